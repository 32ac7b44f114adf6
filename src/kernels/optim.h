// One AdamW step, and the gradients' norm, over many tensors at once.
//
// These entry points have no counterpart in the reference: they are the work
// that follows a ReduceScatter or AllReduce of gradients. A gradient may be
// given as 1 to 8 partial ones in the device's memory (per micro-batch or rank), which the
// kernels add in order, in fp32, as the collectives fold them.
//
// A handle describes tensors of one device; it holds their addresses, not the
// memory, and no device memory of its own. Steps run on the stream given (of
// that device), allocate nothing and can be captured. A handle may be used
// from several threads. Functions that return an int give 0, -1 for bad
// arguments or a CUDA error code, and leave a message in `err` (when
// errcap > 0) for every failure; a create that fails returns null.
#pragma once

#include <cstddef>
#include <cstdint>

extern "C" {

// ncclDataType_t values.
enum { NB_OPTIM_FLOAT16 = 6, NB_OPTIM_FLOAT32 = 7, NB_OPTIM_BFLOAT16 = 9, NB_OPTIM_FLOAT8E4M3 = 10 };

// Elements that share a scale in the 8-bit states; a tensor of n elements has
// ceil(n / 256) scales per state.
enum { NB_OPTIM_BLOCK = 256 };

// `count` tensors; every table has one address per tensor except `grad`,
// which has `parts` (tensor i's are grad[i * parts ...]).
struct nb_adamw_t {
  int32_t device, count, parts;
  int32_t param_dtype;  // fp16, bf16 or fp32
  int32_t grad_dtype;   // fp16, bf16 or fp32
  int32_t copy_dtype;   // fp16 or bf16: a rounded copy of fp32 parameters is written too; 0: none
  int32_t state_dtype;  // fp32, or e4m3 with scales
  uint32_t seed;        // of the 8-bit states' rounding
  const uint64_t* size;
  void* const* param;
  void* const* copy;              // null without copy_dtype
  const void* const* grad;
  void* const* m;
  void* const* v;
  float* const* m_scale;          // e4m3 only
  float* const* v_scale;
  const float* weight_decay;      // per tensor
  double beta1, beta2, eps;
};
void* nb_adamw_create(const nb_adamw_t* a, char* err, size_t errcap);
// Step number t >= 1, learning rate and gradient scale; each may instead be
// read on the device (t_dev: int64, the others float), and the device's scale
// multiplies `scale`. A scale, or an lr / (1 - beta1^t), that is not finite when
// the kernel runs leaves every tensor as it was; t below 1 on the device counts as 1.
int nb_adamw_step(const void* handle, int64_t t, const int64_t* t_dev, double lr, const float* lr_dev, double scale,
                  const float* scale_dev, void* stream, char* err, size_t errcap);
void nb_adamw_destroy(void* handle);

void* nb_grad_norm_create(int device, int count, int parts, int dtype, const uint64_t* size,
                          const void* const* grad, char* err, size_t errcap);
// Doubles of workspace for one call.
int nb_grad_norm_partials(const void* handle);
// out[0] = scale * sqrt(sum of squares), out[1] = scale * min(1, max_norm / (out[0] + 1e-6)), or
// NaN where out[0] is not finite (a step that takes it as its scale is skipped). A root above
// 2^126 counts as infinite.
int nb_grad_norm(const void* handle, double max_norm, double scale, float* out, double* workspace, void* stream,
                 char* err, size_t errcap);
void nb_grad_norm_destroy(void* handle);
}
