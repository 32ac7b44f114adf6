// Root-mean-square norm of a sum: the partial sums of a row-parallel product
// (in one device's memory, in rank order) plus the residual, with the normalised row in
// the input's type or in e4m3 with scales; and its gradient.
//
// These entry points have no counterpart in the reference: they are the work
// that follows an AllReduce of activations, done where the sum is formed.
//
// All pointers are device memory of `device`; the kernels run on `stream`
// (a stream of that device) and allocate nothing, so they can be captured.
// Every call returns 0, -1 for bad arguments or a CUDA error code, and leaves
// a message in `err` (when errcap > 0) for every non-zero return.
#pragma once

#include <cstddef>
#include <cstdint>

extern "C" {

// ncclDataType_t values.
enum { NB_NORM_FLOAT16 = 6, NB_NORM_FLOAT32 = 7, NB_NORM_BFLOAT16 = 9, NB_NORM_FLOAT8E4M3 = 10 };

// Rows are numbered r = o * inner + i; row r of an input starts at
// base + o * outer_stride + i * inner_stride elements. Outputs are contiguous.
struct nb_norm_t {
  const void* x[8];
  int64_t x_outer[8], x_inner[8];
  const void* residual;  // null: none
  int64_t r_outer, r_inner;
  const void* weight;
  void* y;
  float* scale;  // out_dtype e4m3 only: rows x ceil(hidden / group)
  void* h;       // the sum, rounded to dtype; null: not wanted. May be x[0] or the residual (same strides).
  float* rstd;
  int64_t rows, inner;
  int32_t device, hidden, parts, dtype, weight_dtype, out_dtype, group;  // group 0: one scale per row
  float eps;
};
int nb_add_rms_norm(const nb_norm_t* a, void* stream, char* err, size_t errcap);

struct nb_norm_grad_t {
  const void* dy;
  int64_t dy_outer, dy_inner;
  const void* h;
  int64_t h_outer, h_inner;
  const void* dh;  // gradient of the sum from elsewhere (the residual stream); null: none
  int64_t dh_outer, dh_inner;
  const void* weight;
  const float* rstd;
  void* dx;
  void* dweight;     // weight_dtype
  float* workspace;  // nb_add_rms_norm_backward_workspace() bytes
  uint64_t workspace_bytes;
  int64_t rows, inner;
  int32_t device, hidden, dtype, weight_dtype;
};
int nb_add_rms_norm_backward(const nb_norm_grad_t* a, void* stream, char* err, size_t errcap);
// Bytes of workspace for these sizes on `device`, whatever the strides and alignment.
uint64_t nb_add_rms_norm_backward_workspace(int device, int64_t rows, int hidden, int dtype);
}
