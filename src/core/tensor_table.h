// The work list of a kernel over many tensors: which tensor, and which part
// of it, each chunk of a launch covers. Shared by the kernels, the host that
// packs the launches, and the CPU tests.
//
// A tensor of n elements is ceil(n / chunk) chunks; a launch numbers the
// chunks of its tensors one after another. The list travels in the launch's
// parameters (32764 bytes at most on sm_100), so a step needs no copy, no
// device table that a captured graph could outlive, and no workspace; tensors
// beyond one launch's room go to the next launch.
#pragma once

#include <cstddef>
#include <cstdint>
#include <vector>

#ifdef __CUDACC__
#define NB_TT_HD __host__ __device__ __forceinline__
#else
#define NB_TT_HD inline
#endif

namespace nb {

// The tensor of chunk `c`: the last of `count` whose first chunk is not above
// it. `first(i)` gives tensor i's first chunk; first(0) is 0, and a tensor
// without elements (which shares its successor's first chunk) is never chosen
// because it is not listed.
template <typename First>
NB_TT_HD int find_tensor(unsigned c, int count, First first) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first(mid) <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

struct TableLaunch {
  std::vector<int> tensor;         // indexes into the caller's list
  std::vector<unsigned> first;     // each one's first chunk
  unsigned chunks = 0;
};

// Splits the tensors (in order, those without elements left out) into
// launches of at most `room` tensors and fewer than 2^31 chunks.
std::vector<TableLaunch> pack_tensors(const uint64_t* sizes, size_t count, int room, unsigned chunk);

}  // namespace nb
