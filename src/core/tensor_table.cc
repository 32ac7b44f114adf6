#include "core/tensor_table.h"

namespace nb {

std::vector<TableLaunch> pack_tensors(const uint64_t* sizes, size_t count, int room, unsigned chunk) {
  constexpr uint64_t kMost = (1ull << 31) - 1;
  std::vector<TableLaunch> out;
  for (size_t i = 0; i < count; ++i) {
    if (!sizes[i]) continue;
    const uint64_t chunks = (sizes[i] - 1) / chunk + 1;
    if (chunks > kMost) return {};  // more elements than any device holds
    if (out.empty() || int(out.back().tensor.size()) >= room || out.back().chunks + chunks > kMost)
      out.emplace_back();
    TableLaunch& l = out.back();
    l.tensor.push_back(int(i));
    l.first.push_back(l.chunks);
    l.chunks += unsigned(chunks);
  }
  return out;
}

}  // namespace nb
