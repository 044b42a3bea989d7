// The rows of a tree of drafted tokens among the rows of a step.
#pragma once

#include "common.hpp"

namespace spk {
namespace draft {

constexpr int kMaxNodes = 1024;

struct Rows {
  int64_t first;
  int count;
};

__device__ __forceinline__ Rows rows_of(const int32_t *starts, int n, int64_t rows, int max_nodes) {
  Rows r;
  r.first = min<int64_t>(max(starts[n], 0), rows);
  const int64_t end = min(max<int64_t>(starts[n + 1], r.first), rows);
  r.count = static_cast<int>(min<int64_t>(end - r.first, max_nodes));
  return r;
}

}  // namespace draft
}  // namespace spk
