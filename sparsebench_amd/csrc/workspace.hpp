// The workspaces of the calls that run a whole layer (layer.hip,
// gated_layer.hip): one buffer of the caller's, cut into pieces.
#pragma once

#include "common.hpp"

namespace sb {

constexpr int64_t kI32Limit = int64_t{1} << 31;

// Hands out 256-byte aligned pieces of a workspace; with no base it only adds up.
struct Carver {
  uint8_t* base;
  int64_t used = 0;
  template <class T>
  T* take(int64_t count) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += (count * static_cast<int64_t>(sizeof(T)) + 255) / 256 * 256;
    return p;
  }
};

inline int check_workspace(const void* workspace, int64_t workspace_bytes, int64_t needed) {
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return fail(SB_ERR_INVALID, "layer: the workspace must be 256-byte aligned");
  if (workspace_bytes < needed)
    return fail(SB_ERR_INVALID, "layer: workspace of %lld bytes, %lld needed", static_cast<long long>(workspace_bytes),
                static_cast<long long>(needed));
  return SB_OK;
}

}  // namespace sb
