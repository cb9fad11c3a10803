// A [B, H, S, D] bf16 tensor by its element strides; D is contiguous.
#pragma once

#include <cstdint>

namespace b200 {

struct View {
  uint16_t* p;
  int64_t sb, sh, ss;
  __device__ __forceinline__ uint16_t* row(int64_t b, int64_t h, int64_t s) const {
    return p + b * sb + h * sh + s * ss;
  }
};

}  // namespace b200
