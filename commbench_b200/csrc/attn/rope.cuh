// Rotation of pairs by position, shared by the rotary operator and the cache writer.
#pragma once
#include <stdint.h>

namespace cb {

struct RopeTableView {
  const float* cos;   // [positions, rot / 2]
  const float* sin;
  int positions, rot, interleaved;
};

// (a, b) -> (a c - b s, b c + a s)
__device__ __forceinline__ void rotate_pair(float a, float b, float c, float s, float* ya, float* yb) {
  *ya = a * c - b * s;
  *yb = b * c + a * s;
}

}  // namespace cb
