// Rotation of pairs by position, shared by the rotary operator and the cache writer.
#pragma once
#include <stdint.h>

#include "../prim/elem.cuh"
#include "../prim/ptx.cuh"
#include "../prim/status.h"

namespace cb {

struct RopeTableView {
  const float* cos;   // [positions, rot / 2]
  const float* sin;
  int positions, rot, interleaved;
};

// (a, b) -> (a c - b s, b c + a s)
__device__ __forceinline__ void rotate_pair(float a, float b, float c, float s, float* ya, float* yb) {
  const float x = a * c - b * s, y = b * c + a * s;
  *ya = x;
  *yb = y;
}

// How the threads of a CTA share its tokens: thread = (token, head lane, item); an item is V elements of both halves
// (half layout), V neighbouring elements (V / 2 pairs; one pair for V = 1), or V elements to copy.  A head lane
// takes heads hy, hy + head_lanes, ...
struct RopeShare {
  int pair_items, items;        // of a head
  int lanes;                    // threads that share a head
  int head_lanes, tokens;       // of a CTA
  __host__ void set(int threads, int D, int rot, int V, bool half, int heads, int U) {
    pair_items = half ? rot / 2 / V : (V == 1 ? rot / 2 : rot / V);
    items = pair_items + (D - rot) / V;
    lanes = items < threads ? items : threads;
    head_lanes = (heads + U - 1) / U;
    if (head_lanes > threads / lanes) head_lanes = threads / lanes;
    tokens = threads / (lanes * head_lanes);
  }
};

// The rows of one token's heads: the q heads of a first tensor, then those of a second.
template <class T>
struct RopeRows {
  const T *x0, *x1;             // head 0 of the token
  T *y0, *y1;
  long long sh0, sh1;           // element strides between heads (of y: D)
  int heads0, heads;
  int D;
  __device__ __forceinline__ const T* src(int h) const { return h < heads0 ? x0 + h * sh0 : x1 + (h - heads0) * sh1; }
  __device__ __forceinline__ T* dst(int h) const {
    return h < heads0 ? y0 + static_cast<long long>(h) * D : y1 + static_cast<long long>(h - heads0) * D;
  }
};

// One item of up to U heads at a time: their loads are in flight together.
template <class T, int V, bool kHalf, int U>
__device__ __forceinline__ void rope_item(const RopeTableView& table, const RopeShare& sh, const RopeRows<T>& r,
                                          long long pos, float sign, int hy, int item) {
  using W = Vec<T, V>;
  constexpr int P = kHalf || V == 1 ? V : V / 2;   // pairs
  constexpr bool kTwo = kHalf || V == 1;           // an item is two pieces
  const int half = table.rot / 2, first = item * P;
  const bool pair = item < sh.pair_items;
  const int d0 = !pair ? table.rot + (item - sh.pair_items) * V : kHalf ? first : 2 * first;
  const int d1 = kHalf ? half + first : d0 + 1;
  W a[U], b[U];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * sh.head_lanes;
      if (h < r.heads) {
        const T* x = r.src(h);
        a[u] = *reinterpret_cast<const W*>(x + d0);
        if (kTwo && pair) b[u] = *reinterpret_cast<const W*>(x + d1);
      }
    }
  };
  fetch(hy);   // before the position is asked for
  const bool known = pos >= 0 && pos < table.positions;
  float c[P], s[P];
#pragma unroll
  for (int i = 0; i < P; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);   // outside the table: NaN
  if (pair && known) {
    load_vec<float, P>(table.cos + pos * half + first, c);
    load_vec<float, P>(table.sin + pos * half + first, s);
#pragma unroll
    for (int i = 0; i < P; ++i) s[i] *= sign;
  }
  for (int h0 = hy; h0 < r.heads; h0 += U * sh.head_lanes) {
    if (h0 != hy) fetch(h0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * sh.head_lanes;
      if (h >= r.heads) break;
      T* y = r.dst(h);
      if (pair) {
        float x[V];
        unpack(a[u], x);
        if constexpr (kTwo) {
          float z[V];
          unpack(b[u], z);
#pragma unroll
          for (int i = 0; i < V; ++i) rotate_pair(x[i], z[i], c[i], s[i], &x[i], &z[i]);
          store_vec<T, V>(y + d1, z);
        } else {
#pragma unroll
          for (int i = 0; i < V; i += 2) rotate_pair(x[i], x[i + 1], c[i / 2], s[i / 2], &x[i], &x[i + 1]);
        }
        pack(x, a[u]);
      }
      *reinterpret_cast<W*>(y + d0) = a[u];
    }
  }
}

}  // namespace cb
