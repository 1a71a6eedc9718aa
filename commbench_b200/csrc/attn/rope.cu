// Rotary positions: pairs of a head's first `rot` elements are turned by an angle that depends on the position,
//   (a, b) -> (a c - b s, b c + a s),   (c, s) = row `position` of a table,
// the others are copied.  Pairs are (i, i + rot / 2) or (2 i, 2 i + 1).  The transpose (s -> -s) is the gradient.
//
// Bound by memory: one read and one write of x.  The table is fp32 made in 64 bits - an angle of 10^5 turns
// computed in fp32 would be off by a percent of a turn - and a thread keeps its entries for all heads of a token.
#include <cuda_runtime.h>

#include <string>

#include "../prim/elem.cuh"
#include "../prim/pdl.cuh"
#include "../prim/ptx.cuh"
#include "../prim/status.h"
#include "rope.cuh"

namespace cb {
void set_last_error(const std::string& s);

struct RopeTensor {
  const void* x;
  void* y;                           // [B, S, heads, D] dense
  long long sb, ss, sh;              // element strides of x
  int heads;
};
struct RopeParams {
  RopeTensor t[2];
  int tensors, B, S, D;
  RopeTableView table;
  const void* pos;                   // [B, S] or, with pos_batched = 0, [S]
  int pos_i64, pos_batched;
  float sign;                        // -1: transpose
  int pair_items, copy_items;        // work items of a head
  uint32_t* status;
};

// A CTA takes tokens in turn; thread = (head of a group of `hy`, item), an item being V elements of both halves
// (kHalf), V neighbouring elements (V / 2 pairs; a pair for V = 1), or V elements to copy.
template <class T, int V, bool kHalf>
__global__ void __launch_bounds__(256) rope_kernel(const __grid_constant__ RopeParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int items = p.pair_items + p.copy_items;
  const int per_pass = items < 256 ? items : 256;
  const int hy_n = 256 / per_pass;
  const int hy = threadIdx.x / per_pass;
  if (hy >= hy_n) return;
  const int half = p.table.rot / 2;
  const long long tokens = static_cast<long long>(p.B) * p.S;
  for (long long tok = blockIdx.x; tok < tokens; tok += gridDim.x) {
    const int b = static_cast<int>(tok / p.S), s = static_cast<int>(tok - static_cast<long long>(b) * p.S);
    const long long pi = p.pos_batched ? tok : s;
    const long long pos = p.pos_i64 ? static_cast<const long long*>(p.pos)[pi] : static_cast<const int*>(p.pos)[pi];
    const bool known = pos >= 0 && pos < p.table.positions;
    if (!known && threadIdx.x == 0) report_status(p.status, CB_BAD_ARGUMENT, 1, 0xA01);
    for (int item = threadIdx.x - hy * per_pass; item < items; item += per_pass) {
      const bool pair = item < p.pair_items;
      constexpr int P = kHalf || V == 1 ? V : V / 2;   // pairs of an item
      float c[P], sn[P];
      const int first = item * P;                      // first pair
      if (pair) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          // outside the table there is no rotation: the answer is NaN, not some other position's
          c[i] = known ? __ldg(p.table.cos + pos * half + first + i) : __int_as_float(0x7fc00000);
          sn[i] = known ? p.sign * __ldg(p.table.sin + pos * half + first + i) : __int_as_float(0x7fc00000);
        }
      }
      for (int k = 0; k < p.tensors; ++k) {
        const RopeTensor& t = p.t[k];
        const T* x0 = static_cast<const T*>(t.x) + b * t.sb + s * t.ss;
        T* y0 = static_cast<T*>(t.y) + tok * t.heads * p.D;
        for (int h = hy; h < t.heads; h += hy_n) {
          const T* x = x0 + h * t.sh;
          T* y = y0 + static_cast<long long>(h) * p.D;
          if (!pair) {
            const int d = p.table.rot + (item - p.pair_items) * V;
            *reinterpret_cast<Vec<T, V>*>(y + d) = *reinterpret_cast<const Vec<T, V>*>(x + d);
          } else if constexpr (kHalf) {
            float a[V], e[V], ya[V], ye[V];
            load_vec<T, V>(x + first, a);
            load_vec<T, V>(x + half + first, e);
#pragma unroll
            for (int i = 0; i < V; ++i) rotate_pair(a[i], e[i], c[i], sn[i], &ya[i], &ye[i]);
            store_vec<T, V>(y + first, ya);
            store_vec<T, V>(y + half + first, ye);
          } else if constexpr (V > 1) {
            float a[V], ya[V];
            load_vec<T, V>(x + 2 * first, a);
#pragma unroll
            for (int i = 0; i < V; i += 2) rotate_pair(a[i], a[i + 1], c[i / 2], sn[i / 2], &ya[i], &ya[i + 1]);
            store_vec<T, V>(y + 2 * first, ya);
          } else {
            float ya, yb;
            rotate_pair(to_f32(x[2 * first]), to_f32(x[2 * first + 1]), c[0], sn[0], &ya, &yb);
            y[2 * first] = from_f32<T>(ya);
            y[2 * first + 1] = from_f32<T>(yb);
          }
        }
      }
    }
  }
}

template <class T, int V, bool kHalf>
static int rope_go(RopeParams p, cudaStream_t st) {
  const int rot = p.table.rot;
  p.pair_items = kHalf ? rot / 2 / V : (V == 1 ? rot / 2 : rot / V);
  p.copy_items = (p.D - rot) / V;
  const long long tokens = static_cast<long long>(p.B) * p.S;
  const unsigned grid = static_cast<unsigned>(tokens < 148 * 32 ? tokens : 148 * 32);
  const cudaError_t e = launch_pdl(rope_kernel<T, V, kHalf>, dim3(grid), dim3(256), 0, st, p);
  if (e != cudaSuccess) {
    cudaGetLastError();   // reported here, not by the next call
    set_last_error(std::string("rope launch: ") + cudaGetErrorString(e));
    return -1;
  }
  return 0;
}

template <class T>
static int rope_typed(const RopeParams& p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int rot = p.table.rot;
  bool wide = p.D % V == 0 && (p.table.interleaved ? rot % V == 0 : rot % (2 * V) == 0);
  for (int k = 0; k < p.tensors; ++k) {
    const RopeTensor& t = p.t[k];
    wide = wide && reinterpret_cast<uintptr_t>(t.x) % 16 == 0 && reinterpret_cast<uintptr_t>(t.y) % 16 == 0 &&
           t.sb % V == 0 && t.ss % V == 0 && t.sh % V == 0;
  }
  if (p.table.interleaved) return wide ? rope_go<T, V, false>(p, st) : rope_go<T, 1, false>(p, st);
  return wide ? rope_go<T, V, true>(p, st) : rope_go<T, 1, true>(p, st);
}

}  // namespace cb

using namespace cb;

extern "C" {

// One or two tensors [B, S, heads, D] (strides in elements, last one 1) -> dense y of the same type.
int cb_rope(const void* x0, void* y0, long long sb0, long long ss0, long long sh0, int heads0, const void* x1, void* y1,
            long long sb1, long long ss1, long long sh1, int heads1, int B, int S, int D, const void* cos,
            const void* sin, int positions, int rot, int interleaved, const void* pos, int pos_i64, int pos_batched,
            int inverse, int type, void* status, void* stream) {
  if (B < 0 || S < 0 || D < 1 || heads0 < 1 || rot < 2 || rot % 2 != 0 || rot > D || type < 0 || type > 2 ||
      (x1 != nullptr && heads1 < 1)) {
    set_last_error("rope: bad shape or type (an even number of elements, at most the head's, is turned)");
    return -1;
  }
  if (B == 0 || S == 0) return 0;
  RopeParams p;
  p.t[0] = {x0, y0, sb0, ss0, sh0, heads0};
  p.t[1] = {x1, y1, sb1, ss1, sh1, heads1};
  p.tensors = x1 != nullptr ? 2 : 1;
  p.B = B;
  p.S = S;
  p.D = D;
  p.table = {static_cast<const float*>(cos), static_cast<const float*>(sin), positions, rot, interleaved};
  p.pos = pos;
  p.pos_i64 = pos_i64;
  p.pos_batched = pos_batched;
  p.sign = inverse ? -1.f : 1.f;
  p.pair_items = p.copy_items = 0;
  p.status = static_cast<uint32_t*>(status);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (type == ELEM_BF16) return rope_typed<__nv_bfloat16>(p, st);
  if (type == ELEM_F16) return rope_typed<__half>(p, st);
  return rope_typed<float>(p, st);
}

}  // extern "C"
