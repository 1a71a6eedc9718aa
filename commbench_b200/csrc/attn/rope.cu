// Rotary positions: pairs of a head's first `rot` elements are turned by an angle that depends on the position,
//   (a, b) -> (a c - b s, b c + a s),   (c, s) = row `position` of a table,
// the others are copied.  Pairs are (i, i + rot / 2) or (2 i, 2 i + 1).  The transpose (s -> -s) is the gradient.
//
// Bound by memory: one read and one write of x.  The table is fp32 made in 64 bits - an angle of 10^5 turns
// computed in fp32 would be off by a percent of a turn - and a thread uses its entries for several heads, whose loads
// are in flight together.
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
  RopeShare share;
  uint32_t* status;
};

static constexpr int ROPE_THREADS = 256;
// Heads whose loads a thread has in flight.  16384 tokens, 32 + 8 heads of 128 bf16 / the interleaved half of 2 x 2047
// tokens, 16 + 16 heads: 2 heads 98 / -, 3 (64 registers, 4 CTAs an SM) 62.4 / 15.8, 4 (80, 3) 58.9 / 13.0, 8 (128, 2) 56.7 /
// 13.1 us, which is 6.07 TB/s, 0.93 of a copy's.
static constexpr int ROPE_HEADS = 8;

template <class T, int V, bool kHalf>
__global__ void __launch_bounds__(ROPE_THREADS, 2) rope_kernel(const __grid_constant__ RopeParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const RopeShare& sh = p.share;
  const int per_token = sh.lanes * sh.head_lanes;
  const int t = threadIdx.x / per_token, in = threadIdx.x - t * per_token;
  const int s = static_cast<int>(blockIdx.x) * sh.tokens + t;
  if (t >= sh.tokens || s >= p.S) return;
  const int hy = in / sh.lanes, lane = in - hy * sh.lanes;
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
  const long long tok = static_cast<long long>(b) * p.S + s;
  const long long pi = p.pos_batched ? tok : s;
  const long long pos = p.pos_i64 ? static_cast<const long long*>(p.pos)[pi] : static_cast<const int*>(p.pos)[pi];
  if ((pos < 0 || pos >= p.table.positions) && in == 0) report_status(p.status, CB_BAD_ARGUMENT, 1, 0xA01);
  RopeRows<T> r;
  r.x0 = static_cast<const T*>(p.t[0].x) + b * p.t[0].sb + s * p.t[0].ss;
  r.x1 = static_cast<const T*>(p.t[1].x) + b * p.t[1].sb + s * p.t[1].ss;
  r.y0 = static_cast<T*>(p.t[0].y) + tok * p.t[0].heads * p.D;
  r.y1 = static_cast<T*>(p.t[1].y) + tok * p.t[1].heads * p.D;
  r.sh0 = p.t[0].sh;
  r.sh1 = p.t[1].sh;
  r.heads0 = p.t[0].heads;
  r.heads = r.heads0 + (p.tensors > 1 ? p.t[1].heads : 0);
  r.D = p.D;
  for (int item = lane; item < sh.items; item += sh.lanes)
    rope_item<T, V, kHalf, ROPE_HEADS>(p.table, sh, r, pos, p.sign, hy, item);
  }
}

template <class T, int V, bool kHalf>
static int rope_go(RopeParams p, cudaStream_t st) {
  p.share.set(ROPE_THREADS, p.D, p.table.rot, V, kHalf, p.t[0].heads + (p.tensors > 1 ? p.t[1].heads : 0), ROPE_HEADS);
  const int blocks = (p.S + p.share.tokens - 1) / p.share.tokens;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(p.B < 65535 ? p.B : 65535));
  const cudaError_t e = launch_pdl(rope_kernel<T, V, kHalf>, grid, dim3(ROPE_THREADS), 0, st, p);
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
  p.status = static_cast<uint32_t*>(status);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (type == ELEM_BF16) return rope_typed<__nv_bfloat16>(p, st);
  if (type == ELEM_F16) return rope_typed<__half>(p, st);
  return rope_typed<float>(p, st);
}

}  // extern "C"
