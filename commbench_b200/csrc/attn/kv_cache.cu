// Writing and reading the paged 8-bit key/value cache (kv_cache.cuh).
//
// Append, one launch: a CTA takes one (sequence, page, head), reads the new tokens of that page once, turns the
// keys by their positions, finds the block's exponent and writes the e4m3 rows; other CTAs of the launch turn the
// queries.  Bound by memory for prompts (2 bytes an element read, 1 written), by latency for a decode step.
#include <cuda_runtime.h>

#include <string>

#include "../prim/elem.cuh"
#include "../prim/pdl.cuh"
#include "../prim/ptx.cuh"
#include "../prim/status.h"
#include "kv_cache.cuh"
#include "rope.cuh"

namespace cb {
void set_last_error(const std::string& s);

struct KvAppendParams {
  KvCacheView cache;
  KvBatch batch;
  const __nv_bfloat16 *k, *v, *q;                   // q or null
  __nv_bfloat16* q_out;                             // [B, S, hq, 128] dense
  long long k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, q_sb, q_ss, q_sh;
  RopeTableView rope;                               // rot = 0: none
  int hq, pages_per_seq, kv_blocks;
  int wide;                                         // queries in vectors of 8 elements, else of 4
  RopeShare share;                                  // of the queries
  uint32_t* status;
};

// The lane's four elements d = 4 lane .. 4 lane + 3 of a head at `pos`, turned.  Warp-collective.
struct LaneAngles {
  float c[4], s[4];
  bool low;          // elements of the first half (half layout)
  int partner;       // lane that holds the other elements of the pairs
  bool on;
};
__device__ __forceinline__ LaneAngles lane_angles(const RopeTableView& t, long long pos, int lane) {
  LaneAngles a;
  const int d = 4 * lane, half = t.rot / 2;
  a.on = d < t.rot;
  a.low = d < half;
  a.partner = t.interleaved || !a.on ? lane : a.low ? lane + half / 4 : lane - half / 4;
  const bool known = pos >= 0 && pos < t.positions;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a.c[i] = a.s[i] = __int_as_float(0x7fc00000);
    if (a.on && known) {
      const long long at = pos * half + (t.interleaved ? (d + i) / 2 : (a.low ? d : d - half) + i);
      a.c[i] = __ldg(t.cos + at);
      a.s[i] = __ldg(t.sin + at);
    }
  }
  return a;
}
__device__ __forceinline__ void lane_rotate(const RopeTableView& t, const LaneAngles& a, float (&x)[4]) {
  float y[4];
  if (t.interleaved) {
    rotate_pair(x[0], x[1], a.c[0], a.s[0], &y[0], &y[1]);
    rotate_pair(x[2], x[3], a.c[2], a.s[2], &y[2], &y[3]);
  } else {
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __shfl_sync(0xffffffffu, x[i], a.partner);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float lo, hi;
      rotate_pair(a.low ? x[i] : o[i], a.low ? o[i] : x[i], a.c[i], a.s[i], &lo, &hi);
      y[i] = a.low ? lo : hi;
    }
  }
  if (a.on) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = y[i];
  }
}

static constexpr int KV_THREADS = 512;
static constexpr int KV_WARPS = KV_THREADS / 32;
static constexpr int KV_Q_HEADS = 2;   // query heads whose loads a thread has in flight

// The queries of p.share.tokens tokens.
template <int V, bool kHalf>
__device__ __forceinline__ void append_queries(const KvAppendParams& p, int block) {
  const RopeShare& sh = p.share;
  const int per_token = sh.lanes * sh.head_lanes;
  const int t = threadIdx.x / per_token, in = threadIdx.x - t * per_token;
  const long long tok = static_cast<long long>(block) * sh.tokens + t;
  if (t >= sh.tokens || tok >= static_cast<long long>(p.batch.B) * p.batch.S) return;
  const int hy = in / sh.lanes, lane = in - hy * sh.lanes;
  const int b = static_cast<int>(tok / p.batch.S), i = static_cast<int>(tok - static_cast<long long>(b) * p.batch.S);
  __nv_bfloat16* dst = p.q_out + tok * p.hq * KV_D;
  if (i >= p.batch.new_tokens(b)) {      // padding: zeros
    for (int d = in * 4; d < p.hq * KV_D; d += per_token * 4) *reinterpret_cast<uint2*>(dst + d) = make_uint2(0u, 0u);
    return;
  }
  RopeRows<__nv_bfloat16> r;
  r.x0 = r.x1 = p.q + b * p.q_sb + i * p.q_ss;
  r.y0 = r.y1 = dst;
  r.sh0 = r.sh1 = p.q_sh;
  r.heads0 = r.heads = p.hq;
  r.D = KV_D;
  const long long pos = static_cast<long long>(p.batch.start[b]) + i;
  for (int item = lane; item < sh.items; item += sh.lanes)
    rope_item<__nv_bfloat16, V, kHalf, KV_Q_HEADS>(p.rope, sh, r, pos, 1.f, hy, item);
}

// kTokens: token slots of a page per warp.
template <int kTokens>
__global__ void __launch_bounds__(KV_THREADS, kTokens <= 4 ? 2 : 1) kv_append_kernel(const __grid_constant__ KvAppendParams p) {
  __shared__ float sh_max[2][KV_WARPS];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (static_cast<int>(blockIdx.x) >= p.kv_blocks) {
    const int block = static_cast<int>(blockIdx.x) - p.kv_blocks;
    if (p.rope.interleaved)
      p.wide ? append_queries<8, false>(p, block) : append_queries<4, false>(p, block);
    else
      p.wide ? append_queries<8, true>(p, block) : append_queries<4, true>(p, block);
    return;
  }
  const int hkv = p.cache.hkv, page = p.cache.page();
  const int head = blockIdx.x % hkv, rest = blockIdx.x / hkv;
  const int b = rest / p.pages_per_seq;
  const int start = p.batch.start[b], count = p.batch.new_tokens(b);
  if (count == 0) return;
  const long long col = (start >> p.cache.page_log2) + static_cast<long long>(rest - b * p.pages_per_seq);
  const long long t0 = col << p.cache.page_log2;                   // first token of the page
  if (t0 >= static_cast<long long>(start) + count) return;
  const int pid = start >= 0 && col < p.batch.cols ? p.batch.pages[static_cast<long long>(b) * p.batch.cols + col] : -1;
  if (pid < 0 || pid >= p.cache.num_pages) {
    if (threadIdx.x == 0) report_status(p.status, CB_BAD_ARGUMENT, 2, 0xA02);
    return;
  }
  const int lo = start > t0 ? static_cast<int>(start - t0) : 0;     // slots lo .. hi - 1 are new
  const long long left = static_cast<long long>(start) + count - t0;
  const int hi = left < page ? static_cast<int>(left) : page;

  // Values first: a NaN among them is stored as 0 and put into the token's key instead, so that a query that
  // does not see the token has nothing to multiply by zero, and one that does answers NaN.
  uint32_t bad = 0;                                                 // bit per token of the warp
#pragma unroll 1
  for (int side = 1; side >= 0; --side) {
    const __nv_bfloat16* src = side ? p.v + b * p.v_sb + head * p.v_sh : p.k + b * p.k_sb + head * p.k_sh;
    const long long ss = side ? p.v_ss : p.k_ss;
    float x[kTokens][4];
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      const int t = warp + KV_WARPS * i;
      x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
      if (t >= lo && t < hi) load_vec<__nv_bfloat16, 4>(src + (t0 + t - start) * ss + 4 * lane, x[i]);
    }
    if (side == 0 && p.rope.rot > 0) {
#pragma unroll
      for (int i = 0; i < kTokens; ++i) {
        const int t = warp + KV_WARPS * i;
        if (t >= lo && t < hi) {
          if (t0 + t >= p.rope.positions && lane == 0) report_status(p.status, CB_BAD_ARGUMENT, 1, 0xA01);
          lane_rotate(p.rope, lane_angles(p.rope, t0 + t, lane), x[i]);
        }
      }
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      if (side == 1) {
        bool nan = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          nan = nan || x[i][j] != x[i][j];
          if (x[i][j] != x[i][j]) x[i][j] = 0.f;
        }
        if (__any_sync(0xffffffffu, nan)) bad |= 1u << i;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = fabsf(x[i][j]);
        amax = fmaxf(amax, a <= 3.4028234e38f ? a : 0.f);           // infinities become the largest number
      }
    }
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    if (lane == 0) sh_max[side][warp] = amax;
    __syncthreads();
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(sh_max[side][lane & (KV_WARPS - 1)])));
    int8_t* exp_at = p.cache.exp_of(pid, head, side);
    int e = kv_exponent(amax), e_old = e;
    if (lo > 0) {
      e_old = *exp_at;
      e = e > e_old ? e : e_old;
    }
    uint8_t* tile = p.cache.tile(pid, head, side);
    if (e != e_old) {
      const float f = kv_pow2(e_old - e < -126 ? -126 : e_old - e);
      for (int t = warp; t < lo; t += KV_WARPS) {
        uint32_t* at = reinterpret_cast<uint32_t*>(tile + kv_offset(t, 4 * lane));
        const uint32_t old = *at;
        const uint32_t h0 = kv_to_half2(old), h1 = kv_to_half2(old >> 16);
        const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
        const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
        *at = kv_encode4(f0.x * f, f0.y * f, f1.x * f, f1.y * f);
      }
    }
    const float inv = e == KV_EXP_MIN ? 0.f : kv_pow2(-e);          // the least exponent says: all zero
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      const int t = warp + KV_WARPS * i;
      if (t >= lo && t < hi) {
        if (side == 0 && lane == 0 && ((bad >> i) & 1u)) x[i][0] = __int_as_float(0x7fc00000);
        *reinterpret_cast<uint32_t*>(tile + kv_offset(t, 4 * lane)) =
            kv_encode4(x[i][0] * inv, x[i][1] * inv, x[i][2] * inv, x[i][3] * inv);
      }
    }
    if (lo > 0) __syncthreads();   // every warp has read the old exponent
    if (threadIdx.x == 0) *exp_at = static_cast<int8_t>(e);
  }
}

struct KvReadParams {
  KvCacheView cache;
  const int* pages;
  const int* begin;            // [B] or null: 0
  const int* length;           // [B] or null: tokens from here on are zeros
  __nv_bfloat16 *k, *v;        // [B, n, hkv, 128]
  int B, n, cols;
  uint32_t* status;
};

// A thread expands one chunk of 16 elements of a token's key and of its value.
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvReadParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int hkv = p.cache.hkv;
  const long long total = static_cast<long long>(p.B) * p.n * hkv * 8;
  for (long long idx = blockIdx.x * 256ll + threadIdx.x; idx < total; idx += gridDim.x * 256ll) {
    const int chunk = static_cast<int>(idx & 7);
    const long long row = idx >> 3;                     // (b, i, head)
    const int head = static_cast<int>(row % hkv);
    const long long bi = row / hkv;
    const int b = static_cast<int>(bi / p.n);
    const long long t = (p.begin != nullptr ? p.begin[b] : 0) + (bi - static_cast<long long>(b) * p.n);
    uint4 rk = make_uint4(0, 0, 0, 0), rv = rk;
    float sk = 0.f, sv = 0.f;
    if (t >= 0 && (p.length == nullptr || t < p.length[b])) {
      const long long col = t >> p.cache.page_log2;
      const int pid = col < p.cols ? p.pages[static_cast<long long>(b) * p.cols + col] : -1;
      if (pid >= 0 && pid < p.cache.num_pages) {
        const int slot = static_cast<int>(t & (p.cache.page() - 1));
        const int off = kv_offset(slot, chunk * 16);
        rk = *reinterpret_cast<const uint4*>(p.cache.tile(pid, head, 0) + off);
        rv = *reinterpret_cast<const uint4*>(p.cache.tile(pid, head, 1) + off);
        sk = kv_pow2(*p.cache.exp_of(pid, head, 0));
        sv = kv_pow2(*p.cache.exp_of(pid, head, 1));
      } else {
        report_status(p.status, CB_BAD_ARGUMENT, 2, 0xA03);
      }
    }
    kv_expand16(rk, sk, p.k + row * KV_D + chunk * 16);
    kv_expand16(rv, sv, p.v + row * KV_D + chunk * 16);
  }
}

static bool kv_view(KvCacheView* c, void* data, void* exps, int num_pages, int hkv, int page) {
  int lg = 0;
  while ((1 << lg) < page) ++lg;
  *c = {static_cast<uint8_t*>(data), static_cast<int8_t*>(exps), num_pages, hkv, lg};
  if (num_pages >= 1 && hkv >= 1 && page >= 16 && page <= 128 && (1 << lg) == page) return true;
  set_last_error("key/value cache: pages of 16, 32, 64 or 128 tokens, at least one page and head");
  return false;
}

}  // namespace cb

using namespace cb;

extern "C" {

// Strides in elements; k, v, q [B, S, heads, 128] bf16 with rows of 8-byte alignment.  start [B]; count [B] or null.
int cb_kv_append(void* data, void* exps, int num_pages, int hkv, int page, const void* k, const void* v,
                 const long long* strides /* k_sb k_ss k_sh v_sb v_ss v_sh q_sb q_ss q_sh */, const void* pages,
                 int cols, const void* start, const void* count, int B, int S, const void* q, void* q_out, int hq,
                 const void* cos, const void* sin, int positions, int rot, int interleaved, void* status,
                 void* stream) {
  KvAppendParams p;
  if (!kv_view(&p.cache, data, exps, num_pages, hkv, page)) return -1;
  if (B < 0 || S < 0 || cols < 1 || (q != nullptr && hq < 1) || rot < 0 || rot > KV_D || rot % 8 != 0) {
    set_last_error("key/value cache: bad shape (a multiple of 8 elements, at most 128, is turned)");
    return -1;
  }
  if (B == 0 || S == 0) return 0;
  p.batch = {static_cast<const int*>(pages), static_cast<const int*>(start), static_cast<const int*>(count), B, S, cols};
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.k_sb = strides[0], p.k_ss = strides[1], p.k_sh = strides[2];
  p.v_sb = strides[3], p.v_ss = strides[4], p.v_sh = strides[5];
  p.q_sb = strides[6], p.q_ss = strides[7], p.q_sh = strides[8];
  p.rope = {static_cast<const float*>(cos), static_cast<const float*>(sin), positions, rot, interleaved};
  p.hq = hq;
  p.pages_per_seq = (S + page - 2) / page + 1;
  p.status = static_cast<uint32_t*>(status);
  const long long kv_blocks = static_cast<long long>(B) * p.pages_per_seq * hkv;
  p.wide = rot % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(q_out) % 16 == 0 &&
           p.q_sb % 8 == 0 && p.q_ss % 8 == 0 && p.q_sh % 8 == 0;
  p.share = {};
  long long q_blocks = 0;
  if (q != nullptr) {
    p.share.set(KV_THREADS, KV_D, rot, p.wide ? 8 : 4, !interleaved, hq, KV_Q_HEADS);
    q_blocks = (static_cast<long long>(B) * S + p.share.tokens - 1) / p.share.tokens;
  }
  const long long blocks = kv_blocks + q_blocks;
  if (blocks > 0x7fffffffll) {
    set_last_error("key/value cache: too many tokens in one call");
    return -1;
  }
  p.kv_blocks = static_cast<int>(kv_blocks);
  const dim3 grid(static_cast<unsigned>(blocks)), block(KV_THREADS);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (page) {
    case 16: e = launch_pdl(kv_append_kernel<1>, grid, block, 0, st, p); break;
    case 32: e = launch_pdl(kv_append_kernel<2>, grid, block, 0, st, p); break;
    case 64: e = launch_pdl(kv_append_kernel<4>, grid, block, 0, st, p); break;
    default: e = launch_pdl(kv_append_kernel<8>, grid, block, 0, st, p); break;
  }
  if (e != cudaSuccess) {
    cudaGetLastError();   // reported here, not by the next call
    set_last_error(std::string("key/value append launch: ") + cudaGetErrorString(e));
    return -1;
  }
  return 0;
}

// Tokens begin[b] .. begin[b] + n - 1 of each sequence as bf16 [B, n, hkv, 128]; zeros before token 0 and from
// token length[b] on.
int cb_kv_read(const void* data, const void* exps, int num_pages, int hkv, int page, const void* pages, int cols,
               const void* begin, const void* length, int B, int n, void* k, void* v, void* status, void* stream) {
  KvReadParams p;
  if (!kv_view(&p.cache, const_cast<void*>(data), const_cast<void*>(exps), num_pages, hkv, page)) return -1;
  if (B < 0 || n < 0 || cols < 1) {
    set_last_error("key/value cache: bad shape");
    return -1;
  }
  if (B == 0 || n == 0) return 0;
  p.pages = static_cast<const int*>(pages);
  p.begin = static_cast<const int*>(begin);
  p.length = static_cast<const int*>(length);
  p.k = static_cast<__nv_bfloat16*>(k);
  p.v = static_cast<__nv_bfloat16*>(v);
  p.B = B;
  p.n = n;
  p.cols = cols;
  p.status = static_cast<uint32_t*>(status);
  const long long blocks = (static_cast<long long>(B) * n * hkv * 8 + 255) / 256;
  const unsigned grid = static_cast<unsigned>(blocks < 148 * 32 ? blocks : 148 * 32);
  const cudaError_t e = launch_pdl(kv_read_kernel, dim3(grid), dim3(256), 0, static_cast<cudaStream_t>(stream), p);
  if (e != cudaSuccess) {
    cudaGetLastError();   // reported here, not by the next call
    set_last_error(std::string("key/value read launch: ") + cudaGetErrorString(e));
    return -1;
  }
  return 0;
}

}  // extern "C"
