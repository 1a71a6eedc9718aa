// Attention of a few query tokens per sequence over the paged 8-bit cache (kv_cache.cuh): decode steps, draft
// verification, short chunks.
//
//   s_ij = scale q_i . k_j   for the keys j that query i (position p_i) sees: j <= p_i, and with a window
//   j > p_i - window or j < sinks;   o_i = sum_j softmax(s_i)_j v_j;   lse_i = log sum_j exp(s_ij)
//
// What it has to read is the visible part of the cache, 256 bytes a token and head; 16 query rows a key/value head
// want 4096 multiply-adds a token, an eighth of what the tensor cores of an SM do with mma.sync while those bytes
// arrive.  So the tiles are small and every warp works by itself, without a barrier in the loop:
//   * the rows of a tile are 16 (query token, head of the group) couples of one key/value head, so keys are read
//     once for the heads of a group;
//   * a warp takes units of 32 keys from a ring of its own in shared memory, filled by bulk copies that its own
//     lanes issue: the memory system sees 8 KB pieces, and a slot is free again when the warp has read it;
//   * e4m3 becomes fp16 in registers (exactly), scores and products are fp32, probabilities fp16.  With that the
//     scales never touch the data: the key scale is a factor on the score, and the value scale 2^e is the term e in
//     the exponent of the probability, which the running maximum covers too - the sum of the softmax takes it out
//     again per block;
//   * the running maximum is raised only when a score passes it by 2^8;
//   * the work is the flat list of (sequence, head, row tile, unit), cut evenly over the CTAs by the lengths that
//     the device holds: the host needs no lengths, a call can be captured in a graph.  The warps of a CTA merge
//     in shared memory, items that were cut over CTAs in a second small kernel, in the order of the keys.
#include <cuda_runtime.h>
#include <math.h>

#include <string>

#include "../gemm/launch.h"
#include "../prim/mbarrier.cuh"
#include "../prim/pdl.cuh"
#include "../prim/tma.cuh"
#include "kv_cache.cuh"

namespace cb {
void set_last_error(const std::string& s);

static constexpr int KA_UNIT = 32;                     // keys
static constexpr int KA_WARPS = 8;
static constexpr int KA_STAGES = 3;
static constexpr int KA_SIDE = KA_UNIT * KV_D;         // bytes of a unit's keys (and of its values)
static constexpr int KA_RING = KA_WARPS * KA_STAGES * 2 * KA_SIDE;
static constexpr int KA_MAX_B = 1024;
static constexpr float KA_RAISE = 8.f;
static constexpr int KA_MERGE_THREADS = 128;

struct KvAttendParams {
  KvCacheView cache;
  KvBatch batch;
  const __nv_bfloat16* q;
  long long q_sb, q_ss, q_sh;
  __nv_bfloat16* o;              // [B, S, Hq, 128]
  float* lse;                    // [B, Hq, S]
  float* part_o;                 // [CTA][taken over / handed on][tile row][128], unnormalised
  float2* part_ml;               // [CTA][taken over / handed on][tile row] {max (log2 units), sum}
  uint32_t* plan;                // [B + 2]: units before each sequence, units per CTA
  int Hq, group, row_tiles, window, sinks;
  float scale_log2;
  uint32_t* status;
};

struct KaShared {
  uint64_t full[KA_WARPS][KA_STAGES];
  uint32_t base[KA_MAX_B + 1];   // units before each sequence
  uint32_t sums[KA_WARPS];
  float2 ml[KA_WARPS][16];
  int abort_flag;
};
static constexpr int KA_SMEM = KA_RING + static_cast<int>(sizeof(KaShared));

// The units that some query of a sequence sees: the first `sink_units`, then `first` and on; n in all.
struct KaSpan {
  int start, count, end;         // tokens before, new tokens, tokens that exist
  int sink_units, first, n;
};
__device__ __forceinline__ KaSpan ka_span(const KvAttendParams& p, int b) {
  KaSpan s;
  s.start = p.batch.start[b];
  s.count = p.batch.new_tokens(b);
  if (s.start < 0) s.start = 0, s.count = 0;
  s.end = s.start + s.count;
  const int units = (s.end + KA_UNIT - 1) / KA_UNIT;
  s.sink_units = 0;
  s.first = 0;
  if (p.window > 0) {
    const int low = s.start - p.window + 1;            // the first key that the first query's window holds
    s.first = low > 0 ? low / KA_UNIT : 0;
    s.sink_units = (p.sinks + KA_UNIT - 1) / KA_UNIT;
    if (s.sink_units > s.first) s.sink_units = s.first;
  }
  s.n = s.count > 0 ? s.sink_units + units - s.first : 1;   // without a query: one unit, all hidden
  return s;
}

__device__ __forceinline__ float ka_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ka_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ka_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ka_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t ka_half2(float lo, float hi) {
  uint32_t h;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(hi), "f"(lo));
  return h;
}

// The value exponent of a unit's first or second 16 keys.  A block whose values are all zero has the least one; it
// only counts in the sum of the probabilities, and they would be flushed with it.
__device__ __forceinline__ int ka_value_exp(int exps, int h) {
  const int e = static_cast<int8_t>(exps >> (16 * h + 8));
  return e == KV_EXP_MIN ? 0 : e;
}

// Units before each sequence into sh.base, and the units per CTA.  Every CTA does this for itself.
__device__ __forceinline__ uint32_t ka_plan(const KvAttendParams& p, KaShared& sh) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const uint32_t items = static_cast<uint32_t>(p.cache.hkv) * p.row_tiles;
  uint32_t before = 0;
  for (int b0 = 0; b0 < p.batch.B; b0 += KA_WARPS * 32) {
    const int b = b0 + t;
    const uint32_t mine = b < p.batch.B ? static_cast<uint32_t>(ka_span(p, b).n) * items : 0u;
    uint32_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sh.sums[warp] = x;
    __syncthreads();
    uint32_t off = before, all = 0;
#pragma unroll
    for (int w = 0; w < KA_WARPS; ++w) {
      if (w < warp) off += sh.sums[w];
      all += sh.sums[w];
    }
    if (b < p.batch.B) sh.base[b] = off + x - mine;
    before += all;
    __syncthreads();
  }
  if (t == 0) sh.base[p.batch.B] = before;
  __syncthreads();
  const uint32_t per = (before + gridDim.x - 1) / gridDim.x;
  return per < KA_WARPS ? KA_WARPS : per;
}

// What a warp needs to know of one of its units: the page (two pages of 16 tokens), the scales.
struct KaUnit {
  int pid[2];
  int exps;     // key and value exponent bytes of the first and second 16 keys
};

__global__ void __launch_bounds__(KA_WARPS * 32, 1) kv_attend_kernel(const __grid_constant__ KvAttendParams p) {
  extern __shared__ __align__(1024) uint8_t ka_smem[];
  KaShared& sh = *reinterpret_cast<KaShared*>(ka_smem + KA_RING);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  if (lane == 0)
    for (int i = 0; i < KA_STAGES; ++i) mbar_init(&sh.full[warp][i], 1);
  if (threadIdx.x == 0) sh.abort_flag = 0;
  fence_mbar_init();
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t per = ka_plan(p, sh);
  const uint32_t total = sh.base[p.batch.B];
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b <= p.batch.B; b += KA_WARPS * 32) p.plan[b] = sh.base[b];
    if (threadIdx.x == 0) p.plan[p.batch.B + 1] = per;
  }
  uint8_t* ring = ka_smem + warp * KA_STAGES * 2 * KA_SIDE;
  const int page = p.cache.page(), lg = p.cache.page_log2;
  uint32_t used = 0;                                   // units this warp has taken from its ring

  const unsigned long long end64 = static_cast<unsigned long long>(blockIdx.x + 1) * per;
  const uint32_t range_end = end64 < total ? static_cast<uint32_t>(end64) : total;
  uint32_t pos = blockIdx.x * per;
  int b = 0;
  bool ok = true;
  while (pos < range_end) {
    // ------------------------------------------------------------------ the segment
    {
      int lo = b, hi = p.batch.B;                      // the last sequence with base <= pos
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (sh.base[mid] <= pos) lo = mid; else hi = mid;
      }
      b = lo;
    }
    const KaSpan span = ka_span(p, b);
    const uint32_t in_seq = pos - sh.base[b];
    const uint32_t item = in_seq / span.n;
    const int u0 = static_cast<int>(in_seq - item * span.n);
    const int head = static_cast<int>(item) / p.row_tiles, rt = static_cast<int>(item) - head * p.row_tiles;
    int n = span.n - u0;
    if (static_cast<uint32_t>(n) > range_end - pos) n = static_cast<int>(range_end - pos);

    const int mine = n > warp ? (n - warp + KA_WARPS - 1) / KA_WARPS : 0;   // u0 + warp, + 8, ...
    auto key_of = [&](int i) {                         // first key of this warp's i-th unit
      const int u = u0 + warp + KA_WARPS * i;
      return (u < span.sink_units ? u : span.first + u - span.sink_units) * KA_UNIT;
    };
    // Lane l holds what there is to know of unit `base + l`.
    auto look_up = [&](int base) {
      KaUnit k;
      k.pid[0] = k.pid[1] = -1;
      k.exps = 0;
      const int i = base + lane;
      if (i < mine) {
        const int key = key_of(i);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = key + 16 * h;
          if (at >= span.end) continue;                // hidden
          const int col = at >> lg;
          const int pid = col < p.batch.cols ? p.batch.pages[static_cast<long long>(b) * p.batch.cols + col] : -1;
          if (pid < 0 || pid >= p.cache.num_pages) {
            report_status(p.status, CB_BAD_ARGUMENT, 2, 0xA04);
            continue;
          }
          k.pid[h] = pid;
          const uint32_t e = *reinterpret_cast<const uint16_t*>(p.cache.exp_of(pid, head, 0));
          k.exps |= static_cast<int>(e << (16 * h));
        }
      }
      return k;
    };
    KaUnit info = look_up(0);
    // Fills the ring with this warp's i-th unit.  A page that is not there is replaced by any other: its keys are
    // hidden, its values only have to be numbers.
    auto issue = [&](int i) {
      const int src = i & 31;
      const int p0 = __shfl_sync(0xffffffffu, info.pid[0], src), p1 = __shfl_sync(0xffffffffu, info.pid[1], src);
      const uint32_t slot = (used + i) % KA_STAGES;
      uint8_t* dst = ring + slot * 2 * KA_SIDE;
      uint64_t* bar = &sh.full[warp][slot];
      const int a0 = p0 >= 0 ? p0 : 0, a1 = p1 >= 0 ? p1 : a0;
      if (lane == 0) mbar_arrive_expect_tx(bar, 2 * KA_SIDE);
      __syncwarp();
      if (page == 16) {
        if (lane < 4)
          bulk_load_1d(dst + (lane & 1) * KA_SIDE + (lane >> 1) * (KA_SIDE / 2),
                       p.cache.tile(lane >> 1 ? a1 : a0, head, lane & 1), KA_SIDE / 2, bar);
      } else if (lane < 2) {
        const int slot0 = key_of(i) & (page - 1);
        bulk_load_1d(dst + lane * KA_SIDE, p.cache.tile(a0, head, lane) + slot0 * KV_D, KA_SIDE, bar);
      }
    };
    for (int i = 0; i < KA_STAGES && i < mine; ++i) issue(i);

    // ------------------------------------------------------------------ queries of the tile
    // Fragments of m16n8k16 with the head dimension in the order in which the keys' bytes arrive: step m takes
    // dims 16 m + 4 c .. + 3 of lane c.  Rows are brought to [1, 2) by a power of two, so that fp16 holds them.
    uint32_t qa[8][4];
    float row_scale[2];
    int row_pos[2];
    const int rows = p.batch.S * p.group;
#pragma unroll
    for (int r2 = 0; r2 < 2; ++r2) {
      const int r = rt * 16 + g + 8 * r2;
      const int tok = r / p.group;
      const bool there = r < rows && tok < span.count;
      row_pos[r2] = there ? span.start + tok : -1;
      uint2 raw[8];
      float amax = 0.f;
      const __nv_bfloat16* src =
          p.q + b * p.q_sb + tok * p.q_ss + static_cast<long long>(head * p.group + r - tok * p.group) * p.q_sh + 4 * c;
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        raw[m] = there ? *reinterpret_cast<const uint2*>(src + 16 * m) : make_uint2(0u, 0u);
        const float2 f0 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[m].x));
        const float2 f1 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[m].y));
        amax = fmaxf(amax, fmaxf(fmaxf(fabsf(f0.x), fabsf(f0.y)), fmaxf(fabsf(f1.x), fabsf(f1.y))));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
      e = e < -100 ? -100 : e > 100 ? 100 : e;
      const float down = kv_pow2(-e);
      row_scale[r2] = p.scale_log2 * kv_pow2(e);
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        const float2 f0 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[m].x));
        const float2 f1 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[m].y));
        qa[m][r2] = ka_half2(f0.x * down, f0.y * down);
        qa[m][2 + r2] = ka_half2(f1.x * down, f1.y * down);
      }
    }

    // ------------------------------------------------------------------ the units
    float o[8][2][4];
#pragma unroll
    for (int m = 0; m < 8; ++m)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[m][x][j] = 0.f;
    float m_ref[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const int first_pos = span.start, last_pos = span.end - 1;   // of any query of the sequence
    for (int i = 0; ok && i < mine; ++i) {
      const uint32_t slot = (used + i) % KA_STAGES;
      if (!mbar_wait_warp(&sh.full[warp][slot], ((used + i) / KA_STAGES) & 1u, &sh.abort_flag, p.status, 0xA10)) {
        ok = false;
        break;
      }
      const uint32_t keys = smem_u32(ring + slot * 2 * KA_SIDE), values = keys + KA_SIDE;
      const int exps = __shfl_sync(0xffffffffu, info.exps, i & 31);
      const int seen0 = __shfl_sync(0xffffffffu, info.pid[0], i & 31) >= 0;
      const int seen1 = __shfl_sync(0xffffffffu, info.pid[1], i & 31) >= 0;
      const int key = key_of(i);
      // scores: four tiles of 8 keys
      float s[4][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s[t][j] = 0.f;
#pragma unroll
        for (int mh = 0; mh < 2; ++mh) {
          uint32_t r[4];
          const int row = 8 * t + (lane & 7);
          ka_ldsm(keys + row * KV_D + (((4 * mh + (lane >> 3)) ^ (row & 7)) << 4), r);
#pragma unroll
          for (int m = 0; m < 4; ++m) ka_mma(s[t], qa[4 * mh + m], kv_to_half2(r[m]), kv_to_half2(r[m] >> 16));
        }
      }
      // to log2 units with both scales in, hidden ones to -inf
      const bool mask = key + KA_UNIT - 1 > first_pos || !seen0 || !seen1 ||
                        (p.window > 0 && key <= last_pos - p.window && key + KA_UNIT > p.sinks);
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float f = kv_pow2(static_cast<int8_t>(exps >> (16 * (t >> 1))));
        const float add = static_cast<float>(ka_value_exp(exps, t >> 1));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x = fmaf(s[t][j], row_scale[j >> 1] * f, add);
          if (mask) {
            const int at = key + 8 * t + 2 * c + (j & 1), q = row_pos[j >> 1];
            const bool hidden = at > q || (p.window > 0 && at <= q - p.window && at >= p.sinks) ||
                                !(t >> 1 ? seen1 : seen0);
            x = hidden ? -INFINITY : x;
          }
          s[t][j] = x;
          mx[j >> 1] = fmaxf(mx[j >> 1], x);
        }
      }
      const bool grow = mx[0] > m_ref[0] + KA_RAISE || mx[1] > m_ref[1] + KA_RAISE ||
                        (m_ref[0] == -INFINITY && mx[0] > -INFINITY) || (m_ref[1] == -INFINITY && mx[1] > -INFINITY);
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int r2 = 0; r2 < 2; ++r2) {
          float x = mx[r2];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          x = fmaxf(x, m_ref[r2]);
          const float a = m_ref[r2] == -INFINITY ? 0.f : ka_ex2(m_ref[r2] - x);
          m_ref[r2] = x;
          l[r2] *= a;
#pragma unroll
          for (int m = 0; m < 8; ++m)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              o[m][y][2 * r2] *= a;
              o[m][y][2 * r2 + 1] *= a;
            }
        }
      }
      // probabilities (times the value scale) and their sums (without it)
      const float off[2] = {m_ref[0] == -INFINITY ? 0.f : m_ref[0], m_ref[1] == -INFINITY ? 0.f : m_ref[1]};
      uint32_t pa[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            e[j] = ka_ex2(s[2 * h + t][j] - off[j >> 1]);
            sum[j >> 1] += e[j];
          }
          pa[h][2 * t] = ka_half2(e[0], e[1]);
          pa[h][2 * t + 1] = ka_half2(e[2], e[3]);
        }
        const float out = kv_pow2(-ka_value_exp(exps, h));
        l[0] = fmaf(sum[0], out, l[0]);
        l[1] = fmaf(sum[1], out, l[1]);
      }
      // products: the transposing load of byte pairs gives {key, dim}, {key, dim + 1}, {key + 1, dim}, {key + 1,
      // dim + 1}; even and odd dims make a tile of 8 each
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < 8; m += 2) {
          uint32_t r[4];
          const int row = 16 * h + (lane & 15);
          ka_ldsm_t(values + row * KV_D + (((m + (lane >> 4)) ^ (row & 7)) << 4), r);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t b0 = __byte_perm(r[2 * x], 0u, 0x3120), b1 = __byte_perm(r[2 * x + 1], 0u, 0x3120);
            ka_mma(o[m + x][0], pa[h], kv_to_half2(b0), kv_to_half2(b1));
            ka_mma(o[m + x][1], pa[h], kv_to_half2(b0 >> 16), kv_to_half2(b1 >> 16));
          }
        }
      __syncwarp();                                    // the slot has been read
      if (i + 1 < mine && ((i + 1) & 31) == 0) info = look_up(i + 1);
      // units up to the end of the looked-up batch are issued ahead; the rest after the next look-up
      const int ahead = i + KA_STAGES;
      if (ahead < mine && (ahead >> 5) == ((i + 1) >> 5)) issue(ahead);
      if (((i + 1) & 31) == 0)
        for (int x = i + 1; x < ahead && x < mine; ++x) issue(x);
    }
    used += mine;
#pragma unroll
    for (int r2 = 0; r2 < 2; ++r2)
      if (row_pos[r2] < 0) {                           // not a query: zeros
        m_ref[r2] = -INFINITY;
        l[r2] = 0.f;
#pragma unroll
        for (int m = 0; m < 8; ++m)
#pragma unroll
          for (int y = 0; y < 2; ++y) o[m][y][2 * r2] = o[m][y][2 * r2 + 1] = 0.f;
      }

    // ------------------------------------------------------------------ merge of the warps
    float* acc = reinterpret_cast<float*>(ka_smem);    // [warp][16][128], over the rings
#pragma unroll
    for (int r2 = 0; r2 < 2; ++r2) {
      l[r2] += __shfl_xor_sync(0xffffffffu, l[r2], 1);
      l[r2] += __shfl_xor_sync(0xffffffffu, l[r2], 2);
      if (c == 0) sh.ml[warp][g + 8 * r2] = make_float2(m_ref[r2], l[r2]);
    }
    __syncthreads();
#pragma unroll
    for (int r2 = 0; r2 < 2; ++r2)
#pragma unroll
      for (int m = 0; m < 8; ++m)
        *reinterpret_cast<float4*>(acc + (warp * 16 + g + 8 * r2) * KV_D + 16 * m + 4 * c) =
            make_float4(o[m][0][2 * r2], o[m][1][2 * r2], o[m][0][2 * r2 + 1], o[m][1][2 * r2 + 1]);
    __syncthreads();
    const bool whole = n == span.n;
    const uint32_t slot = 2u * blockIdx.x + (u0 == 0 ? 1u : 0u);
#pragma unroll 1
    for (int r = warp; r < 16; r += KA_WARPS) {
      const int row = rt * 16 + r;
      if (row >= rows) continue;
      float m = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < KA_WARPS; ++w) m = fmaxf(m, sh.ml[w][r].x);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < KA_WARPS; ++w) {
        const float2 x = sh.ml[w][r];
        const float f = x.x == -INFINITY ? 0.f : ka_ex2(x.x - m);
        sum += f * x.y;
        const float4 a = *reinterpret_cast<const float4*>(acc + (w * 16 + r) * KV_D + 4 * lane);
        v.x += f * a.x, v.y += f * a.y, v.z += f * a.z, v.w += f * a.w;
      }
      if (whole) {
        const int tok = row / p.group, h = head * p.group + row - tok * p.group;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const __nv_bfloat162 o2[2] = {__floats2bfloat162_rn(v.x * inv, v.y * inv),
                                      __floats2bfloat162_rn(v.z * inv, v.w * inv)};
        *reinterpret_cast<uint2*>(p.o + ((static_cast<long long>(b) * p.batch.S + tok) * p.Hq + h) * KV_D + 4 * lane) =
            *reinterpret_cast<const uint2*>(o2);
        if (lane == 0)
          p.lse[(static_cast<long long>(b) * p.Hq + h) * p.batch.S + tok] =
              sum == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(sum);
      } else {
        const long long at = static_cast<long long>(slot) * 16 + r;
        *reinterpret_cast<float4*>(p.part_o + at * KV_D + 4 * lane) = v;
        if (lane == 0) p.part_ml[at] = make_float2(m, sum);
      }
    }
    fence_proxy_async_smem();   // the next segment's bulk copies write where ordinary accesses were
    __syncthreads();
    if (*static_cast<volatile int*>(&sh.abort_flag) != 0) {
      // A copy never arrived: the others get time to land before the shared memory goes to another CTA.
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
      break;
    }
    pos += n;
  }
}

// Rows of items that were cut: out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i in the order of the keys.  A warp
// takes a row.
__global__ void __launch_bounds__(KA_MERGE_THREADS) kv_attend_merge_kernel(const __grid_constant__ KvAttendParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long row = (blockIdx.x * static_cast<long long>(KA_MERGE_THREADS) + threadIdx.x) >> 5;
  const int S = p.batch.S, hkv = p.cache.hkv;
  const long long rows = static_cast<long long>(S) * p.group;      // of a sequence and key/value head
  if (row >= rows * hkv * p.batch.B) return;
  const long long bh = row / rows;
  const int b = static_cast<int>(bh / hkv), head = static_cast<int>(bh - static_cast<long long>(b) * hkv);
  const int r = static_cast<int>(row - bh * rows), rt = r >> 4;
  const uint32_t base = p.plan[b], per = p.plan[p.batch.B + 1];
  const uint32_t n = (p.plan[b + 1] - base) / static_cast<uint32_t>(hkv * p.row_tiles);
  const uint32_t start = base + static_cast<uint32_t>(head * p.row_tiles + rt) * n;
  const uint32_t cta0 = start / per, cta1 = (start + n - 1) / per;
  if (cta0 == cta1) return;                                        // the row is final
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = -INFINITY, l = 0.f;
#pragma unroll 1
  for (uint32_t i0 = cta0; i0 <= cta1; i0 += 8) {
    float4 v[8];
    float2 x[8];
#pragma unroll
    for (uint32_t u = 0; u < 8; ++u) {
      x[u] = make_float2(-INFINITY, 0.f);
      const uint32_t i = i0 + u;
      if (i <= cta1) {
        const bool begins = i * per <= start;
        const long long at = static_cast<long long>(2u * i + (begins ? 1u : 0u)) * 16 + (r & 15);
        x[u] = p.part_ml[at];
        v[u] = reinterpret_cast<const float4*>(p.part_o + at * KV_D)[lane];
      }
    }
    float m_new = m;
#pragma unroll
    for (int u = 0; u < 8; ++u) m_new = fmaxf(m_new, x[u].x);
    const float keep = m == -INFINITY ? 0.f : ka_ex2(m - m_new);
    m = m_new;
    l *= keep;
    acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (x[u].y == 0.f) continue;            // no visible key in the part
      const float f = ka_ex2(x[u].x - m);
      l += f * x[u].y;
      acc.x += f * v[u].x, acc.y += f * v[u].y, acc.z += f * v[u].z, acc.w += f * v[u].w;
    }
  }
  const int tok = r / p.group, h = head * p.group + r - tok * p.group;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const __nv_bfloat162 o2[2] = {__floats2bfloat162_rn(acc.x * inv, acc.y * inv),
                                __floats2bfloat162_rn(acc.z * inv, acc.w * inv)};
  *reinterpret_cast<uint2*>(p.o + ((static_cast<long long>(b) * S + tok) * p.Hq + h) * KV_D + 4 * lane) =
      *reinterpret_cast<const uint2*>(o2);
  if (lane == 0)
    p.lse[(static_cast<long long>(b) * p.Hq + h) * S + tok] =
        l == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(l);
}

static int ka_sms() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1)
    return 148;
  return n;
}

struct KaLaunch {
  int row_tiles, grid;
  long long bytes, o_at, ml_at;
};
// False when the flat list of units does not fit 31 bits.
static bool ka_shape(KaLaunch* s, int B, int S, int Hq, int Hkv, long long max_len) {
  const long long rows = static_cast<long long>(S) * (Hq / Hkv);
  const long long tiles = (rows + 15) / 16;
  const long long units = static_cast<long long>(B) * Hkv * tiles * ((max_len + KA_UNIT - 1) / KA_UNIT + 1);
  if (units > 0x7fffffffll || B > KA_MAX_B) return false;
  s->row_tiles = static_cast<int>(tiles);
  const long long want = (units + KA_WARPS - 1) / KA_WARPS;
  const int sms = ka_sms();
  s->grid = static_cast<int>(want < sms ? want : sms);
  s->o_at = (static_cast<long long>(B + 2) * 4 + 127) / 128 * 128;
  s->ml_at = s->o_at + 2ll * s->grid * 16 * KV_D * 4;
  s->bytes = s->ml_at + 2ll * s->grid * 16 * 8;
  return true;
}

}  // namespace cb

using namespace cb;

extern "C" {

// Bytes of workspace for cb_kv_attend, or -1: the call is too large for one launch.
long long cb_kv_attend_bytes(int B, int S, int Hq, int Hkv, int max_len) {
  KaLaunch s;
  if (B < 1 || S < 1 || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || max_len < 1 || !ka_shape(&s, B, S, Hq, Hkv, max_len)) {
    set_last_error("key/value attention: bad shape, or more than 1024 sequences or 2^31 units of 32 keys");
    return -1;
  }
  return s.bytes;
}

// q [B, S, Hq, 128] bf16 (strides in elements, rows 8-byte aligned), o [B, S, Hq, 128] and lse [B, Hq, S] dense.
// Query i of sequence b has position start[b] + i; count[b] (null: S) of them exist, the other rows are zeros with
// lse -inf.  max_len bounds start + count; a longer sequence is still right, only not evenly cut.
int cb_kv_attend(void* data, void* exps, int num_pages, int hkv, int page, const void* q, long long q_sb,
                 long long q_ss, long long q_sh, void* o, void* lse, const void* pages, int cols, const void* start,
                 const void* count, int B, int S, int Hq, int window, int sinks, int max_len, float scale,
                 void* workspace, long long workspace_bytes, void* status, void* stream) {
  KvAttendParams p;
  int lg = 0;
  while ((1 << lg) < page) ++lg;
  if (num_pages < 1 || page < 16 || page > 128 || (1 << lg) != page || cols < 1 || window < 0 || sinks < 0) {
    set_last_error("key/value attention: bad cache, window or sinks");
    return -1;
  }
  const long long need = cb_kv_attend_bytes(B, S, Hq, hkv, max_len);
  if (need < 0) return -1;
  if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) {
    set_last_error("key/value attention: workspace missing, misaligned or too small");
    return -1;
  }
  KaLaunch s;
  ka_shape(&s, B, S, Hq, hkv, max_len);
  p.cache = {static_cast<uint8_t*>(data), static_cast<int8_t*>(exps), num_pages, hkv, lg};
  p.batch = {static_cast<const int*>(pages), static_cast<const int*>(start), static_cast<const int*>(count), B, S, cols};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_sb = q_sb, p.q_ss = q_ss, p.q_sh = q_sh;
  p.o = static_cast<__nv_bfloat16*>(o);
  p.lse = static_cast<float*>(lse);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.plan = reinterpret_cast<uint32_t*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + s.o_at);
  p.part_ml = reinterpret_cast<float2*>(ws + s.ml_at);
  p.Hq = Hq;
  p.group = Hq / hkv;
  p.row_tiles = s.row_tiles;
  p.window = window;
  p.sinks = window > 0 ? sinks : 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.status = static_cast<uint32_t*>(status);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  static std::atomic<uint64_t> smem_done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kv_attend_kernel), KA_SMEM, smem_done);
  if (e == cudaSuccess)
    e = launch_pdl(kv_attend_kernel, dim3(static_cast<unsigned>(s.grid)), dim3(KA_WARPS * 32), KA_SMEM, st, p);
  if (e == cudaSuccess) {
    const long long rows = static_cast<long long>(B) * S * Hq;
    const int per = KA_MERGE_THREADS / 32;
    e = launch_pdl(kv_attend_merge_kernel, dim3(static_cast<unsigned>((rows + per - 1) / per)), dim3(KA_MERGE_THREADS), 0,
                   st, p);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();   // reported here, not by the next call
    set_last_error(std::string("key/value attention launch: ") + cudaGetErrorString(e));
    return -1;
  }
  return 0;
}

}  // extern "C"
