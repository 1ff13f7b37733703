// cis2b_kv4_attn.cu -- attention over the 4-bit key/value cache
// (include/cis2b.h, cis2b_kv4_attention).
//
// With key j = kb_j + ks_j c_j and value j = vb_j + vs_j c'_j (c, c' the
// codes), for a query row q of scale s
//   t_j = s (ks_j (q . c_j) + kb_j sum(q))               the score
//   o   = (sum_j p_j vs_j c'_j + sum_j p_j vb_j) / sum_j p_j,  p_j = exp(t_j - M)
// so both products run on the codes themselves and the steps and bases are
// one multiply-add per (key, row).
#include "../../include/cis2b.h"
#include "cis2b_kv4.h"
#include "cis2b_kv4.cuh"

#include <limits.h>
#include <math.h>

#include <algorithm>

namespace cis2b {
namespace {

constexpr int ATT_WARPS = 4;
constexpr int ATT_THREADS = 32 * ATT_WARPS;
constexpr int ATT_CHUNK = 32;       // least records (of 16 keys) per split of a request
constexpr int ATT_MAX_SPLITS = 64;  // per (query tile, KV head)
constexpr uint64_t ATT_PART_BYTES = 64ull << 20;  // partial results of the splits

struct AttArgs {
  const void *q;
  void *out;
  int64_t q_row, q_head, o_row, o_head;
  const uint8_t *pool;
  int32_t *status;
  const int32_t *table, *length, *row_start;
  float *part;        // [part_units][cols][HD + 2]
  uint32_t *counter;  // [query tiles][kv_heads]
  int dtype, requests, rows, width, kv_heads, group, shift, pages, window, sinks;
  int q_wide, o_wide;
  int qt;             // tokens per query tile
  int part_units, counters;
  float scale;
};

// What the splitting rule and the kernel must agree on: the keys that one
// query tile sees, as 16-key records 0 .. sink_recs-1 and lo .. hi-1.
struct Span {
  int p0, p1;     // first and last position of the tile's rows (p1 < 0: none sees anything)
  int sink, lo;   // records before the gap, first record after it (0 and 0 without one)
  int tiles;      // records in all
};

__device__ __forceinline__ Span span_of(const AttArgs &a, int len, int n, int qt_index) {
  Span s;
  const int first = len - n;
  s.p0 = first + qt_index * a.qt;
  s.p1 = min(first + min((qt_index + 1) * a.qt, n), len) - 1;
  s.sink = s.lo = s.tiles = 0;
  if (s.p1 < 0) return s;
  const int hi = (s.p1 >> 4) + 1;
  if (a.window) {
    const int lo = max(0, s.p0 - a.window + 1) >> 4;
    const int sink = (min(a.sinks, s.p1 + 1) + 15) >> 4;
    if (sink < lo) s.sink = sink, s.lo = lo;
  }
  s.tiles = s.sink + hi - s.lo;
  return s;
}

// Splits of a request: by its own length and rows alone, so that what else is
// in the batch does not change its result (unless the partial results outgrow
// the workspace, where `coarse` doubles the chunk).
__device__ __forceinline__ int splits_of(const AttArgs &a, int tiles, int query_tiles, int coarse) {
  const int most = max(1, ATT_MAX_SPLITS * 8 / max(1, query_tiles * a.kv_heads));
  return max(1, min(min((tiles + (ATT_CHUNK << coarse) - 1) / (ATT_CHUNK << coarse), ATT_MAX_SPLITS), most));
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N)); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Codes of a 16-bit half each, as half-precision operands.  EXACT: the normal
// numbers c - 8 (low: bits 0-3) and 16 (c - 8) (high: bits 4-7), one more
// instruction each; else the bits themselves, the subnormals c 2^-24 and
// c 2^-20.
template <bool EXACT> __device__ __forceinline__ uint32_t codes_low(uint32_t x) {
  if constexpr (!EXACT) return x & 0x000f000fu;
  const uint32_t y = (x & 0x000f000fu) | 0x64006400u;  // 1024 + c
  const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&y), __half2half2(__ushort_as_half(0x6408)));
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <bool EXACT> __device__ __forceinline__ uint32_t codes_high(uint32_t x) {
  if constexpr (!EXACT) return x & 0x00f000f0u;
  const uint32_t y = (x & 0x00f000f0u) | 0x64006400u;  // 1024 + 16 c
  const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&y), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t *>(&h);
}

template <int HD, int NT, int LIMBS> __host__ __device__ constexpr int att_stages() { return HD == 64 ? 6 : 4; }
template <int HD, int NT, int LIMBS> __host__ __device__ constexpr int att_ring_bytes() {
  const int ring = ATT_WARPS * att_stages<HD, NT, LIMBS>() * kv4_rec_bytes(HD);
  const int merge = 2 * 8 * NT * HD * 4;  // two warps' sums, reusing the ring
  return ring > merge ? ring : merge;
}
template <int HD, int NT, int LIMBS> __host__ __device__ constexpr int att_smem_bytes() {
  return att_ring_bytes<HD, NT, LIMBS>() + NT * LIMBS * (HD / 32) * 512;
}

// One block takes units (request, query tile, split, KV head) in turn; its
// four warps take the unit's records in turn and meet at the end.
//
// The codes reach the tensor pipe without being converted: a code in bits
// 0-3 of a 16-bit word IS the half-precision number c * 2^-24 (a subnormal),
// and in bits 4-7 c * 2^-20, so `and` makes two operands out of a 32-bit
// word, and the factor of 16 is divided out of every other query element
// (keys) or output row (values).  The tensor pipe lines subnormal products up
// by their exponent field, so its sums keep about 15 bits (measured: 4e-5 of
// fp32 rows' results), enough for 16-bit rows; fp32 rows pay one subtraction
// per operand for the normal numbers c - 8.
//
// Keys are the 16 rows of the first product and head_dim the 16 rows of the
// second, with the query rows (tokens x group) as its 8 columns, so that a
// group of up to 8 heads wastes nothing and a warp's lanes hold 4 scores per
// record.  The probabilities go from the first product's accumulator layout
// to the second's operand layout by an 8 x 8 register transpose.
//
// M is a lazy maximum per column: it moves only when a weight p * vs (the
// number that is rounded to half precision) passes 2^14, or p passes 2^60,
// and then to 2^8 below the top.  Weights keep 11 bits down to 2^-22 of the
// largest; LIMBS = 2 (fp32 rows) adds a second half-precision limb to the
// weights and the query, 22 bits.  Codes are centred at 8, which halves the
// rounding's effect: directly for fp32 rows, by the sum of the rounded
// weights (a product with ones) for 16-bit rows.
template <int HD, int NT, int LIMBS>
__global__ __launch_bounds__(ATT_THREADS) void k_kv4_attention(AttArgs a) {
  constexpr int REC = kv4_rec_bytes(HD), ST = att_stages<HD, NT, LIMBS>();
  constexpr int KS = HD / 16;            // k-steps of the first product, row tiles of the second
  constexpr int W = HD / 32;             // 32-bit words of a key row per lane
  constexpr int COLS = 8 * NT;
  constexpr bool EXACT = LIMBS == 2;
  constexpr float UNIT = EXACT ? 1.0f : 16777216.0f;  // what a code's operand is divided by
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int scan_u[ATT_THREADS + 1], scan_q[ATT_THREADS + 1], warp_u[ATT_WARPS], warp_q[ATT_WARPS];
  __shared__ float red[ATT_WARPS][3][COLS];  // M, l and the base sum of each warp
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint8_t *ring = smem + warp * ST * REC;
  uint4 *qfrag = reinterpret_cast<uint4 *>(smem + att_ring_bytes<HD, NT, LIMBS>());

  // Rows past the last request are zero.
  {
    const int used = max(0, min(__ldg(a.row_start + a.requests), a.rows));
    const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const int64_t per = (int64_t)a.kv_heads * a.group * (HD / 8);
    for (int64_t i = (int64_t)blockIdx.x * ATT_THREADS + tid; i < (a.rows - used) * per; i += gridDim.x * ATT_THREADS) {
      const int64_t row = used + i / per;
      const int h = (int)(i % per) / (HD / 8), d = (int)(i % (HD / 8)) * 8;
      store8(a.out, a.dtype, row * a.o_row + h * a.o_head + d, a.o_wide, zero);
    }
  }

  // Units before each request: thread i sums requests i * per .. of its own.
  const int per = (a.requests + ATT_THREADS - 1) / ATT_THREADS;
  int coarse = 0, total = 0;
  for (;; ++coarse) {
    int64_t units = 0;
    int tiles_q = 0;
    int64_t split_units = 0;
    for (int i = 0; i < per; ++i) {
      const int r = tid * per + i;
      if (r >= a.requests) break;
      const int len = __ldg(a.length + r), n = __ldg(a.row_start + r + 1) - __ldg(a.row_start + r);
      if (n <= 0) continue;
      const int nq = (n + a.qt - 1) / a.qt;
      const int sp = splits_of(a, span_of(a, len, n, nq - 1).tiles, nq, coarse);
      units += (int64_t)nq * sp;
      tiles_q += nq;
      if (sp > 1) split_units += (int64_t)nq * sp;
    }
    int u = (int)min(units, (int64_t)INT_MAX / 1024), sq = tiles_q;
    const int own_u = u, own_q = sq;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, u, d), y = __shfl_up_sync(0xffffffffu, sq, d);
      if (lane >= d) u += x, sq += y;
    }
    __syncthreads();
    if (lane == 31) warp_u[warp] = u, warp_q[warp] = sq;
    __syncthreads();
    int before_u = 0, before_q = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < ATT_WARPS; ++w) {
      if (w < warp) before_u += warp_u[w], before_q += warp_q[w];
      total += warp_u[w];
    }
    scan_u[tid] = before_u + u - own_u;
    scan_q[tid] = before_q + sq - own_q;
    if (tid == ATT_THREADS - 1) scan_u[ATT_THREADS] = before_u + u, scan_q[ATT_THREADS] = before_q + sq;
    // Partial results are kept by unit: enough room, or a coarser chunk (at
    // last one split, which needs none).
    const bool fits = (int64_t)total * a.kv_heads <= a.part_units;
    const int any = __syncthreads_or(split_units > 0);
    if (fits || !any) break;
  }
  const int64_t all_units = (int64_t)total * a.kv_heads;

  for (int64_t unit = blockIdx.x; unit < all_units; unit += gridDim.x) {
    // ---- which unit
    const int head = (int)(unit % a.kv_heads), ub = (int)(unit / a.kv_heads);
    int seg = 0;
    for (int step = ATT_THREADS / 2; step; step >>= 1)
      if (scan_u[seg + step] <= ub) seg += step;
    int u = scan_u[seg], qbase = scan_q[seg], r = seg * per, n = 0, len = 0, nq = 0, sp = 1;
    for (;; ++r) {
      len = __ldg(a.length + r);
      n = __ldg(a.row_start + r + 1) - __ldg(a.row_start + r);
      if (n <= 0) continue;
      nq = (n + a.qt - 1) / a.qt;
      sp = splits_of(a, span_of(a, len, n, nq - 1).tiles, nq, coarse);
      if (ub < u + nq * sp) break;
      u += nq * sp, qbase += nq;
    }
    const int qi = (ub - u) / sp, split = (ub - u) - qi * sp;
    const Span s = span_of(a, len, n, qi);
    const int chunk = (s.tiles + sp - 1) / sp;
    const int t_begin = min(split * chunk, s.tiles), t_end = min(t_begin + chunk, s.tiles);
    const int row0 = __ldg(a.row_start + r) + qi * a.qt;
    const int ncol = min(a.qt, n - qi * a.qt) * a.group;

    // ---- query operands: lane (g, t) holds elements t HD/4 .. of column g
    uint32_t bq[NT == 1 ? LIMBS : 1][NT == 1 ? KS : 1][2];
    float sum_s[NT][2];  // sum(q) * scale * log2 e of this lane's two columns
    int pos[NT][2];
    float code_scale;
    {
      float x[NT][4 * W][2];
      float top = 0.0f;
      const float sl = a.scale * 1.4426950408889634f;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int col = 8 * j + g, tok = col / a.group;
        const int64_t row = row0 + tok;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          float e[8];
          if (col < ncol && row >= 0 && row < a.rows) {
            const int64_t at = row * a.q_row + (int64_t)(head * a.group + col - tok * a.group) * a.q_head + t * (HD / 4) + w * 8;
            if (a.dtype == KV4_F32) load8<KV4_F32>(a.q, at, a.q_wide, e);
            else if (a.dtype == KV4_F16) load8<KV4_F16>(a.q, at, a.q_wide, e);
            else load8<KV4_BF16>(a.q, at, a.q_wide, e);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(e[i])), sum += e[i];
          // Word w's `and`s give the code pairs (0,4) (1,5) (2,6) (3,7).
#pragma unroll
          for (int i = 0; i < 4; ++i) x[j][4 * w + i][0] = e[i], x[j][4 * w + i][1] = e[i + 4];
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum *= sl;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int cc = 8 * j + 2 * t + c;
          sum_s[j][c] = __shfl_sync(0xffffffffu, sum, (2 * t + c) * 4);
          pos[j][c] = cc < ncol ? s.p0 + cc / a.group : -1;
        }
      }
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      // A power of two brings the largest element to 2^13 .. 2^14: 16-bit
      // elements down to 2^-24 of it stay exact.
      const int e = (int)(__float_as_uint(top) >> 23);  // biased exponent
      const int up = e == 0 || e == 255 ? 0 : min(max(13 - (e - 127), -100), 100);
      const float f = __uint_as_float((uint32_t)(127 + up) << 23), back = __uint_as_float((uint32_t)(127 - up) << 23);
      code_scale = sl * UNIT * back;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int w = 0; w < W; ++w) {
          uint32_t v[LIMBS][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float k = (i & 1) ? f * 0.0625f : f;
            const float y0 = x[j][4 * w + i][0] * k, y1 = x[j][4 * w + i][1] * k;
            v[0][i] = pack_half(y0, y1);
            if constexpr (LIMBS == 2) {
              const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&v[0][i]));
              v[1][i] = pack_half(y0 - h.x, y1 - h.y);
            }
          }
#pragma unroll
          for (int l = 0; l < LIMBS; ++l) {
            if constexpr (NT == 1) {
              bq[l][2 * w][0] = v[l][0], bq[l][2 * w][1] = v[l][1];
              bq[l][2 * w + 1][0] = v[l][2], bq[l][2 * w + 1][1] = v[l][3];
            } else if (warp == (j & (ATT_WARPS - 1))) {
              qfrag[((j * LIMBS + l) * W + w) * 32 + lane] = make_uint4(v[l][0], v[l][1], v[l][2], v[l][3]);
            }
          }
        }
    }
    if constexpr (NT > 1) __syncthreads();

    // ---- the unit's records, this warp's share
    float o[NT][KS][4], ones[NT][4], M[NT][2], l[NT][2], z[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int m = 0; m < KS; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][m][i] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ones[j][i] = 0.0f;
#pragma unroll
      for (int c = 0; c < 2; ++c) M[j][c] = -1e30f, l[j][c] = z[j][c] = 0.0f;
    }
    const int32_t *row_table = a.table + (int64_t)r * a.width;
    const int recs_shift = a.shift - 4;
    auto key_rec = [&](int tile) { return tile < s.sink ? tile : tile - s.sink + s.lo; };
    auto page_of = [&](int tile) {  // page of a record, -1 if there is none
      if (tile >= t_end) return -1;
      const int p = key_rec(tile) >> recs_shift;
      const int pg = p < a.width ? __ldg(row_table + p) : -1;
      if (pg >= a.pages || pg < 0) {
        if (a.status && lane == 0) atomicOr(a.status, CIS2B_KV4_BAD_PAGE);
        return -1;
      }
      return pg;
    };
    uint32_t held = 0;  // bit i: stage i holds a record of the pool
    auto issue = [&](int tile, int page, int stage) {
      held &= ~(1u << stage);
      if (tile < t_end && page >= 0) {
        held |= 1u << stage;
        const uint8_t *src = a.pool + ((((int64_t)page * a.kv_heads + head) << recs_shift) +
                                       (key_rec(tile) & ((1 << recs_shift) - 1))) * REC;
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(ring + stage * REC);
#pragma unroll
        for (int i = 0; i < (REC / 16 + 31) / 32; ++i) {
          const int c = lane + 32 * i;
          if (c < REC / 16) {
            // 16-byte pieces of value rows move within their 128 bytes so
            // that the operand loads below touch every bank once.
            const int cv = c - HD / 2;
            const int to = cv >= 0 && cv < HD / 2 ? HD / 2 + (cv ^ (((cv >> 3) & 3) << 1)) : c;
            cp_async16(dst + to * 16, src + c * 16);
          }
        }
      }
      cp_async_commit();
    };
    const int first = t_begin + warp;
    int next_page = page_of(first);
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
      issue(first + i * ATT_WARPS, next_page, i);
      next_page = page_of(first + (i + 1) * ATT_WARPS);
    }
    int stage = 0;
    for (int tile = first; tile < t_end; tile += ATT_WARPS) {
      {
        const int to = stage == 0 ? ST - 1 : stage - 1;
        issue(tile + (ST - 1) * ATT_WARPS, next_page, to);
        next_page = page_of(tile + ST * ATT_WARPS);
      }
      cp_async_wait<ST - 1>();
      __syncwarp();
      const uint8_t *rec = ring + stage * REC;
      const int k0 = key_rec(tile) * 16;

      // scores: keys g and g + 8 by columns 2t, 2t + 1
      float sc[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[j][i] = 0.0f;
      {
        uint32_t ka[W], kb[W];
        if constexpr (HD == 128) {
          const uint4 x = *reinterpret_cast<const uint4 *>(rec + g * 64 + t * 16);
          const uint4 y = *reinterpret_cast<const uint4 *>(rec + (g + 8) * 64 + t * 16);
          ka[0] = x.x, ka[1] = x.y, ka[2] = x.z, ka[3] = x.w;
          kb[0] = y.x, kb[1] = y.y, kb[2] = y.z, kb[3] = y.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2 *>(rec + g * 32 + t * 8);
          const uint2 y = *reinterpret_cast<const uint2 *>(rec + (g + 8) * 32 + t * 8);
          ka[0] = x.x, ka[1] = x.y, kb[0] = y.x, kb[1] = y.y;
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const uint32_t x = ka[w], y = kb[w], xs = x >> 8, ys = y >> 8;
          const uint32_t a0 = codes_low<EXACT>(x), a1 = codes_low<EXACT>(y), a2 = codes_high<EXACT>(x), a3 = codes_high<EXACT>(y);
          const uint32_t c0 = codes_low<EXACT>(xs), c1 = codes_low<EXACT>(ys), c2 = codes_high<EXACT>(xs), c3 = codes_high<EXACT>(ys);
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int lm = 0; lm < LIMBS; ++lm) {
              if constexpr (NT == 1) {
                mma16816(sc[j], a0, a1, a2, a3, bq[lm][2 * w][0], bq[lm][2 * w][1]);
                mma16816(sc[j], c0, c1, c2, c3, bq[lm][2 * w + 1][0], bq[lm][2 * w + 1][1]);
              } else {
                const uint4 f = qfrag[((j * LIMBS + lm) * W + w) * 32 + lane];
                mma16816(sc[j], a0, a1, a2, a3, f.x, f.y);
                mma16816(sc[j], c0, c1, c2, c3, f.z, f.w);
              }
            }
        }
      }
      // parameters of keys g and g + 8; a value's base is taken at code 8
      float ks[2], kz[2], vs[2], vz[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint2 p = *reinterpret_cast<const uint2 *>(rec + 16 * HD + (g + 8 * i) * 8);
        ks[i] = bf16_lo(p.x) * code_scale;
        kz[i] = EXACT ? fmaf(8.0f, bf16_lo(p.x), bf16_hi(p.x)) : bf16_hi(p.x);
        vs[i] = bf16_lo(p.y), vz[i] = fmaf(8.0f, vs[i], bf16_hi(p.y));
      }
      // Every column sees every key of the record: no mask.
      const bool whole = ((held >> stage) & 1) && k0 + 15 <= s.p0 &&
                         (a.window == 0 || k0 > s.p1 - a.window || k0 + 15 < a.sinks);
      uint32_t bw[NT][LIMBS][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float tt[4], p[4], w[4], vse[4], vze[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          tt[i] = fmaf(sc[j][i], ks[i >> 1], kz[i >> 1] * sum_s[j][i & 1]);
          vse[i] = vs[i >> 1], vze[i] = vz[i >> 1];
        }
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = k0 + g + 8 * (i >> 1), at = pos[j][i & 1];
            const bool see = ((held >> stage) & 1) && key <= at &&
                             (a.window == 0 || key > at - a.window || key < a.sinks);
            if (!see) tt[i] = -INFINITY, vse[i] = vze[i] = 0.0f;  // whatever the cache holds there
          }
        }
        float chk[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = ex2(tt[i] - M[j][i & 1]), w[i] = p[i] * vse[i];
#pragma unroll
        for (int c = 0; c < 2; ++c)
          chk[c] = fmaxf(fmaxf(w[c], w[c + 2]), fmaxf(p[c], p[c + 2]) * 0x1p-46f);
        if (__any_sync(0xffffffffu, fmaxf(chk[0], chk[1]) > 0x1p14f)) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float ck = chk[c], tw = fmaxf(tt[c] + lg2(vse[c]), tt[c + 2] + lg2(vse[c + 2])), ts = fmaxf(tt[c], tt[c + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
              ck = fmaxf(ck, __shfl_xor_sync(0xffffffffu, ck, d));
              tw = fmaxf(tw, __shfl_xor_sync(0xffffffffu, tw, d));
              ts = fmaxf(ts, __shfl_xor_sync(0xffffffffu, ts, d));
            }
            if (ck > 0x1p14f) {
              const float m = fmaxf(tw - 8.0f, ts - 54.0f), f = ex2(M[j][c] - m);
              M[j][c] = m;
              l[j][c] *= f, z[j][c] *= f;
              ones[j][c] *= f, ones[j][c + 2] *= f;
#pragma unroll
              for (int k = 0; k < KS; ++k) o[j][k][c] *= f, o[j][k][c + 2] *= f;
#pragma unroll
              for (int i = c; i < 4; i += 2) p[i] = ex2(tt[i] - m), w[i] = p[i] * vse[i];
            }
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          l[j][c] += p[c] + p[c + 2];
          z[j][c] = fmaf(p[c], vze[c], fmaf(p[c + 2], vze[c + 2], z[j][c]));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t h = pack_half(w[2 * i], w[2 * i + 1]);
          bw[j][0][i] = transpose8x8(h);
          if constexpr (LIMBS == 2) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
            bw[j][1][i] = transpose8x8(pack_half(w[2 * i] - f.x, w[2 * i + 1] - f.y));
          }
        }
      }
      // values: lane (g, t) holds elements g HD/8 .. of keys 2t, 2t+1, 2t+8, 2t+9
      {
        uint32_t v[4][HD / 64];
        const uint8_t *vb = rec + 8 * HD;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = 2 * t + (i & 1) + 8 * (i >> 1), at = key * (HD / 2) + g * (HD / 16);
          const int c = at >> 4, to = (c ^ (((c >> 3) & 3) << 1)) * 16 + (at & 15);
          if constexpr (HD == 128) {
            const uint2 x = *reinterpret_cast<const uint2 *>(vb + to);
            v[i][0] = x.x, v[i][1] = x.y;
          } else {
            v[i][0] = *reinterpret_cast<const uint32_t *>(vb + to);
          }
        }
#pragma unroll
        for (int w = 0; w < HD / 64; ++w)
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // low and high 16 bits: codes 0-3 and 4-7 of the word
            uint32_t x = __byte_perm(v[0][w], v[1][w], h ? 0x7632 : 0x5410);
            uint32_t y = __byte_perm(v[2][w], v[3][w], h ? 0x7632 : 0x5410);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int m = 4 * w + 2 * h + q;  // rows of elements 2m and 2m + 1 of this lane's HD/8
              const uint32_t a0 = codes_low<EXACT>(x), a1 = codes_high<EXACT>(x), a2 = codes_low<EXACT>(y), a3 = codes_high<EXACT>(y);
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int lm = 0; lm < LIMBS; ++lm) mma16816(o[j][m], a0, a1, a2, a3, bw[j][lm][0], bw[j][lm][1]);
              x >>= 8, y >>= 8;
            }
          }
#pragma unroll
        for (int j = 0; j < NT && !EXACT; ++j)
#pragma unroll
          for (int lm = 0; lm < LIMBS; ++lm)
            mma16816(ones[j], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, bw[j][lm][0], bw[j][lm][1]);
      }
      __syncwarp();
      stage = stage + 1 == ST ? 0 : stage + 1;
    }
    cp_async_wait<0>();

    // ---- the warps meet: a common M per column, then sums (0 + 2) + (1 + 3)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          l[j][c] += __shfl_xor_sync(0xffffffffu, l[j][c], d);
          z[j][c] += __shfl_xor_sync(0xffffffffu, z[j][c], d);
        }
        if (g == 0) red[warp][0][8 * j + 2 * t + c] = M[j][c];
      }
    __syncthreads();  // also: every warp is done with its ring
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = 8 * j + 2 * t + c;
        float m = red[0][0][col];
#pragma unroll
        for (int w = 1; w < ATT_WARPS; ++w) m = fmaxf(m, red[w][0][col]);
        const float f = ex2(M[j][c] - m);
        M[j][c] = m;
        l[j][c] *= f, z[j][c] *= f;
        const float base = EXACT ? z[j][c] : z[j][c] - 8.0f * f * ones[j][c];
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          // each warp's numerator, the base's part included
          o[j][k][c] = fmaf(o[j][k][c], f * UNIT, base);
          o[j][k][c + 2] = fmaf(o[j][k][c + 2], f * (UNIT / 16.0f), base);
        }
        if (g == 0) red[warp][1][col] = l[j][c];
      }
    float *sum = reinterpret_cast<float *>(smem);
    auto put = [&](int place) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[((place * NT + j) * KS + k) * 128 + i * 32 + lane] = o[j][k][i];
    };
    auto add = [&](int place) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][k][i] += sum[((place * NT + j) * KS + k) * 128 + i * 32 + lane];
    };
    if (warp >= 2) put(warp - 2);
    __syncthreads();
    if (warp < 2) add(warp);
    __syncthreads();
    if (warp == 1) put(0);
    __syncthreads();

    const bool alone = sp == 1;
    float *part = a.part + unit * (int64_t)(COLS * (HD + 2));
    if (warp == 0) {
      add(0);
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col = 8 * j + 2 * t + c;
          float den = red[0][1][col];
#pragma unroll
          for (int w = 1; w < ATT_WARPS; ++w) den += red[w][1][col];
          if (col >= ncol) continue;
          const float f = !alone ? 1.0f : den > 0.0f || den != den ? 1.0f / den : 0.0f;
          const int tok = col / a.group;
          const int64_t row = row0 + tok;
#pragma unroll
          for (int k = 0; k < KS; k += 4) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[2 * i] = o[j][k + i][c] * f, x[2 * i + 1] = o[j][k + i][c + 2] * f;
            const int d = g * (HD / 8) + 2 * k;
            if (alone) {
              if (row >= 0 && row < a.rows)
                store8(a.out, a.dtype,
                       row * a.o_row + (int64_t)(head * a.group + col - tok * a.group) * a.o_head + d, a.o_wide, x);
            } else {
              float4 *to = reinterpret_cast<float4 *>(part + col * HD + d);
              __stcg(to, make_float4(x[0], x[1], x[2], x[3]));
              __stcg(to + 1, make_float4(x[4], x[5], x[6], x[7]));
            }
          }
          if (!alone && g == 0) __stcg(reinterpret_cast<float2 *>(part + COLS * HD) + col, make_float2(M[j][c], den));
        }
    }
    // ---- splits meet: the last one to finish joins them, in their order
    if (!alone) {
      if (warp == 0) {
        __threadfence();
        __syncwarp();
        if (lane == 0) {
          uint32_t *cnt = a.counter + (int64_t)(qbase + qi) * a.kv_heads + head;
          last = (int64_t)(qbase + qi) * a.kv_heads + head < a.counters && atomicAdd(cnt, 1u) == (uint32_t)sp - 1;
          if (last) *cnt = 0;  // ready for the next call
        }
      }
      __syncthreads();
      if (last) {
        __threadfence();
        const int64_t stride = (int64_t)a.kv_heads * (COLS * (HD + 2));
        const float *p0 = part - split * stride;
        float *fac = reinterpret_cast<float *>(smem);  // [splits][cols], then the denominators
        for (int col = tid; col < ncol; col += ATT_THREADS) {
          float m = -INFINITY, den = 0.0f;
          for (int i = 0; i < sp; ++i)
            m = fmaxf(m, __ldcg(reinterpret_cast<const float2 *>(p0 + i * stride + COLS * HD) + col).x);
          for (int i = 0; i < sp; ++i) {
            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(p0 + i * stride + COLS * HD) + col);
            const float f = ex2(ml.x - m);
            fac[i * COLS + col] = f;
            den = fmaf(f, ml.y, den);
          }
          red[0][0][col] = den > 0.0f || den != den ? 1.0f / den : 0.0f;
        }
        __syncthreads();
        for (int i = tid; i < ncol * (HD / 8); i += ATT_THREADS) {
          const int col = i / (HD / 8), d = (i % (HD / 8)) * 8, tok = col / a.group;
          float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
          for (int k = 0; k < sp; ++k) {
            const float4 *from = reinterpret_cast<const float4 *>(p0 + k * stride + col * HD + d);
            const float4 u0 = __ldcg(from), u1 = __ldcg(from + 1);
            const float f = fac[k * COLS + col];
            x[0] = fmaf(f, u0.x, x[0]), x[1] = fmaf(f, u0.y, x[1]), x[2] = fmaf(f, u0.z, x[2]), x[3] = fmaf(f, u0.w, x[3]);
            x[4] = fmaf(f, u1.x, x[4]), x[5] = fmaf(f, u1.y, x[5]), x[6] = fmaf(f, u1.z, x[6]), x[7] = fmaf(f, u1.w, x[7]);
          }
          const float f = red[0][0][col];
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] *= f;
          const int64_t row = row0 + tok;
          if (row >= 0 && row < a.rows)
            store8(a.out, a.dtype, row * a.o_row + (int64_t)(head * a.group + col - tok * a.group) * a.o_head + d,
                   a.o_wide, x);
        }
      }
    }
    __syncthreads();  // the ring and the shared sums are free again
  }
}

struct Shape {
  int nt, limbs, qt, cols;
  uint64_t part_units, counters, bytes;
};

// Query columns per unit: the fewest groups of 8 that hold one request's rows,
// up to 32.
Shape shape_of(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a) {
  Shape s;
  const int group = a->heads / c->kv_heads;
  const int64_t cols = (int64_t)group * a->max_new;
  s.nt = cols <= 8 ? 1 : cols <= 16 ? 2 : 4;
  s.limbs = a->dtype == CIS2B_F32 ? 2 : 1;
  s.cols = 8 * s.nt;
  s.qt = s.cols / group;
  const uint64_t tiles = (uint64_t)a->requests + (uint64_t)a->rows / s.qt;  // query tiles at most
  s.counters = tiles * c->kv_heads;
  const uint64_t unit = (uint64_t)s.cols * (c->head_dim + 2) * 4;
  const uint64_t recs = ((uint64_t)a->width * c->page_size + 15) / 16;
  const uint64_t splits = std::min<uint64_t>((recs + ATT_CHUNK - 1) / ATT_CHUNK, ATT_MAX_SPLITS);
  s.part_units = splits < 2 ? 0 : std::min(s.counters * splits, ATT_PART_BYTES / unit);
  s.bytes = (s.counters * 4 + 127) / 128 * 128 + s.part_units * unit;
  return s;
}

int check_attn(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a) {
  if (!a) return kv4_fail(CIS2B_ERR_ARG, "attention: arguments are NULL");
  if (a->reserved) return kv4_fail(CIS2B_ERR_ARG, "attention: reserved must be zero");
  if (a->dtype < CIS2B_F32 || a->dtype > CIS2B_BF16)
    return kv4_fail(CIS2B_ERR_ARG, "attention: dtype must be CIS2B_F32, CIS2B_F16 or CIS2B_BF16");
  if (a->heads < 1 || a->heads % c->kv_heads || a->heads / c->kv_heads > 32)
    return kv4_fail(CIS2B_ERR_ARG, "attention: heads must be a multiple of kv_heads, at most 32 times as many");
  if (a->requests < 1 || a->rows < 0 || a->width < 1 || a->max_new < 1)
    return kv4_fail(CIS2B_ERR_ARG, "attention: requests, width and max_new must be >= 1 and rows >= 0");
  if ((int64_t)a->width * c->page_size > INT_MAX)
    return kv4_fail(CIS2B_ERR_ARG, "attention: width * page_size must be < 2^31");
  if (a->window < 0 || a->sinks < 0) return kv4_fail(CIS2B_ERR_ARG, "attention: window and sinks must be >= 0");
  if (!isfinite(a->scale)) return kv4_fail(CIS2B_ERR_ARG, "attention: scale must be finite");
  return CIS2B_OK;
}

template <int HD, int NT, int LIMBS>
int launch(const AttArgs &args, const cis2b_kv4_cache *c, uint64_t units, int sms, cudaStream_t stream) {
  static std::atomic<int> resident[64];  // blocks per SM, by device; also: the attribute is set
  const int smem = att_smem_bytes<HD, NT, LIMBS>();
  int n = resident[c->device].load(std::memory_order_relaxed);
  if (!n) {
    if (int rc = kv4_cuda(cudaFuncSetAttribute(k_kv4_attention<HD, NT, LIMBS>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem)))
      return rc;
    if (int rc = kv4_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_kv4_attention<HD, NT, LIMBS>,
                                                                        ATT_THREADS, smem)))
      return rc;
    n = std::max(n, 1);
    resident[c->device].store(n, std::memory_order_relaxed);
  }
  const int grid = (int)std::max<uint64_t>(1, std::min<uint64_t>(units, (uint64_t)sms * n));
  k_kv4_attention<HD, NT, LIMBS><<<grid, ATT_THREADS, smem, stream>>>(args);
  return kv4_cuda(cudaGetLastError());
}

template <int HD>
int dispatch(const Shape &s, const AttArgs &args, const cis2b_kv4_cache *c, uint64_t units, int sms, cudaStream_t st) {
  switch (s.nt * 10 + s.limbs) {
    case 11: return launch<HD, 1, 1>(args, c, units, sms, st);
    case 12: return launch<HD, 1, 2>(args, c, units, sms, st);
    case 21: return launch<HD, 2, 1>(args, c, units, sms, st);
    case 22: return launch<HD, 2, 2>(args, c, units, sms, st);
    case 41: return launch<HD, 4, 1>(args, c, units, sms, st);
    default: return launch<HD, 4, 2>(args, c, units, sms, st);
  }
}

}  // namespace
}  // namespace cis2b

using namespace cis2b;

extern "C" int cis2b_kv4_workspace(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, uint64_t *out_bytes) {
  if (int rc = kv4_check_cache(c, false)) return rc;
  if (int rc = check_attn(c, a)) return rc;
  if (!out_bytes) return kv4_fail(CIS2B_ERR_ARG, "out_bytes is NULL");
  *out_bytes = shape_of(c, a).bytes;
  return CIS2B_OK;
}

extern "C" int cis2b_kv4_attention(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, void *stream) {
  if (int rc = kv4_check_cache(c, true)) return rc;
  if (int rc = check_attn(c, a)) return rc;
  if (!a->table || !a->length || !a->row_start || (a->rows && (!a->q || !a->out)))
    return kv4_fail(CIS2B_ERR_ARG, "attention: a device pointer is NULL");
  const Shape s = shape_of(c, a);
  if (a->work_bytes < s.bytes || !a->work || (reinterpret_cast<uintptr_t>(a->work) & 15))
    return kv4_fail(CIS2B_ERR_ARG, "attention: work must be 16-byte aligned and hold cis2b_kv4_workspace() bytes");
  int sms = 0;
  if (int rc = kv4_sm_count(c->device, &sms)) return rc;
  if (int rc = kv4_cuda(cudaSetDevice(c->device))) return rc;
  if (!a->rows) return CIS2B_OK;
  const int64_t unit = a->dtype == CIS2B_F32 ? 4 : 8;
  AttArgs k;
  k.q = a->q, k.out = a->out;
  k.q_row = a->q_row_stride, k.q_head = a->q_head_stride, k.o_row = a->out_row_stride, k.o_head = a->out_head_stride;
  k.q_wide = !(reinterpret_cast<uintptr_t>(a->q) & 15) && !(k.q_row % unit | k.q_head % unit);
  k.o_wide = !(reinterpret_cast<uintptr_t>(a->out) & 15) && !(k.o_row % unit | k.o_head % unit);
  k.pool = static_cast<const uint8_t *>(c->pool), k.status = c->status;
  k.table = a->table, k.length = a->length, k.row_start = a->row_start;
  k.counter = static_cast<uint32_t *>(a->work);
  k.part = reinterpret_cast<float *>(static_cast<uint8_t *>(a->work) + (s.counters * 4 + 127) / 128 * 128);
  k.dtype = a->dtype, k.requests = a->requests, k.rows = a->rows, k.width = a->width, k.kv_heads = c->kv_heads;
  k.group = a->heads / c->kv_heads, k.pages = c->pages, k.window = a->window, k.sinks = a->sinks;
  k.shift = __builtin_ctz(c->page_size);
  k.qt = s.qt;
  k.part_units = (int)std::min<uint64_t>(s.part_units, INT_MAX), k.counters = (int)std::min<uint64_t>(s.counters, INT_MAX);
  k.scale = a->scale;
  const uint64_t recs = ((uint64_t)a->width * c->page_size + 15) / 16;
  const uint64_t units = s.counters * std::min<uint64_t>((recs + ATT_CHUNK - 1) / ATT_CHUNK, ATT_MAX_SPLITS);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return c->head_dim == 64 ? dispatch<64>(s, k, c, units, sms, st) : dispatch<128>(s, k, c, units, sms, st);
}
