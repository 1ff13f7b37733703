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

#include <float.h>
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

namespace cis2b {
namespace {

constexpr int ATT_WARPS = 8;
constexpr int ATT_THREADS = 32 * ATT_WARPS;
constexpr int ATT_LEAST = 8;   // least records (of 16 keys) that a warp is given
constexpr int ATT_SETUP = 6;   // what an item's fixed costs come to, in records
constexpr int ATT_MEET = 8;    // what joining the parts of several blocks comes to, in records

// log2 of the most that a query is scaled up by: its inverse times a usual scale
// is still a normal number.
constexpr int Q_UP = 116;
// log2 of the most that p = exp(score - M) may be: 2^27 of them stay in fp32, and
// the least steps of the format, 2^-100, still make weights of 2^-6 and more.
constexpr float P_MOST = 100.0f;
constexpr float LOWEST = -FLT_MAX;  // a maximum before anything is seen: below every finite score

struct AttArgs {
  const void *q;
  void *out;
  int64_t q_row, q_head, o_row, o_head;
  const uint8_t *pool;
  int32_t *status;
  const int32_t *table, *length, *row_start;
  float *part;        // [10 or 18 per block][cols][HD + 2], see PART below
  uint32_t *counter;  // [items]
  int dtype, requests, rows, width, kv_heads, group, shift, pages, window, sinks;
  int q_wide, o_wide;
  int qt;             // tokens per query tile
  int items, whole;   // a bound on the items (query tiles x KV heads); whole items per block
  float scale;
  float per_warp;     // 1 / warps of the grid, rounded up
};

// A request's first row and its new tokens; 0 where its row starts do not belong
// to this call.  Tokens past the call's rows count for its positions (the step
// had too few rows for them), but have no row: rows_of().
__device__ __forceinline__ int tokens_of(const AttArgs &a, int r, int &row0) {
  row0 = __ldg(a.row_start + r);
  const int row1 = __ldg(a.row_start + r + 1);
  return row0 >= 0 && row0 < a.rows && row1 > row0 ? row1 - row0 : 0;
}
__device__ __forceinline__ int rows_of(const AttArgs &a, int row0, int n) { return n ? min(n, a.rows - row0) : 0; }

// Records of `keys` tokens of a request, and of all pages in its table.  A
// length past the table counts as one record more, whose page is missing, so
// that no caller's length can pass the 32-bit sums below or the workspace.
__device__ __forceinline__ int records(uint32_t keys) { return (int)((keys + 15) >> 4); }
__device__ __forceinline__ int table_records(const AttArgs &a) { return (int)((uint32_t)a.width << (a.shift - 4)); }

// The keys that one query tile sees, as 16-key records 0 .. sink-1 and
// lo .. hi-1.
struct Span {
  int p0, p1;     // first and last position of the tile's rows (p1 < 0: none sees anything)
  int sink, lo;   // records before the gap, first record after it (0 and 0 without one)
  int tiles;      // records in all
};

// `n` new tokens, of which `rows` have a row.
__device__ __forceinline__ Span span_of(const AttArgs &a, int len, int n, int rows, int qt_index) {
  Span s;
  const int first = len - n;
  s.p0 = first + qt_index * a.qt;
  s.p1 = min(first + min((qt_index + 1) * a.qt, rows), len) - 1;
  s.sink = s.lo = s.tiles = 0;
  if (s.p1 < 0) return s;
  const int hi = min((s.p1 >> 4) + 1, table_records(a) + 1);
  if (a.window) {
    const int lo = s.p0 < a.window ? 0 : min((s.p0 - a.window + 1) >> 4, hi - 1);
    const int sink = records(min(a.sinks, s.p1 + 1));
    if (sink < lo) s.sink = sink, s.lo = lo;
  }
  s.tiles = s.sink + hi - s.lo;
  return s;
}

// A bound on span_of().tiles over the query tiles of a request: what each of
// them counts as when the work is shared out.
__device__ __forceinline__ int tiles_bound(const AttArgs &a, int len) {
  const int all = min(records((uint32_t)max(len, 1)), table_records(a) + 1);
  if (!a.window) return all;
  const uint32_t keys = (uint32_t)all * 16;
  const int some = records(min((uint32_t)a.sinks, keys)) + (int)((min((uint32_t)a.window, keys) + a.qt - 2) >> 4) + 2;
  return min(all, some);
}
// How a query row of largest element `top` becomes an operand: times f, a power
// of two that brings it to 2^13 .. 2^14 (with the scale's sign), so that 16-bit
// elements down to 2^-24 of it stay exact.  The scores are then
//   factor (raw * step_factor * unit * ks + kz * sum_of(sum(q)))
// where raw is the product of the operands in units of the codes' operands.
// With the scale's mantissa in the second factors, factor is a positive power
// of two: a score times it is the same number wherever it is formed, and
// -infinity stays that.
struct QueryScale {
  float f, factor, of_sum;
  // A row with an infinity has NaN for every key that it sees (an infinite sum
  // could make -infinity of each, which is a mask's).
  __device__ __forceinline__ float sum_of(float sum) const { return sum * f * of_sum; }
};
constexpr float SCORE_UNIT = 16384.0f;  // of factor; in the middle of the range of what products can be
__device__ __forceinline__ float mantissa_of(float sl) {
  const uint32_t bits = __float_as_uint(sl) & 0x7fffffffu;
  return bits >> 23 ? __uint_as_float((bits & 0x7fffffu) | 0x3f800000u) : 1.0f;
}
__device__ __forceinline__ float step_factor(float scale) { return mantissa_of(scale * 1.4426950408889634f) / SCORE_UNIT; }
__device__ __forceinline__ QueryScale query_scale(float scale, float top) {
  const float sl = scale * 1.4426950408889634f;
  const int e = (int)(__float_as_uint(top) >> 23);  // biased exponent
  const int up = e == 0 || e == 255 ? 0 : min(13 - (e - 127), Q_UP);
  const float f = __uint_as_float((uint32_t)(127 + up) << 23);
  const float back = __uint_as_float(__float_as_uint(sl) & 0x7f800000u) * __uint_as_float((uint32_t)(127 - up) << 23) * SCORE_UNIT;
  QueryScale s;
  s.f = sl > 0.0f ? f : sl < 0.0f ? -f : 0.0f;
  s.factor = sl == 0.0f ? 1.0f : fminf(fmaxf(back, 0x1p-126f), 0x1p126f);
  s.of_sum = top == INFINITY ? __int_as_float(0x7fffffff) : mantissa_of(sl) / SCORE_UNIT;
  return s;
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
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool on) {
  asm volatile("{.reg .pred p; setp.ne.b32 p, %2, 0; @p cp.async.cg.shared.global [%0], [%1], 16;}" ::"r"(dst), "l"(src),
               "r"((int)on));
}
// Four 8 x 8 matrices of 16-bit units, transposed: lane (g, t) gets units
// (2t, g) and (2t + 1, g) of each; lane l gives row l % 8 of matrix l / 8.
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// Pairs of fp32 numbers in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 x, y, z; mov.b64 x, {%2,%3}; mov.b64 y, {%4,%5}; mul.rn.f32x2 z, x, y; mov.b64 {%0,%1}, z;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 x, y, z; mov.b64 x, {%2,%3}; mov.b64 y, {%4,%5}; add.rn.f32x2 z, x, y; mov.b64 {%0,%1}, z;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{.reg .b64 x, y, z, w; mov.b64 x, {%2,%3}; mov.b64 y, {%4,%5}; mov.b64 z, {%6,%7}; fma.rn.f32x2 w, x, y, z; "
      "mov.b64 {%0,%1}, w;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
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

// What a value's weight is bounded by: its step, and, where that is smaller by
// OF_BASE, its base (at code 7.5).  Numbers that no caller's group has, negative
// steps and NaN, bound nothing.
constexpr float OF_BASE = 0x1p-80f;
__device__ __forceinline__ float size_of(float step, float base) { return fmaxf(fmaxf(step, 0.0f), fabsf(base) * OF_BASE); }

// Four elements of a column's result: numerators over the denominator (zero
// where nothing was seen).
__device__ __forceinline__ void emit(const AttArgs &a, int row0, int head, int col, int d, float4 x, float den) {
  const float f = den > 0.0f || den != den ? 1.0f / den : 0.0f;
  const int tok = col / a.group;
  const int64_t row = (int64_t)row0 + tok;
  if (row >= 0 && row < a.rows)
    store4(a.out, a.dtype, row * a.o_row + (int64_t)(head * a.group + col - tok * a.group) * a.o_head + d, a.o_wide,
           make_float4(x.x * f, x.y * f, x.z * f, x.w * f));
}

// Parts of a column joined, four elements of it: n parts `stride` floats apart,
// then one more at `extra` (unless NULL).  col_at and ml_at are the places of
// the elements and of (maximum, denominator) in a part.
struct Joined {
  float4 x;
  float m, den;
};
__device__ __forceinline__ Joined join_parts(const float *p, int64_t stride, int n, const float *extra, int col_at, int ml_at) {
  Joined s = {make_float4(0, 0, 0, 0), LOWEST, 0.0f};
  const int all = n + (extra != nullptr);
  constexpr int AT_ONCE = 4;
  for (int k = 0; k < all; k += AT_ONCE) {
    float4 y[AT_ONCE];
    float2 ml[AT_ONCE];
    float top = s.m;
#pragma unroll
    for (int e = 0; e < AT_ONCE; ++e) {
      const float *q = k + e < n ? p + (k + e) * stride : extra;
      ml[e] = make_float2(LOWEST, 0.0f), y[e] = make_float4(0, 0, 0, 0);
      if (k + e < all) ml[e] = *reinterpret_cast<const float2 *>(q + ml_at), y[e] = *reinterpret_cast<const float4 *>(q + col_at);
    }
#pragma unroll
    for (int e = 0; e < AT_ONCE; ++e) top = fmaxf(top, ml[e].x);
    const float keep = ex2(s.m - top);
    s.m = top, s.den *= keep, s.x.x *= keep, s.x.y *= keep, s.x.z *= keep, s.x.w *= keep;
#pragma unroll
    for (int e = 0; e < AT_ONCE; ++e) {
      const float f = ex2(ml[e].x - top);
      s.den = fmaf(f, ml[e].y, s.den);
      s.x.x = fmaf(f, y[e].x, s.x.x), s.x.y = fmaf(f, y[e].y, s.x.y);
      s.x.z = fmaf(f, y[e].z, s.x.z), s.x.w = fmaf(f, y[e].w, s.x.w);
    }
  }
  return s;
}

// The codes in bits 4-7 (high) or 0-3 (low) of each 16-bit half as the normal
// half-precision numbers 16 (c - 7.5).  Centred at 7.5, sums over many values
// have no drift that the bases' sums would have to cancel.  The low codes'
// second operation is on the multiply-add pipe, which has room; a shift into
// the high ones' place would be on the other, which has not.
__device__ __forceinline__ uint32_t codes_high(uint32_t x) {
  const uint32_t y = (x & 0x00f000f0u) | 0x64006400u;  // 1024 + 16 c
  const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&y), __half2half2(__ushort_as_half(0x6478)));
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t codes_low(uint32_t x) {
  const uint32_t y = (x & 0x000f000fu) | 0x64006400u;  // 1024 + c
  const __half2 c = __hsub2(*reinterpret_cast<const __half2 *>(&y), __half2half2(__ushort_as_half(0x6400)));
  const __half2 h = __hfma2(c, __half2half2(__ushort_as_half(0x4c00)), __half2half2(__ushort_as_half(0xd780)));  // 16 c - 120
  return *reinterpret_cast<const uint32_t *>(&h);
}
// The four codes of each half in order, as operands that stand for 1 / unit of
// a code: 16 exactly, else 2^-24 (even) and 2^-20 (odd).
template <bool EXACT> __device__ __forceinline__ void codes_of(uint32_t x, uint32_t (&c)[4]) {
  const uint32_t y = x >> 8;
  if constexpr (EXACT) {
    c[0] = codes_low(x), c[1] = codes_high(x), c[2] = codes_low(y), c[3] = codes_high(y);
  } else {
    c[0] = x & 0x000f000fu, c[1] = x & 0x00f000f0u, c[2] = y & 0x000f000fu, c[3] = y & 0x00f000f0u;
  }
}

// Records that a warp takes per iteration (one where two would spill: spilled
// registers come back from L2, since the rings take L1's place; 48 against 44 us
// at 130,051 keys), iterations in its ring, and the shared memory of a block:
// its warps' rings, then their query operands.
__host__ __device__ constexpr int att_pair(int hd, int nt) { return nt < 4 && !(hd == 128 && nt == 1) ? 2 : 1; }
__host__ __device__ constexpr int att_stages(int hd, int nt) { return hd == 128 && nt == 1 ? 6 : nt < 4 ? (hd == 64 ? 4 : 3) : (hd == 64 ? 6 : 4); }
__host__ __device__ constexpr int att_ring_bytes(int hd, int nt) {
  return ATT_WARPS * att_stages(hd, nt) * att_pair(hd, nt) * kv4_rec_bytes(hd);
}
__host__ __device__ constexpr int att_smem_bytes(int hd, int nt, int limbs) {
  return att_ring_bytes(hd, nt) + (nt > 1 ? ATT_WARPS * nt * limbs * (hd / 32) * 512 : 0);
}

// Whether a ring has room for the part of an item that goes on after the warp;
// parts that a block has in the workspace.
__host__ __device__ constexpr bool att_on_shared(int hd, int nt) {
  return 8 * nt * (hd + 2) * 4 <= att_stages(hd, nt) * att_pair(hd, nt) * kv4_rec_bytes(hd);
}
__host__ __device__ constexpr int att_parts(int hd, int nt) { return ATT_WARPS + 2 + (att_on_shared(hd, nt) ? 0 : ATT_WARPS); }

// An item is a query tile of one request and one KV head.  The records of all
// items stand in one row, (request, query tile, KV head, record), with a gap
// of ATT_SETUP before each item for its fixed costs, and every warp of the
// grid takes an equal stretch of it: each has the same work, whatever the
// requests' lengths, and none waits for another on the way.  Items that are
// cut are put together at the end: the parts of a block's eight warps in
// shared memory, the parts of several blocks through the workspace by the
// last block to arrive.  Both join parts in the order of their records, so
// the result does not depend on which block that is.  Where items are short,
// and with CIS2B_KV4_WHOLE, a block takes whole items in turn, an eighth per
// warp, and nothing is left for other blocks; a row's result then does not
// depend on the rest of the batch.
//
// The codes reach the tensor pipe almost as they are.  Of bf16 rows: a code in
// bits 0-3 of a 16-bit word IS the half-precision number c * 2^-24 (a
// subnormal), and in bits 4-7 c * 2^-20, so `and` makes two operands out of a
// 32-bit word, and the factor of 16 is divided out of every other query
// element (keys) or output row (values).  The tensor pipe lines subnormal
// products up by their exponent field and drops what falls below its sums (in
// fp32), so a sum keeps about 15 bits (measured: 4e-5 of fp32 rows' results,
// 2.4 times plain fp16's error at 130,051 keys), enough for 8-bit results: the
// error of bf16 rows is 1.66e-3 there, 1.56e-3 of which is the results' own
// rounding, and exact codes would take 134 us in place of 102 over a ragged
// batch of 64.  fp16 and fp32 rows (EXACT) pay one or two more operations for
// the normal numbers 16 (c - 7.5).
//
// The cache's bytes bound bf16 rows, instructions the others: HBM at its measured
// rate gives an SM a record of head_dim 128 every 93 cycles, and the 280 (bf16),
// 437 (fp16) and 483 (fp32) warp instructions per record, all included, are 70,
// 109 and 121 cycles of issue; a call over 206,616 records takes 109, 136 and 174
// us, 8 rows per request 334, 316 and 412.  Around the records a call spends
// about 10,000 cycles until the first one is there and 10,000 to 20,000 joining
// parts.  Measured on the way: a block per 512 keys with tickets 184 us for the
// ragged batch of 64 (a unit's fixed costs are 12,000 cycles), even stretches
// per block 132, per warp 119 to 105.
//
// Keys are the 16 rows of the first product and head_dim the 16 rows of the
// second, with the query rows (tokens x group) as its 8 columns, so that a
// group of up to 8 heads wastes nothing and a warp's lanes hold 4 scores per
// record.  The probabilities go from the first product's accumulator layout
// to the second's operand layout by an 8 x 8 register transpose.
//
// M is a lazy maximum per column: it moves only when a weight p * vs (the
// number that is rounded to half precision) passes 2^14, or p 2^100, or p |vz|
// 2^94 (whose sum stays in fp32: of groups of one large number, with step 0),
// and then to 2^8 below the top.  Whether one might is asked per lane, unseen
// keys' parameters included; the move goes by the keys that the column sees.  Weights keep 11 bits down to 2^-22 of the
// largest; LIMBS = 2 (fp32 rows) adds a second half-precision limb to the
// weights and the query, 22 bits.  Codes are centred at 7.5, which halves the
// rounding's effect: directly where EXACT, else by the sum of the rounded
// weights (a product with ones).
template <int HD, int NT, int LIMBS, bool EXACT>
__global__ __launch_bounds__(ATT_THREADS, NT == 1 ? 2 : 1) void k_kv4_attention(AttArgs a) {
  constexpr int REC = kv4_rec_bytes(HD), ST = att_stages(HD, NT), RP = att_pair(HD, NT);
  constexpr int KS = HD / 16;            // k-steps of the first product, row tiles of the second
  constexpr int W = HD / 32;             // 32-bit words of a key row per lane
  constexpr int COLS = 8 * NT;
  // Parts that a block has in the workspace: items that end in each warp, the
  // block's first and last item, and, where a ring cannot hold one, items
  // that go on after each warp.
  constexpr bool ON_SHARED = att_on_shared(HD, NT);
  constexpr int PARTS = att_parts(HD, NT);
  // A code's operand is the code over this, of even and odd elements.
  constexpr float EVEN = EXACT ? 1.0f / 16.0f : 16777216.0f, ODD = EXACT ? 1.0f / 16.0f : 1048576.0f;
  // Sums and factors of the query columns, where registers are short (measured 7
  // to 10 percent slower with them in registers, which spill).
  constexpr bool COLUMNS_SHARED = NT == 4;
  __shared__ float4 column_of[COLUMNS_SHARED ? ATT_WARPS : 1][NT][4];
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int scan_t[ATT_THREADS], scan_q[ATT_THREADS], warp_t[ATT_WARPS], warp_top[ATT_WARPS];
  __shared__ int64_t warp_q[ATT_WARPS];
  __shared__ int req_len[ATT_THREADS], req_row[ATT_THREADS], req_n[ATT_THREADS];  // of up to as many requests
  // Each warp's cut items: one that ends in it, one that goes on after it.
  struct Cut {
    int item, row0, head, ncol, begin, size;  // begin and size: its stretch of the row
  };
  __shared__ Cut cut_end[ATT_WARPS], cut_on[ATT_WARPS];
  __shared__ int has_end[ATT_WARPS], on_kind[ATT_WARPS];  // on: 0 none, 1 the item begins here, 2 it began before
  struct Run {  // the parts of one item within the block: `on` of warps w .., then the one that ends it
    int on, end, side;  // end: its warp or -1; side: 0 began before the block, 1 goes on after it, 2 done here, -1 no run
  };
  __shared__ Run run[ATT_WARPS + 1];  // by the warp it begins in; the last: what began before the block
  __shared__ Cut edge[2];       // the block's items that began before it and that go on after it
  __shared__ int edge_last[2];  // 0: no such item, 1: left to another block, 2: to be joined here
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint8_t *ring = smem + warp * ST * RP * REC;
  uint4 *qfrag = reinterpret_cast<uint4 *>(smem + att_ring_bytes(HD, NT)) + warp * (NT * LIMBS * W * 32);

  // Records (with the gaps) and items before each request: thread i sums
  // requests i * per .. of its own.
  const int per = (a.requests + ATT_THREADS - 1) / ATT_THREADS;
  int all_tiles = 0, top_tiles = 1;
  int64_t all_q = 0;
  {
    int st = 0, top = 1;
    int64_t sq = 0;
    for (int r = tid * per; r < min(tid * per + per, a.requests); ++r) {
      int row;
      const int n = tokens_of(a, r, row), on = rows_of(a, row, n), len = __ldg(a.length + r);
      if (per == 1) req_len[r] = len, req_row[r] = row, req_n[r] = n;
      if (n == 0) continue;
      const int nq = on <= a.qt ? 1 : (on + a.qt - 1) / a.qt;
      const int vt = tiles_bound(a, len);
      st += nq * (vt + ATT_SETUP), sq += nq, top = max(top, vt);
    }
    const int own_t = st;
    const int64_t own_q = sq;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, st, d);
      const int64_t y = __shfl_up_sync(0xffffffffu, sq, d);
      if (lane >= d) st += x, sq += y;
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 31) warp_t[warp] = st, warp_q[warp] = sq, warp_top[warp] = top;
    __syncthreads();
    int before_t = 0;
    int64_t before_q = 0;
#pragma unroll
    for (int w = 0; w < ATT_WARPS; ++w) {
      if (w < warp) before_t += warp_t[w], before_q += warp_q[w];
      all_tiles += warp_t[w], all_q += warp_q[w], top_tiles = max(top_tiles, warp_top[w]);
    }
    scan_t[tid] = (before_t + st - own_t) * a.kv_heads;
    scan_q[tid] = (int)(before_q + sq - own_q) * a.kv_heads;
    __syncthreads();
  }
  // Requests that overlap in their rows can have more query tiles than the host
  // counted with: such row starts have no items.
  const bool fits = all_q * a.kv_heads <= a.items;
  all_tiles = fits ? all_tiles * a.kv_heads : 0;
  const int items = fits ? (int)all_q * a.kv_heads : 0;
  // A range's records: an equal share, but not so few that the joins outweigh them.
  const int range = (int)blockIdx.x * ATT_WARPS + warp;
  const int each = max(__float2int_ru(__fmul_ru(__int2float_ru(all_tiles), a.per_warp)), ATT_LEAST);
  // Whole items, too, where the longest is short enough that a block's turns
  // take no longer than an even share and joining its ends.
  const int turns = (int)((uint32_t)(items + gridDim.x - 1) / gridDim.x);
  const bool whole = a.whole || (turns <= 64 && turns * ((top_tiles + ATT_WARPS - 1) / ATT_WARPS + ATT_SETUP) <= each + ATT_SETUP + ATT_MEET);
  const int *scan = whole ? scan_q : scan_t;

  for (int turn_at = blockIdx.x;; turn_at += gridDim.x) {  // once, or once per whole item
  int at = whole ? turn_at : (int)min((int64_t)range * each, (int64_t)all_tiles);
  const int end = whole ? (turn_at < items ? turn_at + 1 : turn_at) : (int)min((int64_t)at + each, (int64_t)all_tiles);
  if (whole ? at >= end : (int64_t)blockIdx.x * ATT_WARPS * each >= all_tiles) break;  // as one block
  if (lane == 0) has_end[warp] = on_kind[warp] = 0;
  while (at < end) {
    // ---- which item, and which of its records
    int seg;
    {
      const uint32_t coarse = __ballot_sync(0xffffffffu, scan[lane * (ATT_THREADS / 32)] <= at);
      seg = (31 - __clz(coarse)) * (ATT_THREADS / 32);
      const uint32_t fine = __ballot_sync(0xffffffffu, scan[seg + (lane & (ATT_THREADS / 32 - 1))] <= at);
      seg += 31 - __clz(fine & ((1u << (ATT_THREADS / 32)) - 1));
    }
    int base = scan[seg], qbase = scan_q[seg], r = seg * per, n, on, len, row0, nq, vt, size;
    for (; r < a.requests; ++r) {
      if (per == 1) {
        len = req_len[r], row0 = req_row[r], n = req_n[r];
      } else {
        len = __ldg(a.length + r), n = tokens_of(a, r, row0);
      }
      if (n == 0) continue;
      on = rows_of(a, row0, n);
      nq = on <= a.qt ? 1 : (on + a.qt - 1) / a.qt;
      vt = tiles_bound(a, len);
      size = whole ? 1 : vt + ATT_SETUP;  // of one item in the row
      const int next = base + nq * a.kv_heads * size;
      if (at < next) break;
      base = next, qbase += nq * a.kv_heads;
    }
    if (r >= a.requests) break;  // row starts that do not belong together
    const int item = (int)((uint32_t)(at - base) / (uint32_t)size);
    const int turn = nq == 1 ? 0 : (int)((uint32_t)item / (uint32_t)a.kv_heads), head = item - turn * a.kv_heads;
    // Later query tiles see more: taken from both ends in turn, so that any
    // stretch of them is about average.
    const int qi = turn & 1 ? nq - 1 - turn / 2 : turn / 2;
    const Span s = span_of(a, len, n, on, qi);
    int from, to, begin = 0;  // records of the item; where it begins in the row
    if (whole) {
      const int share = max((s.tiles + ATT_WARPS - 1) / ATT_WARPS, 1);
      from = min(warp * share, s.tiles), to = min(from + share, s.tiles);
      at = end;
    } else {
      begin = base + item * size + ATT_SETUP;
      if (begin >= end) break;
      from = max(at, begin) - begin, to = min(vt, end - begin);
      at = begin + to;
    }
    const int t_begin = min(from, s.tiles), t_end = min(to, s.tiles);
    row0 += qi * a.qt;
    const int ncol = min(a.qt, on - qi * a.qt) * a.group;

    // ---- this warp's records
    const int32_t *row_table = a.table + (int64_t)r * a.width;
    const int recs_shift = a.shift - 4;
    auto key_rec = [&](int tile) { return tile < s.sink ? tile : tile - s.sink + s.lo; };
    // Records in which every row of the item sees every key: sinks 0 .. all_sink-1
    // and all_lo .. all_hi-1.
    const int shiftr = s.sink - s.lo;
    const int all_hi = ((s.p0 + 1) >> 4) + shiftr;
    const int all_lo = a.window ? max(s.sink, records(max(0, s.p1 - a.window + 1)) + shiftr) : 0;
    const int all_sink = min(a.window ? a.sinks >> 4 : 0, min((s.p0 + 1) >> 4, s.sink));
    // Lane i looks up record i of the next 32: its index in the pool, or NONE.
    constexpr uint32_t NONE = 0xffffffffu;
    auto look_up = [&](int tile) {
      if (tile >= t_end) return NONE;
      const int rec = key_rec(tile), p = rec >> recs_shift;
      const int pg = p < a.width ? __ldg(row_table + p) : -1;
      if (pg >= a.pages || pg < 0) {
        if (a.status) atomicOr(a.status, CIS2B_KV4_BAD_PAGE);
        return NONE;
      }
      return (((uint32_t)pg * a.kv_heads + head) << recs_shift) + (rec & ((1 << recs_shift) - 1));
    };
    uint32_t ids = look_up(t_begin + lane), ids_next = look_up(t_begin + 32 + lane);
    int ahead = t_begin;  // next record to fetch
    uint32_t held = 0;    // bit i: slot i of the ring holds a record of the pool
    // 16-byte pieces move within their 128 bytes so that the operand loads
    // below touch every bank once; the parameters' 8 pieces stay in place.
    const uint32_t ring_base = (uint32_t)__cvta_generic_to_shared(ring), ring_at = ring_base + (lane ^ ((lane >> 3) & 3)) * 16;
    auto fetch = [&](int slot) {
      const int i = (ahead - t_begin) & 31;
      if (i == 0 && ahead != t_begin) ids = ids_next, ids_next = look_up(ahead + 32 + lane);
      const uint32_t id = __shfl_sync(0xffffffffu, ids, i);
      const bool on = id != NONE;
      held = (held & ~(1u << slot)) | (uint32_t)on << slot;
      const uint8_t *src = a.pool + (uint64_t)(on ? id : 0u) * REC + lane * 16;
      const uint32_t dst = ring_at + slot * REC;
#pragma unroll
      for (int k = 0; k < HD / 32; ++k) cp_async16(dst + k * 512, src + k * 512, on);
      cp_async16(dst + HD * 16, src + HD * 16, on && lane < 8);
      ++ahead;
    };
    // ---- query operands: lane (g, t) holds elements t HD/4 .. of column g
    uint32_t bq[NT == 1 ? LIMBS : 1][NT == 1 ? KS : 1][2];
    // Of this lane's two columns: a score is factor (raw * ks + kz * sum_s), see QueryScale.
    float2 sum_s[COLUMNS_SHARED ? 1 : NT], factor[COLUMNS_SHARED ? 1 : NT];
    const float of_step = step_factor(a.scale) * EVEN;
    int pos[NT][2];
    {
      float x[NT][4 * W][2], f[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int col = 8 * j + g, tok = col / a.group;
        const int64_t row = (int64_t)row0 + tok;
        float sum = 0.0f;
        float e[8 * W];
        const bool on = col < ncol && row >= 0 && row < a.rows;
        const int64_t from_q = row * a.q_row + (int64_t)(head * a.group + col - tok * a.group) * a.q_head + t * (HD / 4);
        load_query<LIMBS == 2, 8 * W>(a.q, a.dtype == KV4_BF16, from_q, a.q_wide, on, e);
        if (j == 0) {  // the first records are asked for after the first queries, which would wait behind them
#pragma unroll
          for (int i = 0; i < ST - 1; ++i) {
#pragma unroll
            for (int k = 0; k < RP; ++k) fetch(i * RP + k);
            cp_async_commit();
          }
        }
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8 * W; ++i) top = fmaxf(top, fabsf(e[i])), sum += e[i];
        // Word w's `and`s give the code pairs (0,4) (1,5) (2,6) (3,7).
#pragma unroll
        for (int i = 0; i < 4 * W; ++i) x[j][i][0] = e[(i & ~3) * 2 + (i & 3)], x[j][i][1] = e[(i & ~3) * 2 + (i & 3) + 4];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const QueryScale own = query_scale(a.scale, top);
        f[j] = own.f;
        sum = own.sum_of(sum);
        const int to = COLUMNS_SHARED ? 0 : j;
        sum_s[to] = make_float2(__shfl_sync(0xffffffffu, sum, 8 * t), __shfl_sync(0xffffffffu, sum, 8 * t + 4));
        factor[to] = make_float2(__shfl_sync(0xffffffffu, own.factor, 8 * t), __shfl_sync(0xffffffffu, own.factor, 8 * t + 4));
        if (COLUMNS_SHARED && g == 0) column_of[warp][j][t] = make_float4(sum_s[0].x, sum_s[0].y, factor[0].x, factor[0].y);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int cc = 8 * j + 2 * t + c;
          pos[j][c] = cc < ncol ? s.p0 + cc / a.group : -1;
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          uint32_t v[LIMBS][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float k = (i & 1) && !EXACT ? f[j] * 0.0625f : f[j];
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
            } else {
              qfrag[((j * LIMBS + l) * W + w) * 32 + lane] = make_uint4(v[l][0], v[l][1], v[l][2], v[l][3]);
            }
          }
        }
      }
    }
    if constexpr (NT > 1) __syncwarp();

    float o[NT][KS][4], ones[NT][4];
    float2 M[NT], l[NT], z[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int m = 0; m < KS; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][m][i] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ones[j][i] = 0.0f;
      M[j] = make_float2(LOWEST, LOWEST), l[j] = z[j] = make_float2(0.0f, 0.0f);
    }
    int stage = 0;
    for (int tile = t_begin; tile < t_end; tile += RP) {
      {
        const int to = stage == 0 ? ST - 1 : stage - 1;
#pragma unroll
        for (int k = 0; k < RP; ++k) fetch(to * RP + k);
        cp_async_commit();
      }
      cp_async_wait<ST - 1>();
      __syncwarp();
      const uint32_t here = held >> (stage * RP);
      const bool unmasked = (here & ((1u << RP) - 1)) == (1u << RP) - 1 &&
                         ((tile >= all_lo && tile + RP <= all_hi) || tile + RP <= all_sink);

      // scores: keys g and g + 8 of each record by columns 2t, 2t + 1
      float sc[RP][NT][4];
#pragma unroll
      for (int k = 0; k < RP; ++k) {
        const uint8_t *rec = ring + (stage * RP + k) * REC;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[k][j][i] = 0.0f;
        uint32_t ka[W], kb[W];
        if constexpr (HD == 128) {
          // piece 4 key + t, moved by its line (two keys) within the record
          const int at = (((g & 1) * 4 + t) ^ (g >> 1)) * 16 + (g >> 1) * 128;
          const uint4 x = *reinterpret_cast<const uint4 *>(rec + at);
          const uint4 y = *reinterpret_cast<const uint4 *>(rec + at + 512);
          ka[0] = x.x, ka[1] = x.y, ka[2] = x.z, ka[3] = x.w;
          kb[0] = y.x, kb[1] = y.y, kb[2] = y.z, kb[3] = y.w;
        } else {
          // lines of four keys; keys 8 .. 15 are lines 2 and 3
          const int c = 2 * g + (t >> 1), line = c >> 3;
          const int at = ((c & 7) ^ line) * 16 + line * 128 + (t & 1) * 8;
          const int au = ((c & 7) ^ (line + 2)) * 16 + (line + 2) * 128 + (t & 1) * 8;
          const uint2 x = *reinterpret_cast<const uint2 *>(rec + at);
          const uint2 y = *reinterpret_cast<const uint2 *>(rec + au);
          ka[0] = x.x, ka[1] = x.y, kb[0] = y.x, kb[1] = y.y;
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
          uint32_t x[4], y[4];
          codes_of<EXACT>(ka[w], x);
          codes_of<EXACT>(kb[w], y);
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int lm = 0; lm < LIMBS; ++lm) {
              if constexpr (NT == 1) {
                mma16816(sc[k][j], x[0], y[0], x[1], y[1], bq[lm][2 * w][0], bq[lm][2 * w][1]);
                mma16816(sc[k][j], x[2], y[2], x[3], y[3], bq[lm][2 * w + 1][0], bq[lm][2 * w + 1][1]);
              } else {
                const uint4 f = qfrag[((j * LIMBS + lm) * W + w) * 32 + lane];
                mma16816(sc[k][j], x[0], y[0], x[1], y[1], f.x, f.y);
                mma16816(sc[k][j], x[2], y[2], x[3], y[3], f.z, f.w);
              }
            }
        }
      }
      // parameters of keys g and g + 8; a value's base is taken at code 7.5
      float ks[2 * RP], kz[2 * RP], vs[2 * RP], vz[2 * RP];
#pragma unroll
      for (int i = 0; i < 2 * RP; ++i) {
        const uint8_t *rec = ring + (stage * RP + (i >> 1)) * REC;
        const uint2 p = *reinterpret_cast<const uint2 *>(rec + 16 * HD + (g + 8 * (i & 1)) * 8);
        ks[i] = bf16_lo(p.x) * of_step;
        kz[i] = EXACT ? fmaf(7.5f, bf16_lo(p.x), bf16_hi(p.x)) : bf16_hi(p.x);
        vs[i] = bf16_lo(p.y), vz[i] = fmaf(7.5f, vs[i], bf16_hi(p.y));
      }
      float z_most = 0.0f;
#pragma unroll
      for (int i = 0; i < 2 * RP; ++i) z_most = fmaxf(z_most, fabsf(vz[i]));
      const float p_bound = fmaxf(0x1p-86f, z_most * OF_BASE);  // 2^14 over 2^P_MOST
      uint32_t bw[RP][NT][LIMBS][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        constexpr int E = 2 * RP;  // pair i: key g + 8 (i & 1) of record i >> 1, columns 2t and 2t + 1
        float2 tt[E], p[E], w[E], vse[E], vze[E];
        float2 sum_j, factor_j;
        if constexpr (COLUMNS_SHARED) {
          const float4 c = column_of[warp][j][t];
          sum_j = make_float2(c.x, c.y), factor_j = make_float2(c.z, c.w);
        } else {
          sum_j = sum_s[j], factor_j = factor[j];
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float2 raw = make_float2(sc[i >> 1][j][2 * (i & 1)], sc[i >> 1][j][2 * (i & 1) + 1]);
          tt[i] = fma2(raw, make_float2(ks[i], ks[i]), mul2(make_float2(kz[i], kz[i]), sum_j));
          vse[i] = make_float2(vs[i], vs[i]), vze[i] = make_float2(vz[i], vz[i]);
        }
        if (!unmasked) {
#pragma unroll
          for (int i = 0; i < E; ++i) {
            const int key = key_rec(tile + (i >> 1)) * 16 + g + 8 * (i & 1);
            const bool in = (here >> (i >> 1)) & 1;
            auto sees = [&](int at) { return in && key <= at && (a.window == 0 || key > at - a.window || key < a.sinks); };
            // Whatever the cache holds there.
            if (!sees(pos[j][0])) tt[i].x = -INFINITY, vse[i].x = vze[i].x = 0.0f;
            if (!sees(pos[j][1])) tt[i].y = -INFINITY, vse[i].y = vze[i].y = 0.0f;
          }
        }
        const float2 minus_m = make_float2(-M[j].x, -M[j].y);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float2 u = fma2(tt[i], factor_j, minus_m);
          p[i] = make_float2(ex2(u.x), ex2(u.y));
          w[i] = mul2(p[i], vse[i]);
        }
        float2 chk = w[0], big = p[0];
#pragma unroll
        for (int i = 1; i < E; ++i) {
          chk.x = fmaxf(chk.x, w[i].x), chk.y = fmaxf(chk.y, w[i].y);
          big.x = fmaxf(big.x, p[i].x), big.y = fmaxf(big.y, p[i].y);
        }
        chk.x = fmaxf(chk.x, big.x * p_bound), chk.y = fmaxf(chk.y, big.y * p_bound);
        if (__any_sync(0xffffffffu, fmaxf(chk.x, chk.y) > 0x1p14f)) {
          float2 tw = make_float2(-INFINITY, -INFINITY), ts = tw;
#pragma unroll
          for (int i = 0; i < E; ++i) tt[i] = mul2(tt[i], factor_j);
#pragma unroll
          for (int i = 0; i < E; ++i) {
            tw.x = fmaxf(tw.x, tt[i].x + lg2(size_of(vse[i].x, vze[i].x))), tw.y = fmaxf(tw.y, tt[i].y + lg2(size_of(vse[i].y, vze[i].y)));
            ts.x = fmaxf(ts.x, tt[i].x), ts.y = fmaxf(ts.y, tt[i].y);
          }
          auto raise = [&](float &m, float w_top, float t_top) {  // the factor for what was summed
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
              w_top = fmaxf(w_top, __shfl_xor_sync(0xffffffffu, w_top, d));
              t_top = fmaxf(t_top, __shfl_xor_sync(0xffffffffu, t_top, d));
            }
            if (!(fmaxf(w_top - 14.0f, t_top - P_MOST) > m)) return 1.0f;
            const float before = m;
            m = fmaxf(w_top - 8.0f, t_top - (P_MOST - 6.0f));
            return ex2(before - m);
          };
          const float2 f = make_float2(raise(M[j].x, tw.x, ts.x), raise(M[j].y, tw.y, ts.y));
          l[j] = mul2(l[j], f), z[j] = mul2(z[j], f);
          ones[j][0] *= f.x, ones[j][1] *= f.y;
#pragma unroll
          for (int k = 0; k < KS; ++k) o[j][k][0] *= f.x, o[j][k][1] *= f.y, o[j][k][2] *= f.x, o[j][k][3] *= f.y;
#pragma unroll
          for (int i = 0; i < E; ++i) {
            p[i] = make_float2(ex2(tt[i].x - M[j].x), ex2(tt[i].y - M[j].y));
            w[i] = mul2(p[i], vse[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < E; ++i) l[j] = add2(l[j], p[i]), z[j] = fma2(p[i], vze[i], z[j]);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const uint32_t h = pack_half(w[i].x, w[i].y);
          bw[i >> 1][j][0][i & 1] = transpose8x8(h);
          if constexpr (LIMBS == 2) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
            bw[i >> 1][j][1][i & 1] = transpose8x8(pack_half(w[i].x - f.x, w[i].y - f.y));
          }
        }
      }
      // values: lane (g, t) holds 16-bit units (four codes) of keys 2t, 2t + 1
      // and of 2t + 8, 2t + 9; unit g of the W pieces of 32 elements
#pragma unroll
      for (int k = 0; k < RP; ++k) {
        const uint32_t vb = ring_base + (stage * RP + k) * REC + 8 * HD;
        uint32_t v[2][W];  // [key half][piece]
#pragma unroll
        for (int h = 0; h < W / 2; ++h) {
          // matrices: pieces 2h and 2h + 1 of keys 0-7, then of keys 8-15
          const int key = (lane & 7) + 8 * (lane >> 4), piece = 2 * h + ((lane >> 3) & 1);
          const int c = key * W + piece, line = c >> 3;
          uint32_t r4[4];
          ldmatrix4_trans(r4, vb + line * 128 + ((c & 7) ^ (line & 3)) * 16);
          v[0][2 * h] = r4[0], v[0][2 * h + 1] = r4[1], v[1][2 * h] = r4[2], v[1][2 * h + 1] = r4[3];
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
          uint32_t x[4], y[4];
          codes_of<EXACT>(v[0][w], x);
          codes_of<EXACT>(v[1][w], y);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int m = 2 * w + q;  // rows of elements 32 w + 4 g + 2 q and the next
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int lm = 0; lm < LIMBS; ++lm)
                mma16816(o[j][m], x[2 * q], x[2 * q + 1], y[2 * q], y[2 * q + 1], bw[k][j][lm][0], bw[k][j][lm][1]);
          }
        }
#pragma unroll
        for (int j = 0; j < NT && !EXACT; ++j)
#pragma unroll
          for (int lm = 0; lm < LIMBS; ++lm)
            mma16816(ones[j], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, bw[k][j][lm][0], bw[k][j][lm][1]);
      }
      __syncwarp();
      stage = stage + 1 == ST ? 0 : stage + 1;
    }
    cp_async_wait<0>();

    // ---- the item's numerators and denominators, or this part's
    constexpr int PART = COLS * (HD + 2);  // numerators [col][HD], then (M, denominator) [col]
    const bool ends = !whole && to == vt, alone = ends && from == 0;
    float *mine = nullptr;
    if (!alone) {
      // The last item's part takes this warp's ring where it fits, which it no
      // longer needs; an item that ends here and is followed by others goes
      // to the workspace.
      if (ends) mine = a.part + ((int64_t)blockIdx.x * PARTS + warp) * PART;
      else if (ON_SHARED) mine = reinterpret_cast<float *>(ring);
      else mine = a.part + ((int64_t)blockIdx.x * PARTS + ATT_WARPS + 2 + warp) * PART;
      if (lane == 0) {
        const Cut cut = {qbase + item, row0, head, ncol, begin, vt};
        if (ends) cut_end[warp] = cut, has_end[warp] = 1;
        else cut_on[warp] = cut, on_kind[warp] = whole ? (warp == 0 ? 1 : 2) : (from == 0 ? 1 : 2);
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l[j].x += __shfl_xor_sync(0xffffffffu, l[j].x, d), l[j].y += __shfl_xor_sync(0xffffffffu, l[j].y, d);
        z[j].x += __shfl_xor_sync(0xffffffffu, z[j].x, d), z[j].y += __shfl_xor_sync(0xffffffffu, z[j].y, d);
      }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = 8 * j + 2 * t + c;
        if (col >= ncol) continue;
        const float den = c ? l[j].y : l[j].x, zs = c ? z[j].y : z[j].x;
        const float add = EXACT ? zs : fmaf(-7.5f, ones[j][c], zs);
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          const float4 x = make_float4(fmaf(o[j][k][c], EVEN, add), fmaf(o[j][k][c + 2], ODD, add),
                                       fmaf(o[j][k + 1][c], EVEN, add), fmaf(o[j][k + 1][c + 2], ODD, add));
          const int d = 16 * k + 4 * g;
          if (alone) emit(a, row0, head, col, d, x, den);
          else *reinterpret_cast<float4 *>(mine + col * HD + d) = x;
        }
        if (!alone && g == 0) *reinterpret_cast<float2 *>(mine + COLS * HD + 2 * col) = make_float2(c ? M[j].y : M[j].x, den);
      }
    __syncwarp();
  }

  // ---- parts meet within the block.  A run is an item's parts in it: it
  // begins with the part of warp w that goes on (or, in warp 0, that began
  // before) and takes the following warps up to the one that the item ends in.
  constexpr int PART = COLS * (HD + 2);
  float *block_part = a.part + (int64_t)blockIdx.x * PARTS * PART;
  if (tid < 2) edge_last[tid] = 0;
  __syncthreads();
  auto on_part = [&](int w) {
    return ON_SHARED ? reinterpret_cast<float *>(smem + w * ST * RP * REC) : block_part + (ATT_WARPS + 2 + w) * PART;
  };
  if (tid <= ATT_WARPS) {
    const int w = tid < ATT_WARPS ? tid : 0;
    const bool before = tid == ATT_WARPS;
    Run mine = {0, -1, -1};
    if (before ? has_end[0] : false) {
      mine = {0, 0, 0};
    } else if (on_kind[w] == (before ? 2 : 1)) {
      int x = w + 1;  // the warp after the last part that goes on
      while (x < ATT_WARPS && on_kind[x] == 2) ++x;
      const bool ended = x < ATT_WARPS && has_end[x];
      mine = {x - w, ended ? x : -1, before ? 0 : ended || whole ? 2 : 1};
    }
    run[tid] = mine;
    if (mine.side == 0 || mine.side == 1) edge[mine.side] = mine.on ? cut_on[w] : cut_end[0], edge_last[mine.side] = 1;
  }
  __syncthreads();
  for (int i = 0; i <= ATT_WARPS; ++i) {
    const Run now = run[i];
    if (now.side < 0) continue;
    const int w = i < ATT_WARPS ? i : 0;
    const Cut &cut = now.on ? cut_on[w] : cut_end[0];
    for (int q = tid; q < cut.ncol * (HD / 4); q += ATT_THREADS) {
      const int col = q / (HD / 4), d = (q % (HD / 4)) * 4;
      const Joined y = join_parts(on_part(w), ON_SHARED ? ST * RP * REC / 4 : PART, now.on,
                                  now.end >= 0 ? block_part + now.end * PART : nullptr, col * HD + d, COLS * HD + 2 * col);
      if (now.side == 2) {
        emit(a, cut.row0, cut.head, col, d, y.x, y.den);
      } else {
        float *p = block_part + (ATT_WARPS + now.side) * PART;
        *reinterpret_cast<float4 *>(p + col * HD + d) = y.x;
        if (d == 0) *reinterpret_cast<float2 *>(p + COLS * HD + 2 * col) = make_float2(y.m, y.den);
      }
    }
  }
  __syncthreads();

  // ---- parts of several blocks: the last one to arrive joins them
  if (edge_last[0] | edge_last[1]) {
    auto blocks_of = [&](const Cut &cut, int &first) {  // that share an item
      first = (int)((uint32_t)cut.begin / (uint32_t)each) / ATT_WARPS;
      return (int)((uint32_t)(cut.begin + cut.size - 1) / (uint32_t)each) / ATT_WARPS - first + 1;
    };
    if (tid < 2 && edge_last[tid]) {
      int first;
      const int parts = blocks_of(edge[tid], first);
      // One thread's fence covers the block's writes: the barrier orders them before it.
      asm volatile("fence.acq_rel.gpu;" ::: "memory");
      if (atomicAdd(a.counter + edge[tid].item, 1u) == (uint32_t)parts - 1) {
        a.counter[edge[tid].item] = 0;  // ready for the next call
        edge_last[tid] = 2;
      }
      asm volatile("fence.acq_rel.gpu;" ::: "memory");
    }
    __syncthreads();
    for (int side = 0; side < 2; ++side) {
      if (edge_last[side] != 2) continue;
      const Cut cut = edge[side];
      int first;
      const int parts = blocks_of(cut, first);
      // Part 0 stands second in its block, as one that goes on; the others stand first.
      const float *p0 = a.part + ((int64_t)first * PARTS + ATT_WARPS) * PART;
      // Threads left over by the columns take a stretch of the other parts each.
      const int quads = cut.ncol * (HD / 4), teams = max(1, min(ATT_THREADS / quads, (parts + 2) / 4));
      const int stretch = (parts - 1 + teams - 1) / teams;
      float *team_part = reinterpret_cast<float *>(smem);  // [team][quad][6]: elements, then (M, denominator)
      for (int i = tid; i < quads * teams; i += ATT_THREADS) {
        const int quad = i % quads, team = i / quads, col = quad / (HD / 4), d = (quad % (HD / 4)) * 4;
        const int k0 = 1 + team * stretch, n = max(0, min(stretch, parts - k0));
        const Joined y = join_parts(p0 + (int64_t)k0 * PARTS * PART, PARTS * PART, n, team == 0 ? p0 + PART : nullptr,
                                    col * HD + d, COLS * HD + 2 * col);
        if (teams > 1) {
          *reinterpret_cast<float4 *>(team_part + i * 8) = y.x;
          *reinterpret_cast<float2 *>(team_part + i * 8 + 4) = make_float2(y.m, y.den);
        } else {
          emit(a, cut.row0, cut.head, col, d, y.x, y.den);
        }
      }
      if (teams > 1) {  // then quads < ATT_THREADS
        __syncthreads();
        if (tid < quads) {
          const Joined y = join_parts(team_part, quads * 8, teams, nullptr, tid * 8, tid * 8 + 4);
          emit(a, cut.row0, cut.head, tid / (HD / 4), (tid % (HD / 4)) * 4, y.x, y.den);
        }
        __syncthreads();
      }
    }
  }
  if (!whole) break;
  __syncthreads();  // the rings and the shared words are free again
  }

  // Rows past the last request are zero.
  const int used = max(0, min(__ldg(a.row_start + a.requests), a.rows));
  const int64_t chunks = (int64_t)a.kv_heads * a.group * (HD / 4);
  for (int64_t i = (int64_t)blockIdx.x * ATT_THREADS + tid; i < (a.rows - used) * chunks; i += (int64_t)gridDim.x * ATT_THREADS) {
    const int64_t row = used + i / chunks;
    const int rest = (int)(i % chunks);
    store4(a.out, a.dtype, row * a.o_row + rest / (HD / 4) * a.o_head + rest % (HD / 4) * 4, a.o_wide, make_float4(0, 0, 0, 0));
  }
}

#include "cis2b_kv4_prompt.cuh"

struct Shape {
  bool prompt;  // more than 32 query columns: k_kv4_prompt
  int nt, limbs, qt, cols, blocks;
  uint64_t items, bytes;
  uint64_t slots;  // parts of k_kv4_prompt
};

constexpr int PR_BLOCKS = 320;  // of k_kv4_prompt at most: two for each of 148 SMs, and some to spare

// The workspace begins with every word that has to be zero between calls, at
// places that do not depend on a call's sizes: k_kv4_prompt's tickets and
// counters, then k_kv4_attention's counters.  Parts follow; nothing reads a
// part that its own call has not written.
constexpr uint64_t WORK_PROMPT = 4096, WORK_ITEMS = 65536, WORK_PARTS = WORK_PROMPT + 4 * WORK_ITEMS;
static_assert(WORK_PARTS == CIS2B_KV4_WORK_ZERO, "as include/cis2b.h says");
static_assert(8 + 4 * 2 * PR_BLOCKS <= WORK_PROMPT, "tickets and counters of k_kv4_prompt");

// Query columns per item: the fewest groups of 8 that hold one request's rows,
// up to 32.
constexpr uint64_t ITEMS_MOST = 1u << 30;  // a block's next item, its number plus the grid's, stays in 32 bits
Shape shape_of(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a) {
  Shape s;
  const int group = a->heads / c->kv_heads;
  const int64_t cols = (int64_t)group * a->max_new;
  s.nt = cols <= 8 ? 1 : cols <= 16 ? 2 : 4;
  s.limbs = a->dtype == CIS2B_F32 ? 2 : 1;
  s.prompt = cols > 32;
  s.slots = 0;
  if (s.prompt) {
    s.cols = PR_ROWS;
    s.qt = PR_ROWS / group;
    s.blocks = PR_BLOCKS;
    s.items = ((uint64_t)a->requests + (uint64_t)a->rows / s.qt) * c->kv_heads;  // at most
    // Query tiles of more than 1.25 PR_LEAST key tiles may be cut.
    if ((uint64_t)a->width * c->page_size > PR_KEYS * (PR_LEAST + PR_LEAST / 4)) s.slots = 2 * PR_BLOCKS;
    s.bytes = WORK_PARTS + s.slots * PR_ROWS * (c->head_dim + 2) * 4;
    return s;
  }
  s.cols = 8 * s.nt;
  s.qt = s.cols / group;
  s.blocks = s.nt == 1 ? 320 : 160;  // at most: two or one for each of 148 SMs, and some to spare
  s.items = ((uint64_t)a->requests + (uint64_t)a->rows / s.qt) * c->kv_heads;  // at most
  s.bytes = WORK_PARTS + (uint64_t)s.blocks * att_parts(c->head_dim, s.nt) * s.cols * (c->head_dim + 2) * 4;
  return s;
}

int check_attn(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a) {
  if (!a) return kv4_fail(CIS2B_ERR_ARG, "attention: arguments are NULL");
  if (a->flags & ~CIS2B_KV4_WHOLE) return kv4_fail(CIS2B_ERR_ARG, "attention: unknown flags");
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
  if (shape_of(c, a).items > ITEMS_MOST)
    return kv4_fail(CIS2B_ERR_ARG, "attention: (requests + rows) * kv_heads must be at most 2^30");
  return CIS2B_OK;
}

template <int HD, int NT, int LIMBS, bool EXACT>
int launch(const AttArgs &args, const cis2b_kv4_cache *c, uint64_t most, int sms, cudaStream_t stream) {
  static std::atomic<int> resident[64];  // blocks per SM, by device; also: the attribute is set
  const int smem = att_smem_bytes(HD, NT, LIMBS);
  int n = resident[c->device].load(std::memory_order_relaxed);
  if (!n) {
    if (int rc = kv4_cuda(cudaFuncSetAttribute(k_kv4_attention<HD, NT, LIMBS, EXACT>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem)))
      return rc;
    if (int rc = kv4_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_kv4_attention<HD, NT, LIMBS, EXACT>,
                                                                        ATT_THREADS, smem)))
      return rc;
    n = std::max(n, 1);
    resident[c->device].store(n, std::memory_order_relaxed);
  }
  const int grid = (int)std::max<uint64_t>(1, std::min<uint64_t>(most, (uint64_t)sms * n));
  AttArgs given = args;
  given.per_warp = nextafterf(1.0f / (float)(grid * ATT_WARPS), 1.0f);
  k_kv4_attention<HD, NT, LIMBS, EXACT><<<grid, ATT_THREADS, smem, stream>>>(given);
  return kv4_cuda(cudaGetLastError());
}

template <int HD>
int dispatch(const Shape &s, const AttArgs &args, const cis2b_kv4_cache *c, uint64_t most, int sms, cudaStream_t st) {
  const bool one = s.limbs == 1, bf16 = args.dtype == KV4_BF16;
  switch (s.nt) {
    case 1:
      return !one ? launch<HD, 1, 2, true>(args, c, most, sms, st)
                  : bf16 ? launch<HD, 1, 1, false>(args, c, most, sms, st) : launch<HD, 1, 1, true>(args, c, most, sms, st);
    case 2:
      return !one ? launch<HD, 2, 2, true>(args, c, most, sms, st)
                  : bf16 ? launch<HD, 2, 1, false>(args, c, most, sms, st) : launch<HD, 2, 1, true>(args, c, most, sms, st);
    default:
      return !one ? launch<HD, 4, 2, true>(args, c, most, sms, st)
                  : bf16 ? launch<HD, 4, 1, false>(args, c, most, sms, st) : launch<HD, 4, 1, true>(args, c, most, sms, st);
  }
}

// What both kernels are given.
void fill(AttArgs &k, const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, const Shape &s) {
  const int64_t unit = a->dtype == CIS2B_F32 ? 4 : 8;
  k.q = a->q, k.out = a->out;
  k.q_row = a->q_row_stride, k.q_head = a->q_head_stride, k.o_row = a->out_row_stride, k.o_head = a->out_head_stride;
  k.q_wide = !(reinterpret_cast<uintptr_t>(a->q) & 15) && !(k.q_row % unit | k.q_head % unit);
  k.o_wide = !(reinterpret_cast<uintptr_t>(a->out) & 15) && !(k.o_row % unit | k.o_head % unit);
  k.pool = static_cast<const uint8_t *>(c->pool), k.status = c->status;
  k.table = a->table, k.length = a->length, k.row_start = a->row_start;
  k.dtype = a->dtype, k.requests = a->requests, k.rows = a->rows, k.width = a->width, k.kv_heads = c->kv_heads;
  k.group = a->heads / c->kv_heads, k.pages = c->pages, k.window = a->window, k.sinks = a->sinks;
  k.shift = __builtin_ctz(c->page_size);
  k.qt = s.qt;
  k.items = (int)s.items;
  k.scale = a->scale;
}

template <int HD, int LIMBS>
int launch_prompt(const PromptArgs &args, const cis2b_kv4_cache *c, uint64_t most, int sms, cudaStream_t stream) {
  static std::atomic<bool> ready[64];  // by device: the attribute is set
  const int smem = pr_smem_bytes(HD, LIMBS);
  if (!ready[c->device].load(std::memory_order_relaxed)) {
    if (int rc = kv4_cuda(cudaFuncSetAttribute(k_kv4_prompt<HD, LIMBS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)))
      return rc;
    ready[c->device].store(true, std::memory_order_relaxed);
  }
  const int per_sm = HD == 128 && LIMBS == 2 ? 1 : 2;  // as its launch bounds and shared memory allow
  const int grid = (int)std::max<uint64_t>(1, std::min<uint64_t>(most, std::min(sms * per_sm, PR_BLOCKS)));
  k_kv4_prompt<HD, LIMBS><<<grid, PR_THREADS, smem, stream>>>(args);
  return kv4_cuda(cudaGetLastError());
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
  AttArgs k{};
  if (s.prompt) {
    PromptArgs p{};
    fill(k, c, a, s);
    k.whole = (a->flags & CIS2B_KV4_WHOLE) || !s.slots;
    p.a = k;
    p.ticket = static_cast<uint32_t *>(a->work);
    p.counter = p.ticket + 2;
    p.part = reinterpret_cast<float *>(static_cast<uint8_t *>(a->work) + WORK_PARTS);
    const uint64_t tiles = ((uint64_t)a->width * c->page_size + PR_KEYS - 1) / PR_KEYS;
    const uint64_t most = s.items * ((tiles + PR_LEAST - 1) / PR_LEAST);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->dtype == CIS2B_F32)
      return c->head_dim == 64 ? launch_prompt<64, 2>(p, c, most, sms, st) : launch_prompt<128, 2>(p, c, most, sms, st);
    return c->head_dim == 64 ? launch_prompt<64, 1>(p, c, most, sms, st) : launch_prompt<128, 1>(p, c, most, sms, st);
  }
  k.counter = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(a->work) + WORK_PROMPT);
  k.part = reinterpret_cast<float *>(static_cast<uint8_t *>(a->work) + WORK_PARTS);
  fill(k, c, a, s);
  const uint64_t recs = (uint64_t)a->width * c->page_size / 16 + 1;  // as tiles_bound()
  // The row of records is counted in 32 bits, and an item that is cut has a
  // counter; a batch that could pass that has items enough to take them whole.
  k.whole = (a->flags & CIS2B_KV4_WHOLE) || s.items > WORK_ITEMS || s.items * (recs + ATT_SETUP) > INT_MAX;
  const uint64_t most = std::max(s.items, (s.items * ((recs + ATT_LEAST - 1) / ATT_LEAST) + ATT_WARPS - 1) / ATT_WARPS);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return c->head_dim == 64 ? dispatch<64>(s, k, c, std::min<uint64_t>(most, s.blocks), sms, st)
                           : dispatch<128>(s, k, c, std::min<uint64_t>(most, s.blocks), sms, st);
}
