// cis2b_kv4.cu -- step planning, append and read-back of the 4-bit key/value
// cache (include/cis2b.h).  Attention over it is in
// cis2b_kv4_attn.cuh, drafted trees in cis2b_kv4_tree.cu.
#include "../../include/cis2b.h"
#include "cis2b_kv4.h"
#include "cis2b_kv4.cuh"

#include <limits.h>

#include <algorithm>
#include <type_traits>

namespace cis2b {

// An entry point's error path must not let an exception out (the message is
// a std::string).
int kv4_fail(int code, const char *msg) noexcept {
  try {
    set_last_error(code, msg);
  } catch (...) {
  }
  return code;
}

int kv4_cuda(cudaError_t e) noexcept {
  return e == cudaSuccess ? CIS2B_OK : kv4_fail(CIS2B_ERR_CUDA, cudaGetErrorString(e));
}

int kv4_page_shift(int page_size) noexcept {
  for (int s = 4; s <= 8; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}

int kv4_check_cache(const cis2b_kv4_cache *c, bool pool) noexcept {
  if (!c) return kv4_fail(CIS2B_ERR_ARG, "cache is NULL");
  if (c->reserved) return kv4_fail(CIS2B_ERR_ARG, "cache: reserved must be zero");
  if (c->head_dim != 64 && c->head_dim != 128) return kv4_fail(CIS2B_ERR_ARG, "cache: head_dim must be 64 or 128");
  if (kv4_page_shift(c->page_size) < 0)
    return kv4_fail(CIS2B_ERR_ARG, "cache: page_size must be 16, 32, 64, 128 or 256");
  if (c->kv_heads < 1 || c->kv_heads > 65535) return kv4_fail(CIS2B_ERR_ARG, "cache: kv_heads must be in 1..65535");
  if (c->pages < 1 || (int64_t)c->pages * c->page_size > INT_MAX)
    return kv4_fail(CIS2B_ERR_ARG, "cache: pages must be >= 1 and pages * page_size < 2^31");
  if (pool && (!c->pool || (reinterpret_cast<uintptr_t>(c->pool) & 15)))
    return kv4_fail(CIS2B_ERR_ARG, "cache: pool must be a 16-byte aligned device pointer");
  return CIS2B_OK;
}

int kv4_sm_count(int device, int *sms) noexcept {
  static std::atomic<int> known[64];
  if (device < 0 || device >= 64) return kv4_fail(CIS2B_ERR_ARG, "device ordinal out of range");
  int n = known[device].load(std::memory_order_relaxed);
  if (!n) {
    const cudaError_t e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return kv4_cuda(e);
    known[device].store(n, std::memory_order_relaxed);
  }
  *sms = n;
  return CIS2B_OK;
}

// ---------------------------------------------------------------- plan

constexpr int PLAN_THREADS = 512;
constexpr int PLAN_MAX_REQUESTS = 16384;

struct PlanArgs {
  int requests, rows, width, shift, free_count;
  const int32_t *cached, *fresh, *free_pages;
  int32_t *table, *length, *row_start, *slot, *position, *request, *counts;
};

// Lengths to block tables and slot maps in ONE launch.  Two prefix sums over
// the requests (rows and pages taken) give everything else: every block runs
// both over all requests into its shared memory (8 bytes a request, read from
// L2) and then fills its own part of the rows, finding a row's request by
// binary search.  A row that opens a page enters it in the table, so the
// table needs no pass of its own.  The work is a few hundred kilobytes at
// most: latency bounds it, and a second launch or a grid barrier would cost
// more than the repeated sums.
__global__ __launch_bounds__(PLAN_THREADS, 1) void k_kv4_plan(PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t *row0 = plan_smem;                  // [requests + 1] exclusive sums of new tokens, capped
  int32_t *page0 = plan_smem + a.requests + 1;  // [requests + 1] exclusive sums of pages taken, capped
  __shared__ int64_t warp_rows[PLAN_THREADS / 32], warp_pages[PLAN_THREADS / 32];
  __shared__ int bits;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int page = 1 << a.shift;
  if (tid == 0) bits = 0;
  __syncthreads();

  int64_t rows_before = 0, pages_before = 0;
  for (int base = 0; base < a.requests; base += PLAN_THREADS) {
    const int r = base + tid;
    int64_t n = 0, need = 0;
    if (r < a.requests) {
      int32_t c = __ldg(a.cached + r), f = __ldg(a.fresh + r);
      if (c < 0 || f < 0) atomicOr(&bits, CIS2B_KV4_PLAN_NEGATIVE);
      c = max(c, 0), f = max(f, 0);
      const int64_t len = (int64_t)c + f;
      n = f;
      need = ((len + page - 1) >> a.shift) - (((int64_t)c + page - 1) >> a.shift);
      if (f && len > ((int64_t)a.width << a.shift)) atomicOr(&bits, CIS2B_KV4_PLAN_WIDTH);
      if (blockIdx.x == 0) a.length[r] = (int32_t)min(len, (int64_t)INT_MAX);
    }
    int64_t sn = n, sp = need;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t un = __shfl_up_sync(0xffffffffu, sn, d), up = __shfl_up_sync(0xffffffffu, sp, d);
      if (lane >= d) sn += un, sp += up;
    }
    if (lane == 31) warp_rows[warp] = sn, warp_pages[warp] = sp;
    __syncthreads();
    int64_t before_n = rows_before, before_p = pages_before;
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 32; ++w) {
      const int64_t tn = warp_rows[w], tp = warp_pages[w];
      if (w < warp) before_n += tn, before_p += tp;
      rows_before += tn, pages_before += tp;
    }
    if (r < a.requests) {
      row0[r] = (int32_t)min(before_n + sn - n, (int64_t)INT_MAX);
      page0[r] = (int32_t)min(before_p + sp - need, (int64_t)INT_MAX);
    }
    __syncthreads();
  }
  const int total = (int)min(rows_before, (int64_t)INT_MAX);
  if (tid == 0) row0[a.requests] = total;
  __syncthreads();

  if (blockIdx.x == 0) {
    for (int r = tid; r <= a.requests; r += PLAN_THREADS) a.row_start[r] = row0[r];
    if (tid == 0) {
      int b = bits;
      if (pages_before > a.free_count) b |= CIS2B_KV4_PLAN_FREE;
      if (rows_before > a.rows) b |= CIS2B_KV4_PLAN_ROWS;
      a.counts[0] = min(total, a.rows);
      a.counts[1] = (int32_t)min(pages_before, (int64_t)INT_MAX);
      a.counts[2] = b;
      a.counts[3] = 0;
    }
  }

  const int step = gridDim.x * PLAN_THREADS;
  for (int64_t t64 = (int64_t)blockIdx.x * PLAN_THREADS + tid; t64 < a.rows; t64 += step) {
    const int t = (int)t64;
    int32_t slot = -1, pos = -1, req = -1;
    if (t < total) {
      int lo = 0, hi = a.requests;  // the last request whose first row is at or before t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (row0[mid] <= t) lo = mid; else hi = mid;
      }
      req = lo;
      const int c = max(__ldg(a.cached + req), 0);
      const int64_t p = (int64_t)c + (t - row0[req]);
      pos = (int32_t)min(p, (int64_t)INT_MAX);
      const int64_t col = p >> a.shift;
      const int64_t have = ((int64_t)c + page - 1) >> a.shift;
      if (col < a.width) {
        int32_t *entry = a.table + (int64_t)req * a.width + col;
        int32_t pg = -1;
        if (col < have) {
          pg = *entry;
        } else {
          const int64_t f = page0[req] + (col - have);
          if (f < a.free_count) pg = __ldg(a.free_pages + f);
          if ((p & (page - 1)) == 0) *entry = pg;
        }
        const int64_t s = ((int64_t)pg << a.shift) + (p & (page - 1));
        if (pg >= 0 && s <= INT_MAX) slot = (int32_t)s;
      }
    }
    a.slot[t] = slot;
    a.position[t] = pos;
    a.request[t] = req;
  }
}

// ---------------------------------------------------------------- append and gather

struct RowArgs {
  const uint8_t *pool;
  int32_t *status;
  const int32_t *slot;
  int rows, kv_heads, shift, slots;
  int64_t ks, kh, vs, vh;  // row and head strides of the caller's tensors, elements
};

constexpr int ROW_THREADS = 256;

// Minimum and maximum that are NaN where an operand is.
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Minimum and negated maximum of eight elements, as one pair of their own type
// (fp32: of fp32), NaN where an element is.
struct Range32 {
  float lo, neg_hi;
  __device__ void join(int d) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, d)), neg_hi = min_nan(neg_hi, __shfl_xor_sync(0xffffffffu, neg_hi, d));
  }
  __device__ float2 get() const { return make_float2(lo, -neg_hi); }
};
template <class T2> struct Range16 {
  T2 both;
  __device__ void join(int d) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<const uint32_t *>(&both), d);
    both = __hmin2_nan(both, *reinterpret_cast<const T2 *>(&other));
  }
  __device__ float2 get() const { return make_float2(__low2float(both), -__high2float(both)); }
};
__device__ __forceinline__ Range32 range_of(const float (&x)[8]) {
  Range32 r = {x[0], x[0]};
#pragma unroll
  for (int i = 1; i < 8; ++i) r.lo = min_nan(r.lo, x[i]), r.neg_hi = max_nan(r.neg_hi, x[i]);
  r.neg_hi = -r.neg_hi;
  return r;
}
template <class T2> __device__ __forceinline__ Range16<T2> range_of(const uint32_t (&w)[4]) {
  T2 lo = *reinterpret_cast<const T2 *>(&w[0]), hi = lo;
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    const T2 x = *reinterpret_cast<const T2 *>(&w[i]);
    lo = __hmin2_nan(lo, x), hi = __hmax2_nan(hi, x);
  }
  hi = __hneg2(hi);
  // (lo.x, -hi.x) and (lo.y, -hi.y)
  const uint32_t l = *reinterpret_cast<const uint32_t *>(&lo), h = *reinterpret_cast<const uint32_t *>(&hi);
  const uint32_t a = __byte_perm(l, h, 0x5410), b = __byte_perm(l, h, 0x7632);
  return {__hmin2_nan(*reinterpret_cast<const T2 *>(&a), *reinterpret_cast<const T2 *>(&b))};
}

// A group's step (low 16 bits) and base (high) as bfloat16, and the factor of
// its elements; NaN in both for a group with a NaN, an infinity, or too wide.
__device__ __forceinline__ uint32_t kv4_params(float lo, float hi, float &inv) {
  const uint32_t base16 = bf16_down(lo);
  const float base = __uint_as_float(base16 << 16);
  const float q = __fdiv_rn(__fsub_rn(hi, base), 15.0f);
  const bool fine = q <= 3.3e38f && fabsf(base) <= 3.3e38f;  // bfloat16's largest is 3.39e38
  uint32_t step16 = bf16_up(q);
  float step = __uint_as_float(step16 << 16);
  if (step < 0x1p-100f) step = 0.0f, step16 = 0;
  inv = step > 0.0f ? __frcp_rn(step) : 0.0f;
  return fine ? step16 | base16 << 16 : 0x7fc07fc0u;
}

// Eight codes.  The quotient is at most 15 (1 + 2^-21), since the step is
// rounded up, and at least 0, since the base is rounded down: no clamp.  Adding
// 1.5 * 2^23 rounds it to a whole number, ties to even, in the low bits of the
// sum, and eight sums times powers of 16 make the word, less the constant's own
// part.
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], uint32_t params, float inv) {
  const float base = bf16_hi(params);
  uint32_t word = 0;
#pragma unroll
  for (int i = 7; i >= 0; --i)
    word = word * 16 + __float_as_uint(__fadd_rn(__fmul_rn(__fsub_rn(x[i], base), inv), 12582912.0f));
  return base == base ? word - 0x4b400000u * 0x11111111u : 0u;
}

// Rows to codes: D / 8 lanes take one (row, head), eight key and eight value
// elements each, so one warp instruction reads whole 128-byte lines and a
// group's range is log2(D / 8) shuffles away.  Half of the lanes then find the
// key's parameters and half the value's.  Each element is read once and each
// code written once; instructions bound it: 18 per element, issued in 84 percent
// of the cycles (fp16, 40,009 rows of 8 x 128 in 54 us; its bytes need 32).
template <int HD, int DT>
__global__ __launch_bounds__(ROW_THREADS) void k_kv4_append(RowArgs a, const void *k, const void *v, bool wide) {
  constexpr int LANES = HD / 8;
  const uint32_t item = (uint32_t)blockIdx.x * (ROW_THREADS / LANES) + threadIdx.x / LANES;
  const int part = threadIdx.x & (LANES - 1);
  const int64_t row = item / (uint32_t)a.kv_heads;
  const int head = (int)(item - (uint32_t)row * a.kv_heads);
  int slot = -1;
  if (row < a.rows) slot = __ldg(a.slot + row);
  if (slot >= a.slots) {
    if (a.status && part == 0) atomicOr(a.status, CIS2B_KV4_BAD_SLOT);
    slot = -1;
  }
  const bool on = slot >= 0;
  float x[8], y[8];
  float2 xr, yr;
  if constexpr (DT == KV4_F32) {
    load_query<true, 8>(k, false, row * a.ks + head * a.kh + part * 8, wide, on, x);
    load_query<true, 8>(v, false, row * a.vs + head * a.vh + part * 8, wide, on, y);
    Range32 p = range_of(x), q = range_of(y);
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) p.join(d), q.join(d);
    xr = p.get(), yr = q.get();
  } else {
    using T2 = std::conditional_t<DT == KV4_F16, __half2, __nv_bfloat162>;
    uint32_t xw[4], yw[4];
    load_words(k, row * a.ks + head * a.kh + part * 8, wide, on, xw);
    load_words(v, row * a.vs + head * a.vh + part * 8, wide, on, yw);
    Range16<T2> p = range_of<T2>(xw), q = range_of<T2>(yw);
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) p.join(d), q.join(d);
    xr = p.get(), yr = q.get();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T2 u = *reinterpret_cast<const T2 *>(&xw[i]), w = *reinterpret_cast<const T2 *>(&yw[i]);
      x[2 * i] = __low2float(u), x[2 * i + 1] = __high2float(u), y[2 * i] = __low2float(w), y[2 * i + 1] = __high2float(w);
    }
  }
  const bool of_value = part >= LANES / 2;
  float inv;
  const uint32_t params = kv4_params(of_value ? yr.x : xr.x, of_value ? yr.y : xr.y, inv);
  const uint32_t other = __shfl_xor_sync(0xffffffffu, params, LANES / 2);
  const float other_inv = __shfl_xor_sync(0xffffffffu, inv, LANES / 2);
  if (!on) return;
  const uint32_t kp = of_value ? other : params, vp = of_value ? params : other;
  const uint32_t kc = kv4_codes(x, kp, of_value ? other_inv : inv), vc = kv4_codes(y, vp, of_value ? inv : other_inv);
  const int page = slot >> a.shift, off = slot & ((1 << a.shift) - 1), r = off & 15;
  uint8_t *rec = const_cast<uint8_t *>(a.pool) +
                 ((((int64_t)page * a.kv_heads + head) << (a.shift - 4)) + (off >> 4)) * kv4_rec_bytes(HD);
  reinterpret_cast<uint32_t *>(rec + r * (HD / 2))[part] = kc;
  reinterpret_cast<uint32_t *>(rec + (16 + r) * (HD / 2))[part] = vc;
  if (part == 0) *reinterpret_cast<uint2 *>(rec + 16 * HD + r * 8) = make_uint2(kp, vp);
}

// base + step * code: the product is exact (12 bits), so one rounding.  A code
// under the exponent of 2^23 is the number 2^23 + code.
__device__ __forceinline__ void kv4_values(uint32_t word, uint32_t params, float (&x)[8]) {
  const float step = bf16_lo(params), base = bf16_hi(params);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf(step, __uint_as_float(((word >> (4 * i)) & 15) | 0x4b000000u) - 8388608.0f, base);
}

// Codes to rows, the same split, two rows per lane: 12 instructions per element,
// issued in 74 percent of the cycles, and the wait for the slot and then for the
// codes bound it (fp16, 40,009 rows of 8 x 128 in 42 us; its bytes need 32).
template <int HD>
__global__ __launch_bounds__(ROW_THREADS) void k_kv4_gather(RowArgs a, void *k, void *v, int dt, bool wide) {
  constexpr int LANES = HD / 8, PER = ROW_THREADS / LANES;
  const uint32_t items = (uint32_t)a.rows * a.kv_heads;
  const int part = threadIdx.x & (LANES - 1);
  uint32_t item[2], kc[2], vc[2];
  uint2 p[2];
  int slot[2], head[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    item[i] = (uint32_t)blockIdx.x * (2 * PER) + i * PER + threadIdx.x / LANES;
    const uint32_t row = item[i] / (uint32_t)a.kv_heads;
    head[i] = (int)(item[i] - row * a.kv_heads);
    slot[i] = item[i] < items ? __ldg(a.slot + row) : -1;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (slot[i] >= a.slots) {
      if (a.status && part == 0) atomicOr(a.status, CIS2B_KV4_BAD_SLOT);
      slot[i] = -1;
    }
    kc[i] = vc[i] = 0, p[i] = make_uint2(0, 0);
    if (slot[i] < 0) continue;
    const int page = slot[i] >> a.shift, off = slot[i] & ((1 << a.shift) - 1), r = off & 15;
    const uint8_t *rec =
        a.pool + ((((int64_t)page * a.kv_heads + head[i]) << (a.shift - 4)) + (off >> 4)) * kv4_rec_bytes(HD);
    kc[i] = reinterpret_cast<const uint32_t *>(rec + r * (HD / 2))[part];
    vc[i] = reinterpret_cast<const uint32_t *>(rec + (16 + r) * (HD / 2))[part];
    p[i] = *reinterpret_cast<const uint2 *>(rec + 16 * HD + r * 8);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (item[i] >= items) continue;
    float x[8], y[8];  // step and base 0 where there is nothing
    kv4_values(kc[i], p[i].x, x);
    kv4_values(vc[i], p[i].y, y);
    const int64_t at = (int64_t)item[i] * HD + part * 8;
    store8(k, dt, at, wide, x);
    store8(v, dt, at, wide, y);
  }
}

template <int HD>
static cudaError_t append_launch(const RowArgs &a, int dtype, const void *k, const void *v, bool wide, int grid,
                                 cudaStream_t s) {
  if (dtype == CIS2B_F32) k_kv4_append<HD, KV4_F32><<<grid, ROW_THREADS, 0, s>>>(a, k, v, wide);
  else if (dtype == CIS2B_F16) k_kv4_append<HD, KV4_F16><<<grid, ROW_THREADS, 0, s>>>(a, k, v, wide);
  else k_kv4_append<HD, KV4_BF16><<<grid, ROW_THREADS, 0, s>>>(a, k, v, wide);
  return cudaGetLastError();
}

static int row_args(const cis2b_kv4_cache *c, int32_t dtype, const void *k, const void *v, const int32_t *slot,
                    int32_t rows, RowArgs *a, int *grid) {
  if (int rc = kv4_check_cache(c, true)) return rc;
  if (dtype < CIS2B_F32 || dtype > CIS2B_BF16)
    return kv4_fail(CIS2B_ERR_ARG, "dtype must be CIS2B_F32, CIS2B_F16 or CIS2B_BF16");
  if (rows < 0) return kv4_fail(CIS2B_ERR_ARG, "rows must be >= 0");
  if (rows && (!k || !v || !slot)) return kv4_fail(CIS2B_ERR_ARG, "k, v and slot must be device pointers");
  const int64_t blocks = ((int64_t)rows * c->kv_heads * (c->head_dim / 8) + ROW_THREADS - 1) / ROW_THREADS;
  if ((int64_t)rows * c->kv_heads > INT_MAX || blocks > INT_MAX)
    return kv4_fail(CIS2B_ERR_ARG, "rows * kv_heads must be < 2^31");
  *grid = (int)blocks;
  *a = RowArgs{static_cast<const uint8_t *>(c->pool), c->status, slot, rows, c->kv_heads, kv4_page_shift(c->page_size),
               c->pages * c->page_size, 0, 0, 0, 0};
  return CIS2B_OK;
}

}  // namespace cis2b

using namespace cis2b;

extern "C" int cis2b_kv4_bytes(const cis2b_kv4_cache *c, uint64_t *out_bytes) {
  if (int rc = kv4_check_cache(c, false)) return rc;
  if (!out_bytes) return kv4_fail(CIS2B_ERR_ARG, "out_bytes is NULL");
  *out_bytes = (uint64_t)c->pages * c->page_size * c->kv_heads * (c->head_dim + 8);
  return CIS2B_OK;
}

extern "C" int cis2b_kv4_plan(const cis2b_kv4_step *s, void *stream) {
  if (!s) return kv4_fail(CIS2B_ERR_ARG, "step is NULL");
  if (s->requests < 1 || s->requests > PLAN_MAX_REQUESTS)
    return kv4_fail(CIS2B_ERR_ARG, "step: requests must be in 1..16384");
  const int shift = kv4_page_shift(s->page_size);
  if (shift < 0) return kv4_fail(CIS2B_ERR_ARG, "step: page_size must be 16, 32, 64, 128 or 256");
  if (s->rows < 0 || s->width < 1 || s->free_count < 0)
    return kv4_fail(CIS2B_ERR_ARG, "step: rows and free_count must be >= 0 and width >= 1");
  if (!s->cached || !s->new_tokens || !s->table || !s->length || !s->row_start || !s->counts ||
      (s->free_count && !s->free_pages) || (s->rows && (!s->slot || !s->position || !s->request)))
    return kv4_fail(CIS2B_ERR_ARG, "step: a device pointer is NULL");
  int sms = 0;
  if (int rc = kv4_sm_count(s->device, &sms)) return rc;
  if (int rc = kv4_cuda(cudaSetDevice(s->device))) return rc;
  const PlanArgs a{s->requests, s->rows,      s->width,  shift,        s->free_count, s->cached,  s->new_tokens,
                   s->free_pages, s->table,   s->length, s->row_start, s->slot,       s->position, s->request, s->counts};
  const size_t smem = sizeof(int32_t) * 2 * ((size_t)s->requests + 1);
  // The limit is the kernel's, not the call's: set once, to the most that any
  // call needs, so that no thread lowers it under another.
  static std::atomic<bool> ready[64];  // by device
  if (smem > 47 * 1024 && !ready[s->device].load(std::memory_order_relaxed)) {
    const int most = (int)(sizeof(int32_t) * 2 * (PLAN_MAX_REQUESTS + 1));
    if (int rc = kv4_cuda(cudaFuncSetAttribute(k_kv4_plan, cudaFuncAttributeMaxDynamicSharedMemorySize, most))) return rc;
    ready[s->device].store(true, std::memory_order_relaxed);
  }
  const int grid = std::max(1, std::min(sms, (s->rows + PLAN_THREADS - 1) / PLAN_THREADS));
  k_kv4_plan<<<grid, PLAN_THREADS, smem, static_cast<cudaStream_t>(stream)>>>(a);
  return kv4_cuda(cudaGetLastError());
}

extern "C" int cis2b_kv4_append(const cis2b_kv4_cache *c, int32_t dtype, const void *k, const void *v,
                                int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride,
                                int64_t v_head_stride, const int32_t *slot, int32_t rows, void *stream) {
  RowArgs a;
  int grid = 0;
  if (int rc = row_args(c, dtype, k, v, slot, rows, &a, &grid)) return rc;
  if (int rc = kv4_cuda(cudaSetDevice(c->device))) return rc;
  if (!grid) return CIS2B_OK;
  a.ks = k_row_stride, a.kh = k_head_stride, a.vs = v_row_stride, a.vh = v_head_stride;
  // 16-byte loads where every row and head starts on such a boundary.
  const int64_t unit = dtype == CIS2B_F32 ? 4 : 8;
  const bool wide = !((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) &&
                    !(a.ks % unit | a.kh % unit | a.vs % unit | a.vh % unit);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return kv4_cuda(c->head_dim == 64 ? append_launch<64>(a, dtype, k, v, wide, grid, s)
                                    : append_launch<128>(a, dtype, k, v, wide, grid, s));
}

extern "C" int cis2b_kv4_gather(const cis2b_kv4_cache *c, int32_t dtype, void *k, void *v, const int32_t *slot,
                                int32_t rows, void *stream) {
  RowArgs a;
  int grid = 0;
  if (int rc = row_args(c, dtype, k, v, slot, rows, &a, &grid)) return rc;
  if (int rc = kv4_cuda(cudaSetDevice(c->device))) return rc;
  if (!grid) return CIS2B_OK;
  const bool wide = !((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  grid = (grid + 1) / 2;  // two rows per lane
  if (c->head_dim == 64) k_kv4_gather<64><<<grid, ROW_THREADS, 0, s>>>(a, k, v, dtype, wide);
  else k_kv4_gather<128><<<grid, ROW_THREADS, 0, s>>>(a, k, v, dtype, wide);
  return kv4_cuda(cudaGetLastError());
}
