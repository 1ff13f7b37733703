// cis2b_kv4_prompt.cuh -- attention of many new rows per request over the
// 4-bit cache, on the fifth-generation tensor cores.  Included by
// cis2b_kv4_attn.cu, whose argument and span types it shares.
//
// A unit is 128 query rows (tokens x the group of one KV head) of one request
// against a stretch of its keys.  Per tile of 128 keys:
//   four warps turn codes into half-precision operands in shared memory
//     (16 (c - 7.5), exact), keys as [key][element], values as [element][key];
//   one thread issues S = Q K^T into TMEM (128 x 128 fp32);
//   four warps, one query row per thread, turn S into weights: score =
//     S * ks_j + kz_j sum(q), p = 2^(score - M), w = p vs_j rounded to half
//     precision and put back over S in TMEM; p and p vz_j are summed in fp32;
//   the same thread issues O += W V^T (128 x head_dim fp32 in TMEM).
// The two blocks of an SM fill each other's waits.  Per tile of head_dim 128
// the tensor cores need 1,024 cycles, the exponentials 1,024 and the warps'
// 9,400 instructions 2,350; measured (bf16, 100 GFLOP in 250 us) are 5,200, all
// included.  The row warps' registers leave no room to load ahead, and the
// products cannot overlap their work, since the weights take the scores' place
// in TMEM.  fp32 rows of head_dim 64 need 13,000 instructions a tile (8 x 1,024
// rows in 93 us).
// Measured slower: the products issued by a code warp (it stalls while they
// are queued) or by a ninth warp (96 registers), a pass of its own for the
// row's top, polling without suspension.
//
// M is an integer (a power of two scales exactly) and moves only when a weight
// passes 2^14, p 2^100 or p |vz_j| 2^94 (whose sum stays in fp32); then the row's
// weights already written, its sums and its O are scaled.  Whether one might is
// asked per 32 keys, by the row's top score and the largest step or base, of
// tokens that it does not see too; whether and how far M moves goes by the
// weights of the keys that it sees.
// LIMBS = 2 (fp32 rows): two half-precision limbs of the query and of the
// weights, twice the products.
// The tensor cores cut off what falls below their sums, so the small limbs have
// an O of their own, and are the first in S: that halves the cuts at full size
// (measured 1.5e-6 of the results without it).
//
// Each key's four parameters cost the row warps two 16-byte broadcasts from
// shared memory per pair of keys, 2,048 cycles a tile.  bf16 rows could do
// without where keys and values are rounded to half precision as operands
// (measured 15 percent faster), but then a chunk of 32 keys shares one exponent:
// a token of large values takes its neighbours' bits, and a row's result would
// depend on tokens that it does not see.
#pragma once

constexpr int PR_ROWS = 128, PR_KEYS = 128, PR_RECS = PR_KEYS / KV4_REC;
constexpr int PR_THREADS = 256;      // warps 0-3 rows, 4-7 codes; warp 0 also issues the products
constexpr int PR_MAX_SORT = 512;     // query tiles whose order is chosen (longest first)
constexpr int PR_LEAST = 16;         // least key tiles of a part
constexpr int PR_WAIT = 1 << 18;     // polls of a barrier, of about 4 us each, before the kernel gives up

struct PromptArgs {
  AttArgs a;
  float *part;        // [units that are parts][128 rows][HD], then (M, l) [128]
  uint32_t *counter;  // [query tiles that may be cut][kv_heads]
  uint32_t *ticket;   // next unit; blocks that are done
};

__host__ __device__ constexpr int pr_smem_bytes(int hd, int limbs) {
  return limbs * PR_ROWS * hd * 2 + 2 * PR_KEYS * hd * 2 + 2 * PR_KEYS * 16 + 1024;
}

__device__ __forceinline__ uint32_t smem_of(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(b) : "memory");
}
__device__ __forceinline__ bool bar_poll(uint32_t b, uint32_t parity) {
  uint32_t ok;
  asm volatile("{.reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.b32 %0, 1, 0, p;}"
               : "=r"(ok) : "r"(b), "r"(parity) : "memory");
  return ok;
}
// Waits for the phase of that parity to complete; gives up after PR_WAIT
// polls, or when another thread has.  A warp waits and gives up as one; every
// lane has seen the phase by its own poll, which is what orders its reads.
__device__ __forceinline__ bool bar_wait(uint32_t b, uint32_t parity, volatile int *dead) {
  for (int i = 0; i < PR_WAIT; ++i) {
    const bool ok = bar_poll(b, parity), stop = (i & 63) == 63 && *dead;
    if (__all_sync(0xffffffffu, ok)) return true;
    if (__any_sync(0xffffffffu, stop)) return false;
  }
  *dead = 1;
  return false;
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// The same for one load, whose registers it passes on: other loads may move across it.
__device__ __forceinline__ void tc_wait_ld32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]));
  asm volatile("" : "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_ld32(uint32_t (&r)[32], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}
__device__ __forceinline__ void tc_ld16(uint32_t (&r)[16], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
__device__ __forceinline__ void tc_st16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tc_ld8(uint32_t (&r)[8], uint32_t at) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(at));
}
__device__ __forceinline__ void tc_st8(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// Shared-memory operand with rows of 128 bytes in the 128-byte swizzle (16-byte
// piece p of row r at p ^ (r & 7)), groups of 8 rows 1,024 bytes apart.
__device__ __forceinline__ uint64_t tc_desc(uint32_t at) {
  return (uint64_t)((at >> 4) & 0x3fff) | 1ull << 16 | 64ull << 32 | 1ull << 46 | 2ull << 61;
}
// fp32 accumulators, half-precision operands, both with K contiguous.
__host__ __device__ constexpr uint32_t tc_idesc(int m, int n) {
  return 1u << 4 | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile("{.reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;}" ::"r"(d),
               "l"(a), "l"(b), "r"(idesc), "r"((int)add) : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile("{.reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;}" ::"r"(d),
               "r"(a), "l"(b), "r"(idesc), "r"((int)add) : "memory");
}

template <int HD, int LIMBS>
__global__ __launch_bounds__(PR_THREADS, HD == 128 && LIMBS == 2 ? 1 : 2) void k_kv4_prompt(PromptArgs pa) {
  const AttArgs &a = pa.a;
  constexpr int REC = kv4_rec_bytes(HD);
  constexpr int TMEM = 128 + LIMBS * HD <= 256 ? 256 : 512;  // columns: S, O of each limb
  constexpr int KB = HD / 64;                  // 64-element column blocks of Q and K
  constexpr uint32_t QB = PR_ROWS * 128, VB = HD * 128;  // bytes of a block of Q or K; of V
  extern __shared__ uint8_t pr_smem[];
  __shared__ __align__(8) uint64_t bars[7];
  __shared__ int scan_q[256], req_len[256], req_row[256], req_n[256];
  __shared__ int64_t warp_sum[8];
  __shared__ unsigned long long tile_sum;
  __shared__ uint16_t order[PR_MAX_SORT], tiles_of[PR_MAX_SORT];
  __shared__ int part0[PR_MAX_SORT + 1];       // parts before each query tile, in order
  __shared__ uint32_t tmem_base;
  __shared__ int next_unit, dead, last;
  __shared__ uint32_t held[2][PR_RECS];        // records of each tile that the pool holds
  __shared__ float value_part[2][4];           // log2 of the largest value size (size_of()) of each 32 keys
  __shared__ float4 value_log[2][PR_KEYS / 4];  // log2 of each key's
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint8_t *base = pr_smem + ((1024 - (smem_of(pr_smem) & 1023)) & 1023);
  uint8_t *sq = base, *sk = sq + LIMBS * KB * QB, *sv = sk + KB * QB;
  float4 *sp = reinterpret_cast<float4 *>(sv + 2 * VB);  // [2][64 key pairs][2]: (ks, ks, kz, kz), (vs, vs, vz, vz)
  const uint32_t b_v = smem_of(&bars[1]), b_s = smem_of(&bars[2]), b_p = smem_of(&bars[3]),
                 b_o = smem_of(&bars[4]), b_end = smem_of(&bars[6]);
  // Keys and parameters have a barrier for each parity of the tile: the code
  // warps may be through with the next tile's before a row warp has seen this
  // one's.  They are not through with those of the tile after: that waits for
  // the next tile's scores, which wait for every row warp's weights of this one.
  auto b_k = [&](uint32_t now) { return smem_of(&bars[now & 1 ? 5 : 0]); };
  if (tid == 0) {
    bar_init(b_k(0), 128), bar_init(b_k(1), 128), bar_init(b_v, 128), bar_init(b_s, 1), bar_init(b_p, 128), bar_init(b_o, 1), bar_init(b_end, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    dead = 0;
  }
  if (warp == 7) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_of(&tmem_base)), "n"(TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }

  // ---- query tiles before each request; what the units are
  const int per = (a.requests + 255) / 256;
  int all_q;
  {
    int64_t sum = 0, all = 0;
    {
      for (int r = tid * per; r < min(tid * per + per, a.requests); ++r) {
        int row;
        const int n = tokens_of(a, r, row);
        if (per == 1) req_len[r] = __ldg(a.length + r), req_row[r] = row, req_n[r] = n;
        sum += (rows_of(a, row, n) + a.qt - 1) / a.qt;
      }
      const int64_t own = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += x;
      }
      if (lane == 31) warp_sum[warp] = sum;
      sum -= own;
    }
    __syncthreads();
    int64_t before = 0;
    for (int w = 0; w < 8; ++w) {
      if (w < warp) before += warp_sum[w];
      all += warp_sum[w];
    }
    scan_q[tid] = (int)(before + sum);
    all_q = all * a.kv_heads <= a.items ? (int)all : 0;  // else requests overlap in their rows: no units
    __syncthreads();
  }
  tc_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&tmem_base);

  struct Tile {
    int r, len, n, rows, row0, qi;  // n new tokens, of which `rows` have a row
  };
  auto find = [&](int q) {  // query tile q of the batch
    int seg = 0;
#pragma unroll
    for (int step = 128; step; step >>= 1)
      if (scan_q[seg + step] <= q) seg += step;
    int before = scan_q[seg];
    Tile t;
    t.len = t.n = t.rows = t.row0 = 0;
    for (t.r = seg * per; t.r < a.requests; ++t.r) {
      if (per == 1) {
        t.len = req_len[t.r], t.row0 = req_row[t.r], t.n = req_n[t.r];
      } else {
        t.len = __ldg(a.length + t.r), t.n = tokens_of(a, t.r, t.row0);
      }
      t.rows = rows_of(a, t.row0, t.n);
      const int nq = (t.rows + a.qt - 1) / a.qt;
      if (q < before + nq) break;
      before += nq;
    }
    if (t.r >= a.requests) t.r = 0, t.n = t.rows = t.len = 0;  // row starts that do not belong together: no rows
    t.qi = q - before;
    return t;
  };
  auto key_tiles = [&](const Tile &t) { return (span_of(a, t.len, t.n, t.rows, t.qi).tiles + PR_RECS - 1) / PR_RECS; };

  // Up to PR_MAX_SORT query tiles are taken longest first, and the longest are
  // cut into parts of `each` key tiles where there are too few to go round.
  // Cut ones come first, and are fewer than 2 gridDim.x parts: their number is
  // at most all / each + (those longer than 1.25 each) <= 1.8 gridDim.x.
  const bool sorted = all_q <= PR_MAX_SORT;
  int each, units;
  if (sorted) {
    int sum = 0;  // two query tiles of at most 2^24 key tiles
    for (int q = tid; q < all_q; q += PR_THREADS) {
      const int n = key_tiles(find(q));
      tiles_of[q] = (uint16_t)min(n, 65535);
      sum += n;
    }
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (tid == 0) tile_sum = 0;
    __syncthreads();
    if (lane == 0) atomicAdd(&tile_sum, (unsigned long long)sum);
    __syncthreads();
    const int64_t all = (int64_t)tile_sum * a.kv_heads;
    each = a.whole ? INT_MAX / 2 : (int)min(max((int64_t)PR_LEAST, (all + gridDim.x - 1) / gridDim.x), (int64_t)INT_MAX / 2);
    for (int q = tid; q < all_q; q += PR_THREADS) {
      int rank = 0;
      const int mine = tiles_of[q];
      for (int k = 0; k < all_q; ++k) rank += tiles_of[k] > mine || (tiles_of[k] == mine && k < q);
      order[rank] = (uint16_t)q;
    }
    __syncthreads();
    auto parts_of = [&](int n) { return n > each + each / 4 ? (n + each - 1) / each : 1; };
    if (warp == 0) {  // parts before each
      int before = 0;
      for (int k = 0; k < all_q; k += 32) {
        int n = k + lane < all_q ? parts_of(tiles_of[order[k + lane]]) : 0;
        const int own = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, n, d);
          if (lane >= d) n += x;
        }
        if (k + lane < all_q) part0[k + lane] = before + n - own;
        before += __shfl_sync(0xffffffffu, n, 31);
      }
      if (lane == 0) part0[all_q] = before;
    }
    __syncthreads();
    units = part0[all_q] * a.kv_heads;
  } else {
    units = all_q * a.kv_heads;
  }

  uint32_t phase = 0;  // key tiles that this block has been through: one phase of every barrier each (of b_k's two in turn)
  int unit = blockIdx.x;
  while (unit < units) {
    // ---- the unit
    const int head = unit % a.kv_heads, ui = unit / a.kv_heads;
    int q, parts = 1, part = 0;
    if (sorted) {
      int lo = 0, hi = all_q;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (part0[mid] <= ui) lo = mid; else hi = mid;
      }
      q = order[lo], part = ui - part0[lo], parts = part0[lo + 1] - part0[lo];
    } else {
      q = all_q - 1 - ui;
    }
    const Tile t = find(q);
    const Span s = span_of(a, t.len, t.n, t.rows, t.qi);
    const int all_tiles = (s.tiles + PR_RECS - 1) / PR_RECS, share = (all_tiles + parts - 1) / parts;
    const int j0 = min(part * share, all_tiles), j1 = min(j0 + share, all_tiles);
    const int row0 = t.row0 + t.qi * a.qt, nrow = min(a.qt, t.rows - t.qi * a.qt) * a.group;
    auto key_rec = [&](int rec) { return rec < s.sink ? rec : rec - s.sink + s.lo; };

    // ---- queries: row = token x group + head of the group
    float sum_s = 0.0f, factor = 1.0f;  // a row's scores are factor (S * ks + kz * sum_s), see QueryScale
    int pos = -1;
    const float of_step = step_factor(a.scale) * 0.0625f;  // codes' operands are 16 times as large
    if (warp < 4) {
      const int tok = tid / a.group;
      const int64_t row = (int64_t)row0 + tok;
      const bool on = tid < nrow && row >= 0 && row < a.rows;
      const int64_t from = row * a.q_row + (int64_t)(head * a.group + tid - tok * a.group) * a.q_head;
      if (tid < nrow) pos = s.p0 + tok;
      float top = 0.0f;
#pragma unroll 1
      for (int d = 0; d < HD; d += 32) {
        float e[32];
        load_query<LIMBS == 2, 32>(a.q, a.dtype == KV4_BF16, from + d, a.q_wide, on, e);
#pragma unroll
        for (int i = 0; i < 32; ++i) top = fmaxf(top, fabsf(e[i])), sum_s += e[i];
      }
      const QueryScale own = query_scale(a.scale, top);
      const float f = own.f;
      factor = own.factor, sum_s = own.sum_of(sum_s);
#pragma unroll 1
      for (int d0 = 0; d0 < HD; d0 += 32) {
        float e[32];
        load_query<LIMBS == 2, 32>(a.q, a.dtype == KV4_BF16, from + d0, a.q_wide, on, e);
#pragma unroll
        for (int d = d0; d < d0 + 32; d += 8) {
          uint32_t v[LIMBS][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // elements i and i + 4, as a word's codes come out
            const float y0 = e[d - d0 + i] * f, y1 = e[d - d0 + i + 4] * f;
            v[0][i] = pack_half(y0, y1);
            if constexpr (LIMBS == 2) {
              const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&v[0][i]));
              v[1][i] = pack_half(y0 - h.x, y1 - h.y);
            }
          }
#pragma unroll
          for (int l = 0; l < LIMBS; ++l)
            *reinterpret_cast<uint4 *>(sq + (l * KB + d / 64) * QB + tid * 128 + (((d / 8) & 7) ^ (tid & 7)) * 16) =
                make_uint4(v[l][0], v[l][1], v[l][2], v[l][3]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();

    float M = LOWEST, l = 0.0f, z = 0.0f;
    if (warp >= 4) {
      // ---- codes
      const int pt = tid - 128, pw = warp - 4;
      const int32_t *row_table = a.table + (int64_t)t.r * a.width;
      const int shift = a.shift - 4;
      constexpr uint32_t NONE = 0xffffffffu;
      // Lanes 0-7: the page of a tile's records, which is asked for a tile
      // before it is needed, and the records' index in the pool.
      auto page_of = [&](int j) {
        const int rec = j * PR_RECS + lane;
        if (lane >= PR_RECS || j >= j1 || rec >= s.tiles) return -2;
        const int p = key_rec(rec) >> shift;
        return p < a.width ? __ldg(row_table + p) : -1;
      };
      auto index_of = [&](int j, int pg) {
        if (pg == -2) return NONE;
        if (pg >= a.pages || pg < 0) {
          if (a.status) atomicOr(a.status, CIS2B_KV4_BAD_PAGE);
          return NONE;
        }
        return (((uint32_t)pg * a.kv_heads + head) << shift) + (key_rec(j * PR_RECS + lane) & ((1 << shift) - 1));
      };
      constexpr int KN = HD / 32;          // 16-byte pieces of keys per thread
      constexpr int VN = HD / 64;          // value tasks (8 keys x 8 elements) per thread
      uint4 kw[KN];
      uint32_t vw[VN][8];
      uint2 par;
      uint32_t ids = index_of(j0, page_of(j0));
      int page_next = page_of(j0 + 1);
      auto load_keys = [&]() {
#pragma unroll
        for (int i = 0; i < KN; ++i) {
          const int key = HD == 128 ? i * 32 + pw * 8 + (lane & 7) : i * 64 + pw * 16 + (lane >> 4) * 8 + (lane & 7);
          const int c = HD == 128 ? lane >> 3 : (lane >> 3) & 1;
          const uint32_t id = __shfl_sync(0xffffffffu, ids, key >> 4);
          kw[i] = make_uint4(0, 0, 0, 0);
          if (id != NONE)
            kw[i] = __ldg(reinterpret_cast<const uint4 *>(a.pool + (int64_t)id * REC + (key & 15) * (HD / 2) + c * 16));
        }
        const uint32_t id = __shfl_sync(0xffffffffu, ids, pt >> 4 & 7);
        par = id == NONE ? make_uint2(0, 0)
                         : __ldg(reinterpret_cast<const uint2 *>(a.pool + (int64_t)id * REC + 16 * HD + (pt & 15) * 8));
      };
      auto load_values = [&]() {
#pragma unroll
        for (int i = 0; i < VN; ++i) {
          const int kg = HD == 128 ? i * 8 + pw * 2 + (lane >> 4) : pw * 4 + (lane >> 3), word = lane & (HD / 8 - 1);
          const uint32_t id = __shfl_sync(0xffffffffu, ids, kg >> 1);
          const uint8_t *p = a.pool + (int64_t)(id == NONE ? 0 : id) * REC + 8 * HD + (kg & 1) * 8 * (HD / 2) + word * 4;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            vw[i][k] = id == NONE ? 0u : __ldg(reinterpret_cast<const uint32_t *>(p + k * (HD / 2)));
        }
      };
      auto store_keys = [&](uint32_t now) {
        if (pw == 0 && lane < PR_RECS) held[now & 1][lane] = ids != NONE;
        float *dst = reinterpret_cast<float *>(sp + (now & 1) * 128 + (pt >> 1) * 2) + (pt & 1);
        const float ks = bf16_lo(par.x), vs = bf16_lo(par.y), vz = fmaf(7.5f, vs, bf16_hi(par.y));
        dst[0] = ks * of_step, dst[2] = fmaf(7.5f, ks, bf16_hi(par.x));
        dst[4] = vs, dst[6] = vz;
        // The largest logarithm, not that of the largest, bounds what the row
        // warps add for each key.
        const float log_size = lg2(size_of(vs, vz));
        reinterpret_cast<float *>(value_log[now & 1])[pt] = log_size;
        int most = __float_as_int(log_size);
        most = __reduce_max_sync(0xffffffffu, most ^ (most >> 31 & 0x7fffffff));  // whole numbers in the order of the floats
        if (lane == 0) value_part[now & 1][pw] = __int_as_float(most ^ (most >> 31 & 0x7fffffff));
#pragma unroll
        for (int i = 0; i < KN; ++i) {
          const int key = HD == 128 ? i * 32 + pw * 8 + (lane & 7) : i * 64 + pw * 16 + (lane >> 4) * 8 + (lane & 7);
          const int c = HD == 128 ? lane >> 3 : (lane >> 3) & 1;
          const uint32_t w[4] = {kw[i].x, kw[i].y, kw[i].z, kw[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t v[4];  // elements 0 and 4, 1 and 5, 2 and 6, 3 and 7 of the word
            codes_of<true>(w[k], v);
            const int piece = (c & 1) * 4 + k;
            *reinterpret_cast<uint4 *>(sk + (c >> 1) * QB + key * 128 + (piece ^ (key & 7)) * 16) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        bar_arrive(b_k(now));
      };
      auto store_values = [&](uint32_t now) {
#pragma unroll
        for (int i = 0; i < VN; ++i) {
          const int kg = HD == 128 ? i * 8 + pw * 2 + (lane >> 4) : pw * 4 + (lane >> 3), word = lane & (HD / 8 - 1);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = __byte_perm(vw[i][2 * k], vw[i][2 * k + 1], h ? 0x7632 : 0x5410);
            uint32_t y[4][4];  // [element 8 word + 4 h + e][keys 2 k and 2 k + 1]
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t v[4];
              codes_of<true>(x[k], v);
              y[0][k] = v[0], y[1][k] = v[1], y[2][k] = v[2], y[3][k] = v[3];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int n = (word >> 3) * 64 + (4 * h + e) * 8 + (word & 7);
              *reinterpret_cast<uint4 *>(sv + (kg >> 3) * VB + n * 128 + ((kg & 7) ^ (n & 7)) * 16) =
                  make_uint4(y[e][0], y[e][1], y[e][2], y[e][3]);
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        bar_arrive(b_v);
      };
      if (j0 < j1) {
        load_keys();
        load_values();
        store_keys(phase);
      }
      for (int j = j0; j < j1; ++j) {
        const uint32_t now = phase + (j - j0), parity = now & 1;
        // The next tile's keys are asked for now, its values when these are stored.
        if (j + 1 < j1) {
          ids = index_of(j + 1, page_next);
          page_next = page_of(j + 2);
          load_keys();
        }
        // The last tile's products are done: the values' place is free.
        if (j > j0 && !bar_wait(b_o, parity ^ 1, &dead)) break;
        store_values(now);
        if (j + 1 < j1) {
          load_values();
          // The scores are done: the keys' place is free.
          if (!bar_wait(b_s, parity, &dead)) break;
          store_keys(now + 1);
        }
      }
    } else {
      // ---- weights: one row per thread
      const uint32_t mine = tmem + ((uint32_t)warp << 21);  // lanes 32 warp ..
      constexpr uint32_t S_DESC = tc_idesc(PR_ROWS, PR_KEYS), O_DESC = tc_idesc(PR_ROWS, HD);
      const uint32_t aq = smem_of(sq), ak = smem_of(sk), av = smem_of(sv);
      for (int j = j0; j < j1; ++j) {
        const uint32_t now = phase + (j - j0), parity = now & 1;
        if (warp == 0) {
          // the scores take the place of the last tile's weights
          if (j > j0 && !bar_wait(b_o, parity ^ 1, &dead)) break;
          if (!bar_wait(b_k(now), now >> 1 & 1, &dead)) break;
          if (lane == 0) {
            tc_after();
#pragma unroll
            for (int l2 = 0; l2 < LIMBS; ++l2)
#pragma unroll
              for (int k = 0; k < HD / 16; ++k)
                tc_mma_ss(tmem, tc_desc(aq + ((LIMBS - 1 - l2) * KB + k / 4) * QB + (k & 3) * 32),
                          tc_desc(ak + (k / 4) * QB + (k & 3) * 32), S_DESC, l2 || k);  // the small limb first
            tc_commit(b_s);
          }
          __syncwarp();
        }
        // the parameters come from the code warps, the scores from the products
        if (!bar_wait(b_k(now), now >> 1 & 1, &dead) || !bar_wait(b_s, parity, &dead)) break;
        tc_after();
        const int rec0 = j * PR_RECS;
        // Every row sees every key of the tile: no mask.
        bool unmasked = rec0 + PR_RECS <= s.tiles;
        if (unmasked) {
          const int lo = key_rec(rec0) * 16, hi = key_rec(rec0 + PR_RECS - 1) * 16 + 15;
          unmasked = hi <= s.p0 && (a.window == 0 || lo > s.p1 - a.window || hi < a.sinks);
#pragma unroll
          for (int k = 0; k < PR_RECS; ++k) unmasked = unmasked && held[parity][k];
        }
        const float4 *params = sp + parity * 128;
        // A chunk is two records: 32 scores in; 8 words of weights (and 8 of
        // the second limb) per record out, over the record's scores.
#pragma unroll 1
        for (int c = 0; c < PR_RECS / 2; ++c) {
          const float lv_top = value_part[parity][c];  // log2 of the chunk's largest value size
          uint32_t raw[32];
          tc_ld32(raw, mine + c * 32);
          tc_wait_ld32(raw);
          float2 u[16];  // times factor: scores in units of log2
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float4 kp = params[(c * 16 + i) * 2];
            u[i] = fma2(make_float2(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1])), make_float2(kp.x, kp.y),
                        mul2(make_float2(kp.z, kp.w), make_float2(sum_s, sum_s)));
          }
          if (!unmasked) {
            uint32_t see = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int rec = rec0 + c * 2 + h;
              if (rec >= s.tiles || !held[parity][c * 2 + h]) continue;
              // keys key0 + i: i <= pos - key0, and i > pos - window - key0 or i < sinks - key0
              const int key0 = key_rec(rec) * 16, last_i = pos - key0;
              uint32_t bits = last_i < 0 ? 0u : last_i >= 15 ? 0xffffu : (2u << last_i) - 1;
              if (a.window) {
                const int first_i = last_i - a.window + 1, sink_i = a.sinks - key0;
                const uint32_t late = first_i <= 0 ? 0xffffu : first_i > 15 ? 0u : 0xffffu & ~((1u << first_i) - 1);
                const uint32_t sink = sink_i <= 0 ? 0u : sink_i > 15 ? 0xffffu : (1u << sink_i) - 1;
                bits &= late | sink;
              }
              see |= bits << (16 * h);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              u[i].x = (see >> (2 * i)) & 1 ? u[i].x : -INFINITY;
              u[i].y = (see >> (2 * i + 1)) & 1 ? u[i].y : -INFINITY;
            }
          }
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < 16; i += 2) top = fmaxf(top, fmaxf(fmaxf(u[i].x, u[i].y), fmaxf(u[i + 1].x, u[i + 1].y)));
          top *= factor;
          // Weights stay below 2^14, p below 2^100; if not, M rises to 2^8 below the top.
          bool raise = fmaxf(top + lv_top - 14.0f, top - P_MOST) > M;  // might it have to
          float w_top = -INFINITY;
          if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float4 lv = value_log[parity][c * 8 + i / 2];
              const float2 fact = make_float2(factor, factor);
              const float2 y0 = add2(mul2(u[i], fact), make_float2(lv.x, lv.y)), y1 = add2(mul2(u[i + 1], fact), make_float2(lv.z, lv.w));
              w_top = fmaxf(fmaxf(w_top, fmaxf(y0.x, y0.y)), fmaxf(y1.x, y1.y));
            }
            raise = fmaxf(w_top - 14.0f, top - P_MOST) > M;
          }
          if (__any_sync(0xffffffffu, raise)) {
            float f = 1.0f;
            if (raise) {
              const float m = ceilf(fmaxf(w_top - 8.0f, top - (P_MOST - 6.0f)));
              f = ex2(M - m);
              M = m, l *= f, z *= f;
            }
            // What stands in TMEM: this tile's earlier weights, and O.  The factor
            // may be below half precision's least where the products are not.
            tc_wait_st();  // the weights that are read back were stored asynchronously
#pragma unroll 1
            for (int k = 0; k < 2 * c; ++k) {
              uint32_t w[8 * LIMBS];
              if constexpr (LIMBS == 2) tc_ld16(w, mine + k * 16); else tc_ld8(w, mine + k * 16);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                if constexpr (LIMBS == 2) y = add2(y, __half22float2(*reinterpret_cast<const __half2 *>(&w[8 + i])));
                y = mul2(y, make_float2(f, f));
                w[i] = pack_half(y.x, y.y);
                if constexpr (LIMBS == 2) {
                  const float2 back = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                  w[8 + i] = pack_half(y.x - back.x, y.y - back.y);
                }
              }
              if constexpr (LIMBS == 2) tc_st16(mine + k * 16, w); else tc_st8(mine + k * 16, w);
            }
            if (j > j0) {
              if (!bar_wait(b_o, (now - 1) & 1, &dead)) break;
              tc_after();
#pragma unroll 1
              for (int k = 0; k < LIMBS * HD / 16; ++k) {
                uint32_t w[16];
                tc_ld16(w, mine + 128 + k * 16);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(__uint_as_float(w[i]) * f);
                tc_st16(mine + 128 + k * 16, w);
              }
            }
            tc_wait_st();
          }
          float2 l2 = make_float2(0.0f, 0.0f), z2 = l2;
          const float2 minus = make_float2(-M, -M);
          auto weigh = [&](auto masked) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t hi[8];
              [[maybe_unused]] uint32_t lo[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float2 e = fma2(u[8 * h + i], make_float2(factor, factor), minus), p = make_float2(ex2(e.x), ex2(e.y));
                const float4 vp = params[(c * 16 + 8 * h + i) * 2 + 1];
                float2 vs = make_float2(vp.x, vp.y), vz = make_float2(vp.z, vp.w);
                if constexpr (decltype(masked)::value) {  // whatever the cache holds there
                  vs.x = e.x == -INFINITY ? 0.0f : vs.x, vz.x = e.x == -INFINITY ? 0.0f : vz.x;
                  vs.y = e.y == -INFINITY ? 0.0f : vs.y, vz.y = e.y == -INFINITY ? 0.0f : vz.y;
                }
                const float2 w = mul2(p, vs);
                l2 = add2(l2, p), z2 = fma2(p, vz, z2);
                hi[i] = pack_half(w.x, w.y);
                if constexpr (LIMBS == 2) {
                  const float2 back = __half22float2(*reinterpret_cast<const __half2 *>(&hi[i]));
                  lo[i] = pack_half(w.x - back.x, w.y - back.y);
                }
              }
              tc_st8(mine + c * 32 + h * 16, hi);
              if constexpr (LIMBS == 2) tc_st8(mine + c * 32 + h * 16 + 8, lo);
            }
          };
          if (unmasked) weigh(std::false_type()); else weigh(std::true_type());
          l += l2.x + l2.y, z += z2.x + z2.y;
        }
        tc_wait_st();
        tc_before();
        bar_arrive(b_p);
        if (warp == 0) {
          if (!bar_wait(b_v, parity, &dead) || !bar_wait(b_p, parity, &dead)) break;
          if (lane == 0) {
            tc_after();
#pragma unroll
            for (int k = 0; k < PR_KEYS / 16; ++k)
#pragma unroll
              for (int l2 = 0; l2 < LIMBS; ++l2)
                tc_mma_ts(tmem + 128 + l2 * HD, tmem + k * 16 + l2 * 8, tc_desc(av + (k / 4) * VB + (k & 3) * 32),
                          O_DESC, j > j0 || k);
            tc_commit(b_o);
          }
          __syncwarp();
        }
      }
    }

    // ---- the unit's rows
    const uint32_t done = phase + (j1 - j0);
    const int64_t slot = unit;  // of a part: cut query tiles come first
    constexpr int PART = PR_ROWS * (HD + 2);
    if (warp < 4) {
      const bool any = j1 > j0 && bar_wait(b_o, (done - 1) & 1, &dead);
      tc_after();
      const int tok = tid / a.group;
      const int64_t row = (int64_t)row0 + tok;
      const bool on = tid < nrow && row >= 0 && row < a.rows;
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      const int64_t to = row * a.o_row + (int64_t)(head * a.group + tid - tok * a.group) * a.o_head;
      float *to_part = pa.part + slot * PART;
#pragma unroll 1
      for (int b = 0; b < HD / 64; ++b) {
        uint32_t x0[32], x1[32];  // columns 64 b + 8 i + word: element 8 (8 b + word) + i
#pragma unroll
        for (int i = 0; i < 32; ++i) x0[i] = x1[i] = 0;
        if (any) {
          tc_ld32(x0, tmem + ((uint32_t)warp << 21) + 128 + b * 64);
          tc_ld32(x1, tmem + ((uint32_t)warp << 21) + 128 + b * 64 + 32);
          tc_wait_ld();
          if constexpr (LIMBS == 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t y[32];
              tc_ld32(y, tmem + ((uint32_t)warp << 21) + 128 + HD + b * 64 + h * 32);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                uint32_t &x = h ? x1[i] : x0[i];
                x = __float_as_uint(__uint_as_float(x) + __uint_as_float(y[i]));
              }
            }
          }
        }
#pragma unroll
        for (int word = 0; word < 8; ++word) {
          float y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float v = __uint_as_float(i < 4 ? x0[i * 8 + word] : x1[(i - 4) * 8 + word]);
            y[i] = fmaf(v, 0.0625f, z);
          }
          const int d = 8 * (8 * b + word);
          if (parts > 1) {
            if (tid < nrow) {
              float4 *p = reinterpret_cast<float4 *>(to_part + tid * HD + d);
              p[0] = make_float4(y[0], y[1], y[2], y[3]), p[1] = make_float4(y[4], y[5], y[6], y[7]);
            }
          } else if (on) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] *= inv;
            store8(a.out, a.dtype, to + d, a.o_wide, y);
          }
        }
      }
      if (parts > 1 && tid < nrow) reinterpret_cast<float2 *>(to_part + PR_ROWS * HD)[tid] = make_float2(M, l);
      tc_before();
    }
    if (tid == 0) next_unit = *reinterpret_cast<volatile int *>(&dead) ? INT_MAX : (int)gridDim.x + (int)atomicAdd(pa.ticket, 1u);
    __syncthreads();
    if (parts > 1) {
      // ---- parts meet: the last block to arrive joins them, in their order
      const int tile0 = ui - part;  // the first part's place: cut query tiles come first
      if (tid == 0) {
        asm volatile("fence.acq_rel.gpu;" ::: "memory");  // covers the block's writes: the barrier orders them before it
        uint32_t *c = pa.counter + tile0 * a.kv_heads + head;
        last = !dead && atomicAdd(c, 1u) == (uint32_t)parts - 1;
        if (last) *c = 0;  // ready for the next call
        asm volatile("fence.acq_rel.gpu;" ::: "memory");
      }
      __syncthreads();
      if (last) {
        for (int i = tid; i < nrow * (HD / 4); i += PR_THREADS) {
          const int rr = i / (HD / 4), d = (i % (HD / 4)) * 4;
          const Joined y = join_parts(pa.part + (int64_t)(tile0 * a.kv_heads + head) * PART, (int64_t)a.kv_heads * PART, parts,
                                      nullptr, rr * HD + d, PR_ROWS * HD + 2 * rr);
          emit(a, row0, head, rr, d, y.x, y.den);
        }
      }
    }
    phase = done;
    unit = next_unit;
    __syncthreads();
  }

  // ---- the last block out leaves the tickets as it found them
  __syncthreads();
  if (dead && warp == 0) {  // products may be under way: tensor memory is theirs until they are done
    if (lane == 0) tc_commit(b_end);
    __syncwarp();
    for (int i = 0; i < PR_WAIT && !__all_sync(0xffffffffu, bar_poll(b_end, 0)); ++i) {}
  }
  __syncthreads();
  if (tid == 0) {
    if (dead && a.status) atomicOr(a.status, CIS2B_KV4_STUCK);
    if (atomicAdd(pa.ticket + 1, 1u) == gridDim.x - 1) pa.ticket[0] = pa.ticket[1] = 0;
  }
  if (warp == 7) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM) : "memory");
  // Rows past the last request are zero.
  const int used = max(0, min(__ldg(a.row_start + a.requests), a.rows));
  const int64_t chunks = (int64_t)a.kv_heads * a.group * (HD / 4);
  for (int64_t i = (int64_t)blockIdx.x * PR_THREADS + tid; i < (a.rows - used) * chunks; i += (int64_t)gridDim.x * PR_THREADS) {
    const int64_t row = used + i / chunks;
    const int rest = (int)(i % chunks);
    store4(a.out, a.dtype, row * a.o_row + rest / (HD / 4) * a.o_head + rest % (HD / 4) * 4, a.o_wide, make_float4(0, 0, 0, 0));
  }
}
