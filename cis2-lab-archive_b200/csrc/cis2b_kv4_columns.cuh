// cis2b_kv4_columns.cuh -- attention of bfloat16 rows that see alike (a drafted
// tree's, or those over an encoder's states) over the 4-bit cache, on the
// fifth-generation tensor cores.  Included by cis2b_kv4_tree.cu after
// cis2b_kv4_attn.cuh, whose argument, span and scale types it shares.
//
// An item is up to NC query columns (rows x the group of one KV head) of one
// request against its keys.  Keys are the 128 lanes of both products:
//   S[key][column] = K Q^T       K in tensor memory, Q in shared memory
//   O[element][column] += V^T W  V and W in shared memory
// so a thread of the softmax has ONE key and 16 columns, and what belongs to a
// key stays in its registers.  Per tile of 128 keys
//   a scout looks up the records and copies their codes into shared memory, up to
//     four tiles ahead;
//   four warps make K operands of them (a thread per key, into tensor memory),
//     four the V operands ([key][element], as they come: the product takes them
//     transposed);
//   one warp issues S, another O, so that neither waits for what the other does;
//   four warps for each 16 columns turn S into weights W ([key][column], transposed
//     by the product, too);
//   one warp brings the next item's queries.
// Every block takes an equal stretch of all items' tiles; items that are cut are
// joined by the last block to arrive, in their order.
//
// Operands.  A group (a key, a value) is normalised by a power of two of its own,
// a = the exponent of its largest possible element: its elements base + step c,
// times 2^(-6 - a), are rounded ONCE to half precision (11 bits; the format's
// parameters have 8).  So no token coarsens another.  Scores are S 2^(a - 6)
// factor, factor the row's own (see CO_UNIT), weights w = p 2^(a' - 6) with the
// value's a' and p = 2^(score - M) in fp32, rounded to half precision; O stands
// for 2^-12 of the result's numerator.  M is one integer per column, moves only
// when a weight that the column sees passes 2^14 (or p 2^100), and then to 2^4
// below the top; O and the sums of p are scaled then.  So weights keep 11 bits
// down to 2^-18 of the largest, and 2^-28 of it absolutely.  Sums of p are kept per
// thread in fp32 and joined at the end of the item.  A group that reads NaN makes
// its scores NaN; its operands are zero, so it leaves no trace where unseen.
// Results that are rounded to 8 bits lose nothing by keys and values of 11; with
// fp16 rows the error is 1.5 times that of exact ones, so they have the kernels
// that work on the codes themselves.
//
// What bounds it.  Per tile of head_dim 128 HBM needs 760 cycles and 64 columns'
// exponentials 512.  Their two products hold the tensor pipe for 1,024 each, by its
// counter (512 with 32 columns): four times as long as k_kv4_prompt's do for as much
// work.  The softmax's warps take 1,900, one step after another.  Both overlap in
// part: measured (64 requests, 413K keys, 8 KV heads, bf16), an item's fixed costs
// included, are 3,200 with 64 columns (298 us a call, the pipe busy for 60 percent) and
// 2,440 with 32 (226 us, 37 percent).
// Measured on the way (64 columns): 830 us with every warp walking the requests
// itself (245 KB of code, instruction fetch), 580 with a scout, 412 with the seldom
// run parts in loops (code runs the first time at 10 cycles an instruction), 322
// with codes copied to shared memory in place of loads per key, 311 with operands
// made by `and` and one multiply-add, 292 evenly shared, with a warp for queries
// and one elected lane issuing the products (120 cycles a product before), which
// narrower items gain from: 32 columns 272 to 225.  Named barriers between the softmax's warps take 50
// cycles, memory barriers 500.
#pragma once

constexpr int CO_KEYS = 128, CO_RECS = CO_KEYS / KV4_REC;
constexpr int CO_CODES = 4;      // warps that make K operands, and V operands
constexpr int CO_AHEAD = 4;      // tiles of codes in shared memory: in flight, or being made into operands
constexpr int CO_SEGMENTS = 4;   // and segments that it is ahead of the softmax
constexpr int CO_LEAST = 2;      // least tiles that a block is given
constexpr int CO_SETUP = 4;      // what an item's fixed costs come to, in tiles
constexpr int CO_BLOCKS = 160;   // at most: one for each of 148 SMs, and some to spare
// A row's factor is the scale times CO_UNIT over the power of two that the row is an
// operand with: 2^CO_UP if its largest element is 2^-11 .. 2^8 (those have one factor),
// else one that brings that to 2^3, the largest of all to 2^15.  So factors are 2^-104 to
// 2^124 times the scale and a key's part of a score 2^-112 to 2^122, and neither product
// of the two passes fp32's range where the score does not.
constexpr float CO_UNIT = 4096.0f;
constexpr int CO_UP = 7;

// Warps: the softmax first, four for each 16 columns, then K, V, then one for each
// product, the scout and one for the queries.
__host__ __device__ constexpr int co_sets(int nc) { return nc / 16; }
__host__ __device__ constexpr int co_threads(int nc) { return 32 * (4 * co_sets(nc) + 2 * CO_CODES + 4); }
__host__ __device__ constexpr int co_registers(int nc) { return nc == 64 ? 72 : 96; }  // a thread's at the launch, see below
// Workspace: a counter per block, and two parts of an item per block.
__host__ __device__ constexpr int co_part(int hd, int nc) { return nc * (hd + 2); }
__host__ __device__ constexpr int co_smem_bytes(int hd, int nc) {
  return 2 * nc * hd * 2 + (hd == 128 ? 4 : 3) * CO_KEYS * 128 + 2 * CO_KEYS * nc * 2 + CO_AHEAD * CO_RECS * kv4_rec_bytes(hd) +
         4 * CO_KEYS * 16 + 512 + 1024;
}

// Columns of this thread's lane, there when it returns: the load and its wait are
// one statement, so that nothing which uses them moves between.
__device__ __forceinline__ void tc_read(uint32_t (&r)[16], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16]; tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tc_read(uint32_t (&r)[8], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8]; tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(at)
      : "memory");
}
// Operand of which the rows of M or N lie side by side (ROW bytes of them, in
// ROW's swizzle: 16-byte piece p of line k at p ^ what follows from k) and K goes
// on line by line; `next` bytes to the following ROW bytes of M or N.
template <int ROW> __device__ __forceinline__ uint64_t tc_desc_lines(uint32_t at, uint32_t next) {
  return (uint64_t)((at >> 4) & 0x3fff) | (uint64_t)((next >> 4) & 0x3fff) << 16 | (uint64_t)(8 * ROW >> 4) << 32 | 1ull << 46 |
         (ROW == 128 ? 2ull : 4ull) << 61;
}
template <int ROW> __device__ __forceinline__ int line_piece(int k, int p) {
  static_assert(ROW == 128 || ROW == 64, "lines of 64 or 32 elements");
  return ROW == 128 ? p ^ (k & 7) : p ^ ((k >> 1) & 3);
}
constexpr int CO_WAIT = 1 << 20;  // polls of a barrier, of 0.1 us or more, before the kernel gives up

// Shared memory by its 32-bit address, which stays in a register: the address of
// a __shared__ variable is made anew for every access, from the block's number in
// its cluster, whose reading takes 20 cycles.
__device__ __forceinline__ int lds1(uint32_t at) {
  int x;
  asm volatile("ld.volatile.shared.b32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
  return x;
}
__device__ __forceinline__ uint2 lds2(uint32_t at) {
  uint2 x;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(x.x), "=r"(x.y) : "r"(at) : "memory");
  return x;
}
__device__ __forceinline__ uint4 lds4(uint32_t at) {
  uint4 x;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
  return x;
}
__device__ __forceinline__ void sts1(uint32_t at, int x) { asm volatile("st.volatile.shared.b32 [%0], %1;" ::"r"(at), "r"(x) : "memory"); }
__device__ __forceinline__ void sts4(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// Waits as bar_wait() does, but a warp whose wait gave up goes on.  All later
// waits of the block end at once, so every loop comes to its end; there are no
// other barriers on the way that a warp could be missed at.
// The polls are one statement, and a warp branches as one on their vote: many
// warps wait at any time, and what they issue the others cannot.
__device__ __forceinline__ void co_wait_one(uint32_t b, uint32_t parity, uint32_t dead) {
  if (!bar_poll(b, parity)) {
    int i = 0;
#pragma unroll 1
    while (!bar_poll(b, parity) && !lds1(dead))
      if (++i == CO_WAIT) sts1(dead, 1);
  }
}
__device__ __forceinline__ void co_wait(uint32_t b, uint32_t parity, uint32_t dead) {
  co_wait_one(b, parity, dead);
  __syncwarp();
}
// Barriers of some of the warps, which end soon or not at all: between them the
// softmax's warps go by nothing that they could see differently, a wait that ran
// out included.
__device__ __forceinline__ void co_sync(int id, int threads) { asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
// The same, and whether any thread's x holds.
__device__ __forceinline__ bool co_any(int id, int threads, bool x) {
  uint32_t y;
  asm volatile("{.reg .pred p, q; setp.ne.b32 p, %3, 0; barrier.cta.red.or.pred q, %1, %2, p; selp.b32 %0, 1, 0, q;}"
               : "=r"(y) : "r"(id), "r"(threads), "r"((int)x) : "memory");
  return y;
}
// One lane of a warp that is together.  The compiler knows that it is one, and
// issues products as they stand; behind `lane == 0` it makes a loop of each over
// the lanes that might be there (120 cycles a product).
__device__ __forceinline__ bool elected() {
  uint32_t x;
  asm volatile("{.reg .pred p; elect.sync _|p, 0xffffffff; selp.b32 %0, 1, 0, p;}" : "=r"(x));
  return x;
}
__device__ __forceinline__ float2 pair(float x) { return make_float2(x, x); }
// Powers of two by their exponent, -126 .. 127.
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// The exponent of a group's largest possible element (parameters: step low, base
// high), at least `least`, and whether they are numbers.
__device__ __forceinline__ int group_power(uint32_t params, int least) {
  return max(max((int)(params >> 7 & 0xff) - 123, (int)(params >> 23 & 0xff) - 127), least);
}
__device__ __forceinline__ bool group_fine(uint32_t params) {
  return (params & 0x7f80u) != 0x7f80u && (params & 0x7f800000u) != 0x7f800000u;
}
// Parameters as operands' of a group whose power is a, zeros if they are no
// numbers.  Operands are the elements times 2^-(a + 6): a code in bits 0-3 of a
// 16-bit word is the half-precision number c 2^-24, in bits 4-7 c 2^-20, so one
// `and` and one multiply-add with step 2^24 or 2^20, below 2^15, make each pair.
struct Group {
  __half2 step24, step20, base;
  __device__ __forceinline__ Group(uint32_t params, int a) {
    const int h = a >> 1;
    const float down = group_fine(params) ? power(-h) : 0.0f, rest = power(h - a - 6);
    const float s = group_fine(params) ? bf16_lo(params) * down * rest : 0.0f, b = group_fine(params) ? bf16_hi(params) * down * rest : 0.0f;
    step24 = __float2half2_rn(s * 16777216.0f), step20 = __float2half2_rn(s * 1048576.0f), base = __float2half2_rn(b);
  }
};
// Eight codes of a word as operands: elements 0 and 4, 1 and 5, 2 and 6, 3 and 7.
__device__ __forceinline__ uint32_t operand_of(uint32_t code, __half2 step, __half2 base) {
  const __half2 h = __hfma2(*reinterpret_cast<const __half2 *>(&code), step, base);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void operands_of(uint32_t x, const Group &g, uint32_t *v) {
  const uint32_t y = x >> 8;
  v[0] = operand_of(x & 0x000f000fu, g.step24, g.base), v[1] = operand_of(x & 0x00f000f0u, g.step20, g.base);
  v[2] = operand_of(y & 0x000f000fu, g.step24, g.base), v[3] = operand_of(y & 0x00f000f0u, g.step20, g.base);
}

template <int HD, int NC, Rows SEE>
__global__ __launch_bounds__(co_threads(NC), 1) void k_kv4_columns(AttArgs a) {
  static_assert(SEE != Rows::CAUSAL, "columns of a request see the same tiles");
  constexpr int REC = kv4_rec_bytes(HD), PART = co_part(HD, NC);
  constexpr int CN = 16, SOFT = 4 * co_sets(NC), THREADS = co_threads(NC);  // columns of a softmax warp
  constexpr int WARP_CODES = SOFT, WARP_S = WARP_CODES + 2 * CO_CODES, WARP_O = WARP_S + 1, WARP_SCOUT = WARP_O + 1, WARP_Q = WARP_SCOUT + 1;
  constexpr int WROW = NC * 2;                                    // bytes of a line of W
  constexpr uint32_t KT = HD / 2;                                 // tensor-memory columns of a K operand
  constexpr uint32_t T_K = 0, T_S = 2 * KT, T_O = T_S + 2 * NC;   // places in tensor memory
  constexpr int TMEM = T_O + NC <= 128 ? 128 : T_O + NC <= 256 ? 256 : 512;
  constexpr uint32_t QB = NC * 128, VB = CO_KEYS * 128, WB = CO_KEYS * WROW;
  constexpr int SCAN = 256;
  // A segment: an item's tiles j0 .. j1-1, which this block takes.
  struct Segment {
    int r, head, row0, ncol, n;
    int j0, j1, parts, first;  // parts: blocks that share the item; first: the first of them, -1: no more segments
    Span s;
  };
  extern __shared__ uint8_t co_smem[];
  __shared__ int scan_t[SCAN], scan_q[SCAN], req_len[SCAN], req_row[SCAN], req_n[SCAN];
  __shared__ int warp_t[8];
  __shared__ int64_t warp_q[8];
  __shared__ Segment segments[CO_SEGMENTS], current[2];
  __shared__ float col_factor[2][NC];            // of a segment's columns, where they differ
  __shared__ int col_alike[2];                   // all columns have the common factor
  __shared__ __align__(16) float col_top[NC][4];  // by softmax warp of its set
  __shared__ float col_m[NC], col_scale[NC];     // M; what a raised M scales by, at the end 1 / the sum of p
  __shared__ int64_t col_out[NC];                // a column's place in the output
  __shared__ uint32_t tmem_base;
  __shared__ Segment pending[2];                 // the items that this block began, or ended, and others share
  __shared__ int last[2];
  int tid;  // opaque, so that it stays in a register: reading it again takes 20 cycles each time
  asm volatile("mov.u32 %0, %%tid.x;" : "=r"(tid));
  const int lane = tid & 31, warp = tid >> 5;
  uint32_t s_v;  // opaque as well; what else there is stands behind it
  asm volatile("mov.u32 %0, %1;" : "=r"(s_v) : "r"((smem_of(co_smem) + 1023) & ~1023u));
  const uint32_t s_w = s_v + (HD == 128 ? 4 : 3) * VB, s_q = s_w + 2 * WB, s_raw = s_q + 2 * (HD / 64) * QB;
  const uint32_t s_scale = s_raw + CO_AHEAD * CO_RECS * REC;  // [4][keys] of a tile: of the score, log2 of the weight over p, of the weight (0: not there), of p
  const uint32_t s_kind = s_scale + 4 * CO_KEYS * 16;  // of a tile: 1: its segment's first, 2: its last, 4: there is none; from bit 8 on its records that there are
  const uint32_t s_k_kind = s_kind + 4 * CO_AHEAD, s_w_kind = s_k_kind + 16, dead = s_w_kind + 8;  // the same, passed on with K operands and with weights
  const uint32_t b0 = s_kind + 128;
  // HD = 64: V has 64 rows, the other 64 of the product are one block of zeros after both buffers.
  auto v_at = [&](uint32_t t) { return (HD == 128 ? 2 : 1) * VB * (t & 1); };
  auto v_next = [&](uint32_t t) { return HD == 128 ? VB : (t & 1 ? VB : 2 * VB); };
  auto b_raw = [&](uint32_t t) { return b0 + 8 * (t % CO_AHEAD); };
  auto b_rawfree = [&](uint32_t t) { return b0 + 8 * (CO_AHEAD + t % CO_AHEAD); };
  auto b_seg = [&](uint32_t g) { return b0 + 8 * (2 * CO_AHEAD + g % CO_SEGMENTS); };
  auto b_segfree = [&](uint32_t g) { return b0 + 8 * (2 * CO_AHEAD + CO_SEGMENTS + g % CO_SEGMENTS); };
  const uint32_t b1 = b0 + 8 * (2 * CO_AHEAD + 2 * CO_SEGMENTS);
  auto b_k = [&](uint32_t t) { return b1 + 8 * (t & 3); };
  auto b_v = [&](uint32_t t) { return b1 + 8 * (4 + (t & 1)); };
  auto b_s = [&](uint32_t t) { return b1 + 8 * (6 + (t & 1)); };
  auto b_w = [&](uint32_t t) { return b1 + 8 * (8 + (t & 1)); };
  auto b_o = [&](uint32_t t) { return b1 + 8 * (10 + (t & 1)); };
  auto b_q = [&](uint32_t g) { return b1 + 8 * (12 + (g & 1)); };
  auto b_qfree = [&](uint32_t g) { return b1 + 8 * (14 + (g & 1)); };
  const uint32_t b_end = b1 + 8 * 16;
  if (tid == 0) {
    for (uint32_t i = 0; i < CO_AHEAD; ++i) bar_init(b_raw(i), 33), bar_init(b_rawfree(i), 2 * CO_CODES);
    for (uint32_t i = 0; i < CO_SEGMENTS; ++i) bar_init(b_seg(i), 1), bar_init(b_segfree(i), 2);
    for (uint32_t i = 0; i < 4; ++i) bar_init(b_k(i), CO_CODES);
    for (uint32_t i = 0; i < 2; ++i)
      bar_init(b_v(i), CO_CODES), bar_init(b_s(i), 2), bar_init(b_w(i), SOFT), bar_init(b_o(i), 1), bar_init(b_q(i), 1), bar_init(b_qfree(i), SOFT + 1);
    bar_init(b_end, 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    sts1(dead, 0);
    pending[0].parts = pending[1].parts = 0;
  }
  if (warp == WARP_O) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_of(&tmem_base)), "n"(TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (HD == 64)
#pragma unroll 1
    for (int i = tid; i < (int)VB / 16; i += THREADS) sts4(s_v + 2 * VB + i * 16, 0, 0, 0, 0);

  // ---- tiles (with the items' fixed costs) and items before each request
  auto tiles_of = [&](int len, int n) { return (tiles_bound<SEE>(a, len, n) + CO_RECS - 1) / CO_RECS; };
  const int per = (a.requests + SCAN - 1) / SCAN;
  int all_tiles = 0;
  int64_t all_q = 0;
  {
    int st = 0;
    int64_t sqt = 0;
    if (tid < SCAN)
#pragma unroll 1
      for (int r = tid * per; r < min(tid * per + per, a.requests); ++r) {
        int row;
        const int n = tokens_of(a, r, row), on = rows_of(a, row, n), len = __ldg(a.length + r);
        if (per == 1) req_len[r] = len, req_row[r] = row, req_n[r] = n;
        if (n == 0) continue;
        const int nq = (on + a.qt - 1) / a.qt;
        st += nq * (tiles_of(len, n) + CO_SETUP), sqt += nq;
      }
    const int own_t = st;
    const int64_t own_q = sqt;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, st, d);
      const int64_t y = __shfl_up_sync(0xffffffffu, sqt, d);
      if (lane >= d) st += x, sqt += y;
    }
    if (warp < 8 && lane == 31) warp_t[warp] = st, warp_q[warp] = sqt;
    __syncthreads();
    int before_t = 0;
    int64_t before_q = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if (w < warp) before_t += warp_t[w], before_q += warp_q[w];
      all_tiles += warp_t[w], all_q += warp_q[w];
    }
    if (tid < SCAN) {
      scan_t[tid] = (before_t + st - own_t) * a.kv_heads;
      scan_q[tid] = (int)(before_q + sqt - own_q) * a.kv_heads;
    }
    if (HD == 64) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_before();
    __syncthreads();
    tc_after();
  }
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&tmem_base);
  auto key_rec = [&](const Span &s, int rec) { return rec < s.sink ? rec : rec - s.sink + s.lo; };
  constexpr uint32_t NONE = 0xffffffffu;
  constexpr int64_t NOWHERE = INT64_MIN;
  uint32_t t = 0;  // tiles that this warp has been through

  // Registers go to the softmax's warps from the codes', out of what the launch
  // gives (a scheduler's warps share 512 a lane): 72 for each of 28 warps, or 96
  // for each of 20.
  constexpr int AT_LAUNCH = co_registers(NC), R_SOFT = NC == 64 ? 80 : 128, R_CODES = NC == 64 ? 56 : 64;
  static_assert(SOFT * R_SOFT + 2 * CO_CODES * R_CODES + 4 * AT_LAUNCH <= THREADS / 32 * AT_LAUNCH, "what is taken is what is given");
  if (warp >= WARP_CODES && warp < WARP_S) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R_CODES));
    // ---- operands: a thread per key.  Loops keep the code short: what the warps of
    // an SM run between them has to stay in its instruction cache.
    const bool of_value = warp >= WARP_CODES + CO_CODES;
    const int key = (warp & 3) * 32 + lane;
    const uint32_t k_to = tmem + ((uint32_t)(warp & 3) << 21) + T_K;
#pragma unroll 1
    for (;; ++t) {
      co_wait(b_raw(t), t / CO_AHEAD & 1, dead);
      const int kind = lds1(s_kind + 4 * (t % CO_AHEAD));
      if (tid == WARP_CODES * 32) sts1(s_k_kind + 4 * (t & 3), kind);
      if (kind & 4) break;
      const bool there = kind >> (8 + (key >> 4)) & 1;
      const uint32_t rec = s_raw + (t % CO_AHEAD) * (CO_RECS * REC) + (key >> 4) * REC;
      uint2 p = lds2(rec + 16 * HD + (key & 15) * 8);
      if (!there) p = make_uint2(0, 0);  // operands of 0, whatever the codes
      const int power_k = group_power(p.x, -106), power_v = group_power(p.y, -119);
      const Group group(of_value ? p.y : p.x, of_value ? power_v : power_k);
      auto piece = [&](int from, int i) {  // four words of the key's codes
        const int c = (key & 15) * (HD / 32) + i;
        return lds4(rec + from + (c ^ ((c >> 3) & 3)) * 16);
      };
      // The product that read this place last is done: the scores of the tile
      // before last, or its values.
      if (t >= 2) co_wait(of_value ? b_o(t) : b_s(t), (t / 2 - 1) & 1, dead);
      if (!of_value) {
        // The scales of the tile four back have been read: its weights came before the scores waited for.
        // Of the score: 2^(a + 6) / CO_UNIT.  Of the weight: 2^(a - 6), log2 of it but
        // -86 at least, and the powers that go from one to the other and back to p.
        const int log = power_v - 6, most = max(log, -86);
        sts4(s_scale + ((t & 3) * CO_KEYS + key) * 16, group_fine(p.x) && group_fine(p.y) ? __float_as_uint(power(power_k - 6)) : 0x7fffffffu,
             __float_as_uint(__int_as_float(0x4b400000 + most) - 12582912.0f), there ? __float_as_uint(power(log - most)) : 0u,
             __float_as_uint(power(-most)));
        tc_after();
      }
      if (!of_value) {
#pragma unroll 1
        for (int i = 0; i < HD / 32; ++i) {
          const uint4 x = piece(0, i);
          const uint32_t word[4] = {x.x, x.y, x.z, x.w};
          uint32_t v[16];
#pragma unroll
          for (int w = 0; w < 4; ++w) operands_of(word[w], group, v + 4 * w);
          tc_st16(k_to + KT * (t & 1) + 16 * i, v);
        }
        tc_wait_st();
        tc_before();
      } else {
        const uint32_t to = s_v + v_at(t) + key * 128;
#pragma unroll 1
        for (int i = 0; i < HD / 32; ++i) {
          const uint4 x = piece(8 * HD, i);
          const uint32_t word[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t y[4];
            operands_of(word[w], group, y);
            sts4(to + (i >> 1) * VB + line_piece<128>(key, (i & 1) * 4 + w) * 16, y[0], y[1], y[2], y[3]);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      __syncwarp();
      if (lane == 0) bar_arrive(of_value ? b_v(t) : b_k(t)), bar_arrive(b_rawfree(t));
    }
    if (!of_value && lane == 0) bar_arrive(b_k(t));
  } else if (warp < SOFT) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R_SOFT));
    // ---- weights: a key and a set of 16 columns per thread
    const int set = warp >> 2, key = tid & 127, col0 = set * CN;
    const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21);
    const float common = a.scale * (1.4426950408889634f * CO_UNIT) * power(-CO_UP);
    uint32_t seg = 0, qn = 0;  // segments; those with tiles
    Segment g;
    float2 minus[CN / 2], l[CN / 2];  // -M and the sums of p, pairs of columns
    bool have = false;                // a segment whose sums are under way
#pragma unroll 1
    for (;;) {
      // ---- the last segment's sums, while the next one's first scores are made: over the keys of each warp, then over the warps
      if (have) {
        float *part = a.part + ((int64_t)blockIdx.x * 2 + ((int)blockIdx.x == g.first)) * PART;
        {
          float x[CN];
#pragma unroll
          for (int i = 0; i < CN / 2; ++i) x[2 * i] = l[i].x, x[2 * i + 1] = l[i].y;
#pragma unroll
          for (int w = CN / 2; w >= 1; w /= 2) {  // each lane ends with one column: its number's low bits
            const bool up = lane & w;
#pragma unroll
            for (int i = 0; i < w; ++i) {
              const float keep = up ? x[i + w] : x[i], give = up ? x[i] : x[i + w];
              x[i] = keep + __shfl_xor_sync(0xffffffffu, give, w);
            }
          }
#pragma unroll
          for (int w = CN; w < 32; w *= 2) x[0] += __shfl_xor_sync(0xffffffffu, x[0], w);
          if (lane < CN) col_top[col0 + lane][warp & 3] = x[0];
        }
        co_sync(1 + set, 128);
        // A thread per column: what its results are divided by, and where they go.
        if (key < CN) {
          const int c = col0 + key, tok = c / a.group;
          const float4 y = *reinterpret_cast<const float4 *>(col_top[c]);
          const float den = (y.x + y.y) + (y.z + y.w);
          const int64_t row = (int64_t)g.row0 + tok;
          // 1 / den alone: values of 2^126 leave p of 2^-116, and 2^12 over that is none that fp32 has.
          col_scale[c] = g.parts > 1 ? 1.0f : den > 0.0f || den != den ? 1.0f / den : 0.0f;
          col_out[c] = c >= g.ncol || row < 0 || row >= a.rows ? NOWHERE : row * a.o_row + (int64_t)(g.head * a.group + c - tok * a.group) * a.o_head;
          if (g.parts > 1) *reinterpret_cast<float2 *>(part + NC * HD + 2 * c) = make_float2(col_m[c], den);
        }
        co_sync(1 + set, 128);
        const bool any = g.j1 > g.j0;
        if (any) co_wait(b_o(t - 1), (t - 1) / 2 & 1, dead);
        tc_after();
        const int element = (key & ~7) + ((key & 7) >> 1) + 4 * (key & 1);  // as operands_of() puts them
#pragma unroll 1
        for (int c = col0; c < col0 + CN && c < g.ncol; c += 8) {
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = 0;
          if (any) tc_read(o, mine + T_O + c);
          if (key < HD) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int64_t at = col_out[c + i];
              const float x = __uint_as_float(o[i]) * 4096.0f * col_scale[c + i];  // the powers of V and W do not cancel
              if (at == NOWHERE) continue;
              if (g.parts > 1) part[(c + i) * HD + element] = x;
              else static_cast<__nv_bfloat16 *>(a.out)[at + element] = __float2bfloat16_rn(x);
            }
          }
        }
        tc_before();
        if (g.parts > 1 && tid == 0) pending[(int)blockIdx.x == g.first] = g;
      }
      if (tid == 0) {  // one thread looks, for all: a segment, or none if a wait ran out
        co_wait_one(b_seg(seg), seg / CO_SEGMENTS & 1, dead);
        current[seg & 1] = segments[seg % CO_SEGMENTS];
        if (lds1(dead)) current[seg & 1].first = -1;
        bar_arrive(b_segfree(seg));
      }
      co_sync(15, SOFT * 32);  // and the shared words are free again
      g = current[seg & 1];
      if (g.first < 0) break;
      ++seg, have = true;
      const int sink = g.s.sink, gap = g.s.lo - g.s.sink, recs = g.s.tiles, p0 = g.s.p0, p1 = g.s.p1;
      auto rec_of = [&](int rec) { return rec < sink ? rec : rec + gap; };
      // Records that every row sees: all_lo .. all_hi-1, and those before all_sink.
      const int all_hi = ((p0 + 1) >> 4) - gap, all_sink = a.window ? min(a.sinks >> 4, min((p0 + 1) >> 4, sink)) : 0;
      const int all_lo = a.window ? max(sink, records(max(0, p1 - a.window + 1)) - gap) : 0;
      if (g.j1 > g.j0) co_wait(b_q(qn), qn / 2 & 1, dead);
      const bool alike = col_alike[qn & 1];
#pragma unroll
      for (int i = 0; i < CN / 2; ++i) minus[i] = pair(-LOWEST), l[i] = pair(0.0f);
      if (key < CN) col_m[col0 + key] = LOWEST;  // read behind a barrier
#pragma unroll 1
      for (int j = g.j0; j < g.j1; ++j, ++t) {
        const int rec0 = j * CO_RECS;
        co_wait(b_s(t), t / 2 & 1, dead);
        tc_after();
        const uint4 scale_bits = lds4(s_scale + ((t & 3) * CO_KEYS + key) * 16);
        const float scores = __uint_as_float(scale_bits.x) * (alike ? common : 1.0f), log = __uint_as_float(scale_bits.y);
        const float weight = __uint_as_float(scale_bits.z), back = __uint_as_float(scale_bits.w);
        // Every row sees every key of the tile, if it is there.
        const bool unmasked = __all_sync(0xffffffffu, weight != 0.0f && ((rec0 >= all_lo && rec0 + CO_RECS <= all_hi) || rec0 + CO_RECS <= all_sink));
        uint32_t see = 0xffffffffu;  // bit i: column col0 + i sees the key
        if (!unmasked) {
          see = 0;
          const int rec = rec0 + (key >> 4), at = rec < recs ? rec_of(rec) * 16 + (key & 15) : INT_MAX;
          if (weight != 0.0f && at <= p1) {
            if (SEE == Rows::CROSS) {
              see = 0xffffffffu;
            } else {
#pragma unroll 4
              for (int tok = col0 / a.group; tok * a.group < min(col0 + CN, g.ncol); ++tok) {
                const int64_t row = (int64_t)g.row0 + tok;
                // From the window of the row on, or named by its mask.
                const bool sees = at > p0 ? tree_bits(a, row, at - p0 - 1) & 1
                                          : a.window == 0 || at < a.sinks || at > tree_position(a, row, p0 + 1, g.n) - a.window;
                const int c0 = max(tok * a.group - col0, 0), c1 = min((tok + 1) * a.group - col0, CN);
                if (sees) see |= (0xffffffffu >> (32 - (c1 - c0))) << c0;
              }
            }
          }
        }
        float2 e[CN / 2];
#pragma unroll 1
        for (bool again = false;; again = true) {
          // Scores in units of log2 plus the log of what the weight is times p, over M;
          // -infinity where unseen.
          {
            uint32_t raw[CN];
            tc_read(raw, mine + T_S + NC * (t & 1) + col0);
#pragma unroll
            for (int i = 0; i < CN / 2; ++i) e[i] = make_float2(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1]));
          }
          if (alike) {
#pragma unroll
            for (int i = 0; i < CN / 2; ++i) e[i] = fma2(e[i], pair(scores), pair(log));
          } else {
#pragma unroll
            for (int i = 0; i < CN / 2; ++i)
              e[i] = fma2(mul2(e[i], pair(scores)), *reinterpret_cast<const float2 *>(&col_factor[qn & 1][col0 + 2 * i]), pair(log));
          }
          if (!unmasked) {
#pragma unroll
            for (int i = 0; i < CN / 2; ++i) {
              if (!(see >> (2 * i) & 1)) e[i].x = -INFINITY;
              if (!(see >> (2 * i + 1) & 1)) e[i].y = -INFINITY;
            }
          }
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < CN / 2; ++i) {
            e[i] = add2(e[i], minus[i]);
            top[i & 1] = fmaxf(top[i & 1], fmaxf(e[i].x, e[i].y));
          }
          const bool moves = co_any(1 + set, 128, fmaxf(top[0], top[1]) > 14.0f);
          if (!moves || again) break;  // once is enough: M is as high then as it has to be
          // ---- some column's M may have to move: by the largest of the 128 keys
          // that it sees.  In loops over eight columns, since it is rare: code that is
          // seldom run is fetched at 10 cycles an instruction.
#pragma unroll 1
          for (int c = 0; c < CN; c += 8) {
            uint32_t raw[8];
            tc_read(raw, mine + T_S + NC * (t & 1) + col0 + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float x = alike ? fmaf(__uint_as_float(raw[i]), scores, log) : fmaf(__uint_as_float(raw[i]) * scores, col_factor[qn & 1][col0 + c + i], log);
              int y = x == x && see >> (c + i) & 1 ? __float_as_int(x) : __float_as_int(-INFINITY);
              y = __reduce_max_sync(0xffffffffu, y ^ (y >> 31 & 0x7fffffff));  // whole numbers in the order of the floats
              if (lane == 0) col_top[col0 + c + i][warp & 3] = __int_as_float(y ^ (y >> 31 & 0x7fffffff));
            }
          }
          co_sync(1 + set, 128);
          if (key < CN) {
            const float4 x = *reinterpret_cast<const float4 *>(col_top[col0 + key]);
            const float most = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)), m = col_m[col0 + key];
            const bool moves = most - 14.0f > m;
            const float up = moves ? ceilf(most - 4.0f) : m;
            col_scale[col0 + key] = moves ? ex2(m - up) : 1.0f, col_m[col0 + key] = up;
          }
          co_sync(1 + set, 128);
#pragma unroll
          for (int i = 0; i < CN / 2; ++i) {
            const float2 m = *reinterpret_cast<const float2 *>(&col_m[col0 + 2 * i]);
            minus[i] = make_float2(-m.x, -m.y), l[i] = mul2(l[i], *reinterpret_cast<const float2 *>(&col_scale[col0 + 2 * i]));
          }
          if (j > g.j0) {
            co_wait(b_o(t - 1), (t - 1) / 2 & 1, dead);
            tc_after();
#pragma unroll 1
            for (int c = col0; c < col0 + CN; c += 8) {
              uint32_t o[8];
              tc_read(o, mine + T_O + c);
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * col_scale[c + i]);
              tc_st8(mine + T_O + c, o);
            }
            tc_wait_st();
          }
        }
#pragma unroll
        for (int i = 0; i < CN / 2; ++i) e[i] = make_float2(ex2(e[i].x), ex2(e[i].y));
        tc_before();
        if (t >= 2) co_wait(b_o(t), (t / 2 - 1) & 1, dead);  // the weights of the tile before last have been used
        const uint32_t to = s_w + WB * (t & 1) + key * WROW;
        // In almost all tiles p times the power that `log` is of is the weight.
        if (__any_sync(0xffffffffu, weight != 1.0f)) {
#pragma unroll
          for (int i = 0; i < CN / 2; ++i) l[i] = fma2(e[i], pair(back), l[i]), e[i] = mul2(e[i], pair(weight));
        } else {
#pragma unroll
          for (int i = 0; i < CN / 2; ++i) l[i] = fma2(e[i], pair(back), l[i]);
        }
#pragma unroll
        for (int c = 0; c < CN / 8; ++c) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = pack_half(e[4 * c + i].x, e[4 * c + i].y);
          sts4(to + line_piece<WROW>(key, set * (CN / 8) + c) * 16, w[0], w[1], w[2], w[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (tid == 0) sts1(s_w_kind + 4 * (t & 1), j == g.j0);
        if (lane == 0) bar_arrive(b_w(t));
      }
      if (g.j1 > g.j0) {
        __syncwarp();
        if (lane == 0) bar_arrive(b_qfree(qn));
        ++qn;
      }
    }
    if (tid == 0) sts1(s_w_kind + 4 * (t & 1), 4);
    if (lane == 0) bar_arrive(b_w(t));
    // ---- parts meet: the last block to arrive joins them, in their order
    co_sync(15, SOFT * 32);
    if ((tid & ~32) == 0) {  // a thread for each
      const int side = tid >> 5;
      bool joins = false;
      if (pending[side].parts > 1) {
        asm volatile("fence.acq_rel.gpu;" ::: "memory");  // covers the block's writes: the barrier orders them before it
        joins = !lds1(dead) && atomicAdd(a.counter + pending[side].first, 1u) == (uint32_t)pending[side].parts - 1;
        if (joins) a.counter[pending[side].first] = 0;  // ready for the next call
        asm volatile("fence.acq_rel.gpu;" ::: "memory");
      }
      last[side] = joins;
    }
    co_sync(15, SOFT * 32);
#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
      if (!last[side]) continue;
      const Segment &of = pending[side];
      // The first block's part stands second in its place, the others' first.
      const float *p0 = a.part + (int64_t)of.first * 2 * PART + PART;
#pragma unroll 2
      for (int i = tid; i < of.ncol * (HD / 4); i += SOFT * 32) {
        const int c = i / (HD / 4), d = (i % (HD / 4)) * 4;
        const Joined y = join_parts(p0 + PART, 2 * PART, of.parts - 1, p0, c * HD + d, NC * HD + 2 * c);
        emit(a, of.row0, of.head, c, d, y.x, y.den);
      }
    }
  } else {
    if (warp == WARP_SCOUT) {
      // ---- what this block does, segment by segment and tile by tile, ahead of the others
      // Requests that overlap in their rows can have more items than the host
      // counted with: such row starts have none.
      const bool fits = all_q * a.kv_heads <= a.items;
      all_tiles = fits ? all_tiles * a.kv_heads : 0;
      const int items = fits ? (int)all_q * a.kv_heads : 0;
      const bool whole = a.whole;
      const int each = max((int)(((int64_t)all_tiles + gridDim.x - 1) / gridDim.x), CO_LEAST);
      const int *scan = whole ? scan_q : scan_t;
      int at = whole ? (int)blockIdx.x : (int)min((int64_t)blockIdx.x * each, (int64_t)all_tiles);
      const int end = whole ? items : (int)min((int64_t)at + each, (int64_t)all_tiles);
      const int shift = a.shift - 4;
      uint32_t count = 0;  // segments
      auto put_segment = [&](const Segment &g) {
        if (count >= CO_SEGMENTS) co_wait(b_segfree(count), (count / CO_SEGMENTS - 1) & 1, dead);
        if (lane == 0) segments[count % CO_SEGMENTS] = g, bar_arrive(b_seg(count));
        ++count;
      };
      auto tile_place = [&]() {
        if (t >= CO_AHEAD) co_wait(b_rawfree(t), (t / CO_AHEAD - 1) & 1, dead);
      };
      // Every lane's copies count when they are there.  That arrival is of copies alone:
      // what lane 0 writes itself is released by one of its own.
      auto tile_done = [&](int kind) {
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(b_raw(t)) : "memory");
        if (lane == 0) sts1(s_kind + 4 * (t % CO_AHEAD), kind), bar_arrive(b_raw(t));
      };
      Segment g;
      while (at < end) {
        const uint32_t coarse = __ballot_sync(0xffffffffu, scan[lane * (SCAN / 32)] <= at);
        int seg = (31 - __clz(coarse)) * (SCAN / 32);
        const uint32_t fine = __ballot_sync(0xffffffffu, scan[seg + (lane & (SCAN / 32 - 1))] <= at);
        seg += 31 - __clz(fine & ((1u << (SCAN / 32)) - 1));
        int from = scan[seg], r = seg * per, len = 0, n = 0, row0 = 0, on = 0, vt = 0, size = 1;
#pragma unroll 1
        for (; r < a.requests; ++r) {
          if (per == 1) {
            len = req_len[r], row0 = req_row[r], n = req_n[r];
          } else {
            len = __ldg(a.length + r), n = tokens_of(a, r, row0);
          }
          if (n == 0) continue;
          on = rows_of(a, row0, n);
          vt = tiles_of(len, n);
          size = whole ? 1 : vt + CO_SETUP;
          const int to = from + (on + a.qt - 1) / a.qt * a.kv_heads * size;
          if (at < to) break;
          from = to;
        }
        if (r >= a.requests) break;  // row starts that do not belong together
        const int item = (int)((uint32_t)(at - from) / (uint32_t)size);
        const int qi = (int)((uint32_t)item / (uint32_t)a.kv_heads);
        g.r = r, g.head = item - qi * a.kv_heads, g.n = n;
        g.row0 = row0 + qi * a.qt, g.ncol = min(a.qt, on - qi * a.qt) * a.group;
        g.s = span_of<SEE>(a, len, n, on, qi);
        const int tiles = (g.s.tiles + CO_RECS - 1) / CO_RECS;
        g.parts = 1, g.first = blockIdx.x;
        int j0 = 0, j1 = vt;
        if (whole) {
          at += gridDim.x;
        } else {
          const int begin = from + item * size + CO_SETUP;
          if (begin >= end) break;
          j0 = max(at, begin) - begin, j1 = min(vt, end - begin);
          at = begin + j1;
          if (j0 > 0 || j1 < vt) {
            g.first = (int)((uint32_t)begin / (uint32_t)each);
            g.parts = (int)((uint32_t)(begin + vt - 1) / (uint32_t)each) - g.first + 1;
          }
        }
        g.j0 = min(j0, tiles), g.j1 = min(j1, tiles);
        put_segment(g);
        // Lane i looks up record i of the next 32 (4 tiles).
        auto look_up = [&](int rec) {
          if (rec >= g.j1 * CO_RECS || rec >= g.s.tiles) return NONE;
          const int k = key_rec(g.s, rec), p = k >> shift;
          const int pg = p < a.width ? __ldg(a.table + (int64_t)g.r * a.width + p) : -1;
          if (pg >= a.pages || pg < 0) {
            if (a.status) atomicOr(a.status, CIS2B_KV4_BAD_PAGE);
            return NONE;
          }
          return (((uint32_t)pg * a.kv_heads + g.head) << shift) + (k & ((1 << shift) - 1));
        };
        uint32_t now = look_up(g.j0 * CO_RECS + lane), then = look_up(g.j0 * CO_RECS + 32 + lane);
#pragma unroll 1
        for (int j = g.j0; j < g.j1; ++j, ++t) {
          const int i = (j - g.j0) * CO_RECS & 31;
          if (i == 0 && j > g.j0) now = then, then = look_up(j * CO_RECS + 32 + lane);
          tile_place();
          // 16-byte pieces move within their 128 bytes so that lanes which read a piece
          // of their keys touch every bank once; the parameters' 8 stay in place.
          const uint32_t to = s_raw + (t % CO_AHEAD) * (CO_RECS * REC) + (lane ^ ((lane >> 3) & 3)) * 16;
          uint32_t there = 0;
#pragma unroll
          for (int k = 0; k < CO_RECS; ++k) {
            const uint32_t id = __shfl_sync(0xffffffffu, now, i + k);
            const bool on = id != NONE;
            const uint8_t *src = a.pool + (uint64_t)(on ? id : 0u) * REC + lane * 16;
#pragma unroll
            for (int x = 0; x < HD / 32; ++x) cp_async16(to + k * REC + x * 512, src + x * 512, on);
            cp_async16(to + k * REC + HD * 16, src + HD * 16, on && lane < 8);
            there |= (uint32_t)on << k;
          }
          tile_done((j == g.j0) | (j == g.j1 - 1) << 1 | there << 8);
        }
      }
      g.first = -1;
      put_segment(g);
      tile_place();
      tile_done(4);
    } else if (warp == WARP_Q) {
      // ---- queries: eight lanes a column, four columns at a time, a segment ahead of the softmax
      const float unit = a.scale * (1.4426950408889634f * CO_UNIT);
      constexpr int PIECES = HD / 64;  // of 8 elements
      uint32_t qn = 0;  // segments with tiles
#pragma unroll 1
      for (uint32_t seg = 0;; ++seg) {
        co_wait(b_seg(seg), seg / CO_SEGMENTS & 1, dead);
        const Segment to = segments[seg % CO_SEGMENTS];
        __syncwarp();
        if (lane == 0) bar_arrive(b_segfree(seg));
        if (to.first < 0 || lds1(dead)) break;
        if (to.j1 <= to.j0) continue;
        if (qn >= 2) co_wait(b_qfree(qn), (qn / 2 - 1) & 1, dead);
        bool all = fabsf(unit) < 2.0f * CO_UNIT;  // fp32 has the common factor's product with any key's part
        constexpr int AT_ONCE = 2;
#pragma unroll 1
        for (int c0 = 0; c0 < NC; c0 += 4 * AT_ONCE) {
          uint32_t words[AT_ONCE][PIECES][4];
          bool on[AT_ONCE];
#pragma unroll
          for (int k = 0; k < AT_ONCE; ++k) {
            const int col = c0 + 4 * k + (lane >> 3), tok = col / a.group;
            const int64_t row = (int64_t)to.row0 + tok;
            on[k] = col < to.ncol && row >= 0 && row < a.rows;
            const int64_t from = row * a.q_row + (int64_t)(to.head * a.group + col - tok * a.group) * a.q_head + (lane & 7) * (HD / 8);
#pragma unroll
            for (int w = 0; w < PIECES; ++w) load_words(a.q, from + 8 * w, a.q_wide, on[k], words[k][w]);
          }
          auto element = [&](uint32_t x, bool high) { return high ? bf16_hi(x) : bf16_lo(x); };
#pragma unroll
          for (int k = 0; k < AT_ONCE; ++k) {
            const int col = c0 + 4 * k + (lane >> 3);
            float top = 0.0f;
#pragma unroll
            for (int w = 0; w < PIECES; ++w)
#pragma unroll
              for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(element(words[k][w][i], false)), fabsf(element(words[k][w][i], true))));
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            // What half precision drops of a row of 2^-11 .. 2^8 is below 2^-21 of its largest
            // element, of others 2^-28.
            const int x = (int)(__float_as_uint(top) >> 23) - 127;
            const bool alike = !on[k] || top == 0.0f || (x >= -4 - CO_UP && x < 15 - CO_UP);
            const int up = alike ? CO_UP : x == 128 ? 0 : x == -127 ? Q_UP : max(min(3 - x, Q_UP), -112);
            const float f = top == INFINITY ? __int_as_float(0x7fffffff) : power(up);  // an infinity makes the row NaN
            if ((lane & 7) == 0) col_factor[qn & 1][col] = unit * power(-up);
            all = all && alike;
#pragma unroll
            for (int w = 0; w < PIECES; ++w) {
              const int piece = (lane & 7) * PIECES + w;
              auto two = [&](int i, bool high) { return pack_half(element(words[k][w][i], high) * f, element(words[k][w][i + 2], high) * f); };  // elements 4 apart
              sts4(s_q + ((qn & 1) * (HD / 64) + (piece >> 3)) * QB + col * 128 + line_piece<128>(col, piece & 7) * 16, two(0, false), two(0, true),
                   two(1, false), two(1, true));
            }
          }
        }
        all = __all_sync(0xffffffffu, all);
        if (lane == 0) col_alike[qn & 1] = all;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(b_q(qn));
        ++qn;
      }
    } else if (warp == WARP_S || warp == WARP_O) {
      // ---- products, a warp for each, so that neither waits for what the other waits for
      constexpr uint32_t S_DESC = tc_idesc(CO_KEYS, NC), O_DESC = tc_idesc(128, NC) | 1u << 15 | 1u << 16;  // both transposed
      uint32_t seg = 0;  // segments with tiles
#pragma unroll 1
      for (;; ++t) {
        const uint32_t odd = t & 1;
        if (warp == WARP_S) {
          co_wait(b_k(t), t / 4 & 1, dead);
          const int kind = lds1(s_k_kind + 4 * (t & 3));
          if (kind & 4) break;
          if (kind & 1) co_wait(b_q(seg), seg / 2 & 1, dead), ++seg;
          if (t >= 2) co_wait(b_w(t), (t / 2 - 1) & 1, dead);  // the scores of the tile before last have been read
          if (elected()) {
            tc_after();
            const uint64_t dq = tc_desc(s_q + ((seg - 1) & 1) * (HD / 64) * QB);
            const uint32_t ds = tmem + T_S + NC * odd, dk = tmem + T_K + KT * odd;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) tc_mma_ts(ds, dk + k * 8, dq + (((k / 4) * QB + (k & 3) * 32) >> 4), S_DESC, k);
            tc_commit(b_s(t));
            if (kind & 2) tc_commit(b_qfree(seg - 1));
            bar_arrive(b_s(t));  // who waits for the scores sees what came before b_k, too
          }
        } else {
          co_wait(b_w(t), t / 2 & 1, dead);
          const int kind = lds1(s_w_kind + 4 * odd);
          if (kind & 4) break;
          co_wait(b_v(t), t / 2 & 1, dead);
          if (elected()) {
            tc_after();
            const uint64_t dv = tc_desc_lines<128>(s_v + v_at(t), v_next(t)), dw = tc_desc_lines<WROW>(s_w + WB * odd, WB);
#pragma unroll
            for (int k = 0; k < CO_KEYS / 16; ++k) tc_mma_ss(tmem + T_O, dv + k * (2048 >> 4), dw + k * (16 * WROW >> 4), O_DESC, !(kind & 1) || k);
            tc_commit(b_o(t));
          }
        }
        __syncwarp();
      }
    }
  }

  // ---- the end
  __syncthreads();
  if (lds1(dead) && (warp == WARP_S || warp == WARP_O)) {  // products may be under way: tensor memory is theirs until they are done
    if (elected()) tc_commit(b_end);
    __syncwarp();
#pragma unroll 1
    for (int i = 0; i < CO_WAIT && !__all_sync(0xffffffffu, bar_poll(b_end, 0)); ++i) {}
  }
  __syncthreads();
  if (tid == 0 && lds1(dead) && a.status) atomicOr(a.status, CIS2B_KV4_STUCK);
  if (warp == WARP_O) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM) : "memory");
  // Rows past the last request are zero.
  const int used = max(0, min(__ldg(a.row_start + a.requests), a.rows));
  const int64_t chunks = (int64_t)a.kv_heads * a.group * (HD / 4);
#pragma unroll 1
  for (int64_t i = (int64_t)blockIdx.x * THREADS + tid; i < (a.rows - used) * chunks; i += (int64_t)gridDim.x * THREADS) {
    const int64_t row = used + i / chunks;
    const int rest = (int)(i % chunks);
    store4(a.out, a.dtype, row * a.o_row + rest / (HD / 4) * a.o_head + rest % (HD / 4) * 4, a.o_wide, make_float4(0, 0, 0, 0));
  }
}
