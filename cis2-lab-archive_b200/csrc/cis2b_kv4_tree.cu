// cis2b_kv4_tree.cu -- drafted trees over the 4-bit key/value cache, and
// attention to an encoder's states in it (include/cis2b.h): masks and positions,
// acceptance, moving what was accepted, and the two forms of attention.
#include "cis2b_kv4_attn.cuh"

namespace cis2b {
namespace {

#include "cis2b_kv4_columns.cuh"

// A request's first row and its rows, as tokens_of() and rows_of(); `fresh`
// counts new tokens that have no row, too.
struct Request {
  int row0, fresh, on;
};
__device__ __forceinline__ Request request_of(const int32_t *row_start, int r, int rows) {
  Request q;
  q.row0 = __ldg(row_start + r);
  const int row1 = __ldg(row_start + r + 1);
  q.fresh = q.row0 >= 0 && row1 > q.row0 ? row1 - q.row0 : 0;
  q.on = q.row0 < rows ? min(q.fresh, rows - q.row0) : 0;
  return q;
}

// ---------------------------------------------------------------- plan_tree

constexpr int TREE_THREADS = 128;

// A block per request, a thread per row: it walks from the row to the root
// through the parents in shared memory and fills its words from the top down
// (a parent stands before its child, so the walk only goes to lower words and
// ends).  A walk is as long as the row is deep, about 30 cycles a step; that
// and the launch bound the call.  With a window a first walk finds the depth: the
// ancestor `up` steps above a row is one that the window or the sinks hold.
__global__ __launch_bounds__(TREE_THREADS) void k_kv4_plan_tree(cis2b_kv4_tree a, int window, int sinks) {
  __shared__ int16_t parent[CIS2B_KV4_TREE_MOST];
  const int tid = threadIdx.x, most = 32 * a.words, near = window ? window : INT_MAX;
  int bad = 0;
  for (int r = blockIdx.x; r < a.requests; r += gridDim.x) {
    const Request q = request_of(a.row_start, r, a.rows);
    const int n = min(q.on, most), cached = __ldg(a.length + r) - q.fresh;
    if (q.on > most) bad |= CIS2B_KV4_TREE_ROWS;
    __syncthreads();
    for (int i = tid; i < n; i += TREE_THREADS) {
      int p = __ldg(a.parent + q.row0 + i);
      if (p < -1 || p >= i) bad |= CIS2B_KV4_TREE_PARENT, p = -1;
      parent[i] = (int16_t)p;
    }
    __syncthreads();
    for (int i = tid; i < q.on; i += TREE_THREADS) {
      int32_t *mask = a.mask + (int64_t)(q.row0 + i) * a.words;
      int depth = -1, at = i < n ? i : -1, up = 0;
      int64_t first = INT64_MAX;  // steps up to the last of the sinks
      if (window) {
        for (int x = at; x >= 0; x = parent[x]) ++depth;
        first = (int64_t)cached + depth - sinks + 1;
      }
      for (int w = a.words - 1; w >= 0; --w) {
        uint32_t bits = 0;
        for (; at >= 32 * w; at = parent[at], ++up)
          if (up < near || up >= first) bits |= 1u << (at & 31);
        mask[w] = (int32_t)bits;
      }
      a.position[q.row0 + i] = i < n ? cached + up - 1 : -1;
    }
  }
  // Rows past the last request.
  const int used = max(0, min(__ldg(a.row_start + a.requests), a.rows));
  for (int64_t i = used + (int64_t)blockIdx.x * TREE_THREADS + tid; i < a.rows; i += (int64_t)gridDim.x * TREE_THREADS) {
    for (int w = 0; w < a.words; ++w) a.mask[i * a.words + w] = 0;
    a.position[i] = -1;
  }
  if (bad && a.status) atomicOr(a.status, bad);
}

// ---------------------------------------------------------------- accept

// A block per request.  Every row whose parent agrees with it offers itself as
// the parent's successor, the lowest one counts (a minimum: no order of the
// offers matters); one thread then follows the successors from row 0, about 30
// cycles a step.
__global__ __launch_bounds__(TREE_THREADS) void k_kv4_accept(cis2b_kv4_draft a) {
  __shared__ int next[CIS2B_KV4_TREE_MOST];
  __shared__ int16_t list[CIS2B_KV4_TREE_MOST];
  __shared__ int count;
  const int tid = threadIdx.x;
  int bad = 0;
  for (int r = blockIdx.x; r < a.requests; r += gridDim.x) {
    const Request q = request_of(a.row_start, r, a.rows);
    const int n = min(q.on, CIS2B_KV4_TREE_MOST);
    if (q.on > n) bad |= CIS2B_KV4_TREE_ROWS;
    __syncthreads();
    for (int i = tid; i < n; i += TREE_THREADS) next[i] = INT_MAX;
    __syncthreads();
    for (int i = tid; i < n; i += TREE_THREADS) {
      const int p = __ldg(a.parent + q.row0 + i);
      if (p < -1 || p >= i) bad |= CIS2B_KV4_TREE_PARENT;
      else if (p >= 0 && __ldg(a.token + q.row0 + i) == __ldg(a.target + q.row0 + p)) atomicMin(next + p, i);
    }
    __syncthreads();
    if (tid == 0) {
      int k = 0;
      for (int i = n ? 0 : INT_MAX; i != INT_MAX; i = next[i]) list[k++] = (int16_t)i;
      count = k;
      a.accepted[r] = k;
      a.next_token[r] = k ? __ldg(a.target + q.row0 + list[k - 1]) : -1;
      a.kept[r] = __ldg(a.length + r) - q.fresh + k;
    }
    __syncthreads();
    for (int i = tid; i < q.on; i += TREE_THREADS) a.path[q.row0 + i] = i < count ? list[i] : -1;
  }
  const int used = max(0, min(__ldg(a.row_start + a.requests), a.rows));
  for (int64_t i = used + (int64_t)blockIdx.x * TREE_THREADS + tid; i < a.rows; i += (int64_t)gridDim.x * TREE_THREADS)
    a.path[i] = -1;
  if (bad && a.status) atomicOr(a.status, bad);
}

// ---------------------------------------------------------------- keep

constexpr int KEEP_THREADS = 64, KEEP_LAYERS = 64, KEEP_AT_ONCE = 2;

struct KeepArgs {
  uint8_t *pool[KEEP_LAYERS];
  int32_t *status[KEEP_LAYERS];
  int slots[KEEP_LAYERS];
  cis2b_kv4_kept k;
  int kv_heads, shift;
};

// A block per (request, KV head, layer).  A token's codes and parameters are
// PIECES stretches of 16 bytes (the last of 8), one per thread and turn.  A
// turn reads all its pieces before it writes any, and what it writes lies
// before everything that later turns read (path[k] >= k), so the moves are as
// if made at once.
template <int HD> __global__ __launch_bounds__(KEEP_THREADS) void k_kv4_keep(KeepArgs a) {
  constexpr int ROW = HD / 32, PIECES = 2 * ROW + 1;  // 16-byte pieces of a key or value row; of a token
  constexpr int MOVES = KEEP_THREADS * KEEP_AT_ONCE / PIECES;
  const int r = blockIdx.x, head = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x;
  const Request q = request_of(a.k.row_start, r, a.k.rows);
  const int accepted = min(__ldg(a.k.accepted + r), q.on);
  uint8_t *pool = a.pool[layer];
  const int slots = a.slots[layer];
  int bad = 0;
  auto place = [&](int slot, int piece) {
    const int page = slot >> a.shift, off = slot & ((1 << a.shift) - 1), t = off & 15;
    const int64_t rec = (((int64_t)page * a.kv_heads + head) << (a.shift - 4)) + (off >> 4);
    const int at = piece < 2 * ROW ? (piece >= ROW ? 8 * HD : 0) + t * (HD / 2) + (piece % ROW) * 16 : 16 * HD + t * 8;
    return pool + rec * kv4_rec_bytes(HD) + at;
  };
  for (int k0 = 0; k0 < accepted; k0 += MOVES) {
    uint4 x[KEEP_AT_ONCE];
    uint8_t *to[KEEP_AT_ONCE];
    bool wide[KEEP_AT_ONCE];
#pragma unroll
    for (int e = 0; e < KEEP_AT_ONCE; ++e) {
      const int i = e * KEEP_THREADS + tid, move = i / PIECES, piece = i - move * PIECES, k = k0 + move;
      to[e] = nullptr, wide[e] = piece < 2 * ROW;
      if (move >= MOVES || k >= accepted) continue;
      const int p = __ldg(a.k.path + q.row0 + k);
      if (p == k) continue;
      if (p < k || p >= q.on) {
        bad |= CIS2B_KV4_BAD_PATH;
        continue;
      }
      const int src = __ldg(a.k.slot + q.row0 + p), dst = __ldg(a.k.slot + q.row0 + k);
      if (src >= slots || dst >= slots) bad |= CIS2B_KV4_BAD_SLOT;
      if (src < 0 || dst < 0 || src >= slots || dst >= slots) continue;
      to[e] = place(dst, piece);
      const uint8_t *from = place(src, piece);
      if (wide[e]) {
        x[e] = *reinterpret_cast<const uint4 *>(from);
      } else {
        const uint2 y = *reinterpret_cast<const uint2 *>(from);
        x[e] = make_uint4(y.x, y.y, 0, 0);
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < KEEP_AT_ONCE; ++e) {
      if (!to[e]) continue;
      if (wide[e]) *reinterpret_cast<uint4 *>(to[e]) = x[e];
      else *reinterpret_cast<uint2 *>(to[e]) = make_uint2(x[e].x, x[e].y);
    }
    __syncthreads();
  }
  if (bad && a.status[layer]) atomicOr(a.status[layer], bad);
}

int check_rows(int32_t requests, int32_t rows) {
  if (requests < 1 || rows < 0) return kv4_fail(CIS2B_ERR_ARG, "tree: requests must be >= 1 and rows >= 0");
  return CIS2B_OK;
}

constexpr int TREE_BLOCKS = 65536;  // at most; more requests take turns

// ---------------------------------------------------------------- attention

// bfloat16 rows of 17 to 64 query columns a request take k_kv4_columns, with 32 or
// 64 columns an item.  Fewer columns take k_kv4_attention, more k_kv4_prompt, and so do
// fp16 rows; fp32 rows always take k_kv4_attention.  Measured both ways, us a call,
// columns first (64 requests, 413K keys, 32 over 8 heads of 128): 16 columns 206 and
// 161, 32 columns 226 and 335, 64 columns 295 and 534, 128 columns 547 and 491; 8
// prompts of 1,000 rows to encoders: 612 and 462.
// 65 to 128 columns take k_kv4_columns, twice, where a batch's items are few for the
// keys that its tables hold: k_kv4_prompt cuts only long items and leaves SMs empty, and
// its parts cost more.  Not with CIS2B_KV4_WHOLE, whose rows must not go by the batch.
// Columns first, requests of half to all of these keys, 68 columns over heads of 128:
//   keys     40 items      104          160          320         512
//   500     28 and 32   40 and 33    50 and 34    78 and 52  113 and 64
//   1,000   30 and 49   49 and 49    59 and 50    95 and 72
//   2,000   40 and 79   60 and 79    77 and 85  129 and 113
//   4,000                80 and 105              197 and 200  294 and 264
//   8,000   62 and 89  119 and 182  173 and 219  313 and 359
// 100 columns over heads of 64: 2,000 keys, 48 items 42 and 70, 96 items 61 and 73, 156
// items 81 and 73; 8,000 keys, 156 items 159 and 179, 312 items 293 and 280.
struct Columns {
  bool on;
  int nc, qt;
  uint64_t items, bytes;
};
Columns columns_of(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a) {
  Columns s{};
  const int group = a->heads / c->kv_heads;
  const int64_t cols = (int64_t)group * a->max_new;
  int64_t keys = (int64_t)a->width * c->page_size;  // that a row may see
  if (a->window) keys = std::min(keys, (int64_t)a->window + a->sinks + a->max_new);
  const bool few = !(a->flags & CIS2B_KV4_WHOLE) &&
                   (int64_t)a->requests * c->kv_heads <= std::max<int64_t>(40, std::min<int64_t>(2 * CO_BLOCKS, keys / (c->head_dim == 64 ? 16 : 10)));
  s.on = a->dtype == CIS2B_BF16 && cols > 16 && cols <= (few ? 128 : 64);
  s.nc = cols <= 32 ? 32 : 64;
  s.qt = s.nc / group;
  s.items = ((uint64_t)a->requests + (uint64_t)a->rows / s.qt) * c->kv_heads;  // at most
  s.bytes = WORK_PARTS + (uint64_t)CO_BLOCKS * 2 * co_part(c->head_dim, s.nc) * 4;
  return s;
}
static_assert(CO_BLOCKS <= WORK_ITEMS, "a counter per block");

template <int HD, int NC, Rows SEE>
int launch_columns(const AttArgs &args, const cis2b_kv4_cache *c, uint64_t most, int sms, cudaStream_t stream) {
  static std::atomic<bool> ready[64];  // by device: the attribute is set
  const int smem = co_smem_bytes(HD, NC);
  if (!ready[c->device].load(std::memory_order_relaxed)) {
    if (int rc = kv4_cuda(cudaFuncSetAttribute(k_kv4_columns<HD, NC, SEE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)))
      return rc;
    // The kernel hands registers from warp to warp, out of what it is launched with.  That
    // goes by its launch bounds, whatever its code needs; another count would make it wait.
    cudaFuncAttributes made;
    if (int rc = kv4_cuda(cudaFuncGetAttributes(&made, k_kv4_columns<HD, NC, SEE>))) return rc;
    if (made.numRegs != co_registers(NC)) return kv4_fail(CIS2B_ERR_CUDA, "k_kv4_columns was built with other registers than it counts with");
    ready[c->device].store(true, std::memory_order_relaxed);
  }
  const int grid = (int)std::max<uint64_t>(1, std::min<uint64_t>(most, std::min(sms, CO_BLOCKS)));
  k_kv4_columns<HD, NC, SEE><<<grid, co_threads(NC), smem, stream>>>(args);
  return kv4_cuda(cudaGetLastError());
}

template <Rows SEE> int run_rows(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, const AttArgs &more, void *stream) {
  if (int rc = kv4_check_cache(c, true)) return rc;
  if (int rc = check_attn(c, a)) return rc;
  const Columns s = columns_of(c, a);
  if (!s.on) return run_attention<SEE>(c, a, more, stream);
  if (s.items > ITEMS_MOST) return kv4_fail(CIS2B_ERR_ARG, "attention: (requests + rows) * kv_heads must be at most 2^30");
  if (!a->table || !a->length || !a->row_start || (a->rows && (!a->q || !a->out)))
    return kv4_fail(CIS2B_ERR_ARG, "attention: a device pointer is NULL");
  if (a->work_bytes < s.bytes || !a->work || (reinterpret_cast<uintptr_t>(a->work) & 15))
    return kv4_fail(CIS2B_ERR_ARG, "attention: work must be 16-byte aligned and hold cis2b_kv4_tree_workspace() bytes");
  int sms = 0;
  if (int rc = kv4_sm_count(c->device, &sms)) return rc;
  if (int rc = kv4_cuda(cudaSetDevice(c->device))) return rc;
  if (!a->rows) return CIS2B_OK;
  AttArgs k = more;
  Shape as{};
  as.qt = s.qt, as.items = s.items;
  fill(k, c, a, as);
  k.counter = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(a->work) + WORK_PROMPT);
  k.part = reinterpret_cast<float *>(static_cast<uint8_t *>(a->work) + WORK_PARTS);
  const uint64_t tiles = ((uint64_t)a->width * c->page_size / 16 + 1 + CO_RECS - 1) / CO_RECS;  // as tiles_bound()
  // The row of tiles is counted in 32 bits; a batch that could pass that has items enough to take them whole.
  k.whole = (a->flags & CIS2B_KV4_WHOLE) || s.items * (tiles + CO_SETUP) > INT_MAX;
  const uint64_t most = k.whole ? s.items : s.items * ((tiles + CO_SETUP + CO_LEAST - 1) / CO_LEAST);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (c->head_dim == 64)
    return s.nc == 32 ? launch_columns<64, 32, SEE>(k, c, most, sms, st) : launch_columns<64, 64, SEE>(k, c, most, sms, st);
  return s.nc == 32 ? launch_columns<128, 32, SEE>(k, c, most, sms, st) : launch_columns<128, 64, SEE>(k, c, most, sms, st);
}

}  // namespace
}  // namespace cis2b

using namespace cis2b;

extern "C" int cis2b_kv4_plan_tree(const cis2b_kv4_tree *t, void *stream) { return cis2b_kv4_plan_tree_window(t, 0, 0, stream); }

extern "C" int cis2b_kv4_plan_tree_window(const cis2b_kv4_tree *t, int32_t window, int32_t sinks, void *stream) {
  if (!t) return kv4_fail(CIS2B_ERR_ARG, "tree is NULL");
  if (int rc = check_rows(t->requests, t->rows)) return rc;
  if (t->words < 1 || 32 * t->words > CIS2B_KV4_TREE_MOST) return kv4_fail(CIS2B_ERR_ARG, "tree: words must be in 1..32");
  if (window < 0 || sinks < 0) return kv4_fail(CIS2B_ERR_ARG, "tree: window and sinks must be >= 0");
  if (!t->length || !t->row_start || (t->rows && (!t->parent || !t->mask || !t->position)))
    return kv4_fail(CIS2B_ERR_ARG, "tree: a device pointer is NULL");
  int sms = 0;
  if (int rc = kv4_sm_count(t->device, &sms)) return rc;
  if (int rc = kv4_cuda(cudaSetDevice(t->device))) return rc;
  if (!t->rows) return CIS2B_OK;
  k_kv4_plan_tree<<<std::min(t->requests, TREE_BLOCKS), TREE_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(*t, window, sinks);
  return kv4_cuda(cudaGetLastError());
}

extern "C" int cis2b_kv4_accept(const cis2b_kv4_draft *d, void *stream) {
  if (!d) return kv4_fail(CIS2B_ERR_ARG, "draft is NULL");
  if (int rc = check_rows(d->requests, d->rows)) return rc;
  if (d->reserved) return kv4_fail(CIS2B_ERR_ARG, "draft: reserved must be zero");
  if (!d->length || !d->row_start || !d->accepted || !d->next_token || !d->kept ||
      (d->rows && (!d->token || !d->parent || !d->target || !d->path)))
    return kv4_fail(CIS2B_ERR_ARG, "draft: a device pointer is NULL");
  int sms = 0;
  if (int rc = kv4_sm_count(d->device, &sms)) return rc;
  if (int rc = kv4_cuda(cudaSetDevice(d->device))) return rc;
  k_kv4_accept<<<std::min(d->requests, TREE_BLOCKS), TREE_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(*d);
  return kv4_cuda(cudaGetLastError());
}

extern "C" int cis2b_kv4_keep(const cis2b_kv4_cache *caches, int32_t n, const cis2b_kv4_kept *k, void *stream) {
  if (!k) return kv4_fail(CIS2B_ERR_ARG, "kept is NULL");
  if (int rc = check_rows(k->requests, k->rows)) return rc;
  if (k->reserved) return kv4_fail(CIS2B_ERR_ARG, "kept: reserved must be zero");
  if (n < 1 || !caches) return kv4_fail(CIS2B_ERR_ARG, "keep: at least one cache");
  if (!k->row_start || !k->accepted || (k->rows && (!k->path || !k->slot)))
    return kv4_fail(CIS2B_ERR_ARG, "kept: a device pointer is NULL");
  for (int i = 0; i < n; ++i) {
    const cis2b_kv4_cache &c = caches[i], &first = caches[0];
    if (int rc = kv4_check_cache(&c, true)) return rc;
    if (c.device != first.device || c.page_size != first.page_size || c.kv_heads != first.kv_heads || c.head_dim != first.head_dim)
      return kv4_fail(CIS2B_ERR_ARG, "keep: the caches must agree in device, page_size, kv_heads and head_dim");
  }
  if (caches->device != k->device) return kv4_fail(CIS2B_ERR_ARG, "keep: the caches are on another device");
  int sms = 0;
  if (int rc = kv4_sm_count(k->device, &sms)) return rc;
  if (int rc = kv4_cuda(cudaSetDevice(k->device))) return rc;
  if (!k->rows) return CIS2B_OK;
  for (int at = 0; at < n; at += KEEP_LAYERS) {
    KeepArgs a{};
    const int layers = std::min(n - at, KEEP_LAYERS);
    for (int i = 0; i < layers; ++i) {
      const cis2b_kv4_cache &c = caches[at + i];
      a.pool[i] = static_cast<uint8_t *>(c.pool), a.status[i] = c.status, a.slots[i] = c.pages * c.page_size;
    }
    a.k = *k, a.kv_heads = caches->kv_heads, a.shift = kv4_page_shift(caches->page_size);
    const dim3 grid(k->requests, caches->kv_heads, layers);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (caches->head_dim == 64) k_kv4_keep<64><<<grid, KEEP_THREADS, 0, s>>>(a);
    else k_kv4_keep<128><<<grid, KEEP_THREADS, 0, s>>>(a);
    if (int rc = kv4_cuda(cudaGetLastError())) return rc;
  }
  return CIS2B_OK;
}

extern "C" int cis2b_kv4_tree_workspace(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, uint64_t *out_bytes) {
  if (int rc = kv4_check_cache(c, false)) return rc;
  if (int rc = check_attn(c, a)) return rc;
  if (!out_bytes) return kv4_fail(CIS2B_ERR_ARG, "out_bytes is NULL");
  const Columns s = columns_of(c, a);
  *out_bytes = s.on ? s.bytes : shape_of(c, a, a->dtype == CIS2B_F32).bytes;
  return CIS2B_OK;
}

extern "C" int cis2b_kv4_tree_attention(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, const int32_t *mask, int32_t words,
                                        const int32_t *position, void *stream) {
  if (words < 1 || words > INT_MAX / 32) return kv4_fail(CIS2B_ERR_ARG, "tree attention: words must be in 1..2^26 - 1");
  if (a && a->rows && (!mask || (a->window && !position)))
    return kv4_fail(CIS2B_ERR_ARG, "tree attention: mask, or position with a window, is NULL");
  AttArgs more{};
  more.mask = mask, more.position = position, more.words = words;
  return run_rows<Rows::TREE>(c, a, more, stream);
}

extern "C" int cis2b_kv4_cross_attention(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, void *stream) {
  if (a && (a->window || a->sinks)) return kv4_fail(CIS2B_ERR_ARG, "cross attention: window and sinks must be 0");
  return run_rows<Rows::CROSS>(c, a, AttArgs{}, stream);
}
