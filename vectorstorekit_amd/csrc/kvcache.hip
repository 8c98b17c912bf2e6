// kvcache.hip -- keeping the pages of a key-value cache: growing, forking,
// freeing and compacting, all on the device and in stream order, so that a
// decoding loop never waits for its own bookkeeping.
//
// What decides (reference counts, table rows, lengths) is small: one workgroup
// walks it, 4,096 pages a step, and leaves a list of copies; a second launch
// moves the bytes.  Free pages go out lowest first and moves go in page
// order, so the result does not depend on the order of any atomic.
//
// One workgroup, since free pages are numbered across the whole pool; what
// bounds it is how many trips to memory follow each other.
#include "attn.hpp"
#include "vsk_api.hpp"

namespace vsk {

void check_kv(const vsk_kv *kv) {
  VSK_REQUIRE(kv->dtype >= VSK_DTYPE_F32 && kv->dtype <= VSK_DTYPE_BF16, VSK_ERR_UNSUPPORTED,
              "unknown data type");
  VSK_REQUIRE(kv->layers >= 1 && kv->pages >= 1 && kv->kv_heads >= 1 && kv->slots >= 1 &&
                  kv->width >= 1,
              VSK_ERR_INVALID_ARGUMENT, "an empty cache");
  VSK_REQUIRE(kv->head_dim >= 1 && kv->head_dim <= VSK_MAX_HEAD_DIM, VSK_ERR_UNSUPPORTED,
              "a head holds between 1 and 256 values");
  VSK_REQUIRE(kv->page_size >= 16 && kv->page_size <= (1 << 20) &&
                  (kv->page_size & (kv->page_size - 1)) == 0,
              VSK_ERR_UNSUPPORTED, "a page holds a power of two of tokens, at least 16");
  VSK_REQUIRE((int64_t)kv->width * kv->page_size <= (1ll << 30), VSK_ERR_INVALID_BUFFER_SIZE,
              "a sequence holds at most 2^30 tokens");
  // (row offsets within 16 keys are 32-bit in the kernels)
  VSK_REQUIRE(kv->k_row >= 0 && kv->v_row >= 0 && kv->k_row <= (1 << 26) &&
                  kv->v_row <= (1 << 26),
              VSK_ERR_INVALID_BUFFER_SIZE, "a row stride of more than 2^26 elements");
  VSK_REQUIRE(kv->k && kv->v && kv->table && kv->lengths && is_device_ptr(kv->k) &&
                  is_device_ptr(kv->v) && is_device_ptr(kv->table) && is_device_ptr(kv->lengths),
              VSK_ERR_INVALID_ARGUMENT, "the cache must be device memory");
}

void check_news(const vsk_new_tokens *n) {
  VSK_REQUIRE(n->n >= 0 && n->max_new >= 0 && n->tokens >= 0, VSK_ERR_INVALID_ARGUMENT,
              "negative counts");
  VSK_REQUIRE(n->tokens <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE,
              "at most 2^31 - 1 tokens");
  VSK_REQUIRE((!n->starts || is_device_ptr(n->starts)) && (!n->seqs || is_device_ptr(n->seqs)),
              VSK_ERR_INVALID_ARGUMENT, "offsets and slots must be device memory");
}

void finish_queued(vsk_ctx *ctx, hipStream_t st) {
  if (!ctx->profile) return;
  VSK_HIP(hipStreamSynchronize(st));
  ctx->resolve_pending();
}

namespace {

constexpr int NT = 1024;  // threads of the bookkeeping workgroup

struct Pool {
  char *k, *v;
  int64_t k_layer, k_page, k_row, k_head, v_layer, v_page, v_row, v_head;
  int32_t *table, *lengths, *refs, *status, *scratch;
  int64_t table_stride;
  int32_t layers, pages, page_size, shift, kv_heads, d, size, slots, width;
  // scratch: three lists of a page each, then three of a slot each (reserve: the first
  // of both)
  __device__ int32_t *page_list(int i) const { return scratch + (int64_t)i * pages; }
  __device__ int32_t *slot_list(int i) const {
    return scratch + 3 * (int64_t)pages + (int64_t)i * slots;
  }
};

Pool pool_of(const vsk_kv *kv) {
  check_kv(kv);
  VSK_REQUIRE(kv->refs && kv->status && kv->scratch && is_device_ptr(kv->refs) &&
                  is_device_ptr(kv->status) && is_device_ptr(kv->scratch),
              VSK_ERR_INVALID_ARGUMENT, "page keeping needs refs, status and scratch");
  // (the kernels step past the last page and slot in 32 bits)
  VSK_REQUIRE(kv->pages <= (1 << 30) && kv->slots <= (1 << 30), VSK_ERR_INVALID_BUFFER_SIZE,
              "page keeping for at most 2^30 pages and slots");
  Pool p;
  p.k = static_cast<char *>(kv->k);
  p.v = static_cast<char *>(kv->v);
  p.k_layer = kv->k_layer, p.k_page = kv->k_page, p.k_row = kv->k_row, p.k_head = kv->k_head;
  p.v_layer = kv->v_layer, p.v_page = kv->v_page, p.v_row = kv->v_row, p.v_head = kv->v_head;
  p.table = kv->table, p.lengths = kv->lengths, p.refs = kv->refs;
  p.status = kv->status, p.scratch = kv->scratch;
  p.table_stride = kv->table_stride;
  p.layers = kv->layers, p.pages = kv->pages, p.page_size = kv->page_size;
  p.shift = __builtin_ctz((unsigned)kv->page_size);
  p.kv_heads = kv->kv_heads, p.d = kv->head_dim, p.size = kv->dtype == VSK_DTYPE_F32 ? 4 : 2;
  p.slots = kv->slots, p.width = kv->width;
  return p;
}

// Sum of x over the threads before this one; *total: over all.
template <class I> __device__ inline I scan(I x, I *total) {
  __shared__ I waves[NT / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  I y = x;
  for (int o = 1; o < 64; o <<= 1) {
    const I z = __shfl_up(y, o);
    if (lane >= o) y += z;
  }
  __syncthreads();
  if (lane == 63) waves[w] = y;
  __syncthreads();
  I before = 0, all = 0;
  for (int i = 0; i < NT / 64; ++i) {
    if (i < w) before += waves[i];
    all += waves[i];
  }
  *total = all;
  return before + y - x;
}

// A count that atomics of this workgroup may have changed: read past the L1.
__device__ inline int32_t shared_count(const int32_t *refs, int32_t i) {
  return __hip_atomic_load(refs + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// take(rank, page) for the `want` lowest free pages in order, count(id) the
// sequences that hold one; returns how many there were.  Called by the whole
// workgroup.
template <class C, class F>
__device__ int32_t take_free(const Pool &p, int32_t want, C &&count_of, F &&take) {
  int32_t found = 0;
  for (int32_t c = 0; c < p.pages && found < want; c += 4 * NT) {
    int32_t mask = 0, count[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t id = c + 4 * (int32_t)threadIdx.x + i;
      count[i] = count_of(id < p.pages ? id : p.pages - 1);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + 4 * (int32_t)threadIdx.x + i < p.pages && count[i] <= 0) mask |= 1 << i;
    int32_t all;
    int32_t rank = found + scan((int32_t)__popc(mask), &all);
    for (int i = 0; i < 4; ++i)
      if (mask >> i & 1) {
        if (rank < want) take(rank, c + 4 * (int32_t)threadIdx.x + i);
        ++rank;
      }
    found += all;
  }
  return found < want ? found : want;
}

__device__ inline int32_t held(const Pool &p, int32_t slot) {
  const int32_t l = p.lengths[slot];
  const int32_t most = p.width << p.shift;
  return l < 0 ? 0 : l > most ? most : l;
}

// Gives back what a slot's table row holds; each entry is taken out once.
__device__ inline void release(const Pool &p, int32_t slot, int32_t i) {
  const int32_t page = atomicExch(p.table + slot * p.table_stride + i, -1);
  if ((uint32_t)page < (uint32_t)p.pages) atomicSub(p.refs + page, 1);
}

__global__ __launch_bounds__(NT) void k_kv_reserve(const Pool p, const int32_t *seqs,
                                                   const int32_t *counts, int32_t n) {
  // base: pages that the sequences before want, as far as 32 bits count (there
  // are fewer)
  int32_t *base = p.slot_list(0);
  // pages that sequences which have been cut back held still, in the places of
  // those that are taken
  int32_t *was = p.page_list(0);
  __shared__ int32_t given;
  if (threadIdx.x == 0) given = 0;
  int64_t want = 0;
  const auto counted = [](int64_t x) { return x < INT32_MAX ? (int32_t)x : INT32_MAX; };
  for (int32_t c = 0; c < n; c += NT) {
    const int32_t i = c + threadIdx.x;
    int64_t need = 0;
    if (i < n && (uint32_t)seqs[i] < (uint32_t)p.slots) {
      const int32_t l = held(p, seqs[i]), most = p.width << p.shift;
      const int32_t add = counts[i] > 0 ? counts[i] : 0;
      const int32_t to = add > most - l ? most : l + add;
      need = ((to + p.page_size - 1) >> p.shift) - ((l + p.page_size - 1) >> p.shift);
    }
    int64_t all;
    const int64_t before = scan(need, &all);
    if (i < n) base[i] = counted(want + before);
    want += all;
  }
  __syncthreads();
  const auto count = [&](int32_t id) { return p.refs[id]; };
  const int32_t got = take_free(p, counted(want), count, [&](int32_t rank, int32_t page) {
    int32_t lo = 0, hi = n;  // the last sequence whose first rank is at most this one
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) / 2;
      if (base[mid] <= rank)
        lo = mid;
      else
        hi = mid;
    }
    const int32_t slot = seqs[lo];
    const int32_t first = (held(p, slot) + p.page_size - 1) >> p.shift;
    int32_t *entry = p.table + slot * p.table_stride + first + rank - base[lo];
    const int32_t old = *entry;
    *entry = page;
    if ((uint32_t)old < (uint32_t)p.pages) was[atomicAdd(&given, 1)] = old;
    p.refs[page] = 1;
  });
  __syncthreads();
  // (given back when all are taken, so that which are free does not depend on it)
  for (int32_t r = threadIdx.x; r < given; r += NT) atomicSub(p.refs + was[r], 1);
  __shared__ unsigned long long cut;
  if (threadIdx.x == 0) cut = 0;
  __syncthreads();
  for (int32_t i = threadIdx.x; i < n; i += NT) {
    if ((uint32_t)seqs[i] >= (uint32_t)p.slots) continue;
    const int32_t l = held(p, seqs[i]), most = p.width << p.shift;
    const int32_t add = counts[i] > 0 ? counts[i] : 0;
    const int32_t to = add > most - l ? most : l + add;
    const int32_t end = i + 1 < n ? base[i + 1] : counted(want);
    int32_t have = got - base[i];
    have = have < 0 ? 0 : have > end - base[i] ? end - base[i] : have;
    const int64_t reach = ((int64_t)((l + p.page_size - 1) >> p.shift) + have) << p.shift;
    p.lengths[seqs[i]] = to < reach ? to : (int32_t)reach;
    // pages past the table's width are missing too
    const int64_t wide = ((int64_t)l + add + p.page_size - 1) >> p.shift;
    if (wide > p.width) atomicAdd(&cut, (unsigned long long)(wide - p.width));
  }
  __syncthreads();
  if (threadIdx.x == 0) p.status[0] = counted(want - got + (int64_t)cut);
}

// A wave a child: its row's and its parent's entries are loaded together, and
// nothing waits for the counts before free pages are looked for.  Children go
// in batches of a workgroup's threads, one each; what a batch needs again it
// finds in LDS.
//
// Counts change twice for every page of every child.  LOCAL: in LDS, where
// they are all read at the start and written at the end; else by atomics in
// memory, one a cycle from one workgroup.  48 branches of contexts to 2,000
// over 8,192 pages: 7.1 us, 4 more for the last pages' copies (16.4 by
// atomics behind a fence); a fork over 32,768 pages 13.4 us, over 33,000, by
// atomics, 18.5.
constexpr int32_t LOCAL_PAGES = 32768;
template <bool LOCAL>
__global__ __launch_bounds__(NT) void k_kv_fork(const Pool p, const int32_t *parents,
                                                const int32_t *children, int32_t n) {
  int32_t *src = p.slot_list(0), *dst = p.slot_list(1), *rows = p.slot_list(2);
  __shared__ int32_t sc[NT], sf[NT], sl[NT], who[NT], sd[NT];
  __shared__ int32_t held_by[LOCAL ? LOCAL_PAGES : 1];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (LOCAL) {
#pragma unroll 8
    for (int32_t i = threadIdx.x; i < p.pages; i += NT) held_by[i] = p.refs[i];
  }
  auto change = [&](int32_t page, int32_t by) {
    if ((uint32_t)page >= (uint32_t)p.pages) return;
    atomicAdd(LOCAL ? held_by + page : p.refs + page, by);
  };
  int32_t c = -1, f = -1, l = 0;
  auto stage = [&](int32_t b) {
    const int32_t i = b + threadIdx.x;
    c = f = -1, l = 0;
    if (i < n) {
      c = children[i], f = parents[i];
      if ((uint32_t)c >= (uint32_t)p.slots) c = -1;
      if (c < 0 || (uint32_t)f >= (uint32_t)p.slots) f = -1;
      if (f >= 0) l = held(p, f);
    }
    __syncthreads();
    sc[threadIdx.x] = c, sf[threadIdx.x] = f, sl[threadIdx.x] = l, sd[threadIdx.x] = -1;
    __syncthreads();
  };
  for (int32_t b = 0; b < n; b += NT) {
    stage(b);
    const int32_t m = n - b < NT ? n - b : NT;
    for (int32_t x = w; x < m; x += NT / 64) {
      const int32_t to = sc[x], from = sf[x], full = sl[x] >> p.shift;
      if (to < 0) continue;
      int32_t *mine = p.table + to * p.table_stride;
      const int32_t *its = p.table + (from < 0 ? to : from) * p.table_stride;
#pragma unroll 4
      for (int32_t y = lane; y < p.width; y += 64) {
        const int32_t old = mine[y], now = y < full ? its[y] : -1;
        mine[y] = now;
        change(old, -1);
        change(now, 1);
      }
    }
  }
  int32_t missing = 0;
  for (int32_t b = 0; b < n; b += NT) {
    if (n > NT) stage(b);
    const int32_t i = b + threadIdx.x, part = l & (p.page_size - 1);
    const int32_t last = part ? p.table[f * p.table_stride + (l >> p.shift)] : -1;
    int32_t want;
    const int32_t before = scan((int32_t)(part > 0), &want);
    if (part > 0) who[before] = threadIdx.x;
    // (this wave's atomics are done: the barrier alone would not wait for them)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const auto count = [&](int32_t id) { return LOCAL ? held_by[id] : shared_count(p.refs, id); };
    const int32_t got = take_free(p, want, count, [&](int32_t rank, int32_t page) {
      const int32_t x = who[rank];
      sd[x] = page;
      (LOCAL ? held_by : p.refs)[page] = 1;
      p.table[sc[x] * p.table_stride + (sl[x] >> p.shift)] = page;
    });
    __syncthreads();
    if (i < n) {
      const int32_t to = sd[threadIdx.x];
      src[i] = last, dst[i] = to, rows[i] = part;
      if (c >= 0) p.lengths[c] = part && to < 0 ? l & ~(p.page_size - 1) : l;
    }
    missing += want - got;
  }
  if (threadIdx.x == 0) p.status[0] = missing;
  if (LOCAL) {
#pragma unroll 8
    for (int32_t i = threadIdx.x; i < p.pages; i += NT) p.refs[i] = held_by[i];
  }
}

__global__ __launch_bounds__(256) void k_kv_free(const Pool p, const int32_t *seqs, int32_t n) {
  const int64_t cells = (int64_t)n * p.width;
  for (int64_t x = blockIdx.x * 256ll + threadIdx.x; x < cells; x += gridDim.x * 256ll) {
    const int32_t s = seqs[x / p.width], i = (int32_t)(x % p.width);
    if ((uint32_t)s >= (uint32_t)p.slots) continue;
    release(p, s, i);
    if (i == 0) p.lengths[s] = 0;
  }
}

// Lists the free pages below the number of pages in use and the used ones at
// or above it, each in order: there are as many of the one as of the other.
// place[id]: a moved page's number in the list, -1 for a free one.  Two sweeps
// over the counts, the second's next step in flight: 16,384 pages 10.5 us.
__global__ __launch_bounds__(NT) void k_kv_plan(const Pool p) {
  int32_t *hole = p.page_list(0), *mover = p.page_list(1), *place = p.page_list(2);
  int32_t used = 0;
#pragma unroll 8
  for (int32_t id = threadIdx.x; id < p.pages; id += NT) used += p.refs[id] > 0;
  int32_t live;
  scan(used, &live);
  int32_t moves = 0, holes = 0;
  auto load = [&](int32_t c, int32_t (&on)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t id = c + 4 * (int32_t)threadIdx.x + i;
      on[i] = p.refs[id < p.pages ? id : p.pages - 1];
    }
  };
  int32_t next[4];
  load(0, next);
  for (int32_t c = 0; c < p.pages; c += 4 * NT) {
    // (at most 4,096 of each a step: two counts in one word)
    int32_t count = 0, kind[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t id = c + 4 * (int32_t)threadIdx.x + i;
      const bool on = next[i] > 0;
      kind[i] = id >= p.pages ? 0 : id < live ? (on ? 0 : 1) : (on ? 1 << 16 : 0);
      count += kind[i];
    }
    load(c + 4 * NT, next);
    int32_t all;
    int32_t before = scan(count, &all);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t id = c + 4 * (int32_t)threadIdx.x + i;
      if (kind[i] == 1) hole[holes + (before & 0xFFFF)] = id;
      if (kind[i] > 1) mover[moves + (before >> 16)] = id;
      if (id < p.pages && id >= live) place[id] = kind[i] ? moves + (before >> 16) : -1;
      before += kind[i];
    }
    holes += all & 0xFFFF;
    moves += all >> 16;
  }
  if (threadIdx.x == 0) {
    p.status[1] = live;
    p.status[2] = moves;
  }
}

// Copies rows 0 .. rows[i] of page src[i] to page dst[i] in every layer, keys
// and values.  A page's rows are runs of `run_bytes` dense bytes (whole, where
// heads and rows follow each other); W bytes an access.  Bound by the bytes:
// 4,096 pages of 16 tokens, 8 bf16 heads of 128, 2 layers, 207 us, 5.2 TB/s
// read and written.
struct MoveArgs {
  const int32_t *src, *dst, *rows, *count;  // rows null: whole pages; count null: n
  int32_t n;
  int32_t runs;      // runs of a page's row (1 or kv_heads); 0: the page is one run
  int64_t run_bytes; // of one run (of one row, where the page is one run)
  int32_t pieces;    // blocks that share a page
};
template <int W> struct Word;
template <> struct Word<16> { typedef u32x4 type; };
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<2> { typedef uint16_t type; };

template <int W>
__global__ __launch_bounds__(256) void k_kv_move(const Pool p, const MoveArgs m,
                                                 const int32_t *place) {
  typedef typename Word<W>::type V;
  // compaction: the table's entries at or above the pages in use take their
  // pages' new numbers
  if (place) {
    const int32_t live = p.status[1];
    const int64_t cells = (int64_t)p.slots * p.width;
    for (int64_t x = blockIdx.x * 256ll + threadIdx.x; x < cells; x += gridDim.x * 256ll) {
      int32_t *e = p.table + x / p.width * p.table_stride + x % p.width;
      // (an entry that names a free page keeps its number)
      const int32_t r = *e >= live && *e < p.pages ? place[*e] : -1;
      if (r >= 0) *e = m.dst[r];
    }
  }
  const int32_t n = m.count ? *m.count : m.n;
  const int64_t items = (int64_t)n * p.layers * 2 * m.pieces;
  for (int64_t x = blockIdx.x; x < items; x += gridDim.x) {
    const int32_t piece = (int32_t)(x % m.pieces);
    int64_t y = x / m.pieces;
    const bool val = y & 1;
    y >>= 1;
    const int32_t layer = (int32_t)(y % p.layers), i = (int32_t)(y / p.layers);
    const int32_t from = m.src[i], to = m.dst[i];
    if ((uint32_t)from >= (uint32_t)p.pages || (uint32_t)to >= (uint32_t)p.pages) continue;
    if (place && piece == 0 && layer == 0 && !val && threadIdx.x == 0) {
      p.refs[to] = p.refs[from];
      p.refs[from] = 0;
    }
    const int32_t rows = m.rows ? m.rows[i] : p.page_size;
    const int64_t page = val ? p.v_page : p.k_page, lay = val ? p.v_layer : p.k_layer;
    char *at = (val ? p.v : p.k) + layer * lay * p.size;
    const char *s = at + from * page * p.size;
    char *d = at + to * page * p.size;
    const int64_t row_words = m.run_bytes / W * (m.runs ? m.runs : 1);
    const int64_t words = rows * row_words;
    if (m.runs == 0) {
      const V *sv = reinterpret_cast<const V *>(s);
      V *dv = reinterpret_cast<V *>(d);
      // four loads in flight a thread
      const int64_t step = 256ll * m.pieces;
      int64_t w = piece * 256 + threadIdx.x;
      for (; w + 3 * step < words; w += 4 * step) {
        const V a = sv[w], b = sv[w + step], c = sv[w + 2 * step], e = sv[w + 3 * step];
        dv[w] = a, dv[w + step] = b, dv[w + 2 * step] = c, dv[w + 3 * step] = e;
      }
      for (; w < words; w += step) dv[w] = sv[w];
    } else {
      const int64_t row = (val ? p.v_row : p.k_row) * p.size;
      const int64_t head = (val ? p.v_head : p.k_head) * p.size;
      const int64_t run_words = m.run_bytes / W;
      for (int64_t w = piece * 256 + threadIdx.x; w < words; w += 256 * m.pieces) {
        const int64_t o = w / row_words * row + w % row_words / run_words * head +
                          w % run_words * W;
        *reinterpret_cast<V *>(d + o) = *reinterpret_cast<const V *>(s + o);
      }
    }
  }
}

void launch_move(vsk_ctx *ctx, hipStream_t st, const vsk_kv *kv, const Pool &p, MoveArgs m,
                 int64_t most, const int32_t *place) {
  const int64_t size = p.size, hd = (int64_t)p.kv_heads * p.d;
  const bool whole = p.k_head == p.d && p.v_head == p.d && p.k_row == hd && p.v_row == hd;
  m.runs = whole ? 0 : p.kv_heads;
  m.run_bytes = (whole ? hd : p.d) * size;
  auto fits = [&](int64_t w) {
    const int64_t e = w / size;
    bool ok = e >= 1 && m.run_bytes % w == 0 && (uintptr_t)p.k % w == 0 &&
              (uintptr_t)p.v % w == 0 && p.k_layer % e == 0 && p.v_layer % e == 0 &&
              p.k_page % e == 0 && p.v_page % e == 0;
    if (!whole)
      ok = ok && p.k_row % e == 0 && p.v_row % e == 0 && p.k_head % e == 0 && p.v_head % e == 0;
    return ok;
  };
  const int w = fits(16) ? 16 : fits(4) ? 4 : 2;
  // a block takes about 16 KiB of a page
  const int64_t bytes = hd * size * p.page_size;
  m.pieces = (int32_t)(bytes <= (16 << 10) ? 1 : bytes / (16 << 10));
  int64_t grid = most * p.layers * 2 * m.pieces;
  if (place) {
    const int64_t cells = ceil_div((int64_t)p.slots * p.width, 256);
    grid = grid > cells ? grid : cells;
  }
  const int64_t cap = (int64_t)ctx->cu_count * 16;
  grid = grid < 1 ? 1 : grid > cap ? cap : grid;
  KernelTimer kt(ctx, "kv_move", (double)most, st);
  if (w == 16)
    k_kv_move<16><<<(unsigned)grid, 256, 0, st>>>(p, m, place);
  else if (w == 4)
    k_kv_move<4><<<(unsigned)grid, 256, 0, st>>>(p, m, place);
  else
    k_kv_move<2><<<(unsigned)grid, 256, 0, st>>>(p, m, place);
  check_launch("kv_move");
}

// A workgroup a group: the first page in which a member's table differs from
// the first member's ends the prefix.  A wave takes a member at a time, 256
// pages a step, up to the end that any wave has found so far (64 branches of
// 32,768 tokens in pages of 64: 11 us).
constexpr int SHARE_WAVES = 16;
__global__ __launch_bounds__(64 * SHARE_WAVES) void k_kv_share(
    const int32_t *table, const int32_t *lengths, int64_t stride, int32_t slots, int32_t width,
    int32_t shift, const int32_t *seqs, const int32_t *groups, int32_t n_groups, int32_t n,
    int32_t members, int32_t *prefix) {
  constexpr int NT = 64 * SHARE_WAVES;
  __shared__ int32_t pages;
  auto offset = [&](int32_t g) -> int32_t {
    const int32_t x = groups[g];
    return x < 0 ? 0 : x > n ? n : x;
  };
  const int32_t g = blockIdx.x;
  const int32_t first = offset(g), end = offset(g + 1);
  // (sequences before the first group and behind the last are in none)
  if (g == 0)
    for (int32_t b = threadIdx.x; b < first; b += NT) prefix[b] = 0;
  if (g == n_groups - 1)
    for (int32_t b = (end > first ? end : first) + threadIdx.x; b < n; b += NT) prefix[b] = 0;
  if (end <= first) return;
  auto slot_of = [&](int32_t b) -> int32_t {
    const int32_t x = seqs ? seqs[b] : b;
    return (uint32_t)x < (uint32_t)slots ? x : -1;
  };
  // the whole pages of the shortest member, of one alone its own: its keys are
  // many, as the groups' are, and divided like them (a group of more than
  // attention makes room for has none)
  if (threadIdx.x == 0) pages = end - first <= members ? width : 0;
  __syncthreads();
  for (int32_t b = first + threadIdx.x; b < end; b += NT) {
    const int32_t slot = slot_of(b);
    const int32_t l = slot < 0 ? 0 : lengths[slot], whole = l < 0 ? 0 : l >> shift;
    if (whole < width) atomicMin(&pages, whole);
  }
  __syncthreads();
  const int32_t head = slot_of(first);
  const int32_t lane = threadIdx.x & 63;
  for (int32_t b = first + 1 + (threadIdx.x >> 6); b < end; b += SHARE_WAVES) {
    const int32_t slot = slot_of(b);
    if (slot < 0 || head < 0) break;  // (no pages are left to compare)
    const int32_t *x = table + head * stride, *y = table + slot * stride;
    for (int32_t i = lane;; i += 256) {
      const int32_t most = *(volatile int32_t *)&pages;
      if (i - lane >= most) break;
      int32_t u[4], v[4];
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const int32_t j = i + 64 * z < most ? i + 64 * z : most - 1;
        u[z] = x[j], v[z] = y[j];
      }
      int32_t at = most;
#pragma unroll
      for (int z = 3; z >= 0; --z)
        if (i + 64 * z < most && (u[z] != v[z] || u[z] < 0)) at = i + 64 * z;
      if (at < most) atomicMin(&pages, at);
    }
  }
  __syncthreads();
  const int32_t shared = pages << shift;
  for (int32_t b = first + threadIdx.x; b < end; b += NT) prefix[b] = shared;
}

void check_list(const int32_t *x, int32_t n) {
  VSK_REQUIRE(n >= 0, VSK_ERR_INVALID_ARGUMENT, "negative counts");
  VSK_REQUIRE(n == 0 || (x && is_device_ptr(x)), VSK_ERR_INVALID_ARGUMENT,
              "slots, pages and counts must be device memory");
}

}  // namespace

}  // namespace vsk

using namespace vsk;

extern "C" {

int64_t vsk_kv_scratch_ints(int32_t pages, int32_t slots) {
  return pages < 0 || slots < 0 ? 0 : 3 * ((int64_t)pages + slots);
}

vsk_status vsk_kv_reserve(vsk_ctx *ctx, void *stream, const vsk_kv *kv, const int32_t *seqs,
                          const int32_t *counts, int32_t n) {
  QUEUED_API_BEGIN(ctx);
  VSK_REQUIRE(kv, VSK_ERR_INVALID_ARGUMENT, "null argument");
  const Pool p = pool_of(kv);
  check_list(seqs, n);
  check_list(counts, n);
  VSK_REQUIRE(n <= kv->slots, VSK_ERR_INVALID_ARGUMENT, "more sequences than slots");
  if (n == 0) return VSK_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  {
    KernelTimer kt(ctx, "kv_reserve", n, st);
    k_kv_reserve<<<1, NT, 0, st>>>(p, seqs, counts, n);
    check_launch("kv_reserve");
  }
  finish_queued(ctx, st);
  VSK_API_END(ctx);
}

vsk_status vsk_kv_fork(vsk_ctx *ctx, void *stream, const vsk_kv *kv, const int32_t *parents,
                       const int32_t *children, int32_t n) {
  QUEUED_API_BEGIN(ctx);
  VSK_REQUIRE(kv, VSK_ERR_INVALID_ARGUMENT, "null argument");
  const Pool p = pool_of(kv);
  check_list(parents, n);
  check_list(children, n);
  VSK_REQUIRE(n <= kv->slots, VSK_ERR_INVALID_ARGUMENT, "more sequences than slots");
  if (n == 0) return VSK_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  {
    KernelTimer kt(ctx, "kv_fork", n, st);
    if (p.pages <= LOCAL_PAGES)
      k_kv_fork<true><<<1, NT, 0, st>>>(p, parents, children, n);
    else
      k_kv_fork<false><<<1, NT, 0, st>>>(p, parents, children, n);
    check_launch("kv_fork");
  }
  MoveArgs m{};
  int32_t *lists = p.scratch + 3 * (int64_t)p.pages;
  m.src = lists;
  m.dst = lists + p.slots;
  m.rows = lists + 2 * (int64_t)p.slots;
  m.n = n;
  launch_move(ctx, st, kv, p, m, n, nullptr);
  finish_queued(ctx, st);
  VSK_API_END(ctx);
}

vsk_status vsk_kv_free(vsk_ctx *ctx, void *stream, const vsk_kv *kv, const int32_t *seqs,
                       int32_t n) {
  QUEUED_API_BEGIN(ctx);
  VSK_REQUIRE(kv, VSK_ERR_INVALID_ARGUMENT, "null argument");
  const Pool p = pool_of(kv);
  check_list(seqs, n);
  if (n == 0) return VSK_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  {
    KernelTimer kt(ctx, "kv_free", n, st);
    const int64_t blocks = ceil_div((int64_t)n * p.width, 256);
    k_kv_free<<<(unsigned)(blocks < 2048 ? blocks : 2048), 256, 0, st>>>(p, seqs, n);
    check_launch("kv_free");
  }
  finish_queued(ctx, st);
  VSK_API_END(ctx);
}

vsk_status vsk_kv_compact(vsk_ctx *ctx, void *stream, const vsk_kv *kv) {
  QUEUED_API_BEGIN(ctx);
  VSK_REQUIRE(kv, VSK_ERR_INVALID_ARGUMENT, "null argument");
  const Pool p = pool_of(kv);
  hipStream_t st = static_cast<hipStream_t>(stream);
  {
    KernelTimer kt(ctx, "kv_plan", p.pages, st);
    k_kv_plan<<<1, NT, 0, st>>>(p);
    check_launch("kv_plan");
  }
  MoveArgs m{};
  m.dst = p.scratch;
  m.src = p.scratch + p.pages;
  m.count = p.status + 2;
  launch_move(ctx, st, kv, p, m, p.pages / 2, p.scratch + 2 * (int64_t)p.pages);
  finish_queued(ctx, st);
  VSK_API_END(ctx);
}

vsk_status vsk_kv_share(vsk_ctx *ctx, void *stream, const vsk_kv *kv, const int32_t *seqs,
                        const vsk_shared_prefix *shared) {
  QUEUED_API_BEGIN(ctx);
  VSK_REQUIRE(kv && shared, VSK_ERR_INVALID_ARGUMENT, "null argument");
  check_kv(kv);
  VSK_REQUIRE(shared->n_groups >= 0 && shared->n >= 0, VSK_ERR_INVALID_ARGUMENT,
              "negative counts");
  VSK_REQUIRE(shared->n_groups <= (1 << 30) && shared->n <= (1 << 30),
              VSK_ERR_INVALID_BUFFER_SIZE, "at most 2^30 sequences and groups");
  VSK_REQUIRE(seqs || shared->n <= kv->slots, VSK_ERR_INVALID_ARGUMENT,
              "more sequences than the cache has slots");
  if (shared->n_groups == 0 || shared->n == 0) return VSK_OK;
  VSK_REQUIRE(shared->groups && shared->prefix && is_device_ptr(shared->groups) &&
                  is_device_ptr(shared->prefix) && (!seqs || is_device_ptr(seqs)),
              VSK_ERR_INVALID_ARGUMENT, "groups, prefixes and slots must be device memory");
  hipStream_t st = static_cast<hipStream_t>(stream);
  {
    KernelTimer kt(ctx, "kv_share", shared->n, st);
    k_kv_share<<<(unsigned)shared->n_groups, 64 * SHARE_WAVES, 0, st>>>(
        kv->table, kv->lengths, kv->table_stride, kv->slots, kv->width,
        __builtin_ctz((unsigned)kv->page_size), seqs, shared->groups, shared->n_groups, shared->n,
        shared->max_members, shared->prefix);
    check_launch("kv_share");
  }
  finish_queued(ctx, st);
  VSK_API_END(ctx);
}

vsk_status vsk_kv_copy(vsk_ctx *ctx, void *stream, const vsk_kv *kv, const int32_t *src,
                       const int32_t *dst, int32_t n) {
  QUEUED_API_BEGIN(ctx);
  VSK_REQUIRE(kv, VSK_ERR_INVALID_ARGUMENT, "null argument");
  const Pool p = pool_of(kv);
  check_list(src, n);
  check_list(dst, n);
  if (n == 0) return VSK_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  MoveArgs m{};
  m.src = src;
  m.dst = dst;
  m.n = n;
  launch_move(ctx, st, kv, p, m, n, nullptr);
  finish_queued(ctx, st);
  VSK_API_END(ctx);
}

}  // extern "C"
