// attention.hip -- the attention entry points (of a sequence's new tokens over
// its keys, over keys of another length, over prefixes that sequences share):
// checks, the division of the work, and the choice of kernel.
#include <cmath>

#include "attn.hpp"
#include "vsk_api.hpp"

namespace vsk {

namespace {

int32_t padded_head(int32_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// How a call's work is divided.
struct Plan {
  int32_t tiles, splits, chunk, key_tile;
  int32_t share;  // attn_rows: waves that take a row tile's keys in turn
  bool tile;      // attn_tile
};

// 16-byte loads of every operand, and stores of four values.
bool aligned_operands(const vsk_kv *kv, const vsk_attention_args *args) {
  const int64_t size = kv->dtype == VSK_DTYPE_F32 ? 4 : 2, w = 16 / size;
  const vsk_head_rows &q = args->q;
  auto at = [](const void *p, int64_t bytes) { return (uintptr_t)p % bytes == 0; };
  bool ok = kv->head_dim % w == 0 && at(q.src, 16) && at(kv->k, 16) && at(kv->v, 16) &&
            q.src_row % w == 0 && q.src_head % w == 0 && kv->k_row % w == 0 &&
            kv->k_head % w == 0 && kv->v_row % w == 0 && kv->v_head % w == 0 &&
            at(q.dst, 4 * size) && q.dst_row % 4 == 0 && q.dst_head % 4 == 0;
  if (kv->table)
    ok = ok && kv->k_layer % w == 0 && kv->v_layer % w == 0 && kv->k_page % w == 0 &&
         kv->v_page % w == 0;
  return ok;
}

// What a plan divides: n sequences of at most max_new new tokens and keys keys.
// all: every token sees every key; joined: its parts are joined with another
// plan's; room: blocks a compute unit that it has (of a prefix's row tiles).
struct Span {
  int64_t n, max_new, keys;
  bool all, joined;
  int64_t room = 1;
};

int64_t most_new(const vsk_new_tokens *news) { return news->starts ? news->max_new : 1; }

// keys of a sequence at most, of a bound that the caller gives (0: none)
int64_t most_keys(const vsk_kv *kv, int64_t bound) {
  const int64_t keys = kv->table ? (int64_t)kv->width * kv->page_size : kv->pages;
  return bound > 0 && bound < keys ? bound : keys;
}

Plan plan_of(const vsk_ctx *ctx, const vsk_kv *kv, const vsk_attention_args *args,
             const Span &span) {
  Plan p;
  const int64_t group = args->q.heads / kv->kv_heads;
  const int64_t max_new = span.max_new;
  const int64_t rows = max_new * group, pairs = span.n * kv->kv_heads;
  p.splits = 1;
  p.chunk = 1 << 30;
  p.tile = false;
  p.share = 4;
  const int64_t cus = ctx->cu_count;
  int64_t row_tile = 16, key_tile = kv->dtype == VSK_DTYPE_F32 ? 16 : 32;
  int64_t keys = span.keys;
  // Row tiles of 128 where there are rows to fill them and work for the
  // device.  Under 64 rows of a key head most of a tile would be empty; with
  // few rows in all, and few products, tiles of 16 spread over more waves and
  // end sooner; fewer still where keys are many, whose parts keep the device
  // busy either way.  Measured in 16 bits, tiles of 128 against tiles of 16
  // (us): one prompt of 2,000 tokens, 8 heads of 64 47 / 27, of 4,000 60 / 122;
  // 4 heads of 128 on one 41 / 27; of 333, 32 heads of 128 on 8, 16 / 22; 64
  // new tokens of 8 heads of 64 after 4,000 keys 23 / 15, after 30,000 25 / 33;
  // of one head after 30,000 24 / 16.
  int64_t seen = span.all ? keys : keys - (max_new < keys ? max_new : keys) / 2;
  if (args->window > 0 && args->window + (int64_t)args->sinks < seen)
    seen = args->window + (int64_t)args->sinks;
  const int64_t unit = (kv->head_dim <= 64 ? 64 : 32) * cus;
  const bool few = pairs * rows < unit &&
                   pairs * rows * seen < (seen <= 8192 ? 1024 : 256) * unit;
  if (kv->dtype != VSK_DTYPE_F32 && rows >= 64 && !few && aligned_operands(kv, args)) {
    p.tile = true;
    row_tile = ATTN_TILE_ROWS;
    key_tile = attn_tile_keys(kv->head_dim);
  }
  // In 32 bits such tiles are for rows that share their keys, in large calls: a
  // tile takes some 4 us, and its parts are as large as its keys.  Texts and keys
  // of up to so many, steps of row tiles and key tiles / us / in tiles of 16: 7 of
  // 500 over 3,001, 20 heads of 80 on 5 52,600 / 397 / 746; 6 of 300 over 9,000,
  // 12 of 96 60,900 / 441 / 537; 60 of 50 over 4,000, 28 of 128 on 4 90,000 / 705
  // / 849; 10 of 300 over 1,500, the same heads 32,000 / 233 / 273; 20 of 64 over
  // 2,000, these too 20,200 / 287 / 153; 3 of 128 5,300 / 153 / 102.  (The sides
  // meet between 20,200 and 31,600: calls there are left to tiles of 16.)  Heads
  // of 64, whose tiles of 16 leave registers for four waves, stay with those.
  if (kv->dtype == VSK_DTYPE_F32 && (span.all || span.joined) && rows >= 256 &&
      kv->head_dim > 64 && kv->head_dim <= 128 && aligned_operands(kv, args) &&
      pairs * ceil_div(rows, ATTN_TILE_ROWS) * ceil_div(keys, ATTN_TILE32_KEYS) >= 40000) {
    p.tile = true;
    row_tile = ATTN_TILE_ROWS;
    key_tile = ATTN_TILE32_KEYS;
  }
  p.tiles = (int32_t)ceil_div(rows, row_tile);
  p.key_tile = (int32_t)key_tile;
  const int64_t blocks = pairs * p.tiles;
  if (args->window > 0) {
    const int64_t reach = (int64_t)args->window + args->sinks + ceil_div(row_tile, group) +
                          2 * key_tile;
    if (reach < keys) keys = reach;
  }
  const int64_t tiles = ceil_div(keys, key_tile);
  if (!p.tile) {
    // A wave each for row tiles that fill the device several times over, or
    // with few keys twice; measured against four waves each (us): 8 f32 prompts
    // of 1,000, 32 heads of 128 on 8, window 100 (16,000 row tiles) 160 / 263;
    // one of 4,000, 8 heads of 64, window 64 (2,000) 18 / 88; 8 f16 prompts of
    // 500, 10 heads of 100 (2,560) 357 / 297.
    if (!span.joined && p.tiles >= 4 && (blocks >= 16 * cus || (blocks >= 4 * cus && keys <= 384) ||
                         (blocks >= 2 * cus && keys <= 128))) {
      p.share = 1;
      return p;
    }
    // Eight waves and no parts for short contexts: nothing to join.  Heads over
    // 64 leave room for one such block a compute unit only, in 32 bits with
    // half the bytes in flight.  Against four (us): one context of 777, 32 heads
    // of 128 on 8, 12 / 13; 100 of up to 1,000 37 / 42; 300 117 / 100; with
    // heads of 64 45 / 65; 64 of up to 300 in 32 bits 27 / 22, heads of 64 14 / 22.
    const bool many = kv->head_dim <= 64 || (kv->head_dim <= 128 && kv->dtype != VSK_DTYPE_F32 &&
                                             blocks <= 6 * cus);
    if (!span.joined && many && tiles <= (blocks < cus ? 32 : 64)) {
      // (four over other sequences' keys, which may be few, while eight of such
      // heads take a compute unit: 52 sequences of 12 heads of 96 over 6 keys 20
      // / 11, of 8 of 128 over 380 17 / 13)
      if (!span.all || kv->head_dim <= 64 || blocks <= cus) p.share = 8;
      return p;
    }
  }
  // Parts as many as keep the device supplied with blocks.
  int64_t want, per;
  bool apart = false;
  if (p.tile) {
    // A prompt's rows are many and joining them takes as long as some steps:
    // parts of at least 16 tiles, and only where a quarter of the blocks that
    // fit or less would work.  Unsplit / split after 30,000 keys, 32 heads of
    // 128 on 8 (us): 512 tokens (128 blocks) 519 / 284, 2,000 (504) 893 / 998.
    per = 16;
    want = 2 * blocks > cus ? 1 : 2 * cus;
    if (span.joined && span.all) {
      // A prefix's tiles have the other half of each compute unit's room to the
      // sequences' own keys (64 branches of 32,768, want of 1, 2 and 4 halves:
      // 99, 70 and 81 us), or, where those are few, all of it, and are joined
      // anyway (4 groups of up to 32 branches, four tokens, 23,756 keys, 9 heads
      // of 64 on 3 55 / 44 us; of 1,790, 28 of 128 on 4 48 / 33).
      want = span.room * cus;
    }
    // (parts that are joined anyway may be shorter: 16 sequences of ten tokens
    // over up to 742 keys, 64 heads of 128 on 8 35 / 30)
    if (span.joined && kv->head_dim <= 128) per = 8;
    // In 32 bits a tile takes so long that ragged texts are divided for their
    // balance (7 of up to 500 over three sets of 3,001 keys, want 2 and 12: 575 / 501 us).
    if (kv->dtype == VSK_DTYPE_F32) want = 12 * cus;
  } else {
    // A tile for each of the four waves that share a part at least.  Contexts
    // differ in length, so several rounds of blocks share the work more evenly
    // than one; each starts and is joined, so the fewer the longer a block is
    // by its head.  Measured, blocks a compute unit / us: 64 contexts to 8,192
    // of 8 key heads of 128 2 / 228, 6 / 195, 12 / 197; 200 to 4,000 of 8 heads
    // of 64 8 / 192, 16 / 164, 24 / 203; 17 of 16 f32 heads of 96, window
    // 2,048, 2 / 76, 6 / 86; 60 to 2,000 of 2 heads of 256 1 / 38, 4 / 47.  No
    // more than 64 parts a row, while there is a block for every compute unit:
    // 2 contexts of 100,000 of 8 heads of 128 121 us, in 96 parts 129.  Where a
    // join follows anyway 32-bit rows, whose steps are long, take more (6 groups
    // of drafts, 2 / 8: 216 / 138).
    per = 4;
    int64_t most = kv->head_dim <= 64 ? 16 : kv->head_dim > 128 ? 1
                   : kv->dtype != VSK_DTYPE_F32 ? 6 : span.joined ? 8 : 2;
    // Other sequences' keys of dense rows (and sets of one length) lie in step,
    // and parts that begin powers of two apart meet the same memory channels at
    // a time.  So those of cross attention are many, of 12 tiles at least and
    // never of a multiple of 8: contexts to 4,096 of 16 heads of 64 119 / 111
    // us, 64 to 8,000 of 8 key heads of 128 184 / 170, 200 to 4,000 262 / 238, 50
    // to 4,000 of 16 f32 heads of 96 253 / 205 (parts of 32 tiles 300 instead of
    // 262, of 4 tiles 24 us where 32 contexts to 6,000 of 3 key heads take 21).
    // Of several row tiles the parts to join are as many as the keys: a few
    // blocks a compute unit (20 f32 texts of 128 over 1,000 keys, 8 heads of 128
    // 80 / 61; 3 of 128 over 2,000, 28 on 4 104 / 80).
    apart = span.all && !span.joined && kv->head_dim <= 128;
    if (apart) most = p.tiles > 1 ? 4 : 32;
    // Of a prefix's several row tiles each has a start and a join to the part: four
    // tiles a wave, where that fills the device (23 branches of 2,653 keys, 28
    // heads of 128 on 4 23 / 17, 31 of 4,087, 64 on 8 38 / 33; 3 of 856, four
    // tokens, 32 on 8 13 / 16).
    if (span.joined && span.all && p.tiles > 1 && kv->dtype != VSK_DTYPE_F32 &&
        blocks * ceil_div(tiles, 16) >= cus)
      per = 16;
    want = most * cus < 64 * blocks ? most * cus : 64 * blocks;
    if (want < cus) want = cus;
  }
  int64_t chunk = ceil_div(ceil_div(tiles, ceil_div(want, blocks)), per) * per;
  if (apart) chunk = chunk < 12 ? 12 : chunk + (chunk % 8 == 0 ? 4 : 0);
  p.chunk = (int32_t)(chunk < per ? per : chunk);
  p.splits = (int32_t)ceil_div(tiles, p.chunk);
  if (p.splits < 1) p.splits = 1;
  return p;
}

// The plans of a call: its own, and before it one over the groups' prefixes.
struct Plans {
  Plan own, prefix;
  int64_t group_tokens = 0;  // new tokens of a group at most; 0: no prefixes
  int32_t parts() const { return own.splits + (group_tokens ? prefix.splits : 0); }
};

Plans plans_of(const vsk_ctx *ctx, const vsk_kv *kv, const vsk_new_tokens *news,
               const vsk_attention_args *args, bool all, const vsk_shared_prefix *shared) {
  Plans p;
  const int64_t keys = most_keys(kv, args->max_length);
  // (a window leaves little of a prefix: each sequence reads its own)
  if (shared && shared->n_groups > 0 && shared->max_members > 1 && args->window <= 0) {
    p.group_tokens = (int64_t)shared->max_members * most_new(news);
    if (p.group_tokens > news->tokens) p.group_tokens = news->tokens;
    const int64_t first = most_keys(kv, shared->max_prefix > 0 ? shared->max_prefix : keys);
    const int64_t rest = shared->max_prefix > 0 && shared->max_prefix < keys
                             ? keys - shared->max_prefix : keys;
    const int64_t room = 2 * news->n * rest < shared->n_groups * first ? 3 : 1;
    p.prefix = plan_of(ctx, kv, args,
                       Span{shared->n_groups, p.group_tokens, first, true, true, room});
    p.own = plan_of(ctx, kv, args, Span{news->n, most_new(news), rest, false, true});
  } else {
    p.own = plan_of(ctx, kv, args, Span{news->n, most_new(news), keys, all, false});
  }
  return p;
}

int64_t workspace_of(const Plans &p, const vsk_kv *kv, const vsk_new_tokens *news,
                     const vsk_attention_args *args) {
  if (p.parts() == 1) return 0;
  return (int64_t)sizeof(float) * p.parts() * news->tokens * args->q.heads *
         (padded_head(kv->head_dim) + 2);
}

void check_shapes(const vsk_kv *kv, const vsk_new_tokens *news, const vsk_attention_args *args) {
  VSK_REQUIRE(kv && news && args, VSK_ERR_INVALID_ARGUMENT, "null argument");
  VSK_REQUIRE(kv->dtype >= VSK_DTYPE_F32 && kv->dtype <= VSK_DTYPE_BF16, VSK_ERR_UNSUPPORTED,
              "unknown data type");
  VSK_REQUIRE(kv->kv_heads >= 1 && args->q.heads >= 1 && args->q.heads % kv->kv_heads == 0,
              VSK_ERR_DIMENSION_MISMATCH, "query heads must be a multiple of the key heads");
  VSK_REQUIRE(kv->head_dim >= 1 && kv->head_dim <= VSK_MAX_HEAD_DIM, VSK_ERR_UNSUPPORTED,
              "a head holds between 1 and 256 values");
  VSK_REQUIRE(news->n >= 0 && news->max_new >= 0 && news->tokens >= 0 && kv->pages >= 0 &&
                  args->window >= 0 && args->sinks >= 0 && args->max_length >= 0,
              VSK_ERR_INVALID_ARGUMENT, "negative counts");
  VSK_REQUIRE((int64_t)news->max_new * args->q.heads <= 0x3FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE,
              "too many query rows in one sequence");
}

template <class P> bool aligned_to(const P *p, int64_t bytes) {
  return ((uintptr_t)p % bytes) == 0;
}

bool optional_device(const void *p) { return !p || is_device_ptr(p); }

// sets: cross attention to them; shared: the groups' prefixes
int64_t workspace_call(vsk_ctx *ctx, const vsk_kv *kv, const vsk_new_tokens *news,
                       const vsk_attention_args *args, bool all,
                       const vsk_shared_prefix *shared) {
  if (!ctx) return 0;
  try {
    check_shapes(kv, news, args);
  } catch (...) {
    return 0;  // (the call itself says why)
  }
  // (no rows: nothing to divide)
  if (news->n == 0 || news->tokens == 0 || news->max_new == 0) return 0;
  return workspace_of(plans_of(ctx, kv, news, args, all, shared), kv, news, args);
}

void attend(vsk_ctx *ctx, void *stream, const vsk_kv *kv, int32_t layer,
            const vsk_new_tokens *news, const vsk_attention_args *args, const vsk_key_sets *sets,
            const vsk_shared_prefix *shared) {
  check_shapes(kv, news, args);
  VSK_REQUIRE(std::isfinite(args->scale) && args->scale > 0, VSK_ERR_INVALID_ARGUMENT,
              "scale must be positive and finite");
  check_news(news);
  if (news->n == 0 || news->tokens == 0 || news->max_new == 0) return;
  const bool paged = kv->table != nullptr;
  if (paged) {
    check_kv(kv);
    VSK_REQUIRE(layer >= 0 && layer < kv->layers, VSK_ERR_INVALID_ARGUMENT, "no such layer");
    VSK_REQUIRE(news->seqs || news->n <= kv->slots, VSK_ERR_INVALID_ARGUMENT,
                "more sequences than the cache has slots");
  } else {
    VSK_REQUIRE(kv->page_size == 0 && layer == 0, VSK_ERR_INVALID_ARGUMENT,
                "dense keys have no pages or layers");
    // (positions a few thousand past a sequence's end are formed in 32 bits)
    VSK_REQUIRE(kv->pages <= (1 << 30), VSK_ERR_INVALID_BUFFER_SIZE, "at most 2^30 keys");
    VSK_REQUIRE(sets || (args->k_starts && is_device_ptr(args->k_starts)),
                VSK_ERR_INVALID_ARGUMENT, "dense keys need k_starts in device memory");
    VSK_REQUIRE(kv->k_row >= 0 && kv->v_row >= 0 && kv->k_row <= (1 << 26) &&
                    kv->v_row <= (1 << 26),
                VSK_ERR_INVALID_BUFFER_SIZE, "a row stride of more than 2^26 elements");
    VSK_REQUIRE(kv->k && kv->v && is_device_ptr(kv->k) && is_device_ptr(kv->v),
                VSK_ERR_INVALID_ARGUMENT, "keys and values must be device memory");
  }
  if (sets) {
    VSK_REQUIRE(!paged && args->window == 0 && args->sinks == 0, VSK_ERR_UNSUPPORTED,
                "cross attention is to dense keys, without a window");
    VSK_REQUIRE(sets->n >= 1 && sets->set_rows >= 0, VSK_ERR_INVALID_ARGUMENT,
                "no sets of keys");
    VSK_REQUIRE(news->seqs || news->n <= sets->n, VSK_ERR_INVALID_ARGUMENT,
                "more sequences than sets of keys");
    VSK_REQUIRE(optional_device(sets->starts) && optional_device(sets->lengths),
                VSK_ERR_INVALID_ARGUMENT, "offsets and lengths must be device memory");
  }
  if (shared) {
    VSK_REQUIRE(paged, VSK_ERR_UNSUPPORTED, "only pages are shared");
    VSK_REQUIRE(shared->n_groups >= 0 && shared->max_members >= 0 && shared->max_prefix >= 0,
                VSK_ERR_INVALID_ARGUMENT, "negative counts");
    VSK_REQUIRE(news->n <= shared->n, VSK_ERR_DIMENSION_MISMATCH,
                "more sequences than the prefixes are known of");
    VSK_REQUIRE(shared->n_groups == 0 ||
                    (shared->groups && shared->prefix && is_device_ptr(shared->groups) &&
                     is_device_ptr(shared->prefix)),
                VSK_ERR_INVALID_ARGUMENT, "groups and prefixes must be device memory");
  }
  VSK_REQUIRE(news->starts || news->tokens >= news->n, VSK_ERR_DIMENSION_MISMATCH,
              "fewer rows than sequences");
  VSK_REQUIRE(args->q.src && args->q.dst && is_device_ptr(args->q.src) &&
                  is_device_ptr(args->q.dst) && optional_device(args->lse),
              VSK_ERR_INVALID_ARGUMENT, "queries and outputs must be device memory");
  const Plans p = plans_of(ctx, kv, news, args, sets != nullptr, shared);
  VSK_REQUIRE(p.group_tokens * args->q.heads <= 0x3FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE,
              "too many query rows in one group");
  const int64_t need = workspace_of(p, kv, news, args);
  VSK_REQUIRE(need == 0 || (args->workspace && args->workspace_bytes >= need &&
                            aligned_to(args->workspace, 16) && is_device_ptr(args->workspace)),
              VSK_ERR_INVALID_BUFFER_SIZE,
              "the workspace must be " + std::to_string(need) + " bytes of device memory");
  const int64_t size = kv->dtype == VSK_DTYPE_F32 ? 4 : 2;
  AttnArgs a{};
  a.q = args->q.src;
  a.out = args->q.dst;
  a.lse = args->lse;
  a.q_row = args->q.src_row, a.q_head = args->q.src_head;
  a.o_row = args->q.dst_row, a.o_head = args->q.dst_head;
  a.k = static_cast<const char *>(kv->k) + (paged ? layer * kv->k_layer * size : 0);
  a.v = static_cast<const char *>(kv->v) + (paged ? layer * kv->v_layer * size : 0);
  a.k_row = kv->k_row, a.k_head = kv->k_head, a.v_row = kv->v_row, a.v_head = kv->v_head;
  a.starts = news->starts;
  a.seqs = news->seqs;
  if (paged) {
    a.k_page = kv->k_page, a.v_page = kv->v_page;
    a.table = kv->table, a.lengths = kv->lengths, a.table_stride = kv->table_stride;
    a.pages = kv->pages, a.slots = kv->slots, a.width = kv->width;
    a.page_shift = __builtin_ctz((unsigned)kv->page_size);
  } else if (sets) {
    a.cross = 1;
    a.k_starts = sets->starts, a.k_lengths = sets->lengths;
    a.sets = sets->n, a.set_rows = sets->set_rows;
    // Sequences that see one set read the same part of it at a time (14 over one
    // of 14,841 keys, 12 heads of 96 192 / 106 us); those with a set each would
    // read places of all that may lie in step (64 padded to 4,096, 16 heads of 64
    // 110 / 117).
    a.parts_apart = sets->n < news->n;
    a.k_rows = kv->pages;
  } else {
    a.k_starts = args->k_starts;
    a.k_rows = kv->pages;
  }
  a.tokens = news->tokens;
  a.n = news->n;
  a.heads = args->q.heads;
  a.kv_heads = kv->kv_heads;
  a.group = a.heads / a.kv_heads;
  a.d = kv->head_dim;
  a.window = args->window;
  a.sinks = args->sinks;
  a.max_new = (int32_t)most_new(news);
  a.scale_log2 = args->scale * 1.4426950408889634f;
  if (need) {
    a.part_o = static_cast<float *>(args->workspace);
    a.part_ml = a.part_o + (int64_t)p.parts() * a.tokens * a.heads * padded_head(a.d);
  }
  const bool al = aligned_operands(kv, args);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const AttnForm form = sets || p.group_tokens ? ATTN_FORMS : ATTN_OWN;
  auto launch = [&](const Plan &plan, AttnArgs x) {
    x.tiles = plan.tiles, x.splits = plan.splits, x.chunk = plan.chunk;
    if (plan.tile && kv->dtype == VSK_DTYPE_F32)
      launch_attn_tile32(ctx, st, x);
    else if (plan.tile)
      launch_attn_tile(ctx, st, x, kv->dtype, form);
    else if (form == ATTN_OWN)
      launch_attn_rows(ctx, st, x, kv->dtype, al, plan.share);
    else
      launch_attn_rows_forms(ctx, st, x, kv->dtype, al, plan.share);
  };
  if (p.group_tokens) {
    a.prefix = shared->prefix;
    a.joined = 1;
    a.parts_apart = 1;  // (pages lie anywhere: 12 groups of 16 92 / 88 us)
    a.part0 = p.prefix.splits;
    a.groups = shared->groups;
    a.members = a.n;
    a.pre.n = shared->n_groups, a.pre.max_new = (int32_t)p.group_tokens;
    a.pre.tiles = p.prefix.tiles, a.pre.splits = p.prefix.splits, a.pre.chunk = p.prefix.chunk;
    const int64_t blocks = (int64_t)a.pre.n * a.pre.splits * a.pre.tiles * a.kv_heads;
    VSK_REQUIRE(blocks <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE,
                "too many query rows in one call");
    // one launch for both where one kernel has both
    const bool mixed = p.prefix.tile && !p.own.tile && kv->dtype != VSK_DTYPE_F32 &&
                       kv->head_dim <= 128;
    if (mixed || p.prefix.tile == p.own.tile) {
      a.pre_blocks = (uint32_t)blocks;
    } else {
      AttnArgs g = a;
      g.part0 = 0;
      g.n = a.pre.n, g.max_new = a.pre.max_new;
      launch(p.prefix, g);
      a.groups = nullptr;
    }
    if (mixed) {
      a.tiles = p.own.tiles, a.splits = p.own.splits, a.chunk = p.own.chunk;
      launch_attn_shared(ctx, st, a, kv->dtype);
    } else {
      launch(p.own, a);
    }
  } else {
    launch(p.own, a);
  }
  a.splits = p.parts(), a.chunk = p.own.chunk;
  if (form == ATTN_OWN)
    launch_attn_join(ctx, st, a, kv->dtype, al, p.own.tile ? ATTN_TILE_ROWS : 16);
  else
    launch_attn_join_forms(ctx, st, a, kv->dtype, al, p.own.key_tile);
  finish_queued(ctx, st);
}

}  // namespace

}  // namespace vsk

using namespace vsk;

extern "C" {

int64_t vsk_attention_workspace(vsk_ctx *ctx, const vsk_kv *kv, const vsk_new_tokens *news,
                                const vsk_attention_args *args) {
  return workspace_call(ctx, kv, news, args, false, nullptr);
}

vsk_status vsk_attention(vsk_ctx *ctx, void *stream, const vsk_kv *kv, int32_t layer,
                         const vsk_new_tokens *news, const vsk_attention_args *args) {
  QUEUED_API_BEGIN(ctx);
  attend(ctx, stream, kv, layer, news, args, nullptr, nullptr);
  VSK_API_END(ctx);
}

int64_t vsk_cross_attention_workspace(vsk_ctx *ctx, const vsk_kv *kv, const vsk_new_tokens *news,
                                      const vsk_attention_args *args) {
  return workspace_call(ctx, kv, news, args, true, nullptr);
}

vsk_status vsk_cross_attention(vsk_ctx *ctx, void *stream, const vsk_kv *kv,
                               const vsk_new_tokens *news, const vsk_attention_args *args,
                               const vsk_key_sets *sets) {
  QUEUED_API_BEGIN(ctx);
  VSK_REQUIRE(sets, VSK_ERR_INVALID_ARGUMENT, "null argument");
  attend(ctx, stream, kv, 0, news, args, sets, nullptr);
  VSK_API_END(ctx);
}

int64_t vsk_attention_shared_workspace(vsk_ctx *ctx, const vsk_kv *kv, const vsk_new_tokens *news,
                                       const vsk_attention_args *args,
                                       const vsk_shared_prefix *shared) {
  return workspace_call(ctx, kv, news, args, false, shared);
}

vsk_status vsk_attention_shared(vsk_ctx *ctx, void *stream, const vsk_kv *kv, int32_t layer,
                                const vsk_new_tokens *news, const vsk_attention_args *args,
                                const vsk_shared_prefix *shared) {
  QUEUED_API_BEGIN(ctx);
  VSK_REQUIRE(shared, VSK_ERR_INVALID_ARGUMENT, "null argument");
  attend(ctx, stream, kv, layer, news, args, nullptr, shared);
  VSK_API_END(ctx);
}

}  // extern "C"
