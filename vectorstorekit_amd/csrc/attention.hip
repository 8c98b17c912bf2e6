// attention.hip -- the attention entry points: checks, the division of the
// work, and the choice of kernel.
#include <cmath>

#include "attn.hpp"
#include "vsk_api.hpp"

namespace vsk {

namespace {

int32_t padded_head(int32_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// How a call's work is divided.
struct Plan {
  int32_t tiles, splits, chunk;
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

Plan plan_of(const vsk_ctx *ctx, const vsk_kv *kv, const vsk_new_tokens *news,
             const vsk_attention_args *args) {
  Plan p;
  const int64_t group = args->q.heads / kv->kv_heads;
  const int64_t max_new = news->starts ? news->max_new : 1;
  const int64_t rows = max_new * group, pairs = (int64_t)news->n * kv->kv_heads;
  p.splits = 1;
  p.chunk = 1 << 30;
  p.tile = false;
  p.share = 4;
  const int64_t cus = ctx->cu_count;
  int64_t row_tile = 16, key_tile = kv->dtype == VSK_DTYPE_F32 ? 16 : 32;
  int64_t keys = kv->table ? (int64_t)kv->width * kv->page_size : kv->pages;
  if (args->max_length > 0 && args->max_length < keys) keys = args->max_length;
  // Row tiles of 128 where there are rows to fill them and work for the
  // device.  Under 64 rows of a key head most of a tile would be empty; with
  // few rows in all, and few products, tiles of 16 spread over more waves and
  // end sooner; fewer still where keys are many, whose parts keep the device
  // busy either way.  Measured in 16 bits, tiles of 128 against tiles of 16
  // (us): one prompt of 2,000 tokens, 8 heads of 64 47 / 27, of 4,000 60 / 122;
  // 4 heads of 128 on one 41 / 27; of 333, 32 heads of 128 on 8, 16 / 22; 64
  // new tokens of 8 heads of 64 after 4,000 keys 23 / 15, after 30,000 25 / 33;
  // of one head after 30,000 24 / 16.
  int64_t seen = keys - (max_new < keys ? max_new : keys) / 2;
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
  p.tiles = (int32_t)ceil_div(rows, row_tile);
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
    if (p.tiles >= 4 && (blocks >= 16 * cus || (blocks >= 4 * cus && keys <= 384) ||
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
    if (many && tiles <= (blocks < cus ? 32 : 64)) {
      p.share = 8;
      return p;
    }
  }
  // Parts as many as keep the device supplied with blocks.
  int64_t want, per;
  if (p.tile) {
    // A prompt's rows are many and joining them takes as long as some steps:
    // parts of at least 16 tiles, and only where a quarter of the blocks that
    // fit or less would work.  Unsplit / split after 30,000 keys, 32 heads of
    // 128 on 8 (us): 512 tokens (128 blocks) 519 / 284, 2,000 (504) 893 / 998.
    per = 16;
    want = 2 * blocks > cus ? 1 : 2 * cus;
  } else {
    // A tile for each of the four waves that share a part at least.  Contexts
    // differ in length, so several rounds of blocks share the work more evenly
    // than one; each starts and is joined, so the fewer the longer a block is
    // by its head.  Measured, blocks a compute unit / us: 64 contexts to 8,192
    // of 8 key heads of 128 2 / 228, 6 / 195, 12 / 197; 200 to 4,000 of 8 heads
    // of 64 8 / 192, 16 / 164, 24 / 203; 17 of 16 f32 heads of 96, window
    // 2,048, 2 / 76, 6 / 86; 60 to 2,000 of 2 heads of 256 1 / 38, 4 / 47.  No
    // more than 64 parts a row, while there is a block for every compute unit:
    // 2 contexts of 100,000 of 8 heads of 128 121 us, in 96 parts 129.
    per = 4;
    const int64_t most = kv->head_dim <= 64 ? 16 : kv->head_dim > 128 ? 1
                         : kv->dtype == VSK_DTYPE_F32 ? 2 : 6;
    want = most * cus < 64 * blocks ? most * cus : 64 * blocks;
    if (want < cus) want = cus;
  }
  const int64_t chunk = ceil_div(ceil_div(tiles, ceil_div(want, blocks)), per) * per;
  p.chunk = (int32_t)(chunk < per ? per : chunk);
  p.splits = (int32_t)ceil_div(tiles, p.chunk);
  if (p.splits < 1) p.splits = 1;
  return p;
}

int64_t workspace_of(const Plan &p, const vsk_kv *kv, const vsk_new_tokens *news,
                     const vsk_attention_args *args) {
  if (p.splits == 1) return 0;
  return (int64_t)sizeof(float) * p.splits * news->tokens * args->q.heads *
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

}  // namespace

}  // namespace vsk

using namespace vsk;

extern "C" {

int64_t vsk_attention_workspace(vsk_ctx *ctx, const vsk_kv *kv, const vsk_new_tokens *news,
                                const vsk_attention_args *args) {
  if (!ctx) return 0;
  try {
    check_shapes(kv, news, args);
  } catch (...) {
    return 0;  // (vsk_attention says why)
  }
  // (no rows: nothing to divide)
  if (news->n == 0 || news->tokens == 0 || news->max_new == 0) return 0;
  return workspace_of(plan_of(ctx, kv, news, args), kv, news, args);
}

vsk_status vsk_attention(vsk_ctx *ctx, void *stream, const vsk_kv *kv, int32_t layer,
                         const vsk_new_tokens *news, const vsk_attention_args *args) {
  QUEUED_API_BEGIN(ctx);
  check_shapes(kv, news, args);
  VSK_REQUIRE(std::isfinite(args->scale) && args->scale > 0, VSK_ERR_INVALID_ARGUMENT,
              "scale must be positive and finite");
  check_news(news);
  if (news->n == 0 || news->tokens == 0 || news->max_new == 0) return VSK_OK;
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
    VSK_REQUIRE(args->k_starts && is_device_ptr(args->k_starts), VSK_ERR_INVALID_ARGUMENT,
                "dense keys need k_starts in device memory");
    VSK_REQUIRE(kv->k_row >= 0 && kv->v_row >= 0 && kv->k_row <= (1 << 26) &&
                    kv->v_row <= (1 << 26),
                VSK_ERR_INVALID_BUFFER_SIZE, "a row stride of more than 2^26 elements");
    VSK_REQUIRE(kv->k && kv->v && is_device_ptr(kv->k) && is_device_ptr(kv->v),
                VSK_ERR_INVALID_ARGUMENT, "keys and values must be device memory");
  }
  VSK_REQUIRE(news->starts || news->tokens >= news->n, VSK_ERR_DIMENSION_MISMATCH,
              "fewer rows than sequences");
  VSK_REQUIRE(args->q.src && args->q.dst && is_device_ptr(args->q.src) &&
                  is_device_ptr(args->q.dst) && (!args->lse || is_device_ptr(args->lse)),
              VSK_ERR_INVALID_ARGUMENT, "queries and outputs must be device memory");
  const Plan p = plan_of(ctx, kv, news, args);
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
  a.max_new = news->starts ? news->max_new : 1;
  a.tiles = p.tiles, a.splits = p.splits, a.chunk = p.chunk;
  a.scale_log2 = args->scale * 1.4426950408889634f;
  if (need) {
    a.part_o = static_cast<float *>(args->workspace);
    a.part_ml = a.part_o + (int64_t)p.splits * a.tokens * a.heads * padded_head(a.d);
  }
  const bool al = aligned_operands(kv, args);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p.tile)
    launch_attn_tile(ctx, st, a, kv->dtype);
  else
    launch_attn_rows(ctx, st, a, kv->dtype, al, p.share);
  launch_attn_join(ctx, st, a, kv->dtype, al, p.tile ? ATTN_TILE_ROWS : 16);
  finish_queued(ctx, st);
  VSK_API_END(ctx);
}

}  // extern "C"
