// attn_shared.hip -- attention over shared prefixes in one launch: row tiles of
// 128 over the prefixes (attn_tile.hpp), whose bound is the products, and
// beside them row tiles of 16 over each sequence's own keys (attn_rows.hpp),
// whose bound is their bytes.  64 branches of 32,768 shared keys and up to 512
// of their own, 32 heads of 128 on 8: 64 us and 6 for the join, where the
// products alone are 25 at a large library product's rate and the bytes 38 (one
// call after the other took 93).
#include "attn_rows.hpp"
#include "attn_tile.hpp"
#include "vsk_api.hpp"

namespace vsk {

namespace {

template <class T, int DP, int VW, int NB>
__global__ __launch_bounds__(64 * TILE_WAVES, 2) void k_attn_shared(
    const AttnArgs args) {
  typedef TileLds<DP> Lds;
  typedef RowsLds<T, VW, NB, 4, true> Rows;
  constexpr int TILES = 5 * Lds::TILEB;
  __shared__ __attribute__((aligned(1024))) char pool[TILES > Rows::BYTES ? TILES : Rows::BYTES];
  // Eight blocks (one an XCD) of the one, eight of the other, in turn, and the
  // other way round from 32 such on, so that a compute unit (an XCD has 32, which
  // get their second block when each has its first) has one of each.
  const uint32_t pre = (args.pre_blocks + 7) / 8, own = (args.own_blocks + 7) / 8;
  const uint32_t both = pre < own ? pre : own, g = blockIdx.x / 8;
  const bool paired = g < 2 * both;
  const bool prefix = paired ? (g ^ g >> 5) & 1 : pre > own;
  const uint32_t block = 8 * (paired ? g / 2 : g - both) + blockIdx.x % 8;
  if (block >= (prefix ? args.pre_blocks : args.own_blocks)) return;
  // (each with a copy of its own: one that both changed would hold its values
  // in scalars that neither has left)
  if (prefix) {
    AttnArgs a = args;
    attn_prefix_call(a);
    attn_tile_block<T, DP, ATTN_FORMS>(a, block, pool, pool + 3 * Lds::TILEB, pool);
  } else {
    AttnArgs a = args;
    a.groups = nullptr;
    attn_rows_block<T, VW, NB, 4, true, ATTN_FORMS>(a, block, pool);
  }
}

template <class T> void shared_of(hipStream_t st, const AttnArgs &a, unsigned g) {
  if (a.d <= 64)
    k_attn_shared<T, 64, 4, 1><<<g, 64 * TILE_WAVES, 0, st>>>(a);
  else if (a.d <= 96)
    k_attn_shared<T, 96, 8, 1><<<g, 64 * TILE_WAVES, 0, st>>>(a);
  else
    k_attn_shared<T, 128, 8, 1><<<g, 64 * TILE_WAVES, 0, st>>>(a);
}

}  // namespace

void launch_attn_shared(vsk_ctx *ctx, hipStream_t st, AttnArgs a, int32_t t) {
  const int64_t own = (int64_t)a.n * a.splits * a.tiles * a.kv_heads;
  const int64_t grid = 8 * (ceil_div(a.pre_blocks, 8) + ceil_div(own, 8));
  a.own_blocks = (uint32_t)own;
  VSK_REQUIRE(grid <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "too many query rows in one call");
  KernelTimer kt(ctx, "attn_shared", (double)a.tokens * a.heads, st);
  if (t == VSK_DTYPE_F16)
    shared_of<_Float16>(st, a, (unsigned)grid);
  else
    shared_of<__bf16>(st, a, (unsigned)grid);
  check_launch("attn_shared");
}

}  // namespace vsk
