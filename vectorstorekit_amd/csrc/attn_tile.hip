// attn_tile.hip -- attention of many query rows in 16 bits: 32 rows a wave,
// four waves a workgroup, keys and values shared through LDS.
//
// S^T = K Q^T and O^T = V^T P^T with 32x32x16 products.  As in
// attn_rows.hip a lane owns one query row (lane % 32) and half of the keys of
// a tile, P stays in the registers that S^T was computed in, and the softmax
// exchanges one value a tile with lane ^ 32.  V's columns come out of LDS
// through the transposing read, which hands a lane four keys of one dimension.
//
// Rows of K and V arrive by direct loads into LDS, which write 16 bytes a lane
// in lane order: a row's 16-byte pieces are permuted on the way (each lane
// fetches the piece that belongs in its slot), so that the reads of K (32 rows
// of one piece) and of V (4 rows of 32 bytes) meet every bank once.
//
// A tile's keys are four groups (of a head over 128 two) of 16 that lie
// together: the few first keys that a window leaves visible share a tile with
// the first that it shows.
//
// The weights are rounded to the type of V before the second product, with an
// error of the size of the output's own rounding; sums stay in fp32.
//
// What bounds it: the products, 4 d operations a visible key and row (half of
// them each product), and beside them the exponentials, one a score, on the
// vector unit.  Measured, bf16, 32 heads of 128 on 8: 16,384 tokens, window
// 4,096, 910 to 1,020 us by the card (and its power limit), 945 to 1,060 TFLOP/s
// of visible work, 1,270 in the loop over whole tiles (a library product of
// 16,384 cubed: 1,360); 8 ragged prompts to 4,096, window 1,024, 294 to 310 us,
// 715 to 750 TFLOP/s: 17.3 tiles a block where 16 hold what is seen, three of
// them partly masked and outside the pipelined loop, and a block's start and
// end.  4 prompts of 4,096, 8 heads of 256 on one: 363 us, 758 TFLOP/s (one
// block a compute unit, queries in LDS).  One of 4,000, 8 heads of 64: 60 us,
// 273 TFLOP/s: 16 products a step beside 138 vector instructions, which bound it.
#include "attn_tile.hpp"
#include "vsk_api.hpp"

namespace vsk {

namespace {

template <class T, int DP, AttnForm F>
__global__ __launch_bounds__(64 * TILE_WAVES, DP == 256 ? 1 : 2) void k_attn_tile(
    const AttnArgs args) {
  typedef TileLds<DP> Lds;
  __shared__ __attribute__((aligned(1024))) char keys[3 * Lds::TILEB];
  __shared__ __attribute__((aligned(1024))) char values[2 * Lds::TILEB];
  __shared__ __attribute__((aligned(1024))) char queries[Lds::QUERYB];
  if constexpr (F == ATTN_OWN) {
    attn_tile_block<T, DP, F>(args, blockIdx.x, keys, values, queries);
  } else {
    AttnArgs a = args;
    const uint32_t block = attn_call(a, blockIdx.x);
    attn_tile_block<T, DP, F>(a, block, keys, values, queries);
  }
}

template <class T, AttnForm F> void tile_of(hipStream_t st, const AttnArgs &a, unsigned g) {
  if (a.d <= 64)
    k_attn_tile<T, 64, F><<<g, 64 * TILE_WAVES, 0, st>>>(a);
  else if (a.d <= 96)
    k_attn_tile<T, 96, F><<<g, 64 * TILE_WAVES, 0, st>>>(a);
  else if (a.d <= 128)
    k_attn_tile<T, 128, F><<<g, 64 * TILE_WAVES, 0, st>>>(a);
  else
    k_attn_tile<T, 256, F><<<g, 64 * TILE_WAVES, 0, st>>>(a);
}

}  // namespace

void launch_attn_tile(vsk_ctx *ctx, hipStream_t st, const AttnArgs &a, int32_t t, AttnForm form) {
  const int64_t grid = a.pre_blocks + (int64_t)a.n * a.splits * a.tiles * a.kv_heads;
  VSK_REQUIRE(grid <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "too many query rows in one call");
  KernelTimer kt(ctx, "attn_tile", (double)a.tokens * a.heads, st);
  const unsigned g = (unsigned)grid;
  if (form == ATTN_OWN)
    t == VSK_DTYPE_F16 ? tile_of<_Float16, ATTN_OWN>(st, a, g) : tile_of<__bf16, ATTN_OWN>(st, a, g);
  else
    t == VSK_DTYPE_F16 ? tile_of<_Float16, ATTN_FORMS>(st, a, g)
                       : tile_of<__bf16, ATTN_FORMS>(st, a, g);
  check_launch("attn_tile");
}

}  // namespace vsk
