// attn_rows.hip -- attention over 16 query rows a wave: one new token over a
// long cache, few new tokens, and 32-bit prompts.
//
// S^T = K Q^T and O^T = V^T P^T on the matrix cores, 16 rows (columns of the
// transposed products) at a time.  In the products' layout a lane owns one
// query row (lane % 16) and, of every 16 keys, the four 4 * (lane / 16) on:
// its scores, its running maximum and sum and its outputs belong to that row,
// so the softmax needs two exchanges a tile (the maximum) and the rescaling
// none.  The keys of a product may come in any order as long as both operands
// agree on it: P stays in the registers that S^T was computed in, and a lane
// loads V's rows for just those keys, 16 bytes of each, and turns the 8 x 8
// block of 16-bit values around with byte permutes.  K's fragments straight
// from memory would be 64 accesses of 16 bytes a load: whole rows go into LDS
// that belongs to the wave, and no wave waits for another before the join.
//
// One new token reads K and V once and does 4 * 16 * d operations a key for
// up to 16 heads: far under what the matrix cores do in the time the bytes
// take, so a group's heads ride along at no cost, and P goes in as a sum of
// two 16-bit values (its rounding would be as large as the output's).
//
// What bounds it: the bytes of K and V.  Measured, bf16 and f16, heads of 128:
// 64 contexts to 8,192, 32 heads on 8, 197 us, 5.0 TB/s; 3 to 200,003, 64 on 8,
// 202 us, 5.1 TB/s (a kernel that only reads: 5.8); one of 100,000, 8 on 1,
// 20 us, 2.5 TB/s: what a launch of few blocks and the join take; one of 777,
// 32 on 8, 11 us: one compute unit a key head, and its L1 passes 64 bytes a
// cycle, which is 1 us a round of eight waves and 32 keys; a wave waits for
// memory twice a step (walk).  f32, heads of 96 of their own, 17 contexts,
// window 2,048: 78 us, 4.9 TB/s.  Prompts in 32 bits are bound by the products
// (16x16x4, 157 TFLOP/s) and by keys and values that each wave brings for
// itself: 2 of 2,048, 32 heads of 128 on 8, 731 us, 94 TFLOP/s.  Operands
// without 16-byte alignment are loaded a value at a time: 32 contexts of 4,000,
// 10 f16 heads of 100, 595 us where heads of 104 take 125.
#include "attn_rows.hpp"
#include "vsk_api.hpp"

namespace vsk {

namespace {

// Joins the parts of one output row: sum of the parts' values and sums, each
// times exp(its reference less the largest, scaled).  A block a row, or a block for SL values
// of one; the threads take four values each of several parts at a time.  Its
// bytes are few: it is bound by the chain count, maximum, parts, each a trip to
// memory (5 us behind 64 parts of 192 rows of 128).
template <class T, int DV, int SL, int KTILE, int G, bool ALIGNED>
__global__ __launch_bounds__(256) void k_attn_join(const AttnArgs a, const int32_t RT) {
  constexpr int LANES = SL / 4, WAYS = 256 / LANES;
  __shared__ __attribute__((aligned(16))) float so[WAYS][SL];
  __shared__ float ss[WAYS];
  const uint32_t per = (uint32_t)a.max_new * a.heads;
  const uint32_t block = blockIdx.x / (DV / SL);
  const int e0 = blockIdx.x % (DV / SL) * SL;
  if (e0 >= a.d) return;
  const AttnSeq s = attn_seq<ATTN_OWN>(a, block / per);
  const int32_t x = block % per, t = x / a.heads, head = x % a.heads;
  if (t >= s.T) return;
  const int64_t stride = a.tokens * a.heads;
  const int64_t at = (s.token0 + t) * a.heads + head;
  // the first parts are asked for before it is known how many there are
  const int e = e0 + 4 * (threadIdx.x % LANES), way = threadIdx.x / LANES;
  const int32_t i0 = threadIdx.x & 63;
  const int32_t w0 = way < a.splits ? way : 0;
  const int32_t l0 = i0 < a.splits ? i0 : 0;
  const float m0 = a.part_ml[2 * (l0 * stride + at)];
  const int64_t r0 = w0 * stride + at;
  const float fm0 = a.part_ml[2 * r0], fl0 = a.part_ml[2 * r0 + 1];
  const f32x4 o0 = *reinterpret_cast<const f32x4 *>(a.part_o + r0 * DV + (e < a.d ? e : 0));
  // the parts of the row tile that computed this row
  const int32_t h = head / a.group, row = t * a.group + head - h * a.group;
  const int32_t row0 = row / RT * RT;
  const int32_t all = (s.T < a.max_new ? s.T : a.max_new) * a.group;
  const int32_t last = row0 + RT < all ? row0 + RT - 1 : all - 1;
  const int32_t p0 = s.L - s.T;
  const auto span = attn_span<KTILE, G>(a, p0 + row0 / a.group, p0 + last / a.group);
  const int32_t parts = attn_parts(a, span.tiles);
  if (parts == 1) return;  // written by the row tile itself
  float top = i0 < parts ? m0 : -INFINITY;
  for (int32_t i = i0 + 64; i < parts; i += 64)
    top = fmaxf(top, a.part_ml[2 * (i * stride + at)]);
  for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  top = xor16_32_max(top);
  const float use = top == -INFINITY ? 0.f : top;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
  if (way < parts) {
    const float f = attn_exp2((fm0 - use) * a.scale_log2);
    sum = f * fl0;
    o = f * o0;
  }
#pragma unroll 4
  for (int32_t i = way + WAYS; i < parts; i += WAYS) {
    const int64_t r = i * stride + at;
    const float f = attn_exp2((a.part_ml[2 * r] - use) * a.scale_log2);
    sum += f * a.part_ml[2 * r + 1];
    if (e < a.d) o += f * *reinterpret_cast<const f32x4 *>(a.part_o + r * DV + e);
  }
  *reinterpret_cast<f32x4 *>(&so[way][e - e0]) = o;
  if (threadIdx.x % LANES == 0) ss[way] = sum;
  __syncthreads();
  if (way) return;
#pragma unroll 8
  for (int i = 1; i < WAYS; ++i) {
    o += *reinterpret_cast<f32x4 *>(&so[i][e - e0]);
    sum += ss[i];
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  if (e == 0 && a.lse) a.lse[at] = attn_lse(top * a.scale_log2, sum);
  if (e >= a.d) return;
  T *dst = static_cast<T *>(a.out) + (s.token0 + t) * a.o_row + head * a.o_head + e;
  const float z[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  if constexpr (ALIGNED)
    store4<T>(dst, z, a.d - e);
  else
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (e + i < a.d) dst[i] = (T)z[i];
}

template <class T, int VW, int NB, int SHARE, bool ALIGNED>
__global__ __launch_bounds__(rows_threads(SHARE), rows_waves<T>(SHARE, VW * NB)) void
k_attn_rows(const AttnArgs a) {
  __shared__ __attribute__((aligned(1024))) char pool[RowsLds<T, VW, NB, SHARE, ALIGNED>::BYTES];
  attn_rows_block<T, VW, NB, SHARE, ALIGNED, ATTN_OWN>(a, blockIdx.x, pool);
}

template <class T, int VW, int NB>
void rows_of(hipStream_t st, const AttnArgs &a, bool aligned, int32_t share, unsigned grid) {
  if (share == 8) {
    if constexpr (16 * VW * NB <= (sizeof(T) == 4 ? 64 : 128)) {
      if (aligned)
        k_attn_rows<T, VW, NB, 8, true><<<grid, 512, 0, st>>>(a);
      else
        k_attn_rows<T, VW, NB, 8, false><<<grid, 512, 0, st>>>(a);
    }
  } else if (share == 4) {
    if (aligned)
      k_attn_rows<T, VW, NB, 4, true><<<grid, 256, 0, st>>>(a);
    else
      k_attn_rows<T, VW, NB, 4, false><<<grid, 256, 0, st>>>(a);
  } else {
    if (aligned)
      k_attn_rows<T, VW, NB, 1, true><<<grid, 256, 0, st>>>(a);
    else
      k_attn_rows<T, VW, NB, 1, false><<<grid, 256, 0, st>>>(a);
  }
}

}  // namespace

void launch_attn_rows(vsk_ctx *ctx, hipStream_t st, const AttnArgs &a, int32_t t, bool aligned,
                      int32_t share) {
  const int64_t groups = share > 1 ? a.tiles : (a.tiles + 3) / 4;
  const int64_t grid = (int64_t)a.n * a.splits * groups * a.kv_heads;
  VSK_REQUIRE(grid <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "too many query rows in one call");
  const unsigned g = (unsigned)grid;
  KernelTimer kt(ctx, "attn_rows", (double)a.tokens * a.heads, st);
  if (t == VSK_DTYPE_F32) {
    if (a.d <= 64)
      rows_of<float, 4, 1>(st, a, aligned, share, g);
    else if (a.d <= 128)
      rows_of<float, 4, 2>(st, a, aligned, share, g);
    else
      rows_of<float, 4, 4>(st, a, aligned, share, g);
  } else if (t == VSK_DTYPE_F16) {
    if (a.d <= 64)
      rows_of<_Float16, 4, 1>(st, a, aligned, share, g);
    else if (a.d <= 128)
      rows_of<_Float16, 8, 1>(st, a, aligned, share, g);
    else
      rows_of<_Float16, 8, 2>(st, a, aligned, share, g);
  } else {
    if (a.d <= 64)
      rows_of<__bf16, 4, 1>(st, a, aligned, share, g);
    else if (a.d <= 128)
      rows_of<__bf16, 8, 1>(st, a, aligned, share, g);
    else
      rows_of<__bf16, 8, 2>(st, a, aligned, share, g);
  }
  check_launch("attn_rows");
}

namespace {
template <class T, int DV, int SL>
void join_slice(hipStream_t st, const AttnArgs &a, bool aligned, int32_t rows, unsigned g) {
  constexpr int KR = 16 * SUBS<T>, KB = attn_tile_keys(DV);
  if (rows == ROWS) {
    if (aligned)
      k_attn_join<T, DV, SL, KR, KR, true><<<g, 256, 0, st>>>(a, rows);
    else
      k_attn_join<T, DV, SL, KR, KR, false><<<g, 256, 0, st>>>(a, rows);
  } else if constexpr (sizeof(T) == 2) {  // (tiles are for 16-bit, aligned operands)
    k_attn_join<T, DV, SL, KB, ATTN_TILE_GROUP, true><<<g, 256, 0, st>>>(a, rows);
  }
}
template <class T, int DV>
void join_head(hipStream_t st, const AttnArgs &a, bool aligned, int32_t rows, uint64_t g,
               uint64_t cus) {
  // slices of 16 values where all of them find a compute unit each: one context
  // of 100,000 under 8 heads of 128 on one takes 30 us, 67 without them; 4 of
  // 30,000 under 32 on 8 would take 58 and take 51.  Up to a row a compute unit,
  // slices of 64: 4 f32 contexts to 30,000, 8 heads of 256 on one, 44 us, 49
  // without them; 3 f16 to 200,003, 64 of 128 on 8, 209 / 212.
  if (g * (DV / 16) <= cus)
    join_slice<T, DV, 16>(st, a, aligned, rows, g * (DV / 16));
  else if (DV > 64 && g <= cus)
    join_slice<T, DV, 64>(st, a, aligned, rows, g * (DV / 64));
  else
    join_slice<T, DV, DV>(st, a, aligned, rows, g);
}
template <class T>
void join_of(hipStream_t st, const AttnArgs &a, bool aligned, int32_t rows, uint64_t g,
             uint64_t cus) {
  if (a.d <= 64)
    join_head<T, 64>(st, a, aligned, rows, g, cus);
  else if (a.d <= 128)
    join_head<T, 128>(st, a, aligned, rows, g, cus);
  else
    join_head<T, 256>(st, a, aligned, rows, g, cus);
}
}  // namespace

void launch_attn_join(vsk_ctx *ctx, hipStream_t st, const AttnArgs &a, int32_t t, bool aligned,
                      int32_t rows) {
  if (a.splits == 1) return;
  const int64_t grid = (int64_t)a.n * a.max_new * a.heads;
  VSK_REQUIRE(grid <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "too many query rows in one call");
  KernelTimer kt(ctx, "attn_join", (double)grid, st);
  if (t == VSK_DTYPE_F32)
    join_of<float>(st, a, aligned, rows, grid, ctx->cu_count);
  else if (t == VSK_DTYPE_F16)
    join_of<_Float16>(st, a, aligned, rows, grid, ctx->cu_count);
  else
    join_of<__bf16>(st, a, aligned, rows, grid, ctx->cu_count);
  check_launch("attn_join");
}

}  // namespace vsk
