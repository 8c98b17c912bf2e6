// attn_forms.hip -- the kernels of attn_rows.hip for the other forms of
// attention: to keys of another length that every row sees, and over a prefix
// that sequences share, where a row tile holds rows of several.
//
// What bounds them: the bytes of K and V, as in attn_rows.hip (64 contexts to
// 4,096 of 16 heads of 64, four tokens each, 110 us: 4.4 TB/s, of which the join
// is 5), short ones the launches (one token over 300 keys 9 us; 4 branches of
// 512 shared keys 12, a launch for both calls and one for the join).  In 32 bits
// heads over 64 leave registers for two waves a SIMD, whose products and vector
// instructions, on one unit, take half of the time (6 groups of ten branches and
// up to nine drafts, 16 heads of 96: 109 us for 232 MB).
#include "attn_rows.hpp"
#include "vsk_api.hpp"

namespace vsk {

namespace {

template <class T, int VW, int NB, int SHARE, bool ALIGNED>
__global__ __launch_bounds__(rows_threads(SHARE), rows_waves<T>(SHARE, VW * NB)) void
k_attn_forms(const AttnArgs args) {
  __shared__ __attribute__((aligned(1024))) char pool[RowsLds<T, VW, NB, SHARE, ALIGNED>::BYTES];
  AttnArgs a = args;
  const uint32_t block = attn_call(a, blockIdx.x);
  attn_rows_block<T, VW, NB, SHARE, ALIGNED, ATTN_FORMS>(a, block, pool);
}

// Joins the parts of output rows: a row for DV / 4 lanes, times WAYS that share
// its parts.  Unlike k_attn_join it has the rows of one sequence side by side
// (a block a row took 95 us for 70,000 rows of three parts, this 22).
template <class E, int DV, int WAYS, bool ALIGNED>
__global__ __launch_bounds__(256) void k_attn_join_forms(const AttnArgs a, const int32_t key_tile) {
  constexpr int LANES = DV / 4, WIDE = LANES * WAYS, R = 256 / WIDE;
  __shared__ __attribute__((aligned(16))) float so[WAYS > 1 ? 256 * 4 : 4];
  __shared__ float ss[WAYS > 1 ? 256 / LANES : 1];
  const int32_t per = (int32_t)(((int64_t)a.max_new * a.heads + R - 1) / R);
  const int32_t b = blockIdx.x / per;
  const int32_t x = (int32_t)(blockIdx.x % per) * R + threadIdx.x / WIDE;
  const int32_t t = x / a.heads, head = x - t * a.heads;
  int32_t parts = a.splits, from = 0;
  int64_t token0 = b;
  int32_t T = 1;
  if (a.joined) {
    // the prefix's parts, where the sequence has one, and its own
    from = a.prefix[b] >> a.page_shift > 0 ? 0 : a.part0;
    if (a.starts) {
      int32_t t0 = a.starts[b], t1 = a.starts[b + 1];
      t0 = t0 < 0 ? 0 : t0;
      if (t1 > a.tokens) t1 = (int32_t)a.tokens;
      token0 = t0, T = t1 - t0;
    }
  } else {
    const AttnSeq s = attn_seq<ATTN_FORMS>(a, b);
    token0 = s.token0, T = s.T;
    parts = attn_parts(a, (s.L + key_tile - 1) / key_tile);
    if (parts == 1) return;  // written by the row tile itself
  }
  const bool real = t < T && t < a.max_new;
  if (WAYS == 1 && !real) return;
  const int64_t stride = a.tokens * a.heads;
  const int64_t at = real ? (token0 + t) * a.heads + head : 0;
  const int lane = threadIdx.x % LANES, way = threadIdx.x / LANES % WAYS;
  const int e = 4 * lane < a.d ? 4 * lane : 0;
  // a part's reference, its largest, and (4 parts in flight) its sums
  float top = -INFINITY;
  for (int32_t i = from + lane; i < parts; i += LANES)
    top = fmaxf(top, a.part_ml[2 * (i * stride + at)]);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float use = top == -INFINITY ? 0.f : top;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll 4
  for (int32_t i = from + way; i < parts; i += WAYS) {
    const int64_t r = i * stride + at;
    const float ref = a.part_ml[2 * r], l = a.part_ml[2 * r + 1];
    const f32x4 y = *reinterpret_cast<const f32x4 *>(a.part_o + r * DV + e);
    const float f = attn_exp2((ref - use) * a.scale_log2);
    // (a part that is not there, or of no keys, holds no values; one whose scores
    // are all NaN has no largest either, and its sum is NaN)
    const bool none = ref == -INFINITY && l == 0.f;
    sum += none ? 0.f : f * l;
#pragma unroll
    for (int z = 0; z < 4; ++z) o[z] += none ? 0.f : f * y[z];
  }
  if constexpr (WAYS > 1) {
    *reinterpret_cast<f32x4 *>(&so[4 * threadIdx.x]) = o;
    if (lane == 0) ss[threadIdx.x / LANES] = sum;
    __syncthreads();
    if (way || !real) return;
#pragma unroll
    for (int i = 1; i < WAYS; ++i) {
      o += *reinterpret_cast<f32x4 *>(&so[4 * (threadIdx.x + i * LANES)]);
      sum += ss[threadIdx.x / LANES + i];
    }
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  if (lane == 0 && a.lse) a.lse[at] = attn_lse(top * a.scale_log2, sum);
  if (4 * lane >= a.d) return;
  E *dst = static_cast<E *>(a.out) + (token0 + t) * a.o_row + head * a.o_head + e;
  const float z[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  if constexpr (ALIGNED)
    store4<E>(dst, z, a.d - e);
  else
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (e + i < a.d) dst[i] = (E)z[i];
}

template <class T, int VW, int NB>
void rows_of(hipStream_t st, const AttnArgs &a, bool aligned, int32_t share, unsigned grid) {
  if (share == 8) {
    if constexpr (16 * VW * NB <= (sizeof(T) == 4 ? 64 : 128)) {
      if (aligned)
        k_attn_forms<T, VW, NB, 8, true><<<grid, 512, 0, st>>>(a);
      else
        k_attn_forms<T, VW, NB, 8, false><<<grid, 512, 0, st>>>(a);
    }
  } else if (share == 4) {
    if (aligned)
      k_attn_forms<T, VW, NB, 4, true><<<grid, 256, 0, st>>>(a);
    else
      k_attn_forms<T, VW, NB, 4, false><<<grid, 256, 0, st>>>(a);
  } else {
    if (aligned)
      k_attn_forms<T, VW, NB, 1, true><<<grid, 256, 0, st>>>(a);
    else
      k_attn_forms<T, VW, NB, 1, false><<<grid, 256, 0, st>>>(a);
  }
}

}  // namespace

void launch_attn_rows_forms(vsk_ctx *ctx, hipStream_t st, const AttnArgs &a, int32_t t,
                            bool aligned, int32_t share) {
  const int64_t groups = share > 1 ? a.tiles : (a.tiles + 3) / 4;
  const int64_t grid = a.pre_blocks + (int64_t)a.n * a.splits * groups * a.kv_heads;
  VSK_REQUIRE(grid <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "too many query rows in one call");
  const unsigned g = (unsigned)grid;
  KernelTimer kt(ctx, "attn_forms", (double)a.tokens * a.heads, st);
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
  check_launch("attn_forms");
}

namespace {

template <class E, int DV, int WAYS>
void join_ways(hipStream_t st, const AttnArgs &a, bool aligned, int32_t key_tile) {
  constexpr int R = 256 / (DV / 4 * WAYS);
  const int64_t grid = (int64_t)a.n * ceil_div((int64_t)a.max_new * a.heads, R);
  VSK_REQUIRE(grid <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "too many query rows in one call");
  if (aligned)
    k_attn_join_forms<E, DV, WAYS, true><<<(unsigned)grid, 256, 0, st>>>(a, key_tile);
  else
    k_attn_join_forms<E, DV, WAYS, false><<<(unsigned)grid, 256, 0, st>>>(a, key_tile);
}

template <class E, int DV>
void join_head(hipStream_t st, const AttnArgs &a, bool aligned, int32_t key_tile, int64_t cus) {
  // few rows: a block a row; many: as few ways as keep some parts in flight
  const int64_t rows = (int64_t)a.n * a.max_new * a.heads;
  if (rows < 8 * cus)
    join_ways<E, DV, 1024 / DV>(st, a, aligned, key_tile);
  else if (a.splits > 8)
    join_ways<E, DV, 4>(st, a, aligned, key_tile);
  else
    join_ways<E, DV, 1>(st, a, aligned, key_tile);
}

template <class E>
void join_of(hipStream_t st, const AttnArgs &a, bool aligned, int32_t key_tile, int64_t cus) {
  if (a.d <= 64)
    join_head<E, 64>(st, a, aligned, key_tile, cus);
  else if (a.d <= 128)
    join_head<E, 128>(st, a, aligned, key_tile, cus);
  else
    join_head<E, 256>(st, a, aligned, key_tile, cus);
}

}  // namespace

void launch_attn_join_forms(vsk_ctx *ctx, hipStream_t st, const AttnArgs &a, int32_t t,
                            bool aligned, int32_t key_tile) {
  if (a.splits == 1) return;
  KernelTimer kt(ctx, "attn_join", (double)a.n * a.max_new * a.heads, st);
  if (t == VSK_DTYPE_F32)
    join_of<float>(st, a, aligned, key_tile, ctx->cu_count);
  else if (t == VSK_DTYPE_F16)
    join_of<_Float16>(st, a, aligned, key_tile, ctx->cu_count);
  else
    join_of<__bf16>(st, a, aligned, key_tile, ctx->cu_count);
  check_launch("attn_join");
}

}  // namespace vsk
