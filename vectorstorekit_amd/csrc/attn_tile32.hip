// attn_tile32.hip -- attention of many query rows in 32 bits, of the forms
// whose rows all see (nearly) the same keys: to keys of another length, and
// over prefixes.  32 rows a wave, four waves a workgroup, keys and values
// shared through LDS.
//
// S^T = K Q^T and O^T = V^T P^T with 32x32x2 products.  A lane owns one query
// row (lane % 32); register 4 q + i of the scores is key 8 q + 4 (lane / 32) + i
// of the 32 of a tile, and the second product takes the keys in just those
// pairs, so P stays where it was computed.  The inner order of the first is
// free as well: a lane reads 16 bytes of a key, four places for four products.
// Of a row of V a lane reads DT places that follow each other, one for each of
// the DT products of 32 dimensions: dimension DT r + t of the head is row r of
// product t.
//
// What bounds it: the products, 64 cycles each, and the vector instructions
// beside them, which run on the same units in 32 bits and add to them: a tile
// has 32 DT products or less (of the head's d, not the padding), and some 200
// other instructions (2.3 a product counted).  So the sums are rescaled only when
// a row's largest score has grown by 8 (in log2; weights up to 256 cost fp32
// nothing), and values looked at one by one only in tiles that not every row sees
// whole.  7 texts of up to 500 against three sets of up to 3,001 keys, 20 heads of 80 on 5: 482 us (16
// rows a wave that brings its keys itself: 1,000), 79 of 157 TFLOP/s, 86 with the
// places that the head leaves in a block of 32; the matrix cores are busy 0.62 of
// the time.
#include "attn.hpp"
#include "vsk_api.hpp"

namespace vsk {

namespace {

constexpr int NW = 4;
constexpr int KT = 32;

typedef __attribute__((ext_vector_type(4))) float f4;

// DT: dimensions in blocks of 32, 3 or 4 (the queries of more than 128 would not
// fit the registers), padded to PITCH in LDS
template <int DT>
__global__ __launch_bounds__(64 * NW, 2) void k_attn_tile32(const AttnArgs args) {
  AttnArgs a = args;
  uint32_t at = attn_call(a, blockIdx.x);
  constexpr int PITCH = 128;
  constexpr int CH = PITCH / 4;              // 16-byte pieces of a row
  constexpr int ROWB = 4 * PITCH;
  constexpr int TILEB = KT * ROWB;
  constexpr int RPI = 64 / CH;               // rows that one load of a wave brings
  constexpr int MINE = KT / NW;              // rows of a tile that a wave brings
  constexpr int LD = MINE / RPI;
  constexpr int KS = 32 * DT / 8;            // 16-byte pieces that a lane takes of a key
  constexpr int ROWS = 32 * NW;
  __shared__ __attribute__((aligned(1024))) char pool[4 * TILEB];  // keys twice, values twice
  lds_char *const kbuf = (lds_char *)pool;
  lds_char *const vbuf = kbuf + 2 * TILEB;

  const int lane = threadIdx.x & 63, h2 = lane >> 5, n = lane & 31;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t h = at % a.kv_heads;
  at /= a.kv_heads;
  const int32_t tile = a.tiles - 1 - (int32_t)(at % a.tiles);
  at /= a.tiles;
  const auto [b, part] = attn_turn<ATTN_FORMS>(a, at);
  const AttnSeq s = attn_seq<ATTN_FORMS>(a, b);
  const int32_t row0 = tile * ROWS;
  const int32_t T_used = s.T < a.max_new ? s.T : a.max_new;
  const int32_t rows_all = T_used * a.group;
  if (row0 >= rows_all) return;
  const int32_t last = row0 + ROWS < rows_all ? row0 + ROWS - 1 : rows_all - 1;
  const int32_t my_row = row0 + 32 * w + n, my_t = my_row / a.group;
  const int32_t my_head = h * a.group + my_row - my_t * a.group;
  const bool real = my_row <= last;
  // the positions between which this wave's and the block's rows stand
  const int32_t pos = real ? attn_position<ATTN_FORMS>(a, s, my_t) : -1;
  int32_t q_lo = real ? pos : 0x7FFFFFFF, q_hi = pos;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    q_lo = min(q_lo, __shfl_xor(q_lo, o));
    q_hi = max(q_hi, __shfl_xor(q_hi, o));
  }
  q_lo = __builtin_amdgcn_readfirstlane(q_lo), q_hi = __builtin_amdgcn_readfirstlane(q_hi);
  int32_t b_hi;
  {
    int32_t *ends = reinterpret_cast<int32_t *>(pool);
    if (lane == 0) ends[w] = q_hi;
    __syncthreads();
    b_hi = ends[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) b_hi = max(b_hi, ends[i]);
    b_hi = __builtin_amdgcn_readfirstlane(b_hi);
    __syncthreads();
  }
  const int32_t tiles = (b_hi + KT) / KT;  // (-1: none)
  const int32_t parts = attn_parts(a, tiles);
  if (part >= parts) {
    if (a.joined && real && h2 == 0) attn_empty_part(a, s, h, my_row, part);
    return;
  }
  const int32_t first = part * a.chunk;
  const int32_t end = part == parts - 1 ? tiles : first + a.chunk;

  f4 q[KS];
  {
    const float *src = static_cast<const float *>(a.q) +
                       (real ? (s.token0 + my_t) * a.q_row + my_head * a.q_head : 0);
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int e = 8 * i + 4 * h2;  // (no branch around a load: all are in flight)
      q[i] = *reinterpret_cast<const f4 *>(src + (e < a.d ? e : a.d - 4));
    }
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      if (!real || 8 * i + 4 * h2 >= a.d) q[i] = f4{0.f, 0.f, 0.f, 0.f};
    }
  }
  if (a.d < PITCH) {
    // pieces past the head are never loaded: they stay zero
    u32x4 *z = reinterpret_cast<u32x4 *>(pool);
    for (int i = threadIdx.x; i < 4 * TILEB / 16; i += 64 * NW) z[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
  }

  // The rows that this wave brings lie within 16, on one page.  Lane i holds
  // the addresses of those 16 for tile tb + i.
  const int piece = lane % CH, sub = lane / CH;
  uint32_t k_lo = 0, k_hi = 0, v_lo = 0, v_hi = 0;
  int32_t tb = 0;
  auto addresses = [&](int32_t i) {
    tb = i;
    const int32_t j = attn_row16(s, KT * (i + lane) + (MINE * w & ~15));
    int64_t page = 0, in = s.key0 + j;
    if (a.table) {
      const int32_t x = a.table[s.row + (j >> a.page_shift)];
      page = x < 0 ? 0 : x >= a.pages ? a.pages - 1 : x;
      in = j & ((1 << a.page_shift) - 1);
    }
    const uint64_t k = (uint64_t)(uintptr_t)a.k + 4 * (page * a.k_page + in * a.k_row + h * a.k_head);
    const uint64_t v = (uint64_t)(uintptr_t)a.v + 4 * (page * a.v_page + in * a.v_row + h * a.v_head);
    k_lo = (uint32_t)k, k_hi = (uint32_t)(k >> 32);
    v_lo = (uint32_t)v, v_hi = (uint32_t)(v >> 32);
  };
  // each lane's place in those 16 rows, in bytes (the keys from L on read row L - 1)
  auto place = [&](int x, int32_t most, int64_t stride, int c) -> uint32_t {
    const int32_t in = (MINE * w + x * RPI + sub) & 15;
    return 4 * ((uint32_t)(in < most ? in : most) * (uint32_t)stride + 4 * c);
  };
  uint32_t k_off[LD], v_off[LD];
#pragma unroll
  for (int x = 0; x < LD; ++x) {
    k_off[x] = place(x, 15, a.k_row, piece ^ k_swizzle<CH>(MINE * w + x * RPI + sub));
    v_off[x] = place(x, 15, a.v_row, piece);
  }
  const bool full = a.d == PITCH;
  auto fetch = [&](int32_t i) {
    if (i - tb >= 64) addresses(i);
    const uint64_t kb = lane_of(k_lo, k_hi, i - tb), vb = lane_of(v_lo, v_hi, i - tb);
    const int32_t to = (i & 1) * TILEB + MINE * w * ROWB;
    if (KT * i + KT <= s.L) {
      if (full) {
#pragma unroll
        for (int x = 0; x < LD; ++x) {
          load_to_lds(kb, k_off[x], kbuf + to + x * RPI * ROWB);
          load_to_lds(vb, v_off[x], vbuf + to + x * RPI * ROWB);
        }
        return;
      }
#pragma unroll
      for (int x = 0; x < LD; ++x)
        if (4 * (piece ^ k_swizzle<CH>(MINE * w + x * RPI + sub)) < a.d)
          load_to_lds(kb, k_off[x], kbuf + to + x * RPI * ROWB);
      if (4 * piece < a.d)
#pragma unroll
        for (int x = 0; x < LD; ++x) load_to_lds(vb, v_off[x], vbuf + to + x * RPI * ROWB);
      return;
    }
    const int32_t most = s.L - 1 - attn_row16(s, KT * i + (MINE * w & ~15));
#pragma unroll
    for (int x = 0; x < LD; ++x) {
      const int c = piece ^ k_swizzle<CH>(MINE * w + x * RPI + sub);
      if (4 * c < a.d)
        load_to_lds(kb, place(x, most, a.k_row, c), kbuf + to + x * RPI * ROWB);
      if (4 * piece < a.d)
        load_to_lds(vb, place(x, most, a.v_row, piece), vbuf + to + x * RPI * ROWB);
    }
  };

  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = f32x16{};
  float m = -INFINITY, l = 0.f;  // what the sums are relative to: a score, unscaled
  const int key_at = n * ROWB;

  if (first < end) {
    addresses(first);
    fetch(first);
  }
#pragma unroll 1
  for (int32_t i = first; i < end; ++i) {
    // the tile has arrived, and every wave has read the one before the last
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
    if (i + 1 < end) fetch(i + 1);
    const lds_char *kt = kbuf + (i & 1) * TILEB, *vt = vbuf + (i & 1) * TILEB;
    if (KT * i > q_hi) continue;  // (no row of this wave sees any of it)
    // (one read ahead of its products; left to itself the compiler asks for
    // more than there are registers)
    f32x16 sc = f32x16{};
    auto key = [&](int x) {
      return *(const lds_as f4 *)(kt + key_at + (((2 * x + h2) ^ k_swizzle<CH>(n)) << 4));
    };
    f4 k = key(0);
#pragma unroll
    for (int x = 0; x < KS; ++x)
      if (8 * x < a.d) {
        const f4 next = key(x + 1 < KS ? x + 1 : x);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sc = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q[x][e], sc, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        k = next;
      }
    const bool whole = KT * i + KT - 1 <= q_lo;
    const int32_t mine = KT * i + 4 * h2;  // key of register 0
    if (!whole) {
#pragma unroll
      for (int x = 0; x < 16; ++x)
        if (mine + 8 * (x >> 2) + (x & 3) > pos) sc[x] = -INFINITY;
    }
    float top = product_read(sc[0]);
#pragma unroll
    for (int x = 0; x < 16; x += 2) top = max3(top, sc[x], sc[x + 1]);
    top = xor32_max(top);
    const bool grown = (top - m) * a.scale_log2 > 8.f;
    if (__any(grown)) {
      const float nm = grown ? top : m;
      const float fade = nm == -INFINITY ? 1.f : attn_exp2((m - nm) * a.scale_log2);
      m = nm;
      l *= fade;
#pragma unroll
      for (int t = 0; t < DT; ++t) acc[t] *= fade;
    }
    // (subtracted before the scale comes in: the product of a large score with it
    // is rounded by more than a weight's range.  3 of 490 us)
    const float use = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      sc[x] = attn_exp2((sc[x] - use) * a.scale_log2);
      l += sc[x];
    }
    auto values = [&](int x, float (&v)[DT]) {
      const lds_as float *row =
          (const lds_as float *)(vt + (8 * (x >> 2) + 4 * h2 + (x & 3)) * ROWB) + DT * n;
      if constexpr (DT == 3) {
#pragma unroll
        for (int t = 0; t < DT; ++t) v[t] = row[t];
      } else {
        const f4 y = *(const lds_as f4 *)row;
#pragma unroll
        for (int t = 0; t < DT; ++t) v[t] = y[t];
      }
    };
    // What a masked place holds must not reach a sum, and 0 * NaN is NaN: of a
    // tile that not every row sees whole the products take no value that is
    // not finite, and those that a row sees are added to it alone.
    bool odd = false;
    float v[2][DT];
    values(0, v[0]);
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      if (x < 15) values(x + 1, v[(x + 1) & 1]);
      if (!whole) {
        const bool seen = mine + 8 * (x >> 2) + (x & 3) <= q_hi;
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          const bool fine = fabsf(v[x & 1][t]) < INFINITY;
          odd |= seen && !fine;
          v[x & 1][t] = fine ? v[x & 1][t] : 0.f;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < DT; ++t)
        acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[x & 1][t], sc[x], acc[t], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (!__any(odd)) continue;
    // (a rare path: the sums wait in memory meanwhile, so that it takes no
    // registers from the others)
    float held[16 * DT], wt[16];
#pragma unroll
    for (int x = 0; x < 16 * DT; ++x) held[x] = acc[x >> 4][x & 15];
#pragma unroll
    for (int x = 0; x < 16; ++x) wt[x] = sc[x];
#pragma unroll 1
    for (int j = 0; j < KT; ++j) {
      const float p = __shfl(wt[4 * (j >> 3) + (j & 3)], n + 32 * ((j >> 2) & 1));
      if (KT * i + j > pos) continue;
      const lds_as float *row = (const lds_as float *)(vt + j * ROWB);
#pragma unroll 1
      for (int x = 0; x < 16 * DT; ++x) {
        const float y = row[DT * (8 * ((x & 15) >> 2) + 4 * h2 + (x & 3)) + (x >> 4)];
        if (!(fabsf(y) < INFINITY)) held[x] = fmaf(p, y, held[x]);
      }
    }
#pragma unroll
    for (int x = 0; x < 16 * DT; ++x) acc[x >> 4][x & 15] = held[x];
  }

  const float sum = xor32_sum(l);
  const bool partial = parts > 1 || a.joined;
  const float f = partial ? 1.f : sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const int64_t row = (s.token0 + my_t) * a.heads + my_head;
  const int64_t x0 = (int64_t)(a.part0 + part) * a.tokens * a.heads + row;
  // The outputs leave by way of LDS (this wave's part of it, when no wave reads
  // keys any more), so that a store of a wave is whole rows: 4 bytes of each of
  // 64 rows at a time took as long as 500 keys.
  __syncthreads();
  lds_char *const mine = kbuf + 32 * w * ROWB;
#pragma unroll
  for (int x = 0; x < 16; ++x)
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const int e = DT * (8 * (x >> 2) + 4 * h2 + (x & 3)) + t;
      *(lds_as float *)(mine + n * ROWB + (((e >> 2) ^ k_swizzle<CH>(n)) << 4) + 4 * (e & 3)) =
          acc[t][x] * f;
    }
  const int64_t to = !real     ? INT64_MIN
                     : partial ? x0 * PITCH
                               : (s.token0 + my_t) * a.o_row + my_head * a.o_head;
  float *dst = partial ? a.part_o : static_cast<float *>(a.out);
#pragma unroll 4
  for (int x = 0; x < 32 / RPI; ++x) {
    const int r = x * RPI + sub;
    const f4 y = *(const lds_as f4 *)(mine + r * ROWB + ((piece ^ k_swizzle<CH>(r)) << 4));
    const int64_t at_row = __shfl(to, r);
    if (at_row != INT64_MIN && 4 * piece < a.d) *reinterpret_cast<f4 *>(dst + at_row + 4 * piece) = y;
  }
  if (h2 == 0 && real) {
    if (partial) {
      a.part_ml[2 * x0] = m;
      a.part_ml[2 * x0 + 1] = sum;
    } else if (a.lse) {
      a.lse[row] = attn_lse(m * a.scale_log2, sum);
    }
  }
}

}  // namespace

void launch_attn_tile32(vsk_ctx *ctx, hipStream_t st, const AttnArgs &a) {
  const int64_t grid = a.pre_blocks + (int64_t)a.n * a.splits * a.tiles * a.kv_heads;
  VSK_REQUIRE(grid <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "too many query rows in one call");
  KernelTimer kt(ctx, "attn_tile32", (double)a.tokens * a.heads, st);
  const unsigned g = (unsigned)grid;
  if (a.d <= 96)
    k_attn_tile32<3><<<g, 64 * NW, 0, st>>>(a);
  else
    k_attn_tile32<4><<<g, 64 * NW, 0, st>>>(a);
  check_launch("attn_tile32");
}

}  // namespace vsk
