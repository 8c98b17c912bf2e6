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
#include "attn.hpp"
#include "vsk_api.hpp"

namespace vsk {

namespace {

typedef __attribute__((ext_vector_type(4))) short i16x4;
constexpr int NW = 4;  // waves of a workgroup

// TOP: log2 of a weight where its score sets the reference; weights grow to
// 2^(TOP + 8).  In f16 as large as fits, so that small ones are not lost.
template <class T> struct Mm;
template <> struct Mm<__bf16> {
  typedef bf16x8 V8;
  static constexpr float TOP = 0.f;
  static constexpr uint32_t EXP = 0x7F807F80u;
  static __device__ f32x16 mfma(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mm<_Float16> {
  typedef f16x8 V8;
  static constexpr float TOP = 7.f;
  static constexpr uint32_t EXP = 0x7C007C00u;
  static __device__ f32x16 mfma(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// V's pieces in LDS: the four rows of a transposing read go to different
// banks (K's: attn.hpp).
template <int CH> __device__ inline int v_swizzle(int row) {
  const int x = row & 3;
  return CH >= 16 ? 4 * x + 2 * (x >> 1) : 2 * x;
}

// (fmaxf would first quiet each product, an instruction a value: the maximum
// here passes over NaN without it)
__device__ inline float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// DP: the head, padded to products.  Two workgroups of four waves share a
// compute unit, so that one's start and end hide behind the other's products
// (one of eight waves over twice the rows: 340 us where these take 308, 8
// ragged prompts to 4,096 of 32 heads of 128, window 1,024).
template <class T, int DP>
__global__ __launch_bounds__(64 * NW, DP == 256 ? 1 : 2) void k_attn_tile(const AttnArgs a) {
  typedef typename Mm<T>::V8 V8;
  typedef __attribute__((ext_vector_type(4))) T V4;
  constexpr int KT = attn_tile_keys(DP), U = KT / 32, G = ATTN_TILE_GROUP;
  constexpr int PITCH = DP <= 64 ? 64 : DP <= 128 ? 128 : 256;
  constexpr int CH = PITCH / 8;      // 16-byte pieces of a row
  constexpr int ROWB = 2 * PITCH;    // bytes of a row
  constexpr int TILEB = KT * ROWB;   // bytes of a tile
  constexpr int RPI = 64 / CH;       // rows that one load of a wave brings
  constexpr int MINE = KT / NW;      // rows of a tile that a wave brings
  constexpr int LD = MINE / RPI;     // loads that takes
  constexpr int KS = DP / 16, DT = DP / 32;
  constexpr int ROWS = 32 * NW;      // query rows of the block
  // tile i's keys in kbuf[i % 3], two tiles ahead of their products, its
  // values in vbuf[i % 2], one ahead
  __shared__ __attribute__((aligned(1024))) char keys_lds[3 * TILEB];
  __shared__ __attribute__((aligned(1024))) char values_lds[2 * TILEB];
  lds_char *const kbuf = (lds_char *)keys_lds;
  lds_char *const vbuf = (lds_char *)values_lds;

  const int lane = threadIdx.x & 63, h2 = lane >> 5, n = lane & 31;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t at = blockIdx.x;
  const int32_t h = at % a.kv_heads;
  at /= a.kv_heads;
  const int32_t tile = a.tiles - 1 - (int32_t)(at % a.tiles);
  at /= a.tiles;
  const int32_t part = at % a.splits;
  const AttnSeq s = attn_seq(a, at / a.splits);
  const int32_t row0 = tile * ROWS;
  const int32_t T_used = s.T < a.max_new ? s.T : a.max_new;
  const int32_t rows_all = T_used * a.group;
  if (row0 >= rows_all) return;
  const int32_t last = row0 + ROWS < rows_all ? row0 + ROWS - 1 : rows_all - 1;
  const int32_t p0 = s.L - s.T;
  const auto span = attn_span<KT, G>(a, p0 + row0 / a.group, p0 + last / a.group);
  const int32_t parts = attn_parts(a, span.tiles);
  if (part >= parts) return;
  const int32_t first = part * a.chunk;
  const int32_t end = part == parts - 1 ? span.tiles : first + a.chunk;

  // this wave's rows and what they see
  const int32_t w0 = row0 + 32 * w, w1 = w0 + 31 < last ? w0 + 31 : last;
  const bool have = w0 <= last;
  const int32_t q_lo = p0 + w0 / a.group, q_hi = have ? p0 + w1 / a.group : -1;
  // (a head of 256 leaves no registers for the queries: each lane's wait in LDS)
  constexpr bool QLDS = DP == 256;
  __shared__ __attribute__((aligned(1024))) char queries_lds[QLDS ? NW * KS * 1024 : 16];
  lds_char *const qbuf = (lds_char *)queries_lds + 16 * lane;
  const int32_t my_row = w0 + n, my_t = my_row / a.group;
  const int32_t my_head = h * a.group + my_row - my_t * a.group;
  const bool real = my_row <= last;
  const int32_t pos = real ? p0 + my_t : -1;
  V8 q[QLDS ? 1 : KS];
  auto query = [&](int x) -> V8 {
    if constexpr (QLDS) return *(const lds_as V8 *)(qbuf + (w * KS + x) * 1024);
    return q[QLDS ? 0 : x];
  };
  {
    V8 mine[KS];
    const T *src = static_cast<const T *>(a.q) +
                   (real ? (s.token0 + my_t) * a.q_row + my_head * a.q_head : 0);
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int e = 16 * i + 8 * h2;  // (no branch around a load: all are in flight)
      mine[i] = *reinterpret_cast<const V8 *>(src + (e < a.d ? e : a.d - 8));
    }
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      if (!real || 16 * i + 8 * h2 >= a.d) mine[i] = V8{};
      if constexpr (QLDS)
        *(lds_as V8 *)(qbuf + (w * KS + i) * 1024) = mine[i];
      else
        q[QLDS ? 0 : i] = mine[i];
    }
  }
  if (a.d < PITCH) {
    // pieces past the head are never loaded: they stay zero
    u32x4 *z = reinterpret_cast<u32x4 *>(keys_lds), *y = reinterpret_cast<u32x4 *>(values_lds);
    for (int i = threadIdx.x; i < 3 * TILEB / 16; i += 64 * NW) z[i] = u32x4{0, 0, 0, 0};
    for (int i = threadIdx.x; i < 2 * TILEB / 16; i += 64 * NW) y[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
  }

  f32x16 acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = f32x16{};
  float m = -INFINITY, l = 0.f;

  // The rows of a tile that this wave brings lie within 16, on one page.
  // Lane i holds the addresses of those 16 for tile tb + i, keys and values.
  const int piece = lane % CH, sub = lane / CH;
  uint32_t k_lo = 0, k_hi = 0, v_lo = 0, v_hi = 0;
  int32_t tb = 0;
  auto addresses = [&](int32_t i) {
    tb = i;
    const int32_t j = attn_row16(s, span.group(KT / G * (i + lane) + MINE * w / G));
    int64_t page = 0, in = s.key0 + j;
    if (a.table) {
      int32_t x = a.table[s.slot * a.table_stride + (j >> a.page_shift)];
      page = x < 0 ? 0 : x >= a.pages ? a.pages - 1 : x;
      in = j & ((1 << a.page_shift) - 1);
    }
    const uint64_t k = (uint64_t)(uintptr_t)a.k + 2 * (page * a.k_page + in * a.k_row + h * a.k_head);
    const uint64_t v = (uint64_t)(uintptr_t)a.v + 2 * (page * a.v_page + in * a.v_row + h * a.v_head);
    k_lo = (uint32_t)k, k_hi = (uint32_t)(k >> 32);
    v_lo = (uint32_t)v, v_hi = (uint32_t)(v >> 32);
  };
  // each lane's place in those 16 rows, in bytes
  uint32_t k_off[LD], v_off[LD];
  auto offset = [&](int x, int32_t most, bool keys) -> uint32_t {
    const int lr = MINE * w + x * RPI + sub;
    const int32_t off = (lr & 15) < most ? (lr & 15) : most;
    const int c = piece ^ (keys ? k_swizzle<CH>(lr) : v_swizzle<CH>(lr));
    return 2 * ((uint32_t)off * (uint32_t)(keys ? a.k_row : a.v_row) + 8 * c);
  };
#pragma unroll
  for (int x = 0; x < LD; ++x) k_off[x] = offset(x, 15, true), v_off[x] = offset(x, 15, false);
  const bool full = a.d == PITCH;
  auto fetch = [&](int32_t i, lds_char *to, bool keys) {
    const uint64_t base = keys ? lane_of(k_lo, k_hi, i - tb) : lane_of(v_lo, v_hi, i - tb);
    const int32_t j0 = span.group(KT / G * i + MINE * w / G) + MINE * w % G;
    to += MINE * w * ROWB;
    if (full && j0 + MINE <= s.L) {
#pragma unroll
      for (int x = 0; x < LD; ++x)
        load_to_lds(base, keys ? k_off[x] : v_off[x], to + x * RPI * ROWB);
      return;
    }
    // (the keys from L on read row L - 1, pieces past the head nothing)
    const int32_t left = s.L - 1 - attn_row16(s, j0 & ~15);
#pragma unroll
    for (int x = 0; x < LD; ++x) {
      const int lr = MINE * w + x * RPI + sub;
      const int c = piece ^ (keys ? k_swizzle<CH>(lr) : v_swizzle<CH>(lr));
      const uint32_t off = offset(x, left, keys);
      if (8 * c < a.d) load_to_lds(base, off, to + x * RPI * ROWB);
    }
  };

  // lane's parts of the addresses of the reads
  const int gi = lane & 15, va = gi >> 2, vhalf = (lane >> 4) & 1;
  const int k_at = n * ROWB + ((h2 ^ k_swizzle<CH>(n)) << 4);
  const int v_at = (4 * h2 + va) * ROWB + 8 * (gi & 1) +
                   (((2 * vhalf + ((gi & 3) >> 1)) ^ v_swizzle<CH>(va)) << 4);
  // piece 2 x + h2 of key 32 u + n: the swizzle leaves bit operations only
  auto key_piece = [&](int base, int x, int u) -> V8 {
    return *(const lds_as V8 *)(uintptr_t)(uint32_t)((base ^ (x << 5)) + 32 * u * ROWB);
  };
  // dimensions 32 dt on of keys 16 u + 4 h2 .. + 3 and 8 further
  auto value_piece = [&](int base, int dt, int u) -> V8 {
    const int at = (base ^ (dt << 6)) + 16 * u * ROWB;
    union {
      i16x4 half[2];
      V8 v;
    } f;
    f.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_as i16x4 *)(uintptr_t)(uint32_t)at);
    f.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_as i16x4 *)(uintptr_t)(uint32_t)(at + 8 * ROWB));
    return f.v;
  };
  auto k_base = [&](const lds_char *buf) { return (int)(uintptr_t)buf + k_at; };
  auto v_base = [&](const lds_char *buf) { return (int)(uintptr_t)buf + v_at; };

  // register 16 u + x of the scores belongs to key 32 u + 8 (x / 4) + 4 h2 +
  // x % 4 of the tile
  auto scores = [&](const lds_char *buf, f32x16 (&sc)[U]) {
    const int kb = k_base(buf);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      sc[u] = f32x16{};
#pragma unroll
      for (int x = 0; x < KS; ++x) sc[u] = Mm<T>::mfma(key_piece(kb, x, u), query(x), sc[u]);
    }
  };
  auto largest = [&](const f32x16 (&sc)[U]) {
    float tm = max3(sc[0][0], sc[0][1], sc[0][2]);
#pragma unroll
    for (int x = 3; x < 16 * U - 1; x += 2)
      tm = max3(tm, sc[x >> 4][x & 15], sc[(x + 1) >> 4][(x + 1) & 15]);
    return xor32_max(max3(tm, sc[U - 1][15], sc[U - 1][15]));
  };
  // Past FAR the product of a score and the scale, and so m, is rounded by more
  // than an eighth of one in log2, further on (2^24) by more than the room that
  // f16's weights have, then fp32's.  Rows with such scores, which no model
  // makes, are computed again at the end.
  constexpr float FAR = 2097152.f;
  bool again = false;
  // The sums are kept relative to m, which follows the largest score (less TOP)
  // only when that has grown by 8 (in log2): weights 256 times as large cost no
  // precision, and the sums are seldom rescaled.
  auto settle = [&](float tm) {
    const float top = tm * a.scale_log2 - Mm<T>::TOP;
    if (!__any(top > m + 8.f)) return;
    again |= fabsf(top) > FAR && fabsf(tm) < INFINITY;
    const float nm = top > m + 8.f ? top : m;
    const float fade = nm == -INFINITY ? 1.f : attn_exp2(m - nm);
    m = nm;
    l *= fade;
#pragma unroll
    for (int x = 0; x < DT; ++x) {
      acc[x] *= fade;
      if (DP == 256) __builtin_amdgcn_sched_barrier(0);  // (few registers at a time)
    }
  };
  // -inf for the keys that the lane's row does not see.  Bit c of a
  // word is key c of the 32 that the word is for: comparisons a row, not a key.
  auto up_to = [](int32_t x) -> uint32_t { return x < 0 ? 0u : x > 30 ? ~0u : (2u << x) - 1; };
  auto sees = [&](int32_t b) -> uint32_t {
    uint32_t see = ~0u;
    if (a.window > 0)
      see = (pos < a.window ? ~0u : ~up_to(pos - a.window - b)) | up_to(a.sinks - 1 - b);
    return see & up_to(pos - b);
  };
  auto hide = [&](f32x16 (&sc)[U], int32_t i) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int32_t b = span.group(KT / G * i + 2 * u), c = span.group(KT / G * i + 2 * u + 1);
      uint32_t see = sees(b + 4 * h2);
      if (c != b + G) see = (see & 0xFFFFu) | (sees(c - G + 4 * h2) & 0xFFFF0000u);
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const uint32_t on = (uint32_t)((int32_t)(see << (31 - 8 * (x >> 2) - (x & 3))) >> 31);
        sc[u][x] = __uint_as_float((on & __float_as_uint(sc[u][x])) | (~on & 0xFF800000u));
      }
    }
  };
  // is a value of the tile not finite?  (the largest exponent field)
  auto not_finite = [&](const lds_char *vt) -> bool {
    typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
    u16x2 top = {0, 0};
    const lds_as u32x4 *v4 = (const lds_as u32x4 *)vt;
#pragma unroll 4
    for (int x = lane; x < TILEB / 16; x += 64) {
      const u32x4 y = v4[x];
#pragma unroll
      for (int z = 0; z < 4; ++z)
        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, y[z] & Mm<T>::EXP));
    }
    const unsigned short inf = (unsigned short)(Mm<T>::EXP & 0xFFFF);
    return __any(top[0] == inf || top[1] == inf);
  };
  // tile i, that not every row of the block sees whole
  auto edge = [&](int32_t i, const lds_char *kt, const lds_char *vt) {
    // (a wave whose rows see none of it only brings its rows)
    const int32_t kb = span.base(i), ke = span.group(KT / G * (i + 1) - 1) + G;  // (end)
    const bool any = kb <= q_hi && (a.window <= 0 || q_lo - ke < a.window - 1 || kb < a.sinks);
    if (!any) return;
    const bool whole = ke == kb + KT && ke <= q_lo + 1 &&
                       (a.window <= 0 || q_hi - kb < a.window || ke <= a.sinks);
    f32x16 sc[U];
    if (whole || !not_finite(vt)) {
      scores(kt, sc);
      const int vb = v_base(vt);
      if (!whole) hide(sc, i);
      settle(largest(sc));
      const float use = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int u = 0; u < 2 * U; ++u) {
        V8 p;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float y = attn_exp2(fmaf(sc[u >> 1][8 * (u & 1) + x], a.scale_log2, -use));
          l += y;
          p[x] = (T)y;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] = Mm<T>::mfma(value_piece(vb, dt, u), p, acc[dt]);
      }
      return;
    }
    // a masked place must not reach a sum, and 0 * NaN is NaN: the keys one at
    // a time, each row takes only those it sees.  (A rare path: the sums wait
    // in memory meanwhile, so that it takes no registers from the others.)
    scores(kt, sc);
    hide(sc, i);
    settle(largest(sc));
    const float use = m == -INFINITY ? 0.f : m;
    float held[16 * DT], wt[16 * U];
#pragma unroll
    for (int x = 0; x < 16 * DT; ++x) held[x] = acc[x >> 4][x & 15];
#pragma unroll
    for (int x = 0; x < 16 * U; ++x) {
      wt[x] = attn_exp2(fmaf(sc[x >> 4][x & 15], a.scale_log2, -use));
      l += wt[x];
    }
#pragma unroll 1
    for (int j = 0; j < KT; ++j) {
      // key j is in register 16 (j / 32) + 4 (j / 8 % 4) + j % 4 of the lanes
      // whose h2 is bit 2 of j
      const float y = __shfl(wt[16 * (j >> 5) + 4 * ((j >> 3) & 3) + (j & 3)],
                             n + 32 * ((j >> 2) & 1));
      if (!attn_sees(a, pos, span.group(KT / G * i + j / G) + j % G)) continue;
#pragma unroll 1
      for (int c = 0; c < 4 * DT; ++c) {
        const lds_as T *v =
            (const lds_as T *)(vt + j * ROWB + ((c ^ v_swizzle<CH>(j)) << 4)) + 4 * h2;
#pragma unroll 1
        for (int x = 0; x < 4; ++x) held[4 * c + x] = fmaf(y, (float)v[x], held[4 * c + x]);
      }
    }
#pragma unroll
    for (int x = 0; x < 16 * DT; ++x) acc[x >> 4][x & 15] = held[x];
  };

  // the tiles that every row of the block sees whole: from the window's edge
  // of the last row to the first row's diagonal
  int32_t hot0 = first, hot1 = first;
  {
    const int32_t lo = p0 + row0 / a.group, hi = p0 + last / a.group;
    int32_t x0 = G * span.sink_groups;
    const int32_t x1 = lo + 1 > span.lo ? (x0 + lo + 1 - span.lo) / KT : 0;
    if (a.window > 0 && hi - span.lo >= a.window) x0 += hi - a.window - span.lo + 1;
    x0 = (x0 + KT - 1) / KT;
    hot0 = x0 > first ? x0 : first;
    hot1 = x1 < end ? x1 : end;
  }

  int kslot = 0;  // (i - first) % 3
  if (first < end) {
    addresses(first);
    fetch(first, kbuf, true);
    fetch(first, vbuf, false);
    if (first + 1 < end) fetch(first + 1, kbuf + TILEB, true);
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();

  // a step's copies: the keys of tile i + 2, the values of tile i + 1
  auto ahead = [&](int32_t i) {
    if (i + 2 - tb >= 64) addresses(i + 1);
    if (i + 2 < end) fetch(i + 2, kbuf + (kslot == 0 ? 2 : kslot - 1) * TILEB, true);
    if (i + 1 < end) fetch(i + 1, vbuf + ((i + 1 - first) & 1) * TILEB, false);
  };
  auto done = [&]() {
    kslot = kslot == 2 ? 0 : kslot + 1;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the copies have arrived
    __syncthreads();
  };

  for (int32_t i = first; i < end;) {
    if (i < hot0 || i >= hot1) {
      ahead(i);
      edge(i, kbuf + kslot * TILEB, vbuf + ((i - first) & 1) * TILEB);
      done();
      ++i;
      continue;
    }
    // A step computes the scores of the next tile and the weights and sums of
    // this one, the products on the matrix cores beside the exponentials on
    // the vector unit: the order below is the order they are issued in, one
    // piece of LDS, a read four pieces ahead, and a share of the vector work
    // at a time (left to itself the compiler keeps one read in flight).  The
    // last step's scores are not used: what follows is an edge, or nothing.
    constexpr int NS = U * KS, NV = 2 * U * DT, AHEAD = 4;
    f32x16 sc[U];
    scores(kbuf + kslot * TILEB, sc);
    settle(largest(sc));
#pragma unroll 1
    for (; i < hot1; ++i) {
      ahead(i);
      const int kb = k_base(kbuf + (kslot == 2 ? 0 : kslot + 1) * TILEB);
      const int vb = v_base(vbuf + ((i - first) & 1) * TILEB);
      const float use = m == -INFINITY ? 0.f : m;
      f32x16 sn[U];
      V8 f[AHEAD], p[2 * U], qf[QLDS ? AHEAD : 1];
      float tm = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) sn[u] = f32x16{};
      auto piece_of = [&](int g) -> V8 {
        return g < NS ? key_piece(kb, g / U, g % U) : value_piece(vb, (g - NS) % DT, (g - NS) / DT);
      };
      auto weight = [&](int e) {  // of register e of the scores
        const float y = attn_exp2(fmaf(sc[e >> 4][e & 15], a.scale_log2, -use));
        l += y;
        p[e >> 3][e & 7] = (T)y;
      };
#pragma unroll
      for (int g = 0; g < AHEAD; ++g) {
        f[g] = piece_of(g);
        if (QLDS) qf[QLDS ? g : 0] = query(g / U);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int g = 0; g < NS + NV; ++g) {
        const V8 x = f[g % AHEAD];
        if (g < NS)
          sn[g % U] = Mm<T>::mfma(x, QLDS ? qf[QLDS ? g % AHEAD : 0] : query(g / U), sn[g % U]);
        else
          acc[(g - NS) % DT] = Mm<T>::mfma(x, p[(g - NS) / DT], acc[(g - NS) % DT]);
        if (g + AHEAD < NS + NV) f[g % AHEAD] = piece_of(g + AHEAD);
        if (QLDS && g + AHEAD < NS) qf[QLDS ? g % AHEAD : 0] = query((g + AHEAD) / U);
        // half of the weights beside the scores, half beside the first sums
        if (g < NS) {
#pragma unroll
          for (int e = 8 * U * g / NS; e < 8 * U * (g + 1) / NS; ++e) weight(e);
        } else if (g - NS < NV / 2) {
#pragma unroll
          for (int e = 8 * U * (g - NS) / (NV / 2); e < 8 * U * (g - NS + 1) / (NV / 2); ++e)
            weight(8 * U + e);
        } else {
          const int z = g - NS - NV / 2;
#pragma unroll
          for (int e = 8 * U * z / (NV / 2); e < 8 * U * (z + 1) / (NV / 2); ++e)
            tm = max3(tm, sn[e >> 3][2 * (e & 7)], sn[e >> 3][2 * (e & 7) + 1]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) sc[u] = sn[u];
      if (i + 1 < hot1) settle(xor32_max(tm));
      done();
    }
  }

  float sum = xor32_sum(l);
  // An f16 weight may have been rounded to zero, and zero times an infinite
  // value is NaN.
  if constexpr (Mm<T>::TOP > 0.f) {
    bool odd = false;
#pragma unroll
    for (int x = 0; x < 16 * DT; x += 2)
      odd |= __builtin_isunordered(acc[x >> 4][x & 15], acc[x >> 4][(x & 15) + 1]);
    again |= odd && sum == sum;
  }
  // Key by key on the vector unit, the largest score subtracted before the
  // scale comes in.  Of a row's products a lane has half, of its outputs those
  // in its registers.
  float ref = -INFINITY;  // by_key: the largest score, unscaled
  const bool by_key = __any(again);
  if (by_key) {
#pragma unroll
    for (int x = 0; x < DT; ++x) acc[x] = f32x16{};
    sum = 0.f;
#pragma unroll 1
    for (int32_t x = first * KT; x < end * KT; ++x) {
      const int32_t j = span.group(x / G) + x % G;
      const bool see = attn_sees(a, pos, j);
      if (!__any(see)) continue;
      const AttnRows r = attn_rows(a, s, h, j & ~15, attn_page(a, s, j & ~15));
      const T *kr = static_cast<const T *>(a.k) + r.k + (j & 15) * a.k_row;
      const T *vr = static_cast<const T *>(a.v) + r.v + (j & 15) * a.v_row;
      float sc = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int e = 16 * i + 8 * h2;
        if (e >= a.d) continue;
        const V8 kv = *reinterpret_cast<const V8 *>(kr + e), qv = query(i);
#pragma unroll
        for (int y = 0; y < 8; ++y) sc = fmaf((float)qv[y], (float)kv[y], sc);
      }
      sc = xor32_sum(sc);
      const float top = see ? fmaxf(ref, sc) : ref, use = top == -INFINITY ? 0.f : top;
      const float fade = attn_exp2((ref - use) * a.scale_log2);
      const float p = see ? attn_exp2((sc - use) * a.scale_log2) : 0.f;
      ref = top;
      sum = sum * fade + p;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        acc[dt] *= fade;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int e = 32 * dt + 8 * b + 4 * h2;
          if (!see || e >= a.d) continue;
          const V4 vv = *reinterpret_cast<const V4 *>(vr + e);
#pragma unroll
          for (int y = 0; y < 4; ++y) acc[dt][4 * b + y] = fmaf(p, (float)vv[y], acc[dt][4 * b + y]);
        }
      }
    }
    m = ref * a.scale_log2;
  }
  const int64_t out_row = (s.token0 + my_t) * a.heads + my_head;
  if (parts > 1) {
    if (!real) return;
    // a part's reference is a score: the one that m was made of, or near it
    if (!by_key && m != -INFINITY) {
      ref = (m + Mm<T>::TOP) / a.scale_log2;
      const float f = attn_exp2(-fmaf(ref, a.scale_log2, -m));
      sum *= f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
    }
    const int64_t x = (int64_t)part * a.tokens * a.heads + out_row;
    float *dst = a.part_o + x * PITCH;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        *reinterpret_cast<f32x4 *>(dst + 32 * dt + 8 * b + 4 * h2) =
            f32x4{acc[dt][4 * b], acc[dt][4 * b + 1], acc[dt][4 * b + 2], acc[dt][4 * b + 3]};
    if (h2 == 0) {
      a.part_ml[2 * x] = ref;
      a.part_ml[2 * x + 1] = sum;
    }
    return;
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  // The outputs leave by way of LDS (no wave reads keys any more), so that a
  // store of a wave is whole rows and not eight bytes of each.
  lds_char *const obuf = (QLDS ? (lds_char *)queries_lds : kbuf) + 32 * w * ROWB;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      V4 y;
#pragma unroll
      for (int x = 0; x < 4; ++x) y[x] = (T)(acc[dt][4 * b + x] * inv);
      *(lds_as V4 *)(obuf + n * ROWB + (((4 * dt + b) ^ k_swizzle<CH>(n)) << 4) + 8 * h2) = y;
    }
  const int64_t to = real ? (s.token0 + my_t) * a.o_row + my_head * a.o_head : INT64_MIN;
#pragma unroll
  for (int x = 0; x < 32 / RPI; ++x) {
    const int r = x * RPI + sub;
    typedef __attribute__((ext_vector_type(4), aligned(8))) uint32_t Piece;
    const u32x4 y = *(const lds_as u32x4 *)(obuf + r * ROWB + ((piece ^ k_swizzle<CH>(r)) << 4));
    const int64_t row = __shfl(to, r);
    if (row != INT64_MIN && 8 * piece < a.d)
      *reinterpret_cast<Piece *>(static_cast<T *>(a.out) + row + 8 * piece) = y;
  }
  if (a.lse && h2 == 0 && real)
    a.lse[out_row] = attn_lse(m, sum);
}

template <class T> void tile_of(hipStream_t st, const AttnArgs &a, unsigned g) {
  if (a.d <= 64)
    k_attn_tile<T, 64><<<g, 64 * NW, 0, st>>>(a);
  else if (a.d <= 96)
    k_attn_tile<T, 96><<<g, 64 * NW, 0, st>>>(a);
  else if (a.d <= 128)
    k_attn_tile<T, 128><<<g, 64 * NW, 0, st>>>(a);
  else
    k_attn_tile<T, 256><<<g, 64 * NW, 0, st>>>(a);
}

}  // namespace

void launch_attn_tile(vsk_ctx *ctx, hipStream_t st, const AttnArgs &a, int32_t t) {
  const int64_t grid = (int64_t)a.n * a.splits * a.tiles * a.kv_heads;
  VSK_REQUIRE(grid <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "too many query rows in one call");
  KernelTimer kt(ctx, "attn_tile", (double)a.tokens * a.heads, st);
  if (t == VSK_DTYPE_F16)
    tile_of<_Float16>(st, a, (unsigned)grid);
  else
    tile_of<__bf16>(st, a, (unsigned)grid);
  check_launch("attn_tile");
}

}  // namespace vsk
