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
#include "attn.hpp"
#include "vsk_api.hpp"

namespace vsk {

namespace {

// What a type's 32-bit words hold: E elements; 16 bytes hold 4 * E.
// TOP: log2 of the largest weight.  An f16 of 1 at most loses a weight under
// 2^-25, and a long context may hold many of them behind one large first key;
// bf16 has fp32's exponents.
template <class T> struct Elem;
template <> struct Elem<float> {
  static constexpr int E = 1;
  static constexpr float TOP = 0.f;
  static constexpr uint32_t EXP = 0x7F800000u;  // an infinity's or NaN's exponent
};
template <> struct Elem<__bf16> {
  typedef bf16x8 V8;
  static constexpr int E = 2;
  static constexpr float TOP = 0.f;
  static constexpr uint32_t EXP = 0x7F80u;
  static __device__ f32x4 mfma(u32x4 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V8, a), b, c, 0, 0, 0);
  }
};
template <> struct Elem<_Float16> {
  typedef f16x8 V8;
  static constexpr int E = 2;
  static constexpr float TOP = 15.f;
  static constexpr uint32_t EXP = 0x7C00u;
  static __device__ f32x4 mfma(u32x4 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V8, a), b, c, 0, 0, 0);
  }
};
template <class T> __device__ inline bool not_finite(uint32_t w) {
  constexpr uint32_t X = Elem<T>::EXP;
  if constexpr (sizeof(T) == 4) return (w & X) == X;
  return (w & X) == X || ((w >> 16) & X) == X;
}

// x, as a value that the compiler computes nothing from beforehand: what it
// would (comparisons, a division's reciprocal) waits in registers through the
// loop over the keys, or, with too few of them, in scratch memory, which alone
// costs 64 contexts to 8,192 2 us.
__device__ inline int32_t hidden(int32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// W words of a row of any alignment from element e on, zero from element d on
template <class T, int W>
__device__ inline void load_row(const global_as T *row, int32_t e, int32_t d, uint32_t (&x)[W]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < W; ++i) x[i] = e + i < d ? __builtin_bit_cast(uint32_t, row[e + i]) : 0u;
  } else {
    const global_as uint16_t *h = reinterpret_cast<const global_as uint16_t *>(row);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      x[i] = e + 2 * i < d ? h[e + 2 * i] : 0u;
      if (e + 2 * i + 1 < d) x[i] |= (uint32_t)h[e + 2 * i + 1] << 16;
    }
  }
}

constexpr int ROWS = 16;  // query rows of a wave
// 16-key tiles of a step: the k of a 16-bit product is 32 keys
template <class T> constexpr int SUBS = sizeof(T) == 4 ? 1 : 2;

// The wave's 16 rows over key tiles.  VW: elements of V that a lane takes of a
// row, 16 lanes a block; NB blocks.
template <class T, int VW, int NB, bool ALIGNED> struct RowTile {
  static constexpr int DV = 16 * VW * NB;
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int E = Elem<T>::E;
  static constexpr int KE = 4 * E;          // elements of 16 bytes
  static constexpr int KS = DV / (4 * KE);  // 16-byte loads a lane makes of a key row
  static constexpr int U = SUBS<T>;
  static constexpr int KT = 16 * U;
  static constexpr int WV = VW / E;         // words a lane takes of a row's block
  const AttnArgs &a;
  const AttnSeq &s;
  // (aligned) the step's keys in LDS, this wave's own
  static constexpr int ROWB = DV * (int)sizeof(T), CH = ROWB / 16, RPI = 64 / CH;
  lds_char *const lds;
  const int32_t h;
  int32_t n, g;
  int32_t pos;  // position of this lane's row, -1 if there is none
  uint32_t q[KS][4];
  f32x4 acc[NB][VW];
  float m = -INFINITY;  // the largest score, unscaled
  float l = 0.f;

  __device__ RowTile(const AttnArgs &a_, const AttnSeq &s_, int32_t h_, int lane, lds_char *l_)
      : a(a_), s(s_), lds(l_), h(h_), n(lane & 15), g(lane >> 4) {}

  __device__ void begin(int32_t row) {
    const int32_t t = row / a.group;
    const bool real = t < s.T && t < a.max_new;
    pos = real ? s.L - s.T + t : -1;
    const T *src = static_cast<const T *>(a.q) +
                   (real ? (s.token0 + t) * a.q_row + (h * a.group + row % a.group) * a.q_head : 0);
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int32_t e = (4 * i + g) * KE;
      if constexpr (ALIGNED) {
        // (all of them in flight at once: no branch around any)
        const u32x4 y = *reinterpret_cast<const u32x4 *>(src + (e < a.d ? e : a.d - KE));
#pragma unroll
        for (int z = 0; z < 4; ++z) q[i][z] = y[z];
      } else {
        load_row<T, 4>((const global_as T *)src, e, real ? a.d : 0, q[i]);
      }
    }
    if constexpr (ALIGNED) {
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int z = 0; z < 4; ++z)
          q[i][z] = real && (4 * i + g) * KE < a.d ? q[i][z] : 0u;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int t2 = 0; t2 < VW; ++t2) acc[b][t2] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // acc += V^T P^T; p[u][i] belongs to key 16 u + 4 g + i and v[u][i] is that
  // key's row
  __device__ void weigh(const float (&p)[U][4], const uint32_t (&v)[U][4][NB][WV]) {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int t = 0; t < VW; ++t)
            acc[b][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                __builtin_bit_cast(float, v[0][i][b][t]), p[0][i], acc[b][t], 0, 0, 0);
    } else {
      typename Elem<T>::V8 hi, lo;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          hi[4 * u + i] = (T)p[u][i];
          lo[4 * u + i] = (T)(p[u][i] - (float)hi[4 * u + i]);
        }
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < VW; ++t) {
          // element t of eight rows: the low or high halves of their words
          constexpr uint32_t LOW = 0x05040100u, HIGH = 0x07060302u;
          u32x4 x;
#pragma unroll
          for (int y = 0; y < 4; ++y)
            x[y] = __builtin_amdgcn_perm(v[y >> 1][2 * (y & 1) + 1][b][t / 2],
                                         v[y >> 1][2 * (y & 1)][b][t / 2], t & 1 ? HIGH : LOW);
          acc[b][t] = Elem<T>::mfma(x, hi, acc[b][t]);
          acc[b][t] = Elem<T>::mfma(x, lo, acc[b][t]);
        }
    }
  }

  // Lane i holds the addresses of 16 keys: those of part i % U of the wave's
  // step xb + i / U.
  uint32_t k_lo, k_hi, v_lo, v_hi;
  int32_t xb;
  template <class Base> __device__ void addresses(int32_t x, int32_t steps, Base &&base) {
    xb = x;
    const int32_t lane = hidden(threadIdx.x & 63);
    int32_t at = x + lane / U;
    at = at < steps ? at : steps - 1;
    const int32_t j = attn_row16(s, base(at) + 16 * (lane % U));
    int64_t page = 0, in = s.key0 + j;
    if (a.table) {
      const int32_t y = a.table[s.slot * a.table_stride + (j >> a.page_shift)];
      page = y < 0 ? 0 : y >= a.pages ? a.pages - 1 : y;
      in = j & ((1 << a.page_shift) - 1);
    }
    const uint64_t kp = (uint64_t)(uintptr_t)a.k +
                        (int64_t)sizeof(T) * (page * a.k_page + in * a.k_row + h * a.k_head);
    const uint64_t vp = (uint64_t)(uintptr_t)a.v +
                        (int64_t)sizeof(T) * (page * a.v_page + in * a.v_row + h * a.v_head);
    k_lo = (uint32_t)kp, k_hi = (uint32_t)(kp >> 32);
    v_lo = (uint32_t)vp, v_hi = (uint32_t)(vp >> 32);
  }
  // rows that may be read of the 16 from j16 on, less one
  __device__ int32_t last_of(int32_t j16) const {
    const int32_t left = s.L - 1 - attn_row16(s, j16);
    return left < 15 ? left : 15;
  }
  // The keys from L on read row L - 1, and are masked.  Aligned operands go
  // into LDS whole rows at a time (the products' layout straight from memory
  // is 64 accesses of 16 bytes a load where whole rows are 16 of 64).
  __device__ void load_keys(int32_t x, int32_t kb, uint32_t (&k)[U][KS][4]) {
    const int32_t lane = threadIdx.x & 63, piece = lane % CH, sub = lane / CH;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t base = lane_of(k_lo, k_hi, (x - xb) * U + u);
      const uint32_t stride = (uint32_t)a.k_row * sizeof(T), most = last_of(kb + 16 * u) * stride;
      if constexpr (ALIGNED) {
        const bool full = a.d == DV;
#pragma unroll
        for (int y = 0; y < 16 / RPI; ++y) {
          const int32_t r = y * RPI + sub, c = piece ^ k_swizzle<CH>(r);
          const uint32_t at = (uint32_t)r * stride, row = at < most ? at : most;
          lds_char *to = lds + (16 * u + y * RPI) * ROWB;
          if (full)
            load_to_lds(base, row + 16 * c, to);
          else if (c * KE < a.d)
            load_to_lds(base, row + 16 * c, to);
        }
      } else {
        const uint32_t at = (uint32_t)n * stride, row = at < most ? at : most;
#pragma unroll
        for (int i = 0; i < KS; ++i)
          load_row<T, 4>((const global_as T *)(base + row), (4 * i + g) * KE, a.d, k[u][i]);
      }
    }
  }
  // Elements past the head are the last ones of it: their outputs are dropped.
  __device__ void load_values(int32_t x, int32_t kb, uint32_t (&v)[U][4][NB][WV]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const global_as char *base = (const global_as char *)lane_of(v_lo, v_hi, (x - xb) * U + u);
      const uint32_t stride = (uint32_t)a.v_row * sizeof(T), most = last_of(kb + 16 * u) * stride;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t at = (uint32_t)(4 * g + i) * stride, row = at < most ? at : most;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const int32_t e = (16 * b + n) * VW;
          if constexpr (ALIGNED) {
            typedef __attribute__((ext_vector_type(WV))) uint32_t V;
            const uint32_t in = sizeof(T) * (e < a.d ? e : a.d - VW);
            const V y = *reinterpret_cast<const global_as V *>(base + (row + in));
#pragma unroll
            for (int z = 0; z < WV; ++z) v[u][i][b][z] = y[z];
          } else {
            load_row<T, WV>(reinterpret_cast<const global_as T *>(base + row), e, a.d, v[u][i][b]);
          }
        }
      }
    }
  }

  // The steps of a wave, `steps` of them, step x at key base(x).  q_lo, q_hi:
  // the smallest and largest position of the tile's rows.  The next step's
  // keys are asked for as soon as this one's are in the products and arrive
  // while the weights are computed: the compiler does not count the copies into
  // LDS, so its wait for this step's values is one for them too.  The next
  // step's values arrive during its first product.  The rest of the time to
  // memory is hidden by other waves.
  template <class Base>
  __device__ void walk(int32_t steps, int32_t q_lo, int32_t q_hi, Base &&base) {
    if (steps <= 0) return;
    if (ALIGNED && a.d < DV) {
      // pieces past the head are never loaded: they stay zero
      lds_as u32x4 *z = (lds_as u32x4 *)lds;
      for (int i = threadIdx.x & 63; i < KT * CH; i += 64) z[i] = u32x4{0, 0, 0, 0};
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    uint32_t k[U][KS][4], v[U][4][NB][WV];
    addresses(0, steps, base);
    int32_t kb = base(0);
    load_keys(0, kb, k);
    __builtin_amdgcn_sched_barrier(0);
    load_values(0, kb, v);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
    for (int32_t x = 0;;) {
      f32x4 sc[U];
      // the step's keys have arrived (its values, asked for later, may not:
      // 4 * U * NB global loads, which return in order)
      if constexpr (ALIGNED) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * U * NB) : "memory");
      scores(k, sc);
      __builtin_amdgcn_sched_barrier(0);
      const bool more = x + 1 < steps;
      const int32_t nb = more ? base(x + 1) : 0;
      if (more) {
        if (x + 1 - xb >= 64 / U) addresses(x + 1, steps, base);
        load_keys(x + 1, nb, k);
      }
      __builtin_amdgcn_sched_barrier(0);
      float p[U][4];
      // every row sees every key of most tiles
      const bool whole = kb + KT - 1 <= q_lo &&
                         (a.window <= 0 || q_hi - kb < a.window || kb + KT <= a.sinks);
      weights(kb, whole, sc, p);
      if (whole || !edge(kb, q_lo, q_hi, p, v)) weigh(p, v);
      __builtin_amdgcn_sched_barrier(0);
      if (!more) break;
      load_values(++x, nb, v);
      __builtin_amdgcn_sched_barrier(0);
      kb = nb;
    }
  }

  __device__ void scores(const uint32_t (&k)[U][KS][4], f32x4 (&sc)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      sc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        u32x4 x;
        if constexpr (ALIGNED)
          x = *(const lds_as u32x4 *)(lds + (16 * u + n) * ROWB +
                                      (((4 * i + g) ^ k_swizzle<CH>(n)) << 4));
        else
          x = u32x4{k[u][i][0], k[u][i][1], k[u][i][2], k[u][i][3]};
        const u32x4 y = {q[i][0], q[i][1], q[i][2], q[i][3]};
        if constexpr (F32) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sc[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x[e]),
                                                         __uint_as_float(y[e]), sc[u], 0, 0, 0);
        } else {
          sc[u] = Elem<T>::mfma(x, __builtin_bit_cast(typename Elem<T>::V8, y), sc[u]);
        }
      }
    }
  }

  __device__ void weights(int32_t kb, bool whole, f32x4 (&sc)[U], float (&p)[U][4]) {
    if (!whole) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!attn_sees(a, pos, kb + 16 * u + 4 * g + i)) sc[u][i] = -INFINITY;
    }
    float top = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
    if constexpr (U == 2)
      top = fmaxf(top, fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
    // The largest score is subtracted before the scale comes in: its product
    // with the scale, rounded, would be off by more than a weight's range where
    // scores pass 2^24.
    top = fmaxf(m, xor16_32_max(top));
    const float use = top == -INFINITY ? 0.f : top;
    const float fade = attn_exp2((m - use) * a.scale_log2);
    m = top;
    l *= fade;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[u][i] = attn_exp2(fmaf(sc[u][i] - use, a.scale_log2, Elem<T>::TOP));
        l += p[u][i];
      }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int t = 0; t < VW; ++t) acc[b][t] *= fade;
  }
  // A tile that not every row sees whole: what a masked place holds (memory
  // never written, for one) must not reach a sum, and 0 * NaN is NaN.  Rows of
  // V that no query row sees are cleared; if one that some rows see and some
  // do not is not finite, its keys go one at a time and each row takes only
  // those it sees (returns true).
  __device__ bool edge(int32_t kb, int32_t q_lo, int32_t q_hi, const float (&p)[U][4],
                       uint32_t (&v)[U][4][NB][WV]) {
    bool odd = false;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int32_t j = kb + 16 * u + 4 * g + i;
        // (seen by some row: the last row's side of the diagonal and the
        // first row's side of the window)
        const bool seen = j <= q_hi && (a.window <= 0 || q_lo - j < a.window || j < a.sinks);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int t = 0; t < WV; ++t) {
            v[u][i][b][t] = seen ? v[u][i][b][t] : 0u;
            odd |= not_finite<T>(v[u][i][b][t]);
          }
      }
    if (q_lo == q_hi || !__any(odd)) return false;
    one_by_one(kb, p);
    return true;
  }
  __device__ void one_by_one(int32_t kb, const float (&p)[U][4]) {
#pragma unroll 1
    for (int32_t j = 0; j < KT; ++j) {
      const int32_t at = j & 15, j16 = kb + (j & 16);
      float w = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) w = 16 * u + i == (j & ~12) ? p[u][i] : w;
      w = __shfl(w, n + 16 * (at >> 2));
      const AttnRows r = attn_rows(a, s, h, j16, attn_page(a, s, j16));
      if (!attn_sees(a, pos, kb + j)) continue;
      const T *row = static_cast<const T *>(a.v) + r.v + (at < r.last ? at : r.last) * a.v_row;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int t = 0; t < VW; ++t) {
            const int32_t e = (16 * b + 4 * g + y) * VW + t;
            if (e < a.d) acc[b][t][y] = fmaf(w, (float)row[e], acc[b][t][y]);
          }
    }
  }
  // Has a sum become NaN while the weights are numbers?  Of a weight's two
  // 16-bit parts the second is negative or zero half of the time: the products
  // of an infinite value have both signs, or are NaN.
  __device__ bool lost() const {
    bool odd = false;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int t = 0; t < VW; ++t)
#pragma unroll
        for (int i = 0; i < 4; i += 2)
          odd |= __builtin_isunordered(acc[b][t][i], acc[b][t][i + 1]);
    const float sum = xor16_32_sum(l);
    return odd && sum == sum;
  }
  // Then the steps once more, key by key on the vector unit, with weights in 32
  // bits.  (A rare path: few registers at a time, so that it takes none from
  // the others.)
  template <class Base> __device__ void by_key(int32_t steps, Base &&base) {
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int t = 0; t < VW; ++t) acc[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int32_t x = 0; x < steps * KT; ++x) {
      const int32_t j = base(x / KT) + x % KT, j16 = j & ~15;
      const bool see = attn_sees(a, pos, j);
      if (!__any(see)) continue;
      const int32_t d = hidden(a.d);
      const AttnRows r = attn_rows(a, s, h, j16, attn_page(a, s, j16));
      const T *kr = static_cast<const T *>(a.k) + r.k + (j & 15) * a.k_row;
      const T *vr = static_cast<const T *>(a.v) + r.v + (j & 15) * a.v_row;
      float sc = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int32_t e = (4 * i + g) * KE;
#pragma unroll
        for (int y = 0; y < KE; ++y)
          if (e + y < d) sc = fmaf(query(i, y), (float)kr[e + y], sc);
        __builtin_amdgcn_sched_barrier(0);
      }
      sc = xor16_32_sum(sc);
      const float top = see ? fmaxf(m, sc) : m, use = top == -INFINITY ? 0.f : top;
      const float fade = attn_exp2((m - use) * a.scale_log2);
      const float p = see ? attn_exp2(fmaf(sc - use, a.scale_log2, Elem<T>::TOP)) : 0.f;
      m = top;
      l = l * fade + (g == 0 ? p : 0.f);  // (the row's four lanes are added up later)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < VW; ++t) {
          acc[b][t] *= fade;
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int32_t e = (16 * b + 4 * g + y) * VW + t;
            if (see && e < d) acc[b][t][y] = fmaf(p, (float)vr[e], acc[b][t][y]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
    }
  }
  // element y of the query's piece i
  __device__ float query(int i, int y) const {
    typedef __attribute__((ext_vector_type(KE))) T V;
    const u32x4 w = {q[i][0], q[i][1], q[i][2], q[i][3]};
    return (float)__builtin_bit_cast(V, w)[y];
  }
};

// waves a SIMD, by the registers that the values of a step and the sums take
template <class T> constexpr int row_waves(int elems) {
  return elems * (int)sizeof(T) <= 8 ? 4 : elems * (int)sizeof(T) <= 16 ? 3 : sizeof(T) == 4 && elems == 8 ? 2 : 1;
}

template <class T> __device__ inline void store4(T *dst, const float (&x)[4], int32_t left) {
  if (left >= 4) {
    typedef __attribute__((ext_vector_type(4))) T V4;
    V4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (T)x[i];
    *reinterpret_cast<V4 *>(dst) = y;
  }
}

// One block: a row tile of one sequence and key head, over one part of its
// keys that the block's SHARE waves take in turn, or (SHARE 1) four row tiles,
// a wave each.
template <class T, int VW, int NB, int SHARE, bool ALIGNED>
__global__ __launch_bounds__(SHARE > 4 ? 64 * SHARE : 256,
                             SHARE > 4 ? SHARE / 4 : row_waves<T>(VW * NB)) void
k_attn_rows(const AttnArgs a) {
  typedef RowTile<T, VW, NB, ALIGNED> Tile;
  constexpr int DV = Tile::DV;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // key heads fastest: neighbouring blocks read neighbouring parts of a page
  uint32_t at = blockIdx.x;
  const int32_t h = at % a.kv_heads;
  at /= a.kv_heads;
  const int32_t groups = SHARE > 1 ? a.tiles : (a.tiles + 3) / 4;
  // (the last tiles see the most keys: they go first)
  const int32_t tg = groups - 1 - (int32_t)(at % groups);
  at /= groups;
  const int32_t part = at % a.splits;
  const AttnSeq s = attn_seq(a, at / a.splits);
  const int32_t tile = SHARE > 1 ? tg : 4 * tg + w;
  const int32_t row0 = tile * ROWS;
  const int32_t T_used = s.T < a.max_new ? s.T : a.max_new;
  const int32_t rows_all = T_used * a.group;
  const bool have = row0 < rows_all;
  if (SHARE > 1 ? !have : 4 * tg * ROWS >= rows_all) return;
  const int32_t rows = !have ? 0 : rows_all - row0 < ROWS ? rows_all - row0 : ROWS;
  const int32_t t_lo = row0 / a.group, t_hi = (row0 + rows - 1) / a.group;
  const int32_t q_lo = s.L - s.T + t_lo, q_hi = s.L - s.T + t_hi;
  const auto span = attn_span<Tile::KT, Tile::KT>(a, q_lo, have ? q_hi : -1);
  const int32_t parts = attn_parts(a, span.tiles);
  if (part >= parts) return;
  const int32_t first = part * a.chunk + (SHARE > 1 ? w : 0);
  const int32_t end = part == parts - 1 ? span.tiles : (part + 1) * a.chunk;

  // the waves' keys and, after them, their sums: four waves' at a time
  constexpr int SLOTS = 4, SUMB = SHARE > 1 ? SLOTS * ROWS * (DV + 4) * 4 : 0;
  constexpr int KEYB = ALIGNED ? (SHARE > 4 ? SHARE : 4) * Tile::KT * Tile::ROWB : 16;
  __shared__ __attribute__((aligned(1024))) char pool[KEYB > SUMB ? KEYB : SUMB];
  Tile tl(a, s, h, lane, (lds_char *)pool + (ALIGNED ? w * Tile::KT * Tile::ROWB : 0));
  tl.begin(have ? row0 + tl.n : 0x3fffffff);
  const auto base = [&](int32_t x) { return span.base(first + SHARE * x); };
  const int32_t steps = (end - first + SHARE - 1) / SHARE;
  tl.walk(steps, q_lo, q_hi, base);
  {
    // (the lane's place anew)
    const int32_t tid = hidden(threadIdx.x);
    tl.n = tid & 15, tl.g = (tid >> 4) & 3;
  }
  if constexpr (!Tile::F32)
    if (__any(tl.lost())) tl.by_key(steps, base);
  tl.l = xor16_32_sum(tl.l);

  const bool partial = parts > 1;
  const int32_t group = hidden(a.group);
  const int64_t row_of = (int64_t)part * a.tokens * a.heads;
  if constexpr (SHARE == 1) {
    if (tl.n < rows) {
      const int32_t r = row0 + tl.n;
      const int64_t token = s.token0 + r / group;
      const int32_t head = h * group + r % group;
      const float inv = tl.l > 0.f || tl.l != tl.l ? 1.f / tl.l : 0.f;
      T *dst = static_cast<T *>(a.out) + token * a.o_row + head * a.o_head;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int32_t e = 16 * VW * b + VW * (4 * tl.g + i);
#pragma unroll
          for (int t0 = 0; t0 < VW; t0 += 4) {
            float x[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) x[t] = tl.acc[b][t0 + t][i] * inv;
            if constexpr (ALIGNED)
              store4<T>(dst + e + t0, x, a.d - e - t0);
            else
#pragma unroll
              for (int t = 0; t < 4; ++t)
                if (e + t0 + t < a.d) dst[e + t0 + t] = (T)x[t];
          }
        }
      if (a.lse && tl.g == 0)
        a.lse[token * a.heads + head] =
            attn_lse(tl.m * a.scale_log2 - Elem<T>::TOP, tl.l);
    }
  } else {
    typedef float Sums[ROWS][DV + 4];
    Sums *so = reinterpret_cast<Sums *>(pool);
    __shared__ float sm[SHARE][ROWS], sl[SHARE][ROWS];
    if (tl.g == 0) sm[w][tl.n] = tl.m, sl[w][tl.n] = tl.l;
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int x = 0; x < SHARE; ++x) top = fmaxf(top, sm[x][tl.n]);
    const float use = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int x = 0; x < SHARE; ++x)
      sum += sl[x][tl.n] * attn_exp2((sm[x][tl.n] - use) * a.scale_log2);
    // rows of a part: the sums with weights up to 1; of the whole: the quotient
    constexpr float ONE = Elem<T>::TOP > 0.f ? 1.f / 32768.f : 1.f;  // 2^-TOP
    float f = attn_exp2((tl.m - use) * a.scale_log2);
    f *= partial ? ONE : sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
    for (int turn = 0; turn < (SHARE + SLOTS - 1) / SLOTS; ++turn) {
      if (w / SLOTS == turn && tl.n < rows) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < VW; t += 4) {
              f32x4 x;
#pragma unroll
              for (int y = 0; y < 4; ++y) x[y] = tl.acc[b][t + y][i] * f;
              f32x4 *to = reinterpret_cast<f32x4 *>(
                  &so[w % SLOTS][tl.n][16 * VW * b + VW * (4 * tl.g + i) + t]);
              *to = turn ? *to + x : x;
            }
      }
      __syncthreads();
    }
    if (w == 0 && tl.g == 0 && tl.n < rows) {
      const int32_t r = row0 + tl.n;
      const int64_t row = (s.token0 + r / group) * a.heads + h * group + r % group;
      if (partial) {
        a.part_ml[2 * (row_of + row)] = top;
        a.part_ml[2 * (row_of + row) + 1] = sum * ONE;
      } else if (a.lse) {
        a.lse[row] = attn_lse(top * a.scale_log2 - Elem<T>::TOP, sum);
      }
    }
    for (int32_t x = threadIdx.x; x < rows * (DV / 4); x += 64 * SHARE) {
      const int32_t rr = x / (DV / 4), e = 4 * (x % (DV / 4));
      if (e >= a.d) continue;
      f32x4 y = *reinterpret_cast<f32x4 *>(&so[0][rr][e]);
#pragma unroll
      for (int z = 1; z < SLOTS; ++z) y += *reinterpret_cast<f32x4 *>(&so[z][rr][e]);
      const int32_t r = row0 + rr;
      const int64_t token = s.token0 + r / group;
      const int32_t head = h * group + r % group;
      if (partial) {
        float *dst = a.part_o + (row_of + token * a.heads + head) * DV + e;
        *reinterpret_cast<f32x4 *>(dst) = y;
      } else {
        T *dst = static_cast<T *>(a.out) + token * a.o_row + head * a.o_head + e;
        const float z[4] = {y[0], y[1], y[2], y[3]};
        if constexpr (ALIGNED)
          store4<T>(dst, z, a.d - e);
        else
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (e + t < a.d) dst[t] = (T)z[t];
      }
    }
  }
}

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
  const AttnSeq s = attn_seq(a, block / per);
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
