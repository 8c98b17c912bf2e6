// attn_rows.hpp -- attention over 16 query rows a wave, as the kernels of
// attn_rows.hip (which says how) and attn_forms.hip compute it.
#pragma once

#include "attn.hpp"

namespace vsk {

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
template <class T, int VW, int NB, bool ALIGNED, AttnForm F> struct RowTile {
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
    pos = real ? attn_position<F>(a, s, t) : -1;
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
      const int32_t y = a.table[s.row + (j >> a.page_shift)];
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

// LDS of a block: the waves' keys and, after them, their sums (four waves' at a
// time), then each row's largest scores and sums of weights.
template <class T, int VW, int NB, int SHARE, bool ALIGNED> struct RowsLds {
  static constexpr int DV = 16 * VW * NB, SLOTS = 4;
  static constexpr int SUMB = SHARE > 1 ? SLOTS * ROWS * (DV + 4) * 4 : 0;
  static constexpr int KEYB =
      ALIGNED ? (SHARE > 4 ? SHARE : 4) * 16 * SUBS<T> * DV * (int)sizeof(T) : 16;
  static constexpr int POOL = KEYB > SUMB ? KEYB : SUMB;
  static constexpr int BYTES = POOL + (SHARE > 1 ? 2 * SHARE * ROWS * 4 : 0);
};

// One block: a row tile of one sequence and key head, over one part of its
// keys that the block's SHARE waves take in turn, or (SHARE 1) four row tiles,
// a wave each.
template <class T, int VW, int NB, int SHARE, bool ALIGNED, AttnForm F>
__device__ __forceinline__ void attn_rows_block(const AttnArgs &a, uint32_t at, char *pool) {
  typedef RowTile<T, VW, NB, ALIGNED, F> Tile;
  typedef RowsLds<T, VW, NB, SHARE, ALIGNED> Lds;
  constexpr int DV = Tile::DV, SLOTS = Lds::SLOTS;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // key heads fastest: neighbouring blocks read neighbouring parts of a page
  const int32_t h = at % a.kv_heads;
  at /= a.kv_heads;
  const int32_t groups = SHARE > 1 ? a.tiles : (a.tiles + 3) / 4;
  // (the last tiles see the most keys: they go first)
  const int32_t tg = groups - 1 - (int32_t)(at % groups);
  at /= groups;
  const auto [b, part] = attn_turn<F>(a, at);
  const AttnSeq s = attn_seq<F>(a, b);
  const int32_t tile = SHARE > 1 ? tg : 4 * tg + w;
  const int32_t row0 = tile * ROWS;
  const int32_t T_used = s.T < a.max_new ? s.T : a.max_new;
  const int32_t rows_all = T_used * a.group;
  const bool have = row0 < rows_all;
  if (SHARE > 1 ? !have : 4 * tg * ROWS >= rows_all) return;
  const int32_t rows = !have ? 0 : rows_all - row0 < ROWS ? rows_all - row0 : ROWS;
  const int32_t t_lo = row0 / a.group, t_hi = (row0 + rows - 1) / a.group;
  int32_t q_lo = s.p0 + (t_lo & s.each), q_hi = s.p0 + (t_hi & s.each);
  if (F && SHARE > 1 && a.groups) {
    // (rows of several sequences)
    const int32_t r = (lane & 15) < rows ? row0 + (lane & 15) : row0;
    q_lo = q_hi = attn_position<F>(a, s, r / a.group);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      q_lo = min(q_lo, __shfl_xor(q_lo, o));
      q_hi = max(q_hi, __shfl_xor(q_hi, o));
    }
    q_lo = __builtin_amdgcn_readfirstlane(q_lo), q_hi = __builtin_amdgcn_readfirstlane(q_hi);
  }
  const auto span = attn_span<Tile::KT, Tile::KT>(a, q_lo, have ? q_hi : -1);
  const int32_t parts = attn_parts(a, span.tiles);
  if (part >= parts) {
    if (F && SHARE > 1 && a.joined && (int32_t)threadIdx.x < rows)
      attn_empty_part(a, s, h, row0 + threadIdx.x, part);
    return;
  }
  const int32_t first = part * a.chunk + (SHARE > 1 ? w : 0);
  const int32_t end = part == parts - 1 ? span.tiles : (part + 1) * a.chunk;

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

  const bool partial = parts > 1 || (F && a.joined);
  const int32_t group = hidden(a.group);
  const int64_t row_of = (int64_t)(F ? a.part0 + part : part) * a.tokens * a.heads;
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
    typedef float Ends[ROWS];
    Sums *so = reinterpret_cast<Sums *>(pool);
    Ends *sm = reinterpret_cast<Ends *>(pool + Lds::POOL), *sl = sm + SHARE;
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

constexpr int rows_threads(int share) { return share > 4 ? 64 * share : 256; }
template <class T> constexpr int rows_waves(int share, int elems) {
  return share > 4 ? share / 4 : row_waves<T>(elems);
}

}  // namespace vsk
