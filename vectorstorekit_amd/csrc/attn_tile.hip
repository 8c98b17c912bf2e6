// attn_tile.hip -- attention of many query rows in 16 bits: 32 rows a wave,
// eight (four) waves a workgroup, keys and values shared through LDS.
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
// The weights are rounded to the type of V before the second product, with an
// error of the size of the output's own rounding; sums stay in fp32.
#include "attn.hpp"
#include "vsk_api.hpp"

namespace vsk {

namespace {

constexpr int KT = 64;  // keys of a tile

typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((address_space(3))) char lds_char;

template <class T> struct Mm;
template <> struct Mm<__bf16> {
  typedef bf16x8 V8;
  static constexpr uint32_t EXP = 0x7F807F80u;
  static __device__ f32x16 mfma(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mm<_Float16> {
  typedef f16x8 V8;
  static constexpr uint32_t EXP = 0x7C007C00u;
  static __device__ f32x16 mfma(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// The slot of a row's 16-byte piece c is c ^ swizzle(row).  K: the eight
// (sixteen) rows that a quarter (half) of a wave reads the same piece of go to
// different slots; V: the four rows of a transposing read.
template <int CH> __device__ inline int k_swizzle(int row) {
  return CH >= 16 ? row & 15 : (row & 7) ^ ((row >> 3) & 1);
}
template <int CH> __device__ inline int v_swizzle(int row) {
  const int x = row & 3;
  return CH >= 16 ? 4 * x + 2 * (x >> 1) : 2 * x;
}

// 16 bytes a lane from src to dst + 16 * lane (dst the same in every lane).
// Written as assembly because the compiler makes every read of LDS after the
// builtin wait for it: here a tile's copies fly while the last tile is
// computed with, and one wait before the barrier covers them.  (M0 holds the
// destination of such loads; nothing else in these kernels uses it.)
__device__ inline void load_to_lds(const void *src, const void *dst) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)dst);
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off"
      :
      : "s"(at), "v"(src)
      : "memory");
}

template <class T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, DP == 256 ? 1 : 2) void k_attn_tile(const AttnArgs a) {
  typedef typename Mm<T>::V8 V8;
  constexpr int CH = DP / 8;         // 16-byte pieces of a row
  constexpr int ROWB = 2 * DP;       // bytes of a row
  constexpr int TILEB = KT * ROWB;   // bytes of a tile
  constexpr int RPI = 64 / CH;       // rows that one load of a wave brings
  constexpr int MINE = KT / NW;      // rows of a tile that a wave brings
  constexpr int KS = DP / 16, DT = DP / 32;
  __shared__ __attribute__((aligned(1024))) char kbuf[2][TILEB];
  __shared__ __attribute__((aligned(1024))) char vbuf[2][TILEB];

  const int lane = threadIdx.x & 63, h2 = lane >> 5, n = lane & 31;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t at = blockIdx.x;
  const int32_t h = at % a.kv_heads;
  at /= a.kv_heads;
  const int32_t tile = a.tiles - 1 - (int32_t)(at % a.tiles);
  at /= a.tiles;
  const int32_t part = at % a.splits;
  const AttnSeq s = attn_seq(a, at / a.splits);
  const int32_t row0 = tile * 32 * NW;
  const int32_t T_used = s.T < a.max_new ? s.T : a.max_new;
  const int32_t rows_all = T_used * a.group;
  if (row0 >= rows_all) return;
  const int32_t last = row0 + 32 * NW < rows_all ? row0 + 32 * NW - 1 : rows_all - 1;
  const int32_t p0 = s.L - s.T;
  const AttnSpan<KT> span = attn_span<KT>(a, p0 + row0 / a.group, p0 + last / a.group);
  const int32_t parts = attn_parts(a, span.tiles);
  if (part >= parts) return;
  const int32_t first = part * a.chunk;
  const int32_t end = part == parts - 1 ? span.tiles : first + a.chunk;

  // this wave's rows and what they see
  const int32_t w0 = row0 + 32 * w, w1 = w0 + 31 < last ? w0 + 31 : last;
  const bool have = w0 <= last;
  const int32_t q_lo = p0 + w0 / a.group, q_hi = have ? p0 + w1 / a.group : -1;
  const int32_t row = w0 + n;
  const bool real = row <= last;
  const int32_t t = row / a.group, head = h * a.group + row - t * a.group;
  const int32_t pos = real ? p0 + t : -1;

  V8 q[KS];
  {
    const T *src = static_cast<const T *>(a.q) + (real ? (s.token0 + t) * a.q_row + head * a.q_head : 0);
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      q[i] = V8{};
      if (real && 16 * i + 8 * h2 < a.d) q[i] = *reinterpret_cast<const V8 *>(src + 16 * i + 8 * h2);
    }
  }
  if (a.d < DP) {
    // pieces past the head are never loaded: they stay zero
    u32x4 *z = reinterpret_cast<u32x4 *>(kbuf), *y = reinterpret_cast<u32x4 *>(vbuf);
    for (int i = threadIdx.x; i < 2 * TILEB / 16; i += 64 * NW) z[i] = y[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
  }

  f32x16 acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = f32x16{};
  float m = -INFINITY, l = 0.f;

  // brings the wave's rows of a tile
  const int piece = lane % CH, sub = lane / CH;
  auto fetch = [&](int32_t i, int buf) {
    const int32_t j0 = span.base(i) + MINE * w;
    const AttnRows r = attn_rows(a, s, h, j0 & ~15);
#pragma unroll
    for (int x = 0; x < MINE / RPI; ++x) {
      const int lr = MINE * w + x * RPI + sub;  // the row within the tile
      const int off = (j0 & 15) + x * RPI + sub;
      const int32_t rr = off < r.last ? off : r.last;
      const int kc = piece ^ k_swizzle<CH>(lr), vc = piece ^ v_swizzle<CH>(lr);
      const T *ks = static_cast<const T *>(a.k) + r.k + rr * (int32_t)a.k_row + 8 * kc;
      const T *vs = static_cast<const T *>(a.v) + r.v + rr * (int32_t)a.v_row + 8 * vc;
      const int at = (MINE * w + x * RPI) * ROWB;
      if (8 * kc < a.d) load_to_lds(ks, kbuf[buf] + at);
      if (8 * vc < a.d) load_to_lds(vs, vbuf[buf] + at);
    }
  };

  // lane's parts of the addresses of the reads
  const int kx = h2 ^ k_swizzle<CH>(n);
  const int gi = lane & 15, va = gi >> 2, vhalf = (lane >> 4) & 1;
  const int vrow = (4 * h2 + va) * ROWB + 8 * (gi & 1);
  const int vx = (2 * vhalf + ((gi & 3) >> 1)) ^ v_swizzle<CH>(va);

  if (first < end) fetch(first, 0);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
  for (int32_t i = first; i < end; ++i) {
    const int cur = (i - first) & 1;
    if (i + 1 < end) fetch(i + 1, cur ^ 1);
    const int32_t kb = span.base(i);
    // (a wave whose rows see none of the tile only brings its rows)
    const bool any = kb <= q_hi && (a.window <= 0 || q_lo - (kb + KT - 1) < a.window || kb < a.sinks);
    if (any) {
      const char *kt = kbuf[cur] + n * ROWB;
      f32x16 sc[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        sc[u] = f32x16{};
#pragma unroll
        for (int x = 0; x < KS; ++x) {
          const V8 k = *reinterpret_cast<const V8 *>(kt + 32 * u * ROWB + (((2 * x) ^ kx) << 4));
          sc[u] = Mm<T>::mfma(k, q[x], sc[u]);
        }
      }
      const bool whole = kb + KT - 1 <= q_lo &&
                         (a.window <= 0 || q_hi - kb < a.window || kb + KT <= a.sinks);
      bool odd = false;
      if (!whole) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (!attn_sees(a, pos, kb + 32 * u + 8 * (x >> 2) + 4 * h2 + (x & 3)))
              sc[u][x] = -INFINITY;
        // is every value of the tile finite?  (largest exponent field)
        typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
        u16x2 top = {0, 0};
        const u32x4 *vt = reinterpret_cast<const u32x4 *>(vbuf[cur]);
#pragma unroll 4
        for (int x = lane; x < TILEB / 16; x += 64) {
          const u32x4 y = vt[x];
#pragma unroll
          for (int z = 0; z < 4; ++z)
            top = __builtin_elementwise_max(
                top, __builtin_bit_cast(u16x2, y[z] & Mm<T>::EXP));
        }
        const unsigned short inf = (unsigned short)(Mm<T>::EXP & 0xFFFF);
        odd = __any(top[0] == inf || top[1] == inf);
      }
      float tm = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int x = 0; x < 16; x += 2) tm = fmaxf(tm, fmaxf(sc[u][x], sc[u][x + 1]));
      tm = fmaxf(tm, __shfl_xor(tm, 32));
      const float nm = fmaxf(m, tm * a.scale_log2);
      const float use = nm == -INFINITY ? 0.f : nm;
      const float fade = attn_exp2(m - use);
      m = nm;
      l *= fade;
#pragma unroll
      for (int x = 0; x < DT; ++x) acc[x] *= fade;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          sc[u][x] = attn_exp2(fmaf(sc[u][x], a.scale_log2, -use));
          l += sc[u][x];
        }
      if (!odd) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          V8 p;
#pragma unroll
          for (int x = 0; x < 8; ++x) p[x] = (T)sc[u >> 1][8 * (u & 1) + x];
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const char *vt = vbuf[cur] + vrow + 16 * u * ROWB + (((4 * dt) ^ vx) << 4);
            union {
              i16x4 half[2];
              V8 v;
            } f;
            f.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4 *)(lds_char *)vt);
            f.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4 *)(lds_char *)(vt + 8 * ROWB));
            acc[dt] = Mm<T>::mfma(f.v, p, acc[dt]);
          }
        }
      } else {
        // a value that is not finite, in a tile that not every row sees whole:
        // its keys one at a time, each row takes only those it sees
#pragma unroll 1
        for (int j = 0; j < KT; ++j) {
          float wt = 0.f;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int x = 0; x < 16; ++x)
              wt = 32 * u + 8 * (x >> 2) + (x & 3) == (j & ~4) ? sc[u][x] : wt;
          wt = __shfl(wt, n + 32 * ((j >> 2) & 1));
          if (!attn_sees(a, pos, kb + j)) continue;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const int c = 4 * dt + b;
              const T *v = reinterpret_cast<const T *>(vbuf[cur] + j * ROWB +
                                                       ((c ^ v_swizzle<CH>(j)) << 4)) + 4 * h2;
#pragma unroll
              for (int x = 0; x < 4; ++x)
                acc[dt][4 * b + x] = fmaf(wt, (float)v[x], acc[dt][4 * b + x]);
            }
        }
      }
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the next tile has arrived
    __syncthreads();
  }

  l += __shfl_xor(l, 32);
  if (!real) return;
  const int64_t out_row = (s.token0 + t) * a.heads + head;
  if (parts > 1) {
    const int64_t r = (int64_t)part * a.tokens * a.heads + out_row;
    float *dst = a.part_o + r * DP;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        *reinterpret_cast<f32x4 *>(dst + 32 * dt + 8 * b + 4 * h2) =
            f32x4{acc[dt][4 * b], acc[dt][4 * b + 1], acc[dt][4 * b + 2], acc[dt][4 * b + 3]};
    if (h2 == 0) {
      a.part_ml[2 * r] = m;
      a.part_ml[2 * r + 1] = l;
    }
    return;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  T *dst = static_cast<T *>(a.out) + (s.token0 + t) * a.o_row + head * a.o_head;
  typedef __attribute__((ext_vector_type(4))) T V4;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int e = 32 * dt + 8 * b + 4 * h2;
      V4 y;
#pragma unroll
      for (int x = 0; x < 4; ++x) y[x] = (T)(acc[dt][4 * b + x] * inv);
      if (e < a.d) *reinterpret_cast<V4 *>(dst + e) = y;
    }
  if (a.lse && h2 == 0)
    a.lse[out_row] = l > 0.f ? (m + __log2f(l)) * 0.6931471805599453f : l != l ? l : -INFINITY;
}

template <class T> void tile_of(hipStream_t st, const AttnArgs &a, int nw, unsigned g) {
  if (a.d <= 64) {
    if (nw == 8)
      k_attn_tile<T, 64, 8><<<g, 512, 0, st>>>(a);
    else
      k_attn_tile<T, 64, 4><<<g, 256, 0, st>>>(a);
  } else if (a.d <= 128) {
    if (nw == 8)
      k_attn_tile<T, 128, 8><<<g, 512, 0, st>>>(a);
    else
      k_attn_tile<T, 128, 4><<<g, 256, 0, st>>>(a);
  } else {
    k_attn_tile<T, 256, 4><<<g, 256, 0, st>>>(a);
  }
}

}  // namespace

void launch_attn_tile(vsk_ctx *ctx, hipStream_t st, const AttnArgs &a, int32_t t, int32_t nw) {
  const int64_t grid = (int64_t)a.n * a.splits * a.tiles * a.kv_heads;
  VSK_REQUIRE(grid <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "too many query rows in one call");
  KernelTimer kt(ctx, "attn_tile", (double)a.tokens * a.heads, st);
  if (t == VSK_DTYPE_F16)
    tile_of<_Float16>(st, a, nw, (unsigned)grid);
  else
    tile_of<__bf16>(st, a, nw, (unsigned)grid);
  check_launch("attn_tile");
}

}  // namespace vsk
