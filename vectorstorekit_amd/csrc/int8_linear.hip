// int8_linear.hip -- a linear layer in 8-bit integers: activations quantised
// for each token, weights for each output channel.
//
//   s_m = max_k |x_mk| / 127      c_mk = rint(x_mk * (127 / max_k |x_mk|))
//   y_mn = s_m t_n sum_k c_mk w_nk + b_n
//
// The sums are 32-bit integers and exact: their order changes nothing.
//
// Both operands are kept in the order that the matrix cores read: blocks of 32
// rows and 32 inner places, 1 KB each, in which lane l of a wave has 16 bytes
// of row l % 32 from place 16 * (l / 32) on; a row block's blocks follow each
// other along the inner dimension, which is filled up to a multiple of 64.  A
// block is one load of a wave, contiguous in memory and in LDS, with no bank
// met twice.  Weights are brought into that order once, activations by the
// kernel that quantises them.
//
// What bounds it: few tokens, the weights' bytes and the launches (one token
// through 4,096 x 4,096 5.7 us, 64 through 4,096 x 12,288 14.5, of which the
// weights alone are 8.7 at 5.8 TB/s); many, the matrix cores: 16,384 tokens
// through 4,096 x 12,288 take 43 us to quantise and 700 for the products, 2,350
// TOPS, at which the card holds its power limit and 1.8 GHz.
#include <type_traits>

#include "attn.hpp"
#include "vsk_api.hpp"

namespace vsk {

namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(16))) int i32x16;

constexpr int BLOCK = 1024;       // bytes of a 32 x 32 block
constexpr int FILL = 2;           // the inner dimension is filled up to so many blocks
constexpr int32_t MOST = 131072;  // inner places whose sums (128 * 127 each) fit 32 bits

int64_t inner_blocks(int64_t k) { return ceil_div(k, 32 * FILL) * FILL; }
int64_t packed_bytes(int64_t rows, int64_t k) {
  return ceil_div(rows, 32) * inner_blocks(k) * BLOCK;
}

// ------------------------------------------------------------------ quantising

// 16 values of a row, as they are in memory
template <class T> struct Piece {
  static constexpr int W = 16 / sizeof(T);
  typedef __attribute__((ext_vector_type(W))) T V;
  V v[16 / W];
  __device__ float operator[](int i) const { return (float)v[i / W][i % W]; }
};
// those from element e on, zero past the end
template <class T, bool ALIGNED>
__device__ inline void load16(const T *row, int32_t e, int32_t k, Piece<T> &x) {
  constexpr int W = Piece<T>::W;
  if (ALIGNED && e + 16 <= k) {
#pragma unroll
    for (int i = 0; i < 16 / W; ++i)
      x.v[i] = *reinterpret_cast<const typename Piece<T>::V *>(row + e + W * i);
    return;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) x.v[i / W][i % W] = e + i < k ? row[e + i] : (T)0.f;
}

// What a row's codes are made with.  The largest magnitude is compared as its
// bits, so that an infinity or NaN is the largest: such a row has codes 0 and
// the scale NaN.  Rows of tiny numbers are first made larger by 2^100, so that
// 127 over their largest is finite.
struct RowScale {
  float up, inverse, scale;
};
__device__ inline RowScale row_scale(uint32_t top) {
  RowScale r;
  const float t = __uint_as_float(top);
  r.up = t < 0x1p-100f ? 0x1p100f : 1.f;
  r.inverse = top == 0 || top >= 0x7F800000u ? 0.f : 127.f / (t * r.up);
  r.scale = top >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : t / 127.f;
  return r;
}
__device__ inline uint32_t code(float x, const RowScale &r) {
  // (the largest is 127 times 1 + 2^-22 at most; NaN times 0 is not taken)
  return (r.inverse == 0.f ? 0 : (int)__builtin_rintf(x * r.up * r.inverse)) & 255;
}

struct PackArgs {
  const void *x;
  int64_t x_row, rows;
  char *packed;
  float *scales;
  int32_t k, blocks;  // inner places, inner blocks
};

template <class T> __device__ inline uint32_t magnitude(const Piece<T> &x) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t b = __float_as_uint(x[i]) & 0x7FFFFFFFu;
    top = b > top ? b : top;
  }
  return top;
}

template <class T> __device__ inline u32x4 code16(const Piece<T> &y, const RowScale &r) {
  u32x4 c;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c[i] = code(y[4 * i], r) | code(y[4 * i + 1], r) << 8 | code(y[4 * i + 2], r) << 16 |
           code(y[4 * i + 3], r) << 24;
  return c;
}

// the largest magnitude of a row whose pieces of 16 places a lane takes `step`
// apart from `at` on; the first HELD of them stay in registers
template <class T, bool ALIGNED, int HELD>
__device__ inline uint32_t largest(const T *x, int32_t k, int pieces, int at, int step,
                                   Piece<T> (&held)[HELD]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int p = at + step * i;
    if (p < pieces) load16<T, ALIGNED>(x, 16 * p, k, held[i]);
  }
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (at + step * i < pieces) {
      const uint32_t t = magnitude(held[i]);
      top = t > top ? t : top;
    }
  for (int p = at + step * HELD; p < pieces; p += step) {
    Piece<T> y;
    load16<T, ALIGNED>(x, 16 * p, k, y);
    const uint32_t t = magnitude(y);
    top = t > top ? t : top;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t t = __shfl_xor(top, o);
    top = t > top ? t : top;
  }
  return top;
}

template <class T> constexpr int HELD_PIECES = sizeof(T) == 4 ? 4 : 8;

// Few rows: a workgroup a row.
template <class T, bool ALIGNED>
__global__ __launch_bounds__(256) void k_int8_quantize_row(const PackArgs a) {
  constexpr int HELD = HELD_PIECES<T>;
  const int64_t row = blockIdx.x;
  const int pieces = 2 * a.blocks;
  const T *x = static_cast<const T *>(a.x) + row * a.x_row;
  Piece<T> held[HELD];
  uint32_t top = largest<T, ALIGNED, HELD>(x, a.k, pieces, threadIdx.x, 256, held);
  __shared__ uint32_t tops[4];
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) top = tops[i] > top ? tops[i] : top;
  const RowScale r = row_scale(top);
  if (threadIdx.x == 0) a.scales[row] = r.scale;
  char *to = a.packed + (row >> 5) * a.blocks * BLOCK + (row & 31) * 16;
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int p = threadIdx.x + 256 * i;
    if (p < pieces)
      *reinterpret_cast<u32x4 *>(to + (int64_t)(p >> 1) * BLOCK + (p & 1) * 512) =
          code16(held[i], r);
  }
  for (int p = threadIdx.x + 256 * HELD; p < pieces; p += 256) {
    Piece<T> y;
    load16<T, ALIGNED>(x, 16 * p, a.k, y);
    *reinterpret_cast<u32x4 *>(to + (int64_t)(p >> 1) * BLOCK + (p & 1) * 512) = code16(y, r);
  }
}

// Many rows: eight a workgroup, a wave each.  Their codes leave by way of LDS, so
// that a store has whole lines.  The values wait for their row's largest in the
// type that they came in: as 32-bit numbers they leave room for half as many
// waves (16,384 tokens of 4,096 in bf16 58 us, so 43; read and written at a
// copy's rate it would be 39).
constexpr int PACK_ROWS = 8;
template <class T, bool ALIGNED>
__global__ __launch_bounds__(64 * PACK_ROWS) void k_int8_quantize(const PackArgs a) {
  constexpr int HELD = HELD_PIECES<T>;
  __shared__ __attribute__((aligned(16))) u32x4 codes[2][64 * PACK_ROWS];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t row0 = (int64_t)blockIdx.x * PACK_ROWS, row = row0 + w;
  const int pieces = 2 * a.blocks;
  const bool real = row < a.rows;
  const T *x = static_cast<const T *>(a.x) + (real ? row * a.x_row : 0);
  const int32_t k = real ? a.k : 0;
  Piece<T> held[HELD];
  const RowScale r = row_scale(largest<T, ALIGNED, HELD>(x, k, pieces, lane, 64, held));
  if (real && lane == 0) a.scales[row] = r.scale;
  char *to = a.packed + (row0 >> 5) * a.blocks * BLOCK + (row0 & 31) * 16;
  // 64 pieces of the eight rows: piece p of row y is in slot y ^ (p % 8) of its eight
  auto put = [&](int i, const Piece<T> &y) {
    u32x4 *buf = codes[i & 1];
    buf[lane * 8 + (w ^ (lane & 7))] = code16(y, r);
    __syncthreads();  // (the other buffer's readers have passed the one before)
    const int z = threadIdx.x >> 3, q = threadIdx.x & 7, p = 64 * i + z;
    if (p < pieces && row0 + q < a.rows)
      *reinterpret_cast<u32x4 *>(to + (int64_t)(p >> 1) * BLOCK + (p & 1) * 512 + 16 * q) =
          buf[z * 8 + (q ^ (z & 7))];
  };
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (64 * i < pieces) put(i, held[i]);
  for (int i = HELD; 64 * i < pieces; ++i) {
    Piece<T> y;
    load16<T, ALIGNED>(x, 16 * (64 * i + lane), k, y);
    put(i, y);
  }
}

// codes of the caller's own, a row a wave
__global__ __launch_bounds__(256) void k_int8_pack(const PackArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const int8_t *x = static_cast<const int8_t *>(a.x) + row * a.x_row;
  char *to = a.packed + (row >> 5) * a.blocks * BLOCK + (row & 31) * 16;
  for (int p = threadIdx.x & 63; p < 2 * a.blocks; p += 64) {
    u32x4 c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int32_t e = 16 * p + 4 * i + j;
        w |= (uint32_t)(uint8_t)(e < a.k ? x[e] : 0) << (8 * j);
      }
      c[i] = w;
    }
    *reinterpret_cast<u32x4 *>(to + (int64_t)(p >> 1) * BLOCK + (p & 1) * 512) = c;
  }
}

// -------------------------------------------------------------------- products

struct LinearArgs {
  const char *w, *x;  // packed weights (channels) and activations (tokens)
  const float *w_scales, *x_scales, *bias;
  void *out;
  int64_t out_row, tokens;
  int32_t outputs;
  int32_t blocks;       // inner blocks of both
  int32_t w_blocks;     // row blocks of the weights
  int64_t x_blocks;     // row blocks of the activations
  int32_t tiles_n;      // tiles along the channels
  bool wide;            // the outputs take 16-byte stores
};

// (the weights' scale first: a large token's scale alone could take a sum past f32)
__device__ inline float scaled(int sum, float xs, float ws, float bias) {
  return (float)sum * ws * xs + bias;
}

// A tile of 64 FN channels and 64 FM tokens, four waves of FN x FM products of
// 32 x 32: lane l has token l % 32 and, in register 4 q + i, channel
// 8 q + 4 (l / 32) + i.
template <class T, int FN, int FM, int STEP, int STAGES>
__global__ __launch_bounds__(256, FN * FM >= 16 ? 1 : 2) void k_int8_tile(const LinearArgs a) {
  constexpr int ROWS = 2 * (FN + FM);            // row blocks of a stage
  constexpr int STAGE = ROWS * STEP * BLOCK;     // bytes of it
  constexpr int LOADS = ROWS * STEP / 4;         // blocks of it that a wave brings
  static_assert(ROWS * STEP % 4 == 0 && STEP % 2 == 0 && FILL % STEP == 0, "");
  constexpr int PITCH = FN * 32 * 4 + 16;        // of a token's sums in LDS, in bytes
  constexpr int OUT = 4 * 32 * PITCH;
  __shared__ __attribute__((aligned(1024))) char lds_pool[STAGES * STAGE > OUT ? STAGES * STAGE : OUT];
  lds_char *const lds = (lds_char *)lds_pool;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = w & 1, wm = w >> 1;
  const int32_t tn = blockIdx.x % a.tiles_n;
  const int64_t tm = blockIdx.x / a.tiles_n;
  // the blocks that this wave brings: the channels' first
  uint64_t base[LOADS];
#pragma unroll
  for (int x = 0; x < LOADS; ++x) {
    const int r = (LOADS * w + x) / STEP, j = (LOADS * w + x) % STEP;
    if (r < 2 * FN) {
      const int32_t b = 2 * FN * tn + r;
      base[x] = (uint64_t)(uintptr_t)a.w +
                ((int64_t)(b < a.w_blocks ? b : a.w_blocks - 1) * a.blocks + j) * BLOCK;
    } else {
      const int64_t b = 2 * FM * tm + r - 2 * FN;
      base[x] = (uint64_t)(uintptr_t)a.x +
                ((b < a.x_blocks ? b : a.x_blocks - 1) * a.blocks + j) * BLOCK;
    }
  }
  const int32_t steps = a.blocks / STEP;
  // one of the loads that bring step s, in order of s: the addresses go along
  auto bring = [&](int32_t s, int x) {
    load_to_lds(base[x], 16 * lane, lds + (s % STAGES) * STAGE + (LOADS * w + x) * BLOCK);
    base[x] += STEP * BLOCK;
  };
  i32x4 f[2][FN + FM];
  // operand x of the step's inner block j
  auto read = [&](int32_t s, int j, int x) {
    const int r = x < FN ? FN * wn + x : 2 * FN + FM * wm + x - FN;
    return *(const lds_as i32x4 *)(lds + (s % STAGES) * STAGE + (r * STEP + j) * BLOCK + 16 * lane);
  };
  i32x16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = i32x16{};
  // The products of one inner block, with beside them, a piece after each
  // product, the reads of the next block's operands and the loads of a later
  // step (left to itself the compiler puts all of them before).
  constexpr int PRODUCTS = FN * FM, PIECES_MAX = FN + FM > LOADS ? FN + FM : LOADS;
  auto multiply = [&](const i32x4 (&g)[FN + FM], auto &&piece) {
    constexpr int TURNS = PRODUCTS > PIECES_MAX ? PRODUCTS : PIECES_MAX;
#pragma unroll
    for (int x = 0; x < TURNS; ++x) {
      if (x < PRODUCTS)
        acc[x / FM][x % FM] = __builtin_amdgcn_mfma_i32_32x32x32_i8(
            g[x / FM], g[FN + x % FM], acc[x / FM][x % FM], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      piece(x);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (s < steps)
#pragma unroll
      for (int x = 0; x < LOADS; ++x) bring(s, x);
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
  for (int x = 0; x < FN + FM; ++x) f[0][x] = read(0, 0, x);
  auto up_to_last = [&](int32_t s) {
#pragma unroll
    for (int j = 0; j < STEP - 1; ++j)
      multiply(f[j & 1], [&](int x) {
        if (x < FN + FM) f[(j + 1) & 1][x] = read(s, j + 1, x);
      });
  };
  // Before a step's last block the next step's blocks have arrived, for every
  // wave, and every wave has read the last step's, whose place the step
  // STAGES - 1 on takes.
  int32_t s = 0;
#pragma unroll 1
  for (; s < steps - (STAGES - 1); ++s) {
    up_to_last(s);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 3) * LOADS) : "memory");
    multiply(f[1], [&](int x) {
      if (x < FN + FM) f[0][x] = read(s + 1, 0, x);
      if (x < LOADS) bring(s + STAGES - 1, x);
    });
  }
  // (behind the last step's reads is a step read before: its products are not made)
#pragma unroll 1
  for (; s < steps; ++s) {
    up_to_last(s);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    multiply(f[1], [&](int x) {
      if (x < FN + FM) f[0][x] = read(s + 1, 0, x);
    });
  }
  __syncthreads();
  // The sums leave by way of LDS, this wave's own part of it, so that a store
  // of a wave is whole pieces of rows; a lane has the same channels in each.
  // (Scales and biases of all channels in registers before would not fit.)
  constexpr int V = 16 / (int)sizeof(T);     // outputs of 16 bytes
  constexpr int PIECES = 32 * FN / V;        // pieces of a token's outputs
  const int32_t n0 = 64 * FN * tn + 32 * FN * wn;
  lds_char *const mine = lds + w * 32 * PITCH;
  const int c = lane % PIECES;
  const int32_t n = n0 + V * c, left = a.outputs - n;
  float ws[V], bias[V];
  auto scales_of = [&](int z, int32_t channel) {
    const int32_t at = channel < a.outputs ? channel : a.outputs - 1;
    ws[z] = a.w_scales[at];
    bias[z] = a.bias ? a.bias[at] : 0.f;
  };
  // Rows that take no stores of 16 bytes: a store has the same output of a row in
  // neighbouring lanes, and a lane one or two channels (eight at a time, singly,
  // 12,077 tokens of 846 x 9,931 took 302 us, so 250).
  constexpr int COLUMNS = 32 * FN, EACH = COLUMNS > 64 ? COLUMNS / 64 : 1;
  if (a.wide) {
#pragma unroll
    for (int z = 0; z < V; ++z) scales_of(z, n + z);
  } else {
#pragma unroll
    for (int z = 0; z < EACH; ++z) scales_of(z, n0 + (64 * z + lane) % COLUMNS);
  }
  // the scale of token lane % 32 of each block (asked for where it is used, a trip
  // to memory for every other store: 757 us where 16,384 tokens take 743)
  float xs[FM];
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int64_t m = 64 * FM * tm + 32 * (FM * wm + j) + (lane & 31);
    xs[j] = a.x_scales[m < a.tokens ? m : a.tokens - 1];
  }
#pragma unroll
  for (int j = 0; j < FM; ++j) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(lds_as i32x4 *)(mine + (lane & 31) * PITCH + 4 * (32 * i + 8 * q + 4 * (lane >> 5))) =
            i32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                  acc[i][j][4 * q + 3]};
    const int64_t m0 = 64 * FM * tm + 32 * (FM * wm + j);
    if (!a.wide) {
#pragma unroll 8
      for (int x = 0; x < COLUMNS / 2; x += EACH) {
#pragma unroll
        for (int z = 0; z < EACH; ++z) {
          const int at = 64 * (x + z) + lane, r = at / COLUMNS, o = at % COLUMNS;
          const int64_t m = m0 + r;
          const float scale = __shfl(xs[j], r);
          if (m < a.tokens && n0 + o < a.outputs)
            static_cast<T *>(a.out)[m * a.out_row + n0 + o] =
                (T)scaled(*(const lds_as int *)(mine + r * PITCH + 4 * o), scale, ws[z], bias[z]);
        }
      }
      continue;
    }
#pragma unroll 4
    for (int x = 0; x < PIECES / 2; ++x) {
      const int r = (64 * x + lane) / PIECES;
      const int64_t m = m0 + r;
      const float scale = __shfl(xs[j], r);
      typedef __attribute__((ext_vector_type(V))) T Out;
      Out y;
#pragma unroll
      for (int z = 0; z < V; z += 4) {
        const i32x4 sum = *(const lds_as i32x4 *)(mine + r * PITCH + 4 * (V * c + z));
#pragma unroll
        for (int k = 0; k < 4; ++k) y[z + k] = (T)scaled(sum[k], scale, ws[z + k], bias[z + k]);
      }
      if (m < a.tokens && left > 0)
        *reinterpret_cast<Out *>(static_cast<T *>(a.out) + m * a.out_row + n) = y;
    }
  }
}

// Few tokens: a workgroup has 32 channels and up to 32 F tokens, its waves
// take the inner blocks in turn and add up their sums in LDS.
template <class T, int F, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_int8_few(const LinearArgs a) {
  constexpr int RP = 66;  // (no bank twice when the sums are read by channel)
  __shared__ int sums[WAVES][16 * RP];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t nb = blockIdx.x;
  const int64_t m0 = (int64_t)blockIdx.y * 32 * F;
  const char *wp = a.w + (int64_t)nb * a.blocks * BLOCK + 16 * lane;
  const char *xp[F];
  bool have[F];
#pragma unroll
  for (int j = 0; j < F; ++j) {
    const int64_t b = (m0 >> 5) + j;
    have[j] = m0 + 32 * j + (lane & 31) < a.tokens;
    xp[j] = a.x + (b < a.x_blocks ? b : a.x_blocks - 1) * a.blocks * BLOCK + 16 * lane;
  }
  i32x16 acc[F];
#pragma unroll
  for (int j = 0; j < F; ++j) acc[j] = i32x16{};
  // AHEAD inner blocks in flight
  constexpr int AHEAD = F == 1 ? 8 : 6;
  i32x4 y[AHEAD], z[AHEAD][F];
  auto load = [&](int i, int32_t b) {
    y[i] = *reinterpret_cast<const i32x4 *>(wp + (int64_t)b * BLOCK);
#pragma unroll
    for (int j = 0; j < F; ++j)
      // (tokens that are not there: nothing is read for them)
      if (have[j]) z[i][j] = *reinterpret_cast<const i32x4 *>(xp[j] + (int64_t)b * BLOCK);
  };
  auto step = [&](int i) {
#pragma unroll
    for (int j = 0; j < F; ++j)
      acc[j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(y[i], z[i][j], acc[j], 0, 0, 0);
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) z[i][j] = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (w + WAVES * i < a.blocks) load(i, w + WAVES * i);
  int32_t b = w;
#pragma unroll 1
  for (; b + WAVES * (2 * AHEAD - 1) < a.blocks; b += WAVES * AHEAD)
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      step(i);
      load(i, b + WAVES * (AHEAD + i));
    }
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (b + WAVES * i < a.blocks) step(i);
#pragma unroll 4
  for (b += WAVES * AHEAD; b < a.blocks; b += WAVES) {
    load(0, b);
    step(0);
  }
#pragma unroll
  for (int j = 0; j < F; ++j) {
    if (j) __syncthreads();
#pragma unroll
    for (int r = 0; r < 16; ++r) sums[w][r * RP + lane] = acc[j][r];
    __syncthreads();
    for (int x = threadIdx.x; x < 1024; x += 64 * WAVES) {
      const int c = x & 31, t = x >> 5;
      const int at = (4 * (c >> 3) + (c & 3)) * RP + t + 32 * ((c >> 2) & 1);
      int s = 0;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) s += sums[i][at];
      const int64_t m = m0 + 32 * j + t;
      const int32_t n = 32 * nb + c;
      if (m < a.tokens && n < a.outputs)
        static_cast<T *>(a.out)[m * a.out_row + n] =
            (T)scaled(s, a.x_scales[m], a.w_scales[n], a.bias ? a.bias[n] : 0.f);
    }
  }
}

// A few tokens at once with their quantising: every workgroup quantises them
// for itself, into LDS, while its first weights are on their way.  One launch,
// whose latency is what such a call takes (one token through 4,096 x 4,096 5.7 us, in
// two launches 10.8).
struct TokenArgs {
  LinearArgs l;
  const void *x;
  int64_t x_row;
  int32_t k, pitch;  // bytes of a token's codes in LDS
};
template <class X, class T, int M, bool ALIGNED>
__global__ __launch_bounds__(1024) void k_int8_token(const TokenArgs t) {
  constexpr int WAVES = 16, AHEAD = 8;
  const LinearArgs &a = t.l;
  extern __shared__ __attribute__((aligned(16))) char token_lds[];  // codes, then sums
  __shared__ uint32_t tops[M];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t nb = blockIdx.x;
  const char *wp = a.w + (int64_t)nb * a.blocks * BLOCK + 16 * lane;
  // this wave's inner blocks, w, w + 16, ..., AHEAD of them in flight
  i32x4 ahead[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const int32_t b = w + WAVES * i;
    ahead[i] = *reinterpret_cast<const i32x4 *>(wp + (int64_t)(b < a.blocks ? b : 0) * BLOCK);
  }
  const int64_t token0 = (int64_t)blockIdx.y * M;
  const int32_t tokens = (int32_t)(a.tokens - token0 < M ? a.tokens - token0 : M);
  const int32_t pieces = 2 * a.blocks, all = tokens * pieces;
  // the threads share the tokens' pieces of 16 places; the first stay in registers
  Piece<X> held;
  auto load = [&](int32_t i, Piece<X> &y) -> int32_t {
    const int32_t m = M == 1 ? 0 : i / pieces;
    load16<X, ALIGNED>(static_cast<const X *>(t.x) + (token0 + m) * t.x_row, 16 * (i - m * pieces),
                       t.k, y);
    return m;
  };
  if (threadIdx.x < M) tops[threadIdx.x] = 0;
  __syncthreads();
  for (int32_t i = threadIdx.x; i - lane < all; i += 64 * WAVES) {
    Piece<X> y;
    uint32_t top = 0;
    int32_t m = -1;
    if (i < all) {
      m = load(i, y);
      top = magnitude(y);
      if (i == (int32_t)threadIdx.x)
        held = y;
    }
    // (one access to LDS for a wave whose pieces are one token's)
    const int32_t mine = __builtin_amdgcn_readfirstlane(m);
    if (__all(m == mine || m < 0)) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        const uint32_t z = __shfl_xor(top, o);
        top = z > top ? z : top;
      }
      if (lane == 0) atomicMax(&tops[mine], top);
    } else if (m >= 0) {
      atomicMax(&tops[m], top);
    }
  }
  __syncthreads();
  for (int32_t i = threadIdx.x; i < all; i += 64 * WAVES) {
    Piece<X> y;
    int32_t m = M == 1 ? 0 : i / pieces;
    if (i == (int32_t)threadIdx.x)
      y = held;
    else
      m = load(i, y);
    *reinterpret_cast<u32x4 *>(token_lds + m * t.pitch + 16 * (i - m * pieces)) =
        code16(y, row_scale(tops[m]));
  }
  __syncthreads();
  i32x16 acc = i32x16{};
  const int m0 = lane & 31;
  const char *codes = token_lds + (m0 < tokens ? m0 : 0) * t.pitch + 16 * (lane >> 5);
  auto step = [&](int i, int32_t b) {
    // (columns of tokens that are not there are not used)
    const i32x4 z = *reinterpret_cast<const i32x4 *>(codes + 32 * b);
    acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(ahead[i], z, acc, 0, 0, 0);
  };
  int32_t b = w;
#pragma unroll 1
  for (; b + WAVES * (2 * AHEAD - 1) < a.blocks; b += WAVES * AHEAD)
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      step(i, b + WAVES * i);
      ahead[i] = *reinterpret_cast<const i32x4 *>(wp + (int64_t)(b + WAVES * (AHEAD + i)) * BLOCK);
    }
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (b + WAVES * i < a.blocks) step(i, b + WAVES * i);
#pragma unroll 4
  for (b += WAVES * AHEAD; b < a.blocks; b += WAVES) {
    ahead[0] = *reinterpret_cast<const i32x4 *>(wp + (int64_t)b * BLOCK);
    step(0, b);
  }
  __syncthreads();
  // the waves' sums of the tokens there are, through the codes' LDS
  int(*sums)[32 * M] = reinterpret_cast<int(*)[32 * M]>(token_lds);
  if (m0 < M)
#pragma unroll
    for (int r = 0; r < 16; ++r) sums[w][(2 * r + (lane >> 5)) * M + m0] = acc[r];
  __syncthreads();
  {
    const int x = threadIdx.x & 31, m = threadIdx.x >> 5;
    if (m >= tokens) return;
    const int at = (2 * (4 * (x >> 3) + (x & 3)) + ((x >> 2) & 1)) * M + m;
    int s = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) s += sums[i][at];
    const int32_t n = 32 * nb + x;
    if (n < a.outputs)
      static_cast<T *>(a.out)[(token0 + m) * a.out_row + n] =
          (T)scaled(s, row_scale(tops[m]).scale, a.w_scales[n], a.bias ? a.bias[n] : 0.f);
  }
}

// -------------------------------------------------------------------- launches

template <class T> void quantize_of(hipStream_t st, const PackArgs &a, bool aligned) {
  // (a workgroup a row until eight rows each fill the device)
  if (a.rows < 2048) {
    if (aligned)
      k_int8_quantize_row<T, true><<<(unsigned)a.rows, 256, 0, st>>>(a);
    else
      k_int8_quantize_row<T, false><<<(unsigned)a.rows, 256, 0, st>>>(a);
  } else {
    const unsigned g = (unsigned)ceil_div(a.rows, PACK_ROWS);
    if (aligned)
      k_int8_quantize<T, true><<<g, 64 * PACK_ROWS, 0, st>>>(a);
    else
      k_int8_quantize<T, false><<<g, 64 * PACK_ROWS, 0, st>>>(a);
  }
}

void launch_quantize(vsk_ctx *ctx, hipStream_t st, const PackArgs &a, int32_t t) {
  const int64_t size = t == VSK_DTYPE_F32 ? 4 : 2;
  const bool aligned = (uintptr_t)a.x % 16 == 0 && a.x_row * size % 16 == 0;
  KernelTimer kt(ctx, "int8_quantize", (double)a.rows * a.k, st);
  if (t == VSK_DTYPE_F32)
    quantize_of<float>(st, a, aligned);
  else if (t == VSK_DTYPE_F16)
    quantize_of<_Float16>(st, a, aligned);
  else
    quantize_of<__bf16>(st, a, aligned);
  check_launch("int8_quantize");
}

template <class T, int FN, int FM, int STEP, int STAGES>
void tile_of(hipStream_t st, LinearArgs &a) {
  a.tiles_n = (int32_t)ceil_div(a.outputs, 64 * FN);
  const int64_t grid = a.tiles_n * ceil_div(a.tokens, 64 * FM);
  VSK_REQUIRE(grid <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "too many outputs in one call");
  k_int8_tile<T, FN, FM, STEP, STAGES><<<(unsigned)grid, 256, 0, st>>>(a);
}

template <class X, class T> void token_of(hipStream_t st, const TokenArgs &t, bool aligned) {
  auto launch = [&](auto m) {
    constexpr int M = decltype(m)::value;
    // the tokens' codes, and the sums in their place
    const int64_t codes = (t.l.tokens < M ? t.l.tokens : M) * t.pitch, sums = 16 * 32 * M * 4;
    const dim3 g((unsigned)t.l.w_blocks, (unsigned)ceil_div(t.l.tokens, M));
    const unsigned lds = (unsigned)(codes > sums ? codes : sums);
    if (aligned)
      k_int8_token<X, T, M, true><<<g, 1024, lds, st>>>(t);
    else
      k_int8_token<X, T, M, false><<<g, 1024, lds, st>>>(t);
  };
  if (t.l.tokens == 1)
    launch(std::integral_constant<int, 1>());
  else if (t.l.tokens <= 4)
    launch(std::integral_constant<int, 4>());
  else
    launch(std::integral_constant<int, 8>());
}
template <class T> void token_to(hipStream_t st, const TokenArgs &t, int32_t x, bool aligned) {
  if (x == VSK_DTYPE_F32)
    token_of<float, T>(st, t, aligned);
  else if (x == VSK_DTYPE_F16)
    token_of<_Float16, T>(st, t, aligned);
  else
    token_of<__bf16, T>(st, t, aligned);
}

// The kernel and its tile, by how many workgroups each would have.  Measured over
// weights that come from memory, us a call: under 33 tokens the few-tokens
// kernel; to 64 tokens that or tiles of 64 (64 of 4,096 x 4,096 14.7 / 15.9, of
// 4,096 x 12,288 24.7 / 19.0); then tiles of 64, many steps in flight, while
// two a compute unit cover the outputs (256 of 4,096 x 4,096 17.8, tiles of
// 128 27.4; 1,024 of them 40.7 / 33.3); tiles of 128 in the same way (256 of
// 4,096 x 12,288 30.2, with four steps in flight 33.0; 512 of them 48.0 / 39.7)
// until tiles of 256 reach two thirds of the device (1,024 of 4,096 x 12,288
// 72 / 65; 2,048 of 4,096 x 4,096 50 / 60).  A tile has no more places for tokens
// than it needs (64 of 4,096 x 65,536 in tiles of 64 47.7, of 256 69.7; 128 of
// them in tiles of 128 55.7, of 256 70.7), and up to 1,024 places are over so soon
// that two blocks a compute unit, one's outputs beside the other's products, are
// better (16,384 of 512 x 4,096 99 / 81, of 1,024 120 / 116, 4,096 of 2,048 50 / 55).
enum Products { FEW, FEW_64, TILES_64, TILES_128_AHEAD, TILES_128, TILES_256 };
// (what profiling calls them)
constexpr const char *PRODUCTS_NAME[] = {"int8_few",          "int8_few64",   "int8_tile64",
                                         "int8_tile128_ahead", "int8_tile128", "int8_tile256"};
Products products_for(const vsk_ctx *ctx, const LinearArgs &a) {
  const int64_t cus = ctx->cu_count;
  if (a.tokens <= 32) return FEW;
  if (a.tokens <= 64 && a.w_blocks <= cus) return FEW_64;
  auto tiles = [&](int64_t size) {
    return ceil_div(a.outputs, size) * ceil_div(a.tokens, size);
  };
  if (a.tokens <= 64 || tiles(64) <= 2 * cus) return TILES_64;
  if (a.tokens > 128 && a.blocks > 32 && 3 * tiles(256) >= 2 * cus) return TILES_256;
  return tiles(128) <= cus ? TILES_128_AHEAD : TILES_128;
}
template <class T> void products_of(hipStream_t st, LinearArgs &a, Products by) {
  switch (by) {
    case FEW:
      k_int8_few<T, 1, 8><<<dim3((unsigned)a.w_blocks), 512, 0, st>>>(a);
      break;
    case FEW_64:
      k_int8_few<T, 2, 8><<<dim3((unsigned)a.w_blocks), 512, 0, st>>>(a);
      break;
    case TILES_64:
      tile_of<T, 1, 1, 2, 8>(st, a);
      break;
    case TILES_128_AHEAD:
      tile_of<T, 2, 2, 2, 8>(st, a);
      break;
    case TILES_128:
      tile_of<T, 2, 2, 2, 4>(st, a);
      break;
    case TILES_256:
      tile_of<T, 4, 4, 2, 4>(st, a);
  }
}

// Does k_int8_token take the call?  Each of its workgroups quantises up to eight
// tokens for itself: up to 16,384 places, which take about as long as the launch
// that they save (4 tokens of 4,096 through 4,096 outputs 8.0 us, in two launches
// 9.8; 8 of them 10.3 / 10.0; 64 of 1,024 through 1,024 5.1 / 8.1), and no more
// workgroups than run together (400 of 512 through 512 would take 12.6 us, 7.5
// in two launches), or the same in all.
constexpr int64_t GROUP = 8, PLACES = 16384, TOGETHER = 512;
bool one_launch(int64_t tokens, const vsk_int8_weight *w) {
  const int64_t places = (tokens < GROUP ? tokens : GROUP) * w->inputs;
  const int64_t groups = ceil_div(tokens, GROUP), blocks = groups * ceil_div(w->outputs, 32);
  return places <= PLACES &&
         (blocks <= TOGETHER || (groups == 1 && blocks * places <= TOGETHER * PLACES));
}

void check_layer(const vsk_int8_weight *w) {
  VSK_REQUIRE(w, VSK_ERR_INVALID_ARGUMENT, "null argument");
  VSK_REQUIRE(w->outputs >= 1 && w->inputs >= 1, VSK_ERR_EMPTY_INPUT, "an empty layer");
  VSK_REQUIRE(w->inputs <= MOST, VSK_ERR_INVALID_BUFFER_SIZE,
              "at most 131,072 inputs: their sums fill 32 bits");
  VSK_REQUIRE(w->packed && w->scales && is_device_ptr(w->packed) && is_device_ptr(w->scales) &&
                  (!w->bias || is_device_ptr(w->bias)),
              VSK_ERR_INVALID_ARGUMENT, "a layer's weights must be device memory");
  VSK_REQUIRE((uintptr_t)w->packed % 16 == 0, VSK_ERR_INVALID_ARGUMENT,
              "packed weights must be 16-byte aligned");
}

int64_t scales_bytes(int64_t rows) { return ceil_div(rows * 4, 1024) * 1024; }

}  // namespace

}  // namespace vsk

using namespace vsk;

extern "C" {

int64_t vsk_int8_packed_bytes(int64_t rows, int32_t inputs) {
  return rows < 1 || inputs < 1 || inputs > MOST || rows > 0x7FFFFFFFll ? 0
                                                                       : packed_bytes(rows, inputs);
}

vsk_status vsk_int8_pack(vsk_ctx *ctx, void *stream, int32_t dtype, const void *rows,
                         int64_t row_stride, const vsk_int8_weight *w) {
  QUEUED_API_BEGIN(ctx);
  check_layer(w);
  VSK_REQUIRE(dtype >= VSK_DTYPE_F32 && dtype <= VSK_DTYPE_I8, VSK_ERR_UNSUPPORTED,
              "unknown data type");
  VSK_REQUIRE(rows && is_device_ptr(rows), VSK_ERR_INVALID_ARGUMENT,
              "the rows must be device memory");
  PackArgs a{rows, row_stride, w->outputs, static_cast<char *>(w->packed), w->scales, w->inputs,
             (int32_t)inner_blocks(w->inputs)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == VSK_DTYPE_I8) {
    KernelTimer kt(ctx, "int8_pack", (double)a.rows * a.k, st);
    k_int8_pack<<<(unsigned)ceil_div(a.rows, 4), 256, 0, st>>>(a);
    check_launch("int8_pack");
  } else {
    launch_quantize(ctx, st, a, dtype);
  }
  finish_queued(ctx, st);
  VSK_API_END(ctx);
}

int64_t vsk_int8_linear_workspace(const vsk_int8_weight *w, int64_t tokens) {
  if (!w || tokens < 1 || tokens > 0x7FFFFFFFll || w->inputs < 1 || w->inputs > MOST) return 0;
  return one_launch(tokens, w) ? 0 : scales_bytes(tokens) + packed_bytes(tokens, w->inputs);
}

vsk_status vsk_int8_linear(vsk_ctx *ctx, void *stream, const vsk_int8_weight *w,
                           const vsk_int8_rows *r) {
  QUEUED_API_BEGIN(ctx);
  check_layer(w);
  VSK_REQUIRE(r, VSK_ERR_INVALID_ARGUMENT, "null argument");
  VSK_REQUIRE(r->x_dtype >= VSK_DTYPE_F32 && r->x_dtype <= VSK_DTYPE_BF16 &&
                  r->out_dtype >= VSK_DTYPE_F32 && r->out_dtype <= VSK_DTYPE_BF16,
              VSK_ERR_UNSUPPORTED, "unknown data type");
  VSK_REQUIRE(r->tokens >= 0, VSK_ERR_INVALID_ARGUMENT, "negative counts");
  VSK_REQUIRE(r->tokens <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "at most 2^31 - 1 tokens");
  if (r->tokens == 0) return VSK_OK;
  VSK_REQUIRE(r->x && r->out && is_device_ptr(r->x) && is_device_ptr(r->out),
              VSK_ERR_INVALID_ARGUMENT, "inputs and outputs must be device memory");
  const int64_t need = vsk_int8_linear_workspace(w, r->tokens);
  VSK_REQUIRE(need == 0 || (r->workspace && r->workspace_bytes >= need &&
                            (uintptr_t)r->workspace % 16 == 0 && is_device_ptr(r->workspace)),
              VSK_ERR_INVALID_BUFFER_SIZE,
              "the workspace must be " + std::to_string(need) + " bytes of device memory");
  hipStream_t st = static_cast<hipStream_t>(stream);
  float *scales = static_cast<float *>(r->workspace);
  char *codes = static_cast<char *>(r->workspace) + scales_bytes(r->tokens);
  const int32_t blocks = (int32_t)inner_blocks(w->inputs);
  LinearArgs a{};
  a.w = static_cast<const char *>(w->packed), a.x = codes;
  a.w_scales = w->scales, a.x_scales = scales, a.bias = w->bias;
  a.out = r->out, a.out_row = r->out_row, a.tokens = r->tokens;
  a.outputs = w->outputs, a.blocks = blocks;
  a.w_blocks = (int32_t)ceil_div(w->outputs, 32), a.x_blocks = ceil_div(r->tokens, 32);
  const int64_t pitch = 32 * (int64_t)blocks + 16;
  if (one_launch(r->tokens, w)) {
    const int64_t x_size = r->x_dtype == VSK_DTYPE_F32 ? 4 : 2;
    const bool al = (uintptr_t)r->x % 16 == 0 && r->x_row * x_size % 16 == 0;
    const TokenArgs t{a, r->x, r->x_row, w->inputs, (int32_t)pitch};
    {
      KernelTimer kt(ctx, "int8_token", (double)a.tokens * a.outputs * w->inputs, st);
      if (r->out_dtype == VSK_DTYPE_F32)
        token_to<float>(st, t, r->x_dtype, al);
      else if (r->out_dtype == VSK_DTYPE_F16)
        token_to<_Float16>(st, t, r->x_dtype, al);
      else
        token_to<__bf16>(st, t, r->x_dtype, al);
      check_launch("int8_token");
    }
    finish_queued(ctx, st);
    return VSK_OK;
  }
  launch_quantize(ctx, st, PackArgs{r->x, r->x_row, r->tokens, codes, scales, w->inputs, blocks},
                  r->x_dtype);
  const int64_t size = r->out_dtype == VSK_DTYPE_F32 ? 4 : 2;
  a.wide = (uintptr_t)r->out % 16 == 0 && r->out_row * size % 16 == 0 && w->outputs * size % 16 == 0;
  {
    const Products by = products_for(ctx, a);
    KernelTimer kt(ctx, PRODUCTS_NAME[by], (double)a.tokens * a.outputs * w->inputs, st);
    if (r->out_dtype == VSK_DTYPE_F32)
      products_of<float>(st, a, by);
    else if (r->out_dtype == VSK_DTYPE_F16)
      products_of<_Float16>(st, a, by);
    else
      products_of<__bf16>(st, a, by);
    check_launch("int8_linear");
  }
  finish_queued(ctx, st);
  VSK_API_END(ctx);
}

}  // extern "C"
