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
#include "attn.hpp"
#include "vsk_api.hpp"

namespace vsk {

namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(16))) int i32x16;

constexpr int BLOCK = 1024;       // bytes of a 32 x 32 block
constexpr int STEP = 2;           // blocks of a step along the inner dimension
constexpr int32_t MOST = 131072;  // inner places whose sums (128 * 127 each) fit 32 bits

int64_t inner_blocks(int64_t k) { return ceil_div(k, 32 * STEP) * STEP; }
int64_t packed_bytes(int64_t rows, int64_t k) {
  return ceil_div(rows, 32) * inner_blocks(k) * BLOCK;
}

// ------------------------------------------------------------------ quantising

// 16 values of a row from element e on, zero past the end
template <class T, bool ALIGNED>
__device__ inline void load16(const T *row, int32_t e, int32_t k, float (&x)[16]) {
  if (ALIGNED && e + 16 <= k) {
    constexpr int W = 16 / sizeof(T);
    typedef __attribute__((ext_vector_type(W))) T V;
#pragma unroll
    for (int i = 0; i < 16 / W; ++i) {
      const V v = *reinterpret_cast<const V *>(row + e + W * i);
#pragma unroll
      for (int j = 0; j < W; ++j) x[W * i + j] = (float)v[j];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = e + i < k ? (float)row[e + i] : 0.f;
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
__device__ inline uint32_t code4(const float *x, const RowScale &r) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // (the largest is 127 times 1 + 2^-22 at most; NaN times 0 is not taken)
    const int c = r.inverse == 0.f ? 0 : (int)__builtin_rintf(x[i] * r.up * r.inverse);
    w |= (uint32_t)(c & 255) << (8 * i);
  }
  return w;
}

struct PackArgs {
  const void *x;
  int64_t x_row, rows;
  char *packed;
  float *scales;
  int32_t k, blocks;  // inner places, inner blocks
};

template <class T> __device__ inline uint32_t magnitude(const float (&x)[16]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t b = __float_as_uint(x[i]) & 0x7FFFFFFFu;
    top = b > top ? b : top;
  }
  return top;
}

// WPR waves a row (4 / WPR rows a workgroup).  A lane takes pieces of 16
// places; the first HELD of them stay in registers between the two passes.
template <class T, int WPR, bool ALIGNED>
__global__ __launch_bounds__(256) void k_int8_quantize(const PackArgs a) {
  constexpr int HELD = sizeof(T) == 4 ? 4 : 8;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * (4 / WPR) + w / WPR;
  const int at = WPR > 1 ? threadIdx.x : lane;
  const int pieces = 2 * a.blocks;
  const bool real = row < a.rows;
  const T *x = static_cast<const T *>(a.x) + (real ? row * a.x_row : 0);
  const int32_t k = real ? a.k : 0;
  float held[HELD][16];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int p = at + 64 * WPR * i;
    if (p < pieces) load16<T, ALIGNED>(x, 16 * p, k, held[i]);
  }
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (at + 64 * WPR * i < pieces) {
      const uint32_t t = magnitude<T>(held[i]);
      top = t > top ? t : top;
    }
  for (int p = at + 64 * WPR * HELD; p < pieces; p += 64 * WPR) {
    float y[16];
    load16<T, ALIGNED>(x, 16 * p, k, y);
    const uint32_t t = magnitude<T>(y);
    top = t > top ? t : top;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t t = __shfl_xor(top, o);
    top = t > top ? t : top;
  }
  if constexpr (WPR > 1) {
    __shared__ uint32_t tops[4];
    if (lane == 0) tops[w] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) top = tops[i] > top ? tops[i] : top;
  }
  if (!real) return;
  const RowScale r = row_scale(top);
  if (at == 0) a.scales[row] = r.scale;
  char *to = a.packed + (row >> 5) * a.blocks * BLOCK + (row & 31) * 16;
  auto put = [&](int p, const float (&y)[16]) {
    u32x4 c;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = code4(y + 4 * i, r);
    *reinterpret_cast<u32x4 *>(to + (int64_t)(p >> 1) * BLOCK + (p & 1) * 512) = c;
  };
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (at + 64 * WPR * i < pieces) put(at + 64 * WPR * i, held[i]);
  for (int p = at + 64 * WPR * HELD; p < pieces; p += 64 * WPR) {
    float y[16];
    load16<T, ALIGNED>(x, 16 * p, k, y);
    put(p, y);
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

__device__ inline float scaled(int sum, float xs, float ws, float bias) {
  return (float)sum * xs * ws + bias;
}

// A tile of 64 FN channels and 64 FM tokens, four waves of FN x FM products of
// 32 x 32: lane l has token l % 32 and, in register 4 q + i, channel
// 8 q + 4 (l / 32) + i.
template <class T, int FN, int FM>
__global__ __launch_bounds__(256, FN * FM >= 16 ? 1 : 2) void k_int8_tile(const LinearArgs a) {
  constexpr int ROWS = 2 * (FN + FM);            // row blocks of a stage
  constexpr int STAGE = ROWS * STEP * BLOCK;     // bytes of it
  constexpr int STAGES = 4;
  constexpr int MINE = ROWS / 4;                 // row blocks that a wave brings
  constexpr int LOADS = MINE * STEP;
  constexpr int PITCH = FN * 32 * 4 + 16;        // of a token's sums in LDS, in bytes
  constexpr int OUT = 4 * 32 * PITCH;
  __shared__ __attribute__((aligned(1024))) char lds_pool[STAGES * STAGE > OUT ? STAGES * STAGE : OUT];
  lds_char *const lds = (lds_char *)lds_pool;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = w & 1, wm = w >> 1;
  const int32_t tn = blockIdx.x % a.tiles_n;
  const int64_t tm = blockIdx.x / a.tiles_n;
  // the row blocks that this wave brings: the channels' first
  uint64_t base[MINE];
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int r = MINE * w + i;
    if (r < 2 * FN) {
      const int32_t b = 2 * FN * tn + r;
      base[i] = (uint64_t)(uintptr_t)a.w + (int64_t)(b < a.w_blocks ? b : a.w_blocks - 1) * a.blocks * BLOCK;
    } else {
      const int64_t b = 2 * FM * tm + r - 2 * FN;
      base[i] = (uint64_t)(uintptr_t)a.x + (b < a.x_blocks ? b : a.x_blocks - 1) * a.blocks * BLOCK;
    }
  }
  const int32_t steps = a.blocks / STEP;
  // one of the loads that bring step s, in order of s: the addresses go along
  auto bring = [&](int32_t s, int x) {
    load_to_lds(base[x / STEP] + x % STEP * BLOCK, 16 * lane,
                lds + (s % STAGES) * STAGE + (MINE * w * STEP + x) * BLOCK);
    if (x % STEP == STEP - 1) base[x / STEP] += STEP * BLOCK;
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
  auto first_half = [&](int32_t s) {
    multiply(f[0], [&](int x) {
      if (x < FN + FM) f[1][x] = read(s, 1, x);
    });
  };
  // Between a step's halves the next step's blocks have arrived, for every
  // wave, and every wave has read the last step's, whose place the step after
  // the next two takes.
  int32_t s = 0;
#pragma unroll 1
  for (; s < steps - (STAGES - 1); ++s) {
    first_half(s);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LOADS) : "memory");
    multiply(f[1], [&](int x) {
      if (x < FN + FM) f[0][x] = read(s + 1, 0, x);
      if (x < LOADS) bring(s + STAGES - 1, x);
    });
  }
  // (behind the last step's reads is a step read before: its products are not made)
#pragma unroll 1
  for (; s < steps; ++s) {
    first_half(s);
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
#pragma unroll
  for (int z = 0; z < V; ++z) {
    const int32_t at = z < left ? n + z : a.outputs - 1;
    ws[z] = a.w_scales[at];
    bias[z] = a.bias ? a.bias[at] : 0.f;
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
#pragma unroll 2
    for (int x = 0; x < PIECES / 2; ++x) {
      const int r = (64 * x + lane) / PIECES;
      const int64_t m = m0 + r;
      const float xs = a.x_scales[m < a.tokens ? m : a.tokens - 1];
      typedef __attribute__((ext_vector_type(V))) T Out;
      Out y;
#pragma unroll
      for (int z = 0; z < V; z += 4) {
        const i32x4 sum = *(const lds_as i32x4 *)(mine + r * PITCH + 4 * (V * c + z));
#pragma unroll
        for (int k = 0; k < 4; ++k) y[z + k] = (T)scaled(sum[k], xs, ws[z + k], bias[z + k]);
      }
      T *to = static_cast<T *>(a.out) + m * a.out_row + n;
      const int32_t some = m < a.tokens ? left : 0;
      if (a.wide) {
        if (some > 0) *reinterpret_cast<Out *>(to) = y;
      } else {
#pragma unroll
        for (int z = 0; z < V; ++z)
          if (z < some) to[z] = y[z];
      }
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
#pragma unroll 4
  for (int32_t b = w; b < a.blocks; b += WAVES) {
    const i32x4 y = *reinterpret_cast<const i32x4 *>(wp + (int64_t)b * BLOCK);
#pragma unroll
    for (int j = 0; j < F; ++j) {
      // (tokens that are not there: nothing is read for them)
      i32x4 z = {0, 0, 0, 0};
      if (have[j]) z = *reinterpret_cast<const i32x4 *>(xp[j] + (int64_t)b * BLOCK);
      acc[j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(y, z, acc[j], 0, 0, 0);
    }
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

// -------------------------------------------------------------------- launches

template <class T>
void quantize_of(hipStream_t st, const PackArgs &a, bool aligned) {
  // a workgroup a row while there are too few rows to fill the device with waves
  if (a.rows < 1024) {
    if (aligned)
      k_int8_quantize<T, 4, true><<<(unsigned)a.rows, 256, 0, st>>>(a);
    else
      k_int8_quantize<T, 4, false><<<(unsigned)a.rows, 256, 0, st>>>(a);
  } else {
    const unsigned g = (unsigned)ceil_div(a.rows, 4);
    if (aligned)
      k_int8_quantize<T, 1, true><<<g, 256, 0, st>>>(a);
    else
      k_int8_quantize<T, 1, false><<<g, 256, 0, st>>>(a);
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

template <class T, int FN, int FM> void tile_of(hipStream_t st, LinearArgs &a) {
  a.tiles_n = (int32_t)ceil_div(a.outputs, 64 * FN);
  const int64_t grid = a.tiles_n * ceil_div(a.tokens, 64 * FM);
  VSK_REQUIRE(grid <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "too many outputs in one call");
  k_int8_tile<T, FN, FM><<<(unsigned)grid, 256, 0, st>>>(a);
}

template <class T> void products_of(vsk_ctx *ctx, hipStream_t st, LinearArgs &a) {
  if (a.tokens <= 32) {
    k_int8_few<T, 1, 16><<<dim3((unsigned)a.w_blocks), 1024, 0, st>>>(a);
    return;
  }
  if (a.tokens <= 64) {
    k_int8_few<T, 2, 16><<<dim3((unsigned)a.w_blocks), 1024, 0, st>>>(a);
    return;
  }
  const int64_t large = ceil_div(a.outputs, 256) * ceil_div(a.tokens, 256);
  const int64_t middle = ceil_div(a.outputs, 128) * ceil_div(a.tokens, 128);
  if (large >= ctx->cu_count)
    tile_of<T, 4, 4>(st, a);
  else if (middle >= ctx->cu_count)
    tile_of<T, 2, 2>(st, a);
  else
    tile_of<T, 1, 1>(st, a);
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
  return scales_bytes(tokens) + packed_bytes(tokens, w->inputs);
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
  VSK_REQUIRE(r->workspace && r->workspace_bytes >= need && (uintptr_t)r->workspace % 16 == 0 &&
                  is_device_ptr(r->workspace),
              VSK_ERR_INVALID_BUFFER_SIZE,
              "the workspace must be " + std::to_string(need) + " bytes of device memory");
  hipStream_t st = static_cast<hipStream_t>(stream);
  float *scales = static_cast<float *>(r->workspace);
  char *codes = static_cast<char *>(r->workspace) + scales_bytes(r->tokens);
  const int32_t blocks = (int32_t)inner_blocks(w->inputs);
  launch_quantize(ctx, st, PackArgs{r->x, r->x_row, r->tokens, codes, scales, w->inputs, blocks},
                  r->x_dtype);
  LinearArgs a{};
  a.w = static_cast<const char *>(w->packed), a.x = codes;
  a.w_scales = w->scales, a.x_scales = scales, a.bias = w->bias;
  a.out = r->out, a.out_row = r->out_row, a.tokens = r->tokens;
  a.outputs = w->outputs, a.blocks = blocks;
  a.w_blocks = (int32_t)ceil_div(w->outputs, 32), a.x_blocks = ceil_div(r->tokens, 32);
  const int64_t size = r->out_dtype == VSK_DTYPE_F32 ? 4 : 2;
  a.wide = (uintptr_t)r->out % 16 == 0 && r->out_row * size % 16 == 0 && w->outputs * size % 16 == 0;
  {
    KernelTimer kt(ctx, "int8_linear", (double)a.tokens * a.outputs * w->inputs, st);
    if (r->out_dtype == VSK_DTYPE_F32)
      products_of<float>(ctx, st, a);
    else if (r->out_dtype == VSK_DTYPE_F16)
      products_of<_Float16>(ctx, st, a);
    else
      products_of<__bf16>(ctx, st, a);
    check_launch("int8_linear");
  }
  finish_queued(ctx, st);
  VSK_API_END(ctx);
}

}  // extern "C"
