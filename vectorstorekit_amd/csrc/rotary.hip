// rotary.hip -- rotary positions, alone or on the way into a paged cache.
//
// Pair i of a head's first 2 * pairs values turns by position * inv_freq[i].
// In fp32 that product is off by up to half a radian at a position of 2^20;
// here inv_freq / 2 pi is a 64-bit fraction of a turn, its integer product
// with the position drops the whole turns by itself and the phase is exact to
// 2^-32 of a turn at every int32 position.  16-bit values take the hardware's
// sine and cosine (absolute error about 2^-20, a 500th of the output's
// rounding), 32-bit ones sincospif.
//
// One pass over the heads, bound by their bytes: a thread keeps the sines and
// cosines of its pairs in registers and takes every hs-th head of its token,
// two heads' loads in flight together (16,384 tokens of 40 bf16 heads of 128:
// 69 us, 4.9 TB/s, where one head at a time took 83; a copy does 5.1).  The
// tensors of a call (queries, keys, values) are one sequence of heads, so a
// call is one launch: few tokens take 4 us, the time of a launch and two trips
// to memory.  Into pages (24 ragged prompts to 641, half of each head turned,
// f16, with their queries) 46 us, 3.9 TB/s, or 33 where the last-level cache
// still holds them: 178 MB end before a launch's start and end are small.
#include <cmath>

#include "attn.hpp"
#include "vsk_api.hpp"

struct vsk_rotary {
  vsk::DevBuf turns;  // uint64 per pair: turns a position, in 2^-64
  int32_t pairs = 0, layout = 0;
  float amplitude = 1.f;
};

namespace vsk {

namespace {

struct HeadRows {
  const void *src;
  void *dst;
  int64_t src_row, src_head, dst_row, dst_head;
  int32_t heads;
  int32_t turn;   // rotated, or copied
  int32_t paged;  // dst is a layer of a cache: dst_row within a page, dst_page a page
  int64_t dst_page;
};

struct RotaryArgs {
  HeadRows x[3];
  const uint64_t *turns;
  const int32_t *positions;  // or null: from the sequences
  const int32_t *starts, *seqs, *lengths, *table;
  int64_t table_stride, tokens;
  int32_t n, max_new, slots, width, pages_n, page_shift;
  int32_t pairs, interleaved, d, inverse;
  float amplitude;
  int32_t heads;  // of all tensors
  int32_t hs;     // threads that share a token's heads (per unit)
  int32_t units;  // of 2 * V values a head
};

template <class T> __device__ inline void sin_cos(uint32_t phase, float *s, float *c) {
  const float turns = (float)(int32_t)phase * 2.3283064365386963e-10f;  // [-0.5, 0.5]
  if constexpr (sizeof(T) == 4) {
    sincospif(2.f * turns, s, c);
  } else {
    *s = __builtin_amdgcn_sinf(turns);
    *c = __builtin_amdgcn_cosf(turns);
  }
}

// V: elements of an access; 1: any alignment and parity.
// Unit u of a head: pairs [u V, u V + V) while they last, then 2 V values of
// those that pass through.  In a copied tensor: 2 V values from 2 V u on.
template <class T, int V>
__global__ __launch_bounds__(256) void k_rotary(const RotaryArgs a) {
  const int64_t per = (int64_t)a.max_new * a.hs * a.units;
  const int64_t blocks = (per + 255) / 256;
  const int32_t b = (int32_t)(blockIdx.x / blocks);
  const int64_t at = (blockIdx.x % blocks) * 256 + threadIdx.x;
  if (at >= per) return;
  const int32_t u = (int32_t)(at % a.units);
  const int64_t y = at / a.units;
  const int32_t h0 = (int32_t)(y % a.hs), t = (int32_t)(y / a.hs);

  // the token: its row, its position and its place in the cache
  int64_t row = t;
  int32_t pos;
  int64_t page = -1;
  int32_t in_page = 0;
  if (a.positions) {
    pos = a.positions[t];
  } else {
    int32_t t0 = b, count = 1;
    if (a.starts) {
      t0 = a.starts[b] < 0 ? 0 : a.starts[b];
      const int32_t t1 = a.starts[b + 1] > a.tokens ? (int32_t)a.tokens : a.starts[b + 1];
      count = t1 > t0 ? t1 - t0 : 0;  // (offsets out of order: t1 - t0 may not fit 32 bits)
    }
    if (t >= count) return;
    row = t0 + t;
    const int32_t slot = a.seqs ? a.seqs[b] : b;
    if ((uint32_t)slot >= (uint32_t)a.slots) return;
    pos = a.lengths[slot] - count + t;
    const int32_t i = pos >> a.page_shift;
    if (pos >= 0 && i < a.width) {
      page = a.table[slot * a.table_stride + i];
      if (page >= a.pages_n) page = -1;
      in_page = pos & ((1 << a.page_shift) - 1);
    }
  }
  const bool turned = u * V < a.pairs;
  float c[V], s[V];
  if (turned) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint64_t f = a.turns[u * V + i] * (uint64_t)(int64_t)pos;
      sin_cos<T>((uint32_t)(f >> 32), &s[i], &c[i]);
      c[i] *= a.amplitude;
      s[i] *= a.inverse ? -a.amplitude : a.amplitude;
    }
  }
  // where a head's two runs of V values lie
  struct Place {
    const T *src;
    T *dst;
    int32_t e0, e1;
    bool turn;
  };
  auto place = [&](int32_t h, Place &p) -> bool {
    int32_t hh = h;
    const bool second = hh >= a.x[0].heads;
    if (second) hh -= a.x[0].heads;
    const bool third = second && hh >= a.x[1].heads;
    if (third) hh -= a.x[1].heads;
    const HeadRows &x = third ? a.x[2] : second ? a.x[1] : a.x[0];
    if (h >= a.heads || (x.paged && page < 0)) return false;
    p.src = static_cast<const T *>(x.src) + row * x.src_row + hh * x.src_head;
    p.dst = static_cast<T *>(x.dst) + hh * x.dst_head +
            (x.paged ? page * x.dst_page + in_page * x.dst_row : row * x.dst_row);
    p.turn = x.turn && turned;
    p.e0 = 2 * V * u;
    p.e1 = p.e0 + V;
    if (p.turn && !a.interleaved) {
      p.e0 = V * u;
      p.e1 = a.pairs + V * u;
    }
    return true;
  };
  if constexpr (V == 1) {
    for (int32_t h = h0; h < a.heads; h += a.hs) {
      Place p;
      if (!place(h, p)) continue;
      // (an odd head: the last unit holds one value)
      const bool two = p.e1 < a.d;
      const T p0 = p.src[p.e0], p1 = two ? p.src[p.e1] : T(0.f);
      if (p.turn) {
        const float f0 = (float)p0, f1 = (float)p1;
        p.dst[p.e0] = (T)(f0 * c[0] - f1 * s[0]);
        p.dst[p.e1] = (T)(f0 * s[0] + f1 * c[0]);
      } else {
        p.dst[p.e0] = p0;
        if (two) p.dst[p.e1] = p1;
      }
    }
  } else {
    typedef __attribute__((ext_vector_type(V))) T VT;
    // WAYS heads at a time: their loads are in flight together
    constexpr int WAYS = 2;
    for (int32_t h = h0; h < a.heads; h += WAYS * a.hs) {
      Place p[WAYS];
      VT v0[WAYS], v1[WAYS];
      bool on[WAYS];
#pragma unroll
      for (int y = 0; y < WAYS; ++y) {
        on[y] = place(h + y * a.hs, p[y]);
        if (on[y]) {
          v0[y] = *reinterpret_cast<const VT *>(p[y].src + p[y].e0);
          v1[y] = *reinterpret_cast<const VT *>(p[y].src + p[y].e1);
        }
      }
#pragma unroll
      for (int y = 0; y < WAYS; ++y) {
        if (!on[y]) continue;
        if (p[y].turn) {
          const VT x0 = v0[y], x1 = v1[y];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            if (a.interleaved) {
              const int j = 2 * i;
              const float p0 = (float)(j < V ? x0[j % V] : x1[j % V]);
              const float p1 = (float)(j < V ? x0[(j + 1) % V] : x1[(j + 1) % V]);
              const T r0 = (T)(p0 * c[i] - p1 * s[i]), r1 = (T)(p0 * s[i] + p1 * c[i]);
              if (j < V)
                v0[y][j % V] = r0, v0[y][(j + 1) % V] = r1;
              else
                v1[y][j % V] = r0, v1[y][(j + 1) % V] = r1;
            } else {
              const float p0 = (float)x0[i], p1 = (float)x1[i];
              v0[y][i] = (T)(p0 * c[i] - p1 * s[i]);
              v1[y][i] = (T)(p0 * s[i] + p1 * c[i]);
            }
          }
        }
        *reinterpret_cast<VT *>(p[y].dst + p[y].e0) = v0[y];
        *reinterpret_cast<VT *>(p[y].dst + p[y].e1) = v1[y];
      }
    }
  }
}

template <class T> void rotary_of(hipStream_t st, const RotaryArgs &a, int v, unsigned grid) {
  constexpr int W = 16 / sizeof(T);
  if (v == W)
    k_rotary<T, W><<<grid, 256, 0, st>>>(a);
  else if (v == W / 2)
    k_rotary<T, W / 2><<<grid, 256, 0, st>>>(a);
  else
    k_rotary<T, 1><<<grid, 256, 0, st>>>(a);
}

bool fits(const HeadRows &x, int64_t bytes, int64_t size) {
  const int64_t m = bytes / size;
  return ((uintptr_t)x.src % bytes) == 0 && ((uintptr_t)x.dst % bytes) == 0 &&
         x.src_row % m == 0 && x.src_head % m == 0 && x.dst_row % m == 0 && x.dst_head % m == 0 &&
         x.dst_page % m == 0;
}

void launch_rotary(vsk_ctx *ctx, hipStream_t st, RotaryArgs &a, int32_t dtype) {
  const int64_t size = dtype == VSK_DTYPE_F32 ? 4 : 2;
  a.heads = a.x[0].heads + a.x[1].heads + a.x[2].heads;
  if (a.heads == 0 || a.max_new == 0 || a.n == 0) return;
  // the widest access that the pairs, the values after them and every stride take
  int v = (int)(16 / size);
  for (; v > 1; v = v == 16 / size ? v / 2 : 1) {
    bool ok = a.d % (2 * v) == 0;
    if (a.pairs > 0)
      ok = ok && a.pairs % v == 0 && (a.d - 2 * a.pairs) % (2 * v) == 0;
    for (const auto &x : a.x)
      if (x.heads) ok = ok && fits(x, v * size, size);
    if (ok) break;
  }
  a.units = (a.d + 2 * v - 1) / (2 * v);
  // threads enough to keep the memory busy (4,096 a compute unit: two full
  // sets), and no more: the sines and cosines are a thread's, whatever the
  // number of its heads
  const int64_t one = (int64_t)a.n * a.max_new * a.units;
  a.hs = 1;
  while (a.hs < a.heads && one * a.hs < (int64_t)ctx->cu_count * 4096) a.hs *= 2;
  if (a.hs > a.heads) a.hs = a.heads;
  const int64_t blocks = ceil_div((int64_t)a.max_new * a.hs * a.units, 256) * a.n;
  VSK_REQUIRE(blocks <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE, "too many tokens in one call");
  KernelTimer kt(ctx, "rotary", (double)a.tokens * a.heads, st);
  if (dtype == VSK_DTYPE_F32)
    rotary_of<float>(st, a, v, (unsigned)blocks);
  else if (dtype == VSK_DTYPE_F16)
    rotary_of<_Float16>(st, a, v, (unsigned)blocks);
  else
    rotary_of<__bf16>(st, a, v, (unsigned)blocks);
  check_launch("rotary");
}

HeadRows rows_of(const vsk_head_rows &r, bool turn) {
  VSK_REQUIRE(r.heads >= 1 && r.heads <= (1 << 20), VSK_ERR_INVALID_ARGUMENT,
              "a tensor needs at least one head");
  VSK_REQUIRE(r.src && is_device_ptr(r.src), VSK_ERR_INVALID_ARGUMENT,
              "tensors must be device memory");
  HeadRows x{};
  x.src = r.src;
  x.dst = r.dst;
  x.src_row = r.src_row;
  x.src_head = r.src_head;
  x.dst_row = r.dst_row;
  x.dst_head = r.dst_head;
  x.heads = r.heads;
  x.turn = turn;
  return x;
}

void set_rotary(RotaryArgs &a, const vsk_rotary *r) {
  a.turns = r->turns.as<uint64_t>();
  a.pairs = r->pairs;
  a.interleaved = r->layout == VSK_ROTARY_INTERLEAVED;
  a.amplitude = r->amplitude;
}

}  // namespace

}  // namespace vsk

using namespace vsk;

extern "C" {

vsk_status vsk_rotary_create(vsk_ctx *ctx, const double *inv_freq, int32_t pairs, int32_t layout,
                             double amplitude, vsk_rotary **out) {
  QUEUED_API_BEGIN(ctx);
  VSK_REQUIRE(out, VSK_ERR_INVALID_ARGUMENT, "out is null");
  *out = nullptr;
  VSK_REQUIRE(inv_freq, VSK_ERR_INVALID_ARGUMENT, "inv_freq is null");
  VSK_REQUIRE(pairs >= 1 && pairs <= (1 << 16), VSK_ERR_INVALID_ARGUMENT,
              "pairs must be between 1 and 65536");
  VSK_REQUIRE(layout == VSK_ROTARY_HALF || layout == VSK_ROTARY_INTERLEAVED,
              VSK_ERR_INVALID_ARGUMENT, "unknown rotary layout");
  VSK_REQUIRE(std::isfinite(amplitude), VSK_ERR_INVALID_ARGUMENT, "amplitude must be finite");
  std::vector<uint64_t> turns((size_t)pairs);
  for (int32_t i = 0; i < pairs; ++i) {
    VSK_REQUIRE(std::isfinite(inv_freq[i]) && inv_freq[i] >= 0, VSK_ERR_INVALID_ARGUMENT,
                "inv_freq must be finite and not negative");
    const long double t = (long double)inv_freq[i] / 6.283185307179586476925286766559L;
    const long double frac = t - floorl(t);
    const long double scaled = frac * 18446744073709551616.0L + 0.5L;
    turns[(size_t)i] = scaled >= 18446744073709551616.0L ? 0 : (uint64_t)scaled;
  }
  std::unique_ptr<vsk_rotary> r(new vsk_rotary());
  r->pairs = pairs;
  r->layout = layout;
  r->amplitude = (float)amplitude;
  CallScope cs(ctx);
  r->turns.reserve(sizeof(uint64_t) * (size_t)pairs);
  VSK_HIP(hipMemcpyAsync(r->turns.p, turns.data(), sizeof(uint64_t) * (size_t)pairs,
                         hipMemcpyHostToDevice, ctx->stream));
  cs.finish();
  *out = r.release();
  VSK_API_END(ctx);
}

vsk_status vsk_rotary_free(vsk_ctx *ctx, vsk_rotary *rotary) {
  if (!rotary) return VSK_OK;
  int device = 0;
  (void)hipGetDevice(&device);
  const DeviceScope scope(ctx ? ctx->device : device);
  // (the release waits for the device: work queued on any stream may read it)
  (void)hipDeviceSynchronize();
  delete rotary;
  return VSK_OK;
}

vsk_status vsk_rotary_apply(vsk_ctx *ctx, void *stream, const vsk_rotary *rotary, int32_t dtype,
                            int32_t d, int64_t tokens, const int32_t *positions, int32_t inverse,
                            const vsk_head_rows *tensors, int32_t n_tensors) {
  QUEUED_API_BEGIN(ctx);
  VSK_REQUIRE(rotary && tensors, VSK_ERR_INVALID_ARGUMENT, "null argument");
  VSK_REQUIRE(dtype >= VSK_DTYPE_F32 && dtype <= VSK_DTYPE_BF16, VSK_ERR_UNSUPPORTED,
              "unknown data type");
  VSK_REQUIRE(n_tensors >= 1 && n_tensors <= 3, VSK_ERR_INVALID_ARGUMENT,
              "between one and three tensors");
  VSK_REQUIRE(d >= 2 * rotary->pairs, VSK_ERR_DIMENSION_MISMATCH,
              "a head holds fewer values than the rotation turns");
  VSK_REQUIRE(d <= (1 << 20), VSK_ERR_INVALID_BUFFER_SIZE, "a head holds at most 2^20 values");
  VSK_REQUIRE(tokens >= 0 && tokens <= 0x7FFFFFFFll, VSK_ERR_INVALID_BUFFER_SIZE,
              "between 0 and 2^31 - 1 tokens");
  if (tokens == 0) return VSK_OK;
  VSK_REQUIRE(positions && is_device_ptr(positions), VSK_ERR_INVALID_ARGUMENT,
              "positions must be device memory");
  RotaryArgs a{};
  for (int32_t i = 0; i < n_tensors; ++i) {
    a.x[i] = rows_of(tensors[i], true);
    VSK_REQUIRE(tensors[i].dst && is_device_ptr(tensors[i].dst), VSK_ERR_INVALID_ARGUMENT,
                "tensors must be device memory");
  }
  set_rotary(a, rotary);
  a.positions = positions;
  a.tokens = tokens;
  a.n = 1;
  a.max_new = (int32_t)tokens;
  a.d = d;
  a.inverse = inverse != 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  launch_rotary(ctx, st, a, dtype);
  finish_queued(ctx, st);
  VSK_API_END(ctx);
}

vsk_status vsk_kv_append(vsk_ctx *ctx, void *stream, const vsk_kv *kv, int32_t layer,
                         const vsk_new_tokens *news, const vsk_head_rows *k,
                         const vsk_head_rows *v, const vsk_rotary *rotary,
                         const vsk_head_rows *q) {
  QUEUED_API_BEGIN(ctx);
  VSK_REQUIRE(kv && news && k && v, VSK_ERR_INVALID_ARGUMENT, "null argument");
  check_kv(kv);
  check_news(news);
  VSK_REQUIRE(layer >= 0 && layer < kv->layers, VSK_ERR_INVALID_ARGUMENT, "no such layer");
  VSK_REQUIRE(k->heads == kv->kv_heads && v->heads == kv->kv_heads, VSK_ERR_DIMENSION_MISMATCH,
              "keys and values must have the cache's heads");
  VSK_REQUIRE(!rotary || 2 * rotary->pairs <= kv->head_dim, VSK_ERR_DIMENSION_MISMATCH,
              "a head holds fewer values than the rotation turns");
  if (news->n == 0 || news->tokens == 0 || news->max_new == 0) return VSK_OK;
  VSK_REQUIRE(news->seqs || news->n <= kv->slots, VSK_ERR_INVALID_ARGUMENT,
              "more sequences than the cache has slots");
  VSK_REQUIRE(news->starts || news->tokens >= news->n, VSK_ERR_DIMENSION_MISMATCH,
              "fewer rows than sequences");
  RotaryArgs a{};
  const int64_t size = kv->dtype == VSK_DTYPE_F32 ? 4 : 2;
  int at = 0;
  if (q) {
    VSK_REQUIRE(q->dst && is_device_ptr(q->dst), VSK_ERR_INVALID_ARGUMENT,
                "tensors must be device memory");
    a.x[at++] = rows_of(*q, rotary != nullptr);
  }
  a.x[at] = rows_of(*k, rotary != nullptr);
  a.x[at].dst = static_cast<char *>(kv->k) + layer * kv->k_layer * size;
  a.x[at].dst_page = kv->k_page;
  a.x[at].dst_row = kv->k_row;
  a.x[at].dst_head = kv->k_head;
  a.x[at++].paged = 1;
  a.x[at] = rows_of(*v, false);
  a.x[at].dst = static_cast<char *>(kv->v) + layer * kv->v_layer * size;
  a.x[at].dst_page = kv->v_page;
  a.x[at].dst_row = kv->v_row;
  a.x[at].dst_head = kv->v_head;
  a.x[at++].paged = 1;
  if (rotary) set_rotary(a, rotary);
  a.starts = news->starts;
  a.seqs = news->seqs;
  a.lengths = kv->lengths;
  a.table = kv->table;
  a.table_stride = kv->table_stride;
  a.tokens = news->tokens;
  a.n = news->n;
  a.max_new = news->starts ? news->max_new : 1;
  a.slots = kv->slots;
  a.width = kv->width;
  a.pages_n = kv->pages;
  a.page_shift = __builtin_ctz((unsigned)kv->page_size);
  a.d = kv->head_dim;
  hipStream_t st = static_cast<hipStream_t>(stream);
  launch_rotary(ctx, st, a, kv->dtype);
  finish_queued(ctx, st);
  VSK_API_END(ctx);
}

}  // extern "C"
