// attn.hpp -- what the attention kernels share: the operands of one call, the
// keys that a tile of query rows sees, and the 16- and 32-bit element types.
//
// A sequence's new tokens are its last ones: of T new tokens over a length L
// (the new ones included), token t stands at position L - T + t and sees key
// j when j <= its position and (no window, or position - j < window, or
// j < sinks).  The query heads of one key head are packed into rows, row =
// token * group + head within the group, so that keys and values are read
// once for all of them.
//
// Cross attention: every new token stands at the last key and sees them all.
// A shared prefix is two such calls whose sums are joined: the new tokens of a
// group of sequences, as if of one, over the keys that they share, and each
// sequence over its keys from there on.
#pragma once

#include "device_scope.hpp"
#include "vsk_core.hpp"

// VSK_API_BEGIN (vsk_api.hpp) of a call that a program makes between its own:
// the current device is what it was when the call returns.
#define QUEUED_API_BEGIN(ctx)                              \
  if (!(ctx)) return VSK_ERR_INVALID_ARGUMENT;             \
  const ::vsk::DeviceScope vsk_device_scope_((ctx)->device); \
  VSK_API_BEGIN(ctx)

namespace vsk {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

// Kernels of the plain form (a sequence's own keys, causal) and of the others,
// whose arguments say which.  Apart at compile time: what a block asks of its
// arguments before its first key costs one short context (11.1 us) 0.5 us.
enum AttnForm { ATTN_OWN, ATTN_FORMS };

// The operands of a call, by value to every kernel.  Strides in elements.
struct AttnArgs {
  const void *q, *k, *v;
  void *out;
  float *lse;  // tokens x heads, or null
  int64_t q_row, q_head, o_row, o_head;
  int64_t k_page, k_row, k_head, v_page, v_row, v_head;
  const int32_t *table;    // slots x width page ids; null: dense rows
  const int32_t *lengths;  // per slot (paged)
  const int32_t *starts;   // n + 1 offsets of the sequences' tokens, or null: one each
  const int32_t *seqs;     // slot (cross: set of keys) of each sequence, or null
  const int32_t *prefix;   // per sequence: keys that its group shares, or null
  const int32_t *groups;   // n + 1 offsets of the groups' sequences: a call over prefixes
  const int32_t *k_starts; // n + 1 offsets of the sequences' keys (dense)
  const int32_t *k_lengths;  // (cross, no k_starts) keys of each set, or null: all its rows
  int64_t table_stride;
  int64_t tokens, k_rows;
  int32_t n, heads, kv_heads, group, d;
  int32_t pages, page_shift, slots, width;
  int32_t window, sinks;  // window <= 0: none
  int32_t max_new;
  // ATTN_FORMS
  int32_t cross;        // every token sees every key
  int32_t sets;         // sets of keys (cross)
  int64_t set_rows;     // rows from a set to the next where there are no k_starts
  int32_t members;      // sequences that the groups' offsets may name
  int32_t joined;       // parts are written also where there is one, absent ones marked
  int32_t part0;        // the call's first part
  int32_t parts_apart;  // one part of every sequence, then the next
  // two calls in one launch: the first pre_blocks blocks are those of a call
  // over prefixes, which differs in these
  uint32_t pre_blocks, own_blocks;
  struct {
    int32_t n, max_new, tiles, splits, chunk;
  } pre;
  int32_t tiles;        // row tiles of a sequence's max_new tokens
  int32_t splits;       // parts a tile's keys may be split into
  int32_t chunk;        // key tiles of a part
  float scale_log2;     // scale * log2(e)
  float *part_o;        // splits x tokens x heads x d
  float *part_ml;       // splits x tokens x heads x 2: reference (a score), sum
};

// One sequence of the call (or one group of them, over its prefix).
struct AttnSeq {
  int64_t token0, key0;  // its first row in q; its first dense key
  int64_t row;           // its first entry of the table
  int32_t T, L;          // new tokens, keys
  int32_t p0, each;      // token t stands at p0 + (t & each)
  int32_t first, end;    // (a group) its sequences
};

__device__ inline int32_t attn_length(const AttnArgs &a, int32_t slot) {
  const int64_t most = (int64_t)a.width << a.page_shift;
  const int32_t l = a.lengths[slot];
  return l < 0 ? 0 : l > most ? (int32_t)most : l;
}

// Every index below is taken from device memory, so each is held to its
// buffer here: a slot, length or offset out of range reads no foreign memory.
template <AttnForm F> __device__ inline AttnSeq attn_seq(const AttnArgs &a, int32_t b) {
  AttnSeq s;
  s.first = b, s.end = b + 1;
  if (F && a.groups) {
    s.first = a.groups[b], s.end = a.groups[b + 1];
    s.first = s.first < 0 ? 0 : s.first > a.members ? a.members : s.first;
    s.end = s.end < s.first ? s.first : s.end > a.members ? a.members : s.end;
    b = s.first < a.members ? s.first : 0;  // (whose keys; of an empty group none are read)
  }
  if (a.starts) {
    int32_t t0 = a.starts[s.first], t1 = a.starts[s.end];
    t0 = t0 < 0 ? 0 : t0;
    if (t1 > a.tokens) t1 = (int32_t)a.tokens;
    s.token0 = t0;
    s.T = t1 > t0 ? t1 - t0 : 0;
  } else {
    s.token0 = s.first;
    s.T = s.end - s.first;
  }
  const int32_t slot = a.seqs ? a.seqs[b] : b;
  s.key0 = 0;
  s.row = 0;
  s.L = 0;
  if (a.table) {
    if ((uint32_t)slot < (uint32_t)a.slots) {
      s.row = slot * a.table_stride;
      s.L = attn_length(a, slot);
      if (F && a.prefix) {
        // whole pages: the keys that a group shares, or a sequence's others
        int32_t pages = a.prefix[b] >> a.page_shift;
        pages = pages < 0 ? 0 : pages > a.width ? a.width : pages;
        const int32_t keys = pages << a.page_shift;
        if (a.groups) {
          s.L = keys;  // (also where the first member has been cut back since)
        } else {
          s.row += pages;
          s.L = s.L > keys ? s.L - keys : 0;
        }
      }
    }
  } else if (!F || a.k_starts) {
    const int32_t set = F ? slot : b;
    if (!F || (uint32_t)set < (uint32_t)a.sets) {
      int64_t k0 = a.k_starts[set], k1 = a.k_starts[set + 1];
      k0 = k0 < 0 ? 0 : k0;
      if (k1 > a.k_rows) k1 = a.k_rows;
      s.key0 = k0;
      s.L = k1 > k0 ? (int32_t)(k1 - k0) : 0;
    }
  } else if ((uint32_t)slot < (uint32_t)a.sets) {
    s.key0 = slot * a.set_rows;
    const int32_t l = a.k_lengths ? a.k_lengths[slot] : (int32_t)a.k_rows;
    s.L = l < 0 ? 0 : l > a.k_rows ? (int32_t)a.k_rows : l;
  }
  s.p0 = F && a.cross ? s.L - 1 : s.L - s.T;
  s.each = F && a.cross ? 0 : -1;
  return s;
}

// The sequence (or group) and part of a block, with heads and row tiles taken
// out of its number.
struct AttnTurn {
  int32_t b, part;
};
template <AttnForm F> __device__ inline AttnTurn attn_turn(const AttnArgs &a, uint32_t at) {
  if (F == ATTN_OWN || !a.parts_apart)
    return {(int32_t)(at / a.splits), (int32_t)(at % a.splits)};
  return {(int32_t)(at % a.n), (int32_t)(at / a.n)};
}

// Position of the sequence's new token t among its keys.  Of a group's, it is
// the position in the token's own sequence, found among the group's, or the
// prefix's last.
template <AttnForm F>
__device__ inline int32_t attn_position(const AttnArgs &a, const AttnSeq &s, int32_t t) {
  if (!F || !a.groups) return s.p0 + (t & s.each);
  int32_t b = s.first + t, at = 0, count = 1;
  if (a.starts) {
    const int32_t token = (int32_t)s.token0 + t;
    b = s.first;
    for (int32_t end = s.end; end - b > 1;) {
      const int32_t mid = b + (end - b) / 2;
      if (a.starts[mid] <= token)
        b = mid;
      else
        end = mid;
    }
    at = token - a.starts[b];
    count = a.starts[b + 1] - a.starts[b];
  }
  const int32_t slot = a.seqs ? a.seqs[b] : b;
  if ((uint32_t)slot >= (uint32_t)a.slots) return -1;
  const int64_t pos = (int64_t)attn_length(a, slot) - count + at;
  return pos >= s.L ? s.L - 1 : pos < -1 ? -1 : (int32_t)pos;
}

// the call over prefixes of the two
__device__ inline void attn_prefix_call(AttnArgs &a) {
  a.n = a.pre.n, a.max_new = a.pre.max_new;
  a.tiles = a.pre.tiles, a.splits = a.pre.splits, a.chunk = a.pre.chunk;
  a.part0 = 0;
}
// The call that a block belongs to, and its number there.
__device__ inline uint32_t attn_call(AttnArgs &a, uint32_t block) {
  if (a.pre_blocks == 0) return block;
  if (block >= a.pre_blocks) {
    a.groups = nullptr;
    return block - a.pre_blocks;
  }
  attn_prefix_call(a);
  return block;
}

// The keys that query positions q0 .. q1 see between them, in groups of G keys
// and tiles of KT: the sinks' groups from 0, then the groups from lo on.
template <int KT, int G> struct AttnSpan {
  int32_t lo, hi, sink_groups, tiles;
  // first key of a group
  __device__ int32_t group(int32_t g) const {
    return g < sink_groups ? G * g : lo + G * (g - sink_groups);
  }
  __device__ int32_t base(int32_t t) const { return group(KT / G * t); }
};
template <int KT, int G>
__device__ inline AttnSpan<KT, G> attn_span(const AttnArgs &a, int32_t q0, int32_t q1) {
  AttnSpan<KT, G> s;
  s.hi = q1 + 1 > 0 ? q1 + 1 : 0;
  s.lo = 0;
  s.sink_groups = 0;
  if (a.window > 0) {
    const int64_t first = (int64_t)q0 - a.window + 1;
    if (first > 0) {
      const int32_t lo = (int32_t)first & ~(G - 1);
      const int32_t st = a.sinks / G + (a.sinks % G != 0);
      if ((int64_t)st * G < lo) {
        s.lo = lo;
        s.sink_groups = st;
      }
    }
  }
  const int32_t groups = s.sink_groups + (s.hi > s.lo ? (s.hi - s.lo - 1) / G + 1 : 0);
  s.tiles = (groups + KT / G - 1) / (KT / G);
  return s;
}

// Parts of `tiles` key tiles: part s holds tiles s * chunk on, the last part
// all that is left (a length over the caller's bound only makes it longer).
__device__ inline int32_t attn_parts(const AttnArgs &a, int32_t tiles) {
  const int32_t p = (tiles + a.chunk - 1) / a.chunk;
  return p < 1 ? 1 : p > a.splits ? a.splits : p;
}

// A part that is not there, of query row r of key head h: the sums of no keys.
__device__ inline void attn_empty_part(const AttnArgs &a, const AttnSeq &s, int32_t h, int32_t r,
                                       int32_t part) {
  const int64_t row = (s.token0 + r / a.group) * a.heads + h * a.group + r % a.group;
  const int64_t x = (int64_t)(a.part0 + part) * a.tokens * a.heads + row;
  a.part_ml[2 * x] = -INFINITY;
  a.part_ml[2 * x + 1] = 0.f;
}

__device__ inline bool attn_sees(const AttnArgs &a, int32_t pos, int32_t j) {
  return j <= pos && (a.window <= 0 || pos - j < a.window || j < a.sinks);
}

// Base (in elements) of the 16 keys from j16 on (a multiple of 16; pages hold
// a multiple of 16) and how many of the 16 rows may be read.  The keys from L
// on read row L - 1: they are masked, and their memory may not exist.
struct AttnRows {
  int64_t k, v;
  int32_t last;
};
__device__ inline int32_t attn_row16(const AttnSeq &s, int32_t j16) {
  const int32_t tail = (s.L - 1) & ~15;
  return j16 < tail ? j16 : tail;
}
// The page that holds them, as the table has it (dense: 0): for the paths that
// take keys one at a time.  The index is hidden from the compiler: a scalar load
// of it would keep scalars that the loops around have no registers for (one
// context of 777: 11.3 us, 11.1 with it).
__device__ inline int32_t attn_page(const AttnArgs &a, const AttnSeq &s, int32_t j16) {
  if (!a.table) return 0;
  int32_t i = attn_row16(s, j16) >> a.page_shift;
  asm volatile("" : "+v"(i));
  return a.table[s.row + i];
}
__device__ inline AttnRows attn_rows(const AttnArgs &a, const AttnSeq &s, int32_t h, int32_t j16,
                                     int32_t page) {
  AttnRows r;
  page = __builtin_amdgcn_readfirstlane(page);
  page = page < 0 ? 0 : page >= a.pages && a.table ? a.pages - 1 : page;
  const int32_t j = attn_row16(s, j16);
  r.last = s.L - 1 - j < 15 ? s.L - 1 - j : 15;
  const int64_t in = a.table ? j & ((1 << a.page_shift) - 1) : s.key0 + j;
  r.k = page * a.k_page + in * a.k_row + h * a.k_head;
  r.v = page * a.v_page + in * a.v_row + h * a.v_head;
  return r;
}

#define lds_as __attribute__((address_space(3)))
// A pointer made of an integer is generic unless it says where it points, and
// a generic (flat) load counts as one of LDS too: only a wait for none of them
// is sound behind it.
#define global_as __attribute__((address_space(1)))
typedef lds_as char lds_char;

// 16 bytes a lane from base + off to dst + 16 * lane (base and dst the same in
// every lane).  Written as assembly because the compiler makes every read of
// LDS after the builtin wait for it: here a tile's copies fly while the last
// tile is computed with, and one wait before the barrier covers them.  (M0
// holds the destination of such loads; the compiler is told.)
__device__ inline void load_to_lds(uint64_t base, uint32_t off, const lds_char *dst) {
  const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)dst);
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2"
      :
      : "s"(at), "v"(off), "s"(base)
      : "memory", "m0");
}

__device__ inline uint64_t lane_of(uint32_t lo, uint32_t hi, int i) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, i) << 32 |
         (uint32_t)__builtin_amdgcn_readlane(lo, i);
}

// A row of CH 16-byte pieces in LDS: piece c of it is in slot c ^ swizzle(row),
// so that the rows that a quarter (half) of a wave reads the same piece of
// meet different banks.
template <int CH> __device__ inline int k_swizzle(int row) {
  return CH >= 16 ? row & 15 : (row & 7) ^ ((row >> 3) & 1);
}

// (fmaxf would first quiet each product, an instruction a value: the maximum
// here passes over NaN without it.)  Nothing waits for a matrix product before
// assembly reads it: a chain of maxima starts from product_read() of the last
// products, which it depends on.
__device__ inline float product_read(float x) { return __builtin_canonicalizef(x); }
__device__ inline float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

__device__ inline float attn_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// log of a row's sum, whose weights are 2^(score * scale_log2 - ref)
__device__ inline float attn_lse(float ref, float sum) {
  return sum > 0.f ? (ref + __log2f(sum)) * 0.6931471805599453f : sum != sum ? sum : -INFINITY;
}
// Exchanges between lanes 16 and 32 apart on the vector unit: of x twice, the
// swap of the odd rows (the upper half) of the one with the even rows (the
// lower half) of the other leaves each pair's two values in the two results.
__device__ inline void pair32(float x, float *lo, float *hi) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  *lo = __uint_as_float(r[0]), *hi = __uint_as_float(r[1]);
}
__device__ inline void pair16(float x, float *lo, float *hi) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  *lo = __uint_as_float(r[0]), *hi = __uint_as_float(r[1]);
}
__device__ inline float xor32_max(float x) {
  float a, b;
  pair32(x, &a, &b);
  return fmaxf(a, b);
}
__device__ inline float xor32_sum(float x) {
  float a, b;
  pair32(x, &a, &b);
  return a + b;
}
__device__ inline float xor16_32_max(float x) {
  float a, b;
  pair16(x, &a, &b);
  return xor32_max(fmaxf(a, b));
}
__device__ inline float xor16_32_sum(float x) {
  float a, b;
  pair16(x, &a, &b);
  return xor32_sum(a + b);
}

// what the entry points check of a cache and of a call's tokens (kvcache.hip)
void check_kv(const vsk_kv *kv);
void check_news(const vsk_new_tokens *news);
// the end of a call that is queued: nothing, or, with profiling on, a wait for
// the stream and the timers' results
void finish_queued(vsk_ctx *ctx, hipStream_t stream);

// launches; attn_rows.hip; t: a VSK_DTYPE; aligned: every pointer and
// stride takes 16-byte loads (8-byte stores)
// share: waves that take a row tile's keys in turn: 8 (heads to 128, in 32 bits
// to 64), 4, or 1
void launch_attn_rows(vsk_ctx *ctx, hipStream_t stream, const AttnArgs &a, int32_t t,
                      bool aligned, int32_t share);
// attn_forms.hip: the same of ATTN_FORMS (with a.pre: both of its calls)
void launch_attn_rows_forms(vsk_ctx *ctx, hipStream_t stream, const AttnArgs &a, int32_t t,
                            bool aligned, int32_t share);
// keys of a tile of attn_tile.hip, by the (padded) head
constexpr int attn_tile_keys(int d) { return d > 128 ? 32 : 64; }
// attn_tile.hip: 16-bit types, aligned, row tiles of ATTN_TILE_ROWS
constexpr int ATTN_TILE_ROWS = 128;
constexpr int ATTN_TILE_GROUP = 16;  // keys that lie together in a tile
void launch_attn_tile(vsk_ctx *ctx, hipStream_t stream, const AttnArgs &a, int32_t t,
                      AttnForm form);
// attn_tile32.hip: 32 bits, aligned, heads of 65 to 128, ATTN_FORMS, the same row tiles
constexpr int ATTN_TILE32_KEYS = 32;
void launch_attn_tile32(vsk_ctx *ctx, hipStream_t stream, const AttnArgs &a);
// attn_shared.hip: 16 bits, aligned, heads to 128: a.pre by row tiles of ATTN_TILE_ROWS, the
// call itself by those of 16, four waves each
void launch_attn_shared(vsk_ctx *ctx, hipStream_t stream, AttnArgs a, int32_t t);
// joins the parts that row tiles of `rows` rows left: 16 (launch_attn_rows) or
// ATTN_TILE_ROWS
void launch_attn_join(vsk_ctx *ctx, hipStream_t stream, const AttnArgs &a, int32_t t,
                      bool aligned, int32_t rows);
// attn_forms.hip: the same of ATTN_FORMS; key_tile: keys of a tile of the parts
void launch_attn_join_forms(vsk_ctx *ctx, hipStream_t stream, const AttnArgs &a, int32_t t,
                            bool aligned, int32_t key_tile);

}  // namespace vsk
