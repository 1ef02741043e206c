// The kernels and plans that the attention of many sequences shares: packed prompts and the batch behind a shared prefix
// (fh_packed.hip, whose comment says what they do), and rows over a cache in pages (fh_paged.hip).
#pragma once
#include <math.h>
#include <algorithm>
#include <type_traits>
#include "fh_common.h"

namespace fh {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float floatx16;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short short4v;
typedef __attribute__((__vector_size__(8 * sizeof(short)))) short short8v;
#define SEQ_LDS __attribute__((address_space(3)))
// 16 bytes a lane from memory to LDS, the wave's 1 KB from `to` on in lane order. Written as an instruction so that the compiler
// does not hold every transposed read of LDS for all the loads in flight, as it does behind the builtin (the ring's waits are
// the kernel's own; a count that leaves these loads out only waits longer).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is nobody's here)
__device__ __forceinline__ void load_to_lds(const void* from, uint16_t* to) {
  const uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uintptr_t)(SEQ_LDS uint16_t*)to);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(from), "s"(at) : "memory", "m0");
}
// the same from a wave-uniform base and a lane's own offset
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint16_t* to) {
  const uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uintptr_t)to);  // (an LDS address' low half is its offset)
  const uint64_t b = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)((uint64_t)base >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint64_t)base);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2" :: "v"(offset), "s"(at), "s"(b) : "memory", "m0");
}
#pragma clang diagnostic pop

constexpr int SQ_NW = 4;               // waves a workgroup
constexpr float SQ_SLACK = 8.f;        // how far a score may lie above the running max, in base 2

// which entry point's rows and keys: a batch behind a prefix, packed prompts, or packed rows over a cache in pages
enum SeqForm { SEQ_SHARED, SEQ_PACKED, SEQ_PAGED };

struct SeqArgs {
  const void* q; int q_bf16; int64_t ldq;
  const void* cache; int64_t cache_len; const uint8_t* cache_exps;
  int heads, kv_heads, rep; float scale;
  int64_t rows; int n;          // query rows; sequences
  const int32_t* starts;        // [n + 1] each sequence's first row (NULL: a decode step, row b is sequence b)
  const int32_t* places;        // [n] the place of a sequence's first row
  const int32_t* first_row; const int32_t* prefix_row; const int32_t* shared;
  int64_t max_prefix, max_own;  // bounds of shared, and of the places behind it
  // (pages) each sequence's pages, 2^page_shift rows each; rows a tile, tiles of a row's heads, workgroups a tile of heads shares its
  // keys among, pairs a part holds, the least share of a workgroup (SeqWalk)
  const int32_t* tables; int64_t ldt; int table_cols, pages, page_shift;
  int tile_rows, head_tiles, walkers, slot_pairs, least, unit, uncut, whole;
  int splits, own_splits;       // workgroups the keys are split among (a decode step's prefix; each row's own keys)
  int tiles;                    // tiles of pairs (a decode step's prefix)
  int parts;                    // parts a pair (1: the kernel writes o)
  float* part;                  // [rows][heads][parts][hd + 2]: weighted sum, max (in base 2), sum of weights
  void* o; int o_bf16, o_tiles; int64_t ldo;
};

// what a workgroup does: pairs pair0 .. of `pairs` of the rows from row0 on, keys of tiles first .. last of those they see
struct SeqItem {
  int64_t row0; int pair0, pairs;   // pair p: row row0 + p / rep, head p % rep of the group
  int kvh, split, splits, part;
  int64_t prefix, own; int shared;  // key k's cache row: prefix + k below shared, own + k from there on
  const int32_t* table;             // (pages) the sequence's
  int t0, t1, slot;                 // (pages) the tiles of keys from t0 to t1 alone, into this part (-1: all there are, into o)
  int place0, step;                 // pair p sees keys 0 .. place0 + step (p / rep) of them; step -1: each row's own count
};

__device__ inline int clampi(int64_t v, int64_t lo, int64_t hi) { return (int)(v < lo ? lo : v > hi ? hi : v); }

// A row of a decode step: its prefix's places and its own that it sees
__device__ inline void row_counts(const SeqArgs& a, int64_t b, int& shared, int& in_prefix, int& own) {
  shared = clampi(a.shared[b], 0, a.max_prefix);
  const int64_t seen = (int64_t)a.places[b] + 1;
  in_prefix = clampi(seen, 0, shared);
  own = clampi(seen - shared, 0, a.max_own);
}

// The workgroup's item (false: none). Blocks of one key head lie kv_heads apart: with 8 key heads they share an XCD's L2.
template <int BQ, int FORM>
__device__ inline bool seq_item(const SeqArgs& a, SeqItem& it) {
  int blk = blockIdx.x;
  it.kvh = blk % a.kv_heads;
  blk /= a.kv_heads;
  if constexpr (FORM == SEQ_SHARED) {
    if (blk < a.tiles * a.splits) {  // the prefix: tiles of all rows' pairs
      it.split = blk % a.splits; it.splits = a.splits; it.part = it.split;
      it.row0 = 0; it.pair0 = (blk / a.splits) * BQ; it.pairs = (int)a.rows * a.rep;
      it.prefix = a.prefix_row[0]; it.own = 0; it.shared = 0x7FFFFFFF;
      it.place0 = 0; it.step = -1;
      return true;
    }
    blk -= a.tiles * a.splits;       // a row's own keys: the tiles of its pairs (one, but for more heads a key head than pairs a tile)
    it.split = blk % a.own_splits; it.splits = a.own_splits; it.part = a.splits + it.split;
    const int row_tiles = (a.rep + BQ - 1) / BQ;
    const int64_t b = blk / a.own_splits / row_tiles;
    it.pair0 = blk / a.own_splits % row_tiles * BQ;
    int sh, pre, own;
    row_counts(a, b, sh, pre, own);
    it.row0 = b; it.pairs = a.rep;
    it.prefix = 0; it.own = a.first_row[b]; it.shared = 0;
    it.place0 = own - 1; it.step = 0;
    return true;
  } else {
    it.split = it.part = blk % a.splits; it.splits = a.splits;
    const int tile = blk / a.splits, lane = threadIdx.x & 63;
    const int prefix = a.shared ? a.prefix_row[0] : 0;
    int before = 0;
    for (int s0 = 0; s0 < a.n; s0 += 64) {  // 64 sequences a round: the one whose tiles hold this one
      const int s = min(s0 + lane, a.n - 1);
      const int st = a.starts[s], en = a.starts[s + 1], place = a.places[s], first = a.first_row[s], shd = a.shared ? a.shared[s] : 0;
      const int lo = clampi(st, 0, a.rows), len = s0 + lane < a.n ? clampi(en, lo, a.rows) - lo : 0;
      const int tiles = (int)(((int64_t)len * a.rep + BQ - 1) / BQ);
      int incl = tiles;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d, 64);
        if (lane >= d) incl += o;
      }
      const uint64_t has = __ballot(tile < before + incl);
      if (has) {
        const int at = __builtin_ctzll(has);
        const int nt = __builtin_amdgcn_readlane(tiles, at), in = __builtin_amdgcn_readlane(incl, at);
        const int t = nt - 1 - (tile - (before + in - nt));  // (a sequence's longest tile first)
        it.row0 = __builtin_amdgcn_readlane(lo, at); it.pair0 = t * BQ; it.pairs = __builtin_amdgcn_readlane(len, at) * a.rep;
        it.shared = a.shared ? clampi(__builtin_amdgcn_readlane(shd, at), 0, a.max_prefix) : 0;
        it.prefix = prefix;
        it.own = (int64_t)__builtin_amdgcn_readlane(first, at) - it.shared;
        it.place0 = __builtin_amdgcn_readlane(place, at); it.step = 1;
        return true;
      }
      before += __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
  }
}

// how many keys pair p of the item sees
__device__ inline int pair_limit(const SeqArgs& a, const SeqItem& it, int p) {
  if (p >= it.pairs) return 0;
  if (it.step >= 0) return clampi((int64_t)it.place0 + (int64_t)it.step * (p / a.rep) + 1, 0, it.step ? a.max_own : 0x7FFFFFFF);
  int sh, pre, own;
  row_counts(a, p / a.rep, sh, pre, own);
  return pre;
}

// the largest of a value over the wave
__device__ inline int wave_most(int v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = max(v, __shfl_xor(v, d, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

// Rows over pages: how the work is shared. A sequence's rows go in tiles of `tile_rows`, each a number of tiles of 64 keys, and a
// tile's cost is its keys and SEQ_START more (what it takes before its first key and behind its last, in keys; both in units
// of 2^unit, so that a call's sum stays below 2^30). The tiles of all sequences lie one after another along their cost, and `walkers`
// workgroups a key head take equal shares of it, so that tokens after few and many places, and prompts' tiles, keep the GPU equally long
// together. A share that begins or ends inside a tile leaves a part of it, which seq_join_pages joins; one that begins in a tile's first
// SEQ_START, or anywhere in one that costs less than `uncut`, begins with the tile. For `whole` a workgroup takes a sequence and head as they are. All of it is a function of the arrays alone: a call repeats its bits.
constexpr int SEQ_START = 128;
// the sum of a value over this lane and those before
__device__ inline int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // (within rows of 16 lanes, by 1, 2, 4 and 8)
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // (a row's last lane to the next row, then the lower half's to the upper)
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}
struct SeqWalk {
  int total, share, first;            // `first`: the sequence of held[0]
  int seq, at, lo, len, place, tiles; // the sequence at hand, the cost before it, its rows and tiles
  int4* held;                         // (LDS, the wave's own) 64 sequences' rows, places and the cost up to their end

  // the cost of the first t tiles of rows behind `place` places
  __device__ static int cost(const SeqArgs& a, int place, int t) {
    return (int)((int64_t)t * (((clampi(place, 0, a.max_own) + SEQ_START) >> a.unit) + 1) +  // (a unit at least beyond SEQ_START's)
                  (int64_t)t * (t + 1) / 2 * (a.tile_rows >> a.unit));
  }
  __device__ static int tiles_of(const SeqArgs& a, int len) { return (len + a.tile_rows - 1) / a.tile_rows; }
  // sequences s0 .. s0 + 63, behind cost `before`: into LDS; the cost up to the last of them
  __device__ int load(const SeqArgs& a, int s0, int before) {
    const int lane = threadIdx.x & 63, i = min(s0 + lane, a.n - 1);
    const int st = a.starts[i], en = a.starts[i + 1], p = a.places[i];
    const int l = clampi(st, 0, a.rows), n = s0 + lane < a.n ? clampi(en, l, a.rows) - l : 0;
    const int end = before + wave_scan(cost(a, p, tiles_of(a, n)));
    wave_lds_order();
    held[lane] = make_int4(l, n, p, end);
    wave_lds_order();
    first = s0;
    return __builtin_amdgcn_readlane(end, 63);
  }
  __device__ void start(const SeqArgs& a, int4* lds) {
    held = lds + (threadIdx.x >> 6) * 64;
    total = load(a, 0, 0);
    for (int s0 = 64; s0 < a.n; s0 += 64) total = load(a, s0, total);
    share = max((total + a.walkers - 1) / a.walkers, a.least);
  }
  // to the sequence whose tiles hold cost x < total, from the 64 sequences held on: every x is at least the last one sought
  __device__ void seek(const SeqArgs& a, int x) {
    for (;;) {
      const uint64_t has = __ballot(held[threadIdx.x & 63].w > x);
      if (has) {
        const int l = __builtin_ctzll(has);
        const int4 h = held[l];
        lo = __builtin_amdgcn_readfirstlane(h.x); len = __builtin_amdgcn_readfirstlane(h.y); place = __builtin_amdgcn_readfirstlane(h.z);
        tiles = tiles_of(a, len);
        at = __builtin_amdgcn_readfirstlane(h.w) - cost(a, place, tiles);
        seq = first + l;
        return;
      }
      load(a, first + 64, __builtin_amdgcn_readfirstlane(held[63].w));
    }
  }
  __device__ void seek_from_start(const SeqArgs& a, int x) {
    if (first > 0) load(a, 0, 0);
    seek(a, x);
  }
  // the tile of the sequence at hand that holds cost x (at <= x)
  __device__ int tile_at(const SeqArgs& a, int x) const {
    if (tiles == 1) return 0;
    const float r = a.tile_rows >> a.unit, b = (float)(((clampi(place, 0, a.max_own) + SEQ_START) >> a.unit) + 1) + 0.5f * r, y = (float)(x - at);
    int t = __builtin_amdgcn_readfirstlane(clampi((int64_t)(r > 0.f ? (sqrtf(b * b + 2 * r * y) - b) / r : y / b), 0, tiles - 1));
    while (t > 0 && at + cost(a, place, t) > x) --t;
    while (t + 1 < tiles && at + cost(a, place, t + 1) <= x) ++t;
    return t;
  }
  // tile t's keys, in tiles of `bk`
  __device__ int key_tiles_of(const SeqArgs& a, int t, int bk) const {
    return (clampi((int64_t)place + min((t + 1) * a.tile_rows, len), 0, a.max_own) + bk - 1) / bk;
  }
  // where cost x cuts a tile whose cost is from c0 to c1: at which of its n tiles of keys
  __device__ static int cut(const SeqArgs& a, int c0, int c1, int n, int x) {
    if (x >= c1) return n;
    const int in = x - c0 - (SEQ_START >> a.unit);
    return in <= 0 || c1 - c0 < a.uncut ? 0 : min((int)((float)in * ((float)n / (float)(c1 - c0 - (SEQ_START >> a.unit)))), n);
  }
};

// the first cache row of the page that the sequence's table names for its place k (a page outside the cache: the nearest)
__device__ inline int64_t page_row(const SeqArgs& a, int page) { return (int64_t)clampi(page, 0, a.pages - 1) << a.page_shift; }
template <int FORM>
__device__ inline int64_t key_row(const SeqArgs& a, const SeqItem& it, int k) {
  if constexpr (FORM == SEQ_PAGED) return page_row(a, it.table[min(k >> a.page_shift, a.table_cols - 1)]) + (k & ((1 << a.page_shift) - 1));
  const int64_t r = (k < it.shared ? it.prefix : it.own) + k;
  return r < 0 ? 0 : r >= a.cache_len ? a.cache_len - 1 : r;
}

// the page of place k, the same for the wave, by the scalar unit
__device__ inline int table_page(const SeqArgs& a, const SeqItem& it, int k) {
  return ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)it.table)[min(__builtin_amdgcn_readfirstlane(k) >> a.page_shift, a.table_cols - 1)];
}

__device__ inline uint32_t pack2_rne(float lo, float hi) { return bf16_rne_f(lo) | (bf16_rne_f(hi) << 16); }

// four values of a row of o, columns col .. col + 3
__device__ inline void put4(const SeqArgs& a, int64_t row, int64_t col, float4 v) {
  const int64_t at = a.o_tiles ? tile16_at(row, col, a.ldo) : row * a.ldo + col;
  if (a.o_bf16) *(uint2*)((uint16_t*)a.o + at) = make_uint2(pack2_rne(v.x, v.y), pack2_rne(v.z, v.w));
  else *(float4*)((float*)a.o + at) = v;
}

// a cache row's value, whatever the cache holds
template <int HD, int CF>
__device__ inline float cache_value(const SeqArgs& a, int64_t row, int c) {
  if constexpr (CF == FH_F32) return ((const float*)a.cache)[row * HD + c];
  else if constexpr (CF == FH_BF16) return bf16_to_f(((const uint16_t*)a.cache)[row * HD + c]);
  else {
    const uint32_t e = a.cache_exps[row * (HD / 16) + c / 16];
    int q;
    if constexpr (CF == FH_BFP8) q = ((const int8_t*)a.cache)[row * HD + c];
    else q = (int)(int8_t)(((const uint8_t*)a.cache)[row * (HD / 2) + c / 2] << ((c & 1) ? 0 : 4)) >> 4;
    return bf16_to_f(bfp_value_bf16(CF == FH_BFP4 ? 16 * q : q, e));
  }
}

// 8 values of a cache row as loaded: 16 bytes of bf16, 32 of fp32, or a block float's magnitudes and exponent
struct SeqRaw { uint4 a, b; uint32_t e; };
template <int HD, int CF>
__device__ inline SeqRaw seq_raw(const SeqArgs& a, int64_t row, int c) {
  SeqRaw r;
  if constexpr (CF == FH_BF16) r.a = *(const uint4*)((const uint16_t*)a.cache + row * HD + c);
  else if constexpr (CF == FH_F32) {
    const uint4* p = (const uint4*)((const float*)a.cache + row * HD + c);
    r.a = p[0]; r.b = p[1];
  } else {
    if constexpr (CF == FH_BFP8) { const uint2 m = *(const uint2*)((const uint8_t*)a.cache + row * HD + c); r.a.x = m.x; r.a.y = m.y; }
    else r.a.x = *(const uint32_t*)((const uint8_t*)a.cache + row * (HD / 2) + c / 2);
    r.e = a.cache_exps[row * (HD / 16) + c / 16];
  }
  return r;
}
template <int CF>
__device__ inline uint4 seq_bf16x8(const SeqRaw& r) {
  static_assert(CF != FH_F32, "an fp32 cache goes in as fp32");
  if constexpr (CF == FH_BF16) return r.a;
  else {
    float f[8];
    uint32_t w[4];
    if constexpr (CF == FH_BFP8) magnitudes8(make_uint2(r.a.x, r.a.y), f);
    else magnitudes8(r.a.x, f);
    bfp_run_bf16<8>(f, r.e, w);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// (an fp32 cache's)
__device__ inline void seq_f32x8(const SeqRaw& r, float4& x, float4& y) {
  x = make_float4(__uint_as_float(r.a.x), __uint_as_float(r.a.y), __uint_as_float(r.a.z), __uint_as_float(r.a.w));
  y = make_float4(__uint_as_float(r.b.x), __uint_as_float(r.b.y), __uint_as_float(r.b.z), __uint_as_float(r.b.w));
}

__device__ inline float q_value(const SeqArgs& a, int64_t at) {
  return a.q_bf16 ? bf16_to_f(((const uint16_t*)a.q)[at]) : ((const float*)a.q)[at];
}
// 8 of a row of q
__device__ inline void q8(const SeqArgs& a, int64_t at, float (&f)[8]) {
  if (a.q_bf16) {
    const uint4 w = *(const uint4*)((const uint16_t*)a.q + at);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(u[i] << 16); f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u); }
  } else {
    const float4 u = *(const float4*)((const float*)a.q + at), v = *(const float4*)((const float*)a.q + at + 4);
    f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w; f[4] = v.x; f[5] = v.y; f[6] = v.z; f[7] = v.w;
  }
}

__device__ inline float* part_of(const SeqArgs& a, int64_t row, int h, int part, int hd) {
  return a.part + (((row * a.heads + h) * a.parts) + part) * (hd + 2);
}

// Where pair p of the item leaves its part (a.parts > 1, or pages' item with a slot), hd + 2 floats
template <int FORM>
__device__ inline bool seq_parts(const SeqArgs& a, const SeqItem& it) { return FORM == SEQ_PAGED ? it.slot >= 0 : a.parts > 1; }
template <int FORM>
__device__ inline float* seq_part(const SeqArgs& a, const SeqItem& it, int p, int64_t row, int h, int hd) {
  if constexpr (FORM == SEQ_PAGED) return a.part + ((int64_t)it.slot * a.slot_pairs + (p - it.pair0)) * (hd + 2);
  else return part_of(a, row, h, it.part, hd);
}

// The wave's pairs again, one at a time over the keys k0 .. k1 - 1 that each sees and no other: a lane a key's score, then a
// lane HD / 64 dimensions of p v.
template <int HD, int CF, int FORM>
__device__ void attend_again(const SeqArgs& a, const SeqItem& it, int wpair, int k0, int k1) {
  const int lane = threadIdx.x & 63;
  for (int i = 0; i < 32 && wpair + i < it.pairs; ++i) {
    const int p = wpair + i, h = it.kvh * a.rep + p % a.rep, end = min(pair_limit(a, it, p), k1);
    const int64_t row = it.row0 + p / a.rep, qat = row * a.ldq + (int64_t)h * HD;
    float m = -INFINITY, l = 0.f, o[HD / 64];
    for (int d = 0; d < HD / 64; ++d) o[d] = 0.f;
    for (int k = k0; k < end; k += 64) {
      float sc = -INFINITY;
      if (k + lane < end) {
        const int64_t r = (int64_t)it.kvh * a.cache_len + key_row<FORM>(a, it, k + lane);
        sc = 0.f;
        for (int c = 0; c < HD; ++c) sc = fmaf(q_value(a, qat + c), cache_value<HD, CF>(a, r, c), sc);
        sc *= a.scale * 1.44269504088896341f;
      }
      const float mn = fmaxf(m, wave_max(sc));
      const float pr = k + lane < end ? exp2f(sc - (mn == -INFINITY ? 0.f : mn)) : 0.f, f = m == -INFINITY ? 0.f : exp2f(m - mn);
      l = l * f + wave_sum(pr);
      m = mn;
      for (int d = 0; d < HD / 64; ++d) o[d] *= f;
      for (int j = 0; j < min(64, end - k); ++j) {
        const float pj = __shfl(pr, j, 64);
        const int64_t r = (int64_t)(a.kv_heads + it.kvh) * a.cache_len + key_row<FORM>(a, it, k + j);
        for (int d = 0; d < HD / 64; ++d) o[d] = fmaf(pj, cache_value<HD, CF>(a, r, lane + 64 * d), o[d]);
      }
    }
    if (seq_parts<FORM>(a, it)) {
      float* pp = seq_part<FORM>(a, it, p, row, h, HD);
      for (int d = 0; d < HD / 64; ++d) pp[lane + 64 * d] = o[d];
      if (lane == 0) { pp[HD] = m; pp[HD + 1] = m == -INFINITY && end > k0 ? 1.f : l; }
    } else {
      for (int d = 0; d < HD / 64; ++d) {
        const int64_t col = (int64_t)h * HD + lane + 64 * d, at = a.o_tiles ? tile16_at(row, col, a.ldo) : row * a.ldo + col;
        const float v = end > k0 ? o[d] / l : 0.f;
        if (a.o_bf16) ((uint16_t*)a.o)[at] = (uint16_t)bf16_rne_f(v);
        else ((float*)a.o)[at] = v;
      }
    }
  }
}

// A wave's result: lane (ql, hh) holds dimensions 32 d + 8 (r / 4) + 4 hh + r % 4 of pair wpair + ql
template <int HD, int CF, int FORM>
__device__ inline void seq_finish(const SeqArgs& a, const SeqItem& it, int wpair, int limit, int k0, int k1, floatx16 (&acc)[HD / 32], float m, float l) {
  const int lane = threadIdx.x & 63, ql = lane & 31, hh = lane >> 5, p = wpair + ql;
  float big = l;  // (0 times a sum that is not finite: NaN)
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) big = fmaf(acc[d][r], 0.f, big);
  if (__any(!(fabsf(big) < INFINITY))) { attend_again<HD, CF, FORM>(a, it, wpair, k0, k1); return; }
  if (p >= it.pairs) return;
  const int64_t row = it.row0 + p / a.rep;
  const int h = it.kvh * a.rep + p % a.rep;
  if (seq_parts<FORM>(a, it)) {
    float* pp = seq_part<FORM>(a, it, p, row, h, HD);
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float2* to = (float2*)(pp + 32 * d + 8 * g + 4 * hh);  // (8-byte aligned: hd + 2 floats a part)
        to[0] = make_float2(acc[d][4 * g], acc[d][4 * g + 1]);
        to[1] = make_float2(acc[d][4 * g + 2], acc[d][4 * g + 3]);
      }
    // (a part whose keys all score -inf: no weight beside others, NaN alone; a part without keys: a sum of 0)
    if (hh == 0) *(float2*)(pp + HD) = make_float2(m, m == -INFINITY && limit > k0 ? 1.f : l);
    return;
  }
  const float inv = limit > 0 ? 1.f / l : 0.f;
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      put4(a, row, (int64_t)h * HD + 32 * d + 8 * g + 4 * hh,
           make_float4(acc[d][4 * g] * inv, acc[d][4 * g + 1] * inv, acc[d][4 * g + 2] * inv, acc[d][4 * g + 3] * inv));
}

// The softmax of a tile's NB blocks of 32 keys from key k0: scores in, weights out; the running max (base 2), the sum and
// the output's rescaling
template <int HD, int NB>
__device__ inline void seq_softmax(floatx16* s, int k0, int limit, int wave_min, int hh, float scale2, float& m, float& l, floatx16 (&acc)[HD / 32]) {
  if (k0 + 32 * NB > wave_min) {  // (some pair of the wave does not see all of the tile)
    const int left = limit - k0 - 4 * hh;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 32 * b + 8 * (r >> 2) + (r & 3) < left ? s[b][r] : -INFINITY;
  }
  float mt = -INFINITY;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[b][r]);
  mt = fmaxf(mt, __shfl_xor(mt, 32, 64)) * scale2;
  if (__any(mt > m + SQ_SLACK)) {
    const float mn = fmaxf(m, mt), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= f;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] *= f;
  }
  const float shift = m == -INFINITY ? 0.f : m;  // (no key seen so far: every weight 0)
  float sum = 0.f;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s[b][r], scale2, -shift));
      s[b][r] = p;
      sum += p;
    }
  l += sum;  // (this half's keys; the halves meet at the end)
}

// What the forms do around their tiles: the item, the pair of each lane, the tiles of its keys. A workgroup takes BQ pairs: 32 a
// wave, or with KG = 2 groups of waves half of that, each group half of a tile's keys, and the groups' results meet at the end
// (seq_meet).
#define SEQ_BEGIN(BK, KG, FORM) \
  constexpr int BQ = 32 * SQ_NW / KG, PG = SQ_NW / KG; \
  (void)PG; \
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), ql = lane & 31, hh = lane >> 5; \
  if (it.pair0 >= it.pairs) return; \
  [[maybe_unused]] const int kg = wave / PG; \
  const int wpair = it.pair0 + 32 * (wave % PG), pair = min(wpair + ql, it.pairs - 1); \
  const int limit = wpair + ql < it.pairs ? pair_limit(a, it, pair) : 0; \
  /* what the wave's pairs see at least and at most, and the tile's: a sequence's rows see more and more */ \
  int wave_min, wave_max, keys; \
  if (FORM != SEQ_SHARED || it.step >= 0) { \
    wave_min = pair_limit(a, it, wpair); wave_max = pair_limit(a, it, min(wpair + 31, it.pairs - 1)); \
    keys = pair_limit(a, it, min(it.pair0 + BQ, it.pairs) - 1); \
  } else { \
    wave_max = wave_most(limit); wave_min = -wave_most(wpair + ql < it.pairs ? -limit : -0x7FFFFFFF); \
    keys = wave_most(max(pair_limit(a, it, it.pair0 + lane), BQ > 64 ? pair_limit(a, it, it.pair0 + 64 + lane) : 0)); \
  } \
  wave_min = __builtin_amdgcn_readfirstlane(wave_min); wave_max = __builtin_amdgcn_readfirstlane(wave_max); keys = __builtin_amdgcn_readfirstlane(keys); \
  if (wpair >= it.pairs) wave_max = 0; \
  const int ntiles = (keys + BK - 1) / BK; \
  const int t0 = FORM == SEQ_PAGED ? it.t0 : (int)((int64_t)ntiles * it.split / it.splits), t1 = FORM == SEQ_PAGED ? it.t1 : (int)((int64_t)ntiles * (it.split + 1) / it.splits); \
  const int64_t qat = (it.row0 + pair / a.rep) * a.ldq + (int64_t)(it.kvh * a.rep + pair % a.rep) * HD; \
  const float scale2 = a.scale * 1.44269504088896341f; \
  const int64_t kplane = (int64_t)it.kvh * a.cache_len, vplane = (int64_t)(a.kv_heads + it.kvh) * a.cache_len; \
  floatx16 acc[HD / 32]; \
  for (int d = 0; d < HD / 32; ++d) for (int r = 0; r < 16; ++r) acc[d][r] = 0.f; \
  float m = -INFINITY, l = 0.f;

// The second key group's results into the first's, pair group by pair group, through LDS where the tiles were. False: the
// wave has given its results away. (All waves of the workgroup call it: behind the last tile's barrier.)
template <int HD>
__device__ inline bool seq_meet(float* lds, int pgroups, int kg, int wave, float& m, float& l, floatx16 (&acc)[HD / 32]) {
  const int lane = threadIdx.x & 63;
  float* slot = lds + (wave % pgroups) * (HD / 2 + 2) * 64 + lane;
  if (kg == 1) {
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) slot[(16 * d + r) * 64] = acc[d][r];
    slot[(HD / 2) * 64] = m;
    slot[(HD / 2 + 1) * 64] = l;
  }
  __syncthreads();
  if (kg != 0) return false;
  const float om = slot[(HD / 2) * 64], ol = slot[(HD / 2 + 1) * 64], top = fmaxf(m, om);
  // (a max of -inf, no key seen: no weight; both: 0)
  const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top), g = om == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(om - top);
  m = top;
  l = l * f + ol * g;
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = acc[d][r] * f + slot[(16 * d + r) * 64] * g;
  return true;
}

// x's bf16 terms: the value to nearest, then what is left to nearest
template <int N>
__device__ inline void bf16_terms(const float (&x)[8], bf16x8 (&t)[N]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float left = x[i];
#pragma unroll
    for (int j = 0; j < N; ++j) { t[j][i] = (__bf16)left; left -= (float)t[j][i]; }
  }
}

// Where a tile's values lie in LDS. A bf16 cache's rows go there straight from memory (global_load_lds_dwordx4: no registers, no
// writes of ours): rows unpadded, 1 KB a wave's instruction in lane order, the banks spread by which 16 bytes of its row each
// lane fetches: unit u of a row at unit u ^ f(row). A block float's runs are decoded on the way and written to padded rows.
template <int HD, bool ASYNC>
struct SeqTile {
  static constexpr int KLD = ASYNC ? HD : HD + 8, VLD = ASYNC ? HD : HD + 32;  // (a row's 16-byte reads, and 4 rows' transposed ones, on distinct banks)
  static constexpr int SIZE = 64 * (KLD + VLD);                                // uint16s: 64 keys' rows, then their values'
  // tiles in LDS: a third saves one of two barriers a tile, where it fits two workgroups a CU
  static constexpr int STAGES = ASYNC && HD == 64 ? 3 : 2;
  __device__ static int kswap(int row) { return !ASYNC ? 0 : HD == 128 ? row & 15 : (row >> 1) & 7; }
  __device__ static int vswap(int row) { return !ASYNC ? 0 : HD == 128 ? (row & 3) * 4 : ((row >> 1) & 1) * 4; }
};

// QT, PT: the bf16 terms of q and of the weights; KG: the groups of waves that share a tile's keys; FORM: which entry point's
template <int HD, int CF, int QT, int PT, int KG, int FORM>
__device__ __forceinline__ void seq_bf16_item(const SeqArgs& a, const SeqItem& it, uint16_t* tiles) {
  constexpr bool ASYNC = CF == FH_BF16;
  using Tile = SeqTile<HD, ASYNC>;
  constexpr int BK = 64, KLD = Tile::KLD, VLD = Tile::VLD, NS = Tile::STAGES;
  SEQ_BEGIN(BK, KG, FORM)

  // the lane's q as the product's B: step s holds dimensions 16 s + 8 hh .. + 7, each term
  bf16x8 qf[HD / 16][QT];
#pragma unroll
  for (int s = 0; s < HD / 16; ++s) {
    float f[8];
    q8(a, qat + 16 * s + 8 * hh, f);
    bf16_terms<QT>(f, qf[s]);
  }

  constexpr int NP = BK * HD / 8 / (64 * SQ_NW);  // pieces of 8 a thread
  SeqRaw kraw[ASYNC ? 1 : NP], vraw[ASYNC ? 1 : NP];
  // a thread's pieces of a tile: rows pr + PSTEP j, unit pu of each (a wave's loads into LDS in order: its rows lie together)
  constexpr int PSTEP = (ASYNC ? 64 : 64 * SQ_NW) / (HD / 8);
  const int pr = ASYNC ? (64 * NP * wave + lane) / (HD / 8) : tid / (HD / 8), pu = lane % (HD / 8);
  // (pages) a wave's rows that lie together are 16 or fewer of one page, whose number comes by the scalar unit a tile ahead: pages
  // has those of tile t on their way, load takes them as its base and leaves the next tile's
  constexpr int NPG = ASYNC ? 1 : NP;
  [[maybe_unused]] int page[NPG];
  [[maybe_unused]] const int wrow = __builtin_amdgcn_readfirstlane(pr), mask = (1 << a.page_shift) - 1;
  auto pages = [&](int t) {
    if constexpr (FORM == SEQ_PAGED)
#pragma unroll
      for (int j = 0; j < NPG; ++j) page[j] = table_page(a, it, min(t * BK + wrow + PSTEP * j, keys - 1));
  };
  auto load = [&](int t, int b) {  // tile t's loads: into buffer b, or into registers
    const int k0 = t * BK;
    if constexpr (FORM == SEQ_PAGED) {
      const bool end = k0 + BK > keys;  // (rows behind the last key: its row again)
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int first = k0 + wrow + (ASYNC ? 0 : PSTEP * j);  // the wave's first key of the page
        const int64_t base = page_row(a, page[ASYNC ? 0 : j]);
        const int r = pr + PSTEP * j;
        if (ASYNC && !end) {
          const char* kb = (const char*)a.cache + (kplane + base + (first & mask)) * (HD * 2);
          const char* vb = (const char*)a.cache + (vplane + base + (first & mask)) * (HD * 2);
          uint16_t* to = tiles + b * Tile::SIZE + 512 * (NP * wave + j);
          load_to_lds(kb, (uint32_t)((r - wrow) * HD * 2 + 16 * (pu ^ Tile::kswap(r))), to);
          load_to_lds(vb, (uint32_t)((r - wrow) * HD * 2 + 16 * (pu ^ Tile::vswap(r))), to + BK * HD);
          continue;
        }
        const int64_t row = base + (min(k0 + r, keys - 1) & mask);
        if constexpr (ASYNC) {
          uint16_t* to = tiles + b * Tile::SIZE + 512 * (NP * wave + j);
          load_to_lds((const uint16_t*)a.cache + (kplane + row) * HD + 8 * (pu ^ Tile::kswap(r)), to);
          load_to_lds((const uint16_t*)a.cache + (vplane + row) * HD + 8 * (pu ^ Tile::vswap(r)), to + BK * HD);
        } else {
          kraw[j] = seq_raw<HD, CF>(a, kplane + row, 8 * pu);
          vraw[j] = seq_raw<HD, CF>(a, vplane + row, 8 * pu);
        }
      }
      pages(t + 1);
      return;
    }
    // the tile's rows run on from its first, as they are, unless the keys end or the prefix ends in it, or it leaves the cache
    const int64_t first = (k0 < it.shared ? it.prefix : it.own) + k0;
    const bool plain = k0 + BK <= keys && (k0 >= it.shared || k0 + BK <= it.shared) && first >= 0 && first + BK <= a.cache_len;
    if (ASYNC && plain) {
      const char* kb = (const char*)a.cache + (kplane + first) * (HD * 2);
      const char* vb = (const char*)a.cache + (vplane + first) * (HD * 2);
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int r = pr + PSTEP * j;
        uint16_t* to = tiles + b * Tile::SIZE + 512 * (NP * wave + j);
        load_to_lds(kb + (uint32_t)(r * HD * 2 + 16 * (pu ^ Tile::kswap(r))), to);
        load_to_lds(vb + (uint32_t)(r * HD * 2 + 16 * (pu ^ Tile::vswap(r))), to + BK * HD);
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int r = pr + PSTEP * j;
      const int64_t row = plain ? first + r : key_row<FORM>(a, it, min(k0 + r, keys - 1));
      if constexpr (ASYNC) {
        uint16_t* to = tiles + b * Tile::SIZE + 512 * (NP * wave + j);
        load_to_lds((const uint16_t*)a.cache + (kplane + row) * HD + 8 * (pu ^ Tile::kswap(r)), to);
        load_to_lds((const uint16_t*)a.cache + (vplane + row) * HD + 8 * (pu ^ Tile::vswap(r)), to + BK * HD);
      } else {
        kraw[j] = seq_raw<HD, CF>(a, kplane + row, 8 * pu);
        vraw[j] = seq_raw<HD, CF>(a, vplane + row, 8 * pu);
      }
    }
  };
  auto store = [&](int b) {
    if constexpr (!ASYNC) {
      uint16_t* K = tiles + b * Tile::SIZE;
      uint16_t* V = K + BK * KLD;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int r = pr + PSTEP * j;
        *(uint4*)(K + r * KLD + 8 * pu) = seq_bf16x8<CF>(kraw[j]);
        *(uint4*)(V + r * VLD + 8 * pu) = seq_bf16x8<CF>(vraw[j]);
      }
    }
  };
  if (t0 < t1) pages(t0);
  // this wave's blocks of 32 keys of the tile in buffer b, whose first key is k0
  constexpr int NB = 2 / KG;
  auto work = [&](int b, int k0) {
    const int kb0 = KG == 1 ? 0 : kg;
    const uint16_t* K = tiles + b * Tile::SIZE + 32 * kb0 * KLD;
    const uint16_t* V = tiles + b * Tile::SIZE + BK * KLD + 32 * kb0 * VLD;
    floatx16 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
    if constexpr (NB == 1) {
      // one block: every read of its keys at once, and two chains of products
      bf16x8 kf[HD / 16];
#pragma unroll
      for (int st = 0; st < HD / 16; ++st) kf[st] = *(const bf16x8*)(K + ql * KLD + 8 * ((2 * st + hh) ^ Tile::kswap(ql)));
#pragma unroll
      for (int st = 0; st < HD / 16; st += 2)
#pragma unroll
        for (int u = 0; u < QT; ++u)
#pragma unroll
          for (int c = 0; c < 2; ++c) s[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[st + c], qf[st + c][u], s[c], 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[0][r] += s[1][r];
    } else {
#pragma unroll
      for (int st = 0; st < HD / 16; ++st)
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) {
          const bf16x8 kf = *(const bf16x8*)(K + (32 * kb + ql) * KLD + 8 * ((2 * st + hh) ^ Tile::kswap(ql)));
#pragma unroll
          for (int u = 0; u < QT; ++u) s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[st][u], s[kb], 0, 0, 0);
        }
    }
    seq_softmax<HD, NB>(s, k0 + 32 * kb0, limit, wave_min, hh, scale2, m, l, acc);
    // O^T += V^T P^T, 16 keys a step: the lane's weights 8 j .. 8 j + 7 of block kb are keys 32 kb + 16 j + {4 hh .. 4 hh + 3,
    // 8 + 4 hh .. 8 + 4 hh + 3}; V's columns come transposed, 4 keys of 16 dimensions to 16 lanes
    const int vr = (lane & 15) >> 2, vu = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);  // the lane's row of 4, its 16 bytes of 64
    const uint16_t* vl = V + (4 * hh + vr) * VLD + 4 * (lane & 1);
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float p8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p8[i] = s[kb][8 * j + i];
        bf16x8 pf[PT];
        bf16_terms<PT>(p8, pf);
        const int g = 32 * kb + 16 * j;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) {
          const uint16_t* vd = vl + g * VLD + 8 * ((4 * d + vu) ^ Tile::vswap(vr));
          const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SEQ_LDS short4v*)vd);
          const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SEQ_LDS short4v*)(vd + 8 * VLD));
          const short8v vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
          for (int u = 0; u < PT; ++u) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)&vf, pf[u], acc[d], 0, 0, 0);
        }
      }
  };
  auto work_on = [&](int t, int b) {
    if (t * BK + (KG == 1 ? 0 : 32 * kg) < wave_max) work(b, t * BK);
  };
  if constexpr (ASYNC) {
    // a ring of NS tiles: a tile's wait leaves the next one's loads in flight
    constexpr int W = 2 * NP;
    if (t0 < t1) load(t0, 0);
    if (t0 + 1 < t1) load(t0 + 1, 1);
    int b = 0;
    for (int t = t0; t < t1; ++t) {
      asm volatile("" ::: "memory");
      if (t + 1 < t1) __builtin_amdgcn_s_waitcnt(0x0070 | (W & 15) | (W >> 4) << 14);
      else __builtin_amdgcn_s_waitcnt(0x0070);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (NS == 3 && t + 2 < t1) load(t + 2, b == 0 ? 2 : b - 1);  // (its last readers passed this barrier)
      work_on(t, b);
      if (NS == 2 && t + 2 < t1) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xC07F);  // (this wave's reads of the buffer are done)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        load(t + 2, b);
      }
      b = b + 1 == NS ? 0 : b + 1;
    }
    __syncthreads();
  } else {
    if (t0 < t1) { load(t0, 0); store(0); }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
      const int b = (t - t0) & 1;
      if (t + 1 < t1) load(t + 1, 0);
      work_on(t, b);
      if (t + 1 < t1) store(1 - b);  // (the other buffer: its last readers passed the previous barrier)
      __syncthreads();
    }
  }
  l += __shfl_xor(l, 32, 64);
  static_assert(KG == 1 || PG * 64 * (HD / 2 + 2) * 4 <= NS * Tile::SIZE * 2, "the key groups' place");
  if constexpr (KG > 1)
    if (!seq_meet<HD>((float*)tiles, PG, kg, wave, m, l, acc)) return;
  seq_finish<HD, CF, FORM>(a, it, wpair, limit, t0 * BK, min(t1 * BK, keys), acc, m, l);
}

// A workgroup's items: its own, or over pages those of its share
template <int BQ, int BK, int FORM, typename Work>
__device__ __forceinline__ void seq_items(const SeqArgs& a, Work work) {
  SeqItem it;
  if constexpr (FORM != SEQ_PAGED) {
    if (seq_item<BQ, FORM>(a, it)) work(it);
  } else {
    const int heads = a.kv_heads * a.head_tiles, head = blockIdx.x % heads;
    const int me = a.parts > 1 ? blockIdx.x / heads : a.walkers - 1 - blockIdx.x / heads;  // (without cuts: a sequence's longest tile first)
    it.kvh = head / a.head_tiles;
    it.split = it.splits = it.part = it.shared = 0; it.prefix = it.own = 0; it.step = 1;
    __shared__ __attribute__((aligned(16))) int4 held[64 * SQ_NW];
    SeqWalk w;
    int t = 0, c0 = 0, x0 = 0, x1 = 0x7FFFFFFF;
    if (a.whole) {  // a workgroup a sequence
      const int st = a.starts[me], en = a.starts[me + 1];
      w.seq = me; w.at = 0; w.place = a.places[me];
      w.lo = clampi(st, 0, a.rows);
      w.len = clampi(en, w.lo, a.rows) - w.lo;
      w.tiles = SeqWalk::tiles_of(a, w.len);
      if (!w.tiles) return;
    } else {
      w.start(a, held);
      if ((int64_t)me * w.share >= w.total) return;
      x0 = me * w.share;
      x1 = (int)min((int64_t)x0 + w.share, (int64_t)w.total);
      w.seek_from_start(a, x0);
      t = w.tile_at(a, x0);
      c0 = w.at + SeqWalk::cost(a, w.place, t);
    }
    bool again = false;
    for (;;) {
      const int c1 = w.at + SeqWalk::cost(a, w.place, t + 1), n = w.key_tiles_of(a, t, BK);
      it.t0 = a.whole ? 0 : __builtin_amdgcn_readfirstlane(SeqWalk::cut(a, c0, c1, n, x0));
      it.t1 = a.whole ? n : __builtin_amdgcn_readfirstlane(SeqWalk::cut(a, c0, c1, n, x1));
      if (it.t0 < it.t1 || (n == 0 && x1 >= c1)) {
        if (again) __syncthreads();  // (the last item's tiles are read)
        again = true;
        const int row = t * a.tile_rows;
        it.row0 = w.lo + row;
        it.pair0 = head % a.head_tiles * BQ;
        it.pairs = a.head_tiles > 1 ? a.rep : min(a.tile_rows, w.len - row) * a.rep;
        it.place0 = w.place + row;
        it.table = a.tables + (int64_t)w.seq * a.ldt;
        it.slot = it.t0 == 0 && it.t1 == n ? -1 : (int)(blockIdx.x * 2 + (it.t0 == 0));  // (at most two of a share: its first and its last tile)
        work(it);
      }
      if (c1 >= x1) return;
      c0 = c1;
      if (++t == w.tiles) {
        if (a.whole) return;
        w.seek(a, c1);
        t = 0;
      }
    }
  }
}

template <int HD, int CF, int QT, int PT, int KG, int FORM>
__global__ __launch_bounds__(64 * SQ_NW, HD == 64 && QT < 3 ? 3 : 2) void seq_bf16_kernel(SeqArgs a) {
  using Tile = SeqTile<HD, CF == FH_BF16>;
  __shared__ __attribute__((aligned(256))) uint16_t tiles[Tile::STAGES * Tile::SIZE];
  seq_items<32 * SQ_NW / KG, 64, FORM>(a, [&](const SeqItem& it) { seq_bf16_item<HD, CF, QT, PT, KG, FORM>(a, it, tiles); });
}

// The same in fp32: 32 keys a tile. A lane's q holds dimensions HD / 2 hh .. of its half (the order of a sum's products is free),
// so that K's row is read 16 bytes at a time; P's step r multiplies keys 8 (r / 4) + 4 hh + r % 4, V's rows as they lie.
template <int HD, int FORM>
__device__ __forceinline__ void seq_f32_item(const SeqArgs& a, const SeqItem& it, float (*Ks)[32 * (HD + 4)], float (*Vs)[32 * (HD + 4)]) {
  constexpr int CF = FH_F32;
  constexpr int BK = 32, LD = HD + 4;
  SEQ_BEGIN(BK, 1, FORM)
  float qf[HD / 2];
#pragma unroll
  for (int s = 0; s < HD / 16; ++s) {
    float f[8];
    q8(a, qat + (HD / 2) * hh + 8 * s, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) qf[8 * s + i] = f[i];
  }
  constexpr int NP = BK * HD / 8 / (64 * SQ_NW);
  SeqRaw kraw[NP], vraw[NP];
  [[maybe_unused]] int page[NP];
  auto pages = [&](int t) {  // (pages) as above
    if constexpr (FORM == SEQ_PAGED)
#pragma unroll
      for (int j = 0; j < NP; ++j) page[j] = table_page(a, it, min(t * BK + (tid + 64 * SQ_NW * j) / (HD / 8), keys - 1));
  };
  auto load = [&](int t) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int i = tid + 64 * SQ_NW * j, r = i / (HD / 8), c = (i % (HD / 8)) * 8, k = min(t * BK + r, keys - 1);
      const int64_t row = FORM == SEQ_PAGED ? page_row(a, page[j]) + (k & ((1 << a.page_shift) - 1)) : key_row<FORM>(a, it, k);
      kraw[j] = seq_raw<HD, CF>(a, kplane + row, c);
      vraw[j] = seq_raw<HD, CF>(a, vplane + row, c);
    }
    pages(t + 1);
  };
  if (t0 < t1) pages(t0);
  auto store = [&](int b) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int i = tid + 64 * SQ_NW * j, r = i / (HD / 8), c = (i % (HD / 8)) * 8;
      float4* k = (float4*)(Ks[b] + r * LD + c);
      float4* v = (float4*)(Vs[b] + r * LD + c);
      seq_f32x8(kraw[j], k[0], k[1]);
      seq_f32x8(vraw[j], v[0], v[1]);
    }
  };
  if (t0 < t1) { load(t0); store(0); }
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const int b = (t - t0) & 1, k0 = t * BK;
    if (t + 1 < t1) load(t + 1);
    if (k0 < wave_max) {
      floatx16 s[1];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
      const float* kr = Ks[b] + ql * LD + (HD / 2) * hh;
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) {
        const float4 kf = *(const float4*)(kr + 4 * c);
        s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf.x, qf[4 * c], s[0], 0, 0, 0);
        s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf.y, qf[4 * c + 1], s[0], 0, 0, 0);
        s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf.z, qf[4 * c + 2], s[0], 0, 0, 0);
        s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf.w, qf[4 * c + 3], s[0], 0, 0, 0);
      }
      seq_softmax<HD, 1>(s, k0, limit, wave_min, hh, scale2, m, l, acc);
      const float* vr = Vs[b] + 4 * hh * LD + ql;
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vr[(8 * (r >> 2) + (r & 3)) * LD + 32 * d], s[0][r], acc[d], 0, 0, 0);
    }
    if (t + 1 < t1) store(1 - b);
    __syncthreads();
  }
  l += __shfl_xor(l, 32, 64);
  seq_finish<HD, CF, FORM>(a, it, wpair, limit, t0 * BK, min(t1 * BK, keys), acc, m, l);
}

template <int HD, int FORM>
__global__ __launch_bounds__(64 * SQ_NW, 2) void seq_f32_kernel(SeqArgs a) {
  __shared__ __attribute__((aligned(16))) float Ks[2][32 * (HD + 4)];
  __shared__ __attribute__((aligned(16))) float Vs[2][32 * (HD + 4)];
  seq_items<32 * SQ_NW, 32, FORM>(a, [&](const SeqItem& it) { seq_f32_item<HD, FORM>(a, it, Ks, Vs); });
}

// A pair's parts joined, a wave a pair: lane p holds part p's statistics, then a lane HD / 64 dimensions of each part's sum,
// times 2^(its max - the largest). A part that saw no key (its max -inf) has no weight; a pair with none gives zeros. Parts
// of rows that are no sequence's were never written and are not read. 2048 pairs of 9 parts: 5 us; with the parts stored as
// the products leave them in registers, whole lines a store, and joined 8 dimensions of 32 pairs a wave, 7 to 10: fewer waves,
// each with a longer chain.
template <int HD>
__global__ __launch_bounds__(256) void seq_join(SeqArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= a.rows * a.heads) return;
  const int64_t row = i / a.heads;
  const int h = (int)(i % a.heads);
  if (a.starts && (row < a.starts[0] || row >= a.starts[a.n])) return;
  const float* pp = part_of(a, row, h, 0, HD);
  const bool in = lane < a.parts;
  const float2 st = in ? *(const float2*)(pp + (int64_t)lane * (HD + 2) + HD) : make_float2(-INFINITY, 0.f);
  float o[HD / 64];
  const float top = wave_max(st.x);
  // (a max that is NaN or +inf makes the sum NaN, as one softmax over all keys would)
  const bool none = st.y == 0.f && st.x == -INFINITY;
  const float w = none ? 0.f : __builtin_amdgcn_exp2f(st.x - top);
  const float den = wave_sum(none ? 0.f : w * st.y);
#pragma unroll
  for (int d = 0; d < HD / 64; ++d) o[d] = 0.f;
  const uint64_t some = __ballot(!none && in);
  for (int p0 = 0; p0 < a.parts; p0 += 8) {
    float v[8][HD / 64];
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int d = 0; d < HD / 64; ++d) v[u][d] = pp[(int64_t)min(p0 + u, a.parts - 1) * (HD + 2) + lane * (HD / 64) + d];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float wp = __shfl(w, (p0 + u) & 63, 64);
      if (p0 + u < a.parts && (some >> (p0 + u) & 1))
#pragma unroll
        for (int d = 0; d < HD / 64; ++d) o[d] = fmaf(wp, v[u][d], o[d]);
    }
  }
  const int64_t col = (int64_t)h * HD + lane * (HD / 64), at = a.o_tiles ? tile16_at(row, col, a.ldo) : row * a.ldo + col;
  const float inv = some ? 1.f / den : 0.f;
#pragma unroll
  for (int d = 0; d < HD / 64; ++d) {
    if (a.o_bf16) ((uint16_t*)a.o)[at + d] = (uint16_t)bf16_rne_f(o[d] * inv);
    else ((float*)a.o)[at + d] = o[d] * inv;
  }
}

// The parts of a tile that shares cut, joined as above: a workgroup a cut, which takes the tile whose first cut it is. TOKENS: few
// pairs of many parts, a wave a pair; otherwise HD / 4 lanes a pair, 4 parts on their way at a time.
template <int HD, int BK, bool TOKENS>
__global__ __launch_bounds__(TOKENS || HD == 64 ? 512 : 1024) void seq_join_pages(SeqArgs a) {
  constexpr int NT = TOKENS || HD == 64 ? 512 : 1024;
  __shared__ __attribute__((aligned(16))) int4 held[NT];
  const int heads = a.kv_heads * a.head_tiles, head = blockIdx.x % heads, first = blockIdx.x / heads;  // the share before the cut
  SeqWalk w;
  w.start(a, held);
  if ((int64_t)(first + 1) * w.share >= w.total) return;
  const int x = (first + 1) * w.share;
  w.seek_from_start(a, x);
  const int t = w.tile_at(a, x), n = w.key_tiles_of(a, t, BK);
  const int c0 = w.at + SeqWalk::cost(a, w.place, t), c1 = w.at + SeqWalk::cost(a, w.place, t + 1);
  auto cut = [&](int i) { return SeqWalk::cut(a, c0, c1, n, (int)min((int64_t)i * w.share, (int64_t)w.total)); };  // where share i begins
  const int k = cut(first + 1);
  if (k <= 0 || k >= n || cut(first) > 0) return;
  // the parts: of share `first`, from the tile's first key on, and of those behind it up to the one that ends it
  int last = first + 1;
  while (last + 1 < a.walkers && cut(last + 1) < n) ++last;
  const int parts = last - first + 1, lane = threadIdx.x & 63, row = t * a.tile_rows;
  const int pair0 = head % a.head_tiles * a.slot_pairs, pairs = min(a.slot_pairs, (a.head_tiles > 1 ? a.rep : min(a.tile_rows, w.len - row) * a.rep) - pair0);
  auto part = [&](int i, int p) { return a.part + ((int64_t)(((first + i) * heads + head) * 2 + (i == 0)) * a.slot_pairs + p) * (HD + 2); };
  auto some_of = [&](int i) { return cut(first + i) < cut(first + i + 1); };  // (a share may get no key of the tile)
  auto put_at = [&](int p, int d) {
    return (int64_t)(w.lo + row + (pair0 + p) / a.rep) * a.ldo + (int64_t)(head / a.head_tiles * a.rep + (pair0 + p) % a.rep) * HD + d;
  };
  constexpr int D = TOKENS ? HD / 64 : 4, L = HD / D;  // a lane's dimensions, a pair's lanes
  for (int p = threadIdx.x / L; p < pairs; p += NT / L) {
    float top = -INFINITY, den = 0.f, o[D];
    bool any = false;
#pragma unroll
    for (int d = 0; d < D; ++d) o[d] = 0.f;
    const int d0 = threadIdx.x % L * D;
    if constexpr (TOKENS) {
      for (int i0 = 0; i0 < parts; i0 += 64) {
        const bool in = i0 + lane < parts && some_of(i0 + lane);
        float v[8][D];
        auto load = [&](int i) {
#pragma unroll
          for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int d = 0; d < D; ++d) v[u][d] = part(min(i0 + i + u, parts - 1), p)[d0 + d];
        };
        load(0);  // (on their way with the statistics)
        const float2 st = in ? *(const float2*)(part(i0 + lane, p) + HD) : make_float2(-INFINITY, 0.f);
        const float now = fmaxf(top, wave_max(st.x));
        const bool none = st.y == 0.f && st.x == -INFINITY;
        const float f = any ? __builtin_amdgcn_exp2f(top - now) : 0.f;
        const float wt = none ? 0.f : __builtin_amdgcn_exp2f(st.x - now);
        den = (any ? den * f : 0.f) + wave_sum(none ? 0.f : wt * st.y);
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] = any ? o[d] * f : 0.f;
        const uint64_t some = __ballot(!none && in);
        for (int i = 0; i < min(64, parts - i0); i += 8) {
          if (i) load(i);
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const float wp = __shfl(wt, (i + u) & 63, 64);
            if (some >> ((i + u) & 63) & 1)
#pragma unroll
              for (int d = 0; d < D; ++d) o[d] = fmaf(wp, v[u][d], o[d]);
          }
        }
        any = any || some;
        top = now;
      }
    } else {
      for (int i0 = 0; i0 < parts; i0 += 4) {
        float2 st[4], v[4][2];
        bool some[4];
        float now = top;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float* pp = part(min(i0 + u, parts - 1), p);
          st[u] = *(const float2*)(pp + HD);
          v[u][0] = *(const float2*)(pp + d0); v[u][1] = *(const float2*)(pp + d0 + 2);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          some[u] = i0 + u < parts && some_of(i0 + u) && !(st[u].y == 0.f && st[u].x == -INFINITY);
          if (some[u]) now = fmaxf(now, st[u].x);
        }
        if (any) {
          const float f = __builtin_amdgcn_exp2f(top - now);
          den *= f;
#pragma unroll
          for (int d = 0; d < 4; ++d) o[d] *= f;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (some[u]) {
            const float wt = __builtin_amdgcn_exp2f(st[u].x - now);
            den = fmaf(wt, st[u].y, den);
            o[0] = fmaf(wt, v[u][0].x, o[0]); o[1] = fmaf(wt, v[u][0].y, o[1]); o[2] = fmaf(wt, v[u][1].x, o[2]); o[3] = fmaf(wt, v[u][1].y, o[3]);
            any = true;
          }
        top = now;
      }
    }
    const float inv = any ? 1.f / den : 0.f;
    const int64_t at = put_at(p, d0);
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (a.o_bf16) ((uint16_t*)a.o)[at + d] = (uint16_t)bf16_rne_f(o[d] * inv);
      else ((float*)a.o)[at + d] = o[d] * inv;
    }
  }
}

template <int HD, int CF, int KG, int FORM>
static void launch_seq(unsigned blocks, hipStream_t s, const SeqArgs& a) {
  const dim3 g(blocks), b(64 * SQ_NW);
  if constexpr (CF == FH_F32) hipLaunchKernelGGL((seq_f32_kernel<HD, FORM>), g, b, 0, s, a);
  else if (a.o_bf16) {
    if (a.q_bf16) hipLaunchKernelGGL((seq_bf16_kernel<HD, CF, 1, 2, KG, FORM>), g, b, 0, s, a);
    else hipLaunchKernelGGL((seq_bf16_kernel<HD, CF, 2, 2, KG, FORM>), g, b, 0, s, a);
  } else {
    if (a.q_bf16) hipLaunchKernelGGL((seq_bf16_kernel<HD, CF, 1, 3, KG, FORM>), g, b, 0, s, a);
    else hipLaunchKernelGGL((seq_bf16_kernel<HD, CF, 3, 3, KG, FORM>), g, b, 0, s, a);
  }
}

template <int HD, int CF, bool PAGES>
static void launch_seq(int pairs, unsigned blocks, hipStream_t s, const SeqArgs& a) {
  constexpr int ROWS = PAGES ? SEQ_PAGED : SEQ_PACKED;
  if constexpr (!PAGES)
    if (!a.starts) { launch_seq<HD, CF, 2, SEQ_SHARED>(blocks, s, a); return; }
  if (pairs == 64) launch_seq<HD, CF, 2, ROWS>(blocks, s, a);
  else launch_seq<HD, CF, 1, ROWS>(blocks, s, a);
}

template <int HD, bool PAGES>
static void launch_seq(int cf, int pairs, unsigned blocks, hipStream_t s, const SeqArgs& a) {
  switch (cf) {
    case FH_F32: launch_seq<HD, FH_F32, PAGES>(pairs, blocks, s, a); break;
    case FH_BF16: launch_seq<HD, FH_BF16, PAGES>(pairs, blocks, s, a); break;
    case FH_BFP8: launch_seq<HD, FH_BFP8, PAGES>(pairs, blocks, s, a); break;
    default: launch_seq<HD, FH_BFP4, PAGES>(pairs, blocks, s, a); break;
  }
  if constexpr (PAGES) {
    const dim3 g((unsigned)((a.walkers - 1) * a.kv_heads * a.head_tiles));
    const bool tokens = pairs == 64;
    if (a.parts > 1) {
      if (cf == FH_F32) hipLaunchKernelGGL((seq_join_pages<HD, 32, false>), g, dim3(HD == 64 ? 512 : 1024), 0, s, a);
      else if (tokens) hipLaunchKernelGGL((seq_join_pages<HD, 64, true>), g, dim3(512), 0, s, a);
      else hipLaunchKernelGGL((seq_join_pages<HD, 64, false>), g, dim3(HD == 64 ? 512 : 1024), 0, s, a);
    }
  } else if (a.parts > 1) hipLaunchKernelGGL(seq_join<HD>, dim3((unsigned)((a.rows * a.heads + 3) / 4)), dim3(256), 0, s, a);
}

template <bool PAGES>
static int launch_seq(const char* fn, int head_dim, int cf, int pairs, int64_t blocks, hipStream_t s, const SeqArgs& a) {
  if (blocks >= (1LL << 31) || (a.rows * a.heads + 3) / 4 >= (1LL << 31)) { set_error("%s: too many rows for one grid", fn); return FH_EUNSUP; }
  if (head_dim == 128) launch_seq<128, PAGES>(cf, pairs, (unsigned)blocks, s, a);
  else launch_seq<64, PAGES>(cf, pairs, (unsigned)blocks, s, a);
  return check_launch(fn);
}

// Workgroups the keys of each of `groups` tiles are split among, at most 32 (a wave joins the parts, a lane each): the number
// that takes the least time by what was measured. A workgroup alone on its CU takes a tile of 64 keys in about 1.2 us at 128
// dimensions (8 times that in fp32; one figure for every other cache, number of terms and tile of pairs), two a CU take them together in twice the time, so that more than one a CU gains nothing. It
// weighs splits against each other and is no forecast: a call's start, its end and its second launch are not in it (16 rows
// behind 4096: 7 us by the sum, 18 measured). A second kernel costs 3 us, and each part of a pair is written and read at 4 TB/s (512 rows of 32 heads: 4 us a part). `others`:
// workgroups beside them (a decode step's rows' own keys), of other_tiles each: free until the CUs are one each.
//
// A workspace holds the parts of any call of no more rows, keys and heads (callers take one for their largest), so its size is a
// bound that grows with each of them: a part a split for the pairs there are, up to the most that any sizes choose (below 3 parts
// of 128 pairs a CU for packed prompts, 4 for a decode step, whose own keys are a part more); at most `most` splits keep to it.
constexpr int SQ_CUS = 256, SQ_MAX_SPLITS = 32;
constexpr int64_t SQ_PACKED_PARTS = 3 * 128 * SQ_CUS, SQ_SHARED_PARTS = 4 * 128 * SQ_CUS;
static int64_t key_tiles(int64_t keys) { return std::max<int64_t>(1, (std::min<int64_t>(keys, 1LL << 40) + 63) / 64); }
static int most_splits(int64_t keys) { return (int)std::min<int64_t>(SQ_MAX_SPLITS, key_tiles(keys)); }
static int splits_for(int64_t groups, int64_t keys, int64_t pairs, int head_dim, int cf, double joined, int64_t most, int64_t others = 0, int64_t other_tiles = 0) {
  const double tile = 1.2 * head_dim / 128 * (cf == FH_F32 ? 8 : 1), part = 8e-6 / 4 * pairs * (head_dim + 2);
  const int64_t tiles = key_tiles(keys);
  int best = 1;
  double least = 0;
  for (int s = 1; s <= std::min<int64_t>(most_splits(keys), std::max<int64_t>(1, most)); ++s) {
    const double own = groups * s + others > SQ_CUS ? std::max(1.0, (double)others / SQ_CUS) * other_tiles : 0;
    const double t = tile * (((tiles + s - 1) / s) * std::max(1.0, (double)groups * s / SQ_CUS) + own) + part * s + (s > 1 ? joined : 0);
    if (s == 1 || t < least) { least = t; best = s; }
  }
  return best;
}
// Pairs a workgroup: 128, or 64 with two groups of waves on a tile's keys: for a decode step (one row a sequence) and prompts of
// few rows. An fp32 cache's form has no second group.
static int packed_pairs(int64_t rows, int n, int rep, int cf) { return cf != FH_F32 && rows * rep <= (int64_t)64 * n ? 64 : 128; }
static int64_t packed_tiles(int64_t rows, int n, int rep, int pairs) { return rows * rep / pairs + std::min<int64_t>(n, rows); }
static int packed_splits(int64_t rows, int n, int heads, int kv_heads, int head_dim, int cf, int64_t max_context) {
  return splits_for(packed_tiles(rows, n, heads / kv_heads, 128) * kv_heads, max_context, rows * heads, head_dim, cf, 3, SQ_PACKED_PARTS / (rows * heads));
}
static int shared_pairs(int cf) { return cf == FH_F32 ? 128 : 64; }
static void shared_splits(int batch, int heads, int kv_heads, int head_dim, int cf, int64_t max_prefix, int64_t max_own, int& tiles, int& prefix, int& own) {
  const int pairs = shared_pairs(cf);
  tiles = (int)(((int64_t)batch * (heads / kv_heads) + pairs - 1) / pairs);
  const int64_t rows = (int64_t)batch * heads, most = SQ_SHARED_PARTS / rows, groups = (int64_t)tiles * kv_heads, mine = (int64_t)batch * kv_heads;
  // (a row's own keys taken to be half of max_own, on the mean)
  const int64_t other = (std::min<int64_t>(max_own, 1LL << 40) + 127) / 128;
  const double prefix_work = (double)groups * key_tiles(max_prefix), own_work = (double)mine * std::max<int64_t>(1, other);
  // A row's own keys have half of the GPU beside the prefix, and where that leaves a chain of 8 tiles or more too many, the CUs
  // that their share of all the tiles is worth: 16 rows of 32 heads of 128 after 200 places with 4096 of their own 87 -> 52 us,
  // after 4096 with as many 89 -> 57, after 2048 with 2000 of at most 4096 51 -> 37, with 300 of them 18.1 -> 20.2. For shorter
  // chains that share costs more than it gives (4 rows after 180 with 40 of at most 512 10.2 -> 12.6).
  own = splits_for(mine * 2, max_own, rows, head_dim, cf, 0, most - 1);
  const int more = splits_for((int64_t)std::min(mine * (1 + prefix_work / own_work), 1e9), max_own, rows, head_dim, cf, 0, most - 1);
  if (key_tiles(max_own) / own - key_tiles(max_own) / more >= 8) own = more;
  prefix = splits_for(groups, max_prefix, rows, head_dim, cf, 0, most - own, mine, other);
}

static size_t parts_bytes(int64_t parts, int head_dim) { return (size_t)parts * (head_dim + 2) * sizeof(float); }

// what both entry points ask of their operands (fn: the name in the message)
static int seq_check(const char* fn, const SeqArgs& a, int q_dtype, int cache_dtype, int head_dim, int o_dtype) {
  auto no = [&](int code, const char* what) { set_error("%s: %s", fn, what); return code; };
  if (!a.q || !a.cache || !a.o || !a.places || (!a.first_row && !a.tables)) return no(FH_EINVAL, "null pointer");
  if (a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads) return no(FH_EINVAL, "heads must be a multiple of kv_heads");
  if (a.heads > 65535) return no(FH_EUNSUP, "at most 65535 heads");
  if (head_dim != 64 && head_dim != 128) return no(FH_EUNSUP, "head_dim 64 or 128");
  if (q_dtype != FH_F32 && q_dtype != FH_BF16) return no(FH_EINVAL, "q is FH_F32 or FH_BF16");
  if (cache_dtype < FH_F32 || cache_dtype > FH_BFP4) return no(FH_EUNSUP, "cache is FH_F32, FH_BF16, FH_BFP8 or FH_BFP4");
  if (a.cache_len < 1) return no(FH_EINVAL, "cache_len at least 1");
  if (a.rows * (a.heads / a.kv_heads) >= (1LL << 30) || a.cache_len >= (1LL << 30)) return no(FH_EUNSUP, "fewer than 2^30 cache rows and pairs of a row and a key head's heads");
  if ((a.shared == nullptr) != (a.prefix_row == nullptr)) return no(FH_EINVAL, "prefix_row and shared go together");
  const int64_t cols = (int64_t)a.heads * head_dim;
  if (a.ldq < cols || a.ldo < cols || a.ldq % (q_dtype == FH_F32 ? 4 : 8) || (o_dtype != FH_BF16_T16 && a.ldo % 4) ||
      ((uintptr_t)a.q & 15) || ((uintptr_t)a.cache & 15) || ((uintptr_t)a.o & (o_dtype == FH_F32 ? 15 : 7)))
    return no(FH_EINVAL, "rows at least heads * head_dim, q's and the cache's 16-byte aligned, o's 4 values");
  return FH_OK;
}

}  // namespace fh
