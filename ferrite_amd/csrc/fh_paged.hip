// Attention of ragged rows over a KV cache in pages: prompts, chunks of them and single tokens in one call. A sequence's place p
// lies at row table[p / page] page + p % page of the cache, and a query at place p sees places 0 .. p:
// o = sum_k softmax_k(q k / sqrt(hd)) v. Tiles of (row, head of a key head) pairs against tiles of keys with an online softmax, as
// packed prompts have them (fh_seq.h); what is its own is the pages' reads, how the work is shared (SeqWalk) and token_kernel.
// What bounds it (MI355X; 32 heads of 128, 8 key heads, bf16 cache; whole calls in a replayed graph, and the kernels under a trace, which takes up to
// a tenth longer): a decode step the reads, 48 tokens after up to 8000 places 169 us (890 MB: 5.25 TB/s, a plain read's rate; traced 164 and 6 the join
// of the shares' parts); with fewer keys the chain of a table's page, its rows and the two products: 16 after up to 2000 22.4 us (traced 18 and 5;
// 53 MB, 10 at that rate), 4 short ones in one launch 7.8. Prompts the products: 24 of up to 512 rows or single tokens after up to 4000
// places 206-209 us (traced 201, 95 GF of pairs, 180 with the weights' second term and the unseen pairs of a tile: 895 TFLOP/s; and 20 the join, 58 MB of
// parts). A bfp8 cache's runs are decoded by every workgroup that reads them: 11 of up to 250, 20 heads of 64, 42 us (traced 30 and 15).
//
// For bf16 output an fp32 q and the weights go in as two bf16 terms, as in the packed attention: in that bfp8 case 3.6e-6 off in the mean before the output's
// own rounding of 1.6e-3, so that one value in 280 takes the other neighbour of the exact one (an fp32 computation: one in 1900; q in
// three terms: one in 510).
#include "fh_seq.h"

namespace fh {

typedef __attribute__((__vector_size__(4 * sizeof(float)))) float floatx4;

// Few pairs a tile (a decode step's one row a sequence: the heads of a key head), at most 16, over a bf16 cache: what such a call waits
// for is memory, and behind it a tile's chain of products. Each of the 4 waves takes every fourth block of 32 keys from a ring of
// its own in LDS, so that nothing waits for another wave until the end, where their sums meet. On v_mfma_f32_16x16x32_bf16, the
// pairs 16 across: S^T = K Q^T for 2 x 16 keys, a lane 4 of each for its pair; P^T is the next product's operand as it lies, its 32
// keys in the order 4 g + 0 .. 3, 16 + 4 g + 0 .. 3 of lane group g; O^T += V^T P^T.
template <int HD>
struct TokenRing {
  static constexpr int KEYS = 32, STAGES = 2;
  static constexpr int SIZE = 2 * KEYS * HD;                      // uint16s a stage: keys, then values
  static constexpr int WAVE = STAGES * SIZE;                      // a wave's
  static constexpr int LOADS = KEYS * HD * 2 / 1024;              // instructions of 1 KB for the keys, as many for the values
  // the 16 bytes u of a row lie at u ^ swap: 16 rows' reads of one unit, and 16 rows' transposed reads of two, on distinct banks
  __device__ static int kswap(int row) { return HD == 128 ? row & 15 : (row >> 1) & 7; }
  __device__ static int vswap(int row) { return HD == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3); }
};

template <int HD, int QT, int PT>
__device__ __forceinline__ void token_item(const SeqArgs& a, const SeqItem& it, uint16_t* lds) {
  using Ring = TokenRing<HD>;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
  const int pair = min(r, it.pairs - 1), limit = r < it.pairs ? pair_limit(a, it, pair) : 0;
  const int least = __builtin_amdgcn_readfirstlane(pair_limit(a, it, 0)), keys = __builtin_amdgcn_readfirstlane(pair_limit(a, it, it.pairs - 1));
  const int b0 = 2 * it.t0, b1 = min(2 * it.t1, (keys + 31) / 32);  // blocks of 32 keys
  const float scale2 = a.scale * 1.44269504088896341f;
  const int64_t kplane = (int64_t)it.kvh * a.cache_len, vplane = (int64_t)(a.kv_heads + it.kvh) * a.cache_len;
  const int mask = (1 << a.page_shift) - 1;
  uint16_t* ring = lds + wave * Ring::WAVE;
  constexpr int ROWS = 1024 / (HD * 2), HALF = 16 / ROWS;  // rows an instruction; instructions 16 rows
  const int lrow = lane / (HD / 8), lu = lane % (HD / 8);
  // the pages of a block's halves, a block ahead
  int page[2];
  auto pages = [&](int b) {
#pragma unroll
    for (int h = 0; h < 2; ++h) page[h] = table_page(a, it, min(32 * b + 16 * h, keys - 1));
  };
  auto load = [&](int b, int stage) {
    uint16_t* to = ring + stage * Ring::SIZE;
    const bool end = 32 * b + 32 > keys;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int first = 32 * b + 16 * h;
      const int64_t base = page_row(a, page[h]);
#pragma unroll
      for (int j = 0; j < HALF; ++j) {
        const int row = ROWS * j + lrow;  // of the half's 16
        uint16_t* k = to + 512 * (HALF * h + j);
        if (!end) {
          const char* kb = (const char*)a.cache + (kplane + base + (first & mask)) * (HD * 2);
          const char* vb = (const char*)a.cache + (vplane + base + (first & mask)) * (HD * 2);
          load_to_lds(kb, (uint32_t)(row * HD * 2 + 16 * (lu ^ Ring::kswap(row))), k);
          load_to_lds(vb, (uint32_t)(row * HD * 2 + 16 * (lu ^ Ring::vswap(row))), k + Ring::KEYS * HD);
        } else {  // (behind the last key: its row again)
          const int64_t at = base + (min(first + row, keys - 1) & mask);
          load_to_lds((const uint16_t*)a.cache + (kplane + at) * HD + 8 * (lu ^ Ring::kswap(row)), k);
          load_to_lds((const uint16_t*)a.cache + (vplane + at) * HD + 8 * (lu ^ Ring::vswap(row)), k + Ring::KEYS * HD);
        }
      }
    }
    pages(b + SQ_NW);
  };
  const int first = b0 + wave;
  if (first < b1) pages(first);
  if (first < b1) load(first, 0);
  // q as the product's second operand: step s holds dimensions 32 s + 8 g .. + 7, each term
  bf16x8 qf[HD / 32][QT];
  const int64_t qat = (it.row0 + pair / a.rep) * a.ldq + (int64_t)(it.kvh * a.rep + pair % a.rep) * HD;
#pragma unroll
  for (int s = 0; s < HD / 32; ++s) {
    float f[8];
    q8(a, qat + 32 * s + 8 * g, f);
    bf16_terms<QT>(f, qf[s]);
  }
  floatx4 acc[HD / 16];
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) acc[d] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  if (first + SQ_NW < b1) load(first + SQ_NW, 1);
  int stage = 0;
  for (int b = first; b < b1; b += SQ_NW, stage ^= 1) {
    constexpr int W = 2 * Ring::LOADS;
    asm volatile("" ::: "memory");
    if (b + SQ_NW < b1) __builtin_amdgcn_s_waitcnt(0x0F70 | (W & 15) | (W >> 4) << 14);  // (the next block's loads may be on their way)
    else __builtin_amdgcn_s_waitcnt(0x0F70);
    asm volatile("" ::: "memory");
    const uint16_t* K = ring + stage * Ring::SIZE;
    const uint16_t* V = K + Ring::KEYS * HD;
    floatx4 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      s[kb] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < HD / 32; ++st) {
        const bf16x8 kf = *(const bf16x8*)(K + (16 * kb + r) * HD + 8 * ((4 * st + g) ^ Ring::kswap(r)));
#pragma unroll
        for (int u = 0; u < QT; ++u) s[kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[st][u], s[kb], 0, 0, 0);
      }
    }
    if (32 * b + 32 > least) {  // (some pair does not see all of the block)
      const int left = limit - 32 * b - 4 * g;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[kb][e] = 16 * kb + e < left ? s[kb][e] : -INFINITY;
    }
    float mt = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e) mt = fmaxf(mt, s[kb][e]);
    mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
    mt = fmaxf(mt, __shfl_xor(mt, 32, 64)) * scale2;
    if (__any(mt > m + SQ_SLACK)) {
      const float mn = fmaxf(m, mt), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) acc[d] *= f;
    }
    const float shift = m == -INFINITY ? 0.f : m;  // (no key seen so far: every weight 0)
    float p8[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p8[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], scale2, -shift));
      l += p8[i];
    }
    bf16x8 pf[PT];
    bf16_terms<PT>(p8, pf);
    // V's columns come transposed, 4 keys of 16 dimensions to 16 lanes: lane group g's keys 4 g .. and 16 + 4 g ..
    const int vrow = 4 * g + (r >> 2), vu = (r & 3) >> 1;
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) {
      const uint16_t* v = V + vrow * HD + 8 * ((2 * d + vu) ^ Ring::vswap(vrow)) + 4 * (r & 1);
      const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SEQ_LDS short4v*)v);
      const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SEQ_LDS short4v*)(v + 16 * HD));
      const short8v vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int u = 0; u < PT; ++u) acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8*)&vf, pf[u], acc[d], 0, 0, 0);
    }
    if (b + 2 * SQ_NW < b1) {
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xC07F);  // (this wave's reads of the stage are done)
      asm volatile("" ::: "memory");
      load(b + 2 * SQ_NW, stage);
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  // the waves' sums meet where the rings were: a wave every fourth 16 dimensions
  __syncthreads();
  float4* sums = (float4*)lds;                                     // [4][HD / 16][64]
  float2* stats = (float2*)(lds + SQ_NW * (HD / 16) * 64 * 8);     // [4][16]
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) sums[(wave * (HD / 16) + d) * 64 + lane] = make_float4(acc[d][0], acc[d][1], acc[d][2], acc[d][3]);
  if (g == 0) stats[wave * 16 + r] = make_float2(m, l);
  __syncthreads();
  float2 st[SQ_NW];
  float top = -INFINITY, den = 0.f, w[SQ_NW];
#pragma unroll
  for (int i = 0; i < SQ_NW; ++i) { st[i] = stats[i * 16 + r]; top = fmaxf(top, st[i].x); }
#pragma unroll
  for (int i = 0; i < SQ_NW; ++i) {
    w[i] = st[i].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st[i].x - top);  // (no key of the wave's seen: no weight)
    den = fmaf(w[i], st[i].y, den);
  }
  float4 o[HD / 64];
  float big = den;  // (0 times a sum that is not finite: NaN)
#pragma unroll
  for (int j = 0; j < HD / 64; ++j) {
    o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < SQ_NW; ++i) {
      const float4 v = sums[(i * (HD / 16) + wave + SQ_NW * j) * 64 + lane];
      o[j].x = fmaf(w[i], v.x, o[j].x); o[j].y = fmaf(w[i], v.y, o[j].y); o[j].z = fmaf(w[i], v.z, o[j].z); o[j].w = fmaf(w[i], v.w, o[j].w);
    }
    big = fmaf(o[j].x, 0.f, big); big = fmaf(o[j].y, 0.f, big); big = fmaf(o[j].z, 0.f, big); big = fmaf(o[j].w, 0.f, big);
  }
  const int k0 = 64 * it.t0, k1 = min(64 * it.t1, keys);
  // a key that a pair does not see has the weight 0, but 0 times an infinite or NaN value is NaN: the pairs again, one at a time
  if (__syncthreads_or(!(fabsf(big) < INFINITY))) {
    if (wave == 0) attend_again<HD, FH_BF16, SEQ_PAGED>(a, it, it.pair0, k0, k1);
    return;
  }
  if (r >= it.pairs) return;
  const int64_t row = it.row0 + r / a.rep;
  const int h = it.kvh * a.rep + r % a.rep;
  if (it.slot >= 0) {
    float* pp = seq_part<SEQ_PAGED>(a, it, r, row, h, HD);
#pragma unroll
    for (int j = 0; j < HD / 64; ++j) {
      float2* to = (float2*)(pp + 16 * (wave + SQ_NW * j) + 4 * g);
      to[0] = make_float2(o[j].x, o[j].y);
      to[1] = make_float2(o[j].z, o[j].w);
    }
    // (a part whose keys all score -inf: no weight beside others, NaN alone; a part without keys: a sum of 0)
    if (wave == 0 && g == 0) *(float2*)(pp + HD) = make_float2(top, top == -INFINITY && limit > k0 ? 1.f : den);
    return;
  }
  const float inv = limit > 0 ? 1.f / den : 0.f;
#pragma unroll
  for (int j = 0; j < HD / 64; ++j)
    put4(a, row, (int64_t)h * HD + 16 * (wave + SQ_NW * j) + 4 * g, make_float4(o[j].x * inv, o[j].y * inv, o[j].z * inv, o[j].w * inv));
}

template <int HD, int QT, int PT>
__global__ __launch_bounds__(64 * SQ_NW, HD == 64 ? 2 : 1) void token_kernel(SeqArgs a) {
  __shared__ __attribute__((aligned(256))) uint16_t lds[SQ_NW * TokenRing<HD>::WAVE];
  static_assert(SQ_NW * (HD / 16) * 64 * 16 + SQ_NW * 16 * 8 <= (int)sizeof(lds), "the sums' place");
  seq_items<16, 64, SEQ_PAGED>(a, [&](const SeqItem& it) { token_item<HD, QT, PT>(a, it, lds); });
}

template <int HD>
static void launch_tokens(unsigned blocks, hipStream_t s, const SeqArgs& a) {
  const dim3 g(blocks), b(64 * SQ_NW);
  if (a.o_bf16) {
    if (a.q_bf16) hipLaunchKernelGGL((token_kernel<HD, 1, 2>), g, b, 0, s, a);
    else hipLaunchKernelGGL((token_kernel<HD, 2, 2>), g, b, 0, s, a);
  } else {
    if (a.q_bf16) hipLaunchKernelGGL((token_kernel<HD, 1, 3>), g, b, 0, s, a);
    else hipLaunchKernelGGL((token_kernel<HD, 3, 3>), g, b, 0, s, a);
  }
  if (a.parts > 1) hipLaunchKernelGGL((seq_join_pages<HD, 64, true>), dim3((unsigned)((a.walkers - 1) * a.kv_heads)), dim3(512), 0, s, a);
}

}  // namespace fh

using namespace fh;

// Workgroups that the GPU holds at a time: two a CU, three of the smaller dimensions' where their registers leave room (of token_kernel
// one, and two of the smaller dimensions). They share the keys (SeqWalk). A call of no more rows than sequences and at most PG_WHOLE
// (token_kernel: PG_WHOLE_FEW) places takes a workgroup a sequence and key head instead and needs no second launch: 8 sequences of up to
// 500 11.7 us, shared out 13.8; 16 of up to 2000 30.5, 23.1. The rest is what was measured best: the least share of a workgroup, and
// the cost from which a tile of 128 pairs of 128 dimensions is cut (its parts are 66 KB each, written and read: 16 prompts of up to 300 38 us,
// with every tile cut 55). Prompts of tiles enough for every workgroup that the GPU holds, no sequence of which may outweigh the others' (PG_EACH:
// rows a sequence times rounds of tiles against max_context), go a tile a workgroup as they come, a sequence's longest first, without cuts
// or a join: with bf16 q, lengths and places evenly spaced in three mixed orders, 16 of 100 to 400 rows 53-61 -> 45-50 us, 4 of 1024 to 2048 170-178 -> 148-154,
// one of 2048 86 -> 79, 16 of 512 after up to 4000 places 524-530 -> 462-487; but 8 of these 263-271 -> 261-297, 6 of them beside 24 tokens
// 241-246 -> 265-292, and over an fp32 cache 4 of 512 to 1500 368 -> 370-429.
constexpr int PG_WHOLE = 448, PG_WHOLE_FEW = 1024, PG_LEAST_TOKENS = 128, PG_LEAST = 256, PG_UNCUT = 512;
constexpr int PG_EACH = 4;
static int paged_slots(int head_dim) { return SQ_CUS * (head_dim == 64 ? 3 : 2); }

extern "C" size_t fh_attention_paged_workspace_bytes(int64_t rows, int sequences, int heads, int kv_heads, int head_dim,
                                                     int64_t max_context) {
  if (rows < 1 || sequences < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || max_context < 1) return 0;
  // (two parts a workgroup, at most 128 pairs each and no more than there are: the bound of any call of no more)
  const int64_t pairs = std::min<int64_t>(128, rows * (heads / kv_heads));
  return parts_bytes(2 * std::max<int64_t>(paged_slots(head_dim), (int64_t)kv_heads * ((heads / kv_heads + 63) / 64)) * pairs, head_dim);
}

extern "C" int fh_attention_paged(const void* q, int q_dtype, int64_t ldq, const void* cache, int cache_dtype, int64_t cache_len,
                                  int64_t rows, int sequences, int heads, int kv_heads, int head_dim, const int32_t* starts,
                                  const int32_t* p0, const int32_t* tables, int64_t ldt, int64_t table_cols, int page,
                                  int64_t max_context, void* o, int o_dtype, int64_t ldo, void* workspace, size_t ws_bytes,
                                  void* stream) {
  const char* fn = "fh_attention_paged";
  SeqArgs a = {};
  a.q = q; a.q_bf16 = q_dtype == FH_BF16; a.ldq = ldq; a.cache = cache; a.cache_len = cache_len;
  a.heads = heads; a.kv_heads = kv_heads; a.rows = rows; a.n = sequences;
  a.starts = starts; a.places = p0; a.tables = tables; a.ldt = ldt;
  a.o = o; a.o_bf16 = o_dtype == FH_BF16; a.ldo = ldo;
  if (!starts || !tables) return fail(FH_EINVAL, "fh_attention_paged: null pointer");
  if (rows < 1 || rows >= (1LL << 31) || sequences < 1 || max_context < 1)
    return fail(FH_EINVAL, "fh_attention_paged: need 1 <= rows < 2^31, sequences >= 1 and max_context >= 1");
  if (page < 16 || (page & (page - 1))) return fail(FH_EUNSUP, "fh_attention_paged: pages of 16, 32, 64, ... rows (a power of 2)");
  if (cache_len < page || cache_len % page) return fail(FH_EINVAL, "fh_attention_paged: cache_len is whole pages");
  if (table_cols < 1 || ldt < table_cols) return fail(FH_EINVAL, "fh_attention_paged: tables of at least one page a sequence, rows at least as far apart");
  if (o_dtype != FH_F32 && o_dtype != FH_BF16) return fail(FH_EINVAL, "fh_attention_paged: o is FH_F32 or FH_BF16");
  if (int rc = seq_check(fn, a, q_dtype, cache_dtype, head_dim, o_dtype)) return rc;
  a.page_shift = __builtin_ctz((unsigned)page);
  a.pages = (int)(cache_len >> a.page_shift);
  a.table_cols = (int)std::min<int64_t>(table_cols, 1 << 30);
  max_context = std::min({max_context, (int64_t)a.table_cols << a.page_shift, (int64_t)1 << 30});
  a.max_own = max_context;
  a.rep = heads / kv_heads;
  a.cache_exps = (const uint8_t*)cache + kv_exps_at(cache_dtype, kv_heads, cache_len, head_dim);
  a.scale = 1.0f / sqrtf((float)head_dim);
  const bool few = cache_dtype == FH_BF16 && a.rep <= 16 && rows * a.rep <= (int64_t)16 * sequences;
  const int pairs = few ? 16 : packed_pairs(rows, sequences, a.rep, cache_dtype);
  const bool tokens = pairs <= 64, small = tokens || cache_dtype == FH_F32;
  a.tile_rows = std::max(1, pairs / a.rep);
  a.head_tiles = (a.rep + pairs - 1) / pairs;
  a.slot_pairs = (int)std::min<int64_t>(pairs, rows * a.rep);
  a.whole = tokens && rows <= sequences && max_context <= (few ? PG_WHOLE_FEW : PG_WHOLE) &&
            (int64_t)sequences * kv_heads * a.head_tiles < (1 << 24);  // (a grid's work-items are counted in 32 bits)
  a.walkers = a.whole ? sequences : std::max(1, (few ? SQ_CUS * 128 / head_dim : paged_slots(head_dim)) / (kv_heads * a.head_tiles));
  // (the costs' unit: their sum stays below 2^30)
  const int64_t tiles = rows / a.tile_rows + std::min<int64_t>(sequences, rows), cost = max_context + SEQ_START + a.tile_rows;
  while ((double)tiles * (double)(((cost + rows) >> a.unit) + 1) >= (double)(1 << 30) && a.unit < 30) ++a.unit;
  a.least = std::max(1, (small ? PG_LEAST_TOKENS : PG_LEAST) >> a.unit);
  a.uncut = small ? 0 : PG_UNCUT * head_dim / 128 >> a.unit;
  a.parts = a.walkers > 1 && !a.whole && cost >> a.unit >= a.uncut ? 2 : 1;
  const double each = (double)tiles * kv_heads * a.head_tiles, rounds = each / paged_slots(head_dim);
  if (!small && rounds >= 1 && each < (1 << 24) && max_context < (1 << 29) && rounds * PG_EACH * rows >= (double)max_context * sequences) {
    a.unit = 30; a.least = 1; a.walkers = (int)tiles; a.parts = 1;  // (a cost of 1 a tile, a share of one)
  }
  if (a.parts == 1) a.uncut = 0x7FFFFFFF;
  a.part = (float*)workspace;
  const int64_t blocks = (int64_t)a.walkers * kv_heads * a.head_tiles;
  if (a.parts > 1 && (!workspace || ws_bytes < parts_bytes(2 * blocks * a.slot_pairs, head_dim) || ((uintptr_t)workspace & 15)))
    return fail(FH_EINVAL, "fh_attention_paged: a 16-byte aligned workspace of fh_attention_paged_workspace_bytes");
  if (few) {
    if (head_dim == 128) launch_tokens<128>((unsigned)blocks, as_stream(stream), a);
    else launch_tokens<64>((unsigned)blocks, as_stream(stream), a);
    return check_launch(fn);
  }
  return launch_seq<true>(fn, head_dim, cache_dtype, pairs, blocks, as_stream(stream), a);
}
