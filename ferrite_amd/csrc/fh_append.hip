// The heads of a projection's rows made ready for attention over a cache in pages, in one pass: q's and k's heads through their
// RMSNorm (each head its own mean of squares) and the rotation of their row's place, q out, k and v into the page that the
// sequence's table names for the place, rounded once into whatever the cache holds.
//   n = x rsqrt(mean x^2 + eps) w        (w + 1 centered; q's and k's heads, where weights are given)
//   y = n cos + (-n2, n1) sin            (their halves n1, n2)
//
// A workgroup a row or two, HD / 8 lanes a head: a lane holds columns 4 l .. 4 l + 3 of each half, so that a pair turns in the lane, a
// head's squares meet over 8 or 16 lanes, and a block float's run of 16 columns over 4. What a row waits for is a chain of loads (its
// sequence, its place, its page's number and its row of the tables), so its own values are on their way before the first of them.
// 3517 rows of 32 + 8 + 8 heads of 128, bf16, normed: 21.3-22.3 us for 89 MB, 4.1 TB/s where a copy reaches 5.15; 4 rows a workgroup 27, the
// next row's values loaded behind this one's 27: fewer chains at a time. One row of 9 + 3 + 3 heads of 64: 2.9 us in a graph. Into bfp8,
// 2444 rows of 20 + 4 + 4 heads of 64, normed: 10.1 us for 33 MB (6.3 at a copy's rate); its keys take 64 bits, and with 8 heads of 64 a wave
// the waves that hold both q's and k's run both arithmetics, one after the other (here one of a row's four, all of its keys).
#include <algorithm>
#include <type_traits>
#include "fh_common.h"

namespace fh {

struct AppendArgs {
  const void* x; int64_t ldx;
  int64_t rows; int n, heads, kv_heads;
  const float* q_norm; const float* k_norm; float eps; int centered;
  const float* cos_tab; const float* sin_tab; int64_t rope_rows;
  const int32_t* starts; const int32_t* p0; const int32_t* tables; int64_t ldt; int table_cols, pages, page_shift;
  void* q; int q_bf16; int64_t ldq;
  void* cache; uint8_t* exps; int64_t cache_len;
};

template <bool BF>
__device__ inline float4 load4(const void* p, int at) {
  if constexpr (!BF) return *(const float4*)((const float*)p + at);
  else {
    const uint2 w = *(const uint2*)((const uint16_t*)p + at);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u));
  }
}
__device__ inline uint32_t two_bf16(float lo, float hi) {  // (nearest even, by the chip's conversion)
  typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf2;
  const bf2 v = {(__bf16)lo, (__bf16)hi};
  return *(const uint32_t*)&v;
}
__device__ inline void store4(void* p, bool bf, int at, float4 v) {
  if (bf) *(uint2*)((uint16_t*)p + at) = make_uint2(two_bf16(v.x, v.y), two_bf16(v.z, v.w));
  else *(float4*)((float*)p + at) = v;
}

// 4 columns of a run of 16 of a block float, the run's other columns in the quad's other lanes: their bytes, and the exponent
template <bool FOUR>
__device__ inline uint32_t run4(float4 v, uint32_t& top) {
  const uint32_t b[4] = {bf16_rne_f(v.x), bf16_rne_f(v.y), bf16_rne_f(v.z), bf16_rne_f(v.w)};
  top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, (b[i] >> 7) & 255u);
  top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
  top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t m = bfp_magnitude(b[i], top, FOUR), s = b[i] >> 15 ? 0u - m : m;
    w |= FOUR ? (s & 15u) << (4 * i) : (s & 255u) << (8 * i);
  }
  return w;
}

// A head's norm and rotation, in F's arithmetic: u and v are the lane's columns of its halves. A block float's keys take 64 bits: it
// rounds twice, and a value that 32 bits leave on the other side of a border ends a whole step of its run away.
template <typename F, int HD>
__device__ inline void norm_turn(const AppendArgs& a, const float* w, int64_t turn, int l, float4& u, float4& v) {
  F x[4] = {u.x, u.y, u.z, u.w}, y[4] = {v.x, v.y, v.z, v.w};
  if (w) {
    F ss = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) ss += x[i] * x[i] + y[i] * y[i];
#pragma unroll
    for (int m = 1; m < HD / 8; m <<= 1) ss += __shfl_xor(ss, m, 64);
    const F mean = ss * F(1.0 / HD) + F(a.eps);
    // Squares that overflow give a mean of infinity and 0, as in the framework's other norms. (The chip's reciprocal root with a step of
    // Newton's is 1.5% faster, 3517 rows of 8B's, but the step is 0 times infinity there, and the root takes no number below the normal ones.)
    F r;
    if constexpr (sizeof(F) == 4) r = 1.f / sqrtf(mean);
    else r = F(1) / sqrt(mean);
    const F c = a.centered ? F(1) : F(0);
    const float4 wu = *(const float4*)(w + 4 * l), wv = *(const float4*)(w + HD / 2 + 4 * l);
    const float wx[4] = {wu.x, wu.y, wu.z, wu.w}, wy[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] *= r * (wx[i] + c); y[i] *= r * (wy[i] + c); }
  }
  if (a.cos_tab) {
    const float* cs = a.cos_tab + turn * HD;
    const float* sn = a.sin_tab + turn * HD;
    const float4 c0 = *(const float4*)(cs + 4 * l), c1 = *(const float4*)(cs + HD / 2 + 4 * l), s0 = *(const float4*)(sn + 4 * l), s1 = *(const float4*)(sn + HD / 2 + 4 * l);
    const float cx[4] = {c0.x, c0.y, c0.z, c0.w}, cy[4] = {c1.x, c1.y, c1.z, c1.w}, sx[4] = {s0.x, s0.y, s0.z, s0.w}, sy[4] = {s1.x, s1.y, s1.z, s1.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const F t = x[i] * cx[i] - y[i] * sx[i];
      y[i] = y[i] * cy[i] + x[i] * sy[i];
      x[i] = t;
    }
  }
  u = make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]);
  v = make_float4((float)y[0], (float)y[1], (float)y[2], (float)y[3]);
}

// R rows a workgroup, what each needs on its way together
template <int HD, int CF, bool BF, int R>
__global__ __launch_bounds__(1024) void append_kernel(AppendArgs a) {
  constexpr int G = HD / 8;  // lanes a head
  const int lane = threadIdx.x & 63, l = threadIdx.x % G, total = a.heads + 2 * a.kv_heads;
  const int64_t t0 = (int64_t)blockIdx.x * R;
  float4 u[R], v[R];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const char* x = (const char*)a.x + min(t0 + i, a.rows - 1) * a.ldx * (BF ? 2 : 4);
      u[i] = load4<BF>(x, h * HD + 4 * l); v[i] = load4<BF>(x, h * HD + HD / 2 + 4 * l);
    }
  };
  const int h0 = threadIdx.x / G;
  load(min(h0, total - 1));
  // each row's sequence: as many as end at or before it
  int s[R];
#pragma unroll
  for (int i = 0; i < R; ++i) s[i] = 0;
  const int begin = a.starts[0];
  for (int s0 = 0; s0 < a.n; s0 += 64) {
    const int e = a.starts[min(s0 + lane, a.n - 1) + 1];
#pragma unroll
    for (int i = 0; i < R; ++i) s[i] += __builtin_popcountll(__ballot(s0 + lane < a.n && e <= t0 + i));
  }
  int first[R], from[R];
#pragma unroll
  for (int i = 0; i < R; ++i) { first[i] = a.p0[min(s[i], a.n - 1)]; from[i] = a.starts[min(s[i], a.n - 1)]; }
  int64_t turn[R], row[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t place = (int64_t)first[i] + t0 + i - from[i], at = place >> a.page_shift;
    turn[i] = place < 0 ? 0 : place >= a.rope_rows ? a.rope_rows - 1 : place;
    // (a place or a page outside: k and v are not written)
    const int page = a.tables[min(s[i], a.n - 1) * a.ldt + (at < 0 ? 0 : at >= a.table_cols ? a.table_cols - 1 : at)];
    row[i] = at >= 0 && at < a.table_cols && page >= 0 && page < a.pages ? ((int64_t)page << a.page_shift) + (place & ((1 << a.page_shift) - 1)) : -1;
  }
  for (int h = h0; h < total; h += blockDim.x / G) {
    if (h != h0) load(h);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t t = t0 + i;
      if (t >= a.rows || t < begin || s[i] >= a.n) continue;
      if (h < a.heads + a.kv_heads) {
        const float* w = h < a.heads ? a.q_norm : a.k_norm;
        if (CF == FH_F32 || CF == FH_BF16 || h < a.heads) norm_turn<float, HD>(a, w, turn[i], l, u[i], v[i]);
        else norm_turn<double, HD>(a, w, turn[i], l, u[i], v[i]);
      }
      if (h < a.heads) {
        char* qrow = (char*)a.q + t * a.ldq * (a.q_bf16 ? 2 : 4);
        store4(qrow, a.q_bf16, h * HD + 4 * l, u[i]);
        store4(qrow, a.q_bf16, h * HD + HD / 2 + 4 * l, v[i]);
        continue;
      }
      if (row[i] < 0) continue;
      const int64_t to = (int64_t)(h - a.heads) * a.cache_len + row[i];
      if constexpr (CF == FH_F32 || CF == FH_BF16) {
        char* at = (char*)a.cache + to * (HD * (CF == FH_BF16 ? 2 : 4));
        store4(at, CF == FH_BF16, 4 * l, u[i]);
        store4(at, CF == FH_BF16, HD / 2 + 4 * l, v[i]);
      } else {
        uint32_t tu, tv;
        const uint32_t mu = run4<CF == FH_BFP4>(u[i], tu), mv = run4<CF == FH_BFP4>(v[i], tv);
        if constexpr (CF == FH_BFP8) {
          uint8_t* m = (uint8_t*)a.cache + to * HD + 4 * l;
          *(uint32_t*)m = mu;
          *(uint32_t*)(m + HD / 2) = mv;
        } else {
          uint8_t* m = (uint8_t*)a.cache + to * (HD / 2) + 2 * l;
          *(uint16_t*)m = (uint16_t)mu;
          *(uint16_t*)(m + HD / 4) = (uint16_t)mv;
        }
        if ((l & 3) == 0) {
          a.exps[to * (HD / 16) + l / 4] = (uint8_t)tu;
          a.exps[to * (HD / 16) + HD / 32 + l / 4] = (uint8_t)tv;
        }
      }
    }
  }
}

static int append_threads(int heads, int kv_heads, int head_dim) { return std::min(1024, ((heads + 2 * kv_heads) * (head_dim / 8) + 63) / 64 * 64); }

template <int HD, int CF>
static void launch_append(bool bf, hipStream_t s, const AppendArgs& a) {
  const dim3 b(append_threads(a.heads, a.kv_heads, HD));
  auto launch = [&](auto rows) {
    constexpr int R = decltype(rows)::value;
    const dim3 g((unsigned)((a.rows + R - 1) / R));
    if (bf) hipLaunchKernelGGL((append_kernel<HD, CF, true, R>), g, b, 0, s, a);
    else hipLaunchKernelGGL((append_kernel<HD, CF, false, R>), g, b, 0, s, a);
  };
  // (two rows a workgroup: 8b, 3517 rows 22.7 -> 21.8 us; a block float's arithmetic and fewer rows are faster in one's workgroups)
  if (CF != FH_BFP8 && CF != FH_BFP4 && a.rows >= 1024) launch(std::integral_constant<int, 2>());
  else launch(std::integral_constant<int, 1>());
}

template <int HD>
static void launch_append(int cf, bool bf, hipStream_t s, const AppendArgs& a) {
  switch (cf) {
    case FH_F32: launch_append<HD, FH_F32>(bf, s, a); break;
    case FH_BF16: launch_append<HD, FH_BF16>(bf, s, a); break;
    case FH_BFP8: launch_append<HD, FH_BFP8>(bf, s, a); break;
    default: launch_append<HD, FH_BFP4>(bf, s, a); break;
  }
}

}  // namespace fh

using namespace fh;

extern "C" int fh_rope_append_paged(const void* qkv, int x_dtype, int64_t ldx, int64_t rows, int sequences, int heads, int kv_heads,
                                    int head_dim, const float* q_norm, const float* k_norm, float eps, int centered,
                                    const float* cos_tab, const float* sin_tab, int64_t rope_rows, const int32_t* starts,
                                    const int32_t* p0, const int32_t* tables, int64_t ldt, int64_t table_cols, int page, void* q,
                                    int q_dtype, int64_t ldq, void* cache, int cache_dtype, int64_t cache_len, void* stream) {
  auto no = [](int code, const char* what) { set_error("fh_rope_append_paged: %s", what); return code; };
  if (!qkv || !q || !cache || !starts || !p0 || !tables) return no(FH_EINVAL, "null pointer");
  if (rows < 1 || rows >= (1LL << 31) || sequences < 1) return no(FH_EINVAL, "need 1 <= rows < 2^31 and sequences >= 1");
  if (heads < 1 || kv_heads < 1) return no(FH_EINVAL, "need heads and kv_heads of at least 1");
  if (heads > 65535 || kv_heads > 65535) return no(FH_EUNSUP, "at most 65535 heads");
  if (head_dim != 64 && head_dim != 128) return no(FH_EUNSUP, "head_dim 64 or 128");
  if (x_dtype != FH_F32 && x_dtype != FH_BF16) return no(FH_EINVAL, "qkv is FH_F32 or FH_BF16");
  if (q_dtype != FH_F32 && q_dtype != FH_BF16) return no(FH_EINVAL, "q is FH_F32 or FH_BF16");
  if (cache_dtype < FH_F32 || cache_dtype > FH_BFP4) return no(FH_EUNSUP, "cache is FH_F32, FH_BF16, FH_BFP8 or FH_BFP4");
  if ((cos_tab == nullptr) != (sin_tab == nullptr) || (cos_tab && rope_rows < 1)) return no(FH_EINVAL, "cos_tab and sin_tab go together, with rope_rows, their rows");
  if (page < 16 || (page & (page - 1))) return no(FH_EUNSUP, "pages of 16, 32, 64, ... rows (a power of 2)");
  if (cache_len < page || cache_len % page) return no(FH_EINVAL, "cache_len is whole pages");
  if (cache_len >= (1LL << 30)) return no(FH_EUNSUP, "fewer than 2^30 cache rows");
  if (table_cols < 1 || ldt < table_cols) return no(FH_EINVAL, "tables of at least one page a sequence, rows at least as far apart");
  if (ldx < (int64_t)(heads + 2 * kv_heads) * head_dim || ldq < (int64_t)heads * head_dim || ldx % 4 || ldq % 4 ||
      ((uintptr_t)qkv & (x_dtype == FH_F32 ? 15 : 7)) || ((uintptr_t)q & (q_dtype == FH_F32 ? 15 : 7)) || ((uintptr_t)cache & 15))
    return no(FH_EINVAL, "rows at least their heads, qkv's and q's aligned to 4 values, the cache to 16 bytes");
  if (((uintptr_t)q_norm & 15) || ((uintptr_t)k_norm & 15) || ((uintptr_t)cos_tab & 15) || ((uintptr_t)sin_tab & 15))
    return no(FH_EINVAL, "norms and tables 16-byte aligned");
  if (q == qkv && (q_dtype != x_dtype || (rows > 1 && ldq != ldx))) return no(FH_EINVAL, "q in qkv's own columns has qkv's type and its rows");
  // (a grid's work-items are counted in 32 bits)
  if (rows * append_threads(heads, kv_heads, head_dim) >= (1LL << 32)) return no(FH_EUNSUP, "too many rows for one grid");
  AppendArgs a = {};
  a.x = qkv; a.ldx = ldx; a.rows = rows; a.n = sequences; a.heads = heads; a.kv_heads = kv_heads;
  a.q_norm = q_norm; a.k_norm = k_norm; a.eps = eps; a.centered = centered;
  a.cos_tab = cos_tab; a.sin_tab = sin_tab; a.rope_rows = rope_rows;
  a.starts = starts; a.p0 = p0; a.tables = tables; a.ldt = ldt; a.table_cols = (int)std::min<int64_t>(table_cols, 1 << 30);
  a.page_shift = __builtin_ctz((unsigned)page); a.pages = (int)(cache_len >> a.page_shift);
  a.q = q; a.q_bf16 = q_dtype == FH_BF16; a.ldq = ldq;
  a.cache = cache; a.exps = (uint8_t*)cache + kv_exps_at(cache_dtype, kv_heads, cache_len, head_dim); a.cache_len = cache_len;
  if (head_dim == 128) launch_append<128>(cache_dtype, x_dtype == FH_BF16, as_stream(stream), a);
  else launch_append<64>(cache_dtype, x_dtype == FH_BF16, as_stream(stream), a);
  return check_launch("fh_rope_append_paged");
}
