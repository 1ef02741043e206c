// Low-rank adapters beside a shared projection, each row its own: y = residual + scale_i (x A_i^T) B_i^T for a row whose adapter is
// i, A_i [parts rank][K] and B_i [N][rank] as a checkpoint holds them. A fused projection's parts (q, k and v; gate and up) are
// runs of B's rows, each with its own `rank` rows of A. A row with no adapter keeps its residual.
//
// Two launches: u = x A^T, its K cut into parts that different workgroups sum (u is narrow: without them one prompt tile would be
// one workgroup), then y = residual + scale u B^T, which adds the parts in order as it takes them. A workgroup takes 64
// consecutive rows and goes through the adapters among them, each with its own rows gathered, 16 a matrix operand: a packed
// prompt's rows are one adapter's, a decode step's as many as there are users, shared out among workgroups.
//
// Both matrices' operands are 8 consecutive values along their inner axis, which is the axis that a checkpoint's rows run
// along, so x, A and B go from memory to the matrix cores' registers as they lie. Products are bf16's with fp32 sums
// (v_mfma_f32_16x16x32_bf16): bf16 values go in as they are, fp32 ones (x, u, an fp32 adapter) as two bf16 terms for bf16 output
// (2^-16 of themselves, less than the output's own rounding, 2^-8) and as three for fp32 output (2^-24).
#include <algorithm>
#include "fh_common.h"

namespace fh {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 lr_bf16x8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float lr_floatx4;

constexpr int LR_ROWS = 64;        // rows a tile
constexpr int LR_WAVES = 4;
constexpr int LR_COLS = 64;        // columns of u a workgroup of the first kernel
constexpr int LR_MAX_PARTS = 4;    // parts of a fused projection
constexpr int LR_MAX_RANK = 128;

struct LoraArgs {
  const void* x; int64_t ldx; int64_t rows, K;
  const void* a; const void* b; const float* scale; const int32_t* ids;
  int adapters, rank, parts, C, N;      // C = parts rank
  int col0[LR_MAX_PARTS + 1];           // each part's first column of y
  int chunk0[LR_MAX_PARTS + 1];         // each part's first chunk of `width` columns
  int width, share, splits;             // workgroups a tile's adapters are shared among; parts of K
  int kstep;                            // K a part, a multiple of 64
  float* u;                             // [splits][rows][C]
  const void* residual; int64_t ldr; void* y; int64_t ldy;
};

// x's bf16 terms: the value to nearest, then what is left to nearest
template <int N>
__device__ inline void lr_terms(const float (&x)[8], lr_bf16x8 (&t)[N]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float left = x[i];
#pragma unroll
    for (int j = 0; j < N; ++j) { t[j][i] = (__bf16)left; left -= (float)t[j][i]; }
  }
}

// 8 values from p + at as N bf16 terms (bf16 ones: one); zeros where not `in` (at is inside the buffer all the same)
template <bool BF, int N>
__device__ inline void lr_load(const void* p, int64_t at, bool in, lr_bf16x8 (&t)[N]) {
  if constexpr (BF) {
    uint4 w = *(const uint4*)((const uint16_t*)p + at);
    if (!in) w = make_uint4(0, 0, 0, 0);
    t[0] = *(const lr_bf16x8*)&w;
  } else {
    const float4 a = *(const float4*)((const float*)p + at), b = *(const float4*)((const float*)p + at + 4);
    float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (!in)
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = 0.f;
    lr_terms<N>(f, t);
  }
}

// the products of two operands in terms that matter: those whose terms' places sum to less than the longer operand's count
template <int NA, int NB>
__device__ inline lr_floatx4 lr_mfma(const lr_bf16x8 (&a)[NA], const lr_bf16x8 (&b)[NB], lr_floatx4 c) {
  constexpr int MOST = NA > NB ? NA : NB;
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < MOST) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], c, 0, 0, 0);
  return c;
}

// The adapters of a tile of 64 rows, one after another: each lane's row's, and the rows still to take
struct LoraTile {
  int64_t t0; int id; uint64_t left; int turn;
  __device__ LoraTile(const LoraArgs& a, int64_t tile) {
    const int lane = threadIdx.x & 63;
    t0 = tile * LR_ROWS;
    const int i = a.ids[min(t0 + lane, a.rows - 1)];
    id = i >= 0 && i < a.adapters ? i : -1;
    left = __ballot(t0 + lane < a.rows);
    turn = 0;
  }
  // the next adapter that is this workgroup's (of `share` that take them in turn) and its rows; false: no more
  __device__ bool next(int share, int mine, int& adapter, uint64_t& rows) {
    while (left) {
      adapter = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
      rows = __ballot(id == adapter) & left;
      left &= ~rows;
      if (turn++ % share == mine) return true;
    }
    return false;
  }
};

// the n-th set bit of rows, n a lane's own (n below their count)
__device__ inline int lr_nth(uint64_t rows, int n) {
  int at = 0;
#pragma unroll
  for (int w = 32; w >= 1; w >>= 1) {
    const int c = __builtin_popcountll(rows & ((1ull << w) - 1));
    if (n >= c) { n -= c; rows >>= w; at += w; }
  }
  return at;
}

// u[part][row][c] = the part of K's products of x's row and A's row c
template <bool XB, bool WB, int XT, int WT>
__global__ __launch_bounds__(64 * LR_WAVES) void lora_shrink(LoraArgs a) {
  __shared__ __attribute__((aligned(16))) float sums[LR_WAVES - 1][LR_ROWS * LR_COLS];
  const int split = blockIdx.x % a.splits, group = blockIdx.x / a.splits, c0 = group * LR_COLS;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int cols = min(LR_COLS, a.C - c0), cb = (cols + 15) / 16;
  const int k0 = split * a.kstep, k1 = (int)min((int64_t)k0 + a.kstep, a.K);
  LoraTile tile(a, blockIdx.z);
  int adapter;
  uint64_t rows;
  while (tile.next(a.share, blockIdx.y, adapter, rows)) {
    if (adapter < 0) continue;
    const int n = __builtin_popcountll(rows), mb = (n + 15) / 16;
    const int64_t wbase = (int64_t)adapter * a.C * a.K;
    lr_floatx4 acc[4][4];
    int64_t xat[4], wat[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      xat[i] = (tile.t0 + lr_nth(rows, min(16 * i + r, n - 1))) * a.ldx;
      wat[i] = wbase + (int64_t)(c0 + min(16 * i + r, cols - 1)) * a.K;
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = lr_floatx4{0.f, 0.f, 0.f, 0.f};
    }
    for (int k = k0 + 64 * wave; k < k1; k += 64 * LR_WAVES)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int kk = k + 32 * h + 8 * g;
        const bool in = kk < k1;
        const int at = in ? kk : 0;
        lr_bf16x8 xf[4][XT];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < mb) lr_load<XB, XT>(a.x, xat[i] + at, in, xf[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < cb) {
            lr_bf16x8 wf[WT];
            lr_load<WB, WT>(a.a, wat[j] + at, in, wf);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (i < mb) acc[i][j] = lr_mfma<XT, WT>(xf[i], wf, acc[i][j]);
          }
      }
    // the waves' sums, in order; lane (r, g) holds rows 16 i + 4 g .. + 3 of column 16 j + r
    if (wave > 0)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i < mb && j < cb) *(lr_floatx4*)&sums[wave - 1][((i * 4 + j) * 64 + lane) * 4] = acc[i][j];
    __syncthreads();
    if (wave == 0)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i < mb && j < cb) {
#pragma unroll
            for (int w = 0; w < LR_WAVES - 1; ++w) acc[i][j] += *(const lr_floatx4*)&sums[w][((i * 4 + j) * 64 + lane) * 4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int m = 16 * i + 4 * g + e, c = 16 * j + r;
              if (m < n && c < cols) a.u[((int64_t)split * a.rows + tile.t0 + lr_nth(rows, m)) * a.C + c0 + c] = acc[i][j][e];
            }
          }
    __syncthreads();
  }
}

__device__ inline void lr_read8(const void* p, bool bf, int64_t at, float (&f)[8]) {
  if (bf) {
    const uint4 w = *(const uint4*)((const uint16_t*)p + at);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(u[i] << 16); f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u); }
  } else {
    const float4 u = *(const float4*)((const float*)p + at), v = *(const float4*)((const float*)p + at + 4);
    f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w; f[4] = v.x; f[5] = v.y; f[6] = v.z; f[7] = v.w;
  }
}
template <bool BF>
__device__ inline void lr_write8(void* p, int64_t at, const float (&f)[8]) {
  if constexpr (BF) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = bf16_rne_f(f[2 * i]) | (bf16_rne_f(f[2 * i + 1]) << 16);
    *(uint4*)((uint16_t*)p + at) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    *(float4*)((float*)p + at) = make_float4(f[0], f[1], f[2], f[3]);
    *(float4*)((float*)p + at + 4) = make_float4(f[4], f[5], f[6], f[7]);
  }
}

// y = residual + scale u B^T: a workgroup a chunk of a part's columns. B's rows are the product's rows and x's rows its
// columns: two blocks of 16 of B's rows are rows 8 (r / 4) + r % 4 and those 4 on, so that a lane ends with 8 consecutive columns of
// y's row, 16 or 32 bytes.
template <bool WB, bool YB, int UT, int WT>
__global__ __launch_bounds__(64 * LR_WAVES) void lora_expand(LoraArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint16_t us[];  // [UT][64][ldu] u's terms
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  int part = 0;
  while (part + 1 < a.parts && (int)blockIdx.x >= a.chunk0[part + 1]) ++part;
  const int n0 = a.col0[part] + (blockIdx.x - a.chunk0[part]) * a.width, n1 = min(n0 + a.width, a.col0[part + 1]);
  const int steps = (a.rank + 31) / 32, ldu = 32 * steps + 8;
  LoraTile tile(a, blockIdx.z);
  int adapter;
  uint64_t rows;
  while (tile.next(a.share, blockIdx.y, adapter, rows)) {
    const int n = __builtin_popcountll(rows);
    if (adapter < 0) {  // the residual, or zeros
      if (a.residual == a.y) continue;
      const int pieces = (n1 - n0) / 8;
      for (int i = threadIdx.x; i < n * pieces; i += 64 * LR_WAVES) {
        const int64_t t = tile.t0 + lr_nth(rows, i / pieces), c = n0 + i % pieces * 8;
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (a.residual) lr_read8(a.residual, YB, t * a.ldr + c, f);
        lr_write8<YB>(a.y, t * a.ldy + c, f);
      }
      continue;
    }
    __syncthreads();  // (the last adapter's u is read)
    const float sc = a.scale ? a.scale[adapter] : 1.f;
    for (int i = threadIdx.x; i < n * 4 * steps; i += 64 * LR_WAVES) {  // 8 of a row's u at a time: the parts of K, in order
      const int m = i / (4 * steps), k = i % (4 * steps) * 8;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (k < a.rank) {
        const float* p = a.u + (tile.t0 + lr_nth(rows, m)) * a.C + part * a.rank + k;
        for (int s = 0; s < a.splits; ++s, p += a.rows * a.C) {
          const float4 v = *(const float4*)p, w = *(const float4*)(p + 4);
          f[0] += v.x; f[1] += v.y; f[2] += v.z; f[3] += v.w; f[4] += w.x; f[5] += w.y; f[6] += w.z; f[7] += w.w;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= sc;
      }
      lr_bf16x8 t[UT];
      lr_terms<UT>(f, t);
#pragma unroll
      for (int e = 0; e < UT; ++e) *(lr_bf16x8*)(us + (e * LR_ROWS + m) * ldu + k) = t[e];
    }
    __syncthreads();
    const int mb = (n + 15) / 16;
    int64_t row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) row[i] = tile.t0 + lr_nth(rows, min(16 * i + r, n - 1));
    const int64_t wbase = (int64_t)adapter * a.N * a.rank;
    for (int c = n0 + 32 * wave; c < n1; c += 32 * LR_WAVES) {
      const int col = c + 8 * g;  // the lane's 8 columns of y
      const int64_t w0 = wbase + (int64_t)min(c + 8 * (r >> 2) + (r & 3), n1 - 1) * a.rank;
      const int64_t w1 = wbase + (int64_t)min(c + 8 * (r >> 2) + 4 + (r & 3), n1 - 1) * a.rank;
      lr_floatx4 acc[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i][0] = acc[i][1] = lr_floatx4{0.f, 0.f, 0.f, 0.f};
      for (int s = 0; s < steps; ++s) {
        const int k = 32 * s + 8 * g;
        const bool in = k < a.rank;
        lr_bf16x8 b0[WT], b1[WT];
        lr_load<WB, WT>(a.b, w0 + (in ? k : 0), in, b0);
        lr_load<WB, WT>(a.b, w1 + (in ? k : 0), in, b1);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < mb) {
            lr_bf16x8 uf[UT];
#pragma unroll
            for (int e = 0; e < UT; ++e) uf[e] = *(const lr_bf16x8*)(us + (e * LR_ROWS + min(16 * i + r, n - 1)) * ldu + k);
            acc[i][0] = lr_mfma<WT, UT>(b0, uf, acc[i][0]);
            acc[i][1] = lr_mfma<WT, UT>(b1, uf, acc[i][1]);
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (16 * i + r < n && col < n1) {
          float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          if (a.residual) lr_read8(a.residual, YB, row[i] * a.ldr + col, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] += acc[i][e >> 2][e & 3];
          lr_write8<YB>(a.y, row[i] * a.ldy + col, f);
        }
    }
  }
}

// Parts of K: whole steps of 256 (a wave's 64 each), as many as keep the parts' rows within 16384, so that u's parts stay a
// small share of what a call moves and a decode step's few rows still fill the GPU.
constexpr int LR_MAX_SPLITS = 32;
constexpr int64_t LR_SPLIT_ROWS = 16384;
static int lora_splits(int64_t rows, int64_t K) {
  const int64_t most = std::min<int64_t>(LR_MAX_SPLITS, (K + 255) / 256);
  return (int)std::max<int64_t>(1, std::min(most, LR_SPLIT_ROWS / rows));
}

template <bool XB, bool WB, bool YB>
static void launch_lora(hipStream_t s, const LoraArgs& a) {
  constexpr int T = YB ? 2 : 3, XT = XB ? 1 : T, WT = WB ? 1 : T;
  const unsigned tiles = (unsigned)((a.rows + LR_ROWS - 1) / LR_ROWS), groups = (unsigned)((a.C + LR_COLS - 1) / LR_COLS);
  hipLaunchKernelGGL((lora_shrink<XB, WB, XT, WT>), dim3(a.splits * groups, a.share, tiles), dim3(64 * LR_WAVES), 0, s, a);
  const int ldu = 32 * ((a.rank + 31) / 32) + 8;
  hipLaunchKernelGGL((lora_expand<WB, YB, T, WT>), dim3(a.chunk0[a.parts], a.share, tiles), dim3(64 * LR_WAVES), (size_t)T * LR_ROWS * ldu * 2, s, a);
}

}  // namespace fh

using namespace fh;

extern "C" size_t fh_lora_workspace_bytes(int64_t rows, int64_t K, int rank, int parts) {
  if (rows < 1 || rows >= (1LL << 31) || K < 1 || rank < 1 || rank > LR_MAX_RANK || parts < 1 || parts > LR_MAX_PARTS) return 0;
  // (the parts' rows of any call of no more rows)
  const int64_t most = std::min<int64_t>(LR_MAX_SPLITS, (K + 255) / 256);
  return (size_t)std::max(rows, std::min(rows * most, LR_SPLIT_ROWS)) * rank * parts * sizeof(float);
}

extern "C" int fh_lora(const void* x, int x_dtype, int64_t ldx, int64_t rows, int64_t K, const void* a_w, const void* b_w, int w_dtype,
                       int adapters, int rank, int parts, const int64_t* part_cols, const float* scale, const int32_t* ids,
                       const void* residual, int64_t ldr, void* y, int y_dtype, int64_t ldy, void* workspace, size_t ws_bytes,
                       void* stream) {
  auto no = [](int code, const char* what) { set_error("fh_lora: %s", what); return code; };
  if (!x || !a_w || !b_w || !part_cols || !ids || !y) return no(FH_EINVAL, "null pointer");
  if (rows < 1 || K < 1 || adapters < 1) return no(FH_EINVAL, "need rows, K and adapters of at least 1");
  if (rows > 64LL * 65535 || K >= (1LL << 30)) return no(FH_EUNSUP, "at most 64 * 65535 rows, K below 2^30");
  if (rank < 1 || rank % 8 || rank > LR_MAX_RANK || K % 8) return no(FH_EUNSUP, "rank 8, 16, ..., 128 and K a multiple of 8 (zeros behind what an adapter has)");
  if (parts < 1 || parts > LR_MAX_PARTS) return no(FH_EUNSUP, "1 to 4 parts");
  if (x_dtype != FH_F32 && x_dtype != FH_BF16) return no(FH_EINVAL, "x is FH_F32 or FH_BF16");
  if (w_dtype != FH_F32 && w_dtype != FH_BF16) return no(FH_EINVAL, "the adapters are FH_F32 or FH_BF16");
  if (y_dtype != FH_F32 && y_dtype != FH_BF16) return no(FH_EINVAL, "y is FH_F32 or FH_BF16");
  LoraArgs l = {};
  int64_t N = 0;
  for (int p = 0; p < parts; ++p) {
    if (part_cols[p] < 8 || part_cols[p] % 8 || part_cols[p] >= (1LL << 30)) return no(FH_EUNSUP, "each part's columns a multiple of 8, below 2^30");
    l.col0[p] = (int)N;
    N += part_cols[p];
    if (N >= (1LL << 30)) return no(FH_EUNSUP, "fewer than 2^30 columns");
  }
  l.col0[parts] = (int)N;
  if (ldx < K || ldy < N || (residual && ldr < N) || ldx % (x_dtype == FH_F32 ? 4 : 8) || ldy % (y_dtype == FH_F32 ? 4 : 8) ||
      (residual && ldr % (y_dtype == FH_F32 ? 4 : 8)) || (((uintptr_t)x | (uintptr_t)a_w | (uintptr_t)b_w | (uintptr_t)y | (uintptr_t)residual) & 15))
    return no(FH_EINVAL, "rows at least K and N, 16-byte aligned, as the adapters");
  if (residual == y && ldr != ldy) return no(FH_EINVAL, "a residual that is y itself has y's rows");
  l.splits = lora_splits(rows, K);
  const size_t need = (size_t)l.splits * rows * rank * parts * sizeof(float);
  if (!workspace || ws_bytes < need || ((uintptr_t)workspace & 15)) return no(FH_EINVAL, "a 16-byte aligned workspace of fh_lora_workspace_bytes");
  l.x = x; l.ldx = ldx; l.rows = rows; l.K = K; l.a = a_w; l.b = b_w; l.scale = scale; l.ids = ids;
  l.adapters = adapters; l.rank = rank; l.parts = parts; l.C = rank * parts; l.N = (int)N;
  l.kstep = (int)((K + 64 * l.splits - 1) / (64 * l.splits)) * 64;
  l.u = (float*)workspace; l.residual = residual; l.ldr = residual ? ldr : ldy; l.y = y; l.ldy = ldy;
  const int64_t tiles = (rows + LR_ROWS - 1) / LR_ROWS;
  l.share = (int)(tiles > 16 ? 1 : std::min<int64_t>(std::min<int64_t>(adapters + 1LL, rows), LR_ROWS));
  l.width = 256;
  int chunks = 0;
  for (int p = 0; p < parts; ++p) { l.chunk0[p] = chunks; chunks += (int)((part_cols[p] + l.width - 1) / l.width); }
  l.chunk0[parts] = chunks;
  const hipStream_t s = as_stream(stream);
  const int form = (x_dtype == FH_BF16) * 4 + (w_dtype == FH_BF16) * 2 + (y_dtype == FH_BF16);
  switch (form) {
    case 0: launch_lora<false, false, false>(s, l); break;
    case 1: launch_lora<false, false, true>(s, l); break;
    case 2: launch_lora<false, true, false>(s, l); break;
    case 3: launch_lora<false, true, true>(s, l); break;
    case 4: launch_lora<true, false, false>(s, l); break;
    case 5: launch_lora<true, false, true>(s, l); break;
    case 6: launch_lora<true, true, false>(s, l); break;
    default: launch_lora<true, true, true>(s, l); break;
  }
  return check_launch("fh_lora");
}
