// Low-rank adapters beside a shared projection, each row its own: y = residual + scale_i (x A_i^T) B_i^T for a row whose adapter is
// i, A_i [parts rank][K] and B_i [N][rank] as a checkpoint holds them. A fused projection's parts (q, k and v; gate and up) are
// runs of B's rows, each with its own `rank` rows of A. A row with no adapter keeps its residual.
//
// Two launches: u = x A^T, its K cut into parts that different workgroups sum (u is narrow: without them one prompt tile would be
// one workgroup), then y = residual + scale u B^T, which adds the parts in order as it takes them. A workgroup takes 64
// consecutive rows and goes through the adapters among them, each with its own rows gathered, 16 a matrix operand: a packed
// prompt's rows are one adapter's, a decode step's as many as there are users, shared out among workgroups. A few rows by small
// matrices take one launch (lora_few).
//
// Both matrices' operands are 8 consecutive values along their inner axis, which is the axis that a checkpoint's rows run
// along, so x, A and B go from memory to the matrix cores' registers as they lie. Products are bf16's with fp32 sums
// (v_mfma_f32_16x16x32_bf16): bf16 values go in as they are, fp32 ones (x, u, an fp32 adapter) as two bf16 terms for bf16 output
// (2^-16 of themselves, less than the output's own rounding, 2^-8) and as three for fp32 output (2^-24).
//
// What bounds it (MI355X, calls in a replayed graph): the bytes, and for few rows the chain of loads. Beside an 8B model's gate and up, rank 32,
// 4096 rows of 4 adapters, bf16: 133-137 us for 510 MB, 22 of them u (37 MB: 256 workgroups, one a CU, each wave with one round of 64 of K on its
// way), the rest y's 470 MB read and written at 4.2 TB/s where a copy reaches 5.15; with an fp32 y 211 for 980 MB. 333 fp32 rows of 6 adapters by 3456
// 20 us for 8 MB: fp32 x and A do not go through LDS, a lane's 32 bytes lie in rows K apart, and each of 210 workgroups adds 14 parts of K again;
// beside its q, k and v, rank 16, 32 rows of 24 adapters 12.5 us for 11 MB, a chain of loads in each of two launches.
#include <algorithm>
#include "fh_common.h"

namespace fh {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 lr_bf16x8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float lr_floatx4;

constexpr int LR_ROWS = 64;        // rows a tile
constexpr int LR_WAVES = 4;
constexpr int LR_WIDTH = 256;      // columns of y a workgroup of the second: 512 is 3% faster for 4096 rows, 12% slower for 500
constexpr int LR_FEW_WIDTH = 512;  // of lora_few
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

// 8 values as loaded, and as N bf16 terms (bf16 ones: one); zeros where not `in` (what was loaded is inside the buffer all the same)
template <bool BF>
struct LrRaw {
  uint4 a, b;
  __device__ void load(const void* p, int64_t at) {
    if constexpr (BF) a = *(const uint4*)((const uint16_t*)p + at);
    else { a = *(const uint4*)((const float*)p + at); b = *(const uint4*)((const float*)p + at + 4); }
  }
  __device__ void values(float (&f)[8]) const {
    if constexpr (BF) {
      const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(u[i] << 16); f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u); }
    } else {
      const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(u[i]);
    }
  }
  template <int N>
  __device__ void terms(bool in, lr_bf16x8 (&t)[N]) const {
    if constexpr (BF) {
      const uint4 w = in ? a : make_uint4(0, 0, 0, 0);
      t[0] = *(const lr_bf16x8*)&w;
    } else {
      float f[8];
      values(f);
      if (!in)
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = 0.f;
      lr_terms<N>(f, t);
    }
  }
};

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

// A workgroup's part of u for one adapter: MB blocks of 16 rows, CB of 16 columns. A wave takes 64 of K at a time, every load of them on
// its way before the first product; the waves' sums meet in LDS, in order.
template <bool XB, bool WB, int XT, int WT, int CB, int MB>
__device__ __forceinline__ void shrink_rows(const LoraArgs& a, int64_t t0, uint64_t rows, int n, int adapter, int split, int c0, float* sums) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int cols = min(16 * CB, a.C - c0);
  const int k0 = split * a.kstep, k1 = (int)min((int64_t)k0 + a.kstep, a.K);
  lr_floatx4 acc[MB][CB];
  int64_t xat[MB], wat[CB];
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    xat[i] = (t0 + lr_nth(rows, min(16 * i + r, n - 1))) * a.ldx;
#pragma unroll
    for (int j = 0; j < CB; ++j) acc[i][j] = lr_floatx4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int j = 0; j < CB; ++j) wat[j] = ((int64_t)adapter * a.C + c0 + min(16 * j + r, cols - 1)) * a.K;
  const int kw = (a.kstep / 64 + LR_WAVES - 1) / LR_WAVES * 64, kb = k0 + kw * wave, ke = min(kb + kw, k1);  // the wave's
  if constexpr (XB && WB && MB > 1) {
    // many rows: 8 lanes in a row fetch 128 bytes in a row of x or A, the next 64 of K while these go through LDS to the operands' layout,
    // 16 bytes u of a row at u ^ (row / 2) % 8: 4096 rows of 4096 by 64 columns 24.5 -> 21.6 us
    uint16_t* tile = (uint16_t*)sums + wave * (16 * (MB + CB) * 64);
    const int part = lane & 7;
    int64_t at[2 * MB + 2 * CB];
#pragma unroll
    for (int i = 0; i < 2 * MB; ++i) at[i] = (t0 + lr_nth(rows, min(8 * i + (lane >> 3), n - 1))) * a.ldx;
#pragma unroll
    for (int j = 0; j < 2 * CB; ++j) at[2 * MB + j] = ((int64_t)adapter * a.C + c0 + min(8 * j + (lane >> 3), cols - 1)) * a.K;
    uint4 v[2 * MB + 2 * CB];
    auto load = [&](int k) {
      const bool in = k + 8 * part < ke;
      const int from = in ? k + 8 * part : 0;
#pragma unroll
      for (int i = 0; i < 2 * (MB + CB); ++i) {
        v[i] = *(const uint4*)((const uint16_t*)(i < 2 * MB ? a.x : a.a) + at[i] + from);
        if (!in) v[i] = make_uint4(0, 0, 0, 0);
      }
    };
    if (kb < ke) load(kb);
    for (int k = kb; k < ke; k += 64) {
      wave_lds_order();  // (the last tile is read)
#pragma unroll
      for (int i = 0; i < 2 * (MB + CB); ++i) {
        const int row = 8 * i + (lane >> 3);
        *(uint4*)(tile + row * 64 + 8 * (part ^ (row >> 1 & 7))) = v[i];
      }
      if (k + 64 < ke) load(k + 64);
      wave_lds_order();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        auto operand = [&](int block) { return *(const lr_bf16x8*)(tile + (16 * block + r) * 64 + 8 * ((4 * h + g) ^ (r >> 1 & 7))); };
        lr_bf16x8 xf[MB];
#pragma unroll
        for (int i = 0; i < MB; ++i) xf[i] = operand(i);
#pragma unroll
        for (int j = 0; j < CB; ++j) {
          const lr_bf16x8 wf = operand(MB + j);
#pragma unroll
          for (int i = 0; i < MB; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[i], wf, acc[i][j], 0, 0, 0);
        }
      }
    }
    __syncthreads();  // (the tiles' place is the sums')
  } else
  for (int k = kb; k < ke; k += 64) {
    LrRaw<XB> x[2][MB];
    LrRaw<WB> w[2][CB];
    bool in[2];
    int at[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int kk = k + 32 * h + 8 * g;
      in[h] = kk < ke;
      at[h] = in[h] ? kk : 0;
    }
    // (a line's halves one after the other: far apart, each would be fetched anew)
#pragma unroll
    for (int j = 0; j < CB; ++j) { w[0][j].load(a.a, wat[j] + at[0]); w[1][j].load(a.a, wat[j] + at[1]); }
#pragma unroll
    for (int i = 0; i < MB; ++i) { x[0][i].load(a.x, xat[i] + at[0]); x[1][i].load(a.x, xat[i] + at[1]); }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      lr_bf16x8 xf[MB][XT];
#pragma unroll
      for (int i = 0; i < MB; ++i) x[h][i].template terms<XT>(in[h], xf[i]);
#pragma unroll
      for (int j = 0; j < CB; ++j) {
        lr_bf16x8 wf[WT];
        w[h][j].template terms<WT>(in[h], wf);
#pragma unroll
        for (int i = 0; i < MB; ++i) acc[i][j] = lr_mfma<XT, WT>(xf[i], wf, acc[i][j]);
      }
    }
  }
  // lane (r, g) holds rows 16 i + 4 g .. + 3 of column 16 j + r; a wave adds up every fourth block
  constexpr int BLOCKS = MB * CB;
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < CB; ++j) *(lr_floatx4*)(sums + ((wave * BLOCKS + i * CB + j) * 64 + lane) * 4) = acc[i][j];
  __syncthreads();
  for (int b = wave; b < BLOCKS; b += LR_WAVES) {
    const int i = b / CB, j = b % CB;
    lr_floatx4 v[LR_WAVES];
#pragma unroll
    for (int w = 0; w < LR_WAVES; ++w) v[w] = *(const lr_floatx4*)(sums + ((w * BLOCKS + b) * 64 + lane) * 4);
    const lr_floatx4 t = v[0] + v[1] + v[2] + v[3];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int m = 16 * i + 4 * g + e;
      if (m < n && 16 * j + r < cols) a.u[((int64_t)split * a.rows + t0 + lr_nth(rows, m)) * a.C + c0 + 16 * j + r] = t[e];
    }
  }
  __syncthreads();  // (sums are read)
}

// u[part][row][c] = the part of K's products of x's row and A's row c
template <bool XB, bool WB, int XT, int WT, int CB>
__global__ __launch_bounds__(64 * LR_WAVES) void lora_shrink(LoraArgs a) {
  __shared__ __attribute__((aligned(16))) float sums[LR_WAVES * (XB && WB && CB < 4 ? 512 * (4 + CB) : 4 * CB * 256)];  // (the waves' sums, or their tiles)
  const int split = blockIdx.x % a.splits, c0 = blockIdx.x / a.splits * 16 * CB;
  LoraTile tile(a, blockIdx.z);
  int adapter;
  uint64_t rows;
  while (tile.next(a.share, blockIdx.y, adapter, rows)) {
    if (adapter < 0) continue;
    const int n = __builtin_popcountll(rows);
    if (n <= 16) shrink_rows<XB, WB, XT, WT, CB, 1>(a, tile.t0, rows, n, adapter, split, c0, sums);
    else if (n <= 32) shrink_rows<XB, WB, XT, WT, CB, 2>(a, tile.t0, rows, n, adapter, split, c0, sums);
    else shrink_rows<XB, WB, XT, WT, CB, 4>(a, tile.t0, rows, n, adapter, split, c0, sums);
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

// u of an adapter's rows in LDS as terms: 8 of a row's at a time, the parts of K in order, 8 of them on their way
template <int UT>
__device__ __forceinline__ void expand_u(const LoraArgs& a, int64_t t0, uint64_t rows, int n, int adapter, int part, uint16_t* us, int ldu) {
  const int steps = (a.rank + 31) / 32;
  const float sc = a.scale ? a.scale[adapter] : 1.f;
  for (int i = threadIdx.x; i < n * 4 * steps; i += 64 * LR_WAVES) {
    const int m = i / (4 * steps), k = i % (4 * steps) * 8;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (k < a.rank) {
      const float* p = a.u + (t0 + lr_nth(rows, m)) * a.C + part * a.rank + k;
      for (int s = 0; s < a.splits; s += 8) {
        LrRaw<false> v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e].load(p, min(s + e, a.splits - 1) * a.rows * a.C);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float w[8];
          v[e].values(w);
          if (s + e < a.splits)
#pragma unroll
            for (int d = 0; d < 8; ++d) f[d] += w[d];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= sc;
    }
    lr_bf16x8 t[UT];
    lr_terms<UT>(f, t);
#pragma unroll
    for (int e = 0; e < UT; ++e) *(lr_bf16x8*)(us + (e * LR_ROWS + m) * ldu + k) = t[e];
  }
}

// One adapter's rows, the chunk's columns n0 .. n1: y = residual + u B^T, MB blocks of 16 rows at a time. B's rows are the product's rows and
// x's its columns: two blocks of 16 of B's rows are rows 8 (r / 4) + r % 4 and those 4 on, so that a lane ends with 8 consecutive columns
// of x's row r. They go through LDS (`tile`, the wave's own) to where 8 lanes in a row hold 128 bytes in a row of y: as the products leave them,
// each lane's 16 bytes in a row of their own, 4096 rows of 28672 take 123 us rather than 113.
template <bool YB, int MB>
struct LrTile {
  static constexpr int COLS = YB ? 64 : 32, LD = COLS + 4, SIZE = 16 * MB * LD;  // floats
};
template <bool WB, bool YB, int UT, int WT, int MB>
__device__ __forceinline__ void expand_rows(const LoraArgs& a, int64_t t0, uint64_t rows, int n, int adapter, int n0, int n1, const uint16_t* us, int ldu, float* tile) {
  using Tile = LrTile<YB, MB>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int steps = (a.rank + 31) / 32;
  constexpr int CG = Tile::COLS / 32, V = YB ? 8 : 4, IT = 2 * MB;  // a lane's columns of 16 bytes; rounds of 8 rows
  const int64_t wbase = (int64_t)adapter * a.N * a.rank;
  for (int m0 = 0; m0 < n; m0 += 16 * MB) {
    int64_t row[IT];  // the rows whose 16 bytes the lane moves
#pragma unroll
    for (int i = 0; i < IT; ++i) row[i] = t0 + lr_nth(rows, min(m0 + 8 * i + (lane >> 3), n - 1));
    for (int c = n0 + Tile::COLS * wave; c < n1; c += Tile::COLS * LR_WAVES) {
      const int col = c + V * (lane & 7);
      uint4 res[IT];
      if (a.residual)
#pragma unroll
        for (int i = 0; i < IT; ++i) res[i] = *(const uint4*)((const char*)a.residual + (row[i] * a.ldr + min(col, n1 - V)) * (YB ? 2 : 4));
      lr_floatx4 acc[MB][CG][2];
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int q = 0; q < CG; ++q) acc[i][q][0] = acc[i][q][1] = lr_floatx4{0.f, 0.f, 0.f, 0.f};
      for (int s = 0; s < steps; ++s) {
        const int k = 32 * s + 8 * g;
        LrRaw<WB> b[CG][2];
#pragma unroll
        for (int q = 0; q < CG; ++q)
#pragma unroll
          for (int e = 0; e < 2; ++e) b[q][e].load(a.b, wbase + (int64_t)min(c + 32 * q + 8 * (r >> 2) + 4 * e + (r & 3), n1 - 1) * a.rank + (k < a.rank ? k : 0));
        lr_bf16x8 uf[MB][UT];
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int e = 0; e < UT; ++e) uf[i][e] = *(const lr_bf16x8*)(us + (e * LR_ROWS + min(m0 + 16 * i + r, n - 1)) * ldu + k);
#pragma unroll
        for (int q = 0; q < CG; ++q)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            lr_bf16x8 bf[WT];
            b[q][e].template terms<WT>(k < a.rank, bf);
#pragma unroll
            for (int i = 0; i < MB; ++i) acc[i][q][e] = lr_mfma<WT, UT>(bf, uf[i], acc[i][q][e]);
          }
      }
      wave_lds_order();  // (the last columns are read)
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int q = 0; q < CG; ++q)
#pragma unroll
          for (int e = 0; e < 2; ++e) *(lr_floatx4*)(tile + (16 * i + r) * Tile::LD + 32 * q + 8 * g + 4 * e) = acc[i][q][e];
      wave_lds_order();
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const float* from = tile + (8 * i + (lane >> 3)) * Tile::LD + V * (lane & 7);
        if (m0 + 8 * i + (lane >> 3) >= n || col >= n1) continue;
        uint32_t w[4] = {res[i].x, res[i].y, res[i].z, res[i].w};
        if (!a.residual) w[0] = w[1] = w[2] = w[3] = 0;
        const lr_floatx4 f = *(const lr_floatx4*)from;
        if constexpr (YB) {
          const lr_floatx4 h = *(const lr_floatx4*)(from + 4);
          const float v[8] = {f[0], f[1], f[2], f[3], h[0], h[1], h[2], h[3]};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = bf16_rne_f(__uint_as_float(w[e] << 16) + v[2 * e]) | (bf16_rne_f(__uint_as_float(w[e] & 0xFFFF0000u) + v[2 * e + 1]) << 16);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) + f[e]);
        }
        *(uint4*)((char*)a.y + (row[i] * a.ldy + col) * (YB ? 2 : 4)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

// y = residual + scale u B^T: a workgroup a chunk of a part's columns
template <bool WB, bool YB, int UT, int WT>
__global__ __launch_bounds__(64 * LR_WAVES, WB ? 4 : 3) void lora_expand(LoraArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint16_t us[];  // [UT][64][ldu] u's terms
  __shared__ __attribute__((aligned(16))) float turn[LR_WAVES * LrTile<YB, 2>::SIZE];
  int part = 0;
  while (part + 1 < a.parts && (int)blockIdx.x >= a.chunk0[part + 1]) ++part;
  const int n0 = a.col0[part] + (blockIdx.x - a.chunk0[part]) * a.width, n1 = min(n0 + a.width, a.col0[part + 1]);
  const int ldu = 32 * ((a.rank + 31) / 32) + 8;
  LoraTile tile(a, blockIdx.z);
  int adapter;
  uint64_t rows;
  bool again = false;
  while (tile.next(a.share, blockIdx.y, adapter, rows)) {
    const int n = __builtin_popcountll(rows);
    if (adapter < 0) {  // the residual, or zeros
      if (a.residual == a.y) continue;
      const int pieces = (n1 - n0) / 8;
      for (int i = threadIdx.x; i < n * pieces; i += 64 * LR_WAVES) {
        const int64_t t = tile.t0 + lr_nth(rows, i / pieces), c = n0 + i % pieces * 8;
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (a.residual) {
          LrRaw<YB> x;
          x.load(a.residual, t * a.ldr + c);
          x.values(f);
        }
        lr_write8<YB>(a.y, t * a.ldy + c, f);
      }
      continue;
    }
    if (again) __syncthreads();  // (the last adapter's u is read)
    again = true;
    expand_u<UT>(a, tile.t0, rows, n, adapter, part, us, ldu);
    __syncthreads();
    float* mine = turn + (threadIdx.x >> 6) * LrTile<YB, 2>::SIZE;
    if (n <= 16) expand_rows<WB, YB, UT, WT, 1>(a, tile.t0, rows, n, adapter, n0, n1, us, ldu, mine);
    else expand_rows<WB, YB, UT, WT, 2>(a, tile.t0, rows, n, adapter, n0, n1, us, ldu, mine);
  }
}

// A decode step's few rows in one launch: a workgroup of 16 waves adds up u for its adapter's part itself, though the others of the
// part's columns do the same, and goes on to its columns. Worth it while the part's rows of A (LR_FEW_BYTES at most) take a workgroup less than
// the second launch. The first columns' residual and B are on their way meanwhile; 16 rows at a time.
constexpr int LR_FEW_WAVES = 16;
template <bool XB, bool WB, bool YB, int XT, int WT, int UT, int CB>
__global__ __launch_bounds__(64 * LR_FEW_WAVES) void lora_few(LoraArgs a) {
  constexpr int H = XB && WB && CB <= 2 ? 4 : 2, STEP = 32 * LR_FEW_WAVES;  // loads of 32 of K together; columns a round
  __shared__ __attribute__((aligned(16))) float sums[LR_FEW_WAVES * CB * 256];
  __shared__ __attribute__((aligned(16))) uint16_t us[UT * 16 * (16 * CB + 32 + 8)];  // u's terms, whole steps of 32 columns
  int part = 0;
  while (part + 1 < a.parts && (int)blockIdx.x >= a.chunk0[part + 1]) ++part;
  const int n0 = a.col0[part] + (blockIdx.x - a.chunk0[part]) * a.width, n1 = min(n0 + a.width, a.col0[part + 1]);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int steps = (a.rank + 31) / 32, ldu = 32 * steps + 8;
  const int kw = (int)((a.K + 64 * LR_FEW_WAVES - 1) / (64 * LR_FEW_WAVES)) * 64, kb = kw * wave, ke = (int)min((int64_t)kb + kw, a.K);
  LoraTile tile(a, blockIdx.z);
  int adapter;
  uint64_t rows;
  while (tile.next(a.share, blockIdx.y, adapter, rows)) {
    const int n = __builtin_popcountll(rows);
    if (adapter < 0) {  // the residual, or zeros
      if (a.residual == a.y) continue;
      const int pieces = (n1 - n0) / 8;
      for (int i = threadIdx.x; i < n * pieces; i += 64 * LR_FEW_WAVES) {
        const int64_t t = tile.t0 + lr_nth(rows, i / pieces), c = n0 + i % pieces * 8;
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (a.residual) {
          LrRaw<YB> x;
          x.load(a.residual, t * a.ldr + c);
          x.values(f);
        }
        lr_write8<YB>(a.y, t * a.ldy + c, f);
      }
      continue;
    }
    const float sc = a.scale ? a.scale[adapter] : 1.f;
    const int64_t abase = ((int64_t)adapter * a.C + part * a.rank) * a.K, bbase = (int64_t)adapter * a.N * a.rank;
    for (int m0 = 0; m0 < n; m0 += 16) {
      const int64_t row = tile.t0 + lr_nth(rows, min(m0 + r, n - 1));
      LrRaw<YB> res;
      LrRaw<WB> b[2];
      auto load_b = [&](int c, int k) {
#pragma unroll
        for (int e = 0; e < 2; ++e) b[e].load(a.b, bbase + (int64_t)min(c + 8 * (r >> 2) + 4 * e + (r & 3), n1 - 1) * a.rank + (k < a.rank ? k : 0));
      };
      auto load = [&](int c) {
        if (a.residual) res.load(a.residual, row * a.ldr + min(c + 8 * g, n1 - 8));
        load_b(c, 8 * g);
      };
      int c = n0 + 32 * wave;
      load(c);  // (a chunk's last waves may have no columns: the last ones')
      lr_floatx4 acc[CB];
#pragma unroll
      for (int j = 0; j < CB; ++j) acc[j] = lr_floatx4{0.f, 0.f, 0.f, 0.f};
      const int64_t xat = row * a.ldx;
      for (int k = kb; k < ke; k += 32 * H) {
        LrRaw<XB> x[H];
        LrRaw<WB> w[H][CB];
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const int at = k + 32 * h + 8 * g < ke ? k + 32 * h + 8 * g : 0;
          x[h].load(a.x, xat + at);
#pragma unroll
          for (int j = 0; j < CB; ++j) w[h][j].load(a.a, abase + (int64_t)min(16 * j + r, a.rank - 1) * a.K + at);
        }
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const bool in = k + 32 * h + 8 * g < ke;
          lr_bf16x8 xf[XT];
          x[h].template terms<XT>(in, xf);
#pragma unroll
          for (int j = 0; j < CB; ++j) {
            lr_bf16x8 wf[WT];
            w[h][j].template terms<WT>(in, wf);
            acc[j] = lr_mfma<XT, WT>(xf, wf, acc[j]);
          }
        }
      }
      // the waves' sums, in order; lane (r, g) holds rows 4 g .. + 3 of column 16 j + r
#pragma unroll
      for (int j = 0; j < CB; ++j) *(lr_floatx4*)(sums + ((wave * CB + j) * 64 + lane) * 4) = acc[j];
      __syncthreads();  // (and the last rows' u is read)
      for (int i = threadIdx.x; i < 16 * 32 * steps; i += 64 * LR_FEW_WAVES) {
        const int m = i / (32 * steps), k = i % (32 * steps);
        float v = 0.f;
        if (k < a.rank) {
          const float* p = sums + ((k >> 4) * 64 + (m >> 2) * 16 + (k & 15)) * 4 + (m & 3);
#pragma unroll
          for (int w = 0; w < LR_FEW_WAVES; ++w) v += p[w * CB * 256];
          v *= sc;
        }
#pragma unroll
        for (int e = 0; e < UT; ++e) {
          const __bf16 t = (__bf16)v;
          us[(e * 16 + m) * ldu + k] = *(const uint16_t*)&t;
          v -= (float)t;
        }
      }
      __syncthreads();
      for (; c < n1; c += STEP) {
        lr_floatx4 o[2] = {lr_floatx4{0.f, 0.f, 0.f, 0.f}, lr_floatx4{0.f, 0.f, 0.f, 0.f}};
        for (int s = 0; s < steps; ++s) {
          const int k = 32 * s + 8 * g;
          if (s) load_b(c, k);
          lr_bf16x8 uf[UT];
#pragma unroll
          for (int e = 0; e < UT; ++e) uf[e] = *(const lr_bf16x8*)(us + (e * 16 + r) * ldu + k);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            lr_bf16x8 bf[WT];
            b[e].template terms<WT>(k < a.rank, bf);
            o[e] = lr_mfma<WT, UT>(bf, uf, o[e]);
          }
        }
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (a.residual) res.values(f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += o[e >> 2][e & 3];
        if (c + STEP < n1) load(c + STEP);
        if (m0 + r < n && c + 8 * g < n1) lr_write8<YB>(a.y, row * a.ldy + c + 8 * g, f);
      }
    }
  }
}

// Parts of K: whole steps of 256 (a wave's 64 each), as many as keep the parts' rows within 16384, so that u's parts stay a
// small share of what a call moves and a decode step's few rows still fill the GPU.
constexpr int LR_MAX_SPLITS = 32;
constexpr int64_t LR_SPLIT_ROWS = 16384;  // (32768: 4096 rows 136 -> 146 us)
static int lora_splits(int64_t rows, int64_t K) {
  const int64_t most = std::min<int64_t>(LR_MAX_SPLITS, (K + 255) / 256);
  return (int)std::max<int64_t>(1, std::min(most, LR_SPLIT_ROWS / rows));
}

// One launch where a part's rows of A are at most LR_FEW_BYTES, those of all adapters that the rows may have LR_FEW_ALL, and the rank 32, 16 of
// fp32 weights (more do not fit the registers of 16 waves): smollm's q, k and v of 1 row 8.0 -> 5.1 us; of 16 rows with 8 adapters
// of rank 32 9.7 -> 8.2, of rank 64 10.5 against 9.7 but 10.2 -> 11.9 at K of 1024, in fp32 of rank 16 11.7 -> 8.8, of rank 32 12.2 against 13.1;
// an 8B o of 4 rows with as many adapters 9.1 either way, its q, k and v of 32 with 24 12.5 against 15.2.
constexpr int64_t LR_FEW_BYTES = 160 << 10, LR_FEW_ALL = 1 << 20;
static bool lora_is_few(int64_t rows, int64_t K, int rank, int adapters, int w_dtype) {
  const int64_t bytes = rank * K * (w_dtype == FH_F32 ? 4 : 2);
  return rows <= LR_ROWS && rank <= (w_dtype == FH_F32 ? 16 : 32) && bytes <= LR_FEW_BYTES && bytes * std::min<int64_t>(rows, adapters) <= LR_FEW_ALL;
}

template <bool XB, bool WB, bool YB>
static void launch_lora(bool few, hipStream_t s, const LoraArgs& a) {
  constexpr int T = YB ? 2 : 3, XT = XB ? 1 : T, WT = WB ? 1 : T;
  if (few) {
    const dim3 g(a.chunk0[a.parts], a.share, 1), b(64 * LR_FEW_WAVES);
    if (!WB || a.rank <= 16) hipLaunchKernelGGL((lora_few<XB, WB, YB, XT, WT, T, 1>), g, b, 0, s, a);
    else if constexpr (WB) hipLaunchKernelGGL((lora_few<XB, WB, YB, XT, WT, T, 2>), g, b, 0, s, a);
    return;
  }
  // u's columns in equal groups of up to 4 blocks of 16
  const unsigned tiles = (unsigned)((a.rows + LR_ROWS - 1) / LR_ROWS), blocks = (a.C + 15) / 16, groups = (blocks + 3) / 4, cb = (blocks + groups - 1) / groups;
  const dim3 g(a.splits * groups, a.share, tiles), b(64 * LR_WAVES);
  switch (cb) {
    case 1: hipLaunchKernelGGL((lora_shrink<XB, WB, XT, WT, 1>), g, b, 0, s, a); break;
    case 2: hipLaunchKernelGGL((lora_shrink<XB, WB, XT, WT, 2>), g, b, 0, s, a); break;
    case 3: hipLaunchKernelGGL((lora_shrink<XB, WB, XT, WT, 3>), g, b, 0, s, a); break;
    default: hipLaunchKernelGGL((lora_shrink<XB, WB, XT, WT, 4>), g, b, 0, s, a); break;
  }
  const int ldu = 32 * ((a.rank + 31) / 32) + 8;
  hipLaunchKernelGGL((lora_expand<WB, YB, T, WT>), dim3(a.chunk0[a.parts], a.share, tiles), dim3(64 * LR_WAVES), (size_t)T * LR_ROWS * ldu * 2, s, a);
}

// silu(gate) up for rows whose gate and up are final only behind fh_lora (FH_EP_SILU_GATE does it in the product): a lane 8 columns, which
// two loads and a store of 16 bytes each bound. 16 rows of 14336 out of fp32 into bf16 4-5 us (as a program of fh_map, decoded an element, 15),
// 4096 rows 107 for 587 MB, 5.5 TB/s.
template <bool XB, bool YB>
__global__ __launch_bounds__(256) void silu_gate_kernel(const void* x, int64_t ldx, int64_t rows, int64_t split, void* y, int64_t ldy) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, pieces = split / 8;
  if (i >= rows * pieces) return;
  const int64_t t = i / pieces, c = i % pieces * 8;
  LrRaw<XB> g, u;
  g.load(x, t * ldx + c);
  u.load(x, t * ldx + split + c);
  float a[8], b[8];
  g.values(a);
  u.values(b);
#pragma unroll
  for (int e = 0; e < 8; ++e) a[e] = a[e] / (1.f + expf(-a[e])) * b[e];
  lr_write8<YB>(y, t * ldy + c, a);
}

}  // namespace fh

using namespace fh;

extern "C" int fh_silu_gate_rows(const void* x, int x_dtype, int64_t ldx, int64_t rows, int64_t split, void* y, int y_dtype, int64_t ldy,
                                 void* stream) {
  auto no = [](int code, const char* what) { set_error("fh_silu_gate_rows: %s", what); return code; };
  if (!x || !y) return no(FH_EINVAL, "null pointer");
  if (rows < 1 || split < 1) return no(FH_EINVAL, "need rows and split of at least 1");
  if (x_dtype != FH_F32 && x_dtype != FH_BF16) return no(FH_EINVAL, "x is FH_F32 or FH_BF16");
  if (y_dtype != FH_F32 && y_dtype != FH_BF16) return no(FH_EINVAL, "y is FH_F32 or FH_BF16");
  if (split % 8 || split >= (1LL << 30)) return no(FH_EUNSUP, "split a multiple of 8, below 2^30");
  if (ldx < 2 * split || ldy < split || ldx % (x_dtype == FH_F32 ? 4 : 8) || ldy % (y_dtype == FH_F32 ? 4 : 8) || (((uintptr_t)x | (uintptr_t)y) & 15))
    return no(FH_EINVAL, "rows at least 2 split and split, 16-byte aligned");
  if (rows >= (1LL << 32) / (split / 8 + 1)) return no(FH_EUNSUP, "too many rows for one grid");
  const dim3 g((unsigned)((rows * (split / 8) + 255) / 256)), b(256);
  const hipStream_t s = as_stream(stream);
  if (x_dtype == FH_BF16) {
    if (y_dtype == FH_BF16) hipLaunchKernelGGL((silu_gate_kernel<true, true>), g, b, 0, s, x, ldx, rows, split, y, ldy);
    else hipLaunchKernelGGL((silu_gate_kernel<true, false>), g, b, 0, s, x, ldx, rows, split, y, ldy);
  } else {
    if (y_dtype == FH_BF16) hipLaunchKernelGGL((silu_gate_kernel<false, true>), g, b, 0, s, x, ldx, rows, split, y, ldy);
    else hipLaunchKernelGGL((silu_gate_kernel<false, false>), g, b, 0, s, x, ldx, rows, split, y, ldy);
  }
  return check_launch("fh_silu_gate_rows");
}

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
  const bool few = lora_is_few(rows, K, rank, adapters, w_dtype);
  l.splits = lora_splits(rows, K);
  const size_t need = (size_t)l.splits * rows * rank * parts * sizeof(float);
  if (!workspace || ws_bytes < need || ((uintptr_t)workspace & 15)) return no(FH_EINVAL, "a 16-byte aligned workspace of fh_lora_workspace_bytes");
  if (x == y) return no(FH_EINVAL, "y is not x (a row's x is read until its last column is done)");
  l.x = x; l.ldx = ldx; l.rows = rows; l.K = K; l.a = a_w; l.b = b_w; l.scale = scale; l.ids = ids;
  l.adapters = adapters; l.rank = rank; l.parts = parts; l.C = rank * parts; l.N = (int)N;
  l.kstep = (int)((K + 64 * l.splits - 1) / (64 * l.splits)) * 64;
  l.u = (float*)workspace; l.residual = residual; l.ldr = residual ? ldr : ldy; l.y = y; l.ldy = ldy;
  const int64_t tiles = (rows + LR_ROWS - 1) / LR_ROWS;
  l.share = (int)(tiles > 16 ? 1 : std::min<int64_t>(std::min<int64_t>(adapters + 1LL, rows), LR_ROWS));
  l.width = few ? LR_FEW_WIDTH : LR_WIDTH;
  int chunks = 0;
  for (int p = 0; p < parts; ++p) { l.chunk0[p] = chunks; chunks += (int)((part_cols[p] + l.width - 1) / l.width); }
  l.chunk0[parts] = chunks;
  const hipStream_t s = as_stream(stream);
  const int form = (x_dtype == FH_BF16) * 4 + (w_dtype == FH_BF16) * 2 + (y_dtype == FH_BF16);
  switch (form) {
    case 0: launch_lora<false, false, false>(few, s, l); break;
    case 1: launch_lora<false, false, true>(few, s, l); break;
    case 2: launch_lora<false, true, false>(few, s, l); break;
    case 3: launch_lora<false, true, true>(few, s, l); break;
    case 4: launch_lora<true, false, false>(few, s, l); break;
    case 5: launch_lora<true, false, true>(few, s, l); break;
    case 6: launch_lora<true, true, false>(few, s, l); break;
    default: launch_lora<true, true, true>(few, s, l); break;
  }
  return check_launch("fh_lora");
}
