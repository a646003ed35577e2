// Orthogonalisation of matrices by Newton-Schulz products, and the Muon update built on it.  For every matrix G of a list,
// taken with its shorter side as rows (m x n, m <= n; the transpose otherwise):
//   X_0 = G / max(|G|_F, eps);   A = X X^T,  B = a I + b A + c A^2,  X <- B X   for each step's (a, b, c),
// which pushes the singular values of X towards one and leaves its singular vectors alone.
//
// Bound by matrix products: a step costs m^2 n (A is symmetric: one triangle) + m^3 (so is A^2) + 2 m^2 n operations on
// 4 m n bytes.  The matrix cores have no fast float32 form, and 16-bit operands alone lose small singular values (errors
// grow up to a^steps times).  So every operand is kept as two float16 numbers, x s = hi + lo with a power of two s: hi
// carries 11 bits, lo the next 11, together 32 bits per number with a relative rounding of 2^-23, a half step of
// float32 and one bit more.  A product is hi hi + hi lo + lo hi on v_mfma_f32_16x16x32_f16 with float32 sums; lo lo is
// below 2^-22 of it.  The scales s come from bounds on the spectral norms (host, ortho_scales), so hi never overflows.
//
// Layout: a matrix with rows of K numbers is stored as rows of 32-number blocks [hi x 32 | lo x 32]: one block is one
// 128-byte line, a k-step of 32 is 8 rows x 128 bytes per LDS-DMA instruction, and both halves of a fragment come from
// the same line.  Every product here is D[p][q] = sum_k P[p][k] Q[q][k], both operands contiguous along k:
//   A = X X^T from X;   A^2 from A (symmetric);   (B X)^T = X^T B from Y = X^T and B (symmetric),
// so X and its transpose Y are both kept, and the epilogues store a tile twice, once through a transposing read of LDS.
//
// All matrices of a list share each launch: a workgroup finds its matrix and tile from its index.
#include "common.h"
#include <math.h>

namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

constexpr int MAXM = SNWS_ORTHO_MAX;
constexpr int NORM_CHUNK = 16384;    // elements per partial sum of squares

struct Mat {
  const void* x;       // (rows, cols), row stride ldx: the matrix, or the gradient of a Muon item
  void* out;           // (rows, cols), row stride ldo: the result, or the parameter of a Muon item
  float* mom;          // momentum of a Muon item
  int64_t ldx, ldo;
  int64_t X, Y, A;     // byte offsets into the workspace; the second Y lies behind the first, B behind A
  int64_t part;        // split-K partial tiles of A
  int m, n;            // m <= n
  int flip;            // rows > cols: X is the transpose
  int ks, kc;          // splits of the contraction over n and 32-blocks in each
  int norm0, normc;    // partial sums of squares
  float step;          // learning rate of a Muon item
};

struct Mats {
  Mat mat[MAXM];
  int end[MAXM];       // first workgroup index behind each matrix, for the launch at hand
  int count;
  unsigned char* ws;
};

struct MuonArgs {
  float momentum, grad_scale, decay;
  int nesterov;
};

__host__ __device__ __forceinline__ int up32(int v) { return (v + 31) & ~31; }

__device__ __forceinline__ void glds16(const void* gsrc, unsigned char* lds_wave_base) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)gsrc,
                                   (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}

// blocks dealt to the same XCD (bid % 8) get consecutive logical ids
__device__ __forceinline__ unsigned xcd_order(unsigned bid, unsigned nblk) {
  const unsigned q = nblk >> 3, r = nblk & 7, xcd = bid & 7;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (bid >> 3);
}

// matrix of workgroup id, and the id within it
__device__ __forceinline__ int find_mat(const Mats& a, int id, int& local) {
  const int lane = threadIdx.x & 63;
  const bool past = lane < a.count && id >= a.end[lane];
  const int i = __builtin_amdgcn_readfirstlane(__popcll(__ballot(past)));
  local = i ? id - a.end[i - 1] : id;
  return i;
}

__device__ __forceinline__ void split8(const float (&v)[8], uint4& hi, uint4& lo) {
  f16x8 h, l;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    h[e] = (_Float16)v[e];
    l[e] = (_Float16)(v[e] - (float)h[e]);
  }
  hi = __builtin_bit_cast(uint4, h);
  lo = __builtin_bit_cast(uint4, l);
}
// eight numbers of a row from column c (a multiple of 8), `row` its first byte
__device__ __forceinline__ void store8(unsigned char* row, int c, const float (&v)[8]) {
  uint4 hi, lo;
  split8(v, hi, lo);
  unsigned char* p = row + (c >> 5) * 128 + (c & 31) * 2;
  *reinterpret_cast<uint4*>(p) = hi;
  *reinterpret_cast<uint4*>(p + 64) = lo;
}
__device__ __forceinline__ void load8(const unsigned char* row, int c, float (&v)[8]) {
  const unsigned char* p = row + (c >> 5) * 128 + (c & 31) * 2;
  const f16x8 h = __builtin_bit_cast(f16x8, *reinterpret_cast<const uint4*>(p));
  const f16x8 l = __builtin_bit_cast(f16x8, *reinterpret_cast<const uint4*>(p + 64));
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)h[e] + (float)l[e];
}

// ------------------------------------------------------------------------------------------------ start
template <typename T>
__device__ __forceinline__ float elem(const T* p, int64_t i) { return (float)p[i]; }

// the matrix itself, or a Muon item's update direction from gradient and momentum (already advanced)
__device__ __forceinline__ float direction(float g, float m, const MuonArgs& u) {
  return u.nesterov ? (1.f - u.momentum) * g + u.momentum * m : m;
}

// Partial sums of squares in float64 (no overflow or underflow over float32's range, a fixed order); a Muon item's
// momentum is advanced on the way: m <- momentum m + (1 - momentum) grad_scale g.
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ortho_norm_kernel(Mats a, MuonArgs u, double* __restrict__ partial) {
  __shared__ double red[16];
  int chunk;
  const Mat& t = a.mat[find_mat(a, blockIdx.x, chunk)];
  const int rows = t.flip ? t.n : t.m, cols = t.flip ? t.m : t.n;
  const int64_t total = (int64_t)rows * cols, lo = (int64_t)chunk * NORM_CHUNK;
  const int64_t hi = lo + NORM_CHUNK < total ? lo + NORM_CHUNK : total;
  const T* x = static_cast<const T*>(t.x);
  double s = 0.0;
  const bool flat = t.ldx == cols;
  for (int64_t i = lo + threadIdx.x; i < hi; i += 256) {
    float v = elem(x, flat ? i : (i / cols) * t.ldx + i % cols);
    if (MUON) {
      v *= u.grad_scale;
      const float m = u.momentum * t.mom[i] + (1.f - u.momentum) * v;
      t.mom[i] = m;
      v = direction(v, m, u);
    }
    s += (double)v * (double)v;
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) partial[t.norm0 + chunk] = s;
}

// X_0 and its transpose from 64 x 64 tiles of the source, normalised
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ortho_start_kernel(Mats a, MuonArgs u, const double* __restrict__ partial, float eps,
                                                          float scale) {
  constexpr int LP = 66;
  __shared__ float tile[64 * LP];
  __shared__ double red[16];
  int local;
  const Mat& t = a.mat[find_mat(a, blockIdx.x, local)];
  const int rows = t.flip ? t.n : t.m, cols = t.flip ? t.m : t.n;
  const int tc = (cols + 63) >> 6, r0 = (local / tc) * 64, c0 = (local % tc) * 64;
  double s = 0.0;
  for (int i = threadIdx.x; i < t.normc; i += 256) s += partial[t.norm0 + i];
  const double norm = sqrt(block_sum(s, red));
  const float f = (float)((double)scale / (norm < (double)eps ? (double)eps : norm));      // a NaN stays one
  const T* x = static_cast<const T*>(t.x);
#pragma unroll 4
  for (int k = 0; k < 16; ++k) {
    const int r = k * 4 + (threadIdx.x >> 6), c = threadIdx.x & 63;
    float v = 0.f;
    if (r0 + r < rows && c0 + c < cols) {
      v = elem(x, (int64_t)(r0 + r) * t.ldx + c0 + c);
      if (MUON) v = direction(v * u.grad_scale, t.mom[(int64_t)(r0 + r) * cols + c0 + c], u);
      v *= f;
    }
    tile[r * LP + c] = v;
  }
  __syncthreads();
  unsigned char* direct = a.ws + (t.flip ? t.Y : t.X);      // rows x up32(cols)
  unsigned char* across = a.ws + (t.flip ? t.X : t.Y);      // cols x up32(rows)
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int id = k * 256 + threadIdx.x;
    float v[8];
    const int r = id >> 3, c = (id & 7) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[r * LP + c + e];
    if (r0 + r < rows && c0 + c < up32(cols)) store8(direct + (int64_t)(r0 + r) * up32(cols) * 4, c0 + c, v);
    const int q = (id >> 2 & 15) + (id >> 7) * 16, p = ((id & 3) + (id >> 6 & 1) * 4) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[(p + e) * LP + q];
    if (c0 + q < cols && r0 + p < up32(rows)) store8(across + (int64_t)(c0 + q) * up32(rows) * 4, r0 + p, v);
  }
}

// ------------------------------------------------------------------------------------------------ products
// A workgroup of 4 waves (2 x 2), each WT x WT of a T x T tile, T = 2 WT; k advances by 32 through two LDS stages.
template <int WT>
struct Tile {
  static constexpr int T = 2 * WT, MR = WT / 16, LP = T + 2;
  static constexpr int PIECES = 2 * T / 8, LOADS = PIECES / 4;          // 1 KB LDS-DMA pieces of a stage; per wave
  static constexpr int STAGE = 2 * T * 128;
  static constexpr int LDS = 2 * STAGE > T * LP * 4 ? 2 * STAGE : T * LP * 4;
};

// acc[mr][nr] += P rows p0.. x Q rows q0.. over the k-blocks [kb0, kb1); rows past the last are read as the last.
// Entered and left with the LDS free for anyone's use after a barrier.
template <int WT>
__device__ __forceinline__ void product(f32x4 (&acc)[WT / 16][WT / 16], const unsigned char* P, const unsigned char* Q, int p0,
                                        int q0, int M, int N, int KB, int kb0, int kb1, unsigned char* smem) {
  using G = Tile<WT>;
  constexpr int MR = G::MR;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  // LDS-DMA: piece w + 4 j holds rows 8 (w + 4 j) .. + 7; lane -> row lane >> 3, slot lane & 7, which receives the 16-byte
  // chunk slot ^ ((row >> 1) & 7), so that the 16 lanes of a fragment read hit distinct banks
  const int chunk = (lane & 7) ^ ((4 * (wave & 1) + (lane >> 4)) & 7);
  const unsigned char* src[G::LOADS];
#pragma unroll
  for (int j = 0; j < G::LOADS; ++j) {
    const int r = 8 * (wave + 4 * j) + (lane >> 3);
    const bool isq = j >= G::LOADS / 2;                    // the first half of the pieces is P, the second Q
    int row = isq ? q0 + r - G::T : p0 + r;
    const int last = (isq ? N : M) - 1;
    if (row > last) row = last;
    src[j] = (isq ? Q : P) + ((int64_t)row * KB + kb0) * 128 + chunk * 16;
  }
  auto stage = [&](int kb, int buf) {
#pragma unroll
    for (int j = 0; j < G::LOADS; ++j) glds16(src[j] + (int64_t)(kb - kb0) * 128, smem + buf * G::STAGE + (wave + 4 * j) * 1024);
  };
  int fro[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) fro[h] = (lane & 15) * 128 + (((h * 4 + (lane >> 4)) ^ ((lane >> 1) & 7)) * 16);
  stage(kb0, 0);
  int buf = 0;
  for (int kb = kb0; kb < kb1; ++kb) {
    if (kb + 1 < kb1) {
      stage(kb + 1, buf ^ 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(G::LOADS) : "memory");       // this stage landed, the next in flight
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    const unsigned char* pb = smem + buf * G::STAGE + wm * WT * 128;
    const unsigned char* qb = smem + buf * G::STAGE + (G::T + wn * WT) * 128;
    f16x8 ph[MR], pl[MR], qh[MR], ql[MR];
#pragma unroll
    for (int r = 0; r < MR; ++r) {
      ph[r] = *reinterpret_cast<const f16x8*>(pb + r * 2048 + fro[0]);
      qh[r] = *reinterpret_cast<const f16x8*>(qb + r * 2048 + fro[0]);
    }
#pragma unroll
    for (int r = 0; r < MR; ++r) {
      pl[r] = *reinterpret_cast<const f16x8*>(pb + r * 2048 + fro[1]);
      ql[r] = *reinterpret_cast<const f16x8*>(qb + r * 2048 + fro[1]);
    }
#pragma unroll
    for (int i = 0; i < MR; ++i)
#pragma unroll
      for (int j = 0; j < MR; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[i], qh[j], acc[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[i], ql[j], acc[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[i], qh[j], acc[i][j], 0, 0, 0);
      }
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();                          // every wave is done with this stage before it is refilled
    buf ^= 1;
  }
}

// the accumulators, times f, as a T x LP float tile in LDS; zeros outside M x N
template <int WT>
__device__ __forceinline__ void to_lds(const f32x4 (&acc)[WT / 16][WT / 16], float f, int p0, int q0, int M, int N, float* tile) {
  using G = Tile<WT>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int pr = (wave >> 1) * WT + 4 * (lane >> 4), qc = (wave & 1) * WT + (lane & 15);
#pragma unroll
  for (int i = 0; i < G::MR; ++i)
#pragma unroll
    for (int j = 0; j < G::MR; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int p = pr + i * 16 + r, q = qc + j * 16;
        tile[p * G::LP + q] = p0 + p < M && q0 + q < N ? acc[i][j][r] * f : 0.f;
      }
  __syncthreads();
}
// f(p, q, v): eight columns q .. q + 7 of row p, for every row and octet of the tile
template <int WT, typename F>
__device__ __forceinline__ void by_rows(const float* tile, F&& f) {
  using G = Tile<WT>;
  constexpr int C8 = G::T / 8;
#pragma unroll 2
  for (int id = threadIdx.x; id < G::T * C8; id += 256) {
    const int p = id / C8, q = (id % C8) * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[p * G::LP + q + e];
    f(p, q, v);
  }
}
// f(q, p, v): eight rows p .. p + 7 of column q.  Four lanes take the 32 rows of a block, sixteen the next columns: the
// reads of a wave spread over all banks (8 LP = 16 mod 32) and the stores of four lanes share a line.
template <int WT, typename F>
__device__ __forceinline__ void by_cols(const float* tile, F&& f) {
  using G = Tile<WT>;
  constexpr int B = G::T / 32;
#pragma unroll 2
  for (int id = threadIdx.x; id < G::T * G::T / 8; id += 256) {
    const int g = id >> 6, p = ((g % B) * 4 + (id & 3)) * 8, q = (g / B) * 16 + (id >> 2 & 15);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[(p + e) * G::LP + q];
    f(q, p, v);
  }
}

template <int WT>
__device__ __forceinline__ void clear(f32x4 (&acc)[WT / 16][WT / 16]) {
#pragma unroll
  for (int i = 0; i < WT / 16; ++i)
#pragma unroll
    for (int j = 0; j < WT / 16; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// tile number t of a lower triangle -> (i, j), j <= i
__device__ __forceinline__ void triangle(int t, int& i, int& j) {
  i = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
  while ((i + 1) * (i + 2) / 2 <= t) ++i;
  while (i * (i + 1) / 2 > t) --i;
  j = t - i * (i + 1) / 2;
}

// A = X X^T, one triangle of tiles, stored on both sides of the diagonal.  The contraction over n is split where the tiles
// alone would not fill the chip: partial tiles go to the workspace as they lie in the accumulators.
template <int WT>
__global__ __launch_bounds__(256, 2) void ortho_gram_kernel(Mats a, float f) {
  using G = Tile<WT>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  int local, i, j;
  const Mat& t = a.mat[find_mat(a, xcd_order(blockIdx.x, gridDim.x), local)];
  const int nt = (t.m + G::T - 1) / G::T, tiles = nt * (nt + 1) / 2;
  const int split = local / tiles, tl = local % tiles;      // tiles of one split are neighbours: they share its columns of X
  triangle(tl, i, j);
  const int KB = up32(t.n) >> 5, kb0 = split * t.kc, kb1 = kb0 + t.kc < KB ? kb0 + t.kc : KB;
  const unsigned char* X = a.ws + t.X;
  f32x4 acc[G::MR][G::MR];
  clear<WT>(acc);
  product<WT>(acc, X, X, i * G::T, j * G::T, t.m, t.m, KB, kb0, kb1, smem);
  if (t.ks > 1) {
    f32x4* part = reinterpret_cast<f32x4*>(a.ws + t.part) + (int64_t)(tl * t.ks + split) * (G::T * G::T / 4);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int r = 0; r < G::MR; ++r)
#pragma unroll
      for (int c = 0; c < G::MR; ++c) part[((wave * G::MR + r) * G::MR + c) * 64 + lane] = acc[r][c];
    return;
  }
  float* tile = reinterpret_cast<float*>(smem);
  to_lds<WT>(acc, f, i * G::T, j * G::T, t.m, t.m, tile);
  unsigned char* A = a.ws + t.A;
  const int mp = up32(t.m);
  by_rows<WT>(tile, [&](int p, int q, const float (&v)[8]) {
    if (i * G::T + p < t.m && j * G::T + q < mp) store8(A + (int64_t)(i * G::T + p) * mp * 4, j * G::T + q, v);
  });
  if (i != j)
    by_cols<WT>(tile, [&](int q, int p, const float (&v)[8]) {
      if (j * G::T + q < t.m && i * G::T + p < mp) store8(A + (int64_t)(j * G::T + q) * mp * 4, i * G::T + p, v);
    });
}

// adds the partial tiles of A, a workgroup per 32 x 32 block, in the order of the splits
template <int WT>
__global__ __launch_bounds__(256) void ortho_join_kernel(Mats a, float f) {
  using G = Tile<WT>;
  constexpr int B = G::T / 32;
  __shared__ float tile[32 * 34];
  int local, i, j;
  const Mat& t = a.mat[find_mat(a, blockIdx.x, local)];
  const int tl = local / (B * B), sub = local % (B * B);
  triangle(tl, i, j);
  const int p0 = i * G::T + (sub / B) * 32, q0 = j * G::T + (sub % B) * 32, mp = up32(t.m);
  if (p0 >= mp || q0 >= mp) return;
  // 16 x 16 accumulator blocks (r, c) of the tile's waves that make up this block
  const int r16 = (sub / B) * 2 + (threadIdx.x >> 7), c16 = (sub % B) * 2 + (threadIdx.x >> 6 & 1), lane = threadIdx.x & 63;
  const int wave = (r16 / G::MR) * 2 + c16 / G::MR;
  const f32x4* part = reinterpret_cast<const f32x4*>(a.ws + t.part) + (int64_t)tl * t.ks * (G::T * G::T / 4) +
                      ((wave * G::MR + r16 % G::MR) * G::MR + c16 % G::MR) * 64 + lane;
  f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int k = 0; k < t.ks; ++k) s += part[(int64_t)k * (G::T * G::T / 4)];
  const int pr = (r16 & 1) * 16 + 4 * (lane >> 4), qc = (c16 & 1) * 16 + (lane & 15);
#pragma unroll
  for (int e = 0; e < 4; ++e) tile[(pr + e) * 34 + qc] = p0 + pr + e < t.m && q0 + qc < t.m ? s[e] * f : 0.f;
  __syncthreads();
  unsigned char* A = a.ws + t.A;
  const int id = threadIdx.x & 127, r = id >> 2, c = (id & 3) * 8;
  float v[8];
  if (threadIdx.x < 128) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[r * 34 + c + e];
    if (p0 + r < t.m) store8(A + (int64_t)(p0 + r) * mp * 4, q0 + c, v);
  } else if (i != j) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[(c + e) * 34 + r];
    if (q0 + r < t.m) store8(A + (int64_t)(q0 + r) * mp * 4, p0 + c, v);
  }
}

// B = ca I + cb A + cc A^2 of the stored (scaled) numbers, one triangle of tiles; the host has folded the scales in
template <int WT>
__global__ __launch_bounds__(256, 2) void ortho_poly_kernel(Mats a, float ca, float cb, float cc) {
  using G = Tile<WT>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  int local, i, j;
  const Mat& t = a.mat[find_mat(a, xcd_order(blockIdx.x, gridDim.x), local)];
  triangle(local, i, j);
  const int mp = up32(t.m), KB = mp >> 5;
  const unsigned char* A = a.ws + t.A;
  unsigned char* Bm = a.ws + t.A + (int64_t)t.m * mp * 4;
  f32x4 acc[G::MR][G::MR];
  clear<WT>(acc);
  product<WT>(acc, A, A, i * G::T, j * G::T, t.m, t.m, KB, 0, KB, smem);
  float* tile = reinterpret_cast<float*>(smem);
  to_lds<WT>(acc, cc, i * G::T, j * G::T, t.m, t.m, tile);
  auto put = [&](int r, int c, const float (&v)[8]) {        // eight numbers of row r from column c on
    if (r >= t.m || c >= mp) return;
    float w[8];
    load8(A + (int64_t)r * mp * 4, c, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = v[e] + cb * w[e] + (r == c + e ? ca : 0.f);
    store8(Bm + (int64_t)r * mp * 4, c, w);
  };
  by_rows<WT>(tile, [&](int p, int q, const float (&v)[8]) { put(i * G::T + p, j * G::T + q, v); });
  if (i != j) by_cols<WT>(tile, [&](int q, int p, const float (&v)[8]) { put(j * G::T + q, i * G::T + p, v); });
}

// eight consecutive results at (r, c) of the source's orientation, as many as lie within `cols`
template <typename T, bool MUON>
__device__ __forceinline__ void finish8(const Mat& t, int r, int c, int cols, const float (&v)[8], const MuonArgs& u) {
  T* o = static_cast<T*>(t.out) + (int64_t)r * t.ldo + c;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (c + e < cols) {
      if (MUON) o[e] = (T)((float)o[e] * u.decay - t.step * v[e]);
      else o[e] = (T)v[e];
    }
}

// Y' = Y B (= (B X)^T): the next step's Y and X, or the result
template <int WT, typename T, bool LAST, bool MUON>
__global__ __launch_bounds__(256, 2) void ortho_apply_kernel(Mats a, MuonArgs u, float f, int odd) {
  using G = Tile<WT>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  int local;
  const Mat& t = a.mat[find_mat(a, xcd_order(blockIdx.x, gridDim.x), local)];
  const int mp = up32(t.m), np = up32(t.n), KB = mp >> 5;
  const int tq = (t.m + G::T - 1) / G::T, p0 = (local / tq) * G::T, q0 = (local % tq) * G::T;
  const int64_t ysz = (int64_t)t.n * mp * 4;
  const unsigned char* Yin = a.ws + t.Y + (odd ? ysz : 0);
  unsigned char* Yout = a.ws + t.Y + (odd ? 0 : ysz);
  const unsigned char* Bm = a.ws + t.A + (int64_t)t.m * mp * 4;
  f32x4 acc[G::MR][G::MR];
  clear<WT>(acc);
  product<WT>(acc, Yin, Bm, p0, q0, t.n, t.m, KB, 0, KB, smem);
  float* tile = reinterpret_cast<float*>(smem);
  to_lds<WT>(acc, f, p0, q0, t.n, t.m, tile);
  if (LAST) {
    if (t.flip)
      by_rows<WT>(tile, [&](int p, int q, const float (&v)[8]) {
        if (p0 + p < t.n && q0 + q < t.m) finish8<T, MUON>(t, p0 + p, q0 + q, t.m, v, u);
      });
    else
      by_cols<WT>(tile, [&](int q, int p, const float (&v)[8]) {
        if (q0 + q < t.m && p0 + p < t.n) finish8<T, MUON>(t, q0 + q, p0 + p, t.n, v, u);
      });
    return;
  }
  by_rows<WT>(tile, [&](int p, int q, const float (&v)[8]) {
    if (p0 + p < t.n && q0 + q < mp) store8(Yout + (int64_t)(p0 + p) * mp * 4, q0 + q, v);
  });
  unsigned char* X = a.ws + t.X;
  by_cols<WT>(tile, [&](int q, int p, const float (&v)[8]) {
    if (q0 + q < t.m && p0 + p < np) store8(X + (int64_t)(q0 + q) * np * 4, p0 + p, v);
  });
}

// ------------------------------------------------------------------------------------------------ host
constexpr int MAX_STEPS = 32;

// Powers of two for the stored numbers of each step, from bounds on the spectral norms: |X_0| <= 1, and over singular values
// s in [0, r] the next bound is max |s p(s^2)| with p(l) = a + b l + c l^2; A's numbers are within r^2, B's within max |p|.
struct Scales { float x[MAX_STEPS + 1], a[MAX_STEPS], b[MAX_STEPS]; };

float pow2_for(double bound) { return (float)ldexp(1.0, (int)floor(log2(60000.0 / bound))); }

bool ortho_scales(const float* coeff, int steps, Scales* s) {
  double r = 1.0;
  for (int k = 0; k <= steps; ++k) {
    if (!(r <= 1024.0)) return false;
    if (r < 1e-3) r = 1e-3;
    s->x[k] = pow2_for(r);
    if (k == steps) break;
    const double a = coeff[3 * k], b = coeff[3 * k + 1], c = coeff[3 * k + 2];
    double pm = 1e-3, xm = 0.0;
    for (int i = 0; i <= 4096; ++i) {
      const double v = r * i / 4096.0, p = a + b * v * v + c * v * v * v * v;
      if (!(fabs(p) < 1e9)) return false;
      if (fabs(p) > pm) pm = fabs(p);
      if (fabs(v * p) > xm) xm = fabs(v * p);
    }
    s->a[k] = pow2_for(r * r);
    s->b[k] = pow2_for(pm * 1.01);
    if (pm > 4096.0) return false;
    r = xm * 1.01;
  }
  return true;
}

struct Plan {
  int wg, wp, wa;              // wave tiles of the three products: 64 or 32
  int64_t bytes;
  int norms;
  bool split;
};

int tri(int m, int T) { const int n = cdiv(m, T); return n * (n + 1) / 2; }

// Places the workspace and chooses tiles and splits.  128 x 128 tiles read each operand half as often as 64 x 64 ones, but
// need 256 of them to give every CU one.
int make_plan(Mats& a, Plan& p) {
  int64_t poly = 0, apply = 0, work = 0;
  int mmax = 0;
  for (int i = 0; i < a.count; ++i) {
    const Mat& t = a.mat[i];
    poly += tri(t.m, 128);
    apply += (int64_t)cdiv(t.m, 128) * cdiv(t.n, 128);
    if (t.m > mmax) mmax = t.m;
  }
  p.wg = mmax > 64 ? 64 : 32;
  p.wp = poly >= 256 ? 64 : 32;
  p.wa = apply >= 256 ? 64 : 32;
  const int T = 2 * p.wg;
  for (int i = 0; i < a.count; ++i) work += (int64_t)tri(a.mat[i].m, T) * (up32(a.mat[i].n) >> 5);
  // k-blocks per workgroup so that 512 of them, two per CU, share the whole contraction evenly; at least 8
  int64_t kc = cdiv64(work, 512);
  if (kc < 8) kc = 8;
  int64_t off = 0;
  auto take = [&](int64_t bytes) {
    const int64_t at = off;
    off += (bytes + 255) & ~(int64_t)255;
    return at;
  };
  p.norms = 0;
  p.split = false;
  for (int i = 0; i < a.count; ++i) {
    Mat& t = a.mat[i];
    const int64_t mp = up32(t.m), np = up32(t.n), KB = np >> 5;
    t.normc = (int)cdiv64((int64_t)t.m * t.n, NORM_CHUNK);
    t.norm0 = p.norms;
    p.norms += t.normc;
    t.X = take(t.m * np * 4);
    t.Y = take(2 * t.n * mp * 4);
    t.A = take(2 * t.m * mp * 4);
    t.kc = (int)(kc < KB ? kc : KB);
    t.ks = (int)cdiv64(KB, t.kc);
    t.part = 0;
    if (t.ks > 1) {
      t.part = take((int64_t)tri(t.m, T) * t.ks * T * T * 4);
      p.split = true;
    }
  }
  p.bytes = off + 8 * (int64_t)p.norms;
  return SNWS_OK;
}

// grid of a launch: f(mat) workgroups per matrix
template <typename F>
unsigned grid_of(Mats& a, F&& f) {
  int64_t n = 0;
  for (int i = 0; i < a.count; ++i) {
    n += f(a.mat[i]);
    a.end[i] = (int)n;
  }
  return (unsigned)n;
}

// one instance per kernel, so that each has its own flag
template <auto KERNEL>
int ready(int bytes, const char* what) {
  static PerDeviceOnce once;
  std::atomic<bool>* const set = once.flag();
  if (set && set->load(std::memory_order_acquire)) return SNWS_OK;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) {
    snws_set_error("%s: hipFuncSetAttribute failed: %s", what, hipGetErrorString(e));
    return SNWS_ERR_HIP;
  }
  if (set) set->store(true, std::memory_order_release);
  return SNWS_OK;
}

#define ORTHO_TRY(expr)                    \
  do {                                     \
    const int rc__ = (expr);               \
    if (rc__ != SNWS_OK) return rc__;      \
  } while (0)

template <int WT>
int run_gram(Mats& a, const Plan& p, float f, const char* what, hipStream_t st) {
  ORTHO_TRY((ready<&ortho_gram_kernel<WT>>(Tile<WT>::LDS, what)));
  const unsigned grid = grid_of(a, [](const Mat& t) { return (int64_t)tri(t.m, 2 * WT) * t.ks; });
  ortho_gram_kernel<WT><<<grid, 256, Tile<WT>::LDS, st>>>(a, f);
  SNWS_LAUNCH_CHECK(what);
  if (p.split) {
    constexpr int B = 2 * WT / 32;
    const unsigned blocks = grid_of(a, [](const Mat& t) { return t.ks > 1 ? (int64_t)tri(t.m, 2 * WT) * B * B : 0; });
    ortho_join_kernel<WT><<<blocks, 256, 0, st>>>(a, f);
    SNWS_LAUNCH_CHECK(what);
  }
  return SNWS_OK;
}

template <int WT>
int run_poly(Mats& a, float ca, float cb, float cc, const char* what, hipStream_t st) {
  ORTHO_TRY((ready<&ortho_poly_kernel<WT>>(Tile<WT>::LDS, what)));
  const unsigned grid = grid_of(a, [](const Mat& t) { return (int64_t)tri(t.m, 2 * WT); });
  ortho_poly_kernel<WT><<<grid, 256, Tile<WT>::LDS, st>>>(a, ca, cb, cc);
  SNWS_LAUNCH_CHECK(what);
  return SNWS_OK;
}

template <int WT, typename T, bool LAST, bool MUON>
int run_apply(Mats& a, const MuonArgs& u, float f, int odd, const char* what, hipStream_t st) {
  ORTHO_TRY((ready<&ortho_apply_kernel<WT, T, LAST, MUON>>(Tile<WT>::LDS, what)));
  const unsigned grid = grid_of(a, [](const Mat& t) { return (int64_t)cdiv(t.m, 2 * WT) * cdiv(t.n, 2 * WT); });
  ortho_apply_kernel<WT, T, LAST, MUON><<<grid, 256, Tile<WT>::LDS, st>>>(a, u, f, odd);
  SNWS_LAUNCH_CHECK(what);
  return SNWS_OK;
}

template <typename T, bool MUON>
int run_all(Mats& a, const Plan& p, const MuonArgs& u, const float* coeff, int steps, float eps, const Scales& s,
            const char* what, hipStream_t st) {
  double* norms = reinterpret_cast<double*>(a.ws + (p.bytes - 8 * (int64_t)p.norms));
  unsigned grid = grid_of(a, [](const Mat& t) { return (int64_t)t.normc; });
  ortho_norm_kernel<T, MUON><<<grid, 256, 0, st>>>(a, u, norms);
  SNWS_LAUNCH_CHECK(what);
  grid = grid_of(a, [](const Mat& t) { return (int64_t)cdiv(t.m, 64) * cdiv(t.n, 64); });
  ortho_start_kernel<T, MUON><<<grid, 256, 0, st>>>(a, u, norms, eps, s.x[0]);
  SNWS_LAUNCH_CHECK(what);
  for (int k = 0; k < steps; ++k) {
    // stored numbers are true ones times a scale: the factors turn a product of stored numbers into the next stored ones
    const float fa = (float)((double)s.a[k] / ((double)s.x[k] * s.x[k]));
    ORTHO_TRY(p.wg == 64 ? run_gram<64>(a, p, fa, what, st) : run_gram<32>(a, p, fa, what, st));
    const float ca = (float)((double)coeff[3 * k] * s.b[k]), cb = (float)((double)coeff[3 * k + 1] * s.b[k] / s.a[k]);
    const float cc = (float)((double)coeff[3 * k + 2] * s.b[k] / ((double)s.a[k] * s.a[k]));
    ORTHO_TRY(p.wp == 64 ? run_poly<64>(a, ca, cb, cc, what, st) : run_poly<32>(a, ca, cb, cc, what, st));
    const bool last = k + 1 == steps;
    const float fx = (float)((last ? 1.0 : (double)s.x[k + 1]) / ((double)s.x[k] * s.b[k]));
    if (last)
      ORTHO_TRY((p.wa == 64 ? run_apply<64, T, true, MUON>(a, u, fx, k & 1, what, st)
                            : run_apply<32, T, true, MUON>(a, u, fx, k & 1, what, st)));
    else
      ORTHO_TRY((p.wa == 64 ? run_apply<64, float, false, false>(a, u, fx, k & 1, what, st)
                            : run_apply<32, float, false, false>(a, u, fx, k & 1, what, st)));
  }
  return SNWS_OK;
}

int check_size(int rows, int cols, const char* what) {
  SNWS_CHECK_ARG(rows >= 1 && cols >= 1, "%s: a matrix needs at least one row and one column", what);
  // tile counts stay within 32 bits and every workspace offset within what a card holds
  SNWS_CHECK_ARG(rows <= (1 << 20) && cols <= (1 << 20) && (rows < cols ? rows : cols) <= 32768,
                 "%s: %d x %d is larger than 2^20 on one side or 32768 on both", what, rows, cols);
  return SNWS_OK;
}

void set_shape(Mat& t, int rows, int cols) {
  t.flip = rows > cols;
  t.m = t.flip ? cols : rows;
  t.n = t.flip ? rows : cols;
}

int check_common(const float* coeff, int steps, float eps, Scales* s, const char* what) {
  SNWS_CHECK_ARG(coeff && steps >= 1 && steps <= MAX_STEPS, "%s: 1 to %d steps with three coefficients each", what, MAX_STEPS);
  SNWS_CHECK_ARG(eps >= 0.f && isfinite(eps), "%s: eps must be finite and not negative", what);
  SNWS_CHECK_ARG(ortho_scales(coeff, steps, s), "%s: with these coefficients singular values within [0, 1] can grow beyond 1024", what);
  return SNWS_OK;
}

}  // namespace

extern "C" int64_t snws_ortho_workspace_bytes(const int* rows, const int* cols, int count) {
  if (!rows || !cols || count < 1 || count > MAXM) return -1;
  Mats a{};
  Plan p;
  a.count = count;
  for (int i = 0; i < count; ++i) {
    if (check_size(rows[i], cols[i], "snws_ortho_workspace_bytes") != SNWS_OK) return -1;
    set_shape(a.mat[i], rows[i], cols[i]);
  }
  make_plan(a, p);
  return p.bytes;
}

extern "C" int snws_orthogonalize(const snws_ortho_item* items, int count, int dtype, const float* coeff, int steps, float eps,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "snws_orthogonalize";
  SNWS_CHECK_ARG(dtype == SNWS_F32 || dtype == SNWS_BF16, "%s: dtype must be float32 or bfloat16", what);
  SNWS_CHECK_ARG(items && count >= 1 && count <= MAXM, "%s: 1 to %d matrices", what, MAXM);
  Scales s;
  ORTHO_TRY(check_common(coeff, steps, eps, &s, what));
  Mats a{};
  Plan p;
  a.count = count;
  for (int i = 0; i < count; ++i) {
    const snws_ortho_item& t = items[i];
    ORTHO_TRY(check_size(t.rows, t.cols, what));
    SNWS_CHECK_ARG(t.x && t.out, "%s: NULL pointer", what);
    SNWS_CHECK_ARG(t.ldx >= t.cols && t.ldo >= t.cols, "%s: row strides must be at least the columns", what);
    set_shape(a.mat[i], t.rows, t.cols);
    a.mat[i].x = t.x;
    a.mat[i].out = t.out;
    a.mat[i].ldx = t.ldx;
    a.mat[i].ldo = t.ldo;
  }
  make_plan(a, p);
  SNWS_CHECK_ARG(workspace && workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0,
                 "%s: workspace of %lld bytes, 256-byte aligned, needed", what, (long long)p.bytes);
  a.ws = static_cast<unsigned char*>(workspace);
  const MuonArgs u{};
  return dtype == SNWS_F32 ? run_all<float, false>(a, p, u, coeff, steps, eps, s, what, (hipStream_t)stream)
                           : run_all<bf16_t, false>(a, p, u, coeff, steps, eps, s, what, (hipStream_t)stream);
}

extern "C" int snws_muon_update(const snws_muon_item* items, int count, float momentum, int nesterov, float grad_scale,
                                float weight_decay, const float* coeff, int steps, float eps, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  const char* what = "snws_muon_update";
  SNWS_CHECK_ARG(items && count >= 1 && count <= MAXM, "%s: 1 to %d matrices", what, MAXM);
  SNWS_CHECK_ARG(momentum >= 0.f && momentum <= 1.f, "%s: momentum must lie within [0, 1]", what);
  Scales s;
  ORTHO_TRY(check_common(coeff, steps, eps, &s, what));
  Mats a{};
  Plan p;
  a.count = count;
  for (int i = 0; i < count; ++i) {
    const snws_muon_item& t = items[i];
    ORTHO_TRY(check_size(t.rows, t.cols, what));
    SNWS_CHECK_ARG(t.param && t.grad && t.momentum, "%s: NULL pointer", what);
    set_shape(a.mat[i], t.rows, t.cols);
    a.mat[i].x = t.grad;
    a.mat[i].out = t.param;
    a.mat[i].mom = t.momentum;
    a.mat[i].ldx = a.mat[i].ldo = t.cols;
    a.mat[i].step = t.lr;
  }
  make_plan(a, p);
  SNWS_CHECK_ARG(workspace && workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0,
                 "%s: workspace of %lld bytes, 256-byte aligned, needed", what, (long long)p.bytes);
  a.ws = static_cast<unsigned char*>(workspace);
  const MuonArgs u{momentum, grad_scale, 1.f - weight_decay, nesterov};
  return run_all<float, true>(a, p, u, coeff, steps, eps, s, what, (hipStream_t)stream);
}
