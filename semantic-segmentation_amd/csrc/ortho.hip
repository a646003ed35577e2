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
// 128-byte line, an LDS-DMA instruction copies 8 rows x 128 bytes, and both halves of a fragment come from the same line.
// X X^T and the m x m products read both operands along their rows (all m x m matrices here are symmetric); B X reads
// X down its columns, through the transposing LDS read, so X is kept in one orientation only.
//
// All matrices of a list share each launch: a workgroup finds its matrix and tile from its index.
//
// Measured, float32, five steps: 64 x 126 21 us (one launch), 1024 x 9216 361 us (norm 8, start 16, X X^T 31.5 and its join
// 8 twice, 13 launches of m x m products at 10.8, Q X 53 and 59), the 21 million numbers of 17 filters with their Muon
// update 807 us (nine of 128 rows and more in threes: 44, 50, 56 and 9 twice, 13 x 19, 103 and 124; eight of 64 in single
// steps: 125).
#include "common.h"
#include <math.h>

namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

constexpr int MAXM = SNWS_ORTHO_MAX;
constexpr int NORM_CHUNK = 8192;    // elements per partial sum of squares

struct Mat {
  const void* x;       // (rows, cols), row stride ldx: the matrix, or the gradient of a Muon item
  void* out;           // (rows, cols), row stride ldo: the result, or the parameter of a Muon item
  float* mom;          // momentum of a Muon item
  int64_t ldx, ldo;
  int64_t at;          // its part of the workspace (bytes): X, a second X, the slots, partial tiles of A
  int m, n;            // m <= n
  int flip;            // rows > cols: X is the transpose
  int ks, kc;          // splits of the contraction over n and 32-blocks in each
  int norm0, normc;    // partial sums of squares
  float step;          // learning rate of a Muon item
};

enum Phase { NORM, START, GRAM, JOIN, SQUARE, APPLY, PHASES };

// The first kernel of a call gets this by value and leaves a copy at the start of the workspace for the others: kernel
// arguments lie in host memory, where each dependent read costs a microsecond.
struct Mats {
  Mat mat[MAXM];
  int end[PHASES][MAXM];      // first workgroup index behind each matrix, by the kind of launch
  int count;
  unsigned char* ws;
};

// What the other kernels get: the list's copy in the workspace, and the matrix itself where there is only one: no trip to
// memory before the first copy, 0.4 us of each of the twenty launches.
struct Work {
  unsigned char* ws;
  int count;
  Mat only;
};

// D = ca I + cb C + cc P Q on the slots of every matrix (see square_tile), or a product with X
enum Kind { K_GRAM, K_SQUARE, K_APPLY };
struct Op {
  unsigned char kind, sp, sq, sc, sd, last, pad[2];
  float ca, cb, cc;
};
constexpr int MAX_OPS = 24;    // of a program that one kernel runs: eight single steps
constexpr int GROUP_OPS = 12;  // of a group of three: X X^T, nine products of m x m matrices, Q X
struct Program {
  int n;
  Op op[MAX_OPS];
};

struct MuonArgs {
  float momentum, grad_scale, decay;
  int nesterov;
};

__host__ __device__ __forceinline__ int up32(int v) { return (v + 31) & ~31; }

// parts of a matrix's workspace; every one is a whole number of 128-byte blocks
constexpr int SLOTS = 6;
__host__ __device__ __forceinline__ int64_t size_x(const Mat& t) { return (int64_t)t.m * up32(t.n) * 4; }
__host__ __device__ __forceinline__ int64_t size_slot(const Mat& t) { return (int64_t)t.m * up32(t.m) * 4; }
__device__ __forceinline__ unsigned char* x_of(const Mat& t, unsigned char* ws, int odd) { return ws + t.at + (odd ? size_x(t) : 0); }
__device__ __forceinline__ unsigned char* slot_of(const Mat& t, unsigned char* ws, int k) {
  return ws + t.at + 2 * size_x(t) + k * size_slot(t);
}
__device__ __forceinline__ f32x4* part_of(const Mat& t, unsigned char* ws) {
  return reinterpret_cast<f32x4*>(slot_of(t, ws, SLOTS));
}

// 16 bytes per lane from global memory (base, the same for the whole wave, plus the lane's offset) into LDS, lane after
// lane from byte `lds` on.  Written out because the compiler would wait for every copy in flight before a transposing read;
// it has no result registers, and the waits for it stand in product().  Nothing else here uses m0.
__device__ __forceinline__ void glds16(const unsigned char* base, unsigned offset, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds));
}
__device__ __forceinline__ unsigned lds_offset(const void* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// blocks dealt to the same XCD (bid % 8) get consecutive logical ids
__device__ __forceinline__ unsigned xcd_order(unsigned bid, unsigned nblk) {
  const unsigned q = nblk >> 3, r = nblk & 7, xcd = bid & 7;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (bid >> 3);
}

// Matrix of this workgroup of a list, and its index there.  Workgroups of one XCD (every eighth) get neighbouring indices
// within each matrix: they share operands in its L2, and every XCD gets its share of every matrix.  Every lane reads a matrix
// of its own together with its end, so that the choice costs one trip to memory instead of two.
__device__ __forceinline__ Mat pick_mat(const Mats& a, int count, int phase, int& local) {
  constexpr int V = sizeof(Mat) / 16;
  static_assert(sizeof(Mat) % 16 == 0, "whole vectors");
  const int lane = threadIdx.x & 63, mine = lane < count ? lane : 0, id = blockIdx.x;
  uint4 v[V];
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = reinterpret_cast<const uint4*>(&a.mat[mine])[k];
  const int end = a.end[phase][mine];
  const int i = __builtin_amdgcn_readfirstlane(__popcll(__ballot(lane < count && id >= end)));
  const int from = i ? __builtin_amdgcn_readlane(end, i - 1) : 0;
  local = xcd_order(id - from, __builtin_amdgcn_readlane(end, i) - from);
  union { Mat m; int w[4 * V]; } t;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    t.w[4 * k] = __builtin_amdgcn_readlane((int)v[k].x, i);
    t.w[4 * k + 1] = __builtin_amdgcn_readlane((int)v[k].y, i);
    t.w[4 * k + 2] = __builtin_amdgcn_readlane((int)v[k].z, i);
    t.w[4 * k + 3] = __builtin_amdgcn_readlane((int)v[k].w, i);
  }
  return t.m;
}
// A matrix alone comes with the kernel's arguments.
__device__ __forceinline__ Mat find_mat(const Work& a, int phase, int& local) {
  if (a.count > 1) return pick_mat(*reinterpret_cast<const Mats*>(a.ws), a.count, phase, local);
  local = xcd_order(blockIdx.x, gridDim.x);
  return a.only;
}

typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;

// v = hi + lo: two numbers at a time through the packed conversions, the remainder by one mixed multiply-add
__device__ __forceinline__ void split2(float a, float b, f16x2& hi, f16x2& lo) {
  hi = __builtin_convertvector((f32x2{a, b}), f16x2);
  lo = __builtin_convertvector((f32x2{fmaf((float)hi[0], -1.f, a), fmaf((float)hi[1], -1.f, b)}), f16x2);
}
__device__ __forceinline__ void split4(const float (&v)[4], f16x4& hi, f16x4& lo) {
  f16x2 h0, h1, l0, l1;
  split2(v[0], v[1], h0, l0);
  split2(v[2], v[3], h1, l1);
  hi = f16x4{h0[0], h0[1], h1[0], h1[1]};
  lo = f16x4{l0[0], l0[1], l1[0], l1[1]};
}
__device__ __forceinline__ void split8(const float (&v)[8], uint4& hi, uint4& lo) {
  f16x2 h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) split2(v[2 * e], v[2 * e + 1], h[e], l[e]);
  hi = make_uint4(__builtin_bit_cast(unsigned, h[0]), __builtin_bit_cast(unsigned, h[1]), __builtin_bit_cast(unsigned, h[2]),
                  __builtin_bit_cast(unsigned, h[3]));
  lo = make_uint4(__builtin_bit_cast(unsigned, l[0]), __builtin_bit_cast(unsigned, l[1]), __builtin_bit_cast(unsigned, l[2]),
                  __builtin_bit_cast(unsigned, l[3]));
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
// the matrix itself, or a Muon item's update direction from gradient and momentum (already advanced)
__device__ __forceinline__ float direction(float g, float m, const MuonArgs& u) {
  return u.nesterov ? (1.f - u.momentum) * g + u.momentum * m : m;
}

// Partial sums of squares in float64 (no overflow or underflow over float32's range, a fixed order); a Muon item's
// momentum is advanced on the way: m <- momentum m + (1 - momentum) grad_scale g.  Bound by memory: 4.6 TB/s for a
// 1024 x 9216 matrix, 5.5 TB/s for the gradients and momenta of 21 million parameters.
template <typename T, bool MUON>
__device__ __forceinline__ double norm_chunk(const Mat& t, int chunk, const MuonArgs& u) {
  constexpr int VEC = MUON ? 4 : 16 / (int)sizeof(T);
  const int rows = t.flip ? t.n : t.m, cols = t.flip ? t.m : t.n;
  const int64_t total = (int64_t)rows * cols, lo = (int64_t)chunk * NORM_CHUNK;
  const T* x = static_cast<const T*>(t.x);
  double s = 0.0;
  auto one = [&](int64_t i, float v) {
    if (MUON) {
      v *= u.grad_scale;
      const float m = u.momentum * t.mom[i] + (1.f - u.momentum) * v;
      t.mom[i] = m;
      v = direction(v, m, u);
    }
    s += (double)v * (double)v;
  };
  const bool flat = t.ldx == cols && (((uintptr_t)x | (MUON ? (uintptr_t)t.mom : 0)) & 15) == 0;
  const int64_t hi = lo + NORM_CHUNK < total ? lo + NORM_CHUNK : total;
  if (flat) {       // chunks start at multiples of 16 bytes: all loads of a thread in flight at once
    constexpr int NL = NORM_CHUNK / (256 * VEC);
    uint4 v[NL];
    float4 m[MUON ? NL : 1];
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      const int64_t i = lo + (int64_t)(k * 256 + threadIdx.x) * VEC;
      v[k] = make_uint4(0, 0, 0, 0);
      if (MUON) m[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i + VEC <= hi) {
        v[k] = *reinterpret_cast<const uint4*>(x + i);
        if (MUON) m[k] = *reinterpret_cast<const float4*>(t.mom + i);
      }
    }
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      const T* e8 = reinterpret_cast<const T*>(&v[k]);
      float d[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) d[e] = (float)e8[e];
      if (MUON) {
        float* me = &m[k].x;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          d[e] *= u.grad_scale;
          me[e] = u.momentum * me[e] + (1.f - u.momentum) * d[e];
          d[e] = direction(d[e], me[e], u);
        }
        const int64_t i = lo + (int64_t)(k * 256 + threadIdx.x) * VEC;
        if (i + VEC <= hi) *reinterpret_cast<float4*>(t.mom + i) = m[k];
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += (double)d[e] * (double)d[e];
    }
    const int64_t tail = hi - (hi - lo) % VEC + threadIdx.x;
    if (tail < hi) one(tail, (float)x[tail]);
  } else {
    int64_t i = lo + threadIdx.x;
    if (i < hi) {
      int64_t r = i / cols;
      int c = (int)(i - r * cols);
#pragma unroll 8
      for (; i < hi; i += 256) {
        one(i, (float)x[r * t.ldx + c]);
        for (c += 256; c >= cols; c -= cols) ++r;
      }
    }
  }
  return s;
}

template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ortho_norm_kernel(Mats a, MuonArgs u, double* __restrict__ partial) {
  __shared__ double red[16];
  if (blockIdx.x == 0 && a.count > 1)
    for (int i = threadIdx.x; i < (int)(sizeof(Mats) / 4); i += 256)
      reinterpret_cast<int*>(a.ws)[i] = reinterpret_cast<const int*>(&a)[i];
  int chunk;
  Mat t = a.mat[0];
  if (a.count > 1) t = pick_mat(a, a.count, NORM, chunk);
  else chunk = blockIdx.x;
  const double s = block_sum(norm_chunk<T, MUON>(t, chunk, u), red);
  if (threadIdx.x == 0) partial[t.norm0 + chunk] = s;
}


struct __attribute__((packed, aligned(4))) F4 { float f[4]; };
struct __attribute__((packed, aligned(2))) H8 { unsigned u[4]; };

// eight consecutive elements of any alignment
__device__ __forceinline__ void read8(const float* p, float (&v)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const F4 w = *reinterpret_cast<const F4*>(p + 4 * h);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[4 * h + e] = w.f[e];
  }
}
__device__ __forceinline__ void read8(const bf16_t* p, float (&v)[8]) {
  const H8 w = *reinterpret_cast<const H8*>(p);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[2 * e] = __uint_as_float(w.u[e] << 16);
    v[2 * e + 1] = __uint_as_float(w.u[e] & 0xffff0000u);
  }
}

// A 64 x 64 tile of the source, times f, into X: 16-byte reads to 16-byte stores, row by row, or - where X is the
// transpose - through LDS.  Bound by memory: 4.5 TB/s read and written for 1024 x 9216, 5 TB/s for a model's filters.
template <typename T, bool MUON>
__device__ __forceinline__ void start_tile(const Mat& t, unsigned char* ws, int local, double f, const MuonArgs& u, float* tile) {
  constexpr int LP = 66;
  const int rows = t.flip ? t.n : t.m, cols = t.flip ? t.m : t.n;
  const int tc = (cols + 63) >> 6, r0 = (local / tc) * 64, c0 = (local % tc) * 64;
  const T* x = static_cast<const T*>(t.x);
  unsigned char* X = x_of(t, ws, 0);
  float v[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = r0 + k * 32 + (threadIdx.x >> 3), c = c0 + (threadIdx.x & 7) * 8;
    float m[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[k][e] = m[e] = 0.f;
    if (r < rows) {
      const T* p = x + (int64_t)r * t.ldx + c;
      const float* q = MUON ? t.mom + (int64_t)r * cols + c : nullptr;
      if (c + 8 <= cols) {
        read8(p, v[k]);
        if (MUON) read8(q, m);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < cols) {
            v[k][e] = (float)p[e];
            if (MUON) m[e] = q[e];
          }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[k][e] = (float)(f * (double)(MUON ? direction(v[k][e] * u.grad_scale, m[e], u) : v[k][e]));
  }
  if (!t.flip) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = r0 + k * 32 + (threadIdx.x >> 3), c = c0 + (threadIdx.x & 7) * 8;
      if (r < rows && c < up32(cols)) store8(X + (int64_t)r * up32(cols) * 4, c, v[k]);
    }
    return;
  }
  __syncthreads();                    // the previous tile has been read
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) tile[(k * 32 + (threadIdx.x >> 3)) * LP + (threadIdx.x & 7) * 8 + e] = v[k][e];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int id = k * 256 + threadIdx.x;
    float w[8];
    const int q = (id >> 2 & 15) + (id >> 7) * 16, p = ((id & 3) + (id >> 6 & 1) * 4) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = tile[(p + e) * LP + q];
    if (c0 + q < cols && r0 + p < up32(rows)) store8(X + (int64_t)(c0 + q) * up32(rows) * 4, r0 + p, w);
  }
}

// scale / max(norm, eps): a NaN stays one.  In float64, and multiplied as such: the inverse of a small norm leaves float32.
__device__ __forceinline__ double start_factor(double sum, float eps, float scale) {
  const double norm = sqrt(sum);
  return (double)scale / (norm < (double)eps ? (double)eps : norm);
}

// X_0: the matrices, normalised
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ortho_start_kernel(Work a, MuonArgs u,
                                                          const double* __restrict__ partial, float eps, float scale) {
  __shared__ float tile[64 * 66];
  __shared__ double red[16];
  int local;
  const Mat t = find_mat(a, START, local);
  double s = 0.0;
  for (int i = threadIdx.x; i < t.normc; i += 256) s += partial[t.norm0 + i];
  start_tile<T, MUON>(t, a.ws, local, start_factor(block_sum(s, red), eps, scale), u, tile);
}

// ------------------------------------------------------------------------------------------------ products
// A workgroup of WM x WN waves on a TM x TN tile; k advances by 32 through a ring of S stages, of which S - 1 are on their
// way while one is multiplied.
template <int TM_, int TN_, int WM_, int WN_, int S_>
struct Tile {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, S = S_, W = WM * WN, THREADS = 64 * W;
  static constexpr int MR = TM / WM / 16, NR = TN / WN / 16;              // 16 x 16 products of a wave
  static constexpr int PL = TM / 8 / W, QL = TN / 8 / W;                  // 1 KB LDS-DMA pieces of P and Q, per wave and stage
  static constexpr int LOADS = PL + QL, STAGE = (TM + TN) * 128;
  static constexpr int LP = TN + 2, SLAB = TM * LP * 4 > 80 * 1024 ? 64 : TM;      // the epilogue's LDS tile: row, and rows at once
  static constexpr int LDS = S * STAGE > SLAB * LP * 4 ? S * STAGE : SLAB * LP * 4;
  static constexpr int PER_CU = 2 * LDS <= 160 * 1024 && 2 * W <= 16 ? 2 : 1;
  static_assert(W % 4 == 0 && PL * W * 8 == TM && QL * W * 8 == TN && MR * WM * 16 == TM && NR * WN * 16 == TN && TN % 32 == 0, "whole pieces");
  static_assert(LDS <= 160 * 1024, "LDS of a CU");
};
// Large tiles bring more products with each byte copied, small ones occupy more CUs.  Two workgroups on a CU take turns: one
// multiplies while the other waits.
// 128 x 128, four waves of 64 x 64, two workgroups to a CU: X X^T of 1024 x 9216 in 31.5 us, 0.92 PFLOP/s (64 x 64: 41 us)
typedef Tile<128, 128, 2, 2, 2> Big;
// 128 x 160, four waves of 64 x 80, where that saves a round: Q X there in 53 us, 1.09 PFLOP/s (128 x 128: 67, 64 x 64: 74)
typedef Tile<128, 160, 2, 2, 2> Wide;
// 64 x 64, where there are few tiles; eight waves, so that each SIMD has two to alternate: a product of 1024 x 1024 in
// 10.8 us (128 x 128: 28 us).  Of those about 4 are the launch, the first copies and the epilogue; in the rest the matrix
// units are busy for 2.6: the operands come from beyond the L2s, of which each needs half the matrix: 26 MB, 5 us.  A
// deeper ring or a barrier for every second stage only change nothing.
typedef Tile<64, 64, 2, 4, 4> Fine;
// 96 x 64, four waves of 48 x 32, for m x m products where that makes fewer rounds
typedef Tile<96, 64, 2, 2, 4> Tall;

typedef __attribute__((ext_vector_type(4))) short short4v;

// acc[mr][nr] += P rows p0.. x Q over the k-blocks [kb0, kb1).  P: M rows of KB blocks.  Q: N rows of KB blocks like it,
// rows q0..; or, DOWN, K rows of N numbers in QB blocks each, columns q0...  What lies past the last row or block is read
// as the last one (its results are not stored, and k past the end meets zeros of P).  Entered and left with the LDS free.
template <typename G, bool DOWN = false>
__device__ __forceinline__ void product(f32x4 (&acc)[G::MR][G::NR], const unsigned char* P, const unsigned char* Q, int p0,
                                        int q0, int M, int N, int KB, int kb0, int kb1, unsigned char* smem, int K = 0, int QB = 0) {
  constexpr int MR = G::MR, NR = G::NR, W = G::W, PL = G::PL;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / G::WN, wn = wave % G::WN;
  // LDS-DMA of rows: piece w + W j holds its rows 8 (w + W j) .. + 7; lane -> row lane >> 3, slot lane & 7, which receives the
  // 16-byte chunk slot ^ ((row >> 1) & 7), so that the 16 lanes of a fragment read hit distinct banks
  const int chunk = (lane & 7) ^ ((4 * (wave & 1) + (lane >> 4)) & 7);
  // Offsets from the tile's first row: at most 127 rows (Q: TN - 1) of at most 4 MB, below 2^30.  They are put together anew for
  // every stage: an addition and a minimum each, where keeping them would cost registers the products need.  The last row they
  // may reach is the matrix's or the tile's, whichever comes first: the distance to the matrix's alone would leave 32 bits from
  // 2^30 numbers on.
  const unsigned line = KB * 128, first = (8 * wave + (lane >> 3)) * line;
  const unsigned lastp = (unsigned)(M - 1 - p0 < G::TM - 1 ? M - 1 - p0 : G::TM - 1) * line;
  const int64_t pitch = (int64_t)QB * 128;
  const unsigned lastq = DOWN ? (unsigned)(QB - 1) * 128 : (unsigned)(N - 1 - q0 < G::TN - 1 ? N - 1 - q0 : G::TN - 1) * line;
  // DOWN: piece c of Q is column block c / 4, k-rows 8 (c % 4) .. + 7 of the stage.  A transposing read takes 32 bytes from
  // each of 16 rows 8 g + t (g, t < 4): pairs of chunks trade places by (t >> 1) + 2 (g & 1), so that they meet in twos.
  const unsigned firstq = DOWN ? (unsigned)((q0 >> 5) + (wave >> 2)) * 128 : first;
  unsigned krow = 0, kend = 0;       // offset of this lane's k-row and chunk in a stage; in the last one
  if (DOWN) {
    const int r = 8 * (wave & 3) + (lane >> 3), left = K - (KB - 1) * 32;
    const unsigned dchunk = ((lane & 7) ^ (((lane >> 4 & 1) + 2 * (wave & 1)) << 1)) * 16;
    krow = r * (unsigned)pitch + dchunk;
    kend = (r < left ? r : left - 1) * (unsigned)pitch + dchunk;
  }
  const unsigned char* Pt = P + (int64_t)p0 * line;
  const unsigned char* Qt = DOWN ? Q : Q + (int64_t)q0 * line;
  const unsigned base = __builtin_amdgcn_readfirstlane(lds_offset(smem)) + wave * 1024;
  // copy c of this wave's PL + QL for stage kb
  auto copy = [&](int c, int kb, int buf) {
    const unsigned to = base + buf * G::STAGE;
    if (c < PL) {
      const unsigned at = first + c * (8 * W) * line;
      glds16(Pt + (int64_t)kb * 128, (at < lastp ? at : lastp) + chunk * 16, to + c * (W * 1024));
    } else {
      const int j = c - PL;
      const unsigned krows = kb + 1 < KB ? krow : kend;
      const unsigned at = firstq + j * (DOWN ? (W / 4) * 128u : (8 * W) * line);
      glds16(Qt + (DOWN ? kb * 32 * pitch : (int64_t)kb * 128), (at < lastq ? at : lastq) + (DOWN ? krows : chunk * 16),
             to + G::TM * 128 + j * (W * 1024));
    }
  };
  int fro[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) fro[h] = (lane & 15) * 128 + (((h * 4 + (lane >> 4)) ^ ((lane >> 1) & 7)) * 16);
  // transposing reads: lane -> k-row 8 g + t of the eight 8 g .. (the upper four follow 512 bytes on), four columns 4 c ..
  // [half][odd or even block r of the wave]; where a wave begins in the middle of a 32-column block, `mid`, the sides swap
  // and an odd r belongs to the next block
  int tro[4];
  const int mid = (wn * NR) & 1;
  if (DOWN) {
    const int g = lane >> 4, t = lane >> 2 & 3, c = lane & 3, turn = (t >> 1) + 2 * (g & 1);
#pragma unroll
    for (int v = 0; v < 4; ++v)
      tro[v] = ((wn * NR) >> 1) * 4096 + (8 * g + t) * 128 + ((v ^ mid ^ turn) * 2 + (c >> 1)) * 16 + (c & 1) * 8 + (v & mid) * 4096;
  }
  struct Frags { f16x8 ph[MR], pl[MR], qh[NR], ql[NR]; };
  // read x of the 2 MR + 2 NR fragments of a stage: high halves, low halves of Q, low halves of P, in the order of their use
  auto fetch = [&](Frags& f, int buf, int x) {
    const unsigned char* pb = smem + buf * G::STAGE + wm * (MR * 2048);
    const unsigned char* qb = smem + buf * G::STAGE + G::TM * 128;
    auto q_of = [&](int r, int half) {
      if (!DOWN) return *reinterpret_cast<const f16x8*>(qb + (wn * NR + r) * 2048 + fro[half]);
      typedef __attribute__((ext_vector_type(8))) short short8v;
      const unsigned char* at = qb + (r >> 1) * 4096 + tro[half * 2 + (r & 1)];
      const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)at);
      const short4v b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(at + 512));
      return __builtin_bit_cast(f16x8, short8v{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
    };
    if (x < MR) f.ph[x] = *reinterpret_cast<const f16x8*>(pb + x * 2048 + fro[0]);
    else if (x < MR + NR) f.qh[x - MR] = q_of(x - MR, 0);
    else if (x < MR + 2 * NR) f.ql[x - MR - NR] = q_of(x - MR - NR, 1);
    else f.pl[x - MR - 2 * NR] = *reinterpret_cast<const f16x8*>(pb + (x - MR - 2 * NR) * 2048 + fro[1]);
  };
  // product x of the 3 MR NR of a stage
  auto multiply = [&](const Frags& f, int x) {
    const int w = x / (MR * NR), i = x / NR % MR, j = x % NR;
    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w == 2 ? f.pl[i] : f.ph[i], w == 1 ? f.ql[j] : f.qh[j], acc[i][j], 0, 0, 0);
  };
  // The loop has no branches: the last stages are fetched again where there are no more, so that the number in flight,
  // and with it every wait, is a constant.
  const int nk = kb1 - kb0;
  auto ring = [&](int k) { return (G::S & (G::S - 1)) == 0 ? k & (G::S - 1) : k % G::S; };
  auto issue = [&](int k) {
#pragma unroll
    for (int c = 0; c < G::LOADS; ++c) copy(c, kb0 + (k < nk ? k : nk - 1), ring(k));
  };
  // the oldest stage in flight has landed for every wave, and every wave holds its fragments of the one before
  auto landed = [&] {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((G::S - 2) * G::LOADS) : "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  Frags f[2];
#pragma unroll
  for (int d = 0; d < G::S - 1; ++d) issue(d);
  landed();
#pragma unroll
  for (int x = 0; x < 2 * MR + 2 * NR; ++x) fetch(f[0], 0, x);
  issue(G::S - 1);
  // While stage k is multiplied from registers, the fragments of k + 1 are read and stage k + S is on its way.  A copy
  // instruction occupies the CU's address unit for 16 cycles, as long as a product its matrix unit, and what waits for it
  // holds up all that follows in its wave: so the copies are spread over the step, one to each part of it, with the reads
  // (done before the last part, so that they have arrived at its end) and products.  All copies first: 0.9 us a step
  // of 128 x 128 instead of 0.7.
  // The older of the two workgroups of a CU is served first and would leave the younger alone at the end: they go first in
  // turns (the first 256 workgroups are one to a CU).  Q X of 1024 x 9216 takes 53 us, 56 without; with
  // eight waves it gains nothing.
  auto step = [&](int k, const Frags& now, Frags& next) {
    if (G::PER_CU == 2 && W == 4) {
      if ((k ^ (int)(blockIdx.x >> 8)) & 1) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
    }
    landed();
    constexpr int PARTS = G::LOADS, PRODUCTS = 3 * MR * NR, READS = 2 * MR + 2 * NR, EARLY = PARTS > 2 ? PARTS - 1 : PARTS;
    const int kc = kb0 + (k + G::S < nk ? k + G::S : nk - 1), to = ring(k + G::S), from = ring(k + 1);
#pragma unroll
    for (int c = 0; c < PARTS; ++c) {
      constexpr int most = (PRODUCTS + PARTS - 1) / PARTS;
      copy(c, kc, to);
#pragma unroll
      for (int x = c * READS / EARLY; x < (c + 1) * READS / EARLY && x < READS; ++x) fetch(next, from, x);
#pragma unroll
      for (int x = c * PRODUCTS / PARTS; x < (c + 1) * PRODUCTS / PARTS; ++x) multiply(now, x);
#pragma unroll
      for (int q = 0; q < most; ++q) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, DOWN ? 2 : 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto finish = [&](const Frags& now) {
#pragma unroll
    for (int x = 0; x < 3 * MR * NR; ++x) multiply(now, x);
  };
  int k = 0;
  for (; k + 2 < nk; k += 2) {
    step(k, f[0], f[1]);
    step(k + 1, f[1], f[0]);
  }
  if (k + 1 < nk) {
    step(k, f[0], f[1]);
    finish(f[1]);
  } else {
    finish(f[0]);
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");       // the stages are free for other use
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// rows SLAB h .. of the tile: the accumulators, times f, as SLAB rows of LP floats in LDS; zeros outside M x N
template <typename G>
__device__ __forceinline__ void to_lds(const f32x4 (&acc)[G::MR][G::NR], float f, int h, int p0, int q0, int M, int N, float* tile) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int top = (wave / G::WN) * (16 * G::MR) - h * G::SLAB;
  if (top >= 0 && top < G::SLAB) {
    const int pr = top + 4 * (lane >> 4), qc = (wave % G::WN) * (16 * G::NR) + (lane & 15);
    p0 += h * G::SLAB;
    if (p0 + G::SLAB <= M && q0 + G::TN <= N) {
#pragma unroll
      for (int i = 0; i < G::MR; ++i)
#pragma unroll
        for (int j = 0; j < G::NR; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) tile[(pr + i * 16 + r) * G::LP + qc + j * 16] = acc[i][j][r] * f;
    } else {
#pragma unroll
      for (int i = 0; i < G::MR; ++i)
#pragma unroll
        for (int j = 0; j < G::NR; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int p = pr + i * 16 + r, q = qc + j * 16;
            tile[p * G::LP + q] = p0 + p < M && q0 + q < N ? acc[i][j][r] * f : 0.f;
          }
    }
  }
  __syncthreads();
}
// f(p, q, v): eight columns q .. q + 7 of row p, for every row and octet of a slab
template <typename G, typename F>
__device__ __forceinline__ void by_rows(const float* tile, F&& f) {
  constexpr int C8 = G::TN / 8;
#pragma unroll 2
  for (int id = threadIdx.x; id < G::SLAB * C8; id += G::THREADS) {
    const int p = id / C8, q = (id % C8) * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[p * G::LP + q + e];
    f(p, q, v);
  }
}
// f(q, p, v): eight rows p .. p + 7 of column q.  Four lanes take the 32 rows of a block, sixteen the next columns: the
// reads of a wave spread over all banks (8 LP = 16 mod 32) and the stores of four lanes share a line.
template <typename G, typename F>
__device__ __forceinline__ void by_cols(const float* tile, F&& f) {
  constexpr int B = G::SLAB / 32;
#pragma unroll 2
  for (int id = threadIdx.x; id < G::SLAB * G::TN / 8; id += G::THREADS) {
    const int g = id >> 6, p = ((g % B) * 4 + (id & 3)) * 8, q = (g / B) * 16 + (id >> 2 & 15);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[(p + e) * G::LP + q];
    f(q, p, v);
  }
}

template <int M, int N>
__device__ __forceinline__ void clear(f32x4 (&acc)[M][N]) {
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// Tile number t of a lower triangle of nt tiles a side -> (i, j), j <= i, counted through blocks of 4 x 4 tiles: sixteen
// neighbours read eight rows of tiles, where a row of the triangle would read the whole matrix - in every XCD's L2.
__device__ __forceinline__ void triangle(int t, int nt, int& i, int& j) {
  int I = (int)((sqrtf(2.f + 16.f * (float)t) - 1.f) * 0.125f);          // 8 I^2 + 2 I tiles lie before block row I
  while (8 * (I + 1) * (I + 1) + 2 * (I + 1) <= t) ++I;
  while (8 * I * I + 2 * I > t) --I;
  const int rem = t - 8 * I * I - 2 * I, r = nt - 4 * I < 4 ? nt - 4 * I : 4;
  const int J = rem / (4 * r) < I ? rem / (4 * r) : I;
  const int at = rem - J * 4 * r;
  if (J < I) {
    i = 4 * I + at % r;
    j = 4 * J + at / r;
  } else {
    const int d = at >= 6 ? 3 : at >= 3 ? 2 : at >= 1 ? 1 : 0;
    i = 4 * I + d;
    j = 4 * I + at - d * (d + 1) / 2;
  }
}

// Tiles half as high again as wide: strip i needs columns up to its own end, 3 (i + 1) / 2 tiles; two strips together, column
// by column.
__device__ __forceinline__ void tall_triangle(int t, int rows, int cols, int& i, int& j) {
  int I = (int)((sqrtf(1.f + 3.f * (float)t) - 1.f) * 0.33333333f);      // 3 I^2 + 2 I tiles lie before strip 2 I
  while (3 * (I + 1) * (I + 1) + 2 * (I + 1) <= t) ++I;
  while (3 * I * I + 2 * I > t) --I;
  const int rem = t - 3 * I * I - 2 * I, first = 3 * I + 2 < cols ? 3 * I + 2 : cols;
  const bool alone = 2 * I + 1 >= rows, both = !alone && rem < 2 * first;
  i = alone ? 2 * I : both ? 2 * I + (rem & 1) : 2 * I + 1;
  j = alone ? rem : both ? rem >> 1 : rem - first;
}

template <typename G>
__device__ __forceinline__ void place(int t, int m, int& p0, int& q0) {
  static_assert((G::TM == G::TN || 2 * G::TM == 3 * G::TN) && G::TM == G::SLAB, "symmetric matrices: tiles of one slab");
  int i, j;
  if (G::TM == G::TN) triangle(t, (m + G::TM - 1) / G::TM, i, j);
  else tall_triangle(t, (m + G::TM - 1) / G::TM, (m + G::TN - 1) / G::TN, i, j);
  p0 = i * G::TM;
  q0 = j * G::TN;
}

// Of a symmetric matrix a tile stores what lies left of its strip's end, and the mirror image of what lies left of its strip.
template <typename G>
__device__ __forceinline__ bool own(int p0, int col) { return G::TM == G::TN || col < p0 + G::TM; }
template <typename G>
__device__ __forceinline__ bool mirrored(int p0, int col) { return G::TM == G::TN || col < p0; }

// a tile, times f, into the symmetric matrix D, and its mirror image
template <typename G>
__device__ __forceinline__ void put_symmetric(const f32x4 (&acc)[G::MR][G::NR], float f, const Mat& t, unsigned char* D, int p0, int q0,
                                              unsigned char* smem) {
  float* tile = reinterpret_cast<float*>(smem);
  const int mp = up32(t.m);
  to_lds<G>(acc, f, 0, p0, q0, t.m, t.m, tile);
  by_rows<G>(tile, [&](int p, int q, const float (&v)[8]) {
    if (p0 + p < t.m && q0 + q < mp && own<G>(p0, q0 + q)) store8(D + (int64_t)(p0 + p) * mp * 4, q0 + q, v);
  });
  if (q0 < p0)
    by_cols<G>(tile, [&](int q, int p, const float (&v)[8]) {
      if (q0 + q < t.m && p0 + p < mp && mirrored<G>(p0, q0 + q)) store8(D + (int64_t)(q0 + q) * mp * 4, p0 + p, v);
    });
}

// A = X X^T in slot 0, one triangle of tiles, stored on both sides of the diagonal.  The contraction over n is split where
// the tiles alone would not fill the chip: partial tiles go to the workspace, 16 x 16 blocks as they lie in the accumulators.
template <typename G>
__device__ __forceinline__ void gram_tile(const Mat& t, unsigned char* ws, int local, float f, int odd, unsigned char* smem) {
  const int nt = (t.m + G::TM - 1) / G::TM, tiles = nt * (nt + 1) / 2;
  const int split = local / tiles, tl = local % tiles;      // tiles of one split are neighbours: they share its columns of X
  int p0, q0;
  place<G>(tl, t.m, p0, q0);
  const int KB = up32(t.n) >> 5, kb0 = split * t.kc, kb1 = kb0 + t.kc < KB ? kb0 + t.kc : KB;
  const unsigned char* X = x_of(t, ws, odd);
  f32x4 acc[G::MR][G::NR];
  clear(acc);
  product<G>(acc, X, X, p0, q0, t.m, t.m, KB, kb0, kb1, smem);
  if (t.ks > 1) {
    f32x4* part = part_of(t, ws) + (int64_t)(tl * t.ks + split) * (G::TM * G::TN / 4);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int r = 0; r < G::MR; ++r)
#pragma unroll
      for (int c = 0; c < G::NR; ++c)
        part[(((wave / G::WN) * G::MR + r) * (G::TN / 16) + (wave % G::WN) * G::NR + c) * 64 + lane] = acc[r][c];
    return;
  }
  put_symmetric<G>(acc, f, t, slot_of(t, ws, 0), p0, q0, smem);
}

template <typename G>
__global__ __launch_bounds__(G::THREADS, G::PER_CU * G::W / 4) void ortho_gram_kernel(Work a, float f, int odd) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  int local;
  const Mat t = find_mat(a, GRAM, local);
  gram_tile<G>(t, a.ws, local, f, odd, smem);
}

// Adds the partial tiles of A, a workgroup per 32 x 32 block, in the order of the splits.  Bound by memory: 8 us for the
// 33 MB of 1024 x 9216, 4.1 TB/s.
template <typename G>
__global__ __launch_bounds__(256) void ortho_join_kernel(Work a, float f) {
  constexpr int B = G::TN / 32, BB = (G::TM / 32) * B;
  __shared__ float tile[32 * 34];
  int local, p0, q0;
  const Mat t = find_mat(a, JOIN, local);
  const int tl = local / BB, sub = local % BB;
  place<G>(tl, t.m, p0, q0);
  const bool diagonal = p0 == q0;
  p0 += (sub / B) * 32;
  q0 += (sub % B) * 32;
  const int mp = up32(t.m);
  if (p0 >= mp || q0 >= mp) return;
  // the four 16 x 16 blocks (r, c) of this one, a wave each
  const int r16 = (sub / B) * 2 + (threadIdx.x >> 7), c16 = (sub % B) * 2 + (threadIdx.x >> 6 & 1), lane = threadIdx.x & 63;
  const f32x4* part = part_of(t, a.ws) + (int64_t)tl * t.ks * (G::TM * G::TN / 4) + (r16 * (G::TN / 16) + c16) * 64 + lane;
  f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int k = 0; k < t.ks; ++k) s += part[(int64_t)k * (G::TM * G::TN / 4)];
  const int pr = (r16 & 1) * 16 + 4 * (lane >> 4), qc = (c16 & 1) * 16 + (lane & 15);
#pragma unroll
  for (int e = 0; e < 4; ++e) tile[(pr + e) * 34 + qc] = p0 + pr + e < t.m && q0 + qc < t.m ? s[e] * f : 0.f;
  __syncthreads();
  unsigned char* A = slot_of(t, a.ws, 0);
  const int id = threadIdx.x & 127, r = id >> 2, c = (id & 3) * 8;
  float v[8];
  if (threadIdx.x < 128) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[r * 34 + c + e];
    if (p0 + r < t.m) store8(A + (int64_t)(p0 + r) * mp * 4, q0 + c, v);
  } else if (!diagonal) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[(c + e) * 34 + r];
    if (q0 + r < t.m) store8(A + (int64_t)(q0 + r) * mp * 4, p0 + c, v);
  }
}

// The m x m matrices of one group of steps live in slots of the workspace; all are polynomials in A, so they are symmetric
// and commute, and one triangle of tiles is computed and stored on both sides.
//   D = ca I + cb C + cc P Q of the stored (scaled) numbers; C is not read where ca and cb are 0.  D is none of the others.
template <typename G>
__device__ __forceinline__ void square_tile(const Mat& t, unsigned char* ws, int local, const Op& op, unsigned char* smem) {
  int p0, q0;
  place<G>(local, t.m, p0, q0);
  const int mp = up32(t.m), KB = mp >> 5;
  const unsigned char* C = slot_of(t, ws, op.sc);
  unsigned char* D = slot_of(t, ws, op.sd);
  f32x4 acc[G::MR][G::NR];
  clear(acc);
  product<G>(acc, slot_of(t, ws, op.sp), slot_of(t, ws, op.sq), p0, q0, t.m, t.m, KB, 0, KB, smem);
  if (op.ca == 0.f && op.cb == 0.f) {
    put_symmetric<G>(acc, op.cc, t, D, p0, q0, smem);
    return;
  }
  float* tile = reinterpret_cast<float*>(smem);
  to_lds<G>(acc, op.cc, 0, p0, q0, t.m, t.m, tile);
  auto put = [&](int r, int c, const float (&v)[8]) {        // eight numbers of row r from column c on
    if (r >= t.m || c >= mp) return;
    float w[8];
    load8(C + (int64_t)r * mp * 4, c, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = v[e] + op.cb * w[e] + (r == c + e ? op.ca : 0.f);
    store8(D + (int64_t)r * mp * 4, c, w);
  };
  by_rows<G>(tile, [&](int p, int q, const float (&v)[8]) {
    if (own<G>(p0, q0 + q)) put(p0 + p, q0 + q, v);
  });
  if (q0 < p0)
    by_cols<G>(tile, [&](int q, int p, const float (&v)[8]) {
      if (mirrored<G>(p0, q0 + q)) put(q0 + q, p0 + p, v);
    });
}

// one or two operations that do not depend on each other: gridDim.y of them
template <typename G>
__global__ __launch_bounds__(G::THREADS, G::PER_CU * G::W / 4) void ortho_square_kernel(Work a, Op first, Op second) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  int local;
  const Mat t = find_mat(a, SQUARE, local);
  square_tile<G>(t, a.ws, local, blockIdx.y ? second : first, smem);
}

// eight consecutive results at (r, c) of the source's orientation, as many as lie within `cols`: 16-byte accesses of any
// alignment, single elements at the row's end
template <typename T, bool MUON>
__device__ __forceinline__ void finish8(const Mat& t, int r, int c, int cols, const float (&v)[8], const MuonArgs& u) {
  T* o = static_cast<T*>(t.out) + (int64_t)r * t.ldo + c;
  if (c + 8 <= cols) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        F4 w;
        if (MUON) w = *reinterpret_cast<const F4*>(o + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) w.f[e] = MUON ? w.f[e] * u.decay - t.step * v[4 * h + e] : v[4 * h + e];
        *reinterpret_cast<F4*>(o + 4 * h) = w;
      }
    } else {
      H8 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w.u[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
      *reinterpret_cast<H8*>(o) = w;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (c + e < cols) {
      if (MUON) o[e] = (T)((float)o[e] * u.decay - t.step * v[e]);
      else o[e] = (T)v[e];
    }
}

// Q X with Q from slot sq: the next group's X, or the result.  Tiles of a column panel of X are neighbours.
template <typename G, typename T, bool LAST, bool MUON>
__device__ __forceinline__ void apply_tile(const Mat& t, unsigned char* ws, int local, const MuonArgs& u, int sq, float f, int odd,
                                           unsigned char* smem) {
  const int np = up32(t.n), KB = up32(t.m) >> 5;
  const int tp = (t.m + G::TM - 1) / G::TM, p0 = (local % tp) * G::TM, q0 = (local / tp) * G::TN;
  f32x4 acc[G::MR][G::NR];
  clear(acc);
  product<G, true>(acc, slot_of(t, ws, sq), x_of(t, ws, odd), p0, q0, t.m, t.n, KB, 0, KB, smem, t.m, np >> 5);
  float* tile = reinterpret_cast<float*>(smem);
  unsigned char* X = x_of(t, ws, odd ^ 1);
#pragma unroll
  for (int h = 0; h < G::TM / G::SLAB; ++h) {
    const int ph = p0 + h * G::SLAB;
    if (ph >= t.m) break;
    if (h) __syncthreads();
    to_lds<G>(acc, f, h, p0, q0, t.m, t.n, tile);
    if (!LAST)
      by_rows<G>(tile, [&](int p, int q, const float (&v)[8]) {
        if (ph + p < t.m && q0 + q < np) store8(X + (int64_t)(ph + p) * np * 4, q0 + q, v);
      });
    else if (!t.flip)
      by_rows<G>(tile, [&](int p, int q, const float (&v)[8]) {
        if (ph + p < t.m && q0 + q < t.n) finish8<T, MUON>(t, ph + p, q0 + q, t.n, v, u);
      });
    else
      by_cols<G>(tile, [&](int q, int p, const float (&v)[8]) {
        if (q0 + q < t.n && ph + p < t.m) finish8<T, MUON>(t, q0 + q, ph + p, t.m, v, u);
      });
  }
}

template <typename G, typename T, bool LAST, bool MUON>
__global__ __launch_bounds__(G::THREADS, G::PER_CU * G::W / 4) void ortho_apply_kernel(Work a, MuonArgs u, int sq, float f,
                                                             int odd) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  int local;
  const Mat t = find_mat(a, APPLY, local);
  apply_tile<G, T, LAST, MUON>(t, a.ws, local, u, sq, f, odd, smem);
}

// ------------------------------------------------------------------------------------------------ few rows
// a value in memory, the same for all lanes, in scalar registers
template <typename V>
__device__ __forceinline__ V uniform(const V* p) {
  static_assert(sizeof(V) % 4 == 0, "whole words");
  union { V v; int w[sizeof(V) / 4]; } u;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / 4); ++i) u.w[i] = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(p)[i]);
  return u.v;
}
// kernel arguments into LDS, all at once
template <typename V>
__device__ __forceinline__ void keep(V* lds, const V& arg) {
  for (int i = threadIdx.x; i < (int)(sizeof(V) / 4); i += blockDim.x) reinterpret_cast<int*>(lds)[i] = reinterpret_cast<const int*>(&arg)[i];
}

// A program from the kernel's arguments, an operation to a lane: read once, and the next one is a few lane reads away.
struct Ops {
  int w[sizeof(Op) / 4];
  __device__ __forceinline__ explicit Ops(const Program& p) {
    const int lane = threadIdx.x & 63;
    const int* from = reinterpret_cast<const int*>(&p.op[lane < MAX_OPS ? lane : 0]);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Op) / 4); ++i) w[i] = from[i];
  }
  __device__ __forceinline__ Op operator[](int k) const {
    union { Op op; int v[sizeof(Op) / 4]; } u;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Op) / 4); ++i) u.v[i] = __builtin_amdgcn_readlane(w[i], k);
    return u.op;
  }
};
static_assert(MAX_OPS <= 64 && sizeof(Op) % 4 == 0, "an operation to a lane");

// Up to 64 rows the m x m matrices stay in LDS, 16 KB each: slot k, 32-column block b, row r, 16-byte chunks as in the
// stages of product().  A workgroup computes the whole 64 x 64 product, and a lane's four rows of one column are, by
// symmetry (of X X^T and A A^T, up to rounding), four columns of one row: they go back without any transposition.  An operation takes 0.9 us this way (1.2 with
// four waves), 2.7 us through global memory.
constexpr int SLOT64 = 64 * 2 * 128;

constexpr int THREADS64 = 1024;      // 16 waves, a 16 x 16 block each: what counts is how soon each is done

struct Lane64 {
  int wm, wn, r, g, fro[2];      // the wave's block of columns and of rows
  int at[2];                     // byte of this lane's four numbers, [half], within a slot
  int col, row;                  // of the first of them
  __device__ __forceinline__ Lane64() {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), turn = (lane >> 1) & 7;
    wm = wave >> 2; wn = wave & 3; r = lane & 15; g = lane >> 4;
    col = wm * 16 + 4 * g; row = wn * 16 + r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      fro[h] = r * 128 + (((h * 4 + g) ^ turn) * 16);
      at[h] = (wm >> 1) * 8192 + wn * 2048 + r * 128 + ((((wm & 1) * 2 + (g >> 1)) + 4 * h) ^ turn) * 16 + (g & 1) * 8;
    }
  }
};

// a lane's four numbers in a matrix C
struct Old64 { f16x4 hi, lo; };

// D = ca I + cb C + cc acc into slot D.  What lies outside m x m is zero in C and in acc, and stays zero.
__device__ __forceinline__ void put64(const f32x4& acc, float ca, float cb, float cc, int m, unsigned char* D, const Old64& C,
                                      const Lane64& L) {
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = cc * acc[e];
  if (cb != 0.f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fmaf((float)C.lo[e], cb, fmaf((float)C.hi[e], cb, v[e]));
  }
  if (ca != 0.f && L.wm == L.wn) {         // a block on the diagonal
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += L.row == L.col + e && L.row < m ? ca : 0.f;
  }
  f16x4 hi, lo;
  split4(v, hi, lo);
  *reinterpret_cast<f16x4*>(D + L.at[0]) = hi;
  *reinterpret_cast<f16x4*>(D + L.at[1]) = lo;
}
__device__ __forceinline__ void lds_done() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}
// 32 columns of both operands, [half]
struct Block64 { f16x8 p[2], q[2]; };
__device__ __forceinline__ void multiply64(f32x4& acc, const Block64& f) {
#pragma unroll
  for (int w = 0; w < 3; ++w) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.p[w == 2], f.q[w == 1], acc, 0, 0, 0);
}
// P Q^T over nb 32-column blocks of two matrices of 64 rows in LDS; a block is read while the one before is multiplied
__device__ __forceinline__ f32x4 product64(const unsigned char* P, const unsigned char* Q, int nb, const Lane64& L) {
  P += L.wm * 2048;
  Q += L.wn * 2048;
  auto load = [&](Block64& f, int b) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f.p[h] = *reinterpret_cast<const f16x8*>(P + b * 8192 + L.fro[h]);
      f.q[h] = *reinterpret_cast<const f16x8*>(Q + b * 8192 + L.fro[h]);
    }
  };
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  Block64 one, two;
  load(one, 0);
  int b = 0;
  for (; b + 1 < nb; b += 2) {
    load(two, b + 1);
    multiply64(acc, one);
    if (b + 2 < nb) load(one, b + 2);
    multiply64(acc, two);
  }
  if (b < nb) multiply64(acc, one);
  return acc;
}
// the polynomial of A in slot 0 into slot 1
__device__ __forceinline__ void polynomial64(const Op& op, int m, unsigned char* slots, const Lane64& L) {
  Old64 old{};
  if (op.cb != 0.f) {
    old.hi = *reinterpret_cast<const f16x4*>(slots + L.at[0]);
    old.lo = *reinterpret_cast<const f16x4*>(slots + L.at[1]);
  }
  const f32x4 acc = product64(slots, slots, up32(m) >> 5, L);
  put64(acc, op.ca, op.cb, op.cc, m, slots + SLOT64, old, L);
  lds_done();
}

// A step's polynomial P = ca I + cb A + cc A^2 for matrices of up to 64 rows, a workgroup each, from the parts of A = X X^T.
__global__ __launch_bounds__(THREADS64) void ortho_few_kernel(Work a, float f, Op op) {
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * SLOT64];
  const Mat t = a.count > 1 ? uniform(&reinterpret_cast<const Mats*>(a.ws)->mat[blockIdx.x]) : a.only;
  const Lane64 L;
  const int m = t.m, nb = up32(m) >> 5;
  unsigned char* A = slot_of(t, a.ws, op.sp);
  if (t.ks > 1) {
    // the partial tiles of A, in the order of the splits
    const f32x4* part = part_of(t, a.ws) + threadIdx.x;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int k = 0; k < t.ks; ++k) acc += part[k * (64 * 64 / 4)];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = L.col + e < m && L.row < m ? acc[e] : 0.f;      // rows past the last repeat it
    put64(acc, 0.f, 0.f, f, m, smem, Old64{}, L);
  } else {
    for (int id = threadIdx.x; id < 64 * nb * 8; id += THREADS64) {
      const int r = id / (nb * 8), b = (id >> 3) % nb, c = id & 7;
      const uint4 v = r < m ? *reinterpret_cast<const uint4*>(A + ((int64_t)r * nb + b) * 128 + c * 16) : make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(smem + b * 8192 + r * 128 + (c ^ ((r >> 1) & 7)) * 16) = v;
    }
  }
  __syncthreads();
  polynomial64(op, m, smem, L);
  unsigned char* P = slot_of(t, a.ws, op.sd);
  for (int id = threadIdx.x; id < m * nb * 8; id += THREADS64) {
    const int r = id / (nb * 8), b = (id >> 3) % nb, c = id & 7;
    *reinterpret_cast<uint4*>(P + ((int64_t)r * nb + b) * 128 + c * 16) =
        *reinterpret_cast<const uint4*>(smem + SLOT64 + b * 8192 + r * 128 + (c ^ ((r >> 1) & 7)) * 16);
  }
}

// The whole call for small matrices, a workgroup each and a single launch: here the time of a launch, and of the latencies
// behind it, is all there is to save.  X lives in LDS too, as 32-column blocks of 64 rows in the layout of the slots; Q X
// replaces it 64 columns at a time, each depending on themselves only.  As many columns as LDS holds beside A and P: 64 x 256
// takes 35 us this way and 65 in the launches of FEW, 64 x 448 54 and 65, eight of them 55 and 77.
constexpr int SMALL_N = 448, SMALL_LDS = (2 + SMALL_N / 64) * SLOT64;

// columns 64 c .. of X <- f Q X, or the result.  The operands trade sides, D[j][i] = sum_k X[k][j] Q[i][k]: a lane then has
// four columns of one row of the result.
template <typename T, bool MUON>
__device__ __forceinline__ void apply64(const Mat& t, unsigned char* X, const unsigned char* Q, int c, float f, bool last,
                                        const MuonArgs& u, const Lane64& L) {
  const int lane = threadIdx.x & 63, m = t.m, n = t.n, nb = up32(m) >> 5, KB = up32(n) >> 5;
  X += c * SLOT64;
  // transposing reads: k-row 8 g + t (+ 4), columns 4 q ..; the chunk a row holds them in: base ^ 4 half ^ 2 (side ^ upper four)
  const int tt = lane >> 2 & 3, cq = lane & 3, base = (cq >> 1) ^ (4 * (L.g & 1) + (tt >> 1));
  const bool past = 2 * c + (L.wm >> 1) >= KB;
  const unsigned char* row = X + (past ? 0 : L.wm >> 1) * 8192 + (8 * L.g + tt) * 128 + (cq & 1) * 8;
  auto load = [&](Block64& in, int b) {
    const unsigned char* at = row + b * 4096;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      typedef __attribute__((ext_vector_type(8))) short short8v;
      const int side = 2 * (L.wm & 1);
      const short4v a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) short4v*)(at + (base ^ (4 * h) ^ side) * 16));
      const short4v a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) short4v*)(at + 512 + (base ^ (4 * h) ^ (side ^ 2)) * 16));
      in.p[h] = __builtin_bit_cast(f16x8, short8v{a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]});
      in.q[h] = *reinterpret_cast<const f16x8*>(Q + b * 8192 + L.wn * 2048 + L.fro[h]);
    }
  };
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  Block64 one, two;
  load(one, 0);
  if (nb > 1) load(two, 1);
  multiply64(acc, one);
  if (nb > 1) multiply64(acc, two);
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = acc[e] * f;
  lds_done();                                                 // every wave has read the old columns
  if (past) return;
  if (!last) {
    f16x4 hi, lo;
    split4(v, hi, lo);
    *reinterpret_cast<f16x4*>(X + L.at[0]) = hi;
    *reinterpret_cast<f16x4*>(X + L.at[1]) = lo;
    return;
  }
  const int col = c * 64 + L.col;
  if (L.row >= m) return;
  T* o = static_cast<T*>(t.out) + (t.flip ? (int64_t)col * t.ldo + L.row : (int64_t)L.row * t.ldo + col);
  const int64_t next = t.flip ? t.ldo : 1;
  float old[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) old[e] = MUON && col + e < n ? (float)o[e * next] : 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < n) o[e * next] = MUON ? (T)(old[e] * u.decay - t.step * v[e]) : (T)v[e];
}

template <typename T, bool MUON>
__global__ __launch_bounds__(THREADS64) void ortho_small_kernel(Mats a, MuonArgs u, float eps, float scale, Program prog) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ double red[16];
  __shared__ Mat mine;
  const Ops ops(prog);
  keep(&mine, a.mat[blockIdx.x]);
  __syncthreads();
  const Mat t = uniform(&mine);
  unsigned char* X = smem + 2 * SLOT64;
  const Lane64 L;
  const int m = t.m, n = t.n, KB = up32(n) >> 5;
  // the matrix, eight elements at a time, stays in registers until its norm is known
  constexpr int MOST = (64 * SMALL_N / 8 + THREADS64 - 1) / THREADS64;
  const int rows = t.flip ? n : m, cols = t.flip ? m : n, c8 = (cols + 7) >> 3, chunks = rows * c8;
  const T* x = static_cast<const T*>(t.x);
  float v[MOST][8];
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    const int id = k * THREADS64 + threadIdx.x, r = id / c8, c = (id - r * c8) * 8;
    float mo[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[k][e] = mo[e] = 0.f;
    if (id < chunks) {
      const T* p = x + (int64_t)r * t.ldx + c;
      float* q = MUON ? t.mom + (int64_t)r * cols + c : nullptr;
      if (c + 8 <= cols) {
        read8(p, v[k]);
        if (MUON) read8(q, mo);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < cols) {
            v[k][e] = (float)p[e];
            if (MUON) mo[e] = q[e];
          }
      }
      if (MUON) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[k][e] *= u.grad_scale;
          mo[e] = u.momentum * mo[e] + (1.f - u.momentum) * v[k][e];
          if (c + e < cols) q[e] = mo[e];
          v[k][e] = direction(v[k][e], mo[e], u);
        }
      }
    }
  }
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < MOST; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) s += (double)v[k][e] * (double)v[k][e];
  const double f = start_factor(block_sum(s, red), eps, scale);
  for (int i = threadIdx.x; i < KB * 512; i += THREADS64) reinterpret_cast<uint4*>(X)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    const int id = k * THREADS64 + threadIdx.x, r = id / c8, c = (id - r * c8) * 8;
    if (id >= chunks) continue;
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = (float)(f * (double)v[k][e]);
    uint4 hi, lo;
    split8(w, hi, lo);
    if (!t.flip) {      // row r, columns c ..: two chunks of 16 bytes (zeros past the end)
      unsigned char* p = X + (c >> 5) * 8192 + r * 128;
      const int turn = (r >> 1) & 7, q = (c & 31) >> 3;
      *reinterpret_cast<uint4*>(p + (q ^ turn) * 16) = hi;
      *reinterpret_cast<uint4*>(p + ((q + 4) ^ turn) * 16) = lo;
    } else {            // rows c .., column r
      const unsigned hs[4] = {hi.x, hi.y, hi.z, hi.w}, ls[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < cols) {
          unsigned char* p = X + (r >> 5) * 8192 + (c + e) * 128 + (r & 7) * 2;
          const int turn = ((c + e) >> 1) & 7, q = (r & 31) >> 3;
          *reinterpret_cast<unsigned short*>(p + (q ^ turn) * 16) = (unsigned short)(hs[e >> 1] >> (16 * (e & 1)));
          *reinterpret_cast<unsigned short*>(p + ((q + 4) ^ turn) * 16) = (unsigned short)(ls[e >> 1] >> (16 * (e & 1)));
        }
    }
  }
  __syncthreads();
  for (int k = 0; k < prog.n; ++k) {
    const Op op = ops[k];
    if (op.kind == K_GRAM) {
      put64(product64(X, X, KB, L), 0.f, 0.f, op.cc, m, smem, Old64{}, L);
      lds_done();
    } else if (op.kind == K_SQUARE) {
      polynomial64(op, m, smem, L);
    } else {
      for (int c = 0; c * 64 < n; ++c) apply64<T, MUON>(t, X, smem + SLOT64, c, op.cc, op.last, u, L);
      lds_done();
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
constexpr int MAX_STEPS = 32;

// Powers of two for the stored numbers of each step, from bounds on the spectral norms: |X_0| <= 1, and over singular values
// s in [0, r] the next bound is max |s p(s^2)| with p(l) = a + b l + c l^2; A's numbers are within r^2, B's within max |p|.
struct Scales { double x[MAX_STEPS + 1], a[MAX_STEPS], pa[MAX_STEPS], p[MAX_STEPS], pmax[MAX_STEPS]; };

double pow2_for(double bound) { return ldexp(1.0, (int)floor(log2(60000.0 / bound))); }

bool ortho_scales(const float* coeff, int steps, Scales* s) {
  double r = 1.0;
  for (int k = 0; k <= steps; ++k) {
    if (!(r <= 1024.0)) return false;
    if (r < 1e-3) r = 1e-3;
    s->x[k] = pow2_for(r);
    if (k == steps) break;
    const double a = coeff[3 * k], b = coeff[3 * k + 1], c = coeff[3 * k + 2];
    // p(l), s p(s^2) and l p(l) over l = s^2 in [0, r^2]: the ends, and where their derivatives vanish
    double pm = 1e-3, xm = 0.0, am = 1e-3;
    auto look = [&](double l) {
      if (!(l >= 0.0 && l <= r * r)) return;
      const double p = fabs(a + b * l + c * l * l);
      pm = fmax(pm, p);
      xm = fmax(xm, sqrt(l) * p);
      am = fmax(am, l * p);
    };
    auto roots = [&](double q, double h, double w) {       // q l^2 + h l + w = 0
      if (q == 0.0) {
        if (h != 0.0) look(-w / h);
        return;
      }
      const double d = h * h - 4.0 * q * w;
      if (d < 0.0) return;
      look((-h + sqrt(d)) / (2.0 * q));
      look((-h - sqrt(d)) / (2.0 * q));
    };
    if (!(fabs(a) + fabs(b) + fabs(c) < 1e6)) return false;
    look(0.0);
    look(r * r);
    roots(0.0, 2.0 * c, b);
    roots(5.0 * c, 3.0 * b, a);
    roots(3.0 * c, 2.0 * b, a);
    if (!(pm <= 4096.0)) return false;
    s->pmax[k] = pm * 1.01;
    s->a[k] = pow2_for(r * r);
    s->pa[k] = pow2_for(am * 1.01);
    s->p[k] = pow2_for(s->pmax[k]);
    r = xm * 1.001;       // (rounding; more would grow through steps such as s^5, which stay within 1)
  }
  return true;
}

// How a run is done.  GENERAL: every product a launch over all its tiles.  FEW: up to 64 rows, where one workgroup adds the
// parts of X X^T and makes a step's polynomial of it.  SMALL: one launch for everything.
enum Mode { GENERAL, FEW, SMALL };

struct Plan {
  Mode mode;
  int wg, wp, wa;              // tiles of the three kinds of products: 64 and 128 square, 96 x 64, 128 x 160
  int group;                   // steps taken together
  int64_t bytes, norms;        // of the workspace; where the partial sums of squares begin
};

int tri(int m, int T) { const int n = cdiv(m, T); return n * (n + 1) / 2; }
// tiles of an m x m product by the rows of a tile: 64 or 128 (square), or 96 (by 64)
int square_tiles(int m, int T) {
  if (T != 96) return tri(m, T);
  int n = 0;
  for (int i = 0; 96 * i < m; ++i) {
    const int end = 96 * (i + 1) < m ? 96 * (i + 1) : m;
    n += cdiv(end, 64);
  }
  return n;
}

// Steps in groups: with A = X X^T a step multiplies X by P = a I + b A + c A^2, and the next A is P A P.  Three steps then cost
// one product each way with X and nine with m x m matrices instead of three each way and three.  That pays where n >= 2 m:
// 1024 x 9216 takes 708 us in single steps, 557 in twos, 481 in threes (with the tiles of that time).
// Its price is rounding: A is not taken anew from X, so directions far below the largest lose digits, the more the fewer there
// are to share the error.  Largest error against float64, over that of single steps with float32 products, of twelve kinds of
// spectra: single steps 3.6 (3 x 9), 2.7 (8 x 72), 1.5 to 1.6 (from 36 x 324 to 1024 x 9216); threes 4.0 (65 x 200), 3.1
// (80 x 170), 2.6 (100 x 300), 2.2 (128 x 300), 2.0 (512 x 1100), 2.2 (1024 x 9216), but 6 to 33 up to 64 rows (emulated).  So: threes from
// m = 128 on, else single steps, whatever the type.
bool in_threes(const Mat& t) { return t.m >= 128 && t.n >= 2 * t.m; }

// the matrices of a call in one run or two
struct Parts {
  int count;
  Mats list[2];
  int group[2];      // steps taken together
};
// A list with both kinds is two runs where the threes save more than the twenty launches of a second run cost, in multiplications
// of halves; else all go in single steps.  Muon for the 17 filters of a model, two runs and one (us): 0.6e10 saved 228 and 138,
// 3.3e10 299 and 247, 7.0e10 350 and 348, 9.6e10 381 and 400, 4.0e11 798 and 1017.
constexpr double RUN_PRODUCTS = 7e10;
void split(const Mats& a, Parts& s) {
  double saved = 0.0;
  int threes = 0;
  for (int i = 0; i < a.count; ++i) {
    const double m = a.mat[i].m, n = a.mat[i].n;
    if (in_threes(a.mat[i])) {
      ++threes;
      saved += 3.0 * m * m * (9.0 * n - 8.0 * m);
    }
  }
  const bool both = threes && threes < a.count && saved >= RUN_PRODUCTS;
  s.count = both ? 2 : 1;
  s.group[0] = both || threes == a.count ? 3 : 1;
  s.group[1] = 1;
  for (int k = 0; k < s.count; ++k) {
    Mats& l = s.list[k];
    l.count = 0;
    l.ws = a.ws;
    for (int i = 0; i < a.count; ++i)
      if (!both || in_threes(a.mat[i]) == (k == 0)) l.mat[l.count++] = a.mat[i];
  }
}

// Places the workspace, chooses mode, tiles and splits, and counts workgroups.
void make_plan(Mats& a, Plan& p, int steps, int group) {
  int64_t apply = 0, grams = 0;
  int mmax = 0, nmax = 0;
  for (int i = 0; i < a.count; ++i) {
    const Mat& t = a.mat[i];
    grams += tri(t.m, 128) * cdiv64(up32(t.n) >> 5, 8);
    apply += (int64_t)cdiv(t.m, 128) * cdiv(t.n, 128);
    mmax = t.m > mmax ? t.m : mmax;
    nmax = t.n > nmax ? t.n : nmax;
  }
  p.group = group;
  p.mode = GENERAL;
  if (mmax <= 64) p.mode = nmax <= SMALL_N && 3 * steps <= MAX_OPS ? SMALL : FEW;
  // Few tiles: 64 x 64, to occupy CUs; fewer than 256 of 128 x 128 are few (Q X of 333 x 1000, 24: 13.5 us against 6.6).
  // X X^T splits its contraction, at least eight blocks to a workgroup: 512 x 4608, 180 workgroups of 128 x 128, 12.1 us
  // against 9.8, but 1024 x 9216, 512 of them, 32 against 41.  From 256 on 128 rows, and for Q X the width whose rounds of 512
  // workgroups make the least work: 9216 columns by 1024 rows are 576 tiles of 128 columns, two rounds, but 464 of 160, one.
  p.wg = mmax > 64 && grams >= 256 ? 128 : 64;
  p.wp = 64;
  if (p.mode == GENERAL) {
    // Products of m x m matrices take as long as the CU with the most tiles.  In units of a 64 x 64 tile, one of 96 x 64 takes
    // 1.5, one of 128 x 128 3.7, and two of these, that share a CU, 5.9; a tile of a smaller matrix counts by its share of the
    // longest contraction.  Whole calls of m x 2 m with 64, 96, 128 rows (us): m = 1100 283, 296, 508; 1409 475, 425, 665;
    // 1800 654, 692, 867; 2200 1133, 1047, 1242; 2750 1859, 1922, 1747; 3700 4192, 4038, 3568; 4096 6168, 5649, 6020.
    double n64 = 0.0, n96 = 0.0, n128 = 0.0;
    for (int i = 0; i < a.count; ++i) {
      const double share = (double)a.mat[i].m / mmax;
      n64 += square_tiles(a.mat[i].m, 64) * share;
      n96 += square_tiles(a.mat[i].m, 96) * share;
      n128 += square_tiles(a.mat[i].m, 128) * share;
    }
    const double c64 = ceil(n64 / 256), c96 = 1.5 * ceil(n96 / 256), left = fmod(n128, 512.0);
    const double c128 = 5.9 * floor(n128 / 512) + (left > 256.0 ? 5.9 : left > 0.0 ? 3.7 : 0.0);
    p.wp = c128 <= c96 && c128 <= c64 ? 128 : c96 <= c64 ? 96 : 64;
  }
  p.wa = apply >= 256 ? 128 : 64;
  if (apply >= 256) {
    int64_t wide = 0;
    for (int i = 0; i < a.count; ++i) wide += (int64_t)cdiv(a.mat[i].m, 128) * cdiv(a.mat[i].n, 160);
    if (cdiv64(wide, 512) * 160 < cdiv64(apply, 512) * 128) p.wa = 160;
  }
  const int T = p.wg, AM = p.wa == 64 ? 64 : 128, AN = p.wa;
  int64_t work = 0;
  for (int i = 0; i < a.count; ++i) work += (int64_t)tri(a.mat[i].m, T) * (up32(a.mat[i].n) >> 5);
  // k-blocks per workgroup so that as many as the chip holds at once share the whole contraction evenly; at least 8.
  const int64_t round = 512;
  int64_t kc = cdiv64(work, round);
  if (kc < 8) kc = 8;
  for (;; ++kc) {        // each matrix rounds up: not more than one round in all
    int64_t n = 0;
    for (int i = 0; i < a.count; ++i) n += tri(a.mat[i].m, T) * cdiv64(up32(a.mat[i].n) >> 5, kc);
    if (n <= round || kc >= 4 * cdiv64(work, round)) break;
  }
  int64_t off = (sizeof(Mats) + 255) & ~(int64_t)255;
  int norms = 0;
  for (int i = 0; i < a.count; ++i) {
    Mat& t = a.mat[i];
    const int64_t KB = up32(t.n) >> 5;
    t.normc = (int)cdiv64((int64_t)t.m * t.n, NORM_CHUNK);
    t.norm0 = norms;
    norms += t.normc;
    int64_t k = kc;
    // A block takes 0.2 us, and about as long a part to be added, where few workgroups do it: their sum is least with
    // sqrt(KB) of each; tiles of 128 have more workgroups to add them, and longer blocks.  64 x 9216: 62 us with 16 parts, 71
    // with 8, 66 with 24; 64 x 131072: 171 with 64, 287 with 512; 100 x 131072: 282 with 128, 375 with 512.
    const int64_t least = (int64_t)ceil(sqrt((double)KB) * (T == 128 ? 0.5 : 1.0));
    if (k < least) k = least;
    t.kc = (int)(p.mode == SMALL || k > KB ? KB : k);
    t.ks = (int)cdiv64(KB, t.kc);
    t.at = off;
    off += 2 * size_x(t) + SLOTS * size_slot(t);
    if (t.ks > 1) off += (int64_t)tri(t.m, T) * t.ks * T * T * 4;
    off = (off + 255) & ~(int64_t)255;
    const int B = (T / 32) * (T / 32);
    const int64_t n[PHASES] = {t.normc, (int64_t)cdiv(t.m, 64) * cdiv(t.n, 64), (int64_t)tri(t.m, T) * t.ks,
                               t.ks > 1 ? (int64_t)tri(t.m, T) * B : 0, square_tiles(t.m, p.wp),
                               (int64_t)cdiv(t.m, AM) * cdiv(t.n, AN)};
    for (int k2 = 0; k2 < PHASES; ++k2) a.end[k2][i] = (int)n[k2] + (i ? a.end[k2][i - 1] : 0);
  }
  p.norms = off;
  p.bytes = off + 8 * (int64_t)norms;
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

// A call in flight: the copy of the matrices in the workspace, grid sizes and the stream
struct Run {
  const Mats& a;
  const Plan& p;
  const MuonArgs& u;
  const char* what;
  hipStream_t st;
  unsigned grid(Phase k) const { return (unsigned)a.end[k][a.count - 1]; }
  Work work() const { return Work{a.ws, a.count, a.mat[0]}; }

  template <typename G>
  int gram(float f, int odd) const {
    ORTHO_TRY((ready<&ortho_gram_kernel<G>>(G::LDS, what)));
    ortho_gram_kernel<G><<<grid(GRAM), G::THREADS, G::LDS, st>>>(work(), f, odd);
    SNWS_LAUNCH_CHECK(what);
    if (p.mode == GENERAL && grid(JOIN)) {
      ortho_join_kernel<G><<<grid(JOIN), 256, 0, st>>>(work(), f);
      SNWS_LAUNCH_CHECK(what);
    }
    return SNWS_OK;
  }
  template <typename G>
  int squares(const Op& first, const Op* second) const {
    ORTHO_TRY((ready<&ortho_square_kernel<G>>(G::LDS, what)));
    ortho_square_kernel<G><<<dim3(grid(SQUARE), second ? 2 : 1), G::THREADS, G::LDS, st>>>(work(), first, second ? *second : first);
    SNWS_LAUNCH_CHECK(what);
    return SNWS_OK;
  }
  int few(float f, const Op& op) const {
    ortho_few_kernel<<<(unsigned)a.count, THREADS64, 0, st>>>(work(), f, op);
    SNWS_LAUNCH_CHECK(what);
    return SNWS_OK;
  }
  template <typename G, typename T, bool LAST, bool MUON>
  int apply_by(const Op& op, int odd) const {
    ORTHO_TRY((ready<&ortho_apply_kernel<G, T, LAST, MUON>>(G::LDS, what)));
    ortho_apply_kernel<G, T, LAST, MUON><<<grid(APPLY), G::THREADS, G::LDS, st>>>(work(), u, op.sq, op.cc, odd);
    SNWS_LAUNCH_CHECK(what);
    return SNWS_OK;
  }
  template <typename T, bool LAST, bool MUON>
  int apply(const Op& op, int odd) const {
    switch (p.wa) {
      case 160: return apply_by<Wide, T, LAST, MUON>(op, odd);
      case 128: return apply_by<Big, T, LAST, MUON>(op, odd);
      default: return apply_by<Fine, T, LAST, MUON>(op, odd);
    }
  }
  template <typename T, bool MUON>
  int small(const Program& prog, float eps, float scale) const {
    ORTHO_TRY((ready<&ortho_small_kernel<T, MUON>>(SMALL_LDS, what)));
    ortho_small_kernel<T, MUON><<<(unsigned)a.count, THREADS64, SMALL_LDS, st>>>(a, u, eps, scale, prog);
    SNWS_LAUNCH_CHECK(what);
    return SNWS_OK;
  }
};

// The operations of steps k .. k + g - 1; returns how many.  Stored numbers are true ones times a power of two: the factors
// turn a product of stored numbers into stored ones.
int group_ops(const float* coeff, const Scales& s, int k, int g, bool last, Op* op) {
  int n = 0;
  auto square = [&](int sp, int sq, int sd, double ca, double cb, double cc) {
    op[n++] = Op{K_SQUARE, (unsigned char)sp, (unsigned char)sq, (unsigned char)sp, (unsigned char)sd, 0, {0, 0}, (float)ca, (float)cb,
                 (float)cc};
  };
  op[n++] = Op{K_GRAM, 0, 0, 0, 0, 0, {0, 0}, 0.f, 0.f, (float)(s.a[k] / (s.x[k] * s.x[k]))};
  int A = 0, Q = 1, spare[4] = {2, 3, 4, 5};
  double qs = s.p[k], qmax = s.pmax[k];                  // scale of Q, bound of its numbers
  for (int j = k; j < k + g; ++j) {
    const int P = j == k ? Q : spare[0];
    square(A, A, P, (double)coeff[3 * j] * s.p[j], (double)coeff[3 * j + 1] * s.p[j] / s.a[j],
           (double)coeff[3 * j + 2] * s.p[j] / (s.a[j] * s.a[j]));
    const bool more = j + 1 < k + g;
    if (more) square(P, A, spare[2], 0.0, 0.0, s.pa[j] / (s.p[j] * s.a[j]));      // P A, and beside it
    if (j > k) {                                                                  // Q <- P Q
      qmax *= s.pmax[j];
      const double to = pow2_for(qmax);
      square(P, Q, spare[1], 0.0, 0.0, to / (s.p[j] * qs));
      const int old = Q;
      Q = spare[1];
      spare[1] = old;
      qs = to;
    }
    // A <- P (P A)^T, the next X X^T.  Rows by rows, so that it is P A P^T of the rounded P: with (P A) P^T in its place the
    // error grows tens of times.
    if (more) {
      square(P, spare[2], spare[3], 0.0, 0.0, s.a[j + 1] / (s.p[j] * s.pa[j]));
      const int old = A;
      A = spare[3];
      spare[3] = old;
    }
  }
  op[n++] = Op{K_APPLY, 0, (unsigned char)Q, 0, 0, last, {0, 0}, 0.f, 0.f, (float)((last ? 1.0 : s.x[k + g]) / (s.x[k] * qs))};
  return n;
}

template <typename T, bool MUON>
int run_all(const Mats& a, const Plan& p, const MuonArgs& u, const float* coeff, int steps, float eps, const Scales& s,
            const char* what, hipStream_t st) {
  const Run run{a, p, u, what, st};
  if (p.mode == SMALL) {
    Program prog{};
    for (int k = 0; k < steps;) {
      const int g = p.group < steps - k ? p.group : steps - k;
      prog.n += group_ops(coeff, s, k, g, k + g == steps, prog.op + prog.n);
      k += g;
    }
    return run.small<T, MUON>(prog, eps, (float)s.x[0]);
  }
  double* partial = reinterpret_cast<double*>(a.ws + p.norms);
  ortho_norm_kernel<T, MUON><<<run.grid(NORM), 256, 0, st>>>(a, u, partial);
  SNWS_LAUNCH_CHECK(what);
  ortho_start_kernel<T, MUON><<<run.grid(START), 256, 0, st>>>(run.work(), u, partial, eps, (float)s.x[0]);
  SNWS_LAUNCH_CHECK(what);
  int odd = 0;
  for (int k = 0; k < steps;) {
    const int g = p.group < steps - k ? p.group : steps - k;
    Op op[GROUP_OPS];
    const int n = group_ops(coeff, s, k, g, k + g == steps, op);
    ORTHO_TRY(p.wg == 128 ? run.gram<Big>(op[0].cc, odd) : run.gram<Fine>(op[0].cc, odd));
    if (p.mode == FEW) {
      ORTHO_TRY(run.few(op[0].cc, op[1]));
    } else {
      for (int i = 1; i + 1 < n; ++i) {
        // P A and P Q read the same matrices and write different ones: one launch for both
        const bool both = i + 2 < n && op[i].cb == 0.f && op[i + 1].cb == 0.f && op[i + 1].sp != op[i].sd && op[i + 1].sq != op[i].sd;
        const Op* second = both ? &op[i + 1] : nullptr;
        ORTHO_TRY(p.wp == 128 ? run.squares<Big>(op[i], second) : p.wp == 96 ? run.squares<Tall>(op[i], second)
                                                                             : run.squares<Fine>(op[i], second));
        if (both) ++i;
      }
    }
    k += g;
    const Op& ap = op[n - 1];
    ORTHO_TRY((ap.last ? run.apply<T, true, MUON>(ap, odd) : run.apply<float, false, false>(ap, odd)));
    odd ^= 1;
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

// runs use the workspace one after the other
int64_t bytes_of(const Mats& a, int steps) {
  Parts s;
  split(a, s);
  int64_t most = 0;
  for (int i = 0; i < s.count; ++i) {
    Plan p;
    make_plan(s.list[i], p, steps, s.group[i]);
    most = p.bytes > most ? p.bytes : most;
  }
  return most;
}

template <typename T, bool MUON>
int run_parts(Mats& a, const MuonArgs& u, const float* coeff, int steps, float eps, const Scales& scales, void* workspace,
              int64_t workspace_bytes, const char* what, hipStream_t st) {
  const int64_t need = bytes_of(a, steps);
  SNWS_CHECK_ARG(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0,
                 "%s: workspace of %lld bytes, 256-byte aligned, needed", what, (long long)need);
  a.ws = static_cast<unsigned char*>(workspace);
  Parts s;
  split(a, s);
  for (int i = 0; i < s.count; ++i) {
    Plan p;
    make_plan(s.list[i], p, steps, s.group[i]);
    ORTHO_TRY((run_all<T, MUON>(s.list[i], p, u, coeff, steps, eps, scales, what, st)));
  }
  return SNWS_OK;
}

}  // namespace

extern "C" int64_t snws_ortho_workspace_bytes(const int* rows, const int* cols, int count, int steps) {
  if (!rows || !cols || count < 1 || count > MAXM || steps < 1 || steps > MAX_STEPS) {
    snws_set_error("snws_ortho_workspace_bytes: 1 to %d matrices, 1 to %d steps", MAXM, MAX_STEPS);
    return -1;
  }
  Mats a{};
  a.count = count;
  for (int i = 0; i < count; ++i) {
    if (check_size(rows[i], cols[i], "snws_ortho_workspace_bytes") != SNWS_OK) return -1;
    set_shape(a.mat[i], rows[i], cols[i]);
  }
  return bytes_of(a, steps);
}

extern "C" int snws_orthogonalize(const snws_ortho_item* items, int count, int dtype, const float* coeff, int steps, float eps,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "snws_orthogonalize";
  SNWS_CHECK_ARG(dtype == SNWS_F32 || dtype == SNWS_BF16, "%s: dtype must be float32 or bfloat16", what);
  SNWS_CHECK_ARG(items && count >= 1 && count <= MAXM, "%s: 1 to %d matrices", what, MAXM);
  Scales s;
  ORTHO_TRY(check_common(coeff, steps, eps, &s, what));
  Mats a{};
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
  const MuonArgs u{};
  return dtype == SNWS_F32
             ? run_parts<float, false>(a, u, coeff, steps, eps, s, workspace, workspace_bytes, what, (hipStream_t)stream)
             : run_parts<bf16_t, false>(a, u, coeff, steps, eps, s, workspace, workspace_bytes, what, (hipStream_t)stream);
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
  const MuonArgs u{momentum, grad_scale, 1.f - weight_decay, nesterov};
  return run_parts<float, true>(a, u, coeff, steps, eps, s, workspace, workspace_bytes, what, (hipStream_t)stream);
}
