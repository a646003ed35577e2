// Layer normalisation over the last axis, forward: y = (x - mean) * rstd * weight + bias per row, mean and variance of the
// row's own C elements (the channels of one pixel in NHWC), rstd = 1 / sqrt(var + eps).
//
// Bound by memory: x is read once and y written once.  A row stays in registers between the two (ln.h), so the variance is
// taken around the mean in a second sweep over registers, in float32.  A float32 sum of C elements is off by some roundings of
// the mean, which for a row far from zero is no small part of its spread: a constant row of 1000.1 came out as up to 0.4
// instead of 0 (512 to 16384 elements).  So the second sweep also adds up the distances to that mean - exact numbers, where the
// row is far from zero - and their mean corrects it.  The bfloat16 elements of such a row are multiples of one unit, at most 2^9
// of it each: up to 2^15 of them, as many as the registers take, add exactly in float32, and there is nothing to correct.
// Measured: 262144 x 64 bfloat16 11.6 us (5.8 TB/s), 1048576 x 320 bfloat16 222 us (6.0 TB/s), 997 x 9216 float32 17.1 us
// (4.3 TB/s), 10 x 512 float32 2.2 us (a launch).
#include "ln.h"
#include <math.h>

namespace {
using namespace ln;

struct FwdArgs {
  const void* x;
  void* y;
  const float* w;      // nullptr: ones
  const float* b;      // nullptr: zeros
  float* mean;         // nullptr: not kept (evaluation)
  float* rstd;
  int64_t ldx, ldy, rows;
  int C;
  float eps;
};

// s / C to the last bit (a constant row has to give exactly its value): one Newton correction of s * (1 / C)
__device__ __forceinline__ float over(float s, float C, float inv) {
  const float m = s * inv;
  const float r = fmaf(-m, C, s);
  return isfinite(m) ? fmaf(r, inv, m) : m;
}

// whether the mean of a row in registers is corrected (see above)
template <typename T> constexpr bool CORRECT = sizeof(T) == 4;
// mean square around a number `off` below the mean -> variance; not below zero, and infinite where the squares overflow
__device__ __forceinline__ float variance(float square, float off) {
  return isfinite(square) ? fmaxf(fmaf(-off, off, square), 0.f) : square;
}

template <typename T, int G, int NV, bool TAIL>
__global__ __launch_bounds__(G <= 256 ? 256 : G) void ln_fwd_kernel(FwdArgs a) {
  constexpr int VEC = Geo<T>::VEC, BT = G <= 256 ? 256 : G, GB = BT / G;
  __shared__ float red[2 * (BT / 64)];
  const int t = threadIdx.x % G, grp = threadIdx.x / G;
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  int col[NV], dup[NV];
  float w[NV][VEC], b[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c0 = (t + k * G) * VEC;
    col[k] = TAIL && c0 + VEC > a.C ? a.C - VEC : c0;
    dup[k] = TAIL ? (c0 - col[k] < VEC ? c0 - col[k] : VEC) : 0;
    load_param<VEC>(a.w, col[k], 1.f, w[k]);
    load_param<VEC>(a.b, col[k], 0.f, b[k]);
  }
  const float inv = 1.f / (float)a.C;
  for (int64_t row = (int64_t)blockIdx.x * GB + grp; row < a.rows; row += (int64_t)gridDim.x * GB) {
    uint4 v[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k] = load_raw(x + row * a.ldx + col[k]);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float f[VEC];
      unpack(v[k], f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += !TAIL || e >= dup[k] ? f[e] : 0.f;
    }
    const float near = over(group_sum<G>(s, red), (float)a.C, inv);
    float q = 0.f, r = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float f[VEC];
      unpack(v[k], f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = f[e] - near;
        q += !TAIL || e >= dup[k] ? d * d : 0.f;
        if (CORRECT<T>) r += !TAIL || e >= dup[k] ? d : 0.f;
      }
    }
    if (CORRECT<T>) group_sum2<G>(q, r, red);
    else q = group_sum<G>(q, red);
    const float off = r * inv;
    const float rstd = 1.f / sqrtf(variance(q * inv, off) + a.eps);
    T* yr = y + row * a.ldy;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float f[VEC];
      unpack(v[k], f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = (CORRECT<T> ? f[e] - near - off : f[e] - near) * rstd * w[k][e] + b[k][e];
      if (!TAIL || dup[k] == 0) {
        store_raw(yr + col[k], pack(f));
      } else {
#pragma unroll
        for (int e = 1; e < VEC; ++e)
          if (e >= dup[k]) yr[col[k] + e] = (T)f[e];
      }
    }
    if (a.mean && t == 0) {
      a.mean[row] = near + off;
      a.rstd[row] = rstd;
    }
  }
}

// rows shorter than one chunk: a thread per row
template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_narrow_kernel(FwdArgs a) {
  constexpr int M = 7;
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  const float inv = 1.f / (float)a.C;
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.rows; row += (int64_t)gridDim.x * 256) {
    float f[M], s = 0.f, q = 0.f;
#pragma unroll
    for (int e = 0; e < M; ++e) {
      f[e] = e < a.C ? (float)x[row * a.ldx + e] : 0.f;
      s += f[e];
    }
    const float near = over(s, (float)a.C, inv);
    float r = 0.f;
#pragma unroll
    for (int e = 0; e < M; ++e) {
      const float d = e < a.C ? f[e] - near : 0.f;
      q += d * d;
      r += d;
    }
    const float off = r * inv;
    const float rstd = 1.f / sqrtf(variance(q * inv, off) + a.eps);
#pragma unroll
    for (int e = 0; e < M; ++e)
      if (e < a.C) y[row * a.ldy + e] = (T)((f[e] - near - off) * rstd * (a.w ? a.w[e] : 1.f) + (a.b ? a.b[e] : 0.f));
    if (a.mean) {
      a.mean[row] = near + off;
      a.rstd[row] = rstd;
    }
  }
}

// Longer rows: the first 8 chunks of each of 1024 threads stay in registers, what lies behind them is read for each sweep, out
// of the caches.  4096 x 20000 float32 184 us (3.6 TB/s; three sweeps over memory with 4-byte loads: 249), 1000 x 33000 bfloat16
// 40 us (71).  A row is one workgroup's, however long: 1 x 100000 takes as long as 8.  A thread adds up to 2^18 elements: the sum
// of a chunk is float32, the thread's float64.
template <typename T>
__global__ __launch_bounds__(WIDE) void ln_fwd_wide_kernel(FwdArgs a) {
  constexpr int VEC = Geo<T>::VEC, KEEP = 8;
  __shared__ float red[2 * (WIDE / 64)];
  const T* x = static_cast<const T*>(a.x) + (int64_t)blockIdx.x * a.ldx;
  T* y = static_cast<T*>(a.y) + (int64_t)blockIdx.x * a.ldy;
  uint4 v[KEEP];
#pragma unroll
  for (int i = 0; i < KEEP; ++i) v[i] = make_uint4(0, 0, 0, 0);
  double s = 0.0, q = 0.0, r = 0.0;
  wide_row<VEC, KEEP>(a.C, [&](int kept, int c, int dup) {
    const uint4 raw = load_raw(x + c);
    if (kept >= 0) v[kept] = raw;
    float f[VEC], sc = 0.f;
    unpack(raw, f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sc += e >= dup ? f[e] : 0.f;
    s += (double)sc;
  });
  const float near = over(group_sum<WIDE>((float)s, red), (float)a.C, 1.f / (float)a.C);
  wide_row<VEC, KEEP>(a.C, [&](int kept, int c, int dup) {
    float f[VEC], qc = 0.f, rc = 0.f;
    unpack(kept >= 0 ? v[kept] : load_raw(x + c), f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float d = e >= dup ? f[e] - near : 0.f;
      qc += d * d;
      rc += d;
    }
    q += (double)qc;
    r += (double)rc;
  });
  float square = (float)q, off = (float)r;
  group_sum2<WIDE>(square, off, red);
  off /= (float)a.C;
  const float rstd = 1.f / sqrtf(variance(square / (float)a.C, off) + a.eps);
  wide_row<VEC, KEEP>(a.C, [&](int kept, int c, int dup) {
    float f[VEC], w[VEC], b[VEC];
    unpack(kept >= 0 ? v[kept] : load_raw(x + c), f);
    load_param<VEC>(a.w, c, 1.f, w);
    load_param<VEC>(a.b, c, 0.f, b);
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = (f[e] - near - off) * rstd * w[e] + b[e];
    if (dup == 0) {
      store_raw(y + c, pack(f));
    } else {
#pragma unroll
      for (int e = 1; e < VEC; ++e)
        if (e >= dup) y[c + e] = (T)f[e];
    }
  });
  if (a.mean && threadIdx.x == 0) {
    a.mean[blockIdx.x] = near + off;
    a.rstd[blockIdx.x] = rstd;
  }
}

template <typename T>
struct Fwd {
  const FwdArgs& a;
  hipStream_t st;
  template <int G, int NV>
  int run() {
    constexpr int VEC = Geo<T>::VEC, BT = G <= 256 ? 256 : G, GB = BT / G;
    // Workgroups that walk over rows keep the parameters in registers: eight per CU fill it.  Very many rows go to more of
    // them, which evens out what the parts of the chip reach: 1048576 rows of 320 bfloat16 take 222 us with 16384, 244 us
    // with 2048, but 262144 rows 57 us instead of 54.
    int64_t blocks = cdiv64(a.rows, GB);
    if (blocks > 2048) blocks = blocks < 16384 ? 2048 : 16384;
    if (a.C == G * NV * VEC) ln_fwd_kernel<T, G, NV, false><<<(unsigned)blocks, BT, 0, st>>>(a);
    else ln_fwd_kernel<T, G, NV, true><<<(unsigned)blocks, BT, 0, st>>>(a);
    SNWS_LAUNCH_CHECK("snws_ln_fwd");
    return SNWS_OK;
  }
  int wide() {
    if (a.rows >= MAX_WIDE_ROWS) SNWS_UNSUPPORTED("snws_ln_fwd: too many rows of this length");
    ln_fwd_wide_kernel<T><<<(unsigned)a.rows, WIDE, 0, st>>>(a);
    SNWS_LAUNCH_CHECK("snws_ln_fwd");
    return SNWS_OK;
  }
  int go() {
    constexpr int VEC = Geo<T>::VEC;
    if (a.C < VEC) {
      int64_t blocks = cdiv64(a.rows, 256);
      if (blocks > 4096) blocks = 4096;
      ln_fwd_narrow_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(a);
      SNWS_LAUNCH_CHECK("snws_ln_fwd");
      return SNWS_OK;
    }
    return dispatch(cdiv64(a.C, VEC), *this);
  }
};

}  // namespace

extern "C" int snws_ln_fwd(const void* x, int64_t ldx, const float* weight, const float* bias, void* y, int64_t ldy, int dtype,
                           int64_t rows, int C, float eps, float* mean, float* rstd, void* stream) {
  SNWS_CHECK_ARG(dtype == SNWS_F32 || dtype == SNWS_BF16, "snws_ln_fwd: dtype must be float32 or bfloat16");
  SNWS_CHECK_ARG(rows >= 0 && C >= 1 && C <= LN_MAX_C && ldx >= C && ldy >= C, "snws_ln_fwd: bad sizes");
  SNWS_CHECK_ARG(eps >= 0.f && isfinite(eps), "snws_ln_fwd: eps must be finite and not negative");
  if (rows == 0) return SNWS_OK;
  SNWS_CHECK_ARG(x && y, "snws_ln_fwd: NULL pointer");
  SNWS_CHECK_ARG((mean == nullptr) == (rstd == nullptr), "snws_ln_fwd: mean and rstd go together");
  const FwdArgs a{x, y, weight, bias, mean, rstd, ldx, ldy, rows, C, eps};
  const hipStream_t st = (hipStream_t)stream;
  return dtype == SNWS_F32 ? Fwd<float>{a, st}.go() : Fwd<bf16_t>{a, st}.go();
}
