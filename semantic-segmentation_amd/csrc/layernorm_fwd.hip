// Layer normalisation over the last axis, forward: y = (x - mean) * rstd * weight + bias per row, mean and variance of the
// row's own C elements (the channels of one pixel in NHWC), rstd = 1 / sqrt(var + eps).
//
// Bound by memory: x is read once and y written once.  A row stays in registers between the two (ln.h), so the variance is
// taken around the mean in a second sweep over registers - no cancellation however large the mean - in float32.
// Measured: 262144 x 64 bfloat16 11.6 us (5.8 TB/s), 1048576 x 320 bfloat16 222 us (6.0 TB/s), 997 x 9216 float32 16.7 us
// (4.4 TB/s), 10 x 512 float32 2.2 us (a launch).
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
    const float mean = over(group_sum<G>(s, red), (float)a.C, inv);
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float f[VEC];
      unpack(v[k], f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = f[e] - mean;
        q += !TAIL || e >= dup[k] ? d * d : 0.f;
      }
    }
    const float rstd = 1.f / sqrtf(group_sum<G>(q, red) * inv + a.eps);
    T* yr = y + row * a.ldy;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float f[VEC];
      unpack(v[k], f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = (f[e] - mean) * rstd * w[k][e] + b[k][e];
      if (!TAIL || dup[k] == 0) {
        store_raw(yr + col[k], pack(f));
      } else {
#pragma unroll
        for (int e = 1; e < VEC; ++e)
          if (e >= dup[k]) yr[col[k] + e] = (T)f[e];
      }
    }
    if (a.mean && t == 0) {
      a.mean[row] = mean;
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
    const float mean = over(s, (float)a.C, inv);
#pragma unroll
    for (int e = 0; e < M; ++e) q += e < a.C ? (f[e] - mean) * (f[e] - mean) : 0.f;
    const float rstd = 1.f / sqrtf(q * inv + a.eps);
#pragma unroll
    for (int e = 0; e < M; ++e)
      if (e < a.C) y[row * a.ldy + e] = (T)((f[e] - mean) * rstd * (a.w ? a.w[e] : 1.f) + (a.b ? a.b[e] : 0.f));
    if (a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// rows longer than the registers of a workgroup hold: three sweeps, the later two out of the caches
template <typename T>
__global__ __launch_bounds__(512) void ln_fwd_wide_kernel(FwdArgs a) {
  __shared__ float red[16];
  const T* x = static_cast<const T*>(a.x) + (int64_t)blockIdx.x * a.ldx;
  T* y = static_cast<T*>(a.y) + (int64_t)blockIdx.x * a.ldy;
  float s = 0.f, q = 0.f;
  for (int c = threadIdx.x; c < a.C; c += 512) s += (float)x[c];
  const float mean = group_sum<512>(s, red) / (float)a.C;
  for (int c = threadIdx.x; c < a.C; c += 512) {
    const float d = (float)x[c] - mean;
    q += d * d;
  }
  const float rstd = 1.f / sqrtf(group_sum<512>(q, red) / (float)a.C + a.eps);
  for (int c = threadIdx.x; c < a.C; c += 512)
    y[c] = (T)(((float)x[c] - mean) * rstd * (a.w ? a.w[c] : 1.f) + (a.b ? a.b[c] : 0.f));
  if (a.mean && threadIdx.x == 0) {
    a.mean[blockIdx.x] = mean;
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
    if (a.rows > 0x7fffffff) SNWS_UNSUPPORTED("snws_ln_fwd: too many rows of this length");
    ln_fwd_wide_kernel<T><<<(unsigned)a.rows, 512, 0, st>>>(a);
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
