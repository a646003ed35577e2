// Layer normalisation over the last axis, backward.  With z = (x - mean) * rstd and g = dy * weight, per row
//   dx = rstd * (g - sum(g) / C - z * sum(g * z) / C),
// and over all rows dweight = sum(dy * z), dbias = sum(dy).
//
// Bound by memory: x and dy are read once and dx is written once.  One sweep does it all: a group of lanes holds a row
// in registers (ln.h) and walks over rows, so its columns stay the same and their share of the two parameter gradients
// is summed on the spot.  A workgroup folds its groups and stores one partial row; a second, small launch adds the
// partial rows in a fixed order in float64.  Runs with the same sizes give the same bits.
// A lane holds its columns of x, dy, the weight and both sums: 32 registers per bfloat16 chunk, 20 per float32 one.  Seven or eight
// chunks of bfloat16, and 512 lanes from five (seven of float32) on, are more than the registers, and the rest lies in
// scratch memory: 69905 x 3840 bfloat16 660 us (2.4 TB/s), but 65536 x 4096 328 us; 9362 x 28672 1195 us (1.4 TB/s).
// Few rows are bound by launches: there one launch does both, with workgroups of their own for the parameter gradients, which
// read their columns of x and dy once more out of the caches, and no partial rows.
// Measured, with the second launch: 1048576 x 320 bfloat16 390 + 5 us (5.2 TB/s), 16384 x 1024 bfloat16 22 + 4 us (4.6 TB/s
// for the sweep), 50001 x 77 float32 rows of a wider buffer 16 + 4 us.
#include "ln.h"

namespace {
using namespace ln;

struct BwdArgs {
  const void* dy;
  const void* x;
  const float* mean;
  const float* rstd;
  const float* w;      // nullptr: ones
  void* dx;            // nullptr: not wanted
  float* part;         // [blocks][2][C], nullptr: no parameter gradient wanted, or few rows
  float* dw;           // few rows: the parameter gradients themselves, nullptr: not wanted
  float* db;
  int64_t lddy, ldx, lddx, rows;
  int C;
  int row_blocks;      // workgroups that take rows; those behind them take columns
};

// One launch up to here: 160 rows of 512 float32 take 4.1 us instead of 5.4 + 2.7 us in two launches.
constexpr int64_t FEW_ROWS = 256;
constexpr int64_t SLICE_ROWS = 16;     // rows to a thread of the columns' sums, where rows are longer than registers hold

// parameter gradients of 32 columns, by all threads of a workgroup: float32 over a thread's rows, float64 over the threads
template <typename T, int BT>
__device__ __forceinline__ void column_sums(const BwdArgs& a, int c0) {
  constexpr int LANES = BT / 32;
  __shared__ double red[2][LANES][33];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5, c = c0 + cl;
  float sw = 0.f, sb = 0.f;
  if (c < a.C) {
    const T* x = static_cast<const T*>(a.x) + c;
    const T* dy = static_cast<const T*>(a.dy) + c;
#pragma unroll 8
    for (int r = rl; r < (int)a.rows; r += LANES) {
      const float g = (float)dy[r * a.lddy];
      sb += g;
      sw += g * (((float)x[r * a.ldx] - a.mean[r]) * a.rstd[r]);
    }
  }
  red[0][rl][cl] = sw;
  red[1][rl][cl] = sb;
  __syncthreads();
  if (rl < 2 && c < a.C) {
    double s = 0.0;
#pragma unroll
    for (int r = 0; r < LANES; ++r) s += red[rl][r][cl];
    float* o = rl ? a.db : a.dw;
    if (o) o[c] = (float)s;
  }
}

// Workgroups that stay, and so partial rows: one per CU, four waves, has enough loads in flight where a lane holds three
// chunks or more of each operand, two where it holds fewer (1048576 rows of 64 bfloat16: 80 us instead of 130; 1048576
// rows of 320, five chunks: 387 us and 5 us for the partial rows, instead of 390 and 9).
constexpr int64_t most_blocks(int nv) { return nv <= 2 ? 512 : 256; }

template <typename T, int G, int NV, bool TAIL>
__global__ __launch_bounds__(G <= 256 ? 256 : G) void ln_bwd_kernel(BwdArgs a) {
  constexpr int VEC = Geo<T>::VEC, BT = G <= 256 ? 256 : G, GB = BT / G;
  constexpr int NW = BT / 64, WC = (G < 64 ? G : 64) * NV * VEC;       // waves; columns that one wave holds
  __shared__ float red[2 * NW];
  __shared__ float fold[G < 256 ? 2 * WC : 1];
  if ((int)blockIdx.x >= a.row_blocks) {
    column_sums<T, BT>(a, ((int)blockIdx.x - a.row_blocks) * 32);
    return;
  }
  const int t = threadIdx.x % G, grp = threadIdx.x / G;
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  T* dx = static_cast<T*>(a.dx);
  int col[NV], dup[NV];
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c0 = (t + k * G) * VEC;
    col[k] = TAIL && c0 + VEC > a.C ? a.C - VEC : c0;
    dup[k] = TAIL ? (c0 - col[k] < VEC ? c0 - col[k] : VEC) : 0;
    load_param<VEC>(a.w, col[k], 1.f, w[k]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[k][e] = db[k][e] = 0.f;
  }
  const float inv = 1.f / (float)a.C;
  for (int64_t row = (int64_t)blockIdx.x * GB + grp; row < a.rows; row += (int64_t)a.row_blocks * GB) {
    uint4 vx[NV], vg[NV];
    const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      vx[k] = load_raw(x + row * a.ldx + col[k]);
      vg[k] = load_raw(dy + row * a.lddy + col[k]);
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float f[VEC], g[VEC];
      unpack(vx[k], f);
      unpack(vg[k], g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float z = (f[e] - mean) * rstd;
        const bool on = !TAIL || e >= dup[k];
        const float d = on ? g[e] : 0.f, dz = on ? g[e] * z : 0.f;
        db[k][e] += d;
        dw[k][e] += dz;
        s1 += d * w[k][e];
        s2 += dz * w[k][e];
      }
    }
    if (!dx) continue;
    group_sum2<G>(s1, s2, red);
    const float m1 = s1 * inv, m2 = s2 * inv;
    T* o = dx + row * a.lddx;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float f[VEC], g[VEC];
      unpack(vx[k], f);
      unpack(vg[k], g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float z = (f[e] - mean) * rstd;
        f[e] = rstd * (g[e] * w[k][e] - m1 - z * m2);
      }
      if (!TAIL || dup[k] == 0) {
        store_raw(o + col[k], pack(f));
      } else {
#pragma unroll
        for (int e = 1; e < VEC; ++e)
          if (e >= dup[k]) o[col[k] + e] = (T)f[e];
      }
    }
  }
  if (!a.part) return;
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.C;
  if (G >= 256) {               // the workgroup is one group: its sums are the workgroup's
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (!TAIL || e >= dup[k]) {
          part[col[k] + e] = dw[k][e];
          part[a.C + col[k] + e] = db[k][e];
        }
    return;
  }
  // fold the groups of a wave by shuffles, then the waves one after the other through one row of LDS: a fixed order
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
#pragma unroll
      for (int o = G; o < 64; o <<= 1) {
        dw[k][e] += __shfl_xor(dw[k][e], o, 64);
        db[k][e] += __shfl_xor(db[k][e], o, 64);
      }
    }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int q = 0; q < NW; ++q) {
    if (q == wave && lane < G) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (!TAIL || e >= dup[k]) {
            const int c = col[k] + e;
            fold[c] = q ? fold[c] + dw[k][e] : dw[k][e];
            fold[WC + c] = q ? fold[WC + c] + db[k][e] : db[k][e];
          }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 2 * a.C; i += BT) part[i] = fold[i < a.C ? i : WC + i - a.C];
}

template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_narrow_kernel(BwdArgs a) {
  constexpr int M = 7;
  __shared__ float red[16];
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  T* dx = static_cast<T*>(a.dx);
  const float inv = 1.f / (float)a.C;
  float dw[M], db[M];
#pragma unroll
  for (int e = 0; e < M; ++e) dw[e] = db[e] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.rows; row += (int64_t)gridDim.x * 256) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float z[M], g[M], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int e = 0; e < M; ++e) {
      z[e] = e < a.C ? ((float)x[row * a.ldx + e] - mean) * rstd : 0.f;
      g[e] = e < a.C ? (float)dy[row * a.lddy + e] : 0.f;
      db[e] += g[e];
      dw[e] += g[e] * z[e];
      g[e] *= e < a.C && a.w ? a.w[e] : 1.f;
      s1 += g[e];
      s2 += g[e] * z[e];
    }
    if (dx) {
#pragma unroll
      for (int e = 0; e < M; ++e)
        if (e < a.C) dx[row * a.lddx + e] = (T)(rstd * (g[e] - s1 * inv - z[e] * s2 * inv));
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int e = 0; e < M; ++e) {
    const float sw = block_sum(dw[e], red), sb = block_sum(db[e], red);
    if (threadIdx.x == 0 && e < a.C) {
      a.part[(int64_t)blockIdx.x * 2 * a.C + e] = sw;
      a.part[(int64_t)blockIdx.x * 2 * a.C + a.C + e] = sb;
    }
  }
}

// rows beyond what the kernel above holds: 4 chunks of x and dy of each of 1024 threads stay in registers; the sum
// of a chunk is float32, a thread's, of up to 2^18 elements, float64
template <typename T>
__global__ __launch_bounds__(WIDE) void ln_bwd_wide_kernel(BwdArgs a) {
  constexpr int VEC = Geo<T>::VEC, KEEP = 4;
  __shared__ float red[2 * (WIDE / 64)];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
  T* dx = static_cast<T*>(a.dx) + row * a.lddx;
  const float mean = a.mean[row], rstd = a.rstd[row];
  uint4 vx[KEEP], vg[KEEP];
#pragma unroll
  for (int i = 0; i < KEEP; ++i) vx[i] = vg[i] = make_uint4(0, 0, 0, 0);
  double s1 = 0.0, s2 = 0.0;
  wide_row<VEC, KEEP>(a.C, [&](int kept, int c, int dup) {
    const uint4 rx = load_raw(x + c), rg = load_raw(dy + c);
    if (kept >= 0) {
      vx[kept] = rx;
      vg[kept] = rg;
    }
    float f[VEC], g[VEC], w[VEC], c1 = 0.f, c2 = 0.f;
    unpack(rx, f);
    unpack(rg, g);
    load_param<VEC>(a.w, c, 1.f, w);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float d = e >= dup ? g[e] * w[e] : 0.f;
      c1 += d;
      c2 += e >= dup ? d * ((f[e] - mean) * rstd) : 0.f;
    }
    s1 += (double)c1;
    s2 += (double)c2;
  });
  float m1 = (float)s1, m2 = (float)s2;
  group_sum2<WIDE>(m1, m2, red);
  m1 /= (float)a.C;
  m2 /= (float)a.C;
  wide_row<VEC, KEEP>(a.C, [&](int kept, int c, int dup) {
    float f[VEC], g[VEC], w[VEC];
    unpack(kept >= 0 ? vx[kept] : load_raw(x + c), f);
    unpack(kept >= 0 ? vg[kept] : load_raw(dy + c), g);
    load_param<VEC>(a.w, c, 1.f, w);
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = rstd * (g[e] * w[e] - m1 - (f[e] - mean) * rstd * m2);
    if (dup == 0) {
      store_raw(dx + c, pack(f));
    } else {
#pragma unroll
      for (int e = 1; e < VEC; ++e)
        if (e >= dup) dx[c + e] = (T)f[e];
    }
  });
}

// Parameter gradients of such rows: a thread per column, rows dealt to gridDim.y slices.  The slices get fewer as rows get longer,
// and a thread's rows many, so it adds them in float64.
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_wide_param_kernel(BwdArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  double dw = 0.0, db = 0.0;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float g = (float)dy[row * a.lddy + c];
    db += (double)g;
    dw += (double)(g * (((float)x[row * a.ldx + c] - a.mean[row]) * a.rstd[row]));
  }
  if (!a.part) {               // one slice: no partial rows
    if (a.dw) a.dw[c] = (float)dw;
    if (a.db) a.db[c] = (float)db;
    return;
  }
  float* part = a.part + (int64_t)blockIdx.y * 2 * a.C;
  part[c] = (float)dw;
  part[a.C + c] = (float)db;
}

// dweight[c] / dbias[c] = sum over the partial rows, in float64 and a fixed order: 32 columns x 32 row lanes at a time
__global__ __launch_bounds__(1024) void ln_param_sum_kernel(const float* __restrict__ part, int blocks, int C,
                                                            float* __restrict__ dw, float* __restrict__ db) {
  constexpr int LOADS = 8;
  __shared__ double red[32][33];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  for (int i0 = blockIdx.x * 32; i0 < 2 * C; i0 += gridDim.x * 32) {
    const int i = i0 + cl;
    double s = 0.0;
    if (i < 2 * C)
      for (int r = rl; r < blocks; r += 32 * LOADS) {
        float f[LOADS];        // in flight together
#pragma unroll
        for (int k = 0; k < LOADS; ++k) f[k] = r + 32 * k < blocks ? part[(int64_t)(r + 32 * k) * 2 * C + i] : 0.f;
#pragma unroll
        for (int k = 0; k < LOADS; ++k) s += (double)f[k];
      }
    __syncthreads();           // the previous columns have been read
    red[rl][cl] = s;
    __syncthreads();
    if (rl == 0 && i < 2 * C) {
      s = 0.0;
#pragma unroll
      for (int r = 0; r < 32; ++r) s += red[r][cl];
      float* o = i < C ? dw : db;
      if (o) o[i < C ? i : i - C] = (float)s;
    }
  }
}

// workgroups of the sweep = partial rows
template <typename T>
int64_t bwd_blocks(int64_t rows, int C) {
  constexpr int VEC = Geo<T>::VEC;
  int64_t need, most = most_blocks(1);
  if (C < VEC) {
    need = cdiv64(rows, 256);
  } else {
    const int64_t chunks = cdiv64(C, VEC);
    const int G = pick_group(chunks);
    if (!G) {
      need = cdiv64(rows, SLICE_ROWS);               // slices of the column sums
      const int64_t cb = cdiv64(C, 256);
      most = cdiv64(1024, cb);
      return need < most ? need : most;
    }
    need = cdiv64(rows, G <= 256 ? 256 / G : 1);
    most = most_blocks((int)cdiv64(chunks, G));
  }
  return need < most ? need : most;
}

// few rows: no partial rows
template <typename T>
bool few_rows(int64_t rows, int C) {
  constexpr int VEC = Geo<T>::VEC;
  return C >= VEC && rows <= (pick_group(cdiv64(C, VEC)) ? FEW_ROWS : SLICE_ROWS);
}
bool few_rows(int dtype, int64_t rows, int C) {
  return dtype == SNWS_F32 ? few_rows<float>(rows, C) : few_rows<bf16_t>(rows, C);
}

template <typename T>
struct Bwd {
  const BwdArgs& a;
  int64_t blocks;      // of the whole launch
  hipStream_t st;
  template <int G, int NV>
  int run() {
    constexpr int VEC = Geo<T>::VEC, BT = G <= 256 ? 256 : G;
    if (a.C == G * NV * VEC) ln_bwd_kernel<T, G, NV, false><<<(unsigned)blocks, BT, 0, st>>>(a);
    else ln_bwd_kernel<T, G, NV, true><<<(unsigned)blocks, BT, 0, st>>>(a);
    SNWS_LAUNCH_CHECK("snws_ln_bwd");
    return SNWS_OK;
  }
  int wide() {
    if (a.rows >= MAX_WIDE_ROWS) SNWS_UNSUPPORTED("snws_ln_bwd: too many rows of this length");
    if (a.dx) {
      ln_bwd_wide_kernel<T><<<(unsigned)a.rows, WIDE, 0, st>>>(a);
      SNWS_LAUNCH_CHECK("snws_ln_bwd");
    }
    if (a.dw || a.db) {
      ln_bwd_wide_param_kernel<T><<<dim3((unsigned)cdiv64(a.C, 256), a.part ? (unsigned)blocks : 1), 256, 0, st>>>(a);
      SNWS_LAUNCH_CHECK("snws_ln_bwd");
    }
    return SNWS_OK;
  }
  int go() {
    constexpr int VEC = Geo<T>::VEC;
    if (a.C < VEC) {
      ln_bwd_narrow_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(a);
      SNWS_LAUNCH_CHECK("snws_ln_bwd");
      return SNWS_OK;
    }
    return dispatch(cdiv64(a.C, VEC), *this);
  }
};

}  // namespace

extern "C" int64_t snws_ln_bwd_workspace_floats(int dtype, int64_t rows, int C) {
  if (rows < 1 || C < 1 || C > LN_MAX_C || few_rows(dtype, rows, C)) return 0;
  return 2 * (int64_t)C * (dtype == SNWS_F32 ? bwd_blocks<float>(rows, C) : bwd_blocks<bf16_t>(rows, C));
}

extern "C" int snws_ln_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* mean, const float* rstd,
                           const float* weight, int dtype, int64_t rows, int C, void* dx, int64_t lddx, float* dweight,
                           float* dbias, float* workspace, int64_t workspace_floats, void* stream) {
  SNWS_CHECK_ARG(dtype == SNWS_F32 || dtype == SNWS_BF16, "snws_ln_bwd: dtype must be float32 or bfloat16");
  SNWS_CHECK_ARG(rows >= 0 && C >= 1 && C <= LN_MAX_C && lddy >= C && ldx >= C && (!dx || lddx >= C), "snws_ln_bwd: bad sizes");
  SNWS_CHECK_ARG(rows == 0 || (dy && x && mean && rstd), "snws_ln_bwd: NULL pointer");
  const bool params = dweight || dbias;
  const int64_t need = params ? snws_ln_bwd_workspace_floats(dtype, rows, C) : 0;
  SNWS_CHECK_ARG(need == 0 || (workspace && workspace_floats >= need), "snws_ln_bwd: workspace of %lld floats needed",
                 (long long)need);
  const hipStream_t st = (hipStream_t)stream;
  int64_t blocks = 0;
  if (rows > 0 && (dx || params)) {
    blocks = dtype == SNWS_F32 ? bwd_blocks<float>(rows, C) : bwd_blocks<bf16_t>(rows, C);
    const bool few = few_rows(dtype, rows, C);
    const BwdArgs a{dy, x, mean, rstd, weight, dx, params && !few ? workspace : nullptr, dweight, dbias, lddy, ldx, lddx, rows, C,
                    few && !dx ? 0 : (int)blocks};
    if (few) blocks = a.row_blocks + (params ? cdiv64(C, 32) : 0);
    const int rc = dtype == SNWS_F32 ? Bwd<float>{a, blocks, st}.go() : Bwd<bf16_t>{a, blocks, st}.go();
    if (rc != SNWS_OK || few) return rc;
  }
  if (params) {
    // (a launch holds less than 2^32 threads: the longest rows have more columns)
    const int64_t most = 1 << 16, need = cdiv64(2 * (int64_t)C, 32);
    ln_param_sum_kernel<<<(unsigned)(need < most ? need : most), 1024, 0, st>>>(workspace, (int)blocks, C, dweight, dbias);
    SNWS_LAUNCH_CHECK("snws_ln_bwd");
  }
  return SNWS_OK;
}
