// What the forward and the backward layer-normalisation kernels share: how a row is spread over lanes, 16-byte loads and
// stores of any alignment, sums over the lanes of a row, and the choice of a kernel for a row length.
//
// A row of C elements is held in registers by a group of G lanes, NV chunks of 16 bytes (VEC elements) per lane: chunk
// t + k * G belongs to lane t.  Every load instruction of a group then covers G * 16 consecutive bytes, and each element
// is fetched from memory once.  A row whose length is no multiple of VEC ends in a chunk that is moved back to end with
// the row: it overlaps its predecessor, and its first `dup` elements count for nothing and are not stored (chunks past
// the end are such a chunk with dup == VEC).  Rows need no alignment beyond their element's.
#pragma once
#include "common.h"

namespace ln {

constexpr int LN_MAX_C = 1 << 28;      // 2 C and a column counter's last step stay within 31 bits

template <typename T> struct Geo;
template <> struct Geo<float> { static constexpr int VEC = 4; };
template <> struct Geo<bf16_t> { static constexpr int VEC = 8; };

// 16 bytes at an address aligned to the element only (global memory takes any alignment; whole lines are fetched once)
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Raw { unsigned u[4]; };
struct __attribute__((packed, aligned(4))) Raw32 { float f[4]; };

template <typename T>
__device__ __forceinline__ uint4 load_raw(const T* p) {
  const Raw<T> r = *reinterpret_cast<const Raw<T>*>(p);
  return make_uint4(r.u[0], r.u[1], r.u[2], r.u[3]);
}
template <typename T>
__device__ __forceinline__ void store_raw(T* p, uint4 v) {
  Raw<T> r;
  r.u[0] = v.x; r.u[1] = v.y; r.u[2] = v.z; r.u[3] = v.w;
  *reinterpret_cast<Raw<T>*>(p) = r;
}
__device__ __forceinline__ void unpack(uint4 v, float (&f)[4]) {
  f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(uint4 v, float (&f)[8]) {
  const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(u[i] << 16);
    f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack(const float (&f)[4]) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 pack(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
// VEC float32 parameters from an address aligned to 4 bytes, or `fill` without a parameter
template <int VEC>
__device__ __forceinline__ void load_param(const float* p, int col, float fill, float (&f)[VEC]) {
#pragma unroll
  for (int q = 0; q < VEC / 4; ++q) {
    if (p) {
      const Raw32 r = *reinterpret_cast<const Raw32*>(p + col + 4 * q);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * q + e] = r.f[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * q + e] = fill;
    }
  }
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// sum over a group of G <= 64 consecutive lanes, the same bits in each of them (partners 1, 2, then the other quad, the
// other eight, then 16 and 32 lanes away)
template <int G>
__device__ __forceinline__ float lane_sum(float v) {
  v = dpp_add<0xB1>(v);                      // lane ^ 1
  v = dpp_add<0x4E>(v);                      // lane ^ 2
  if (G >= 8) v = dpp_add<0x141>(v);         // mirrored within 8: the quads' sums are uniform by now
  if (G >= 16) v = dpp_add<0x140>(v);        // mirrored within 16
  if (G >= 32) v += __shfl_xor(v, 16, 64);
  if (G >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}
// two sums over the G threads of a row; G > 64: over the whole workgroup, by way of 2 * G / 64 floats of LDS
template <int G>
__device__ __forceinline__ void group_sum2(float& a, float& b, float* red) {
  if (G <= 64) {
    a = lane_sum<G>(a);
    b = lane_sum<G>(b);
  } else {
    constexpr int NW = G > 64 ? G / 64 : 1;
    a = lane_sum<64>(a);
    b = lane_sum<64>(b);
    __syncthreads();                          // the previous sums have been read
    if ((threadIdx.x & 63) == 0) {
      red[threadIdx.x >> 6] = a;
      red[NW + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      a += red[i];
      b += red[NW + i];
    }
  }
}
template <int G>
__device__ __forceinline__ float group_sum(float a, float* red) {
  if (G <= 64) return lane_sum<G>(a);
  constexpr int NW = G > 64 ? G / 64 : 1;
  a = lane_sum<64>(a);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  a = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) a += red[i];
  return a;
}

// A row by a workgroup of 1024 threads, chunk after chunk: f(kept index or -1, chunk's first column, its dup).  The first KEEP
// chunks of a thread have a constant index, so that what is kept of them stays in registers.
constexpr int WIDE = 1024;
constexpr int64_t MAX_WIDE_ROWS = (1ll << 32) / WIDE;      // a launch holds less than 2^32 threads: 4 million rows of 64 KB or more
template <int VEC, int KEEP, typename F>
__device__ __forceinline__ void wide_row(int C, F&& f) {
  const int chunks = (C + VEC - 1) / VEC;
  auto one = [&](int kept, int k) {
    const int c0 = k * VEC, c = c0 + VEC > C ? C - VEC : c0;
    f(kept, c, c0 - c);
  };
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if ((int)threadIdx.x + i * WIDE < chunks) one(i, threadIdx.x + i * WIDE);
#pragma unroll 4
  for (int k = threadIdx.x + KEEP * WIDE; k < chunks; k += WIDE) one(-1, k);
}

// Lanes per row and chunks per lane for a row of `chunks` chunks.  The narrowest group that needs at most five chunks per
// lane wastes the fewest lanes on a ragged end (320 bfloat16 channels: 40 chunks = 8 lanes x 5, none idle); from 160
// chunks on a whole wave, then a workgroup of 4 or 8 waves takes a row, with up to eight.  0: longer than registers hold.
// (A whole wave per row of 320 bfloat16, 24 of its lanes idle: forward 358 us instead of 244, backward 542 instead of 390.)
inline int pick_group(int64_t chunks) {
  if (chunks <= 40) return 8;
  if (chunks <= 80) return 16;
  if (chunks <= 160) return 32;
  if (chunks <= 512) return 64;
  if (chunks <= 2048) return 256;
  if (chunks <= 4096) return 512;
  return 0;
}

// calls F<G, NV>() for the pair that pick_group and the row length give
#define LN_CASE(G_, NV_) \
  case NV_: return f.template run<G_, NV_>();
template <typename F>
int dispatch(int64_t chunks, F&& f) {
  const int G = pick_group(chunks), nv = G ? (int)((chunks + G - 1) / G) : 0;
  switch (G) {
    case 8:
      switch (nv) { LN_CASE(8, 1) LN_CASE(8, 2) LN_CASE(8, 3) LN_CASE(8, 4) LN_CASE(8, 5) }
      break;
    case 16:
      switch (nv) { LN_CASE(16, 3) LN_CASE(16, 4) LN_CASE(16, 5) }
      break;
    case 32:
      switch (nv) { LN_CASE(32, 3) LN_CASE(32, 4) LN_CASE(32, 5) }
      break;
    case 64:
      switch (nv) { LN_CASE(64, 3) LN_CASE(64, 4) LN_CASE(64, 5) LN_CASE(64, 6) LN_CASE(64, 7) LN_CASE(64, 8) }
      break;
    case 256:
      switch (nv) { LN_CASE(256, 3) LN_CASE(256, 4) LN_CASE(256, 5) LN_CASE(256, 6) LN_CASE(256, 7) LN_CASE(256, 8) }
      break;
    case 512:
      switch (nv) { LN_CASE(512, 5) LN_CASE(512, 6) LN_CASE(512, 7) LN_CASE(512, 8) }
      break;
  }
  return f.wide();
}
#undef LN_CASE

}  // namespace ln
