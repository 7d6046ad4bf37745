// Shared parts of the selective state-space scan's kernels.
#pragma once

#include "gdn_common.cuh"
#include "gdn_internal.h"

namespace gdn {

constexpr int kScanThreads = 128;
constexpr int kScanLanes = 4;                            // lanes of a channel
constexpr int kScanCh = kScanThreads / kScanLanes;       // channels of a block

// log(1 + e) for 0 <= e <= 1 as 2 atanh(e / (2 + e)): with s = e / (2 + e) <= 1/3
// the series s + s^3 / 3 + ... + s^15 / 15 leaves less than s^17 / 17 / (1 - s^2) <
// 2^-29 of it out.  No cancellation at small e, where step sizes lie.
__device__ __forceinline__ float log1p_unit(float e) {
  const float s = __fdividef(e, 2.f + e);
  const float q = s * s;
  float p = fmaf(q, 1.f / 15.f, 1.f / 13.f);
  p = fmaf(q, p, 1.f / 11.f);
  p = fmaf(q, p, 1.f / 9.f);
  p = fmaf(q, p, 1.f / 7.f);
  p = fmaf(q, p, 1.f / 5.f);
  p = fmaf(q, p, 1.f / 3.f);
  return 2.f * fmaf(q * p, s, s);
}

// softplus(v) and, through `sig`, its derivative sigmoid(v).  A NaN stays one.
__device__ __forceinline__ float softplus_sig(float v, float& sig) {
  const float e = expf(-fabsf(v));
  const float r = __fdividef(1.f, 1.f + e);
  sig = v >= 0.f ? r : e * r;
  return (v > 0.f ? v : (v == v ? 0.f : v)) + log1p_unit(e);
}

// One element, zero where `ok` is false.
template <typename T>
__device__ __forceinline__ float load1(const T* p, bool ok) {
  return ok ? to_f32(*p) : 0.f;
}

// Four consecutive channels of a row: one vector when the row allows it, else
// element by element.  `n`: channels in range (<= 0: none).
template <typename T>
__device__ __forceinline__ void load_ch4(const T* p, int n, bool vec, float (&v)[4]) {
  if (vec && n >= 4) {
    const float4 q = load4(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = load1(p + e, e < n);
  }
}
template <typename T>
__device__ __forceinline__ void store_ch4(T* p, int n, bool vec, const float (&v)[4]) {
  if (vec && n >= 4) {
    store4(p, make_float4(v[0], v[1], v[2], v[3]));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) p[e] = from_f32<T>(v[e]);
  }
}

// Sums four tokens' values over the four lanes of a channel in three shuffles:
// lane j (lane & 3) returns the sum of v[j].
__device__ __forceinline__ float quad_sum4(float v0, float v1, float v2, float v3, int lane) {
  const bool hi = lane & 2, odd = lane & 1;
  // lanes 0, 1 keep tokens 0, 1; lanes 2, 3 keep tokens 2, 3
  float k0 = hi ? v2 : v0, k1 = hi ? v3 : v1;
  const float g0 = hi ? v0 : v2, g1 = hi ? v1 : v3;
  k0 += __shfl_xor_sync(0xffffffffu, g0, 2);
  k1 += __shfl_xor_sync(0xffffffffu, g1, 2);
  const float k = odd ? k1 : k0, g = odd ? k0 : k1;
  return k + __shfl_xor_sync(0xffffffffu, g, 1);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLog2e = 1.4426950408889634f;

// NL fp32 values to / from memory in 16-byte vectors where NL allows.
template <int NL>
__device__ __forceinline__ void store_states(float* p, const float (&v)[NL]) {
  if constexpr (NL % 4 == 0) {
#pragma unroll
    for (int i = 0; i < NL; i += 4) store4(p + i, make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
  } else {
#pragma unroll
    for (int i = 0; i < NL; ++i) p[i] = v[i];
  }
}
template <int NL>
__device__ __forceinline__ void load_states(const float* p, float (&v)[NL]) {
  if constexpr (NL % 4 == 0) {
#pragma unroll
    for (int i = 0; i < NL; i += 4) {
      const float4 q = load4(p + i);
      v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NL; ++i) v[i] = p[i];
  }
}

// Tokens of the backward's tile (and the distance of the forward's checkpoints)
// for NL states a lane: 64 decay factors a lane stay in registers.
template <int NL>
constexpr int scan_tile() { return NL <= 4 ? 16 : 64 / NL; }

}  // namespace gdn
