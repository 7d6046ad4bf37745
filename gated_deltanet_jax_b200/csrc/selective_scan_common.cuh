// Shared parts of the selective state-space scan's kernels.
#pragma once

#include "gdn_common.cuh"
#include "gdn_internal.h"

namespace gdn {

constexpr int kScanLanes = 4;   // lanes of a channel
constexpr int kScanCh = 32;     // channels of a block

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The same, formed again where it stands (not kept in a register from an equal
// argument's earlier use).
__device__ __forceinline__ float ex2_again(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLog2e = 1.4426950408889634f;

// Added to the argument of every decay factor exp2(delta A log2 e), in the multiply-
// add that forms it.  ex2.approx comes out too small by 0.1 to 0.45 of 2^-24 in the
// mean for arguments in [-0.3, 0] (measured over random ones), and a state near a
// decay of one keeps that over hundreds of tokens: this makes the mean -0.1 to 0.2.
// exp2 of it alone is 1 exactly, so a step of zero leaves the state as it is.
constexpr float kDecayBias = 0x1p-25f;

// softplus(v) = max(v, 0) + log(1 + e), e = exp(-|v|) <= 1, the logarithm as
// 2 atanh(s) with s = e / (2 + e) <= 1/3: the series s + s^3 / 3 + ... + s^13 / 13
// leaves less than 2 s^15 / 15 / (1 - s^2) out, 1.1e-8 at s = 1/3 and there 2^-26 of the
// logarithm, less of it at smaller s.  No cancellation at small
// e, where step sizes lie.  A NaN stays one (through e).
__device__ __forceinline__ float softplus_e(float v, float e) {
  const float s = e * fast_rcp(2.f + e);
  const float q = s * s, s2 = s + s;
  float p = fmaf(q, 1.f / 13.f, 1.f / 11.f);
  p = fmaf(q, p, 1.f / 9.f);
  p = fmaf(q, p, 1.f / 7.f);
  p = fmaf(q, p, 1.f / 5.f);
  p = fmaf(q, p, 1.f / 3.f);
  return fmaxf(v, 0.f) + fmaf(q * p, s2, s2);
}
__device__ __forceinline__ float softplus_fast(float v) {
  return softplus_e(v, ex2(-fabsf(v) * kLog2e));
}
// The same and its derivative sigmoid(v).
__device__ __forceinline__ float softplus_sig(float v, float& sig) {
  const float e = ex2(-fabsf(v) * kLog2e);
  const float r = fast_rcp(1.f + e);
  sig = v >= 0.f ? r : e * r;
  return softplus_e(v, e);
}

__device__ __forceinline__ float2 decay_arg(float2 delta, float2 a2) {
  return fma2(delta, a2, make_float2(kDecayBias, kDecayBias));
}

// Four consecutive elements as they lie in memory (a load in flight holds two
// registers in bf16), the ones past `n` zero.  `vec`: the row allows one vector.
template <typename T>
struct Raw4;
template <>
struct Raw4<__nv_bfloat16> {
  uint2 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int n, bool vec) {
    u = make_uint2(0u, 0u);
    if (n <= 0) return;
    if (vec && n >= 4) {
      u = *reinterpret_cast<const uint2*>(p);
    } else {
      const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
      u.x = q[0];
      if (n > 1) u.x |= (uint32_t)q[1] << 16;
      if (n > 2) u.y = q[2];
      if (n > 3) u.y |= (uint32_t)q[3] << 16;
    }
  }
  __device__ __forceinline__ void get(float (&v)[4]) const {
    v[0] = __uint_as_float(u.x << 16);
    v[1] = __uint_as_float(u.x & 0xffff0000u);
    v[2] = __uint_as_float(u.y << 16);
    v[3] = __uint_as_float(u.y & 0xffff0000u);
  }
};
template <>
struct Raw4<float> {
  float4 u;
  __device__ __forceinline__ void load(const float* p, int n, bool vec) {
    u = make_float4(0.f, 0.f, 0.f, 0.f);
    if (n <= 0) return;
    if (vec && n >= 4) {
      u = load4(p);
    } else {
      u.x = p[0];
      if (n > 1) u.y = p[1];
      if (n > 2) u.z = p[2];
      if (n > 3) u.w = p[3];
    }
  }
  __device__ __forceinline__ void get(float (&v)[4]) const {
    v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
  }
};

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

// A lane's states as pairs (NL = 1: one state and an idle second).
template <int NL>
constexpr int scan_pairs() { return NL == 1 ? 1 : NL / 2; }

// One token's row of B or C for a lane from shared memory.
template <int NL>
__device__ __forceinline__ void load_pairs(const float* p, float2 (&v)[scan_pairs<NL>()]) {
  if constexpr (NL == 1) {
    v[0] = make_float2(p[0], 0.f);
  } else if constexpr (NL == 2) {
    v[0] = *reinterpret_cast<const float2*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < NL; i += 4) {
      const float4 q = load4(p + i);
      v[i / 2] = make_float2(q.x, q.y);
      v[i / 2 + 1] = make_float2(q.z, q.w);
    }
  }
}
template <int NL>
__device__ __forceinline__ void store_pairs(float* p, const float2 (&v)[scan_pairs<NL>()]) {
  if constexpr (NL == 1) {
    p[0] = v[0].x;
  } else if constexpr (NL == 2) {
    *reinterpret_cast<float2*>(p) = v[0];
  } else {
#pragma unroll
    for (int i = 0; i < NL; i += 4)
      store4(p + i, make_float4(v[i / 2].x, v[i / 2].y, v[i / 2 + 1].x, v[i / 2 + 1].y));
  }
}
__device__ __forceinline__ float& pair_at(float2& v, int i) { return i ? v.y : v.x; }

// Tokens of the backward's tile (and the distance of the forward's checkpoints)
// for NL states a lane: half a tile's states of the lane's two channels, 64 of them at
// most, stay in registers.
template <int NL>
constexpr int scan_tile() { return NL <= 4 ? 16 : 64 / NL; }

}  // namespace gdn
