// The layer's elementwise work around the delta-rule op, for the shapes whose
// op kernels do not fuse it (model.py:15-53, 119-153):
//
//   short_conv_kernel   ShortConvolution (model.py:15-40): a causal depthwise
//                       convolution over time, kernel K, optional bias, then SiLU,
//                       with an optional state of the K - 1 inputs before the
//                       first token (decode) and the K - 1 last inputs out;
//   gated_norm_kernel   FusedRMSNormGated (model.py:41-53) over the op's output:
//                       y = o rsqrt(mean(o^2) + eps) w silu(gate), in place.
//
// Each element is read once and written once: the norm is HBM-bound, the convolution
// takes 70 % of the issue slots at 4 TB/s.  A thread of
// the norm owns 16-byte vectors (8 bf16 or 4 fp32), one of the convolution four
// channels.
#include <type_traits>

#include "gdn_common.cuh"
#include "gdn_internal.h"

namespace gdn {

namespace {

template <typename Tin>
struct Vec16;
template <>
struct Vec16<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void load(const __nv_bfloat16* p, float (&f)[N]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = __bfloat1622float2(h[i]);
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  }
  __device__ static void store(__nv_bfloat16* p, const float (&f)[N]) {
    uint4 u;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = u;
  }
};
template <>
struct Vec16<float> {
  static constexpr int N = 4;
  __device__ static void load(const float* p, float (&f)[N]) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w;
  }
  __device__ static void store(float* p, const float (&f)[N]) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  }
};

__device__ __forceinline__ float silu_acc(float x) { return x / (1.f + expf(-x)); }

// Four consecutive channels (8 bytes of bf16, 16 of fp32): with eight of bf16 the
// windows and weights of K = 4 take 139 registers, and too few warps fit an SM
// to cover the loads (142 us at 8 x 2048 x 4096).
template <typename Tin>
struct Vec4 {
  static constexpr int N = 4;
  using Raw = typename std::conditional<sizeof(Tin) == 2, uint2, float4>::type;
  __device__ static Raw load_raw(const Tin* p) { return *reinterpret_cast<const Raw*>(p); }
  __device__ static void get(const uint2& u, float2 (&f)[N / 2]) {
    f[0] = make_float2(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u));
    f[1] = make_float2(__uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
  }
  __device__ static void get(const float4& u, float2 (&f)[N / 2]) {
    f[0] = make_float2(u.x, u.y);
    f[1] = make_float2(u.z, u.w);
  }
  __device__ static void store(Tin* p, const float (&f)[N]) {
    store4(p, make_float4(f[0], f[1], f[2], f[3]));
  }
};

// silu_acc of four values to be rounded to bf16, with the bits that silu_acc gives and
// fewer instructions: formed from the fast exponential and reciprocal, and again by
// silu_acc where that could round to another bf16.  For v >= -8, in units of 2^-24 of the
// result: the fast form's argument v log2 e is off by half of 2^-20 (5.5 with the ln 2)
// and by the constant's rounding (1.8), the exponential by 4, sum, reciprocal and product
// by 1, 2 and 1; silu_acc by 4 (expf) and 1 and 1.  Together 21.3, which is at most 21.3
// of the fp32 result's last places, so the two can only round apart when the fast
// result's low half lies within 24 of the tie at 0x8000 (one in 1340 values).  Below -8
// (infinities among them) silu_acc serves alone; a NaN stays one.  The convolution of
// 8 x 2048 x 4096: 93 us with silu_acc throughout, 66 so (4.0 TB/s).
constexpr uint32_t kTieBand = 24;
__device__ __forceinline__ void silu_acc_bf16(float (&v)[4]) {
  float f[4];
  auto near_tie = [](float r) {
    return ((__float_as_uint(r) - (0x8000u - kTieBand)) & 0xffffu) <= 2 * kTieBand;
  };
  bool again = fminf(fminf(v[0], v[1]), fminf(v[2], v[3])) < -8.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[e] = v[e] * fast_sigmoid(v[e]);
    again |= near_tie(f[e]);
  }
  if (again) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (v[e] < -8.f || near_tie(f[e])) f[e] = silu_acc(v[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = f[e];
}

constexpr int kConvThreads = 128;
constexpr int kConvAhead = 4;

// x, y [B, T, C]; w [K, C] fp32 (the flax kernel (K, 1, C) as stored); bias [C]
// fp32 or NULL;
// state_in / state_out [B, K - 1, C] in x's dtype (NULL: zeros / not wanted).
// Block (channel vectors, b, token tile of TT).  The K - 1 inputs before the
// tile are read as its halo (from the state before token 0); the tile then
// slides a register window.  The last tile writes the final K - 1 inputs.
template <typename Tin, int K>
__global__ void __launch_bounds__(kConvThreads, sizeof(Tin) == 2 && K <= 4 ? 6 : 1)
short_conv_kernel(const Tin* __restrict__ x, const float* __restrict__ w,
                  const float* __restrict__ bias, const Tin* state_in, Tin* state_out, Tin* __restrict__ y, int T, int C,
                  int TT, int act) {
  using V = Vec4<Tin>;
  constexpr int N = V::N;
  const int c = (blockIdx.x * kConvThreads + threadIdx.x) * N;
  if (c >= C) return;
  const int b = blockIdx.y;
  const int t0 = blockIdx.z * TT;
  const int t1 = T - t0 > TT ? t0 + TT : T;
  float2 wk[K][N / 2], bs[N / 2];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const float4 q = load4(w + (size_t)j * C + c);
    wk[j][0] = make_float2(q.x, q.y);
    wk[j][1] = make_float2(q.z, q.w);
  }
  const float4 bq = bias ? load4(bias + c) : make_float4(0.f, 0.f, 0.f, 0.f);
  bs[0] = make_float2(bq.x, bq.y);
  bs[1] = make_float2(bq.z, bq.w);
  const Tin* xb = x + (size_t)b * T * C + c;
  // win[j] = input at token t - (K - 1) + j for the next output t
  float2 win[K > 1 ? K - 1 : 1][N / 2];
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    const int tt = t0 - (K - 1) + j;
    if (tt >= 0) {
      V::get(V::load_raw(xb + (size_t)tt * C), win[j]);
    } else if (state_in) {
      V::get(V::load_raw(state_in + ((size_t)b * (K - 1) + (K - 1) + tt) * C + c), win[j]);
    } else {
#pragma unroll
      for (int e = 0; e < N / 2; ++e) win[j][e] = make_float2(0.f, 0.f);
    }
  }
  typename V::Raw nxt[kConvAhead];   // loads of four tokens in flight under four others' work
  const Tin* xt = xb + (size_t)t0 * C;   // the next row to load
  Tin* yt = y + ((size_t)b * T + t0) * C + c;
  auto fetch = [&](int tb) {
#pragma unroll
    for (int i = 0; i < kConvAhead; ++i)
      if (tb + i < t1) nxt[i] = V::load_raw(xt + (size_t)i * C);
    xt += (size_t)kConvAhead * C;
  };
  fetch(t0);
  for (int tb = t0; tb < t1; tb += kConvAhead) {
    float2 cur[kConvAhead][N / 2];
#pragma unroll
    for (int i = 0; i < kConvAhead; ++i) V::get(nxt[i], cur[i]);
    if (tb + kConvAhead < t1) fetch(tb + kConvAhead);
#pragma unroll
    for (int i = 0; i < kConvAhead; ++i, yt += C) {
      if (tb + i >= t1) break;
      float out[N];
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        float2 acc = mul2(wk[K - 1][e], cur[i][e]);
#pragma unroll
        for (int j = 0; j < K - 1; ++j) acc = fma2(wk[j][e], win[j][e], acc);
        if (bias) acc = add2(acc, bs[e]);
        out[2 * e] = acc.x;
        out[2 * e + 1] = acc.y;
      }
      if (act) {
        if constexpr (sizeof(Tin) == 2) {
          silu_acc_bf16(out);
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) out[e] = silu_acc(out[e]);
        }
      }
      V::store(yt, out);
#pragma unroll
      for (int j = 0; j + 1 < K - 1; ++j)
#pragma unroll
        for (int e = 0; e < N / 2; ++e) win[j][e] = win[j + 1][e];
      if constexpr (K > 1) {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) win[K - 2][e] = cur[i][e];
      }
    }
  }
  if (state_out && blockIdx.z == gridDim.z - 1) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      const float v[N] = {win[j][0].x, win[j][0].y, win[j][1].x, win[j][1].y};
      V::store(state_out + ((size_t)b * (K - 1) + j) * C + c, v);
    }
  }
}

// One warp per row of dv elements (rows = tokens x heads): y = o rsqrt(mean(o^2)
// + eps) w (silu(gate) when gate is given).  o and y may be the same array.
constexpr int kNormWarps = 8;
constexpr int kNormMaxVec = 4;  // 16-byte vectors per lane: dv <= 4 * 32 * N

template <typename Tin>
__global__ void __launch_bounds__(kNormWarps * 32)
gated_norm_kernel(const Tin* o, const Tin* __restrict__ gate, const float* __restrict__ wt,
                  Tin* y, long long rows, int dv, float eps) {
  using V = Vec16<Tin>;
  constexpr int N = V::N;
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * kNormWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int nvec = dv / N;
  const Tin* orow = o + row * dv;
  float v[kNormMaxVec][N];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < kNormMaxVec; ++i) {
    const int cv = lane + 32 * i;
    if (cv < nvec) {
      V::load(orow + cv * N, v[i]);
#pragma unroll
      for (int e = 0; e < N; ++e) ss = fmaf(v[i][e], v[i][e], ss);
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
  const float r = rsqrtf(ss / (float)dv + eps);
#pragma unroll
  for (int i = 0; i < kNormMaxVec; ++i) {
    const int cv = lane + 32 * i;
    if (cv < nvec) {
      float gv[N], out[N];
      if (gate) V::load(gate + row * dv + cv * N, gv);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float wv = wt[cv * N + e];
        out[e] = v[i][e] * r * wv * (gate ? silu_acc(gv[e]) : 1.f);
      }
      V::store(y + row * dv + cv * N, out);
    }
  }
}

template <typename Tin>
cudaError_t conv_dispatch(const void* x, const float* w, const float* bias, const void* si,
                          void* so, void* y, int B, int T, int C, int K, int TT, int act, cudaStream_t st) {
  constexpr int N = Vec4<Tin>::N;
  const dim3 grid((C / N + kConvThreads - 1) / kConvThreads, B, (T - 1) / TT + 1);
  const Tin* xi = static_cast<const Tin*>(x);
  const Tin* s_in = static_cast<const Tin*>(si);
  Tin* sout = static_cast<Tin*>(so);
  Tin* yo = static_cast<Tin*>(y);
#define GDN_CONV_CASE(KK)                                                                   \
  case KK:                                                                                  \
    short_conv_kernel<Tin, KK><<<grid, kConvThreads, 0, st>>>(xi, w, bias, s_in, sout, yo, T, C, \
                                                              TT, act);                     \
    break;
  switch (K) {
    GDN_CONV_CASE(1)
    GDN_CONV_CASE(2)
    GDN_CONV_CASE(3)
    GDN_CONV_CASE(4)
    GDN_CONV_CASE(5)
    GDN_CONV_CASE(6)
    GDN_CONV_CASE(7)
    GDN_CONV_CASE(8)
    default: return cudaErrorInvalidValue;
  }
#undef GDN_CONV_CASE
  return cudaGetLastError();
}

}  // namespace

bool short_conv_supported(int C, int K, int dtype) {
  const int n = dtype == kBF16 ? 8 : 4;
  return K >= 1 && K <= kShortConvMaxK && C > 0 && C % n == 0;
}

cudaError_t launch_short_conv(const void* x, const float* w, const float* bias,
                              const void* state_in, void* state_out, void* y, int B, int T, int C, int K, int act,
                              int dtype, cudaStream_t st) {
  if (B == 0 || T == 0) return cudaSuccess;
  if (!short_conv_supported(C, K, dtype) || B > 65535) return cudaErrorInvalidValue;
  // Token tiles of 64, shorter ones (down to 16) where 64 leave SMs with fewer
  // than eight blocks: a tile is a serial walk.  A state updated in place is read
  // by the first tile and written by the last, so it takes one tile over all T.
  int TT = 64;
  const long long per = (long long)((C / 4 + kConvThreads - 1) / kConvThreads) * B;
  while (TT > 16 && per * ((T - 1) / TT + 1) < 8LL * device_sm_count()) TT /= 2;
  if (state_in && state_in == state_out) TT = T;
  if ((T - 1) / TT + 1 > 65535) TT = (T - 1) / 65535 + 1;
  return dtype == kBF16
             ? conv_dispatch<__nv_bfloat16>(x, w, bias, state_in, state_out, y, B, T, C, K, TT, act,
                                            st)
             : conv_dispatch<float>(x, w, bias, state_in, state_out, y, B, T, C, K, TT, act, st);
}

bool gated_norm_supported(int dv, int dtype) {
  const int n = dtype == kBF16 ? 8 : 4;
  return dv > 0 && dv % n == 0 && dv <= kNormMaxVec * 32 * n;
}

cudaError_t launch_gated_norm(const void* o, const void* gate, const float* w, void* y,
                              long long rows, int dv, float eps, int dtype, cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  if (!gated_norm_supported(dv, dtype)) return cudaErrorInvalidValue;
  const long long blocks = (rows + kNormWarps - 1) / kNormWarps;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (dtype == kBF16)
    gated_norm_kernel<__nv_bfloat16><<<(unsigned)blocks, kNormWarps * 32, 0, st>>>(
        static_cast<const __nv_bfloat16*>(o), static_cast<const __nv_bfloat16*>(gate), w,
        static_cast<__nv_bfloat16*>(y), rows, dv, eps);
  else
    gated_norm_kernel<float><<<(unsigned)blocks, kNormWarps * 32, 0, st>>>(
        static_cast<const float*>(o), static_cast<const float*>(gate), w,
        static_cast<float*>(y), rows, dv, eps);
  return cudaGetLastError();
}

}  // namespace gdn
