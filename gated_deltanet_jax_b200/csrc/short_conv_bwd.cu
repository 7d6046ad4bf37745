// Gradients of the short convolution (layer_ops.cu: a causal depthwise
// convolution over time, kernel K, optional bias, then SiLU or nothing).
//
// With xe the inputs behind the K - 1 rows of the entering window,
//   pre[t] = bias + sum_j w[j] xe[t + j],   y[t] = act(pre[t]),
//   dpre[t] = dy[t] act'(pre[t]),
//   dxe[s]  = sum_j w[j] dpre[s - j]   (+ the final window's gradient on the last K - 1 rows),
//   dw[j]   = sum_{b,t} dpre[t] xe[t + j],   dbias = sum_{b,t} dpre[t].
//
// In bytes HBM-bound: x and dy are read once and dx is written once (pre is formed
// again from x; it is not kept between the passes).  A thread owns two channels
// (the two halves of every multiply-add instruction) and walks a tile of tokens
// with x and dpre in sliding register windows; it copies its own words of the next
// twelve tokens to shared memory ahead of their use (in registers four tokens ahead
// fitted, and 83 registers: 110 us); a tile reads K - 1 rows before it and K - 1
// after it again, and inside it nothing is checked.  8 x 2048 x 4096 in bf16: 101 us
// with the sums below (4.0 TB/s), about 60 % of the issue slots; with four channels a
// thread 275 us (registers left too few warps), with every row's edges checked 155 us.
// The sums over tokens stay in registers (fp32) and leave as one partial row per tile,
// which a second kernel adds up in a fixed order: no atomics, the same bits on every
// run.
#include "gdn_common.cuh"
#include "gdn_internal.h"

namespace gdn {

namespace {

constexpr int kThreads = 128;
constexpr int kVec = 2;        // channels of a thread: a warp reads 128 bytes of bf16 a row
constexpr int kAhead = 4;      // tokens of a group
constexpr int kGroups = 4;     // groups in flight or worked on, in shared memory

// Blocks of an SM: by registers in bf16 (72 of them at K = 4), by shared memory in fp32.
constexpr int bwd_blocks(int K, int bytes) {
  return K > 6 ? 3 : K > 4 ? 4 : bytes == 2 ? 7 : 6;
}

// Two channels as they lie in memory.
template <typename T>
struct Raw2;
template <>
struct Raw2<float> {
  float2 u;
  __device__ __forceinline__ float2 get() const { return u; }
};
template <>
struct Raw2<__nv_bfloat16> {
  uint32_t u;
  __device__ __forceinline__ float2 get() const {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
};
template <typename T>
__device__ __forceinline__ Raw2<T> ldr(const T* p) {
  Raw2<T> r;
  r.u = *reinterpret_cast<const decltype(r.u)*>(p);
  return r;
}
// A thread's own copy of them to shared memory; nothing is read and zeros are written
// without `on` (p is then any valid address).
template <typename T>
__device__ __forceinline__ void copy2(Raw2<T>* dst, const T* p, bool on) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  const int n = on ? (int)sizeof(Raw2<T>) : 0;
  if constexpr (sizeof(Raw2<T>) == 4)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d), "l"(p), "r"(n)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(d), "l"(p), "r"(n)
                 : "memory");
}
__device__ __forceinline__ void st2(float* p, float2 v) { *reinterpret_cast<float2*>(p) = v; }
__device__ __forceinline__ void st2(__nv_bfloat16* p, float2 v) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v.x, v.y);
}

// Block (channel group, token tile, row b).  part [B * tiles][K + 1][C]: this
// tile's sums for dw[0 .. K - 1] and dbias.
template <typename Tin, int K>
__global__ void __launch_bounds__(kThreads, bwd_blocks(K, sizeof(Tin)))
short_conv_bwd_kernel(const Tin* __restrict__ x, const float* __restrict__ w,
                      const float* __restrict__ bias, const Tin* __restrict__ state_in,
                      const Tin* __restrict__ dy, const Tin* __restrict__ dstate_out,
                      Tin* __restrict__ dx, Tin* __restrict__ dstate_in,
                      float* __restrict__ part, int T, int C, int TT, int act) {
  const int c = (blockIdx.x * kThreads + threadIdx.x) * kVec;
  if (c >= C) return;
  const int b = blockIdx.z;
  const int t0 = blockIdx.y * TT;
  const int t1 = T - t0 > TT ? t0 + TT : T;
  constexpr int W = K > 1 ? K - 1 : 1;
  const float2 zero = make_float2(0.f, 0.f), one = make_float2(1.f, 1.f);
  float2 wk[K], win[W], dwin[W], dw[K], db = zero, bs = zero;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    wk[j] = ldr(w + (size_t)j * C + c).get();
    dw[j] = zero;
  }
  if (bias) bs = ldr(bias + c).get();
#pragma unroll
  for (int j = 0; j < W; ++j) win[j] = dwin[j] = zero;
  const size_t row0 = (size_t)b * T;
  // win[j] = xe[t + j] for the next token t (the K - 1 inputs before it)
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    const int tt = t0 - (K - 1) + j;
    if (tt >= 0)
      win[j] = ldr(x + (row0 + tt) * C + c).get();
    else if (state_in)
      win[j] = ldr(state_in + ((size_t)b * (K - 1) + (K - 1) + tt) * C + c).get();
  }
  // Token t closes row s = t - (K - 1) of dxe: dxe[s] takes dpre[s .. t].
  const int tend = t1 + K - 1, tload = min(T, tend);
  const size_t step = (size_t)kAhead * C;
  const Tin* xt = x + (row0 + t0) * C + c;   // the next rows to load
  const Tin* gt = dy + (row0 + t0) * C + c;
  Tin* ot = dx + (row0 + t0) * C + c;        // the row of token tb
  __shared__ Raw2<Tin> ring[kGroups][kAhead][2][kThreads];
  Raw2<Tin>* mine = &ring[0][0][0][threadIdx.x];
  auto fetch = [&](int tb, int slot) {
    Raw2<Tin>* r = mine + slot * (kAhead * 2 * kThreads);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const bool on = tb + i < tload;
      copy2(r + 2 * i * kThreads, on ? xt + (size_t)i * C : x, on);
      copy2(r + (2 * i + 1) * kThreads, on ? gt + (size_t)i * C : x, on);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    xt += step;
    gt += step;
  };
  // One token: dpre into the sums (own: a token of this tile) and the row it closes.
  auto token = [&](float2 xv, float2 d, bool own) {
    float2 pre = fma2(wk[K - 1], xv, bs);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) pre = fma2(wk[j], win[j], pre);
    if (act) {
      const float2 sg = make_float2(fast_sigmoid(pre.x), fast_sigmoid(pre.y));
      const float2 q = fma2(sg, make_float2(-1.f, -1.f), one);
      d = mul2(mul2(d, sg), fma2(pre, q, one));
    }
    if (own) {
      db = add2(db, d);
      dw[K - 1] = fma2(d, xv, dw[K - 1]);
#pragma unroll
      for (int j = 0; j < K - 1; ++j) dw[j] = fma2(d, win[j], dw[j]);
    }
    // dxe[s] = w[0] dpre[t] + w[1] dpre[t - 1] + ...
    float2 out = mul2(wk[0], d);
#pragma unroll
    for (int j = 1; j < K; ++j) out = fma2(wk[j], dwin[K - 1 - j], out);
#pragma unroll
    for (int j = 0; j + 1 < K - 1; ++j) {
      win[j] = win[j + 1];
      dwin[j] = dwin[j + 1];
    }
    if constexpr (K > 1) {
      win[K - 2] = xv;
      dwin[K - 2] = d;
    }
    return out;
  };
#pragma unroll
  for (int g = 0; g < kGroups - 1; ++g) fetch(t0 + g * kAhead, g);
  int slot = 0;
  for (int tb = t0; tb < tend; tb += kAhead, ot += step) {
    // (a thread reads what it copied itself: no barrier)
    asm volatile("cp.async.wait_group %0;" ::"n"(kGroups - 2) : "memory");
    float2 xv[kAhead], gv[kAhead];   // (gradients past the last token are zero)
    const Raw2<Tin>* r = mine + slot * (kAhead * 2 * kThreads);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      xv[i] = r[2 * i * kThreads].get();
      gv[i] = r[(2 * i + 1) * kThreads].get();
    }
    fetch(tb + (kGroups - 1) * kAhead, slot == 0 ? kGroups - 1 : slot - 1);
    slot = slot + 1 == kGroups ? 0 : slot + 1;
    if (tb >= t0 + K - 1 && tb + kAhead <= t1) {
      // inside the tile: every token its own, every row closed one of dx
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        st2(ot + (i - (K - 1)) * (ptrdiff_t)C, token(xv[i], gv[i], true));
      continue;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int t = tb + i;
      if (t >= tend) break;
      float2 out = token(xv[i], gv[i], t < t1);
      const int s = t - (K - 1);
      if (s < t0 && blockIdx.y != 0) continue;
      // the final window's rows are the inputs s = T - (K - 1) .. T - 1
      if (dstate_out && s >= T - (K - 1))
        out = add2(out, ldr(dstate_out + ((size_t)b * (K - 1) + (s - (T - (K - 1)))) * C + c)
                            .get());
      if (s >= 0)
        st2(dx + (row0 + s) * C + c, out);
      else if (dstate_in)
        st2(dstate_in + ((size_t)b * (K - 1) + (K - 1) + s) * C + c, out);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");   // (zeros past the last token)
  float* pr = part + ((size_t)b * gridDim.y + blockIdx.y) * (K + 1) * C + c;
#pragma unroll
  for (int j = 0; j < K; ++j) st2(pr + (size_t)j * C, dw[j]);
  st2(pr + (size_t)K * C, db);
}

template <typename Tin>
cudaError_t bwd_dispatch(const ShortConvBwdArgs& a, int TT, int tiles, cudaStream_t st) {
  const dim3 grid((a.C / kVec + kThreads - 1) / kThreads, tiles, a.B);
#define GDN_CONV_BWD_CASE(KK)                                                                  \
  case KK:                                                                                     \
    short_conv_bwd_kernel<Tin, KK><<<grid, kThreads, 0, st>>>(                                 \
        static_cast<const Tin*>(a.x), a.w, a.bias, static_cast<const Tin*>(a.state_in),        \
        static_cast<const Tin*>(a.dy), static_cast<const Tin*>(a.dstate_out),                  \
        static_cast<Tin*>(a.dx), static_cast<Tin*>(a.dstate_in), a.part, a.T, a.C, TT, a.act); \
    break;
  switch (a.K) {
    GDN_CONV_BWD_CASE(1)
    GDN_CONV_BWD_CASE(2)
    GDN_CONV_BWD_CASE(3)
    GDN_CONV_BWD_CASE(4)
    GDN_CONV_BWD_CASE(5)
    GDN_CONV_BWD_CASE(6)
    GDN_CONV_BWD_CASE(7)
    GDN_CONV_BWD_CASE(8)
    default: return cudaErrorInvalidValue;
  }
#undef GDN_CONV_BWD_CASE
  return cudaGetLastError();
}

// Token tiles such that the blocks fill the SMs a whole number of times, of at most 256
// tokens where eight times allow it (a tile reads 2 (K - 1) rows more than it owns).
// 8 x 2048 x 4096: 256 tokens, one wave, 101 us; 208 tokens 105, 352 tokens 118.
int conv_bwd_tile(int B, int T, int C, int K, int dtype) {
  const long long per = (long long)((C / kVec + kThreads - 1) / kThreads) * B;
  const long long slots = (long long)device_sm_count() * bwd_blocks(K, dtype == kBF16 ? 2 : 4);
  long long tt = T;
  for (int n = 1; per > 0 && n <= 8; ++n) {
    const long long tiles = n * slots / per;
    if (tiles > 0) tt = (T + tiles - 1) / tiles;
    if (tiles > 0 && tt <= 256) break;
  }
  if (tt < 16) tt = 16;
  if ((T + tt - 1) / tt > 65535) tt = ((long long)T + 65534) / 65535;
  return (int)tt;
}

}  // namespace

size_t short_conv_bwd_workspace_bytes(int B, int T, int C, int K, int dtype) {
  if (B <= 0 || T <= 0 || C <= 0) return 0;
  const int TT = conv_bwd_tile(B, T, C, K, dtype);
  return (size_t)B * ((T - 1) / TT + 1) * (K + 1) * C * sizeof(float);
}

cudaError_t launch_short_conv_bwd(const ShortConvBwdArgs& a, cudaStream_t st) {
  if (!short_conv_supported(a.C, a.K, a.dtype) || a.B > 65535) return cudaErrorInvalidValue;
  const int TT = conv_bwd_tile(a.B, a.T, a.C, a.K, a.dtype);
  const int tiles = (a.T - 1) / TT + 1;
  cudaError_t e = a.dtype == kBF16 ? bwd_dispatch<__nv_bfloat16>(a, TT, tiles, st)
                                   : bwd_dispatch<float>(a, TT, tiles, st);
  if (e != cudaSuccess) return e;
  // dw rows 0 .. K - 1, dbias row K of every partial
  const long long n = (long long)a.K * a.C;
  const SumSegments out{{a.dw, a.dbias, nullptr}, {n, a.C, 0}};
  return launch_sum_partials(a.part, (long long)a.B * tiles, n + a.C, out, st);
}

// ---------------------------------------------------------------------------
// Sums of partial rows, in a fixed order
// ---------------------------------------------------------------------------

namespace {

constexpr int kSumCols = 32;   // columns of a block
constexpr int kSumRows = 16;   // rows of threads, each over every 16th partial

__global__ void __launch_bounds__(kSumCols * kSumRows)
sum_partials_kernel(const float* __restrict__ part, const SumSegments out, long long parts,
                    long long stride) {
  __shared__ float red[kSumRows][kSumCols];
  const int col = threadIdx.x % kSumCols, row = threadIdx.x / kSumCols;
  const long long i = (long long)blockIdx.x * kSumCols + col;
  float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
  if (i < stride) {
    long long p = row;
    for (; p + 3 * kSumRows < parts; p += 4 * kSumRows) {
      s0 += part[p * stride + i];
      s1 += part[(p + kSumRows) * stride + i];
      s2 += part[(p + 2 * kSumRows) * stride + i];
      s3 += part[(p + 3 * kSumRows) * stride + i];
    }
    for (; p < parts; p += kSumRows) s0 += part[p * stride + i];
  }
  red[row][col] = (s0 + s1) + (s2 + s3);
  __syncthreads();
  if (row == 0 && i < stride) {
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < kSumRows; ++r) s += red[r][col];
    long long at = i;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (at >= 0 && at < out.n[k] && out.dst[k]) out.dst[k][at] = s;
      at -= out.n[k];
    }
  }
}

}  // namespace

cudaError_t launch_sum_partials(const float* part, long long parts, long long stride,
                                const SumSegments& out, cudaStream_t st) {
  if (stride <= 0) return cudaSuccess;
  const long long blocks = (stride + kSumCols - 1) / kSumCols;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  sum_partials_kernel<<<(unsigned)blocks, kSumCols * kSumRows, 0, st>>>(part, out, parts, stride);
  return cudaGetLastError();
}

}  // namespace gdn
