// Selective state-space scan, forward (no counterpart in the reference, whose
// only recurrence is the gated delta rule).  Per channel c with N states,
//   delta_t = softplus(dt_t + dt_bias)          (or dt_t + dt_bias)
//   h_t[n]  = exp(delta_t A[n]) h_{t-1}[n] + delta_t x_t B_t[n]
//   y_t     = (sum_n C_t[n] h_t[n] + D x_t) silu(z_t)
// with an fp32 state.  B and C are shared by the channels of a group.
//
// What it has to move is x, dt, z and y once (8 bytes a token and channel in
// bf16); what it has to compute is one exponential and four multiply-adds per
// state, which at N = 16 takes longer than the bytes.  Four lanes share a
// channel, each with a quarter of its states in registers, so the exponentials
// of a token run side by side and few sequences still fill the SMs.  A block
// owns 32 channels of one row and walks tiles of 32 tokens: every thread forms
// delta and delta x of eight (token, channel) pairs into shared memory with the
// next tile's loads in flight, all lanes then run the recurrence over the tile,
// and four tokens' read-outs at a time are summed over the four lanes in three
// shuffles.
#include "selective_scan_common.cuh"

namespace gdn {

namespace {

constexpr int kTT = 32;   // tokens of a tile
constexpr int kRows = kTT * kScanCh / (kScanThreads * 4);   // staging rows per thread

template <typename T, int NL>
__global__ void __launch_bounds__(kScanThreads)
scan_fwd_kernel(const ScanArgs a, int tiles_per_group, int vec) {
  constexpr int NP = NL * kScanLanes;
  constexpr int CK = scan_tile<NL>();
  __shared__ float2 sDU[kTT][kScanCh];
  __shared__ float sY[kTT][kScanCh + 8];   // padded: four tokens of eight channels at once
  __shared__ __align__(16) float sB[kTT][NP], sC[kTT][NP];

  const int tid = threadIdx.x, lane = tid & 31;
  const int Cg = a.C / a.G;
  const int grp = blockIdx.x / tiles_per_group;
  const int cl0 = (blockIdx.x % tiles_per_group) * kScanCh;   // first channel in the group
  const int nch = min(kScanCh, Cg - cl0);
  const int c0 = grp * Cg + cl0;
  const int b = blockIdx.y;
  const T* x = static_cast<const T*>(a.x);
  const T* dt = static_cast<const T*>(a.dt);
  const T* z = static_cast<const T*>(a.z);
  const T* Bp = static_cast<const T*>(a.Bm) + ((size_t)b * a.T * a.G + grp) * a.N;
  const T* Cp = static_cast<const T*>(a.Cm) + ((size_t)b * a.T * a.G + grp) * a.N;
  T* y = static_cast<T*>(a.y);

  // the lane's channel and states
  const int chl = tid / kScanLanes, q = tid % kScanLanes;
  const bool chan = chl < nch;
  float A2[NL], h[NL];
  const size_t st = ((size_t)b * a.C + c0 + chl) * a.N + q * NL;
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const bool ok = chan && q * NL + i < a.N;
    A2[i] = ok ? a.A[(size_t)(c0 + chl) * a.N + q * NL + i] * kLog2e : 0.f;
    h[i] = ok && a.h0 ? a.h0[st + i] : 0.f;
  }
  // the staging role: channels sc .. sc + 3 of rows sr, sr + 16
  const int sc = tid % 8 * 4, sr = tid / 8;
  const int sn = nch - sc;
  float bias[4], Dv[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    bias[e] = a.dt_bias && e < sn ? a.dt_bias[c0 + sc + e] : 0.f;
    Dv[e] = a.D && e < sn ? a.D[c0 + sc + e] : 0.f;
  }
  const size_t row0 = (size_t)b * a.T;
  float xv[kRows][4], dv[kRows][4], zv[kRows][4];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int t = t0 + sr + r * 16;
      const int n = t < a.T ? sn : 0;
      const size_t off = (row0 + t) * a.C + c0 + sc;
      load_ch4(x + off, n, vec, xv[r]);
      load_ch4(dt + off, n, vec, dv[r]);
      if (z) load_ch4(z + off, n, vec, zv[r]);
    }
  };
  fetch(0);
  for (int t0 = 0; t0 < a.T; t0 += kTT) {
    float xs[kRows][4], zs[kRows][4];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int tl = sr + r * 16;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float sig, d = dv[r][e] + bias[e];
        if (a.softplus) d = softplus_sig(d, sig);
        if (t0 + tl >= a.T) d = 0.f;   // past the end: the state stays
        sDU[tl][sc + e] = make_float2(d, d * xv[r][e]);
        xs[r][e] = xv[r][e];
        zs[r][e] = z ? zv[r][e] : 0.f;
      }
    }
    for (int i = tid; i < kTT * NP; i += kScanThreads) {
      const int tl = i / NP, n = i % NP;
      const bool ok = t0 + tl < a.T && n < a.N;
      const size_t off = (size_t)(t0 + tl) * a.G * a.N + n;
      sB[tl][n] = load1(Bp + off, ok);
      sC[tl][n] = load1(Cp + off, ok);
    }
    __syncthreads();
    if (t0 + kTT < a.T) fetch(t0 + kTT);
#pragma unroll 1
    for (int g = 0; g < kTT; g += 4) {
      if (a.ckpt && g % CK == 0 && t0 + g < a.T && chan) {
        float* ck = a.ckpt + (((size_t)b * a.nck + (t0 + g) / CK) * a.C + c0 + chl) * NP + q * NL;
        store_states(ck, h);
      }
      float ys[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 du = sDU[g + j][chl];
        float acc = 0.f;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const float dec = ex2(du.x * A2[i]);
          h[i] = fmaf(dec, h[i], du.y * sB[g + j][q * NL + i]);
          acc = fmaf(sC[g + j][q * NL + i], h[i], acc);
        }
        ys[j] = acc;
      }
      sY[g + q][chl] = quad_sum4(ys[0], ys[1], ys[2], ys[3], lane);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int tl = sr + r * 16, t = t0 + tl;
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = fmaf(Dv[e], xs[r][e], sY[tl][sc + e]);
        if (z) o[e] *= __fdividef(zs[r][e], 1.f + __expf(-zs[r][e]));
      }
      if (t < a.T) store_ch4(y + (row0 + t) * a.C + c0 + sc, sn, vec, o);
    }
  }
  if (a.hT && chan) {
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (q * NL + i < a.N) a.hT[st + i] = h[i];
  }
}

// One token (decode): HBM-bound on the state, which is read and written once.
// A lane owns four states (16 bytes), N / 4 lanes a channel; in place when
// h0 == hT, since a lane reads its states before it writes them.
template <typename T, int L>
__global__ void __launch_bounds__(256)
scan_step_kernel(const ScanArgs a) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const int b = blockIdx.y, q = (int)(id % L);
  const long long cl = id / L;
  const bool chan = cl < a.C;
  const int c = chan ? (int)cl : 0;
  const int N = 4 * L, grp = c / (a.C / a.G);
  const size_t row = (size_t)b * a.C + c;
  const size_t st = row * N + 4 * q;
  const size_t bc = ((size_t)b * a.G + grp) * N + 4 * q;
  float4 h = make_float4(0.f, 0.f, 0.f, 0.f);
  if (a.h0 && chan) h = load4_stream(a.h0 + st);
  const float4 A = load4(a.A + (size_t)c * N + 4 * q);
  const float4 B = load4(static_cast<const T*>(a.Bm) + bc);
  const float4 Cv = load4(static_cast<const T*>(a.Cm) + bc);
  const float x = to_f32(static_cast<const T*>(a.x)[row]);
  float d = to_f32(static_cast<const T*>(a.dt)[row]) + (a.dt_bias ? a.dt_bias[c] : 0.f);
  float sig;
  if (a.softplus) d = softplus_sig(d, sig);
  const float u = d * x, d2 = d * kLog2e;
  h.x = fmaf(ex2(d2 * A.x), h.x, u * B.x);
  h.y = fmaf(ex2(d2 * A.y), h.y, u * B.y);
  h.z = fmaf(ex2(d2 * A.z), h.z, u * B.z);
  h.w = fmaf(ex2(d2 * A.w), h.w, u * B.w);
  if (a.hT && chan) store4_stream(a.hT + st, h);
  float y = fmaf(Cv.x, h.x, fmaf(Cv.y, h.y, fmaf(Cv.z, h.z, Cv.w * h.w)));
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  if (q == 0 && chan) {
    if (a.D) y = fmaf(a.D[c], x, y);
    if (a.z) {
      const float zv = to_f32(static_cast<const T*>(a.z)[row]);
      y *= __fdividef(zv, 1.f + __expf(-zv));
    }
    static_cast<T*>(a.y)[row] = from_f32<T>(y);
  }
}

template <typename T, int L>
cudaError_t launch_step(const ScanArgs& a, cudaStream_t st) {
  const long long blocks = ((long long)a.C * L + 255) / 256;
  scan_step_kernel<T, L><<<dim3((unsigned)blocks, a.B), 256, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t fwd_dispatch(const ScanArgs& a, cudaStream_t st) {
  if (a.T == 1 && !a.ckpt) {
    switch (a.N) {
      case 4: return launch_step<T, 1>(a, st);
      case 8: return launch_step<T, 2>(a, st);
      case 16: return launch_step<T, 4>(a, st);
      case 32: return launch_step<T, 8>(a, st);
      case 64: return launch_step<T, 16>(a, st);
      default: break;   // the general kernel
    }
  }
  const int Cg = a.C / a.G;
  const int tpg = (Cg + kScanCh - 1) / kScanCh;
  const int vec = a.C % 4 == 0 && Cg % 4 == 0;
  const dim3 grid((unsigned)(tpg * a.G), a.B);
  if (a.N <= 4) scan_fwd_kernel<T, 1><<<grid, kScanThreads, 0, st>>>(a, tpg, vec);
  else if (a.N <= 8) scan_fwd_kernel<T, 2><<<grid, kScanThreads, 0, st>>>(a, tpg, vec);
  else if (a.N <= 16) scan_fwd_kernel<T, 4><<<grid, kScanThreads, 0, st>>>(a, tpg, vec);
  else if (a.N <= 32) scan_fwd_kernel<T, 8><<<grid, kScanThreads, 0, st>>>(a, tpg, vec);
  else scan_fwd_kernel<T, 16><<<grid, kScanThreads, 0, st>>>(a, tpg, vec);
  return cudaGetLastError();
}

}  // namespace

int scan_padded_states(int N) { return N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }

int scan_checkpoint_tokens(int N) { return N <= 16 ? 16 : N <= 32 ? 8 : 4; }

size_t scan_checkpoint_bytes(int B, int T, int C, int N) {
  const int k = scan_checkpoint_tokens(N);
  return (size_t)B * ((T + k - 1) / k) * C * scan_padded_states(N) * sizeof(float);
}

cudaError_t launch_selective_scan(const ScanArgs& a, cudaStream_t st) {
  if (a.B == 0 || a.C == 0) return cudaSuccess;
  return a.dtype == kBF16 ? fwd_dispatch<__nv_bfloat16>(a, st) : fwd_dispatch<float>(a, st);
}

}  // namespace gdn
