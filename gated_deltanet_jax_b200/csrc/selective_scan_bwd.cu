// Selective state-space scan, backward (formulas of the forward in
// selective_scan.cu).  With dyp = dy silu(z) and the adjoint state r,
//   r_t[n]   = C_t[n] dyp_t + a_{t+1}[n] r_{t+1}[n]      (a_t = exp(delta_t A)),
//   dB_t[n]  = sum_c r delta x,      dC_t[n] = sum_c dyp h_t[n],
//   dx_t     = delta_t sum_n r B + D dyp,
//   ddelta_t = sum_n r a_t h_{t-1} A + x_t sum_n r B,    ddt = ddelta sigmoid(dt + bias),
//   dA[n]    = sum_t r delta a_t h_{t-1},   dD = sum dyp x,   dz = dy ypre silu'(z).
//
// A block owns 32 channels of one row, four lanes a channel as in the forward,
// and walks its tiles backwards.  A tile restarts from the state that the
// forward kept at its first token (one fp32 state every 16 tokens at N <= 16:
// four bytes a token and channel, less time than forming it again), runs the
// recurrence over the tile with the decay factors in registers and the states
// in shared memory, then the adjoint recurrence backwards.  Bound by issue
// slots: about a dozen multiply-adds a state and token, and seven shuffles a
// token that sum dB and dC over a warp's eight channels.  Sums over channels,
// rows and tokens leave as one partial per block and are added up in a fixed
// order by further kernels: no atomics, the same bits on every run.
#include "selective_scan_common.cuh"

namespace gdn {

namespace {

// Reduces NV values per lane over the eight channels of a warp (lane bits 2 to
// 4), halving the values kept where it can; afterwards the lane holds
// max(1, NV / 8) totals, value index first + i.
template <int NV>
struct ChanSum {
  static constexpr int K1 = NV >= 2 ? NV / 2 : 1;
  static constexpr int K2 = NV >= 4 ? NV / 4 : 1;
  static constexpr int K3 = NV >= 8 ? NV / 8 : 1;
  template <int NI, int NO>
  __device__ __forceinline__ static void half(const float (&v)[NI], float (&o)[NO], int mask,
                                              bool up) {
    if constexpr (NI == 2 * NO) {
#pragma unroll
      for (int i = 0; i < NO; ++i) {
        const float keep = up ? v[NO + i] : v[i], give = up ? v[i] : v[NO + i];
        o[i] = keep + __shfl_xor_sync(0xffffffffu, give, mask);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NO; ++i) o[i] = v[i] + __shfl_xor_sync(0xffffffffu, v[i], mask);
    }
  }
  __device__ __forceinline__ static void run(const float (&v)[NV], float (&o)[K3], int lane) {
    float p[K1], q[K2];
    half(v, p, 4, (lane & 4) != 0);
    half(p, q, 8, (lane & 8) != 0);
    half(q, o, 16, (lane & 16) != 0);
  }
  __device__ __forceinline__ static int first(int lane) {
    int f = 0;
    if (NV >= 2 && (lane & 4)) f += NV / 2;
    if (NV >= 4 && (lane & 8)) f += NV / 4;
    if (NV >= 8 && (lane & 16)) f += NV / 8;
    return f;
  }
};

template <int NL>
struct BwdSmem {
  static constexpr int CK = scan_tile<NL>();
  static constexpr int NP = NL * kScanLanes;
  float h[CK][kScanThreads][NL];          // states after each token of the tile
  float4 p[CK][kScanCh];                  // delta, delta x, dyp, x
  float o[3][CK][kScanCh + 8];            // sum C h, sum r B, sum r a h A
  float B[CK][NP];
  float C[CK][NP];
  float red[kScanThreads / 32][CK][2 * NP];   // a warp's dB and dC
};

template <typename T, int NL>
__global__ void __launch_bounds__(kScanThreads)
scan_bwd_kernel(const ScanBwdArgs a, int tiles_per_group, int vec, float* __restrict__ pBC,
                float* __restrict__ pA, float* __restrict__ pD) {
  using S = BwdSmem<NL>;
  constexpr int CK = S::CK, NP = S::NP;
  constexpr int RPT = CK * kScanCh / (kScanThreads * 4);    // staging rows per thread
  constexpr int ROWS = RPT > 0 ? RPT : 1;
  constexpr int RT = CK < 16 ? CK : 16;                     // rows of one staging pass
  extern __shared__ __align__(16) unsigned char smem_raw[];
  S& s = *reinterpret_cast<S*>(smem_raw);

  const ScanArgs& f = a.fwd;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int Cg = f.C / f.G;
  const int grp = blockIdx.x / tiles_per_group;
  const int cl0 = (blockIdx.x % tiles_per_group) * kScanCh;
  const int nch = min(kScanCh, Cg - cl0);
  const int c0 = grp * Cg + cl0;
  const int b = blockIdx.y;
  const T* x = static_cast<const T*>(f.x);
  const T* dt = static_cast<const T*>(f.dt);
  const T* z = static_cast<const T*>(f.z);
  const T* dy = static_cast<const T*>(a.dy);
  const T* Bp = static_cast<const T*>(f.Bm) + ((size_t)b * f.T * f.G + grp) * f.N;
  const T* Cp = static_cast<const T*>(f.Cm) + ((size_t)b * f.T * f.G + grp) * f.N;

  const int chl = tid / kScanLanes, q = tid % kScanLanes;
  const bool chan = chl < nch;
  float A2[NL], ar[NL], dA[NL];
  const size_t st = ((size_t)b * f.C + c0 + chl) * f.N + q * NL;
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const bool ok = chan && q * NL + i < f.N;
    A2[i] = ok ? f.A[(size_t)(c0 + chl) * f.N + q * NL + i] * kLog2e : 0.f;
    ar[i] = ok && a.dhT ? a.dhT[st + i] : 0.f;
    dA[i] = 0.f;
  }
  const int sc = tid % 8 * 4, sr = tid / 8;
  const bool stages = sr < CK;
  const int sn = nch - sc;
  float bias[4], Dv[4], accD[4], accB[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    bias[e] = f.dt_bias && e < sn ? f.dt_bias[c0 + sc + e] : 0.f;
    Dv[e] = f.D && e < sn ? f.D[c0 + sc + e] : 0.f;
    accD[e] = accB[e] = 0.f;
  }
  const size_t row0 = (size_t)b * f.T;
  const int ntiles = (f.T + CK - 1) / CK;
  Raw4<T> xr[ROWS], dr[ROWS], zr[ROWS], gr[ROWS];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int t = t0 + sr + r * RT;
      const int n = stages && t < f.T ? sn : 0;
      const size_t off = (row0 + t) * f.C + c0 + sc;
      xr[r].load(x + off, n, vec);
      dr[r].load(dt + off, n, vec);
      gr[r].load(dy + off, n, vec);
      if (z) zr[r].load(z + off, n, vec);
    }
  };
  if (ntiles > 0) fetch((ntiles - 1) * CK);
  for (int k = ntiles - 1; k >= 0; --k) {
    const int t0 = k * CK;
    // kept for the tile's last step: sigmoid(dt + bias), dy silu'(z), delta, dyp, x
    float ks[ROWS][4], kz[ROWS][4];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int tl = sr + r * RT;
      float xv[4], dv[4], gv[4], zv[4];
      xr[r].get(xv);
      dr[r].get(dv);
      gr[r].get(gv);
      if (z) zr[r].get(zv);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float sig = 1.f, d = dv[e] + bias[e];
        if (f.softplus) d = softplus_sig(d, sig);
        if (t0 + tl >= f.T) d = 0.f;
        float g = gv[e];
        kz[r][e] = 0.f;
        if (z) {
          const float zz = zv[e];
          const float sz = fast_sigmoid(zz);
          kz[r][e] = g * (sz * fmaf(zz, 1.f - sz, 1.f));
          g *= zz * sz;
        }
        ks[r][e] = sig;
        if (stages) s.p[tl][sc + e] = make_float4(d, d * xv[e], g, xv[e]);
      }
    }
    for (int i = tid; i < CK * NP; i += kScanThreads) {
      const int tl = i / NP, n = i % NP;
      const bool ok = t0 + tl < f.T && n < f.N;
      const size_t off = (size_t)(t0 + tl) * f.G * f.N + n;
      s.B[tl][n] = load1(Bp + off, ok);
      s.C[tl][n] = load1(Cp + off, ok);
    }
    float h0[NL];
    if (chan) {
      load_states(f.ckpt + (((size_t)b * f.nck + k) * f.C + c0 + chl) * NP + q * NL, h0);
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) h0[i] = 0.f;
    }
    __syncthreads();
    if (k > 0) fetch((k - 1) * CK);

    // the recurrence over the tile
    float dec[CK][NL], h[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) h[i] = h0[i];
#pragma unroll
    for (int g = 0; g < CK; g += 4) {
      float ys[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 p = s.p[g + j][chl];
        float acc = 0.f;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          dec[g + j][i] = ex2(p.x * A2[i]);
          h[i] = fmaf(dec[g + j][i], h[i], p.y * s.B[g + j][q * NL + i]);
          acc = fmaf(s.C[g + j][q * NL + i], h[i], acc);
        }
        ys[j] = acc;
        store_states(s.h[g + j][tid], h);
      }
      if (z) s.o[0][g + q][chl] = quad_sum4(ys[0], ys[1], ys[2], ys[3], lane);
    }
    // the adjoint recurrence, backwards; h holds h_t and becomes h_{t-1}
#pragma unroll
    for (int g = CK - 4; g >= 0; g -= 4) {
      float rb[4], fa[4];
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        const int t = g + j;
        const float4 p = s.p[t][chl];
        float hp[NL];
        if (t > 0) {
          load_states(s.h[t > 0 ? t - 1 : 0][tid], hp);
        } else {
#pragma unroll
          for (int i = 0; i < NL; ++i) hp[i] = h0[i];
        }
        float v[2 * NL];
        float sb = 0.f, sa = 0.f;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const float r = fmaf(s.C[t][q * NL + i], p.z, ar[i]);
          v[i] = r * p.y;
          v[NL + i] = p.z * h[i];
          sb = fmaf(r, s.B[t][q * NL + i], sb);
          ar[i] = dec[t][i] * r;
          const float fl = ar[i] * hp[i];
          dA[i] = fmaf(fl, p.x, dA[i]);
          sa = fmaf(fl, A2[i], sa);
          h[i] = hp[i];
        }
        rb[j] = sb;
        fa[j] = sa;
        using CS = ChanSum<2 * NL>;
        float tot[CS::K3];
        CS::run(v, tot, lane);
        const int first = CS::first(lane);
#pragma unroll
        for (int i = 0; i < CS::K3; ++i) {
          const int w = first + i;   // < NL: dB of state q NL + w, else dC
          s.red[warp][t][w < NL ? q * NL + w : NP + q * NL + w - NL] = tot[i];
        }
      }
      s.o[1][g + q][chl] = quad_sum4(rb[0], rb[1], rb[2], rb[3], lane);
      s.o[2][g + q][chl] = quad_sum4(fa[0], fa[1], fa[2], fa[3], lane);
    }
    __syncthreads();
    // the block's dB and dC of the tile
    for (int i = tid; i < CK * 2 * NP; i += kScanThreads) {
      const int tl = i / (2 * NP), n = i % (2 * NP);
      if (t0 + tl < f.T) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kScanThreads / 32; ++w) sum += s.red[w][tl][n];
        pBC[(((size_t)blockIdx.x * f.B + b) * f.T + t0 + tl) * (2 * NP) + n] = sum;
      }
    }
    // dx, ddt, dz
    if (stages) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const int tl = sr + r * RT, t = t0 + tl;
        float ox[4], ot[4], oz[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 p = s.p[tl][sc + e];
          const float rbv = s.o[1][tl][sc + e];
          ox[e] = fmaf(rbv, p.x, Dv[e] * p.z);
          // the factors A came in as A log2(e)
          ot[e] = fmaf(s.o[2][tl][sc + e], 0.6931471805599453f, rbv * p.w) * ks[r][e];
          oz[e] = kz[r][e] * (z ? fmaf(Dv[e], p.w, s.o[0][tl][sc + e]) : 0.f);
          if (t < f.T) {
            accD[e] = fmaf(p.z, p.w, accD[e]);
            accB[e] += ot[e];
          }
        }
        if (t < f.T) {
          const size_t off = (row0 + t) * f.C + c0 + sc;
          store_ch4(static_cast<T*>(a.dx) + off, sn, vec, ox);
          store_ch4(static_cast<T*>(a.ddt) + off, sn, vec, ot);
          if (z) store_ch4(static_cast<T*>(a.dz) + off, sn, vec, oz);
        }
      }
    }
    __syncthreads();
  }
  if (chan) {
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (q * NL + i < f.N) {
        pA[st + i] = dA[i];
        if (a.dh0) a.dh0[st + i] = ar[i];
      }
  }
  // dD and ddt_bias: the staging rows' sums
  float* red = &s.h[0][0][0];
  static_assert(sizeof(s.h) >= kScanThreads * 8 * sizeof(float), "room for the rows' sums");
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    red[(sr * 2 + 0) * kScanCh + sc + e] = accD[e];
    red[(sr * 2 + 1) * kScanCh + sc + e] = accB[e];
  }
  __syncthreads();
  if (tid < 2 * kScanCh) {
    const int which = tid / kScanCh, c = tid % kScanCh;
    if (c < nch) {
      float sum = 0.f;
      for (int r = 0; r < kScanThreads / 8; ++r) sum += red[(r * 2 + which) * kScanCh + c];
      pD[((size_t)b * 2 + which) * f.C + c0 + c] = sum;
    }
  }
}

// dB, dC [rows, G, N] from the blocks' partials [tiles][rows][2 NP].
template <typename T>
__global__ void __launch_bounds__(256)
sum_bc_kernel(const float* __restrict__ part, T* __restrict__ dB, T* __restrict__ dC,
              long long rows, int G, int N, int NP, int tiles) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;   // row, group, 2 NP
  const int n = (int)(i % (2 * NP));
  const long long rg = i / (2 * NP);
  if (rg >= rows * G || n % NP >= N) return;
  const int g = (int)(rg % G);
  const long long row = rg / G;
  float s = 0.f;
  for (int t = 0; t < tiles; ++t)
    s += part[(((long long)g * tiles + t) * rows + row) * (2 * NP) + n];
  T* out = n < NP ? dB : dC;
  out[rg * N + n % NP] = from_f32<T>(s);
}

template <typename T, int NL>
cudaError_t bwd_form(const ScanBwdArgs& a, int tpg, int vec, float* pBC, float* pA, float* pD,
                     cudaStream_t st) {
  static std::atomic<int> slot[kMaxDevices] = {};
  const int smem = (int)sizeof(BwdSmem<NL>);
  const cudaError_t e = ensure_smem(scan_bwd_kernel<T, NL>, smem, slot);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)(tpg * a.fwd.G), a.fwd.B);
  scan_bwd_kernel<T, NL><<<grid, kScanThreads, smem, st>>>(a, tpg, vec, pBC, pA, pD);
  return cudaGetLastError();
}

template <typename T>
cudaError_t bwd_dispatch(const ScanBwdArgs& a, cudaStream_t st) {
  const ScanArgs& f = a.fwd;
  const int Cg = f.C / f.G, NP = scan_padded_states(f.N);
  const int tpg = (Cg + kScanCh - 1) / kScanCh;
  const int vec = f.C % 4 == 0 && Cg % 4 == 0;
  const long long rows = (long long)f.B * f.T;
  float* pBC = a.part;
  float* pA = pBC + (size_t)tpg * f.G * rows * 2 * NP;
  float* pD = pA + ((size_t)f.B * f.C * f.N + 3) / 4 * 4;
  cudaError_t e;
  if (f.N <= 4) e = bwd_form<T, 1>(a, tpg, vec, pBC, pA, pD, st);
  else if (f.N <= 8) e = bwd_form<T, 2>(a, tpg, vec, pBC, pA, pD, st);
  else if (f.N <= 16) e = bwd_form<T, 4>(a, tpg, vec, pBC, pA, pD, st);
  else if (f.N <= 32) e = bwd_form<T, 8>(a, tpg, vec, pBC, pA, pD, st);
  else e = bwd_form<T, 16>(a, tpg, vec, pBC, pA, pD, st);
  if (e != cudaSuccess) return e;
  const long long n = rows * f.G * 2 * NP;
  if (n > 0) {
    const long long blocks = (n + 255) / 256;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    sum_bc_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(pBC, static_cast<T*>(a.dB),
                                                       static_cast<T*>(a.dC), rows, f.G, f.N, NP,
                                                       tpg);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  e = launch_sum_partials(pA, a.dA, f.B, (long long)f.C * f.N, (long long)f.C * f.N, st);
  if (e == cudaSuccess && a.dD) e = launch_sum_partials(pD, a.dD, f.B, 2LL * f.C, f.C, st);
  if (e == cudaSuccess && a.ddt_bias)
    e = launch_sum_partials(pD + f.C, a.ddt_bias, f.B, 2LL * f.C, f.C, st);
  return e;
}

}  // namespace

size_t selective_scan_bwd_workspace_bytes(int B, int T, int C, int N, int G) {
  if (B <= 0 || C <= 0 || G <= 0 || N <= 0 || T < 0) return 0;
  const size_t tiles = (size_t)((C / G + kScanCh - 1) / kScanCh) * G;
  const size_t pA = ((size_t)B * C * N + 3) / 4 * 4;
  return (tiles * B * T * 2 * scan_padded_states(N) + pA + (size_t)B * 2 * C) * sizeof(float);
}

cudaError_t launch_selective_scan_bwd(const ScanBwdArgs& a, cudaStream_t st) {
  if (a.fwd.B == 0 || a.fwd.C == 0) return cudaSuccess;
  return a.fwd.dtype == kBF16 ? bwd_dispatch<__nv_bfloat16>(a, st) : bwd_dispatch<float>(a, st);
}

}  // namespace gdn
