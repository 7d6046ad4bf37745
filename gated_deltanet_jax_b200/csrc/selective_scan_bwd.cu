// Selective state-space scan, backward (formulas of the forward in
// selective_scan.cu).  With dyp = dy silu(z) and the adjoint state r,
//   r_t[n]   = C_t[n] dyp_t + a_{t+1}[n] r_{t+1}[n]      (a_t = exp(delta_t A)),
//   dB_t[n]  = sum_c r delta x,      dC_t[n] = sum_c dyp h_t[n],
//   dx_t     = delta_t sum_n r B + D dyp,
//   ddelta_t = sum_n r a_t h_{t-1} A + x_t sum_n r B,    ddt = ddelta sigmoid(dt + bias),
//   dA[n]    = sum_t r delta a_t h_{t-1},   dD = sum dyp x,   dz = dy ypre silu'(z).
//
// A block owns 32 channels of one row, four lanes and two channels a lane as in
// the forward, and walks its tiles backwards.  A tile restarts from the state
// that the forward kept at its first token (one fp32 state every 16 tokens at
// N <= 16: four bytes a token and channel, less time than forming it again).  Its
// halves take turns, the later one first: the recurrence runs over the half with
// the states in registers, then the adjoint recurrence backwards.  Rows that
// leave most SMs idle are cut as in the forward, the chunks' adjoint states
// chained from the end.  Sums over channels, rows and tokens leave as one partial
// per block and are added up in a fixed order by further kernels: no atomics, the
// same bits on every run.
//
// Bound by issue slots and latency at eight warps an SM: two to three exponentials
// and about a dozen multiply-adds a state and token.  4 x 2048 x 2048 with 16 states:
// the main pass 394 us (issue 44 %, exponential pipe 42 %, shared memory 59 %), the
// first pass 89 (exponential pipe 79 %).  The sums of dB and dC over the block's
// channels go through shared memory half a tile at a time (shuffles took 31
// instructions a token for them, this takes 15: 425 to 394 us).
#include <type_traits>

#include "selective_scan_common.cuh"

namespace gdn {

namespace {

constexpr int kBwdThreads = 64;   // 16 slots of four lanes, two channels a lane
constexpr int kBwdSlots = kBwdThreads / kScanLanes;

// kLocal: the first pass of a cut row (chunks 1 ..: the adjoint from zero over
// the chunk and the steps' sum out, no gradients).  kTail: the row ends inside a
// tile.  The factors of the tokens past its end are not formed: with A = -inf a step of
// zero would make them NaN.  (A form of its own: 4 x 2048 x 2048 with 16 states 538 us
// with it, 511 without.)
template <typename T, int NL, bool kLocal, bool kTail>
__global__ void __launch_bounds__(kBwdThreads, 4)
scan_bwd_kernel(const ScanBwdArgs a, int tiles_per_group, int vec, int chunk, int nchunk,
                float* __restrict__ pBC, float* __restrict__ pP) {
  constexpr int CK = scan_tile<NL>(), SUB = CK / 2;
  constexpr int NP = NL * kScanLanes;
  constexpr int P = scan_pairs<NL>();
  constexpr int RT = CK < kBwdThreads / 8 ? CK : kBwdThreads / 8;   // rows staged side by side
  constexpr int ROWS = CK / RT;
  constexpr int BV = CK * NL, BPT = (BV + kBwdThreads - 1) / kBwdThreads;
  __shared__ __align__(16) float2 sDU[CK][kScanCh];       // delta, delta x
  __shared__ __align__(16) float sG[CK][kScanCh];         // dyp
  __shared__ __align__(16) float sB[CK][NP], sC[CK][NP];
  __shared__ __align__(16) float sPar[2][kScanCh];        // dt_bias, D
  // x, sigmoid(dt + bias), dy silu'(z); sum C h, sum r B, sum r a h A
  __shared__ __align__(16) float sK[kLocal ? 1 : 3][CK][kScanCh];
  __shared__ __align__(16) float sO[kLocal ? 1 : 3][CK][kScanCh + 8];
  // the lanes' dB and dC of half a tile, in vectors of VW
  constexpr int VW = NL >= 2 ? 4 : 2, PARTS = 2 * NL / VW;
  __shared__ __align__(16) float sV[kLocal ? 1 : SUB][PARTS][kBwdThreads][VW];
  __shared__ __align__(16) float sSum[2][kBwdThreads / 8][kScanCh];

  const ScanArgs& f = a.fwd;
  const int tid = threadIdx.x, lane = tid & 31;
  const int Cg = f.C / f.G;
  const int grp = blockIdx.x / tiles_per_group;
  const int cl0 = (blockIdx.x % tiles_per_group) * kScanCh;
  const int nch = min(kScanCh, Cg - cl0);
  const int c0 = grp * Cg + cl0;
  const int b = blockIdx.y, kc = blockIdx.z + (kLocal ? 1 : 0);
  const int tbeg = kc * chunk, tend = min(f.T, tbeg + chunk);
  const T* x = static_cast<const T*>(f.x);
  const T* dt = static_cast<const T*>(f.dt);
  const T* z = static_cast<const T*>(f.z);
  const T* dy = static_cast<const T*>(a.dy);
  const T* Bp = static_cast<const T*>(f.Bm) + ((size_t)b * f.T * f.G + grp) * f.N;
  const T* Cp = static_cast<const T*>(f.Cm) + ((size_t)b * f.T * f.G + grp) * f.N;
  const bool vecn = f.N % 4 == 0;

  const int chl = tid / kScanLanes * 2, q = tid % kScanLanes;
  const size_t row = (size_t)b * f.C + c0 + chl;
  float* slot = f.chunk_state + (((size_t)kc * f.B + b) * f.C + c0 + chl) * NP + q * NL;
  float2 A2[2][P], ar[2][P], dA[2][P];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int i = 0; i < 2 * P; ++i) {
      const bool ok = chl + c < nch && i < NL && q * NL + i < f.N;
      pair_at(A2[c][i / 2], i & 1) =
          ok ? f.A[(size_t)(c0 + chl + c) * f.N + q * NL + i] * kLog2e : 0.f;
      pair_at(ar[c][i / 2], i & 1) =
          !kLocal && nchunk == 1 && ok && a.dhT ? a.dhT[(row + c) * f.N + q * NL + i] : 0.f;
      pair_at(dA[c][i / 2], i & 1) = 0.f;
    }
    if (!kLocal && nchunk > 1 && chl + c < nch) load_pairs<NL>(slot + c * NP, ar[c]);
  }
  const int sc = tid % 8 * 4, sr = tid / 8;
  const bool stages = sr < RT;
  const int sn = stages ? nch - sc : 0;
  if (tid < kScanCh) {
    sPar[0][tid] = f.dt_bias && tid < nch ? f.dt_bias[c0 + tid] : 0.f;
    sPar[1][tid] = f.D && tid < nch ? f.D[c0 + tid] : 0.f;
  }
  __syncthreads();
  float accD[4] = {0.f, 0.f, 0.f, 0.f}, accB[4] = {0.f, 0.f, 0.f, 0.f};
  const size_t row0 = (size_t)b * f.T;
  Raw4<T> xr[ROWS], dr[ROWS], zr[ROWS], gr[ROWS], bv[BPT], cv[BPT];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int t = t0 + sr + r * RT;
      const int n = t < tend ? sn : 0;
      const size_t off = (row0 + t) * f.C + c0 + sc;
      if (!kLocal) xr[r].load(x + off, n, vec);
      dr[r].load(dt + off, n, vec);
      gr[r].load(dy + off, n, vec);
      if (z) zr[r].load(z + off, n, vec);
    }
#pragma unroll
    for (int r = 0; r < BPT; ++r) {
      const int i = tid + r * kBwdThreads, t = t0 + i / NL, n0 = i % NL * 4;
      const int n = i < BV && t < tend ? f.N - n0 : 0;
      const size_t off = (size_t)t * f.G * f.N + n0;
      if (!kLocal) bv[r].load(Bp + off, n, vecn);
      cv[r].load(Cp + off, n, vecn);
    }
  };
  const int ntiles = (tend - tbeg + CK - 1) / CK;
  if (ntiles > 0) fetch(tbeg + (ntiles - 1) * CK);
  for (int k = ntiles - 1; k >= 0; --k) {
    const int t0 = tbeg + k * CK;
    if (stages) {
      const float4 b4 = load4(&sPar[0][sc]);
      const float bias[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const int tl = sr + r * RT;
        float xv[4] = {0.f, 0.f, 0.f, 0.f}, d[4], g[4], sg[4], kz[4] = {0.f, 0.f, 0.f, 0.f};
        if (!kLocal) xr[r].get(xv);
        dr[r].get(d);
        gr[r].get(g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          d[e] += bias[e];
          sg[e] = 1.f;
          if (f.softplus) d[e] = softplus_sig(d[e], sg[e]);
          if (t0 + tl >= tend) d[e] = 0.f;
          if (kLocal) accD[e] += d[e];
        }
        if (z) {
          float zz[4];
          zr[r].get(zz);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float sz = fast_sigmoid(zz[e]);
            kz[e] = g[e] * (sz * fmaf(zz[e], 1.f - sz, 1.f));
            g[e] *= zz[e] * sz;
          }
        }
        float* du = reinterpret_cast<float*>(&sDU[tl][sc]);
        store4(du, make_float4(d[0], d[0] * xv[0], d[1], d[1] * xv[1]));
        store4(du + 4, make_float4(d[2], d[2] * xv[2], d[3], d[3] * xv[3]));
        store4(&sG[tl][sc], make_float4(g[0], g[1], g[2], g[3]));
        if (!kLocal) {
          store4(&sK[0][tl][sc], make_float4(xv[0], xv[1], xv[2], xv[3]));
          store4(&sK[1][tl][sc], make_float4(sg[0], sg[1], sg[2], sg[3]));
          if (z) store4(&sK[2][tl][sc], make_float4(kz[0], kz[1], kz[2], kz[3]));
        }
      }
    }
#pragma unroll
    for (int r = 0; r < BPT; ++r) {
      const int i = tid + r * kBwdThreads;
      if (i < BV) {
        float v[4];
        cv[r].get(v);
        store4(&sC[i / NL][i % NL * 4], make_float4(v[0], v[1], v[2], v[3]));
        if (!kLocal) {
          bv[r].get(v);
          store4(&sB[i / NL][i % NL * 4], make_float4(v[0], v[1], v[2], v[3]));
        }
      }
    }
    __syncthreads();
    if (k > 0) fetch(t0 - CK);
    if (kLocal) {
#pragma unroll 4
      for (int t = (kTail ? min(CK, tend - t0) : CK) - 1; t >= 0; --t) {
        const float4 du = load4(reinterpret_cast<const float*>(&sDU[t][chl]));
        const float2 g = *reinterpret_cast<const float2*>(&sG[t][chl]);
        float2 C2[P];
        load_pairs<NL>(&sC[t][q * NL], C2);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float dd = c ? du.z : du.x, gg = c ? g.y : g.x;
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 e = decay_arg(make_float2(dd, dd), A2[c][i]);
            ar[c][i] = mul2(make_float2(ex2(e.x), ex2(e.y)),
                            fma2(C2[i], make_float2(gg, gg), ar[c][i]));
          }
        }
      }
      __syncthreads();
      continue;
    }
    // Halves of the tile, the later one first, each with its states in registers.
    // kRagged: the row ends in this one.
    const float* ck = f.ckpt + (((size_t)b * f.nck + t0 / CK) * f.C + c0 + chl) * NP + q * NL;
    const int left = kTail ? tend - t0 : CK;
    auto half = [&](int hf, auto ragged) {
      constexpr bool kRagged = decltype(ragged)::value;
      float2 hs[2][P], h[SUB][2][P];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int i = 0; i < P; ++i) hs[c][i] = make_float2(0.f, 0.f);
        if (chl + c < nch) load_pairs<NL>(ck + c * NP, hs[c]);
      }
      auto advance = [&](int t, float2 (&s)[2][P]) {
        const float4 du = load4(reinterpret_cast<const float*>(&sDU[t][chl]));
        float2 B2[P];
        load_pairs<NL>(&sB[t][q * NL], B2);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float2 d2 = c ? make_float2(du.z, du.z) : make_float2(du.x, du.x);
          const float2 u2 = c ? make_float2(du.w, du.w) : make_float2(du.y, du.y);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 e = decay_arg(d2, A2[c][i]);
            s[c][i] = fma2(make_float2(ex2(e.x), ex2(e.y)), s[c][i], mul2(u2, B2[i]));
          }
        }
      };
      if (hf) {
#pragma unroll
        for (int t = 0; t < SUB; ++t) {
          advance(t, hs);
        }
      }
      const int base = hf * SUB;
      {
        float2 s[2][P];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < P; ++i) s[c][i] = hs[c][i];
#pragma unroll
        for (int t = 0; t < SUB; ++t) {
          if (!kRagged || base + t < left) advance(base + t, s);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < P; ++i) h[t][c][i] = s[c][i];
        }
      }
      // the adjoint recurrence, backwards
      constexpr int QT = SUB < 4 ? SUB : 4;   // tokens whose lane sums are taken together
#pragma unroll
      for (int g0 = SUB - QT; g0 >= 0; g0 -= QT) {
        float yc[2][4] = {}, rb[2][4] = {}, fa[2][4] = {};
#pragma unroll
        for (int j = QT - 1; j >= 0; --j) {
          const int tl = g0 + j, t = base + tl;
          if (kRagged && t >= left) continue;
          const float4 du = load4(reinterpret_cast<const float*>(&sDU[t][chl]));
          const float2 gg = *reinterpret_cast<const float2*>(&sG[t][chl]);
          float2 B2[P], C2[P], dBv[P], dCv[P];
          load_pairs<NL>(&sB[t][q * NL], B2);
          load_pairs<NL>(&sC[t][q * NL], C2);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float2 d2 = c ? make_float2(du.z, du.z) : make_float2(du.x, du.x);
            const float2 u2 = c ? make_float2(du.w, du.w) : make_float2(du.y, du.y);
            const float2 g2 = c ? make_float2(gg.y, gg.y) : make_float2(gg.x, gg.x);
            float2 sy = make_float2(0.f, 0.f), sb = sy, sa = sy;
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const float2 r = fma2(C2[i], g2, ar[c][i]);
              const float2 hn = h[tl][c][i], hp = tl > 0 ? h[tl > 0 ? tl - 1 : 0][c][i] : hs[c][i];
              dBv[i] = c ? fma2(r, u2, dBv[i]) : mul2(r, u2);
              dCv[i] = c ? fma2(hn, g2, dCv[i]) : mul2(hn, g2);
              sy = i ? fma2(C2[i], hn, sy) : mul2(C2[i], hn);
              sb = i ? fma2(r, B2[i], sb) : mul2(r, B2[i]);
              // (kept from the walk above, the factors spilled: 1.24 against 0.83 ms
              // for the training pass of 4 x 2048 x 2048)
              const float2 e = decay_arg(d2, A2[c][i]);
              const float2 dk = make_float2(ex2_again(e.x), ex2_again(e.y));
              ar[c][i] = mul2(dk, r);
              const float2 fl = mul2(ar[c][i], hp);
              dA[c][i] = fma2(fl, d2, dA[c][i]);
              sa = i ? fma2(fl, A2[c][i], sa) : mul2(fl, A2[c][i]);
            }
            yc[c][j] = sy.x + sy.y;
            rb[c][j] = sb.x + sb.y;
            fa[c][j] = sa.x + sa.y;
          }
          if constexpr (NL == 1) {
            *reinterpret_cast<float2*>(sV[tl][0][tid]) = make_float2(dBv[0].x, dCv[0].x);
          } else if constexpr (NL == 2) {
            store4(sV[tl][0][tid], make_float4(dBv[0].x, dBv[0].y, dCv[0].x, dCv[0].y));
          } else {
#pragma unroll
            for (int i = 0; i < NL / 4; ++i) {
              store4(sV[tl][i][tid], make_float4(dBv[2 * i].x, dBv[2 * i].y, dBv[2 * i + 1].x,
                                                 dBv[2 * i + 1].y));
              store4(sV[tl][NL / 4 + i][tid], make_float4(dCv[2 * i].x, dCv[2 * i].y,
                                                          dCv[2 * i + 1].x, dCv[2 * i + 1].y));
            }
          }
        }
        const int t = base + g0 + q;
        float s0, s1;
        if (z) {
          s0 = quad_sum4(yc[0][0], yc[0][1], yc[0][2], yc[0][3], lane);
          s1 = quad_sum4(yc[1][0], yc[1][1], yc[1][2], yc[1][3], lane);
          if (q < QT) *reinterpret_cast<float2*>(&sO[0][t][chl]) = make_float2(s0, s1);
        }
        s0 = quad_sum4(rb[0][0], rb[0][1], rb[0][2], rb[0][3], lane);
        s1 = quad_sum4(rb[1][0], rb[1][1], rb[1][2], rb[1][3], lane);
        if (q < QT) *reinterpret_cast<float2*>(&sO[1][t][chl]) = make_float2(s0, s1);
        s0 = quad_sum4(fa[0][0], fa[0][1], fa[0][2], fa[0][3], lane);
        s1 = quad_sum4(fa[1][0], fa[1][1], fa[1][2], fa[1][3], lane);
        if (q < QT) *reinterpret_cast<float2*>(&sO[2][t][chl]) = make_float2(s0, s1);
      }
      __syncthreads();
      // The half's dB and dC: a thread sums one vector of one token over the 16 slots,
      // from a slot of its own on, so that the threads' reads fall on other banks.
      if (tid < SUB * PARTS * kScanLanes) {
        const int qu = tid % kScanLanes, part = tid / kScanLanes % PARTS;
        const int tl = tid / (kScanLanes * PARTS), t = t0 + base + tl;
        float sum[VW] = {};
#pragma unroll
        for (int i = 0; i < kBwdSlots; ++i) {
          const int sl = (i + tid / kScanLanes) % kBwdSlots;
          const float* v = sV[tl][part][sl * kScanLanes + qu];
          if constexpr (VW == 4) {
            const float4 w = load4(v);
            sum[0] += w.x; sum[1] += w.y; sum[2] += w.z; sum[3] += w.w;
          } else {
            const float2 w = *reinterpret_cast<const float2*>(v);
            sum[0] += w.x; sum[1] += w.y;
          }
        }
        if (t < tend) {
          float* o = pBC + (((size_t)blockIdx.x * f.B + b) * f.T + t) * (2 * NP) + qu * NL;
          if constexpr (NL >= 4) {
            constexpr int H = PARTS / 2;
            store4(o + (part < H ? part * 4 : NP + (part - H) * 4),
                   make_float4(sum[0], sum[1], sum[2], sum[3]));
          } else {
#pragma unroll
            for (int e = 0; e < VW; ++e) o[e < NL ? e : NP + e - NL] = sum[e];
          }
        }
      }
      __syncthreads();
    };
#pragma unroll 1
    for (int hf = 1; hf >= 0; --hf) {
      if (hf * SUB + SUB <= left) half(hf, std::false_type{});
      else if (kTail && hf * SUB < left) half(hf, std::true_type{});
    }
    // dx, ddt, dz
    if (stages) {
      const float4 D4 = load4(&sPar[1][sc]);
      const float Dv[4] = {D4.x, D4.y, D4.z, D4.w};
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const int tl = sr + r * RT, t = t0 + tl;
        if (t >= tend) continue;
        float ox[4], ot[4], oz[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float d = sDU[tl][sc + e].x, g = sG[tl][sc + e];
          const float xv = sK[0][tl][sc + e], rbv = sO[1][tl][sc + e];
          ox[e] = fmaf(rbv, d, Dv[e] * g);
          // the factors A came in as A log2(e)
          ot[e] = fmaf(sO[2][tl][sc + e], 0.6931471805599453f, rbv * xv) * sK[1][tl][sc + e];
          if (z) oz[e] = sK[2][tl][sc + e] * fmaf(Dv[e], xv, sO[0][tl][sc + e]);
          accD[e] = fmaf(g, xv, accD[e]);
          accB[e] += ot[e];
        }
        const size_t off = (row0 + t) * f.C + c0 + sc;
        store_ch4(static_cast<T*>(a.dx) + off, sn, vec, ox);
        store_ch4(static_cast<T*>(a.ddt) + off, sn, vec, ot);
        if (z) store_ch4(static_cast<T*>(a.dz) + off, sn, vec, oz);
      }
    }
    __syncthreads();
  }
  // this chunk's and row's sums for the parameters: dA [C][N], dD [C], ddt_bias [C]
  const size_t prow = ((size_t)kc * f.B + b) * f.C * (f.N + 2);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (chl + c >= nch) continue;
    if (kLocal) {
      store_pairs<NL>(slot + c * NP, ar[c]);
      continue;
    }
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (q * NL + i < f.N) {
        pP[prow + (size_t)(c0 + chl + c) * f.N + q * NL + i] = pair_at(dA[c][i / 2], i & 1);
        if (a.dh0 && kc == 0)
          a.dh0[(row + c) * f.N + q * NL + i] = pair_at(ar[c][i / 2], i & 1);
      }
  }
  // the staging rows' sums: dD and ddt_bias, or the local pass's steps
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    sSum[0][sr][sc + e] = accD[e];
    sSum[1][sr][sc + e] = accB[e];
  }
  __syncthreads();
  const int which = tid / kScanCh, c = tid % kScanCh;
  if (c < nch) {
    float sum = 0.f;
    for (int r = 0; r < kBwdThreads / 8; ++r) sum += sSum[which][r][c];
    if (!kLocal)
      pP[prow + (size_t)f.C * (f.N + which) + c0 + c] = sum;
    else if (which == 0)
      f.chunk_sum[((size_t)kc * f.B + b) * f.C + c0 + c] = sum;
  }
}

// dB, dC [rows, G, N] from the blocks' partials [tiles][rows][2 NP]: four states a
// thread, 16-byte reads with eight in flight.
template <typename T>
__global__ void __launch_bounds__(256)
sum_bc_kernel(const float* __restrict__ part, T* __restrict__ dB, T* __restrict__ dC,
              long long rows, int G, int N, int NP, int tiles) {
  const int per = NP / 2;                                          // vectors of a row and group
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;   // row, group, vector
  const int n = (int)(i % per) * 4;
  const long long rg = i / per;
  if (rg >= rows * G) return;
  const int g = (int)(rg % G);
  const long long row = rg / G, step = rows * 2 * NP;
  const float* p = part + ((long long)g * tiles * rows + row) * (2 * NP) + n;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int t = 0; t < tiles; ++t) {
    const float4 v = load4(p + t * step);
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  T* out = (n < NP ? dB : dC) + rg * N;
  const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n % NP + e < N) out[n % NP + e] = from_f32<T>(v[e]);
}

template <typename T, int NL, bool kTail>
cudaError_t bwd_form(const ScanBwdArgs& a, int tpg, int vec, const ScanSplit& sp, float* pBC,
                     float* pP, cudaStream_t st) {
  const dim3 grid((unsigned)(tpg * a.fwd.G), a.fwd.B, sp.chunks);
  if (sp.chunks > 1) {
    scan_bwd_kernel<T, NL, true, kTail>
        <<<dim3(grid.x, grid.y, sp.chunks - 1), kBwdThreads, 0, st>>>(
            a, tpg, vec, sp.tokens, sp.chunks, nullptr, nullptr);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = launch_scan_chain(a.fwd, a.dhT, sp.chunks, true, st);
    if (e != cudaSuccess) return e;
  }
  scan_bwd_kernel<T, NL, false, kTail><<<grid, kBwdThreads, 0, st>>>(a, tpg, vec, sp.tokens,
                                                                     sp.chunks, pBC, pP);
  return cudaGetLastError();
}

template <typename T, int NL>
cudaError_t bwd_form(const ScanBwdArgs& a, int tpg, int vec, const ScanSplit& sp, float* pBC,
                     float* pP, cudaStream_t st) {
  return a.fwd.T % scan_tile<NL>() ? bwd_form<T, NL, true>(a, tpg, vec, sp, pBC, pP, st)
                                   : bwd_form<T, NL, false>(a, tpg, vec, sp, pBC, pP, st);
}

// The workspace's parts, in floats from its start.
struct BwdLayout {
  ScanSplit sp;
  size_t bc, params, split, total;
  BwdLayout(int B, int T, int C, int N, int G) {
    sp = scan_split(B, T, C, G, true);
    const size_t tiles = (size_t)((C / G + kScanCh - 1) / kScanCh) * G;
    bc = 0;
    params = tiles * B * T * 2 * scan_padded_states(N);
    split = params + ((size_t)sp.chunks * B * C * (N + 2) + 3) / 4 * 4;
    total = split + scan_split_bytes(B, C, N, sp) / sizeof(float);
  }
};

template <typename T>
cudaError_t bwd_dispatch(const ScanBwdArgs& args, cudaStream_t st) {
  ScanBwdArgs a = args;
  const ScanArgs& f = a.fwd;
  const int Cg = f.C / f.G, NP = scan_padded_states(f.N);
  const int tpg = (Cg + kScanCh - 1) / kScanCh;
  const int vec = f.C % 4 == 0 && Cg % 4 == 0;
  const long long rows = (long long)f.B * f.T;
  const BwdLayout lay(f.B, f.T, f.C, f.N, f.G);
  float *pBC = a.part + lay.bc, *pP = a.part + lay.params;
  scan_split_workspace(a.fwd, a.part + lay.split, lay.sp);
  cudaError_t e;
  if (f.N <= 4) e = bwd_form<T, 1>(a, tpg, vec, lay.sp, pBC, pP, st);
  else if (f.N <= 8) e = bwd_form<T, 2>(a, tpg, vec, lay.sp, pBC, pP, st);
  else if (f.N <= 16) e = bwd_form<T, 4>(a, tpg, vec, lay.sp, pBC, pP, st);
  else if (f.N <= 32) e = bwd_form<T, 8>(a, tpg, vec, lay.sp, pBC, pP, st);
  else e = bwd_form<T, 16>(a, tpg, vec, lay.sp, pBC, pP, st);
  if (e != cudaSuccess) return e;
  const long long n = rows * f.G * (NP / 2);
  if (n > 0) {
    const long long blocks = (n + 255) / 256;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    sum_bc_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(pBC, static_cast<T*>(a.dB),
                                                       static_cast<T*>(a.dC), rows, f.G, f.N, NP,
                                                       tpg);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  const SumSegments out{{a.dA, a.dD, a.ddt_bias}, {(long long)f.C * f.N, f.C, f.C}};
  return launch_sum_partials(pP, (long long)lay.sp.chunks * f.B, (long long)f.C * (f.N + 2), out,
                             st);
}

}  // namespace

size_t selective_scan_bwd_workspace_bytes(int B, int T, int C, int N, int G) {
  if (B <= 0 || C <= 0 || G <= 0 || N <= 0 || T < 0) return 0;
  return BwdLayout(B, T, C, N, G).total * sizeof(float);
}

cudaError_t launch_selective_scan_bwd(const ScanBwdArgs& a, cudaStream_t st) {
  if (a.fwd.B == 0 || a.fwd.C == 0) return cudaSuccess;
  return a.fwd.dtype == kBF16 ? bwd_dispatch<__nv_bfloat16>(a, st) : bwd_dispatch<float>(a, st);
}

}  // namespace gdn
