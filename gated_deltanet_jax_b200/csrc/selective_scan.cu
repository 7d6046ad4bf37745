// Selective state-space scan, forward (no counterpart in the reference, whose
// only recurrence is the gated delta rule).  Per channel c with N states,
//   delta_t = softplus(dt_t + dt_bias)          (or dt_t + dt_bias)
//   h_t[n]  = exp(delta_t A[n]) h_{t-1}[n] + delta_t x_t B_t[n]
//   y_t     = (sum_n C_t[n] h_t[n] + D x_t) silu(z_t)
// with an fp32 state.  B and C are shared by the channels of a group.
//
// What it has to move is x, dt, z and y once (8 bytes a token and channel in
// bf16); what it has to compute is one exponential and four multiply-adds per
// state, which at N = 16 takes longer than the bytes (16 exponentials a clock
// and SM: 0.30 ms with the gates' for 8 x 2048 x 4096 against 0.08 ms for its
// bytes).  Four lanes share a channel, each with a quarter of its states in
// registers as pairs (two multiply-adds an instruction), and a lane serves two
// channels with each row of B and C that it reads: a 16-byte read takes four
// shared-memory cycles of a warp whatever its lanes share, and with one channel a
// lane those cycles (87 % busy) set the time.  A block owns 32 channels of one row
// and walks tiles of 32 tokens: every thread forms delta and delta x of its share
// into shared memory with the next tile's loads in flight, all lanes then run the
// recurrence over the tile, and four tokens' read-outs at a time are summed over
// the four lanes in three shuffles.  0.50 ms at that size: the exponential pipe 60 %
// busy, issue slots 58 %, shared memory 54 %, 7 blocks (14 warps) an SM.  Part of
// the exponentials on the multiply-add pipes, more warps of fewer registers, and
// the read-out or the reads moved ahead by hand each measured slower.
//
// Few rows and a long axis: the recurrence is linear, so a row is cut into
// chunks.  A first pass runs each from a zero state (no read-out) and keeps its
// end and the sum of its steps; since the decay over a chunk is exp(A sum delta),
// a second kernel chains the chunks' entering states, and the main pass starts
// every chunk from its own.  The exponentials are computed twice, so only rows
// that leave most SMs idle are cut.
#include <type_traits>

#include "selective_scan_common.cuh"

namespace gdn {

namespace {

constexpr int kFwdThreads = 64;       // 16 slots of four lanes, two channels a lane
constexpr int kTT = 32;               // tokens of a tile
constexpr int kSRows = kFwdThreads / 8;                     // rows staged side by side
constexpr int kRows = kTT / kSRows;                         // staging rows per thread

// kLocal: the first pass of a cut row (from zero; the end state and the steps'
// sum out, no y).  chunk / nchunk: tokens of a chunk and their number (grid z).
// kTail: the row ends inside a tile.  The factors of the tokens past its end are not
// formed: with A = -inf a step of zero would make them NaN.  (A form of its own, so that
// whole tiles do not carry it: 8 x 2048 x 4096 in bf16 514 us with it, 500 without.)
template <typename T, int NL, bool kLocal, bool kTail>
__global__ void __launch_bounds__(kFwdThreads, NL > 8 ? 4 : 7)
scan_fwd_kernel(const ScanArgs a, int tiles_per_group, int vec, int chunk, int nchunk) {
  constexpr int NP = NL * kScanLanes;
  constexpr int P = scan_pairs<NL>();
  constexpr int CK = scan_tile<NL>();
  constexpr int BV = kTT * NL;                                    // vectors of B in a tile
  constexpr int BPT = (BV + kFwdThreads - 1) / kFwdThreads;       // per thread
  __shared__ __align__(16) float2 sDU[kTT][kScanCh];              // delta, delta x
  __shared__ __align__(16) float sY[kLocal ? 1 : kTT][kScanCh + 8];
  __shared__ __align__(16) float sB[kTT][NP], sC[kLocal ? 1 : kTT][NP];
  __shared__ __align__(16) float sPar[2][kScanCh];                // dt_bias, D

  const int tid = threadIdx.x, lane = tid & 31;
  const int Cg = a.C / a.G;
  const int grp = blockIdx.x / tiles_per_group;
  const int cl0 = (blockIdx.x % tiles_per_group) * kScanCh;   // first channel in the group
  const int nch = min(kScanCh, Cg - cl0);
  const int c0 = grp * Cg + cl0;
  const int b = blockIdx.y, kc = blockIdx.z;
  const int tbeg = kc * chunk, tend = min(a.T, tbeg + chunk);
  const T* x = static_cast<const T*>(a.x);
  const T* dt = static_cast<const T*>(a.dt);
  const T* z = kLocal ? nullptr : static_cast<const T*>(a.z);
  const T* Bp = static_cast<const T*>(a.Bm) + ((size_t)b * a.T * a.G + grp) * a.N;
  const T* Cp = static_cast<const T*>(a.Cm) + ((size_t)b * a.T * a.G + grp) * a.N;
  const bool vecn = a.N % 4 == 0;

  // the lane's channels chl, chl + 1 and its quarter of their states
  const int chl = tid / kScanLanes * 2, q = tid % kScanLanes;
  const size_t row = (size_t)b * a.C + c0 + chl;
  float* slot = a.chunk_state + (((size_t)kc * a.B + b) * a.C + c0 + chl) * NP + q * NL;
  float2 A2[2][P], h[2][P];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int i = 0; i < 2 * P; ++i) {
      const bool ok = chl + c < nch && i < NL && q * NL + i < a.N;
      pair_at(A2[c][i / 2], i & 1) =
          ok ? a.A[(size_t)(c0 + chl + c) * a.N + q * NL + i] * kLog2e : 0.f;
      pair_at(h[c][i / 2], i & 1) =
          !kLocal && nchunk == 1 && ok && a.h0 ? a.h0[(row + c) * a.N + q * NL + i] : 0.f;
    }
    if (!kLocal && nchunk > 1 && chl + c < nch) load_pairs<NL>(slot + c * NP, h[c]);
  }
  // the staging role: channels sc .. sc + 3 of rows sr, sr + kSRows, ...
  const int sc = tid % 8 * 4, sr = tid / 8;
  const int sn = nch - sc;
  if (tid < kScanCh) {
    sPar[0][tid] = a.dt_bias && tid < nch ? a.dt_bias[c0 + tid] : 0.f;
    sPar[1][tid] = !kLocal && a.D && tid < nch ? a.D[c0 + tid] : 0.f;
  }
  __syncthreads();
  float dsum[4] = {0.f, 0.f, 0.f, 0.f};
  const size_t row0 = (size_t)b * a.T;
  Raw4<T> xv[kRows], dv[kRows], zv[kRows], bv[BPT], cv[BPT];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int t = t0 + sr + r * kSRows;
      const int n = t < tend ? sn : 0;
      const size_t off = (row0 + t) * a.C + c0 + sc;
      xv[r].load(x + off, n, vec);
      dv[r].load(dt + off, n, vec);
    }
#pragma unroll
    for (int r = 0; r < BPT; ++r) {
      const int i = tid + r * kFwdThreads, t = t0 + i / NL, n0 = i % NL * 4;
      const int n = i < BV && t < tend ? a.N - n0 : 0;
      const size_t off = (size_t)t * a.G * a.N + n0;
      bv[r].load(Bp + off, n, vecn);
      if (!kLocal) cv[r].load(Cp + off, n, vecn);
    }
  };
  fetch(tbeg);
  for (int t0 = tbeg; t0 < tend; t0 += kTT) {
    const float4 bias4 = load4(&sPar[0][sc]), D4 = load4(&sPar[1][sc]);
    const float bias[4] = {bias4.x, bias4.y, bias4.z, bias4.w};
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int tl = sr + r * kSRows;
      float xf[4], d[4];
      xv[r].get(xf);
      dv[r].get(d);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        d[e] += bias[e];
        if (a.softplus) d[e] = softplus_fast(d[e]);
        if (kLocal) dsum[e] += d[e];   // (its chunks are whole tiles)
      }
      float* du = reinterpret_cast<float*>(&sDU[tl][sc]);
      store4(du, make_float4(d[0], d[0] * xf[0], d[1], d[1] * xf[1]));
      store4(du + 4, make_float4(d[2], d[2] * xf[2], d[3], d[3] * xf[3]));
      if (!kLocal)
        store4(&sY[tl][sc], make_float4(D4.x * xf[0], D4.y * xf[1], D4.z * xf[2], D4.w * xf[3]));
    }
#pragma unroll
    for (int r = 0; r < BPT; ++r) {
      const int i = tid + r * kFwdThreads;
      if (i < BV) {
        float v[4];
        bv[r].get(v);
        store4(&sB[i / NL][i % NL * 4], make_float4(v[0], v[1], v[2], v[3]));
        if (!kLocal) {
          cv[r].get(v);
          store4(&sC[i / NL][i % NL * 4], make_float4(v[0], v[1], v[2], v[3]));
        }
      }
    }
    __syncthreads();
    if (z) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int t = t0 + sr + r * kSRows;
        zv[r].load(z + (row0 + t) * a.C + c0 + sc, t < tend ? sn : 0, vec);
      }
    }
    if (t0 + kTT < tend) fetch(t0 + kTT);
    // Four tokens from g on; kRagged: the row ends among them.
    const int left = kTail ? min(kTT, tend - t0) : kTT;
    auto group = [&](int g, auto ragged) {
      constexpr bool kRagged = decltype(ragged)::value;
      if (!kLocal && a.ckpt && g % CK == 0 && t0 + g < a.T) {
        float* ck = a.ckpt + (((size_t)b * a.nck + (t0 + g) / CK) * a.C + c0 + chl) * NP + q * NL;
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (chl + c < nch) store_pairs<NL>(ck + c * NP, h[c]);
      }
      float ys[2][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (kRagged && g + j >= left) {
          ys[0][j] = ys[1][j] = 0.f;
          continue;
        }
        const float4 du = load4(reinterpret_cast<const float*>(&sDU[g + j][chl]));
        float2 B2[P], C2[P];
        load_pairs<NL>(&sB[g + j][q * NL], B2);
        if (!kLocal) load_pairs<NL>(&sC[g + j][q * NL], C2);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float2 d2 = c ? make_float2(du.z, du.z) : make_float2(du.x, du.x);
          const float2 u2 = c ? make_float2(du.w, du.w) : make_float2(du.y, du.y);
          float2 acc = make_float2(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 e = decay_arg(d2, A2[c][i]);
            h[c][i] = fma2(make_float2(ex2(e.x), ex2(e.y)), h[c][i], mul2(u2, B2[i]));
            if (!kLocal) acc = i ? fma2(C2[i], h[c][i], acc) : mul2(C2[i], h[c][i]);
          }
          ys[c][j] = acc.x + acc.y;
        }
      }
      if (!kLocal) {
        float2* yp = reinterpret_cast<float2*>(&sY[g + q][chl]);
        float2 v = *yp;
        v.x += quad_sum4(ys[0][0], ys[0][1], ys[0][2], ys[0][3], lane);
        v.y += quad_sum4(ys[1][0], ys[1][1], ys[1][2], ys[1][3], lane);
        *yp = v;
      }
    };
    const int whole = left / 4 * 4;
#pragma unroll 1
    for (int g = 0; g < whole; g += 4) group(g, std::false_type{});
    if (kTail && whole < left) group(whole, std::true_type{});
    __syncthreads();
    if (!kLocal) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int tl = sr + r * kSRows, t = t0 + tl;
        const float4 yv = load4(&sY[tl][sc]);
        float o[4] = {yv.x, yv.y, yv.z, yv.w};
        if (z) {
          float zf[4];
          zv[r].get(zf);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] *= zf[e] * fast_sigmoid(zf[e]);
        }
        if (t < tend) store_ch4(static_cast<T*>(a.y) + (row0 + t) * a.C + c0 + sc, sn, vec, o);
      }
    }
  }
  if (kLocal) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (chl + c < nch) store_pairs<NL>(slot + c * NP, h[c]);
    // the staging rows' sums of delta, added up in a fixed order
    float* red = reinterpret_cast<float*>(sDU);
#pragma unroll
    for (int e = 0; e < 4; ++e) red[sr * kScanCh + sc + e] = dsum[e];
    __syncthreads();
    if (tid < nch) {
      float s = 0.f;
      for (int r = 0; r < kSRows; ++r) s += red[r * kScanCh + tid];
      a.chunk_sum[((size_t)kc * a.B + b) * a.C + c0 + tid] = s;
    }
  } else if (a.hT && kc == nchunk - 1) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < NL; ++i)
        if (chl + c < nch && q * NL + i < a.N)
          a.hT[(row + c) * a.N + q * NL + i] = pair_at(h[c][i / 2], i & 1);
  }
}

// Chains a cut row's chunks: state [chunk][rows = B C][NP] holds each chunk's end
// from zero (the last chunk's is not read) and takes the state entering it.
// kReverse: from the last chunk to the first (the backward's adjoint states),
// the sum of steps being that of the chunk the state leaves through.  A chunk's decay may
// leave fp32's range where the state does not (A > 0 and a state of zero or near it, or a
// large one that shrinks): it enters as its square root, twice, and not at all at zero.
template <bool kReverse>
__global__ void __launch_bounds__(256)
scan_chain_kernel(float* __restrict__ state, const float* __restrict__ sum,
                  const float* __restrict__ A, const float* __restrict__ first, long long rows,
                  int C, int N, int NP, int nchunk) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = i / NP;
  const int n = (int)(i % NP);
  if (row >= rows) return;
  const float a2 = n < N ? A[(row % C) * N + n] * (0.5f * kLog2e) : 0.f;
  float h = n < N && first ? first[row * N + n] : 0.f;
  constexpr int kAt = 8;   // chunks whose loads are in flight under eight others' steps
  float loc[kAt], dec[kAt];
  auto fetch = [&](int s0) {
#pragma unroll
    for (int j = 0; j < kAt; ++j) {
      const int s = s0 + j;
      const long long k = kReverse ? nchunk - 1 - s : s;
      const bool on = s + 1 < nchunk;
      loc[j] = on ? state[k * rows * NP + i] : 0.f;
      dec[j] = on ? sum[k * rows + row] : 0.f;
    }
  };
  fetch(0);
  for (int s0 = 0; s0 < nchunk; s0 += kAt) {
    float l[kAt], d[kAt];
#pragma unroll
    for (int j = 0; j < kAt; ++j) {
      l[j] = loc[j];
      d[j] = ex2(fmaf(a2, dec[j], kDecayBias));
    }
    fetch(s0 + kAt);
#pragma unroll
    for (int j = 0; j < kAt; ++j) {
      const int s = s0 + j;
      if (s >= nchunk) break;
      state[(kReverse ? nchunk - 1 - s : s) * rows * NP + i] = h;
      h = h == 0.f ? l[j] : fmaf(d[j], d[j] * h, l[j]);
    }
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
  if (a.softplus) d = softplus_fast(d);
  const float u = d * x, d2 = d * kLog2e;
  h.x = fmaf(ex2(fmaf(d2, A.x, kDecayBias)), h.x, u * B.x);
  h.y = fmaf(ex2(fmaf(d2, A.y, kDecayBias)), h.y, u * B.y);
  h.z = fmaf(ex2(fmaf(d2, A.z, kDecayBias)), h.z, u * B.z);
  h.w = fmaf(ex2(fmaf(d2, A.w, kDecayBias)), h.w, u * B.w);
  if (a.hT && chan) store4_stream(a.hT + st, h);
  float y = fmaf(Cv.x, h.x, fmaf(Cv.y, h.y, fmaf(Cv.z, h.z, Cv.w * h.w)));
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  if (q == 0 && chan) {
    if (a.D) y = fmaf(a.D[c], x, y);
    if (a.z) {
      const float zv = to_f32(static_cast<const T*>(a.z)[row]);
      y *= zv * fast_sigmoid(zv);
    }
    static_cast<T*>(a.y)[row] = from_f32<T>(y);
  }
}

// The same at 16 states where four channels in a row share a group: four lanes
// take four channels together, each forming the step and the gate of one (four
// lanes a channel form them four times over, and issue slots, 71 % of them in use,
// then hold the loads back: 12.2 us for 64 x 4096 channels).
template <typename T>
__global__ void __launch_bounds__(256)
scan_step4_kernel(const ScanArgs a) {
  constexpr int N = 16;
  const int lane = threadIdx.x & 31, q = lane & 3, b = blockIdx.y;
  const long long cl = (long long)blockIdx.x * 256 + threadIdx.x;   // this lane's channel
  const bool chan = cl < a.C;
  const int c = chan ? (int)cl : a.C - 1;
  const int cq = c - q >= 0 ? c - q : 0;     // the four lanes' first channel
  const int grp = cq / (a.C / a.G);
  const bool quad = cl - q < a.C;            // C is a multiple of four: all four or none
  const size_t row = (size_t)b * a.C;
  const size_t st = (row + cq) * N + 4 * q;
  float4 h[4], A[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (quad && a.h0) h[j] = load4_stream(a.h0 + st + j * N);
  }
  const float x = to_f32(static_cast<const T*>(a.x)[row + c]);
  float d = to_f32(static_cast<const T*>(a.dt)[row + c]) + (a.dt_bias ? a.dt_bias[c] : 0.f);
  const float zv = a.z ? to_f32(static_cast<const T*>(a.z)[row + c]) : 0.f;
  const float Dv = a.D ? a.D[c] : 0.f;
  const size_t bc = ((size_t)b * a.G + grp) * N + 4 * q;
  const float4 B = load4(static_cast<const T*>(a.Bm) + bc);
  const float4 Cv = load4(static_cast<const T*>(a.Cm) + bc);
#pragma unroll
  for (int j = 0; j < 4; ++j) A[j] = load4(a.A + (size_t)(quad ? cq + j : 0) * N + 4 * q);
  if (a.softplus) d = softplus_fast(d);
  const float u = d * x;
  float y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float dj = __shfl_sync(0xffffffffu, d, (lane & ~3) | j) * kLog2e;
    const float uj = __shfl_sync(0xffffffffu, u, (lane & ~3) | j);
    h[j].x = fmaf(ex2(fmaf(dj, A[j].x, kDecayBias)), h[j].x, uj * B.x);
    h[j].y = fmaf(ex2(fmaf(dj, A[j].y, kDecayBias)), h[j].y, uj * B.y);
    h[j].z = fmaf(ex2(fmaf(dj, A[j].z, kDecayBias)), h[j].z, uj * B.z);
    h[j].w = fmaf(ex2(fmaf(dj, A[j].w, kDecayBias)), h[j].w, uj * B.w);
    if (quad && a.hT) store4_stream(a.hT + st + j * N, h[j]);
    y[j] = fmaf(Cv.x, h[j].x, fmaf(Cv.y, h[j].y, fmaf(Cv.z, h[j].z, Cv.w * h[j].w)));
  }
  float o = fmaf(Dv, x, quad_sum4(y[0], y[1], y[2], y[3], lane));
  if (a.z) o *= zv * fast_sigmoid(zv);
  if (chan) static_cast<T*>(a.y)[row + c] = from_f32<T>(o);
}

template <typename T, int L>
cudaError_t launch_step(const ScanArgs& a, cudaStream_t st) {
  if (L == 4 && a.C / a.G % 4 == 0) {
    scan_step4_kernel<T><<<dim3((unsigned)((a.C + 255LL) / 256), a.B), 256, 0, st>>>(a);
    return cudaGetLastError();
  }
  const long long blocks = ((long long)a.C * L + 255) / 256;
  scan_step_kernel<T, L><<<dim3((unsigned)blocks, a.B), 256, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T, int NL>
cudaError_t launch_fwd(const ScanArgs& a, int tpg, int vec, const ScanSplit& sp, cudaStream_t st) {
  const dim3 grid((unsigned)(tpg * a.G), a.B, sp.chunks);
  if (sp.chunks > 1) {
    scan_fwd_kernel<T, NL, true, false>
        <<<dim3(grid.x, grid.y, sp.chunks - 1), kFwdThreads, 0, st>>>(a, tpg, vec, sp.tokens,
                                                                      sp.chunks);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = launch_scan_chain(a, a.h0, sp.chunks, false, st);
    if (e != cudaSuccess) return e;
  }
  if (a.T % kTT)
    scan_fwd_kernel<T, NL, false, true><<<grid, kFwdThreads, 0, st>>>(a, tpg, vec, sp.tokens,
                                                                      sp.chunks);
  else
    scan_fwd_kernel<T, NL, false, false><<<grid, kFwdThreads, 0, st>>>(a, tpg, vec, sp.tokens,
                                                                       sp.chunks);
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
  const ScanSplit sp = scan_split(a.B, a.T, a.C, a.G, false);
  if (a.N <= 4) return launch_fwd<T, 1>(a, tpg, vec, sp, st);
  if (a.N <= 8) return launch_fwd<T, 2>(a, tpg, vec, sp, st);
  if (a.N <= 16) return launch_fwd<T, 4>(a, tpg, vec, sp, st);
  if (a.N <= 32) return launch_fwd<T, 8>(a, tpg, vec, sp, st);
  return launch_fwd<T, 16>(a, tpg, vec, sp, st);
}

}  // namespace

// How a row is cut.  Whole rows are bound by one warp's walk until about three
// blocks share an SM (2048 tokens, 16 states: 0.24 ms forward from 1 to 256 blocks,
// 0.31 at 512), while a cut row costs 1.4 (forward) to 1.2 times the work.  The
// chunks make two waves of the forward's blocks (seven an SM) and four of the
// backward's (four an SM), which measured best: at 256 blocks the forward takes
// 0.21 ms cut, 0.24 whole, the backward 0.54 and 0.98; at 8192 tokens and 512 blocks
// the forward 1.42 cut, 1.22 whole, the backward 3.9 and 4.6.
ScanSplit scan_split(int B, int T, int C, int G, bool backward) {
  const long long blocks = (long long)((C / G + kScanCh - 1) / kScanCh) * G * B;
  ScanSplit s{1, T};
  if (T <= 0 || blocks <= 0 || blocks > (backward ? 512 : 384)) return s;
  const long long want = ((long long)device_sm_count() * (backward ? 16 : 14) + blocks - 1) / blocks;
  long long tokens = (T + want - 1) / want;
  if (tokens < 128) tokens = 128;   // a chunk's launch and chaining against its walk
  tokens = (tokens + 31) / 32 * 32;
  s.tokens = (int)tokens;
  s.chunks = (int)((T + tokens - 1) / tokens);
  return s;
}

size_t scan_split_bytes(int B, int C, int N, const ScanSplit& s) {
  if (s.chunks <= 1) return 0;
  return (size_t)s.chunks * B * C * (scan_padded_states(N) + 1) * sizeof(float);
}

void scan_split_workspace(ScanArgs& a, float* ws, const ScanSplit& s) {
  a.chunk_state = ws;
  a.chunk_sum = ws ? ws + (size_t)s.chunks * a.B * a.C * scan_padded_states(a.N) : nullptr;
}

cudaError_t launch_scan_chain(const ScanArgs& a, const float* first, int chunks, bool reverse,
                              cudaStream_t st) {
  const int NP = scan_padded_states(a.N);
  const long long rows = (long long)a.B * a.C, blocks = (rows * NP + 255) / 256;
  if (reverse)
    scan_chain_kernel<true><<<(unsigned)blocks, 256, 0, st>>>(a.chunk_state, a.chunk_sum, a.A,
                                                              first, rows, a.C, a.N, NP, chunks);
  else
    scan_chain_kernel<false><<<(unsigned)blocks, 256, 0, st>>>(a.chunk_state, a.chunk_sum, a.A,
                                                               first, rows, a.C, a.N, NP, chunks);
  return cudaGetLastError();
}

int scan_padded_states(int N) { return N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }

int scan_checkpoint_tokens(int N) { return N <= 16 ? 16 : N <= 32 ? 8 : 4; }

size_t scan_checkpoint_bytes(int B, int T, int C, int N) {
  const int k = scan_checkpoint_tokens(N);
  return (size_t)B * ((T + k - 1) / k) * C * scan_padded_states(N) * sizeof(float);
}

size_t selective_scan_workspace_bytes(int B, int T, int C, int N, int G) {
  return scan_split_bytes(B, C, N, scan_split(B, T, C, G, false));
}

cudaError_t launch_selective_scan(const ScanArgs& a, cudaStream_t st) {
  if (a.B == 0 || a.C == 0) return cudaSuccess;
  return a.dtype == kBF16 ? fwd_dispatch<__nv_bfloat16>(a, st) : fwd_dispatch<float>(a, st);
}

}  // namespace gdn
