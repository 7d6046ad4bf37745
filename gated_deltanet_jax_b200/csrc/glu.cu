// The gated linear unit of the feed-forward block (model.py:162-180 before its
// down projection): h = silu(x Wg^T) * (x Wu^T), and its gradients
//   dg = dh u s (1 + g (1 - s)),  du = dh g s   (s = sigmoid(g)),
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x.
//
// This file holds the CUDA-core form, for fp32 inputs (the products are fp32
// fused multiply-adds) and for bf16 widths that the tensor-core form does not
// take, and the elementwise step between the two halves of the backward, which
// every form shares.  One tiled kernel computes all products: 256 threads,
// square tiles with the operands transposed into shared memory and prefetched
// a step ahead in registers, fp32 accumulators (53 TFLOP/s forward at 4096 x 1024 x
// 2048 in fp32, 46 with the gradients).  The two projections share one
// tile of x: half of a tile's columns come from Wg and half from Wu, so that a
// thread ends with g and u of the same elements.
#include "gdn_common.cuh"
#include "gdn_internal.h"

namespace gdn {

namespace {

constexpr int kThreads = 256;
constexpr int kBK = 16;

// Four consecutive elements of `p`, the first `n` of them in range.
template <typename T>
__device__ __forceinline__ void load_vec(const T* p, int n, bool vec, float (&v)[4]) {
  if (n >= 4 && vec) {
    const float4 q = load4(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? to_f32(p[e]) : 0.f;
  }
}

enum GluMode : int {
  kFwd = 0,    // [g | u] = x [Wg | Wu]^T, h out (g, u out when asked for)
  kDx = 1,     // dx = dg Wg + du Wu
  kDw = 2,     // dWg = dg^T x (even blockIdx.z), dWu = du^T x (odd), over the K rows of part z / 2
};

// out [M, N] = sum_k A(m, k) B(n, k).  A and B per mode:
//   kFwd  A = x [M, K], B = the rows of Wg and Wu [N, K];
//   kDx   A = dg, du [M, K], B(n, k) = W[k, n]  (two passes over k);
//   kDw   A(m, k) = dg[k, m], B(n, k) = x[k, n].
template <typename T, int MODE, int TM>
__global__ void __launch_bounds__(kThreads, 2)
glu_simt_kernel(const T* __restrict__ A0, const T* __restrict__ A1, const T* __restrict__ B0,
                const T* __restrict__ B1, T* __restrict__ O0, T* __restrict__ O1,
                T* __restrict__ O2, int M, int N, int K, int kpart, bool vec) {
  constexpr int BM = 16 * TM, BN = 16 * TM, H = TM / 2;
  constexpr int BNH = MODE == kFwd ? BN / 2 : BN;   // output columns of a tile
  constexpr int LV = BM * kBK / 4 / kThreads;       // vectors of a tile per thread
  constexpr int LD = BM + 4;
  __shared__ __align__(16) float As[2][kBK][LD], Bs[2][kBK][LD];
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  const long long m0 = (long long)blockIdx.y * BM, n0 = (long long)blockIdx.x * BNH;
  // kDw: this block's share of the contraction (kpart rows of it)
  const int kbeg = MODE == kDw ? (int)(blockIdx.z / 2) * kpart : 0;
  const int kend = MODE == kDw ? min(K, kbeg + kpart) : K;
  const int ksteps = (kend - kbeg + kBK - 1) / kBK;
  const int total = MODE == kDx ? 2 * ksteps : ksteps;
  float ra[LV][4], rb[LV][4];

  auto fetch = [&](int s) {
    const bool second = MODE == kDx ? s >= ksteps : (MODE == kDw ? blockIdx.z % 2 != 0 : false);
    const int k0 = kbeg + (MODE == kDx && second ? s - ksteps : s) * kBK;
    const T* A = second ? A1 : A0;
    const T* B = MODE == kDx && second ? B1 : B0;
#pragma unroll
    for (int i = 0; i < LV; ++i) {
      const int idx = tid + i * kThreads;
      if (MODE != kDw) {   // rows of K: four consecutive k of one row
        const int r = idx / (kBK / 4), k = k0 + idx % (kBK / 4) * 4;
        const long long m = m0 + r;
        load_vec(A + m * K + k, m < M ? K - k : 0, vec, ra[i]);
        if (MODE == kFwd) {
          const long long n = n0 + r % BNH;
          load_vec((r < BNH ? B0 : B1) + n * K + k, n < N ? K - k : 0, vec, rb[i]);
        }
      }
      if (MODE != kFwd) {  // rows over k: four consecutive columns of one row
        const int k = k0 + idx / (BM / 4), c = idx % (BM / 4) * 4;
        if (MODE == kDw)
          load_vec(A + (long long)k * M + m0 + c, k < kend ? (int)min(4LL, M - m0 - c) : 0, vec,
                   ra[i]);
        load_vec(B + (long long)k * N + n0 + c, k < kend ? (int)min(4LL, N - n0 - c) : 0, vec, rb[i]);
      }
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int i = 0; i < LV; ++i) {
      const int idx = tid + i * kThreads;
      const int r = idx / (kBK / 4), kr = idx % (kBK / 4) * 4;      // row-of-K order
      const int kc = idx / (BM / 4), c = idx % (BM / 4) * 4;        // rows-over-k order
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (MODE == kDw) As[buf][kc][c + e] = ra[i][e];
        else As[buf][kr + e][r] = ra[i][e];
        if (MODE == kFwd) Bs[buf][kr + e][r] = rb[i][e];
        else Bs[buf][kc][c + e] = rb[i][e];
      }
    }
  };

  // pairs of columns: two multiply-adds an instruction
  float2 acc2[TM][TM / 2];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TM / 2; ++j) acc2[i][j] = make_float2(0.f, 0.f);

  if (total > 0) {
    fetch(0);
    put(0);
  }
  __syncthreads();
  for (int s = 0; s < total; ++s) {
    const int buf = s & 1;
    if (s + 1 < total) fetch(s + 1);
#pragma unroll
    for (int k = 0; k < kBK; ++k) {
      float a[TM];
      float2 b[TM / 2];
#pragma unroll
      for (int i = 0; i < TM; i += 4) {
        const float4 v = load4(&As[buf][k][ty * TM + i]);
        a[i] = v.x; a[i + 1] = v.y; a[i + 2] = v.z; a[i + 3] = v.w;
      }
#pragma unroll
      for (int j = 0; j < H; j += 2) {
        b[j / 2] = *reinterpret_cast<const float2*>(&Bs[buf][k][tx * H + j]);
        b[(H + j) / 2] = *reinterpret_cast<const float2*>(&Bs[buf][k][BN / 2 + tx * H + j]);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TM / 2; ++j)
          acc2[i][j] = fma2(make_float2(a[i], a[i]), b[j], acc2[i][j]);
    }
    if (s + 1 < total) put(buf ^ 1);
    __syncthreads();
  }

#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const long long m = m0 + ty * TM + i;
    if (m >= M) continue;
    float acc[TM];
#pragma unroll
    for (int j = 0; j < TM / 2; ++j) {
      acc[2 * j] = acc2[i][j].x;
      acc[2 * j + 1] = acc2[i][j].y;
    }
#pragma unroll
    for (int j = 0; j < H; ++j) {
      if (MODE == kFwd) {
        const long long n = n0 + tx * H + j;
        if (n >= N) continue;
        const float g = acc[j], u = acc[H + j];
        const float sg = 1.f / (1.f + expf(-g));
        O0[m * N + n] = from_f32<T>(g * sg * u);
        if (O1) {
          O1[m * N + n] = from_f32<T>(g);
          O2[m * N + n] = from_f32<T>(u);
        }
      } else {
        T* O = MODE == kDw && blockIdx.z % 2 ? O1 : O0;
        if (MODE == kDw) O += (long long)(blockIdx.z / 2) * 2 * M * N;   // (the parts' sums)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const long long n = n0 + hf * (BN / 2) + tx * H + j;
          if (n < N) O[m * N + n] = from_f32<T>(acc[hf * H + j]);
        }
      }
    }
  }
}

// Tiles of 128 do four times the products per shared-memory word of tiles of 64;
// the small tiles only where the big ones leave SMs idle.
bool big_tiles(int mode, int M, int N) {
  const long long rows = mode == kFwd ? 64 : 128;
  return (N + rows - 1) / rows * ((M + 127LL) / 128) * (mode == kDw ? 2 : 1) >= 148;
}

template <typename T, int MODE>
cudaError_t launch_simt(const T* A0, const T* A1, const T* B0, const T* B1, T* O0, T* O1, T* O2,
                        int M, int N, int K, int parts, cudaStream_t st) {
  // 16-byte (fp32) or 8-byte (bf16) vectors need rows that are a multiple of four elements
  const bool vec = MODE == kDw ? (M % 4 == 0 && N % 4 == 0)
                               : (K % 4 == 0 && (MODE == kFwd || N % 4 == 0));
  const int z = MODE == kDw ? 2 * parts : 1;
  const int kpart = ((K + parts - 1) / parts + kBK - 1) / kBK * kBK;
  const long long rows = MODE == kFwd ? 64 : 128;
  if (big_tiles(MODE, M, N)) {
    const dim3 grid((unsigned)((N + rows - 1) / rows), (unsigned)((M + 127LL) / 128), z);
    glu_simt_kernel<T, MODE, 8><<<grid, kThreads, 0, st>>>(A0, A1, B0, B1, O0, O1, O2, M, N, K,
                                                           kpart, vec);
  } else {
    const dim3 grid((unsigned)((N + rows / 2 - 1) / (rows / 2)), (unsigned)((M + 63LL) / 64), z);
    glu_simt_kernel<T, MODE, 4><<<grid, kThreads, 0, st>>>(A0, A1, B0, B1, O0, O1, O2, M, N, K,
                                                           kpart, vec);
  }
  return cudaGetLastError();
}

// dg, du from g, u, dh (n elements each): HBM-bound, three arrays read and two
// written (8200 x 5632 in bf16: 77 us, 6.0 TB/s).
template <typename T, bool kVec>
__global__ void __launch_bounds__(256)
glu_act_bwd_kernel(const T* __restrict__ g, const T* __restrict__ u, const T* __restrict__ dh,
                   T* __restrict__ dg, T* __restrict__ du, long long n) {
  constexpr int E = kVec ? 4 : 1;
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * E;
  if (i >= n) return;
  float gv[E], uv[E], dv[E], a[E], b[E];
  if constexpr (kVec) {
    const float4 p = load4(g + i), q = load4(u + i), r = load4(dh + i);
    gv[0] = p.x; gv[1] = p.y; gv[2] = p.z; gv[3] = p.w;
    uv[0] = q.x; uv[1] = q.y; uv[2] = q.z; uv[3] = q.w;
    dv[0] = r.x; dv[1] = r.y; dv[2] = r.z; dv[3] = r.w;
  } else {
    gv[0] = to_f32(g[i]); uv[0] = to_f32(u[i]); dv[0] = to_f32(dh[i]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float s = 1.f / (1.f + expf(-gv[e]));
    a[e] = dv[e] * uv[e] * (s * fmaf(gv[e], 1.f - s, 1.f));
    b[e] = dv[e] * (gv[e] * s);
  }
  if constexpr (kVec) {
    store4(dg + i, make_float4(a[0], a[1], a[2], a[3]));
    store4(du + i, make_float4(b[0], b[1], b[2], b[3]));
  } else {
    dg[i] = from_f32<T>(a[0]);
    du[i] = from_f32<T>(b[0]);
  }
}

template <typename T>
cudaError_t fwd_simt(const GluArgs& a, cudaStream_t st) {
  return launch_simt<T, kFwd>(static_cast<const T*>(a.x), nullptr, static_cast<const T*>(a.wg),
                              static_cast<const T*>(a.wu), static_cast<T*>(a.h),
                              static_cast<T*>(a.g), static_cast<T*>(a.u), a.M, a.I, a.D, 1, st);
}

template <typename T>
cudaError_t act_bwd(const GluBwdArgs& a, cudaStream_t st) {
  const long long n = (long long)a.M * a.I;
  const bool vec = n % 4 == 0;
  const long long blocks = (n / (vec ? 4 : 1) + 255) / 256;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const T *g = static_cast<const T*>(a.g), *u = static_cast<const T*>(a.u),
          *dh = static_cast<const T*>(a.dh);
  T *dg = static_cast<T*>(a.dg), *du = static_cast<T*>(a.du);
  if (vec) glu_act_bwd_kernel<T, true><<<(unsigned)blocks, 256, 0, st>>>(g, u, dh, dg, du, n);
  else glu_act_bwd_kernel<T, false><<<(unsigned)blocks, 256, 0, st>>>(g, u, dh, dg, du, n);
  return cudaGetLastError();
}

template <typename T>
cudaError_t bwd_products_simt(const GluBwdArgs& a, cudaStream_t st) {
  const T *x = static_cast<const T*>(a.x), *wg = static_cast<const T*>(a.wg),
          *wu = static_cast<const T*>(a.wu), *dg = static_cast<const T*>(a.dg),
          *du = static_cast<const T*>(a.du);
  cudaError_t e = cudaSuccess;
  if (a.dx)
    e = launch_simt<T, kDx>(dg, du, wg, wu, static_cast<T*>(a.dx), nullptr, nullptr, a.M, a.D,
                            a.I, 1, st);
  if (e != cudaSuccess || !a.dwg) return e;
  T *dwg = static_cast<T*>(a.dwg), *dwu = static_cast<T*>(a.dwu);
  const int parts = glu_dw_parts(a.M, a.D, a.I, a.dtype);
  const long long n = (long long)a.I * a.D;
  if (parts > 1) {
    dwg = reinterpret_cast<T*>(a.part);
    dwu = dwg + n;
  }
  e = launch_simt<T, kDw>(dg, du, x, nullptr, dwg, dwu, nullptr, a.I, a.D, a.M, parts, st);
  if (e != cudaSuccess || parts == 1) return e;
  const SumSegments out{{static_cast<float*>(a.dwg), static_cast<float*>(a.dwu), nullptr},
                        {n, n, 0}};
  return launch_sum_partials(a.part, parts, 2 * n, out, st);
}

}  // namespace

// The weights' gradients in fp32 contract over the tokens: few output tiles leave
// SMs idle, and the tokens are cut into parts (of 512 or more) whose sums a second
// kernel adds up (10000 x 128 x 330: 0.5 ms in one part).
int glu_dw_parts(int M, int D, int I, int dtype) {
  if (dtype != kFP32 || M < 1024 || big_tiles(kDw, I, D)) return 1;
  const long long tiles = 2LL * ((I + 63) / 64) * ((D + 63) / 64);
  if (tiles >= 148) return 1;
  long long p = 296 / tiles;
  if (p > M / 512) p = M / 512;
  return p < 1 ? 1 : p > 16 ? 16 : (int)p;
}

cudaError_t launch_glu_fwd(const GluArgs& a, cudaStream_t st) {
  if (a.M == 0 || a.I == 0) return cudaSuccess;
  if (glu_tc_supported(a.M, a.D, a.I, a.dtype)) return launch_glu_tc_fwd(a, st);
  return a.dtype == kBF16 ? fwd_simt<__nv_bfloat16>(a, st) : fwd_simt<float>(a, st);
}

cudaError_t launch_glu_bwd(const GluBwdArgs& a, cudaStream_t st) {
  if (a.M > 0 && a.I > 0) {
    const cudaError_t e =
        a.dtype == kBF16 ? act_bwd<__nv_bfloat16>(a, st) : act_bwd<float>(a, st);
    if (e != cudaSuccess) return e;
  }
  if (a.D == 0) return cudaSuccess;
  if (glu_tc_supported(a.M, a.D, a.I, a.dtype)) return launch_glu_tc_bwd(a, st);
  return a.dtype == kBF16 ? bwd_products_simt<__nv_bfloat16>(a, st)
                          : bwd_products_simt<float>(a, st);
}

}  // namespace gdn
