// The gated linear unit of the feed-forward block (model.py:162-180 before its
// down projection): h = silu(x Wg^T) * (x Wu^T), and its gradients
//   dg = dh u s (1 + g (1 - s)),  du = dh g s   (s = sigmoid(g)),
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x.
//
// This file holds the CUDA-core form, for fp32 inputs (the products are fp32
// fused multiply-adds) and for bf16 widths that the tensor-core form does not
// take, and the elementwise step between the two halves of the backward, which
// every form shares.  One tiled kernel computes all products: 256 threads,
// the operands transposed into shared memory and prefetched a step ahead in
// registers, fp32 accumulators (4100 x 1024 x 2048 in fp32: forward 745 us, 46 TFLOP/s;
// dx 779, both weights' gradients 653).  The two projections share one
// tile of x: half of a tile's columns come from Wg and half from Wu, so that a
// thread ends with g and u of the same elements.  Few tokens have a kernel of
// their own, bound by the weights' bytes up to four of them (2048 x 5632 in fp32: one
// token 16 us from HBM, 10.5 with part of them in L2, where the tiles took 147).
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

// A projection kept for the backward, in T or (keep32) in fp32.
template <typename T>
__device__ __forceinline__ void keep(T* p, long long i, float v, bool keep32) {
  if (sizeof(T) < 4 && keep32) reinterpret_cast<float*>(p)[i] = v;
  else p[i] = from_f32<T>(v);
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
// A thread takes TR rows and TC columns, half of them from either half of the tile.  A
// step's shared-memory reads take as many cycles of a warp as a thread reads words, TR +
// TC for TR TC multiply-adds: at 8 x 8 as many as the multiply-adds, which then run at
// 48 to 53 TFLOP/s (8 x 16 reads fewer, but leaves two warps a scheduler: no faster).
template <typename T, int MODE, int TR, int TC>
__global__ void __launch_bounds__(kThreads, TR * TC >= 64 ? 2 : TR * TC >= 32 ? 3 : 4)
glu_simt_kernel(const T* __restrict__ A0, const T* __restrict__ A1, const T* __restrict__ B0,
                const T* __restrict__ B1, T* __restrict__ O0, T* __restrict__ O1,
                T* __restrict__ O2, int M, int N, int K, int kpart, bool vec, bool keep32) {
  constexpr int BM = 16 * TR, BN = 16 * TC, H = TC / 2;
  constexpr int BNH = MODE == kFwd ? BN / 2 : BN;   // output columns of a tile
  constexpr int LA = BM * kBK / 4 / kThreads;        // vectors of A's tile per thread
  constexpr int LB = BN * kBK / 4 / kThreads;
  constexpr int CG = H < 4 ? H : 4;                 // columns side by side
  __shared__ __align__(16) float As[2][kBK][BM + 4], Bs[2][kBK][BN + 4];
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  const long long m0 = (long long)blockIdx.y * BM, n0 = (long long)blockIdx.x * BNH;
  const int mleft = (int)min((long long)BM, M - m0), nleft = (int)min((long long)BNH, N - n0);
  // this block's share of the contraction: kpart elements (kDw), kpart steps (kDx)
  const int kbeg = MODE == kDw ? (int)(blockIdx.z / 2) * kpart : 0;
  const int kend = MODE == kDw ? min(K, kbeg + kpart) : K;
  const int ksteps = (kend - kbeg + kBK - 1) / kBK;
  const int first = MODE == kDx ? (int)blockIdx.z * kpart : 0;
  const int total = MODE == kDx ? min(2 * ksteps, first + kpart) : ksteps;
  float ra[LA][4], rb[LB][4];

  // (offsets inside a tile fit 32 bits: its rows are at most 128 of 2^22 elements)
  auto fetch = [&](int s) {
    const bool second = MODE == kDx ? s >= ksteps : (MODE == kDw ? blockIdx.z % 2 != 0 : false);
    const int k0 = kbeg + (MODE == kDx && second ? s - ksteps : s) * kBK, left = kend - k0;
    const T* A = (second ? A1 : A0) + (MODE == kDw ? (long long)k0 * M + m0 : m0 * K + k0);
    const T* B = (MODE == kDx && second ? B1 : B0) +
                 (MODE == kFwd ? n0 * K + k0 : (long long)k0 * N + n0);
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      const int idx = tid + i * kThreads;
      if (MODE == kDw) {   // rows over k: four consecutive columns of one row
        const int r = idx / (BM / 4), c = idx % (BM / 4) * 4;
        load_vec(A + (r * M + c), r < left ? mleft - c : 0, vec, ra[i]);
      } else {             // rows of K: four consecutive k of one row
        const int r = idx / (kBK / 4), k = idx % (kBK / 4) * 4;
        load_vec(A + (r * K + k), r < mleft ? left - k : 0, vec, ra[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      const int idx = tid + i * kThreads;
      if (MODE == kFwd) {
        const int r = idx / (kBK / 4), k = idx % (kBK / 4) * 4;
        const bool up = LB > 1 ? i >= LB / 2 : r >= BNH;   // a row of Wu
        const int rr = r - (up ? BNH : 0);
        // (Wu by its distance from Wg, both 16-byte aligned: a second pointer spills, and
        // 4100 x 1024 x 2048 takes 826 us instead of 745)
        load_vec((up ? B + (B1 - B0) : B) + (rr * K + k), rr < nleft ? left - k : 0, vec, rb[i]);
      } else {
        const int r = idx / (BN / 4), c = idx % (BN / 4) * 4;
        load_vec(B + (r * N + c), r < left ? nleft - c : 0, vec, rb[i]);
      }
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      const int idx = tid + i * kThreads;
      if (MODE == kDw) {
        store4(&As[buf][idx / (BM / 4)][idx % (BM / 4) * 4],
               make_float4(ra[i][0], ra[i][1], ra[i][2], ra[i][3]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) As[buf][idx % (kBK / 4) * 4 + e][idx / (kBK / 4)] = ra[i][e];
      }
    }
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      const int idx = tid + i * kThreads;
      if (MODE == kFwd) {
#pragma unroll
        for (int e = 0; e < 4; ++e) Bs[buf][idx % (kBK / 4) * 4 + e][idx / (kBK / 4)] = rb[i][e];
      } else if (MODE == kDx) {   // (as a vector it spills: 903 against 780 us, 4100 x 1024 x 2048)
#pragma unroll
        for (int e = 0; e < 4; ++e) Bs[buf][idx / (BN / 4)][idx % (BN / 4) * 4 + e] = rb[i][e];
      } else {
        store4(&Bs[buf][idx / (BN / 4)][idx % (BN / 4) * 4],
               make_float4(rb[i][0], rb[i][1], rb[i][2], rb[i][3]));
      }
    }
  };

  // pairs of columns: two multiply-adds an instruction
  float2 acc2[TR][TC / 2];
#pragma unroll
  for (int i = 0; i < TR; ++i)
#pragma unroll
    for (int j = 0; j < TC / 2; ++j) acc2[i][j] = make_float2(0.f, 0.f);

  if (first < total) {
    fetch(first);
    put(0);
  }
  __syncthreads();
  for (int s = first; s < total; ++s) {
    const int buf = (s - first) & 1;
    if (s + 1 < total) fetch(s + 1);
#pragma unroll
    for (int k = 0; k < kBK; ++k) {
      float a[TR];
      float2 b[TC / 2];
#pragma unroll
      for (int i = 0; i < TR; i += 4) {
        const float4 v = load4(&As[buf][k][ty * TR + i]);
        a[i] = v.x; a[i + 1] = v.y; a[i + 2] = v.z; a[i + 3] = v.w;
      }
#pragma unroll
      for (int j = 0; j < TC; j += CG) {
        const float* p = &Bs[buf][k][j / CG * 16 * CG + tx * CG];
        if constexpr (CG == 4) {
          const float4 v = load4(p);
          b[j / 2] = make_float2(v.x, v.y);
          b[j / 2 + 1] = make_float2(v.z, v.w);
        } else {
          b[j / 2] = *reinterpret_cast<const float2*>(p);
        }
      }
#pragma unroll
      for (int i = 0; i < TR; ++i)
#pragma unroll
        for (int j = 0; j < TC / 2; ++j)
          acc2[i][j] = fma2(make_float2(a[i], a[i]), b[j], acc2[i][j]);
    }
    if (s + 1 < total) put(buf ^ 1);
    __syncthreads();
  }

#pragma unroll
  for (int i = 0; i < TR; ++i) {
    const long long m = m0 + ty * TR + i;
    if (m >= M) continue;
    float acc[TC];
#pragma unroll
    for (int j = 0; j < TC / 2; ++j) {
      acc[2 * j] = acc2[i][j].x;
      acc[2 * j + 1] = acc2[i][j].y;
    }
#pragma unroll
    for (int j = 0; j < H; ++j) {
      const int cj = j / CG * 16 * CG + tx * CG + j % CG;   // column in the tile's half
      if (MODE == kFwd) {
        const long long n = n0 + cj;
        if (n >= N) continue;
        const float g = acc[j], u = acc[H + j];
        const float sg = 1.f / (1.f + expf(-g));
        O0[m * N + n] = from_f32<T>(g * sg * u);
        if (O1) {
          keep(O1, m * N + n, g, keep32);
          keep(O2, m * N + n, u, keep32);
        }
      } else {
        T* O = MODE == kDw && blockIdx.z % 2 ? O1 : O0;
        // (the parts' sums)
        if (MODE == kDw) O += (long long)(blockIdx.z / 2) * 2 * M * N;
        if (MODE == kDx) O += (long long)blockIdx.z * M * N;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const long long n = n0 + hf * (BN / 2) + cj;
          if (n < N) O[m * N + n] = from_f32<T>(acc[hf * H + j]);
        }
      }
    }
  }
}

struct SimtPlan {
  int tile;    // 0: 64 x 64, 1: 64 x 128, 2: 128 x 128
  int parts;   // of the contraction, whose sums are added up afterwards
  double us;   // its estimate
};

constexpr int kTileTR[3] = {4, 4, 8}, kTileTC[3] = {4, 8, 8};

long long simt_tiles(int mode, int tile, int M, int N) {
  const long long rows = 16 * kTileTR[tile], cols = (mode == kFwd ? 8 : 16) * kTileTC[tile];
  return (M + rows - 1) / rows * ((N + cols - 1) / cols) * (mode == kDw ? 2 : 1);
}

// Tile and parts by the time they take: the fullest SM's tiles times a tile's, which per
// 1024 elements of the contraction measured 35, 58 and 94 us (a lone tile on its SM 43,
// 73 and 112: nothing covers its waits), and the partial sums' bytes.  A tile of 128 x
// 128 does twice the products per shared-memory word of one of 64 x 64, but fills 148
// SMs in coarser steps: 513 x 1024 x 2048 forward 124 us on 64 x 128 (143 on 64 x 64, 194
// on 128 x 128).  In parts: dx of 64 tokens of 296 x 11000 47 us, in one 0.95 ms.
SimtPlan simt_plan(int mode, int M, int N, int K, bool parts_ok) {
  static const double kStep[3] = {35., 58., 94.}, kLone[3] = {8., 15., 18.};
  const int sms = device_sm_count();
  const double depth = (mode == kDx ? 2. : 1.) * K / 1024.;
  SimtPlan best{0, 1, 1e300};
  for (int parts = 1; parts <= (parts_ok ? 64 : 1); parts *= 2) {
    if (parts > 1 && depth * 1024. / parts < 128.) break;
    for (int tile = 0; tile < 3; ++tile) {
      const long long n = simt_tiles(mode, tile, M, N) * parts;
      const long long per_sm = (n + sms - 1) / sms;
      double t = (kStep[tile] * per_sm + (per_sm == 1 ? kLone[tile] : 0.)) * depth / parts;
      if (parts > 1) t += 4. + (mode == kDw ? 2. : 1.) * M * N * parts * 8. / 3e6;
      if (t < best.us * 0.98) best = SimtPlan{tile, parts, t};
    }
  }
  return best;
}

template <typename T, int MODE>
cudaError_t launch_simt(const T* A0, const T* A1, const T* B0, const T* B1, T* O0, T* O1, T* O2,
                        int M, int N, int K, const SimtPlan& p, cudaStream_t st,
                        bool keep32 = false) {
  // 16-byte (fp32) or 8-byte (bf16) vectors need rows that are a multiple of four elements
  const bool vec = MODE == kDw ? (M % 4 == 0 && N % 4 == 0)
                               : (K % 4 == 0 && (MODE == kFwd || N % 4 == 0));
  const int steps = (K + kBK - 1) / kBK * (MODE == kDx ? 2 : 1);
  const int kpart = (steps + p.parts - 1) / p.parts * (MODE == kDw ? kBK : 1);
  const long long rows = 16 * kTileTR[p.tile], cols = (MODE == kFwd ? 8 : 16) * kTileTC[p.tile];
  const dim3 grid((unsigned)((N + cols - 1) / cols), (unsigned)((M + rows - 1) / rows),
                  (MODE == kDw ? 2 : 1) * p.parts);
  auto go = [&](auto kernel) {
    kernel<<<grid, kThreads, 0, st>>>(A0, A1, B0, B1, O0, O1, O2, M, N, K, kpart, vec, keep32);
    return cudaGetLastError();
  };
  switch (p.tile) {
    case 0: return go(glu_simt_kernel<T, MODE, 4, 4>);
    case 1: return go(glu_simt_kernel<T, MODE, 4, 8>);
    default: return go(glu_simt_kernel<T, MODE, 8, 8>);
  }
}

// The parts' sums in their order: out[i] over part[p][i], the first `split` elements to
// out0 and the rest to out1 (HBM-bound; all three counts multiples of four with kVec).
template <bool kVec>
__global__ void __launch_bounds__(256)
glu_sum_kernel(const float* __restrict__ part, int parts, long long n, long long split,
               float* __restrict__ out0, float* __restrict__ out1) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * (kVec ? 4 : 1);
  if (i >= n) return;
  float* out = i < split ? out0 + i : out1 + (i - split);
  if constexpr (kVec) {
    float4 s = load4(part + i);
#pragma unroll 4
    for (int p = 1; p < parts; ++p) {
      const float4 v = load4(part + p * n + i);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    store4(out, s);
  } else {
    float s = part[i];
#pragma unroll 4
    for (int p = 1; p < parts; ++p) s += part[p * n + i];
    *out = s;
  }
}

cudaError_t sum_parts(const float* part, int parts, long long n, long long split, void* out0,
                      void* out1, cudaStream_t st) {
  const bool vec = n % 4 == 0 && split % 4 == 0;
  const long long blocks = (n / (vec ? 4 : 1) + 255) / 256;
  if (blocks == 0) return cudaSuccess;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  float *o0 = static_cast<float*>(out0), *o1 = static_cast<float*>(out1);
  if (vec) glu_sum_kernel<true><<<(unsigned)blocks, 256, 0, st>>>(part, parts, n, split, o0, o1);
  else glu_sum_kernel<false><<<(unsigned)blocks, 256, 0, st>>>(part, parts, n, split, o0, o1);
  return cudaGetLastError();
}

// dg, du from g, u, dh (n elements each): HBM-bound, three arrays read and two
// written (8200 x 5632 in bf16 with g and u kept in fp32: 90 us for 647 MB; kept in bf16
// 77 us, 6.0 TB/s).
template <typename T, typename Kept, bool kVec>
__global__ void __launch_bounds__(256)
glu_act_bwd_kernel(const Kept* __restrict__ g, const Kept* __restrict__ u,
                   const T* __restrict__ dh, T* __restrict__ dg, T* __restrict__ du, long long n) {
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

// Four elements from `p` on: one vector (kVec), or one by one; all of them in range
// (kAll) or the first `n`.  No branch in the full form, so that loads of many rows
// go out together.
template <typename T, bool kVec, bool kAll>
__device__ __forceinline__ float4 load_four(const T* p, int n) {
  if constexpr (kAll && kVec) return load4(p);
  if constexpr (kAll) return make_float4(to_f32(p[0]), to_f32(p[1]), to_f32(p[2]), to_f32(p[3]));
  float v[4];
  load_vec(p, n, kVec, v);
  return make_float4(v[0], v[1], v[2], v[3]);
}

// Adds 2 N float2 values over the lanes by halves: each step keeps one half of the
// values and takes the partner lane's sums of it.  v[0] ends as the sum of value
// lane / (32 / N) for N values of the start.
template <int N, int O>
__device__ __forceinline__ void lane_sums(float2* v, int lane) {
  if constexpr (O > 0) {
    if constexpr (N > 1) {
      const bool hi = lane & O;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 keep = hi ? v[i + N / 2] : v[i], give = hi ? v[i] : v[i + N / 2];
        v[i].x = keep.x + __shfl_xor_sync(0xffffffffu, give.x, O);
        v[i].y = keep.y + __shfl_xor_sync(0xffffffffu, give.y, O);
      }
      lane_sums<N / 2, O / 2>(v, lane);
    } else {
      v[0].x += __shfl_xor_sync(0xffffffffu, v[0].x, O);
      v[0].y += __shfl_xor_sync(0xffffffffu, v[0].y, O);
      lane_sums<1, O / 2>(v, lane);
    }
  }
}

// Few tokens on the CUDA cores: a warp owns two columns of the result, that is four
// weight rows, and walks them 128 elements a step with the next steps' loads in
// flight; every 16 bytes of x (in L1, the SM's warps walk it together) serve the four
// rows.  Even and odd elements are summed apart (two multiply-adds an instruction),
// then the 32 lanes' sums are added up by halves in a fixed order, which leaves g and
// u of one token and column in a lane.
template <typename T, int MB, bool kVec>
__global__ void __launch_bounds__(128)
glu_rows_kernel(const T* __restrict__ x, const T* __restrict__ wg, const T* __restrict__ wu,
                T* __restrict__ h, T* __restrict__ go, T* __restrict__ uo, int M, int I, int K,
                bool keep32) {
  const int lane = threadIdx.x % 32;
  const long long n0 = ((long long)blockIdx.x * 4 + threadIdx.x / 32) * 2;
  if (n0 >= I) return;
  const int m0 = blockIdx.y * MB;
  const int last = n0 + 1 < I;
  const T* w[4] = {wg + n0 * K + lane * 4, wu + n0 * K + lane * 4, wg + (n0 + last) * K + lane * 4,
                   wu + (n0 + last) * K + lane * 4};
  // (tokens past the last read the last one again; their sums are not stored)
  const T* xr = x + (long long)m0 * K + lane * 4;
  const int mlast = min(MB, M - m0) - 1;
  float2 acc[MB][4];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[m][r] = make_float2(0.f, 0.f);
  auto add = [&](int m, const float4& xv, const float4 (&wv)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      acc[m][r] = fma2(make_float2(wv[r].x, wv[r].y), make_float2(xv.x, xv.y), acc[m][r]);
      acc[m][r] = fma2(make_float2(wv[r].z, wv[r].w), make_float2(xv.z, xv.w), acc[m][r]);
    }
  };
  const int full = K / 128 * 128;
  // Steps whose weights are in flight (from HBM, 2048 x 5632 and 4096 x 4096: one token 16.3
  // and 24.5 us, with one step ahead 18.2 and 27.9; four tokens 20.5 and 27.3, 24.8 and 51.4).
  constexpr int kAhead = MB <= 2 ? 2 : MB == 4 ? 4 : 1;
  float4 wn[kAhead][4];
  if (full > 0) {
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        wn[s][r] = load_four<T, kVec, true>(w[r] + min(s * 128, full - 128), 4);
  }
#pragma unroll kAhead
  for (int k = 0; k < full; k += 128) {
    float4 wv[4], xv[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m)
      xv[m] = load_four<T, kVec, true>(xr + (long long)min(m, mlast) * K + k, 4);
    const int next = min(k + kAhead * 128, full - 128);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      wv[r] = wn[0][r];
#pragma unroll
      for (int s = 0; s + 1 < kAhead; ++s) wn[s][r] = wn[s + 1][r];
      wn[kAhead - 1][r] = load_four<T, kVec, true>(w[r] + next, 4);
    }
#pragma unroll
    for (int m = 0; m < MB; ++m) add(m, xv[m], wv);
  }
  if (full < K) {
    const int n = K - full - lane * 4;
    float4 wv[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) wv[r] = load_four<T, kVec, false>(w[r] + full, n);
#pragma unroll
    for (int m = 0; m < MB; ++m)
      add(m, load_four<T, kVec, false>(xr + (long long)min(m, mlast) * K + full, n), wv);
  }
  // value 2 m + c: g and u of token m and column c
  float2 v[2 * MB];
#pragma unroll
  for (int i = 0; i < 2 * MB; ++i) {
    const float2 a = acc[i / 2][i % 2 * 2], b = acc[i / 2][i % 2 * 2 + 1];
    v[i] = make_float2(a.x + a.y, b.x + b.y);
  }
  lane_sums<2 * MB, 16>(v, lane);
  constexpr int kSame = 16 / MB;   // lanes that hold the same value
  const int i = lane / kSame;
  const long long m = m0 + i / 2, c = n0 + i % 2;
  if (lane % kSame == 0 && m < M && c < I) {
    const float g = v[0].x, u = v[0].y;
    const float sg = 1.f / (1.f + expf(-g));
    h[m * I + c] = from_f32<T>(g * sg * u);
    if (go) {
      keep(go, m * I + c, g, keep32);
      keep(uo, m * I + c, u, keep32);
    }
  }
}

template <typename T, int MB>
cudaError_t launch_rows(const GluArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)((a.I + 7) / 8), (unsigned)((a.M + MB - 1) / MB));
  const T *x = static_cast<const T*>(a.x), *wg = static_cast<const T*>(a.wg),
          *wu = static_cast<const T*>(a.wu);
  T *h = static_cast<T*>(a.h), *g = static_cast<T*>(a.g), *u = static_cast<T*>(a.u);
  if (a.D % 4 == 0)
    glu_rows_kernel<T, MB, true><<<grid, 128, 0, st>>>(x, wg, wu, h, g, u, a.M, a.I, a.D,
                                                       a.kept == kFP32);
  else
    glu_rows_kernel<T, MB, false><<<grid, 128, 0, st>>>(x, wg, wu, h, g, u, a.M, a.I, a.D,
                                                        a.kept == kFP32);
  return cudaGetLastError();
}

template <typename T>
cudaError_t fwd_simt(const GluArgs& a, cudaStream_t st) {
  if (a.M <= 1) return launch_rows<T, 1>(a, st);
  if (a.M <= 2) return launch_rows<T, 2>(a, st);
  if (a.M <= 4) return launch_rows<T, 4>(a, st);
  if (a.M <= 8) return launch_rows<T, 8>(a, st);
  // 16 tokens at a time: 2.7 us for a million weights of one projection (and 250 a column
  // for the sums over the lanes): 37 tokens of 2048 x 5632 107 us, on the tiles 150; 64
  // of 296 x 11000 82 us, on the tiles 36.
  const SimtPlan p = simt_plan(kFwd, a.M, a.I, a.D, false);
  const double rows_us = 3. + (a.M + 15) / 16 * 2.7e-6 * a.I * (a.D + 250.);
  if (a.M <= 16 || (a.M <= 128 && rows_us < p.us)) return launch_rows<T, 16>(a, st);
  return launch_simt<T, kFwd>(static_cast<const T*>(a.x), nullptr, static_cast<const T*>(a.wg),
                              static_cast<const T*>(a.wu), static_cast<T*>(a.h),
                              static_cast<T*>(a.g), static_cast<T*>(a.u), a.M, a.I, a.D,
                              p, st, a.kept == kFP32);
}

template <typename T, typename Kept>
cudaError_t act_bwd(const GluBwdArgs& a, cudaStream_t st) {
  const long long n = (long long)a.M * a.I;
  const bool vec = n % 4 == 0;
  const long long blocks = (n / (vec ? 4 : 1) + 255) / 256;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const Kept *g = static_cast<const Kept*>(a.g), *u = static_cast<const Kept*>(a.u);
  const T* dh = static_cast<const T*>(a.dh);
  T *dg = static_cast<T*>(a.dg), *du = static_cast<T*>(a.du);
  if (vec) glu_act_bwd_kernel<T, Kept, true><<<(unsigned)blocks, 256, 0, st>>>(g, u, dh, dg, du, n);
  else glu_act_bwd_kernel<T, Kept, false><<<(unsigned)blocks, 256, 0, st>>>(g, u, dh, dg, du, n);
  return cudaGetLastError();
}

template <typename T>
cudaError_t bwd_products_simt(const GluBwdArgs& a, cudaStream_t st) {
  const T *x = static_cast<const T*>(a.x), *wg = static_cast<const T*>(a.wg),
          *wu = static_cast<const T*>(a.wu), *dg = static_cast<const T*>(a.dg),
          *du = static_cast<const T*>(a.du);
  cudaError_t e = cudaSuccess;
  if (a.dx) {
    const SimtPlan p = simt_plan(kDx, a.M, a.D, a.I, a.dtype == kFP32);
    const long long n = (long long)a.M * a.D;
    T* dx = p.parts > 1 ? reinterpret_cast<T*>(a.part) : static_cast<T*>(a.dx);
    e = launch_simt<T, kDx>(dg, du, wg, wu, dx, nullptr, nullptr, a.M, a.D, a.I, p, st);
    if (e == cudaSuccess && p.parts > 1)
      e = sum_parts(a.part, p.parts, n, n, a.dx, nullptr, st);
  }
  if (e != cudaSuccess || !a.dwg) return e;
  T *dwg = static_cast<T*>(a.dwg), *dwu = static_cast<T*>(a.dwu);
  const SimtPlan p = simt_plan(kDw, a.I, a.D, a.M, a.dtype == kFP32);
  const long long n = (long long)a.I * a.D;
  if (p.parts > 1) {
    dwg = reinterpret_cast<T*>(a.part);
    dwu = dwg + n;
  }
  e = launch_simt<T, kDw>(dg, du, x, nullptr, dwg, dwu, nullptr, a.I, a.D, a.M, p, st);
  if (e != cudaSuccess || p.parts == 1) return e;
  return sum_parts(a.part, p.parts, 2 * n, n, a.dwg, a.dwu, st);
}

}  // namespace

// A product with few output tiles leaves SMs idle; its contraction is cut into parts (in
// fp32, and dx on the tensor cores, whose accumulators also take no more than 32768 terms
// each), whose sums a second kernel adds up in a fixed order.
size_t glu_part_floats(int M, int D, int I, int dtype) {
  if (glu_tc_widths(D, I, dtype)) return glu_tc_part_floats(M, D, I);
  if (dtype != kFP32) return 0;
  const size_t dx = simt_plan(kDx, M, D, I, true).parts, dw = simt_plan(kDw, I, D, M, true).parts;
  const size_t a = dx > 1 ? dx * M * D : 0, b = dw > 1 ? dw * 2 * I * D : 0;
  return a > b ? a : b;
}

cudaError_t launch_glu_fwd(const GluArgs& a, cudaStream_t st) {
  if (a.M == 0 || a.I == 0) return cudaSuccess;
  if (glu_tc_supported(a.M, a.D, a.I, a.dtype)) return launch_glu_tc_fwd(a, st);
  return a.dtype == kBF16 ? fwd_simt<__nv_bfloat16>(a, st) : fwd_simt<float>(a, st);
}

cudaError_t launch_glu_bwd(const GluBwdArgs& a, cudaStream_t st) {
  const cudaError_t e = a.dtype == kFP32   ? act_bwd<float, float>(a, st)
                        : a.kept == kFP32 ? act_bwd<__nv_bfloat16, float>(a, st)
                                          : act_bwd<__nv_bfloat16, __nv_bfloat16>(a, st);
  if (e != cudaSuccess) return e;
  if (glu_tc_supported(a.M, a.D, a.I, a.dtype)) return launch_glu_tc_bwd(a, st);
  return a.dtype == kBF16 ? bwd_products_simt<__nv_bfloat16>(a, st)
                          : bwd_products_simt<float>(a, st);
}

}  // namespace gdn
