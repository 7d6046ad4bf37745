// The gated linear unit's products on tcgen05 (bf16; formulas in glu.cu).
//
// One kernel, three products, each a tile of 256 x 256 fp32 accumulators held by
// a pair of CTAs (cta_group::2, 128 rows each):
//   kFwd  [g | u] = x [Wg | Wu]^T: 128 columns of Wg in the pair's first CTA, the
//         same columns of Wu in its second, so that every epilogue thread finds g
//         and u of its row in its own TMEM and writes silu(g) u (and g, u in
//         training) without the projections ever reaching HBM between;
//   kDx   dx = dg Wg + du Wu, one accumulation over both;
//   kDw   dWg = dg^T x, then dWu = du^T x, as tiles of one launch.
// Operands that run along the contraction are K-major tiles, the others MN-major
// ones (the transposes cost nothing: the tensor cores read either order).
//
// Compute-bound.  A pair halves what each SM has to read and write in shared
// memory per product against a tile of its own (each CTA stages half of B), and
// 256 x 256 is the largest tile whose accumulator fits TMEM twice, so that a
// tile's epilogue runs under the next tile's products.  Persistent: one pair per
// two SMs, tiles in panels of 16 row tiles so that what runs at one time shares
// its operands in L2.  Warp 0 loads (TMA, 128-byte swizzle, five stages of 64
// along the contraction), warp 1 of the even CTA issues the products, eight
// warps run the epilogue through 128-byte-swizzled staging and TMA stores, which
// clip ragged edges (loads fill them with zeros).
#include "gdn_common.cuh"
#include "gdn_internal.h"
#include "ptx.cuh"

namespace gdn {

namespace {

enum Kind : int { kFwd = 0, kDx = 1, kDw = 2 };

constexpr int kStages = 5;
constexpr int kTile = 256;              // rows and accumulator columns of a pair's tile
constexpr int kBK = 64;
constexpr int kOperand = 16384;         // bytes of a CTA's half of A or B in a stage
constexpr int kStageBytes = 2 * kOperand;
constexpr int kBox = 16384;             // 128 rows x 64 bf16 columns of staging
constexpr int kEpiWarps = 8;
constexpr int kTcThreads = 64 + 32 * kEpiWarps;
constexpr int kOffStaging = kStages * kStageBytes;
constexpr int kOffBars = kOffStaging + 4 * kBox;
constexpr int kNumBars = 2 * kStages + 4;
constexpr int kSmemBytes = kOffBars + kNumBars * 8 + 16 + 1024;   // + alignment
constexpr int kPanel = 16;              // row tiles of a panel
constexpr uint32_t kSW128 = 2;

struct alignas(64) GluMaps {
  CUtensorMap a[2];
  CUtensorMap b[2];
  CUtensorMap out[3];
};

struct GluShape {
  int tiles_m, tiles_n;   // output tiles (kDw: of dWg; dWu has as many again)
  int kblocks;            // 64-wide steps along the contraction (kDx: of each half)
  int keep;               // kFwd: g and u are stored
  int rows, cols;         // of the output
};

template <int KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTcThreads, 1)
glu_tc_kernel(const __grid_constant__ GluMaps maps, const GluShape sh) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = smem_raw + (1024u - (smem_u32(smem_raw) & 1023u)) % 1024u;
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + kOffBars);
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;    // an accumulator is complete
  uint64_t* tempty = tfull + 2;         // an accumulator has been read (even CTA's is used)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 2 * kEpiWarps);
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int npairs = gridDim.x / 2, pair = blockIdx.x / 2;
  const int tm = KIND == kDw ? 2 * sh.tiles_m : sh.tiles_m;
  const long long tiles = (long long)tm * sh.tiles_n;
  const int ksteps = KIND == kDx ? 2 * sh.kblocks : sh.kblocks;
  // Panels of kPanel row tiles; within a panel, row tiles run fastest.
  auto decode = [&](long long t, int& m, int& n) {
    const long long per = (long long)kPanel * sh.tiles_n;
    const int p = (int)(t / per);
    const int rows = min(kPanel, tm - p * kPanel);
    const int r = (int)(t - p * per);
    m = p * kPanel + r % rows;
    n = r / rows;
  };

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      uint32_t it = 0;
      for (long long t = pair; ok && t < tiles; t += npairs) {
        int m, n;
        decode(t, m, n);
        const int half = KIND == kDw && m >= sh.tiles_m;
        if (half) m -= sh.tiles_m;
        const int row = m * kTile + (int)rank * 128;
        for (int k = 0; k < ksteps; ++k, ++it) {
          const int s = it % kStages;
          ok = mbar_wait(&empty[s], ((it / kStages) & 1) ^ 1);
          if (!ok) break;
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kStageBytes);
          const uint32_t bar = mapa_shared(smem_u32(&full[s]), 0);
          unsigned char* a = sm + s * kStageBytes;
          unsigned char* b = a + kOperand;
          const int second = KIND == kDx && k >= sh.kblocks;
          const int kk = (second ? k - sh.kblocks : k) * kBK;
          if (KIND == kDw) {
            // A(m, k) = dg[k, m], B(n, k) = x[k, n]: 64 x 64 blocks, MN-major
            const CUtensorMap* ma = &maps.a[half];
            const int col = n * kTile + (int)rank * 128;
            tma_load_2d_pair(a, ma, row, kk, bar);
            tma_load_2d_pair(a + 8192, ma, row + 64, kk, bar);
            tma_load_2d_pair(b, &maps.b[0], col, kk, bar);
            tma_load_2d_pair(b + 8192, &maps.b[0], col + 64, kk, bar);
          } else {
            tma_load_2d_pair(a, &maps.a[second], kk, row, bar);
            if (KIND == kFwd) {
              tma_load_2d_pair(b, &maps.b[rank], kk, n * 128, bar);
            } else {
              const int col = n * kTile + (int)rank * 128;
              tma_load_2d_pair(b, &maps.b[second], col, kk, bar);
              tma_load_2d_pair(b + 8192, &maps.b[second], col + 64, kk, bar);
            }
          }
        }
      }
      // every stage's last use has been read (its arrival is not left in flight)
      for (uint32_t i = 0; ok && i < (uint32_t)kStages && i < it; ++i) {
        const uint32_t last = it - 1 - i;
        ok = mbar_wait(&empty[last % kStages], (last / kStages) & 1);
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      constexpr uint32_t idesc =
          idesc_bf16(256, 256, KIND == kDw ? 1 : 0, KIND == kFwd ? 0 : 1);
      const uint32_t sbase = smem_u32(sm);
      bool ok = true;
      uint32_t it = 0, j = 0;
      for (long long t = pair; ok && t < tiles; t += npairs, ++j) {
        const uint32_t acc = tmem + (j & 1) * 256;
        ok = mbar_wait_cluster(&tempty[j & 1], ((j >> 1) & 1) ^ 1);
        tc_fence_after();
        for (int k = 0; ok && k < ksteps; ++k, ++it) {
          const int s = it % kStages;
          ok = mbar_wait_cluster(&full[s], (it / kStages) & 1);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = sbase + s * kStageBytes, b = a + kOperand;
#pragma unroll
          for (int q = 0; q < kBK / 16; ++q) {
            const uint64_t ad = KIND == kDw ? umma_desc(a + q * 2048, 8192, 1024, kSW128)
                                            : umma_desc(a + q * 32, 16, 1024, kSW128);
            const uint64_t bd = KIND == kFwd ? umma_desc(b + q * 32, 16, 1024, kSW128)
                                             : umma_desc(b + q * 2048, 8192, 1024, kSW128);
            mma_bf16_pair(acc, ad, bd, idesc, (k | q) != 0);
          }
          mma_commit_pair(&empty[s]);
        }
        if (ok) mma_commit_pair(&tfull[j & 1]);
      }
    }
  } else {
    // Epilogue: warp w reads TMEM lanes 32 (w % 4) .., columns of its half.
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const int row = quad * 32 + lane;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    unsigned char* box0 = sm + kOffStaging + half * 2 * kBox;
    const bool issuer = quad == 2 && lane == 0;   // first warp of the half
    const int bar_id = 1 + half;
    const uint32_t tempty0 = mapa_shared(smem_u32(tempty), 0);
    int nbuf = 0;
    // Staging buffer for the next box: its last store has been read.
    auto begin_box = [&]() {
      if (issuer) bulk_wait_read<1>();
      named_barrier(bar_id, 128);
      return box0 + (nbuf & 1) * kBox;
    };
    auto end_box = [&](const CUtensorMap* map, int c0, int c1, unsigned char* box) {
      fence_proxy_async_smem();
      named_barrier(bar_id, 128);
      if (issuer) {
        if (c0 < sh.cols && c1 < sh.rows) tma_store_2d(map, c0, c1, box);
        bulk_commit();
      }
      ++nbuf;
    };
    auto put = [&](unsigned char* box, int chunk, const float (&v)[32]) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint4 q;
        __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = __floats2bfloat162_rn(v[8 * c + 2 * e], v[8 * c + 2 * e + 1]);
        *reinterpret_cast<uint4*>(box + sw128(row, chunk + c)) = q;
      }
    };
    uint32_t j = 0;
    bool ok = true;
    for (long long t = pair; ok && t < tiles; t += npairs, ++j) {
      int m, n;
      decode(t, m, n);
      const int second = KIND == kDw && m >= sh.tiles_m;
      if (second) m -= sh.tiles_m;
      const int r0 = m * kTile + (int)rank * 128;
      // (agreed by the half's warps, so that none waits at a barrier for one that gave up)
      ok = named_barrier_and(bar_id, 128, mbar_wait(&tfull[j & 1], (j >> 1) & 1));
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + (j & 1) * 256 + lanes;
      auto release = [&]() {   // this warp has read its part of the accumulator
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tempty0 + (j & 1) * 8);
      };
      if (KIND == kFwd) {
        const int c0 = n * 128 + half * 64;
        unsigned char* box = begin_box();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float g[32], u[32];
          tmem_ld32(acc + half * 64 + c * 32, g);
          tmem_ld32(acc + 128 + half * 64 + c * 32, u);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            g[e] = g[e] * fast_sigmoid(g[e]) * u[e];
          put(box, c * 4, g);
        }
        if (!sh.keep) release();
        end_box(&maps.out[0], c0, r0, box);
        if (sh.keep) {
#pragma unroll 1
          for (int w = 0; w < 2; ++w) {   // g, then u
            box = begin_box();
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float v[32];
              tmem_ld32(acc + w * 128 + half * 64 + c * 32, v);
              put(box, c * 4, v);
            }
            if (w == 1) release();
            end_box(&maps.out[1 + w], c0, r0, box);
          }
        }
      } else {
#pragma unroll 1
        for (int w = 0; w < 2; ++w) {
          unsigned char* box = begin_box();
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float v[32];
            tmem_ld32(acc + half * 128 + w * 64 + c * 32, v);
            put(box, c * 4, v);
          }
          if (w == 1) release();
          end_box(&maps.out[second], n * kTile + half * 128 + w * 64, r0, box);
        }
      }
    }
    if (issuer) bulk_wait<0>();
  }
  tc_fence_before();
  // neither CTA leaves while the other may still reach its barriers or operands
  cluster_sync_all();
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// ---------------------------------------------------------------------------
// Few tokens: the weights are streamed once
// ---------------------------------------------------------------------------
//
// HBM-bound on Wg and Wu (46 MB at 2048 x 5632).  A CTA owns W output columns:
// W rows of Wg and the same W of Wu form B (2 W columns of the accumulator), the
// tokens are A's rows, of which only the ones in use are loaded (the others'
// products are never read).  Two CTAs share an SM and each keeps as many 64-wide
// stages in flight as half its shared memory holds.  The same tiles serve
// products too small to fill the GPU with 256 x 256 tiles.
constexpr int kNarrowThreads = 192;
constexpr int kNarrowMaxStages = 12;
constexpr int kNarrowSmem = 110 * 1024;

struct NarrowShape {
  int M, I, tiles_m, tiles_n, kblocks, rows_a, stages;
};
struct alignas(64) NarrowMaps {
  CUtensorMap x, wg, wu;
};

template <int W>
__global__ void __launch_bounds__(kNarrowThreads, 2)
glu_narrow_kernel(const __grid_constant__ NarrowMaps maps, const NarrowShape sh,
                  __nv_bfloat16* __restrict__ h, __nv_bfloat16* __restrict__ gk,
                  __nv_bfloat16* __restrict__ uk) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = smem_raw + (1024u - (smem_u32(smem_raw) & 1023u)) % 1024u;
  __shared__ __align__(8) uint64_t full[kNarrowMaxStages], empty[kNarrowMaxStages], tfull[2],
      tempty[2];
  __shared__ uint32_t tmem_slot;
  constexpr int kCols = 4 * W;                       // two accumulators of 2 W columns
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bytes_a = sh.rows_a * 128;               // rows of 128 bytes, 8 an atom
  constexpr int kBytesB = 2 * W * 128;
  const int stage_bytes = bytes_a + kBytesB;         // both multiples of 1024
  if (threadIdx.x == 0) {
    for (int i = 0; i < sh.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 4);
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const long long tiles = (long long)sh.tiles_m * sh.tiles_n;

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      uint32_t it = 0, s = 0, ph = 1;
      for (long long t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
        const int m = (int)(t % sh.tiles_m), n = (int)(t / sh.tiles_m);
        for (int k = 0; k < sh.kblocks; ++k, ++it) {
          ok = mbar_wait(&empty[s], ph);
          if (!ok) break;
          mbar_arrive_expect_tx(&full[s], (uint32_t)stage_bytes);
          unsigned char* b = sm + s * stage_bytes;
          tma_load_2d(b, &maps.wg, k * kBK, n * W, &full[s]);
          tma_load_2d(b + kBytesB / 2, &maps.wu, k * kBK, n * W, &full[s]);
          tma_load_2d(b + kBytesB, &maps.x, k * kBK, m * 128, &full[s]);
          if (++s == (uint32_t)sh.stages) { s = 0; ph ^= 1; }
        }
      }
      // the loads still in flight land before the CTA leaves
      for (int i = 0; ok && i < sh.stages && (uint32_t)i < it; ++i) {
        ok = mbar_wait(&empty[s], ph);
        if (++s == (uint32_t)sh.stages) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_bf16(128, 2 * W, 0, 0);
      const uint32_t sbase = smem_u32(sm);
      bool ok = true;
      uint32_t j = 0, s = 0, ph = 0;
      for (long long t = blockIdx.x; ok && t < tiles; t += gridDim.x, ++j) {
        const uint32_t acc = tmem + (j & 1) * 2 * W;
        ok = mbar_wait(&tempty[j & 1], ((j >> 1) & 1) ^ 1);
        tc_fence_after();
        for (int k = 0; ok && k < sh.kblocks; ++k) {
          ok = mbar_wait(&full[s], ph);
          if (!ok) break;
          tc_fence_after();
          const uint32_t b = sbase + s * stage_bytes, x = b + kBytesB;
#pragma unroll
          for (int q = 0; q < kBK / 16; ++q)
            mma_bf16(acc, umma_desc(x + q * 32, 16, 1024, kSW128),
                     umma_desc(b + q * 32, 16, 1024, kSW128), idesc, (k | q) != 0);
          mma_commit(&empty[s]);
          if (++s == (uint32_t)sh.stages) { s = 0; ph ^= 1; }
        }
        if (ok) mma_commit(&tfull[j & 1]);
      }
    }
  } else {
    const int quad = warp & 3;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    uint32_t j = 0;
    bool ok = true;
    for (long long t = blockIdx.x; ok && t < tiles; t += gridDim.x, ++j) {
      const int m = (int)(t % sh.tiles_m), n = (int)(t / sh.tiles_m);
      ok = mbar_wait(&tfull[j & 1], (j >> 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + (j & 1) * 2 * W + lanes;
      const long long row = (long long)m * 128 + quad * 32 + lane;
#pragma unroll
      for (int c = 0; c < W / 16; ++c) {
        float g[16], u[16];
        tmem_ld16x2(acc + c * 16, acc + W + c * 16, g, u);
        const int col = n * W + c * 16;
        if (row < sh.M) {
          auto put = [&](__nv_bfloat16* p, const float (&v)[16]) {
#pragma unroll
            for (int e = 0; e < 16; e += 8)
              if (col + e < sh.I) {   // I is a multiple of 8
                uint4 q;
                __nv_bfloat162* b2 = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  b2[i] = __floats2bfloat162_rn(v[e + 2 * i], v[e + 2 * i + 1]);
                *reinterpret_cast<uint4*>(p + row * sh.I + col + e) = q;
              }
          };
          if (gk) {
            put(gk, g);
            put(uk, u);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) g[e] = g[e] * fast_sigmoid(g[e]) * u[e];
          put(h, g);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[j & 1]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, kCols);
}

// [rows, cols] bf16 row-major, boxes of 64 columns x `box_rows`, 128-byte swizzle.
bool make_map(CUtensorMap* m, const void* base, long long rows, long long cols, int box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)cols * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <int KIND>
cudaError_t launch_kind(const GluMaps& maps, const GluShape& sh, cudaStream_t st) {
  static std::atomic<int> slot[kMaxDevices] = {};
  const cudaError_t e = ensure_smem(glu_tc_kernel<KIND>, kSmemBytes, slot);
  if (e != cudaSuccess) return e;
  const long long tiles = (long long)sh.tiles_m * sh.tiles_n * (KIND == kDw ? 2 : 1);
  const int pairs = device_sm_count() / 2;
  const int grid = 2 * (int)(tiles < pairs ? tiles : pairs);
  glu_tc_kernel<KIND><<<grid, kTcThreads, kSmemBytes, st>>>(maps, sh);
  return cudaGetLastError();
}

template <int W>
cudaError_t launch_narrow(const GluArgs& a, cudaStream_t st) {
  NarrowMaps m;
  NarrowShape sh;
  sh.M = a.M;
  sh.I = a.I;
  sh.tiles_m = ceil_div(a.M, 128);
  sh.tiles_n = ceil_div(a.I, W);
  sh.kblocks = ceil_div(a.D, kBK);
  sh.rows_a = a.M >= 128 ? 128 : ceil_div(a.M, 8) * 8;
  // The products read all 128 rows of A's tile from a stage's start of it (rows past
  // rows_a are whatever lies there): the last stage's end inside the allocation too.
  const int bytes_a = sh.rows_a * 128;
  sh.stages = (kNarrowSmem - 1024 - 128 * 128 + bytes_a) / (bytes_a + 2 * W * 128);
  if (sh.stages > kNarrowMaxStages) sh.stages = kNarrowMaxStages;
  if (!make_map(&m.x, a.x, a.M, a.D, sh.rows_a) || !make_map(&m.wg, a.wg, a.I, a.D, W) ||
      !make_map(&m.wu, a.wu, a.I, a.D, W))
    return cudaErrorInvalidValue;
  static std::atomic<int> slot[kMaxDevices] = {};
  const cudaError_t e = ensure_smem(glu_narrow_kernel<W>, kNarrowSmem, slot);
  if (e != cudaSuccess) return e;
  const long long tiles = (long long)sh.tiles_m * sh.tiles_n, most = 2LL * device_sm_count();
  glu_narrow_kernel<W><<<(unsigned)(tiles < most ? tiles : most), kNarrowThreads, kNarrowSmem,
                         st>>>(m, sh, static_cast<__nv_bfloat16*>(a.h),
                               static_cast<__nv_bfloat16*>(a.g), static_cast<__nv_bfloat16*>(a.u));
  return cudaGetLastError();
}

}  // namespace

GDN_DEVICE_ERROR_ACCESSOR(device_error_glu_tc)

bool glu_tc_supported(int M, int D, int I, int dtype) {
  return dtype == kBF16 && M > 0 && D > 0 && I > 0 && D % 8 == 0 && I % 8 == 0 &&
         encode_fn() != nullptr;
}

cudaError_t launch_glu_tc_fwd(const GluArgs& a, cudaStream_t st) {
#ifndef NARROW_M
#define NARROW_M 128
#endif
#ifndef NARROW_W
#define NARROW_W 0
#endif
  if (a.M <= NARROW_M) {
    const int w = NARROW_W ? NARROW_W : a.I > 296 * 32 ? 64 : a.I > 296 * 16 ? 32 : 16;
    if (w == 64) return launch_narrow<64>(a, st);
    return w == 32 ? launch_narrow<32>(a, st) : launch_narrow<16>(a, st);
  }
  GluMaps m;
  if (!make_map(&m.a[0], a.x, a.M, a.D, 128) || !make_map(&m.b[0], a.wg, a.I, a.D, 128) ||
      !make_map(&m.b[1], a.wu, a.I, a.D, 128) || !make_map(&m.out[0], a.h, a.M, a.I, 128) ||
      (a.g && (!make_map(&m.out[1], a.g, a.M, a.I, 128) ||
               !make_map(&m.out[2], a.u, a.M, a.I, 128))))
    return cudaErrorInvalidValue;
  m.a[1] = m.a[0];
  if (!a.g) m.out[1] = m.out[2] = m.out[0];
  const GluShape sh{ceil_div(a.M, kTile), ceil_div(a.I, 128), ceil_div(a.D, kBK),
                    a.g != nullptr, a.M, a.I};
  return launch_kind<kFwd>(m, sh, st);
}

cudaError_t launch_glu_tc_bwd(const GluBwdArgs& a, cudaStream_t st) {
  GluMaps m;
  if (a.dx) {
    if (!make_map(&m.a[0], a.dg, a.M, a.I, 128) || !make_map(&m.a[1], a.du, a.M, a.I, 128) ||
        !make_map(&m.b[0], a.wg, a.I, a.D, 64) || !make_map(&m.b[1], a.wu, a.I, a.D, 64) ||
        !make_map(&m.out[0], a.dx, a.M, a.D, 128))
      return cudaErrorInvalidValue;
    m.out[1] = m.out[2] = m.out[0];
    const GluShape sh{ceil_div(a.M, kTile), ceil_div(a.D, kTile), ceil_div(a.I, kBK), 0,
                      a.M, a.D};
    const cudaError_t e = launch_kind<kDx>(m, sh, st);
    if (e != cudaSuccess) return e;
  }
  if (a.dwg) {
    if (!make_map(&m.a[0], a.dg, a.M, a.I, 64) || !make_map(&m.a[1], a.du, a.M, a.I, 64) ||
        !make_map(&m.b[0], a.x, a.M, a.D, 64) || !make_map(&m.out[0], a.dwg, a.I, a.D, 128) ||
        !make_map(&m.out[1], a.dwu, a.I, a.D, 128))
      return cudaErrorInvalidValue;
    m.b[1] = m.b[0];
    m.out[2] = m.out[1];
    const GluShape sh{ceil_div(a.I, kTile), ceil_div(a.D, kTile), ceil_div(a.M, kBK), 0,
                      a.I, a.D};
    return launch_kind<kDw>(m, sh, st);
  }
  return cudaSuccess;
}

}  // namespace gdn
