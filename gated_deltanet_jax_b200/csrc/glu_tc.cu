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
// clip ragged edges (loads fill them with zeros).  16384 tokens of 2048 x 5632:
// 478 us in short runs, 1582 TFLOP/s (0.96 of the measured bf16 rate), 0.54 to 0.56
// ms back to back under the power cap; 8200 tokens: 280 us storing g and u in fp32 too
// (257 in bf16), dx 260 and both weights' gradients 244 us (tensor pipe 95 % busy).
//
// Roundings: accumulators are fp32.  dg, du are rounded to bf16 as the backward's
// operands, by at most 2^-8 of the value, which takes a gradient's error in the norm from
// 1.7e-3 (its own rounding) to 2.4e-3.  g and u are kept in fp32 for it: in bf16 they
// would halve what a training step keeps of them, and their roundings would make it 3.1e-3
// (a caller of the library may ask for that).
#include <algorithm>

#include "gdn_common.cuh"
#include "gdn_internal.h"
#include "glu_few_plan.h"
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
  int keep;               // kFwd: g and u are stored (1: bf16, 2: fp32)
  int rows, cols;         // of the output
  // kDx, kDw: the contraction's parts and their steps.  With more than one, part p's sums
  // leave in fp32 for rows 256 tiles_m p .. (kDw: 512 tiles_m p, dWg's before dWu's) of out[2].
  int parts = 1, part_steps = 0;
};

// The most 64-wide steps that one accumulator takes.  A sum in TMEM does not round to
// nearest: over terms of one sign it came out too small by 0.7e-4 after 16384 of them, 3.5e-4
// after 65536, 1.6e-3 after 262144 and 2.6 % after 4 million.  Longer contractions are cut into
// parts of 32768 terms, added up in fp32: at 2048 x 5632 the weights' gradients of 65536 tokens
// then write and read 0.37 GB more beside 2 ms of products.
constexpr int kMaxSteps = 512;

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
  const long long items = KIND == kFwd ? tiles : tiles * sh.parts;
  const int ksteps = KIND == kDx ? 2 * sh.kblocks : sh.kblocks;
  // Panels of kPanel row tiles; within a panel, row tiles run fastest.
  // k0 .. k1: the item's steps.
  auto decode = [&](long long t, int& m, int& n, int& part, int& k0, int& k1) {
    part = 0;
    k0 = 0;
    k1 = ksteps;
    if (KIND != kFwd) {
      part = (int)(t / tiles);
      t -= part * tiles;
      k0 = part * sh.part_steps;
      k1 = min(ksteps, k0 + sh.part_steps);
    }
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
      for (long long t = pair; ok && t < items; t += npairs) {
        int m, n, part, k0, k1;
        decode(t, m, n, part, k0, k1);
        const int half = KIND == kDw && m >= sh.tiles_m;
        if (half) m -= sh.tiles_m;
        const int row = m * kTile + (int)rank * 128;
        for (int k = k0; k < k1; ++k, ++it) {
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
      for (long long t = pair; ok && t < items; t += npairs, ++j) {
        const uint32_t acc = tmem + (j & 1) * 256;
        int m, n, part, k0, k1;
        decode(t, m, n, part, k0, k1);
        ok = mbar_wait_cluster(&tempty[j & 1], ((j >> 1) & 1) ^ 1);
        tc_fence_after();
        for (int k = k0; ok && k < k1; ++k, ++it) {
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
            mma_bf16_pair(acc, ad, bd, idesc, k > k0 || q != 0);
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
    auto put_fp32 = [&](unsigned char* box, const float (&v)[32]) {
#pragma unroll
      for (int c = 0; c < 8; ++c)
        *reinterpret_cast<float4*>(box + sw128(row, c)) =
            make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
    };
    uint32_t j = 0;
    bool ok = true;
    for (long long t = pair; ok && t < items; t += npairs, ++j) {
      int m, n, part, k0, k1;
      decode(t, m, n, part, k0, k1);
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
        if (sh.keep == 2) {
#pragma unroll 1
          for (int w = 0; w < 4; ++w) {   // g, then u, 32 columns a box
            box = begin_box();
            float v[32];
            tmem_ld32(acc + (w >> 1) * 128 + half * 64 + (w & 1) * 32, v);
            put_fp32(box, v);
            if (w == 3) release();
            end_box(&maps.out[1 + (w >> 1)], c0 + (w & 1) * 32, r0, box);
          }
        } else if (sh.keep) {
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
      } else if (sh.parts > 1) {
#pragma unroll 1
        for (int w = 0; w < 4; ++w) {
          unsigned char* box = begin_box();
          float v[32];
          tmem_ld32(acc + half * 128 + w * 32, v);
          put_fp32(box, v);
          if (w == 3) release();
          end_box(&maps.out[2], n * kTile + half * 128 + w * 32,
                  (KIND == kDw ? 2 * part + second : part) * sh.tiles_m * kTile + r0, box);
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
// HBM-bound on Wg and Wu (46 MB at 2048 x 5632).  The operands change places: 64
// rows of Wg and the same 64 of Wu are the 128 rows of A, the tokens (rounded up
// to 16) the columns.  A product of 128 rows takes about 150 clocks however few its
// columns are, so an SM takes in 27 bytes of weights a clock at most, and only all
// SMs together keep up with HBM: the contraction is cut over a cluster of S CTAs,
// S chosen so that tiles x S spread evenly (88 tiles at 5632 columns: S = 3, two
// CTAs an SM; on 88 SMs alone the same work took 15 us).  Each CTA of the cluster
// then sums the S partial accumulators of its share of the tokens, sent through
// distributed shared memory in a fixed order, and writes their silu(g) u.
constexpr int kFewThreads = 192;
static_assert(kFewBK == kBK, "the operands' boxes are shared");

struct FewShape {
  int M, I, kblocks, n, stages, cols, split;   // n: tokens rounded up to 16
  int share;                                   // tokens a CTA finishes (a multiple of 4)
  bool keep32;                                 // g and u are kept in fp32
};
struct alignas(64) FewMaps {
  CUtensorMap x, wg, wu;
};

__global__ void __launch_bounds__(kFewThreads)
glu_few_kernel(const __grid_constant__ FewMaps maps, const FewShape sh,
               __nv_bfloat16* __restrict__ h, void* __restrict__ gk, void* __restrict__ uk) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = smem_raw + (1024u - (smem_u32(smem_raw) & 1023u)) % 1024u;
  __shared__ __align__(8) uint64_t full[kFewMaxStages], empty[kFewMaxStages], done;
  __shared__ uint32_t tmem_slot;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stage_bytes = kFewA + sh.n * 128;        // a multiple of 1024
  const int rank = sh.split > 1 ? (int)cluster_ctarank() : 0;
  const int tile = blockIdx.x / sh.split;
  const int k0 = rank * sh.kblocks / sh.split, k1 = (rank + 1) * sh.kblocks / sh.split;
  if (threadIdx.x == 0) {
    for (int i = 0; i < sh.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&done, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, sh.cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // The set-up above overlaps the launch before this one on its stream; nothing in
  // global memory is touched before that has completed.
  griddep_wait();
  if (threadIdx.x == 0) griddep_launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      uint32_t s = 0, ph = 1;
      for (int k = k0; k < k1; ++k) {
        if (!mbar_wait(&empty[s], ph)) break;
        mbar_arrive_expect_tx(&full[s], (uint32_t)stage_bytes);
        unsigned char* a = sm + s * stage_bytes;
        tma_load_2d(a, &maps.wg, k * kBK, tile * kFewRows, &full[s]);
        tma_load_2d(a + kFewA / 2, &maps.wu, k * kBK, tile * kFewRows, &full[s]);
        tma_load_2d(a + kFewA, &maps.x, k * kBK, 0, &full[s]);
        if (++s == (uint32_t)sh.stages) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_bf16(128, sh.n, 0, 0);
      const uint32_t sbase = smem_u32(sm);
      uint32_t s = 0, ph = 0;
      bool ok = true;
      for (int k = k0; k < k1; ++k) {
        ok = mbar_wait(&full[s], ph);
        if (!ok) break;
        tc_fence_after();
        const uint32_t a = sbase + s * stage_bytes, b = a + kFewA;
#pragma unroll
        for (int q = 0; q < kBK / 16; ++q)
          mma_bf16(tmem, umma_desc(a + q * 32, 16, 1024, kSW128),
                   umma_desc(b + q * 32, 16, 1024, kSW128), idesc, (k > k0) || q != 0);
        mma_commit(&empty[s]);
        if (++s == (uint32_t)sh.stages) { s = 0; ph ^= 1; }
      }
      if (ok) mma_commit(&done);
    }
  }
  // The accumulator is complete: every load has landed and been read (a wait that
  // gives up is recorded, and its results are invalid; the barriers below are met
  // by every thread either way).
  mbar_wait(&done, 0);
  __syncwarp();
  tc_fence_after();
  if (sh.split > 1) cluster_sync_all();
  else __syncthreads();
  // part [source][four tokens of my share][128 rows], over the stages' memory: a warp's
  // lanes write and read 512 bytes in a row
  float4* part = reinterpret_cast<float4*>(sm);
  const int quads = sh.share / 4;
  if (warp >= 2) {
    const int quad = warp & 3;
    const uint32_t mine = smem_u32(part + rank * quads * 128 + quad * 32 + lane);
    int to = 0, tl = 0;                   // tokens c ..: CTA `to`, its tokens tl ..
    uint32_t dst = sh.split > 1 ? mapa_shared(mine, 0) : mine;
    for (int c = 0; c < sh.n; c += 16) {
      float v[16];
      tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + c, v);
#pragma unroll
      for (int e = 0; e < 16; e += 4) {   // a share is a multiple of four tokens
        if (c + e < sh.M)
          st_cluster_f32x4(dst + tl * 512, v[e], v[e + 1], v[e + 2], v[e + 3]);
        tl += 4;
        if (tl >= sh.share && to + 1 < sh.split) {
          tl = 0;
          dst = mapa_shared(mine, (uint32_t)++to);
        }
      }
    }
    tc_fence_before();
  }
  __syncwarp();
  if (sh.split > 1) cluster_sync_all();
  else __syncthreads();
  // four tokens of one column a thread
  const int first = rank * sh.share, mine = min(sh.share, sh.M - first);
  for (int i = threadIdx.x; i < (mine + 3) / 4 * kFewRows; i += kFewThreads) {
    const int tl = i / kFewRows * 4, r = i % kFewRows, col = tile * kFewRows + r;
    if (col >= sh.I) continue;
    float4 g = make_float4(0.f, 0.f, 0.f, 0.f), u = g;
    for (int s = 0; s < sh.split; ++s) {
      const float4* p = part + (s * quads + tl / 4) * 128 + r;
      const float4 a = p[0], b = p[kFewRows];
      g.x += a.x; g.y += a.y; g.z += a.z; g.w += a.w;
      u.x += b.x; u.y += b.y; u.z += b.z; u.w += b.w;
    }
    const float gv[4] = {g.x, g.y, g.z, g.w}, uv[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (tl + e >= mine) break;
      const size_t o = (size_t)(first + tl + e) * sh.I + col;
      h[o] = __float2bfloat16_rn(gv[e] * fast_sigmoid(gv[e]) * uv[e]);
      if (gk && sh.keep32) {
        static_cast<float*>(gk)[o] = gv[e];
        static_cast<float*>(uk)[o] = uv[e];
      } else if (gk) {
        static_cast<__nv_bfloat16*>(gk)[o] = __float2bfloat16_rn(gv[e]);
        static_cast<__nv_bfloat16*>(uk)[o] = __float2bfloat16_rn(uv[e]);
      }
    }
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, sh.cols);
  }
}

// [rows, cols] bf16 row-major, boxes of 64 columns x `box_rows` (fp32: of 32 columns),
// 128-byte swizzle.
bool make_map(CUtensorMap* m, const void* base, long long rows, long long cols, int box_rows,
              bool fp32 = false) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)cols * (fp32 ? 4 : 2)};
  cuuint32_t box[2] = {fp32 ? 32u : 64u, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(m, fp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
            const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <int KIND>
cudaError_t launch_kind(const GluMaps& maps, const GluShape& sh, cudaStream_t st) {
  static std::atomic<int> slot[kMaxDevices] = {};
  const cudaError_t e = ensure_smem(glu_tc_kernel<KIND>, kSmemBytes, slot);
  if (e != cudaSuccess) return e;
  const long long tiles = (long long)sh.tiles_m * sh.tiles_n * sh.parts * (KIND == kDw ? 2 : 1);
  const int pairs = device_sm_count() / 2;
  const int grid = 2 * (int)(tiles < pairs ? tiles : pairs);
  glu_tc_kernel<KIND><<<grid, kTcThreads, kSmemBytes, st>>>(maps, sh);
  return cudaGetLastError();
}

// The parts added up in their order: n vectors of four, `stride` of them a part.
__global__ void __launch_bounds__(256)
glu_part_sum_kernel(const float* __restrict__ part, int parts, long long n, long long stride,
                    __nv_bfloat16* __restrict__ out) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float4 s = load4(part + 4 * i);
#pragma unroll 4
  for (int p = 1; p < parts; ++p) {
    const float4 v = load4(part + 4 * (p * stride + i));
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  store4(out + 4 * i, s);
}

cudaError_t sum_parts(const float* part, int parts, long long n, long long stride, void* out,
                      cudaStream_t st) {
  glu_part_sum_kernel<<<(unsigned)((n / 4 + 255) / 256), 256, 0, st>>>(
      part, parts, n / 4, stride / 4, static_cast<__nv_bfloat16*>(out));
  return cudaGetLastError();
}

// Parts of dx's contraction: of kMaxSteps at most, and where its output tiles are at most
// half the pairs of SMs (a tile walks 2 I / 64 steps alone) up to 16 of 8 steps or more.  The
// whole backward of 2048 x 5632: 16 tokens 74 -> 40 us, 256 81 -> 46, 1000 105 -> 88.
int tc_dx_parts(int M, int D, int I, int* steps) {
  const int ksteps = 2 * ceil_div(I, kBK), pairs = device_sm_count() / 2;
  const long long tiles = (long long)ceil_div(M, kTile) * ceil_div(D, kTile);
  int parts = ceil_div(ksteps, kMaxSteps);
  if (tiles > 0 && 2 * tiles <= pairs)
    parts = std::max(parts, (int)std::min({pairs / tiles, 16LL, ksteps / 8LL}));
  *steps = parts > 1 ? ceil_div(ksteps, parts) : ksteps;
  return parts > 1 ? ceil_div(ksteps, *steps) : 1;
}

// Parts of the weights' gradients' contraction over M tokens.
int tc_dw_parts(int M, int* steps) {
  const int ksteps = ceil_div(M, kBK), parts = ceil_div(ksteps, kMaxSteps);
  *steps = parts > 1 ? ceil_div(ksteps, parts) : ksteps;
  return parts > 1 ? ceil_div(ksteps, *steps) : 1;
}

cudaError_t launch_few(const GluArgs& a, cudaStream_t st) {
  FewMaps m;
  const FewPlan p = few_plan(a.M, a.D, a.I, device_sm_count());
  if (!p.fits()) return cudaErrorInvalidValue;
  const FewShape sh{a.M, a.I, p.kblocks, p.n, p.stages, p.cols, p.split, p.share,
                    a.kept == kFP32};
  // (a box of n rows past the M there are is filled with zeros)
  if (!make_map(&m.x, a.x, a.M, a.D, sh.n) || !make_map(&m.wg, a.wg, a.I, a.D, kFewRows) ||
      !make_map(&m.wu, a.wu, a.I, a.D, kFewRows))
    return cudaErrorInvalidValue;
  static std::atomic<int> slot[kMaxDevices] = {};
  const cudaError_t e = ensure_smem(glu_few_kernel, 226 * 1024, slot);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.tiles * p.split);
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = kernel_overrides().decode_pdl ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = sh.split;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = sh.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, glu_few_kernel, m, sh, static_cast<__nv_bfloat16*>(a.h), a.g,
                            a.u);
}

}  // namespace

GDN_DEVICE_ERROR_ACCESSOR(device_error_glu_tc)

// The forward's contraction is not cut (its sums never reach HBM), so D ends where an
// accumulator would take 2048 steps (0.7e-3 short at most, by the figures at kMaxSteps);
// wider inputs run on the CUDA cores, whose sums round to nearest.
bool glu_tc_widths(int D, int I, int dtype) {
  return dtype == kBF16 && D % 8 == 0 && I % 8 == 0 && D <= 4 * kMaxSteps * kBK;
}

bool glu_tc_supported(int M, int D, int I, int dtype) {
  return M > 0 && D > 0 && I > 0 && glu_tc_widths(D, I, dtype) && encode_fn() != nullptr;
}

cudaError_t launch_glu_tc_fwd(const GluArgs& a, cudaStream_t st) {
  // 37 / 64 / 128 tokens of 2048 x 5632: 12.7 / 13.0 / 16.6 us against 17.0 / 17.0 / 17.5
  if (a.M <= kFewTokens) return launch_few(a, st);
  GluMaps m;
  if (!make_map(&m.a[0], a.x, a.M, a.D, 128) || !make_map(&m.b[0], a.wg, a.I, a.D, 128) ||
      !make_map(&m.b[1], a.wu, a.I, a.D, 128) || !make_map(&m.out[0], a.h, a.M, a.I, 128) ||
      (a.g && (!make_map(&m.out[1], a.g, a.M, a.I, 128, a.kept == kFP32) ||
               !make_map(&m.out[2], a.u, a.M, a.I, 128, a.kept == kFP32))))
    return cudaErrorInvalidValue;
  m.a[1] = m.a[0];
  if (!a.g) m.out[1] = m.out[2] = m.out[0];
  const GluShape sh{ceil_div(a.M, kTile), ceil_div(a.I, 128), ceil_div(a.D, kBK),
                    a.g == nullptr ? 0 : a.kept == kFP32 ? 2 : 1, a.M, a.I};
  return launch_kind<kFwd>(m, sh, st);
}

size_t glu_tc_part_floats(int M, int D, int I) {
  int steps;
  const int dx = tc_dx_parts(M, D, I, &steps), dw = tc_dw_parts(M, &steps);
  return std::max(dx > 1 ? (size_t)dx * ceil_div(M, kTile) * kTile * D : 0,
                  dw > 1 ? (size_t)dw * 2 * ceil_div(I, kTile) * kTile * D : 0);
}

cudaError_t launch_glu_tc_bwd(const GluBwdArgs& a, cudaStream_t st) {
  GluMaps m;
  if (a.dx) {
    if (!make_map(&m.a[0], a.dg, a.M, a.I, 128) || !make_map(&m.a[1], a.du, a.M, a.I, 128) ||
        !make_map(&m.b[0], a.wg, a.I, a.D, 64) || !make_map(&m.b[1], a.wu, a.I, a.D, 64) ||
        !make_map(&m.out[0], a.dx, a.M, a.D, 128))
      return cudaErrorInvalidValue;
    m.out[1] = m.out[2] = m.out[0];
    GluShape sh{ceil_div(a.M, kTile), ceil_div(a.D, kTile), ceil_div(a.I, kBK), 0, a.M, a.D};
    sh.parts = tc_dx_parts(a.M, a.D, a.I, &sh.part_steps);
    const int padded = sh.tiles_m * kTile;   // rows of a part
    if (sh.parts > 1) {
      sh.rows = sh.parts * padded;
      if (!make_map(&m.out[2], a.part, sh.rows, a.D, 128, true)) return cudaErrorInvalidValue;
    }
    cudaError_t e = launch_kind<kDx>(m, sh, st);
    if (e == cudaSuccess && sh.parts > 1)
      e = sum_parts(a.part, sh.parts, (long long)a.M * a.D, (long long)padded * a.D, a.dx, st);
    if (e != cudaSuccess) return e;
  }
  if (a.dwg) {
    if (!make_map(&m.a[0], a.dg, a.M, a.I, 64) || !make_map(&m.a[1], a.du, a.M, a.I, 64) ||
        !make_map(&m.b[0], a.x, a.M, a.D, 64) || !make_map(&m.out[0], a.dwg, a.I, a.D, 128) ||
        !make_map(&m.out[1], a.dwu, a.I, a.D, 128))
      return cudaErrorInvalidValue;
    m.b[1] = m.b[0];
    m.out[2] = m.out[1];
    GluShape sh{ceil_div(a.I, kTile), ceil_div(a.D, kTile), ceil_div(a.M, kBK), 0, a.I, a.D};
    sh.parts = tc_dw_parts(a.M, &sh.part_steps);
    const long long seg = (long long)sh.tiles_m * kTile * a.D;   // a part's dWg, or its dWu
    if (sh.parts > 1) {
      sh.rows = sh.parts * 2 * sh.tiles_m * kTile;
      if (!make_map(&m.out[2], a.part, sh.rows, a.D, 128, true)) return cudaErrorInvalidValue;
    }
    cudaError_t e = launch_kind<kDw>(m, sh, st);
    const long long n = (long long)a.I * a.D;
    if (e == cudaSuccess && sh.parts > 1)
      e = sum_parts(a.part, sh.parts, n, 2 * seg, a.dwg, st);
    if (e == cudaSuccess && sh.parts > 1)
      e = sum_parts(a.part + seg, sh.parts, n, 2 * seg, a.dwu, st);
    return e;
  }
  return cudaSuccess;
}

}  // namespace gdn
