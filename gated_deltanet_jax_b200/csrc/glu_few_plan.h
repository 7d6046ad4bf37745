// How the gated linear unit's kernel for few tokens (glu_tc.cu) is laid out: host
// arithmetic alone, so that it can be checked for every size without a GPU.
#pragma once

namespace gdn {

constexpr int kFewRows = 64;                         // output columns of a cluster
constexpr int kFewTokens = 128;                      // the most this form takes
constexpr int kFewBK = 64;                           // of the contraction, a step
constexpr int kFewA = 2 * kFewRows * 128;            // bytes of a stage's weights
constexpr int kFewMaxStages = 11;
constexpr int kFewMaxSplit = 8;
constexpr int kFewMaxShare = 2;                      // CTAs of an SM
constexpr int kFewAlign = 1024;                      // bytes lost to the stages' alignment

struct FewPlan {
  int tiles;     // clusters
  int split;     // CTAs of a cluster, the contraction's parts
  int kblocks;   // steps of the contraction
  int n;         // tokens rounded up to 16: rows of a stage's x
  int cols;      // of TMEM
  int share;     // tokens a CTA finishes (a multiple of 4)
  int stages;
  int smem;      // dynamic shared memory, bytes

  int stage_bytes() const { return kFewA + n * 128; }
  int exchange_bytes() const { return split * share * 512; }
  // the stages and, over their memory afterwards, the exchange end inside the allocation
  bool fits() const {
    return stages >= 1 && kFewAlign + stages * stage_bytes() <= smem &&
           kFewAlign + exchange_bytes() <= smem;
  }
};

inline FewPlan few_plan(int M, int D, int I, int sms) {
  auto ceil_div = [](int a, int b) { return (a + b - 1) / b; };
  FewPlan p;
  p.tiles = ceil_div(I, kFewRows);
  p.kblocks = ceil_div(D, kFewBK);
  p.n = ceil_div(M, 16) * 16;
  p.cols = p.n <= 32 ? 32 : p.n <= 64 ? 64 : 128;
  // The split whose busiest SM has the least work (tiles / S each), the smallest
  // such, with at most two CTAs sharing an SM and four steps left to each (the
  // exchange costs 1 to 2 us).
  p.split = 1;
  double best = ceil_div(p.tiles, sms);
  for (int S = 2; S <= kFewMaxSplit && 4 * S <= p.kblocks; ++S) {
    const long long c = ((long long)p.tiles * S + sms - 1) / sms;
    if (c <= kFewMaxShare && (double)c / S < 0.95 * best) {
      best = (double)c / S;
      p.split = S;
    }
  }
  p.smem = ((long long)p.tiles * p.split <= sms ? 226 : 112) * 1024;   // and 1 KB static
  p.share = ceil_div(ceil_div(M, p.split), 4) * 4;
  p.stages = (p.smem - kFewAlign) / p.stage_bytes();
  if (p.stages > kFewMaxStages) p.stages = kFewMaxStages;
  return p;
}

}  // namespace gdn
