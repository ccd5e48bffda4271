// latent_decode_args.h - arguments of the latent decode kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace pcamd {
namespace decode {

struct Args {
  const void* q_latent; const void* q_rope;
  int64_t qlb, qls, qlh, qrb, qrs, qrh;
  const void* latent; const void* rope; const float* scale;
  uint32_t slp, slt, srp, srt, ssp, sst;
  const int32_t* table; int64_t table_stride; const int32_t* lens;
  void* out; int64_t ob, os, oh;
  float* lse; int64_t lb, ls, lh;
  uint32_t pages, page_mul;
  int batch, new_tokens, heads, rows, row_tiles, page, page_shift, capacity;
  float scale_log2;
  // the division of the work, and where its pieces meet
  int groups, min_steps;
  int4* joins; float* parts; float2* part_ml;

  // place in the page table of the page that holds token t, t / page: with l =
  // ceil(log2 page) = page_shift and page_mul = ceil(2^(31 + l) / page), exact
  // for every t below 2^31
  __device__ __forceinline__ int page_index(int t) const {
    return static_cast<int>(__umulhi(2u * static_cast<uint32_t>(t), page_mul) >> page_shift);
  }
};

// What a piece costs whatever its length (queries in, output out, latencies),
// in steps of its kernel
template <int MR>
constexpr int kFixed = MR == 32 ? 10 : 2;

// Rows of a tile and tokens of a step for `rows` rows a sequence: up to 16 (32,
// 64) rows fill one (two, four) waves of 16 rows, and the other waves of a
// workgroup take other tokens; above that, four waves of 32 rows.
struct Shape {
  int mr, wr;
  int tile_rows() const { return mr * wr; }
  int step() const { return 32 * (4 / wr); }
};
inline Shape shape_for(int64_t rows) {
  if (rows <= 16) return {16, 1};
  if (rows <= 32) return {16, 2};
  if (rows <= 64) return {16, 4};
  return {32, 4};
}

// launches decode_kernel and, where a.parts is set, combine_kernel
template <int DT, int DL, int DR>
int launch(const Args& a, Shape shape, bool fp8, hipStream_t st);

// fp16 weights times an fp8 cache's scales (a 448th of its group's maximum)
// would reach the subnormal numbers; bf16 has fp32's range
template <int DT>
constexpr float kScaleUp = DT == 2 /* PCAMD_F16 */ ? 256.0f : 1.0f;

}  // namespace decode
}  // namespace pcamd
