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

constexpr int kWorkgroups = 256;  // one (four waves, most of the LDS) a CU

// What a piece costs whatever its length (queries in, output out, latencies),
// in steps of its kernel. With two workgroups a tile: 8 takes 72.4 us for 48
// sequences of up to 5003 tokens and 128 rows and 92.2 for 19 of up to 6007 and
// 384 rows in fp8; 4 takes 84.8 and 100.5, 10 takes 74.9 and 93.8. Waves of 16
// rows: 3 takes 52.2 and 33.7 us for 48 sequences of 4000 tokens and 16 rows and
// of 1000 and 64; 1 takes 53.9 and 37.2.
template <int MR, int SPLIT>
constexpr int kFixed = MR == 32 ? (SPLIT == 2 ? 8 : 10) : 3;

// Rows of a tile and tokens of a step. Up to 16 (32, 64) rows a sequence fill
// one (two, four) waves of 16 rows, and the other waves of a workgroup take
// other tokens. Above that a tile has 128 rows, in waves of 32, as four waves
// of one workgroup or as two workgroups side by side on the same tokens, each
// with two waves on its 64 rows and two on other tokens of them. Two halve what
// a piece reads of queries and writes of partial sums, but copy the cache twice
// to LDS (the second time from the XCD's L2) and cannot overlap a tile's
// softmax with the next one's scores: they win where sequences are cut into
// pieces, up to half as many tiles as CUs. 128 heads over a bf16 cache, us, two
// workgroups against one: 16 sequences of 4096 tokens 47 / 66, 48 of 2048 65 /
// 71, 128 of 1024 and of 4096 63 / 80 and 185 / 182, 160 of 1024 and of 4096 94 /
// 98 and 249 / 233, 256 of 300 and of 2048 64 / 50 and 200 / 168. fp8: 16 of 4096
// 55 / 66, 48 of 2048 67 / 67, 128 of 1024 and of 4096 65 / 80 and 193 / 199, 160
// of 1024 100 / 96, 256 of 300 70 / 49.
struct Shape {
  int mr, wr, split;  // rows of a wave, waves over rows, workgroups over rows
  int tile_rows() const { return mr * wr * split; }
  int step() const { return 32 * (4 / wr); }
};
inline Shape shape_for(int64_t batch, int64_t rows) {
  if (rows <= 16) return {16, 1, 1};
  if (rows <= 32) return {16, 2, 1};
  if (rows <= 64) return {16, 4, 1};
  return batch * ((rows + 127) / 128) <= kWorkgroups / 2 ? Shape{32, 2, 2} : Shape{32, 4, 1};
}

// Whether each row tile is cut by itself: a workgroup then never has parts of
// two (it would work on them one after the other), and at most an eighth of the
// workgroups is lost to tiles that do not divide evenly.
__host__ __device__ inline bool few_tiles(int64_t tiles, int split) { return tiles * 8 <= kWorkgroups / split; }

// launches decode_kernel and, where a.parts is set, combine_kernel
template <int DT, int DL, int DR>
int launch(const Args& a, Shape shape, bool fp8, hipStream_t st);

}  // namespace decode
}  // namespace pcamd
