// int8_bmm.h - what the kernels of the int8 product share.
//
//   C[row, col] = act(float(sum_k A[row, k] B[col, k]) * (sa[row] * sb[col]) + bias[row, col])
//
// with the sum in int32, exact for k up to 131071 (128 * 128 * 131071 < 2^31),
// and one rounding to C's type. With the gated activation B holds 2 n rows, n
// gates and then n others, and C = silu(gate) * other.
//
// Plain: a batch of matrices. Grouped: rows starts[e] .. starts[e + 1] - 1 of C
// go with matrix e; row s of A is s itself, or with `choices` the row
// order[s] / choices (the token of pair order[s]); rows behind the last group
// are written as zeros.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "abi_util.h"
#include "fp8_common.h"

namespace pcamd {
namespace int8 {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int64_t kMaxK = 131071;

struct Args {
  const int8_t* a;
  const int8_t* b;
  void* c;
  const void* bias;
  const float* sa;
  const float* sb;
  int64_t sab, lda, sbb, ldb;        // bytes from matrix to matrix, from row to row
  int64_t scb, scm;                  // elements, as those below
  int64_t sbiasb, sbiasm, sbiasn;
  int64_t ssab, ssam, ssbb, ssbn;
  int32_t m, n, k, batch;            // n: columns of C
  int32_t c_dtype, bias_dtype, act;
  // grouped
  const int32_t* starts;
  const int32_t* order;              // null: rows of A are in C's order
  int32_t pairs, choices, a_rows;
};

// Rows of C that a workgroup computes: [row, end) of matrix `mat`; rows of none are zeros.
struct Rows {
  int32_t mat, row, end;
  bool zeros;
};

PCAMD_DEV int32_t start_at(const Args& a, int e) { return min(max(a.starts[e], 0), a.pairs); }

// Tile `q` of the grouped rows cut into tiles of `height`: a wave's lanes take 64 groups at a time and count their
// tiles; all waves of a workgroup find the same one. false: there are fewer tiles.
PCAMD_DEV bool grouped_tile(const Args& a, int q, int height, Rows& r) {
  const int lane = threadIdx.x & 63;
  int ahead = 0;
  for (int e0 = 0; e0 <= a.batch; e0 += 64) {
    const int e = e0 + lane;
    int lo = 0, hi = 0;  // group a.batch: the rows behind the last one
    if (e <= a.batch) {
      lo = start_at(a, e);
      hi = e < a.batch ? start_at(a, e + 1) : a.pairs;
    }
    const int tiles = hi > lo ? (hi - lo + height - 1) / height : 0;
    int sum = tiles;
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(sum, d, 64);
      if (lane >= d) sum += up;
    }
    const uint64_t past = __ballot(ahead + sum > q);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int first = ahead + __shfl(sum - tiles, at, 64);
      r.mat = __builtin_amdgcn_readfirstlane(e0 + at);
      r.row = __builtin_amdgcn_readfirstlane(__shfl(lo, at, 64) + (q - first) * height);
      r.end = __builtin_amdgcn_readfirstlane(min(r.row + height, __shfl(hi, at, 64)));
      r.zeros = r.mat == a.batch;
      return true;
    }
    ahead += __shfl(sum, 63, 64);
  }
  return false;
}

// Upper bound of grouped_tile's tiles, from what the host knows
inline int64_t grouped_tiles(int64_t pairs, int64_t groups, int64_t height) {
  const int64_t filled = groups + 1 < pairs ? groups + 1 : pairs;
  return (pairs - filled) / height + filled;
}

// Row of A that goes with row s of C
template <bool GROUPED>
PCAMD_DEV int64_t a_row(const Args& a, int s) {
  if constexpr (GROUPED) {
    if (a.order) s = a.order[s] / a.choices;
    return min(max(s, 0), a.a_rows - 1);
  }
  return s;
}

PCAMD_DEV float load_as(const void* p, int dt, int64_t i) {
  if (dt == kF32) return static_cast<const float*>(p)[i];
  return dt == kBF16 ? load_one<kBF16>(p, i) : load_one<kF16>(p, i);
}

// expf and a division in fp32: what gate gets is within a few units in the last place of 32 bits
PCAMD_DEV float silu(float x) { return x / (1.0f + expf(-x)); }

PCAMD_DEV float activate(float x, int act) {
  return act == PCAMD_ACT_GELU ? 0.5f * x * (1.0f + erff(x * 0.7071067811865475f)) : x;
}

// Four values in the 16-bit type dt
PCAMD_DEV uint2 pack4(int dt, const float (&v)[4]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  if (dt == kBF16) {
    typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
    return make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[0], v[1]}, b16x2)),
                      __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[2], v[3]}, b16x2)));
  }
  typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
  return make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[0], v[1]}, h16x2)),
                    __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[2], v[3]}, h16x2)));
}

// Up to four neighbouring columns of a row of C, rounded once
PCAMD_DEV void store4(void* c, int dt, int64_t off, int valid, const float (&v)[4]) {
  if (dt == kF32) {
    float* p = static_cast<float*>(c) + off;
    if (valid >= 4 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < valid) p[i] = v[i];
    }
    return;
  }
  const uint2 w = pack4(dt, v);
  uint16_t* p = static_cast<uint16_t*>(c) + off;
  if (valid >= 4 && (reinterpret_cast<uintptr_t>(p) & 7) == 0) {
    *reinterpret_cast<uint2*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < valid) p[i] = static_cast<uint16_t>((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
  }
}

// The same of up to eight
PCAMD_DEV void store8(void* c, int dt, int64_t off, int valid, const float (&v)[8]) {
  const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
  if (dt != kF32) {
    uint16_t* p = static_cast<uint16_t*>(c) + off;
    if (valid >= 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      const uint2 a = pack4(dt, lo), b = pack4(dt, hi);
      *reinterpret_cast<uint4*>(p) = make_uint4(a.x, a.y, b.x, b.y);
      return;
    }
  }
  store4(c, dt, off, valid, lo);
  if (valid > 4) store4(c, dt, off + 4, valid - 4, hi);
}

// 16 bytes of a row from k0 on; those at or past k become zeros
PCAMD_DEV v4i mask_tail(v4i v, int k0, int k) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int left = k - k0 - 4 * w;  // valid bytes of this word
    v[w] = left >= 4 ? v[w] : left <= 0 ? 0 : v[w] & ((1 << (8 * left)) - 1);
  }
  return v;
}

// tiles of 16 rt x 16 ct (int8_bmm_rows.hip)
int launch_rows(const Args& a, bool grouped, int rt, int ct, hipStream_t st);
// tiles of 256 x 256 or 128 x 128 (int8_bmm_tiles.hip), where tiles_ok
bool tiles_ok(const Args& a, bool grouped);
int launch_tiles(const Args& a, bool grouped, bool wide, hipStream_t st);

}  // namespace int8
}  // namespace pcamd
