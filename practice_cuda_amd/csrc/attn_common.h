// attn_common.h - matrix-instruction tiles shared by the latent attention
// kernels.
//
// Scores are computed transposed, S^T = K Q^T (m = key token, n = query row),
// and so is the output, O^T = V^T P^T (m = value column, n = query row). Both
// put a query row on a lane: its maximum and sum are reductions over the
// lane's own registers and one or two lane exchanges, its rescaling factor is
// one register, and the registers that hold S^T hold the operand P^T of the
// second product: the order of tokens within a contraction is free, so V^T is
// read in the order in which S^T came out. P never leaves the registers.
//
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <utility>

#include "fp8_common.h"

namespace pcamd {
namespace attn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_ptr;

// f(0), f(1), .. f(N - 1), each with its number as a type: unrolled whatever
// the body's size
template <typename F, int... I>
PCAMD_DEV void unrolled(F& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
PCAMD_DEV void unrolled(F f) {
  unrolled(f, std::make_integer_sequence<int, N>{});
}

// The running maximum (of scores times scale and log2(e) in the decode kernels,
// of bare products q . k in the prefill kernels) starts at a finite value below
// every score that is told apart from -inf, so that a row that has seen nothing
// (all scores -inf) gets weights exp2(-inf) = 0 and no NaN. Times a scale above
// 0.78 it is not finite any more: the prefill kernels keep it out of the weights.
constexpr float kNoMax = -3.0e38f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <int DT>
struct Elem;
template <>
struct Elem<kBF16> {
  typedef bf16x8 vec8;
  static PCAMD_DEV uint32_t narrow2(float a, float b) {
    const bf16x2 h = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, h);
  }
};
template <>
struct Elem<kF16> {
  typedef f16x8 vec8;
  static PCAMD_DEV uint32_t narrow2(float a, float b) {
    const f16x2 h = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, h);
  }
};

// MR query rows a wave: one 32x32x16 product, or one 16x16x32. Both take
// 8 consecutive k per lane and operand; lane = (k group h = lane / MR, row
// lane % MR). D: n = lane % MR; register quad q holds m = QSTEP q + 4 h + 0..3.
template <int DT, int MR>
struct Mfma;
template <int DT>
struct Mfma<DT, 32> {
  typedef f32x16 acc;
  static constexpr int K = 16, REGS = 16, QSTEP = 8;
  static PCAMD_DEV acc mul(uint4 a, uint4 b, acc c) {
    typedef typename Elem<DT>::vec8 v;
    if constexpr (DT == kBF16)
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v, a), __builtin_bit_cast(v, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v, a), __builtin_bit_cast(v, b), c, 0, 0, 0);
  }
};
template <int DT>
struct Mfma<DT, 16> {
  typedef f32x4 acc;
  static constexpr int K = 32, REGS = 4, QSTEP = 16;
  static PCAMD_DEV acc mul(uint4 a, uint4 b, acc c) {
    typedef typename Elem<DT>::vec8 v;
    if constexpr (DT == kBF16)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v, a), __builtin_bit_cast(v, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v, a), __builtin_bit_cast(v, b), c, 0, 0, 0);
  }
};

// The same product where its sum stays in ordinary vector registers: with 256
// accumulation registers taken by the output, the compiler would move 16 of
// them out and back for every tile of scores. The compiler does not see these
// as matrix instructions, so the waits that it would insert stand here: two
// wait states ahead of each for operands that an ordinary instruction wrote
// last, and 12 (settle: 16) between the last of a sum and its first ordinary
// read. Where other products of this kind follow at once, two of them take
// longer than that: mul_holding() makes reads of `held` wait for its own issue.
template <int DT, int MR>
struct ScoreMfma : Mfma<DT, MR> {
  typedef typename Mfma<DT, MR>::acc acc;
  static PCAMD_DEV acc first(uint4 a, uint4 b) { return Mfma<DT, MR>::mul(a, b, acc{}); }
  static PCAMD_DEV acc mul_holding(uint4 a, uint4 b, acc c, acc&) { return Mfma<DT, MR>::mul(a, b, c); }
  static PCAMD_DEV void settle(acc&) {}
};
template <int DT>
struct ScoreMfma<DT, 32> {
  typedef f32x16 acc;
  typedef typename Elem<DT>::vec8 v;
#define PCAMD_SCORE_MFMA(C, ...)                                                             \
  if constexpr (DT == kBF16) asm("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %[a], %[b], " C : __VA_ARGS__); \
  else asm("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %[a], %[b], " C : __VA_ARGS__)
  static PCAMD_DEV acc first(uint4 a, uint4 b) {
    acc c;
    PCAMD_SCORE_MFMA("0", "=&v"(c) : [a] "v"(__builtin_bit_cast(v, a)), [b] "v"(__builtin_bit_cast(v, b)));
    return c;
  }
  static PCAMD_DEV acc mul(uint4 a, uint4 b, acc c) {
    PCAMD_SCORE_MFMA("%0", "+v"(c) : [a] "v"(__builtin_bit_cast(v, a)), [b] "v"(__builtin_bit_cast(v, b)));
    return c;
  }
  static PCAMD_DEV acc mul_holding(uint4 a, uint4 b, acc c, acc& held) {
    PCAMD_SCORE_MFMA("%0", "+v"(c), "+v"(held) : [a] "v"(__builtin_bit_cast(v, a)), [b] "v"(__builtin_bit_cast(v, b)));
    return c;
  }
#undef PCAMD_SCORE_MFMA
  static PCAMD_DEV void settle(acc& c) { asm volatile("s_nop 15" : "+v"(c)); }
};

// Four rows' 16-bit elements of one column, transposed within groups of 16
// lanes: lane i addresses 8 bytes of row i / 4 at columns 4 (i % 4), and
// receives column i of the four rows.
PCAMD_DEV uint2 read_tr4(const uint8_t* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p)));
}

// ---- global -> LDS copies. Lane i's 16 (4) bytes at p land at lds + 16 i
// (4 i). Inline asm: the compiler would wait for every copy in flight before any
// read of LDS.
PCAMD_DEV void copy16(const void* p, uint32_t lds) {
  asm volatile("global_load_lds_dwordx4 %0, off" ::"v"(p), "{m0}"(lds) : "memory");
}
PCAMD_DEV void copy4(const void* p, uint32_t lds) {
  asm volatile("global_load_lds_dword %0, off" ::"v"(p), "{m0}"(lds) : "memory");
}
// until at most N copies are in flight
template <int N>
PCAMD_DEV void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// all waves' reads of LDS are behind them, and their copies that they waited for are there
PCAMD_DEV void tile_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Tiles of 128-byte rows: chunk c (16 bytes) of row t lies at c ^ f(t). t & 1 is
// a half of the 256 bytes that 16 lanes may read without conflict; the rest of
// t spreads 16 consecutive rows' equal chunks (keys) over all eight places, and
// the four rows that a transposing read takes at once (64 bytes each) over both
// halves of a row: the reversed bits of t / 2.
PCAMD_DEV int swizzle16(int t) { return ((t & 2) << 1) | ((t >> 1) & 2) | ((t >> 3) & 1); }

// max / sum over the lane groups that share a row: swapping rows of 16 (32)
// lanes between two copies leaves one group's values in each
template <int MR, typename F>
PCAMD_DEV float row_reduce(float v, F f) {
  if constexpr (MR == 16) {
    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(x[0]), __uint_as_float(x[1]));
  }
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
template <int MR>
PCAMD_DEV float row_max(float v) {
  return row_reduce<MR>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int MR>
PCAMD_DEV float row_sum(float v) {
  return row_reduce<MR>(v, [](float a, float b) { return a + b; });
}

// Eight rows' bytes of one column: lane i of 16 addresses 8 bytes of row i / 2
// at columns 8 (i % 2), and receives column i of the eight rows.
PCAMD_DEV uint2 read_tr8(const uint8_t* p) {
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  typedef __attribute__((address_space(3))) i32x2* lds_ptr;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_ptr)(p)));
}

// two of four fp8 codes as 16-bit elements, times a power of two (exact where it is one)
template <int DT, bool HI>
PCAMD_DEV uint32_t widen2(uint32_t c, float unit) {
  if constexpr (DT == kBF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, unit, HI));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, unit, HI));
}

}  // namespace attn
}  // namespace pcamd
