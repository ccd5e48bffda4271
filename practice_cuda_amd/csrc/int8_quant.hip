// int8_quant.hip - int8 codes with one fp32 scale for each row.
//
//   top = max(max|x|, eps), scale = top / 127,
//   code = rint(127 x / top), ties to even
//
// The code is that of the real quotient, not of its fp32 form: x * (127 / top)
// in fp32 is within 127 * 2^-22 = 3.1e-5 of it, so a value whose fp32 form lies
// further than 1e-4 from the border of two codes has its code already; the
// others (one in 5000) are divided in fp64. There 127 x is exact, and a
// quotient that is not a tie misses one by more than 2^-33 of its size, far
// more than fp64 rounds by. So codes do not depend on how a kernel rounds.
//
// A row with a NaN or an infinity, which no code stands for, gets the scale
// NaN and codes of zero: its products are NaN.
//
// A row of up to 32768 values is read once and held in registers between the
// maximum and the codes (a wave a row up to 2048 values, a workgroup above).
#include <hip/hip_runtime.h>

#include <cstdint>

#include "abi_util.h"
#include "fp8_common.h"

namespace pcamd {
namespace int8q {

struct Args {
  const void* x;
  int8_t* y;
  float* scale;
  int64_t sxb, sxm, syb, sym, ssb, ssm;  // elements
  int64_t rows;                          // batch * m
  int32_t m, n;
  float eps;
};

// 16-byte vectors at any element alignment
typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// elements [off, off + 8) of a row of n, zeros behind its end
template <int DT>
PCAMD_DEV void load8(Chunk<DT>& c, const void* row, int off, int n) {
  const uint8_t* p = static_cast<const uint8_t*>(row) + int64_t(off) * elem_bytes<DT>();
  if (off + 8 <= n) {
    const u32x4_any a = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
    c.r[0] = make_uint4(a.x, a.y, a.z, a.w);
    if constexpr (DT == kF32) {
      const u32x4_any b = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p) + 1);
      c.r[1] = make_uint4(b.x, b.y, b.z, b.w);
    }
    return;
  }
  zero_chunk<DT>(c);
  uint32_t w[DT == kF32 ? 8 : 4] = {};
  for (int i = 0; i < n - off; ++i) {
    if constexpr (DT == kF32) {
      w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    } else {
      w[i >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1));
    }
  }
  c.r[0] = make_uint4(w[0], w[1], w[2], w[3]);
  if constexpr (DT == kF32) c.r[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

// bits of the largest |x| of a chunk as fp32: they order like the values, and NaN lies above infinity
template <int DT>
PCAMD_DEV uint32_t chunk_top(const Chunk<DT>& c) {
  if constexpr (DT == kBF16) return __float_as_uint(chunk_amax<kBF16>(c));
  float v[8];
  unpack_chunk<DT>(c, v);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return top;
}

constexpr uint32_t kInf = 0x7F800000u;

struct Row {
  float top;      // 0: every code is 0
  float factor;   // 127 / top
  bool by_fp64;   // factor is not finite, or too rough: every code is divided in fp64
};

PCAMD_DEV Row row_of(uint32_t bits, float eps) {
  Row r;
  r.top = bits >= kInf ? 0.0f : fmaxf(__uint_as_float(bits), eps);
  r.factor = r.top > 0.0f ? 127.0f / r.top : 0.0f;
  r.by_fp64 = r.top > 0.0f && r.top < 1e-30f;
  return r;
}

PCAMD_DEV float scale_of(uint32_t bits, const Row& r) {
  return bits >= kInf ? __uint_as_float(0x7FC00000u) : r.top / 127.0f;
}

// eight codes, four a word
template <int DT>
PCAMD_DEV uint2 codes(const Chunk<DT>& c, const Row& r) {
  float v[8];
  unpack_chunk<DT>(c, v);
  if (r.top == 0.0f) return make_uint2(0, 0);
  // adding 1.5 * 2^23 rounds to an integer, ties to even, and leaves it in the low byte
  constexpr float kMagic = 12582912.0f;
  uint32_t q[8];
  float far = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = v[i] * r.factor;
    const float m = t + kMagic;
    far = fmaxf(far, fabsf(t - (m - kMagic)));
    q[i] = __float_as_uint(m);
  }
  if (far > 0.4999f || r.by_fp64) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      q[i] = static_cast<uint32_t>(static_cast<int>(rint(127.0 * static_cast<double>(v[i]) / static_cast<double>(r.top))));
  }
  auto four = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0C0C0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000C0Cu);
    return lo | hi;
  };
  return make_uint2(four(q[0], q[1], q[2], q[3]), four(q[4], q[5], q[6], q[7]));
}

// The maximum over a team: a wave, or the workgroup (TEAM_WAVE false)
template <bool TEAM_WAVE>
PCAMD_DEV uint32_t team_top(uint32_t top, uint32_t* shared) {
  top = __float_as_uint(group_max<64>(__uint_as_float(top)));
  if constexpr (!TEAM_WAVE) {
    const int waves = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int w = 0; w < waves; ++w) top = max(top, shared[w]);
  }
  return top;
}

// Lane i of a row's team takes the chunks i, i + team, .. (C of them); ONCE: all of them stay in registers.
template <int DT, int C, bool TEAM_WAVE, bool ONCE>
__global__ __launch_bounds__(TEAM_WAVE ? 256 : 1024) void quant_rows_kernel(Args a) {
  __shared__ uint32_t shared[16];
  const int team = TEAM_WAVE ? 64 : blockDim.x;
  const int t = TEAM_WAVE ? threadIdx.x & 63 : threadIdx.x;
  const int64_t block = int64_t(blockIdx.y) * gridDim.x + blockIdx.x;
  const int64_t row = TEAM_WAVE ? block * 4 + (threadIdx.x >> 6) : block;
  if (row >= a.rows) return;  // a whole wave; a workgroup that synchronizes has one row
  const int64_t b = row / a.m, i = row - b * a.m;
  const uint8_t* x = static_cast<const uint8_t*>(a.x) + (b * a.sxb + i * a.sxm) * elem_bytes<DT>();
  int8_t* y = a.y + b * a.syb + i * a.sym;
  const int chunks = ((a.n + 15) / 16) * 2;  // the padding up to 16 bytes is written as zeros
  uint32_t top = 0;
  if constexpr (ONCE) {
    Chunk<DT> c[C];
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int at = t + k * team;
      if (at * 8 < a.n) load8<DT>(c[k], x, at * 8, a.n);
      else zero_chunk<DT>(c[k]);
    }
#pragma unroll
    for (int k = 0; k < C; ++k) top = max(top, chunk_top<DT>(c[k]));
    top = team_top<TEAM_WAVE>(top, shared);
    const Row r = row_of(top, a.eps);
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int at = t + k * team;
      if (at < chunks) *reinterpret_cast<uint2*>(y + at * 8) = codes<DT>(c[k], r);
    }
    if (t == 0) a.scale[b * a.ssb + i * a.ssm] = scale_of(top, r);
  } else {
    for (int at = t; at * 8 < a.n; at += team) {
      Chunk<DT> c;
      load8<DT>(c, x, at * 8, a.n);
      top = max(top, chunk_top<DT>(c));
    }
    top = team_top<TEAM_WAVE>(top, shared);
    const Row r = row_of(top, a.eps);
    for (int at = t; at < chunks; at += team) {
      Chunk<DT> c;
      if (at * 8 < a.n) load8<DT>(c, x, at * 8, a.n);
      else zero_chunk<DT>(c);
      *reinterpret_cast<uint2*>(y + at * 8) = codes<DT>(c, r);
    }
    if (t == 0) a.scale[b * a.ssb + i * a.ssm] = scale_of(top, r);
  }
}

// a dimension of a grid may have up to 2^32 - 1 threads
dim3 grid_of(int64_t blocks) {
  const int64_t x = blocks < (1 << 20) ? blocks : 1 << 20;
  return dim3(static_cast<unsigned>(x), static_cast<unsigned>((blocks + x - 1) / x));
}

template <int DT>
int launch(const Args& a, hipStream_t st) {
  const int chunks = (a.n + 7) / 8;
  if (chunks <= 256) {
    const dim3 grid = grid_of((a.rows + 3) / 4);
    if (chunks <= 64) quant_rows_kernel<DT, 1, true, true><<<grid, 256, 0, st>>>(a);
    else if (chunks <= 128) quant_rows_kernel<DT, 2, true, true><<<grid, 256, 0, st>>>(a);
    else quant_rows_kernel<DT, 4, true, true><<<grid, 256, 0, st>>>(a);
    return check_launch("quant_rows_kernel");
  }
  const dim3 grid = grid_of(a.rows);
  if (chunks > 4096) {
    quant_rows_kernel<DT, 1, false, false><<<grid, 1024, 0, st>>>(a);
    return check_launch("quant_rows_kernel");
  }
  const int threads = (((chunks + 3) / 4) + 63) / 64 * 64;
  quant_rows_kernel<DT, 4, false, true><<<grid, threads, 0, st>>>(a);
  return check_launch("quant_rows_kernel");
}

}  // namespace int8q
}  // namespace pcamd

extern "C" int pcamd_quant_int8(const void* x, int x_dtype, int64_t batch, int64_t m, int64_t n, int64_t sxb,
                                int64_t sxm, void* y, int64_t syb, int64_t sym, float* scale, int64_t ssb, int64_t ssm,
                                float eps, void* stream) {
  using namespace pcamd;
  clear_error();
  if (x_dtype != kF32 && x_dtype != kBF16 && x_dtype != kF16)
    return set_error(PCAMD_ERR_INVALID, "input dtype must be fp32, bf16 or fp16, got code %d", x_dtype);
  if (batch < 0 || m < 0 || n < 0) return set_error(PCAMD_ERR_INVALID, "negative size");
  if (!(eps >= 0.0f) || eps > 3e38f) return set_error(PCAMD_ERR_INVALID, "eps must be finite and not negative");
  if (batch == 0 || m == 0) return PCAMD_OK;
  if ((n && (!x || !y)) || !scale) return set_error(PCAMD_ERR_INVALID, "null pointer");
  const int size = x_dtype == kF32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(x) % size) return set_error(PCAMD_ERR_INVALID, "x is not aligned to its elements");
  if ((reinterpret_cast<uintptr_t>(y) & 15) || (m > 1 && sym % 16) || (batch > 1 && syb % 16))
    return set_error(PCAMD_ERR_INVALID, "rows of codes must be 16-byte aligned");
  // a thread's place in a long row steps on by 1024 * 8 values, past the row's end, in 32 bits
  if (m > INT32_MAX || n > INT32_MAX - 16384 || batch > INT32_MAX / m)
    return set_error(PCAMD_ERR_UNSUPPORTED, "int8 quant: more than 2^31 - 1 rows or 2^31 - 16385 columns");
  int8q::Args a{x, static_cast<int8_t*>(y), scale, sxb, sxm, syb, sym, ssb, ssm, batch * m, static_cast<int32_t>(m),
                static_cast<int32_t>(n), eps};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (x_dtype == kF32) return int8q::launch<kF32>(a, st);
  if (x_dtype == kBF16) return int8q::launch<kBF16>(a, st);
  return int8q::launch<kF16>(a, st);
}
