// rms_norm.hip - root-mean-square norm with the residual's addition and an
// fp8 output in 1 x 128 groups, and the same norm written into the pages of a
// latent cache.
//
//   r = x + residual           (fp32; also stored, rounded to x's type)
//   y = r * rsqrt(mean(r^2) + norm_eps) * w
//   per group of 128 columns: qs = fp8_max / max(max|y|, eps),
//   codes = fp8(clamp(y * qs)), scale = 1 / qs
//
// One team of lanes holds a row of up to 16384 values in registers between the
// two reductions (the sum of squares over the row, the maxima over 16-lane
// groups), so every input is read once. Lane i of the team takes the 8-element chunks i, i + TEAM, ..;
// 16 neighbouring lanes then hold one quantization group.
//
// Bound by memory: 4096 x 7168 bf16 with a residual, 206 MB, takes 50.2 us, 4.1
// TB/s (a large copy 5.9 to 6.4). Rows that are not 16-byte aligned take longer: 29
// million values in rows of 5003 columns 58 us, of 5120 45. By the launch where
// rows are few: 56 tokens of 512 + 64 into an fp8 cache 9 us a call, most of it
// the host's.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "abi_util.h"
#include "fp8_common.h"

namespace pcamd {
namespace norm {

constexpr int kGroup = 128;

// 16-byte vectors at any element alignment: gfx950 loads and stores them
// unaligned, so odd row lengths keep the wide accesses.
typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// elements [off, off + valid) of a row, zeros behind them
template <int DT>
PCAMD_DEV void load8(const void* base, int64_t off, int64_t valid, float (&v)[8]) {
  if (valid >= 8) {
    const u32x4_any* p = reinterpret_cast<const u32x4_any*>(static_cast<const uint8_t*>(base) + off * elem_bytes<DT>());
    Chunk<DT> c;
    const u32x4_any a = p[0];
    c.r[0] = make_uint4(a.x, a.y, a.z, a.w);
    if constexpr (DT == kF32) {
      const u32x4_any b = p[1];
      c.r[1] = make_uint4(b.x, b.y, b.z, b.w);
    }
    unpack_chunk<DT>(c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? load_one<DT>(base, off + i) : 0.0f;
  }
}

PCAMD_DEV void load8_as(int dt, const void* base, int64_t off, int64_t valid, float (&v)[8]) {
  if (dt == kF32) load8<kF32>(base, off, valid, v);
  else if (dt == kBF16) load8<kBF16>(base, off, valid, v);
  else load8<kF16>(base, off, valid, v);
}

// round to nearest even
template <int DT>
PCAMD_DEV uint32_t narrow2(float a, float b) {
  if constexpr (DT == kBF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 h = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, h);
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 h = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, h);
  }
}

template <int DT>
PCAMD_DEV void store8(void* base, int64_t off, int64_t valid, const float (&v)[8]) {
  uint8_t* p = static_cast<uint8_t*>(base) + off * elem_bytes<DT>();
  if constexpr (DT == kF32) {
    if (valid >= 8) {
      u32x4_any a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) { a[i] = __float_as_uint(v[i]); b[i] = __float_as_uint(v[4 + i]); }
      reinterpret_cast<u32x4_any*>(p)[0] = a;
      reinterpret_cast<u32x4_any*>(p)[1] = b;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < valid) reinterpret_cast<float*>(p)[i] = v[i];
    }
  } else {
    u32x4_any a;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = narrow2<DT>(v[2 * i], v[2 * i + 1]);
    if (valid >= 8) {
      *reinterpret_cast<u32x4_any*>(p) = a;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < valid) reinterpret_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(a[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// max |y| of a chunk; NaN elements do not count, as in the quantizers
PCAMD_DEV float amax8(const float (&y)[8]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(y[i]));
  return m;
}

// Scales of a group of y = t * inv, t = r * w: as block_scales of y, with inv
// left out of the codes' factor where y's largest value sets it: codes come of
// r * w, one division and their product, without the roundings of inv and of y.
// Which side of a boundary between two codes a value falls on still differs from
// one order of operations to another. (inf * 0, of a row with an infinity, takes
// the floor: its other values are zeros.)
PCAMD_DEV Scales normed_scales(float amax_t, float inv, float fp8_max, float eps) {
  const bool above = amax_t * inv >= eps;
  const float qs = fp8_max / (above ? amax_t : eps);
  return above ? Scales{qs, inv / qs} : Scales{qs * inv, 1.0f / qs};
}

// fp8 of clamp(y * qs); a NaN stays one (the clamp alone would make it -fp8_max)
template <int FMT>
PCAMD_DEV uint2 codes8(const float (&y)[8], float qs, float fp8_max) {
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = y[i] * qs;
    q[i] = t != t ? t : clamp_sym(t, fp8_max);
  }
  return make_uint2(pack4<FMT>(q[0], q[1], q[2], q[3]), pack4<FMT>(q[4], q[5], q[6], q[7]));
}

PCAMD_DEV void store_codes(uint8_t* p, int64_t valid, uint2 c) {
  if (valid >= 8) {
    const u32x2_any w = {c.x, c.y};
    *reinterpret_cast<u32x2_any*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) p[i] = static_cast<uint8_t>((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
  }
}

// over groups of LANES neighbouring lanes
template <int LANES>
PCAMD_DEV float lanes_sum(float v) {
#pragma unroll
  for (int d = LANES / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

struct NormArgs {
  const void* x; const void* residual; const void* weight;
  uint8_t* y; float* scale; void* residual_out;
  int64_t rows, m, n;
  int64_t sxb, sxm, srb, srm, syb, sym, ssb, ssm, sob, som;
  int w_dtype;
  float norm_eps, fp8_max, eps;
};

// NV chunks per lane in registers; NV = 0: rows of any length, read a second
// time (from the caches where they fit) instead of held.
template <int DT, int FMT, int TEAM, int NV>
__global__ __launch_bounds__(TEAM < 256 ? 256 : TEAM) void norm_quant_kernel(NormArgs a) {
  constexpr int WG = TEAM < 256 ? 256 : TEAM;
  constexpr int TEAMS = WG / TEAM;
  __shared__ float sums[2][WG / 64];
  const int lane = threadIdx.x % TEAM;
  const int64_t chunks = (a.n + 7) / 8;
  int parity = 0;
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * TEAMS; row0 < a.rows;
       row0 += static_cast<int64_t>(gridDim.x) * TEAMS, parity ^= 1) {
    const int64_t want = row0 + (TEAMS > 1 ? threadIdx.x / TEAM : 0);
    const bool live = want < a.rows;
    const int64_t row = live ? want : a.rows - 1;  // a spare team computes the last row and stores nothing
    const int64_t b = row / a.m, r = row - b * a.m;
    const int64_t x0 = b * a.sxb + r * a.sxm, r0 = b * a.srb + r * a.srm, o0 = b * a.sob + r * a.som;

    auto load_sum = [&](int64_t c, float (&v)[8], bool store) {
      const int64_t valid = c < chunks ? a.n - 8 * c : 0;
      load8<DT>(a.x, x0 + 8 * c, valid, v);
      if (a.residual) {
        float t[8];
        load8<DT>(a.residual, r0 + 8 * c, valid, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += t[i];
        if (store && live) store8<DT>(a.residual_out, o0 + 8 * c, valid, v);
      }
    };
    float v[NV > 0 ? NV : 1][8];
    float s = 0.0f;
    if constexpr (NV > 0) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        load_sum(lane + static_cast<int64_t>(k) * TEAM, v[k], true);
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[k][i] * v[k][i];
      }
    } else {
      for (int64_t c = lane; c < chunks; c += TEAM) {
        load_sum(c, v[0], false);
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[0][i] * v[0][i];
      }
    }
    s = lanes_sum<(TEAM < 64 ? TEAM : 64)>(s);
    if constexpr (TEAM > 64) {
      if (threadIdx.x % 64 == 0) sums[parity][threadIdx.x / 64] = s;
      __syncthreads();  // the other parity's sums may still be read: two buffers, one barrier a row
      s = 0.0f;
#pragma unroll
      for (int w = 0; w < TEAM / 64; ++w) s += sums[parity][threadIdx.x / TEAM * (TEAM / 64) + w];
    }
    const float inv = rsqrtf(s / static_cast<float>(a.n) + a.norm_eps);

    auto finish = [&](int64_t c, float (&y)[8]) {
      const int64_t valid = c < chunks ? a.n - 8 * c : 0;
      float w[8];
      load8_as(a.w_dtype, a.weight, 8 * c, valid, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= w[i];
      const Scales sc = normed_scales(group_max<16>(amax8(y)), inv, a.fp8_max, a.eps);
      if (!live || valid <= 0) return;
      if (lane % 16 == 0) a.scale[b * a.ssb + r * a.ssm + c / 16] = sc.ds;
      store_codes(a.y + b * a.syb + r * a.sym + 8 * c, valid, codes8<FMT>(y, sc.qs, a.fp8_max));
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int k = 0; k < NV; ++k) finish(lane + static_cast<int64_t>(k) * TEAM, v[k]);
    } else {
      // whole rounds of the team: the group maxima take every lane
      for (int64_t c0 = 0; c0 < chunks; c0 += TEAM) {
        load_sum(c0 + lane, v[0], true);
        finish(c0 + lane, v[0]);
      }
    }
  }
}

struct AppendArgs {
  const void* latent; const void* rope; const void* weight; const void* slots;
  uint8_t* c_latent; uint8_t* c_rope; float* c_scale;
  int64_t tokens, slt, srt, clp, clt, crp, crt, csp, cst, places;
  int dl, dr, page, w_dtype, slot_bytes;
  float norm_eps, eps;
};

// One wave a token: its latent (up to 512 values) is one chunk a lane.
template <int DT, bool FP8>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  const int lane = threadIdx.x % 64;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 4;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 64; t < a.tokens; t += step) {
    const int64_t slot = a.slot_bytes == 8 ? static_cast<const int64_t*>(a.slots)[t]
                                           : static_cast<const int32_t*>(a.slots)[t];
    if (slot < 0 || slot >= a.places) continue;  // the wave's lanes agree
    const int64_t page = slot / a.page, at = slot - page * a.page;
    const int64_t valid = a.dl - 8 * lane;  // >= 8 or <= 0
    float v[8];
    load8<DT>(a.latent, t * a.slt + 8 * lane, valid > 0 ? valid : 0, v);
    float inv = 1.0f;
    if (a.weight) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i] * v[i];
      inv = rsqrtf(lanes_sum<64>(s) / static_cast<float>(a.dl) + a.norm_eps);
      float w[8];
      load8_as(a.w_dtype, a.weight, 8 * lane, valid > 0 ? valid : 0, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= w[i];
    }
    if constexpr (FP8) {
      const Scales sc = normed_scales(group_max<16>(amax8(v)), inv, fmt_max<kE4M3>(), a.eps);
      if (valid > 0) {
        if (lane % 16 == 0) a.c_scale[page * a.csp + at * a.cst + lane / 16] = sc.ds;
        store_codes(a.c_latent + page * a.clp + at * a.clt + 8 * lane, 8, codes8<kE4M3>(v, sc.qs, fmt_max<kE4M3>()));
      }
    } else if (valid > 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= inv;
      store8<DT>(a.c_latent, page * a.clp + at * a.clt + 8 * lane, 8, v);
    }
    for (int c = lane; 8 * c < a.dr; c += 64) {
      const u32x4_any raw =
          *reinterpret_cast<const u32x4_any*>(static_cast<const uint16_t*>(a.rope) + t * a.srt + 8 * c);
      *reinterpret_cast<u32x4_any*>(reinterpret_cast<uint16_t*>(a.c_rope) + page * a.crp + at * a.crt + 8 * c) = raw;
    }
  }
}

template <int DT, int FMT>
int launch_norm(const NormArgs& a, hipStream_t st) {
  // workgroups beyond the cap take further rows
  auto go = [&](auto team, auto nv) {
    constexpr int TEAM = decltype(team)::value, NV = decltype(nv)::value;
    constexpr int WG = TEAM < 256 ? 256 : TEAM;
    const int64_t groups = (a.rows + WG / TEAM - 1) / (WG / TEAM);
    const int64_t cap = int64_t{1} << 20;
    norm_quant_kernel<DT, FMT, TEAM, NV><<<static_cast<uint32_t>(groups < cap ? groups : cap), WG, 0, st>>>(a);
    return check_launch("norm_quant_kernel");
  };
  using std::integral_constant;
  // A team that a row fills, with two chunks a lane and more where it can: the loads of both are in flight at once. 29 million
  // values (16384 rows at most), bf16 with a residual, us, the team taken and the ones beside it:
  //   64 columns 16 x 1 5.1, 64 x 1 11.0; 129 16 x 2 7.8, 32 x 1 10.0; 300 32 x 2 16.0, 64 x 1 20.0; 1024 64 x 2 29.2, 128 x 1
  //   30.9, 64 x 4 42.2; 1031 64 x 3 49.1, 128 x 2 54.1; 2000 128 x 2 50.0, 64 x 4 59.2; 4096 256 x 2 47.3, 512 x 1 48.3, 128 x 4
  //   56.0; 5120 256 x 3 49.7, 512 x 2 57.0; 7168 512 x 2 51.1, 256 x 4 55.0, 1024 x 1 65.2; 10007 512 x 3 73.5, 1024 x 2 96.2;
  //   16384 512 x 4 53.9, 1024 x 2 54.0
  if (a.n <= 128) return go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  if (a.n <= 256) return go(integral_constant<int, 16>{}, integral_constant<int, 2>{});
  if (a.n <= 512) return go(integral_constant<int, 32>{}, integral_constant<int, 2>{});
  if (a.n <= 1024) return go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  if (a.n <= 1536) return go(integral_constant<int, 64>{}, integral_constant<int, 3>{});
  if (a.n <= 2048) return go(integral_constant<int, 128>{}, integral_constant<int, 2>{});
  if (a.n <= 4096) return go(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  if (a.n <= 6144) return go(integral_constant<int, 256>{}, integral_constant<int, 3>{});
  if (a.n <= 8192) return go(integral_constant<int, 512>{}, integral_constant<int, 2>{});
  if (a.n <= 12288) return go(integral_constant<int, 512>{}, integral_constant<int, 3>{});
  if (a.n <= 16384) return go(integral_constant<int, 512>{}, integral_constant<int, 4>{});
  // Longer rows are read twice, the second time from the caches. 1024 lanes with eight chunks hold rows of up to 65536 columns,
  // but not within their registers: 16390 columns, bf16, 70 us (held 178), 32768 59 (113), 65536 61 (76), one row of 16390
  // 8.4 (19.6); fp32 102 (190), 104 (134) and, the only loss, 110 (105).
  return go(integral_constant<int, 1024>{}, integral_constant<int, 0>{});
}

bool in16(int dt) { return dt == kBF16 || dt == kF16; }

}  // namespace norm
}  // namespace pcamd

extern "C" int pcamd_rms_norm_quant(const void* x, int x_dtype, int64_t batch, int64_t m, int64_t n, int64_t sxb,
                                    int64_t sxm, const void* residual, int64_t srb, int64_t srm, const void* weight,
                                    int w_dtype, void* y, int y_dtype, int64_t syb, int64_t sym, float* scale,
                                    int64_t ssb, int64_t ssm, void* residual_out, int64_t sob, int64_t som,
                                    float norm_eps, float fp8_max, float eps, void* stream) {
  using namespace pcamd;
  clear_error();
  if (batch < 0 || m < 0 || n < 0) return set_error(PCAMD_ERR_INVALID, "negative size");
  if (x_dtype < kF32 || x_dtype > kF16) return set_error(PCAMD_ERR_INVALID, "bad x dtype code %d", x_dtype);
  if (w_dtype < kF32 || w_dtype > kF16) return set_error(PCAMD_ERR_INVALID, "bad weight dtype code %d", w_dtype);
  if (y_dtype != kE4M3 && y_dtype != kE5M2) return set_error(PCAMD_ERR_INVALID, "bad fp8 dtype code %d", y_dtype);
  if (batch == 0 || m == 0 || n == 0) return PCAMD_OK;
  if (!x || !weight || !y || !scale) return set_error(PCAMD_ERR_INVALID, "null pointer");
  if ((residual == nullptr) != (residual_out == nullptr))
    return set_error(PCAMD_ERR_INVALID, "residual and residual_out come together");
  if (!(fp8_max > 0.0f) || !(eps >= 0.0f) || !(norm_eps >= 0.0f))
    return set_error(PCAMD_ERR_INVALID, "fp8_max must be positive, eps and norm_eps not negative");
  if (m > INT64_MAX / batch) return set_error(PCAMD_ERR_INVALID, "too many rows");
  norm::NormArgs a{x, residual, weight, static_cast<uint8_t*>(y), scale, residual_out, batch * m, m, n,
                   sxb, sxm, srb, srm, syb, sym, ssb, ssm, sob, som, w_dtype, norm_eps, fp8_max, eps};
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto by_fmt = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return y_dtype == kE4M3 ? norm::launch_norm<DT, kE4M3>(a, st) : norm::launch_norm<DT, kE5M2>(a, st);
  };
  if (x_dtype == kF32) return by_fmt(std::integral_constant<int, kF32>{});
  if (x_dtype == kBF16) return by_fmt(std::integral_constant<int, kBF16>{});
  return by_fmt(std::integral_constant<int, kF16>{});
}

extern "C" int pcamd_latent_append(const void* latent, const void* rope, int dtype, int64_t tokens,
                                   int64_t latent_dim, int64_t rope_dim, int64_t slt, int64_t srt, const void* weight,
                                   int w_dtype, const void* slots, int slot_bytes, void* cache_latent, int cache_dtype,
                                   int64_t clp, int64_t clt, void* cache_rope, int64_t crp, int64_t crt,
                                   float* cache_scale, int64_t csp, int64_t cst, int64_t pages, int64_t page_size,
                                   float norm_eps, float eps, void* stream) {
  using namespace pcamd;
  clear_error();
  if (tokens < 0 || pages < 0) return set_error(PCAMD_ERR_INVALID, "negative size");
  if (!norm::in16(dtype)) return set_error(PCAMD_ERR_INVALID, "tokens must be bf16 or fp16, got code %d", dtype);
  if (cache_dtype != dtype && cache_dtype != kE4M3)
    return set_error(PCAMD_ERR_INVALID, "the cache holds the tokens' type or e4m3fn, got code %d", cache_dtype);
  if (weight && (w_dtype < kF32 || w_dtype > kF16))
    return set_error(PCAMD_ERR_INVALID, "bad weight dtype code %d", w_dtype);
  if (slot_bytes != 4 && slot_bytes != 8) return set_error(PCAMD_ERR_INVALID, "slots are int32 or int64");
  if (latent_dim <= 0 || latent_dim > 512 || latent_dim % 128)
    return set_error(PCAMD_ERR_UNSUPPORTED, "latent width must be a multiple of 128 up to 512, got %lld",
                     (long long)latent_dim);
  if (rope_dim < 0 || rope_dim % 8 || rope_dim > 512)
    return set_error(PCAMD_ERR_UNSUPPORTED, "rotary width must be a multiple of 8 up to 512, got %lld",
                     (long long)rope_dim);
  if (page_size <= 0 || page_size > INT32_MAX) return set_error(PCAMD_ERR_INVALID, "bad page size");
  if (pages > INT64_MAX / page_size) return set_error(PCAMD_ERR_INVALID, "too many places");
  if (!(eps >= 0.0f) || !(norm_eps >= 0.0f)) return set_error(PCAMD_ERR_INVALID, "eps and norm_eps must not be negative");
  if (tokens == 0 || pages == 0) return PCAMD_OK;
  if (!latent || !slots || !cache_latent || (rope_dim && (!rope || !cache_rope)) || (cache_dtype == kE4M3 && !cache_scale))
    return set_error(PCAMD_ERR_INVALID, "null pointer");
  norm::AppendArgs a{latent, rope, weight, slots, static_cast<uint8_t*>(cache_latent), static_cast<uint8_t*>(cache_rope),
                     cache_scale, tokens, slt, srt, clp, clt, crp, crt, csp, cst, pages * page_size,
                     static_cast<int>(latent_dim), static_cast<int>(rope_dim), static_cast<int>(page_size), w_dtype,
                     slot_bytes, norm_eps, eps};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t groups = (tokens + 3) / 4, cap = int64_t{1} << 20;
  const uint32_t grid = static_cast<uint32_t>(groups < cap ? groups : cap);
  const bool f8 = cache_dtype == kE4M3;
  if (dtype == kBF16) {
    if (f8) norm::append_kernel<kBF16, true><<<grid, 256, 0, st>>>(a);
    else norm::append_kernel<kBF16, false><<<grid, 256, 0, st>>>(a);
  } else {
    if (f8) norm::append_kernel<kF16, true><<<grid, 256, 0, st>>>(a);
    else norm::append_kernel<kF16, false><<<grid, 256, 0, st>>>(a);
  }
  return check_launch("append_kernel");
}
