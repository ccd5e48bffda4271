// latent_decode.h - attention of absorbed queries over a paged cache of latent
// vectors (one key and value vector a token, shared by all heads).
//
//   s[r, t] = scale * (q_latent[r] . c[t] + q_rope[r] . k_rope[t])
//   o[r] = sum_t softmax(s[r])[t] * c[t],   lse[r] = log sum_t exp(s[r, t])
//
// Rows r are (new token, head) pairs: all of a sequence's rows read the same
// cache, so a cache row is read once for up to 128 of them. New token i of S
// sees the tokens before length - S + i + 1.
//
// A cache in fp8 holds codes and one scale for each token and 128 columns. The
// codes enter the products as they are (16 bits hold them exactly); the scales
// multiply fp32 values: the four groups' partial scores, and the weights p
// ahead of their rounding to 16 bits, once for each group of value columns.
//
// The work is one list of steps of 32 * WT tokens: for each sequence, for each
// tile of rows, the steps over its tokens. Workgroup w of G takes the w-th of
// G equal pieces, whatever the lengths are; pieces of one (sequence, row tile)
// are joined by combine_kernel through their maxima and sums.
#pragma once

#include "attn_common.h"
#include "latent_decode_args.h"

namespace pcamd {
namespace decode {

using namespace attn;

constexpr int NT = 256;
constexpr int TOK = 32;  // tokens of a wave's step

// [first, last) unit of workgroup w, and the workgroup that unit u belongs to
PCAMD_DEV int64_t first_unit(int64_t w, int64_t units, int64_t groups) { return w * units / groups; }
PCAMD_DEV int64_t group_of(int64_t u, int64_t units, int64_t groups) { return ((u + 1) * groups - 1) / units; }

PCAMD_DEV int length_of(const Args& a, int64_t b) {
  const int n = a.lens[b];
  return n < 0 ? 0 : n > a.capacity ? a.capacity : n;
}
PCAMD_DEV int steps_of(int len, int step) { return len > step ? (len + step - 1) / step : 1; }

// sum of v over the workgroup's threads before this one, and over all of them
PCAMD_DEV int64_t block_scan(int64_t v, int64_t* wave_total, int64_t& total) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  int64_t inc = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up(inc, d, 64);
    if (lane >= d) inc += o;
  }
  if (lane == 63) wave_total[wave] = inc;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) before += wave_total[w];
    total += wave_total[w];
  }
  __syncthreads();
  return before + inc - v;
}

template <int DT, bool FP8, int DL, int DR, int MR, int WR>
struct Kernel {
  static constexpr int WT = 4 / WR;
  static constexpr int STEP = TOK * WT;
  static constexpr int ROWS = MR * WR;
  static constexpr int CL = DL / 8, CR = DR / 8;  // chunks of a latent and a rotary row
  static constexpr int GROUPS = DL / 128;
  typedef Mfma<DT, MR> M;
  typedef typename M::acc acc;
  static constexpr int QUADS = TOK / M::QSTEP;     // register quads of a wave's S^T
  static constexpr int SUB = QUADS * 4 / M::REGS;  // S^T products side by side
  static constexpr int KL = DL / M::K, KR = DR / M::K;
  static constexpr int OB = DL / MR;               // blocks of value columns
  static constexpr int PK = TOK / M::K;            // contraction steps of the second product
  static constexpr int LANES_K = 64 / MR;
  // LDS: latent tile, rotary tile, scales; the epilogue reuses all of it
  static constexpr int LAT = STEP * DL * 2, ROPE = STEP * DR * 2, SCALES = FP8 ? STEP * GROUPS * 4 : 0;
  static constexpr int DC = MR == 32 && DL > 256 ? 256 : DL;  // columns of an epilogue pass
  static constexpr int PITCH = DC + 4;
  static constexpr int EPI = 4 * MR * PITCH * 4 + 4 * MR * 8;
  static constexpr int LDS = LAT + ROPE + SCALES > EPI ? LAT + ROPE + SCALES : EPI;

  static PCAMD_DEV void stage(const Args& a, uint8_t* lds, const int32_t* table, int t0, int len) {
    for (int j = threadIdx.x; j < STEP * CL / (FP8 ? 2 : 1); j += NT) {
      constexpr int PER = CL / (FP8 ? 2 : 1);
      const int row = j / PER, c = j % PER, tok = t0 + row;
      uint4 v = make_uint4(0, 0, 0, 0);
      const uint8_t* src = nullptr;
      if (tok < len) {
        const int64_t page = a.page_of(table, tok);
        const int64_t at = page * a.slp + a.offset_of(tok) * a.slt;
        src = static_cast<const uint8_t*>(a.latent) + at * (FP8 ? 1 : 2) + c * 16;
        v = *reinterpret_cast<const uint4*>(src);
      }
      if constexpr (FP8) {
        const uint2 w0 = widen4<DT>(v.x), w1 = widen4<DT>(v.y), w2 = widen4<DT>(v.z), w3 = widen4<DT>(v.w);
        uint8_t* d = lds + row * (DL * 2);
        *reinterpret_cast<uint4*>(d + (((2 * c) ^ swz<CL>(row)) << 4)) = make_uint4(w0.x, w0.y, w1.x, w1.y);
        *reinterpret_cast<uint4*>(d + (((2 * c + 1) ^ swz<CL>(row)) << 4)) = make_uint4(w2.x, w2.y, w3.x, w3.y);
      } else {
        *reinterpret_cast<uint4*>(lds + row * (DL * 2) + ((c ^ swz<CL>(row)) << 4)) = v;
      }
    }
    for (int j = threadIdx.x; j < STEP * CR; j += NT) {
      const int row = j / CR, c = j % CR, tok = t0 + row;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (tok < len) {
        const int64_t at = a.page_of(table, tok) * a.srp + a.offset_of(tok) * a.srt;
        v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.rope) + at + 8 * c);
      }
      *reinterpret_cast<uint4*>(lds + LAT + row * (DR * 2) + ((c ^ swz<CR>(row)) << 4)) = v;
    }
    if constexpr (FP8) {
      for (int j = threadIdx.x; j < STEP * GROUPS; j += NT) {
        const int row = j / GROUPS, g = j % GROUPS, tok = t0 + row;
        float v = 0.0f;
        if (tok < len) v = a.scale[a.page_of(table, tok) * a.ssp + a.offset_of(tok) * a.sst + g];
        reinterpret_cast<float*>(lds + LAT + ROPE)[g * STEP + row] = v;
      }
    }
  }

  static PCAMD_DEV void run(const Args& a, uint8_t* lds) {
    __shared__ int64_t wave_total[NT / 64];
    __shared__ int64_t found[2];
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int wr = wave % WR, wt = wave / WR;
    const int h = lane / MR, ln = lane % MR;

    // ---- this workgroup's piece of the list
    int64_t sum = 0, units;
    for (int64_t b = tid; b < a.batch; b += NT) sum += steps_of(length_of(a, b), STEP);
    block_scan(sum, wave_total, units);
    units *= a.row_tiles;
    int64_t groups = (units + a.min_units - 1) / a.min_units;
    if (groups > a.groups) groups = a.groups;
    if (blockIdx.x == 0 && tid == 0 && a.parts) {
      a.plan[0] = units;
      a.plan[1] = groups;
    }
    const bool writes_plan = blockIdx.x == 0 && a.parts;
    const int64_t w = blockIdx.x;
    if (w >= groups) return;
    int64_t u = first_unit(w, units, groups);
    const int64_t end = first_unit(w + 1, units, groups);
    const int64_t begin = u;
    int64_t base = 0;
    if (tid == 0) found[0] = -1;
    __syncthreads();
    for (int64_t b0 = 0; b0 < a.batch; b0 += NT) {
      const int64_t b = b0 + tid;
      const int64_t mine = b < a.batch ? int64_t{steps_of(length_of(a, b), STEP)} * a.row_tiles : 0;
      int64_t total;
      const int64_t before = base + block_scan(mine, wave_total, total);
      if (b < a.batch) {
        if (writes_plan) a.plan[2 + b] = before;
        if (u >= before && u < before + mine) {
          found[0] = b;
          found[1] = u - before;
        }
      }
      base += total;
      __syncthreads();
      if (found[0] >= 0 && !writes_plan) break;
    }
    int64_t b = found[0], in_seq = found[1];

    while (u < end) {
      const int len = length_of(a, b);
      const int steps = steps_of(len, STEP);
      const int rt = static_cast<int>(in_seq / steps), s0 = static_cast<int>(in_seq % steps);
      const int64_t left = end - u;
      const int n = left < steps - s0 ? static_cast<int>(left) : steps - s0;
      segment(a, lds, b, rt, s0, n, steps, len, u == begin ? 2 * w : 2 * w + 1, wr, wt, h, ln);
      u += n;
      in_seq += n;
      if (in_seq >= int64_t{steps} * a.row_tiles) {
        ++b;
        in_seq = 0;
      }
    }
  }

  static PCAMD_DEV void segment(const Args& a, uint8_t* lds, int64_t b, int rt, int s0, int n, int steps, int len,
                                int64_t slot, int wr, int wt, int h, int ln) {
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int row = rt * ROWS + wr * MR + ln;  // this lane's row
    const bool live = row < a.rows;
    const int tok_new = live ? row / a.heads : 0, head = live ? row % a.heads : 0;
    // queries, in registers for the whole segment
    uint4 ql[KL], qr[KR];
    {
      const uint16_t* p = static_cast<const uint16_t*>(a.q_latent) + b * a.qlb + tok_new * a.qls + head * a.qlh;
      const uint16_t* r = static_cast<const uint16_t*>(a.q_rope) + b * a.qrb + tok_new * a.qrs + head * a.qrh;
#pragma unroll
      for (int k = 0; k < KL; ++k)
        ql[k] = live ? *reinterpret_cast<const uint4*>(p + k * M::K + 8 * h) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int k = 0; k < KR; ++k)
        qr[k] = live ? *reinterpret_cast<const uint4*>(r + k * M::K + 8 * h) : make_uint4(0, 0, 0, 0);
    }
    const int limit = live ? len - a.new_tokens + 1 + tok_new : 0;  // tokens this row sees
    acc o[OB];
#pragma unroll
    for (int i = 0; i < OB; ++i) o[i] = acc{};
    float m = kNoMax, l = 0.0f;
    const int32_t* table = a.table + b * a.table_stride;
    const float* scales = reinterpret_cast<const float*>(lds + LAT + ROPE);

    for (int i = 0; i < n; ++i) {
      const int t0 = (s0 + i) * STEP;
      __syncthreads();
      stage(a, lds, table, t0, len);
      __syncthreads();
      const int tb = t0 + wt * TOK;
      if (tb >= len) continue;
      const int lr = wt * TOK;  // first row of this wave's tokens in the tile

      // ---- S^T
      float s[QUADS * 4];
      auto operand = [&](int sub, int chunk_pitch, int chunk, const uint8_t* tile, auto f) {
        const int t = lr + sub * MR + ln;
        return *reinterpret_cast<const uint4*>(tile + t * (chunk_pitch * 16) + ((chunk ^ f(t)) << 4));
      };
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub) {
        acc c = {};
#pragma unroll
        for (int k = 0; k < KR; ++k)
          c = M::mul(operand(sub, CR, k * LANES_K + h, lds + LAT, [](int t) { return swz<CR>(t); }), qr[k], c);
        if constexpr (FP8) {
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) {
            acc d = {};
#pragma unroll
            for (int k = g * (KL / GROUPS); k < (g + 1) * (KL / GROUPS); ++k)
              d = M::mul(operand(sub, CL, k * LANES_K + h, lds, [](int t) { return swz<CL>(t); }), ql[k], d);
#pragma unroll
            for (int r = 0; r < M::REGS; ++r) {
              const int quad = sub * (M::REGS / 4) + r / 4;
              c[r] += scales[g * STEP + lr + quad * M::QSTEP + 4 * h + r % 4] * d[r];
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < KL; ++k)
            c = M::mul(operand(sub, CL, k * LANES_K + h, lds, [](int t) { return swz<CL>(t); }), ql[k], c);
        }
#pragma unroll
        for (int r = 0; r < M::REGS; ++r) s[sub * M::REGS + r] = c[r];
      }

      // ---- softmax, one row a lane
      float top = kNoMax;
#pragma unroll
      for (int r = 0; r < QUADS * 4; ++r) {
        const int t = tb + (r / 4) * M::QSTEP + 4 * h + r % 4;
        s[r] = t < limit ? s[r] * a.scale_log2 : -INFINITY;
        top = fmaxf(top, s[r]);
      }
      top = fmaxf(row_max<MR>(top), m);
      const float alpha = exp2f(m - top);
      m = top;
      float part = 0.0f;
#pragma unroll
      for (int r = 0; r < QUADS * 4; ++r) {
        s[r] = exp2f(s[r] - m);
        part += s[r];
      }
      l = l * alpha + part;
#pragma unroll
      for (int j = 0; j < OB; ++j) o[j] *= alpha;

      // ---- O^T += V^T P^T
#pragma unroll
      for (int g = 0; g < (FP8 ? GROUPS : 1); ++g) {
        uint4 p[PK];
#pragma unroll
        for (int kk = 0; kk < PK; ++kk) {
          uint32_t w[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int r = kk * 8 + 2 * q;
            float x0 = s[r], x1 = s[r + 1];
            if constexpr (FP8) {
              const float* f = scales + g * STEP + lr + (r / 4) * M::QSTEP + 4 * h + r % 4;
              x0 *= f[0] * kScaleUp<DT>;
              x1 *= f[1] * kScaleUp<DT>;
            }
            w[q] = Elem<DT>::narrow2(x0, x1);
          }
          p[kk] = make_uint4(w[0], w[1], w[2], w[3]);
        }
#pragma unroll
        for (int j = g * (FP8 ? OB / GROUPS : OB); j < (g + 1) * (FP8 ? OB / GROUPS : OB); ++j) {
#pragma unroll
          for (int kk = 0; kk < PK; ++kk) {
            const int i16 = lane % 16, g16 = lane / 16;
            const int col = j * MR + (MR == 32 ? 16 * (g16 & 1) : 0) + 4 * (i16 & 3);
            uint2 v[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int t = lr + (2 * kk + q) * M::QSTEP + 4 * h + i16 / 4;
              v[q] = read_tr4(lds + t * (DL * 2) + (((col >> 3) ^ swz<CL>(t)) << 4) + ((col & 4) << 1));
            }
            o[j] = M::mul(make_uint4(v[0].x, v[0].y, v[1].x, v[1].y), p[kk], o[j]);
          }
        }
      }
    }
    l = row_sum<MR>(l);

    // ---- epilogue: the waves' rows meet in LDS and leave as whole rows
    const bool whole = n == steps;
    float* ep = reinterpret_cast<float*>(lds);
    float2* ml = reinterpret_cast<float2*>(lds + 4 * MR * PITCH * 4);
    constexpr float down = FP8 ? 1.0f / kScaleUp<DT> : 1.0f;
#pragma unroll
    for (int d0 = 0; d0 < DL; d0 += DC) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < DC / MR; ++j) {
#pragma unroll
        for (int q = 0; q < M::REGS / 4; ++q) {
          const acc& x = o[d0 / MR + j];
          float* d = ep + (wave * MR + ln) * PITCH + j * MR + q * 8 + 4 * h;
          *reinterpret_cast<float4*>(d) = make_float4(x[4 * q] * down, x[4 * q + 1] * down, x[4 * q + 2] * down,
                                                      x[4 * q + 3] * down);
        }
      }
      if (lane < MR) ml[wave * MR + ln] = make_float2(m, l);
      __syncthreads();
      for (int i = tid; i < ROWS * (DC / 4); i += NT) {
        const int r = i / (DC / 4), d = 4 * (i % (DC / 4));
        const int rr = rt * ROWS + r;
        if (rr >= a.rows) continue;
        const int src = (r / MR) * MR + r % MR;  // wave wr = r / MR of the first token group
        float big = kNoMax;
#pragma unroll
        for (int t = 0; t < WT; ++t) big = fmaxf(big, ml[t * WR * MR + src].x);
        float4 x = make_float4(0, 0, 0, 0);
        float total = 0.0f;
#pragma unroll
        for (int t = 0; t < WT; ++t) {
          const float2 s = ml[t * WR * MR + src];
          const float f = exp2f(s.x - big);
          const float4 y = *reinterpret_cast<const float4*>(ep + (t * WR * MR + src) * PITCH + d);
          x.x += f * y.x; x.y += f * y.y; x.z += f * y.z; x.w += f * y.w;
          total += f * s.y;
        }
        if (whole) {
          const int sn = rr / a.heads, hd = rr % a.heads;
          const float inv = total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : NAN;
          const uint2 out = make_uint2(Elem<DT>::narrow2(x.x * inv, x.y * inv), Elem<DT>::narrow2(x.z * inv, x.w * inv));
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + b * a.ob + sn * a.os + hd * a.oh + d0 + d) = out;
          if (a.lse && d0 + d == 0)
            a.lse[b * a.lb + sn * a.ls + hd * a.lh] = total == 0.0f ? -INFINITY : (big + log2f(total)) * kLn2;
        } else {
          const int64_t at = slot * ROWS + r;
          *reinterpret_cast<float4*>(a.parts + at * DL + d0 + d) = x;
          if (d0 + d == 0) a.part_ml[at] = make_float2(big, total);
        }
      }
    }
    __syncthreads();
  }
};

template <int DT, bool FP8, int DL, int DR, int MR, int WR>
__global__ __launch_bounds__(NT, 1) void decode_kernel(Args a) {
  extern __shared__ __align__(16) uint8_t lds[];
  Kernel<DT, FP8, DL, DR, MR, WR>::run(a, lds);
}

// Joins the pieces of a (sequence, row tile): one workgroup a row, its waves
// take the pieces in turn, each lane DL / 64 columns.
template <int DT, int DL>
__global__ __launch_bounds__(NT) void combine_kernel(Args a, int tile_rows, int step) {
  constexpr int V = DL / 64;
  __shared__ float sums[NT / 64][DL];
  __shared__ float2 ml[NT / 64];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int64_t units = a.plan[0], groups = a.plan[1];
  for (int64_t i = blockIdx.x; i < a.batch * a.rows; i += gridDim.x) {
    const int64_t b = i / a.rows;
    const int row = static_cast<int>(i % a.rows), rt = row / tile_rows, r = row % tile_rows;
    const int steps = steps_of(length_of(a, b), step);
    const int64_t u0 = a.plan[2 + b] + int64_t{rt} * steps, u1 = u0 + steps;
    const int64_t w0 = group_of(u0, units, groups), w1 = group_of(u1 - 1, units, groups);
    if (w0 == w1) continue;  // one workgroup had it all and wrote it
    float m = kNoMax, l = 0.0f, x[V];
#pragma unroll
    for (int k = 0; k < V; ++k) x[k] = 0.0f;
    for (int64_t w = w0 + wave; w <= w1; w += NT / 64) {
      const int64_t slot = first_unit(w, units, groups) >= u0 ? 2 * w : 2 * w + 1;
      const int64_t at = slot * tile_rows + r;
      const float2 s = a.part_ml[at];
      const float* p = a.parts + at * DL + lane * 4;
      float y[V];
#pragma unroll
      for (int k = 0; k < V; k += 4) *reinterpret_cast<float4*>(y + k) = *reinterpret_cast<const float4*>(p + k * 64);
      const float top = fmaxf(m, s.x), f = exp2f(m - top), g = exp2f(s.x - top);
      m = top;
      l = l * f + s.y * g;
#pragma unroll
      for (int k = 0; k < V; ++k) x[k] = x[k] * f + y[k] * g;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; k += 4) *reinterpret_cast<float4*>(&sums[wave][k * 64 + lane * 4]) = *reinterpret_cast<float4*>(x + k);
    if (lane == 0) ml[wave] = make_float2(m, l);
    __syncthreads();
    float big = kNoMax, total = 0.0f;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) big = fmaxf(big, ml[w].x);
    float f[NT / 64];
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
      f[w] = exp2f(ml[w].x - big);
      total += f[w] * ml[w].y;
    }
    const float inv = total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : NAN;
    const int sn = row / a.heads, hd = row % a.heads;
    for (int d = threadIdx.x; d < DL; d += NT) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) v += f[w] * sums[w][d];
      store_elem<DT>(a.out, b * a.ob + sn * a.os + hd * a.oh + d, v * inv);
    }
    if (a.lse && threadIdx.x == 0)
      a.lse[b * a.lb + sn * a.ls + hd * a.lh] = total == 0.0f ? -INFINITY : (big + log2f(total)) * kLn2;
    __syncthreads();
  }
}

}  // namespace decode
}  // namespace pcamd
