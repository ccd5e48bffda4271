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

// How far (log2) a score may pass the reference point of its row's weights
// before the reference moves and the wave's sums are rescaled. Weights and sums
// are floating point: bf16 and fp32 hold 2^40 as exactly as 1, so the first
// tile's maximum nearly always stays the reference. fp16 ends at 2^16, and has
// no room left where an fp8 cache's scales multiply the weights.
template <int DT, bool FP8>
constexpr float kSlack = DT == kF16 ? (FP8 ? 0.0f : 8.0f) : 40.0f;

// Registers that hold operands read ahead of their products, in operands
template <bool FP8>
constexpr int kAheadKeys = FP8 ? 4 : 6;
template <bool FP8>
constexpr int kAheadValues = 6;

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
  static constexpr int GROUPS = DL / 128;
  typedef Mfma<DT, MR> M;
  typedef ScoreMfma<DT, MR> S;
  typedef typename M::acc acc;
  static constexpr int QUADS = TOK / M::QSTEP;     // register quads of a wave's S^T
  static constexpr int SUB = QUADS * 4 / M::REGS;  // S^T products side by side
  static constexpr int KL = DL / M::K, KR = DR / M::K;
  static constexpr int OB = DL / MR;               // blocks of value columns
  static constexpr int PK = TOK / M::K;            // contraction steps of the second product
  static constexpr int LANES_K = 64 / MR;
  // A tile of 32 tokens as it lies in LDS: latent rows (in the cache's type),
  // rotary rows, and with fp8 the scales [group][token].
  static constexpr int LROW = DL * (FP8 ? 1 : 2), RROW = DR * 2;
  static constexpr int CL = LROW / 16, CR = RROW / 16;  // 16-byte chunks of a row
  static constexpr int ROPE = TOK * LROW, SCALES = ROPE + TOK * RROW;
  static constexpr int TILE = SCALES + (FP8 ? TOK * GROUPS * 4 : 0);
  // Tiles per token group: all that fit, up to four
  static constexpr int FIT = 150000 / (WT * TILE);
  static constexpr int NB = FIT > 4 ? 4 : FIT;
  static_assert(NB >= (WR > 1 ? 2 : 1), "a shared ring needs two tiles");
  static constexpr int PAGES = 256;  // page numbers kept in LDS
  static constexpr int RING = WT * NB * TILE;
  // epilogue, in the ring's place: DC columns of every row at a time
  static constexpr int DC = MR == 32 && DL > 256 ? 256 : DL;
  static constexpr int PITCH = DC + 4;
  static constexpr int EPI = 4 * MR * PITCH * 4 + 4 * MR * 8;
  static constexpr int BODY = RING > EPI ? RING : EPI;
  static constexpr int LDS = BODY + PAGES * 4 + 64;  // and a few words of the division of the work
  static_assert(TILE % 256 == 0, "see Lane");

  // ---- global -> LDS copies. The WR waves of a token group share a tile's
  // rows; every wave issues the same number of copies for each tile, so the
  // count of copies in flight says which tiles have arrived.
  static constexpr int RW = TOK / WR;                                // a wave's rows of a tile
  static constexpr int L_COPIES = RW * CL / 64;                      // 64 chunks a copy
  static constexpr int R_COPIES = (RW * CR + 63) / 64;
  static constexpr int S_LANES = FP8 ? TOK * GROUPS / WR : 0;        // scales of a wave
  static constexpr int S_COPIES = (S_LANES + 63) / 64;
  static constexpr int COPIES = L_COPIES + R_COPIES + S_COPIES;
  static_assert(L_COPIES * 64 == RW * CL, "whole copies of latent rows");

  // lane i's 16 (4) bytes at p land at lds + 16 i (4 i). Inline asm: the
  // compiler would wait for every copy in flight before any read of LDS.
  static PCAMD_DEV void copy16(const void* p, uint32_t lds) {
    asm volatile("global_load_lds_dwordx4 %0, off" ::"v"(p), "{m0}"(lds) : "memory");
  }
  static PCAMD_DEV void copy16(uint32_t off, const void* base, uint32_t lds) {
    asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
  }
  static PCAMD_DEV void copy4(const void* p, uint32_t lds) {
    asm volatile("global_load_lds_dword %0, off" ::"v"(p), "{m0}"(lds) : "memory");
  }
  template <int N>
  static PCAMD_DEV void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
  }

  struct Source {
    const int32_t* pages;  // in LDS: the table from page number `first` on
    int first, len;
  };
  // page and place of a token, cut to the sequence's last one: what lies
  // behind it is not read, and a copy of a row that is seen adds nothing once
  // its weight is zero
  static PCAMD_DEV void locate(const Args& a, const Source& src, int t, int64_t& page, int64_t& place) {
    t = t < src.len ? t : src.len - 1;
    const int n = a.page_index(t);
    const uint32_t p = static_cast<uint32_t>(src.pages[n - src.first]);
    page = p < static_cast<uint64_t>(a.pages) ? p : a.pages - 1;
    place = t - n * a.page;
  }

  static PCAMD_DEV void issue(const Args& a, const Source& src, uint32_t tile, int t0, int wr, int lane) {
    const int row0 = wr * RW;
    int64_t page, place;
    locate(a, src, t0 + lane % TOK, page, place);
    const uint64_t mine = static_cast<uint64_t>(page * a.slp + place * a.slt) * (FP8 ? 1 : 2);
    const uint32_t lo = static_cast<uint32_t>(mine), hi = static_cast<uint32_t>(mine >> 32);
    const uint8_t* latent = static_cast<const uint8_t*>(a.latent);
#pragma unroll
    for (int i = 0; i < L_COPIES; ++i) {
      const int r = row0 + i * 64 / CL + (CL < 64 ? lane / CL : 0);  // this lane's row
      const int c = (lane % CL) ^ swz<16>(r);                        // and chunk
      const uint32_t to = tile + row0 * LROW + i * 1024;
      if constexpr (CL == 64) {
        const uint64_t at = static_cast<uint64_t>(__builtin_amdgcn_readlane(hi, row0 + i)) << 32 |
                            static_cast<uint32_t>(__builtin_amdgcn_readlane(lo, row0 + i));
        copy16(16 * c, latent + at, to);
      } else {
        const uint64_t at = static_cast<uint64_t>(static_cast<uint32_t>(__shfl(static_cast<int>(hi), r, 64))) << 32 |
                            static_cast<uint32_t>(__shfl(static_cast<int>(lo), r, 64));
        copy16(latent + at + 16 * c, to);
      }
    }
#pragma unroll
    for (int i = 0; i < R_COPIES; ++i) {
      const int j = i * 64 + lane, r = row0 + j / CR;
      if (RW * CR % 64 == 0 || j < RW * CR) {
        locate(a, src, t0 + r, page, place);
        const uint16_t* p = static_cast<const uint16_t*>(a.rope) + page * a.srp + place * a.srt;
        copy16(p + 8 * ((j % CR) ^ swz<CR>(r)), tile + ROPE + row0 * RROW + i * 1024);
      }
    }
#pragma unroll
    for (int i = 0; i < S_COPIES; ++i) {
      const int j = wr * S_LANES + i * 64 + lane;  // [group][token]
      if (S_LANES % 64 == 0 || i * 64 + lane < S_LANES) {
        locate(a, src, t0 + j % TOK, page, place);
        copy4(a.scale + page * a.ssp + place * a.sst + j / TOK, tile + SCALES + (wr * S_LANES + i * 64) * 4);
      }
    }
  }

  static PCAMD_DEV void run(const Args& a, uint8_t* lds) {
    int64_t* wave_total = reinterpret_cast<int64_t*>(lds + BODY + PAGES * 4);
    int64_t* found = wave_total + NT / 64;
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

  // 8 fp8 codes as 16-bit elements (exact)
  static PCAMD_DEV uint4 widen8(uint2 c) {
    return make_uint4(widen2<DT, false>(c.x), widen2<DT, true>(c.x), widen2<DT, false>(c.y), widen2<DT, true>(c.y));
  }

  // Where this lane reads in a tile. A row's chunks lie at c ^ f(row), and
  // tiles start at multiples of 256 bytes, so the place of another chunk
  // differs by an exclusive or with a constant (within 256 bytes, or a rotary
  // row) and an added one: three registers serve all reads.
  struct Lane {
    int h, ln;
    uint32_t k, kr, v;
    PCAMD_DEV explicit Lane(int lane) : h(lane / MR), ln(lane % MR) {
      const int i16 = lane % 16, g16 = lane / 16;
      k = ln * LROW + ((h ^ swz<16>(ln)) << 4);
      kr = ROPE + ln * RROW + ((h ^ swz<CR>(ln)) << 4);
      if constexpr (FP8) {
        const int t = (i16 >> 3) * M::QSTEP + 4 * h + ((i16 >> 1) & 3);
        v = t * LROW + (((MR == 32 ? g16 & 1 : 0) ^ swz<16>(t)) << 4) + 8 * (i16 & 1);
      } else {
        const int t = 4 * h + (i16 >> 2);
        v = t * LROW + (((MR == 32 ? 2 * (g16 & 1) : 0) + ((i16 >> 1) & 1) ^ swz<16>(t)) << 4) + 8 * (i16 & 1);
      }
    }
    // 16 bytes of a token's latent (rotary) row, as step i reads them; token MR * sub + ln
    PCAMD_DEV uint4 key(const uint8_t* lds, uint32_t tile, int sub, int i) const {
      constexpr int P = 16 / LANES_K;
      return *reinterpret_cast<const uint4*>(lds + ((tile + k) ^ (i % P * LANES_K << 4)) + sub * MR * LROW + i / P * 256);
    }
    PCAMD_DEV uint4 rope(const uint8_t* lds, uint32_t tile, int sub, int i) const {
      return *reinterpret_cast<const uint4*>(lds + ((tile + kr) ^ (i * LANES_K << 4)) + sub * MR * RROW);
    }
    // value columns j * MR .. of contraction step kk: raw codes, or the operand itself
    PCAMD_DEV uint4 value(const uint8_t* lds, uint32_t tile, int j, int kk) const {
      if constexpr (FP8) {
        constexpr int P = MR == 32 ? 8 : 16, C = MR / 16;
        const uint2 x = read_tr8(lds + ((tile + v) ^ (j % P * C << 4)) + kk * 16 * LROW + j / P * 256);
        return make_uint4(x.x, x.y, 0, 0);
      } else {
        constexpr int P = MR == 32 ? 4 : 8, C = MR / 8;
        const uint32_t c = j % P * C;
        // the second four tokens are QSTEP rows on, whose f differs in bit 1 (MR 32) or not at all
        const uint2 x = read_tr4(lds + ((tile + v) ^ (c << 4)) + kk * 16 * LROW + j / P * 256);
        const uint2 y = read_tr4(lds + ((tile + v) ^ ((MR == 32 ? c ^ 2 : c) << 4)) + (kk * 16 + M::QSTEP) * LROW + j / P * 256);
        return make_uint4(x.x, x.y, y.x, y.y);
      }
    }
  };

  static PCAMD_DEV void segment(const Args& a, uint8_t* lds, int64_t b, int rt, int s0, int n, int steps, int len,
                                int64_t slot, int wr, int wt, int h, int ln) {
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int row = rt * ROWS + wr * MR + ln;  // this lane's row
    const bool live = row < a.rows;
    const int tok_new = live ? row / a.heads : 0, head = live ? row % a.heads : 0;
    // Queries, in registers for the whole segment, in the order in which the
    // keys are read: 16 bytes of a key row a lane (with fp8 two steps' worth).
    uint4 ql[KL], qr[KR];
    {
      const uint16_t* p = static_cast<const uint16_t*>(a.q_latent) + b * a.qlb + tok_new * a.qls + head * a.qlh;
      const uint16_t* r = static_cast<const uint16_t*>(a.q_rope) + b * a.qrb + tok_new * a.qrs + head * a.qrh;
#pragma unroll
      for (int k = 0; k < KL; ++k) {
        const int at = FP8 ? (k / 2 * LANES_K + h) * 16 + k % 2 * 8 : (k * LANES_K + h) * 8;
        ql[k] = live ? *reinterpret_cast<const uint4*>(p + at) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < KR; ++k)
        qr[k] = live ? *reinterpret_cast<const uint4*>(r + k * M::K + 8 * h) : make_uint4(0, 0, 0, 0);
      // arrived before the loop: a wait inside it would wait for the copies too
#pragma unroll
      for (int k = 0; k < KL; ++k) asm volatile("" : "+v"(ql[k].x), "+v"(ql[k].y), "+v"(ql[k].z), "+v"(ql[k].w));
#pragma unroll
      for (int k = 0; k < KR; ++k) asm volatile("" : "+v"(qr[k].x), "+v"(qr[k].y), "+v"(qr[k].z), "+v"(qr[k].w));
    }
    const int limit = live ? len - a.new_tokens + 1 + tok_new : len;  // tokens this row sees
    const int all_see = len - a.new_tokens + 1;                       // tokens that every row sees
    const Lane L(lane);
    acc o[OB];
#pragma unroll
    for (int i = 0; i < OB; ++i) o[i] = acc{};
    float m = kNoMax, l = 0.0f;

    // ---- one tile of 32 tokens from tb on
    // Reads of LDS run a few steps ahead of the products that take them
    // (kAhead registers' worth), and sched_barrier keeps them there: left
    // alone, the scheduler saves registers by waiting for every read.
    auto compute = [&](uint32_t tile, int tb) {
      const float* scales = reinterpret_cast<const float*>(lds + tile + SCALES) + 4 * h;

      // ---- S^T: products n = 0 .. NA - 1, rotary steps first
      constexpr int PER_LOAD = FP8 ? 2 : 1;
      constexpr int LOADS = KR + KL / PER_LOAD, PER = KR + KL;
      constexpr int NA = SUB * PER, TA = SUB * LOADS;
      constexpr int DA = kAheadKeys<FP8> < TA ? kAheadKeys<FP8> : TA;
      uint4 raw[DA];
      auto load_key = [&](int i) {
        const int sub = i / LOADS, r = i % LOADS;
        return r < KR ? L.rope(lds, tile, sub, r) : L.key(lds, tile, sub, r - KR);
      };
      auto load_of = [](int n) { return n / PER * LOADS + (n % PER < KR ? n % PER : KR + (n % PER - KR) / PER_LOAD); };
      auto operand = [&](int n) {
        const uint4 x = raw[load_of(n) % DA];
        if constexpr (FP8) {
          if (n % PER >= KR) return (n % PER - KR) % 2 ? widen8(make_uint2(x.z, x.w)) : widen8(make_uint2(x.x, x.y));
        }
        return x;
      };
#pragma unroll
      for (int i = 0; i < DA; ++i) raw[i] = load_key(i);
      __builtin_amdgcn_sched_barrier(0);
      acc c[SUB], d[2];
      uint4 next = operand(0);
#pragma unroll
      for (int n = 0; n < NA; ++n) {
        const int sub = n / PER, r = n % PER;
        const uint4 x = next;
        if (n + 1 < NA) {
          if (load_of(n + 1) != load_of(n) && load_of(n) + DA < TA) raw[load_of(n) % DA] = load_key(load_of(n) + DA);
          next = operand(n + 1);
        }
        if (r < KR) {
          c[sub] = r == 0 ? S::first(x, qr[0]) : S::mul(x, qr[r], c[sub]);
        } else if constexpr (!FP8) {
          c[sub] = S::mul(x, ql[r - KR], c[sub]);
        } else {
          // a group's partial scores in d, scaled into c while the next group's are summed
          constexpr int G = KL / GROUPS;
          const int k = r - KR, g = k / G;
          if (k % G == 0) d[g & 1] = S::first(x, ql[k]);
          else if (k % G == 1 && g > 0) d[g & 1] = S::mul_holding(x, ql[k], d[g & 1], d[(g - 1) & 1]);
          else d[g & 1] = S::mul(x, ql[k], d[g & 1]);
          auto scale_in = [&](int group, int reg) {
            const int q = sub * (M::REGS / 4) + reg / 4;
            const float2 f = *reinterpret_cast<const float2*>(scales + group * TOK + q * M::QSTEP + reg % 4);
            c[sub][reg] += f.x * d[group & 1][reg];
            c[sub][reg + 1] += f.y * d[group & 1][reg + 1];
          };
          if (g > 0) {
            // from the group's third product on the last of the group before has been written
#pragma unroll
            for (int reg = 0; reg < M::REGS; reg += 2)
              if (2 + reg / 2 * (G - 2) / (M::REGS / 2) == k % G) scale_in(g - 1, reg);
          }
          if (r == PER - 1) {
            S::settle(d[g & 1]);
#pragma unroll
            for (int reg = 0; reg < M::REGS; reg += 2) scale_in(g, reg);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }

      // ---- the first values are on their way during the softmax
      constexpr int NP = OB * PK;  // products of the second kind: block n / PK, step n % PK
      constexpr int DV = kAheadValues<FP8> < NP ? kAheadValues<FP8> : NP;
      uint4 val[DV];
#pragma unroll
      for (int n = 0; n < DV; ++n) val[n] = L.value(lds, tile, n / PK, n % PK);
      if constexpr (!FP8) {
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub) S::settle(c[sub]);
      }
      __builtin_amdgcn_sched_barrier(0);

      // ---- softmax, one row a lane
      float s[QUADS * 4];
#pragma unroll
      for (int r = 0; r < QUADS * 4; ++r) s[r] = c[r / M::REGS][r % M::REGS] * a.scale_log2;
      if (tb + TOK > all_see) {
#pragma unroll
        for (int r = 0; r < QUADS * 4; ++r)
          s[r] = tb + (r / 4) * M::QSTEP + 4 * h + r % 4 < limit ? s[r] : -INFINITY;
      }
      float top = s[0];
#pragma unroll
      for (int r = 1; r < QUADS * 4; ++r) top = fmaxf(top, s[r]);
      top = row_max<MR>(top);
      if (__any(top > m + kSlack<DT, FP8>)) {
        const float to = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= alpha;
#pragma unroll
        for (int j = 0; j < OB; ++j) {
          // block by block through the vector registers, back to where the products keep it
          asm volatile("" : "+a"(o[j]));
          o[j] *= alpha;
          asm volatile("" : "+a"(o[j]));
        }
      }
#pragma unroll
      for (int r = 0; r < QUADS * 4; ++r) {
        s[r] = __builtin_amdgcn_exp2f(s[r] - m);
        l += s[r];
      }

      // ---- O^T += V^T P^T
      uint32_t p[2][PK * 4];  // P^T of a group of value columns, and of the next
      auto weights = [&](int g, int i) {  // dword i: registers 2 i and 2 i + 1
        float x0 = s[2 * i], x1 = s[2 * i + 1];
        if constexpr (FP8) {
          const float2 f = *reinterpret_cast<const float2*>(scales + g * TOK + (2 * i / 4) * M::QSTEP + 2 * i % 4);
          x0 *= f.x * kScaleUp<DT>;
          x1 *= f.y * kScaleUp<DT>;
        }
        p[g & 1][i] = Elem<DT>::narrow2(x0, x1);
      };
#pragma unroll
      for (int i = 0; i < PK * 4; ++i) weights(0, i);
      auto value_operand = [&](int n) {
        const uint4 x = val[n % DV];
        if constexpr (FP8) return widen8(make_uint2(x.x, x.y));
        else return x;
      };
      next = value_operand(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        constexpr int PER_GROUP = NP / (FP8 ? GROUPS : 1);
        const int j = n / PK, kk = n % PK, g = n / PER_GROUP;
        const uint4 x = next;
        if (n + DV < NP) val[n % DV] = L.value(lds, tile, (n + DV) / PK, (n + DV) % PK);
        if (n + 1 < NP) next = value_operand(n + 1);
        const uint32_t* w = p[g & 1] + 4 * kk;
        o[j] = M::mul(x, make_uint4(w[0], w[1], w[2], w[3]), o[j]);
        if constexpr (FP8) {
          if (g + 1 < GROUPS) {
#pragma unroll
            for (int i = 0; i < PK * 4; ++i)
              if (i * PER_GROUP / (PK * 4) == n % PER_GROUP) weights(g + 1, i);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    // ---- the loop over tiles, window by window of the page table
    const int32_t* table = a.table + b * a.table_stride;
    int32_t* pages = reinterpret_cast<int32_t*>(lds + BODY);
    const uint32_t ring = wt * NB * TILE;  // the dynamic LDS starts at address 0 (see decode_kernel)
    int done = len > 0 ? 0 : n;
    while (done < n) {
      const int first_t = (s0 + done) * STEP;
      Source src{pages, a.page_index(first_t), len};
      // steps whose tokens all lie within the window's pages (one at least:
      // a step is at most 128 tokens, the window 256 pages)
      const int64_t covered = (static_cast<int64_t>(src.first) + PAGES) * a.page;
      int upto = covered >= len ? n : static_cast<int>(covered / STEP) - s0;
      if (upto > n) upto = n;
      __syncthreads();
      {
        const int last = a.page_index(len - 1), at = src.first + tid;
        pages[tid] = table[at < last ? at : last];
      }
      __syncthreads();
      const int count = upto - done;
      auto start = [&](int i) {  // i: step of this window
        issue(a, src, ring + i % NB * TILE, (s0 + done + i) * STEP + wt * TOK, wr, lane);
      };
      auto wait = [&](int later) {  // copies of `later` further steps may be in flight
        if (NB > 2 && later >= 2) wait_copies<2 * COPIES <= 63 ? 2 * COPIES : 63>();
        else if (later == 1) wait_copies<COPIES>();
        else wait_copies<0>();
      };
      constexpr int AHEAD = WR > 1 ? NB - 1 : NB;
      static_assert(AHEAD <= 3 || WR == 1, "wait() counts up to two further steps");
      for (int i = 0; i < AHEAD && i < count; ++i) start(i);
      for (int i = 0; i < count; ++i) {
        const int later = count - 1 - i < AHEAD - 1 ? count - 1 - i : AHEAD - 1;
        wait(later);
        if constexpr (WR > 1) {
          // the tile is there for all waves, and all have left the one before it
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
          if (i + AHEAD < count) start(i + AHEAD);
        }
        const int tb = (s0 + done + i) * STEP + wt * TOK;
        if (WT == 1 || tb < len) compute(ring + i % NB * TILE, tb);
        if constexpr (WR == 1) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if (i + AHEAD < count) start(i + AHEAD);
        }
      }
      done = upto;
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
  // all of the kernel's LDS, so that it starts at address 0: copies and tile addresses count on it
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
