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
// fp16 has no room for scales of any size there: a wave takes the power of two
// out of its tile's largest scale of a group and widens the group's value codes
// times it instead, so that the weights stay p times a scale of one to two.
//
// What bounds it. With up to 16 rows the cache's bytes: 48 sequences of 32768
// tokens, 16 heads, bf16: 1.81 GB in 329 us, 5.5 TB/s. With 128 rows the
// products and the operands that they read from LDS, level with each other: 256
// sequences of 8192 tokens 974 TFLOP/s in whole tiles. Where sequences are cut
// into pieces, what a piece costs beside its steps: queries in, the first
// tokens' way, partial sums out and in again. 48 sequences of 1 to 5003 tokens,
// 128 heads: 63 us (34 of them in steps) and the joins 10; 19 of up to 6007
// tokens with 3 new ones each over an fp8 cache: 85 us, the steps' 60 bound by
// widening the codes.
#pragma once

#include "attn_common.h"
#include "latent_decode_args.h"

namespace pcamd {
namespace decode {

using namespace attn;

constexpr int NT = 256;
constexpr int TOK = 32;  // tokens of a wave's step
// 16 bytes of an output row, which is 8-byte aligned
typedef uint32_t u32x4_out __attribute__((ext_vector_type(4), aligned(8)));

// How far (log2) a score may pass the reference point of its row's weights
// before the reference moves and the wave's sums are rescaled. Weights and sums
// are floating point: bf16 and fp32 hold 2^40 as exactly as 1, so the first
// tile's maximum nearly always stays the reference. fp16 ends at 2^16:
// half of its room is left to an fp8 cache's scales past kTopUnit.
template <int DT>
constexpr float kSlack = DT == kF16 ? 8.0f : 40.0f;

// fp16 over an fp8 cache: bounds of the power of two that goes from a tile's
// scales to its value codes. Codes of up to 448 times 2^7 are finite in fp16;
// what is lost below its smallest number, 2^-25 of a value, the output loses too.
constexpr float kTopUnit = 128.0f, kLeastUnit = 0x1p-100f;

// Registers that hold operands read ahead of their products, in operands
template <bool FP8>
constexpr int kAheadKeys = FP8 ? 4 : 6;
constexpr int kAheadValues = 6;

// ---------------------------------------------------------------------------
// The division of the work. Few row tiles are cut one by one into equal pieces,
// one a workgroup. Many tiles are one list of units: for each sequence, for each tile
// of its rows, kFixed units for what a piece costs whatever its length (its
// queries, its output) and one for each step over the tokens. Workgroup w takes
// the w-th of `groups` equal pieces of the list, whatever the lengths are (with
// SPLIT, workgroups SPLIT w and on take its rows); what more than one piece has
// a part of, combine_kernel joins.
// ---------------------------------------------------------------------------
struct Division {
  int units, groups, q, r;
  PCAMD_DEV Division(int n, int g) : units(n), groups(g), q(n / g), r(n - n / g * g) {}
  PCAMD_DEV int first(int w) const { return w * q + (w < r ? w : r); }
  PCAMD_DEV int group_of(int u) const { return u < r * (q + 1) ? u / (q + 1) : r + (u - r * (q + 1)) / q; }
};

// Sequence b's tokens
PCAMD_DEV int length_of(const Args& a, int b) {
  const int n = a.lens[b];
  return n < 0 ? 0 : n > a.capacity ? a.capacity : n;
}
PCAMD_DEV int steps_of(int len, int step) { return len > step ? (len + step - 1) / step : 1; }

// sum of v over the workgroup's threads before this one, and over all of them
PCAMD_DEV int block_scan(int v, int* wave_total, int& total) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  int inc = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(inc, d, 64);
    if (lane >= d) inc += o;
  }
  if (lane == 63) wave_total[wave] = inc;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) before += wave_total[w];
    total += wave_total[w];
  }
  __syncthreads();
  return before + inc - v;
}

template <int DT, bool FP8, int DL, int DR, int MR, int WR, int SPLIT>
struct Kernel {
  static constexpr int WT = 4 / WR;
  static constexpr int STEP = TOK * WT;
  static constexpr int ROWS = MR * WR, TILE_ROWS = ROWS * SPLIT;
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
  // A tile of 32 tokens as it lies in LDS: the latent rows in blocks of 128
  // bytes, [block][token][128 bytes], then the rotary rows as one more block
  // (half filled where they are 64 bytes), and with fp8 the scales
  // [group][token].
  static constexpr int LROW = DL * (FP8 ? 1 : 2), BLOCKS = LROW / 128, BLOCK = TOK * 128;
  static constexpr int CR = DR / 8;  // 16-byte chunks of a rotary row
  static constexpr int ROPE = BLOCKS * BLOCK, SCALES = ROPE + BLOCK;
  static constexpr int TILE = SCALES + (FP8 ? TOK * GROUPS * 4 : 0);
  // Tiles per token group: all that fit, up to four
  static constexpr int FIT = 150000 / (WT * TILE);
  static constexpr int NB = FIT > 4 ? 4 : FIT;
  static_assert(NB >= (WR > 1 ? 2 : 1), "a shared ring needs two tiles");
  static constexpr int AHEAD = WR > 1 ? NB - 1 : NB;  // tiles on their way or in use
  // With 128 rows a workgroup and a 16-bit cache one tile's softmax overlaps the
  // next one's scores.
  static constexpr bool PIPE = MR == 32 && WR == 4 && !FP8;
  static_assert(!PIPE || NB == 4, "the overlapped loop holds two tiles while two more are on their way");
  static constexpr int PAGES = 256;  // page numbers kept in LDS
  static constexpr int RING = WT * NB * TILE;
  // epilogue, in the ring's place: what the waves of a row hand each other, and
  // whole rows on their way out
  static constexpr int OWN = OB / WT, QN = M::REGS / 4;  // blocks that a wave brings to their end; quads of a block
  static constexpr int PACK = OWN * QN * 64 * 16;        // what it gets from each of the others
  static constexpr int OUT_PITCH = OWN * MR * 2 + 16, STAGE = WT > 1 ? (WT - 1) * PACK : MR * OUT_PITCH;
  static_assert(STAGE >= MR * OUT_PITCH, "a wave's rows leave through what it was handed");
  static constexpr int EPI = 4 * STAGE + 4 * MR * 8 + 4 * MR * 8;
  // prologue, there too: each wave's query rows, [block][row][128 bytes]
  static constexpr int QBLOCKS = DL / 64, QBLOCK = MR * 128;
  static constexpr int QUERIES = (QBLOCKS + 1) * QBLOCK;
  static constexpr int BODY0 = RING > EPI ? RING : EPI;
  static constexpr int BODY = BODY0 > 4 * QUERIES ? BODY0 : 4 * QUERIES;
  static constexpr int LDS = BODY + PAGES * 4 + 64;  // and a few words of the division of the work

  // Chunk c of row t lies at c ^ f(t). Rows are 128 bytes apart, so t & 1 is a
  // half of the 256 bytes that 16 lanes may read without conflict, and the rest
  // of t has to spread 16 consecutive rows' equal chunks (keys) over all eight
  // places, and what a transposing read takes at once over disjoint ones:
  //   16-bit values: rows 4 h .. + 3 (MR 32: 64 bytes each; MR 16, two h: 32
  //   bytes each) - the reversed bits of t / 2;
  //   8-bit values: rows 4 h .. + 3 and QSTEP further on, 32 (16) bytes each.
  static PCAMD_DEV int swizzle(int t) {
    if constexpr (FP8) return ((t & 2) << 1) | (((t >> 2) ^ (t >> 3)) & 2) | ((t >> 2) & 1);
    else return swizzle16(t);
  }

  // ---- global -> LDS copies: 8 rows x 128 bytes each. The WR waves of a token
  // group share a tile's rows, and every wave issues the same number of copies
  // for every tile (past the last one too, of rows it has already), so a count
  // of copies in flight says which tiles have arrived.
  static constexpr int RW = TOK / WR, RR = RW / 8;             // a wave's rows of a tile, in eights
  static constexpr int S_LANES = FP8 ? TOK * GROUPS / WR : 0;  // scales of a wave
  static constexpr int S_COPIES = (S_LANES + 63) / 64;
  static constexpr int COPIES = RR * (BLOCKS + 1) + S_COPIES;
  static_assert((AHEAD - 1) * COPIES < 64, "the counter of copies in flight ends at 63");

  struct Source {
    const int32_t* pages;  // in LDS: the table from page number `first` on
    int first, last;       // last: the last token that they and the sequence hold
  };
  // Where a token is: its page's number and its place in the page. Cut to the
  // last token: what lies behind it is not read, and a row that is there twice
  // adds nothing, its second weight is zero.
  struct Place {
    uint32_t page, place;
    PCAMD_DEV void find(const Args& a, const Source& src, int t) {
      t = t < src.last ? t : src.last;
      const int n = a.page_index(t);
      page = static_cast<uint32_t>(src.pages[n - src.first]);
      place = t - n * a.page;
    }
    PCAMD_DEV uint64_t at(const Args& a, uint32_t page_stride, uint32_t token_stride) const {
      return uint64_t{page < a.pages ? page : a.pages - 1} * page_stride + uint64_t{place} * token_stride;
    }
  };

  // the addresses of a tile's copies, and the copies
  struct Copies {
    const uint8_t* latent[RR];
    const uint8_t* rope[RR];
    const float* scale[S_COPIES > 0 ? S_COPIES : 1];

    Place of_row[RR], of_scale[S_COPIES > 0 ? S_COPIES : 1];
    uint32_t rotation;  // a multiple of 256 bytes where a row has so many
    PCAMD_DEV explicit Copies(int wave) : rotation(wave * (BLOCKS > 4 ? 2 : 1)) {}

    // in two parts: the page numbers come from LDS, and the first part's reads have arrived when the second uses them
    PCAMD_DEV void find(const Args& a, const Source& src, int t0, int wr, int lane) {
#pragma unroll
      for (int i = 0; i < RR; ++i) of_row[i].find(a, src, t0 + wr * RW + 8 * i + lane / 8);
#pragma unroll
      for (int i = 0; i < S_COPIES; ++i) of_scale[i].find(a, src, t0 + (wr * S_LANES + i * 64 + lane) % TOK);
    }
    PCAMD_DEV void address(const Args& a, int wr, int lane) {
#pragma unroll
      for (int i = 0; i < RR; ++i) {
        const int c = (lane % 8) ^ swizzle(wr * RW + 8 * i + lane / 8);
        latent[i] = static_cast<const uint8_t*>(a.latent) + of_row[i].at(a, a.slp, a.slt) * (FP8 ? 1 : 2) + 16 * c;
        rope[i] = c < CR ? static_cast<const uint8_t*>(a.rope) + of_row[i].at(a, a.srp, a.srt) * 2 + 16 * c : nullptr;
      }
#pragma unroll
      for (int i = 0; i < S_COPIES; ++i)  // [group][token]
        scale[i] = a.scale + of_scale[i].at(a, a.ssp, a.sst) + (wr * S_LANES + i * 64 + lane) / TOK;
    }
    PCAMD_DEV void prepare(const Args& a, const Source& src, int t0, int wr, int lane) {
      find(a, src, t0, wr, lane);
      address(a, wr, lane);
    }
    PCAMD_DEV void emit_latent(uint32_t tile, int wr, int i, uint32_t block) const {  // eight rows' 128 bytes
      copy16(latent[i] + block * 128, tile + block * BLOCK + (wr * RW + 8 * i) * 128);
    }
    PCAMD_DEV void emit_rope(uint32_t tile, int wr, int i) const {
      if (CR == 8 || rope[i]) copy16(rope[i], tile + ROPE + (wr * RW + 8 * i) * 128);
    }
    PCAMD_DEV void emit_scale(uint32_t tile, int wr, int lane, int i) const {
      if (S_LANES % 64 == 0 || i * 64 + lane < S_LANES) copy4(scale[i], tile + SCALES + (wr * S_LANES + i * 64) * 4);
    }
    // Copy k of COPIES into the tile at LDS address `tile`. The latent rows'
    // blocks come in an order that starts elsewhere in every wave: eight rows'
    // equal 128 bytes lie in few memory channels, and waves that asked for the
    // same block at the same time would leave the other channels idle.
    template <int K>
    PCAMD_DEV void emit(uint32_t tile, int wr, int lane) const {
      if constexpr (K < RR * BLOCKS) emit_latent(tile, wr, K / BLOCKS, (K + rotation) % BLOCKS);
      else if constexpr (K < RR * (BLOCKS + 1)) emit_rope(tile, wr, K - RR * BLOCKS);
      else emit_scale(tile, wr, lane, K - RR * (BLOCKS + 1));
    }
    template <int K = 0>
    PCAMD_DEV void emit_all(uint32_t tile, int wr, int lane) const {
      if constexpr (K < COPIES) {
        emit<K>(tile, wr, lane);
        emit_all<K + 1>(tile, wr, lane);
      }
    }
    // the copies that step n of `steps` gives time for: from step 8 on, evenly
    template <int K = 0>
    PCAMD_DEV void emit_at(int n, int steps, uint32_t tile, int wr, int lane) const {
      if constexpr (K < COPIES) {
        if (8 + K * (steps - 9) / COPIES == n) emit<K>(tile, wr, lane);
        emit_at<K + 1>(n, steps, tile, wr, lane);
      }
    }
  };

  // 8 fp8 codes as 16-bit elements, times a power of two
  static PCAMD_DEV uint4 widen8(uint2 c, float unit = 1.0f) {
    return make_uint4(widen2<DT, false>(c.x, unit), widen2<DT, true>(c.x, unit), widen2<DT, false>(c.y, unit),
                      widen2<DT, true>(c.y, unit));
  }
  static constexpr bool UNITS = FP8 && DT == kF16;  // value codes times a power of two of their tile and group

  // Where this lane reads in a tile. Chunks of a row lie at c ^ f(row), so
  // another chunk's place differs by an exclusive or with a constant (bits 4-6
  // of the address), another block's by a constant to add.
  struct Lane {
    int h, ln;
    uint32_t k, v;
    PCAMD_DEV explicit Lane(int lane) : h(lane / MR), ln(lane % MR) {
      const int i16 = lane % 16, g16 = lane / 16;
      k = ln * 128 + ((h ^ swizzle(ln)) << 4);
      // the transposing read's row, and its chunk's part that is the lane's
      const int t = FP8 ? (i16 >> 3) * M::QSTEP + 4 * h + ((i16 >> 1) & 3) : 4 * h + (i16 >> 2);
      const int c = FP8 ? (MR == 32 ? g16 & 1 : 0) : (MR == 32 ? 2 * (g16 & 1) : 0) + ((i16 >> 1) & 1);
      v = t * 128 + ((c ^ swizzle(t)) << 4) + 8 * (i16 & 1);
    }
    // 16 bytes of a token's latent (rotary) row, as step i reads them; token MR * sub + ln
    PCAMD_DEV uint4 key(const uint8_t* lds, uint32_t tile, int sub, int i) const {
      constexpr int P = 8 / LANES_K;
      // 16 rows on, f is the same (16-bit rows) or differs in bit 1
      const int x = (i % P * LANES_K ^ (FP8 && sub ? 2 : 0)) << 4;
      return *reinterpret_cast<const uint4*>(lds + ((tile + k) ^ x) + i / P * BLOCK + sub * MR * 128);
    }
    PCAMD_DEV uint4 rope(const uint8_t* lds, uint32_t tile, int sub, int i) const {
      const int x = (i * LANES_K ^ (FP8 && sub ? 2 : 0)) << 4;
      return *reinterpret_cast<const uint4*>(lds + ((tile + k) ^ x) + ROPE + sub * MR * 128);
    }
    // value columns j * MR .. of contraction step kk: raw codes, or the operand itself
    PCAMD_DEV uint4 value(const uint8_t* lds, uint32_t tile, int j, int kk) const {
      if constexpr (FP8) {
        const int c = j * (MR / 16), x = (c % 8 ^ (kk ? 2 : 0)) << 4;
        const uint2 y = read_tr8(lds + ((tile + v) ^ x) + c / 8 * BLOCK + kk * 16 * 128);
        return make_uint4(y.x, y.y, 0, 0);
      } else {
        const int c = j * (MR / 8), x = c % 8 << 4, at = c / 8 * BLOCK + kk * 16 * 128;
        // the second four tokens are QSTEP rows on: 8 rows change bit 0 of f, 16 do not
        const uint2 y = read_tr4(lds + ((tile + v) ^ x) + at);
        const uint2 z = read_tr4(lds + ((tile + v) ^ (MR == 32 ? x ^ 16 : x)) + at + M::QSTEP * 128);
        return make_uint4(y.x, y.y, z.x, z.y);
      }
    }
  };

  static PCAMD_DEV void run(const Args& a, uint8_t* lds) {
    int* wave_total = reinterpret_cast<int*>(lds + BODY + PAGES * 4);
    int* found = wave_total + NT / 64;
    const int tid = threadIdx.x;

    // ---- this workgroup's piece: steps [in_seq, in_seq + end - begin) of
    // sequence b's row tiles one after the other, and of the sequences behind it
    const int tiles = a.batch * a.row_tiles;
    int b, in_seq, begin, end, w, share, FIXED = 0;
    auto take_place = [&](int groups) {  // false: nothing to do here
      const int wgs = groups * SPLIT, eighth = (wgs + 8 * SPLIT - 1) / (8 * SPLIT) * SPLIT;
      // Neighbouring pieces belong to the same sequence, and a piece's workgroups
      // read the same tokens at the same time: put them on the same XCD (workgroups
      // go round the eight of them), whose L2 then holds its queries and the tokens.
      int place = blockIdx.x;
      if (8 * eighth <= static_cast<int>(gridDim.x) && place < 8 * eighth) place = place % 8 * eighth + place / 8;
      w = place / SPLIT;
      share = place % SPLIT * ROWS;  // its first row of the tile
      if (place < wgs) return true;
      if (a.parts && tid == 0) a.joins[w] = make_int4(0, 0, -1, 0);
      return false;
    };
    if (few_tiles(tiles, SPLIT)) {
      // Each row tile alone, in equal pieces of up to `most` steps. Every wave
      // works it out for itself, a lane a sequence.
      const int lane = tid % 64;
      const int len = lane < a.batch ? length_of(a, lane) : 0, steps = lane < a.batch ? steps_of(len, STEP) : 0;
      int all = steps;
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) all += __shfl_xor(all, d, 64);
      const int spare = kWorkgroups / SPLIT - tiles;  // sum ceil(steps / most) <= sum steps / most + tiles
      int most = (all * a.row_tiles + spare - 1) / spare;
      if (most < a.min_steps) most = a.min_steps;
      const int pieces = (steps + most - 1) / most;
      int upto = pieces * a.row_tiles;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d, 64);
        if (lane >= d) upto += o;
      }
      if (!take_place(__builtin_amdgcn_readlane(upto, 63))) return;
      b = __popcll(__ballot(upto <= w));
      const int of_b = __builtin_amdgcn_readlane(pieces, b), steps_b = __builtin_amdgcn_readlane(steps, b);
      const int at = w - (__builtin_amdgcn_readlane(upto, b) - of_b * a.row_tiles), rt = at / of_b, i = at - rt * of_b;
      const int q = steps_b / of_b, r = steps_b - q * of_b;
      begin = 0;
      end = q + (i < r);
      in_seq = rt * steps_b + i * q + (i < r ? i : r);
      // the second piece's workgroup notes which tile it is and the last piece's workgroup
      if (a.parts && tid == 0 && share == 0)
        a.joins[w] = i == 1 ? make_int4(b, rt, 1, w + of_b - 2) : make_int4(0, 0, -1, 0);
    } else {
      int sum = 0, steps_all;
      for (int i = tid; i < a.batch; i += NT) sum += steps_of(length_of(a, i), STEP);
      int before = block_scan(sum, wave_total, steps_all);
      steps_all = __builtin_amdgcn_readfirstlane(steps_all);
      const int wanted = (steps_all * a.row_tiles + a.min_steps - 1) / a.min_steps;
      int groups = wanted > tiles ? wanted : tiles;
      if (groups > a.groups) groups = a.groups;
      FIXED = kFixed<MR, SPLIT>;
      const Division div(a.row_tiles * (steps_all + a.batch * FIXED), groups);
      if (!take_place(groups)) return;
      begin = div.first(w);
      end = div.first(w + 1);
      int base = 0;
      for (int b0 = 0; b0 < a.batch; b0 += NT) {
        const int i = b0 + tid;
        const int mine = i < a.batch ? (steps_of(length_of(a, i), STEP) + FIXED) * a.row_tiles : 0;
        int total;
        if (a.batch <= NT) before = (before + tid * FIXED) * a.row_tiles;  // the first scan's answer, where it had one sequence a thread
        else before = base + block_scan(mine, wave_total, total);
        if (mine && begin >= before && begin < before + mine) {
          found[0] = i;
          found[1] = begin - before;
        }
        if (a.batch > NT) {
          base += total;
          if (base > begin) break;
        }
      }
      __syncthreads();
      // in scalar registers, as all that steers the segments: branches on them are scalar branches
      b = __builtin_amdgcn_readfirstlane(found[0]);
      in_seq = __builtin_amdgcn_readfirstlane(found[1]);
      if (a.parts && tid == 0 && share == 0) {
        // Where pieces meet: the first workgroup that starts inside a (sequence,
        // row tile) notes which it is and which workgroup holds the last piece;
        // the one before it holds the first.
        const int tile = steps_of(length_of(a, b), STEP) + FIXED;
        const int in_tile = in_seq % tile, real = begin - in_tile + FIXED;  // its first step's unit
        a.joins[w] = begin > real && div.first(w - 1) <= real
                         ? make_int4(b, in_seq / tile, 1, div.group_of(real + tile - FIXED - 1))
                         : make_int4(0, 0, -1, 0);
      }
    }

    for (int u = begin; u < end;) {
      const int len = length_of(a, b);
      const int steps = steps_of(len, STEP), tile = steps + FIXED;
      const int rt = in_seq / tile, at = in_seq - rt * tile;
      const int n = end - u < tile - at ? end - u : tile - at;
      const int s0 = at > FIXED ? at - FIXED : 0, s1 = at + n - FIXED;
      const int row0 = rt * TILE_ROWS + share;
      if (s1 > s0 && row0 < a.rows) segment(a, lds, b, row0, share, s0, s1 - s0, steps, len, s0 > 0 ? 2 * w : 2 * w + 1);
      u += n;
      in_seq += n;
      if (in_seq >= tile * a.row_tiles) {
        ++b;
        in_seq = 0;
      }
    }
  }

  // Steps s0 .. s0 + n - 1 of a row tile's `steps`.
  static PCAMD_DEV void segment(const Args& a, uint8_t* lds, int b, int row0, int share, int s0, int n, int steps,
                                int len, int slot) {
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wr = wave % WR, wt = wave / WR;
    const Lane L(lane);
    const int h = L.h, ln = L.ln;
    const int row = row0 + wr * MR + ln;  // this lane's row
    const bool live = row < a.rows;
    const int tok_new = live ? row / a.heads : 0, head = live ? row % a.heads : 0;

    // ---- the page numbers and the queries, then the first tiles. Queries stay
    // in registers for the whole segment, in the order in which the keys are
    // read: 16 bytes of a key row a lane (with fp8 two products' worth).
    const int32_t* table = a.table + static_cast<int64_t>(b) * a.table_stride;
    int32_t* pages = reinterpret_cast<int32_t*>(lds + BODY);
    Source src{pages, 0, 0};
    int done = len > 0 ? 0 : n, upto = n;  // steps behind and, with the pages at hand, ahead of the loop
    auto window = [&]() {                  // this thread's entry of the page numbers from step `done` on
      src.first = a.page_index((s0 + done) * STEP);
      // A step is at most 128 tokens and a window 256 pages, so it covers one at least.
      const int64_t covered = (static_cast<int64_t>(src.first) + PAGES) * a.page;
      src.last = (covered < len ? static_cast<int>(covered) : len) - 1;
      upto = covered >= len ? n : static_cast<int>(covered / STEP) - s0;
      if (upto > n) upto = n;
      const int last = a.page_index(len - 1), at = src.first + tid;
      return table[at < last ? at : last];
    };
    int entry = 0;
    if (len > 0) entry = window();
    // The queries pass through LDS: whole 128-byte lines come in, and a lane
    // takes its row's pieces from there.
    {
      const uint32_t to = wave * QUERIES;
#pragma unroll
      for (int i = 0; i < MR / 8; ++i) {
        const int r = 8 * i + lane / 8, c = (lane % 8) ^ swizzle16(r);
        int from = row0 + wr * MR + r;
        if (from >= a.rows) from = a.rows - 1;  // a spare row computes what another one does, and is not stored
        const int tn = from / a.heads, hd = from - tn * a.heads;
        const uint16_t* p = static_cast<const uint16_t*>(a.q_latent) + b * a.qlb + tn * a.qls + hd * a.qlh + 8 * c;
#pragma unroll
        for (int k = 0; k < QBLOCKS; ++k) {
          const uint32_t blk = (k + 2 * wave) % QBLOCKS;  // in another order in every wave, as the tiles' copies
          copy16(p + blk * 64, to + blk * QBLOCK + 8 * i * 128);
        }
        if (c < CR)
          copy16(static_cast<const uint16_t*>(a.q_rope) + b * a.qrb + tn * a.qrs + hd * a.qrh + 8 * c,
                    to + QBLOCKS * QBLOCK + 8 * i * 128);
      }
    }
    wait_copies<0>();
    uint4 ql[KL], qr[KR];
    {
      const uint8_t* from = lds + wave * QUERIES + ln * 128;
      auto piece = [&](int c) {  // c: a constant and h
        return *reinterpret_cast<const uint4*>(from + c / 8 * QBLOCK + ((c % 8 ^ swizzle16(ln)) << 4));
      };
#pragma unroll
      for (int k = 0; k < KL; ++k) ql[k] = piece(FP8 ? 2 * (k / 2 * LANES_K + h) + k % 2 : k * LANES_K + h);
#pragma unroll
      for (int k = 0; k < KR; ++k) qr[k] = piece(QBLOCKS * 8 + k * LANES_K + h);
#pragma unroll
      for (int k = 0; k < KL; ++k) asm volatile("" : "+v"(ql[k].x), "+v"(ql[k].y), "+v"(ql[k].z), "+v"(ql[k].w));
#pragma unroll
      for (int k = 0; k < KR; ++k) asm volatile("" : "+v"(qr[k].x), "+v"(qr[k].y), "+v"(qr[k].z), "+v"(qr[k].w));
    }
    __syncthreads();  // the tiles take the queries' place
    const int limit = live ? len - a.new_tokens + 1 + tok_new : len;  // tokens this row sees
    const int all_see = len - a.new_tokens + 1;                       // tokens that every row sees
    const uint32_t ring = wt * NB * TILE;  // the dynamic LDS starts at address 0 (see decode_kernel)
    auto tile_of = [&](int i) { return ring + static_cast<uint32_t>(i % NB) * TILE; };
    auto first_token = [&](int i) { return (s0 + done + i) * STEP + wt * TOK; };  // of this wave in step i of the window
    auto start = [&]() {
      pages[tid] = entry;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        Copies c(wave);
        c.prepare(a, src, first_token(i), wr, lane);
        c.emit_all(tile_of(i), wr, lane);
      }
    };
    if (len > 0) start();
    acc o[OB];
#pragma unroll
    for (int i = 0; i < OB; ++i) o[i] = acc{};
    float m = kNoMax, l = 0.0f;

    // ---- The parts of a step. Reads of LDS run a few products ahead of those
    // that take them, and sched_barrier keeps them there: left alone, the
    // scheduler saves registers by waiting for every read. `beside(i)` is other
    // work for the time of product i.
    constexpr int PER_LOAD = FP8 ? 2 : 1;
    constexpr int LOADS = KR + KL / PER_LOAD, PER = KR + KL;
    constexpr int NA = SUB * PER, TA = SUB * LOADS;  // products of S^T, rotary ones first; their loads
    constexpr int NP = OB * PK;                      // products of O^T: block n / PK, step n % PK
    constexpr int DV = kAheadValues < NP ? kAheadValues : NP;
    uint4 val[DV];
    auto scores = [&](uint32_t tile, acc (&c)[SUB], auto beside) {
      const float* scales = reinterpret_cast<const float*>(lds + tile + SCALES) + 4 * h;
      constexpr int DA = kAheadKeys<FP8> < TA ? kAheadKeys<FP8> : TA;
      uint4 raw[DA];
      auto load_key = [&](int i) {
        const int sub = i / LOADS, r = i % LOADS;
        return r < KR ? L.rope(lds, tile, sub, r) : L.key(lds, tile, sub, r - KR);
      };
      auto load_of = [](int k) { return k / PER * LOADS + (k % PER < KR ? k % PER : KR + (k % PER - KR) / PER_LOAD); };
      auto operand = [&](int k) {
        const uint4 x = raw[load_of(k) % DA];
        if constexpr (FP8) {
          if (k % PER >= KR) return (k % PER - KR) % 2 ? widen8(make_uint2(x.z, x.w)) : widen8(make_uint2(x.x, x.y));
        }
        return x;
      };
#pragma unroll
      for (int i = 0; i < DA; ++i) raw[i] = load_key(i);
      __builtin_amdgcn_sched_barrier(0);
      acc d[2];
      float4 f;  // four tokens' scales of a group, read a step before their use
      uint4 next = operand(0);
      unrolled<NA>([&](auto number) {
        constexpr int k = decltype(number)::value, sub = k / PER, r = k % PER;
        const uint4 x = next;
        if (k + 1 < NA) {
          if (load_of(k + 1) != load_of(k) && load_of(k) + DA < TA) raw[load_of(k) % DA] = load_key(load_of(k) + DA);
          next = operand(k + 1);
        }
        if constexpr (r < KR) {
          c[sub] = r == 0 ? S::first(x, qr[0]) : S::mul(x, qr[r], c[sub]);
        } else if constexpr (!FP8) {
          c[sub] = S::mul(x, ql[r - KR], c[sub]);
        } else {
          // a group's partial scores in d, scaled into c while the next group's are summed
          constexpr int G = KL / GROUPS;
          constexpr int i = r - KR, g = i / G;
          if (i % G == 0) d[g & 1] = S::first(x, ql[i]);
          else if (i % G == 1 && g > 0) d[g & 1] = S::mul_holding(x, ql[i], d[g & 1], d[(g - 1) & 1]);
          else d[g & 1] = S::mul(x, ql[i], d[g & 1]);
          constexpr int QD = M::REGS / 4;  // quads of a sum
          auto scales_of = [&](int group, int q) {
            return *reinterpret_cast<const float4*>(scales + group * TOK + (sub * QD + q) * M::QSTEP);
          };
          auto scale_in = [&](int group, int q, float4 x) {
            c[sub][4 * q] += x.x * d[group & 1][4 * q];
            c[sub][4 * q + 1] += x.y * d[group & 1][4 * q + 1];
            c[sub][4 * q + 2] += x.z * d[group & 1][4 * q + 2];
            c[sub][4 * q + 3] += x.w * d[group & 1][4 * q + 3];
          };
          // from the group's third product on the last of the group before has been written
#pragma unroll
          for (int q = 0; q < QD; ++q) {
            const int at = 2 + q * (G - 2) / QD;
            if (g > 0 && at == i % G) scale_in(g - 1, q, f);
          }
#pragma unroll
          for (int q = 0; q < QD; ++q) {
            const int at = 2 + q * (G - 2) / QD;
            if (g > 0 && at == i % G + 1) f = scales_of(g - 1, q);
          }
          if (r == PER - 1) {
            float4 last[QD];
#pragma unroll
            for (int q = 0; q < QD; ++q) last[q] = scales_of(g, q);
            S::settle(d[g & 1]);
#pragma unroll
            for (int q = 0; q < QD; ++q) scale_in(g, q, last[q]);
          }
        }
        beside(k);
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    auto first_values = [&](uint32_t tile) {
#pragma unroll
      for (int k = 0; k < DV; ++k) val[k] = L.value(lds, tile, k / PK, k % PK);
    };
    auto settle = [&](acc (&c)[SUB]) {
      if constexpr (!FP8) {
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub) S::settle(c[sub]);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    // The powers of two in a tile's scales. Each lane takes one or two of them, and
    // 16 lanes have what belongs to one group. Exponents compare as integers.
    float unit[UNITS ? GROUPS : 1];
    uint32_t exponent = 0;
    auto find_unit = [&](uint32_t tile) {
      const uint32_t* at = reinterpret_cast<const uint32_t*>(lds + tile + SCALES) + lane * (GROUPS / 2);
      exponent = at[0] & 0x7f800000u;
      if constexpr (GROUPS == 4) {
        const uint32_t other = at[1] & 0x7f800000u;
        exponent = exponent > other ? exponent : other;
      }
    };
    auto set_unit = [&]() {
      unrolled<4>([&](auto n) {  // rotations by 1, 2, 4 and 8 within 16 lanes
        const uint32_t other = __builtin_amdgcn_update_dpp(0, exponent, 0x120 + (1 << decltype(n)::value), 0xf, 0xf, true);
        exponent = exponent > other ? exponent : other;
      });
      constexpr uint32_t least = __builtin_bit_cast(uint32_t, kLeastUnit), most = __builtin_bit_cast(uint32_t, kTopUnit);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        uint32_t top = least;
#pragma unroll
        for (int i = 0; i < 4 / GROUPS; ++i) {
          const uint32_t part = __builtin_amdgcn_readlane(exponent, 64 / GROUPS * g + 16 * i);
          top = top > part ? top : part;
        }
        unit[g] = __uint_as_float(top < most ? top : most);
      }
    };
    float s[QUADS * 4];
    auto mask = [&](int tb) {
#pragma unroll
      for (int r = 0; r < QUADS * 4; ++r) s[r] = tb + (r / 4) * M::QSTEP + 4 * h + r % 4 < limit ? s[r] : -INFINITY;
    };
    auto maximum = [&]() {
      float top = s[0];
#pragma unroll
      for (int r = 1; r < QUADS * 4; ++r) top = fmaxf(top, s[r]);
      return top;
    };
    auto refer = [&](float top) {  // top: of the row
      if (__any(top > m + kSlack<DT>)) {
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
    };
    uint32_t p[FP8 ? 2 : 1][PK * 4];  // P^T of a group of value columns, and of the next
    float4 fw;                        // with fp8: the scales of a quad of the weights' tokens
    auto scales_of_weights = [&](uint32_t tile, int g, int q) {
      if constexpr (FP8)
        fw = *reinterpret_cast<const float4*>(lds + tile + SCALES + 4 * (4 * h + g * TOK + q * M::QSTEP));
    };
    auto weights = [&](int g, int q) {  // registers 4 q .. + 3
      float x0 = s[4 * q], x1 = s[4 * q + 1], x2 = s[4 * q + 2], x3 = s[4 * q + 3];
      if constexpr (UNITS) {
        const float per = __uint_as_float((254u << 23) - __float_as_uint(unit[g]));  // 1 / unit
        x0 *= fw.x * per;
        x1 *= fw.y * per;
        x2 *= fw.z * per;
        x3 *= fw.w * per;
      } else if constexpr (FP8) {
        x0 *= fw.x;
        x1 *= fw.y;
        x2 *= fw.z;
        x3 *= fw.w;
      }
      p[FP8 ? g & 1 : 0][2 * q] = Elem<DT>::narrow2(x0, x1);
      p[FP8 ? g & 1 : 0][2 * q + 1] = Elem<DT>::narrow2(x2, x3);
    };
    auto values = [&](uint32_t tile, auto beside) {  // O^T += V^T P^T
      auto operand = [&](int k) {
        const uint4 x = val[k % DV];
        if constexpr (UNITS) return widen8(make_uint2(x.x, x.y), unit[k * GROUPS / NP]);
        else if constexpr (FP8) return widen8(make_uint2(x.x, x.y));
        else return x;
      };
      uint4 next = operand(0);
      unrolled<NP>([&](auto number) {
        constexpr int PER_GROUP = NP / (FP8 ? GROUPS : 1);
        constexpr int k = decltype(number)::value, j = k / PK, kk = k % PK, g = FP8 ? k / PER_GROUP : 0;
        const uint4 x = next;
        if (k + DV < NP) val[k % DV] = L.value(lds, tile, (k + DV) / PK, (k + DV) % PK);
        if (k + 1 < NP) next = operand(k + 1);
        const uint32_t* w = p[g & 1] + 4 * kk;
        o[j] = M::mul(x, make_uint4(w[0], w[1], w[2], w[3]), o[j]);
        if constexpr (FP8) {
          if (g + 1 < GROUPS) {
            // a quad of the next group's weights, its scales read a product before
#pragma unroll
            for (int q = 0; q < QUADS; ++q) {
              if (q * PER_GROUP / QUADS == k % PER_GROUP) scales_of_weights(tile, g + 1, q);
              if (q * PER_GROUP / QUADS + 1 == k % PER_GROUP) weights(g + 1, q);
            }
          }
        }
        beside(k);
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    auto nothing = [](int) {};

    // ---- the loop over steps, window by window of the page table
    while (done < n) {
      if (done > 0) {
        __syncthreads();
        entry = window();
        start();
      }
      const int count = upto - done;
      if constexpr (PIPE) {
        acc c[1];
        auto to_scores = [&](int k) { s[k] = c[0][k] * a.scale_log2; };
        auto look = [&](int i, float top) {  // before step i's weights: its mask and reference point; top: the row's
          const int tb = first_token(i);
          if (tb + TOK > all_see) {
            mask(tb);
            top = row_max<MR>(maximum());
          }
          refer(top);
        };
        wait_copies<(AHEAD - 1) * COPIES>();
        tile_barrier();
        scores(tile_of(0), c, nothing);
        settle(c);
#pragma unroll
        for (int k = 0; k < 16; ++k) to_scores(k);
        look(0, row_max<MR>(maximum()));
        auto step = [&](int i, auto more) {
          constexpr bool MORE = decltype(more)::value;  // another step follows
          auto weigh = [&](int k) { s[k] = __builtin_amdgcn_exp2f(s[k] - m); };  // element k of step i's weights
          auto add = [&](int k) {
            l += s[k];
            if (k % 4 == 3) weights(0, k / 4);
          };
          if constexpr (MORE) {
            wait_copies<(AHEAD - 2) * COPIES>();
            tile_barrier();
            Copies copies(wave);
            scores(tile_of(i + 1), c, [&](int k) {
              if (k == 1) copies.find(a, src, first_token(i + AHEAD), wr, lane);
              if (k == 6) copies.address(a, wr, lane);
              copies.emit_at(k, NA, tile_of(i + AHEAD), wr, lane);
              constexpr int EVERY = NA / 16;  // products an element
              if (k % EVERY == 0 && k / EVERY < 16) weigh(k / EVERY);
              if (k % EVERY == EVERY - 1 && k / EVERY < 16) add(k / EVERY);
              if (k == NA - 3) first_values(tile_of(i));
            });
            settle(c);
            float top = kNoMax;
            values(tile_of(i), [&](int k) {
              constexpr int EACH = NP < 32 ? 2 : 1;  // elements a product, from the second on
              if (k > 0 && (k - 1) * EACH < 16) {
#pragma unroll
                for (int e = (k - 1) * EACH; e < k * EACH; ++e) to_scores(e);
              }
              if (k > 1 && (k - 2) * EACH < 16) {
#pragma unroll
                for (int e = (k - 2) * EACH; e < (k - 1) * EACH; ++e) top = fmaxf(top, s[e]);
              }
              if (k == 16 / EACH + 3) top = row_max<MR>(top);
            });
            look(i + 1, top);
          } else {
            first_values(tile_of(i));
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              weigh(k);
              add(k);
            }
            values(tile_of(i), nothing);
          }
        };
        for (int i = 0; i + 1 < count; ++i) step(i, std::true_type{});
        step(count - 1, std::false_type{});
      } else {
        for (int i = 0; i < count; ++i) {
          wait_copies<(AHEAD - 1) * COPIES>();
          if constexpr (WR > 1) tile_barrier();
          const uint32_t tile = tile_of(i);
          const int tb = first_token(i);
          Copies copies(wave);
          acc c[SUB];
          // (in waves of 32 rows an fp8 cache leaves no registers for it beside the scores)
          if constexpr (WR > 1 && MR == 32 && FP8) {
            copies.prepare(a, src, first_token(i + AHEAD), wr, lane);
            copies.emit_all(tile_of(i + AHEAD), wr, lane);
          }
          auto ahead = [&](int k) {
            if constexpr (UNITS) {
              if (k == 2) find_unit(tile);
              if (k == 8) set_unit();
            }
            if constexpr (MR == 16 || !FP8) {
              if (k == 1) copies.find(a, src, first_token(i + AHEAD), wr, lane);
              if (k == 6) copies.address(a, wr, lane);
              if constexpr (WR > 1) copies.emit_at(k, NA, tile_of(i + AHEAD), wr, lane);
            }
          };
          scores(tile, c, ahead);
          first_values(tile);
          settle(c);
#pragma unroll
          for (int r = 0; r < QUADS * 4; ++r) s[r] = c[r / M::REGS][r % M::REGS] * a.scale_log2;
          if (tb + TOK > all_see) mask(tb);
          refer(row_max<MR>(maximum()));
#pragma unroll
          for (int r = 0; r < QUADS * 4; ++r) {
            s[r] = __builtin_amdgcn_exp2f(s[r] - m);
            l += s[r];
          }
#pragma unroll
          for (int q = 0; q < QUADS; ++q) {
            scales_of_weights(tile, 0, q);
            weights(0, q);
          }
          const uint32_t into = tile_of(i + AHEAD);
          values(tile, [&](int k) {
            if constexpr (WR == 1) {
              // A wave of its own refills what it has read: the rotary rows
              // during the first block's products, each block of the latent rows
              // during the next one's.
              constexpr int SB = NP / BLOCKS;  // products of a block
#pragma unroll
              for (int r = 0; r < RR; ++r) {
                if (r * SB / RR + (SB > RR ? 1 : 0) != k % SB) continue;
                if (k < SB) copies.emit_rope(into, wr, r);
                else copies.emit_latent(into, wr, r, k / SB - 1);
              }
            }
          });
          if constexpr (WR == 1) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int r = 0; r < RR; ++r) copies.emit_latent(into, wr, r, BLOCKS - 1);
#pragma unroll
            for (int r = 0; r < S_COPIES; ++r) copies.emit_scale(into, wr, lane, r);
          }
        }
      }
      wait_copies<0>();  // the copies past the last step: LDS has other uses next
      done = upto;
    }
    l = row_sum<MR>(l);

    // ---- epilogue. The WT waves of a row split its columns: each hands the
    // others their blocks through LDS and adds up its own.
    const bool whole = n == steps;
    float2* ml = reinterpret_cast<float2*>(lds + 4 * STAGE);                     // of each wave's rows
    int64_t* place = reinterpret_cast<int64_t*>(lds + 4 * STAGE + 4 * MR * 8) + wave * MR;  // where its rows go; -1: nowhere
    float big = m, total = l, factor = 1.0f;  // of this lane's row
    __syncthreads();
    if constexpr (WT > 1) {
      if (lane < MR) ml[wave * MR + ln] = make_float2(m, l);
      __syncthreads();
      big = kNoMax;
      total = 0.0f;
#pragma unroll
      for (int t = 0; t < WT; ++t) big = fmaxf(big, ml[(t * WR + wr) * MR + ln].x);
#pragma unroll
      for (int t = 0; t < WT; ++t) {
        const float2 s = ml[(t * WR + wr) * MR + ln];
        total += __builtin_amdgcn_exp2f(s.x - big) * s.y;
      }
      factor = __builtin_amdgcn_exp2f(m - big);
    }
    if (whole) factor *= total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : NAN;
    const int64_t at = static_cast<int64_t>(slot) * TILE_ROWS + share + wr * MR;  // of its first row among the partial sums
    if (lane < MR) {
      place[ln] = live ? b * a.ob + tok_new * a.os + head * a.oh : -1;
      if (wt == 0) {
        if (!whole) a.part_ml[at + ln] = make_float2(big, total);
        else if (live && a.lse)
          a.lse[b * a.lb + tok_new * a.ls + head * a.lh] = total == 0.0f ? -INFINITY : (big + log2f(total)) * kLn2;
      }
    }
    auto quad = [&](int j, int q) {
      return make_float4(o[j][4 * q] * factor, o[j][4 * q + 1] * factor, o[j][4 * q + 2] * factor, o[j][4 * q + 3] * factor);
    };
    float4 own[WT > 1 ? OWN * QN : 1];
    if constexpr (WT > 1) {
#pragma unroll
      for (int w = 0; w < WT; ++w) {
        if (wt != w) continue;
#pragma unroll
        for (int j = 0; j < OB; ++j) {
#pragma unroll
          for (int q = 0; q < QN; ++q) {
            const int to = j / OWN, i = j % OWN * QN + q;
            if (to == w) own[i] = quad(j, q);
            else *reinterpret_cast<float4*>(lds + (wr * WT + to) * STAGE + (w < to ? w : w - 1) * PACK + (i * 64 + lane) * 16) = quad(j, q);
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int t = 0; t < WT - 1; ++t) {
#pragma unroll
        for (int i = 0; i < OWN * QN; ++i) {
          const float4 x = *reinterpret_cast<const float4*>(lds + (wr * WT + wt) * STAGE + t * PACK + (i * 64 + lane) * 16);
          own[i].x += x.x; own[i].y += x.y; own[i].z += x.z; own[i].w += x.w;
        }
      }
    }
    auto sum = [&](int i) {  // columns i / QN * MR + i % QN * 8 + 4 h .. of the wave's blocks
      if constexpr (WT > 1) return own[i];
      else return quad(i / QN, i % QN);
    };
    if (!whole) {
      // as the lanes hold them, 1 KB a store: [row block][column block][quad][lane]
      float4* to = reinterpret_cast<float4*>(a.parts + at * DL) + wt * (PACK / 16) + lane;
#pragma unroll
      for (int i = 0; i < OWN * QN; ++i) to[i * 64] = sum(i);
    } else {
      uint8_t* rows = lds + (wr * WT + wt) * STAGE;
#pragma unroll
      for (int i = 0; i < OWN * QN; ++i) {
        const float4 x = sum(i);
        *reinterpret_cast<uint2*>(rows + ln * OUT_PITCH + 2 * (i / QN * MR + i % QN * 8 + 4 * h)) =
            make_uint2(Elem<DT>::narrow2(x.x, x.y), Elem<DT>::narrow2(x.z, x.w));
      }
      constexpr int CHUNKS = OWN * MR / 8;  // 16-byte chunks of a row
#pragma unroll 4
      for (int i = lane; i < MR * CHUNKS; i += 64) {
        const int r = i / CHUNKS, c = i % CHUNKS;
        const uint4 x = *reinterpret_cast<const uint4*>(rows + r * OUT_PITCH + 16 * c);
        const u32x4_out y = {x.x, x.y, x.z, x.w};
        if (place[r] >= 0)
          *reinterpret_cast<u32x4_out*>(static_cast<uint16_t*>(a.out) + place[r] + wt * (OWN * MR) + 8 * c) = y;
      }
    }
    __syncthreads();
  }
};

template <int DT, bool FP8, int DL, int DR, int MR, int WR, int SPLIT>
__global__ __launch_bounds__(NT, 1) void decode_kernel(Args a) {
  // all of the kernel's LDS, so that it starts at address 0: copies and tile addresses count on it
  extern __shared__ __align__(16) uint8_t lds[];
  Kernel<DT, FP8, DL, DR, MR, WR, SPLIT>::run(a, lds);
}

// Joins the pieces of the (sequence, row tile)s that more than one workgroup
// worked on: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i. Every workgroup
// lists the joins from the main kernel's notes. Partial sums lie as that
// kernel's lanes held them, in units of 1 KB: MR rows (a lane's is lane % MR)
// and 256 / MR columns (four of them its own). Few pieces: a wave takes two
// units, all pieces' loads at once. Many (a long context split over the whole
// device): a workgroup takes a unit, and its waves share the pieces.
constexpr int kFewPieces = 8;
constexpr int kJoinThreads = 512, kJoinWaves = kJoinThreads / 64;
constexpr int kJoinGroups = 512;  // two workgroups a CU

struct Joins {
  int4 join[2][kWorkgroups];  // few pieces, many: {sequence, row tile, 1, last workgroup}
  int first[2][kWorkgroups];  // workgroup of the second piece
  int count[2][kJoinWaves];
  float red[kJoinWaves][32];
  float4 sums[kJoinWaves][64];
  float total[kJoinWaves][64];
};

template <int DT, int DL, int MR>
__global__ __launch_bounds__(kJoinThreads) void combine_kernel(Args a, int tile_rows) {
  __shared__ Joins L;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const int ln = lane % MR, h = lane / MR;
  constexpr int UNITS = DL * MR / 256, COLS = 256 / MR;  // units of a row block, columns of a unit

  // ---- the lists, in the same order in every workgroup
  const int4 mine = tid < a.groups ? a.joins[tid] : make_int4(0, 0, -1, 0);
  const bool some = mine.z >= 0, many = mine.w - tid + 2 > kFewPieces;
  const uint64_t masks[2] = {__ballot(some && !many), __ballot(some && many)};
  if (lane < 2) L.count[lane][wave] = __popcll(masks[lane]);
  __syncthreads();
  int total[2] = {0, 0}, before[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) {
      before[k] += w < wave ? L.count[k][w] : 0;
      total[k] += L.count[k][w];
    }
  if (some) {
    const int k = many, at = before[k] + __popcll(masks[k] & ((uint64_t{1} << lane) - 1));
    L.join[k][at] = mine;
    L.first[k][at] = tid;
  }
  __syncthreads();

  auto address = [&](const int4& j, int r, int64_t& out, int64_t& lse) {  // false: no such row
    const int row = j.y * tile_rows + r, sn = row / a.heads, hd = row % a.heads;
    out = j.x * a.ob + sn * a.os + hd * a.oh;
    lse = j.x * a.lb + sn * a.ls + hd * a.lh;
    return row < a.rows;
  };
  // piece i: the first one was cut at its end, the others at their start
  auto slot_of = [](int first, int i) { return int64_t{i == 0 ? 2 * (first - 1) + 1 : 2 * (first + i - 1)}; };
  auto finish = [&](int64_t lse, float m, float l) {
    if (a.lse) a.lse[lse] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
  };
  auto inverse = [](float l) { return l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : NAN; };

  const int blocks = tile_rows / MR;  // row blocks of a tile

  // ---- few pieces: a wave for two units
  const int of_tile = blocks * (UNITS / 2);
  for (int i = blockIdx.x * kJoinWaves + wave; i < total[0] * of_tile; i += gridDim.x * kJoinWaves) {
    const int t = i / of_tile, block = i / (UNITS / 2) % blocks, u = i % (UNITS / 2) * 2;
    const int4 j = L.join[0][t];
    const int first = L.first[0][t], n = j.w - first + 2;
    float4 x[kFewPieces][2];
    float2 s[kFewPieces];
#pragma unroll
    for (int p = 0; p < kFewPieces; ++p) {
      const int64_t at = slot_of(first, p < n ? p : 0) * tile_rows + block * MR;
      s[p] = a.part_ml[at + ln];
      if (p >= n) s[p] = make_float2(kNoMax, 0.0f);
      if (p < n) {
#pragma unroll
        for (int v = 0; v < 2; ++v) x[p][v] = reinterpret_cast<const float4*>(a.parts + at * DL)[(u + v) * 64 + lane];
      }
    }
    float m = kNoMax, l = 0.0f;
#pragma unroll
    for (int p = 0; p < kFewPieces; ++p) m = fmaxf(m, s[p].x);
    float4 o[2];
#pragma unroll
    for (int v = 0; v < 2; ++v) o[v] = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int p = 0; p < kFewPieces; ++p) {
      if (p >= n) break;
      const float f = __builtin_amdgcn_exp2f(s[p].x - m);
      l += f * s[p].y;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        o[v].x += f * x[p][v].x; o[v].y += f * x[p][v].y; o[v].z += f * x[p][v].z; o[v].w += f * x[p][v].w;
      }
    }
    int64_t out, lse;
    const bool live = address(j, block * MR + ln, out, lse);
    const float inv = inverse(l);
    uint2 y[2];
#pragma unroll
    for (int v = 0; v < 2; ++v)
      y[v] = make_uint2(Elem<DT>::narrow2(o[v].x * inv, o[v].y * inv), Elem<DT>::narrow2(o[v].z * inv, o[v].w * inv));
    uint16_t* to = static_cast<uint16_t*>(a.out) + out + u * COLS;
    if constexpr (MR == 32) {
      // a lane's four columns of both units for eight of one
      const auto p = __builtin_amdgcn_permlane32_swap(y[0].x, y[1].x, false, false);
      const auto q = __builtin_amdgcn_permlane32_swap(y[0].y, y[1].y, false, false);
      const u32x4_out z = {p[0], q[0], p[1], q[1]};
      if (live) *reinterpret_cast<u32x4_out*>(to + 8 * h) = z;
    } else if (live) {
#pragma unroll
      for (int v = 0; v < 2; ++v) *reinterpret_cast<uint2*>(to + v * COLS + 4 * h) = y[v];
    }
    if (live && u == 0 && h == 0) finish(lse, m, l);
  }

  // ---- many: a workgroup for a unit
  for (int i = blockIdx.x; i < total[1] * blocks * UNITS; i += gridDim.x) {
    const int t = i / (blocks * UNITS), block = i / UNITS % blocks, u = i % UNITS;
    const int4 j = L.join[1][t];
    const int first = L.first[1][t], n = j.w - first + 2;  // up to one more than there are workgroups
    auto row_of = [&](int p) { return slot_of(first, p) * tile_rows + block * MR; };
    float m = kNoMax;
#pragma unroll 4
    for (int p = tid / MR; p < n; p += kJoinThreads / MR) m = fmaxf(m, a.part_ml[row_of(p) + ln].x);
    m = row_max<MR>(m);
    if (lane < MR) L.red[wave][ln] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) m = fmaxf(m, L.red[w][ln]);
    float l = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 8
    for (int p = wave; p < n; p += kJoinWaves) {
      const int64_t at = row_of(p);
      const float2 s = a.part_ml[at + ln];
      const float4 x = reinterpret_cast<const float4*>(a.parts + at * DL)[u * 64 + lane];
      const float f = __builtin_amdgcn_exp2f(s.x - m);
      l += f * s.y;
      o.x += f * x.x; o.y += f * x.y; o.z += f * x.z; o.w += f * x.w;
    }
    L.sums[wave][lane] = o;
    L.total[wave][lane] = l;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int w = 1; w < kJoinWaves; ++w) {
        const float4 x = L.sums[w][lane];
        o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
        l += L.total[w][lane];
      }
      int64_t out, lse;
      if (address(j, block * MR + ln, out, lse)) {
        const float inv = inverse(l);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + out + u * COLS + 4 * h) =
            make_uint2(Elem<DT>::narrow2(o.x * inv, o.y * inv), Elem<DT>::narrow2(o.z * inv, o.w * inv));
        if (u == 0 && h == 0) finish(lse, m, l);
      }
    }
    __syncthreads();
  }
}

}  // namespace decode
}  // namespace pcamd
