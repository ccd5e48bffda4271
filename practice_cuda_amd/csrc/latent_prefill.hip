// latent_prefill.hip - attention of packed sequences with keys and values
// expanded from the latent vectors: head h of token t has the key
// [k_nope[t, h] | k_rope[t]], its rotary part shared by all heads, and the
// value v[t, h].
//
//   s[i, j] = scale * q[i] . k[j], j <= i + (keys - queries) where causal
//   o[i] = sum_j softmax(s[i])[j] v[j],   lse[i] = log sum_j exp(s[i, j])
//
// One workgroup holds NR x 128 query rows of one head, NR x 32 a wave, and
// walks over the keys they see in steps of 32 with a running maximum and sum.
// With NR = 2 every operand read from LDS serves two matrix products; with NR =
// 1 two workgroups share a CU, and one's queries, first tiles and output pass
// beside the other's products.
//
// Bound by the matrix products: 2 (DN + DR + DV) operations for each seen pair
// and head, beside an exponential and a rounding to 16 bits a pair, which the
// vector units do while the products run. 8192 tokens, 32 heads, causal, bf16:
// 688 GFLOP in 646 us, 1.06 PFLOP/s, where an 8192^3 product of the library
// reaches 1.25; 6 prompts of up to 1111 tokens behind up to 700 cached ones, 128
// heads: 310 GFLOP in 413 us (their ends fill tiles in part; a workgroup a CU
// took 467). Under this load the clock falls to about 1.6 GHz, so what remains
// is power.
#include <hip/hip_runtime.h>

#include <atomic>
#include <cstdint>

#include "abi_util.h"
#include "attn_common.h"

namespace pcamd {
namespace prefill {

using namespace attn;

constexpr int NT = 256;
constexpr int BN = 32;  // keys of a tile and step

struct Args {
  const void* q; const void* k; const void* kr; const void* v;
  int64_t sqt, sqh, skh, svh;
  uint32_t skt, srt, svt;  // of a token, in bytes
  const int32_t* cu_q; const int32_t* cu_k;
  void* out; int64_t sot, soh;
  float* lse; int64_t slt, slh;
  int64_t total_q, total_k;
  int sequences, heads, causal, max_tiles;  // max_tiles: bound of a head's row tiles
  float scale_log2;                         // not negative: run() is told of a sign by `negate`
  uint32_t negate;                          // sign bits of two elements, or 0
};

struct Tile {
  int64_t q0, k0;  // first token of the sequence's queries and keys (below 2^31)
  int qn, kn;
  int ahead, gap;  // queries from `ahead` on lie `gap` tokens further on
  PCAMD_DEV int query(int row) const { return row + (row >= ahead ? gap : 0); }  // from q0 on
};

PCAMD_DEV int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// Sequence i: its queries and keys, within the tensors whatever the offsets
// say. "Sequence" n (past the last) is the tokens ahead of the first one and
// behind the last, which see no key and get zeros.
PCAMD_DEV Tile sequence(const Args& a, int i) {
  Tile t;
  const bool own = i < a.sequences;
  const int64_t q0 = clamp64(a.cu_q[own ? i : 0], 0, a.total_q), q1 = clamp64(a.cu_q[own ? i + 1 : i], q0, a.total_q);
  const int n = static_cast<int>(q1 - q0);
  t.q0 = own ? q0 : 0;
  t.qn = own ? n : static_cast<int>(a.total_q) - n;
  t.ahead = own ? 0 : static_cast<int>(q0);
  t.gap = own ? 0 : n;
  t.k0 = t.kn = 0;
  if (own) {
    t.k0 = clamp64(a.cu_k[i], 0, a.total_k);
    t.kn = static_cast<int>(clamp64(a.cu_k[i + 1], t.k0, a.total_k) - t.k0);
  }
  return t;
}

// How far (log2) a score may pass its row's reference point before that moves
// (as in the decode kernels: weights are floating point).
template <int DT>
constexpr float kSlack = DT == kF16 ? 8.0f : 40.0f;

template <int DT, int DN, int DR, int DV, int NR>
struct Kernel {
  typedef Mfma<DT, 32> M;
  static constexpr int BM = NR * 128;
  static constexpr int DK = DN + DR;
  static constexpr int KS = DK / 16, OB = DV / 32;
  // A tile in LDS: blocks of 128 bytes a key, [block][key]: the key's own part,
  // its rotary part (one block, half filled where it is 64 bytes), the value.
  static constexpr int KB = DN / 64, VB = DV / 64, CR = DR / 8;
  static constexpr int BLOCK = BN * 128, VALUES = (KB + 1) * BLOCK, TILE = (KB + 1 + VB) * BLOCK;
  // Tiles: the one in use, the next, and others on their way. With 128 rows a
  // workgroup has half of the registers and takes half of the LDS.
  static constexpr int HALF = 163840 / 2, FIT = HALF / TILE;
  static constexpr int NB = NR == 1 && FIT < 6 ? FIT : 6;
  // In the ring's place: queries [block][row][128 bytes] first, behind the tiles
  // that are copied meanwhile; output rows last
  static constexpr int QROWS = NR * 32, QBLOCK = QROWS * 128, QUERIES = (KB + 1) * QBLOCK;
  static constexpr int EARLY = NB < 6 ? 1 : 2, QAT = EARLY * TILE;
  static constexpr int OPITCH = DV * 2 + 16, OUT = QROWS * OPITCH;
  static constexpr int max3(int a, int b, int c) { return a > b ? (a > c ? a : c) : (b > c ? b : c); }
  static constexpr int BODY = max3(NB * TILE, QAT + 4 * QUERIES, 4 * OUT);
  static constexpr int LDS = BODY;
  static_assert(NR > 1 || LDS <= HALF, "two workgroups share a CU's LDS");
  static constexpr int COPIES = KB + 1 + VB;  // of a wave for a tile: 8 keys x 128 bytes each

  // a wave's share of a tile's copies: 8 of its keys
  struct Copies {
    const uint8_t* k;
    const uint8_t* r;
    const uint8_t* v;
    // Keys past the last are copies of it: their weights are zero.
    PCAMD_DEV void address(const uint8_t* kn, const uint8_t* kr, const uint8_t* kv, const Args& a, int t0, int last,
                           int wave, int lane) {
      const int row = wave * 8 + lane / 8, c = (lane % 8) ^ swizzle16(row);
      const uint32_t t = t0 + row < last ? t0 + row : last;
      k = kn + uint64_t{t} * a.skt + 16 * c;
      r = c < CR ? kr + uint64_t{t} * a.srt + 16 * c : nullptr;
      v = kv + uint64_t{t} * a.svt + 16 * c;
    }
    template <int K>
    PCAMD_DEV void emit(uint32_t tile, int wave) const {
      const uint32_t to = tile + K * BLOCK + wave * 8 * 128;
      if constexpr (K < KB) copy16(k + K * 128, to);
      else if constexpr (K > KB) copy16(v + (K - KB - 1) * 128, to);
      else if (CR == 8 || r) copy16(r, to);
    }
    template <int K = 0>
    PCAMD_DEV void emit_all(uint32_t tile, int wave) const {
      if constexpr (K < COPIES) {
        emit<K>(tile, wave);
        emit_all<K + 1>(tile, wave);
      }
    }
    template <int K = 0>
    PCAMD_DEV void emit_at(int n, uint32_t tile, int wave) const {  // spread over the products, from the third on
      if constexpr (K < COPIES) {
        if (2 + K * (KS - 2) / COPIES == n) emit<K>(tile, wave);
        emit_at<K + 1>(n, tile, wave);
      }
    }
  };

  static PCAMD_DEV void run(const Args& a, uint8_t* lds) {
    int* wave_total = reinterpret_cast<int*>(lds);
    int* found = wave_total + NT / 64;
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    // Workgroups go round the eight XCDs: each gets a run of neighbouring heads,
    // one head's tiles after the other's, so that its L2 holds the keys in use
    // and they lie in all of its channels.
    const int per = gridDim.x / 8, item = blockIdx.x % 8 * per + blockIdx.x / 8;
    const int head = item / a.max_tiles;
    int want = item - head * a.max_tiles;
    if (head >= a.heads) return;

    // ---- the tile's sequence, found in a running count of tiles over the
    // sequences, and its tile, the longest rows of a causal sequence first
    Tile t;
    int row0;
    if (a.sequences < 64) {
      // a sequence a lane; every wave finds it by itself
      const Tile own = sequence(a, lane <= a.sequences ? lane : a.sequences);
      const int mine = lane <= a.sequences ? (own.qn + BM - 1) / BM : 0;
      int inc = mine;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(inc, d, 64);
        if (lane >= d) inc += o;
      }
      // Every second head, counted from the last, the other way round: workgroups
      // that share a CU then have long rows and short ones.
      const int total = __builtin_amdgcn_readlane(inc, 63);
      if (((a.heads - 1 - head) & 1) && want < total) want = total - 1 - want;
      const uint64_t here = __ballot(want >= inc - mine && want < inc);
      if (!here) return;
      const int from = __builtin_ctzll(here);
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, from); };
      t.q0 = of(static_cast<int>(own.q0));
      t.k0 = of(static_cast<int>(own.k0));
      t.qn = of(own.qn);
      t.kn = of(own.kn);
      t.ahead = of(own.ahead);
      t.gap = of(own.gap);
      row0 = (of(inc) - 1 - want) * BM;
    } else {
      if (tid == 0) found[0] = -1;
      int base = 0;
      for (int i0 = 0; i0 <= a.sequences; i0 += NT) {
        const int i = i0 + tid;
        const int mine = i <= a.sequences ? (sequence(a, i).qn + BM - 1) / BM : 0;
        int inc = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const int o = __shfl_up(inc, d, 64);
          if (lane >= d) inc += o;
        }
        __syncthreads();
        if (lane == 63) wave_total[wave] = inc;
        __syncthreads();
        int before = base + inc - mine, total = 0;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) {
          if (w < wave) before += wave_total[w];
          total += wave_total[w];
        }
        if (want >= before && want < before + mine) {
          found[0] = i;
          found[1] = mine - 1 - (want - before);
        }
        base += total;
        __syncthreads();
        if (found[0] >= 0) break;
      }
      if (found[0] < 0) return;
      t = sequence(a, __builtin_amdgcn_readfirstlane(found[0]));
      row0 = __builtin_amdgcn_readfirstlane(found[1]) * BM;
      __syncthreads();  // the queries take this place
    }
    // a tile of at most 128 rows, the rest of a sequence, goes to all four waves too
    if (NR == 2 && t.qn - row0 <= 128) Kernel<DT, DN, DR, DV, 1>::rows(a, lds, t, row0, head);
    else rows(a, lds, t, row0, head);
  }

  // rows row0 .. of a sequence's queries
  static PCAMD_DEV void rows(const Args& a, uint8_t* lds, const Tile& t, int row0, int head) {
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int h = lane / 32, ln = lane % 32;
    const int past = t.kn - t.qn;

    // ---- queries: whole lines into LDS, a lane's row from there
    const uint8_t* qp = static_cast<const uint8_t*>(a.q) + 2 * (t.q0 * a.sqt + head * a.sqh);
#pragma unroll
    for (int i = 0; i < QROWS / 8; ++i) {
      const int r = 8 * i + lane / 8, c = (lane % 8) ^ swizzle16(r);
      int row = row0 + wave * QROWS + r;
      if (row >= t.qn) row = t.qn - 1;  // a spare row computes what another one does, and is not stored
      const uint8_t* p = qp + 2 * row * a.sqt + 16 * c;
      const uint32_t to = QAT + wave * QUERIES + 8 * i * 128;
#pragma unroll
      for (int b = 0; b < KB; ++b) copy16(p + b * 128, to + b * QBLOCK);
      if (c < CR) copy16(p + DN * 2, to + KB * QBLOCK);
    }
    // ---- the first tiles' copies, behind the queries'
    const uint8_t* kn = static_cast<const uint8_t*>(a.k) + t.k0 * a.skt + 2 * head * a.skh;
    const uint8_t* kr = static_cast<const uint8_t*>(a.kr) + t.k0 * a.srt;
    const uint8_t* kv = static_cast<const uint8_t*>(a.v) + t.k0 * a.svt + 2 * head * a.svh;
    const int end = row0 + BM < t.qn ? row0 + BM : t.qn;  // of the tile's rows
    int keys = a.causal ? end + past : t.kn;              // that they see
    if (keys > t.kn) keys = t.kn;
    const int tiles = keys > 0 ? (keys + BN - 1) / BN : 0;
    Copies copies;
    if (tiles > 0) {
#pragma unroll
      for (int i = 0; i < EARLY; ++i) {
        copies.address(kn, kr, kv, a, i * BN, t.kn - 1, wave, lane);
        copies.emit_all(i * TILE, wave);
      }
      wait_copies<EARLY * COPIES>();
    } else {
      wait_copies<0>();
    }
    uint4 q[NR][KS];
#pragma unroll
    for (int u = 0; u < NR; ++u)
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int c = 2 * k < DN / 8 ? 2 * k : 2 * k - DN / 8, b = 2 * k < DN / 8 ? c / 8 : KB;
        uint4 x = *reinterpret_cast<const uint4*>(lds + QAT + wave * QUERIES + b * QBLOCK + (u * 32 + ln) * 128 +
                                                  (((c % 8 + h) ^ swizzle16(ln)) << 4));
        x.x ^= a.negate; x.y ^= a.negate; x.z ^= a.negate; x.w ^= a.negate;
        q[u][k] = x;
      }
#pragma unroll
    for (int u = 0; u < NR; ++u)
#pragma unroll
      for (int k = 0; k < KS; ++k) asm volatile("" : "+v"(q[u][k].x), "+v"(q[u][k].y), "+v"(q[u][k].z), "+v"(q[u][k].w));
    __syncthreads();  // the tiles take the queries' place

    int row[NR], limit[NR];  // this lane's rows, and how many keys they see
#pragma unroll
    for (int u = 0; u < NR; ++u) {
      row[u] = row0 + wave * QROWS + u * 32 + ln;
      const int n = a.causal ? row[u] + past + 1 : t.kn;
      limit[u] = n < t.kn ? n : t.kn;
    }
    const int first = row0 + wave * QROWS + past + 1;
    const int all_see = a.causal && first < t.kn ? first : t.kn;  // keys that every row of the wave sees
    // The wave's own steps: up to the last key that one of its rows sees, none
    // if it has no rows. It waits out the others' steps.
    const int mine0 = row0 + wave * QROWS, mine1 = mine0 + QROWS < t.qn ? mine0 + QROWS : t.qn;
    int seen = mine1 <= mine0 ? 0 : a.causal ? mine1 + past : t.kn;
    if (seen > t.kn) seen = t.kn;
    const int steps = seen > 0 ? (seen + BN - 1) / BN : 0;
    f32x16 o[NR][OB];
    float m[NR], nm[NR], l[NR];  // reference point (in units of s), minus its log2, sum of weights
#pragma unroll
    for (int u = 0; u < NR; ++u) {
#pragma unroll
      for (int j = 0; j < OB; ++j) o[u][j] = f32x16{};
      m[u] = kNoMax;
      nm[u] = 0.0f;
      l[u] = 0.0f;
    }

    // ---- The parts of a step. As in the decode kernels, reads of LDS run ahead
    // of the products that take them, held in place by sched_barrier; `beside(i)`
    // is other work for the time of the products with operand i.
    const uint32_t lane_k = ln * 128 + ((h ^ swizzle16(ln)) << 4);
    const int i16 = lane % 16, tv = 4 * h + (i16 >> 2);
    const uint32_t lane_v =
        VALUES + tv * 128 + (((2 * ((lane / 16) & 1) + ((i16 >> 1) & 1)) ^ swizzle16(tv)) << 4) + 8 * (i16 & 1);
    auto key = [&](uint32_t tile, int k) {
      const int c = 2 * k < DN / 8 ? 2 * k : 2 * k - DN / 8, b = 2 * k < DN / 8 ? c / 8 : KB;
      return *reinterpret_cast<const uint4*>(lds + ((tile + lane_k) ^ (c % 8 << 4)) + b * BLOCK);
    };
    auto value = [&](uint32_t tile, int j, int kk) {
      const int x = 4 * j % 8 << 4, at = 4 * j / 8 * BLOCK + kk * 16 * 128;
      const uint2 y = read_tr4(lds + ((tile + lane_v) ^ x) + at);
      const uint2 z = read_tr4(lds + ((tile + lane_v) ^ (x ^ 16)) + at + 8 * 128);
      return make_uint4(y.x, y.y, z.x, z.y);
    };
    constexpr int DA = KS < 8 ? KS : 8;                      // key operands read ahead
    constexpr int NP = 2 * OB, DVA = NP < 6 ? NP : 6;        // value operands (contraction step n / OB, block n % OB), ahead
    uint4 val[DVA];
    f32x16 c[NR];
    float s[NR][16];
    uint32_t p[NR][8];
    auto scores = [&](uint32_t tile, auto beside) {
      uint4 raw[DA];
#pragma unroll
      for (int k = 0; k < DA; ++k) raw[k] = key(tile, k);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const uint4 x = raw[k % DA];
#pragma unroll
        for (int u = 0; u < NR; ++u) c[u] = M::mul(x, q[u][k], k == 0 ? f32x16{} : c[u]);
        if (k + DA < KS) raw[k % DA] = key(tile, k + DA);
        beside(k);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto first_values = [&](uint32_t tile) {
#pragma unroll
      for (int n = 0; n < DVA; ++n) val[n] = value(tile, n % OB, n / OB);
    };
    auto values = [&](uint32_t tile, auto beside) {
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        const int j = n % OB, kk = n / OB;
        const uint4 x = val[n % DVA];
#pragma unroll
        for (int u = 0; u < NR; ++u) {
          const uint32_t* w = p[u] + 4 * kk;
          o[u][j] = M::mul(x, make_uint4(w[0], w[1], w[2], w[3]), o[u][j]);
        }
        if (n + DVA < NP) val[n % DVA] = value(tile, (n + DVA) % OB, (n + DVA) / OB);
        beside(n);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // element e of NR * 16: row u = e / 16, register e % 16
    // A score out of the accumulation registers. Inline asm: the compiler would
    // keep the copy there too. It does not see the product that wrote the score
    // (12 wait states, 48 clocks), so two later ones (32 clocks each) stand in
    // between, or settle().
    auto take = [&](int e) {
      asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(s[e / 16][e % 16]) : "a"(c[e / 16][e % 16]));
    };
    auto settle = [&]() {
#pragma unroll
      for (int u = 0; u < NR; ++u) asm volatile("s_nop 15" : "+a"(c[u]));
    };
    auto weigh = [&](int e) {
      const int u = e / 16, r = e % 16;
      s[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], a.scale_log2, nm[u]));
    };
    auto add = [&](int e) {  // two elements at a time
      const int u = e / 16, r = e % 16;
      if (r & 1) {
        l[u] += s[u][r - 1] + s[u][r];
        asm volatile("" : "+v"(l[u]));  // here, beside the products: left alone, it sinks to the end of the step
        p[u][r / 2] = Elem<DT>::narrow2(s[u][r - 1], s[u][r]);
      }
    };
    float top[NR];
    auto look = [&](int t0, auto masked) {  // before the weights of the step at key t0: its mask and reference point
      if constexpr (decltype(masked)::value) {
#pragma unroll
        for (int u = 0; u < NR; ++u) {
          top[u] = kNoMax;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[u][r] = t0 + (r / 4) * 8 + 4 * h + r % 4 < limit[u] ? s[u][r] : -INFINITY;
            top[u] = fmaxf(top[u], s[u][r]);
          }
          top[u] = row_max<32>(top[u]);
        }
      }
      bool passed = false;
#pragma unroll
      for (int u = 0; u < NR; ++u) passed |= (top[u] - m[u]) * a.scale_log2 > kSlack<DT>;
      if (__any(passed)) {
#pragma unroll
        for (int u = 0; u < NR; ++u) {
          const float to = fmaxf(m[u], top[u]), alpha = __builtin_amdgcn_exp2f((m[u] - to) * a.scale_log2);
          m[u] = to;
          // A row that has seen nothing keeps a factor of zero: kNoMax itself times a scale_log2 above 1.13 is not
          // finite, and its scores of -inf would become NaN.
          nm[u] = to == kNoMax ? 0.0f : -to * a.scale_log2;
          l[u] *= alpha;
#pragma unroll
          for (int j = 0; j < OB; ++j) {
            // block by block through the vector registers, back to where the products keep it
            asm volatile("" : "+a"(o[u][j]));
            o[u][j] *= alpha;
            asm volatile("" : "+a"(o[u][j]));
          }
        }
      }
    };
    auto maxima = [&]() {
#pragma unroll
      for (int u = 0; u < NR; ++u) {
        top[u] = s[u][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top[u] = fmaxf(top[u], s[u][r]);
        top[u] = row_max<32>(top[u]);
      }
    };
    auto nothing = [](int) {};
    constexpr int E = NR * 16;
    // the step with a tile whose scores are in s; the next tile's scores are computed beside
    auto step = [&](uint32_t tile, int t0, uint32_t next, auto more, auto masked, auto copies) {
      if constexpr (decltype(more)::value) {
        scores(next, [&](int k) {
          copies(k);
          // E elements over KS operands' time, each pair's sum and rounding one operand later
#pragma unroll
          for (int e = 0; e < E; ++e) {
            if (e * (KS - 1) / E == k) weigh(e);
            if (e * (KS - 1) / E + 1 == k) add(e);
          }
          if (k == KS - 2) first_values(tile);
        });
#pragma unroll
        for (int u = 0; u < NR; ++u) top[u] = kNoMax;
        values(tile, [&](int n) {
          constexpr int FROM = NR == 1 ? 2 : 1, OVER = NP - 1 - FROM;  // elements over operands FROM .. FROM + OVER - 1
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (FROM + e * OVER / E == n) {
              take(e);
              top[e / 16] = fmaxf(top[e / 16], s[e / 16][e % 16]);
            }
          if (n == NP - 1) {
#pragma unroll
            for (int u = 0; u < NR; ++u) top[u] = row_max<32>(top[u]);
          }
        });
        look(t0 + 32, masked);
      } else {
        first_values(tile);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          weigh(e);
          add(e);
        }
        __builtin_amdgcn_sched_barrier(0);
        values(tile, nothing);
      }
    };

    if (tiles > 0) {
#pragma unroll
      for (int i = EARLY; i < NB - 1; ++i) {
        copies.address(kn, kr, kv, a, i * BN, t.kn - 1, wave, lane);
        copies.emit_all(i * TILE, wave);
      }
      wait_copies<(NB - 2) * COPIES>();
      tile_barrier();
      uint32_t tile = 0, into = (NB - 1) * TILE;
      int i = 0;
      auto turn = [&]() {
        // The next tile has arrived for all waves, and all have left the one
        // before this: a tile further on takes its place.
        wait_copies<(NB - 3) * COPIES>();
        tile_barrier();
        return tile + TILE < NB * TILE ? tile + TILE : 0;
      };
      auto walk = [&](int to, auto masked) {  // up to step `to`, whose scores then wait in s
        for (; i < to; ++i) {
          const uint32_t next = turn();
          step(tile, i * BN, next, std::true_type{}, masked, [&](int k) {
            if (k == 1) copies.address(kn, kr, kv, a, (i + NB - 1) * BN, t.kn - 1, wave, lane);
            copies.emit_at(k, into, wave);
          });
          into = tile;
          tile = next;
        }
      };
      if (steps > 0) {
        scores(0, nothing);
        settle();
#pragma unroll
        for (int e = 0; e < E; ++e) take(e);
        maxima();
        if (all_see < BN) look(0, std::true_type{});
        else look(0, std::false_type{});
        // Steps that some row of the wave does not see all of come last. Masking
        // in a branch of one loop would cost every step copies of its scores.
        const int whole = all_see / BN - 1;
        walk(whole < steps - 1 ? whole : steps - 1, std::false_type{});
        walk(steps - 1, std::true_type{});
        step(tile, i * BN, 0, std::false_type{}, std::false_type{}, nothing);
      }
      for (; i + 1 < tiles; ++i) {
        const uint32_t next = turn();
        copies.address(kn, kr, kv, a, (i + NB - 1) * BN, t.kn - 1, wave, lane);
        copies.emit_all(into, wave);
        into = tile;
        tile = next;
      }
      wait_copies<0>();
    }

    // ---- epilogue: output rows gather in LDS and leave as whole lines
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NR; ++u) {
      const float sum = row_sum<32>(l[u]);
      const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : NAN;
      if (a.lse && h == 0 && row[u] < t.qn)
        a.lse[(t.q0 + t.query(row[u])) * a.slt + head * a.slh] =
            sum == 0.0f ? -INFINITY : (m[u] * a.scale_log2 + log2f(sum)) * kLn2;
#pragma unroll
      for (int j = 0; j < OB; ++j)
#pragma unroll
        for (int y = 0; y < 4; ++y)
          *reinterpret_cast<uint2*>(lds + wave * OUT + (u * 32 + ln) * OPITCH + 64 * j + 16 * y + 8 * h) =
              make_uint2(Elem<DT>::narrow2(o[u][j][4 * y] * inv, o[u][j][4 * y + 1] * inv),
                         Elem<DT>::narrow2(o[u][j][4 * y + 2] * inv, o[u][j][4 * y + 3] * inv));
    }
    // each wave's rows are its own
    uint16_t* out = static_cast<uint16_t*>(a.out) + t.q0 * a.sot + head * a.soh;
    constexpr int PER = DV / 4;  // 8-byte pieces of a row
#pragma unroll 4
    for (int i = lane; i < QROWS * PER; i += 64) {
      const int r = i / PER, d = i % PER, to = row0 + wave * QROWS + r;
      const uint2 x = *reinterpret_cast<const uint2*>(lds + wave * OUT + r * OPITCH + 8 * d);
      if (to < t.qn) *reinterpret_cast<uint2*>(out + t.query(to) * a.sot + 4 * d) = x;
    }
  }
};

template <int DT, int DN, int DR, int DV, int NR>
__global__ __launch_bounds__(NT, NR == 1 ? 2 : 1) void prefill_kernel(Args a) {
  // all of the kernel's LDS, so that it starts at address 0: copies and tile addresses count on it
  extern __shared__ __align__(16) uint8_t lds[];
  Kernel<DT, DN, DR, DV, NR>::run(a, lds);
}

template <int DT, int DN, int DR, int DV, int NR>
int launch_rows(Args a, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  typedef Kernel<DT, DN, DR, DV, NR> K;
  const auto kern = prefill_kernel<DT, DN, DR, DV, NR>;
  const int64_t max_tiles = a.total_q / K::BM + a.sequences + 1, per = (max_tiles * a.heads + 7) / 8;
  if (per * 8 >= (int64_t{1} << 32) / NT)
    return set_error(PCAMD_ERR_UNSUPPORTED, "latent prefill: grid too large (%lld workgroups)", (long long)per * 8);
  const int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(kern), K::LDS, st, done);
  if (rc != PCAMD_OK) return rc;
  a.max_tiles = static_cast<int>(max_tiles);
  kern<<<static_cast<uint32_t>(per * 8), NT, K::LDS, st>>>(a);
  return check_launch("prefill_kernel");
}

template <int DT, int DN, int DR, int DV>
int launch(const Args& a, hipStream_t st) {
  // 256-row tiles for prompts that are long on average. Tokens x heads, causal, bf16, us with 128 and 256 rows: 4096 x 16
  // 108 / 135, 4096 x 32 206 / 206, 8192 x 16 321 / 316, 8192 x 32 643 / 632, 16384 x 16 1265 / 1216, 32768 x 16 5174 / 4929;
  // 4096 x 128 704 / 737, 2 sequences of 7000, 32 heads 979 / 992 and of 8192, 16 heads 689 / 703, 4 of 10 to 4000, 32 heads
  // 294 / 333, 16 of 512, 16 heads 52 / 66, 40 of 300, 128 heads 465 / 830
  const bool many = a.total_q >= int64_t{8192} * a.sequences && a.total_q * a.heads >= 8192 * 16;
  return many ? launch_rows<DT, DN, DR, DV, 2>(a, st) : launch_rows<DT, DN, DR, DV, 1>(a, st);
}

}  // namespace prefill
}  // namespace pcamd

extern "C" int pcamd_latent_prefill(const void* q, const void* k_nope, const void* k_rope, const void* v, int dtype,
                                    int64_t total_q, int64_t total_k, int64_t heads, int64_t nope_dim,
                                    int64_t rope_dim, int64_t v_dim, int64_t sqt, int64_t sqh, int64_t skt,
                                    int64_t skh, int64_t srt, int64_t svt, int64_t svh, const int32_t* cu_q,
                                    const int32_t* cu_k, int64_t sequences, void* out, int64_t sot, int64_t soh,
                                    float* lse, int64_t slt, int64_t slh, float softmax_scale, int causal,
                                    void* stream) {
  using namespace pcamd;
  clear_error();
  if (total_q < 0 || total_k < 0 || heads < 0 || sequences < 0) return set_error(PCAMD_ERR_INVALID, "negative size");
  if (dtype != kBF16 && dtype != kF16) return set_error(PCAMD_ERR_INVALID, "queries must be bf16 or fp16, got code %d", dtype);
  const bool wide = nope_dim == 128 && rope_dim == 64 && v_dim == 128;
  const bool narrow = nope_dim == 64 && rope_dim == 32 && v_dim == 64;
  if (!wide && !narrow)
    return set_error(PCAMD_ERR_UNSUPPORTED, "key, rotary and value widths must be 128, 64, 128 or 64, 32, 64; got %lld, %lld, %lld",
                     (long long)nope_dim, (long long)rope_dim, (long long)v_dim);
  if (total_q > (1 << 30) || total_k > (1 << 30) || sequences > (1 << 30) || heads > (1 << 20))
    return set_error(PCAMD_ERR_UNSUPPORTED, "latent prefill: more than 2^30 tokens or sequences, or 2^20 heads");
  if (total_q == 0 || heads == 0) return PCAMD_OK;
  if (!q || !cu_q || !cu_k || !out || (total_k && (!k_nope || !k_rope || !v)))
    return set_error(PCAMD_ERR_INVALID, "null pointer");
  auto odd = [](const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; };
  auto bad = [](int64_t places, int64_t stride, int64_t unit) { return places > 1 && stride % unit; };  // one place: any stride
  if (odd(q, 16) || odd(k_nope, 16) || odd(k_rope, 16) || odd(v, 16) || odd(out, 8) || bad(total_q, sqt, 8) ||
      bad(heads, sqh, 8) || bad(total_k, skt, 8) || bad(heads, skh, 8) || bad(total_k, srt, 8) || bad(total_k, svt, 8) ||
      bad(heads, svh, 8) || bad(total_q, sot, 4) || bad(heads, soh, 4))
    return set_error(PCAMD_ERR_INVALID, "rows of queries, keys and values must be 16-byte aligned, of the output 8-byte");
  if (total_k <= 1) skt = srt = svt = 0;
  for (const int64_t stride : {skt, srt, svt})
    if (stride < 0 || stride > (1 << 30)) return set_error(PCAMD_ERR_UNSUPPORTED, "latent prefill: a token stride past 2^30 elements");
  prefill::Args a{};
  a.q = q; a.k = k_nope; a.kr = k_rope; a.v = v;
  a.sqt = sqt; a.sqh = sqh; a.skh = skh; a.svh = svh;
  a.skt = static_cast<uint32_t>(2 * skt); a.srt = static_cast<uint32_t>(2 * srt); a.svt = static_cast<uint32_t>(2 * svt);
  a.cu_q = cu_q; a.cu_k = cu_k;
  a.out = out; a.sot = sot; a.soh = soh; a.lse = lse; a.slt = slt; a.slh = slh;
  a.total_q = total_q; a.total_k = total_k;
  a.sequences = static_cast<int>(sequences); a.heads = static_cast<int>(heads); a.causal = causal != 0;
  // The kernel compares scores before they are scaled: a negative scale's sign
  // goes to the queries, and none is so small that a masked score's times it is not -inf.
  a.scale_log2 = fabsf(softmax_scale) * attn::kLog2e;
  if (a.scale_log2 < 1e-30f) a.scale_log2 = 1e-30f;
  a.negate = softmax_scale < 0.0f ? 0x80008000u : 0u;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == kBF16) return wide ? prefill::launch<kBF16, 128, 64, 128>(a, st) : prefill::launch<kBF16, 64, 32, 64>(a, st);
  return wide ? prefill::launch<kF16, 128, 64, 128>(a, st) : prefill::launch<kF16, 64, 32, 64>(a, st);
}
