// int8_bmm_tiles.hip - int8 products of many rows, bound by the matrix cores.
//
// Tiles of A and B go global -> LDS with buffer_load_dwordx4 ... lds, 64 bytes
// of k a step, into a ring of LDS stages, all but one of them ahead of the
// products. A row's 64 bytes are four chunks of 16; chunk c of row r sits at
// position c ^ swz(r), so that the 16 lanes that LDS serves together read
// different banks. Lane 16 g + r holds
// chunk g of its row, the operand of v_mfma_i32_16x16x64_i8. B is the first
// operand of the instruction, so a lane ends with four neighbouring columns of
// a row.
#include <algorithm>
#include <type_traits>

#include "bmm_lds.h"
#include "int8_bmm.h"

namespace pcamd {
namespace int8 {
namespace {

using lds::lds_addr;
using lds::make_rsrc;

constexpr int BK = 64;

// ds_read_b128 serves 16 lanes at once: 0-3, 12-15 and 20-27, then 4-11, 16-19 and 28-31, and so on, as counted bank
// conflicts say. With i = r / 4, the rows a, a + 12 of chunk g and a + 4, a + 8 of chunk g ^ 1 then need four different
// positions: 0, 1, 1 ^ 3 and 1 ^ 2. Conflicts are under 0.5 % of the LDS's busy clocks at 8192 x 14336 x 4096.
PCAMD_DEV int swz(int r) {
  const int i = (r >> 2) & 3;
  return i ^ ((i & 1) << 1);
}

// WM x WN waves of 64 rows by 64 NB columns. PP: two waves share a SIMD and take turns, one on the matrix cores
// while the other reads LDS.
template <int WM_, int WN_, int NB_, int NS_, bool PP_>
struct Geom {
  static constexpr int WM = WM_, WN = WN_, NB = NB_, WAVES = WM * WN, THREADS = WAVES * 64;
  static constexpr int NS = NS_, AHEAD = NS - 1;  // stages, steps copied ahead
  static constexpr bool PP = PP_;
  static constexpr int BM = 64 * WM, BN = 64 * NB * WN;
  static constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK, STAGE = A_BYTES + B_BYTES, RING = NS * STAGE, LDS = RING + (BM + 2 * BN) * 4;
  static constexpr int A_INSTS = BM / WAVES / 16, B_INSTS = BN / WAVES / 16, INSTS = A_INSTS + B_INSTS;
  static_assert(A_INSTS * WAVES * 16 == BM && B_INSTS * WAVES * 16 == BN, "rows a wave copies");
};
using Wide = Geom<4, 2, 2, 4, true>;    // 256 x 256, a workgroup a CU
using Small = Geom<2, 2, 1, 4, false>;  // 128 x 128, two workgroups a CU

template <typename G, bool GROUPED, bool GATED>
__global__ __launch_bounds__(G::THREADS, G::WAVES == 8 ? 1 : 2) void tiles_kernel(Args a, int tiles_m, int tiles_n) {
  constexpr int OUT = GATED ? G::BN / 2 : G::BN;  // columns of C a tile
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const int wm = wave % G::WM, wn = wave / G::WM;

  // consecutive tiles on one XCD (workgroup i runs on XCD i % 8), in groups of 8 rows of tiles
  const int total = tiles_m * tiles_n, per_xcd = (total + 7) >> 3;
  const int pid = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (pid >= total) return;
  constexpr int GROUP_M = 8;
  const int group = pid / (GROUP_M * tiles_n), in_group = pid - group * GROUP_M * tiles_n;
  const int gm = min(tiles_m - group * GROUP_M, GROUP_M);
  const int tile_m = __builtin_amdgcn_readfirstlane(group * GROUP_M + in_group % gm);
  const int n0 = __builtin_amdgcn_readfirstlane(in_group / gm * OUT);
  Rows rows;
  if constexpr (GROUPED) {
    if (!grouped_tile(a, tile_m, G::BM, rows)) return;
    if (rows.zeros) {
      const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int i = threadIdx.x; i < G::BM * OUT / 4; i += G::THREADS) {
        const int row = rows.row + i / (OUT / 4), n = n0 + 4 * (i % (OUT / 4));
        if (row < rows.end && n < a.n) store4(a.c, a.c_dtype, int64_t(row) * a.scm + n, a.n - n, zero);
      }
      return;
    }
  } else {
    rows.mat = blockIdx.y;
    rows.row = tile_m * G::BM;
    rows.end = min(rows.row + G::BM, a.m);
    rows.zeros = false;
  }

  // Where the copies read: instruction i of wave w fills 16 rows from (w * INSTS + i) * 16 on, lane l chunk (l & 3) ^
  // swz of row l >> 2 of them. Rows and columns past the matrix read its last one; their outputs are not stored.
  const int chunk = ((lane & 3) ^ swz(lane >> 2)) * 16;
  const int8_t* base_a = a.a + (GROUPED ? 0 : rows.mat * a.sab + int64_t(rows.row) * a.lda);
  const int8_t* base_b = a.b + rows.mat * a.sbb + int64_t(n0) * a.ldb;
  const lds::v4i rsa = make_rsrc(base_a, 0xFFFFFFFFu), rsb = make_rsrc(base_b, 0xFFFFFFFFu);
  uint32_t off_a[G::A_INSTS], off_b[G::B_INSTS];
#pragma unroll
  for (int i = 0; i < G::A_INSTS; ++i) {
    const int r = min(rows.row + (wave * G::A_INSTS + i) * 16 + (lane >> 2), rows.end - 1);
    const int64_t row = GROUPED ? a_row<GROUPED>(a, r) : r - rows.row;
    off_a[i] = static_cast<uint32_t>(row * a.lda) + chunk;
  }
#pragma unroll
  for (int i = 0; i < G::B_INSTS; ++i) {
    const int c = (wave * G::B_INSTS + i) * 16 + (lane >> 2);
    // gated: 16 gates, then the 16 columns they go with
    const int col = GATED ? min(16 * (c >> 5) + (c & 15), a.n - 1 - n0) + ((c >> 4) & 1) * a.n : min(c, a.n - 1 - n0);
    off_b[i] = static_cast<uint32_t>(col * int64_t(a.ldb)) + chunk;
  }
  const int steps = (a.k + BK - 1) / BK, tail = a.k - (steps - 1) * BK;
  const uint32_t to_a = lds_addr(smem) + wave * G::A_INSTS * 16 * BK;
  const uint32_t to_b = lds_addr(smem) + G::A_BYTES + wave * G::B_INSTS * 16 * BK;
  // The copies of step ks; stage: its offset in LDS. Chunks past a row's end read its first one (the masked A makes
  // zeros of them).
  auto issue = [&](int ks, uint32_t stage) {
    const int k0 = ks * BK;
    const uint32_t step = k0 + chunk < a.k ? k0 : -chunk;
#pragma unroll
    for (int i = 0; i < G::A_INSTS; ++i) lds::lds_dma16(rsa, to_a + stage + i * 16 * BK, off_a[i] + step);
#pragma unroll
    for (int i = 0; i < G::B_INSTS; ++i) lds::lds_dma16(rsb, to_b + stage + i * 16 * BK, off_b[i] + step);
  };

  constexpr int NJ = 4 * G::NB;
  v4i acc[4][NJ];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = v4i{0, 0, 0, 0};
  v4i fa[4], fb[NJ];
  const int frag = lr * BK + ((lg ^ swz(lr)) << 4);  // a lane's place in 16 rows
  auto read = [&](uint32_t stage) {
    const uint8_t* at_a = smem + stage + wm * 64 * BK + frag;
    const uint8_t* at_b = smem + stage + G::A_BYTES + wn * 64 * G::NB * BK + frag;
#pragma unroll
    for (int i = 0; i < 4; ++i) fa[i] = *reinterpret_cast<const v4i*>(at_a + 16 * BK * i);
#pragma unroll
    for (int j = 0; j < NJ; ++j) fb[j] = *reinterpret_cast<const v4i*>(at_b + 16 * BK * j);
  };
  auto products = [&] {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[j], fa[i], acc[i][j], 0, 0, 0);
  };
  auto fence = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // Once step k + AHEAD is issued: step k + 1 has landed. Where no more are issued (last), all have.
  auto landed = [&](bool last) {
    if (!last) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((G::AHEAD - 1) * G::INSTS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  auto barrier = [&] {
    fence();
    __builtin_amdgcn_s_barrier();
    fence();
  };
  auto mask_a = [&](int ks) {
#pragma unroll
    for (int i = 0; i < 4; ++i) fa[i] = mask_tail(fa[i], ks * BK + lg * 16, a.k);
  };
  auto after = [](uint32_t stage) { return stage + G::STAGE == G::NS * G::STAGE ? 0u : stage + G::STAGE; };

  for (int ks = 0; ks < G::AHEAD && ks < steps; ++ks) issue(ks, ks * G::STAGE);
  // scales, and the bias where it is one for all rows, for the end
  float* sa_l = reinterpret_cast<float*>(smem + G::RING);
  float* sb_l = sa_l + G::BM;
  float* bias_l = sb_l + G::BN;
  const bool row_bias = !GROUPED && a.bias && a.sbiasm != 0;
  auto bias_at = [&](int row, int col) {
    return load_as(a.bias, a.bias_dtype, rows.mat * a.sbiasb + (GROUPED ? 0 : row * a.sbiasm) + int64_t(col) * a.sbiasn);
  };
  for (int t = threadIdx.x; t < G::BM; t += G::THREADS) {
    const int r = min(rows.row + t, rows.end - 1);
    sa_l[t] = a.sa[(GROUPED ? 0 : rows.mat * a.ssab) + a_row<GROUPED>(a, r) * a.ssam];
  }
  for (int t = threadIdx.x; t < G::BN; t += G::THREADS) {
    const int col = GATED ? min(n0 + 16 * (t >> 5) + (t & 15), a.n - 1) + ((t >> 4) & 1) * a.n : min(n0 + t, a.n - 1);
    sb_l[t] = a.sb[rows.mat * a.ssbb + int64_t(col) * a.ssbn];
    bias_l[t] = a.bias && !row_bias ? bias_at(0, col) : 0.0f;
  }
  landed(steps <= G::AHEAD);
  __syncthreads();
  uint32_t cur = 0, fill = G::AHEAD * G::STAGE;
  if constexpr (G::PP) {
    // Time runs in slots between barriers. The first four waves read step k in slot 2 k and multiply in slot 2 k + 1;
    // the last four, one on each SIMD with one of the first, do the same one slot later. A wave issues the copies of
    // step k + AHEAD behind its reads of step k: the stage that they fill held step k - 1, whose last reads (slot
    // 2 k - 1) ended in front of that slot's barrier. Step k + 1 has landed in front of the barrier of slot 2 k + 1.
    const bool second = wave >= G::WAVES / 2;
    if (second) barrier();
    for (int ks = 0; ks < steps; ++ks) {
      const bool more = ks + G::AHEAD < steps;
      read(cur);
      if (more) issue(ks + G::AHEAD, fill);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (ks == steps - 1 && tail < BK) mask_a(ks);
      if (second) landed(!more);
      barrier();
      __builtin_amdgcn_s_setprio(1);
      products();
      __builtin_amdgcn_s_setprio(0);
      if (!second) landed(!more);
      barrier();
      cur = after(cur);
      fill = after(fill);
    }
    if (!second) barrier();
  } else {
    // The stage of step k + AHEAD held step k - 1, whose reads ended in front of the barrier.
    for (int ks = 0; ks < steps; ++ks) {
      const bool more = ks + G::AHEAD < steps;
      if (more) issue(ks + G::AHEAD, fill);
      read(cur);
      if (ks == steps - 1 && tail < BK) mask_a(ks);
      products();
      landed(!more);
      __syncthreads();
      cur = after(cur);
      fill = after(fill);
    }
  }

  // ---- C ----
  // Each wave lays 16 rows of its sums down in LDS at a time and takes them up again row by row, eight neighbouring
  // columns a lane: whole lines of C, and the scales of a lane's columns stay in registers.
  __syncthreads();
  constexpr int PITCH = 64 * G::NB + 4, COLS = GATED ? 32 * G::NB : 64 * G::NB, PIECES = COLS / 8, AT_ONCE = 64 / PIECES;
  int32_t* sums = reinterpret_cast<int32_t*>(smem) + wave * 16 * PITCH;
  static_assert(G::WAVES * 16 * PITCH * 4 <= G::RING, "the sums take the ring's place");
  const int piece = lane % PIECES;
  const int at = GATED ? (piece >> 1) * 32 + (piece & 1) * 8 : piece * 8;  // among the wave's columns of B
  const int n = n0 + wn * COLS + piece * 8, valid = min(8, a.n - n);
  float sb[8], bias[8], sb2[GATED ? 8 : 1], bias2[GATED ? 8 : 1];
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const int c = wn * 64 * G::NB + at + q;
    sb[q] = sb_l[c];
    bias[q] = bias_l[c];
    if constexpr (GATED) {
      sb2[q] = sb_l[c + 16];
      bias2[q] = bias_l[c + 16];
    }
  }
  const int64_t c_mat = GROUPED ? 0 : rows.mat * a.scb;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) *reinterpret_cast<v4i*>(sums + lr * PITCH + 16 * j + 4 * lg) = acc[i][j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll 2
    for (int r = lane / PIECES; r < 16; r += AT_ONCE) {
      const int lrow = wm * 64 + 16 * i + r, row = rows.row + lrow;
      if (row >= rows.end || valid <= 0) continue;
      const float sa = sa_l[lrow];
      const int32_t* x = sums + r * PITCH + at;
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = static_cast<float>(x[q]) * (sa * sb[q]) + bias[q];
      if constexpr (GATED) {
        if (row_bias) {
          for (int q = 0; q < 8; ++q) v[q] += bias_at(row, min(n + q, a.n - 1));
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          float u = static_cast<float>(x[16 + q]) * (sa * sb2[q]) + bias2[q];
          if (row_bias) u += bias_at(row, min(n + q, a.n - 1) + a.n);
          v[q] = silu(v[q]) * u;
        }
      } else {
        if (row_bias) {
          for (int q = 0; q < 8; ++q) v[q] += bias_at(row, min(n + q, a.n - 1));
        }
        if (a.act == PCAMD_ACT_GELU) {
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = activate(v[q], PCAMD_ACT_GELU);
        }
      }
      store8(a.c, a.c_dtype, c_mat + int64_t(row) * a.scm + n, valid, v);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <typename G, bool GROUPED, bool GATED>
int launch(const Args& a, hipStream_t st) {
  constexpr int OUT = GATED ? G::BN / 2 : G::BN;
  const int64_t tiles_n = (a.n + OUT - 1) / OUT;
  const int64_t tiles_m = GROUPED ? grouped_tiles(a.pairs, a.batch, G::BM) : (a.m + G::BM - 1) / G::BM;
  if (tiles_m * tiles_n > INT32_MAX / G::THREADS - 8 || (!GROUPED && a.batch > 65535))
    return set_error(PCAMD_ERR_UNSUPPORTED, "int8 product: too many tiles or matrices for one launch");
  auto kern = tiles_kernel<G, GROUPED, GATED>;
  static std::atomic<uint64_t> done{0};
  const int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(kern), G::LDS, st, done);
  if (rc != PCAMD_OK) return rc;
  const dim3 grid(static_cast<unsigned>((tiles_m * tiles_n + 7) / 8 * 8), GROUPED ? 1 : a.batch);
  kern<<<grid, G::THREADS, G::LDS, st>>>(a, static_cast<int>(tiles_m), static_cast<int>(tiles_n));
  return check_launch("tiles_kernel");
}

template <typename G>
int launch(const Args& a, bool grouped, hipStream_t st) {
  const bool gated = a.act == PCAMD_ACT_SWIGLU;
  if (grouped) return gated ? launch<G, true, true>(a, st) : launch<G, true, false>(a, st);
  return gated ? launch<G, false, true>(a, st) : launch<G, false, false>(a, st);
}

}  // namespace

// The copies' offsets are 32 bits wide from a tile's first row (the gathered A's: from its first row of all).
bool tiles_ok(const Args& a, bool grouped) {
  constexpr int64_t kMost = (int64_t{1} << 32) - (1 << 18);
  const int64_t rows_b = a.act == PCAMD_ACT_SWIGLU ? a.n + 256 : 256;
  return a.k > 0 && rows_b * a.ldb < kMost && (grouped ? a.a_rows : 256) * a.lda < kMost;
}

int launch_tiles(const Args& a, bool grouped, bool wide, hipStream_t st) {
  return wide ? launch<Wide>(a, grouped, st) : launch<Small>(a, grouped, st);
}

}  // namespace int8
}  // namespace pcamd
