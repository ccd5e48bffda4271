// int8_bmm_rows.hip - int8 products of few rows, bound by the weights' bytes.
//
// A workgroup computes 16 RT rows by 16 CT columns of C. Its eight waves split
// k: wave w takes the 128-byte blocks w, w + 8, .. of every row, straight from
// memory into the operand registers of v_mfma_i32_16x16x64_i8 (lane 16 g + r
// holds 16 bytes of row r; which of the block's bytes they are is the same for
// both operands, and the order of a sum of whole numbers does not matter). The
// eight partial sums meet in LDS.
#include "int8_bmm.h"

namespace pcamd {
namespace int8 {
namespace {

constexpr int kWaves = 8, kThreads = kWaves * 64;
constexpr int kBlock = 128;  // bytes of k a wave takes at once

template <int RT, int CT, bool GROUPED, bool GATED>
__global__ __launch_bounds__(kThreads) void rows_kernel(Args a, int tiles_n) {
  constexpr int R = 16 * RT, CN = 16 * CT, LD = CN + 4;  // columns of B here; of C half as many where gated
  constexpr int OUT = GATED ? CN / 2 : CN;
  constexpr int PARTS = RT * CT > 8 ? 4 : 8;             // partial sums in LDS at a time
  __shared__ int32_t parts[PARTS][R * LD];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = (blockIdx.x % tiles_n) * OUT;
  Rows rows;
  if constexpr (GROUPED) {
    if (!grouped_tile(a, blockIdx.x / tiles_n, R, rows)) return;
  } else {
    rows.mat = blockIdx.y;
    rows.row = (blockIdx.x / tiles_n) * R;
    rows.end = min(rows.row + R, a.m);
    rows.zeros = false;
  }
  const int64_t c_mat = GROUPED ? 0 : rows.mat * a.scb;
  if (GROUPED && rows.zeros) {
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = threadIdx.x; i < R * OUT / 4; i += kThreads) {
      const int row = rows.row + i / (OUT / 4), n = n0 + 4 * (i % (OUT / 4));
      if (row < rows.end && n < a.n) store4(a.c, a.c_dtype, int64_t(row) * a.scm + n, a.n - n, zero);
    }
    return;
  }

  const int8_t* pa[RT];
  const int8_t* pb[CT];
#pragma unroll
  for (int j = 0; j < CT; ++j) {
    const int col = GATED ? min(n0 + 16 * (j >> 1) + r, a.n - 1) + (j & 1) * a.n : min(n0 + 16 * j + r, a.n - 1);
    pb[j] = a.b + rows.mat * a.sbb + int64_t(col) * a.ldb + 16 * g;
  }
#pragma unroll
  for (int i = 0; i < RT; ++i)
    pa[i] = a.a + (GROUPED ? 0 : rows.mat * a.sab) + a_row<GROUPED>(a, min(rows.row + 16 * i + r, rows.end - 1)) * a.lda + 16 * g;

  v4i acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j) acc[i][j] = v4i{0, 0, 0, 0};

  // Pieces of 64 bytes of k: piece p is half p & 1 of the wave's block p >> 1. Two are on their way while one is
  // multiplied: four took registers that more waves use better (192 rows through 64 experts of 4096 x 7168, 16 x 32
  // tiles: 232 us with two, 284 with four).
  constexpr int AHEAD = 2;
  const int full = a.k / kBlock;  // whole blocks
  const int pieces = 2 * (full > wave ? (full - wave + kWaves - 1) / kWaves : 0);
  struct Piece {
    v4i a[RT], b[CT];
  };
  Piece ring[AHEAD];
  auto load = [&](Piece& x, int p) {
    const int at = (wave + (p >> 1) * kWaves) * kBlock + (p & 1) * 64;
#pragma unroll
    for (int j = 0; j < CT; ++j) x.b[j] = *reinterpret_cast<const v4i*>(pb[j] + at);
#pragma unroll
    for (int i = 0; i < RT; ++i) x.a[i] = *reinterpret_cast<const v4i*>(pa[i] + at);
  };
  auto multiply = [&](const Piece& x) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.b[j], x.a[i], acc[i][j], 0, 0, 0);
  };
#pragma unroll
  for (int q = 0; q < AHEAD; ++q)
    if (q < pieces) load(ring[q], q);
  int p = 0;
  for (; p + 2 * AHEAD <= pieces; p += AHEAD) {
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      multiply(ring[q]);
      load(ring[q], p + q + AHEAD);
    }
  }
  for (; p < pieces; p += AHEAD) {
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      if (p + q < pieces) multiply(ring[q]);
      if (p + q + AHEAD < pieces) load(ring[q], p + q + AHEAD);
    }
  }
  // the last bytes of k: rows start at multiples of 16 bytes, so a 16-byte piece with a valid byte is the row's own or
  // its padding, which the masked A makes zeros of
  const int left = a.k - full * kBlock;
  if (left && wave == full % kWaves) {
    for (int h = 0; 64 * h < left; ++h) {
      const int at = full * kBlock + 64 * h, k0 = at + 16 * g;
      const bool in = k0 < a.k;
      Piece x;
#pragma unroll
      for (int j = 0; j < CT; ++j) x.b[j] = in ? *reinterpret_cast<const v4i*>(pb[j] + at) : v4i{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < RT; ++i)
        x.a[i] = in ? mask_tail(*reinterpret_cast<const v4i*>(pa[i] + at), k0, a.k) : v4i{0, 0, 0, 0};
      multiply(x);
    }
  }
  // The waves' sums meet in LDS (whole numbers: any order). With PARTS = 4 the upper four waves hand theirs to the lower.
  auto at_of = [&](int i, int j) { return (16 * i + r) * LD + 16 * j + 4 * g; };
  if constexpr (PARTS == 4) {
    if (wave >= 4) {
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) *reinterpret_cast<v4i*>(&parts[wave - 4][at_of(i, j)]) = acc[i][j];
    }
    __syncthreads();
    if (wave < 4) {
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) acc[i][j] += *reinterpret_cast<v4i*>(&parts[wave][at_of(i, j)]);
    }
  }
  if (wave < PARTS) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j) *reinterpret_cast<v4i*>(&parts[wave][at_of(i, j)]) = acc[i][j];
  }
  __syncthreads();

  for (int i = threadIdx.x; i < R * OUT / 4; i += kThreads) {
    const int lr = i / (OUT / 4), row = rows.row + lr, c4 = 4 * (i % (OUT / 4)), n = n0 + c4;
    if (row >= rows.end || n >= a.n) continue;
    const int64_t arow = a_row<GROUPED>(a, row);
    const float sa = a.sa[(GROUPED ? 0 : rows.mat * a.ssab) + arow * a.ssam];
    const int valid = min(4, a.n - n);
    auto total = [&](int at) {
      v4i sum = *reinterpret_cast<const v4i*>(&parts[0][lr * LD + at]);
#pragma unroll
      for (int w = 1; w < PARTS; ++w) sum += *reinterpret_cast<const v4i*>(&parts[w][lr * LD + at]);
      return sum;
    };
    auto value = [&](int x, int col) {
      float y = static_cast<float>(x) * (sa * a.sb[rows.mat * a.ssbb + int64_t(col) * a.ssbn]);
      if (a.bias)
        y += load_as(a.bias, a.bias_dtype, rows.mat * a.sbiasb + (GROUPED ? 0 : row * a.sbiasm) + int64_t(col) * a.sbiasn);
      return y;
    };
    const int at = GATED ? 32 * (c4 >> 4) + (c4 & 15) : c4;
    const v4i x = total(at);
    v4i up = x;
    if constexpr (GATED) up = total(at + 16);
    float v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int col = min(n + q, a.n - 1);
      if constexpr (GATED) v[q] = silu(value(x[q], col)) * value(up[q], col + a.n);
      else v[q] = activate(value(x[q], col), a.act);
    }
    store4(a.c, a.c_dtype, c_mat + int64_t(row) * a.scm + n, valid, v);
  }
}

template <int RT, int CT>
int launch(const Args& a, bool grouped, hipStream_t st) {
  const bool gated = a.act == PCAMD_ACT_SWIGLU;
  const int64_t out = gated ? 8 * CT : 16 * CT, tiles_n = (a.n + out - 1) / out;
  const int64_t tiles_m = grouped ? grouped_tiles(a.pairs, a.batch, 16 * RT) : (a.m + 16 * RT - 1) / (16 * RT);
  if (tiles_m * tiles_n > UINT32_MAX / kThreads || (!grouped && a.batch > 65535))
    return set_error(PCAMD_ERR_UNSUPPORTED, "int8 product: too many tiles or matrices for one launch");
  const dim3 grid(static_cast<unsigned>(tiles_m * tiles_n), grouped ? 1 : a.batch);
  const int tn = static_cast<int>(tiles_n);
  if constexpr (CT > 1) {
    if (grouped && gated) rows_kernel<RT, CT, true, true><<<grid, kThreads, 0, st>>>(a, tn);
    else if (gated) rows_kernel<RT, CT, false, true><<<grid, kThreads, 0, st>>>(a, tn);
    if (gated) return check_launch("rows_kernel");
  }
  if (grouped) rows_kernel<RT, CT, true, false><<<grid, kThreads, 0, st>>>(a, tn);
  else rows_kernel<RT, CT, false, false><<<grid, kThreads, 0, st>>>(a, tn);
  return check_launch("rows_kernel");
}

}  // namespace

int launch_rows(const Args& a, bool grouped, int rt, int ct, hipStream_t st) {
  if (rt == 1 && ct == 1) return launch<1, 1>(a, grouped, st);
  if (rt == 1 && ct == 2) return launch<1, 2>(a, grouped, st);
  if (rt == 1) return launch<1, 4>(a, grouped, st);
  if (rt == 2 && ct == 1) return launch<2, 1>(a, grouped, st);
  if (rt == 2 && ct == 2) return launch<2, 2>(a, grouped, st);
  if (rt == 2) return launch<2, 4>(a, grouped, st);
  return launch<4, 4>(a, grouped, st);
}

}  // namespace int8
}  // namespace pcamd
