// int8_bmm_rows.hip - int8 products of few rows, bound by the weights' bytes.
//
// A workgroup computes 16 RT rows by 16 CT columns of C. Its eight waves split
// k: wave w takes the 128-byte blocks w, w + 8, .. of every row, straight from
// memory into the operand registers of v_mfma_i32_16x16x64_i8 (lane 16 g + r
// holds 16 bytes of row r; which of the block's bytes they are is the same for
// both operands, and the order of a sum of whole numbers does not matter). The
// eight partial sums meet in LDS by integer atomics: exact, whatever their
// order.
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
  __shared__ int32_t sums[R * LD];
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
  for (int i = threadIdx.x; i < R * LD; i += kThreads) sums[i] = 0;

  const int8_t* pa[RT];
  const int8_t* pb[CT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
    pa[i] = a.a + (GROUPED ? 0 : rows.mat * a.sab) + a_row<GROUPED>(a, min(rows.row + 16 * i + r, rows.end - 1)) * a.lda + 16 * g;
#pragma unroll
  for (int j = 0; j < CT; ++j) {
    const int col = GATED ? min(n0 + 16 * (j >> 1) + r, a.n - 1) + (j & 1) * a.n : min(n0 + 16 * j + r, a.n - 1);
    pb[j] = a.b + rows.mat * a.sbb + int64_t(col) * a.ldb + 16 * g;
  }

  v4i acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j) acc[i][j] = v4i{0, 0, 0, 0};

  const int full = a.k / kBlock;  // whole blocks
  auto load = [&](const int8_t* p, int at) { return *reinterpret_cast<const v4i*>(p + at); };
  for (int kb = wave; kb < full; kb += kWaves) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = kb * kBlock + 64 * h;
      v4i fa[RT], fb[CT];
#pragma unroll
      for (int j = 0; j < CT; ++j) fb[j] = load(pb[j], at);
#pragma unroll
      for (int i = 0; i < RT; ++i) fa[i] = load(pa[i], at);
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[j], fa[i], acc[i][j], 0, 0, 0);
    }
  }
  // the last bytes of k: rows start at multiples of 16 bytes, so a 16-byte piece with a valid byte is the row's own or
  // its padding, which the masked A makes zeros of
  const int left = a.k - full * kBlock;
  if (left && wave == full % kWaves) {
    for (int h = 0; 64 * h < left; ++h) {
      const int at = full * kBlock + 64 * h, k0 = at + 16 * g;
      const bool in = k0 < a.k;
      v4i fa[RT], fb[CT];
#pragma unroll
      for (int j = 0; j < CT; ++j) fb[j] = in ? load(pb[j], at) : v4i{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < RT; ++i) fa[i] = in ? mask_tail(load(pa[i], at), k0, a.k) : v4i{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[j], fa[i], acc[i][j], 0, 0, 0);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) atomicAdd(&sums[(16 * i + r) * LD + 16 * j + 4 * g + q], acc[i][j][q]);
  __syncthreads();

  for (int i = threadIdx.x; i < R * OUT / 4; i += kThreads) {
    const int lr = i / (OUT / 4), row = rows.row + lr, c4 = 4 * (i % (OUT / 4)), n = n0 + c4;
    if (row >= rows.end || n >= a.n) continue;
    const int64_t arow = a_row<GROUPED>(a, row);
    const float sa = a.sa[(GROUPED ? 0 : rows.mat * a.ssab) + arow * a.ssam];
    const int valid = min(4, a.n - n);
    auto value = [&](int at, int col) {
      float x = static_cast<float>(sums[lr * LD + at]) * (sa * a.sb[rows.mat * a.ssbb + int64_t(col) * a.ssbn]);
      if (a.bias)
        x += load_as(a.bias, a.bias_dtype, rows.mat * a.sbiasb + (GROUPED ? 0 : row * a.sbiasm) + int64_t(col) * a.sbiasn);
      return x;
    };
    float v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[q] = 0.0f;
      if (q >= valid) continue;
      if constexpr (GATED) {
        const int at = 32 * (c4 >> 4) + (c4 & 15) + q;
        v[q] = silu(value(at, n + q)) * value(at + 16, n + q + a.n);
      } else {
        v[q] = activate(value(c4 + q, n + q), a.act);
      }
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
  if (grouped && gated) rows_kernel<RT, CT, true, true><<<grid, kThreads, 0, st>>>(a, tn);
  else if (grouped) rows_kernel<RT, CT, true, false><<<grid, kThreads, 0, st>>>(a, tn);
  else if (gated) rows_kernel<RT, CT, false, true><<<grid, kThreads, 0, st>>>(a, tn);
  else rows_kernel<RT, CT, false, false><<<grid, kThreads, 0, st>>>(a, tn);
  return check_launch("rows_kernel");
}

}  // namespace

int launch_rows(const Args& a, bool grouped, hipStream_t st) {
  const int64_t rows = !grouped ? a.m : a.batch ? (a.pairs + a.batch - 1) / a.batch : a.pairs;
  if (rows <= 16) return launch<1, 2>(a, grouped, st);
  if (rows <= 32) return launch<2, 2>(a, grouped, st);
  return launch<4, 4>(a, grouped, st);
}

}  // namespace int8
}  // namespace pcamd
