// latent_prefill.hip - attention of packed sequences with keys and values
// expanded from the latent vectors: head h of token t has the key
// [k_nope[t, h] | k_rope[t]], its rotary part shared by all heads, and the
// value v[t, h].
//
//   s[i, j] = scale * q[i] . k[j], j <= i + (keys - queries) where causal
//   o[i] = sum_j softmax(s[i])[j] v[j],   lse[i] = log sum_j exp(s[i, j])
//
// One workgroup holds 128 query rows of one head (32 a wave) and walks over
// the keys it sees in tiles of 64 with a running maximum and sum.
#include <hip/hip_runtime.h>

#include <atomic>
#include <cstdint>

#include "abi_util.h"
#include "attn_common.h"

namespace pcamd {
namespace prefill {

using namespace attn;

constexpr int NT = 256;
constexpr int BM = 128, BN = 64;

struct Args {
  const void* q; const void* k; const void* kr; const void* v;
  int64_t sqt, sqh, skt, skh, srt, svt, svh;
  const int32_t* cu_q; const int32_t* cu_k;
  void* out; int64_t sot, soh;
  float* lse; int64_t slt, slh;
  int64_t total_q, total_k;
  int sequences, heads, causal;
  float scale_log2;
};

struct Tile {
  int64_t q0, k0;  // first token of the sequence's queries and keys
  int qn, kn, row0;
};

PCAMD_DEV int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// Sequence i: its queries and keys, within the tensors whatever the offsets
// say. "Sequence" n (past the last) is the tokens behind the last one, which
// see no key and get zeros.
PCAMD_DEV Tile sequence(const Args& a, int i) {
  Tile t;
  t.q0 = clamp64(a.cu_q[i], 0, a.total_q);
  const int64_t q1 = i < a.sequences ? clamp64(a.cu_q[i + 1], t.q0, a.total_q) : a.total_q;
  t.qn = static_cast<int>(q1 - t.q0);
  t.k0 = t.kn = 0;
  if (i < a.sequences) {
    t.k0 = clamp64(a.cu_k[i], 0, a.total_k);
    t.kn = static_cast<int>(clamp64(a.cu_k[i + 1], t.k0, a.total_k) - t.k0);
  }
  t.row0 = 0;
  return t;
}

template <int DT, int DN, int DR, int DV>
struct Kernel {
  typedef Mfma<DT, 32> M;
  static constexpr int DK = DN + DR;
  static constexpr int CN = DN / 8, CK = DK / 8, CV = DV / 8;
  static constexpr int KS = DK / 16, OB = DV / 32, SUB = BN / 32;
  static constexpr int KT = BN * DK * 2, VT = BN * DV * 2;
  static constexpr int LDS = KT + VT;

  static PCAMD_DEV void run(const Args& a, uint8_t* lds) {
    __shared__ int wave_total[NT / 64];
    __shared__ int found[2];
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int h = lane / 32, ln = lane % 32;
    const int head = blockIdx.x % a.heads;
    const int want = blockIdx.x / a.heads;

    // ---- the tile's sequence: a running count of tiles over the sequences
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
        found[1] = mine - 1 - (want - before);  // the longest rows of a causal sequence first
      }
      base += total;
      __syncthreads();
      if (found[0] >= 0) break;
    }
    if (found[0] < 0) return;
    Tile t = sequence(a, found[0]);
    t.row0 = found[1] * BM;

    // ---- this lane's row
    const int row = t.row0 + wave * 32 + ln;
    const bool live = row < t.qn;
    const int past = t.kn - t.qn;
    const int limit = !live ? 0 : a.causal ? row + past + 1 : t.kn;
    uint4 q[KS];
    {
      const uint16_t* p = static_cast<const uint16_t*>(a.q) + (t.q0 + row) * a.sqt + head * a.sqh;
#pragma unroll
      for (int k = 0; k < KS; ++k)
        q[k] = live ? *reinterpret_cast<const uint4*>(p + 16 * k + 8 * h) : make_uint4(0, 0, 0, 0);
    }
    const int last = t.row0 + BM < t.qn ? t.row0 + BM : t.qn;  // end of the tile's rows
    int keys = a.causal ? last + past : t.kn;
    if (keys > t.kn) keys = t.kn;
    const uint16_t* kn = static_cast<const uint16_t*>(a.k) + t.k0 * a.skt + head * a.skh;
    const uint16_t* kr = static_cast<const uint16_t*>(a.kr) + t.k0 * a.srt;
    const uint16_t* kv = static_cast<const uint16_t*>(a.v) + t.k0 * a.svt + head * a.svh;

    f32x16 o[OB];
#pragma unroll
    for (int j = 0; j < OB; ++j) o[j] = f32x16{};
    float m = kNoMax, l = 0.0f;
    for (int t0 = 0; t0 < keys; t0 += BN) {
      __syncthreads();
      for (int j = tid; j < BN * CK; j += NT) {
        const int r = j / CK, c = j % CK;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (t0 + r < t.kn)
          x = *reinterpret_cast<const uint4*>(c < CN ? kn + (t0 + r) * a.skt + 8 * c : kr + (t0 + r) * a.srt + 8 * (c - CN));
        *reinterpret_cast<uint4*>(lds + r * (DK * 2) + ((c ^ swz<CK>(r)) << 4)) = x;
      }
      for (int j = tid; j < BN * CV; j += NT) {
        const int r = j / CV, c = j % CV;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (t0 + r < t.kn) x = *reinterpret_cast<const uint4*>(kv + (t0 + r) * a.svt + 8 * c);
        *reinterpret_cast<uint4*>(lds + KT + r * (DV * 2) + ((c ^ swz_v<CV>(r)) << 4)) = x;
      }
      __syncthreads();

      f32x16 s[SUB];
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub) {
        s[sub] = f32x16{};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const int r = sub * 32 + ln;
          const uint4 x = *reinterpret_cast<const uint4*>(lds + r * (DK * 2) + (((2 * k + h) ^ swz<CK>(r)) << 4));
          s[sub] = M::mul(x, q[k], s[sub]);
        }
      }
      float top = m;
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = t0 + sub * 32 + (r / 4) * 8 + 4 * h + r % 4;
          s[sub][r] = key < limit ? s[sub][r] * a.scale_log2 : -INFINITY;
          top = fmaxf(top, s[sub][r]);
        }
      top = row_max<32>(top);
      const float alpha = exp2f(m - top);
      m = top;
      float part = 0.0f;
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[sub][r] = exp2f(s[sub][r] - m);
          part += s[sub][r];
        }
      l = l * alpha + part;
#pragma unroll
      for (int j = 0; j < OB; ++j) o[j] *= alpha;
#pragma unroll
      for (int kk = 0; kk < BN / 16; ++kk) {
        const f32x16& x = s[kk / 2];
        const int r0 = (kk & 1) * 8;
        const uint4 p = make_uint4(Elem<DT>::narrow2(x[r0], x[r0 + 1]), Elem<DT>::narrow2(x[r0 + 2], x[r0 + 3]),
                                   Elem<DT>::narrow2(x[r0 + 4], x[r0 + 5]), Elem<DT>::narrow2(x[r0 + 6], x[r0 + 7]));
#pragma unroll
        for (int j = 0; j < OB; ++j) {
          const int i16 = lane % 16, g16 = lane / 16;
          const int col = j * 32 + 16 * (g16 & 1) + 4 * (i16 & 3);
          uint2 w[2];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int r = kk * 16 + y * 8 + 4 * h + i16 / 4;
            w[y] = read_tr4(lds + KT + r * (DV * 2) + (((col >> 3) ^ swz_v<CV>(r)) << 4) + ((col & 4) << 1));
          }
          o[j] = M::mul(make_uint4(w[0].x, w[0].y, w[1].x, w[1].y), p, o[j]);
        }
      }
    }
    l = row_sum<32>(l);
    if (!live) return;
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : NAN;
    uint16_t* out = static_cast<uint16_t*>(a.out) + (t.q0 + row) * a.sot + head * a.soh;
#pragma unroll
    for (int j = 0; j < OB; ++j)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint2 w = make_uint2(Elem<DT>::narrow2(o[j][4 * y] * inv, o[j][4 * y + 1] * inv),
                                   Elem<DT>::narrow2(o[j][4 * y + 2] * inv, o[j][4 * y + 3] * inv));
        *reinterpret_cast<uint2*>(out + 32 * j + 8 * y + 4 * h) = w;
      }
    if (a.lse && h == 0) a.lse[(t.q0 + row) * a.slt + head * a.slh] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
  }
};

template <int DT, int DN, int DR, int DV>
__global__ __launch_bounds__(NT, 2) void prefill_kernel(Args a) {
  extern __shared__ __align__(16) uint8_t lds[];
  Kernel<DT, DN, DR, DV>::run(a, lds);
}

template <int DT, int DN, int DR, int DV>
int launch(const Args& a, int64_t grid, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  const auto kern = prefill_kernel<DT, DN, DR, DV>;
  constexpr int bytes = Kernel<DT, DN, DR, DV>::LDS;
  const int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(kern), bytes, st, done);
  if (rc != PCAMD_OK) return rc;
  kern<<<static_cast<uint32_t>(grid), NT, bytes, st>>>(a);
  return check_launch("prefill_kernel");
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
  if (total_q > INT32_MAX || total_k > INT32_MAX || sequences > INT32_MAX / 2)
    return set_error(PCAMD_ERR_UNSUPPORTED, "latent prefill: more than 2^31 - 1 tokens");
  if (total_q == 0 || heads == 0) return PCAMD_OK;
  if (!q || !cu_q || !cu_k || !out || (total_k && (!k_nope || !k_rope || !v)))
    return set_error(PCAMD_ERR_INVALID, "null pointer");
  auto odd = [](const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; };
  if (odd(q, 16) || odd(k_nope, 16) || odd(k_rope, 16) || odd(v, 16) || odd(out, 8) || sqt % 8 || sqh % 8 || skt % 8 ||
      skh % 8 || srt % 8 || svt % 8 || svh % 8 || sot % 4 || soh % 4)
    return set_error(PCAMD_ERR_INVALID, "rows of queries, keys and values must be 16-byte aligned, of the output 8-byte");
  const int64_t grid = heads * (total_q / prefill::BM + sequences + 1);
  if (grid >= (int64_t{1} << 32) / prefill::NT)
    return set_error(PCAMD_ERR_UNSUPPORTED, "latent prefill: grid too large (%lld workgroups)", (long long)grid);
  prefill::Args a{q, k_nope, k_rope, v, sqt, sqh, skt, skh, srt, svt, svh, cu_q, cu_k, out, sot, soh, lse, slt, slh,
                  total_q, total_k, static_cast<int>(sequences), static_cast<int>(heads), causal != 0,
                  softmax_scale * attn::kLog2e};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == kBF16)
    return wide ? prefill::launch<kBF16, 128, 64, 128>(a, grid, st) : prefill::launch<kBF16, 64, 32, 64>(a, grid, st);
  return wide ? prefill::launch<kF16, 128, 64, 128>(a, grid, st) : prefill::launch<kF16, 64, 32, 64>(a, grid, st);
}
