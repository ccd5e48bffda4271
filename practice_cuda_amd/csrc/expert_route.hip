// expert_route.hip - tokens sorted by expert and back.
//
// A token t has `choices` experts; pair p = t * choices + j is its j-th choice.
//   sort:     order[place] = pair, pairs of expert e at starts[e] .. starts[e + 1] - 1 in
//             their own order, pairs without an expert behind them all;
//             place[pair] = its place, or -1 - place without an expert
//   dispatch: out[place] = x[order[place] / choices], zeros without an expert
//   combine:  out[t] = sum_j w[t, j] y[place[t, j]]   (fp32, j ascending)
//             d y[place[t, j]] = w[t, j] g[t],  d w[t, j] = y[place[t, j]] . g[t]
// The gradient of dispatch is combine with weights of one.
//
// The sort counts: each chunk of pairs is counted by expert, and a pair's place
// is its expert's start, plus what earlier chunks, earlier waves of its chunk
// and earlier lanes of its wave hold of that expert. Every count is a sum of
// whole numbers in a fixed order, so the result is the stable sort, each time.
//
// The row movers are bound by memory: a workgroup takes one token, so x and g
// are read once however many choices there are, and each pair's row is written
// (read) once.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "abi_util.h"
#include "fp8_common.h"

namespace pcamd {
namespace route {

// ---------------------------------------------------------------------------
// sort
// ---------------------------------------------------------------------------
constexpr int kMaxExperts = 1024;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kMaxChunks = 128;

struct SortArgs {
  const void* ids;
  int64_t pairs;
  int32_t* order;
  int32_t* place;
  int32_t* starts;
  int32_t* counts;  // [chunks][experts + 1] where there are several chunks
  int32_t experts, chunks, chunk;  // chunk: pairs a chunk, a multiple of kSortThreads
};

// key of a pair: its expert, or `experts` without one
template <int BYTES>
PCAMD_DEV int key_of(const SortArgs& a, int64_t pair) {
  const int64_t id = BYTES == 8 ? static_cast<const int64_t*>(a.ids)[pair]
                                : static_cast<int64_t>(static_cast<const int32_t*>(a.ids)[pair]);
  return id < 0 || id >= a.experts ? a.experts : static_cast<int>(id);
}

// lanes of this wave with the same key, among the active ones given by `live`
PCAMD_DEV uint64_t same_key(int key, uint64_t live, int bits) {
  uint64_t same = live;
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = __ballot((key >> b) & 1);
    same &= ((key >> b) & 1) ? set : ~set;
  }
  return same;
}

// Counts of each wave's share of a chunk: wave w takes the pairs [w, w + 1) * chunk / waves of it.
template <int BYTES>
PCAMD_DEV void count_waves(const SortArgs& a, int64_t first, int32_t* counts, int bits) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, keys = a.experts + 1;
  for (int i = threadIdx.x; i < kSortWaves * keys; i += kSortThreads) counts[i] = 0;
  __syncthreads();
  const int share = a.chunk / kSortWaves;
  for (int at = 0; at < share; at += 64) {
    const int64_t pair = first + wave * share + at + lane;
    const uint64_t live = __ballot(pair < a.pairs);
    if (live == 0) break;
    const int key = pair < a.pairs ? key_of<BYTES>(a, pair) : 0;
    const uint64_t same = same_key(key, live, bits);
    // the first lane of each key counts for all; keys of different leaders differ, and the row is the wave's own
    if (pair < a.pairs && (same & ((uint64_t{1} << lane) - 1)) == 0) counts[wave * keys + key] += __popcll(same);
  }
  __syncthreads();
}

template <int BYTES>
__global__ __launch_bounds__(kSortThreads) void count_kernel(SortArgs a) {
  extern __shared__ int32_t counts[];
  const int keys = a.experts + 1, bits = 32 - __clz(a.experts);
  count_waves<BYTES>(a, int64_t(blockIdx.x) * a.chunk, counts, bits);
  for (int e = threadIdx.x; e < keys; e += kSortThreads) {
    int sum = 0;
    for (int w = 0; w < kSortWaves; ++w) sum += counts[w * keys + e];
    a.counts[int64_t(blockIdx.x) * keys + e] = sum;
  }
}

template <int BYTES>
__global__ __launch_bounds__(kSortThreads) void place_kernel(SortArgs a) {
  extern __shared__ int32_t shared[];
  const int keys = a.experts + 1, bits = 32 - __clz(a.experts);
  int32_t* counts = shared;                       // [waves][keys]: then the next place of each wave and key
  int32_t* base = shared + kSortWaves * keys;     // [2 keys]: sums over the chunks, then this one's first places
  int32_t* sums = base + 2 * keys;                // [waves]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t first = int64_t(blockIdx.x) * a.chunk;
  count_waves<BYTES>(a, first, counts, bits);
  // All pairs of each key, and those of earlier chunks. Several threads share a key where there are few: each sums every
  // parts-th chunk (131288 pairs of 128 experts, 65 chunks: a call of 13 us, 26 with one thread a key).
  int32_t before[2] = {0, 0}, total[2] = {0, 0};  // of keys threadIdx.x and threadIdx.x + 1024
  if (a.chunks == 1) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int e = threadIdx.x + k * kSortThreads;
      for (int w = 0; e < keys && w < kSortWaves; ++w) total[k] += counts[w * keys + e];
    }
  } else {
    for (int i = threadIdx.x; i < 2 * keys; i += kSortThreads) base[i] = 0;
    __syncthreads();
    const int parts = keys < kSortThreads ? kSortThreads / keys : 1;
    for (int i = threadIdx.x; i < keys * parts; i += kSortThreads) {
      const int e = i % keys, part = i / keys;
      int32_t all = 0, ahead = 0;
#pragma unroll 8
      for (int c = part; c < a.chunks; c += parts) {
        const int n = a.counts[int64_t(c) * keys + e];
        all += n;
        ahead += c < static_cast<int>(blockIdx.x) ? n : 0;
      }
      atomicAdd(&base[e], all);  // whole numbers: any order
      atomicAdd(&base[keys + e], ahead);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int e = threadIdx.x + k * kSortThreads;
      if (e >= keys) continue;
      total[k] = base[e];
      before[k] = base[keys + e];
    }
    __syncthreads();
  }
  // exclusive sums over the keys
  int32_t start = 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    int32_t sum = total[k];
    for (int d = 1; d < 64; d <<= 1) {
      const int32_t up = __shfl_up(sum, d, 64);
      if (lane >= d) sum += up;
    }
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    int32_t ahead = start, all = 0;
    for (int w = 0; w < kSortWaves; ++w) {
      ahead += w < wave ? sums[w] : 0;
      all += sums[w];
    }
    const int e = threadIdx.x + k * kSortThreads;
    if (e < keys) {
      const int32_t s = ahead + sum - total[k];
      base[e] = s + before[k];
      if (blockIdx.x == 0) a.starts[e] = s;
    }
    start += all;
    __syncthreads();
  }
  for (int e = threadIdx.x; e < keys; e += kSortThreads) {
    int32_t next = base[e];
    for (int w = 0; w < kSortWaves; ++w) {
      const int32_t n = counts[w * keys + e];
      counts[w * keys + e] = next;
      next += n;
    }
  }
  __syncthreads();
  const int share = a.chunk / kSortWaves;
  for (int at = 0; at < share; at += 64) {
    const int64_t pair = first + wave * share + at + lane;
    const uint64_t live = __ballot(pair < a.pairs);
    if (live == 0) break;
    const int key = pair < a.pairs ? key_of<BYTES>(a, pair) : 0;
    const uint64_t same = same_key(key, live, bits);
    if (pair < a.pairs) {
      const uint64_t ahead = same & ((uint64_t{1} << lane) - 1);
      // every lane of a key reads its wave's next place before the first of them moves it on
      const int32_t place = counts[wave * keys + key] + __popcll(ahead);
      __builtin_amdgcn_wave_barrier();
      if (ahead == 0) counts[wave * keys + key] += __popcll(same);
      __builtin_amdgcn_wave_barrier();
      a.order[place] = static_cast<int32_t>(pair);
      a.place[pair] = key < a.experts ? place : -1 - place;
    }
  }
}

struct SortPlan {
  int chunks, chunk;
};

SortPlan sort_plan(int64_t pairs) {
  // one workgroup up to 4096 pairs, else chunks of 2048 and more, at most kMaxChunks of them
  int64_t chunk = pairs <= 4096 ? pairs : (pairs + kMaxChunks - 1) / kMaxChunks;
  if (pairs > 4096 && chunk < 2048) chunk = 2048;
  chunk = (chunk + kSortThreads - 1) / kSortThreads * kSortThreads;
  if (chunk == 0) chunk = kSortThreads;
  return {static_cast<int>((pairs + chunk - 1) / chunk), static_cast<int>(chunk)};
}

template <int BYTES>
int sort(SortArgs a, hipStream_t st) {
  const int lds = (kSortWaves * (a.experts + 1) + 2 * (a.experts + 1) + kSortWaves) * 4;
  if (a.chunks > 1) {
    static std::atomic<uint64_t> done{0};
    int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(count_kernel<BYTES>), 80 * 1024, st, done);
    if (rc != PCAMD_OK) return rc;
    count_kernel<BYTES><<<a.chunks, kSortThreads, lds, st>>>(a);
    rc = check_launch("count_kernel");
    if (rc != PCAMD_OK) return rc;
  }
  static std::atomic<uint64_t> done{0};
  const int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(place_kernel<BYTES>), 80 * 1024, st, done);
  if (rc != PCAMD_OK) return rc;
  place_kernel<BYTES><<<a.chunks ? a.chunks : 1, kSortThreads, lds, st>>>(a);
  return check_launch("place_kernel");
}

// ---------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;
constexpr int kMaxChoices = 128;

// V elements a lane: 16 bytes at once, or one element where rows are not 16-byte aligned
template <int DT, int V>
PCAMD_DEV void load_v(const void* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = load_one<DT>(p, 0);
  } else {
    const u32x4_t w = *static_cast<const u32x4_t*>(p);
    if constexpr (DT == kF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = DT == kBF16 ? bf16_lo(w[i]) : f16_lo(w[i]);
        v[2 * i + 1] = DT == kBF16 ? bf16_hi(w[i]) : f16_hi(w[i]);
      }
    }
  }
}

template <int DT>
PCAMD_DEV uint32_t pair16(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  if constexpr (DT == kBF16) {
    typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, b16x2));
  } else {
    typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, h16x2));
  }
}

template <int DT, int V, bool NT = false>
PCAMD_DEV void store_v(void* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    if constexpr (DT == kF32) *static_cast<float*>(p) = v[0];
    else if constexpr (DT == kBF16) *static_cast<__bf16*>(p) = static_cast<__bf16>(v[0]);
    else *static_cast<_Float16*>(p) = static_cast<_Float16>(v[0]);
  } else {
    u32x4_t w;
    if constexpr (DT == kF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pair16<DT>(v[2 * i], v[2 * i + 1]);
    }
    if constexpr (NT) __builtin_nontemporal_store(w, static_cast<u32x4_t*>(p));
    else *static_cast<u32x4_t*>(p) = w;
  }
}

PCAMD_DEV float weight_at(const void* w, int dt, int64_t i) {
  if (w == nullptr) return 1.0f;
  if (dt == kF32) return static_cast<const float*>(w)[i];
  return dt == kBF16 ? load_one<kBF16>(w, i) : load_one<kF16>(w, i);
}

struct RowArgs {
  const void* x;        // dispatch: tokens; combine: rows
  void* out;
  const int32_t* place;
  const void* weights;  // [tokens, choices], or null: ones
  const void* grad;     // backward of combine: [tokens, width]
  float* grad_weights;  // or null
  int64_t sx, so, sg;   // elements from row to row
  int64_t tokens, pairs;
  int32_t choices, width, w_dtype;
};

// A pair's row: its place, or with `used` false the place that -1 - place gives. Places past the pairs (of no sorted
// plan) are left alone.
struct Place {
  int64_t row;
  bool used, in;
};
PCAMD_DEV Place place_at(const RowArgs& a, int64_t t, int j) {
  const int32_t s = a.place[t * a.choices + j];
  Place p;
  p.used = s >= 0;
  p.row = p.used ? int64_t(s) : int64_t(-1) - s;
  p.in = p.row < a.pairs;
  return p;
}

PCAMD_DEV int64_t token_of() { return int64_t(blockIdx.y) * gridDim.x + blockIdx.x; }

// Rows are moved as words, whatever they hold.
template <typename W, bool NT>
__global__ __launch_bounds__(kRowThreads) void dispatch_kernel(RowArgs a, int words) {
  const int64_t t = token_of();
  if (t >= a.tokens) return;
  const W* x = static_cast<const W*>(a.x) + t * a.sx;
  for (int at = blockIdx.z * kRowThreads + threadIdx.x; at < words; at += gridDim.z * kRowThreads) {
    const W v = x[at];
    for (int j = 0; j < a.choices; ++j) {
      const Place p = place_at(a, t, j);
      W o = v;
      if (!p.used) o = W{};
      if (!p.in) continue;
      W* to = static_cast<W*>(a.out) + p.row * a.so + at;
      if constexpr (NT) __builtin_nontemporal_store(o, to);
      else *to = o;
    }
  }
}

template <int DT, int V>
__global__ __launch_bounds__(kRowThreads) void combine_kernel(RowArgs a) {
  const int64_t t = token_of();
  if (t >= a.tokens) return;
  for (int64_t at = (int64_t(blockIdx.z) * kRowThreads + threadIdx.x) * V; at < a.width;
       at += int64_t(gridDim.z) * kRowThreads * V) {
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0f;
    for (int j = 0; j < a.choices; ++j) {
      const Place p = place_at(a, t, j);
      if (!p.used || !p.in) continue;
      const float w = weight_at(a.weights, a.w_dtype, t * a.choices + j);
      float v[V];
      load_v<DT, V>(static_cast<const uint8_t*>(a.x) + (p.row * a.sx + at) * elem_bytes<DT>(), v);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += w * v[i];
    }
    store_v<DT, V>(static_cast<uint8_t*>(a.out) + (t * a.so + at) * elem_bytes<DT>(), sum);
  }
}

PCAMD_DEV float wave_sum(float v) {
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

// out: the rows' gradient, or null; the weights' products are summed in a fixed order
template <int DT, int V, bool NT>
__global__ __launch_bounds__(kRowThreads) void combine_back_kernel(RowArgs a) {
  extern __shared__ float dots[];  // [choices][waves]
  constexpr int kWaves = kRowThreads / 64;
  const int64_t t = token_of();
  if (t >= a.tokens) return;
  const int wave = threadIdx.x >> 6;
  if (a.grad_weights) {
    for (int i = threadIdx.x; i < a.choices * kWaves; i += kRowThreads) dots[i] = 0.0f;
    __syncthreads();
  }
  const int64_t block = int64_t(kRowThreads) * V;
  for (int64_t from = 0; from < a.width; from += block) {
    const int64_t at = from + int64_t(threadIdx.x) * V;
    const bool in = at < a.width;
    float g[V];
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] = 0.0f;
    if (in) load_v<DT, V>(static_cast<const uint8_t*>(a.grad) + (t * a.sg + at) * elem_bytes<DT>(), g);
    for (int j = 0; j < a.choices; ++j) {
      const Place p = place_at(a, t, j);
      if (!p.in) continue;
      if (a.out && in) {
        const float w = p.used ? weight_at(a.weights, a.w_dtype, t * a.choices + j) : 0.0f;
        float v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = p.used ? w * g[i] : 0.0f;
        store_v<DT, V, NT>(static_cast<uint8_t*>(a.out) + (p.row * a.so + at) * elem_bytes<DT>(), v);
      }
      if (a.grad_weights && p.used) {
        float dot = 0.0f;
        if (in) {
          float y[V];
          load_v<DT, V>(static_cast<const uint8_t*>(a.x) + (p.row * a.sx + at) * elem_bytes<DT>(), y);
#pragma unroll
          for (int i = 0; i < V; ++i) dot += y[i] * g[i];
        }
        dot = wave_sum(dot);
        if ((threadIdx.x & 63) == 0) dots[j * kWaves + wave] += dot;
      }
    }
  }
  if (a.grad_weights) {
    __syncthreads();
    for (int j = threadIdx.x; j < a.choices; j += kRowThreads) {
      float sum = 0.0f;
      for (int w = 0; w < kWaves; ++w) sum += dots[j * kWaves + w];
      a.grad_weights[t * a.choices + j] = sum;
    }
  }
}

// Rows that the 256 MB cache behind the L2 cannot hold for their reader go past it.
constexpr int64_t kStream = 128 << 20;
bool streams(int64_t bytes) { return bytes > kStream; }
template <int DT>
constexpr int64_t elem_size() { return DT == kF32 ? 4 : 2; }

// One workgroup a token, cut along the row where tokens are few.
dim3 row_grid(int64_t tokens, int64_t pieces, bool cut) {
  const int64_t x = tokens < (1 << 20) ? tokens : 1 << 20;
  const int64_t z = cut && tokens < 2048 ? (pieces < 64 ? pieces : 64) : 1;
  return dim3(static_cast<unsigned>(x), static_cast<unsigned>((tokens + x - 1) / x), static_cast<unsigned>(z ? z : 1));
}

// Whether rows of a tensor (address, elements from row to row) can be moved in 16-byte pieces
bool rows16(const void* p, int64_t stride, int size) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride * size) % 16 == 0;
}

int size_of(int dtype) { return dtype == kF32 ? 4 : 2; }

int check_rows(int dtype, int64_t tokens, int64_t choices, int64_t width, const void* place) {
  if (dtype != kF32 && dtype != kBF16 && dtype != kF16)
    return set_error(PCAMD_ERR_INVALID, "rows must be fp32, bf16 or fp16, got code %d", dtype);
  if (tokens < 0 || choices < 0 || width < 0) return set_error(PCAMD_ERR_INVALID, "negative size");
  if (choices > kMaxChoices)
    return set_error(PCAMD_ERR_UNSUPPORTED, "at most %d choices a token, got %lld", kMaxChoices, (long long)choices);
  // a thread's column steps on by up to 64 workgroups of 256, past the row's end, in 32 bits
  if (width > INT32_MAX - 65536 || (choices && tokens > INT32_MAX / choices))
    return set_error(PCAMD_ERR_UNSUPPORTED, "more than 2^31 - 1 pairs or 2^31 - 65537 columns");
  if (tokens && choices && !place) return set_error(PCAMD_ERR_INVALID, "null pointer");
  return PCAMD_OK;
}

template <int DT>
int combine(const RowArgs& a, bool wide, hipStream_t st) {
  constexpr int V = DT == kF32 ? 4 : 8;
  if (wide) {
    combine_kernel<DT, V><<<row_grid(a.tokens, (a.width + kRowThreads * V - 1) / (kRowThreads * V), true), kRowThreads,
                            0, st>>>(a);
  } else {
    combine_kernel<DT, 1><<<row_grid(a.tokens, (a.width + kRowThreads - 1) / kRowThreads, true), kRowThreads, 0, st>>>(a);
  }
  return check_launch("combine_kernel");
}

template <int DT>
int combine_back(const RowArgs& a, bool wide, hipStream_t st) {
  constexpr int V = DT == kF32 ? 4 : 8;
  const int lds = a.choices * (kRowThreads / 64) * 4;
  const dim3 grid = row_grid(a.tokens, 1, false);
  if (!wide) combine_back_kernel<DT, 1, false><<<grid, kRowThreads, lds, st>>>(a);
  else if (streams(a.pairs * a.width * elem_size<DT>())) combine_back_kernel<DT, V, true><<<grid, kRowThreads, lds, st>>>(a);
  else combine_back_kernel<DT, V, false><<<grid, kRowThreads, lds, st>>>(a);
  return check_launch("combine_back_kernel");
}

}  // namespace route
}  // namespace pcamd

extern "C" int64_t pcamd_expert_sort_workspace(int64_t pairs, int64_t experts) {
  using namespace pcamd;
  clear_error();
  if (pairs < 0 || experts < 0) return set_error(PCAMD_ERR_INVALID, "negative size");
  if (pairs > INT32_MAX || experts > route::kMaxExperts)
    return set_error(PCAMD_ERR_UNSUPPORTED, "expert sort: at most %d experts and 2^31 - 1 pairs, got %lld and %lld",
                     route::kMaxExperts, (long long)experts, (long long)pairs);
  const route::SortPlan p = route::sort_plan(pairs);
  return p.chunks > 1 ? int64_t(p.chunks) * (experts + 1) * 4 : 0;
}

extern "C" int pcamd_expert_sort(const void* ids, int id_bytes, int64_t pairs, int64_t experts, int32_t* order,
                                 int32_t* place, int32_t* starts, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  using namespace pcamd;
  const int64_t need = pcamd_expert_sort_workspace(pairs, experts);
  if (need < 0) return static_cast<int>(need);
  if (id_bytes != 4 && id_bytes != 8) return set_error(PCAMD_ERR_INVALID, "ids must be int32 or int64");
  if (!starts || (pairs && (!ids || !order || !place))) return set_error(PCAMD_ERR_INVALID, "null pointer");
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3)))
    return set_error(PCAMD_ERR_INVALID, "expert sort needs a workspace of %lld bytes, got %lld", (long long)need,
                     (long long)workspace_bytes);
  const route::SortPlan p = route::sort_plan(pairs);
  route::SortArgs a{ids, pairs, order, place, starts, static_cast<int32_t*>(workspace), static_cast<int32_t>(experts),
                    p.chunks ? p.chunks : 1, p.chunk};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return id_bytes == 8 ? route::sort<8>(a, st) : route::sort<4>(a, st);
}

extern "C" int pcamd_expert_dispatch(const void* x, int dtype, int64_t tokens, int64_t choices, int64_t width,
                                     int64_t sxt, const int32_t* place, void* out, int64_t sos, void* stream) {
  using namespace pcamd;
  clear_error();
  int rc = route::check_rows(dtype, tokens, choices, width, place);
  if (rc != PCAMD_OK) return rc;
  if (tokens == 0 || choices == 0 || width == 0) return PCAMD_OK;
  if (!x || !out) return set_error(PCAMD_ERR_INVALID, "null pointer");
  const int size = route::size_of(dtype);
  route::RowArgs a{};
  a.x = x; a.out = out; a.place = place; a.sx = sxt; a.so = sos;
  a.tokens = tokens; a.pairs = tokens * choices; a.choices = static_cast<int32_t>(choices); a.width = static_cast<int32_t>(width);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool wide = route::rows16(x, sxt, size) && route::rows16(out, sos, size) && width * size % 16 == 0;
  const int bytes = wide ? 16 : size, words = static_cast<int>(width * size / bytes);
  a.sx = sxt * size / bytes;
  a.so = sos * size / bytes;
  const dim3 grid = route::row_grid(tokens, (words + route::kRowThreads - 1) / route::kRowThreads, true);
  if (wide && route::streams(a.pairs * width * size))
    route::dispatch_kernel<u32x4_t, true><<<grid, route::kRowThreads, 0, st>>>(a, words);
  else if (wide) route::dispatch_kernel<u32x4_t, false><<<grid, route::kRowThreads, 0, st>>>(a, words);
  else if (size == 4) route::dispatch_kernel<uint32_t, false><<<grid, route::kRowThreads, 0, st>>>(a, words);
  else route::dispatch_kernel<uint16_t, false><<<grid, route::kRowThreads, 0, st>>>(a, words);
  return check_launch("dispatch_kernel");
}

extern "C" int pcamd_expert_combine(const void* rows, int dtype, int64_t tokens, int64_t choices, int64_t width,
                                    int64_t srs, const int32_t* place, const void* weights, int w_dtype, void* out,
                                    int64_t sot, void* stream) {
  using namespace pcamd;
  clear_error();
  int rc = route::check_rows(dtype, tokens, choices, width, place);
  if (rc != PCAMD_OK) return rc;
  if (weights && w_dtype != kF32 && w_dtype != kBF16 && w_dtype != kF16)
    return set_error(PCAMD_ERR_INVALID, "weights must be fp32, bf16 or fp16, got code %d", w_dtype);
  if (tokens == 0 || width == 0) return PCAMD_OK;
  if (!out || (choices && !rows)) return set_error(PCAMD_ERR_INVALID, "null pointer");
  const int size = route::size_of(dtype);
  route::RowArgs a{};
  a.x = rows; a.out = out; a.place = place; a.weights = weights; a.w_dtype = w_dtype; a.sx = srs; a.so = sot;
  a.tokens = tokens; a.pairs = tokens * choices; a.choices = static_cast<int32_t>(choices); a.width = static_cast<int32_t>(width);
  const bool wide = route::rows16(rows, srs, size) && route::rows16(out, sot, size) && width * size % 16 == 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == kF32) return route::combine<kF32>(a, wide, st);
  if (dtype == kBF16) return route::combine<kBF16>(a, wide, st);
  return route::combine<kF16>(a, wide, st);
}

extern "C" int pcamd_expert_combine_backward(const void* grad, const void* rows, int dtype, int64_t tokens,
                                             int64_t choices, int64_t width, int64_t sgt, int64_t srs,
                                             const int32_t* place, const void* weights, int w_dtype, void* grad_rows,
                                             int64_t sos, float* grad_weights, void* stream) {
  using namespace pcamd;
  clear_error();
  int rc = route::check_rows(dtype, tokens, choices, width, place);
  if (rc != PCAMD_OK) return rc;
  if (w_dtype != kF32 && w_dtype != kBF16 && w_dtype != kF16)
    return set_error(PCAMD_ERR_INVALID, "weights must be fp32, bf16 or fp16, got code %d", w_dtype);
  if (tokens == 0 || choices == 0) return PCAMD_OK;
  if ((width && (!grad || (grad_weights && !rows))) || (grad_rows && !weights))
    return set_error(PCAMD_ERR_INVALID, "null pointer");
  if (!grad_rows && !grad_weights) return PCAMD_OK;
  const int size = route::size_of(dtype);
  route::RowArgs a{};
  a.x = rows; a.out = grad_rows; a.place = place; a.weights = weights; a.w_dtype = w_dtype; a.grad = grad;
  a.grad_weights = grad_weights; a.sx = srs; a.so = sos; a.sg = sgt;
  a.tokens = tokens; a.pairs = tokens * choices; a.choices = static_cast<int32_t>(choices); a.width = static_cast<int32_t>(width);
  const bool wide = route::rows16(grad, sgt, size) && (!grad_weights || route::rows16(rows, srs, size)) &&
                    (!grad_rows || route::rows16(grad_rows, sos, size)) && width * size % 16 == 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == kF32) return route::combine_back<kF32>(a, wide, st);
  if (dtype == kBF16) return route::combine_back<kBF16>(a, wide, st);
  return route::combine_back<kF16>(a, wide, st);
}
