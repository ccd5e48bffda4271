// latent_decode.hip - C entry of attention over a paged latent cache.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "abi_util.h"
#include "fp8_common.h"
#include "latent_decode_args.h"

namespace pcamd {
namespace decode {

extern template int launch<kBF16, 512, 64>(const Args&, Shape, bool, hipStream_t);
extern template int launch<kBF16, 256, 32>(const Args&, Shape, bool, hipStream_t);
extern template int launch<kF16, 512, 64>(const Args&, Shape, bool, hipStream_t);
extern template int launch<kF16, 256, 32>(const Args&, Shape, bool, hipStream_t);

struct Layout {
  Shape shape;
  int64_t row_tiles, groups, min_steps;
  bool split;  // pieces may have to be joined
  int64_t join_bytes, ml_bytes, part_bytes;
  int64_t bytes() const { return split ? join_bytes + ml_bytes + part_bytes : 0; }
};

// From sizes that the host knows: the table's capacity bounds the lengths.
Layout lay_out(int64_t batch, int64_t rows, int64_t latent_dim, int64_t capacity) {
  Layout d;
  d.shape = shape_for(batch, rows);
  const int64_t tile = d.shape.tile_rows(), step = d.shape.step();
  d.row_tiles = (rows + tile - 1) / tile;
  const int64_t steps = capacity > step ? (capacity + step - 1) / step : 1;
  d.min_steps = step == 128 ? 1 : 2;
  const int64_t tiles = batch * d.row_tiles, cap = kWorkgroups / d.shape.split;
  d.groups = few_tiles(tiles, d.shape.split) ? tiles * ((steps + d.min_steps - 1) / d.min_steps)
                                             : (tiles * steps + d.min_steps - 1) / d.min_steps;
  if (d.groups < tiles) d.groups = tiles;
  if (d.groups > cap) d.groups = cap;
  d.split = steps > 1 && d.groups > 1;
  d.join_bytes = (d.groups * 16 + 255) / 256 * 256;
  d.ml_bytes = 2 * d.groups * tile * 8;
  d.part_bytes = 2 * d.groups * tile * latent_dim * 4;
  return d;
}

// A sequence's tokens: the kernels count them in 32 bits, and name tokens past the last one by up to a workgroup's
// tiles on their way (four steps of 128 tokens) ahead of cutting them to it.
constexpr int64_t kMaxTokens = (int64_t{1} << 31) - 1024;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_sizes(int64_t batch, int64_t new_tokens, int64_t heads, int64_t latent_dim, int64_t page_size,
                int64_t max_pages) {
  if (batch < 0 || new_tokens < 0 || heads < 0 || max_pages < 0)
    return set_error(PCAMD_ERR_INVALID, "negative size");
  if (page_size <= 0 || page_size > INT32_MAX) return set_error(PCAMD_ERR_INVALID, "bad page size");
  if (latent_dim != 512 && latent_dim != 256)
    return set_error(PCAMD_ERR_UNSUPPORTED, "latent width must be 512 or 256, got %lld", (long long)latent_dim);
  if (batch > (1 << 20) || new_tokens > (1 << 20) || heads > (1 << 20) || new_tokens * heads > (1 << 24) ||
      max_pages > kMaxTokens / page_size ||
      batch * ((new_tokens * heads + 15) / 16) * ((page_size * max_pages) / 32 + 32) > INT32_MAX)
    return set_error(PCAMD_ERR_UNSUPPORTED, "latent decode: too many rows or tokens a sequence");
  return PCAMD_OK;
}

}  // namespace decode
}  // namespace pcamd

extern "C" int64_t pcamd_latent_decode_workspace(int64_t batch, int64_t new_tokens, int64_t heads, int64_t latent_dim,
                                                 int64_t page_size, int64_t max_pages) {
  using namespace pcamd;
  clear_error();
  const int rc = decode::check_sizes(batch, new_tokens, heads, latent_dim, page_size, max_pages);
  if (rc != PCAMD_OK) return rc;
  if (batch == 0 || new_tokens * heads == 0) return 0;
  return decode::lay_out(batch, new_tokens * heads, latent_dim, page_size * max_pages).bytes();
}

extern "C" int pcamd_latent_decode(
    const void* q_latent, const void* q_rope, int dtype, int64_t batch, int64_t new_tokens, int64_t heads,
    int64_t latent_dim, int64_t rope_dim, int64_t qlb, int64_t qls, int64_t qlh, int64_t qrb, int64_t qrs, int64_t qrh,
    const void* cache_latent, int cache_dtype, int64_t clp, int64_t clt, const void* cache_rope, int64_t crp,
    int64_t crt, const float* cache_scale, int64_t csp, int64_t cst, int64_t pages, int64_t page_size,
    const int32_t* table, int64_t table_stride, int64_t max_pages, const int32_t* lens, void* out, int64_t ob,
    int64_t os, int64_t oh, float* lse, int64_t lb, int64_t ls, int64_t lh, float softmax_scale, void* workspace,
    int64_t workspace_bytes, void* stream) {
  using namespace pcamd;
  clear_error();
  const int rc = decode::check_sizes(batch, new_tokens, heads, latent_dim, page_size, max_pages);
  if (rc != PCAMD_OK) return rc;
  if (dtype != kBF16 && dtype != kF16) return set_error(PCAMD_ERR_INVALID, "queries must be bf16 or fp16, got code %d", dtype);
  if (cache_dtype != dtype && cache_dtype != kE4M3)
    return set_error(PCAMD_ERR_INVALID, "the cache holds the queries' type or e4m3fn, got code %d", cache_dtype);
  const bool f8 = cache_dtype == kE4M3;
  if (!(latent_dim == 512 && rope_dim == 64) && !(latent_dim == 256 && rope_dim == 32))
    return set_error(PCAMD_ERR_UNSUPPORTED, "latent and rotary widths must be 512 and 64, or 256 and 32; got %lld and %lld",
                     (long long)latent_dim, (long long)rope_dim);
  if (pages < 0) return set_error(PCAMD_ERR_INVALID, "negative size");
  if (batch == 0 || new_tokens == 0 || heads == 0) return PCAMD_OK;
  if (!q_latent || !q_rope || !lens || !out || (max_pages && !table) ||
      (pages && (!cache_latent || !cache_rope || (f8 && !cache_scale))))
    return set_error(PCAMD_ERR_INVALID, "null pointer");
  // a dimension with one place has any stride
  auto bad = [](int64_t places, int64_t stride, int64_t unit) { return places > 1 && stride % unit; };
  const int64_t per16 = f8 ? 16 : 8;
  if (!decode::aligned16(q_latent) || !decode::aligned16(q_rope) || !decode::aligned16(cache_latent) ||
      !decode::aligned16(cache_rope) || (reinterpret_cast<uintptr_t>(out) & 7) || bad(batch, qlb, 8) ||
      bad(new_tokens, qls, 8) || bad(heads, qlh, 8) || bad(batch, qrb, 8) || bad(new_tokens, qrs, 8) ||
      bad(heads, qrh, 8) || bad(pages, clp, per16) || bad(page_size, clt, per16) || bad(pages, crp, 8) ||
      bad(page_size, crt, 8) || bad(batch, ob, 4) || bad(new_tokens, os, 4) || bad(heads, oh, 4))
    return set_error(PCAMD_ERR_INVALID, "rows of queries and cache must be 16-byte aligned, of the output 8-byte");
  if (pages <= 1) clp = crp = csp = 0;
  if (page_size == 1) clt = crt = cst = 0;
  for (const int64_t stride : {clp, clt, crp, crt, csp, cst})
    if (stride < 0 || stride > INT32_MAX) return set_error(PCAMD_ERR_UNSUPPORTED, "latent decode: a cache stride past 2^31 elements");
  if (pages > UINT32_MAX) return set_error(PCAMD_ERR_UNSUPPORTED, "latent decode: more than 2^32 - 1 pages");
  decode::Args a{};
  a.q_latent = q_latent; a.q_rope = q_rope;
  a.qlb = qlb; a.qls = qls; a.qlh = qlh; a.qrb = qrb; a.qrs = qrs; a.qrh = qrh;
  a.latent = cache_latent; a.rope = cache_rope; a.scale = cache_scale;
  a.slp = static_cast<uint32_t>(clp); a.slt = static_cast<uint32_t>(clt);
  a.srp = static_cast<uint32_t>(crp); a.srt = static_cast<uint32_t>(crt);
  a.ssp = static_cast<uint32_t>(csp); a.sst = static_cast<uint32_t>(cst);
  a.table = table; a.table_stride = table_stride; a.lens = lens;
  a.out = out; a.ob = ob; a.os = os; a.oh = oh;
  a.lse = lse; a.lb = lb; a.ls = ls; a.lh = lh;
  a.batch = static_cast<int>(batch); a.pages = static_cast<uint32_t>(pages);
  a.new_tokens = static_cast<int>(new_tokens);
  a.heads = static_cast<int>(heads);
  a.rows = static_cast<int>(new_tokens * heads);
  a.page = static_cast<int>(page_size);
  while ((int64_t{1} << a.page_shift) < page_size) ++a.page_shift;
  a.page_mul = static_cast<uint32_t>(((int64_t{1} << (31 + a.page_shift)) + page_size - 1) / page_size);
  a.capacity = pages ? static_cast<int>(page_size * max_pages) : 0;  // no pool: every sequence is empty
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  const decode::Layout d = decode::lay_out(batch, a.rows, latent_dim, page_size * max_pages);
  a.row_tiles = static_cast<int>(d.row_tiles);
  a.groups = static_cast<int>(d.groups);
  a.min_steps = static_cast<int>(d.min_steps);
  if (d.split) {
    if (!workspace || workspace_bytes < d.bytes() || !decode::aligned16(workspace))
      return set_error(PCAMD_ERR_INVALID, "latent decode needs a 16-byte aligned workspace of %lld bytes, got %lld",
                       (long long)d.bytes(), (long long)workspace_bytes);
    uint8_t* w = static_cast<uint8_t*>(workspace);
    a.joins = reinterpret_cast<int4*>(w);
    a.part_ml = reinterpret_cast<float2*>(w + d.join_bytes);
    a.parts = reinterpret_cast<float*>(w + d.join_bytes + d.ml_bytes);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == kBF16)
    return latent_dim == 512 ? decode::launch<kBF16, 512, 64>(a, d.shape, f8, st)
                             : decode::launch<kBF16, 256, 32>(a, d.shape, f8, st);
  return latent_dim == 512 ? decode::launch<kF16, 512, 64>(a, d.shape, f8, st)
                           : decode::launch<kF16, 256, 32>(a, d.shape, f8, st);
}
