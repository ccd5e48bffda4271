// int8_bmm.hip - C entries of the int8 products (int8_bmm.h) and the choice of kernel.
#include "int8_bmm.h"

namespace pcamd {
namespace int8 {
namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_common(int64_t n, int64_t k, int c_dtype, const void* bias, int bias_dtype, int act) {
  if (n < 0 || k < 0) return set_error(PCAMD_ERR_INVALID, "negative size");
  if (c_dtype != kF32 && c_dtype != kBF16 && c_dtype != kF16)
    return set_error(PCAMD_ERR_INVALID, "output dtype must be fp32, bf16 or fp16, got code %d", c_dtype);
  if (bias && bias_dtype != kF32 && bias_dtype != kBF16 && bias_dtype != kF16)
    return set_error(PCAMD_ERR_INVALID, "bias dtype must be fp32, bf16 or fp16, got code %d", bias_dtype);
  if (act != PCAMD_ACT_NONE && act != PCAMD_ACT_GELU && act != PCAMD_ACT_SWIGLU)
    return set_error(PCAMD_ERR_INVALID, "unknown activation code %d", act);
  if (k > kMaxK)
    return set_error(PCAMD_ERR_UNSUPPORTED, "int8 product: k up to %lld (sums of 32 bits), got %lld", (long long)kMaxK,
                     (long long)k);
  if (n > (INT32_MAX - 65536) / 2) return set_error(PCAMD_ERR_UNSUPPORTED, "int8 product: too many columns");
  return PCAMD_OK;
}

// rows of an operand: 16-byte aligned, and at least as far apart as they are long
int check_operand(const char* name, const void* p, int64_t rows, int64_t stride, int64_t k) {
  if (k && (!aligned16(p) || (rows > 1 && (stride % 16 || stride < k))))
    return set_error(PCAMD_ERR_INVALID, "rows of %s must be 16-byte aligned and not overlap", name);
  return PCAMD_OK;
}

}  // namespace
}  // namespace int8
}  // namespace pcamd

extern "C" int pcamd_bmm_int8(const void* a, const void* b, int64_t batch, int64_t m, int64_t n, int64_t k, int64_t sab,
                              int64_t sam, int64_t sbb, int64_t sbn, void* c, int c_dtype, int64_t scb, int64_t scm,
                              const void* bias, int bias_dtype, int64_t sbiasb, int64_t sbiasm, int64_t sbiasn,
                              const float* sa, int64_t ssab, int64_t ssam, const float* sb, int64_t ssbb, int64_t ssbn,
                              int activation, void* stream) {
  using namespace pcamd;
  clear_error();
  int rc = int8::check_common(n, k, c_dtype, bias, bias_dtype, activation);
  if (rc != PCAMD_OK) return rc;
  if (batch < 0 || m < 0) return set_error(PCAMD_ERR_INVALID, "negative size");
  if (batch == 0 || m == 0 || n == 0) return PCAMD_OK;
  if (!c || !sa || !sb || (k && (!a || !b))) return set_error(PCAMD_ERR_INVALID, "null pointer");
  const int64_t cols = activation == PCAMD_ACT_SWIGLU ? 2 * n : n;
  if ((rc = int8::check_operand("a", a, m, sam, k)) != PCAMD_OK) return rc;
  if ((rc = int8::check_operand("b", b, cols, sbn, k)) != PCAMD_OK) return rc;
  if (k && batch > 1 && (sab % 16 || sbb % 16))
    return set_error(PCAMD_ERR_INVALID, "matrices must start at multiples of 16 bytes");
  if (m > INT32_MAX - 65536) return set_error(PCAMD_ERR_UNSUPPORTED, "int8 product: too many rows");
  int8::Args x{};
  x.a = static_cast<const int8_t*>(a); x.b = static_cast<const int8_t*>(b); x.c = c; x.bias = bias; x.sa = sa; x.sb = sb;
  x.sab = sab; x.lda = m > 1 ? sam : 0; x.sbb = sbb; x.ldb = cols > 1 ? sbn : 0; x.scb = scb; x.scm = scm;
  x.sbiasb = sbiasb; x.sbiasm = sbiasm; x.sbiasn = sbiasn;
  x.ssab = ssab; x.ssam = ssam; x.ssbb = ssbb; x.ssbn = ssbn;
  x.m = static_cast<int32_t>(m); x.n = static_cast<int32_t>(n); x.k = static_cast<int32_t>(k);
  x.batch = static_cast<int32_t>(batch < INT32_MAX ? batch : INT32_MAX);
  x.c_dtype = c_dtype; x.bias_dtype = bias_dtype; x.act = activation;
  return int8::launch_rows(x, false, static_cast<hipStream_t>(stream));
}

extern "C" int pcamd_expert_bmm_int8(const void* a, int64_t a_rows, const void* b, int64_t experts, int64_t n, int64_t k,
                                     int64_t sam, int64_t sbe, int64_t sbn, void* c, int c_dtype, int64_t scm,
                                     const void* bias, int bias_dtype, int64_t sbiase, int64_t sbiasn, const float* sa,
                                     int64_t ssam, const float* sb, int64_t ssbe, int64_t ssbn, const int32_t* starts,
                                     const int32_t* order, int64_t pairs, int64_t choices, int activation, void* stream) {
  using namespace pcamd;
  clear_error();
  int rc = int8::check_common(n, k, c_dtype, bias, bias_dtype, activation);
  if (rc != PCAMD_OK) return rc;
  if (pairs < 0 || experts < 0 || a_rows < 0) return set_error(PCAMD_ERR_INVALID, "negative size");
  if (order ? choices < 1 || a_rows > pairs || (a_rows && pairs / a_rows < choices) || a_rows * choices != pairs
            : a_rows != pairs)
    return set_error(PCAMD_ERR_INVALID, "a has %lld rows, which do not go with %lld pairs", (long long)a_rows,
                     (long long)pairs);
  if (pairs == 0 || n == 0) return PCAMD_OK;
  if (!c || !sa || !starts || (experts && (!sb || (k && (!a || !b)))))
    return set_error(PCAMD_ERR_INVALID, "null pointer");
  const int64_t cols = activation == PCAMD_ACT_SWIGLU ? 2 * n : n;
  if ((rc = int8::check_operand("a", a, a_rows, sam, k)) != PCAMD_OK) return rc;
  if ((rc = int8::check_operand("b", b, cols, sbn, k)) != PCAMD_OK) return rc;
  if (k && experts > 1 && sbe % 16) return set_error(PCAMD_ERR_INVALID, "matrices must start at multiples of 16 bytes");
  if (pairs > INT32_MAX - 65536 || experts > 65535)
    return set_error(PCAMD_ERR_UNSUPPORTED, "int8 product: too many pairs or experts");
  int8::Args x{};
  x.a = static_cast<const int8_t*>(a); x.b = static_cast<const int8_t*>(b); x.c = c; x.bias = bias; x.sa = sa; x.sb = sb;
  x.lda = a_rows > 1 ? sam : 0; x.sbb = sbe; x.ldb = cols > 1 ? sbn : 0; x.scm = scm;
  x.sbiasb = sbiase; x.sbiasn = sbiasn; x.ssam = ssam; x.ssbb = ssbe; x.ssbn = ssbn;
  x.n = static_cast<int32_t>(n); x.k = static_cast<int32_t>(k); x.batch = static_cast<int32_t>(experts);
  x.c_dtype = c_dtype; x.bias_dtype = bias_dtype; x.act = activation;
  x.starts = starts; x.order = order; x.pairs = static_cast<int32_t>(pairs);
  x.choices = static_cast<int32_t>(choices); x.a_rows = static_cast<int32_t>(a_rows);
  return int8::launch_rows(x, true, static_cast<hipStream_t>(stream));
}
