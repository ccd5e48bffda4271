// int8_bmm.hip - C entries of the int8 products (int8_bmm.h) and the choice of kernel.
#include <algorithm>
#include <cmath>

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

// What a form of tiles would take, in us, from the tile counts. The constants are fitted to timings on MI355X; us as
// modelled / measured (rotating inputs, a captured graph of calls):
//   rows 16 rt x 16 ct: a tile costs more with rt + ct, as its waves load that many operands;
//     24 x 14336 x 4096: 2 x 4 14.5 / 16.8, 2 x 2 16.4 / 19.2, 4 x 4 18.9 / 18.9;
//     64 x 4096 x 4096: 2 x 2 10.7 / 10.5, 4 x 4 18.9 / 19.4;
//     192 rows by 64 experts of 7168 x 4096: 1 x 2 196 / 220, 2 x 4 270 / 226
//   128 x 128: two workgroups a CU; 512 x 14336 x 4096 43.5 / 49.3, 2048 x 4096 x 4096 48.0 / 46.4,
//     1024 x 4096 x 4096 30.0 / 29.4
//   256 x 256: 2048 x 4096 x 4096 53.0 / 48.6, 4096 x 4096 x 4096 61.0 / 63.4, 8192 x 14336 x 4096 379 / 432
// Of 24 drawn plain products the chosen form took 1.03 times the fastest on average and 1.30 at worst, of 24 drawn
// grouped ones 1.04 and 1.19.
struct Form {
  int rows, cols;  // of C, before a gated activation halves the columns
  int rt, ct;      // of the rows kernel; 0: the tiled one
};
// in the order that the test entries count in
constexpr Form kForms[] = {{16, 16, 1, 1}, {16, 32, 1, 2}, {16, 64, 1, 4}, {32, 16, 2, 1}, {32, 32, 2, 2},
                           {32, 64, 2, 4}, {64, 64, 4, 4}, {128, 128, 0, 0}, {256, 256, 0, 0}};

double cost(const Form& f, double tiles, double cus, double k) {
  k /= 4096.0;
  const double rounds = tiles / cus;
  if (f.rt) {
    const double s = f.rt + f.ct, each = 1.1 * s + 0.08 * s * s;
    // Many small tiles share a CU and cover each other's start and end: 68 rows by 128 experts of 3344 x 968 take 28 / 24
    // as 1 x 2, and without the factor would go to 1 x 4, at 31 / 32.
    return 5.0 + k * each * (rounds >= 4.0 ? (s <= 3.0 ? 0.85 * rounds : rounds) : std::ceil(rounds));
  }
  if (f.rows == 128) {
    const double pairs = std::floor(rounds / 2.0), rest = rounds - 2.0 * pairs;
    return 6.0 + k * (42.0 * pairs + (rest == 0.0 ? 0.0 : rest <= 1.0 ? 21.0 + 3.0 * rest : 6.0 + 18.0 * rest));
  }
  return 8.0 + k * std::ceil(rounds) * (37.0 + 16.0 * std::min(1.0, rounds));
}

// The cheapest form, or the one with the given place in kForms. Of grouped rows the host knows no more than their
// number: groups of one size are assumed, each with half a tile more than it fills.
int launch(const Args& a, bool grouped, int form, hipStream_t st) {
  const bool gated = a.act == PCAMD_ACT_SWIGLU, tiled = tiles_ok(a, grouped);
  const int found = device_cu_count(st);
  const double cus = found > 0 ? found : 256.0;
  const Form* best = nullptr;
  double least = 0.0;
  for (const Form& f : kForms) {
    if ((!f.rt && !tiled) || (gated && f.ct == 1) || (form >= 0 && &f - kForms != form)) continue;
    const double n = std::ceil(double(a.n) * (gated ? 2 : 1) / f.cols);
    double m = std::ceil(double(a.m) / f.rows) * a.batch;
    if (grouped) {
      const double used = std::max(1, std::min(a.batch, a.pairs));
      m = used * std::max(1.0, a.pairs / used / f.rows + 0.5);
    }
    const double c = cost(f, m * n, cus, a.k);
    if (!best || c < least) {
      best = &f;
      least = c;
    }
  }
  if (!best) return set_error(PCAMD_ERR_UNSUPPORTED, "int8 product: form %d does not take this call", form);
  if (best->rt) return launch_rows(a, grouped, best->rt, best->ct, st);
  return launch_tiles(a, grouped, best->rows == 256, st);
}

int bmm(int form, const void* a, const void* b, int64_t batch, int64_t m, int64_t n, int64_t k, int64_t sab,
        int64_t sam, int64_t sbb, int64_t sbn, void* c, int c_dtype, int64_t scb, int64_t scm, const void* bias,
        int bias_dtype, int64_t sbiasb, int64_t sbiasm, int64_t sbiasn, const float* sa, int64_t ssab, int64_t ssam,
        const float* sb, int64_t ssbb, int64_t ssbn, int activation, void* stream) {
  clear_error();
  int rc = check_common(n, k, c_dtype, bias, bias_dtype, activation);
  if (rc != PCAMD_OK) return rc;
  if (batch < 0 || m < 0) return set_error(PCAMD_ERR_INVALID, "negative size");
  if (batch == 0 || m == 0 || n == 0) return PCAMD_OK;
  if (!c || !sa || !sb || (k && (!a || !b))) return set_error(PCAMD_ERR_INVALID, "null pointer");
  const int64_t cols = activation == PCAMD_ACT_SWIGLU ? 2 * n : n;
  if ((rc = check_operand("a", a, m, sam, k)) != PCAMD_OK) return rc;
  if ((rc = check_operand("b", b, cols, sbn, k)) != PCAMD_OK) return rc;
  if (k && batch > 1 && (sab % 16 || sbb % 16))
    return set_error(PCAMD_ERR_INVALID, "matrices must start at multiples of 16 bytes");
  if (m > INT32_MAX - 65536) return set_error(PCAMD_ERR_UNSUPPORTED, "int8 product: too many rows");
  Args x{};
  x.a = static_cast<const int8_t*>(a); x.b = static_cast<const int8_t*>(b); x.c = c; x.bias = bias; x.sa = sa; x.sb = sb;
  x.sab = sab; x.lda = m > 1 ? sam : 0; x.sbb = sbb; x.ldb = cols > 1 ? sbn : 0; x.scb = scb; x.scm = scm;
  x.sbiasb = sbiasb; x.sbiasm = sbiasm; x.sbiasn = sbiasn;
  x.ssab = ssab; x.ssam = ssam; x.ssbb = ssbb; x.ssbn = ssbn;
  x.m = static_cast<int32_t>(m); x.n = static_cast<int32_t>(n); x.k = static_cast<int32_t>(k);
  x.batch = static_cast<int32_t>(batch < INT32_MAX ? batch : INT32_MAX);
  x.c_dtype = c_dtype; x.bias_dtype = bias_dtype; x.act = activation;
  return launch(x, false, form, static_cast<hipStream_t>(stream));
}

int expert_bmm(int form, const void* a, int64_t a_rows, const void* b, int64_t experts, int64_t n, int64_t k,
               int64_t sam, int64_t sbe, int64_t sbn, void* c, int c_dtype, int64_t scm, const void* bias,
               int bias_dtype, int64_t sbiase, int64_t sbiasn, const float* sa, int64_t ssam, const float* sb,
               int64_t ssbe, int64_t ssbn, const int32_t* starts, const int32_t* order, int64_t pairs,
               int64_t choices, int activation, void* stream) {
  clear_error();
  int rc = check_common(n, k, c_dtype, bias, bias_dtype, activation);
  if (rc != PCAMD_OK) return rc;
  if (pairs < 0 || experts < 0 || a_rows < 0) return set_error(PCAMD_ERR_INVALID, "negative size");
  if (pairs == 0 && choices == 0) return PCAMD_OK;  // tokens, if any, without a choice: no rows
  if (order ? choices < 1 || a_rows > pairs || (a_rows && pairs / a_rows < choices) || a_rows * choices != pairs
            : a_rows != pairs)
    return set_error(PCAMD_ERR_INVALID, "a has %lld rows, which do not go with %lld pairs", (long long)a_rows,
                     (long long)pairs);
  if (pairs == 0 || n == 0) return PCAMD_OK;
  if (!c || !sa || !starts || (experts && (!sb || (k && (!a || !b)))))
    return set_error(PCAMD_ERR_INVALID, "null pointer");
  const int64_t cols = activation == PCAMD_ACT_SWIGLU ? 2 * n : n;
  if ((rc = check_operand("a", a, a_rows, sam, k)) != PCAMD_OK) return rc;
  if ((rc = check_operand("b", b, cols, sbn, k)) != PCAMD_OK) return rc;
  if (k && experts > 1 && sbe % 16) return set_error(PCAMD_ERR_INVALID, "matrices must start at multiples of 16 bytes");
  if (pairs > INT32_MAX - 65536 || experts > 65535)
    return set_error(PCAMD_ERR_UNSUPPORTED, "int8 product: too many pairs or experts");
  Args x{};
  x.a = static_cast<const int8_t*>(a); x.b = static_cast<const int8_t*>(b); x.c = c; x.bias = bias; x.sa = sa; x.sb = sb;
  x.lda = a_rows > 1 ? sam : 0; x.sbb = sbe; x.ldb = cols > 1 ? sbn : 0; x.scm = scm;
  x.sbiasb = sbiase; x.sbiasn = sbiasn; x.ssam = ssam; x.ssbb = ssbe; x.ssbn = ssbn;
  x.n = static_cast<int32_t>(n); x.k = static_cast<int32_t>(k); x.batch = static_cast<int32_t>(experts);
  x.c_dtype = c_dtype; x.bias_dtype = bias_dtype; x.act = activation;
  x.starts = starts; x.order = order; x.pairs = static_cast<int32_t>(pairs);
  x.choices = static_cast<int32_t>(choices); x.a_rows = static_cast<int32_t>(a_rows);
  return launch(x, true, form, static_cast<hipStream_t>(stream));
}

}  // namespace
}  // namespace int8
}  // namespace pcamd

extern "C" int pcamd_bmm_int8(const void* a, const void* b, int64_t batch, int64_t m, int64_t n, int64_t k,
                              int64_t sab, int64_t sam, int64_t sbb, int64_t sbn, void* c, int c_dtype, int64_t scb,
                              int64_t scm, const void* bias, int bias_dtype, int64_t sbiasb, int64_t sbiasm,
                              int64_t sbiasn, const float* sa, int64_t ssab, int64_t ssam, const float* sb,
                              int64_t ssbb, int64_t ssbn, int activation, void* stream) {
  return pcamd::int8::bmm(-1, a, b, batch, m, n, k, sab, sam, sbb, sbn, c, c_dtype, scb, scm, bias, bias_dtype,
                          sbiasb, sbiasm, sbiasn, sa, ssab, ssam, sb, ssbb, ssbn, activation, stream);
}

extern "C" int pcamd_selftest_bmm_int8(int form, const void* a, const void* b, int64_t batch, int64_t m, int64_t n,
                                       int64_t k, int64_t sab, int64_t sam, int64_t sbb, int64_t sbn, void* c,
                                       int c_dtype, int64_t scb, int64_t scm, const void* bias, int bias_dtype,
                                       int64_t sbiasb, int64_t sbiasm, int64_t sbiasn, const float* sa, int64_t ssab,
                                       int64_t ssam, const float* sb, int64_t ssbb, int64_t ssbn, int activation,
                                       void* stream) {
  return pcamd::int8::bmm(form, a, b, batch, m, n, k, sab, sam, sbb, sbn, c, c_dtype, scb, scm, bias, bias_dtype,
                          sbiasb, sbiasm, sbiasn, sa, ssab, ssam, sb, ssbb, ssbn, activation, stream);
}

extern "C" int pcamd_expert_bmm_int8(const void* a, int64_t a_rows, const void* b, int64_t experts, int64_t n,
                                     int64_t k, int64_t sam, int64_t sbe, int64_t sbn, void* c, int c_dtype,
                                     int64_t scm, const void* bias, int bias_dtype, int64_t sbiase, int64_t sbiasn,
                                     const float* sa, int64_t ssam, const float* sb, int64_t ssbe, int64_t ssbn,
                                     const int32_t* starts, const int32_t* order, int64_t pairs, int64_t choices,
                                     int activation, void* stream) {
  return pcamd::int8::expert_bmm(-1, a, a_rows, b, experts, n, k, sam, sbe, sbn, c, c_dtype, scm, bias, bias_dtype,
                                 sbiase, sbiasn, sa, ssam, sb, ssbe, ssbn, starts, order, pairs, choices, activation,
                                 stream);
}

extern "C" int pcamd_selftest_expert_bmm_int8(int form, const void* a, int64_t a_rows, const void* b,
                                              int64_t experts, int64_t n, int64_t k, int64_t sam, int64_t sbe,
                                              int64_t sbn, void* c, int c_dtype, int64_t scm, const void* bias,
                                              int bias_dtype, int64_t sbiase, int64_t sbiasn, const float* sa,
                                              int64_t ssam, const float* sb, int64_t ssbe, int64_t ssbn,
                                              const int32_t* starts, const int32_t* order, int64_t pairs,
                                              int64_t choices, int activation, void* stream) {
  return pcamd::int8::expert_bmm(form, a, a_rows, b, experts, n, k, sam, sbe, sbn, c, c_dtype, scm, bias, bias_dtype,
                                 sbiase, sbiasn, sa, ssam, sb, ssbe, ssbn, starts, order, pairs, choices, activation,
                                 stream);
}
