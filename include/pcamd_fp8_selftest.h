/*
 * pcamd_fp8_selftest.h - test and measurement entry points of
 * libpcamd_fp8.so.
 *
 * Not part of the product interface (include/pcamd_fp8.h): the test suite
 * calls them to pin the hardware fp8 conversion the quantizers use, and
 * bench.py to measure the plain-copy and narrowing ceilings the quantizers
 * are compared with. They have no counterpart in the reference (xuOAO/practice_cuda),
 * whose fp8 casts are Triton's `.to(fp8)`
 * (fp8_training/fp8_bench/kernels/quant/per_block.py:47).
 */
#ifndef PCAMD_FP8_SELFTEST_H
#define PCAMD_FP8_SELFTEST_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Device self-test of the fp32 -> fp8 conversion used by the quantizers:
 * compares the gfx950 hardware conversion with an integer restatement of
 * round-to-nearest-even over every fp32 bit pattern with |x| <= fp8 max.
 * result (device, 4 x uint32) receives {mismatches, first mismatching
 * pattern, checked count low 32 bits, 0}. fmt is PCAMD_E4M3FN (3) or
 * PCAMD_E5M2 (4). Returns 0 or a negative status (see pcamd_fp8.h).
 */
int pcamd_selftest_fp8_convert(int fmt, uint32_t *result, void *stream);

/*
 * Plain device copy y[i] = x[i] of `bytes` bytes (a multiple of 16, both
 * pointers 16-byte aligned) in the quantizers' streaming layout: one 16-byte
 * non-temporal load and store per lane, 256-thread workgroups. The 1 : 1
 * read/write ceiling the dual quantizer is measured against. Returns 0 or a
 * negative status.
 */
int pcamd_selftest_copy16(const void *x, void *y, int64_t bytes, void *stream);

/*
 * Plain device narrowing: y receives the high byte of every 16-bit element
 * of x (in_bytes a multiple of 16; x 16-byte and y 8-byte aligned; y holds
 * in_bytes / 2 bytes), in the 1 x 128 quantizer's streaming layout: each
 * lane loads two 16-byte chunks 64 apart (non-temporal) and then stores
 * their 8-byte results (non-temporal), 256-thread workgroups. The
 * quantizers' 2 : 1 read/write mix with no arithmetic, the ceiling they are
 * measured against.
 * Returns 0 or a negative status.
 */
int pcamd_selftest_narrow16(const void *x, void *y, int64_t in_bytes, void *stream);

/*
 * pcamd_bmm_int8 and pcamd_expert_bmm_int8 (pcamd_fp8.h) in one of the forms
 * that these choose from by size, so that the tests reach each form at any
 * size: 0 to 6 the kernel of few rows with tiles of 16 x 16, 16 x 32, 16 x 64,
 * 32 x 16, 32 x 32, 32 x 64 and 64 x 64, 7 and 8 the kernel of many rows with
 * 128 x 128 and 256 x 256; -1: as the product entries choose. A form that does
 * not take the call (the gated activation in forms 0 and 3, no inner size or
 * operands of 4 GiB in 7 and 8) returns PCAMD_ERR_UNSUPPORTED.
 */
int pcamd_selftest_bmm_int8(int form, const void *a, const void *b,
                            int64_t batch, int64_t m, int64_t n, int64_t k,
                            int64_t sab, int64_t sam, int64_t sbb, int64_t sbn,
                            void *c, int c_dtype, int64_t scb, int64_t scm,
                            const void *bias, int bias_dtype, int64_t sbiasb,
                            int64_t sbiasm, int64_t sbiasn, const float *sa,
                            int64_t ssab, int64_t ssam, const float *sb,
                            int64_t ssbb, int64_t ssbn, int activation,
                            void *stream);
int pcamd_selftest_expert_bmm_int8(int form, const void *a, int64_t a_rows,
                                   const void *b, int64_t experts, int64_t n,
                                   int64_t k, int64_t sam, int64_t sbe,
                                   int64_t sbn, void *c, int c_dtype,
                                   int64_t scm, const void *bias,
                                   int bias_dtype, int64_t sbiase,
                                   int64_t sbiasn, const float *sa,
                                   int64_t ssam, const float *sb, int64_t ssbe,
                                   int64_t ssbn, const int32_t *starts,
                                   const int32_t *order, int64_t pairs,
                                   int64_t choices, int activation,
                                   void *stream);

#ifdef __cplusplus
}
#endif

#endif /* PCAMD_FP8_SELFTEST_H */
