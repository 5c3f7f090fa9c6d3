/*
 * tgis_w8.h -- products with 8-bit weights of libtgis_engine.so, on the caller's stream.
 *
 * Numbers v of a group (128 neighbours of a row of activations; a block of 128 x 128 of a weight matrix; smaller at the ends) are e4m3 codes
 * c and one fp32 scale s:
 *     s = max(max |v| * (1 / 448), 2^-126),   c = e4m3(v / s) (nearest, ties to even),   a number stands for c * s,
 * with 1 / 448, the product and the quotient rounded to fp32.  A group that holds a NaN or an infinity has a NaN for its scale and zeros for
 * codes: what is summed over it is NaN, in its row (activations) or its 128 columns (weights).  Codes and scales made elsewhere in this form
 * (a checkpoint of block-scaled e4m3) serve as well, whatever rule their scales follow.
 *
 * Conventions: every pointer inside the records and every other one is device memory of the current device, the records themselves are
 * host memory and read before the call returns; `stream` is a cudaStream_t.  Calls return after the launch: 0, or < 0 with
 * tgis_w8_last_error() (per thread) and nothing launched.  They may be captured into CUDA graphs and keep no workspace: calls may run at
 * the same time.  Inputs and outputs do not overlap but for residual_out, which may be the residual or x.  A result is the same in every call; its
 * last bits depend on the call's sizes (which kernel, how many pieces of k), never on the other rows.
 * *status (int32, may be NULL) collects TGIS_W8_* bits.
 */
#ifndef TGIS_W8_H_
#define TGIS_W8_H_
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

#define TGIS_W8_GROUP 128
#define TGIS_W8_BF16 0
#define TGIS_W8_F32 1
#define TGIS_W8_MAX_K 131072       /* numbers of a row */
#define TGIS_W8_STALLED 1          /* a wait inside a kernel ran out: the results of the call are not to be used */

/* codes [n][ld] (ld a multiple of 16, codes on 16 bytes), scales [(n + 127) / 128][(k + 127) / 128] */
typedef struct {
  void* codes;
  float* scales;
  int64_t ld;
  int32_t n, k;
} tgis_w8_matrix;

/* codes [t][ld] (ld a multiple of 16, codes on 16 bytes), scales [(k + 127) / 128][lds] (lds >= t) */
typedef struct {
  void* codes;
  float* scales;
  int64_t ld, lds;
  int32_t t, k;
} tgis_w8_rows;

/* Rows of x [t, ldx] (TGIS_W8_BF16 or _F32) in 8 bits; t, k are the record's, its ld no less than k rounded up to 128 (the rest of a row's last
 * group is zeroed).  residual (may be NULL; type of x): r = x + residual, rounded to the type and stored at residual_out (may be residual
 * or x itself), takes x's place.  norm [k] (bf16, may be NULL): the row is v = r * norm / sqrt(mean r^2 + eps): the codes are those of r * norm and
 * its groups' scales are multiplied by the root's reciprocal, both in fp32 (a row whose sum of squares passes 2^128 has scales of 0). */
int tgis_w8_quantise_rows(const void* x, int32_t type, int64_t ldx, const void* norm, float eps, const void* residual, int64_t ldr,
                          void* residual_out, int64_t ldro, const tgis_w8_rows* out, void* stream);

/* A weight matrix w [n, ldw] (TGIS_W8_BF16 or _F32) in 8 bits; its record's ld no less than k rounded up to 128 (zeroed there). */
int tgis_w8_quantise_weight(const void* w, int32_t type, int64_t ldw, const tgis_w8_matrix* out, void* stream);

/* y[t, n] (TGIS_W8_BF16 or _F32, rows of ldy numbers) = x w^T: every group's sum of code products in fp32, times the product of both scales, groups added in
 * fp32.  That product of scales is one number of fp32: below 2^-126 it keeps fewer bits, above 2^128 it is an infinity (and NaN where the sum is 0). */
int tgis_w8_product(const tgis_w8_rows* x, const tgis_w8_matrix* w, void* y, int32_t type, int64_t ldy, int32_t* status, void* stream);

/* h = g / (1 + exp(-g)) * u, g = x gate^T, u = x up^T, in 8 bits (out: t = x's, k = the matrices' n, ld as for tgis_w8_quantise_rows); g, u and h are
 * fp32 before that.  exp and the quotient are within (4 + 1.2 |g|) * 2^-22 of what they stand for (below -87 the quotient may be 0), and codes are e4m3(h * fl(1 / s)) where other rows'
 * are of the rounded quotient: that product is off by 3 * 2^-24 at most, so a code is the quotient's neighbour where that lies so near to the middle of two, a few in a million. */
int tgis_w8_gated(const tgis_w8_rows* x, const tgis_w8_matrix* gate, const tgis_w8_matrix* up, const tgis_w8_rows* out, int32_t* status,
                  void* stream);

/* tgis_w8_gated into `hidden`, then tgis_w8_product of it with `down` */
int tgis_w8_feed_forward(const tgis_w8_rows* x, const tgis_w8_matrix* gate, const tgis_w8_matrix* up, const tgis_w8_matrix* down,
                         const tgis_w8_rows* hidden, void* y, int32_t type, int64_t ldy, int32_t* status, void* stream);

const char* tgis_w8_last_error(void);

#ifdef __cplusplus
}
#endif
#endif
