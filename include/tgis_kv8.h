/*
 * tgis_kv8.h -- the 8-bit paged cache of libtgis_engine.so and the attention that reads it, on the caller's stream.
 *
 * A stored row (one token, one key / value head, 128 numbers x) is 128 e4m3 codes c and one fp32 scale s:
 *     s = max(max |x| * (1 / 448), 2^-126),   c = e4m3(x / s) (nearest, ties to even),   the row stands for c * s,
 * with 1 / 448, the product and the quotient rounded to fp32.
 * A row that holds a NaN or an infinity is stored with a NaN for its scale and zeros for codes: whoever sees it gets NaN, whoever does
 * not gets what it would have got without it.  Finite rows of any size cost those that do not see them, or give them no weight, nothing either.
 * Numbers of a query count to 2^-39 of its row's largest.
 *
 * Memory of one layer: `pages` [n_pages][n_kv][TGIS_KV8_PAGE_BYTES], 16-byte aligned, 32 tokens a page; slot = page * 32 + place.  It is
 * filled with zeros before the first use and written by tgis_kv8_write (or copied from another such cache) alone: that keeps
 * every code a number, which the attention counts on for places that no row was written to.
 *
 * Conventions: every pointer is device memory of the current device unless marked host, `stream` is a cudaStream_t.  Calls return after
 * the launch: 0, or < 0 with tgis_kv8_last_error() (per thread) and nothing launched.  They may be captured into CUDA graphs; lengths,
 * slots and tables are read on the device when the work runs, so a replay sees what they hold then.  What the host cannot check is
 * checked there: nothing is read or written out of range, and *status (int32, may be NULL) collects TGIS_KV8_BAD_* bits.
 */
#ifndef TGIS_KV8_H_
#define TGIS_KV8_H_
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

#define TGIS_KV8_PAGE_TOKENS 32
#define TGIS_KV8_PAGE_BYTES 8448   /* per head: 4096 key codes, 4096 value codes, 32 key scales, 32 value scales */
#define TGIS_KV8_MAX_TREE 64       /* drafted tokens of one sequence */
#define TGIS_KV8_MAX_SEQS 4096

#define TGIS_KV8_BAD_SLOT 1        /* a slot behind the last page: the row was not stored / was read as zeros */
#define TGIS_KV8_BAD_POSITION 2    /* a position outside the rotation table: its nearest row was taken */
#define TGIS_KV8_BAD_SEQ 4         /* a sequence record that contradicts the call: its rows were left as they were */
#define TGIS_KV8_BAD_PAGE 8        /* a page number outside the cache: its keys were left out */
#define TGIS_KV8_STALLED 16         /* a wait inside a kernel ran out: the results of the call are not to be used */

/* Queries and keys of qkv [T, ld] bf16 = [n_q query heads | n_kv key heads | n_kv value heads], 128 numbers each, are rotated by
 * cos_sin [n_positions][cos 64 | sin 64] bf16 at positions[t] (pairs i, i + 64; in fp32); the queries go to q_out [T, ldq] bf16 (may be
 * qkv itself; NULL: not wanted), keys and values as rows to slots[t] (< 0: not stored).  The slots >= 0 of one call differ. */
int tgis_kv8_write(void* pages, int32_t n_pages, int32_t n_kv, const void* qkv, int64_t ld, int32_t T, int32_t n_q, const int32_t* positions,
                   const int32_t* slots, const void* cos_sin, int32_t n_positions, void* q_out, int64_t ldq, int32_t* status, void* stream);

/* Rows at slots[t] as bf16: k_out [T, ldk], v_out [T, ldv], n_kv * 128 numbers a row (either may be NULL; slot < 0: zeros) */
int tgis_kv8_read(const void* pages, int32_t n_pages, int32_t n_kv, const int32_t* slots, int32_t T, void* k_out, int64_t ldk, void* v_out,
                  int64_t ldv, int32_t* status, void* stream);

/* Bytes of workspace that tgis_kv8_attention needs for these bounds (host only); < 0: bad arguments.  No fewer for more sequences, for more queries
 * of a sequence or for longer ones, and 43 MB at most: one for the largest of each that a program calls with serves all its calls. */
int64_t tgis_kv8_attention_workspace(int32_t T, int32_t n_seqs, int32_t n_q, int32_t n_kv, int32_t max_q, int32_t max_kv);

/* out[t, h] = sum_j softmax_j(scale * q[t, h] . k_j) v_j over the rows that the query sees, h's head being h / (n_q / n_kv).
 * seqs [n_seqs] of {q_start, q_len, kv_len, block_row}: queries q_start .. q_start + q_len - 1 are the last q_len of the sequence's kv_len
 * tokens, whose pages are block_table[block_row][0 .. (kv_len - 1) / 32].  tree NULL: query i sees tokens 0 .. kv_len - q_len + i.
 * tree [T]: the last q_len (<= 64) tokens are a draft; query t sees tokens 0 .. kv_len - q_len - 1 and those nodes j of the draft whose
 * bit j is set in tree[t] (its own has to be set to be seen).  A query that sees nothing gives zeros.  Rows of q and out [T, ld*] bf16
 * that no sequence names are not touched; no two sequences name the same.  max_q, max_kv: no sequence has more queries / tokens (host; they choose kernels and
 * shapes, so a captured call can be replayed for any lengths within them).  Calls that may run at the same time need workspaces of their own. */
int tgis_kv8_attention(const void* pages, int32_t n_pages, int32_t n_kv, const void* q, int64_t ldq, int32_t T, int32_t n_q, const int32_t* seqs,
                       int32_t n_seqs, const int32_t* block_table, int32_t bt_rows, int32_t bt_stride, const uint64_t* tree, float scale,
                       int32_t max_q, int32_t max_kv, void* out, int64_t ldo, void* workspace, int64_t workspace_bytes, int32_t* status,
                       void* stream);

const char* tgis_kv8_last_error(void);

#ifdef __cplusplus
}
#endif
#endif
