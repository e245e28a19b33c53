/*
 * vgemm_kv -- a paged key-value cache in the library's exact integer arithmetic: part of libvgemm.so, beside the decode-step
 * operators of vgemm_lm.h. No counterparts in the reference.
 *
 *   vgemm_kv_plan        block tables and slot maps from request lengths, on the GPU
 *   vgemm_kv_write       keys and values of tokens into the pages, 8 or 16 bits with a shift a row
 *   vgemm_kv_read        rows of the cache back as int32
 *   vgemm_kv_attention   attention of one new token a sequence over the pages of its block table
 *   vgemm_beam_select    beam search: the best continuations over a group's beams and the vocabulary
 *   vgemm_beam_tables    its reordering: block tables and lengths by parent
 *   vgemm_kv_copy        pages copied (what vgemm_beam_tables lists)
 *
 * Conventions of vgemm_lm.h hold: device pointers of the current device, asynchronous on `stream`, no allocation, legal under stream
 * capture, VGEMM_OK or a negative code with a message in vgemm_last_error(). Every result is a whole number that does not
 * depend on the order of sums or on how the work is split. An output overlaps no input except where it says so. Values are
 * Q16; rshr, sat32 and the exp table are those of the attention (lutexp(d): linear between entries d >> 10 and (d >> 10) + 1 of Lexp,
 * 1025 entries in [0, 2^31); 0 from d = 2^20 on).
 */
#ifndef VGEMM_KV_H
#define VGEMM_KV_H
#include <stddef.h>
#include <stdint.h>

#include "vgemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Pages of `page` tokens (16, 32, 64, 128 or 256) for `heads` heads (1..1024) of D values (a multiple of 16 up to 256); bits 8 or
 * 16; pages * page < 2^31. data: pages * vgemm_kv_page_bytes() bytes, 16-byte aligned; shift: pages * heads * 2 * page bytes, 16-byte aligned. Token t of
 * a page is slot page_number * page + t. A row x of D values is held as q 2^e: e = the least shift >= 0 with max |x| < 2^(bits - 1 + e),
 * q = clamp(rshr(x, e), -(2^(bits - 1) - 1), 2^(bits - 1) - 1); 16 bits as two int8 planes, q = 256 hi + lo + 128.
 * Layout, for each page and head: keys, then values, in groups of 16 tokens; within a group the planes hi, lo one after the other, of
 * 16 D bytes each. Keys: [4 quarters of 4 tokens][D / 16][4 tokens][16 values]; values: [D][16 tokens]. shift: [page][head][keys, values][token]. */
typedef struct VgemmKv {
    int pages, page, heads, D, bits;
    void* data;
    uint8_t* shift;
} VgemmKv;
/* bytes of one page's data over all heads (0: unsupported) */
size_t vgemm_kv_page_bytes(int page, int heads, int D, int bits);

/* R requests of len[r] tokens in the cache and add[r] new ones (below 0: 0; both at most 2^23). Request r has
 * have = ceil(len / page) pages in table [R x ldt] (width <= ldt entries in use) and needs need = min(ceil((len + add) / page), width); its entries
 * [have, need) are written with page numbers taken from free [nfree[0]] in order of request and entry, -1 where the list has ended (or holds no page number).
 * The new tokens, in order of request: token t of `tokens` rows belongs to the request r with start[r] <= t < start[r + 1], start
 * the running sum of add (R + 1 values); pos[t] = len[r] + t - start[r], and slot[t] its slot by the table, -1 where there is no page (entry
 * outside [0, pages), or pos >= width * page). Rows t >= start[R] get pos = slot = -1. new_len[r] = len[r] + add[r]; used[0] = the pages asked for, those past
 * the list included: more than nfree[0] means that some tokens have no slot. new_len, start, pos and used may be NULL; sums saturate at 2^31 - 1.
 * R <= 4096. R == 0: every row gets -1. */
typedef struct VgemmKvPlan {
    int R, tokens, pages, page, width, ldt;
    const int32_t *len, *add;
    int32_t* table;
    const int32_t *free, *nfree;
    int32_t *new_len, *start, *slot, *pos, *used;
} VgemmKvPlan;
int vgemm_kv_plan(void* stream, const VgemmKvPlan* P);

/* Keys K and values V of M tokens, int32 rows of heads * D values ld apart (16-byte aligned, ld % 4 == 0; they may be parts of one
 * merged projection's rows), into slots slot[t]; tokens whose slot lies outside [0, pages * page) are not written. Two tokens of a call have
 * different slots. M == 0 is a no-op; M <= 2^24. */
int vgemm_kv_write(void* stream, const VgemmKv* C, const int32_t* K, const int32_t* V, int ld, const int32_t* slot, int M);
/* The rows q 2^e of slots slot[t], saturated to 32 bits; rows of 0 where the slot lies outside [0, pages * page). K or V may be NULL. */
int vgemm_kv_read(void* stream, const VgemmKv* C, const int32_t* slot, int M, int32_t* K, int32_t* V, int ld);
/* Page dst[i] becomes a copy of page src[i], i < n <= 2^23, data and shifts; pairs with a number outside [0, pages) are left out. No page is the dst of
 * two pairs, or the dst of one and the src of another. */
int vgemm_kv_copy(void* stream, const VgemmKv* C, const int32_t* src, const int32_t* dst, int n);

/* Attention of one new token for each of `rows` sequences. Q [rows x ldq]: Hq heads of D values (Hq a multiple of the cache's
 * heads; query head h reads head h / (Hq / heads)). Sequence r holds n = min(max(len[r], 0), max_len, width * page) tokens (the new one among them,
 * written before), token j in page table[r, j / page]; with window > 0 only the last `window` of them count, and none
 * whose table entry lies outside [0, pages); the slots of those that count have been written by vgemm_kv_write (or copied). For a query head:
 *   q = rshr(x, eq), eq the least shift >= 0 with max |x| < 2^(14 + eq)
 *   s_j = rshr(m sum_d q_d k_jd, s - eq - ek_j)                         1 <= m <= 32768, -64 <= s <= 128
 * Tokens go in spans of 256 positions, [256 u, 256 u + 256). In a span, over the tokens that count:
 *   mx_u = max s_j; P_j = min(32767, rshr(lutexp(mx_u - s_j), 15)); L_u = sum P_j
 *   A_u = sat32(floor((sum P_j v_j 2^ev_j + floor(L_u / 2)) / L_u)), 0 where L_u = 0
 * and over the spans with L_u > 0:
 *   mx = max mx_u; G_u = rshr(lutexp(mx - mx_u), 7) L_u, at least L_u where mx_u = mx; h = the least shift >= 0 with sum G_u < 2^(30 + h); g_u = floor(G_u / 2^h + 1/2)
 *   out = sat32(floor((sum g_u A_u + floor(T / 2)) / T)), T = sum g_u; 0 where no token counts.
 * out [rows x ldo]; rowmax[r] = max(rowmax[r], max |out|) if not NULL. Q and out 16-byte aligned, ldq % 4 == ldo % 4 == 0. rows <= 65535, 0 <= max_len <= 2^23,
 * Hq <= 4096. ws: vgemm_kv_attention_workspace_bytes(), 16-byte aligned, of any content (none up to 256 tokens); calls, or replays of captured ones, that share one must not run at the
 * same time. */
typedef struct VgemmKvAttn {
    const int32_t* Q; int ldq;
    int rows, Hq;
    const int32_t* table; int ldt, width;
    const int32_t* len;
    int max_len, window, m, s;
    const int64_t* Lexp;
    int32_t* out; int ldo;
    uint32_t* rowmax;
    void* ws; size_t ws_bytes;
} VgemmKvAttn;
size_t vgemm_kv_attention_workspace_bytes(int rows, int Hq, int D, int max_len);
int vgemm_kv_attention(void* stream, const VgemmKv* C, const VgemmKvAttn* A);

/* For each of `groups` requests the n best continuations of its `beams` beams. Row r = group * beams + beam of logits [groups * beams
 * x ldz] holds V of them; INT32_MIN bans its token. score[r]: what the beam has so far, |score| < 2^61; INT64_MIN: no such beam. With
 * spans of 4096 tokens: mx_c = max z, S_c = sum lutexp(mx_c - z) over the tokens of a span that are not banned; mx = max mx_c,
 *   S = max(1, sum_c floor((lutexp(mx - mx_c) floor((S_c + 2^11) / 2^12) + 2^17) / 2^18))
 *   t = floor(log2 S), f = floor(S 2^(30 - t)) - 2^30, i = floor(f / 2^20), l = Lln[i] + floor((Lln[i + 1] - Lln[i]) (f mod 2^20) / 2^20)
 *   logZ = rshr((t - 30) Lln[1024] + l, 14)              Lln[i] = ln(1 + i / 1024) in Q30, 1025 entries in [0, 2^30)
 * a continuation's score is score[r] + z - mx - logZ, in 64 bits. out_score, parent (the row) and token [groups x n]: the n
 * largest, in falling order, equal ones by beam and token; INT64_MIN, -1, -1 where there are fewer. 1 <= beams <= 32, 1 <= n <= 64, 1 <= V <= 2^18,
 * groups * beams <= 65535; ws: vgemm_beam_workspace_bytes(), 16-byte aligned, of any content, not shared by calls that run at the same time. */
typedef struct VgemmBeam {
    int groups, beams, V, n;
    const int32_t* logits; int ldz;
    const int64_t* score;
    const int64_t* Lexp; const int64_t* Lln;
    int64_t* out_score; int32_t* parent; int32_t* token;
    void* ws; size_t ws_bytes;
} VgemmBeam;
size_t vgemm_beam_workspace_bytes(int groups, int beams, int V, int n);
int vgemm_beam_select(void* stream, const VgemmBeam* B);

/* Row r continues row parent[r]: n = len[parent[r]] (below 0: 0, at most width * page); out_len[r] = n; out_table[r, j] = table[parent[r], j] for the
 * whole pages j < n / page; a partly filled last page becomes fresh[r], with the pair (src[r], dst[r]) = (its page, fresh[r]) for vgemm_kv_copy, else
 * (-1, -1); one that is no page (an entry below 0, as vgemm_kv_plan writes where its list has ended) becomes -1, without a pair: its tokens do not count
 * afterwards either. Last pages' entries from 0 on are pages of the cache. The entries behind are -1. parent[r] outside [0, rows): n = 0.
 * Tables [rows x ldt], width <= ldt. rows <= 65535, page as in VgemmKv. */
typedef struct VgemmBeamTables {
    int rows, page, width, ldt;
    const int32_t *parent, *len, *table, *fresh;
    int32_t *out_len, *out_table, *src, *dst;
} VgemmBeamTables;
int vgemm_beam_tables(void* stream, const VgemmBeamTables* T);

#ifdef __cplusplus
}
#endif
#endif
