/*
 * vgemm_lm -- operators of a language model's decode step in the library's exact integer arithmetic: part of
 * libvgemm.so, beside the W8A16 products, norms and GEGLU blocks of vgemm.h. No counterparts in the reference. Of such a
 * step these are the norms, the projections and the feed-forward layers, dense or of experts; rotary positions, attention over a
 * cache and sampling are not there, and no engine block or container of vgemm_engine.h / vgemm_model.h uses them.
 *
 *   vgemm_rmsnorm_q     residual addition, root-mean-square norm, 8-bit rows (or the int16 view)
 *   vgemm_w4_pack       4-bit weights with group scales and zero points, laid out for the products
 *   vgemm_w4            products of few rows with such weights: PLAIN or GEGLU epilogue
 *   vgemm_moe_route     the router of a mixture-of-experts layer: logits, the chosen experts, their shares
 *   vgemm_moe           the chosen experts' feed-forward on 4-bit weights and their combination
 *
 * Conventions of vgemm.h hold: device pointers of the current device, asynchronous on `stream`, no allocation, legal under
 * stream capture, VGEMM_OK or a negative code with a message in vgemm_last_error(). Every result is a whole
 * number that does not depend on the order of sums. An output overlaps no input except where it says so. A row is
 *   8-bit:  q = hi          (VgemmASrc.src = VGEMM_SRC_I8 with lo == NULL)
 *   16-bit: q = 256 hi + lo + 128                (VGEMM_SRC_I8 with both planes)
 * and stands for q 2^e with a shift e per row (e == NULL: 0).
 */
#ifndef VGEMM_LM_H
#define VGEMM_LM_H
#include <stddef.h>
#include <stdint.h>

#include "vgemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* h = sat32(X + R) (R may be NULL: h = X); ex = max(0, row_exp(max |h|) - 5); var = floor(sum rshr(h, ex)^2 / C);
 * sd = isqrt((var + eps) << 16), eps = floor((2^(32 - 2 ex) + den / 2) / den);
 * y = sat32(rshr(floor((h 2^(25 - ex) + sd) / 2 sd) g, 16)). With lo == NULL: 8-bit rows hi [M x Kp], e = the
 * least shift >= 0 with max |y| < 2^(7 + e), q = clamp(rshr(y, e), -127, 127); else the int16 view of vgemm_lnorm_q. Columns
 * [C, Kp) hold the value 0. H (may be NULL, X or R) receives h. X, R, H [M x C] and g [C] 16-byte aligned,
 * C % 4 == 0, C <= 8192, Kp >= C, Kp % 4 == 0, hi / lo 4-byte aligned, M <= 2^22. M == 0 is a no-op. */
int vgemm_rmsnorm_q(void* stream, const int32_t* X, const int32_t* R, int M, int C, const int32_t* g, int64_t den, int32_t* H, int8_t* hi, int8_t* lo,
                    int32_t* e, int Kp);

/* `count` matrices of N x K 4-bit weights, w[n, k] = (u[n, k] - z[n, k / group]) sc[n, k / group] with u, z in 0..15 and
 * sc in 0..4095; group 32, 64 or 128 (the last group of a row may be short), 1 <= N <= 2^24, 1 <= K <= 32768. q holds count *
 * vgemm_w4_bytes(N, K, group) bytes, cst [count x N16 x 4] int32 {m, s, b, wsum} with N16 = N rounded up to 16; both
 * 16-byte aligned, written by vgemm_w4_pack. */
typedef struct VgemmW4 {
    int N, K, group, count;
    void* q;
    int32_t* cst;
} VgemmW4;
/* bytes of one matrix (0: unsupported N, K or group) */
size_t vgemm_w4_bytes(int N, int K, int group);
/* Lay out matrices [first, first + n) of W from rows: nib [n x N x ldn] bytes (column 2 i in the low half of byte i, 2 i + 1
 * in the high half), scale [n x N x lds] (values above 4095 are taken as 4095) and zero [n x N x lds] bytes (their low four
 * bits; NULL: 8 throughout), lds >= the groups of a row, msb [n x N x 4] int32 {m, s, b, unused}. A load-time operation. */
int vgemm_w4_pack(void* stream, const VgemmW4* W, int first, int n, const uint8_t* nib, int ldn, const uint16_t* scale, const uint8_t* zero, int lds,
                  const int32_t* msb);

/* Y = A W^T for M rows (W->count == 1): acc = sum_k q[r, k] w[n, k], y = sat32(rshr(acc m, s - e) + b) (acc m wraps in 64 bits),
 * then as vgemm_hl2's epilogues
 *   VGEMM_EPI_PLAIN  + residual (stride ldy, may be Y), saturated; gnstat must be NULL
 *   VGEMM_EPI_GEGLU  columns (a, g) interleaved, N even: sat32(rshr(a sat32(rshr(g lut16i(g, Lphi), 16)), 16)); with a sigmoid
 *                    table it is a * SiLU(g)
 * and rowmax[r] = max(rowmax[r], |y|) when E->rowmax != NULL. A: VGEMM_SRC_I8 (lo may be NULL; ld8 >= K rounded up to 16, ld8 % 16
 * == 0, 16-byte aligned planes; columns past K are not used) or VGEMM_SRC_X32 (K == W->K, K % 4 == 0; row maxima in
 * rowmax). Made for rows up to a few tens: the weights are read once for every 8, 16 or 32 of them.
 * M <= 2^18, ld8 <= 2^21, ldx <= 2^23 (else VGEMM_ERR_UNSUPPORTED). M == 0 is a no-op. */
int vgemm_w4(void* stream, const VgemmASrc* A, int M, const VgemmW4* W, const VgemmAEpi* E);

/* Router of M tokens (rows of A, VGEMM_SRC_I8): logits z[x] = sat32(rshr(acc m, s - e) + b) of the int8 weights W [experts x ldw]
 * (K = A->K columns, ldw >= K, ldw % 16 == 0) and cst {m, s, b, wsum}; idx [M x topk] = the topk largest, in falling order, equal
 * ones by their index; p [M x topk] their shares in Q15: E_x = lutexp(max z - z[x]) by the attention's exp table Lexp (1025 entries in [0, 2^31)),
 * r = floor(2^62 / sum E) over the chosen (renorm != 0) or all experts, p = min(32767, (E r + 2^46) >> 47). logits [M x experts]
 * may be NULL; given, it lets the logits of a layer above 256 KiB of weights be computed by many CUs (p = 0 where sum E = 0). experts <= 512, topk <= 16, topk <= experts, K % 16 == 0, K <= 16384, M <= 2^18. */
typedef struct VgemmMoeRoute {
    const int8_t* W; int ldw; const int32_t* cst;
    int experts, topk, renorm;
    const int64_t* Lexp;
    int32_t* idx; int32_t* p; int32_t* logits;
} VgemmMoeRoute;
int vgemm_moe_route(void* stream, const VgemmASrc* A, int M, const VgemmMoeRoute* R);

/* The experts' part of the layer for M tokens: per token t and choice j with x = idx[t, j] in [0, up.count) (others
 * contribute nothing), v = GEGLU row of up[x] (N = 2F) on row t of A, y = PLAIN row of down[x] (K = F) on the int16 quantisation of v
 * by its own maximum, Y[t] = sat32(sat32(rshr(sum_j p[t, j] y, 15)) + residual[t]). residual (stride ldy) may be NULL or Y. A:
 * VGEMM_SRC_I8 as for vgemm_w4. p: any int32 (the sum wraps in 64 bits); an expert may be chosen more than once. ws:
 * vgemm_moe_workspace_bytes(M, topk, F) bytes, 16-byte aligned, of any content; calls, or replays of captured ones, that share one must not
 * run at the same time. F % 4 == 0, topk <= 16, up.count == down.count <= 512. */
typedef struct VgemmMoe {
    VgemmW4 up, down;
    int topk;
    const int32_t* idx; const int32_t* p;
    const int32_t* Lphi;
    int32_t* Y; int ldy; const int32_t* residual;
    void* ws; size_t ws_bytes;
} VgemmMoe;
/* 0: no tokens, or a topk or F that a layer does not take */
size_t vgemm_moe_workspace_bytes(int M, int topk, int F);
int vgemm_moe(void* stream, const VgemmASrc* A, int M, const VgemmMoe* P);

#ifdef __cplusplus
}
#endif
#endif
