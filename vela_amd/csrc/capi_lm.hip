// C ABI of the language-model operators (include/vgemm_lm.h): argument checks and dispatch.
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/vgemm_lm.h"
#include "moe.h"
#include "w4.h"

namespace vk {
int set_error(int code, const std::string& msg);
void clear_error();
hipError_t launch_rmsnorm_q(hipStream_t st, const int32_t* X, const int32_t* R, int M, int C, const int32_t* g, i64 den, int32_t* H, int8_t* hi, int8_t* lo,
                            int32_t* e, int Kp);
}  // namespace vk

namespace {

__attribute__((format(printf, 2, 3))) int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return vk::set_error(code, buf);
}

int ok() {
    vk::clear_error();
    return VGEMM_OK;
}

int hip_status(hipError_t e, const char* what) {
    if (e != hipSuccess) return fail(VGEMM_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    return ok();
}

bool aligned(const void* p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

bool w4_shape(int N, int K, int group) { return N >= 1 && N <= (1 << 24) && K >= 1 && K <= 32768 && (group == 32 || group == 64 || group == 128); }

int w4_weights(const char* what, const VgemmW4* W) {
    if (!W || !W->q || !W->cst || !aligned(W->q, 16) || !aligned(W->cst, 16) || W->count < 1)
        return fail(VGEMM_ERR_ARG, "%s: weights need q and cst, 16-byte aligned, and count >= 1", what);
    if (!w4_shape(W->N, W->K, W->group)) return fail(VGEMM_ERR_ARG, "%s: weights need N >= 1, N <= 2^24, 1 <= K <= 32768 and a group of 32, 64 or 128", what);
    return VGEMM_OK;
}

vk::W4View w4_view(const VgemmW4& W) {
    const int KT = vk::w4_kt(W.K), CT = vk::w4_ct(W.N);
    const uint8_t* q = static_cast<const uint8_t*>(W.q);
    return vk::W4View{q, q + size_t(CT) * KT * 1024, reinterpret_cast<const int4*>(W.cst), W.N, W.K, KT, CT};
}

// strides that keep the rows a kernel addresses with 32-bit offsets within 2^30 bytes: 512 int8 rows, 32 int32 rows
constexpr int MAX_LD8 = 1 << 21, MAX_LDX = 1 << 23;
// rows of a call: what a grid holds (65535 tiles of eight rows along its second axis, 2^32 threads)
constexpr int MAX_ROWS = 1 << 18, MAX_NORM_ROWS = 1 << 22;

int rows_limit(const char* what, int M, int most) { return M > most ? fail(VGEMM_ERR_UNSUPPORTED, "%s: at most %d rows a call, not %d", what, most, M) : VGEMM_OK; }

int up16(int v) { return (v + 15) / 16 * 16; }

// int8 rows of K values (lo may be null)
int i8_rows(const char* what, const VgemmASrc* A, int K) {
    if (A->src != VGEMM_SRC_I8) return fail(VGEMM_ERR_ARG, "%s: the rows must be VGEMM_SRC_I8", what);
    if (!A->hi || A->ld8 < up16(K) || A->ld8 % 16 || !aligned(A->hi, 16) || !aligned(A->lo, 16))
        return fail(VGEMM_ERR_ARG, "%s: SRC_I8 planes must be 16-byte aligned with ld8 >= K rounded up to 16, ld8 %% 16 == 0", what);
    if (A->ld8 > MAX_LD8) return fail(VGEMM_ERR_UNSUPPORTED, "%s: ld8 above %d", what, MAX_LD8);
    return VGEMM_OK;
}

}  // namespace

extern "C" {

int vgemm_rmsnorm_q(void* stream, const int32_t* X, const int32_t* R, int M, int C, const int32_t* g, int64_t den, int32_t* H, int8_t* hi, int8_t* lo,
                    int32_t* e, int Kp) {
    if (M == 0) return ok();
    if (!X || M < 0 || !g || !hi || !e || den <= 0) return fail(VGEMM_ERR_ARG, "rmsnorm_q: bad arguments");
    if (C <= 0 || C % 4 || C > 8192) return fail(VGEMM_ERR_ARG, "rmsnorm_q: C must be a multiple of 4 and at most 8192");
    if (!aligned(X, 16) || !aligned(R, 16) || !aligned(H, 16) || !aligned(g, 16)) return fail(VGEMM_ERR_ARG, "rmsnorm_q: X, R, H and g must be 16-byte aligned");
    if (int rc = rows_limit("rmsnorm_q", M, MAX_NORM_ROWS)) return rc;
    if (Kp < C || Kp % 4 || !aligned(hi, 4) || !aligned(lo, 4)) return fail(VGEMM_ERR_ARG, "rmsnorm_q: Kp >= C, Kp %% 4 == 0 and 4-byte aligned rows required");
    return hip_status(vk::launch_rmsnorm_q(static_cast<hipStream_t>(stream), X, R, M, C, g, den, H, hi, lo, e, Kp), "rmsnorm_q launch");
}

size_t vgemm_w4_bytes(int N, int K, int group) { return w4_shape(N, K, group) ? vk::w4_bytes(N, K, group) : 0; }

int vgemm_w4_pack(void* stream, const VgemmW4* W, int first, int n, const uint8_t* nib, int ldn, const uint16_t* scale, const uint8_t* zero, int lds,
                  const int32_t* msb) {
    if (int rc = w4_weights("w4_pack", W)) return rc;
    if (first < 0 || n < 0 || first > W->count - n) return fail(VGEMM_ERR_ARG, "w4_pack: matrices [%d, %d + %d) of %d", first, first, n, W->count);
    if (n == 0) return ok();
    if (n > 65535) return fail(VGEMM_ERR_UNSUPPORTED, "w4_pack: at most 65535 matrices a call");
    if (!nib || !scale || !msb || ldn < (W->K + 1) / 2 || lds < (W->K + W->group - 1) / W->group || !aligned(scale, 2) || !aligned(msb, 4))
        return fail(VGEMM_ERR_ARG, "w4_pack: nib with ldn >= K / 2, scale with lds >= the row's groups, and msb required");
    uint8_t* q = static_cast<uint8_t*>(W->q) + size_t(first) * vk::w4_bytes(W->N, W->K, W->group);
    int4* cst = reinterpret_cast<int4*>(W->cst) + size_t(first) * up16(W->N);
    return hip_status(vk::launch_w4_pack(static_cast<hipStream_t>(stream), W->N, W->K, W->group, q, cst, n, nib, ldn, scale, zero, lds, msb), "w4_pack launch");
}

int vgemm_w4(void* stream, const VgemmASrc* A, int M, const VgemmW4* W, const VgemmAEpi* E) {
    if (!A || !E || M < 0) return fail(VGEMM_ERR_ARG, "w4: bad arguments");
    if (int rc = w4_weights("w4", W)) return rc;
    if (W->count != 1) return fail(VGEMM_ERR_ARG, "w4: one matrix expected, not %d", W->count);
    if (E->epi == VGEMM_EPI_PLAIN && E->gnstat) return fail(VGEMM_ERR_ARG, "w4: no GroupNorm statistics (gnstat must be NULL)");
    if (M == 0) return ok();
    if (int rc = rows_limit("w4", M, MAX_ROWS)) return rc;
    vk::W4Args a{};
    a.w = w4_view(*W);
    a.group = W->group;
    a.M = M;
    a.Kp16 = up16(W->K);
    if (A->src == VGEMM_SRC_X32) {
        if (!A->x || !A->rowmax || A->K != W->K || A->K % 4 || A->ldx < A->K || A->ldx % 4 || !aligned(A->x, 16))
            return fail(VGEMM_ERR_ARG, "w4: SRC_X32 needs x, rowmax, K == the weights' K, K %% 4 == 0, ldx >= K, ldx %% 4 == 0, 16-byte alignment");
        if (A->ldx > MAX_LDX) return fail(VGEMM_ERR_UNSUPPORTED, "w4: ldx above %d", MAX_LDX);
        a.x = A->x; a.ldx = A->ldx; a.xmax = A->rowmax;
    } else {
        if (int rc = i8_rows("w4", A, W->K)) return rc;
        a.hi = A->hi; a.lo = A->lo; a.ld8 = A->ld8; a.e = A->e;
    }
    if (!E->Y) return fail(VGEMM_ERR_ARG, "w4: null Y");
    if (E->epi == VGEMM_EPI_GEGLU) {
        if (W->N % 2 || !E->Lphi || E->ldy < W->N / 2) return fail(VGEMM_ERR_ARG, "w4: EPI_GEGLU needs an even N, Lphi and ldy >= N / 2");
    } else if (E->epi == VGEMM_EPI_PLAIN) {
        if (E->ldy < W->N) return fail(VGEMM_ERR_ARG, "w4: ldy < N");
        a.R = E->residual;
    } else {
        return fail(VGEMM_ERR_ARG, "w4: EPI_PLAIN or EPI_GEGLU expected");
    }
    a.geglu = E->epi == VGEMM_EPI_GEGLU;
    a.Y = E->Y; a.ldy = E->ldy; a.Lphi = E->Lphi; a.rowmax = E->rowmax;
    return hip_status(vk::launch_w4(static_cast<hipStream_t>(stream), a), "w4 launch");
}

int vgemm_moe_route(void* stream, const VgemmASrc* A, int M, const VgemmMoeRoute* R) {
    if (!A || !R || M < 0) return fail(VGEMM_ERR_ARG, "moe_route: bad arguments");
    if (R->experts < 1 || R->experts > vk::MOE_EXPERTS || R->topk < 1 || R->topk > vk::MOE_TOPK || R->topk > R->experts)
        return fail(VGEMM_ERR_ARG, "moe_route: 1 <= topk <= experts, experts <= %d and topk <= %d required", vk::MOE_EXPERTS, vk::MOE_TOPK);
    if (M == 0) return ok();
    if (int rc = rows_limit("moe_route", M, MAX_ROWS)) return rc;
    if (!R->W || !R->cst || !R->Lexp || !R->idx || !R->p || !aligned(R->W, 16) || !aligned(R->cst, 16)) return fail(VGEMM_ERR_ARG, "moe_route: W, cst (16-byte aligned), Lexp, idx and p required");
    if (A->K < 16 || A->K % 16 || A->K > 16384 || R->ldw < A->K || R->ldw % 16) return fail(VGEMM_ERR_ARG, "moe_route: K %% 16 == 0, K <= 16384, ldw >= K, ldw %% 16 == 0 required");
    if (int rc = i8_rows("moe_route", A, A->K)) return rc;
    const vk::RouteArgs a{A->hi, A->lo, A->ld8, A->e, A->K, R->W, R->ldw, reinterpret_cast<const int4*>(R->cst), R->experts, R->topk, R->renorm,
                          reinterpret_cast<const long long*>(R->Lexp), R->idx, R->p, R->logits};
    return hip_status(vk::launch_moe_route(static_cast<hipStream_t>(stream), a, M), "moe_route launch");
}

// tokens one pass takes; a pass's workspace holds for each pair the row of the down product, v and the maxima of v's segments
static int moe_pass(int M, int topk) { return std::min(M, vk::MOE_PAIRS / topk); }

size_t vgemm_moe_workspace_bytes(int M, int topk, int F) {
    if (M <= 0 || topk < 1 || topk > vk::MOE_TOPK || F < 1 || F > 32768 || F % 4) return 0;
    return size_t(moe_pass(M, topk)) * topk * (size_t(F) + vk::MOE_COLS + vk::w4_ct(2 * F)) * 4;
}

int vgemm_moe(void* stream, const VgemmASrc* A, int M, const VgemmMoe* P) {
    if (!A || !P || M < 0) return fail(VGEMM_ERR_ARG, "moe: bad arguments");
    if (int rc = w4_weights("moe", &P->up)) return rc;
    if (int rc = w4_weights("moe", &P->down)) return rc;
    const int F = P->down.K, D = P->down.N;
    if (P->up.N != 2 * F || P->up.count != P->down.count || P->up.count > vk::MOE_EXPERTS || F % 4)
        return fail(VGEMM_ERR_ARG, "moe: up.N == 2 down.K, down.K %% 4 == 0 and equal counts of at most %d required", vk::MOE_EXPERTS);
    if (P->topk < 1 || P->topk > vk::MOE_TOPK) return fail(VGEMM_ERR_ARG, "moe: 1 <= topk <= %d required", vk::MOE_TOPK);
    if (M == 0) return ok();
    if (!P->idx || !P->p || !P->Lphi || !P->Y || P->ldy < D) return fail(VGEMM_ERR_ARG, "moe: idx, p, Lphi and Y with ldy >= down.N required");
    if (int rc = i8_rows("moe", A, P->up.K)) return rc;
    if (!P->ws || !aligned(P->ws, 16) || P->ws_bytes < vgemm_moe_workspace_bytes(M, P->topk, F)) return fail(VGEMM_ERR_ARG, "moe: workspace of vgemm_moe_workspace_bytes() required, 16-byte aligned");
    const int pass = moe_pass(M, P->topk);
    vk::MoeArgs a{};
    a.up = w4_view(P->up);
    a.down = w4_view(P->down);
    a.up_stride = vk::w4_bytes(P->up.N, P->up.K, P->up.group);
    a.down_stride = vk::w4_bytes(D, F, P->down.group);
    a.experts = P->up.count;
    a.group_up = P->up.group;
    a.group_down = P->down.group;
    a.ld8 = A->ld8;
    a.topk = P->topk;
    a.Kp16 = up16(P->up.K);
    a.Lphi = P->Lphi;
    a.ldy = P->ldy;
    a.y = static_cast<int32_t*>(P->ws);
    a.v = a.y + size_t(pass) * P->topk * vk::MOE_COLS;
    a.vmax = reinterpret_cast<uint32_t*>(a.v + size_t(pass) * P->topk * F);
    for (int t = 0; t < M; t += pass) {
        a.M = std::min(pass, M - t);
        a.hi = A->hi + size_t(t) * A->ld8;
        a.lo = A->lo ? A->lo + size_t(t) * A->ld8 : nullptr;
        a.e = A->e ? A->e + t : nullptr;
        a.idx = P->idx + size_t(t) * P->topk;
        a.p = P->p + size_t(t) * P->topk;
        a.Y = P->Y + size_t(t) * P->ldy;
        a.R = P->residual ? P->residual + size_t(t) * P->ldy : nullptr;
        if (int rc = hip_status(vk::launch_moe(static_cast<hipStream_t>(stream), a), "moe launch")) return rc;
    }
    return ok();
}

}  // extern "C"
