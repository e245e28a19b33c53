// C ABI of the paged key-value cache (include/vgemm_kv.h): argument checks and dispatch.
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "kv.h"

namespace vk {
int set_error(int code, const std::string& msg);
void clear_error();
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

int page_log2(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : page == 256 ? 8 : -1; }

bool kv_shape(int page, int heads, int D, int bits) {
    return page_log2(page) >= 0 && heads >= 1 && heads <= 1024 && D >= 16 && D <= 256 && D % 16 == 0 && (bits == 8 || bits == 16);
}

int kv_cache(const char* what, const VgemmKv* C) {
    if (!C || !C->data || !C->shift || !aligned(C->data, 16) || !aligned(C->shift, 16)) return fail(VGEMM_ERR_ARG, "%s: a cache needs data and shift, 16-byte aligned", what);
    if (!kv_shape(C->page, C->heads, C->D, C->bits))
        return fail(VGEMM_ERR_ARG, "%s: a cache needs a page of 16, 32, 64, 128 or 256 tokens, 1 to 1024 heads, D %% 16 == 0, 16 <= D <= 256 and 8 or 16 bits", what);
    if (C->pages < 1 || (int64_t(C->pages) << page_log2(C->page)) > 0x7fffffffLL) return fail(VGEMM_ERR_ARG, "%s: a cache needs pages >= 1 and pages * page < 2^31", what);
    return VGEMM_OK;
}

vk::KvView kv_view(const VgemmKv& C) { return vk::KvView{static_cast<int8_t*>(C.data), C.shift, C.pages, page_log2(C.page), C.heads, C.D, C.bits / 8}; }

int kv_rows(const char* what, const VgemmKv* C, const void* K, const void* V, int ld, int M) {
    if (!aligned(K, 16) || !aligned(V, 16) || ld < C->heads * C->D || ld % 4) return fail(VGEMM_ERR_ARG, "%s: K and V must be 16-byte aligned with ld >= heads * D, ld %% 4 == 0", what);
    if (M > (1 << 24)) return fail(VGEMM_ERR_UNSUPPORTED, "%s: at most %d tokens a call, not %d", what, 1 << 24, M);
    return VGEMM_OK;
}

int attn_spans(int max_len) { return (max_len + vk::KV_SPAN - 1) / vk::KV_SPAN; }
int beam_spans(int V) { return (V + vk::BEAM_SPAN - 1) / vk::BEAM_SPAN; }

}  // namespace

extern "C" {

size_t vgemm_kv_page_bytes(int page, int heads, int D, int bits) { return kv_shape(page, heads, D, bits) ? size_t(heads) * 2 * page * D * (bits / 8) : 0; }

int vgemm_kv_plan(void* stream, const VgemmKvPlan* P) {
    if (!P || P->R < 0 || P->tokens < 0) return fail(VGEMM_ERR_ARG, "kv_plan: bad arguments");
    const int lp = page_log2(P->page);
    if (lp < 0 || P->pages < 1 || (int64_t(P->pages) << lp) > 0x7fffffffLL) return fail(VGEMM_ERR_ARG, "kv_plan: a page of 16, 32, 64, 128 or 256 tokens, pages >= 1 and pages * page < 2^31 required");
    if (P->R > vk::KV_PLAN_ROWS) return fail(VGEMM_ERR_UNSUPPORTED, "kv_plan: at most %d requests, not %d", vk::KV_PLAN_ROWS, P->R);
    if (P->width < 0 || P->ldt < P->width) return fail(VGEMM_ERR_ARG, "kv_plan: 0 <= width <= ldt required");
    if (P->R && (!P->len || !P->add || !P->nfree || (P->width && (!P->table || !P->free)))) return fail(VGEMM_ERR_ARG, "kv_plan: len, add, table, free and nfree required");
    if (P->tokens && !P->slot) return fail(VGEMM_ERR_ARG, "kv_plan: slot required");
    return hip_status(vk::launch_kv_plan(static_cast<hipStream_t>(stream), *P, lp), "kv_plan launch");
}

int vgemm_kv_write(void* stream, const VgemmKv* C, const int32_t* K, const int32_t* V, int ld, const int32_t* slot, int M) {
    if (int rc = kv_cache("kv_write", C)) return rc;
    if (M < 0) return fail(VGEMM_ERR_ARG, "kv_write: bad arguments");
    if (M == 0) return ok();
    if (!K || !V || !slot) return fail(VGEMM_ERR_ARG, "kv_write: K, V and slot required");
    if (int rc = kv_rows("kv_write", C, K, V, ld, M)) return rc;
    return hip_status(vk::launch_kv_write(static_cast<hipStream_t>(stream), kv_view(*C), K, V, ld, slot, M), "kv_write launch");
}

int vgemm_kv_read(void* stream, const VgemmKv* C, const int32_t* slot, int M, int32_t* K, int32_t* V, int ld) {
    if (int rc = kv_cache("kv_read", C)) return rc;
    if (M < 0) return fail(VGEMM_ERR_ARG, "kv_read: bad arguments");
    if (M == 0 || (!K && !V)) return ok();
    if (!slot) return fail(VGEMM_ERR_ARG, "kv_read: slot required");
    if (int rc = kv_rows("kv_read", C, K, V, ld, M)) return rc;
    return hip_status(vk::launch_kv_read(static_cast<hipStream_t>(stream), kv_view(*C), slot, M, K, V, ld), "kv_read launch");
}

int vgemm_kv_copy(void* stream, const VgemmKv* C, const int32_t* src, const int32_t* dst, int n) {
    if (int rc = kv_cache("kv_copy", C)) return rc;
    if (n < 0) return fail(VGEMM_ERR_ARG, "kv_copy: bad arguments");
    if (n == 0) return ok();
    if (!src || !dst) return fail(VGEMM_ERR_ARG, "kv_copy: src and dst required");
    if (n > (1 << 23)) return fail(VGEMM_ERR_UNSUPPORTED, "kv_copy: at most %d pages a call, not %d", 1 << 23, n);   // what a grid holds
    return hip_status(vk::launch_kv_copy(static_cast<hipStream_t>(stream), kv_view(*C), src, dst, n), "kv_copy launch");
}

// per row, query head and span: two words of statistics, and the means
size_t vgemm_kv_attention_workspace_bytes(int rows, int Hq, int D, int max_len) {
    if (rows < 1 || rows > 65535 || Hq < 1 || Hq > 4096 || D < 16 || D > 256 || D % 16 || max_len <= vk::KV_SPAN || max_len > vk::KV_MAX_LEN) return 0;
    return (size_t(rows) * Hq * attn_spans(max_len) * 8 + 15) / 16 * 16 + size_t(rows) * Hq * attn_spans(max_len) * D * 4;
}

int vgemm_kv_attention(void* stream, const VgemmKv* C, const VgemmKvAttn* A) {
    if (int rc = kv_cache("kv_attention", C)) return rc;
    if (!A || A->rows < 0) return fail(VGEMM_ERR_ARG, "kv_attention: bad arguments");
    if (A->Hq < 1 || A->Hq % C->heads || A->Hq > 4096) return fail(VGEMM_ERR_ARG, "kv_attention: Hq must be a multiple of the cache's heads and at most 4096");
    if (A->m < 1 || A->m > 32768 || A->s < -64 || A->s > 128) return fail(VGEMM_ERR_ARG, "kv_attention: 1 <= m <= 32768 and -64 <= s <= 128 required");
    if (A->max_len < 0 || A->window < 0 || A->width < 0 || A->ldt < A->width) return fail(VGEMM_ERR_ARG, "kv_attention: max_len >= 0, window >= 0 and 0 <= width <= ldt required");
    if (A->rows > 65535) return fail(VGEMM_ERR_UNSUPPORTED, "kv_attention: at most 65535 rows a call, not %d", A->rows);
    if (A->max_len > vk::KV_MAX_LEN) return fail(VGEMM_ERR_UNSUPPORTED, "kv_attention: at most %d tokens a sequence, not %d", vk::KV_MAX_LEN, A->max_len);
    if (A->rows == 0) return ok();
    if (!A->Q || !A->len || (A->width && !A->table) || !A->Lexp || !A->out) return fail(VGEMM_ERR_ARG, "kv_attention: Q, len, table, Lexp and out required");
    if (!aligned(A->Q, 16) || !aligned(A->out, 16) || A->ldq < A->Hq * C->D || A->ldo < A->Hq * C->D || A->ldq % 4 || A->ldo % 4)
        return fail(VGEMM_ERR_ARG, "kv_attention: Q and out must be 16-byte aligned with ldq, ldo >= Hq * D and multiples of 4");
    const size_t nb = vgemm_kv_attention_workspace_bytes(A->rows, A->Hq, C->D, A->max_len);
    if (nb && (!A->ws || !aligned(A->ws, 16) || A->ws_bytes < nb)) return fail(VGEMM_ERR_ARG, "kv_attention: workspace of vgemm_kv_attention_workspace_bytes() required, 16-byte aligned");
    vk::KvAttnArgs a{};
    a.c = kv_view(*C);
    a.Q = A->Q; a.ldq = A->ldq; a.rows = A->rows; a.Hq = A->Hq;
    a.group = A->Hq / C->heads;
    a.qtiles = (a.group + 15) / 16;
    a.table = A->table; a.ldt = A->ldt; a.width = A->width;
    a.len = A->len; a.max_len = A->max_len; a.window = A->window;
    a.m = A->m; a.s = A->s;
    a.Lexp = reinterpret_cast<const long long*>(A->Lexp);
    a.out = A->out; a.ldo = A->ldo; a.rowmax = A->rowmax;
    a.spans = std::max(1, attn_spans(A->max_len));
    a.stat = static_cast<int2*>(A->ws);
    a.part = reinterpret_cast<int32_t*>(static_cast<char*>(A->ws) + (size_t(A->rows) * A->Hq * a.spans * 8 + 15) / 16 * 16);
    return hip_status(vk::launch_kv_attention(static_cast<hipStream_t>(stream), a), "kv_attention launch");
}

static bool beam_shape(int groups, int beams, int V, int n) {
    return groups >= 1 && beams >= 1 && beams <= vk::BEAM_MOST && groups <= 65535 / beams && V >= 1 && V <= vk::BEAM_V && n >= 1 && n <= vk::BEAM_N;
}

// per row and span: its statistics and n candidates
size_t vgemm_beam_workspace_bytes(int groups, int beams, int V, int n) {
    return beam_shape(groups, beams, V, n) ? size_t(groups) * beams * beam_spans(V) * (sizeof(vk::BeamStat) + size_t(n) * 8) : 0;
}

int vgemm_beam_select(void* stream, const VgemmBeam* B) {
    if (!B || B->groups < 0) return fail(VGEMM_ERR_ARG, "beam_select: bad arguments");
    if (B->groups == 0) return ok();
    if (!beam_shape(B->groups, B->beams, B->V, B->n))
        return fail(VGEMM_ERR_ARG, "beam_select: 1 <= beams <= %d, groups * beams <= 65535, 1 <= V <= %d and 1 <= n <= %d required", vk::BEAM_MOST, vk::BEAM_V, vk::BEAM_N);
    if (!B->logits || B->ldz < B->V || !B->score || !B->Lexp || !B->Lln || !B->out_score || !B->parent || !B->token)
        return fail(VGEMM_ERR_ARG, "beam_select: logits with ldz >= V, score, Lexp, Lln, out_score, parent and token required");
    const size_t nb = vgemm_beam_workspace_bytes(B->groups, B->beams, B->V, B->n);
    if (!B->ws || !aligned(B->ws, 16) || B->ws_bytes < nb) return fail(VGEMM_ERR_ARG, "beam_select: workspace of vgemm_beam_workspace_bytes() required, 16-byte aligned");
    vk::BeamArgs a{};
    a.b = *B;
    a.spans = beam_spans(B->V);
    a.stat = static_cast<vk::BeamStat*>(B->ws);
    a.cand = reinterpret_cast<int2*>(a.stat + size_t(B->groups) * B->beams * a.spans);
    return hip_status(vk::launch_beam_select(static_cast<hipStream_t>(stream), a), "beam_select launch");
}

int vgemm_beam_tables(void* stream, const VgemmBeamTables* T) {
    if (!T || T->rows < 0) return fail(VGEMM_ERR_ARG, "beam_tables: bad arguments");
    const int lp = page_log2(T->page);
    if (lp < 0 || T->width < 0 || T->ldt < T->width) return fail(VGEMM_ERR_ARG, "beam_tables: a page of 16, 32, 64, 128 or 256 tokens and 0 <= width <= ldt required");
    if (T->rows > 65535) return fail(VGEMM_ERR_UNSUPPORTED, "beam_tables: at most 65535 rows, not %d", T->rows);
    if (T->rows == 0) return ok();
    if (!T->parent || !T->len || !T->fresh || !T->out_len || !T->src || !T->dst || (T->width && (!T->table || !T->out_table)))
        return fail(VGEMM_ERR_ARG, "beam_tables: parent, len, table, fresh, out_len, out_table, src and dst required");
    return hip_status(vk::launch_beam_tables(static_cast<hipStream_t>(stream), *T, lp), "beam_tables launch");
}

}  // extern "C"
