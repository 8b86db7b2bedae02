// A gated MLP's forward or backward as one call: the launches of its products made one after the other from native code, for the host's work through the Python
// wrappers, 10 - 15 us each, is more than a small block's kernels take.  Forward: the gate's products, the down projection.  Backward: the way back through the down projection and the gate,
// the weight gradients, the input gradient over both products.
#include "common.h"
#include "gated_rows.h"
#include "gemm_list.h"
#include "gemm_rows.h"
#include "../../include/ezl.h"

namespace {

int64_t aligned256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t max64(int64_t a, int64_t b) { return a > b ? a : b; }
int64_t block_bytes(const ezl_gated_mlp& m) { return aligned256(m.M * m.f * 2); }

// The weight gradients, down's in front: the order in which they are written where two of them are one tensor's.  All of them, or gate's and up's, go out as one list of tiles where
// that is estimated to be faster; results that do not stay in the caches only on 256 x 256 tiles.  A block forward and backward with the three apart or in pairs, and so: 1024 tokens,
// 256 x 688 47.0 and 40.1 us; 2048, 768 x 2048 123.5 and 108.0; 4000, 1536 x 4096 491 and 462; 8192, 2048 x 5504 1476 and 1407 (from 256 x 256 tiles on: the last round of one
// list is fuller than those of three); where the estimates lie close, 1531 to 4096 tokens at 4096 x 11008, within 1 %.
struct Products {
    int64_t M[3], N[3], three, two;  // bytes of workspace, -1: as fewer
    Products(const ezl_gated_mlp& m, int result_bytes) : M{m.n, m.f, m.f}, N{m.f, m.h, m.h}, three(-1), two(-1) {
        if (m.M == 0) return;
        const int pieces[2] = {1, 2};
        two = ezl_gemm_group_form_workspace_bytes(0, 2, M + 1, N + 1, m.M);
        three = gemm_list_workspace_bytes(2, pieces, M, N, m.M, (m.n + 2 * m.h) * m.f * result_bytes > (384LL << 20));
    }
};

bool wanted(const ezl_layer_grad* g) { return g && (g->f32 || g->bf16); }

int check(const char* name, const ezl_gated_mlp* m) {
    EZL_REQUIRE(m && m->M >= 0 && m->h > 0 && m->f > 0 && m->n > 0, EZL_EINVAL, "%s: bad size", name);
    EZL_REQUIRE(m->gate && m->up && m->down, EZL_EINVAL, "%s: null pointer", name);
    EZL_REQUIRE(m->h % 8 == 0 && m->f % 8 == 0 && m->n % 8 == 0 && m->f < (1LL << 21) && m->h < (1LL << 21) && m->n < (1LL << 21) && m->M < (1LL << 31), EZL_EUNSUPPORTED,
                "%s: widths must be multiples of 8 below 2^21", name);
    return EZL_OK;
}

int weight_gradient(const void* d, int64_t out, const void* in, int64_t ldin, int64_t width, const ezl_layer_grad* g, int64_t tokens, void* ws, int64_t ws_bytes, void* stream) {
    return ezl_gemm_bf16(d, in, g->f32 ? g->f32 : g->bf16, out, width, tokens, out, ldin, width, 0, 0, g->f32 ? 1 : 0, g->f32 && g->accumulate ? 1 : 0, ws, ws_bytes, stream);
}

}  // namespace

extern "C" int64_t ezl_gated_mlp_bytes(const ezl_gated_mlp* m, int backward) {
    if (!m || m->M < 0 || m->h <= 0 || m->f <= 0 || m->n <= 0 || m->M >= (1LL << 31)) return -1;
    if (m->M == 0) return 0;
    if (!backward) return block_bytes(*m) + max64(ezl_gated_workspace_bytes(m->M, m->f, m->h), ezl_gemm_workspace_bytes(m->M, m->n, m->f));
    int64_t ws = max64(ezl_gemm_workspace_bytes(m->M, m->f, m->n), ezl_gemm_workspace_bytes(m->M, m->h, 2 * m->f));
    ws = max64(ws, ezl_gemm_workspace_bytes(m->n, m->f, m->M));
    const Products bf16(*m, 2), f32(*m, 4);
    ws = max64(ws, max64(max64(bf16.two, max64(bf16.three, f32.three)), ezl_gemm_workspace_bytes(m->f, m->h, m->M)));
    return 3 * block_bytes(*m) + ws;
}

extern "C" int ezl_gated_mlp_fwd(const ezl_gated_mlp* m, const void* x, int64_t ldx, void* y, void* kept, void* temp, int64_t temp_bytes, void* stream) {
    const char* name = "ezl_gated_mlp_fwd";
    if (const int rc = check(name, m)) return rc;
    if (m->M == 0) return EZL_OK;
    EZL_REQUIRE(y && temp && ezl_aligned16(temp) && ezl_aligned16(y) && temp_bytes >= ezl_gated_mlp_bytes(m, 0), EZL_EINVAL, "%s: null, misaligned or too small a buffer", name);
    char* const ws = (char*)temp + block_bytes(*m);
    const int64_t ws_bytes = temp_bytes - block_bytes(*m);
    if (const int rc = ezl_gated_fwd(m->act, x, m->gate, m->up, temp, kept, m->M, m->f, m->h, ldx, m->ldw, ws, ws_bytes, stream)) return rc;
    const ezl_epilogue none = {nullptr, nullptr, nullptr, 0, 0, EZL_ACT_NONE};
    if (gemm_rows_pays(m->M, m->n, m->f)) return ezl_gemm_bf16_epilogue(temp, m->down, y, m->M, m->n, m->f, m->f, m->ldd, m->n, &none, ws, ws_bytes, stream);
    if (stream_down_pays(m->M, m->f)) {
        EZL_REQUIRE(ezl_aligned16(m->down) && m->ldd % 8 == 0 && m->ldd >= m->f && m->ldd < (1LL << 22), EZL_EINVAL, "%s: bad down projection", name);
        stream_rows_launch(temp, m->down, nullptr, y, Kept{}, (int)m->M, (int)m->n, (int)m->f, m->f, m->ldd, 0, (hipStream_t)stream);
        EZL_LAUNCH_CHECK(name);
        return EZL_OK;
    }
    return ezl_gemm_bf16(temp, m->down, y, m->M, m->n, m->f, m->f, m->ldd, m->n, 1, 1, 0, 0, ws, ws_bytes, stream);
}

extern "C" int ezl_gated_mlp_bwd(const ezl_gated_mlp* m, const void* x, int64_t ldx, const void* dy, const void* kept, void* dx, const ezl_layer_grad* dgate, const ezl_layer_grad* dup,
                                 const ezl_layer_grad* ddown, void* temp, int64_t temp_bytes, void* stream) {
    const char* name = "ezl_gated_mlp_bwd";
    if (const int rc = check(name, m)) return rc;
    EZL_REQUIRE(m->M == 0 || (x && dy && kept && temp && ezl_aligned16(temp) && temp_bytes >= ezl_gated_mlp_bytes(m, 1)), EZL_EINVAL, "%s: null, misaligned or too small a buffer", name);
    EZL_REQUIRE(m->M == 0 || !dx || ezl_aligned16(dx), EZL_EINVAL, "%s: misaligned dx", name);
    const int64_t block = block_bytes(*m);
    char* const t = (char*)temp;
    void *const dg = t, *const du = t + block, *const mid = t + 2 * block, *const ws = t + 3 * block;
    const int64_t ws_bytes = m->M ? temp_bytes - 3 * block : 0;
    if (m->M)
        if (const int rc = ezl_gated_bwd(m->act, dy, m->down, kept, dg, du, wanted(ddown) ? mid : nullptr, m->M, m->f, m->n, m->n, m->ldd, ws, ws_bytes, stream)) return rc;
    const bool pair = wanted(dgate) && wanted(dup) && !dgate->f32 == !dup->f32;
    const Products products(*m, pair && dgate->f32 ? 4 : 2);
    const bool three = pair && wanted(ddown) && !dgate->f32 == !ddown->f32 && products.three >= 0;
    if (wanted(ddown) && !three)
        if (const int rc = weight_gradient(dy, m->n, mid, m->f, m->f, ddown, m->M, ws, ws_bytes, stream)) return rc;
    if (three || (pair && products.two >= 0)) {
        const ezl_layer_grad* const g[3] = {ddown, dgate, dup};
        const void *a[3] = {dy, dg, du}, *b[3] = {mid, x, x};
        void* c[3] = {};
        const int64_t lda[3] = {m->n, m->f, m->f}, ldb[3] = {m->f, ldx, ldx};
        int accumulate[3] = {};
        const int first = three ? 0 : 1;
        for (int i = first; i < 3; ++i) {
            c[i] = g[i]->f32 ? (void*)g[i]->f32 : (void*)g[i]->bf16;
            accumulate[i] = g[i]->f32 && g[i]->accumulate;
        }
        if (const int rc = gemm_list(3 - first, a + first, b + first, c + first, products.M + first, products.N + first, m->M, lda + first, ldb + first, products.N + first, 0, 0,
                                     dgate->f32 ? 1 : 0, accumulate + first, ws, ws_bytes, stream, three))
            return rc;
    } else {
        if (wanted(dgate))
            if (const int rc = weight_gradient(dg, m->f, x, ldx, m->h, dgate, m->M, ws, ws_bytes, stream)) return rc;
        if (wanted(dup))
            if (const int rc = weight_gradient(du, m->f, x, ldx, m->h, dup, m->M, ws, ws_bytes, stream)) return rc;
    }
    if (!dx || m->M == 0) return EZL_OK;
    const void *a[2] = {dg, du}, *b[2] = {m->gate, m->up};
    const int64_t k[2] = {m->f, m->f};
    return ezl_gemm_bf16_ksplit(2, a, b, dx, m->M, m->h, k, m->f, m->ldw, m->h, 1, 0, 0, 0, ws, ws_bytes, stream);
}
