// A linear map and its gradients in 8-bit block-scaled form, each as one call over clt_pack8 and clt_gemm8.  Why: with few tokens a training
// step costs what the host needs between launches.  Inside a step of 16 tokens and 2 layers of 110 -> 32: forward 41 us and
// backward 51 us with a call from Python for every launch, 32 and 37 us so (the step, autograd's own 60 us included: 170 and 142).
//
// Bytes kept between the two: x transposed (codes [L][K][up(T)], scale bytes [L][up(T) / 128][up(K)]), then W for the input gradient (codes
// [L][K][up(N)], scale bytes [L][up(N) / 128][up(K)]), either part only where it is kept.  All parts are multiples of 128 bytes.
#include "block8_common.h"

namespace {
long codes(long L, long rows, long cols) { return L * rows * up128(cols); }
long held(long L, long rows, long cols) { return codes(L, rows, cols) + L * (up128(cols) / B8) * up128(rows); }

// densely held e4m3 operands [L][rows][K]
struct Operand { const uint8_t *q, *s; int rows; };
int product(Operand a, Operand b, int L, int K, void* c, int dtype, long ldc, long cb, const float* bias, long bias_batch, void* ws, size_t bytes, void* stream) {
    const long k = up128(K), sa = up128(a.rows), sb = up128(b.rows);
    return clt_gemm8(a.q, a.s, CLT_F8_E4M3, k, sa, a.rows * k, k / B8 * sa, b.q, b.s, CLT_F8_E4M3, k, sb, b.rows * k, k / B8 * sb, c, dtype, ldc, cb, bias, bias_batch,
                     a.rows, b.rows, K, L, 0, bytes ? ws : nullptr, bytes, stream);
}
uint8_t* take(uint8_t*& at, long n) { uint8_t* p = at; at += n; return p; }
bool bad(int T, int L, int K, int N) { return T < 0 || L <= 0 || K <= 0 || N <= 0; }
}  // namespace

extern "C" size_t clt_linear8_kept_bytes(int T, int L, int K, int N, int keep_x, int keep_w) {
    return bad(T, L, K, N) ? 0 : (size_t)((keep_x ? held(L, K, T) : 0) + (keep_w ? held(L, K, N) : 0));
}

extern "C" size_t clt_linear8_forward_workspace_bytes(int T, int L, int K, int N) {
    return bad(T, L, K, N) ? 0 : (size_t)(held(L, T, K) + held(L, N, K)) + clt_gemm8_workspace_bytes(T, N, K, L);
}

extern "C" int clt_linear8_forward(const void* x, int x_dtype, long x_token_stride, long x_layer_stride, const void* w, int w_dtype,
                                   long w_row_stride, long w_batch_stride, int kn, const float* bias, void* y, int T, int L, int K, int N,
                                   int keep_x, int keep_w, void* kept, void* workspace, size_t workspace_bytes, void* stream) {
    if (bad(T, L, K, N)) return CLT_ERR_SHAPE;
    if (!T && !keep_w) return CLT_OK;
    if (!workspace || !aligned16(workspace) || workspace_bytes < clt_linear8_forward_workspace_bytes(T, L, K, N)) return CLT_ERR_WORKSPACE;
    if ((keep_x || keep_w) && (!kept || !aligned16(kept))) return CLT_ERR_WORKSPACE;
    uint8_t *at = static_cast<uint8_t*>(workspace), *kp = static_cast<uint8_t*>(kept);
    uint8_t *q = take(at, codes(L, T, K)), *s = take(at, held(L, T, K) - codes(L, T, K));
    uint8_t *f = take(at, codes(L, N, K)), *fs = take(at, held(L, N, K) - codes(L, N, K));
    uint8_t *xt = nullptr, *xs = nullptr, *wk = nullptr, *wks = nullptr;
    if (keep_x) { xt = take(kp, codes(L, K, T)); xs = take(kp, held(L, K, T) - codes(L, K, T)); }
    if (keep_w) { wk = take(kp, codes(L, K, N)); wks = take(kp, held(L, K, N) - codes(L, K, N)); }
    // the contraction over K reads the [N, K] form of W, the input gradient its [K, N] form
    const int rows = kn ? K : N, cols = kn ? N : K;
    int rc = clt_pack8(w, w_dtype, w_row_stride, w_batch_stride, L, rows, cols, CLT_F8_E4M3, 1, kn ? wk : f, kn ? wks : fs, kn ? f : wk, kn ? fs : wks,
                       nullptr, nullptr, 0, stream);
    if (rc != CLT_OK || !T) return rc;
    rc = clt_pack8(x, x_dtype, x_token_stride, x_layer_stride, L, T, K, CLT_F8_E4M3, 0, q, s, xt, xs, nullptr, nullptr, 0, stream);
    if (rc != CLT_OK) return rc;
    return product({q, s, T}, {f, fs, N}, L, K, y, x_dtype, (long)L * N, N, bias, N, at, clt_gemm8_workspace_bytes(T, N, K, L), stream);
}

extern "C" size_t clt_linear8_backward_workspace_bytes(int T, int L, int K, int N, int need_dx, int need_dw, int need_db) {
    if (bad(T, L, K, N)) return 0;
    const size_t px = need_dx ? clt_gemm8_workspace_bytes(T, K, N, L) : 0;
    const size_t pa = need_dw ? clt_gemm8_workspace_bytes(K, N, T, L) : 0, pb = need_dw ? clt_gemm8_workspace_bytes(N, K, T, L) : 0;
    const size_t pw = pa > pb ? pa : pb, sums = need_db ? clt_pack8_sums_workspace_bytes(L, T, N) : 0;
    const size_t part = px > pw ? px : pw;
    return (size_t)((need_dx || !need_dw ? held(L, T, N) : 0) + (need_dw ? held(L, N, T) : 0)) + (part > sums ? part : sums);
}

extern "C" int clt_linear8_backward(const void* dy, int dtype, long token_stride, long layer_stride, const void* kept, int has_x, int kn, int T,
                                    int L, int K, int N, void* dx, void* dw, int dw_dtype, float* db, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    if (bad(T, L, K, N) || (!dx && !dw && !db)) return CLT_ERR_SHAPE;
    if ((dx || dw) && T && (!kept || !aligned16(kept))) return CLT_ERR_WORKSPACE;
    const size_t need = clt_linear8_backward_workspace_bytes(T, L, K, N, dx != nullptr, dw != nullptr, db != nullptr);
    if (need && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return CLT_ERR_WORKSPACE;
    uint8_t* at = static_cast<uint8_t*>(workspace);
    const uint8_t *kp = static_cast<const uint8_t*>(kept), *xs = kp + codes(L, K, T), *wk = kp + (has_x ? held(L, K, T) : 0), *wks = wk + codes(L, K, N);
    uint8_t *q = nullptr, *s = nullptr, *qt = nullptr, *qs = nullptr;
    if (dx || !dw) { q = take(at, codes(L, T, N)); s = take(at, held(L, T, N) - codes(L, T, N)); }   // (the bias gradient rides along with a pack; alone it takes one)
    if (dw) { qt = take(at, codes(L, N, T)); qs = take(at, held(L, N, T) - codes(L, N, T)); }
    int rc = CLT_OK;
    if (T) rc = clt_pack8(dy, dtype, token_stride, layer_stride, L, T, N, CLT_F8_E4M3, 0, q, s, qt, qs, db, at, db ? clt_pack8_sums_workspace_bytes(L, T, N) : 0, stream);
    if (rc == CLT_OK && T && dx)
        rc = product({q, s, T}, {wk, wks, K}, L, N, dx, dtype, (long)L * K, K, nullptr, 0, at, clt_gemm8_workspace_bytes(T, K, N, L), stream);
    if (rc == CLT_OK && dw) {
        const Operand a = {kp, xs, K}, b = {qt, qs, N};
        const int m = kn ? K : N, n = kn ? N : K;
        rc = product(kn ? a : b, kn ? b : a, L, T, dw, dw_dtype, n, (long)m * n, nullptr, 0, at, clt_gemm8_workspace_bytes(m, n, T, L), stream);
    }
    return rc;
}
