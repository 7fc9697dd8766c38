// C entry points of the 8-bit integer products: argument checks and the choice between the tiled
// form (int8_gemm.cu) and the split one (int8_skinny.cu).
#include "int8_gemm.cu"
#include "int8_skinny.cu"

namespace {

// Bytes that a lane may store at once into rows of `ld` elements at p: the widest power of two up to 16 that
// divides both the address and the row's bytes.
int store_width(const void* p, int64_t ld, int esize) {
    int w = 16;
    while (w > esize && ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * esize)) & (w - 1))) w /= 2;
    return w;
}

int64_t i8_steps(int64_t Ka) { return (Ka + I8_KT - 1) / I8_KT; }

// The form with the shorter estimate.
template <int P, int EPI>
int run_codes(I8Params& p, const I8Operands& o, int ops, cudaStream_t st) {
    const int64_t k_steps = i8_steps(o.Ka);
    const SkPlan q = sk_plan(p.M, p.N, k_steps, P, ops, -1);
    const TilePlan t = tile_plan<P, EPI>(p.M, p.N, k_steps, EPI == I8_DIGIT && p.tail, p.dependent != 0);
    if (q.ok && q.ns < t.ns) return run_skinny_codes<EPI, P>(p, o, q, st);
    return launch_i8<P, EPI>(p, o, t, st);
}

template <int EPI>
int run_fused(SkParams& p, int x_dtype, const SkPlan& q, cudaStream_t st) {
    if (x_dtype == IMA_DTYPE_BF16) return launch_skinny<EPI, 1, IMA_DTYPE_BF16>(p, q, st);
    if (x_dtype == IMA_DTYPE_F16) return launch_skinny<EPI, 1, IMA_DTYPE_F16>(p, q, st);
    return launch_skinny<EPI, 1, IMA_DTYPE_F32>(p, q, st);
}

// Whether the tokens are quantised inside the product: if it can, and that costs no more than a launch of the row
// quantiser, whose work the product's start hides in part.  A short product is over before the host has issued
// the next call, so the launch counts by the host's 2 us; behind a longer one (from 10 us on) it counts half of one: 3584 x
// 18944 with one token takes 19.5 us fused and 18.2 apart, 4864 x 896 8.8 and 7.7 but 12.7 and 15 issued one by one.
bool fused_plan(int64_t M, int64_t N, int64_t K, int ops, int x_dtype, SkPlan& q) {
    if (M < 1 || M > SK_MAX_TM || N < 1) return false;
    q = sk_plan(M, N, i8_steps(K), 1, ops, x_dtype);
    if (!q.ok) return false;
    const SkPlan codes = sk_plan(M, N, i8_steps(K), 1, ops, -1);
    const double tiled = ops == 2 ? tile_plan<1, I8_GATED>(M, N, i8_steps(K), false, true).ns
                                  : tile_plan<1, I8_LINEAR>(M, N, i8_steps(K), false, true).ns;
    const double apart = std::min(codes.ok ? codes.ns : tiled, tiled);
    return q.ns <= apart + (apart < 10000.0 ? 2000.0 : 500.0);
}

}  // namespace

namespace {

// What the launch before a product wrote of its operands: nothing, its activations, or weights too.
constexpr int AFTER_NOTHING = 0, AFTER_TOKENS = 1, AFTER_WEIGHTS = 2;

struct Pair8 { int8_t* p[2]; };
struct PairL { int64_t v[2]; };
struct PairF { float* p[2]; };
struct PairV { const void* p[2]; };

// The quantisers before a product: of the activations unless it quantises them itself, and of the weights that are
// given as floating tensors; one launch where the types agree.  `after`: see above.
int quantise_all(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                 bool fused, Pair8 w, PairL ldw, PairF w_scale, PairV src, PairL ldsrc, int src_dtype, int64_t N, int& after,
                 cudaStream_t st) {
    QuantRows weights = {}, tokens = {};
    weights.K = tokens.K = K;
    int nw = 0, nt = 0, rc = IMA_OK;
    const bool any = src.p[0] || src.p[1];
    if (any && !known_dtype(src_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    const bool together = any && !fused && src_dtype == x_dtype;
    if (!fused) rc = add_quantize(together ? weights : tokens, together ? nw : nt, x, M, ldx, q, ldq, scale);
    for (int i = 0; i < 2 && rc == IMA_OK; ++i)
        if (src.p[i]) rc = add_quantize(weights, nw, src.p[i], N, ldsrc.v[i], w.p[i], ldw.v[i], w_scale.p[i]);
    if (rc == IMA_OK && nw > 0) rc = run_quantize(weights, src_dtype, st);
    if (rc == IMA_OK && nt > 0) rc = run_quantize(tokens, x_dtype, st);
    // a product that starts early may read weights before it waits unless the launch right before it wrote them
    after = fused || M == 0 ? AFTER_NOTHING : together ? AFTER_WEIGHTS : AFTER_TOKENS;
    return rc;
}

int int8_gemm_entry(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, int64_t M, int64_t N, int64_t K,
                  int32_t* c, int64_t ldc, const float* x_scale, const float* w_scale, const void* bias, int bias_dtype,
                  void* y, int y_dtype, int64_t ldy, int dependent, void* stream) {
    int rc = check_i8_operand(a, M, K, lda);
    if (rc == IMA_OK) rc = check_i8_operand(b, N, K, ldb);
    if (rc != IMA_OK) return rc;
    if (M == 0 || N == 0) return IMA_OK;
    if (!c && !y) return IMA_ERR_INVALID_ARGUMENT;
    if (c && ldc < N && M > 1) return IMA_ERR_INVALID_ARGUMENT;
    if (y && (!x_scale || !w_scale || (ldy < N && M > 1) || !known_dtype(y_dtype))) return IMA_ERR_INVALID_ARGUMENT;
    if (y && bias && !known_dtype(bias_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    I8Params p;
    memset(&p, 0, sizeof(p));
    p.c = c; p.y = y; p.xs = x_scale; p.ws[0] = w_scale; p.bias[0] = bias; p.bias_dtype = bias_dtype;
    p.ldc = ldc; p.ldy = ldy; p.y_dtype = y_dtype;
    p.M = (int32_t)M; p.N = (int32_t)N; p.dependent = dependent;
    p.c_width = store_width(c, ldc, 4);
    p.y_width = store_width(y, ldy, y ? dtype_bytes(y_dtype) : 4);
    return run_codes<1, I8_LINEAR>(p, {a, b, nullptr, lda, ldb, 0, K, K, M * lda}, 1, (cudaStream_t)stream);
}

int int8_gated_entry(const int8_t* a, int64_t lda, const int8_t* gate, int64_t ldg, const int8_t* up, int64_t ldu,
                        int64_t M, int64_t N, int64_t K, const float* x_scale, const float* gate_scale,
                        const float* up_scale, const void* gate_bias, const void* up_bias, int bias_dtype,
                        int activation, void* y, int y_dtype, int64_t ldy, int dependent, void* stream) {
    int rc = check_i8_operand(a, M, K, lda);
    if (rc == IMA_OK) rc = check_i8_operand(gate, N, K, ldg);
    if (rc == IMA_OK) rc = check_i8_operand(up, N, K, ldu);
    if (rc != IMA_OK) return rc;
    if (activation != IMA_ACT_SILU && activation != IMA_ACT_GELU && activation != IMA_ACT_GELU_TANH) return IMA_ERR_UNSUPPORTED;
    if (M == 0 || N == 0) return IMA_OK;
    if (!y || !x_scale || !gate_scale || !up_scale || (ldy < N && M > 1) || !known_dtype(y_dtype))
        return IMA_ERR_INVALID_ARGUMENT;
    if ((gate_bias || up_bias) && !known_dtype(bias_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    I8Params p;
    memset(&p, 0, sizeof(p));
    p.y = y; p.xs = x_scale; p.ws[0] = gate_scale; p.ws[1] = up_scale; p.bias[0] = gate_bias; p.bias[1] = up_bias;
    p.bias_dtype = bias_dtype; p.ldy = ldy; p.y_dtype = y_dtype; p.act = act_form(activation, y_dtype == IMA_DTYPE_F32);
    p.M = (int32_t)M; p.N = (int32_t)N; p.dependent = dependent;
    p.y_width = store_width(y, ldy, dtype_bytes(y_dtype));
    return run_codes<1, I8_GATED>(p, {a, gate, up, lda, ldg, ldu, K, K, M * lda}, 2, (cudaStream_t)stream);
}

}  // namespace

extern "C" {

int ima_int8_gemm(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, int64_t M, int64_t N, int64_t K,
                  int32_t* c, int64_t ldc, const float* x_scale, const float* w_scale, const void* bias, int bias_dtype,
                  void* y, int y_dtype, int64_t ldy, void* stream) {
    return int8_gemm_entry(a, lda, b, ldb, M, N, K, c, ldc, x_scale, w_scale, bias, bias_dtype, y, y_dtype, ldy, 0, stream);
}

// Operator entries: floating activations in.  Few tokens: one launch, quantiser inside.  Otherwise the row
// quantiser into q and scale, then the product.
int ima_int8_fused(int64_t M, int64_t N, int64_t K, int gated, int x_dtype) {
    SkPlan plan;
    return K >= 0 && K <= I8_MAX_K && fused_plan(M, N, K, gated ? 2 : 1, x_dtype, plan) ? 1 : 0;
}

int ima_int8_linear(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                    int keep_codes, int8_t* w, int64_t ldw, int64_t N, float* w_scale, const void* w_src,
                    int w_src_dtype, int64_t ldw_src, const void* bias, int bias_dtype, void* y, int64_t ldy,
                    void* stream) {
    if (M < 0 || K < 0 || !known_dtype(x_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    cudaStream_t st = (cudaStream_t)stream;
    int rc = check_i8_operand(w, N, K, ldw);
    if (rc != IMA_OK) return rc;
    if (M > 0 && K > 0 && (!x || (M > 1 && ldx < K))) return IMA_ERR_INVALID_ARGUMENT;
    SkPlan plan;
    const bool fused = !keep_codes && fused_plan(M, N, K, 1, x_dtype, plan);
    int after = AFTER_NOTHING;
    rc = quantise_all(x, x_dtype, M, K, ldx, q, ldq, scale, fused, {w, nullptr}, {ldw, 0}, {w_scale, nullptr},
                      {w_src, nullptr}, {ldw_src, 0}, w_src_dtype, N, after, st);
    if (rc != IMA_OK) return rc;
    if (fused) {
        if (!y || !w_scale || (ldy < N && M > 1) || (bias && !known_dtype(bias_dtype))) return IMA_ERR_INVALID_ARGUMENT;
        SkParams p;
        memset(&p, 0, sizeof(p));
        p.x = x; p.ldx = ldx; p.K = K; p.M = (int32_t)M; p.N = (int32_t)N;
        p.y = y; p.ldy = ldy; p.y_dtype = x_dtype; p.ws[0] = w_scale; p.bias[0] = bias; p.bias_dtype = bias_dtype;
        p.vec_y = store_width(y, ldy, dtype_bytes(x_dtype)) >= 4 * dtype_bytes(x_dtype);
        rc = sk_weight_maps(p, {nullptr, w, nullptr, 0, ldw, 0, K, K, 0});
        if (rc != IMA_OK) return rc;
        return run_fused<I8_LINEAR>(p, x_dtype, plan, st);
    }
    return int8_gemm_entry(q, ldq, w, ldw, M, N, K, nullptr, N, scale, w_scale, bias, bias_dtype, y, x_dtype, ldy, after, stream);
}

int ima_int8_gated(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                   int keep_codes, int8_t* gate, int64_t ldg, int8_t* up, int64_t ldu, int64_t N, float* gate_scale,
                   float* up_scale, const void* gate_src, int64_t ldgate_src, const void* up_src, int64_t ldup_src,
                   int w_src_dtype, const void* gate_bias, const void* up_bias, int bias_dtype, int activation, void* y,
                   int64_t ldy, void* stream) {
    if (M < 0 || K < 0 || !known_dtype(x_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    cudaStream_t st = (cudaStream_t)stream;
    int rc = check_i8_operand(gate, N, K, ldg);
    if (rc == IMA_OK) rc = check_i8_operand(up, N, K, ldu);
    if (rc != IMA_OK) return rc;
    if (activation != IMA_ACT_SILU && activation != IMA_ACT_GELU && activation != IMA_ACT_GELU_TANH) return IMA_ERR_UNSUPPORTED;
    if (M > 0 && K > 0 && (!x || (M > 1 && ldx < K))) return IMA_ERR_INVALID_ARGUMENT;
    SkPlan plan;
    const bool fused = !keep_codes && fused_plan(M, N, K, 2, x_dtype, plan);
    int after = AFTER_NOTHING;
    rc = quantise_all(x, x_dtype, M, K, ldx, q, ldq, scale, fused, {gate, up}, {ldg, ldu}, {gate_scale, up_scale},
                      {gate_src, up_src}, {ldgate_src, ldup_src}, w_src_dtype, N, after, st);
    if (rc != IMA_OK) return rc;
    if (fused) {
        if (!y || !gate_scale || !up_scale || (ldy < N && M > 1) || ((gate_bias || up_bias) && !known_dtype(bias_dtype)))
            return IMA_ERR_INVALID_ARGUMENT;
        SkParams p;
        memset(&p, 0, sizeof(p));
        p.x = x; p.ldx = ldx; p.K = K; p.M = (int32_t)M; p.N = (int32_t)N;
        p.y = y; p.ldy = ldy; p.y_dtype = x_dtype; p.act = act_form(activation, x_dtype == IMA_DTYPE_F32);
        p.ws[0] = gate_scale; p.ws[1] = up_scale; p.bias[0] = gate_bias; p.bias[1] = up_bias; p.bias_dtype = bias_dtype;
        p.vec_y = store_width(y, ldy, dtype_bytes(x_dtype)) >= 4 * dtype_bytes(x_dtype);
        rc = sk_weight_maps(p, {nullptr, gate, up, 0, ldg, ldu, K, K, 0});
        if (rc != IMA_OK) return rc;
        return run_fused<I8_GATED>(p, x_dtype, plan, st);
    }
    return int8_gated_entry(q, ldq, gate, ldg, up, ldu, M, N, K, scale, gate_scale, up_scale, gate_bias, up_bias,
                            bias_dtype, activation, y, x_dtype, ldy, after, stream);
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Backward passes.  Launches, in order: W and q transposed (and the maxima zeroed), [g and u again, their
// gradients D and D's maxima | D's maxima], the digits of D by rows and by columns with the partial bias
// sums, dx, dW, bias sums.
// ---------------------------------------------------------------------------
namespace {

constexpr int BWD_DX = 1, BWD_DW = 2, BWD_DB = 4, BWD_OWN_WT = 8;

struct BwdPlan {
    int64_t pitch, W, ldm, ldwt;
    int64_t maxima, maxima_bytes, d, rows, row_scale, cols, col_scale, q_t, w_t, partial, tail, total;   // offsets
    bool has_tail;
};

BwdPlan bwd_plan(int64_t M, int64_t N, int64_t K, int segs, int planes, int want) {
    BwdPlan b = {};
    // segments of a pair start on a k-tile of the dx product and on a row tile of the dW product
    b.pitch = segs == 2 ? (N + 127) / 128 * 128 : (N + 15) / 16 * 16;
    b.W = segs * b.pitch;
    b.ldm = (M + 15) / 16 * 16;
    b.ldwt = (N + 15) / 16 * 16;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at += (bytes + 255) / 256 * 256;
        return o;
    };
    const bool dx = want & BWD_DX, dw = want & BWD_DW;
    b.maxima_bytes = (M + b.W) * 4;
    b.maxima = take(b.maxima_bytes);
    if (segs == 2) b.d = take(M * b.W * 4);
    if (dx) {
        b.rows = take(planes * M * b.W);
        b.row_scale = take(M * 4);
    }
    if (dw) {
        b.cols = take(planes * b.W * b.ldm);
        b.col_scale = take(b.W * 4);
        b.q_t = take(K * b.ldm);
    }
    if (want & BWD_OWN_WT) b.w_t = take(segs * K * b.ldwt);
    if (want & BWD_DB) b.partial = take((M + 127) / 128 * b.W * 8);
    // more 128 x 128 blocks than workers: the tiled form may have a tail to split
    const int64_t kb = (K + 127) / 128;
    b.has_tail = (dx && (M + 127) / 128 * kb > 74) || (dw && (b.W + 127) / 128 * kb > 74);
    if (b.has_tail) b.tail = take(I8_TAIL_BYTES);
    b.total = at;
    return b;
}

struct BwdArgs {
    const void* grad;
    int grad_dtype;
    int64_t ldg, M, N, K;
    const int8_t* q;
    int64_t ldq;
    const float* scale;
    int segs;
    const int8_t* w[2];
    int64_t ldw[2];
    const int8_t* w_t[2];          // [K, N] (NULL: made in the workspace)
    int64_t ldwt[2];
    const float* w_scale[2];
    const void* bias[2];
    int bias_dtype, activation, planes;
    void* dx;
    int dx_dtype;
    void* dw[2];
    int dw_dtype;
    void* db[2];
    int db_dtype;
    void* workspace;
};

int zero_out(void* p, int64_t n, int dtype, cudaStream_t st) {
    if (!p || n == 0) return IMA_OK;
    return ima_note_cuda(cudaMemsetAsync(p, 0, (size_t)(n * dtype_bytes(dtype)), st));
}

template <int P>
int bwd_products(const BwdArgs& a, const BwdPlan& b, unsigned char* ws, cudaStream_t st) {
    int rc = IMA_OK;
    if (a.dx) {
        const int8_t* wt[2] = {a.w_t[0], a.w_t[1]};
        int64_t ldwt[2] = {a.ldwt[0], a.ldwt[1]};
        for (int i = 0; i < a.segs; ++i)
            if (!wt[i]) {
                wt[i] = reinterpret_cast<const int8_t*>(ws + b.w_t) + i * a.K * b.ldwt;
                ldwt[i] = b.ldwt;
            }
        I8Params p;
        memset(&p, 0, sizeof(p));
        p.y = a.dx; p.ldy = a.K; p.y_dtype = a.dx_dtype; p.xs = reinterpret_cast<const float*>(ws + b.row_scale);
        p.M = (int32_t)a.M; p.N = (int32_t)a.K;
        p.y_width = store_width(a.dx, a.K, dtype_bytes(a.dx_dtype));
        p.seg_tiles = (int32_t)i8_steps(a.N);
        p.tail = b.has_tail ? reinterpret_cast<int32_t*>(ws + b.tail) : nullptr;
        const I8Operands o = {reinterpret_cast<const int8_t*>(ws + b.rows), wt[0], a.segs == 2 ? wt[1] : nullptr, b.W,
                              ldwt[0], ldwt[1], (a.segs - 1) * b.pitch + a.N, a.N, a.M * b.W};
        if (a.K > 0) rc = run_codes<P, I8_DIGIT>(p, o, 1, st);
        if (rc != IMA_OK) return rc;
    }
    if ((a.dw[0] || a.dw[1]) && a.K > 0) {
        const int8_t* qt = reinterpret_cast<const int8_t*>(ws + b.q_t);
        const int first = a.dw[0] ? 0 : 1;
        const bool both = a.dw[0] && a.dw[1];
        I8Params p;
        memset(&p, 0, sizeof(p));
        p.y = a.dw[first]; p.ldy = a.K; p.y_dtype = a.dw_dtype;
        p.xs = reinterpret_cast<const float*>(ws + b.col_scale) + first * b.pitch;
        p.M = (int32_t)(both ? b.pitch + a.N : a.N); p.N = (int32_t)a.K;
        p.y_width = store_width(p.y, a.K, dtype_bytes(a.dw_dtype));
        if (both) {
            p.y2 = a.dw[1]; p.split_row = b.pitch; p.seg_rows = a.N;
            p.y_width = std::min(p.y_width, store_width(p.y2, a.K, dtype_bytes(a.dw_dtype)));
        }
        p.seg_tiles = (int32_t)i8_steps(a.M);
        p.tail = b.has_tail ? reinterpret_cast<int32_t*>(ws + b.tail) : nullptr;
        const I8Operands o = {reinterpret_cast<const int8_t*>(ws + b.cols) + first * b.pitch * b.ldm, qt, nullptr, b.ldm,
                              b.ldm, 0, a.M, a.M, b.W * b.ldm};
        rc = run_codes<P, I8_DIGIT>(p, o, 1, st);
    }
    return rc;
}

int run_backward(const BwdArgs& a, cudaStream_t st) {
    const bool want_dw = a.dw[0] || a.dw[1], want_db = a.db[0] || a.db[1];
    if (a.M < 0 || a.N < 0 || a.K < 0 || !known_dtype(a.grad_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    if (a.planes != 2 && a.planes != 3) return IMA_ERR_UNSUPPORTED;
    if ((a.dx && !known_dtype(a.dx_dtype)) || (want_dw && !known_dtype(a.dw_dtype)) || (want_db && !known_dtype(a.db_dtype)))
        return IMA_ERR_INVALID_ARGUMENT;
    int rc = check_i8_operand(a.q, a.M, a.K, a.ldq);
    for (int i = 0; i < a.segs && rc == IMA_OK; ++i) {
        rc = check_i8_operand(a.w[i], a.N, a.K, a.ldw[i]);
        if (rc == IMA_OK && a.dx && a.w_t[i]) rc = check_i8_operand(a.w_t[i], a.K, a.N, a.ldwt[i]);
    }
    if (rc != IMA_OK) return rc;
    const bool own = a.dx && (!a.w_t[0] || (a.segs == 2 && !a.w_t[1]));
    const BwdPlan b = bwd_plan(a.M, a.N, a.K, a.segs, a.planes,
                               (a.dx ? BWD_DX : 0) | (want_dw ? BWD_DW : 0) | (want_db ? BWD_DB : 0) | (own ? BWD_OWN_WT : 0));
    if ((a.dx && (a.segs - 1) * b.pitch + a.N > I8_MAX_K) || (want_dw && a.M > I8_MAX_K)) return IMA_ERR_UNSUPPORTED;
    if (b.W > INT32_MAX / 2 || (a.M + 63) / 64 > 65535 || (a.N + 127) / 128 > 65535) return IMA_ERR_UNSUPPORTED;
    if (a.M == 0 || a.N == 0) {   // empty sums
        if (a.dx) rc = zero_out(a.dx, a.M * a.K, a.dx_dtype, st);
        for (int i = 0; i < a.segs && rc == IMA_OK; ++i) {
            rc = zero_out(a.dw[i], a.N * a.K, a.dw_dtype, st);
            if (rc == IMA_OK) rc = zero_out(a.db[i], a.N, a.db_dtype, st);
        }
        return rc;
    }
    if (!a.dx && !want_dw && !want_db) return IMA_OK;
    if (!a.grad || !a.scale || !a.workspace || (a.M > 1 && a.ldg < a.N)) return IMA_ERR_INVALID_ARGUMENT;
    for (int i = 0; i < a.segs; ++i)
        if (!a.w_scale[i]) return IMA_ERR_INVALID_ARGUMENT;
    unsigned char* ws = reinterpret_cast<unsigned char*>(a.workspace);
    uint32_t* row_max = reinterpret_cast<uint32_t*>(ws + b.maxima);
    GradDigits d;
    memset(&d, 0, sizeof(d));
    GradSrc& g = d.g;
    g.src = a.grad; g.ld = a.ldg; g.M = a.M; g.n = a.N; g.pitch = b.pitch; g.W = b.W; g.xs = a.scale;
    g.ws[0] = a.w_scale[0]; g.ws[1] = a.w_scale[1];
    g.row_max = a.dx ? row_max : nullptr;
    g.col_max = want_dw ? row_max + a.M : nullptr;
    if (a.dx || want_dw) {   // the transposed operands, and the maxima at zero
        TransposeJobs t = {};
        int n = 0;
        t.zero = row_max;
        t.zero_words = b.maxima_bytes / 4;
        if (a.K > 0) {
            for (int i = 0; i < a.segs && a.dx; ++i)
                if (!a.w_t[i])
                    add_transpose(t, n, a.w[i], a.N, a.K, a.ldw[i], reinterpret_cast<int8_t*>(ws + b.w_t) + i * a.K * b.ldwt, b.ldwt);
            if (want_dw) add_transpose(t, n, a.q, a.M, a.K, a.ldq, reinterpret_cast<int8_t*>(ws + b.q_t), b.ldm);
        }
        rc = run_transposes(t, st);
        if (rc != IMA_OK) return rc;
    }
    int src_dtype = a.grad_dtype;
    if (a.segs == 2) {
        I8Params p;
        memset(&p, 0, sizeof(p));
        p.xs = a.scale; p.ws[0] = a.w_scale[0]; p.ws[1] = a.w_scale[1]; p.bias[0] = a.bias[0]; p.bias[1] = a.bias[1];
        p.bias_dtype = a.bias_dtype; p.act = a.activation; p.dh = a.grad; p.dh_dtype = a.grad_dtype; p.ldh = a.ldg;
        p.d = reinterpret_cast<float*>(ws + b.d); p.ldd = b.W; p.seg_pitch = b.pitch;
        p.row_max = g.row_max; p.col_max = g.col_max;
        p.M = (int32_t)a.M; p.N = (int32_t)a.N;
        rc = launch_i8<1, I8_GATED_BWD>(p, {a.q, a.w[0], a.w[1], a.ldq, a.ldw[0], a.ldw[1], a.K, a.K, a.M * a.ldq},
                                         tile_plan<1, I8_GATED_BWD>(a.M, a.N, i8_steps(a.K), false, false), st);
        if (rc != IMA_OK) return rc;
        g.src = p.d;
        g.ld = b.W;
        src_dtype = IMA_DTYPE_F32;
    } else if (a.dx || want_dw) {
        rc = run_grad_max(g, src_dtype, st);
        if (rc != IMA_OK) return rc;
    }
    if (a.dx) {
        d.rows = reinterpret_cast<int8_t*>(ws + b.rows);
        d.row_scale = reinterpret_cast<float*>(ws + b.row_scale);
    }
    if (want_dw) {
        d.cols = reinterpret_cast<int8_t*>(ws + b.cols);
        d.col_scale = reinterpret_cast<float*>(ws + b.col_scale);
    }
    if (want_db) d.partial = reinterpret_cast<double*>(ws + b.partial);
    d.ldm = b.ldm;
    rc = run_grad_digits(d, src_dtype, a.planes, st);
    if (rc != IMA_OK) return rc;
    rc = a.planes == 2 ? bwd_products<2>(a, b, ws, st) : bwd_products<3>(a, b, ws, st);
    if (rc == IMA_OK && want_db) {
        const dim3 grid((unsigned)((a.N + 255) / 256), (unsigned)a.segs);
        int8_col_sum_kernel<<<grid, 256, 0, st>>>(d.partial, (a.M + 127) / 128, b.W, a.N, b.pitch, a.db[0], a.db[1],
                                                  a.db_dtype);
        rc = IMA_LAUNCH_STATUS();
    }
    return rc;
}

}  // namespace

extern "C" {

int64_t ima_int8_backward_workspace_bytes(int64_t M, int64_t N, int64_t K, int gated, int planes, int dx, int dw, int db,
                                          int own_transposed) {
    if (M < 0 || N < 0 || K < 0) return 0;
    const int want = (dx ? BWD_DX : 0) | (dw ? BWD_DW : 0) | (db ? BWD_DB : 0) | (dx && own_transposed ? BWD_OWN_WT : 0);
    return bwd_plan(M, N, K, gated ? 2 : 1, planes, want).total;
}

int ima_int8_linear_backward(const void* grad, int grad_dtype, int64_t ldg, int64_t M, int64_t N, int64_t K,
                             const int8_t* q, int64_t ldq, const float* scale, const int8_t* w, int64_t ldw,
                             const int8_t* w_t, int64_t ldwt, const float* w_scale, int planes, void* dx, int dx_dtype,
                             void* dw, int dw_dtype, void* db, int db_dtype, void* workspace, void* stream) {
    BwdArgs a;
    memset(&a, 0, sizeof(a));
    a.grad = grad; a.grad_dtype = grad_dtype; a.ldg = ldg; a.M = M; a.N = N; a.K = K; a.q = q; a.ldq = ldq; a.scale = scale;
    a.segs = 1; a.w[0] = w; a.ldw[0] = ldw; a.w_t[0] = w_t; a.ldwt[0] = ldwt; a.w_scale[0] = w_scale; a.planes = planes;
    a.dx = dx; a.dx_dtype = dx_dtype; a.dw[0] = dw; a.dw_dtype = dw_dtype; a.db[0] = db; a.db_dtype = db_dtype;
    a.workspace = workspace;
    return run_backward(a, (cudaStream_t)stream);
}

int ima_int8_gated_backward(const void* grad, int grad_dtype, int64_t ldg, int64_t M, int64_t N, int64_t K,
                            const int8_t* q, int64_t ldq, const float* scale, const int8_t* gate, int64_t ldgate,
                            const int8_t* up, int64_t ldup, const int8_t* gate_t, int64_t ldgate_t, const int8_t* up_t,
                            int64_t ldup_t, const float* gate_scale, const float* up_scale, const void* gate_bias,
                            const void* up_bias, int bias_dtype, int activation, int planes, void* dx, int dx_dtype,
                            void* dgate, void* dup, int dw_dtype, void* dgate_bias, void* dup_bias, int db_dtype,
                            void* workspace, void* stream) {
    if (activation != IMA_ACT_SILU && activation != IMA_ACT_GELU && activation != IMA_ACT_GELU_TANH) return IMA_ERR_UNSUPPORTED;
    if ((gate_bias || up_bias) && !known_dtype(bias_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    const BwdArgs a = {grad, grad_dtype, ldg, M, N, K, q, ldq, scale, 2, {gate, up}, {ldgate, ldup}, {gate_t, up_t},
                       {ldgate_t, ldup_t}, {gate_scale, up_scale}, {gate_bias, up_bias}, bias_dtype, activation, planes,
                       dx, dx_dtype, {dgate, dup}, dw_dtype, {dgate_bias, dup_bias}, db_dtype, workspace};
    return run_backward(a, (cudaStream_t)stream);
}

}  // extern "C"
