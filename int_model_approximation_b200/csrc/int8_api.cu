// C entry points of the 8-bit integer products: argument checks and the choice between the tiled
// form (int8_gemm.cu) and the split one (int8_skinny.cu).
#include "int8_gemm.cu"
#include "int8_skinny.cu"

namespace {

int64_t i8_steps(int64_t Ka) { return (Ka + I8_KT - 1) / I8_KT; }

// Time of the tiled form in ns: rounds of 128 x BN tiles over the machine at the tensor core's rate (8192
// multiplications per clock and SM at 1.6 GHz), two thirds of it while a stage's loads limit it, and
// the fill and drain of its pipeline.
double tiled_ns(int64_t M, int64_t N, int64_t k_steps, int planes, int bn) {
    const int64_t tiles = ((M + I8_BM - 1) / I8_BM) * ((N + bn - 1) / bn);
    const int64_t rounds = (tiles + gemm_grid_limit() - 1) / gemm_grid_limit();
    return (double)rounds * (double)k_steps * planes * bn * 128.0 * 128.0 / (8192.0 * 1.6 * 0.67) + 3000.0;
}

// The form with the shorter estimate.
int run_linear(I8Params& p, const I8Operands& o, cudaStream_t st) {
    const SkPlan q = sk_plan(p.M, p.N, i8_steps(o.K), 1, 1, false);
    if (q.ok && q.ns < tiled_ns(p.M, p.N, i8_steps(o.K), 1, 256)) return run_skinny_codes<I8_LINEAR, 1>(p, o, q, st);
    return launch_i8<1, 256, I8_LINEAR>(p, o, st);
}

int run_gated(I8Params& p, const I8Operands& o, cudaStream_t st) {
    const SkPlan q = sk_plan(p.M, p.N, i8_steps(o.K), 1, 2, false);
    if (q.ok && q.ns < tiled_ns(p.M, 2 * (int64_t)p.N, i8_steps(o.K), 1, 256))
        return run_skinny_codes<I8_GATED, 1>(p, o, q, st);
    return launch_i8<1, 256, I8_GATED>(p, o, st);
}

template <int P, int BN>
int run_digits(I8Params& p, const I8Operands& o, cudaStream_t st) {
    const SkPlan q = sk_plan(p.M, p.N, i8_steps(o.Ka), P, 1, false);
    if (q.ok && q.ns < tiled_ns(p.M, p.N, i8_steps(o.Ka), P, BN)) return run_skinny_codes<I8_DIGIT, P>(p, o, q, st);
    return launch_i8<P, BN, I8_DIGIT>(p, o, st);
}

template <int EPI>
int run_fused(SkParams& p, int x_dtype, const SkPlan& q, cudaStream_t st) {
    if (x_dtype == IMA_DTYPE_BF16) return launch_skinny<EPI, 1, IMA_DTYPE_BF16>(p, q, st);
    if (x_dtype == IMA_DTYPE_F16) return launch_skinny<EPI, 1, IMA_DTYPE_F16>(p, q, st);
    return launch_skinny<EPI, 1, IMA_DTYPE_F32>(p, q, st);
}

// Whether the tokens are quantised inside the product: every cluster then does it for itself, which
// pays while the workers hold a CTA's share in one batch of loads.
bool fused_wanted(int64_t M, const SkPlan& q) {
    return q.ok && M <= 16 && M * ((q.k_steps + q.splits - 1) / q.splits) * I8_KT <= SK_WORKERS * 32 * SK_BATCH * 8;
}

}  // namespace

namespace {

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
    p.vec_c = c && aligned16(c, ldc * 4);
    p.vec_y = y && aligned16(y, ldy * dtype_bytes(y_dtype));
    return run_linear(p, {a, b, nullptr, lda, ldb, 0, K, K}, (cudaStream_t)stream);
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
    p.bias_dtype = bias_dtype; p.ldy = ldy; p.y_dtype = y_dtype; p.act = activation;
    p.M = (int32_t)M; p.N = (int32_t)N; p.dependent = dependent;
    p.vec_y = aligned16(y, ldy * dtype_bytes(y_dtype));
    return run_gated(p, {a, gate, up, lda, ldg, ldu, K, K}, (cudaStream_t)stream);
}

}  // namespace

extern "C" {

int ima_int8_gemm(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, int64_t M, int64_t N, int64_t K,
                  int32_t* c, int64_t ldc, const float* x_scale, const float* w_scale, const void* bias, int bias_dtype,
                  void* y, int y_dtype, int64_t ldy, void* stream) {
    return int8_gemm_entry(a, lda, b, ldb, M, N, K, c, ldc, x_scale, w_scale, bias, bias_dtype, y, y_dtype, ldy, 0, stream);
}

int ima_int8_gated_gemm(const int8_t* a, int64_t lda, const int8_t* gate, int64_t ldg, const int8_t* up, int64_t ldu,
                        int64_t M, int64_t N, int64_t K, const float* x_scale, const float* gate_scale,
                        const float* up_scale, const void* gate_bias, const void* up_bias, int bias_dtype,
                        int activation, void* y, int y_dtype, int64_t ldy, void* stream) {
    return int8_gated_entry(a, lda, gate, ldg, up, ldu, M, N, K, x_scale, gate_scale, up_scale, gate_bias, up_bias,
                            bias_dtype, activation, y, y_dtype, ldy, 0, stream);
}

int ima_int8_gated_backward_gemm(const int8_t* a, int64_t lda, const int8_t* gate, int64_t ldg, const int8_t* up,
                                 int64_t ldu, int64_t M, int64_t N, int64_t K, const float* x_scale,
                                 const float* gate_scale, const float* up_scale, const void* gate_bias,
                                 const void* up_bias, int bias_dtype, int activation, const void* dh, int dh_dtype,
                                 int64_t ldh, float* d, int64_t ldd, int64_t seg_pitch, void* stream) {
    int rc = check_i8_operand(a, M, K, lda);
    if (rc == IMA_OK) rc = check_i8_operand(gate, N, K, ldg);
    if (rc == IMA_OK) rc = check_i8_operand(up, N, K, ldu);
    if (rc != IMA_OK) return rc;
    if (activation != IMA_ACT_SILU && activation != IMA_ACT_GELU && activation != IMA_ACT_GELU_TANH) return IMA_ERR_UNSUPPORTED;
    if (M == 0 || N == 0) return IMA_OK;
    if (!dh || !d || !x_scale || !gate_scale || !up_scale || !known_dtype(dh_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    if ((ldh < N && M > 1) || seg_pitch < N || (ldd < seg_pitch + N && M > 1)) return IMA_ERR_INVALID_ARGUMENT;
    if ((gate_bias || up_bias) && !known_dtype(bias_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    I8Params p;
    memset(&p, 0, sizeof(p));
    p.xs = x_scale; p.ws[0] = gate_scale; p.ws[1] = up_scale; p.bias[0] = gate_bias; p.bias[1] = up_bias;
    p.bias_dtype = bias_dtype; p.act = activation; p.dh = dh; p.dh_dtype = dh_dtype; p.ldh = ldh;
    p.d = d; p.ldd = ldd; p.seg_pitch = seg_pitch;
    p.M = (int32_t)M; p.N = (int32_t)N;
    p.vec_d = aligned16(d, ldd * 4) && seg_pitch % 4 == 0;
    return launch_i8<1, 256, I8_GATED_BWD>(p, {a, gate, up, lda, ldg, ldu, K, K}, (cudaStream_t)stream);
}

int ima_int8_digit_gemm(const int8_t* a_planes, int planes, int64_t lda, const float* row_scale, const int8_t* b,
                        int64_t ldb, const int8_t* b2, int64_t ldb2, int64_t M, int64_t N, int64_t K, void* y,
                        int y_dtype, int64_t ldy, void* stream) {
    if (planes != 2 && planes != 3) return IMA_ERR_UNSUPPORTED;
    // with a second B the planes hold two segments of K columns, the second on a k-tile boundary
    const int64_t seg = b2 ? (K + I8_KT - 1) / I8_KT * I8_KT : 0;
    int rc = check_i8_operand(a_planes, M, seg + K, lda);
    if (rc == IMA_OK) rc = check_i8_operand(b, N, K, ldb);
    if (rc == IMA_OK && b2) rc = check_i8_operand(b2, N, K, ldb2);
    if (rc != IMA_OK) return rc;
    if (M == 0 || N == 0) return IMA_OK;
    if (!y || !row_scale || (ldy < N && M > 1) || !known_dtype(y_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    I8Params p;
    memset(&p, 0, sizeof(p));
    p.y = y; p.xs = row_scale; p.ldy = ldy; p.y_dtype = y_dtype;
    p.M = (int32_t)M; p.N = (int32_t)N;
    p.vec_y = aligned16(y, ldy * dtype_bytes(y_dtype));
    p.seg_tiles = (int32_t)((K + I8_KT - 1) / I8_KT);
    const I8Operands o = {a_planes, b, b2, lda, ldb, ldb2, seg + K, K};
    if (planes == 2) return run_digits<2, 256>(p, o, (cudaStream_t)stream);
    return run_digits<3, 128>(p, o, (cudaStream_t)stream);
}

// Operator entries: floating activations in.  Few tokens: one launch, quantiser inside.  Otherwise the row
// quantiser into q and scale, then the product.
int ima_int8_linear(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                    int keep_codes, const int8_t* w, int64_t ldw, int64_t N, const float* w_scale, const void* bias,
                    int bias_dtype, void* y, int64_t ldy, void* stream) {
    if (M < 0 || K < 0 || !known_dtype(x_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    int rc = check_i8_operand(w, N, K, ldw);
    if (rc != IMA_OK) return rc;
    if (M > 0 && K > 0 && (!x || (M > 1 && ldx < K))) return IMA_ERR_INVALID_ARGUMENT;
    if (M > 0 && M <= 16 && N > 0 && !keep_codes) {
        const SkPlan plan = sk_plan(M, N, i8_steps(K), 1, 1, true);
        if (fused_wanted(M, plan)) {
            if (!y || !w_scale || (ldy < N && M > 1) || (bias && !known_dtype(bias_dtype))) return IMA_ERR_INVALID_ARGUMENT;
            SkParams p;
            memset(&p, 0, sizeof(p));
            p.x = x; p.ldx = ldx; p.K = K; p.M = (int32_t)M; p.N = (int32_t)N;
            p.y = y; p.ldy = ldy; p.y_dtype = x_dtype; p.ws[0] = w_scale; p.bias[0] = bias; p.bias_dtype = bias_dtype;
            p.vec_y = aligned16(y, ldy * dtype_bytes(x_dtype));
            rc = sk_weight_maps(p, {nullptr, w, nullptr, 0, ldw, 0, K, K});
            if (rc != IMA_OK) return rc;
            return run_fused<I8_LINEAR>(p, x_dtype, plan, (cudaStream_t)stream);
        }
    }
    rc = ima_int8_quantize_rows(x, x_dtype, M, K, ldx, q, ldq, scale, stream);
    if (rc != IMA_OK) return rc;
    return int8_gemm_entry(q, ldq, w, ldw, M, N, K, nullptr, N, scale, w_scale, bias, bias_dtype, y, x_dtype, ldy, 1, stream);
}

int ima_int8_gated(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                   int keep_codes, const int8_t* gate, int64_t ldg, const int8_t* up, int64_t ldu, int64_t N,
                   const float* gate_scale, const float* up_scale, const void* gate_bias, const void* up_bias,
                   int bias_dtype, int activation, void* y, int64_t ldy, void* stream) {
    if (M < 0 || K < 0 || !known_dtype(x_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    int rc = check_i8_operand(gate, N, K, ldg);
    if (rc == IMA_OK) rc = check_i8_operand(up, N, K, ldu);
    if (rc != IMA_OK) return rc;
    if (activation != IMA_ACT_SILU && activation != IMA_ACT_GELU && activation != IMA_ACT_GELU_TANH) return IMA_ERR_UNSUPPORTED;
    if (M > 0 && K > 0 && (!x || (M > 1 && ldx < K))) return IMA_ERR_INVALID_ARGUMENT;
    if (M > 0 && M <= 16 && N > 0 && !keep_codes) {
        const SkPlan plan = sk_plan(M, N, i8_steps(K), 1, 2, true);
        if (fused_wanted(M, plan)) {
            if (!y || !gate_scale || !up_scale || (ldy < N && M > 1) || ((gate_bias || up_bias) && !known_dtype(bias_dtype)))
                return IMA_ERR_INVALID_ARGUMENT;
            SkParams p;
            memset(&p, 0, sizeof(p));
            p.x = x; p.ldx = ldx; p.K = K; p.M = (int32_t)M; p.N = (int32_t)N;
            p.y = y; p.ldy = ldy; p.y_dtype = x_dtype; p.act = activation;
            p.ws[0] = gate_scale; p.ws[1] = up_scale; p.bias[0] = gate_bias; p.bias[1] = up_bias; p.bias_dtype = bias_dtype;
            p.vec_y = aligned16(y, ldy * dtype_bytes(x_dtype));
            rc = sk_weight_maps(p, {nullptr, gate, up, 0, ldg, ldu, K, K});
            if (rc != IMA_OK) return rc;
            return run_fused<I8_GATED>(p, x_dtype, plan, (cudaStream_t)stream);
        }
    }
    rc = ima_int8_quantize_rows(x, x_dtype, M, K, ldx, q, ldq, scale, stream);
    if (rc != IMA_OK) return rc;
    return int8_gated_entry(q, ldq, gate, ldg, up, ldu, M, N, K, scale, gate_scale, up_scale, gate_bias, up_bias,
                            bias_dtype, activation, y, x_dtype, ldy, 1, stream);
}

}  // extern "C"
