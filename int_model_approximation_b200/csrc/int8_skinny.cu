// 8-bit integer products of few tokens: the weight is streamed once, and the contraction is split
// over a cluster of CTAs.
//
// Roles of the operands are the other way round than in int8_gemm.cu: a tile is 128 weight rows
// (the M side of the MMA) by tm tokens (its N side, a multiple of 16 up to 128), so a single token
// costs one 16-column MMA and the work is the weight's bytes.  The gated form has 128 rows of G and
// 128 of U in a tile, the digit form stacks the P planes of the tokens: P * tm columns.
//
// Split: the k-steps (128 bytes) of a tile are dealt to the S CTAs of a cluster (1, 2, 4 or 8; see
// sk_plan).  Output rows are owned by CTAs, 128 / S each: every CTA pushes its int32 partial sums into
// the owners' shared memory, and after one cluster barrier each owner adds S of them and applies
// the epilogue.  Integer sums do not depend on the order.
//
// Fused quantiser: with the activations still floating and few, the 8 worker warps find the row
// maxima of the CTA's k-slice (exchanged through the cluster) and quantise the slice into the swizzled
// layout that the MMA reads, in shared memory, while the first weight tiles are on their way.  This
// saves a launch and a round trip of the codes.  Otherwise the row quantiser runs before, and this
// kernel is launched so that it starts, and loads its first weight tiles, while that one finishes.
//
// Measured: 16 tokens by 3584 x 18944 (68 MB of weights) 18.3 to 18.9 us, where a kernel that only loads them takes
// 15.0 and the measured copy rate would allow 10.4; the gated form of one token by 18944 x 3584 (136 MB) 27.8 us,
// 4.9 TB/s; one token by 4864 x 896 8.5 us, all of it latency.
#include "sm100_pair.cuh"

namespace {

constexpr int SK_ROWS = 128;                       // weight rows per tile and operand
constexpr int SK_WORKERS = 8;
constexpr int SK_THREADS = 64 + SK_WORKERS * 32;
constexpr int SK_MAX_STAGES = 8;
constexpr int SK_SMEM = 221 * 1024;              // with 5 KB static and 1 KB of the system: one CTA per SM at most
constexpr int SK_SMEM_HALF = 107 * 1024;           // two CTAs per SM
constexpr int SK_MAX_TM = 128;

// Groups of eight elements that a lane of the fused quantiser has in flight (32 registers).
__host__ __device__ constexpr int sk_batch(int dtype) { return dtype == IMA_DTYPE_F32 ? 4 : 8; }

struct __align__(64) SkParams {
    CUtensorMap mw, mw2, mt;       // weight rows (or G), U (or the second segment's rows), token codes
    const void* x;                 // fused: activations
    int32_t* c;
    void* y;
    const float* xs;               // [M] token scales (not fused)
    const float* ws[2];            // [N] channel scales
    const void* bias[2];
    void* y2;                      // I8_DIGIT: rows from split_row on, seg_rows of each part (NULL: all to y)
    int64_t ldx, ldc, ldy, K, split_row, seg_rows;
    int32_t M, N, tm, k_steps, seg_steps, splits, stages, codes_bytes, tmem_cols;
    int32_t y_dtype, bias_dtype, act, vec_c, vec_y;
    int32_t dependent;             // launched while the kernel before it still runs: 1: it writes the tokens, 2: weights too
    uint64_t stall_ns;             // test knob (ima_set_gemm_wait_test); 0 in normal use
};

IMA_DEVINL uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
IMA_DEVINL void st_cluster_u32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
IMA_DEVINL void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
IMA_DEVINL void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Four consecutive outputs of one row in y's type (all valid and aligned: one store).
IMA_DEVINL void store_quad(void* y, int dtype, int64_t off, const float (&v)[4], int valid, bool vec) {
    if (dtype == IMA_DTYPE_F32) {
        float* p = reinterpret_cast<float*>(y) + off;
        if (vec && valid >= 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else
            for (int e = 0; e < valid && e < 4; ++e) p[e] = v[e];
    } else {
        uint16_t* p = reinterpret_cast<uint16_t*>(y) + off;
        const uint32_t w[2] = {pack_half2(v[0], v[1], dtype), pack_half2(v[2], v[3], dtype)};
        if (vec && valid >= 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else
            for (int e = 0; e < valid && e < 4; ++e) p[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
    }
}

IMA_DEVINL float gated_value(int form, float g, float u) {
    float h;
    with_form(form, [&](auto tag) { h = act_value<decltype(tag)::value>(g) * u; });
    return h;
}

// EPI: I8_LINEAR, I8_GATED or I8_DIGIT; P digit planes (1 otherwise); DT: type of the activations when
// the quantiser is fused, -1 when the tokens come as codes.
template <int EPI, int P, int DT>
__global__ void __launch_bounds__(SK_THREADS, 2) int8_skinny_kernel(const __grid_constant__ SkParams p) {
    constexpr bool FUSED = DT >= 0;
    constexpr int OPS = EPI == I8_GATED ? 2 : 1;
    constexpr int XT = FUSED ? DT : IMA_DTYPE_F32;
    constexpr int BATCH = sk_batch(XT);
    extern __shared__ unsigned char sk_raw[];
    __shared__ uint64_t full[SK_MAX_STAGES], empty[SK_MAX_STAGES], tok_ready, acc_full, drained;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    __shared__ uint32_t s_amax[FUSED ? 8 * SK_MAX_TM : 1];      // [source CTA][token] maxima, as bits
    __shared__ float s_scale[SK_MAX_TM];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(sk_raw) + 1023) & ~(uintptr_t)1023);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = p.splits;
    const uint32_t rank = S > 1 ? cluster_ctarank() : 0;
    const int32_t m0 = blockIdx.y * p.tm;
    const int rows = min(p.tm, p.M - m0);                       // tokens of this tile
    const int32_t n0 = (int32_t)(blockIdx.x / S) * SK_ROWS;
    const int s0 = (int)((int64_t)rank * p.k_steps / S), s1 = (int)((int64_t)(rank + 1) * p.k_steps / S);
    const int steps = s1 - s0;
    const int tok_bytes = P * p.tm * I8_KT;                     // tokens of one k-step
    constexpr int W_BYTES = SK_ROWS * I8_KT;
    const int stage_bytes = OPS * W_BYTES + (FUSED ? 0 : tok_bytes);
    unsigned char* codes = smem;                                // fused: [k-step][token][128], swizzled
    unsigned char* tiles = smem + p.codes_bytes;
    int32_t* part = reinterpret_cast<int32_t*>(tiles + p.stages * stage_bytes);   // [S][OPS][P][tm][128 / S]

    auto load_weights = [&](int i) {   // i-th k-step of this CTA
        const int st = i % p.stages, ks = s0 + i;
        unsigned char* sb = tiles + st * stage_bytes;
        mbar_arrive_expect_tx(&full[st], (uint32_t)stage_bytes);
        if (EPI == I8_DIGIT && ks >= p.seg_steps) tma_load_2d(sb, &p.mw2, &full[st], (ks - p.seg_steps) * I8_KT, n0);
        else tma_load_2d(sb, &p.mw, &full[st], ks * I8_KT, n0);
        if (EPI == I8_GATED) tma_load_2d(sb + W_BYTES, &p.mw2, &full[st], ks * I8_KT, n0);
    };
    const int first = min(steps, p.stages);
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&tok_ready, SK_WORKERS);
        mbar_init(&acc_full, 1);
        mbar_init(&drained, 1);
        abort_flag = 0;
        mbar_fence_init();
        if (p.dependent == 2) wait_previous_kernel();   // the weights come from there too
        for (int i = 0; i < first; ++i) load_weights(i);        // on their way before anything else is set up
    }
    if (FUSED)
        for (int i = threadIdx.x; i < 8 * SK_MAX_TM; i += SK_THREADS) s_amax[i] = 0;
    if (warp == 1) {
        tmem_alloc(&tmem_slot, (uint32_t)p.tmem_cols);
        tmem_relinquish();
    }
    __syncthreads();
    if (S > 1) cluster_arrive();                                // barrier A: every CTA of the cluster runs
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    auto load_tokens = [&](int i) {
        const int st = i % p.stages;
        unsigned char* sb = tiles + st * stage_bytes + OPS * W_BYTES;
#pragma unroll
        for (int d = 0; d < P; ++d) tma_load_3d(sb + d * p.tm * I8_KT, &p.mt, &full[st], (s0 + i) * I8_KT, m0, d);
    };

    // ---- phase 1: row maxima of this CTA's slice ----
    const int64_t kbeg = (int64_t)s0 * I8_KT, kend = min(p.K, (int64_t)s1 * I8_KT);
    // units of 256 elements of a token's slice, dealt to the warps in turn, at most BATCH each (sk_plan): loaded
    // once, kept until the scales are known
    const int per_tok = FUSED ? max(1, (int)((kend - kbeg + 255) / 256)) : 1;
    const int units = FUSED && kend > kbeg ? rows * per_tok : 0;
    Raw8<XT> batch[FUSED ? BATCH : 1];
    auto load_batch = [&](int u0) {
#pragma unroll
        for (int i = 0; i < (FUSED ? BATCH : 0); ++i) {
            const int u = u0 + i * SK_WORKERS;
            batch[i].clear();
            if (u < units) {
                const int t = u / per_tok;
                const int64_t k = kbeg + (int64_t)(u - t * per_tok) * 256 + lane * 8;
                const unsigned char* row =
                    reinterpret_cast<const unsigned char*>(p.x) + (int64_t)(m0 + t) * p.ldx * dtype_bytes(XT);
                if ((reinterpret_cast<uintptr_t>(row) & 15) == 0 && k + 8 <= kend) batch[i].load_whole(row, k);
                else if (k < kend) batch[i].load(row, k, kend, false);
            }
        }
    };
    if (warp == 0 && lane == 0) {
        if (!FUSED) {
            if (p.dependent) wait_previous_kernel();
            for (int i = 0; i < first; ++i) load_tokens(i);
        }
    } else if (FUSED && warp >= 2) {
        load_batch(warp - 2);
#pragma unroll
        for (int i = 0; i < (FUSED ? BATCH : 0); ++i) {
            const int u = warp - 2 + i * SK_WORKERS;
            if (u >= units) break;
            const uint32_t mx = __reduce_max_sync(0xFFFFFFFFu, batch[i].max_bits());
            if (lane == 0) atomicMax(&s_amax[rank * SK_MAX_TM + u / per_tok], mx);
        }
    }
    if (S > 1) {
        __syncwarp();
        cluster_wait();                                         // A
        if (FUSED) {
            __syncthreads();
            for (int i = threadIdx.x; i < rows * S; i += SK_THREADS) {
                const int t = i % rows, r = i / rows;
                if (r != (int)rank)
                    st_cluster_u32(cluster_addr(smem_u32(&s_amax[rank * SK_MAX_TM + t]), (uint32_t)r),
                                   s_amax[rank * SK_MAX_TM + t]);
            }
            __syncwarp();
            cluster_arrive();                                   // B: the maxima are exchanged
            cluster_wait();
        }
    } else if (FUSED) {
        __syncthreads();
    }

    // ---- phase 2 ----
    if (warp == 0 && lane == 0) {
        int issued = first;
        for (; issued < steps; ++issued) {
            const int st = issued % p.stages;
            if (!mbar_wait_or_abort(&empty[st], (uint32_t)((issued / p.stages - 1) & 1), &abort_flag, IMA_WAIT_LIMIT_NS,
                                    IMA_WHERE_INT8_SKINNY, st))
                break;
            load_weights(issued);
            if (!FUSED) load_tokens(issued);
        }
        // every load issued lands before the CTA goes on, also after a give-up
        for (int i = max(0, issued - p.stages); i < issued; ++i)
            mbar_wait_bounded(&full[i % p.stages], (uint32_t)((i / p.stages) & 1), IMA_WHERE_INT8_SKINNY, 150);
    } else if (warp == 1 && lane == 0) {
        const uint32_t idesc = idesc_i8(SK_ROWS, P * p.tm);
        bool fed = !FUSED || mbar_wait_or_abort(&tok_ready, 0u, &abort_flag, IMA_WAIT_LIMIT_NS, IMA_WHERE_INT8_SKINNY, 50);
        if (p.stall_ns)   // test knob: a wait that nothing ends runs out
            fed = mbar_wait_or_abort(&drained, 0u, &abort_flag, p.stall_ns, IMA_WHERE_INT8_SKINNY, -2) && fed;
        for (int i = 0; fed && i < steps; ++i) {
            const int st = i % p.stages;
            fed = mbar_wait_or_abort(&full[st], (uint32_t)((i / p.stages) & 1), &abort_flag, IMA_WAIT_LIMIT_NS,
                                     IMA_WHERE_INT8_SKINNY, 100 + st);
            if (!fed) break;
            tc_fence_after();
            const uint32_t sw = smem_u32(tiles + st * stage_bytes);
            const uint32_t sx = FUSED ? smem_u32(codes + (int64_t)i * tok_bytes) : sw + OPS * W_BYTES;
#pragma unroll
            for (int ks = 0; ks < I8_KT / 32; ++ks)
#pragma unroll
                for (int o = 0; o < OPS; ++o)
                    mma_i8(tmem + (uint32_t)(o * P * p.tm), umma_desc_sw128_kmajor(sw + o * W_BYTES + ks * 32),
                           umma_desc_sw128_kmajor(sx + ks * 32), idesc, (i | ks) ? 1u : 0u);
            mma_commit(&empty[st]);
        }
        if (fed) mma_commit(&acc_full);
        // every MMA issued completes before the CTA goes on
        mma_commit(&drained);
        mbar_wait_bounded(&drained, 0u, IMA_WHERE_INT8_SKINNY, -3);
    } else if (warp >= 2) {
        if constexpr (FUSED) {
            // scales of all tokens, from the maxima of every CTA of the cluster
            for (int t = threadIdx.x - 64; t < rows; t += SK_WORKERS * 32) {
                uint32_t mx = 0;
                for (int r = 0; r < S; ++r) mx = max(mx, s_amax[r * SK_MAX_TM + t]);
                const float a = __uint_as_float(mx);
                s_scale[t] = i8_row_scale(a, a != a);
            }
            named_barrier_sync(1, SK_WORKERS * 32);
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int u = warp - 2 + i * SK_WORKERS;
                if (u >= units) break;
                const int t = u / per_tok;
                const int off = (u - t * per_tok) * 256 + lane * 8;     // element of the slice
                if (kbeg + off >= kend) continue;
                const float s = s_scale[t];
                float v[8];
                batch[i].unpack(v);
                // k-step off / 128, token t, 16-byte piece (off % 128) / 16 at its swizzled place
                unsigned char* dst = codes + (off >> 7) * tok_bytes + t * I8_KT +
                                     ((((off >> 4) & 7) ^ (t & 7)) << 4) + (off & 8);
                *reinterpret_cast<uint2*>(dst) = i8_codes8<XT>(v, s, i8_inv(s));
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tok_ready);
        }
        if (!FUSED) {   // the token scales
            if (p.dependent) wait_previous_kernel();
            for (int t = threadIdx.x - 64; t < rows; t += SK_WORKERS * 32) s_scale[t] = p.xs ? p.xs[m0 + t] : 0.0f;
            named_barrier_sync(1, SK_WORKERS * 32);
        }
        // scales and biases while the products run: of the lane's weight row (one CTA), or of the four
        // columns that the thread will own (a cluster).  Plain loads: the kernel before this one may have written the
        // scales since this one started.  No bias is -0, which changes no sum.
        const int q = warp & 3, hw = (warp - 2) >> 2, wt = threadIdx.x - 64;
        const int own = SK_ROWS / S, per = own / 4, j4 = (wt % per) * 4;
        const int32_t nq = S > 1 ? n0 + (int32_t)rank * own + j4 : n0 + q * 32 + lane;
        const int valid = max(0, min(S > 1 ? 4 : 1, p.N - nq));
        float ws[OPS][4], bias[OPS][4];
#pragma unroll
        for (int o = 0; o < OPS; ++o)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                ws[o][e] = EPI != I8_DIGIT && p.y && e < valid ? p.ws[o][nq + e] : 0.0f;
                bias[o][e] = EPI != I8_DIGIT && p.bias[o] && e < valid ? load_as_f32(p.bias[o], p.bias_dtype, nq + e) : -0.0f;
            }
        // the value of one output from its exact sums: a[plane], or a[0] of the operand(s)
        auto value = [&](const int32_t (&a)[P], int32_t b, float xs, int e) {
            if constexpr (EPI == I8_DIGIT) {
                int64_t sum = 0;
#pragma unroll
                for (int d = 0; d < P; ++d) sum += (int64_t)a[d] << (8 * d);
                return __fmul_rn(__ll2float_rn(sum), xs);
            } else {
                float v = __fmul_rn(__fmul_rn(__int2float_rn(a[0]), xs), ws[0][e]);
                if (EPI == I8_GATED) {
                    const float u = __fmul_rn(__fmul_rn(__int2float_rn(b), xs), ws[OPS - 1][e]);
                    return gated_value(p.act, __fadd_rn(v, bias[0][e]), __fadd_rn(u, bias[OPS - 1][e]));
                }
                return __fadd_rn(v, bias[0][e]);
            }
        };
        // row of y that token t of the tile goes to (false: none)
        auto place = [&](int t, void*& y, int64_t& m) {
            y = p.y;
            m = m0 + t;
            if (EPI == I8_DIGIT && p.y2) {
                if (m >= p.split_row) { m -= p.split_row; y = p.y2; }
                return m < p.seg_rows;
            }
            return true;
        };
        const bool ok = mbar_wait_or_abort(&acc_full, 0u, &abort_flag, IMA_WAIT_LIMIT_NS, IMA_WHERE_INT8_SKINNY, 200);
        __syncwarp();
        const bool all_ok = __all_sync(0xFFFFFFFFu, ok);
        tc_fence_after();
        const uint32_t tq = tmem + ((uint32_t)(q * 32) << 16);   // TMEM lane = weight row, column = (operand, plane, token)
        if (all_ok && S == 1) {
            // straight from tensor memory: a warp stores 32 consecutive outputs of a token
            for (int c0 = hw * 8; c0 < rows; c0 += 16) {
                uint32_t r[OPS * P][8];
#pragma unroll
                for (int o = 0; o < OPS * P; ++o) tmem_ld8(tq + (uint32_t)(o * p.tm + c0), r[o]);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    void* y;
                    int64_t m;
                    if (c0 + i >= rows || valid == 0 || !place(c0 + i, y, m)) continue;
                    int32_t a[P];
#pragma unroll
                    for (int d = 0; d < P; ++d) a[d] = steps > 0 ? (int32_t)r[d][i] : 0;
                    const int32_t b = steps > 0 ? (int32_t)r[OPS * P - 1][i] : 0;
                    if (EPI == I8_LINEAR && p.c) p.c[m * p.ldc + nq] = a[0];
                    if (!p.y) continue;
                    const float v = value(a, b, s_scale[c0 + i], 0);
                    const int64_t at = m * p.ldy + nq;
                    if (p.y_dtype == IMA_DTYPE_F32) reinterpret_cast<float*>(y)[at] = v;
                    else if (p.y_dtype == IMA_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
                    else reinterpret_cast<__half*>(y)[at] = __float2half_rn(v);
                }
            }
        } else if (all_ok) {
            // push the partial sums to the owners
            const int n = q * 32 + lane;
            const uint32_t base = cluster_addr(smem_u32(part), (uint32_t)(n / own));
            for (int c0 = hw * 8; c0 < OPS * P * p.tm; c0 += 16) {
                if (c0 % p.tm >= rows) continue;                // tokens beyond the last one
                uint32_t r[8];
                tmem_ld8(tq + (uint32_t)c0, r);
                tmem_wait_ld();
                const uint32_t at = base + (uint32_t)((((int)rank * OPS * P * p.tm + c0) * own + n % own) * 4);
#pragma unroll
                for (int j = 0; j < 8; ++j) st_cluster_u32(at + (uint32_t)(j * own * 4), steps > 0 ? r[j] : 0u);
            }
        }
        tc_fence_before();
        if (S > 1) {
            __syncwarp();
            cluster_arrive();                                   // C: all partial sums are with their owners
            cluster_wait();
            // the outputs this CTA owns: a thread keeps its four columns and walks the tokens
            if (all_ok && valid > 0) {
                auto gather = [&](int col) {   // sum over the cluster of 4 partial sums of one column
                    int4 a = make_int4(0, 0, 0, 0);
                    for (int r = 0; r < S; ++r) {
                        const int4 b = *reinterpret_cast<const int4*>(part + (r * OPS * P * p.tm + col) * own + j4);
                        a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
                    }
                    return a;
                };
#pragma unroll 2
                for (int t = wt / per; t < rows; t += 256 / per) {
                    void* y;
                    int64_t m;
                    if (!place(t, y, m)) continue;
                    int4 a[P], b = make_int4(0, 0, 0, 0);
#pragma unroll
                    for (int d = 0; d < P; ++d) a[d] = gather(d * p.tm + t);
                    if (EPI == I8_GATED) b = gather(p.tm + t);
                    if (EPI == I8_LINEAR && p.c) {
                        int32_t* dst = p.c + m * p.ldc + nq;
                        if (p.vec_c && valid == 4) *reinterpret_cast<int4*>(dst) = a[0];
                        else {
                            const int32_t av[4] = {a[0].x, a[0].y, a[0].z, a[0].w};
                            for (int e = 0; e < valid; ++e) dst[e] = av[e];
                        }
                    }
                    if (!p.y) continue;
                    float v[4];
                    const float xs = s_scale[t];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        int32_t ae[P];
#pragma unroll
                        for (int d = 0; d < P; ++d) ae[d] = e == 0 ? a[d].x : e == 1 ? a[d].y : e == 2 ? a[d].z : a[d].w;
                        v[e] = value(ae, e == 0 ? b.x : e == 1 ? b.y : e == 2 ? b.z : b.w, xs, e);
                    }
                    store_quad(y, p.y_dtype, m * p.ldy + nq, v, valid, p.vec_y);
                }
            }
        }
    }
    if (S > 1 && warp < 2) {
        __syncwarp();
        cluster_arrive();                                       // C, of the two warps without outputs
        cluster_wait();
    }
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, (uint32_t)p.tmem_cols);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct SkPlan {
    int tm, m_tiles, n_tiles, k_steps, splits, stages, codes_bytes, smem;
    bool ok;
    double ns;   // estimate
};

// The split form of a product of M tokens by N outputs over k_steps k-steps: tokens per tile, split and
// stages with the shortest estimate, which follows measurements.  A CTA streams its weights at 45 bytes/ns
// whatever its stages beyond three (a kernel that only loads 68 MB with one CTA per SM takes 15.0 us), token codes,
// which other CTAs read too, at 100 from L2, and the machine 5500; so two CTAs of four stages per SM beat one of
// eight (3584 x 18944 with 16 tokens: 18.9 us with 224 CTAs, 24.6 with 112).  A round of CTAs takes 5 us from launch to
// exit besides, the epilogue of the outputs that a CTA keeps 16 ns per token column (32 of two that share an SM), the
// exchange in a cluster 4 ns per column and 1 us.
// The fused quantiser (x_dtype >= 0) takes what its workers hold in registers at once: another pass over the
// activations costs 6 us (64 tokens, K = 3584), more than the row quantiser and its launch.
SkPlan sk_plan(int64_t M, int64_t N, int64_t k_steps, int planes, int ops, int x_dtype) {
    const bool fused = x_dtype >= 0;
    const int max_tm = planes == 3 ? 32 : (planes == 2 || ops == 2 ? 64 : SK_MAX_TM);
    SkPlan best = {};
    const int64_t m_tiles = (M + max_tm - 1) / max_tm, n_tiles = (N + SK_ROWS - 1) / SK_ROWS;
    const int64_t tm = ((M + m_tiles - 1) / m_tiles + 15) / 16 * 16;
    if (m_tiles > 65535 || (fused && m_tiles > 1)) return best;
    for (int s = 1; s <= 8 && s <= std::max<int64_t>(k_steps, 1); s *= 2) {
        SkPlan q = {};
        const int64_t steps = (k_steps + s - 1) / s;
        if (fused && M * ((steps * I8_KT + 255) / 256) > SK_WORKERS * sk_batch(x_dtype)) continue;
        const int64_t tok = (int64_t)planes * tm * I8_KT;
        const int64_t codes = fused ? steps * tok : 0;
        const int64_t stage = (int64_t)ops * SK_ROWS * I8_KT + (fused ? 0 : tok);
        const int64_t partial = s > 1 ? (int64_t)ops * planes * tm * SK_ROWS * 4 : 0;
        const int64_t least = std::min<int64_t>(3, std::max<int64_t>(steps, 1));
        const int64_t fixed = 1024 + codes + partial;
        int64_t per_sm = 2, stages = std::min<int64_t>((SK_SMEM_HALF - fixed) / stage, 4);
        if (stages < least) {
            per_sm = 1;
            stages = std::min<int64_t>((SK_SMEM - fixed) / stage, SK_MAX_STAGES);
        }
        if (stages < least) continue;
        stages = std::min<int64_t>(stages, std::max<int64_t>(steps, 1));
        q.tm = (int)tm; q.m_tiles = (int)m_tiles; q.n_tiles = (int)n_tiles; q.k_steps = (int)k_steps;
        q.splits = s; q.stages = (int)stages; q.codes_bytes = (int)codes;
        q.smem = (int)(fixed + stages * stage);
        const int64_t ctas = m_tiles * n_tiles * s;
        // clusters of 8 leave some SMs out, and so do those of 4
        const int64_t room = std::max<int64_t>(1, gemm_grid_limit() * per_sm * (s == 8 ? 14 : s == 4 ? 15 : 16) / 16);
        const double rounds = (double)((ctas + room - 1) / room);
        const int64_t w_bytes = ops * SK_ROWS * I8_KT;
        const double stream = std::max(rounds * (double)steps * ((double)w_bytes / 45.0 + (double)(stage - w_bytes) / 100.0),
                                       (double)(N * k_steps * I8_KT * ops * m_tiles) / 5500.0);
        const double column = 4.0 + 16.0 * (double)per_sm / (double)s;
        q.ns = rounds * ((fused ? 6000.0 + 100.0 * (double)M : 5000.0) + column * (double)(ops * planes * tm)) + stream +
               (s > 1 ? 1000.0 : 0.0);
        q.ok = true;
        if (!best.ok || q.ns < best.ns) best = q;
    }
    return best;
}

template <int EPI, int P, int DT>
int launch_skinny(SkParams& p, const SkPlan& q, cudaStream_t stream) {
    auto kern = int8_skinny_kernel<EPI, P, DT>;
    static std::atomic<uint64_t> ready{0};
    const int rc = set_smem_once(ready, (const void*)kern, SK_SMEM);
    if (rc != IMA_OK) return rc;
    p.tm = q.tm;
    p.k_steps = q.k_steps;
    p.splits = q.splits;
    p.stages = q.stages;
    p.codes_bytes = q.codes_bytes;
    p.stall_ns = g_gemm_stall_ns;
    p.tmem_cols = 32;
    while (p.tmem_cols < (EPI == I8_GATED ? 2 : 1) * P * q.tm) p.tmem_cols *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(q.splits * q.n_tiles), (unsigned)q.m_tiles);
    cfg.blockDim = dim3(SK_THREADS);
    cfg.dynamicSmemBytes = (size_t)q.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (q.splits > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)q.splits;
        attr[n].val.clusterDim.y = 1;
        attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (p.dependent) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = (unsigned)n;
    return ima_note_cuda(cudaLaunchKernelEx(&cfg, kern, p));
}

// Weight maps of the split form: o.b (and o.b2) in boxes of a tile's rows.
int sk_weight_maps(SkParams& p, const I8Operands& o) {
    if (o.K == 0) return IMA_OK;
    int rc = make_i8_map(&p.mw, o.b, o.K, o.ldb, p.N, 1, 0, SK_ROWS);
    if (rc == IMA_OK && o.b2) rc = make_i8_map(&p.mw2, o.b2, o.K, o.ldb2, p.N, 1, 0, SK_ROWS);
    return rc;
}

// Codes (or digit planes) in, split form.
template <int EPI, int P>
int run_skinny_codes(const I8Params& g, const I8Operands& o, const SkPlan& q, cudaStream_t stream) {
    SkParams p;
    memset(&p, 0, sizeof(p));
    p.c = g.c; p.y = g.y; p.xs = g.xs; p.ws[0] = g.ws[0]; p.ws[1] = g.ws[1]; p.bias[0] = g.bias[0]; p.bias[1] = g.bias[1];
    p.y2 = g.y2; p.split_row = g.split_row; p.seg_rows = g.seg_rows;
    p.ldc = g.ldc; p.ldy = g.ldy; p.M = g.M; p.N = g.N; p.K = o.K; p.y_dtype = g.y_dtype; p.bias_dtype = g.bias_dtype;
    p.act = g.act; p.vec_c = g.c_width == 16; p.vec_y = g.y_width >= 4 * dtype_bytes(g.y_dtype); p.dependent = g.dependent;
    p.seg_steps = g.seg_tiles;
    int rc = sk_weight_maps(p, o);
    if (rc == IMA_OK && o.K > 0) rc = make_i8_map(&p.mt, o.a, o.Ka, o.lda, p.M, P, o.a_planes, q.tm);
    if (rc != IMA_OK) return rc;
    return launch_skinny<EPI, P, -1>(p, q, stream);
}

}  // namespace
