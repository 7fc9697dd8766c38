// 8-bit integer products of few tokens: the weight is streamed once, and the contraction is split
// over a cluster of CTAs.
//
// Roles of the operands are the other way round than in int8_gemm.cu: a tile is 128 weight rows
// (the M side of the MMA) by TM tokens (its N side, 16 .. 128), so a single token costs one 16-column
// MMA and the work is the weight's bytes.  The gated form puts 64 rows of G and 64 rows of U into
// the 128; the digit form stacks the P planes of the tokens, P * TM columns.
//
// Split: the k-steps of a tile are dealt to the S <= 8 CTAs of a cluster, S chosen so that about two
// CTAs per SM are in flight.  Each CTA leaves its int32 partial sums in its shared memory; after
// a cluster barrier every CTA adds a share of the outputs from all of them (distributed shared
// memory) and applies the epilogue.  Integer sums do not depend on the order.
//
// Fused quantiser: with the activations still floating, the 8 worker warps find the row maxima of
// the CTA's k-slice (exchanged through the cluster), quantise the slice into the swizzled layout the
// MMA reads, and keep it in shared memory, while the first weight tiles are on their way.  This saves a
// launch and a round trip of the codes.
#include "sm100_primitives.cuh"

namespace {

constexpr int SK_ROWS = 128;                       // weight rows per tile
constexpr int SK_WORKERS = 8;
constexpr int SK_THREADS = 64 + SK_WORKERS * 32;
constexpr int SK_MAX_STAGES = 8;
constexpr int SK_SMEM = 112 * 1024;                // two CTAs per SM

struct __align__(64) SkParams {
    CUtensorMap mw, mw2, mt;       // weight rows (or G), U (or the second segment's rows), token codes
    const void* x;                 // fused: activations
    int32_t* c;
    void* y;
    const float* xs;               // [M] token scales (not fused)
    const float* ws[2];            // [N] channel scales
    const void* bias[2];
    int64_t ldx, ldc, ldy, K;
    int32_t M, N, tm, k_steps, seg_steps, splits, stages, codes_bytes, tmem_cols;
    int32_t y_dtype, bias_dtype, act, vec_c, vec_y, pad;
    uint64_t stall_ns;             // test knob (ima_set_gemm_wait_test); 0 in normal use
};

IMA_DEVINL uint4 ld_cluster_v4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
IMA_DEVINL uint32_t ld_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

// Four consecutive outputs of one row in y's type (n + 3 < N and aligned: one store).
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

IMA_DEVINL float gated_value(int act, float g, float u) {
    if (act == IMA_ACT_SILU) return act_value<IMA_ACT_SILU>(g) * u;
    if (act == IMA_ACT_GELU) return act_value<IMA_ACT_GELU>(g) * u;
    return act_value<IMA_ACT_GELU_TANH>(g) * u;
}

// EPI: I8_LINEAR, I8_GATED or I8_DIGIT; P digit planes (1 otherwise); DT: type of the activations when
// the quantiser is fused, -1 when the tokens come as codes.
template <int EPI, int P, int DT>
__global__ void __launch_bounds__(SK_THREADS, 2) int8_skinny_kernel(const __grid_constant__ SkParams p) {
    constexpr bool FUSED = DT >= 0;
    extern __shared__ unsigned char sk_raw[];
    __shared__ uint64_t full[SK_MAX_STAGES], empty[SK_MAX_STAGES], tok_ready, acc_full, drained;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    __shared__ uint32_t s_amax[SK_ROWS];
    __shared__ float s_scale[SK_ROWS];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(sk_raw) + 1023) & ~(uintptr_t)1023);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = p.splits;
    const uint32_t rank = S > 1 ? cluster_ctarank() : 0;
    const int nt = blockIdx.x / S;
    const int32_t m0 = blockIdx.y * p.tm;
    const int rows = min(p.tm, p.M - m0);                       // tokens of this tile
    constexpr int OUT = EPI == I8_GATED ? SK_ROWS / 2 : SK_ROWS;   // output columns of this tile
    const int32_t n0 = nt * OUT;
    const int s0 = (int)((int64_t)rank * p.k_steps / S), s1 = (int)((int64_t)(rank + 1) * p.k_steps / S);
    const int tok_bytes = P * p.tm * I8_KT;                     // tokens of one k-step
    const int w_bytes = SK_ROWS * I8_KT;
    const int stage_bytes = w_bytes + (FUSED ? 0 : tok_bytes);
    unsigned char* codes = smem;                                // fused: [k-step][token row][128], swizzled
    unsigned char* tiles = smem + p.codes_bytes;

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
    }
    if (FUSED && threadIdx.x >= 64 && threadIdx.x < 64 + SK_ROWS) s_amax[threadIdx.x - 64] = 0;
    if (warp == 1) {
        tmem_alloc(&tmem_slot, (uint32_t)p.tmem_cols);
        tmem_relinquish();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    auto load_step = [&](int i) {   // i-th k-step of this CTA into its stage
        const int st = i % p.stages, ks = s0 + i;
        unsigned char* sb = tiles + st * stage_bytes;
        mbar_arrive_expect_tx(&full[st], (uint32_t)stage_bytes);
        if (EPI == I8_GATED) {
            tma_load_2d(sb, &p.mw, &full[st], ks * I8_KT, n0);
            tma_load_2d(sb + w_bytes / 2, &p.mw2, &full[st], ks * I8_KT, n0);
        } else if (EPI == I8_DIGIT && ks >= p.seg_steps) {
            tma_load_2d(sb, &p.mw2, &full[st], (ks - p.seg_steps) * I8_KT, n0);
        } else {
            tma_load_2d(sb, &p.mw, &full[st], ks * I8_KT, n0);
        }
        if (!FUSED) {
#pragma unroll
            for (int i2 = 0; i2 < P; ++i2)
                tma_load_3d(sb + w_bytes + i2 * p.tm * I8_KT, &p.mt, &full[st], ks * I8_KT, m0, i2);
        }
    };

    // ---- phase 1: first weight tiles on their way; row maxima of this CTA's slice ----
    const int steps = s1 - s0;
    const int first = min(steps, p.stages);
    const int64_t kbeg = (int64_t)s0 * I8_KT, kend = min(p.K, (int64_t)s1 * I8_KT);
    const int blocks = FUSED ? (int)((kend - kbeg + 255) / 256) : 0;   // 256-element pieces of a row
    if (warp == 0 && lane == 0) {
        for (int i = 0; i < first; ++i) load_step(i);
    } else if (FUSED && warp >= 2) {
        constexpr int U = 4;
        const int units = rows * blocks;
        for (int u0 = warp - 2; u0 < units; u0 += SK_WORKERS * U) {
            Raw8<FUSED ? DT : 0> r[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int u = u0 + i * SK_WORKERS;
                const int t = min(u / blocks, rows - 1);
                const int64_t k = u < units ? kbeg + (int64_t)(u % blocks) * 256 + lane * 8 : kend;
                const unsigned char* row = reinterpret_cast<const unsigned char*>(p.x) + (int64_t)(m0 + t) * p.ldx * dtype_bytes(DT);
                r[i].load(row, k, kend, (reinterpret_cast<uintptr_t>(row) & 15) == 0);
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int u = u0 + i * SK_WORKERS;
                if (u >= units) break;
                const uint32_t mx = __reduce_max_sync(0xFFFFFFFFu, r[i].max_bits());
                if (lane == 0) atomicMax(&s_amax[u / blocks], mx);
            }
        }
    }
    if (FUSED) {
        __syncwarp();
        if (S > 1) cluster_sync_all();
        else __syncthreads();
    }

    // ---- phase 2 ----
    if (warp == 0 && lane == 0) {
        int issued = first;
        for (; issued < steps; ++issued) {
            const int st = issued % p.stages;
            if (!mbar_wait_or_abort(&empty[st], (uint32_t)((issued / p.stages - 1) & 1), &abort_flag, IMA_WAIT_LIMIT_NS,
                                    IMA_WHERE_INT8_SKINNY, st))
                break;
            load_step(issued);
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
            const uint32_t sx = FUSED ? smem_u32(codes + (int64_t)i * tok_bytes) : sw + w_bytes;
#pragma unroll
            for (int ks = 0; ks < I8_KT / 32; ++ks)
                mma_i8(tmem, umma_desc_sw128_kmajor(sw + ks * 32), umma_desc_sw128_kmajor(sx + ks * 32), idesc,
                       (i | ks) ? 1u : 0u);
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
                uint32_t mx = s_amax[t];
                for (int r = 0; r < S; ++r)
                    if (S > 1) mx = max(mx, ld_cluster_u32(cluster_map(&s_amax[t], (uint32_t)r)));
                const float a = __uint_as_float(mx);
                s_scale[t] = i8_row_scale(a, a != a);
            }
            named_barrier_sync(1, SK_WORKERS * 32);
            const int units = rows * blocks;
            constexpr int U = 4;
            for (int u0 = warp - 2; u0 < units; u0 += SK_WORKERS * U) {
                Raw8<FUSED ? DT : 0> r[U];
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int u = u0 + i * SK_WORKERS;
                    const int t = min(u / blocks, rows - 1);
                    const int64_t k = u < units ? kbeg + (int64_t)(u % blocks) * 256 + lane * 8 : kend;
                    const unsigned char* row = reinterpret_cast<const unsigned char*>(p.x) + (int64_t)(m0 + t) * p.ldx * dtype_bytes(DT);
                    r[i].load(row, k, kend, (reinterpret_cast<uintptr_t>(row) & 15) == 0);
                }
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int u = u0 + i * SK_WORKERS;
                    if (u >= units) break;
                    const int t = u / blocks;
                    const int off = (u % blocks) * 256 + lane * 8;      // element of the slice
                    if (kbeg + off >= kend) continue;
                    float v[8];
                    r[i].unpack(v);
                    const float s = s_scale[t];
                    // k-step off / 128, token row t, 16-byte piece (off % 128) / 16 at its swizzled place
                    unsigned char* dst = codes + (int64_t)(off >> 7) * tok_bytes + t * I8_KT +
                                         ((((off >> 4) & 7) ^ (t & 7)) << 4) + (off & 8);
                    *reinterpret_cast<uint2*>(dst) = i8_codes8(v, s, __frcp_rn(s));
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tok_ready);
        }
        // partial sums: TMEM lane = weight row, column = token (plane after plane)
        const bool ok = mbar_wait_or_abort(&acc_full, 0u, &abort_flag, IMA_WAIT_LIMIT_NS, IMA_WHERE_INT8_SKINNY, 200);
        __syncwarp();
        const bool all_ok = __all_sync(0xFFFFFFFFu, ok);
        tc_fence_after();
        int32_t* part = reinterpret_cast<int32_t*>(smem);       // [P * tm][128], over the tiles and codes
        const int q = warp & 3, hw = (warp - 2) >> 2;
        if (all_ok) {
            for (int c0 = hw * 8; c0 < P * p.tm; c0 += 16) {
                uint32_t r[8];
                tmem_ld8(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c0, r);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 8; ++j) part[(c0 + j) * SK_ROWS + q * 32 + lane] = steps > 0 ? (int32_t)r[j] : 0;
            }
        }
        tc_fence_before();
    }
    __syncwarp();
    if (S > 1) cluster_sync_all();
    else __syncthreads();

    // ---- phase 3: this CTA's share of the outputs, four consecutive columns at a time ----
    if (!abort_flag) {
        const int quads = rows * (OUT / 4);
        const uint32_t part_addr = smem_u32(smem);
        for (int i = (int)rank * SK_THREADS + threadIdx.x; i < quads; i += S * SK_THREADS) {
            const int t = i / (OUT / 4), j = (i % (OUT / 4)) * 4;
            const int32_t n = n0 + j;
            if (n >= p.N) continue;
            const int valid = min(4, p.N - n);
            const int64_t m = m0 + t;
            auto gather = [&](int col, int at) {   // sum over the cluster of 4 partials of one column
                uint4 a = make_uint4(0, 0, 0, 0);
                const uint32_t off = (uint32_t)((col * SK_ROWS + at) * 4);
                for (int r = 0; r < S; ++r) {
                    uint4 b;
                    if (S > 1) {
                        uint32_t base;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(base) : "r"(part_addr), "r"(r));
                        b = ld_cluster_v4(base + off);
                    } else {
                        b = *reinterpret_cast<const uint4*>(smem + off);
                    }
                    a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
                }
                return a;
            };
            float v[4];
            if constexpr (EPI == I8_DIGIT) {
                int64_t s[4] = {0, 0, 0, 0};
#pragma unroll
                for (int d = 0; d < P; ++d) {
                    const uint4 a = gather(d * p.tm + t, j);
                    s[0] += (int64_t)(int32_t)a.x << (8 * d);
                    s[1] += (int64_t)(int32_t)a.y << (8 * d);
                    s[2] += (int64_t)(int32_t)a.z << (8 * d);
                    s[3] += (int64_t)(int32_t)a.w << (8 * d);
                }
                const float xs = p.xs[m];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __fmul_rn(__ll2float_rn(s[e]), xs);
            } else {
                const float xs = FUSED ? s_scale[t] : (p.xs ? p.xs[m] : 0.0f);
                const uint4 a = gather(t, j);
                const int32_t av[4] = {(int32_t)a.x, (int32_t)a.y, (int32_t)a.z, (int32_t)a.w};
                if constexpr (EPI == I8_GATED) {
                    const uint4 b = gather(t, OUT + j);
                    const int32_t bv[4] = {(int32_t)b.x, (int32_t)b.y, (int32_t)b.z, (int32_t)b.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[e] = 0.0f;
                        if (e >= valid) continue;
                        const float gb = p.bias[0] ? load_as_f32(p.bias[0], p.bias_dtype, n + e) : 0.0f;
                        const float ub = p.bias[1] ? load_as_f32(p.bias[1], p.bias_dtype, n + e) : 0.0f;
                        const float g = __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(av[e]), xs), p.ws[0][n + e]), gb);
                        const float u = __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(bv[e]), xs), p.ws[1][n + e]), ub);
                        v[e] = gated_value(p.act, g, u);
                    }
                } else {
                    if (p.c) {
                        int32_t* dst = p.c + m * p.ldc + n;
                        if (p.vec_c && valid == 4) *reinterpret_cast<uint4*>(dst) = a;
                        else
                            for (int e = 0; e < valid; ++e) dst[e] = av[e];
                    }
                    if (!p.y) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[e] = 0.0f;
                        if (e >= valid) continue;
                        v[e] = __fmul_rn(__fmul_rn(__int2float_rn(av[e]), xs), p.ws[0][n + e]);
                        if (p.bias[0]) v[e] = __fadd_rn(v[e], load_as_f32(p.bias[0], p.bias_dtype, n + e));
                    }
                }
            }
            store_quad(p.y, p.y_dtype, m * p.ldy + n, v, valid, p.vec_y);
        }
    }
    // no CTA leaves while another still reads its partial sums
    __syncwarp();
    if (S > 1) cluster_sync_all();
    else __syncthreads();
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
};

// Tokens per tile, split and stages for a product of M tokens by N outputs over k_steps k-steps.
// `max_tm`: most tokens a tile may have.  Splits: about two CTAs per SM, at least one k-step each.
SkPlan sk_plan(int64_t M, int64_t N, int64_t k_steps, int planes, int out, int max_tm, bool fused) {
    SkPlan q = {};
    const int64_t tiles = (M + max_tm - 1) / max_tm;
    q.tm = (int)(((M + tiles - 1) / tiles + 15) / 16 * 16);
    q.m_tiles = (int)((M + q.tm - 1) / q.tm);
    q.n_tiles = (int)((N + out - 1) / out);
    q.k_steps = (int)k_steps;
    const int64_t all = (int64_t)q.m_tiles * q.n_tiles;
    int64_t s = 2 * (int64_t)gemm_grid_limit() / std::max<int64_t>(all, 1);
    s = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(s, 8), k_steps));
    q.splits = (int)s;
    const int64_t steps = (k_steps + s - 1) / s;
    const int64_t tok = (int64_t)planes * q.tm * I8_KT;
    const int64_t codes = fused ? steps * tok : 0;
    const int64_t stage = SK_ROWS * I8_KT + (fused ? 0 : tok);
    const int64_t partial = (int64_t)planes * q.tm * SK_ROWS * 4;
    const int64_t room = SK_SMEM - 1024 - 2048;
    int64_t stages = std::min<int64_t>((room - codes) / stage, SK_MAX_STAGES);
    stages = std::min<int64_t>(stages, std::max<int64_t>(steps, 1));
    q.codes_bytes = (int)codes;
    q.ok = stages >= std::min<int64_t>(2, std::max<int64_t>(steps, 1)) && partial <= room && q.m_tiles <= 65535;
    q.stages = (int)std::max<int64_t>(stages, 1);
    q.smem = (int)(std::max<int64_t>(codes + q.stages * stage, partial) + 1024);
    return q;
}

template <int EPI, int P, int DT>
int launch_skinny(SkParams& p, const SkPlan& q, cudaStream_t stream) {
    auto kern = int8_skinny_kernel<EPI, P, DT>;
    int rc = ima_note_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SK_SMEM));
    if (rc != IMA_OK) return rc;
    p.tm = q.tm;
    p.k_steps = q.k_steps;
    p.splits = q.splits;
    p.stages = q.stages;
    p.codes_bytes = q.codes_bytes;
    p.stall_ns = g_gemm_stall_ns;
    p.tmem_cols = 32;
    while (p.tmem_cols < P * q.tm) p.tmem_cols *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(q.splits * q.n_tiles), (unsigned)q.m_tiles);
    cfg.blockDim = dim3(SK_THREADS);
    cfg.dynamicSmemBytes = (size_t)q.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)q.splits;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = q.splits > 1 ? 1 : 0;
    return ima_note_cuda(cudaLaunchKernelEx(&cfg, kern, p));
}

// A product whose tiles would occupy at most half the machine in int8_gemm.cu is split here instead.
bool sk_wanted(int64_t M, int64_t N, int tile_n) {
    return ((M + I8_BM - 1) / I8_BM) * ((N + tile_n - 1) / tile_n) * 2 <= gemm_grid_limit();
}

// Weight maps of the split form: o.b (and o.b2) in boxes of a tile's rows.
int sk_weight_maps(SkParams& p, const I8Operands& o, int box) {
    if (o.K == 0) return IMA_OK;
    int rc = make_i8_map(&p.mw, o.b, o.K, o.ldb, p.N, 1, box, false);
    if (rc == IMA_OK && o.b2) rc = make_i8_map(&p.mw2, o.b2, o.K, o.ldb2, p.N, 1, box, false);
    return rc;
}

// Codes (or digit planes) in, split form.
template <int EPI, int P>
int run_skinny_codes(const I8Params& g, const I8Operands& o, const SkPlan& q, cudaStream_t stream) {
    SkParams p;
    memset(&p, 0, sizeof(p));
    p.c = g.c; p.y = g.y; p.xs = g.xs; p.ws[0] = g.ws[0]; p.ws[1] = g.ws[1]; p.bias[0] = g.bias[0]; p.bias[1] = g.bias[1];
    p.ldc = g.ldc; p.ldy = g.ldy; p.M = g.M; p.N = g.N; p.K = o.K; p.y_dtype = g.y_dtype; p.bias_dtype = g.bias_dtype;
    p.act = g.act; p.vec_c = g.vec_c; p.vec_y = g.vec_y;
    p.seg_steps = g.seg_tiles;
    int rc = sk_weight_maps(p, o, EPI == I8_GATED ? SK_ROWS / 2 : SK_ROWS);
    if (rc == IMA_OK && o.K > 0) rc = make_i8_map(&p.mt, o.a, o.Ka, o.lda, p.M, P, q.tm, true);
    if (rc != IMA_OK) return rc;
    return launch_skinny<EPI, P, -1>(p, q, stream);
}

}  // namespace
