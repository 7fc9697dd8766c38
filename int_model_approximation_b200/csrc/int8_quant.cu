// Memory-bound kernels of the 8-bit integer linears: the per-token / per-channel int8
// quantiser, the digit planes of gradients (by rows, and transposed by columns), the int8
// transpose and the column sums of bias gradients.
//
// Quantiser, one row:  s = max(RN32(amax_k |x_k| / 127), 1e-12),  q_k = rint(RN32(x_k / s)),
// both divisions IEEE, ties to even.  |q| <= 127 because RN32(amax / s) < 127.5.  A row with a
// NaN or an infinity has scale NaN or inf and codes 0, so that its products rescale to NaN.
//
// Gradient digits.  A gradient product has one integer factor (codes) and one real factor D.  D
// is written against its row maximum as v = rint(D / s), s = amax / V_P, in P balanced base-256
// digits, v = sum_p 256^p d_p with d_p in [-128, 127] (V_2 = 127 * 256 + 127, V_3 = 127 * 65536 +
// 127 * 256 + 127), so the product runs on the int8 tensor cores exactly.  The rounding is the
// one place where a gradient loses bits: half a step of amax / V_P, i.e. at most 2^-16 (P = 2, for
// bf16) or 2^-24 (P = 3, for fp16 and fp32) of the row's largest element.  Against the rms of
// the row's products that is at most sqrt(L / 3) 2^-16 for L summands, reached only when one
// element carries the whole row; 4e-5 for Gaussian rows, 6e-4 measured for columns of token
// gradients of very different sizes, where a bf16 result is off by 2e-3 and an fp16 one by 2e-4.
#include <algorithm>
#include "ima_common.cuh"

namespace {

// Reciprocals of a scale that bracket it: x * lo and x * hi lie on either side of RN32(x / s), which is off
// by at most 2^-24 of the quotient, as are the products.
struct I8Inv {
    float lo, hi;
};
IMA_DEVINL I8Inv i8_inv(float s) {
    const float inv = __frcp_rn(s);
    return {__fmul_rn(inv, 1.0f - 0x1p-21f), __fmul_rn(inv, 1.0f + 0x1p-21f)};
}

// Codes of eight elements, rint(RN32(x / s)) each, without a division per element: fma(x, inv, 1.5 *
// 2^23) holds rint(x * inv) in its low mantissa bits, and rounding is monotonic, so where both
// brackets round to the same integer the quotient does too.  Where they differ (a quotient within
// 2^-20 of itself of a half-integer, some 3 in 10^5) the division decides.  A scale that is NaN or
// inf gives codes 0.
IMA_DEVINL uint2 i8_codes8(const float (&v)[8], float s, I8Inv inv) {
    constexpr float kRound = 12582912.0f;
    uint32_t b[8], differ = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        b[j] = __float_as_uint(__fmaf_rn(v[j], inv.lo, kRound));
        differ |= b[j] ^ __float_as_uint(__fmaf_rn(v[j], inv.hi, kRound));
    }
    if (differ) {
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
            float x = v[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) x = j == e ? v[e] : x;
            if (__fmaf_rn(x, inv.lo, kRound) != __fmaf_rn(x, inv.hi, kRound)) {
                const uint32_t k = (uint32_t)__float2int_rn(__fdiv_rn(x, s));
#pragma unroll
                for (int e = 0; e < 8; ++e) b[e] = j == e ? k : b[e];
            }
        }
    }
    if (!(s <= 3.402823466e38f)) return make_uint2(0, 0);
    return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

IMA_DEVINL float i8_row_scale(float amax, bool nan) {
    if (nan) return __int_as_float(0x7FC00000);
    const float s = __fdiv_rn(amax, 127.0f);
    return s < 1e-12f ? 1e-12f : s;
}

IMA_DEVINL uint32_t pack4(const int32_t* v) {
    return __byte_perm(__byte_perm((uint32_t)v[0], (uint32_t)v[1], 0x0040),
                       __byte_perm((uint32_t)v[2], (uint32_t)v[3], 0x0040), 0x5410);
}

// Eight consecutive elements as loaded (16 bytes of a 16-bit type, 32 of fp32).  max_bits() is the fp32
// bit pattern of the largest magnitude: magnitudes order like their bit patterns, NaN above all.
template <int DT>
struct Raw8;
template <>
struct Raw8<IMA_DTYPE_F32> {
    float v[8];
    IMA_DEVINL void clear() {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    }
    IMA_DEVINL void load_whole(const void* row, int64_t k0) {
        const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + k0);
        const float4 a = __ldg(p), b = __ldg(p + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    IMA_DEVINL void load(const void* row, int64_t k0, int64_t K, bool vec) { load8(row, IMA_DTYPE_F32, k0, K, vec, v); }
    IMA_DEVINL void unpack(float (&o)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = v[j];
    }
    IMA_DEVINL uint32_t max_bits() const {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
        return m;
    }
};
template <bool BF16>
struct RawHalf8 {
    uint4 u;
    IMA_DEVINL void clear() { u = make_uint4(0, 0, 0, 0); }
    IMA_DEVINL void load_whole(const void* row, int64_t k0) {
        u = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(row) + k0));
    }
    IMA_DEVINL void load(const void* row, int64_t k0, int64_t K, bool vec) {
        u = qz_load_half8(reinterpret_cast<const uint16_t*>(row), k0, K, vec);
    }
    IMA_DEVINL void unpack(float (&o)[8]) const { qz_unpack_half8(u, BF16, o); }
    IMA_DEVINL uint32_t max_bits() const {
        uint32_t m = __vmaxu2(__vmaxu2(u.x & 0x7FFF7FFFu, u.y & 0x7FFF7FFFu),
                              __vmaxu2(u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu));
        m = max(m & 0xFFFFu, m >> 16);
        return BF16 ? m << 16 : __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
    }
};
template <>
struct Raw8<IMA_DTYPE_BF16> : RawHalf8<true> {};
template <>
struct Raw8<IMA_DTYPE_F16> : RawHalf8<false> {};

__host__ __device__ __forceinline__ int dtype_bytes(int dtype) { return dtype == IMA_DTYPE_F32 ? 4 : 2; }

// Maximum over the TPR threads of a row (TPR == 32, or the block).
template <int TPR>
IMA_DEVINL uint32_t row_max(uint32_t m, uint32_t* s_max) {
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    if (TPR > 32) {
        if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPR / 32; ++i) m = max(m, s_max[i]);
        __syncthreads();
    }
    return m;
}

// ---------------------------------------------------------------------------
// Row quantiser.  TPR threads take one row; a row of up to TPR * 8 * V elements is read once
// and kept in registers between the maximum and the codes, a longer one is read again (from
// L2).  Bound by memory: 2 or 4 bytes in and 1 out per element.
// ---------------------------------------------------------------------------
template <int DT, int TPR, int V>
__global__ void __launch_bounds__(256, 2) int8_quantize_rows_kernel(const void* x, int64_t M, int64_t K, int64_t ldx,
                                                                    int8_t* q, int64_t ldq, float* scale) {
    // a product launched to follow this kernel may start now; it waits for this kernel's end before it reads
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ uint32_t s_max[8];
    constexpr int ROWS = 256 / TPR;
    const int tid = threadIdx.x % TPR;
    for (int64_t m = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR; m < M; m += (int64_t)gridDim.x * ROWS) {
        const unsigned char* row = reinterpret_cast<const unsigned char*>(x) + m * ldx * dtype_bytes(DT);
        const bool vec = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
        // whole aligned groups of eight that this thread keeps; the rest is loaded twice
        const int64_t whole = vec ? min(K / 8 * 8, (int64_t)V * TPR * 8) : 0;
        Raw8<DT> keep[V];
        uint32_t mx = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            keep[i].clear();
            if ((i * TPR + tid) * 8 < whole) keep[i].load_whole(row, (int64_t)(i * TPR + tid) * 8);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) mx = max(mx, keep[i].max_bits());
#pragma unroll 1
        for (int64_t k0 = whole + tid * 8; k0 < K; k0 += TPR * 8) {
            Raw8<DT> r;
            r.load(row, k0, K, vec);
            mx = max(mx, r.max_bits());
        }
        const float amax = __uint_as_float(row_max<TPR>(mx, s_max));
        const float s = i8_row_scale(amax, amax != amax);
        const I8Inv inv = i8_inv(s);
        if (tid == 0) scale[m] = s;
        int8_t* qr = q + m * ldq;
        auto emit = [&](const Raw8<DT>& r, int64_t k0) {
            float v[8];
            r.unpack(v);
            *reinterpret_cast<uint2*>(qr + k0) = i8_codes8(v, s, inv);
        };
#pragma unroll
        for (int i = 0; i < V; ++i)
            if ((i * TPR + tid) * 8 < whole) emit(keep[i], (int64_t)(i * TPR + tid) * 8);
#pragma unroll 1
        for (int64_t k0 = whole + tid * 8; k0 < K; k0 += TPR * 8) {
            Raw8<DT> r;
            r.load(row, k0, K, vec);
            emit(r, k0);
        }
    }
}

// ---------------------------------------------------------------------------
// Digits
// ---------------------------------------------------------------------------
template <int P>
IMA_DEVINL float digit_limit() { return P == 2 ? 32639.0f : 8355711.0f; }

// Scale of a row (or column) with largest magnitude `amax`: never zero, so that a row of zeros has
// codes 0, and never so small that its reciprocal overflows.
template <int P>
IMA_DEVINL float digit_scale(float amax, bool nan) {
    if (nan) return __int_as_float(0x7FC00000);
    return fmaxf(__fdiv_rn(amax, digit_limit<P>()), 1.17549435e-38f);
}

// Balanced base-256 digits of rint(x * inv): |rint| <= V_P + 1 after rounding, clamped to V_P.
template <int P>
IMA_DEVINL void digits_of(float x, float inv, int32_t (&d)[P]) {
    const int32_t lim = P == 2 ? 32639 : 8355711;
    int32_t v = min(max(__float2int_rn(__fmul_rn(x, inv)), -lim), lim);
#pragma unroll
    for (int p = 0; p < P - 1; ++p) {
        d[p] = (int32_t)(int8_t)(v & 255);
        v = (v - d[p]) >> 8;
    }
    d[P - 1] = v;
}

// Row digits of D[m, j] = src[m, j] * col_scale[j].  The row is `segs` segments of `seg_len`
// columns, segment i starting at column i * seg_pitch of the source, of col_scale and of the
// planes; columns between segments are zero in the planes.
struct DigitRows {
    const void* src;
    const float* col_scale;   // NULL: 1
    int8_t* planes;           // plane p at planes + p * plane_stride
    float* row_scale;
    int64_t ld, M, seg_len, seg_pitch, ldp, plane_stride;
    int32_t segs, pad;
};

template <int DT, int P>
__global__ void __launch_bounds__(256) int8_digit_rows_kernel(const DigitRows a) {
    __shared__ uint32_t s_max[8];
    const int tid = threadIdx.x;
    for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
        const unsigned char* row = reinterpret_cast<const unsigned char*>(a.src) + m * a.ld * dtype_bytes(DT);
        float v[8];
        uint32_t mx = 0;
        auto scaled = [&](int sg, int64_t j0, float (&o)[8]) {
            const unsigned char* base = row + sg * a.seg_pitch * dtype_bytes(DT);
            Raw8<DT> r;
            r.load(base, j0, a.seg_len, (reinterpret_cast<uintptr_t>(base) & 15) == 0);
            r.unpack(o);
            if (a.col_scale) {
                const float* cs = a.col_scale + sg * a.seg_pitch;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j0 + j < a.seg_len) o[j] = __fmul_rn(o[j], __ldg(cs + j0 + j));
            }
        };
        for (int sg = 0; sg < a.segs; ++sg)
            for (int64_t j0 = (int64_t)tid * 8; j0 < a.seg_len; j0 += 2048) {
                scaled(sg, j0, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) mx = max(mx, __float_as_uint(v[j]) & 0x7FFFFFFFu);
            }
        const float amax = __uint_as_float(row_max<256>(mx, s_max));
        const float s = digit_scale<P>(amax, amax != amax);
        const float inv = __frcp_rn(s);
        if (tid == 0) a.row_scale[m] = s;
        for (int sg = 0; sg < a.segs; ++sg) {
            const int64_t width = sg + 1 < a.segs ? a.seg_pitch : a.ldp - sg * a.seg_pitch;
            for (int64_t j0 = (int64_t)tid * 8; j0 < width; j0 += 2048) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = 0.0f;
                if (j0 < a.seg_len) scaled(sg, j0, v);
                int32_t d[P][8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    int32_t t[P];
                    digits_of<P>(v[j], inv, t);
#pragma unroll
                    for (int p = 0; p < P; ++p) d[p][j] = t[p];
                }
#pragma unroll
                for (int p = 0; p < P; ++p)
                    *reinterpret_cast<uint2*>(a.planes + p * a.plane_stride + m * a.ldp + sg * a.seg_pitch + j0) =
                        make_uint2(pack4(d[p]), pack4(d[p] + 4));
            }
        }
    }
}

// Column statistics of src [M, L]: col_max[j] = bits of max_m |src[m, j] * row_scale[m]| (unsigned
// order equals float order for non-negative floats, and NaN is above everything), and the partial
// column sums of src itself over chunks of rows.  Both are independent of the order of execution.
struct DigitCols {
    const void* src;
    const float* row_scale;   // [M]
    uint32_t* col_max;        // [L], zeroed before
    float* partial;           // [chunks][L] (NULL: no sums)
    int8_t* planes;           // [P][L][ldp]
    float* col_scale;         // [L] written by the digit pass
    int64_t ld, M, L, ldp, plane_stride, rows_per_chunk;
};

template <int DT>
__global__ void __launch_bounds__(256) int8_col_stats_kernel(const DigitCols a) {
    // 32 groups of 8 columns by 8 row lanes
    __shared__ float s_amax[8][256], s_sum[8][256];
    const int cg = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int64_t j0 = ((int64_t)blockIdx.x * 32 + cg) * 8;
    const int64_t m0 = (int64_t)blockIdx.y * a.rows_per_chunk;
    const int64_t m1 = min(a.M, m0 + a.rows_per_chunk);
    uint32_t mx[8];
    float sum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { mx[j] = 0; sum[j] = 0.0f; }
    if (j0 < a.L) {
        for (int64_t m = m0 + rl; m < m1; m += 8) {
            const unsigned char* row = reinterpret_cast<const unsigned char*>(a.src) + m * a.ld * dtype_bytes(DT);
            Raw8<DT> r;
            float v[8];
            r.load(row, j0, a.L, (reinterpret_cast<uintptr_t>(row) & 15) == 0);
            r.unpack(v);
            const float rs = a.row_scale ? __ldg(a.row_scale + m) : 1.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum[j] += v[j];
                mx[j] = max(mx[j], __float_as_uint(fabsf(__fmul_rn(v[j], rs))));
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        s_amax[rl][cg * 8 + j] = __uint_as_float(mx[j]);
        s_sum[rl][cg * 8 + j] = sum[j];
    }
    __syncthreads();
    const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (col >= a.L) return;
    uint32_t m = 0;
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        m = max(m, __float_as_uint(s_amax[i][threadIdx.x]));
        t += s_sum[i][threadIdx.x];
    }
    if (a.col_max) atomicMax(a.col_max + col, m);
    if (a.partial) a.partial[(int64_t)blockIdx.y * a.L + col] = t;
}

// out[j] = sum over chunks of partial[chunk][j], in the type of the bias.
__global__ void __launch_bounds__(256) int8_col_sum_kernel(const float* partial, int64_t chunks, int64_t L, void* out,
                                                           int dtype) {
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (j >= L) return;
    double t = 0.0;
    for (int64_t c = 0; c < chunks; ++c) t += (double)partial[c * L + j];
    const float f = (float)t;
    if (dtype == IMA_DTYPE_F32) reinterpret_cast<float*>(out)[j] = f;
    else if (dtype == IMA_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(out)[j] = __float2bfloat16_rn(f);
    else reinterpret_cast<__half*>(out)[j] = __float2half_rn(f);
}

// Transposed digits: planes[p][j][m] of src[m, j] * row_scale[m] against the column maximum.
// A block turns 128 rows by 32 columns through shared memory: it reads 64 or 128 bytes of a row
// and writes 128 bytes of a plane row at a time.
template <int DT, int P>
__global__ void __launch_bounds__(256) int8_digit_cols_kernel(const DigitCols a) {
    __shared__ float tile[128][33];
    const int64_t m0 = (int64_t)blockIdx.y * 128, j0 = (int64_t)blockIdx.x * 32;
    for (int i = threadIdx.x; i < 128 * 32; i += 256) {
        const int r = i >> 5, c = i & 31;
        float v = 0.0f;
        if (m0 + r < a.M && j0 + c < a.L) {
            v = load_as_f32(a.src, DT, (m0 + r) * a.ld + j0 + c);
            if (a.row_scale) v = __fmul_rn(v, __ldg(a.row_scale + m0 + r));
        }
        tile[r][c] = v;
    }
    __syncthreads();
    const int c = threadIdx.x >> 3, r0 = (threadIdx.x & 7) * 16;
    const int64_t j = j0 + c;
    if (j >= a.L) return;
    const float mx = __uint_as_float(a.col_max[j]);
    const float s = digit_scale<P>(mx, mx != mx);
    const float inv = __frcp_rn(s);
    if (blockIdx.y == 0 && r0 == 0) a.col_scale[j] = s;
    if (m0 + r0 >= a.ldp) return;   // ldp is a multiple of 16
    uint32_t w[P][4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        int32_t d[P][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            int32_t t[P];
            digits_of<P>(tile[r0 + g * 4 + e][c], inv, t);
#pragma unroll
            for (int p = 0; p < P; ++p) d[p][e] = t[p];
        }
#pragma unroll
        for (int p = 0; p < P; ++p) w[p][g] = pack4(d[p]);
    }
#pragma unroll
    for (int p = 0; p < P; ++p)
        *reinterpret_cast<uint4*>(a.planes + p * a.plane_stride + j * a.ldp + m0 + r0) =
            make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
}

// dst[c][r] = src[r][c], int8; columns rows..round16(rows) of dst are zero.
__global__ void __launch_bounds__(256) int8_transpose_kernel(const int8_t* src, int64_t rows, int64_t cols, int64_t ld,
                                                             int8_t* dst, int64_t ldd, int vec) {
    __shared__ uint32_t tile[128][33];   // 128 rows of 128 bytes
    const int64_t r0 = (int64_t)blockIdx.y * 128, c0 = (int64_t)blockIdx.x * 128;
    for (int i = threadIdx.x; i < 128 * 32; i += 256) {
        const int r = i >> 5, w = i & 31;
        uint32_t v = 0;
        if (r0 + r < rows) {
            const int8_t* p = src + (r0 + r) * ld + c0 + w * 4;
            if (vec && c0 + w * 4 + 4 <= cols) {
                v = *reinterpret_cast<const uint32_t*>(p);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c0 + w * 4 + e < cols) v |= (uint32_t)(uint8_t)p[e] << (8 * e);
            }
        }
        tile[r][w] = v;
    }
    __syncthreads();
    // each thread turns 4 x 4 blocks: rows 4 rr .. + 3, columns 4 cw .. + 3
    const int64_t width = (rows + 15) / 16 * 16;
    for (int i = threadIdx.x; i < 32 * 32; i += 256) {
        const int rr = i & 31, cw = i >> 5;
        if (r0 + rr * 4 >= width) continue;
        const uint32_t a = tile[rr * 4][cw], b = tile[rr * 4 + 1][cw], c = tile[rr * 4 + 2][cw], d = tile[rr * 4 + 3][cw];
        const uint32_t ab = __byte_perm(a, b, 0x5140), AB = __byte_perm(a, b, 0x7362);
        const uint32_t cd = __byte_perm(c, d, 0x5140), CD = __byte_perm(c, d, 0x7362);
        const uint32_t o[4] = {__byte_perm(ab, cd, 0x5410), __byte_perm(ab, cd, 0x7632), __byte_perm(AB, CD, 0x5410),
                               __byte_perm(AB, CD, 0x7632)};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c0 + cw * 4 + e < cols)
                *reinterpret_cast<uint32_t*>(dst + (c0 + cw * 4 + e) * ldd + r0 + rr * 4) = o[e];
    }
}

bool known_dtype(int d) { return d == IMA_DTYPE_F32 || d == IMA_DTYPE_BF16 || d == IMA_DTYPE_F16; }

template <int DT>
int launch_quantize(const void* x, int64_t M, int64_t K, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                    cudaStream_t st) {
    // A warp per row where the row fits its registers and the rows fill the machine (no barrier across the
    // block), else a block per row: all of a long row's loads in flight at once.
    constexpr int W = DT == IMA_DTYPE_F32 ? 8 : 16;
    if (K <= 32 * 8 * 4 || (K <= 32 * 8 * W && M >= 148 * 8)) {
        const unsigned grid = (unsigned)std::min<int64_t>((M + 7) / 8, 148 * 32);
        if (K <= 1024) int8_quantize_rows_kernel<DT, 32, 4><<<grid, 256, 0, st>>>(x, M, K, ldx, q, ldq, scale);
        else int8_quantize_rows_kernel<DT, 32, W><<<grid, 256, 0, st>>>(x, M, K, ldx, q, ldq, scale);
    } else {
        const unsigned grid = (unsigned)std::min<int64_t>(M, 148 * 32);
        if (K <= 4096) int8_quantize_rows_kernel<DT, 256, 2><<<grid, 256, 0, st>>>(x, M, K, ldx, q, ldq, scale);
        else int8_quantize_rows_kernel<DT, 256, 10><<<grid, 256, 0, st>>>(x, M, K, ldx, q, ldq, scale);
    }
    return IMA_LAUNCH_STATUS();
}

template <int DT>
int launch_digit_rows(const DigitRows& a, int planes, cudaStream_t st) {
    const unsigned grid = (unsigned)std::min<int64_t>(a.M, 148 * 32);
    if (planes == 2) int8_digit_rows_kernel<DT, 2><<<grid, 256, 0, st>>>(a);
    else int8_digit_rows_kernel<DT, 3><<<grid, 256, 0, st>>>(a);
    return IMA_LAUNCH_STATUS();
}

constexpr int64_t I8_COL_CHUNK = 256;   // rows per partial column sum

template <int DT>
int launch_col_stats(const DigitCols& a, cudaStream_t st) {
    const dim3 grid((unsigned)((a.L + 255) / 256), (unsigned)((a.M + a.rows_per_chunk - 1) / a.rows_per_chunk));
    int8_col_stats_kernel<DT><<<grid, 256, 0, st>>>(a);
    return IMA_LAUNCH_STATUS();
}

template <int DT>
int launch_digit_cols(const DigitCols& a, int planes, cudaStream_t st) {
    const dim3 grid((unsigned)((a.L + 31) / 32), (unsigned)((a.ldp + 127) / 128));
    if (planes == 2) int8_digit_cols_kernel<DT, 2><<<grid, 256, 0, st>>>(a);
    else int8_digit_cols_kernel<DT, 3><<<grid, 256, 0, st>>>(a);
    return IMA_LAUNCH_STATUS();
}

}  // namespace

extern "C" {

int ima_int8_quantize_rows(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, int8_t* q, int64_t ldq,
                           float* scale, void* stream) {
    if (M < 0 || K < 0 || !known_dtype(x_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    if (M == 0) return IMA_OK;
    if (!scale || (K > 0 && (!x || !q || (M > 1 && ldx < K)))) return IMA_ERR_INVALID_ARGUMENT;
    if (ldq < K || ldq % 16 || (reinterpret_cast<uintptr_t>(q) & 15)) return IMA_ERR_INVALID_ARGUMENT;
    cudaStream_t st = (cudaStream_t)stream;
    if (x_dtype == IMA_DTYPE_BF16) return launch_quantize<IMA_DTYPE_BF16>(x, M, K, ldx, q, ldq, scale, st);
    if (x_dtype == IMA_DTYPE_F16) return launch_quantize<IMA_DTYPE_F16>(x, M, K, ldx, q, ldq, scale, st);
    return launch_quantize<IMA_DTYPE_F32>(x, M, K, ldx, q, ldq, scale, st);
}

int ima_int8_transpose(const int8_t* src, int64_t rows, int64_t cols, int64_t ld, int8_t* dst, int64_t ldd,
                       void* stream) {
    if (rows < 0 || cols < 0) return IMA_ERR_INVALID_ARGUMENT;
    if (rows == 0 || cols == 0) return IMA_OK;
    if (!src || !dst || ld < cols || ldd < rows || ldd % 16 || (reinterpret_cast<uintptr_t>(dst) & 15))
        return IMA_ERR_INVALID_ARGUMENT;
    if ((rows + 127) / 128 > 65535) return IMA_ERR_UNSUPPORTED;
    const int vec = !((reinterpret_cast<uintptr_t>(src) | (uintptr_t)ld) & 3);
    const dim3 grid((unsigned)((cols + 127) / 128), (unsigned)((rows + 127) / 128));
    int8_transpose_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(src, rows, cols, ld, dst, ldd, vec);
    return IMA_LAUNCH_STATUS();
}

int ima_int8_digits_rows(const void* src, int src_dtype, int64_t M, int64_t seg_len, int64_t seg_pitch, int segs,
                         int64_t ld, const float* col_scale, int planes, int8_t* out, int64_t ldp, float* row_scale,
                         void* stream) {
    if (M < 0 || seg_len < 0 || segs < 1 || segs > 2 || !known_dtype(src_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    if (planes != 2 && planes != 3) return IMA_ERR_UNSUPPORTED;
    if (M == 0) return IMA_OK;
    if (!row_scale || !out || (seg_len > 0 && !src)) return IMA_ERR_INVALID_ARGUMENT;
    if (seg_pitch < seg_len || ldp % 16 || (segs > 1 && seg_pitch % 16)) return IMA_ERR_INVALID_ARGUMENT;
    const int64_t width = (segs - 1) * seg_pitch + seg_len;
    if (ldp < width || (M > 1 && ld < width) || (reinterpret_cast<uintptr_t>(out) & 15)) return IMA_ERR_INVALID_ARGUMENT;
    const DigitRows a = {src, col_scale, out, row_scale, ld, M, seg_len, seg_pitch, ldp, M * ldp, segs, 0};
    cudaStream_t st = (cudaStream_t)stream;
    if (src_dtype == IMA_DTYPE_BF16) return launch_digit_rows<IMA_DTYPE_BF16>(a, planes, st);
    if (src_dtype == IMA_DTYPE_F16) return launch_digit_rows<IMA_DTYPE_F16>(a, planes, st);
    return launch_digit_rows<IMA_DTYPE_F32>(a, planes, st);
}

int64_t ima_int8_cols_workspace_bytes(int64_t M, int64_t L) {
    if (M < 0 || L < 0) return 0;
    return ((M + I8_COL_CHUNK - 1) / I8_COL_CHUNK + 1) * L * 4;
}

int ima_int8_digits_cols(const void* src, int src_dtype, int64_t M, int64_t L, int64_t ld, const float* row_scale,
                         int planes, int8_t* out, int64_t ldp, float* col_scale, void* sum_out, int sum_dtype,
                         void* workspace, void* stream) {
    if (M < 0 || L < 0 || !known_dtype(src_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    if (planes != 0 && planes != 2 && planes != 3) return IMA_ERR_UNSUPPORTED;
    if (L == 0) return IMA_OK;
    if (!workspace || (M > 0 && (!src || (M > 1 && ld < L)))) return IMA_ERR_INVALID_ARGUMENT;
    if (planes && (!out || !col_scale || ldp < M || ldp % 16 || (reinterpret_cast<uintptr_t>(out) & 15)))
        return IMA_ERR_INVALID_ARGUMENT;
    if (sum_out && !known_dtype(sum_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    if ((ldp + 127) / 128 > 65535 || (M + I8_COL_CHUNK - 1) / I8_COL_CHUNK > 65535) return IMA_ERR_UNSUPPORTED;
    cudaStream_t st = (cudaStream_t)stream;
    uint32_t* col_max = reinterpret_cast<uint32_t*>(workspace);
    float* partial = reinterpret_cast<float*>(workspace) + L;
    int rc = IMA_OK;
    if (planes) {
        rc = ima_note_cuda(cudaMemsetAsync(col_max, 0, (size_t)L * 4, st));
        if (rc != IMA_OK) return rc;
    }
    DigitCols a = {src, row_scale, planes ? col_max : nullptr, sum_out ? partial : nullptr, out, col_scale, ld, M, L,
                   ldp, L * ldp, I8_COL_CHUNK};
    if (M > 0) {
        if (src_dtype == IMA_DTYPE_BF16) rc = launch_col_stats<IMA_DTYPE_BF16>(a, st);
        else if (src_dtype == IMA_DTYPE_F16) rc = launch_col_stats<IMA_DTYPE_F16>(a, st);
        else rc = launch_col_stats<IMA_DTYPE_F32>(a, st);
        if (rc != IMA_OK) return rc;
    }
    if (sum_out) {
        int8_col_sum_kernel<<<(unsigned)((L + 255) / 256), 256, 0, st>>>(partial, (M + I8_COL_CHUNK - 1) / I8_COL_CHUNK,
                                                                        L, sum_out, sum_dtype);
        rc = IMA_LAUNCH_STATUS();
        if (rc != IMA_OK) return rc;
    }
    if (!planes || M == 0) return IMA_OK;
    if (src_dtype == IMA_DTYPE_BF16) return launch_digit_cols<IMA_DTYPE_BF16>(a, planes, st);
    if (src_dtype == IMA_DTYPE_F16) return launch_digit_cols<IMA_DTYPE_F16>(a, planes, st);
    return launch_digit_cols<IMA_DTYPE_F32>(a, planes, st);
}

}  // extern "C"
