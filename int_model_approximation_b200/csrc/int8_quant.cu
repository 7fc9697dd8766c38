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
// digits, v = sum_p 256^p d_p with d_p in [-128, 127] (V_2 = 127 * 256 + 127, V_3 = 8355000, a little
// below 127 * 65536 + 127 * 256 + 127), so the product runs on the int8 tensor cores exactly.  The rounding is the
// one place where a gradient loses bits: half a step of amax / V_P, i.e. at most 2^-16 (P = 2) or
// 2^-24 (P = 3) of the row's largest element; elements below that vanish.  Against the rms of
// the row's products that is at most sqrt(L / 3) 2^-16 for L summands, reached only when one
// element carries the whole row: 1.7e-3 over the 37888 columns of a pair, 3.2e-3 over the longest sum.
// Measured: 4e-5 for Gaussian rows, 6e-4 for columns of 4096 token gradients of very different sizes.  bf16 rounds
// by up to 2^-8 of a value, 1.6e-3 of a norm, fp16 by an eighth of that: the callers take P = 2 for bf16 and L <=
// 65536, where the worst case is 2.3e-3, else P = 3.
#include <algorithm>
#include <type_traits>
#include "sm100_pair.cuh"

namespace {

// Reciprocals of a scale that bracket it: x * lo and x * hi lie on either side of RN32(x / s), which is off
// by at most 2^-24 of the quotient, as are the products.
struct I8Inv {
    float mid, lo, hi;
};
IMA_DEVINL I8Inv i8_inv(float s) {
    const float inv = __frcp_rn(s);
    return {inv, __fmul_rn(inv, 1.0f - 0x1p-21f), __fmul_rn(inv, 1.0f + 0x1p-21f)};
}

// rint(RN32(x / s)) where x * inv rounds to a on one side of its bracket and to c on the other, without
// dividing.  h = (a + c) / 2 is the half-integer between; e = x - h s is exact (h has 8 bits, s 24, and
// the difference few).  RN32(x / s) equals h, a tie, when |x / s - h| is below half a step of fp32 at
// h (a quotient of two fp32 numbers is never exactly on that boundary); otherwise e's sign decides.
IMA_DEVINL uint32_t i8_near_tie(float x, float s, float a, float c) {
    const float h = 0.5f * (a + c);
    const float e = __fmaf_rn(-h, s, x);
    const float half_step = __uint_as_float((__float_as_uint(h) & 0x7F800000u) - (24u << 23));
    const float even = __fmul_rn(2.0f, rintf(__fmul_rn(0.5f, h)));   // the even one of a and c
    const float k = fabsf(e) < __fmul_rn(s, half_step) ? even : (e > 0.0f ? fmaxf(a, c) : fminf(a, c));
    return (uint32_t)(int32_t)k;
}

// Codes of eight elements, rint(RN32(x / s)) each, without a division per element.  A scale that is NaN
// or inf gives codes 0.  1.5 * 2^23 is added to have the rounded integer in the low mantissa bits.
//   16-bit inputs: Markstein's correction (see the fp8 quantiser), q0 = x y, q = q0 + (x - s q0) y with y =
//     RN(1/s), which is RN32(x / s) to the last bit or at least rounds like it for every pair of a bf16
//     or fp16 maximum and element (powers of two apart, 128^2 and 1024^2 pairs of significands times ten
//     binades; a GPU test goes through them).  No branch: these inputs have few bits, and near-ties
//     are common (0.2 % of bf16 elements).
//   fp32: fma(x, inv, 1.5 * 2^23) for both brackets; rounding is monotonic, so where they agree the
//     quotient rounds alike, and elsewhere (3 in 10^5) i8_near_tie decides.
template <int DT>
IMA_DEVINL uint2 i8_codes8(const float (&v)[8], float s, I8Inv inv) {
    constexpr float kRound = 12582912.0f;
    uint32_t b[8];
    if (DT != IMA_DTYPE_F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float q0 = __fmul_rn(v[j], inv.mid);
            const float q = __fmaf_rn(__fmaf_rn(-q0, s, v[j]), inv.mid, q0);
            b[j] = __float_as_uint(__fadd_rn(q, kRound));
        }
    } else {
        float lo[8], hi[8];
        uint32_t differ = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            lo[j] = __fmaf_rn(v[j], inv.lo, kRound);
            hi[j] = __fmaf_rn(v[j], inv.hi, kRound);
            b[j] = __float_as_uint(lo[j]);
            differ |= b[j] ^ __float_as_uint(hi[j]);
        }
        if (differ) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (lo[j] != hi[j]) b[j] = i8_near_tie(v[j], s, lo[j] - kRound, hi[j] - kRound);
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

// N words that start d bytes (0..15) into the N + 4 aligned ones of w.
template <int N>
IMA_DEVINL void shift_words(const uint32_t (&w)[N + 4], uint32_t d, uint32_t (&o)[N]) {
    uint32_t x[N + 2], y[N + 1];
#pragma unroll
    for (int j = 0; j < N + 2; ++j) x[j] = d & 8 ? w[j + 2] : w[j];
#pragma unroll
    for (int j = 0; j < N + 1; ++j) y[j] = d & 4 ? x[j + 1] : x[j];
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = __funnelshift_r(y[j], y[j + 1], (d & 3) * 8);
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
    // the same from a row that lies d bytes behind a 16-byte boundary, by aligned loads (all of which
    // touch bytes of the eight elements)
    IMA_DEVINL void load_shifted(const void* row, int64_t k0, uint32_t d) {
        const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned char*>(row) + k0 * 4 - d);
        const uint4 a = __ldg(p), b = __ldg(p + 1), c = __ldg(p + 2);
        const uint32_t w[12] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, c.x, c.y, c.z, c.w};
        uint32_t o[8];
        shift_words<8>(w, d, o);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(o[j]);
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
    IMA_DEVINL void load_shifted(const void* row, int64_t k0, uint32_t d) {
        const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned char*>(row) + k0 * 2 - d);
        const uint4 a = __ldg(p), b = __ldg(p + 1);
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        uint32_t o[4];
        shift_words<4>(w, d, o);
        u = make_uint4(o[0], o[1], o[2], o[3]);
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

// Maximum over the TPR threads of a row (whole warps of a block of 256).
template <int TPR>
IMA_DEVINL uint32_t row_max(uint32_t m, uint32_t* s_max) {
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    if (TPR > 32) {
        const int warp = threadIdx.x >> 5, group = threadIdx.x / TPR;
        if ((threadIdx.x & 31) == 0) s_max[warp] = m;
        named_barrier_sync(1 + group, TPR);
#pragma unroll
        for (int i = 0; i < TPR / 32; ++i) m = max(m, s_max[group * (TPR / 32) + i]);
        named_barrier_sync(1 + group, TPR);
    }
    return m;
}

// ---------------------------------------------------------------------------
// Row quantiser.  TPR threads take one row; a row of up to TPR * 8 * V elements is read once
// and kept in registers between the maximum and the codes, a longer one is read again (from
// L2).  Bound by memory: 2 or 4 bytes in and 1 out per element.  16384 x 3584 from bf16 takes 35 us (27 at the
// measured copy rate), 16384 x 18944 156 (142; 177 with two blocks per SM instead of three); fp32 rows are at the
// copy rate.
// ---------------------------------------------------------------------------
struct QuantRows {           // up to three matrices of K columns, one after the other (activations, weights)
    const void* x[3];
    int8_t* q[3];
    float* scale[3];
    int64_t ldx[3], ldq[3], end[3];   // end: rows of this and the matrices before it
    int64_t K;
};

template <int DT, int TPR, int V>
__global__ void __launch_bounds__(256, DT != IMA_DTYPE_F32 && V <= 10 ? 3 : 2) int8_quantize_rows_kernel(const __grid_constant__ QuantRows a) {
    // a product launched to follow this kernel may start now; it waits for this kernel's end before it reads
    allow_next_kernel();
    __shared__ uint32_t s_max[8];
    constexpr int ROWS = 256 / TPR;
    const int tid = threadIdx.x % TPR;
    const int64_t K = a.K;
    for (int64_t row_at = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR; row_at < a.end[2];
         row_at += (int64_t)gridDim.x * ROWS) {
        const int which = (row_at >= a.end[0]) + (row_at >= a.end[1]);
        const int64_t m = row_at - (which ? a.end[which - 1] : 0);
        const unsigned char* row = reinterpret_cast<const unsigned char*>(a.x[which]) + m * a.ldx[which] * dtype_bytes(DT);
        const uint32_t d = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15;   // the same for a warp
        const bool vec = d == 0;
        // whole groups of eight that this thread keeps; the rest is loaded twice
        const int64_t whole = min(K / 8 * 8, (int64_t)V * TPR * 8);
        // the last K % 8 elements, where all groups before them are kept
        const bool ends = whole == K / 8 * 8;
        const int64_t rest = ends ? K : whole;
        Raw8<DT> keep[V], last;
        last.clear();
        if (ends && whole < K && tid == 0) last.load(row, whole, K, vec);
        uint32_t mx = 0;
        if (vec) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                keep[i].clear();
                if ((i * TPR + tid) * 8 < whole) keep[i].load_whole(row, (int64_t)(i * TPR + tid) * 8);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                keep[i].clear();
                if ((i * TPR + tid) * 8 < whole) keep[i].load_shifted(row, (int64_t)(i * TPR + tid) * 8, d);
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) mx = max(mx, keep[i].max_bits());
        mx = max(mx, last.max_bits());
#pragma unroll 1
        for (int64_t k0 = rest + tid * 8; k0 < K; k0 += TPR * 8) {
            Raw8<DT> r;
            if (vec || k0 + 8 > K) r.load(row, k0, K, vec);
            else r.load_shifted(row, k0, d);
            mx = max(mx, r.max_bits());
        }
        const float amax = __uint_as_float(row_max<TPR>(mx, s_max));
        const float s = i8_row_scale(amax, amax != amax);
        const I8Inv inv = i8_inv(s);
        if (tid == 0) a.scale[which][m] = s;
        int8_t* qr = a.q[which] + m * a.ldq[which];
        auto emit = [&](const Raw8<DT>& r, int64_t k0) {
            float v[8];
            r.unpack(v);
            *reinterpret_cast<uint2*>(qr + k0) = i8_codes8<DT>(v, s, inv);
        };
#pragma unroll
        for (int i = 0; i < V; ++i)
            if ((i * TPR + tid) * 8 < whole) emit(keep[i], (int64_t)(i * TPR + tid) * 8);
        if (ends && whole < K && tid == 0) emit(last, whole);
#pragma unroll 1
        for (int64_t k0 = rest + tid * 8; k0 < K; k0 += TPR * 8) {
            Raw8<DT> r;
            if (vec || k0 + 8 > K) r.load(row, k0, K, vec);
            else r.load_shifted(row, k0, d);
            emit(r, k0);
        }
    }
}

// ---------------------------------------------------------------------------
// Digits
// ---------------------------------------------------------------------------
template <int P>
IMA_DEVINL float digit_limit() { return P == 2 ? 32639.0f : 8355000.0f; }

// Scale of a row (or column) with largest magnitude `amax`: never zero, so that a row of zeros has
// codes 0, and never so small that its reciprocal overflows; NaN where an element is NaN or infinite,
// so that its products are NaN.
template <int P>
IMA_DEVINL float digit_scale(float amax) {
    if (!(amax <= 3.402823466e38f)) return __int_as_float(0x7FC00000);
    return fmaxf(__fdiv_rn(amax, digit_limit<P>()), 1.17549435e-38f);
}

// The P digit bytes of eight values x * inv, packed.  Two digits: fma(x, inv, 1.5 * 2^23) holds v in its
// low mantissa bits; its lowest byte is d_0 and (v + 128) >> 8 is d_1.  |x * inv| <= V_P (1 + 2^-22):
// 32639.01, and 8355002 where the digits end at 8355711, so no rounding leaves the range.
template <int P>
IMA_DEVINL void digits8(const float (&x)[8], float inv, uint2 (&out)[P]) {
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
        v[j] = P == 2 ? __float_as_uint(__fmaf_rn(x[j], inv, 12582912.0f)) : (uint32_t)__float2int_rn(__fmul_rn(x[j], inv));
#pragma unroll
    for (int p = 0; p < P; ++p) {
        out[p] = make_uint2(__byte_perm(__byte_perm(v[0], v[1], 0x0040), __byte_perm(v[2], v[3], 0x0040), 0x5410),
                            __byte_perm(__byte_perm(v[4], v[5], 0x0040), __byte_perm(v[6], v[7], 0x0040), 0x5410));
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (uint32_t)((int32_t)(v[j] + 128u) >> 8);
    }
}

// A gradient D [M, W]: `segs` segments of n columns, `pitch` columns apart (W = segs * pitch; columns
// between segments hold nothing).  Its row form is D ws (channel scales, one vector per segment), its
// column form D xs (token scales), each with its own maxima, as bit patterns of non-negative fp32.
struct GradSrc {
    const void* src;
    const float* ws[2];
    const float* xs;
    uint32_t* row_max;        // [M]
    uint32_t* col_max;        // [W]
    int64_t ld, M, n, pitch, W;
};

// Maxima of both forms.  A block takes 64 rows by 256 columns: a warp has one row's 256 columns at a
// time, so the row maximum is one warp reduction and the column maxima stay in registers.
template <int DT>
__global__ void __launch_bounds__(256) int8_grad_max_kernel(const GradSrc a) {
    __shared__ uint32_t s_max[8][256];
    const int cg = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int64_t j0 = (int64_t)blockIdx.x * 256 + cg * 8;
    const int64_t m0 = (int64_t)blockIdx.y * 64;
    uint32_t mx[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = a.row_max && j0 + j < a.n ? __ldg(a.ws[0] + j0 + j) : 0.0f;
    Raw8<DT> r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t m = m0 + rl + i * 8;
        const unsigned char* row = reinterpret_cast<const unsigned char*>(a.src) + m * a.ld * dtype_bytes(DT);
        r[i].clear();
        if (m < a.M && j0 < a.n) r[i].load(row, j0, a.n, (reinterpret_cast<uintptr_t>(row) & 15) == 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t m = m0 + rl + i * 8;
        if (m >= a.M) break;
        float v[8];
        r[i].unpack(v);
        const float xs = a.col_max ? __ldg(a.xs + m) : 0.0f;
        uint32_t rm = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            rm = max(rm, __float_as_uint(fabsf(__fmul_rn(v[j], w[j]))));
            mx[j] = max(mx[j], __float_as_uint(fabsf(__fmul_rn(v[j], xs))));
        }
        if (a.row_max) {
            rm = __reduce_max_sync(0xFFFFFFFFu, rm);
            if (cg == 0) atomicMax(a.row_max + m, rm);
        }
    }
    if (!a.col_max) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) s_max[rl][cg * 8 + j] = mx[j];
    __syncthreads();
    const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, s_max[i][threadIdx.x]);
    if (col < a.n) atomicMax(a.col_max + col, m);
}

// Digit planes of both forms, and partial column sums of D (in 64 bits), in one pass over D.  A block takes 128 rows
// by 64 columns; the transposed form goes through shared memory.  There a row is 16 quads of columns, the
// two of its thread t at t ^ (row / 16) and (t + 8) ^ (row / 16): eight threads that write a row, and eight
// 16-row groups that read a quad, meet no bank conflicts.  Every plane row is written
// in pieces of 64 (rows) or 128 (columns) contiguous bytes.  Either form and the sums may be absent.  Bound by
// memory: 4096 x 37888 from fp32 to two planes both ways (1.24 GB) takes 212 us, 189 at the measured copy rate.
struct GradDigits {
    GradSrc g;
    int8_t* rows;             // [P][M][W]
    float* row_scale;         // [M]
    int8_t* cols;             // [P][W][ldm]
    float* col_scale;         // [W]
    double* partial;          // [ceil(M / 128)][W]
    int64_t ldm;
};

template <int DT, int P>
__global__ void __launch_bounds__(256) int8_grad_digits_kernel(const GradDigits a) {
    __shared__ float4 tile[128 * 16];                           // four columns each
    __shared__ float4 s_xs[32];                                 // token scales of the 128 rows, 0 beyond the last
    __shared__ float s_row_inv[128], s_col_inv[64];             // reciprocals of the digit scales
    const GradSrc& g = a.g;
    const int64_t m0 = (int64_t)blockIdx.y * 128, c0 = (int64_t)blockIdx.x * 64;
    const int seg = c0 >= g.pitch ? 1 : 0;
    const int valid = (int)min((int64_t)64, g.n - (c0 - seg * g.pitch));   // columns of this tile that hold something
    const int rows = (int)min((int64_t)128, g.M - m0);
    // eight columns of rows r0 + 32 i, in two quads: neighbours of 16 bits, 32 columns apart of fp32, so that eight
    // threads load 128 contiguous bytes either way
    constexpr bool F32 = DT == IMA_DTYPE_F32;
    const int ch = threadIdx.x & 7, r0 = threadIdx.x >> 3;
    const int ca = F32 ? 4 * ch : 8 * ch, cb = F32 ? 4 * ch + 32 : 8 * ch + 4;
    Raw8<DT> raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = r0 + i * 32;
        raw[i].clear();
        if (r < rows && ca < valid) {
            const unsigned char* p = reinterpret_cast<const unsigned char*>(g.src) + ((m0 + r) * g.ld + c0) * dtype_bytes(DT);
            const bool vec = (reinterpret_cast<uintptr_t>(p) & 15) == 0;
            if constexpr (F32) {
                const float* f = reinterpret_cast<const float*>(p);
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int c = hf ? cb : ca;
                    if (vec && c + 4 <= valid) {
                        const float4 q = __ldg(reinterpret_cast<const float4*>(f + c));
                        raw[i].v[4 * hf] = q.x; raw[i].v[4 * hf + 1] = q.y; raw[i].v[4 * hf + 2] = q.z; raw[i].v[4 * hf + 3] = q.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) raw[i].v[4 * hf + e] = c + e < valid ? __ldg(f + c + e) : 0.0f;
                    }
                }
            } else {
                if (vec && ca + 8 <= valid) raw[i].load_whole(p, ca);
                else raw[i].load(p, ca, valid, false);
            }
        }
    }
    if (threadIdx.x < 128) {
        const int r = threadIdx.x;
        if (a.cols) reinterpret_cast<float*>(s_xs)[r] = r < rows ? __ldg(g.xs + m0 + r) : 0.0f;
        if (a.rows && r < rows) {
            const float s = digit_scale<P>(__uint_as_float(g.row_max[m0 + r]));
            if (blockIdx.x == 0) a.row_scale[m0 + r] = s;
            s_row_inv[r] = __frcp_rn(s);
        }
    } else if (a.cols && threadIdx.x < 192) {
        const int c = threadIdx.x - 128;
        if (c < valid) {
            const float s = digit_scale<P>(__uint_as_float(g.col_max[c0 + c]));
            if (blockIdx.y == 0) a.col_scale[c0 + c] = s;
            s_col_inv[c] = __frcp_rn(s);
        }
    }
    float w[8];
    if (a.rows) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = j < 4 ? ca + j : cb + j - 4;
            w[j] = c < valid ? __ldg(g.ws[seg] + (c0 - seg * g.pitch) + c) : 0.0f;
        }
    }
    __syncthreads();
    const bool in_a = a.rows && c0 + ca < g.W, in_b = a.rows && c0 + cb < g.W;
    int8_t* row_out = a.rows + (m0 + r0) * g.W + c0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = r0 + i * 32;
        float v[8];
        raw[i].unpack(v);
        if (in_a && r < rows) {
            const float inv = s_row_inv[r];
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __fmul_rn(v[j], w[j]);
            uint2 d[P];
            digits8<P>(x, inv, d);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                int8_t* out = row_out + (int64_t)p * g.M * g.W + (int64_t)i * 32 * g.W;
                if (F32) {
                    *reinterpret_cast<uint32_t*>(out + ca) = d[p].x;
                    if (in_b) *reinterpret_cast<uint32_t*>(out + cb) = d[p].y;
                } else {
                    *reinterpret_cast<uint2*>(out + ca) = d[p];
                }
            }
        }
        if (a.cols || a.partial) {
            tile[r * 16 + (ch ^ (r >> 4))] = make_float4(v[0], v[1], v[2], v[3]);
            tile[r * 16 + ((ch + 8) ^ (r >> 4))] = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
    if (!a.cols && !a.partial) return;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sg = lane >> 2;                                   // rows 16 sg .. + 15
#pragma unroll
    for (int it = 0; it < 2; ++it) {
        const int c = (F32 ? it * 32 + warp * 4 : warp * 8 + it * 4) + (lane & 3);
        const float* from = reinterpret_cast<const float*>(tile + sg * 256 + ((warp + it * 8) ^ sg)) + (lane & 3);
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = from[i * 64];
        if (a.partial) {
            double sum = 0.0;   // 64 bits throughout: one rounding, to the bias' type, at the end
#pragma unroll
            for (int i = 0; i < 16; ++i) sum += (double)v[i];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            if (lane < 4 && c < valid) a.partial[(int64_t)blockIdx.y * g.W + c0 + c] = sum;
        }
        if (a.cols && c < valid && m0 + sg * 16 < a.ldm) {
            const float inv = s_col_inv[c];
            uint2 d[2][P];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const float4 x0 = s_xs[sg * 4 + hf * 2], x1 = s_xs[sg * 4 + hf * 2 + 1];
                const float* u = v + hf * 8;
                const float x[8] = {__fmul_rn(u[0], x0.x), __fmul_rn(u[1], x0.y), __fmul_rn(u[2], x0.z),
                                    __fmul_rn(u[3], x0.w), __fmul_rn(u[4], x1.x), __fmul_rn(u[5], x1.y),
                                    __fmul_rn(u[6], x1.z), __fmul_rn(u[7], x1.w)};
                digits8<P>(x, inv, d[hf]);
            }
#pragma unroll
            for (int p = 0; p < P; ++p)
                *reinterpret_cast<uint4*>(a.cols + ((int64_t)p * g.W + c0 + c) * a.ldm + m0 + sg * 16) =
                    make_uint4(d[0][p].x, d[0][p].y, d[1][p].x, d[1][p].y);
        }
    }
}

// out[j] = sum over chunks of partial[chunk][j], in the type of the bias; blockIdx.y: which of two
// segments, `pitch` columns apart (out NULL: not wanted).
__global__ void __launch_bounds__(256) int8_col_sum_kernel(const double* partial, int64_t chunks, int64_t W, int64_t n,
                                                           int64_t pitch, void* out0, void* out1, int dtype) {
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
    void* out = blockIdx.y ? out1 : out0;
    if (j >= n || !out) return;
    double t = 0.0;
    for (int64_t c = 0; c < chunks; ++c) t += partial[c * W + blockIdx.y * pitch + j];
    if (dtype == IMA_DTYPE_F32) reinterpret_cast<float*>(out)[j] = (float)t;
    else if (dtype == IMA_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(out)[j] = __double2bfloat16(t);
    else reinterpret_cast<__half*>(out)[j] = __double2half(t);
}

// dst[c][r] = src[r][c], int8; columns rows..round16(rows) of dst are zero.  A block turns 128 x 128
// bytes: 16-byte loads, 4 x 4 byte blocks turned in registers, 128 contiguous bytes out per row.  Up to three
// matrices in one launch, and words to be zeroed.
struct TransposeJobs {
    const int8_t* src[3];
    int8_t* dst[3];
    int64_t rows[3], cols[3], ld[3], ldd[3], end[3];   // end: blocks of this and the matrices before it
    uint32_t* zero;
    int64_t zero_words;
};

__global__ void __launch_bounds__(256) int8_transpose_kernel(const __grid_constant__ TransposeJobs a) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.zero_words; i += (int64_t)gridDim.x * 256) a.zero[i] = 0;
    const int64_t block = blockIdx.x;
    if (block >= a.end[2]) return;
    const int which = (block >= a.end[0]) + (block >= a.end[1]);
    const int64_t rows = a.rows[which], cols = a.cols[which], ld = a.ld[which], ldd = a.ldd[which];
    const int8_t* src = a.src[which];
    int8_t* dst = a.dst[which];
    const bool vec = ((reinterpret_cast<uintptr_t>(src) | (uintptr_t)ld) & 15) == 0;
    const int64_t across = (cols + 127) / 128, at = block - (which ? a.end[which - 1] : 0);
    const int64_t r0 = at / across * 128, c0 = at % across * 128;
    __shared__ uint32_t tile[128][33];   // 128 rows of 128 bytes
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = i * 32 + (threadIdx.x >> 3), b = (threadIdx.x & 7) * 16;
        v[i] = make_uint4(0, 0, 0, 0);
        if (r0 + r < rows && c0 + b < cols) {
            const int8_t* p = src + (r0 + r) * ld + c0 + b;
            if (vec && c0 + b + 16 <= cols) {
                v[i] = __ldg(reinterpret_cast<const uint4*>(p));
            } else {
                uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (c0 + b + e < cols) w[e >> 2] |= (uint32_t)(uint8_t)p[e] << (8 * (e & 3));
                v[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = i * 32 + (threadIdx.x >> 3), w = (threadIdx.x & 7) * 4;
        tile[r][w] = v[i].x; tile[r][w + 1] = v[i].y; tile[r][w + 2] = v[i].z; tile[r][w + 3] = v[i].w;
    }
    __syncthreads();
    const int64_t width = (rows + 15) / 16 * 16;
    const int rr = threadIdx.x & 31;     // rows 4 rr .. + 3: a warp writes 128 contiguous bytes
    if (r0 + rr * 4 >= width) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int cw = i * 8 + (threadIdx.x >> 5);
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

// Rows of int8 codes moved to rows that start on 16 bytes, as the tile loads need them: dst[r][c] = src[r][c], and zeros in
// columns cols..round16(cols).  Up to two matrices of one width in a launch.  A thread makes 16 bytes from the
// aligned 4-byte words that hold them, shifted into place.
struct PackRows {
    const int8_t* src[2];
    int8_t* dst[2];
    int64_t ld[2], end[2];   // end: rows of this and the matrix before it
    int64_t cols, ldd;
};

__global__ void __launch_bounds__(256) int8_pack_rows_kernel(const __grid_constant__ PackRows a) {
    const int64_t chunks = (a.cols + 15) / 16, total = a.end[1] * chunks;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / chunks, c = (i - row * chunks) * 16;
        const int which = row >= a.end[0];
        const int64_t r = row - (which ? a.end[0] : 0);
        const uintptr_t from = reinterpret_cast<uintptr_t>(a.src[which] + r * a.ld[which] + c);
        const int n = (int)min((int64_t)16, a.cols - c), shift = (int)(from & 3);
        const uint32_t* p = reinterpret_cast<const uint32_t*>(from - shift);
        uint32_t w[5], o[4];
#pragma unroll
        for (int j = 0; j < 5; ++j) w[j] = j * 4 < n + shift ? __ldg(p + j) : 0;   // words with a wanted byte
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[j] = __funnelshift_r(w[j], w[j + 1], shift * 8);
            const int left = n - j * 4;
            if (left < 4) o[j] = left > 0 ? o[j] & ((1u << (left * 8)) - 1) : 0;
        }
        *reinterpret_cast<uint4*>(a.dst[which] + r * a.ldd + c) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

bool known_dtype(int d) { return d == IMA_DTYPE_F32 || d == IMA_DTYPE_BF16 || d == IMA_DTYPE_F16; }

template <int DT>
int launch_quantize(const QuantRows& a, cudaStream_t st) {
    const int64_t M = a.end[2], K = a.K;
    if (M == 0) return IMA_OK;
    // As few threads per row as hold it in registers, when the rows fill the machine: 8 KB of a row in flight
    // per warp and no barrier, or a barrier of two to eight warps.  Few rows: a block each, for latency.
    // Rows off 16 bytes take two loads per group, so half as many groups per thread (12638 x 2269 from bf16: 44 us,
    // 54 with 16; aligned rows 35 us either way at 16384 x 3584).
    constexpr bool F = DT == IMA_DTYPE_F32;
    const bool many = M >= 148 * 8;
    bool shifted = false;
    for (int i = 0; i < 3; ++i)
        shifted |= a.end[i] > (i ? a.end[i - 1] : 0) &&
                   ((reinterpret_cast<uintptr_t>(a.x[i]) | (uintptr_t)(a.ldx[i] * dtype_bytes(DT))) & 15) != 0;
    auto run = [&](auto tpr, auto v) {
        constexpr int TPR = decltype(tpr)::value, V = decltype(v)::value;
        const unsigned grid = (unsigned)std::min<int64_t>((M * TPR + 255) / 256, 148 * 32);
        int8_quantize_rows_kernel<DT, TPR, V><<<grid, 256, 0, st>>>(a);
    };
    if (K <= 1024) run(std::integral_constant<int, 32>{}, std::integral_constant<int, 4>{});
    else if (many && K <= (F ? 2048 : 4096) && (F || !shifted)) run(std::integral_constant<int, 32>{}, std::integral_constant<int, F ? 8 : 16>{});
    else if (many && !F && K <= 4096) run(std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
    else if (many && K <= 5120) run(std::integral_constant<int, 64>{}, std::integral_constant<int, 10>{});
    else if (many && K <= 10240) run(std::integral_constant<int, 128>{}, std::integral_constant<int, 10>{});
    else if (K <= 4096) run(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else run(std::integral_constant<int, 256>{}, std::integral_constant<int, 10>{});
    return IMA_LAUNCH_STATUS();
}

template <int DT>
int launch_grad_max(const GradSrc& a, cudaStream_t st) {
    const dim3 grid((unsigned)((a.n + 255) / 256), (unsigned)((a.M + 63) / 64));
    int8_grad_max_kernel<DT><<<grid, 256, 0, st>>>(a);
    return IMA_LAUNCH_STATUS();
}

template <int DT>
int launch_grad_digits(const GradDigits& a, int planes, cudaStream_t st) {
    const dim3 grid((unsigned)((a.g.W + 63) / 64), (unsigned)((a.g.M + 127) / 128));
    if (planes == 2) int8_grad_digits_kernel<DT, 2><<<grid, 256, 0, st>>>(a);
    else int8_grad_digits_kernel<DT, 3><<<grid, 256, 0, st>>>(a);
    return IMA_LAUNCH_STATUS();
}

int run_grad_max(const GradSrc& a, int dtype, cudaStream_t st) {
    if (dtype == IMA_DTYPE_BF16) return launch_grad_max<IMA_DTYPE_BF16>(a, st);
    if (dtype == IMA_DTYPE_F16) return launch_grad_max<IMA_DTYPE_F16>(a, st);
    return launch_grad_max<IMA_DTYPE_F32>(a, st);
}

int run_grad_digits(const GradDigits& a, int dtype, int planes, cudaStream_t st) {
    if (dtype == IMA_DTYPE_BF16) return launch_grad_digits<IMA_DTYPE_BF16>(a, planes, st);
    if (dtype == IMA_DTYPE_F16) return launch_grad_digits<IMA_DTYPE_F16>(a, planes, st);
    return launch_grad_digits<IMA_DTYPE_F32>(a, planes, st);
}

void add_transpose(TransposeJobs& a, int& n, const int8_t* src, int64_t rows, int64_t cols, int64_t ld, int8_t* dst,
                   int64_t ldd) {
    a.src[n] = src; a.dst[n] = dst; a.rows[n] = rows; a.cols[n] = cols; a.ld[n] = ld; a.ldd[n] = ldd;
    const int64_t before = n ? a.end[n - 1] : 0;
    for (int i = n; i < 3; ++i) a.end[i] = before + (rows + 127) / 128 * ((cols + 127) / 128);
    ++n;
}

int run_transposes(const TransposeJobs& a, cudaStream_t st) {
    const int64_t blocks = std::max(a.end[2], std::min<int64_t>((a.zero_words + 255) / 256, 296));
    if (blocks == 0) return IMA_OK;
    if (blocks > INT32_MAX) return IMA_ERR_UNSUPPORTED;
    int8_transpose_kernel<<<(unsigned)blocks, 256, 0, st>>>(a);
    return IMA_LAUNCH_STATUS();
}

int run_quantize(const QuantRows& a, int dtype, cudaStream_t st) {
    if (dtype == IMA_DTYPE_BF16) return launch_quantize<IMA_DTYPE_BF16>(a, st);
    if (dtype == IMA_DTYPE_F16) return launch_quantize<IMA_DTYPE_F16>(a, st);
    return launch_quantize<IMA_DTYPE_F32>(a, st);
}

// Append a matrix to `a` (fewer than three so far, `n` of them).
int add_quantize(QuantRows& a, int& n, const void* x, int64_t M, int64_t ldx, int8_t* q, int64_t ldq, float* scale) {
    const int64_t K = a.K;
    if (M < 0 || K < 0) return IMA_ERR_INVALID_ARGUMENT;
    if (M > 0) {
        if (!scale || (K > 0 && (!x || !q || (M > 1 && ldx < K)))) return IMA_ERR_INVALID_ARGUMENT;
        if (ldq < K || ldq % 16 || (reinterpret_cast<uintptr_t>(q) & 15)) return IMA_ERR_INVALID_ARGUMENT;
    }
    a.x[n] = x; a.q[n] = q; a.scale[n] = scale; a.ldx[n] = ldx; a.ldq[n] = ldq;
    const int64_t before = n ? a.end[n - 1] : 0;
    for (int i = n; i < 3; ++i) a.end[i] = before + M;
    ++n;
    return IMA_OK;
}

}  // namespace

extern "C" {

int ima_int8_quantize_rows(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, int8_t* q, int64_t ldq,
                           float* scale, void* stream) {
    if (!known_dtype(x_dtype)) return IMA_ERR_INVALID_ARGUMENT;
    QuantRows a = {};
    a.K = K;
    int n = 0;
    const int rc = add_quantize(a, n, x, M, ldx, q, ldq, scale);
    return rc != IMA_OK ? rc : run_quantize(a, x_dtype, (cudaStream_t)stream);
}

int ima_int8_transpose(const int8_t* src, int64_t rows, int64_t cols, int64_t ld, int8_t* dst, int64_t ldd,
                       void* stream) {
    if (rows < 0 || cols < 0) return IMA_ERR_INVALID_ARGUMENT;
    if (rows == 0 || cols == 0) return IMA_OK;
    if (!src || !dst || ld < cols || ldd < rows || ldd % 16 || (reinterpret_cast<uintptr_t>(dst) & 15))
        return IMA_ERR_INVALID_ARGUMENT;
    TransposeJobs a = {};
    int n = 0;
    add_transpose(a, n, src, rows, cols, ld, dst, ldd);
    return run_transposes(a, (cudaStream_t)stream);
}

int ima_int8_pack_rows(const int8_t* a, int64_t rows_a, int64_t lda, int8_t* dst_a, const int8_t* b, int64_t rows_b,
                       int64_t ldb, int8_t* dst_b, int64_t cols, int64_t ldd, void* stream) {
    if (rows_a < 0 || rows_b < 0 || cols < 0) return IMA_ERR_INVALID_ARGUMENT;
    if (cols == 0 || rows_a + rows_b == 0) return IMA_OK;
    if (ldd % 16 || ldd < cols) return IMA_ERR_INVALID_ARGUMENT;
    if (rows_a > 0 && (!a || !dst_a || (rows_a > 1 && lda < cols) || (reinterpret_cast<uintptr_t>(dst_a) & 15)))
        return IMA_ERR_INVALID_ARGUMENT;
    if (rows_b > 0 && (!b || !dst_b || (rows_b > 1 && ldb < cols) || (reinterpret_cast<uintptr_t>(dst_b) & 15)))
        return IMA_ERR_INVALID_ARGUMENT;
    const PackRows p = {{a, b}, {dst_a, dst_b}, {lda, ldb}, {rows_a, rows_a + rows_b}, cols, ldd};
    const int64_t total = (rows_a + rows_b) * ((cols + 15) / 16);
    const unsigned grid = (unsigned)std::min<int64_t>((total + 255) / 256, 148 * 32);
    int8_pack_rows_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(p);
    return IMA_LAUNCH_STATUS();
}

}  // extern "C"
