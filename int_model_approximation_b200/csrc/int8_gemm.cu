// Products of 8-bit integer matrices on tcgen05 kind::i8, with the epilogues of the 8-bit linears.
//
//   I8_LINEAR     C = A B^T (int32, exact),  y = (fp32(C) s_m) t_n + b_n
//   I8_GATED      two products of one A:  h = act(g) u,  g = (fp32(A G^T) s_m) t^g_n + b^g_n, u likewise
//   I8_GATED_BWD  the same two products again, then with dh read in the epilogue
//                 D^g = dh u act'(g),  D^u = dh act(g)
//   I8_DIGIT      A in P base-256 digit planes (int8_quant.cu):  y = s_m sum_p 256^p (A_p B^T)
//
// Sums.  |C| <= 128 * 128 * K < 2^31 for K <= 131,071, the longest contraction accepted, so the
// int32 accumulators are exact; they, or the digits' accumulators together, are rounded to fp32 once.
//
// Tile and roles (persistent, 10 or 18 warps per CTA): a tile is 128 rows of A by BN rows of B.  A stage
// holds 128 bytes of K of the P planes of A and of the tile's rows of B, 128-byte swizzled.
//   warp 0    TMA producer;
//   warp 1    allocates tensor memory and issues the MMAs (one thread);
//   warps 2.. epilogue: warp w reads TMEM lanes 32 (w % 4) .. + 31 (one output row per thread) and
//             half (of 8 warps) or a quarter (of 16) of the tile's columns, and stores 64-byte row pieces
//             through shared memory, so that a warp store covers 8 rows of 64 contiguous bytes.
// Where two accumulators fit (P BN <= 256), the epilogue of a tile runs under the MMAs of the next.  The
// gated forms put 128 rows of G and 128 rows of U into one B tile: a single MMA of N = 256 forms g and u of
// the same 128 output columns, and A is read once for both.
//
// Measured.  Long contractions are bound by power: 16384 x 18944 x 3584 with its quantiser takes 0.74 to 0.79 ms (cards
// differ) in the first 20 ms after a pause, 0.92 after seconds of it, when the card draws 1 kW and clocks 1.24 GHz:
// 2.85e15 and 2.42e15 operations/s, 0.89 and 0.88 of twice the bf16 rates measured the same two ways.  The gated form
// takes 1.53 and 1.78 (2.91e15 and 2.50e15); with zeros for operands the kernel reaches 3.75e15.  Below 14 k-tiles or so the epilogue bounds: 4096 x 4864 x 896 to
// bf16 takes 25 us, its products alone 12; per 128 x 256 outputs it takes 5700 clocks, most of them in
// the shared-memory pipe (tensor memory out, staging in and out).  Small products are bound by the
// latency of launch, first loads and last epilogue, 8 us.
//
// Every wait is bounded: one that runs out records IMA_ERR_TIMEOUT, and every role drains and
// returns.
#pragma once
#include <cudaTypedefs.h>
#include <algorithm>
#include <atomic>
#include "sm100_pair.cuh"

namespace {

constexpr int I8_BM = 128;      // rows of A per CTA
constexpr int I8_KT = 128;      // bytes of K per stage: one 128-byte swizzle row
constexpr int64_t I8_MAX_K = 131071;

enum I8Epi { I8_LINEAR = 0, I8_GATED = 1, I8_GATED_BWD = 2, I8_DIGIT = 3 };
// Epilogue warps: the gradients of the gated block do 45 instructions per column where the others do 10 to
// 25, waiting for loads in between; with 8 warps they would take longer than the tile's MMAs.
constexpr int i8_epi_warps(int epi) { return epi == I8_GATED_BWD ? 16 : 8; }

template <int P, int BN, int CG, int EPI>
struct I8Cfg {
    static constexpr int EW = i8_epi_warps(EPI);
    static constexpr int THREADS = 64 + EW * 32;
    static constexpr int A_PLANE = I8_BM * I8_KT;
    static constexpr int B_BYTES = BN / CG * I8_KT;          // a CTA pair holds half of B each
    static constexpr int STAGE_BYTES = P * A_PLANE + B_BYTES;
    static constexpr int EPI_BYTES = EW * 2048 + EW * 128 * 8;   // output staging; scales and biases
    static constexpr int ROOM = (225 * 1024 - EPI_BYTES) / STAGE_BYTES;
    static constexpr int STAGES = ROOM < 6 ? ROOM : 6;
    static constexpr int ACC = P * BN;                       // tensor-memory columns of one tile
    static constexpr int BUFS = 2 * ACC <= 512 ? 2 : 1;
    static_assert(ACC <= 512, "accumulators exceed tensor memory");
    static constexpr int STG_OFFSET = STAGES * STAGE_BYTES;  // 2 KB of output staging per epilogue warp
    static constexpr int COL_OFFSET = STG_OFFSET + EW * 2048;    // 256 floats per epilogue warp (128 of 16 warps)
    static constexpr int BAR_OFFSET = STG_OFFSET + EPI_BYTES;
    static constexpr int TOTAL = BAR_OFFSET + (2 * STAGES + 2 * BUFS + 1) * 8 + 16;
    static constexpr int ALLOC = TOTAL + 1024;               // slack to align the base to 1024 B
    static_assert(ALLOC <= 227 * 1024, "shared memory per CTA");
};

struct __align__(64) I8Params {
    CUtensorMap ma, mb, mb2;        // A planes, B (or G), U
    int32_t* c;
    void* y;
    const float* xs;                // [M] row scales
    const float* ws[2];             // [N] column scales of B (or G) and U
    const void* bias[2];
    const void* dh;
    float* d;                       // I8_GATED_BWD: D^g, and D^u seg_pitch columns further
    uint32_t *row_max, *col_max;    // I8_GATED_BWD: maxima of |D t| by rows and |D s| by columns (NULL: none)
    void* y2;                       // I8_DIGIT: rows from split_row on go here (NULL: all to y)
    int64_t split_row, seg_rows;    // and of each part only seg_rows exist
    int64_t ldc, ldy, ldh, ldd, seg_pitch;
    int32_t* tail;                  // I8_DIGIT: sums of the tail tiles, [tile][plane][BN][rows], and their counters
    uint32_t* tail_count;           // [tile][CTA of the pair][epilogue warp]; both zero at launch
    int32_t full_tiles;             // tiles taken whole; each of the rest is split over tail_splits workers
    int32_t tail_splits;
    int32_t M, N, m_tiles, n_tiles, k_tiles, group_m;
    int32_t y_dtype, bias_dtype, dh_dtype, act, c_width, y_width;   // act: act_form() (I8_GATED_BWD: the activation); width: see stage_store
    int32_t dependent;              // launched while the kernel before it (a quantiser) still runs
    int32_t seg_tiles;              // I8_DIGIT: k-tiles of the first B; later ones read the second (mb2)
    uint64_t stall_ns;              // test knob (ima_set_gemm_wait_test); 0 in normal use
};

// Tile t -> (row tile, column tile): groups of group_m row tiles, rows fastest within a group, so
// that the tiles in flight share their k-slices of both operands in L2.
IMA_DEVINL void i8_tile(const I8Params& p, int32_t t, int32_t& mt, int32_t& nt) {
    const int32_t per_group = p.group_m * p.n_tiles, g = t / per_group, within = t - g * per_group;
    const int32_t gm = min(p.group_m, p.m_tiles - g * p.group_m);
    mt = g * p.group_m + within % gm;
    nt = within / gm;
}

// The work of one worker (a CTA, or a pair): whole tiles first, first + step, ..., then at most one part of
// the k-range of a tail tile.
struct I8Work {
    int32_t t, k0, k1;    // tile, k-tiles
    bool split;
    IMA_DEVINL bool get(const I8Params& p, int32_t i, int32_t first, int32_t step) {
        t = first + i * step;
        k0 = 0;
        k1 = p.k_tiles;
        split = false;
        if (t < p.full_tiles) return true;
        // the worker's item after its last whole tile
        if (p.tail_splits == 0 || (i > 0 && t - step >= p.full_tiles)) return false;
        const int32_t tail = first / p.tail_splits, part = first % p.tail_splits;
        t = p.full_tiles + tail;
        if (t >= p.m_tiles * p.n_tiles) return false;
        k0 = part * p.k_tiles / p.tail_splits;
        k1 = (part + 1) * p.k_tiles / p.tail_splits;
        split = true;
        return true;
    }
};

// ---------------------------------------------------------------------------
// activations and their derivatives, fp32
// ---------------------------------------------------------------------------
// An activation as the forward epilogues take it: IMA_ACT_..., with ACT_FINE for fp32 results.  Results of 16 bits take the
// hardware's 2^x for e^-|z|: off by 2^-22 + |z| 2^-24 of it, and 0 from |z| = 87 on, where the activation is below 2^-119.
// 4096 x 4864 x 896 takes 52.7 us to bf16 so, 57.6 with expf.
constexpr int ACT_FINE = 4;
inline int act_form(int activation, bool fine) { return activation + (fine ? ACT_FINE : 0); }

template <bool FINE>
IMA_DEVINL float exp_minus(float x) {   // e^-x, x >= 0
    if (FINE) return expf(-x);
    float t;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(x * -1.44269504f));
    return t;
}
// r = 1 / (1 + e^-z) and c = 1 - r, both from e^-|z|, so that neither cancels, overflows or divides by more than 2 (where
// the estimate of the reciprocal is off by a unit in the last place).
template <bool FINE>
IMA_DEVINL void sigmoid_both(float z, float& r, float& c) {
    const float t = exp_minus<FINE>(fabsf(z));
    float hi;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(hi) : "f"(1.0f + t));
    const float lo = t * hi;
    r = z < 0.0f ? lo : hi;
    c = z < 0.0f ? hi : lo;
}
// gelu_tanh(g) = g / (1 + e^-z) with z = 2 sqrt(2 / pi) (g + 0.044715 g^3); slope: z'.  Both quotients are 0
// or 1 from |g| = 13 on, where g may stop: its cube does not overflow.
IMA_DEVINL float gelu_tanh_z(float g, float& slope) {
    const float x = fminf(fmaxf(g, -32.0f), 32.0f), x2 = x * x;
    slope = 1.5957691f + 0.21406444f * x2;
    return x * (1.5957691f + 0.071354814f * x2);
}
template <int FORM>
IMA_DEVINL float act_value(float g) {
    constexpr int ACT = FORM % ACT_FINE;
    if (ACT == IMA_ACT_GELU) return 0.5f * g * erfcf(-0.70710678f * g);
    float r, c, slope, z = g;
    if (ACT == IMA_ACT_GELU_TANH) z = gelu_tanh_z(g, slope);
    sigmoid_both<(FORM >= ACT_FINE)>(z, r, c);
    return g * r;
}
// value a = act(g) and slope act'(g), as exact as fp32 results need for all types: the gradients are formed in fp32,
// and the estimate would save 0.5 % of a backward pass
template <int ACT>
IMA_DEVINL void act_both(float g, float& a, float& da) {
    if (ACT == IMA_ACT_GELU) {
        const float cdf = 0.5f * erfcf(-0.70710678f * g);
        a = g * cdf;
        da = cdf + g * 0.39894228f * expf(-0.5f * g * g);
    } else {
        float r, c, slope = 1.0f, z = g;
        if (ACT == IMA_ACT_GELU_TANH) z = gelu_tanh_z(g, slope);
        sigmoid_both<true>(z, r, c);
        a = g * r;
        da = r + a * c * slope;
    }
}
// f(integral_constant of the form); gelu has one, with erfc
template <typename F>
IMA_DEVINL void with_form(int form, F&& f) {
    if (form == IMA_ACT_SILU) f(std::integral_constant<int, IMA_ACT_SILU>{});
    else if (form == IMA_ACT_GELU_TANH) f(std::integral_constant<int, IMA_ACT_GELU_TANH>{});
    else if (form == IMA_ACT_SILU + ACT_FINE) f(std::integral_constant<int, IMA_ACT_SILU + ACT_FINE>{});
    else if (form == IMA_ACT_GELU_TANH + ACT_FINE) f(std::integral_constant<int, IMA_ACT_GELU_TANH + ACT_FINE>{});
    else f(std::integral_constant<int, IMA_ACT_GELU>{});
}

// Two fp32 values in one register pair, and arithmetic on both in one instruction; each rounds as the plain form does.
IMA_DEVINL uint64_t pair2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
IMA_DEVINL float2 halves(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
IMA_DEVINL uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
IMA_DEVINL uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
IMA_DEVINL uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Sums as fp32, rounded once.  A sum is written hi * 2^s + lo with parts that fp32 holds exactly, so that one fma rounds it.
// 0x4B000000 and 0x4B400000 are the bits of 2^23 and 1.5 * 2^23: an integer of up to 23 bits, added to them as
// bits, is a float after one subtraction.  The conversion instruction has an eighth of the multiplier's rate and
// took half of the epilogue's time; this form takes 2 integer and 1.5 floating instructions per value.
//   one plane:  s = 16
//   two planes: r0 + 2^8 r1.  |r1| <= 127 * 128 * 131071 leaves room for r0 >> 8 in 32 bits: t = r1 + (r0 >> 8),
//               the sum is 2^8 t + (r0 & 255); s = 17, and |t >> 9| < 2^22
//   three:      in 64 bits, below 2^47; s = 23
IMA_DEVINL void sum_parts(const int32_t (&r)[1], uint32_t& hi, uint32_t& lo) {
    hi = (uint32_t)((r[0] >> 16) + 0x4B400000);
    lo = __byte_perm((uint32_t)r[0], 0x4B000000u, 0x7610);
}
IMA_DEVINL void sum_parts(const int32_t (&r)[2], uint32_t& hi, uint32_t& lo) {
    const int32_t t = r[1] + (r[0] >> 8);
    hi = (uint32_t)((t >> 9) + 0x4B400000);
    lo = (__byte_perm((uint32_t)t, (uint32_t)r[0], 0x1104) & 0x1FFFFu) | 0x4B000000u;
}
template <int P>
IMA_DEVINL uint64_t sums_to_float2(const int32_t (&a)[P], const int32_t (&b)[P]) {
    if constexpr (P <= 2) {
        uint32_t ah, al, bh, bl;
        sum_parts(a, ah, al);
        sum_parts(b, bh, bl);
        const uint64_t hi = add2(pair2(__uint_as_float(ah), __uint_as_float(bh)), pair2(-12582912.0f, -12582912.0f));
        const uint64_t lo = add2(pair2(__uint_as_float(al), __uint_as_float(bl)), pair2(-8388608.0f, -8388608.0f));
        constexpr float S = P == 1 ? 65536.0f : 131072.0f;
        return fma2(hi, pair2(S, S), lo);
    } else {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int32_t(&r)[P] = e ? b : a;
            const int64_t s = ((int64_t)r[2] << 16) + ((int64_t)r[1] << 8) + r[0];
            const float lo = __uint_as_float(((uint32_t)s & 0x7FFFFFu) | 0x4B000000u) - 8388608.0f;
            f[e] = __fmaf_rn(__int2float_rn((int32_t)(s >> 23)), 8388608.0f, lo);
        }
        return pair2(f[0], f[1]);
    }
}

IMA_DEVINL uint64_t sum2(uint32_t a, uint32_t b) {
    const int32_t x[1] = {(int32_t)a}, y[1] = {(int32_t)b};
    return sums_to_float2<1>(x, y);
}

// (sum * x scale) * column scale + bias of four neighbouring columns
template <bool BIASED>
IMA_DEVINL void rescaled4(const uint32_t* sums, bool zero, uint64_t x2, const float* scale, const float* bias, float (&o)[4]) {
    const float4 w = *reinterpret_cast<const float4*>(scale);
    uint64_t a = mul2(mul2(zero ? 0ull : sum2(sums[0], sums[1]), x2), pair2(w.x, w.y));
    uint64_t b = mul2(mul2(zero ? 0ull : sum2(sums[2], sums[3]), x2), pair2(w.z, w.w));
    if (BIASED) {
        const float4 t = *reinterpret_cast<const float4*>(bias);
        a = add2(a, pair2(t.x, t.y));
        b = add2(b, pair2(t.z, t.w));
    }
    const float2 lo = halves(a), hi = halves(b);
    o[0] = lo.x; o[1] = lo.y; o[2] = hi.x; o[3] = hi.y;
}

IMA_DEVINL uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&b);
}
IMA_DEVINL uint32_t pack_f16(float lo, float hi) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}
IMA_DEVINL uint32_t pack_half2(float lo, float hi, int dtype) {
    return dtype == IMA_DTYPE_BF16 ? pack_bf16(lo, hi) : pack_f16(lo, hi);
}

// Staged rows out, W bytes a lane: 64 / W neighbouring lanes write one row's 64 bytes together.
template <int W>
IMA_DEVINL void stage_out(const unsigned char* st, int lane, unsigned char* base, int64_t pitch, int rows, int bytes,
                          int esize) {
    using Small = std::conditional_t<W == 4, uint32_t, uint16_t>;
    using T = std::conditional_t<W == 16, uint4, std::conditional_t<W == 8, uint2, Small>>;
    constexpr int ACROSS = 64 / W;
    const int o = lane % ACROSS * W, left = bytes - o;
#pragma unroll 4
    for (int it = 0; it < ACROSS; ++it) {
        const int r = it * (32 / ACROSS) + lane / ACROSS;
        if (r >= rows || left <= 0) continue;
        const unsigned char* src = st + r * 64 + (((o >> 4) ^ ((r >> 1) & 3)) << 4) + (o & 15);
        unsigned char* dst = base + r * pitch + o;
        if (left >= W) {
            *reinterpret_cast<T*>(dst) = *reinterpret_cast<const T*>(src);
        } else if (esize == 4) {
            for (int e = 0; e < left; e += 4) *reinterpret_cast<uint32_t*>(dst + e) = *reinterpret_cast<const uint32_t*>(src + e);
        } else {
            for (int e = 0; e < left; e += 2) *reinterpret_cast<uint16_t*>(dst + e) = *reinterpret_cast<const uint16_t*>(src + e);
        }
    }
}

// 64 bytes of each of a warp's 32 rows (w: this lane's row) through 2 KB of shared memory to
// base + row * pitch.  Slot j of row r lies at j ^ (r / 2 % 4), which keeps both sides free of bank
// conflicts.  `bytes` of each row and `rows` rows are written, `width` bytes (16, 8, 4 or 2, as the rows' alignment
// allows) by a lane, neighbouring lanes always side by side in a row: with lanes that write 16 bytes of their own
// row in pieces, a 3759 x 2116 x 1728 product to bf16 took 54 us, 69 at 2113 columns, so 30 and 38 (2112: 27).
IMA_DEVINL void stage_store(unsigned char* st, int lane, const uint32_t (&w)[16], unsigned char* base, int64_t pitch,
                            int rows, int bytes, int width, int esize) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint4*>(st + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
            make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    __syncwarp();
    if (width == 16 && rows == 32 && bytes >= 64) {   // all of it
        uint4 v[4];
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const int r = it * 8 + (lane >> 2);
            v[it] = *reinterpret_cast<const uint4*>(st + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
        }
        unsigned char* dst = base + (lane >> 2) * pitch + (lane & 3) * 16;
#pragma unroll
        for (int it = 0; it < 4; ++it) *reinterpret_cast<uint4*>(dst + it * 8 * pitch) = v[it];
    } else if (width == 16) stage_out<16>(st, lane, base, pitch, rows, bytes, esize);
    else if (width == 8) stage_out<8>(st, lane, base, pitch, rows, bytes, esize);
    else if (width == 4) stage_out<4>(st, lane, base, pitch, rows, bytes, esize);
    else stage_out<2>(st, lane, base, pitch, rows, bytes, esize);
}

// 32 fp32 values of this lane's row at column `col` of y, in y's type.
IMA_DEVINL void store_y32(const I8Params& p, unsigned char* st, int lane, const float (&v)[32], int64_t row0, int rows,
                          int32_t col, void* y_base) {
    unsigned char* y = reinterpret_cast<unsigned char*>(y_base);
    uint32_t w[16];
    if (p.y_dtype == IMA_DTYPE_F32) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(v[hf * 16 + j]);
            const int32_t c = col + hf * 16;
            stage_store(st, lane, w, y + (row0 * p.ldy + c) * 4, p.ldy * 4, rows, min(p.N - c, 16) * 4, p.y_width, 4);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
        if (p.y_dtype != IMA_DTYPE_BF16) {
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = pack_f16(v[2 * j], v[2 * j + 1]);
        }
        stage_store(st, lane, w, y + (row0 * p.ldy + col) * 2, p.ldy * 2, rows, min(p.N - col, 32) * 2, p.y_width, 2);
    }
}

template <int P, int BN, int EPI, int CG>
__global__ void __launch_bounds__(64 + 32 * i8_epi_warps(EPI), 1) int8_gemm_kernel(const __grid_constant__ I8Params p) {
    using L = I8Cfg<P, BN, CG, EPI>;
    constexpr bool PAIR = EPI == I8_GATED || EPI == I8_GATED_BWD;   // B tile = BN / 2 rows of G, then of U
    constexpr int TN = PAIR ? BN / 2 : BN;                          // output columns of a tile
    constexpr int HALF = TN / (L::EW / 4);                          // output columns of an epilogue warp
    constexpr int COLS = L::EW == 16 ? 128 : 256;                   // its scales and biases
    static_assert((PAIR ? 4 : 2) * HALF <= COLS, "scales and biases of an epilogue warp");
    // The gated forward forms spill a few registers: 5 loads and 4 stores per warp and tile whatever the activation, 0.1 to
    // 0.4 % of the instructions (counted for 256 and 4096 x 4864 x 896).
    extern __shared__ unsigned char i8_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(i8_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFFSET);
    uint64_t* empty = full + L::STAGES;
    uint64_t* acc_full = empty + L::STAGES;
    uint64_t* acc_empty = acc_full + L::BUFS;
    uint64_t* drained = acc_empty + L::BUFS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? cluster_ctarank() : 0;   // CTA of the pair; 0 issues its MMAs
    const int32_t first = (int32_t)(blockIdx.x / CG), step = (int32_t)(gridDim.x / CG);

    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < L::BUFS; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], L::EW * CG);
        }
        mbar_init(drained, 1);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        if (CG == 2) {
            tmem_alloc_pair(tmem_slot, 512);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(tmem_slot, 512);
            tmem_relinquish();
        }
    }
    __syncthreads();
    if (CG == 2) cluster_sync_all();   // both CTAs' barriers exist before either signals the other's
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (p.dependent) wait_previous_kernel();   // codes and scales are complete

    if (warp == 0 && lane == 0) {
        // ---------------- TMA producer ----------------
        uint32_t stage = 0, phase = 0;
        uint64_t issued = 0;
        I8Work w;
        for (int32_t i = 0; !*abort_flag && w.get(p, i, first, step); ++i) {
            int32_t mt, nt;
            i8_tile(p, w.t, mt, nt);
            for (int kt = w.k0; kt < w.k1; ++kt) {
                if (!mbar_wait_or_abort(&empty[stage], phase ^ 1u, abort_flag, IMA_WAIT_LIMIT_NS, IMA_WHERE_INT8_GEMM,
                                        (int)stage))
                    break;
                ++issued;
                unsigned char* sb = smem + stage * L::STAGE_BYTES;
                unsigned char* bb = sb + P * L::A_PLANE;
                const bool second = EPI == I8_DIGIT && kt >= p.seg_tiles;
                const int32_t bx = (second ? kt - p.seg_tiles : kt) * I8_KT;
                if constexpr (CG == 1) {
                    mbar_arrive_expect_tx(&full[stage], (uint32_t)L::STAGE_BYTES);
#pragma unroll
                    for (int pl = 0; pl < P; ++pl)
                        tma_load_3d(sb + pl * L::A_PLANE, &p.ma, &full[stage], kt * I8_KT, mt * I8_BM, pl);
                    tma_load_2d(bb, second ? &p.mb2 : &p.mb, &full[stage], bx, nt * TN);
                    if (PAIR) tma_load_2d(bb + TN * I8_KT, &p.mb2, &full[stage], bx, nt * TN);
                } else {
                    // both CTAs' loads count on the barrier of CTA 0, whose MMA thread waits for them; the
                    // stage is free in both (a commit of that thread), so its barrier is in this round's phase
                    const uint32_t bar = cluster_map(&full[stage], 0);
                    if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2u * (uint32_t)L::STAGE_BYTES);
#pragma unroll
                    for (int pl = 0; pl < P; ++pl)
                        tma_load_3d_pair(sb + pl * L::A_PLANE, &p.ma, bar, kt * I8_KT, (mt * 2 + (int)rank) * I8_BM, pl);
                    if (PAIR)
                        tma_load_2d_pair(bb, rank ? &p.mb2 : &p.mb, bar, bx, nt * TN);
                    else
                        tma_load_2d_pair(bb, second ? &p.mb2 : &p.mb, bar, bx, nt * TN + (int)rank * (BN / 2));
                }
                if (++stage == (uint32_t)L::STAGES) { stage = 0; phase ^= 1u; }
            }
        }
        // Every load issued lands before the CTA exits, also after an abort; in a pair, the commits
        // that free this CTA's stages have arrived as well.
        for (int s = 0; s < L::STAGES; ++s) {
            const uint64_t rounds = issued / L::STAGES + ((uint64_t)s < issued % L::STAGES ? 1u : 0u);
            if (rounds > 0 && rank == 0)
                mbar_wait_bounded(&full[s], (uint32_t)((rounds - 1) & 1u), IMA_WHERE_INT8_GEMM, 100 + s);
            if (CG == 2 && rounds > 0 && !*abort_flag)
                mbar_wait_or_abort(&empty[s], (uint32_t)((rounds - 1) & 1u), abort_flag, IMA_WAIT_LIMIT_NS,
                                   IMA_WHERE_INT8_GEMM, 150 + s);
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {
        // ---------------- MMA issuer ----------------
        constexpr uint32_t idesc = idesc_i8(I8_BM * CG, BN);
        uint32_t stage = 0, phase = 0, buf = 0, bphase = 0;
        if (p.stall_ns)   // test knob: a wait that nothing ends runs out
            mbar_wait_or_abort(drained, 0u, abort_flag, p.stall_ns, IMA_WHERE_INT8_GEMM, -2);
        I8Work w;
        for (int32_t i = 0; !*abort_flag && w.get(p, i, first, step); ++i) {
            if (!mbar_wait_or_abort(&acc_empty[buf], bphase ^ 1u, abort_flag, IMA_WAIT_LIMIT_NS, IMA_WHERE_INT8_GEMM, -1))
                break;
            tc_fence_after();
            const uint32_t acc = tmem_base + buf * L::ACC;
            bool fed = true;
            for (int kt = w.k0; kt < w.k1; ++kt) {
                if (!mbar_wait_or_abort(&full[stage], phase, abort_flag, IMA_WAIT_LIMIT_NS, IMA_WHERE_INT8_GEMM,
                                        50 + (int)stage)) {
                    fed = false;
                    break;
                }
                tc_fence_after();
                const uint32_t sa = smem_u32(smem + stage * L::STAGE_BYTES);
                const uint32_t sb = sa + P * L::A_PLANE;
#pragma unroll
                for (int ks = 0; ks < I8_KT / 32; ++ks)
#pragma unroll
                    for (int pl = 0; pl < P; ++pl) {
                        const uint64_t da = umma_desc_sw128_kmajor(sa + pl * L::A_PLANE + ks * 32);
                        const uint64_t db = umma_desc_sw128_kmajor(sb + ks * 32);
                        if (CG == 2) mma_i8_pair(acc + pl * BN, da, db, idesc, (kt > w.k0 || ks) ? 1u : 0u);
                        else mma_i8(acc + pl * BN, da, db, idesc, (kt > w.k0 || ks) ? 1u : 0u);
                    }
                if (CG == 2) mma_commit_pair(&empty[stage]);
                else mma_commit(&empty[stage]);
                if (++stage == (uint32_t)L::STAGES) { stage = 0; phase ^= 1u; }
            }
            if (!fed) break;
            if (CG == 2) mma_commit_pair(&acc_full[buf]);
            else mma_commit(&acc_full[buf]);
            if (++buf == (uint32_t)L::BUFS) { buf = 0; bphase ^= 1u; }
        }
        // Every MMA issued completes before the CTA frees tensor memory.
        if (CG == 2) mma_commit_pair_local(drained);
        else mma_commit(drained);
        mbar_wait_bounded(drained, 0u, IMA_WHERE_INT8_GEMM, -3);
    } else if (warp >= 2) {
        // ---------------- epilogue ----------------
        const int ew = warp - 2, q = warp & 3, h = ew >> 2;
        unsigned char* st = smem + L::STG_OFFSET + ew * 2048;
        float* cols = reinterpret_cast<float*>(smem + L::COL_OFFSET) + ew * COLS;
        uint32_t buf = 0, bphase = 0;
        // this warp's column scales and biases, [2 operands][scale, bias][HALF] in shared memory, and its lane's row
        // scale: loaded one tile ahead where registers allow (16 warps have 96 each, and hide the loads anyway)
        constexpr bool AHEAD = EPI != I8_GATED_BWD;
        constexpr int OPS = PAIR ? 2 : 1, EACH = EPI == I8_DIGIT ? 0 : HALF / 32;
        float ahead[OPS * 2 * EACH + 1], xs_ahead = 0.0f;
        auto fetch = [&](const I8Work& w, int32_t& mt, int32_t& nt) {
            i8_tile(p, w.t, mt, nt);
            const int64_t row = ((int64_t)mt * CG + rank) * I8_BM + q * 32 + lane;
            xs_ahead = row < p.M && p.xs ? p.xs[row] : 0.0f;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int32_t n = nt * TN + h * HALF + i * 32 + lane;
#pragma unroll
                for (int o = 0; o < OPS; ++o) {
                    ahead[(2 * o) * EACH + i] = n < p.N && p.ws[o] ? p.ws[o][n] : 0.0f;
                    // no bias is -0, which changes no sum
                    ahead[(2 * o + 1) * EACH + i] =
                        n < p.N && p.bias[o] ? load_as_f32(p.bias[o], p.bias_dtype, n) : -0.0f;
                }
            }
        };
        I8Work wk, next;
        int32_t mt = 0, nt = 0, mt_next = 0, nt_next = 0;
        bool more = wk.get(p, 0, first, step);
        if (AHEAD && more) fetch(wk, mt, nt);
        for (int32_t item = 0; more; ++item) {
            if (!AHEAD) fetch(wk, mt, nt);
            const int64_t row0 = ((int64_t)mt * CG + rank) * I8_BM + q * 32;
            const int rows = (int)max((int64_t)0, min((int64_t)32, (int64_t)p.M - row0));
            const int32_t n0 = nt * TN + h * HALF;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < OPS * 2 * EACH; ++i) cols[i * 32 + lane] = ahead[i];
            const float xs = xs_ahead;
            if (AHEAD) {
                more = next.get(p, item + 1, first, step);
                if (more) fetch(next, mt_next, nt_next);
            }
            const bool ok = mbar_wait_or_abort(&acc_full[buf], bphase, abort_flag, IMA_WAIT_LIMIT_NS,
                                               IMA_WHERE_INT8_GEMM, 200);
            __syncwarp();
            if (!__all_sync(0xFFFFFFFFu, ok)) { *abort_flag = 1; break; }
            tc_fence_after();
            const uint32_t tq = tmem_base + ((uint32_t)(q * 32) << 16) + buf * L::ACC + h * HALF;
            const bool zero = p.k_tiles == 0;   // K == 0: no MMA wrote the accumulators
            const uint64_t x2 = pair2(xs, xs);
            if constexpr (EPI == I8_LINEAR) {
#pragma unroll 1
                for (int c0 = 0; c0 < HALF; c0 += 32) {
                    uint32_t r[32];
                    tmem_ld32(tq + c0, r);
                    tmem_wait_ld();
                    if (zero) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) r[j] = 0;
                    }
                    if (n0 + c0 >= p.N || rows == 0) continue;
                    if (p.c) {
                        uint32_t w[16];
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) w[j] = r[hf * 16 + j];
                            const int32_t c = n0 + c0 + hf * 16;
                            stage_store(st, lane, w, reinterpret_cast<unsigned char*>(p.c + row0 * p.ldc + c),
                                        p.ldc * 4, rows, min(p.N - c, 16) * 4, p.c_width, 4);
                        }
                    }
                    if (p.y) {
                        float v[32];
                        auto scaled = [&](auto with_bias) {
#pragma unroll
                            for (int j = 0; j < 32; j += 4) {
                                float f[4];
                                rescaled4<decltype(with_bias)::value>(r + j, false, x2, cols + c0 + j, cols + HALF + c0 + j, f);
#pragma unroll
                                for (int e = 0; e < 4; ++e) v[j + e] = f[e];
                            }
                        };
                        if (p.bias[0]) scaled(std::true_type{});
                        else scaled(std::false_type{});
                        store_y32(p, st, lane, v, row0, rows, n0 + c0, p.y);
                    }
                }
            } else if constexpr (EPI == I8_GATED) {
                auto chunks = [&](auto tag, auto with_bias) {
                    constexpr int ACT = decltype(tag)::value;
                    constexpr bool BIASED = decltype(with_bias)::value;
#pragma unroll 1
                    for (int c0 = 0; c0 < HALF; c0 += 32) {
                        uint32_t rg[32], ru[32];
                        tmem_ld32(tq + c0, rg);
                        tmem_ld32(tq + TN + c0, ru);
                        tmem_wait_ld();
                        if (n0 + c0 >= p.N || rows == 0) continue;
                        float v[32];
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            float g[4], u[4];
                            rescaled4<BIASED>(rg + j, zero, x2, cols + c0 + j, cols + HALF + c0 + j, g);
                            rescaled4<BIASED>(ru + j, zero, x2, cols + 2 * HALF + c0 + j, cols + 3 * HALF + c0 + j, u);
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[j + e] = act_value<ACT>(g[e]) * u[e];
                        }
                        store_y32(p, st, lane, v, row0, rows, n0 + c0, p.y);
                    }
                };
                auto both = [&](auto tag) {
                    if (p.bias[0] || p.bias[1]) chunks(tag, std::true_type{});
                    else chunks(tag, std::false_type{});
                };
                with_form(p.act, both);
            } else if constexpr (EPI == I8_GATED_BWD) {
                uint32_t rm = 0;
                auto chunks = [&](auto tag) {
                    constexpr int ACT = decltype(tag)::value;
#pragma unroll 1
                    for (int c0 = 0; c0 < HALF; c0 += 16) {
                        uint32_t rg[16], ru[16];
                        tmem_ld16(tq + c0, rg);
                        tmem_ld16(tq + TN + c0, ru);
                        const int32_t n = n0 + c0;
                        float dh[16];
                        if (lane < rows && n < p.N) {
                            const unsigned char* src = reinterpret_cast<const unsigned char*>(p.dh) +
                                                       ((row0 + lane) * p.ldh + n) * dtype_bytes(p.dh_dtype);
                            const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
                            float a[8], b[8];
                            load8(src, p.dh_dtype, 0, p.N - n, vec, a);
                            load8(src, p.dh_dtype, 8, p.N - n, vec, b);
#pragma unroll
                            for (int j = 0; j < 8; ++j) { dh[j] = a[j]; dh[8 + j] = b[j]; }
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; ++j) dh[j] = 0.0f;
                        }
                        tmem_wait_ld();
                        if (n >= p.N || rows == 0) continue;
                        uint32_t wg[16], wu[16], cm = 0;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            // the conversion instruction: 16 warps hide it, and the two-value form needs
                            // registers that they do not have (477 us for 4096 x 18944 x 3584, 445 so)
                            const float g0 = zero ? 0.0f : __int2float_rn((int32_t)rg[j]);
                            const float u0 = zero ? 0.0f : __int2float_rn((int32_t)ru[j]);
                            const float g = __fadd_rn(__fmul_rn(__fmul_rn(g0, xs), cols[c0 + j]), cols[HALF + c0 + j]);
                            const float u = __fadd_rn(__fmul_rn(__fmul_rn(u0, xs), cols[2 * HALF + c0 + j]),
                                                      cols[3 * HALF + c0 + j]);
                            float a, da;
                            act_both<ACT>(g, a, da);
                            const float dg = dh[j] * u * da, du = dh[j] * a;
                            wg[j] = __float_as_uint(dg);
                            wu[j] = __float_as_uint(du);
                            // maxima of the bit patterns of magnitudes: order like the values, NaN above all
                            rm = max(rm, max(__float_as_uint(fabsf(__fmul_rn(dg, cols[c0 + j]))),
                                             __float_as_uint(fabsf(__fmul_rn(du, cols[2 * HALF + c0 + j])))));
                            if (p.col_max) {
                                const uint32_t mg = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(fabsf(__fmul_rn(dg, xs))));
                                const uint32_t mu = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(fabsf(__fmul_rn(du, xs))));
                                cm = lane == j ? mg : (lane == 16 + j ? mu : cm);
                            }
                        }
                        if (p.col_max && n + (lane & 15) < p.N)
                            atomicMax(p.col_max + n + (lane & 15) + (lane >= 16 ? p.seg_pitch : 0), cm);
                        float* d = p.d + row0 * p.ldd + n;
                        stage_store(st, lane, wg, reinterpret_cast<unsigned char*>(d), p.ldd * 4, rows, min(p.N - n, 16) * 4,
                                    16, 4);
                        stage_store(st, lane, wu, reinterpret_cast<unsigned char*>(d + p.seg_pitch), p.ldd * 4, rows,
                                    min(p.N - n, 16) * 4, 16, 4);
                    }
                };
                if (p.act == IMA_ACT_SILU) chunks(std::integral_constant<int, IMA_ACT_SILU>{});
                else if (p.act == IMA_ACT_GELU) chunks(std::integral_constant<int, IMA_ACT_GELU>{});
                else chunks(std::integral_constant<int, IMA_ACT_GELU_TANH>{});
                if (p.row_max && lane < rows) atomicMax(p.row_max + row0 + lane, rm);
            } else {
                // the second part's rows start on a multiple of 128: a warp's 32 rows lie in one part
                const bool second = p.y2 && row0 >= p.split_row;
                const int64_t out_row = second ? row0 - p.split_row : row0;
                const int out_rows = p.y2 ? (int)max((int64_t)0, min((int64_t)rows, p.seg_rows - out_row)) : rows;
                void* out = second ? p.y2 : p.y;
                bool store = true;
                int32_t* sums = nullptr;   // this warp's rows and columns of a split tile: [plane][column][row]
                if (wk.split) {
                    // exact sums in any order; the last worker to add to this warp's part writes it out
                    sums = p.tail + (((int64_t)(wk.t - p.full_tiles) * P * BN + h * HALF) * CG + rank) * I8_BM + q * 32 + lane;
#pragma unroll 1
                    for (int c0 = 0; c0 < HALF; c0 += 32)
#pragma unroll 1
                        for (int i = 0; i < P; ++i) {
                            uint32_t r[32];
                            tmem_ld32(tq + i * BN + c0, r);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                atomicAdd(sums + (int64_t)(i * BN + c0 + j) * CG * I8_BM, (int32_t)r[j]);
                        }
                    __threadfence();
                    __syncwarp();
                    uint32_t before = 0;
                    if (lane == 0)
                        before = atomicAdd(p.tail_count + ((wk.t - p.full_tiles) * CG + rank) * L::EW + ew, 1u);
                    store = __shfl_sync(0xFFFFFFFFu, before, 0) + 1 == (uint32_t)p.tail_splits;
                    __threadfence();
                }
#pragma unroll 1
                for (int c0 = 0; c0 < HALF && store; c0 += 32) {
                    uint32_t r[P][32];
                    if (wk.split) {
#pragma unroll
                        for (int i = 0; i < P; ++i)
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                r[i][j] = load_l2(sums + (int64_t)(i * BN + c0 + j) * CG * I8_BM);
                    } else {
#pragma unroll
                        for (int i = 0; i < P; ++i) tmem_ld32(tq + i * BN + c0, r[i]);
                        tmem_wait_ld();
                    }
                    if (n0 + c0 >= p.N || out_rows <= 0) continue;
                    float v[32];
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        int32_t a[P], b[P];
#pragma unroll
                        for (int i = 0; i < P; ++i) { a[i] = (int32_t)r[i][j]; b[i] = (int32_t)r[i][j + 1]; }
                        const float2 f = halves(mul2(zero ? 0ull : sums_to_float2<P>(a, b), x2));
                        v[j] = f.x; v[j + 1] = f.y;
                    }
                    store_y32(p, st, lane, v, out_row, out_rows, n0 + c0, out);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 2) mbar_arrive_cluster(cluster_map(&acc_empty[buf], 0));
                else mbar_arrive(&acc_empty[buf]);
            }
            if (++buf == (uint32_t)L::BUFS) { buf = 0; bphase ^= 1u; }
            if (AHEAD) {
                wk = next; mt = mt_next; nt = nt_next;
            } else {
                more = wk.get(p, item + 1, first, step);
            }
        }
    }
    __syncthreads();
    if (CG == 2) cluster_sync_all();   // no CTA leaves while the other may still signal or use its memory
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        if (CG == 2) tmem_dealloc_pair(tmem_base, 512);
        else tmem_dealloc(tmem_base, 512);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Map over [planes][rows][K] bytes (row pitch ld, planes plane_stride apart; 0: a matrix) with a {128 B,
// box_rows(, 1)} box, 128-byte swizzle.
int make_i8_map(CUtensorMap* map, const int8_t* base, int64_t K, int64_t ld, int64_t rows, int planes,
                int64_t plane_stride, int box_rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)K, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)ld, (cuuint64_t)plane_stride};
    const cuuint32_t box[3] = {(cuuint32_t)I8_KT, (cuuint32_t)box_rows, 1};
    return encode_bytes(map, plane_stride ? 3 : 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Allow `kern` its dynamic shared memory, once per device (a bit each for the first 64).
int set_smem_once(std::atomic<uint64_t>& ready, const void* kern, int bytes) {
    int dev = 0;
    int rc = ima_note_cuda(cudaGetDevice(&dev));
    if (rc != IMA_OK) return rc;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (ready.load(std::memory_order_acquire) & bit) return IMA_OK;
    rc = ima_note_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (rc == IMA_OK) ready.fetch_or(bit, std::memory_order_release);
    return rc;
}

// An int8 operand as the loads need it: 16-byte aligned rows of at least K bytes.
int check_i8_operand(const int8_t* p, int64_t rows, int64_t K, int64_t ld) {
    if (rows < 0 || K < 0) return IMA_ERR_INVALID_ARGUMENT;
    if (K > 0 && rows > 0 && !p) return IMA_ERR_INVALID_ARGUMENT;
    if (ld < K || ld % 16 || (reinterpret_cast<uintptr_t>(p) & 15)) return IMA_ERR_INVALID_ARGUMENT;
    if (rows > INT32_MAX / 2 || ld > INT32_MAX || K > I8_MAX_K) return IMA_ERR_UNSUPPORTED;
    return IMA_OK;
}


// Rows of B in a load box: a CTA's share of a tile, of each operand in the gated forms.
template <int BN, int EPI, int CG>
constexpr int i8_box_rows() { return EPI == I8_GATED || EPI == I8_GATED_BWD ? BN / 2 : BN / CG; }

struct I8Operands {
    const int8_t *a, *b, *b2;
    int64_t lda, ldb, ldb2, Ka, K;   // A has Ka columns per plane, B and b2 K
    int64_t a_planes;                // bytes between the planes of A
};

// Tail tiles of a digit product that the workspace of a backward pass has room for (I8_TAIL_BYTES), and
// the bytes that `tiles` of them take: their sums and counters.
constexpr int64_t I8_TAIL_BYTES = 24ll << 20;
template <int P, int BN>
int64_t tail_bytes(int cg, int64_t tiles) { return tiles * cg * ((int64_t)P * BN * I8_BM * 4 + i8_epi_warps(I8_DIGIT) * 4); }
template <int P, int BN>
int64_t tail_tiles(int cg) { return I8_TAIL_BYTES / tail_bytes<P, BN>(cg, 1); }

template <int P, int BN, int EPI, int CG>
int launch_i8_tile(I8Params& p, const I8Operands& o, cudaStream_t stream) {
    using L = I8Cfg<P, BN, CG, EPI>;
    constexpr int TN = EPI == I8_GATED || EPI == I8_GATED_BWD ? BN / 2 : BN;
    constexpr int BOX = i8_box_rows<BN, EPI, CG>();
    p.m_tiles = (p.M + CG * I8_BM - 1) / (CG * I8_BM);
    p.n_tiles = (p.N + TN - 1) / TN;
    p.k_tiles = (int32_t)((o.Ka + I8_KT - 1) / I8_KT);
    p.group_m = 16 / CG;
    p.stall_ns = g_gemm_stall_ns;
    int rc = IMA_OK;
    if (o.K > 0) {   // K == 0 loads nothing
        rc = make_i8_map(&p.ma, o.a, o.Ka, o.lda, p.M, P, o.a_planes, I8_BM);
        if (rc == IMA_OK) rc = make_i8_map(&p.mb, o.b, o.K, o.ldb, p.N, 1, 0, BOX);
        if (rc == IMA_OK && o.b2) rc = make_i8_map(&p.mb2, o.b2, o.K, o.ldb2, p.N, 1, 0, BOX);
        if (rc != IMA_OK) return rc;
    }
    const int64_t all = (int64_t)p.m_tiles * p.n_tiles, workers = std::max<int64_t>(1, gemm_grid_limit() / CG);
    if (all > INT32_MAX - workers) return IMA_ERR_UNSUPPORTED;   // tiles are counted in 32 bits
    p.full_tiles = (int32_t)all;
    p.tail_splits = 0;
    if (EPI == I8_DIGIT && p.tail && all > workers) {
        // a last round that fills less than 5/8 of the machine: its tiles split over all workers (at least 8 k-tiles
        // each, and at most 16 of them per tile, whose sums meet in L2)
        const int64_t rest = all % workers;
        const int64_t splits = rest ? std::min<int64_t>(std::min<int64_t>(workers / rest, 16), p.k_tiles / 8) : 0;
        if (rest * 8 <= workers * 5 && splits >= 2 && rest <= tail_tiles<P, BN>(CG)) {
            p.full_tiles = (int32_t)(all - rest);
            p.tail_splits = (int32_t)splits;
            rc = ima_note_cuda(cudaMemsetAsync(p.tail, 0, tail_bytes<P, BN>(CG, rest), stream));
            if (rc != IMA_OK) return rc;
            p.tail_count = reinterpret_cast<uint32_t*>(p.tail + rest * P * BN * CG * I8_BM);
        }
    }
    auto kern = int8_gemm_kernel<P, BN, EPI, CG>;
    static std::atomic<uint64_t> ready{0};
    rc = set_smem_once(ready, (const void*)kern, L::ALLOC);
    if (rc != IMA_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(std::min<int64_t>(all, workers) * CG));
    cfg.blockDim = dim3(L::THREADS);
    cfg.dynamicSmemBytes = L::ALLOC;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (CG == 2) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = CG;
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

// Tile forms: a CTA pair (256 rows, each CTA holds half of B), one CTA, or one CTA with half the columns.  Per
// unit of work the pair loads least (L2 to SM is 64 bytes a clock and SM), the small tile most; the small one fills the
// machine with few tiles, ends a last round sooner, and with two digit planes has room for a second accumulator, so that
// the epilogue of a tile runs during the products of the next.
struct TilePlan {
    double ns;
    int bn, cg;
};

// Time of a form in ns, fitted to 160 measured times of 40 products of 128 to 16384 rows, and within 15 % of those
// with one plane.  A k-tile takes the tensor core 2 clocks per plane and column, and its loads 1 per 64 bytes; measured,
// the wide pair needs 650 and the wide CTA 720 clocks with one plane, 1065 and 1100 with two.  The epilogue of a tile
// takes 22 to 24 clocks per column (two planes 27, three 80, the gated gradients 35), behind the products of the
// next tile where two accumulators fit.  3.5 us from launch to the first products, 0.6 more for a cluster; 1 more after a
// quantiser, whose end the split form awaits with its weights already on their way.
inline double tile_ns(int64_t M, int64_t N, int64_t k_steps, int planes, int epi, int bn, int cg, bool tail,
                      bool dependent) {
    const bool pair = epi == I8_GATED || epi == I8_GATED_BWD;
    const int64_t tn = pair ? bn / 2 : bn, tiles = ((M + cg * I8_BM - 1) / (cg * I8_BM)) * ((N + tn - 1) / tn);
    const int64_t workers = std::max<int64_t>(1, gemm_grid_limit() / cg);
    const double step = planes == 3 ? 850.0 : planes == 2 ? (bn == 128 ? 800.0 : cg == 2 ? 1065.0 : 1100.0)
                                                          : (bn == 128 ? 530.0 : cg == 2 ? 650.0 : 720.0);
    const double products = (double)k_steps * step;
    const double epilogue = (double)(std::min(tn, N) * (pair ? 2 : 1)) *
                            (epi == I8_GATED_BWD ? 35.0 : planes == 1 ? 20.0 + 2.0 * cg : planes == 2 ? 27.0 : 80.0);
    int64_t rounds = (tiles + workers - 1) / workers;
    double extra = 0.0;
    const int64_t rest = tiles % workers;
    if (tail && rounds > 1 && rest && rest * 8 <= workers * 5) {   // the last round's tiles are split over all workers
        rounds -= 1;
        extra = products * (double)rest / (double)workers + 2.0 * epilogue;
    }
    const double clocks = 2 * planes * bn <= 512
        ? products + (double)(rounds - 1) * std::max(products, epilogue) + epilogue
        : (double)rounds * (products + epilogue);
    const double streams = (double)((N * (pair ? 2 : 1) + M * planes) * k_steps * I8_KT) / 4700.0;
    return std::max((clocks + extra) / 1.77, streams) + (cg == 2 ? 4100.0 : 3500.0) + (dependent ? 1000.0 : 0.0);
}

template <int P, int EPI>
TilePlan tile_plan(int64_t M, int64_t N, int64_t k_steps, bool tail, bool dependent) {
    constexpr int WIDE = P == 3 ? 128 : 256;
    TilePlan best = {tile_ns(M, N, k_steps, P, EPI, WIDE, 1, tail, dependent), WIDE, 1};
    auto consider = [&](int bn, int cg) {
        const double ns = tile_ns(M, N, k_steps, P, EPI, bn, cg, tail, dependent);
        if (ns < best.ns) best = {ns, bn, cg};
    };
    if (gemm_grid_limit() >= 2) consider(WIDE, 2);
    if (P < 3 && EPI != I8_GATED_BWD) consider(128, 1);
    return best;
}

template <int P, int EPI>
int launch_i8(I8Params& p, const I8Operands& o, const TilePlan& t, cudaStream_t stream) {
    constexpr int WIDE = P == 3 ? 128 : 256;
    if (t.cg == 2) return launch_i8_tile<P, WIDE, EPI, 2>(p, o, stream);
    if constexpr (P < 3 && EPI != I8_GATED_BWD) {
        if (t.bn == 128) return launch_i8_tile<P, 128, EPI, 1>(p, o, stream);
    }
    return launch_i8_tile<P, WIDE, EPI, 1>(p, o, stream);
}

}  // namespace
