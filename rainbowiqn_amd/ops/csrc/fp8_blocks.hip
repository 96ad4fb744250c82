// 8-bit block matrices for gfx950: e4m3 values with one power-of-two scale per
// block of 128 columns and 1 or 128 rows, their products, and the backward
// pass of a linear layer whose input is kept in that form.
//
// Layout of a matrix [R, C] with nb = ceil(C / 128):
//   q     [R, 128 nb]            e4m3 bytes, zeros behind column C
//   scale [R or ceil(R/128), S]  e8m0 bytes (e + 127), S = nb rounded up to 4
// A value stands for q 2^e.  e = floor(log2(amax)) - 7 over the block's finite
// values (0 for a block of zeros, at least -127), so |x| 2^-e < 256 stays
// inside e4m3's 448 and every scale is a power of two: scaling is exact, and
// the only rounding is the one to 4 significant bits (nearest, ties to even).
// Values that are not finite become e4m3's NaN and leave the scale alone.
//
// Products are exact and sums fp32 wherever the caller does not ask for less.
// e4m3 times a power of two is exact in bf16, and bf16 products are summed in
// full: expanding the operands (v_cvt_scalef32_pk_bf16_fp8, two values and
// their scale an instruction) costs half the peak rate and nothing in precision.
// The scaled 8-bit instruction keeps less: it sums products in groups of 8 and
// cuts each to a multiple of 2^(E - 13), E the group's largest sum of
// exponents.  Sums of random terms end some 1e-5 of their size off, sums of
// terms that cancel may lose all that is left.  It runs only where `exact` is 0
// and the result has 16 bits.
#include "common.h"
#include "riqn_kernels.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <type_traits>

namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(2))) int i32x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) short s16x4;

struct bf16_t { unsigned short v; };
struct fp16_t { _Float16 v; };
DEV float to_f(float x) { return x; }
DEV float to_f(bf16_t x) { return bf16_to_f32(x.v); }
DEV float to_f(fp16_t x) { return (float)x.v; }
template <typename T> DEV T from_f(float x);
template <> DEV float from_f<float>(float x) { return x; }
template <> DEV bf16_t from_f<bf16_t>(float x) {
    // the integer rounding of f32_to_bf16 would carry a NaN into infinity
    return bf16_t{__builtin_bit_cast(unsigned short, (__bf16)x)};
}
template <> DEV fp16_t from_f<fp16_t>(float x) { return fp16_t{(_Float16)x}; }

// relu and the truth value that its gradient goes by; NaN passes both
DEV bool passes(float z) { return !(z <= 0.0f); }

// 2^e for e in [-126, 127]
DEV float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

DEV int block_exp(float amax) {
    if (amax <= 0.0f) return 0;
    return max((int)(__float_as_uint(amax) >> 23) - 134, -127);
}

// max over each group of 16 lanes, in every lane of it
template <int N>
DEV float ror16_max(float v) {
    int o = __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf,
                                        0xf, false);
    return fmaxf(v, __int_as_float(o));
}
DEV float max16(float v) {
    v = ror16_max<8>(v);
    v = ror16_max<4>(v);
    v = ror16_max<2>(v);
    return ror16_max<1>(v);
}

DEV float finite_abs(float x) {
    const float a = fabsf(x);
    return a < __builtin_inff() ? a : 0.0f;  // false for NaN too
}

// 8 scaled values -> 8 e4m3 bytes
DEV i32x2 pack8(const float* v, float inv) {
    i32x2 r;
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] * inv,
                                                v[4 * i + 1] * inv, 0, false);
        r[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] * inv,
                                               v[4 * i + 3] * inv, w, true);
    }
    return r;
}

// 8 consecutive values of a row, zeros behind column C.  VEC: every 8th
// element of every row is 16-byte aligned and C is a multiple of 8.  Otherwise
// 8 are loaded all the same, the row's last where it has not as many there, and
// moved up: [20001, 2999] in bf16 takes 33 us, with loads one by one, in
// branches, 72.
template <typename T, bool VEC>
DEV void load8(const T* p, int col, int C, float* v) {
    if (VEC) {
        if (col < C) {
            struct alignas(16) Pack { T t[8]; };
            const Pack x = *(const Pack*)(p + col);
            #pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_f(x.t[i]);
        } else {
            #pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        }
    } else if (C < 8) {
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = col + i < C ? to_f(p[col + i]) : 0.0f;
    } else {
        const int from = min(col, C - 8), up = col - from;
        T t[8];
        __builtin_memcpy(t, p + from, sizeof(t));
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f(t[i]);
        if (up > 0) {
            #pragma unroll
            for (int by = 4; by > 0; by >>= 1)
                #pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (up & by) v[i] = i + by < 8 ? v[i + by] : 0.0f;
            if (up >= 8) {
                #pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.0f;
            }
        }
    }
}

// N values to a place of any alignment, those that are there.  [20001, 2999]
// back to bf16 takes 34 us, one by one 76; [20001, 1001, 300] 36 and 64.
template <int N, typename T>
DEV void store_some(T* p, const T (&t)[N], int there) {
    if (there >= N) {
        __builtin_memcpy(p, t, sizeof(t));
    } else {
        #pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < there) p[i] = t[i];
    }
}

// ---------------------------------------------------------------------------
// Quantisation with a scale per 1 x 128 block.  16 lanes hold one block, 8
// columns each; BPW blocks of a row per wave (1 for narrow matrices, so that
// the wave's other lanes take further rows).  Bound by memory: reads the
// input once, writes half (bf16) or a quarter (fp32) of it.  [32768, 3136] in
// bf16: 63 us, 4.9 TB/s.
//
// MASK: values whose bit is clear are taken as zero (the gradient of a relu).
// SUM: also adds up the columns, for the bias gradient: each workgroup writes
// its partial sums in fp32 to part[blockIdx.y][C]; no atomics, so the result
// does not depend on the order in which workgroups run.  Both, [32768, 1024] in
// bf16: 29 us, 3.7 TB/s, and 4 to add up the parts.
// ---------------------------------------------------------------------------
template <typename T, bool VEC, int BPW, bool MASK, bool SUM, int WAVES>
DEV void quant_rows(const T* __restrict__ x, int64_t ldx,
                    const uint8_t* __restrict__ mask, uint8_t* __restrict__ q,
                    uint8_t* __restrict__ scale, int R, int C, int nb, int S,
                    int strip, int group, int groups, float (&sum)[8]) {
    constexpr int RPW = 4 / BPW;  // rows of a wave
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int grp = lane >> 4, l15 = lane & 15;
    const int blk = strip * BPW + (BPW == 4 ? grp : 0);
    const int col = blk * 128 + l15 * 8;
    const int step = WAVES * RPW * groups;
    if (blk < nb) {
        for (int r = (group * WAVES + wave) * RPW + (BPW == 4 ? 0 : grp);
             r < R; r += step) {
            float v[8];
            load8<T, VEC>(x + r * ldx, col, C, v);
            if (MASK) {
                const unsigned m = mask[(int64_t)r * (nb * 16) + blk * 16 + l15];
                #pragma unroll
                for (int i = 0; i < 8; ++i)
                    v[i] = (m >> i) & 1 ? v[i] : 0.0f;
            }
            float am = 0.0f;
            #pragma unroll
            for (int i = 0; i < 8; ++i) {
                am = fmaxf(am, finite_abs(v[i]));
                if (SUM) sum[i] += v[i];
            }
            const int e = block_exp(max16(am));
            *(i32x2*)(q + (int64_t)r * (nb * 128) + col) = pack8(v, pow2i(-e));
            if (l15 == 0) scale[(int64_t)r * S + blk] = (uint8_t)(e + 127);
            // bytes between nb and S are read with the others as one dword
            if (l15 == 0 && blk == nb - 1)
                for (int i = nb; i < S; ++i) scale[(int64_t)r * S + i] = 0;
        }
    }
}

template <typename T, bool VEC, int BPW, bool MASK, bool SUM>
__global__ __launch_bounds__(256) void quant_rows_kernel(
    const T* __restrict__ x, int64_t ldx, const uint8_t* __restrict__ mask,
    uint8_t* __restrict__ q, uint8_t* __restrict__ scale,
    float* __restrict__ part, int R, int C, int nb, int S) {
    constexpr int RPW = 4 / BPW;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    quant_rows<T, VEC, BPW, MASK, SUM, 4>(x, ldx, mask, q, scale, R, C, nb, S,
                                          blockIdx.x, blockIdx.y, gridDim.y,
                                          sum);
    if (SUM) {
        __shared__ float red[4][64][9];  // 9: lanes on different banks
        #pragma unroll
        for (int i = 0; i < 8; ++i) red[wave][lane][i] = sum[i];
        __syncthreads();
        for (int c = threadIdx.x; c < BPW * 128; c += 256) {
            float t = 0.0f;
            #pragma unroll
            for (int w = 0; w < 4; ++w) {
                #pragma unroll
                for (int g = 0; g < RPW; ++g)
                    t += red[w][(BPW == 4 ? c >> 3 : g * 16 + (c >> 3))][c & 7];
            }
            const int cc = blockIdx.x * BPW * 128 + c;
            if (cc < C) part[(int64_t)blockIdx.y * C + cc] = t;
        }
    }
}

// out[c] = sum over G rows of part[g][c]; 64 columns and 16 shares of the rows
// a workgroup, so that no load waits for another.  A share goes in runs of 64
// rows, then the runs: one register over thousands of terms of one sign is 1e-5
// and more off.
template <typename T>
__global__ __launch_bounds__(1024) void column_sum_kernel(
    const float* __restrict__ part, T* __restrict__ out, int G, int C) {
    __shared__ float red[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), g0 = threadIdx.x >> 6;
    float t = 0.0f;
    if (c < C) {
        for (int from = g0; from < G; from += 16 * 64) {
            float p = 0.0f;
            const int end = min(from + 16 * 64, G);
            #pragma unroll 8
            for (int g = from; g < end; g += 16) p += part[(int64_t)g * C + c];
            t += p;
        }
    }
    red[g0][threadIdx.x & 63] = t;
    __syncthreads();
    if (g0 == 0 && c < C) {
        #pragma unroll
        for (int i = 1; i < 16; ++i) t += red[i][threadIdx.x];
        out[c] = from_f<T>(t);
    }
}

// ---------------------------------------------------------------------------
// Quantisation with a scale per 128 x 128 block, for weights; qt/scale_t (may
// be null) get the transposed matrix, whose blocks have the same scales.  One
// workgroup per block: 32 values a thread stay in registers between the
// maximum and the conversion; the transposed bytes go through LDS.  Bound by
// the launch at the sizes of a layer's weight: [1024, 3136] in bf16 takes 4.4 us.
// ---------------------------------------------------------------------------
struct Tiles {
    const void* x;           // [R, C] of T, rows ldx apart
    int64_t ldx;
    uint8_t *q, *scale, *qt, *scale_t;
    int R, C, nb, S, nbt, St;
};

template <typename T, bool VEC>
DEV void quant_tile(const Tiles& a, int bc, int br) {
    __shared__ float wmax[8];
    __shared__ uint8_t tile[128][132];  // 132: columns fall on all banks
    const int t = threadIdx.x, l15 = t & 15, rr = t >> 4;
    const T* const x = (const T*)a.x;
    const int64_t ldx = a.ldx;
    uint8_t *const q = a.q, *const scale = a.scale, *const qt = a.qt,
            *const scale_t = a.scale_t;
    const int R = a.R, C = a.C, nb = a.nb, S = a.S, nbt = a.nbt, St = a.St;
    const int col = bc * 128 + l15 * 8;
    float v[4][8];
    float am = 0.0f;
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = br * 128 + i * 32 + rr;
        if (r < R) {
            load8<T, VEC>(x + r * ldx, col, C, v[i]);
        } else {
            #pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        }
        #pragma unroll
        for (int j = 0; j < 8; ++j) am = fmaxf(am, finite_abs(v[i][j]));
    }
    #pragma unroll
    for (int off = 32; off > 0; off >>= 1) am = fmaxf(am, __shfl_xor(am, off, 64));
    if ((t & 63) == 0) wmax[t >> 6] = am;
    __syncthreads();
    #pragma unroll
    for (int i = 0; i < 8; ++i) am = fmaxf(am, wmax[i]);
    const int e = block_exp(am);
    const float inv = pow2i(-e);
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = br * 128 + i * 32 + rr;
        const i32x2 w = pack8(v[i], inv);
        if (r < R) *(i32x2*)(q + (int64_t)r * (nb * 128) + col) = w;
        if (qt) {
            *(int*)&tile[i * 32 + rr][l15 * 8] = w[0];
            *(int*)&tile[i * 32 + rr][l15 * 8 + 4] = w[1];
        }
    }
    if (t == 0) {
        scale[(int64_t)br * S + bc] = (uint8_t)(e + 127);
        if (bc == nb - 1)
            for (int i = nb; i < S; ++i) scale[(int64_t)br * S + i] = 0;
        if (qt) {
            scale_t[(int64_t)bc * St + br] = (uint8_t)(e + 127);
            if (br == nbt - 1)
                for (int i = nbt; i < St; ++i) scale_t[(int64_t)bc * St + i] = 0;
        }
    }
    if (!qt) return;
    __syncthreads();
    // 8 rows x 4 columns a thread, transposed by byte permutes; 16 lanes write
    // the 128 bytes of one row of the transposed block
    {
        const int n8 = t & 15, c4 = t >> 4;
        uint32_t d[8], o[4][2];
        #pragma unroll
        for (int r = 0; r < 8; ++r)
            d[r] = *(const uint32_t*)&tile[n8 * 8 + r][c4 * 4];
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t* e = d + 4 * h;
            const uint32_t aa = __builtin_amdgcn_perm(e[1], e[0], 0x05010400);
            const uint32_t b = __builtin_amdgcn_perm(e[1], e[0], 0x07030602);
            const uint32_t u = __builtin_amdgcn_perm(e[3], e[2], 0x05010400);
            const uint32_t v = __builtin_amdgcn_perm(e[3], e[2], 0x07030602);
            o[0][h] = __builtin_amdgcn_perm(u, aa, 0x05040100);
            o[1][h] = __builtin_amdgcn_perm(u, aa, 0x07060302);
            o[2][h] = __builtin_amdgcn_perm(v, b, 0x05040100);
            o[3][h] = __builtin_amdgcn_perm(v, b, 0x07060302);
        }
        #pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int c = bc * 128 + c4 * 4 + r;
            if (c < C)
                *(i32x2*)(qt + (int64_t)c * (nbt * 128) + br * 128 + n8 * 8) =
                    i32x2{(int)o[r][0], (int)o[r][1]};
        }
    }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(512) void quant_tiles_kernel(Tiles a) {
    quant_tile<T, VEC>(a, blockIdx.x, blockIdx.y);
}

// A weight's tiles and an activation's rows in one launch, the forward pass of
// a training step: the first `tiles` workgroups take the weight.  x [32768,
// 3136] and w [1024, 3136] in bf16: 62 us, what x takes alone; x [256, 3136]:
// 9.6 us.
template <typename T, int BPW>
__global__ __launch_bounds__(512) void quant_both_kernel(
    Tiles a, const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q,
    uint8_t* __restrict__ scale, int R, int nb, int S, int tiles, int strips,
    int groups) {
    if ((int)blockIdx.x < tiles) {
        quant_tile<T, true>(a, blockIdx.x % nb, blockIdx.x / nb);
    } else {
        const int id = blockIdx.x - tiles;
        float none[8];
        quant_rows<T, true, BPW, false, false, 8>(
            x, ldx, nullptr, q, scale, R, a.C, nb, S, id % strips, id / strips,
            groups, none);
    }
}

// 8-bit blocks -> T; 8 columns a thread.  q 2^e is exact in fp32, and in bf16
// wherever it is a normal number.  Bound by memory: [32768, 3136] to bf16 54 us,
// 5.8 TB/s right after it was quantised, as part of it is still in the last cache.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dequant_kernel(
    const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale,
    T* __restrict__ out, int R, int C, int nb, int S, int shift) {
    const int per = (C + 7) >> 3;  // groups of 8 columns in a row
    for (int64_t i = threadIdx.x + (int64_t)blockIdx.x * 256;
         i < (int64_t)R * per; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per;
        const int col = (int)(i - r * per) * 8;
        const i32x2 w = *(const i32x2*)(q + r * (nb * 128) + col);
        const int e = (int)scale[(r >> shift) * S + (col >> 7)] - 127;
        // 2^-127 is no normal number: two factors, each a power of two
        const float s0 = pow2i(e < 0 ? e + 1 : e), s1 = e < 0 ? 0.5f : 1.0f;
        struct alignas(16) Pack { T t[8]; } p;
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
            auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], false);
            auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], true);
            p.t[4 * j] = from_f<T>(lo[0] * s0 * s1);
            p.t[4 * j + 1] = from_f<T>(lo[1] * s0 * s1);
            p.t[4 * j + 2] = from_f<T>(hi[0] * s0 * s1);
            p.t[4 * j + 3] = from_f<T>(hi[1] * s0 * s1);
        }
        T* o = out + r * C + col;
        if (VEC) {
            *(Pack*)o = p;
        } else {
            store_some(o, p.t, C - col);
        }
    }
}

// ---------------------------------------------------------------------------
// C[m][n] = sum_k A[m][k] B[n][k] (+ bias[n], relu).  The MFMA's row operand
// is B, so a lane's 4 results are 4 neighbours of one row of C.
// ---------------------------------------------------------------------------
struct Gemm {
    const uint8_t *a, *as, *b, *bs;  // [M, 128 nb], [M >> ash, S] and so on
    const void* bias;                // [N] of bias_t, or null
    void* c;                         // [M, N]
    uint8_t* mask;                   // [M, 16 ceil(N / 128)] bits, or null
    int M, N, nb, S, ash, bsh, bias_t, relu;
    const void* x;                   // [M, K], rows ldx apart, in place of a
    int64_t ldx;
    int K;
};

DEV float bias_at(const Gemm& g, int n) {
    if (!g.bias) return 0.0f;
    return g.bias_t == 0   ? ((const float*)g.bias)[n]
           : g.bias_t == 1 ? to_f(((const bf16_t*)g.bias)[n])
                           : to_f(((const fp16_t*)g.bias)[n]);
}

// 8 e4m3 values and a scale byte -> bf16.  The conversion takes the exponent
// field of its fp32 scale alone, so a byte of 0 stands for 2^-127.
DEV bf16x8 expand8(int w0, int w1, int sbyte) {
    const float s = __uint_as_float((uint32_t)sbyte << 23);
    union { bf16x2 h[4]; bf16x8 v; } u;
    u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, false);
    u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, true);
    u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, false);
    u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, true);
    return u.v;
}

// adds the partial tiles of 8 waves in a fixed order and stores the result
template <int TM, int TN, typename T>
DEV void finish_direct(const Gemm& g, float (&red)[8][TM][TN + 4], int m0,
                       int n0) {
    const int t = threadIdx.x;
    __syncthreads();
    constexpr int QUADS = TM * TN / 4;
    if (t >= QUADS) return;
    const int mm = t / (TN / 4), nn = (t % (TN / 4)) * 4;
    f32x4 z = *(const f32x4*)&red[0][mm][nn];
    #pragma unroll
    for (int w = 1; w < 8; ++w) z += *(const f32x4*)&red[w][mm][nn];
    const int m = m0 + mm, n = n0 + nn;
    unsigned bits = 0;
    struct alignas(4 * sizeof(T)) Pack { T t[4]; } p;
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        float y = z[j] + (n + j < g.N ? bias_at(g, n + j) : 0.0f);
        const bool on = passes(y);
        bits |= (unsigned)(on && n + j < g.N) << j;
        if (g.relu && !on) y = 0.0f;
        p.t[j] = from_f<T>(y);
    }
    if (g.mask) {
        // four neighbours make 16 columns; quads of a row are 4-aligned
        bits <<= 4 * (t & 3);
        bits |= __shfl_xor(bits, 1, 64);
        bits |= __shfl_xor(bits, 2, 64);
        if ((t & 3) == 0 && m < g.M)
            *(uint16_t*)(g.mask + (int64_t)m * (((g.N + 127) >> 7) * 16) +
                         (n >> 3)) = (uint16_t)bits;
    }
    if (m >= g.M) return;
    T* out = (T*)g.c + (int64_t)m * g.N + n;
    if ((g.N & 3) == 0) {
        if (n < g.N) *(Pack*)out = p;
    } else {
        store_some(out, p.t, g.N - n);
    }
}

// Few rows or small results: a workgroup of 8 waves computes a tile of
// 16 MI x 16 NI, each wave a share of the 128-column blocks (kb = wave,
// wave + 8, ...), with operands straight from memory into registers: no
// staging, so a wave has all its loads in flight at once.  The 8 partial
// tiles are added in LDS in a fixed order.  Bound by the loads, 64 bytes of each
// of 16 rows at a time, so the products are the exact bf16 ones.  [1, 1024,
// 3136]: 4.3 us, [256, 1024, 3136]: 8.9.
template <int MI, int NI, typename T>
__global__ __launch_bounds__(512) void gemm_direct_kernel(Gemm g) {
    constexpr int TM = 16 * MI, TN = 16 * NI;
    __shared__ float red[8][TM][TN + 4];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int l15 = lane & 15, l4 = lane >> 4;
    const int nt = (g.N + TN - 1) / TN;
    const int m0 = (blockIdx.x / nt) * TM, n0 = (blockIdx.x % nt) * TN;
    const int64_t ld = (int64_t)g.nb * 128;
    const uint8_t *pa[MI], *sa[MI], *pb[NI], *sb[NI];
    #pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int64_t r = min(m0 + i * 16 + l15, g.M - 1);
        pa[i] = g.a + r * ld + l4 * 16;
        sa[i] = g.as + (r >> g.ash) * g.S;
    }
    #pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int64_t r = min(n0 + i * 16 + l15, g.N - 1);
        pb[i] = g.b + r * ld + l4 * 16;
        sb[i] = g.bs + (r >> g.bsh) * g.S;
    }
    f32x4 acc[MI][NI];
    #pragma unroll
    for (int i = 0; i < MI; ++i)
        #pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    #pragma unroll 2
    for (int kb = wave; kb < g.nb; kb += 8) {
        i32x4 fa[MI][2], fb[NI][2];
        int ea[MI], eb[NI];
        #pragma unroll
        for (int i = 0; i < MI; ++i) {
            fa[i][0] = *(const i32x4*)(pa[i] + kb * 128);
            fa[i][1] = *(const i32x4*)(pa[i] + kb * 128 + 64);
            ea[i] = sa[i][kb];
        }
        #pragma unroll
        for (int i = 0; i < NI; ++i) {
            fb[i][0] = *(const i32x4*)(pb[i] + kb * 128);
            fb[i][1] = *(const i32x4*)(pb[i] + kb * 128 + 64);
            eb[i] = sb[i][kb];
        }
        // the order of the 128 products is free, as both operands have it
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            #pragma unroll
            for (int u = 0; u < 4; u += 2) {
                bf16x8 xb[NI];
                #pragma unroll
                for (int j = 0; j < NI; ++j)
                    xb[j] = expand8(fb[j][h][u], fb[j][h][u + 1], eb[j]);
                #pragma unroll
                for (int i = 0; i < MI; ++i) {
                    const bf16x8 xa =
                        expand8(fa[i][h][u], fa[i][h][u + 1], ea[i]);
                    #pragma unroll
                    for (int j = 0; j < NI; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            xb[j], xa, acc[i][j], 0, 0, 0);
                }
            }
        }
    }
    #pragma unroll
    for (int i = 0; i < MI; ++i)
        #pragma unroll
        for (int j = 0; j < NI; ++j)
            *(f32x4*)&red[wave][i * 16 + l15][j * 16 + l4 * 4] = acc[i][j];
    finish_direct<TM, TN, T>(g, red, m0, n0);
}

// A product of up to 16 rows that are not in 8 bits yet, for serving: one
// launch instead of two, which is what such a call takes its time with.  The
// workgroup first quantises the rows into LDS, exactly as quant_rows_kernel
// does, while its first piece of B is on the way; then as above.
// [1, 1024, 3136]: 5.7 us a call, 10.4 by two launches.
template <typename T, bool VEC>
__global__ __launch_bounds__(512) void gemm_few_kernel(Gemm g) {
    __shared__ float red[8][16][20];
    extern __shared__ __align__(16) uint8_t lds[];  // rows, then their scales
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int l15 = lane & 15, l4 = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int pitch = g.nb * 128 + 16;  // 16: rows begin on different banks
    uint8_t* const scales = lds + g.M * pitch;
    const int64_t rb = min(n0 + l15, g.N - 1);
    const uint8_t* pb = g.b + rb * ((int64_t)g.nb * 128) + l4 * 16;
    const uint8_t* sb = g.bs + (rb >> g.bsh) * g.S;
    i32x4 fb[2];
    int eb = 0;
    auto load = [&](int kb) {
        fb[0] = *(const i32x4*)(pb + kb * 128);
        fb[1] = *(const i32x4*)(pb + kb * 128 + 64);
        eb = sb[kb];
    };
    load(min(wave, g.nb - 1));
    for (int i = t >> 4; i < g.M * g.nb; i += 32) {
        const int r = i / g.nb, blk = i - r * g.nb;
        float v[8];
        load8<T, VEC>((const T*)g.x + r * g.ldx, blk * 128 + l15 * 8, g.K, v);
        float am = 0.0f;
        #pragma unroll
        for (int j = 0; j < 8; ++j) am = fmaxf(am, finite_abs(v[j]));
        const int e = block_exp(max16(am));
        *(i32x2*)(lds + r * pitch + blk * 128 + l15 * 8) = pack8(v, pow2i(-e));
        if (l15 == 0) scales[i] = (uint8_t)(e + 127);
    }
    __syncthreads();
    const int ra = min(l15, g.M - 1);
    f32x4 acc = {0, 0, 0, 0};
    for (int kb = wave; kb < g.nb; kb += 8) {
        const i32x4 b0 = fb[0], b1 = fb[1];
        const int e1 = eb;
        load(min(kb + 8, g.nb - 1));  // the next piece
        const uint8_t* p = lds + ra * pitch + kb * 128 + l4 * 16;
        const i32x4 a0 = *(const i32x4*)p, a1 = *(const i32x4*)(p + 64);
        const int e0 = scales[ra * g.nb + kb];
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            const i32x4 a = h ? a1 : a0, b = h ? b1 : b0;
            #pragma unroll
            for (int u = 0; u < 4; u += 2)
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    expand8(b[u], b[u + 1], e1), expand8(a[u], a[u + 1], e0),
                    acc, 0, 0, 0);
        }
    }
    *(f32x4*)&red[wave][l15][l4 * 4] = acc;
    finish_direct<16, 16, T>(g, red, 0, n0);
}

// ---------------------------------------------------------------------------
// Larger results.  A workgroup of WM x WN waves, each with 16 MI rows of C and
// 16 NJ columns, walks over K in steps of 128 with two LDS buffers: while one is
// multiplied the next is on its way into the other, straight from memory
// (global_load_lds, 16 bytes a lane).  The walk goes on over the workgroup's
// next tile without a pause: its first step is under way during the epilogue.
//
// LDS rows are 128 bytes; the 16-byte piece p of row r lies at p ^ (r / 2 % 8),
// so the 16 rows that a fragment reads fall on all 64 banks.  B's rows lie in
// the order in which lane group l4 of a pair of fragments gets columns 8 l4
// ... 8 l4 + 7 of 32: a lane then ends up with 8 neighbours of one row of C,
// the 4 groups with 32, and a store of 16 bits a value fills 64 bytes of each
// of 16 rows.
//
// EXACT: operands expanded to bf16, every product summed in full.  Otherwise
// the scaled 8-bit instruction, at twice the rate.
//
// 256 x 256, 8 waves of 128 x 64, to bf16: 8192^3 exact in 766 us (1436 TF) and
// scaled in 451 (2440 TF); [32768, 1024, 3136] in 160 to 183 and 102 to 118,
// [32768, 3136, 1024] in 224 to 252 and 155 to 171, where results are written for as long as two of a tile's 8 steps
// take.  Products are under way 53 % of the time (8 bits): a step's reads from
// LDS and its loads into it need as long as they do.  Two groups of waves that
// read and multiply by turns took 504 us for 8192^3, 4 waves of 128 x 128 more
// than 8 of 128 x 64, and stores counted so as to go on under two steps of the
// next tile the same as now.
// ---------------------------------------------------------------------------
DEV i32x8 two(i32x4 lo, i32x4 hi) {
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// a buffer of `bytes` from a uniform address
DEV __amdgpu_buffer_rsrc_t buffer_of(const uint8_t* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(
        (void*)p, 0, (int)min(bytes, (int64_t)0xffffffffu), 0x00027000);
}

// B's row at place r of a tile, see above
DEV int place_b(int r) {
    return (r & ~31) + ((r & 15) >> 2) * 8 + ((r >> 4) & 1) * 4 + (r & 3);
}

// The results of a wave: columns n ... n + 7 of rows m0 + 16 i + lane % 16, for
// each 32 columns.  A row's stores follow each other, so that whole lines are
// written.
template <int MI, int NJ, typename T>
DEV void store_tile(const Gemm& g, const f32x4 (&acc)[MI][NJ], int m0, int n0,
                    int lane) {
    const int l15 = lane & 15, l4 = lane >> 4;
    const bool even = (g.N & 7) == 0;  // all 8 there, and aligned
    auto finish = [&](auto plain, const float (&bias)[NJ / 2][8]) {
        #pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int m = m0 + i * 16 + l15;
            #pragma unroll
            for (int c = 0; c < NJ / 2; ++c) {
                const int n = n0 + c * 32 + l4 * 8;
                unsigned bits = 0;
                struct alignas(16) Pack { T t[8]; } p;
                #pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float z = acc[i][c * 2 + (e >> 2)][e & 3];
                    if (!decltype(plain)::value) {
                        z += bias[c][e];
                        const bool on = passes(z);
                        bits |= (unsigned)(on && n + e < g.N) << e;
                        if (g.relu && !on) z = 0.0f;
                    }
                    p.t[e] = from_f<T>(z);
                }
                if (m >= g.M || n >= g.N) continue;
                if (!decltype(plain)::value && g.mask)
                    g.mask[(int64_t)m * (((g.N + 127) >> 7) * 16) + (n >> 3)] =
                        (uint8_t)bits;
                T* out = (T*)g.c + (int64_t)m * g.N + n;
                if (even) {
                    *(Pack*)out = p;
                } else {
                    store_some(out, p.t, g.N - n);
                }
            }
        }
    };
    // without any of them the results go out as they are: the rest is 10
    // instructions a value, as long as 4 steps of products
    float bias[NJ / 2][8];
    if (g.bias || g.relu || g.mask) {
        #pragma unroll
        for (int c = 0; c < NJ / 2; ++c)
            #pragma unroll
            for (int e = 0; e < 8; ++e)
                bias[c][e] = bias_at(g, min(n0 + c * 32 + l4 * 8 + e, g.N - 1));
        finish(std::false_type{}, bias);
    } else {
        finish(std::true_type{}, bias);
    }
}

template <int WM, int WN, int MI, int NJ, bool EXACT, typename T>
__global__ __launch_bounds__(64 * WM * WN) void gemm_tile_kernel(Gemm g) {
#ifdef __HIP_DEVICE_COMPILE__  // the host needs its launch alone
    constexpr int TM = WM * MI * 16, TN = WN * NJ * 16, WAVES = WM * WN;
    constexpr int BUF = (TM + TN) * 128;
    // [2][BUF] tiles, [2][TM + TN] dwords of scales
    extern __shared__ __align__(16) uint8_t lds[];
    uint32_t* const lds_s = (uint32_t*)(lds + 2 * BUF);
    static_assert(TM + TN <= 64 * WAVES && TM % 64 == 0, "a scale a lane");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l15 = lane & 15, l4 = lane >> 4;
    const int wm = (wave / WN) * MI * 16, wn = (wave % WN) * NJ * 16;
    const int nt = (g.N + TN - 1) / TN, mt = (g.M + TM - 1) / TM;
    const int64_t ld = (int64_t)g.nb * 128;
    // each XCD (workgroups are dealt to 8 in turn) takes one run of tiles,
    // neighbours in n first, so that its L2 serves a row of tiles' A once
    const int tiles = mt * nt, xcd = blockIdx.x & 7;
    const int q = tiles >> 3, rem = tiles & 7;
    const int first = xcd * q + min(xcd, rem), end = first + q + (xcd < rem);
    const int stride = gridDim.x >> 3;
    int tile = first + (blockIdx.x >> 3);
    if (tile >= end) return;

    // Loads go by a buffer that begins at the tile's first row, a lane's
    // offset in it and a uniform one for the step.  One instruction fills 8
    // rows: lane -> row lane / 8, stored piece lane % 8; rows behind the last
    // one are read as the last.
    constexpr int LA = TM / 8 / WAVES, LB = TN / 8 / WAVES;
    __amdgpu_buffer_rsrc_t buf_a, buf_b, buf_s;
    uint32_t off[LA + LB], off_s;
    auto enter = [&](int tile) {
        const int m0 = (tile / nt) * TM, n0 = (tile % nt) * TN;
        buf_a = buffer_of(g.a + m0 * ld, (g.M - m0) * ld);
        buf_b = buffer_of(g.b + n0 * ld, (g.N - n0) * ld);
        #pragma unroll
        for (int i = 0; i < LA + LB; ++i) {
            const int inst = (i < LA ? i : i - LA) * WAVES + wave;
            const int r = inst * 8 + (lane >> 3);
            const int from = i < LA ? min(r, g.M - 1 - m0)
                                    : min(place_b(r), g.N - 1 - n0);
            off[i] = (uint32_t)from * (uint32_t)ld +
                     ((lane & 7) ^ ((r >> 1) & 7)) * 16;
        }
        // scales: a wave takes those of 64 rows, A's or B's
        const int r = wave * 64 + lane;
        if (wave * 64 < TM) {
            const int r0 = m0 >> g.ash;
            buf_s = buffer_of(g.as + (int64_t)r0 * g.S,
                              (((g.M - 1) >> g.ash) + 1 - r0) * (int64_t)g.S);
            off_s = ((min(m0 + r, g.M - 1) >> g.ash) - r0) * g.S;
        } else {
            const int r0 = n0 >> g.bsh;
            buf_s = buffer_of(g.bs + (int64_t)r0 * g.S,
                              (((g.N - 1) >> g.bsh) + 1 - r0) * (int64_t)g.S);
            off_s = (((n0 + min(place_b(r - TM), g.N - 1 - n0)) >> g.bsh) - r0) * g.S;
        }
    };
    int sbuf = 1;  // which scales are in use
    // loads [from, to) of a wave's share of a step
    auto stage = [&](int buf, int kb, int from, int to) {
        // the scales of 4 steps are a dword a row
        if (from == 0 && (kb & 3) == 0 && wave * 64 < TM + TN)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                buf_s,
                (__attribute__((address_space(3))) void*)(
                    lds_s + (sbuf ^ 1) * (TM + TN) + wave * 64),
                4, off_s, kb, 0, 0);
        #pragma unroll
        for (int i = 0; i < LA + LB; ++i) {
            if (i < from || i >= to) continue;
            const int inst = (i < LA ? i : i - LA) * WAVES + wave;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                i < LA ? buf_a : buf_b,
                (__attribute__((address_space(3))) void*)(
                    lds + buf * BUF + (i < LA ? 0 : TM * 128) + inst * 1024),
                16, off[i], kb * 128, 0, 0);
        }
    };
    enter(tile);
    stage(0, 0, 0, LA + LB);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    int buf = 0;
    for (; tile < end; tile += stride) {
        const int m0 = (tile / nt) * TM + wm, n0 = (tile % nt) * TN + wn;
        f32x4 acc[MI][NJ];
        #pragma unroll
        for (int i = 0; i < MI; ++i)
            #pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
        int ea[MI], eb[NJ];
        for (int kb = 0; kb < g.nb; ++kb, buf ^= 1) {
            // a tile's first step was waited for before the last one's stores
            if (kb > 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if ((kb & 3) == 0) {
                sbuf ^= 1;
                #pragma unroll
                for (int i = 0; i < MI; ++i)
                    ea[i] = lds_s[sbuf * (TM + TN) + wm + i * 16 + l15];
                #pragma unroll
                for (int j = 0; j < NJ; ++j)
                    eb[j] = lds_s[sbuf * (TM + TN) + TM + wn + j * 16 + l15];
            } else {
                #pragma unroll
                for (int i = 0; i < MI; ++i) ea[i] >>= 8;
                #pragma unroll
                for (int j = 0; j < NJ; ++j) eb[j] >>= 8;
            }
            // The next step goes into the other buffer, which all waves are
            // past reading; behind the last step the tile's first, for
            // nothing.  Its loads are issued between the products of the
            // first half of this step: a wave that issues them at once waits
            // for the memory pipe to take them, and multiplies nothing.
            const bool last = kb + 1 == g.nb;
            if (last && tile + stride < end) enter(tile + stride);
            const int next = last ? 0 : kb + 1;
            constexpr int PER = 2 * (LA + LB) / MI;
            const uint8_t* A = lds + buf * BUF;
            const uint8_t* B = A + TM * 128;
            auto piece = [&](const uint8_t* base, int row, int p) {
                return *(const i32x4*)(base + row * 128 +
                                       ((p ^ ((row >> 1) & 7)) * 16));
            };
            auto row_a = [&](int i) {
                return two(piece(A, wm + i * 16 + l15, l4),
                           piece(A, wm + i * 16 + l15, 4 + l4));
            };
            if (!EXACT) {
                // reads run two fragments ahead of the products
                i32x8 fa[3], fb[NJ];
                fa[0] = row_a(0);
                #pragma unroll
                for (int j = 0; j < NJ; ++j)
                    fb[j] = two(piece(B, wn + j * 16 + l15, l4),
                                piece(B, wn + j * 16 + l15, 4 + l4));
                fa[1] = row_a(1);
                #pragma unroll
                for (int i = 0; i < MI; ++i) {
                    if (i + 2 < MI) fa[(i + 2) % 3] = row_a(i + 2);
                    stage(buf ^ 1, next, i * PER, (i + 1) * PER);
                    __builtin_amdgcn_sched_barrier(0);
                    #pragma unroll
                    for (int j = 0; j < NJ; ++j)
                        acc[i][j] =
                            __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                                fb[j], fa[i % 3], acc[i][j], 0, 0, 0, eb[j], 0,
                                ea[i]);
                }
            } else {
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    bf16x8 fb[NJ][2];
                    i32x4 fa[3];
                    fa[0] = piece(A, wm + l15, h * 4 + l4);
                    #pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        const i32x4 w = piece(B, wn + j * 16 + l15, h * 4 + l4);
                        fb[j][0] = expand8(w[0], w[1], eb[j] & 255);
                        fb[j][1] = expand8(w[2], w[3], eb[j] & 255);
                    }
                    fa[1] = piece(A, wm + 16 + l15, h * 4 + l4);
                    #pragma unroll
                    for (int i = 0; i < MI; ++i) {
                        if (i + 2 < MI)
                            fa[(i + 2) % 3] =
                                piece(A, wm + (i + 2) * 16 + l15, h * 4 + l4);
                        if (h == 0) stage(buf ^ 1, next, i * PER / 2, (i + 1) * PER / 2);
                        __builtin_amdgcn_sched_barrier(0);
                        const i32x4 w = fa[i % 3];
                        const bf16x8 lo = expand8(w[0], w[1], ea[i] & 255);
                        const bf16x8 hi = expand8(w[2], w[3], ea[i] & 255);
                        #pragma unroll
                        for (int j = 0; j < NJ; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                fb[j][0], lo, acc[i][j], 0, 0, 0);
                        #pragma unroll
                        for (int j = 0; j < NJ; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                fb[j][1], hi, acc[i][j], 0, 0, 0);
                    }
                }
            }
        }
        // The next tile's first step is waited for here: behind the stores it
        // would be waited for with them, as the counter knows one order only.
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        store_tile<MI, NJ, T>(g, acc, m0, n0, lane);
    }
    // no load may come in after the workgroup has given its LDS back
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#endif
}

template <int WM, int WN, int MI, int NJ, typename T>
void launch_tiles(const Gemm& g, bool exact, hipStream_t st) {
    constexpr int TM = WM * MI * 16, TN = WN * NJ * 16;
    constexpr int bytes = 2 * (TM + TN) * (128 + 4);
    const int64_t tiles =
        (int64_t)((g.M + TM - 1) / TM) * ((g.N + TN - 1) / TN);
    // as many workgroups as the 256 CUs hold, in whole rounds of the 8 XCDs
    const int64_t most = 256 * (163840 / bytes);
    const dim3 grid((uint32_t)min((tiles + 7) / 8 * 8, most));
    if (sizeof(T) == 4 || exact)
        hipLaunchKernelGGL((gemm_tile_kernel<WM, WN, MI, NJ, true, T>), grid,
                           dim3(64 * WM * WN), bytes, st, g);
    else
        hipLaunchKernelGGL((gemm_tile_kernel<WM, WN, MI, NJ, sizeof(T) == 4, T>),
                           grid, dim3(64 * WM * WN), bytes, st, g);
}

// The same for fewer results, where a workgroup or two fall to a CU and a step
// takes as long as the way from one barrier to the next: loads, LDS reads and
// products one behind the other.  One tile of 64 x 64 a workgroup; two groups
// of 4 waves take every other step, so that there are half as many barriers and
// one group's reads go on under the other's products.  Their sums are added at
// the end, through LDS.  [1024, 1024, 3136]: scaled 9.3 us, exact in fp32 13.7;
// with one group 11.9 and 16.0, with four 9.7 and 13.4.
template <bool EXACT, typename T>
__global__ __launch_bounds__(512) void gemm_shared_kernel(Gemm g) {
#ifdef __HIP_DEVICE_COMPILE__
    constexpr int TM = 64, TN = 64, MI = 2, NJ = 2, WAVES = 4, LOADS = 4;
    // a step's rows, then the dwords of scales of them
    constexpr int BUF = (TM + TN) * (128 + 4);
    extern __shared__ __align__(16) uint8_t lds[];  // [2 buffers][2 groups][BUF]
    const int lane = threadIdx.x & 63;
    const int all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = all / WAVES, wave = all % WAVES;
    const int l15 = lane & 15, l4 = lane >> 4;
    const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
    const int nt = (g.N + TN - 1) / TN;
    const int64_t ld = (int64_t)g.nb * 128;
    // each XCD takes one run of tiles, as above
    const int xcd = blockIdx.x & 7, q = gridDim.x >> 3, rem = gridDim.x & 7;
    const int tile = xcd * q + min(xcd, rem) + (blockIdx.x >> 3);
    const int m0 = (tile / nt) * TM, n0 = (tile % nt) * TN;
    const auto buf_a = buffer_of(g.a + m0 * ld, (g.M - m0) * ld);
    const auto buf_b = buffer_of(g.b + n0 * ld, (g.N - n0) * ld);
    uint32_t off[LOADS];  // A, A, B, B
    #pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int r = ((i & 1) * WAVES + wave) * 8 + (lane >> 3);
        const int from = i < 2 ? min(r, g.M - 1 - m0)
                               : min(place_b(r), g.N - 1 - n0);
        off[i] = (uint32_t)from * (uint32_t)ld +
                 ((lane & 7) ^ ((r >> 1) & 7)) * 16;
    }
    // scales: wave 0 takes those of A's rows, wave 1 those of B's
    const int r0 = wave ? n0 >> g.bsh : m0 >> g.ash;
    const int rows = wave ? ((g.N - 1) >> g.bsh) + 1 : ((g.M - 1) >> g.ash) + 1;
    const auto buf_s = buffer_of((wave ? g.bs : g.as) + (int64_t)r0 * g.S,
                                 (rows - r0) * (int64_t)g.S);
    const uint32_t off_s =
        (wave ? ((n0 + min(place_b(lane), g.N - 1 - n0)) >> g.bsh) - r0
              : (min(m0 + lane, g.M - 1) >> g.ash) - r0) * g.S;
    typedef __attribute__((address_space(3))) void* lds_t;
    // a group's step of a round; behind the last one the last, for nothing
    auto stage = [&](int round) {
        const int kb = min(round * 2 + group, g.nb - 1);
        uint8_t* const to = lds + ((round & 1) * 2 + group) * BUF;
        if (wave < 2)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                buf_s, (lds_t)(to + (TM + TN) * 128 + wave * 256), 4, off_s,
                kb & ~3, 0, 0);
        #pragma unroll
        for (int i = 0; i < LOADS; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                i < 2 ? buf_a : buf_b,
                (lds_t)(to + (i < 2 ? 0 : TM * 128) +
                        ((i & 1) * WAVES + wave) * 1024),
                16, off[i], kb * 128, 0, 0);
    };
    f32x4 acc[MI][NJ];
    #pragma unroll
    for (int i = 0; i < MI; ++i)
        #pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    stage(0);
    for (int round = 0; round * 2 < g.nb; ++round) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        stage(round + 1);  // into the buffer that all are past reading
        const int kb = round * 2 + group;
        if (kb >= g.nb) continue;
        const uint8_t* A = lds + ((round & 1) * 2 + group) * BUF;
        const uint8_t* B = A + TM * 128;
        const uint32_t* sc = (const uint32_t*)(A + (TM + TN) * 128);
        auto piece = [&](const uint8_t* base, int row, int p) {
            return *(const i32x4*)(base + row * 128 +
                                   ((p ^ ((row >> 1) & 7)) * 16));
        };
        const int shift = (kb & 3) * 8;
        int ea[MI], eb[NJ];
        i32x4 fa[MI][2], fb[NJ][2];
        #pragma unroll
        for (int i = 0; i < MI; ++i)
            ea[i] = (sc[wm + i * 16 + l15] >> shift) & 255;
        #pragma unroll
        for (int j = 0; j < NJ; ++j)
            eb[j] = (sc[TM + wn + j * 16 + l15] >> shift) & 255;
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            #pragma unroll
            for (int j = 0; j < NJ; ++j)
                fb[j][h] = piece(B, wn + j * 16 + l15, h * 4 + l4);
            #pragma unroll
            for (int i = 0; i < MI; ++i)
                fa[i][h] = piece(A, wm + i * 16 + l15, h * 4 + l4);
        }
        if (!EXACT) {
            #pragma unroll
            for (int i = 0; i < MI; ++i)
                #pragma unroll
                for (int j = 0; j < NJ; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        two(fb[j][0], fb[j][1]), two(fa[i][0], fa[i][1]),
                        acc[i][j], 0, 0, 0, eb[j], 0, ea[i]);
        } else {
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
                #pragma unroll
                for (int u = 0; u < 4; u += 2) {
                    bf16x8 xb[NJ];
                    #pragma unroll
                    for (int j = 0; j < NJ; ++j)
                        xb[j] = expand8(fb[j][h][u], fb[j][h][u + 1], eb[j]);
                    #pragma unroll
                    for (int i = 0; i < MI; ++i) {
                        const bf16x8 xa =
                            expand8(fa[i][h][u], fa[i][h][u + 1], ea[i]);
                        #pragma unroll
                        for (int j = 0; j < NJ; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                xb[j], xa, acc[i][j], 0, 0, 0);
                    }
                }
            }
        }
    }
    // no load may come in behind this, over the sums or after the workgroup
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    f32x4* const part = (f32x4*)lds + wave * (MI * NJ * 64) + lane;
    __syncthreads();
    if (group == 1) {
        #pragma unroll
        for (int i = 0; i < MI * NJ; ++i) part[i * 64] = acc[i / NJ][i % NJ];
    }
    __syncthreads();
    if (group == 1) return;
    #pragma unroll
    for (int i = 0; i < MI * NJ; ++i) acc[i / NJ][i % NJ] += part[i * 64];
    store_tile<MI, NJ, T>(g, acc, m0 + wm, n0 + wn, lane);
#endif
}

template <typename T>
void launch_shared(const Gemm& g, bool exact, hipStream_t st) {
    constexpr int bytes = 2 * 2 * (64 + 64) * (128 + 4);
    const dim3 grid(((g.M + 63) / 64) * ((g.N + 63) / 64));
    if (sizeof(T) == 4 || exact)
        hipLaunchKernelGGL((gemm_shared_kernel<true, T>), grid, dim3(512), bytes,
                           st, g);
    else
        hipLaunchKernelGGL((gemm_shared_kernel<sizeof(T) == 4, T>), grid,
                           dim3(512), bytes, st, g);
}

// ---------------------------------------------------------------------------
// dW[n][k] = sum_m G[m][n] X[m][k]: both operands have a scale per row m, the
// summed index, so tiles are expanded to bf16 on their way into LDS; nothing
// is rounded before the fp32 sums.  LDS keeps rows of m; ds_read_b64_tr_b16
// hands each lane 4 rows of one column, the operand layout of a product that
// sums over rows.
//
// A tile is 256 x 128, 32 rows a step, 4 waves of 128 x 64; two LDS buffers
// of 24 KB leave room for a second workgroup on the CU, whose waves multiply
// while this one's wait at a barrier.  Loads run 3 steps ahead in registers: a
// step is shorter than the way to memory.  They go by a buffer that ends with
// the last row, behind which they give zeros: none is conditional, so the
// compiler waits for those of one step only.
//
// LDS keeps rows of m in an order that spreads what 16 rows of a transposed
// read, or 16 lanes of a write, touch over all banks.  Within 64 columns of X,
// column 16 a + 4 j + b lies at 16 j + 4 a + b, so that a lane ends up with 16
// neighbours of one row of dW.
//
// A workgroup takes one tile and one share of the rows; with more than one
// share each writes fp32 partials [share][N][K], added in a fixed order by
// add_shares_kernel.
//
// [32768, 1024, 3136]: 216 us (973 TF) and 14 to add 5 shares up.  The matrix
// unit is busy 44 % of the time, LDS 38 %: reading and multiplying take turns
// around the step's barrier.  Fragments of the next step read between the
// products took 30 us more, operands turned in registers 60; an order of X
// whose stores have no bank conflicts (14 % of LDS's time) took the same.
// ---------------------------------------------------------------------------
struct Wgrad {
    const uint8_t *g, *gs, *x, *xs;  // [M, 128 nbn], [M, Sn], [M, 128 nbk], ...
    void* dw;                        // [N, K] of T, or fp32 [shares][N][K]
    int M, N, K, nbn, Sn, nbk, Sk;
    int shares, rows;  // rows of a share: multiple of 64
};

// Where 8 bytes (4 columns from c) of a row lie.  G: rows of 256 columns, the
// two 16-byte halves of 16 columns 256 bytes apart; X: rows of 128 columns, 16
// columns together.
DEV int at_g(int row, int c) {
    const int half = (c >> 3) & 1;
    return row * 256 + half * 128 + ((c >> 4) ^ (8 * half) ^ (row & 7)) * 8 +
           (c & 7);
}
DEV int at_x(int row, int c) {
    return row * 128 + ((c >> 4) ^ (row & 7)) * 16 + (c & 15);
}

// the 32 rows of the 16 columns from c; lane group l4 gets rows 4 l4 ... and
// 16 + 4 l4 ..., in both operands alike
template <bool G>
DEV bf16x8 tr_frag(const uint16_t* tile, int c, int lane) {
    const int l15 = lane & 15, l4 = lane >> 4;
    bf16x8 f;
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = h * 16 + l4 * 4 + (l15 >> 2), cc = c + (l15 & 3) * 4;
        auto* p = (__attribute__((address_space(3))) s16x4*)(
            tile + (G ? at_g(row, cc) : at_x(row, cc)));
        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p);
        const bf16x4 b = __builtin_bit_cast(bf16x4, v);
        #pragma unroll
        for (int j = 0; j < 4; ++j) f[h * 4 + j] = b[j];
    }
    return f;
}

template <typename T>
__global__ __launch_bounds__(256, 2) void wgrad_kernel(Wgrad w) {
#ifdef __HIP_DEVICE_COMPILE__
    __shared__ __align__(16) uint16_t gt[2][32 * 256], xt[2][32 * 128];
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int l15 = lane & 15, l4 = lane >> 4;
    // each XCD takes one run of tiles of the same share, which walk over the
    // same rows side by side: its L2 fetches them once.  Dealt out one by one
    // instead, every XCD fetches everything, and memory sets the pace.
    const int xcd = blockIdx.x & 7, q = gridDim.x >> 3, rem = gridDim.x & 7;
    const int at = xcd * q + min(xcd, rem) + (blockIdx.x >> 3);
    const int tiles = gridDim.x / w.shares;
    const int share = at / tiles, tile = at - share * tiles;
    const int bn = tile / w.nbk * 2, bk = tile % w.nbk;
    const int wn = (wave >> 1) * 128, wk = (wave & 1) * 64;
    const int64_t ldg = (int64_t)w.nbn * 128, ldx = (int64_t)w.nbk * 128;
    const int lo = share * w.rows, hi = min(lo + w.rows, w.M);
    // an even number of steps; the last may lie behind row M, among zeros
    const int steps = ((hi - lo + 63) >> 6) * 2;  // <= 0: nothing is left

    // 16 bytes each: rows t / 16 and 16 + t / 16 of G, row t / 8 of X.  A
    // second block of G that is not there is read as the first.
    const int pg = t & 15, px = t & 7, rg = t >> 4, rx = t >> 3;
    const bool there = bn + (pg >> 3) < w.nbn;
    const int og = rg * (int)ldg + bn * 128 + (there ? pg : pg & 7) * 16;
    const int os = rg * w.Sn + bn + (there ? pg >> 3 : 0);
    const int ox = rx * (int)ldx + bk * 128 + px * 16, ot = rx * w.Sk + bk;
    // rows behind the last one are told by the lane's own offset alone
    const int og2[2] = {og, og + 16 * (int)ldg}, os2[2] = {os, os + 16 * w.Sn};
    struct Held { i32x4 v[3]; int e[3]; };
    auto load = [&](Held& h, int step) {
        const int64_t m = lo + (int64_t)step * 32;
        const int64_t left = max((int64_t)0, w.M - m);
        const auto bg = buffer_of(w.g + m * ldg, left * ldg);
        const auto bs = buffer_of(w.gs + m * w.Sn, left * w.Sn);
        const auto bx = buffer_of(w.x + m * ldx, left * ldx);
        const auto bt = buffer_of(w.xs + m * w.Sk, left * w.Sk);
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
            h.v[i] = __builtin_amdgcn_raw_buffer_load_b128(bg, og2[i], 0, 0);
            h.e[i] = __builtin_amdgcn_raw_buffer_load_b8(bs, os2[i], 0, 0);
        }
        h.v[2] = __builtin_amdgcn_raw_buffer_load_b128(bx, ox, 0, 0);
        h.e[2] = __builtin_amdgcn_raw_buffer_load_b8(bt, ot, 0, 0);
    };
    auto store = [&](const Held& h, int buf) {
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = i * 16 + rg;
            *(bf16x8*)&gt[buf][at_g(row, pg * 16)] =
                expand8(h.v[i][0], h.v[i][1], h.e[i]);
            *(bf16x8*)&gt[buf][at_g(row, pg * 16 + 8)] =
                expand8(h.v[i][2], h.v[i][3], h.e[i]);
        }
        #pragma unroll
        for (int j = 0; j < 4; j += 2) {
            const i32x4 u = __builtin_bit_cast(
                i32x4, expand8(h.v[2][j], h.v[2][j + 1], h.e[2]));
            const int c = (px >> 2) * 64 + (px & 3) * 4;
            *(i32x2*)&xt[buf][at_x(rx, c + j * 16)] = i32x2{u[0], u[1]};
            *(i32x2*)&xt[buf][at_x(rx, c + j * 16 + 16)] = i32x2{u[2], u[3]};
        }
    };
    f32x4 acc[8][4];
    #pragma unroll
    for (int i = 0; i < 8; ++i)
        #pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    Held h0, h1;  // even and odd steps
    load(h0, 0);
    load(h1, 1);
    store(h0, 0);
    load(h0, 2);
    __syncthreads();
    auto turn = [&](Held& next, int step, int buf) {
        store(next, buf ^ 1);  // all waves are past reading it
        load(next, step + 3);
        __builtin_amdgcn_sched_barrier(0);  // the loads are under way
        // all reads first: the way to LDS is waited for once
        bf16x8 fx[4], fg[8];
        #pragma unroll
        for (int j = 0; j < 4; ++j)
            fx[j] = tr_frag<false>(xt[buf], wk + j * 16, lane);
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            fg[i] = tr_frag<true>(gt[buf], wn + i * 16, lane);
        __builtin_amdgcn_sched_barrier(0);
        // rows of the MFMA's result are k, columns n
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            #pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    fx[j], fg[i], acc[i][j], 0, 0, 0);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
    };
    for (int step = 0; step < steps; step += 2) {
        turn(h1, step, 0);
        turn(h0, step + 1, 1);
    }
    const int k = bk * 128 + wk + l4 * 16;
    if (k >= w.K) return;
    const bool whole = k + 16 <= w.K && (w.K * sizeof(T) & 15) == 0;
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int n = bn * 128 + wn + i * 16 + l15;
        if (n >= w.N) continue;
        struct alignas(16) Pack { T t[16]; } p;
        #pragma unroll
        for (int j = 0; j < 4; ++j)
            #pragma unroll
            for (int e = 0; e < 4; ++e) p.t[j * 4 + e] = from_f<T>(acc[i][j][e]);
        T* out = (T*)w.dw + ((int64_t)share * w.N + n) * w.K + k;
        if (whole) {
            *(Pack*)out = p;
        } else {
            store_some(out, p.t, w.K - k);
        }
    }
#endif
}

template <typename T>
__global__ __launch_bounds__(256) void add_shares_kernel(
    const float* __restrict__ part, T* __restrict__ out, int shares,
    int64_t n) {
    for (int64_t i = threadIdx.x + (int64_t)blockIdx.x * 256; i < n;
         i += (int64_t)gridDim.x * 256) {
        float t = part[i];
        for (int s = 1; s < shares; ++s) t += part[s * n + i];
        out[i] = from_f<T>(t);
    }
}

#define RIQN_TYPE(code, T, ...)                     \
    switch (code) {                                 \
        case 0: { using T = float; __VA_ARGS__; } break;   \
        case 1: { using T = bf16_t; __VA_ARGS__; } break;  \
        default: { using T = fp16_t; __VA_ARGS__; } break; \
    }

// workgroups of 512 threads in a grid's first dimension, which holds less than
// 2^32 threads
constexpr int64_t MOST_512 = (1 << 23) - 1;

bool vec8(const void* p, int64_t ld, int C, int type) {
    const int size = type == 0 ? 4 : 2;
    return ((uintptr_t)p & 15) == 0 && (ld * size & 15) == 0 && (C & 7) == 0;
}

}  // namespace

extern "C" {

int riqn_fp8_quant_rows(const void* x, int type, int64_t ldx,
                        const uint8_t* mask, uint8_t* q, uint8_t* scale,
                        float* part, int groups, int R, int C, void* stream) {
    const int nb = (C + 127) >> 7, S = (nb + 3) & ~3;
    const bool wide = nb >= 4, vec = vec8(x, ldx, C, type);
    dim3 grid(wide ? (nb + 3) / 4 : nb, groups);
    hipStream_t st = (hipStream_t)stream;
#define RIQN_Q4(V, B, MK, SM)                                              \
    hipLaunchKernelGGL((quant_rows_kernel<T, V, B, MK, SM>), grid,         \
                       dim3(256), 0, st, (const T*)x, ldx, mask, q, scale, \
                       part, R, C, nb, S)
#define RIQN_Q3(V, B)                     \
    if (mask && part) RIQN_Q4(V, B, true, true);         \
    else if (mask) RIQN_Q4(V, B, true, false);           \
    else if (part) RIQN_Q4(V, B, false, true);           \
    else RIQN_Q4(V, B, false, false)
    RIQN_TYPE(type, T, {
        if (vec && wide) { RIQN_Q3(true, 4); }
        else if (vec) { RIQN_Q3(true, 1); }
        else if (wide) { RIQN_Q3(false, 4); }
        else { RIQN_Q3(false, 1); }
    })
    return (int)hipGetLastError();
}

int riqn_column_sum(const float* part, void* out, int type, int G, int C,
                    void* stream) {
    RIQN_TYPE(type, T, hipLaunchKernelGGL(
        column_sum_kernel<T>, dim3((C + 63) / 64), dim3(1024), 0,
        (hipStream_t)stream, part, (T*)out, G, C))
    return (int)hipGetLastError();
}

static Tiles tiles_of(const void* x, int64_t ldx, uint8_t* q, uint8_t* scale,
                      uint8_t* qt, uint8_t* scale_t, int R, int C) {
    const int nb = (C + 127) >> 7, nbt = (R + 127) >> 7;
    return {x, ldx, q, scale, qt, scale_t, R, C, nb, (nb + 3) & ~3, nbt,
            (nbt + 3) & ~3};
}

int riqn_fp8_quant_tiles(const void* x, int type, int64_t ldx, uint8_t* q,
                         uint8_t* scale, uint8_t* qt, uint8_t* scale_t, int R,
                         int C, void* stream) {
    const Tiles a = tiles_of(x, ldx, q, scale, qt, scale_t, R, C);
    hipStream_t st = (hipStream_t)stream;
    RIQN_TYPE(type, T, {
        if (vec8(x, ldx, C, type))
            hipLaunchKernelGGL((quant_tiles_kernel<T, true>), dim3(a.nb, a.nbt),
                               dim3(512), 0, st, a);
        else
            hipLaunchKernelGGL((quant_tiles_kernel<T, false>),
                               dim3(a.nb, a.nbt), dim3(512), 0, st, a);
    })
    return (int)hipGetLastError();
}

// x [M, C] by rows and w [N, C] by tiles, both of one type; where they are not
// laid out for it, by two launches
int riqn_fp8_quant_both(const void* x, int64_t ldx, uint8_t* xq, uint8_t* xs,
                        int groups, int M, const void* w, int64_t ldw,
                        uint8_t* wq, uint8_t* ws, uint8_t* wtq, uint8_t* wts,
                        int N, int C, int type, void* stream) {
    const int nb = (C + 127) >> 7, strips = nb >= 4 ? (nb + 3) / 4 : nb;
    const int64_t tiles = (int64_t)nb * ((N + 127) >> 7);
    if (!vec8(x, ldx, C, type) || !vec8(w, ldw, C, type) ||
        tiles + strips > MOST_512) {
        const int err = riqn_fp8_quant_rows(x, type, ldx, nullptr, xq, xs,
                                            nullptr, groups, M, C, stream);
        return err ? err
                   : riqn_fp8_quant_tiles(w, type, ldw, wq, ws, wtq, wts, N, C,
                                          stream);
    }
    const Tiles a = tiles_of(w, ldw, wq, ws, wtq, wts, N, C);
    // 8 waves here, 4 there
    const int half =
        (int)min((int64_t)(groups + 1) / 2, (MOST_512 - tiles) / strips);
    const dim3 grid((uint32_t)(tiles + strips * half));
    hipStream_t st = (hipStream_t)stream;
    RIQN_TYPE(type, T, {
        if (nb >= 4)
            hipLaunchKernelGGL((quant_both_kernel<T, 4>), grid, dim3(512), 0, st,
                               a, (const T*)x, ldx, xq, xs, M, nb, a.S,
                               (int)tiles, strips, half);
        else
            hipLaunchKernelGGL((quant_both_kernel<T, 1>), grid, dim3(512), 0, st,
                               a, (const T*)x, ldx, xq, xs, M, nb, a.S,
                               (int)tiles, strips, half);
    })
    return (int)hipGetLastError();
}

int riqn_fp8_dequant(const uint8_t* q, const uint8_t* scale, void* out,
                     int type, int R, int C, int shift, void* stream) {
    const int nb = (C + 127) >> 7, S = (nb + 3) & ~3;
    const int64_t n = (int64_t)R * ((C + 7) >> 3);
    const uint32_t blocks = (uint32_t)min((n + 255) / 256, (int64_t)1 << 20);
    const bool vec = vec8(out, C, C, type);
    RIQN_TYPE(type, T, {
        if (vec)
            hipLaunchKernelGGL((dequant_kernel<T, true>), dim3(blocks),
                               dim3(256), 0, (hipStream_t)stream, q, scale,
                               (T*)out, R, C, nb, S, shift);
        else
            hipLaunchKernelGGL((dequant_kernel<T, false>), dim3(blocks),
                               dim3(256), 0, (hipStream_t)stream, q, scale,
                               (T*)out, R, C, nb, S, shift);
    })
    return (int)hipGetLastError();
}

int riqn_fp8_gemm(const uint8_t* a, const uint8_t* as, int a_block_rows,
                  const uint8_t* b, const uint8_t* bs, int b_block_rows,
                  const void* bias, int bias_type, int relu, void* c,
                  int c_type, uint8_t* mask, int exact, int M, int N, int K,
                  void* stream) {
    const int nb = (K + 127) >> 7;
    Gemm g{a, as, b, bs, bias, c, mask, M, N, nb, (nb + 3) & ~3,
           a_block_rows == 128 ? 7 : 0, b_block_rows == 128 ? 7 : 0, bias_type,
           relu, nullptr, 0, K};
    hipStream_t st = (hipStream_t)stream;
    auto tiles = [&](int t) {
        return (int64_t)((M + t - 1) / t) * ((N + t - 1) / t);
    };
    // The largest tile of which there are enough for the 256 CUs: it moves the
    // fewest bytes.  Tiles of 64 that all fit at once, two on a CU, share their
    // steps out over two groups of waves.  Measured in us, scaled products in
    // bf16 / exact ones in fp32 (in bf16 2 to 6 % less), tiles of 32 (direct) | 64 shared | 64 | 128 | 256; [M, 1024, 3136]:
    //   M =  256    9 /  9 |  9 / 13 | 12 / 15 | 19 / 29 | 43 / 74
    //       1024   30 /    |  9 / 14 | 12 / 16 | 20 / 30 | 44 / 75
    //       2048           | 14 / 21 | 18 / 22 | 23 / 31 | 44 / 76
    //       2900           | 24 / 30 | 20 / 28 | 25 / 32 | 45 / 77
    //       4096           | 27 / 38 | 23 / 35 | 25 / 33 | 45 / 78
    //       8192           | 54 / 75 | 47 /    | 32 / 53 | 48 / 80
    //      16384           |         | 91 /    | 61 /    | 52 / 89
    // and [30000, 64, 512]:   6 /  8 |  6 /  8 |  7 / 10 | 11 / 17
    RIQN_TYPE(c_type, T, {
        if (M <= 16 && (N + 15) / 16 <= MOST_512) {
            hipLaunchKernelGGL((gemm_direct_kernel<1, 1, T>),
                               dim3((N + 15) / 16), dim3(512), 0, st, g);
        } else if (tiles(256) >= 192) {
            launch_tiles<2, 4, 8, 4, T>(g, exact, st);
        } else if (tiles(64) > 512) {
            if (tiles(128) >= 192) launch_tiles<2, 2, 4, 4, T>(g, exact, st);
            else launch_tiles<2, 2, 2, 2, T>(g, exact, st);
        } else if (tiles(32) > 256) {
            launch_shared<T>(g, exact, st);
        } else {
            hipLaunchKernelGGL((gemm_direct_kernel<2, 2, T>),
                               dim3((uint32_t)tiles(32)), dim3(512), 0, st, g);
        }
    })
    return (int)hipGetLastError();
}

// LDS that riqn_fp8_gemm_from takes for M rows of K columns
static int few_bytes(int64_t M, int K) {
    const int nb = (K + 127) >> 7;
    return (int)min(M * (nb * 128 + 16 + nb), (int64_t)1 << 30);
}

// whether a product of M rows that are not in 8 bits goes by one kernel
int riqn_fp8_few(int64_t M, int64_t N, int K) {
    return M <= 16 && few_bytes(M, K) <= 65536 && (N + 15) / 16 <= MOST_512;
}

// the product of a few rows that are not in 8 bits yet; c has x's type
int riqn_fp8_gemm_from(const void* x, int type, int64_t ldx, const uint8_t* b,
                       const uint8_t* bs, int b_block_rows, const void* bias,
                       int bias_type, int relu, void* c, int M, int N, int K,
                       void* stream) {
    const int nb = (K + 127) >> 7;
    Gemm g{nullptr, nullptr, b, bs, bias, c, nullptr, M, N, nb, (nb + 3) & ~3,
           0, b_block_rows == 128 ? 7 : 0, bias_type, relu, x, ldx, K};
    const dim3 grid((N + 15) / 16);
    const int bytes = few_bytes(M, K);
    hipStream_t st = (hipStream_t)stream;
    RIQN_TYPE(type, T, {
        if (vec8(x, ldx, K, type))
            hipLaunchKernelGGL((gemm_few_kernel<T, true>), grid, dim3(512),
                               bytes, st, g);
        else
            hipLaunchKernelGGL((gemm_few_kernel<T, false>), grid, dim3(512),
                               bytes, st, g);
    })
    return (int)hipGetLastError();
}

int riqn_fp8_wgrad(const uint8_t* g, const uint8_t* gs, const uint8_t* x,
                   const uint8_t* xs, void* dw, int type, float* part,
                   int shares, int M, int N, int K, void* stream) {
    const int nbn = (N + 127) >> 7, nbk = (K + 127) >> 7;
    const int rows = ((M + shares - 1) / shares + 63) & ~63;
    Wgrad w{g, gs, x, xs, shares > 1 ? (void*)part : dw, M, N, K, nbn,
            (nbn + 3) & ~3, nbk, (nbk + 3) & ~3, shares, rows};
    hipStream_t st = (hipStream_t)stream;
    dim3 grid((nbn + 1) / 2 * nbk * shares);
    RIQN_TYPE(shares > 1 ? 0 : type, T, hipLaunchKernelGGL(
        wgrad_kernel<T>, grid, dim3(256), 0, st, w))
    if (shares > 1) {
        const int64_t n = (int64_t)N * K;
        RIQN_TYPE(type, T, hipLaunchKernelGGL(
            add_shares_kernel<T>,
            dim3((uint32_t)min((n + 255) / 256, (int64_t)4096)), dim3(256), 0,
            st, part, (T*)dw, shares, n))
    }
    return (int)hipGetLastError();
}

}  // extern "C"
