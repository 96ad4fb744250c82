// Layer norm over the last axis for gfx950, forward and backward.
//
//   y  = h w + b           h = (x - mean) rstd, rstd = 1 / sqrt(var + eps)
//   dx = rstd (g - mean(g) - h mean(g h)),  g = dy w
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// The variance is the mean of squared distances from the mean, not a
// difference of squares: rows with a large offset keep their digits.  All of
// it in fp32, rounded once on the way out.  A register that adds up more than
// some 4096 columns would not do: terms of one sign are rounded the same way
// again and again, 2^16 of them 1e-3 off.  Longer sums go by runs.
//
// Both passes are bound by memory: forward reads x and writes y, backward
// reads x and dy and writes dx.  Rows of up to 4096 columns stay in registers
// between the sums and the result, 8 neighbours a lane and NV times that, so
// they are read once: [32768, 3136] in bf16 takes 79 to 85 us forward (4.8 TB/s
// and more), 139 to 143 backward and 5 to add up the parts (4.2 TB/s).  A team of 1 wave (up to 1024 columns) or 4 waves takes
// 4 rows at a time: 4 rows of loads in flight, one exchange of sums through
// LDS for all of them, and the weights stay in registers for the next 4.
// Longer rows are walked over again by a workgroup, value by value: [8192, 8192]
// in bf16 takes 177 us forward (1.5 TB/s) and 373 backward.
//
// dw and db: a lane adds its columns up in registers over all its rows,
// workgroup g writes part[g], and a second kernel adds the parts.  No atomics:
// the same inputs give the same bits.  A register takes 256 rows at most, there
// are as many workgroups as that needs: of 8192 terms of one sign the sum is
// 6e-5 off.
#include "common.h"
#include "riqn_kernels.h"

namespace {

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

struct bf16_t { unsigned short v; };
struct fp16_t { _Float16 v; };
DEV float to_f(float x) { return x; }
DEV float to_f(bf16_t x) { return bf16_to_f32(x.v); }
DEV float to_f(fp16_t x) { return (float)x.v; }
template <typename T> DEV T from_f(float x);
template <> DEV float from_f<float>(float x) { return x; }
template <> DEV bf16_t from_f<bf16_t>(float x) {
    return bf16_t{__builtin_bit_cast(unsigned short, (__bf16)x)};
}
template <> DEV fp16_t from_f<fp16_t>(float x) { return fp16_t{(_Float16)x}; }

template <typename T> struct Bits { using type = unsigned short; };
template <> struct Bits<float> { using type = uint32_t; };

// 8 values as they lie in memory.  Kept as whole registers: as single 16-bit
// values the compiler gives each a register of its own.
template <typename T>
struct Pack8 {
    static constexpr int WORDS = 2 * sizeof(T);
    uint32_t w[WORDS];
    DEV float get(int i) const {
        if (sizeof(T) == 4) return __uint_as_float(w[i]);
        const uint32_t u = w[i >> 1];
        const unsigned short h = (unsigned short)(i & 1 ? u >> 16 : u);
        return to_f(__builtin_bit_cast(T, (typename Bits<T>::type)h));
    }
    DEV void set(int i, float v) {
        const auto bits = __builtin_bit_cast(typename Bits<T>::type, from_f<T>(v));
        if (sizeof(T) == 4) w[i] = bits;
        else if (i & 1) w[i >> 1] |= (uint32_t)bits << 16;
        else w[i >> 1] = bits;
    }
};

// 8 neighbours from column `col`, or the row's last 8 where it has not as many
// there: loads are unconditional, as a branch around each would keep them apart.
// VEC: rows are 16-byte aligned and C is a multiple of 8; behind column C the
// values are then zeros where ZERO is set.  Otherwise the last lane takes some
// columns that the lane before it has too: `fresh` says which count.  Both store
// the same values for them.  [20001, 2999] in bf16 takes 133 us a step, with the
// last columns one by one, in a branch, 273.  A weight that alone lies off 16
// bytes costs nothing: [32768, 3136] takes 207 us a step, aligned 208.
template <typename T, bool VEC, bool ZERO>
DEV Pack8<T> load8(const T* p, int col, int C) {
    Pack8<T> v;
    if (VEC) {
        const uint32_t* q = (const uint32_t*)(p + min(col, C - 8));
        #pragma unroll
        for (int i = 0; i < Pack8<T>::WORDS; i += 4)
            *(u32x4*)&v.w[i] = *(const u32x4*)(q + i);
        if (ZERO) {
            #pragma unroll
            for (int i = 0; i < Pack8<T>::WORDS; ++i)
                v.w[i] = col < C ? v.w[i] : 0;
        }
    } else {
        __builtin_memcpy(v.w, p + min(col, C - 8), sizeof(v.w));
    }
    return v;
}
// whether the i-th of those 8 is a column of this lane's own
template <bool VEC>
DEV bool fresh(int col, int i, int C) {
    return VEC ? col < C : min(col, C - 8) + i >= col;
}
template <typename T>
DEV Pack8<T> all8(float x) {
    Pack8<T> v;
    #pragma unroll
    for (int i = 0; i < 8; ++i) v.set(i, x);
    return v;
}
template <typename T, bool VEC>
DEV void store8(T* p, int col, int C, const Pack8<T>& v) {
    if (col >= C) return;
    if (VEC) {
        #pragma unroll
        for (int i = 0; i < Pack8<T>::WORDS; i += 4)
            *(u32x4*)((uint32_t*)(p + col) + i) = *(const u32x4*)&v.w[i];
    } else {
        __builtin_memcpy(p + min(col, C - 8), v.w, sizeof(v.w));
    }
}

template <int N>
DEV float ror16_add(float v) {
    int o = __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf,
                                        0xf, false);
    return v + __int_as_float(o);
}
// sum over the wave, in every lane
DEV float wave_sum(float v) {
    v = ror16_add<8>(v);
    v = ror16_add<4>(v);
    v = ror16_add<2>(v);
    v = ror16_add<1>(v);
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
// sums over 4 waves, in every thread; `lds` is [4][2] floats
DEV void group_sums(float& s, float& t, float* lds) {
    s = wave_sum(s);
    t = wave_sum(t);
    __syncthreads();  // the last sums have been read
    if ((threadIdx.x & 63) == 0) {
        lds[(threadIdx.x >> 6) * 2] = s;
        lds[(threadIdx.x >> 6) * 2 + 1] = t;
    }
    __syncthreads();
    s = (lds[0] + lds[2]) + (lds[4] + lds[6]);
    t = (lds[1] + lds[3]) + (lds[5] + lds[7]);
}

struct NormFwd {
    const void *x, *w, *b;  // w, b may be null
    void* y;                // [R, C] contiguous
    float *mean, *rstd;     // [R], or null
    int64_t ldx;
    int R, C;
    float eps;
};

constexpr int RB = 4;  // rows a team takes at a time

// Sums of N values over a team of TW waves, in every lane.  `lds` is
// [2][4][N] floats; `turn` alternates, so that one barrier a sum is enough:
// what a slow wave still reads is not written before the next barrier.
template <int TW, int N>
DEV void team_sum(float (&v)[N], float* lds, int& turn) {
    #pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if (TW == 1) return;
    float* s = lds + turn * 4 * N;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) {
        #pragma unroll
        for (int i = 0; i < N; ++i) s[(threadIdx.x >> 6) * N + i] = v[i];
    }
    __syncthreads();
    #pragma unroll
    for (int i = 0; i < N; ++i)
        v[i] = (s[i] + s[N + i]) + (s[2 * N + i] + s[3 * N + i]);
}

// Makes the compiler take a loaded value for a new one: what was derived from
// it before a sum is derived again after it.  Kept instead, the fp32 values
// of 4 rows would take twice the registers and halve the waves in flight.
template <typename T>
DEV void forget(Pack8<T>& p) {
    #pragma unroll
    for (int i = 0; i < Pack8<T>::WORDS; ++i) asm volatile("" : "+v"(p.w[i]));
}

template <typename T, typename W, int TW, int NV, bool VEC>
__global__ __launch_bounds__(256) void norm_fwd_kernel(NormFwd a) {
    __shared__ float lds[2 * 4 * RB];
    const int t = threadIdx.x % (64 * TW);  // place in the team
    constexpr int TEAMS = 4 / TW;
    int turn = 0;
    Pack8<W> w[NV], b[NV];
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int col = (i * 64 * TW + t) * 8;
        w[i] = a.w ? load8<W, VEC, false>((const W*)a.w, col, a.C) : all8<W>(1.0f);
        b[i] = a.b ? load8<W, VEC, false>((const W*)a.b, col, a.C) : all8<W>(0.0f);
    }
    for (int64_t r0 = ((int64_t)blockIdx.x * TEAMS + threadIdx.x / (64 * TW)) * RB;
         r0 < a.R; r0 += (int64_t)gridDim.x * TEAMS * RB) {
        Pack8<T> x[RB][NV];
        #pragma unroll
        for (int k = 0; k < RB; ++k) {
            // rows behind the last one are read as the last
            const int64_t r = min(r0 + k, (int64_t)a.R - 1);
            #pragma unroll
            for (int i = 0; i < NV; ++i)
                x[k][i] = load8<T, VEC, true>((const T*)a.x + r * a.ldx,
                                        (i * 64 * TW + t) * 8, a.C);
        }
        float mean[RB], rstd[RB];
        #pragma unroll
        for (int k = 0; k < RB; ++k) {
            mean[k] = 0.0f;
            #pragma unroll
            for (int i = 0; i < NV; ++i)
                #pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (VEC || fresh<VEC>((i * 64 * TW + t) * 8, j, a.C))
                        mean[k] += x[k][i].get(j);
        }
        team_sum<TW, RB>(mean, lds, turn);
        #pragma unroll
        for (int k = 0; k < RB; ++k) {
            mean[k] /= a.C;
            #pragma unroll
            for (int i = 0; i < NV; ++i) forget(x[k][i]);
            rstd[k] = 0.0f;
            #pragma unroll
            for (int i = 0; i < NV; ++i) {
                #pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float d = x[k][i].get(j) - mean[k];
                    // what is not there counts for nothing
                    if (fresh<VEC>((i * 64 * TW + t) * 8, j, a.C))
                        rstd[k] += d * d;
                }
            }
        }
        team_sum<TW, RB>(rstd, lds, turn);
        #pragma unroll
        for (int k = 0; k < RB; ++k) {
            rstd[k] = 1.0f / sqrtf(rstd[k] / a.C + a.eps);
            const int64_t r = r0 + k;
            if (r >= a.R) continue;
            #pragma unroll
            for (int i = 0; i < NV; ++i) forget(x[k][i]);
            if (a.mean && t == 0) {
                a.mean[r] = mean[k];
                a.rstd[r] = rstd[k];
            }
            #pragma unroll
            for (int i = 0; i < NV; ++i) {
                Pack8<T> o;
                #pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float h = (x[k][i].get(j) - mean[k]) * rstd[k];
                    o.set(j, h * w[i].get(j) + b[i].get(j));
                }
                store8<T, VEC>((T*)a.y + r * a.C, (i * 64 * TW + t) * 8, a.C, o);
            }
        }
    }
}

// Sums of two values a column over the row, in every thread.  A thread's
// columns go in runs of 256: off by 2^-24 of its magnitude for each of 256 +
// C / 2^16 additions at most, where one after the other would be C / 256.
template <typename F>
DEV void long_sums(int C, float* lds, float& s, float& t, F add) {
    constexpr int RUN = 256 * 256;
    s = t = 0.0f;
    for (int c0 = threadIdx.x; c0 < C; c0 += RUN) {
        float p = 0.0f, q = 0.0f;
        const int end = min(c0 + RUN, C);
        for (int c = c0; c < end; c += 256) add(c, p, q);
        s += p;
        t += q;
    }
    group_sums(s, t, lds);
}

// any number of columns, for those above 4096 and below 8: a workgroup walks
// over its row three times.  The second walk also sums up the distances: their
// mean is what the first one's mean is off by, and its square what the mean of
// their squares has too much.
template <typename T, typename W>
__global__ __launch_bounds__(256) void norm_fwd_long_kernel(NormFwd a) {
    __shared__ float lds[8];
    for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.ldx;
        float s, s2;
        long_sums(a.C, lds, s, s2,
                  [&](int c, float& p, float&) { p += to_f(x[c]); });
        const float near = s / a.C;
        long_sums(a.C, lds, s, s2, [&](int c, float& p, float& q) {
            const float d = to_f(x[c]) - near;
            p += d;
            q += d * d;
        });
        const float off = s / a.C, mean = near + off;
        // squares past fp32's range leave an infinite variance, not inf - inf
        const float var = s2 < __builtin_inff() ? s2 / a.C - off * off : s2;
        // rounding may leave less than nothing; a NaN stays one
        const float rstd = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + a.eps);
        if (a.mean && threadIdx.x == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        T* y = (T*)a.y + r * a.C;
        for (int c = threadIdx.x; c < a.C; c += 256) {
            float z = (to_f(x[c]) - mean) * rstd;
            if (a.w) z *= to_f(((const W*)a.w)[c]);
            if (a.b) z += to_f(((const W*)a.b)[c]);
            y[c] = from_f<T>(z);
        }
    }
}

struct NormBwd {
    const void *dy, *x, *w;     // w may be null
    const float *mean, *rstd;   // [R]
    void* dx;                   // [R, C] contiguous, or null
    float* part;                // [gridDim.x][2][C]: dw, db, or null
    int64_t lddy, ldx;
    int R, C;
};

// 2 waves a SIMD: held to 3 the compiler spills, and [32768, 3136] in bf16
// took 165 us, the adding up of the parts included, where it takes 144 to 148
// (the bytes alone take 121 at the rate of a large copy).
template <typename T, typename W, int TW, int NV, bool VEC>
__global__ __launch_bounds__(256, 2) void norm_bwd_kernel(NormBwd a) {
    constexpr int TEAMS = 4 / TW;
    // sums of the teams; where teams are waves, also their parts in turn
    __shared__ float lds[TW == 1 ? 4 * NV * 512 : 2 * 2 * 4 * RB];
    const int t = threadIdx.x % (64 * TW);
    int turn = 0;
    Pack8<W> w[NV];
    float dw[NV][8], db[NV][8];
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
        // zeros behind column C: an infinite weight times dy's zeros were NaN
        w[i] = a.w ? load8<W, VEC, true>((const W*)a.w, (i * 64 * TW + t) * 8, a.C)
                   : all8<W>(1.0f);
        #pragma unroll
        for (int j = 0; j < 8; ++j) dw[i][j] = db[i][j] = 0.0f;
    }
    for (int64_t r0 = ((int64_t)blockIdx.x * TEAMS + threadIdx.x / (64 * TW)) * RB;
         r0 < a.R; r0 += (int64_t)gridDim.x * TEAMS * RB) {
        Pack8<T> x[RB][NV], dy[RB][NV];
        float mean[RB], rstd[RB];
        #pragma unroll
        for (int k = 0; k < RB; ++k) {
            const int64_t r = min(r0 + k, (int64_t)a.R - 1);
            mean[k] = a.mean[r];
            rstd[k] = a.rstd[r];
            #pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int col = (i * 64 * TW + t) * 8;
                x[k][i] = load8<T, VEC, false>((const T*)a.x + r * a.ldx, col, a.C);
                dy[k][i] = load8<T, VEC, true>((const T*)a.dy + r * a.lddy, col, a.C);
            }
        }
        float s[2 * RB];  // sums of g and of g h
        #pragma unroll
        for (int k = 0; k < RB; ++k) {
            s[2 * k] = s[2 * k + 1] = 0.0f;
            const bool there = r0 + k < a.R;
            #pragma unroll
            for (int i = 0; i < NV; ++i) {
                #pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // behind column C dy is zero, so nothing is added there
                    const bool own =
                        VEC || fresh<VEC>((i * 64 * TW + t) * 8, j, a.C);
                    const float d = there && own ? dy[k][i].get(j) : 0.0f;
                    const float h = (x[k][i].get(j) - mean[k]) * rstd[k];
                    // a weight of another lane's column may be infinite
                    const float g = own ? d * w[i].get(j) : 0.0f;
                    db[i][j] += d;
                    dw[i][j] += d * h;
                    // here, not at the loop's end with d and h of all rows
                    // kept until then, which is what the compiler would do
                    asm volatile("" : "+v"(db[i][j]), "+v"(dw[i][j]));
                    s[2 * k] += g;
                    s[2 * k + 1] += g * h;
                }
            }
            asm volatile("" : "+v"(s[2 * k]), "+v"(s[2 * k + 1]));
        }
        if (!a.dx) continue;
        team_sum<TW, 2 * RB>(s, lds, turn);
        #pragma unroll
        for (int k = 0; k < RB; ++k) {
            const int64_t r = r0 + k;
            if (r >= a.R) continue;
            const float c1 = s[2 * k] / a.C, c2 = s[2 * k + 1] / a.C;
            #pragma unroll
            for (int i = 0; i < NV; ++i) {
                forget(x[k][i]);
                forget(dy[k][i]);
                Pack8<T> o;
                #pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float d = dy[k][i].get(j);
                    const float h = (x[k][i].get(j) - mean[k]) * rstd[k];
                    const float g = d * w[i].get(j);
                    o.set(j, rstd[k] * (g - c1 - h * c2));
                }
                store8<T, VEC>((T*)a.dx + r * a.C, (i * 64 * TW + t) * 8, a.C, o);
            }
        }
    }
    if (!a.part) return;
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.C;
    #pragma unroll
    for (int which = 0; which < 2; ++which, part += a.C) {
        if (TW == 1) {  // the waves' parts, added in their order
            __syncthreads();
            #pragma unroll
            for (int i = 0; i < NV; ++i)
                #pragma unroll
                for (int j = 0; j < 8; ++j)
                    lds[(threadIdx.x >> 6) * NV * 512 + (i * 8 + j) * 64 + t] =
                        which ? db[i][j] : dw[i][j];
            __syncthreads();
            for (int c = threadIdx.x; c < a.C; c += 256) {
                const int j = c - (VEC ? c & ~7 : min(c & ~7, a.C - 8));
                const int at = ((c >> 9) * 8 + j) * 64 + ((c >> 3) & 63);
                part[c] = (lds[at] + lds[NV * 512 + at]) +
                          (lds[2 * NV * 512 + at] + lds[3 * NV * 512 + at]);
            }
        } else {
            #pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int col = (i * 64 * TW + t) * 8;
                #pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (fresh<VEC>(col, j, a.C))
                        part[(VEC ? col : min(col, a.C - 8)) + j] =
                            which ? db[i][j] : dw[i][j];
            }
        }
    }
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void norm_dx_long_kernel(NormBwd a) {
    __shared__ float lds[8];
    for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.ldx;
        const T* dy = (const T*)a.dy + r * a.lddy;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1, s2;
        long_sums(a.C, lds, s1, s2, [&](int c, float& p, float& q) {
            float g = to_f(dy[c]);
            if (a.w) g *= to_f(((const W*)a.w)[c]);
            p += g;
            q += g * ((to_f(x[c]) - mean) * rstd);
        });
        const float c1 = s1 / a.C, c2 = s2 / a.C;
        for (int c = threadIdx.x; c < a.C; c += 256) {
            float g = to_f(dy[c]);
            if (a.w) g *= to_f(((const W*)a.w)[c]);
            const float h = (to_f(x[c]) - mean) * rstd;
            ((T*)a.dx)[r * a.C + c] = from_f<T>(rstd * (g - c1 - h * c2));
        }
    }
}

// a column a thread, a share of the rows a workgroup; columns along x, of which
// a grid may have more than along y
template <typename T>
__global__ __launch_bounds__(256) void norm_part_long_kernel(NormBwd a) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.C) return;
    float dw = 0.0f, db = 0.0f;
    // in runs of 256 rows, then the runs
    for (int64_t r0 = blockIdx.y; r0 < a.R; r0 += 256 * (int64_t)gridDim.y) {
        float p = 0.0f, q = 0.0f;
        const int64_t end = min(r0 + 256 * (int64_t)gridDim.y, (int64_t)a.R);
        for (int64_t r = r0; r < end; r += gridDim.y) {
            const float d = to_f(((const T*)a.dy)[r * a.lddy + c]);
            const float h =
                (to_f(((const T*)a.x)[r * a.ldx + c]) - a.mean[r]) * a.rstd[r];
            p += d * h;
            q += d;
        }
        dw += p;
        db += q;
    }
    float* part = a.part + (int64_t)blockIdx.y * 2 * a.C;
    part[c] = dw;
    part[a.C + c] = db;
}

// dw, db [C] = sum over G of part[g][2][C]; either may be null.  64 columns
// and 16 shares of the parts a workgroup: a load depends on none before it.  A
// share goes in runs of 64 parts, then the runs.
template <typename W>
__global__ __launch_bounds__(1024) void norm_add_parts_kernel(
    const float* __restrict__ part, W* __restrict__ dw, W* __restrict__ db,
    int G, int C) {
    __shared__ float red[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), g0 = threadIdx.x >> 6;
    float t = 0.0f;
    if (c < 2 * C) {
        for (int from = g0; from < G; from += 16 * 64) {
            float p = 0.0f;
            const int end = min(from + 16 * 64, G);
            #pragma unroll 8
            for (int g = from; g < end; g += 16) p += part[(int64_t)g * 2 * C + c];
            t += p;
        }
    }
    red[g0][threadIdx.x & 63] = t;
    __syncthreads();
    if (g0 == 0 && c < 2 * C) {
        #pragma unroll
        for (int i = 1; i < 16; ++i) t += red[i][threadIdx.x];
        if (c < C) {
            if (dw) dw[c] = from_f<W>(t);
        } else if (db) {
            db[c - C] = from_f<W>(t);
        }
    }
}

bool aligned8(const void* p, int64_t ld, int size) {
    return ((uintptr_t)p & 15) == 0 && (ld * size & 15) == 0;
}

// types: 0 fp32, 1 bf16, 2 fp16; weights have x's type or fp32
#define RIQN_NORM_TYPES(type, wtype, ...)                                     \
    if (type == 0) { using T = float; using W = float; __VA_ARGS__; }         \
    else if (type == 1 && wtype == 1) { using T = bf16_t; using W = bf16_t; __VA_ARGS__; } \
    else if (type == 1) { using T = bf16_t; using W = float; __VA_ARGS__; }   \
    else if (wtype == 2) { using T = fp16_t; using W = fp16_t; __VA_ARGS__; } \
    else { using T = fp16_t; using W = float; __VA_ARGS__; }

// Columns -> waves a row and registers: 512 NV columns a wave.
#define RIQN_NORM_SHAPE(C, ...)                                                \
    if (C <= 512) { constexpr int TW = 1, NV = 1; __VA_ARGS__; }               \
    else if (C <= 1024) { constexpr int TW = 1, NV = 2; __VA_ARGS__; }         \
    else if (C <= 2048) { constexpr int TW = 4, NV = 1; __VA_ARGS__; }         \
    else { constexpr int TW = 4, NV = 2; __VA_ARGS__; }

int teams_of(int C) { return C <= 1024 ? 4 : 1; }

}  // namespace

extern "C" {

int riqn_norm_fwd(const void* x, int type, int64_t ldx, const void* w,
                  const void* b, int wtype, void* y, float* mean, float* rstd,
                  int R, int C, float eps, void* stream) {
    NormFwd a{x, w, b, y, mean, rstd, ldx, R, C, eps};
    const int size = type == 0 ? 4 : 2;
    const bool vec = (C & 7) == 0 && aligned8(x, ldx, size) &&
                     aligned8(y, C, size) && aligned8(w, 0, 1) &&
                     aligned8(b, 0, 1);
    hipStream_t st = (hipStream_t)stream;
    RIQN_NORM_TYPES(type, wtype, {
        if (C > 4096 || C < 8) {
            hipLaunchKernelGGL((norm_fwd_long_kernel<T, W>),
                               dim3(min(R, 1 << 16)), dim3(256), 0, st, a);
        } else {
            const int rows = RB * teams_of(C);  // of a workgroup at a time
            const dim3 grid(min((R + rows - 1) / rows, 2048));
            RIQN_NORM_SHAPE(C, {
                if (vec)
                    hipLaunchKernelGGL((norm_fwd_kernel<T, W, TW, NV, true>),
                                       grid, dim3(256), 0, st, a);
                else
                    hipLaunchKernelGGL((norm_fwd_kernel<T, W, TW, NV, false>),
                                       grid, dim3(256), 0, st, a);
            })
        }
    })
    return (int)hipGetLastError();
}

// workgroups of the backward pass, each of which leaves a part: 512, two a CU,
// but as many as hold a register to 256 rows, or where it folds its runs to
// 256 of them
int riqn_norm_groups(int R, int C) {
    const bool folds = C > 4096 || C < 8;
    const int rows = folds ? 4 : RB * teams_of(C);
    const int most = folds ? 256 * 256 : 256 * teams_of(C);
    return min((R + rows - 1) / rows, max(512, (R + most - 1) / most));
}

// part: [groups][2][C] fp32 workspace, or null where neither dw nor db is
// asked for
int riqn_norm_bwd(const void* dy, const void* x, int type, int64_t lddy,
                  int64_t ldx, const void* w, int wtype, const float* mean,
                  const float* rstd, void* dx, void* dw, void* db, float* part,
                  int groups, int R, int C, void* stream) {
    NormBwd a{dy, x, w, mean, rstd, dx, part, lddy, ldx, R, C};
    const int size = type == 0 ? 4 : 2;
    const bool vec = (C & 7) == 0 && aligned8(x, ldx, size) &&
                     aligned8(dy, lddy, size) && aligned8(dx, C, size) &&
                     aligned8(w, 0, 1);
    hipStream_t st = (hipStream_t)stream;
    RIQN_NORM_TYPES(type, wtype, {
        if (C > 4096 || C < 8) {
            if (dx)
                hipLaunchKernelGGL((norm_dx_long_kernel<T, W>),
                                   dim3(min(R, 1 << 16)), dim3(256), 0, st, a);
            if (part)
                hipLaunchKernelGGL((norm_part_long_kernel<T>),
                                   dim3((C + 255) / 256, groups), dim3(256), 0,
                                   st, a);
        } else {
            RIQN_NORM_SHAPE(C, {
                if (vec)
                    hipLaunchKernelGGL((norm_bwd_kernel<T, W, TW, NV, true>),
                                       dim3(groups), dim3(256), 0, st, a);
                else
                    hipLaunchKernelGGL((norm_bwd_kernel<T, W, TW, NV, false>),
                                       dim3(groups), dim3(256), 0, st, a);
            })
        }
        if (part)
            hipLaunchKernelGGL((norm_add_parts_kernel<W>),
                               dim3((2 * C + 63) / 64), dim3(1024), 0, st,
                               part, (W*)dw, (W*)db, groups, C);
    })
    return (int)hipGetLastError();
}

}  // extern "C"
