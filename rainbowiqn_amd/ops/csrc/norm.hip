// Layer norm over the last axis for gfx950, forward and backward.
//
//   y  = h w + b           h = (x - mean) rstd, rstd = 1 / sqrt(var + eps)
//   dx = rstd (g - mean(g) - h mean(g h)),  g = dy w
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// The variance is the mean of squared distances from the mean, not a
// difference of squares: rows with a large offset keep their digits.  All of
// it in fp32, rounded once on the way out.
//
// Both passes are bound by memory: forward reads x and writes y, backward
// reads x and dy and writes dx.  Up to 4096 columns one wave holds a row in
// registers (8 neighbours a lane, NV times), so a row is read once and no
// wave waits for another; longer rows are walked over again by a workgroup,
// out of the cache.
//
// dw and db: each wave adds its rows up in registers, the workgroup's waves
// add theirs in LDS one after the other, and workgroup g writes part[g]; a
// second kernel adds the parts.  No atomics: the same inputs give the same
// bits.
#include "common.h"
#include "riqn_kernels.h"

namespace {

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

template <typename T, bool VEC> struct Pack8;
template <typename T> struct alignas(16) Pack8<T, true> { T t[8]; };
template <typename T> struct Pack8<T, false> { T t[8]; };

// 8 neighbours from column `col`, zeros behind column C.  VEC: rows are
// 16-byte aligned and C is a multiple of 8.
template <typename T, bool VEC>
DEV Pack8<T, VEC> load8(const T* p, int col, int C) {
    Pack8<T, VEC> v;
    if (col + 8 <= C) {
        v = *(const Pack8<T, VEC>*)(p + col);
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            v.t[i] = (!VEC && col + i < C) ? p[col + i] : T{};
    }
    return v;
}
template <typename T, bool VEC>
DEV void store8(T* p, int col, int C, const Pack8<T, VEC>& v) {
    if (col + 8 <= C) {
        *(Pack8<T, VEC>*)(p + col) = v;
    } else if (!VEC) {
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < C) p[col + i] = v.t[i];
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
// sum over 4 waves, in every thread
DEV float group_sum(float v, float* lds) {
    v = wave_sum(v);
    __syncthreads();  // the last sum has been read
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

struct NormFwd {
    const void *x, *w, *b;  // w, b may be null
    void* y;                // [R, C] contiguous
    float *mean, *rstd;     // [R], or null
    int64_t ldx;
    int R, C;
    float eps;
};

template <typename T, typename W, int NV, bool VEC>
__global__ __launch_bounds__(256) void norm_fwd_kernel(NormFwd a) {
    const int lane = threadIdx.x & 63;
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= a.R) return;
    const T* x = (const T*)a.x + r * a.ldx;
    float v[NV][8];
    float s = 0.0f;
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
        const auto p = load8<T, VEC>(x, (i * 64 + lane) * 8, a.C);
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[i][j] = to_f(p.t[j]);
            s += v[i][j];
        }
    }
    const float mean = wave_sum(s) / a.C;
    s = 0.0f;
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            // what is not there counts for nothing
            v[i][j] = (i * 64 + lane) * 8 + j < a.C ? v[i][j] - mean : 0.0f;
            s += v[i][j] * v[i][j];
        }
    }
    const float rstd = 1.0f / sqrtf(wave_sum(s) / a.C + a.eps);
    if (a.mean && lane == 0) {
        a.mean[r] = mean;
        a.rstd[r] = rstd;
    }
    T* y = (T*)a.y + r * a.C;
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int col = (i * 64 + lane) * 8;
        Pack8<W, VEC> w, b;
        if (a.w) w = load8<W, VEC>((const W*)a.w, col, a.C);
        if (a.b) b = load8<W, VEC>((const W*)a.b, col, a.C);
        Pack8<T, VEC> o;
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            float z = v[i][j] * rstd;
            if (a.w) z *= to_f(w.t[j]);
            if (a.b) z += to_f(b.t[j]);
            o.t[j] = from_f<T>(z);
        }
        store8<T, VEC>(y, col, a.C, o);
    }
}

// any number of columns: a workgroup walks over its row three times
template <typename T, typename W>
__global__ __launch_bounds__(256) void norm_fwd_long_kernel(NormFwd a) {
    __shared__ float lds[4];
    for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.ldx;
        float s = 0.0f;
        for (int c = threadIdx.x; c < a.C; c += 256) s += to_f(x[c]);
        const float mean = group_sum(s, lds) / a.C;
        s = 0.0f;
        for (int c = threadIdx.x; c < a.C; c += 256) {
            const float d = to_f(x[c]) - mean;
            s += d * d;
        }
        const float rstd = 1.0f / sqrtf(group_sum(s, lds) / a.C + a.eps);
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

template <typename T, typename W, int NV, bool VEC>
__global__ __launch_bounds__(256) void norm_bwd_kernel(NormBwd a) {
    extern __shared__ float lds[];  // [2][C] where part is asked for
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float dw[NV][8], db[NV][8];
    #pragma unroll
    for (int i = 0; i < NV; ++i)
        #pragma unroll
        for (int j = 0; j < 8; ++j) dw[i][j] = db[i][j] = 0.0f;
    for (int64_t r = (int64_t)blockIdx.x * 4 + wave; r < a.R;
         r += (int64_t)gridDim.x * 4) {
        Pack8<T, VEC> x[NV], dy[NV];
        #pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * 64 + lane) * 8;
            x[i] = load8<T, VEC>((const T*)a.x + r * a.ldx, col, a.C);
            dy[i] = load8<T, VEC>((const T*)a.dy + r * a.lddy, col, a.C);
        }
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
        #pragma unroll
        for (int i = 0; i < NV; ++i) {
            Pack8<W, VEC> w;
            if (a.w) w = load8<W, VEC>((const W*)a.w, (i * 64 + lane) * 8, a.C);
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                // behind column C dy is zero, so nothing is added there
                const float d = to_f(dy[i].t[j]);
                const float h = (to_f(x[i].t[j]) - mean) * rstd;
                const float g = a.w ? d * to_f(w.t[j]) : d;
                db[i][j] += d;
                dw[i][j] += d * h;
                s1 += g;
                s2 += g * h;
            }
        }
        if (!a.dx) continue;
        const float c1 = wave_sum(s1) / a.C, c2 = wave_sum(s2) / a.C;
        #pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * 64 + lane) * 8;
            Pack8<W, VEC> w;
            if (a.w) w = load8<W, VEC>((const W*)a.w, col, a.C);
            Pack8<T, VEC> o;
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = to_f(dy[i].t[j]);
                const float h = (to_f(x[i].t[j]) - mean) * rstd;
                const float g = a.w ? d * to_f(w.t[j]) : d;
                o.t[j] = from_f<T>(rstd * (g - c1 - h * c2));
            }
            store8<T, VEC>((T*)a.dx + r * a.C, col, a.C, o);
        }
    }
    if (!a.part) return;
    for (int k = 0; k < 4; ++k) {
        if (wave == k) {
            #pragma unroll
            for (int i = 0; i < NV; ++i) {
                #pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = (i * 64 + lane) * 8 + j;
                    if (c < a.C) {
                        lds[c] = dw[i][j] + (k ? lds[c] : 0.0f);
                        lds[a.C + c] = db[i][j] + (k ? lds[a.C + c] : 0.0f);
                    }
                }
            }
        }
        __syncthreads();
    }
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.C;
    for (int c = threadIdx.x; c < 2 * a.C; c += 256) part[c] = lds[c];
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void norm_dx_long_kernel(NormBwd a) {
    __shared__ float lds[4];
    for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.ldx;
        const T* dy = (const T*)a.dy + r * a.lddy;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
        for (int c = threadIdx.x; c < a.C; c += 256) {
            float g = to_f(dy[c]);
            if (a.w) g *= to_f(((const W*)a.w)[c]);
            s1 += g;
            s2 += g * ((to_f(x[c]) - mean) * rstd);
        }
        const float c1 = group_sum(s1, lds) / a.C, c2 = group_sum(s2, lds) / a.C;
        for (int c = threadIdx.x; c < a.C; c += 256) {
            float g = to_f(dy[c]);
            if (a.w) g *= to_f(((const W*)a.w)[c]);
            const float h = (to_f(x[c]) - mean) * rstd;
            ((T*)a.dx)[r * a.C + c] = from_f<T>(rstd * (g - c1 - h * c2));
        }
    }
}

// a column a thread, a share of the rows a workgroup
template <typename T>
__global__ __launch_bounds__(256) void norm_part_long_kernel(NormBwd a) {
    const int c = blockIdx.y * 256 + threadIdx.x;
    if (c >= a.C) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
        const float d = to_f(((const T*)a.dy)[r * a.lddy + c]);
        const float h =
            (to_f(((const T*)a.x)[r * a.ldx + c]) - a.mean[r]) * a.rstd[r];
        dw += d * h;
        db += d;
    }
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.C;
    part[c] = dw;
    part[a.C + c] = db;
}

// dw, db [C] = sum over G of part[g][2][C]; either may be null
template <typename W>
__global__ __launch_bounds__(256) void norm_add_parts_kernel(
    const float* __restrict__ part, W* __restrict__ dw, W* __restrict__ db,
    int G, int C) {
    __shared__ float red[8][32];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), g0 = threadIdx.x >> 5;
    float t = 0.0f;
    if (c < 2 * C)
        for (int g = g0; g < G; g += 8) t += part[(int64_t)g * 2 * C + c];
    red[g0][threadIdx.x & 31] = t;
    __syncthreads();
    if (g0 == 0 && c < 2 * C) {
        #pragma unroll
        for (int i = 1; i < 8; ++i) t += red[i][threadIdx.x];
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

#define RIQN_NORM_NV(C, ...)                                   \
    if (C <= 512) { constexpr int NV = 1; __VA_ARGS__; }       \
    else if (C <= 1024) { constexpr int NV = 2; __VA_ARGS__; } \
    else if (C <= 2048) { constexpr int NV = 4; __VA_ARGS__; } \
    else { constexpr int NV = 8; __VA_ARGS__; }

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
        if (C > 4096) {
            hipLaunchKernelGGL((norm_fwd_long_kernel<T, W>),
                               dim3(min(R, 1 << 16)), dim3(256), 0, st, a);
        } else {
            const dim3 grid((R + 3) / 4);
            RIQN_NORM_NV(C, {
                if (vec)
                    hipLaunchKernelGGL((norm_fwd_kernel<T, W, NV, true>), grid,
                                       dim3(256), 0, st, a);
                else
                    hipLaunchKernelGGL((norm_fwd_kernel<T, W, NV, false>),
                                       grid, dim3(256), 0, st, a);
            })
        }
    })
    return (int)hipGetLastError();
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
        if (C > 4096) {
            if (dx)
                hipLaunchKernelGGL((norm_dx_long_kernel<T, W>),
                                   dim3(min(R, 1 << 16)), dim3(256), 0, st, a);
            if (part)
                hipLaunchKernelGGL((norm_part_long_kernel<T>),
                                   dim3(groups, (C + 255) / 256), dim3(256), 0,
                                   st, a);
        } else {
            const uint32_t bytes = part ? 2 * C * sizeof(float) : 0;
            RIQN_NORM_NV(C, {
                if (vec)
                    hipLaunchKernelGGL((norm_bwd_kernel<T, W, NV, true>),
                                       dim3(groups), dim3(256), bytes, st, a);
                else
                    hipLaunchKernelGGL((norm_bwd_kernel<T, W, NV, false>),
                                       dim3(groups), dim3(256), bytes, st, a);
            })
        }
        if (part)
            hipLaunchKernelGGL((norm_add_parts_kernel<W>),
                               dim3((2 * C + 31) / 32), dim3(256), 0, st, part,
                               (W*)dw, (W*)db, groups, C);
    })
    return (int)hipGetLastError();
}

}  // extern "C"
