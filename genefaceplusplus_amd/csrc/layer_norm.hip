// layer_norm.hip -- layer norm over the last axis, forward and backward, with the reduction of the weight's and bias' gradients (gfx950).
//
//   mean = sum x / N, rstd = 1 / sqrt(sum (x - mean)^2 / N + eps), xhat = (x - mean) rstd, y = xhat w + b
//   g = dy w:   dx = rstd (g - mean(g) - xhat mean(g xhat)),   dw = sum_rows dy xhat,   db = sum_rows dy
//
// Bound by memory: a forward pass reads x and writes y, a backward pass reads x and dy and writes dx.  A row is therefore held in registers between its
// statistics and its output (the variance is that of the centred values, not E x^2 - mean^2), by one wavefront or one workgroup of 256.  Forward: rows of up to 8 192 elements,
// fp32 rows in vectors up to 4 096; backward, which holds two rows and the column sums: up to 4 096, fp32 rows in vectors up to 2 048.  Longer rows are read again out of the
// caches, three times in the forward pass, twice for dx, and once more from memory for the column sums (8 192 x 8 192 bf16: forward 50 us, backward 209; fp32 157 and 339;
// 13 000 x 4 096 bf16, still in registers: 37 and 108).  Statistics, both row sums of the backward pass and the column sums are fp32 for every type; the outputs
// are rounded once.  The column sums of dw / db stay in registers over the rows of a workgroup, leave as one partial row per workgroup and are added in a fixed
// order by a second launch: no atomics, the same bits every time.
// Measured: 13 000 x 1 024 bf16 with fp32 parameters: forward 12.5 us (53 MB, 4.3 TB/s), backward 21.2 (80 MB, 3.8 TB/s) and 3.9 for the column sums; 65 537 x 204 fp32: forward
// 23.9 us (107 MB, 4.5 TB/s), backward 28.8 (160 MB, 5.6 TB/s) and 3.9.  Rows that 16-byte vectors do not divide go one element at a time: 24.7 and 36.3, 32.2 and 47.0.
// One row of 1 024: 2.7 us, a launch.
#include <algorithm>

#include "gfpp_common.h"

namespace gfpp {

template <typename T>
struct LnVec;      // 16 bytes of T
template <> struct LnVec<float> { typedef float v __attribute__((ext_vector_type(4))); };
template <> struct LnVec<_Float16> { typedef _Float16 v __attribute__((ext_vector_type(8))); };
template <> struct LnVec<__bf16> { typedef __bf16 v __attribute__((ext_vector_type(8))); };

// VEC elements at p, widened (VEC == 1: the rows whose start, pitch or width is no multiple of 16 bytes)
template <typename T, int VEC>
__device__ __forceinline__ void ln_load(const T *p, float (&out)[VEC]) {
    if constexpr (VEC == 1) {
        out[0] = (float)p[0];
    } else {
        const typename LnVec<T>::v t = *reinterpret_cast<const typename LnVec<T>::v *>(p);
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[e] = (float)t[e];
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void ln_store(T *p, const float (&in)[VEC]) {
    if constexpr (VEC == 1) {
        p[0] = (T)in[0];
    } else {
        typename LnVec<T>::v t;
#pragma unroll
        for (int e = 0; e < VEC; ++e) t[e] = (T)in[e];
        *reinterpret_cast<typename LnVec<T>::v *>(p) = t;
    }
}
// parameters: fp32 or the type of x (wave-uniform choice); NULL: the given constant
template <typename T, int VEC>
__device__ __forceinline__ void ln_param(const void *p, bool f32, uint32_t at, float none, float (&out)[VEC]) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[e] = none;
    } else if (f32) {
        const float *q = static_cast<const float *>(p) + at;
        if constexpr (VEC == 1) {
            out[0] = q[0];
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
                const LnVec<float>::v t = *reinterpret_cast<const LnVec<float>::v *>(q + e);
#pragma unroll
                for (int k = 0; k < 4; ++k) out[e + k] = t[k];
            }
        }
    } else {
        ln_load<T, VEC>(static_cast<const T *>(p) + at, out);
    }
}

// sum over the wavefront, in a scalar register: data-parallel moves inside the vector unit (shifts within rows of 16 lanes, then row to row) instead of six round
// trips through the LDS crossbar
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float wave_sum(float v) {
    v = dpp_add<0x111, 0xf>(v);                        // row_shr 1, 2, 4, 8: lane 15 of a row has its sum
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);                        // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3: lane 63 has all
    v = dpp_add<0x143, 0xc>(v);
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
// sum over the WG threads that share a row, in every one of them; `box`: LDS of one float per wavefront, free again after the next call's first barrier
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *box) {
    v = wave_sum(v);
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) v += box[w];
    }
    return v;
}

struct LnArgs {
    const void *x, *dy, *weight, *bias;
    void *y;                      // forward: y; backward: dx (may be NULL)
    float *mean, *rstd;           // forward: may be NULL
    float *partial;               // backward: [gridDim.x][2][N], or NULL
    uint64_t M;
    int64_t xs, dys;              // row pitches in elements
    uint32_t N;
    float eps;
    int param_f32;
};

// TPR threads per row (64: a wavefront, 256: the workgroup), NV vectors of VEC elements per thread, R rows of a wavefront at a time: their loads are in flight together
template <typename T, int VEC, int TPR, int NV, int R>
__global__ __launch_bounds__(256) void k_layer_norm(LnArgs a) {
    __shared__ float box[4];
    constexpr int RPW = 256 / TPR;
    const uint32_t t = threadIdx.x % TPR, sub = TPR == 64 ? (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / TPR)) : 0;
    const float n = (float)a.N;
    for (uint64_t row0 = ((uint64_t)blockIdx.x * RPW + sub) * R; row0 < a.M; row0 += (uint64_t)gridDim.x * RPW * R) {      // (TPR 256: the same in all threads)
        float v[R][NV][VEC];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const T *x = static_cast<const T *>(a.x) + (int64_t)(row0 + q < a.M ? row0 + q : a.M - 1) * a.xs;            // (the last row again: nothing is written twice)
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const uint32_t c = (k * TPR + t) * VEC;
                if (c < a.N) ln_load<T, VEC>(x + c, v[q][k]);
            }
        }
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const uint64_t row = row0 + q;
            if (row >= a.M) break;
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if ((k * TPR + t) * VEC < a.N)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) s += v[q][k][e];
            const float mean = row_sum<TPR>(s, box) / n;
            s = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if ((k * TPR + t) * VEC < a.N)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float d = v[q][k][e] - mean;
                        s = fmaf(d, d, s);
                    }
            const float rstd = 1.0f / sqrtf(row_sum<TPR>(s, box) / n + a.eps);
            T *y = static_cast<T *>(a.y) + row * a.N;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const uint32_t c = (k * TPR + t) * VEC;
                if (c < a.N) {
                    float w[VEC], b[VEC];
                    ln_param<T, VEC>(a.weight, a.param_f32, c, 1.0f, w);
                    ln_param<T, VEC>(a.bias, a.param_f32, c, 0.0f, b);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) w[e] = fmaf((v[q][k][e] - mean) * rstd, w[e], b[e]);
                    ln_store<T, VEC>(y + c, w);
                }
            }
            if (t == 0 && a.mean) {
                a.mean[row] = mean;
                a.rstd[row] = rstd;
            }
        }
    }
}

// rows beyond the register forms: three readings, the second and third out of the cache
template <typename T, int VEC>
__global__ __launch_bounds__(256) void k_layer_norm_long(LnArgs a) {
    __shared__ float box[4];
    const uint32_t t = threadIdx.x;
    const float n = (float)a.N;
    for (uint64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.xs;
        float v[VEC], s = 0.0f;
        for (uint32_t c = t * VEC; c < a.N; c += 256 * VEC) {
            ln_load<T, VEC>(x + c, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += v[e];
        }
        const float mean = row_sum<256>(s, box) / n;
        s = 0.0f;
        for (uint32_t c = t * VEC; c < a.N; c += 256 * VEC) {
            ln_load<T, VEC>(x + c, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = v[e] - mean;
                s = fmaf(d, d, s);
            }
        }
        const float rstd = 1.0f / sqrtf(row_sum<256>(s, box) / n + a.eps);
        T *y = static_cast<T *>(a.y) + row * a.N;
        for (uint32_t c = t * VEC; c < a.N; c += 256 * VEC) {
            float w[VEC], b[VEC];
            ln_load<T, VEC>(x + c, v);
            ln_param<T, VEC>(a.weight, a.param_f32, c, 1.0f, w);
            ln_param<T, VEC>(a.bias, a.param_f32, c, 0.0f, b);
#pragma unroll
            for (int e = 0; e < VEC; ++e) w[e] = fmaf((v[e] - mean) * rstd, w[e], b[e]);
            ln_store<T, VEC>(y + c, w);
        }
        if (t == 0 && a.mean) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

// dx of every row, and this workgroup's share of dw and db: a thread keeps the sums of its own columns over all its rows
template <typename T, int VEC, int TPR, int NV, int R>
__global__ __launch_bounds__(256) void k_layer_norm_bwd(LnArgs a) {
    __shared__ float box[4];
    extern __shared__ float cols[];                    // TPR == 64: [2][N], the wavefronts' sums one after the other
    constexpr int RPW = 256 / TPR;
    const uint32_t t = threadIdx.x % TPR, sub = TPR == 64 ? (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / TPR)) : 0;
    const float n = (float)a.N;
    float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const uint32_t c = (k * TPR + t) * VEC;
        if (c < a.N) ln_param<T, VEC>(a.weight, a.param_f32, c, 1.0f, w[k]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[k][e] = db[k][e] = 0.0f;
    }
    for (uint64_t row0 = ((uint64_t)blockIdx.x * RPW + sub) * R; row0 < a.M; row0 += (uint64_t)gridDim.x * RPW * R) {      // (TPR 256: the same in all threads)
        float xs[R][NV][VEC], gs[R][NV][VEC], means[R], rstds[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const uint64_t row = row0 + q < a.M ? row0 + q : a.M - 1;
            const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.xs, *dy = static_cast<const T *>(a.dy) + (int64_t)row * a.dys;
            means[q] = a.mean[row];
            rstds[q] = a.rstd[row];
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const uint32_t c = (k * TPR + t) * VEC;
                if (c < a.N) {
                    ln_load<T, VEC>(x + c, xs[q][k]);
                    ln_load<T, VEC>(dy + c, gs[q][k]);
                }
            }
        }
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const uint64_t row = row0 + q;
            if (row >= a.M) break;
            const float mean = means[q], rstd = rstds[q];
            float(&xh)[NV][VEC] = xs[q], (&g)[NV][VEC] = gs[q];
            float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if ((k * TPR + t) * VEC < a.N)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        xh[k][e] = (xh[k][e] - mean) * rstd;
                        db[k][e] += g[k][e];
                        dw[k][e] = fmaf(g[k][e], xh[k][e], dw[k][e]);
                        g[k][e] *= w[k][e];
                        s0 += g[k][e];
                        s1 = fmaf(g[k][e], xh[k][e], s1);
                    }
            if (a.y) {
                s0 = row_sum<TPR>(s0, box) / n;
                s1 = row_sum<TPR>(s1, box) / n;
                T *dx = static_cast<T *>(a.y) + row * a.N;
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const uint32_t c = (k * TPR + t) * VEC;
                    if (c < a.N) {
                        float o[VEC];
#pragma unroll
                        for (int e = 0; e < VEC; ++e) o[e] = rstd * (g[k][e] - s0 - xh[k][e] * s1);
                        ln_store<T, VEC>(dx + c, o);
                    }
                }
            }
        }
    }
    if (!a.partial) return;
    float *out = a.partial + (uint64_t)blockIdx.x * 2 * a.N;
    if constexpr (TPR == 64) {
        for (uint32_t turn = 0; turn < 4; ++turn) {
            if (sub == turn) {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const uint32_t c = (k * TPR + t) * VEC;
                    if (c < a.N)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            cols[c + e] = turn ? cols[c + e] + dw[k][e] : dw[k][e];
                            cols[a.N + c + e] = turn ? cols[a.N + c + e] + db[k][e] : db[k][e];
                        }
                }
            }
            __syncthreads();
        }
        for (uint32_t c = threadIdx.x; c < 2 * a.N; c += 256) out[c] = cols[c];
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t c = (k * TPR + t) * VEC;
            if (c < a.N)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    out[c + e] = dw[k][e];
                    out[a.N + c + e] = db[k][e];
                }
        }
    }
}

// the same for rows beyond the register forms: a workgroup takes 256 VEC columns at a time (blockIdx.y) for the column sums, dx by a launch of its own
template <typename T, int VEC>
__global__ __launch_bounds__(256) void k_layer_norm_bwd_long(LnArgs a) {
    __shared__ float box[4];
    const uint32_t t = threadIdx.x;
    const float n = (float)a.N;
    for (uint64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.xs, *dy = static_cast<const T *>(a.dy) + (int64_t)row * a.dys;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float xh[VEC], g[VEC], w[VEC], s0 = 0.0f, s1 = 0.0f;
        for (uint32_t c = t * VEC; c < a.N; c += 256 * VEC) {
            ln_load<T, VEC>(x + c, xh);
            ln_load<T, VEC>(dy + c, g);
            ln_param<T, VEC>(a.weight, a.param_f32, c, 1.0f, w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float gw = g[e] * w[e];
                s0 += gw;
                s1 = fmaf(gw, (xh[e] - mean) * rstd, s1);
            }
        }
        s0 = row_sum<256>(s0, box) / n;
        s1 = row_sum<256>(s1, box) / n;
        T *dx = static_cast<T *>(a.y) + row * a.N;
        for (uint32_t c = t * VEC; c < a.N; c += 256 * VEC) {
            float o[VEC];
            ln_load<T, VEC>(x + c, xh);
            ln_load<T, VEC>(dy + c, g);
            ln_param<T, VEC>(a.weight, a.param_f32, c, 1.0f, w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = rstd * (g[e] * w[e] - s0 - (xh[e] - mean) * rstd * s1);
            ln_store<T, VEC>(dx + c, o);
        }
    }
}
template <typename T, int VEC>
__global__ __launch_bounds__(256) void k_layer_norm_cols_long(LnArgs a) {
    for (uint32_t c = (blockIdx.y * 256 + threadIdx.x) * VEC; c < a.N; c += gridDim.y * 256 * VEC) {
        float dw[VEC], db[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[e] = db[e] = 0.0f;
        for (uint64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
            float x[VEC], g[VEC];
            ln_load<T, VEC>(static_cast<const T *>(a.x) + (int64_t)row * a.xs + c, x);
            ln_load<T, VEC>(static_cast<const T *>(a.dy) + (int64_t)row * a.dys + c, g);
            const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                db[e] += g[e];
                dw[e] = fmaf(g[e], (x[e] - mean) * rstd, dw[e]);
            }
        }
        float *out = a.partial + (uint64_t)blockIdx.x * 2 * a.N + c;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            out[e] = dw[e];
            out[a.N + e] = db[e];
        }
    }
}

// [P][2][N] partial rows -> dw, db: 32 columns per workgroup at a time, 32 threads down each column, added in a fixed tree
template <typename P>
__global__ __launch_bounds__(1024) void k_layer_norm_cols(const float *__restrict__ partial, uint32_t rows, uint32_t N, P *__restrict__ dw, P *__restrict__ db) {
    __shared__ float s[32][33];
    const uint32_t r0 = threadIdx.x >> 5;
    for (uint32_t c0 = blockIdx.x * 32; c0 < 2 * N; c0 += gridDim.x * 32) {
        const uint32_t c = c0 + (threadIdx.x & 31);
        float acc = 0.0f;
        if (c < 2 * N) {
            uint32_t r = r0;
            for (; r + 7 * 32 < rows; r += 8 * 32) {               // (eight loads in flight)
                float v[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) v[x] = partial[(uint64_t)(r + x * 32) * 2 * N + c];
#pragma unroll
                for (int x = 0; x < 8; ++x) acc += v[x];
            }
            for (; r < rows; r += 32) acc += partial[(uint64_t)r * 2 * N + c];
        }
        s[r0][threadIdx.x & 31] = acc;
        __syncthreads();
        // 32 columns x 32 partial sums: the wavefronts read them transposed, 32 lanes per column
        float v = s[threadIdx.x & 31][threadIdx.x >> 5];
        __syncthreads();                                           // (read before the next columns' are written)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor(v, o);
        const uint32_t col = c0 + (threadIdx.x >> 5);
        if ((threadIdx.x & 31) == 0 && col < 2 * N) {
            if (col < N) {
                if (dw) dw[col] = (P)v;
            } else if (db) {
                db[col - N] = (P)v;
            }
        }
    }
}

// Most workgroups along an axis of columns (wider rows go round again): a grid's axis has to stay below 2^32 threads, and a launch beyond that is not refused -- the count wraps
// and the columns behind keep what their memory held.
constexpr uint32_t kLnMostGrid = 32768;

// workgroups of the backward pass = partial rows: four per CU (65 537 x 204 fp32: 28.5 us, two per CU 37.7; 13 000 x 1 024 bf16: 21.9, six per CU 28.9), no more than there
// are rows to take.  Four rows a workgroup are counted up to 1 024 columns; fp32 rows of 513 to 1 024 take a whole workgroup each and so share one by fours.  Measured at these two
// widths: from 4 096 columns on the partial rows weigh as much as the data (3 250 x 4 096 bf16: backward 68 us for 80 MB).
static uint32_t ln_bwd_groups(uint64_t M, uint32_t N) {
    const uint64_t rpw = N <= 1024 ? 4 : 1;
    const uint64_t want = (M + rpw - 1) / rpw;
    const uint64_t most = (uint64_t)cu_count() * 4;
    return (uint32_t)(want < most ? (want ? want : 1) : most);
}

static bool ln_aligned(const void *p, int64_t pitch, size_t size) { return ((uintptr_t)p | (uint64_t)(pitch * (int64_t)size)) % 16 == 0; }

template <typename T, int VEC>
static void ln_forward(const LnArgs &a, hipStream_t st) {
    const uint64_t most = 1u << 22, waves = (a.M + 3) / 4;
    const uint32_t g4 = (uint32_t)(waves < most ? waves : most), g1 = (uint32_t)(a.M < most ? a.M : most);
    constexpr int E = VEC == 1 ? 8 : VEC;              // elements of a "step" per thread
    constexpr int S = E / VEC;                         // vectors per step
    // Rows of a wavefront at a time: four where half its lanes have a row's elements and there are rows for every wavefront of the chip, so that as many bytes are in flight
    // (200 000 x 64 fp32: 39 us one by one, 33 four at a time; 32 768 x 512: 22 either way).  16-bit rows are bound by their conversions instead (65 537 x 128: 18.0 one by one,
    // 19.0 four at a time).
    constexpr int MANY = VEC == 1 || sizeof(T) == 2 ? 1 : 4;
    if (MANY > 1 && a.N <= 32u * E && a.M >= (uint64_t)cu_count() * 64) k_layer_norm<T, VEC, 64, S, MANY><<<div_up(g4, MANY), 256, 0, st>>>(a);
    else if (a.N <= 64u * E) k_layer_norm<T, VEC, 64, S, 1><<<g4, 256, 0, st>>>(a);
    else if (a.N <= 128u * E) k_layer_norm<T, VEC, 64, 2 * S, 1><<<g4, 256, 0, st>>>(a);
    else if (a.N <= 256u * E) k_layer_norm<T, VEC, 256, S, 1><<<g1, 256, 0, st>>>(a);
    else if (a.N <= 512u * E) k_layer_norm<T, VEC, 256, 2 * S, 1><<<g1, 256, 0, st>>>(a);
    else if (a.N <= 1024u * E) k_layer_norm<T, VEC, 256, 4 * S, 1><<<g1, 256, 0, st>>>(a);
    else k_layer_norm_long<T, VEC><<<g1, 256, 0, st>>>(a);
}

template <typename T, int VEC>
static void ln_backward(const LnArgs &a, uint32_t groups, hipStream_t st) {
    constexpr int E = VEC == 1 ? 8 : VEC, S = E / VEC;
    const uint32_t lds = a.partial ? 2 * a.N * 4 : 0;
    // (as in the forward pass; 200 000 x 64: fp32 56 us one by one, 48 four at a time, bf16 73 and 65)
    constexpr int MANY = VEC == 1 ? 1 : 4;
    if (MANY > 1 && a.N <= 32u * E && a.M >= (uint64_t)cu_count() * 64) k_layer_norm_bwd<T, VEC, 64, S, MANY><<<groups, 256, lds, st>>>(a);
    else if (a.N <= 64u * E) k_layer_norm_bwd<T, VEC, 64, S, 1><<<groups, 256, lds, st>>>(a);
    else if (a.N <= 128u * E) k_layer_norm_bwd<T, VEC, 64, 2 * S, 1><<<groups, 256, lds, st>>>(a);
    else if (a.N <= 256u * E) k_layer_norm_bwd<T, VEC, 256, S, 1><<<groups, 256, 0, st>>>(a);
    else if (a.N <= 512u * E) k_layer_norm_bwd<T, VEC, 256, 2 * S, 1><<<groups, 256, 0, st>>>(a);
    else {
        const uint64_t most = 1u << 22;
        if (a.y && a.M) k_layer_norm_bwd_long<T, VEC><<<(uint32_t)(a.M < most ? a.M : most), 256, 0, st>>>(a);
        if (a.partial) k_layer_norm_cols_long<T, VEC><<<dim3(groups, std::min(div_up(a.N, 256 * VEC), kLnMostGrid)), 256, 0, st>>>(a);
    }
}

}  // namespace gfpp

using namespace gfpp;

#define LN_REQUIRE(cond, what)                                              \
    do {                                                                    \
        if (!(cond)) {                                                      \
            set_error("%s: invalid argument (%s)", what, #cond);            \
            return GFPP_EINVAL;                                             \
        }                                                                   \
    } while (0)

GFPP_API unsigned long long gfpp_layer_norm_backward_scratch_floats(uint64_t M, uint32_t N) { return 2ull * N * ln_bwd_groups(M, N); }

GFPP_API int gfpp_layer_norm_forward(const void *x, int64_t x_pitch, const void *weight, const void *bias, int param_dtype, uint64_t M, uint32_t N, float eps, int dtype,
                                     void *y, float *mean, float *rstd, gfpp_stream_t stream) {
    const char *what = "gfpp_layer_norm_forward";
    LN_REQUIRE(dtype == GFPP_F32 || dtype == GFPP_F16 || dtype == GFPP_BF16, what);
    LN_REQUIRE(param_dtype == GFPP_F32 || param_dtype == dtype, what);
    LN_REQUIRE(N > 0 && N <= (1u << 30), what);
    LN_REQUIRE((mean == nullptr) == (rstd == nullptr), what);
    LN_REQUIRE(eps >= 0.0f, what);
    if (M == 0) return 0;
    LN_REQUIRE(x && y, what);
    LN_REQUIRE(x_pitch >= 0, what);
    LnArgs a{x, nullptr, weight, bias, y, mean, rstd, nullptr, M, x_pitch, 0, N, eps, param_dtype == GFPP_F32};
    const size_t size = dtype == GFPP_F32 ? 4 : 2;
    const bool vec = (N * size) % 16 == 0 && ln_aligned(x, x_pitch, size) && ln_aligned(y, 0, size) && ln_aligned(weight, 0, size) && ln_aligned(bias, 0, size);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GFPP_F32) vec ? ln_forward<float, 4>(a, st) : ln_forward<float, 1>(a, st);
    else if (dtype == GFPP_F16) vec ? ln_forward<_Float16, 8>(a, st) : ln_forward<_Float16, 1>(a, st);
    else vec ? ln_forward<__bf16, 8>(a, st) : ln_forward<__bf16, 1>(a, st);
    return check_launch(what);
}

GFPP_API int gfpp_layer_norm_backward(const void *dy, int64_t dy_pitch, const void *x, int64_t x_pitch, const void *weight, int param_dtype, const float *mean,
                                      const float *rstd, uint64_t M, uint32_t N, int dtype, void *dx, void *dweight, void *dbias, float *scratch,
                                      gfpp_stream_t stream) {
    const char *what = "gfpp_layer_norm_backward";
    LN_REQUIRE(dtype == GFPP_F32 || dtype == GFPP_F16 || dtype == GFPP_BF16, what);
    LN_REQUIRE(param_dtype == GFPP_F32 || param_dtype == dtype, what);
    LN_REQUIRE(N > 0 && N <= (1u << 30), what);
    const bool cols = dweight || dbias;
    if (!dx && !cols) return 0;
    LN_REQUIRE(M == 0 || (dy && x && mean && rstd), what);
    LN_REQUIRE(!cols || scratch, what);
    LN_REQUIRE(x_pitch >= 0 && dy_pitch >= 0, what);
    const uint32_t groups = ln_bwd_groups(M, N);
    LnArgs a{x, dy, weight, nullptr, dx, const_cast<float *>(mean), const_cast<float *>(rstd), cols ? scratch : nullptr, M, x_pitch, dy_pitch, N, 0.0f,
             param_dtype == GFPP_F32};
    const size_t size = dtype == GFPP_F32 ? 4 : 2;
    const bool vec = (N * size) % 16 == 0 && ln_aligned(x, x_pitch, size) && ln_aligned(dy, dy_pitch, size) && ln_aligned(dx, 0, size) && ln_aligned(weight, 0, size);
    hipStream_t st = (hipStream_t)stream;
    // (M == 0: one workgroup without rows leaves zero sums)
    if (dtype == GFPP_F32) vec ? ln_backward<float, 4>(a, groups, st) : ln_backward<float, 1>(a, groups, st);
    else if (dtype == GFPP_F16) vec ? ln_backward<_Float16, 8>(a, groups, st) : ln_backward<_Float16, 1>(a, groups, st);
    else vec ? ln_backward<__bf16, 8>(a, groups, st) : ln_backward<__bf16, 1>(a, groups, st);
    int rc = check_launch(what);
    if (rc || !cols) return rc;
    const uint32_t blocks = std::min(div_up(2 * N, 32), kLnMostGrid);
    if (param_dtype == GFPP_F32) k_layer_norm_cols<float><<<blocks, 1024, 0, st>>>(scratch, groups, N, (float *)dweight, (float *)dbias);
    else if (dtype == GFPP_F16) k_layer_norm_cols<_Float16><<<blocks, 1024, 0, st>>>(scratch, groups, N, (_Float16 *)dweight, (_Float16 *)dbias);
    else k_layer_norm_cols<__bf16><<<blocks, 1024, 0, st>>>(scratch, groups, N, (__bf16 *)dweight, (__bf16 *)dbias);
    return check_launch(what);
}
