// window_attn_device.h -- what the windowed-attention kernels share (window_attn.hip, window_attn_bwd.hip; gfx950).
//
// A query at position p = q_start + i sees key j iff  j < n  and  p < n  and  j <= p + right  and  (j >= p - left  or  j < sinks),  n = the sequence's length.
//
// Fragments of v_mfma_f32_32x32x16_*: lane (c = lane & 31, h = lane >> 5) supplies row / column c at contraction indices 8 h .. 8 h + 7 of a step, and holds of a
// 32 x 32 product column c at rows  8 (r >> 2) + 4 h + (r & 3), r = 0 .. 15.  The contraction index may be permuted as long as both operands agree, so the 16
// values of a product that a lane holds ARE the operand of the next product's two steps (values 8 s .. 8 s + 7 = rows 16 s + {4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3}):
// probabilities never leave their registers, the other operand is read with the rows in that order.  fp32: a "step" is eight v_mfma_f32_32x32x2_f32, element e of
// both fragments each (lp_mfma_device.h).
#pragma once

#include "gfpp_common.h"
#include "lp_mfma_device.h"

namespace gfpp {

constexpr int kWaThreads = 256, kWaRows = 128;      // four wavefronts of 32 queries (forward, dq); dk and dv: 64 keys, two wavefronts for every 32

template <int N>
struct WaInt {
    static constexpr int value = N;
};
struct WaTensor {
    void *p;
    int64_t sb, st, sh;            // strides of sequence, token and head in elements
};
struct WaArgs {
    WaTensor q, k, v, o, dout, dq, dk, dv;
    void *low;                     // out's rounding errors (o's strides), or NULL
    float *lse, *delta;            // [B][Hq][Tq]
    float *partial;                // sink tiles' dk and dv: [sink tiles][splits][B][Hk][2][keys][D]
    const int32_t *lengths;        // [B] or NULL
    int32_t B, Tq, Tk, Hq, Hk, D, G;
    int32_t left, right, sinks;    // left, right < 2^30
    int32_t q_start;
    float scale, c;                // c = scale log2(e)
    uint32_t sink_tiles, splits;
};

// two query heads per workgroup: an even group, and enough workgroups left to fill the chip (16 384 x 16 heads on 4 x 128, window 2 049, bf16, forward, in turn on one card: 313 to
// 329 us, one head each 342; the backward kernels do not gain)
inline bool wa_pair_heads(const WaArgs &a, uint64_t grid) { return a.G % 2 == 0 && grid / 2 >= (uint64_t)cu_count(); }

// Workgroups are dealt out to the 8 XCDs in turn, each with an L2 of its own: the work items of one XCD are made neighbours (which read the same keys or
// queries) by giving it a contiguous stretch of them (dk and dv at 16 384 x 16 heads x 128: 824 us, in the grid's order 856).  A permutation of 0 .. total - 1 for any total.
__device__ __forceinline__ uint32_t wa_item(uint32_t block, uint32_t total) {
    const uint32_t xcd = block % 8, each = total / 8, more = total % 8;
    return xcd * each + (xcd < more ? xcd : more) + block / 8;
}

template <typename T>
struct WaTraits;
template <>
struct WaTraits<_Float16> {
    static constexpr int V = 8;                                        // elements of 16 bytes
    typedef __fp16 raw4 __attribute__((__vector_size__(8)));
    typedef _Float16 half4 __attribute__((ext_vector_type(4)));
};
template <>
struct WaTraits<__bf16> {
    static constexpr int V = 8;
    typedef __bf16 half4 __attribute__((ext_vector_type(4)));
};
template <>
struct WaTraits<float> {
    static constexpr int V = 4;
};

// Bytes of an LDS row of DP elements, padded for what reads it (64 banks of 4 bytes): row fragments want an odd number of 16-byte units (16 rows at one column
// then cover all banks), transposing reads 64 or 192 modulo 256 bytes (the 4 rows x 64 bytes of one read lie apart); rows that are read both ways take the odd
// number next to that.  32-bit columns are read a word per lane: any pitch.
template <typename T, int DP>
constexpr int wa_pitch_row() { return DP * (int)sizeof(T) + 16; }
template <typename T, int DP>
constexpr int wa_pitch_col() { return DP * (int)sizeof(T) % 128 == 0 ? DP * (int)sizeof(T) + 64 : DP * (int)sizeof(T); }
template <typename T, int DP>
constexpr int wa_pitch_both() { return DP * (int)sizeof(T) + (sizeof(T) == 2 ? (DP == 32 ? 16 : 80) : 16); }

// Rows r0 .. r0 + ROWS - 1 of a [tokens][D] head into registers, the thread's share: 16 bytes per vector.  Rows from `end` on and columns from D on are zeros and
// are not read: what lies behind a sequence may hold anything.  VEC: buffer loads, whose range check gives those zeros without a branch or a clear per vector -- the
// tile's base and its end are scalar, a lane keeps ONE 32-bit offset for all its vectors (the host has seen to it that 64 rows span less than 2^31 bytes and
// that a row's pitch is at least its width).
template <typename T, int DP, int ROWS, bool VEC, int THREADS = kWaThreads>
struct WaStage {
    static constexpr int V = WaTraits<T>::V, PER_ROW = DP / V, ALL = ROWS * PER_ROW, N = (ALL + THREADS - 1) / THREADS, STEP = THREADS / PER_ROW;      // rows between a lane's vectors
    static_assert(ALL % THREADS == 0 || ALL < THREADS, "whole vectors per thread, or one for some of them");
    typedef T vec __attribute__((ext_vector_type(V)));
    vec r[N];

    // r0 >= 0 and the same in all lanes
    __device__ __forceinline__ void load(const T *base, int64_t stride, int r0, int end, int D) {
        const T *tile = base + (int64_t)r0 * stride;
        const int row = (int)threadIdx.x / PER_ROW, col = (int)threadIdx.x % PER_ROW * V;
        if constexpr (VEC) {
            const int rows = end - r0 < ROWS ? (end - r0 > 0 ? end - r0 : 0) : ROWS, pitch = (int)stride * (int)sizeof(T);
            // (a scalar by its making: the compiler clamps in the vector unit and would then load lane group by lane group)
            const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(tile), 0, __builtin_amdgcn_readfirstlane(rows * pitch), 0x00020000);
            const uint32_t at = col < D && (ALL >= THREADS || (int)threadIdx.x < ALL) ? (uint32_t)(row * pitch + col * (int)sizeof(T)) : 0x7ffffff0u;
#pragma unroll
            for (int n = 0; n < N; ++n)                        // (the whole offset in the lane: the range check subtracts a scalar offset from the size, without a sign)
                r[n] = __builtin_bit_cast(vec, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)(at + (uint32_t)(n * STEP * pitch)), 0, 0));
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                vec t = (vec)(T)0.0f;
                if (row + n * STEP < end - r0 && (ALL >= THREADS || (int)threadIdx.x < ALL)) {
                    const T *p = tile + (int64_t)(row + n * STEP) * stride + col;
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (col + e < D) t[e] = p[e];
                }
                r[n] = t;
            }
        }
    }
    __device__ __forceinline__ void store(unsigned char *lds, int pitch) const {
        unsigned char *at = lds + (int)threadIdx.x / PER_ROW * pitch + (int)threadIdx.x % PER_ROW * 16;
        if (ALL >= THREADS || (int)threadIdx.x < ALL)
#pragma unroll
            for (int n = 0; n < N; ++n) *reinterpret_cast<vec *>(at + n * STEP * pitch) = r[n];
    }
};

// row fragment: elements 16 s + 8 h .. + 7 of row c of a tile (`at` = the lane's row + 8 h elements)
template <typename T>
__device__ __forceinline__ typename LpTraits<T>::vec wa_row(const unsigned char *at, int s) {
    return *reinterpret_cast<const typename LpTraits<T>::vec *>(at + s * 16 * (int)sizeof(T));
}
template <>
__device__ __forceinline__ LpTraits<float>::vec wa_row<float>(const unsigned char *at, int s) {
    typedef float f4 __attribute__((ext_vector_type(4)));
    const f4 a = *reinterpret_cast<const f4 *>(at + s * 64), b = *reinterpret_cast<const f4 *>(at + s * 64 + 16);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// column fragment of the 16 rows from row0 (tile bytes `tile`): column 32 t + c at rows {4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3}.  16 bits: two transposing reads
// (ds_read_b64_tr_b16: a quarter wavefront reads 4 rows x 16 columns, lane p the four elements at its own address -- row p >> 2, columns 4 (p & 3) .. -- and lane l
// is given column l); 32 bits: eight reads.
template <typename T>
__device__ __forceinline__ int wa_col_offset(int lane, int pitch) {
    const int c = lane & 31, h = lane >> 5;
    if constexpr (sizeof(T) == 4) return 4 * h * pitch + c * 4;
    const int p = lane & 15, gi = (lane >> 4) & 1;
    return (4 * h + (p >> 2)) * pitch + (16 * gi + 4 * (p & 3)) * 2;
}
template <typename T, int PITCH>
__device__ __forceinline__ typename LpTraits<T>::vec wa_col(const unsigned char *tile_at, int row0, int t) {
    const unsigned char *at = tile_at + row0 * PITCH + t * 32 * (int)sizeof(T);
    if constexpr (sizeof(T) == 4) {
        typename LpTraits<T>::vec f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = *reinterpret_cast<const float *>(at + ((e & 3) + 8 * (e >> 2)) * PITCH);
        return f;
    } else {
        typedef __attribute__((__vector_size__(4 * sizeof(__fp16)))) __fp16 fp16x4;
        typedef __attribute__((address_space(3))) fp16x4 *lds_ptr;
        typedef T half4 __attribute__((ext_vector_type(4)));
        const fp16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_ptr)(at));
        const fp16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_ptr)(at + 8 * PITCH));
        return __builtin_shufflevector(__builtin_bit_cast(half4, lo), __builtin_bit_cast(half4, hi), 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// the lane's row of a head straight from memory as NS row fragments; zeros where `have` is false and behind column D
template <typename T, int NS, bool VEC>
__device__ __forceinline__ void wa_global_rows(typename LpTraits<T>::vec (&f)[NS], const T *row, bool have, int h, int D) {
    typedef T vec16 __attribute__((ext_vector_type(WaTraits<T>::V)));
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int col = 16 * s + 8 * h;
#pragma unroll
        for (int e0 = 0; e0 < 8; e0 += WaTraits<T>::V) {
            vec16 t = (vec16)(T)0.0f;
            if (have && col + e0 < D) {
                if constexpr (VEC) {
                    t = *reinterpret_cast<const vec16 *>(row + col + e0);
                } else {
#pragma unroll
                    for (int e = 0; e < WaTraits<T>::V; ++e)
                        if (col + e0 + e < D) t[e] = row[col + e0 + e];
                }
            }
#pragma unroll
            for (int e = 0; e < WaTraits<T>::V; ++e) f[s][e0 + e] = t[e];
        }
    }
}

// Has the fragments in their registers here.  Loads that are still in flight where a loop begins are otherwise waited for at their first use INSIDE it, in every
// iteration, and with them the tile that the iteration has just requested.
template <typename V, int N>
__device__ __forceinline__ void wa_arrived(V (&f)[N]) {
#pragma unroll
    for (int x = 0; x < N; ++x) {
        if constexpr (sizeof(V) == 16) {
            asm volatile("" : "+v"(f[x]));
        } else {
            typedef float f4 __attribute__((ext_vector_type(4)));
            f4 a = __builtin_shufflevector(f[x], f[x], 0, 1, 2, 3), b = __builtin_shufflevector(f[x], f[x], 4, 5, 6, 7);
            asm volatile("" : "+v"(a), "+v"(b));
            f[x] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
}

// N matrix instructions whose LDS operands are read a few instructions before their use: `read(x)` is the fragment of instruction x, `use(x, f)` the instruction.
// prime() is called where the reads may start, in front of the arithmetic that the first instruction waits for.  (dk and dv of 64-wide heads 168 -> 154 us; elsewhere within
// 2 % of the compiler's own order, pinned or not: with two wavefronts on a SIMD the products of one already run under the reads of the other.)
template <typename T, int N>
struct WaStream {
    typedef typename LpTraits<T>::vec vec;
    static constexpr int AHEAD = (sizeof(T) == 4 ? 2 : 4) < N ? (sizeof(T) == 4 ? 2 : 4) : N;
    vec ring[AHEAD];
    template <typename Read>
    __device__ __forceinline__ void prime(Read read) {
#pragma unroll
        for (int x = 0; x < AHEAD; ++x) ring[x] = read(x);
        __builtin_amdgcn_sched_barrier(0);
    }
    template <typename Read, typename Use>
    __device__ __forceinline__ void run(Read read, Use use) {
#pragma unroll
        for (int x = 0; x < N; ++x) {
            use(x, ring[x % AHEAD]);
            if (x + AHEAD < N) ring[x % AHEAD] = read(x + AHEAD);
        }
    }
};

// values 8 s .. 8 s + 7 of a product, rounded to the operand type (pairs: one conversion instruction each)
template <typename T>
__device__ __forceinline__ typename LpTraits<T>::vec wa_pack(const v16f &x, int s) {
    if constexpr (sizeof(T) == 4) {
        typename LpTraits<T>::vec f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = x[8 * s + e];
        return f;
    } else {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typename LpTraits<T>::vec f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const typename LpTraits<T>::pair p = __builtin_convertvector(((f32x2){x[8 * s + e], x[8 * s + e + 1]}), typename LpTraits<T>::pair);
            f[e] = p[0];
            f[e + 1] = p[1];
        }
        return f;
    }
}

// exp2((s - m) c), base = m c.  16-bit modes: one fused multiply-add; its rounding of base is far below theirs.  EXACT (fp32, two-part probabilities): the
// difference first, so that the largest score's probability is exactly 1 and a query with one visible key copies its value
template <bool EXACT>
__device__ __forceinline__ float wa_prob(float s, float m, float base, float c) {
    if constexpr (EXACT) return __builtin_amdgcn_exp2f((s - m) * c);
    return __builtin_amdgcn_exp2f(fmaf(s, c, -base));
}

__device__ __forceinline__ float half_wave_max(float t) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(t), __float_as_uint(t), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// x f rounded to 32 bits and then to T in every form of the kernels: left alone, the compiler makes some scalar f16 stores a mixed-precision multiply that rounds once
template <typename T>
__device__ __forceinline__ T wa_scaled(float x, float f) {
    float y = x * f;
    asm("" : "+v"(y));
    return (T)y;
}

// what rounding x f to T leaves of it
template <typename T>
__device__ __forceinline__ T wa_remainder(float x, float f) {
    float y = x * f;
    asm("" : "+v"(y));
    return (T)(y - (float)(T)y);
}

// a product tile [32 T rows = features][32 columns = tokens] to the lane's token row: 4 consecutive features per store
template <typename T, int NT, bool VEC, bool LOW = false>
__device__ __forceinline__ void wa_store_rows(const v16f (&acc)[NT], float f, T *row, int h, int D) {
    typedef T vec4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int col = 32 * t + 2 * r + 4 * h;
            if (col >= D) continue;
            if (VEC || col + 3 < D) {
                vec4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = LOW ? wa_remainder<T>(acc[t][r + e], f) : wa_scaled<T>(acc[t][r + e], f);
                if constexpr (VEC) {
                    *reinterpret_cast<vec4 *>(row + col) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) row[col + e] = v[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (col + e < D) row[col + e] = LOW ? wa_remainder<T>(acc[t][r + e], f) : wa_scaled<T>(acc[t][r + e], f);
            }
        }
}

// The two-part rule.  Rounding a probability costs half a step of its weight; over many keys these errors average out below the output's own rounding, over few they
// do not, and delta, the backward pass' row sum, carries both into every score gradient of the row.  Where a query sees at most 64 keys the forward pass therefore
// takes its probabilities as a rounded value and a rounded remainder (a second product: such calls are bound by latency and memory), and a training pass keeps
// the output's remainder for delta.  Goes by the arguments alone, so that a pass with gradients and one without give the same bits.
inline bool wa_few(int64_t Tk, int64_t left, int64_t right, int64_t sinks) {
    const int64_t window = left + right + 1 + sinks;
    return (window < Tk ? window : Tk) <= 64;
}
inline bool wa_two_part(int64_t Tk, int64_t left, int64_t right, int64_t sinks, int dtype) { return dtype != GFPP_F32 && wa_few(Tk, left, right, sinks); }

// tiles of BN keys that queries at positions p0 .. p1 can see: [0, head) for the sinks in front of the band, [lo, hi) for the band (merged where they touch)
struct WaRange {
    int head, lo, hi;
};
template <int BN>
__device__ __forceinline__ WaRange wa_keys(const WaArgs &a, int p0, int p1, int n) {
    WaRange r{0, 0, 0};
    if (p1 >= n) p1 = n - 1;
    if (p0 > p1) return r;
    const int last = p1 + a.right < n - 1 ? p1 + a.right : n - 1, first = p0 - a.left > 0 ? p0 - a.left : 0;
    r.lo = first / BN;
    r.hi = last / BN + 1;
    const int s = a.sinks < n ? a.sinks : n;
    r.head = (s + BN - 1) / BN;
    if (r.head >= r.lo) {
        r.lo = 0;
        r.head = 0;
    }
    return r;
}

}  // namespace gfpp
