// window_attn.hip -- attention with a sliding window and visible first tokens: forward pass (gfx950).  The rule of visibility and the fragment layout are in
// window_attn_device.h, the backward pass in window_attn_bwd.hip, the single-token form in window_attn_step.hip.
//
//   s_ij = scale q_i . k_j over the visible keys,  p_ij = exp(s_ij - m_i) / l_i,  o_i = sum_j p_ij v_j,   m the running maximum, l the running sum (fp32)
//
// A workgroup takes 128 queries of one head, a wavefront 32 of them, and walks the tiles of keys that they can see (the sinks' tiles, then the band's): keys and
// values go through LDS, double-buffered, the tile after next in flight in registers, one barrier per tile.  S^T = K Q^T puts a query's scores into ONE lane pair: the
// row maximum and sum are register arithmetic, the probabilities are the operand of O^T = V^T P^T without leaving their registers, and the accumulators are rescaled
// by one factor per lane -- only when a maximum has grown by more than 2^8, since exp2(s - m) with a slightly old m is as exact.
// Probabilities are rounded to the operand type (16-bit modes) for the matrix instruction; l sums the unrounded ones in fp32.  That is a choice: against 64 bits the output is off by
// 2.4e-3 of its norm (bf16, window 1 024) where its own rounding alone is 1.7e-3.  The matrix pipe takes fp32 operands at an eighth of the rate, and as a rounded value and its
// remainder (done where it shows: window_attn_device.h, the two-part rule) half as many products again.
#include "window_attn_device.h"

namespace gfpp {

// Keys per tile.  64 let one half's products run under the other's arithmetic where registers allow it (128-wide 16-bit heads); up to 64 features 32 keys fit four wavefronts to a
// SIMD instead of three (13 000 x 8 heads x 64, window 1024: 78 -> 71 us), and a query that sees few keys has less of a tile to mask.
template <typename T, int DP, bool FEW>
constexpr int wa_bn() { return FEW || (sizeof(T) == 4 && DP == 128) || (sizeof(T) == 2 && DP <= 64) ? 32 : 64; }

// FEW: a query sees at most 64 keys (wa_few): small tiles, and in the 16-bit modes probabilities as a rounded value and its remainder (window_attn_device.h).
// HEADS 2: eight wavefronts, four for each of two query heads of a group, share the tiles of keys and values -- half the loads and LDS writes per query.
// WAVES 1: 32 queries a workgroup instead of 128, for few keys and a grid that would leave CUs empty (296 x 4 heads x 16, window 8, fp32: 8.5 us, with 128 queries 13.8).
// VEC: 16-byte accesses (wa_vectors); one element at a time otherwise (13 000 x 8 heads x 64, window 1 024: 69 and 180 us).
//
// No unit is full: what is left is waiting (a third of the wavefronts' time for data and barriers, near a third for their turn to issue).  Measured (bf16): 16 384 x 16 heads on 4 x 128,
// window 2 049: 295 us (266 GFLOP, 0.90 PFLOP/s; of the CUs' cycles the matrix pipe is busy in 45 %, the LDS in 28 %); 13 000 x 8 on 2 x 64, window 1 024, 4 sinks: 68 us (26 GFLOP,
// 0.39 PFLOP/s; 26 and 20 %: at 64 features every 64 products come with an exponential).
template <typename T, int DP, bool VEC, bool FEW, int HEADS, int WAVES>
__global__ __launch_bounds__(64 * WAVES * HEADS, WAVES == 1 ? 1 : (sizeof(T) == 2 ? (DP <= 64 && VEC ? (FEW ? 3 : 4) : (VEC || HEADS == 2 ? 2 : 1)) : 1)) void k_window_attn(WaArgs a) {
    constexpr int BN = wa_bn<T, DP, FEW>(), ROWS = 32 * WAVES, NS = DP / 16, NT = DP / 32, NSUB = BN / 32, PK = wa_pitch_row<T, DP>(), PV = wa_pitch_col<T, DP>();
    constexpr bool TWO = FEW && sizeof(T) == 2;
    typedef typename LpTraits<T>::vec vec;
    __shared__ __attribute__((aligned(16))) unsigned char s_k[2][BN * PK], s_v[2][BN * PV];
    const int q_tiles = (a.Tq + ROWS - 1) / ROWS;
    // items: sequence, key head, tile of queries, query head of the group -- those that read the same keys side by side
    uint32_t item = wa_item(blockIdx.x, gridDim.x);
    const int in_group = (int)(item % (a.G / HEADS)) * HEADS + (HEADS == 2 ? __builtin_amdgcn_readfirstlane((int)(threadIdx.x / (64 * WAVES))) : 0);
    item /= a.G / HEADS;
    const int i0 = (int)(item % q_tiles) * ROWS;
    item /= q_tiles;
    const int hk = (int)(item % a.Hk), hq = hk * a.G + in_group, b = (int)(item / a.Hk);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6) % WAVES), c = lane & 31, h = lane >> 5;
    const int n = a.lengths ? a.lengths[b] < a.Tk ? a.lengths[b] : a.Tk : a.Tk;
    const int i = i0 + wave * 32 + c, p = a.q_start + i;
    const bool have = i < a.Tq && p < n;
    vec q[NS];
    wa_global_rows<T, NS, VEC>(q, static_cast<const T *>(a.q.p) + b * a.q.sb + (int64_t)i * a.q.st + hq * a.q.sh, have, h, a.D);
    const int i1 = i0 + ROWS < a.Tq ? i0 + ROWS - 1 : a.Tq - 1;
    const WaRange range = wa_keys<BN>(a, a.q_start + i0, a.q_start + i1, n);
    const int tiles = range.head + range.hi - range.lo;
    const int last = have ? (p + a.right < n - 1 ? p + a.right : n - 1) : -1, first = p - a.left;          // this lane's query
    const int pw0 = a.q_start + i0 + wave * 32, pw1 = pw0 + 31;                                               // the wavefront's
    v16f acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    const T *kb = static_cast<const T *>(a.k.p) + b * a.k.sb + hk * a.k.sh, *vb = static_cast<const T *>(a.v.p) + b * a.v.sb + hk * a.v.sh;
    // two tiles in flight: the one that the next step stores and the one after it (one alone arrives later than the step that it was requested in takes)
    WaStage<T, DP, BN, VEC, 64 * WAVES * HEADS> rk[2], rv[2];
    auto tile_row = [&](int k) { return (k < range.head ? k : range.lo + k - range.head) * BN; };
    // Loads and stores of tiles are unconditional -- past the last tile a load's range is empty, nothing is read --: a load behind a branch may or may not be in flight, and
    // every wait would then be for all of them.
    auto load = [&](int which, int k) {
        const int r0 = k < tiles ? tile_row(k) : (n > 0 ? n : 0);
        rk[which].load(kb, a.k.st, r0, n, a.D);
        rv[which].load(vb, a.v.st, r0, n, a.D);
    };
    load(0, 0);
    load(1, 1);
    rk[0].store(s_k[0], PK);
    rv[0].store(s_v[0], PV);
    load(0, 2);
    wa_arrived(q);
    __syncthreads();
    const int row_at = c * PK + 8 * h * (int)sizeof(T), col_at = wa_col_offset<T>(lane, PV);
    auto step = [&](int k, auto which) {
        constexpr int buf = decltype(which)::value, other = buf ^ 1;     // of tile k (LDS) and of tile k + 1 (LDS, registers)
        const int j0 = tile_row(k), j1 = j0 + BN - 1;
        rk[other].store(s_k[other], PK);                         // (last read before the previous barrier)
        rv[other].store(s_v[other], PV);
        load(other, k + 3);
        const bool seen = pw0 < n && j0 <= pw1 + a.right && (j1 >= pw0 - a.left || j0 < a.sinks);
        if (seen) {
            v16f s[NSUB];
#pragma unroll
            for (int u = 0; u < NSUB; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[u][r] = 0.0f;
            {
                WaStream<T, NSUB * NS> keys;
                const auto read = [&](int x) { return wa_row<T>(s_k[buf] + row_at + 32 * (x / NS) * PK, x % NS); };
                keys.prime(read);
                keys.run(read, [&](int x, const vec &f) { s[x / NS] = LpTraits<T>::mfma(f, q[x % NS], s[x / NS]); });
            }
            WaStream<T, NSUB * 2 * NT> values;                 // (32 keys u, their step x, the feature tile t: u, x, t)
            const auto read_v = [&](int x) { return wa_col<T, PV>(s_v[buf] + col_at, 32 * (x / (2 * NT)) + 16 * (x / NT % 2), x % NT); };
            values.prime(read_v);
            const bool full = pw1 < n && j1 < n && j1 <= pw0 + a.right && (j0 >= pw1 - a.left || j1 < a.sinks);
            if (!full) {
#pragma unroll
                for (int u = 0; u < NSUB; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int j = j0 + 32 * u + 8 * (r >> 2) + 4 * h + (r & 3);
                        s[u][r] = j <= last && (j >= first || j < a.sinks) ? s[u][r] : -INFINITY;
                    }
            }
            float top = s[0][0];
#pragma unroll
            for (int u = 0; u < NSUB; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
            top = half_wave_max(top);
            // (both -inf: NaN, which is not > 8; the first visible score: inf > 8)
            if (__any((top - m) * a.c > 8.0f)) {
                const float grown = fmaxf(m, top), f = m == -INFINITY ? 0.0f : exp2f((m - grown) * a.c);
                m = grown;
                l *= f;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[t][r] *= f;
            }
            const float top0 = m == -INFINITY ? 0.0f : m, base = top0 * a.c;
#pragma unroll
            for (int u = 0; u < NSUB; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[u][r] = wa_prob<TWO || sizeof(T) == 4>(s[u][r], top0, base, a.c);
                    l += s[u][r];
                }
            vec pr;
            values.run(read_v, [&](int x, const vec &f) {
                const int u = x / (2 * NT), step = x / NT % 2, t = x % NT;
                if (t == 0) pr = wa_pack<T>(s[u], step);
                acc[t] = LpTraits<T>::mfma(f, pr, acc[t]);
            });
            if constexpr (TWO) {                               // what the rounding left, over the same values once more
#pragma unroll
                for (int u = 0; u < NSUB; ++u)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const vec p = wa_pack<T>(s[u], x);
#pragma unroll
                        for (int e = 0; e < 8; ++e) s[u][8 * x + e] -= (float)p[e];
                    }
                values.prime(read_v);
                values.run(read_v, [&](int x, const vec &f) {
                    const int u = x / (2 * NT), step = x / NT % 2, t = x % NT;
                    if (t == 0) pr = wa_pack<T>(s[u], step);
                    acc[t] = LpTraits<T>::mfma(f, pr, acc[t]);
                });
            }
        }
        __syncthreads();
    };
    for (int k = 0; k < tiles; ++k) {
        step(k, WaInt<0>{});
        if (++k >= tiles) break;                               // (no way from an even step to the next even one: what is in flight is the same at every wait)
        step(k, WaInt<1>{});
    }
    l = half_wave_sum(l);
    if (i >= a.Tq) return;
    T *o = static_cast<T *>(a.o.p) + b * a.o.sb + (int64_t)i * a.o.st + hq * a.o.sh;
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    wa_store_rows<T, NT, VEC>(acc, inv, o, h, a.D);
    if constexpr (TWO)
        if (a.low) wa_store_rows<T, NT, VEC, true>(acc, inv, static_cast<T *>(a.low) + (o - static_cast<T *>(a.o.p)), h, a.D);
    // log2 of the row's sum, +inf for a row without visible keys: every probability of the backward pass is then exp2(-inf) = 0
    if (a.lse && h == 0) a.lse[((int64_t)b * a.Hq + hq) * a.Tq + i] = l > 0.0f ? m * a.c + log2f(l) : INFINITY;
}

// whether a tensor's rows can be read as 16-byte vectors whose place in a tile of 64 rows is a 32-bit offset (WaStage)
bool wa_vectors(const WaTensor &t, int D, size_t size) {
    return t.st >= D && t.st <= (int64_t)(((1u << 31) - 1024) / (64 * size)) && ((uintptr_t)t.p | (uint64_t)(t.sb * (int64_t)size) | (uint64_t)(t.st * (int64_t)size) | (uint64_t)(t.sh * (int64_t)size) | (uint64_t)(D * size)) % 16 == 0;
}

// the arguments that both passes share; 0 or an error code
int wa_arguments(const char *what, WaArgs &a, const int64_t *strides, int n_tensors, uint32_t B, uint32_t Tq, uint32_t Tk, uint32_t Hq, uint32_t Hk, uint32_t D, int32_t left,
                 int32_t right, int32_t sinks, int32_t q_start, const int32_t *lengths, float scale, int dtype) {
    const uint32_t most = 1u << 29;
#define WA_REQUIRE(cond)                                               \
    do {                                                               \
        if (!(cond)) {                                                 \
            set_error("%s: invalid argument (%s)", what, #cond);       \
            return GFPP_EINVAL;                                        \
        }                                                              \
    } while (0)
    WA_REQUIRE(dtype == GFPP_F32 || dtype == GFPP_F16 || dtype == GFPP_BF16);
    WA_REQUIRE(B <= most && Tq <= most && Tk <= most && Hq <= most && Hk <= most && strides);
    WA_REQUIRE(Hk >= 1 && Hq >= 1 && Hq % Hk == 0);
    WA_REQUIRE(left >= 0 && right >= 0 && sinks >= 0 && q_start >= 0 && (uint32_t)q_start <= most);
    WA_REQUIRE(scale > 0.0f && scale < INFINITY);
    if (D < 1 || D > 128) {
        set_error("%s: head width %u (1 .. 128 are supported)", what, D);
        return GFPP_EUNSUPPORTED;
    }
    WaTensor *t[8] = {&a.q, &a.k, &a.v, &a.o, &a.dout, &a.dq, &a.dk, &a.dv};
    for (int k = 0; k < n_tensors; ++k) {
        t[k]->sb = strides[3 * k];
        t[k]->st = strides[3 * k + 1];
        t[k]->sh = strides[3 * k + 2];
    }
    a.lengths = lengths;
    a.B = (int)B;
    a.Tq = (int)Tq;
    a.Tk = (int)Tk;
    a.Hq = (int)Hq;
    a.Hk = (int)Hk;
    a.G = (int)(Hq / Hk);
    a.D = (int)D;
    a.left = left < (int)most ? left : (int)most;
    a.right = right < (int)most ? right : (int)most;
    a.sinks = sinks < (int)Tk ? sinks : (int)Tk;
    a.q_start = q_start;
    a.scale = scale;
    a.c = scale * 1.4426950408889634f;
    return 0;
}

template <typename T, int DP, bool FEW, int HEADS, int WAVES>
static void wa_forward_launch(const WaArgs &a, bool vec, hipStream_t st) {
    const uint32_t grid = div_up((uint32_t)a.Tq, 32 * WAVES) * (uint32_t)(a.Hq / HEADS) * (uint32_t)a.B;
    if (vec) k_window_attn<T, DP, true, FEW, HEADS, WAVES><<<grid, 64 * WAVES * HEADS, 0, st>>>(a);
    else if constexpr (HEADS == 1) k_window_attn<T, DP, false, FEW, HEADS, WAVES><<<grid, 64 * WAVES, 0, st>>>(a);
}
template <typename T, int DP>
static void wa_forward_width(const WaArgs &a, bool vec, bool few, uint32_t grid, hipStream_t st) {
    if constexpr (DP * sizeof(T) <= 128)                       // (wider rows: a wavefront alone has no registers for two tiles in flight)
        if (few && grid < 2u * (uint32_t)cu_count()) return wa_forward_launch<T, DP, true, 1, 1>(a, vec, st);
    if constexpr (DP == 128 && sizeof(T) == 2)
        if (!few && vec && wa_pair_heads(a, grid)) return wa_forward_launch<T, DP, false, 2, 4>(a, vec, st);
    few ? wa_forward_launch<T, DP, true, 1, 4>(a, vec, st) : wa_forward_launch<T, DP, false, 1, 4>(a, vec, st);
}
template <typename T>
static void wa_forward(const WaArgs &a, bool vec, bool few, uint32_t grid, hipStream_t st) {
    if (a.D <= 32) wa_forward_width<T, 32>(a, vec, few, grid, st);
    else if (a.D <= 64) wa_forward_width<T, 64>(a, vec, few, grid, st);
    else wa_forward_width<T, 128>(a, vec, few, grid, st);
}

}  // namespace gfpp

using namespace gfpp;

GFPP_API int gfpp_window_attn_two_part(uint32_t Tk, int32_t left, int32_t right, int32_t sinks, int dtype) { return wa_two_part(Tk, left, right, sinks, dtype); }

GFPP_API int gfpp_window_attn_forward(const void *q, const void *k, const void *v, void *out, void *out_low, float *lse, const int64_t *strides, uint32_t B, uint32_t Tq, uint32_t Tk,
                                      uint32_t Hq, uint32_t Hk, uint32_t D, int32_t left, int32_t right, int32_t sinks, int32_t q_start, const int32_t *lengths, float scale,
                                      int dtype, gfpp_stream_t stream) {
    const char *what = "gfpp_window_attn_forward";
    WaArgs a{};
    if (int rc = wa_arguments(what, a, strides, 4, B, Tq, Tk, Hq, Hk, D, left, right, sinks, q_start, lengths, scale, dtype)) return rc;
    if ((uint64_t)B * Tq == 0) return 0;
    WA_REQUIRE(q && out && (Tk == 0 || (k && v)));
    a.q.p = const_cast<void *>(q);
    a.k.p = const_cast<void *>(k);
    a.v.p = const_cast<void *>(v);
    a.o.p = out;
    a.lse = lse;
    const bool few = wa_few(Tk, left, right, sinks);
    a.low = wa_two_part(Tk, left, right, sinks, dtype) ? out_low : nullptr;
    WA_REQUIRE(grid_fits(kWaThreads, div_up(Tq, kWaRows), Hq, B));
    const uint32_t grid = div_up(Tq, kWaRows) * Hq * B;
    const size_t size = dtype == GFPP_F32 ? 4 : 2;
    const bool vec = wa_vectors(a.q, a.D, size) && wa_vectors(a.k, a.D, size) && wa_vectors(a.v, a.D, size) && wa_vectors(a.o, a.D, size) && (uintptr_t)a.low % 16 == 0;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GFPP_F32) wa_forward<float>(a, vec, few, grid, st);
    else if (dtype == GFPP_F16) wa_forward<_Float16>(a, vec, few, grid, st);
    else wa_forward<__bf16>(a, vec, few, grid, st);
    return check_launch(what);
}
