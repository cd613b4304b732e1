// window_attn_step.hip -- one new token per stream against a rolling cache: the single-token form of the windowed attention (gfx950).
//
// The cache of a stream holds its first `sinks` tokens and its last W = slots - sinks ones; the token at position n lives in slot  n < sinks ? n : sinks +
// (n - sinks) mod W.  A step writes the new key and value into their slot and attends over the min(n + 1, slots) slots that are filled: exactly the keys that
// window_attn.hip's rule shows position n with left = W - 1, right = 0.  Softmax does not ask for an order, so the ring is read as it lies.
// A negative position leaves its stream as it is.
//
// Bound by memory: the filled slots are read once for all query heads of a group.  The group's heads are the 32 columns of the matrix products (window_attn_device.h's
// layout): keys come straight from memory as row fragments, values pass through a wavefront's own 32 rows of LDS for the transposing read.  A wavefront takes every
// fourth tile of 32 slots of its workgroup's stretch, the next tile in flight in registers; the four partial softmaxes meet in LDS.  Few streams: the
// slots of a stream are split over several workgroups, whose partial results a second launch joins.
// Probabilities enter the products as a rounded value and its rounded remainder, so that the output carries its own rounding alone.
// Measured (bf16): 64 streams x 32 heads on 8 x 128, 4 100 slots (1.08 GB): 180 us (6.0 TB/s; a copy of 2 GiB moves 5.2) and 7 for the join; one stream x 8 on 2 x 64, 260 slots:
// 6.3 us, a launch's latency and four dependent trips to memory.  One element at a time (unaligned rows) takes 1 000 and 23 us.
// The row of the new token is taken from the arguments by whoever reads that slot, and written by one wavefront: no order between workgroups is needed.
#include "window_attn_device.h"

namespace gfpp {

constexpr int kWsJoinThreads = 128;                    // a thread per feature

struct WsArgs {
    const void *q, *k, *v;
    void *ck, *cv, *out;
    const void *pos;
    float *part;                   // [B][Hq][splits][D + 2]: accumulators, maximum, sum
    int64_t qb, qh, kb, kh, vb, vh, ckb, cks, ckh, cvb, cvs, cvh, ob, oh;
    int32_t B, Hq, Hk, D, G, slots, sinks, chunks, per_split;
    uint32_t splits;
    int pos64;
    float c;
};

template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(kWaThreads, sizeof(T) == 2 ? 2 : 1) void k_window_attn_step(WsArgs a) {
    constexpr int NS = DP / 16, NT = DP / 32, PV = wa_pitch_col<T, DP>(), V = WaTraits<T>::V, PER_ROW = DP / V, NV = 32 * PER_ROW / 64;
    typedef typename LpTraits<T>::vec vec;
    typedef T vec16 __attribute__((ext_vector_type(V)));
    // the wavefronts' value tiles; after the loop their results: [4][32 heads][DP] accumulators, [4][32] maxima and sums
    constexpr int TILES = 4 * 32 * PV, RESULTS = 4 * 32 * (DP + 4) * 4;
    __shared__ __attribute__((aligned(16))) unsigned char lds[TILES > RESULTS ? TILES : RESULTS];
    __shared__ float s_m[4][32], s_l[4][32];
    // Consecutive workgroups go to the 8 XCDs in turn.  Heads taken in order would give an XCD the same few heads of every stream, whose rows, a whole token apart, lie on
    // the same few channels of its L2; turned by the stretch and the stream, every XCD sees all of them (64 streams x 8 heads x 128, 4 100 slots in 4 stretches: 227 -> 206 us).
    const uint32_t split = blockIdx.x % a.splits;
    uint32_t item = blockIdx.x / a.splits;
    const int chunk = (int)(item % a.chunks);
    item /= a.chunks;
    const int b = (int)(item / a.Hk), hk = (int)((item % a.Hk + split + b) % a.Hk);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
    const int64_t n = a.pos64 ? static_cast<const int64_t *>(a.pos)[b] : (int64_t)static_cast<const int32_t *>(a.pos)[b];
    const int window = a.slots - a.sinks;
    const int at = n < 0 ? -1 : (int)(n < a.sinks ? n : a.sinks + (n - a.sinks) % window);
    const int filled = n < 0 ? 0 : (int)(n < a.slots - 1 ? n + 1 : a.slots);
    const int g0 = chunk * 32, heads = a.G - g0 < 32 ? a.G - g0 : 32, hq0 = hk * a.G + g0;
    const T *kb = static_cast<const T *>(a.ck) + b * a.ckb + hk * a.ckh, *vb = static_cast<const T *>(a.cv) + b * a.cvb + hk * a.cvh;
    const T *kn = static_cast<const T *>(a.k) + b * a.kb + hk * a.kh, *vn = static_cast<const T *>(a.v) + b * a.vb + hk * a.vh;
    const int s0 = (int)split * a.per_split, s1 = s0 + a.per_split < filled ? s0 + a.per_split : filled;
    if (at >= s0 && at < s0 + a.per_split && chunk == 0 && wave == 0) {
        T *dk = static_cast<T *>(a.ck) + b * a.ckb + (int64_t)at * a.cks + hk * a.ckh, *dv = static_cast<T *>(a.cv) + b * a.cvb + (int64_t)at * a.cvs + hk * a.cvh;
        for (int d = lane; d < a.D; d += 64) {
            dk[d] = kn[d];
            dv[d] = vn[d];
        }
    }
    vec q[NS];
    wa_global_rows<T, NS, VEC>(q, static_cast<const T *>(a.q) + b * a.qb + (hq0 + c) * a.qh, c < heads && n >= 0, h, a.D);
    v16f acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    vec kf[NS];
    vec16 vr[NV];
    auto load = [&](int row0) {
        const int r = row0 + c;
        wa_global_rows<T, NS, VEC>(kf, r == at ? kn : kb + (int64_t)r * a.cks, r < s1, h, a.D);
#pragma unroll
        for (int x = 0; x < NV; ++x) {
            const int i = x * 64 + lane, row = row0 + i / PER_ROW, col = i % PER_ROW * V;
            vec16 t = (vec16)(T)0.0f;
            if (row < s1 && col < a.D) {
                const T *p = (row == at ? vn : vb + (int64_t)row * a.cvs) + col;
                if constexpr (VEC) {
                    t = *reinterpret_cast<const vec16 *>(p);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (col + e < a.D) t[e] = p[e];
                }
            }
            vr[x] = t;
        }
    };
    unsigned char *mine = lds + wave * 32 * PV;
    const int col_at = wa_col_offset<T>(lane, PV);
    int row0 = s0 + wave * 32;
    wa_arrived(q);
    if (row0 < s1) load(row0);
    for (; row0 < s1; row0 += 128) {
        // (the wavefront's own tile: the LDS serves a wavefront's accesses in the order of its instructions, no barrier -- the fences hold the compiler to it)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int x = 0; x < NV; ++x) {
            const int i = x * 64 + lane;
            *reinterpret_cast<vec16 *>(mine + i / PER_ROW * PV + i % PER_ROW * 16) = vr[x];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        v16f s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
        for (int x = 0; x < NS; ++x) s = LpTraits<T>::mfma(kf[x], q[x], s);
        if (row0 + 128 < s1) load(row0 + 128);
        if (row0 + 32 > s1) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = row0 + 8 * (r >> 2) + 4 * h + (r & 3) < s1 ? s[r] : -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
        top = half_wave_max(top);
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
        for (int r = 0; r < 16; ++r) {
            s[r] = wa_prob<sizeof(T) == 4>(s[r], top0, base, a.c);
            l += s[r];
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const vec pr = wa_pack<T>(s, x);
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t] = LpTraits<T>::mfma(wa_col<T, PV>(mine + col_at, 16 * x, t), pr, acc[t]);
            if constexpr (sizeof(T) == 2) {                    // what the rounding left of them: the products are not what bounds this kernel
#pragma unroll
                for (int e = 0; e < 8; ++e) s[8 * x + e] -= (float)pr[e];
                const vec rest = wa_pack<T>(s, x);
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[t] = LpTraits<T>::mfma(wa_col<T, PV>(mine + col_at, 16 * x, t), rest, acc[t]);
            }
        }
    }
    l = half_wave_sum(l);
    __syncthreads();
    // the four wavefronts' softmaxes: accumulators [wave][head][DP + 4]
    float *res = reinterpret_cast<float *>(lds);
    constexpr int RP = DP + 4;
    if (c < heads) {
        float *row = res + (wave * 32 + c) * RP;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) row[32 * t + 8 * (r >> 2) + 4 * h + (r & 3)] = acc[t][r];
        if (h == 0) {
            s_m[wave][c] = m;
            s_l[wave][c] = l;
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < heads * a.D; e += kWaThreads) {
        const int g = e / a.D, d = e % a.D;
        const float top = fmaxf(fmaxf(s_m[0][g], s_m[1][g]), fmaxf(s_m[2][g], s_m[3][g]));
        float o = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = s_m[w][g] == -INFINITY ? 0.0f : exp2f((s_m[w][g] - top) * a.c);
            o = fmaf(f, res[(w * 32 + g) * RP + d], o);
            sum = fmaf(f, s_l[w][g], sum);
        }
        if (a.splits == 1) {
            static_cast<T *>(a.out)[b * a.ob + (hq0 + g) * a.oh + d] = (T)(sum > 0.0f ? o / sum : 0.0f);
        } else {
            float *out = a.part + (((int64_t)b * a.Hq + hq0 + g) * a.splits + split) * (a.D + 2);
            out[d] = o;
            if (d == 0) {
                out[a.D] = top;
                out[a.D + 1] = sum;
            }
        }
    }
}

// joins the splits of one (stream, head): a thread per feature
template <typename T>
__global__ __launch_bounds__(kWsJoinThreads) void k_window_attn_step_join(WsArgs a) {
    const int b = (int)(blockIdx.x / a.Hq), hq = (int)(blockIdx.x % a.Hq), d = threadIdx.x;
    if (d >= a.D) return;
    const float *part = a.part + ((int64_t)b * a.Hq + hq) * a.splits * (a.D + 2);
    float top = -INFINITY, o = 0.0f, sum = 0.0f;
    for (uint32_t s = 0; s < a.splits; ++s) top = fmaxf(top, part[s * (a.D + 2) + a.D]);
    for (uint32_t s = 0; s < a.splits; ++s) {
        const float *p = part + s * (a.D + 2);
        const float f = p[a.D] == -INFINITY ? 0.0f : exp2f((p[a.D] - top) * a.c);
        o = fmaf(f, p[d], o);
        sum = fmaf(f, p[a.D + 1], sum);
    }
    static_cast<T *>(a.out)[b * a.ob + hq * a.oh + d] = (T)(sum > 0.0f ? o / sum : 0.0f);
}

template <typename T>
static void ws_launch(const WsArgs &a, bool vec, uint32_t grid, hipStream_t st) {
    if (a.D <= 32) vec ? k_window_attn_step<T, 32, true><<<grid, kWaThreads, 0, st>>>(a) : k_window_attn_step<T, 32, false><<<grid, kWaThreads, 0, st>>>(a);
    else if (a.D <= 64) vec ? k_window_attn_step<T, 64, true><<<grid, kWaThreads, 0, st>>>(a) : k_window_attn_step<T, 64, false><<<grid, kWaThreads, 0, st>>>(a);
    else vec ? k_window_attn_step<T, 128, true><<<grid, kWaThreads, 0, st>>>(a) : k_window_attn_step<T, 128, false><<<grid, kWaThreads, 0, st>>>(a);
    if (a.splits > 1) k_window_attn_step_join<T><<<(uint32_t)a.B * a.Hq, kWsJoinThreads, 0, st>>>(a);
}

// Stretches that a stream's slots are cut into, us measured with 8 key heads of 128 features, 4 100 slots.
// Groups (of query heads that share keys) for half the CUs at most: one workgroup per CU (4 streams: 88 whole, 28 in 8 stretches; 16 streams: 97 and 65 in 2), of 320
// slots at least -- below, the second launch costs what the stretches save (1 stream, 64 features, 516 slots: 8.4 whole, 9.0 in 2; 1 028 slots: 11.5 whole, 10.1 in 3).
// More groups: five stretches, so that one workgroup's start and end lie under the loads of others (64 streams: 219 whole, 204 in 5, 221 in 12), of 768 slots at least
// (32 streams x 8 heads x 64, 1 028 slots: 22 whole, 26 in 2).  The one size in between that would rather stay whole is one group per CU (107, 114 in 5).
static uint32_t ws_splits(uint32_t B, uint32_t Hq, uint32_t Hk, uint32_t slots) {
    const uint64_t groups = (uint64_t)B * Hk * (((uint64_t)Hq / Hk + 31) / 32), cus = (uint64_t)cu_count();
    if (groups == 0) return 1;
    const bool few = groups * 2 <= cus;
    const uint64_t want = few ? (cus + groups - 1) / groups : 5, most = slots / (few ? 320 : 768), n = want < most ? want : most;
    return n < 1 ? 1 : (uint32_t)n;
}

}  // namespace gfpp

using namespace gfpp;

#define WS_REQUIRE(cond)                                                                        \
    do {                                                                                        \
        if (!(cond)) {                                                                          \
            set_error("gfpp_window_attn_step: invalid argument (%s)", #cond);                   \
            return GFPP_EINVAL;                                                                 \
        }                                                                                       \
    } while (0)

GFPP_API unsigned long long gfpp_window_attn_step_scratch_floats(uint32_t B, uint32_t Hq, uint32_t Hk, uint32_t D, uint32_t slots) {
    if (Hk == 0 || Hq % Hk) return 0;
    const uint32_t s = ws_splits(B, Hq, Hk, slots);
    return s > 1 ? (unsigned long long)B * Hq * s * (D + 2) : 0;
}

GFPP_API int gfpp_window_attn_step(const void *q, const void *k, const void *v, void *cache_k, void *cache_v, const void *positions, int positions64, void *out,
                                   const int64_t *strides, uint32_t B, uint32_t Hq, uint32_t Hk, uint32_t D, uint32_t slots, uint32_t sinks, float scale, int dtype,
                                   float *scratch, gfpp_stream_t stream) {
    const uint32_t most = 1u << 29;
    WS_REQUIRE(dtype == GFPP_F32 || dtype == GFPP_F16 || dtype == GFPP_BF16);
    WS_REQUIRE(B <= most && Hq >= 1 && Hk >= 1 && Hq <= most && Hq % Hk == 0 && strides);
    WS_REQUIRE(slots >= 1 && slots <= most && sinks < slots);
    WS_REQUIRE(scale > 0.0f && scale < INFINITY);
    if (D < 1 || D > 128) {
        set_error("gfpp_window_attn_step: head width %u (1 .. 128 are supported)", D);
        return GFPP_EUNSUPPORTED;
    }
    if (B == 0) return 0;
    WS_REQUIRE(q && k && v && cache_k && cache_v && positions && out);
    WsArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.ck = cache_k;
    a.cv = cache_v;
    a.out = out;
    a.pos = positions;
    a.pos64 = positions64 != 0;
    a.part = scratch;
    const int64_t *s = strides;
    a.qb = s[0], a.qh = s[1], a.kb = s[2], a.kh = s[3], a.vb = s[4], a.vh = s[5];
    a.ckb = s[6], a.cks = s[7], a.ckh = s[8], a.cvb = s[9], a.cvs = s[10], a.cvh = s[11], a.ob = s[12], a.oh = s[13];
    a.B = (int)B;
    a.Hq = (int)Hq;
    a.Hk = (int)Hk;
    a.D = (int)D;
    a.G = (int)(Hq / Hk);
    a.slots = (int)slots;
    a.sinks = (int)sinks;
    a.chunks = (a.G + 31) / 32;
    a.c = scale * 1.4426950408889634f;
    a.splits = ws_splits(B, Hq, Hk, slots);
    WS_REQUIRE(a.splits == 1 || scratch);
    a.per_split = (int)(div_up(div_up(slots, a.splits), 32) * 32);
    WS_REQUIRE(grid_fits(kWaThreads, B, Hk, a.chunks, a.splits) && (a.splits == 1 || grid_fits(kWsJoinThreads, B, Hq)));
    const uint32_t grid = B * Hk * (uint32_t)a.chunks * a.splits;
    const size_t size = dtype == GFPP_F32 ? 4 : 2;
    uint64_t bits = (uint64_t)(uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)cache_k | (uintptr_t)cache_v | (uint64_t)D * size;
    for (int x = 0; x < 12; ++x) bits |= (uint64_t)s[x] * size;
    const bool vec = bits % 16 == 0;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GFPP_F32) ws_launch<float>(a, vec, grid, st);
    else if (dtype == GFPP_F16) ws_launch<_Float16>(a, vec, grid, st);
    else ws_launch<__bf16>(a, vec, grid, st);
    return check_launch("gfpp_window_attn_step");
}
