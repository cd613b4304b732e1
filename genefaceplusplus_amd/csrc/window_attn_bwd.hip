// window_attn_bwd.hip -- backward pass of the windowed attention (gfx950; rule of visibility and fragments: window_attn_device.h).
//
//   p_ij = exp(s_ij - lse_i),  delta_i = sum_d dout_id out_id,  ds_ij = p_ij (dout_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij dout_i
//
// Two launches that both recompute the probabilities from the saved row sums: dq by tiles of queries (it also leaves delta), then dk and dv by tiles of keys.  No
// atomics: every gradient is summed by one workgroup in a fixed order, the heads of a group one after the other.  The tiles that hold sinks are seen by ALL later
// queries; their queries are cut into slices that leave fp32 partial sums, which a third launch adds in the slices' order.
// delta is a matrix product's diagonal, taken by the instructions that compute dout . v: where a query sees one key only, out = v and ds is exactly zero.
// p and ds are rounded to the operand type (16-bit modes) for the matrix instruction; every sum is fp32.
#include "window_attn_device.h"

namespace gfpp {

int wa_arguments(const char *what, WaArgs &a, const int64_t *strides, int n_tensors, uint32_t B, uint32_t Tq, uint32_t Tk, uint32_t Hq, uint32_t Hk, uint32_t D, int32_t left,
                 int32_t right, int32_t sinks, int32_t q_start, const int32_t *lengths, float scale, int dtype);
bool wa_vectors(const WaTensor &t, int D, size_t size);

template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(kWaThreads, sizeof(T) == 2 ? 2 : 1) void k_window_attn_dq(WaArgs a) {
    constexpr int BN = sizeof(T) == 4 && DP == 128 ? 32 : 64, NS = DP / 16, NT = DP / 32, PK = wa_pitch_both<T, DP>(), PV = wa_pitch_row<T, DP>();
    typedef typename LpTraits<T>::vec vec;
    __shared__ __attribute__((aligned(16))) unsigned char s_k[2][BN * PK], s_v[2][BN * PV];
    const int q_tiles = (a.Tq + kWaRows - 1) / kWaRows;
    const int hq = (int)(blockIdx.x / q_tiles) % a.Hq, b = (int)(blockIdx.x / q_tiles) / a.Hq, i0 = (int)(blockIdx.x % q_tiles) * kWaRows, hk = hq / a.G;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
    const int n = a.lengths ? a.lengths[b] < a.Tk ? a.lengths[b] : a.Tk : a.Tk;
    const int i = i0 + wave * 32 + c, p = a.q_start + i;
    const bool have = i < a.Tq && p < n;                       // (rows behind the sequence: zeros, whatever they hold)
    vec q[NS], g[NS];
    wa_global_rows<T, NS, VEC>(q, static_cast<const T *>(a.q.p) + b * a.q.sb + (int64_t)i * a.q.st + hq * a.q.sh, have, h, a.D);
    wa_global_rows<T, NS, VEC>(g, static_cast<const T *>(a.dout.p) + b * a.dout.sb + (int64_t)i * a.dout.st + hq * a.dout.sh, have, h, a.D);
    const int64_t stat = ((int64_t)b * a.Hq + hq) * a.Tq + i;
    const float lse = have ? a.lse[stat] : INFINITY;
    float delta = 0.0f;
    {
        v16f d;
#pragma unroll
        for (int r = 0; r < 16; ++r) d[r] = 0.0f;
        vec o[NS];
        wa_global_rows<T, NS, VEC>(o, static_cast<const T *>(a.o.p) + b * a.o.sb + (int64_t)i * a.o.st + hq * a.o.sh, have, h, a.D);
#pragma unroll
        for (int x = 0; x < NS; ++x) d = LpTraits<T>::mfma(o[x], g[x], d);
        if (a.low) {                                           // (wa_two_part: what the rounding of out took)
            wa_global_rows<T, NS, VEC>(o, static_cast<const T *>(a.low) + b * a.o.sb + (int64_t)i * a.o.st + hq * a.o.sh, have, h, a.D);
#pragma unroll
            for (int x = 0; x < NS; ++x) d = LpTraits<T>::mfma(o[x], g[x], d);
        }
        // the diagonal: column c's value of row c is in the half (c >> 2) & 1, register 4 (c >> 3) + (c & 3)
#pragma unroll
        for (int r = 0; r < 16; ++r) delta = (4 * (c >> 3) + (c & 3)) == r ? d[r] : delta;
        delta = ((c >> 2) & 1) == h ? delta : 0.0f;
        delta = half_wave_sum(delta);
        if (h == 0 && i < a.Tq) a.delta[stat] = delta;
    }
    const int i1 = i0 + kWaRows < a.Tq ? i0 + kWaRows - 1 : a.Tq - 1;
    const WaRange range = wa_keys<BN>(a, a.q_start + i0, a.q_start + i1, n);
    const int tiles = range.head + range.hi - range.lo;
    const int last = have ? (p + a.right < n - 1 ? p + a.right : n - 1) : -1, first = p - a.left;
    const int pw0 = a.q_start + i0 + wave * 32, pw1 = pw0 + 31;
    v16f acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.0f;
    const T *kb = static_cast<const T *>(a.k.p) + b * a.k.sb + hk * a.k.sh, *vb = static_cast<const T *>(a.v.p) + b * a.v.sb + hk * a.v.sh;
    WaStage<T, DP, BN, VEC> rk, rv;
    auto tile_row = [&](int k) { return (k < range.head ? k : range.lo + k - range.head) * BN; };
    if (tiles > 0) {
        rk.load(kb, a.k.st, tile_row(0), n, a.D);
        rv.load(vb, a.v.st, tile_row(0), n, a.D);
        rk.store(s_k[0], PK);
        rv.store(s_v[0], PV);
        if (tiles > 1) {
            rk.load(kb, a.k.st, tile_row(1), n, a.D);
            rv.load(vb, a.v.st, tile_row(1), n, a.D);
        }
    }
    wa_arrived(q);
    wa_arrived(g);
    __syncthreads();
    const int row_k = c * PK + 8 * h * (int)sizeof(T), row_v = c * PV + 8 * h * (int)sizeof(T), col_at = wa_col_offset<T>(lane, PK);
    for (int k = 0; k < tiles; ++k) {
        const int buf = k & 1, j0 = tile_row(k), j1 = j0 + BN - 1;
        if (k + 1 < tiles) {
            rk.store(s_k[buf ^ 1], PK);
            rv.store(s_v[buf ^ 1], PV);
            if (k + 2 < tiles) {
                rk.load(kb, a.k.st, tile_row(k + 2), n, a.D);
                rv.load(vb, a.v.st, tile_row(k + 2), n, a.D);
            }
        }
        const bool seen = pw0 < n && j0 <= pw1 + a.right && (j1 >= pw0 - a.left || j0 < a.sinks);
        if (seen) {
            const bool full = pw1 < n && j1 < n && j1 <= pw0 + a.right && (j0 >= pw1 - a.left || j1 < a.sinks);
            // Two bodies without a branch inside: the products of one half tile may then overlap the arithmetic of the other.  The widest heads have no registers
            // for two half tiles at once (two wavefronts per SIMD overlap instead): one body, the branch between its products.
            auto body = [&](auto masked, auto always) {
#pragma unroll
                for (int u = 0; u < BN / 32; ++u) {
                    v16f s, d;
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = d[r] = 0.0f;
#pragma unroll
                    for (int x = 0; x < NS; ++x) s = LpTraits<T>::mfma(wa_row<T>(s_k[buf] + row_k + 32 * u * PK, x), q[x], s);
#pragma unroll
                    for (int x = 0; x < NS; ++x) d = LpTraits<T>::mfma(wa_row<T>(s_v[buf] + row_v + 32 * u * PV, x), g[x], d);
                    if (decltype(masked)::value && (decltype(always)::value || !full)) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int j = j0 + 32 * u + 8 * (r >> 2) + 4 * h + (r & 3);
                            s[r] = j <= last && (j >= first || j < a.sinks) ? s[r] : -INFINITY;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -lse)) * (d[r] - delta);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const vec ds = wa_pack<T>(s, x);
#pragma unroll
                        for (int t = 0; t < NT; ++t) acc[t] = LpTraits<T>::mfma(wa_col<T, PK>(s_k[buf] + col_at, 32 * u + 16 * x, t), ds, acc[t]);
                    }
                }
            };
            if constexpr (DP == 128) body(WaFlag<true>{}, WaFlag<false>{});
            else if (full) body(WaFlag<false>{}, WaFlag<false>{});
            else body(WaFlag<true>{}, WaFlag<true>{});
        }
        __syncthreads();
    }
    if (i < a.Tq) wa_store_rows<T, NT, VEC>(acc, a.scale, static_cast<T *>(a.dq.p) + b * a.dq.sb + (int64_t)i * a.dq.st + hq * a.dq.sh, h, a.D);
}

// dk and dv of 128 keys (a wavefront: 32), the queries in tiles of BQ through LDS.  Work items: first the slices of the tiles with sinks (a.splits each, partial
// sums), then the other tiles.
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(kWaThreads, 1) void k_window_attn_dkv(WaArgs a) {
    constexpr int BQ = sizeof(T) == 2 ? 64 : 32, NS = DP / 16, NT = DP / 32, PITCH = wa_pitch_both<T, DP>();
    typedef typename LpTraits<T>::vec vec;
    typedef float f4 __attribute__((ext_vector_type(4)));
    __shared__ __attribute__((aligned(16))) unsigned char s_q[2][BQ * PITCH], s_g[2][BQ * PITCH];
    __shared__ __attribute__((aligned(16))) float s_lse[2][BQ], s_delta[2][BQ];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
    const uint32_t bh = (uint32_t)a.B * a.Hk, sliced = a.sink_tiles * a.splits * bh;
    const bool slice = blockIdx.x < sliced;
    uint32_t item = slice ? blockIdx.x : blockIdx.x - sliced;
    const uint32_t hkb = item % bh;
    item /= bh;
    const uint32_t part = slice ? item % a.splits : 0;
    const int j0 = (int)(slice ? item / a.splits : item + a.sink_tiles) * kWaRows;
    const int hk = (int)(hkb % a.Hk), b = (int)(hkb / a.Hk);
    const int n = a.lengths ? a.lengths[b] < a.Tk ? a.lengths[b] : a.Tk : a.Tk;
    const int j = j0 + wave * 32 + c, jw0 = j0 + wave * 32, jw1 = jw0 + 31;
    const bool have = j < n;
    vec kf[NS], vf[NS];
    wa_global_rows<T, NS, VEC>(kf, static_cast<const T *>(a.k.p) + b * a.k.sb + (int64_t)j * a.k.st + hk * a.k.sh, have, h, a.D);
    wa_global_rows<T, NS, VEC>(vf, static_cast<const T *>(a.v.p) + b * a.v.sb + (int64_t)j * a.v.st + hk * a.v.sh, have, h, a.D);
    v16f dk[NT], dv[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[t][r] = dv[t][r] = 0.0f;
    // query rows [i_lo, i_hi) that can see a key of the tile; rows from `end` on are behind the sequence
    const int end = n - a.q_start < a.Tq ? n - a.q_start : a.Tq;
    const int jn = j0 + kWaRows <= n ? j0 + kWaRows - 1 : n - 1;
    int i_lo = j0 - a.right - a.q_start, i_hi = (j0 < a.sinks ? end : jn + a.left + 1 - a.q_start);
    i_lo = i_lo < 0 ? 0 : i_lo / BQ * BQ;
    i_hi = i_hi < end ? i_hi : end;
    if (j0 >= n) i_hi = i_lo;
    int tiles = i_hi > i_lo ? (i_hi - i_lo + BQ - 1) / BQ : 0;
    if (slice) {
        const int per = (tiles + (int)a.splits - 1) / (int)a.splits, t0 = per * (int)part;
        i_lo += t0 * BQ;
        tiles = tiles - t0 < per ? tiles - t0 : per;
        tiles = tiles < 0 ? 0 : tiles;
    }
    const int steps = tiles * a.G;
    WaStage<T, DP, BQ, VEC> rq, rg;
    float r_stat = 0.0f;
    auto load = [&](int s) {
        const int hq = hk * a.G + s / tiles, i = i_lo + s % tiles * BQ;
        rq.load(static_cast<const T *>(a.q.p) + b * a.q.sb + hq * a.q.sh, a.q.st, i, end, a.D);
        rg.load(static_cast<const T *>(a.dout.p) + b * a.dout.sb + hq * a.dout.sh, a.dout.st, i, end, a.D);
        if (threadIdx.x < 2 * BQ) {
            const int row = i + (int)(threadIdx.x % BQ);
            const int64_t at = ((int64_t)b * a.Hq + hq) * a.Tq + row;
            if (threadIdx.x < BQ) r_stat = row < end ? a.lse[at] : INFINITY;
            else r_stat = row < end ? a.delta[at] : 0.0f;
        }
    };
    auto store = [&](int buf) {
        rq.store(s_q[buf], PITCH);
        rg.store(s_g[buf], PITCH);
        if (threadIdx.x < BQ) s_lse[buf][threadIdx.x] = r_stat;
        else if (threadIdx.x < 2 * BQ) s_delta[buf][threadIdx.x - BQ] = r_stat;
    };
    if (steps > 0) {
        load(0);
        store(0);
        if (steps > 1) load(1);
    }
    wa_arrived(kf);
    wa_arrived(vf);
    __syncthreads();
    const int row_at = c * PITCH + 8 * h * (int)sizeof(T), col_at = wa_col_offset<T>(lane, PITCH);
    for (int k = 0; k < steps; ++k) {
        const int buf = k & 1, p0 = a.q_start + i_lo + k % tiles * BQ, p1 = p0 + BQ - 1;
        if (k + 1 < steps) {
            store(buf ^ 1);
            if (k + 2 < steps) load(k + 2);
        }
        const bool seen = jw0 < n && p1 >= jw0 - a.right && (p0 <= jw1 + a.left || jw0 < a.sinks);
        if (seen) {
            const bool full = jw1 < n && p0 >= jw1 - a.right && (p1 <= jw0 + a.left || jw1 < a.sinks);
            // (two bodies without a branch inside: the compiler overlaps the products of one sub-tile with the arithmetic of the other)
            auto body = [&](auto masked) {
#pragma unroll
                for (int u = 0; u < BQ / 32; ++u) {
                    v16f s, d;
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = d[r] = 0.0f;
#pragma unroll
                    for (int x = 0; x < NS; ++x) s = LpTraits<T>::mfma(wa_row<T>(s_q[buf] + row_at + 32 * u * PITCH, x), kf[x], s);
#pragma unroll
                    for (int x = 0; x < NS; ++x) d = LpTraits<T>::mfma(wa_row<T>(s_g[buf] + row_at + 32 * u * PITCH, x), vf[x], d);
                    if constexpr (decltype(masked)::value) {
                        const int from = have ? j - a.right : 0x7fffffff, to = j < a.sinks ? 0x7fffffff : j + a.left;
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int p = p0 + 32 * u + 8 * (r >> 2) + 4 * h + (r & 3);
                            s[r] = p >= from && p <= to ? s[r] : -INFINITY;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const f4 lse = *reinterpret_cast<const f4 *>(&s_lse[buf][32 * u + 2 * r + 4 * h]), delta = *reinterpret_cast<const f4 *>(&s_delta[buf][32 * u + 2 * r + 4 * h]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[r + e] = __builtin_amdgcn_exp2f(fmaf(s[r + e], a.c, -lse[e]));
                            d[r + e] = s[r + e] * (d[r + e] - delta[e]);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const vec pr = wa_pack<T>(s, x), ds = wa_pack<T>(d, x);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            dv[t] = LpTraits<T>::mfma(wa_col<T, PITCH>(s_g[buf] + col_at, 32 * u + 16 * x, t), pr, dv[t]);
                            dk[t] = LpTraits<T>::mfma(wa_col<T, PITCH>(s_q[buf] + col_at, 32 * u + 16 * x, t), ds, dk[t]);
                        }
                    }
                }
            };
            if (full) body(WaFlag<false>{});
            else body(WaFlag<true>{});
        }
        __syncthreads();
    }
    if (j >= a.Tk) return;
    if (slice) {
        float *out = a.partial + ((((int64_t)(j0 / kWaRows) * a.splits + part) * bh + hkb) * 2 * kWaRows + (j - j0)) * a.D;
        wa_store_rows<float, NT, false>(dk, a.scale, out, h, a.D);
        wa_store_rows<float, NT, false>(dv, 1.0f, out + kWaRows * a.D, h, a.D);
    } else {
        wa_store_rows<T, NT, VEC>(dk, a.scale, static_cast<T *>(a.dk.p) + b * a.dk.sb + (int64_t)j * a.dk.st + hk * a.dk.sh, h, a.D);
        wa_store_rows<T, NT, VEC>(dv, 1.0f, static_cast<T *>(a.dv.p) + b * a.dv.sb + (int64_t)j * a.dv.st + hk * a.dv.sh, h, a.D);
    }
}

// the slices' sums of the tiles with sinks, added in order
template <typename T>
__global__ __launch_bounds__(kWaThreads) void k_window_attn_join(WaArgs a) {
    const uint32_t bh = (uint32_t)a.B * a.Hk, hkb = blockIdx.y, tile = blockIdx.z;
    const int hk = (int)(hkb % a.Hk), b = (int)(hkb / a.Hk);
    const int64_t size = 2ll * kWaRows * a.D, stride = (int64_t)bh * size;
    const float *src = a.partial + ((int64_t)tile * a.splits * bh + hkb) * size;
    for (int64_t e = blockIdx.x * kWaThreads + threadIdx.x; e < size; e += (int64_t)gridDim.x * kWaThreads) {
        const int which = e >= (int64_t)kWaRows * a.D, r = (int)(e / a.D) - which * kWaRows, d = (int)(e % a.D);
        const int64_t j = (int64_t)tile * kWaRows + r;
        if (j >= a.Tk) continue;
        float sum = 0.0f;
        for (uint32_t s = 0; s < a.splits; ++s) sum += src[s * stride + e];
        const WaTensor &t = which ? a.dv : a.dk;
        static_cast<T *>(t.p)[b * t.sb + j * t.st + hk * t.sh + d] = (T)sum;
    }
}

// slices of a tile with sinks: enough for the chip, at least 512 queries each
static uint32_t wa_splits(uint32_t sink_tiles, uint64_t bh, uint32_t Tq) {
    if (sink_tiles == 0) return 1;
    const uint64_t want = ((uint64_t)cu_count() + sink_tiles * bh - 1) / (sink_tiles * bh), most = Tq / 512;
    const uint64_t n = want < most ? want : most;
    return n < 1 ? 1 : (uint32_t)n;
}
static uint32_t wa_sink_tiles(const WaArgs &a) {
    // a window that reaches every query from its first key makes the sinks ordinary keys
    if (a.sinks == 0 || (int64_t)a.left + 1 >= (int64_t)a.q_start + a.Tq) return 0;
    return (uint32_t)(a.sinks + kWaRows - 1) / kWaRows;
}

template <typename T>
static void wa_backward(const WaArgs &a, bool vec, uint32_t gq, uint32_t gk, hipStream_t st) {
#define WA_BOTH(DP)                                                                                                                    \
    do {                                                                                                                               \
        if (gq) vec ? k_window_attn_dq<T, DP, true><<<gq, kWaThreads, 0, st>>>(a) : k_window_attn_dq<T, DP, false><<<gq, kWaThreads, 0, st>>>(a);    \
        if (gk) vec ? k_window_attn_dkv<T, DP, true><<<gk, kWaThreads, 0, st>>>(a) : k_window_attn_dkv<T, DP, false><<<gk, kWaThreads, 0, st>>>(a);  \
    } while (0)
    if (a.D <= 32) WA_BOTH(32);
    else if (a.D <= 64) WA_BOTH(64);
    else WA_BOTH(128);
#undef WA_BOTH
    if (a.sink_tiles && gk)
        k_window_attn_join<T><<<dim3(div_up(2 * kWaRows * a.D, kWaThreads), (uint32_t)(a.B * a.Hk), a.sink_tiles), kWaThreads, 0, st>>>(a);
}

}  // namespace gfpp

using namespace gfpp;

#define WA_REQUIRE(cond)                                               \
    do {                                                               \
        if (!(cond)) {                                                 \
            set_error("%s: invalid argument (%s)", what, #cond);       \
            return GFPP_EINVAL;                                        \
        }                                                              \
    } while (0)

static void wa_bwd_setup(WaArgs &a) {
    a.sink_tiles = wa_sink_tiles(a);
    a.splits = wa_splits(a.sink_tiles, (uint64_t)a.B * a.Hk, (uint32_t)a.Tq);
    if (a.splits == 1) a.sink_tiles = 0;                       // whole tiles write their gradients themselves
}

GFPP_API unsigned long long gfpp_window_attn_backward_scratch_floats(uint32_t B, uint32_t Tq, uint32_t Tk, uint32_t Hq, uint32_t Hk, uint32_t D, int32_t left,
                                                                     int32_t sinks, int32_t q_start) {
    if (Hk == 0 || Tq > (1u << 29) || Tk > (1u << 29) || sinks < 0 || left < 0) return 0;
    WaArgs a{};
    a.B = (int)B;
    a.Hk = (int)Hk;
    a.Tq = (int)Tq;
    a.left = left < (1 << 29) ? left : 1 << 29;                // (as wa_arguments has them)
    a.sinks = sinks < (int)Tk ? sinks : (int)Tk;
    a.q_start = q_start;
    wa_bwd_setup(a);
    return (unsigned long long)B * Hq * Tq + (unsigned long long)a.sink_tiles * a.splits * B * Hk * 2 * kWaRows * D;
}

GFPP_API int gfpp_window_attn_backward(const void *q, const void *k, const void *v, const void *out, const void *out_low, const void *dout, const float *lse, void *dq, void *dk, void *dv,
                                       float *scratch, const int64_t *strides, uint32_t B, uint32_t Tq, uint32_t Tk, uint32_t Hq, uint32_t Hk, uint32_t D, int32_t left,
                                       int32_t right, int32_t sinks, int32_t q_start, const int32_t *lengths, float scale, int dtype, gfpp_stream_t stream) {
    const char *what = "gfpp_window_attn_backward";
    WaArgs a{};
    if (int rc = wa_arguments(what, a, strides, 8, B, Tq, Tk, Hq, Hk, D, left, right, sinks, q_start, lengths, scale, dtype)) return rc;
    if (B == 0 || (Tq == 0 && Tk == 0)) return 0;
    WA_REQUIRE(Tq == 0 || (q && out && dout && lse && dq && scratch));
    WA_REQUIRE(Tk == 0 || (k && v && dk && dv));
    a.q.p = const_cast<void *>(q);
    a.k.p = const_cast<void *>(k);
    a.v.p = const_cast<void *>(v);
    a.o.p = const_cast<void *>(out);
    a.dout.p = const_cast<void *>(dout);
    a.dq.p = dq;
    a.dk.p = dk;
    a.dv.p = dv;
    a.low = wa_two_part(Tk, left, right, sinks, dtype) ? const_cast<void *>(out_low) : nullptr;
    a.lse = const_cast<float *>(lse);
    wa_bwd_setup(a);
    a.delta = scratch;
    a.partial = scratch ? scratch + (uint64_t)B * Hq * Tq : nullptr;
    const uint64_t bh = (uint64_t)B * Hk, gq = (uint64_t)div_up(Tq, kWaRows) * Hq * B;
    const uint64_t gk = ((uint64_t)div_up(Tk, kWaRows) - a.sink_tiles + (uint64_t)a.sink_tiles * a.splits) * bh;
    WA_REQUIRE(gq <= 0x7fffffffull && gk <= 0x7fffffffull && (a.sink_tiles == 0 || (bh <= 65535 && a.sink_tiles <= 65535)));
    const size_t size = dtype == GFPP_F32 ? 4 : 2;
    bool vec = (uintptr_t)a.low % 16 == 0;
    for (const WaTensor *t : {&a.q, &a.k, &a.v, &a.o, &a.dout, &a.dq, &a.dk, &a.dv}) vec = vec && wa_vectors(*t, a.D, size);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GFPP_F32) wa_backward<float>(a, vec, (uint32_t)gq, (uint32_t)gk, st);
    else if (dtype == GFPP_F16) wa_backward<_Float16>(a, vec, (uint32_t)gq, (uint32_t)gk, st);
    else wa_backward<__bf16>(a, vec, (uint32_t)gq, (uint32_t)gk, st);
    return check_launch(what);
}
