// window_attn_bwd.hip -- backward pass of the windowed attention (gfx950; rule of visibility and fragments: window_attn_device.h).
//
//   p_ij = exp(s_ij - lse_i),  delta_i = sum_d dout_id out_id,  ds_ij = p_ij (dout_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij dout_i
//
// Two launches that both recompute the probabilities from the saved row sums: dq by tiles of queries (it also leaves delta), then dk and dv by tiles of keys.  No
// atomics: every gradient is summed by one workgroup in a fixed order, the heads of a group one after the other.  The tiles that hold sinks are seen by ALL later
// queries; their queries are cut into slices that leave fp32 partial sums, which a third launch adds in the slices' order.
// delta is a matrix product's diagonal, taken by the instructions that compute dout . v: where a query sees one key only, out = v and ds is exactly zero.
// p and ds are rounded to the operand type (16-bit modes) for the matrix instruction; every sum is fp32.  A choice, as in the forward pass: the gradients' error against 64 bits grows
// from 1.7e-3 of their norm (their own rounding) to 2.4e-3 (bf16), and two parts each would take half as many products again for dk and dv, a third for dq.
#include "window_attn_device.h"

namespace gfpp {

int wa_arguments(const char *what, WaArgs &a, const int64_t *strides, int n_tensors, uint32_t B, uint32_t Tq, uint32_t Tk, uint32_t Hq, uint32_t Hk, uint32_t D, int32_t left,
                 int32_t right, int32_t sinks, int32_t q_start, const int32_t *lengths, float scale, int dtype);
bool wa_vectors(const WaTensor &t, int D, size_t size);

// dq of 128 queries of one head, 32 a wavefront, over tiles of keys and values in LDS; s and dout . v both as K Q^T and V dout^T, so that ds is the operand of dq^T += K^T ds^T
// without leaving its registers.  Measured (bf16): 16 384 x 16 heads on 4 x 128, window 2 049: 406 us (400 GFLOP, 0.98 PFLOP/s; matrix pipe busy in 49 % of the CUs' cycles,
// LDS in 41 %, a fifth of that bank conflicts; two heads of a group on one workgroup, as in the forward pass: no difference); 13 000 x 8 on 2 x 64, window 1 024, 4 sinks: 84 us
// (39 GFLOP, 0.47 PFLOP/s; 36 and 31 %).
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(kWaThreads, sizeof(T) == 2 && (VEC || DP <= 64) ? 2 : 1) void k_window_attn_dq(WaArgs a) {
    constexpr int BN = DP == 128 ? 32 : 64, NS = DP / 16, NT = DP / 32, PK = wa_pitch_both<T, DP>(), PV = wa_pitch_row<T, DP>();
    typedef typename LpTraits<T>::vec vec;
    __shared__ __attribute__((aligned(16))) unsigned char s_k[2][BN * PK], s_v[2][BN * PV];
    const int q_tiles = (a.Tq + kWaRows - 1) / kWaRows;
    // items: sequence, key head, tile of queries, query head of the group -- those that read the same keys side by side
    uint32_t item = wa_item(blockIdx.x, gridDim.x);
    const int in_group = (int)(item % a.G);
    item /= a.G;
    const int i0 = (int)(item % q_tiles) * kWaRows;
    item /= q_tiles;
    const int hk = (int)(item % a.Hk), hq = hk * a.G + in_group, b = (int)(item / a.Hk);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), c = lane & 31, h = lane >> 5;
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
    // two tiles in flight: the one that the next step stores and the one after it (one alone arrives later than the step that it was requested in takes)
    WaStage<T, DP, BN, VEC, kWaThreads> rk[2], rv[2];
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
    wa_arrived(g);
    __syncthreads();
    const int row_k = c * PK + 8 * h * (int)sizeof(T), row_v = c * PV + 8 * h * (int)sizeof(T), col_at = wa_col_offset<T>(lane, PK);
    auto step = [&](int k, auto which) {
        constexpr int buf = decltype(which)::value, other = buf ^ 1;
        const int j0 = tile_row(k), j1 = j0 + BN - 1;
        rk[other].store(s_k[other], PK);                         // (last read before the previous barrier)
        rv[other].store(s_v[other], PV);
        load(other, k + 3);
        const bool seen = pw0 < n && j0 <= pw1 + a.right && (j1 >= pw0 - a.left || j0 < a.sinks);
        if (seen) {
            const bool full = pw1 < n && j1 < n && j1 <= pw0 + a.right && (j0 >= pw1 - a.left || j1 < a.sinks);
#pragma unroll
            for (int u = 0; u < BN / 32; ++u) {
                v16f s, d;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = d[r] = 0.0f;
                {
                    WaStream<T, 2 * NS> rows;                  // keys, then values
                    const auto read = [&](int x) { return x < NS ? wa_row<T>(s_k[buf] + row_k + 32 * u * PK, x) : wa_row<T>(s_v[buf] + row_v + 32 * u * PV, x - NS); };
                    rows.prime(read);
                    rows.run(read, [&](int x, const vec &f) {
                        if (x < NS) s = LpTraits<T>::mfma(f, q[x % NS], s);
                        else d = LpTraits<T>::mfma(f, g[x % NS], d);
                    });
                }
                WaStream<T, 2 * NT> cols;
                const auto read_k = [&](int x) { return wa_col<T, PK>(s_k[buf] + col_at, 32 * u + 16 * (x / NT), x % NT); };
                cols.prime(read_k);
                if (!full) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int j = j0 + 32 * u + 8 * (r >> 2) + 4 * h + (r & 3);
                        s[r] = j <= last && (j >= first || j < a.sinks) ? s[r] : -INFINITY;
                    }
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -lse)) * (d[r] - delta);
                vec ds;
                cols.run(read_k, [&](int x, const vec &f) {
                    if (x % NT == 0) ds = wa_pack<T>(s, x / NT);
                    acc[x % NT] = LpTraits<T>::mfma(f, ds, acc[x % NT]);
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
    if (i < a.Tq) wa_store_rows<T, NT, VEC>(acc, a.scale, static_cast<T *>(a.dq.p) + b * a.dq.sb + (int64_t)i * a.dq.st + hq * a.dq.sh, h, a.D);
}

// dk and dv of 64 keys, the queries in tiles of 32 through LDS.  Two wavefronts for every 32 keys: one makes the probabilities and sums dv, the other takes
// them a tile later (through LDS, in fp32), makes ds and sums dk.  One wavefront doing both would hold 128 accumulators, 64 registers of K and V and both products, and
// be alone on its SIMD.  Halved, two or three share a SIMD and fill each other's waits; the work is the same (four products per tile, none twice).
// Three tiles are held: the one being stored, the one that is read by the first wavefronts and the one that is read by the second.  AHEAD (16-bit heads of 33 to 64
// features): the second take their product with dout a tile early and hold it, so that two tiles of dout are enough and three workgroups fit a CU.
// Work items: first the slices of the tiles with sinks (a.splits each, partial sums), then the other tiles.
// Neither the matrix pipe nor the LDS is full; the wavefronts of a pair wait for one another at every tile's barrier.  Measured (bf16): 16 384 x 16 heads on 4 x 128, window 2 049:
// 725 us (533 GFLOP, 0.74 PFLOP/s; matrix pipe busy in 33 % of the CUs' cycles, LDS in 44 %, a fifth of that bank conflicts); 13 000 x 8 on 2 x 64, window 1 024, 4 sinks: 153 us
// (53 GFLOP, 0.35 PFLOP/s; 18 and 30 %: 430 workgroups where 768 fit).  128 keys a workgroup instead of 64 took within 1.5 % of that at 128 features and 3 to 20 %
// more at 64 and fewer (16 384 x 16 heads x 64, window 301: dq, dk and dv together 289 us against 237, and 206 with AHEAD).
constexpr int kWaBq = 32, kWaKeys = 64, kWaPairs = kWaKeys / 32;
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(kWaThreads, DP == 128 && (sizeof(T) == 4 || !VEC) ? 1 : (DP == 64 && sizeof(T) == 2 && VEC ? 3 : 2)) void k_window_attn_dkv(WaArgs a) {
    constexpr int BQ = kWaBq, NS = DP / 16, NT = DP / 32, PITCH = wa_pitch_both<T, DP>();
    constexpr bool AHEAD = DP == 64 && sizeof(T) == 2;
    typedef typename LpTraits<T>::vec vec;
    typedef float f4 __attribute__((ext_vector_type(4)));
    __shared__ __attribute__((aligned(16))) unsigned char s_q[3][BQ * PITCH], s_g[AHEAD ? 2 : 3][BQ * PITCH];
    __shared__ __attribute__((aligned(16))) float s_p[2][kWaPairs][4][64][4];                 // [tile & 1][32 keys][quad of rows][lane][row]
    __shared__ __attribute__((aligned(16))) float s_lse[3][BQ], s_delta[3][BQ];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), keys = wave % kWaPairs, c = lane & 31, h = lane >> 5;
    const bool second = wave >= kWaPairs;
    const uint32_t bh = (uint32_t)a.B * a.Hk, sliced = a.sink_tiles * a.splits * bh;
    const bool slice = blockIdx.x < sliced;
    uint32_t item = slice ? blockIdx.x : wa_item(blockIdx.x - sliced, gridDim.x - sliced);
    const uint32_t per_head = slice ? a.sink_tiles * a.splits : (gridDim.x - sliced) / bh, hkb = item / per_head;
    item %= per_head;
    const uint32_t part = slice ? item % a.splits : 0;
    const int j0 = (int)(slice ? item / a.splits : item + a.sink_tiles) * kWaKeys;
    const int hk = (int)(hkb % a.Hk), b = (int)(hkb / a.Hk);
    const int n = a.lengths ? a.lengths[b] < a.Tk ? a.lengths[b] : a.Tk : a.Tk;
    const int jw0 = j0 + keys * 32, jw1 = jw0 + 31, j = jw0 + c;
    const bool have = j < n;
    vec f[NS];                                                                         // the lane's key (first) or value (second)
    const WaTensor &own = second ? a.v : a.k;
    wa_global_rows<T, NS, VEC>(f, static_cast<const T *>(own.p) + b * own.sb + (int64_t)j * own.st + hk * own.sh, have, h, a.D);
    v16f acc[NT];                                                                      // dv (first) or dk (second)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.0f;
    // query rows [i_lo, i_hi) that can see a key of the tile; rows from `end` on are behind the sequence
    const int end = n - a.q_start < a.Tq ? n - a.q_start : a.Tq;
    const int jn = j0 + kWaKeys <= n ? j0 + kWaKeys - 1 : n - 1;
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
    WaStage<T, DP, BQ, VEC, kWaThreads> rq[2], rg[2];                                 // two tiles in flight (k_window_attn)
    float r_lse[2], r_delta[2];
    int next_tile = 0, next_head = 0, loaded = 0;                                      // of the tile that is loaded next: the heads of a group one after the other
    // (unconditional, as in the forward pass: past the last tile the ranges are empty)
    auto load = [&](int which) {
        const bool more = loaded < steps;
        const int hq = hk * a.G + (more ? next_head : 0), i = more ? i_lo + next_tile * BQ : (end > 0 ? end : 0);
        rq[which].load(static_cast<const T *>(a.q.p) + b * a.q.sb + hq * a.q.sh, a.q.st, i, end, a.D);
        rg[which].load(static_cast<const T *>(a.dout.p) + b * a.dout.sb + hq * a.dout.sh, a.dout.st, i, end, a.D);
        const int64_t at = ((int64_t)b * a.Hq + hq) * a.Tq + i;
        const int rows = __builtin_amdgcn_readfirstlane(end - i < BQ ? (end - i > 0 ? end - i : 0) : BQ);
        const int off = threadIdx.x < BQ ? (int)threadIdx.x * 4 : 0x7ffffff0;
        r_lse[which] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(__builtin_amdgcn_make_buffer_rsrc(a.lse + at, 0, rows * 4, 0x00020000), off, 0, 0));
        r_delta[which] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(__builtin_amdgcn_make_buffer_rsrc(a.delta + at, 0, rows * 4, 0x00020000), off, 0, 0));
        if ((int)threadIdx.x >= rows) r_lse[which] = INFINITY;                         // rows behind the sequence: probability 0
        ++loaded;
        if (++next_tile == tiles) {
            next_tile = 0;
            ++next_head;
        }
    };
    auto store = [&](int buf, int which) {
        rq[which].store(s_q[buf], PITCH);
        rg[which].store(s_g[AHEAD ? which : buf], PITCH);
        if (threadIdx.x < BQ) {
            s_lse[buf][threadIdx.x] = r_lse[which];
            s_delta[buf][threadIdx.x] = r_delta[which];
        }
    };
    load(0);
    load(1);
    store(0, 0);
    load(0);
    wa_arrived(f);
    __syncthreads();
    const int row_at = c * PITCH + 8 * h * (int)sizeof(T), col_at = wa_col_offset<T>(lane, PITCH);
    const int from = have ? j - a.right : 0x7fffffff, to = j < a.sinks ? 0x7fffffff : j + a.left;
    int now = 0, tile = 0, before = 2;                                                 // buffer of tile k, the tile, the buffer of tile k - 1
    bool seen_before = false;
    v16f d;                                                                            // second: dout . v of the tile before
    auto step = [&](int k, auto parity) {
        constexpr int odd = decltype(parity)::value;                                   // k & 1; tile k + 1 is in the other registers
        const int next = now == 2 ? 0 : now + 1;
        store(next, odd ^ 1);                                                          // (tile k - 2's: last read a step ago, before the barrier)
        load(odd ^ 1);
        const int p0 = a.q_start + i_lo + tile * BQ, p1 = p0 + BQ - 1;
        const bool seen = k < steps && jw0 < n && p1 >= jw0 - a.right && (p0 <= jw1 + a.left || jw0 < a.sinks);
        if (!second) {
            if (seen) {
                v16f s;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = 0.0f;
                {
                    WaStream<T, NS> rows;
                    const auto read = [&](int x) { return wa_row<T>(s_q[now] + row_at, x); };
                    rows.prime(read);
                    rows.run(read, [&](int x, const vec &y) { s = LpTraits<T>::mfma(y, f[x], s); });
                }
                WaStream<T, 2 * NT> cols;
                const auto read_g = [&](int x) { return wa_col<T, PITCH>(s_g[AHEAD ? odd : now] + col_at, 16 * (x / NT), x % NT); };
                cols.prime(read_g);
                if (!(jw1 < n && p0 >= jw1 - a.right && (p1 <= jw0 + a.left || jw1 < a.sinks))) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int p = p0 + 8 * (r >> 2) + 4 * h + (r & 3);
                        s[r] = p >= from && p <= to ? s[r] : -INFINITY;
                    }
                }
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f4 lse = *reinterpret_cast<const f4 *>(&s_lse[now][2 * r + 4 * h]);
                    f4 pr;
#pragma unroll
                    for (int e = 0; e < 4; ++e) pr[e] = s[r + e] = __builtin_amdgcn_exp2f(fmaf(s[r + e], a.c, -lse[e]));
                    *reinterpret_cast<f4 *>(s_p[odd][keys][r >> 2][lane]) = pr;
                }
                vec pr;
                cols.run(read_g, [&](int x, const vec &y) {
                    if (x % NT == 0) pr = wa_pack<T>(s, x / NT);
                    acc[x % NT] = LpTraits<T>::mfma(y, pr, acc[x % NT]);
                });
            }
        } else {
            auto product = [&](const unsigned char *g) {
#pragma unroll
                for (int r = 0; r < 16; ++r) d[r] = 0.0f;
                WaStream<T, NS> rows;
                const auto read = [&](int x) { return wa_row<T>(g + row_at, x); };
                rows.prime(read);
                rows.run(read, [&](int x, const vec &y) { d = LpTraits<T>::mfma(y, f[x], d); });
            };
            if (seen_before) {
                if constexpr (!AHEAD) product(s_g[before]);
                WaStream<T, 2 * NT> cols;
                const auto read_q = [&](int x) { return wa_col<T, PITCH>(s_q[before] + col_at, 16 * (x / NT), x % NT); };
                cols.prime(read_q);
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f4 delta = *reinterpret_cast<const f4 *>(&s_delta[before][2 * r + 4 * h]), pr = *reinterpret_cast<const f4 *>(s_p[odd ^ 1][keys][r >> 2][lane]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[r + e] = pr[e] * (d[r + e] - delta[e]);
                }
                vec ds;
                cols.run(read_q, [&](int x, const vec &y) {
                    if (x % NT == 0) ds = wa_pack<T>(d, x / NT);
                    acc[x % NT] = LpTraits<T>::mfma(y, ds, acc[x % NT]);
                });
            }
            if constexpr (AHEAD)
                if (seen) product(s_g[odd]);
            seen_before = seen;
        }
        __syncthreads();
        before = now;
        now = next;
        if (++tile == tiles) tile = 0;
    };
    for (int k = 0; k <= steps; k += 2) {
        step(k, WaInt<0>{});
        if (k + 1 <= steps) step(k + 1, WaInt<1>{});
    }
    if (j >= a.Tk) return;
    const float f_out = second ? a.scale : 1.0f;
    if (slice) {
        float *out = a.partial + (((((int64_t)(j0 / kWaKeys) * a.splits + part) * bh + hkb) * 2 + (second ? 0 : 1)) * kWaKeys + (j - j0)) * a.D;
        wa_store_rows<float, NT, false>(acc, f_out, out, h, a.D);
    } else {
        const WaTensor &o = second ? a.dk : a.dv;
        wa_store_rows<T, NT, VEC>(acc, f_out, static_cast<T *>(o.p) + b * o.sb + (int64_t)j * o.st + hk * o.sh, h, a.D);
    }
}

// the slices' sums of the tiles with sinks, added in order (4 us, a launch)
template <typename T>
__global__ __launch_bounds__(kWaThreads) void k_window_attn_join(WaArgs a) {
    const uint32_t bh = (uint32_t)a.B * a.Hk, hkb = blockIdx.y, tile = blockIdx.z;
    const int hk = (int)(hkb % a.Hk), b = (int)(hkb / a.Hk);
    const int64_t size = 2ll * kWaKeys * a.D, stride = (int64_t)bh * size;
    const float *src = a.partial + ((int64_t)tile * a.splits * bh + hkb) * size;
    for (int64_t e = blockIdx.x * kWaThreads + threadIdx.x; e < size; e += (int64_t)gridDim.x * kWaThreads) {
        const int which = e >= (int64_t)kWaKeys * a.D, r = (int)(e / a.D) - which * kWaKeys, d = (int)(e % a.D);
        const int64_t j = (int64_t)tile * kWaKeys + r;
        if (j >= a.Tk) continue;
        float sum = 0.0f;
        uint32_t s = 0;
        for (; s + 8 <= a.splits; s += 8) {                    // (eight loads in flight; the order of the sum stays)
            float v[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) v[x] = src[(s + x) * stride + e];
#pragma unroll
            for (int x = 0; x < 8; ++x) sum += v[x];
        }
        for (; s < a.splits; ++s) sum += src[s * stride + e];
        const WaTensor &t = which ? a.dv : a.dk;
        static_cast<T *>(t.p)[b * t.sb + j * t.st + hk * t.sh + d] = (T)sum;
    }
}

// Slices of a tile with sinks: each about the queries that a tile without sinks has, so that no workgroup ends long after the others; at least 256, 64 slices at most
// (13 000 queries, window 1 024, 4 sinks: 155 us, whole 1 515; a padded batch of 6 x 777, window 251, 3 sinks: 29 us, whole 49).  All tiles' slices together: 4 096 at most, five
// times what the chip holds at once, so that their partial sums end at 256 MB (128 features) however many sinks and heads there are (whole backward pass, bf16: 13 000 x 8 heads x 128, window 129, 1 000
// sinks 506 us, without that end 597; 64 x 4 096 x 8 x 64, window 128, 4 sinks 1 350 and 1 417).
constexpr uint32_t kWaMostSlices = 4096;
static uint32_t wa_splits(const WaArgs &a) {
    const int64_t ordinary = (int64_t)kWaKeys + a.left + a.right, each = ordinary > 256 ? ordinary : 256, want = ((int64_t)a.Tq + each - 1) / each;
    const uint64_t tiles = (uint64_t)a.sink_tiles * a.B * a.Hk, room = kWaMostSlices / (tiles ? tiles : 1), most = room < 64 ? room : 64;
    return (uint32_t)(want < 1 || most < 1 ? 1 : ((uint64_t)want > most ? most : want));
}
static uint32_t wa_sink_tiles(const WaArgs &a) {
    // a window that reaches every query from its first key makes the sinks ordinary keys
    if (a.sinks == 0 || (int64_t)a.left + 1 >= (int64_t)a.q_start + a.Tq) return 0;
    return (uint32_t)((a.sinks + kWaKeys - 1) / kWaKeys);
}

template <typename T, int DP>
static void wa_backward_launch(const WaArgs &a, bool vec, uint32_t gq, uint32_t gk, hipStream_t st) {
    if (gq) vec ? k_window_attn_dq<T, DP, true><<<gq, kWaThreads, 0, st>>>(a) : k_window_attn_dq<T, DP, false><<<gq, kWaThreads, 0, st>>>(a);
    if (!gk) return;
    vec ? k_window_attn_dkv<T, DP, true><<<gk, kWaThreads, 0, st>>>(a) : k_window_attn_dkv<T, DP, false><<<gk, kWaThreads, 0, st>>>(a);
    if (a.sink_tiles) k_window_attn_join<T><<<dim3(div_up(2 * kWaKeys * a.D, kWaThreads), (uint32_t)(a.B * a.Hk), a.sink_tiles), kWaThreads, 0, st>>>(a);
}
template <typename T>
static void wa_backward(const WaArgs &a, bool vec, uint32_t gq, uint32_t gk, hipStream_t st) {
    if (a.D <= 32) wa_backward_launch<T, 32>(a, vec, gq, gk, st);
    else if (a.D <= 64) wa_backward_launch<T, 64>(a, vec, gq, gk, st);
    else wa_backward_launch<T, 128>(a, vec, gq, gk, st);
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
    a.splits = a.sink_tiles ? wa_splits(a) : 1;
    if (a.splits == 1) a.sink_tiles = 0;                       // whole tiles write their gradients themselves
}

GFPP_API unsigned long long gfpp_window_attn_backward_scratch_floats(uint32_t B, uint32_t Tq, uint32_t Tk, uint32_t Hq, uint32_t Hk, uint32_t D, int32_t left,
                                                                     int32_t right, int32_t sinks, int32_t q_start, int) {
    if (Hk == 0 || Tq > (1u << 29) || Tk > (1u << 29) || sinks < 0 || left < 0 || right < 0) return 0;
    WaArgs a{};
    a.B = (int)B;
    a.Hk = (int)Hk;
    a.Tq = (int)Tq;
    a.Tk = (int)Tk;
    a.D = (int)D;
    a.left = left < (1 << 29) ? left : 1 << 29;                // (as wa_arguments has them)
    a.right = right < (1 << 29) ? right : 1 << 29;
    a.sinks = sinks < (int)Tk ? sinks : (int)Tk;
    a.q_start = q_start;
    wa_bwd_setup(a);
    return (unsigned long long)B * Hq * Tq + (unsigned long long)a.sink_tiles * a.splits * B * Hk * 2 * kWaKeys * D;
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
    const uint32_t q_tiles = div_up(Tq, kWaRows), k_tiles = div_up(Tk, (uint32_t)kWaKeys) - a.sink_tiles + a.sink_tiles * a.splits;
    WA_REQUIRE(grid_fits(kWaThreads, q_tiles, Hq, B) && grid_fits(kWaThreads, k_tiles, Hk, B));
    const uint32_t bh = B * Hk, gq = q_tiles * Hq * B, gk = k_tiles * bh;
    const size_t size = dtype == GFPP_F32 ? 4 : 2;
    bool vec = (uintptr_t)a.low % 16 == 0;
    for (const WaTensor *t : {&a.q, &a.k, &a.v, &a.o, &a.dout, &a.dq, &a.dk, &a.dv}) vec = vec && wa_vectors(*t, a.D, size);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GFPP_F32) wa_backward<float>(a, vec, gq, gk, st);
    else if (dtype == GFPP_F16) wa_backward<_Float16>(a, vec, gq, gk, st);
    else wa_backward<__bf16>(a, vec, gq, gk, st);
    return check_launch(what);
}
