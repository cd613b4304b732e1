// rotary.hip -- rotary positions over several axes (gfx950): pairs of a head's features turned by position x frequency, forward and (by the opposite angle) backward.
//
//   pair i of axis a(i):  t = position[a(i)] frequency[i],  (u, v) -> (u cos t - v sin t, u sin t + v cos t)
//
// A pair is (i, i + P) of the head's first 2 P features, or (2 i, 2 i + 1) when interleaved; the features behind the first 2 P pass through.  The angle is taken
// in 64 bits and reduced to a fraction of a turn there -- a 32-bit product of a position of 10^6 and a frequency is off by a sixteenth of a radian -- and only the
// fraction is narrowed, so that cosine and sine are good to fp32's last bits at any position.
//
// Bound by memory: every element is read and written once.  A workgroup takes a few tokens, computes their cosines and sines once into LDS (they are shared by all
// heads of both tensors: queries and keys go through in ONE launch) and streams the heads in 16-byte vectors.
// Measured: 16 384 tokens x (16 + 4) heads x 128 bf16: 34 us (168 MB, 4.9 TB/s; one element at a time, which is what pairs that do not fill 16-byte vectors take: 87); 3 x 1 023 x 9 x 40 fp32: 5.4 us (8.8 MB); 8 tokens: 3.4 us, a launch.
#include "gfpp_common.h"

namespace gfpp {

template <typename T>
struct RoVec;
template <> struct RoVec<float> { typedef float v __attribute__((ext_vector_type(4))); };
template <> struct RoVec<_Float16> { typedef _Float16 v __attribute__((ext_vector_type(8))); };
template <> struct RoVec<__bf16> { typedef __bf16 v __attribute__((ext_vector_type(8))); };

constexpr int kRoThreads = 256, kRoMaxAxes = 4, kRoAngles = 512;

struct RoTensor {
    const void *x;
    void *y;                       // [B][T][heads][D] contiguous
    int64_t sb, st, sh;            // x's strides in elements
    uint32_t heads;
};
struct RoArgs {
    RoTensor t[2];
    const void *pos;               // [B or 1][T][axes]
    const double *freq;            // [P] radians per position
    int64_t pos_sb;                // 0: one set of positions for every sequence
    uint32_t B, T, D, P, axes, tokens_wg;
    uint32_t first[kRoMaxAxes];    // first pair of every axis
    int pos_type;                  // 0 int32, 1 int64, 2 float32
    float sign;
};

template <typename T, bool VEC, bool INTER>
__global__ __launch_bounds__(kRoThreads) void k_rotary(RoArgs a) {
    __shared__ float s_cos[kRoAngles], s_sin[kRoAngles];
    typedef typename RoVec<T>::v vec;
    constexpr uint32_t V = VEC ? 16 / sizeof(T) : 1;
    const uint64_t tokens = (uint64_t)a.B * a.T, tok0 = (uint64_t)blockIdx.x * a.tokens_wg;
    const uint32_t n_tok = (uint32_t)(tokens - tok0 < a.tokens_wg ? tokens - tok0 : a.tokens_wg);
    for (uint32_t i = threadIdx.x; i < n_tok * a.P; i += kRoThreads) {
        const uint32_t pr = i % a.P;
        const uint64_t tok = tok0 + i / a.P;
        uint32_t ax = 0;
#pragma unroll
        for (uint32_t k = 1; k < kRoMaxAxes; ++k)
            if (k < a.axes && pr >= a.first[k]) ax = k;
        const uint64_t at = (tok / a.T) * (uint64_t)a.pos_sb + (tok % a.T) * a.axes + ax;
        double p;
        if (a.pos_type == 0) p = (double)static_cast<const int32_t *>(a.pos)[at];
        else if (a.pos_type == 1) p = (double)static_cast<const int64_t *>(a.pos)[at];
        else p = (double)static_cast<const float *>(a.pos)[at];
        const double turns = p * a.freq[pr] * 0.15915494309189533577;      // 1 / (2 pi)
        float sn, cs;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
        s_cos[i] = cs;
        s_sin[i] = sn * a.sign;
    }
    __syncthreads();
    // work items: (token, head of either tensor, chunk).  A chunk is V pairs (both their vectors, or the one vector that holds V / 2 interleaved pairs), or V
    // features of the part that passes through
    const uint32_t turned = INTER ? (VEC ? 2 * a.P / V : a.P) : a.P / V, chunks = turned + (a.D - 2 * a.P) / V, heads = a.t[0].heads + a.t[1].heads;
    const uint32_t items = n_tok * heads * chunks;
    for (uint32_t i = threadIdx.x; i < items; i += kRoThreads) {
        const uint32_t c = i % chunks, r = i / chunks;
        uint32_t h = r % heads;
        const uint32_t lt = r / heads;
        const uint64_t tok = tok0 + lt;
        const RoTensor &t = h < a.t[0].heads ? a.t[0] : a.t[1];
        if (h >= a.t[0].heads) h -= a.t[0].heads;
        const T *x = static_cast<const T *>(t.x) + (int64_t)(tok / a.T) * t.sb + (int64_t)(tok % a.T) * t.st + (int64_t)h * t.sh;
        T *y = static_cast<T *>(t.y) + (tok * t.heads + h) * a.D;
        if (c >= turned) {
            const uint32_t at = 2 * a.P + (c - turned) * V;
            if constexpr (VEC) *reinterpret_cast<vec *>(y + at) = *reinterpret_cast<const vec *>(x + at);
            else y[at] = x[at];
            continue;
        }
        const float *cs = s_cos + lt * a.P, *sn = s_sin + lt * a.P;
        if constexpr (!VEC) {
            const uint32_t i0 = INTER ? 2 * c : c, i1 = INTER ? 2 * c + 1 : c + a.P;
            const float u = (float)x[i0], v = (float)x[i1];
            y[i0] = (T)(u * cs[c] - v * sn[c]);
            y[i1] = (T)(u * sn[c] + v * cs[c]);
        } else if constexpr (INTER) {
            const uint32_t at = c * V;
            vec d = *reinterpret_cast<const vec *>(x + at);
#pragma unroll
            for (uint32_t e = 0; e < V; e += 2) {
                const float u = (float)d[e], v = (float)d[e + 1], cc = cs[(at + e) / 2], ss = sn[(at + e) / 2];
                d[e] = (T)(u * cc - v * ss);
                d[e + 1] = (T)(u * ss + v * cc);
            }
            *reinterpret_cast<vec *>(y + at) = d;
        } else {
            const uint32_t at = c * V;
            vec d0 = *reinterpret_cast<const vec *>(x + at), d1 = *reinterpret_cast<const vec *>(x + a.P + at);
#pragma unroll
            for (uint32_t e = 0; e < V; ++e) {
                const float u = (float)d0[e], v = (float)d1[e], cc = cs[at + e], ss = sn[at + e];
                d0[e] = (T)(u * cc - v * ss);
                d1[e] = (T)(u * ss + v * cc);
            }
            *reinterpret_cast<vec *>(y + at) = d0;
            *reinterpret_cast<vec *>(y + a.P + at) = d1;
        }
    }
}

template <typename T>
static void ro_launch(const RoArgs &a, bool vec, bool inter, uint32_t grid, hipStream_t st) {
    if (vec) inter ? k_rotary<T, true, true><<<grid, kRoThreads, 0, st>>>(a) : k_rotary<T, true, false><<<grid, kRoThreads, 0, st>>>(a);
    else inter ? k_rotary<T, false, true><<<grid, kRoThreads, 0, st>>>(a) : k_rotary<T, false, false><<<grid, kRoThreads, 0, st>>>(a);
}

}  // namespace gfpp

using namespace gfpp;

#define RO_REQUIRE(cond)                                                       \
    do {                                                                       \
        if (!(cond)) {                                                         \
            set_error("gfpp_rotary: invalid argument (%s)", #cond);            \
            return GFPP_EINVAL;                                                \
        }                                                                      \
    } while (0)

GFPP_API int gfpp_rotary(const void *x0, const int64_t *x0_strides, uint32_t heads0, void *y0, const void *x1, const int64_t *x1_strides, uint32_t heads1, void *y1,
                         const void *positions, int position_type, int64_t position_stride, const double *frequencies, const uint32_t *sections, uint32_t axes,
                         uint32_t B, uint32_t T, uint32_t D, int interleaved, int backward, int dtype, gfpp_stream_t stream) {
    RO_REQUIRE(dtype == GFPP_F32 || dtype == GFPP_F16 || dtype == GFPP_BF16);
    RO_REQUIRE(axes >= 1 && axes <= kRoMaxAxes && sections);
    RO_REQUIRE(position_type >= 0 && position_type <= 2 && position_stride >= 0);
    RoArgs a{};
    for (uint32_t k = 0; k < axes; ++k) {
        a.first[k] = a.P;
        RO_REQUIRE(sections[k] <= kRoAngles);
        a.P += sections[k];
    }
    RO_REQUIRE(a.P >= 1 && a.P <= kRoAngles && 2 * a.P <= D);
    RO_REQUIRE(D <= 65536 && heads0 <= 65536 && heads1 <= 65536 && ((uint64_t)heads0 + heads1) * D <= (1u << 26));      // (a workgroup's items: 32 bits)
    if ((uint64_t)B * T == 0 || heads0 + heads1 == 0) return 0;
    RO_REQUIRE(positions && frequencies);
    const size_t size = dtype == GFPP_F32 ? 4 : 2;
    const uint32_t V = (uint32_t)(16 / size);
    bool vec = interleaved ? (2 * a.P) % V == 0 : a.P % V == 0;
    vec = vec && D % V == 0;
    const void *xs[2] = {x0, x1};
    void *ys[2] = {y0, y1};
    const int64_t *ss[2] = {x0_strides, x1_strides};
    const uint32_t hs[2] = {heads0, heads1};
    for (int k = 0; k < 2; ++k) {
        a.t[k].heads = hs[k];
        if (!hs[k]) continue;
        RO_REQUIRE(xs[k] && ys[k] && ss[k]);
        a.t[k].x = xs[k];
        a.t[k].y = ys[k];
        a.t[k].sb = ss[k][0];
        a.t[k].st = ss[k][1];
        a.t[k].sh = ss[k][2];
        vec = vec && ((uintptr_t)xs[k] | (uintptr_t)ys[k]) % 16 == 0 && ((uint64_t)(ss[k][0] | ss[k][1] | ss[k][2]) * size) % 16 == 0;
    }
    a.pos = positions;
    a.freq = frequencies;
    a.pos_sb = position_stride;
    a.pos_type = position_type;
    a.B = B;
    a.T = T;
    a.D = D;
    a.axes = axes;
    a.sign = backward ? -1.0f : 1.0f;
    // tokens per workgroup: as many as fill the threads with angles (16 384 x 20 heads x 128: four 34 us, one 39), fewer while the chip is not full
    // (3 069 x 9 heads x 40: two 5.3 us, sixteen 9.3, one 7.0)
    const uint64_t tokens = (uint64_t)B * T;
    uint32_t tw = kRoThreads / a.P;
    tw = tw < 1 ? 1 : (tw > 16 ? 16 : tw);
    while (tw > 1 && (tokens + tw - 1) / tw < (uint64_t)cu_count() * 4) tw /= 2;
    a.tokens_wg = tw;
    const uint64_t grid = (tokens + tw - 1) / tw;
    RO_REQUIRE(grid_fits(kRoThreads, grid));
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GFPP_F32) ro_launch<float>(a, vec, interleaved != 0, (uint32_t)grid, st);
    else if (dtype == GFPP_F16) ro_launch<_Float16>(a, vec, interleaved != 0, (uint32_t)grid, st);
    else ro_launch<__bf16>(a, vec, interleaved != 0, (uint32_t)grid, st);
    return check_launch("gfpp_rotary");
}
