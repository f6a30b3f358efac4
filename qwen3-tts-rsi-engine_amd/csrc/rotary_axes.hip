// Rotary positions with several axes: query and key rows of tokens that have a position on each
// axis (reference: the talker's rotary_emb with mrope_section, continuous.py:193,
// packed_attention.py:66-69).
//
//   angle_i = positions[axis(i)] * frequency_i,  i < half
//   y[i] = x[i] c_i - x[i + half] s_i,  y[i + half] = x[i + half] c_i + x[i] s_i
//
// One workgroup takes the rows of a few tokens, queries and keys: its threads form the tokens'
// cosines and sines once, in LDS, for all heads.  The angle is a number of turns in 64 bits, and
// only what is left after whole turns goes on to sincospi in 32: an angle kept in 32 bits would
// be off by radians at far positions.  What that rounding takes off the angle (below 2^-25) is put back by
// cos(a + r) = cos a - r sin a, sin(a + r) = sin a + r cos a: without it a cosine near zero has 24 bits of 1 and not of
// itself (rms error of float32 rows 3.9e-8 of their rms, with it 2.9e-8, in the same time).  Products and sums are
// float32, and each element is rounded once, to nearest even.
// Bound by HBM (every row read and written once: 16396 tokens of 32 heads of 128, 269 MB, 57 us, 4.7
// TB/s, and 49 where the outputs' memory is in the caches; one row of a thread on its way at a time 65, four
// 57), by the launch for a decode step (64 tokens 3.5 us); the first rows are on their way while the
// angles are formed.  Rows are loaded with the non-temporal policy and stored with the plain one: whoever
// reads the outputs next finds more of them in the caches (with a copy of both outputs behind it 97 us;
// plain loads 120, non-temporal stores too 109).
#include "paged_index.hpp"
#include "q3t_common.hpp"

#include <type_traits>

namespace q3t {
namespace axes {

constexpr int kThreads = 256;
constexpr int kAngles = 512;  // cosines and sines of a workgroup (4 KiB of LDS)
constexpr int kFlight = 2;    // a thread's items whose rows are on their way at once

struct Rows {
    const char *x;
    char *y;
    int64_t x_sb, x_ss, x_sh, y_sb, y_ss, y_sh;  // bytes
};
struct Params {
    Rows q, k;
    const int64_t *positions;
    const double *turns;
    int64_t p_sa, p_sb, p_ss;
    uint32_t rows;            // batch * tokens
    uint32_t group;           // tokens of a workgroup
    uint32_t half, q_heads, heads, units, rotated;  // units of a row: `rotated` pairs, then copies
    uint32_t tail;            // first element that is copied
    Divisor by_tokens, by_half, by_units, by_heads;
    uint32_t limit[4];        // first frequency behind each axis's section, or axes * section
    uint32_t axes, interleaved;
    float scaling;
};

template <typename T> struct Type;
template <> struct Type<float> {
    static constexpr int vec = 4;
    static Q3T_DEVICE void widen(const U4 &v, float (&x)[4]) { __builtin_memcpy(x, &v, 16); }
    static Q3T_DEVICE U4 narrow(const float (&x)[4]) { U4 v; __builtin_memcpy(&v, x, 16); return v; }
    static Q3T_DEVICE float one(float x) { return x; }
};
template <> struct Type<__bf16> {
    static constexpr int vec = 8;
    static Q3T_DEVICE void widen(const U4 &v, float (&x)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = bf16_lo(w[i]);
            x[2 * i + 1] = bf16_hi(w[i]);
        }
    }
    static Q3T_DEVICE U4 narrow(const float (&x)[8]) {
        return U4{cvt_pk_bf16_canon(x[0], x[1]), cvt_pk_bf16_canon(x[2], x[3]), cvt_pk_bf16_canon(x[4], x[5]),
                  cvt_pk_bf16_canon(x[6], x[7])};
    }
    static Q3T_DEVICE __bf16 one(float x) { return __builtin_bit_cast(__bf16, (uint16_t)float_to_bf16(x)); }
};
template <> struct Type<_Float16> {
    static constexpr int vec = 8;
    typedef _Float16 halves_t __attribute__((ext_vector_type(8)));
    static Q3T_DEVICE void widen(const U4 &v, float (&x)[8]) {
        const halves_t h = __builtin_bit_cast(halves_t, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
    }
    static Q3T_DEVICE U4 narrow(const float (&x)[8]) {
        halves_t h;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = (_Float16)x[i];
        return __builtin_bit_cast(U4, h);
    }
    static Q3T_DEVICE _Float16 one(float x) { return (_Float16)x; }
};

// VEC: 16-byte vectors (row pointers, strides and both halves are multiples of one); else single
// elements.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) rotary_axes_kernel(Params p) {
    constexpr int V = VEC ? Type<T>::vec : 1;
    __shared__ float cosv[kAngles], sinv[kAngles];
    const uint32_t first = blockIdx.x * p.group;
    const uint32_t count = min(p.group, p.rows - first);

    // item -> (token, head, unit) of the workgroup, units fastest
    struct Item {
        const char *x;
        char *y;
        uint32_t unit, token;
    };
    auto item_of = [&](uint32_t i) {
        const uint32_t row = divide(i, p.by_units), token = divide(row, p.by_heads);
        const uint32_t head = row - token * p.heads;
        const uint32_t b = divide(first + token, p.by_tokens), s = first + token - b * p.by_tokens.d;
        Item it;
        it.unit = i - row * p.units;
        it.token = token;
        const bool is_key = head >= p.q_heads;
        const Rows &r = is_key ? p.k : p.q;
        const uint32_t h = is_key ? head - p.q_heads : head;
        const uint32_t element = it.unit < p.rotated ? it.unit * V : p.tail + (it.unit - p.rotated) * V;
        it.x = r.x + b * r.x_sb + s * r.x_ss + h * r.x_sh + element * sizeof(T);
        it.y = r.y + b * r.y_sb + s * r.y_ss + h * r.y_sh + element * sizeof(T);
        return it;
    };
    typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
    typedef std::conditional_t<VEC, U4, T> Word;
    auto load_word = [](const char *x) {
        if constexpr (VEC) {
            const u32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(x));
            return U4{v[0], v[1], v[2], v[3]};
        } else {
            return *reinterpret_cast<const T *>(x);
        }
    };
    const uint32_t items = count * p.heads * p.units, apart = p.half * sizeof(T);
    Item it[kFlight];
    Word a[kFlight], b[kFlight];
    auto load = [&](uint32_t first_item) {
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            const uint32_t i = first_item + j * kThreads;
            if (i >= items) break;
            it[j] = item_of(i);
            a[j] = load_word(it[j].x);
            if (it[j].unit < p.rotated) b[j] = load_word(it[j].x + apart);
        }
    };
    load(threadIdx.x);

    for (uint32_t n = threadIdx.x; n < count * p.half; n += kThreads) {
        const uint32_t token = divide(n, p.by_half), f = n - token * p.half;
        uint32_t axis = 0;
        if (p.interleaved) {
            const uint32_t at = f % p.axes;
            if (f < p.limit[at]) axis = at;
        } else {
            while (axis + 1 < p.axes && f >= p.limit[axis]) ++axis;
        }
        const uint32_t rb = divide(first + token, p.by_tokens), s = first + token - rb * p.by_tokens.d;
        const double turn = (double)p.positions[axis * p.p_sa + rb * p.p_sb + s * p.p_ss] * p.turns[f];
        const double part = 2.0 * (turn - rint(turn));  // of half turns
        const float nearest = (float)part, rest = 3.14159274f * (float)(part - nearest);
        float sn, cs;
        sincospif(nearest, &sn, &cs);
        cosv[n] = __builtin_fmaf(-rest, sn, cs) * p.scaling;
        sinv[n] = __builtin_fmaf(rest, cs, sn) * p.scaling;
    }
    __syncthreads();

    for (uint32_t first_item = threadIdx.x; first_item < items; first_item += kFlight * kThreads) {
        if (first_item != threadIdx.x) load(first_item);
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            if (first_item + j * kThreads >= items) break;
            if (it[j].unit < p.rotated) {
                const uint32_t at = it[j].token * p.half + it[j].unit * V;
                if constexpr (VEC) {
                    float x1[V], x2[V], y1[V], y2[V];
                    Type<T>::widen(a[j], x1);
                    Type<T>::widen(b[j], x2);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        y1[e] = x1[e] * cosv[at + e] - x2[e] * sinv[at + e];
                        y2[e] = x2[e] * cosv[at + e] + x1[e] * sinv[at + e];
                    }
                    *reinterpret_cast<U4 *>(it[j].y) = Type<T>::narrow(y1);
                    *reinterpret_cast<U4 *>(it[j].y + apart) = Type<T>::narrow(y2);
                } else {
                    const float x1 = (float)a[j], x2 = (float)b[j];
                    *reinterpret_cast<T *>(it[j].y) = Type<T>::one(x1 * cosv[at] - x2 * sinv[at]);
                    *reinterpret_cast<T *>(it[j].y + apart) = Type<T>::one(x2 * cosv[at] + x1 * sinv[at]);
                }
            } else {
                *reinterpret_cast<Word *>(it[j].y) = a[j];
            }
        }
    }
}

template <typename T>
static void launch(const Params &p, bool vec, uint32_t blocks, hipStream_t stream) {
    if (vec) hipLaunchKernelGGL((rotary_axes_kernel<T, true>), dim3(blocks), dim3(kThreads), 0, stream, p);
    else hipLaunchKernelGGL((rotary_axes_kernel<T, false>), dim3(blocks), dim3(kThreads), 0, stream, p);
}

}  // namespace axes
}  // namespace q3t

using namespace q3t;

extern "C" int q3t_rotary_axes(const q3t_rotary_axes_args *a, void *stream) {
    using namespace axes;
    if (!a) return Q3T_EINVAL;
    if (a->batch < 0 || a->tokens < 0 || a->q_heads < 1 || a->k_heads < 0 || a->width < 2 || a->axes < 1 || a->axes > 4)
        return Q3T_EINVAL;
    if (a->dtype != Q3T_BF16 && a->dtype != Q3T_F16 && a->dtype != Q3T_F32) return Q3T_EUNSUPPORTED;
    int64_t half = 0;
    for (int64_t i = 0; i < a->axes; ++i) {
        if (a->sections[i] < 0 || a->sections[i] > a->width) return Q3T_EINVAL;
        half += a->sections[i];
    }
    if (half < 1 || 2 * half > a->width) return Q3T_EINVAL;
    if (half > kAngles || a->width > 1 << 16 || a->q_heads > 1 << 16 || a->k_heads > 1 << 16) return Q3T_EUNSUPPORTED;
    if (a->batch == 0 || a->tokens == 0) return Q3T_OK;
    if (a->batch > INT32_MAX / a->tokens) return Q3T_EUNSUPPORTED;
    const int64_t rows = a->batch * a->tokens;
    const bool keys = a->k_heads > 0;
    if (!a->turns || !a->positions || !a->query || !a->q_out || (keys && (!a->key || !a->k_out))) return Q3T_EINVAL;

    const int64_t es = a->dtype == Q3T_F32 ? 4 : 2, vec = 16 / es;
    auto bytes = [&](const void *x, void *y, int64_t xb, int64_t xs, int64_t xh, int64_t yb, int64_t ys, int64_t yh) {
        return Rows{(const char *)x, (char *)y, xb * es, xs * es, xh * es, yb * es, ys * es, yh * es};
    };
    Params p = {};
    p.q = bytes(a->query, a->q_out, a->q_stride_b, a->q_stride_s, a->q_stride_h, a->qo_stride_b, a->qo_stride_s, a->qo_stride_h);
    p.k = p.q;
    if (keys) p.k = bytes(a->key, a->k_out, a->k_stride_b, a->k_stride_s, a->k_stride_h, a->ko_stride_b, a->ko_stride_s, a->ko_stride_h);
    auto whole = [&](const Rows &r, int64_t unit) {
        return aligned(r.x, unit) && aligned(r.y, unit) &&
               ((r.x_sb | r.x_ss | r.x_sh | r.y_sb | r.y_ss | r.y_sh) & (unit - 1)) == 0;
    };
    if (!whole(p.q, es) || !whole(p.k, es) || !aligned(a->positions, 8) || !aligned(a->turns, 8)) return Q3T_EINVAL;
    const bool vectors = whole(p.q, 16) && whole(p.k, 16) && half % vec == 0 && a->width % vec == 0;
    const int64_t v = vectors ? vec : 1;
    p.positions = a->positions;
    p.turns = a->turns;
    p.p_sa = a->p_stride_a; p.p_sb = a->p_stride_b; p.p_ss = a->p_stride_s;
    p.rows = (uint32_t)rows;
    p.half = (uint32_t)half;
    p.q_heads = (uint32_t)a->q_heads;
    p.heads = (uint32_t)(a->q_heads + a->k_heads);
    p.rotated = (uint32_t)(half / v);
    p.tail = (uint32_t)(2 * half);
    // what is not rotated needs no copy where every output is its input
    auto same = [](const Rows &r) { return r.x == r.y && r.x_sb == r.y_sb && r.x_ss == r.y_ss && r.x_sh == r.y_sh; };
    const bool in_place = same(p.q) && same(p.k);
    p.units = p.rotated + (in_place ? 0u : (uint32_t)((a->width - 2 * half) / v));
    p.axes = (uint32_t)a->axes;
    p.interleaved = a->interleaved != 0;
    p.scaling = a->scaling;
    uint32_t end = 0;
    for (int64_t i = 0; i < a->axes; ++i) {
        end += (uint32_t)a->sections[i];
        p.limit[i] = p.interleaved ? (uint32_t)(a->axes * a->sections[i]) : end;
    }
    // as many tokens as the angles' LDS holds, but fewer where that leaves the card short of workgroups
    int64_t group = kAngles / half;
    while (group > 1 && rows / group < 2048) group /= 2;
    // items of a workgroup, and threads of the launch, stay below 2^31 and 2^32
    while (group > 1 && group * p.heads > INT32_MAX / 2 / p.units) group /= 2;
    if (p.heads > INT32_MAX / 2 / p.units) return Q3T_EUNSUPPORTED;
    p.group = (uint32_t)group;
    p.by_tokens = divisor((uint32_t)a->tokens);
    p.by_half = divisor(p.half);
    p.by_units = divisor(p.units);
    p.by_heads = divisor(p.heads);
    const uint32_t blocks = (uint32_t)((rows + group - 1) / group);
    if ((uint64_t)blocks * kThreads >= (uint64_t)1 << 32) return Q3T_EUNSUPPORTED;
    if (a->dtype == Q3T_F32) launch<float>(p, vectors, blocks, (hipStream_t)stream);
    else if (a->dtype == Q3T_BF16) launch<__bf16>(p, vectors, blocks, (hipStream_t)stream);
    else launch<_Float16>(p, vectors, blocks, (hipStream_t)stream);
    return launch_status();
}
