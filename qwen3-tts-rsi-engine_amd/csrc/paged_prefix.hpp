// Attention of a whole batch over the keys that all of its requests share.
//
// The query heads of all requests that read one KV head are the columns of the products S^T = K . Q^T and
// O^T += V^T . P^T, so a key and a value row is read once for all of them.  For each column the result is a softmax state,
// maximum, sum and weighted values, that the attention over the request's own keys takes in at its end.
//   * A workgroup of four waves takes one KV head, a block of CW * CT * 16 columns and a part of the keys.  CW waves
//     share a stage of keys in LDS, each with CT tiles of 16 columns in registers; the 4 / CW groups of waves take stages
//     in turn and are merged at the end.
//   * Stages come straight from memory to LDS, two ahead of the one that is multiplied.
//   * The weights go into the second product in one part of the type's own bits (half a step of 2^-8 in bf16, as the
//     prefill's weights have; float32 is multiplied as such): here, unlike in the attention of one request, the matrix
//     cores are the bound.  Their sum is that of the rounded weights, by a product with ones, so that what rounding takes
//     from a weight is taken from both.
#pragma once

#include "paged_kernel.hpp"

namespace q3t {
namespace paged {

struct PrefixParams {
    const char *q, *kp, *vp, *mask;
    const int32_t *table;               // request 0's row
    const int64_t *positions;
    float *states, *ml;                 // (part, KV head, column): D values; maximum and sum
    uint32_t q_sb, q_sh, kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st;  // 16 bytes
    uint32_t m_sb, m_st;                // elements
    int32_t mask_dtype;
    uint32_t heads, columns, blocks;    // KV heads; columns of one, and their blocks
    uint32_t parts, keys, chunk;        // parts of `chunk` keys
    uint32_t pages, ctx;
    Divisor by_page, by_group;
    float scale;                        // unmasked: times log2(e)
};

// The products of a wave's CT tiles of 16 columns with a stage's keys.
template <typename T, int D, int CT> struct Wide {
    typedef Shape<T, D> S;
    static constexpr int tiles = 2, keys = 32;  // of 16 keys; keys of a stage
    static constexpr float shift = Half<T>::shift, threshold = Half<T>::threshold;
    U4 q[CT][D / 32];
    f32x4_t acc[CT][D / 16], sum[CT];
    uint32_t key_at[D / 32], value_at[D / 16];

    Q3T_DEVICE void load_query(int ct, const char *row, int g, bool live) {
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) q[ct][kk] = live ? load16(row + (4 * kk + g) * 16) : U4{0u, 0u, 0u, 0u};
    }
    Q3T_DEVICE void clear() {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            sum[ct] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < D / 16; ++d) acc[ct][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
    }
    Q3T_DEVICE void rescale(int ct, float a) {
        sum[ct] *= a;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) acc[ct][d] *= a;
    }
    Q3T_DEVICE void place(int g, int c) {
        const int r = 4 * g + (c >> 2);
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) key_at[kk] = c * S::row + (((4 * kk + g) ^ S::key_swizzle(c)) & (S::chunks - 1)) * 16;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
            value_at[d] = (keys + r) * S::row + (((2 * d + ((c >> 1) & 1)) ^ S::value_swizzle(r)) & (S::chunks - 1)) * 16 + 8 * (c & 1);
    }
    Q3T_DEVICE void scores(uint32_t stage, f32x4_t (&s)[CT][tiles]) const {
#pragma unroll
        for (int t = 0; t < tiles; ++t) {
            U4 k[D / 32];
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk) k[kk] = lds_read16(key_at[kk] + stage + t * 16 * S::row);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) s[ct][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) s[ct][t] = Half<T>::scores(k[kk], q[ct][kk], s[ct][t]);
        }
    }
    // Rounded weights as an operand: inner index 8 g + j stands for key 4 g + j of the first tile (j < 4), and 4 g + j - 4 of the second.
    Q3T_DEVICE static U4 pack(const float (&w)[tiles][4]) {
        return U4{Half<T>::round2(w[0][0], w[0][1]), Half<T>::round2(w[0][2], w[0][3]), Half<T>::round2(w[1][0], w[1][1]),
                  Half<T>::round2(w[1][2], w[1][3])};
    }
    Q3T_DEVICE void sums(const float (&w)[CT][tiles][4]) {
        const uint32_t one = std::is_same<T, __bf16>::value ? 0x3f803f80u : 0x3c003c00u;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) sum[ct] = Half<T>::scores(U4{one, one, one, one}, pack(w[ct]), sum[ct]);
    }
    Q3T_DEVICE void values(uint32_t stage, const float (&w)[CT][tiles][4]) {
        U4 p[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) p[ct] = pack(w[ct]);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            const uint2 lo = lds_read_tr16(value_at[d] + stage), hi = lds_read_tr16(value_at[d] + stage + 16 * S::row);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) acc[ct][d] = Half<T>::scores(U4{lo.x, lo.y, hi.x, hi.y}, p[ct], acc[ct][d]);
        }
    }
    Q3T_DEVICE float total(int ct) const { return sum[ct][0]; }
    // element i of acc[][a] is that of dim:
    Q3T_DEVICE static int dim(int a, int i, int g) { return 16 * a + 4 * g + i; }
    Q3T_DEVICE static float element(uint32_t row, int r, int d) {
        const uint32_t at = row + (((d / 8) ^ S::value_swizzle(r)) & (S::chunks - 1)) * 16 + d % 8 * 2;
        return (float)*(Q3T_LDS const T *)(uintptr_t)at;
    }
    Q3T_DEVICE static bool finite(U4 x) {
        const uint32_t step = std::is_same<T, __bf16>::value ? 0x00800080u : 0x04000400u;  // carries an exponent of all ones into the sign
        const uint32_t any = ((x.x & 0x7fff7fffu) + step) | ((x.y & 0x7fff7fffu) + step) | ((x.z & 0x7fff7fffu) + step) | ((x.w & 0x7fff7fffu) + step);
        return !(any & 0x80008000u);
    }
    static Q3T_DEVICE float visible(float w) { return Half<T>::visible(w); }
};

template <int D, int CT> struct Wide<float, D, CT> {
    typedef Shape<float, D> S;
    static constexpr int tiles = 1, keys = 16;
    static constexpr float shift = 0.f, threshold = 8.f;
    f32x4_t q[CT][D / 16], acc[CT][D / 16];
    float sum[CT];
    uint32_t key_at[D / 16], value_at;

    Q3T_DEVICE void load_query(int ct, const char *row, int g, bool live) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
            q[ct][kk] = __builtin_bit_cast(f32x4_t, live ? load16(row + (4 * kk + g) * 16) : U4{0u, 0u, 0u, 0u});
    }
    Q3T_DEVICE void clear() {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            sum[ct] = 0.f;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) acc[ct][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
    }
    Q3T_DEVICE void rescale(int ct, float a) {
        sum[ct] *= a;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) acc[ct][d] *= a;
    }
    Q3T_DEVICE void place(int g, int c) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) key_at[kk] = c * S::row + ((4 * kk + g) ^ S::key_swizzle(c)) * 16;
        value_at = (keys + 4 * g) * S::row + c * 16;
    }
    Q3T_DEVICE void scores(uint32_t stage, f32x4_t (&s)[CT][tiles]) const {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) s[ct][0] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            const f32x4_t k = __builtin_bit_cast(f32x4_t, lds_read16(key_at[kk] + stage));
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) s[ct][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[e], q[ct][kk][e], s[ct][0], 0, 0, 0);
        }
    }
    Q3T_DEVICE void sums(const float (&w)[CT][tiles][4]) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) sum[ct] += (w[ct][0][0] + w[ct][0][1]) + (w[ct][0][2] + w[ct][0][3]);
    }
    Q3T_DEVICE void values(uint32_t stage, const float (&w)[CT][tiles][4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
                const f32x4_t v = __builtin_bit_cast(f32x4_t, lds_read16(value_at + stage + i * S::row + j * 256));
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct)
                        acc[ct][4 * j + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e], w[ct][0][i], acc[ct][4 * j + e], 0, 0, 0);
            }
    }
    Q3T_DEVICE float total(int ct) const {
        const float l = sum[ct] + xor16(sum[ct]);
        return l + xor32(l);
    }
    Q3T_DEVICE static int dim(int a, int i, int g) { return 64 * (a >> 2) + 16 * g + 4 * i + (a & 3); }
    Q3T_DEVICE static float element(uint32_t row, int, int d) { return *(Q3T_LDS const float *)(uintptr_t)(row + d * 4); }
    Q3T_DEVICE static bool finite(U4 x) {
        auto fine = [](uint32_t e) { return (e & 0x7fffffffu) < 0x7f800000u; };
        return fine(x.x) && fine(x.y) && fine(x.z) && fine(x.w);
    }
    static Q3T_DEVICE float visible(float w) { return w; }
};

constexpr uint32_t kWindow = 1024;  // page numbers that a workgroup holds

template <typename T, int D, int CW, int CT>
struct PrefixLds {
    typedef Wide<T, D, CT> X;
    static constexpr int groups = 4 / CW, stage = 2 * X::keys * Shape<T, D>::row, buffers = CW == 4 ? 3 : 2;
    union {
        alignas(1024) char ring[buffers][groups][stage];
        alignas(1024) float merge[groups == 1 ? 1 : 4][groups == 1 ? 1 : CT * kColumns][D];  // the groups' states
    };
    uint32_t ids[kWindow];
    float ml[4][CT * kColumns][2];
    uint32_t odd[buffers][4];  // whether a wave has found values that are not finite among its rows of a stage
    uint32_t least;            // keys that all live columns see
};

template <typename T, int D, bool MASK, int CW, int CT>
__global__ void __launch_bounds__(256, sizeof(PrefixLds<T, D, CW, CT>) <= 80 * 1024 ? 2 : 1)
prefix_kernel(PrefixParams p) {
    typedef Shape<T, D> S;
    typedef Wide<T, D, CT> X;
    typedef PrefixLds<T, D, CW, CT> L;
    constexpr int GROUPS = L::groups, SK = X::keys, TILES = X::tiles, AHEAD = L::buffers - 1;
    constexpr int LOADS = L::stage / 1024 / CW;  // of a wave's share of a stage: keys' rows in the first half, values' in the second
    constexpr uint32_t kAll = (uint32_t)((1ull << SK) - 1);
    static_assert(GROUPS == 1 || sizeof(float) * 4 * CT * kColumns * D <= sizeof(char) * L::buffers * GROUPS * L::stage, "");
    __shared__ L s;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int wave = (int)uniform(tid >> 6), cw = wave % CW, group = wave / CW;

    // all column blocks of a KV head's part follow each other on one XCD
    const uint32_t unit = blockIdx.x / (8 * p.blocks) * 8 + blockIdx.x % 8, block = blockIdx.x / 8 % p.blocks;
    if (unit >= p.heads * p.parts) return;
    const uint32_t part = unit / p.heads, head = unit - part * p.heads;
    const uint32_t begin = part * p.chunk, end = min(p.keys, begin + p.chunk);

    // ---- columns ----
    X x;
    uint32_t column[CT], seen[CT], request[CT];  // keys that a column sees (one that attends nothing: all of them, for no state)
    bool live[CT];
    if (tid == 0) s.least = p.keys;
    __syncthreads();
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        column[ct] = (block * CW * CT + cw * CT + ct) * kColumns + c;
        const bool real = column[ct] < p.columns;
        request[ct] = real ? divide(column[ct], p.by_group) : 0;
        const uint32_t i = column[ct] - request[ct] * p.by_group.d;
        const int64_t pos = real ? p.positions[request[ct]] : -1;
        live[ct] = pos >= 0 && pos < (int64_t)p.ctx;
        seen[ct] = live[ct] && pos < (int64_t)p.keys ? (uint32_t)pos + 1 : p.keys;
        if (seen[ct] < p.keys) atomicMin(&s.least, seen[ct]);
        x.load_query(ct, p.q + ((uint64_t)request[ct] * p.q_sb + (uint64_t)(head * p.by_group.d + (real ? i : 0)) * p.q_sh) * 16, g, real);
    }
    x.place(g, c);
    x.clear();
    __syncthreads();
    const uint32_t least = uniform(s.least);

    // ---- stages ----
    const uint32_t ring = uniform(lds_at(&s.ring[0][0][0]));
    uint32_t window = ~0u;  // first entry of the window
    auto buffer = [&](uint32_t n) { return ring + ((n % L::buffers) * GROUPS + group) * L::stage; };
    const uint32_t sets = (end - begin + GROUPS * SK - 1) / (GROUPS * SK);  // of a stage for every group
    // row and chunk of the lane's 16 bytes of load i of the wave's share
    auto row_of = [&](int i) { return ((cw * LOADS + i) * 64 + lane) / S::chunks % SK; };
    auto is_value = [&](int i) { return cw * LOADS + i >= L::stage / 2048; };
    auto load = [&](uint32_t n) {
        const uint32_t first = begin + n * GROUPS * SK, last = min(end, first + GROUPS * SK) - 1;
        const uint32_t from = divide(first, p.by_page), to = divide(last, p.by_page);
        if (window == ~0u || to - window >= kWindow) {  // (the same for all waves)
            if (window != ~0u) __syncthreads();
            window = from;
            const uint32_t entries = min(kWindow, divide(end - 1, p.by_page) - from + 1);
            for (uint32_t i = tid; i < entries; i += 256) s.ids[i] = (uint32_t)p.table[from + i];
            __syncthreads();
        }
        const uint32_t key0 = first + group * SK;
        const uint32_t mine = min(key0 + lane % SK, end - 1);
        const bool there = (uint32_t)lane < SK && key0 + lane < end && s.ids[divide(mine, p.by_page) - window] < p.pages;
        const uint32_t exists = (uint32_t)__builtin_amdgcn_ballot_w64(there);
        uint64_t at[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r = row_of(i);
            const uint32_t key = min(key0 + r, end - 1), entry = divide(key, p.by_page), row = key - entry * p.by_page.d;
            uint32_t id = s.ids[entry - window];
            if (id >= p.pages) id = 0;  // a key on no page: not looked at
            const uint32_t chunk = ((cw * LOADS + i) * 64 + lane) % S::chunks;
            const bool value = is_value(i);
            const uint64_t o = value ? (uint64_t)id * p.vp_sp + (uint64_t)row * p.vp_st + (uint64_t)head * p.vp_sh + (chunk ^ S::value_swizzle(r))
                                     : (uint64_t)id * p.kp_sp + (uint64_t)row * p.kp_st + (uint64_t)head * p.kp_sh + (chunk ^ S::key_swizzle(r));
            at[i] = reinterpret_cast<uint64_t>(value ? p.vp : p.kp) + o * 16 - 1024 * (LOADS == 2 ? i : i & 3);
        }
        const uint32_t base = uniform(buffer(n) + cw * LOADS * 1024);
        if constexpr (LOADS == 2) load_half(at, base);
        else
#pragma unroll
            for (int i = 0; i < LOADS; i += 4) load_rows(at + i, base + i * 1024);
        return exists;
    };

    float m[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) m[ct] = -INFINITY;
    const float unit_of = MASK ? kLog2e : 1.f;  // scores are natural under a mask, else in log2 units
    const float threshold = MASK ? X::threshold / kLog2e : X::threshold;
    uint32_t exists[AHEAD + 1];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) exists[n] = (uint32_t)n < sets ? load(n) : 0u;

    for (uint32_t n = 0; n < sets; ++n) {
        const uint32_t key0 = begin + (n * GROUPS + group) * SK, here = exists[0], at = buffer(n);
        if (AHEAD == 1 || n + 1 == sets) wait_loads<0>();
        else wait_loads<LOADS>();
        // value rows of keys that do not exist become zeros (zero times NaN would be NaN); where some column does not see
        // all keys, those that are not finite are looked for
        const bool partial = MASK || key0 + SK > least;
        if (here != kAll || partial) {
            uint32_t odd = 0;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                if (!is_value(i)) continue;
                const uint32_t to = at + (cw * LOADS + i) * 1024 + lane * 16;
                if (!(here >> row_of(i) & 1u)) lds_write16(to, U4{0u, 0u, 0u, 0u});
                else if (partial && !X::finite(lds_read16(to))) odd = 1;
            }
            odd = __builtin_amdgcn_ballot_w64(odd) != 0;
            if (lane == 0) s.odd[n % L::buffers][wave] = odd;
        }
        lds_barrier();  // the stage is there for all waves, and all have left the one before
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) exists[i] = exists[i + 1];
        exists[AHEAD - 1] = n + AHEAD < sets ? load(n + AHEAD) : 0u;

        f32x4_t score[CT][TILES];
        x.scores(at, score);
        float w[CT][TILES][4];
        bool pass = false;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            float highest = -INFINITY;
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = score[ct][t][i] * p.scale;
                    if (MASK || here != kAll || partial) {
                        const uint32_t k = 16 * t + 4 * g + i, key = key0 + k;
                        bool hidden = !(here >> k & 1u) || key >= seen[ct];
                        if constexpr (MASK) {
                            if (!hidden) {
                                const uint64_t element = (uint64_t)request[ct] * p.m_sb + (uint64_t)key * p.m_st;
                                const uint32_t e = p.mask_dtype == Q3T_F32 ? reinterpret_cast<const uint32_t *>(p.mask)[element]
                                                 : p.mask_dtype == Q3T_BOOL ? reinterpret_cast<const uint8_t *>(p.mask)[element]
                                                                            : reinterpret_cast<const uint16_t *>(p.mask)[element];
                                const float term = mask_term(e, p.mask_dtype);
                                hidden = term == -INFINITY;
                                v += term;
                            }
                        }
                        if (hidden) v = -INFINITY;
                    }
                    w[ct][t][i] = v;
                    highest = fmaxf(highest, v);
                }
            pass |= highest > m[ct] + threshold;
        }
        if (__builtin_amdgcn_ballot_w64(pass)) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                float highest = m[ct];
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) highest = fmaxf(highest, w[ct][t][i]);
                highest = fmaxf(highest, xor16(highest));
                highest = fmaxf(highest, xor32(highest));
                x.rescale(ct, fexp2((m[ct] - (highest == -INFINITY ? 0.f : highest)) * unit_of));
                m[ct] = highest;
            }
        }
        const bool slow = (here != kAll || partial) && [&] {
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < CW; ++i) any |= s.odd[n % L::buffers][group * CW + i];
            return uniform(any) != 0;
        }();
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const float from = m[ct] == -INFINITY ? 0.f : m[ct];
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = X::visible(fexp2((w[ct][t][i] - from) * unit_of + X::shift));
                    w[ct][t][i] = w[ct][t][i] == -INFINITY && (MASK || here != kAll || partial) ? (slow ? -1.f : 0.f) : e;
                }
        }
        if (!slow) {
            x.sums(w);
            x.values(at, w);
            continue;
        }
        // Values that are not finite, among keys that not all columns see: key by key, those that a column sees.
        for (int t = 0; t < TILES; ++t)
            for (int i = 0; i < 4; ++i)
                for (int o = 0; o < 4; ++o) {
                    const int r = 16 * t + 4 * o + i;
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) {
                        float mine = 0.f;
#pragma unroll
                        for (int k = 0; k < TILES * 4; ++k)
                            if (k == 4 * t + i) mine = w[ct][k / 4][k % 4];
                        const float weight = __shfl(mine, 16 * o + c);
                        if (weight < 0.f) continue;
#pragma unroll
                        for (int a = 0; a < D / 16; ++a)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                x.acc[ct][a][e] += weight * X::element(at + (SK + r) * S::row, r, X::dim(a, e, g));
                    }
                }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[ct][t][i] = w[ct][t][i] < 0.f ? 0.f : w[ct][t][i];
        x.sums(w);
    }

    // ---- the groups' states, into one ----
    const uint64_t rows = ((uint64_t)part * p.heads + head) * p.columns;
    float l[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        l[ct] = x.total(ct);
        if (!live[ct] || l[ct] == 0.f) {
            m[ct] = -INFINITY;
            l[ct] = 0.f;
#pragma unroll
            for (int a = 0; a < D / 16; ++a) x.acc[ct][a] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
    }
    if constexpr (GROUPS == 1) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            if (column[ct] >= p.columns) continue;
            if (g == 0) *reinterpret_cast<f32x2_t *>(p.ml + 2 * (rows + column[ct])) = f32x2_t{m[ct], l[ct]};
#pragma unroll
            for (int a = 0; a < D / 16; ++a) {
                if constexpr (sizeof(T) == 4) {
                    for (int i = 0; i < 4; ++i) p.states[(rows + column[ct]) * D + X::dim(a, i, g)] = x.acc[ct][a][i];
                } else {
                    *reinterpret_cast<f32x4_t *>(p.states + (rows + column[ct]) * D + X::dim(a, 0, g)) = x.acc[ct][a];
                }
            }
        }
    } else {
        lds_barrier();  // all have left the last stage
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const int row = ct * kColumns + c;
            if (g == 0) {
                s.ml[wave][row][0] = m[ct];
                s.ml[wave][row][1] = l[ct];
            }
#pragma unroll
            for (int a = 0; a < D / 16; ++a)
#pragma unroll
                for (int i = 0; i < 4; ++i) s.merge[wave][row][X::dim(a, i, g) ^ (c & 7) * 4] = x.acc[ct][a][i];
        }
        lds_barrier();
        constexpr int items = CW * CT * kColumns * (D / 4);
        for (int item = tid; item < items; item += 256) {
            const int col = item / (D / 4), d = item % (D / 4) * 4, of = col / (CT * kColumns), row = col % (CT * kColumns);
            const uint32_t to = block * CW * CT * kColumns + col;
            if (to >= p.columns) continue;
            State sum = {};
            sum.m = -INFINITY;
#pragma unroll
            for (int n = 0; n < GROUPS; ++n) {
                const int from = n * CW + of;
                sum.add(State{s.ml[from][row][0], s.ml[from][row][1], *reinterpret_cast<const f32x4_t *>(&s.merge[from][row][d ^ (row & 7) * 4])}, unit_of);
            }
            *reinterpret_cast<f32x4_t *>(p.states + (rows + to) * D + d) = sum.a;
            if (d == 0) *reinterpret_cast<f32x2_t *>(p.ml + 2 * (rows + to)) = f32x2_t{sum.m, sum.l};
        }
    }
}

// What a launch over a prefix does.
struct PrefixPlan {
    int64_t cw, ct, columns, blocks, parts, chunk, bytes;  // bytes of states
};

// By sizes alone: tiles for the columns that there are, and as many parts as fill the card with a chunk of kLeastChunk keys at least (a
// state is written and read again for every part).
constexpr int64_t kLeastChunk = 256;

template <typename T>
static PrefixPlan prefix_plan(const q3t_paged_args *a, int64_t keys) {
    PrefixPlan z;
    z.columns = a->batch * (a->q_heads / a->kv_heads);
    z.ct = z.columns <= kColumns ? 1 : 2;
    z.cw = z.columns <= 2 * kColumns ? 1 : z.columns <= 4 * kColumns ? 2 : 4;
    z.blocks = (z.columns + z.cw * z.ct * kColumns - 1) / (z.cw * z.ct * kColumns);
    const int64_t step = (4 / z.cw) * (sizeof(T) == 4 ? 16 : 32), workgroups = (z.cw == 1 ? 1 : 2) * 256;
    int64_t parts = workgroups / (z.blocks * a->kv_heads);
    if (parts < 1) parts = 1;
    z.chunk = (keys + parts - 1) / parts;
    if (z.chunk < kLeastChunk) z.chunk = kLeastChunk;
    z.chunk = (z.chunk + step - 1) / step * step;
    z.parts = (keys + z.chunk - 1) / z.chunk;
    z.bytes = z.parts * a->kv_heads * z.columns * (a->head_dim + 2) * 4;
    return z;
}

// `p` the arguments that the attention of the requests' own keys takes, whose strides the prefix' are.
template <typename T>
static int prefix_run(const q3t_paged_args *a, const PrefixPlan &z, int64_t keys, const Params &p, const int32_t *table, const void *mask,
                      float *states, hipStream_t stream) {
    PrefixParams x = {};
    x.q = p.q; x.kp = p.kp; x.vp = p.vp; x.mask = (const char *)mask;
    x.table = table;
    x.positions = a->positions;
    x.states = states;
    x.ml = states + z.parts * a->kv_heads * z.columns * a->head_dim;
    x.q_sb = p.q_sb; x.q_sh = p.q_sh;
    x.kp_sp = p.kp_sp; x.kp_sh = p.kp_sh; x.kp_st = p.kp_st; x.vp_sp = p.vp_sp; x.vp_sh = p.vp_sh; x.vp_st = p.vp_st;
    x.m_sb = p.m_sb; x.m_st = p.m_st; x.mask_dtype = p.mask_dtype;
    x.heads = (uint32_t)a->kv_heads; x.columns = (uint32_t)z.columns; x.blocks = (uint32_t)z.blocks;
    x.parts = (uint32_t)z.parts; x.keys = (uint32_t)keys; x.chunk = (uint32_t)z.chunk;
    x.pages = p.pages;
    x.ctx = (uint32_t)(a->ctx + keys);
    x.by_page = p.by_page;
    x.by_group = divisor(p.group);
    x.scale = p.scale;
    const int64_t units = a->kv_heads * z.parts;
    const dim3 grid((uint32_t)((units + 7) / 8 * 8 * z.blocks));
    auto shape = [&](auto d, auto masked) {
        constexpr int D = decltype(d)::value;
        constexpr bool MASK = decltype(masked)::value;
        auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, x); };
        if (z.cw == 4) launch(prefix_kernel<T, D, MASK, 4, 2>);
        else if (z.cw == 2) launch(prefix_kernel<T, D, MASK, 2, 2>);
        else if (z.ct == 2) launch(prefix_kernel<T, D, MASK, 1, 2>);
        else launch(prefix_kernel<T, D, MASK, 1, 1>);
    };
    auto width = [&](auto masked) {
        if (a->head_dim == 128) shape(std::integral_constant<int, 128>{}, masked);
        else shape(std::integral_constant<int, 64>{}, masked);
    };
    if (mask) width(std::true_type{});
    else width(std::false_type{});
    return launch_status();
}

}  // namespace paged
}  // namespace q3t
