// Rows into a paged cache of 8-bit elements, and rows out of a paged cache.
//
// Written: with a = max(2^-100, max |x|) of a row, int8 elements round(x * (127 / a)) and the scale a / 127;
// e4m3 elements x / s and the scale s, the smallest power of two with a <= 448 s.  A row with an infinity or a NaN gets
// the scale NaN.  Read: scale * element, or the elements of an unquantised pool.
// One pass each: a row lies in 8 or 16 lanes, whose maximum four steps over the lanes find, so it is read once and held in
// registers.  Both are bound by HBM where rows are many and by the launch where they are few.  us per launch, the rows not in the
// caches: 16 prompts of up to 1024 rows, 8 heads of 128, bf16 into int8 16.4 (3.4 TB/s), and read back behind the write, padding
// and all, 16.4 (5.3); both in a graph 33.0 (4.3, nine tenths of a copy's rate); 48 requests of up to 777 rows, 12 heads of 64,
// e4m3 into fp16 34.8 (4.3); one token of 64 requests 2.5 each way; 300 rows of one request 3.2.  Out of pools of the rows' own type:
// the 48 requests in fp16 34.8 (5.1), in bf16 with 8 heads of 128 45.3 (5.2, a copy's rate and a little more); the one of 300 2.7.
#include "paged_index.hpp"
#include "q3t_common.hpp"

#include <type_traits>

namespace q3t {
namespace paged_quantized {

constexpr int kThreads = 256;

struct Rows {  // one of keys and values
    char *rows, *pages;                         // of the call, of the pool
    float *scales;
    int64_t r_sb, r_sh, r_st, p_sp, p_sh, p_st;  // bytes
    int64_t s_sp, s_sh, s_st;                   // elements
};
struct Params {
    Rows x[2];
    const int64_t *positions;
    const int32_t *lengths, *table;
    int64_t table_sb, rows;  // rows: table_width * page_size
    uint32_t batch, heads, tokens, units, pages;
    uint32_t token_last;  // rows are taken head by head, else token by token
    Divisor by_units, by_inner, by_page;  // inner: tokens, or heads
};

// Token and head of a request's row in the order that rows are taken in, some past the end.
Q3T_DEVICE void row_of(const Params &p, uint32_t row, uint32_t &t, uint32_t &h) {
    const uint32_t outer = divide(row, p.by_inner), inner = row - outer * p.by_inner.d;
    t = p.token_last ? inner : outer;
    h = p.token_last ? outer : inner;
}

// Rows of a request that the call has.
Q3T_DEVICE uint32_t used_rows(const Params &p, uint32_t b) {
    return p.lengths ? (uint32_t)max(0, min(p.lengths[b], (int32_t)p.tokens)) : p.tokens;
}
// Place of row t of request b, whose first row is at `start`: page and row of it, page -1 for a row that it has not.
struct Place { int32_t page; uint32_t row; };
Q3T_DEVICE Place place(const Params &p, uint32_t b, int64_t start, uint32_t used, uint32_t t, uint32_t h) {
    // (start + t overflows for no start that is left)
    if (h >= p.heads || t >= used || start >= p.rows || start < -(int64_t)p.tokens || start + t < 0 || start + t >= p.rows) return {-1, 0u};
    const uint32_t j = (uint32_t)(start + t), entry = divide(j, p.by_page);
    const int32_t page = p.table[b * p.table_sb + entry];
    return {(uint32_t)page < p.pages ? page : -1, j - entry * p.by_page.d};
}

// The call's rows are read and written once: the non-temporal policy.  The pools' are not, which what follows reads (16 prompts of
// up to 1024 rows in int8 written and read back 32.5 us; all with the policy 37.3, none 37.1).
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

template <typename T> struct Eight { alignas(16) T x[8]; };

// Eight elements of a row; VEC: by 16-byte accesses.
template <bool VEC, typename T>
Q3T_DEVICE void load8(const char *from, Eight<T> &e) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(e) / 16; ++i)
            reinterpret_cast<u32x4_t *>(&e)[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(from) + i);
    } else {
        for (int i = 0; i < 8; ++i) e.x[i] = reinterpret_cast<const T *>(from)[i];
    }
}
template <bool VEC, typename T>
Q3T_DEVICE void store8(char *to, const Eight<T> &e) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(e) / 16; ++i)
            __builtin_nontemporal_store(reinterpret_cast<const u32x4_t *>(&e)[i], reinterpret_cast<u32x4_t *>(to) + i);
    } else {
        for (int i = 0; i < 8; ++i) reinterpret_cast<T *>(to)[i] = e.x[i];
    }
}

Q3T_DEVICE uint32_t dpp_max(uint32_t x, uint32_t y) { return x > y ? x : y; }
template <int CTRL> Q3T_DEVICE uint32_t dpp_u(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false);
}

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
Q3T_DEVICE uint32_t pairs_max(uint32_t x, uint32_t y) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, x), __builtin_bit_cast(u16x2_t, y)));
}

// The largest |x| of a row of L lanes of eight elements, as float32's bits: NaN above infinity above the rest.  Types of 16
// bits are compared as such, two at once.
template <int L, typename T> Q3T_DEVICE uint32_t row_largest(const Eight<T> &e) {
    const uint32_t *bits = reinterpret_cast<const uint32_t *>(&e);
    auto over_lanes = [](uint32_t m, auto max) {
        m = max(m, dpp_u<kDppXor1>(m));
        m = max(m, dpp_u<kDppXor2>(m));
        m = max(m, dpp_u<kDppHalfMirror>(m));
        return L == 16 ? max(m, xor8u(m)) : m;
    };
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) m = dpp_max(m, bits[i] & 0x7fffffffu);
        return over_lanes(m, dpp_max);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = pairs_max(m, bits[i] & 0x7fff7fffu);
        m = over_lanes(m, pairs_max);
        m = dpp_max(m & 0xffffu, m >> 16);
        if constexpr (std::is_same<T, _Float16>::value) return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)m));
        return m << 16;
    }
}

// x / 127 for x of 2^-100 and above, rounded as a division is: a quotient from the nearest reciprocal, put right by what it
// leaves (Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990).
Q3T_DEVICE float by_127(float x) {
    const float r = 1.f / 127.f, q = x * r;
    return __builtin_fmaf(__builtin_fmaf(-q, 127.f, x), r, q);
}
// 127 / x for the same: of its mantissa alone, whose reciprocal is a normal number (tried for all 2^23 of them).
Q3T_DEVICE float of_127(float x) {
    const uint32_t bits = __float_as_uint(x);
    const float m = __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
    float r = __builtin_amdgcn_rcpf(m);
    r = __builtin_fmaf(__builtin_fmaf(-m, r, 1.f), r, r);
    float q = 127.f * r;
    q = __builtin_fmaf(__builtin_fmaf(-q, m, 127.f), r, q);
    return __uint_as_float(__float_as_uint(q) - ((bits >> 23) - 127) * (1u << 23));
}

// A row's scale and the lane's eight elements.
template <bool E4M3> Q3T_DEVICE uint2 quantise(const float (&x)[8], uint32_t largest, float &scale) {
#pragma clang fp contract(off)
    const bool finite = largest < 0x7f800000u;
    const uint32_t a = dpp_max(largest, 0x0d800000u);  // 2^-100
    float inverse;
    if constexpr (E4M3) {
        // a = m 2^E: s = 2^(E - 8) where m <= 1.75, else 2^(E - 7); the carry out of the mantissa says which
        const uint32_t exponent = ((a + 0x1fffffu) >> 23) - 8;
        scale = __uint_as_float(exponent << 23);
        inverse = __uint_as_float((254 - exponent) << 23);
    } else {
        scale = by_127(__uint_as_float(a));
        inverse = of_127(__uint_as_float(a));
    }
    if (!finite) scale = __uint_as_float(0x7fc00000u);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (E4M3) {
            w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inverse, x[4 * i + 1] * inverse, 0, false);
            w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inverse, x[4 * i + 3] * inverse, (int)w[i], true);
        } else {
            // products of at most 127, rounded to whole numbers by an addition to 1.5 2^23, whose low byte they then are
            uint32_t u[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k] = __float_as_uint(x[4 * i + k] * inverse + 0x1.8p23f);
            w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x00000400u), __builtin_amdgcn_perm(u[1], u[0], 0x00000400u), 0x05040100u);
        }
        if (!finite) w[i] = 0;
    }
    return uint2{w[0], w[1]};
}

// A thread takes eight elements of N rows of the keys and of the values, 256 / L rows apart; L threads have a row.  The rows are on
// their way before the positions and page numbers are known; with two of them (launches that fill the card) those past a request's
// length are not read.
template <typename T, int L, bool E4M3, bool VEC, int N>
__global__ void __launch_bounds__(kThreads) write_kernel(Params p) {
    for (uint32_t b = blockIdx.y; b < p.batch; b += gridDim.y) {
        const int64_t start = p.positions[b];
        const uint32_t used = used_rows(p, b), unit = threadIdx.x % L;
        Eight<T> e[N][2];
        uint32_t t[N], h[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const uint32_t row = ((blockIdx.x * N + k) * kThreads + threadIdx.x) / L;
            row_of(p, row, t[k], h[k]);
            if (h[k] >= p.heads || t[k] >= (N == 1 ? p.tokens : used)) continue;
#pragma unroll
            for (int n = 0; n < 2; ++n)
                load8<VEC>(p.x[n].rows + b * p.x[n].r_sb + h[k] * p.x[n].r_sh + t[k] * p.x[n].r_st + unit * 8 * sizeof(T), e[k][n]);
        }
        Place at[N];
#pragma unroll
        for (int k = 0; k < N; ++k) at[k] = place(p, b, start, used, t[k], h[k]);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (at[k].page < 0) continue;  // (the same for all lanes of a row)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const Rows &r = p.x[n];
                float x[8], scale;
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = (float)e[k][n].x[i];
                const uint2 w = quantise<E4M3>(x, row_largest<L>(e[k][n]), scale);
                *reinterpret_cast<u32x2_t *>(r.pages + at[k].page * r.p_sp + h[k] * r.p_sh + at[k].row * r.p_st + unit * 8) = u32x2_t{w.x, w.y};
                if (unit == 0) r.scales[at[k].page * r.s_sp + h[k] * r.s_sh + at[k].row * r.s_st] = scale;
            }
        }
    }
}

// Eight elements, from their bytes.
template <bool E4M3> Q3T_DEVICE void elements(uint2 w, float (&x)[8]) {
    const uint32_t u[2] = {w.x, w.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (E4M3) {
            const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], true);
            x[4 * i] = lo[0]; x[4 * i + 1] = lo[1]; x[4 * i + 2] = hi[0]; x[4 * i + 3] = hi[1];
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) x[4 * i + k] = (float)(int8_t)(u[i] >> 8 * k);
        }
    }
}

template <typename T> Q3T_DEVICE T rounded(float x) { return (T)x; }
// (a product and its rounding become one instruction otherwise, which adds a zero: -0 would be 0)
template <> Q3T_DEVICE _Float16 rounded<_Float16>(float x) {
    asm("" : "+v"(x));
    return (_Float16)x;
}
template <> Q3T_DEVICE __bf16 rounded<__bf16>(float x) { return __builtin_bit_cast(__bf16, (uint16_t)float_to_bf16(x)); }

template <typename T, int L, bool E4M3, bool VEC, int N>
__global__ void __launch_bounds__(kThreads) read_kernel(Params p) {
    for (uint32_t b = blockIdx.y; b < p.batch; b += gridDim.y) {
        const int64_t start = p.positions[b];
        const uint32_t used = used_rows(p, b), unit = threadIdx.x % L;
        uint32_t t[N], h[N];
        Place at[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const uint32_t row = ((blockIdx.x * N + k) * kThreads + threadIdx.x) / L;
            row_of(p, row, t[k], h[k]);
            at[k] = place(p, b, start, used, t[k], h[k]);
        }
        u32x2_t w[N][2];
        float scale[N][2];
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const Rows &r = p.x[n];
                w[k][n] = u32x2_t{0u, 0u};
                scale[k][n] = 0.f;
                if (at[k].page < 0) continue;
                w[k][n] = *reinterpret_cast<const u32x2_t *>(r.pages + at[k].page * r.p_sp + h[k] * r.p_sh + at[k].row * r.p_st + unit * 8);
                scale[k][n] = r.scales[at[k].page * r.s_sp + h[k] * r.s_sh + at[k].row * r.s_st];
            }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (h[k] >= p.heads || t[k] >= p.tokens) continue;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const Rows &r = p.x[n];
                float x[8];
                elements<E4M3>(uint2{w[k][n][0], w[k][n][1]}, x);
                Eight<T> e;
#pragma unroll
                for (int i = 0; i < 8; ++i) e.x[i] = at[k].page < 0 ? (T)0.f : rounded<T>(x[i] * scale[k][n]);
                store8<VEC>(r.rows + b * r.r_sb + h[k] * r.r_sh + t[k] * r.r_st + unit * 8 * sizeof(T), e);
            }
        }
    }
}

// Units of V bytes out of pools of the rows' own type.
template <int V> struct Unit { typedef uint32_t T __attribute__((ext_vector_type(V / 4))); };
template <> struct Unit<4> { typedef uint32_t T; };
template <> struct Unit<2> { typedef uint16_t T; };

template <int V, int N>
__global__ void __launch_bounds__(kThreads) copy_kernel(Params p) {
    typedef typename Unit<V>::T T;
    for (uint32_t b = blockIdx.y; b < p.batch; b += gridDim.y) {
        const int64_t start = p.positions[b];
        const uint32_t used = used_rows(p, b);
        uint32_t t[N], h[N];
        int64_t unit[N];
        Place at[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const uint32_t i = (blockIdx.x * N + k) * kThreads + threadIdx.x, row = divide(i, p.by_units);
            row_of(p, row, t[k], h[k]);
            unit[k] = (int64_t)(i - row * p.units) * V;
            at[k] = place(p, b, start, used, t[k], h[k]);
        }
        T v[N][2];
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const Rows &r = p.x[n];
                v[k][n] = T{};
                if (at[k].page >= 0)
                    v[k][n] = __builtin_nontemporal_load(reinterpret_cast<const T *>(r.pages + at[k].page * r.p_sp + h[k] * r.p_sh + at[k].row * r.p_st + unit[k]));
            }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (h[k] >= p.heads || t[k] >= p.tokens) continue;
#pragma unroll
            for (int n = 0; n < 2; ++n)
                __builtin_nontemporal_store(v[k][n], reinterpret_cast<T *>(p.x[n].rows + b * p.x[n].r_sb + h[k] * p.x[n].r_sh + t[k] * p.x[n].r_st + unit[k]));
        }
    }
}

// The fields that writes and reads share; Q3T_OK, or the status to return.
template <typename A>
static int common(const A *a, int64_t es, int64_t held, const q3t_paged_scales *s, Params &p) {
    if (!a || a->batch < 0 || a->heads < 1 || a->tokens < 0 || a->width < 1 || a->pages < 1 || a->page_size < 1 || a->table_width < 1)
        return Q3T_EINVAL;
    if (s && s->format != Q3T_I8 && s->format != Q3T_E4M3) return Q3T_EUNSUPPORTED;
    if (s && a->width != 64 && a->width != 128) return Q3T_EUNSUPPORTED;
    if (a->batch == 0 || a->tokens == 0) return Q3T_OK;
    if (!a->keys || !a->values || !a->key_pages || !a->value_pages || !a->page_table || !a->positions) return Q3T_EINVAL;
    if (s && (!s->key_scales || !s->value_scales || !aligned(s->key_scales, 4) || !aligned(s->value_scales, 4))) return Q3T_EINVAL;
    if (a->pages > INT32_MAX || a->table_width > INT32_MAX / a->page_size || a->batch > INT32_MAX || a->heads > INT32_MAX ||
        a->tokens > INT32_MAX || a->width > 1 << 20)
        return Q3T_EUNSUPPORTED;
    p.x[0] = {(char *)a->keys, (char *)a->key_pages, s ? s->key_scales : nullptr, a->k_stride_b * es, a->k_stride_h * es,
              a->k_stride_t * es, a->kp_stride_p * held, a->kp_stride_h * held, a->kp_stride_t * held,
              s ? s->ks_stride_p : 0, s ? s->ks_stride_h : 0, s ? s->ks_stride_t : 0};
    p.x[1] = {(char *)a->values, (char *)a->value_pages, s ? s->value_scales : nullptr, a->v_stride_b * es, a->v_stride_h * es,
              a->v_stride_t * es, a->vp_stride_p * held, a->vp_stride_h * held, a->vp_stride_t * held,
              s ? s->vs_stride_p : 0, s ? s->vs_stride_h : 0, s ? s->vs_stride_t : 0};
    p.positions = a->positions; p.lengths = a->lengths; p.table = a->page_table;
    p.table_sb = a->table_stride_b;
    p.rows = a->table_width * a->page_size;
    p.batch = (uint32_t)a->batch; p.heads = (uint32_t)a->heads; p.tokens = (uint32_t)a->tokens;
    p.pages = (uint32_t)a->pages;
    // In the order of the call's rows: a projection's heads lie side by side, a prefill cache's tokens, as they do in pages.  us,
    // token by token / head by head: written in int8, 16 prompts of 600 rows of a cache, 8 heads of 128, 16.6 / 16.1, 4 of 200 3.6 /
    // 3.3, 48 of 700, 12 heads of 64, 37.5 / 35.6; the last read 35.7 / 33.1, 48 of up to 777 in e4m3 36.1 / 34.4; 16 of up to 1024
    // read behind their write 15.8 / 16.4.
    p.token_last = a->k_stride_t <= a->k_stride_h;
    p.by_inner = divisor(p.token_last ? p.tokens : p.heads);
    p.by_page = divisor((uint32_t)a->page_size);
    if (!aligned(a->page_table, 4) || !aligned(a->positions, 8) || (a->lengths && !aligned(a->lengths, 4))) return Q3T_EINVAL;
    for (const Rows &r : p.x) {
        const int64_t at = r.p_sp | r.p_sh | r.p_st | (int64_t)(uintptr_t)r.pages;
        if (s ? at % 16 : at % es) return Q3T_EINVAL;
        if ((r.r_sb | r.r_sh | r.r_st | (int64_t)(uintptr_t)r.rows) % es) return Q3T_EINVAL;
    }
    return Q3T_OK;
}

// What every row of the call, and every pool row, is a multiple of, in bytes.
static int64_t strides(const Params &p, bool pools) {
    int64_t all = 0;
    for (const Rows &r : p.x) {
        all |= r.r_sb | r.r_sh | r.r_st | (int64_t)(uintptr_t)r.rows;
        if (pools) all |= r.p_sp | r.p_sh | r.p_st | (int64_t)(uintptr_t)r.pages;
    }
    return all;
}

// Launches one of two kernels, of one and of two units a thread, for `units` units of a row; Q3T_OK, or the status to return.
constexpr int64_t kManyBlocks = 2048;  // workgroups of one unit a thread that the card holds at once
template <typename K1, typename K2>
static int launch(K1 one, K2 two, Params &p, uint32_t units, void *stream) {
    p.units = units;
    p.by_units = divisor(units);
    // units of a request stay below 2^31, and threads of a launch below 2^32
    if (p.heads > INT32_MAX / units || p.tokens > (INT32_MAX - 2 * kThreads) / (p.heads * units)) return Q3T_EUNSUPPORTED;
    const int64_t all = (int64_t)p.tokens * p.heads * units;
    const bool many = all / kThreads * p.batch >= kManyBlocks;
    const int64_t each = kThreads * (many ? 2 : 1), blocks = (all + each - 1) / each, most = ((int64_t)1 << 24) - 1;
    if (blocks > most) return Q3T_EUNSUPPORTED;
    int64_t across = p.batch < 65535 ? p.batch : 65535;
    if (across > most / blocks) across = most / blocks;
    hipLaunchKernelGGL(many ? two : one, dim3((uint32_t)blocks, (uint32_t)across), dim3(kThreads), 0, (hipStream_t)stream, p);
    return launch_status();
}

// f(type, lanes of a row, e4m3, vectors) for a call's rows
template <typename F>
static int with(int64_t dtype, int64_t width, int64_t format, bool vec, F f) {
    auto by_vec = [&](auto t, auto l, auto e) { return vec ? f(t, l, e, std::true_type{}) : f(t, l, e, std::false_type{}); };
    auto by_format = [&](auto t, auto l) { return format == Q3T_E4M3 ? by_vec(t, l, std::true_type{}) : by_vec(t, l, std::false_type{}); };
    auto by_width = [&](auto t) {
        return width == 64 ? by_format(t, std::integral_constant<int, 8>{}) : by_format(t, std::integral_constant<int, 16>{});
    };
    if (dtype == Q3T_F32) return by_width(float{});
    return dtype == Q3T_BF16 ? by_width(__bf16{}) : by_width(_Float16{});
}

}  // namespace paged_quantized
}  // namespace q3t

using namespace q3t;

extern "C" int q3t_paged_write_quantized(const q3t_paged_write_args *a, int64_t dtype, const q3t_paged_scales *s, void *stream) {
    using namespace paged_quantized;
    if (!a || !s) return Q3T_EINVAL;
    if (dtype != Q3T_BF16 && dtype != Q3T_F16 && dtype != Q3T_F32) return Q3T_EUNSUPPORTED;
    if (a->elem_size != (dtype == Q3T_F32 ? 4 : 2)) return Q3T_EINVAL;
    Params p = {};
    const int status = common(a, a->elem_size, 1, s, p);
    if (status != Q3T_OK || a->batch == 0 || a->tokens == 0) return status;
    return with(dtype, a->width, s->format, strides(p, false) % 16 == 0, [&](auto t, auto l, auto e, auto vec) {
        constexpr int L = decltype(l)::value;
        constexpr bool E = decltype(e)::value, VEC = decltype(vec)::value;
        return launch(write_kernel<decltype(t), L, E, VEC, 1>, write_kernel<decltype(t), L, E, VEC, 2>, p, L, stream);
    });
}

extern "C" int q3t_paged_read(const q3t_paged_read_args *a, const q3t_paged_scales *s, void *stream) {
    using namespace paged_quantized;
    if (!a) return Q3T_EINVAL;
    if (a->dtype != Q3T_BF16 && a->dtype != Q3T_F16 && a->dtype != Q3T_F32) return Q3T_EUNSUPPORTED;
    const int64_t es = a->dtype == Q3T_F32 ? 4 : 2;
    Params p = {};
    const int status = common(a, es, s ? 1 : es, s, p);
    if (status != Q3T_OK || a->batch == 0 || a->tokens == 0) return status;
    if (s)
        return with(a->dtype, a->width, s->format, strides(p, false) % 16 == 0, [&](auto t, auto l, auto e, auto vec) {
            constexpr int L = decltype(l)::value;
            constexpr bool E = decltype(e)::value, VEC = decltype(vec)::value;
            return launch(read_kernel<decltype(t), L, E, VEC, 1>, read_kernel<decltype(t), L, E, VEC, 2>, p, L, stream);
        });
    const int64_t all = strides(p, true) | a->width * es;  // the widest unit that divides the row, every stride and every pointer
    int64_t v = 16;
    while (v > es && all % v) v >>= 1;
    const uint32_t units = (uint32_t)(a->width * es / v);
    switch (v) {
        case 16: return launch(copy_kernel<16, 1>, copy_kernel<16, 2>, p, units, stream);
        case 8: return launch(copy_kernel<8, 1>, copy_kernel<8, 2>, p, units, stream);
        case 4: return launch(copy_kernel<4, 1>, copy_kernel<4, 2>, p, units, stream);
        default: return launch(copy_kernel<2, 1>, copy_kernel<2, 2>, p, units, stream);
    }
}
