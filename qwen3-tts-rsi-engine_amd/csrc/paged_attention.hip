// Attention of one new token per request over a cache kept in pages (the paged counterpart of the
// decode attention; reference: packed_attention.py:75-84).
//
//   s_j = scale q . k_j (+ mask_j),  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// in one pass over the keys, with a running maximum m that moves when it is passed by more than a
// threshold.  Every key and value row is read once, so HBM bounds a launch of many keys (2 to 16
// operations per byte), and the chain arguments - positions - page numbers - rows - merge one of few.
//   * Work: a workgroup of four waves takes an equal share of the rounds of all (request, KV head)
//     pairs (paged_index.hpp), whatever the requests' lengths; it finds its place by adding up
//     all requests' rounds.  A pair that lies in several shares leaves its parts' states in the
//     workspace, and the workgroup that arrives last merges them, in the parts' order.
//   * A wave takes every fourth stage of 16 (rows of 128 bytes: 32) keys of a pair.  A stage's rows
//     go straight from memory to the wave's own two LDS slots, one stage ahead of the one that is
//     scored, over the ends of pairs: no barrier but where a pair ends.  The stages' page numbers
//     come the same way, two stages before the rows that they place; each lane works out the
//     address of its own row, so that any page size will do.
//   * The rows of a KV head's query heads are the columns of 16x16 products, S^T = K . Q^T and
//     O^T += V^T . P^T.  The matrix cores idle (under a twentieth of their rate), so the weights are
//     not rounded to the cache's type: bf16 weights go in three parts (all 24 bits of their
//     float32), fp16 ones in two (22 bits), float32 is multiplied as such.  The first part has
//     accumulators of its own: an infinite value times a remainder of zero would be NaN.
//   * A key that does not exist (past the request's end, under a mask's minus infinity, on no page)
//     scores minus infinity, and its value row is zeroed in LDS: zero times NaN would be NaN.
#include "paged_index.hpp"
#include "q3t_common.hpp"

namespace q3t {
namespace paged {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kColumns = 16;           // query heads of a workgroup: columns of a product
constexpr int kWindow = 256;           // requests whose lengths are at hand
constexpr uint32_t kLeastRounds = 4;   // rounds that are not shared out
constexpr int kCounters = 65536;       // counter words in front of a decode workspace
constexpr float kLog2e = 1.4426950408889634f;

struct Params {
    const char *q, *kp, *vp, *mask;
    char *out;
    const int32_t *table;
    const int64_t *positions;
    int32_t *counters;
    float *states;
    int64_t q_sb, q_sh, o_sb, o_sh;                    // bytes
    int64_t m_sb, m_st, table_sb;                      // elements
    uint32_t kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st; // 16 bytes
    int32_t ctx, mask_dtype, stream, vec_out;
    uint32_t batch, pages, group, heads, blocks;       // heads: pairs of a request; blocks: of a KV head
    uint32_t columns;                                  // of a state
    Divisor by_page;
    float scale;                                       // unmasked: times log2(e)
};

template <typename T, int D>
struct Shape {
    static constexpr int row = D * (int)sizeof(T);
    static constexpr int chunks = row / 16;                // 16-byte chunks of a row
    static constexpr int keys = row == 128 ? 32 : 16;      // of a wave's stage
    static constexpr int stage = 2 * keys * row;           // key rows, then value rows
    static constexpr int loads = keys * row / 1024;        // 1 KiB loads of either
    static constexpr int round = kWaves * keys;
    static constexpr int log_round = keys == 32 ? 7 : 6;
    static constexpr bool f32 = sizeof(T) == 4;
    // the queries of two pairs, and accumulators of at least 4 KiB (8 of 512-byte rows)
    static constexpr int shared = 2 * kColumns * row + (row == 512 ? 8192 : 4096);
    static constexpr int per_cu = row == 512 ? 1 : 2;      // workgroups that fit a CU's LDS
    // chunk c of key (value) row r sits at c ^ swizzle: the products' reads meet distinct banks
    static Q3T_DEVICE int key_swizzle(int r) { return chunks == 8 ? (r >> 1) & 7 : r & 15; }
    static Q3T_DEVICE int value_swizzle(int r) { return f32 ? 0 : chunks == 8 ? (2 * (r >> 1)) & 7 : (2 * r) & 15; }
};

template <typename T, int D, bool MASK>
struct Lds {
    alignas(1024) char ring[kWaves][2][Shape<T, D>::stage];
    alignas(16) char shared[Shape<T, D>::shared];
    alignas(16) int32_t ids[kWaves][4][Shape<T, D>::keys];
    alignas(16) uint32_t maskw[MASK ? kWaves : 1][2][MASK ? Shape<T, D>::keys : 4];
    float ml[kWaves][kColumns][2];
    int32_t lengths[kWindow];
    uint32_t sums[kWaves][2];
    uint32_t start[4];
};

#define Q3T_LDS __attribute__((address_space(3)))
#define Q3T_GLOBAL __attribute__((address_space(1)))
Q3T_DEVICE uint32_t lds_at(const void *x) { return (uint32_t)(uintptr_t)(Q3T_LDS const char *)x; }
Q3T_DEVICE uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

// Four 16-byte loads per lane into LDS, 1 KiB apart there: the instructions' offsets move both
// addresses, so load i's pointer is 1024 i short of its row.
#define Q3T_LOAD4(POLICY)                                                                             \
    asm volatile("s_mov_b32 m0, %0\n\t" Q3T_VMEM_SGPR_WAIT                                            \
                 "global_load_lds_dwordx4 %1, off" POLICY "\n\t"                                      \
                 "global_load_lds_dwordx4 %2, off offset:1024" POLICY "\n\t"                          \
                 "global_load_lds_dwordx4 %3, off offset:2048" POLICY "\n\t"                          \
                 "global_load_lds_dwordx4 %4, off offset:3072" POLICY                                 \
                 :: "s"(base), "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]) : "memory", "m0")
Q3T_DEVICE void load_rows(const uint64_t *p, uint32_t base, bool stream) {
    if (stream) Q3T_LOAD4(" nt");
    else Q3T_LOAD4("");
}
#undef Q3T_LOAD4
Q3T_DEVICE void load_lds16(uint64_t from, uint32_t base) {
    asm volatile("s_mov_b32 m0, %0\n\t" Q3T_VMEM_SGPR_WAIT "global_load_lds_dwordx4 %1, off"
                 :: "s"(base), "v"(from) : "memory", "m0");
}
Q3T_DEVICE void load_lds4(uint64_t from, uint32_t base) {
    asm volatile("s_mov_b32 m0, %0\n\t" Q3T_VMEM_SGPR_WAIT "global_load_lds_dword %1, off"
                 :: "s"(base), "v"(from) : "memory", "m0");
}

// States pass between workgroups through device-scope accesses, which are coherent across the
// XCDs' L2 caches; a writer's stores have completed before the barrier ahead of its count.
Q3T_DEVICE void publish(float *p, float a, float b) {
    const uint64_t v = (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32;
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
Q3T_DEVICE void collect(const float *p, float &a, float &b) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    a = __uint_as_float((uint32_t)v);
    b = __uint_as_float((uint32_t)(v >> 32));
}

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// The products of a wave's tile of 16 keys, by type.  Lane (g, c) = (lane / 16, lane % 16) holds
// column c; of S^T the keys 4 g ... 4 g + 3.
template <typename T, int D> struct Tile;

// 16-bit types: Type gives the products and the weights' parts.
template <typename T> struct Half;
template <> struct Half<__bf16> {
    static constexpr int parts = 3;
    static constexpr float shift = 0.f, threshold = 8.f;
    static Q3T_DEVICE f32x4_t scores(const U4 &k, const U4 &q, f32x4_t s) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(k), as_bf16x8(q), s, 0, 0, 0);
    }
    static Q3T_DEVICE f32x4_t values(uint2 v, uint2 p, f32x4_t a) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, v), __builtin_bit_cast(s16x4_t, p), a, 0, 0, 0);
    }
    static Q3T_DEVICE uint32_t round2(float a, float b) { return cvt_pk_bf16(a, b); }
    static Q3T_DEVICE float lo(uint32_t x) { return bf16_lo(x); }
    static Q3T_DEVICE float hi(uint32_t x) { return bf16_hi(x); }
    static Q3T_DEVICE uint32_t store2(float a, float b) { return cvt_pk_bf16_canon(a, b); }
};
// fp16 weights are kept 2^8 larger than exp(s - m), so that small ones keep their bits, and stay
// below 2^14 with the smaller threshold.
template <> struct Half<_Float16> {
    static constexpr int parts = 2;
    static constexpr float shift = 8.f, threshold = 6.f;
    static Q3T_DEVICE f32x4_t scores(const U4 &k, const U4 &q, f32x4_t s) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, k), __builtin_bit_cast(f16x8_t, q), s, 0, 0, 0);
    }
    static Q3T_DEVICE f32x4_t values(uint2 v, uint2 p, f32x4_t a) {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_t, v), __builtin_bit_cast(f16x4_t, p), a, 0, 0, 0);
    }
    static Q3T_DEVICE uint32_t round2(float a, float b) {
        const f16x2_t h = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(uint32_t, h);
    }
    static Q3T_DEVICE float lo(uint32_t x) { return (float)__builtin_bit_cast(f16x2_t, x)[0]; }
    static Q3T_DEVICE float hi(uint32_t x) { return (float)__builtin_bit_cast(f16x2_t, x)[1]; }
    static Q3T_DEVICE uint32_t store2(float a, float b) { return round2(a, b); }
};

template <typename T, int D> struct Tile {
    typedef Shape<T, D> S;
    static constexpr float shift = Half<T>::shift, threshold = Half<T>::threshold;
    U4 q[D / 32];
    f32x4_t first[D / 16], rest[D / 16];  // O^T by the weights' first part, and by the others

    // Lane (g, c) takes dims 32 kk + 8 g ... of the query row of column c.
    Q3T_DEVICE void load_query(uint32_t rows, int g, int c, bool live) {
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) q[kk] = live ? lds_read16(rows + c * S::row + (4 * kk + g) * 16) : U4{0u, 0u, 0u, 0u};
    }
    Q3T_DEVICE void clear() {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) first[d] = rest[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    Q3T_DEVICE void rescale(float a) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            first[d] *= a;
            rest[d] *= a;
        }
    }
    Q3T_DEVICE f32x4_t scores(uint32_t keys, int t, int g, int c) const {
        const int r = 16 * t + c;
        f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk)
            s = Half<T>::scores(lds_read16(keys + r * S::row + (((4 * kk + g) ^ S::key_swizzle(r)) & (S::chunks - 1)) * 16), q[kk], s);
        return s;
    }
    Q3T_DEVICE void values(uint32_t rows, int t, int g, int c, const float (&w)[4]) {
        uint2 part[3];
        float x[4] = {w[0], w[1], w[2], w[3]};
#pragma unroll
        for (int i = 0; i < Half<T>::parts; ++i) {
            part[i] = uint2{Half<T>::round2(x[0], x[1]), Half<T>::round2(x[2], x[3])};
            x[0] -= Half<T>::lo(part[i].x);
            x[1] -= Half<T>::hi(part[i].x);
            x[2] -= Half<T>::lo(part[i].y);
            x[3] -= Half<T>::hi(part[i].y);
        }
        const int r = 16 * t + 4 * g + (c >> 2);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            const int chunk = ((2 * d + ((c >> 1) & 1)) ^ S::value_swizzle(r)) & (S::chunks - 1);
            const uint2 v = lds_read_tr16(rows + r * S::row + chunk * 16 + 8 * (c & 1));
            first[d] = Half<T>::values(v, part[0], first[d]);
#pragma unroll
            for (int i = 1; i < Half<T>::parts; ++i) rest[d] = Half<T>::values(v, part[i], rest[d]);
        }
    }
    // Elements of column c into its row of D floats.
    Q3T_DEVICE void store(uint32_t to, int g) const {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            f32x4_t x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __builtin_fabsf(first[d][i]) < INFINITY ? first[d][i] + rest[d][i] : first[d][i];
            lds_write16(to + (16 * d + 4 * g) * 4, __builtin_bit_cast(U4, x));
        }
    }
};

// float32: products of four, whose inner index g stands for dims 16 kk + 4 g + e (scores) and for key
// 4 g + i (values); row c of a value product is dim 64 j + 4 c + e.
template <int D> struct Tile<float, D> {
    typedef Shape<float, D> S;
    static constexpr float shift = 0.f, threshold = 8.f;
    f32x4_t q[D / 16], acc[D / 16];

    static Q3T_DEVICE f32x4_t read(uint32_t at) { return __builtin_bit_cast(f32x4_t, lds_read16(at)); }
    Q3T_DEVICE void load_query(uint32_t rows, int g, int c, bool live) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) q[kk] = live ? read(rows + c * S::row + (4 * kk + g) * 16) : f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    Q3T_DEVICE void clear() {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) acc[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    Q3T_DEVICE void rescale(float a) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) acc[d] *= a;
    }
    Q3T_DEVICE f32x4_t scores(uint32_t keys, int t, int g, int c) const {
        const int r = 16 * t + c;
        f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            const f32x4_t k = read(keys + r * S::row + ((4 * kk + g) ^ S::key_swizzle(r)) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[e], q[kk][e], s, 0, 0, 0);
        }
        return s;
    }
    Q3T_DEVICE void values(uint32_t rows, int t, int g, int c, const float (&w)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
                const f32x4_t v = read(rows + (16 * t + 4 * g + i) * S::row + (16 * j + c) * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[4 * j + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e], w[i], acc[4 * j + e], 0, 0, 0);
            }
    }
    Q3T_DEVICE void store(uint32_t to, int g) const {
#pragma unroll
        for (int j = 0; j < D / 64; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4_t x = {acc[4 * j][i], acc[4 * j + 1][i], acc[4 * j + 2][i], acc[4 * j + 3][i]};
                lds_write16(to + (64 * j + 4 * (4 * g + i)) * 4, __builtin_bit_cast(U4, x));
            }
    }
};

// The mask term of a word that holds the element at byte `low` of it.
Q3T_DEVICE float mask_term(uint32_t word, uint32_t low, int dtype) {
    switch (dtype) {
        case Q3T_BF16: return bf16_to_float((word >> (8 * low)) & 0xffffu);
        case Q3T_F16: return (float)__builtin_bit_cast(_Float16, (uint16_t)(word >> (8 * low)));
        case Q3T_F32: return __uint_as_float(word);
        default: return (word >> (8 * low)) & 0xffu ? 0.0f : -INFINITY;  // bool: true attends
    }
}

template <typename T>
Q3T_DEVICE void store_out(char *at, const float (&y)[4], bool vec) {
    if constexpr (sizeof(T) == 4) {
        if (vec) *(Q3T_GLOBAL f32x4_t *)(uintptr_t)at = f32x4_t{y[0], y[1], y[2], y[3]};
        else
            for (int i = 0; i < 4; ++i) ((Q3T_GLOBAL float *)(uintptr_t)at)[i] = y[i];
    } else {
        typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
        const u32x2_t v = {Half<T>::store2(y[0], y[1]), Half<T>::store2(y[2], y[3])};
        if (vec) *(Q3T_GLOBAL u32x2_t *)(uintptr_t)at = v;
        else
            for (int i = 0; i < 4; ++i) ((Q3T_GLOBAL uint16_t *)(uintptr_t)at)[i] = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
    }
}

// A wave's stage: keys from key0 on of request b (length keys) under pair `head`, in the share's run.
struct Stage {
    uint32_t b, head, length, key0;
    int32_t run;  // -1: none
};

template <typename T, int D, bool MASK>
__global__ void __launch_bounds__(kThreads, (Shape<T, D>::per_cu)) paged_kernel(Params p) {
    typedef Shape<T, D> S;
    typedef Tile<T, D> Products;
    constexpr int LOADS = 2 * S::loads;
    __shared__ Lds<T, D, MASK> s;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int wave = (int)uniform(tid >> 6);

    // ---- the share: all requests' rounds and pieces, then the request that it starts in --------
    auto length_of = [&](int64_t pos) { return pos >= 0 && pos < p.ctx ? (int)pos + 1 : 0; };
    auto rounds_of = [&](int length) { return (uint32_t)max(1, (length + S::round - 1) >> S::log_round); };
    const uint32_t each = (p.batch + kThreads - 1) / kThreads;  // requests of a thread, one after the other
    uint32_t rounds = 0, pieces = 0;
    for (uint32_t i = 0; i < each; ++i) {
        const uint32_t b = tid * each + i;
        if (b >= p.batch) break;
        const int length = length_of(p.positions[b]);
        if (each == 1) s.lengths[tid] = length;
        rounds += rounds_of(length);
        pieces += (rounds_of(length) + kLeastRounds - 1) / kLeastRounds;
    }
    uint32_t rounds_to = rounds, pieces_to = pieces;  // sums up to and with this thread
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t a = __shfl_up(rounds_to, o), b = __shfl_up(pieces_to, o);
        if (lane >= o) {
            rounds_to += a;
            pieces_to += b;
        }
    }
    if (lane == 63) {
        s.sums[wave][0] = rounds_to;
        s.sums[wave][1] = pieces_to;
    }
    __syncthreads();
    uint32_t all_rounds = 0, all_pieces = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w == wave) {
            rounds_to += all_rounds;
            pieces_to += all_pieces;
        }
        all_rounds += s.sums[w][0];
        all_pieces += s.sums[w][1];
    }
    const Sharing sh = sharing(uniform(all_rounds) * p.heads, uniform(all_pieces) * p.heads, kLeastRounds, gridDim.x);
    Cursor at = {};
    at.x = blockIdx.x * sh.share;
    if (at.x >= sh.total) return;
    at.left = min(sh.share, sh.total - at.x);
    {
        const bool cut = sh.unit > 1;
        const uint32_t mine = cut ? pieces * kLeastRounds : rounds;
        uint32_t from = ((cut ? pieces_to * kLeastRounds : rounds_to) - mine) * p.heads;
        if (at.x >= from && at.x - from < mine * p.heads) {
            for (uint32_t i = 0; i < each; ++i) {
                const uint32_t b = tid * each + i, one = places(rounds_of(length_of(p.positions[b])), sh.unit);
                if (at.x - from < one * p.heads) {
                    s.start[0] = b;
                    s.start[1] = (at.x - from) / one;
                    s.start[2] = (at.x - from) % one;
                    break;
                }
                from += one * p.heads;
            }
        }
    }
    __syncthreads();
    at.b = uniform(s.start[0]);
    at.head = uniform(s.start[1]);
    at.off = uniform(s.start[2]);
    const uint32_t window = each == 1 ? 0 : at.b;  // s.lengths holds the requests from here on
    if (each > 1) {
        s.lengths[tid] = window + tid < p.batch ? length_of(p.positions[window + tid]) : 0;
        __syncthreads();
    }
    auto request_length = [&](uint32_t b) {
        return b - window < kWindow ? uniform(s.lengths[b - window]) : uniform(length_of(p.positions[b]));
    };

    // ---- the wave's stages, in the order of the share ------------------------------------------
    Cursor ahead = at;
    Run run = {};
    uint32_t run_length = 0, round = 0;
    int32_t run_index = -1;
    auto next_stage = [&]() {
        ++round;
        while (true) {
            const uint32_t key0 = (round * kWaves + wave) * S::keys;
            if (run_index >= 0 && round < run.hi && key0 < run_length) return Stage{run.b, run.head, run_length, key0, run_index};
            if (ahead.left == 0) return Stage{0u, 0u, 1u, 0u, -1};
            run_length = request_length(ahead.b);
            run = next_run(ahead, rounds_of(run_length), p.heads, sh);
            round = run.lo;
            ++run_index;
        }
    };
    const uint32_t ring = uniform(lds_at(&s.ring[wave][0][0]));
    const uint32_t ids = uniform(lds_at(&s.ids[wave][0][0]));
    const uint32_t maskw = MASK ? uniform(lds_at(&s.maskw[wave][0][0])) : 0u;
    const int mask_size = !MASK ? 0 : p.mask_dtype == Q3T_F32 ? 4 : p.mask_dtype == Q3T_BOOL ? 1 : 2;
    // page numbers of a stage's keys; past the request's end its last key's
    auto load_ids = [&](const Stage &st, uint32_t n) {
        const uint32_t key = min(st.key0 + lane, st.length - 1);
        const uint64_t from = reinterpret_cast<uint64_t>(p.table + (int64_t)st.b * p.table_sb + divide(key, p.by_page));
        if (lane < S::keys) load_lds4(from, uniform(ids + (n & 3) * S::keys * 4));
    };
    auto mask_byte = [&](uint32_t b, uint32_t key) { return ((int64_t)b * p.m_sb + (int64_t)key * p.m_st) * mask_size; };
    auto load_stage = [&](const Stage &st, uint32_t n) {
        if constexpr (MASK) {
            const uint32_t key = min(st.key0 + lane, st.length - 1);
            const uint64_t from = (reinterpret_cast<uint64_t>(p.mask) + (uint64_t)mask_byte(st.b, key)) & ~(uint64_t)3;
            if (lane < S::keys) load_lds4(from, uniform(maskw + (n & 1) * S::keys * 4));
        }
        const uint32_t h = st.head / p.blocks, base = uniform(ring + (n & 1) * S::stage);
        const uint64_t kh = (uint64_t)h * p.kp_sh, vh = (uint64_t)h * p.vp_sh;
        uint64_t kf[S::loads], vf[S::loads];
#pragma unroll
        for (int i = 0; i < S::loads; ++i) {
            const int r = (i * 64 + lane) / S::chunks, slot = (i * 64 + lane) % S::chunks;
            const uint32_t key = min(st.key0 + r, st.length - 1), at_row = key - divide(key, p.by_page) * p.by_page.d;
            int32_t id = *(Q3T_LDS const int32_t *)(uintptr_t)(ids + ((n & 3) * S::keys + r) * 4);
            if ((uint32_t)id >= p.pages) id = 0;  // a key on no page: not looked at
            const uint64_t ko = (uint64_t)(uint32_t)id * p.kp_sp + (uint64_t)at_row * p.kp_st + kh;
            const uint64_t vo = (uint64_t)(uint32_t)id * p.vp_sp + (uint64_t)at_row * p.vp_st + vh;
            kf[i] = reinterpret_cast<uint64_t>(p.kp) + (ko + (uint32_t)(slot ^ S::key_swizzle(r))) * 16 - 1024 * (i & 3);
            vf[i] = reinterpret_cast<uint64_t>(p.vp) + (vo + (uint32_t)(slot ^ S::value_swizzle(r))) * 16 - 1024 * (i & 3);
        }
#pragma unroll
        for (int i = 0; i < S::loads; i += 4) load_rows(kf + i, base + i * 1024, p.stream);
#pragma unroll
        for (int i = 0; i < S::loads; i += 4) load_rows(vf + i, base + (S::loads + i) * 1024, p.stream);
    };
    // the query rows of a pair, by the last wave, into one of two places
    auto columns_of = [&](uint32_t head) { return min((uint32_t)kColumns, p.group - head % p.blocks * kColumns); };
    auto first_head = [&](uint32_t head) { return head / p.blocks * p.group + head % p.blocks * kColumns; };
    const uint32_t shared = uniform(lds_at(s.shared));
    auto load_query = [&](uint32_t b, uint32_t head, uint32_t place) {
        const uint32_t items = columns_of(head) * S::chunks;
        for (uint32_t i = 0; i < items; i += 64) {
            const uint32_t item = i + lane;
            const uint64_t from = reinterpret_cast<uint64_t>(p.q) + (uint64_t)((int64_t)b * p.q_sb) +
                                  (uint64_t)((int64_t)(first_head(head) + item / S::chunks) * p.q_sh) + item % S::chunks * 16;
            if (item < items) load_lds16(from, uniform(shared + (place * p.columns * S::chunks + i) * 16));
        }
    };

    Stage s0 = next_stage(), s1 = s0.run < 0 ? s0 : next_stage(), s2 = s1.run < 0 ? s1 : next_stage();
    if (wave == kWaves - 1) load_query(at.b, at.head, 0);
    if (s0.run >= 0) load_ids(s0, 0);
    if (s1.run >= 0) load_ids(s1, 1);
    if (s2.run >= 0) load_ids(s2, 2);
    wait_loads<0>();
    if (s0.run >= 0) load_stage(s0, 0);
    lds_barrier();  // the first query rows are there

    // ---- run by run -----------------------------------------------------------------------------
    Products x;
    const uint32_t buffer = shared + 2 * p.columns * S::row;  // accumulators of `pass` columns per wave
    const uint32_t pass = min(p.columns, (S::shared - 2 * p.columns * S::row) / (kWaves * D * 4));
    const float unit = MASK ? kLog2e : 1.f;  // scores are natural under a mask, else in log2 units
    const float threshold = MASK ? Products::threshold / kLog2e : Products::threshold;
    float m, l;
    uint32_t n = 0;
    auto score = [&](const Stage &st) {
        const uint32_t keys = ring + (n & 1) * S::stage, rows = keys + S::keys * S::row;
        float v[S::keys / 16][4];
        bool hidden[S::keys / 16][4], any = false;
#pragma unroll
        for (int t = 0; t < S::keys / 16; ++t) {
            const U4 id = lds_read16(ids + ((n & 3) * S::keys + 16 * t + 4 * g) * 4);
            const uint32_t page[4] = {id.x, id.y, id.z, id.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t key = st.key0 + 16 * t + 4 * g + i;
                hidden[t][i] = key >= st.length || page[i] >= p.pages;
                if constexpr (MASK) {
                    const uint32_t low = (uint32_t)(reinterpret_cast<uint64_t>(p.mask) + (uint64_t)mask_byte(st.b, min(key, st.length - 1))) & 3u;
                    const uint32_t word = *(Q3T_LDS const uint32_t *)(uintptr_t)(maskw + ((n & 1) * S::keys + 16 * t + 4 * g + i) * 4);
                    v[t][i] = mask_term(word, low, p.mask_dtype);
                    hidden[t][i] = hidden[t][i] || v[t][i] == -INFINITY;
                }
                any = any || hidden[t][i];
            }
        }
        if (__builtin_amdgcn_ballot_w64(any)) {
            const U4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int t = 0; t < S::keys / 16; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (hidden[t][i])
                        for (int chunk = c; chunk < S::chunks; chunk += 16) lds_write16(rows + (16 * t + 4 * g + i) * S::row + chunk * 16, zero);
            asm volatile("" ::: "memory");
        }
        float highest = -INFINITY;
#pragma unroll
        for (int t = 0; t < S::keys / 16; ++t) {
            const f32x4_t st4 = x.scores(keys, t, g, c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float scaled = MASK ? st4[i] * p.scale + v[t][i] : st4[i] * p.scale;
                v[t][i] = hidden[t][i] ? -INFINITY : scaled;
                highest = fmaxf(highest, v[t][i]);
            }
        }
        if (__builtin_amdgcn_ballot_w64(highest > m + threshold)) {
            highest = fmaxf(highest, xor16(highest));
            highest = fmaxf(highest, xor32(highest));
            highest = fmaxf(highest, m);
            const float alpha = fexp2((m - (highest == -INFINITY ? 0.f : highest)) * unit);
            l *= alpha;
            x.rescale(alpha);
            m = highest;
        }
        const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int t = 0; t < S::keys / 16; ++t) {
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = fexp2((v[t][i] - from) * unit + Products::shift);
            l += (w[0] + w[1]) + (w[2] + w[3]);
            x.values(rows, t, g, c, w);
        }
    };
    auto finish = [&](const Run &r, uint32_t column, uint32_t d, float sum, const float (&a)[4]) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = sum == 0.f ? 0.f : a[i] / sum;
        store_out<T>(p.out + (int64_t)r.b * p.o_sb + (int64_t)(first_head(r.head) + column) * p.o_sh + d * sizeof(T), y, p.vec_out);
    };
    // what a state weighs against a maximum
    auto weight = [&](float mine, float highest) { return fexp2((mine - (highest == -INFINITY ? 0.f : highest)) * unit); };
    const uint32_t state_size = p.columns * (D + 2);

    for (int32_t index = 0; at.left > 0; ++index) {
        const Run r = next_run(at, rounds_of(request_length(at.b)), p.heads, sh);
        const uint32_t columns = columns_of(r.head);
        if (wave == kWaves - 1 && at.left > 0) load_query(at.b, at.head, (index + 1) & 1);
        x.load_query(shared + (index & 1) * p.columns * S::row, g, c, (uint32_t)c < columns);
        x.clear();
        m = -INFINITY;
        l = 0.f;
        if (s0.run != index) wait_loads<0>();  // no stage here: the next query rows may be in flight
        while (s0.run == index) {
            const Stage now = s0;
            if (s1.run >= 0) {
                // the next stage, into the slot that was scored last, once its reads have returned
                const Stage s3 = s2.run < 0 ? s2 : next_stage();
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                load_ids(s3.run < 0 ? s1 : s3, n + 3);  // (always, so that the loads behind the stage can be counted)
                load_stage(s1, n + 1);
                wait_loads<LOADS + 1 + (MASK ? 1 : 0)>();
                s0 = s1;
                s1 = s2;
                s2 = s3;
            } else {
                wait_loads<0>();
                s0 = s1;
            }
            score(now);
            ++n;
        }

        // the waves' states into one, `pass` columns at a time
        l += xor16(l);
        l += xor32(l);
        if (g == 0) {
            s.ml[wave][c][0] = m;
            s.ml[wave][c][1] = l;
        }
        const bool whole = r.parts == 1;
        float *state = p.states + (2 * blockIdx.x + r.begins) * (uint64_t)state_size;
        for (uint32_t c0 = 0; c0 < columns; c0 += pass) {
            const uint32_t count = min(pass, columns - c0);
            if (c >= c0 && c < c0 + count) x.store(buffer + (wave * pass + c - c0) * D * 4, g);
            lds_barrier();
            for (uint32_t item = tid; item < count * (D / 4); item += kThreads) {
                const uint32_t column = c0 + item / (D / 4), d = item % (D / 4) * 4;
                float highest = -INFINITY, sum = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < kWaves; ++w) highest = fmaxf(highest, s.ml[w][column][0]);
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    const float e = weight(s.ml[w][column][0], highest);
                    const f32x4_t part = __builtin_bit_cast(f32x4_t, lds_read16(buffer + ((w * pass + column - c0) * D + d) * 4));
                    sum += s.ml[w][column][1] * e;
#pragma unroll
                    for (int i = 0; i < 4; ++i) a[i] += part[i] * e;
                }
                if (whole) {
                    finish(r, column, d, sum, a);
                } else {
                    publish(state + column * D + d, a[0], a[1]);
                    publish(state + column * D + d + 2, a[2], a[3]);
                    if (d == 0) publish(state + p.columns * D + 2 * column, highest, sum);
                }
            }
            if (!whole && c0 + pass >= columns) wait_loads<0>();  // the state has been stored
            lds_barrier();
        }
        if (whole) continue;

        int32_t *counter = p.counters + r.b * p.heads + r.head;
        if (tid == 0) s.start[3] = (uint32_t)__hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (uniform(s.start[3]) != r.parts - 1) continue;
        // the last to arrive: thread (part % groups, item) takes every groups-th part's four elements
        const uint32_t items = columns * (D / 4), groups = max(1u, kThreads / items);
        for (uint32_t first = 0; first < items; first += kThreads) {
            const uint32_t item = first + tid % items, group = groups == 1 ? 0 : tid / items;
            const bool live = groups == 1 ? first + tid < items : group < groups;
            const uint32_t own = groups == 1 ? first + tid : item, column = own / (D / 4), d = own % (D / 4) * 4;
            float highest = -INFINITY, sum = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
            if (live) {
                for (uint32_t i = group; i < r.parts; i += groups) {
                    const float *from = p.states + (2 * (r.first + i) + (i == 0)) * (uint64_t)state_size;
                    float pm, pl, v[4];
                    collect(from + p.columns * D + 2 * column, pm, pl);
                    collect(from + column * D + d, v[0], v[1]);
                    collect(from + column * D + d + 2, v[2], v[3]);
                    const float top = fmaxf(highest, pm), e0 = weight(highest, top), e1 = weight(pm, top);
                    sum = sum * e0 + pl * e1;
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[j] = a[j] * e0 + v[j] * e1;
                    highest = top;
                }
            }
            if (groups == 1) {
                if (live) finish(r, column, d, sum, a);
                continue;
            }
            const uint32_t mine = buffer + tid * 16, mine_ml = buffer + kThreads * 16 + tid * 8;
            if (live) {
                lds_write16(mine, U4{__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]), __float_as_uint(a[3])});
                *(Q3T_LDS float *)(uintptr_t)mine_ml = highest;
                *(Q3T_LDS float *)(uintptr_t)(mine_ml + 4) = sum;
            }
            lds_barrier();
            if (live && group == 0) {
                for (uint32_t o = 1; o < groups; ++o) {
                    const uint32_t from = buffer + o * items * 16 + tid * 16, ml = buffer + kThreads * 16 + o * items * 8 + tid * 8;
                    const f32x4_t v = __builtin_bit_cast(f32x4_t, lds_read16(from));
                    const float pm = *(Q3T_LDS const float *)(uintptr_t)ml, pl = *(Q3T_LDS const float *)(uintptr_t)(ml + 4);
                    const float top = fmaxf(highest, pm), e0 = weight(highest, top), e1 = weight(pm, top);
                    sum = sum * e0 + pl * e1;
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[j] = a[j] * e0 + v[j] * e1;
                    highest = top;
                }
                finish(r, column, d, sum, a);
            }
        }
        if (tid == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        lds_barrier();  // the buffer is free again
    }
}

template <typename T, int D>
struct Launch {
    static int64_t workgroups(const q3t_paged_args *a, int64_t pairs) {
        const int64_t rounds = (a->ctx + Shape<T, D>::round - 1) / Shape<T, D>::round;
        const int64_t pieces = pairs * ((rounds + kLeastRounds - 1) / kLeastRounds), most = 256 * Shape<T, D>::per_cu;
        return pieces < most ? pieces : most;
    }
    static int64_t rounds(const q3t_paged_args *a, int64_t pairs) { return pairs * ((a->ctx + Shape<T, D>::round - 1) / Shape<T, D>::round); }
    static void run(const Params &p, uint32_t blocks, hipStream_t s) {
        if (p.mask) hipLaunchKernelGGL((paged_kernel<T, D, true>), dim3(blocks), dim3(kThreads), 0, s, p);
        else hipLaunchKernelGGL((paged_kernel<T, D, false>), dim3(blocks), dim3(kThreads), 0, s, p);
    }
};
// f on the Launch of a call's type and width
template <typename F>
static auto with(const q3t_paged_args *a, F f) {
    const bool wide = a->head_dim == 128;
    if (a->dtype == Q3T_F32) return wide ? f(Launch<float, 128>{}) : f(Launch<float, 64>{});
    if (a->dtype == Q3T_BF16) return wide ? f(Launch<__bf16, 128>{}) : f(Launch<__bf16, 64>{});
    return wide ? f(Launch<_Float16, 128>{}) : f(Launch<_Float16, 64>{});
}

struct Sizes {
    int64_t group, blocks, pairs, columns, workgroups, workspace;
};

// The sizes of a launch; Q3T_OK, or the status to return.
static int sizes_of(const q3t_paged_args *a, Sizes &z) {
    if (!a || a->batch < 0 || a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads || a->ctx < 1 || a->pages < 1 ||
        a->page_size < 1 || a->table_width < 1)
        return Q3T_EINVAL;
    if (a->dtype != Q3T_BF16 && a->dtype != Q3T_F16 && a->dtype != Q3T_F32) return Q3T_EUNSUPPORTED;
    if (a->head_dim != 64 && a->head_dim != 128) return Q3T_EUNSUPPORTED;
    if (a->pages > INT32_MAX || a->page_size > INT32_MAX || a->table_width > INT32_MAX) return Q3T_EUNSUPPORTED;
    if (a->ctx > a->table_width * a->page_size) return Q3T_EINVAL;
    if (a->ctx >= 1 << 30 || a->batch > kCounters || a->q_heads > 1 << 16) return Q3T_EUNSUPPORTED;
    z.group = a->q_heads / a->kv_heads;
    z.blocks = (z.group + kColumns - 1) / kColumns;
    z.pairs = a->batch * a->kv_heads * z.blocks;
    z.columns = z.group < kColumns ? z.group : kColumns;
    if (z.pairs > kCounters) return Q3T_EUNSUPPORTED;  // a counter each
    if (with(a, [&](auto l) { return l.rounds(a, z.pairs); }) >= INT32_MAX - kCounters) return Q3T_EUNSUPPORTED;
    z.workgroups = with(a, [&](auto l) { return l.workgroups(a, z.pairs); });
    z.workspace = kCounters * 4 + 2 * z.workgroups * z.columns * (a->head_dim + 2) * 4;
    return Q3T_OK;
}

}  // namespace paged
}  // namespace q3t

using namespace q3t;

extern "C" int64_t q3t_paged_workspace_bytes(const q3t_paged_args *a) {
    paged::Sizes z;
    return paged::sizes_of(a, z) == Q3T_OK ? z.workspace : -1;
}

extern "C" int q3t_paged_attention(const q3t_paged_args *a, void *stream) {
    using namespace paged;
    Sizes z;
    const int status = sizes_of(a, z);
    if (status != Q3T_OK) return status;
    if (a->batch == 0) return Q3T_OK;
    if (!a->query || !a->key_pages || !a->value_pages || !a->page_table || !a->positions || !a->out) return Q3T_EINVAL;
    if (a->mask && (a->mask_dtype < Q3T_BF16 || a->mask_dtype > Q3T_BOOL)) return Q3T_EINVAL;
    const int64_t es = a->dtype == Q3T_F32 ? 4 : 2;
    auto chunks = [&](int64_t stride, uint32_t &to) {  // a stride of whole 16-byte chunks
        if (stride < 0 || stride * es % 16) return Q3T_EINVAL;
        if (stride > (int64_t)UINT32_MAX * 16 / es) return Q3T_EUNSUPPORTED;
        to = (uint32_t)(stride * es / 16);
        return Q3T_OK;
    };
    Params p = {};
    const int64_t strides[6] = {a->kp_stride_p, a->kp_stride_h, a->kp_stride_t, a->vp_stride_p, a->vp_stride_h, a->vp_stride_t};
    uint32_t *const to[6] = {&p.kp_sp, &p.kp_sh, &p.kp_st, &p.vp_sp, &p.vp_sh, &p.vp_st};
    for (int i = 0; i < 6; ++i) {
        const int s = chunks(strides[i], *to[i]);
        if (s != Q3T_OK) return s;
    }
    p.q = (const char *)a->query; p.kp = (const char *)a->key_pages; p.vp = (const char *)a->value_pages;
    p.mask = (const char *)a->mask; p.out = (char *)a->out;
    p.table = a->page_table; p.positions = a->positions;
    p.q_sb = a->q_stride_b * es; p.q_sh = a->q_stride_h * es;
    p.o_sb = a->o_stride_b * es; p.o_sh = a->o_stride_h * es;
    p.m_sb = a->mask_stride_b; p.m_st = a->mask_stride_t; p.table_sb = a->table_stride_b;
    const int64_t mask_size = a->mask_dtype == Q3T_F32 ? 4 : a->mask_dtype == Q3T_BOOL ? 1 : 2;
    if ((p.q_sb | p.q_sh) % 16 || !aligned(p.q, 16) || !aligned(p.kp, 16) || !aligned(p.vp, 16) || !aligned(p.out, es) ||
        !aligned(p.table, 4) || !aligned(p.positions, 8) || (p.mask && !aligned(p.mask, mask_size)))
        return Q3T_EINVAL;
    if (!a->workspace || a->workspace_bytes < z.workspace) return Q3T_EWORKSPACE;
    if (!aligned(a->workspace, 16)) return Q3T_EINVAL;
    p.counters = (int32_t *)a->workspace;
    p.states = (float *)((char *)a->workspace + kCounters * 4);
    p.ctx = (int32_t)a->ctx; p.mask_dtype = (int32_t)a->mask_dtype;
    p.stream = 1;
    p.vec_out = aligned(p.out, 4 * es) && (p.o_sb | p.o_sh) % (4 * es) == 0;
    p.batch = (uint32_t)a->batch; p.pages = (uint32_t)a->pages;
    p.group = (uint32_t)z.group; p.blocks = (uint32_t)z.blocks;
    p.heads = (uint32_t)(a->kv_heads * z.blocks);
    p.columns = (uint32_t)z.columns;
    p.by_page = divisor((uint32_t)a->page_size);
    p.scale = a->mask ? a->scale : a->scale * kLog2e;
    with(a, [&](auto l) { l.run(p, (uint32_t)z.workgroups, (hipStream_t)stream); });
    return launch_status();
}
