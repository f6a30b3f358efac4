// Attention of one new token per request over a cache kept in pages (the paged counterpart of the
// decode attention; reference: packed_attention.py:75-84).
//
//   s_j = scale q . k_j (+ mask_j),  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// in one pass over the keys, with a running maximum m that moves when it is passed by more than a
// threshold.  Every key and value row is read once for 16 query heads of its KV head, so HBM bounds a launch of
// many keys (2 to 16 operations per byte), and the chain arguments - positions - page numbers - rows - merge one of few.
// us per launch in a graph, rows not in the caches (TB/s of them): 128 requests of 100..4095 keys, 8 KV heads of
// 128, bf16 175 (6.0, the rate of a large read); 64 of 64..1023 30.7 (4.9); one of 65000, 4 heads, fp16 32.7 (4.1);
// 32 of 30..2047 under a mask, 4 heads 22.3 (3.3); 21 of 1..700 in float32 under a mask, 12 heads of 64 18.0
// (3.1); one of 300 7.6.  The first rows are there after 5.8 us.
// float32 rows of 128: 64 of 64..1023 54.0 (5.5), 128 of 100..2000 192 (5.9), one of 30000 49.3 (5.0), one of 300
// 11.6.  Pages that hold no whole stages: 128 of 100..2000 in bf16 in pages of 16 / 24 / 100 96.0 / 101 / 98.7.
// Each further block of 16 query heads of a KV head reads that head's rows again, from memory: 64 requests of 2000
// keys, 2 KV heads of 128 in bf16, with 16 / 20 / 32 / 48 query heads each 30.3 / 47.4 / 46.8 / 67.6 us (135 / 263 / 264 /
// 381 MB fetched); 8 requests of 4000 18.2 / 19.1 / 19.6 / 25.9.
//   * Work: a workgroup takes an equal share of the stages of all (request, KV head) pairs
//     (paged_index.hpp), whatever the requests' lengths; its waves find their place by adding up all
//     requests' stages.  A pair that lies in several shares leaves its parts' states in the
//     workspace, and the workgroup that arrives last merges them, in the parts' order.
//     Where no pair can have more than one share a workgroup takes the pair of its own number, and its page
//     numbers are on their way together with the position.
//   * Of a run of a pair's stages of 16 (rows of 128 bytes: 32) keys each of the workgroup's W waves takes
//     every W-th.  A stage's rows go straight from memory to the wave's own two LDS slots, one stage
//     ahead of the one that is scored, over the ends of runs: no barrier but where a run ends.  The
//     page numbers of up to 64 stages come the same way, while the stages before them are read.
//     Where pages hold whole stages the rows are one range of memory; for other page sizes each lane works out
//     the address of its own row.  In pages of halves of a stage of 32 (16 rows of 128 bytes each) they are two
//     ranges where a pair has a workgroup to itself, and single rows elsewhere, where ranges gain nothing (us, rows /
//     ranges, 64 columns in fp16, pages of 16: 128 requests of 100..4000 keys 89.7 / 90.2, 64 of 64..2047 32.8 / 33.0, 200 of
//     10..400 25.8 / 26.1).
//   * The rows of a KV head's query heads are the columns of 16x16 products, S^T = K . Q^T and
//     O^T += V^T . P^T.  The matrix cores idle (under a twentieth of their rate), so the weights are
//     not rounded to the cache's type: bf16 weights go in three parts (all 24 bits of their
//     float32), fp16 ones in two (22 bits), float32 is multiplied as such.  The first part has
//     accumulators of its own: an infinite value times a remainder of zero would be NaN.
//   * A key that does not exist (past the request's end, under a mask's minus infinity, on no page)
//     scores minus infinity, and its value row is zeroed in LDS: zero times NaN would be NaN.
#include "paged_index.hpp"
#include "q3t_common.hpp"

#include <type_traits>

namespace q3t {
namespace paged {

constexpr int kColumns = 16;           // query heads of a workgroup: columns of a product
// Stages that are not shared out, as a power of two: two of each wave; all of a pair that a workgroup has to
// itself (below).  us with 4 / 8 / 16 for four waves: one request of 4000 keys 13.4 / 12.9 / -, 4 of 300..1000 11.3 /
// 10.8 / -, 3 of 5000..9000 with one KV head 22.5 / 20.8 / 20.8, 8 of 100..2000 14.0 / 14.0 / 15.0; with 16 / 32 for
// eight: one of 1000 with one KV head and 16 others 11.8 / 13.7.
constexpr uint32_t kLogLeast4 = 3, kLogLeast8 = 4, kLogLeastSingle = 6;
// Stages that the end of a run of W waves costs as much as.  us with 1 / 8 / 24 for four waves: 200 requests of
// 10..400 keys 44 / 27.2 / 28.3, 128 of 32..511 42 / 32.9 / 34.6; with 8 / 16 / 24 for eight: 64 of 64..1023
// 31.6 / 30.8 / 31.2, 128 of 100..4095 174.8 / 174.4 / 176.2.
constexpr uint32_t run_cost(int waves) { return 2 * waves; }
constexpr int kCounters = 65536;       // counter words in front of a decode workspace: of the pairs,
constexpr int kPairs = kCounters - 1024;  // then of the state slots, two for each of up to 512 workgroups
// Parts that are merged in one step.  us with 4 / 16 / all: one request of 65000 keys 35.6 / 33.9 / 49.4, 8 of
// 100..2000 15.9 / 14.0 / 14.1.
constexpr uint32_t kTogether = 16;
constexpr float kLog2e = 1.4426950408889634f;

struct Params {
    const char *q, *kp, *vp, *mask;
    char *out;
    const int32_t *table;
    int32_t *counters;
    float *states;
    uint32_t q_sb, q_sh, kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st;  // 16 bytes
    uint32_t o_sb, o_sh, m_sb, m_st, table_sb;                      // elements
    int32_t mask_dtype, vec_out;
    uint32_t pages, group, heads, blocks;       // heads: pairs of a request; blocks: of a KV head
    uint32_t columns, log_least;                       // of a state; of eight waves
    Divisor by_page, by_grid;
    float scale;                                       // unmasked: times log2(e)
};

template <typename T, int D>
struct Shape {
    static constexpr int row = D * (int)sizeof(T);
    static constexpr int chunks = row / 16;                // 16-byte chunks of a row
    static constexpr int keys = row == 128 ? 32 : 16;      // of a wave's stage
    static constexpr int stage = 2 * keys * row;           // key rows, then value rows
    static constexpr int loads = keys * row / 1024;        // 1 KiB loads of either
    static constexpr int log_keys = keys == 32 ? 5 : 4;
    static constexpr bool f32 = sizeof(T) == 4;
    static_assert(kColumns * D * 4 <= stage, "a free slot holds a wave's accumulators");
    // chunk c of key (value) row r sits at c ^ swizzle: the products' reads meet distinct banks
    static Q3T_DEVICE int key_swizzle(int r) { return chunks == 8 ? (r >> 1) & 7 : r & 15; }
    static Q3T_DEVICE int value_swizzle(int r) { return f32 ? 0 : chunks == 8 ? (2 * (r >> 1)) & 7 : (2 * r) & 15; }
};

// Workgroups of W waves, as many as fit the LDS of 256 CUs.
template <typename T, int D, int W> struct Workgroups {
    static constexpr int per_cu = 2 * W * Shape<T, D>::stage > 64 * 1024 ? 1 : 2;
    static constexpr int count = 256 * per_cu;
};

template <typename T, int D, bool MASK, int W>
struct Lds {
    alignas(1024) char ring[W][2][Shape<T, D>::stage];
    alignas(16) char query[2][kColumns * Shape<T, D>::row];  // of this run's pair and the next's
    uint32_t ids[W][2][64];
    alignas(16) uint32_t maskw[MASK ? W : 1][2][MASK ? Shape<T, D>::keys : 4];
    float ml[W][kColumns][2];
    uint32_t slot[W];  // each wave's free slot
    uint32_t there;    // the count of a pair of two parts, ahead of the waves' merge
    uint32_t count;    // parts that have arrived
};

#define Q3T_LDS __attribute__((address_space(3)))
#define Q3T_GLOBAL __attribute__((address_space(1)))
Q3T_DEVICE uint32_t lds_at(const void *x) { return (uint32_t)(uintptr_t)(Q3T_LDS const char *)x; }
Q3T_DEVICE uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

// Four 16-byte loads per lane into LDS, 1 KiB apart there: the instructions' offsets move both
// addresses, so load i's address is 1024 i short of its row.
#define Q3T_LOAD4(OPCODE, ADDRESS, POLICY, ...)                                                    \
    asm volatile("s_mov_b32 m0, %0\n\t" Q3T_VMEM_SGPR_WAIT                                         \
                 OPCODE " %1, " ADDRESS POLICY "\n\t"                                              \
                 OPCODE " %2, " ADDRESS " offset:1024" POLICY "\n\t"                               \
                 OPCODE " %3, " ADDRESS " offset:2048" POLICY "\n\t"                               \
                 OPCODE " %4, " ADDRESS " offset:3*1024" POLICY                                      \
                 :: "s"(base), "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]) __VA_ARGS__ : "memory", "m0")
// Rows are read once: the non-temporal policy (64 requests of 64..1023 keys without it 35.1 us, with it 32.8;
// 128 of 100..4095 194.9, 176.2).  From a pointer per lane:
Q3T_DEVICE void load_rows(const uint64_t *p, uint32_t base) { Q3T_LOAD4("global_load_lds_dwordx4", "off", " nt"); }
// from an offset per lane into a resource; past its range zeros are written without a memory access: four
// loads, or two
#define Q3T_RSRC , "s"(rsrc)
Q3T_DEVICE void load_rows(i32x4_t rsrc, const uint32_t *p, uint32_t base) {
    Q3T_LOAD4("buffer_load_dwordx4", "%5, 0 offen", " nt lds", Q3T_RSRC);
}
Q3T_DEVICE void load_half(i32x4_t rsrc, const uint32_t *p, uint32_t base) {
    asm volatile("s_mov_b32 m0, %0\n\t" Q3T_VMEM_SGPR_WAIT
                 "buffer_load_dwordx4 %1, %3, 0 offen nt lds\n\t"
                 "buffer_load_dwordx4 %2, %3, 0 offen offset:1024 nt lds"
                 :: "s"(base), "v"(p[0]), "v"(p[1]), "s"(rsrc) : "memory", "m0");
}
#undef Q3T_RSRC
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
Q3T_DEVICE f32x2_t collect(const float *p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return f32x2_t{__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))};
}

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// LDS reads above are issued before anything below: left alone, the compiler waits for each one alone.
Q3T_DEVICE void together() { __builtin_amdgcn_sched_barrier(0); }

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
    static Q3T_DEVICE float visible(float w) { return w; }
    static Q3T_DEVICE uint32_t round2(float a, float b) { return cvt_pk_bf16(a, b); }
    static Q3T_DEVICE float lo(uint32_t x) { return bf16_lo(x); }
    static Q3T_DEVICE float hi(uint32_t x) { return bf16_hi(x); }
    static Q3T_DEVICE uint32_t store2(float a, float b) { return cvt_pk_bf16_canon(a, b); }
};
// fp16 weights are kept 2^8 larger than exp(s - m), so that small ones keep their bits, and stay
// below 2^14 with the smaller threshold.  The first part is 2^-24, fp16's smallest, at least: an infinite value
// under a weight that rounds to zero is an infinity of the output, as the definition has it, where zero times it
// would be NaN.  The second part takes it off again (a key adds 2^-32 of its value's size to the error at most; the
// value rows of hidden keys are zeros).  us without / with it: 64 requests of 64..1023 keys 30.6 / 30.5, 200 of
// 10..400, 64 columns 25.9 / 26.2.
template <> struct Half<_Float16> {
    static constexpr int parts = 2;
    static constexpr float shift = 8.f, threshold = 6.f;
    static Q3T_DEVICE f32x4_t scores(const U4 &k, const U4 &q, f32x4_t s) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, k), __builtin_bit_cast(f16x8_t, q), s, 0, 0, 0);
    }
    static Q3T_DEVICE f32x4_t values(uint2 v, uint2 p, f32x4_t a) {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_t, v), __builtin_bit_cast(f16x4_t, p), a, 0, 0, 0);
    }
    static Q3T_DEVICE float visible(float w) { return fmaxf(w, 0x1p-24f); }
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
    uint32_t key_at[D / 32], value_at[D / 16];  // the lane's places in a stage's first 16 rows (the swizzles repeat every 16)

    Q3T_DEVICE void place(uint32_t ring, int g, int c) {
        const int r = 4 * g + (c >> 2);
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) key_at[kk] = ring + c * S::row + (((4 * kk + g) ^ S::key_swizzle(c)) & (S::chunks - 1)) * 16;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
            value_at[d] = ring + (S::keys + r) * S::row + (((2 * d + ((c >> 1) & 1)) ^ S::value_swizzle(r)) & (S::chunks - 1)) * 16 + 8 * (c & 1);
    }
    // tile t of the stage at byte `stage` of the ring
    Q3T_DEVICE f32x4_t scores(uint32_t stage, int t) const {
        U4 k[D / 32];
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) k[kk] = lds_read16(key_at[kk] + stage + t * 16 * S::row);
        together();
        f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) s = Half<T>::scores(k[kk], q[kk], s);
        return s;
    }
    uint2 v[D / 16];  // the next value fragments
    Q3T_DEVICE void read_values(uint32_t stage, int t) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) v[d] = lds_read_tr16(value_at[d] + stage + t * 16 * S::row);
        together();
    }
    Q3T_DEVICE void values(const float (&w)[4]) {
        uint2 part[3];
        float x[4] = {w[0], w[1], w[2], w[3]};
#pragma unroll
        for (int i = 0; i < Half<T>::parts; ++i) {
            auto kept = [&](int k) { return i == 0 ? Half<T>::visible(x[k]) : x[k]; };
            part[i] = uint2{Half<T>::round2(kept(0), kept(1)), Half<T>::round2(kept(2), kept(3))};
            x[0] -= Half<T>::lo(part[i].x);
            x[1] -= Half<T>::hi(part[i].x);
            x[2] -= Half<T>::lo(part[i].y);
            x[3] -= Half<T>::hi(part[i].y);
        }
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            first[d] = Half<T>::values(v[d], part[0], first[d]);
#pragma unroll
            for (int i = 1; i < Half<T>::parts; ++i) rest[d] = Half<T>::values(v[d], part[i], rest[d]);
        }
    }
    // Elements of column c into its row of D floats, four to a chunk, chunk k at k ^ c.
    Q3T_DEVICE void store(uint32_t to, int g, int c) const {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            f32x4_t x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __builtin_fabsf(first[d][i]) < INFINITY ? first[d][i] + rest[d][i] : first[d][i];
            lds_write16(to + c * D * 4 + ((4 * d + g) ^ c) * 16, __builtin_bit_cast(U4, x));
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
    uint32_t key_at[D / 16], value_at;

    Q3T_DEVICE void place(uint32_t ring, int g, int c) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) key_at[kk] = ring + c * S::row + ((4 * kk + g) ^ S::key_swizzle(c)) * 16;
        value_at = ring + (S::keys + 4 * g) * S::row + c * 16;
    }
    Q3T_DEVICE f32x4_t scores(uint32_t stage, int t) const {
        f32x4_t k[D / 16], s = {0.f, 0.f, 0.f, 0.f}, s2 = s;  // two chains: one waits for its last product
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) k[kk] = read(key_at[kk] + stage + t * 16 * S::row);
        together();
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[kk][e], q[kk][e], s, 0, 0, 0);
                s2 = __builtin_amdgcn_mfma_f32_16x16x4f32(k[kk][e + 1], q[kk][e + 1], s2, 0, 0, 0);
            }
        return s + s2;
    }
    f32x4_t v[D / 16];
    Q3T_DEVICE void read_values(uint32_t stage, int t) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < D / 64; ++j) v[i * (D / 64) + j] = read(value_at + stage + (16 * t + i) * S::row + j * 256);
        together();
    }
    Q3T_DEVICE void values(const float (&w)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < D / 64; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[4 * j + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i * (D / 64) + j][e], w[i], acc[4 * j + e], 0, 0, 0);
    }
    Q3T_DEVICE void store(uint32_t to, int g, int c) const {
#pragma unroll
        for (int j = 0; j < D / 64; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4_t x = {acc[4 * j][i], acc[4 * j + 1][i], acc[4 * j + 2][i], acc[4 * j + 3][i]};
                lds_write16(to + c * D * 4 + ((16 * j + 4 * g + i) ^ c) * 16, __builtin_bit_cast(U4, x));
            }
    }
};

// The mask term whose element lies in a word's low bytes.
Q3T_DEVICE float mask_term(uint32_t e, int dtype) {
    switch (dtype) {
        case Q3T_BF16: return bf16_to_float(e & 0xffffu);
        case Q3T_F16: return (float)__builtin_bit_cast(_Float16, (uint16_t)e);
        case Q3T_F32: return __uint_as_float(e);
        default: return e & 0xffu ? 0.0f : -INFINITY;  // bool: true attends
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

// Four elements of a column's softmax state: maximum, sum, weighted values.
struct State {
    float m, l;
    f32x4_t a;
    // Another state's keys added; fused products by name, so that every copy of this code rounds alike.
    Q3T_DEVICE void add(const State &o, float unit) {
        const float top = fmaxf(m, o.m), from = top == -INFINITY ? 0.f : top;
        const float e0 = fexp2((m - from) * unit), e1 = fexp2((o.m - from) * unit);
        l = __builtin_fmaf(l, e0, o.l * e1);
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = __builtin_fmaf(a[i], e0, o.a[i] * e1);
        m = top;
    }
    Q3T_DEVICE void publish(float *to, uint32_t sums, uint32_t column, uint32_t d, int D) const {
        paged::publish(to + column * D + d, a[0], a[1]);
        paged::publish(to + column * D + d + 2, a[2], a[3]);
        if (d == 0) paged::publish(to + sums + 2 * column, m, l);
    }
    Q3T_DEVICE void collect(const float *from, uint32_t sums, uint32_t column, uint32_t d, int D) {
        const f32x2_t ml = paged::collect(from + sums + 2 * column);
        const f32x2_t lo = paged::collect(from + column * D + d), hi = paged::collect(from + column * D + d + 2);
        m = ml[0];
        l = ml[1];
        a = f32x4_t{lo[0], lo[1], hi[0], hi[1]};
    }
};

// Stages of a wave in one run, every W-th from key `key` on below `end`, up to the number of
// stages whose page numbers fit its 64 words.
struct Batch {
    uint32_t b, kv_head, length, key, end;
    int32_t run;  // of the share; -1: none
};
// A wave's stage; bit k of `exists`: key0 + k is a key of the request and on a page.
struct Stage {
    uint32_t b, key0, exists;
    int32_t run;
};

// Sums over the wave's lanes up to and with each lane.
Q3T_DEVICE uint32_t scan(uint32_t x) {
    auto add = [&](auto control, auto rows) {
        x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(control)::value, decltype(rows)::value, 0xf, false);
    };
    add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // from 1, 2, 4 and 8 lanes
    add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});  // below in rows of 16
    add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
    add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // lanes 15 and 47 to the next rows
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // lane 31 to the upper half
    return x;
}

// RANGES: ranges of memory that a stage's rows are in, in pages that hold whole ones; 0: any page size.
// SINGLE: no pair can have more than one share (without the code for others 64 requests of 64 keys take 8.2 us
// instead of 9.0; as a branch of one instance it cost 1024 of 20..200 98 -> 105).
template <typename T, int D, bool MASK, int RANGES, int W, bool SINGLE>
__global__ void __launch_bounds__(64 * W, (W / 4 * Workgroups<T, D, W>::per_cu))
paged_kernel(const int64_t *positions, uint32_t batch, uint32_t ctx, Params p) {
    typedef Shape<T, D> S;
    typedef Tile<T, D> Products;
    constexpr int LOADS = 2 * S::loads, kThreads = 64 * W;
    constexpr bool WHOLE = RANGES > 0;
    constexpr uint32_t kRows = S::keys / (WHOLE ? RANGES : S::keys);  // of a page number
    __shared__ Lds<T, D, MASK, W> s;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int wave = (int)uniform(tid >> 6);

    // ---- the share: every wave adds up all requests' stages and pieces for itself ---------------
    auto length_at = [&](uint32_t b) {
        const int64_t pos = b < batch ? positions[b] : -1;
        return pos >= 0 && pos < (int64_t)ctx ? (uint32_t)pos + 1 : 0u;
    };
    auto stages_of = [&](uint32_t length) { return max(1u, (length + S::keys - 1) >> S::log_keys); };
    const uint32_t log_least = W == 4 ? kLogLeast4 : p.log_least, least = 1u << log_least;
    uint32_t lengths, window = 0;  // of requests window + lane
    Sharing sh;
    Cursor at = {};
    auto find_share = [&]() {
        const uint32_t each = (batch + 63) / 64;  // requests of a lane, one after the other
        uint32_t stages = 0, pieces = 0;
        lengths = length_at(lane);
        auto count = [&](uint32_t r) {
            stages += r;
            pieces += (r + least - 1) >> log_least;
        };
        if (each == 1) {
            if ((uint32_t)lane < batch) count(stages_of(lengths));
        } else {
            constexpr uint32_t kFlight = 8;  // positions on their way at once (4096 requests: one 118 us, eight 116)
            for (uint32_t i = 0; i < each; i += kFlight) {
                uint32_t r[kFlight];
#pragma unroll
                for (uint32_t j = 0; j < kFlight; ++j) r[j] = stages_of(length_at(min(lane * each + i + j, batch - 1)));
#pragma unroll
                for (uint32_t j = 0; j < kFlight; ++j)
                    if (i + j < each && lane * each + i + j < batch) count(r[j]);
            }
        }
        const uint32_t stages_to = scan(stages), pieces_to = scan(pieces);
        auto last_lane = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); };
        sh = sharing(batch * p.heads, last_lane(stages_to) * p.heads, last_lane(pieces_to) * p.heads,
                     least, run_cost(W), p.by_grid);
        at.x = blockIdx.x * sh.share;
        if (at.x >= sh.total) return false;
        at.left = min(sh.share, sh.total - at.x);
        // the lane whose requests hold the share's first place, then the request
        auto holder = [&](uint32_t to, uint32_t &from) {  // `from`: the first place of the lane found
            const uint64_t below = __builtin_amdgcn_ballot_w64(to * p.heads <= at.x - from);
            const int j = __builtin_popcountll(below);
            if (j) from += (uint32_t)__builtin_amdgcn_readlane((int)to, j - 1) * p.heads;
            return (uint32_t)j;
        };
        uint32_t from = 0;
        at.b = holder(sh.unit > 1 ? pieces_to * least : stages_to + sh.cost * min((lane + 1) * each, batch), from);
        if (each > 1) {
            window = at.b * each;
            while (true) {  // (once, for up to 4096 requests)
                lengths = length_at(window + lane);
                const uint32_t j = holder(scan(window + lane < batch ? places(stages_of(lengths), sh) : 0), from);
                at.b = window + j;
                if (j < 64) break;
                window += 64;
            }
        }
        const uint32_t stages_here = stages_of((uint32_t)__builtin_amdgcn_readlane((int)lengths, (int)(at.b - window)));
        const uint32_t length = places(stages_here, sh);
        at.head = (at.x - from) / length;
        at.off = (at.x - from) - at.head * length;
        if (at.off >= stages_here) end_pair(at, length, p.heads);
        at = Cursor{uniform(at.x), uniform(at.left), uniform(at.b), uniform(at.head), uniform(at.off)};
        return at.left > 0;
    };
    if constexpr (SINGLE) {
        constexpr uint32_t kRoom = 1u << kLogLeastSingle;  // holds any such pair's stages
        sh = {kRoom, 0u, kRoom, batch * p.heads * kRoom};
        const uint32_t b = blockIdx.x / p.heads;
        at = Cursor{blockIdx.x * kRoom, kRoom, b, blockIdx.x - b * p.heads, 0u};
        window = b;
        lengths = length_at(b + lane);
    } else if (!find_share()) {
        return;
    }
    auto request_length = [&](uint32_t b) {
        return b - window < 64 ? (uint32_t)__builtin_amdgcn_readlane((int)lengths, (int)(b - window)) : uniform(length_at(b));
    };

    // ---- the wave's stages, in the order of the share ------------------------------------------
    // pairs of a request: the blocks of up to 16 query heads of each KV head
    auto kv_head = [&](uint32_t head) { return p.blocks == 1 ? head : head / p.blocks; };
    Cursor ahead = at;
    int32_t runs = -1;
    constexpr uint32_t kIds = S::keys / kRows;                        // page numbers of a stage
    constexpr uint32_t kStep = W * S::keys, kBatch = 64 / kIds * kStep;  // keys
    Batch batches = {0u, 0u, 0u, 0u, 0u, -1};  // the next one, whose page numbers are on their way
    auto next_batch = [&]() {
        if (batches.key + kBatch < batches.end) {
            batches.key += kBatch;
            return;
        }
        while (ahead.left) {
            const uint32_t length = request_length(ahead.b);
            const Run run = next_run(ahead, stages_of(length), p.heads, sh);
            ++runs;
            batches.b = run.b;
            batches.kv_head = kv_head(run.head);
            batches.length = length;
            batches.key = (run.lo + ((wave - run.lo) & (W - 1))) * S::keys;  // every W-th stage is the wave's
            batches.end = min(run.hi * S::keys, length);
            batches.run = runs;
            if (batches.key < batches.end) return;
        }
        batches = Batch{0u, 0u, 0u, 0u, 0u, -1};
    };
    const uint32_t ring = uniform(lds_at(&s.ring[wave][0][0]));
    const uint32_t ids = uniform(lds_at(&s.ids[wave][0][0]));
    const uint32_t maskw = MASK ? uniform(lds_at(&s.maskw[wave][0][0])) : 0u;
    const uint32_t mask_size = !MASK ? 0 : p.mask_dtype == Q3T_F32 ? 4 : p.mask_dtype == Q3T_BOOL ? 1 : 2;
    // The batch's page numbers: lane i's is that of range (WHOLE) or key i % kIds of stage i / kIds; past the
    // request's end that of its last key.
    auto load_ids = [&](uint32_t half) {
        const uint32_t key = batches.key + lane / kIds * kStep + lane % kIds * kRows;
        const uint32_t at_page = divide(min(key, batches.length - 1), p.by_page);
        load_lds4(reinterpret_cast<uint64_t>(p.table + (uint64_t)batches.b * p.table_sb + at_page), uniform(ids + half * 256));
    };
    // row and chunk of the lane's 16 bytes of load i, before the swizzle
    auto row_of = [&](int i) { return (i * 64 + lane) / S::chunks; };
    auto chunk_of = [&](int i) { return (i * 64 + lane) % S::chunks; };
    uint32_t key_offset[WHOLE ? S::loads : 1], value_offset[WHOLE ? S::loads : 1];
    if constexpr (WHOLE) {
#pragma unroll
        for (int i = 0; i < S::loads; ++i) {
            const int r = row_of(i) % kRows;  // of its range (the swizzles repeat every 16 rows)
            const uint32_t ahead = 1024 * (RANGES == 1 ? i & 3 : i & 1);
            key_offset[i] = (uint32_t)(r * p.kp_st + (chunk_of(i) ^ S::key_swizzle(r))) * 16 - ahead;
            value_offset[i] = (uint32_t)(r * p.vp_st + (chunk_of(i) ^ S::value_swizzle(r))) * 16 - ahead;
        }
    }
    // stage `index` of a batch into ring slot n % 2
    auto load_stage = [&](const Batch &bt, uint32_t index, uint32_t half, uint32_t n) {
        const uint32_t key0 = bt.key + index * kStep, at_ids = ids + half * 256 + index * (4 * kIds);
        if constexpr (MASK) {
            const uint32_t key = min(key0 + lane, bt.length - 1);
            const uint64_t byte = ((uint64_t)bt.b * p.m_sb + (uint64_t)key * p.m_st) * mask_size;
            const uint64_t from = (reinterpret_cast<uint64_t>(p.mask) + byte) & ~(uint64_t)3;
            if (lane < S::keys) load_lds4(from, uniform(maskw + (n & 1) * S::keys * 4));
        }
        const uint32_t base = uniform(ring + (n & 1) * S::stage);
        Stage st = {bt.b, key0, 0u, bt.run};
        if constexpr (WHOLE) {
            i32x4_t keys[RANGES], values[RANGES];
#pragma unroll
            for (int n = 0; n < RANGES; ++n) {
                // the range's rows that exist, none on no page
                const uint32_t id = uniform(*(Q3T_LDS const uint32_t *)(uintptr_t)(at_ids + 4 * n));
                const uint32_t key = key0 + kRows * n, row = key - divide(key, p.by_page) * p.by_page.d;
                const uint32_t count = id < p.pages && bt.length > key ? min(kRows, bt.length - key) : 0u;
                st.exists |= (count == 32 ? ~0u : (1u << count) - 1) << kRows * n % 32;
                auto range = [&](const char *pool, uint32_t page_stride, uint32_t head_stride, uint32_t row_stride) {
                    const uint64_t from = reinterpret_cast<uint64_t>(pool) +
                                          (count ? ((uint64_t)id * page_stride + (uint64_t)row * row_stride + (uint64_t)bt.kv_head * head_stride) * 16 : 0);
                    return scalar_rsrc(reinterpret_cast<const void *>(from), count ? (count - 1) * row_stride * 16 + S::row : 0u);
                };
                keys[n] = range(p.kp, p.kp_sp, p.kp_sh, p.kp_st);
                values[n] = range(p.vp, p.vp_sp, p.vp_sh, p.vp_st);
            }
            auto load = [&](const i32x4_t *ranges, const uint32_t *offset, uint32_t to) {
                if constexpr (RANGES == 1) {
#pragma unroll
                    for (int i = 0; i < S::loads; i += 4) load_rows(ranges[0], offset + i, to + i * 1024);
                } else {
                    static_assert(S::loads == 2 * RANGES, "two loads a range");
#pragma unroll
                    for (int n = 0; n < RANGES; ++n) load_half(ranges[n], offset + 2 * n, to + n * 2048);
                }
            };
            load(keys, key_offset, base);
            load(values, value_offset, base + S::loads * 1024);
        } else {
            const uint32_t rest = bt.length - key0;  // keys from key0 on
            const uint32_t mine = *(Q3T_LDS const uint32_t *)(uintptr_t)(at_ids + lane % S::keys * 4);
            st.exists = (uint32_t)__builtin_amdgcn_ballot_w64(lane < S::keys && (uint32_t)lane < rest && mine < p.pages);
            const uint64_t kh = (uint64_t)bt.kv_head * p.kp_sh, vh = (uint64_t)bt.kv_head * p.vp_sh;
            uint64_t kf[S::loads], vf[S::loads];
#pragma unroll
            for (int i = 0; i < S::loads; ++i) {
                const int r = row_of(i);
                const uint32_t key = min(key0 + r, bt.length - 1), row = key - divide(key, p.by_page) * p.by_page.d;
                uint32_t id = *(Q3T_LDS const uint32_t *)(uintptr_t)(at_ids + r * 4);
                if (id >= p.pages) id = 0;  // a key on no page: not looked at
                const uint64_t ko = (uint64_t)id * p.kp_sp + (uint64_t)row * p.kp_st + kh;
                const uint64_t vo = (uint64_t)id * p.vp_sp + (uint64_t)row * p.vp_st + vh;
                kf[i] = reinterpret_cast<uint64_t>(p.kp) + (ko + (uint32_t)(chunk_of(i) ^ S::key_swizzle(r))) * 16 - 1024 * (i & 3);
                vf[i] = reinterpret_cast<uint64_t>(p.vp) + (vo + (uint32_t)(chunk_of(i) ^ S::value_swizzle(r))) * 16 - 1024 * (i & 3);
            }
#pragma unroll
            for (int i = 0; i < S::loads; i += 4) load_rows(kf + i, base + i * 1024);
#pragma unroll
            for (int i = 0; i < S::loads; i += 4) load_rows(vf + i, base + (S::loads + i) * 1024);
        }
        return st;
    };
    // the query rows of a pair, by the last wave, into one of two places
    auto first_head = [&](uint32_t head) {
        const uint32_t h = kv_head(head);
        return h * p.group + (head - h * p.blocks) * kColumns;
    };
    auto columns_of = [&](uint32_t head) { return min((uint32_t)kColumns, (kv_head(head) + 1) * p.group - first_head(head)); };
    const uint32_t queries = uniform(lds_at(s.query[0]));
    auto load_query = [&](uint32_t b, uint32_t head, uint32_t place) {
        const uint32_t items = columns_of(head) * S::chunks;
        for (uint32_t i = 0; i < items; i += 64) {
            const uint32_t item = i + lane;
            const uint64_t from = reinterpret_cast<uint64_t>(p.q) + ((uint64_t)b * p.q_sb +
                                  (uint64_t)(first_head(head) + item / S::chunks) * p.q_sh + item % S::chunks) * 16;
            if (item < items) load_lds16(from, uniform(queries + (place * kColumns * S::chunks + i) * 16));
        }
    };

    if (wave == W - 1) load_query(at.b, at.head, 0);
    if constexpr (SINGLE) {  // the first batch's page numbers, whatever the length
        batches.b = at.b;
        batches.key = wave * S::keys;
        batches.length = ctx;
        load_ids(0);
    }
    next_batch();
    Batch now = batches;  // the batch whose rows are being loaded, its page numbers in half `half`
    uint32_t index = 0, half = 0;
    Stage s0 = {0u, 0u, 0u, -1};
    if (now.run >= 0) {
        if (!SINGLE) load_ids(0);
        next_batch();
        if (batches.run >= 0) load_ids(1);
        wait_loads<0>();
        s0 = load_stage(now, 0, 0, 0);
    } else {
        wait_loads<0>();
    }
    lds_barrier();  // the first query rows are there

    // ---- run by run -----------------------------------------------------------------------------
    Products x;
    const float unit = MASK ? kLog2e : 1.f;  // scores are natural under a mask, else in log2 units
    const float threshold = MASK ? Products::threshold / kLog2e : Products::threshold;
    float m, l;
    uint32_t n = 0;
    x.place(ring, g, c);
    constexpr uint32_t kAllKeys = (uint32_t)((1ull << S::keys) - 1);
    auto score = [&](const Stage &st) {
        const uint32_t stage = (n & 1) * S::stage;
        // Keys that do not exist.  Their value rows are zeroed, unless they are rows past a range, for
        // which the loads left zeros.
        bool zero_rows = !WHOLE && st.exists != kAllKeys;
        U4 terms[MASK ? S::keys / 16 : 1];
        if constexpr (MASK) {
            // lane k's term is that of key k, from its word; then, through LDS, each lane takes its own four
            const uint32_t k = lane % S::keys, words = maskw + (n & 1) * S::keys * 4;
            const uint32_t low = (uint32_t)reinterpret_cast<uint64_t>(p.mask) + (st.b * p.m_sb + (st.key0 + k) * p.m_st) * mask_size;
            float term = mask_term(*(Q3T_LDS const uint32_t *)(uintptr_t)(words + 4 * k) >> (8 * (low & 3u)), p.mask_dtype);
            if (!(st.exists >> k & 1u)) term = -INFINITY;
            *(Q3T_LDS float *)(uintptr_t)(words + 4 * k) = term;
            zero_rows = __builtin_amdgcn_ballot_w64(term == -INFINITY) != 0;
            asm volatile("" ::: "memory");
#pragma unroll
            for (int t = 0; t < S::keys / 16; ++t) terms[t] = lds_read16(words + (16 * t + 4 * g) * 4);
        }
        f32x4_t scores[S::keys / 16];
#pragma unroll
        for (int t = 0; t < S::keys / 16; ++t) scores[t] = x.scores(stage, t);
        float v[S::keys / 16][4], highest = -INFINITY;
        bool hidden[S::keys / 16][4] = {};
        if (MASK || st.exists != kAllKeys) {
#pragma unroll
            for (int t = 0; t < S::keys / 16; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (MASK) {
                        v[t][i] = __uint_as_float(i == 0 ? terms[t].x : i == 1 ? terms[t].y : i == 2 ? terms[t].z : terms[t].w);
                        hidden[t][i] = v[t][i] == -INFINITY;
                    } else {
                        hidden[t][i] = !(st.exists >> (16 * t + 4 * g) & (1u << i));
                    }
                }
            if ((!WHOLE || MASK) && zero_rows) {
                const U4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int t = 0; t < S::keys / 16; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (hidden[t][i])
                            for (int chunk = c; chunk < S::chunks; chunk += 16)
                                lds_write16(ring + stage + (S::keys + 16 * t + 4 * g + i) * S::row + chunk * 16, zero);
                asm volatile("" ::: "memory");
            }
        }
#pragma unroll
        for (int t = 0; t < S::keys / 16; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float scaled = MASK ? scores[t][i] * p.scale + v[t][i] : scores[t][i] * p.scale;
                v[t][i] = hidden[t][i] ? -INFINITY : scaled;
                highest = fmaxf(highest, v[t][i]);
            }
        x.read_values(stage, 0);  // on their way during the softmax
        if (__builtin_amdgcn_ballot_w64(highest > m + threshold)) {
            highest = fmaxf(highest, xor16(highest));
            highest = fmaxf(highest, xor32(highest));
            highest = fmaxf(highest, m);
            if (__builtin_amdgcn_ballot_w64(m != -INFINITY)) {  // something has been added up
                const float alpha = fexp2((m - (highest == -INFINITY ? 0.f : highest)) * unit);
                l *= alpha;
                x.rescale(alpha);
            }
            m = highest;
        }
        const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int t = 0; t < S::keys / 16; ++t) {
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = fexp2((v[t][i] - from) * unit + Products::shift);
            l += (w[0] + w[1]) + (w[2] + w[3]);
            if (t > 0) x.read_values(stage, t);
            x.values(w);
        }
    };
    auto finish = [&](const Run &r, uint32_t column, uint32_t d, const State &sum) {
        float y[4];
        const float inverse = sum.l == 0.f ? 0.f : 1.f / sum.l;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = sum.a[i] * inverse;
        store_out<T>(p.out + ((uint64_t)r.b * p.o_sb + (uint64_t)(first_head(r.head) + column) * p.o_sh + d) * sizeof(T), y, p.vec_out);
    };
    const uint32_t state_size = p.columns * (D + 2);

    for (int32_t order = 0; at.left > 0; ++order) {
        const Run r = next_run(at, stages_of(request_length(at.b)), p.heads, sh);
        const uint32_t columns = columns_of(r.head);
        if (wave == W - 1 && at.left > 0) load_query(at.b, at.head, (order + 1) & 1);
        x.load_query(queries + (order & 1) * kColumns * S::row, g, c, (uint32_t)c < columns);
        x.clear();
        m = -INFINITY;
        l = 0.f;
        if (s0.run != order) wait_loads<0>();  // no stage here: the next query rows may be in flight
        while (s0.run == order) {
            // the next stage, into the slot that was scored last, once its reads have returned
            Stage s1 = {0u, 0u, 0u, -1};
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            ++index;
            if (index * kStep < kBatch && now.key + index * kStep < now.end) {
                s1 = load_stage(now, index, half, n + 1);
                wait_loads<LOADS + (MASK ? 1 : 0)>();
            } else if (batches.run >= 0) {
                wait_loads<LOADS + (MASK ? 1 : 0)>();  // the batch's page numbers, loaded ahead of the last batch's rows
                now = batches;
                index = 0;
                half ^= 1;
                next_batch();
                const bool more = batches.run >= 0;
                if (more) load_ids(half ^ 1);
                s1 = load_stage(now, 0, half, n + 1);
                if (more) wait_loads<LOADS + (MASK ? 1 : 0) + 1>();
                else wait_loads<LOADS + (MASK ? 1 : 0)>();
            } else {
                wait_loads<0>();
            }
            score(s0);
            s0 = s1;
            ++n;
            // Of two workgroups on a CU the older one's loads go first, and the younger one (of the later half, as
            // they are dealt out) would end after it: it goes first on every second stage (200 requests of
            // 10..400 keys 28.0 -> 27.2 us).  Not in one workgroup of eight waves, where all wait for the
            // last (64 of 64..1023 with it 33.0, without 31.6).
            if (W == 4 && blockIdx.x >= 256) {
                if (n & 1) __builtin_amdgcn_s_setprio(2);
                else __builtin_amdgcn_s_setprio(0);
            }
        }

        // the waves' states, each in the slot that its next stage is not in, into one
        l += xor16(l);
        l += xor32(l);
        const uint32_t slot = ring + ((n + 1) & 1) * S::stage;
        if (g == 0) {
            s.ml[wave][c][0] = m;
            s.ml[wave][c][1] = l;
        }
        if (lane == 0) s.slot[wave] = slot;
        const bool whole = SINGLE || r.parts == 1;
        // The first of two parts is done last in its share, and the other first in the next one: where that
        // one is there already, it is merged at once and nothing is published.
        int32_t *counter = p.counters + r.b * p.heads + r.head;
        if (!whole && tid == kThreads - 1 && r.parts == 2 && r.begins)
            s.there = (uint32_t)__hip_atomic_load(counter, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if ((uint32_t)c < columns) x.store(slot, g, c);
        lds_barrier();
        const bool two = !whole && r.parts == 2 && r.begins && uniform(s.there) == 1;
        float *state = p.states + (2 * blockIdx.x + r.begins) * (uint64_t)state_size;
        for (uint32_t item = tid; item < columns * (D / 4); item += kThreads) {
            const uint32_t column = item / (D / 4), chunk = item % (D / 4);
            State own = {};
            own.m = -INFINITY;
#pragma unroll
            for (int w = 0; w < W; ++w) own.m = fmaxf(own.m, s.ml[w][column][0]);
            const float from = own.m == -INFINITY ? 0.f : own.m;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float e = fexp2((s.ml[w][column][0] - from) * unit);
                own.l += s.ml[w][column][1] * e;
                own.a += __builtin_bit_cast(f32x4_t, lds_read16(s.slot[w] + column * D * 4 + (chunk ^ column) * 16)) * e;
            }
            if (two) {
                State other;
                other.collect(p.states + 2 * (r.first + 1) * (uint64_t)state_size, p.columns * D, column, chunk * 4, D);
                own.add(other, unit);
            }
            if (whole || two) finish(r, column, chunk * 4, own);
            else own.publish(state, p.columns * D, column, chunk * 4, D);
        }
        if (!whole && !two) wait_loads<0>();  // the state has been stored
        lds_barrier();
        if (two && tid == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (whole || two) continue;

        // Parts beyond kTogether are merged in two steps: kTogether neighbours' last to arrive merges
        // theirs into the first one's state, and the last of those merges them.
        const uint32_t part = blockIdx.x - r.first;
        auto slot_of = [&](uint32_t i) { return 2 * (r.first + i) + (i == 0); };  // part i's state
        auto arrive = [&](int32_t *counter, uint32_t expected) {
            if (tid == 0) s.count = (uint32_t)__hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();  // (the waves' merge or a merge of parts, with barriers, lies before the next count)
            const bool last = uniform(s.count) == expected - 1;
            if (last && tid == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            return last;
        };
        // every `step`-th part from `begin` on, `count` of them, in one order whoever merges them: thread
        // (part % groups, item) adds up every groups-th part's four elements, and thread (0, item) the groups'
        auto merge = [&](uint32_t begin, uint32_t step, uint32_t count, bool last) {
            const uint32_t items = columns * (D / 4), groups = max(1u, kThreads / items);
            for (uint32_t first = 0; first < items; first += kThreads) {
                const uint32_t group = groups == 1 ? 0 : tid / items, item = groups == 1 ? first + tid : tid - group * items;
                const bool live = group < groups && item < items;
                const uint32_t column = item / (D / 4), d = item % (D / 4) * 4;
                State sum = {};
                sum.m = -INFINITY;
                if (live) {
                    constexpr uint32_t kFlight = 4;  // states on their way at once
                    for (uint32_t i = group; i < count; i += kFlight * groups) {
                        State parts[kFlight];
#pragma unroll
                        for (uint32_t j = 0; j < kFlight; ++j) {
                            const uint32_t at_part = min(i + j * groups, count - 1);
                            parts[j].collect(p.states + slot_of(begin + at_part * step) * (uint64_t)state_size, p.columns * D, column, d, D);
                        }
#pragma unroll
                        for (uint32_t j = 0; j < kFlight; ++j)
                            if (i + j * groups < count) sum.add(parts[j], unit);
                    }
                }
                if (groups > 1) {
                    // 32 bytes a thread, in its wave's free slot
                    auto place = [&](uint32_t t) { return s.slot[t >> 6] + (t & 63) * 32; };
                    if (live) {
                        lds_write16(place(tid), __builtin_bit_cast(U4, sum.a));
                        lds_write16(place(tid) + 16, U4{__float_as_uint(sum.m), __float_as_uint(sum.l), 0u, 0u});
                    }
                    lds_barrier();
                    if (live && group == 0) {
                        for (uint32_t o = 1; o < min(groups, count); ++o) {
                            const U4 ml = lds_read16(place(tid + o * items) + 16);
                            const State other = {__uint_as_float(ml.x), __uint_as_float(ml.y),
                                                 __builtin_bit_cast(f32x4_t, lds_read16(place(tid + o * items)))};
                            sum.add(other, unit);
                        }
                    }
                    lds_barrier();  // the slots are free again
                }
                if (!last) {  // the first part's state is written where other threads have read it
                    wait_loads<0>();
                    lds_barrier();
                }
                if (live && group == 0) {
                    if (last) finish(r, column, d, sum);
                    else sum.publish(p.states + slot_of(begin) * (uint64_t)state_size, p.columns * D, column, d, D);
                }
            }
        };
        bool last = r.parts <= kTogether;
        uint32_t begin = last ? 0 : part / kTogether * kTogether, step = 1, count = min(kTogether, r.parts - begin);
        while (arrive(last ? counter : p.counters + kPairs + slot_of(begin), count)) {
            merge(begin, step, count, last);
            if (last) break;
            wait_loads<0>();
            lds_barrier();  // the merged state has been stored
            begin = 0;
            step = kTogether;
            count = (r.parts + kTogether - 1) / kTogether;
            last = true;
        }
    }
}

// What a launch does, by what the host sees: capacities, not lengths.  The figures are of tables as wide as the longest
// request; requests in a wider table run as the table's width has it.  us, 8 KV heads of 128 in bf16, exact / 1024 /
// 4096 / 32000 rows: one request of 300 keys 7.6 / 10.3 / 10.3 / 9.7, 8 of 300 8.3 / 10.9 / 10.1 / 10.2, 32 of 300 10.7 /
// 10.7 / 12.0 / 12.0, 64 of 64 8.0 / 11.9 / 11.9 / 12.0, 48 of 100..400 15.4 / 18.6 / 18.7 / 18.6, 64 of 64..1023 31.7 / 30.6 /
// 30.5 / 30.5.
//   * Few short pairs, a workgroup each: nothing to find or share, and no states pass through memory.  Eight waves
//     for a pair a CU, us shared out / a workgroup each (8 KV heads of 128, bf16): one request of 100 keys 7.7 / 6.0,
//     of 300 10.2 / 7.5, of 600 10.6 / 9.9, of 700 10.5 / 10.5, 8 of 300 10.5 / 8.4, 8 of 600 12.5 / 11.9, 8 of
//     100..700 11.2 / 11.5; from half of the CUs on longer ones too: 32 of 1..700 17.9 / 14.3, 20 of 900 21.7 / 17.2,
//     24 of 100..1000 18.0 / 16.3, 32 of 1000 26.6 / 24.9, but 32 of 30..2047 with 4 KV heads 22.5 / 27.7.  Up to
//     700 keys, or 1024; twice that for rows of 128 bytes (one of 1000 9.4 / 8.6, 32 of 100..1800 18.3 / 16.0, 24 of
//     2000 25.0 / 20.3; where a stage's rows are not one range one of 1000 9.7 / 11.1, so 700 stays).
//     Four waves for as many pairs as there are workgroups (rows of 256 bytes): 64 of 64 9.0 / 7.5, 48 of 100..400
//     19.0 / 15.4, 64 of 10..500 21.1 / 17.7, 40 of 600 27.5 / 23.5, 64 of 700 35.7 / 33.1, 64 of 10..750 23.7 / 22.3;
//     40 of 64..1023 23.4 / 25.1.  Up to 768 keys.
//   * Many stages: eight waves, half as many shares, so half as many cut pairs, but more waves with nothing to
//     do in a short one.  us, four / eight: 128 requests of 100..4095 keys 180 / 174, 64 of 64..1023 33.4 / 30.8, 40 of
//     64..1023 25.5 / 23.4, one of 65000 33.1 / 31.7, 8 of 1000..4000 24.7 / 24.3; 8 of 100..2000 14.1 / 14.7, 512 of
//     20..200 32.8 / 41.6.  From 769 keys a request and 15000 stages and run ends in all, for up to 1024 pairs,
//     where short requests cost little.  Under a mask too: 64 of 64..1023 33.3 / 31.8, 32 of 30..2047 33.2 / 32.1, 128 of
//     100..2000 with 4 KV heads 57.7 / 53.8, 8 of 1000..4000 25.1 / 25.1; the rule costs 1 to 3% in the smallest masked
//     launches that it takes (32 of 30..2047 with 4 KV heads of 4 query heads 21.6 / 21.9, of 8 21.9 / 22.4).  Not
//     rows of 128 bytes: 64 of 64..2047 33.5 / 36.9, 128 of 100..4000 94.6 / 95.6.
//   * Groups of more than 8 query heads, whose states are large: eight waves, half as many parts.  us, four / eight: 16
//     heads on one KV head, one request of 1000 keys 12.6 / 11.7, of 8000 18.8 / 16.4, of 60000 31.6 / 21.0, 8 of
//     2000 16.5 / 13.2, 128 of 64..1023 20.5 / 19.1, 32 of 4000 26.1 / 22.3; 256 of 100..1000 24.8 / 25.2, 512 of
//     20..200 20.1 / 20.4, 300 of 10..60 10.1 / 13.9.  From 192 keys on.  Groups of 8 lose as often (one of
//     1000 and two KV heads 10.7 / 11.8, of 4000 and four 14.4 / 13.1).  Rows of 128 bytes from 2500 keys on: one
//     of 1000 9.9 / 11.3, 8 of 2000 10.9 / 11.7, 32 of 4000 17.3 / 14.4, one of 8000 13.9 / 12.4.
constexpr int64_t kLongRequest = 769, kManyStages = 15000, kFewPairs = 1024;
constexpr int64_t kShortRequest = 700, kMiddleRequest = 1024, kCUs = 256;
constexpr int64_t kSmallRequest = 768;
constexpr int64_t kWideGroup = 8, kWideRequest = 192, kWideNarrow = 2500;

template <typename T, int D>
struct Launch {
    typedef Shape<T, D> S;
    static int64_t stages(const q3t_paged_args *a, int64_t pairs, int waves) { return pairs * ((a->ctx + S::keys - 1) / S::keys + run_cost(waves)); }
    // Ranges of memory that a stage's rows are in: whole pages, rows that do not overlap, 32-bit offsets; else 0.
    static int ranges(const q3t_paged_args *a) {
        const int64_t es = sizeof(T), most = ((int64_t)1 << 30) / S::keys;
        if (a->kp_stride_t * es < S::row || a->vp_stride_t * es < S::row || a->kp_stride_t * es >= most || a->vp_stride_t * es >= most)
            return 0;
        return a->page_size % S::keys == 0 ? 1 : a->page_size % 16 == 0 ? 2 : 0;
    }
    // one workgroup of eight waves, or of four, for each pair
    static bool few(const q3t_paged_args *a, int64_t pairs) {
        constexpr int64_t narrow = 256 / S::row;
        return S::row < 512 && pairs <= kCUs &&
               a->ctx <= (pairs >= kCUs / 2 ? kMiddleRequest * narrow : kShortRequest * (ranges(a) == 1 ? narrow : 1));
    }
    static bool small(const q3t_paged_args *a, int64_t pairs) {
        return S::row == 256 && ranges(a) == 1 && !eight(a, pairs) && pairs > kCUs && pairs <= Workgroups<T, D, 4>::count &&
               a->ctx <= kSmallRequest;
    }
    static bool single(const q3t_paged_args *a, int64_t pairs) {
        // a pair is one piece, and there is a workgroup for it
        static_assert(S::row == 512 || kMiddleRequest * 256 / S::row <= (int64_t)S::keys << kLogLeastSingle, "");
        static_assert(kSmallRequest <= (int64_t)S::keys << kLogLeastSingle && kCUs <= Workgroups<T, D, 8>::count, "");
        return few(a, pairs) || small(a, pairs);
    }
    static bool eight(const q3t_paged_args *a, int64_t pairs) {
        const bool many = S::row > 128 && a->ctx >= kLongRequest && pairs <= kFewPairs && stages(a, pairs, 4) >= kManyStages;
        const bool wide = a->q_heads / a->kv_heads > kWideGroup && a->ctx >= (S::row == 128 ? kWideNarrow : kWideRequest);
        return few(a, pairs) || (S::row < 512 && ranges(a) == 1 && (many || wide));
    }
    static uint32_t log_least(const q3t_paged_args *a, int64_t pairs) {
        return single(a, pairs) ? kLogLeastSingle : eight(a, pairs) ? kLogLeast8 : kLogLeast4;
    }
    static int64_t workgroups(const q3t_paged_args *a, int64_t pairs) {
        const bool wide = eight(a, pairs);
        const int64_t least = (int64_t)1 << log_least(a, pairs), stages = (a->ctx + S::keys - 1) / S::keys;
        const int64_t pieces = pairs * ((stages + least - 1) / least);
        const int64_t most = wide ? Workgroups<T, D, 8>::count : Workgroups<T, D, 4>::count;
        return pieces < most ? pieces : most;
    }
    static void run(const q3t_paged_args *a, int64_t pairs, const Params &p, uint32_t blocks, hipStream_t s) {
        auto launch = [&](auto kernel, int waves) {
            hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * waves), 0, s, a->positions, (uint32_t)a->batch, (uint32_t)a->ctx, p);
        };
        auto masked = [&](auto mask) {
            constexpr bool MASK = decltype(mask)::value;
            if constexpr (S::row < 512) {
                if (few(a, pairs)) {
                    if constexpr (S::keys == 32)
                        if (ranges(a) == 2) return launch(paged_kernel<T, D, MASK, 2, 8, true>, 8);
                    return ranges(a) == 1 ? launch(paged_kernel<T, D, MASK, 1, 8, true>, 8) : launch(paged_kernel<T, D, MASK, 0, 8, true>, 8);
                }
                if constexpr (S::row == 256)
                    if (small(a, pairs)) return launch(paged_kernel<T, D, MASK, 1, 4, true>, 4);
                if (eight(a, pairs)) return launch(paged_kernel<T, D, MASK, 1, 8, false>, 8);
            }
            if (ranges(a) == 1) launch(paged_kernel<T, D, MASK, 1, 4, false>, 4);
            else launch(paged_kernel<T, D, MASK, 0, 4, false>, 4);
        };
        if (a->mask) masked(std::true_type{});
        else masked(std::false_type{});
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
    if (a->ctx >= 1 << 30 || a->batch > kPairs || a->q_heads > 1 << 16) return Q3T_EUNSUPPORTED;
    z.group = a->q_heads / a->kv_heads;
    z.blocks = (z.group + kColumns - 1) / kColumns;
    z.pairs = a->batch * a->kv_heads * z.blocks;
    z.columns = z.group < kColumns ? z.group : kColumns;
    if (z.pairs > kPairs) return Q3T_EUNSUPPORTED;  // a counter each
    if (with(a, [&](auto l) { return l.stages(a, z.pairs, 8); }) >= INT32_MAX / 2) return Q3T_EUNSUPPORTED;
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
    const int64_t strides[8] = {a->q_stride_b, a->q_stride_h, a->kp_stride_p, a->kp_stride_h, a->kp_stride_t, a->vp_stride_p, a->vp_stride_h, a->vp_stride_t};
    uint32_t *const to[8] = {&p.q_sb, &p.q_sh, &p.kp_sp, &p.kp_sh, &p.kp_st, &p.vp_sp, &p.vp_sh, &p.vp_st};
    for (int i = 0; i < 8; ++i) {
        const int s = chunks(strides[i], *to[i]);
        if (s != Q3T_OK) return s;
    }
    p.q = (const char *)a->query; p.kp = (const char *)a->key_pages; p.vp = (const char *)a->value_pages;
    p.mask = (const char *)a->mask; p.out = (char *)a->out;
    p.table = a->page_table;
    const int64_t elements[5] = {a->o_stride_b, a->o_stride_h, a->mask ? a->mask_stride_b : 0, a->mask ? a->mask_stride_t : 0, a->table_stride_b};
    uint32_t *const in[5] = {&p.o_sb, &p.o_sh, &p.m_sb, &p.m_st, &p.table_sb};
    for (int i = 0; i < 5; ++i) {
        if (elements[i] < 0) return Q3T_EINVAL;
        if (elements[i] > UINT32_MAX) return Q3T_EUNSUPPORTED;
        *in[i] = (uint32_t)elements[i];
    }
    const int64_t mask_size = a->mask_dtype == Q3T_F32 ? 4 : a->mask_dtype == Q3T_BOOL ? 1 : 2;
    if (!aligned(p.q, 16) || !aligned(p.kp, 16) || !aligned(p.vp, 16) || !aligned(p.out, es) ||
        !aligned(p.table, 4) || !aligned(a->positions, 8) || (p.mask && !aligned(p.mask, mask_size)))
        return Q3T_EINVAL;
    if (!a->workspace || a->workspace_bytes < z.workspace) return Q3T_EWORKSPACE;
    if (!aligned(a->workspace, 16)) return Q3T_EINVAL;
    p.counters = (int32_t *)a->workspace;
    p.states = (float *)((char *)a->workspace + kCounters * 4);
    p.mask_dtype = (int32_t)a->mask_dtype;
    p.vec_out = aligned(p.out, 4 * es) && (p.o_sb | p.o_sh) % 4 == 0;
    p.pages = (uint32_t)a->pages;
    p.group = (uint32_t)z.group; p.blocks = (uint32_t)z.blocks;
    p.heads = (uint32_t)(a->kv_heads * z.blocks);
    p.columns = (uint32_t)z.columns;
    p.log_least = with(a, [&](auto l) { return l.log_least(a, z.pairs); });
    p.by_page = divisor((uint32_t)a->page_size);
    p.by_grid = divisor((uint32_t)z.workgroups);
    p.scale = a->mask ? a->scale : a->scale * kLog2e;
    with(a, [&](auto l) { l.run(a, z.pairs, p, (uint32_t)z.workgroups, (hipStream_t)stream); });
    return launch_status();
}
