// Attention of a whole batch over the keys that all of its requests share.
//
// The query heads of all requests that read one KV head are the columns of the products S^T = K . Q^T and
// O^T += V^T . P^T, so a key and a value row is read once for all of them.  For each column the result is a softmax state,
// maximum, sum and weighted values, that the attention over the request's own keys takes in at its end.
//   * A workgroup takes one KV head, a block of CW * CT * 16 columns and a part of the keys.  CW waves share a stage of
//     keys in LDS, each with CT tiles of 16 columns in registers; KW such groups take the stages in turn and are merged
//     at the end.
//   * Stages come straight from memory to LDS, ahead of the one that is multiplied.
//   * The weights go into the second product in two parts of the type's bits, 16 of a float32's in bf16 and 22 in fp16 (float32 is
//     multiplied as such), and their sum is that of the float32 weights: outputs are those of requests that each read the prefix, up to
//     what the outputs' own rounding hides.  In one part the largest launch below takes 50 us for 64, but outputs are
//     off by 0.0022 of their norm where the type's rounding alone is 0.0017.
//   * A value that is not finite would reach, as zero times NaN, columns that do not see its key, and as infinity times a part that
//     is zero those that do.  A launch that meets such a one says so, and its states are not used: the requests then attend the prefix
//     each for itself.
// The matrix cores bound it from some hundred columns on (4 * 16384 keys, 128 requests, 32 query heads over 8 KV heads of 128 in
// bf16: 51.5 GFLOP, the weights' two parts counted, in 64 us, 0.80 PFLOP/s and 0.94 past the start of 9 us, where a large library
// product reaches 1.2), the start and the stages' chain below it (8 KV heads, 128 columns each, 4096 keys 18.6 us).  Waves that
// share a stage alternate between matrix and vector instructions in two groups (with the addresses of a part worked out once, 65 ->
// 57 us, with weights in one part).
#pragma once

#include "paged_kernel.hpp"

namespace q3t {
namespace paged {

struct PrefixParams {
    const char *q, *kp, *vp, *mask;
    const int32_t *table;
    const int64_t *positions;
    float *states, *ml;                 // (part, KV head, column): D values; maximum and sum
    uint32_t *odd;                      // of each workgroup: its states are not to be used, nor any other
    uint32_t q_sb, q_sh, kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st;  // 16 bytes
    uint32_t m_sb, m_st;                // elements
    int32_t mask_dtype, mask_vec;       // four terms at once: unit strides, aligned, keys a multiple of 4
    uint32_t heads, columns, blocks;    // KV heads; columns of one, and their blocks
    uint32_t parts, keys, chunk;        // parts of `chunk` keys
    uint32_t pages, ctx;
    uint32_t table_sb, batch;
    int32_t flip, zero;                 // unmasked: the scale is below zero, is zero
    Divisor by_page, by_group;
    float scale;                        // unmasked: its size times log2(e), 1 for none
};

// The products of a wave's CT tiles of 16 columns with a stage's keys.
template <typename T, int D, int CT> struct Wide {
    typedef Shape<T, D> S;
    static constexpr int tiles = 2, keys = 32;  // of 16 keys; keys of a stage
    static constexpr float shift = Half<T>::shift, threshold = Half<T>::threshold;
    static constexpr int parts = 2;  // of a weight
    U4 q[CT][D / 32];
    f32x4_t acc[CT][D / 16];
    float sum[CT];
    uint32_t key_at[D / 32], value_at[D / 16];

    Q3T_DEVICE void load_query(int ct, const char *row, int g, bool live, bool flip) {
        const uint32_t sign = flip ? 0x80008000u : 0u;
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {
            const U4 x = live ? load16(row + (4 * kk + g) * 16) : U4{0u, 0u, 0u, 0u};
            q[ct][kk] = U4{x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign};
        }
    }
    // The query rows have come: no wait for them is left to the loop, where it would hold up the stages.
    Q3T_DEVICE void settle() {
#pragma unroll
        for (int i = 0; i < CT * (D / 32); ++i) asm volatile("" : "+v"(q[i / (D / 32)][i % (D / 32)].x), "+v"(q[i / (D / 32)][i % (D / 32)].y),
                                                                 "+v"(q[i / (D / 32)][i % (D / 32)].z), "+v"(q[i / (D / 32)][i % (D / 32)].w));
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
        const int r = 4 * g + (c >> 2);
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) key_at[kk] = c * S::row + (((4 * kk + g) ^ S::key_swizzle(c)) & (S::chunks - 1)) * 16;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
            value_at[d] = (keys + r) * S::row + (((2 * d + ((c >> 1) & 1)) ^ S::value_swizzle(r)) & (S::chunks - 1)) * 16 + 8 * (c & 1);
    }
    U4 k[tiles][D / 32], v[D / 16], p[CT][parts];  // a stage's fragments of keys and values, its weights
    Q3T_DEVICE void read_keys(uint32_t stage) {
#pragma unroll
        for (int t = 0; t < tiles; ++t)
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk) k[t][kk] = lds_read16(key_at[kk] + stage + t * 16 * S::row);
        together();
    }
    Q3T_DEVICE void scores(f32x4_t (&s)[CT][tiles]) const {
#pragma unroll
        for (int t = 0; t < tiles; ++t)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) s[ct][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
            for (int t = 0; t < tiles; ++t)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) s[ct][t] = Half<T>::scores(k[t][kk], q[ct][kk], s[ct][t]);
    }
    Q3T_DEVICE void read_values(uint32_t stage) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            const uint2 lo = lds_read_tr16(value_at[d] + stage), hi = lds_read_tr16(value_at[d] + stage + 16 * S::row);
            v[d] = U4{lo.x, lo.y, hi.x, hi.y};
        }
        together();
    }
    // The weights as operands, in parts: inner index 8 g + j stands for key 4 g + j of the first tile (j < 4), and 4 g + j - 4 of
    // the second.
    Q3T_DEVICE void weights(int ct, const float (&w)[tiles][4]) {
        float rest[tiles * 4];
#pragma unroll
        for (int k = 0; k < tiles * 4; ++k) rest[k] = w[k / 4][k % 4];
        sum[ct] += ((rest[0] + rest[1]) + (rest[2] + rest[3])) + ((rest[4] + rest[5]) + (rest[6] + rest[7]));
#pragma unroll
        for (int n = 0; n < parts; ++n) {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                u[i] = Half<T>::round2(rest[2 * i], rest[2 * i + 1]);
                rest[2 * i] -= Half<T>::lo(u[i]);
                rest[2 * i + 1] -= Half<T>::hi(u[i]);
            }
            p[ct][n] = U4{u[0], u[1], u[2], u[3]};
            // (worked out here, not where they are used)
            asm volatile("" : "+v"(p[ct][n].x), "+v"(p[ct][n].y), "+v"(p[ct][n].z), "+v"(p[ct][n].w));
        }
    }
    Q3T_DEVICE void values() {
#pragma unroll
        for (int n = 0; n < parts; ++n)
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) acc[ct][d] = Half<T>::scores(v[d], p[ct][n], acc[ct][d]);
    }
    Q3T_DEVICE float total(int ct) const {
        const float l = sum[ct] + xor16(sum[ct]);
        return l + xor32(l);
    }
    // the values' dims, as they are stored: 16 bytes of acc[][a] from dim
    Q3T_DEVICE static int dim(int a, int g) { return 16 * a + 4 * g; }
    Q3T_DEVICE f32x4_t four(int ct, int a) const { return acc[ct][a]; }
};

template <int D, int CT> struct Wide<float, D, CT> {
    typedef Shape<float, D> S;
    static constexpr int tiles = 1, keys = 16;
    static constexpr float shift = 0.f, threshold = 8.f;
    f32x4_t q[CT][D / 16], acc[CT][D / 16];
    float sum[CT];
    uint32_t key_at[D / 16], value_at;

    Q3T_DEVICE void load_query(int ct, const char *row, int g, bool live, bool flip) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            const f32x4_t x = __builtin_bit_cast(f32x4_t, live ? load16(row + (4 * kk + g) * 16) : U4{0u, 0u, 0u, 0u});
            q[ct][kk] = flip ? -x : x;
        }
    }
    Q3T_DEVICE void settle() {
#pragma unroll
        for (int i = 0; i < CT * (D / 16); ++i) asm volatile("" : "+v"(q[i / (D / 16)][i % (D / 16)]));
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
    f32x4_t k[D / 16], v[4 * (D / 64)];
    float p[CT][4];
    Q3T_DEVICE void read_keys(uint32_t stage) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) k[kk] = __builtin_bit_cast(f32x4_t, lds_read16(key_at[kk] + stage));
        together();
    }
    Q3T_DEVICE void scores(f32x4_t (&s)[CT][tiles]) const {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) s[ct][0] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) s[ct][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[kk][e], q[ct][kk][e], s[ct][0], 0, 0, 0);
    }
    Q3T_DEVICE void read_values(uint32_t stage) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < D / 64; ++j) v[i * (D / 64) + j] = __builtin_bit_cast(f32x4_t, lds_read16(value_at + stage + i * S::row + j * 256));
        together();
    }
    Q3T_DEVICE void weights(int ct, const float (&w)[tiles][4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[ct][i] = w[0][i];
            asm volatile("" : "+v"(p[ct][i]));
        }
        sum[ct] += (w[0][0] + w[0][1]) + (w[0][2] + w[0][3]);
    }
    Q3T_DEVICE void values() {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < D / 64; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct)
                        acc[ct][4 * j + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i * (D / 64) + j][e], p[ct][i], acc[ct][4 * j + e], 0, 0, 0);
    }
    Q3T_DEVICE float total(int ct) const {
        const float l = sum[ct] + xor16(sum[ct]);
        return l + xor32(l);
    }
    // (row 4 g + i of the products 4 j + e is dim 64 j + 16 g + 4 i + e)
    Q3T_DEVICE static int dim(int a, int g) { return 64 * (a >> 2) + 16 * g + 4 * (a & 3); }
    Q3T_DEVICE f32x4_t four(int ct, int a) const {
        const int j = a & ~3, i = a & 3;
        return f32x4_t{acc[ct][j][i], acc[ct][j + 1][i], acc[ct][j + 2][i], acc[ct][j + 3][i]};
    }
};

// Loads into LDS from an address per lane (load_rows and load_half, for rows that several workgroups read).
Q3T_DEVICE void load_shared(const uint64_t *p, uint32_t base) {
    asm volatile("s_mov_b32 m0, %0\n\t" Q3T_VMEM_SGPR_WAIT
                 "global_load_lds_dwordx4 %1, off\n\t"
                 "global_load_lds_dwordx4 %2, off offset:1024\n\t"
                 "global_load_lds_dwordx4 %3, off offset:2048\n\t"
                 "global_load_lds_dwordx4 %4, off offset:3*1024"
                 :: "s"(base), "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]) : "memory", "m0");
}
Q3T_DEVICE void load_shared_half(const uint64_t *p, uint32_t base) {
    asm volatile("s_mov_b32 m0, %0\n\t" Q3T_VMEM_SGPR_WAIT
                 "global_load_lds_dwordx4 %1, off\n\t"
                 "global_load_lds_dwordx4 %2, off offset:1024"
                 :: "s"(base), "v"(p[0]), "v"(p[1]) : "memory", "m0");
}

constexpr uint32_t kEntries = 1024;  // pages that a workgroup knows: those of its part

template <typename T, int D, int CW, int KW, int CT>
struct PrefixLds {
    typedef Wide<T, D, CT> X;
    static constexpr int stage = 2 * X::keys * Shape<T, D>::row, buffers = CW == 1 ? 2 : 4;
    union {
        alignas(1024) char ring[buffers][KW][stage];
        alignas(1024) f32x4_t merge[KW == 1 ? 1 : KW - 1][CW][CT][D / 16][64];  // the groups' states, each in the first group's order
    };
    float ml[KW][CW][CT][2][64];
    uint64_t pages[kEntries][2];     // addresses of the head's first key and value row on a page, kBias short; odd for no page
    uint32_t odd;                    // values that are not finite were met
    uint32_t least;                  // keys that all live columns see
    uint32_t holes;                  // entries that are no page
    uint32_t row;                    // the first of the table whose first entry is a page
};

// CW waves share the columns, KW groups of them the stages.
// WHOLE: a stage lies in one page, or pages of whole loads in a stage.
template <typename T, int D, bool MASK, bool WHOLE, int CW, int KW, int CT>
__global__ void __launch_bounds__(64 * CW * KW, (CW * KW / 4 * (sizeof(PrefixLds<T, D, CW, KW, CT>) <= 80 * 1024 ? 2 : 1)))
prefix_kernel(PrefixParams p) {
    typedef Shape<T, D> S;
    typedef Wide<T, D, CT> X;
    typedef PrefixLds<T, D, CW, KW, CT> L;
    constexpr int SK = X::keys, TILES = X::tiles, B = L::buffers, kThreads = 64 * CW * KW;
    constexpr int LOADS = L::stage / 1024 / CW;  // of a wave's share of a stage: keys' rows in the first half, values' in the second
    constexpr uint32_t kAll = (uint32_t)((1ull << SK) - 1);
    static_assert(CW == 1 || KW == 2, "");
    static_assert(sizeof(f32x4_t) * (KW - 1) * CW * CT * (D / 16) * 64 <= sizeof(char) * L::buffers * KW * L::stage, "");
    __shared__ L s;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int wave = (int)uniform(tid >> 6), cw = wave % CW, group = wave / CW;

    // all column blocks of a KV head's part follow each other on one XCD
    const uint32_t task = blockIdx.x / (8 * p.blocks) * 8 + blockIdx.x % 8, block = blockIdx.x / 8 % p.blocks;
    if (task >= p.heads * p.parts) return;
    const uint32_t part = task / p.heads, head = task - part * p.heads;
    const uint32_t begin = part * p.chunk, end = min(p.keys, begin + p.chunk);

    // ---- stages ----
    const uint32_t ring = uniform(lds_at(&s.ring[0][0][0]));
    const uint32_t entry0 = divide(begin, p.by_page);
    auto buffer = [&](uint32_t n) { return ring + (n % B * KW + group) * L::stage; };
    const uint32_t sets = (end - begin + KW * SK - 1) / (KW * SK);  // of a stage for every group
    // row and chunk of the lane's 16 bytes of load i of the wave's share
    auto row_of = [&](int i) { return ((cw * LOADS + i) * 64 + lane) / S::chunks % SK; };
    auto is_value = [&](int i) { return cw * LOADS + i >= L::stage / 2048; };
    // the lane's place in load i: entry and offset from those of the stage's first row (WHOLE), or the chunk of its row
    uint32_t entry_of[LOADS], offset[LOADS];
    constexpr uint32_t kBias = 4096;  // (the loads' offsets move both of their addresses: load i's is 1024 i short)
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const uint32_t r = row_of(i), chunk = lane % S::chunks ^ (is_value(i) ? S::value_swizzle(r) : S::key_swizzle(r));
        const uint32_t ahead = p.by_page.d < (uint32_t)SK ? r / p.by_page.d : 0;
        entry_of[i] = ahead;
        offset[i] = chunk * 16 + kBias - 1024 * (LOADS == 2 ? i : i & 3);
        if constexpr (WHOLE) offset[i] += (r - ahead * p.by_page.d) * (is_value(i) ? p.vp_st : p.kp_st) * 16;
    }
    const uint32_t pages = uniform(lds_at(&s.pages[0][0]));
    const uint32_t last_entry = divide(end - 1, p.by_page) - entry0;
    uint32_t holes = 0;
    uint64_t at[LOADS];  // of the next stage's loads
    // works them out, and says which of stage n's keys exist
    auto locate = [&](uint32_t n) {
        const uint32_t key0 = begin + (n * KW + group) * SK;
        if constexpr (WHOLE) {
            const uint32_t entry = divide(key0, p.by_page) - entry0;
            const uint32_t row = p.by_page.d < (uint32_t)SK ? 0 : key0 - divide(key0, p.by_page) * p.by_page.d;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                // (past the end, the part's last page: its rows are not looked at)
                const uint64_t from = *(Q3T_LDS const uint64_t *)(uintptr_t)(pages + min(entry + entry_of[i], last_entry) * 16 + (is_value(i) ? 8 : 0));
                at[i] = (from & ~(uint64_t)1) + (offset[i] + row * (is_value(i) ? p.vp_st : p.kp_st) * 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const uint32_t key = min(key0 + row_of(i), end - 1), entry = divide(key, p.by_page);
                const uint64_t from = *(Q3T_LDS const uint64_t *)(uintptr_t)(pages + (entry - entry0) * 16 + (is_value(i) ? 8 : 0));
                at[i] = (from & ~(uint64_t)1) + (uint64_t)(key - entry * p.by_page.d) * (is_value(i) ? p.vp_st : p.kp_st) * 16 + offset[i];
            }
        }
        const uint32_t count = key0 < end ? min((uint32_t)SK, end - key0) : 0u;
        uint32_t exists = (uint32_t)((1ull << count) - 1);
        if (holes) {
            const uint32_t key = min(key0 + lane % SK, end - 1);
            exists &= (uint32_t)__builtin_amdgcn_ballot_w64(!(s.pages[divide(key, p.by_page) - entry0][0] & 1));
        }
        return exists;
    };

    auto load = [&](uint32_t n) {
        const uint32_t base = uniform(buffer(n) + cw * LOADS * 1024);
        if constexpr (LOADS == 2) load_shared_half(at, base);
        else
#pragma unroll
            for (int i = 0; i < LOADS; i += 4) load_shared(at + i, base + i * 1024);
    };

    // ---- columns ----
    X x;
    uint32_t column[CT], seen[CT], request[CT];  // keys that a column sees (one that attends nothing: all of them, for no state)
    bool live[CT];
    // what all of it starts with, on its way together: positions, query rows, page numbers
    int64_t position[CT];
    uint32_t lead[CT];  // the first entry of the request's row of the table
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        column[ct] = (block * CW * CT + cw * CT + ct) * kColumns + c;
        const bool real = column[ct] < p.columns;
        request[ct] = real ? divide(column[ct], p.by_group) : 0;
        const uint32_t i = column[ct] - request[ct] * p.by_group.d;
        position[ct] = p.positions[request[ct]];
        lead[ct] = (uint32_t)p.table[(uint64_t)request[ct] * p.table_sb];
        if (!real) position[ct] = -1;
        x.load_query(ct, p.q + ((uint64_t)request[ct] * p.q_sb + (uint64_t)(head * p.by_group.d + (real ? i : 0)) * p.q_sh) * 16, g, real && !p.zero, p.flip);
    }
    uint32_t first_id = (uint32_t)p.table[entry0 + min((uint32_t)tid, last_entry)];
    const bool first_leads = uniform((uint32_t)p.table[0]) < p.pages;
    if (tid == 0) {
        s.least = p.keys;
        s.odd = s.holes = 0;
        s.row = p.batch;
    }
    __syncthreads();
    // The entries are those of the first row whose first one is a page: a retired request's row holds none.  Where no row's is, row 0's.
    uint32_t row = 0;
    bool leads = first_leads;
    if (!first_leads) {
        for (uint32_t b = tid; b < p.batch; b += kThreads)
            if ((uint32_t)p.table[(uint64_t)b * p.table_sb] < p.pages) {
                atomicMin(&s.row, b);
                break;
            }
        __syncthreads();
        leads = uniform(s.row) < p.batch;
        if (leads) {
            row = uniform(s.row);
            first_id = (uint32_t)p.table[(uint64_t)row * p.table_sb + entry0 + min((uint32_t)tid, last_entry)];
        }
    }
    const int32_t *table = p.table + (uint64_t)row * p.table_sb + entry0;
    for (uint32_t i = tid; i <= last_entry; i += kThreads) {
        const uint32_t id = i == (uint32_t)tid ? first_id : (uint32_t)table[i], none = id >= p.pages;
        auto first = [&](const char *pool, uint32_t page_stride, uint32_t head_stride) {
            return reinterpret_cast<uint64_t>(pool) + ((uint64_t)(none ? 0 : id) * page_stride + (uint64_t)head * head_stride) * 16 - kBias + none;
        };
        s.pages[i][0] = first(p.kp, p.kp_sp, p.kp_sh);
        s.pages[i][1] = first(p.vp, p.vp_sp, p.vp_sh);
        if (none) s.holes = 1;
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        live[ct] = position[ct] >= 0 && position[ct] < (int64_t)p.ctx && (lead[ct] < p.pages) == leads;
        seen[ct] = live[ct] && position[ct] < (int64_t)p.keys ? (uint32_t)position[ct] + 1 : p.keys;
        if (seen[ct] < p.keys) atomicMin(&s.least, seen[ct]);
    }
    x.place(g, c);
    x.clear();
    x.settle();
    __syncthreads();
    const uint32_t least = uniform(s.least);
    holes = uniform(s.holes);

    float m[CT], w[CT][TILES][4];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) m[ct] = -INFINITY;
    // exponents are unit (v - m) in log2 units: v the products themselves, or, under a mask, the natural scores
    // (a threshold that is finite: m is below any score at first)
    const float unit = MASK ? kLog2e : p.scale, threshold = fminf(X::threshold / unit, __FLT_MAX__);
    auto partial = [&](uint32_t key0) { return MASK || key0 + SK > least; };
    // Stage n, whose loads of this wave have ended.  Value rows of keys that do not exist become zeros: zero times NaN would
    // be NaN.
    auto arrived = [&](uint32_t n, uint32_t here) {
        if (here == kAll) return;
        const uint32_t at = buffer(n);
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            if (is_value(i) && !(here >> row_of(i) & 1u)) lds_write16(at + (cw * LOADS + i) * 1024 + lane * 16, U4{0u, 0u, 0u, 0u});
    };
    // The mask's words of stage n, four keys of a column at once where they lie so, and the terms in them.
    uint32_t words[CT][TILES][4] = {};
    float terms[MASK ? CT : 1][TILES][4] = {};
    auto fetch_terms = [&](uint32_t n) {
        if constexpr (MASK) {
            const uint32_t key0 = begin + (n * KW + group) * SK;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    uint32_t (&to)[4] = words[ct][t];
                    const uint32_t key = key0 + 16 * t + 4 * g;
                    const uint64_t row = (uint64_t)request[ct] * p.m_sb;
                    if (p.mask_vec) {
                        const uint64_t at = row + min(key, end - 4);
                        if (p.mask_dtype == Q3T_F32) {
                            const U4 x = load16(p.mask + at * 4);
                            to[0] = x.x; to[1] = x.y; to[2] = x.z; to[3] = x.w;
                        } else if (p.mask_dtype == Q3T_BOOL) {
                            to[0] = *reinterpret_cast<const uint32_t *>(p.mask + at);
                        } else {
                            const uint2 x = *reinterpret_cast<const uint2 *>(p.mask + at * 2);
                            to[0] = x.x; to[1] = x.y;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint64_t at = row + (uint64_t)min(key + i, end - 1) * p.m_st;
                            to[i] = p.mask_dtype == Q3T_F32 ? reinterpret_cast<const uint32_t *>(p.mask)[at]
                                  : p.mask_dtype == Q3T_BOOL ? reinterpret_cast<const uint8_t *>(p.mask)[at]
                                                             : reinterpret_cast<const uint16_t *>(p.mask)[at];
                        }
                    }
                }
        }
    };
    auto read_terms = [&] {
        if constexpr (MASK) {
            const int of_word = !p.mask_vec || p.mask_dtype == Q3T_F32 ? 1 : p.mask_dtype == Q3T_BOOL ? 4 : 2;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t (&from)[4] = words[ct][t];
                        const uint32_t e = of_word == 1 ? from[i] : of_word == 4 ? from[0] >> 8 * i : from[i / 2] >> 16 * (i & 1);
                        terms[ct][t][i] = mask_term(e, p.mask_dtype);
                    }
        }
    };
    auto scores = [&] {
        f32x4_t score[CT][TILES];
        x.scores(score);
#pragma unroll
        for (int k = 0; k < CT * TILES * 4; ++k) w[k / (TILES * 4)][k / 4 % TILES][k % 4] = score[k / (TILES * 4)][k / 4 % TILES][k % 4];
    };
    auto softmax = [&](uint32_t n, uint32_t here) {
        const uint32_t key0 = begin + (n * KW + group) * SK;
        if (here != kAll || partial(key0)) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    float term[4] = {};
                    if constexpr (MASK)
#pragma unroll
                        for (int i = 0; i < 4; ++i) term[i] = terms[ct][t][i];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t k = 16 * t + 4 * g + i;
                        const bool hidden = !(here >> k & 1u) || key0 + k >= seen[ct] || term[i] == -INFINITY;
                        w[ct][t][i] = hidden ? -INFINITY : MASK ? w[ct][t][i] * p.scale + term[i] : w[ct][t][i];
                    }
                }
        }
        float highest[CT];
        bool pass = false;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            highest[ct] = w[ct][0][0];
#pragma unroll
            for (int k = 1; k < TILES * 4; ++k) highest[ct] = fmaxf(highest[ct], w[ct][k / 4][k % 4]);
            pass |= highest[ct] > m[ct] + threshold;
        }
        if (__builtin_amdgcn_ballot_w64(pass)) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                float top = fmaxf(highest[ct], m[ct]);
                top = fmaxf(top, xor16(top));
                top = fmaxf(top, xor32(top));
                x.rescale(ct, fexp2((m[ct] - (top == -INFINITY ? 0.f : top)) * unit));
                m[ct] = top;
            }
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            // (under a mask the difference first: a mask's lowest term times the unit is no float32)
            const float top = m[ct] == -INFINITY ? 0.f : m[ct], from = X::shift - top * unit;
#pragma unroll
            for (int k = 0; k < TILES * 4; ++k) {
                float &e = w[ct][k / 4][k % 4];
                e = fexp2(MASK ? __builtin_fmaf(e - top, unit, X::shift) : __builtin_fmaf(e, unit, from));
            }
            x.weights(ct, w[ct]);
        }
    };

    if constexpr (CW == 1) {
        // each wave has stages of its own, and no barriers
        uint32_t here = locate(0);
        load(0);
        fetch_terms(0);
        for (uint32_t n = 0; n < sets; ++n) {
            wait_loads<0>();
            read_terms();
            arrived(n, here);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the other buffer's reads have returned, too)
            uint32_t next = 0;
            if (n + 1 < sets) {
                next = locate(n + 1);
                load(n + 1);
                fetch_terms(n + 1);
            }
            x.read_keys(buffer(n));
            scores();
            x.read_values(buffer(n));  // on their way during the softmax
            softmax(n, here);
            x.values();
            here = next;
        }
    } else {
        // Two groups of waves in turn: while one multiplies, the values of its last stage and the scores of the next, the other one
        // works out its weights, so that matrix cores and vector units are both busy.  Four buffers: of the stages whose values and
        // whose keys are read, and of two that are on their way.
        static_assert(B == 4, "");
        uint32_t exists[4];  // of stages n ... n + 3
        exists[0] = locate(0);
        load(0);
        exists[1] = exists[2] = exists[3] = 0;
        if (sets > 1) {
            exists[1] = locate(1);
            load(1);
            wait_loads<LOADS>();
        } else {
            wait_loads<0>();
        }
        if (sets > 2) exists[2] = locate(2);
        arrived(0, exists[0]);
        lds_barrier();
        if (group) lds_barrier();
        for (uint32_t n = 0; n < sets; ++n) {
            __builtin_amdgcn_s_setprio(1);
            // (the terms' words are waited for below, and what is on its way before them: the next stage, which is needed then)
            if (MASK) fetch_terms(n);
            else if (n + 2 < sets) load(n + 2);
            if (n) x.read_values(buffer(n - 1));
            x.read_keys(buffer(n));
            if (n) x.values();
            scores();
            __builtin_amdgcn_s_setprio(0);
            lds_barrier();
            if (!MASK && n + 3 < sets) exists[3] = locate(n + 3);
            read_terms();
            softmax(n, exists[0]);
            if (MASK && n + 2 < sets) load(n + 2);
            if (n + 2 < sets) wait_loads<LOADS>();
            else wait_loads<0>();
            if (n + 1 < sets) arrived(n + 1, exists[1]);
            if (MASK && n + 3 < sets) exists[3] = locate(n + 3);
#pragma unroll
            for (int i = 0; i < 3; ++i) exists[i] = exists[i + 1];
            lds_barrier();
        }
        x.read_values(buffer(sets - 1));
        x.values();
        if (!group) lds_barrier();
    }

    // ---- the groups' states, into the first one's ----
    float l[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        l[ct] = x.total(ct);
        // A value that is not finite leaves the sums of its dim so, whatever its weight.  (Where the weights are not either, so is
        // what they should give.)
        bool fine = true;
#pragma unroll
        for (int a = 0; a < D / 16; ++a)
#pragma unroll
            for (int i = 0; i < 4; ++i) fine &= __builtin_fabsf(x.acc[ct][a][i]) < INFINITY;
        if (live[ct] && !fine && __builtin_fabsf(l[ct]) < INFINITY) s.odd = 1;
    }
    lds_barrier();  // all have left the last stage
    if (tid == 0) p.odd[task * p.blocks + block] = s.odd;
    if constexpr (KW > 1) {
        if (group > 0) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                s.ml[group][cw][ct][0][lane] = m[ct];
                s.ml[group][cw][ct][1][lane] = l[ct];
#pragma unroll
                for (int a = 0; a < D / 16; ++a) s.merge[group - 1][cw][ct][a][lane] = x.acc[ct][a];
            }
        }
        lds_barrier();
        if (group > 0) return;
#pragma unroll
        for (int n = 1; n < KW; ++n)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const float om = s.ml[n][cw][ct][0][lane], top = fmaxf(m[ct], om), from = top == -INFINITY ? 0.f : top;
                const float e0 = fexp2((m[ct] - from) * unit), e1 = fexp2((om - from) * unit);
                l[ct] = l[ct] * e0 + s.ml[n][cw][ct][1][lane] * e1;
                m[ct] = top;
#pragma unroll
                for (int a = 0; a < D / 16; ++a) x.acc[ct][a] = x.acc[ct][a] * e0 + s.merge[n - 1][cw][ct][a][lane] * e1;
            }
    }
    const uint64_t rows = ((uint64_t)part * p.heads + head) * p.columns;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        if (column[ct] >= p.columns) continue;
        const bool none = !live[ct] || l[ct] == 0.f;
        if (g == 0) *reinterpret_cast<f32x2_t *>(p.ml + 2 * (rows + column[ct])) = none ? f32x2_t{-INFINITY, 0.f} : f32x2_t{MASK ? m[ct] : m[ct] * unit, l[ct]};
#pragma unroll
        for (int a = 0; a < D / 16; ++a)
            *reinterpret_cast<f32x4_t *>(p.states + (rows + column[ct]) * D + X::dim(a, g)) = none ? f32x4_t{0.f, 0.f, 0.f, 0.f} : x.four(ct, a);
    }
}

// What a launch over a prefix does.
struct PrefixPlan {
    int64_t cw, kw, ct, columns, blocks, parts, chunk, step;  // step: keys of a stage for every group
    int64_t states, workgroups, bytes;  // states: in all
};

// By sizes alone: tiles for the columns that there are, and a part for each CU that blocks and heads leave, but some keys each at
// least, as a state is written and read again for every part, and no more than a request's end reads at once (8 for groups of 16 query
// heads of 128: with few KV heads the card is not filled).  Only pages of few rows, of which a workgroup knows 1022, make more parts:
// 896 keys each in pages of one row.  us of both launches with 64 / 256 / 512 keys at least, bf16, weights in one part: 64 requests
// over 4096 keys 57.6 / 56.2 / 57.2, 64 over 2048 30.0 / 27.8 / 31.9, 32 over 1024 19.5 / 20.2 / 24.0, 128 over 1024 46.9 / 42.3 / 44.7;
// with 64 / 128 / 256, float32 under a mask: 21 over 792 25.3 / 27.2 / 33.0.

template <typename T>
static PrefixPlan prefix_plan(const q3t_paged_args *a, int64_t keys) {
    PrefixPlan z;
    z.columns = a->batch * (a->q_heads / a->kv_heads);
    z.ct = z.columns <= kColumns || (z.columns > 2 * kColumns && z.columns <= 4 * kColumns) ? 1 : 2;
    z.cw = z.columns <= 2 * kColumns ? 1 : 4;
    z.kw = z.cw == 4 ? 2 : 4;
    z.blocks = (z.columns + z.cw * z.ct * kColumns - 1) / (z.cw * z.ct * kColumns);
    const int64_t step = z.step = z.kw * (sizeof(T) == 4 ? 16 : 32), workgroups = 256;
    int64_t parts = workgroups / (z.blocks * a->kv_heads);
    // each request's end reads the states of its columns: up to eight for a thread of 512, as far as pages allow
    const int64_t group = a->q_heads / a->kv_heads, most_parts = 16384 / ((group < kColumns ? group : kColumns) * a->head_dim);
    if (parts > most_parts) parts = most_parts;
    if (parts < 1) parts = 1;
    z.chunk = (keys + parts - 1) / parts;
    const int64_t least = sizeof(T) == 4 ? 64 : 256;
    if (z.chunk < least) z.chunk = least;
    z.chunk = (z.chunk + step - 1) / step * step;
    const int64_t most = (kEntries - 2) * a->page_size / step * step;  // whose page numbers a workgroup holds
    if (z.chunk > most) z.chunk = most;
    z.parts = (keys + z.chunk - 1) / z.chunk;
    z.states = z.parts * a->kv_heads * z.columns;
    z.workgroups = z.parts * a->kv_heads * z.blocks;
    z.bytes = (z.states * (a->head_dim + 2) + z.workgroups) * 4;
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
    x.ml = states + z.states * a->head_dim;
    x.odd = (uint32_t *)(x.ml + 2 * z.states);
    x.q_sb = p.q_sb; x.q_sh = p.q_sh;
    x.kp_sp = p.kp_sp; x.kp_sh = p.kp_sh; x.kp_st = p.kp_st; x.vp_sp = p.vp_sp; x.vp_sh = p.vp_sh; x.vp_st = p.vp_st;
    x.m_sb = p.m_sb; x.m_st = p.m_st; x.mask_dtype = p.mask_dtype;
    const int64_t mask_size = a->mask_dtype == Q3T_F32 ? 4 : a->mask_dtype == Q3T_BOOL ? 1 : 2;
    x.mask_vec = p.m_st == 1 && p.m_sb % 4 == 0 && aligned(mask, 4 * mask_size) && keys % 4 == 0;
    x.heads = (uint32_t)a->kv_heads; x.columns = (uint32_t)z.columns; x.blocks = (uint32_t)z.blocks;
    x.parts = (uint32_t)z.parts; x.keys = (uint32_t)keys; x.chunk = (uint32_t)z.chunk;
    x.pages = p.pages;
    x.ctx = (uint32_t)(a->ctx + keys);
    x.table_sb = p.table_sb; x.batch = (uint32_t)a->batch;
    x.by_page = p.by_page;
    x.by_group = divisor(p.group);
    x.scale = p.scale;
    if (!mask) {
        x.flip = p.scale < 0.f;
        x.zero = p.scale == 0.f;
        x.scale = x.zero ? 1.f : p.scale < 0.f ? -p.scale : p.scale;
    }
    const int64_t units = a->kv_heads * z.parts;
    const dim3 grid((uint32_t)((units + 7) / 8 * 8 * z.blocks));
    // (offsets within a page have 32 bits)
    const int64_t stage = sizeof(T) == 4 ? 16 : 32, rows = 1024 / (a->head_dim * (int64_t)sizeof(T));
    const bool whole = (a->page_size % stage == 0 || (stage % a->page_size == 0 && a->page_size % rows == 0)) &&
                       (int64_t)(p.kp_st > p.vp_st ? p.kp_st : p.vp_st) * a->page_size < (1 << 27) - 1024;
    auto shape = [&](auto d, auto masked, auto in_one) {
        constexpr int D = decltype(d)::value;
        constexpr bool MASK = decltype(masked)::value, WHOLE = decltype(in_one)::value;
        auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3((uint32_t)(64 * z.cw * z.kw)), 0, stream, x); };
        if (z.cw == 4 && z.ct == 2) launch(prefix_kernel<T, D, MASK, WHOLE, 4, 2, 2>);
        else if (z.cw == 4) launch(prefix_kernel<T, D, MASK, WHOLE, 4, 2, 1>);
        else if (z.ct == 2) launch(prefix_kernel<T, D, MASK, WHOLE, 1, 4, 2>);
        else launch(prefix_kernel<T, D, MASK, WHOLE, 1, 4, 1>);
    };
    auto width = [&](auto masked, auto in_one) {
        if (a->head_dim == 128) shape(std::integral_constant<int, 128>{}, masked, in_one);
        else shape(std::integral_constant<int, 64>{}, masked, in_one);
    };
    auto pages = [&](auto masked) {
        if (whole) width(masked, std::true_type{});
        else width(masked, std::false_type{});
    };
    if (mask) pages(std::true_type{});
    else pages(std::false_type{});
    return launch_status();
}

}  // namespace paged
}  // namespace q3t
