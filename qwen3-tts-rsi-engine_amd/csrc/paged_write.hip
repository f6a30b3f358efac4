// New key/value rows into a cache kept in pages (the paged counterpart of q3t_kv_write; reference:
// continuous.py:152-166, 118-132).
//
// A copy: bound by HBM for a batch of prompts (16 of 60..1024 rows, 74 MB, 16.7 us, 4.5 TB/s; a plain
// copy of as many bytes 15.7), by the launch for a decode step (64 rows 2.9 us).  A workgroup takes
// rows of one request, in the order token, head, vector (the fused projection's own order); the
// rows are loaded while the position and the page number are on their way.  Workgroups past a
// request's length end at once.
#include "paged_index.hpp"
#include "q3t_common.hpp"

namespace q3t {
namespace paged_write {

constexpr int kThreads = 256;
constexpr int64_t kManyBlocks = 2048;  // workgroups of one unit a thread that the card holds at once

// Units of V bytes, read and written once each: the non-temporal policy (16 prompts 16.6 us; plain stores 17.4,
// plain loads 17.6, both 19.2; a launch of 64 requests' rows and the attention over them the same).
template <int V> struct Unit { typedef uint32_t T __attribute__((ext_vector_type(V / 4))); };
template <> struct Unit<4> { typedef uint32_t T; };
template <> struct Unit<2> { typedef uint16_t T; };

struct Params {
    const char *k, *v;
    char *kp, *vp;
    const int32_t *table;
    int64_t k_sb, k_sh, k_st, v_sb, v_sh, v_st;           // bytes
    int64_t kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st;     // bytes
    int64_t table_sb, rows;                               // rows: table_width * page_size
    uint32_t batch, heads, tokens, units, pages;
    Divisor by_units, by_heads, by_page;
};

// N units a thread, 256 apart, all of their rows on the way before the first is stored.  With one unit
// (launches of few rows) they are on the way before anything else is known; with more, rows past a
// request's length are not read.
template <int V, int N>
__global__ void __launch_bounds__(kThreads)
paged_write_kernel(const int64_t *__restrict__ positions, const int32_t *__restrict__ lengths, Params p) {
    typedef typename Unit<V>::T T;
    for (uint32_t b = blockIdx.y; b < p.batch; b += gridDim.y) {
        const int64_t start = positions[b];
        const uint32_t used = lengths ? (uint32_t)max(0, min(lengths[b], (int32_t)p.tokens)) : p.tokens;
        T kv[N], vv[N];
        uint32_t t[N];
        int64_t at_k[N], at_v[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const uint32_t i = (blockIdx.x * N + n) * kThreads + threadIdx.x;
            const uint32_t row = divide(i, p.by_units), h = row - divide(row, p.by_heads) * p.heads;
            const int64_t unit = (int64_t)(i - row * p.units) * V;
            t[n] = divide(row, p.by_heads);
            at_k[n] = h * p.kp_sh + unit;
            at_v[n] = h * p.vp_sh + unit;
            if (t[n] >= (N == 1 ? p.tokens : used)) continue;
            kv[n] = __builtin_nontemporal_load(reinterpret_cast<const T *>(p.k + b * p.k_sb + h * p.k_sh + t[n] * p.k_st + unit));
            vv[n] = __builtin_nontemporal_load(reinterpret_cast<const T *>(p.v + b * p.v_sb + h * p.v_sh + t[n] * p.v_st + unit));
        }
        int32_t page[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            page[n] = -1;
            // (start + t overflows for no start that is left)
            if (t[n] >= used || start >= p.rows || start < -(int64_t)p.tokens || start + t[n] < 0 || start + t[n] >= p.rows) continue;
            const uint32_t j = (uint32_t)(start + t[n]), entry = divide(j, p.by_page), r = j - entry * p.by_page.d;
            page[n] = p.table[b * p.table_sb + entry];
            at_k[n] += r * p.kp_st;
            at_v[n] += r * p.vp_st;
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if ((uint32_t)page[n] >= p.pages) continue;
            __builtin_nontemporal_store(kv[n], reinterpret_cast<T *>(p.kp + page[n] * p.kp_sp + at_k[n]));
            __builtin_nontemporal_store(vv[n], reinterpret_cast<T *>(p.vp + page[n] * p.vp_sp + at_v[n]));
        }
    }
}

}  // namespace paged_write
}  // namespace q3t

using namespace q3t;

extern "C" int q3t_paged_write(const q3t_paged_write_args *a, void *stream) {
    using namespace paged_write;
    if (!a || a->batch < 0 || a->heads < 1 || a->tokens < 0 || a->width < 1 || a->pages < 1 || a->page_size < 1 ||
        a->table_width < 1)
        return Q3T_EINVAL;
    if (a->elem_size != 2 && a->elem_size != 4) return Q3T_EUNSUPPORTED;
    if (a->batch == 0 || a->tokens == 0) return Q3T_OK;
    if (!a->keys || !a->values || !a->key_pages || !a->value_pages || !a->page_table || !a->positions) return Q3T_EINVAL;
    if (a->pages > INT32_MAX || a->table_width > INT32_MAX / a->page_size || a->batch > INT32_MAX || a->width > 1 << 20)
        return Q3T_EUNSUPPORTED;
    const int64_t es = a->elem_size;
    Params p = {};
    p.k = (const char *)a->keys; p.v = (const char *)a->values;
    p.kp = (char *)a->key_pages; p.vp = (char *)a->value_pages;
    p.table = a->page_table;
    p.k_sb = a->k_stride_b * es; p.k_sh = a->k_stride_h * es; p.k_st = a->k_stride_t * es;
    p.v_sb = a->v_stride_b * es; p.v_sh = a->v_stride_h * es; p.v_st = a->v_stride_t * es;
    p.kp_sp = a->kp_stride_p * es; p.kp_sh = a->kp_stride_h * es; p.kp_st = a->kp_stride_t * es;
    p.vp_sp = a->vp_stride_p * es; p.vp_sh = a->vp_stride_h * es; p.vp_st = a->vp_stride_t * es;
    p.table_sb = a->table_stride_b;
    p.rows = a->table_width * a->page_size;
    // the widest unit that divides the row, every stride and every pointer
    const int64_t strides = p.k_sb | p.k_sh | p.k_st | p.v_sb | p.v_sh | p.v_st | p.kp_sp | p.kp_sh | p.kp_st |
                            p.vp_sp | p.vp_sh | p.vp_st | (a->width * es) | (int64_t)(uintptr_t)a->keys |
                            (int64_t)(uintptr_t)a->values | (int64_t)(uintptr_t)a->key_pages | (int64_t)(uintptr_t)a->value_pages;
    int64_t v = 16;
    while (v > es && strides % v) v >>= 1;
    if (strides % v || !aligned(a->page_table, 4) || !aligned(a->positions, 8) || (a->lengths && !aligned(a->lengths, 4)))
        return Q3T_EINVAL;
    p.batch = (uint32_t)a->batch; p.heads = (uint32_t)a->heads; p.tokens = (uint32_t)a->tokens;
    p.units = (uint32_t)(a->width * es / v);
    p.pages = (uint32_t)a->pages;
    // items of a request, and the threads of a launch, stay below 2^31 and 2^32
    if (a->heads > INT32_MAX / p.units || a->tokens > (INT32_MAX - 2 * kThreads) / (a->heads * p.units)) return Q3T_EUNSUPPORTED;
    // two units a thread where the card is full all the same (16 prompts of 1024: one 20.2 us, two 16.7, 4 17.3)
    const int64_t units = a->tokens * a->heads * p.units;
    const bool two = units / kThreads * a->batch >= kManyBlocks;
    const int64_t blocks = (units + kThreads * (two ? 2 : 1) - 1) / (kThreads * (two ? 2 : 1));
    const int64_t most = ((int64_t)1 << 24) - 1;
    if (blocks > most) return Q3T_EUNSUPPORTED;
    int64_t across = a->batch < 65535 ? a->batch : 65535;
    if (across > most / blocks) across = most / blocks;
    p.by_units = divisor(p.units);
    p.by_heads = divisor(p.heads);
    p.by_page = divisor((uint32_t)a->page_size);
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks, (uint32_t)across), dim3(kThreads), 0, (hipStream_t)stream,
                           a->positions, a->lengths, p);
    };
    switch (v) {
        case 16: two ? launch(paged_write_kernel<16, 2>) : launch(paged_write_kernel<16, 1>); break;
        case 8: two ? launch(paged_write_kernel<8, 2>) : launch(paged_write_kernel<8, 1>); break;
        case 4: two ? launch(paged_write_kernel<4, 2>) : launch(paged_write_kernel<4, 1>); break;
        default: two ? launch(paged_write_kernel<2, 2>) : launch(paged_write_kernel<2, 1>); break;
    }
    return launch_status();
}
