// New key/value rows into a cache kept in pages (the paged counterpart of q3t_kv_write; reference:
// continuous.py:152-166, 118-132).
//
// A copy: bound by HBM for a batch of prompts, by the launch for a decode step.  A workgroup takes
// rows of one request, in the order token, head, vector (the fused projection's own order); the
// rows are loaded while the position and the page number are on their way.  Workgroups past a
// request's length end at once.
#include "paged_index.hpp"
#include "q3t_common.hpp"

namespace q3t {
namespace paged_write {

constexpr int kThreads = 256;

template <int V> struct Unit;
template <> struct Unit<16> { typedef U4 T; };
template <> struct Unit<8> { typedef uint2 T; };
template <> struct Unit<4> { typedef uint32_t T; };
template <> struct Unit<2> { typedef uint16_t T; };

struct Params {
    const char *k, *v;
    char *kp, *vp;
    const int32_t *table;
    const int64_t *positions;
    const int32_t *lengths;
    int64_t k_sb, k_sh, k_st, v_sb, v_sh, v_st;           // bytes
    int64_t kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st;     // bytes
    int64_t table_sb, rows;                               // rows: table_width * page_size
    uint32_t batch, heads, tokens, units, pages;
    Divisor by_units, by_heads, by_page;
};

template <int V>
__global__ void __launch_bounds__(kThreads) paged_write_kernel(Params p) {
    typedef typename Unit<V>::T T;
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    const uint32_t row = divide(i, p.by_units), c = i - row * p.units;
    const uint32_t t = divide(row, p.by_heads), h = row - t * p.heads;
    for (uint32_t b = blockIdx.y; b < p.batch; b += gridDim.y) {
        const uint32_t used = p.lengths ? (uint32_t)max(0, min(p.lengths[b], (int32_t)p.tokens)) : p.tokens;
        if (t >= used) continue;
        const int64_t start = p.positions[b];
        const T kv = *reinterpret_cast<const T *>(p.k + b * p.k_sb + h * p.k_sh + t * p.k_st + (int64_t)c * V);
        const T vv = *reinterpret_cast<const T *>(p.v + b * p.v_sb + h * p.v_sh + t * p.v_st + (int64_t)c * V);
        // start + t overflows for no start that is left
        if (start >= p.rows || start < -(int64_t)p.tokens || start + t < 0 || start + t >= p.rows) continue;
        const uint32_t j = (uint32_t)(start + t), at = divide(j, p.by_page), r = j - at * p.by_page.d;
        const int32_t page = p.table[b * p.table_sb + at];
        if ((uint32_t)page >= p.pages) continue;
        *reinterpret_cast<T *>(p.kp + page * p.kp_sp + h * p.kp_sh + r * p.kp_st + (int64_t)c * V) = kv;
        *reinterpret_cast<T *>(p.vp + page * p.vp_sp + h * p.vp_sh + r * p.vp_st + (int64_t)c * V) = vv;
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
    p.table = a->page_table; p.positions = a->positions; p.lengths = a->lengths;
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
    if (a->heads > INT32_MAX / p.units || a->tokens > (INT32_MAX - kThreads) / (a->heads * p.units)) return Q3T_EUNSUPPORTED;
    const int64_t blocks = (a->tokens * a->heads * p.units + kThreads - 1) / kThreads;
    const int64_t most = ((int64_t)1 << 24) - 1;
    if (blocks > most) return Q3T_EUNSUPPORTED;
    int64_t across = a->batch < 65535 ? a->batch : 65535;
    if (across > most / blocks) across = most / blocks;
    p.by_units = divisor(p.units);
    p.by_heads = divisor(p.heads);
    p.by_page = divisor((uint32_t)a->page_size);
    const dim3 grid((uint32_t)blocks, (uint32_t)across);
    hipStream_t s = (hipStream_t)stream;
    switch (v) {
        case 16: hipLaunchKernelGGL(paged_write_kernel<16>, grid, dim3(kThreads), 0, s, p); break;
        case 8: hipLaunchKernelGGL(paged_write_kernel<8>, grid, dim3(kThreads), 0, s, p); break;
        case 4: hipLaunchKernelGGL(paged_write_kernel<4>, grid, dim3(kThreads), 0, s, p); break;
        default: hipLaunchKernelGGL(paged_write_kernel<2>, grid, dim3(kThreads), 0, s, p); break;
    }
    return launch_status();
}
