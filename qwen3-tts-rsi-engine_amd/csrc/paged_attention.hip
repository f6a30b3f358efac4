// Attention of one new token per request over a cache kept in pages (the paged counterpart of the
// decode attention; reference: packed_attention.py:75-84).
//
// The plain form: one workgroup per (request, query head), its waves taking keys in turn with one
// softmax state each, merged in LDS.
#include "paged_index.hpp"
#include "q3t_common.hpp"

namespace q3t {
namespace paged {

struct Params {
    const char *q, *kp, *vp, *mask;
    char *out;
    const int32_t *table;
    const int64_t *positions;
    int64_t q_sb, q_sh, o_sb, o_sh, kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st;  // bytes
    int64_t m_sb, m_st, table_sb;                                              // elements
    int32_t ctx, mask_dtype;
    uint32_t pages, q_heads, group;
    Divisor by_page, by_heads;
    float scale;
};

Q3T_DEVICE float mask_value(const char *m, int64_t i, int dtype) {
    switch (dtype) {
        case Q3T_BF16: return bf16_to_float(reinterpret_cast<const uint16_t *>(m)[i]);
        case Q3T_F16: return (float)reinterpret_cast<const _Float16 *>(m)[i];
        case Q3T_F32: return reinterpret_cast<const float *>(m)[i];
        default: return m[i] ? 0.0f : -INFINITY;
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(256) paged_plain_kernel(Params p) {
    constexpr int E = D / 64;
    __shared__ float sm[4], sl[4], sa[4][D];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t b = divide(blockIdx.x, p.by_heads), hq = blockIdx.x - b * p.q_heads, h = hq / p.group;
    const int64_t pos = p.positions[b];
    const int length = pos >= 0 && pos < p.ctx ? (int)pos + 1 : 0;
    const T *q = reinterpret_cast<const T *>(p.q + b * p.q_sb + hq * p.q_sh);
    float qv[E], acc[E] = {}, m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; ++e) qv[e] = (float)q[lane * E + e];
    for (int j = wave; j < length; j += 4) {
        const uint32_t at = divide((uint32_t)j, p.by_page), r = j - at * p.by_page.d;
        const int32_t page = p.table[b * p.table_sb + at];
        const float term = p.mask ? mask_value(p.mask, b * p.m_sb + j * p.m_st, p.mask_dtype) : 0.f;
        if ((uint32_t)page >= p.pages || term == -INFINITY) continue;
        const T *k = reinterpret_cast<const T *>(p.kp + page * p.kp_sp + h * p.kp_sh + r * p.kp_st);
        const T *v = reinterpret_cast<const T *>(p.vp + page * p.vp_sp + h * p.vp_sh + r * p.vp_st);
        float s = 0.f;
        for (int e = 0; e < E; ++e) s += qv[e] * (float)k[lane * E + e];
        for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
        s = s * p.scale + term;
        const float mn = fmaxf(m, s), shift = mn == -INFINITY ? 0.f : mn;
        const float alpha = expf(m - shift), w = expf(s - shift);
        l = l * alpha + w;
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * alpha + w * (float)v[lane * E + e];
        m = s != s ? s : mn;
    }
    if (lane == 0) {
        sm[wave] = m;
        sl[wave] = l;
    }
    for (int e = 0; e < E; ++e) sa[wave][lane * E + e] = acc[e];
    __syncthreads();
    if (threadIdx.x >= D) return;
    float mm = -INFINITY, tl = 0.f, ta = 0.f;
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sm[w]);
    const float shift = mm == -INFINITY ? 0.f : mm;
    for (int w = 0; w < 4; ++w) {
        const float x = expf(sm[w] - shift);
        tl += sl[w] * x;
        ta += sa[w][threadIdx.x] * x;
    }
    const float y = tl == 0.f ? 0.f : ta / tl;
    reinterpret_cast<T *>(p.out + b * p.o_sb + hq * p.o_sh)[threadIdx.x] = (T)y;
}

template <typename T>
static void launch(const Params &p, int64_t D, uint32_t blocks, hipStream_t s) {
    if (D == 64) hipLaunchKernelGGL((paged_plain_kernel<T, 64>), dim3(blocks), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((paged_plain_kernel<T, 128>), dim3(blocks), dim3(256), 0, s, p);
}

// Sizes that this operator takes; Q3T_OK, or the status to return.
static int check_sizes(const q3t_paged_args *a) {
    if (!a || a->batch < 0 || a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads || a->ctx < 1 || a->pages < 1 ||
        a->page_size < 1 || a->table_width < 1)
        return Q3T_EINVAL;
    if (a->dtype != Q3T_BF16 && a->dtype != Q3T_F16 && a->dtype != Q3T_F32) return Q3T_EUNSUPPORTED;
    if (a->head_dim != 64 && a->head_dim != 128) return Q3T_EUNSUPPORTED;
    if (a->pages > INT32_MAX || a->page_size > INT32_MAX || a->table_width > INT32_MAX) return Q3T_EUNSUPPORTED;
    if (a->ctx > a->table_width * a->page_size) return Q3T_EINVAL;
    if (a->ctx >= 1 << 30 || a->batch > 1 << 16 || a->q_heads > 1 << 16 || a->batch * a->q_heads > 1 << 20) return Q3T_EUNSUPPORTED;
    return Q3T_OK;
}

}  // namespace paged
}  // namespace q3t

using namespace q3t;

extern "C" int64_t q3t_paged_workspace_bytes(const q3t_paged_args *a) {
    return paged::check_sizes(a) == Q3T_OK ? 0 : -1;
}

extern "C" int q3t_paged_attention(const q3t_paged_args *a, void *stream) {
    using namespace paged;
    const int status = check_sizes(a);
    if (status != Q3T_OK) return status;
    if (a->batch == 0) return Q3T_OK;
    if (!a->query || !a->key_pages || !a->value_pages || !a->page_table || !a->positions || !a->out) return Q3T_EINVAL;
    if (a->mask && (a->mask_dtype < Q3T_BF16 || a->mask_dtype > Q3T_BOOL)) return Q3T_EINVAL;
    const int64_t es = a->dtype == Q3T_F32 ? 4 : 2;
    Params p = {};
    p.q = (const char *)a->query; p.kp = (const char *)a->key_pages; p.vp = (const char *)a->value_pages;
    p.mask = (const char *)a->mask; p.out = (char *)a->out;
    p.table = a->page_table; p.positions = a->positions;
    p.q_sb = a->q_stride_b * es; p.q_sh = a->q_stride_h * es;
    p.o_sb = a->o_stride_b * es; p.o_sh = a->o_stride_h * es;
    p.kp_sp = a->kp_stride_p * es; p.kp_sh = a->kp_stride_h * es; p.kp_st = a->kp_stride_t * es;
    p.vp_sp = a->vp_stride_p * es; p.vp_sh = a->vp_stride_h * es; p.vp_st = a->vp_stride_t * es;
    p.m_sb = a->mask_stride_b; p.m_st = a->mask_stride_t; p.table_sb = a->table_stride_b;
    if ((p.q_sb | p.q_sh | p.kp_sp | p.kp_sh | p.kp_st | p.vp_sp | p.vp_sh | p.vp_st) % 16 || !aligned(p.q, 16) ||
        !aligned(p.kp, 16) || !aligned(p.vp, 16) || !aligned(p.out, es) || !aligned(p.table, 4) || !aligned(p.positions, 8))
        return Q3T_EINVAL;
    p.ctx = (int32_t)a->ctx; p.mask_dtype = (int32_t)a->mask_dtype;
    p.pages = (uint32_t)a->pages; p.q_heads = (uint32_t)a->q_heads; p.group = (uint32_t)(a->q_heads / a->kv_heads);
    p.by_page = divisor((uint32_t)a->page_size);
    p.by_heads = divisor(p.q_heads);
    p.scale = a->scale;
    const uint32_t blocks = (uint32_t)(a->batch * a->q_heads);
    hipStream_t s = (hipStream_t)stream;
    if (a->dtype == Q3T_F32) launch<float>(p, a->head_dim, blocks, s);
    else if (a->dtype == Q3T_BF16) launch<__bf16>(p, a->head_dim, blocks, s);
    else launch<_Float16>(p, a->head_dim, blocks, s);
    return launch_status();
}
