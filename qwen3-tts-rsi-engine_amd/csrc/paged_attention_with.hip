// Attention of one new token per request over a paged cache of 8-bit rows, or over one whose first pages are
// shared by all requests of the batch.
//
//   s_j = scale ks_j (q . k_j) (+ mask_j),  out = sum_j exp(s_j - m) vs_j v_j / sum_j exp(s_j - m)
//
// A workgroup takes one query head of a request, its waves every fourth key, with a running maximum.
#include "paged_with.hpp"

namespace q3t {
namespace paged_with {

constexpr int kWaves = 4;

struct Params {
    q3t_paged_args a;
    q3t_paged_scales s;
    int64_t shared;  // pages that are request 0's
};

Q3T_DEVICE float element(const void *pool, int64_t at, int64_t type) {
    switch (type) {
        case Q3T_BF16: return bf16_to_float(((const uint16_t *)pool)[at]);
        case Q3T_F16: return (float)((const _Float16 *)pool)[at];
        case Q3T_F32: return ((const float *)pool)[at];
        case Q3T_I8: return (float)((const int8_t *)pool)[at];
        case Q3T_BOOL: return ((const uint8_t *)pool)[at] ? 0.f : -INFINITY;
        default: return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t *)pool)[at], 0);
    }
}

__global__ void __launch_bounds__(64 * kWaves) simple_kernel(Params p) {
    const q3t_paged_args &a = p.a;
    __shared__ float ml[kWaves][2], acc[kWaves][128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, D = (int)a.head_dim, n = D / 64;
    const int64_t b = blockIdx.x / a.q_heads, hq = blockIdx.x % a.q_heads, h = hq / (a.q_heads / a.kv_heads);
    const int64_t position = a.positions[b], length = position >= 0 && position < a.ctx ? position + 1 : 0;
    const int64_t held = p.s.format ? p.s.format : a.dtype;
    float q[2] = {}, o[2] = {}, m = -INFINITY, l = 0.f;
    for (int i = 0; i < n; ++i) q[i] = element(a.query, b * a.q_stride_b + hq * a.q_stride_h + lane + 64 * i, a.dtype);
    for (int64_t j = wave; j < length; j += kWaves) {
        const int64_t entry = j / a.page_size, row = j % a.page_size;
        const int64_t page = a.page_table[(entry < p.shared ? 0 : b * a.table_stride_b) + entry];
        const float term = a.mask ? element(a.mask, b * a.mask_stride_b + j * a.mask_stride_t, a.mask_dtype) : 0.f;
        if (page < 0 || page >= a.pages || term == -INFINITY) continue;
        float s = 0.f;
        for (int i = 0; i < n; ++i)
            s += q[i] * element(a.key_pages, page * a.kp_stride_p + h * a.kp_stride_h + row * a.kp_stride_t + lane + 64 * i, held);
        for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
        s *= a.scale;
        float vs = 1.f;
        if (p.s.format) {
            s *= p.s.key_scales[page * p.s.ks_stride_p + h * p.s.ks_stride_h + row * p.s.ks_stride_t];
            vs = p.s.value_scales[page * p.s.vs_stride_p + h * p.s.vs_stride_h + row * p.s.vs_stride_t];
        }
        s += term;
        const float top = s > m || s != s ? s : m, from = top == -INFINITY ? 0.f : top;
        const float alpha = expf(m - from), w = expf(s - from);
        l = l * alpha + w;
        for (int i = 0; i < n; ++i)
            o[i] = o[i] * alpha + w * vs * element(a.value_pages, page * a.vp_stride_p + h * a.vp_stride_h + row * a.vp_stride_t + lane + 64 * i, held);
        m = top;
    }
    if (lane == 0) { ml[wave][0] = m; ml[wave][1] = l; }
    for (int i = 0; i < n; ++i) acc[wave][lane + 64 * i] = o[i];
    __syncthreads();
    if ((int)threadIdx.x >= D) return;
    float top = -INFINITY, sum = 0.f, y = 0.f;
    for (int w = 0; w < kWaves; ++w) top = ml[w][0] > top || ml[w][0] != ml[w][0] ? ml[w][0] : top;
    const float from = top == -INFINITY ? 0.f : top;
    for (int w = 0; w < kWaves; ++w) {
        const float e = expf(ml[w][0] - from);
        sum += ml[w][1] * e;
        y += acc[w][threadIdx.x] * e;
    }
    y = sum == 0.f ? 0.f : y / sum;
    const int64_t at = b * a.o_stride_b + hq * a.o_stride_h + threadIdx.x;
    if (a.dtype == Q3T_F32) ((float *)a.out)[at] = y;
    else if (a.dtype == Q3T_F16) ((_Float16 *)a.out)[at] = (_Float16)y;
    else ((uint16_t *)a.out)[at] = (uint16_t)float_to_bf16(y);
}

// The sizes of a launch; Q3T_OK, or the status to return.
static int check(const q3t_paged_args *a, const q3t_paged_scales *s, int64_t shared_pages, paged::Sizes &z) {
    if (!a) return Q3T_EINVAL;
    if (s && s->format != Q3T_I8 && s->format != Q3T_E4M3) return Q3T_EUNSUPPORTED;
    const int status = s && s->format == Q3T_I8 ? paged::sizes_int8(a, z) : paged::sizes_e4m3(a, z);
    if (status != Q3T_OK) return status;
    if (shared_pages < 0 || shared_pages > a->table_width || shared_pages * a->page_size >= a->ctx) return Q3T_EINVAL;
    return Q3T_OK;
}

}  // namespace paged_with
}  // namespace q3t

using namespace q3t;

extern "C" int64_t q3t_paged_workspace_bytes_with(const q3t_paged_args *a, const q3t_paged_scales *s, int64_t shared_pages) {
    paged::Sizes z;
    return paged_with::check(a, s, shared_pages, z) == Q3T_OK ? z.workspace : -1;
}

extern "C" int q3t_paged_attention_with(const q3t_paged_args *a, const q3t_paged_scales *s, int64_t shared_pages, void *stream) {
    using namespace paged_with;
    paged::Sizes z;
    const int status = check(a, s, shared_pages, z);
    if (status != Q3T_OK || a->batch == 0) return status;
    if (s && shared_pages == 0)
        return (s->format == Q3T_I8 ? paged::attend_int8 : paged::attend_e4m3)(a, z, s, paged::Behind{}, (hipStream_t)stream);
    if (!a->query || !a->key_pages || !a->value_pages || !a->page_table || !a->positions || !a->out) return Q3T_EINVAL;
    if (s && (!s->key_scales || !s->value_scales || !aligned(s->key_scales, 4) || !aligned(s->value_scales, 4))) return Q3T_EINVAL;
    if (a->mask && (a->mask_dtype < Q3T_BF16 || a->mask_dtype > Q3T_BOOL)) return Q3T_EINVAL;
    const int64_t es = a->dtype == Q3T_F32 ? 4 : 2, held = s ? 1 : es;
    const int64_t query[2] = {a->q_stride_b, a->q_stride_h};
    const int64_t pools[6] = {a->kp_stride_p, a->kp_stride_h, a->kp_stride_t, a->vp_stride_p, a->vp_stride_h, a->vp_stride_t};
    const int64_t others[5] = {a->o_stride_b, a->o_stride_h, a->mask ? a->mask_stride_b : 0, a->mask ? a->mask_stride_t : 0, a->table_stride_b};
    for (int64_t x : query) if (x < 0 || x * es % 16) return Q3T_EINVAL;
    for (int64_t x : pools) if (x < 0 || x * held % 16) return Q3T_EINVAL;
    for (int64_t x : others) if (x < 0) return Q3T_EINVAL;
    const int64_t mask_size = a->mask_dtype == Q3T_F32 ? 4 : a->mask_dtype == Q3T_BOOL ? 1 : 2;
    if (!aligned(a->query, 16) || !aligned(a->key_pages, 16) || !aligned(a->value_pages, 16) || !aligned(a->out, es) ||
        !aligned(a->page_table, 4) || !aligned(a->positions, 8) || (a->mask && !aligned(a->mask, mask_size)))
        return Q3T_EINVAL;
    if (!a->workspace || a->workspace_bytes < z.workspace) return Q3T_EWORKSPACE;
    Params p = {};
    p.a = *a;
    if (s) p.s = *s;
    p.shared = shared_pages;
    hipLaunchKernelGGL(simple_kernel, dim3((uint32_t)(a->batch * a->q_heads)), dim3(64 * kWaves), 0, (hipStream_t)stream, p);
    return launch_status();
}
