// Attention over pools of 8 bits, and behind a prefix that the batch shares: what paged_attention_with.hip asks of the
// sources that hold the kernels' instances.
#pragma once

#include "paged_prefix.hpp"

namespace q3t {
namespace paged {

int sizes_int8(const q3t_paged_args *args, Sizes &sizes);
int sizes_e4m3(const q3t_paged_args *args, Sizes &sizes);
int attend_int8(const q3t_paged_args *args, const Sizes &sizes, const q3t_paged_scales *scales, hipStream_t stream);
int attend_e4m3(const q3t_paged_args *args, const Sizes &sizes, const q3t_paged_scales *scales, hipStream_t stream);

// A call behind `keys` shared keys, for each type of pools: bytes of workspace, or the status; the launches.
int64_t bytes_shared_bf16(const q3t_paged_args *args, int64_t keys);
int64_t bytes_shared_f16(const q3t_paged_args *args, int64_t keys);
int64_t bytes_shared_f32(const q3t_paged_args *args, int64_t keys);
int attend_shared_bf16(const q3t_paged_args *args, int64_t keys, hipStream_t stream);
int attend_shared_f16(const q3t_paged_args *args, int64_t keys, hipStream_t stream);
int attend_shared_f32(const q3t_paged_args *args, int64_t keys, hipStream_t stream);

template <typename With>
static int attend_with(const q3t_paged_args *a, const Sizes &z, const q3t_paged_scales *s, hipStream_t stream, With with) {
    MoreParams p = {};
    const int status = fill(a, z, 1, p, with);
    if (status != Q3T_OK) return status;
    if (!s->key_scales || !s->value_scales || !aligned(s->key_scales, 4) || !aligned(s->value_scales, 4)) return Q3T_EINVAL;
    const int64_t strides[6] = {s->ks_stride_p, s->ks_stride_h, s->ks_stride_t, s->vs_stride_p, s->vs_stride_h, s->vs_stride_t};
    uint32_t *const to[6] = {&p.ks_sp, &p.ks_sh, &p.ks_st, &p.vs_sp, &p.vs_sh, &p.vs_st};
    for (int i = 0; i < 6; ++i) {
        if (strides[i] < 0) return Q3T_EINVAL;
        if (strides[i] > UINT32_MAX) return Q3T_EUNSUPPORTED;
        *to[i] = (uint32_t)strides[i];
    }
    p.ks = s->key_scales;
    p.vs = s->value_scales;
    with(a, [&](auto l) { l.run(a, z.pairs, p, (uint32_t)z.workgroups, stream); });
    return launch_status();
}

// The call's part behind its first `keys` keys.
static q3t_paged_args behind(const q3t_paged_args *a, int64_t keys) {
    q3t_paged_args b = *a;
    b.ctx -= keys;
    b.table_width -= keys / a->page_size;
    if (a->page_table) b.page_table += keys / a->page_size;
    const int64_t mask_size = a->mask_dtype == Q3T_F32 ? 4 : a->mask_dtype == Q3T_BOOL ? 1 : 2;
    if (a->mask) b.mask = (const char *)a->mask + keys * a->mask_stride_t * mask_size;
    return b;
}

// The two launches of a call, `with` of the type T.
template <typename T, typename With>
static int64_t shared_bytes(const q3t_paged_args *a, int64_t keys, With with) {
    const q3t_paged_args b = behind(a, keys);
    Sizes z;
    int status = sizes_of(a, z, with);  // of all keys too: the requests may have to attend the prefix each for itself
    if (status == Q3T_OK) status = sizes_of(&b, z, with);
    return status != Q3T_OK ? status : (z.workspace + 15) / 16 * 16 + prefix_plan<T>(&b, keys).bytes;
}

template <typename T, typename With>
static int shared_attend(const q3t_paged_args *a, int64_t keys, hipStream_t stream, With with) {
    const q3t_paged_args b = behind(a, keys);
    Sizes z;
    MoreParams p = {};
    int status = sizes_of(&b, z, with);
    if (status == Q3T_OK) status = fill(&b, z, (int64_t)sizeof(T), p, with);
    if (status != Q3T_OK) return status;
    const PrefixPlan plan = prefix_plan<T>(&b, keys);
    const int64_t own = (z.workspace + 15) / 16 * 16;
    if (a->workspace_bytes < own + plan.bytes) return Q3T_EWORKSPACE;
    float *states = (float *)((char *)a->workspace + own);
    status = prefix_run<T>(&b, plan, keys, p, a->page_table, a->mask, states, stream);
    if (status != Q3T_OK) return status;
    p.skip = (uint32_t)keys;
    p.parts = (uint32_t)plan.parts;
    p.columns_all = (uint32_t)plan.columns;
    p.prefix = states;
    p.prefix_ml = states + plan.states * a->head_dim;
    p.odd = (const uint32_t *)(p.prefix_ml + 2 * plan.states);
    p.odds = (uint32_t)plan.workgroups;
    p.skip_pages = (uint32_t)(keys / a->page_size);
    with(&b, [&](auto l) { l.run(&b, z.pairs, p, (uint32_t)z.workgroups, stream); });
    return launch_status();
}

}  // namespace paged
}  // namespace q3t
