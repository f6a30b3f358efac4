// Attention over pools of 8 bits, and behind a prefix that the batch shares: what paged_attention_with.hip asks of the
// sources that hold the kernels' instances.
#pragma once

#include "paged_kernel.hpp"

namespace q3t {
namespace paged {

// The keys behind a prefix: `args` are those of the keys behind it alone, with positions still counted from its start.
struct Behind {
    int64_t skip;                      // keys of the prefix
    uint32_t parts;                    // states of each query head over it, 0: none
    const float *prefix, *prefix_ml;
};

int sizes_int8(const q3t_paged_args *args, Sizes &sizes);
int sizes_e4m3(const q3t_paged_args *args, Sizes &sizes);
int attend_int8(const q3t_paged_args *args, const Sizes &sizes, const q3t_paged_scales *scales, const Behind &behind, hipStream_t stream);
int attend_e4m3(const q3t_paged_args *args, const Sizes &sizes, const q3t_paged_scales *scales, const Behind &behind, hipStream_t stream);

template <typename With>
static int attend_with(const q3t_paged_args *a, const Sizes &z, const q3t_paged_scales *s, const Behind &behind, hipStream_t stream, With with) {
    MoreParams p = {};
    const int status = fill(a, z, s ? 1 : a->dtype == Q3T_F32 ? 4 : 2, p, with);
    if (status != Q3T_OK) return status;
    if (s) {
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
    }
    p.skip = (uint32_t)behind.skip;
    p.parts = behind.parts;
    p.columns_all = (uint32_t)(a->batch * z.group);
    p.prefix = behind.prefix;
    p.prefix_ml = behind.prefix_ml;
    with(a, [&](auto l) { l.run(a, z.pairs, p, (uint32_t)z.workgroups, stream); });
    return launch_status();
}

}  // namespace paged
}  // namespace q3t
