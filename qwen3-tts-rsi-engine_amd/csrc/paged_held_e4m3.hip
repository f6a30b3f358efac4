// The attention over pages of e4m3 rows (paged_attention_with.hip).
#include "paged_with.hpp"

namespace q3t {
namespace paged {

// f on the Launch of a call's type and width
constexpr auto with = [](const q3t_paged_args *a, auto f) {
    const bool wide = a->head_dim == 128;
    if (a->dtype == Q3T_F32) return wide ? f(Launch<Held<float, true>, 128>{}) : f(Launch<Held<float, true>, 64>{});
    if (a->dtype == Q3T_BF16) return wide ? f(Launch<Held<__bf16, true>, 128>{}) : f(Launch<Held<__bf16, true>, 64>{});
    return wide ? f(Launch<Held<_Float16, true>, 128>{}) : f(Launch<Held<_Float16, true>, 64>{});
};

int sizes_e4m3(const q3t_paged_args *a, Sizes &z) { return sizes_of(a, z, with); }
int attend_e4m3(const q3t_paged_args *a, const Sizes &z, const q3t_paged_scales *s, hipStream_t stream) {
    return attend_with(a, z, s, stream, with);
}

}  // namespace paged
}  // namespace q3t
