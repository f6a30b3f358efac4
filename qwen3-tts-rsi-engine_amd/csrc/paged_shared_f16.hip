// The attention of requests that share their first pages, for pools of f16 (paged_attention_with.hip).
#include "paged_with.hpp"

namespace q3t {
namespace paged {

// f on the Launch of a call's width
constexpr auto with = [](const q3t_paged_args *a, auto f) { return a->head_dim == 128 ? f(Launch<_Float16, 128>{}) : f(Launch<_Float16, 64>{}); };

int64_t bytes_shared_f16(const q3t_paged_args *a, int64_t keys) { return shared_bytes<_Float16>(a, keys, with); }
int attend_shared_f16(const q3t_paged_args *a, int64_t keys, hipStream_t stream) { return shared_attend<_Float16>(a, keys, stream, with); }

}  // namespace paged
}  // namespace q3t
