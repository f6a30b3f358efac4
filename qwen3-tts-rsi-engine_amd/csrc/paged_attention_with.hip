// Attention of one new token per request over a paged cache of 8-bit rows, or over one whose first pages are
// shared by all requests of the batch.
//
//   s_j = scale ks_j (q . k_j) (+ mask_j),  out = sum_j exp(s_j - m) vs_j v_j / sum_j exp(s_j - m)
#include "paged_with.hpp"

namespace q3t {
namespace paged {

// Bytes of workspace, or the status to return.
static int64_t bytes_with(const q3t_paged_args *a, const q3t_paged_scales *s, int64_t shared_pages) {
    if (!a) return Q3T_EINVAL;
    if (s && s->format != Q3T_I8 && s->format != Q3T_E4M3) return Q3T_EUNSUPPORTED;
    Sizes z;
    const int status = s && s->format == Q3T_I8 ? sizes_int8(a, z) : sizes_e4m3(a, z);
    if (status != Q3T_OK) return status;
    if (shared_pages < 0 || shared_pages > a->table_width || shared_pages * a->page_size >= a->ctx) return Q3T_EINVAL;
    if (s) return z.workspace;
    if (shared_pages == 0) return q3t_paged_workspace_bytes(a);
    const int64_t keys = shared_pages * a->page_size;
    return a->dtype == Q3T_BF16 ? bytes_shared_bf16(a, keys) : a->dtype == Q3T_F16 ? bytes_shared_f16(a, keys) : bytes_shared_f32(a, keys);
}

}  // namespace paged
}  // namespace q3t

using namespace q3t;

extern "C" int64_t q3t_paged_workspace_bytes_with(const q3t_paged_args *a, const q3t_paged_scales *s, int64_t shared_pages) {
    const int64_t bytes = paged::bytes_with(a, s, shared_pages);
    return bytes < 0 ? -1 : bytes;
}

extern "C" int q3t_paged_attention_with(const q3t_paged_args *a, const q3t_paged_scales *s, int64_t shared_pages, void *stream) {
    using namespace paged;
    const int64_t bytes = bytes_with(a, s, shared_pages);
    if (bytes < 0) return (int)bytes;
    if (a->batch == 0) return Q3T_OK;
    if (s) {
        Sizes z;
        const int status = s->format == Q3T_I8 ? sizes_int8(a, z) : sizes_e4m3(a, z);
        if (status != Q3T_OK) return status;
        return (s->format == Q3T_I8 ? attend_int8 : attend_e4m3)(a, z, s, (hipStream_t)stream);
    }
    if (shared_pages == 0) return q3t_paged_attention(a, stream);
    const int64_t keys = shared_pages * a->page_size;
    return (a->dtype == Q3T_BF16 ? attend_shared_bf16 : a->dtype == Q3T_F16 ? attend_shared_f16 : attend_shared_f32)(a, keys, (hipStream_t)stream);
}
