// Attention of one new token per request over a paged cache of 8-bit rows, or over one whose first pages are
// shared by all requests of the batch.
//
//   s_j = scale ks_j (q . k_j) (+ mask_j),  out = sum_j exp(s_j - m) vs_j v_j / sum_j exp(s_j - m)
//
// 8-bit rows run through the kernel of the rows of 16 bits (paged_kernel.hpp): half the bytes, so its start and its matrix and
// vector instructions weigh twice as much, and HBM bounds long launches alone.  A stage has 32 keys; rows and scales go straight
// to LDS, elements are widened to bf16 (exact) on the way into the products, and a key's scale multiplies its score and
// a value's its weight, outside of them.  us per launch in a graph (TB/s of rows and scales; the same in bf16): 128 requests of
// 100..4095 keys, 8 KV heads of 128, 32 query heads, int8 95 (5.7; 175), 64 of 64..1023 in e4m3 23.0 (3.4; 30.7), 21 of 1..700
// with float32 queries under a mask, 12 heads of 64, e4m3 12.2 (1.2; float32 rows 18.0), one of 300 8.1 (7.6).
//
// A shared prefix is read once for the batch, by a launch ahead of that for the requests' own keys (paged_prefix.hpp): 128 requests
// behind 16384 keys, 32 query heads, 103 us (64 for the prefix) where requests that each read it take 960, 64 behind 4096 58.6 (18.6)
// and 154.
#include "paged_with.hpp"

namespace q3t {
namespace paged {

// Whether the prefix is attended once for all: a launch of its own (9 us, and 1.1 for each set of stages that a workgroup has),
// whose states every pair's end reads (16 ns a pair, 1.2 us for each time that a thread has four on their way), against the
// time that reading the prefix again takes, at 5.5 TB/s.  us with / without it, requests x prefix, 8 KV heads of 128 and two
// query heads each in bf16: 2 x 16384 28.6 / 29.4, 4 x 4096 19.3 / 19.9, 8 x 512 15.4 / 11.8, 8 x 2048 17.7 / 18.2, 8 x 4096
// 19.6 / 24.0, 32 x 512 18.5 / 12.4, 32 x 1024 19.4 / 26.1, 64 x 256 23.8 / 16.3, 64 x 512 24.6 / 30.4, 64 x 4096 57.8 / 153, 128
// x 256 38.9 / 36.0; one KV head of 16 query heads: 32 x 4096 30.0 / 19.2, 100 x 4096 32.5 / 35.5.
static bool once_for_all(const q3t_paged_args *a, int64_t shared_pages) {
    if (shared_pages == 0 || a->reserved == Q3T_SHARE_NEVER) return false;
    if (a->reserved == Q3T_SHARE_ALWAYS) return true;
    const int64_t size = a->dtype == Q3T_F32 ? 4 : 2, group = a->q_heads / a->kv_heads, keys = shared_pages * a->page_size;
    const int64_t blocks = (group + kColumns - 1) / kColumns, columns = group < kColumns ? group : kColumns;
    const PrefixPlan plan = size == 4 ? prefix_plan<float>(a, keys) : prefix_plan<__bf16>(a, keys);
    const double again = 2.0 * (double)(a->head_dim * size * a->kv_heads) * (double)(a->batch * blocks - 1) * (double)keys / 5.5e6;
    const double rounds = (double)((plan.parts * columns * a->head_dim / 4 + 2047) / 2048);
    return again > 9.0 + 1.1 * (double)(plan.chunk / plan.step) + 0.016 * (double)(a->batch * a->kv_heads * blocks) + 1.2 * rounds;
}

// Bytes of workspace, or the status to return.
static int64_t bytes_with(const q3t_paged_args *a, const q3t_paged_scales *s, int64_t shared_pages) {
    if (!a) return Q3T_EINVAL;
    if (s && s->format != Q3T_I8 && s->format != Q3T_E4M3) return Q3T_EUNSUPPORTED;
    if (a->reserved < Q3T_SHARE_AUTO || a->reserved > Q3T_SHARE_NEVER) return Q3T_EINVAL;
    Sizes z;
    const int status = s && s->format == Q3T_I8 ? sizes_int8(a, z) : sizes_e4m3(a, z);
    if (status != Q3T_OK) return status;
    if (shared_pages < 0 || shared_pages > a->table_width || shared_pages * a->page_size >= a->ctx) return Q3T_EINVAL;
    if (s || a->batch == 0) return z.workspace;
    if (!once_for_all(a, shared_pages)) return q3t_paged_workspace_bytes(a);
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
    if (!once_for_all(a, shared_pages)) return q3t_paged_attention(a, stream);
    const int64_t keys = shared_pages * a->page_size;
    return (a->dtype == Q3T_BF16 ? attend_shared_bf16 : a->dtype == Q3T_F16 ? attend_shared_f16 : attend_shared_f32)(a, keys, (hipStream_t)stream);
}
