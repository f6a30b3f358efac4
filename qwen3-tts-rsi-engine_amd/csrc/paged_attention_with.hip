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
// with float32 queries under a mask, 12 heads of 64, e4m3 12.1 (1.2; float32 rows 18.0), one of 300 8.1 (7.6).  With
// fp16 queries the first two take 98 and 25.9, under a bool mask 94 and 25.9.
//
// A shared prefix is read once for the batch, by a launch ahead of that for the requests' own keys (paged_prefix.hpp): 128 requests
// behind 16384 keys, 32 query heads, 102 us (64 for the prefix) where requests that each read it take 960, 64 behind 4096 58.1 (18.6)
// and 154; under a bool mask 214 and 73, where the prefix' launch waits for each stage's terms.
#include "paged_with.hpp"

namespace q3t {
namespace paged {

// Whether the prefix is attended once for all: what its launch adds, against what reading the prefix again for every request takes.
// The costs, in us, are those of a line through 478 pairs of times, of requests x prefix, heads, types, masks and pages of all kinds:
// the choice is the quicker one or within 3% of it for all but 13 of them (0.35% off on average, 42% at worst, for 4720 columns under a
// mask).  us once / for each, 8 KV heads of 128 and two query heads each in bf16 unless said: 2 x 16384 28.7 / 29.5, 8 x 512
// 16.9 / 12.1, 8 x 4096 19.7 / 24.5, 64 x 512 28.8 / 31.1, 64 x 4096 32.3 / 108, float32 70.5 / 260, 64 x 512 under a mask 47.2 / 33.2;
// one KV head of 16 query heads: 100 x 4096 35.7 / 34.3, float32 102 / 71; 40 query heads on 2: 16 x 4096 33.3 / 27.0, float32 99 / 49.
static bool once_for_all(const q3t_paged_args *a, int64_t shared_pages) {
    if (shared_pages == 0 || a->reserved == Q3T_SHARE_NEVER) return false;
    if (a->reserved == Q3T_SHARE_ALWAYS) return true;
    const bool f32 = a->dtype == Q3T_F32;
    const int64_t group = a->q_heads / a->kv_heads, keys = shared_pages * a->page_size, blocks = (group + kColumns - 1) / kColumns;
    const PrefixPlan plan = f32 ? prefix_plan<float>(a, keys) : prefix_plan<__bf16>(a, keys);
    const double width = (double)a->head_dim, pairs = (double)(a->batch * a->kv_heads * blocks);
    // read again: 8.4 TB/s, out of the caches where it fits them
    const double again = 2.0 * width * (f32 ? 4 : 2) * (pairs - (double)a->kv_heads) * (double)keys / 8.4e6;
    // a set of stages: its start, the products (two a weight in 16 bits) at a CU's rate, the mask's terms
    const double products = (f32 ? 4 : 6) * width * (double)(plan.cw * plan.ct * kColumns * plan.step) / (f32 ? 0.6e6 : 9.8e6);
    const double set = 0.37 + 1.2 * products + (a->mask ? (f32 ? 0.72 : 1.15) * (double)plan.ct : 0.0);
    const double sets = (double)((plan.workgroups + 255) / 256 * (plan.chunk / plan.step));
    // a launch; the pairs' ends; the states, written and read
    return again > 5.0 + sets * set + 0.0061 * pairs + (double)(plan.states * (a->head_dim + 2) * 4) / 0.7e6;
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
