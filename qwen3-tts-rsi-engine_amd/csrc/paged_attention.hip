// Attention of one new token per request over a cache kept in pages (the paged counterpart of the
// decode attention; reference: packed_attention.py:75-84).
//
//   s_j = scale q . k_j (+ mask_j),  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// in one pass over the keys, with a running maximum m that moves when it is passed by more than a
// threshold.  Every key and value row is read once for 16 query heads of its KV head, so HBM bounds a launch of
// many keys (2 to 16 operations per byte), and the chain arguments - positions - page numbers - rows - merge one of few.
// us per launch in a graph, rows not in the caches (TB/s of them): 128 requests of 100..4095 keys, 8 KV heads of
// 128, bf16 175 (6.0, the rate of a large read); 64 of 64..1023 30.7 (4.9); one of 65000, 4 heads, fp16 32.7 (4.1);
// 32 of 30..2047 under a mask, 4 heads 22.3 (3.3); 21 of 1..700 in float32 under a mask, 12 heads of 64 18.0
// (3.1); one of 300 7.6.  The first rows are there after 5.8 us.
// float32 rows of 128: 64 of 64..1023 54.0 (5.5), 128 of 100..2000 192 (5.9), one of 30000 49.3 (5.0), one of 300
// 11.6.  Pages that hold no whole stages: 128 of 100..2000 in bf16 in pages of 16 / 24 / 100 96.0 / 101 / 98.7.
// Each further block of 16 query heads of a KV head reads that head's rows again, from memory: 64 requests of 2000
// keys, 2 KV heads of 128 in bf16, with 16 / 20 / 32 / 48 query heads each 30.3 / 47.4 / 46.8 / 67.6 us (135 / 263 / 264 /
// 381 MB fetched); 8 requests of 4000 18.2 / 19.1 / 19.6 / 25.9.
//   * Work: a workgroup takes an equal share of the stages of all (request, KV head) pairs
//     (paged_index.hpp), whatever the requests' lengths; its waves find their place by adding up all
//     requests' stages.  A pair that lies in several shares leaves its parts' states in the
//     workspace, and the workgroup that arrives last merges them, in the parts' order.
//     Where no pair can have more than one share a workgroup takes the pair of its own number, and its page
//     numbers are on their way together with the position.
//   * Of a run of a pair's stages of 16 (rows of 128 bytes: 32) keys each of the workgroup's W waves takes
//     every W-th.  A stage's rows go straight from memory to the wave's own two LDS slots, one stage
//     ahead of the one that is scored, over the ends of runs: no barrier but where a run ends.  The
//     page numbers of up to 64 stages come the same way, while the stages before them are read.
//     Where pages hold whole stages the rows are one range of memory; for other page sizes each lane works out
//     the address of its own row.  In pages of halves of a stage of 32 (16 rows of 128 bytes each) they are two
//     ranges where a pair has a workgroup to itself, and single rows elsewhere, where ranges gain nothing (us, rows /
//     ranges, 64 columns in fp16, pages of 16: 128 requests of 100..4000 keys 89.7 / 90.2, 64 of 64..2047 32.8 / 33.0, 200 of
//     10..400 25.8 / 26.1).
//   * The rows of a KV head's query heads are the columns of 16x16 products, S^T = K . Q^T and
//     O^T += V^T . P^T.  The matrix cores idle (under a twentieth of their rate), so the weights are
//     not rounded to the cache's type: bf16 weights go in three parts (all 24 bits of their
//     float32), fp16 ones in two (22 bits), float32 is multiplied as such.  The first part has
//     accumulators of its own: an infinite value times a remainder of zero would be NaN.
//   * A key that does not exist (past the request's end, under a mask's minus infinity, on no page)
//     scores minus infinity, and its value row is zeroed in LDS: zero times NaN would be NaN.
#include "paged_kernel.hpp"

namespace q3t {
namespace paged {

// f on the Launch of a call's type and width
constexpr auto with = [](const q3t_paged_args *a, auto f) {
    const bool wide = a->head_dim == 128;
    if (a->dtype == Q3T_F32) return wide ? f(Launch<float, 128>{}) : f(Launch<float, 64>{});
    if (a->dtype == Q3T_BF16) return wide ? f(Launch<__bf16, 128>{}) : f(Launch<__bf16, 64>{});
    return wide ? f(Launch<_Float16, 128>{}) : f(Launch<_Float16, 64>{});
};

}  // namespace paged
}  // namespace q3t

using namespace q3t;

extern "C" int64_t q3t_paged_workspace_bytes(const q3t_paged_args *a) {
    paged::Sizes z;
    return paged::sizes_of(a, z, paged::with) == Q3T_OK ? z.workspace : -1;
}

extern "C" int q3t_paged_attention(const q3t_paged_args *a, void *stream) {
    using namespace paged;
    Sizes z;
    int status = sizes_of(a, z, with);
    if (status != Q3T_OK || a->batch == 0) return status;
    Params p = {};
    status = fill(a, z, a->dtype == Q3T_F32 ? 4 : 2, p, with);
    if (status != Q3T_OK) return status;
    with(a, [&](auto l) { l.run(a, z.pairs, p, (uint32_t)z.workgroups, (hipStream_t)stream); });
    return launch_status();
}
