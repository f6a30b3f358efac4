// Index arithmetic of the paged cache, the same on the host and in the kernels (it includes no HIP
// header, so a host compiler alone can check it).
#pragma once

#include <stdint.h>

#if defined(__HIP__) || defined(__HIPCC__)
#define Q3T_BOTH __host__ __device__ inline __attribute__((always_inline))
#else
#define Q3T_BOTH inline
#endif

namespace q3t {

// Division of 0 <= n < 2^31 by a divisor in [1, 2^31) as a multiplication, an addition and a
// shift (Granlund and Montgomery, Division by Invariant Integers using Multiplication, 1994): with
// 2^(l-1) < d <= 2^l and m = floor(2^32 (2^l - d) / d) + 1, floor(n / d) is
// (floor(m n / 2^32) + n) >> l (the sum stays below 2^32 since floor(m n / 2^32) <= n < 2^31).
struct Divisor {
    uint32_t d, m, l;
};
inline Divisor divisor(uint32_t d) {
    uint32_t l = 0;
    while (((uint64_t)1 << l) < d) ++l;
    return {d, (uint32_t)(((((uint64_t)1 << l) - d) << 32) / d + 1), l};
}
Q3T_BOTH uint32_t divide(uint32_t n, const Divisor &v) {
    return ((uint32_t)(((uint64_t)v.m * n) >> 32) + n) >> v.l;
}

// ---- how the paged attention's work is shared out ------------------------------------------
//
// A pair is a request with one KV head (and up to 16 of its query heads).  A pair's keys are read
// in stages of a fixed number of keys, at least one.  All pairs lie on one line, request by request,
// head by head, each with a place for every stage and some empty ones behind them, and workgroup w
// takes the share [w * share, (w + 1) * share) of it.  A pair whose stages lie in several shares
// is merged from its parts.
//   * When every pair cut into pieces of `least` stages gives no more pieces than there are
//     workgroups, each piece is a share of its own: a pair takes a multiple of that many places.
//   * Otherwise a pair takes `cost` places more than it has stages, for what ends a run (the waves'
//     merge, the output), and the shares are equal.

struct Sharing {
    uint32_t unit, cost;  // places of a pair: a multiple of unit (a power of two), and cost more
    uint32_t share;       // places of a workgroup
    uint32_t total;       // places in all
};

// From the number of pairs, their stages (fewer than 2^30 together), and their pieces of `least`
// stages, a power of two.
Q3T_BOTH Sharing sharing(uint32_t pairs, uint32_t stages, uint32_t pieces, uint32_t least, uint32_t cost, const Divisor &workgroups) {
    if (pieces <= workgroups.d) return {least, 0u, least, pieces * least};
    const uint32_t total = stages + cost * pairs;
    return {1u, cost, divide(total + workgroups.d - 1, workgroups), total};
}

Q3T_BOTH uint32_t places(uint32_t stages, const Sharing &s) {
    return ((stages + s.unit - 1) & ~(s.unit - 1)) + s.cost;
}

// Where a workgroup is on the line: place x, `left` places to go, at place `off` of pair (b, head).
struct Cursor {
    uint32_t x, left, b, head, off;
};

// Past the pair's last stage: on to the next pair.
Q3T_BOTH void end_pair(Cursor &c, uint32_t length, uint32_t heads) {
    const uint32_t rest = length - c.off;
    c.x += rest;
    c.left -= rest < c.left ? rest : c.left;
    c.off = 0;
    if (++c.head == heads) {
        c.head = 0;
        ++c.b;
    }
}

// A run of one pair's stages [lo, hi) in one share: part (its workgroup - first) of the pair's `parts`
// (first only if there are several).  Its state's slot is 2 w for a pair that began in an earlier share
// (a workgroup's first run at most), 2 w + 1 for one that begins in this one (the last at most, if
// there are more parts).
struct Run {
    uint32_t b, head, lo, hi, first, parts, begins;
};

// The run at the cursor, for a pair of `stages` stages, and the cursor moved past it.
Q3T_BOTH Run next_run(Cursor &c, uint32_t stages, uint32_t heads, const Sharing &s) {
    const uint32_t rest = stages - c.off, take = rest < c.left ? rest : c.left;
    Run r;
    r.b = c.b;
    r.head = c.head;
    r.lo = c.off;
    r.hi = c.off + take;
    r.begins = c.off == 0;
    r.first = 0;
    r.parts = 1;
    if (c.off || take < rest) {  // (no division for a pair that lies in one share)
        const uint32_t start = c.x - c.off;
        r.first = start / s.share;
        r.parts = (start + stages - 1) / s.share - r.first + 1;
    }
    c.x += take;
    c.left -= take;
    c.off = r.hi;
    if (r.hi == stages) end_pair(c, places(stages, s), heads);
    return r;
}

// The share of a workgroup that has one pair to itself, in one run: of any number of stages below 2^30.
constexpr uint32_t kWholePair = 1u << 30;
Q3T_BOTH Sharing whole_pair() { return {kWholePair, 0u, kWholePair, kWholePair}; }
Q3T_BOTH Cursor whole_pair_at(uint32_t b, uint32_t head) { return {0u, kWholePair, b, head, 0u}; }

}  // namespace q3t
