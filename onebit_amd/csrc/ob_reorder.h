// States of hypotheses brought to the slots that go on with them, in place, gfx950: slot (g, b) takes what slot (g, parents[g][b]) held.
// A thread owns one unit of 16 (4, 1) bytes at the same place of all slots of a group: it loads every unit that a slot takes from another one, then
// stores them.  No other thread touches that place, so any map is right in place (permutations, one slot to many), and slots that keep their state move
// nothing.  Bound by HBM: each moved byte is read (a source that several slots take comes from the L1 after its first load) and written once:
// 403 MB of 64 caches, 4 or 8 beams, 82 us, 4.9 TB/s; 32 beams, 805 MB, 168 us.
#pragma once
#include "ob_common.h"

#define OB_RE_THREADS 256
#define OB_RE_BUFFERS 128                          // buffers of one launch (their addresses travel in the kernel arguments)
#define OB_RE_MAX_BEAMS 32

struct ObReArgs {
    const int *parents;              // device [groups][beams]
    long long slot_bytes, outer_bytes, first_byte;
    long long units;                 // of a slot: outer * units_per
    int units_per, beams;            // units_per: of a slot's one outer row
    char *buf[OB_RE_BUFFERS];
};

template <int W, typename U>
__global__ __launch_bounds__(OB_RE_THREADS) void ob_re_kernel(const ObReArgs A)
{
    const int group = blockIdx.y;
    const int *par = A.parents + (int64_t)group * A.beams;
    int src[W];
    bool any = false;
#pragma unroll
    for (int b = 0; b < W; ++b) {
        const int p = b < A.beams ? par[b] : b;
        src[b] = p >= 0 && p < A.beams ? p : b;                                  // (a parent outside the group: the slot stays as it is)
        any = any || src[b] != b;
    }
    if (!any) return;
    const int64_t u = (int64_t)blockIdx.x * OB_RE_THREADS + threadIdx.x;
    if (u >= A.units) return;
    const int64_t row = u / A.units_per;
    char *p = A.buf[blockIdx.z] + (int64_t)group * A.beams * A.slot_bytes + row * A.outer_bytes + A.first_byte + (u - row * A.units_per) * sizeof(U);
    U v[W];
#pragma unroll
    for (int b = 0; b < W; ++b)
        if (src[b] != b) v[b] = *reinterpret_cast<const U *>(p + src[b] * A.slot_bytes);
#pragma unroll
    for (int b = 0; b < W; ++b)
        if (src[b] != b) *reinterpret_cast<U *>(p + b * A.slot_bytes) = v[b];
}
