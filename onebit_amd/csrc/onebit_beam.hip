// libonebit_hip.so, beam search's operators:
//   onebit_attention_shared_rows   attention of single-token rows over a shared prefix and their own cache slots (ob_shattn.h)
//   onebit_beam_select             the best continuations over beams and vocabulary (ob_beamsel.h)
//   onebit_reorder_slots           surviving hypotheses' states brought to their slots, in place (ob_reorder.h)
#include <hip/hip_runtime.h>
#include <algorithm>
#include <math.h>

#include "../../include/onebit.h"
#include "ob_host.h"
#include "ob_shattn.h"
#include "ob_beamsel.h"
#include "ob_reorder.h"

static inline int64_t ob_up(int64_t n, int64_t m) { return (n + m - 1) / m; }
static const int64_t OB_MAX_WGS = 0xffffff;            // workgroups of 256 threads of one launch
static const int64_t OB_SH_MAX_LEN = 1 << 30;         // (positions and their chunks are counted in 32 bits)

// memory of a call (sizes of products that may pass 64 bits)
struct ObMem { const void *p; unsigned __int128 n; };
static inline bool ob_overlap(const ObMem &a, const ObMem &b)
{
    const unsigned __int128 x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    return a.p && b.p && a.n && b.n && x < y + b.n && y < x + a.n;
}

// ------------------------------------------------------------------------------------------- attention over a shared prefix --
// form: ob_sh_one_kernel; ob_sh_wide_kernel of 64 / 128 queries and ob_sh_own_kernel; the latter alone.  osplits 0: a row's own keys are one chunk, no part
enum { OB_SH_INLINE, OB_SH_ONE, OB_SH_WIDE64, OB_SH_WIDE128 };
struct ObShPlan { int form, per, pchunk, ochunk, psplits, osplits, own_mb; bool among, alone; };
#define OB_SH_TICKETS 16384                           // their place in front of the scratch memory does not depend on a call's sizes

static ObShPlan ob_sh_plan(const onebit_prefix_t *groups, int32_t n_groups, int64_t rows, int32_t n_heads, int32_t n_kv_heads, int64_t max_own)
{
    ObShPlan p = {};
    const int64_t rep = n_heads / n_kv_heads;
    int64_t most = 1, longest = 0, again = 0;
    for (int i = 0; i < n_groups; ++i) {
        if (groups[i].len > 0) most = std::max<int64_t>(most, groups[i].n * rep);
        longest = std::max<int64_t>(longest, groups[i].len);
        again += (int64_t)groups[i].n * groups[i].len;
    }
    // (us of kernels at D = 128, rows x heads / kv heads; the other side in brackets)
    p.own_mb = (int)ob_up(rep, 16);
    const int64_t own = rows * n_kv_heads * p.own_mb;                    // workgroups of one chunk per row
    p.ochunk = (int)(128 * std::max<int64_t>(1, ob_up(max_own, 128)));
    // a row's own keys in chunks where the rows are few: 8 x 8 / 8 with 1000 own keys each 10.8 (in one chunk 17.3), 16 x 8 / 8 with 600 12.4 (14.2), 30 x 8 / 8 18.7 (18.7)
    if (own < 256 && max_own > 512) p.ochunk = (int)(128 * std::max<int64_t>(2, ob_up(own * max_own, 512 * 128)));
    p.osplits = (int)ob_up(max_own, p.ochunk);
    // one launch that reads short prefixes once a row: 4 x 8 / 8 sharing 96 5.8 (ob_sh_one_kernel 7.2), 8 x 32 / 32 sharing 256 8.4 (8.8), 64 x 64 / 8 sharing 200 11.0
    // (16.1); behind the bound 8 x 32 / 32 sharing 500 11.0 (9.6), 32 x 32 / 32 sharing 256 19.4 (16.6), 64 x 32 / 32 sharing 128 26.4 (wide 22.5)
    if (p.osplits <= 1 && longest <= 256 && again * n_kv_heads * p.own_mb <= 128 * 1024) {
        p.form = OB_SH_INLINE;
        p.osplits = 0;
        return p;
    }
    const auto tiles = [&](int per) {                                    // keys of all workgroups of `per` queries together
        int64_t n = 0;
        for (int i = 0; i < n_groups; ++i) n += ob_up(groups[i].n * rep, per) * groups[i].len * n_kv_heads;
        return n;
    };
    // up to 32 queries of a group and kv head in blocks of 16, one launch: 17 x 32 / 32 sharing 1000 15.0 (blocks of 64 16.7), 32 x 32 / 32 sharing 4000 27.8 (31.0), 4 rows x
    // 8 groups x 40 / 40 of 2000 82 (91); more: 64 x 32 / 32 sharing 8000 56.8 (48.8), 48 x 32 / 8 sharing 2000 23.6 (17.7).
    // Blocks of 128 where 512 workgroups of them have 512 keys and more: 64 x 64 / 8 sharing 32768 95 (of 64 108), sharing 8000 41 (39), 48 x 32 / 8 sharing 2000 19.8 (17.4)
    p.form = most <= 32 && rows * n_kv_heads <= OB_SH_TICKETS ? OB_SH_ONE : most > 64 && tiles(128) >= 512 * 512 ? OB_SH_WIDE128 : OB_SH_WIDE64;
    p.per = p.form == OB_SH_ONE ? 16 : p.form == OB_SH_WIDE64 ? 64 : 128;
    // own keys' workgroups among the prefix's and a launch that joins: 64 x 40 / 40 sharing 2000 with 20 own 37.5 (after them, started from their parts, 44.5), 64 x 32 / 32
    // sharing 8000 49.9 (57.8); with more queries of a row per kv head, whose parts fill the lanes that fetch them, 64 x 64 / 8 sharing 2000 30.7 (23.9)
    p.among = p.form == OB_SH_WIDE64 && rep <= 2;
    // there a wave of its own for 128 of a row's own keys while those are few: 64 x 40 / 40 sharing 2000 with 20 own, not in the caches, 33 (a workgroup for a row's 43), 48 x 40 / 40
    // sharing 4000 with 100 50 (56), 64 x 32 / 32 sharing 2040 with 200 60 (64), with 300 82 (81); 64 x 40 / 40 sharing 500 with 500 135 (127)
    p.alone = p.among && max_own <= 384;
    if (p.alone) {
        p.ochunk = 128;
        p.osplits = (int)ob_up(max_own, p.ochunk);
    }
    if (p.form == OB_SH_ONE || p.among) p.osplits = std::max(p.osplits, 1);
    else if (p.osplits <= 1) p.osplits = 0;
    // chunks for 256 workgroups where a row's last one joins them (1 x 32 / 32 of 8192 26.8, for 512 29.0; 16 x 32 / 32 of 4000 23.7 and 26.4), for 512 else (64 x 64 / 8
    // sharing 32768 79 of the prefix, for 256 118), no fewer than 256 keys (32 x 32 / 8 sharing 8192 28.7, from 128 on 35.0)
    p.pchunk = (int)(128 * std::max<int64_t>(p.form == OB_SH_ONE ? 1 : 2, ob_up(tiles(p.per), (p.form == OB_SH_ONE ? 256 : 512) * 128)));
    p.psplits = (int)ob_up(longest, p.pchunk);
    return p;
}

static int ob_sh_check(const onebit_prefix_t *groups, int32_t n_groups, int64_t rows, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int64_t max_own)
{
    if (n_groups < 0 || rows < 0 || n_heads <= 0 || n_kv_heads <= 0 || max_own < 0) return ob_fail(ONEBIT_E_ARG, "attention_shared_rows: bad size");
    if (head_dim < 8 || head_dim % 8 != 0 || head_dim > 128 || n_heads % n_kv_heads != 0)
        return ob_fail(ONEBIT_E_SHAPE, "attention_shared_rows: head_dim %d (multiple of 8, <= 128), heads %d / %d", head_dim, n_heads, n_kv_heads);
    if (rows > 65535 || n_heads > 65535 || max_own > OB_SH_MAX_LEN) return ob_fail(ONEBIT_E_ARG, "attention_shared_rows: dimension too large");
    if (rows > 0 && !groups) return ob_fail(ONEBIT_E_ARG, "attention_shared_rows: null pointer");
    int64_t r = 0;
    for (int i = 0; i < n_groups && rows > 0; ++i) {
        const onebit_prefix_t &g = groups[i];
        if (g.row0 != r || g.n < 1 || g.len < 0 || g.first < 0 || g.len > OB_SH_MAX_LEN || g.first > OB_SH_MAX_LEN)
            return ob_fail(ONEBIT_E_SHAPE, "attention_shared_rows: group %d starts at row %d (expected %lld) with %d rows, a prefix of %d, own positions from %d", i,
                           g.row0, (long long)r, g.n, g.len, g.first);
        r += g.n;
    }
    if (r != rows) return ob_fail(ONEBIT_E_SHAPE, "attention_shared_rows: the groups have %lld rows of %lld", (long long)r, (long long)rows);
    return 0;
}

extern "C" size_t onebit_attention_shared_scratch_bytes(const onebit_prefix_t *groups, int32_t n_groups, int64_t rows, int32_t n_heads, int32_t n_kv_heads,
                                                        int32_t head_dim, int64_t max_own)
{
    if (rows <= 0 || ob_sh_check(groups, n_groups, rows, n_heads, n_kv_heads, head_dim, max_own)) return 0;
    const ObShPlan p = ob_sh_plan(groups, n_groups, rows, n_heads, n_kv_heads, max_own);
    return OB_SH_TICKETS * 4 + (size_t)rows * n_heads * (p.psplits + p.osplits) * (head_dim + 2) * 4;
}

template <int DP, bool EXACT>
static void ob_sh_launch(ObShArgs &a, const ObShPlan &p, int64_t prefix_items, int64_t own_items, hipStream_t s)
{
    const dim3 block(OB_SH_THREADS), own((unsigned)(own_items * a.Hkv)), all((unsigned)((prefix_items + own_items) * a.Hkv));
    if (p.form == OB_SH_ONE) {
        hipLaunchKernelGGL((ob_sh_one_kernel<DP, 1, EXACT>), all, block, 0, s, a);
        return;
    }
    a.own_alone = p.alone;
    a.own_blocks = p.among ? (int)(p.alone ? ob_up(own.x, 4) : own.x) : 0;
    const dim3 wide(all.x - own.x + a.own_blocks);
    if (wide.x > 0) {
        if (p.form == OB_SH_WIDE64) hipLaunchKernelGGL((ob_sh_wide_kernel<DP, 1, EXACT>), wide, block, 0, s, a);
        else if (p.form == OB_SH_WIDE128) hipLaunchKernelGGL((ob_sh_wide_kernel<DP, 2, EXACT>), wide, block, 0, s, a);
    }
    if (!p.among) hipLaunchKernelGGL((ob_sh_own_kernel<DP, EXACT>), own, block, 0, s, a);
    if (a.osplits) hipLaunchKernelGGL(ob_sh_join_kernel, dim3((unsigned)ob_up((int64_t)a.rows * a.H, OB_SH_THREADS / 32)), block, 0, s, a);
}

extern "C" int onebit_attention_shared_rows(const void *q, const void *prefix_k, const void *prefix_v, const void *k_cache, const void *v_cache, void *o,
                                            const void *h_next, const onebit_prefix_t *groups, int32_t n_groups, const int32_t *row_slot,
                                            const int32_t *row_pos, int64_t rows, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                                            int64_t n_prefix_slots, int64_t prefix_max_len, int64_t n_slots, int64_t max_len, int64_t max_own, void *scratch,
                                            size_t scratch_bytes, void *stream)
{
    const int rc = ob_sh_check(groups, n_groups, rows, n_heads, n_kv_heads, head_dim, max_own);
    if (rc) return rc;
    if (n_prefix_slots < 0 || prefix_max_len < 0 || n_slots <= 0 || max_len <= 0 || n_slots > 0x7fffffffLL || max_len > OB_SH_MAX_LEN)
        return ob_fail(ONEBIT_E_ARG, "attention_shared_rows: bad cache size");
    bool prefixes = false;
    for (int i = 0; i < n_groups && rows > 0; ++i) {
        const onebit_prefix_t &g = groups[i];
        prefixes = prefixes || g.len > 0;
        if (g.len > 0 && (g.slot < 0 || g.slot >= n_prefix_slots || g.len > prefix_max_len))
            return ob_fail(ONEBIT_E_SHAPE, "attention_shared_rows: group %d's prefix (slot %d, %d positions) outside %lld slots x %lld positions", i, g.slot, g.len,
                           (long long)n_prefix_slots, (long long)prefix_max_len);
    }
    if (rows == 0) return 0;
    if (!q || !k_cache || !v_cache || !o || !row_pos || (prefixes && (!prefix_k || !prefix_v))) return ob_fail(ONEBIT_E_ARG, "attention_shared_rows: null pointer");
    if (!ob_aligned(q, 16) || !ob_aligned(k_cache, 16) || !ob_aligned(v_cache, 16) || !ob_aligned(o, 8) || (h_next && !ob_aligned(h_next, 2)) ||
        (prefixes && (!ob_aligned(prefix_k, 16) || !ob_aligned(prefix_v, 16))))
        return ob_fail(ONEBIT_E_ALIGN, "attention_shared_rows: q and the caches must be 16-byte aligned");
    const size_t need = onebit_attention_shared_scratch_bytes(groups, n_groups, rows, n_heads, n_kv_heads, head_dim, max_own);
    if (!scratch || scratch_bytes < need || !ob_aligned(scratch, 16)) return ob_fail(ONEBIT_E_WSPACE, "attention_shared_rows: needs %zu bytes of zero-initialised, 16-byte aligned scratch", need);
    const auto mem = [](const void *p, int64_t n0, int64_t n1, int64_t n2, int64_t n3) { return ObMem{p, (unsigned __int128)n0 * n1 * n2 * n3}; };
    const ObMem out = mem(o, rows, n_heads, head_dim, 2), work = {scratch, need};
    const int64_t pre = prefixes ? prefix_max_len : 0;
    const ObMem in[] = {mem(q, rows, n_heads, head_dim, 2), mem(k_cache, n_slots, n_kv_heads, max_len, head_dim * 2), mem(v_cache, n_slots, n_kv_heads, max_len, head_dim * 2),
                        mem(prefix_k, n_prefix_slots, n_kv_heads, pre, head_dim * 2), mem(prefix_v, n_prefix_slots, n_kv_heads, pre, head_dim * 2), mem(h_next, n_heads, head_dim, 2, 1),
                        mem(row_slot, rows, 4, 1, 1), mem(row_pos, rows, 4, 1, 1)};
    bool overlap = ob_overlap(out, work);
    for (const ObMem &m : in) overlap = overlap || ob_overlap(out, m) || ob_overlap(work, m);
    if (overlap) return ob_fail(ONEBIT_E_ARG, "attention_shared_rows: the output and the scratch memory overlap nothing else");
    const ObShPlan p = ob_sh_plan(groups, n_groups, rows, n_heads, n_kv_heads, max_own);
    const int64_t rep = n_heads / n_kv_heads;
    ObShArgs a = {};
    a.q = (const _Float16 *)q; a.pk = (const _Float16 *)prefix_k; a.pv = (const _Float16 *)prefix_v; a.k = (const _Float16 *)k_cache; a.v = (const _Float16 *)v_cache;
    a.o = (_Float16 *)o; a.h_next = (const _Float16 *)h_next; a.row_slot = row_slot; a.row_pos = row_pos;
    a.p_max_len = prefix_max_len; a.max_len = max_len; a.H = n_heads; a.Hkv = n_kv_heads; a.rep = (int)rep; a.D = head_dim; a.n_slots = (int)n_slots;
    a.pchunk = p.pchunk; a.ochunk = p.ochunk; a.psplits = p.psplits; a.osplits = p.osplits; a.own_mb = p.own_mb; a.max_own = (int)max_own;
    a.inline_prefix = p.form == OB_SH_INLINE;
    a.scale_log2e = 1.4426950408889634f / sqrtf((float)head_dim);
    const size_t parts = (size_t)rows * n_heads * (p.psplits + p.osplits);
    a.tickets = (int *)scratch;
    a.part_o = (float *)scratch + OB_SH_TICKETS;
    a.part_ml = a.part_o + parts * head_dim;
    const auto chunks_of = [&](const onebit_prefix_t &g) { return p.form == OB_SH_INLINE ? 0 : ob_up(g.len, p.pchunk); };
    for (int g0 = 0; g0 < n_groups; g0 += OB_SH_GROUPS) {                        // (all launches are looked at before the first)
        int64_t items = 0;
        for (int i = g0; i < std::min(n_groups, g0 + OB_SH_GROUPS); ++i) {
            const int64_t chunks = chunks_of(groups[i]);
            items += (chunks ? chunks * ob_up(groups[i].n * rep, p.per) : 0) + (int64_t)groups[i].n * p.own_mb * std::max(p.osplits, 1);
        }
        if (items * n_kv_heads > OB_MAX_WGS) return ob_fail(ONEBIT_E_ARG, "attention_shared_rows: too many workgroups");
    }
    for (int g0 = 0; g0 < n_groups; g0 += OB_SH_GROUPS) {
        a.n_groups = std::min(n_groups - g0, OB_SH_GROUPS);
        a.row_base = groups[g0].row0; a.rows = 0;
        int64_t items = 0;
        for (int i = 0; i < a.n_groups; ++i) {
            const onebit_prefix_t &g = groups[g0 + i];
            const int64_t chunks = chunks_of(g);
            items += chunks ? chunks * ob_up(g.n * rep, p.per) : 0;
            a.g[i] = {g.row0, g.n, g.slot, g.len, g.first, (int)chunks, (int)items};
            a.rows += g.n;
        }
        const int64_t own_items = (int64_t)a.rows * p.own_mb * std::max(p.osplits, 1);
        a.one_items = (int)items;
        hipStream_t s = (hipStream_t)stream;
        if (head_dim == 128) ob_sh_launch<128, true>(a, p, items, own_items, s);
        else if (head_dim == 64) ob_sh_launch<64, true>(a, p, items, own_items, s);
        else if (head_dim > 64) ob_sh_launch<128, false>(a, p, items, own_items, s);
        else ob_sh_launch<64, false>(a, p, items, own_items, s);
        const int rc2 = ob_launch_status("attention_shared_rows");
        if (rc2) return rc2;
    }
    return 0;
}

// ---------------------------------------------------------------------------------------------- the choice of hypotheses --
static int ob_bs_check(int64_t groups, int32_t beams, int64_t vocab, int32_t keep)
{
    if (groups < 0 || vocab < 1) return ob_fail(ONEBIT_E_ARG, "beam_select: bad size");
    if (beams < 1 || beams > OB_BS_MAX_BEAMS || keep < 1 || keep > OB_BS_MAX_KEEP)
        return ob_fail(ONEBIT_E_SHAPE, "beam_select: %d beams (1 .. %d), %d kept (1 .. %d)", beams, OB_BS_MAX_BEAMS, keep, OB_BS_MAX_KEEP);
    if (vocab > (1 << 20) || groups > 65535 || groups * beams > 65535) return ob_fail(ONEBIT_E_ARG, "beam_select: dimension too large");
    return 0;
}

// pieces of 8 elements per thread, chunks of a row and pieces of a chunk (as even as they go); fused: the scan's last workgroups pick
struct ObBsPlan { int nv, chunks, vecs; bool fused; };
static ObBsPlan ob_bs_plan(int64_t groups, int32_t beams, int64_t vocab, int32_t keep)
{
    const int64_t all = ob_up(vocab, 8), one = ob_up(all, OB_BS_THREADS), few = 256 * OB_BS_PLACES;
    ObBsPlan p;
    // (us of both halves, groups x beams, vocabulary 32000 if not said otherwise; the other side in brackets)
    // four pieces a thread: 1 x 4 12.4 (one piece 13.7), 16 x 1 11.0 (12.1), 16 x 4 13.0 (15.1), 64 x 4 16.1 (22.1), 64 x 4 of 50257 18.4 (26.7); one: 1 x 1 9.6 (four 9.9), 64 x 4 of 512
    // 13.4 (15.4)
    p.nv = one >= 4 && (beams * one >= 64 || groups * beams * one > 128) ? 4 : 1;
    p.chunks = (int)ob_up(all, p.nv * OB_BS_THREADS);
    p.vecs = (int)ob_up(all, p.chunks);
    // one launch: 1 x 4 12.4 (two 12.1), 2 x 8 16.0 (15.7), 4 x 4 12.8 (12.8), and 4 less on the host; 16 x 4, 256 workgroups, 15.1 (13.0), 64 x 4, 1024, 18.6 (16.1)
    p.fused = groups <= OB_BS_TICKETS && groups * beams * p.chunks <= 128 && (int64_t)beams * p.chunks * ob_bs_list(keep) <= few;
    return p;
}

extern "C" size_t onebit_beam_select_scratch_bytes(int64_t rows, int64_t vocab, int32_t keep)
{
    if (rows <= 0 || vocab <= 0 || keep <= 0 || rows > 65535 || vocab > (1 << 20) || keep > OB_BS_MAX_KEEP) return 0;
    return OB_BS_TICKETS * 4 + (size_t)rows * ob_up(vocab, 8 * OB_BS_THREADS) * (16 + 4 + 8 * (size_t)ob_bs_list(keep));
}

template <typename T>
static void ob_bs_scan(const ObBsArgs &a, const ObBsPlan &p, const dim3 &grid, const dim3 &block, hipStream_t s)
{
    if (p.fused) {
        if (p.nv == 1) hipLaunchKernelGGL((ob_bs_scan_kernel<T, 1, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((ob_bs_scan_kernel<T, 4, true>), grid, block, 0, s, a);
    } else if (p.nv == 1) hipLaunchKernelGGL((ob_bs_scan_kernel<T, 1, false>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((ob_bs_scan_kernel<T, 4, false>), grid, block, 0, s, a);
}

extern "C" int onebit_beam_select(const void *logits, int64_t ld, int dtype, const float *scores, int64_t groups, int32_t beams, int64_t vocab, int32_t keep,
                                  float *out_scores, int32_t *out_beams, int32_t *out_tokens, void *scratch, size_t scratch_bytes, void *stream)
{
    const int rc = ob_bs_check(groups, beams, vocab, keep);
    if (rc) return rc;
    if (dtype != ONEBIT_F16 && dtype != ONEBIT_F32) return ob_fail(ONEBIT_E_DTYPE, "beam_select: dtype %d", dtype);
    if (ld < vocab) return ob_fail(ONEBIT_E_SHAPE, "beam_select: row pitch %lld below %lld logits", (long long)ld, (long long)vocab);
    if (groups == 0) return 0;
    if (!logits || !scores || !out_scores || !out_beams || !out_tokens) return ob_fail(ONEBIT_E_ARG, "beam_select: null pointer");
    if (!ob_aligned(logits, dtype == ONEBIT_F16 ? 2 : 4) || !ob_aligned(scores, 4) || !ob_aligned(out_scores, 4) || !ob_aligned(out_beams, 4) || !ob_aligned(out_tokens, 4))
        return ob_fail(ONEBIT_E_ALIGN, "beam_select: misaligned pointer");
    const int64_t rows = groups * beams;
    const size_t need = onebit_beam_select_scratch_bytes(rows, vocab, keep);
    if (!scratch || scratch_bytes < need || !ob_aligned(scratch, 16)) return ob_fail(ONEBIT_E_WSPACE, "beam_select: needs %zu bytes of zero-initialised, 16-byte aligned scratch", need);
    // (a group's results are written while others' scores and logits are still read)
    const unsigned __int128 n_out = (unsigned __int128)groups * keep * 4;
    const ObMem mem[] = {{out_scores, n_out}, {out_beams, n_out}, {out_tokens, n_out}, {scratch, need}, {scores, (unsigned __int128)rows * 4},
                         {logits, ((unsigned __int128)(rows - 1) * ld + vocab) * (dtype == ONEBIT_F16 ? 2 : 4)}};
    for (int i = 0; i < 4; ++i)
        for (int j = i + 1; j < 6; ++j)
            if (ob_overlap(mem[i], mem[j])) return ob_fail(ONEBIT_E_ARG, "beam_select: outputs and scratch memory overlap nothing else");
    ObBsArgs a = {};
    const ObBsPlan p = ob_bs_plan(groups, beams, vocab, keep);
    a.logits = logits; a.ld = ld; a.scores = scores; a.beams = beams; a.keep = keep; a.vocab = (int)vocab; a.chunks = p.chunks; a.vecs = p.vecs;
    a.inv_room = ob_bs_inverse(ob_bs_list(keep)); a.inv_chunks = ob_bs_inverse(p.chunks);
    const size_t lists = (size_t)rows * p.chunks;
    a.tickets = (int *)scratch;
    a.sums = (double *)(a.tickets + OB_BS_TICKETS);
    a.counts = (int *)(a.sums + 2 * lists);
    a.list_x = (float *)(a.counts + lists);
    a.list_t = (int *)(a.list_x + lists * ob_bs_list(keep));
    a.out_scores = out_scores; a.out_beams = out_beams; a.out_tokens = out_tokens;
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)a.chunks, (unsigned)rows), block(OB_BS_THREADS);
    if (dtype == ONEBIT_F16) ob_bs_scan<_Float16>(a, p, grid, block, s);
    else ob_bs_scan<float>(a, p, grid, block, s);
    const bool few = (int64_t)beams * p.chunks * ob_bs_list(keep) <= 256 * OB_BS_PLACES;
    if (!p.fused && few) hipLaunchKernelGGL((ob_bs_pick_kernel<256>), dim3((unsigned)groups), dim3(256), 0, s, a);
    else if (!p.fused) hipLaunchKernelGGL((ob_bs_pick_kernel<1024>), dim3((unsigned)groups), dim3(1024), 0, s, a);
    return ob_launch_status("beam_select");
}

// ------------------------------------------------------------------------------------------------------ states reordered --
template <typename U>
static void ob_re_launch(const ObReArgs &a, const dim3 &grid, hipStream_t s)
{
    if (a.beams <= 4) hipLaunchKernelGGL((ob_re_kernel<4, U>), grid, dim3(OB_RE_THREADS), 0, s, a);
    else if (a.beams <= 16) hipLaunchKernelGGL((ob_re_kernel<16, U>), grid, dim3(OB_RE_THREADS), 0, s, a);
    else hipLaunchKernelGGL((ob_re_kernel<32, U>), grid, dim3(OB_RE_THREADS), 0, s, a);
}

extern "C" int onebit_reorder_slots(void *const *buffers, int32_t n_buffers, const int32_t *parents, int64_t groups, int32_t beams, int64_t slot_bytes,
                                    int64_t outer, int64_t outer_bytes, int64_t first_byte, int64_t n_bytes, void *stream)
{
    if (n_buffers < 0 || groups < 0 || outer < 0 || first_byte < 0 || n_bytes < 0 || outer_bytes < 0 || slot_bytes < 0)
        return ob_fail(ONEBIT_E_ARG, "reorder_slots: negative size");
    if (beams < 1 || beams > OB_RE_MAX_BEAMS || groups > 65535) return ob_fail(ONEBIT_E_SHAPE, "reorder_slots: %lld groups of %d beams (1 .. %d)", (long long)groups, beams, OB_RE_MAX_BEAMS);
    const int64_t most = (int64_t)1 << 46;
    if (slot_bytes > most || outer > most / std::max<int64_t>(n_bytes, 1) || (outer > 0 && first_byte + n_bytes > outer_bytes) ||
        (outer > 0 && outer_bytes > slot_bytes / outer))
        return ob_fail(ONEBIT_E_SHAPE, "reorder_slots: %lld rows of %lld bytes (%lld from %lld on) do not lie in slots of %lld", (long long)outer, (long long)outer_bytes,
                       (long long)n_bytes, (long long)first_byte, (long long)slot_bytes);
    if (n_buffers == 0 || groups == 0 || outer == 0 || n_bytes == 0) return 0;
    if (!buffers || !parents) return ob_fail(ONEBIT_E_ARG, "reorder_slots: null pointer");
    if (!ob_aligned(parents, 4)) return ob_fail(ONEBIT_E_ALIGN, "reorder_slots: misaligned parents");
    uint64_t low = (uint64_t)(slot_bytes | outer_bytes | first_byte | n_bytes);
    for (int i = 0; i < n_buffers; ++i) {
        if (!buffers[i]) return ob_fail(ONEBIT_E_ARG, "reorder_slots: null buffer %d", i);
        low |= (uint64_t)(uintptr_t)buffers[i];
    }
    for (int i = 0; i < n_buffers; ++i)                                          // (workgroups that come later would read what others have written)
        if (ob_overlap({buffers[i], (unsigned __int128)groups * beams * slot_bytes}, {parents, (unsigned __int128)groups * beams * 4}))
            return ob_fail(ONEBIT_E_ARG, "reorder_slots: the parents overlap buffer %d", i);
    const int unit = low % 16 == 0 ? 16 : low % 4 == 0 ? 4 : 1;
    ObReArgs a = {};
    a.parents = parents; a.slot_bytes = slot_bytes; a.outer_bytes = outer_bytes; a.first_byte = first_byte; a.beams = beams;
    if (n_bytes / unit > 0x7fffffffLL) return ob_fail(ONEBIT_E_ARG, "reorder_slots: dimension too large");
    a.units_per = (int)(n_bytes / unit);
    a.units = outer * a.units_per;
    const int64_t wgs = ob_up(a.units, OB_RE_THREADS);
    if (wgs > OB_MAX_WGS) return ob_fail(ONEBIT_E_ARG, "reorder_slots: dimension too large");
    for (int b0 = 0; b0 < n_buffers; b0 += OB_RE_BUFFERS) {
        const int n = std::min(n_buffers - b0, OB_RE_BUFFERS);
        for (int i = 0; i < n; ++i) a.buf[i] = (char *)buffers[b0 + i];
        const dim3 grid((unsigned)wgs, (unsigned)groups, (unsigned)n);
        if (unit == 16) ob_re_launch<ob_u32x4>(a, grid, (hipStream_t)stream);
        else if (unit == 4) ob_re_launch<uint32_t>(a, grid, (hipStream_t)stream);
        else ob_re_launch<uint8_t>(a, grid, (hipStream_t)stream);
        const int rc = ob_launch_status("reorder_slots");
        if (rc) return rc;
    }
    return 0;
}
