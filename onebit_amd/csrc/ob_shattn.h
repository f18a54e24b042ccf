// Attention of single-token rows that share a prefix of their keys and values, gfx950: row r of group g attends to the group's
// prefix (len rows of one slot of the prefix cache, stored once for all rows of the group) and to its own later positions (rows
// first .. pos of its own slot):
//   o = sum_j e^{s_j} v_j / sum_j e^{s_j},  s_j = q . k_j / sqrt(D),  j over prefix and own keys together
// A range of keys leaves a PART: its maximum m, l = sum e^{s - m} and o = sum e^{s - m} v in fp32.  A part is also a state of the running
// softmax, so parts join by starting from them:  M = max m_p,  l = sum e^{m_p - M} l_p,  o = sum e^{m_p - M} o_p / l.
//   ob_sh_one_kernel     few workgroups: parts of the prefixes, (kv head) x (block of the group's queries) x (chunk of keys), and of the rows' own
//                        keys in one launch; the last workgroup to arrive at a row joins its parts
//   ob_sh_wide_kernel    many: parts of the prefixes, up to 128 queries of a group at a time, then
//   ob_sh_own_kernel     the rows' own keys, started from the prefix's parts: the outputs, or, where a row's own keys are split as well, parts
//                        again, which ob_sh_join_kernel joins.  Where a prefix is so short that every row may read it again, this kernel does, alone.
//                        Where the rows' own keys are the larger share, their workgroups run among the wide kernel's and leave parts
// Parts are joined in their order, whoever does it: deterministic.
//
// Both products are computed transposed, S^T = K Q^T and O^T = V^T P^T (MFMA 16x16x32): a lane holds 4 consecutive keys of one query
// per 16-key tile, which are, for two tiles, its 8 k elements of the second product; V lies row-major in the LDS and is transposed by
// ds_read_b64_tr_b16.  The sum of the weights is one more such product, with ones in V's place.
// Scores, maxima, sums and outputs are fp32.  The weights e^{s - m} enter the second product as fp16 (relative error 2^-11 each, which the
// sum averages; the output is rounded to fp16 anyway), the denominator sums the same rounded weights.
#pragma once
#include <type_traits>
#include "ob_common.h"

#define OB_SH_THREADS 256
#define OB_SH_GROUPS 64            // groups of one launch (they travel in the kernel arguments)

struct ObShGroup { int row0, n, slot, len, first, chunks, item_end; };

struct ObShArgs {
    const _Float16 *q;                 // [rows][H][D]
    const _Float16 *pk, *pv;           // prefix cache [p_slots][Hkv][p_max_len][D]
    const _Float16 *k, *v;             // own cache [n_slots][Hkv][max_len][D]
    _Float16 *o;                       // [rows][H][D]
    const _Float16 *h_next;            // optional [H * D]
    const int *row_slot, *row_pos;     // device [rows]; row_slot NULL: slot = row
    float *part_o;                     // [rows][H][psplits + osplits][D]
    float *part_ml;                    // [rows][H][psplits + osplits][2]   {max (log2 domain), sum}
    long long p_max_len, max_len;
    int H, Hkv, rep, D, n_slots, rows, row_base;      // rows: of this launch, from row_base on
    int pchunk, ochunk, psplits, osplits;             // keys per chunk; parts of a row: psplits of the prefix, then osplits of its own (0: one chunk, no part)
    int own_mb, max_own;                              // query blocks per row and kv head; most own positions
    int inline_prefix;                                // the own kernel reads the prefixes itself
    int one_items;                                    // ob_sh_one_kernel: items of the prefixes, in front of the rows'
    int own_blocks;                                   // ob_sh_wide_kernel: workgroups of the rows' own keys among its others
    int own_alone;                                    // their waves each take a row's keys of a kv head
    int *tickets;                                     // [rows][Hkv] arrivals at a row, zero between launches
    float scale_log2e;                                // log2(e) / sqrt(D)
    int n_groups;
    ObShGroup g[OB_SH_GROUPS];
};

typedef short ob_sh_v4s __attribute__((ext_vector_type(4)));
typedef short ob_sh_v8s __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) ob_sh_v4s ob_sh_lds_v4s;

// largest over the wave's four 16-lane rows (same lane & 15)
__device__ __forceinline__ float ob_sh_rows_max(float v)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
#define OB_SH_NONE -3e38f                // the maximum of no key (finite: differences of two stay numbers)
__device__ __forceinline__ float ob_sh_weight(float m, float M) { return __builtin_amdgcn_exp2f(m - M); }

// LDS place (halves) of 16-byte piece p of row r of a tile of DP columns: pairs of pieces swizzled by the row
template <int DP> __device__ __forceinline__ int ob_sh_place(int r, int p) { return r * DP + 8 * (2 * ((p >> 1) ^ (r & (DP / 16 - 1))) + (p & 1)); }

// The running softmax of 16 MT queries of a wave: query lane & 15 of each tile, output column 16 dt + 4 (lane >> 4) + i
template <int DP, int MT, bool EXACT>
struct ObShWave {
    static constexpr int DK = DP / 32, DT = DP / 16;
    ob_half8 qf[MT][DK];
    ob_float4 m;                       // log2 domain, of the MT tiles (a vector: hipcc keeps an array of them in memory)
    ob_float4 l[MT];                   // sum of the weights, in each of the four
    ob_float4 acc[MT][DT];

    // query i of the block is query qi0 + i of nq: row row0 + (qi0 + i) / rep, head kvh rep + (qi0 + i) % rep
    __device__ __forceinline__ void init(const ObShArgs &A, int row0, int qi0, int nq, int kvh)
    {
        const int lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4, D = EXACT ? DP : A.D;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const int qi = min(qi0 + 16 * mt + lr, nq - 1);
            const _Float16 *qr = A.q + ((int64_t)(row0 + qi / A.rep) * A.H + kvh * A.rep + qi % A.rep) * D;
#pragma unroll
            for (int j = 0; j < DK; ++j) {
                const int d = 32 * j + 8 * g;
                qf[mt][j] = EXACT || d < D ? *reinterpret_cast<const ob_half8 *>(qr + d) : (ob_half8)(_Float16)0;
            }
            m[mt] = OB_SH_NONE;
            l[mt] = (ob_float4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[mt][dt] = (ob_float4){0.f, 0.f, 0.f, 0.f};
        }
    }

    // Scores of 32 keys (kf: their rows); TAIL: only the first `n` count
    template <bool TAIL>
    __device__ __forceinline__ void scores(const ob_half8 (&kf)[2][DK], int n, ob_float4 (&s)[MT][2])
    {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                s[mt][kt] = (ob_float4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < DK; ++j) s[mt][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[kt][j], qf[mt][j], s[mt][kt], 0, 0, 0);
            }
        if (TAIL)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (16 * (e >> 2) + 4 * g + (e & 3) >= n)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) s[mt][e >> 2][e & 3] = -INFINITY;
    }

    // Their weights
    __device__ __forceinline__ void weights(const ob_float4 (&s)[MT][2], float scale, ob_half8 (&pb)[MT])
    {
        // the running maximum moves only where a weight would exceed 2^15 (the first ones do), to where the largest is 2^7: the weights stay inside fp16, those of 2^-21 of
        // the largest and more as normal numbers, and neither the tile's maximum nor a rescaled output is needed otherwise
        float x[MT][8], top = -INFINITY;
        const auto exponents = [&]() {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[mt][e] = __builtin_fmaf(s[mt][e >> 2][e & 3], scale, -m[mt]);
        };
        exponents();
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, x[mt][e]);
        if (__any(top > 15.f)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float mx = s[mt][0][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[mt][e >> 2][e & 3]);
                const float mn = fmaxf(m[mt], __builtin_fmaf(ob_sh_rows_max(mx), scale, -7.f)), f = ob_sh_weight(m[mt], mn);
                l[mt] *= f;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[mt][dt] *= f;
                m[mt] = mn;
            }
            exponents();
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 8; ++e) pb[mt][e] = (_Float16)__builtin_amdgcn_exp2f(x[mt][e]);
    }

    // columns 16 dt .. of the 32 values from vt on, as the second product takes them
    __device__ __forceinline__ ob_half8 columns(const _Float16 *vt, int dt)
    {
        const int lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4;
        ob_sh_v4s a[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
            a[kt] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ob_sh_lds_v4s *)(vt + ob_sh_place<DP>(16 * kt + 4 * g + (lr >> 2), 2 * dt + ((lr & 3) >> 1)) + 4 * (lr & 1)));
        const ob_sh_v8s av = {a[0][0], a[0][1], a[0][2], a[0][3], a[1][0], a[1][1], a[1][2], a[1][3]};
        return __builtin_bit_cast(ob_half8, av);
    }

    // acc += weights . values, vt: the 32 keys' rows in the LDS
    __device__ __forceinline__ void values(const _Float16 *vt, const ob_half8 (&pb)[MT])
    {
        const ob_half8 one = (ob_half8)(_Float16)1;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) l[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, pb[mt], l[mt], 0, 0, 0);
        ob_half8 av[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) av[dt] = columns(vt, dt);
        __builtin_amdgcn_sched_barrier(0);                                       // (all of them on their way: left to itself hipcc waits for one after the other)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[mt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av[dt], pb[mt], acc[mt][dt], 0, 0, 0);
    }
};

// The keys of a workgroup's item: keys begin .. end - 1 of the rows from k, v on
struct ObShRange { const _Float16 *k, *v; int begin, end; };
__device__ __forceinline__ int ob_sh_tiles(int n) { return (n + 31) >> 5; }

// A workgroup's four waves over the keys of two ranges one after the other, 32 in turn; each starts from what W holds, the four results are joined in wave 0's W.  STEP 1: every
// wave goes over ranges of its own, alone.
// meanwhile(W) runs while the first loads are on their way.
// K goes from memory to registers in the layout of its product, V by registers into the wave's own part of the LDS: no barrier in the loop, the
// next 32 keys and values are on their way while a wave computes.
template <int DP, int MT, bool EXACT> constexpr int ob_sh_body_floats() { return (4 * 32 * DP * 2 > 2 * MT * 16 * DP * 4 ? 4 * 32 * DP * 2 : 2 * MT * 16 * DP * 4) / 4; }
template <int DP, int MT, bool EXACT> constexpr int ob_sh_lds_floats() { return ob_sh_body_floats<DP, MT, EXACT>() + 4 * MT * 16 * 2; }

template <int DP, int MT, bool EXACT, int STEP = 4, typename F>
__device__ __forceinline__ void ob_sh_sweep(const ObShArgs &A, const ObShRange &R0, const ObShRange &R1, ObShWave<DP, MT, EXACT> &W, float *sm, F meanwhile)
{
    constexpr int DK = DP / 32, DT = DP / 16, PPR = DP / 8, RPL = 64 / PPR, NV = 32 / RPL;       // pieces of 16 bytes per row, rows per load, loads of a V tile
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 15, g = lane >> 4;
    const int D = EXACT ? DP : A.D;
    _Float16 *vt = reinterpret_cast<_Float16 *>(sm) + wave * 32 * DP;
    ob_half8 kf[2][DK], vr[NV];
    const int vrow = lane / PPR, vpc = lane % PPR;                     // this lane's piece of a V load: row vrow + RPL i, piece vpc
    const int n0 = ob_sh_tiles(R0.end - R0.begin), n = n0 + ob_sh_tiles(R1.end - R1.begin);
    const auto load_k = [&](int t) {
        const bool one = t < n0;
        const int last = (one ? R0.end : R1.end) - 1, base = one ? R0.begin + 32 * t : R1.begin + 32 * (t - n0);
        const _Float16 *kb = one ? R0.k : R1.k;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const _Float16 *p = kb + (int64_t)min(base + 16 * kt + lr, last) * D;
#pragma unroll
            for (int j = 0; j < DK; ++j) {
                const int d = 32 * j + 8 * g;
                kf[kt][j] = EXACT || d < D ? *reinterpret_cast<const ob_half8 *>(p + d) : (ob_half8)(_Float16)0;
            }
        }
    };
    const auto load_v = [&](int t) {
        const bool one = t < n0;
        const int last = (one ? R0.end : R1.end) - 1, base = one ? R0.begin + 32 * t : R1.begin + 32 * (t - n0);
        const _Float16 *vb = one ? R0.v : R1.v;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const _Float16 *p = vb + (int64_t)min(base + vrow + RPL * i, last) * D + 8 * vpc;
            vr[i] = EXACT || 8 * vpc < D ? *reinterpret_cast<const ob_half8 *>(p) : (ob_half8)(_Float16)0;
        }
    };
    const int t0 = STEP == 4 ? wave : 0;
    if (t0 < n) { load_v(t0); load_k(t0); }                            // (values first, as in the loop: what waits for them lets the keys come)
    meanwhile(W);
    for (int t = t0; t < n; t += STEP) {
        const bool one = t < n0;
        const int end = one ? R0.end : R1.end, base = one ? R0.begin + 32 * t : R1.begin + 32 * (t - n0);
        // rows beyond the range as zeros (their weights are zero, their values may be anything)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int row = vrow + RPL * i;
            if (base + 32 > end && base + row >= end) vr[i] = (ob_half8)(_Float16)0;
            *reinterpret_cast<ob_half8 *>(vt + ob_sh_place<DP>(row, vpc)) = vr[i];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (t + STEP < n) load_v(t + STEP);
        ob_half8 pb[MT];
        ob_float4 s[MT][2];
        W.template scores<true>(kf, end - base, s);
        W.weights(s, A.scale_log2e, pb);
        if (t + STEP < n) load_k(t + STEP);
        W.values(vt, pb);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    if (STEP == 1) return;
    // ---- join the four waves: statistics, then the outputs in two steps through two buffers
    float *st = sm + ob_sh_body_floats<DP, MT, EXACT>();               // [4 waves][16 MT][2]
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
        if (g == 0) *reinterpret_cast<ob_float2 *>(st + (wave * 16 * MT + 16 * mt + lr) * 2) = (ob_float2){W.m[mt], W.l[mt][0]};
    __syncthreads();
    ob_float4 *buf = reinterpret_cast<ob_float4 *>(sm);                // [2][MT][DT][64]
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const float *sq = st + (16 * mt + lr) * 2;
        const float M = fmaxf(fmaxf(sq[0], sq[32 * MT]), fmaxf(sq[64 * MT], sq[96 * MT])), f = ob_sh_weight(W.m[mt], M);
        float lt = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) lt += sq[32 * MT * w + 1] * ob_sh_weight(sq[32 * MT * w], M);
        W.m[mt] = M;
        W.l[mt][0] = lt;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) W.acc[mt][dt] *= f;
    }
    if (wave >= 2)
#pragma unroll
        for (int i = 0; i < MT * DT; ++i) buf[((wave - 2) * MT * DT + i) * 64 + lane] = W.acc[i / DT][i % DT];
    __syncthreads();
    if (wave < 2) {
#pragma unroll
        for (int i = 0; i < MT * DT; ++i) W.acc[i / DT][i % DT] += buf[(wave * MT * DT + i) * 64 + lane];
        if (wave == 1)
#pragma unroll
            for (int i = 0; i < MT * DT; ++i) buf[(MT * DT + i) * 64 + lane] = W.acc[i / DT][i % DT];
    }
    __syncthreads();
    if (wave == 0)
#pragma unroll
        for (int i = 0; i < MT * DT; ++i) W.acc[i / DT][i % DT] += buf[(MT * DT + i) * 64 + lane];
}

// What W holds of the queries qi0 .. of nq as their part `split`; AGENT: past the XCD's L2, for readers of the same launch
template <int DP, int MT, bool EXACT, bool AGENT = false>
__device__ __forceinline__ void ob_sh_store(const ObShArgs &A, const ObShWave<DP, MT, EXACT> &W, int row0, int qi0, int nq, int kvh, int split)
{
    const int lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4, D = EXACT ? DP : A.D;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int qi = qi0 + 16 * mt + lr;
        if (qi >= nq) continue;
        const int64_t p = ((int64_t)(row0 + qi / A.rep) * A.H + kvh * A.rep + qi % A.rep) * (A.psplits + A.osplits) + split;
        const auto two = [](float *to, float a, float b) {
            const ob_float2 v = {a, b};
            if (AGENT) __hip_atomic_store(reinterpret_cast<unsigned long long *>(to), __builtin_bit_cast(unsigned long long, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            else *reinterpret_cast<ob_float2 *>(to) = v;
        };
        if (g == 0) two(A.part_ml + 2 * p, W.m[mt], W.l[mt][0]);
#pragma unroll
        for (int dt = 0; dt < DP / 16; ++dt) {
            float *to = A.part_o + p * D + 16 * dt + 4 * g;
            if (!EXACT && 16 * dt + 4 * g >= D) continue;
            if (!AGENT) { *reinterpret_cast<ob_float4 *>(to) = W.acc[mt][dt]; continue; }
            two(to, W.acc[mt][dt][0], W.acc[mt][dt][1]);
            two(to + 2, W.acc[mt][dt][2], W.acc[mt][dt][3]);
        }
    }
}

// own keys of a row (0: none), false for an idle row
__device__ __forceinline__ bool ob_sh_row(const ObShArgs &A, int row, int first, int &slot, int &own)
{
    slot = A.row_slot ? A.row_slot[row] : row;
    const int pos = A.row_pos[row];
    if (slot < 0 || slot >= A.n_slots || pos < 0 || pos >= A.max_len) return false;
    own = max(0, min(pos + 1 - first, A.max_own));
    return true;
}

// a prefix item: kv head kvh, keys k0 .. k1 - 1 of the group's prefix (rows from kb, vb on), chunk and block of `per` queries
struct ObShItem { int kvh, chunk, qi0, k0, k1; const _Float16 *kb, *vb; };
__device__ __forceinline__ ObShItem ob_sh_item(const ObShArgs &A, int block, int per, ObShGroup &G)
{
    ObShItem I;
    const int item = block / A.Hkv;
    I.kvh = block - item * A.Hkv;
    int gi = 0;
    while (item >= A.g[gi].item_end) ++gi;
    G = A.g[gi];
    const int at = item - (gi ? A.g[gi - 1].item_end : 0), mb = at / G.chunks;
    I.chunk = at - mb * G.chunks;
    I.qi0 = per * mb;
    I.k0 = I.chunk * A.pchunk;
    I.k1 = min(G.len, I.k0 + A.pchunk);
    const int64_t row = ((int64_t)G.slot * A.Hkv + I.kvh) * A.p_max_len * A.D;
    I.kb = A.pk + row;
    I.vb = A.pv + row;
    return I;
}

// More queries: the four waves share the queries out, 16 MT each, over tiles of 64 keys and values that they read from the LDS together (two tiles
// there, brought by DMA; one barrier a tile).  The second half's keys are read while the first one's exponentials run.
// MT = 2: 64 rows of 64 / 8 heads over 32768 keys 79 us, 0.87 PFLOP/s (tiles through registers 88; MT = 4 140: 490 registers, one wave a SIMD): products, vector
// instructions and LDS reads, 31, 28 and 29 us of them each, mostly in turn.
template <int DP, int MT, bool EXACT>
__device__ __forceinline__ void ob_sh_wide(const ObShArgs &A, const ObShItem &I, const ObShGroup &G, _Float16 (*kv)[2][64 * DP])
{
    constexpr int DK = DP / 32, PPR = DP / 8, RPL = 64 / PPR, NL = 64 / RPL / 4;      // pieces of 16 bytes per row, rows per DMA, DMAs of a wave
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 15, g = lane >> 4;
    const int D = EXACT ? DP : A.D, qi0 = I.qi0 + 16 * MT * wave, nq = G.n * A.rep;
    ObShWave<DP, MT, EXACT> W;
    W.init(A, G.row0, qi0, nq, I.kvh);
    // a lane brings what belongs at its place of RPL rows: row lane / PPR of them (the same of every eight), place lane % PPR
    const int row = lane / PPR, at = lane % PPR;
    const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char *)&kv[0][0][0];
    const auto load = [&](int base, int b) {
        const int most = I.k1 - 1 - base;                                        // (rows behind the last one: the last one again; its scores there are left out, its values written over)
        const char *kb = reinterpret_cast<const char *>(I.kb + (int64_t)base * D), *vb = reinterpret_cast<const char *>(I.vb + (int64_t)base * D);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int r = RPL * (NL * wave + i) + row, p = 2 * ((at >> 1) ^ (r & (DP / 16 - 1))) + (at & 1);
            const uint32_t off = (uint32_t)(min(r, most) * D + 8 * p) * 2, to = lds0 + (uint32_t)b * (2 * 64 * DP * 2) + (NL * wave + i) * 1024;
            if (EXACT || 8 * p < D) {
                ob_dma_1k(kb, off, to);
                ob_dma_1k(vb, off, to + 64 * DP * 2);
            }
        }
    };
    const auto landed = [&]() {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    if (!EXACT) {                                                                // columns from D on are not brought: zeros
        for (int i = tid; i < 4 * 64 * PPR; i += OB_SH_THREADS) *reinterpret_cast<ob_half8 *>(&kv[0][0][8 * i]) = (ob_half8)(_Float16)0;
        __syncthreads();
    }
    load(I.k0, 0);
    landed();
    int b = 0, base = I.k0;
    const auto keys = [&](int h, ob_half8 (&kf)[2][DK]) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int j = 0; j < DK; ++j) kf[kt][j] = *reinterpret_cast<const ob_half8 *>(&kv[b][0][ob_sh_place<DP>(32 * h + 16 * kt + lr, 4 * j + g)]);
    };
    ob_half8 kf[2][DK], pb[MT];
    ob_float4 s[MT][2];
    for (; base + 64 <= I.k1; base += 64, b ^= 1) {
        if (base + 64 < I.k1) load(base + 64, b ^ 1);
        keys(0, kf);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const _Float16 *vt = &kv[b][1][32 * h * DP];
            W.template scores<false>(kf, 32, s);
            if (h == 0) keys(1, kf);
            W.weights(s, A.scale_log2e, pb);
            W.values(vt, pb);
        }
        landed();
    }
    if (base < I.k1) {                                                           // a last tile that is not full: weights of zero, and values that no infinity is among
        for (int i = (I.k1 - base) * PPR + tid; i < 64 * PPR; i += OB_SH_THREADS) *reinterpret_cast<ob_half8 *>(&kv[b][1][8 * i]) = (ob_half8)(_Float16)0;
        __syncthreads();
    }
#pragma unroll 1
    for (int h = 0; base + 32 * h < I.k1; ++h) {
        keys(h, kf);
        W.template scores<true>(kf, I.k1 - base - 32 * h, s);
        W.weights(s, A.scale_log2e, pb);
        W.values(&kv[b][1][32 * h * DP], pb);
    }
    ob_sh_store<DP, MT, EXACT>(A, W, G.row0, qi0, nq, I.kvh, I.chunk);
}

template <int DP, int MT, bool EXACT>
__global__ __launch_bounds__(OB_SH_THREADS, 2) void ob_sh_wide_kernel(const ObShArgs A)
{
    __shared__ __attribute__((aligned(16))) _Float16 kv[2][2][64 * DP];
    const int before = (int)((long long)blockIdx.x * A.own_blocks / gridDim.x);
    if ((int)((long long)(blockIdx.x + 1) * A.own_blocks / gridDim.x) == before) {
        ObShGroup G;
        const ObShItem I = ob_sh_item(A, blockIdx.x - before, 64 * MT, G);
        ob_sh_wide<DP, MT, EXACT>(A, I, G, kv);
        return;
    }
    // (a wave of its own for every row and kv head, or four)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), unit = A.own_alone ? 4 * before + wave : before;
    const int item = unit / A.Hkv, kvh = unit - item * A.Hkv;
    const int at = item / A.rows, r = A.row_base + item - at * A.rows, split = at / A.own_mb, mb = at - split * A.own_mb;
    if (split >= A.osplits) return;
    int gi = 0, slot, own;
    while (r >= A.g[gi].row0 + A.g[gi].n) ++gi;
    const int first = A.g[gi].first;
    if (!ob_sh_row(A, r, first, slot, own) || split * A.ochunk >= own) return;
    const int64_t row = ((int64_t)slot * A.Hkv + kvh) * A.max_len * A.D;
    const ObShRange keys = {A.k + row, A.v + row, first + split * A.ochunk, first + min(own, (split + 1) * A.ochunk)}, none = {A.k + row, A.v + row, 0, 0};
    ObShWave<DP, 1, EXACT> W;
    W.init(A, r, 16 * mb, A.rep, kvh);
    if (A.own_alone) ob_sh_sweep<DP, 1, EXACT, 1>(A, keys, none, W, reinterpret_cast<float *>(kv), [](auto &) {});
    else {
        ob_sh_sweep<DP, 1, EXACT>(A, keys, none, W, reinterpret_cast<float *>(kv), [](auto &) {});
        if (wave) return;
    }
    ob_sh_store<DP, 1, EXACT>(A, W, r, 16 * mb, A.rep, kvh, A.psplits + split);
}

// Bound by HBM: 8 rows x 32 heads of 1000 own keys each 24.7 us, 5.3 TB/s.
// One row's queries of a kv head (16 of them: block mb) over its own keys.  osplits 0: all of them, started from the prefix's parts (the waves take
// them in turn) or from its keys; the output.  Else chunk `split` of them as a part.
template <int DP, bool EXACT>
__global__ __launch_bounds__(OB_SH_THREADS, 2) void ob_sh_own_kernel(const ObShArgs A)
{
    constexpr int DT = DP / 16;
    __shared__ __attribute__((aligned(16))) float sm[ob_sh_lds_floats<DP, 1, EXACT>()];
    const int item = blockIdx.x / A.Hkv, kvh = blockIdx.x - item * A.Hkv;
    const int at = item / A.rows, r = A.row_base + item - at * A.rows, split = at / A.own_mb, mb = at - split * A.own_mb;
    int gi = 0, slot, own;
    while (r >= A.g[gi].row0 + A.g[gi].n) ++gi;
    const ObShGroup &G = A.g[gi];
    const int first = G.first;
    if (!ob_sh_row(A, r, first, slot, own)) return;                               // idle: its output stays as it is
    const bool parts = A.osplits > 0;
    if (parts && split * A.ochunk >= own) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, g = lane >> 4, D = EXACT ? DP : A.D;
    ObShWave<DP, 1, EXACT> W;
    W.init(A, r, 16 * mb, A.rep, kvh);
    const int qi = 16 * mb + lr, head = kvh * A.rep + qi;
    const bool mine = qi < A.rep;
    // the prefix's parts, this wave's of them: two at a time
    const auto start = [&](ObShWave<DP, 1, EXACT> &W) {
        if (parts || A.inline_prefix) return;
        const int64_t p0 = ((int64_t)r * A.H + (mine ? head : 0)) * A.psplits;
        for (int s0 = wave; s0 < G.chunks; s0 += 8) {
            ob_float2 ml[2];
            ob_float4 o[2][DT];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const bool in = mine && s0 + 4 * j < G.chunks;
                const int64_t p = p0 + min(s0 + 4 * j, G.chunks - 1);
                ml[j] = in ? *reinterpret_cast<const ob_float2 *>(A.part_ml + 2 * p) : (ob_float2){OB_SH_NONE, 0.f};
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    o[j][dt] = in && (EXACT || 16 * dt + 4 * g < D) ? *reinterpret_cast<const ob_float4 *>(A.part_o + p * D + 16 * dt + 4 * g) : (ob_float4){0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float M = fmaxf(W.m[0], ml[j][0]), f = ob_sh_weight(W.m[0], M), x = ob_sh_weight(ml[j][0], M);
                W.m[0] = M;
                W.l[0] = W.l[0] * f + x * ml[j][1];
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) W.acc[0][dt] = W.acc[0][dt] * f + o[j][dt] * x;
            }
        }
    };
    const int64_t row = ((int64_t)slot * A.Hkv + kvh) * A.max_len * A.D;
    const int64_t prow = A.inline_prefix ? ((int64_t)G.slot * A.Hkv + kvh) * A.p_max_len * A.D : 0;
    const int k0 = first + (parts ? split * A.ochunk : 0), k1 = first + (parts ? min(own, (split + 1) * A.ochunk) : own);
    ob_sh_sweep<DP, 1, EXACT>(A, {A.pk + prow, A.pv + prow, 0, A.inline_prefix ? G.len : 0}, {A.k + row, A.v + row, k0, k1}, W, sm, start);
    if (wave) return;
    if (parts) {
        ob_sh_store<DP, 1, EXACT>(A, W, r, 16 * mb, A.rep, kvh, A.psplits + split);
        return;
    }
    if (!mine) return;
    const bool any = G.len > 0 || own > 0;                                         // no key at all: zeros
    const float inv = 1.f / W.l[0][0];
    _Float16 *out = A.o + ((int64_t)r * A.H + head) * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        const int d = 16 * dt + 4 * g;
        if (!EXACT && d >= D) continue;
        ob_half4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = (_Float16)(any ? W.acc[0][dt][i] * inv : 0.f);
            if (A.h_next) y[i] *= A.h_next[head * D + d + i];
        }
        *reinterpret_cast<ob_half4 *>(out + d) = y;
    }
}

// Half a wave joins the n parts of (row, head), np of them the prefix's, in order, four output columns a lane (n = 0: zeros)
template <bool AGENT>
__device__ __forceinline__ void ob_sh_join(const ObShArgs &A, int r, int head, int np, int n)
{
    const int d = 4 * (threadIdx.x & 31);
    if (d >= A.D) return;
    const int64_t p0 = ((int64_t)r * A.H + head) * (A.psplits + A.osplits);
    const auto two = [](const float *p) -> ob_float2 {
        if (!AGENT) return *reinterpret_cast<const ob_float2 *>(p);
        return __builtin_bit_cast(ob_float2, __hip_atomic_load(reinterpret_cast<const unsigned long long *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    };
    float M = OB_SH_NONE, l = 0.f;
    ob_float4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < n; s0 += 8) {
        ob_float2 ml[8], po[8][2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int s = min(s0 + j, n - 1);
            const int64_t p = p0 + (s < np ? s : A.psplits + s - np);
            ml[j] = two(A.part_ml + 2 * p);
            po[j][0] = two(A.part_o + p * A.D + d);
            po[j][1] = two(A.part_o + p * A.D + d + 2);
        }
        float mb = M;
#pragma unroll
        for (int j = 0; j < 8; ++j) mb = fmaxf(mb, ml[j][0]);
        const float f = ob_sh_weight(M, mb);
        l *= f; o *= f; M = mb;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (s0 + j < n) {
                const float x = ob_sh_weight(ml[j][0], M);
                l += x * ml[j][1];
                o += x * (ob_float4){po[j][0][0], po[j][0][1], po[j][1][0], po[j][1][1]};
            }
    }
    ob_half4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = n ? (_Float16)(o[i] / l) : (_Float16)0;
        if (A.h_next) y[i] *= A.h_next[head * A.D + d + i];
    }
    *reinterpret_cast<ob_half4 *>(A.o + ((int64_t)r * A.H + head) * A.D + d) = y;
}

__global__ __launch_bounds__(OB_SH_THREADS) void ob_sh_join_kernel(const ObShArgs A)
{
    const int w = blockIdx.x * (OB_SH_THREADS / 32) + (threadIdx.x >> 5);
    if (w >= A.rows * A.H) return;
    const int r = A.row_base + w / A.H, head = w % A.H;
    int gi = 0, slot, own;
    while (r >= A.g[gi].row0 + A.g[gi].n) ++gi;
    if (!ob_sh_row(A, r, A.g[gi].first, slot, own)) return;                       // idle: its output stays as it is
    const int np = A.g[gi].chunks;
    ob_sh_join<false>(A, r, head, np, np + (own + A.ochunk - 1) / A.ochunk);
}

// One launch: the items of the prefixes (up to 16 MT queries of a group), then those of the rows' own keys.  A workgroup publishes its part WRITE-THROUGH
// (agent-scope stores), waits until it has left, and takes a ticket of every row that it holds queries of; the last one at a row joins the row's parts and
// sets the ticket back to zero.  Every row has own items, an empty one if it has no key of its own.  One row of 32 heads over 8192 keys 26.3 us, 5.2 TB/s; 8 rows sharing
// 1000 12 us, of which some 5 are the parts' way out, the ticket and the join (in launches of their own 13.8, and 5 more on the host).
template <int DP, int MT, bool EXACT>
__global__ __launch_bounds__(OB_SH_THREADS, 2) void ob_sh_one_kernel(const ObShArgs A)
{
    __shared__ __attribute__((aligned(16))) float sm[ob_sh_lds_floats<DP, MT, EXACT>()];
    __shared__ int last_s[64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int row0, r_lo, r_hi, kvh, chunks, per, first, n_query;              // rows that this workgroup holds queries of
    if ((int)blockIdx.x < A.one_items * A.Hkv) {
        ObShGroup G;
        const ObShItem I = ob_sh_item(A, blockIdx.x, 16 * MT, G);
        ObShWave<DP, MT, EXACT> W;
        n_query = G.n * A.rep;
        W.init(A, G.row0, I.qi0, n_query, I.kvh);
        ob_sh_sweep<DP, MT, EXACT>(A, {I.kb, I.vb, I.k0, I.k1}, {I.kb, I.vb, 0, 0}, W, sm, [](auto &) {});
        if (wave == 0) ob_sh_store<DP, MT, EXACT, true>(A, W, G.row0, I.qi0, n_query, I.kvh, I.chunk);
        row0 = G.row0; kvh = I.kvh; chunks = G.chunks; first = G.first;
        r_lo = G.row0 + I.qi0 / A.rep;
        r_hi = G.row0 + (min(I.qi0 + 16 * MT, n_query) - 1) / A.rep;
    } else {
        const int at0 = blockIdx.x - A.one_items * A.Hkv, item = at0 / A.Hkv;
        kvh = at0 - item * A.Hkv;
        const int at = item / A.rows, r = A.row_base + item - at * A.rows, split = at / A.own_mb, mb = at - split * A.own_mb;
        int gi = 0, slot, own;
        while (r >= A.g[gi].row0 + A.g[gi].n) ++gi;
        const ObShGroup &G = A.g[gi];
        first = G.first;
        if (!ob_sh_row(A, r, first, slot, own)) return;                          // idle: its output stays as it is
        if (split && split * A.ochunk >= own) return;
        const int64_t row = ((int64_t)slot * A.Hkv + kvh) * A.max_len * A.D;
        ObShWave<DP, 1, EXACT> W;
        W.init(A, r, 16 * mb, A.rep, kvh);
        ob_sh_sweep<DP, 1, EXACT>(A, {A.k + row, A.v + row, first + split * A.ochunk, first + min(own, (split + 1) * A.ochunk)}, {A.k + row, A.v + row, 0, 0}, W, sm,
                                  [](auto &) {});
        if (wave == 0) ob_sh_store<DP, 1, EXACT, true>(A, W, r, 16 * mb, A.rep, kvh, A.psplits + split);
        row0 = G.row0; chunks = G.chunks; n_query = G.n * A.rep;
        r_lo = r_hi = r;
    }
    per = 16 * MT;
    if (wave == 0) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                         // the part has left
        for (int r = r_lo + lane; r <= r_hi; r += 64) {                          // (at most 16 MT rows: one turn)
            int slot, own, last = 0;
            if (ob_sh_row(A, r, first, slot, own)) {
                const int q = (r - row0) * A.rep, blocks = (q + A.rep - 1) / per - q / per + 1;
                const int all = chunks * blocks + A.own_mb * max(1, (own + A.ochunk - 1) / A.ochunk);
                int *t = A.tickets + (int64_t)r * A.Hkv + kvh;
                last = __hip_atomic_fetch_add(t, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == all - 1;
                if (last) __hip_atomic_store(t, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                last = last ? chunks + (own + A.ochunk - 1) / A.ochunk : -1;      // its parts
            } else last = -1;
            last_s[r - r_lo] = last;
        }
    }
    __syncthreads();
    const int pairs = (r_hi - r_lo + 1) * A.rep;
    for (int i = tid >> 5; i < pairs; i += OB_SH_THREADS / 32) {
        const int r = i / A.rep, n = last_s[r];
        if (n >= 0) ob_sh_join<true>(A, r_lo + r, kvh * A.rep + i - r * A.rep, chunks, n);
    }
}
