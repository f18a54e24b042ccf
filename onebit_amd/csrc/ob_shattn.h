// Attention of single-token rows that share a prefix of their keys and values, gfx950: row r of group g attends to the group's
// prefix (len rows of one slot of the prefix cache, stored once for all rows of the group) and to its own later positions (rows
// first .. pos of its own slot):
//   o = sum_j e^{s_j} v_j / sum_j e^{s_j},  s_j = q . k_j / sqrt(D),  j over prefix and own keys together
// A key range is a PART: its maximum m, sum l = sum e^{s - m} and o = sum e^{s - m} v in fp32; parts join by
//   M = max m_p,  l = sum e^{m_p - M} l_p,  o = sum e^{m_p - M} o_p / l          (ob_sh_join_kernel)
// so prefix chunks and own chunks are workgroups of one launch, and the order of the join is the order of the parts.
//
// Workgroup = (16 MT queries of one kv head) x (one chunk of keys): the queries of a prefix chunk are the rows of the group times
// the query heads of the kv head, those of an own chunk one row's query heads.  Four waves take 32 keys in turn, each with its
// own (m, l, o), joined through LDS at the end: no barrier in the loop, a wave's next 32 keys and values are on their way in
// registers while it computes.  Both products are computed transposed, S^T = K Q^T and O^T = V^T P^T (MFMA 16x16x32): a lane holds
// 4 consecutive keys of one query per 16-key tile, which are, for two tiles, its 8 k elements of the second product; V stays
// row-major in the wave's part of the LDS and is transposed by ds_read_b64_tr_b16.
// Scores, maxima, sums and outputs are fp32.  The weights e^{s - m} enter the second product as fp16 (relative error 2^-11 each, which the
// sum averages; the output is rounded to fp16 anyway), the denominator sums the same rounded weights.
#pragma once
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
    float *part_o;                     // [rows][H][splits][D]
    float *part_ml;                    // [rows][H][splits][2]   {max (log2 domain), sum}
    long long p_max_len, max_len;
    int H, Hkv, rep, D, n_slots, rows, row_base;      // rows: of this launch, from row_base on
    int pchunk, ochunk, psplits, osplits;             // keys per chunk; parts of a row: psplits of the prefix, then osplits of its own
    int own_item0, own_mb, max_own;                   // first item of the own chunks; query blocks per row; most own positions
    float scale_log2e;                                // log2(e) / sqrt(D)
    int n_groups;
    ObShGroup g[OB_SH_GROUPS];
};

typedef short ob_sh_v4s __attribute__((ext_vector_type(4)));
typedef short ob_sh_v8s __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) ob_sh_v4s ob_sh_lds_v4s;

// v over the wave's four 16-lane rows (same lane & 15)
__device__ __forceinline__ float ob_sh_rows_sum(float v)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float ob_sh_rows_max(float v)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float ob_sh_weight(float m, float M) { return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M); }

// LDS of a workgroup, floats: four waves' V tiles [32][DP] fp16, later two output buffers of 16 MT queries; behind them the waves' statistics
template <int DP, int MT> constexpr int ob_sh_body_floats() { return (4 * 32 * DP * 2 > 2 * MT * 16 * DP * 4 ? 4 * 32 * DP * 2 : 2 * MT * 16 * DP * 4) / 4; }
template <int DP, int MT> constexpr int ob_sh_lds_floats() { return ob_sh_body_floats<DP, MT>() + 4 * MT * 16 * 2; }

// Keys k0 .. k1 - 1 of one slot and kv head (kb, vb: its rows) for queries qi0 .. of nq, query i = (row row0 + i / rep, head kvh rep + i % rep);
// the result is part `split` of each.  DP: head size padded to 64 or 128 (EXACT: it is the head size).
template <int DP, int MT, bool EXACT>
__device__ __forceinline__ void ob_sh_body(const ObShArgs &A, const _Float16 *kb, const _Float16 *vb, int k0, int k1, int row0, int qi0, int nq, int kvh,
                                           int split, float *sm)
{
    constexpr int DK = DP / 32, DT = DP / 16, PPR = DP / 8, RPL = 64 / PPR, NV = 32 / RPL;       // pieces of 16 bytes per row, rows per load, loads of a V tile
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, g = lane >> 4;
    const int D = EXACT ? DP : A.D;
    _Float16 *vt = reinterpret_cast<_Float16 *>(sm) + wave * 32 * DP;
    ob_half8 qf[MT][DK];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int qi = min(qi0 + 16 * mt + lr, nq - 1);
        const _Float16 *qr = A.q + ((int64_t)(row0 + qi / A.rep) * A.H + kvh * A.rep + qi % A.rep) * D;
#pragma unroll
        for (int j = 0; j < DK; ++j) {
            const int d = 32 * j + 8 * g;
            qf[mt][j] = EXACT || d < D ? *reinterpret_cast<const ob_half8 *>(qr + d) : (ob_half8)(_Float16)0;
        }
    }
    float m[MT], l[MT];
    ob_float4 acc[MT][DT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        m[mt] = -INFINITY; l[mt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[mt][dt] = (ob_float4){0.f, 0.f, 0.f, 0.f};
    }
    ob_half8 kf[2][DK], vr[NV];
    const int vrow = lane / PPR, vpc = lane % PPR;                     // this lane's piece of a V load: row vrow + RPL i, piece vpc
    const auto load_k = [&](int base) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const _Float16 *r = kb + (int64_t)min(base + 16 * kt + lr, k1 - 1) * D;
#pragma unroll
            for (int j = 0; j < DK; ++j) {
                const int d = 32 * j + 8 * g;
                kf[kt][j] = EXACT || d < D ? *reinterpret_cast<const ob_half8 *>(r + d) : (ob_half8)(_Float16)0;
            }
        }
    };
    const auto load_v = [&](int base) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const _Float16 *r = vb + (int64_t)min(base + vrow + RPL * i, k1 - 1) * D + 8 * vpc;
            vr[i] = EXACT || 8 * vpc < D ? *reinterpret_cast<const ob_half8 *>(r) : (ob_half8)(_Float16)0;
        }
    };
    int base = k0 + 32 * wave;
    if (base < k1) { load_k(base); load_v(base); }
    for (; base < k1; base += 128) {
        const bool tail = base + 32 > k1, more = base + 128 < k1;
        // V tile into the LDS, pairs of pieces swizzled by the row; rows beyond the range as zeros (their weights are zero, their values may be anything)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int row = vrow + RPL * i;
            if (tail && base + row >= k1) vr[i] = (ob_half8)(_Float16)0;
            *reinterpret_cast<ob_half8 *>(vt + row * DP + 8 * (2 * ((vpc >> 1) ^ (row & (DT - 1))) + (vpc & 1))) = vr[i];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (more) load_v(base + 128);
        ob_float4 s[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                s[mt][kt] = (ob_float4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < DK; ++j) s[mt][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[kt][j], qf[mt][j], s[mt][kt], 0, 0, 0);
            }
        if (more) load_k(base + 128);
        ob_half8 pb[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float x[8], mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = s[mt][e >> 2][e & 3] * A.scale_log2e;
                if (tail && base + 16 * (e >> 2) + 4 * g + (e & 3) >= k1) x[e] = -INFINITY;
                mx = fmaxf(mx, x[e]);
            }
            mx = ob_sh_rows_max(mx);
            // the running maximum moves only where a tile exceeds it by 2^8: the weights stay far inside fp16, the output is rescaled seldom
            if (__any(mx > m[mt] + 8.f)) {
                const float mn = fmaxf(m[mt], mx), f = ob_sh_weight(m[mt], mn);
                l[mt] *= f;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[mt][dt] *= f;
                m[mt] = mn;
            }
            const float mu = m[mt] == -INFINITY ? 0.f : m[mt];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                pb[mt][e] = (_Float16)__builtin_amdgcn_exp2f(x[e] - mu);
                l[mt] += (float)pb[mt][e];
            }
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            ob_sh_v4s a[2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const int row = 16 * kt + 4 * g + (lr >> 2);
                a[kt] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (ob_sh_lds_v4s *)(vt + row * DP + 8 * (2 * (dt ^ (row & (DT - 1))) + ((lr & 3) >> 1)) + 4 * (lr & 1)));
            }
            const ob_sh_v8s av = {a[0][0], a[0][1], a[0][2], a[0][3], a[1][0], a[1][1], a[1][2], a[1][3]};
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[mt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ob_half8, av), pb[mt], acc[mt][dt], 0, 0, 0);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    // ---- join the four waves: statistics, then the outputs in two steps through two buffers
    float *st = sm + ob_sh_body_floats<DP, MT>();                      // [4 waves][16 MT][2]
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        l[mt] = ob_sh_rows_sum(l[mt]);
        if (g == 0) { st[(wave * 16 * MT + 16 * mt + lr) * 2] = m[mt]; st[(wave * 16 * MT + 16 * mt + lr) * 2 + 1] = l[mt]; }
    }
    __syncthreads();
    ob_float4 *buf = reinterpret_cast<ob_float4 *>(sm);                // [2][MT][DT][64]
    float M[MT], lt[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const float *sq = st + (16 * mt + lr) * 2;
        M[mt] = fmaxf(fmaxf(sq[0], sq[32 * MT]), fmaxf(sq[64 * MT], sq[96 * MT]));
        lt[mt] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) lt[mt] += sq[32 * MT * w + 1] * ob_sh_weight(sq[32 * MT * w], M[mt]);
        const float f = ob_sh_weight(m[mt], M[mt]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            acc[mt][dt] *= f;
            if (wave >= 2) buf[((wave - 2) * MT * DT + mt * DT + dt) * 64 + lane] = acc[mt][dt];
        }
    }
    __syncthreads();
    if (wave < 2)
#pragma unroll
        for (int i = 0; i < MT * DT; ++i) {
            acc[i / DT][i % DT] += buf[(wave * MT * DT + i) * 64 + lane];
            if (wave == 1) buf[(MT * DT + i) * 64 + lane] = acc[i / DT][i % DT];
        }
    __syncthreads();
    if (wave == 0) {
        const int splits = A.psplits + A.osplits;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const int qi = qi0 + 16 * mt + lr;
            if (qi < nq) {
                const int64_t p = ((int64_t)(row0 + qi / A.rep) * A.H + kvh * A.rep + qi % A.rep) * splits + split;
                if (g == 0) *reinterpret_cast<ob_float2 *>(A.part_ml + 2 * p) = (ob_float2){M[mt], lt[mt]};
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    if (EXACT || 16 * dt + 4 * g < D)
                        *reinterpret_cast<ob_float4 *>(A.part_o + p * D + 16 * dt + 4 * g) = acc[mt][dt] + buf[((MT + mt) * DT + dt) * 64 + lane];
            }
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

template <int DP, int MT, bool EXACT>
__global__ __launch_bounds__(OB_SH_THREADS) void ob_sh_part_kernel(const ObShArgs A)
{
    __shared__ __attribute__((aligned(16))) float sm[ob_sh_lds_floats<DP, MT>()];
    const int item = blockIdx.x / A.Hkv, kvh = blockIdx.x % A.Hkv;
    if (item < A.own_item0) {
        int gi = 0;
        while (item >= A.g[gi].item_end) ++gi;
        const ObShGroup G = A.g[gi];
        const int at = item - (gi ? A.g[gi - 1].item_end : 0), chunk = at % G.chunks, mb = at / G.chunks;
        const int64_t row = ((int64_t)G.slot * A.Hkv + kvh) * A.p_max_len * A.D;
        ob_sh_body<DP, MT, EXACT>(A, A.pk + row, A.pv + row, chunk * A.pchunk, min(G.len, (chunk + 1) * A.pchunk), G.row0, 16 * MT * mb, G.n * A.rep, kvh, chunk, sm);
        return;
    }
    const int at = item - A.own_item0, r = A.row_base + at % A.rows, mb = at / A.rows % A.own_mb, split = at / A.rows / A.own_mb;
    int gi = 0, slot, own;
    while (r >= A.g[gi].row0 + A.g[gi].n) ++gi;
    const int first = A.g[gi].first;
    if (!ob_sh_row(A, r, first, slot, own) || split * A.ochunk >= own) return;
    const int64_t row = ((int64_t)slot * A.Hkv + kvh) * A.max_len * A.D;
    ob_sh_body<DP, 1, EXACT>(A, A.k + row, A.v + row, first + split * A.ochunk, first + min(own, (split + 1) * A.ochunk), r, 16 * mb, A.rep, kvh, A.psplits + split, sm);
}

// A wave per (row, head): its parts in order, two output columns a lane.
__global__ __launch_bounds__(OB_SH_THREADS) void ob_sh_join_kernel(const ObShArgs A)
{
    const int w = blockIdx.x * (OB_SH_THREADS / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (w >= A.rows * A.H) return;
    const int r = A.row_base + w / A.H, head = w % A.H;
    int gi = 0, slot, own;
    while (r >= A.g[gi].row0 + A.g[gi].n) ++gi;
    if (!ob_sh_row(A, r, A.g[gi].first, slot, own)) return;                       // idle: its output stays as it is
    const int np = A.g[gi].chunks, n = np + (own + A.ochunk - 1) / A.ochunk;
    const int64_t p0 = ((int64_t)r * A.H + head) * (A.psplits + A.osplits);
    const int d = 2 * lane;
    if (d >= A.D) return;
    float M = -INFINITY, l = 0.f;
    ob_float2 o = {0.f, 0.f};
    for (int s0 = 0; s0 < n; s0 += 8) {
        ob_float2 ml[8], po[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int s = min(s0 + j, n - 1);
            const int64_t p = p0 + (s < np ? s : A.psplits + s - np);
            ml[j] = *reinterpret_cast<const ob_float2 *>(A.part_ml + 2 * p);
            po[j] = *reinterpret_cast<const ob_float2 *>(A.part_o + p * A.D + d);
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
                o += x * po[j];
            }
    }
    _Float16 *out = A.o + ((int64_t)r * A.H + head) * A.D + d;
    ob_half2 y = {(_Float16)0, (_Float16)0};                                       // no key at all: zeros
    if (n) { y[0] = (_Float16)(o[0] / l); y[1] = (_Float16)(o[1] / l); }
    if (A.h_next) { y[0] *= A.h_next[head * A.D + d]; y[1] *= A.h_next[head * A.D + d + 1]; }
    out[0] = y[0]; out[1] = y[1];
}
