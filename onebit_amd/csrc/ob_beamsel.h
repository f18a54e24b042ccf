// The continuations that a beam search goes on with, gfx950.  Row r = (group r / beams, beam r % beams) holds the logits of one
// hypothesis; its continuation by token t is worth  v = score_r + (x_t - ln sum_u e^{x_u}),  and a group's `keep` best of beams x vocab
// continuations are wanted in the order (v descending, beam, x descending, token).  Within a row the logits themselves order; between rows v, added and compared in
// 64 bits (two beams' values often lie closer than fp32 resolves), decides as far as the logarithm of the row's sum is known (below).
//   ob_bs_scan_kernel   (row, chunk of the vocabulary): max and sum e^{x - max} of the chunk, and a list of candidates that holds its `keep` best
//   ob_bs_pick          (group): the rows' sums joined, then the `keep` best of the lists; a launch of its own, or, where the scan is small, by the scan's
//                       last workgroup to arrive at the group
// Both find the best by a threshold instead of one after the other: every wave publishes the largest of its lanes' largest values, its share of `keep` and
// two more; at least `keep` candidates reach the keep-th of all published, and few more do; those are listed (the scan) or ranked by counting (the
// pick).  Where too many reach it (rows of equal logits), the best are taken one after the other.
// The logits are read once.  A term e^d, d = x - max, is computed in fp32 and added in 64 bits.  It is off by 2^-24 |d| of itself for the rounded difference (fp32 logits; of
// fp16 ones it is exact where their sizes are alike), by as much for the rounded product with log2 e, by 2^-26 |d| for the rounded constant (always the same way) and by 2^-23 for the
// exponential.  The logarithm of the sum is off by at most  2^-23 (1 + 9/8 mean |d|),  the mean over the row's probabilities (below ln vocab, 10.4 for 32000): 2^-22 .. 2^-20.
// Measured over rows of 32003: values 2.6e-8 too low in the mean, 5e-8 at most (normal logits, sigma 2), 1.3e-7 where many logits are equal.  Values of two beams that lie
// closer than that can come in either order; the scores that a search hands back in fp32 are no finer (2^-24 of themselves).  A row's elements belong to threads by
// their index alone, not by the row's alignment: equal rows have equal sums, bit for bit, and tie exactly.
#pragma once
#include <type_traits>
#include "ob_common.h"

#define OB_BS_THREADS 256
#define OB_BS_MAX_KEEP 64
#define OB_BS_MAX_BEAMS 32
#define OB_BS_LISTS 2048                           // lists of a group that the pick can choose from first
#define OB_BS_TICKETS 4096                         // groups whose pick may be the scan's: counters in front of the scratch memory, zero between launches

// room for the candidates of a chunk
static inline __host__ __device__ int ob_bs_list(int keep) { return keep + keep / 2 + 16; }

struct ObBsArgs {
    const void *logits;
    long long ld;                    // row pitch, elements
    const float *scores;             // [groups * beams]
    int beams, keep, vocab, chunks, vecs;                // vecs: pieces of 8 elements of a chunk
    double *sums;                    // [rows][chunks][2]  {max, sum}
    int *counts;                     // [rows][chunks]
    float *list_x;                   // [rows][chunks][ob_bs_list(keep)]
    int *list_t;
    float *out_scores; int *out_beams, *out_tokens;      // [groups][keep]
    int *tickets;
    unsigned inv_room, inv_chunks;   // ob_bs_inverse of a list's places, of a row's chunks
};
// n / d for n d < 2^31 as one product
static inline unsigned ob_bs_inverse(int d) { return (unsigned)(((1u << 31) + (unsigned)d - 1) / (unsigned)d); }
__device__ __forceinline__ int ob_bs_div(int n, unsigned inverse) { return (int)__umulhi(2u * (unsigned)n, inverse); }

// what a later launch reads, or (AGENT) another workgroup of this one: past the XCD's L2
template <bool AGENT, typename V> __device__ __forceinline__ void ob_bs_put(V *p, V v)
{
    if (AGENT) __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else *p = v;
}
template <bool AGENT, typename V> __device__ __forceinline__ V ob_bs_get(const V *p) { return AGENT ? __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : *p; }

template <int CTRL, int ROWS> __device__ __forceinline__ double ob_bs_dpp(double v)
{
    const ob_u32x2 u = __builtin_bit_cast(ob_u32x2, v);
    const ob_u32x2 o = {(uint32_t)__builtin_amdgcn_update_dpp(0, (int)u[0], CTRL, ROWS, 0xF, false), (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u[1], CTRL, ROWS, 0xF, false)};
    return __builtin_bit_cast(double, o);
}
// sums over 16 lanes, in every one of them, and over the wave, on the DPP network (as ob_wave_sum)
__device__ __forceinline__ double ob_bs_row_sum(double v)
{
    v += ob_bs_dpp<0xB1, 0xF>(v);
    v += ob_bs_dpp<0x4E, 0xF>(v);
    v += ob_bs_dpp<0x141, 0xF>(v);
    return v + ob_bs_dpp<0x140, 0xF>(v);
}
__device__ __forceinline__ double ob_bs_wave_sum(double v)
{
    v = ob_bs_row_sum(v);
    v += ob_bs_dpp<0x142, 0xA>(v);
    v += ob_bs_dpp<0x143, 0xC>(v);
    const ob_u32x2 u = __builtin_bit_cast(ob_u32x2, v);
    const ob_u32x2 t = {(uint32_t)__builtin_amdgcn_readlane((int)u[0], 63), (uint32_t)__builtin_amdgcn_readlane((int)u[1], 63)};
    return __builtin_bit_cast(double, t);
}
__device__ __forceinline__ float ob_bs_row_max(float v)
{
    v = fmaxf(v, OB_DPP_F(v, 0xB1, 0xF));
    v = fmaxf(v, OB_DPP_F(v, 0x4E, 0xF));
    v = fmaxf(v, OB_DPP_F(v, 0x141, 0xF));
    return fmaxf(v, OB_DPP_F(v, 0x140, 0xF));
}

// the k largest of the lanes' values (equal ones one by one; -inf where there are fewer), in order, to out
__device__ __forceinline__ void ob_bs_publish(float v, int k, float *out)
{
    const int lane = threadIdx.x & 63;
    for (int i = 0; i < k; ++i) {
        const float w = ob_wave_max(v);
        if (lane == 0) out[i] = w;
        if (w > -INFINITY && lane == __builtin_ctzll(__ballot(v == w))) v = -INFINITY;
    }
}
// thread i < n: the i-th of the n published values is the keep-th largest (equal ones in their order)?
__device__ __forceinline__ bool ob_bs_is_kth(const float *pub, int n, int keep, int i)
{
    if (i >= n) return false;
    const float v = pub[i];
    int rank = 0;
    for (int k = 0; k < n; ++k) rank += pub[k] > v || (pub[k] == v && k < i);
    return rank == keep - 1;
}

// candidate a in front of candidate b?  (value, beam, logit, token)
struct ObBsCand { double v; float x; int beam, tok; };
__device__ __forceinline__ bool ob_bs_before(const ObBsCand &a, const ObBsCand &b)
{
    if (a.v != b.v) return a.v > b.v;
    if (a.beam != b.beam) return a.beam < b.beam;
    return a.x != b.x ? a.x > b.x : a.tok < b.tok;
}

#define OB_BS_PLACES 8                                                            // candidate places of a thread of the pick that stay in registers

// THREADS: 256, where their registers hold all places of a group, or 1024
template <int THREADS, bool AGENT>
__device__ __forceinline__ void ob_bs_pick(const ObBsArgs &A, int group)
{
    constexpr int WAVES = THREADS / 64, NS = OB_BS_PLACES, RANKED = THREADS;       // candidates that are ranked by counting
    constexpr bool MORE = THREADS > 256;                                          // places beyond the registers
    __shared__ double row_v[OB_BS_MAX_BEAMS], cand_v[RANKED];                     // lse of a beam; NaN: it offers nothing
    __shared__ float pub[WAVES * (OB_BS_MAX_KEEP + 2)], t_s, row_s[OB_BS_MAX_BEAMS];
    __shared__ ObBsCand cand[RANKED];
    __shared__ int n_s, lists_s;
    __shared__ unsigned short live[MORE ? OB_BS_LISTS : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int room = ob_bs_list(A.keep), lists = A.beams * A.chunks, total = lists * room;
    // more places than registers, in many lists: a threshold from the lists' largest logits first, then the lists that reach it alone (32 rows of 128256, 64 kept: 84 ->
    // 42 us of both kernels)
    const bool by_lists = MORE && total > THREADS * NS && lists <= OB_BS_LISTS && lists >= 2 * A.keep;
    const int64_t list0 = (int64_t)group * A.beams * A.chunks;
    if (tid == 0) { n_s = 0; lists_s = 0; t_s = -INFINITY; }
    // place e of list l: its logit (NaN behind the list's end) and token
    const auto fetch = [&](int l, int e, float &x, int &tok) {                   // (all loads at once: what lies behind a list's end is memory of the list, not used)
        const int n = ob_bs_get<AGENT>(A.counts + list0 + l);
        x = ob_bs_get<AGENT>(A.list_x + (list0 + l) * room + e);
        tok = ob_bs_get<AGENT>(A.list_t + (list0 + l) * room + e);
        if (e >= n) x = NAN;
    };
    const auto beam_of = [&](int l) { return ob_bs_div(l, A.inv_chunks); };
    const auto value = [&](float x, int beam) { return (double)row_s[beam] + ((double)x - row_v[beam]); };        // (NaN: no candidate)
    float px[NS];
    int ptok[NS];
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        const int i = tid + THREADS * k, l = ob_bs_div(i, A.inv_room);
        px[k] = NAN; ptok[k] = 0;
        if (!by_lists && i < total) fetch(l, i - l * room, px[k], ptok[k]);
    }
    // a chunk's sum in terms of the row's largest logit
    const auto term = [](double m, double part, float M) { return m == -INFINITY ? part : part * exp(m - (double)M); };
    if (A.chunks <= 16)                                                          // a row of 16 lanes for a beam
        for (int b0 = 4 * wave; b0 < A.beams; b0 += 4 * WAVES) {
            const int b = b0 + (lane >> 4), c = lane & 15;
            const bool in = b < A.beams && c < A.chunks;
            const double *sm = A.sums + (list0 + (int64_t)min(b, A.beams - 1) * A.chunks + min(c, A.chunks - 1)) * 2;
            const double m = ob_bs_get<AGENT>(sm), part = ob_bs_get<AGENT>(sm + 1);
            const float M = ob_bs_row_max(in ? (float)m : -INFINITY);
            const double s = ob_bs_row_sum(in ? term(m, part, M) : 0.);
            if (b < A.beams && c == 0) { row_v[b] = (double)M + log(s); row_s[b] = A.scores[group * A.beams + b]; }
        }
    else
        for (int b = wave; b < A.beams; b += WAVES) {
            const double *sm = A.sums + (list0 + (int64_t)b * A.chunks) * 2;
            float M = -INFINITY;                                                 // (a logit)
            for (int c = lane; c < A.chunks; c += 64) M = fmaxf(M, (float)ob_bs_get<AGENT>(sm + 2 * c));
            M = ob_wave_max(M);
            double s = 0.;
            for (int c = lane; c < A.chunks; c += 64) s += term(ob_bs_get<AGENT>(sm + 2 * c), ob_bs_get<AGENT>(sm + 2 * c + 1), M);
            s = ob_bs_wave_sum(s);
            if (lane == 0) { row_v[b] = (double)M + log(s); row_s[b] = A.scores[group * A.beams + b]; }
        }
    __syncthreads();
    // their values, in registers; the other places' (where there are more) with every look at them
    double pv[NS];
#pragma unroll
    for (int k = 0; k < NS; ++k) pv[k] = value(px[k], min(beam_of(ob_bs_div(tid + THREADS * k, A.inv_room)), A.beams - 1));
    const auto others = [&](auto f) {
        if constexpr (MORE) for (int i = tid + (by_lists ? 0 : THREADS * NS); i < total; i += THREADS) {
            const int l = ob_bs_div(i, A.inv_room);
            ObBsCand c;
            fetch(l, i - l * room, c.x, c.tok);
            c.beam = beam_of(l);
            c.v = value(c.x, c.beam);
            if (c.v > -INFINITY) f(c);
        }
    };
    const auto keep_it = [&](const ObBsCand &c) {
        const int k = atomicAdd(&n_s, 1);
        if (k < RANKED) { cand_v[k] = c.v; cand[k] = c; }
    };
    float best = -INFINITY;
    if (MORE && by_lists) {
        constexpr int NL = OB_BS_LISTS / THREADS;
        float top[NL];
#pragma unroll
        for (int k = 0; k < NL; ++k) {
            const int l = min(tid + THREADS * k, lists - 1), beam = beam_of(l);
            const double v = (double)row_s[beam] + (ob_bs_get<AGENT>(A.sums + 2 * (list0 + l)) - row_v[beam]);
            top[k] = tid + THREADS * k < lists && v > -INFINITY ? __double2float_rd(v) : -INFINITY;
            best = fmaxf(best, top[k]);
        }
        const int waves = min(WAVES, (lists + 63) / 64), share = min(64, (A.keep + waves - 1) / waves + 2);
        if (wave < waves) ob_bs_publish(best, share, pub + wave * share);
        __syncthreads();
        if (ob_bs_is_kth(pub, waves * share, A.keep, tid)) t_s = pub[tid];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NL; ++k)
            if (top[k] >= t_s && top[k] > -INFINITY) live[atomicAdd(&lists_s, 1)] = (unsigned short)(tid + THREADS * k);
        __syncthreads();
        const double t = t_s;
        for (int i = tid; i < lists_s * room; i += THREADS) {
            const int at = ob_bs_div(i, A.inv_room);
            ObBsCand c;
            fetch(live[at], i - at * room, c.x, c.tok);
            c.beam = beam_of(live[at]);
            c.v = value(c.x, c.beam);
            if (c.v > -INFINITY && c.v >= t) keep_it(c);
        }
    } else {
        double most = -INFINITY;
#pragma unroll
        for (int k = 0; k < NS; ++k) most = fmax(most, pv[k]);
        others([&](const ObBsCand &c) { most = fmax(most, c.v); });
        best = __double2float_rd(most);                                          // (rounded down: what reaches the threshold reaches it in 64 bits, too)
        const int waves = min(WAVES, (total + 63) / 64), share = min(64, (A.keep + waves - 1) / waves + 2);
        if (wave < waves) ob_bs_publish(best, share, pub + wave * share);
        __syncthreads();
        if (ob_bs_is_kth(pub, waves * share, A.keep, tid)) t_s = pub[tid];
        __syncthreads();
        const double t = t_s;
        if (best >= t_s) {
            unsigned left = 0;
#pragma unroll
            for (int k = 0; k < NS; ++k) left |= pv[k] >= t && pv[k] > -INFINITY ? 1u << k : 0u;
            for (; left; left &= left - 1) {                                     // (few: one piece of code for all places)
                const int k = __builtin_ctz(left);
                ObBsCand c = {pv[0], px[0], beam_of(ob_bs_div(tid + THREADS * k, A.inv_room)), ptok[0]};
#pragma unroll
                for (int j = 1; j < NS; ++j)
                    if (k == j) { c.v = pv[j]; c.x = px[j]; c.tok = ptok[j]; }
                keep_it(c);
            }
            others([&](const ObBsCand &c) { if (c.v >= t) keep_it(c); });
        }
    }
    __syncthreads();
    int n = n_s;
    const int64_t out = (int64_t)group * A.keep;
    const auto put = [&](int k, const ObBsCand &c) { A.out_scores[out + k] = (float)c.v; A.out_beams[out + k] = c.beam; A.out_tokens[out + k] = c.tok; };
    if (n <= RANKED) {
        for (int i = tid; i < n; i += THREADS) {
            const ObBsCand c = cand[i];
            int rank = 0;
#pragma unroll 4
            for (int k = 0; k < n; ++k) {
                const double v = cand_v[k];
                rank += v > c.v;
                if (v == c.v && k != i) rank += ob_bs_before(cand[k], c);
            }
            if (rank < A.keep) put(rank, c);
        }
    } else {                                                                     // one after the other: the best behind the last one
        ObBsCand last = {INFINITY, INFINITY, -1, -1};
        for (n = 0; n < A.keep; ++n) {
            ObBsCand b = {-INFINITY, -INFINITY, 0x7fffffff, 0x7fffffff};
            const auto look = [&](const ObBsCand &c) { if (ob_bs_before(last, c) && ob_bs_before(c, b)) b = c; };
#pragma unroll
            for (int k = 0; k < NS; ++k)
                if (pv[k] > -INFINITY) look({pv[k], px[k], beam_of(ob_bs_div(tid + THREADS * k, A.inv_room)), ptok[k]});
            others(look);
            __syncthreads();
            cand[tid] = b;
            __syncthreads();
            for (int h = THREADS / 2; h; h >>= 1) {
                if (tid < h && ob_bs_before(cand[tid + h], cand[tid])) cand[tid] = cand[tid + h];
                __syncthreads();
            }
            last = cand[0];
            if (last.v == -INFINITY) break;
            if (tid == 0) put(n, last);
        }
    }
    if (tid >= n && tid < A.keep) put(tid, {-INFINITY, 0.f, -1, -1});
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void ob_bs_pick_kernel(const ObBsArgs A) { ob_bs_pick<THREADS, false>(A, blockIdx.x); }

// NV: pieces of 8 elements of a thread, OB_BS_THREADS apart.  PICK: the last workgroup of a group picks.
// 256 rows of 50257 fp16 11.5 us (2.2 TB/s; NV = 4 in 72 registers, so that the 1792 workgroups run in one round: in 85 two us more), 8 rows of 32000 with the pick 15.
// What a launch of few workgroups runs is fetched as it goes: code that few lanes need is there once, not for every element (8 rows of 32000 16.2, 4 rows of 512 11.1, with
// one for each).
template <typename T, int NV, bool PICK>
__global__ __launch_bounds__(OB_BS_THREADS, PICK ? 4 : NV == 1 ? 8 : 7) void ob_bs_scan_kernel(const ObBsArgs A)
{
    __shared__ float red_m[4], pub[4 * (OB_BS_MAX_KEEP + 2)], t_s;
    __shared__ double red_s[4];
    __shared__ int n_s, red_i[8];
    const int chunk = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T *x_row = (const T *)A.logits + (int64_t)row * A.ld;
    const int c0 = chunk * A.vecs * 8, c1 = min(A.vocab, c0 + A.vecs * 8);
    float x[NV][8];
    if (tid == 0) { n_s = 0; t_s = -INFINITY; }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int t0 = c0 + 8 * (tid + OB_BS_THREADS * j);
        if (t0 + 8 <= c1) {
            typedef T vec __attribute__((ext_vector_type(8)));
            struct __attribute__((packed, aligned(sizeof(T)))) U { vec v; };
            const vec v = reinterpret_cast<const U *>(x_row + t0)->v;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[j][e] = (float)v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[j][e] = t0 + e < c1 ? (float)x_row[t0 + e] : -INFINITY;
        }
    }
    float best = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) best = fmaxf(best, x[j][e]);
    const int n_thr = min((c1 - c0 + 7) / 8, OB_BS_THREADS), share = min(64, (A.keep * min(64, n_thr) + n_thr - 1) / n_thr + 2);     // (of a wave all of whose lanes have elements)
    const float wm = ob_wave_max(best);
    if (lane == 0) red_m[wave] = wm;
    ob_bs_publish(best, share, pub + wave * share);
    __syncthreads();
    if (ob_bs_is_kth(pub, 4 * share, A.keep, tid)) t_s = pub[tid];
    __syncthreads();
    const float m = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3])), t = t_s;
    const int room = ob_bs_list(A.keep);
    const int64_t list = (int64_t)row * A.chunks + chunk;
    float *lx = A.list_x + list * room;
    int *lt = A.list_t + list * room;
    const float least = fmaxf(t, -3.402823466e38f);                             // (-inf is no candidate)
    if (best >= least) {
        unsigned left = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) left |= x[j][e] >= least ? 1u << (8 * j + e) : 0u;
        for (; left; left &= left - 1) {                                         // (few: one piece of code for all elements, their logits read again)
            const int k = __builtin_ctz(left), tok = c0 + 8 * (tid + OB_BS_THREADS * (k >> 3)) + (k & 7), at = atomicAdd(&n_s, 1);
            if (at < room) { ob_bs_put<PICK>(lx + at, (float)x_row[tok]); ob_bs_put<PICK>(lt + at, tok); }
        }
    }
    double s = 0.;                                                              // (a NaN makes the row's sum NaN, +inf as well)
    if (m > -INFINITY) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) s += (double)__builtin_amdgcn_exp2f((x[j][e] - m) * 1.44269504f);
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) s += x[j][e] == -INFINITY ? 0. : (double)x[j][e];
    }
    s = ob_bs_wave_sum(s);
    if (lane == 0) red_s[wave] = s;
    __syncthreads();
    int n = n_s;
    if (n > room) {
        // too many reach the threshold: a search for one that `keep` reach and the list has room for, bit by bit (x as whole numbers of its order; NaN the lowest), and,
        // where that is one of too many equal logits, for the last index that is taken
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                         // (what is listed already is written over)
        int turn = 0;
        const auto count = [&](auto in) -> int {                                 // elements that `in` holds for, over the workgroup
            int c = 0;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) c += __popcll(__ballot(in(__float_as_uint(x[j][e]), 8 * (tid + OB_BS_THREADS * j) + e)));
            int *to = red_i + 4 * turn;
            turn ^= 1;
            if (lane == 0) to[wave] = c;
            __syncthreads();
            return (to[0] + to[1]) + (to[2] + to[3]);
        };
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t u = __float_as_uint(x[j][e] + 0.f);               // (-0 is 0)
                x[j][e] = __uint_as_float(x[j][e] != x[j][e] ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u);
            }
        uint32_t kth = 0;
        int reach = n;
        for (uint32_t bit = 0x80000000u; bit && reach > room; bit >>= 1) {
            const uint32_t k = kth | bit;
            const int c = count([&](uint32_t u, int) { return u >= k; });
            if (c >= A.keep) { kth = k; reach = c; }
        }
        int last = 8 * OB_BS_THREADS * NV;
        if (reach > room) {
            const int want = A.keep - count([&](uint32_t u, int) { return u > kth; });
            last = 0;
            for (int bit = 4 * OB_BS_THREADS * NV; bit; bit >>= 1)
                if (count([&](uint32_t u, int at) { return u == kth && at < (last | bit); }) < want) last |= bit;
        }
        if (tid == 0) n_s = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t u = __float_as_uint(x[j][e]);
                const int at0 = 8 * (tid + OB_BS_THREADS * j) + e;
                if (u > kth || (u == kth && at0 <= last)) {
                    const int at = atomicAdd(&n_s, 1);
                    if (at < room) { ob_bs_put<PICK>(lx + at, __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u)); ob_bs_put<PICK>(lt + at, c0 + at0); }
                }
            }
        __syncthreads();
        n = min(n_s, room);
    }
    if (tid == 0) {
        ob_bs_put<PICK>(A.sums + 2 * list, (double)m);
        ob_bs_put<PICK>(A.sums + 2 * list + 1, (red_s[0] + red_s[1]) + (red_s[2] + red_s[3]));
        ob_bs_put<PICK>(A.counts + list, n);
    }
    if constexpr (PICK) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                         // every wave: what it wrote has left
        __syncthreads();
        const int group = row / A.beams;
        if (tid == 0) {
            const int all = A.beams * A.chunks, last = __hip_atomic_fetch_add(A.tickets + group, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == all - 1;
            if (last) __hip_atomic_store(A.tickets + group, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            n_s = last;
        }
        __syncthreads();
        if (n_s) ob_bs_pick<OB_BS_THREADS, true>(A, group);
    }
}
