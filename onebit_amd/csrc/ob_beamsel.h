// The continuations that a beam search goes on with, gfx950.  Row r = (group r / beams, beam r % beams) holds the logits of one
// hypothesis; its continuation by token t is worth  v = score_r + (x_t - ln sum_u e^{x_u}),  and a group's `keep` best of beams x vocab
// continuations are wanted in the order (v descending, beam, x descending, token).  v is a sum in 64 bits: two beams' values often lie closer
// than fp32 resolves, while within a row the logits themselves order.
//   ob_bs_scan_kernel   (row, chunk of the vocabulary): max and sum e^{x - max} of the chunk, and each wave's `keep` best of it, in order
//   ob_bs_pick_kernel   (group): the rows' sums joined, then the best heads of the waves' lists, one after the other
// The logits are read once.  e^x: the product x log2 e is carried in two parts, so a term is off by 2^-23 at most however far x lies below the
// maximum; terms are added in fp32 over a thread's elements and in 64 bits from there on.  A row's elements belong to threads by their index
// alone, not by the row's alignment: equal rows have equal sums, bit for bit.
#pragma once
#include "ob_common.h"

#define OB_BS_THREADS 256
#define OB_BS_EPT 8                                // elements of a thread
#define OB_BS_CHUNK (OB_BS_THREADS * OB_BS_EPT)    // elements of a workgroup
#define OB_BS_MAX_KEEP 64

struct ObBsArgs {
    const void *logits;
    long long ld;                    // row pitch, elements
    const float *scores;             // [groups * beams]
    int beams, keep, vocab, chunks;
    double *sums;                    // [rows][chunks][2]  {max, sum}
    float *list_x;                   // [rows][4 chunks][keep]
    int *list_t;                     // token, or -1 behind the list's end
    float *out_scores; int *out_beams, *out_tokens;      // [groups][keep]
};

__device__ __forceinline__ float ob_bs_exp(float d)              // e^d, d <= 0
{
    d = d < -1000.f ? -1000.f : d;                               // (-inf has no two parts; NaN stays)
    const float hi = d * 1.44269502162933349609375f;             // log2 e = 1.44269502... + 1.925963033e-8
    const float lo = __builtin_fmaf(d, 1.44269502162933349609375f, -hi) + d * 1.925963033500011e-8f;
    return __builtin_amdgcn_exp2f(hi) * __builtin_fmaf(lo, 0.693147180559945f, 1.f);
}

__device__ __forceinline__ double ob_bs_wave_sum(double v)
{
#pragma unroll
    for (int k = 32; k; k >>= 1) v += __shfl_xor(v, k, 64);
    return v;
}

template <typename T>
__global__ __launch_bounds__(OB_BS_THREADS) void ob_bs_scan_kernel(const ObBsArgs A)
{
    __shared__ float red_m[4];
    __shared__ double red_s[4];
    const int chunk = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T *x_row = (const T *)A.logits + (int64_t)row * A.ld;
    const int t0 = chunk * OB_BS_CHUNK + tid * OB_BS_EPT;
    float x[OB_BS_EPT];
    if (t0 + OB_BS_EPT <= A.vocab) {
        typedef T vec __attribute__((ext_vector_type(OB_BS_EPT)));
        struct __attribute__((packed, aligned(sizeof(T)))) U { vec v; };
        const vec v = reinterpret_cast<const U *>(x_row + t0)->v;
#pragma unroll
        for (int e = 0; e < OB_BS_EPT; ++e) x[e] = (float)v[e];
    } else {
#pragma unroll
        for (int e = 0; e < OB_BS_EPT; ++e) x[e] = t0 + e < A.vocab ? (float)x_row[t0 + e] : -INFINITY;
    }
    float m = x[0];
#pragma unroll
    for (int e = 1; e < OB_BS_EPT; ++e) m = fmaxf(m, x[e]);
    m = ob_wave_max(m);
    if (lane == 0) red_m[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
    float s = 0.f;
    if (m != -INFINITY) {
#pragma unroll
        for (int e = 0; e < OB_BS_EPT; ++e) s += ob_bs_exp(x[e] - m);           // (a NaN logit makes the row's sum NaN, +inf as well)
    } else {
#pragma unroll
        for (int e = 0; e < OB_BS_EPT; ++e) s += x[e] == -INFINITY ? 0.f : x[e];
    }
    const double ds = ob_bs_wave_sum((double)s);
    if (lane == 0) red_s[wave] = ds;
    __syncthreads();
    if (tid == 0) {
        double *out = A.sums + ((int64_t)row * A.chunks + chunk) * 2;
        out[0] = (double)m;
        out[1] = (red_s[0] + red_s[1]) + (red_s[2] + red_s[3]);
    }
    // ---- the wave's best, one after the other: the largest of the lanes' largest, in the lowest lane that has it
    const int64_t list = ((int64_t)row * 4 * A.chunks + 4 * chunk + wave) * A.keep;
    float bx = -INFINITY;
    int be = 0;
    for (int e = OB_BS_EPT - 1; e >= 0; --e)
        if (x[e] >= bx) { bx = x[e]; be = e; }
    for (int k = 0; k < A.keep; ++k) {
        const float w = ob_wave_max(bx);
        const unsigned long long who = __ballot(bx == w);
        if (w == -INFINITY || !who) {                                            // nothing is left: the list ends here
            if (lane == 0) A.list_t[list + k] = -1;
            break;
        }
        const int first = __builtin_ctzll(who);
        if (lane == first) {
            A.list_x[list + k] = bx;
            A.list_t[list + k] = t0 + be;
#pragma unroll
            for (int e = 0; e < OB_BS_EPT; ++e)
                if (e == be) x[e] = -INFINITY;
            bx = -INFINITY;
#pragma unroll
            for (int e = OB_BS_EPT - 1; e >= 0; --e)
                if (x[e] >= bx) { bx = x[e]; be = e; }
        }
    }
}

// candidate a in front of candidate b?  (value, logit, list); lists of a beam come one after the other, in the order of their tokens
__device__ __forceinline__ bool ob_bs_before(double va, float xa, int la, double vb, float xb, int lb, int lists)
{
    if (va != vb) return va > vb;
    return xa != xb && la / lists == lb / lists ? xa > xb : la < lb;
}

__global__ __launch_bounds__(OB_BS_THREADS) void ob_bs_pick_kernel(const ObBsArgs A)
{
    __shared__ double row_v[32];                                                 // score - lse of a beam; NaN: it offers nothing
    __shared__ double best_v[4];
    __shared__ float best_x[4];
    __shared__ int best_l[4];
    const int group = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int lists = 4 * A.chunks, total = lists * A.beams;
    for (int b = wave; b < A.beams; b += 4) {
        const double *sm = A.sums + ((int64_t)(group * A.beams + b) * A.chunks) * 2;
        double M = -INFINITY, s = 0.;
        for (int c = lane; c < A.chunks; c += 64) M = fmax(M, sm[2 * c]);
#pragma unroll
        for (int k = 32; k; k >>= 1) M = fmax(M, __shfl_xor(M, k, 64));
        for (int c = lane; c < A.chunks; c += 64) s += sm[2 * c] == -INFINITY ? sm[2 * c + 1] : sm[2 * c + 1] * exp(sm[2 * c] - M);
        s = ob_bs_wave_sum(s);
        if (lane == 0) row_v[b] = M + log(s);
    }
    __syncthreads();
    // a thread's lists tid, tid + 256, ..: the best of their heads
    const auto value = [&](int l, int at, float &x) -> double {
        const int b = l / lists;
        const int64_t i = ((int64_t)group * total + l) * A.keep + at;
        if (at >= A.keep || A.list_t[i] < 0) return -INFINITY;
        x = A.list_x[i];
        const double v = (double)A.scores[group * A.beams + b] + ((double)x - row_v[b]);
        return v > -INFINITY ? v : -INFINITY;                                    // (NaN: no candidate)
    };
    extern __shared__ unsigned char at_s[];                                      // how many of a list are taken, [total]
    for (int l = tid; l < total; l += OB_BS_THREADS) at_s[l] = 0;
    double bv;
    float bx;
    int bl;
    const auto rescan = [&]() {
        bv = -INFINITY; bx = 0.f; bl = 0x7fffffff;
        for (int l = tid; l < total; l += OB_BS_THREADS) {
            float x = 0.f;
            const double v = value(l, at_s[l], x);
            if (v > -INFINITY && ob_bs_before(v, x, l, bv, bx, bl, lists)) { bv = v; bx = x; bl = l; }
        }
    };
    rescan();
    for (int k = 0; k < A.keep; ++k) {
        double v = bv;
        float x = bx;
        int l = bl;
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            const double v2 = __shfl_xor(v, o, 64);
            const float x2 = __shfl_xor(x, o, 64);
            const int l2 = __shfl_xor(l, o, 64);
            if (ob_bs_before(v2, x2, l2, v, x, l, lists)) { v = v2; x = x2; l = l2; }
        }
        if (lane == 0) { best_v[wave] = v; best_x[wave] = x; best_l[wave] = l; }
        __syncthreads();
        v = best_v[0]; x = best_x[0]; l = best_l[0];
#pragma unroll
        for (int w = 1; w < 4; ++w)
            if (ob_bs_before(best_v[w], best_x[w], best_l[w], v, x, l, lists)) { v = best_v[w]; x = best_x[w]; l = best_l[w]; }
        const int64_t out = (int64_t)group * A.keep + k;
        if (v == -INFINITY) {
            if (tid == 0) { A.out_scores[out] = -INFINITY; A.out_beams[out] = -1; A.out_tokens[out] = -1; }
        } else if (bl == l) {
            A.out_scores[out] = (float)v;
            A.out_beams[out] = l / lists;
            A.out_tokens[out] = A.list_t[((int64_t)group * total + l) * A.keep + at_s[l]];
            at_s[l] = (unsigned char)(at_s[l] + 1);
            rescan();
        }
        __syncthreads();
    }
}
