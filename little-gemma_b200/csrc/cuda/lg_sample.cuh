// lg_sample.cuh -- a token from a row of logits: temperature, top-k, top-p, min-p and a given random number.  Included by lg_serve.cu.
//
// What is kept is a beginning of the order (larger logits first, the lower index first among equals), so it is described by a
// threshold: every token with a larger logit, and the first `ties` tokens whose logit equals it; min_p is a property of the logit
// alone.  Weights enter as integers, w = round(exp((l - max) / T) 2^shift) with shift = 62 - ceil(log2 vocab): sums of them are
// exact, so where a running weight passes a target does not depend on how a sum is cut up.  Their error of 2^-(shift+1) of
// the largest weight is far below the step of a 32-bit random number.
#pragma once
#include "lg_device.cuh"
#include <cuda_bf16.h>

#define LG_SAMPLE_THREADS 1024

struct LgSampleArgs {
    const void *logits;
    long long ld;
    int vocab, shift;
    const float *temperature; const int *top_k; const float *top_p; const float *min_p; const float *u;
    int *token; float *prob;
};

// Logits as unsigned integers in the same order; NaN lowest, -0 equal to 0.
__device__ __forceinline__ uint32_t logit_key(float l) {
    if (l != l) return 0;
    const uint32_t b = l == 0.0f ? 0u : __float_as_uint(l);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }
#define LG_KEY_DEAD 0x007FFFFFu        // -inf; this and below is never drawn
#define LG_KEY_INF 0xFF800000u

struct LgWeight {                      // exp((l - top) / T) of a row
    double top, inv;                   // inv: log2(e) / T
    bool inf;                          // the largest logit is +inf: 1 for those, 0 for the others
    __device__ __forceinline__ double real(uint32_t key) const {
        if (inf) return key == LG_KEY_INF ? 1.0 : 0.0;
        if (key <= LG_KEY_DEAD) return 0.0;
        return exp2(((double)key_logit(key) - top) * inv);
    }
    __device__ __forceinline__ unsigned long long fixed(uint32_t key, int shift) const {
        return (unsigned long long)__double2ull_rn(real(key) * (double)(1ull << shift));
    }
};

__device__ __forceinline__ unsigned long long block_sum_u64(unsigned long long v, unsigned long long *red) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned long long t = red[threadIdx.x & 31];
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
}

template <typename T> __device__ __forceinline__ float logit_at(const T *p, int i);
template <> __device__ __forceinline__ float logit_at<float>(const float *p, int i) { return p[i]; }
template <> __device__ __forceinline__ float logit_at<__half>(const __half *p, int i) { return __half2float(p[i]); }
template <> __device__ __forceinline__ float logit_at<__nv_bfloat16>(const __nv_bfloat16 *p, int i) { return __bfloat162float(p[i]); }

// One CTA per row.  Thresholds by bisection on the key: the largest key t for which what lies at t and above reaches the target.
template <typename T> __global__ void __launch_bounds__(LG_SAMPLE_THREADS) lg_sample_kernel(LgSampleArgs a) {
    __shared__ unsigned long long red[32];
    const int row = blockIdx.x, tid = threadIdx.x, V = a.vocab;
    const T *x = (const T *)a.logits + (long long)row * a.ld;
    // largest logit and its first place
    unsigned long long top = 0;
    for (int i = tid; i < V; i += LG_SAMPLE_THREADS) {
        const unsigned long long k = (unsigned long long)logit_key(logit_at(x, i)) << 32 | (uint32_t)~i;
        top = k > top ? k : top;
    }
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) { const unsigned long long t = __shfl_xor_sync(0xffffffffu, top, o); top = t > top ? t : top; }
    if ((tid & 31) == 0) red[tid >> 5] = top;
    __syncthreads();
    top = red[tid & 31];
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) { const unsigned long long t = __shfl_xor_sync(0xffffffffu, top, o); top = t > top ? t : top; }
    const uint32_t top_key = (uint32_t)(top >> 32);
    const float T1 = a.temperature ? a.temperature[row] : 1.0f, top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f;
    const int top_k = a.top_k ? a.top_k[row] : 0;
    if (top_key <= LG_KEY_DEAD || !(T1 > 0.0f) || top_k == 1 || top_p <= 0.0f || min_p > 1.0f) {
        if (tid == 0) {
            const bool none = top_key <= LG_KEY_DEAD;
            a.token[row] = none ? -1 : (int)~(uint32_t)top;
            if (a.prob) a.prob[row] = none ? 0.0f : 1.0f;
        }
        return;
    }
    LgWeight w;
    w.top = (double)key_logit(top_key); w.inv = 1.4426950408889634 / (double)T1; w.inf = top_key == LG_KEY_INF;
    uint32_t t = LG_KEY_DEAD + 1;                       // threshold; below: nothing
    unsigned long long ties = ~0ull;                    // tokens kept at the threshold
    if (top_k > 0 && top_k < V) {
        uint32_t lo = LG_KEY_DEAD, hi = top_key;        // the count at lo and above is top_k or more, or nothing below counts
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            unsigned long long n = 0;
            for (int i = tid; i < V; i += LG_SAMPLE_THREADS) n += logit_key(logit_at(x, i)) >= mid;
            if (block_sum_u64(n, red) >= (unsigned long long)top_k) lo = mid; else hi = mid - 1;
        }
        if (lo > LG_KEY_DEAD) {
            unsigned long long n = 0;
            for (int i = tid; i < V; i += LG_SAMPLE_THREADS) n += logit_key(logit_at(x, i)) > lo;
            t = lo;
            ties = (unsigned long long)top_k - block_sum_u64(n, red);
        }
    }
    if (top_p < 1.0f) {
        // weight above a key, the threshold's share limited to its kept ties
        auto above = [&](uint32_t key) {                // of keys >= key, key > t
            unsigned long long s = 0;
            for (int i = tid; i < V; i += LG_SAMPLE_THREADS) { const uint32_t k = logit_key(logit_at(x, i)); if (k >= key) s += w.fixed(k, a.shift); }
            return block_sum_u64(s, red);
        };
        unsigned long long n_at = 0;
        for (int i = tid; i < V; i += LG_SAMPLE_THREADS) n_at += logit_key(logit_at(x, i)) == t;
        n_at = block_sum_u64(n_at, red);
        if (ties < n_at) n_at = ties;
        const unsigned long long total = above(t + 1) + n_at * w.fixed(t, a.shift);
        const unsigned long long p64 = __double2ull_rz((double)top_p * 18446744073709551616.0);
        unsigned long long target = __umul64hi(p64, total) + (p64 * total != 0);
        if (target < 1) target = 1;
        uint32_t lo = t, hi = top_key;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            if (above(mid) >= target) lo = mid; else hi = mid - 1;
        }
        const unsigned long long before = lo == 0xFFFFFFFFu ? 0 : above(lo + 1), one = w.fixed(lo, a.shift);
        const unsigned long long c = one ? (target - before + one - 1) / one : 1;
        ties = lo == t && ties < c ? ties : c;
        t = lo;
    }
    // the draw: every warp has a piece of the row; first what each piece keeps, then the piece in which the running weight passes the target
    __shared__ unsigned long long part[32], tie0[32];
    const int lane = tid & 31, warp = tid >> 5, per = ((V + 31) / 32 + 31) & ~31, i0 = warp * per, i1 = min(V, i0 + per);
    const unsigned long long at_t = w.fixed(t, a.shift) * (w.real(t) >= (double)min_p || !(min_p > 0.0f));
    unsigned long long s = 0, n = 0;
    for (int i = i0 + lane; i < i1; i += 32) {
        const uint32_t k = logit_key(logit_at(x, i));
        if (k > t) { const double e = w.real(k); if (!(min_p > 0.0f) || e >= (double)min_p) s += (unsigned long long)__double2ull_rn(e * (double)(1ull << a.shift)); }
        n += k == t;
    }
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, o); n += __shfl_xor_sync(0xffffffffu, n, o); }
    __syncthreads();
    if (lane == 0) { part[warp] = s; tie0[warp] = n; }
    __syncthreads();
    unsigned long long total = 0, seen = 0, mine = 0, mine_ties = 0;
    for (int j = 0; j < 32; j++) {
        const unsigned long long left = ties > seen ? ties - seen : 0, c = tie0[j] < left ? tie0[j] : left;
        if (j == warp) { mine = total; mine_ties = seen; }
        total += part[j] + c * at_t;
        seen += tie0[j];
        if (j == warp) s = total;
    }
    const float u = a.u[row];
    const unsigned long long u64 = u > 0.0f ? u < 1.0f ? __double2ull_rz((double)u * 18446744073709551616.0) : ~0ull : 0ull;
    const unsigned long long target = __umul64hi(u64, total);
    if (mine <= target && target < s) {                 // one warp: the running weight passes the target in its piece
        unsigned long long run = mine, rank = mine_ties;
        for (int i = i0; i < i1; i += 32) {
            const uint32_t k = i + lane < i1 ? logit_key(logit_at(x, i + lane)) : 0;
            const uint32_t eq = __ballot_sync(0xffffffffu, k == t && i + lane < i1);
            unsigned long long v = 0;
            if (k > t) { const double e = w.real(k); if (!(min_p > 0.0f) || e >= (double)min_p) v = (unsigned long long)__double2ull_rn(e * (double)(1ull << a.shift)); }
            else if (k == t && i + lane < i1 && rank + __popc(eq & ((1u << lane) - 1)) < ties) v = at_t;
            rank += __popc(eq);
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const unsigned long long z = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += z; }
            const uint32_t hit = __ballot_sync(0xffffffffu, run + v > target);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    a.token[row] = i + lane;
                    if (a.prob) a.prob[row] = (float)(w.real(k) / ((double)total / (double)(1ull << a.shift)));
                }
                break;
            }
            run += __shfl_sync(0xffffffffu, v, 31);
        }
    }
}
