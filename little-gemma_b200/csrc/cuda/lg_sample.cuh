// lg_sample.cuh -- a token from a row of logits: temperature, top-k, top-p, min-p and a given random number.  Included by lg_serve.cu.
//
// What is kept is a beginning of the order (larger logits first, the lower index first among equals), so it is described by a
// threshold: every token with a larger logit, and the first `ties` tokens whose logit equals it; min_p is a property of the logit
// alone.  Weights enter as integers, w = round(exp((l - max) / T) 2^shift) with shift = 44 (42 for the largest vocabularies): sums of them are
// exact, so where a running weight passes a target does not depend on how a sum is cut up.  Their error of 2^-(shift+1) of
// the largest weight is far below the step of a 32-bit random number.
//
// A cluster of CTAs holds a row in shared memory after one read of HBM (the part that does not fit is read again from L2); what all
// CTAs have to know -- the maximum, histograms, sums -- goes through distributed shared memory with one cluster barrier each, and every CTA draws the same
// conclusions from it.  A threshold is found without sorting:
//   coarse  bins of 1/32 of a power of two of the weight (2048: beyond, a weight is 0); the tokens' number, or their weights to a part in 2000, added up per
//           bin, tell the bin (two where it is close) that the threshold lies in, and with it an interval of logits
//   list    each warp notes its tokens in that interval (top-k: and above, later passes then read the list instead of the row)
//   fine    exact counts or weights over 1024 equal parts of that interval of keys (the logits as ordered integers), then of the part that holds the threshold,
//           until a part is a single key: at most four rounds.  Where the lists hold the interval, every CTA fetches its tokens and does the rounds alone;
//           otherwise (flat rows) the histograms of a round are added up over the cluster
// Not at a limit of the device: 61 warp instructions per 32 tokens with temperature alone (29 of them a weight, 14 in 64 bits) and 170 with top-p and min-p fill
// 57 and 43 % of the issue slots of two CTAs an SM (64 registers allow no third); the rest is waiting, for block and cluster barriers, results and the 64-bit
// pipe, and a second round of CTAs where there are more than 296.  Few rows: cluster barriers, and code that is fetched for the first time.  One row of
// 262144 with top-k and top-p 30 us, 48 rows with top-p and min-p 137 us, 512 rows of 32768 without filters 49 us.
#pragma once
#include "lg_device.cuh"
#include <cuda_bf16.h>

#define LG_SAMPLE_THREADS 512
#define LG_SAMPLE_WARPS (LG_SAMPLE_THREADS / 32)
#define LG_SAMPLE_COARSE 2048          // bins, four a thread
#define LG_SAMPLE_BINS 1024            // parts of an interval
#define LG_SAMPLE_LIST 224             // tokens a warp's list holds
#define LG_SAMPLE_NEAR 2816            // of these, tokens of a CTA whose place at a threshold is open
#define LG_SAMPLE_HIST (3 * LG_SAMPLE_BINS)    // words of a histogram: the coarse bins, or three arrays of the parts
#define LG_SAMPLE_TOOLS (2 * LG_SAMPLE_HIST * 4 + LG_SAMPLE_COARSE * 8 + LG_SAMPLE_WARPS * LG_SAMPLE_LIST * 8 + LG_SAMPLE_NEAR * 4)
#define LG_SAMPLE_MAX_CLUSTER 8

typedef unsigned long long u64;

struct LgSampleArgs {
    const void *logits;
    long long ld;
    int rows, vocab, shift;
    int slice, cap;                    // tokens per CTA of a cluster; of these, tokens held in shared memory
    const float *temperature; const int *top_k; const float *top_p; const float *min_p; const float *u;
    int *token; float *prob;
};

// A logit as its f32 value, four at a time, and the larger of two words of logits (NaN loses); LOW: bits that are the same in every f32 that the
// type holds.
template <typename T> struct LogitType;
template <> struct LogitType<float> {
    static constexpr int LOW = 0;
    static __device__ __forceinline__ float value(const float *p) { return *p; }
    static __device__ __forceinline__ void value4(const float *p, float (&l)[4]) {
        const float4 v = *(const float4 *)p;
        l[0] = v.x; l[1] = v.y; l[2] = v.z; l[3] = v.w;
    }
    static __device__ __forceinline__ uint32_t lowest() { return 0xFF800000u; }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ float most(uint32_t a) { return __uint_as_float(a); }
};
template <> struct LogitType<__half> {
    static constexpr int LOW = 13;
    static __device__ __forceinline__ float value(const __half *p) { return __half2float(*p); }
    static __device__ __forceinline__ void value4(const __half *p, float (&l)[4]) {
        const uint2 v = *(const uint2 *)p;
        const float2 f = __half22float2(*(const __half2 *)&v.x), h = __half22float2(*(const __half2 *)&v.y);
        l[0] = f.x; l[1] = f.y; l[2] = h.x; l[3] = h.y;
    }
    static __device__ __forceinline__ uint32_t lowest() { return 0xFC00FC00u; }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { const __half2 m = __hmax2(*(const __half2 *)&a, *(const __half2 *)&b); return *(const uint32_t *)&m; }
    static __device__ __forceinline__ float most(uint32_t a) { const float2 f = __half22float2(*(const __half2 *)&a); return fmaxf(f.x, f.y); }
};
template <> struct LogitType<__nv_bfloat16> {
    static constexpr int LOW = 16;
    static __device__ __forceinline__ float value(const __nv_bfloat16 *p) { return __uint_as_float((uint32_t)*(const uint16_t *)p << 16); }
    static __device__ __forceinline__ void value4(const __nv_bfloat16 *p, float (&l)[4]) {
        const uint2 v = *(const uint2 *)p;
        l[0] = __uint_as_float(v.x << 16); l[1] = __uint_as_float(v.x & 0xFFFF0000u);
        l[2] = __uint_as_float(v.y << 16); l[3] = __uint_as_float(v.y & 0xFFFF0000u);
    }
    static __device__ __forceinline__ uint32_t lowest() { return 0xFF80FF80u; }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { const __nv_bfloat162 m = __hmax2(*(const __nv_bfloat162 *)&a, *(const __nv_bfloat162 *)&b); return *(const uint32_t *)&m; }
    static __device__ __forceinline__ float most(uint32_t a) { return fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u)); }
};
// Logits as unsigned integers in their order (-0 is 0; no NaN), without the bits that are always the same
template <int LOW> __device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = l == 0.0f ? 0u : __float_as_uint(l);
    return (b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u)) >> LOW;
}
template <int LOW> __device__ __forceinline__ float key_value(uint32_t k) {
    const uint32_t full = k << LOW;
    return __uint_as_float((full >> 31) ? full ^ 0x80000000u : ~(full | ((1u << LOW) - 1)));
}

// exp((l - top) / T) of a row
#define LG_TWO52 4503599627370496.0
#define LG_MAGIC 6755399441055744.0    // 1.5 2^52: adding it rounds to a whole number, which the low word then holds
struct LgWeight {
    double top, inv32, root;           // inv32: 32 log2(e) / T; root: 2^(shift - lane / 32).  Where the largest logit is +inf: f32's largest number and 0
    // y = 32 log2(e) (top - l) / T rounded, and behind it what rounding left over; false: the weight is 0
    __device__ __forceinline__ bool bin(float l, int &k, double &rest) const {
        const double d = top - (double)fminf(l, 3.402823466e38f);
        const double t = fma(d, inv32, LG_MAGIC);
        rest = fma(d, inv32, -(t - LG_MAGIC));
        k = __double2loint(t);
        return __double2hiint(t) == 0x43380000 && (uint32_t)k < LG_SAMPLE_COARSE;
    }
    // 2^(shift - (k + rest) / 32), all lanes of a warp together: the power of the whole number from a lane's root times a polynomial (Taylor in
    // rest ln 2 / 32, at most ln 2 / 64: the first term left out is below 2^-48)
    __device__ __forceinline__ double scaled(int k, double rest) const {
        double p;
        return scaled(k, rest, p);
    }
    __device__ __forceinline__ double scaled(int k, double rest, double &p) const {       // p: of that, 2^(-rest / 32)
        const double c = 0.02166084939249829;                                 // ln 2 / 32
        p = fma(rest, -c * c * c * c * c / 120.0, c * c * c * c / 24.0);
        p = fma(p, rest, -c * c * c / 6.0);
        p = fma(p, rest, c * c / 2.0);
        p = fma(p, rest, -c);
        p = fma(p, rest, 1.0);
        const int hi = __shfl_sync(0xffffffffu, __double2hiint(root), k), lo = __shfl_sync(0xffffffffu, __double2loint(root), k);
        return __dmul_rn(p, __hiloint2double(hi - (k & ~31) * 32768, lo));    // (never joined with an addition: a weight is the same wherever it is computed)
    }
    static __device__ __forceinline__ double whole(double s) { return __dadd_rn(__dadd_rn(s, LG_TWO52), -LG_TWO52); }    // to the nearest integer; s < 2^51
    // of one logit, the same in all lanes: 0 where it has no weight
    __device__ __forceinline__ double of(float l) const {
        int k;
        double rest;
        const bool live = bin(l, k, rest) && l > -INFINITY;
        const double x = scaled(k, rest);
        return live ? x : 0.0;
    }
};

__device__ __forceinline__ u64 ld_peer_u64(const u64 *p, uint32_t rank) {
    uint32_t ra; u64 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(ra) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t ld_peer_u32(const uint32_t *p, uint32_t rank) {
    uint32_t ra, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(ra) : "memory");
    return v;
}
__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_half_sum_u64(u64 v) {
    #pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Inclusive sum over the lanes
__device__ __forceinline__ u64 warp_scan_u64(u64 v, int lane) {
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const u64 t = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += t; }
    return v;
}

template <typename T> struct LgSampler {
    typedef LogitType<T> L;
    static constexpr int LOW = L::LOW;
    static constexpr uint32_t DEAD = 0x007FFFFFu >> LOW;                      // -inf; this key and below are never drawn

    const LgSampleArgs &a;
    const T *g;                        // the slice in global memory
    T *data;                           // and in shared memory: cap tokens, the last ones filled up with NaN
    uint32_t *hist;                    // two histograms of `limbs` arrays, used in turn
    float *lv; int *li;                // this warp's list: logits, places in the slice; -inf behind the last
    u64 *fine; uint32_t *near;         // histogram of this CTA alone; keys of its tokens in an interval
    u64 *word;                         // words for the other CTAs: a place per exchange
    u64 *red;                          // block-wide
    int n, first, ranks, rank, lane, warp, turn = 0, at_word = 0;             // tokens here, index of the first
    int w0, w1;                        // this warp's tokens: places in the slice, or 0 .. of its list
    bool listed = false;
    LgWeight w;

    // four tokens a lane from place i on
    __device__ __forceinline__ void fetch4(int i, float (&l)[4]) const {
        if (listed) {
            float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (i < LG_SAMPLE_LIST) v = *(const float4 *)(lv + i);
            l[0] = v.x; l[1] = v.y; l[2] = v.z; l[3] = v.w;
        }
        else if (i + 4 <= a.cap) L::value4(data + i, l);
        else {
            #pragma unroll
            for (int j = 0; j < 4; j++) l[j] = i + j < n ? i + j < a.cap ? L::value(data + i + j) : L::value(g + i + j) : -INFINITY;
        }
    }
    // Four tokens' bins and weights side by side; in: above lt and with a weight
    __device__ __forceinline__ void weigh4(const float (&l)[4], float lt, int (&k)[4], double (&x)[4], bool (&in)[4]) const {
        double p[4];
        weigh4(l, lt, k, x, in, p);
    }
    __device__ __forceinline__ void weigh4(const float (&l)[4], float lt, int (&k)[4], double (&x)[4], bool (&in)[4], double (&p)[4]) const {
        double rest[4];
        #pragma unroll
        for (int j = 0; j < 4; j++) in[j] = w.bin(l[j], k[j], rest[j]) && l[j] > lt;
        #pragma unroll
        for (int j = 0; j < 4; j++) x[j] = w.scaled(k[j], rest[j], p[j]);
    }
    // This warp's tokens of at least `least` into its list, in their order, where they fit
    __device__ void make_list(float least) {
        if (listed) return;
        int count = 0;
        for (int i = w0; i < w1; i += 128) {
            float l[4];
            fetch4(i + lane * 4, l);
            const bool in[4] = {l[0] >= least, l[1] >= least, l[2] >= least, l[3] >= least};
            if (!__any_sync(0xffffffffu, in[0] || in[1] || in[2] || in[3])) continue;
            int at = count;
            #pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t m = __ballot_sync(0xffffffffu, in[j]);
                at += __popc(m & ((1u << lane) - 1));
                count += __popc(m);
            }
            if (count > LG_SAMPLE_LIST) return;
            #pragma unroll
            for (int j = 0; j < 4; j++) if (in[j]) { lv[at] = l[j]; li[at++] = i + lane * 4 + j; }
        }
        for (int i = count + lane; i < LG_SAMPLE_LIST; i += 32) lv[i] = -INFINITY;
        __syncwarp();
        listed = true; w0 = 0; w1 = count;
    }
    // Sums of two numbers a thread over the cluster; `at` (or NULL): the place of the CTAs' own sums
    __device__ void sum2(u64 x, u64 y, u64 &sx, u64 &sy, const u64 **at = nullptr) {
        x = warp_sum_u64(x); y = warp_sum_u64(y);
        __syncthreads();
        if (lane == 0) { red[warp] = x; red[LG_SAMPLE_WARPS + warp] = y; }
        __syncthreads();
        u64 *p = word + at_word;
        at_word += 2;
        if (warp == 0) {
            const u64 v = warp_half_sum_u64(red[lane]);                       // 16 warps: x in the lower half of the lanes, y in the upper
            if ((lane & 15) == 0) p[lane >> 4] = v;
        }
        cluster_sync_all();
        const u64 v = warp_half_sum_u64((lane & 15) < ranks ? ld_peer_u64(p + (lane >> 4), lane & 15) : 0);
        sx = __shfl_sync(0xffffffffu, v, 0); sy = __shfl_sync(0xffffffffu, v, 16);
        if (at) *at = p;
    }
    // An empty histogram (block-wide; the cluster has passed a barrier since the one before it was read)
    __device__ uint32_t *fresh_hist(int words) {
        uint32_t *h = hist + turn * LG_SAMPLE_HIST;
        turn ^= 1;
        for (int i = threadIdx.x; i < words; i += LG_SAMPLE_THREADS) h[i] = 0;
        __syncthreads();
        return h;
    }
    static __device__ __forceinline__ void add_weight(uint32_t *h, int bin, u64 x) {      // 15 bits per array: 2^17 tokens fit 32 bits
        if (const uint32_t v = (uint32_t)x & 0x7FFFu) atomicAdd(h + bin, v);
        if (const uint32_t v = (uint32_t)(x >> 15) & 0x7FFFu) atomicAdd(h + LG_SAMPLE_BINS + bin, v);
        if (const uint32_t v = (uint32_t)(x >> 30)) atomicAdd(h + 2 * LG_SAMPLE_BINS + bin, v);
    }
    // The first bin at which before + the running sum of v reaches the target, and the sum before it; the last bin where none does (found = false).
    template <int N> __device__ bool first_reaching(const u64 (&v)[N], u64 before, u64 target, int &bin, u64 &sum) {
        u64 mine = 0;
        #pragma unroll
        for (int j = 0; j < N; j++) mine += v[j];
        const u64 incl = warp_scan_u64(mine, lane);
        __syncthreads();
        if (lane == 31) red[warp] = incl;
        if (threadIdx.x == 0) red[2 * LG_SAMPLE_WARPS] = ~0ull;
        __syncthreads();
        const u64 ws = lane < LG_SAMPLE_WARPS ? red[lane] : 0, wi = warp_scan_u64(ws, lane);
        u64 at = before + incl - mine + __shfl_sync(0xffffffffu, wi - ws, warp);
        const u64 all = before + __shfl_sync(0xffffffffu, wi, 31);
        if (at < target && target <= at + mine) {
            int k = 0;
            #pragma unroll
            for (int j = 0; j < N - 1; j++) if (k == j && at + v[j] < target) { at += v[j]; k++; }
            red[2 * LG_SAMPLE_WARPS] = threadIdx.x * N + k;
            red[2 * LG_SAMPLE_WARPS + 1] = at;
        }
        __syncthreads();
        const u64 b = red[2 * LG_SAMPLE_WARPS];
        const bool found = b != ~0ull;
        bin = found ? (int)b : N * LG_SAMPLE_THREADS - 1;
        sum = found ? red[2 * LG_SAMPLE_WARPS + 1] : all;
        return found;
    }
    // The bins at which the running sums of `up` and of `low` (smaller ones) first reach the target, four bins a thread
    __device__ void bracket(const u64 (&up)[4], const u64 (&low)[4], u64 target, int &b0, int &b1) {
        const u64 mine[2] = {up[0] + up[1] + up[2] + up[3], low[0] + low[1] + low[2] + low[3]}, incl[2] = {warp_scan_u64(mine[0], lane), warp_scan_u64(mine[1], lane)};
        __syncthreads();
        if (lane == 31) { red[warp] = incl[0]; red[LG_SAMPLE_WARPS + warp] = incl[1]; }
        if (threadIdx.x < 2) red[2 * LG_SAMPLE_WARPS + threadIdx.x] = LG_SAMPLE_COARSE - 1;
        __syncthreads();
        #pragma unroll
        for (int h = 0; h < 2; h++) {
            const u64 ws = lane < LG_SAMPLE_WARPS ? red[h * LG_SAMPLE_WARPS + lane] : 0, wi = warp_scan_u64(ws, lane);
            u64 at = incl[h] - mine[h] + __shfl_sync(0xffffffffu, wi - ws, warp);
            if (at < target && target <= at + mine[h]) {
                int k = 0;
                #pragma unroll
                for (int j = 0; j < 3; j++) { const u64 v = h ? low[j] : up[j]; if (k == j && at + v < target) { at += v; k++; } }
                red[2 * LG_SAMPLE_WARPS + h] = threadIdx.x * 4 + k;
            }
        }
        __syncthreads();
        b0 = (int)red[2 * LG_SAMPLE_WARPS]; b1 = (int)red[2 * LG_SAMPLE_WARPS + 1];
    }
    // Keys of the coarse bins b0 .. b1 with room on either side, within low .. top_key
    __device__ void interval(int b0, int b1, uint32_t low, uint32_t top_key, uint32_t &klo, uint32_t &khi) const {
        klo = low; khi = top_key;
        if (!(w.inv32 > 0.0)) return;
        klo = max(low, key_of<LOW>(__double2float_rd(w.top - (b1 + 0.51) / w.inv32)));
        khi = min(top_key, key_of<LOW>(__double2float_ru(w.top - (b0 - 0.51) / w.inv32)));
    }
    // What one token adds: its weight, or 1
    __device__ __forceinline__ u64 mass(bool weighted, float l) const {
        int k;
        double rest;
        const bool live = w.bin(l, k, rest);
        const double x = LgWeight::whole(w.scaled(k, rest));
        return !weighted ? 1 : live ? (u64)(long long)x : 0;
    }
    // Part of the interval at which the target is reached, and the interval narrowed to it; `above`: of what lies above it
    static __device__ __forceinline__ void narrow(int part, int sh, uint32_t &klo, uint32_t &khi) {
        khi -= (uint32_t)part << sh;
        const uint32_t low = khi - ((1u << sh) - 1);
        klo = max(klo, low > khi ? 0u : low);
    }
    static __device__ __forceinline__ int shift_of(uint32_t range) { return range >= LG_SAMPLE_BINS ? 22 - __clz(range) : 0; }    // range >> shift < 1024
    // This CTA's share of the bins of a histogram, summed over the cluster and left for the others: adding up all bins in every CTA would
    // move ranks^2 histograms through the cluster
    __device__ void share_bins(const uint32_t *h, int bins, int limbs) {
        const int per = (bins + ranks - 1) / ranks;
        for (int b = threadIdx.x; b < per && rank * per + b < bins; b += LG_SAMPLE_THREADS) {
            u64 v = 0;
            for (int l = 0; l < limbs; l++) {
                #pragma unroll
                for (int c = 0; c < LG_SAMPLE_MAX_CLUSTER; c++) if (c < ranks) v += (u64)ld_peer_u32(h + l * bins + rank * per + b, c) << 15 * l;
            }
            fine[b] = v;
        }
        cluster_sync_all();
    }
    template <int N> __device__ __forceinline__ void shared_bins(u64 (&v)[N]) const {     // N a thread
        const int per = (N * LG_SAMPLE_THREADS + ranks - 1) / ranks;
        #pragma unroll
        for (int j = 0; j < N; j++) { const int b = threadIdx.x * N + j, c = b / per; v[j] = ld_peer_u64(fine + b - c * per, c); }
    }
    // The keys of a row's tokens from some threshold up, where every CTA has them (refine leaves them here): the histograms' place
    __device__ __forceinline__ uint32_t *pool() const { return hist; }
    // Rounds over tokens that this CTA has, eight a thread (x: what each counts): klo .. khi narrowed to the key at which the target is reached, `above`
    // brought to what lies above it
    __device__ void settle(const uint32_t (&key)[8], const u64 (&x)[8], u64 &above, u64 target, uint32_t &klo, uint32_t &khi) {
        for (int round = 0; round < 4; round++) {                             // 10 bits of at most 32 a round
            const int sh = shift_of(khi - klo);
            fine[2 * threadIdx.x] = fine[2 * threadIdx.x + 1] = 0;
            __syncthreads();
            #pragma unroll
            for (int q = 0; q < 8; q++) if (x[q] && key[q] >= klo && key[q] <= khi) atomicAdd(fine + ((khi - key[q]) >> sh), x[q]);
            __syncthreads();
            const u64 v[2] = {fine[2 * threadIdx.x], fine[2 * threadIdx.x + 1]};
            int part;
            first_reaching(v, above, target, part, above);
            narrow(part, sh, klo, khi);
            if (sh == 0) break;
        }
    }
    // Sums of two numbers a thread over this CTA
    __device__ void own_sum2(u64 x, u64 y, u64 &sx, u64 &sy) {
        x = warp_sum_u64(x); y = warp_sum_u64(y);
        __syncthreads();
        if (lane == 0) { red[warp] = x; red[LG_SAMPLE_WARPS + warp] = y; }
        __syncthreads();
        const u64 v = warp_half_sum_u64(red[lane]);
        sx = __shfl_sync(0xffffffffu, v, 0); sy = __shfl_sync(0xffffffffu, v, 16);
    }
    // The threshold at which counts (weighted: weights) of the keys from the largest down reach the target; it lies in klo .. khi.  Kept then: keys
    // above t and `ties` of key t.  Passes that read the row itself note its tokens in the interval in the warp's list: over_w is then this lane's part
    // of the warp's weight above the list's tokens and n_list their number; n_list < 0: there is no such list.  n_pool (or NULL): receives the number
    // of keys left in pool(), where every CTA has fetched all of the interval's.
    __device__ void refine(bool weighted, u64 target, uint32_t klo, uint32_t khi, uint32_t &t, u64 &ties, u64 &over_w, int &n_list, int *n_pool) {
        uint32_t *n_near = (uint32_t *)(red + 2 * LG_SAMPLE_WARPS + 4);
        u64 above, found;
        for (int wide = 0;; wide++) {
            // what lies above the interval, and the tokens in it
            __syncthreads();
            if (threadIdx.x == 0) *n_near = 0;
            __syncthreads();
            const float lo = key_value<LOW>(klo), hi = key_value<LOW>(khi);
            int open = 0;
            bool full = false;
            double over = 0.0;
            found = 0;
            for (int i = w0; i < w1; i += 128) {
                float l[4];
                fetch4(i + lane * 4, l);
                const bool any = l[0] >= lo || l[1] >= lo || l[2] >= lo || l[3] >= lo;
                if (!__any_sync(0xffffffffu, any)) continue;
                if (weighted) {
                    int k[4];
                    double x[4];
                    bool in[4];
                    weigh4(l, hi, k, x, in);
                    #pragma unroll
                    for (int j = 0; j < 4; j++) if (in[j]) over += LgWeight::whole(x[j]);
                } else found += (u64)((l[0] > hi) + (l[1] > hi) + (l[2] > hi) + (l[3] > hi)) << 32;
                uint32_t m[4], all = 0;
                #pragma unroll
                for (int j = 0; j < 4; j++) { m[j] = __ballot_sync(0xffffffffu, l[j] >= lo && l[j] <= hi); all |= m[j]; }
                if (!all) continue;
                int at = open;
                uint32_t put = 0;
                #pragma unroll
                for (int j = 0; j < 4; j++) { at += __popc(m[j] & ((1u << lane) - 1)); open += __popc(m[j]); }
                if (lane == 0) put = atomicAdd(n_near, (uint32_t)(__popc(m[0]) + __popc(m[1]) + __popc(m[2]) + __popc(m[3])));
                put = __shfl_sync(0xffffffffu, put, 0) + at - (open - __popc(m[0]) - __popc(m[1]) - __popc(m[2]) - __popc(m[3]));
                #pragma unroll
                for (int j = 0; j < 4; j++)
                    if (m[j] >> lane & 1) {
                        if (put < LG_SAMPLE_NEAR) near[put] = key_of<LOW>(l[j]); else full = true;
                        if (!listed) { if (at < LG_SAMPLE_LIST) { lv[at] = l[j]; li[at] = i + lane * 4 + j; } else full = true; }
                        put++; at++;
                    }
            }
            if (lane == 0) found += open;
            if (full) found += 1u << 30;
            over_w = weighted ? (u64)(long long)over : 0;
            n_list = listed || !weighted ? -1 : open;
            const u64 *counts;
            sum2(weighted ? over_w : found >> 32, found & 0xFFFFFFFFull, above, found, &counts);
            if (found <= 8 * LG_SAMPLE_THREADS) {
                // eight tokens a thread, from the CTA that has them; the rounds need no other CTA
                uint32_t key[8];
                u64 x[8];
                const uint32_t n_c = (lane < ranks) ? (uint32_t)ld_peer_u64(counts + 1, lane) : 0, up = (uint32_t)warp_scan_u64(n_c, lane);
                #pragma unroll
                for (int q = 0; q < 8; q++) {
                    const uint32_t i = threadIdx.x + q * LG_SAMPLE_THREADS;
                    x[q] = 0; key[q] = 0;
                    if (q * LG_SAMPLE_THREADS + warp * 32 >= found) continue;
                    int c = 0;
                    uint32_t before = 0;
                    for (int o = 0; o < ranks; o++) { const uint32_t e = __shfl_sync(0xffffffffu, up, o); if (i >= e) { c = o + 1; before = e; } }
                    if (i < found) key[q] = ld_peer_u32(near + (i - before), c);
                    const u64 v = mass(weighted, key_value<LOW>(key[q]));
                    if (i < found) x[q] = v;
                }
                if (n_pool && wide == 0) {
                    #pragma unroll
                    for (int q = 0; q < 8; q++) if (threadIdx.x + q * LG_SAMPLE_THREADS < found) pool()[threadIdx.x + q * LG_SAMPLE_THREADS] = key[q];
                    *n_pool = (int)found;
                }
                settle(key, x, above, target, klo, khi);
                break;
            }
            // too many: one round of the whole cluster
            const int sh = shift_of(khi - klo);
            uint32_t *h = fresh_hist(weighted ? 3 * LG_SAMPLE_BINS : LG_SAMPLE_BINS);
            for (int i = w0; i < w1; i += 128) {
                float l[4];
                fetch4(i + lane * 4, l);
                bool in[4];
                #pragma unroll
                for (int j = 0; j < 4; j++) in[j] = l[j] >= lo && l[j] <= hi;
                if (!__any_sync(0xffffffffu, in[0] || in[1] || in[2] || in[3])) continue;
                #pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (!__any_sync(0xffffffffu, in[j])) continue;
                    const int part = (int)((khi - key_of<LOW>(l[j])) >> sh);
                    const u64 x = mass(weighted, l[j]);
                    if (in[j] && weighted) add_weight(h, part, x);
                    else if (in[j]) atomicAdd(h + part, 1u);
                }
            }
            cluster_sync_all();
            share_bins(h, LG_SAMPLE_BINS, weighted ? 3 : 1);
            u64 v[2];
            int part;
            shared_bins(v);
            first_reaching(v, above, target, part, above);
            narrow(part, sh, klo, khi);
            n_list = -1;
            cluster_sync_all();                                               // `fine` and the lists are used again
            if (sh == 0 || wide == 3) break;
        }
        t = khi;
        if (!weighted) { ties = target - above; return; }
        const u64 one = mass(true, key_value<LOW>(t));
        ties = one ? (target - above + one - 1) / one : 1;
    }
};

// grid: rows x ranks, clusters of `ranks` CTAs
template <typename T> __global__ void __launch_bounds__(LG_SAMPLE_THREADS, 2) lg_sample_kernel(LgSampleArgs a) {
    extern __shared__ __align__(16) unsigned char lg_sample_sm[];
    __shared__ u64 word[48], red[2 * LG_SAMPLE_WARPS + 5];
    __shared__ int kind[LG_SAMPLE_WARPS];               // tokens of a warp's list; -1: it has the row's own, -2: and min_p takes none of those above the threshold
    typedef LogitType<T> L;
    constexpr int LOW = L::LOW;
    uint32_t ranks;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
    const int rank = (int)cluster_rank(), row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = rank * a.slice, n = max(0, min(a.vocab - first, a.slice));
    LgSampler<T> s{a};
    s.g = (const T *)a.logits + (long long)row * a.ld + first;
    s.data = (T *)lg_sample_sm;
    s.hist = (uint32_t *)(lg_sample_sm + (size_t)a.cap * sizeof(T));
    s.fine = (u64 *)(s.hist + 2 * LG_SAMPLE_HIST);
    s.near = (uint32_t *)(s.fine + LG_SAMPLE_COARSE);
    s.lv = (float *)(s.near + LG_SAMPLE_NEAR) + warp * LG_SAMPLE_LIST * 2; s.li = (int *)(s.lv + LG_SAMPLE_LIST);
    s.word = word; s.red = red; s.n = n; s.first = first; s.ranks = ranks; s.rank = rank; s.lane = lane; s.warp = warp;
    const int per = ((a.slice + LG_SAMPLE_WARPS - 1) / LG_SAMPLE_WARPS + 127) / 128 * 128;
    s.w0 = min(warp * per, n); s.w1 = min(s.w0 + per, n);
    const float T1 = a.temperature ? a.temperature[row] : 1.0f, top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f;
    const int top_k = a.top_k ? a.top_k[row] : 0;

    // the row, once: into shared memory, and its largest logit
    float best = -INFINITY;
    {
        constexpr int V = 16 / sizeof(T);
        const int held = min(n, a.cap), vec = ((uintptr_t)s.g & 15) ? 0 : held / V * V;
        uint32_t m = L::lowest();
        for (int i = tid * V; i < vec; i += LG_SAMPLE_THREADS * V * 4) {
            uint4 v[4];
            #pragma unroll
            for (int q = 0; q < 4; q++) {
                const int at = i + q * LG_SAMPLE_THREADS * V;
                v[q] = make_uint4(L::lowest(), L::lowest(), L::lowest(), L::lowest());
                if (at < vec) v[q] = ldg_stream16((const uint4 *)(s.g + at));
            }
            #pragma unroll
            for (int q = 0; q < 4; q++) {
                const int at = i + q * LG_SAMPLE_THREADS * V;
                if (at < vec) *(uint4 *)(s.data + at) = v[q];
                m = L::larger(L::larger(m, L::larger(v[q].x, v[q].y)), L::larger(v[q].z, v[q].w));
            }
        }
        best = L::most(m);
        for (int i = vec + tid; i < held; i += LG_SAMPLE_THREADS) { const T x = s.g[i]; s.data[i] = x; best = fmaxf(best, L::value(&x)); }
        for (int i = held + tid; i < a.cap; i += LG_SAMPLE_THREADS) ((uint16_t *)s.data)[i * (sizeof(T) / 2) + sizeof(T) / 2 - 1] = 0x7FFF;      // NaN in any of the types
        for (int i = held + tid; i < n; i += LG_SAMPLE_THREADS) best = fmaxf(best, L::value(s.g + i));
    }
    best = warp_max(best);
    if (lane == 0) red[warp] = __float_as_uint(best);
    __syncthreads();
    if (warp == 0) {
        best = warp_max(lane < LG_SAMPLE_WARPS ? __uint_as_float((uint32_t)red[lane]) : -INFINITY);
        if (lane == 0) word[0] = __float_as_uint(best);
    }
    cluster_sync_all();
    for (uint32_t c = 0; c < ranks; c++) best = fmaxf(best, __uint_as_float((uint32_t)ld_peer_u64(word, c)));
    s.at_word = 1;
    if (best == -INFINITY || !(T1 > 0.0f) || top_k == 1 || top_p <= 0.0f || min_p > 1.0f) {
        // nothing to draw, or the first token of the order: the lowest place of the largest logit
        u64 place = ~0ull;
        if (best > -INFINITY)
            for (int i = s.w0; i < s.w1; i += 128) {
                float l[4];
                s.fetch4(i + lane * 4, l);
                #pragma unroll
                for (int j = 3; j >= 0; j--) if (l[j] == best) place = min(place, (u64)(first + i + lane * 4 + j));
            }
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) place = min(place, (u64)__shfl_xor_sync(0xffffffffu, place, o));
        __syncthreads();
        if (lane == 0) red[warp] = place;
        __syncthreads();
        if (tid == 0) {
            for (int i = 1; i < LG_SAMPLE_WARPS; i++) place = min(place, red[i]);
            word[1] = place;
        }
        cluster_sync_all();
        if (rank == 0 && tid == 0) {
            for (uint32_t c = 1; c < ranks; c++) place = min(place, ld_peer_u64(word + 1, c));
            a.token[row] = place == ~0ull ? -1 : (int)place;
            if (a.prob) a.prob[row] = place == ~0ull ? 0.0f : 1.0f;
        }
        cluster_sync_all();                             // no CTA leaves while another reads its words
        return;
    }
    const uint32_t top_key = key_of<LOW>(best);
    s.w.top = (double)fminf(best, 3.402823466e38f); s.w.inv32 = best == INFINITY ? 0.0 : 46.166241308446828 / (double)T1; s.w.root = exp2(a.shift - lane / 32.0);

    uint32_t t = best == INFINITY ? top_key - 1 : LgSampler<T>::DEAD;          // threshold; at first everything above -inf
    u64 ties = 0, over_w = 0;
    int n_pool = 0;                                     // keys in pool(): all from the threshold up
    int n_list = -1;                                    // >= 0: this warp's list and over_w say what it keeps (LgSampler::refine)
    if (top_k > 0 && top_k < a.vocab) {
        uint32_t *h = s.fresh_hist(LG_SAMPLE_COARSE);
        const float lt = key_value<LOW>(t);
        for (int i = s.w0; i < s.w1; i += 128) {
            float l[4];
            s.fetch4(i + lane * 4, l);
            #pragma unroll
            for (int j = 0; j < 4; j++) {
                int k;
                double rest;
                if (s.w.bin(l[j], k, rest) && l[j] > lt) atomicAdd(h + k, 1u);
            }
        }
        cluster_sync_all();
        s.share_bins(h, LG_SAMPLE_COARSE, 1);
        u64 v[4], before;
        int bin;
        s.shared_bins(v);
        if (s.first_reaching(v, 0, (u64)top_k, bin, before)) {              // otherwise fewer than top_k tokens have a weight
            uint32_t klo, khi;
            s.interval(bin, bin, t + 1, top_key, klo, khi);
            s.make_list(key_value<LOW>(klo));
            // few: every CTA fetches them all, and needs no other for top_p either
            if (top_k <= 2048) khi = top_key;
            s.refine(false, (u64)top_k, klo, khi, t, ties, over_w, n_list, top_k <= 2048 ? &n_pool : nullptr);
        }
    }
    const u64 p64 = top_p < 1.0f ? __double2ull_rz((double)top_p * 18446744073709551616.0) : 0;
    // the weight that top_p asks for of `total`
    auto share = [&](u64 total) { const u64 w = __umul64hi(p64, total) + (p64 * total != 0); return w < 1 ? (u64)1 : w; };
    if (top_p < 1.0f && n_pool) {
        uint32_t key[8];
        u64 x[8], over = 0, at_t = 0;
        __syncthreads();
        #pragma unroll
        for (int q = 0; q < 8; q++) {
            x[q] = 0; key[q] = 0;
            if (q * LG_SAMPLE_THREADS + warp * 32 >= n_pool) continue;
            const int i = tid + q * LG_SAMPLE_THREADS;
            if (i < n_pool) key[q] = s.pool()[i];
            const u64 v = s.mass(true, key_value<LOW>(key[q]));
            if (i < n_pool && key[q] > t) { x[q] = v; over += v; }
            at_t += i < n_pool && key[q] == t;
        }
        s.own_sum2(over, at_t, over, at_t);
        const u64 one = s.mass(true, key_value<LOW>(t));
        if (ties < at_t) at_t = ties;
        const u64 target = share(over + at_t * one);
        if (target > over) ties = min(ties, one ? (target - over + one - 1) / one : ties);
        else {
            uint32_t klo = t + 1, khi = top_key;
            u64 above = 0;
            s.settle(key, x, above, target, klo, khi);
            t = khi;
            const u64 w_t = s.mass(true, key_value<LOW>(t));
            ties = w_t ? (target - above + w_t - 1) / w_t : 1;
        }
    } else if (top_p < 1.0f) {
        // weight above the threshold, tokens at it
        uint32_t *h = s.fresh_hist(LG_SAMPLE_COARSE);
        const float lt = key_value<LOW>(t);
        double sum = 0.0;
        u64 over, at_t;
        uint32_t n_at = 0;
        for (int i = s.w0; i < s.w1; i += 128) {
            float l[4];
            int k[4];
            double x[4];
            bool in[4];
            s.fetch4(i + lane * 4, l);
            if (ties) n_at += (l[0] == lt) + (l[1] == lt) + (l[2] == lt) + (l[3] == lt);
            if (!__any_sync(0xffffffffu, l[0] > lt || l[1] > lt || l[2] > lt || l[3] > lt)) continue;
            double p[4];
            s.weigh4(l, lt, k, x, in, p);
            #pragma unroll
            for (int j = 0; j < 4; j++)
                if (in[j]) { sum += LgWeight::whole(x[j]); atomicAdd(h + k[j], (uint32_t)__double2loint(fma(p[j], 1000.0, LG_TWO52))); }
        }
        s.sum2((u64)(long long)sum, n_at, over, at_t);
        const u64 one = (u64)(long long)LgWeight::whole(s.w.of(lt));
        if (ties < at_t) at_t = ties;
        const u64 target = share(over + at_t * one);
        if (target > over) ties = min(ties, one ? (target - over + one - 1) / one : ties);
        else {
            // a bin's tokens count 989 .. 1011 each: their weights in thousandths of the bin's own, to half of one
            u64 c[4], v[4], low[4];
            int b0, b1;
            s.share_bins(h, LG_SAMPLE_COARSE, 1);
            s.shared_bins(c);
            #pragma unroll
            for (int j = 0; j < 4; j++) {
                const double edge = (double)c[j] * (s.w.scaled(4 * tid + j, 0.0) * 0.001);
                const u64 least = __double2ull_rd(edge * 0.9994);
                v[j] = __double2ull_ru(edge * 1.0006) + c[j];                 // (and half a unit for the rounding of each weight)
                low[j] = least > c[j] ? least - c[j] : 0;
            }
            s.bracket(v, low, target, b0, b1);
            uint32_t klo, khi;
            s.interval(b0, max(b0, b1), t + 1, top_key, klo, khi);
            s.refine(true, target, klo, khi, t, ties, over_w, n_list, nullptr);
        }
    }
    // the draw: what each warp's tokens weigh and how many lie at the threshold, then the warp in which the running weight passes the target
    const double floor_w = min_p > 0.0f ? (double)min_p * (double)(1ull << a.shift) : 0.0;
    const float lt = key_value<LOW>(t);
    const double x_t = s.w.of(lt);
    const u64 one = x_t >= floor_w ? (u64)(long long)LgWeight::whole(x_t) : 0;
    u64 over, at_t;
    const bool noted = n_list >= 0 && (ties ? x_t : 0.0) >= floor_w;
    if (noted) {
        // min_p takes nothing away: the weight above the list, and the list's own tokens
        over = over_w; at_t = 0;
        for (int i = 0; i < n_list; i += 32) {
            const float l = i + lane < n_list ? s.lv[i + lane] : -INFINITY;
            const u64 x = s.mass(true, l);
            if (l > lt) over += x;
            at_t += l == lt && ties;
        }
    } else {
        // min_p's own threshold, a little lower: what is below it needs no weight
        const float from = floor_w > 0.0 && s.w.inv32 > 0.0 ? fmaxf(lt, __double2float_rd(s.w.top + (32.0 * log2((double)min_p) - 0.01) / s.w.inv32)) : lt;
        double sum = 0.0;
        uint32_t n_at = 0;
        for (int i = s.w0; i < s.w1; i += 128) {
            float l[4];
            int k[4];
            double x[4];
            bool in[4];
            s.fetch4(i + lane * 4, l);
            if (ties) n_at += (l[0] == lt) + (l[1] == lt) + (l[2] == lt) + (l[3] == lt);
            if (!__any_sync(0xffffffffu, l[0] >= from || l[1] >= from || l[2] >= from || l[3] >= from)) continue;
            s.weigh4(l, lt, k, x, in);
            #pragma unroll
            for (int j = 0; j < 4; j++) if (in[j] && x[j] >= floor_w) sum += LgWeight::whole(x[j]);
        }
        over = (u64)(long long)sum; at_t = n_at;
    }
    // ties before one of several pieces of the row (a lane each), the weight before it and in it, where a piece's tokens at the threshold are kept while
    // there are ties left; `all`: the weight behind the last piece
    auto before = [&](u64 x, u64 y, u64 ties0, u64 run0, u64 &y0, u64 &x0, u64 &all) {
        const u64 y_up = warp_scan_u64(y, lane);
        y0 = ties0 + y_up - y;
        const u64 left = ties > y0 ? ties - y0 : 0, x_all = x + (y < left ? y : left) * one, x_up = warp_scan_u64(x_all, lane);
        x0 = run0 + x_up - x_all;
        all = run0 + __shfl_sync(0xffffffffu, x_up, 31);
        return x_all;
    };
    if (lane == 0) kind[warp] = s.listed ? s.w1 : noted ? -2 : -1;
    const u64 *mine;
    u64 total, none, y0, x0;
    s.sum2(over, at_t, total, none, &mine);
    u64 x_all = before(lane < (int)ranks ? ld_peer_u64(mine, lane) : 0, lane < (int)ranks ? ld_peer_u64(mine + 1, lane) : 0, 0, 0, y0, x0, total);
    const float u = a.u[row];
    const u64 u_64 = u > 0.0f ? u < 1.0f ? __double2ull_rz((double)u * 18446744073709551616.0) : ~0ull : 0ull, target = __umul64hi(u_64, total);
    uint32_t hit = __ballot_sync(0xffffffffu, x0 <= target && target < x0 + x_all);
    if (hit && __ffs(hit) - 1 == rank) {
        // this CTA: the warp in whose tokens the running weight passes the target, then a sixteenth of those, each by a warp
        u64 ties0 = __shfl_sync(0xffffffffu, y0, rank), run = __shfl_sync(0xffffffffu, x0, rank);
        x_all = before(lane < LG_SAMPLE_WARPS ? red[lane] : 0, lane < LG_SAMPLE_WARPS ? red[LG_SAMPLE_WARPS + lane] : 0, ties0, run, y0, x0, none);
        hit = __ballot_sync(0xffffffffu, x0 <= target && target < x0 + x_all);
        const int who = hit ? __ffs(hit) - 1 : 0;
        ties0 = __shfl_sync(0xffffffffu, y0, who); run = __shfl_sync(0xffffffffu, x0, who);
        s.listed = kind[who] >= 0;
        const double least = kind[who] == -2 ? 0.0 : floor_w;
        s.lv += (who - warp) * LG_SAMPLE_LIST * 2; s.li += (who - warp) * LG_SAMPLE_LIST * 2;
        const int from = s.listed ? 0 : min(who * per, n), to = s.listed ? kind[who] : min(from + per, n), sub = ((to - from + LG_SAMPLE_WARPS - 1) / LG_SAMPLE_WARPS + 127) / 128 * 128;
        const int i0 = min(from + warp * sub, to), i1 = min(i0 + sub, to);
        // four tokens a lane: what each weighs if it is kept, ties aside, and which lie at the threshold
        auto kept4 = [&](int i, double (&x)[4], u64 (&v)[4]) {
            float l[4];
            int k[4];
            bool in[4];
            s.fetch4(i + lane * 4, l);
            s.weigh4(l, lt, k, x, in);
            uint32_t eq = 0;
            #pragma unroll
            for (int j = 0; j < 4; j++) {
                v[j] = in[j] && x[j] >= least ? (u64)(long long)LgWeight::whole(x[j]) : 0;
                eq |= (uint32_t)(ties && l[j] == lt) << j;
                if (l[j] == lt) x[j] = x_t;
            }
            return eq;
        };
        double x[4];
        u64 v[4];
        over = at_t = 0;
        for (int i = i0; i < i1; i += 128) { const uint32_t eq = kept4(i, x, v); over += v[0] + v[1] + v[2] + v[3]; at_t += __popc(eq); }
        over = warp_sum_u64(over); at_t = warp_sum_u64(at_t);
        __syncthreads();
        if (lane == 0) { red[warp] = over; red[LG_SAMPLE_WARPS + warp] = at_t; }
        __syncthreads();
        x_all = before(lane < LG_SAMPLE_WARPS ? red[lane] : 0, lane < LG_SAMPLE_WARPS ? red[LG_SAMPLE_WARPS + lane] : 0, ties0, run, y0, x0, none);
        hit = __ballot_sync(0xffffffffu, x0 <= target && target < x0 + x_all);
        if (hit && __ffs(hit) - 1 == warp) {
            run = __shfl_sync(0xffffffffu, x0, warp);
            u64 rank_t = __shfl_sync(0xffffffffu, y0, warp);
            for (int i = i0; i < i1; i += 128) {
                const uint32_t eq = kept4(i, x, v);
                const u64 ties_up = warp_scan_u64(__popc(eq), lane);
                u64 rk = rank_t + ties_up - __popc(eq), sum = 0;
                #pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (eq >> j & 1) v[j] = rk++ < ties ? one : 0;
                    sum += v[j];
                }
                const u64 up = warp_scan_u64(sum, lane);
                hit = __ballot_sync(0xffffffffu, run + up > target);
                if (hit) {
                    if (lane == __ffs(hit) - 1) {
                        u64 at = run + up - sum;
                        int at_j = 0;
                        double got = x[0];
                        #pragma unroll
                        for (int j = 0; j < 3; j++) if (at_j == j && at + v[j] <= target) { at += v[j]; at_j++; got = x[j + 1]; }
                        a.token[row] = first + (s.listed ? s.li[i + lane * 4 + at_j] : i + lane * 4 + at_j);
                        if (a.prob) a.prob[row] = (float)(got / (double)total);
                    }
                    break;
                }
                run += __shfl_sync(0xffffffffu, up, 31);
                rank_t += __shfl_sync(0xffffffffu, ties_up, 31);
            }
        }
    }
    cluster_sync_all();
}
