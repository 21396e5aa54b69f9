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
//   coarse  y = 32 log2(e) (max - l) / T, rounded, is the bin of a token (at most 2047: beyond, a weight is 0); counts per bin and the bounds of a bin's
//           weights tell the bins that the threshold can lie in, and with them an interval of logits
//   fine    exact counts or weights over 2048 equal parts of that interval of keys (the logits as ordered integers), then of the part that holds the threshold,
//           until a part is a single key: at most three rounds
// Bound by 64-bit arithmetic (about 11 operations a weight, 64 a cycle and SM) and, for few rows, by the cluster barriers.
#pragma once
#include "lg_device.cuh"
#include <cuda_bf16.h>

#define LG_SAMPLE_THREADS 512
#define LG_SAMPLE_WARPS (LG_SAMPLE_THREADS / 32)
#define LG_SAMPLE_BINS 2048
#define LG_SAMPLE_MAX_CLUSTER 8

typedef unsigned long long u64;

struct LgSampleArgs {
    const void *logits;
    long long ld;
    int rows, vocab, shift;
    int slice, cap;                    // tokens per CTA of a cluster; of these, tokens held in shared memory
    int limbs;                         // histograms: 0 none, 1 counts, 3 weights too
    const float *temperature; const int *top_k; const float *top_p; const float *min_p; const float *u;
    int *token; float *prob;
};

// A logit as the bits of its f32 value, and as an unsigned integer in the order of the logits (LOW: bits that are the same in every f32 that the type
// holds; they are dropped).  NaN lowest, -0 equal to 0.
template <typename T> struct LogitType;
template <> struct LogitType<float> {
    static constexpr int LOW = 0;
    static __device__ __forceinline__ uint32_t bits(const float *p) { return __float_as_uint(*p); }
    static __device__ __forceinline__ void bits4(const float *p, uint32_t (&b)[4]) {
        const uint4 v = *(const uint4 *)p;
        b[0] = v.x; b[1] = v.y; b[2] = v.z; b[3] = v.w;
    }
};
template <> struct LogitType<__half> {
    static constexpr int LOW = 13;
    static __device__ __forceinline__ uint32_t bits(const __half *p) { return __float_as_uint(__half2float(*p)); }
    static __device__ __forceinline__ void bits4(const __half *p, uint32_t (&b)[4]) {
        const uint2 v = *(const uint2 *)p;
        const float2 f = __half22float2(*(const __half2 *)&v.x), h = __half22float2(*(const __half2 *)&v.y);
        b[0] = __float_as_uint(f.x); b[1] = __float_as_uint(f.y); b[2] = __float_as_uint(h.x); b[3] = __float_as_uint(h.y);
    }
};
template <> struct LogitType<__nv_bfloat16> {
    static constexpr int LOW = 16;
    static __device__ __forceinline__ uint32_t bits(const __nv_bfloat16 *p) { return (uint32_t)*(const uint16_t *)p << 16; }
    static __device__ __forceinline__ void bits4(const __nv_bfloat16 *p, uint32_t (&b)[4]) {
        const uint2 v = *(const uint2 *)p;
        b[0] = v.x << 16; b[1] = v.x & 0xFFFF0000u; b[2] = v.y << 16; b[3] = v.y & 0xFFFF0000u;
    }
};
#define LG_NAN_BITS 0x7FC00000u
template <int LOW> __device__ __forceinline__ uint32_t key_of(uint32_t b) {
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0;
    if (b == 0x80000000u) b = 0;
    return (b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u)) >> LOW;
}
template <int LOW> __device__ __forceinline__ uint32_t key_bits(uint32_t k) {
    const uint32_t full = k << LOW;
    return (full >> 31) ? full ^ 0x80000000u : ~(full | ((1u << LOW) - 1));
}
// the same of a number, rounded down or up to a f32
template <int LOW> __device__ __forceinline__ uint32_t key_below(double x) { return key_of<LOW>(__float_as_uint(__double2float_rd(x))); }
template <int LOW> __device__ __forceinline__ uint32_t key_above(double x) { return key_of<LOW>(__float_as_uint(__double2float_ru(x))); }

// exp((l - top) / T) of a row
struct LgWeight {
    double top, inv32, root;           // inv32: 32 log2(e) / T; root: 2^(-lane / 32)
    int shift;
    bool inf;                          // the largest logit is +inf: 1 for those, 0 for the others
    // y of a logit; false: its weight is 0
    __device__ __forceinline__ bool arg(uint32_t b, double &y) const {
        y = 0.0;
        const uint32_t e = b & 0x7F800000u;
        if (inf) return b == 0x7F800000u;
        if (e == 0x7F800000u) return false;                                   // -inf, NaN
        // f32 -> f64 by moving bits: the conversion instruction runs at a quarter of the rate of the arithmetic
        const double l = e ? __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7FFFFFFFu) >> 3) + 0x38000000u)), (int)(b << 29)) : (double)__uint_as_float(b);
        const double x = (top - l) * inv32;
        const bool live = (uint32_t)__double2hiint(x) < 0x409FFC00u;          // x < 2047
        if (live) y = x;
        return live;
    }
    // w = 2^(shift - y / 32), all lanes of a warp together: 2^(-k / 32) of the nearest whole k, from its lane, times a polynomial of the rest
    // (Taylor, |x| <= ln 2 / 64: the first term left out is below 2^-48).  k: the coarse bin.
    __device__ __forceinline__ double scaled(double y, int &k) const {
        const double magic = 6755399441055744.0;                              // 1.5 2^52: adding it rounds to a whole number
        const double t = y + magic;
        k = __double2loint(t);
        const double x = (y - (t - magic)) * -0.02166084939249829;            // -ln 2 / 32
        double p = fma(x, 1.0 / 120.0, 1.0 / 24.0);
        p = fma(p, x, 1.0 / 6.0);
        p = fma(p, x, 0.5);
        p = fma(p, x, 1.0);
        p = fma(p, x, 1.0);
        const int hi = __shfl_sync(0xffffffffu, __double2hiint(root), k & 31), lo = __shfl_sync(0xffffffffu, __double2loint(root), k & 31);
        return p * __hiloint2double(hi + ((shift - (k >> 5)) << 20), lo);
    }
    static __device__ __forceinline__ u64 whole(double s) {                   // to the nearest integer, s < 2^51
        return (u64)__double_as_longlong(s + 4503599627370496.0) - 0x4330000000000000ull;
    }
};

__device__ __forceinline__ uint32_t ld_peer_u32(uint32_t addr, uint32_t rank) {
    uint32_t ra, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(ra) : "memory");
    return v;
}
__device__ __forceinline__ u64 ld_peer_u64(const u64 *p, uint32_t rank) {
    uint32_t ra; u64 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(ra) : "memory");
    return v;
}
__device__ __forceinline__ uint4 ld_peer_u32x4(const uint32_t *p, uint32_t rank) {
    uint32_t ra; uint4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(ra) : "memory");
    return v;
}
__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
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
    u64 *word;                         // words for the other CTAs: a place per exchange
    u64 *red;                          // [2 * warps] and more, block-wide
    int n, first, ranks, rank, lane, warp, turn = 0, at_word = 0;             // tokens here, index of the first
    int w0, w1;                        // this warp's tokens
    LgWeight w;

    __device__ __forceinline__ void fetch4(int i, uint32_t (&b)[4]) const {
        if (i + 4 <= a.cap) L::bits4(data + i, b);
        else {
            #pragma unroll
            for (int j = 0; j < 4; j++) b[j] = i + j < n ? i + j < a.cap ? L::bits(data + i + j) : L::bits(g + i + j) : LG_NAN_BITS;
        }
    }
    // Sums of two numbers a thread over the cluster; each CTA's own sums are left in own[0], own[1]
    __device__ void sum2(u64 x, u64 y, u64 &sx, u64 &sy) {
        x = warp_sum_u64(x); y = warp_sum_u64(y);
        __syncthreads();
        if (lane == 0) { red[warp] = x; red[LG_SAMPLE_WARPS + warp] = y; }
        __syncthreads();
        u64 *p = word + at_word;
        at_word += 2;
        if (warp == 0) {
            x = lane < LG_SAMPLE_WARPS ? red[lane] : 0; y = lane < LG_SAMPLE_WARPS ? red[LG_SAMPLE_WARPS + lane] : 0;
            x = warp_sum_u64(x); y = warp_sum_u64(y);
            if (lane == 0) { p[0] = x; p[1] = y; }
        }
        cluster_sync_all();
        sx = sy = 0;
        for (int c = 0; c < ranks; c++) { sx += ld_peer_u64(p, c); sy += ld_peer_u64(p + 1, c); }
    }
    // An empty histogram (block-wide; the cluster has passed a barrier since the one before it was read)
    __device__ uint32_t *fresh_hist(int limbs) {
        uint32_t *h = hist + turn * a.limbs * LG_SAMPLE_BINS;
        turn ^= 1;
        for (int i = threadIdx.x; i < limbs * LG_SAMPLE_BINS; i += LG_SAMPLE_THREADS) h[i] = 0;
        __syncthreads();
        return h;
    }
    static __device__ __forceinline__ void add_weight(uint32_t *h, int bin, u64 x) {      // 15 bits per array: 2^17 tokens fit 32 bits
        if (const uint32_t v = (uint32_t)x & 0x7FFFu) atomicAdd(h + bin, v);
        if (const uint32_t v = (uint32_t)(x >> 15) & 0x7FFFu) atomicAdd(h + LG_SAMPLE_BINS + bin, v);
        if (const uint32_t v = (uint32_t)(x >> 30)) atomicAdd(h + 2 * LG_SAMPLE_BINS + bin, v);
    }
    // This thread's four bins, summed over the cluster
    __device__ __forceinline__ void bins4(const uint32_t *h, int limbs, u64 (&v)[4]) const {
        v[0] = v[1] = v[2] = v[3] = 0;
        for (int l = 0; l < limbs; l++)
            for (int c = 0; c < ranks; c++) {
                const uint4 x = ld_peer_u32x4(h + l * LG_SAMPLE_BINS + threadIdx.x * 4, c);
                v[0] += (u64)x.x << 15 * l; v[1] += (u64)x.y << 15 * l; v[2] += (u64)x.z << 15 * l; v[3] += (u64)x.w << 15 * l;
            }
    }
    // The first bin at which before + the running sum of v reaches the target, and the sum before it; the last bin where none does (found = false).
    // `slot` keeps two results of one call apart.
    __device__ bool first_reaching(const u64 (&v)[4], u64 before, u64 target, int slot, int &bin, u64 &sum) {
        const u64 mine = v[0] + v[1] + v[2] + v[3], incl = warp_scan_u64(mine, lane);
        __syncthreads();
        if (lane == 31) red[warp] = incl;
        if (threadIdx.x == 0) red[2 * LG_SAMPLE_WARPS + slot] = ~0ull;
        __syncthreads();
        u64 at = before + incl - mine, all = before;
        #pragma unroll
        for (int i = 0; i < LG_SAMPLE_WARPS; i++) { if (i < warp) at += red[i]; all += red[i]; }
        if (at < target && target <= at + mine) {
            int j = 0;
            while (at + v[j] < target) at += v[j++];
            red[2 * LG_SAMPLE_WARPS + slot] = threadIdx.x * 4 + j;
            red[2 * LG_SAMPLE_WARPS + 2 + slot] = at;
        }
        __syncthreads();
        const u64 b = red[2 * LG_SAMPLE_WARPS + slot];
        const bool found = b != ~0ull;
        bin = found ? (int)b : LG_SAMPLE_BINS - 1;
        sum = found ? red[2 * LG_SAMPLE_WARPS + 2 + slot] : all;
        return found;
    }
    // Keys of the bins b0 .. b1 of the coarse histogram, a bin more on either side
    __device__ void interval(int b0, int b1, uint32_t low, uint32_t top_key, uint32_t &klo, uint32_t &khi) const {
        klo = low; khi = top_key;
        if (w.inf || !(w.inv32 > 0.0)) return;
        const double lo = w.top - (b1 + 1) / w.inv32, hi = w.top - (b0 - 1) / w.inv32;
        klo = max(low, key_below<LOW>(lo));
        khi = min(top_key, key_above<LOW>(hi));
    }
    // The threshold at which counts (weighted: weights) of the keys from the largest down reach the target; it lies in klo .. khi, and all keys
    // in question are above `floor_key`.  Kept then: keys above t and `ties` of key t.
    __device__ void refine(bool weighted, u64 target, uint32_t klo, uint32_t khi, uint32_t &t, u64 &ties) {
        u64 above = 0;
        for (int round = 0; round < 3; round++) {                             // 11 bits of at most 32 a round
            const bool begin = round == 0;
            const uint32_t range = khi - klo;
            const int sh = range >= LG_SAMPLE_BINS ? 21 - __clz(range) : 0;    // range >> sh < 2048
            uint32_t *h = fresh_hist(weighted ? 3 : 1);
            u64 over = 0;
            for (int i = w0; i < w1; i += 128) {
                uint32_t b[4];
                fetch4(i + lane * 4, b);
                #pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t k = key_of<LOW>(b[j]);
                    const bool in = k >= klo && k <= khi, more = begin && k > khi;
                    if (weighted) {
                        if (!__any_sync(0xffffffffu, in || more)) continue;
                        double y;
                        int bin;
                        const bool live = w.arg(b[j], y);
                        const u64 x = LgWeight::whole(w.scaled(y, bin));
                        if (live && more) over += x;
                        if (live && in) add_weight(h, (khi - k) >> sh, x);
                    } else {
                        if (more) over++;
                        if (in) atomicAdd(h + ((khi - k) >> sh), 1u);
                    }
                }
            }
            if (begin) { u64 none; sum2(over, 0, above, none); }               // (its barrier also makes the histograms complete)
            else cluster_sync_all();
            u64 v[4];
            int bin;
            bins4(h, weighted ? 3 : 1, v);
            first_reaching(v, above, target, 0, bin, above);
            // `above` is now what lies above the part `bin`
            khi -= (uint32_t)bin << sh;
            klo = max(klo, khi - ((1u << sh) - 1) > khi ? 0u : khi - ((1u << sh) - 1));
            if (sh == 0) break;
        }
        t = khi;
        if (!weighted) { ties = target - above; return; }
        double y;
        int bin;
        const bool live = w.arg(key_bits<LOW>(t), y);
        const u64 one = LgWeight::whole(w.scaled(y, bin));
        ties = live && one ? (target - above + one - 1) / one : 1;
    }
};

// grid: rows x ranks, clusters of `ranks` CTAs
template <typename T> __global__ void __launch_bounds__(LG_SAMPLE_THREADS) lg_sample_kernel(LgSampleArgs a) {
    extern __shared__ __align__(16) unsigned char lg_sample_sm[];
    __shared__ u64 word[48], red[2 * LG_SAMPLE_WARPS + 4];
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
    s.word = word; s.red = red; s.n = n; s.first = first; s.ranks = ranks; s.rank = rank; s.lane = lane; s.warp = warp;
    const int per = ((a.slice + LG_SAMPLE_WARPS - 1) / LG_SAMPLE_WARPS + 127) / 128 * 128;
    s.w0 = min(warp * per, n); s.w1 = min(s.w0 + per, n);
    const float T1 = a.temperature ? a.temperature[row] : 1.0f, top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f;
    const int top_k = a.top_k ? a.top_k[row] : 0;

    // the row, once: into shared memory, and its largest logit with its first place
    u64 best = 0;
    auto seen = [&](uint32_t b, int i) {
        const u64 k = (u64)key_of<LOW>(b) << 32 | (uint32_t)~(first + i);
        best = k > best ? k : best;
    };
    {
        constexpr int V = 16 / sizeof(T);
        const int held = min(n, a.cap), vec = ((uintptr_t)s.g & 15) ? 0 : held / V * V;
        for (int i = tid * V; i < vec; i += LG_SAMPLE_THREADS * V * 4) {
            uint4 v[4];
            #pragma unroll
            for (int q = 0; q < 4; q++) if (i + q * LG_SAMPLE_THREADS * V < vec) v[q] = ldg_stream16((const uint4 *)(s.g + i + q * LG_SAMPLE_THREADS * V));
            #pragma unroll
            for (int q = 0; q < 4; q++) {
                const int at = i + q * LG_SAMPLE_THREADS * V;
                if (at < vec) {
                    *(uint4 *)(s.data + at) = v[q];
                    uint32_t b[4];
                    #pragma unroll
                    for (int h = 0; h < V / 4; h++) {
                        L::bits4((const T *)&v[q] + 4 * h, b);
                        #pragma unroll
                        for (int j = 0; j < 4; j++) seen(b[j], at + 4 * h + j);
                    }
                }
            }
        }
        for (int i = vec + tid; i < held; i += LG_SAMPLE_THREADS) { const T x = s.g[i]; s.data[i] = x; seen(L::bits(&x), i); }
        for (int i = held + tid; i < a.cap; i += LG_SAMPLE_THREADS) ((uint16_t *)s.data)[i * (sizeof(T) / 2) + sizeof(T) / 2 - 1] = 0x7FFF;      // NaN in any of the types
        for (int i = held + tid; i < n; i += LG_SAMPLE_THREADS) seen(L::bits(s.g + i), i);
    }
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) { const u64 t = __shfl_xor_sync(0xffffffffu, best, o); best = t > best ? t : best; }
    if (lane == 0) red[warp] = best;
    __syncthreads();
    if (warp == 0) {
        best = lane < LG_SAMPLE_WARPS ? red[lane] : 0;
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) { const u64 t = __shfl_xor_sync(0xffffffffu, best, o); best = t > best ? t : best; }
        if (lane == 0) word[0] = best;
    }
    cluster_sync_all();
    best = 0;
    for (uint32_t c = 0; c < ranks; c++) { const u64 t = ld_peer_u64(word, c); best = t > best ? t : best; }
    s.at_word = 1;
    const uint32_t top_key = (uint32_t)(best >> 32);
    if (top_key <= LgSampler<T>::DEAD || !(T1 > 0.0f) || top_k == 1 || top_p <= 0.0f || min_p > 1.0f) {
        if (rank == 0 && tid == 0) {
            const bool none = top_key <= LgSampler<T>::DEAD;
            a.token[row] = none ? -1 : (int)~(uint32_t)best;
            if (a.prob) a.prob[row] = none ? 0.0f : 1.0f;
        }
        cluster_sync_all();                             // no CTA leaves while another reads its words
        return;
    }
    const uint32_t top_bits = key_bits<LOW>(top_key);
    s.w.inf = top_bits == 0x7F800000u;
    s.w.top = (double)__uint_as_float(top_bits); s.w.inv32 = 46.166241308446828 / (double)T1; s.w.root = exp2(-lane / 32.0); s.w.shift = a.shift;

    uint32_t t = LgSampler<T>::DEAD;                    // threshold; at first everything above -inf
    u64 ties = 0;
    if (top_k > 0 && top_k < a.vocab) {
        uint32_t *h = s.fresh_hist(1);
        for (int i = s.w0; i < s.w1; i += 128) {
            uint32_t b[4];
            s.fetch4(i + lane * 4, b);
            #pragma unroll
            for (int j = 0; j < 4; j++) {
                double y;
                if (s.w.arg(b[j], y)) atomicAdd(h + __double2loint(y + 6755399441055744.0), 1u);
            }
        }
        cluster_sync_all();
        u64 v[4], before;
        int bin;
        s.bins4(h, 1, v);
        if (s.first_reaching(v, 0, (u64)top_k, 0, bin, before)) {              // otherwise fewer than top_k tokens have a weight
            uint32_t klo, khi;
            s.interval(bin, bin, LgSampler<T>::DEAD + 1, top_key, klo, khi);
            s.refine(false, (u64)top_k, klo, khi, t, ties);
        }
    }
    if (top_p < 1.0f) {
        // weight above the threshold, tokens at it
        uint32_t *h = s.fresh_hist(1);
        u64 over = 0, at_t = 0;
        for (int i = s.w0; i < s.w1; i += 128) {
            uint32_t b[4];
            s.fetch4(i + lane * 4, b);
            #pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t k = key_of<LOW>(b[j]);
                at_t += k == t;
                if (!__any_sync(0xffffffffu, k > t)) continue;
                double y;
                int bin;
                const bool live = s.w.arg(b[j], y);
                const u64 x = LgWeight::whole(s.w.scaled(y, bin));
                if (live && k > t) { over += x; atomicAdd(h + bin, 1u); }
            }
        }
        s.sum2(over, at_t, over, at_t);
        double y;
        int bin;
        const bool live = s.w.arg(key_bits<LOW>(t), y);
        u64 one = LgWeight::whole(s.w.scaled(y, bin));
        if (!live) one = 0;
        if (ties < at_t) at_t = ties;
        const u64 total = over + at_t * one, p64 = __double2ull_rz((double)top_p * 18446744073709551616.0);
        u64 target = __umul64hi(p64, total) + (p64 * total != 0);
        if (target < 1) target = 1;
        if (target > over) ties = min(ties, one ? (target - over + one - 1) / one : ties);
        else {
            // weights of a bin: between those of its borders, half a bin to either side of its number
            u64 c[4], v[4], before;
            int b0, b1;
            s.bins4(h, 1, c);
            #pragma unroll
            for (int j = 0; j < 4; j++) v[j] = c[j] ? c[j] * (u64)__double2ull_ru(exp2(a.shift - (tid * 4 + j - 0.51) / 32.0)) : 0;
            s.first_reaching(v, 0, target, 0, b0, before);
            #pragma unroll
            for (int j = 0; j < 4; j++) v[j] = c[j] ? c[j] * (u64)__double2ull_rd(exp2(a.shift - (tid * 4 + j + 0.51) / 32.0)) : 0;
            s.first_reaching(v, 0, target, 1, b1, before);
            uint32_t klo, khi;
            s.interval(b0, max(b0, b1), t + 1, top_key, klo, khi);
            s.refine(true, target, klo, khi, t, ties);
        }
    }
    // the draw: what each warp's tokens weigh and how many lie at the threshold, then the warp in which the running weight passes the target
    const double floor_w = min_p > 0.0f ? (double)min_p * (double)(1ull << a.shift) : 0.0;
    u64 over = 0, at_t = 0, one;
    {
        double y;
        int bin;
        const bool live = s.w.arg(key_bits<LOW>(t), y);
        const double x = s.w.scaled(y, bin);
        one = live && x >= floor_w ? LgWeight::whole(x) : 0;
    }
    for (int i = s.w0; i < s.w1; i += 128) {
        uint32_t b[4];
        s.fetch4(i + lane * 4, b);
        #pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t k = key_of<LOW>(b[j]);
            at_t += k == t;
            if (!__any_sync(0xffffffffu, k > t)) continue;
            double y;
            int bin;
            const bool live = s.w.arg(b[j], y) && k > t;
            const double x = s.w.scaled(y, bin);
            if (live && x >= floor_w) over += LgWeight::whole(x);
        }
    }
    over = warp_sum_u64(over); at_t = warp_sum_u64(at_t);
    __syncthreads();
    if (lane == 0) { red[warp] = over; red[LG_SAMPLE_WARPS + warp] = at_t; }
    __syncthreads();
    u64 *mine = word + s.at_word;
    if (warp == 0) {
        const u64 x = warp_sum_u64(lane < LG_SAMPLE_WARPS ? red[lane] : 0), y = warp_sum_u64(lane < LG_SAMPLE_WARPS ? red[LG_SAMPLE_WARPS + lane] : 0);
        if (lane == 0) { mine[0] = x; mine[1] = y; }
    }
    cluster_sync_all();
    u64 total = 0, tied = 0, run = 0, end = 0, rank_t = 0;                     // run .. end: of this warp; rank_t: ties before it
    for (uint32_t c = 0; c < ranks; c++) {
        const u64 x = ld_peer_u64(mine, c), y = ld_peer_u64(mine + 1, c);
        if ((int)c == rank) {
            u64 at = total, seen_t = tied;
            for (int i = 0; i <= warp; i++) {
                const u64 left = ties > seen_t ? ties - seen_t : 0, m = red[LG_SAMPLE_WARPS + i];
                run = at; rank_t = seen_t;
                at += red[i] + (m < left ? m : left) * one;
                seen_t += m;
            }
            end = at;
        }
        const u64 left = ties > tied ? ties - tied : 0;
        total += x + (y < left ? y : left) * one;
        tied += y;
    }
    const float u = a.u[row];
    const u64 u64_ = u > 0.0f ? u < 1.0f ? __double2ull_rz((double)u * 18446744073709551616.0) : ~0ull : 0ull;
    const u64 target = __umul64hi(u64_, total);
    if (run <= target && target < end) {
        for (int i = s.w0; i < s.w1; i += 128) {
            uint32_t b[4], eq = 0;
            double x[4];
            u64 v[4], sum = 0;
            s.fetch4(i + lane * 4, b);
            #pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t k = key_of<LOW>(b[j]);
                double y;
                int bin;
                const bool live = s.w.arg(b[j], y);
                x[j] = s.w.scaled(y, bin);
                v[j] = live && k > t && x[j] >= floor_w ? LgWeight::whole(x[j]) : 0;
                eq |= (uint32_t)(k == t) << j;
            }
            const u64 ties_up = warp_scan_u64(__popc(eq), lane);
            u64 rk = rank_t + ties_up - __popc(eq);
            #pragma unroll
            for (int j = 0; j < 4; j++) {
                if (eq >> j & 1) v[j] = rk++ < ties ? one : 0;
                sum += v[j];
            }
            const u64 up = warp_scan_u64(sum, lane);
            const uint32_t hit = __ballot_sync(0xffffffffu, run + up > target);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    u64 at = run + up - sum;
                    int j = 0;
                    while (at + v[j] <= target) at += v[j++];
                    a.token[row] = first + i + lane * 4 + j;
                    if (a.prob) a.prob[row] = (float)(x[j] / (double)total);
                }
                break;
            }
            run += __shfl_sync(0xffffffffu, up, 31);
            rank_t += __shfl_sync(0xffffffffu, ties_up, 31);
        }
    }
    cluster_sync_all();
}
