// lg_paged.cuh -- kernels of a paged K / V cache: the step that hands out pages and slots, the append of rows, the attention of the
// newest rows.  Included by lg_serve.cu.
#pragma once
#include "lg_device.cuh"
#include <cuda_bf16.h>
#include "lg_serve.h"

struct LgPaged {                       // struct lg_paged_cache as the kernels need it
    void *k, *v;
    long long page_stride, row_stride, head_stride;
    int n_pages, page_size, n_kv, hd;
    int max_pages, table_stride;
    int *table, *len, *free_pages, *n_free, *status;
};

__device__ __forceinline__ void paged_raise(const LgPaged &c, int bit) { if (c.status) atomicOr(c.status, bit); }

// Element types.  8 elements at a time: one 16-byte word of a 16-bit type, two of f32.
template <typename T> struct Elem;
template <> struct Elem<float> {
    static __device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
        const float4 a = *(const float4 *)p, b = *(const float4 *)(p + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
    static __device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
        *(float4 *)p = make_float4(x[0], x[1], x[2], x[3]);
        *(float4 *)(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    }
    static __device__ __forceinline__ float get(const float *p) { return *p; }
    static __device__ __forceinline__ float put(float x) { return x; }
};
template <> struct Elem<__half> {
    static __device__ __forceinline__ void load8(const __half *p, float (&x)[8]) {
        const uint4 a = *(const uint4 *)p;
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*(const __half2 *)&w[i]);
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ void store8(__half *p, const float (&x)[8]) {
        uint32_t w[4];
        #pragma unroll
        for (int i = 0; i < 4; i++) { const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]); w[i] = *(const uint32_t *)&h; }
        *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float get(const __half *p) { return __half2float(*p); }
    static __device__ __forceinline__ __half put(float x) { return __float2half_rn(x); }
};
template <> struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&x)[8]) {
        const uint4 a = *(const uint4 *)p;
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
        #pragma unroll
        for (int i = 0; i < 4; i++) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
    }
    static __device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&x)[8]) {
        uint32_t w[4];
        #pragma unroll
        for (int i = 0; i < 4; i++) { const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]); w[i] = *(const uint32_t *)&h; }
        *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float get(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
};

// ---------------------------------------------------------------------------------------------
// the step
// ---------------------------------------------------------------------------------------------
#define LG_STEP_THREADS 1024

struct LgStepArgs {
    LgPaged c;
    int n_req, cap;
    const int *keep, *fresh;           // rows kept (or NULL), new rows
    int *start, *pos, *slot, *req;
};

// Exclusive sum over the block of one number a thread; *total gets the sum of all.
__device__ __forceinline__ long long block_scan(long long v, long long *red, long long *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long s = v;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const long long t = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += t; }
    __syncthreads();
    if (lane == 31) red[warp] = s;
    __syncthreads();
    if (warp == 0) {
        long long w = red[lane];                       // LG_STEP_THREADS / 32 = 32 warps
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const long long t = __shfl_up_sync(0xffffffffu, w, o); if (lane >= o) w += t; }
        red[lane] = w;
    }
    __syncthreads();
    *total = red[31];
    return s - v + (warp ? red[warp - 1] : 0);
}

// What request r asks for: rows kept, new rows, pages held and needed.  false: it does not fit its row of the table.
__device__ __forceinline__ bool step_request(const LgStepArgs &a, int r, int &kept, int &fresh, int &have, int &need) {
    const int ps = a.c.page_size;
    const long long room = (long long)a.c.max_pages * ps;
    const int raw = a.c.len[r];
    const int len = raw < 0 ? 0 : (int)(raw > room ? room : raw);
    if (len != raw) paged_raise(a.c, LG_PAGED_BAD_PAGE);
    kept = a.keep ? min(max(a.keep[r], 0), len) : len;
    fresh = max(a.fresh[r], 0);
    have = (int)(((long long)len + ps - 1) / ps);
    const bool fits = (long long)kept + fresh <= room;
    if (!fits) { kept = len; fresh = 0; }
    need = (int)(((long long)kept + fresh + ps - 1) / ps);
    return fits;
}

// One step: one CTA (a larger grid would have every CTA scan all requests and share the rest; the barrier between reading the old
// state and writing the new one is the block's).  Three sums over the requests decide who is served -- pages, then rows -- and
// where each request's tokens, taken pages and returned pages go; after that every token and page finds its place on its own.
// A request that is not served takes no pages, and neither does any later one that needs some, so the pages taken are the top of the stack in one piece.
__global__ void __launch_bounds__(LG_STEP_THREADS) lg_paged_step_kernel(LgStepArgs a) {
    extern __shared__ int sm[];
    __shared__ long long red[32];
    const int R = a.n_req, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int *start = sm, *pop = start + R + 1, *push = pop + R + 1;       // exclusive sums; push[r] < 0: the request is not served
    const int per = (R + LG_STEP_THREADS - 1) / LG_STEP_THREADS;      // <= 8
    const int r0 = min(R, tid * per), r1 = min(R, r0 + per);
    const int n_free = min(max(*a.c.n_free, 0), a.c.n_pages);
    uint32_t served = 0;
    long long total, sum = 0;
    int kept, fresh, have, need;
    for (int r = r0; r < r1; r++) {
        if (!step_request(a, r, kept, fresh, have, need)) { paged_raise(a.c, LG_PAGED_TOO_LONG); continue; }
        served |= 1u << (r - r0);
        sum += max(0, need - have);
    }
    long long at = block_scan(sum, red, &total);
    sum = 0;
    for (int r = r0; r < r1; r++) {
        if (!(served >> (r - r0) & 1)) continue;
        step_request(a, r, kept, fresh, have, need);
        if (need > have && (at += need - have) > n_free) { served &= ~(1u << (r - r0)); paged_raise(a.c, LG_PAGED_NO_PAGES); continue; }
        sum += fresh;
    }
    at = block_scan(sum, red, &total);
    long long n_tok = 0, n_pop = 0, n_push = 0;
    for (int r = r0; r < r1; r++) {
        if (!(served >> (r - r0) & 1)) continue;
        step_request(a, r, kept, fresh, have, need);
        if (fresh && (at += fresh) > a.cap) { served &= ~(1u << (r - r0)); paged_raise(a.c, LG_PAGED_NO_ROWS); continue; }
        n_tok += fresh; n_pop += max(0, need - have); n_push += max(0, have - need);
    }
    long long all_tok, all_pop, all_push;
    n_tok = block_scan(n_tok, red, &all_tok);
    n_pop = block_scan(n_pop, red, &all_pop);
    n_push = block_scan(n_push, red, &all_push);
    for (int r = r0; r < r1; r++) {
        const bool ok = served >> (r - r0) & 1;
        start[r] = (int)n_tok; pop[r] = (int)n_pop; push[r] = ok ? (int)n_push : -1;
        a.start[r] = (int)n_tok;
        if (!ok) continue;
        step_request(a, r, kept, fresh, have, need);
        n_tok += fresh; n_pop += max(0, need - have); n_push += max(0, have - need);
    }
    if (tid == 0) { start[R] = (int)all_tok; a.start[R] = (int)all_tok; }
    __syncthreads();
    const int ps = a.c.page_size;
    // tokens: the request whose rows hold row i, its place, and the page there -- from the table, or from the stack if this step takes it
    for (int i = tid; i < a.cap; i += LG_STEP_THREADS) {
        int pos = -1, slot = -1, req = -1;
        if (i < (int)all_tok) {
            int lo = 0, hi = R;                        // start[lo] <= i < start[hi]
            while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (start[mid] <= i) lo = mid; else hi = mid; }
            step_request(a, lo, kept, fresh, have, need);
            req = lo;
            pos = kept + i - start[lo];
            const int pg = pos / ps;
            const int page = pg < have ? a.c.table[(size_t)lo * a.c.table_stride + pg] : a.c.free_pages[n_free - 1 - (pop[lo] + pg - have)];
            if (page >= 0 && page < a.c.n_pages) slot = page * ps + pos % ps;
            else paged_raise(a.c, LG_PAGED_BAD_PAGE);
        }
        if (a.pos) a.pos[i] = pos;
        if (a.slot) a.slot[i] = slot;
        if (a.req) a.req[i] = req;
    }
    // pages taken go into the tables, behind every entry that a token above reads
    for (int r = warp; r < R; r += LG_STEP_THREADS / 32) {
        if (push[r] < 0) continue;
        step_request(a, r, kept, fresh, have, need);
        for (int p = have + lane; p < need; p += 32) a.c.table[(size_t)r * a.c.table_stride + p] = a.c.free_pages[n_free - 1 - (pop[r] + p - have)];
    }
    __syncthreads();
    // pages returned go onto the stack, over what was taken from it; lengths
    const int base = n_free - (int)all_pop;
    for (int r = warp; r < R; r += LG_STEP_THREADS / 32) {
        if (push[r] < 0) continue;
        step_request(a, r, kept, fresh, have, need);
        __syncwarp();
        for (int p = need + lane; p < have; p += 32) {
            const long long to = base + all_push - 1 - (push[r] + (long long)p - need);
            int *e = &a.c.table[(size_t)r * a.c.table_stride + p];
            if (to < a.c.n_pages && *e >= 0 && *e < a.c.n_pages) a.c.free_pages[to] = *e;
            else paged_raise(a.c, LG_PAGED_BAD_PAGE);
            *e = -1;
        }
        if (lane == 0) a.c.len[r] = kept + fresh;
    }
    if (tid == 0) *a.c.n_free = (int)min((long long)a.c.n_pages, base + all_push);
}

// ---------------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------------
struct LgAppendArgs {
    LgPaged c;
    const void *k, *v;
    long long ld_k, ld_v;
    int n, wide;                       // wide: rows can be read 16 bytes at a time
    const int *slot;
};

// A thread moves 8 elements of a row at a time, K's then V's; bound by the bytes in and out.
template <typename TI, typename TC> __global__ void __launch_bounds__(256) lg_paged_append_kernel(LgAppendArgs a) {
    const int per_head = a.c.hd >> 3, half = per_head * a.c.n_kv, units = 2 * half;
    const long long all = (long long)a.n * units;
    const long long n_slots = (long long)a.c.n_pages * a.c.page_size;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (long long)gridDim.x * blockDim.x) {
        const int row = (int)(i / units);
        int u = (int)(i - (long long)row * units);
        const bool is_v = u >= half;
        if (is_v) u -= half;
        const int slot = a.slot[row];
        if (slot < 0 || slot >= n_slots) { if (slot != -1) paged_raise(a.c, LG_PAGED_BAD_SLOT); continue; }
        const int page = slot / a.c.page_size, head = u / per_head;
        const TI *src = (const TI *)(is_v ? a.v : a.k) + (is_v ? a.ld_v : a.ld_k) * row + u * 8;
        TC *dst = (TC *)(is_v ? a.c.v : a.c.k) + (long long)page * a.c.page_stride + (long long)(slot - page * a.c.page_size) * a.c.row_stride +
                  head * a.c.head_stride + (u - head * per_head) * 8;
        float x[8];
        if (a.wide) Elem<TI>::load8(src, x);
        else {
            #pragma unroll
            for (int j = 0; j < 8; j++) x[j] = Elem<TI>::get(src + j);
        }
        Elem<TC>::store8(dst, x);
    }
}

// ---------------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------------
struct LgPagedAttnArgs {
    LgPaged c;
    const void *q; void *out;
    long long ld_q, ld_out;
    int n_req, n_new, n_rows, n_heads, window;
    float scale;                       // times log2(e)
    const int *start;
};

// The block of rows of request r: first row, rows to compute, rows it has.
__device__ __forceinline__ void paged_rows(const LgPagedAttnArgs &a, int r, int &first, int &m, int &held) {
    if (!a.start) { first = r * a.n_new; m = held = a.n_new; return; }
    first = a.start[r];
    const long long d = (long long)a.start[r + 1] - first;
    held = (int)(d < 0 ? 0 : d > 0x7fffffff ? 0x7fffffff : d);
    if (d < 0 || first < 0 || (long long)first + held > a.n_rows) { held = 0; if (d) paged_raise(a.c, LG_PAGED_BAD_ROWS); }
    m = min(held, a.n_new);
    if (m < held) paged_raise(a.c, LG_PAGED_BAD_ROWS);
}
__device__ __forceinline__ int paged_len(const LgPagedAttnArgs &a, int r) {
    const int len = a.c.len[r];
    const long long room = (long long)a.c.max_pages * a.c.page_size;
    if (len < 0 || len > room) { paged_raise(a.c, LG_PAGED_BAD_PAGE); return len < 0 ? 0 : (int)room; }
    return len;
}

// One query row and head per CTA (grid: rows of a block, heads, requests), a key per warp at a time, softmax with a running maximum and sum:
//   m' = max(m, s),  l' = l 2^(m - m') + 2^(s - m'),  o' = o 2^(m - m') + 2^(s - m') v
// Sums in f32.  The queries of a KV head each read its rows on their own.
#define LG_PATTN_WARPS 8
template <typename TQ, typename TC> __global__ void __launch_bounds__(LG_PATTN_WARPS * 32) lg_paged_attn_rows_kernel(LgPagedAttnArgs a) {
    __shared__ float po[LG_PATTN_WARPS][512], pm[LG_PATTN_WARPS], pl[LG_PATTN_WARPS];
    const int t = blockIdx.x, h = blockIdx.y, r = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int first, m, held;
    paged_rows(a, r, first, m, held);
    if (t >= m) return;
    const int hd = a.c.hd, units = hd >> 3, ps = a.c.page_size;
    const int pos = paged_len(a, r) - held + t;
    const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const long long head = (long long)(h / (a.n_heads / a.c.n_kv)) * a.c.head_stride;
    const TQ *q = (const TQ *)a.q + (long long)(first + t) * a.ld_q + (long long)h * hd;
    float qv[2][8], o[2][8] = {}, x[8], mx = -INFINITY, l = 0.0f;
    #pragma unroll
    for (int j = 0; j < 2; j++)
        #pragma unroll
        for (int i = 0; i < 8; i++) qv[j][i] = lane + 32 * j < units ? Elem<TQ>::get(q + (lane + 32 * j) * 8 + i) : 0.0f;
    for (int key = lo + warp; key <= pos; key += LG_PATTN_WARPS) {
        const int page = a.c.table[(size_t)r * a.c.table_stride + key / ps];
        if (page < 0 || page >= a.c.n_pages) { paged_raise(a.c, LG_PAGED_BAD_PAGE); continue; }
        const long long at = (long long)page * a.c.page_stride + (long long)(key % ps) * a.c.row_stride + head;
        float s = 0.0f;
        #pragma unroll
        for (int j = 0; j < 2; j++)
            if (lane + 32 * j < units) {
                Elem<TC>::load8((const TC *)a.c.k + at + (lane + 32 * j) * 8, x);
                #pragma unroll
                for (int i = 0; i < 8; i++) s += qv[j][i] * x[i];
            }
        s = warp_sum(s) * a.scale;
        const float m2 = fmaxf(mx, s), f = mx == -INFINITY ? 0.0f : exp2f(mx - m2), p = s == -INFINITY ? 0.0f : exp2f(s - m2);
        mx = m2; l = l * f + p;
        #pragma unroll
        for (int j = 0; j < 2; j++)
            if (lane + 32 * j < units) {
                Elem<TC>::load8((const TC *)a.c.v + at + (lane + 32 * j) * 8, x);
                #pragma unroll
                for (int i = 0; i < 8; i++) o[j][i] = o[j][i] * f + p * x[i];
            }
    }
    #pragma unroll
    for (int j = 0; j < 2; j++)
        if (lane + 32 * j < units)
            #pragma unroll
            for (int i = 0; i < 8; i++) po[warp][(lane + 32 * j) * 8 + i] = o[j][i];
    if (lane == 0) { pm[warp] = mx; pl[warp] = l; }
    __syncthreads();
    float top = -INFINITY;
    for (int w = 0; w < LG_PATTN_WARPS; w++) top = fmaxf(top, pm[w]);
    float sum = 0.0f, f[LG_PATTN_WARPS];
    #pragma unroll
    for (int w = 0; w < LG_PATTN_WARPS; w++) { f[w] = pl[w] == 0.0f ? 0.0f : exp2f(pm[w] - top); sum += pl[w] * f[w]; }
    TQ *out = (TQ *)a.out + (long long)(first + t) * a.ld_out + (long long)h * hd;
    for (int d = threadIdx.x; d < hd; d += blockDim.x) {
        float y = 0.0f;
        #pragma unroll
        for (int w = 0; w < LG_PATTN_WARPS; w++) y += po[w][d] * f[w];
        out[d] = Elem<TQ>::put(sum == 0.0f ? 0.0f : y / sum);
    }
}
