// lg_paged.cuh -- kernels of a paged K / V cache: the step that hands out pages and slots, the append of rows, the attention of the
// newest rows.  Included by lg_serve.cu.
#pragma once
#include "lg_device.cuh"
#include <cuda_bf16.h>
#include <type_traits>
#include "lg_serve.h"

struct LgPaged {                       // struct lg_paged_cache as the kernels need it
    void *k, *v;
    long long page_stride, row_stride, head_stride;
    int n_pages, page_size, n_kv, hd;
    int max_pages, table_stride;
    int *table, *len, *free_pages, *n_free, *status;
};

// Where a row of a page begins, for one head, in elements; -1: there is no such row.
__host__ __device__ __forceinline__ long long paged_place(const LgPaged &c, int page, int row, int head) {
    if (page < 0 || page >= c.n_pages || row < 0 || row >= c.page_size || head < 0 || head >= c.n_kv) return -1;
    return (long long)page * c.page_stride + (long long)row * c.row_stride + (long long)head * c.head_stride;
}
__device__ __forceinline__ void paged_raise(const LgPaged &c, int bit) { if (c.status) atomicOr(c.status, bit); }

// Element types.  store8: 8 elements rounded into a 16-byte word.
template <typename T> struct Elem;
template <> struct Elem<float> {
    static __device__ __forceinline__ float get(const float *p) { return *p; }
    static __device__ __forceinline__ float put(float x) { return x; }
};
template <> struct Elem<__half> {
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

// Exclusive sums over the block of three numbers a thread, in place; total: of all threads.
__device__ __forceinline__ void block_scan3(long long (&v)[3], long long (&total)[3], long long (*red)[3]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long s[3];
    #pragma unroll
    for (int k = 0; k < 3; k++) {
        s[k] = v[k];
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const long long t = __shfl_up_sync(0xffffffffu, s[k], o); if (lane >= o) s[k] += t; }
    }
    __syncthreads();
    if (lane == 31) { red[warp][0] = s[0]; red[warp][1] = s[1]; red[warp][2] = s[2]; }
    __syncthreads();
    #pragma unroll
    for (int k = 0; k < 3; k++) {
        long long w = red[lane][k];                    // LG_STEP_THREADS / 32 = 32 warps
        const long long own = w;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const long long t = __shfl_up_sync(0xffffffffu, w, o); if (lane >= o) w += t; }
        total[k] = __shfl_sync(0xffffffffu, w, 31);
        v[k] = s[k] - v[k] + __shfl_sync(0xffffffffu, w - own, warp);
    }
}

// One step, in one CTA or in a cluster of them: each CTA adds up all requests (a thread has PER in a row) and takes a share of the tokens, tables and
// returned pages; what the old state is read for lies before the cluster's barrier, what overwrites it behind.  Sums over the requests -- pages
// taken, tokens, pages returned -- say where each request's things go, and every token and page then finds its place on its own.  Where
// pages or rows do not suffice, two more sums decide who is served: a request that is not takes no pages, and neither does any later one
// that needs some, so the pages taken are always the top of the stack in one piece.  Bound by latency: a step and its roll-back
// take 10.3 us for 48 requests, 23 us for 2048 with 40576 tokens (one CTA, with the requests looked up again for every token: 274).
template <int PER> __global__ void __launch_bounds__(LG_STEP_THREADS, 1) lg_paged_step_kernel(LgStepArgs a) {
    extern __shared__ int sm[];
    __shared__ long long red[32][3];
    const int R = a.n_req, tid = threadIdx.x, lane = tid & 31, ps = a.c.page_size;
    uint32_t ranks;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
    const int rank = (int)cluster_rank();
    int *start = sm, *pop = start + R + 1, *kept_of = pop + R, *have_of = kept_of + R;
    const long long room = (long long)a.c.max_pages * ps;
    const int n_free = min(max(*a.c.n_free, 0), a.c.n_pages);
    int kept[PER], fresh[PER], have[PER], need[PER];
    long long sum[3] = {0, 0, 0}, all[3];
    uint32_t served = 0;
    #pragma unroll
    for (int q = 0; q < PER; q++) {
        const int r = tid * PER + q;
        kept[q] = fresh[q] = have[q] = need[q] = 0;
        if (r >= R) continue;
        const int raw = a.c.len[r], len = raw < 0 ? 0 : (int)(raw > room ? room : raw);
        if (len != raw) paged_raise(a.c, LG_PAGED_BAD_PAGE);
        kept[q] = a.keep ? min(max(a.keep[r], 0), len) : len;
        fresh[q] = max(a.fresh[r], 0);
        have[q] = (int)(((long long)len + ps - 1) / ps);
        if ((long long)kept[q] + fresh[q] > room) { kept[q] = len; fresh[q] = 0; paged_raise(a.c, LG_PAGED_TOO_LONG); }
        else served |= 1u << q;
        need[q] = (int)(((long long)kept[q] + fresh[q] + ps - 1) / ps);
    }
    auto add_up = [&]() {
        sum[0] = sum[1] = sum[2] = 0;
        #pragma unroll
        for (int q = 0; q < PER; q++)
            if (served >> q & 1) { sum[0] += max(0, need[q] - have[q]); sum[1] += fresh[q]; sum[2] += max(0, have[q] - need[q]); }
        block_scan3(sum, all, red);
    };
    add_up();
    if (all[0] > n_free || all[1] > a.cap) {
        long long at = sum[0];
        #pragma unroll
        for (int q = 0; q < PER; q++)
            if ((served >> q & 1) && need[q] > have[q] && (at += need[q] - have[q]) > n_free) { served &= ~(1u << q); paged_raise(a.c, LG_PAGED_NO_PAGES); }
        add_up();
        at = sum[1];
        #pragma unroll
        for (int q = 0; q < PER; q++)
            if ((served >> q & 1) && fresh[q] && (at += fresh[q]) > a.cap) { served &= ~(1u << q); paged_raise(a.c, LG_PAGED_NO_ROWS); }
        add_up();
    }
    long long at_pop = sum[0], at_tok = sum[1], at_push = sum[2];
    int pop0[PER], push0[PER];
    #pragma unroll
    for (int q = 0; q < PER; q++) {
        const int r = tid * PER + q;
        pop0[q] = (int)at_pop; push0[q] = (int)at_push;
        if (r >= R) continue;
        start[r] = (int)at_tok; pop[r] = (int)at_pop; kept_of[r] = kept[q]; have_of[r] = have[q];
        if (rank == 0) a.start[r] = (int)at_tok;
        if (served >> q & 1) { at_pop += max(0, need[q] - have[q]); at_tok += fresh[q]; at_push += max(0, have[q] - need[q]); }
    }
    if (tid == 0) { start[R] = (int)all[1]; if (rank == 0) a.start[R] = (int)all[1]; }
    __syncthreads();
    // tokens: the request whose rows hold row i, its place, and the page there -- from the table, or from the stack if this step takes it
    const long long rows = a.pos || a.slot || a.req ? a.cap : all[1];         // (at most cap)
    for (long long row = rank * LG_STEP_THREADS + tid; row < rows; row += (long long)ranks * LG_STEP_THREADS) {
        const int i = (int)row;
        int pos = -1, slot = -1, req = -1;
        if (i < (int)all[1]) {
            int lo = 0, hi = R;                        // start[lo] <= i < start[hi]
            while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (start[mid] <= i) lo = mid; else hi = mid; }
            req = lo;
            pos = kept_of[lo] + i - start[lo];
            const int pg = pos / ps, had = have_of[lo];
            const int page = pg < had ? a.c.table[(size_t)lo * a.c.table_stride + pg] : a.c.free_pages[n_free - 1 - (pop[lo] + pg - had)];
            if (page >= 0 && page < a.c.n_pages) slot = page * ps + pos - pg * ps;
            else paged_raise(a.c, LG_PAGED_BAD_PAGE);
        }
        if (a.pos) a.pos[i] = pos;
        if (a.slot) a.slot[i] = slot;
        if (a.req) a.req[i] = req;
    }
    // pages of a request, by its thread, or by the warp where they are many
    auto pages = [&](int n, auto &&one, auto &&give) {
        uint32_t many = __ballot_sync(0xffffffffu, n > 4);
        if (n <= 4) for (int p = 0; p < n; p++) one(p);
        while (many) {
            const int who = __ffs(many) - 1;
            many &= many - 1;
            give(who, __shfl_sync(0xffffffffu, n, who));
        }
    };
    // those taken go into the tables, behind every entry that a token above reads
    #pragma unroll
    for (int q = 0; q < PER; q++) {
        const int r = tid * PER + q, n = (served >> q & 1) && r % (int)ranks == rank ? max(0, need[q] - have[q]) : 0;
        const int from = n_free - 1 - pop0[q];
        int *row = a.c.table + (size_t)r * a.c.table_stride + have[q];
        pages(n, [&](int p) { row[p] = a.c.free_pages[from - p]; }, [&](int who, int count) {
            int *to = (int *)__shfl_sync(0xffffffffu, (unsigned long long)row, who);
            const int f = __shfl_sync(0xffffffffu, from, who);
            for (int p = lane; p < count; p += 32) to[p] = a.c.free_pages[f - p];
        });
    }
    cluster_sync_all();
    // those given up go onto the stack, over what was taken from it, the last one first; lengths
    const int base = n_free - (int)all[0];
    auto back = [&](int *e, long long to) {
        const bool page = *e >= 0 && *e < a.c.n_pages;                        // what is none has a place on the stack all the same, and must not leave a page there
        if (to < a.c.n_pages) a.c.free_pages[to] = page ? *e : -1;            // that another request took from it
        if (!page || to >= a.c.n_pages) paged_raise(a.c, LG_PAGED_BAD_PAGE);
        *e = -1;
    };
    #pragma unroll
    for (int q = 0; q < PER; q++) {
        const int r = tid * PER + q;
        const bool own = (served >> q & 1) && r % (int)ranks == rank;
        const int n = own ? max(0, have[q] - need[q]) : 0;
        const long long top = base + all[2] - 1 - push0[q];
        int *row = a.c.table + (size_t)r * a.c.table_stride + need[q];
        pages(n, [&](int p) { back(row + p, top - p); }, [&](int who, int count) {
            int *e = (int *)__shfl_sync(0xffffffffu, (unsigned long long)row, who);
            const long long t = __shfl_sync(0xffffffffu, top, who);
            for (int p = lane; p < count; p += 32) back(e + p, t - p);
        });
        if (own) a.c.len[r] = kept[q] + fresh[q];
    }
    if (rank == 0 && tid == 0) *a.c.n_free = (int)min((long long)a.c.n_pages, base + all[2]);
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

#define LG_APPEND_THREADS 256

// Eight elements on their way from a row to the cache: as they are, or rounded.
template <typename TI, typename TC> struct Eight {
    float x[8];
    __device__ __forceinline__ void load(const TI *p, bool wide) {
        if (wide) {
            const float4 a = __ldcs((const float4 *)p), b = __ldcs((const float4 *)(p + 4));
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        } else {
            #pragma unroll
            for (int j = 0; j < 8; j++) x[j] = p[j];
        }
    }
    __device__ __forceinline__ void store(TC *p) const { Elem<TC>::store8(p, x); }
};
template <typename T> struct Eight<T, T> {
    uint4 x[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *p, bool wide) {
        if (wide) {
            #pragma unroll
            for (int j = 0; j < (int)sizeof(T) / 2; j++) x[j] = __ldcs((const uint4 *)p + j);
        } else {
            T *e = (T *)x;
            #pragma unroll
            for (int j = 0; j < 8; j++) e[j] = p[j];
        }
    }
    __device__ __forceinline__ void store(T *p) const {
        #pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; j++) ((uint4 *)p)[j] = x[j];
    }
};

// A thread moves 8 elements of a row at a time, two such pieces under way, K's and V's; a CTA has one row, or as many whole ones as its threads cover, and
// goes on to the next.  Rows of one type are not looked at.  Bound by the bytes in and out: 8191 rows of 8 heads of 256 in bf16 take 24 us (134 MB, three sets in turn; a division a piece and
// conversion through f32 cost 30), 48 rows 2.1 us.
template <typename TI, typename TC> __global__ void __launch_bounds__(LG_APPEND_THREADS) lg_paged_append_kernel(LgAppendArgs a) {
    const int per_head = a.c.hd >> 3, half = per_head * a.c.n_kv, units = 2 * half;
    const int here = units < LG_APPEND_THREADS ? (int)threadIdx.x / units : 0, rows = units < LG_APPEND_THREADS ? LG_APPEND_THREADS / units : 1;
    const int u0 = (int)threadIdx.x - here * units;
    const bool packed = a.c.head_stride == a.c.hd;
    const int n_slots = a.c.n_pages * a.c.page_size;
    if (here >= rows) return;
    for (long long row = (long long)blockIdx.x * rows + here; row < a.n; row += (long long)gridDim.x * rows) {
        const int slot = a.slot[row];
        const TI *k = (const TI *)a.k + a.ld_k * row, *v = (const TI *)a.v + a.ld_v * row;
        for (int u = u0; u < units; u += 2 * LG_APPEND_THREADS) {
            Eight<TI, TC> x[2];                                               // on their way before the slot is looked at
            #pragma unroll
            for (int q = 0; q < 2; q++) {
                const int w = u + q * LG_APPEND_THREADS;
                if (w < units) x[q].load(w < half ? k + w * 8 : v + (w - half) * 8, a.wide);
            }
            if (slot < 0 || slot >= n_slots) { if (slot != -1) paged_raise(a.c, LG_PAGED_BAD_SLOT); break; }
            const int page = slot / a.c.page_size;
            const long long to = paged_place(a.c, page, slot - page * a.c.page_size, 0);
            #pragma unroll
            for (int q = 0; q < 2; q++) {
                const int w = u + q * LG_APPEND_THREADS, c = w < half ? w : w - half;
                long long at = to + c * 8;
                if (!packed) { const int head = c / per_head; at += head * (a.c.head_stride - a.c.hd); }
                if (w < units) x[q].store((TC *)(w < half ? a.c.k : a.c.v) + at);
            }
        }
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
    int gqa, group_rows;               // query heads of a KV head, query rows of an item
    int whole;                         // pages are whole slices
    float *part; float2 *part_ml;      // [CTA][2][query row of an item]: output over the part's keys; maximum and sum
    int4 *jobs;                        // [CTA]: the item that it leaves unfinished (first row of the request, KV head, last CTA, first of its rows and their number), or -1
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

// The work is a line of slices of 16 keys: request by request, KV head by KV head, group of 8 NT query rows by group (an item).  Every CTA of a
// persistent grid takes a stretch of equal length of that line, so ragged lengths cost nothing; an item that one stretch holds is written at once,
// of one that several stretches share each leaves (max, sum, output), and lg_paged_merge_kernel adds those in their order.
// (Spans fixed by a request's own length took 876 us for 96 requests of 1.6K to 16K rows where this took 539, one set of inputs replayed: short spans cost
// merges, and about as many items as CTAs leave SMs idle: 153 us for two requests of 120000 rows where this took 97.)
//
// Inside a CTA every warp works alone: it takes 16 keys (a slice) at a time, brings K and V in with 16-byte asynchronous copies through a ring
// of U units of its own (a unit: 16 rows of K or of V; rows that no query may see are filled with zeros and never read), so the loop has no block barrier and
// runs ahead across items.  Both products have the keys / head dims on the 16-row side and 8 queries as columns:
//   S^T (16 keys x 8) = K Q^T, softmax with a running maximum per column in the accumulator's own lanes, O^T (16 dims x 8) += V^T P^T,
// P^T turned from accumulator order into operand order by movmatrix.
//
// Numerics.  An f32 query enters as a sum of 16-bit parts (f16: 2 parts behind a power of two per row, 22 bits; bf16: 3, 24 bits), P as 2 parts (3 where the
// answer is f32 and the cache bf16; 2 of bf16 are 16 bits of a weight, off by 2^-18 of it at most, for an answer of 8 bits: the third takes 5 % more time
// over many calls of 96 requests up to 16383 rows); P carries a factor 2^15 in f16 so that weights down to 2^-29 of the largest stay normal numbers.  Rows of an
// f32 cache are split in registers into three bf16 parts (24 bits); of the nine products of parts the six that reach the last bits of an f32 are
// computed.  The matrix instructions' additions cut off, always towards zero.  So a slice's products are added to the outputs outside of them, with rounding to
// nearest and the factor of a moved maximum in the same operation: over 131072 f16 rows of one sign a sum inside took 8.6e-5 from the result (0.18 of half
// a step), this 1.7e-6; it costs nothing where copies are the bound, 15 % with 16-bit heads of 512, 4 to 7 % with 16 query rows a KV head and more.  And products
// of lower parts are added up before the first ones or apart from them: f32 caches are 1.3e-7 to 6e-7 (norm) off the 64-bit answer, with all in one sum
// 3e-7 to 1.8e-6.  Everything else is f32.  Outputs that are not finite are computed again, see paged_key_by_key.
#define LG_PA_MAX_CTAS 296             // two per SM
#define LG_PA_ITEM_COST 6              // of an item beside its slices, in slices: queries in, warps' results together, rows out
#define LG_PA_MIN_STRETCH 8

template <typename T> __device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { mma_f16(c, a, b0, b1); }
template <> __device__ __forceinline__ void mma_16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two numbers rounded and packed, the first in the low half; x and y keep what the rounding left over.
template <typename T> __device__ __forceinline__ uint32_t split2(float &x, float &y);
template <> __device__ __forceinline__ uint32_t split2<__half>(float &x, float &y) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    x -= f.x; y -= f.y;
    return *(const uint32_t *)&h;
}
template <> __device__ __forceinline__ uint32_t split2<__nv_bfloat16>(float &x, float &y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const uint32_t w = *(const uint32_t *)&h;
    x -= __uint_as_float(w << 16); y -= __uint_as_float(w & 0xFFFF0000u);
    return w;
}
__device__ __forceinline__ float lds_f(uint32_t p) { float v; asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(p)); return v; }
__device__ __forceinline__ float2 lds_f2(uint32_t p) { float2 v; asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(p)); return v; }
__device__ __forceinline__ uint16_t lds_u16(uint32_t p) { uint16_t v; asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(p)); return v; }
// One element of a cache in shared memory
template <typename T> __device__ __forceinline__ float lds_elem(uint32_t p);
template <> __device__ __forceinline__ float lds_elem<float>(uint32_t p) { return lds_f(p); }
template <> __device__ __forceinline__ float lds_elem<__half>(uint32_t p) { return __half2float(__ushort_as_half(lds_u16(p))); }
template <> __device__ __forceinline__ float lds_elem<__nv_bfloat16>(uint32_t p) { return __uint_as_float((uint32_t)lds_u16(p) << 16); }
// A factor that is not 0, so that inf times it is inf; NaN stays
__device__ __forceinline__ float above_zero(float x) { return x < 1.17549435e-38f ? 1.17549435e-38f : x; }
// x = x f + a, y = y g + b in one instruction
__device__ __forceinline__ void fma2(float &x, float &y, float f, float g, float a, float b) {
    asm("{\n.reg .b64 o, f, a;\nmov.b64 o, {%0, %1};\nmov.b64 f, {%2, %3};\nmov.b64 a, {%4, %5};\nfma.rn.f32x2 o, o, f, a;\nmov.b64 {%0, %1}, o;\n}"
        : "+f"(x), "+f"(y) : "f"(f), "f"(g), "f"(a), "f"(b));
}
__device__ __forceinline__ uint32_t movm(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// 16 bytes from global memory, or 16 zero bytes without a read
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void *src, bool read) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

// A request as the walk over items sees it.
struct LgReq {
    int first, m, held, len;           // rows, see paged_rows
    int groups;                        // of query rows, per KV head
    int s0, n_sl;                      // first slice, slices
};
__device__ __forceinline__ LgReq paged_request(const LgPagedAttnArgs &a, int r) {
    LgReq q;
    paged_rows(a, r, q.first, q.m, q.held);
    q.len = paged_len(a, r);
    q.groups = (q.m * a.gqa + a.group_rows - 1) / a.group_rows;
    // keys lo .. hi-1 are seen by some row
    const int hi = max(0, q.len - q.held + q.m), lo = a.window > 0 ? max(0, q.len - q.held - a.window + 1) : 0;
    q.s0 = min(lo, hi) >> 4;
    q.n_sl = ((hi + 15) >> 4) - q.s0;
    return q;
}
// Places of an item in the line: its slices and a cost of its own, or, where short stretches suffice (pad), whole stretches
template <int W> __device__ __forceinline__ int paged_weight(const LgReq &q, bool pad) {
    constexpr int least = (LG_PA_MIN_STRETCH + W - 1) / W * W;
    return pad ? max(1, (q.n_sl + least - 1) / least) * least : q.n_sl + LG_PA_ITEM_COST;
}

// The walk of one CTA over the items that begin before the end of its stretch: places 0 .. length-1, the item's beginning at `at` (below 0: another stretch has
// its first slices).
template <int W> struct LgWalk {
    LgReq q;
    int r, hg, at;                     // request, KV head * groups + group
    __device__ __forceinline__ bool valid(const LgPagedAttnArgs &a, int length) const { return r < a.n_req && at < length; }
    __device__ __forceinline__ int begin() const { return max(-at, 0); }                                   // the item's slices in the stretch
    __device__ __forceinline__ int end(int length) const { return min(length - at, q.n_sl); }
    __device__ __forceinline__ void next(const LgPagedAttnArgs &a, int length, bool pad) {
        at += paged_weight<W>(q, pad);
        hg++;
        while (r < a.n_req && hg >= q.groups * a.c.n_kv) {                    // past requests without rows
            if (++r < a.n_req) {
                if (at < length) { q = paged_request(a, r); hg = 0; } else r = a.n_req;
            }
        }
    }
};

template <typename TQ, typename TC, int HD, int NT> struct LgPagedTile {
    typedef typename std::conditional<std::is_same<TC, __half>::value, __half, __nv_bfloat16>::type TM;      // the matrix instructions' type
    static constexpr bool SAME16 = sizeof(TQ) == 2, F32 = sizeof(TC) == 4;    // 16-bit queries; f32 cache
    static constexpr bool F16 = std::is_same<TC, __half>::value;
    static constexpr int NQ = SAME16 ? 1 : F16 ? 2 : 3;                       // parts of a query
    static constexpr int NP = SAME16 || F16 ? 2 : 3;                          // parts of a weight
    static constexpr bool LONG = sizeof(TQ) == 4 && HD > 128;                 // f32 answers: scores added up with rounding to nearest too, every 128 dims
    static constexpr int KS = HD / 16;
    static constexpr int ROWS = 8 * NT;
    static constexpr int ROW = HD * (int)sizeof(TC), UNIT = 16 * ROW, CHUNKS = ROW / 16;
    // Chunk of 16 bytes that a row's chunk c lies in.  16-bit rows: eight rows' chunks in the eight 16-byte columns (ldmatrix); 32-bit rows: pairs of chunks so
    // that neither rows g .. g + 3 (K) nor rows 0, 2, 4, 6 (V) of a column meet in a bank.
    static __device__ __forceinline__ int place(int row, int c) { return F32 ? c ^ (((row ^ (row >> 2)) & 3) << 1) : c ^ (row & 7); }
    static constexpr int LDB = HD + 4;                                        // floats from row to row of the merge buffer: no bank conflicts
    static constexpr bool QREG = (NT * NQ * 2 + NT * 4) * KS <= 160;          // queries stay in registers beside the outputs
    static constexpr bool OWN = UNIT >= ROWS * HD * 4;                        // a warp's outputs fit the ring's free unit on their way to the others'
    static constexpr int Q_BYTES = NT * NQ * KS * 32 * 8, BUF_BYTES = OWN ? 0 : ROWS * LDB * 4;
    static constexpr int SHARED = QREG ? (Q_BYTES > BUF_BYTES ? Q_BYTES : BUF_BYTES) : Q_BYTES + BUF_BYTES;   // in registers they need the room only on the way
    static constexpr int fixed(int w) { return SHARED + 2 * w * ROWS * 8 + ROWS * 4 + 144 + w * 17 * 4; }
    // Two CTAs of 4 warps per SM where three units a warp fit (one merges while the other streams), else one of as many warps as fit
    static constexpr int CTAS = fixed(4) + 12 * UNIT <= 115712 ? 2 : 1;
    static constexpr int ROOM = CTAS == 2 ? 115712 : 232448;
    static constexpr int W = CTAS == 2 ? 4 : fixed(8) + 24 * UNIT <= ROOM ? 8 : fixed(6) + 18 * UNIT <= ROOM ? 6 : fixed(4) + 12 * UNIT <= ROOM ? 4 : fixed(3) + 9 * UNIT <= ROOM ? 3 : 2;
    static constexpr int U0 = (ROOM - fixed(W)) / (W * UNIT);
    static constexpr int U = U0 > 8 ? 8 : U0;
    static constexpr int SMEM = fixed(W) + W * U * UNIT;
    static_assert(U >= 2, "a unit in use and one on its way");
};

// 16 rows of K or V into a unit; lane i (and i + 16) knows where row i lies, in bytes, bit i of `there` whether it is read
template <typename P> __device__ __forceinline__ void paged_copy_unit(const void *from, uint32_t dst, long long place, uint32_t there, int row_chunks, int lane) {
    const unsigned char *base = (const unsigned char *)from;
    #pragma unroll
    for (int i = 0; i < P::CHUNKS / 2; i++) {                                 // 32 chunks of 16 bytes at a time
        const int idx = i * 32 + lane, row = idx / P::CHUNKS, c = idx % P::CHUNKS;
        const long long off = __shfl_sync(0xffffffffu, place, row);
        const bool rd = (there >> row & 1) && c < row_chunks;
        cp_async16_or_zero(dst + row * P::ROW + (P::place(row, c) << 4), rd ? base + off + c * 16 : base, rd);
    }
}
// Scores of a slice whose K lies at `at`; query(i): fragment i of the queries
template <typename P, int NT, typename Q> __device__ __forceinline__ void paged_scores(uint32_t at, int lane, Q &&query, float (&x)[NT][4]) {
    const int g = lane >> 2, t4 = lane & 3;
    // chains of products: those of the first parts in one, as each addition to a large sum cuts off, the others in one (f32 caches: two) of their own
    constexpr int CH = P::F32 ? 3 : 2;
    float sc[NT][CH][4];
    #pragma unroll
    for (int nt = 0; nt < NT; nt++)
        #pragma unroll
        for (int c = 0; c < CH; c++) sc[nt][c][0] = sc[nt][c][1] = sc[nt][c][2] = sc[nt][c][3] = 0.0f;
    auto total = [&](int nt, int j) { return P::F32 ? sc[nt][0][j] + (sc[nt][1][j] + sc[nt][CH - 1][j]) : sc[nt][0][j] + sc[nt][1][j]; };
    float sum[P::LONG ? NT : 1][4];
    if (P::LONG) {
        #pragma unroll
        for (int nt = 0; nt < NT; nt++) sum[nt][0] = sum[nt][1] = sum[nt][2] = sum[nt][3] = 0.0f;
    }
    #pragma unroll
    for (int ks = 0; ks < P::KS; ks++) {
        uint32_t k4[P::F32 ? 3 : 1][4];                                       // parts of 16 rows x 16 dims
        if constexpr (P::F32) {
            #pragma unroll
            for (int e = 0; e < 4; e++) {
                const int row = g + (e & 1) * 8;
                float2 x = lds_f2(at + row * P::ROW + (P::place(row, 4 * ks + 2 * (e >> 1) + (t4 >> 1)) << 4) + (t4 & 1) * 8);
                #pragma unroll
                for (int part = 0; part < 3; part++) k4[part][e] = split2<typename P::TM>(x.x, x.y);
            }
        } else {
            const int row = (lane & 7) + (lane & 8);
            ldsm_x4_u32(k4[0], at + row * P::ROW + (P::place(row, 2 * ks + (lane >> 4)) << 4));
        }
        #pragma unroll
        for (int nt = 0; nt < NT; nt++)
            #pragma unroll
            for (int part = 0; part < P::NQ; part++) {
                const uint2 v = query((nt * P::NQ + part) * P::KS + ks);
                #pragma unroll
                for (int own = 0; own < (P::F32 ? 3 : 1); own++)
                    if (own + part < 3) mma_16<typename P::TM>(sc[nt][P::SAME16 ? ks & 1 : !own && !part ? 0 : P::F32 ? 1 + (own + part + ks & 1) : 1], k4[own], v.x, v.y);
            }
        if (P::LONG && ks % 8 == 7 && ks != P::KS - 1) {
            #pragma unroll
            for (int nt = 0; nt < NT; nt++)
                #pragma unroll
                for (int j = 0; j < 4; j++) {
                    sum[nt][j] += total(nt, j);
                    #pragma unroll
                    for (int c = 0; c < CH; c++) sc[nt][c][j] = 0.0f;
                }
        }
    }
    #pragma unroll
    for (int nt = 0; nt < NT; nt++)
        #pragma unroll
        for (int j = 0; j < 4; j++) {
            x[nt][j] = total(nt, j);
            if (P::LONG) x[nt][j] += sum[nt][j];
        }
}
// -inf for the scores of keys that a query (at position top) does not see
__device__ __forceinline__ void paged_mask(float (&x)[4], const int (&top)[2], uint32_t ok, int k0, int window, int g) {
    #pragma unroll
    for (int j = 0; j < 4; j++) {
        const int key = k0 + g + (j >> 1) * 8, pos = top[j & 1];
        if (!(ok >> (g + (j >> 1) * 8) & 1) || key > pos || (window > 0 && key <= pos - window)) x[j] = -INFINITY;
    }
}
// Scores of two columns into weights 2^(score - reference); the reference is the running maximum (and `lift`), f: what an old sum is multiplied by
template <typename P> __device__ __forceinline__ void paged_weights(float (&x)[4], const float (&cs)[2], float (&mx)[2], float (&l)[2], float lift, float (&f)[2]) {
    #pragma unroll
    for (int j = 0; j < 2; j++) {
        float m2 = fmaxf(x[j], x[j + 2]) * cs[j];
        m2 = fmaxf(m2, __shfl_xor_sync(0xffffffffu, m2, 4));
        m2 = fmaxf(m2, __shfl_xor_sync(0xffffffffu, m2, 8));
        m2 = fmaxf(m2, __shfl_xor_sync(0xffffffffu, m2, 16));
        m2 = fmaxf(lift != 0.0f ? m2 + lift : m2, mx[j]);
        const float ref = m2 == -INFINITY ? 0.0f : m2;
        f[j] = ex2(mx[j] - ref);
        mx[j] = m2;
        const float up = P::F16 ? 15.0f : 0.0f;
        // score minus maximum in one rounding: small next to the maximum, where the weight is
        x[j] = ex2(fmaf(x[j], cs[j], up - ref));
        x[j + 2] = ex2(fmaf(x[j + 2], cs[j], up - ref));
        l[j] = l[j] * f[j] + (x[j] + x[j + 2]);
    }
}

// A warp's slices s, s + W .. of an item once more, where inf or NaN was among its outputs: the matrix instructions multiply every loaded row with all parts of a
// weight, and 0 times inf is NaN -- for a query that does not see the row (the last rows of a block, the first of its windows), and for a part that is 0; f32
// numbers above bf16's largest become inf in parts; and sums of numbers near the largest run over.  Here V is multiplied key by key, where a query
// sees the key, with the whole weight, 2^-32 of what it is elsewhere (f16, which runs over nowhere: the same).  8 query rows at a time, so that it takes few
// registers from the loop's; copies go to `unit` and are waited for.  res: [NT][KS + 1][4], 2 maxima and 2 sums, then the outputs.
template <typename TQ, typename TC, int HD, int NT>
__device__ __forceinline__ void paged_key_by_key(const LgPagedAttnArgs &a, const LgReq &q, int r, int head, int row0, int n_rows, int s0, int s_end, uint32_t unit,
                                                 const uint32_t *sq, const float *cscale, float *res) {
    typedef LgPagedTile<TQ, TC, HD, NT> P;
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3, ps = a.c.page_size, row_chunks = a.c.hd * (int)sizeof(TC) / 16;
    const int hi = q.len - q.held + q.m, lo = a.window > 0 ? q.len - q.held - a.window + 1 : 0;
    #pragma unroll 1
    for (int nt = 0; nt < NT; nt++) {
        float cs[2], mx[2], l[2], o[P::KS][4];
        int top[2];
        #pragma unroll
        for (int j = 0; j < 2; j++) {
            const int n = nt * 8 + 2 * t4 + j;
            cs[j] = cscale[n]; mx[j] = -INFINITY; l[j] = 0.0f;
            top[j] = q.len - q.held + (row0 + min(n, n_rows - 1)) / a.gqa;
        }
        #pragma unroll
        for (int ks = 0; ks < P::KS; ks++)
            #pragma unroll
            for (int j = 0; j < 4; j++) o[ks][j] = 0.0f;
        #pragma unroll 1
        for (int s = s0; s < s_end; s += P::W) {
            const int key = s * 16 + (lane & 15), n = key / ps;
            const long long place = key < hi && key >= lo ? paged_place(a.c, a.c.table[(size_t)r * a.c.table_stride + n], key - n * ps, head) : -1;
            const uint32_t ok = __ballot_sync(0xffffffffu, place >= 0) & 0xFFFFu;
            auto bring = [&](const void *from) {
                __syncwarp();                                                 // what lies there has been read
                paged_copy_unit<P>(from, unit, max(place, 0LL) * (int)sizeof(TC), ok, row_chunks, lane);
                cp_async_commit();
                cp_async_wait<0>();
                __syncwarp();
            };
            float x[1][4], f[2];
            bring(a.c.k);
            paged_scores<P, 1>(unit, lane, [&](int i) { return *(const uint2 *)(sq + ((nt * P::NQ * P::KS + i) * 32 + lane) * 2); }, x);
            paged_mask(x[0], top, ok, s * 16, a.window, g);
            paged_weights<P>(x[0], cs, mx, l, P::F16 ? 0.0f : 32.0f, f);
            bring(a.c.v);
            #pragma unroll
            for (int ks = 0; ks < P::KS; ks++)
                #pragma unroll
                for (int j = 0; j < 4; j++) o[ks][j] *= above_zero(f[j & 1]);
            #pragma unroll 1
            for (int row = 0; row < 16; row++) {
                const int at = s * 16 + row;
                #pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float p = __shfl_sync(0xffffffffu, row < 8 ? x[0][j] : x[0][2 + j], (row & 7) * 4 + t4);
                    if (!(ok >> row & 1) || at > top[j] || (a.window > 0 && at <= top[j] - a.window)) continue;
                    #pragma unroll
                    for (int ks = 0; ks < P::KS; ks++)
                        #pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int byte = (16 * ks + 8 * h + g) * (int)sizeof(TC);
                            const float y = lds_elem<TC>(unit + row * P::ROW + (P::place(row, byte >> 4) << 4) + (byte & 15));
                            o[ks][2 * h + j] += fabsf(y) < INFINITY ? p * y : y;               // (the smallest weights are 0 here)
                        }
                }
            }
        }
        float *to = res + nt * 4 * (P::KS + 1);
        #pragma unroll
        for (int j = 0; j < 2; j++) { to[j] = mx[j]; to[2 + j] = l[j]; }
        #pragma unroll
        for (int ks = 0; ks < P::KS; ks++)
            #pragma unroll
            for (int j = 0; j < 4; j++) to[4 + ks * 4 + j] = o[ks][j];
    }
    __syncwarp();
}

template <typename TQ, typename TC, int HD, int NT>
__global__ void __launch_bounds__((LgPagedTile<TQ, TC, HD, NT>::W * 32), (LgPagedTile<TQ, TC, HD, NT>::CTAS)) lg_paged_attn_kernel(const __grid_constant__ LgPagedAttnArgs a) {
    typedef LgPagedTile<TQ, TC, HD, NT> P;
    extern __shared__ __align__(128) unsigned char lg_pa_sm[];
    unsigned char *ring = lg_pa_sm;
    uint32_t *sq = (uint32_t *)(lg_pa_sm + P::W * P::U * P::UNIT);           // [nt][part][ks][lane][2]
    float *buf = P::QREG ? (float *)sq : (float *)((unsigned char *)sq + P::Q_BYTES);      // [row][LDB]
    float2 *stats = (float2 *)((unsigned char *)sq + P::SHARED);              // [2][warp][row]: max, sum; items take turns
    float *cscale = (float *)(stats + 2 * P::W * P::ROWS);                  // [row]: scale of the scores
    long long *red = (long long *)(cscale + P::ROWS);                         // 18 words
    uint32_t *vmask = (uint32_t *)(red + 18);                                  // [warp][16]: keys of a slice that are there
    int *free_of = (int *)(vmask + P::W * 16);                                // [warp]: its ring's free unit
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    pdl_launch();

    // this CTA's stretch: weights of all requests, thread by thread, and where the stretch begins
    LgWalk<P::W> w;
    int stretch, length;                                                      // of every CTA; of this one (the last may be shorter)
    bool pad;
    {
        const int per = (a.n_req + P::W * 32 - 1) / (P::W * 32), r0 = min(a.n_req, tid * per), r1 = min(a.n_req, r0 + per);
        long long mine[2] = {0, 0}, s[2], before[2] = {0, 0}, total[2] = {0, 0};
        for (int r = r0; r < r1; r++) {
            const LgReq q = paged_request(a, r);
            const int items = q.groups * a.c.n_kv;
            mine[0] += (long long)paged_weight<P::W>(q, false) * items; mine[1] += (long long)paged_weight<P::W>(q, true) * items;
        }
        #pragma unroll
        for (int k = 0; k < 2; k++) {
            s[k] = mine[k];
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const long long x = __shfl_up_sync(0xffffffffu, s[k], o); if (lane >= o) s[k] += x; }
            if (lane == 31) red[2 * warp + k] = s[k];
        }
        if (tid == 0) red[16] = a.n_req;
        __syncthreads();
        #pragma unroll
        for (int i = 0; i < P::W; i++)
            #pragma unroll
            for (int k = 0; k < 2; k++) { if (i < warp) before[k] += red[2 * i + k]; total[k] += red[2 * i + k]; }
        // Stretches of the least length, if there are CTAs for them with no item's end inside of one: a CTA then has one item (each further one takes it
        // about 3 us, of 13 for a short call)
        constexpr int least = (LG_PA_MIN_STRETCH + P::W - 1) / P::W * P::W;
        pad = total[1] <= (long long)least * gridDim.x;
        const long long all = pad ? total[1] : total[0], own = pad ? mine[1] : mine[0];
        long long at = pad ? before[1] + s[1] - mine[1] : before[0] + s[0] - mine[0];
        stretch = pad ? least : (int)max((long long)least, ((all + gridDim.x - 1) / gridDim.x + P::W - 1) / P::W * P::W);
        const long long lo = (long long)stretch * blockIdx.x;
        length = (int)max(0LL, min((long long)stretch, all - lo));
        if (own && at <= lo && lo < at + own) {
            int r = r0;
            for (;; r++) {
                const LgReq q = paged_request(a, r);
                const long long x = (long long)paged_weight<P::W>(q, pad) * q.groups * a.c.n_kv;
                if (lo < at + x) break;
                at += x;
            }
            red[16] = r; red[17] = at;
        }
        __syncthreads();
        w.r = (int)red[16];
        if (tid == 0) a.jobs[blockIdx.x] = make_int4(-1, 0, 0, 0);
        if (w.r >= a.n_req) return;
        w.q = paged_request(a, w.r);
        const int n = paged_weight<P::W>(w.q, pad);
        w.hg = (int)((lo - red[17]) / n);
        w.at = (int)(red[17] + (long long)w.hg * n - lo);
    }
    // the copies run ahead of the arithmetic with a walk of their own
    LgWalk<P::W> p = w;
    int ps = 0, ps_end = 0, n_issued = 0, slot_in = 0, page = -1, rem = 0, nth = 0;         // next slice of this warp, end of the item's slices
    long long poff = 0;
    uint32_t pok = 0;
    const int ps_size = a.c.page_size, row_chunks = a.c.hd * (int)sizeof(TC) / 16;
    auto begin_item = [&]() {                                                 // first slice of this warp in walk p's item, or the next item that has one
        while (p.valid(a, length)) {
            ps = p.q.s0 + p.begin() + warp;
            ps_end = p.q.s0 + p.end(length);
            if (ps < ps_end) return true;
            p.next(a, length, pad);
        }
        return false;
    };
    bool more = begin_item();
    // Pages ahead of their use.  Pages of whole slices: lane i looks up the page of this warp's i-th slice from here, one round of loads for 32 slices.
    // Others: a lane per row of the next slice.
    auto fetch_pages = [&]() {
        page = -1; nth = 0;
        const int hi = p.q.len - p.q.held + p.q.m, lo = a.window > 0 ? p.q.len - p.q.held - a.window + 1 : 0;
        const int slice = a.whole ? ps + lane * P::W : ps, key = a.whole ? slice * 16 : slice * 16 + (lane & 15);
        if (slice < ps_end && (a.whole || (key < hi && key >= lo))) {
            const int n = key / ps_size;
            page = a.c.table[(size_t)p.r * a.c.table_stride + n];
            rem = key - n * ps_size;
            if (page < 0 || page >= a.c.n_pages) { paged_raise(a.c, LG_PAGED_BAD_PAGE); page = -1; }
        }
    };
    if (more) fetch_pages();
    const uint32_t ring_u32 = smem_u32(ring) + warp * (P::U * P::UNIT);
    auto issue = [&]() {                                                      // one unit: K of a slice, then its V
        if (more) {
            const bool is_v = n_issued & 1;
            if (!is_v) {
                // rows of the slice that some query may see, and where they lie, a lane each (lanes 16 .. 31: the same rows)
                const int hi = p.q.len - p.q.held + p.q.m, lo = a.window > 0 ? p.q.len - p.q.held - a.window + 1 : 0;
                const int first = max(lo - ps * 16, 0), last = min(hi - ps * 16, 16);
                int pg = page, rm = rem;
                if (a.whole) { pg = __shfl_sync(0xffffffffu, page, nth); rm = __shfl_sync(0xffffffffu, rem, nth) + (lane & 15); }
                poff = max(paged_place(a.c, pg, rm, p.hg / p.q.groups), 0LL) * (int)sizeof(TC);
                pok = a.whole ? pg >= 0 ? (0xFFFFu << first) & (0xFFFFu >> (16 - last)) : 0u : __ballot_sync(0xffffffffu, pg >= 0) & 0xFFFFu;
                if (lane == 0) vmask[warp * 16 + ((n_issued >> 1) & 15)] = pok;
            }
            paged_copy_unit<P>(is_v ? a.c.v : a.c.k, ring_u32 + slot_in * P::UNIT, poff, pok, row_chunks, lane);
            if (is_v) {
                ps += P::W;
                nth++;
                if (ps >= ps_end) { p.next(a, length, pad); more = begin_item(); nth = 32; }
                if (more && (!a.whole || nth == 32)) fetch_pages();
            }
            n_issued++;
            if (++slot_in == P::U) slot_in = 0;
        }
        cp_async_commit();
    };
    #pragma unroll
    for (int i = 0; i < P::U - 1; i++) issue();

    int slot = 0, n_used = 0, q_r = -1, q_hg = -1, turn = 0;
    uint32_t qr[P::QREG ? NT * P::NQ * P::KS * 2 : 1];
    for (; w.valid(a, length); w.next(a, length, pad)) {
        const int s_begin = w.q.s0 + w.begin(), s_end = w.q.s0 + w.end(length);
        if (s_begin >= s_end && (w.q.n_sl || w.at < 0)) continue;          // another stretch has its slices, or writes its zeros
        float2 *stat = stats + turn * P::W * P::ROWS;
        turn ^= 1;
        const int kvh = w.hg / w.q.groups, row0 = (w.hg - kvh * w.q.groups) * P::ROWS;      // first of the group's rows: row = token * gqa + head of the group
        const int n_rows = min(P::ROWS, w.q.m * a.gqa - row0);
        if (q_r != w.r || q_hg != w.hg) {                                     // queries of the group into operand order
            q_r = w.r; q_hg = w.hg;
            if (P::QREG && !P::OWN) __syncthreads();                          // the merge buffer lies there
            for (int n = warp; n < P::ROWS; n += P::W) {
                const int rho = row0 + n, t = rho / a.gqa;
                const TQ *src = (const TQ *)a.q + (long long)(w.q.first + t) * a.ld_q + (long long)(kvh * a.gqa + rho - t * a.gqa) * a.c.hd;
                float x[HD / 32];
                #pragma unroll
                for (int i = 0; i < HD / 64; i++) {
                    const int d = 64 * i + 2 * lane;
                    x[2 * i] = n < n_rows && d < a.c.hd ? Elem<TQ>::get(src + d) : 0.0f;
                    x[2 * i + 1] = n < n_rows && d < a.c.hd ? Elem<TQ>::get(src + d + 1) : 0.0f;
                }
                float back = a.scale;
                if (P::NQ == 2) {                                             // a power of two that takes the row's largest element to 2^14 .. 2^15
                    float top = 0.0f;
                    #pragma unroll
                    for (int i = 0; i < HD / 32; i++) top = fmaxf(top, fabsf(x[i]));
                    top = warp_max(top);
                    if (top > 0.0f && top < INFINITY) {
                        int e;
                        frexpf(top, &e);
                        const int up = 15 - e;
                        #pragma unroll
                        for (int i = 0; i < HD / 32; i++) x[i] = ldexpf(x[i], up);
                        back = ldexpf(back, -up);
                    }
                }
                #pragma unroll
                for (int i = 0; i < HD / 64; i++) {
                    const int d = 64 * i + 2 * lane, ks = d >> 4, half = (d >> 3) & 1, t = (d & 7) >> 1;
                    #pragma unroll
                    for (int part = 0; part < P::NQ; part++)
                        sq[((((n >> 3) * P::NQ + part) * P::KS + ks) * 32 + (n & 7) * 4 + t) * 2 + half] = split2<typename P::TM>(x[2 * i], x[2 * i + 1]);
                }
                if (lane == 0) cscale[n] = fmaxf(back, 1e-37f);               // above 0: a masked score times it is -inf
            }
            __syncthreads();
            if (P::QREG) {
                #pragma unroll
                for (int i = 0; i < NT * P::NQ * P::KS; i++) {
                    const uint2 v = *(const uint2 *)(sq + (i * 32 + lane) * 2);
                    qr[2 * i] = v.x; qr[2 * i + 1] = v.y;
                }
            }
        }
        float cs[NT][2], mx[NT][2], l[NT][2], o[P::KS][NT][4];
        int top[NT][2];                                                       // position of the column's query
        const int pos0 = w.q.len - w.q.held;
        #pragma unroll
        for (int nt = 0; nt < NT; nt++)
            #pragma unroll
            for (int j = 0; j < 2; j++) {
                const int n = nt * 8 + 2 * t4 + j;
                cs[nt][j] = cscale[n];
                top[nt][j] = pos0 + (row0 + min(n, n_rows - 1)) / a.gqa;
            }
        const int pos_lo = pos0 + row0 / a.gqa, pos_hi = pos0 + (row0 + n_rows - 1) / a.gqa;
        #pragma unroll
        for (int nt = 0; nt < NT; nt++) { mx[nt][0] = mx[nt][1] = -INFINITY; l[nt][0] = l[nt][1] = 0.0f; }
        #pragma unroll
        for (int ks = 0; ks < P::KS; ks++)
            #pragma unroll
            for (int nt = 0; nt < NT; nt++)
                #pragma unroll
                for (int j = 0; j < 4; j++) o[ks][nt][j] = 0.0f;
        for (int s = s_begin + warp; s < s_end; s += P::W) {
            cp_async_wait<P::U - 2>();
            __syncwarp();
            issue();
            const uint32_t ok = vmask[warp * 16 + ((n_used++) & 15)];
            uint32_t at = ring_u32 + slot * P::UNIT;
            if (++slot == P::U) slot = 0;
            float x[NT][4], f[NT][2];
            paged_scores<P, NT>(at, lane, [&](int i) {
                if (P::QREG) return make_uint2(qr[P::QREG ? 2 * i : 0], qr[P::QREG ? 2 * i + 1 : 0]);
                return *(const uint2 *)(sq + (i * 32 + lane) * 2);
            }, x);
            const bool all = ok == 0xFFFFu && s * 16 + 15 <= pos_lo && (a.window <= 0 || s * 16 > pos_hi - a.window);
            uint32_t pb[NT][P::NP][2];
            #pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                if (!all) paged_mask(x[nt], top[nt], ok, s * 16, a.window, g);
                paged_weights<P>(x[nt], cs[nt], mx[nt], l[nt], 0.0f, f[nt]);
                #pragma unroll
                for (int part = 0; part < P::NP; part++) {
                    pb[nt][part][0] = movm(split2<typename P::TM>(x[nt][0], x[nt][1]));
                    pb[nt][part][1] = movm(split2<typename P::TM>(x[nt][2], x[nt][3]));
                }
            }
            cp_async_wait<P::U - 2>();
            __syncwarp();
            issue();
            at = ring_u32 + slot * P::UNIT;
            if (++slot == P::U) slot = 0;
            #pragma unroll
            for (int ks = 0; ks < P::KS; ks++) {
                uint32_t v4[P::F32 ? 3 : 1][4];                               // parts of 16 dims x 16 rows
                if constexpr (P::F32) {
                    #pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int row = 2 * t4 + (e >> 1) * 8, d = 16 * ks + (e & 1) * 8 + g;
                        float x = lds_f(at + row * P::ROW + (P::place(row, d >> 2) << 4) + (d & 3) * 4);
                        float y = lds_f(at + (row + 1) * P::ROW + (P::place(row + 1, d >> 2) << 4) + (d & 3) * 4);
                        #pragma unroll
                        for (int part = 0; part < 3; part++) v4[part][e] = split2<typename P::TM>(x, y);
                    }
                } else {
                    const int row = (lane & 7) + ((lane >> 4) << 3);
                    ldsm_x4_t_u32(v4[0], at + row * P::ROW + (P::place(row, 2 * ks + ((lane >> 3) & 1)) << 4));
                }
                #pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float add[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    #pragma unroll
                    for (int part = P::NP - 1; part >= 0; part--)             // the smallest first: each addition to a large sum cuts off
                        #pragma unroll
                        for (int own = P::F32 ? 2 : 0; own >= 0; own--)
                            if (own + part < 3) mma_16<typename P::TM>(add, v4[own], pb[nt][part][0], pb[nt][part][1]);
                    #pragma unroll
                    for (int j = 0; j < 4; j += 2) fma2(o[ks][nt][j], o[ks][nt][j + 1], f[nt][0], f[nt][1], add[j], add[j + 1]);
                }
            }
        }
        __syncwarp();
        float odd = 0.0f;                                                     // NaN where an output is inf or NaN
        #pragma unroll
        for (int ks = 0; ks < P::KS; ks++)
            #pragma unroll
            for (int nt = 0; nt < NT; nt++)
                #pragma unroll
                for (int j = 0; j < 4; j++) odd = fmaf(o[ks][nt][j], 0.0f, odd);
        if (__any_sync(0xffffffffu, odd != odd)) {
            float res[NT * 4 * (P::KS + 1)];
            paged_key_by_key<TQ, TC, HD, NT>(a, w.q, w.r, kvh, row0, n_rows, s_begin + warp, s_end, ring_u32 + slot_in * P::UNIT, sq, cscale, res);
            #pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const float *from = res + nt * 4 * (P::KS + 1);
                #pragma unroll
                for (int j = 0; j < 2; j++) { mx[nt][j] = from[j]; l[nt][j] = from[2 + j]; }
                #pragma unroll
                for (int ks = 0; ks < P::KS; ks++)
                    #pragma unroll
                    for (int j = 0; j < 4; j++) o[ks][nt][j] = from[4 + ks * 4 + j];
            }
        }
        // the warps' results into one, in warp order
        #pragma unroll
        for (int nt = 0; nt < NT; nt++)
            #pragma unroll
            for (int j = 0; j < 2; j++) {
                float x = l[nt][j];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (g == 0) stat[warp * P::ROWS + nt * 8 + 2 * t4 + j] = make_float2(mx[nt][j], x);
            }
        // the item's other slices: before this stretch, behind it (its last slice then lies in the stretch of CTA `last`)
        const bool head = w.at < 0, tail = w.at + w.q.n_sl > length;
        const long long part = ((long long)blockIdx.x * 2 + !head) * P::ROWS;
        if (!head && tail && tid == 0) a.jobs[blockIdx.x] = make_int4(w.q.first, kvh, (int)blockIdx.x + (w.at + w.q.n_sl - 1) / stretch, row0 << 8 | n_rows);
        // row n of the item: its maximum and sum, and what the warps' outputs are multiplied by -- together at most 1, so that their sum does not run over
        auto factors = [&](int n, float &m2, float &sum, float (&fw)[P::W]) {
            m2 = -INFINITY; sum = 0.0f;
            #pragma unroll
            for (int i = 0; i < P::W; i++) m2 = fmaxf(m2, stat[i * P::ROWS + n].x);
            #pragma unroll
            for (int i = 0; i < P::W; i++) { fw[i] = ex2(stat[i * P::ROWS + n].x - (m2 == -INFINITY ? 0.0f : m2)); sum += stat[i * P::ROWS + n].y * fw[i]; }
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            #pragma unroll
            for (int i = 0; i < P::W; i++) fw[i] = above_zero(fw[i] * inv);
        };
        auto finish = [&](int n, int first, int step, auto &&number) {
            float m2, sum, fw[P::W];
            factors(n, m2, sum, fw);
            const int rho = row0 + n, t = rho / a.gqa, h = kvh * a.gqa + rho - t * a.gqa;
            if (!head && !tail) {
                TQ *out = (TQ *)a.out + (long long)(w.q.first + t) * a.ld_out + (long long)h * a.c.hd;
                for (int d = first; d < a.c.hd; d += step) out[d] = Elem<TQ>::put(number(d, fw));
            } else {
                for (int d = first; d < a.c.hd; d += step) a.part[(part + n) * a.c.hd + d] = number(d, fw);
                if (first == 0) a.part_ml[part + n] = make_float2(m2, sum);
            }
        };
        if constexpr (P::OWN) {
            // each warp's outputs into the unit of its ring that no copy is under way to; the columns of a row pair moved by 8 so that a store meets no bank twice
            float *mine = (float *)(ring + warp * (P::U * P::UNIT) + slot_in * P::UNIT);
            #pragma unroll
            for (int ks = 0; ks < P::KS; ks++)
                #pragma unroll
                for (int nt = 0; nt < NT; nt++)
                    #pragma unroll
                    for (int j = 0; j < 4; j++) mine[(nt * 8 + 2 * t4 + (j & 1)) * HD + ((ks * 16 + g + (j >> 1) * 8) ^ (t4 << 3))] = o[ks][nt][j];
            if (lane == 0) free_of[warp] = slot_in;
            __syncthreads();
            const float *from[P::W];
            #pragma unroll
            for (int i = 0; i < P::W; i++) from[i] = (const float *)(ring + i * (P::U * P::UNIT) + free_of[i] * P::UNIT);
            const bool each = n_rows >= P::W;                                 // a row a warp, or every row by all of them
            for (int n = each ? warp : 0; n < n_rows; n += each ? P::W : 1)
                finish(n, each ? lane : tid, each ? 32 : P::W * 32, [&](int d, const float (&fw)[P::W]) {
                    const int at = n * HD + (d ^ (((n >> 1) & 3) << 3));
                    float y = 0.0f;
                    #pragma unroll
                    for (int i = 0; i < P::W; i++) y += from[i][at] * fw[i];
                    return y;
                });
            __syncthreads();                                                  // before the units are filled again
        } else {
            __syncthreads();
            float f[NT][2];
            #pragma unroll
            for (int nt = 0; nt < NT; nt++)
                #pragma unroll
                for (int j = 0; j < 2; j++) {
                    float m2, sum, fw[P::W];
                    factors(nt * 8 + 2 * t4 + j, m2, sum, fw);
                    #pragma unroll
                    for (int i = 0; i < P::W; i++) if (i == warp) f[nt][j] = fw[i];
                }
            for (int i = 0; i < P::W; i++) {
                if (warp == i) {
                    #pragma unroll
                    for (int ks = 0; ks < P::KS; ks++)
                        #pragma unroll
                        for (int nt = 0; nt < NT; nt++)
                            #pragma unroll
                            for (int j = 0; j < 4; j++) {
                                float *e = buf + (nt * 8 + 2 * t4 + (j & 1)) * P::LDB + ks * 16 + g + (j >> 1) * 8;
                                const float x = o[ks][nt][j] * f[nt][j & 1];
                                *e = i ? *e + x : x;
                            }
                }
                __syncthreads();
            }
            for (int n = warp; n < n_rows; n += P::W) finish(n, lane, 32, [&](int d, const float (&)[P::W]) { return buf[n * P::LDB + d]; });
        }
    }
}

// One item that CTA b began and did not end, one query row (grid: CTAs, rows of a group): the parts, b's own and those of the CTAs behind it, each
// warp every eighth, then the warps in order.  Bound by latency.
template <typename TQ> __global__ void __launch_bounds__(256) lg_paged_merge_kernel(LgPagedAttnArgs a) {
    __shared__ float po[8][512], pl[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockIdx.y, b = blockIdx.x;
    pdl_wait();
    const int4 job = a.jobs[b];
    if (job.x < 0 || n >= (job.w & 255)) return;
    const int parts = job.z - b + 1;
    // part i: the last place of CTA b, the first one of those behind it
    auto place = [&](int i) { return ((long long)(b + i) * 2 + (i == 0)) * a.group_rows + n; };
    float4 v[4];                                                              // dims lane * 4 .. of every 128
    auto load = [&](int i) {
        #pragma unroll
        for (int k = 0; k < 4; k++) {
            const int d = k * 128 + lane * 4;
            if (d < a.c.hd) v[k] = *(const float4 *)(a.part + place(i) * a.c.hd + d);
        }
    };
    if (warp < parts) load(warp);                                             // beside the maxima
    float top = -INFINITY;
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, a.part_ml[place(i)].x);
    top = warp_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    float y[16], sum = 0.0f;
    #pragma unroll
    for (int k = 0; k < 16; k++) y[k] = 0.0f;
    for (int i = warp; i < parts; i += 8) {
        const float2 ml = a.part_ml[place(i)];
        const float f = above_zero(ex2(ml.x - ref) * (ml.y * 0x1p-46f));      // sums are at most 2^15 of 2^30 rows: outputs times this do not run over
        sum += f;
        if (i != warp) load(i);
        #pragma unroll
        for (int k = 0; k < 4; k++)
            if (k * 128 + lane * 4 < a.c.hd) { y[4 * k] += v[k].x * f; y[4 * k + 1] += v[k].y * f; y[4 * k + 2] += v[k].z * f; y[4 * k + 3] += v[k].w * f; }
    }
    #pragma unroll
    for (int k = 0; k < 4; k++) {
        const int d = k * 128 + lane * 4;
        if (d < a.c.hd) *(float4 *)&po[warp][d] = make_float4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
    }
    if (lane == 0) pl[warp] = sum;
    __syncthreads();
    sum = 0.0f;
    #pragma unroll
    for (int i = 0; i < 8; i++) sum += pl[i];
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int rho = (job.w >> 8) + n, t = rho / a.gqa;
    TQ *out = (TQ *)a.out + (long long)(job.x + t) * a.ld_out + (long long)(job.y * a.gqa + rho - t * a.gqa) * a.c.hd;
    for (int d = threadIdx.x; d < a.c.hd; d += 256) {
        float x = 0.0f;
        #pragma unroll
        for (int i = 0; i < 8; i++) x += po[i][d];
        out[d] = Elem<TQ>::put(x * inv);
    }
}
