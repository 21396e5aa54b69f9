// lg_serve.cu -- operators of a decode step of many requests (include/lg_serve.h): the entry points, their checks and launches.
// Kernels: lg_paged.cuh (block tables and slots, append, attention of a paged cache), lg_sample.cuh.
#include <algorithm>
#include "lg_engine.h"
#include "lg_serve.h"
#include "lg_paged.cuh"
#include "lg_sample.cuh"

using namespace lg;

namespace {

#define SERVE_FAIL(code, ...) do { fprintf(stderr, __VA_ARGS__); fputc('\n', stderr); return (code); } while (0)

enum { TY_F32 = 0, TY_F16 = 1, TY_BF16 = 30 };
bool known_type(int t) { return t == TY_F32 || t == TY_F16 || t == TY_BF16; }
int type_bytes(int t) { return t == TY_F32 ? 4 : 2; }

// The device of a call: where its memory lies.  Made current for the call, the caller's is put back.
struct OnDevice {
    int dev = -1, prev = -1;
    bool ok = true;
    // p is device memory on the same device as the pointers before it
    void add(const void *p) {
        cudaPointerAttributes at;
        if (!ok) return;
        if (cudaPointerGetAttributes(&at, p) != cudaSuccess) { cudaGetLastError(); ok = false; return; }
        if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) ok = false;
        else if (dev < 0) dev = at.device;
        else if (dev != at.device) ok = false;
    }
    void add_opt(const void *p) { if (p) add(p); }
    bool enter() {
        if (!ok || cudaGetDevice(&prev) != cudaSuccess) return false;
        if (prev == dev) { prev = -1; return true; }
        if (cudaSetDevice(dev) == cudaSuccess) return true;
        cudaGetLastError();
        prev = -1;
        return false;
    }
    ~OnDevice() { if (prev >= 0) cudaSetDevice(prev); }
};

// early: the kernel may start while the one before it drains (it begins with pdl_wait); cluster: CTAs of one, along x
template <typename... KArgs> int launch_serve(const char *who, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, void *stream, bool early, int cluster, KArgs... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at; cfg.numAttrs = early ? 2 : 1;
    const cudaError_t rc = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (rc != cudaSuccess) { cudaGetLastError(); SERVE_FAIL(-6, "%s: launch failed: %s", who, cudaGetErrorString(rc)); }
    return 0;
}
// Dynamic shared memory above 48 KB, up to `most`: once per device and kernel
template <typename K> bool allow_smem(K *kernel, size_t bytes, size_t most, int dev, unsigned char *done) {
    if (bytes <= 48 * 1024 || (dev < 64 && done[dev])) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess) { cudaGetLastError(); return false; }
    if (dev < 64) done[dev] = 1;
    return true;
}

int device_sms(int dev) {
    static int n[64];
    int v = dev < 64 ? n[dev] : 0;
    if (!v) {
        if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) { cudaGetLastError(); v = 148; }
        if (dev < 64) n[dev] = v;
    }
    return v;
}

// NULL where the description of a cache is good, else what is wrong with it
const char *cache_fault(const struct lg_paged_cache *c) {
    if (!c || !c->k || !c->v || !c->table || !c->len) return "a NULL pointer in the cache";
    if (!known_type(c->type)) return "the cache's type is not f32, f16 or bf16";
    if (c->n_pages < 1 || c->page_size < 1 || c->n_kv_heads < 1 || c->max_req < 1 || c->max_pages < 1 || c->table_stride < c->max_pages)
        return "a size of the cache out of range";
    if (c->head_dim < 8 || c->head_dim > 512 || c->head_dim % 8) return "head_dim is not a multiple of 8 up to 512";
    if ((long long)c->n_pages * c->page_size > 0x7fffffffLL) return "more slots than 2^31 - 1";
    if ((long long)c->max_pages * c->page_size > 1LL << 30 || c->n_kv_heads > 65535) return "more rows in a request than 2^30, or more KV heads than 65535";
    if (c->page_stride < 0 || c->row_stride < 0 || c->head_stride < 0 || (c->page_stride | c->row_stride | c->head_stride) % 8)
        return "a stride is negative or not a multiple of 8";
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return "k and v must be 16-byte aligned";
    if (((uintptr_t)c->table | (uintptr_t)c->len | (uintptr_t)c->free_pages | (uintptr_t)c->n_free | (uintptr_t)c->status) & 3)
        return "table, len and the stack must be 4-byte aligned";
    return nullptr;
}
LgPaged paged_of(const struct lg_paged_cache *c) {
    LgPaged p;
    p.k = c->k; p.v = c->v; p.page_stride = c->page_stride; p.row_stride = c->row_stride; p.head_stride = c->head_stride;
    p.n_pages = c->n_pages; p.page_size = c->page_size; p.n_kv = c->n_kv_heads; p.hd = c->head_dim;
    p.max_pages = c->max_pages; p.table_stride = c->table_stride;
    p.table = c->table; p.len = c->len; p.free_pages = c->free_pages; p.n_free = c->n_free; p.status = c->status;
    return p;
}
void add_cache(OnDevice &on, const struct lg_paged_cache *c) {
    on.add(c->k); on.add(c->v); on.add(c->table); on.add(c->len);
    on.add_opt(c->status);
}

}  // namespace

// The kernels' own arithmetic, on the host
extern "C" long long lg_debug_paged_place(const struct lg_paged_cache *c, int page, int row, int head) {
    if (const char *f = cache_fault(c)) SERVE_FAIL(-2, "lg_debug_paged_place: %s", f);
    return paged_place(paged_of(c), page, row, head);
}

extern "C" int lg_paged_step(const struct lg_paged_cache *c, int n_req, const int *d_keep, const int *d_new, int cap, int *d_start, int *d_pos,
                             int *d_slot, int *d_req, void *stream) {
    if (const char *f = cache_fault(c)) SERVE_FAIL(-1, "lg_paged_step: %s", f);
    if (!c->free_pages || !c->n_free) SERVE_FAIL(-1, "lg_paged_step: the cache has no stack of free pages");
    if (n_req < 1 || n_req > c->max_req || cap < 0 || !d_new || !d_start) SERVE_FAIL(-1, "lg_paged_step: bad arguments");
    if (n_req > LG_PAGED_MAX_REQ) SERVE_FAIL(-2, "lg_paged_step: %d requests, at most %d", n_req, LG_PAGED_MAX_REQ);
    if (((uintptr_t)d_keep | (uintptr_t)d_new | (uintptr_t)d_start | (uintptr_t)d_pos | (uintptr_t)d_slot | (uintptr_t)d_req) & 3)
        SERVE_FAIL(-1, "lg_paged_step: arrays must be 4-byte aligned");
    OnDevice on;
    add_cache(on, c);
    on.add(c->free_pages); on.add(c->n_free); on.add(d_new); on.add(d_start);
    on.add_opt(d_keep); on.add_opt(d_pos); on.add_opt(d_slot); on.add_opt(d_req);
    if (!on.enter()) SERVE_FAIL(-1, "lg_paged_step: pointers are not memory of one device");
    LgStepArgs a;
    a.c = paged_of(c); a.n_req = n_req; a.cap = cap; a.keep = d_keep; a.fresh = d_new;
    a.start = d_start; a.pos = d_pos; a.slot = d_slot; a.req = d_req;
    const size_t smem = (4 * (size_t)n_req + 1) * sizeof(int);
    // a cluster where one CTA would go over its threads' rows more than twice
    const int ctas = cap > 2 * LG_STEP_THREADS ? 8 : 1;
    static unsigned char done[64];
    if (!allow_smem(lg_paged_step_kernel<8>, smem, (4 * (size_t)LG_PAGED_MAX_REQ + 1) * sizeof(int), on.dev, done)) SERVE_FAIL(-6, "lg_paged_step: no %zu bytes of shared memory", smem);
    void (*kernel)(LgStepArgs) = n_req <= LG_STEP_THREADS ? lg_paged_step_kernel<1> : n_req <= 2 * LG_STEP_THREADS ? lg_paged_step_kernel<2> : lg_paged_step_kernel<8>;
    return launch_serve("lg_paged_step", kernel, dim3(ctas), dim3(LG_STEP_THREADS), smem, stream, false, ctas, a);
}

extern "C" int lg_paged_append(const struct lg_paged_cache *c, const void *d_k, const void *d_v, int type, long long ld_k, long long ld_v, int n,
                               const int *d_slot, void *stream) {
    if (const char *f = cache_fault(c)) SERVE_FAIL(-1, "lg_paged_append: %s", f);
    const long long width = (long long)c->n_kv_heads * c->head_dim;
    if (n == 0) return 0;
    if (n < 0 || !d_k || !d_v || !d_slot || ld_k < width || ld_v < width) SERVE_FAIL(-1, "lg_paged_append: bad arguments");
    if (type != TY_F32 && type != c->type) SERVE_FAIL(-1, "lg_paged_append: rows are f32 or of the cache's type");
    const int eb = type_bytes(type);
    if (((uintptr_t)d_k | (uintptr_t)d_v) % eb || (uintptr_t)d_slot & 3) SERVE_FAIL(-1, "lg_paged_append: a pointer into the middle of an element");
    OnDevice on;
    add_cache(on, c);
    on.add(d_k); on.add(d_v); on.add(d_slot);
    if (!on.enter()) SERVE_FAIL(-1, "lg_paged_append: pointers are not memory of one device");
    LgAppendArgs a;
    a.c = paged_of(c); a.k = d_k; a.v = d_v; a.ld_k = ld_k; a.ld_v = ld_v; a.n = n; a.slot = d_slot;
    a.wide = !(((uintptr_t)d_k | (uintptr_t)d_v | (uintptr_t)(ld_k * eb) | (uintptr_t)(ld_v * eb)) & 15);
    const long long units = width / 4, rows = units < LG_APPEND_THREADS ? LG_APPEND_THREADS / units : 1;
    const long long ctas = (n + rows - 1) / rows, most = device_sms(on.dev) * 8LL;
    const dim3 grid((unsigned)(ctas < most ? ctas : most));
    void (*kernel)(LgAppendArgs) = nullptr;
    if (c->type == TY_F32) kernel = lg_paged_append_kernel<float, float>;
    else if (c->type == TY_F16) kernel = type == TY_F32 ? lg_paged_append_kernel<float, __half> : lg_paged_append_kernel<__half, __half>;
    else kernel = type == TY_F32 ? lg_paged_append_kernel<float, __nv_bfloat16> : lg_paged_append_kernel<__nv_bfloat16, __nv_bfloat16>;
    return launch_serve("lg_paged_append", kernel, grid, dim3(LG_APPEND_THREADS), 0, stream, false, 1, a);
}

namespace {
// Query rows of an item, 8 nt: more rows share one read of the cache and more matrix work; 8 nt x head_dim outputs have to fit a
// warp's registers.
struct AttnCut { int hd, nt; };
AttnCut attn_cut(const struct lg_paged_cache *c, int n_new, int n_heads) {
    AttnCut k;
    const int rows = n_new * (n_heads / c->n_kv_heads);
    k.hd = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : c->head_dim <= 256 ? 256 : 512;
    const int most = k.hd <= 128 ? 4 : k.hd == 256 ? 2 : 1;
    k.nt = rows <= 8 || most == 1 ? 1 : rows <= 16 || most == 2 ? 2 : 4;
    return k;
}

template <typename TQ, typename TC, int HD, int NT> int launch_attn_tile(LgPagedAttnArgs &a, int dev, void *stream) {
    typedef LgPagedTile<TQ, TC, HD, NT> P;
    static unsigned char done[64];
    if (!allow_smem(lg_paged_attn_kernel<TQ, TC, HD, NT>, P::SMEM, P::SMEM, dev, done)) SERVE_FAIL(-6, "lg_paged_attn: no %d bytes of shared memory", P::SMEM);
    const int sms = device_sms(dev), ctas = sms * P::CTAS < LG_PA_MAX_CTAS ? sms * P::CTAS : LG_PA_MAX_CTAS;
    // slices that there can be at most, so that no CTA comes for nothing
    const long long slices = ((long long)a.c.max_pages * a.c.page_size + 15) / 16 + 1 + LG_PA_ITEM_COST;
    const long long all = slices * a.n_req * a.c.n_kv * ((a.n_new * a.gqa + a.group_rows - 1) / a.group_rows) / LG_PA_MIN_STRETCH + 1;
    const int grid = all < ctas ? (int)all : ctas;
    const int rc = launch_serve("lg_paged_attn", lg_paged_attn_kernel<TQ, TC, HD, NT>, dim3(grid), dim3(P::W * 32), P::SMEM, stream, false, 1, a);
    if (rc || grid == 1) return rc;
    const int rows = a.n_new * a.gqa;
    return launch_serve("lg_paged_attn", lg_paged_merge_kernel<TQ>, dim3(grid - 1, rows < a.group_rows ? rows : a.group_rows), dim3(256), 0, stream, true, 1, a);
}
template <typename TQ, typename TC> int launch_attn_type(LgPagedAttnArgs &a, const AttnCut &k, int dev, void *stream) {
    int rc;
    if (k.hd == 64) rc = k.nt == 1 ? launch_attn_tile<TQ, TC, 64, 1>(a, dev, stream) : k.nt == 2 ? launch_attn_tile<TQ, TC, 64, 2>(a, dev, stream) : launch_attn_tile<TQ, TC, 64, 4>(a, dev, stream);
    else if (k.hd == 128) rc = k.nt == 1 ? launch_attn_tile<TQ, TC, 128, 1>(a, dev, stream) : k.nt == 2 ? launch_attn_tile<TQ, TC, 128, 2>(a, dev, stream) : launch_attn_tile<TQ, TC, 128, 4>(a, dev, stream);
    else if (k.hd == 256) rc = k.nt == 1 ? launch_attn_tile<TQ, TC, 256, 1>(a, dev, stream) : launch_attn_tile<TQ, TC, 256, 2>(a, dev, stream);
    else rc = launch_attn_tile<TQ, TC, 512, 1>(a, dev, stream);
    return rc;
}
}  // namespace

extern "C" long long lg_paged_attn_work(const struct lg_paged_cache *c, int n_req, int n_new, int n_heads) {
    if (const char *f = cache_fault(c)) SERVE_FAIL(-1, "lg_paged_attn_work: %s", f);
    if (n_req < 1 || n_req > c->max_req || n_new < 1 || n_new > LG_PAGED_MAX_NEW || n_heads < 1 || n_heads % c->n_kv_heads)
        SERVE_FAIL(-1, "lg_paged_attn_work: bad arguments");
    const AttnCut k = attn_cut(c, n_new, n_heads);
    return LG_PA_MAX_CTAS * (16 + 2LL * 8 * k.nt * (c->head_dim + 2) * 4);
}

extern "C" int lg_paged_attn(const struct lg_paged_cache *c, const void *d_q, int type, long long ld_q, int n_req, int n_new, int n_rows,
                             const int *d_start, int n_heads, float scale, int window, void *d_out, long long ld_out, void *d_work,
                             long long work_bytes, void *stream) {
    if (const char *f = cache_fault(c)) SERVE_FAIL(-1, "lg_paged_attn: %s", f);
    if (n_rows == 0 && d_start) return 0;
    if (n_req < 1 || n_req > c->max_req || n_new < 1 || n_new > LG_PAGED_MAX_NEW || n_heads < 1 || n_heads % c->n_kv_heads || n_rows < 0 ||
        !d_q || !d_out || !d_work || window < 0 || !(scale >= 0.0f) || isinf(scale))
        SERVE_FAIL(-1, "lg_paged_attn: bad arguments");
    if (!d_start && (long long)n_req * n_new != n_rows) SERVE_FAIL(-1, "lg_paged_attn: %d rows for %d requests of %d tokens", n_rows, n_req, n_new);
    if (type != TY_F32 && type != c->type) SERVE_FAIL(-1, "lg_paged_attn: q and out are f32 or of the cache's type");
    const long long width = (long long)n_heads * c->head_dim;
    if (ld_q < width || ld_out < width) SERVE_FAIL(-1, "lg_paged_attn: rows overlap");
    const int eb = type_bytes(type);
    if (((uintptr_t)d_q | (uintptr_t)d_out) % eb || (uintptr_t)d_start & 3 || (uintptr_t)d_work & 15)
        SERVE_FAIL(-1, "lg_paged_attn: a misaligned pointer");
    if (n_heads > 65535 || n_rows > 1 << 30) SERVE_FAIL(-2, "lg_paged_attn: %d rows of %d heads", n_rows, n_heads);
    const long long need = lg_paged_attn_work(c, n_req, n_new, n_heads);
    if (work_bytes < need) SERVE_FAIL(-3, "lg_paged_attn: a workspace of %lld bytes, %lld are needed", work_bytes, need);
    OnDevice on;
    add_cache(on, c);
    on.add(d_q); on.add(d_out); on.add(d_work); on.add_opt(d_start);
    if (!on.enter()) SERVE_FAIL(-1, "lg_paged_attn: pointers are not memory of one device");
    const AttnCut k = attn_cut(c, n_new, n_heads);
    LgPagedAttnArgs a;
    a.c = paged_of(c); a.q = d_q; a.out = d_out; a.ld_q = ld_q; a.ld_out = ld_out; a.n_req = n_req; a.n_new = n_new; a.n_rows = n_rows;
    a.n_heads = n_heads; a.start = d_start;
    a.window = window < (long long)c->max_pages * c->page_size ? window : 0;             // a window of all rows is none
    a.scale = (scale > 0.0f ? scale : 1.0f / sqrtf((float)c->head_dim)) * LG_LOG2E;
    a.gqa = n_heads / c->n_kv_heads; a.group_rows = 8 * k.nt; a.whole = c->page_size % 16 == 0;
    a.jobs = (int4 *)d_work;
    a.part = (float *)(a.jobs + LG_PA_MAX_CTAS);
    a.part_ml = (float2 *)(a.part + LG_PA_MAX_CTAS * 2LL * a.group_rows * c->head_dim);
    if (c->type == TY_F32) return launch_attn_type<float, float>(a, k, on.dev, stream);
    if (c->type == TY_F16) return type == TY_F32 ? launch_attn_type<float, __half>(a, k, on.dev, stream) : launch_attn_type<__half, __half>(a, k, on.dev, stream);
    return type == TY_F32 ? launch_attn_type<float, __nv_bfloat16>(a, k, on.dev, stream) : launch_attn_type<__nv_bfloat16, __nv_bfloat16>(a, k, on.dev, stream);
}

namespace {
// CTAs that share a row, a cluster of at most 8 (what every device places; 16 were slower).  A CTA's time goes with its tokens, and its fixed work -- barriers, scans of
// histograms -- with some 10000 more; two on an SM take 1.7 times as long as one; clusters that the device cannot hold at once follow in rounds.  That
// estimate is within 15 % of what was measured, and its choice within 5 % of the best: CTAs a row 1 / 2 / 3 / 4 / 5 / 6 / 8, rows of 262144 with top-p:
//   1 row - / 69 / 55 / 47 / 43 / 40 / 29 us     18 - / 160 / 114 / 92 / 78 / 70 / 81     48 - / 167 / 195 / 149 / 127 / 148 / 142     100 - / 262 / 251 / 232 / 225 / 241 / 250
// and 512 rows of 32768 without filters 48 / 55 / 79 / 86 / 107 / 126 / 162.
template <typename T> int launch_sample(LgSampleArgs &a, int dev, void *stream) {
    static unsigned char done[64];
    static int fit[64][2][LG_SAMPLE_MAX_CLUSTER + 1];                         // clusters of so many CTAs that are on the device at once, with one and two CTAs per SM
    const int both[2] = {220 * 1024, 112 * 1024}, tools = a.top_k || a.top_p ? LG_SAMPLE_TOOLS : 0, slot = dev & 63;
    if (!allow_smem(lg_sample_kernel<T>, both[0], both[0], dev, done)) SERVE_FAIL(-6, "lg_sample: no %d bytes of shared memory", both[0]);
    if (!fit[slot][1][1] || dev >= 64)
        for (int two = 0; two < 2; two++)
            for (int r = LG_SAMPLE_MAX_CLUSTER; r >= 1; r--) {
                cudaLaunchConfig_t cfg = {};
                cudaLaunchAttribute at[1];
                at[0].id = cudaLaunchAttributeClusterDimension;
                at[0].val.clusterDim.x = r; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
                cfg.gridDim = dim3(r); cfg.blockDim = dim3(LG_SAMPLE_THREADS); cfg.dynamicSmemBytes = both[two]; cfg.attrs = at; cfg.numAttrs = 1;
                int n = 0;
                if (cudaOccupancyMaxActiveClusters(&n, lg_sample_kernel<T>, &cfg) != cudaSuccess || n < 1) { cudaGetLastError(); n = std::max(1, (two + 1) * device_sms(dev) / r); }
                fit[slot][two][r] = n;
            }
    int ranks = 0;
    double least = 0.0;
    for (int r = 1; r <= LG_SAMPLE_MAX_CLUSTER; r++) {
        if (a.vocab > r << 17 || (r > 1 && a.vocab / r < 4096)) continue;
        const int rest = a.rows % fit[slot][1][r];
        const double cost = (a.vocab / r + 10000.0) * (a.rows / fit[slot][1][r] * 1.7 + (rest == 0 ? 0.0 : rest <= fit[slot][0][r] ? 1.0 : 1.7));
        if (!ranks || cost < least) { ranks = r; least = cost; }
    }
    a.slice = ((a.vocab + ranks - 1) / ranks + 127) / 128 * 128;
    // what of the slice does not fit is read again
    const int most = both[a.rows > fit[slot][0][ranks]];
    const long long held = (most - tools) / (int)sizeof(T) / 128 * 128;
    a.cap = (int)(a.slice < held ? a.slice : held);
    const size_t smem = (size_t)a.cap * sizeof(T) + tools;
    return launch_serve("lg_sample", lg_sample_kernel<T>, dim3((unsigned)a.rows * ranks), dim3(LG_SAMPLE_THREADS), smem, stream, false, ranks, a);
}
}  // namespace

extern "C" int lg_sample(const void *d_logits, int type, long long ld, int rows, int vocab, const float *d_temperature, const int *d_top_k,
                         const float *d_top_p, const float *d_min_p, const float *d_u, int *d_token, float *d_prob, void *stream) {
    if (rows == 0) return 0;
    if (!d_logits || !d_u || !d_token || rows < 0 || vocab < 1 || ld < vocab || !known_type(type)) SERVE_FAIL(-1, "lg_sample: bad arguments");
    if (vocab > 1 << 20 || rows > 1 << 27) SERVE_FAIL(-2, "lg_sample: %d rows of %d, at most %d of %d", rows, vocab, 1 << 27, 1 << 20);
    if ((uintptr_t)d_logits % type_bytes(type) ||
        ((uintptr_t)d_temperature | (uintptr_t)d_top_k | (uintptr_t)d_top_p | (uintptr_t)d_min_p | (uintptr_t)d_u | (uintptr_t)d_token | (uintptr_t)d_prob) & 3)
        SERVE_FAIL(-1, "lg_sample: a pointer into the middle of an element");
    OnDevice on;
    on.add(d_logits); on.add(d_u); on.add(d_token);
    on.add_opt(d_temperature); on.add_opt(d_top_k); on.add_opt(d_top_p); on.add_opt(d_min_p); on.add_opt(d_prob);
    if (!on.enter()) SERVE_FAIL(-1, "lg_sample: pointers are not memory of one device");
    LgSampleArgs a;
    a.logits = d_logits; a.ld = ld; a.rows = rows; a.vocab = vocab;
    int bits = 0;
    while ((1 << bits) < vocab) bits++;
    a.shift = 62 - bits < 44 ? 62 - bits : 44;
    a.temperature = d_temperature; a.top_k = d_top_k; a.top_p = d_top_p; a.min_p = d_min_p; a.u = d_u; a.token = d_token; a.prob = d_prob;
    return type == TY_F32 ? launch_sample<float>(a, on.dev, stream) : type == TY_F16 ? launch_sample<__half>(a, on.dev, stream) : launch_sample<__nv_bfloat16>(a, on.dev, stream);
}

// The parameters of the one row go to the device beside its forward; the token and its probability return behind it.
extern "C" int lg_forward_sample(struct model *m, struct kvcache *kv, int token, int pos, float temperature, int top_k, float top_p, float min_p,
                                 float u, float *prob) {
    Engine *e = nullptr;
    const float *logits = forward_device_logits(m, kv, token, pos, &e);
    struct Words { float temperature; int top_k; float top_p, min_p, u; int token; float prob; };
    if (!e->draw) e->draw = dalloc<float>(sizeof(Words) / 4);
    if (!e->draw_host) LG_CHECK(cudaMallocHost(&e->draw_host, sizeof(Words)));
    Words *d = (Words *)e->draw, *h = (Words *)e->draw_host;
    *h = Words{temperature, top_k, top_p, min_p, u, -1, 0.0f};
    LG_CHECK(cudaMemcpyAsync(d, h, sizeof(Words), cudaMemcpyHostToDevice, e->stream));
    const int n_vocab = m->cfg.n_vocab;
    if (lg_sample(logits, TY_F32, n_vocab, 1, n_vocab, &d->temperature, &d->top_k, &d->top_p, &d->min_p, &d->u, &d->token, &d->prob, e->stream)) exit(1);
    LG_CHECK(cudaMemcpyAsync(&h->token, &d->token, 8, cudaMemcpyDeviceToHost, e->stream));
    check_err(e);
    e->host_syncs++;
    if (prob) *prob = h->prob;
    return h->token;
}
