// rq_pages.cu -- page tables and slot maps built on the device from the
// lengths of a batch's sequences, and the return of their pages.  The
// bookkeeping of a paged cache (rq_kv4.cuh) without a host round trip; the
// reference has one contiguous buffer per sequence and rolls its length back
// on the host (truncate_caches, src/streaming_quantized.rs:603-609).
#include <algorithm>

#include "rq_kv4.cuh"

namespace rq {
namespace {

constexpr int kThreads = 512;

struct PagesP {
    int batch, page_size;
    const int32_t* ctx;
    const int32_t* fresh;
    int32_t* table;
    int64_t table_stride, table_width;
    const int32_t* ring;
    int64_t n_pages;
    const int32_t* state_in;
    int32_t* state_out;
    int32_t* kv_lens;
    int32_t* cu;
    int32_t* positions;
    int32_t* slots;
    int64_t n_tokens;
    int ctas;
};

// Inclusive sums of a over the CTA (in thread order).
__device__ __forceinline__ int64_t block_scan(int64_t a, int64_t* tmp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, a, o);
        if (lane >= o) a += v;
    }
    __syncthreads();  // tmp of an earlier call is no longer read
    if (lane == 31) tmp[warp] = a;
    __syncthreads();
    int64_t before = 0;
    for (int w = 0; w < warp; w++) before += tmp[w];
    return a + before;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// first index i in 0..n-1 with v[i + 1] > x (v ascending, v[n] > x)
__device__ __forceinline__ int owner(const int64_t* v, int n, int64_t x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (v[mid + 1] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// One cluster (1 to 8 CTAs).  Requests go in chunks of a CTA's threads; every
// CTA sums the chunk's tokens and pages by itself and then fills its share of
// the chunk's page entries and token rows, finding a row's request by
// bisection in shared memory.  New entries of the table are written and old
// ones read, never the same ones, so the CTAs need one barrier a chunk: before
// kv_lens (which may be ctx_lens) and the state (which may be its own output)
// are written.  Bound by latencies: 4 us for 16 sequences of one new token (the
// lengths, two sums over the CTA, a barrier, the writes), 9.7 us for 200 of which
// most take in a prompt (354 KB written; 14 us before a warp took runs of tokens).
__global__ void __launch_bounds__(kThreads) pages_extend_kernel(const __grid_constant__ PagesP p) {
    pdl_wait();
    __shared__ int64_t tok[kThreads + 1], pg[kThreads + 1];
    __shared__ int32_t ctx[kThreads], held[kThreads];
    __shared__ int64_t tmp[kThreads / 32];
    const int rank = (int)blockIdx.x, tid = threadIdx.x;
    const int64_t step = (int64_t)p.ctas * kThreads, me = (int64_t)rank * kThreads + tid;
    const int64_t head = p.state_in[0], free = min((int64_t)max(p.state_in[1], 0), p.n_pages);
    const int64_t start = ((head % p.n_pages) + p.n_pages) % p.n_pages;
    const int64_t ps = p.page_size;
    int64_t tok0 = 0, pg0 = 0;  // tokens and pages of earlier chunks
    if (rank == 0 && tid == 0) p.cu[0] = 0;
    for (int64_t b0 = 0; b0 < p.batch; b0 += kThreads) {
        const int n = (int)min((int64_t)kThreads, p.batch - b0);
        int64_t c = 0, f = 0, need = 0, h = 0;
        if (tid < n) {
            c = max(p.ctx[b0 + tid], 0);
            f = max(p.fresh[b0 + tid], 0);
            h = min((c + ps - 1) / ps, p.table_width);
            need = min((c + f + ps - 1) / ps, p.table_width) - h;
        }
        const int64_t ts = block_scan(f, tmp);
        const int64_t gs = block_scan(need, tmp);
        if (tid == 0) tok[0] = pg[0] = 0;
        tok[tid + 1] = ts;
        pg[tid + 1] = gs;
        ctx[tid] = (int32_t)c;
        held[tid] = (int32_t)h;
        if (p.ctas > 1) cluster_sync();  // every CTA has read the chunk's lengths (and the state)
        else __syncthreads();
        if (rank == 0 && tid < n) {
            p.kv_lens[b0 + tid] = (int32_t)min(c + f, (int64_t)INT32_MAX);
            p.cu[b0 + tid + 1] = (int32_t)min(tok0 + ts, (int64_t)INT32_MAX);
        }
        // page i (counted over the batch) is ring[(start + i) % n_pages], if there
        auto taken = [&](int64_t i) {
            if (i >= free) return (int32_t)-1;
            int64_t at = start + i;
            if (at >= p.n_pages) at -= p.n_pages;
            return p.ring[at];
        };
        for (int64_t i = me; i < pg[n]; i += step) {
            const int b = owner(pg, n, i);
            p.table[(b0 + b) * p.table_stride + held[b] + (i - pg[b])] = taken(pg0 + i);
        }
        // token rows: a warp takes a run of them, so that a lane bisects once and
        // then walks; four pages at a time are on their way
        {
            const int64_t all = min(tok[n], max(p.n_tokens - tok0, (int64_t)0)), warps = step / 32;
            const int64_t run = ((all + warps - 1) / warps + 127) & ~(int64_t)127;
            const int64_t i0 = me / 32 * run, i1 = min(i0 + run, all);
            int b = i0 < i1 ? owner(tok, n, min(i0 + (tid & 31), all - 1)) : 0;
            for (int64_t i = i0 + (tid & 31); i < i1; i += 128) {
                int32_t pos[4], off[4], page[4];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int64_t at = i + 32 * x;
                    page[x] = -1;
                    pos[x] = off[x] = 0;
                    if (at >= i1) continue;
                    while (tok[b + 1] <= at) b++;
                    const int64_t ps64 = ctx[b] + (at - tok[b]);
                    pos[x] = (int32_t)min(ps64, (int64_t)INT32_MAX);
                    const int64_t col = (uint32_t)pos[x] / (uint32_t)p.page_size;
                    off[x] = (int32_t)(pos[x] - col * ps);
                    if (col < held[b]) page[x] = p.table[(b0 + b) * p.table_stride + col];
                    else if (col < p.table_width) page[x] = taken(pg0 + pg[b] + (col - held[b]));
                }
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int64_t at = i + 32 * x;
                    if (at >= i1) continue;
                    const int64_t slot = (int64_t)page[x] * ps + off[x];
                    p.positions[tok0 + at] = pos[x];
                    p.slots[tok0 + at] = page[x] < 0 || slot > INT32_MAX ? -1 : (int32_t)slot;
                }
            }
        }
        tok0 += tok[n];
        pg0 += pg[n];
        __syncthreads();  // the chunk's sums are no longer read
    }
    for (int64_t i = tok0 + me; i < p.n_tokens; i += step) {
        p.positions[i] = -1;
        p.slots[i] = -1;
    }
    if (rank == 0 && tid == 0) {
        const int64_t used = min(pg0, free);
        p.state_out[0] = (int32_t)((start + used) % p.n_pages);
        p.state_out[1] = (int32_t)(free - used);
        p.state_out[2] = (int32_t)min(pg0 - used, (int64_t)INT32_MAX);
    }
}

struct ReleaseP {
    int batch, page_size;
    const int32_t* held;
    const int32_t* keep;
    int32_t* table;
    int64_t table_stride, table_width;
    int32_t* ring;
    int64_t n_pages;
    int32_t* state;
};

// One CTA: the entries to give back are walked in order, a CTA's threads at a
// time; those that are pages are numbered by a scan and appended to the ring.
// Bound by the scan's barriers, four a run of 512 entries: 200 sequences that give
// back 978 pages take 6 us, 16 with 1854 9, and 64 with 60237 200.
__global__ void __launch_bounds__(kThreads) pages_release_kernel(const __grid_constant__ ReleaseP p) {
    pdl_wait();
    __shared__ int64_t first[kThreads + 1];
    __shared__ int32_t keep[kThreads];
    __shared__ int64_t tmp[kThreads / 32];
    const int tid = threadIdx.x;
    const int64_t start = (((int64_t)p.state[0] % p.n_pages) + p.n_pages) % p.n_pages;
    int64_t free = min((int64_t)max(p.state[1], 0), p.n_pages);
    const int64_t ps = p.page_size;
    for (int64_t b0 = 0; b0 < p.batch; b0 += kThreads) {
        const int n = (int)min((int64_t)kThreads, p.batch - b0);
        int64_t k = 0, cnt = 0;
        if (tid < n) {
            k = min(((int64_t)max(p.keep[b0 + tid], 0) + ps - 1) / ps, p.table_width);
            cnt = max(min(((int64_t)max(p.held[b0 + tid], 0) + ps - 1) / ps, p.table_width) - k, (int64_t)0);
        }
        const int64_t s = block_scan(cnt, tmp);
        if (tid == 0) first[0] = 0;
        first[tid + 1] = s;
        keep[tid] = (int32_t)k;
        __syncthreads();
        const int64_t total = first[n];
        for (int64_t i0 = 0; i0 < total; i0 += kThreads) {
            const int64_t i = i0 + tid;
            int32_t page = -1;
            if (i < total) {
                const int b = owner(first, n, i);
                int32_t* e = p.table + (b0 + b) * p.table_stride + keep[b] + (i - first[b]);
                page = *e;
                *e = -1;
            }
            const bool ok = page >= 0 && page < p.n_pages;
            const int64_t at = block_scan(ok ? 1 : 0, tmp);
            // more pages than the ring holds would be pages given back twice
            if (ok && free + at <= p.n_pages) p.ring[(start + free + at - 1) % p.n_pages] = page;
            __shared__ int64_t last;
            if (tid == kThreads - 1) last = at;
            __syncthreads();
            free = min(free + last, p.n_pages);
            __syncthreads();
        }
    }
    __syncthreads();
    if (tid == 0) p.state[1] = (int32_t)free;
}

int check_pages(const rq_ctx* ctx, int64_t batch, int page_size, int64_t table_stride, int64_t table_width, int64_t n_pages,
                const char* fn) {
    if (!ctx) return set_error(RQ_ERR_INVALID, "%s: NULL argument", fn);
    if (batch < 0 || batch > (1 << 24) || page_size < 1 || page_size > (1 << 20) || n_pages < 1 || n_pages > INT32_MAX ||
        table_width < 0 || table_width > INT32_MAX || (batch > 1 && table_stride < table_width))
        return set_error(RQ_ERR_INVALID, "%s: batch %lld, page_size %d, %lld pages, table of %lld (stride %lld)", fn,
                         (long long)batch, page_size, (long long)n_pages, (long long)table_width, (long long)table_stride);
    return RQ_OK;
}

}  // namespace

int pages_extend(int64_t batch, int page_size, const int32_t* ctx_lens, const int32_t* new_lens, int32_t* table,
                 int64_t table_stride, int64_t table_width, const int32_t* ring, int64_t n_pages, const int32_t* state_in,
                 int32_t* state_out, int32_t* kv_lens, int32_t* cu_new, int32_t* positions, int32_t* slots, int64_t n_tokens,
                 cudaStream_t st) {
    PagesP p{(int)batch, page_size, ctx_lens, new_lens, table, table_stride, table_width, ring, n_pages, state_in,
             state_out, kv_lens, cu_new, positions, slots, n_tokens, 1};
    // one CTA writes 4096 rows in about the time a cluster takes to meet
    while (p.ctas < 8 && (int64_t)p.ctas * 4096 < n_tokens) p.ctas *= 2;
    void* args[] = {&p};
    return launch_pdl((const void*)pages_extend_kernel, (unsigned)p.ctas, kThreads, 0, st, args, "page table kernel",
                      (unsigned)p.ctas);
}

int pages_release(int64_t batch, int page_size, const int32_t* held_lens, const int32_t* keep_lens, int32_t* table,
                  int64_t table_stride, int64_t table_width, int32_t* ring, int64_t n_pages, int32_t* state, cudaStream_t st) {
    ReleaseP p{(int)batch, page_size, held_lens, keep_lens, table, table_stride, table_width, ring, n_pages, state};
    void* args[] = {&p};
    return launch_pdl((const void*)pages_release_kernel, 1, kThreads, 0, st, args, "page release kernel");
}

}  // namespace rq

using namespace rq;

extern "C" {

int rq_pages_extend(rq_ctx* ctx, int64_t batch, int page_size, const int32_t* ctx_lens, const int32_t* new_lens, int32_t* table,
                    int64_t table_stride, int64_t table_width, const int32_t* ring, int64_t n_pages, const int32_t* state_in,
                    int32_t* state_out, int32_t* kv_lens, int32_t* cu_new, int32_t* positions, int32_t* slots,
                    int64_t n_tokens, void* stream) {
    static const char* fn = "rq_pages_extend";
    int rc = check_pages(ctx, batch, page_size, table_stride, table_width, n_pages, fn);
    if (rc) return rc;
    if (n_tokens < 0 || n_tokens > INT32_MAX) return set_error(RQ_ERR_INVALID, "%s: n_tokens %lld", fn, (long long)n_tokens);
    DevGuard g(ctx->device);
    struct { const void* p; const char* name; bool used; } ptrs[] = {
        {ctx_lens, "ctx_lens", batch > 0}, {new_lens, "new_lens", batch > 0}, {table, "table", batch > 0 && table_width > 0},
        {ring, "ring", true},              {state_in, "state_in", true},      {state_out, "state_out", true},
        {kv_lens, "kv_lens", batch > 0},   {cu_new, "cu_new", true},          {positions, "positions", n_tokens > 0},
        {slots, "slots", n_tokens > 0}};
    for (auto& q : ptrs)
        if (q.used && (rc = check_device_ptr(ctx, q.p, fn, q.name))) return rc;
    return pages_extend(batch, page_size, ctx_lens, new_lens, table, table_stride, table_width, ring, n_pages, state_in,
                        state_out, kv_lens, cu_new, positions, slots, n_tokens, (cudaStream_t)stream);
}

int rq_pages_release(rq_ctx* ctx, int64_t batch, int page_size, const int32_t* held_lens, const int32_t* keep_lens,
                     int32_t* table, int64_t table_stride, int64_t table_width, int32_t* ring, int64_t n_pages, int32_t* state,
                     void* stream) {
    static const char* fn = "rq_pages_release";
    int rc = check_pages(ctx, batch, page_size, table_stride, table_width, n_pages, fn);
    if (rc) return rc;
    if (!batch || !table_width) return RQ_OK;
    DevGuard g(ctx->device);
    rc = check_device_ptr(ctx, held_lens, fn, "held_lens");
    if (!rc) rc = check_device_ptr(ctx, keep_lens, fn, "keep_lens");
    if (!rc) rc = check_device_ptr(ctx, table, fn, "table");
    if (!rc) rc = check_device_ptr(ctx, ring, fn, "ring");
    if (!rc) rc = check_device_ptr(ctx, state, fn, "state");
    if (rc) return rc;
    return pages_release(batch, page_size, held_lens, keep_lens, table, table_stride, table_width, ring, n_pages, state,
                         (cudaStream_t)stream);
}

}  // extern "C"
