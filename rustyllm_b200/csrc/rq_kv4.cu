// rq_kv4.cu -- the 4-bit paged key/value cache: create, append, read; and the
// pass that normalises queries and keys per head and rotates them by their
// positions, with or without the append in the same launch.  No counterpart
// in the reference, whose cache is contiguous f32 (QuantStreamCache,
// src/streaming_quantized.rs:93-152) and whose rotation is a pass of its own
// (QAttn::forward, :201-240).

#include <algorithm>
#include <new>
#include <utility>

#include "rq_kv4.cuh"

namespace rq {

int check_device_ptr(const rq_ctx* ctx, const void* p, const char* fn, const char* name) {
    if (!p) return set_error(RQ_ERR_INVALID, "%s: %s is NULL", fn, name);
    cudaPointerAttributes a;
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
        cudaGetLastError();
        return set_error(RQ_ERR_INVALID, "%s: %s must be device memory", fn, name);
    }
    if (a.type != cudaMemoryTypeManaged && (a.type != cudaMemoryTypeDevice || a.device != ctx->device))
        return set_error(RQ_ERR_INVALID, "%s: %s must be device memory on device %d", fn, name, ctx->device);
    return RQ_OK;
}

int check_rows_apart(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t len, const char* fn, const char* name) {
    using wide = __int128;
    if (n0 < 1 || n1 < 1) return RQ_OK;
    // the larger stride's axis is `a`; an axis of one row has none
    wide sa = n0 > 1 ? (s0 < 0 ? -(wide)s0 : s0) : 0, sb = n1 > 1 ? (s1 < 0 ? -(wide)s1 : s1) : 0;
    if (sa < sb) {
        std::swap(sa, sb);
        std::swap(n0, n1);
    }
    bool meet = (n0 > 1 && sa < len) || (n1 > 1 && sb < len);
    // rows i of a and j of b lie i sa - j sb apart: nothing meets where a steps
    // over all of b, else the nearest j of each i say
    const wide span = n1 > 1 ? sb * (n1 - 1) : 0;
    for (int64_t i = 1; !meet && n1 > 1 && i < n0 && i * sa < span + len; i++) {
        const wide j = i * sa / sb, off = i * sa - j * sb;
        meet = (j < n1 && off < len) || (j + 1 < n1 && sb - off < len);
    }
    return meet ? set_error(RQ_ERR_INVALID, "%s: %s: its rows lie on one another", fn, name) : RQ_OK;
}

int launch_pdl(const void* fn, unsigned grid, unsigned block, size_t smem, cudaStream_t st, void** args, const char* what,
               unsigned cluster) {
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cuda_error(cudaLaunchKernelExC(&cfg, fn, args), what);
}

namespace {

size_t dtype_size(int dtype) { return dtype == RQ_F32 ? 4 : dtype == RQ_F16 || dtype == RQ_BF16 ? 2 : 0; }

bool wide_ok(const void* p, int64_t s0, int64_t s1, size_t size) {
    return (((uintptr_t)p | (uintptr_t)(s0 * (int64_t)size) | (uintptr_t)(s1 * (int64_t)size)) & 15) == 0;
}

// ------------------------------------------------------------------ append
//
// A lane takes 8 elements of a block of 32 (an item) and a CTA whole tokens
// (`per_cta`, see tokens_per_cta), so that a warp's reads are whole lines and indexes
// are 32-bit inside it; the largest magnitude crosses four lanes by shuffles, a
// code is decided without rounding (rq_kv4.cuh).  Bound by the issue of the
// quantizer's instructions (84 % of the slots; 46 an element): 16001 tokens of 8
// heads of 128 in bf16 take 50 us (84 MB, 1.7 TB/s), in f32 49; 64 in f32 2.3 us,
// one launch and one round trip.
struct AppendP {
    const void* x[2];          // k, v
    int64_t tok[2], head[2];   // strides in elements
    bool wide[2];
    const int32_t* slots;
    int64_t n, n_slots;
    uint8_t* data;
    int page_size, n_kv, nb, per_cta;
};

// Item i of a CTA's tokens: row (K's heads, then V's, of a token) and 8 elements
struct Item {
    int64_t n;
    int head, e;
    bool is_v;
    __device__ __forceinline__ Item(unsigned i, int64_t first, int n_kv, unsigned nb) {
        const unsigned per = 4 * nb, row = i / per;
        const unsigned tok = row / (2u * n_kv), r = row - tok * 2u * n_kv;
        e = (int)(i - row * per);
        is_v = r >= (unsigned)n_kv;
        head = (int)(is_v ? r - n_kv : r);
        n = first + tok;
    }
};

template <typename T, int NB>
__global__ void __launch_bounds__(256) kv4_append_kernel(const __grid_constant__ AppendP p) {
    pdl_wait();
    const int64_t first = (int64_t)blockIdx.x * p.per_cta;
    const unsigned items = (unsigned)(min((int64_t)p.per_cta, p.n - first) * 2 * p.n_kv * 4 * NB);
    for (unsigned i = threadIdx.x; i < items; i += 256) {
        const Item it(i, first, p.n_kv, NB);
        const int32_t slot = p.slots[it.n];
        float x[8];
        load8(static_cast<const T*>(p.x[it.is_v]) + it.n * p.tok[it.is_v] + it.head * p.head[it.is_v] + 8 * it.e,
              p.wide[it.is_v], x);
        uint8_t* rec = kv4_record(p.data, p.n_slots, p.page_size, p.n_kv, 576 * NB, slot, it.head);
        kv4_store(rec, NB, slot & 15, it.e >> 2, it.is_v, x);
    }
}

// k and v rows of the given slots, dequantized; zeros for a slot outside the
// cache.  The append's thread mapping.  Bound by memory and the
// scattered code words: 16001 tokens of 8 heads of 128 take 28 us into bf16 (84 MB,
// 3.0 TB/s), 35 into f32 (150 MB, 4.3 TB/s).
struct ReadP {
    const uint8_t* data;
    const int32_t* slots;
    int64_t n, n_slots;
    int page_size, n_kv, per_cta;
    void* x[2];  // [n][n_kv][head_dim]
    bool wide;
};

template <typename T, int NB>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ ReadP p) {
    pdl_wait();
    const int64_t first = (int64_t)blockIdx.x * p.per_cta;
    const unsigned items = (unsigned)(min((int64_t)p.per_cta, p.n - first) * 2 * p.n_kv * 4 * NB);
    for (unsigned i = threadIdx.x; i < items; i += 256) {
        const Item it(i, first, p.n_kv, NB);
        const int32_t slot = p.slots[it.n];
        const uint8_t* rec =
            kv4_record(const_cast<uint8_t*>(p.data), p.n_slots, p.page_size, p.n_kv, 576 * NB, slot, it.head);
        float x[8];
        kv4_load(rec, NB, slot & 15, it.e >> 2, it.is_v, x);
        store8(static_cast<T*>(p.x[it.is_v]) + (it.n * p.n_kv + it.head) * (32 * NB) + 8 * it.e, p.wide, x);
    }
}

// --------------------------------------------------- norm and rotation
//
// y = x / sqrt(mean(x^2) + eps) * w per head (w NULL: y = x), then the first
// rot elements rotated in pairs by the angles of the token's position.  A row
// is cut into units of E elements (four, or one where alignment or sizes forbid
// that); a lane holds the unit with the first halves of its
// pairs and the one with the second, so the rotation needs no exchange and a
// row may be its own output.  Bound by memory.
constexpr int kRopeRows = 2;  // heads that a group of lanes takes at once where the rows are many
struct RopeP {
    const void* x[2];  // q, k
    void* y[2];
    int64_t xt[2], xh[2], yt[2], yh[2];  // strides in elements: token, head
    const float* w[2];
    const float* cos;
    const float* sin;
    const int32_t* pos;
    int64_t n, max_pos;
    int heads[2];
    int hd, rot, inter, lpr, lpr_log;
    unsigned q_ctas;
    float eps, inv_hd;
};

template <typename T, int E>
struct alignas(sizeof(T) * E > 16 ? 16 : sizeof(T) * E) Unit {
    T v[E];
    Unit() = default;
    __device__ __forceinline__ explicit Unit(const float (&x)[E]) {
#pragma unroll
        for (int i = 0; i < E; i++) v[i] = from_f32<T>(x[i]);
    }
};

// What a lane holds of one head's row: units u0 and u1 (-1: none), the first and
// second halves of its pairs where i < P = rot / 2 E (interleaved: its pairs are
// neighbours), elements that are not rotated behind them.
template <int E>
struct Lane {
    int u0, u1;
    bool turns;
    __device__ __forceinline__ Lane(const RopeP& p, int i) {
        const int P = p.rot / (2 * E), rest = (p.hd - p.rot) / E, r = 2 * (i - P);
        turns = i < P;
        u0 = turns ? i : r < rest ? 2 * P + r : -1;
        u1 = turns ? i + P : r + 1 < rest ? 2 * P + r + 1 : -1;
        if (p.inter && E == 1 && turns) {  // single elements: the pair is (2 i, 2 i + 1)
            u0 = 2 * i;
            u1 = 2 * i + 1;
        }
    }
};
// The angles of a position for a lane's pairs, in element order of u0 and u1
// (halves: a pair takes one of each; interleaved: the pairs of u0 first)
template <int E>
struct Angles {
    Unit<float, E> cs, sn;
    __device__ __forceinline__ void load(const RopeP& p, const Lane<E>& l, int64_t pos) {
        if (!l.turns || pos < 0 || pos >= p.max_pos) return;
        const float* c = p.cos + pos * (p.rot / 2);
        const float* z = p.sin + pos * (p.rot / 2);
        if (E == 1 || !p.inter) {
            const int at = E == 1 && p.inter ? l.u0 / 2 : l.u0 * E;
            cs = *reinterpret_cast<const Unit<float, E>*>(c + at);
            sn = *reinterpret_cast<const Unit<float, E>*>(z + at);
        } else if constexpr (E > 1) {
            using Half = Unit<float, E / 2>;
            const Half c0 = *reinterpret_cast<const Half*>(c + l.u0 * (E / 2)), c1 = *reinterpret_cast<const Half*>(c + l.u1 * (E / 2));
            const Half z0 = *reinterpret_cast<const Half*>(z + l.u0 * (E / 2)), z1 = *reinterpret_cast<const Half*>(z + l.u1 * (E / 2));
#pragma unroll
            for (int e = 0; e < E / 2; e++) {
                cs.v[e] = c0.v[e];
                sn.v[e] = z0.v[e];
                cs.v[E / 2 + e] = c1.v[e];
                sn.v[E / 2 + e] = z1.v[e];
            }
        }
    }
};
// The norm's weights taken into the rotation: per pair (f, g) of elements
//   f' = r (f A + g B), g' = r (f C + g D)   (A = wf cos, B = -wg sin, ..);
// elements that are not rotated use A and D alone.
template <int E>
struct Coeffs {
    float A[E], B[E], C[E], D[E];
    __device__ __forceinline__ Coeffs(const RopeP& p, const Lane<E>& l, const Angles<E>& t, const float* w) {
        Unit<float, E> w0, w1;
#pragma unroll
        for (int e = 0; e < E; e++) w0.v[e] = w1.v[e] = 1.0f;
        if (w) {
            if (l.u0 >= 0) w0 = *reinterpret_cast<const Unit<float, E>*>(w + l.u0 * E);
            if (l.u1 >= 0) w1 = *reinterpret_cast<const Unit<float, E>*>(w + l.u1 * E);
        }
#pragma unroll
        for (int e = 0; e < E; e++) {
            float f = w0.v[e], g = w1.v[e];
            if (E > 1 && p.inter && l.turns) {
                f = 2 * e < E ? w0.v[2 * e % E] : w1.v[2 * e % E];
                g = 2 * e < E ? w0.v[(2 * e + 1) % E] : w1.v[(2 * e + 1) % E];
            }
            const float cs = l.turns ? t.cs.v[e] : 1.0f, sn = l.turns ? t.sn.v[e] : 0.0f;
            A[e] = f * cs;
            B[e] = -g * sn;
            C[e] = f * sn;
            D[e] = g * cs;
        }
    }
    __device__ __forceinline__ void turn(const RopeP& p, const Lane<E>& l, float (&a)[E], float (&b)[E]) const {
        if (!l.turns) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                a[e] *= A[e];
                b[e] *= D[e];
            }
        } else if (E == 1 || !p.inter) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float2 v = fma2(make_float2(a[e], a[e]), make_float2(A[e], C[e]),
                                      mul2(make_float2(b[e], b[e]), make_float2(B[e], D[e])));
                a[e] = v.x;
                b[e] = v.y;
            }
        } else if constexpr (E > 1) {
#pragma unroll
            for (int e = 0; e < E / 2; e++) {
                float f = a[2 * e], g = a[2 * e + 1];
                a[2 * e] = f * A[e] + g * B[e];
                a[2 * e + 1] = f * C[e] + g * D[e];
                f = b[2 * e];
                g = b[2 * e + 1];
                b[2 * e] = f * A[E / 2 + e] + g * B[E / 2 + e];
                b[2 * e + 1] = f * C[E / 2 + e] + g * D[E / 2 + e];
            }
        }
    }
};
__device__ __forceinline__ float group_sum(float v, int lpr, unsigned group) {
    for (int o = lpr >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(group, v, o);
    return v;
}
__device__ __forceinline__ unsigned group_mask(int lpr, int lane) {
    return (lpr == 32 ? 0xffffffffu : ((1u << lpr) - 1u)) << (lane & ~(lpr - 1));
}

// q (0) or k (1), the same for a whole CTA: selected once, since a pointer
// picked from the parameters by a thread's index costs every access
template <typename T>
struct Side {
    const T* x;
    T* y;
    const float* w;
    int64_t xt, xh, yt, yh;
    int heads;
    __device__ __forceinline__ Side(const RopeP& p, bool k)
        : x(static_cast<const T*>(k ? p.x[1] : p.x[0])), y(static_cast<T*>(k ? p.y[1] : p.y[0])), w(k ? p.w[1] : p.w[0]),
          xt(k ? p.xt[1] : p.xt[0]), xh(k ? p.xh[1] : p.xh[0]), yt(k ? p.yt[1] : p.yt[0]), yh(k ? p.yh[1] : p.yh[0]),
          heads(k ? p.heads[1] : p.heads[0]) {}
};

// One row a group of lanes: few rows, where a launch and one round trip bound it
// (5 tokens of 64 + 8 heads of 128 in f32: 2.1 us), and what units of 16 bytes
// cannot take.
// The first q_ctas CTAs take q's rows, the others k's.
template <typename T, int E, int S>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const __grid_constant__ RopeP p) {
    pdl_wait();
    const int lane = threadIdx.x & 31, sl = lane & (p.lpr - 1);
    const unsigned group = group_mask(p.lpr, lane);
    const bool is_k = blockIdx.x >= p.q_ctas;
    const Side<T> o(p, is_k);
    const unsigned gi = (blockIdx.x - (is_k ? p.q_ctas : 0)) * (256u >> p.lpr_log) + (threadIdx.x >> p.lpr_log);
    const int64_t n = gi / (unsigned)o.heads;
    if (n >= p.n) return;
    const int head = (int)(gi - (unsigned)n * (unsigned)o.heads);
    const T* x = o.x + n * o.xt + head * o.xh;
    T* y = o.y + n * o.yt + head * o.yh;
    // the row's loads come first: the position, the tables behind it and the
    // row are then not three round trips to memory
    float a[S][E], b[S][E], ss = 0.0f;
#pragma unroll
    for (int s = 0; s < S; s++) {
        const Lane<E> l(p, sl + s * p.lpr);
        Unit<T, E> ra, rb;
        if (l.u0 >= 0) ra = *reinterpret_cast<const Unit<T, E>*>(x + l.u0 * E);
        if (l.u1 >= 0) rb = *reinterpret_cast<const Unit<T, E>*>(x + l.u1 * E);
#pragma unroll
        for (int e = 0; e < E; e++) {
            a[s][e] = l.u0 >= 0 ? to_f32(ra.v[e]) : 0.0f;
            b[s][e] = l.u1 >= 0 ? to_f32(rb.v[e]) : 0.0f;
            ss = fmaf(a[s][e], a[s][e], fmaf(b[s][e], b[s][e], ss));
        }
    }
    const int64_t pos = p.pos[n];
    if (pos < 0 || pos >= p.max_pos) return;  // the row stays as it was
    const float r = o.w ? rsqrtf(fmaf(group_sum(ss, p.lpr, group), p.inv_hd, p.eps)) : 1.0f;
#pragma unroll
    for (int s = 0; s < S; s++) {
        const Lane<E> l(p, sl + s * p.lpr);
        Angles<E> t;
        t.load(p, l, pos);
        const Coeffs<E> c(p, l, t, o.w);
#pragma unroll
        for (int e = 0; e < E; e++) {
            a[s][e] *= r;
            b[s][e] *= r;
        }
        c.turn(p, l, a[s], b[s]);
        if (l.u0 >= 0) *reinterpret_cast<Unit<T, E>*>(y + l.u0 * E) = Unit<T, E>(a[s]);
        if (l.u1 >= 0) *reinterpret_cast<Unit<T, E>*>(y + l.u1 * E) = Unit<T, E>(b[s]);
    }
}

// Many rows: a group of lanes takes U heads of a token (E = 8 elements a unit
// for 16-bit types, 4 for f32: 16 bytes), all rows' loads before the first use.
// Bound by the loads that three CTAs an SM keep in flight: 8191 tokens of 64 + 8
// heads of 128 in bf16 take 88 us (3.4 TB/s read and written) with two heads a
// group, 93 with four (fewer CTAs), 112 with one (the angles loaded for each).
template <typename T, int U>
__global__ void __launch_bounds__(256, 3) qk_norm_rope_rows_kernel(const __grid_constant__ RopeP p) {
    constexpr int E = 16 / sizeof(T);
    pdl_wait();
    const int lane = threadIdx.x & 31, sl = lane & (p.lpr - 1);
    const unsigned group = group_mask(p.lpr, lane);
    const bool is_k = blockIdx.x >= p.q_ctas;
    const Side<T> o(p, is_k);
    const unsigned i = (blockIdx.x - (is_k ? p.q_ctas : 0)) * (256u >> p.lpr_log) + (threadIdx.x >> p.lpr_log);
    const unsigned per = (unsigned)(o.heads + U - 1) / U;
    const unsigned n = i / per;
    if (n >= p.n) return;
    const int h0 = (int)(i - n * per) * U, hn = min(U, o.heads - h0);
    const Lane<E> l(p, sl);
    const T* x = o.x + n * o.xt + h0 * o.xh;
    T* y = o.y + n * o.yt + h0 * o.yh;
    Unit<T, E> ra[U], rb[U];
#pragma unroll
    for (int h = 0; h < U; h++)
        if (h < hn) {
            if (l.u0 >= 0) ra[h] = *reinterpret_cast<const Unit<T, E>*>(x + h * o.xh + l.u0 * E);
            if (l.u1 >= 0) rb[h] = *reinterpret_cast<const Unit<T, E>*>(x + h * o.xh + l.u1 * E);
        }
    const int64_t pos = p.pos[n];
    if (pos < 0 || pos >= p.max_pos) return;  // the rows stay as they were
    Angles<E> t;
    t.load(p, l, pos);
    const Coeffs<E> c(p, l, t, o.w);
#pragma unroll
    for (int h = 0; h < U; h++) {
        if (h >= hn) break;
        float a[E], b[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            a[e] = l.u0 >= 0 ? to_f32(ra[h].v[e]) : 0.0f;
            b[e] = l.u1 >= 0 ? to_f32(rb[h].v[e]) : 0.0f;
        }
        if (o.w) {
            float2 s2 = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int e = 0; e < E; e++) s2 = fma2(make_float2(a[e], b[e]), make_float2(a[e], b[e]), s2);
            const float r = rsqrtf(fmaf(group_sum(s2.x + s2.y, p.lpr, group), p.inv_hd, p.eps));
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float2 v = mul2(make_float2(a[e], b[e]), make_float2(r, r));
                a[e] = v.x;
                b[e] = v.y;
            }
        }
        c.turn(p, l, a, b);
        if (l.u0 >= 0) *reinterpret_cast<Unit<T, E>*>(y + h * o.yh + l.u0 * E) = Unit<T, E>(a);
        if (l.u1 >= 0) *reinterpret_cast<Unit<T, E>*>(y + h * o.yh + l.u1 * E) = Unit<T, E>(b);
    }
}

// The same with the append: 16 lanes a row of q, k or v (head_dim <= 128),
// 8 consecutive elements a lane as the blocks of the cache want them; the
// rotation's partner comes through shared memory.  For decode steps: 5 tokens of 64
// + 8 + 8 heads of 128 take 3.5 us in f32 (rotation and append one after the other
// 4.2), 64 4.5 (4.8).  At 8191 tokens the angles and weights fetched by element,
// the row's way through shared memory and a 64-bit division a row bound it: 189 us
// in bf16 and 211 in f32, where the two passes take 114 and 134.
struct RopeAppendP {
    RopeP r;  // y[1] unused
    bool wide_q, wide_qo;
    AppendP a;  // x[0] = k, x[1] = v
};

template <typename T>
__global__ void __launch_bounds__(256) qk_norm_rope_append_kernel(const __grid_constant__ RopeAppendP p) {
    pdl_wait();
    __shared__ float rows[16][132];
    const int lane = threadIdx.x & 31, sl = lane & 15, gidx = threadIdx.x >> 4;
    const int H = p.r.heads[0], kv = p.a.n_kv, per = H + 2 * kv, nb = p.a.nb;
    const int64_t gi = (int64_t)blockIdx.x * 16 + gidx;
    const int64_t n = gi / per;
    bool live = n < p.a.n;
    const int r = live ? (int)(gi - n * per) : 0;
    const int kind = r < H ? 0 : r < H + kv ? 1 : 2;  // q, k, v
    const int64_t pos = live ? p.r.pos[n] : -1;
    live = live && pos >= 0 && pos < p.r.max_pos;
    const bool mine = live && sl < 4 * nb;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = 0.0f;
    if (mine) {
        if (kind == 0) load8(static_cast<const T*>(p.r.x[0]) + n * p.r.xt[0] + r * p.r.xh[0] + 8 * sl, p.wide_q, x);
        else
            load8(static_cast<const T*>(p.a.x[kind - 1]) + n * p.a.tok[kind - 1] +
                      (r - H - (kind - 1) * kv) * p.a.head[kind - 1] + 8 * sl,
                  p.a.wide[kind - 1], x);
    }
    if (kind < 2) {
        const float* w = p.r.w[kind];
        if (w) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffu << (lane & 16), ss, o);
            const float s = rsqrtf(fmaf(ss, p.r.inv_hd, p.r.eps));
            if (mine)
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = x[i] * s * w[8 * sl + i];
        }
    }
    float* row = rows[gidx];
    if (mine)
#pragma unroll
        for (int i = 0; i < 8; i++) row[8 * sl + i] = x[i];
    __syncwarp();
    if (mine && kind < 2) {
        const int rot = p.r.rot, half = rot / 2;
        const float* cs = p.r.cos + pos * half;
        const float* sn = p.r.sin + pos * half;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int d = 8 * sl + i;
            if (d < rot) {
                int a, f, g;  // angle, first and second of the pair
                if (p.r.inter) {
                    a = d >> 1;
                    f = d & ~1;
                    g = f + 1;
                } else {
                    a = d < half ? d : d - half;
                    f = a;
                    g = a + half;
                }
                const float c = cs[a], s = sn[a];
                x[i] = d == f ? row[f] * c - row[g] * s : row[f] * s + row[g] * c;
            }
        }
    }
    if (kind == 0) {
        if (mine) store8(static_cast<T*>(p.r.y[0]) + n * p.r.yt[0] + r * p.r.yh[0] + 8 * sl, p.wide_qo, x);
    } else {
        const int head = r - H - (kind - 1) * kv;
        uint8_t* rec = nullptr;
        int tok = 0;
        if (mine) {
            const int32_t slot = p.a.slots[n];
            rec = kv4_record(p.a.data, p.a.n_slots, p.a.page_size, kv, 576 * nb, slot, head);
            tok = slot & 15;
        }
        kv4_store(rec, nb, tok, sl >> 2, kind == 2, x);
    }
}

int check_cache(const rq_kv4* c, const char* fn) {
    return c ? RQ_OK : set_error(RQ_ERR_INVALID, "%s: NULL cache", fn);
}

int check_rope(const rq_ctx* ctx, const rq_qk_rope* a, bool append, const char* fn) {
    if (!ctx || !a) return set_error(RQ_ERR_INVALID, "%s: NULL argument", fn);
    if (!dtype_size(a->dtype)) return set_error(RQ_ERR_UNSUPPORTED, "%s: dtype %d (f32 = 0, f16 = 1, bf16 = 2)", fn, a->dtype);
    if (a->n_tokens < 0 || a->n_heads < 0 || a->n_kv_heads < 0 || a->n_heads > 65536 || a->n_kv_heads > 65536 ||
        a->n_tokens > INT32_MAX)
        return set_error(RQ_ERR_INVALID, "%s: %lld tokens, %lld / %lld heads", fn, (long long)a->n_tokens,
                         (long long)a->n_heads, (long long)a->n_kv_heads);
    if (a->head_dim < 2 || a->head_dim > 256 || a->head_dim % 2 || a->rot_dim < 0 || a->rot_dim > a->head_dim || a->rot_dim % 2)
        return set_error(RQ_ERR_INVALID, "%s: head_dim %lld (even, 2..256), rot_dim %lld (even, 0..head_dim)", fn,
                         (long long)a->head_dim, (long long)a->rot_dim);
    if (a->rot_dim && a->max_pos < 1) return set_error(RQ_ERR_INVALID, "%s: max_pos %lld", fn, (long long)a->max_pos);
    int rc = RQ_OK;
    if (a->n_tokens) {
        if (!rc) rc = check_device_ptr(ctx, a->positions, fn, "positions");
        if (!rc && a->n_heads) rc = check_device_ptr(ctx, a->q, fn, "q");
        if (!rc && a->n_heads) rc = check_device_ptr(ctx, a->q_out, fn, "q_out");
        if (!rc) rc = check_rows_apart(a->n_tokens, a->q_out_stride[0], a->n_heads, a->q_out_stride[1], a->head_dim, fn, "q_out");
        if (!rc && a->n_kv_heads) rc = check_device_ptr(ctx, a->k, fn, "k");
        if (!rc && a->n_kv_heads && !append) rc = check_device_ptr(ctx, a->k_out, fn, "k_out");
        if (!rc && !append)
            rc = check_rows_apart(a->n_tokens, a->k_out_stride[0], a->n_kv_heads, a->k_out_stride[1], a->head_dim, fn, "k_out");
        if (!rc && a->rot_dim) rc = check_device_ptr(ctx, a->cos, fn, "cos");
        if (!rc && a->rot_dim) rc = check_device_ptr(ctx, a->sin, fn, "sin");
        if (!rc && a->q_weight) rc = check_device_ptr(ctx, a->q_weight, fn, "q_weight");
        if (!rc && a->k_weight) rc = check_device_ptr(ctx, a->k_weight, fn, "k_weight");
    }
    return rc;
}

RopeP rope_params(const rq_qk_rope* a) {
    RopeP p{};
    p.x[0] = a->q;
    p.x[1] = a->k;
    p.y[0] = a->q_out;
    p.y[1] = a->k_out;
    p.xt[0] = a->q_stride[0];
    p.xh[0] = a->q_stride[1];
    p.xt[1] = a->k_stride[0];
    p.xh[1] = a->k_stride[1];
    p.yt[0] = a->q_out_stride[0];
    p.yh[0] = a->q_out_stride[1];
    p.yt[1] = a->k_out_stride[0];
    p.yh[1] = a->k_out_stride[1];
    p.w[0] = a->q_weight;
    p.w[1] = a->k_weight;
    p.cos = a->cos;
    p.sin = a->sin;
    p.pos = a->positions;
    p.n = a->n_tokens;
    p.max_pos = a->rot_dim ? a->max_pos : INT32_MAX;
    p.heads[0] = (int)a->n_heads;
    p.heads[1] = (int)a->n_kv_heads;
    p.hd = (int)a->head_dim;
    p.inv_hd = 1.0f / (float)p.hd;
    p.rot = (int)a->rot_dim;
    p.inter = a->interleaved != 0;
    p.eps = a->eps;
    return p;
}

int check_grid(int64_t blocks, const char* fn) {
    return blocks > INT32_MAX ? set_error(RQ_ERR_INVALID, "%s: too many rows for one call", fn) : RQ_OK;
}

template <typename T>
const void* append_fn(int nb) {
    return nb == 1   ? (const void*)kv4_append_kernel<T, 1>
           : nb == 2 ? (const void*)kv4_append_kernel<T, 2>
           : nb == 3 ? (const void*)kv4_append_kernel<T, 3>
                     : (const void*)kv4_append_kernel<T, 4>;
}
const void* append_fn(int dtype, int nb) {
    return dtype == RQ_F32 ? append_fn<float>(nb) : dtype == RQ_F16 ? append_fn<__half>(nb) : append_fn<__nv_bfloat16>(nb);
}
template <typename T>
const void* read_fn(int nb) {
    return nb == 1   ? (const void*)kv4_read_kernel<T, 1>
           : nb == 2 ? (const void*)kv4_read_kernel<T, 2>
           : nb == 3 ? (const void*)kv4_read_kernel<T, 3>
                     : (const void*)kv4_read_kernel<T, 4>;
}
const void* read_fn(int dtype, int nb) {
    return dtype == RQ_F32 ? read_fn<float>(nb) : dtype == RQ_F16 ? read_fn<__half>(nb) : read_fn<__nv_bfloat16>(nb);
}

// Tokens of an append or read CTA: four items a thread where the tokens fill the
// device anyway, else one (more where a token alone has more items than threads).
int tokens_per_cta(const rq_kv4* c, int64_t n) {
    const int64_t items = (int64_t)2 * c->n_kv * (c->head_dim / 8);
    const int64_t want = n * items > (int64_t)c->ctx->sm_count * 2048 * 4 ? 1024 : 256;
    return (int)std::max<int64_t>(1, want / items);
}

AppendP append_params(const rq_kv4* c, const void* k, int64_t kt, int64_t kh, const void* v, int64_t vt, int64_t vh,
                      const int32_t* slots, int64_t n, size_t size) {
    AppendP p{};
    p.x[0] = k;
    p.x[1] = v;
    p.tok[0] = kt;
    p.head[0] = kh;
    p.tok[1] = vt;
    p.head[1] = vh;
    p.wide[0] = wide_ok(k, kt, kh, size);
    p.wide[1] = wide_ok(v, vt, vh, size);
    p.slots = slots;
    p.n = n;
    p.n_slots = c->n_pages * c->page_size;
    p.data = c->data;
    p.page_size = c->page_size;
    p.n_kv = c->n_kv;
    p.nb = c->head_dim / 32;
    p.per_cta = tokens_per_cta(c, n);
    return p;
}

}  // namespace

int qk_norm_rope(const rq_ctx* ctx, const rq_qk_rope* a, cudaStream_t st) {
    RopeP p = rope_params(a);
    const size_t size = dtype_size(a->dtype);
    // units of E elements: 16 bytes for many rows, four elements for few (twice
    // the lanes for 16-bit types), one where sizes or alignment ask for it
    auto fits = [&](int e) { return p.hd % e == 0 && p.rot % (2 * e) == 0; };
    bool vec = fits(4);
    for (int i = 0; i < 2; i++)
        if (p.heads[i])
            vec = vec && wide_ok(p.x[i], p.xt[i], p.xh[i], size) && wide_ok(p.y[i], p.yt[i], p.yh[i], size) &&
                  ((uintptr_t)p.w[i] & 15) == 0;
    vec = vec && (((uintptr_t)p.cos | (uintptr_t)p.sin) & 15) == 0;
    const int64_t rows = p.n * (p.heads[0] + p.heads[1]);
    if (rows > INT32_MAX) return set_error(RQ_ERR_INVALID, "rq_qk_norm_rope: too many rows for one call");
    const bool many = vec && fits((int)(16 / size)) && rows * (p.hd / 8) > 2 * (int64_t)ctx->sm_count * 2048;
    const int E = many ? (int)(16 / size) : vec ? 4 : 1, U = many ? kRopeRows : 1;
    const int slots = p.rot / (2 * E) + ((p.hd - p.rot) / E + 1) / 2;
    p.lpr = 1;
    for (; p.lpr < slots && p.lpr < 32; p.lpr *= 2) p.lpr_log++;
    const int64_t groups = 256 >> p.lpr_log;
    p.q_ctas = (unsigned)((p.n * ((p.heads[0] + U - 1) / U) + groups - 1) / groups);
    const int64_t blocks = p.q_ctas + (p.n * ((p.heads[1] + U - 1) / U) + groups - 1) / groups;
    const void* fn;
    if (a->dtype == RQ_F32)
        fn = many  ? (const void*)qk_norm_rope_rows_kernel<float, kRopeRows>
             : vec ? (const void*)qk_norm_rope_kernel<float, 4, 1>
                   : (const void*)qk_norm_rope_kernel<float, 1, 4>;
    else if (a->dtype == RQ_F16)
        fn = many  ? (const void*)qk_norm_rope_rows_kernel<__half, kRopeRows>
             : vec ? (const void*)qk_norm_rope_kernel<__half, 4, 1>
                   : (const void*)qk_norm_rope_kernel<__half, 1, 4>;
    else
        fn = many  ? (const void*)qk_norm_rope_rows_kernel<__nv_bfloat16, kRopeRows>
             : vec ? (const void*)qk_norm_rope_kernel<__nv_bfloat16, 4, 1>
                   : (const void*)qk_norm_rope_kernel<__nv_bfloat16, 1, 4>;
    void* args[] = {&p};
    return launch_pdl(fn, (unsigned)blocks, 256, 0, st, args, "q/k norm and rotation kernel");
}

int qk_norm_rope_append(const rq_kv4* c, const rq_qk_rope* a, const void* v, const int64_t v_stride[2], const int32_t* slots,
                        cudaStream_t st) {
    const size_t size = dtype_size(a->dtype);
    RopeAppendP p{};
    p.r = rope_params(a);
    p.wide_q = wide_ok(p.r.x[0], p.r.xt[0], p.r.xh[0], size);
    p.wide_qo = wide_ok(p.r.y[0], p.r.yt[0], p.r.yh[0], size);
    p.a = append_params(c, a->k, a->k_stride[0], a->k_stride[1], v, v_stride[0], v_stride[1], slots, a->n_tokens, size);
    const int64_t blocks = (a->n_tokens * (a->n_heads + 2 * a->n_kv_heads) + 15) / 16;
    const int rc = check_grid(blocks, "rq_qk_norm_rope_append");
    if (rc) return rc;
    const void* fn = a->dtype == RQ_F32 ? (const void*)qk_norm_rope_append_kernel<float>
                     : a->dtype == RQ_F16 ? (const void*)qk_norm_rope_append_kernel<__half>
                                          : (const void*)qk_norm_rope_append_kernel<__nv_bfloat16>;
    void* args[] = {&p};
    return launch_pdl(fn, (unsigned)blocks, 256, 0, st, args, "q/k norm, rotation and append kernel");
}

}  // namespace rq

using namespace rq;

extern "C" {

int rq_kv4_create(rq_ctx* ctx, int64_t n_pages, int page_size, int n_kv_heads, int head_dim, rq_kv4** out) {
    if (!ctx || !out) return set_error(RQ_ERR_INVALID, "rq_kv4_create: NULL argument");
    *out = nullptr;
    if (n_pages < 1 || page_size < kKv4Tile || page_size > 4096 || page_size % kKv4Tile || n_kv_heads < 1 || n_kv_heads > 65536)
        return set_error(RQ_ERR_INVALID,
                         "rq_kv4_create: %lld pages of %d positions (a multiple of 16 up to 4096), %d kv heads",
                         (long long)n_pages, page_size, n_kv_heads);
    if (head_dim != 32 && head_dim != 64 && head_dim != 96 && head_dim != 128)
        return set_error(RQ_ERR_UNSUPPORTED, "rq_kv4_create: head_dim %d (32, 64, 96 or 128)", head_dim);
    if (n_pages > INT32_MAX / page_size)
        return set_error(RQ_ERR_INVALID, "rq_kv4_create: %lld pages of %d positions pass 2^31 slots", (long long)n_pages,
                         page_size);
    DevGuard g(ctx->device);
    rq_kv4* c = new (std::nothrow) rq_kv4();
    if (!c) return set_error(RQ_ERR_OOM, "host allocation failed");
    c->ctx = ctx;
    c->n_pages = n_pages;
    c->page_size = page_size;
    c->n_kv = n_kv_heads;
    c->head_dim = head_dim;
    c->bytes = (size_t)n_pages * n_kv_heads * (page_size / kKv4Tile) * 576 * (head_dim / 32);
    int rc = cuda_error(cudaMalloc((void**)&c->data, c->bytes), "cudaMalloc(kv4)");
    if (!rc) {
        // zero scales: positions never written read as zeros
        rc = cuda_error(cudaMemset(c->data, 0, c->bytes), "kv4 clear");
        if (!rc) rc = cuda_error(cudaDeviceSynchronize(), "kv4 clear");
        if (rc) cudaFree(c->data);
    }
    if (rc) {
        delete c;
        return rc;
    }
    *out = c;
    return RQ_OK;
}

int rq_kv4_free(rq_kv4* c) {
    if (!c) return RQ_OK;
    DevGuard g(c->ctx->device);
    cudaFree(c->data);
    delete c;
    return RQ_OK;
}

int rq_kv4_info(const rq_kv4* c, int64_t* n_pages, int* page_size, int* n_kv_heads, int* head_dim, size_t* device_bytes) {
    int rc = check_cache(c, "rq_kv4_info");
    if (rc) return rc;
    if (n_pages) *n_pages = c->n_pages;
    if (page_size) *page_size = c->page_size;
    if (n_kv_heads) *n_kv_heads = c->n_kv;
    if (head_dim) *head_dim = c->head_dim;
    if (device_bytes) *device_bytes = c->bytes;
    return RQ_OK;
}

int rq_kv4_append(rq_kv4* c, int dtype, const void* k, const int64_t k_stride[2], const void* v, const int64_t v_stride[2],
                  const int32_t* slots, int64_t n, void* stream) {
    int rc = check_cache(c, "rq_kv4_append");
    if (rc) return rc;
    const size_t size = dtype_size(dtype);
    if (!size) return set_error(RQ_ERR_UNSUPPORTED, "rq_kv4_append: dtype %d (f32 = 0, f16 = 1, bf16 = 2)", dtype);
    if (n < 0 || n > INT32_MAX || !k_stride || !v_stride)
        return set_error(RQ_ERR_INVALID, "rq_kv4_append: n = %lld, strides %s", (long long)n, k_stride && v_stride ? "given" : "NULL");
    if (n == 0) return RQ_OK;
    DevGuard g(c->ctx->device);
    rc = check_device_ptr(c->ctx, k, "rq_kv4_append", "k");
    if (!rc) rc = check_device_ptr(c->ctx, v, "rq_kv4_append", "v");
    if (!rc) rc = check_device_ptr(c->ctx, slots, "rq_kv4_append", "slots");
    if (rc) return rc;
    AppendP p = append_params(c, k, k_stride[0], k_stride[1], v, v_stride[0], v_stride[1], slots, n, size);
    const int64_t blocks = (n + p.per_cta - 1) / p.per_cta;
    rc = check_grid(blocks, "rq_kv4_append");
    if (rc) return rc;
    const void* fn = append_fn(dtype, c->head_dim / 32);
    void* args[] = {&p};
    return launch_pdl(fn, (unsigned)blocks, 256, 0, (cudaStream_t)stream, args, "kv4 append kernel");
}

int rq_kv4_read(rq_kv4* c, const int32_t* slots, int64_t n, int dtype, void* k, void* v, void* stream) {
    int rc = check_cache(c, "rq_kv4_read");
    if (rc) return rc;
    const size_t size = dtype_size(dtype);
    if (!size) return set_error(RQ_ERR_UNSUPPORTED, "rq_kv4_read: dtype %d (f32 = 0, f16 = 1, bf16 = 2)", dtype);
    if (n < 0 || n > INT32_MAX) return set_error(RQ_ERR_INVALID, "rq_kv4_read: n = %lld", (long long)n);
    if (n == 0) return RQ_OK;
    DevGuard g(c->ctx->device);
    rc = check_device_ptr(c->ctx, slots, "rq_kv4_read", "slots");
    if (!rc) rc = check_device_ptr(c->ctx, k, "rq_kv4_read", "k");
    if (!rc) rc = check_device_ptr(c->ctx, v, "rq_kv4_read", "v");
    if (rc) return rc;
    ReadP p{};
    p.data = c->data;
    p.slots = slots;
    p.n = n;
    p.n_slots = c->n_pages * c->page_size;
    p.page_size = c->page_size;
    p.n_kv = c->n_kv;
    p.x[0] = k;
    p.x[1] = v;
    p.wide = (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
    p.per_cta = tokens_per_cta(c, n);
    const int64_t blocks = (n + p.per_cta - 1) / p.per_cta;
    rc = check_grid(blocks, "rq_kv4_read");
    if (rc) return rc;
    const void* fn = read_fn(dtype, c->head_dim / 32);
    void* args[] = {&p};
    return launch_pdl(fn, (unsigned)blocks, 256, 0, (cudaStream_t)stream, args, "kv4 read kernel");
}

int rq_qk_norm_rope(rq_ctx* ctx, const rq_qk_rope* a, void* stream) {
    static const char* fn_name = "rq_qk_norm_rope";
    if (!ctx) return set_error(RQ_ERR_INVALID, "%s: NULL argument", fn_name);
    DevGuard g(ctx->device);
    int rc = check_rope(ctx, a, false, fn_name);
    if (rc) return rc;
    if (!a->n_tokens || !(a->n_heads + a->n_kv_heads)) return RQ_OK;
    return qk_norm_rope(ctx, a, (cudaStream_t)stream);
}

int rq_qk_norm_rope_append(rq_kv4* c, const rq_qk_rope* a, const void* v, const int64_t v_stride[2], const int32_t* slots,
                           void* stream) {
    static const char* fn_name = "rq_qk_norm_rope_append";
    int rc = check_cache(c, fn_name);
    if (rc) return rc;
    DevGuard g(c->ctx->device);
    rc = check_rope(c->ctx, a, true, fn_name);
    if (rc) return rc;
    if (a->head_dim != c->head_dim || a->n_kv_heads != c->n_kv)
        return set_error(RQ_ERR_INVALID, "%s: %lld kv heads of %lld, the cache holds %d of %d", fn_name,
                         (long long)a->n_kv_heads, (long long)a->head_dim, c->n_kv, c->head_dim);
    if (!v_stride) return set_error(RQ_ERR_INVALID, "%s: v_stride is NULL", fn_name);
    if (!a->n_tokens) return RQ_OK;
    rc = check_device_ptr(c->ctx, v, fn_name, "v");
    if (!rc) rc = check_device_ptr(c->ctx, slots, fn_name, "slots");
    if (rc) return rc;
    return qk_norm_rope_append(c, a, v, v_stride, slots, (cudaStream_t)stream);
}

}  // extern "C"
