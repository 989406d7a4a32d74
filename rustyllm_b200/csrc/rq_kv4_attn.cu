// rq_kv4_attn.cu -- attention over the 4-bit paged cache (rq_kv4.cuh), for
// single new tokens, drafted tokens and prompt chunks.
//
// For a query row q and the positions j it sees, with K = (c - 8) d per block
// of 32 elements:
//   s_j = scale * sum_b dK_jb (q_b . (cK_jb - 8)),  o = sum_j softmax(s)_j V_j.
// The codes c - 8 are exact in f16, so both products run on mma.m16n8k16
// without rounding the cache: q is scaled by a power of two to [-1, 1] and
// split into f16 hi + lo (f32 input; 16-bit inputs need hi alone), the K
// scales multiply the f32 block sums, and the V scales multiply the
// probabilities, P_jb = p_j dV_jb, which again enter as hi + lo (one f16 for
// 16-bit outputs, whose own rounding is coarser).  For f32 the hi and lo parts
// are the two row halves of one m16 operand: eight query rows a tile, no
// extra instructions.  To keep P_jb inside f16's range whatever the scale of V,
// the running maximum is taken over s_j + log2 max_b dV_jb (base 2), so that
// |P_jb| <= 1 (2^8 between lazy rescales) with the largest near 1; 22 bits
// then hold f32's accuracy.  Sums stay in f32 throughout.
#include <algorithm>

#include "rq_async.cuh"
#include "rq_kv4.cuh"

namespace rq {
namespace {

constexpr int kWarps = 4;    // warps of a CTA, each walking its own tiles
constexpr int kStages = 4;   // tiles in flight per warp
constexpr float kLazy = 8.0f;  // rescale once the maximum grew by 2^8

enum Mode { kSplit8 = 0, kOne8 = 1, kOne16 = 2 };  // rows 8 hi + lo, 8, 16

struct AttnP {
    const uint8_t* data;
    int64_t n_pages;
    int page_size, n_kv;
    const void* q;
    int64_t qt, qh;
    void* out;
    int64_t ot, oh;
    bool wide;
    int64_t n_tokens;
    int n_heads, group, batch, max_q, row_tiles, splits;
    const int32_t* cu_q;
    const int32_t* kv_lens;
    const int32_t* table;
    int64_t table_stride, table_width;
    int64_t window;
    float scale;  // times log2(e)
    float* part;  // [n_tokens * n_heads][splits][head_dim]
    float2* ml;   // [n_tokens * n_heads][splits]
    int* err;
};

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// nibbles 0 and 4 (even) or 1 and 5 (odd) of w as f16 pairs c - 8: a nibble
// placed in the mantissa of 1024 (or, four bits up, of 64) is that value + c
__device__ __forceinline__ uint32_t codes_even(uint32_t w) {
    const uint32_t h = (w & 0x000F000Fu) | 0x64006400u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6408)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t codes_odd(uint32_t w) {
    const uint32_t h = (w & 0x00F000F0u) | 0x54005400u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x5480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// The 2 NB words of this lane in a code region
template <int NB>
__device__ __forceinline__ void load_words(const uint8_t* region, int lane, uint32_t (&w)[2 * NB]) {
#pragma unroll
    for (int p = 0; p < NB / 2; p++) {
        const uint4 v = *reinterpret_cast<const uint4*>(region + p * 512 + lane * 16);
        w[4 * p] = v.x;
        w[4 * p + 1] = v.y;
        w[4 * p + 2] = v.z;
        w[4 * p + 3] = v.w;
    }
    if (NB & 1) {
        const uint2 v = *reinterpret_cast<const uint2*>(region + (NB / 2) * 512 + lane * 8);
        w[2 * NB - 2] = v.x;
        w[2 * NB - 1] = v.y;
    }
}

// The rows of one (sequence, kv head, row tile): what main and join kernels
// agree on.
struct Rows {
    int b, kvh, r0, rows, n_q, q0;
    int64_t pos0;  // position of query 0
    int tile0, tile1, per;  // tiles seen by any row; tiles of a split
};

template <int R>
__device__ __forceinline__ bool find_rows(const AttnP& p, int64_t unit, Rows& o) {
    const int rt = (int)(unit % p.row_tiles);
    unit /= p.row_tiles;
    o.kvh = (int)(unit % p.n_kv);
    o.b = (int)(unit / p.n_kv);
    o.q0 = p.cu_q ? p.cu_q[o.b] : o.b;
    o.n_q = p.cu_q ? min(max(p.cu_q[o.b + 1] - o.q0, 0), p.max_q) : 1;
    o.rows = o.n_q * p.group;
    o.r0 = rt * R;
    if (o.r0 >= o.rows) return false;
    const int64_t len = max(p.kv_lens[o.b], 0);
    const int64_t held = min(len, p.table_width * p.page_size);
    o.pos0 = len - o.n_q;
    const int i0 = o.r0 / p.group, i1 = min(o.n_q - 1, (o.r0 + R - 1) / p.group);
    const int64_t hi = max((int64_t)0, min(held, o.pos0 + i1 + 1));
    const int64_t lo = p.window > 0 ? max((int64_t)0, o.pos0 + i0 - p.window + 1) : 0;
    o.tile0 = (int)(lo / kKv4Tile);
    o.tile1 = max(o.tile0, (int)((hi + kKv4Tile - 1) / kKv4Tile));
    o.per = max((o.tile1 - o.tile0 + p.splits - 1) / p.splits, kWarps);
    return true;
}

template <int NB, int MODE, typename T>
__global__ void __launch_bounds__(kWarps * 32) kv4_attn_kernel(const __grid_constant__ AttnP p) {
    using Rec = Kv4Rec<NB>;
    constexpr int R = MODE == kOne16 ? 16 : 8;
    constexpr int H = MODE == kOne16 ? 2 : 1;  // rows a lane
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[kWarps][kStages];
    __shared__ float s_m[kWarps][R], s_l[kWarps][R];
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int split = (int)(blockIdx.x % p.splits);
    Rows o;
    if (!find_rows<R>(p, blockIdx.x / p.splits, o)) return;
    const int t0 = o.tile0 + split * o.per, t1 = min(t0 + o.per, o.tile1);
    if (p.splits > 1 && t0 >= t1) return;  // the join does not read this split
    const int tiles = p.page_size / kKv4Tile;
    const int n_mine = t1 > t0 + warp ? (t1 - t0 - warp + kWarps - 1) / kWarps : 0;  // tiles t0 + warp + k * kWarps
    const uint8_t* ring = smem + warp * kStages * Rec::kBytes;
    const uint32_t ring32 = smem_u32(ring), bar32 = smem_u32(&bars[warp][0]);
    if (lane == 0) {
        for (int s = 0; s < kStages; s++) mbar_init(bar32 + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    // pages of tiles k = base .. base + 31 of this warp, one a lane; -1: not in the cache
    int page_base = -32, my_page = -1;
    auto page_of = [&](int k) {
        if (k >= page_base + 32) {
            page_base = k & ~31;
            const int kk = page_base + lane;
            my_page = -1;
            if (kk < n_mine) {
                const int64_t col = (int64_t)(t0 + warp + kk * kWarps) / tiles;
                const int pg = p.table[o.b * p.table_stride + col];
                my_page = pg >= 0 && pg < p.n_pages ? pg : -1;
            }
        }
        return __shfl_sync(0xffffffffu, my_page, k & 31);
    };
    const uint64_t pol = policy_evict_normal();
    uint32_t absent = 0;  // bit per stage: the tile there is not in the cache
    auto issue = [&](int k) {
        const int s = k % kStages;
        const int pg = page_of(k);
        absent = (absent & ~(1u << s)) | ((pg < 0 ? 1u : 0u) << s);
        if (pg >= 0 && lane == 0) {
            const int tile = t0 + warp + k * kWarps;
            const uint8_t* src = p.data + (((int64_t)pg * p.n_kv + o.kvh) * tiles + tile % tiles) * Rec::kBytes;
            mbar_expect_tx(bar32 + 8 * s, Rec::kBytes);
            bulk_g2s(ring32 + s * Rec::kBytes, src, Rec::kBytes, bar32 + 8 * s, pol);
        }
    };
    for (int k = 0; k < min(kStages, n_mine); k++) issue(k);

    // ---- query rows: normalise by a power of two, split
    uint32_t aq[NB][2][4];
    float qs[H];       // back from the normalised row, times the softmax scale
    int64_t rpos[H];   // position of the row's query; -1: no row
#pragma unroll
    for (int h = 0; h < H; h++) {
        const int r = o.r0 + g + 8 * h;
        const int i = r / p.group;
        const int64_t tok = (int64_t)o.q0 + i;
        const bool ok = r < o.rows && tok >= 0 && tok < p.n_tokens;
        rpos[h] = ok ? o.pos0 + i : -1;
        float x[NB][8];
        float mx = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[b][e] = 0.0f;
            if (ok)
                load8(static_cast<const T*>(p.q) + tok * p.qt + (o.kvh * p.group + r % p.group) * p.qh + 32 * b + 8 * t,
                      p.wide, x[b]);
#pragma unroll
            for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[b][e]));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // 2^e with mx in [2^(e-1), 2^e), kept where its reciprocal is finite;
        // an infinite or NaN row stays so
        int e2 = 0;
        if (mx > 0.0f && mx < INFINITY) frexpf(mx, &e2);
        e2 = max(-120, min(120, e2));
        const float inv = __int_as_float((127 - e2) << 23);
        qs[h] = __int_as_float((127 + e2) << 23) * p.scale;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int j = 0; j < 2; j++) {  // elements 4 s + 2 j, + 1: operand half j of step s
                    const float f0 = x[b][4 * s + 2 * j] * inv, f1 = x[b][4 * s + 2 * j + 1] * inv;
                    const uint32_t hi = pack(f0, f1);
                    if (MODE == kOne16) {
                        aq[b][s][2 * j + h] = hi;
                    } else {
                        aq[b][s][2 * j] = hi;
                        if (MODE == kSplit8) {
                            const float2 back = unpack(hi);
                            aq[b][s][2 * j + 1] = pack(f0 - back.x, f1 - back.y);
                        } else {
                            aq[b][s][2 * j + 1] = 0u;
                        }
                    }
                }
    }
    const int i_first = o.r0 / p.group, i_last = min(o.n_q - 1, (o.r0 + R - 1) / p.group);
    const int64_t held = min((int64_t)max(p.kv_lens[o.b], 0), p.table_width * p.page_size);

    float oacc[NB][4][4];
    float m[H], l[H];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) oacc[b][n][i] = 0.0f;
#pragma unroll
    for (int h = 0; h < H; h++) {
        m[h] = -INFINITY;
        l[h] = 0.0f;
    }
    uint32_t phase = 0;  // bit per stage
    bool bad = false;
    for (int k = 0; k < n_mine; k++) {
        const int s = k % kStages;
        if ((absent >> s) & 1u) {  // not in the cache: nothing to see
            if (k + kStages < n_mine) issue(k + kStages);
            continue;
        }
        if (!mbar_wait(bar32 + 8 * s, (phase >> s) & 1u)) bad = true;
        if (__any_sync(0xffffffffu, bad)) {
            bad = true;
            break;
        }
        phase ^= 1u << s;
        const uint8_t* rec = ring + s * Rec::kBytes;
        uint32_t kw[2 * NB], vw[2 * NB];
        uint2 ks[NB], vs[NB];  // scales of tokens 4 t .. 4 t + 3
        load_words<NB>(rec, lane, kw);
        load_words<NB>(rec + Rec::kV, lane, vw);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            ks[b] = *reinterpret_cast<const uint2*>(rec + Rec::kKs + t * 8 * NB + 8 * b);
            vs[b] = *reinterpret_cast<const uint2*>(rec + Rec::kVs + t * 8 * NB + 8 * b);
        }
        __syncwarp();
        if (k + kStages < n_mine) issue(k + kStages);

        // ---- scores: sc[n][.] of tokens 4 t + 2 n, + 1
        float sc[2][2 * H];
#pragma unroll
        for (int n = 0; n < 2; n++) {
#pragma unroll
            for (int i = 0; i < 2 * H; i++) sc[n][i] = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const uint32_t w = kw[2 * b + n], w8 = w >> 8;
                mma16816(c, aq[b][0], codes_even(w), codes_odd(w));
                mma16816(c, aq[b][1], codes_even(w8), codes_odd(w8));
                const float2 d = unpack(n ? ks[b].y : ks[b].x);
                if (MODE == kOne16) {
                    sc[n][0] = fmaf(c[0], d.x, sc[n][0]);
                    sc[n][1] = fmaf(c[1], d.y, sc[n][1]);
                    sc[n][2 * H - 2] = fmaf(c[2], d.x, sc[n][2 * H - 2]);
                    sc[n][2 * H - 1] = fmaf(c[3], d.y, sc[n][2 * H - 1]);
                } else {
                    sc[n][0] = fmaf(MODE == kSplit8 ? c[0] + c[2] : c[0], d.x, sc[n][0]);
                    sc[n][1] = fmaf(MODE == kSplit8 ? c[1] + c[3] : c[1], d.y, sc[n][1]);
                }
            }
        }
        // ---- log2 of each token's largest V scale
        float lg[4];
        {
            float2 d01 = make_float2(0.0f, 0.0f), d23 = d01;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float2 u = unpack(vs[b].x), v = unpack(vs[b].y);
                d01.x = fmaxf(d01.x, fabsf(u.x));
                d01.y = fmaxf(d01.y, fabsf(u.y));
                d23.x = fmaxf(d23.x, fabsf(v.x));
                d23.y = fmaxf(d23.y, fabsf(v.y));
            }
            lg[0] = lg2(fmaxf(d01.x, 5.9604645e-8f));
            lg[1] = lg2(fmaxf(d01.y, 5.9604645e-8f));
            lg[2] = lg2(fmaxf(d23.x, 5.9604645e-8f));
            lg[3] = lg2(fmaxf(d23.y, 5.9604645e-8f));
        }
        const int64_t j0 = (int64_t)(t0 + warp + k * kWarps) * kKv4Tile;
        const bool full = j0 + kKv4Tile <= held && j0 + kKv4Tile - 1 <= o.pos0 + i_first &&
                          (p.window <= 0 || j0 > o.pos0 + i_last - p.window);
        uint32_t hidden[H];  // bit i: token 4 t + i is not seen by the row
        float pr[H][4];
        float mx[H];
#pragma unroll
        for (int h = 0; h < H; h++) {
            hidden[h] = 0;
            mx[h] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                pr[h][i] = sc[i >> 1][2 * h + (i & 1)] * qs[h];
                if (!full) {
                    const int64_t j = j0 + 4 * t + i;
                    if (j >= held || j > rpos[h] || (p.window > 0 && j <= rpos[h] - p.window)) {
                        hidden[h] |= 1u << i;
                        pr[h][i] = -INFINITY;
                    }
                }
                mx[h] = fmaxf(mx[h], pr[h][i] + lg[i]);
            }
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        }
        bool grow = false;
#pragma unroll
        for (int h = 0; h < H; h++) grow |= mx[h] > m[h] + kLazy || (m[h] == -INFINITY && mx[h] > -INFINITY);
        if (__any_sync(0xffffffffu, grow)) {
            float al[H];
#pragma unroll
            for (int h = 0; h < H; h++) {
                const float mn = fmaxf(m[h], mx[h]);
                al[h] = m[h] == -INFINITY ? 0.0f : ex2(m[h] - mn);
                m[h] = mn;
                l[h] *= al[h];
            }
            // rows g and g + 8 of the accumulators: in the split modes both
            // halves belong to row g
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    oacc[b][n][0] *= al[0];
                    oacc[b][n][1] *= al[0];
                    oacc[b][n][2] *= al[H - 1];
                    oacc[b][n][3] *= al[H - 1];
                }
        }
#pragma unroll
        for (int h = 0; h < H; h++) {
            const float base = m[h] == -INFINITY ? 0.0f : m[h];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                pr[h][i] = ex2(pr[h][i] - base);
                l[h] += pr[h][i];
            }
        }
        // ---- values
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const float2 d01 = unpack(vs[b].x), d23 = unpack(vs[b].y);
            uint32_t a[4];
#pragma unroll
            for (int h = 0; h < H; h++) {
                float f[4] = {pr[h][0] * d01.x, pr[h][1] * d01.y, pr[h][2] * d23.x, pr[h][3] * d23.y};
                if (!full) {  // whatever a hidden position holds (a NaN scale too) does not enter
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if ((hidden[h] >> i) & 1u) f[i] = 0.0f;
                }
                const uint32_t h01 = pack(f[0], f[1]), h23 = pack(f[2], f[3]);
                if (MODE == kOne16) {
                    a[h] = h01;
                    a[2 + h] = h23;
                } else {
                    a[0] = h01;
                    a[2] = h23;
                    a[1] = a[3] = 0u;
                    if (MODE == kSplit8) {
                        const float2 u = unpack(h01), v = unpack(h23);
                        a[1] = pack(f[0] - u.x, f[1] - u.y);
                        a[3] = pack(f[2] - v.x, f[3] - v.y);
                    }
                }
            }
            const uint32_t w0 = vw[2 * b], w1 = vw[2 * b + 1];
            mma16816(oacc[b][0], a, codes_even(w0), codes_even(w1));
            mma16816(oacc[b][1], a, codes_odd(w0), codes_odd(w1));
            mma16816(oacc[b][2], a, codes_even(w0 >> 8), codes_even(w1 >> 8));
            mma16816(oacc[b][3], a, codes_odd(w0 >> 8), codes_odd(w1 >> 8));
        }
    }
    if (bad) {
        // a copy did not arrive within the bound: report it, and give the
        // copies still in flight the same bound before the memory goes
        if (lane == 0) {
            atomicExch(p.err, 1);
            for (int s = 0; s < kStages; s++)
                if (!((absent >> s) & 1u)) mbar_wait(bar32 + 8 * s, (phase >> s) & 1u);
        }
        __syncwarp();
    }
    // ---- join the warps: each one's m, l and row sums through shared memory
    // (the rings are drained: every issued copy has been waited for)
    float* so = reinterpret_cast<float*>(smem) + warp * (R * 32 * NB);
    __syncthreads();
#pragma unroll
    for (int h = 0; h < H; h++) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if (t == 0) {
            s_m[warp][g + 8 * h] = m[h];
            s_l[warp][g + 8 * h] = l[h];
        }
    }
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const int d = 32 * b + 8 * n + 2 * t;
            float2 v = make_float2(oacc[b][n][0], oacc[b][n][1]);
            if (MODE == kOne16) {
                *reinterpret_cast<float2*>(so + (g + 8) * 32 * NB + d) = make_float2(oacc[b][n][2], oacc[b][n][3]);
            } else if (MODE == kSplit8) {
                v.x += oacc[b][n][2];
                v.y += oacc[b][n][3];
            }
            *reinterpret_cast<float2*>(so + g * 32 * NB + d) = v;
        }
    __syncthreads();
    const float* all = reinterpret_cast<const float*>(smem);
    for (int e = threadIdx.x; e < R * 32 * NB; e += kWarps * 32) {
        const int row = e / (32 * NB), d = e % (32 * NB);
        const int r = o.r0 + row;
        if (r >= o.rows) break;
        const int64_t tok = (int64_t)o.q0 + r / p.group;
        if (tok < 0 || tok >= p.n_tokens) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; w++) M = fmaxf(M, s_m[w][row]);
        float L = 0.0f, acc = 0.0f;
        if (M > -INFINITY) {
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float f = ex2(s_m[w][row] - M);
                L = fmaf(f, s_l[w][row], L);
                acc = fmaf(f, all[w * (R * 32 * NB) + e], acc);
            }
        }
        const int head = o.kvh * p.group + r % p.group;
        if (p.splits == 1) {
            static_cast<T*>(p.out)[tok * p.ot + head * p.oh + d] = from_f32<T>(M > -INFINITY ? acc / L : 0.0f);
        } else {
            const int64_t at = (tok * p.n_heads + head) * p.splits + split;
            p.part[at * (32 * NB) + d] = acc;
            if (d == 0) p.ml[at] = make_float2(M, L);
        }
    }
}

// Joins the splits of a row in split order; one CTA of head_dim threads a row.
template <int NB, int R, typename T>
__global__ void __launch_bounds__(32 * NB) kv4_join_kernel(const __grid_constant__ AttnP p) {
    pdl_wait();
    Rows o;
    if (!find_rows<R>(p, blockIdx.x / R, o)) return;
    const int r = o.r0 + (int)(blockIdx.x % R);
    if (r >= o.rows) return;
    const int64_t tok = (int64_t)o.q0 + r / p.group;
    if (tok < 0 || tok >= p.n_tokens) return;
    const int head = o.kvh * p.group + r % p.group, d = threadIdx.x;
    const int used = (o.tile1 - o.tile0 + o.per - 1) / o.per;  // splits that had tiles
    const int64_t at = (tok * p.n_heads + head) * p.splits;
    float M = -INFINITY;
    for (int s = 0; s < used; s++) M = fmaxf(M, p.ml[at + s].x);
    float L = 0.0f, acc = 0.0f;
    if (M > -INFINITY) {
#pragma unroll 4
        for (int s = 0; s < used; s++) {
            const float2 v = p.ml[at + s];
            const float f = ex2(v.x - M);
            L = fmaf(f, v.y, L);
            acc = fmaf(f, p.part[(at + s) * (32 * NB) + d], acc);
        }
    }
    static_cast<T*>(p.out)[tok * p.ot + head * p.oh + d] = from_f32<T>(M > -INFINITY ? acc / L : 0.0f);
}

// f32 queries take the hi + lo rows, 16-bit ones one operand row each (eight
// or sixteen rows a tile)
template <int NB, typename T>
const void* main_fn(int mode) {
    if constexpr (sizeof(T) == 4) return (const void*)kv4_attn_kernel<NB, kSplit8, T>;
    else return mode == kOne8 ? (const void*)kv4_attn_kernel<NB, kOne8, T> : (const void*)kv4_attn_kernel<NB, kOne16, T>;
}
template <int NB, typename T>
const void* join_fn(int mode) {
    if constexpr (sizeof(T) == 4) return (const void*)kv4_join_kernel<NB, 8, T>;
    else return mode == kOne8 ? (const void*)kv4_join_kernel<NB, 8, T> : (const void*)kv4_join_kernel<NB, 16, T>;
}
template <typename T>
const void* pick(int nb, bool join, int mode) {
    switch (nb) {
    case 1: return join ? join_fn<1, T>(mode) : main_fn<1, T>(mode);
    case 2: return join ? join_fn<2, T>(mode) : main_fn<2, T>(mode);
    case 3: return join ? join_fn<3, T>(mode) : main_fn<3, T>(mode);
    default: return join ? join_fn<4, T>(mode) : main_fn<4, T>(mode);
    }
}
const void* pick(int dtype, int nb, bool join, int mode) {
    return dtype == RQ_F32 ? pick<float>(nb, join, mode)
           : dtype == RQ_F16 ? pick<__half>(nb, join, mode)
                             : pick<__nv_bfloat16>(nb, join, mode);
}

struct Plan {
    int mode, R, row_tiles, splits;
    int64_t units;
};

int check_query(const rq_kv4* c, const rq_kv4_query* a, const char* fn) {
    if (!c || !a) return set_error(RQ_ERR_INVALID, "%s: NULL argument", fn);
    if (a->dtype != RQ_F32 && a->dtype != RQ_F16 && a->dtype != RQ_BF16)
        return set_error(RQ_ERR_UNSUPPORTED, "%s: dtype %d (f32 = 0, f16 = 1, bf16 = 2)", fn, a->dtype);
    if (a->n_heads < 1 || a->n_heads > 65536 || a->n_heads % c->n_kv)
        return set_error(RQ_ERR_INVALID, "%s: %lld query heads over %d kv heads", fn, (long long)a->n_heads, c->n_kv);
    if (a->batch < 0 || a->batch > INT32_MAX - 1 || a->n_tokens < 0 || a->n_tokens > INT32_MAX || a->max_q < 1 ||
        a->max_q > (1 << 24) || a->table_width < 0 || a->table_width > INT32_MAX || a->max_len < 0 || a->window < 0)
        return set_error(RQ_ERR_INVALID,
                         "%s: batch %lld, n_tokens %lld, max_q %lld, table_width %lld, max_len %lld, window %lld", fn,
                         (long long)a->batch, (long long)a->n_tokens, (long long)a->max_q, (long long)a->table_width,
                         (long long)a->max_len, (long long)a->window);
    if (a->table_width * c->page_size > INT32_MAX)
        return set_error(RQ_ERR_INVALID, "%s: a table of %lld pages passes 2^31 positions", fn, (long long)a->table_width);
    if (!a->cu_q && a->n_tokens < a->batch)
        return set_error(RQ_ERR_INVALID, "%s: %lld tokens for %lld sequences of one query each", fn, (long long)a->n_tokens,
                         (long long)a->batch);
    if (!(a->scale == a->scale) || a->scale - a->scale != 0.0f)
        return set_error(RQ_ERR_INVALID, "%s: scale is not finite", fn);
    return RQ_OK;
}

Plan make_plan(const rq_kv4* c, const rq_kv4_query* a) {
    Plan pl{};
    const int64_t group = a->n_heads / c->n_kv;
    const int64_t rows = group * (a->cu_q ? a->max_q : 1);
    pl.mode = a->dtype == RQ_F32 ? kSplit8 : rows <= 8 ? kOne8 : kOne16;
    pl.R = pl.mode == kOne16 ? 16 : 8;
    pl.row_tiles = (int)((rows + pl.R - 1) / pl.R);
    pl.units = a->batch * c->n_kv * pl.row_tiles;
    // Splits of the long axis: enough CTAs for about two waves, but none
    // shorter than two tiles a warp
    int64_t len = a->table_width * c->page_size;
    if (a->max_len > 0) len = std::min(len, a->max_len);
    if (a->window > 0) len = std::min(len, a->window + a->max_q);
    const int64_t tiles = (len + kKv4Tile - 1) / kKv4Tile;
    const int64_t want = ((int64_t)c->ctx->sm_count * 6 + pl.units - 1) / std::max<int64_t>(pl.units, 1);
    pl.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, tiles / (2 * kWarps)));
    return pl;
}

size_t plan_bytes(const rq_kv4* c, const rq_kv4_query* a, const Plan& pl) {
    if (pl.splits == 1) return 0;
    return (size_t)a->n_tokens * a->n_heads * pl.splits * ((size_t)c->head_dim * 4 + 8);
}

}  // namespace

int kv4_attention(const rq_kv4* c, const rq_kv4_query* a, int* err, cudaStream_t st) {
    const Plan pl = make_plan(c, a);
    const size_t need = plan_bytes(c, a, pl);
    if (need) {
        if (a->workspace_bytes < need)
            return set_error(RQ_ERR_INVALID, "rq_kv4_attention: workspace of %zu bytes, need %zu", a->workspace_bytes, need);
        if (!a->workspace || (uintptr_t)a->workspace & 15) return set_error(RQ_ERR_INVALID, "rq_kv4_attention: workspace is NULL or not 16-byte aligned");
    }
    if (pl.units * pl.splits > INT32_MAX || pl.units * pl.R > INT32_MAX)
        return set_error(RQ_ERR_INVALID, "rq_kv4_attention: too many rows for one call");
    const size_t size = a->dtype == RQ_F32 ? 4 : 2;
    AttnP p{};
    p.data = c->data;
    p.n_pages = c->n_pages;
    p.page_size = c->page_size;
    p.n_kv = c->n_kv;
    p.q = a->q;
    p.qt = a->q_stride[0];
    p.qh = a->q_stride[1];
    p.out = a->out;
    p.ot = a->out_stride[0];
    p.oh = a->out_stride[1];
    p.wide = (((uintptr_t)a->q | (uintptr_t)(p.qt * (int64_t)size) | (uintptr_t)(p.qh * (int64_t)size)) & 15) == 0;
    p.n_tokens = a->n_tokens;
    p.n_heads = (int)a->n_heads;
    p.group = (int)(a->n_heads / c->n_kv);
    p.batch = (int)a->batch;
    p.max_q = a->cu_q ? (int)a->max_q : 1;
    p.row_tiles = pl.row_tiles;
    p.splits = pl.splits;
    p.cu_q = a->cu_q;
    p.kv_lens = a->kv_lens;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.table_width = a->table_width;
    p.window = a->window;
    p.scale = a->scale * 1.44269504088896340736f;
    p.part = static_cast<float*>(a->workspace);
    if (need) {
        const int64_t rows = a->n_tokens * a->n_heads * pl.splits;
        p.ml = reinterpret_cast<float2*>(p.part + rows * c->head_dim);
    }
    p.err = err;
    const int nb = c->head_dim / 32;
    const size_t smem = (size_t)kWarps * std::max(kStages * 576 * nb, pl.R * 32 * nb * 4);
    const void* fn = pick(a->dtype, nb, false, pl.mode);
    void* args[] = {&p};
    const int rc = launch_pdl(fn, (unsigned)(pl.units * pl.splits), kWarps * 32, smem, st, args,
                    "kv4 attention kernel");
    if (rc || pl.splits == 1) return rc;
    const void* jf = pick(a->dtype, nb, true, pl.mode);
    return launch_pdl(jf, (unsigned)(pl.units * pl.R), 32 * nb, 0, st, args, "kv4 join kernel");
}


}  // namespace rq

using namespace rq;

extern "C" {

int rq_kv4_attention_workspace(const rq_kv4* c, const rq_kv4_query* a, size_t* bytes) {
    if (!bytes) return set_error(RQ_ERR_INVALID, "rq_kv4_attention_workspace: NULL argument");
    int rc = check_query(c, a, "rq_kv4_attention_workspace");
    if (rc) return rc;
    *bytes = plan_bytes(c, a, make_plan(c, a));
    return RQ_OK;
}

int rq_kv4_attention(rq_kv4* c, const rq_kv4_query* a, void* stream) {
    static const char* fn_name = "rq_kv4_attention";
    int rc = check_query(c, a, fn_name);
    if (rc) return rc;
    if (!a->batch || !a->n_tokens) return RQ_OK;
    DevGuard g(c->ctx->device);
    const rq_ctx* ctx = c->ctx;
    rc = check_device_ptr(ctx, a->q, fn_name, "q");
    if (!rc) rc = check_device_ptr(ctx, a->out, fn_name, "out");
    if (!rc) rc = check_device_ptr(ctx, a->kv_lens, fn_name, "kv_lens");
    if (!rc && a->cu_q) rc = check_device_ptr(ctx, a->cu_q, fn_name, "cu_q");
    if (!rc && a->table_width) rc = check_device_ptr(ctx, a->block_table, fn_name, "block_table");
    if (!rc && a->workspace) rc = check_device_ptr(ctx, a->workspace, fn_name, "workspace");
    return rc ? rc : kv4_attention(c, a, ctx->derr, (cudaStream_t)stream);
}

}  // extern "C"
