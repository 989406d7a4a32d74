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
// probabilities, P_jb = p_j dV_jb.  For f32 the hi and lo parts are the two row
// halves of one m16 operand: eight query rows a tile, no extra instructions.
//
// P enters as f16: for f32, p = ph + pl (22 bits) and ph d = h + r exactly (h
// the rounded product, r = fma(ph, d, -h)), so P = h + (r + pl d) costs three
// packed operations a pair of tokens; 16-bit outputs take h alone (two
// roundings of 2^-12, below the output's own).  f16's range is kept whatever
// the scale of V: the scales are divided by a power of two 2^E that follows
// the largest one seen, and the running maximum m is taken over s_j + log2 of
// the lane's largest scale (not below 2^-7), so that |P| <= 2^8 with the
// largest near 1, and p <= 2^15.  m and E move lazily, when P would pass 2^8
// or a scale 2^E.  Sums stay in f32 throughout.
//
// Two forms of one kernel:
//  - few rows (decode): every warp of a CTA walks its own tiles of 16
//    positions for the same rows, so one row tile uses all lanes of the GPU;
//    its operands are built in registers from the record that one bulk copy
//    brought to shared memory.  The warps join through shared memory, the
//    splits of the long axis through a second launch.
//  - many rows (prompts): the warps hold different rows; each turns one record
//    into f16 operands in shared memory and all use them, which takes the
//    unpacking (144 of about 340 instructions a tile) off three of four warps.
#include <algorithm>

#include "rq_async.cuh"
#include "rq_kv4.cuh"

namespace rq {
namespace {

constexpr int kWarps = 4;       // warps of a CTA
constexpr int kStages = 4;      // records in flight per warp (few rows)
constexpr int kStagesRows = 2;  // (many rows: a step of kWarps records each)
constexpr float kLazy = 8.0f;   // log2 of the largest |P|
constexpr float kFloor = 0.0078125f;  // 2^-7

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
    int64_t table_stride;
    int table_slots;  // positions of a table row
    int window;       // 0: none
    float scale;      // times log2(e)
    float* part;  // [n_tokens * n_heads][splits][head_dim]
    float2* ml;   // [n_tokens * n_heads][splits]
    int* err;
};

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the same from a zero accumulator
__device__ __forceinline__ void mma16816_0(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
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
// two f32 operations an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
        " fma.rn.f32x2 w, x, y, z;\n mov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 x, y, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 w, x, y;\n mov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
// nibbles 0 and 4 (even) or 1 and 5 (odd) of w as f16 pairs c - 8: a nibble
// placed in the mantissa of 1024 (or, four bits up, of 64) is that value + c
__device__ __forceinline__ uint32_t codes_even(uint32_t w) {
    return as_u32(__hsub2(as_h2((w & 0x000F000Fu) | 0x64006400u), __half2half2(__ushort_as_half(0x6408))));
}
__device__ __forceinline__ uint32_t codes_odd(uint32_t w) {
    return as_u32(__hsub2(as_h2((w & 0x00F000F0u) | 0x54005400u), __half2half2(__ushort_as_half(0x5480))));
}
__device__ __forceinline__ uint32_t pack(float a, float b) { return as_u32(__floats2half2_rn(a, b)); }
__device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(as_h2(v)); }

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

// The four operand words of one code word of K (two steps of two), of two
// words of V (four column tiles of two)
__device__ __forceinline__ uint4 k_operands(uint32_t w) {
    return make_uint4(codes_even(w), codes_odd(w), codes_even(w >> 8), codes_odd(w >> 8));
}

// The rows of one (sequence, kv head, row tile of R): what the main and the
// join kernel agree on.
struct Rows {
    int b, kvh, r0, rows, n_q, q0;
    int pos0, held;         // position of query 0; positions that the table can hold
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
    const int len = max(p.kv_lens[o.b], 0);
    o.held = min(len, p.table_slots);
    o.pos0 = len - o.n_q;
    const int i0 = o.r0 / p.group, i1 = min(o.n_q - 1, (o.r0 + R - 1) / p.group);
    const int hi = max(0, min(o.held, o.pos0 + i1 + 1));
    const int lo = p.window > 0 ? max(0, o.pos0 + i0 - p.window + 1) : 0;
    o.tile0 = lo / kKv4Tile;
    o.tile1 = max(o.tile0, hi / kKv4Tile + (hi % kKv4Tile != 0));
    o.per = max((o.tile1 - o.tile0 + p.splits - 1) / p.splits, kWarps);
    return true;
}

// One warp's query rows, running sums and the work on one tile.
template <int NB, int MODE, typename T>
struct Warp {
    static constexpr int R = MODE == kOne16 ? 16 : 8;
    static constexpr int H = MODE == kOne16 ? 2 : 1;  // rows a lane
    uint32_t aq[NB][2][4];
    float qs[H];      // back from the normalised row, times the softmax scale
    int rpos[H];      // position of the row's query; -1: no row
    float oacc[NB][4][4];
    float m[H], l[H];
    float E;
    float bound;      // 2^E
    __half2 inv;      // 2^-E
    int full0, full1;      // tiles that every row sees whole
    int seen;              // positions that any row sees end here

    __device__ __forceinline__ void init(const AttnP& p, const Rows& o, int r0, int g, int t) {
#pragma unroll
        for (int h = 0; h < H; h++) {
            const int r = r0 + g + 8 * h;
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
            // 2^e with mx in [2^(e-1), 2^e), kept where its reciprocal is
            // finite; an infinite or NaN row stays so
            int e2 = 0;
            if (mx > 0.0f && mx < INFINITY) frexpf(mx, &e2);
            e2 = max(-120, min(120, e2));
            const float down = __int_as_float((127 - e2) << 23);
            qs[h] = __int_as_float((127 + e2) << 23) * p.scale;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int s = 0; s < 2; s++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {  // elements 4 s + 2 j, + 1: operand half j of step s
                        const float f0 = x[b][4 * s + 2 * j] * down, f1 = x[b][4 * s + 2 * j + 1] * down;
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
            m[h] = -INFINITY;
            l[h] = 0.0f;
        }
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) oacc[b][n][i] = 0.0f;
        set_scale(-15);
        const int i0 = r0 / p.group, i1 = min(o.n_q - 1, (r0 + R - 1) / p.group);
        full1 = max(0, min(o.held, o.pos0 + i0 + 1)) / kKv4Tile;
        const int before = o.pos0 + i1 - p.window;  // positions up to here the last row no longer sees
        full0 = p.window > 0 && before >= 0 ? before / kKv4Tile + 1 : 0;
        seen = min(o.held, o.pos0 + i1 + 1);
    }
    __device__ __forceinline__ void set_scale(int e) {
        E = (float)e;
        bound = __int_as_float((127 + e) << 23);
        inv = __float2half2_rn(__int_as_float((127 - e) << 23));
    }
    __device__ __forceinline__ void scale_rows(const float (&f)[H]) {
        // rows g and g + 8 of the accumulators: in the 8-row modes both
        // halves belong to row g
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int n = 0; n < 4; n++) {
                oacc[b][n][0] *= f[0];
                oacc[b][n][1] *= f[0];
                oacc[b][n][2] *= f[H - 1];
                oacc[b][n][3] *= f[H - 1];
            }
    }

    // kop(n, b): four operand words of score tile n, block b; ksc(n, b): the
    // f16 pair of K scales of tokens 4 t + 2 n, + 1; vop(b, half): operand
    // words of column tiles 2 half, 2 half + 1 of block b; vs: the V scales of
    // tokens 4 t .. + 3.
    template <class KOp, class KSc, class VOp, class VSc>
    __device__ __forceinline__ void tile(const AttnP& p, int tile_at, int t, KOp kop, KSc ksc, VOp vop, VSc vsc) {
        if (tile_at >= full0 && tile_at < full1) tile<true>(p, tile_at, t, kop, ksc, vop, vsc);
        else tile<false>(p, tile_at, t, kop, ksc, vop, vsc);
    }
    template <bool full, class KOp, class KSc, class VOp, class VSc>
    __device__ __forceinline__ void tile(const AttnP& p, int tile_at, int t, KOp kop, KSc ksc, VOp vop, VSc vsc) {
        float2 sc[2][H];
#pragma unroll
        for (int n = 0; n < 2; n++) {
#pragma unroll
            for (int h = 0; h < H; h++) sc[n][h] = make_float2(0.0f, 0.0f);
            float c[NB][4];  // all blocks' first steps, then the second ones: no product waits for the one before
            uint4 w[NB];
#pragma unroll
            for (int b = 0; b < NB; b++) {
                w[b] = kop(n, b);
                mma16816_0(c[b], aq[b][0], w[b].x, w[b].y);
            }
#pragma unroll
            for (int b = 0; b < NB; b++) mma16816(c[b], aq[b][1], w[b].z, w[b].w);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float2 d = unpack(ksc(n, b));
                const float2 lo = make_float2(c[b][0], c[b][1]), hi = make_float2(c[b][2], c[b][3]);
                if (MODE == kOne16) {
                    sc[n][0] = fma2(lo, d, sc[n][0]);
                    sc[n][H - 1] = fma2(hi, d, sc[n][H - 1]);
                } else {
                    sc[n][0] = fma2(MODE == kSplit8 ? add2(lo, hi) : lo, d, sc[n][0]);
                }
            }
        }
        uint2 vs[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) vs[b] = vsc(b);
        const int j0 = tile_at * kKv4Tile + 4 * t;
        uint32_t hid01[H], hid23[H];  // halves of all ones: tokens that the row sees
#pragma unroll
        for (int h = 0; h < H; h++) hid01[h] = hid23[h] = 0xFFFFFFFFu;
        if constexpr (!full) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int j = j0 + i;
                const uint32_t half = (i & 1) ? 0xFFFF0000u : 0x0000FFFFu;
                if (j >= seen) {  // nobody's: whatever scale lies there counts for nothing
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        if (i < 2) vs[b].x &= ~half;
                        else vs[b].y &= ~half;
                    }
                }
#pragma unroll
                for (int h = 0; h < H; h++)
                    if (j >= seen || j > rpos[h] || (p.window > 0 && rpos[h] - j >= p.window)) {
                        if (i < 2) hid01[h] &= ~half;
                        else hid23[h] &= ~half;
                    }
            }
        }
        // the largest V scale of this lane's tokens
        __half2 big = __hmax2(__habs2(as_h2(vs[0].x)), __habs2(as_h2(vs[0].y)));
#pragma unroll
        for (int b = 1; b < NB; b++) big = __hmax2(big, __hmax2(__habs2(as_h2(vs[b].x)), __habs2(as_h2(vs[b].y))));
        const float2 big2 = __half22float2(big);
        const float dmax = fmaxf(big2.x, big2.y);
        float pr[H][4], top[H], mx[H];
#pragma unroll
        for (int h = 0; h < H; h++) {
            pr[h][0] = sc[0][h].x * qs[h];
            pr[h][1] = sc[0][h].y * qs[h];
            pr[h][2] = sc[1][h].x * qs[h];
            pr[h][3] = sc[1][h].y * qs[h];
            if constexpr (!full) {
                if (!(hid01[h] & 0xFFFFu)) pr[h][0] = -INFINITY;
                if (!(hid01[h] >> 16)) pr[h][1] = -INFINITY;
                if (!(hid23[h] & 0xFFFFu)) pr[h][2] = -INFINITY;
                if (!(hid23[h] >> 16)) pr[h][3] = -INFINITY;
            }
            top[h] = fmaxf(fmaxf(pr[h][0], pr[h][1]), fmaxf(pr[h][2], pr[h][3]));
        }
        float lg = fmaxf(lg2(dmax) - E, -7.0f);
        bool move = dmax > bound;
#pragma unroll
        for (int h = 0; h < H; h++) {
            mx[h] = top[h] + lg;
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
            move |= mx[h] > m[h] + kLazy || (m[h] == -INFINITY && mx[h] > -INFINITY);
        }
        if (__any_sync(0xffffffffu, move)) {
            if (__any_sync(0xffffffffu, dmax > bound)) {
                float w = dmax;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, o));
                int e;
                frexpf(w, &e);  // w <= 2^e
                const float down = __int_as_float((127 + (int)E - e) << 23);
                float f[H];
#pragma unroll
                for (int h = 0; h < H; h++) f[h] = down;
                scale_rows(f);
                set_scale(e);
                lg = fmaxf(lg2(dmax) - E, -7.0f);
#pragma unroll
                for (int h = 0; h < H; h++) {
                    mx[h] = top[h] + lg;
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                }
            }
            float al[H];
#pragma unroll
            for (int h = 0; h < H; h++) {
                const float mn = fmaxf(m[h], mx[h]);
                al[h] = m[h] == -INFINITY ? 0.0f : ex2(m[h] - mn);
                m[h] = mn;
                l[h] *= al[h];
            }
            scale_rows(al);
        }
        uint32_t ph[H][2], pl[H][2], nh[2];
#pragma unroll
        for (int h = 0; h < H; h++) {
            const float base = m[h] == -INFINITY ? 0.0f : m[h];
#pragma unroll
            for (int i = 0; i < 4; i++) pr[h][i] = ex2(pr[h][i] - base);
            l[h] += (pr[h][0] + pr[h][1]) + (pr[h][2] + pr[h][3]);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                ph[h][i] = pack(pr[h][2 * i], pr[h][2 * i + 1]);
                if (MODE == kSplit8) {
                    const float2 back = unpack(ph[h][i]);
                    pl[h][i] = pack(back.x - pr[h][2 * i], back.y - pr[h][2 * i + 1]);  // -pl
                    nh[i] = ph[h][i] ^ 0x80008000u;
                }
            }
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const __half2 d01 = __hmul2(as_h2(vs[b].x), inv), d23 = __hmul2(as_h2(vs[b].y), inv);
            uint32_t a[4];
#pragma unroll
            for (int h = 0; h < H; h++) {
                const __half2 x = __hmul2(as_h2(ph[h][0]), d01), y = __hmul2(as_h2(ph[h][1]), d23);
                if (MODE == kOne16) {
                    a[h] = as_u32(x);
                    a[2 + h] = as_u32(y);
                } else {
                    a[0] = as_u32(x);
                    a[2] = as_u32(y);
                    a[1] = a[3] = 0u;
                    if (MODE == kSplit8) {
                        // minus the low part, which spares the negations: value() subtracts
                        a[1] = as_u32(__hfma2(as_h2(pl[h][0]), d01, __hfma2(as_h2(nh[0]), d01, x)));
                        a[3] = as_u32(__hfma2(as_h2(pl[h][1]), d23, __hfma2(as_h2(nh[1]), d23, y)));
                    }
                }
                if constexpr (!full) {  // whatever a hidden position holds (a NaN scale too) does not enter
                    if (MODE == kOne16) {
                        a[h] &= hid01[h];
                        a[2 + h] &= hid23[h];
                    } else {
                        a[0] &= hid01[h];
                        a[1] &= hid01[h];
                        a[2] &= hid23[h];
                        a[3] &= hid23[h];
                    }
                }
            }
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const uint4 w = vop(b, half);
                mma16816(oacc[b][2 * half], a, w.x, w.y);
                mma16816(oacc[b][2 * half + 1], a, w.z, w.w);
            }
        }
    }

    // Row sums complete, accumulators back at the values' scale.
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int h = 0; h < H; h++) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        }
    }
    // elements 32 b + 8 n + 2 t, + 1 of row h
    __device__ __forceinline__ float2 value(int b, int n, int h) const {
        float2 v = h ? make_float2(oacc[b][n][2], oacc[b][n][3]) : make_float2(oacc[b][n][0], oacc[b][n][1]);
        if (MODE == kSplit8) {
            v.x -= oacc[b][n][2];
            v.y -= oacc[b][n][3];
        }
        return make_float2(v.x * bound, v.y * bound);
    }
};

// The records of one warp's tiles t0 + warp, + kWarps, ...: `Stages` bulk copies in
// flight, pages looked up 32 tiles at a time.
template <int Stages, int Bytes>
struct Stream {
    uint32_t ring, bar;
    const AttnP& p;
    const Rows& o;
    int first, n, lane, tiles;
    int base = -32;
    int64_t addr = -1;  // of tile base + lane: byte offset of its record, -1: not in the cache
    uint32_t phase = 0, absent = 0;

    __device__ __forceinline__ Stream(const AttnP& p, const Rows& o, uint32_t ring, uint32_t bar, int first, int n, int lane)
        : ring(ring), bar(bar), p(p), o(o), first(first), n(n), lane(lane), tiles(p.page_size / kKv4Tile) {
        if (lane == 0) {
            for (int s = 0; s < Stages; s++) mbar_init(bar + 8 * s, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        for (int k = 0; k < min(Stages, n); k++) issue(k);
    }
    __device__ __forceinline__ void issue(int k) {
        if (k >= base + 32) {
            base = k & ~31;
            addr = -1;
            if (base + lane < n) {
                const int tile = first + (base + lane) * kWarps, col = tile / tiles;
                const int pg = p.table[o.b * p.table_stride + col];
                if (pg >= 0 && pg < p.n_pages)
                    addr = (((int64_t)pg * p.n_kv + o.kvh) * tiles + (tile - col * tiles)) * Bytes;
            }
        }
        const int s = k % Stages;
        const int64_t a = __shfl_sync(0xffffffffu, addr, k & 31);
        absent = (absent & ~(1u << s)) | ((a < 0 ? 1u : 0u) << s);
        if (a >= 0 && lane == 0) {
            mbar_expect_tx(bar + 8 * s, Bytes);
            bulk_g2s(ring + s * Bytes, p.data + a, Bytes, bar + 8 * s, policy_evict_normal());
        }
    }
    __device__ __forceinline__ bool missing(int k) const { return (absent >> (k % Stages)) & 1u; }
    // false: the copy did not arrive within the bound
    __device__ __forceinline__ bool wait(int k) {
        const int s = k % Stages;
        const bool ok = mbar_wait(bar + 8 * s, (phase >> s) & 1u);
        if (!__all_sync(0xffffffffu, ok)) return false;
        phase ^= 1u << s;
        return true;
    }
    // after a wait that gave up: the same bound for the copies still in
    // flight, before their memory goes
    __device__ __forceinline__ void abandon(int k) {
        if (lane == 0) {
            atomicExch(p.err, 1);
            for (int i = k; i < min(k + Stages, n); i++)
                if (!missing(i)) mbar_wait(bar + 8 * (i % Stages), (phase >> (i % Stages)) & 1u);
        }
        __syncwarp();
    }
};

template <typename T>
__device__ __forceinline__ void store2(T* p, bool pair, float a, float b) {
    if constexpr (sizeof(T) == 4) {
        if (pair) {
            *reinterpret_cast<float2*>(p) = make_float2(a, b);
            return;
        }
    }
    p[0] = from_f32<T>(a);
    p[1] = from_f32<T>(b);
}

template <int NB, int MODE, typename T>
__global__ void __launch_bounds__(kWarps * 32, 3) kv4_attn_kernel(const __grid_constant__ AttnP p) {
    using Rec = Kv4Rec<NB>;
    using W = Warp<NB, MODE, T>;
    constexpr int R = W::R, H = W::H;
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
    const int n_mine = t1 > t0 + warp ? (t1 - t0 - warp + kWarps - 1) / kWarps : 0;
    const uint8_t* ring = smem + warp * kStages * Rec::kBytes;
    Stream<kStages, Rec::kBytes> in(p, o, smem_u32(ring), smem_u32(&bars[warp][0]), t0 + warp, n_mine, lane);
    W w;
    w.init(p, o, o.r0, g, t);
    for (int k = 0; k < n_mine; k++) {
        if (in.missing(k)) {  // not in the cache: nothing to see
            if (k + kStages < n_mine) in.issue(k + kStages);
            continue;
        }
        if (!in.wait(k)) {
            in.abandon(k);
            break;
        }
        const uint8_t* rec = ring + (k % kStages) * Rec::kBytes;
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
        if (k + kStages < n_mine) in.issue(k + kStages);
        w.tile(
            p, t0 + warp + k * kWarps, t, [&](int n, int b) { return k_operands(kw[2 * b + n]); },
            [&](int n, int b) { return n ? ks[b].y : ks[b].x; },
            [&](int b, int half) {
                const uint32_t w0 = vw[2 * b] >> (8 * half), w1 = vw[2 * b + 1] >> (8 * half);
                return make_uint4(codes_even(w0), codes_even(w1), codes_odd(w0), codes_odd(w1));
            },
            [&](int b) { return vs[b]; });
    }
    w.finish();
    // ---- join the warps: each one's m, l and row sums through shared memory
    // (the rings are drained: every issued copy has been waited for)
    float* so = reinterpret_cast<float*>(smem) + warp * (R * 32 * NB);
    __syncthreads();
#pragma unroll
    for (int h = 0; h < H; h++) {
        if (t == 0) {
            s_m[warp][g + 8 * h] = w.m[h];
            s_l[warp][g + 8 * h] = w.l[h];
        }
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int n = 0; n < 4; n++)
                *reinterpret_cast<float2*>(so + (g + 8 * h) * 32 * NB + 32 * b + 8 * n + 2 * t) = w.value(b, n, h);
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
        for (int i = 0; i < kWarps; i++) M = fmaxf(M, s_m[i][row]);
        float L = 0.0f, acc = 0.0f;
        if (M > -INFINITY) {
#pragma unroll
            for (int i = 0; i < kWarps; i++) {
                const float f = ex2(s_m[i][row] - M);
                L = fmaf(f, s_l[i][row], L);
                acc = fmaf(f, all[i * (R * 32 * NB) + e], acc);
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

// Many rows: warp i holds rows r0 + i R ..; a step is kWarps tiles, each
// unpacked by one warp into f16 operands that all four use.
template <int NB, int MODE, typename T>
__global__ void __launch_bounds__(kWarps * 32, 3) kv4_attn_rows_kernel(const __grid_constant__ AttnP p) {
    using Rec = Kv4Rec<NB>;
    using W = Warp<NB, MODE, T>;
    constexpr int R = W::R, H = W::H;
    constexpr int kOps = 2048 * NB;  // K and V operands of a tile, 1024 NB each
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[kWarps][kStagesRows];
    __shared__ int s_state[kWarps];  // of the step's tiles: 1 there, 0 not in the cache, -1 gave up
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int split = (int)(blockIdx.x % p.splits);
    Rows o;
    if (!find_rows<R * kWarps>(p, blockIdx.x / p.splits, o)) return;
    const int t0 = o.tile0 + split * o.per, t1 = min(t0 + o.per, o.tile1);
    if (p.splits > 1 && t0 >= t1) return;
    const int n_mine = t1 > t0 + warp ? (t1 - t0 - warp + kWarps - 1) / kWarps : 0;
    const int steps = t1 > t0 ? (t1 - t0 + kWarps - 1) / kWarps : 0;
    uint8_t* ops = smem;                                 // [kWarps][kOps]
    uint8_t* scl = smem + kWarps * kOps;                 // [kWarps][64 NB]: K scales, V scales
    const uint8_t* ring = scl + kWarps * 64 * NB + warp * kStagesRows * Rec::kBytes;
    Stream<kStagesRows, Rec::kBytes> in(p, o, smem_u32(ring), smem_u32(&bars[warp][0]), t0 + warp, n_mine, lane);
    W w;
    const int r0 = o.r0 + warp * R;
    w.init(p, o, r0, g, t);
    // tiles that this warp's rows see
    const int last = r0 < o.rows ? (max(w.seen, 0) + kKv4Tile - 1) / kKv4Tile : 0;
    for (int k = 0; k < steps; k++) {
        int state = 0;
        if (k < n_mine && !in.missing(k)) {
            state = in.wait(k) ? 1 : -1;
            if (state > 0) {
                const uint8_t* rec = ring + (k % kStagesRows) * Rec::kBytes;
                uint32_t kw[2 * NB], vw[2 * NB];
                load_words<NB>(rec, lane, kw);
                load_words<NB>(rec + Rec::kV, lane, vw);
                uint4* dst = reinterpret_cast<uint4*>(ops + warp * kOps) + lane;
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        dst[(2 * b + n) * 32] = k_operands(kw[2 * b + n]);
                        const uint32_t w0 = vw[2 * b] >> (8 * n), w1 = vw[2 * b + 1] >> (8 * n);
                        dst[(2 * NB + 2 * b + n) * 32] =
                            make_uint4(codes_even(w0), codes_even(w1), codes_odd(w0), codes_odd(w1));
                    }
                if (lane < 4 * NB)
                    reinterpret_cast<uint4*>(scl + warp * 64 * NB)[lane] = reinterpret_cast<const uint4*>(rec + Rec::kKs)[lane];
            }
        }
        if (lane == 0) s_state[warp] = state;
        __syncthreads();
        if (k + kStagesRows < n_mine && state >= 0) in.issue(k + kStagesRows);
        bool stop = false;
#pragma unroll 1
        for (int i = 0; i < kWarps; i++) {
            const int st = s_state[i], tile = t0 + k * kWarps + i;
            stop |= st < 0;
            if (st <= 0 || tile >= last) continue;
            const uint4* src = reinterpret_cast<const uint4*>(ops + i * kOps) + lane;
            const uint8_t* sc = scl + i * 64 * NB + t * 8 * NB;
            w.tile(
                p, tile, t, [&](int n, int b) { return src[(2 * b + n) * 32]; },
                [&](int n, int b) { return *reinterpret_cast<const uint32_t*>(sc + 8 * b + 4 * n); },
                [&](int b, int half) { return src[(2 * NB + 2 * b + half) * 32]; },
                [&](int b) { return *reinterpret_cast<const uint2*>(sc + 32 * NB + 8 * b); });
        }
        __syncthreads();
        if (stop) {
            in.abandon(k + (state >= 0 ? 1 : 0));
            break;
        }
    }
    w.finish();
#pragma unroll
    for (int h = 0; h < H; h++) {
        const int r = r0 + g + 8 * h;
        const int64_t tok = (int64_t)o.q0 + r / p.group;
        if (r >= o.rows || tok < 0 || tok >= p.n_tokens) continue;
        const int head = o.kvh * p.group + r % p.group;
        if (p.splits == 1) {
            T* dst = static_cast<T*>(p.out) + tok * p.ot + head * p.oh + 2 * t;
            const bool pair = ((uintptr_t)dst & 7) == 0;
            const float f = w.m[h] > -INFINITY ? 1.0f / w.l[h] : 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const float2 v = w.value(b, n, h);
                    store2(dst + 32 * b + 8 * n, pair, w.m[h] > -INFINITY ? v.x * f : 0.0f, w.m[h] > -INFINITY ? v.y * f : 0.0f);
                }
        } else {
            const int64_t at = (tok * p.n_heads + head) * p.splits + split;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int n = 0; n < 4; n++)
                    *reinterpret_cast<float2*>(p.part + at * (32 * NB) + 32 * b + 8 * n + 2 * t) = w.value(b, n, h);
            if (t == 0) p.ml[at] = make_float2(w.m[h], w.l[h]);
        }
    }
}

// Joins the splits of a row, a CTA a row: groups of 8 NB threads (four
// elements each) take every kJoin / (8 NB)-th split, and add up in group order.
constexpr int kJoin = 256;
template <int NB, int R, typename T>
__global__ void __launch_bounds__(kJoin) kv4_join_kernel(const __grid_constant__ AttnP p) {
    pdl_wait();
    Rows o;
    if (!find_rows<R>(p, blockIdx.x / R, o)) return;
    const int r = o.r0 + (int)(blockIdx.x % R);
    if (r >= o.rows) return;
    const int64_t tok = (int64_t)o.q0 + r / p.group;
    if (tok < 0 || tok >= p.n_tokens) return;
    constexpr int per = 8 * NB, groups = kJoin / per;
    __shared__ float4 s_o[groups][per];
    __shared__ float s_l[groups], s_m[kJoin / 32];
    const int head = o.kvh * p.group + r % p.group, tid = threadIdx.x;
    const int used = (o.tile1 - o.tile0 + o.per - 1) / o.per;  // splits that had tiles
    const int64_t at = (tok * p.n_heads + head) * p.splits;
    float M = -INFINITY;
    for (int s = tid; s < used; s += kJoin) M = fmaxf(M, p.ml[at + s].x);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, i));
    if ((tid & 31) == 0) s_m[tid >> 5] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kJoin / 32; i++) M = fmaxf(M, s_m[i]);
    const int grp = tid / per, e = tid % per;
    float L = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (grp < groups) {
        if (M > -INFINITY) {
#pragma unroll 4
            for (int s = grp; s < used; s += groups) {
                const float2 v = p.ml[at + s];
                const float4 x = reinterpret_cast<const float4*>(p.part + (at + s) * (32 * NB))[e];
                const float f = ex2(v.x - M);
                L = fmaf(f, v.y, L);
                acc.x = fmaf(f, x.x, acc.x);
                acc.y = fmaf(f, x.y, acc.y);
                acc.z = fmaf(f, x.z, acc.z);
                acc.w = fmaf(f, x.w, acc.w);
            }
        }
        s_o[grp][e] = acc;
        if (e == 0) s_l[grp] = L;
    }
    __syncthreads();
    if (tid < 32 * NB) {
        float sum = 0.0f, l = 0.0f;
#pragma unroll
        for (int i = 0; i < groups; i++) {
            l += s_l[i];
            sum += reinterpret_cast<const float*>(s_o[i])[tid];
        }
        static_cast<T*>(p.out)[tok * p.ot + head * p.oh + tid] = from_f32<T>(M > -INFINITY ? sum / l : 0.0f);
    }
}

// f32 queries take the hi + lo rows, 16-bit ones one operand row each (eight
// or sixteen rows a tile)
enum Which { kMain, kRows, kJoinSplits };
template <int NB, int MODE, typename T>
const void* fn_of(Which which, bool rows) {
    constexpr int R = MODE == kOne16 ? 16 : 8;
    if (which == kMain) return (const void*)kv4_attn_kernel<NB, MODE, T>;
    if constexpr (MODE == kOne8) return (const void*)kv4_join_kernel<NB, R, T>;  // 8 rows have no rows form
    else if (which == kRows) return (const void*)kv4_attn_rows_kernel<NB, MODE, T>;
    else return rows ? (const void*)kv4_join_kernel<NB, R * kWarps, T> : (const void*)kv4_join_kernel<NB, R, T>;
}
template <int NB, typename T>
const void* fn_of(Which which, int mode, bool rows) {
    if constexpr (sizeof(T) == 4) return fn_of<NB, kSplit8, T>(which, rows);
    else return mode == kOne8 ? fn_of<NB, kOne8, T>(which, rows) : fn_of<NB, kOne16, T>(which, rows);
}
template <typename T>
const void* fn_of(int nb, Which which, int mode, bool rows) {
    switch (nb) {
    case 1: return fn_of<1, T>(which, mode, rows);
    case 2: return fn_of<2, T>(which, mode, rows);
    case 3: return fn_of<3, T>(which, mode, rows);
    default: return fn_of<4, T>(which, mode, rows);
    }
}
const void* fn_of(int dtype, int nb, Which which, int mode, bool rows) {
    return dtype == RQ_F32 ? fn_of<float>(nb, which, mode, rows)
           : dtype == RQ_F16 ? fn_of<__half>(nb, which, mode, rows)
                             : fn_of<__nv_bfloat16>(nb, which, mode, rows);
}

struct Plan {
    int mode, R, row_tiles, splits;  // R: rows of a CTA
    bool rows;                       // the many-rows form
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
    pl.rows = rows > 2 * pl.R;
    if (pl.rows) pl.R *= kWarps;
    pl.row_tiles = (int)((rows + pl.R - 1) / pl.R);
    pl.units = a->batch * c->n_kv * pl.row_tiles;
    // Splits of the long axis: one CTA for each place on the device (three an
    // SM) where the rows are few, four where the sequences' different lengths
    // have to even out, but none shorter than two tiles a warp
    int64_t len = a->table_width * c->page_size;
    if (a->max_len > 0) len = std::min(len, a->max_len);
    if (a->window > 0) len = std::min(len, a->window + a->max_q);
    const int64_t tiles = (len + kKv4Tile - 1) / kKv4Tile;
    const int64_t places = (int64_t)c->ctx->sm_count * 3;
    const int64_t want = a->batch == 1 ? places / std::max<int64_t>(pl.units, 1)
                                       : (4 * places + pl.units - 1) / std::max<int64_t>(pl.units, 1);
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
    p.table_slots = (int)(a->table_width * c->page_size);
    // positions stay below 2^31 and a query is never more than max_q below 0,
    // so a window this long hides nothing and its differences fit 32 bits
    p.window = a->window < (1 << 30) * 2ll - (1 << 25) ? (int)a->window : 0;
    p.scale = a->scale * 1.44269504088896340736f;
    p.part = static_cast<float*>(a->workspace);
    if (need) {
        const int64_t rows = a->n_tokens * a->n_heads * pl.splits;
        p.ml = reinterpret_cast<float2*>(p.part + rows * c->head_dim);
    }
    p.err = err;
    const int nb = c->head_dim / 32;
    const size_t smem = pl.rows ? (size_t)kWarps * (2048 * nb + 64 * nb + kStagesRows * 576 * nb)
                                : (size_t)kWarps * std::max(kStages * 576 * nb, pl.R * 32 * nb * 4);
    const void* fn = fn_of(a->dtype, nb, pl.rows ? kRows : kMain, pl.mode, pl.rows);
    if (smem > 48 * 1024) {
        const int rc = cuda_error(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                                  "kv4 attention kernel");
        if (rc) return rc;
    }
    void* args[] = {&p};
    const int rc = launch_pdl(fn, (unsigned)(pl.units * pl.splits), kWarps * 32, smem, st, args, "kv4 attention kernel");
    if (rc || pl.splits == 1) return rc;
    const void* jf = fn_of(a->dtype, nb, kJoinSplits, pl.mode, pl.rows);
    return launch_pdl(jf, (unsigned)(pl.units * pl.R), kJoin, 0, st, args, "kv4 join kernel");
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
