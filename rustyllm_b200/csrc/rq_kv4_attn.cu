// rq_kv4_attn.cu -- attention over the 4-bit paged cache (rq_kv4.cuh), for
// single new tokens, drafted tokens and prompt chunks.
//
// For a query row q and the positions j it sees, with K = (c - 8) d per block
// of 32 elements:
//   s_j = scale * sum_b dK_jb (q_b . (cK_jb - 8)),  o = sum_j softmax(s)_j V_j.
// The codes c - 8 are exact in f16.
//
// Three forms, chosen by make_plan:
//  - few rows (decode, drafted tokens), on mma.m16n8k16: every warp of a CTA
//    walks its own tiles of 16 positions for the same rows, so one row tile uses
//    all lanes of the GPU; its operands are built in registers from the record
//    that one bulk copy brought to shared memory.  The warps join through shared
//    memory, the pieces of a unit that went to several CTAs through a second
//    launch.
//  - many rows of f32 and f16 queries (prompts), on mma.m16n8k16: the warps hold
//    different rows, two operand tiles each; the records are turned into f16
//    operands in shared memory once for all four, and an operand read from there
//    serves two tiles of rows (with one tile a warp, reading them took as long as
//    the products).
//  - many rows of bf16 queries, on tcgen05: see there.
//
// The first two do not round the cache: q is scaled by a power of two to [-1, 1]
// and split into f16 hi + lo (16-bit inputs need hi alone), the K
// scales multiply the f32 block sums, and the V scales multiply the
// probabilities, P_jb = p_j dV_jb.  The hi and lo parts are the two row halves of
// one m16 operand: eight query rows a tile, no extra instructions.  (Nine to
// sixteen bf16 rows take both halves for one part.)
//
// P enters as f16: in two parts, p = ph + pl (22 bits) and ph d = h + r exactly (h
// the rounded product, r = fma(ph, d, -h)), so P = h + (r + pl d) costs three
// packed operations a pair of tokens; one part takes h alone (two roundings of
// 2^-11, an eighth of bf16's own).  f16's range is kept position by position: the
// scales of position j are divided by their power 2^Dj (the smallest with all
// |dV_jb| <= 2^Dj, within f16's normal numbers), p_j 2^Dj takes it, and the reference
// m follows the largest s_j + Dj that the row sees: the products of the positions
// that count most lie in [2^4, 2^14], and a huge value that a row does not see,
// or sees with no weight, takes no bits from the others (a power that followed the
// largest scale seen cost the f32 output up to 3 % behind one value of 5e5).  A
// scale 2^14 below the largest of its own position keeps fewer bits, of its 2^-25.
// m moves lazily, by 2^8.  Sums stay in f32 throughout.
#include <algorithm>

#include "rq_async.cuh"
#include "rq_kv4.cuh"
#include "rq_tcgen05.cuh"

namespace rq {
namespace {

constexpr int kWarps = 4;       // warps of a CTA
constexpr int kStages = 3;      // pairs of tiles in flight per warp (few rows)
constexpr int kStagesRows = 2;  // (many rows)
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxQ = 1 << 24;  // queries of a sequence
constexpr float kLazy = 8.0f;   // log2 of how far P grows before the reference moves
constexpr float kTop = 5.0f;    // log2 of the largest p 2^D where it has moved

enum Mode { kSplit8, kOne16 };  // 8 rows of hi + lo parts, 16 rows of one part

struct Magic {  // see codes_even
    uint32_t even, odd;
};

struct AttnP {
    const uint8_t* data;
    int64_t n_pages;
    int page_size, n_kv;
    const void* q;
    int64_t qt, qh;
    void* out;
    int64_t ot, oh;
    bool wide, wide_out;  // rows of q, of out on 16-byte borders
    int64_t n_tokens;
    int n_heads, group, batch, max_q, row_tiles, splits;
    const int32_t* cu_q;
    const int32_t* kv_lens;
    const int32_t* table;
    int64_t table_stride;
    int table_slots;  // positions of a table row
    int window;       // 0: none
    float scale;      // times log2(e)
    // sums of pieces: few rows, [2 ctas][8 or 16 rows][head_dim], CTA i's piece
    // at its range's start and one that starts later; many rows, [n_tokens *
    // n_heads][splits][head_dim]
    float* part;
    float2* ml;  // their running maxima and sums
    int4* desc;  // few rows, [ctas]: the unit that starts in CTA i and goes on behind it
    Magic magic;
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
// What sums kept relative to maximum m count relative to M, the largest: where
// no position was seen m and M are -inf and the sums are zeros -- or not numbers,
// if all scores were none, which have to stay so.
__device__ __forceinline__ float weight(float m, float M) { return M > -INFINITY ? ex2(m - M) : 1.0f; }
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
// For halves w >= 0: the smallest 2^D >= w with D in -14 .. 14 (above, 2^14: w is
// 4 times that at most), 0 for 0.  2^-D has the exponent field 30 less this one's,
// and for 0 some finite value.
__device__ __forceinline__ uint32_t power(__half2 w) {
    return as_u32(__hmin2(as_h2((as_u32(w) + 0x03FF03FFu) & 0x7C007C00u), __half2half2(__ushort_as_half(0x7400))));
}
// nibbles 0 and 4 (even) or 1 and 5 (odd) of w as f16 pairs c - 8: a nibble
// placed in the mantissa of 1024 (or, four bits up, of 64) is that value + c.
// The two constants come from the launch's parameters: known ones would be
// immediates, and a second immediate costs lop3 another instruction (33 of 400 a
// tile).
constexpr uint32_t kEven = 0x64006400u, kOdd = 0x54005400u;
__device__ __forceinline__ uint32_t codes_even(uint32_t w, Magic m) {
    uint32_t h;
    asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(h) : "r"(w), "r"(m.even));
    return as_u32(__hsub2(as_h2(h), __half2half2(__ushort_as_half(0x6408))));
}
__device__ __forceinline__ uint32_t codes_odd(uint32_t w, Magic m) {
    uint32_t h;
    asm("lop3.b32 %0, %1, 0x00F000F0, %2, 0xEA;" : "=r"(h) : "r"(w), "r"(m.odd));
    return as_u32(__hsub2(as_h2(h), __half2half2(__ushort_as_half(0x5480))));
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
__device__ __forceinline__ uint4 k_operands(uint32_t w, Magic m) {
    return make_uint4(codes_even(w, m), codes_odd(w, m), codes_even(w >> 8, m), codes_odd(w >> 8, m));
}
__device__ __forceinline__ uint4 v_operands(uint32_t w0, uint32_t w1, Magic m) {
    return make_uint4(codes_even(w0, m), codes_even(w1, m), codes_odd(w0, m), codes_odd(w1, m));
}

// A sequence's queries and positions
struct Seq {
    int n_q, q0;
    int pos0, held;    // position of query 0; positions that the table can hold
    __device__ __forceinline__ Seq(const AttnP& p, int b) {
        q0 = p.cu_q ? p.cu_q[b] : b;
        const int64_t n = p.cu_q ? max((int64_t)p.cu_q[b + 1] - q0, (int64_t)0) : 1;
        n_q = (int)min(n, (int64_t)p.max_q);  // of more than the caller announced, the first ones, where they are
        const int len = max(p.kv_lens[b], 0);
        held = min(len, p.table_slots);
        // no query that is computed lies further than max_q behind this bound, so
        // those below it see nothing either way
        pos0 = (int)max(len - n, -(int64_t)kMaxQ);
    }
    // tiles that queries i0 .. i1 see
    __device__ __forceinline__ void tiles(const AttnP& p, int i0, int i1, int& tile0, int& tile1) const {
        const int hi = max(0, min(held, pos0 + i1 + 1));
        const int lo = p.window > 0 ? max(0, pos0 + i0 - p.window + 1) : 0;
        tile0 = lo / kKv4Tile;
        tile1 = max(tile0, hi / kKv4Tile + (hi % kKv4Tile != 0));
    }
};
// A unit of work: rows r0 .. of kv head kvh of sequence b
struct Rows : Seq {
    int b, kvh, r0, rows;
    __device__ __forceinline__ Rows(const AttnP& p, int b, int kvh, int r0)
        : Seq(p, b), b(b), kvh(kvh), r0(r0), rows(n_q * p.group) {}
};
// Unit `unit` of the many-rows forms, row tiles of R; its r0 may lie behind the rows
template <int R>
__device__ __forceinline__ Rows unit_rows(const AttnP& p, int unit) {
    const int bk = unit / p.row_tiles, b = bk / p.n_kv;
    return Rows(p, b, bk - b * p.n_kv, (unit - bk * p.row_tiles) * R);
}
template <int R>
__device__ __forceinline__ void unit_tiles(const AttnP& p, const Rows& o, int& tile0, int& tile1, int& per) {
    o.tiles(p, o.r0 / p.group, min(o.n_q - 1, (o.r0 + R - 1) / p.group), tile0, tile1);
    per = max((tile1 - tile0 + 2 * p.splits - 1) / (2 * p.splits), kWarps) * 2;  // of a split, whole pairs
}

// One warp's query rows, running sums and the work on one tile.  MT operand
// tiles of rows: one, its query operands in registers, or two, theirs in shared
// memory (`as`: [MT][NB][2][32 lanes]).
template <int NB, int MODE, typename T, int MT, bool AS>
struct Warp {
    static_assert(MODE == kSplit8 || MT == 1, "16 rows of one part fill an operand tile's both halves");
    static constexpr int R1 = MODE == kOne16 ? 16 : 8, R = R1 * MT;
    static constexpr int HH = MODE == kOne16 ? 2 : 1, H = HH * MT;  // rows a lane: of an operand tile, in all
    uint32_t aq[AS ? 1 : NB][2][4];
    uint4* as;
    float qs[H];      // back from the normalised row, times the softmax scale
    int rpos[H];      // position of the row's query; -1: no row
    // The tensor cores cut their sums off rather than round them: over the tiles
    // of a long walk that grows to 1.3e-5 of the output (60000 positions), nothing
    // to 16-bit outputs, but for f32 a tile's products are summed alone and added
    // here (7e-7; 1 to 5 % slower).
    static constexpr bool kAlone = sizeof(T) == 4;
    static constexpr int kAcc = kAlone ? 2 : 4;  // kAlone: hi and lo rows together
    float oacc[MT][NB][4][kAcc];
    float m[H], l[H];
    int full0, full1;      // tiles that every row sees whole
    int seen;              // positions that any row sees end here

    // row of lane group g's h-th
    static __device__ __forceinline__ int row_of(int g, int h) { return (h / HH) * R1 + g + 8 * (h % HH); }

    __device__ __forceinline__ void init(const AttnP& p, const Rows& o, int r0, int g, int t) {
#pragma unroll
        for (int h = 0; h < H; h++) {
            const int mt = h / HH, hh = h % HH;
            const int r = r0 + row_of(g, h);
            const int i = r / p.group, head = o.kvh * p.group + r - i * p.group;
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
                    load8(static_cast<const T*>(p.q) + tok * p.qt + head * p.qh + 32 * b + 8 * t,
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
                        const float2 back = unpack(hi);
                        const uint32_t lo = MODE == kOne16 ? 0u : pack(f0 - back.x, f1 - back.y);
                        if constexpr (AS) {
                            uint32_t* at = reinterpret_cast<uint32_t*>(as + ((mt * NB + b) * 2 + s) * 32 + 4 * g + t);
                            at[2 * j + hh] = hi;
                            if (MODE != kOne16) at[2 * j + 1] = lo;
                        } else {
                            aq[b][s][2 * j + hh] = hi;
                            if (MODE != kOne16) aq[b][s][2 * j + 1] = lo;
                        }
                    }
            m[h] = -INFINITY;
            l[h] = 0.0f;
        }
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int n = 0; n < 4; n++)
#pragma unroll
                    for (int i = 0; i < kAcc; i++) oacc[mt][b][n][i] = 0.0f;
        __syncwarp();  // the operands in shared memory are there
        const int i0 = r0 / p.group, i1 = min(o.n_q - 1, (r0 + R - 1) / p.group);
        full1 = max(0, min(o.held, o.pos0 + i0 + 1)) / kKv4Tile;
        const int before = o.pos0 + i1 - p.window;  // positions up to here the last row no longer sees
        full0 = p.window > 0 && before >= 0 ? before / kKv4Tile + 1 : 0;
        seen = min(o.held, o.pos0 + i1 + 1);
    }
    static __device__ __forceinline__ void add_products(float (&o)[kAcc], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        if constexpr (kAlone) {
            float c[4];
            mma16816_0(c, a, b0, b1);
            const float2 d = add2(make_float2(c[0], c[1]), make_float2(-c[2], -c[3]));
            const float2 s = add2(make_float2(o[0], o[1]), d);
            o[0] = s.x;
            o[1] = s.y;
        } else {
            mma16816(o, a, b0, b1);
        }
    }
    __device__ __forceinline__ void scale_rows(const float (&f)[H]) {
        // rows g and g + 8 of an accumulator: in the 8-row mode both halves
        // belong to row g
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int n = 0; n < 4; n++) {
#pragma unroll
                    for (int i = 0; i < kAcc; i++) oacc[mt][b][n][i] *= f[mt * HH + (i < 2 ? 0 : HH - 1)];
                }
    }

    // NT tiles at tile_at, + 1 that the operand source `src` holds:
    //   src.k(i) / src.v(i)  make tile i's K / V operands available
    //   src.kop(i, n, b)     four operand words of score tile n, block b
    //   src.ksc(i, n, b)     the f16 pair of K scales of tokens 4 t + 2 n, + 1
    //   src.vop(i, b, half)  operand words of column tiles 2 half, 2 half + 1
    //   src.vsc(i, b)        the V scales of tokens 4 t .. + 3
    // full: every row sees every position.
    template <int NT, bool full, class Src>
    __device__ __forceinline__ void tiles(const AttnP& p, int tile_at, int t, Src& src) {
        float2 sc[NT][2][H];
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int h = 0; h < H; h++) sc[i][n][h] = make_float2(0.0f, 0.0f);
        auto add = [&](float2 (&to)[H], int mt, const float (&c)[4], float2 d) {
            const float2 lo = make_float2(c[0], c[1]), hi = make_float2(c[2], c[3]);
            if (MODE == kOne16) {
                to[mt * HH] = fma2(lo, d, to[mt * HH]);
                to[mt * HH + HH - 1] = fma2(hi, d, to[mt * HH + HH - 1]);
            } else {
                to[mt] = fma2(add2(lo, hi), d, to[mt]);
            }
        };
        if constexpr (!AS) {
#pragma unroll
            for (int i = 0; i < NT; i++) {
                src.k(i);
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    float c[NB][4];  // all blocks' first steps, then the second ones: no product waits for the one before
                    uint4 w[NB];
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        w[b] = src.kop(i, n, b);
                        mma16816_0(c[b], aq[b][0], w[b].x, w[b].y);
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++) mma16816(c[b], aq[b][1], w[b].z, w[b].w);
#pragma unroll
                    for (int b = 0; b < NB; b++) add(sc[i][n], 0, c[b], unpack(src.ksc(i, n, b)));
                }
            }
        } else {
            // block by block, so that its query operands are fetched once for
            // all tiles
#pragma unroll
            for (int b = 0; b < NB; b++) {
                uint32_t a[MT][2][4];
                float c[MT][NT][2][4];
                uint4 w[NT][2];
                src.template kblock<NT>(b);
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const uint4 v = as[((mt * NB + b) * 2 + s) * 32 + (threadIdx.x & 31)];
                        a[mt][s][0] = v.x;
                        a[mt][s][1] = v.y;
                        a[mt][s][2] = v.z;
                        a[mt][s][3] = v.w;
                    }
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        w[i][n] = src.kop(i, n, b);
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) mma16816_0(c[mt][i][n], a[mt][0], w[i][n].x, w[i][n].y);
                    }
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) mma16816(c[mt][i][n], a[mt][1], w[i][n].z, w[i][n].w);
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const float2 d = unpack(src.ksc(i, n, b));
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) add(sc[i][n], mt, c[mt][i][n], d);
                    }
            }
        }
        uint2 vs[NT][NB];
        uint32_t see[NT][H][2];  // halves of all ones: tokens that the row sees (used where !full)
        uint32_t pw[NT][2];      // 2^D of the lane's tokens, f16; zero where all scales are
        float pr[NT][H][4], top[H];
        __half2 big = __half2half2(__ushort_as_half(0));
#pragma unroll
        for (int h = 0; h < H; h++) top[h] = -INFINITY;
#pragma unroll
        for (int i = 0; i < NT; i++) {
#pragma unroll
            for (int b = 0; b < NB; b++) vs[i][b] = src.vsc(i, b);
            if constexpr (!full) {
#pragma unroll
                for (int h = 0; h < H; h++) see[i][h][0] = see[i][h][1] = 0xFFFFFFFFu;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int j = (tile_at + i) * kKv4Tile + 4 * t + x;
                    const uint32_t half = (x & 1) ? 0xFFFF0000u : 0x0000FFFFu;
#pragma unroll
                    for (int h = 0; h < H; h++)
                        if (j >= seen || j > rpos[h] || (p.window > 0 && rpos[h] - j >= p.window)) see[i][h][x >> 1] &= ~half;
                }
            }
            // the power of each token's scales (a not-a-number one is passed over)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                __half2 w = __habs2(as_h2(x ? vs[i][0].y : vs[i][0].x));
#pragma unroll
                for (int b = 1; b < NB; b++) w = __hmax2(w, __habs2(as_h2(x ? vs[i][b].y : vs[i][b].x)));
                big = __hmax2(big, w);
                pw[i][x] = power(w);
            }
#pragma unroll
            for (int h = 0; h < H; h++) {
                pr[i][h][0] = sc[i][0][h].x * qs[h];
                pr[i][h][1] = sc[i][0][h].y * qs[h];
                pr[i][h][2] = sc[i][1][h].x * qs[h];
                pr[i][h][3] = sc[i][1][h].y * qs[h];
                if constexpr (!full) {
                    if (!(see[i][h][0] & 0xFFFFu)) pr[i][h][0] = -INFINITY;
                    if (!(see[i][h][0] >> 16)) pr[i][h][1] = -INFINITY;
                    if (!(see[i][h][1] & 0xFFFFu)) pr[i][h][2] = -INFINITY;
                    if (!(see[i][h][1] >> 16)) pr[i][h][3] = -INFINITY;
                }
#pragma unroll
                for (int x = 0; x < 4; x++) top[h] = fmaxf(top[h], pr[i][h][x]);
            }
        }
        // No s + D of this lane passes its largest s plus its largest D: where that
        // says that P stays in range the reference is not looked at
        const float2 big2 = __half22float2(big);
        const float lg = kTop + kLazy - fmaxf(lg2(fmaxf(big2.x, big2.y)), -14.0f);
        bool move = false;
#pragma unroll
        for (int h = 0; h < H; h++) move |= top[h] > m[h] + lg;  // (m -inf: anything that is seen)
        if (__any_sync(0xffffffffu, move)) {
            float al[H];
#pragma unroll
            for (int h = 0; h < H; h++) {
                float k = -INFINITY;
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        // no value at all counts for the sum of weights alone, which
                        // holds 2^60 times the others' (and not infinity)
                        const float2 u = unpack(pw[i][x]);
                        k = fmaxf(k, fmaxf(pr[i][h][2 * x] + fmaxf(lg2(u.x), -60.0f), pr[i][h][2 * x + 1] + fmaxf(lg2(u.y), -60.0f)));
                    }
                k = fmaxf(k, __shfl_xor_sync(0xffffffffu, k, 1));
                k = fmaxf(k, __shfl_xor_sync(0xffffffffu, k, 2));
                const float mn = fmaxf(m[h], k - kTop);
                al[h] = m[h] == -INFINITY ? 0.0f : ex2(m[h] - mn);
                m[h] = mn;
                l[h] *= al[h];
            }
            scale_rows(al);
        }
#pragma unroll
        for (int i = 0; i < NT; i++) {
            uint32_t ph[H][2], pl[MT][2], nh[MT][2];
#pragma unroll
            for (int h = 0; h < H; h++) {
                const float base = m[h] == -INFINITY ? 0.0f : m[h];
#pragma unroll
                for (int x = 0; x < 4; x++) pr[i][h][x] = ex2(pr[i][h][x] - base);
                l[h] += (pr[i][h][0] + pr[i][h][1]) + (pr[i][h][2] + pr[i][h][3]);
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const float2 u = unpack(pw[i][x]);
                    pr[i][h][2 * x] *= u.x;
                    pr[i][h][2 * x + 1] *= u.y;
                    ph[h][x] = pack(pr[i][h][2 * x], pr[i][h][2 * x + 1]);
                    if (MODE == kSplit8) {
                        const float2 back = unpack(ph[h][x]);
                        pl[h / HH][x] = pack(back.x - pr[i][h][2 * x], back.y - pr[i][h][2 * x + 1]);  // -pl
                        nh[h / HH][x] = ph[h][x] ^ 0x80008000u;
                    }
                }
            }
            src.v(i);
            const uint32_t inv0 = 0x78007800u - pw[i][0], inv1 = 0x78007800u - pw[i][1];  // 2^-D
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const __half2 d01 = __hmul2(as_h2(vs[i][b].x), as_h2(inv0)), d23 = __hmul2(as_h2(vs[i][b].y), as_h2(inv1));
                uint32_t a[MT][4];
#pragma unroll
                for (int h = 0; h < H; h++) {
                    const int mt = h / HH, hh = h % HH;
                    const __half2 x = __hmul2(as_h2(ph[h][0]), d01), y = __hmul2(as_h2(ph[h][1]), d23);
                    a[mt][hh] = as_u32(x);
                    a[mt][2 + hh] = as_u32(y);
                    if (MODE == kSplit8) {
                        // minus the low part, which spares the negations: value() subtracts
                        a[mt][1] = as_u32(__hfma2(as_h2(pl[mt][0]), d01, __hfma2(as_h2(nh[mt][0]), d01, x)));
                        a[mt][3] = as_u32(__hfma2(as_h2(pl[mt][1]), d23, __hfma2(as_h2(nh[mt][1]), d23, y)));
                    }
                    if constexpr (!full) {  // whatever a hidden position holds (a NaN scale too) does not enter
                        a[mt][hh] &= see[i][h][0];
                        a[mt][2 + hh] &= see[i][h][1];
                        if (MODE == kSplit8) {
                            a[mt][1] &= see[i][h][0];
                            a[mt][3] &= see[i][h][1];
                        }
                    }
                }
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const uint4 w = src.vop(i, b, half);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        add_products(oacc[mt][b][2 * half], a[mt], w.x, w.y);
                        add_products(oacc[mt][b][2 * half + 1], a[mt], w.z, w.w);
                    }
                }
            }
        }
    }
    // Tiles tile_at, + 1, of which bits of `there` are in the cache.
    template <class Src>
    __device__ __forceinline__ void pair(const AttnP& p, int tile_at, uint32_t there, int t, Src& src) {
        if (there == 3u && tile_at >= full0 && tile_at + 1 < full1) {
            tiles<2, true>(p, tile_at, t, src);
            return;
        }
#pragma unroll 1
        for (int i = 0; i < 2; i++)
            if ((there >> i) & 1u) {
                src.first = i;
                tiles<1, false>(p, tile_at + i, t, src);
            }
        src.first = 0;
    }

    // Row sums complete.
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int h = 0; h < H; h++) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        }
    }
    // elements 32 b + 8 n + 2 t, + 1 of row h
    __device__ __forceinline__ float2 value(int b, int n, int h) const {
        const float(&o)[kAcc] = oacc[h / HH][b][n];
        float2 v = make_float2(o[0], o[1]);
        if constexpr (!kAlone) {
            if (h % HH) v = make_float2(o[2], o[3]);
            if (MODE == kSplit8) {
                v.x -= o[2];
                v.y -= o[3];
            }
        }
        return v;
    }
};

// The records of a warp's pairs of tiles: pair k is tiles first + 2 Lists k
// and the next one, below `end` (Lists: such streams a CTA); `Stages` pairs in
// flight, one bulk copy a tile, issued by two lanes of the warp that `issues`.
// Pages are looked up 16 pairs (one tile a lane) at a time.
template <int Stages, int Bytes, int Lists>
struct Stream {
    const AttnP& p;
    uint32_t ring, bar;
    int lane, tiles;
    bool issues;
    const int32_t* table;
    int kvh, first, end, n = 0, base;
    int64_t addr;   // of this lane's tile: byte offset of its record
    uint32_t mask;  // lanes whose tile is in the cache
    uint32_t phase = 0, have = 0;  // bit per stage; two bits per stage: tiles that are there

    __device__ __forceinline__ Stream(const AttnP& p, uint32_t ring, uint32_t bar, int lane, bool issues = true)
        : p(p), ring(ring), bar(bar), lane(lane), tiles(p.page_size / kKv4Tile), issues(issues) {
        if (lane == 0 && issues) {
            for (int s = 0; s < Stages; s++) mbar_init(bar + 8 * s, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
    }
    __device__ __forceinline__ void begin(int b, int kv_head, int first_tile, int end_tile) {
        table = p.table + b * p.table_stride;
        kvh = kv_head;
        first = first_tile;
        end = end_tile;
        n = end > first ? (end - first + 2 * Lists - 1) / (2 * Lists) : 0;
        base = -16;
        have = 0;
        for (int k = 0; k < min(Stages, n); k++) issue(k, k);
    }
    // pair k into stage s
    __device__ __forceinline__ void issue(int k, int s) {
        if (k >= base + 16) {
            base = k & ~15;
            addr = -1;
            const int tile = first + 2 * Lists * (base + (lane >> 1)) + (lane & 1);
            if (tile < end) {
                const int col = tile / tiles;
                const int pg = table[col];
                if (pg >= 0 && pg < p.n_pages) addr = (((int64_t)pg * p.n_kv + kvh) * tiles + (tile - col * tiles)) * Bytes;
            }
            mask = __ballot_sync(0xffffffffu, addr >= 0);
        }
        const uint32_t there = (mask >> (2 * (k - base))) & 3u;
        have = (have & ~(3u << (2 * s))) | (there << (2 * s));
        if (!issues || (lane >> 1) != k - base) return;
        // one lane expects both tiles' bytes, before either copy can arrive:
        // the other one's is issued behind the group's own barrier
        const uint32_t two = 3u << (lane & ~1);
        if (there && (lane & 1) == 0) mbar_expect_tx(bar + 8 * s, __popc(there) * Bytes);
        __syncwarp(two);
        if ((there >> (lane & 1)) & 1u)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                             ring + (2 * s + (lane & 1)) * Bytes),
                         "l"(p.data + addr), "r"((uint32_t)Bytes), "r"(bar + 8 * s)
                         : "memory");
    }
    __device__ __forceinline__ uint32_t there(int s) const { return (have >> (2 * s)) & 3u; }
    // false: a copy did not arrive within the bound
    __device__ __forceinline__ bool wait(int s) {
        const bool ok = mbar_wait(bar + 8 * s, (phase >> s) & 1u);
        if (!__all_sync(0xffffffffu, ok)) return false;
        phase ^= 1u << s;
        return true;
    }
    // after a wait that gave up: the same bound for the copies of pairs k .. k +
    // Stages - 1, before their memory goes
    __device__ __forceinline__ void abandon(int k) {
        if (lane == 0) {
            atomicExch(p.err, 1);
            for (int i = k; i < min(k + Stages, n); i++)
                if (there(i % Stages)) mbar_wait(bar + 8 * (i % Stages), (phase >> (i % Stages)) & 1u);
        }
        __syncwarp();
    }
};

// Operands built in registers from the records of a pair
template <int NB, bool kAS>
struct RecordSrc {
    const uint8_t* rec;
    Magic magic;
    int lane, t, first = 0;
    uint32_t w[2 * NB];
    uint32_t kb[2][4];  // K words of blocks b (even) and b + 1 of both tiles
    template <int NT>
    __device__ __forceinline__ void kblock(int b) {
        if (b & 1) return;
#pragma unroll
        for (int i = 0; i < NT; i++) {
            if (b + 1 < NB) {
                const uint4 v = *reinterpret_cast<const uint4*>(at(i) + (b >> 1) * 512 + lane * 16);
                kb[i][0] = v.x;
                kb[i][1] = v.y;
                kb[i][2] = v.z;
                kb[i][3] = v.w;
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(at(i) + (b >> 1) * 512 + lane * 8);
                kb[i][0] = v.x;
                kb[i][1] = v.y;
            }
        }
    }
    __device__ __forceinline__ const uint8_t* at(int i) const { return rec + (first + i) * Kv4Rec<NB>::kBytes; }
    __device__ __forceinline__ void k(int i) { load_words<NB>(at(i), lane, w); }
    __device__ __forceinline__ void v(int i) { load_words<NB>(at(i) + Kv4Rec<NB>::kV, lane, w); }
    __device__ __forceinline__ uint4 kop(int i, int n, int b) const { return k_operands(kAS ? kb[i][2 * (b & 1) + n] : w[2 * b + n], magic); }
    __device__ __forceinline__ uint32_t ksc(int i, int n, int b) const {
        return *reinterpret_cast<const uint32_t*>(at(i) + Kv4Rec<NB>::kKs + t * 8 * NB + 8 * b + 4 * n);
    }
    __device__ __forceinline__ uint4 vop(int, int b, int half) const {
        return v_operands(w[2 * b] >> (8 * half), w[2 * b + 1] >> (8 * half), magic);
    }
    __device__ __forceinline__ uint2 vsc(int i, int b) const {
        return *reinterpret_cast<const uint2*>(at(i) + Kv4Rec<NB>::kVs + t * 8 * NB + 8 * b);
    }
};
// Operands that some warp has put into shared memory
template <int NB>
struct SharedSrc {
    static constexpr int kOps = 2048 * NB;  // K and V operands of a tile, 1024 NB each
    const uint8_t *ops, *scl;               // [..][kOps], [..][64 NB]: K scales, V scales
    int lane, t, first = 0;
    __device__ __forceinline__ void k(int) {}
    __device__ __forceinline__ void v(int) {}
    template <int NT>
    __device__ __forceinline__ void kblock(int) {}
    __device__ __forceinline__ uint4 kop(int i, int n, int b) const {
        return reinterpret_cast<const uint4*>(ops + (first + i) * kOps)[(2 * b + n) * 32 + lane];
    }
    __device__ __forceinline__ uint32_t ksc(int i, int n, int b) const {
        return *reinterpret_cast<const uint32_t*>(scl + (first + i) * 64 * NB + t * 8 * NB + 8 * b + 4 * n);
    }
    __device__ __forceinline__ uint4 vop(int i, int b, int half) const {
        return reinterpret_cast<const uint4*>(ops + (first + i) * kOps)[(2 * NB + 2 * b + half) * 32 + lane];
    }
    __device__ __forceinline__ uint2 vsc(int i, int b) const {
        return *reinterpret_cast<const uint2*>(scl + (first + i) * 64 * NB + 32 * NB + t * 8 * NB + 8 * b);
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

// CTAs of an SM: what 168 (head_dim 96, 128) or 128 registers a thread allow
template <int NB>
constexpr int kPerSm = NB > 2 ? 3 : 4;
// query operands in shared memory where the accumulators leave no registers
template <int NB>
constexpr bool kInShared = NB > 2;

// Few rows.  The work is the line of all units' pairs of tiles (units in the
// order of sequence, kv head, row tile), each unit headed by kHead empty places
// for what starting and joining it costs (5 us of a CTA, about 8 pairs); CTA i of
// n takes places [P i / n, P (i + 1) / n) of it, whatever the sequences' lengths,
// so one wave of CTAs ends together.  A border inside a head counts as the
// unit's start.  A unit that lies in one CTA is written out; of one that goes
// over several, each CTA leaves its sums in `part` (slot 2 i where the piece
// begins its range, 2 i + 1 where it starts later) and the CTA that starts it
// says in desc[i] how many there are.
//
// Bound by the issue of the instructions that unpack the codes (some 430 a tile of
// 16 positions, head_dim 128, at 2 a cycle and SM): 64 sequences of up to 8192
// positions, 32 bf16 heads on 8, take 109 us (2.8 TB/s of the cache), 131072
// positions of one under 64 f32 heads on 8 59 us (2.5 TB/s), 2000 of one 12.7 us
// (two launches and a CTA's latencies).
constexpr int kHead = 8;
constexpr int kChunk = 128;  // sequences looked up at a time

struct Piece {
    int b, kvh, r0, t0, t1, slot, whole, more;
};
// A CTA's way along the line, in shared memory; warp 0 walks it one piece ahead
// of the work.
template <int R>
struct Line {
    int64_t total, x0, x1, at, before, end;  // places; `before`: of the chunks so far; `end`: of sequence b
    int64_t ends[kChunk];                    // of the chunk's sequences
    int b0, b, tile0, tile1, places, row_tiles, cta, ctas;
    Piece piece[2];

    // places of a unit of sequence q, and of the sequence (a pair at least:
    // rows that see nothing are written too)
    static __device__ __forceinline__ int places_of(const AttnP& p, const Seq& q, int& tile0, int& tile1) {
        q.tiles(p, 0, q.n_q - 1, tile0, tile1);
        return max((tile1 - tile0 + 1) / 2, 1) + kHead;
    }
    static __device__ __forceinline__ int64_t line_of(const AttnP& p, int b) {
        if (b >= p.batch) return 0;
        const Seq q(p, b);
        int tile0, tile1;
        const int row_tiles = (q.n_q * p.group + R - 1) / R;
        return (int64_t)places_of(p, q, tile0, tile1) * p.n_kv * row_tiles;
    }
    // warp 0: the next piece
    __device__ __noinline__ void next(const AttnP& p, Piece& o) {
        const int lane = threadIdx.x & 31;
        if (lane == 0) o.more = 0;
        if (at >= x1) return;
        if (at >= end) {
            while (at >= before) {  // the chunk that holds the place
                const int first = b0 + kChunk;
                if (first >= p.batch) return;
                int64_t v[kChunk / 32], sum = 0;
#pragma unroll
                for (int i = 0; i < kChunk / 32; i++) v[i] = line_of(p, first + lane * (kChunk / 32) + i);
#pragma unroll
                for (int i = 0; i < kChunk / 32; i++) sum += v[i];
                int64_t upto = sum;
#pragma unroll
                for (int i = 1; i < 32; i <<= 1) {
                    const int64_t u = __shfl_up_sync(0xffffffffu, upto, i);
                    if (lane >= i) upto += u;
                }
                int64_t e = before + upto - sum;
#pragma unroll
                for (int i = 0; i < kChunk / 32; i++) ends[lane * (kChunk / 32) + i] = e += v[i];
                const int64_t all = before + __shfl_sync(0xffffffffu, upto, 31);
                __syncwarp();
                if (lane == 0) {
                    b0 = first;
                    before = all;
                }
                __syncwarp();
            }
            int lo = 0, hi = kChunk - 1;  // the first sequence whose end lies behind it
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (ends[mid] > at) hi = mid;
                else lo = mid + 1;
            }
            const Seq q(p, b0 + lo);
            int ta, tb;
            const int n = places_of(p, q, ta, tb);
            __syncwarp();
            if (lane == 0) {
                b = b0 + lo;
                end = ends[lo];
                tile0 = ta;
                tile1 = tb;
                places = n;
                row_tiles = (q.n_q * p.group + R - 1) / R;
            }
            __syncwarp();
        }
        if (lane != 0) return;
        // counted from the sequence's end, which needs no start
        const int64_t left = end - at;
        const int unit = (int)(((int64_t)p.n_kv * row_tiles * places - left) / places);
        int off = places - (int)((left - 1) % places) - 1;
        const bool first = at == x0;
        if (off <= kHead) {  // (only the range's start can lie inside a head)
            at -= off;
            off = 0;
        }
        const int stop = (int)min((int64_t)places, off + (x1 - at));
        if (stop <= kHead) {  // the next CTA's
            at = x1;
            return;
        }
        o.whole = off == 0 && stop == places;
        o.slot = 2 * cta + (first ? 0 : 1);
        o.b = b;
        o.kvh = unit / row_tiles;
        o.r0 = (unit - o.kvh * row_tiles) * R;
        o.t0 = tile0 + 2 * max(off - kHead, 0);
        o.t1 = min(tile0 + 2 * (stop - kHead), tile1);
        o.more = 1;
        at += stop - off;
        if (off == 0 && !o.whole) {
            // the CTA that holds the unit's last place: the largest i with
            // total * i / ctas <= it
            const int64_t behind = at - stop + places;
            p.desc[cta] = make_int4(b, unit, (int)((behind * ctas + total - 1) / total - cta), o.slot);
        }
    }
};

template <int NB, int MODE, typename T>
__global__ void __launch_bounds__(kWarps * 32, kPerSm<NB>) kv4_attn_kernel(const __grid_constant__ AttnP p) {
    using Rec = Kv4Rec<NB>;
    constexpr bool kAs = kInShared<NB>;
    using W = Warp<NB, MODE, T, 1, kAs>;
    constexpr int R = W::R, H = W::H, HD = 32 * NB, kThreads = kWarps * 32;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[kWarps][kStages];
    __shared__ float s_m[kWarps][R], s_l[kWarps][R], s_f[R][kWarps];
    __shared__ int64_t s_at[R], s_sum[kWarps];
    __shared__ Line<R> line;
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int cta = (int)blockIdx.x;
    // the line's length: every thread sums some sequences
    int64_t total = 0;
    for (int b = threadIdx.x; b < p.batch; b += kThreads) total += Line<R>::line_of(p, b);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) total += __shfl_xor_sync(0xffffffffu, total, i);
    if (lane == 0) s_sum[warp] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int x = 0; x < kWarps; x++) total += s_sum[x];
    if (threadIdx.x == 0 && p.desc) p.desc[cta] = make_int4(0, 0, 0, 0);
    // no more CTAs than places, so that none in the middle of a unit is idle
    const int ctas = (int)min((int64_t)gridDim.x, total);
    if (cta >= ctas) return;
    if (warp == 0) {
        if (lane == 0) {
            line.total = total;
            line.at = line.x0 = total * cta / ctas;
            line.x1 = total * (cta + 1) / ctas;
            line.before = line.end = 0;
            line.b0 = -kChunk;
            line.cta = cta;
            line.ctas = ctas;
        }
        __syncwarp();
        line.next(p, line.piece[0]);
    }
    const uint8_t* ring = smem + warp * kStages * 2 * Rec::kBytes;
    Stream<kStages, Rec::kBytes, kWarps> in(p, smem_u32(ring), smem_u32(&bars[warp][0]), lane);
    RecordSrc<NB, kAs> src;
    src.lane = lane;
    src.t = t;
    src.magic = p.magic;
    float* const joint = reinterpret_cast<float*>(smem + kWarps * kStages * 2 * Rec::kBytes);
    __syncthreads();
    if (line.piece[0].more) in.begin(line.piece[0].b, line.piece[0].kvh, line.piece[0].t0 + 2 * warp, line.piece[0].t1);
    bool bad = false;
    for (int turn = 0; line.piece[turn].more; turn ^= 1) {
        const Piece& cur = line.piece[turn];
        if (warp == 0) line.next(p, line.piece[turn ^ 1]);
        const Rows o(p, cur.b, cur.kvh, cur.r0);
        W w;
        w.as = reinterpret_cast<uint4*>(joint + warp * (R * HD));  // this warp's part, free until the join
        w.init(p, o, o.r0, g, t);
        const int t0 = cur.t0;
        int s = 0;
        for (int k = 0; k < in.n; k++) {
            const uint32_t there = in.there(s);
            if (there) {  // what is not in the cache is not seen
                if (!in.wait(s)) {
                    in.abandon(k);
                    bad = true;
                    break;
                }
                src.rec = ring + s * 2 * Rec::kBytes;
                w.pair(p, t0 + 2 * (warp + k * kWarps), there, t, src);
                __syncwarp();
            }
            if (k + kStages < in.n) in.issue(k + kStages, s);
            s = s + 1 == kStages ? 0 : s + 1;
        }
        w.finish();
        // ---- join the warps: each one's m, l and row sums through shared
        // memory (where the query operands were), while the next piece's first
        // copies are under way
        if (kAs) __syncwarp();
        float* so = joint + warp * (R * HD);
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
                    *reinterpret_cast<float2*>(so + (g + 8 * h) * HD + 32 * b + 8 * n + 2 * t) = w.value(b, n, h);
        }
        if (__syncthreads_or(bad)) return;
        {
            const Piece& nxt = line.piece[turn ^ 1];
            if (nxt.more) in.begin(nxt.b, nxt.kvh, nxt.t0 + 2 * warp, nxt.t1);
        }
        if (threadIdx.x < R) {  // a thread a row: the warps' weights, and where the row goes
            const int row = threadIdx.x, r = o.r0 + row;
            const int i = r / p.group, head = o.kvh * p.group + r - i * p.group;
            const int64_t tok = (int64_t)o.q0 + i;
            float M = -INFINITY, L = 0.0f, f[kWarps];
#pragma unroll
            for (int x = 0; x < kWarps; x++) M = fmaxf(M, s_m[x][row]);
#pragma unroll
            for (int x = 0; x < kWarps; x++) {
                f[x] = weight(s_m[x][row], M);
                L = fmaf(f[x], s_l[x][row], L);
            }
            const bool ok = r < o.rows && tok >= 0 && tok < p.n_tokens;
            const float scale = cur.whole && L != 0.0f ? 1.0f / L : 1.0f;
#pragma unroll
            for (int x = 0; x < kWarps; x++) s_f[row][x] = f[x] * scale;
            s_at[row] = !ok ? -1 : cur.whole ? tok * p.ot + head * p.oh : ((int64_t)cur.slot * R + row) * HD;
            if (ok && !cur.whole) p.ml[cur.slot * R + row] = make_float2(M, L);
        }
        __syncthreads();
#pragma unroll
        for (int e = threadIdx.x * 2; e < R * HD; e += kThreads * 2) {
            const int row = e / HD, d = e % HD;
            const int64_t to = s_at[row];
            const float4 f = *reinterpret_cast<const float4*>(s_f[row]);
            const float ff[kWarps] = {f.x, f.y, f.z, f.w};
            float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int x = 0; x < kWarps; x++) {
                const float2 v = *reinterpret_cast<const float2*>(joint + x * (R * HD) + e);
                acc.x = fmaf(ff[x], v.x, acc.x);
                acc.y = fmaf(ff[x], v.y, acc.y);
            }
            if (to < 0) continue;
            if (cur.whole) {
                T* dst = static_cast<T*>(p.out) + to + d;
                dst[0] = from_f32<T>(acc.x);
                dst[1] = from_f32<T>(acc.y);
            } else {
                *reinterpret_cast<float2*>(p.part + to + d) = acc;
            }
        }
        __syncthreads();  // the sums (and this piece) have been read
    }
}

// Many rows: warp i holds rows r0 + i R ..; a step is kWarps tiles, two to a
// stream.  Two warps share a stream: one unpacks its K, the other its V into
// f16 operands that all four use.
// Bound by the issue of products and of what surrounds them (mma.sync, 255
// registers, two CTAs an SM): three prompts of 300, 150 and 225 tokens on 1600,
// 3100 and 4500 positions, 64 heads on 8, head_dim 128, take 552 us in f32 and
// 548 in f16 (bf16, on tcgen05: 132).
template <int NB, typename T>
__global__ void __launch_bounds__(kWarps * 32, 2) kv4_attn_rows_kernel(const __grid_constant__ AttnP p) {
    using Rec = Kv4Rec<NB>;
    using W = Warp<NB, kSplit8, T, 2, true>;
    constexpr int R = W::R, H = W::H, HD = 32 * NB, kLists = kWarps / 2;
    constexpr int kOps = SharedSrc<NB>::kOps;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[kLists][kStagesRows];
    __shared__ uint32_t s_there[kWarps];  // of the step's pairs; bit 2: a copy did not arrive
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int list = warp >> 1, is_v = warp & 1;
    const int unit = (int)(blockIdx.x / p.splits), split = (int)blockIdx.x - unit * p.splits;
    const Rows o = unit_rows<R * kWarps>(p, unit);
    if (o.r0 >= o.rows) return;
    int tile0, tile1, per;
    unit_tiles<R * kWarps>(p, o, tile0, tile1, per);
    const int t0 = tile0 + split * per, t1 = min(t0 + per, tile1);
    if (p.splits > 1 && t0 >= t1) return;  // the join does not read this split
    uint8_t* ops = smem;                  // [kWarps][kOps]
    uint8_t* scl = smem + kWarps * kOps;  // [kWarps][64 NB]
    const uint8_t* ring = scl + kWarps * 64 * NB + list * kStagesRows * 2 * Rec::kBytes;
    Stream<kStagesRows, Rec::kBytes, kLists> in(p, smem_u32(ring), smem_u32(&bars[list][0]), lane, !is_v);
    in.begin(o.b, o.kvh, t0 + 2 * list, t1);
    const int steps = t1 > t0 ? (t1 - t0 + kWarps - 1) / kWarps : 0;
    W w;
    w.as = reinterpret_cast<uint4*>(scl + kWarps * 64 * NB + kLists * kStagesRows * 2 * Rec::kBytes) + warp * (2 * NB * 2 * 32);
    const int r0 = o.r0 + warp * R;
    w.init(p, o, r0, g, t);
    // tiles that this warp's rows see
    const int last = r0 < o.rows ? (max(w.seen, 0) + kKv4Tile - 1) / kKv4Tile : 0;
    SharedSrc<NB> src;
    src.lane = lane;
    src.t = t;
    __syncthreads();  // the barriers are there
    int s = 0;
    for (int k = 0; k < steps; k++) {
        uint32_t there = k < in.n ? in.there(s) : 0;
        if (there && !in.wait(s)) there = 4;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (!((there >> i) & 1u)) continue;
            const uint8_t* rec = ring + (2 * s + i) * Rec::kBytes;
            uint4* dst = reinterpret_cast<uint4*>(ops + (2 * list + i) * kOps) + lane;
            uint32_t x[2 * NB];
            load_words<NB>(rec + is_v * Rec::kV, lane, x);
            if (is_v) {
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int n = 0; n < 2; n++)
                        dst[(2 * NB + 2 * b + n) * 32] = v_operands(x[2 * b] >> (8 * n), x[2 * b + 1] >> (8 * n), p.magic);
            } else {
#pragma unroll
                for (int b = 0; b < 2 * NB; b++) dst[b * 32] = k_operands(x[b], p.magic);
            }
            if (lane < 2 * NB)  // its scales
                reinterpret_cast<uint4*>(scl + (2 * list + i) * 64 * NB)[is_v * 2 * NB + lane] =
                    reinterpret_cast<const uint4*>(rec + Rec::kKs)[is_v * 2 * NB + lane];
        }
        if (lane == 0) s_there[warp] = there;
        __syncthreads();
        if (k + kStagesRows < in.n && there < 4) in.issue(k + kStagesRows, s);
        s = s + 1 == kStagesRows ? 0 : s + 1;
        bool stop = false;
#pragma unroll 1
        for (int i = 0; i < kLists; i++) {
            const int tile = t0 + 2 * (k * kLists + i);
            uint32_t at = s_there[2 * i];
            stop |= at >= 4 || s_there[2 * i + 1] >= 4;
            if (tile + 1 >= last) at &= tile < last ? 1u : 0u;
            src.ops = ops + 2 * i * kOps;
            src.scl = scl + 2 * i * 64 * NB;
            w.pair(p, tile, at & 3u, t, src);
        }
        __syncthreads();
        if (stop) {
            in.abandon(k + (there < 4 ? 1 : 0));
            break;
        }
    }
    w.finish();
#pragma unroll
    for (int h = 0; h < H; h++) {
        const int r = r0 + W::row_of(g, h);
        const int i = r / p.group, head = o.kvh * p.group + r - i * p.group;
        const int64_t tok = (int64_t)o.q0 + i;
        if (r >= o.rows || tok < 0 || tok >= p.n_tokens) continue;
        if (p.splits == 1) {
            T* dst = static_cast<T*>(p.out) + tok * p.ot + head * p.oh + 2 * t;
            const bool two = ((uintptr_t)dst & 7) == 0;
            const bool any = w.l[h] != 0.0f;  // (not a number counts)
            const float f = 1.0f / w.l[h];
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const float2 v = w.value(b, n, h);
                    store2(dst + 32 * b + 8 * n, two, any ? v.x * f : 0.0f, any ? v.y * f : 0.0f);
                }
        } else {
            const int64_t at = (tok * p.n_heads + head) * p.splits + split;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int n = 0; n < 4; n++)
                    *reinterpret_cast<float2*>(p.part + at * HD + 32 * b + 8 * n + 2 * t) = w.value(b, n, h);
            if (t == 0) p.ml[at] = make_float2(w.m[h], w.l[h]);
        }
    }
}

// Many rows of bf16 queries: 128 rows and steps of 64 positions on tcgen05.
//
// K and V enter as f16 values (c - 8) d / 2^E, one rounding of 2^-11 of each, and
// P as f16: an eighth each of the rounding that bf16 gives the output.  (Kept exact --
// a product a block, scaled in the softmax, P times each block's scales -- S and
// P crossed TMEM head_dim / 32 times, for 1.3 times the softmax's time.)  E is
// that of 32 positions: their largest scale comes to [2^11, 2^12) -- so that 8 d
// still is an f16 -- or stays below it with the power at its floor, and only scales
// 2^26 times smaller than that lose bits.  A row's reference m follows the largest
// s_j + E_j that it sees, and P is 2^(s_j + E_j - m): the products that count most
// keep their bits beside values of any size that count little (with E's largest and
// the scores' each followed for itself, one value of 5e5 without weight took 12 bits
// from all weights: 75 % of an output made of weights of 2^-18).  A value that
// is not a number cannot lie in an operand that rows share which do not see it:
// it enters as zero, and the rows that do see it are marked and get it at the
// end.
//
// Two groups of four warps do the softmax, a thread a row, each with its own S (64
// columns of TMEM), P as the A operand (32) and O (32 NB): with PAIR of a tile of
// 128 rows each, so that unpacking a step serves 256 rows; else of even and of odd
// steps of one tile, with their own maxima and sums, joined at the end (one group
// with half the positions a warp, which agreed on every step's maximum, took 318 us
// where the two took 279).  PAIR from 129 rows: 192 rows of 8 heads a kv head of 8,
// head_dim 128, 16 x 2048 positions 84 -> 66 us, 64 x 1024 182 -> 158, 1 x 40000
// 94 -> 83; at 128 rows, where its second tile would be empty, the steps' latencies
// are not hidden (41, 102, 54 us as it is).
//
// Roles (17 warps):
//   0 - 7   softmax, group w / 4, rows 32 (w % 4) + lane of the tile
//   8       issues the products: S ahead of P V by a step of the group
//   9 - 16  unpack, even steps the first four, odd ones the others: two warps a
//           half of the step, one K, one V, into the 128-byte-swizzled operands
//           (three or four buffers: with two, and one group, unpacking a step
//           waited for the products two steps before, 3400 cycles a step where
//           this takes 2000)
//
// Three prompts of 512 tokens on 4500 positions, 64 query heads on 8, head_dim 128:
// 377 us (567 TFLOP/s); of 256, 384 and 512 tokens on up to 4500 positions each, 220
// to 252 as the lengths fall out (some 300 TFLOP/s).  The chains of the softmax
// (TMEM read, maximum, exponentials, TMEM write) and of the unpacking bound these,
// at 1.8 instructions a cycle and SM, and the last wave's length: in the second case
// 288 CTAs on 148 SMs, the tensor pipe busy for a quarter of the time.
constexpr int kTcRows = 128, kTcStep = 64, kTcWarps = 17;
constexpr int kTcTop = 12, kTcLow = -8;  // see E
constexpr float kTcUp = 7.0f;  // the largest P lies in [2^7, 2^15], so that f16 has it to 2^-11 down to 2^-21 of that

template <int NB, bool PAIR>
struct TcSmem {  // dynamic shared memory from a 1024-byte border
    static constexpr int kOps = PAIR ? 3 : 4;    // operand buffers
    static constexpr int kAtoms = (NB + 1) / 2;  // 64 elements = 128 bytes of a row
    static constexpr int kQ = 0, kK = (PAIR ? 2 : 1) * kAtoms * 16384, kV = kK + kOps * kAtoms * 8192,
                         kRing = kV + kOps * NB * 4096;
    static constexpr int kScl = kRing + 4 * 2 * 2 * 576 * NB;  // [8 unpacking warps][2 tiles][32 NB]
    static constexpr int kBytes = kScl + 8 * 2 * 32 * NB;
    static constexpr int kCols = NB == 1 ? 256 : 512;
};
// byte of 16-byte chunk c of row r in a 128-byte-swizzled operand
__device__ __forceinline__ int sw128(int r, int c) { return (r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4); }
__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) { return as_u32(__hmul2(as_h2(a), as_h2(b))); }
// halves of all ones where w's f16 is not a number
__device__ __forceinline__ uint32_t nan_halves(uint32_t w) {
    return __hne2_mask(as_h2(w), as_h2(w));
}

template <int NB, bool PAIR, typename T>
__global__ void __launch_bounds__(kTcWarps * 32, 1) kv4_attn_tc_kernel(const __grid_constant__ AttnP p) {
    using Rec = Kv4Rec<NB>;
    using S = TcSmem<NB, PAIR>;
    constexpr int kTcOps = S::kOps, kAllRows = PAIR ? 2 * kTcRows : kTcRows;
    constexpr int HD = 32 * NB, kPCol = 128, kOCol = 192;  // TMEM: the groups' S, P, O
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[4][2], b_ops_full[kTcOps], b_ops_empty[kTcOps], b_s_full[2], b_s_empty[2],
        b_p_full[2], b_pv_done[2];
    __shared__ float s_qs[kAllRows], s_m[2][kTcRows], s_l[2][kTcRows];
    __shared__ float s_kf[kTcOps][2];  // of a step's half: 2^E of K, E of V, tiles that are there
    __shared__ int s_E[kTcOps][2], s_there[kTcOps][2], s_any_nan[kTcOps][2];
    __shared__ uint32_t s_nan[kTcOps][2][NB], s_bad[2][kTcRows];  // positions that are not numbers: of a step's half, by block
    __shared__ uint32_t s_tmem;
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a sequence's last rows, which see the most, first
    const int at0 = (int)(blockIdx.x / p.splits), split = (int)blockIdx.x - at0 * p.splits;
    const int unit = (int)(gridDim.x / p.splits) - 1 - at0;
    const Rows o = unit_rows<kAllRows>(p, unit);
    if (o.r0 >= o.rows) return;
    int tile0, tile1, per;
    unit_tiles<kAllRows>(p, o, tile0, tile1, per);
    const int t0 = tile0 + split * per, t1 = min(t0 + per, tile1);
    if (p.splits > 1 && t0 >= t1) return;  // the join does not read this split
    const int steps = t1 > t0 ? (t1 - t0 + 3) / 4 : 0;
    const int i1 = min(o.n_q - 1, (o.r0 + kAllRows - 1) / p.group);
    const int groups = PAIR && o.rows - o.r0 <= kTcRows ? 1 : 2;
    const int seen = max(0, min(o.held, o.pos0 + i1 + 1));  // positions that any row sees end here
    uint8_t* const sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sm32 = smem_u32(sm);

    // ---- set-up: barriers, TMEM, the query operand, the first records
    const int pw = warp - 9, list = pw >> 1, is_v = pw & 1;
    Stream<2, Rec::kBytes, 4> in(p, sm32 + S::kRing + (warp >= 9 ? list : 0) * 2 * 2 * Rec::kBytes,
                                 smem_u32(&bars[warp >= 9 ? list : 0][0]), lane, warp >= 9 && !is_v);
    if (warp >= 9) {
        in.begin(o.b, o.kvh, t0 + 2 * list, t1);
    } else if (warp == 8) {
        if (lane == 0) {
            for (int i = 0; i < kTcOps; i++) {
                mbar_init(smem_u32(&b_ops_full[i]), 4);
                mbar_init(smem_u32(&b_ops_empty[i]), 1);
            }
            for (int i = 0; i < 2; i++) {
                mbar_init(smem_u32(&b_s_full[i]), 1);
                mbar_init(smem_u32(&b_s_empty[i]), 4);
                mbar_init(smem_u32(&b_p_full[i]), 4);
                mbar_init(smem_u32(&b_pv_done[i]), 1);
            }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                     "r"((uint32_t)S::kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
        // two lanes a row: normalised by a power of two to f16, which is exact
        // for f16 and (but for elements below 2^-14 of the largest) bf16
#pragma unroll 1
        for (int tile = 0; tile < (PAIR ? groups : 1); tile++) {
            const int row = tile * kTcRows + (threadIdx.x >> 1), r = o.r0 + row;
            const int i = r / p.group, head = o.kvh * p.group + r - i * p.group;
            const int64_t tok = (int64_t)o.q0 + i;
            const bool ok = r < o.rows && tok >= 0 && tok < p.n_tokens;
            const T* q = static_cast<const T*>(p.q) + tok * p.qt + head * p.qh;
            float x[2 * NB][8];  // chunks 2 c + (lane & 1)
            float mx = 0.0f;
#pragma unroll
            for (int c = 0; c < 2 * NB; c++) {
#pragma unroll
                for (int e = 0; e < 8; e++) x[c][e] = 0.0f;
                if (ok) load8(q + 8 * (2 * c + (lane & 1)), p.wide, x[c]);
            }
#pragma unroll
            for (int c = 0; c < 2 * NB; c++)
#pragma unroll
                for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[c][e]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            int e2 = 0;
            if (mx > 0.0f && mx < INFINITY) frexpf(mx, &e2);
            e2 = max(-120, min(120, e2));
            // the scale's sign is the operand's, so that scores grow with their sums
            const float down = p.scale == 0.0f ? 0.0f : copysignf(__int_as_float((127 - e2) << 23), p.scale);
            if ((lane & 1) == 0) s_qs[row] = p.scale == 0.0f ? 1.0f : __int_as_float((127 + e2) << 23) * fabsf(p.scale);
#pragma unroll
            for (int c = 0; c < 2 * NB; c++) {
                const int at = 2 * c + (lane & 1);
                *reinterpret_cast<uint4*>(sm + S::kQ + (tile * S::kAtoms + (at >> 3)) * 16384 + sw128(row & (kTcRows - 1), at & 7)) =
                    make_uint4(pack(x[c][0] * down, x[c][1] * down), pack(x[c][2] * down, x[c][3] * down),
                               pack(x[c][4] * down, x[c][5] * down), pack(x[c][6] * down, x[c][7] * down));
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc::tmem_fence_before();
    __syncthreads();
    tc::tmem_fence_after();
    const uint32_t tmem = s_tmem;
    bool ok = true;

    if (warp >= 9) {
        // ---------------------------------------------------------- unpack
        const int g = lane >> 2, t = lane & 3, half = list & 1;
        const Magic magic = p.magic;
        uint8_t* const scl = sm + S::kScl + pw * 2 * 32 * NB;
        // where the lane's values go: V, elements g, + 8, .. and positions 4 t .. + 3
        // of tile i; K, elements 8 t .. (chunk t, or t + 4 for odd blocks) of positions
        // 4 (g / 2) + g % 2 + 2 n of the half's first tile
        int at[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
            at[i] = is_v ? sw128(g, 4 * half + 2 * i + (t >> 1)) + 8 * (t & 1)
                         : half * 4096 + sw128(4 * (g >> 1) + (g & 1) + 2 * i, t);
        const uint32_t pick = g & 1 ? 0x3232u : 0x1010u;
        for (int j = 0; 2 * j + (list >> 1) < steps; j++) {
            const int k = 2 * j + (list >> 1), st = k % kTcOps, s = j & 1;
            if (ok && k >= kTcOps && !mbar_wait(smem_u32(&b_ops_empty[st]), ((k / kTcOps) - 1) & 1)) ok = false;
            uint32_t there = j < in.n ? in.there(s) : 0;
            if (ok && there && !in.wait(s)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) there = 0;
            const uint8_t* rec = sm + S::kRing + (list * 2 + s) * 2 * Rec::kBytes;
            // ---- scales: lane u holds those of token group u / NB, block u % NB
            // (four tokens) of both tiles; positions that nobody sees count
            // for nothing, whatever lies there
            uint2 sc[2];
            uint32_t bad[2] = {0u, 0u};  // tokens (bits 0 - 3) whose value is not a number
            __half2 big = __half2half2(__ushort_as_half(0));
            const bool ends = (t0 + 4 * k + 2 * half + 2) * kKv4Tile > seen;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                sc[i] = make_uint2(0u, 0u);
                if (((there >> i) & 1u) && lane < 4 * NB) {
                    sc[i] = *reinterpret_cast<const uint2*>(rec + i * Rec::kBytes + Rec::kKs + is_v * 32 * NB + lane * 8);
                    if (ends) {
                        const int left = seen - ((t0 + 4 * k + 2 * half + i) * kKv4Tile + 4 * (lane / NB));
                        if (left < 4) {
                            sc[i].y &= left > 2 ? 0x0000FFFFu : 0u;
                            sc[i].x &= left > 1 ? 0xFFFFFFFFu : left > 0 ? 0x0000FFFFu : 0u;
                        }
                    }
                    if (is_v) {
                        const uint32_t nx = nan_halves(sc[i].x), ny = nan_halves(sc[i].y);
                        bad[i] = (nx & 1u) | ((nx >> 15) & 2u) | ((ny & 1u) << 2) | ((ny >> 13) & 8u);
                        sc[i].x &= ~nx;
                        sc[i].y &= ~ny;
                    }
                }
                big = __hmax2(big, __hmax2(__habs2(as_h2(sc[i].x)), __habs2(as_h2(sc[i].y))));
            }
            float dm = fmaxf(__half2float(__low2half(big)), __half2float(__high2half(big)));
            int E = kTcLow;
            if (__any_sync(0xffffffffu, dm > __int_as_float((127 + kTcTop + kTcLow) << 23))) {
#pragma unroll
                for (int i = 16; i > 0; i >>= 1) dm = fmaxf(dm, __shfl_xor_sync(0xffffffffu, dm, i));
                frexpf(dm, &E);
                E -= kTcTop;
            }
            if (is_v) {
                const bool some = __any_sync(0xffffffffu, bad[0] | bad[1]);
                if (lane < NB) s_nan[st][half][lane] = 0u;
                if (lane == 0) {
                    s_any_nan[st][half] = some;
                    s_E[st][half] = E;
                }
                __syncwarp();
            } else if (lane == 0) {
                s_kf[st][half] = __int_as_float((127 + E) << 23);
                s_there[st][half] = (int)there;
            }
            const uint32_t inv = as_u32(__float2half2_rn(__int_as_float((127 - E) << 23)));
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (lane < 4 * NB)
                    *reinterpret_cast<uint2*>(scl + i * 32 * NB + lane * 8) = make_uint2(times(sc[i].x, inv), times(sc[i].y, inv));
                if (bad[i]) atomicOr(&s_nan[st][half][lane % NB], bad[i] << (16 * i + 4 * (lane / NB)));
            }
            __syncwarp();
            // ---- values
#pragma unroll
            for (int i = 0; i < 2; i++) {
                uint32_t x[2 * NB];
                if ((there >> i) & 1u) {
                    load_words<NB>(rec + i * Rec::kBytes + is_v * Rec::kV, lane, x);
                } else {
#pragma unroll
                    for (int b = 0; b < 2 * NB; b++) x[b] = 0x88888888u;  // zeros
                }
                if (is_v) {
                    uint8_t* dst = sm + S::kV + st * NB * 4096 + at[i];
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const uint2 d = *reinterpret_cast<const uint2*>(scl + i * 32 * NB + (t * NB + b) * 8);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const uint4 v = v_operands(x[2 * b] >> (8 * h), x[2 * b + 1] >> (8 * h), magic);
                            *reinterpret_cast<uint2*>(dst + b * 4096 + h * 2048) = make_uint2(times(v.x, d.x), times(v.y, d.y));
                            *reinterpret_cast<uint2*>(dst + b * 4096 + h * 2048 + 1024) = make_uint2(times(v.z, d.x), times(v.w, d.y));
                        }
                    }
                } else {
                    uint8_t* dst = sm + S::kK + st * S::kAtoms * 8192 + i * 2048;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const uint2 d = *reinterpret_cast<const uint2*>(scl + i * 32 * NB + ((g >> 1) * NB + b) * 8);
#pragma unroll
                        for (int n = 0; n < 2; n++) {
                            const uint32_t dd = __byte_perm(n ? d.y : d.x, 0u, pick);
                            const uint4 v = k_operands(x[2 * b + n], magic);
                            *reinterpret_cast<uint4*>(dst + (b >> 1) * 8192 + (b & 1 ? at[n] ^ 64 : at[n])) =
                                make_uint4(times(v.x, dd), times(v.y, dd), times(v.z, dd), times(v.w, dd));
                        }
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&b_ops_full[st]));
            named_bar_sync(5 + list, 64);  // both warps have read the records
            if (ok && j + 2 < in.n) in.issue(j + 2, s);
        }
        if (!ok) in.abandon(0);
    } else if (warp == 8) {
        // -------------------------------------------------------- products
        constexpr uint32_t kIdS = (1u << 4) | ((uint32_t)(kTcStep >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
        constexpr uint32_t kIdO = (1u << 4) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
        constexpr int kAhead = PAIR ? 1 : 2;  // steps from S to P V
        for (int k = -kAhead; k < steps; k++) {
            // (without PAIR a step belongs to one group, as its n-th)
            if (const int j = k + kAhead; j < steps) {
                const int os = j % kTcOps, n = PAIR ? j : j >> 1;
                if (ok && !mbar_wait(smem_u32(&b_ops_full[os]), (j / kTcOps) & 1)) ok = false;
                for (int g = PAIR ? 0 : j & 1; g < (PAIR ? groups : (j & 1) + 1); g++) {
                    if (ok && n > 0 && !mbar_wait(smem_u32(&b_s_empty[g]), (n - 1) & 1)) ok = false;
                    ok = __all_sync(0xffffffffu, ok);
                    tc::tmem_fence_after();
                    if (tc::elect_one()) {
                        if (ok) {
                            const uint32_t qa = sm32 + S::kQ + (PAIR ? g * S::kAtoms * 16384 : 0);
#pragma unroll
                            for (int x = 0; x < 2 * NB; x++)
                                tc::umma_f16(tmem + 64 * g, tc::desc_sw128(qa + (x >> 2) * 16384 + 32 * (x & 3)),
                                             tc::desc_sw128(sm32 + S::kK + (os * S::kAtoms + (x >> 2)) * 8192 + 32 * (x & 3)), kIdS,
                                             x ? 1u : 0u);
                        }
                        tc::umma_commit(smem_u32(&b_s_full[g]));
                    }
                    __syncwarp();
                }
            }
            if (k >= 0) {
                const int os = k % kTcOps, n = PAIR ? k : k >> 1;
                const int last = PAIR ? groups - 1 : k & 1;
                for (int g = PAIR ? 0 : k & 1; g <= last; g++) {
                    if (ok && !mbar_wait(smem_u32(&b_p_full[g]), n & 1)) ok = false;
                    ok = __all_sync(0xffffffffu, ok);
                    tc::tmem_fence_after();
                    if (tc::elect_one()) {
                        if (ok) {
#pragma unroll
                            for (int x = 0; x < 4; x++)
                                tc::umma_f16_ts(tmem + kOCol + g * HD, tmem + kPCol + 32 * g + 8 * x,
                                                tc::desc_sw128(sm32 + S::kV + os * NB * 4096 + 32 * x), kIdO, n > 0 || x > 0 ? 1u : 0u);
                        }
                        tc::umma_commit(smem_u32(&b_pv_done[g]));
                        if (g == last) tc::umma_commit(smem_u32(&b_ops_empty[os]));
                    }
                    __syncwarp();
                }
            }
        }
        // the last commits' arrivals, which nobody else may wait for, may not
        // find the CTA gone
        for (int k = max(0, steps - kTcOps); k < steps; k++)
            if (ok && !mbar_wait(smem_u32(&b_ops_empty[k % kTcOps]), (k / kTcOps) & 1)) ok = false;
        if (!ok && lane == 0) atomicExch(p.err, 1);
    } else {
        // --------------------------------------------------------- softmax
        const int q = warp & 3, h = warp >> 2, row = 32 * q + lane, at_row = row + (PAIR ? h * kTcRows : 0);
        const int r = o.r0 + at_row, i = r / p.group, head = o.kvh * p.group + r - i * p.group;
        const int64_t tok = (int64_t)o.q0 + i;
        const bool live = r < o.rows && tok >= 0 && tok < p.n_tokens;
        const int rpos = live ? o.pos0 + i : -1;
        const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16);
        const float qs = s_qs[at_row];
        const uint32_t s_at = lanes + 64 * h, p_at = lanes + kPCol + 32 * h, o_at = lanes + kOCol + HD * h;
        float m = -INFINITY, l = 0.0f;
        uint32_t bad = 0;  // blocks of O that a value which is not a number reaches
        const int mine = h >= groups ? 0 : PAIR ? steps : (steps + 1 - h) / 2;
        for (int n = 0; n < mine; n++) {
            const int k = PAIR ? n : 2 * n + h, ph = n & 1, os = k % kTcOps;
            if (ok && !mbar_wait(smem_u32(&b_ops_full[os]), (k / kTcOps) & 1)) ok = false;
            if (ok && !mbar_wait(smem_u32(&b_s_full[h]), ph)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            tc::tmem_fence_after();
            // ---- scores of positions j0 .. j0 + 63
            const int j0 = (t0 + 4 * k) * kKv4Tile;
            uint32_t a[2][32];
            tc::tmem_ld32(s_at, a[0]);
            tc::tmem_ld32(s_at + 32, a[1]);
            tc::tmem_wait_ld();
            tc::tmem_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&b_s_empty[h]));
            // ---- which of them the row sees
            uint32_t sees[2];
            float f[2], e[2], mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t there = (uint32_t)s_there[os][i];
                const int at = j0 + 32 * i;
                f[i] = fmaxf(qs * s_kf[os][i], 1.2e-38f);  // (times -inf of a masked place)
                e[i] = (float)s_E[os][i];
                const int hi = min(min(rpos + 1, o.held) - at, 32), lo = p.window > 0 ? max(rpos - p.window + 1 - at, 0) : 0;
                sees[i] = (hi >= 32 ? 0xFFFFFFFFu : hi > 0 ? (1u << hi) - 1u : 0u) & (lo >= 32 ? 0u : 0xFFFFFFFFu << lo);
                sees[i] &= (there & 1u ? 0xFFFFu : 0u) | (there & 2u ? 0xFFFF0000u : 0u);
                if (__any_sync(0xffffffffu, sees[i] != 0xFFFFFFFFu)) {
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        if (!((sees[i] >> j) & 1u)) a[i][j] = 0xFF800000u;  // -inf
                }
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 32; j++) top = fmaxf(top, __uint_as_float(a[i][j]));
                mx = fmaxf(mx, fmaf(top, f[i], e[i]));
            }
            if (s_any_nan[os][0] | s_any_nan[os][1]) {
                for (int b = 0; b < NB; b++)
                    if ((s_nan[os][0][b] & sees[0]) | (s_nan[os][1][b] & sees[1])) bad |= 1u << b;
            }
            // ---- move the row's reference where s + E grew
            float al = 1.0f;
            if (mx > m + kLazy || (m == -INFINITY && mx > -INFINITY)) {
                al = m == -INFINITY ? 0.0f : ex2(m - mx);
                l *= al;
                m = mx;
            }
            // ---- P and O are free once the group's last products are done
            if (ok && n > 0 && !mbar_wait(smem_u32(&b_pv_done[h]), ph ^ 1)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            tc::tmem_fence_after();
            if (n > 0 && __any_sync(0xffffffffu, al != 1.0f)) {
#pragma unroll 1
                for (int c = 0; c < 2 * NB; c++) {
                    uint32_t v[16];
                    tc::tmem_ld16(o_at + 16 * c, v);
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int x = 0; x < 16; x++) v[x] = __float_as_uint(__uint_as_float(v[x]) * al);
                    tc::tmem_st16u(o_at + 16 * c, v);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float base = (m == -INFINITY ? 0.0f : m) - e[i] - kTcUp;
                float2 sum = make_float2(0.0f, 0.0f);
                uint32_t pk[16];
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const float2 x = fma2(make_float2(__uint_as_float(a[i][2 * j]), __uint_as_float(a[i][2 * j + 1])),
                                          make_float2(f[i], f[i]), make_float2(-base, -base));
                    const float2 y = make_float2(ex2(x.x), ex2(x.y));
                    sum = add2(sum, y);
                    pk[j] = pack(y.x, y.y);
                }
                tc::tmem_st16u(p_at + 16 * i, pk);
                l = fmaf(sum.x + sum.y, __int_as_float((127 - (int)e[i]) << 23), l);
            }
            tc::tmem_wait_st();
            tc::tmem_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&b_p_full[h]));
        }
        if (ok && mine > 0 && !mbar_wait(smem_u32(&b_pv_done[h]), (mine - 1) & 1)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok && lane == 0) atomicExch(p.err, 1);
        float f0 = 1.0f, f1 = 0.0f;  // what the groups' O counts
        if constexpr (!PAIR) {  // the row's even and odd steps together
            s_m[h][row] = m;
            s_l[h][row] = l;
            s_bad[h][row] = bad;
            tc::tmem_fence_before();
            named_bar_sync(1 + q, 64);
            m = fmaxf(s_m[0][row], s_m[1][row]);
            const float w0 = weight(s_m[0][row], m), w1 = weight(s_m[1][row], m);
            l = s_l[0][row] * w0 + s_l[1][row] * w1;
            bad = s_bad[0][row] | s_bad[1][row];
            f0 = w0;
            f1 = w1;
        }
        tc::tmem_fence_after();
        const bool any = l != 0.0f;  // (not a number counts)
        if (p.splits == 1) {
            const float f = 1.0f / l;
            f0 *= f;
            f1 *= f;
        }
        const int64_t at = (tok * p.n_heads + head) * p.splits + split;
        T* out = static_cast<T*>(p.out) + tok * p.ot + head * p.oh;
        // PAIR: all columns of the group's rows; else columns 16 NB h .. of the tile's
#pragma unroll
        for (int c = 0; c < (PAIR ? 2 * NB : NB); c++) {
            uint32_t a0[16], a1[16];
            const int col = 16 * (PAIR ? c : h * NB + c);
            if (mine > 0 || (!PAIR && steps > 0)) tc::tmem_ld16(lanes + kOCol + (PAIR ? HD * h : 0) + col, a0);
            if (!PAIR && steps > 1) tc::tmem_ld16(lanes + kOCol + HD + col, a1);
            tc::tmem_wait_ld();
            if (!live) continue;
            const bool not_number = (bad >> (col >> 5)) & 1u;
#pragma unroll
            for (int x = 0; x < 16; x += 8) {
                float v[8];
#pragma unroll
                for (int y = 0; y < 8; y++) {
                    v[y] = any ? __uint_as_float(a0[x + y]) * f0 : 0.0f;
                    if (!PAIR && any && steps > 1) v[y] = fmaf(__uint_as_float(a1[x + y]), f1, v[y]);
                    if (not_number) v[y] = __int_as_float(0x7fffffff);
                }
                if (p.splits == 1) store8(out + col + x, p.wide_out, v);
                else store8(p.part + at * HD + col + x, true, v);
            }
        }
        if (p.splits > 1 && live && (PAIR || h == 0)) p.ml[at] = make_float2(m, l);
    }
    // every product and copy has been waited for (or its wait gave up)
    tc::tmem_fence_before();
    __syncthreads();
    tc::tmem_fence_after();
    if (warp == 8)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)S::kCols));
}

// Joins the pieces of a row, a CTA a row: groups of 8 NB threads (four elements
// each) take every kJoin / (8 NB)-th piece, and add up in group order.  slot(s):
// where piece s lies.
constexpr int kJoin = 256;
template <int NB, typename T, class Slot>
__device__ __forceinline__ void join_row(const AttnP& p, int64_t dst, int used, Slot slot) {
    constexpr int per = 8 * NB, groups = kJoin / per;
    __shared__ float4 s_o[groups][per];
    __shared__ float s_l[groups], s_m[kJoin / 32];
    const int tid = threadIdx.x;
    float M = -INFINITY;
    for (int s = tid; s < used; s += kJoin) M = fmaxf(M, p.ml[slot(s)].x);
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
#pragma unroll 4
        for (int s = grp; s < used; s += groups) {
            const int64_t at = slot(s);
            const float2 v = p.ml[at];
            const float4 x = reinterpret_cast<const float4*>(p.part + at * (32 * NB))[e];
            const float f = weight(v.x, M);
            L = fmaf(f, v.y, L);
            acc.x = fmaf(f, x.x, acc.x);
            acc.y = fmaf(f, x.y, acc.y);
            acc.z = fmaf(f, x.z, acc.z);
            acc.w = fmaf(f, x.w, acc.w);
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
        static_cast<T*>(p.out)[dst + tid] = from_f32<T>(l != 0.0f ? sum / l : 0.0f);
    }
}
// Few rows: CTA i R + row joins row `row` of the unit that starts in CTA i.
template <int NB, int R, typename T>
__global__ void __launch_bounds__(kJoin) kv4_join_kernel(const __grid_constant__ AttnP p) {
    pdl_wait();
    const int i = (int)(blockIdx.x / R), row = (int)blockIdx.x - i * R;
    const int4 d = p.desc[i];
    if (d.z < 2) return;
    const Seq q(p, d.x);
    const int row_tiles = (q.n_q * p.group + R - 1) / R, kvh = d.y / row_tiles;
    const int r = (d.y - kvh * row_tiles) * R + row;
    const int64_t tok = (int64_t)q.q0 + r / p.group;
    if (r >= q.n_q * p.group || tok < 0 || tok >= p.n_tokens) return;
    join_row<NB, T>(p, tok * p.ot + (kvh * p.group + r % p.group) * p.oh, d.z,
                    [&](int s) { return (int64_t)(s ? 2 * (i + s) : d.w) * R + row; });
}
// Many rows: the splits of every row.
template <int NB, int R, typename T>
__global__ void __launch_bounds__(kJoin) kv4_join_rows_kernel(const __grid_constant__ AttnP p) {
    pdl_wait();
    const Rows o = unit_rows<R>(p, (int)(blockIdx.x / R));
    const int r = o.r0 + (int)(blockIdx.x % R);
    if (r >= o.rows) return;
    const int64_t tok = (int64_t)o.q0 + r / p.group;
    if (tok < 0 || tok >= p.n_tokens) return;
    int tile0, tile1, per;
    unit_tiles<R>(p, o, tile0, tile1, per);
    const int head = o.kvh * p.group + r % p.group;
    const int64_t at = (tok * p.n_heads + head) * p.splits;
    join_row<NB, T>(p, tok * p.ot + head * p.oh, (tile1 - tile0 + per - 1) / per, [&](int s) { return at + s; });
}

struct Fns {
    const void *main, *join;
};
template <int NB, int MODE, typename T>
Fns fns_of(bool rows, bool pair) {
    constexpr int R = MODE == kOne16 ? 16 : 8;
    if (rows) {
        if constexpr (MODE == kOne16) {
            if (pair)
                return Fns{(const void*)kv4_attn_tc_kernel<NB, true, T>, (const void*)kv4_join_rows_kernel<NB, 2 * kTcRows, T>};
            return Fns{(const void*)kv4_attn_tc_kernel<NB, false, T>, (const void*)kv4_join_rows_kernel<NB, kTcRows, T>};
        } else {
            return Fns{(const void*)kv4_attn_rows_kernel<NB, T>, (const void*)kv4_join_rows_kernel<NB, 2 * R * kWarps, T>};
        }
    }
    return Fns{(const void*)kv4_attn_kernel<NB, MODE, T>, (const void*)kv4_join_kernel<NB, R, T>};
}
template <int NB, typename T>
Fns fns_of(int mode, bool rows, bool pair) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
        if (mode == kOne16) return fns_of<NB, kOne16, T>(rows, pair);
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
        return Fns{(const void*)kv4_attn_kernel<NB, kSplit8, T>, (const void*)kv4_join_kernel<NB, 8, T>};
    else
        return fns_of<NB, kSplit8, T>(rows, pair);
}
template <typename T>
Fns fns_of(int nb, int mode, bool rows, bool pair) {
    switch (nb) {
    case 1: return fns_of<1, T>(mode, rows, pair);
    case 2: return fns_of<2, T>(mode, rows, pair);
    case 3: return fns_of<3, T>(mode, rows, pair);
    default: return fns_of<4, T>(mode, rows, pair);
    }
}
Fns fns_of(int dtype, int nb, int mode, bool rows, bool pair) {
    return dtype == RQ_F32 ? fns_of<float>(nb, mode, rows, pair)
           : dtype == RQ_F16 ? fns_of<__half>(nb, mode, rows, pair)
                             : fns_of<__nv_bfloat16>(nb, mode, rows, pair);
}

struct Plan {
    int mode, R;       // R: rows of a CTA
    bool rows, tc;     // a many-rows form; the one on tcgen05
    bool pair;         // two tiles of rows a CTA there
    int64_t ctas;      // of the main launch
    int row_tiles, splits;  // many rows
    int64_t pieces;    // row sums kept for the join: 0, no join
};

int check_query(const rq_kv4* c, const rq_kv4_query* a, const char* fn) {
    if (!c || !a) return set_error(RQ_ERR_INVALID, "%s: NULL argument", fn);
    if (a->dtype != RQ_F32 && a->dtype != RQ_F16 && a->dtype != RQ_BF16)
        return set_error(RQ_ERR_UNSUPPORTED, "%s: dtype %d (f32 = 0, f16 = 1, bf16 = 2)", fn, a->dtype);
    if (a->n_heads < 1 || a->n_heads > 65536 || a->n_heads % c->n_kv)
        return set_error(RQ_ERR_INVALID, "%s: %lld query heads over %d kv heads", fn, (long long)a->n_heads, c->n_kv);
    if (a->batch < 0 || a->batch > INT32_MAX - 1 || a->n_tokens < 0 || a->n_tokens > INT32_MAX || a->max_q < 1 ||
        a->max_q > kMaxQ || a->table_width < 0 || a->table_width > INT32_MAX || a->max_len < 0 || a->window < 0)
        return set_error(RQ_ERR_INVALID,
                         "%s: batch %lld, n_tokens %lld, max_q %lld, table_width %lld, max_len %lld, window %lld", fn,
                         (long long)a->batch, (long long)a->n_tokens, (long long)a->max_q, (long long)a->table_width,
                         (long long)a->max_len, (long long)a->window);
    if (a->table_width * c->page_size > INT32_MAX)
        return set_error(RQ_ERR_INVALID, "%s: a table of %lld pages passes 2^31 positions", fn, (long long)a->table_width);
    // (in floating point: the product of the largest passes 64 bits)
    if ((double)a->batch * (double)a->n_heads * (double)(a->cu_q ? a->max_q : 1) > (double)INT32_MAX)
        return set_error(RQ_ERR_INVALID, "%s: too many rows for one call: %lld sequences of up to %lld queries of %lld heads", fn,
                         (long long)a->batch, (long long)(a->cu_q ? a->max_q : 1), (long long)a->n_heads);
    if (!a->cu_q && a->n_tokens < a->batch)
        return set_error(RQ_ERR_INVALID, "%s: %lld tokens for %lld sequences of one query each", fn, (long long)a->n_tokens,
                         (long long)a->batch);
    const float scale = a->scale * kLog2e;
    if (scale - scale != 0.0f) return set_error(RQ_ERR_INVALID, "%s: scale is not finite (or passes f32 in base 2)", fn);
    return RQ_OK;
}

Plan make_plan(const rq_kv4* c, const rq_kv4_query* a) {
    Plan pl{};
    const int64_t group = a->n_heads / c->n_kv;
    const int64_t rows = group * (a->cu_q ? a->max_q : 1);
    // f32 needs the two parts, and f16 does too: its own output rounding is no
    // larger than the roundings of one part (errors of 1.4 to 1.8 of the output
    // rounding's alone, where two parts leave 1.0; bf16: 1.02).  Up to eight bf16
    // rows take them as well, since the other half of the operand would be empty.
    pl.mode = a->dtype != RQ_BF16 || rows <= 8 ? kSplit8 : kOne16;
    pl.R = pl.mode == kOne16 ? 16 : 8;
    // Where the many-rows forms win, few rows -> many rows (us, 8 heads a kv head of
    // 8, head_dim 128; other geometries follow the same rule): bf16 at 16 rows,
    // 16 x 2048 keys 43 -> 41, 64 x 1024 74 -> 98, 1 x 40000 45 -> 49; at 24 rows
    // 40 -> 41, 112 -> 98, 63 -> 50; at 128 rows 174 -> 42, 364 -> 104, 192 -> 54.
    // f32 at 32 rows 65 -> 95, 118 -> 151, 68 -> 87; at 48 rows 87 -> 100, 166 -> 153,
    // 91 -> 88; at 64 rows 109 -> 106, 216 -> 158, 129 -> 89; f16 within 5 % of f32.
    // The rows are those that the caller announces (max_q), not those that are there.
    pl.rows = rows > (a->dtype == RQ_BF16 ? 16 : 48);
    const int64_t tiles_of_row = (rows + pl.R - 1) / pl.R;
    int64_t len = a->table_width * c->page_size;
    if (a->max_len > 0) len = std::min(len, a->max_len);
    if (a->window > 0) len = std::min(len, a->window + a->max_q);
    const int64_t tiles = (len + kKv4Tile - 1) / kKv4Tile, sms = c->ctx->sm_count;
    if (!pl.rows) {
        // one wave, but no CTA shorter than a pair a warp at the longest lengths
        const int64_t pairs = a->batch * c->n_kv * tiles_of_row * (std::max<int64_t>((tiles + 1) / 2, 1) + kHead);
        const int64_t places = sms * (c->head_dim > 64 ? kPerSm<4> : kPerSm<2>);
        pl.ctas = std::max<int64_t>(1, std::min(places, pairs / (kWarps + 1)));
        // units of one length (a single sequence's) then begin where CTAs do
        const int64_t units = a->batch * c->n_kv * tiles_of_row;
        if (pl.ctas > units) pl.ctas -= pl.ctas % units;
        pl.pieces = pl.ctas > 1 ? 2 * pl.ctas * pl.R : 0;
        return pl;
    }
    pl.tc = a->dtype == RQ_BF16;
    pl.pair = pl.tc && rows > kTcRows;  // (times: see the kernel)
    pl.R = pl.tc ? (pl.pair ? 2 : 1) * kTcRows : 2 * kWarps * pl.R;
    pl.row_tiles = (int)((rows + pl.R - 1) / pl.R);
    const int64_t units = a->batch * c->n_kv * pl.row_tiles;
    // splits of the long axis where the units leave the device's places (two
    // CTAs an SM) empty, none shorter than two steps
    const int64_t want = sms * (pl.tc ? 1 : 2) / std::max<int64_t>(units, 1);
    pl.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, tiles / (2 * kWarps)));
    pl.ctas = units * pl.splits;
    pl.pieces = pl.splits > 1 ? a->n_tokens * a->n_heads * pl.splits : 0;
    return pl;
}

size_t plan_bytes(const rq_kv4* c, const Plan& pl) {
    return (size_t)pl.pieces * ((size_t)c->head_dim * 4 + 8) + (pl.pieces && !pl.rows ? (size_t)pl.ctas * 16 : 0);
}

}  // namespace

int kv4_attention(const rq_kv4* c, const rq_kv4_query* a, int* err, cudaStream_t st) {
    const Plan pl = make_plan(c, a);
    const size_t need = plan_bytes(c, pl);
    if (need) {
        if (a->workspace_bytes < need)
            return set_error(RQ_ERR_INVALID, "rq_kv4_attention: workspace of %zu bytes, need %zu", a->workspace_bytes, need);
        if (!a->workspace || (uintptr_t)a->workspace & 15) return set_error(RQ_ERR_INVALID, "rq_kv4_attention: workspace is NULL or not 16-byte aligned");
    }
    if (pl.ctas * (pl.rows ? 1 : pl.R) > INT32_MAX || (pl.rows && a->batch * c->n_kv * pl.row_tiles * pl.R > INT32_MAX))
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
    p.wide_out = (((uintptr_t)a->out | (uintptr_t)(p.ot * (int64_t)size) | (uintptr_t)(p.oh * (int64_t)size)) & 15) == 0;
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
    // positions stay below 2^31 and a query is never more than kMaxQ below 0,
    // so a window this long hides nothing and its differences fit 32 bits
    p.window = a->window < (1 << 30) * 2ll - (1 << 25) ? (int)a->window : 0;
    p.scale = a->scale * kLog2e;
    p.part = static_cast<float*>(a->workspace);
    if (need) {
        // sums, then the pairs (descriptions first: they want 16 bytes)
        p.desc = pl.rows ? nullptr : reinterpret_cast<int4*>(p.part + pl.pieces * c->head_dim);
        p.ml = pl.rows ? reinterpret_cast<float2*>(p.part + pl.pieces * c->head_dim) : reinterpret_cast<float2*>(p.desc + pl.ctas);
    }
    p.magic = Magic{kEven, kOdd};
    p.err = err;
    const int nb = c->head_dim / 32;
    constexpr int tc_smem[2][4] = {
        {TcSmem<1, false>::kBytes, TcSmem<2, false>::kBytes, TcSmem<3, false>::kBytes, TcSmem<4, false>::kBytes},
        {TcSmem<1, true>::kBytes, TcSmem<2, true>::kBytes, TcSmem<3, true>::kBytes, TcSmem<4, true>::kBytes}};
    const size_t smem = pl.tc     ? (size_t)tc_smem[pl.pair][nb - 1] + 1024
                        : pl.rows ? (size_t)kWarps * (2048 * nb + 64 * nb + kStagesRows * 576 * nb + 2048 * nb)
                                : (size_t)kWarps * (kStages * 2 * 576 * nb + pl.R * 32 * nb * 4);
    const Fns fn = fns_of(a->dtype, nb, pl.mode, pl.rows, pl.pair);
    if (smem > 32 * 1024) {  // (48 KB without asking, the kernels' static part included)
        const int rc = cuda_error(cudaFuncSetAttribute(fn.main, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                                  "kv4 attention kernel");
        if (rc) return rc;
    }
    void* args[] = {&p};
    const int rc = launch_pdl(fn.main, (unsigned)pl.ctas, (pl.tc ? kTcWarps : kWarps) * 32, smem, st, args, "kv4 attention kernel");
    if (rc || !pl.pieces) return rc;
    const int64_t joins = pl.rows ? a->batch * c->n_kv * pl.row_tiles * pl.R : pl.ctas * pl.R;
    return launch_pdl(fn.join, (unsigned)joins, kJoin, 0, st, args, "kv4 join kernel");
}


}  // namespace rq

using namespace rq;

extern "C" {

int rq_kv4_attention_workspace(const rq_kv4* c, const rq_kv4_query* a, size_t* bytes) {
    if (!bytes) return set_error(RQ_ERR_INVALID, "rq_kv4_attention_workspace: NULL argument");
    int rc = check_query(c, a, "rq_kv4_attention_workspace");
    if (rc) return rc;
    *bytes = plan_bytes(c, make_plan(c, a));
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
    if (!rc) rc = check_rows_apart(a->n_tokens, a->out_stride[0], a->n_heads, a->out_stride[1], c->head_dim, fn_name, "out");
    if (!rc) rc = check_device_ptr(ctx, a->kv_lens, fn_name, "kv_lens");
    if (!rc && a->cu_q) rc = check_device_ptr(ctx, a->cu_q, fn_name, "cu_q");
    if (!rc && a->table_width) rc = check_device_ptr(ctx, a->block_table, fn_name, "block_table");
    if (!rc && a->workspace) rc = check_device_ptr(ctx, a->workspace, fn_name, "workspace");
    return rc ? rc : kv4_attention(c, a, ctx->derr, (cudaStream_t)stream);
}

}  // extern "C"
