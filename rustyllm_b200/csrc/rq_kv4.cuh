// rq_kv4.cuh -- the paged key/value cache held in 4 bits: layout, rounding and
// the helpers that its kernels (append, read, attention) share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "rq_internal.cuh"

// A block is 32 consecutive elements of one head's row: an f16 scale d and 32
// codes, value = (code - 8) * d.  The cache is [page][kv head][tile], a tile
// being 16 consecutive positions of one head, so a tile is one contiguous
// record of 576 * NB bytes (NB = head_dim / 32) that one bulk copy brings in:
//   K codes 256 NB | V codes 256 NB | K scales 32 NB | V scales 32 NB
// Codes lie in the order in which the lanes of a warp feed them to
// mma.m16n8k16 (lane = 4 g + t), so attention reads them with 16-byte
// conflict-free loads and turns them into f16 operands without a shuffle:
//   K  lane (g, t), word 2 b + n: the 8 elements 32 b + 8 t .. + 7 of token
//      4 (g / 2) + (g % 2) + 2 n (column g of score tile n); element 2 i + h
//      in nibble i + 4 h, so a 16-bit lane mask yields two neighbours.
//   V  lane (g, t), word 2 b + p: tokens 4 t + 2 p (low half) and 4 t + 2 p + 1
//      (high half); nibble k of a half is element 32 b + 8 k + g.
//   scales: [token / 4][b][token % 4] f16.
// A token's K words and V halves are its own: an append writes no byte that
// holds another token's codes.
struct rq_kv4 {
    rq_ctx* ctx;
    uint8_t* data;
    int64_t n_pages;
    int page_size, n_kv, head_dim;
    size_t bytes;
};

namespace rq {

constexpr int kKv4Tile = 16;  // positions of a tile

template <int NB>
struct Kv4Rec {
    static constexpr int kCodes = 256 * NB;  // bytes of one code region
    static constexpr int kV = kCodes, kKs = 2 * kCodes, kVs = kKs + 32 * NB;
    static constexpr int kBytes = 576 * NB;
};

// Byte of word w (0 .. 2 NB - 1) of `lane` inside a code region: planes of
// four words a lane (16 bytes), then one of two where 2 NB is not a multiple
// of four.
__host__ __device__ __forceinline__ int kv4_word(int nb, int lane, int w) {
    const int full = nb >> 1;  // planes of four words
    return (w >> 2) < full ? (w >> 2) * 512 + lane * 16 + (w & 3) * 4 : full * 512 + lane * 8 + (w & 3) * 4;
}
__host__ __device__ __forceinline__ int kv4_scale(int nb, int tok, int b) {
    return 2 * ((tok >> 2) * 4 * nb + b * 4 + (tok & 3));
}
// K: token and the group t of 8 elements inside block b -> lane and word
__host__ __device__ __forceinline__ int kv4_k_at(int nb, int tok, int b, int t) {
    const int g = 2 * (tok >> 2) + (tok & 1);
    return kv4_word(nb, g * 4 + t, 2 * b + ((tok >> 1) & 1));
}
// V: the 16-bit item of token tok, block b, column g
__host__ __device__ __forceinline__ int kv4_v_at(int nb, int tok, int b, int g) {
    return kv4_word(nb, g * 4 + (tok >> 2), 2 * b + ((tok >> 1) & 1)) + 2 * (tok & 1);
}

// The record of (slot, head); NULL for a slot outside the cache.
__device__ __forceinline__ uint8_t* kv4_record(uint8_t* data, int64_t n_slots, int page_size, int n_kv, int rec_bytes,
                                               int32_t slot, int head) {
    if (slot < 0 || slot >= n_slots) return nullptr;
    const int page = (int)((unsigned)slot / (unsigned)page_size), off = slot - page * page_size;
    return data + (((int64_t)page * n_kv + head) * (page_size / kKv4Tile) + off / kKv4Tile) * rec_bytes;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

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
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 x, y, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 w, x, y;\n mov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// 8 consecutive elements as f32; `wide`: p is 16-byte aligned
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, bool wide, float (&x)[8]) {
    if (wide) {
        T tmp[8];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++)
            reinterpret_cast<uint4*>(tmp)[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_f32(tmp[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_f32(p[i]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, bool wide, const float (&x)[8]) {
    if (wide) {
        T tmp[8];
#pragma unroll
        for (int i = 0; i < 8; i++) tmp[i] = from_f32<T>(x[i]);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++)
            reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(tmp)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = from_f32<T>(x[i]);
    }
}

__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN wins
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float c;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}

// The four lanes of an aligned group hold a block, 8 elements each.  Returns
// the block's scale (f16 value in f32) and this lane's 8 codes.  d = f16(m /
// -8), m the element of the largest magnitude (the lowest index of equals); m /
// 8 is exact, so d is one rounding.  A code is the nearest multiple of d (ties
// to the higher code): k = rint(x / d) by an approximate quotient is off by one
// at most, and what is left, r = x - k d (k d has at most 15 bits), compares with
// d / 2 exactly, whatever the quotient's rounding.  A NaN makes the scale NaN
// (the block reads back as NaN); infinities saturate it at 65504.
__device__ __forceinline__ float kv4_quantize(const float (&x)[8], uint32_t (&c)[8]) {
    float top = x[0], low = x[0];
#pragma unroll
    for (int i = 1; i < 8; i++) {
        top = max_nan(top, x[i]);
        low = min_nan(low, x[i]);
    }
    const unsigned lane = threadIdx.x & 31;
    const unsigned group = 0xFu << (lane & 28);
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
        top = max_nan(top, __shfl_xor_sync(group, top, o));
        low = min_nan(low, __shfl_xor_sync(group, low, o));
    }
    float m = top > -low ? top : low;
    if (top == -low) {  // both signs reach it: the first element decides
        int first = 8;  // 2 * index + (negative)
#pragma unroll
        for (int i = 7; i >= 0; i--)
            if (fabsf(x[i]) == top) first = 2 * i + (x[i] < 0.0f ? 1 : 0);
        bool here = false;
#pragma unroll
        for (int i = 0; i < 8; i++) here |= fabsf(x[i]) == top;
        const unsigned who = __ballot_sync(group, here) & group;
        if (__shfl_sync(group, first, who ? __ffs((int)who) - 1 : (int)lane) & 1) m = low;
        else m = top;
    }
    const float d = __half2float(__float2half_rn(fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f)));
    if (!(top == top) || d == 0.0f) {
#pragma unroll
        for (int i = 0; i < 8; i++) c[i] = 8;
        return top == top ? d : __int_as_float(0x7fffffff);
    }
    // with the sign of d taken into x
    const uint32_t sign = __float_as_uint(d) & 0x80000000u;
    const float D = fabsf(d), inv = __frcp_rn(D), half = 0.5f * D;
    constexpr int kMid = 0x4B400000;  // 12582912.0f
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float v = __uint_as_float(__float_as_uint(x[i]) ^ sign);
        const float z = fmaf(v, inv, 12582912.0f);  // 1.5 * 2^23: an integer in the low bits
        const float r = fmaf(12582912.0f - z, D, v);
        int k = __float_as_int(z);  // kMid + the multiple, and in the order of z elsewhere (a negative z is a negative k)
        if (r >= half) k++;
        if (r < -half) k--;
        c[i] = (uint32_t)(min(max(k, kMid - 8), kMid + 7) - (kMid - 8));
    }
    return d;
}

// Writes one lane's share of a token's block: x holds elements 32 b + 8 t ..
// + 7 (t = lane % 4; the aligned four lanes hold the block).  rec NULL: the
// lane takes part in the group's exchange and writes nothing.
__device__ __forceinline__ void kv4_store(uint8_t* rec, int nb, int tok, int b, bool is_v, const float (&x)[8]) {
    uint32_t c[8];
    const float d = kv4_quantize(x, c);
    const unsigned lane = threadIdx.x & 31, t = lane & 3;
    const unsigned group = 0xFu << (lane & 28);
    uint8_t* codes = rec + (is_v ? 256 * nb : 0);
    if (!is_v) {
        uint32_t w = 0;  // element 2 i + h in nibble i + 4 h
#pragma unroll
        for (int i = 0; i < 8; i++) w |= c[i] << (4 * ((i >> 1) + 4 * (i & 1)));
        if (rec) *reinterpret_cast<uint32_t*>(codes + kv4_k_at(nb, tok, b, (int)t)) = w;
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) w |= c[i] << (4 * i);
        // element 8 k + g of lane k goes to nibble k of item g: lane t writes
        // items 2 t and 2 t + 1, bytes t of the four words
        uint32_t a = 0, e = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t o = __shfl_sync(group, w, (int)((lane & 28) + k)) >> (8 * t);
            a |= (o & 15u) << (4 * k);
            e |= ((o >> 4) & 15u) << (4 * k);
        }
        if (rec) {
            *reinterpret_cast<uint16_t*>(codes + kv4_v_at(nb, tok, b, (int)(2 * t))) = (uint16_t)a;
            *reinterpret_cast<uint16_t*>(codes + kv4_v_at(nb, tok, b, (int)(2 * t + 1))) = (uint16_t)e;
        }
    }
    if (rec && t == 0)
        *reinterpret_cast<__half*>(rec + 512 * nb + (is_v ? 32 * nb : 0) + kv4_scale(nb, tok, b)) = __float2half_rn(d);
}

// The inverse: this lane's 8 values of a token's block.
__device__ __forceinline__ void kv4_load(const uint8_t* rec, int nb, int tok, int b, bool is_v, float (&x)[8]) {
    const unsigned lane = threadIdx.x & 31, t = lane & 3;
    const unsigned group = 0xFu << (lane & 28);
    float d = 0.0f;
    if (rec) d = __half2float(*reinterpret_cast<const __half*>(rec + 512 * nb + (is_v ? 32 * nb : 0) + kv4_scale(nb, tok, b)));
    if (!is_v) {
        const uint32_t w = rec ? *reinterpret_cast<const uint32_t*>(rec + kv4_k_at(nb, tok, b, (int)t)) : 0;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = ((float)((w >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15u) - 8.0f) * d;
    } else {
        uint32_t w = 0;
        uint32_t items = 0;
        if (rec)
            items = *reinterpret_cast<const uint16_t*>(rec + 256 * nb + kv4_v_at(nb, tok, b, (int)(2 * t))) |
                    ((uint32_t)*reinterpret_cast<const uint16_t*>(rec + 256 * nb + kv4_v_at(nb, tok, b, (int)(2 * t + 1))) << 16);
#pragma unroll
        for (int k = 0; k < 4; k++) {  // items 2 k, 2 k + 1 of lane k: its nibble t is this lane's elements 2 k, 2 k + 1
            const uint32_t o = __shfl_sync(group, items, (int)((lane & 28) + k));
            w |= ((o >> (4 * t)) & 15u) << (8 * k);
            w |= ((o >> (16 + 4 * t)) & 15u) << (8 * k + 4);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = ((float)((w >> (4 * i)) & 15u) - 8.0f) * d;
    }
}

// shared host helpers of the paged operators (rq_kv4.cu)
struct DevGuard {  // the context's device for the duration of a call
    int prev = -1;
    explicit DevGuard(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev) cudaSetDevice(dev);
    }
    ~DevGuard() {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
    }
};
// RQ_OK when p is device memory on ctx's device, else an error that names it
int check_device_ptr(const rq_ctx* ctx, const void* p, const char* fn, const char* name);
// RQ_OK when no two rows of an output [n0][n1] (strides s0, s1, rows of len
// contiguous elements) share an element
int check_rows_apart(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t len, const char* fn, const char* name);
// a launch that may begin while the previous kernel of the stream drains
// (the kernel waits with griddepcontrol.wait before it touches memory);
// cluster > 1: thread-block clusters of that many CTAs along x
int launch_pdl(const void* fn, unsigned grid, unsigned block, size_t smem, cudaStream_t st, void** args, const char* what,
               unsigned cluster = 1);

// The operators for callers inside the library that know their pointers
// (rq_llama.cu): no checks of memory kinds, the device already current, a
// bounded wait that gives up reported in *err.
int kv4_attention(const rq_kv4* c, const rq_kv4_query* a, int* err, cudaStream_t st);
int qk_norm_rope(const rq_ctx* ctx, const rq_qk_rope* a, cudaStream_t st);
int qk_norm_rope_append(const rq_kv4* c, const rq_qk_rope* a, const void* v, const int64_t v_stride[2], const int32_t* slots,
                        cudaStream_t st);
int pages_extend(int64_t batch, int page_size, const int32_t* ctx_lens, const int32_t* new_lens, int32_t* table,
                 int64_t table_stride, int64_t table_width, const int32_t* ring, int64_t n_pages, const int32_t* state_in,
                 int32_t* state_out, int32_t* kv_lens, int32_t* cu_new, int32_t* positions, int32_t* slots, int64_t n_tokens,
                 cudaStream_t st);
int pages_release(int64_t batch, int page_size, const int32_t* held_lens, const int32_t* keep_lens, int32_t* table,
                  int64_t table_stride, int64_t table_width, int32_t* ring, int64_t n_pages, int32_t* state, cudaStream_t st);

__device__ __forceinline__ void pdl_wait() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
}

}  // namespace rq
