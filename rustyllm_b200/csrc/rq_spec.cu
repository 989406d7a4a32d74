// rq_spec.cu -- verification of drafted tokens against the target's
// probabilities from given random numbers: the sampled counterpart of the
// greedy accept of examples/spec_decode_70b.rs:262-283.
//
// Draft x_i is accepted while u_i q_i(x_i) < p_i(x_i); the next token is drawn
// from the leftover w = max(p - q, 0) of the first rejected row (or from p of
// the row after the last draft): the first j with sum_{i<=j} w_i > r * sum w.
// A product of two f32 values is exact in f64, and f64 sums put a border
// between two tokens off by 1e-16 of the mass, so the drawn token does not
// depend on the order of the sum; f32 sums over a large vocabulary would move
// borders by many tokens' mass.
//
// Bound by memory: one row of p and of q per sequence.  A cluster of up to 8
// CTAs takes a sequence; each CTA sums a contiguous share of the row in groups
// of kGroup consecutive elements (one warp a group, 2 x 16 whole lines in
// flight), the CTAs exchange their sums through distributed shared memory, and
// the one whose share holds the target re-reads one group (from L2), 16
// elements a lane, and scans it.  8.4 us for one sequence of four drafts over
// 32000 tokens (four dependent round trips to memory and two cluster barriers),
// 17.4 us for 32 of seven over 128003 (1.9 TB/s of the f32 rows read: 5 us at the
// copy's rate, the round trips before and behind it the rest).
#include <algorithm>

#include "rq_kv4.cuh"

namespace rq {
namespace {

constexpr int kThreads = 512, kWarpsV = kThreads / 32;
constexpr int kPer = 16, kGroup = 32 * kPer;  // elements a warp sums at a time
constexpr int kMaxGroups = 512;               // groups of a CTA's share kept in shared memory

struct VerifyP {
    const void* p;
    const void* q;
    int64_t ps, pr, qs, qr;  // strides: sequence, row
    const int32_t* drafts;
    const int32_t* n_drafts;
    const float* u;
    const float* r;
    int max_drafts;
    int64_t vocab;
    int32_t* tokens;
    int32_t* accepted;
    int ctas;        // CTAs of a sequence
    int per_group;   // kGroup-element runs a group of the sum holds
};

// a probability as a weight: NaN and negatives are none, infinities the largest finite
__device__ __forceinline__ double mass(float x) { return x > 0.0f ? (double)fminf(x, 3.402823466e38f) : 0.0; }

struct Row {  // the weights that the token is drawn from
    const void* p;
    const void* q;  // NULL: none
    int64_t hole;   // element without weight (a certain draft), or -1
};

__device__ __forceinline__ double weight(float p, float q) { return fmax(mass(p) - mass(q), 0.0); }

__device__ __forceinline__ void cluster_arrive_wait() {
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
// the double at the same shared address of the cluster's CTA `rank`
__device__ __forceinline__ double remote(const double* v, int rank) {
    uint32_t a = (uint32_t)__cvta_generic_to_shared(v), b;
    double x;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(a), "r"(rank));
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(x) : "r"(b) : "memory");
    return x;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) spec_verify_kernel(const __grid_constant__ VerifyP p) {
    pdl_wait();
    __shared__ double sums[kMaxGroups];
    __shared__ double total_s;   // this CTA's mass, read by the cluster
    __shared__ int s_acc, s_n;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)(blockIdx.x % p.ctas);
    const int64_t b = blockIdx.x / p.ctas;
    const T* P = static_cast<const T*>(p.p) + b * p.ps;
    const T* Q = p.q ? static_cast<const T*>(p.q) + b * p.qs : nullptr;
    const int32_t* drafts = p.drafts + b * p.max_drafts;
    // ---- accepted drafts (every CTA by itself).  The first 32 drafts and their
    // numbers are loaded beside the count, not behind it.
    if (warp == 0) {
        int32_t x0 = 0;
        float u0 = 0.0f;
        if (lane < p.max_drafts) {
            x0 = drafts[lane];
            u0 = p.u[b * p.max_drafts + lane];
        }
        const int n = p.n_drafts ? min(max(p.n_drafts[b], 0), p.max_drafts) : p.max_drafts;
        int acc = n;
        for (int i0 = 0; i0 < n && acc == n; i0 += 32) {
            const int i = i0 + lane;
            bool good = true;
            if (i < n) {
                const int64_t x = i0 ? drafts[i] : x0;
                good = x >= 0 && x < p.vocab;
                if (good) {
                    const double px = mass(to_f32(P[i * p.pr + x]));
                    const double qx = Q ? mass(to_f32(Q[i * p.qr + x])) : 1.0;
                    good = (double)(i0 ? p.u[b * p.max_drafts + i] : u0) * qx < px;
                }
            }
            const unsigned no = __ballot_sync(0xffffffffu, !good);
            if (no) acc = i0 + __ffs((int)no) - 1;
        }
        if (lane == 0) {
            s_acc = acc;
            s_n = n;
        }
    }
    __syncthreads();
    const int acc = s_acc, n = s_n;
    Row w{P + (int64_t)acc * p.pr, nullptr, -1};
    bool leftover = acc < n;
    if (leftover) {
        if (Q) w.q = Q + (int64_t)acc * p.qr;
        else w.hole = drafts[acc];
    }
    // ---- sums of this CTA's share, group by group
    const int64_t glen = (int64_t)kGroup * p.per_group;
    const int64_t groups = (p.vocab + glen - 1) / glen;
    const int64_t gper = (groups + p.ctas - 1) / p.ctas;
    const int64_t g0 = min(rank * gper, groups), g1 = min(g0 + gper, groups);
    double total, before;
    for (int pass = 0; pass < 2; pass++) {
        for (int64_t g = g0 + warp; g < g1; g += kWarpsV) {
            double a = 0.0;
            for (int64_t j0 = g * glen; j0 < min((g + 1) * glen, p.vocab); j0 += kGroup) {
                float x[kPer], y[kPer];
#pragma unroll
                for (int i = 0; i < kPer; i++) {
                    const int64_t j = j0 + 32 * i + lane;
                    x[i] = j < p.vocab ? to_f32(static_cast<const T*>(w.p)[j]) : 0.0f;
                    y[i] = w.q && j < p.vocab ? to_f32(static_cast<const T*>(w.q)[j]) : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < kPer; i++) a += j0 + 32 * i + lane == w.hole ? 0.0 : weight(x[i], y[i]);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
            if (lane == 0) sums[g - g0] = a;
        }
        __syncthreads();
        if (warp == 0) {
            double a = 0.0;
            for (int64_t i = lane; i < g1 - g0; i += 32) a += sums[i];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
            if (lane == 0) total_s = a;
        }
        __syncthreads();
        total = total_s;
        before = 0.0;
        if (p.ctas > 1) {
            cluster_arrive_wait();
            total = 0.0;
            for (int c = 0; c < p.ctas; c++) {
                if (c == rank) before = total;
                total += remote(&total_s, c);
            }
            cluster_arrive_wait();  // total_s may be written again, or its CTA leave
        }
        if (total > 0.0 || !leftover) break;
        // nothing is left over (p <= q everywhere): draw from p itself
        leftover = false;
        w.q = nullptr;
        w.hole = -1;
    }
    // ---- the token: the CTA, the group and the element whose running sum
    // passes r * total; r below 1 keeps the target below the total, so exactly
    // one CTA's share passes it (all add the shares in the same order)
    const float rb = p.r[b];
    const double target = (double)(rb > 0.0f ? fminf(rb, 0.99999994f) : 0.0f) * total;
    const double mine = total_s;
    int32_t* out = p.tokens + b * (p.max_drafts + 1);
    if (rank == 0) {
        for (int i = tid; i <= p.max_drafts; i += kThreads)
            if (i != acc || !(total > 0.0)) out[i] = i < acc ? drafts[i] : -1;
        if (tid == 0) p.accepted[b] = acc;
    }
    if (!(total > 0.0) || !(mine > 0.0)) return;
    if (!(before <= target) || !(before + mine > target) || warp != 0) return;
    // the group: the lanes scan the sums of 32 groups at a time.  Where
    // rounding lets no group pass, the last with weight.
    int64_t pick = -1, last = -1;
    double run = before, pick_run = before, last_run = before;
    for (int64_t i0 = 0; i0 < g1 - g0 && pick < 0; i0 += 32) {
        const double x = i0 + lane < g1 - g0 ? sums[i0 + lane] : 0.0;
        double s = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += v;
        }
        const unsigned pos = __ballot_sync(0xffffffffu, x > 0.0);
        const unsigned hit = __ballot_sync(0xffffffffu, x > 0.0 && run + s > target);
        const int at = hit ? __ffs((int)hit) - 1 : pos ? 31 - __clz((int)pos) : 0;
        const double upto = run + __shfl_sync(0xffffffffu, s - x, at);
        if (hit) {
            pick = i0 + at;
            pick_run = upto;
        } else if (pos) {
            last = i0 + at;
            last_run = upto;
        }
        run += __shfl_sync(0xffffffffu, s, 31);
    }
    if (pick < 0) {
        pick = last;
        pick_run = last_run;
    }
    // the element: kPer consecutive ones a lane, a scan over the lanes, and the
    // lane that passes goes over its own
    const int64_t e0 = (g0 + pick) * glen, e1 = min(e0 + glen, p.vocab);
    int64_t last_el = -1;
    double upto = pick_run;
    for (int64_t j0 = e0; j0 < e1; j0 += kGroup) {
        double x[kPer], sum = 0.0;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int64_t j = j0 + lane * kPer + i;
            x[i] = 0.0;
            if (j < e1 && j != w.hole)
                x[i] = weight(to_f32(static_cast<const T*>(w.p)[j]), w.q ? to_f32(static_cast<const T*>(w.q)[j]) : 0.0f);
        }
        int mine_last = -1;  // this lane's last element with weight
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            sum += x[i];
            if (x[i] > 0.0) mine_last = i;
        }
        double s = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += v;
        }
        int hit = -1;
        if (mine_last >= 0 && upto + s > target) {
            double r = upto + (s - sum);
            bool found = false;
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                r += x[i];
                if (!found && x[i] > 0.0 && r > target) {
                    found = true;
                    hit = i;
                }
            }
            if (!found) hit = mine_last;  // rounding let no single one pass
        }
        const unsigned who = __ballot_sync(0xffffffffu, hit >= 0);
        if (who) {
            if (lane == __ffs((int)who) - 1) out[acc] = (int32_t)(j0 + lane * kPer + hit);
            return;
        }
        const unsigned some = __ballot_sync(0xffffffffu, mine_last >= 0);
        if (some) {
            const int l = 31 - __clz((int)some);
            last_el = j0 + l * kPer + __shfl_sync(0xffffffffu, mine_last, l);
        }
        upto += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) out[acc] = (int32_t)last_el;  // rounding let none pass: the last with weight
}

}  // namespace
}  // namespace rq

using namespace rq;

extern "C" int rq_spec_verify(rq_ctx* ctx, int dtype, const void* p, const int64_t p_stride[2], const void* q,
                              const int64_t q_stride[2], const int32_t* drafts, const int32_t* n_drafts, const float* u,
                              const float* r, int64_t batch, int64_t max_drafts, int64_t vocab, int32_t* tokens,
                              int32_t* accepted, void* stream) {
    static const char* fn_name = "rq_spec_verify";
    if (!ctx || !p_stride || (q && !q_stride)) return set_error(RQ_ERR_INVALID, "%s: NULL argument", fn_name);
    if (dtype != RQ_F32 && dtype != RQ_F16 && dtype != RQ_BF16)
        return set_error(RQ_ERR_UNSUPPORTED, "%s: dtype %d (f32 = 0, f16 = 1, bf16 = 2)", fn_name, dtype);
    if (batch < 0 || batch > (1 << 24) || max_drafts < 0 || max_drafts > 65536 || vocab < 1 || vocab > (1 << 28))
        return set_error(RQ_ERR_INVALID, "%s: batch %lld, max_drafts %lld (<= 65536), vocab %lld (<= 2^28)", fn_name,
                         (long long)batch, (long long)max_drafts, (long long)vocab);
    if (!batch) return RQ_OK;
    DevGuard g(ctx->device);
    int rc = check_device_ptr(ctx, p, fn_name, "p");
    if (!rc && q && max_drafts) rc = check_device_ptr(ctx, q, fn_name, "q");
    if (!rc && max_drafts) rc = check_device_ptr(ctx, drafts, fn_name, "drafts");
    if (!rc && max_drafts) rc = check_device_ptr(ctx, u, fn_name, "u");
    if (!rc && n_drafts) rc = check_device_ptr(ctx, n_drafts, fn_name, "n_drafts");
    if (!rc) rc = check_device_ptr(ctx, r, fn_name, "r");
    if (!rc) rc = check_device_ptr(ctx, tokens, fn_name, "tokens");
    if (!rc) rc = check_device_ptr(ctx, accepted, fn_name, "accepted");
    if (rc) return rc;
    VerifyP v{};
    v.p = p;
    v.q = max_drafts ? q : nullptr;
    v.ps = p_stride[0];
    v.pr = p_stride[1];
    v.qs = q ? q_stride[0] : 0;
    v.qr = q ? q_stride[1] : 0;
    v.drafts = drafts;
    v.n_drafts = n_drafts;
    v.u = u;
    v.r = r;
    v.max_drafts = (int)max_drafts;
    v.vocab = vocab;
    v.tokens = tokens;
    v.accepted = accepted;
    v.ctas = 1;
    while (v.ctas < 8 && (int64_t)v.ctas * kGroup * kWarpsV < vocab) v.ctas *= 2;
    v.per_group = (int)((vocab + (int64_t)kGroup * kMaxGroups * v.ctas - 1) / ((int64_t)kGroup * kMaxGroups * v.ctas));
    const void* fn = dtype == RQ_F32 ? (const void*)spec_verify_kernel<float>
                     : dtype == RQ_F16 ? (const void*)spec_verify_kernel<__half>
                                       : (const void*)spec_verify_kernel<__nv_bfloat16>;
    void* args[] = {&v};
    return launch_pdl(fn, (unsigned)(batch * v.ctas), kThreads, 0, (cudaStream_t)stream, args, "draft verification kernel",
                      (unsigned)v.ctas);
}
