// Losses of preference and policy tuning over rows of logits: target log-probabilities and their
// gradient, the paired log-ratio loss over sequences, and the clipped policy loss with a KL term
// with its gradient in the same pass.
//
// Per row: lse = M + log(sum_j exp(x_j - M)), logp = x_t - M - log(sum); the gradient of anything that
// depends on the row through logp is dlogits_j = g ([j == t] - exp(x_j - M) / sum). Statistics are fp32.
// The exponent is fma(x, log2(e), -B) with B = M log2(e) rounded; what the rounding of B left out,
// r = fma(M, log2(e), -B), is the same for every x and is taken out of the sum by one factor 2^-r: left
// in, it would reach logp with an error that grows with |M|. Beyond |M| = 2^20, where r itself grows (rows
// masked with the type's lowest value are there), the exponent is (x - M) * log2(e).
#include <algorithm>
#include <type_traits>

#include "pk_common.cuh"
#include "pk_tc.cuh"

namespace pk {
namespace {

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The kernels of this file are launched while their predecessor on the stream still runs, and wait for it here
// before they touch memory: the cost of a launch is then behind them. None of their parameters is __restrict__: that
// would allow loads that are defined only for data that nobody writes while the kernel lives, and the predecessor does.
// The three calls of a paired loss over 32000 words in bf16, 8192 rows: 224 -> 218 us; 2 x 40 rows, called from Python,
// 25 -> 23, and replayed from a graph, where a launch costs little, 9.6 -> 10.7.
__device__ __forceinline__ void after_predecessor() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Running maximum and sum of exponentials of a thread's or a row's values. An empty one has m = -inf and s = 0, and
// so has a row of nothing but -inf. Merging scales by expf: ex2.approx is 5.5e-8 low on the average, which would enter
// once per merge and add up over a sequence's rows (mean error of logp over 4000 x 32000: 7e-9, with ex2 36e-9).
struct __align__(8) Stat {
    float m, s;
};
__device__ __forceinline__ float stat_base(float m) { return m == -INFINITY ? 0.0f : m; }  // no inf - inf below
__device__ __forceinline__ Stat merge(Stat a, Stat b) {
    const float m = fmaxf(a.m, b.m), base = stat_base(m);
    return {m, a.s * expf(a.m - base) + b.s * expf(b.m - base)};
}
// Exponentials against a maximum m: of(x) = exp(x - m) * 2^r.
struct Base {
    float m, nb, r;
    bool plain;  // |m| small enough for the fused form
    __device__ __forceinline__ explicit Base(float top) {
        m = stat_base(top);
        plain = fabsf(m) < 1048576.0f;
        nb = -__fmul_rn(m, LOG2E);
        r = plain ? __fmaf_rn(m, LOG2E, nb) : 0.0f;
    }
    template <bool PLAIN> __device__ __forceinline__ float of(float x) const {
        return PLAIN ? ex2(__fmaf_rn(x, LOG2E, nb)) : ex2((x - m) * LOG2E);
    }
    // two at a time: the same bits
    template <bool PLAIN> __device__ __forceinline__ uint64_t of2(uint64_t x) const {
        const uint64_t c = tc::f2_pack(LOG2E, LOG2E);
        const uint64_t y = PLAIN ? tc::f2_fma(x, c, tc::f2_pack(nb, nb)) : tc::f2_mul(tc::f2_add(x, tc::f2_pack(-m, -m)), c);
        float lo, hi;
        tc::f2_unpack(y, lo, hi);
        return tc::f2_pack(ex2(lo), ex2(hi));
    }
};

// A row of V values that may start anywhere: `head` values up to the first 16-byte boundary, nv
// vectors, and a tail.
template <typename T> struct RowSplit {
    int64_t head, nv, tail0;
    __device__ __forceinline__ RowSplit(const T* row, int64_t V) {
        constexpr int N = Vec<T>::N;
        const int to = (-static_cast<int>(reinterpret_cast<uintptr_t>(row) / sizeof(T))) & (N - 1);
        head = to < V ? to : V;
        nv = (V - head) >> (N == 8 ? 3 : 2);
        tail0 = head + nv * N;
    }
};

// dx[j] = g [j == t] - k exp(x_j - base): `threads` threads, of which this is `tid`, write one row. x and dx may be
// the same row; they are read and written by the same thread, element by element or vector by vector.
template <typename T>
__device__ __forceinline__ void row_grad(const T* x, T* dx, int64_t V, int64_t t, float base, float k, float g, int64_t tid, int64_t threads) {
    constexpr int N = Vec<T>::N;
    const RowSplit<T> sp(x, V);
    const bool wide = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15u) == 0;
    if (wide) {
        const T* body = x + sp.head;
        T* out = dx + sp.head;
        for (int64_t i = tid; i < sp.nv; i += threads) {
            float f[N];
            Vec<T>::load(body + i * N, f);
            const int64_t te = t - sp.head - i * N;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                f[e] = ex2((f[e] - base) * LOG2E) * -k;
                if (te == e) f[e] += g;
            }
            Vec<T>::store(out + i * N, f);
        }
    }
    const int64_t edge = wide ? sp.head + V - sp.tail0 : V;  // elements outside the vectors
    for (int64_t i = tid; i < edge; i += threads) {
        const int64_t c = !wide || i < sp.head ? i : sp.tail0 + i - sp.head;
        float f = ex2((to_f32(x[c]) - base) * LOG2E) * -k;
        if (c == t) f += g;
        dx[c] = from_f32<T>(f);
    }
}
template <typename T>
__device__ __forceinline__ void row_zero(T* dx, int64_t V, int64_t tid, int64_t threads) {
    constexpr int N = Vec<T>::N;
    const RowSplit<T> sp(dx, V);
    for (int64_t i = tid; i < sp.nv; i += threads) *reinterpret_cast<uint4*>(dx + sp.head + i * N) = make_uint4(0, 0, 0, 0);
    for (int64_t c = tid; c < sp.head; c += threads) dx[c] = from_f32<T>(0.0f);
    for (int64_t c = sp.tail0 + tid; c < V; c += threads) dx[c] = from_f32<T>(0.0f);
}

// x - (m + log(s)) and m + log(s), each as if rounded once: log(s) = k log(2) + log(f) with f in [sqrt(1/2), sqrt(2)),
// k times the upper bits of log(2) is exact, and what the sums round off is carried along. A logarithm of fp32
// taken whole rounds at its own size, and its sum with m once more; a KL term of two close policies feels both.
constexpr float LN2_HI = 11355.0f / 16384, LN2_LO = 9.2981341195e-5f;
__device__ __forceinline__ float sum2(float a, float b, float& left) {  // a + b, and what its rounding left out (Knuth's two-sum)
    const float c = __fadd_rn(a, b), t = __fsub_rn(c, a);
    left += __fadd_rn(__fsub_rn(a, __fsub_rn(c, t)), __fsub_rn(b, t));
    return c;
}
struct LogSum {
    float m, k, rest, whole;
    bool fine;
    __device__ __forceinline__ explicit LogSum(const Stat& st) : m(st.m) {
        fine = fabsf(st.m) < 1e30f && st.s > 1e-30f && st.s < 1e30f;
        const int e = (__float_as_int(st.s) - __float_as_int(0.70710678f)) >> 23;
        k = static_cast<float>(e);
        const float l = logf(fine ? __int_as_float(__float_as_int(st.s) - (e << 23)) : st.s);
        rest = __fmaf_rn(k, LN2_LO, l);
        whole = l;
    }
    __device__ __forceinline__ float lse() const {
        if (!fine) return m + whole;
        float left = rest;
        const float a = sum2(m, k * LN2_HI, left);
        return a + left;
    }
    __device__ __forceinline__ float logp(float x) const {
        if (!fine || !(fabsf(x) < 1e30f)) return x - m - (fine ? k * LN2_HI + rest : whole);
        float left = -rest;
        const float a = sum2(x, -m, left), b = sum2(a, -k * LN2_HI, left);
        return b + left;
    }
};

// The same for a row whose lse has few bits behind the point. exp(x - lse) is off by the rounding of lse, |lse| 2^-24
// (by a factor of V in a row of the type's lowest value alone), so maximum and sum are found again from the row, and
// serve where the lse is theirs (one over more words than the row holds is taken as it is). A block reads all of the row
// before it writes any, so one block has it to itself. From 64 on for fp32 (below, at most 2^-18, what an exponential
// may be off), from 1024 for bf16 (2^-14, against its own rounding of 2^-9); ordinary rows never come here.
template <typename T>
__device__ __noinline__ void row_grad_large(const T* x, T* dx, int64_t V, int64_t t, float lse, float g) {
    __shared__ float red[32];
    if (blockIdx.y != 0) return;
    constexpr int N = Vec<T>::N;
    const RowSplit<T> sp(x, V);
    const int tid = threadIdx.x, threads = blockDim.x;
    const int64_t edge = sp.head + V - sp.tail0;
    float m = -INFINITY, s = 0.0f;
    for (int64_t i = tid; i < sp.nv; i += threads) {
        float f[N];
        Vec<T>::load(x + sp.head + i * N, f);
#pragma unroll
        for (int e = 0; e < N; ++e) m = fmaxf(m, f[e]);
    }
    for (int64_t i = tid; i < edge; i += threads) m = fmaxf(m, to_f32(x[i < sp.head ? i : sp.tail0 + i - sp.head]));
    m = block_max(m, red);
    for (int64_t i = tid; i < sp.nv; i += threads) {
        float f[N], part = 0.0f;
        Vec<T>::load(x + sp.head + i * N, f);
#pragma unroll
        for (int e = 0; e < N; ++e) part += expf(f[e] - m);
        s += part;
    }
    for (int64_t i = tid; i < edge; i += threads) s += expf(to_f32(x[i < sp.head ? i : sp.tail0 + i - sp.head]) - m);
    s = block_sum(s, red);
    const float own = LogSum({m, s}).lse();
    const bool mine = fabsf(own - lse) <= fminf(fabsf(lse) * 0x1p-22f, 1e38f);  // two to four steps of fp32; not an infinite one
    row_grad(x, dx, V, t, mine ? m : lse, mine ? g / s : g, g, tid, threads);
    __syncthreads();  // red is free for the block's next such row
}

template <typename T>
__global__ void __launch_bounds__(512, 4)  // 32 registers at most: large rows must not cost the others their residency
token_logprob_bwd_kernel(const T* logits, int64_t ld, const int32_t* targets, const float* lse,
                         const float* dlogp, T* dlogits, int64_t ldd, int64_t R, int64_t V, int32_t* status) {
    // gridDim.y blocks share a row. Last rows first: the pass that took the log-probabilities has left them in L2.
    const int64_t tid = blockIdx.y * blockDim.x + threadIdx.x, threads = gridDim.y * blockDim.x;
    after_predecessor();
    for (int64_t row = R - 1 - blockIdx.x; row >= 0; row -= gridDim.x) {
        float g = dlogp[row];
        T* dx = dlogits + row * ldd;
        if (g != 0.0f) {
            const int64_t t = targets[row];
            if (t >= 0 && t < V) {
                const float l = lse[row];
                if (fabsf(l) >= (sizeof(T) == 2 ? 1024.0f : 64.0f)) row_grad_large(logits + row * ld, dx, V, t, l, g);
                else row_grad(logits + row * ld, dx, V, t, l, g, g, tid, threads);
                continue;
            }
            if (tid == 0 && status) atomicOr(status, PK_ERR_INDEX);
        }
        row_zero(dx, V, tid, threads);
    }
}

struct PolicyArgs {
    const int32_t* targets;
    const float *old_logp, *ref_logp, *advantage, *weight;
    float lo, hi, kl_coef, gscale;  // lo = 1 - clip_lo, hi = 1 + clip_hi
    float *row_loss, *logp, *kl;
    int32_t* status;
};

// e^u - u - 1 without the cancellation near zero: its series there (the next term is below 2^-24 of
// the first for |u| < 0.1), expm1 elsewhere, alone where u is below its last bit (and may be infinite).
__device__ __forceinline__ float kl_term(float u) {
    if (fabsf(u) < 0.1f)
        return u * u * (0.5f + u * (1.0f / 6 + u * (1.0f / 24 + u * (1.0f / 120 + u * (1.0f / 720 + u * (1.0f / 5040))))));
    return u > 64.0f ? expm1f(u) : expm1f(u) - u;
}
// What the loss takes from a row besides its logits: fetched before the row's reduction, so that the
// fetch does not stand behind it.
struct PolicyRow {
    float adv, old, ref, w;
    __device__ __forceinline__ void load(const PolicyArgs& a, int64_t row) {
        adv = a.advantage[row];
        old = a.old_logp ? a.old_logp[row] : 0.0f;
        ref = a.ref_logp ? a.ref_logp[row] : 0.0f;
        w = a.weight ? a.weight[row] : 1.0f;
    }
};
// d loss / d logp of a row, for every thread that asks; one of them writes the row's loss.
__device__ __forceinline__ float policy_row(const PolicyArgs& a, int64_t row, const PolicyRow& q, float logp, bool writer) {
    float r = a.old_logp ? expf(logp - q.old) : (logp == logp ? 1.0f : logp);
    if (q.adv == 0.0f && r == INFINITY) r = 1.0f;  // a ratio past the type's range counts for nothing all the same
    const float free_ = r * q.adv, held = fminf(fmaxf(r, a.lo), a.hi) * q.adv;
    float loss = -held, g = 0.0f, kl = 0.0f;
    if (free_ <= held) loss = g = -free_;
    if (free_ != free_) loss = g = free_;
    if (a.ref_logp) {
        const float u = q.ref - logp;
        kl = kl_term(u);
        if (a.kl_coef != 0.0f) {  // without it e^u may be infinite
            loss += a.kl_coef * kl;
            g -= a.kl_coef * expm1f(u);
        }
    }
    if (writer) {
        a.row_loss[row] = q.w * loss;
        if (a.logp) a.logp[row] = logp;
        if (a.kl) a.kl[row] = kl;
    }
    return q.w * g * a.gscale;
}
__device__ __forceinline__ void policy_row_out(const PolicyArgs& a, int64_t row) {
    a.row_loss[row] = 0.0f;
    if (a.logp) a.logp[row] = 0.0f;
    if (a.kl) a.kl[row] = 0.0f;
}

// ---- losses and log-probabilities, a row per warp, CTA or cluster ---------------------------------
struct RowArgs {
    const void* logits;
    void* dlogits;       // null: no gradient
    int64_t ld, ldd, R, V;
    PolicyArgs p;        // policy; of it, targets, weight, logp and status for log-probabilities
    float* lse;          // log-probabilities
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_store(uint32_t addr, uint32_t rank, Stat v) {
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\tst.shared::cluster.v2.f32 [a], {%2, %3};\n\t}"
                 ::"r"(addr), "r"(rank), "f"(v.m), "f"(v.s) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Statistics over the lanes of a warp, the same bits in every lane.
__device__ __forceinline__ Stat warp_stat(Stat st) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(st.m));
    return {m, warp_sum(st.s * expf(st.m - stat_base(m)))};
}

// The values of a 16-byte vector as packed fp32 pairs: (0, 1), (2, 3), ...
__device__ __forceinline__ void unpack2(const uint4& v, uint64_t (&p)[4]) {  // bf16
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = tc::f2_pack_bits(w[i] << 16, w[i] & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(const uint4& v, uint64_t (&p)[2]) {  // fp32
    p[0] = tc::f2_pack_bits(v.x, v.y);
    p[1] = tc::f2_pack_bits(v.z, v.w);
}
template <typename T> struct RowVec;  // maximum over 16-byte vectors
template <> struct RowVec<bf16> {
    static constexpr int N = 8;
    __nv_bfloat162 m = __halves2bfloat162(__ushort_as_bfloat16(0xff80), __ushort_as_bfloat16(0xff80));  // -inf
    __device__ __forceinline__ void add(const uint4& v) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __hmax2(m, *reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    }
    __device__ __forceinline__ float top(float with) const { return fmaxf(with, fmaxf(__low2float(m), __high2float(m))); }
};
template <> struct RowVec<float> {
    static constexpr int N = 4;
    float m = -INFINITY;
    __device__ __forceinline__ void add(const uint4& v) {
        m = tc::fmax3(m, __uint_as_float(v.x), __uint_as_float(v.y));
        m = tc::fmax3(m, __uint_as_float(v.z), __uint_as_float(v.w));
    }
    __device__ __forceinline__ float top(float with) const { return fmaxf(with, m); }
};

__device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A row belongs to a warp (THREADS = 32, four rows to a CTA), a CTA, or a cluster of 2 to 8 CTAs with a
// stretch of it each. A thread holds K vectors in flight and a running sum of exponentials against its
// running maximum. (A reference that follows the maximum only when that has moved by 8 saves no time, and
// costs the large terms' exponents a rounding at 2^-21.) With a gradient the stretch is read once more,
// backwards: what was read last is still in L1, and the stretches of all resident CTAs are in L2, so DRAM sees the
// logits once. Nothing orders the rows: the chain from a row's last byte over its reductions to its scalars is
// hidden by what else is resident.
//
// Bound by memory and its latency. Policy loss with its gradient, bf16: 8192 x 32000 185 - 189 us from card to card, 5.6
// TB/s (second reading forwards 195), 60000 x 4000 168 us, 5.7 TB/s, 8192 x 151936 930 - 1010 us, 5.2 TB/s, where the
// second reading is no cause: DRAM moves 931 MB of the 934 that 1536 such rows and their gradient have, and 833 of 817
// with a quarter of dead rows. A row that stays in the registers or the shared memory of its CTAs while the next one is
// on its way with cp.async took 207 at the first size and 385 at the second (kept: 189 and 168 on that card): its warps
// wait for one another between the rows. Holding a part of the stretch in shared memory for the second reading costs
// L1 as much as it saves (190; five CTAs per SM). Without a gradient:
// 8192 x 50257 150 us, 5.5 TB/s.
constexpr int CLUSTER_MOST = 8, SWEEP_K = 4;
constexpr int64_t ROWS_MOST = 0x7fffffff / CLUSTER_MOST;  // of a call with one grid for all rows
template <bool GRAD, int THREADS> struct Sweep {
    static constexpr int CTA = THREADS < 128 ? 128 : THREADS;  // threads of a CTA
    static constexpr int PER_SM = GRAD ? (CTA == 128 ? 10 : 6) : 2048 / CTA;
};

// The second reading is the last, and nobody reads the gradient before the kernel's end: both are marked to leave L2
// first, so that they do not push out stretches that have yet to be read again (8192 x 32000 bf16 209 -> 189 us).
__device__ __forceinline__ uint4 load_last(const void* p) { return __ldcs(static_cast<const uint4*>(p)); }

template <typename T, bool POLICY, bool GRAD, int THREADS>
__global__ void __launch_bounds__((Sweep<GRAD, THREADS>::CTA), (Sweep<GRAD, THREADS>::PER_SM))
sweep_kernel(const RowArgs a) {
    constexpr bool WARP = THREADS == 32;  // a warp per row, four to a CTA, no barrier
    constexpr int N = RowVec<T>::N, K = SWEEP_K, NW = THREADS / 32;
    __shared__ Stat boxes[CLUSTER_MOST * NW];
    __shared__ float4 result;  // maximum, factor of the exponentials, gradient at the target, 1 when there is any
    __shared__ int64_t target;
    const int tid = threadIdx.x % THREADS, lane = tid & 31, warp = tid >> 5;
    const int C = WARP ? 1 : static_cast<int>(cluster_size()), rank = WARP ? 0 : static_cast<int>(cluster_rank());
    const int64_t r = WARP ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x / static_cast<unsigned>(C);
    after_predecessor();
    if (WARP && r >= a.R) return;
    const bool writer = rank == 0 && tid == 0;
    T* dx = GRAD ? static_cast<T*>(a.dlogits) + r * a.ldd : nullptr;
    if (a.p.weight != nullptr && a.p.weight[r] == 0.0f) {  // the whole cluster
        if (writer) {
            if constexpr (POLICY) {
                policy_row_out(a.p, r);
            } else {
                a.lse[r] = 0.0f;
                a.p.logp[r] = 0.0f;
            }
        }
        if constexpr (GRAD) row_zero(dx, a.V, rank * THREADS + tid, C * THREADS);
        return;
    }
    if (C > 1) cluster_arrive();  // nobody writes to a CTA's boxes before it runs
    const T* x = static_cast<const T*>(a.logits) + r * a.ld;
    const RowSplit<T> sp(x, a.V);
    int64_t t = 0;
    bool ok = false;
    float xt = 0.0f;
    PolicyRow q;
    if (tid == 0 && (GRAD || rank == 0)) {  // read before any CTA of the row may write a gradient over it
        t = a.p.targets[r];
        ok = t >= 0 && t < a.V;
        if constexpr (POLICY) q.load(a.p, r);
        if (ok) xt = to_f32(x[t]);
    }
    // the elements before the first and behind the last vector belong to the first threads
    int64_t edge_at = -1;
    if (rank == 0 && tid < sp.head + a.V - sp.tail0) edge_at = tid < sp.head ? tid : sp.tail0 + tid - sp.head;
    const float edge = edge_at < 0 ? -INFINITY : to_f32(x[edge_at]);

    const int64_t slice = (sp.nv + C - 1) / C, from = rank * slice, to = min(from + slice, sp.nv);
    const T* body = x + sp.head;
    Stat st;
    {
        Base base(-INFINITY);
        float top = -INFINITY, sum = 0.0f;
        auto follow = [&](float m) {
            if (m > top) {
                const Base next(m);
                if (top != -INFINITY) sum *= ex2((top - next.m) * LOG2E - base.r + next.r);  // else it is 0, or NaN
                top = m;
                base = next;
            }
        };
        constexpr uint32_t FILL = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;  // -inf
        for (int64_t i = from + tid; i < to; i += K * THREADS) {
            uint4 raw[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                raw[k] = make_uint4(FILL, FILL, FILL, FILL);
                if (i + k * THREADS < to) raw[k] = Vec<T>::load_raw(body + (i + k * THREADS) * N);
            }
            RowVec<T> most;
#pragma unroll
            for (int k = 0; k < K; ++k) most.add(raw[k]);
            follow(most.top(-INFINITY));
            uint64_t part[2] = {};
            auto take = [&](auto form) {
                constexpr bool PLAIN = decltype(form)::value;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    uint64_t p[N / 2];
                    unpack2(raw[k], p);
#pragma unroll
                    for (int e = 0; e < N / 2; ++e) part[e & 1] = tc::f2_add(part[e & 1], base.template of2<PLAIN>(p[e]));
                }
            };
            if (base.plain) take(std::true_type());
            else take(std::false_type());
            float lo, hi;
            tc::f2_unpack(tc::f2_add(part[0], part[1]), lo, hi);
            sum += lo + hi;
        }
        follow(edge);
        sum += base.plain ? base.template of<true>(edge) : base.template of<false>(edge);
        st = warp_stat({top, sum * ex2(-base.r)});
        if (WARP) {
        } else if (C == 1) {
            if (lane == 0) boxes[warp] = st;
            __syncthreads();
        } else {
            cluster_wait();
            if (lane < (GRAD ? C : 1)) cluster_store(tc::smem_u32(&boxes[rank * NW + warp]), lane, st);
            __syncwarp();
            cluster_arrive();
            cluster_wait();
        }
    }
    if (!GRAD && rank != 0) return;
    float4 res = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (warp == 0) {
        if (!WARP) {
            st = {-INFINITY, 0.0f};
            for (int k = lane; k < C * NW; k += 32) st = merge(st, boxes[k]);
            st = warp_stat(st);
        }
        if (tid == 0) {
            const LogSum sum(st);
            const float logp = sum.logp(xt);
            if (writer && !ok && a.p.status) atomicOr(a.p.status, PK_ERR_INDEX);
            if constexpr (!POLICY) {
                a.lse[r] = sum.lse();
                a.p.logp[r] = ok ? logp : 0.0f;
            } else if (ok) {
                const float g = policy_row(a.p, r, q, logp, writer);
                // a gradient of exactly zero (held back by its bound, no KL term) leaves nothing to read
                res = make_float4(st.m, -g / st.s * ex2(-Base(st.m).r), g, g == 0.0f ? 0.0f : 1.0f);
            } else if (writer) {
                policy_row_out(a.p, r);
            }
        }
    }
    if constexpr (GRAD) {
        if (WARP) {
            res.x = __shfl_sync(0xffffffffu, res.x, 0);
            res.y = __shfl_sync(0xffffffffu, res.y, 0);
            res.z = __shfl_sync(0xffffffffu, res.z, 0);
            res.w = __shfl_sync(0xffffffffu, res.w, 0);
            t = __shfl_sync(0xffffffffu, t, 0);
        } else {
            if (tid == 0) {
                result = res;
                target = t;
            }
            __syncthreads();
            res = result;
            t = target;
        }
        if (res.w == 0.0f) {
            row_zero(dx, a.V, rank * THREADS + tid, C * THREADS);
            return;
        }
        const Base base(res.x);
        const uint64_t k2 = tc::f2_pack(res.y, res.y);
        const int64_t tv = t >= sp.head && t < sp.tail0 ? (t - sp.head) / N : -1;
        const int te = static_cast<int>((t - sp.head) % N);
        const bool wide = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15u) == 0;
        T* out = dx + sp.head;
        auto give = [&](auto form, auto aligned) {
            constexpr bool PLAIN = decltype(form)::value;
            for (int64_t i = from + (to - from - 1) / (K * THREADS) * (K * THREADS) + tid; i >= from; i -= K * THREADS) {
                uint4 raw[K];
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (i + k * THREADS < to) raw[k] = load_last(body + (i + k * THREADS) * N);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const int64_t v = i + k * THREADS;
                    if (v >= to) break;
                    uint64_t p[N / 2];
                    unpack2(raw[k], p);
                    float f[N];
#pragma unroll
                    for (int e = 0; e < N / 2; ++e) tc::f2_unpack(tc::f2_mul(base.template of2<PLAIN>(p[e]), k2), f[2 * e], f[2 * e + 1]);
                    if (v == tv)
#pragma unroll
                        for (int e = 0; e < N; ++e)
                            if (e == te) f[e] += res.z;
                    if constexpr (decltype(aligned)::value) {
                        __stcs(reinterpret_cast<uint4*>(out + v * N), pack(f));
                    } else {
#pragma unroll
                        for (int e = 0; e < N; ++e) out[v * N + e] = from_f32<T>(f[e]);
                    }
                }
            }
        };
        if (from < to) {
            // the form goes by the row's maximum alone: res.y carries the 2^-r of the plain one
            if (base.plain && wide) give(std::true_type(), std::true_type());
            else if (base.plain) give(std::true_type(), std::false_type());
            else if (wide) give(std::false_type(), std::true_type());
            else give(std::false_type(), std::false_type());
        }
        if (edge_at >= 0) {
            const float e = ex2((edge - base.m) * LOG2E) * (res.y * ex2(base.r));  // res.y carries 2^-r
            dx[edge_at] = from_f32<T>(e + (edge_at == t ? res.z : 0.0f));
        }
    }
}

// One block per pair. Sums in fp64: a thread's rows in ascending order, then a fixed tree. A pair is a few
// thousand rows, so the time is latency: four rows per thread are loaded side by side (12 -> 7 us for four
// pairs of 2 x 800 rows).
constexpr int PAIR_THREADS = 512;
__global__ void __launch_bounds__(PAIR_THREADS)
preference_loss_kernel(const float* logp, const float* ref, const float* weight,
                       const int32_t* seq, int64_t R, float beta, float eps, float gscale,
                       float* loss, float* margin, float* dlogp, int32_t* status) {
    constexpr int U = 4, WARPS = PAIR_THREADS / 32;
    __shared__ double red[WARPS];
    __shared__ float dz_s;
    const int64_t pair = blockIdx.x;
    after_predecessor();
    const int64_t a = seq[2 * pair], b = seq[2 * pair + 1], c = seq[2 * pair + 2];
    if (a < 0 || b < a || c < b || c > R) {
        if (threadIdx.x == 0) {
            if (status) atomicOr(status, PK_ERR_INDEX);
            loss[pair] = __int_as_float(0x7fffffff);
            if (margin) margin[pair] = __int_as_float(0x7fffffff);
        }
        return;
    }
    double acc = 0.0;
    for (int64_t i0 = a + threadIdx.x; i0 < c; i0 += U * PAIR_THREADS) {
        float w[U], l[U], r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = i0 + u * PAIR_THREADS;
            const bool in = i < c;
            w[u] = in ? (weight ? weight[i] : 1.0f) : 0.0f;
            l[u] = in ? logp[i] : 0.0f;
            r[u] = in && ref ? ref[i] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (w[u] == 0.0f) continue;  // whatever the row holds
            const double v = static_cast<double>(w[u]) * (static_cast<double>(l[u]) - static_cast<double>(r[u]));
            acc += i0 + u * PAIR_THREADS < b ? v : -v;
        }
    }
    acc = warp_sum_f64(acc);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        double z = 0.0;
        for (int k = 0; k < WARPS; ++k) z += red[k];
        z *= static_cast<double>(beta);
        // -log sigmoid(z) = softplus(-z); both it and the gradient from e^-|z|
        const double q = exp(-fabs(z)), small = log1p(q);
        const double down = small + fmax(-z, 0.0), up = small + fmax(z, 0.0);
        const double e = eps;
        double l = 0.0;  // a term of coefficient 0 is left out: 0 * inf
        if (e < 1.0) l += (1.0 - e) * down;
        if (e > 0.0) l += e * up;
        if (z != z) l = z;
        loss[pair] = static_cast<float>(l);
        if (margin) margin[pair] = static_cast<float>(z);
        const double below = z >= 0.0 ? q / (1.0 + q) : (z != z ? z : 1.0 / (1.0 + q));  // sigmoid(-z)
        dz_s = static_cast<float>((e - below) * static_cast<double>(beta) * static_cast<double>(gscale));
    }
    __syncthreads();
    if (dlogp == nullptr) return;
    const float dz = dz_s;
    for (int64_t i = a + threadIdx.x; i < c; i += PAIR_THREADS) {
        const float w = weight ? weight[i] : 1.0f;
        dlogp[i] = w == 0.0f ? 0.0f : (i < b ? dz : -dz) * w;
    }
}

int row_threads(int64_t V) { return V >= 4096 ? 512 : (V >= 1024 ? 256 : 128); }
unsigned row_blocks(int64_t R) { return static_cast<unsigned>(std::min<int64_t>(R, static_cast<int64_t>(sm_count()) * 8)); }

// A launch in clusters of `size` CTAs (1: none) that may start before its predecessor has ended.
template <typename... P, typename... A>
int launch(cudaStream_t st, void (*kernel)(P...), dim3 grid, int size, int threads, const A&... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = static_cast<unsigned>(size);
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = size > 1 ? 2 : 1;
    PK_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
    return PK_OK;
}

template <typename T, bool POLICY, bool GRAD>
int launch_rows(cudaStream_t st, const RowArgs& a) {
    constexpr int N = Vec<T>::N;
    const int64_t vectors = (a.V + N - 1) / N;
    const int sms = sm_count();
    // Threads per row, us with a gradient in bf16 for 32 / 128 / 256: 32000 x 6000 145 / 178 / 221, 32000 x 8000
    // 203 / 201 / 240, 16000 x 16000 - / 182 / 195, 12000 x 24000 - / 218 / 207. Few rows take more: 400 x 6000
    // 16 / 12 / 12.
    int threads = vectors <= 896 ? 32 : (vectors <= 2048 ? 128 : 256);
    if (threads == 32 && vectors >= 256 && a.R <= sms * 8) threads = 128;
    if (threads == 128 && vectors >= 512 && a.R <= sms * 4) threads = 256;
    if (threads == 32) return launch(st, sweep_kernel<T, POLICY, GRAD, 32>, dim3(static_cast<unsigned>((a.R + 3) / 4)), 1, 128, a);
    int size = 1;
    // With a gradient a CTA's stretch is at most 100 KB, so that the stretches of all resident CTAs stay in L2:
    // 2048 x 151936 bf16 295 us with one CTA per row, 266 with two, 246 with four, 292 with eight.
    if (GRAD)
        while (size < CLUSTER_MOST && vectors > static_cast<int64_t>(6400) * size) size *= 2;
    // few rows: as many CTAs as are resident, down to two vectors per thread (100 x 151936 bf16 without a gradient:
    // 27 us with one CTA per row, 16 with eight; 400 rows 39, with two 36, with eight 43)
    while (size < CLUSTER_MOST && a.R * size * 2 <= sms * 6 && vectors >= static_cast<int64_t>(4) * threads * size) size *= 2;
    const dim3 grid(static_cast<unsigned>(a.R * size));
    return threads == 128 ? launch(st, sweep_kernel<T, POLICY, GRAD, 128>, grid, size, 128, a)
                          : launch(st, sweep_kernel<T, POLICY, GRAD, 256>, grid, size, 256, a);
}

// dlogits may be logits itself or must not touch it.
bool bad_alias(const void* x, int64_t ld, const void* dx, int64_t ldd, int64_t R, int64_t V, size_t es) {
    if (dx == nullptr) return false;
    if (x == dx) return ld != ldd;
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(dx);
    const uintptr_t an = static_cast<uintptr_t>((R - 1) * ld + V) * es, bn = static_cast<uintptr_t>((R - 1) * ldd + V) * es;
    return a < b + bn && b < a + an;
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" {

int pk_token_logprob(void* stream, int dtype, const void* logits, int64_t ld, const int32_t* targets,
                     const float* weight, float* logp, float* lse, int64_t R, int64_t V, int32_t* status) {
    PK_REQUIRE(valid_dtype(dtype), "bad dtype");
    PK_REQUIRE(R >= 0 && V > 0 && ld >= V, "bad shape");
    PK_REQUIRE(R <= ROWS_MOST, "too many rows");
    if (R == 0) return PK_OK;
    PK_REQUIRE(logits && targets && logp && lse, "null pointer");
    PK_REQUIRE(aligned_to(dtype_size(dtype), logits) && aligned_to(4, targets, weight, logp, lse, status), "buffer not aligned to its type");
    RowArgs a{};
    a.logits = logits; a.ld = ld; a.R = R; a.V = V; a.lse = lse;
    a.p.targets = targets; a.p.weight = weight; a.p.logp = logp; a.p.status = status;
    return dtype == PK_F32 ? launch_rows<float, false, false>(as_stream(stream), a) : launch_rows<bf16, false, false>(as_stream(stream), a);
}

int pk_token_logprob_bwd(void* stream, int dtype, const void* logits, int64_t ld, const int32_t* targets,
                         const float* lse, const float* dlogp, void* dlogits, int64_t ldd, int64_t R, int64_t V,
                         int32_t* status) {
    PK_REQUIRE(valid_dtype(dtype), "bad dtype");
    PK_REQUIRE(R >= 0 && V > 0 && ld >= V && ldd >= V, "bad shape");
    if (R == 0) return PK_OK;
    PK_REQUIRE(logits && targets && lse && dlogp && dlogits, "null pointer");
    PK_REQUIRE(aligned_to(dtype_size(dtype), logits, dlogits) && aligned_to(4, targets, lse, dlogp, status), "buffer not aligned to its type");
    PK_REQUIRE(!bad_alias(logits, ld, dlogits, ldd, R, V, dtype_size(dtype)), "dlogits overlaps logits");
    const int threads = row_threads(V);
    // few rows: several blocks to a row, down to two vectors per thread (80 rows of 32000 bf16: 9.7 -> 7.0 us)
    const int64_t most = std::max<int64_t>(1, V * static_cast<int64_t>(dtype_size(dtype)) / (threads * 32));
    const dim3 grid(row_blocks(R), static_cast<unsigned>(std::min<int64_t>(most, std::max<int64_t>(1, sm_count() * 4 / R))));
    cudaStream_t st = as_stream(stream);
    return dtype == PK_F32 ? launch(st, token_logprob_bwd_kernel<float>, grid, 1, threads, static_cast<const float*>(logits), ld, targets,
                                    lse, dlogp, static_cast<float*>(dlogits), ldd, R, V, status)
                           : launch(st, token_logprob_bwd_kernel<bf16>, grid, 1, threads, static_cast<const bf16*>(logits), ld, targets,
                                    lse, dlogp, static_cast<bf16*>(dlogits), ldd, R, V, status);
}

int pk_preference_loss(void* stream, const float* logp, const float* ref_logp, const float* weight,
                       const int32_t* seq, int64_t n_pairs, int64_t R, float beta, float label_smoothing,
                       float grad_scale, float* loss, float* margin, float* dlogp, int32_t* status) {
    PK_REQUIRE(n_pairs >= 0 && n_pairs <= 0x3fffffff && R >= 0, "bad shape");
    PK_REQUIRE(label_smoothing >= 0.0f && label_smoothing <= 1.0f, "label_smoothing must be in [0, 1]");
    if (n_pairs == 0) return PK_OK;
    PK_REQUIRE(seq && loss && (R == 0 || logp), "null pointer");
    PK_REQUIRE(aligned_to(4, logp, ref_logp, weight, seq, loss, margin, dlogp, status), "buffer not aligned to its type");
    return launch(as_stream(stream), preference_loss_kernel, dim3(static_cast<unsigned>(n_pairs)), 1, PAIR_THREADS, logp, ref_logp, weight, seq,
                  R, beta, label_smoothing, grad_scale, loss, margin, dlogp, status);
}

int pk_policy_loss(void* stream, int dtype, const void* logits, int64_t ld, const int32_t* targets,
                   const float* old_logp, const float* ref_logp, const float* advantage, const float* weight,
                   float clip_lo, float clip_hi, float kl_coef, float grad_scale, float* row_loss, float* logp,
                   float* kl, void* dlogits, int64_t ldd, int64_t R, int64_t V, int32_t* status) {
    PK_REQUIRE(valid_dtype(dtype), "bad dtype");
    PK_REQUIRE(R >= 0 && V > 0 && ld >= V && (dlogits == nullptr || ldd >= V), "bad shape");
    PK_REQUIRE(R <= ROWS_MOST, "too many rows");
    PK_REQUIRE(clip_lo >= 0.0f && clip_lo <= 1.0f && clip_hi >= 0.0f, "clip bounds must not be negative, the lower at most 1");
    if (R == 0) return PK_OK;
    PK_REQUIRE(logits && targets && advantage && row_loss, "null pointer");
    PK_REQUIRE(aligned_to(dtype_size(dtype), logits, dlogits) &&
                   aligned_to(4, targets, old_logp, ref_logp, advantage, weight, row_loss, logp, kl, status),
               "buffer not aligned to its type");
    PK_REQUIRE(!bad_alias(logits, ld, dlogits, ldd, R, V, dtype_size(dtype)), "dlogits overlaps logits");
    const PolicyArgs a = {targets, old_logp, ref_logp, advantage, weight, 1.0f - clip_lo, 1.0f + clip_hi, kl_coef, grad_scale,
                          row_loss, logp, kl, status};
    RowArgs ra{};
    ra.logits = logits; ra.dlogits = dlogits; ra.ld = ld; ra.ldd = ldd; ra.R = R; ra.V = V; ra.p = a;
    cudaStream_t st = as_stream(stream);
    if (dlogits == nullptr) return dtype == PK_F32 ? launch_rows<float, true, false>(st, ra) : launch_rows<bf16, true, false>(st, ra);
    return dtype == PK_F32 ? launch_rows<float, true, true>(st, ra) : launch_rows<bf16, true, true>(st, ra);
}

}  // extern "C"
