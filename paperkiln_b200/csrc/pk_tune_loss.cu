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

// Running maximum and sum of exponentials of a thread's or a row's values. An empty one has
// m = -inf and s = 0, and so has a row of nothing but -inf.
struct __align__(8) Stat {
    float m, s;
};
__device__ __forceinline__ float stat_base(float m) { return m == -INFINITY ? 0.0f : m; }  // no inf - inf below
__device__ __forceinline__ Stat merge(Stat a, Stat b) {
    const float m = fmaxf(a.m, b.m), base = stat_base(m);
    return {m, a.s * ex2((a.m - base) * LOG2E) + b.s * ex2((b.m - base) * LOG2E)};
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
template <int N>
__device__ __forceinline__ void absorb(Stat& st, const float (&f)[N]) {
    float m = f[0];
#pragma unroll
    for (int e = 1; e < N; ++e) m = fmaxf(m, f[e]);
    if (m > st.m) {
        st.s *= ex2((st.m - m) * LOG2E);  // 0 * exp(-inf) for the first values
        st.m = m;
    }
    const float base = stat_base(st.m);
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) s += ex2((f[e] - base) * LOG2E);
    st.s += s;
}
// All threads of the block get the row's statistics, merged in a fixed order.
__device__ __forceinline__ Stat block_stat(Stat st, Stat* red) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Stat other = {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o)};
        // both partners merge in the same order, so all lanes hold the same bits
        st = (lane & o) ? merge(other, st) : merge(st, other);
    }
    __syncthreads();
    if (lane == 0) red[wid] = st;
    __syncthreads();
    st = red[0];
    for (int w = 1; w < nw; ++w) st = merge(st, red[w]);
    return st;
}

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

template <typename T>
__device__ __forceinline__ Stat row_stat(const T* __restrict__ x, int64_t V) {
    constexpr int N = Vec<T>::N, K = 4;  // K wide loads in flight per thread
    const RowSplit<T> sp(x, V);
    Stat st = {-INFINITY, 0.0f};
    const T* body = x + sp.head;
    int64_t i = threadIdx.x;
    for (; i + (K - 1) * static_cast<int64_t>(blockDim.x) < sp.nv; i += K * static_cast<int64_t>(blockDim.x)) {
        uint4 raw[K];
#pragma unroll
        for (int k = 0; k < K; ++k) raw[k] = Vec<T>::load_raw(body + (i + k * static_cast<int64_t>(blockDim.x)) * N);
        float f[K * N];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float v[N];
            Vec<T>::unpack(raw[k], v);
#pragma unroll
            for (int e = 0; e < N; ++e) f[k * N + e] = v[e];
        }
        absorb(st, f);
    }
    for (; i < sp.nv; i += blockDim.x) {
        float f[N];
        Vec<T>::load(body + i * N, f);
        absorb(st, f);
    }
    for (int64_t c = threadIdx.x; c < sp.head; c += blockDim.x) {
        const float f[1] = {to_f32(x[c])};
        absorb(st, f);
    }
    for (int64_t c = sp.tail0 + threadIdx.x; c < V; c += blockDim.x) {
        const float f[1] = {to_f32(x[c])};
        absorb(st, f);
    }
    return st;
}

// dx[j] = g ([j == t] - exp(x_j - base) * inv): `threads` threads, of which this is `tid`, write one row. x
// and dx may be the same row; they are read and written by the same thread, element by element or vector by vector.
template <typename T>
__device__ __forceinline__ void row_grad(const T* x, T* dx, int64_t V, int64_t t, float base, float inv, float g, int64_t tid, int64_t threads) {
    constexpr int N = Vec<T>::N;
    const RowSplit<T> sp(x, V);
    const bool wide = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15u) == 0;
    const float k = -g * inv;
    if (wide) {
        const T* body = x + sp.head;
        T* out = dx + sp.head;
        for (int64_t i = tid; i < sp.nv; i += threads) {
            float f[N];
            Vec<T>::load(body + i * N, f);
            const int64_t te = t - sp.head - i * N;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                f[e] = ex2((f[e] - base) * LOG2E) * k;
                if (te == e) f[e] += g;
            }
            Vec<T>::store(out + i * N, f);
        }
    }
    const int64_t edge = wide ? sp.head + V - sp.tail0 : V;  // elements outside the vectors
    for (int64_t i = tid; i < edge; i += threads) {
        const int64_t c = !wide || i < sp.head ? i : sp.tail0 + i - sp.head;
        float f = ex2((to_f32(x[c]) - base) * LOG2E) * k;
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

template <typename T>
__global__ void __launch_bounds__(512)
token_logprob_bwd_kernel(const T* logits, int64_t ld, const int32_t* __restrict__ targets, const float* __restrict__ lse,
                         const float* __restrict__ dlogp, T* dlogits, int64_t ldd, int64_t R, int64_t V, int32_t* status) {
    // gridDim.y blocks share a row. Last rows first: the pass that took the log-probabilities has left them in L2.
    const int64_t tid = blockIdx.y * blockDim.x + threadIdx.x, threads = gridDim.y * blockDim.x;
    for (int64_t row = R - 1 - blockIdx.x; row >= 0; row -= gridDim.x) {
        float g = dlogp[row];
        T* dx = dlogits + row * ldd;
        if (g != 0.0f) {
            const int64_t t = targets[row];
            if (t >= 0 && t < V) {
                row_grad(logits + row * ld, dx, V, t, lse[row], 1.0f, g, tid, threads);
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
// the first for |u| < 0.1), expm1 elsewhere.
__device__ __forceinline__ float kl_term(float u) {
    if (fabsf(u) < 0.1f)
        return u * u * (0.5f + u * (1.0f / 6 + u * (1.0f / 24 + u * (1.0f / 120 + u * (1.0f / 720 + u * (1.0f / 5040))))));
    return expm1f(u) - u;
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
    const float r = a.old_logp ? expf(logp - q.old) : (logp == logp ? 1.0f : logp);
    const float free_ = r * q.adv, held = fminf(fmaxf(r, a.lo), a.hi) * q.adv;
    float loss = -held, g = 0.0f, kl = 0.0f;
    if (free_ <= held) loss = g = -free_;
    if (free_ != free_) loss = g = free_;
    if (a.ref_logp) {
        const float u = q.ref - logp;
        kl = kl_term(u);
        loss += a.kl_coef * kl;
        g -= a.kl_coef * expm1f(u);
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

// Loss and gradient of rows too long for a cluster: a CTA sweeps its row twice, the second time through L2
// where it fits (2048 x 400000 bf16).
template <typename T>
__global__ void __launch_bounds__(512)
policy_loss_kernel(const T* logits, int64_t ld, PolicyArgs a, T* dlogits, int64_t ldd, int64_t R, int64_t V) {
    __shared__ Stat red[16];
    __shared__ float grad;
    for (int64_t row = blockIdx.x; row < R; row += gridDim.x) {
        const float w = a.weight ? a.weight[row] : 1.0f;
        const int64_t t = a.targets[row];
        const bool ok = t >= 0 && t < V;
        if (w == 0.0f || !ok) {
            if (threadIdx.x == 0) {
                if (w != 0.0f && a.status) atomicOr(a.status, PK_ERR_INDEX);
                policy_row_out(a, row);
            }
            row_zero(dlogits + row * ldd, V, threadIdx.x, blockDim.x);
            continue;
        }
        const T* x = logits + row * ld;
        const Stat st = block_stat(row_stat(x, V), red);
        if (threadIdx.x == 0) {
            PolicyRow q;
            q.load(a, row);
            grad = policy_row(a, row, q, to_f32(x[t]) - st.m - logf(st.s), true);
        }
        __syncthreads();
        // a gradient of exactly zero (held back by its bound, no KL term) leaves nothing to read
        if (grad == 0.0f) row_zero(dlogits + row * ldd, V, threadIdx.x, blockDim.x);
        else row_grad(x, dlogits + row * ldd, V, t, st.m, 1.0f / st.s, grad, threadIdx.x, blockDim.x);
        __syncthreads();
    }
}

// ---- rows kept on the chip --------------------------------------------------------------------
// One read of the logits: a row stays on the chip between its statistics and its gradient. Short rows
// belong to one or four warps (row_kernel), long ones to a CTA or a cluster (stream_kernel).
constexpr int ROW_THREADS = 512, ROW_WARPS = ROW_THREADS / 32;
template <typename T> struct RowK;
template <> struct RowK<float> { static constexpr int K = 8; };  // 32 registers of exponentials
template <> struct RowK<bf16> { static constexpr int K = 8; };   // 64 registers

struct RowArgs {
    const void* logits;
    void* dlogits;       // null: no gradient
    int64_t ld, ldd, R, V;
    int slots;           // row_kernel: vectors per thread that this row length needs, at most K
    PolicyArgs p;        // policy; of it, targets, weight, logp and status for log-probabilities
    float* lse;          // log-probabilities
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The same under a condition, without a branch around it.
__device__ __forceinline__ void cp_async16_if(bool on, uint32_t dst, const void* src) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %0, 0;\n\t@p cp.async.cg.shared.global [%1], [%2], 16;\n\t}"
                 ::"r"(static_cast<int>(on)), "r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void store16_if(bool on, void* p, const uint4& v) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %0, 0;\n\t@p st.global.v4.b32 [%1], {%2, %3, %4, %5};\n\t}"
                 ::"r"(static_cast<int>(on)), "l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
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
    return {m, warp_sum(st.s * ex2((st.m - stat_base(m)) * LOG2E))};
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
// N gradients to a row that is aligned as the logits are (wide), or not.
template <typename T, int N>
__device__ __forceinline__ void put(T* p, const float (&f)[N], bool wide) {
    if (wide) {
        Vec<T>::store(p, f);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) p[e] = from_f32<T>(f[e]);
    }
}

// Rows of up to K * 32 * WPR vectors: WPR warps own a row, K vectors per thread. A thread takes its
// values' maximum, then their exponentials once, which stay in registers; the warps merge their
// (maximum, sum) pairs, and the gradient is the held exponential times one factor per thread. The
// next two rows are on their way meanwhile: every thread copies its own vectors with cp.async into its
// own slots of shared memory, so the copies need no barrier.
template <typename T, int WPR, bool POLICY>
__global__ void __launch_bounds__(ROW_THREADS, 1)
row_kernel(const RowArgs a) {
    constexpr int N = RowVec<T>::N, K = RowK<T>::K, GT = WPR * 32, GROUPS = ROW_WARPS / WPR;
    extern __shared__ __align__(16) uint4 slots[];  // [2][a.slots][ROW_THREADS]
    __shared__ Stat partial[2][ROW_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = warp / WPR, gtid = tid % GT;
    const int64_t hop = static_cast<int64_t>(gridDim.x) * GROUPS;
    int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + group;
    const T* logits = static_cast<const T*>(a.logits);
    T* dlogits = static_cast<T*>(a.dlogits);
    const uint32_t mine = tc::smem_u32(slots) + tid * 16;

    auto live = [&](int64_t r) { return r < a.R && (a.p.weight == nullptr || a.p.weight[r] != 0.0f); };
    auto fetch = [&](int64_t r, bool wanted, int buf) {
        if (wanted) {
            const T* x = logits + r * a.ld;
            const RowSplit<T> sp(x, a.V);
            const T* body = x + sp.head;
            const int nv = static_cast<int>(sp.nv);
            uint32_t dst = mine + buf * a.slots * (ROW_THREADS * 16);
            for (int v = gtid; v < nv; v += GT, dst += ROW_THREADS * 16) cp_async16(dst, body + static_cast<int64_t>(v) * N);
        }
        cp_async_commit();
    };
    // the elements before the first and behind the last vector of a row belong to the first threads
    auto edge_at = [&](const RowSplit<T>& sp) -> int64_t {
        const int64_t n = sp.head + a.V - sp.tail0;
        if (gtid >= n) return -1;
        return gtid < sp.head ? gtid : sp.tail0 + gtid - sp.head;
    };
    auto fetch_edge = [&](int64_t r, bool wanted) -> float {
        if (!wanted) return -INFINITY;
        const T* x = logits + r * a.ld;
        const int64_t c = edge_at(RowSplit<T>(x, a.V));
        return c < 0 ? -INFINITY : to_f32(x[c]);
    };

    bool now = live(row), next = live(row + hop), later = live(row + 2 * hop);
    fetch(row, now, 0);
    fetch(row + hop, next, 1);
    float edge = fetch_edge(row, now);
    int32_t target = row < a.R ? a.p.targets[row] : 0;
    int buf = 0, side = 0;
    for (; row < a.R; row += hop, buf ^= 1) {
        cp_async_wait<1>();
        const T* x = logits + row * a.ld;
        const RowSplit<T> sp(x, a.V);
        const int nv = static_cast<int>(sp.nv);
        const bool afterwards = live(row + 3 * hop);
        const float edge_next = fetch_edge(row + hop, next);
        T* dx = dlogits ? dlogits + row * a.ldd : nullptr;
        const bool wide = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15u) == 0;
        const int64_t t = target;
        target = row + hop < a.R ? a.p.targets[row + hop] : 0;
        const bool ok = t >= 0 && t < a.V;
        if (now && (ok || !POLICY)) {
            const float xt = ok ? to_f32(x[t]) : 0.0f;
            PolicyRow q;
            if constexpr (POLICY) q.load(a.p, row);
            // maximum, then exponentials against the thread's own maximum
            uint4 raw[K];
            const uint4* from = slots + (buf * a.slots) * ROW_THREADS + tid;
            RowVec<T> most;
#pragma unroll
            for (int j = 0; j < K; ++j)
                if (j * GT + gtid < nv) {
                    raw[j] = from[j * ROW_THREADS];
                    most.add(raw[j]);
                }
            const float m = most.top(edge);
            const Base base(m);
            float ex[K][N], sum = 0.0f, edge_ex;
            auto take = [&](auto plain) {
                constexpr bool PLAIN = decltype(plain)::value;
#pragma unroll
                for (int j = 0; j < K; ++j)
                    if (j * GT + gtid < nv) {
                        float f[N];
                        Vec<T>::unpack(raw[j], f);
#pragma unroll
                        for (int e = 0; e < N; ++e) sum += ex[j][e] = base.template of<PLAIN>(f[e]);
                    }
                edge_ex = base.template of<PLAIN>(edge);
            };
            if (base.plain) take(std::true_type());
            else take(std::false_type());
            const float unit = ex2(-base.r);  // the exponentials carry 2^r
            Stat st = warp_stat({m, (sum + edge_ex) * unit});
            if (WPR > 1) {
                // rows that count take turns between two sets of boxes: a set is written again only behind the
                // next row's barrier, which every reader of the set has passed
                Stat* const box = partial[side];
                side ^= 1;
                if (lane == 0) box[warp] = st;
                asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(GT) : "memory");
                st = {-INFINITY, 0.0f};
                if (lane < WPR) st = box[group * WPR + lane];
                st = warp_stat(st);
            }
            fetch(row + 2 * hop, later, buf);  // every value of this buffer has gone into the statistics
            const float ls = logf(st.s);
            const bool writer = gtid == 0;
            if constexpr (!POLICY) {
                if (writer) {
                    if (!ok && a.p.status) atomicOr(a.p.status, PK_ERR_INDEX);
                    a.lse[row] = st.m + ls;
                    a.p.logp[row] = ok ? xt - st.m - ls : 0.0f;
                }
            } else {
                const float g = policy_row(a.p, row, q, xt - st.m - ls, writer);
                if (dx) {
                    const float k = -g / st.s * ex2((m - st.m) * LOG2E) * unit;
                    T* out = dx + sp.head;
                    const int tv = t >= sp.head && t < sp.tail0 ? static_cast<int>((t - sp.head) / N) : -1;
#pragma unroll
                    for (int j = 0; j < K; ++j) {
                        const int v = j * GT + gtid;
                        if (v < nv) {
                            float f[N];
#pragma unroll
                            for (int e = 0; e < N; ++e) f[e] = ex[j][e] * k;
                            if (v == tv) {
                                const int te = static_cast<int>((t - sp.head) % N);
#pragma unroll
                                for (int e = 0; e < N; ++e)
                                    if (e == te) f[e] += g;
                            }
                            put<T, N>(out + static_cast<int64_t>(v) * N, f, wide);
                        }
                    }
                    const int64_t c = edge_at(sp);
                    if (c >= 0) dx[c] = from_f32<T>(edge_ex * k + (c == t ? g : 0.0f));
                }
            }
        } else {
            fetch(row + 2 * hop, later, buf);
            if (gtid == 0) {
                if (now && a.p.status) atomicOr(a.p.status, PK_ERR_INDEX);
                if constexpr (POLICY) {
                    policy_row_out(a.p, row);
                } else {
                    a.p.logp[row] = 0.0f;
                    a.lse[row] = 0.0f;
                }
            }
            if (POLICY && dx) row_zero(dx, a.V, gtid, GT);
        }
        edge = edge_next;
        now = next;
        next = later;
        later = afterwards;
    }
}

// Long rows: a cluster of 1 to 16 small CTAs owns a row, SLOTS 16-byte vectors per thread. A thread's
// logits stay in registers as they were read (half the registers of fp32 values) from the maximum to the
// gradient, so the exponential is taken twice, once for the sum and once for the gradient. Four CTAs of
// different rows share an SM: while one takes maxima or waits for its cluster's sums, the others keep the
// memory busy. The next row of the CTA is on its way meanwhile: every thread copies its own vectors with
// cp.async into its own slots of shared memory, so the copies need no barrier. What lies behind a row in its
// last slots is filled with -inf, whose exponential is 0: the loops need no bounds. What a row takes besides
// its logits (target, log-probabilities) is loaded for 32 rows at a time, a lane per row, one batch ahead.
//
// Policy loss with gradient, 8192 x 32000 bf16: 207 us, 5.1 TB/s (sweeps through L2: 325). One CTA per
// SM with its warps in lock step took 373, exponentials held in fp32 at two CTAs per SM 227. The kernel
// without any exponential takes 180 to 188: most of what it lacks to the copy's 162 is the chain from a row's
// last byte over the reductions and the cluster's barrier to its scalars, no longer the memory.
constexpr int CLUSTER_MOST = 16, CLUSTER_PORTABLE = 8, STREAM_THREADS = 256, STREAM_WARPS = STREAM_THREADS / 32;
template <typename T, bool POLICY, int SLOTS> struct Stream {
    static constexpr int SLICE = SLOTS * STREAM_THREADS;  // vectors of a row per CTA
    static constexpr int PER_SM = 4;  // 64 registers
    static constexpr size_t SMEM = static_cast<size_t>(SLICE) * 16;
};

template <typename T, bool POLICY, int SLOTS>
__global__ void __launch_bounds__(STREAM_THREADS, Stream<T, POLICY, SLOTS>::PER_SM)
stream_kernel(const RowArgs a) {
    constexpr int N = RowVec<T>::N, THREADS = STREAM_THREADS, SLICE = Stream<T, POLICY, SLOTS>::SLICE;
    extern __shared__ __align__(16) uint4 slots[];  // [SLICE]
    __shared__ Stat boxes[2][CLUSTER_MOST * STREAM_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int C = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
    const int64_t hop = gridDim.x / C, row0 = blockIdx.x / C;
    const int n = static_cast<int>((a.R - row0 + hop - 1) / hop);  // rows of this cluster
    const T* logits = static_cast<const T*>(a.logits);
    T* dlogits = static_cast<T*>(a.dlogits);
    auto meet = [&] {
        if (C == 1) {
            __syncthreads();
        } else {
            cluster_arrive();
            cluster_wait();
        }
    };
    if (C > 1) meet();  // nobody writes to a CTA's boxes before it runs

    __shared__ float4 result;  // maximum, factor of the exponentials, gradient at the target, 1 when there is any
    __shared__ int32_t target;
    __shared__ float target_logit;
    // What rows take besides their logits, for two batches of 32 rows; the first warp's alone.
    struct RowScalars {
        int32_t t;
        float xt;
        PolicyRow q;
    };
    __shared__ RowScalars ahead[2][32];
    auto load_batch = [&](int at) {  // a lane per row; past the end the last row again, not used
        const int64_t r = row0 + min(at + lane, n - 1) * hop;
        RowScalars s{};
        s.t = a.p.targets[r];
        if constexpr (POLICY) s.q.load(a.p, r);
        const bool counts = a.p.weight == nullptr || a.p.weight[r] != 0.0f;
        // the target's logit is read long before the row's gradient may be written over it
        if (counts && s.t >= 0 && s.t < a.V) s.xt = to_f32(logits[r * a.ld + s.t]);
        ahead[(at >> 5) & 1][lane] = s;
        __syncwarp();
    };
    if (warp == 0) {
        load_batch(0);
        load_batch(32);
    }

    const uint32_t mine = tc::smem_u32(slots) + tid * 16;
    const int before = rank * SLICE;  // vectors of the row in the CTAs before this one
    // rows that are not whole vectors from a 16-byte boundary have elements of their own on both sides
    const bool ragged = a.V % N != 0 || (reinterpret_cast<uintptr_t>(logits) & 15u) != 0 || a.ld % N != 0;
    const int even = min(static_cast<int>(a.V / N) - before, SLICE) - tid;
    auto head_of = [&](const T* x) { return ragged ? static_cast<int>(RowSplit<T>(x, a.V).head) : 0; };
    // vectors of a row from this thread's first one to the end of the CTA's slice
    auto span_of = [&](const T* x) { return ragged ? min(static_cast<int>(RowSplit<T>(x, a.V).nv) - before, SLICE) - tid : even; };
    constexpr uint32_t FILL = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;  // -inf
    const uint4 fill = make_uint4(FILL, FILL, FILL, FILL);
    for (int j = 0; j < SLOTS; ++j) slots[j * THREADS + tid] = fill;
    // which of the cluster's next rows count: a bit per row, 32 rows at a time
    auto load_w = [&](int at) {
        const int i = at + lane;
        return i < n ? (a.p.weight ? a.p.weight[row0 + i * hop] : 1.0f) : 0.0f;
    };
    auto fetch = [&](int64_t r, bool wanted) {
        if (wanted) {
            const T* x = logits + r * a.ld;
            const char* from = reinterpret_cast<const char*>(x + head_of(x)) + static_cast<int64_t>(before + tid) * 16;
            const int left = span_of(x);
#pragma unroll
            for (int j = 0; j < SLOTS; ++j) cp_async16_if(j * THREADS < left, mine + j * (THREADS * 16), from + j * (THREADS * 16));
            if (ragged) {  // the row before may have had a vector more
#pragma unroll
                for (int j = 0; j < SLOTS; ++j)
                    if (j * THREADS >= left) slots[j * THREADS + tid] = fill;
            }
        }
        cp_async_commit();
    };
    // the elements before the first and behind the last vector of a row belong to the first threads
    auto edge_at = [&](const RowSplit<T>& sp) -> int64_t {
        if (rank != 0 || tid >= sp.head + a.V - sp.tail0) return -1;
        return tid < sp.head ? tid : sp.tail0 + tid - sp.head;
    };
    auto fetch_edge = [&](int64_t r, bool wanted) -> float {
        if (!ragged || !wanted) return -INFINITY;
        const T* x = logits + r * a.ld;
        const int64_t c = edge_at(RowSplit<T>(x, a.V));
        return c < 0 ? -INFINITY : to_f32(x[c]);
    };

    uint32_t bits = __ballot_sync(0xffffffffu, load_w(0) != 0.0f), bits_next = __ballot_sync(0xffffffffu, load_w(32) != 0.0f);
    float w_ahead = load_w(64);
    auto live = [&](int l) { return ((l < 32 ? bits >> l : bits_next >> (l - 32)) & 1u) != 0; };  // row l of this batch
    int64_t r = row0;
    fetch(r, live(0));
    float edge = fetch_edge(r, live(0));
    int side = 0;
    for (int i = 0; i < n; ++i, r += hop) {
        const int l = i & 31;
        if (i > 0 && l == 0) {
            bits = bits_next;
            bits_next = __ballot_sync(0xffffffffu, w_ahead != 0.0f);
            w_ahead = load_w(i + 64);
            if (warp == 0) load_batch(i + 32);
        }
        const float edge_next = fetch_edge(r + hop, live(l + 1));
        const bool writer = rank == 0 && tid == 0;
        T* dx = dlogits + r * a.ldd;
        if (!live(l)) {
            fetch(r + hop, live(l + 1));
            if constexpr (POLICY) {
                if (writer) policy_row_out(a.p, r);
                if (dlogits) row_zero(dx, a.V, rank * THREADS + tid, C * THREADS);
            } else if (writer) {
                a.lse[r] = 0.0f;
                a.p.logp[r] = 0.0f;
            }
            edge = edge_next;
            continue;
        }
        // ---- statistics of the slice
        cp_async_wait<0>();
        uint4 raw[SLOTS];
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) raw[j] = slots[j * THREADS + tid];
        RowVec<T> most;
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) most.add(raw[j]);
        const float m = most.top(edge);
        fetch(r + hop, live(l + 1));  // this thread's slots have been read
        {
            const Base base(m);
            const bool plain = __all_sync(0xffffffffu, base.plain);
            uint64_t sum[2] = {};
            float edge_ex = 0.0f;
            auto take = [&](auto form) {
                constexpr bool PLAIN = decltype(form)::value;
#pragma unroll
                for (int j = 0; j < SLOTS; ++j) {
                    uint64_t p[N / 2];
                    unpack2(raw[j], p);
#pragma unroll
                    for (int e = 0; e < N / 2; ++e) sum[e & 1] = tc::f2_add(sum[e & 1], base.template of2<PLAIN>(p[e]));
                }
                if (ragged) edge_ex = base.template of<PLAIN>(edge);
            };
            if (plain) take(std::true_type());
            else take(std::false_type());
            float lo, hi;
            tc::f2_unpack(tc::f2_add(sum[0], sum[1]), lo, hi);
            const Stat st = warp_stat({m, (lo + hi + edge_ex) * ex2(plain ? -base.r : 0.0f)});
            if (C == 1) {
                if (lane == 0) boxes[side][warp] = st;
            } else if (lane < C) {
                cluster_store(tc::smem_u32(&boxes[side][rank * STREAM_WARPS + warp]), lane, st);
            }
            __syncwarp();
        }
        meet();  // the row's pairs are in the boxes
        // ---- the row's scalars, by one warp (by every warp they were an eighth of the instructions)
        if (warp == 0) {
            Stat st = {-INFINITY, 0.0f};
            for (int k = lane; k < C * STREAM_WARPS; k += 32) st = merge(st, boxes[side][k]);
            st = warp_stat(st);
            const RowScalars& own = ahead[(i >> 5) & 1][l];
            const int32_t t = own.t;
            const bool ok = t >= 0 && t < a.V;
            const float ls = logf(st.s), logp = own.xt - st.m - ls;
            if (writer && !ok && a.p.status) atomicOr(a.p.status, PK_ERR_INDEX);
            if constexpr (!POLICY) {
                if (writer) {
                    a.lse[r] = st.m + ls;
                    a.p.logp[r] = ok ? logp : 0.0f;
                }
            } else {
                float4 out = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (ok) {
                    const float g = policy_row(a.p, r, own.q, logp, writer);
                    out = make_float4(st.m, -g / st.s * ex2(-Base(st.m).r), g, 1.0f);
                } else if (writer) {
                    policy_row_out(a.p, r);
                }
                if (lane == 0) {
                    result = out;
                    target = t;
                    target_logit = own.xt;
                }
            }
            __syncwarp();
        }
        // rows that count take turns between two sets of boxes: a set is written again only behind the
        // next row's meeting, for which its readers have to be done
        side ^= 1;
        if constexpr (POLICY) {
            if (dlogits) {
                __syncthreads();
                // ---- gradient of the slice
                const float4 res = result;
                if (res.w == 0.0f) {
                    row_zero(dx, a.V, rank * THREADS + tid, C * THREADS);
                } else {
                    const T* x = logits + r * a.ld;
                    const int head = head_of(x), left = span_of(x);
                    const bool wide = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15u) == 0;
                    const Base base(res.x);
                    const uint64_t k = tc::f2_pack(res.y, res.y);
                    T* out = dx + head + static_cast<int64_t>(before + tid) * N;
                    auto give = [&](auto form, auto aligned) {
                        constexpr bool PLAIN = decltype(form)::value;
#pragma unroll
                        for (int j = 0; j < SLOTS; ++j) {
                            uint64_t p[N / 2];
                            unpack2(raw[j], p);
                            float f[N];
#pragma unroll
                            for (int e = 0; e < N / 2; ++e) tc::f2_unpack(tc::f2_mul(base.template of2<PLAIN>(p[e]), k), f[2 * e], f[2 * e + 1]);
                            if constexpr (decltype(aligned)::value) store16_if(j * THREADS < left, out + j * (THREADS * N), pack(f));
                            else if (j * THREADS < left) put<T, N>(out + j * (THREADS * N), f, false);
                        }
                    };
                    if (base.plain && wide) give(std::true_type(), std::true_type());
                    else if (wide) give(std::false_type(), std::true_type());
                    else give(std::false_type(), std::false_type());
                    // the target's element once more, by the thread that has just written it
                    auto value = [&](float v) { return ex2((v - base.m) * LOG2E) * (res.y * ex2(base.r)); };  // res.y carries 2^-r
                    const unsigned te = static_cast<unsigned>(target - head - before * N), at = te / N;
                    if (at < static_cast<unsigned>(SLICE) && at % THREADS == static_cast<unsigned>(tid) && static_cast<int>(at) - tid < left)
                        dx[target] = from_f32<T>(value(target_logit) + res.z);
                    if (ragged) {
                        const int64_t c = edge_at(RowSplit<T>(x, a.V));
                        if (c >= 0) dx[c] = from_f32<T>(value(edge) + (c == target ? res.z : 0.0f));
                    }
                }
            }
        }
        edge = edge_next;
    }
}

// Long rows without a gradient: one pass, nothing is kept. A CTA, or a cluster of CTAs when there are few
// rows, per row; a thread holds FORWARD_K vectors in flight and a running sum of exponentials against a
// reference that follows its maximum only when that has moved by more than 8 (a term stays below e^8, the
// rounding of its exponent below 2^-20). Nothing orders the rows: the memory stays busy by what else is
// resident, eight CTAs to an SM. 8192 x 50257 bf16: 150 us, 5.5 TB/s (the kernel above, which waits for a
// row before it takes the next: 228; four CTAs of 128 registers 158).
constexpr int FORWARD_THREADS = 256, FORWARD_WARPS = FORWARD_THREADS / 32, FORWARD_K = 4, FORWARD_PER_SM = 8;

template <typename T, bool POLICY>
__global__ void __launch_bounds__(FORWARD_THREADS, FORWARD_PER_SM)
forward_kernel(const RowArgs a) {
    constexpr int N = RowVec<T>::N, THREADS = FORWARD_THREADS, K = FORWARD_K;
    __shared__ Stat boxes[CLUSTER_PORTABLE * FORWARD_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int C = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
    const int64_t r = blockIdx.x / static_cast<unsigned>(C);
    const bool writer = rank == 0 && tid == 0;
    if (a.p.weight != nullptr && a.p.weight[r] == 0.0f) {  // the whole cluster
        if (writer) {
            if constexpr (POLICY) {
                policy_row_out(a.p, r);
            } else {
                a.lse[r] = 0.0f;
                a.p.logp[r] = 0.0f;
            }
        }
        return;
    }
    if (C > 1) cluster_arrive();  // nobody writes to a CTA's boxes before it runs
    const T* x = static_cast<const T*>(a.logits) + r * a.ld;
    const RowSplit<T> sp(x, a.V);
    int64_t t = 0;
    bool ok = false;
    float xt = 0.0f;
    PolicyRow q;
    if (writer) {
        t = a.p.targets[r];
        ok = t >= 0 && t < a.V;
        if constexpr (POLICY) q.load(a.p, r);
        if (ok) xt = to_f32(x[t]);
    }
    float edge = -INFINITY;  // the elements before the first and behind the last vector belong to the first threads
    if (rank == 0 && tid < sp.head + a.V - sp.tail0) edge = to_f32(x[tid < sp.head ? tid : sp.tail0 + tid - sp.head]);

    const int64_t slice = (sp.nv + C - 1) / C, from = rank * slice, to = min(from + slice, sp.nv);
    const T* body = x + sp.head;
    Base base(-INFINITY);
    float top = -INFINITY, sum = 0.0f;
    auto follow = [&](float m) {
        if (m > top + 8.0f) {
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
    Stat st = warp_stat({top, sum * ex2(-base.r)});
    if (C == 1) {
        if (lane == 0) boxes[warp] = st;
        __syncthreads();
    } else {
        cluster_wait();
        if (lane == 0) cluster_store(tc::smem_u32(&boxes[rank * FORWARD_WARPS + warp]), 0, st);
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
    if (rank != 0 || warp != 0) return;
    st = {-INFINITY, 0.0f};
    for (int k = lane; k < C * FORWARD_WARPS; k += 32) st = merge(st, boxes[k]);
    st = warp_stat(st);
    if (!writer) return;
    const float ls = logf(st.s);
    if (!ok && a.p.status) atomicOr(a.p.status, PK_ERR_INDEX);
    if constexpr (!POLICY) {
        a.lse[r] = st.m + ls;
        a.p.logp[r] = ok ? xt - st.m - ls : 0.0f;
    } else if (ok) {
        policy_row(a.p, r, q, xt - st.m - ls, true);
    } else {
        policy_row_out(a.p, r);
    }
}

// One block per pair. Sums in fp64: a thread's rows in ascending order, then a fixed tree. A pair is a few
// thousand rows, so the time is latency: four rows per thread are loaded side by side (12 -> 7 us for four
// pairs of 2 x 800 rows).
constexpr int PAIR_THREADS = 512;
__global__ void __launch_bounds__(PAIR_THREADS)
preference_loss_kernel(const float* __restrict__ logp, const float* __restrict__ ref, const float* __restrict__ weight,
                       const int32_t* __restrict__ seq, int64_t R, float beta, float eps, float gscale,
                       float* __restrict__ loss, float* __restrict__ margin, float* __restrict__ dlogp, int32_t* status) {
    constexpr int U = 4, WARPS = PAIR_THREADS / 32;
    __shared__ double red[WARPS];
    __shared__ float dz_s;
    const int64_t pair = blockIdx.x;
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

// Clusters of `size` CTAs of a kernel that are resident at once (asked once per kernel, size and GPU).
int resident_clusters(const void* kernel, int size, int threads, size_t smem, size_t smem_most) {
    struct Known {
        const void* kernel;
        int size, device, count;
        size_t smem;
    };
    static thread_local Known known[16] = {};
    static thread_local int used = 0;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return 0;
    for (int i = 0; i < std::min(used, 16); ++i)
        if (known[i].kernel == kernel && known[i].size == size && known[i].device == device && known[i].smem == smem) return known[i].count;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = static_cast<unsigned>(size);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(size));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_most)) != cudaSuccess ||
        (size > CLUSTER_PORTABLE && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    known[used++ % 16] = {kernel, size, device, n, smem};
    return n;
}

template <typename T, bool POLICY, int SLOTS>
void stream_form(const void** kernel, size_t* smem) {
    *kernel = reinterpret_cast<const void*>(stream_kernel<T, POLICY, SLOTS>);
    *smem = Stream<T, POLICY, SLOTS>::SMEM;
}

int launch_clusters(cudaStream_t st, const void* kernel, int64_t ctas, int size, int threads, size_t smem, RowArgs& a) {
    PK_REQUIRE(ctas <= 0x7fffffff, "too many rows");
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = static_cast<unsigned>(size);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &at;
    cfg.numAttrs = size > 1 ? 1 : 0;
    void* args[] = {&a};
    PK_CHECK_CUDA(cudaLaunchKernelExC(&cfg, kernel, args));
    return PK_OK;
}

// Launches the kernels that read the logits once; *taken is false when there is a gradient and a row does
// not fit a cluster.
template <typename T, bool POLICY>
int launch_rows(cudaStream_t st, RowArgs a, bool* taken) {
    constexpr int N = Vec<T>::N, K = RowK<T>::K;
    const int64_t vectors = (a.V + N - 1) / N;
    const int sms = sm_count();
    *taken = true;
    // From 7 vectors per thread on the free-running rows win (16000 x 16000 bf16 101 against 108 us, 24000 x
    // 10000 133 against 104).
    if (a.dlogits == nullptr && vectors >= 7 * FORWARD_THREADS) {
        // few rows: clusters, down to two vectors per thread (100 x 151936 bf16: 27 us with one CTA, 16 with eight)
        int size = 1;
        while (size < CLUSTER_PORTABLE && a.R * size * 2 <= sms * 6 && vectors >= static_cast<int64_t>(4) * FORWARD_THREADS * size) size *= 2;
        return launch_clusters(st, reinterpret_cast<const void*>(forward_kernel<T, POLICY>), a.R * size, size, FORWARD_THREADS, 0, a);
    }
    *taken = vectors <= static_cast<int64_t>(Stream<T, POLICY, 10>::SLICE) * CLUSTER_MOST;
    if (!*taken) return PK_OK;
    // the fewest warps that hold a row, and more while that leaves SMs without a row
    int wpr = vectors <= K * 32 ? 1 : (vectors <= K * 128 ? 4 : ROW_WARPS);
    while (wpr < ROW_WARPS && a.R * wpr < static_cast<int64_t>(sms) * 8) wpr *= 4;
    int size = 1, threads = ROW_THREADS;
    size_t smem = 0, most = static_cast<size_t>(2) * K * ROW_THREADS * 16;
    const void* kernel = wpr == 1 ? reinterpret_cast<const void*>(row_kernel<T, 1, POLICY>) : reinterpret_cast<const void*>(row_kernel<T, 4, POLICY>);
    if (wpr < ROW_WARPS) {
        a.slots = static_cast<int>((vectors + wpr * 32 - 1) / (wpr * 32));
        smem = static_cast<size_t>(2) * a.slots * ROW_THREADS * 16;
    } else {
        threads = STREAM_THREADS;
        // The fewest CTAs of up to 8 vectors per thread: every CTA more makes a row's chain longer (8192 x 50257
        // bf16: 4 CTAs 387 us, 5 405, 6 479). Seven fill the SMs' groups badly (1021 x 50257 fp32: 100 us, with
        // eight 92). Beyond eight CTAs 10 vectors per thread, although some of them spill, beat more CTAs (2048 x
        // 200064 bf16: 10 CTAs 362 us, 13 407; sweeps 481).
        constexpr int64_t SLICE8 = Stream<T, POLICY, 8>::SLICE, SLICE10 = Stream<T, POLICY, 10>::SLICE;
        size = static_cast<int>((vectors + SLICE8 - 1) / SLICE8);
        if (size == 7) size = 8;
        if (size > 8) size = static_cast<int>((vectors + SLICE10 - 1) / SLICE10);
        // few rows: more CTAs to a row, down to two vectors per thread; beyond 8 CTAs nothing is gained
        while (size < CLUSTER_PORTABLE && a.R * size * 2 <= sms * 4 && vectors >= static_cast<int64_t>(4) * STREAM_THREADS * size)
            size = std::min(size * 2, CLUSTER_PORTABLE);
        const int64_t slice = (vectors + size - 1) / size;
        if (slice <= Stream<T, POLICY, 4>::SLICE) stream_form<T, POLICY, 4>(&kernel, &smem);
        else if (slice <= Stream<T, POLICY, 5>::SLICE) stream_form<T, POLICY, 5>(&kernel, &smem);
        else if (slice <= Stream<T, POLICY, 6>::SLICE) stream_form<T, POLICY, 6>(&kernel, &smem);
        else if (slice <= Stream<T, POLICY, 7>::SLICE) stream_form<T, POLICY, 7>(&kernel, &smem);
        else if constexpr (POLICY) {  // log-probabilities of longer rows are taken above
            if (slice <= SLICE8) stream_form<T, POLICY, 8>(&kernel, &smem);
            else stream_form<T, POLICY, 10>(&kernel, &smem);
        }
        most = smem;
    }
    const int resident = resident_clusters(kernel, size, threads, smem, most);
    if (resident == 0 && a.dlogits == nullptr)
        return launch_clusters(st, reinterpret_cast<const void*>(forward_kernel<T, POLICY>), a.R, 1, FORWARD_THREADS, 0, a);
    if (resident == 0) {
        *taken = false;
        return PK_OK;
    }
    const int64_t groups = wpr == ROW_WARPS ? a.R : (a.R + ROW_WARPS / wpr - 1) / (ROW_WARPS / wpr);
    return launch_clusters(st, kernel, std::min<int64_t>(groups, resident) * size, size, threads, smem, a);
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
    if (R == 0) return PK_OK;
    PK_REQUIRE(logits && targets && logp && lse, "null pointer");
    RowArgs a{};
    a.logits = logits; a.ld = ld; a.R = R; a.V = V; a.lse = lse;
    a.p.targets = targets; a.p.weight = weight; a.p.logp = logp; a.p.status = status;
    bool taken = false;  // always, without a gradient
    return dtype == PK_F32 ? launch_rows<float, false>(as_stream(stream), a, &taken) : launch_rows<bf16, false>(as_stream(stream), a, &taken);
}

int pk_token_logprob_bwd(void* stream, int dtype, const void* logits, int64_t ld, const int32_t* targets,
                         const float* lse, const float* dlogp, void* dlogits, int64_t ldd, int64_t R, int64_t V,
                         int32_t* status) {
    PK_REQUIRE(valid_dtype(dtype), "bad dtype");
    PK_REQUIRE(R >= 0 && V > 0 && ld >= V && ldd >= V, "bad shape");
    if (R == 0) return PK_OK;
    PK_REQUIRE(logits && targets && lse && dlogp && dlogits, "null pointer");
    PK_REQUIRE(!bad_alias(logits, ld, dlogits, ldd, R, V, dtype_size(dtype)), "dlogits overlaps logits");
    const int threads = row_threads(V);
    // few rows: several blocks to a row, down to two vectors per thread (80 rows of 32000 bf16: 9.7 -> 7.0 us)
    const int64_t most = std::max<int64_t>(1, V * static_cast<int64_t>(dtype_size(dtype)) / (threads * 32));
    const dim3 grid(row_blocks(R), static_cast<unsigned>(std::min<int64_t>(most, std::max<int64_t>(1, sm_count() * 4 / R))));
    if (dtype == PK_F32)
        token_logprob_bwd_kernel<float><<<grid, threads, 0, as_stream(stream)>>>(
            static_cast<const float*>(logits), ld, targets, lse, dlogp, static_cast<float*>(dlogits), ldd, R, V, status);
    else
        token_logprob_bwd_kernel<bf16><<<grid, threads, 0, as_stream(stream)>>>(
            static_cast<const bf16*>(logits), ld, targets, lse, dlogp, static_cast<bf16*>(dlogits), ldd, R, V, status);
    PK_LAUNCH_CHECK();
    return PK_OK;
}

int pk_preference_loss(void* stream, const float* logp, const float* ref_logp, const float* weight,
                       const int32_t* seq, int64_t n_pairs, int64_t R, float beta, float label_smoothing,
                       float grad_scale, float* loss, float* margin, float* dlogp, int32_t* status) {
    PK_REQUIRE(n_pairs >= 0 && n_pairs <= 0x3fffffff && R >= 0, "bad shape");
    PK_REQUIRE(label_smoothing >= 0.0f && label_smoothing <= 1.0f, "label_smoothing must be in [0, 1]");
    if (n_pairs == 0) return PK_OK;
    PK_REQUIRE(seq && loss && (R == 0 || logp), "null pointer");
    preference_loss_kernel<<<static_cast<unsigned>(n_pairs), PAIR_THREADS, 0, as_stream(stream)>>>(
        logp, ref_logp, weight, seq, R, beta, label_smoothing, grad_scale, loss, margin, dlogp, status);
    PK_LAUNCH_CHECK();
    return PK_OK;
}

int pk_policy_loss(void* stream, int dtype, const void* logits, int64_t ld, const int32_t* targets,
                   const float* old_logp, const float* ref_logp, const float* advantage, const float* weight,
                   float clip_lo, float clip_hi, float kl_coef, float grad_scale, float* row_loss, float* logp,
                   float* kl, void* dlogits, int64_t ldd, int64_t R, int64_t V, int32_t* status) {
    PK_REQUIRE(valid_dtype(dtype), "bad dtype");
    PK_REQUIRE(R >= 0 && V > 0 && ld >= V && (dlogits == nullptr || ldd >= V), "bad shape");
    PK_REQUIRE(clip_lo >= 0.0f && clip_lo <= 1.0f && clip_hi >= 0.0f, "clip bounds must not be negative, the lower at most 1");
    if (R == 0) return PK_OK;
    PK_REQUIRE(logits && targets && advantage && row_loss, "null pointer");
    PK_REQUIRE(!bad_alias(logits, ld, dlogits, ldd, R, V, dtype_size(dtype)), "dlogits overlaps logits");
    const PolicyArgs a = {targets, old_logp, ref_logp, advantage, weight, 1.0f - clip_lo, 1.0f + clip_hi, kl_coef, grad_scale,
                          row_loss, logp, kl, status};
    RowArgs ra{};
    ra.logits = logits; ra.dlogits = dlogits; ra.ld = ld; ra.ldd = ldd; ra.R = R; ra.V = V; ra.p = a;
    bool taken = false;
    const int rc = dtype == PK_F32 ? launch_rows<float, true>(as_stream(stream), ra, &taken) : launch_rows<bf16, true>(as_stream(stream), ra, &taken);
    if (rc != PK_OK || taken) return rc;
    const int threads = row_threads(V);
    if (dtype == PK_F32)
        policy_loss_kernel<float><<<row_blocks(R), threads, 0, as_stream(stream)>>>(
            static_cast<const float*>(logits), ld, a, static_cast<float*>(dlogits), ldd, R, V);
    else
        policy_loss_kernel<bf16><<<row_blocks(R), threads, 0, as_stream(stream)>>>(
            static_cast<const bf16*>(logits), ld, a, static_cast<bf16*>(dlogits), ldd, R, V);
    PK_LAUNCH_CHECK();
    return PK_OK;
}

}  // extern "C"
