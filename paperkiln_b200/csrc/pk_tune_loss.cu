// Losses of preference and policy tuning over rows of logits: target log-probabilities and their
// gradient, the paired log-ratio loss over sequences, and the clipped policy loss with a KL term
// with its gradient in the same pass.
//
// Per row: lse = M + log(sum_j exp(x_j - M)), logp = x_t - M - log(sum); the gradient of anything that
// depends on the row through logp is dlogits_j = g ([j == t] - exp(x_j - M) / sum). The exponent is
// formed as (x - M) * log2(e), two roundings, not as fma(x, log2(e), -M log2(e)): the latter's
// error grows with |M| and would reach logp, and M log2(e) overflows for rows masked with the type's
// lowest value. Statistics are fp32.
#include <algorithm>

#include "pk_common.cuh"

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
struct Stat {
    float m, s;
};
__device__ __forceinline__ float stat_base(float m) { return m == -INFINITY ? 0.0f : m; }  // no inf - inf below
__device__ __forceinline__ Stat merge(Stat a, Stat b) {
    const float m = fmaxf(a.m, b.m), base = stat_base(m);
    return {m, a.s * ex2((a.m - base) * LOG2E) + b.s * ex2((b.m - base) * LOG2E)};
}
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
        const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(row) & 15u) / static_cast<int64_t>(sizeof(T));
        head = off == 0 ? 0 : min(V, static_cast<int64_t>(Vec<T>::N) - off);
        nv = (V - head) / Vec<T>::N;
        tail0 = head + nv * Vec<T>::N;
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

// dx[j] = g ([j == t] - exp(x_j - base) * inv): the block writes one row. x and dx may be the same
// row; they are read and written by the same thread, element by element or vector by vector.
template <typename T>
__device__ __forceinline__ void row_grad(const T* x, T* dx, int64_t V, int64_t t, float base, float inv, float g) {
    constexpr int N = Vec<T>::N;
    const RowSplit<T> sp(x, V);
    const bool wide = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15u) == 0;
    const float k = -g * inv;
    if (wide) {
        const T* body = x + sp.head;
        T* out = dx + sp.head;
        for (int64_t i = threadIdx.x; i < sp.nv; i += blockDim.x) {
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
    for (int64_t i = threadIdx.x; i < edge; i += blockDim.x) {
        const int64_t c = !wide || i < sp.head ? i : sp.tail0 + i - sp.head;
        float f = ex2((to_f32(x[c]) - base) * LOG2E) * k;
        if (c == t) f += g;
        dx[c] = from_f32<T>(f);
    }
}
template <typename T>
__device__ __forceinline__ void row_zero(T* dx, int64_t V) {
    constexpr int N = Vec<T>::N;
    const RowSplit<T> sp(dx, V);
    for (int64_t i = threadIdx.x; i < sp.nv; i += blockDim.x) *reinterpret_cast<uint4*>(dx + sp.head + i * N) = make_uint4(0, 0, 0, 0);
    for (int64_t c = threadIdx.x; c < sp.head; c += blockDim.x) dx[c] = from_f32<T>(0.0f);
    for (int64_t c = sp.tail0 + threadIdx.x; c < V; c += blockDim.x) dx[c] = from_f32<T>(0.0f);
}

template <typename T>
__global__ void __launch_bounds__(512)
token_logprob_kernel(const T* __restrict__ logits, int64_t ld, const int32_t* __restrict__ targets,
                     const float* __restrict__ weight, float* __restrict__ logp, float* __restrict__ lse, int64_t R, int64_t V,
                     int32_t* status) {
    __shared__ Stat red[16];
    for (int64_t row = blockIdx.x; row < R; row += gridDim.x) {
        if (weight != nullptr && weight[row] == 0.0f) {
            if (threadIdx.x == 0) {
                logp[row] = 0.0f;
                lse[row] = 0.0f;
            }
            continue;
        }
        const T* x = logits + row * ld;
        const Stat st = block_stat(row_stat(x, V), red);
        if (threadIdx.x == 0) {
            const int64_t t = targets[row];
            const bool ok = t >= 0 && t < V;
            if (!ok && status) atomicOr(status, PK_ERR_INDEX);
            const float ls = logf(st.s);
            lse[row] = st.m + ls;
            logp[row] = ok ? to_f32(x[t]) - st.m - ls : 0.0f;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(512)
token_logprob_bwd_kernel(const T* logits, int64_t ld, const int32_t* __restrict__ targets, const float* __restrict__ lse,
                         const float* __restrict__ dlogp, T* dlogits, int64_t ldd, int64_t R, int64_t V, int32_t* status) {
    for (int64_t row = blockIdx.x; row < R; row += gridDim.x) {
        float g = dlogp[row];
        T* dx = dlogits + row * ldd;
        if (g != 0.0f) {
            const int64_t t = targets[row];
            if (t >= 0 && t < V) {
                row_grad(logits + row * ld, dx, V, t, lse[row], 1.0f, g);
                continue;
            }
            if (threadIdx.x == 0 && status) atomicOr(status, PK_ERR_INDEX);
        }
        row_zero(dx, V);
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
// The row's loss, written by one thread, and d loss / d logp.
__device__ __forceinline__ float policy_row(const PolicyArgs& a, int64_t row, float logp, float w) {
    const float adv = a.advantage[row];
    const float r = a.old_logp ? expf(logp - a.old_logp[row]) : (logp == logp ? 1.0f : logp);
    const float free_ = r * adv, held = fminf(fmaxf(r, a.lo), a.hi) * adv;
    float loss = -held, g = 0.0f, kl = 0.0f;
    if (free_ <= held) loss = g = -free_;
    if (free_ != free_) loss = g = free_;
    if (a.ref_logp) {
        const float u = a.ref_logp[row] - logp;
        kl = kl_term(u);
        loss += a.kl_coef * kl;
        g -= a.kl_coef * expm1f(u);
    }
    a.row_loss[row] = w * loss;
    if (a.logp) a.logp[row] = logp;
    if (a.kl) a.kl[row] = kl;
    return w * g * a.gscale;
}
__device__ __forceinline__ void policy_row_out(const PolicyArgs& a, int64_t row) {
    a.row_loss[row] = 0.0f;
    if (a.logp) a.logp[row] = 0.0f;
    if (a.kl) a.kl[row] = 0.0f;
}

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
            if (dlogits) row_zero(dlogits + row * ldd, V);
            continue;
        }
        const T* x = logits + row * ld;
        const Stat st = block_stat(row_stat(x, V), red);
        if (threadIdx.x == 0) grad = policy_row(a, row, to_f32(x[t]) - st.m - logf(st.s), w);
        __syncthreads();
        // a gradient of exactly zero (held back by its bound, no KL term) leaves nothing to read
        if (dlogits) {
            if (grad == 0.0f) row_zero(dlogits + row * ldd, V);
            else row_grad(x, dlogits + row * ldd, V, t, st.m, 1.0f / st.s, grad);
        }
        __syncthreads();
    }
}

// One block per pair. Sums in fp64: a thread's rows in ascending order, then a fixed tree.
__global__ void __launch_bounds__(256)
preference_loss_kernel(const float* __restrict__ logp, const float* __restrict__ ref, const float* __restrict__ weight,
                       const int32_t* __restrict__ seq, int64_t R, float beta, float eps, float gscale,
                       float* __restrict__ loss, float* __restrict__ margin, float* __restrict__ dlogp, int32_t* status) {
    __shared__ double red[8];
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
    for (int64_t i = a + threadIdx.x; i < c; i += blockDim.x) {
        const float w = weight ? weight[i] : 1.0f;
        if (w == 0.0f) continue;
        const double v = static_cast<double>(w) * (static_cast<double>(logp[i]) - (ref ? static_cast<double>(ref[i]) : 0.0));
        acc += i < b ? v : -v;
    }
    acc = warp_sum_f64(acc);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        double z = 0.0;
        for (int k = 0; k < 8; ++k) z += red[k];
        z *= static_cast<double>(beta);
        // -log sigmoid(z) = softplus(-z)
        const double small = log1p(exp(-fabs(z)));
        const double down = small + fmax(-z, 0.0), up = small + fmax(z, 0.0);
        const double e = eps;
        double l = 0.0;  // a term of coefficient 0 is left out: 0 * inf
        if (e < 1.0) l += (1.0 - e) * down;
        if (e > 0.0) l += e * up;
        if (z != z) l = z;
        loss[pair] = static_cast<float>(l);
        if (margin) margin[pair] = static_cast<float>(z);
        dz_s = static_cast<float>((e - 1.0 / (1.0 + exp(z))) * static_cast<double>(beta) * static_cast<double>(gscale));
    }
    __syncthreads();
    if (dlogp == nullptr) return;
    const float dz = dz_s;
    for (int64_t i = a + threadIdx.x; i < c; i += blockDim.x) {
        const float w = weight ? weight[i] : 1.0f;
        dlogp[i] = w == 0.0f ? 0.0f : (i < b ? dz : -dz) * w;
    }
}

int row_threads(int64_t V) { return V >= 4096 ? 512 : (V >= 1024 ? 256 : 128); }
unsigned row_blocks(int64_t R) { return static_cast<unsigned>(std::min<int64_t>(R, static_cast<int64_t>(sm_count()) * 8)); }

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
    const int threads = row_threads(V);
    if (dtype == PK_F32)
        token_logprob_kernel<float><<<row_blocks(R), threads, 0, as_stream(stream)>>>(
            static_cast<const float*>(logits), ld, targets, weight, logp, lse, R, V, status);
    else
        token_logprob_kernel<bf16><<<row_blocks(R), threads, 0, as_stream(stream)>>>(
            static_cast<const bf16*>(logits), ld, targets, weight, logp, lse, R, V, status);
    PK_LAUNCH_CHECK();
    return PK_OK;
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
    if (dtype == PK_F32)
        token_logprob_bwd_kernel<float><<<row_blocks(R), threads, 0, as_stream(stream)>>>(
            static_cast<const float*>(logits), ld, targets, lse, dlogp, static_cast<float*>(dlogits), ldd, R, V, status);
    else
        token_logprob_bwd_kernel<bf16><<<row_blocks(R), threads, 0, as_stream(stream)>>>(
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
    preference_loss_kernel<<<static_cast<unsigned>(n_pairs), 256, 0, as_stream(stream)>>>(
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
