// RMS norm of every query and key head with the rotary embedding in the same pass, forward and
// backward.
//
// Forward, per head x of dk values: inv = rsqrt(mean(x^2) + eps), y = R(pos) (x inv w). With g the
// upstream gradient and g' = R(-pos) g:
//     dx = inv (w g' - x inv^2 mean(w g' x)),   dw += g' x inv  (summed over tokens and heads).
// Both sums of a head (x^2 and w g' x) are over what the pass reads anyway, so the backward needs
// nothing saved by the forward and reduces once.
//
// Bound by memory: 2 (forward) or 3 (backward) accesses per element. A team of LANES threads owns a
// head (16 bytes per thread), a warp walks the heads of one token and keeps the token's part of the
// rotation table and the gains in registers; heads are taken U at a time so that U wide loads
// per thread are in flight.
#include <algorithm>

#include "pk_common.cuh"

namespace pk {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int U = 4;  // heads per team in flight

struct QkArgs {
    const void* x[2];     // q, k: inputs of the forward
    const void* g[2];     // upstream gradients (backward)
    void* y[2];           // outputs: y or dx
    int64_t ldx[2], ldg[2], ldy[2];
    const float* w[2];
    int heads[2], rot[2];
    int dk;
    float eps;
    const int32_t* pos;
    const float* cs;
    int64_t n_pos, T;
    int parts;            // warps that share a token
    float* partial;       // backward: [blocks][2][dk] partial sums of dw, or null
};

// N consecutive elements. Wide accesses need 16-byte aligned rows; the narrow form (N = 2, one
// rotation pair) takes any alignment.
template <typename T, int N> struct Piece {
    static constexpr bool WIDE = N * sizeof(T) == 16;
    __device__ __forceinline__ static void load(const T* p, float (&f)[N]) {
        if constexpr (WIDE) Vec<T>::load(p, f);
        else {
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = to_f32(p[e]);
        }
    }
    __device__ __forceinline__ static void store(T* p, const float (&f)[N]) {
        if constexpr (WIDE) Vec<T>::store(p, f);
        else {
#pragma unroll
            for (int e = 0; e < N; ++e) p[e] = from_f32<T>(f[e]);
        }
    }
};

template <int LANES>
__device__ __forceinline__ float team_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A thread holds PIECES pieces of N elements of its head: piece j covers elements
// (j * LANES + lane) * N. Every warp works on whole warps of threads; teams past the last head and
// lanes past dk hold zeros, so that the shuffles always take all lanes.
template <typename T, int N, int LANES, int PIECES, bool BACK>
__global__ void __launch_bounds__(THREADS)
qk_norm_rope_kernel(QkArgs a) {
    constexpr int TEAMS = 32 / LANES;
    const int lane = threadIdx.x & 31, team = lane / LANES, tl = lane % LANES;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * WARPS;
    const int64_t tasks = a.T * a.parts;
    const float inv_dk = 1.0f / static_cast<float>(a.dk);
    float dw[2][PIECES][N] = {};
    float w[2][PIECES][N];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int j = 0; j < PIECES; ++j)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int c = (j * LANES + tl) * N + e;
                w[r][j][e] = c < a.dk ? a.w[r][c] : 0.0f;
            }
    for (int64_t task = static_cast<int64_t>(blockIdx.x) * WARPS + (threadIdx.x >> 5); task < tasks; task += warps) {
        const int64_t t = task / a.parts;
        const int part = static_cast<int>(task - t * a.parts);
        float cs[PIECES][N];  // (cos, sin) of the thread's pairs; the backward turns by the negative angle
        if (a.rot[0] + a.rot[1] > 0) {
            int64_t p = a.pos[t];
            p = p < 0 ? 0 : (p >= a.n_pos ? a.n_pos - 1 : p);
            const float* row = a.cs + p * a.dk;
#pragma unroll
            for (int j = 0; j < PIECES; ++j)
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const int c = (j * LANES + tl) * N + e;
                    float2 v = make_float2(1.0f, 0.0f);
                    if (c < a.dk) v = *reinterpret_cast<const float2*>(row + c);
                    cs[j][e] = v.x;
                    cs[j][e + 1] = BACK ? -v.y : v.y;
                }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const T* x = static_cast<const T*>(a.x[r]) + t * a.ldx[r];
            const T* g = BACK ? static_cast<const T*>(a.g[r]) + t * a.ldg[r] : nullptr;
            T* y = static_cast<T*>(a.y[r]) + t * a.ldy[r];
            const int H = a.heads[r];
            for (int h0 = part * TEAMS * U; h0 < H; h0 += a.parts * TEAMS * U) {
                float xv[U][PIECES][N], gv[BACK ? U : 1][PIECES][N];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int h = h0 + u * TEAMS + team;
#pragma unroll
                    for (int j = 0; j < PIECES; ++j) {
                        const int c = (j * LANES + tl) * N;
#pragma unroll
                        for (int e = 0; e < N; ++e) {
                            xv[u][j][e] = 0.0f;
                            if constexpr (BACK) gv[u][j][e] = 0.0f;
                        }
                        if (h < H && c < a.dk) {
                            Piece<T, N>::load(x + h * a.dk + c, xv[u][j]);
                            if constexpr (BACK) Piece<T, N>::load(g + h * a.dk + c, gv[u][j]);
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int h = h0 + u * TEAMS + team;
                    const bool turn = h < a.rot[r];
                    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
                    for (int j = 0; j < PIECES; ++j) {
                        if constexpr (BACK) {
                            if (turn)
#pragma unroll
                                for (int e = 0; e < N; e += 2) {
                                    float o0, o1;
                                    rope_rotate(gv[u][j][e], gv[u][j][e + 1], cs[j][e], cs[j][e + 1], o0, o1);
                                    gv[u][j][e] = o0;
                                    gv[u][j][e + 1] = o1;
                                }
                        }
#pragma unroll
                        for (int e = 0; e < N; ++e) {
                            s1 += xv[u][j][e] * xv[u][j][e];
                            if constexpr (BACK) s2 += gv[u][j][e] * w[r][j][e] * xv[u][j][e];
                        }
                    }
                    s1 = team_sum<LANES>(s1);
                    const float inv = rsqrtf(s1 * inv_dk + a.eps);
                    float k2 = 0.0f;
                    if constexpr (BACK) k2 = team_sum<LANES>(s2) * inv_dk * inv * inv;
#pragma unroll
                    for (int j = 0; j < PIECES; ++j) {
                        float o[N];
                        if constexpr (BACK) {
#pragma unroll
                            for (int e = 0; e < N; ++e) {
                                o[e] = inv * (gv[u][j][e] * w[r][j][e] - xv[u][j][e] * k2);
                                dw[r][j][e] += gv[u][j][e] * (xv[u][j][e] * inv);
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < N; e += 2) {
                                const float y0 = xv[u][j][e] * inv * w[r][j][e], y1 = xv[u][j][e + 1] * inv * w[r][j][e + 1];
                                o[e] = y0;
                                o[e + 1] = y1;
                                if (turn) rope_rotate(y0, y1, cs[j][e], cs[j][e + 1], o[e], o[e + 1]);
                            }
                        }
                        const int c = (j * LANES + tl) * N;
                        if (h < H && c < a.dk) Piece<T, N>::store(y + h * a.dk + c, o);
                    }
                }
            }
        }
    }
    if constexpr (BACK) {
        if (a.partial == nullptr) return;
        // teams of a warp, then the warps of the block, in a fixed order
        __shared__ float red[WARPS][PIECES * LANES * N];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (int j = 0; j < PIECES; ++j)
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    float v = dw[r][j][e];
#pragma unroll
                    for (int o = 16; o >= LANES; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                    if (team == 0) red[threadIdx.x >> 5][(j * LANES + tl) * N + e] = v;
                }
            __syncthreads();
            for (int c = threadIdx.x; c < a.dk; c += THREADS) {
                float v = 0.0f;
#pragma unroll
                for (int k = 0; k < WARPS; ++k) v += red[k][c];
                a.partial[(static_cast<int64_t>(blockIdx.x) * 2 + r) * a.dk + c] = v;
            }
            __syncthreads();
        }
    }
}

// dw[r][c] += sum of the blocks' partials, in a fixed order: a block owns 32 columns, its 32 warps
// take every 32nd partial and are then added in ascending order.
__global__ void __launch_bounds__(1024)
qk_gain_grad_kernel(const float* __restrict__ partial, int blocks, int dk, float* __restrict__ dwq, float* __restrict__ dwk) {
    __shared__ float red[32][33];
    const int r = blockIdx.y, c = blockIdx.x * 32 + threadIdx.x;
    float* out = r == 0 ? dwq : dwk;
    if (out == nullptr) return;
    float v = 0.0f;
    if (c < dk)
        for (int b = threadIdx.y; b < blocks; b += 32) v += partial[(static_cast<int64_t>(b) * 2 + r) * dk + c];
    red[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y == 0 && c < dk) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; ++k) s += red[k][threadIdx.x];
        out[c] += s;
    }
}

int bwd_blocks_most() { return sm_count() * 4; }

// Warps that share a token: as many as keep the grid full when there are few tokens, never more than
// the token has head groups of one warp.
int parts_for(int64_t T, int Hq, int Hkv, int teams) {
    const int groups = std::max((Hq + teams * U - 1) / (teams * U), (Hkv + teams * U - 1) / (teams * U));
    const int64_t want = (static_cast<int64_t>(sm_count()) * 16 + T - 1) / T;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(groups, want)));
}

template <typename T, int N, int LANES, int PIECES, bool BACK>
int launch(cudaStream_t st, QkArgs a, int* blocks_out) {
    a.parts = parts_for(a.T, a.heads[0], a.heads[1], 32 / LANES);
    const int64_t need = (a.T * a.parts + WARPS - 1) / WARPS;
    const int64_t cap = BACK ? bwd_blocks_most() : static_cast<int64_t>(sm_count()) * 16;
    const int blocks = static_cast<int>(std::min(need, cap));
    *blocks_out = blocks;
    qk_norm_rope_kernel<T, N, LANES, PIECES, BACK><<<blocks, THREADS, 0, st>>>(a);
    PK_LAUNCH_CHECK();
    return PK_OK;
}

template <typename T, bool BACK>
int dispatch(cudaStream_t st, const QkArgs& a, bool wide, int* blocks) {
    constexpr int N = Vec<T>::N;
    if (wide) {
        const int lanes = (a.dk + N - 1) / N;
        if (lanes <= 4) return launch<T, N, 4, 1, BACK>(st, a, blocks);
        if (lanes <= 8) return launch<T, N, 8, 1, BACK>(st, a, blocks);
        if (lanes <= 16) return launch<T, N, 16, 1, BACK>(st, a, blocks);
        if (lanes <= 32) return launch<T, N, 32, 1, BACK>(st, a, blocks);
        return launch<T, N, 32, 2, BACK>(st, a, blocks);
    }
    return launch<T, 2, 32, 4, BACK>(st, a, blocks);
}

const char* check_args(int dtype, int64_t T, int Hq, int Hkv, int dk, int rot_q, int rot_k, float eps) {
    if (!valid_dtype(dtype)) return "bad dtype";
    if (T < 0 || Hq < 0 || Hkv < 0) return "negative size";
    if (dk <= 0 || dk % 2 != 0 || dk > 256) return "head_dim must be even and at most 256";
    if (rot_q < 0 || rot_q > Hq || rot_k < 0 || rot_k > Hkv) return "more rotated heads than heads";
    if (!(eps >= 0.0f)) return "eps must not be negative";
    return nullptr;
}

bool rows_aligned(const void* p, int64_t ld, int dtype) {
    return aligned16(p) && static_cast<size_t>(ld) * dtype_size(dtype) % 16 == 0;
}

}  // namespace
}  // namespace pk

using namespace pk;

#define PK_QK_CHECK(cond, msg)                     \
    do {                                           \
        if (!(cond)) {                             \
            pk::set_error("%s: %s", __func__, msg); \
            return PK_ERR_INVALID;                 \
        }                                          \
    } while (0)

extern "C" {

int pk_qk_norm_rope_fwd(void* stream, int dtype, const void* q, int64_t ldq, const void* k, int64_t ldk,
                        const float* wq, const float* wk, void* qo, int64_t ldqo, void* ko, int64_t ldko,
                        int64_t T, int Hq, int Hkv, int head_dim, int rot_q, int rot_k, float eps,
                        const int32_t* pos, const float* cos_sin, int64_t n_pos) {
    const char* bad = check_args(dtype, T, Hq, Hkv, head_dim, rot_q, rot_k, eps);
    PK_QK_CHECK(bad == nullptr, bad);
    if (T == 0 || Hq + Hkv == 0) return PK_OK;
    const int64_t cq = static_cast<int64_t>(Hq) * head_dim, ck = static_cast<int64_t>(Hkv) * head_dim;
    PK_REQUIRE(cq <= 0x7fffffff && ck <= 0x7fffffff, "a row is too long");
    PK_REQUIRE(ldq >= cq && ldqo >= cq && ldk >= ck && ldko >= ck, "a row stride is smaller than its row");
    PK_REQUIRE(Hq == 0 || (q && qo && wq), "null pointer");
    PK_REQUIRE(Hkv == 0 || (k && ko && wk), "null pointer");
    const bool turn = rot_q + rot_k > 0;
    PK_REQUIRE(!turn || (pos && cos_sin && n_pos > 0), "the rotation needs positions and a table");
    PK_REQUIRE(!turn || (reinterpret_cast<uintptr_t>(cos_sin) & 7u) == 0, "the table must be 8-byte aligned");
    PK_REQUIRE((q != qo || ldq == ldqo) && (k != ko || ldk == ldko), "in place needs equal row strides");
    QkArgs a{};
    a.x[0] = q; a.x[1] = k;
    a.y[0] = qo; a.y[1] = ko;
    a.ldx[0] = ldq; a.ldx[1] = ldk;
    a.ldy[0] = ldqo; a.ldy[1] = ldko;
    a.w[0] = wq ? wq : wk; a.w[1] = wk ? wk : wq;
    a.heads[0] = Hq; a.heads[1] = Hkv;
    a.rot[0] = rot_q; a.rot[1] = rot_k;
    a.dk = head_dim; a.eps = eps; a.pos = pos; a.cs = cos_sin; a.n_pos = n_pos; a.T = T;
    const int vec = dtype == PK_F32 ? 4 : 8;
    const bool wide = head_dim % vec == 0 && (Hq == 0 || (rows_aligned(q, ldq, dtype) && rows_aligned(qo, ldqo, dtype))) &&
                      (Hkv == 0 || (rows_aligned(k, ldk, dtype) && rows_aligned(ko, ldko, dtype)));
    int blocks = 0;
    return dtype == PK_F32 ? dispatch<float, false>(as_stream(stream), a, wide, &blocks)
                           : dispatch<bf16, false>(as_stream(stream), a, wide, &blocks);
}

size_t pk_qk_norm_rope_bwd_scratch_bytes(int64_t T, int Hq, int Hkv, int head_dim) {
    (void)T; (void)Hq; (void)Hkv;
    return static_cast<size_t>(bwd_blocks_most()) * 2 * static_cast<size_t>(std::max(head_dim, 0)) * sizeof(float);
}

int pk_qk_norm_rope_bwd(void* stream, int dtype, const void* dqo, int64_t lddqo, const void* dko, int64_t lddko,
                        const void* q, int64_t ldq, const void* k, int64_t ldk, const float* wq, const float* wk,
                        void* dq, int64_t lddq, void* dk, int64_t lddk, float* dwq, float* dwk, void* scratch,
                        int64_t T, int Hq, int Hkv, int head_dim, int rot_q, int rot_k, float eps,
                        const int32_t* pos, const float* cos_sin, int64_t n_pos) {
    const char* bad = check_args(dtype, T, Hq, Hkv, head_dim, rot_q, rot_k, eps);
    PK_QK_CHECK(bad == nullptr, bad);
    if (T == 0 || Hq + Hkv == 0) return PK_OK;
    const int64_t cq = static_cast<int64_t>(Hq) * head_dim, ck = static_cast<int64_t>(Hkv) * head_dim;
    PK_REQUIRE(cq <= 0x7fffffff && ck <= 0x7fffffff, "a row is too long");
    PK_REQUIRE(ldq >= cq && lddq >= cq && lddqo >= cq && ldk >= ck && lddk >= ck && lddko >= ck, "a row stride is smaller than its row");
    PK_REQUIRE(Hq == 0 || (q && dqo && dq && wq), "null pointer");
    PK_REQUIRE(Hkv == 0 || (k && dko && dk && wk), "null pointer");
    const bool turn = rot_q + rot_k > 0;
    PK_REQUIRE(!turn || (pos && cos_sin && n_pos > 0), "the rotation needs positions and a table");
    PK_REQUIRE(!turn || (reinterpret_cast<uintptr_t>(cos_sin) & 7u) == 0, "the table must be 8-byte aligned");
    PK_REQUIRE((dqo != dq || lddqo == lddq) && (dko != dk || lddko == lddk), "in place needs equal row strides");
    const bool gains = dwq != nullptr || dwk != nullptr;
    PK_REQUIRE(!gains || scratch, "the gains' gradients need scratch");
    PK_REQUIRE(!gains || dwq != dwk, "the two gains' gradients must be two buffers");
    QkArgs a{};
    a.x[0] = q; a.x[1] = k;
    a.g[0] = dqo; a.g[1] = dko;
    a.y[0] = dq; a.y[1] = dk;
    a.ldx[0] = ldq; a.ldx[1] = ldk;
    a.ldg[0] = lddqo; a.ldg[1] = lddko;
    a.ldy[0] = lddq; a.ldy[1] = lddk;
    a.w[0] = wq ? wq : wk; a.w[1] = wk ? wk : wq;
    a.heads[0] = Hq; a.heads[1] = Hkv;
    a.rot[0] = rot_q; a.rot[1] = rot_k;
    a.dk = head_dim; a.eps = eps; a.pos = pos; a.cs = cos_sin; a.n_pos = n_pos; a.T = T;
    a.partial = gains ? static_cast<float*>(scratch) : nullptr;
    const int vec = dtype == PK_F32 ? 4 : 8;
    const bool wide = head_dim % vec == 0 &&
                      (Hq == 0 || (rows_aligned(q, ldq, dtype) && rows_aligned(dqo, lddqo, dtype) && rows_aligned(dq, lddq, dtype))) &&
                      (Hkv == 0 || (rows_aligned(k, ldk, dtype) && rows_aligned(dko, lddko, dtype) && rows_aligned(dk, lddk, dtype)));
    int blocks = 0;
    const int rc = dtype == PK_F32 ? dispatch<float, true>(as_stream(stream), a, wide, &blocks)
                                   : dispatch<bf16, true>(as_stream(stream), a, wide, &blocks);
    if (rc != PK_OK || !gains) return rc;
    qk_gain_grad_kernel<<<dim3((head_dim + 31) / 32, 2), dim3(32, 32), 0, as_stream(stream)>>>(
        static_cast<const float*>(scratch), blocks, head_dim, dwq, dwk);
    PK_LAUNCH_CHECK();
    return PK_OK;
}

}  // extern "C"
