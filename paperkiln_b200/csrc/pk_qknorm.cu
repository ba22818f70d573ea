// RMS norm of every query and key head with the rotary embedding in the same pass, forward and
// backward.
//
// Forward, per head x of dk values: inv = rsqrt(mean(x^2) + eps), y = R(pos) (x inv w). With g the
// upstream gradient and g' = R(-pos) g:
//     dx = inv (w g' - x inv^2 mean(w g' x)),   dw += g' x inv  (summed over tokens and heads).
// Both sums of a head (x^2 and w g' x) are over what the pass reads anyway, so the backward needs
// nothing saved by the forward and reduces once.
//
// Bound by memory: 2 (forward) or 3 (backward) accesses per element. bf16: 65536 x 40 heads of 64 take
// 118 - 124 us forward from card to card, 5.6 TB/s; 16381 x 32 heads of 128 73 - 75 us backward, 5.5 TB/s, the sum
// of dw included.
// A team of LANES threads owns a head, 16 bytes per thread. A warp's task is a group of heads of one kind
// and one token (of several tokens where a token has fewer heads than the warp has teams): U heads per
// team, all loaded before the first is computed, with the rotation table's row and the gains in registers.
#include <algorithm>
#include <numeric>
#include <type_traits>

#include "pk_common.cuh"
#include "pk_tc.cuh"

namespace pk {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;  // of the backward
// Small CTAs in the forward, nine to an SM at 56 registers (65536 x 40 heads of 64, on one card: 120 us; four of 256 at
// 64 registers 130, ten at 48 120, and 118 against 114 at head_dim 128).
constexpr int FWD_THREADS = 128, FWD_WARPS = FWD_THREADS / 32;
constexpr int U = 4;  // heads per team in flight, at most

// One kind of heads (queries or keys) and how its tasks are cut.
struct Kind {
    const void* x;        // input of the forward
    const void* g;        // upstream gradient (backward)
    void* y;              // y or dx
    int64_t ldx, ldg, ldy;
    const float* w;
    int heads, rot;
    int step;             // heads side by side in a warp: a power of two, at most the warp's teams
    int u;                // heads per team and task: at most U (7 in the forward), chosen so that rounds are full
    int rounds;           // tasks per group of tokens (teams / step tokens)
    int64_t groups;
    int blocks;           // backward: blocks that work on this kind
};

struct QkArgs {
    Kind kind[2];
    int dk;
    float eps;
    const int32_t* pos;   // null: nothing is rotated
    const float* cs;
    int64_t n_pos, T;
    float* partial;       // backward: [blocks][dk] partial sums of dw (queries' blocks first), or null
};

using tc::f2_add;
using tc::f2_fma;
using tc::f2_mul;
using tc::f2_pack;
using tc::f2_pack_bits;
using tc::f2_unpack;

__device__ __forceinline__ uint64_t f2_both(float v) { return f2_pack(v, v); }
__device__ __forceinline__ float f2_sum(uint64_t v) {
    float lo, hi;
    f2_unpack(v, lo, hi);
    return lo + hi;
}
__device__ __forceinline__ uint64_t f2_neg(uint64_t v) { return v ^ 0x8000000080000000ull; }

// N consecutive elements of a head, held as even and odd ones (the two members of each rotation
// pair) in packed fp32 pairs: the arithmetic of both kernels is two elements per instruction, which
// matters because at copy speed an SM has 22 issue slots per bf16 element. Wide pieces are 16
// bytes and need 16-byte aligned rows; the narrow one (N = 2) takes any alignment and leaves the
// upper halves zero.
template <typename T, int N> struct Piece {
    static constexpr int P = N >= 4 ? N / 4 : 1;
    uint64_t even[P], odd[P];
    static __device__ __forceinline__ uint4 load_raw(const T* p) {
        if constexpr (N * sizeof(T) == 16) return Vec<T>::load_raw(p);
        else if constexpr (sizeof(T) == 4) return make_uint4(__float_as_uint(p[0]), __float_as_uint(p[1]), 0, 0);
        else return make_uint4(__bfloat16_as_ushort(p[0]), __bfloat16_as_ushort(p[1]), 0, 0);
    }
    __device__ __forceinline__ explicit Piece(const uint4& v) {
        if constexpr (N == 8) {
            even[0] = f2_pack_bits(v.x << 16, v.y << 16);
            odd[0] = f2_pack_bits(v.x & 0xffff0000u, v.y & 0xffff0000u);
            even[1] = f2_pack_bits(v.z << 16, v.w << 16);
            odd[1] = f2_pack_bits(v.z & 0xffff0000u, v.w & 0xffff0000u);
        } else if constexpr (N == 4) {
            even[0] = f2_pack_bits(v.x, v.z);
            odd[0] = f2_pack_bits(v.y, v.w);
        } else {
            even[0] = f2_pack_bits(sizeof(T) == 4 ? v.x : v.x << 16, 0);
            odd[0] = f2_pack_bits(sizeof(T) == 4 ? v.y : v.y << 16, 0);
        }
    }
    __device__ __forceinline__ Piece() {}
    __device__ __forceinline__ void store(T* p) const {
        float f[P * 4];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            f2_unpack(even[i], f[4 * i], f[4 * i + 2]);
            f2_unpack(odd[i], f[4 * i + 1], f[4 * i + 3]);
        }
        if constexpr (N * sizeof(T) == 16) {
            float w[N];
#pragma unroll
            for (int e = 0; e < N; ++e) w[e] = f[e];
            Vec<T>::store(p, w);
        } else {
            p[0] = from_f32<T>(f[0]);
            p[1] = from_f32<T>(f[1]);
        }
    }
    // fp32 values of columns c .. c + N - 1 (zeros past dk); wide pieces need 16-byte aligned tables
    __device__ __forceinline__ void table(const float* w, int c, int dk) {
        float f[P * 4] = {};
        if (c < dk) {
            if constexpr (N >= 4) {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const float4 v = *reinterpret_cast<const float4*>(w + c + 4 * i);
                    f[4 * i] = v.x; f[4 * i + 1] = v.y; f[4 * i + 2] = v.z; f[4 * i + 3] = v.w;
                }
            } else {
                f[0] = w[c];
                f[1] = w[c + 1];
            }
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
            even[i] = f2_pack(f[4 * i], f[4 * i + 2]);
            odd[i] = f2_pack(f[4 * i + 1], f[4 * i + 3]);
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
// (j * LANES + lane) * N. Lanes past dk hold zeros, teams past the last head or token zeros or ones, so
// that the shuffles always take all lanes.
template <typename T, int N, int LANES, int PIECES>
struct Place {
    int team, tl;
    __device__ __forceinline__ Place() : team((threadIdx.x & 31) / LANES), tl((threadIdx.x & 31) % LANES) {}
    __device__ __forceinline__ int col(int j) const { return (j * LANES + tl) * N; }
};

__device__ __forceinline__ const float* table_row(const QkArgs& a, int64_t p) {
    return a.cs + (p < 0 ? 0 : (p >= a.n_pos ? a.n_pos - 1 : p)) * a.dk;
}

// What a warp's task is like as a whole. The bounds, and whether a head turns, are a third of the
// instructions of a task; where every head of the round exists, fills its lanes and turns (or none
// does), they are left out.
enum Form { ANY = 0, FULL_TURN = 1, FULL_PLAIN = 2, PART_TURN = 3 };  // PART: lanes past dk are idle
template <Form F, int UU> struct Shape {};
template <typename T, int N, int LANES, int PIECES, bool BACK, typename Run>
__device__ __forceinline__ void with_shape(const QkArgs& a, const Kind& k, int first, bool tokens, Run run) {
    const int last = first + k.step * k.u;
    const bool heads = last <= k.heads && tokens, full = heads && PIECES * LANES * N == a.dk;
    const bool turn = full && last <= k.rot, plain = full && first >= k.rot;
    if constexpr (!BACK) {
        const bool part = heads && !full && last <= k.rot;
        if (k.u == 7) return turn ? run(Shape<FULL_TURN, 7>()) : (part ? run(Shape<PART_TURN, 7>()) : run(Shape<ANY, 7>()));
        if (turn && k.u == 3) return run(Shape<FULL_TURN, 3>());
        if (part) return k.u == 1 ? run(Shape<PART_TURN, 1>()) : (k.u == 2 ? run(Shape<PART_TURN, 2>()) : (k.u == 3 ? run(Shape<PART_TURN, 3>()) : run(Shape<PART_TURN, 4>())));
    }
    if (turn && k.u == 4) run(Shape<FULL_TURN, 4>());
    else if (turn && k.u == 2) run(Shape<FULL_TURN, 2>());
    else if (turn) run(Shape<FULL_TURN, 1>());
    else if (plain && k.u == 4) run(Shape<FULL_PLAIN, 4>());
    else run(Shape<ANY, U>());
}

template <typename T, int N, int LANES, int PIECES, Form F, int UU>
__device__ __forceinline__ void forward_task(const QkArgs& a, const Kind& k, const Place<T, N, LANES, PIECES>& at, int64_t t, int first,
                                             Shape<F, UU>) {
    constexpr bool FULL = F == FULL_TURN || F == FULL_PLAIN, TURNS = F == FULL_TURN || F == PART_TURN;
    const int h0 = first + at.team % k.step;
    const bool token = F != ANY || t < a.T;
    const int heads = min(k.heads, first + k.step * k.u);  // ANY: where the round ends
    const int hop = k.step * a.dk;
    const T* x = static_cast<const T*>(k.x) + t * k.ldx + h0 * a.dk + at.tl * N;
    T* y = static_cast<T*>(k.y) + t * k.ldy + h0 * a.dk + at.tl * N;
    int64_t p = 0;
    if (TURNS || (F == ANY && a.pos && token)) p = a.pos[t];
    uint4 raw[UU][PIECES];
#pragma unroll
    for (int u = 0; u < UU; ++u)
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            if (F == ANY || F == PART_TURN) raw[u][j] = make_uint4(0, 0, 0, 0);
            if (FULL || (at.col(j) < a.dk && (F == PART_TURN || (token && h0 + u * k.step < heads))))
                raw[u][j] = Piece<T, N>::load_raw(x + u * hop + j * (LANES * N));
        }
    // gain and angle of a pair in one: with c, s the angle's and w, w' the pair's gains,
    // (x, x') -> inv (x wc - x' w's, x ws + x' w'c)
    Piece<T, N> w[PIECES], wc[PIECES], ws[PIECES];  // ws.even = w s, ws.odd = -w' s
#pragma unroll
    for (int j = 0; j < PIECES; ++j) w[j].table(k.w, at.col(j), a.dk);
    if (TURNS || (F == ANY && a.pos)) {
        const float* row = table_row(a, p);
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            Piece<T, N> cs;
            cs.table(row, at.col(j), a.dk);  // cos in even, sin in odd
#pragma unroll
            for (int i = 0; i < Piece<T, N>::P; ++i) {
                wc[j].even[i] = f2_mul(w[j].even[i], cs.even[i]);
                wc[j].odd[i] = f2_mul(w[j].odd[i], cs.even[i]);
                ws[j].even[i] = f2_mul(w[j].even[i], cs.odd[i]);
                ws[j].odd[i] = f2_neg(f2_mul(w[j].odd[i], cs.odd[i]));
            }
        }
    }
    const float inv_dk = 1.0f / static_cast<float>(a.dk);
#pragma unroll
    for (int u = 0; u < UU; ++u) {
        const int h = h0 + u * k.step;
        if (F == ANY && first + u * k.step >= heads) break;  // the same for the whole warp
        const bool turn = TURNS || (F == ANY && h < k.rot);
        uint64_t sq = 0;
        Piece<T, N> v[PIECES];
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            v[j] = Piece<T, N>(raw[u][j]);
#pragma unroll
            for (int i = 0; i < Piece<T, N>::P; ++i) sq = f2_fma(v[j].odd[i], v[j].odd[i], f2_fma(v[j].even[i], v[j].even[i], sq));
        }
        const uint64_t inv = f2_both(rsqrtf(team_sum<LANES>(f2_sum(sq)) * inv_dk + a.eps));
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            Piece<T, N> o;
#pragma unroll
            for (int i = 0; i < Piece<T, N>::P; ++i) {
                if (turn) {
                    o.even[i] = f2_mul(inv, f2_fma(v[j].odd[i], ws[j].odd[i], f2_mul(v[j].even[i], wc[j].even[i])));
                    o.odd[i] = f2_mul(inv, f2_fma(v[j].odd[i], wc[j].odd[i], f2_mul(v[j].even[i], ws[j].even[i])));
                } else {
                    o.even[i] = f2_mul(inv, f2_mul(v[j].even[i], w[j].even[i]));
                    o.odd[i] = f2_mul(inv, f2_mul(v[j].odd[i], w[j].odd[i]));
                }
            }
            if (FULL || (at.col(j) < a.dk && (F == PART_TURN || (token && h < heads)))) o.store(y + u * hop + j * (LANES * N));
        }
    }
}

template <typename T, int N, int LANES, int PIECES>
__global__ void __launch_bounds__(FWD_THREADS, PIECES == 1 ? 9 : 1)
qk_norm_rope_fwd_kernel(QkArgs a) {
    constexpr int TEAMS = 32 / LANES;
    const Place<T, N, LANES, PIECES> at;
    const bool keys = static_cast<int>(blockIdx.y) >= a.kind[0].rounds;
    const Kind& k = a.kind[keys];
    const int first = (static_cast<int>(blockIdx.y) - (keys ? a.kind[0].rounds : 0)) * k.step * k.u;
    const int64_t group = static_cast<int64_t>(blockIdx.x) * FWD_WARPS + (threadIdx.x >> 5);
    if (group >= k.groups) return;
    const int per = TEAMS / k.step;
    const int64_t t = group * per + at.team / k.step;
    with_shape<T, N, LANES, PIECES, false>(a, k, first, (group + 1) * per <= a.T, [&](auto shape) { forward_task(a, k, at, t, first, shape); });
}

// One task of the backward; adds the thread's share of dw.
template <typename T, int N, int LANES, int PIECES, Form F, int UU>
__device__ __forceinline__ void backward_task(const QkArgs& a, const Kind& k, const Place<T, N, LANES, PIECES>& at, const T* x,
                                              const T* g, T* y, int first, bool token, int64_t p, const Piece<T, N> (&w)[PIECES],
                                              Piece<T, N> (&dw)[PIECES], Shape<F, UU>) {
    const int h0 = first + at.team % k.step, hop = k.step * a.dk;
    const int heads = min(k.heads, first + k.step * k.u);  // ANY: where the round ends
    uint4 xr[UU][PIECES], gr[UU][PIECES];
#pragma unroll
    for (int u = 0; u < UU; ++u)
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            if (F == ANY) {
                // A team without a head or token holds x = 1 and g = 0, and so adds 0 to dw: with x = 0 and eps = 0 its root
                // would be infinite, and 0 * inf. (The root set to 0 there instead: 191 -> 199 us at 65536 x 14 / 2 heads of 96.)
                const uint32_t one = at.col(j) < a.dk ? (sizeof(T) == 2 ? 0x3f803f80u : 0x3f800000u) : 0u;
                xr[u][j] = make_uint4(one, one, one, one);
                gr[u][j] = make_uint4(0, 0, 0, 0);
            }
            if (F != ANY || (token && h0 + u * k.step < heads && at.col(j) < a.dk)) {
                xr[u][j] = Piece<T, N>::load_raw(x + u * hop + j * (LANES * N));
                gr[u][j] = Piece<T, N>::load_raw(g + u * hop + j * (LANES * N));
            }
        }
    Piece<T, N> cs[PIECES];
    if (F == FULL_TURN || (F == ANY && a.pos)) {
        const float* row = table_row(a, p);
#pragma unroll
        for (int j = 0; j < PIECES; ++j) cs[j].table(row, at.col(j), a.dk);  // cos in even, sin in odd
    }
    const float inv_dk = 1.0f / static_cast<float>(a.dk);
#pragma unroll
    for (int u = 0; u < UU; ++u) {
        const int h = h0 + u * k.step;
        if (F == ANY && first + u * k.step >= heads) break;  // the same for the whole warp
        const bool turn = F == FULL_TURN || (F == ANY && h < k.rot);
        Piece<T, N> xv[PIECES], gv[PIECES];
        uint64_t q1 = 0, q2 = 0;
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            xv[j] = Piece<T, N>(xr[u][j]);
            gv[j] = Piece<T, N>(gr[u][j]);
#pragma unroll
            for (int i = 0; i < Piece<T, N>::P; ++i) {
                if (turn) {  // by the negative angle
                    const uint64_t e = gv[j].even[i], o = gv[j].odd[i];
                    gv[j].even[i] = f2_fma(o, cs[j].odd[i], f2_mul(e, cs[j].even[i]));
                    gv[j].odd[i] = f2_fma(f2_neg(e), cs[j].odd[i], f2_mul(o, cs[j].even[i]));
                }
                q1 = f2_fma(xv[j].odd[i], xv[j].odd[i], f2_fma(xv[j].even[i], xv[j].even[i], q1));
                q2 = f2_fma(f2_mul(gv[j].even[i], w[j].even[i]), xv[j].even[i], q2);
                q2 = f2_fma(f2_mul(gv[j].odd[i], w[j].odd[i]), xv[j].odd[i], q2);
            }
        }
        const float inv = rsqrtf(team_sum<LANES>(f2_sum(q1)) * inv_dk + a.eps);
        const uint64_t inv2 = f2_both(inv), k2 = f2_both(-team_sum<LANES>(f2_sum(q2)) * inv_dk * inv * inv);
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            Piece<T, N> o;
#pragma unroll
            for (int i = 0; i < Piece<T, N>::P; ++i) {
                o.even[i] = f2_mul(inv2, f2_fma(xv[j].even[i], k2, f2_mul(gv[j].even[i], w[j].even[i])));
                o.odd[i] = f2_mul(inv2, f2_fma(xv[j].odd[i], k2, f2_mul(gv[j].odd[i], w[j].odd[i])));
                dw[j].even[i] = f2_fma(f2_mul(gv[j].even[i], xv[j].even[i]), inv2, dw[j].even[i]);
                dw[j].odd[i] = f2_fma(f2_mul(gv[j].odd[i], xv[j].odd[i]), inv2, dw[j].odd[i]);
            }
            if (F != ANY || (token && h < heads && at.col(j) < a.dk)) o.store(y + u * hop + j * (LANES * N));
        }
    }
}

// A warp keeps one round of heads of one kind and walks the groups of tokens, so that what depends on
// the heads is set up once and a thread's share of dw stays in registers. The next group's position is
// fetched a group ahead: only one memory latency (data beside table) stands in a group's way.
template <typename T, int N, int LANES, int PIECES>
__global__ void __launch_bounds__(THREADS, PIECES == 1 ? 2 : 1)
qk_norm_rope_bwd_kernel(QkArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the sum of the partials, if it follows
    constexpr int TEAMS = 32 / LANES;
    __shared__ float red[WARPS][PIECES * LANES * N];
    const Place<T, N, LANES, PIECES> at;
    const bool keys = static_cast<int>(blockIdx.x) >= a.kind[0].blocks;
    const Kind& k = a.kind[keys];
    const int warp = (blockIdx.x - (keys ? a.kind[0].blocks : 0)) * WARPS + (threadIdx.x >> 5);
    const int walkers = k.blocks * WARPS / k.rounds;  // warps per round; the remainder has no work
    const int round = warp / walkers, first = round * k.step * k.u;
    const int per = TEAMS / k.step, sub = at.team / k.step;
    Piece<T, N> dw[PIECES], w[PIECES];
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
        w[j].table(k.w, at.col(j), a.dk);
#pragma unroll
        for (int i = 0; i < Piece<T, N>::P; ++i) dw[j].even[i] = dw[j].odd[i] = 0;
    }
    if (round < k.rounds) {
        int64_t t = static_cast<int64_t>(warp % walkers) * per + sub;
        const int64_t end = (k.groups - 1) * per + sub, hop = static_cast<int64_t>(walkers) * per;
        const int c0 = (first + at.team % k.step) * a.dk + at.tl * N;
        const T* x = static_cast<const T*>(k.x) + t * k.ldx + c0;
        const T* g = static_cast<const T*>(k.g) + t * k.ldg + c0;
        T* y = static_cast<T*>(k.y) + t * k.ldy + c0;
        const bool turns = a.pos != nullptr;
        int64_t p = turns && t < a.T ? a.pos[t] : 0;
        with_shape<T, N, LANES, PIECES, true>(a, k, first, a.T % per == 0, [&](auto shape) {
            for (; t <= end; t += hop, x += hop * k.ldx, g += hop * k.ldg, y += hop * k.ldy) {
                const int64_t ahead = turns && t + hop < a.T ? a.pos[t + hop] : 0;
                backward_task(a, k, at, x, g, y, first, t < a.T, p, w, dw, shape);
                p = ahead;
            }
        });
    }
    if (a.partial == nullptr) return;
    // teams of a warp, then the warps of the block, in a fixed order
#pragma unroll
    for (int j = 0; j < PIECES; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            float lo, hi;
            f2_unpack(e % 2 == 0 ? dw[j].even[e / 4] : dw[j].odd[e / 4], lo, hi);
            float v = e % 4 < 2 ? lo : hi;
#pragma unroll
            for (int o = 16; o >= LANES; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (at.team == 0) red[threadIdx.x >> 5][at.col(j) + e] = v;
        }
    __syncthreads();
    for (int c = threadIdx.x; c < a.dk; c += THREADS) {
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < WARPS; ++q) v += red[q][c];
        a.partial[static_cast<int64_t>(blockIdx.x) * a.dk + c] = v;
    }
}

// dw += sum of the kind's partials, in a fixed order: a block owns 32 columns, its 32 warps take every
// 32nd partial and are then added in ascending order.
__global__ void __launch_bounds__(1024)
qk_gain_grad_kernel(const float* partial, int nq, int nk, int dk, float* dwq, float* dwk) {
    __shared__ float red[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x, n = blockIdx.y == 0 ? nq : nk;
    float* out = blockIdx.y == 0 ? dwq : dwk;
    if (blockIdx.y == 1) partial += static_cast<int64_t>(nq) * dk;
    // launched while the backward still runs, whose partials it waits for here (and so no __restrict__: what is written in
    // this kernel's lifetime must be read coherently)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (out == nullptr) return;
    float v = 0.0f;
    if (c < dk)
        for (int b = threadIdx.y; b < n; b += 32) v += partial[static_cast<int64_t>(b) * dk + c];
    red[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y == 0 && c < dk) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; ++k) s += red[k][threadIdx.x];
        out[c] += s;
    }
}

// Blocks of the backward: one resident wave at 128 registers, shared out by the tasks of a kind and what a task
// takes, at least a warp for every round. A task of u heads per team takes about as long as u + 4 heads: its loads'
// latency is that of four. (By heads alone the warps of few key heads were the last: 65536 x 32 / 8 heads of 64
// 205 -> 176 us, 16 / 1 of 128 266 -> 160, 14 / 2 of 64 126 -> 98; u + 2 182 / 176 / 102, u + 6 179 / 159 / 99.)
constexpr int TASK = 4;
int wave_blocks() { return sm_count() * 2; }
void share_blocks(QkArgs& a) {
    double cost[2];
    for (int r = 0; r < 2; ++r) {
        const Kind& k = a.kind[r];
        cost[r] = k.heads == 0 ? 0.0 : static_cast<double>(k.rounds) * static_cast<double>(k.groups) * (k.u + TASK);
    }
    for (int r = 0; r < 2; ++r) {
        Kind& k = a.kind[r];
        if (k.heads == 0) continue;
        const int least = (k.rounds + WARPS - 1) / WARPS;
        k.blocks = std::max(least, static_cast<int>(wave_blocks() * (cost[r] / (cost[0] + cost[1]))));
        // a few tokens need no full wave
        k.blocks = static_cast<int>(std::min<int64_t>(k.blocks, (k.groups * k.rounds + WARPS - 1) / WARPS));
    }
}
void cut(QkArgs& a, int teams, bool back) {
    for (Kind& k : a.kind) {
        k.step = 1;
        while (k.step < teams && k.step < k.heads) k.step *= 2;
        // a round of U heads per team; fewer where that leaves no round half empty
        k.u = k.heads % (k.step * U) == 0 || k.heads > k.step * U ? U : (k.heads % (k.step * 2) == 0 ? 2 : (k.heads <= k.step ? 1 : U));
        // Head counts that this leaves ragged: fewer side by side, in full rounds of 4, 7 or 3 (forward of 65536 x 14 / 2
        // heads of 64: 77 -> 61 us). A few tokens have time for the bounds, not for longer tasks (37: 2.5 us, else 3.2).
        for (int s = a.T >= 1024 ? k.step : 0; s > 0 && k.heads % (k.step * k.u) != 0; s /= 2)
            for (int u : {4, back ? 2 : 7, back ? 2 : 3})
                if (k.heads % (s * u) == 0) {
                    k.step = s;
                    k.u = u;
                    break;
                }
        k.rounds = (k.heads + k.step * k.u - 1) / (k.step * k.u);
        k.groups = (a.T + teams / k.step - 1) / (teams / k.step);
    }
}

template <typename T, int N, int LANES, int PIECES, bool BACK>
int launch(cudaStream_t st, QkArgs a, int (&blocks)[2]) {
    cut(a, 32 / LANES, BACK);
    if constexpr (BACK) {
        share_blocks(a);
        for (int r = 0; r < 2; ++r) blocks[r] = a.kind[r].blocks;
        qk_norm_rope_bwd_kernel<T, N, LANES, PIECES><<<static_cast<unsigned>(blocks[0] + blocks[1]), THREADS, 0, st>>>(a);
    } else {
        const int64_t gx = (std::max(a.kind[0].heads ? a.kind[0].groups : 0, a.kind[1].heads ? a.kind[1].groups : 0) + FWD_WARPS - 1) / FWD_WARPS;
        const int gy = a.kind[0].rounds + a.kind[1].rounds;
        PK_REQUIRE(gx <= 0x7fffffff && gy <= 65535, "too many rows or heads");
        qk_norm_rope_fwd_kernel<T, N, LANES, PIECES><<<dim3(static_cast<unsigned>(gx), gy), FWD_THREADS, 0, st>>>(a);
    }
    PK_LAUNCH_CHECK();
    return PK_OK;
}

template <typename T, bool BACK>
int dispatch(cudaStream_t st, const QkArgs& a, bool wide, int (&blocks)[2]) {
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

// T rows of a kind of heads.
struct Rows {
    const void* p;
    int64_t ld, cols;
};
// Whether rows of a and b share memory. Two column ranges of one buffer span the same memory and do not, when they stay
// apart within the rows' stride (of two strides, within their common measure).
bool meet(const Rows& a, const Rows& b, int64_t T, size_t es) {
    if (a.cols == 0 || b.cols == 0) return false;
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
    const uintptr_t na = static_cast<uintptr_t>((T - 1) * a.ld + a.cols) * es, nb = static_cast<uintptr_t>((T - 1) * b.ld + b.cols) * es;
    if (pa + na <= pb || pb + nb <= pa) return false;
    if (T == 1) return true;
    const uintptr_t m = static_cast<uintptr_t>(std::gcd(a.ld, b.ld)) * es, ca = a.cols * es, cb = b.cols * es;
    const uintptr_t d = pb >= pa ? (pb - pa) % m : (m - (pa - pb) % m) % m;  // where b starts in a's stride
    return !(d >= ca && d + cb <= m);
}
bool same(const Rows& a, const Rows& b) { return a.p == b.p && a.ld == b.ld; }

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
    PK_REQUIRE((q != qo || ldq == ldqo) && (k != ko || ldk == ldko), "in place needs equal row strides");
    PK_REQUIRE((Hq == 0 || aligned_to(dtype_size(dtype), q, qo)) && (Hkv == 0 || aligned_to(dtype_size(dtype), k, ko)) &&
                   aligned_to(4, Hq ? wq : nullptr, Hkv ? wk : nullptr, turn ? pos : nullptr, turn ? cos_sin : nullptr),
               "buffer not aligned to its type");
    {
        const size_t es = dtype_size(dtype);
        const Rows in[2] = {{q, ldq, cq}, {k, ldk, ck}}, out[2] = {{qo, ldqo, cq}, {ko, ldko, ck}};
        for (int r = 0; r < 2; ++r) {
            PK_REQUIRE(same(out[r], in[r]) || !meet(out[r], in[r], T, es), "an output overlaps its input");
            PK_REQUIRE(!meet(out[r], in[1 - r], T, es), "an output overlaps the input of the other kind");
        }
        PK_REQUIRE(!meet(out[0], out[1], T, es), "the outputs overlap");
    }
    QkArgs a{};
    a.kind[0] = {q, nullptr, qo, ldq, 0, ldqo, wq, Hq, rot_q, 0, 0, 0, 0, 0};
    a.kind[1] = {k, nullptr, ko, ldk, 0, ldko, wk, Hkv, rot_k, 0, 0, 0, 0, 0};
    a.dk = head_dim; a.eps = eps; a.pos = turn ? pos : nullptr; a.cs = cos_sin; a.n_pos = n_pos; a.T = T;
    const int vec = dtype == PK_F32 ? 4 : 8;
    const bool wide = head_dim % vec == 0 && (!turn || aligned16(cos_sin)) && (Hq == 0 || aligned16(wq)) && (Hkv == 0 || aligned16(wk)) &&
                      (Hq == 0 || (rows_aligned(q, ldq, dtype) && rows_aligned(qo, ldqo, dtype))) &&
                      (Hkv == 0 || (rows_aligned(k, ldk, dtype) && rows_aligned(ko, ldko, dtype)));
    int blocks[2] = {};
    return dtype == PK_F32 ? dispatch<float, false>(as_stream(stream), a, wide, blocks)
                           : dispatch<bf16, false>(as_stream(stream), a, wide, blocks);
}

size_t pk_qk_norm_rope_bwd_scratch_bytes(int64_t T, int Hq, int Hkv, int head_dim) {
    (void)T;
    if (Hq < 0 || Hkv < 0 || head_dim <= 0) return 0;
    // a wave, and a warp for every round where that is more: a head per round makes the most rounds
    const size_t blocks = static_cast<size_t>(wave_blocks()) + static_cast<size_t>(Hq + WARPS - 1) / WARPS + static_cast<size_t>(Hkv + WARPS - 1) / WARPS;
    return blocks * static_cast<size_t>(head_dim) * sizeof(float);
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
    PK_REQUIRE((dqo != dq || lddqo == lddq) && (dko != dk || lddko == lddk), "in place needs equal row strides");
    const bool gains = dwq != nullptr || dwk != nullptr;
    PK_REQUIRE(!gains || scratch, "the gains' gradients need scratch");
    PK_REQUIRE(!gains || dwq != dwk, "the two gains' gradients must be two buffers");
    PK_REQUIRE((Hq == 0 || aligned_to(dtype_size(dtype), q, dqo, dq)) && (Hkv == 0 || aligned_to(dtype_size(dtype), k, dko, dk)) &&
                   aligned_to(4, Hq ? wq : nullptr, Hkv ? wk : nullptr, dwq, dwk, turn ? pos : nullptr, turn ? cos_sin : nullptr) &&
                   (!gains || aligned_to(4, static_cast<const char*>(scratch))),
               "buffer not aligned to its type");
    {
        const size_t es = dtype_size(dtype);
        const Rows in[2] = {{q, ldq, cq}, {k, ldk, ck}}, up[2] = {{dqo, lddqo, cq}, {dko, lddko, ck}}, out[2] = {{dq, lddq, cq}, {dk, lddk, ck}};
        for (int r = 0; r < 2; ++r) {
            PK_REQUIRE((same(out[r], in[r]) || !meet(out[r], in[r], T, es)) && (same(out[r], up[r]) || !meet(out[r], up[r], T, es)),
                       "an output overlaps its input");
            PK_REQUIRE(!meet(out[r], in[1 - r], T, es) && !meet(out[r], up[1 - r], T, es), "an output overlaps an input of the other kind");
        }
        PK_REQUIRE(!meet(out[0], out[1], T, es), "the outputs overlap");
    }
    QkArgs a{};
    a.kind[0] = {q, dqo, dq, ldq, lddqo, lddq, wq, Hq, rot_q, 0, 0, 0, 0, 0};
    a.kind[1] = {k, dko, dk, ldk, lddko, lddk, wk, Hkv, rot_k, 0, 0, 0, 0, 0};
    a.dk = head_dim; a.eps = eps; a.pos = turn ? pos : nullptr; a.cs = cos_sin; a.n_pos = n_pos; a.T = T;
    a.partial = gains ? static_cast<float*>(scratch) : nullptr;
    const int vec = dtype == PK_F32 ? 4 : 8;
    const bool wide = head_dim % vec == 0 && (!turn || aligned16(cos_sin)) && (Hq == 0 || aligned16(wq)) && (Hkv == 0 || aligned16(wk)) &&
                      (Hq == 0 || (rows_aligned(q, ldq, dtype) && rows_aligned(dqo, lddqo, dtype) && rows_aligned(dq, lddq, dtype))) &&
                      (Hkv == 0 || (rows_aligned(k, ldk, dtype) && rows_aligned(dko, lddko, dtype) && rows_aligned(dk, lddk, dtype)));
    int blocks[2] = {};
    const int rc = dtype == PK_F32 ? dispatch<float, true>(as_stream(stream), a, wide, blocks)
                                   : dispatch<bf16, true>(as_stream(stream), a, wide, blocks);
    if (rc != PK_OK || !gains) return rc;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((head_dim + 31) / 32, 2);
    cfg.blockDim = dim3(32, 32);
    cfg.stream = as_stream(stream);
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    PK_CHECK_CUDA(cudaLaunchKernelEx(&cfg, qk_gain_grad_kernel, static_cast<const float*>(scratch), blocks[0], blocks[1], head_dim, dwq, dwk));
    return PK_OK;
}

}  // extern "C"
