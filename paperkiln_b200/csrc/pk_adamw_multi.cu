// AdamW over many tensors in one launch, with fp32 or 8-bit moments.
//
// The plan is a table of chunks in device memory, one CTA each. Per element the step reads p, g and both
// moments and writes p, both moments and the bf16 shadow: 30 bytes with fp32 moments and gradients, 18.1 with
// 8-bit moments. Bound by memory: 124 M parameters with fp32 moments 535 us, as fast as a copy; 243 M with 8-bit
// moments 795 - 815 us from card to card, 5.4 TB/s (85 % of a copy), where the coding of the moments shares the
// issue slots.
//
// 8-bit moments: E4M3 codes, one power-of-two scale per 32 elements. A scale that is a power of two
// makes both directions exact but for the rounding of the code itself. sqrt(v) is stored instead
// of v because it halves the binades a block spans (E4M3 holds 17).
#include <new>
#include <algorithm>
#include <vector>

#include "pk_common.cuh"

namespace pk {
namespace {

constexpr int BLOCK = 32;          // elements per scale
constexpr int THREADS = 256;
constexpr int WIDE = THREADS * 4;  // elements of a CTA's pass: 4 per thread
// Passes of a full chunk, all loaded before the first is computed. Four keep enough bytes in flight
// for large plans; a plan that would not fill the GPU four CTAs deep that way takes chunks of one.
constexpr int MANY = 4;
constexpr uint64_t PLAN_MAGIC = 0x706b5f6164616d77ull;

// What a CTA needs: up to passes * WIDE consecutive elements of one tensor. A record per chunk rather than per
// tensor: the CTA's first loads are then one step from its data instead of two or a search.
struct Chunk {
    float* p;
    const void* g;
    void* m;
    void* v;
    uint8_t* ms;
    uint8_t* vs;
    bf16* shadow;
    int64_t number;       // number of the first element in the plan (tensors padded to BLOCK)
    float lr_mult, wd;
    int n;
    int vec;              // every buffer of the tensor allows the wide accesses
};

struct Plan {
    uint64_t magic;
    int device;
    int g_dtype, bits, passes;
    int64_t chunks;
    Chunk* dev;
};

// 32 random bits of element i under the step's key: two rounds of xor-shift and multiplication by
// odd constants (fractional bits of the golden ratio and of sqrt 3), enough to decorrelate
// neighbouring elements and steps, which is all that the rounding needs.
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t v) {
    v = (v ^ (v >> 16)) * 0x9E3779B1u;
    v = (v ^ (v >> 15)) * 0xBB67AE85u;
    return v ^ (v >> 16);
}
__device__ __forceinline__ uint32_t element_key(int64_t i) {
    return static_cast<uint32_t>(i) + 0x3C6EF372u * static_cast<uint32_t>(i >> 32);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// Exponent byte of a block whose largest finite magnitude is a: the power of two 2^(b - 127) with
// a / 2^(b - 127) in (224, 448], so that the largest value never saturates; at least 1.
__device__ __forceinline__ uint32_t scale_byte(float a) {
    const uint32_t u = __float_as_uint(a);
    const int b = static_cast<int>(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return static_cast<uint32_t>(b < 1 ? 1 : b);
}
__device__ __forceinline__ float pow2_of(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float inverse_of(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Four E4M3 codes to fp32 (exact) and back (to nearest even).
__device__ __forceinline__ void decode4(uint32_t c, float s, float (&f)[4]) {
    uint32_t lo, hi;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(c));
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
        : "=f"(f[0]), "=f"(f[1]) : "r"(lo));
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
        : "=f"(f[2]), "=f"(f[3]) : "r"(hi));
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] *= s;
}
__device__ __forceinline__ uint32_t encode4(const float (&f)[4]) {
    uint32_t c;
    asm("{\n\t.reg .b16 l, h;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(c) : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]));
    return c;
}

// x / 2^e with what is not finite turned into NaN (E4M3 has no infinity and would saturate).
__device__ __forceinline__ float scaled(float x, float inv) {
    return finite(x) ? x * inv : __int_as_float(0x7fffffff);
}
// The E4M3 neighbour of y >= 0 above or below, chosen with 20 random bits so that the mean is y. The
// codes from 2^-6 up are the floats whose low 20 mantissa bits are zero: adding the random bits
// and cutting them off rounds up with the right probability. Below 2^-6 the codes are 2^-9
// apart, as they are in [2^-6, 2^-5): there y is shifted up by 2^-6, cut, and shifted back.
constexpr float SMALLEST_NORMAL = 0.015625f, SMALLEST = 0.001953125f;  // 2^-6, 2^-9
__device__ __forceinline__ float cut_by_chance(float y, uint32_t rnd) {
    return __uint_as_float((__float_as_uint(y) + (rnd & 0xfffffu)) & 0xfff00000u);
}
__device__ __forceinline__ float round_by_chance(float y, uint32_t rnd, bool positive) {
    const bool low = y < SMALLEST_NORMAL;
    float r = cut_by_chance(low ? __fadd_rn(y, SMALLEST_NORMAL) : y, rnd);
    if (low) r -= SMALLEST_NORMAL;
    if (positive && r == 0.0f) r = SMALLEST;
    return y == y ? r : y;
}
__device__ __forceinline__ float round_root_nearest(float y, bool positive) {
    return positive && y < SMALLEST ? SMALLEST : y;
}

struct Step32 {
    float lr, b1, b2, eps, wd, c1, c2;
};

// One element with fp32 moments. The result has the bits of pk_adamw, whose wide and narrow loops
// the compiler contracts differently: which product of a moment's sum is rounded on its own is
// written out here for each (WIDE).
template <bool WIDE>
__device__ __forceinline__ void adamw_element(float& p, float g, float& m, float& v, const Step32& s) {
    const float omb1 = 1.0f - s.b1, omb2 = 1.0f - s.b2;
    const float g2 = __fmul_rn(omb2, g);
    if (WIDE) {
        m = __fmaf_rn(s.b1, m, __fmul_rn(omb1, g));
        v = __fmaf_rn(s.b2, v, __fmul_rn(g2, g));
    } else {
        m = __fmaf_rn(omb1, g, __fmul_rn(s.b1, m));
        v = __fmaf_rn(g2, g, __fmul_rn(s.b2, v));
    }
    const float upd = __fdiv_rn(__fdiv_rn(m, s.c1), __fadd_rn(__fsqrt_rn(__fdiv_rn(v, s.c2)), s.eps));
    p = __fmaf_rn(-s.lr, __fmaf_rn(s.wd, p, upd), p);
}

// sqrt(x) within half a unit of the last place and a hair: with q near 1 / sqrt(x) and s = x q, one step of Newton's
// iteration for s^2 = x, s + (x - s^2) / (2 s), where 1 / (2 s) is taken as q / 2. (The correctly rounded form takes 13 % of the kernel's time; the
// approximate one alone, two units off, moves one stored code in 10^5 to its neighbour.) Below the
// smallest normal number the approximation serves.
__device__ __forceinline__ float root(float x) {
    float q, low;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(x));
    asm("sqrt.approx.f32 %0, %1;" : "=f"(low) : "f"(x));
    const float s = __fmul_rn(x, q);
    const float r = __fmaf_rn(__fmaf_rn(-s, s, x), __fmul_rn(0.5f, q), s);
    return x >= 1.17549435e-38f && x <= 3.402823466e38f ? r : low;
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

struct Step8 {
    float lr, b1, b2, eps, ic1, isc2;  // ic1 = 1 / c1, isc2 = 1 / sqrt(c2)
    uint32_t key;
};

// One element with 8-bit moments: m and r = sqrt(v) in, both new ones out (fp32). With the root
// stored, one square root serves the state and the denominator: sqrt(v / c2) = r / sqrt(c2).
// Every product and sum of the moments is rounded on its own, as a program that writes the step out in fp32
// rounds them: the stored codes are that program's, and the wide and the narrow loop's the same. (With fused
// multiply-adds a third of the moments differs by its last bit, and of 243 M parameters some 300 get the
// neighbouring code and one to three blocks a scale twice as large; the time is the same, 808 and 809 us.)
__device__ __forceinline__ void adamw8_element(float& p, float g, float& m, float& r, const Step8& s, float wd) {
    m = __fadd_rn(__fmul_rn(s.b1, m), __fmul_rn(1.0f - s.b1, g));
    r = root(__fadd_rn(__fmul_rn(s.b2, __fmul_rn(r, r)), __fmul_rn(__fmul_rn(1.0f - s.b2, g), g)));
    const float upd = __fdividef(__fmul_rn(m, s.ic1), __fmaf_rn(r, s.isc2, s.eps));
    p = __fmaf_rn(-s.lr, __fmaf_rn(wd, p, upd), p);
}

// Four gradients as loaded, and their conversion.
template <typename G> struct Grad4;
template <> struct Grad4<float> {
    uint4 raw;
    __device__ __forceinline__ void load(const float* g) { raw = *reinterpret_cast<const uint4*>(g); }
    __device__ __forceinline__ void get(float (&f)[4]) const { Vec<float>::unpack(raw, f); }
};
template <> struct Grad4<bf16> {
    uint2 raw;
    __device__ __forceinline__ void load(const bf16* g) { raw = *reinterpret_cast<const uint2*>(g); }
    __device__ __forceinline__ void get(float (&f)[4]) const {
        f[0] = __uint_as_float(raw.x << 16);
        f[1] = __uint_as_float(raw.x & 0xffff0000u);
        f[2] = __uint_as_float(raw.y << 16);
        f[3] = __uint_as_float(raw.y & 0xffff0000u);
    }
};
__device__ __forceinline__ void store_shadow4(bf16* s, const float (&p)[4]) {
    __nv_bfloat162 h0 = __floats2bfloat162_rn(p[0], p[1]), h1 = __floats2bfloat162_rn(p[2], p[3]);
    uint2 w;
    w.x = *reinterpret_cast<uint32_t*>(&h0);
    w.y = *reinterpret_cast<uint32_t*>(&h1);
    *reinterpret_cast<uint2*>(s) = w;
}

// fp32 moments.
template <typename G>
__global__ void __launch_bounds__(THREADS)
adamw_multi32_kernel(const Chunk* __restrict__ chunks, Step32 s) {
    const Chunk c = chunks[blockIdx.x];
    s.lr *= c.lr_mult;
    s.wd = c.wd;
    float* m = static_cast<float*>(c.m);
    float* v = static_cast<float*>(c.v);
    const G* g = static_cast<const G*>(c.g);
    const int nv = c.vec ? c.n / 4 : 0;
    for (int i = threadIdx.x; i < nv; i += THREADS) {
        float pp[4], gg[4], mm[4], vv[4];
        Grad4<G> raw;
        Vec<float>::load(c.p + i * 4, pp);
        raw.load(g + i * 4);
        Vec<float>::load(m + i * 4, mm);
        Vec<float>::load(v + i * 4, vv);
        raw.get(gg);
#pragma unroll
        for (int e = 0; e < 4; ++e) adamw_element<true>(pp[e], gg[e], mm[e], vv[e], s);
        Vec<float>::store(c.p + i * 4, pp);
        Vec<float>::store(m + i * 4, mm);
        Vec<float>::store(v + i * 4, vv);
        if (c.shadow) store_shadow4(c.shadow + i * 4, pp);
    }
    for (int i = nv * 4 + threadIdx.x; i < c.n; i += THREADS) {
        float pi = c.p[i], mi = m[i], vi = v[i];
        adamw_element<false>(pi, to_f32(g[i]), mi, vi, s);
        c.p[i] = pi;
        m[i] = mi;
        v[i] = vi;
        if (c.shadow) c.shadow[i] = __float2bfloat16_rn(pi);
    }
}

// 8-bit moments. Wide part: a lane holds 4 consecutive elements, 8 lanes a block of 32; the rest (and
// tensors whose buffers are not aligned): a lane holds one element, a warp one block.
// A pass of the CTA moves 18 KB, so every load of the chunk is issued before the first pass is
// computed: with one pass in flight at a time the kernel waited for memory (24 % of the copy
// bandwidth, 27 % of the issue slots).
template <typename G>
struct Pass8 {
    float4 p;
    Grad4<G> g;
    uint32_t m, v;
    uint8_t ms, vs;
    __device__ __forceinline__ void load(const Chunk& c, int i) {
        p = *reinterpret_cast<const float4*>(c.p + i);
        g.load(static_cast<const G*>(c.g) + i);
        m = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(c.m) + i);
        v = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(c.v) + i);
        ms = c.ms[i / BLOCK];
        vs = c.vs[i / BLOCK];
    }
    // Called by whole warps: lanes of a block exchange their maxima.
    __device__ __forceinline__ void step(const Chunk& c, int i, const Step8& s) const {
        float pp[4] = {p.x, p.y, p.z, p.w}, gg[4], mm[4], vv[4];
        g.get(gg);
        decode4(m, pow2_of(ms), mm);
        decode4(v, pow2_of(vs), vv);
        uint32_t am = 0, av = 0;  // magnitudes compared as bits: NaN and infinity are the largest
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            adamw8_element(pp[e], gg[e], mm[e], vv[e], s, c.wd);
            am = max(am, __float_as_uint(mm[e]) & 0x7fffffffu);
            av = max(av, __float_as_uint(vv[e]) & 0x7fffffffu);
        }
        Vec<float>::store(c.p + i, pp);
        if (c.shadow) store_shadow4(c.shadow + i, pp);
        if (__any_sync(0xffffffffu, max(am, av) >= 0x7f800000u)) {  // rare: what is not finite becomes NaN and has no say
            am = av = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (finite(mm[e])) am = max(am, __float_as_uint(mm[e]) & 0x7fffffffu);
                else mm[e] = __int_as_float(0x7fffffff);
                if (finite(vv[e])) av = max(av, __float_as_uint(vv[e]) & 0x7fffffffu);
                else vv[e] = __int_as_float(0x7fffffff);
            }
        }
        // both maxima in one word, rounded up to their upper 16 bits: scale_byte asks for nothing below
        uint32_t top = ((am + 0xffffu) >> 16) | ((av + 0xffffu) & 0xffff0000u);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) top = max_u16x2(top, __shfl_xor_sync(0xffffffffu, top, o));
        const uint32_t bm = scale_byte(__uint_as_float(top << 16)), bv = scale_byte(__uint_as_float(top & 0xffff0000u));
        const float im = inverse_of(bm), iv = inverse_of(bv);
        const uint32_t k0 = element_key(c.number + i);
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            mm[e] *= im;
            y[e] = vv[e] * iv;
        }
        // every value of the warp at or above the smallest normal code: the plain cut
        if (__all_sync(0xffffffffu, fminf(fminf(y[0], y[1]), fminf(y[2], y[3])) >= SMALLEST_NORMAL && y[0] + y[1] + y[2] + y[3] < INFINITY)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) vv[e] = cut_by_chance(y[e], mix32((k0 + e) ^ s.key));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) vv[e] = round_by_chance(y[e], mix32((k0 + e) ^ s.key), vv[e] > 0.0f);
        }
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(c.m) + i) = encode4(mm);
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(c.v) + i) = encode4(vv);
        if ((threadIdx.x & 7) == 0) {
            c.ms[i / BLOCK] = static_cast<uint8_t>(bm);
            c.vs[i / BLOCK] = static_cast<uint8_t>(bv);
        }
    }
};

template <typename G, int PASSES>
__global__ void __launch_bounds__(THREADS, 3)
adamw_multi8_kernel(const Chunk* __restrict__ chunks, Step8 s) {
    const Chunk c = chunks[blockIdx.x];
    s.lr *= c.lr_mult;
    if (c.vec && c.n == PASSES * WIDE) {
        Pass8<G> pass[PASSES];
#pragma unroll
        for (int k = 0; k < PASSES; ++k) pass[k].load(c, k * WIDE + threadIdx.x * 4);
#pragma unroll
        for (int k = 0; k < PASSES; ++k) pass[k].step(c, k * WIDE + threadIdx.x * 4, s);
        return;
    }
    const int wide = c.vec ? c.n / 128 * 128 : 0;  // whole warps only: the shuffles take all lanes
    for (int i = threadIdx.x * 4; i < wide; i += WIDE) {
        Pass8<G> pass;
        pass.load(c, i);
        pass.step(c, i, s);
    }
    const int lane = threadIdx.x & 31;
    const G* g = static_cast<const G*>(c.g);
    uint8_t* m = static_cast<uint8_t*>(c.m);
    uint8_t* v = static_cast<uint8_t*>(c.v);
    for (int b = wide / BLOCK + (threadIdx.x >> 5); b * BLOCK < c.n; b += THREADS / 32) {
        const int i = b * BLOCK + lane;
        const bool in = i < c.n;
        float pp = 0.0f, mm[4] = {}, vv[4] = {};
        if (in) {
            pp = c.p[i];
            decode4(m[i], pow2_of(c.ms[b]), mm);
            decode4(v[i], pow2_of(c.vs[b]), vv);
            adamw8_element(pp, to_f32(g[i]), mm[0], vv[0], s, c.wd);
            c.p[i] = pp;
            if (c.shadow) c.shadow[i] = __float2bfloat16_rn(pp);
        }
        const uint32_t bm = scale_byte(warp_max(in && finite(mm[0]) ? fabsf(mm[0]) : 0.0f));
        const uint32_t bv = scale_byte(warp_max(in && finite(vv[0]) ? vv[0] : 0.0f));
        if (in) {
            const bool positive = vv[0] > 0.0f;
            const float cm[4] = {scaled(mm[0], inverse_of(bm)), 0.0f, 0.0f, 0.0f};
            const float cv[4] = {round_by_chance(scaled(vv[0], inverse_of(bv)), mix32(element_key(c.number + i) ^ s.key), positive),
                                 0.0f, 0.0f, 0.0f};
            m[i] = static_cast<uint8_t>(encode4(cm));
            v[i] = static_cast<uint8_t>(encode4(cv));
        }
        if (lane == 0) {  // after every lane has read the old scales: the shuffles above order it
            c.ms[b] = static_cast<uint8_t>(bm);
            c.vs[b] = static_cast<uint8_t>(bv);
        }
    }
}

// Conversions of whole moment tensors, a warp per block of 32.
__global__ void __launch_bounds__(THREADS)
moment_unpack_kernel(const uint8_t* __restrict__ c, const uint8_t* __restrict__ b, float* __restrict__ x, int64_t n, bool root) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * THREADS) {
        float f[4];
        decode4(c[i], pow2_of(b[i / BLOCK]), f);
        x[i] = root ? f[0] * f[0] : f[0];
    }
}
__global__ void __launch_bounds__(THREADS)
moment_pack_kernel(const float* __restrict__ x, uint8_t* __restrict__ c, uint8_t* __restrict__ b, int64_t n, bool root) {
    const int lane = threadIdx.x & 31;
    const int64_t blocks = (n + BLOCK - 1) / BLOCK;
    for (int64_t k = static_cast<int64_t>(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5); k < blocks;
         k += static_cast<int64_t>(gridDim.x) * (THREADS / 32)) {
        const int64_t i = k * BLOCK + lane;
        float f = i < n ? x[i] : 0.0f;
        if (root) f = sqrtf(f);
        const uint32_t e = scale_byte(warp_max(finite(f) ? fabsf(f) : 0.0f));
        float y = scaled(f, inverse_of(e));
        if (root) y = round_root_nearest(y, f > 0.0f);
        const float y4[4] = {y, 0.0f, 0.0f, 0.0f};
        if (i < n) c[i] = static_cast<uint8_t>(encode4(y4));
        if (lane == 0) b[k] = static_cast<uint8_t>(e);
    }
}

// A device buffer of the current GPU?
bool on_device(const void* p, int device) {
    cudaPointerAttributes a;
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    return (a.type == cudaMemoryTypeDevice || a.type == cudaMemoryTypeManaged) && a.device == device;
}

struct Range {
    uintptr_t lo, hi;
    bool written;
};

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" {

int pk_adamw_plan_create(const pk_adamw_tensor* tensors_h, int n_tensors, int g_dtype, int state_bits, void** plan_h) {
    PK_REQUIRE(plan_h != nullptr, "null pointer");
    *plan_h = nullptr;
    PK_REQUIRE(n_tensors >= 0 && (n_tensors == 0 || tensors_h), "bad tensor list");
    PK_REQUIRE(valid_dtype(g_dtype), "bad dtype");
    PK_REQUIRE(state_bits == 8 || state_bits == 32, "state_bits must be 8 or 32");
    const size_t gs = dtype_size(g_dtype), ss = state_bits == 8 ? 1 : 4;
    for (int t = 0; t < n_tensors; ++t) {  // what needs no GPU is checked first
        const pk_adamw_tensor& x = tensors_h[t];
        PK_REQUIRE(x.n >= 0 && x.n <= (int64_t(1) << 40), "bad element count");
        if (x.n == 0) continue;
        PK_REQUIRE(x.p && x.g && x.m && x.v, "null pointer");
        PK_REQUIRE(state_bits == 32 || (x.m_scale && x.v_scale), "8-bit moments need their scales");
        PK_REQUIRE((reinterpret_cast<uintptr_t>(x.p) & 3u) == 0 && (reinterpret_cast<uintptr_t>(x.g) & (gs - 1)) == 0 &&
                       (reinterpret_cast<uintptr_t>(x.m) & (ss - 1)) == 0 && (reinterpret_cast<uintptr_t>(x.v) & (ss - 1)) == 0 &&
                       (reinterpret_cast<uintptr_t>(x.shadow) & 1u) == 0,
                   "buffer not aligned to its type");
    }
    int device = 0;
    PK_CHECK_CUDA(cudaGetDevice(&device));
    try {
        int64_t large = 0;
        for (int t = 0; t < n_tensors; ++t) large += (tensors_h[t].n + MANY * WIDE - 1) / (MANY * WIDE);
        const int passes = large >= static_cast<int64_t>(sm_count()) * 4 ? MANY : 1, CHUNK = passes * WIDE;
        std::vector<Chunk> chunks;
        std::vector<Range> ranges;
        int64_t base = 0;
        for (int t = 0; t < n_tensors; ++t) {
            const pk_adamw_tensor& x = tensors_h[t];
            if (x.n == 0) continue;
            const size_t n = static_cast<size_t>(x.n), nb = (n + BLOCK - 1) / BLOCK;
            const struct { const void* p; size_t bytes; bool written; } bufs[] = {
                {x.p, n * 4, true}, {x.g, n * gs, false}, {x.m, n * ss, true}, {x.v, n * ss, true},
                {state_bits == 8 ? x.m_scale : nullptr, nb, true}, {state_bits == 8 ? x.v_scale : nullptr, nb, true},
                {x.shadow, n * 2, true}};
            for (const auto& b : bufs) {
                if (b.p == nullptr) continue;
                PK_REQUIRE(on_device(b.p, device), "a buffer is not in the current GPU's memory");
                const uintptr_t lo = reinterpret_cast<uintptr_t>(b.p);
                ranges.push_back({lo, lo + b.bytes, b.written});
            }
            const uintptr_t mask = 4 * ss - 1;
            const int vec = aligned16(x.p) && (reinterpret_cast<uintptr_t>(x.g) & (4 * gs - 1)) == 0 &&
                            (reinterpret_cast<uintptr_t>(x.m) & mask) == 0 && (reinterpret_cast<uintptr_t>(x.v) & mask) == 0 &&
                            (reinterpret_cast<uintptr_t>(x.shadow) & 7u) == 0;
            PK_REQUIRE(static_cast<int64_t>(chunks.size()) + (x.n + CHUNK - 1) / CHUNK <= 0x7fffffff, "too many elements");
            for (int64_t at = 0; at < x.n; at += CHUNK) {
                Chunk c{};
                c.p = x.p + at;
                c.g = static_cast<const char*>(x.g) + at * static_cast<int64_t>(gs);
                c.m = static_cast<char*>(x.m) + at * static_cast<int64_t>(ss);
                c.v = static_cast<char*>(x.v) + at * static_cast<int64_t>(ss);
                c.ms = x.m_scale ? x.m_scale + at / BLOCK : nullptr;
                c.vs = x.v_scale ? x.v_scale + at / BLOCK : nullptr;
                c.shadow = x.shadow ? static_cast<bf16*>(x.shadow) + at : nullptr;
                c.number = base + at;
                c.lr_mult = x.lr_mult;
                c.wd = x.weight_decay;
                c.n = static_cast<int>(std::min<int64_t>(CHUNK, x.n - at));
                c.vec = vec;
                chunks.push_back(c);
            }
            base += static_cast<int64_t>(nb) * BLOCK;
        }
        std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
        uintptr_t end_any = 0, end_written = 0;  // furthest ends seen so far
        for (const Range& r : ranges) {
            PK_REQUIRE(r.lo >= end_written && (!r.written || r.lo >= end_any), "a written buffer overlaps another one");
            end_any = std::max(end_any, r.hi);
            if (r.written) end_written = std::max(end_written, r.hi);
        }
        Plan* plan = new Plan{};
        plan->magic = PLAN_MAGIC;
        plan->device = device;
        plan->g_dtype = g_dtype;
        plan->bits = state_bits;
        plan->passes = passes;
        plan->chunks = static_cast<int64_t>(chunks.size());
        if (!chunks.empty()) {
            const size_t bytes = chunks.size() * sizeof(Chunk);
            void* dev = nullptr;
            cudaError_t e = cudaMalloc(&dev, bytes);
            if (e == cudaSuccess) e = cudaMemcpy(dev, chunks.data(), bytes, cudaMemcpyHostToDevice);
            // a copy from pageable memory may still be under way when the call returns, in order with the legacy
            // stream only: a step on a stream that does not wait for that one would read what was there before
            if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamLegacy);
            plan->dev = static_cast<Chunk*>(dev);
            if (e != cudaSuccess) {
                if (dev) cudaFree(dev);
                delete plan;
                set_error("%s: %s", __func__, cudaGetErrorString(e));
                return PK_ERR_CUDA;
            }
        }
        *plan_h = plan;
    } catch (const std::bad_alloc&) {
        set_error("%s: out of host memory", __func__);
        return PK_ERR_INVALID;
    }
    return PK_OK;
}

int pk_adamw_plan_destroy(void* plan_h) {
    if (plan_h == nullptr) return PK_OK;
    Plan* plan = static_cast<Plan*>(plan_h);
    PK_REQUIRE(plan->magic == PLAN_MAGIC, "not an AdamW plan");
    plan->magic = 0;
    void* dev = plan->dev;
    delete plan;
    if (dev) PK_CHECK_CUDA(cudaFree(dev));
    return PK_OK;
}

int pk_adamw_multi(void* stream, void* plan_h, float lr, float b1, float b2, float eps, float c1, float c2,
                   uint64_t seed) {
    const Plan* plan = static_cast<const Plan*>(plan_h);
    PK_REQUIRE(plan != nullptr && plan->magic == PLAN_MAGIC, "not an AdamW plan");
    PK_REQUIRE(c1 > 0.0f && c2 > 0.0f, "c1 and c2 must be positive");
    if (plan->chunks == 0) return PK_OK;
    int device = 0;
    PK_CHECK_CUDA(cudaGetDevice(&device));
    PK_REQUIRE(device == plan->device, "the plan's tensors are on another GPU than the current one");
    const unsigned grid = static_cast<unsigned>(plan->chunks);
    cudaStream_t st = as_stream(stream);
    if (plan->bits == 32) {
        const Step32 s = {lr, b1, b2, eps, 0.0f, c1, c2};
        if (plan->g_dtype == PK_F32) adamw_multi32_kernel<float><<<grid, THREADS, 0, st>>>(plan->dev, s);
        else adamw_multi32_kernel<bf16><<<grid, THREADS, 0, st>>>(plan->dev, s);
    } else {
        const uint32_t key = mix32(static_cast<uint32_t>(seed) + 0x632BE5ABu * static_cast<uint32_t>(seed >> 32));
        const Step8 s = {lr, b1, b2, eps, static_cast<float>(1.0 / c1), static_cast<float>(1.0 / sqrt(static_cast<double>(c2))), key};
        const bool f = plan->g_dtype == PK_F32;
        if (plan->passes == MANY) (f ? adamw_multi8_kernel<float, MANY> : adamw_multi8_kernel<bf16, MANY>)<<<grid, THREADS, 0, st>>>(plan->dev, s);
        else (f ? adamw_multi8_kernel<float, 1> : adamw_multi8_kernel<bf16, 1>)<<<grid, THREADS, 0, st>>>(plan->dev, s);
    }
    PK_LAUNCH_CHECK();
    return PK_OK;
}

int pk_adamw_moment_unpack(void* stream, const void* codes, const uint8_t* scales, float* x, int64_t n, int root) {
    PK_REQUIRE(n >= 0, "negative size");
    if (n == 0) return PK_OK;
    PK_REQUIRE(codes && scales && x, "null pointer");
    PK_REQUIRE(aligned_to(4, x), "buffer not aligned to its type");
    const int64_t blocks = std::min<int64_t>((n + THREADS - 1) / THREADS, static_cast<int64_t>(sm_count()) * 16);
    moment_unpack_kernel<<<static_cast<unsigned>(blocks), THREADS, 0, as_stream(stream)>>>(
        static_cast<const uint8_t*>(codes), scales, x, n, root != 0);
    PK_LAUNCH_CHECK();
    return PK_OK;
}

int pk_adamw_moment_pack(void* stream, const float* x, void* codes, uint8_t* scales, int64_t n, int root) {
    PK_REQUIRE(n >= 0, "negative size");
    if (n == 0) return PK_OK;
    PK_REQUIRE(x && codes && scales, "null pointer");
    PK_REQUIRE(aligned_to(4, x), "buffer not aligned to its type");
    const int64_t blocks = std::min<int64_t>((n + THREADS - 1) / THREADS, static_cast<int64_t>(sm_count()) * 16);
    moment_pack_kernel<<<static_cast<unsigned>(blocks), THREADS, 0, as_stream(stream)>>>(
        x, static_cast<uint8_t*>(codes), scales, n, root != 0);
    PK_LAUNCH_CHECK();
    return PK_OK;
}

}  // extern "C"
