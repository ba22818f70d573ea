"""What the tuning operators promise to the hardware and to their callers, checked without a GPU: the upload of an optimizer
plan, loads of kernels that start early, row weights of the C++ operators, overlaps of the head norms."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

from paperkiln_b200 import _capi
from paperkiln_b200 import build as b

# A runtime without a GPU. A copy from pageable host memory returns when the data is staged, as the CUDA documentation
# has it: the bytes reach their destination with the next wait for the legacy stream (0 or 1) or the device.
RUNTIME = r'''
#include <cuda_runtime_api.h>
#include <cstdarg>
#include <cstdlib>
#include <cstring>
#include <vector>
struct Late { void* to; std::vector<char> data; };
static std::vector<Late> late;
static int live = 0, fail = 0;
extern "C" {
int test_late() { return static_cast<int>(late.size()); }
int test_live() { return live; }
void test_fail(int on) { fail = on; }
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "made by the test"; }
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes* a, const void*) {
    std::memset(a, 0, sizeof(*a));
    a->type = cudaMemoryTypeDevice;
    return cudaSuccess;
}
cudaError_t cudaMalloc(void** p, size_t n) { *p = std::calloc(1, n); ++live; return cudaSuccess; }
cudaError_t cudaFree(void* p) { std::free(p); --live; return cudaSuccess; }
static cudaError_t arrive() {
    if (fail) return cudaErrorUnknown;
    for (auto& c : late) std::memcpy(c.to, c.data.data(), c.data.size());
    late.clear();
    return cudaSuccess;
}
cudaError_t cudaMemcpy(void* to, const void* from, size_t n, cudaMemcpyKind) {
    const char* f = static_cast<const char*>(from);
    late.push_back({to, std::vector<char>(f, f + n)});
    return cudaSuccess;
}
cudaError_t cudaStreamSynchronize(cudaStream_t s) { return reinterpret_cast<size_t>(s) <= 1 ? arrive() : cudaSuccess; }
cudaError_t cudaDeviceSynchronize() { return arrive(); }
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { return cudaSuccess; }
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, cudaStream_t) { return 0; }
cudaError_t __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return cudaSuccess; }
void** __cudaRegisterFatBinary(void*) { static void* h = nullptr; return &h; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, void*, void*, void*, void*, int*) {}
}
namespace pk {
int sm_count() { return 148; }
void set_error(const char*, ...) {}
}
'''


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    """The optimizer's entries over that runtime, from this tree's source. (Bound to it, not to a runtime that another
    library of the process has brought.)"""
    at = tmp_path_factory.mktemp("plans")
    src, obj = b.CSRC / "pk_adamw_multi.cu", b.OBJ / "pk_adamw_multi.o"
    if not b._newer(obj, [src, *b.CSRC.glob("*.cuh"), *b.INCLUDE.glob("*.h")]):
        obj = at / "pk_adamw_multi.o"
        subprocess.run([b._nvcc(), "-ccbin", b._host_cxx(), *b.NVCC_FLAGS, "-c", str(src), "-o", str(obj)], check=True)
    (at / "runtime.cpp").write_text(RUNTIME)
    cuda = Path(b._nvcc()).resolve().parent.parent / "include"
    subprocess.run([b._host_cxx(), "-shared", "-fPIC", "-std=c++17", "-Wl,-Bsymbolic", "-I", str(cuda), "-o", str(at / "plans.so"), str(at / "runtime.cpp"),
                    str(obj)], check=True)
    return ctypes.CDLL(str(at / "plans.so"))


def table(count, n):
    return (_capi.AdamwTensor * count)(*[_capi.AdamwTensor(
        p=(i * 8 + 1) << 24, g=(i * 8 + 2) << 24, m=(i * 8 + 3) << 24, v=(i * 8 + 4) << 24, n=n, lr_mult=1.0, weight_decay=0.0)
        for i in range(count)])


@pytest.mark.parametrize("count, n", [(1, 5), (40, 300001)])
def test_a_plan_is_on_the_gpu_when_it_is_given_out(plans, count, n):
    """The step may follow at once, on a stream that waits for no other: nothing may still be under way."""
    h = ctypes.c_void_p()
    assert plans.pk_adamw_plan_create(table(count, n), count, 0, 32, ctypes.byref(h)) == 0 and h.value
    assert plans.test_late() == 0
    assert plans.test_live() == 1
    assert plans.pk_adamw_plan_destroy(h) == 0 and plans.test_live() == 0


def test_a_plan_whose_upload_fails_leaves_nothing(plans):
    h = ctypes.c_void_p()
    plans.test_fail(1)
    try:
        assert plans.pk_adamw_plan_create(table(2, 100), 2, 0, 32, ctypes.byref(h)) == 2 and not h.value
    finally:
        plans.test_fail(0)
    assert plans.test_live() == 0


def kernels(text):
    """(name, parameters, body) of every kernel of a source file, comments left out."""
    text = re.sub(r"//[^\n]*", "", text)
    for head in re.finditer(r"__global__", text):
        at = text.index("{", head.end())
        sign, depth, end = text[head.end():at], 0, at
        for end in range(at, len(text)):
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            if depth == 0:
                break
        name = re.findall(r"(\w+)\s*\((?!\()", re.sub(r"__launch_bounds__\s*\((?:[^()]|\([^()]*\))*\)", "", sign))[0]
        yield name, sign, text[at:end]


def test_kernels_that_start_early_read_coherently():
    """A kernel that is launched before its predecessor has ended lives while that one writes what it will read. `const
    __restrict__` parameters allow loads that are defined only for data that nobody writes in a kernel's lifetime."""
    early = []
    for src in sorted(b.CSRC.glob("*.cu")):
        for name, sign, body in kernels(src.read_text()):
            if "griddepcontrol.wait" in body or "after_predecessor" in body:
                early.append(name)
                assert "__restrict__" not in sign, (src.name, name)
                assert "__ldg" not in body and ".nc." not in body, (src.name, name)
    assert {"token_logprob_bwd_kernel", "sweep_kernel", "preference_loss_kernel", "qk_gain_grad_kernel"} <= set(early)


# ---- the C++ operators -------------------------------------------------------------------------

WEIGHTS = r'''
#include <cstdio>
#include <functional>
#include <stdexcept>
#include <string>
#include "microtorch/ops.hpp"
using namespace microtorch;
int main() {
    Var h = make_var(Matrix(5, 4, 0.5f), false), W = make_var(Matrix(4, 7, 0.5f), false);
    const std::vector<int> targets = {1, 2, -100, 3, -100};
    const std::vector<float> rows(5, 1.0f), few(2, 1.0f), many(6, 0.0f);
    ops::PolicyTerms policy;
    ops::PreferenceTerms pref;
    policy.advantage = rows;
    pref.seq = {0, 2, 5};
    int bad = 0;
    for (const auto& w : {few, many}) {
        policy.weight = pref.weight = w;
        const std::function<void()> calls[] = {[&] { ops::linear_token_logprob(h, W, false, targets, w); },
                                               [&] { ops::linear_policy_loss(h, W, false, targets, policy); },
                                               [&] { ops::linear_preference_loss(h, W, false, targets, pref); }};
        for (const auto& call : calls) {
            std::string said = "nothing";
            try { call(); } catch (const std::exception& e) { said = e.what(); }
            if (said.find("one weight per row") == std::string::npos) { std::printf("%zu weights: %s\n", w.size(), said.c_str()); ++bad; }
        }
    }
    return bad;
}
'''


def test_weights_of_another_length_are_refused_before_they_are_read(tmp_path):
    (tmp_path / "weights.cpp").write_text(WEIGHTS)
    exe = tmp_path / "weights"
    subprocess.run([b._host_cxx(), "-O1", "-std=c++17", "-I", str(b.INCLUDE), "-I", str(b.HOST / "include"), str(tmp_path / "weights.cpp"), "-o",
                    str(exe), "-L", str(b.PKG), "-lmicrotorch", "-lpk", f"-Wl,-rpath,{b.PKG}"], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


# ---- overlaps of the head norms ----------------------------------------------------------------

BASE, FAR = 1 << 20, 1 << 30   # addresses that nothing reads: every call below is refused, or has no GPU to run on


def address(base, elements, size):
    return ctypes.c_void_p(base + elements * size)


@pytest.fixture(scope="module")
def pk():
    return _capi.libpk()


def forward(pk, q, k, qo, ko, size=4, T=3, Hq=4, Hkv=2, dk=16):
    """q, k, qo, ko: (base, first element, row stride). True when the call is refused for an overlap."""
    at = [(address(base, first, size), ld) for base, first, ld in (q, k, qo, ko)]
    w = ctypes.c_void_p(FAR * 3)
    rc = pk.pk_qk_norm_rope_fwd(None, 0 if size == 4 else 1, *at[0], *at[1], w, w, *at[2], *at[3], T, Hq, Hkv, dk, 0, 0, 1e-6, None, None, 0)
    assert rc != 0   # no GPU here
    return rc == 1 and b"overlap" in pk.pk_last_error()


def backward(pk, dqo, dko, q, k, dq, dk_, size=4, T=3):
    at = [(address(base, first, size), ld) for base, first, ld in (dqo, dko, q, k, dq, dk_)]
    w = ctypes.c_void_p(FAR * 3)
    rc = pk.pk_qk_norm_rope_bwd(None, 0 if size == 4 else 1, *at[0], *at[1], *at[2], *at[3], w, w, *at[4], *at[5], None, None, None, T, 4, 2, 16, 0, 0,
                                1e-6, None, None, 0)
    assert rc != 0
    return rc == 1 and b"overlap" in pk.pk_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls that are let through name addresses without memory")
@pytest.mark.parametrize("size", [2, 4])
def test_head_norms_refuse_outputs_inside_their_inputs(pk, size):
    q, k, qo, ko = (BASE, 0, 64), (2 * BASE, 0, 32), (FAR, 0, 64), (FAR + BASE, 0, 32)
    f = lambda **o: forward(pk, **({"q": q, "k": k, "qo": qo, "ko": ko} | o), size=size)  # noqa: E731
    assert not f()
    assert not f(qo=q, ko=k)                                   # in place
    assert not f(qo=q) and not f(ko=k)
    assert f(qo=(BASE, 16, 64))                                # one head on: another team reads what this one writes
    assert f(qo=(BASE, 64, 64))                                # one row on
    assert f(qo=(BASE, 2 * 64 + 63, 64))                       # the last element of q alone
    assert not f(qo=(BASE, 3 * 64, 64))                        # right behind it
    assert f(qo=(2 * BASE, 0, 64)) and f(ko=q)                 # over the other kind
    assert f(ko=(FAR, 48, 32))                                 # the outputs over each other
    # column ranges of one packed projection: q | k | free, rows of 160
    q, k = (BASE, 0, 160), (BASE, 64, 160)
    g = lambda **o: forward(pk, **({"q": q, "k": k, "qo": qo, "ko": ko} | o), size=size)  # noqa: E731
    assert not g() and not g(qo=q, ko=k)
    assert not g(qo=(BASE, 96, 160)) and not g(ko=(BASE, 96, 160))
    assert g(qo=(BASE, 97, 160))                               # reaches the next row's queries
    assert g(qo=(BASE, 95, 160))                               # starts at the keys' end
    assert not g(qo=(BASE, 160 + 96, 160))                     # a row further down the same columns
    assert g(ko=(BASE, 160 + 80, 160))
    # rows of another stride: apart when the columns are, in the strides' common measure
    assert not g(qo=(BASE, 96, 320)) and g(qo=(BASE, 90, 320)) and g(qo=(BASE, 96, 176))
    assert not forward(pk, (BASE, 0, 64), (2 * BASE, 0, 32), (BASE, 64, 80), ko, size=size, T=1)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls that are let through name addresses without memory")
@pytest.mark.parametrize("size", [2, 4])
def test_head_norm_gradients_refuse_outputs_inside_their_inputs(pk, size):
    at = {"dqo": (BASE, 0, 64), "dko": (2 * BASE, 0, 32), "q": (3 * BASE, 0, 64), "k": (4 * BASE, 0, 32), "dq": (FAR, 0, 64),
          "dk_": (FAR + BASE, 0, 32)}
    f = lambda **o: backward(pk, **(at | o), size=size)  # noqa: E731
    assert not f() and not f(dq=at["dqo"], dk_=at["dko"])
    assert not f(dq=at["q"], dk_=at["k"])                      # every thread reads its elements before it writes them
    assert f(dq=(BASE, 16, 64)) and f(dq=(3 * BASE, 16, 64)) and f(dk_=(2 * BASE, 32, 32)) and f(dk_=(4 * BASE, 1, 32))
    assert f(dq=(4 * BASE, 0, 64)) and f(dk_=at["dqo"]) and f(dk_=at["q"]) and f(dk_=(FAR, 0, 64))
    packed = {"dqo": (BASE, 0, 160), "dko": (BASE, 64, 160), "dq": (BASE, 0, 160), "dk_": (BASE, 64, 160)}
    assert not f(**packed) and not f(**(packed | {"dk_": (BASE, 96, 160)})) and f(**(packed | {"dk_": (BASE, 60, 160)}))


# ---- addresses that no element of the type can have --------------------------------------------

@pytest.mark.skipif(torch.cuda.is_available(), reason="names addresses without memory")
def test_buffers_off_their_type_are_refused(pk):
    """Rows may start at any element, but not between two bytes of one: the kernels' loads would fault."""
    P = [ctypes.c_void_p((i + 1) << 26) for i in range(20)]
    odd = lambda p, n: ctypes.c_void_p(p.value + n)  # noqa: E731

    def each(call, args, sizes):
        """call(*args) gets as far as the GPU; with any one buffer (sizes: {index: bytes of an element}) moved it is refused."""
        assert call(*args) == 2
        for i, size in sizes.items():
            for off in (1, 2) if size == 4 else (1,):
                moved = list(args)
                moved[i] = odd(args[i], off)
                assert call(*moved) == 1 and b"aligned" in pk.pk_last_error(), (i, off)

    for dtype, es in ((0, 4), (1, 2)):
        each(pk.pk_token_logprob, [None, dtype, P[0], 8, P[1], P[2], P[3], P[4], 2, 8, P[5]], {2: es, 4: 4, 5: 4, 6: 4, 7: 4, 10: 4})
        each(pk.pk_token_logprob_bwd, [None, dtype, P[0], 8, P[1], P[2], P[3], P[4], 8, 2, 8, P[5]], {2: es, 4: 4, 5: 4, 6: 4, 7: es, 11: 4})
        each(pk.pk_policy_loss, [None, dtype, P[0], 8, P[1], P[2], P[3], P[4], P[5], 0.2, 0.2, 0.1, 1.0, P[6], P[7], P[8], P[9], 8, 2, 8, P[10]],
             {2: es, 4: 4, 5: 4, 6: 4, 7: 4, 8: 4, 13: 4, 14: 4, 15: 4, 16: es, 20: 4})
        each(pk.pk_qk_norm_rope_fwd, [None, dtype, P[0], 64, P[1], 32, P[2], P[3], P[4], 64, P[5], 32, 3, 4, 2, 16, 4, 2, 1e-6, P[6], P[7], 8],
             {2: es, 4: es, 6: 4, 7: 4, 8: es, 10: es, 19: 4, 20: 4})
        each(pk.pk_qk_norm_rope_bwd, [None, dtype, P[0], 64, P[1], 32, P[2], 64, P[3], 32, P[4], P[5], P[6], 64, P[7], 32, P[8], P[9], P[10], 3, 4, 2, 16,
                                      4, 2, 1e-6, P[11], P[12], 8],
             {2: es, 4: es, 6: es, 8: es, 10: 4, 11: 4, 12: es, 14: es, 16: 4, 17: 4, 18: 4, 26: 4, 27: 4})
    each(pk.pk_preference_loss, [None, P[0], P[1], P[2], P[3], 1, 4, 0.1, 0.0, 1.0, P[4], P[5], P[6], P[7]], {1: 4, 2: 4, 3: 4, 4: 4, 10: 4, 11: 4, 12: 4, 13: 4})
    each(pk.pk_adamw_moment_unpack, [None, P[0], P[1], P[2], 4, 0], {3: 4})
    each(pk.pk_adamw_moment_pack, [None, P[0], P[1], P[2], 4, 0], {1: 4})
