"""What the tuning operators promise to the hardware and to their callers, checked without a GPU: the upload of an optimizer
plan, loads of kernels that start early, row weights of the C++ operators."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest

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
