"""Edges of the tuning operators on the GPU: stored codes bit by bit, rows and heads where a number runs out of its
range, gradients that sit differently from their logits. Tolerances as derived in tests/test_tuning_ops_gpu.py."""
import ctypes

import pytest
import torch

from paperkiln_b200 import _capi
from tests import pkt
from tests import test_tuning_ops_gpu as ops
from tests import tuning_ref as ref
from tests.pkt import ptr, stream
from tests.test_tuning_ops_gpu import HYPER, Many, f32, gen, pk  # noqa: F401

pytestmark = pytest.mark.gpu


def to_codes(x, bits=None):
    """E4M3 codes (as bytes) and scale bytes of x [n], fp32, to the nearest or by the chance of `bits`."""
    n = x.numel()
    x = torch.nn.functional.pad(x, (0, -n % 32))
    f, e = torch.frexp(x.abs().view(-1, 32).amax(1))
    b = torch.where(f > 0.875, e - 8, e - 9) + 127
    b = torch.where(f == 0, torch.ones_like(b), b.clamp(1, 254))
    y = x * torch.ldexp(torch.ones_like(f), 127 - b).repeat_interleave(32)
    if bits is not None:
        low = y < 2.0 ** -6
        z = torch.where(low, y + 2.0 ** -6, y)
        z = ((z.view(torch.int32) + torch.nn.functional.pad(bits, (0, -n % 32)).int()) & ~0xFFFFF).view(torch.float32)
        z = torch.where(low, z - 2.0 ** -6, z)
        y = torch.where((x > 0) & (z == 0), torch.full_like(z, 2.0 ** -9), z)
    return y[:n].to(torch.float8_e4m3fn).view(torch.uint8), b.to(torch.uint8)


@pytest.mark.parametrize("g_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])
def test_stored_codes_are_those_of_the_step_in_fp32(pk, g_dtype, shift):  # noqa: F811
    """m and v are each product and sum rounded to fp32 on its own, as written: a rounding left out would move a value
    in three by its last bit, and of those one in 2^20 to another code, that is several here. (The root under the
    codes of v is off its correctly rounded value in fewer than one of 2^20, so fewer than one of 2^40 codes by it.)"""
    sizes = [(1 << 24) + 77, 4096 * 5, 33]
    s = Many(sizes, 8, g_dtype, shift=shift, seed=6)
    b1, b2, seed, base = f32(HYPER["b1"]), f32(HYPER["b2"]), 31, 0
    before = [[ops.decode(c, b).float() for c, b in ((s.m[i], s.ms[i]), (s.v[i], s.vs[i]))] for i in range(len(sizes))]
    s.step(seed=seed)
    for i, n in enumerate(sizes):
        (m, r), g = before[i], s.g[i].float()
        m = b1 * m + (1 - b1) * g
        v = b2 * (r * r) + (1 - b2) * g * g
        bits = ref.random_bits(torch.arange(n, device="cuda") + base, seed)
        base += -(-n // 32) * 32
        for what, (c, b), got_c, got_b in (("m", to_codes(m), s.m[i], s.ms[i]), ("v", to_codes(torch.sqrt(v), bits), s.v[i], s.vs[i])):
            assert torch.equal(b, got_b), what
            assert int((c != got_c).sum()) == 0, (what, n, int((c != got_c).sum()))


def test_a_step_right_behind_its_plan_on_a_stream_of_its_own(pk):  # noqa: F811
    """A table of several megabytes, and the step at once on a stream that waits for no other."""
    count, n = 60000, 32
    side = torch.cuda.Stream()
    p0, g, m0, v0 = (torch.randn(count * n, device="cuda", generator=gen(i)) for i in range(4))
    v0 = v0.square()
    want = [t.clone() for t in (p0, m0, v0)]
    pkt.check(pk.pk_adamw(stream(), ptr(want[0]), ptr(g), ptr(want[1]), ptr(want[2]), count * n, 1e-3, 0.9, 0.999, 1e-8, 0.1, 0.2, 0.01, None))
    for _ in range(4):
        p, m, v = p0.clone(), m0.clone(), v0.clone()
        tensors = [_capi.AdamwTensor(p=p.data_ptr() + 4 * a, g=g.data_ptr() + 4 * a, m=m.data_ptr() + 4 * a, v=v.data_ptr() + 4 * a, n=n,
                                     lr_mult=1.0, weight_decay=0.1) for a in range(0, count * n, n)]
        torch.cuda.synchronize()
        plan = _capi.AdamwPlan(tensors, 0, 32)
        pkt.check(pk.pk_adamw_multi(ctypes.c_void_p(side.cuda_stream), plan.handle, 1e-3, 0.9, 0.999, 1e-8, 0.2, 0.01, 1))
        side.synchronize()
        plan.close()
        assert all(torch.equal(a, b) for a, b in zip((p, m, v), want))
