"""Edges of the tuning operators on the GPU: stored codes bit by bit, rows and heads where a number runs out of its
range, gradients that sit differently from their logits. Tolerances as derived in tests/test_tuning_ops_gpu.py."""
import ctypes

import pytest
import torch

from paperkiln_b200 import _capi
from tests import pkt
from tests import test_tuning_ops_gpu as ops
from tests import tuning_ref as ref
from tests.pkt import dt, ptr, scratch, stream
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


# ---- q / k norms without an epsilon ------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(5, 3, 2, 64), (7, 14, 2, 64), (1, 1, 1, 2), (3, 5, 3, 96), (9, 6, 1, 34), (1027, 14, 2, 64), (1025, 3, 1, 80),
                                   (1501, 16, 2, 128)])
def test_gain_gradients_without_epsilon(pk, dtype, shape):  # noqa: F811
    """eps = 0 where a round of heads or a group of tokens is not full: places without a head add nothing to the gains'
    gradients."""
    T, Hq, Hkv, dk = shape
    n_pos, hs = 50, ops.half_step(dtype)
    q, gq = (torch.randn(T, Hq * dk, device="cuda", generator=gen(i)).to(dtype) for i in (1, 2))
    k, gk = (torch.randn(T, Hkv * dk, device="cuda", generator=gen(i)).to(dtype) for i in (3, 4))
    wq, wk = (1 + 0.3 * torch.randn(dk, device="cuda", generator=gen(i)) for i in (5, 6))
    pos = torch.randint(0, n_pos, (T,), device="cuda", generator=gen(7)).to(torch.int32)
    cs32 = ref.table(n_pos, dk, 1e4).float().cuda()
    oq, ok, dq, dk_ = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q), torch.empty_like(k)
    dwq, dwk = torch.zeros(dk, device="cuda"), torch.zeros(dk, device="cuda")
    buf = scratch(pk.pk_qk_norm_rope_bwd_scratch_bytes(T, Hq, Hkv, dk))
    lq, lk = Hq * dk, Hkv * dk
    pkt.check(pk.pk_qk_norm_rope_fwd(stream(), dt(q), ptr(q), lq, ptr(k), lk, ptr(wq), ptr(wk), ptr(oq), lq, ptr(ok), lk, T, Hq, Hkv, dk, Hq, Hkv,
                                     0.0, ptr(pos), ptr(cs32), n_pos))
    pkt.check(pk.pk_qk_norm_rope_bwd(stream(), dt(q), ptr(gq), lq, ptr(gk), lk, ptr(q), lq, ptr(k), lk, ptr(wq), ptr(wk), ptr(dq), lq, ptr(dk_), lk,
                                     ptr(dwq), ptr(dwk), ptr(buf), T, Hq, Hkv, dk, Hq, Hkv, 0.0, ptr(pos), ptr(cs32), n_pos))
    for x, g, w, H, y, dx, dw in ((q, gq, wq, Hq, oq, dq, dwq), (k, gk, wk, Hkv, ok, dk_, dwk)):
        want, size = ref.qk_forward(x.double(), w.double(), H, cs32.double(), pos.long(), H, 0.0, sizes=True)
        ops.within(y, want, hs * want.abs() + 2.0 ** -19 * size)
        want, wdw, (size, wsize) = ref.qk_backward(g.double(), x.double(), w.double(), H, cs32.double(), pos.long(), H, 0.0)
        ops.within(dx, want, hs * want.abs() + 2.0 ** -18 * size)
        ops.within(dw, wdw, 2.0 ** -17 * wsize + 4 * ops.U * wdw.abs())


# ---- gradients that sit differently from their logits ------------------------------------------

def raised(R, V, ld, offset, dtype, base, seed=0):
    """Logits around `base`, as far as the type holds them apart."""
    x, t = ops.make_logits(R, V, ld, offset, torch.float32, seed)
    _, y = ops.strided(R, V, ld, offset, dtype)
    y.copy_(x + base)
    return y, t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [519, 5003, 40000])
@pytest.mark.parametrize("base", [0.0, 12345.6, -1e5, 9e5, 3e6])
def test_policy_gradient_of_another_alignment(pk, dtype, V, base):  # noqa: F811
    """Where logits and gradient sit differently against 16 bytes the gradient has the bits that it has side by side, and
    is right, whatever the rows' size."""
    R, ld = 5, (V + 15) // 8 * 8
    x, t = raised(R, V, ld, 0, dtype, base)
    ti, adv = t.to(torch.int32), torch.randn(R, device="cuda", generator=gen(3))
    loss, got = torch.empty(R, device="cuda"), []
    for ldd, off in ((ld, 0), (ld + 3, 1), (V, 2)):
        buf, dx = ops.strided(R, V, ldd, off, dtype)
        pkt.check(pk.pk_policy_loss(stream(), dt(x), ptr(x), ld, ptr(ti), None, None, ptr(adv), None, 0.2, 0.2, 0.0, 1.0, ptr(loss), None, None,
                                    ptr(dx), ldd, R, V, None))
        got.append(dx.clone())
        outside = torch.ones_like(buf, dtype=torch.bool)
        outside[off:].as_strided((R, V), (ldd, 1))[:] = False
        assert bool((buf[outside] == 7).all())
    x64, g = x.double(), -adv.double()
    _, lse = ref.logprob(x64, t)
    want = ref.logprob_back(x64, t, lse, g)
    p = torch.exp(x64 - lse[:, None])
    lim = ops.half_step(dtype) * want.abs() + g.abs()[:, None] * (p * (2.0 ** -18 + 2.0 ** -21 * (x64 - lse[:, None]).abs()) + 2 * ops.U) + 1e-38
    for dx in got:
        ops.within(dx, want, lim)
        assert torch.equal(dx, got[0])


# ---- gradients of log-probabilities whose sum has few bits left --------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [37, 2056, 40000])
@pytest.mark.parametrize("R", [4, 3000])
def test_logprob_gradient_of_large_rows(pk, dtype, V, R):  # noqa: F811
    """exp(x - lse) with an lse of 24 bits is off by up to |lse| 2^-24, a row of the lowest value alone by a factor of V:
    such rows get their probabilities from the row itself. Few rows (several blocks to a row) and many, apart and in place."""
    if R > 4 and V > 10000:
        R = 700
    low = torch.finfo(dtype).min
    x, t = raised(R, V, V, 0, dtype, 0.0)
    for i, base in enumerate((1e5, -2e6, 300.0, -5000.0, 70.0, -60.0, 4e4, 0.0)):
        x[i::11] += base
    x[8::11] = low            # nothing but masked words: uniform
    x[0] = low
    x[1, 1::2] = low          # and some of a row's
    x[R - 1, ::3] = -float("inf")
    t[1] = 0
    t[R - 1] = 1
    ti, g = t.to(torch.int32), torch.randn(R, device="cuda", generator=gen(9))
    logp, lse = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    pkt.check(pk.pk_token_logprob(stream(), dt(x), ptr(x), V, ptr(ti), None, ptr(logp), ptr(lse), R, V, None))
    x64, g64 = x.double(), g.double()
    top = x64.amax(1, keepdim=True)
    e = torch.exp(x64 - top)
    p = e / e.sum(1, keepdim=True)
    want = -g64[:, None] * p
    want[torch.arange(R, device="cuda"), t] += g64
    far = (x64 - top).clamp(min=-1e4).abs() + torch.log(torch.tensor(float(V)))
    # below 64 (fp32) and 1024 (bf16) the lse serves as it is: half a step of it is 2^-18 (2^-14, of the rounding to come 2^-5)
    rel = 2.0 ** -17 + 2.0 ** -21 * far + (2.0 ** -18 if dtype == torch.float32 else 2.0 ** -14)
    lim = ops.half_step(dtype) * want.abs() + g64.abs()[:, None] * (p * rel + 2 * ops.U) + 1e-38
    dx = torch.full_like(x, 3.0)
    call = lambda out: pkt.check(pk.pk_token_logprob_bwd(stream(), dt(x), ptr(x), V, ptr(ti), ptr(lse), ptr(g), ptr(out), V, R, V, None))  # noqa: E731
    call(dx)
    ops.within(dx, want, lim)
    call(x)
    assert torch.equal(dx, x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logprob_gradient_under_a_sum_over_more_words(pk, dtype):  # noqa: F811
    """An lse that is not this row's own (the words of a row lie in two tensors, say) is taken as it is given."""
    R, V = 6, 1000
    x, t = raised(R, V, V, 0, dtype, 0.0)
    x += 3000.0
    ti, g = t.to(torch.int32), torch.randn(R, device="cuda", generator=gen(9))
    lse = (torch.logsumexp(x.double(), 1) + 1.5).float()
    dx = torch.empty_like(x)
    pkt.check(pk.pk_token_logprob_bwd(stream(), dt(x), ptr(x), V, ptr(ti), ptr(lse), ptr(g), ptr(dx), V, R, V, None))
    want = ref.logprob_back(x.double(), t, lse.double(), g.double())
    p = torch.exp(x.double() - lse.double()[:, None])
    far = (x.double() - lse.double()[:, None]).abs()
    ops.within(dx, want, ops.half_step(dtype) * want.abs() + g.double().abs()[:, None] * (p * (2.0 ** -18 + 2.0 ** -21 * far) + 2 * ops.U) + 1e-38)


# ---- terms of the policy loss that do not count ------------------------------------------------

def test_policy_terms_of_coefficient_zero(pk):  # noqa: F811
    """A KL coefficient of zero and an advantage of zero leave their terms out, also where e^u or the ratio passes the
    type's range (a reference or an old policy that had all but excluded the word): 0 * inf is no loss."""
    V = 64
    x = torch.randn(4, V, device="cuda", generator=gen(2))
    t = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    lp = ref.logprob(x.double(), t.long())[0].float()
    loss, kl, dx = torch.empty(4, device="cuda"), torch.empty(4, device="cuda"), torch.empty(4, V, device="cuda")

    def run(old, refp, adv, c):
        pkt.check(pk.pk_policy_loss(stream(), 0, ptr(x), V, ptr(t), ptr(old), ptr(refp), ptr(adv), None, 0.2, 0.2, c, 1.0, ptr(loss), None,
                                    ptr(kl), ptr(dx), V, 4, V, None))
        return loss.clone(), dx.clone()

    adv = torch.tensor([1.0, -1.0, 0.5, 0.0], device="cuda")
    want = run(lp, None, adv, 0.0)
    got = run(lp, lp + torch.tensor([100.0, 200.0, float("inf"), 1.0], device="cuda"), adv, 0.0)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert kl[:3].tolist() == [float("inf")] * 3   # still told
    # the ratio e^200 counts for nothing with an advantage of 0; the KL term does
    none = torch.zeros(4, device="cuda")
    a = run(lp - 200.0, lp + 0.1, none, 0.1)
    b = run(lp, lp + 0.1, none, 0.1)
    assert all(torch.equal(u, v) and bool(torch.isfinite(u).all()) for u, v in zip(a, b)) and bool((a[1] != 0).any())
    a = run(lp - 200.0, None, none, 0.0)
    assert not a[0].any() and not a[1].any()
    x[1, 5] = float("nan")   # a row that holds NaN stays one
    assert torch.isnan(run(lp, None, none, 0.0)[0]).tolist() == [False, True, False, False]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(37, 14, 2, 64), (130, 3, 1, 80), (1027, 16, 4, 128)])
def test_head_norm_gradients_over_the_inputs(pk, dtype, shape):  # noqa: F811
    """dq / dk written over q / k: the same bits as elsewhere."""
    T, Hq, Hkv, dk = shape
    lq, lk = Hq * dk, Hkv * dk
    q, gq = (torch.randn(T, lq, device="cuda", generator=gen(i)).to(dtype) for i in (1, 2))
    k, gk = (torch.randn(T, lk, device="cuda", generator=gen(i)).to(dtype) for i in (3, 4))
    w = 1 + 0.3 * torch.randn(dk, device="cuda", generator=gen(5))
    buf, got = scratch(pk.pk_qk_norm_rope_bwd_scratch_bytes(T, Hq, Hkv, dk)), []
    for a, b in ((torch.empty_like(q), torch.empty_like(k)), (q, k)):
        dw = torch.zeros(2, dk, device="cuda")
        pkt.check(pk.pk_qk_norm_rope_bwd(stream(), dt(q), ptr(gq), lq, ptr(gk), lk, ptr(q), lq, ptr(k), lk, ptr(w), ptr(w), ptr(a), lq, ptr(b), lk,
                                         ptr(dw[0]), ptr(dw[1]), ptr(buf), T, Hq, Hkv, dk, 0, 0, 1e-6, None, None, 0))
        got.append((a, b, dw))
    assert all(torch.equal(x, y) for x, y in zip(*got))


@pytest.mark.parametrize("root, first, last", [(0, 1, 246), (1, 65, 182)])
def test_every_stored_moment_survives_fp32(pk, root, first, last):  # noqa: F811
    """All codes under all scales through fp32 and back: the same values. For roots the scales whose smallest code is
    2^-71 and whose largest is below 2^64."""
    codes = torch.arange(128, device="cuda", dtype=torch.uint8) % 127   # no NaN
    scales = torch.arange(first, last + 1, device="cuda", dtype=torch.uint8)
    c, b = codes.repeat(scales.numel()), scales.repeat_interleave(4)
    if not root:
        c = c | (torch.arange(c.numel(), device="cuda") % 3 == 0).to(torch.uint8) * 128
    n = c.numel()
    x, c2, b2 = torch.empty(n, device="cuda"), torch.empty_like(c), torch.empty_like(b)
    pkt.check(pk.pk_adamw_moment_unpack(stream(), ptr(c), ptr(b), ptr(x), n, root))
    pkt.check(pk.pk_adamw_moment_pack(stream(), ptr(x), ptr(c2), ptr(b2), n, root))
    assert torch.equal(ops.decode(c2, b2), ops.decode(c, b))
