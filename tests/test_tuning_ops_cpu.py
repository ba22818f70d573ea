"""Refusals of the tuning operators (policy / preference losses, q / k norm with rotation, AdamW over
many tensors): arguments that the headers rule out are rejected before any CUDA call, and the 64-bit
formulas that the GPU tests compare with are checked against differences."""
import ctypes

import pytest
import torch

from paperkiln_b200 import _capi
from tests import tuning_ref as ref

P = ctypes.c_void_p(1 << 20)   # an address that nothing reads: every call below is refused first
Q = ctypes.c_void_p(1 << 30)


@pytest.fixture(scope="module")
def pk():
    return _capi.libpk()


def refused(pk, rc, word):
    assert rc == 1
    assert word in pk.pk_last_error()


def test_token_logprob_refusals(pk):
    f = pk.pk_token_logprob
    refused(pk, f(None, 5, P, 8, P, None, P, P, 1, 8, None), b"dtype")
    refused(pk, f(None, 0, P, 7, P, None, P, P, 1, 8, None), b"shape")       # ld < V
    refused(pk, f(None, 0, P, 8, P, None, P, P, -1, 8, None), b"shape")
    refused(pk, f(None, 0, P, 8, P, None, P, P, 1, 0, None), b"shape")
    refused(pk, f(None, 0, None, 8, P, None, P, P, 1, 8, None), b"null")
    refused(pk, f(None, 0, P, 8, P, None, P, None, 1, 8, None), b"null")
    assert f(None, 0, None, 8, None, None, None, None, 0, 8, None) == 0       # no rows
    b = pk.pk_token_logprob_bwd
    refused(pk, b(None, 0, P, 8, P, P, P, Q, 7, 1, 8, None), b"shape")
    refused(pk, b(None, 0, P, 8, P, P, P, None, 8, 1, 8, None), b"null")
    refused(pk, b(None, 0, P, 8, P, P, P, P, 9, 4, 8, None), b"overlaps")     # in place with another stride
    inside = ctypes.c_void_p((1 << 20) + 64)
    refused(pk, b(None, 0, P, 8, P, P, P, inside, 8, 4, 8, None), b"overlaps")
    assert b(None, 0, None, 8, None, None, None, None, 8, 0, 8, None) == 0


def test_more_rows_than_a_grid_holds(pk):
    R = 1 << 28
    refused(pk, pk.pk_token_logprob(None, 0, P, 8, P, None, P, P, R, 8, None), b"too many rows")
    refused(pk, pk.pk_policy_loss(None, 1, P, 8, P, None, None, P, None, 0.2, 0.2, 0.0, 1.0, P, None, None, None, 8, R, 8, None), b"too many rows")


def test_preference_refusals(pk):
    f = pk.pk_preference_loss
    refused(pk, f(None, P, P, None, P, -1, 4, 0.1, 0.0, 1.0, P, None, None, None), b"shape")
    refused(pk, f(None, P, P, None, P, 1, 4, 0.1, 1.5, 1.0, P, None, None, None), b"label_smoothing")
    refused(pk, f(None, P, P, None, P, 1, 4, 0.1, float("nan"), 1.0, P, None, None, None), b"label_smoothing")
    refused(pk, f(None, P, P, None, None, 1, 4, 0.1, 0.0, 1.0, P, None, None, None), b"null")
    refused(pk, f(None, None, P, None, P, 1, 4, 0.1, 0.0, 1.0, P, None, None, None), b"null")
    assert f(None, None, None, None, None, 0, 4, 0.1, 0.0, 1.0, None, None, None, None) == 0


def test_policy_refusals(pk):
    f = pk.pk_policy_loss

    def call(dtype=0, x=P, ld=8, t=P, adv=P, lo=0.2, hi=0.2, loss=P, dx=Q, ldd=8, R=4, V=8):
        return f(None, dtype, x, ld, t, None, None, adv, None, lo, hi, 0.0, 1.0, loss, None, None, dx, ldd, R, V, None)

    refused(pk, call(dtype=2), b"dtype")
    refused(pk, call(ld=7), b"shape")
    refused(pk, call(ldd=7), b"shape")
    refused(pk, call(lo=-0.1), b"clip")
    refused(pk, call(lo=1.1), b"clip")
    refused(pk, call(hi=float("nan")), b"clip")
    refused(pk, call(adv=None), b"null")
    refused(pk, call(loss=None), b"null")
    refused(pk, call(dx=P, ldd=16), b"overlaps")
    refused(pk, call(dx=ctypes.c_void_p((1 << 20) + 4)), b"overlaps")
    assert call(x=None, R=0) == 0


def test_qk_norm_rope_refusals(pk):
    f = pk.pk_qk_norm_rope_fwd

    def call(dtype=0, q=P, ldq=64, wq=P, qo=Q, ldqo=64, T=2, Hq=4, Hkv=2, dk=16, rq=4, rk=2, eps=1e-6, pos=P, cs=P, n_pos=8):
        return f(None, dtype, q, ldq, P, 32, wq, P, qo, ldqo, Q, 32, T, Hq, Hkv, dk, rq, rk, eps, pos, cs, n_pos)

    refused(pk, call(dtype=9), b"dtype")
    refused(pk, call(dk=15), b"head_dim")
    refused(pk, call(dk=258), b"head_dim")
    refused(pk, call(T=-1), b"negative")
    refused(pk, call(rq=5), b"rotated")
    refused(pk, call(eps=-1.0), b"eps")
    refused(pk, call(eps=float("nan")), b"eps")
    refused(pk, call(ldq=63), b"stride")
    refused(pk, call(wq=None), b"null")
    refused(pk, call(pos=None), b"table")
    refused(pk, call(n_pos=0), b"table")
    refused(pk, call(qo=P, ldqo=80), b"in place")
    assert call(T=0) == 0
    b = pk.pk_qk_norm_rope_bwd

    def back(dwq=P, dwk=Q, scratch=P, ldd=64):
        return b(None, 0, P, 64, P, 32, P, 64, P, 32, P, P, Q, ldd, Q, 32, dwq, dwk, scratch, 2, 4, 2, 16, 4, 2, 1e-6, P, P, 8)

    refused(pk, back(scratch=None), b"scratch")
    refused(pk, back(dwk=P), b"two buffers")
    refused(pk, back(ldd=60), b"stride")


def test_adamw_plan_refusals(pk):
    def make(n=64, bits=8, g_dtype=0, count=1, **other):
        f = dict(p=1 << 20, g=2 << 20, m=3 << 20, v=4 << 20, m_scale=5 << 20, v_scale=6 << 20, shadow=None, n=n, lr_mult=1.0,
                 weight_decay=0.0) | other
        table = (_capi.AdamwTensor * 1)(_capi.AdamwTensor(**f))
        h = ctypes.c_void_p()
        rc = pk.pk_adamw_plan_create(table, count, g_dtype, bits, ctypes.byref(h))
        assert not h.value or rc == 0
        return rc

    refused(pk, make(bits=16), b"state_bits")
    refused(pk, make(g_dtype=3), b"dtype")
    refused(pk, make(count=-1), b"list")
    refused(pk, make(n=-1), b"count")
    refused(pk, make(p=None), b"null")
    refused(pk, make(m_scale=None), b"scales")
    refused(pk, make(p=(1 << 20) + 2), b"aligned")
    refused(pk, make(bits=32, m=(3 << 20) + 1), b"aligned")
    refused(pk, make(g_dtype=1, g=(2 << 20) + 1), b"aligned")
    refused(pk, pk.pk_adamw_plan_create(None, 0, 0, 8, None), b"null")
    not_a_plan = (ctypes.c_uint64 * 16)()
    refused(pk, pk.pk_adamw_multi(None, ctypes.byref(not_a_plan), 1e-3, 0.9, 0.999, 1e-8, 0.1, 0.1, 0), b"not an AdamW plan")
    refused(pk, pk.pk_adamw_multi(None, None, 1e-3, 0.9, 0.999, 1e-8, 0.1, 0.1, 0), b"not an AdamW plan")
    assert pk.pk_adamw_plan_destroy(None) == 0
    refused(pk, pk.pk_adamw_moment_pack(None, P, None, P, 4, 0), b"null")
    refused(pk, pk.pk_adamw_moment_unpack(None, P, P, P, -4, 0), b"negative")


# ---- the formulas of the GPU tests against differences -----------------------------------------

def central(f, x, i, h=1e-6):
    a, b = x.clone(), x.clone()
    a.view(-1)[i] += h
    b.view(-1)[i] -= h
    return (f(a) - f(b)) / (2 * h)


def test_policy_formula_against_differences():
    g = torch.Generator().manual_seed(3)
    R, V = 6, 11
    x = torch.randn(R, V, generator=g, dtype=torch.float64)
    t = torch.randint(0, V, (R,), generator=g)
    lp = torch.log_softmax(x, 1)[torch.arange(R), t]
    kw = dict(old=lp + torch.tensor([0.0, 0.5, -0.5, 0.1, -0.1, 0.6]).double(), refp=lp + torch.randn(R, generator=g).double() * 0.3,
              adv=torch.tensor([1.0, 1.0, 1.0, -1.0, -1.0, -1.0]).double(), w=torch.tensor([1, 0.5, 1, 2, 0, 1]).double(),
              lo=0.8, hi=1.28, c=0.1)
    out = ref.policy(x, t, **kw)
    f = lambda z: float(ref.policy(z, t, **kw)["loss"].sum())  # noqa: E731
    for i in range(0, R * V):
        assert abs(central(f, x, i) - float(out["dx"].view(-1)[i])) < 1e-8


def test_preference_formula_against_differences():
    g = torch.Generator().manual_seed(4)
    R = 13
    logp, refp, w = (torch.randn(R, generator=g, dtype=torch.float64) for _ in range(3))
    seq = [0, 4, 4, 9, 12]
    kw = dict(refp=refp, w=w, seq=seq, beta=0.3, eps=0.1)
    out = ref.preference(logp, **kw)
    f = lambda z: float(ref.preference(z, **kw)["loss"].sum())  # noqa: E731
    for i in range(R):
        assert abs(central(f, logp, i) - float(out["dlogp"][i])) < 1e-8


def test_qk_norm_rope_formula_against_differences():
    g = torch.Generator().manual_seed(5)
    T, H, dk = 3, 2, 6
    x, dy = (torch.randn(T, H * dk, generator=g, dtype=torch.float64) for _ in range(2))
    w = torch.randn(dk, generator=g, dtype=torch.float64)
    cs = ref.table(5, dk, 100.0)
    pos = torch.tensor([0, 4, 2])
    y = lambda x_, w_: ref.qk_forward(x_, w_, H, cs, pos, H - 1, 1e-6)  # noqa: E731
    dx, dw, _ = ref.qk_backward(dy, x, w, H, cs, pos, H - 1, 1e-6)
    for i in range(T * H * dk):
        assert abs(central(lambda z: float((y(z, w) * dy).sum()), x, i) - float(dx.view(-1)[i])) < 1e-8
    for i in range(dk):
        assert abs(central(lambda z: float((y(x, z) * dy).sum()), w, i) - float(dw[i])) < 1e-8


def test_rounding_bits_are_spread():
    """The 20 bits that round a moment: uniform over elements, and independent of the next seed's."""
    i = torch.arange(1 << 16)
    a, b = ref.random_bits(i, 7).double() / 2 ** 20, ref.random_bits(i, 8).double() / 2 ** 20
    n = i.numel()
    # mean of n uniform numbers: sigma = 1 / sqrt(12 n); six sigma
    assert abs(float(a.mean()) - 0.5) < 6 / (12 * n) ** 0.5
    assert abs(float(((a - 0.5) * (b - 0.5)).mean())) < 6 / 12 / n ** 0.5
    assert abs(float(((a[1:] - 0.5) * (a[:-1] - 0.5)).mean())) < 6 / 12 / (n - 1) ** 0.5
