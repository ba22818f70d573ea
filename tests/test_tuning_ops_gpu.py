"""Tuning operators on the GPU against 64-bit restatements (tests/tuning_ref.py).

Tolerances, from the kernels' arithmetic (u = 2^-24, one fp32 rounding):
  log-probabilities  an exponential has relative error 2^-22 (ex2.approx) plus that of its argument
      d = x - M, rounded twice: |d| 2^-23, weighted by e^-|d| <= 1; a sum takes at most 64 additions in
      a chain at the sizes here: 2^-18 relative in all, which is 2^-18 absolute in the logarithm; the
      differences that form logp and lse round at most four times at |x_t| + |lse| + |logp|.
  gradients          p (2^-18 + 2^-21 |x - lse|) relative from p, what the row's g carries, one
      rounding to the stored type (half a step: finfo.eps / 2).
  heads' norms       a sum of dk squares in a tree (under 16 roundings), rsqrt.approx 2^-22, the two
      products: 2^-19 relative on each term of a rotated pair.
  8-bit moments      E4M3: to nearest 2^-4 relative or 2^-10 of the scale, by chance twice that.
"""
import ctypes

import pytest
import torch

from paperkiln_b200 import _capi
from tests import pkt
from tests import tuning_ref as ref
from tests.pkt import dt, ptr, scratch, stream

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def pk():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return _capi.libpk()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(a, b, tol):
    a, b = a.double(), b.double()
    bad = ~((a - b).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} off, worst {float(((a - b).abs() - tol).max()):.3e} over its limit"


def half_step(t):
    return torch.finfo(t).eps / 2


def status_word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def strided(R, V, ld, offset, dtype):
    """A [R, V] window with row stride ld that starts `offset` elements into its buffer."""
    buf = torch.full((offset + (R - 1) * ld + V + 16,), 7.0, dtype=dtype, device="cuda")
    return buf, buf[offset:].as_strided((R, V), (ld, 1))


def make_logits(R, V, ld, offset, dtype, seed=0, spread=3.0):
    buf, x = strided(R, V, ld, offset, dtype)
    x.copy_(torch.randn(R, V, device="cuda", generator=gen(seed)) * spread)
    t = torch.randint(0, V, (R,), device="cuda", generator=gen(seed + 1))
    x[torch.arange(R, device="cuda"), t] += 4
    return x, t


# rows, words, row stride, first element: short and long rows, odd lengths, every alignment
LOGITS = [(1, 1, 1, 0), (3, 5, 5, 0), (2, 8, 8, 0), (5, 37, 40, 3), (67, 133, 133, 1), (9, 1000, 1024, 0), (4, 4099, 4099, 5),
          (300, 2048, 2048, 0), (3, 50257, 50264, 0), (2, 50257, 50257, 1), (2, 151936, 151936, 0), (1, 300001, 300001, 0),
          (700, 515, 515, 0)]


def lp_tol(x64, t, logp, lse):
    xt = x64[torch.arange(x64.shape[0], device=x64.device), t]
    return 2.0 ** -18 + 4 * U * (xt.abs() + lse.abs() + logp.abs())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", LOGITS)
def test_token_logprob_and_gradient(pk, dtype, shape):
    R, V, ld, off = shape
    x, t = make_logits(R, V, ld, off, dtype)
    x64 = x.double()
    w = torch.ones(R, device="cuda")
    if R > 2:
        w[1::3] = 0
        x[1::3] = float("nan")  # rows that do not count hold anything
        x64[1::3] = 0
    ti = t.to(torch.int32)
    ti[w == 0] = -100
    live = w != 0
    logp, lse = torch.full((R,), 9.0, device="cuda"), torch.full((R,), 9.0, device="cuda")
    st = status_word()
    pkt.check(pk.pk_token_logprob(stream(), dt(x), ptr(x), ld, ptr(ti), ptr(w), ptr(logp), ptr(lse), R, V, ptr(st)))
    elogp, else_ = ref.logprob(x64, t)
    tol = lp_tol(x64, t, elogp, else_)
    within(logp[live], elogp[live], tol[live])
    within(lse[live], else_[live], tol[live])
    assert bool((logp[~live] == 0).all()) and bool((lse[~live] == 0).all()) and int(st) == 0

    g = torch.randn(R, device="cuda", generator=gen(5)) * live
    for same_place in (False, True):
        _, dx = strided(R, V, ld, off, dtype) if not same_place else (None, x)
        pkt.check(pk.pk_token_logprob_bwd(stream(), dt(x), ptr(x), ld, ptr(ti), ptr(lse), ptr(g), ptr(dx), ld, R, V, ptr(st)))
        want = ref.logprob_back(x64, t, else_, g.double())
        p = torch.exp(x64 - else_[:, None])
        rel = 2.0 ** -18 + 2.0 ** -21 * (x64 - else_[:, None]).abs() + (4 * U * else_.abs())[:, None]
        lim = half_step(dtype) * want.abs() + g.double().abs()[:, None] * (p * rel + 2 * U) + 1e-38
        within(dx[live], want[live], lim[live])
        assert bool((dx[~live] == 0).all()) and int(st) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_of_another_stride(pk, dtype):
    """logits and dlogits whose rows sit differently against 16 bytes; what lies between rows stays."""
    R, V, ld, ldd = 6, 519, 520, 523
    x, t = make_logits(R, V, ld, 0, dtype)
    buf, dx = strided(R, V, ldd, 1, dtype)
    ti, g = t.to(torch.int32), torch.randn(R, device="cuda", generator=gen(9))
    logp, lse = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    pkt.check(pk.pk_token_logprob(stream(), dt(x), ptr(x), ld, ptr(ti), None, ptr(logp), ptr(lse), R, V, None))
    pkt.check(pk.pk_token_logprob_bwd(stream(), dt(x), ptr(x), ld, ptr(ti), ptr(lse), ptr(g), ptr(dx), ldd, R, V, None))
    x64 = x.double()
    _, else_ = ref.logprob(x64, t)
    want = ref.logprob_back(x64, t, else_, g.double())
    p = torch.exp(x64 - else_[:, None])
    within(dx, want, half_step(dtype) * want.abs() + g.double().abs()[:, None] * (p * 2.0 ** -16 + 2 * U) + 1e-38)
    outside = torch.ones_like(buf, dtype=torch.bool)
    outside[1:].as_strided((R, V), (ldd, 1))[:] = False
    assert bool((buf[outside] == 7).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [40, 2056, 40000])
def test_masked_words_and_odd_rows(pk, dtype, V):
    """-inf and the type's lowest value mask words; a row of the lowest value alone is uniform; a row of
    -inf alone, or with NaN or +inf, is NaN and says nothing about its neighbours."""
    low = torch.finfo(dtype).min
    x = torch.randn(7, V, device="cuda", generator=gen(1)).to(dtype)
    x[0, 1::2] = -float("inf")
    x[1, 1::2] = low
    x[2] = low
    x[3] = -float("inf")
    x[4, 3] = float("nan")
    x[5, 3] = float("inf")
    t = torch.zeros(7, dtype=torch.int32, device="cuda")
    logp, lse = torch.empty(7, device="cuda"), torch.empty(7, device="cuda")
    pkt.check(pk.pk_token_logprob(stream(), dt(x), ptr(x), V, ptr(t), None, ptr(logp), ptr(lse), 7, V, None))
    x64 = x.double()
    el, es = ref.logprob(x64, t.long())
    for i in (0, 1, 6):
        within(logp[i], el[i], 2.0 ** -17)
        within(lse[i], es[i], 2.0 ** -17)
    within(logp[2], -torch.log(torch.tensor(float(V), dtype=torch.float64)), 2.0 ** -17)
    assert bool(torch.isnan(logp[3:6]).all())
    dx = torch.empty_like(x)
    old, adv, loss = logp.clone(), torch.ones(7, device="cuda"), torch.empty(7, device="cuda")
    old[3:6] = 0
    pkt.check(pk.pk_policy_loss(stream(), dt(x), ptr(x), V, ptr(t), ptr(old), None, ptr(adv), None, 0.2, 0.2, 0.0, 1.0, ptr(loss),
                                None, None, ptr(dx), V, 7, V, None))
    assert bool((dx[0, 1::2] == 0).all()) and bool((dx[1, 1::2] == 0).all())
    within(dx[2, 1:], torch.full((V - 1,), 1.0 / V, dtype=torch.float64, device="cuda"), half_step(dtype) / V + 2.0 ** -17 / V)
    assert bool(torch.isnan(dx[3:6]).any(1).all()) and bool(torch.isnan(loss[3:6]).all())
    assert bool(torch.isfinite(dx[6]).all()) and bool(torch.isfinite(loss[[0, 1, 2, 6]]).all())


def policy_inputs(R, seed, logp):
    g = gen(seed)
    d = torch.randn(R, device="cuda", generator=g) * 0.3
    for b in (0.8, 1.28):  # the gradient jumps on a bound
        b = torch.tensor(b).log().item()
        d = torch.where((d - b).abs() < 1e-3, torch.full_like(d, b + 2e-3), d)
    old = (logp - d).float()
    return old, (logp + torch.randn(R, device="cuda", generator=g) * 0.4).float(), torch.randn(R, device="cuda", generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", LOGITS)
@pytest.mark.parametrize("form", ["all", "on policy", "no kl", "forward"])
def test_policy_loss(pk, dtype, shape, form):
    R, V, ld, off = shape
    x, t = make_logits(R, V, ld, off, dtype)
    x64 = x.double()
    e0, _ = ref.logprob(x64, t)
    old, refp, adv = policy_inputs(R, 11, e0)
    w = torch.rand(R, device="cuda", generator=gen(12)) + 0.5
    ti = t.to(torch.int32)
    if R > 2:
        w[2::4] = 0
        ti[2::4] = -100
        x[2::4] = float("inf")
        x64[2::4] = 0
    if form == "on policy":
        old = None
    if form == "no kl":
        refp = None
    c, gs = 0.05, 0.5
    lo, hi = float(1 - torch.tensor(0.2)), float(1 + torch.tensor(0.28))
    want = ref.policy(x64, t, None if old is None else old.double(), None if refp is None else refp.double(), adv.double(), w.double(),
                      lo, hi, float(torch.tensor(c)))
    loss, logp, kl = (torch.full((R,), 9.0, device="cuda") for _ in range(3))
    st = status_word()
    _, dx = strided(R, V, ld, off, dtype)
    back = form != "forward"
    args = lambda out: (stream(), dt(x), ptr(x), ld, ptr(ti), ptr(old), ptr(refp), ptr(adv), ptr(w), 0.2, 0.28, c, gs,  # noqa: E731
                        ptr(loss), ptr(logp), ptr(kl), ptr(out) if back else None, ld, R, V, ptr(st))
    pkt.check(pk.pk_policy_loss(*args(dx)))
    live = w != 0
    dlp = lp_tol(x64, t, want["logp"], want["lse"])
    within(logp[live], want["logp"][live], dlp[live])
    a = adv.double().abs()
    eu = torch.exp(refp.double() - want["logp"]) if refp is not None else torch.zeros_like(dlp)
    # r and e^u have the error of their exponents (dlp) and of expf / expm1f (2^-21); three products and sums
    gt = w.double() * ((a * want["r"] + c * (eu + 1)) * (dlp + 2.0 ** -20))
    within(loss[live], want["loss"][live], (gt + w.double() * c * (dlp * (eu + 1) + 2.0 ** -20))[live])
    if refp is not None:
        u = refp.double() - want["logp"]
        within(kl[live], want["kl"][live], (dlp * (torch.expm1(u).abs() + dlp) + 2.0 ** -20 * (want["kl"] + u.abs()))[live])
    else:
        assert bool((kl[live] == 0).all())
    for out in (loss, logp, kl):
        assert bool((out[~live] == 0).all())
    if back:
        p = torch.exp(x64 - want["lse"][:, None])
        rel = 2.0 ** -18 + 2.0 ** -21 * (x64 - want["lse"][:, None]).abs()
        on = torch.zeros_like(p)
        on[torch.arange(R, device="cuda"), t] = 1
        lim = half_step(dtype) * gs * want["dx"].abs() + gs * (gt[:, None] * (p + on) + want["g"].abs()[:, None] * (p * rel + 2 * U)) + 1e-38
        within(dx[live], gs * want["dx"][live], lim[live])
        assert bool((dx[~live] == 0).all())
        first = dx.clone()
        pkt.check(pk.pk_policy_loss(*args(dx)))
        assert torch.equal(first, dx)          # the same call gives the same bits
        pkt.check(pk.pk_policy_loss(*args(x)))  # in place
        assert torch.equal(first[live], x[live]) and bool((x[~live] == 0).all())
    assert int(st) == 0


def test_policy_on_its_bounds(pk):
    """Far past a bound the gradient is exactly zero, on the free side it is not."""
    V = 64
    x = torch.randn(4, V, device="cuda", generator=gen(2))
    t = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    lp, _ = ref.logprob(x.double(), t.long())
    old = (lp - torch.tensor([1.0, 1.0, -1.0, -1.0], device="cuda")).float()   # r = e, e, 1/e, 1/e
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0], device="cuda")
    loss, dx = torch.empty(4, device="cuda"), torch.full((4, V), 5.0, device="cuda")
    pkt.check(pk.pk_policy_loss(stream(), 0, ptr(x), V, ptr(t), ptr(old), None, ptr(adv), None, 0.2, 0.2, 0.0, 1.0, ptr(loss), None,
                                None, ptr(dx), V, 4, V, None))
    assert bool((dx[0] == 0).all()) and bool((dx[3] == 0).all())
    assert bool((dx[1] != 0).all()) and bool((dx[2] != 0).all())
    within(loss[[0, 3]], torch.tensor([-1.2, 0.8], dtype=torch.float64, device="cuda"), 2 * U)


def test_bad_targets_are_reported(pk):
    V = 24
    x = torch.randn(3, V, device="cuda", generator=gen(2))
    t = torch.tensor([1, V, -100], dtype=torch.int32, device="cuda")
    st, logp, lse = status_word(), torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
    pkt.check(pk.pk_token_logprob(stream(), 0, ptr(x), V, ptr(t), None, ptr(logp), ptr(lse), 3, V, ptr(st)))
    assert int(st) == 5 and bool((logp[1:] == 0).all()) and float(logp[0]) < 0
    st.zero_()
    g, dx = torch.ones(3, device="cuda"), torch.full((3, V), 4.0, device="cuda")
    pkt.check(pk.pk_token_logprob_bwd(stream(), 0, ptr(x), V, ptr(t), ptr(lse), ptr(g), ptr(dx), V, 3, V, ptr(st)))
    assert int(st) == 5 and bool((dx[1:] == 0).all()) and bool((dx[0] != 0).all())
    st.zero_()
    adv, loss = torch.ones(3, device="cuda"), torch.empty(3, device="cuda")
    pkt.check(pk.pk_policy_loss(stream(), 0, ptr(x), V, ptr(t), None, None, ptr(adv), None, 0.2, 0.2, 0.0, 1.0, ptr(loss), None, None,
                                ptr(dx), V, 3, V, ptr(st)))
    assert int(st) == 5 and bool((dx[1:] == 0).all()) and bool((loss[1:] == 0).all())


@pytest.mark.parametrize("lengths", [[1, 1], [3, 0], [0, 0], [5, 700, 64, 1], [33, 2, 0, 31, 300, 256], [40000, 39999]])
@pytest.mark.parametrize("weights", [True, False])
def test_preference_loss(pk, lengths, weights):
    g = gen(21)
    at = [2]
    for n in lengths:
        at.append(at[-1] + n)
    R, P = at[-1] + 3, len(lengths) // 2
    logp = -torch.rand(R, device="cuda", generator=g) * 4
    refp = logp + torch.randn(R, device="cuda", generator=g) * 0.05
    w = (torch.rand(R, device="cuda", generator=g) > 0.3).float() * 0.7 if weights else None
    seq = torch.tensor(at, dtype=torch.int32, device="cuda")
    if weights:  # rows that do not count hold anything
        skip = w == 0
        logp[skip] = float("nan")
        refp[skip] = -float("inf")
    beta, eps, gs = 0.1, 0.05, 0.25
    loss, margin = torch.empty(P, device="cuda"), torch.empty(P, device="cuda")
    dlogp = torch.full((R,), 3.0, device="cuda")
    st = status_word()
    call = lambda: pkt.check(pk.pk_preference_loss(stream(), ptr(logp), ptr(refp), ptr(w), ptr(seq), P, R, beta, eps, gs, ptr(loss),  # noqa: E731
                                                   ptr(margin), ptr(dlogp), ptr(st)))
    call()
    w64 = w.double() if weights else torch.ones(R, device="cuda", dtype=torch.float64)
    clean = lambda v: torch.where(w64 == 0, torch.zeros_like(v, dtype=torch.float64), v.double())  # noqa: E731
    f = lambda v: float(torch.tensor(v))  # noqa: E731
    want = ref.preference(clean(logp).cpu(), clean(refp).cpu(), w64.cpu(), at, f(beta), f(eps))
    # sums are in 64 bits (1e-11 at these lengths); loss and margin round once, dlogp rounds its factor and the product
    within(margin.cpu(), want["margin"], U * want["margin"].abs() + 1e-10)
    within(loss.cpu(), want["loss"], U * want["loss"].abs() + 1e-10)
    inside = torch.zeros(R, dtype=torch.bool)
    inside[at[0]:at[-1]] = True
    within(dlogp.cpu()[inside], gs * want["dlogp"][inside], (3 * U * gs * want["dlogp"].abs() + 1e-10)[inside])
    assert bool((dlogp.cpu()[~inside] == 3).all()) and int(st) == 0
    a, b = loss.clone(), dlogp.clone()
    call()
    assert torch.equal(a, loss) and torch.equal(b, dlogp)


def test_preference_without_reference_and_bad_offsets(pk):
    logp = -torch.rand(10, device="cuda", generator=gen(1))
    seq = torch.tensor([0, 3, 5, 4, 9, 9, 11], dtype=torch.int32, device="cuda")  # pair 1 descends, pair 2 leaves the rows
    loss, dlogp, st = torch.empty(3, device="cuda"), torch.full((10,), 2.0, device="cuda"), status_word()
    pkt.check(pk.pk_preference_loss(stream(), ptr(logp), None, None, ptr(seq), 3, 10, 0.5, 0.0, 1.0, ptr(loss), None, ptr(dlogp), ptr(st)))
    z = 0.5 * (float(logp[:3].double().sum()) - float(logp[3:5].double().sum()))
    within(loss[:1].cpu(), torch.nn.functional.softplus(torch.tensor([-z], dtype=torch.float64)), 4 * U)
    assert bool(torch.isnan(loss[1:]).all()) and int(st) == 5 and bool((dlogp[5:] == 2).all()) and bool((dlogp[:5] != 2).all())
    pkt.check(pk.pk_preference_loss(stream(), ptr(logp), None, None, ptr(seq), 1, 10, 0.5, 0.0, 1.0, ptr(loss), None, None, None))


def test_preference_margins_without_end(pk):
    """A chosen or rejected answer that the policy excludes: infinite margins, finite gradients."""
    logp = torch.tensor([-float("inf"), -1.0, -1.0, -float("inf")], device="cuda")
    seq = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device="cuda")
    loss, margin, dlogp = torch.empty(2, device="cuda"), torch.empty(2, device="cuda"), torch.empty(4, device="cuda")
    pkt.check(pk.pk_preference_loss(stream(), ptr(logp), None, None, ptr(seq), 2, 4, 0.5, 0.0, 1.0, ptr(loss), ptr(margin), ptr(dlogp), None))
    assert loss.tolist() == [float("inf"), 0.0] and margin.tolist() == [-float("inf"), float("inf")]
    assert dlogp.tolist() == [-0.5, 0.5, 0.0, 0.0]


# ---- q / k norm with rotation ------------------------------------------------------------------

HEADS = [(1, 1, 1, 2), (5, 4, 2, 8), (37, 14, 2, 64), (130, 3, 1, 80), (7, 8, 8, 128), (3, 5, 5, 96), (64, 2, 1, 256), (9, 6, 3, 34),
         (2000, 16, 4, 128), (33, 40, 0, 64), (33, 0, 5, 32), (4, 2, 2, 254)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", HEADS)
@pytest.mark.parametrize("layout", ["apart", "packed", "unaligned"])
@pytest.mark.parametrize("turn", ["all", "first", "none"])
def test_qk_norm_rope(pk, dtype, shape, layout, turn):
    T, Hq, Hkv, dk = shape
    nq, nk, eps, n_pos = Hq * dk, Hkv * dk, 1e-6, 50
    g = gen(7)

    def pair(seed, empty=False):
        r = lambda *s: torch.full(s, 3.0, device="cuda", dtype=dtype) if empty else torch.randn(*s, device="cuda", generator=gen(seed)).to(dtype)  # noqa: E731
        if layout == "apart":
            return r(T, max(nq, 1))[:, :nq], r(T + 1, max(nk, 1))[:T, :nk]
        extra = 8 if layout == "packed" else 3
        z = r(T + 1, nq + 2 * nk + extra)
        if layout == "unaligned":
            z = z.view(-1)[1:1 + T * (nq + 2 * nk + extra)].view(T, -1)
        return z[:T, :nq], z[:T, nq:nq + nk]

    q, k = pair(1)
    wq, wk = (1 + 0.3 * torch.randn(dk, device="cuda", generator=g) for _ in range(2))
    pos = torch.randint(0, n_pos, (T,), device="cuda", generator=g).to(torch.int32)
    cs32 = ref.table(n_pos, dk, 1e4).float().cuda()
    cs = cs32.double()
    rq, rk = {"all": (Hq, Hkv), "first": (min(1, Hq), min(1, Hkv)), "none": (0, 0)}[turn]
    table = (ptr(pos), ptr(cs32), n_pos) if turn != "none" else (None, None, 0)
    oq, ok = pair(0, empty=True)
    ld = lambda t: max(1, t.stride(0))  # noqa: E731
    fwd = lambda yq, yk: pkt.check(pk.pk_qk_norm_rope_fwd(  # noqa: E731
        stream(), dt(q), ptr(q), ld(q), ptr(k), ld(k), ptr(wq), ptr(wk), ptr(yq), ld(yq), ptr(yk), ld(yk), T, Hq, Hkv, dk, rq, rk,
        eps, *table))
    fwd(oq, ok)
    hs = half_step(dtype)
    for x, w, H, y, rot in ((q, wq, Hq, oq, rq), (k, wk, Hkv, ok, rk)):
        if H:
            want, size = ref.qk_forward(x.double(), w.double(), H, cs, pos.long(), rot, eps, sizes=True)
            within(y, want, hs * want.abs() + 2.0 ** -19 * size)
    gq, gk = pair(2)
    dq, dk_ = pair(0, empty=True)
    dwq, dwk = torch.full((dk,), 2.0, device="cuda"), torch.full((dk,), 3.0, device="cuda")
    buf = scratch(pk.pk_qk_norm_rope_bwd_scratch_bytes(T, Hq, Hkv, dk))
    bwd = lambda a, b, u, v: pkt.check(pk.pk_qk_norm_rope_bwd(  # noqa: E731
        stream(), dt(q), ptr(gq), ld(gq), ptr(gk), ld(gk), ptr(q), ld(q), ptr(k), ld(k), ptr(wq), ptr(wk), ptr(a), ld(a), ptr(b),
        ld(b), ptr(u), ptr(v), ptr(buf) if u is not None or v is not None else None, T, Hq, Hkv, dk, rq, rk, eps, *table))
    bwd(dq, dk_, dwq, dwk)
    for x, gy, w, H, dx, dw, rot, start in ((q, gq, wq, Hq, dq, dwq, rq, 2.0), (k, gk, wk, Hkv, dk_, dwk, rk, 3.0)):
        if not H:
            assert bool((dw == start).all())
            continue
        want, wdw, (size, wsize) = ref.qk_backward(gy.double(), x.double(), w.double(), H, cs, pos.long(), rot, eps)
        within(dx, want, hs * want.abs() + 2.0 ** -18 * size)
        # at most 64 additions in a chain, and what each term carries
        within(dw - start, wdw, 2.0 ** -17 * wsize + 4 * U * (wdw.abs() + start))
    # the same bits again; without the gains; in place
    a, b = dq.clone(), dk_.clone()
    u, v = torch.full((dk,), 2.0, device="cuda"), torch.full((dk,), 3.0, device="cuda")
    bwd(dq, dk_, u, v)
    assert torch.equal(a, dq) and torch.equal(b, dk_) and torch.equal(u, dwq) and torch.equal(v, dwk)
    bwd(gq, gk, None, None)
    assert torch.equal(a, gq) and torch.equal(b, gk)
    a, b = oq.clone(), ok.clone()
    fwd(q, k)
    assert torch.equal(a, q) and torch.equal(b, k)


def test_qk_norm_rope_clamps_positions_like_pk_rope(pk):
    T, H, dk, n_pos = 4, 2, 64, 8
    q, k = (torch.randn(T, H * dk, device="cuda", generator=gen(s)) for s in (1, 2))
    one = torch.ones(dk, device="cuda")
    cs = ref.table(n_pos, dk, 1e4).float().cuda()
    out = []
    for p in ([-3, 0, 7, 100], [0, 0, 7, 7]):
        pos = torch.tensor(p, dtype=torch.int32, device="cuda")
        oq, ok = torch.empty_like(q), torch.empty_like(k)
        pkt.check(pk.pk_qk_norm_rope_fwd(stream(), 0, ptr(q), H * dk, ptr(k), H * dk, ptr(one), ptr(one), ptr(oq), H * dk, ptr(ok), H * dk,
                                         T, H, H, dk, H, H, 1e-6, ptr(pos), ptr(cs), n_pos))
        out.append((oq, ok))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


# ---- AdamW over many tensors -------------------------------------------------------------------

HYPER = dict(lr=1e-3, b1=0.9, b2=0.999, eps=1e-8)
SIZES = [1, 31, 32, 33, 128, 129, 1000, 4096, 4097, 8191, 100003, 5]


class Many:
    """Tensors of the given sizes with their moments; `shift` moves every buffer off its alignment."""

    def __init__(self, sizes, bits, g_dtype=torch.float32, shadow=True, shift=0, seed=0, fresh=False):
        self.sizes, self.bits, r = sizes, bits, gen(seed)
        cut = lambda t: t[shift:]  # noqa: E731
        self.p = [cut(torch.randn(n + shift, device="cuda", generator=r)) for n in sizes]
        self.g = [cut((torch.randn(n + shift, device="cuda", generator=r) * torch.exp(torch.randn(n + shift, device="cuda", generator=r))).to(g_dtype)) for n in sizes]
        kind = torch.uint8 if bits == 8 else torch.float32
        self.m, self.v = ([cut(torch.zeros(n + shift, device="cuda", dtype=kind)) for n in sizes] for _ in range(2))
        self.ms, self.vs = ([torch.zeros((n + 31) // 32, device="cuda", dtype=torch.uint8) for n in sizes] for _ in range(2))
        self.sh = [cut(torch.zeros(n + shift, device="cuda", dtype=torch.bfloat16)) for n in sizes] if shadow else None
        self.rate = [1.0 if i % 2 else 0.5 for i in range(len(sizes))]
        self.decay = [0.1 if i % 3 else 0.0 for i in range(len(sizes))]
        if not fresh:  # moments as after some steps
            pk = _capi.libpk()
            for i, n in enumerate(sizes):
                m = torch.randn(n, device="cuda", generator=r)
                v = torch.rand(n, device="cuda", generator=r) * torch.exp(2 * torch.randn(n, device="cuda", generator=r))
                if bits == 8:
                    pkt.check(pk.pk_adamw_moment_pack(stream(), ptr(m), ptr(self.m[i]), ptr(self.ms[i]), n, 0))
                    pkt.check(pk.pk_adamw_moment_pack(stream(), ptr(v), ptr(self.v[i]), ptr(self.vs[i]), n, 1))
                else:
                    self.m[i].copy_(m), self.v[i].copy_(v)
        self.plan = _capi.AdamwPlan([_capi.AdamwTensor(
            p=self.p[i].data_ptr(), g=self.g[i].data_ptr(), m=self.m[i].data_ptr(), v=self.v[i].data_ptr(),
            m_scale=self.ms[i].data_ptr(), v_scale=self.vs[i].data_ptr(), shadow=self.sh[i].data_ptr() if shadow else None,
            n=n, lr_mult=self.rate[i], weight_decay=self.decay[i]) for i, n in enumerate(sizes)],
            dt(self.g[0]) if sizes else 0, bits)

    def moments(self, i):
        """(m, v in fp32 or sqrt(v)) as the step reads them, in 64 bits."""
        if self.bits == 32:
            return self.m[i].double(), self.v[i].double()
        return decode(self.m[i], self.ms[i]), decode(self.v[i], self.vs[i]).square()

    def step(self, t=3, seed=1, h=HYPER):
        c1, c2 = (float(torch.tensor(1 - b ** t)) for b in (h["b1"], h["b2"]))
        pkt.check(_capi.libpk().pk_adamw_multi(stream(), self.plan.handle, h["lr"], h["b1"], h["b2"], h["eps"], c1, c2, seed))
        return c1, c2

    def state(self):
        out = [*self.p, *self.m, *self.v, *self.ms, *self.vs, *(self.sh or [])]
        return [t.clone() for t in out]


def spread(scales, n):
    return torch.exp2(scales.double() - 127).repeat_interleave(32)[:n]


def decode(codes, scales):
    return codes.contiguous().view(torch.float8_e4m3fn).double() * spread(scales, codes.numel())


def f32(v):
    return float(torch.tensor(v))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("g_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])
def test_adamw_multi(pk, bits, g_dtype, shift):
    s = Many(SIZES, bits, g_dtype, shadow=shift == 0, shift=shift)
    before = [(s.p[i].double(), *s.moments(i)) for i in range(len(SIZES))]
    c1, c2 = s.step(seed=(5 << 32) + 9)
    h = {k: f32(v) for k, v in HYPER.items()}
    base = 0
    for i, n in enumerate(SIZES):
        p, m, v = before[i]
        g = s.g[i].double()
        m1 = h["b1"] * m + (1 - h["b1"]) * g
        v1 = h["b2"] * v + (1 - h["b2"]) * g * g
        up = m1 / c1 / ((v1 / c2).sqrt() + h["eps"])
        lr, wd = h["lr"] * f32(s.rate[i]), f32(s.decay[i])
        p1 = p - lr * (up + wd * p)
        # m1 is a sum of two products (3 roundings of their magnitudes), the quotient takes five more, p one
        carry = (h["b1"] * m.abs() + (1 - h["b1"]) * g.abs()) / c1 / ((v1 / c2).sqrt() + h["eps"])
        within(s.p[i], p1, lr * (12 * U * carry + 4 * U * wd * p.abs()) + U * p1.abs() + 1e-30)
        if s.sh:
            assert torch.equal(s.sh[i], s.p[i].to(torch.bfloat16))
        got_m, got_v = s.moments(i)
        if bits == 32:
            within(got_m, m1, 3 * U * (h["b1"] * m.abs() + (1 - h["b1"]) * g.abs()))
            within(got_v, v1, 5 * U * v1)
        else:
            for got, want, codes, scales, step in ((got_m, m1, s.m[i], s.ms[i], 0.5), (got_v.sqrt(), v1.sqrt(), s.v[i], s.vs[i], 1.0)):
                sc = spread(scales, n)
                lim = torch.maximum(want.abs() * 2.0 ** -3, sc * 2.0 ** -9) * step
                slack = 8 * U * (want.abs() + (0.1 * g.abs() + 0.9 * m.abs() if step == 0.5 else 0))
                within(got, want, lim + slack)
                top = torch.nn.functional.pad(want.abs(), (0, -n % 32)).view(-1, 32).amax(1) / torch.exp2(scales.double() - 127)
                assert bool((top <= 448 * (1 + 2.0 ** -20)).all()) and bool((top > 224 * (1 - 2.0 ** -20)).all())
            assert bool((got_v[v1 > 0] > 0).all())
            # the side that chance chose: up when the fraction between the codes plus the element's bits passes one
            sc = spread(s.vs[i], n)
            y = v1.sqrt() / sc
            st = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
            u = ref.random_bits(torch.arange(n, device="cuda") + base, (5 << 32) + 9).double() / 2 ** 20
            low = torch.floor(y / st)
            sure = ((y / st - low + u) - 1).abs() > 2.0 ** -16  # u has 20 bits, y/st < 16 an error below 2^-19
            want_code = torch.maximum((low + (y / st - low + u >= 1)) * st, torch.tensor(2.0 ** -9, device="cuda"))
            assert torch.equal((got_v.sqrt() / sc)[sure], want_code[sure])
        base += -(-n // 32) * 32


@pytest.mark.parametrize("g_dtype", [torch.float32, torch.bfloat16])
def test_adamw_multi_alignment_changes_nothing(pk, g_dtype):
    """Wide and narrow accesses give the same bits, moments in 8 bits."""
    a, b = Many(SIZES, 8, g_dtype, shift=0), Many(SIZES, 8, g_dtype, shift=3)
    for x, y in zip((*a.p, *a.g, *a.m, *a.v, *a.ms, *a.vs), (*b.p, *b.g, *b.m, *b.v, *b.ms, *b.vs)):
        y.copy_(x)
    a.step(), b.step()
    for x, y in zip(a.state(), b.state()):
        assert torch.equal(x, y)


@pytest.mark.parametrize("shift", [0, 1])
def test_adamw_multi_32_has_the_bits_of_pk_adamw(pk, shift):
    a = Many(SIZES, 32, shift=shift)
    p, m, v, sh = ([t.clone() for t in x] for x in (a.p, a.m, a.v, a.sh))
    if shift:  # the same misalignment for the single calls
        p, m, v, sh = ([torch.cat([t[:1], t])[1:] for t in x] for x in (p, m, v, sh))
    c1, c2 = a.step()
    for i, n in enumerate(SIZES):
        pkt.check(pk.pk_adamw(stream(), ptr(p[i]), ptr(a.g[i]), ptr(m[i]), ptr(v[i]), n, HYPER["lr"] * a.rate[i], 0.9, 0.999, 1e-8,
                              a.decay[i], c1, c2, ptr(sh[i])))
        for x, y in ((p, a.p), (m, a.m), (v, a.v), (sh, a.sh)):
            assert torch.equal(x[i], y[i]), i


def test_adamw_multi_is_repeatable_and_moves_by_seed(pk):
    a, b, c = (Many(SIZES, 8) for _ in range(3))
    a.step(seed=4), b.step(seed=4), c.step(seed=5)
    for x, y in zip(a.state(), b.state()):
        assert torch.equal(x, y)
    for i in range(len(SIZES)):
        assert torch.equal(a.p[i], c.p[i]) and torch.equal(a.m[i], c.m[i])
    assert any(not torch.equal(x, y) for x, y in zip(a.v, c.v))


def test_second_moment_is_unbiased_and_does_not_freeze(pk):
    """With gradients of zero, v falls by b2 a step in the mean although a step is far below half a code."""
    n, steps = 1 << 16, 40
    s = Many([n], 8, fresh=True)
    one = torch.ones(n, device="cuda")
    pkt.check(pk.pk_adamw_moment_pack(stream(), ptr(one), ptr(s.v[0]), ptr(s.vs[0]), n, 1))
    s.g[0].zero_()
    for k in range(steps):
        s.step(t=1000, seed=k)
    r = decode(s.v[0], s.vs[0])
    # every step keeps the mean of sqrt(v) but for the factor sqrt(b2); a rounding's variance is at most (step / 2)^2,
    # step <= 1/8 here: six sigma of the mean of n values after `steps` roundings
    want = f32(0.999) ** (steps / 2)
    assert abs(float(r.mean()) - want) < 6 * (steps ** 0.5) * (1 / 16) / n ** 0.5
    assert float((r < 1).float().mean()) > 0.05


def test_adamw_multi_starts_from_zero_memory(pk):
    s = Many([100, 64], 8, fresh=True)
    s.g[1].zero_()
    p1 = s.p[1].clone()
    s.step(t=1)
    m, v = s.moments(0)
    within(m, 0.1 * s.g[0].double(), torch.maximum(0.1 * s.g[0].double().abs() * 2.0 ** -4, spread(s.ms[0], 100) * 2.0 ** -10) * 1.001)
    assert bool((v[s.g[0] != 0] > 0).all())
    assert not s.m[1].any() and not s.v[1].any() and bool((s.ms[1] == 1).all())
    within(s.p[1], p1.double() * (1 - 1e-3 * f32(s.decay[1])), 4 * U * p1.abs().double() + 1e-30)


def test_adamw_multi_non_finite_gradients_stay_alone(pk):
    s, clean = Many([96, 70], 8), Many([96, 70], 8)
    for i, at in ((0, 40), (1, 66)):  # a whole block, and the ragged last one
        s.g[i][at] = float("nan")
        s.g[i][at + 1] = float("inf")
        clean.g[i][at:at + 2] = 0
    s.step(), clean.step()
    for i, at in ((0, 40), (1, 66)):
        keep = torch.ones(s.sizes[i], dtype=torch.bool, device="cuda")
        keep[at:at + 2] = False
        m, v = s.moments(i)
        assert bool(torch.isnan(m[~keep]).all()) and bool(torch.isnan(v[~keep]).all())
        assert bool(torch.isfinite(m[keep]).all()) and bool(torch.isfinite(v[keep]).all())
        assert torch.equal(s.p[i][keep], clean.p[i][keep])


@pytest.mark.parametrize("root", [0, 1])
@pytest.mark.parametrize("n", [1, 32, 33, 5000])
def test_moment_pack_and_unpack(pk, root, n):
    x = torch.randn(n, device="cuda", generator=gen(3)) * torch.exp(4 * torch.randn(n, device="cuda", generator=gen(4)))
    if root:
        x = x.square()
    c, b = torch.empty(n, dtype=torch.uint8, device="cuda"), torch.empty((n + 31) // 32, dtype=torch.uint8, device="cuda")
    pkt.check(pk.pk_adamw_moment_pack(stream(), ptr(x), ptr(c), ptr(b), n, root))
    want = x.double().sqrt() if root else x.double()
    got, sc = decode(c, b), spread(b, n)
    lim = torch.maximum(want.abs() * 2.0 ** -4, sc * 2.0 ** -10)
    if root:  # nothing above zero becomes zero
        lim = torch.maximum(lim, sc * 2.0 ** -9)
        assert bool((got[x > 0] > 0).all())
    within(got, want, lim + 2 * U * want.abs())
    y = torch.empty(n, device="cuda")
    pkt.check(pk.pk_adamw_moment_unpack(stream(), ptr(c), ptr(b), ptr(y), n, root))
    within(y, got.square() if root else got, U * (got.square() if root else got * 0).abs())
    c2, b2 = torch.empty_like(c), torch.empty_like(b)   # packing what was unpacked changes nothing
    pkt.check(pk.pk_adamw_moment_pack(stream(), ptr(y), ptr(c2), ptr(b2), n, root))
    assert torch.equal(decode(c2, b2), got)


def test_adamw_plan_refuses_overlaps_and_host_memory(pk):
    a = torch.zeros(4096, device="cuda")
    base = a.data_ptr()

    def make(*tensors):
        rows = [_capi.AdamwTensor(p=base + p, g=base + g, m=base + m, v=base + v, shadow=None, n=64, lr_mult=1.0, weight_decay=0.0)
                for p, g, m, v in tensors]
        return _capi.AdamwPlan(rows, 0, 32)

    make((0, 1024, 2048, 2560), (256, 1024, 2304, 2816)).close()     # two tensors may read one gradient
    for second in ((0, 1280, 4096, 5120), (128, 1280, 4096, 5120), (512, 1024 + 252, 1024 + 128, 5120)):
        with pytest.raises(_capi.PkError, match="overlaps"):
            make((0, 1024, 2048, 2560), second)
    host = torch.zeros(64)
    with pytest.raises(_capi.PkError, match="not in the current GPU"):
        _capi.AdamwPlan([_capi.AdamwTensor(p=host.data_ptr(), g=base, m=base + 1024, v=base + 2048, n=64)], 0, 32)
    empty = Many([], 8)
    empty.step()


# ---- together ----------------------------------------------------------------------------------

def test_on_another_stream_and_replayed_from_a_graph(pk):
    """The losses' calls and the optimizer's on a side stream, captured once and replayed."""
    R, V, P = 24, 515, 2
    x, t = make_logits(R, V, 520, 0, torch.bfloat16)
    ti = t.to(torch.int32)
    seq = torch.tensor([0, 5, 12, 18, 24], dtype=torch.int32, device="cuda")
    refp = torch.randn(R, device="cuda", generator=gen(3)) - 4
    adv = torch.randn(R, device="cuda", generator=gen(4))
    opt = Many(SIZES, 8)

    def make():
        return {k: torch.zeros(n, device="cuda") for k, n in (("logp", R), ("lse", R), ("loss", P), ("dlogp", R), ("rl", R))} | {
            "dx": torch.zeros(R, V, device="cuda", dtype=x.dtype), "px": torch.zeros(R, V, device="cuda", dtype=x.dtype)}

    def steps(o, m):
        s = stream()
        pkt.check(pk.pk_token_logprob(s, 1, ptr(x), 520, ptr(ti), None, ptr(o["logp"]), ptr(o["lse"]), R, V, None))
        pkt.check(pk.pk_preference_loss(s, ptr(o["logp"]), ptr(refp), None, ptr(seq), P, R, 0.1, 0.0, 1.0, ptr(o["loss"]), None, ptr(o["dlogp"]), None))
        pkt.check(pk.pk_token_logprob_bwd(s, 1, ptr(x), 520, ptr(ti), ptr(o["lse"]), ptr(o["dlogp"]), ptr(o["dx"]), V, R, V, None))
        pkt.check(pk.pk_policy_loss(s, 1, ptr(x), 520, ptr(ti), None, ptr(refp), ptr(adv), None, 0.2, 0.2, 0.1, 1.0, ptr(o["rl"]), None, None,
                                    ptr(o["px"]), V, R, V, None))
        m.step(seed=11)

    plain, plain_opt = make(), Many(SIZES, 8)
    steps(plain, plain_opt)
    torch.cuda.synchronize()
    out, side, graph = make(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        steps(out, opt)
    graph.replay()
    torch.cuda.synchronize()
    for k in plain:
        assert torch.equal(plain[k], out[k]), k
    for a, b in zip(plain_opt.state(), opt.state()):
        assert torch.equal(a, b)
    x.copy_(torch.randn(R, V, device="cuda", generator=gen(77)))   # new inputs in the same place
    graph.replay()
    steps(plain, plain_opt)
    torch.cuda.synchronize()
    for k in plain:
        assert torch.equal(plain[k], out[k]), k
    for a, b in zip(plain_opt.state(), opt.state()):
        assert torch.equal(a, b)
