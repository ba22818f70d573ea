"""The tuning operators where ordinary tests do not go: vocabularies beyond a cluster of eight CTAs and beyond any
cluster, offsets past 2^31 elements, two streams at once, a process whose first calls are captured into a graph.
Tolerances as in tests/test_tuning_ops_gpu.py."""
import os
import subprocess
import sys

import pytest
import torch

from tests import pkt
from tests import test_tuning_ops_gpu as ops
from tests.pkt import dt, ptr, scratch, stream
from tests.test_tuning_ops_gpu import gen, pk  # noqa: F401

pytestmark = pytest.mark.gpu
WIDE = [(5, 131080, 131080, 0), (3, 200064, 200064, 0), (3, 262147, 262147, 1), (2, 400009, 400016, 0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", WIDE)
def test_wide_vocabularies(pk, dtype, shape):  # noqa: F811
    ops.test_policy_loss(pk, dtype, shape, "all")
    ops.test_policy_loss(pk, dtype, shape, "forward")
    ops.test_token_logprob_and_gradient(pk, dtype, shape)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [200064, 400009])
def test_masked_words_in_wide_vocabularies(pk, dtype, V):  # noqa: F811
    ops.test_masked_words_and_odd_rows(pk, dtype, V)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1025, 14, 2, 64), (1100, 14, 2, 96), (1031, 3, 6, 80), (1024, 12, 12, 64), (1500, 7, 1, 256), (1026, 24, 3, 34),
                                   (1501, 16, 1, 128), (1200, 6, 5, 64), (1027, 40, 0, 64), (1027, 0, 7, 32), (2051, 28, 4, 8)])
@pytest.mark.parametrize("layout, turn", [("packed", "all"), ("apart", "first"), ("apart", "none"), ("unaligned", "all")])
def test_head_norms_of_many_tokens(pk, dtype, shape, layout, turn):  # noqa: F811
    """Rounds of heads are cut another way from a thousand tokens on."""
    ops.test_qk_norm_rope(pk, dtype, shape, layout, turn)


def policy(pk, x, t, old, adv, w, dx, ld, ldd, R, V, loss, logp):  # noqa: F811
    pkt.check(pk.pk_policy_loss(stream(), dt(x), ptr(x), ld, ptr(t), ptr(old), None, ptr(adv), ptr(w), 0.2, 0.2, 0.0, 1.0, ptr(loss),
                                ptr(logp), None, ptr(dx), ldd, R, V, None))


def test_losses_past_32_bit_offsets(pk):  # noqa: F811
    """The last rows of logits with more than 2^31 elements have the bits of the same rows alone."""
    R, V, tail = 42800, 50264, 48
    assert R * V > 2 ** 31
    x = torch.zeros(R, V, device="cuda", dtype=torch.bfloat16)
    x[-tail:] = torch.randn(tail, V, device="cuda", generator=gen(1)) * 3
    mine = x[-tail:].clone()
    t = torch.randint(0, V, (R,), device="cuda", dtype=torch.int32, generator=gen(2))
    old, adv = torch.full((R,), -9.0, device="cuda"), torch.randn(R, device="cuda", generator=gen(3))
    w = torch.zeros(R, device="cuda")
    w[-tail:] = 1
    loss, logp, lse = (torch.full((R,), 5.0, device="cuda") for _ in range(3))
    a_loss, a_logp, a_dx = torch.empty(tail, device="cuda"), torch.empty(tail, device="cuda"), torch.empty_like(mine)
    policy(pk, mine, t[-tail:], old[-tail:], adv[-tail:], w[-tail:], a_dx, V, V, tail, V, a_loss, a_logp)
    pkt.check(pk.pk_token_logprob(stream(), 1, ptr(x), V, ptr(t), ptr(w), ptr(logp), ptr(lse), R, V, None))
    within = lambda a, b: ops.within(a, b, 2.0 ** -17 * (1 + b.double().abs()))  # noqa: E731  (another split of the row's sum)
    within(logp[-tail:], a_logp)
    assert bool((logp[:-tail] == 0).all())
    policy(pk, x, t, old, adv, w, x, V, V, R, V, loss, logp)
    within(loss[-tail:], a_loss)
    assert bool((loss[:-tail] == 0).all()) and bool((x[0] == 0).all())
    # a gradient may round to the neighbouring code where the two sums differ in their last bits
    ops.within(x[-tail:], a_dx, 2.0 ** -7 * a_dx.double().abs() + 1e-12)
    # every row of the whole in the backward of the log-probabilities; the last rows sit past 2^31
    x[-tail:] = mine
    g = torch.zeros(R, device="cuda")
    g[-tail:] = adv[-tail:]
    pkt.check(pk.pk_token_logprob_bwd(stream(), 1, ptr(x), V, ptr(t), ptr(lse), ptr(g), ptr(x), V, R, V, None))
    pkt.check(pk.pk_token_logprob_bwd(stream(), 1, ptr(mine), V, ptr(t[-tail:]), ptr(lse[-tail:]), ptr(adv[-tail:]), ptr(mine), V, tail, V, None))
    assert torch.equal(x[-tail:], mine) and bool((x[R // 2] == 0).all())


def test_head_norms_past_32_bit_offsets(pk):  # noqa: F811
    T, H, Hk, d, tail = 330000, 96, 4, 64, 33
    ld = (H + Hk + 4) * d
    assert T * ld > 2 ** 31
    buf = torch.zeros(T, ld, device="cuda", dtype=torch.bfloat16)
    buf[-tail:] = torch.randn(tail, ld, device="cuda", generator=gen(1))
    small = buf[-tail:].clone()
    wq, wk = (1 + torch.randn(d, device="cuda", generator=gen(i)) * 0.2 for i in (2, 3))
    table = torch.randn(40, d, device="cuda", generator=gen(4))
    pos = (torch.arange(T, device="cuda", dtype=torch.int32) % 40).contiguous()

    def forward(b, p, n):
        q, k = b, b[:, H * d:]
        pkt.check(pk.pk_qk_norm_rope_fwd(stream(), 1, ptr(q), ld, ptr(k), ld, ptr(wq), ptr(wk), ptr(q), ld, ptr(k), ld, n, H, Hk, d, H, Hk,
                                         1e-5, ptr(p), ptr(table), 40))

    def backward(b, src, p, n):
        dw = [torch.zeros(d, device="cuda") for _ in range(2)]
        s = scratch(pk.pk_qk_norm_rope_bwd_scratch_bytes(n, H, Hk, d))
        pkt.check(pk.pk_qk_norm_rope_bwd(stream(), 1, ptr(b), ld, ptr(b[:, H * d:]), ld, ptr(src), ld, ptr(src[:, H * d:]), ld, ptr(wq), ptr(wk),
                                         ptr(b), ld, ptr(b[:, H * d:]), ld, ptr(dw[0]), ptr(dw[1]), ptr(s), n, H, Hk, d, H, Hk, 1e-5, ptr(p),
                                         ptr(table), 40))
        return dw

    src, src_small = buf.clone(), small.clone()
    forward(buf, pos, T)
    forward(small, pos[-tail:], tail)
    assert torch.equal(buf[-tail:], small) and bool((buf[:1000] == 0).all())
    dw = backward(buf, src, pos, T)
    dw_small = backward(small, src_small, pos[-tail:], tail)
    assert torch.equal(buf[-tail:], small)
    for a, b, heads in zip(dw, dw_small, (H, Hk)):
        # all other rows add zeros; the order of the sums differs: at most 128 additions in a chain, over terms g x inv whose
        # magnitudes are below 1 in the mean
        ops.within(a, b, 128 * ops.U * tail * heads)


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_past_32_bit_offsets(pk, bits):  # noqa: F811
    n, tail = 2 ** 31 + 5077, 5077
    kind = torch.uint8 if bits == 8 else torch.float32

    def state(n):
        return dict(p=torch.zeros(n, device="cuda"), g=torch.zeros(n, device="cuda", dtype=torch.bfloat16), m=torch.zeros(n, device="cuda", dtype=kind),
                    v=torch.zeros(n, device="cuda", dtype=kind), ms=torch.zeros((n + 31) // 32, device="cuda", dtype=torch.uint8),
                    vs=torch.zeros((n + 31) // 32, device="cuda", dtype=torch.uint8))

    g, p = torch.randn(tail, device="cuda", generator=gen(1)).bfloat16(), torch.randn(tail, device="cuda", generator=gen(2))
    outs = []
    for size in (n, tail):
        s = state(size)
        s["g"][-tail:] = g
        s["p"][-tail:] = p
        plan = ops._capi.AdamwPlan([ops._capi.AdamwTensor(p=s["p"].data_ptr(), g=s["g"].data_ptr(), m=s["m"].data_ptr(), v=s["v"].data_ptr(),
                                                          m_scale=s["ms"].data_ptr(), v_scale=s["vs"].data_ptr(), shadow=None, n=size,
                                                          lr_mult=1.0, weight_decay=0.1)], 1, bits)
        pkt.check(pk.pk_adamw_multi(stream(), plan.handle, 1e-2, 0.9, 0.999, 1e-8, 0.1, 1e-3, 5))
        torch.cuda.synchronize()
        plan.close()
        outs.append([s["p"][-tail:].clone(), s["m"][-tail:].clone(), s["ms"][-((tail + 31) // 32):].clone(), s["vs"][-((tail + 31) // 32):].clone()])
        assert not bool(s["p"][:-tail][::4097].any())
        del s
    # the tail starts at a whole block of 32 and of every chunk size: the same bits (but for the codes of v, whose
    # random bits belong to the element's number)
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    torch.cuda.empty_cache()


def test_two_streams_at_once(pk):  # noqa: F811
    """The kernels keep nothing between calls that another stream's call could meet."""
    R, V = 300, 50257
    sets = []
    for i in range(2):
        x, t = ops.make_logits(R, V, V, 0, torch.bfloat16, seed=10 * i)
        sets.append(dict(x=x, t=t.to(torch.int32), old=torch.full((R,), -9.0, device="cuda"), adv=torch.randn(R, device="cuda", generator=gen(i)),
                         w=(torch.rand(R, device="cuda", generator=gen(i + 5)) > 0.3).float()))

    def run(s):
        o = dict(dx=torch.empty(R, V, device="cuda", dtype=torch.bfloat16), loss=torch.empty(R, device="cuda"), logp=torch.empty(R, device="cuda"))
        policy(pk, s["x"], s["t"], s["old"], s["adv"], s["w"], o["dx"], V, V, R, V, o["loss"], o["logp"])
        return o

    alone = [run(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        both = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                both.append(run(s))
        torch.cuda.synchronize()
        for a, b in zip(alone, both):
            assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("R, V", [(40, 32000), (2000, 515), (3000, 8192)])
def test_calls_wait_for_what_runs_before_them(pk, R, V):  # noqa: F811
    """Kernels that start early still see what their predecessors write and leave alone what those read: other kernels, copies,
    each other, and a join of two streams, on a stream and in a graph."""
    base, t = ops.make_logits(R, V, V, 0, torch.bfloat16)
    ti, adv, old = t.to(torch.int32), torch.randn(R, device="cuda", generator=gen(3)), torch.full((R,), -9.0, device="cuda")
    seq = torch.tensor([0, R // 4, R // 2, R // 2 + 3, R], dtype=torch.int32, device="cuda")
    x, x2 = torch.zeros_like(base), torch.zeros_like(base)
    o = {k: torch.zeros(n, device="cuda") for k, n in (("logp", R), ("lse", R), ("loss", 2), ("dlogp", R), ("rl", R), ("dw", 64))}
    heads, gain = torch.randn(R, 64, device="cuda", generator=gen(4)), torch.ones(64, device="cuda")
    s_heads = scratch(pk.pk_qk_norm_rope_bwd_scratch_bytes(R, 1, 0, 64))
    dheads = torch.zeros_like(heads)
    side = torch.cuda.Stream()

    def work(scale, wait=lambda: None):
        here = torch.cuda.current_stream()
        torch.mul(base, scale, out=x)                      # a kernel right before
        wait()
        pkt.check(pk.pk_token_logprob(stream(), 1, ptr(x), V, ptr(ti), None, ptr(o["logp"]), ptr(o["lse"]), R, V, None))
        wait()
        pkt.check(pk.pk_preference_loss(stream(), ptr(o["logp"]), None, None, ptr(seq), 2, R, 0.1, 0.0, 1.0, ptr(o["loss"]), None, ptr(o["dlogp"]), None))
        wait()
        pkt.check(pk.pk_token_logprob_bwd(stream(), 1, ptr(x), V, ptr(ti), ptr(o["lse"]), ptr(o["dlogp"]), ptr(x), V, R, V, None))
        side.wait_stream(here)
        with torch.cuda.stream(side):
            x2.copy_(x)                                    # another stream between
        here.wait_stream(side)
        wait()
        pkt.check(pk.pk_policy_loss(stream(), 1, ptr(x2), V, ptr(ti), ptr(old), None, ptr(adv), None, 0.2, 0.2, 0.0, 1.0, ptr(o["rl"]), None, None,
                                    ptr(x2), V, R, V, None))
        wait()
        o["dw"].zero_()
        pkt.check(pk.pk_qk_norm_rope_bwd(stream(), 0, ptr(heads), 64, None, 0, ptr(heads), 64, None, 0, ptr(gain), None, ptr(dheads), 64, None, 0,
                                         ptr(o["dw"]), None, ptr(s_heads), R, 1, 0, 64, 0, 0, 1e-5, None, None, 0))
        wait()
        return [v.clone() for v in (*o.values(), x, x2, dheads)]

    want = {k: work(k, torch.cuda.synchronize) for k in (1.0, 0.5, 2.0)}
    for i in range(30):
        k = (1.0, 0.5, 2.0)[i % 3]
        got = work(k)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[k]))
    graph, main = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=main):
        got = work(0.5)
    for _ in range(5):
        for v in got:
            v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[0.5]))


FIRST = r'''
import torch
from tests import pkt
from tests import test_tuning_ops_gpu as ops
from tests.pkt import ptr, scratch, stream
pk = ops._capi.libpk()
R, V, d = 200, 50257, 64
x = torch.randn(R, V, device="cuda").bfloat16()
t = torch.randint(0, V, (R,), device="cuda", dtype=torch.int32)
adv, old = torch.randn(R, device="cuda"), torch.full((R,), -9.0, device="cuda")
loss, logp, lse, dx = torch.zeros(R, device="cuda"), torch.zeros(R, device="cuda"), torch.zeros(R, device="cuda"), torch.zeros_like(x)
q, k, w = torch.randn(R, 4 * d, device="cuda"), torch.randn(R, 2 * d, device="cuda"), torch.ones(d, device="cuda")
dq, dk, dw = torch.zeros_like(q), torch.zeros_like(k), torch.zeros(2, d, device="cuda")
s = scratch(pk.pk_qk_norm_rope_bwd_scratch_bytes(R, 4, 2, d))
opt = ops.Many([1000, 33], 8, fresh=True)
def work():
    pkt.check(pk.pk_policy_loss(stream(), 1, ptr(x), V, ptr(t), ptr(old), None, ptr(adv), None, 0.2, 0.2, 0.0, 1.0, ptr(loss), None, None, ptr(dx), V, R, V, None))
    pkt.check(pk.pk_token_logprob(stream(), 1, ptr(x), V, ptr(t), None, ptr(logp), ptr(lse), R, V, None))
    pkt.check(pk.pk_qk_norm_rope_bwd(stream(), 0, ptr(q), 4 * d, ptr(k), 2 * d, ptr(q), 4 * d, ptr(k), 2 * d, ptr(w), ptr(w), ptr(dq), 4 * d, ptr(dk), 2 * d,
                                     ptr(dw[0]), ptr(dw[1]), ptr(s), R, 4, 2, d, 0, 0, 1e-5, None, None, 0))
    opt.step()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    work()
graph.replay()
torch.cuda.synchronize()
got = [v.clone() for v in (loss, dx, logp, lse, dq, dk, dw)]
for v in (loss, dx, logp, lse, dq, dk, dw): v.zero_()
work()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, (loss, dx, logp, lse, dq, dk, dw))) and bool(dx.any()) and bool(dw.any())
print("same")
'''


def test_first_calls_of_a_process_are_captured():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]
