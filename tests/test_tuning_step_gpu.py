"""Preference and policy tuning through the model-level calls: blocks with q / k norms, the losses over
the fused head, AdamW with 8-bit moments and rates per parameter, and a run of them together.

Tolerances as in tests/test_step_gpu.py: fp32 losses 1e-4 relative, gradients 1e-4 of their largest
element (a logit's gradient carries at most 2^-18 relative from its softmax; the products that
contract it sum terms within a factor of 25 of the result); bf16 gradients cosine 0.99."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mt():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from paperkiln_b200 import model
    model.init(0, model.FP32)
    yield model
    model.init(0, model.FP32)


SPEC = dict(family="llama", vocab=211, d=64, layers=2, heads=4, kv_heads=2, dff=96, nctx=64, rope_all=1, seed=5)


def tokens(n, vocab=211, seed=0):
    s = np.random.RandomState(seed).randint(0, vocab, size=n + 1).astype(np.int32)
    return s[:-1].copy(), s[1:].copy()


def close_grads(a, b, tol=1e-4):
    assert a.keys() == b.keys()
    for n in a:
        if a[n] is None or b[n] is None:
            assert a[n] is None and b[n] is None
            continue
        assert np.abs(a[n] - b[n]).max() <= tol * max(1e-6, np.abs(b[n]).max()), n


# ---- q / k norms in the block ------------------------------------------------------------------

def torch_block(p, x, B, S, H, Hkv, dk, theta, rot_q, rot_k):
    import torch

    def rms(t, w):
        return t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-5) * w

    def heads(t, n, w, rot):
        t = rms(t.view(-1, n, dk), w)
        pos = torch.arange(S, dtype=torch.float64).repeat(B)
        ang = pos[:, None] / torch.pow(torch.tensor(theta, dtype=torch.float64), torch.arange(0, dk, 2, dtype=torch.float64) / dk)[None]
        c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
        a, b = t[..., 0::2], t[..., 1::2]
        turned = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
        return torch.cat((turned[:, :rot], t[:, rot:]), 1).reshape(B, S, n, dk).transpose(1, 2)

    h = rms(x, p["input_layernorm.weight"])
    q = heads(h @ p["self_attn.q_proj.weight"], H, p["self_attn.q_norm.weight"], rot_q)
    k = heads(h @ p["self_attn.k_proj.weight"], Hkv, p["self_attn.k_norm.weight"], rot_k).repeat_interleave(H // Hkv, 1)
    v = (h @ p["self_attn.v_proj.weight"]).view(B, S, Hkv, dk).transpose(1, 2).repeat_interleave(H // Hkv, 1)
    s = (q @ k.transpose(-1, -2)) / math.sqrt(dk)
    s = s.masked_fill(~torch.ones(S, S, dtype=torch.bool).tril(), float("-inf"))
    a = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B * S, H * dk)
    x = x + a @ p["self_attn.o_proj.weight"]
    h = rms(x, p["post_attention_layernorm.weight"])
    return x + (torch.nn.functional.silu(h @ p["mlp.gate_proj.weight"]) * (h @ p["mlp.up_proj.weight"])) @ p["mlp.down_proj.weight"]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("dk", [16, 64])
@pytest.mark.parametrize("rope_all", [0, 1])
def test_block_with_qk_norm(mt, dtype, dk, rope_all):
    import torch
    mt.init(0, mt.BF16 if dtype == "bf16" else mt.FP32)
    B, S, H, Hkv, dff = 2, 40, 4, 2, 96
    d = H * dk
    rng = np.random.RandomState(3)
    x, dy = rng.randn(B * S, d).astype(np.float32), (rng.randn(B * S, d) * 1e-2).astype(np.float32)
    got = []
    for ckpt in (0, 1):
        m = mt.Model(family="block", d=d, heads=H, kv_heads=Hkv, dff=dff, theta=10000.0, rope_all=rope_all, qk_norm=1, seed=5, ckpt=ckpt)
        for i, n in enumerate(("self_attn.q_norm.weight", "self_attn.k_norm.weight")):
            m.set_param(n, 1 + 0.3 * np.random.RandomState(i).randn(1, dk).astype(np.float32))
        m.block_set_input(x, dy, S)
        m.block_forward()
        y = m.block_output()
        m.block_backward()
        got.append((y, m.block_input_grad(), m.grads()))
        if ckpt:
            continue
        p = {n: torch.tensor(m.get_param(n).astype(np.float64), requires_grad=True) for n in m.names}
        xt = torch.tensor(x.astype(np.float64), requires_grad=True)
        ref = torch_block(p, xt, B, S, H, Hkv, dk, 10000.0, H if rope_all else 1, Hkv if rope_all else 1)
        ref.backward(torch.tensor(dy.astype(np.float64)))
        pairs = [(y, ref.detach().numpy()), (got[0][1], xt.grad.numpy())] + [(got[0][2][n], p[n].grad.numpy()) for n in m.names]
        for a, b in pairs:
            if dtype == "fp32":
                assert np.abs(a - b).max() <= 1e-4 * np.abs(b).max()
            else:
                assert (a.ravel() @ b.ravel()) / (np.linalg.norm(a) * np.linalg.norm(b)) >= 0.99
        m.close()
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])   # recomputed: the same bits
    for n in got[0][2]:
        assert np.array_equal(got[0][2][n], got[1][2][n]), n
    mt.init(0, mt.FP32)


def test_qk_norm_model_files(mt, tmp_path):
    """The gains are parameters of their own: saved, loaded, taken over by a QLoRA model; no place in GGUF."""
    m = mt.Model(**SPEC, qk_norm=1)
    assert "layers.1.self_attn.k_norm.weight" in m.names
    m.set_param("layers.1.self_attn.k_norm.weight", np.full((1, 16), 1.5, np.float32))
    m.save(str(tmp_path / "w.safetensors"))
    q = mt.Model(**SPEC, qk_norm=1, qlora=1, rank=4)
    assert not any("norm" in n for n in q.names)   # frozen
    ids, targets = tokens(32)
    before = q.step(ids, targets, 16, backward=False)
    q.load_base(str(tmp_path / "w.safetensors"))
    after = q.step(ids, targets, 16, backward=False)
    assert before != after and math.isfinite(after)
    q.save_merged(str(tmp_path / "merged.safetensors"))
    r = mt.Model(**SPEC, qk_norm=1)
    r.load(str(tmp_path / "merged.safetensors"))
    assert float(r.get_param("layers.1.self_attn.k_norm.weight")[0, 0]) == 1.5
    with pytest.raises(mt.MtError, match="query and key norms"):
        m.export_gguf(str(tmp_path / "m.gguf"))
    mt.Model(**SPEC).save(str(tmp_path / "plain.safetensors"))
    with pytest.raises(mt.MtError, match="no tensor"):
        r.load(str(tmp_path / "plain.safetensors"))


# ---- the losses over the head ------------------------------------------------------------------

FAMILIES = {"tied": dict(SPEC), "untied": dict(SPEC, tie=0), "qk_norm": dict(SPEC, qk_norm=1), "qlora": dict(SPEC, qlora=1, rank=4),
            "gpt2": dict(family="gpt2", vocab=211, d=64, layers=2, heads=4, nctx=64, seed=5)}


@pytest.mark.parametrize("family", sorted(FAMILIES))
@pytest.mark.parametrize("chunk", [0, 13, 1000])
def test_policy_gradient_of_a_fresh_policy_is_the_cross_entropy_gradient(mt, family, chunk):
    """r = 1, A = 1, weight 1 / n: d loss / d logp = -1 / n, which is the mean cross entropy's."""
    m = mt.Model(**FAMILIES[family], ckpt=1)
    m.set_loss_chunk(chunk)
    ids, targets = tokens(48)
    n = ids.size
    loss = m.step(ids, targets, 16)
    want = m.grads()
    lp = m.token_logprob(ids, targets, 16)
    assert abs(loss + lp.mean()) <= 1e-4 * loss
    out = m.policy_step(ids, targets, np.ones(n), 16, weight=np.full(n, 1 / n))
    assert abs(out["loss"] + 1.0) <= 1e-5 and np.array_equal(out["logp"], lp) and not out["kl"].any()
    close_grads(m.grads(), want)
    half = m.policy_step(ids, targets, np.ones(n), 16, weight=np.full(n, 1 / n), loss_scale=0.5)
    close_grads(m.grads(), {k: None if v is None else v / 2 for k, v in want.items()})
    assert half["loss"] == out["loss"]


def test_flex_models_and_heads_apart(mt):
    """The flex family's untied head: policy and preference gradients against each other and the cross entropy's."""
    m = mt.Model(family="flex", vocab=131, d=64, layers=2, heads=4, dff=96, nctx=64, norm="rmsnorm", act="swiglu", pos="sinusoidal", seed=3)
    ids, targets = tokens(32, vocab=131)
    m.step(ids, targets, 16)
    want = m.grads()
    m.policy_step(ids, targets, np.ones(32), 16, weight=np.full(32, 1 / 32))
    close_grads(m.grads(), want)
    out = m.preference_step(ids, targets, [0, 16, 32], 16, beta=0.2)
    got = m.grads()
    lp = m.token_logprob(ids, targets, 16).astype(np.float64)
    z = 0.2 * (lp[:16].sum() - lp[16:].sum())
    assert abs(out["margin"][0] - z) <= 1e-5 * max(1, abs(z))
    dlogp = -0.2 / (1 + np.exp(z)) * np.repeat([1.0, -1.0], 16)
    m.policy_step(ids, targets, -dlogp, 16)
    close_grads(got, m.grads())


@pytest.mark.parametrize("chunk", [0, 7])
def test_micro_batches_add_up(mt, chunk):
    """Two accumulated halves give the gradient of the whole batch, for both losses; a step without backward leaves it alone."""
    ids, targets = tokens(64)
    adv = np.random.RandomState(4).randn(64)
    old = -5 + 0.1 * np.random.RandomState(5).randn(64)
    seq = np.arange(0, 65, 16, dtype=np.int32)
    whole = mt.Model(**SPEC, ckpt=1)
    halves = mt.Model(**SPEC, ckpt=1)
    halves.set_loss_chunk(chunk)
    for kind in ("policy", "preference"):
        if kind == "policy":
            run = lambda m, a, b, scale: m.policy_step(ids[a:b], targets[a:b], adv[a:b], 16, old_logp=old[a:b], loss_scale=scale)  # noqa: E731
            run(whole, 0, 64, 1.0)
        else:
            run = lambda m, a, b, scale: m.preference_step(ids[a:b], targets[a:b], seq[:(b - a) // 16 + 1], 16, loss_scale=scale)  # noqa: E731
            run(whole, 0, 64, 1.0)
        want = whole.grads()
        halves.zero_grad()
        halves.set_accumulate(True)
        scale = 1.0 if kind == "policy" else 0.5   # a sum over rows; a mean over pairs
        run(halves, 0, 32, scale)
        halves.policy_step(ids, targets, adv, 16, backward=False)
        halves.token_logprob(ids, targets, 16)
        run(halves, 32, 64, scale)
        halves.set_accumulate(False)
        close_grads(halves.grads(), want)


def test_policy_step_values_and_rows_that_do_not_count(mt):
    m = mt.Model(**SPEC, ckpt=1)
    m.set_loss_chunk(17)
    ids, targets = tokens(48)
    n = ids.size
    rng = np.random.RandomState(2)
    w = (rng.rand(n) > 0.4).astype(np.float32) / n
    lp = m.token_logprob(ids, targets, 16, weight=w)
    assert not lp[w == 0].any()
    old, refp, adv = lp - 0.3 * rng.randn(n), lp + 0.2 * rng.randn(n), rng.randn(n)
    kw = dict(seq_len=16, old_logp=old, ref_logp=refp, weight=w, clip_lo=0.2, clip_hi=0.3, kl_coef=0.1)
    out = m.policy_step(ids, targets, adv, **kw)
    g1 = m.grads()
    o32, r32 = old.astype(np.float32).astype(np.float64), refp.astype(np.float32).astype(np.float64)
    l64, a64 = lp.astype(np.float64), adv.astype(np.float32).astype(np.float64)
    r, u = np.exp(l64 - o32), r32 - l64
    rows = -np.minimum(r * a64, np.clip(r, 0.8, 1.3) * a64) + 0.1 * (np.expm1(u) - u)
    assert abs(out["loss"] - (w * rows).sum()) <= 1e-5 * np.abs(w * rows).sum()
    # targets of rows that do not count say nothing
    masked = targets.copy()
    masked[w == 0] = -100
    again = m.policy_step(ids, masked, adv, **kw)
    g2 = m.grads()
    assert again["loss"] == out["loss"]
    for k in g1:
        assert np.array_equal(g1[k], g2[k]), k
    with pytest.raises(mt.MtError, match="target out of range"):
        m.policy_step(ids, np.where(w > 0, -100, targets), adv, **kw)
    with pytest.raises(ValueError):
        m.policy_step(ids, targets, adv[:-1])


@pytest.mark.parametrize("family", ["tied", "untied", "gpt2"])
@pytest.mark.parametrize("chunk", [11, 1000])
def test_preference_gradient_is_that_of_weighted_log_probabilities(mt, family, chunk):
    """dlogp of the paired loss, as advantages of a fresh policy, gives the same gradients; in one chunk of
    logits or in several that are produced twice."""
    m = mt.Model(**FAMILIES[family], ckpt=1)
    m.set_loss_chunk(chunk)
    ids, targets = tokens(48)
    n = ids.size
    seq = np.array([0, 16, 29, 32, 48], np.int32)
    w = np.ones(n, np.float32)
    w[:4] = w[16:20] = w[30:31] = 0
    lp = m.token_logprob(ids, targets, 16, weight=w)
    refp = lp + np.random.RandomState(1).randn(n).astype(np.float32) * 0.5
    beta, eps = 0.3, 0.1
    out = m.preference_step(ids, targets, seq, 16, ref_logp=refp, weight=w, beta=beta, label_smoothing=eps)
    got = m.grads()
    v = w.astype(np.float64) * (lp.astype(np.float64) - refp.astype(np.float64))
    z = beta * np.array([v[0:16].sum() - v[16:29].sum(), v[29:32].sum() - v[32:48].sum()])
    want = (1 - eps) * np.log1p(np.exp(-z)) + eps * np.log1p(np.exp(z))
    assert np.abs(out["margin"] - z).max() <= 1e-5 and np.abs(out["pair_loss"] - want).max() <= 1e-5
    assert abs(out["loss"] - want.mean()) <= 1e-5
    dz = (eps - 1 / (1 + np.exp(z))) / 2
    dlogp = np.zeros(n)
    for i, (a, b, c) in enumerate(((0, 16, 29), (29, 32, 48))):
        dlogp[a:b], dlogp[b:c] = beta * dz[i] * w[a:b], -beta * dz[i] * w[b:c]
    m.policy_step(ids, targets, -dlogp, 16, weight=w)
    close_grads(got, m.grads())
    # loss by differences along the gradient's direction
    name = m.names[-1]
    g, p = got[name], m.get_param(name)
    step = 1e-2 * g / np.linalg.norm(g)
    side = []
    for s in (1, -1):
        m.set_param(name, p + s * step)
        side.append(m.preference_step(ids, targets, seq, 16, ref_logp=refp, weight=w, beta=beta, label_smoothing=eps, backward=False)["loss"])
    # the difference of two fp32 losses near 0.7 is good to 2^-23; the third derivative adds at most 1 % at this step
    assert abs((side[0] - side[1]) / 2 - 1e-2 * np.linalg.norm(g)) <= 2 ** -22 + 0.02 * 1e-2 * np.linalg.norm(g)
    with pytest.raises(mt.MtError, match="ascend"):
        m.preference_step(ids, targets, [0, 5, 3], 16)
    with pytest.raises(mt.MtError, match="ascend"):
        m.preference_step(ids, targets, [0, 5, 49], 16)


# ---- the optimizer -----------------------------------------------------------------------------

def train(mt, steps, bits=32, rates=None, spec=SPEC, dtype=None, model=None):
    m = model or mt.Model(**spec)
    if model is None:
        m.set_adamw(lr=1e-2, weight_decay=0.1)
        m.set_adamw_state_bits(bits)
        for name, r in (rates or {}).items():
            m.set_param_rates(name, *r)
    for k in range(steps):
        ids, targets = tokens(32, seed=k)
        m.step(ids, targets, 16)
        m.optimizer_step()
    return m


def test_unpacked_parameters_step_as_packed_ones(mt):
    a, b = train(mt, 3), train(mt, 3, spec=dict(SPEC, pack=0))
    for n in a.names:
        assert np.array_equal(a.get_param(n), b.get_param(n)), n
    sa, sb = a.optimizer_state(), b.optimizer_state()
    for n in a.names:
        assert np.array_equal(sa["m"][n], sb["m"][n]) and np.array_equal(sa["v"][n], sb["v"][n]), n


@pytest.mark.parametrize("bits", [8, 32])
def test_rates_of_single_parameters(mt, bits):
    still, free = "layers.0.self_attn.q_proj.weight", "norm.weight"
    a = train(mt, 1, bits)
    b = train(mt, 1, bits, rates={still: (0.0, 0.1), free: (1.0, 0.0)})
    fresh = mt.Model(**SPEC)
    assert np.array_equal(b.get_param(still), fresh.get_param(still))
    for n in a.names:
        same = np.array_equal(a.get_param(n), b.get_param(n))
        assert same == (n not in (still, free)), n
    # p -= lr (update + wd p): without the decay the gains of one stay higher by lr wd
    diff = b.get_param(free) - a.get_param(free)
    assert np.abs(diff - 1e-2 * 0.1).max() <= 4 * 2.0 ** -24


def test_optimizer_settings_in_any_order(mt):
    """Rates before the hyper-parameters, bits between them: the same run."""
    a = train(mt, 2, 8, rates={"norm.weight": (0.5, 0.0)})
    b = mt.Model(**SPEC)
    b.set_param_rates("norm.weight", 0.5, 0.0)
    b.set_adamw_state_bits(8)
    b.set_adamw(lr=1e-2, weight_decay=0.1)
    train(mt, 2, model=b)
    for n in a.names:
        assert np.array_equal(a.get_param(n), b.get_param(n)), n


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_eight_bit_moments_follow_the_gradients(mt, dtype):
    mt.init(0, mt.BF16 if dtype == "bf16" else mt.FP32)
    m = train(mt, 1, bits=8)
    g, s = m.grads(), m.optimizer_state()
    for n in m.names:
        want_m, want_r = 0.1 * g[n].astype(np.float64), math.sqrt(1e-3) * np.abs(g[n].astype(np.float64))
        # a code is off by half a step (m) or a step (sqrt v): 2^-4 and 2^-3 of the value, or of 2^-6 of its block's scale,
        # which the block's largest value bounds by 2^-7.8 / 448 and 2^-9 / 224
        pad = lambda a: np.pad(a.ravel(), (0, -a.size % 32)).reshape(-1, 32)  # noqa: E731
        block = lambda a: np.repeat(pad(np.abs(a)).max(1), 32)[:a.size].reshape(a.shape)  # noqa: E731
        assert (np.abs(s["m"][n] - want_m) <= 1.001 * np.maximum(2.0 ** -4 * np.abs(want_m), 2.0 ** -10 / 224 * block(want_m)) + 1e-30).all(), n
        assert (np.abs(np.sqrt(s["v"][n].astype(np.float64)) - want_r) <= 1.001 * np.maximum(2.0 ** -3 * want_r, 2.0 ** -9 / 224 * block(want_r)) + 1e-30).all(), n
        assert (s["v"][n][g[n] != 0] > 0).all()
    mt.init(0, mt.FP32)


def test_eight_bit_moments_resume_bitwise(mt, tmp_path):
    a = train(mt, 3, bits=8, rates={"norm.weight": (1.0, 0.0)})
    a.save(str(tmp_path / "w"), str(tmp_path / "o"))
    b = mt.Model(**SPEC)
    b.set_adamw(lr=1e-2, weight_decay=0.1)
    b.set_adamw_state_bits(8)
    b.set_param_rates("norm.weight", 1.0, 0.0)
    b.load(str(tmp_path / "w"), str(tmp_path / "o"))
    train(mt, 3, model=a), train(mt, 3, model=b)
    for n in a.names:
        assert np.array_equal(a.get_param(n), b.get_param(n)), n
    with pytest.raises(mt.MtError, match="already exist"):
        a.set_adamw_state_bits(32)
    with pytest.raises(mt.MtError, match="8 or 32"):
        b.set_adamw_state_bits(16)


# ---- together ----------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_a_tuning_run(mt, dtype):
    """A QLoRA model with q / k norms: reference log-probabilities, then preference and policy steps with
    8-bit moments. Two runs give the same bits, and the margins move towards the chosen answers."""
    mt.init(0, mt.BF16 if dtype == "bf16" else mt.FP32)
    spec = dict(family="llama", vocab=515, d=128, layers=2, heads=2, kv_heads=1, dff=256, nctx=64, rope_all=1, qk_norm=1, qlora=1, rank=8,
                seed=3, ckpt=1)
    ids, targets = tokens(128, vocab=515)
    seq, w = np.arange(0, 129, 32, dtype=np.int32), np.ones(128, np.float32)
    w[::32] = w[1::32] = 0
    ends = []
    for _ in range(2):
        m = mt.Model(**spec)
        m.set_adamw(lr=3e-2, weight_decay=0.0)
        m.set_adamw_state_bits(8)
        refp = m.token_logprob(ids, targets, 32, weight=w)
        margins = []
        for k in range(6):
            margins.append(m.preference_step(ids, targets, seq, 32, ref_logp=refp, weight=w, beta=0.5)["margin"])
            m.clip_grad_norm(1.0)
            m.optimizer_step()
        old = m.token_logprob(ids, targets, 32, weight=w)
        out = m.policy_step(ids, targets, np.where(np.arange(128) % 2 == 0, 1.0, -1.0), 32, old_logp=old, ref_logp=refp, weight=w / w.sum(), kl_coef=0.05)
        m.optimizer_step()
        assert math.isfinite(out["loss"]) and np.array_equal(out["logp"], old)
        assert not margins[0].any()   # the policy is its own reference at first
        ends.append((m.state_dict(), np.stack(margins), out["loss"]))
        assert m.optimizer_steps() == 7
        m.close()
    assert np.array_equal(ends[0][1], ends[1][1]) and ends[0][2] == ends[1][2]
    for n in ends[0][0]:
        assert np.array_equal(ends[0][0][n], ends[1][0][n]), n
    mt.init(0, mt.FP32)
