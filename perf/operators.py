"""Cases, plain forms and 64-bit values of the operators of a preference- or policy-tuning step.

Four operators, each reached through the C entries of include/pk.h:

  policy      clipped policy loss with a KL term over rows of logits, and its gradient
              (pk_policy_loss)
  preference  log-probabilities of the targets, the paired log-ratio loss over sequences and the
              gradient of the logits (pk_token_logprob, pk_preference_loss, pk_token_logprob_bwd)
  qknorm      RMS norm of every query and key head with the rotary embedding in the same pass,
              forward and backward (pk_qk_norm_rope_fwd, pk_qk_norm_rope_bwd)
  adamw       one AdamW step over many tensors, moments in 32 or in 8 bits (pk_adamw_multi)

``own`` selects what ``run`` does: False computes the plain form with elementary torch operations
in 32 bits, True calls the library. ``exact`` restates every operator in 64 bits.
"""
import math
import random

import torch

own = False

_DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_BLOCK = 32  # elements that share one scale of an 8-bit moment


# ------------------------------------------------------------------------------- cases

def listed():
    return [
        # A few sampled continuations of an interactive tuning run: launch latency counts.
        {"name": "policy small", "op": "policy", "dtype": "bf16", "R": 48, "V": 32000, "pad": 0, "dead": 10, "old": True},
        # fp32 logits of a 50257-word vocabulary: rows start at every 4-byte offset.
        {"name": "policy fp32 odd", "op": "policy", "dtype": "fp32", "R": 1021, "V": 50257, "pad": 0, "dead": 0, "old": True},
        # Two 4096-token rollouts over the largest vocabulary; a quarter of the rows is prompt.
        {"name": "policy large", "op": "policy", "dtype": "bf16", "R": 8192, "V": 151936, "pad": 0, "dead": 25, "old": True},
        # One pair of short answers.
        {"name": "preference small", "op": "preference", "dtype": "bf16", "pairs": 1, "length": 40, "V": 32000, "pad": 0, "dead": 10},
        # Ragged answers over an odd vocabulary whose rows are padded to 16 bytes.
        {"name": "preference odd", "op": "preference", "dtype": "bf16", "pairs": 5, "length": 211, "V": 50257, "pad": 7, "dead": 20},
        # Eight pairs of up to 2048 tokens, 32000 words: 2 GB of logits.
        {"name": "preference large", "op": "preference", "dtype": "bf16", "pairs": 8, "length": 2048, "V": 32000, "pad": 0, "dead": 20},
        # The tokens of one small batch of the 14 / 2-head shape.
        {"name": "qknorm small", "op": "qknorm", "dir": "fwd", "dtype": "bf16", "T": 37, "Hq": 14, "Hkv": 2, "dk": 64, "rot": True, "packed": True},
        # 32 / 8 heads of 64 over 16 sequences of 4096 (one micro-batch of the 1B shape).
        {"name": "qknorm forward", "op": "qknorm", "dir": "fwd", "dtype": "bf16", "T": 65536, "Hq": 32, "Hkv": 8, "dk": 64, "rot": True, "packed": False},
        # 16 heads of 128, four sequences of 4096 with a ragged end, gradients of both gains.
        {"name": "qknorm backward", "op": "qknorm", "dir": "bwd", "dtype": "bf16", "T": 16381, "Hq": 16, "Hkv": 16, "dk": 128, "rot": True, "packed": True},
        # The LoRA matrices of the 24-layer QLoRA shape: 96 small tensors, 8-bit moments.
        {"name": "adamw adapters 8", "op": "adamw", "set": "lora", "count": 24, "largest": 0, "bits": 8, "g": "fp32", "shadow": True},
        # Every tensor of the GPT-2-small shape, 32-bit moments, gradients left in bf16.
        {"name": "adamw gpt2 32", "op": "adamw", "set": "gpt2", "count": 12, "largest": 0, "bits": 32, "g": "bf16", "shadow": True},
        # Four blocks of the 1B shape with moments in 8 bits.
        {"name": "adamw blocks 8", "op": "adamw", "set": "block", "count": 4, "largest": 0, "bits": 8, "g": "fp32", "shadow": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["policy", "preference", "qknorm", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op in ("policy", "preference"):
        V = rng.choice([32000, 50257, 151936, _log_int(rng, 300, 200000)])
        pad = rng.choice([0, 0, rng.randrange(1, 16)])
        dead = rng.choice([0, rng.randrange(1, 60)])
        rows = max(2, int(1e9 / V / (1 if dtype == "bf16" else 2)))
        if op == "policy":
            return {"op": op, "dtype": dtype, "R": _log_int(rng, 1, min(rows, 32768)), "V": V, "pad": pad, "dead": dead,
                    "old": rng.random() < 0.7}
        pairs = _log_int(rng, 1, max(1, min(64, rows // 16)))
        return {"op": op, "dtype": dtype, "pairs": pairs, "length": _log_int(rng, 8, max(8, min(2048, rows // (2 * pairs)))),
                "V": V, "pad": pad, "dead": dead}
    if op == "qknorm":
        Hkv = rng.choice([1, 2, 4, 8])
        Hq = Hkv * rng.choice([1, 2, 4, 7])
        dk = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        most = max(2, int(2e8 / ((Hq + Hkv) * dk)))
        return {"op": op, "dir": rng.choice(["fwd", "bwd"]), "dtype": dtype, "T": _log_int(rng, 1, min(most, 65536)), "Hq": Hq,
                "Hkv": Hkv, "dk": dk, "rot": rng.random() < 0.8, "packed": rng.random() < 0.5}
    return {"op": op, "set": "mixed", "count": _log_int(rng, 1, 300), "largest": _log_int(rng, 100, 4000000),
            "sizes": rng.randrange(1 << 30), "bits": rng.choice([8, 8, 32]), "g": rng.choice(["fp32", "bf16"]),
            "shadow": rng.random() < 0.7}


def _sizes(case):
    """Element counts of the tensors of an adamw case, in order."""
    n = case["count"]
    if case["set"] == "lora":  # rank 16 on q (896 -> 896) and v (896 -> 128)
        return [896 * 16, 16 * 896, 896 * 16, 16 * 128] * n
    if case["set"] == "gpt2":
        d = 768
        per = [d, d, d * 3 * d, 3 * d, d * d, d, d, d, d * 4 * d, 4 * d, 4 * d * d, d]
        return per * n + [50257 * d, 1024 * d, d, d]
    if case["set"] == "block":
        d, kv, f = 2048, 512, 8192
        return [d, d, d * d, d * kv, d * kv, d * d, d * f, d * f, f * d] * n
    r, sizes, left = random.Random(case["sizes"]), [], 60_000_000
    for _ in range(n):
        k = min(_log_int(r, 1, case["largest"]), max(1, left))
        left -= k
        sizes.append(k)
    return sizes


def _seqs(case, seed):
    """Offsets of 2 * pairs ragged sequences, between half the length and the whole."""
    r, at = random.Random(seed * 7 + 1), [0]
    for _ in range(2 * case["pairs"]):
        at.append(at[-1] + r.randint(max(1, case["length"] // 2), case["length"]))
    return at


def _rows_most(case):
    return 2 * case["pairs"] * case["length"]


# ------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(int(seed) * 1000003 + 17)


def _logits(case, R, g):
    """Logits [R, V] (rows V + pad apart) with one likelier word per row, the targets, and the
    log-probability of each target."""
    V, dt = case["V"], _DT[case["dtype"]]
    x = torch.empty(R, V + case["pad"], device=_DEV, dtype=dt)
    step = max(1, (1 << 27) // (V + case["pad"]))
    for a in range(0, R, step):
        x[a:a + step] = torch.randn(min(step, R - a), V + case["pad"], device=_DEV, generator=g) * 2.0
    x = x[:, :V]
    t = torch.randint(0, V, (R,), device=_DEV, generator=g)
    r = torch.arange(R, device=_DEV)
    x[r, t] += (torch.rand(R, device=_DEV, generator=g) * 10 + 3).to(dt)
    logp = torch.empty(R, device=_DEV)
    for a in range(0, R, step):
        logp[a:a + step] = x[r[a:a + step], t[a:a + step]].float() - torch.logsumexp(x[a:a + step].float(), 1)
    return x, t.to(torch.int32), logp


def _live(R, percent, g):
    w = (torch.rand(R, device=_DEV, generator=g) * 100 >= percent).float()
    return w


_CLIP = (0.2, 0.28)
_KL, _BETA, _SMOOTH = 0.04, 0.1, 0.05


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case, "op": case["op"]}
    if case["op"] == "policy":
        R, V = case["R"], case["V"]
        x, t, logp = _logits(case, R, g)
        d = torch.randn(R, device=_DEV, generator=g) * 0.25
        # the gradient jumps where a ratio crosses its bound: no sampled ratio sits on one
        for b in (math.log(1 - _CLIP[0]), math.log(1 + _CLIP[1])):
            d = torch.where((d - b).abs() < 1e-3, torch.full_like(d, b + 2e-3), d)
        live = _live(R, case["dead"], g)
        t = torch.where(live == 0, torch.full_like(t, -100), t)  # labels of prompt and padding rows
        s |= {"x": x, "t": t, "old": (logp - d) if case["old"] else None,
              "ref": logp + torch.randn(R, device=_DEV, generator=g) * 0.3,
              "adv": torch.randn(R, device=_DEV, generator=g), "w": live / max(1.0, R * (100 - case["dead"]) / 100),
              "loss": torch.zeros(R, device=_DEV), "logp": torch.zeros(R, device=_DEV), "kl": torch.zeros(R, device=_DEV),
              "dx": torch.zeros(R, V + case["pad"], device=_DEV, dtype=x.dtype)[:, :V]}
    elif case["op"] == "preference":
        at, V = _seqs(case, seed), case["V"]
        R = _rows_most(case)  # rows behind the last sequence are padding
        x, t, logp = _logits(case, R, g)
        w = _live(R, case["dead"], g)
        w[at[-1]:] = 0
        t = torch.where(w == 0, torch.full_like(t, -100), t)
        P = case["pairs"]
        # the policy has moved towards the chosen answers, by about the same for a whole answer of any length
        start = torch.tensor(at, device=_DEV)
        sign = 1 - 2.0 * (torch.searchsorted(start[1:], torch.arange(R, device=_DEV), right=True) % 2)
        ref = logp - sign * 15 / case["length"] + torch.randn(R, device=_DEV, generator=g) * 0.3
        s |= {"x": x, "t": t, "w": w, "ref": ref,
              "seq": torch.tensor(at, device=_DEV, dtype=torch.int32),
              "logp": torch.zeros(R, device=_DEV), "lse": torch.zeros(R, device=_DEV), "dlogp": torch.zeros(R, device=_DEV),
              "loss": torch.zeros(P, device=_DEV), "margin": torch.zeros(P, device=_DEV),
              "dx": torch.zeros(R, V + case["pad"], device=_DEV, dtype=x.dtype)[:, :V]}
    elif case["op"] == "qknorm":
        T, Hq, Hkv, dk, dt = case["T"], case["Hq"], case["Hkv"], case["dk"], _DT[case["dtype"]]

        def qk():
            if case["packed"]:  # column ranges of one q | k | v projection
                z = torch.randn(T, (Hq + 2 * Hkv) * dk, device=_DEV, generator=g).to(dt)
                return z[:, :Hq * dk], z[:, Hq * dk:(Hq + Hkv) * dk]
            return (torch.randn(T, Hq * dk, device=_DEV, generator=g).to(dt),
                    torch.randn(T, Hkv * dk, device=_DEV, generator=g).to(dt))

        S = min(T, 4096)
        ang = (torch.arange(S, device=_DEV, dtype=torch.float64)[:, None]
               * (5e5 ** (-torch.arange(0, dk, 2, device=_DEV, dtype=torch.float64) / dk))[None])
        q, k = qk()
        s |= {"q": q, "k": k, "wq": 1 + 0.2 * torch.randn(dk, device=_DEV, generator=g),
              "wk": 1 + 0.2 * torch.randn(dk, device=_DEV, generator=g),
              "pos": (torch.arange(T, device=_DEV) % S).to(torch.int32),
              "cs": torch.stack([ang.cos(), ang.sin()], -1).float().contiguous(),
              "oq": torch.zeros(T, Hq * dk, device=_DEV, dtype=dt), "ok": torch.zeros(T, Hkv * dk, device=_DEV, dtype=dt)}
        if case["dir"] == "bwd":
            gq, gk = qk()
            s |= {"gq": gq, "gk": gk, "dwq": torch.zeros(dk, device=_DEV), "dwk": torch.zeros(dk, device=_DEV)}
            if own:
                n = _lib().libpk().pk_qk_norm_rope_bwd_scratch_bytes(T, Hq, Hkv, dk)
                s["scratch"] = torch.empty(max(16, n), device=_DEV, dtype=torch.uint8)
    else:
        n = _sizes(case)
        at, total = [], 0
        for k in n:
            at.append(total)
            total += -(-k // _BLOCK) * _BLOCK
        inside = torch.zeros(total, device=_DEV)
        for a, k in zip(at, n):
            inside[a:a + k] = 1
        blocks = total // _BLOCK
        wide = torch.exp(torch.randn(blocks, device=_DEV, generator=g) * 1.5).repeat_interleave(_BLOCK) * inside * 1e-3
        grad = (torch.randn(total, device=_DEV, generator=g) * wide).to(_DT[case["g"]])
        m = torch.randn(total, device=_DEV, generator=g) * wide * 0.3
        r = (torch.rand(total, device=_DEV, generator=g) + 0.5) * wide
        s |= {"n": n, "at": at, "p": torch.randn(total, device=_DEV, generator=g) * 0.02 * inside, "g": grad, "t": 101,
              "decay": [0.0 if k < 4096 else 0.1 for k in n],  # norm gains and biases are not decayed
              "rate": [1.0 if i % 3 else 0.5 for i in range(len(n))], "seed": 1234567 + int(seed)}
        s["shadow"] = s["p"].to(torch.bfloat16) if case["shadow"] else None
        if case["bits"] == 8:
            s["m"], s["ms"] = _pack(m, None)
            s["v"], s["vs"] = _pack(r, torch.zeros(total, device=_DEV, dtype=torch.int64))
        else:
            s["m"], s["v"], s["ms"], s["vs"] = m, r * r, None, None
        # one number per block, kept beside the tensors as a program keeps its parameter groups
        lens = torch.tensor([-(-k // _BLOCK) for k in n], device=_DEV)
        s["block_decay"] = torch.tensor(s["decay"], device=_DEV).repeat_interleave(lens)
        s["block_rate"] = torch.tensor(s["rate"], device=_DEV).repeat_interleave(lens)
        if own:
            s["plan"] = _plan(s)
    return s


# ------------------------------------------------------------------------------- plain forms

def _policy(s):
    """-min(r A, clip(r) A) + kl (e^u - u - 1), r = exp(logp - old), u = ref - logp, per row."""
    x, live = s["x"].float(), s["w"] != 0
    t = torch.where(live, s["t"], torch.zeros_like(s["t"])).long()[:, None]
    mx = x.max(1, keepdim=True).values
    e = torch.exp(x - mx)
    total = e.sum(1, keepdim=True)
    logp = (x.gather(1, t) - mx - torch.log(total))[:, 0]
    d = (logp - s["old"]) if s["old"] is not None else torch.zeros_like(logp)
    r, a, w = torch.exp(d), s["adv"], s["w"]
    u = (s["ref"] - logp).double()
    kl = (torch.expm1(u) - u).float()
    free, held = r * a, r.clamp(1 - _CLIP[0], 1 + _CLIP[1]) * a
    loss = w * (-torch.minimum(free, held) + _KL * kl)
    gl = w * (torch.where(free <= held, -free, torch.zeros_like(free)) + _KL * (1 - torch.exp(s["ref"] - logp)))
    zero = torch.zeros_like(logp)
    gl = torch.where(live, gl, zero)[:, None]
    dx = e / total * -gl
    dx.scatter_add_(1, t, gl)
    s["dx"].copy_(torch.where(live[:, None], dx, torch.zeros((), device=dx.device)))
    return {"loss": torch.where(live, loss, zero), "logp": torch.where(live, logp, zero),
            "kl": torch.where(live, kl, zero), "dx": s["dx"]}


def _preference(s):
    """-(1 - e) log sigmoid(z) - e log sigmoid(-z), z = beta (sum of chosen - sum of rejected log ratios)."""
    x, w = s["x"].float(), s["w"]
    live = w != 0
    t = torch.where(live, s["t"], torch.zeros_like(s["t"])).long()[:, None]
    mx = x.max(1, keepdim=True).values
    e = torch.exp(x - mx)
    total = e.sum(1, keepdim=True)
    lse = (mx + torch.log(total))[:, 0]
    logp = x.gather(1, t)[:, 0] - lse
    zero = torch.zeros_like(logp)
    logp, lse = torch.where(live, logp, zero), torch.where(live, lse, zero)
    P, R = s["loss"].numel(), logp.numel()
    ratio = torch.where(live, w * (logp - s["ref"]), zero).double()
    upto = torch.cat([torch.zeros(1, device=_DEV, dtype=torch.float64), ratio.cumsum(0)])
    ends = upto[s["seq"].long()]
    sums = (ends[1:] - ends[:-1]).view(P, 2)
    z = _BETA * (sums[:, 0] - sums[:, 1])
    down, up = torch.log1p(torch.exp(-z.abs())) + (-z).clamp(min=0), torch.log1p(torch.exp(-z.abs())) + z.clamp(min=0)
    loss = (1 - _SMOOTH) * down + _SMOOTH * up
    dz = (_SMOOTH - 1 / (1 + torch.exp(z))).float() / P
    which = torch.searchsorted(s["seq"][1:].long(), torch.arange(R, device=_DEV), right=True).clamp(max=2 * P - 1)
    sign = torch.where(which % 2 == 0, torch.ones_like(logp), -torch.ones_like(logp))
    gl = torch.where(live, _BETA * dz[which // 2] * sign * w, zero)
    dx = e / total * -gl[:, None]
    dx.scatter_add_(1, t, gl[:, None])
    s["dx"].copy_(torch.where(live[:, None], dx, torch.zeros((), device=dx.device)))
    return {"logp": logp, "lse": lse, "loss": loss.float(), "margin": z.float(), "dlogp": gl, "dx": s["dx"]}


_EPS = 1e-6


def _norm_rope(x, H, w, c, sn, rot):
    T, dk = x.shape[0], w.numel()
    x = x.float().reshape(T, H, dk)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w
    if rot:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * c - b * sn, a * sn + b * c], -1)
    return y.reshape(T, H * dk)


def _norm_rope_back(g, x, H, w, c, sn, rot):
    T, dk = x.shape[0], w.numel()
    x, g = x.float().reshape(T, H, dk), g.float().reshape(T, H, dk)
    if rot:
        a, b = g[..., 0::2], g[..., 1::2]
        g = torch.stack([a * c + b * sn, b * c - a * sn], -1).reshape(T, H, dk)
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    hat = x * inv
    gw = g * w
    dx = inv * (gw - hat * (gw * hat).mean(-1, keepdim=True))
    return dx.reshape(T, H * dk), (g * hat).sum((0, 1))


def _qknorm(s):
    c, sn = s["cs"][s["pos"].long()].unbind(-1)
    c, sn, k = c[:, None], sn[:, None], s["case"]
    if k["dir"] == "fwd":
        s["oq"].copy_(_norm_rope(s["q"], k["Hq"], s["wq"], c, sn, k["rot"]))
        s["ok"].copy_(_norm_rope(s["k"], k["Hkv"], s["wk"], c, sn, k["rot"]))
        return {"q": s["oq"], "k": s["ok"]}
    dq, dwq = _norm_rope_back(s["gq"], s["q"], k["Hq"], s["wq"], c, sn, k["rot"])
    dkk, dwk = _norm_rope_back(s["gk"], s["k"], k["Hkv"], s["wk"], c, sn, k["rot"])
    s["oq"].copy_(dq)
    s["ok"].copy_(dkk)
    s["dwq"] += dwq
    s["dwk"] += dwk
    return {"dq": s["oq"], "dk": s["ok"], "dwq": s["dwq"], "dwk": s["dwk"]}


_LR, _B1, _B2, _ADAM_EPS = 1e-4, 0.9, 0.999, 1e-8


def _f32(v):
    return float(torch.tensor(v, dtype=torch.float32))


def _rates(t):
    """The step's numbers as the fp32 values that the entry takes."""
    b1, b2 = _f32(_B1), _f32(_B2)
    return _f32(_LR), b1, b2, _f32(_ADAM_EPS), _f32(1 - b1 ** t), _f32(1 - b2 ** t)


def _mix32(v):
    v &= 0xFFFFFFFF
    v = ((v ^ (v >> 16)) * 0x9E3779B1) & 0xFFFFFFFF
    v = ((v ^ (v >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return v ^ (v >> 16)


def _random_bits(total, seed):
    """20 bits for each element's rounding: a function of the seed and the element's number."""
    i = torch.arange(total, device=_DEV, dtype=torch.int64)
    v = _mix32((seed & 0xFFFFFFFF) + 0x632BE5AB * (seed >> 32))
    return _mix32(i + 0x3C6EF372 * (i >> 32) ^ v) & 0xFFFFF


def _scale(x):
    """Per block of 32 the power of two 2^e with max|x| / 2^e in (224, 448], e >= -126, as its byte e + 127."""
    f, e = torch.frexp(x.abs().view(-1, _BLOCK).amax(1))  # max = f 2^e, f in [0.5, 1)
    b = torch.where(f > 0.875, e - 8, e - 9) + 127
    return torch.where(f == 0, torch.ones_like(b), b.clamp(1, 254)).to(torch.uint8)


def _pack(x, bits):
    """E4M3 codes and block scales of x: to the nearest, or, with random bits, up or down by chance
    (and then no value above zero becomes zero)."""
    b = _scale(x)
    y = x * torch.ldexp(torch.ones_like(b, dtype=torch.float32), 127 - b.int()).repeat_interleave(_BLOCK)
    if bits is not None:
        # steps of 2^-9 below 2^-6: shifted up by 2^-6 the same cut of the mantissa gives them
        low = y < 2.0 ** -6
        z = torch.where(low, y + 2.0 ** -6, y)
        z = ((z.view(torch.int32) + bits.int()) & ~0xFFFFF).view(torch.float32)
        z = torch.where(low, z - 2.0 ** -6, z)
        y = torch.where((x > 0) & (z == 0), torch.full_like(z, 2.0 ** -9), z)
    return y.to(torch.float8_e4m3fn), b


def _unpack(c, b):
    return c.float() * torch.ldexp(torch.ones_like(b, dtype=torch.float32), b.int() - 127).repeat_interleave(_BLOCK)


def _adamw(s):
    lr, b1, b2, eps, c1, c2 = _rates(s["t"])
    bits, g, p = s["case"]["bits"], s["g"].float(), s["p"]
    m, v = (_unpack(s["m"], s["ms"]), _unpack(s["v"], s["vs"]).square()) if bits == 8 else (s["m"], s["v"])
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    up = (m / c1) / (torch.sqrt(v / c2) + eps) + s["block_decay"].repeat_interleave(_BLOCK) * p
    p -= (lr * s["block_rate"]).repeat_interleave(_BLOCK) * up
    if bits == 8:
        c, e = _pack(m, None)
        s["m"].copy_(c), s["ms"].copy_(e)
        c, e = _pack(torch.sqrt(v), _random_bits(v.numel(), s["seed"]))
        s["v"].copy_(c), s["vs"].copy_(e)
    else:
        s["m"].copy_(m), s["v"].copy_(v)
    if s["shadow"] is not None:
        s["shadow"].copy_(p)
    return _adamw_out(s)


def _adamw_out(s):
    """The updated buffers; block scales as the powers of two that their bytes stand for."""
    power = lambda b: None if b is None else b.view(torch.float8_e8m0fnu)  # noqa: E731
    return {"p": s["p"], "m": s["m"], "v": s["v"], "ms": power(s["ms"]), "vs": power(s["vs"]), "shadow": s["shadow"]}


# ------------------------------------------------------------------------------- the library's calls

def _lib():
    from paperkiln_b200 import _capi
    return _capi


def _ptr(t):
    return None if t is None else t.data_ptr()


def _dt(t):
    return 1 if t.dtype == torch.bfloat16 else 0


def _plan(s):
    """The handle of the many-tensor step: made once, as a program makes its optimizer."""
    c, out = _lib(), []
    size = {torch.float32: 4, torch.bfloat16: 2}
    for i, (a, n) in enumerate(zip(s["at"], s["n"])):
        wide = 1 if s["ms"] is not None else 4
        out.append(c.AdamwTensor(
            p=s["p"].data_ptr() + 4 * a, g=s["g"].data_ptr() + size[s["g"].dtype] * a,
            m=s["m"].data_ptr() + wide * a, v=s["v"].data_ptr() + wide * a,
            m_scale=s["ms"].data_ptr() + a // _BLOCK if wide == 1 else None,
            v_scale=s["vs"].data_ptr() + a // _BLOCK if wide == 1 else None,
            shadow=s["shadow"].data_ptr() + 2 * a if s["shadow"] is not None else None, n=n, lr_mult=s["rate"][i],
            weight_decay=s["decay"][i]))
    return c.AdamwPlan(out, g_dtype=_dt(s["g"]), state_bits=s["case"]["bits"])


def _run_own(s):
    c = _lib()
    pk, k, st = c.libpk(), s["case"], torch.cuda.current_stream().cuda_stream
    if s["op"] == "policy":
        x, dx = s["x"], s["dx"]
        c.check(pk.pk_policy_loss(st, _dt(x), _ptr(x), x.stride(0), _ptr(s["t"]), _ptr(s["old"]), _ptr(s["ref"]), _ptr(s["adv"]),
                                  _ptr(s["w"]), _CLIP[0], _CLIP[1], _KL, 1.0, _ptr(s["loss"]), _ptr(s["logp"]), _ptr(s["kl"]),
                                  _ptr(dx), dx.stride(0), x.shape[0], x.shape[1], None))
        return {"loss": s["loss"], "logp": s["logp"], "kl": s["kl"], "dx": dx}
    if s["op"] == "preference":
        x, dx = s["x"], s["dx"]
        R, V, P = x.shape[0], x.shape[1], s["loss"].numel()
        c.check(pk.pk_token_logprob(st, _dt(x), _ptr(x), x.stride(0), _ptr(s["t"]), _ptr(s["w"]), _ptr(s["logp"]), _ptr(s["lse"]),
                                    R, V, None))
        c.check(pk.pk_preference_loss(st, _ptr(s["logp"]), _ptr(s["ref"]), _ptr(s["w"]), _ptr(s["seq"]), P, R, _BETA, _SMOOTH,
                                      1.0 / P, _ptr(s["loss"]), _ptr(s["margin"]), _ptr(s["dlogp"]), None))
        c.check(pk.pk_token_logprob_bwd(st, _dt(x), _ptr(x), x.stride(0), _ptr(s["t"]), _ptr(s["lse"]), _ptr(s["dlogp"]), _ptr(dx),
                                        dx.stride(0), R, V, None))
        return {"logp": s["logp"], "lse": s["lse"], "loss": s["loss"], "margin": s["margin"], "dlogp": s["dlogp"], "dx": dx}
    if s["op"] == "qknorm":
        q, kk, T, Hq, Hkv, dk = s["q"], s["k"], k["T"], k["Hq"], k["Hkv"], k["dk"]
        rq, rk = (Hq, Hkv) if k["rot"] else (0, 0)
        if k["dir"] == "fwd":
            c.check(pk.pk_qk_norm_rope_fwd(st, _dt(q), _ptr(q), q.stride(0), _ptr(kk), kk.stride(0), _ptr(s["wq"]), _ptr(s["wk"]),
                                           _ptr(s["oq"]), Hq * dk, _ptr(s["ok"]), Hkv * dk, T, Hq, Hkv, dk, rq, rk, _EPS,
                                           _ptr(s["pos"]), _ptr(s["cs"]), s["cs"].shape[0]))
            return {"q": s["oq"], "k": s["ok"]}
        gq, gk = s["gq"], s["gk"]
        c.check(pk.pk_qk_norm_rope_bwd(st, _dt(q), _ptr(gq), gq.stride(0), _ptr(gk), gk.stride(0), _ptr(q), q.stride(0), _ptr(kk),
                                       kk.stride(0), _ptr(s["wq"]), _ptr(s["wk"]), _ptr(s["oq"]), Hq * dk, _ptr(s["ok"]), Hkv * dk,
                                       _ptr(s["dwq"]), _ptr(s["dwk"]), _ptr(s["scratch"]), T, Hq, Hkv, dk, rq, rk, _EPS,
                                       _ptr(s["pos"]), _ptr(s["cs"]), s["cs"].shape[0]))
        return {"dq": s["oq"], "dk": s["ok"], "dwq": s["dwq"], "dwk": s["dwk"]}
    lr, b1, b2, eps, c1, c2 = _rates(s["t"])
    c.check(pk.pk_adamw_multi(st, s["plan"].handle, lr, b1, b2, eps, c1, c2, s["seed"]))
    return _adamw_out(s)


def run(state):
    if own:
        return _run_own(state)
    return {"policy": _policy, "preference": _preference, "qknorm": _qknorm, "adamw": _adamw}[state["op"]](state)


# ------------------------------------------------------------------------------- work

def work(case):
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        state = 4 * (1 + 1 / _BLOCK) if case["bits"] == 8 else 16  # both moments, read and written
        return {"bytes": n * (8 + (4 if case["g"] == "fp32" else 2) + state + (2 if case["shadow"] else 0)), "flops": 16 * n}
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "qknorm":
        n = case["T"] * (case["Hq"] + case["Hkv"]) * case["dk"]
        back = case["dir"] == "bwd"
        table = min(case["T"], 4096) * case["dk"] * 4 + case["T"] * 4 if case["rot"] else 0
        return {"bytes": n * e * (3 if back else 2) + table, "flops": n * (14 if back else 8)}
    if case["op"] == "policy":
        R, live = case["R"], 1 - case["dead"] / 100
    else:
        R = _rows_most(case)
        live = 0.75 * (1 - case["dead"] / 100)  # sequences fill three quarters on average
    return {"bytes": R * case["V"] * e * (1 + live) + R * 32, "flops": 6 * live * R * case["V"]}


# ------------------------------------------------------------------------------- in 64 bits

def _exact_rows(x, t, live):
    """log-sum-exp and the target's log-probability of every row that counts, in 64 bits."""
    R = x.shape[0]
    lse, logp = torch.zeros(R, device=_DEV, dtype=torch.float64), torch.zeros(R, device=_DEV, dtype=torch.float64)
    step = max(1, (1 << 27) // x.shape[1])
    for a in range(0, R, step):
        z = x[a:a + step].double()
        lse[a:a + step] = torch.logsumexp(z, 1)
        logp[a:a + step] = z.gather(1, t[a:a + step].long().clamp(min=0)[:, None])[:, 0] - lse[a:a + step]
    return lse * live, logp * live


def _exact_dx(x, t, lse, gl):
    R, step = x.shape[0], max(1, (1 << 27) // x.shape[1])
    dx = torch.empty(x.shape, device=_DEV, dtype=torch.float64)
    for a in range(0, R, step):
        gz = gl[a:a + step, None]
        z = -gz * torch.exp(x[a:a + step].double() - lse[a:a + step, None])
        z.scatter_add_(1, t[a:a + step].long().clamp(min=0)[:, None], gz)
        z[gl[a:a + step] == 0] = 0
        dx[a:a + step] = z
    return dx


def _exact_policy(s):
    w, live = s["w"].double(), (s["w"] != 0).double()
    lse, logp = _exact_rows(s["x"], s["t"], live)
    r = torch.exp(logp - s["old"].double()) if s["old"] is not None else torch.ones_like(logp)
    u, a = s["ref"].double() - logp, s["adv"].double()
    lo, hi = 1 - _f32(_CLIP[0]), 1 + _f32(_CLIP[1])
    # with a positive advantage only the upper bound holds the ratio back, with a negative one the lower
    held = torch.where(a >= 0, r > hi, r < lo)
    kl = torch.expm1(u) - u
    loss = w * (-a * torch.where(a >= 0, r.clamp(max=hi), r.clamp(min=lo)) + _f32(_KL) * kl)
    gl = w * (-(a * r) * (~held).double() - _f32(_KL) * torch.expm1(u))
    return {"loss": loss, "logp": logp, "kl": kl * live, "dx": _exact_dx(s["x"], s["t"], lse, gl)}


def _exact_preference(s):
    w, live = s["w"].double(), (s["w"] != 0).double()
    lse, logp = _exact_rows(s["x"], s["t"], live)
    ratio, at = w * (logp - s["ref"].double()), s["seq"].tolist()
    P = len(at) // 2
    gl, loss, margin = torch.zeros_like(logp), [], []
    for i in range(P):
        a, b, c = at[2 * i], at[2 * i + 1], at[2 * i + 2]
        z = _f32(_BETA) * float(ratio[a:b].sum() - ratio[b:c].sum())
        soft = lambda v: math.log1p(math.exp(-abs(v))) + max(0.0, v)  # noqa: E731
        e = _f32(_SMOOTH)
        loss.append((1 - e) * soft(-z) + e * soft(z))
        margin.append(z)
        dz = (e - 1 / (1 + math.exp(z))) / P
        gl[a:b] = _f32(_BETA) * dz * w[a:b]
        gl[b:c] = -_f32(_BETA) * dz * w[b:c]
    as64 = lambda v: torch.tensor(v, device=_DEV, dtype=torch.float64)  # noqa: E731
    return {"logp": logp, "lse": lse, "loss": as64(loss), "margin": as64(margin), "dlogp": gl,
            "dx": _exact_dx(s["x"], s["t"], lse, gl)}


def _exact_qknorm(s):
    k, dk = s["case"], s["case"]["dk"]
    z = torch.view_as_complex(s["cs"].double())[s["pos"].long()][:, None] if k["rot"] else None

    def turn(v, by):
        return v if by is None else torch.view_as_real(torch.view_as_complex(v.unflatten(-1, (-1, 2)).contiguous()) * by).flatten(-2)

    got = []
    for x, g, w, H in ((s["q"], s.get("gq"), s["wq"], k["Hq"]), (s["k"], s.get("gk"), s["wk"], k["Hkv"])):
        x, w = x.double().unflatten(-1, (H, dk)), w.double()
        n = (x.square().mean(-1, keepdim=True) + _f32(_EPS)).sqrt()
        if g is None:
            got.append(turn(x / n * w, z).flatten(-2))
            continue
        g = turn(g.double().unflatten(-1, (H, dk)), None if z is None else z.conj())
        proj = (g * w * x).sum(-1, keepdim=True) / (dk * n * n)
        got += [((g * w - x * proj) / n).flatten(-2), (g * x / n).sum((0, 1))]
    if k["dir"] == "fwd":
        return {"q": got[0], "k": got[1]}
    return {"dq": got[0], "dk": got[2], "dwq": got[1], "dwk": got[3]}


def _exact_codes(x, bits):
    """Values that 8-bit codes of x (64 bits) stand for before scaling, and the scales."""
    top = x.abs().view(-1, _BLOCK).amax(1)
    e = torch.where(top > 0, torch.ceil(torch.log2(top / 448)), torch.full_like(top, -126)).clamp(-126, 127)
    y = x / torch.exp2(e).repeat_interleave(_BLOCK)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    if bits is None:
        q = torch.round(y / step) * step
    else:
        q = torch.floor(y / step + bits.double() / 2 ** 20) * step
        q = torch.where((x > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
    return q, torch.exp2(e)


def _exact_adamw(s):
    lr, b1, b2, eps, c1, c2 = _rates(s["t"])
    bits, g, p = s["case"]["bits"], s["g"].double(), s["p"].double()
    if bits == 8:
        m = s["m"].double() * torch.exp2(s["ms"].double() - 127).repeat_interleave(_BLOCK)
        v = (s["v"].double() * torch.exp2(s["vs"].double() - 127).repeat_interleave(_BLOCK)).square()
    else:
        m, v = s["m"].double(), s["v"].double()
    m = m + (1 - b1) * (g - m)
    v = v + (1 - b2) * (g * g - v)
    decay = torch.tensor([_f32(d) for d in s["decay"]], device=_DEV, dtype=torch.float64)
    rate = torch.tensor([_f32(d) for d in s["rate"]], device=_DEV, dtype=torch.float64)
    lens = torch.tensor([-(-k // _BLOCK) * _BLOCK for k in s["n"]], device=_DEV)
    p = p - lr * rate.repeat_interleave(lens) * (m / c1 / ((v / c2).sqrt() + eps) + decay.repeat_interleave(lens) * p)
    out = {"p": p, "m": m, "v": v, "ms": None, "vs": None, "shadow": p if s["shadow"] is not None else None}
    if bits == 8:
        out["m"], out["ms"] = _exact_codes(m, None)
        out["v"], out["vs"] = _exact_codes(v.sqrt(), _random_bits(v.numel(), s["seed"]))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"policy": _exact_policy, "preference": _exact_preference, "qknorm": _exact_qknorm, "adamw": _exact_adamw}[case["op"]](s)
