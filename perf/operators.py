"""Operators of a decoder's training step beside the AXS-6 Linear: rotary positions, attention with its backward pass and
distillation from a teacher's top logits.  Each in its plain form (elementary torch operations in 32 bits, angles in 64) and
as the calls that a user makes of this package.

A case is a dict of plain values.  ``op`` names the operator; the other keys are its sizes, its types and its masks.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # ---- rotary positions
        # one generated token for each of 16 requests, at far positions: latency
        rotary("rotary_token", B=16, S=1, Hq=16, Hkv=16, D=64, R=64, layout="half", far=131072, train=False),
        # the step of the benchmark's 12-layer GPT (batch 8, sequence 1024, 16 heads of 64): forward and backward
        rotary("rotary_train", B=8, S=1024, Hq=16, Hkv=16, D=64, R=64, layout="interleaved", far=0, train=True),
        # one long document with shared key heads, half of each head rotated, scaled for sixteen times the length
        rotary("rotary_long", B=1, S=65536, Hq=32, Hkv=8, D=128, R=64, layout="half", far=0, train=False, scaling="yarn", factor=16.0),
        # fp32 graph, odd sizes, one key head
        rotary("rotary_fp32_odd", B=3, S=2039, Hq=5, Hkv=1, D=72, R=36, layout="half", far=4096, train=True, dtype="fp32", scaling="linear", factor=4.0),
        # ---- attention
        # one generated token for each of 16 requests over caches of up to 8192 tokens, four query heads to a key head
        attention("attention_token", B=16, Hq=32, Hkv=8, Sq=1, Sk=8192, D=128, lengths=True, train=False),
        # the step of the benchmark's 12-layer GPT
        attention("attention_train", B=8, Hq=16, Hkv=16, Sq=1024, Sk=1024, D=64, causal=True, train=True),
        # one long sequence, four query heads to a key head: the largest
        attention("attention_train_long", B=1, Hq=32, Hkv=8, Sq=8192, Sk=8192, D=128, causal=True, train=True),
        # a padded batch of an encoder, odd lengths, a head size between the powers of two
        attention("attention_padded", B=6, Hq=12, Hkv=4, Sq=1531, Sk=1531, D=96, lengths=True, train=True),
        # a sliding window, the queries the last part of the keys
        attention("attention_window", B=2, Hq=16, Hkv=2, Sq=1000, Sk=9001, D=128, causal=True, window=2048, train=False),
        # the fp32 modules: a mask tensor added to the scores
        attention("attention_fp32_mask", B=2, Hq=8, Hkv=8, Sq=512, Sk=512, D=64, mask="added", train=True, dtype="fp32"),
        # ---- distillation
        # a few positions of a small batch: latency
        distillation("distill_few", T=7, V=32000, K=20, temperature=1.0),
        # the benchmark's vocabulary and batch
        distillation("distill_train", T=8192, V=32000, K=64, temperature=2.0),
    ]


def rotary(name, B, S, Hq, Hkv, D, R, layout, far, train, dtype="bf16", scaling="none", factor=1.0):
    """``far``: the first position of a batch entry lies in [0, far]."""
    return {"name": name, "op": "rotary", "B": B, "S": S, "Hq": Hq, "Hkv": Hkv, "D": D, "R": R, "layout": layout, "far": far, "train": train,
            "dtype": dtype, "scaling": scaling, "factor": factor}


def attention(name, B, Hq, Hkv, Sq, Sk, D, causal=False, window=0, lengths=False, mask="none", train=False, dtype="bf16"):
    """``window`` 0: none.  ``lengths``: each batch entry has its own number of keys.  ``mask``: none, "added" (values added to the scores,
    -inf among them) or "kept" (truth values), one for every batch entry and shared by the heads."""
    return {"name": name, "op": "attention", "B": B, "Hq": Hq, "Hkv": Hkv, "Sq": Sq, "Sk": Sk, "D": D, "causal": causal, "window": window,
            "lengths": lengths, "mask": mask, "train": train, "dtype": dtype}


def distillation(name, T, V, K, temperature, dtype="bf16"):
    return {"name": name, "op": "distillation", "T": T, "V": V, "K": K, "temperature": temperature, "dtype": dtype}


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    op = rng.choice(["rotary", "attention", "attention", "distillation"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if op == "rotary":
        D = rng.choice([32, 40, 64, 64, 72, 80, 96, 128, 128, 256])
        R = rng.choice([D, D, D // 2, D // 4 * 2 - 4])
        Hkv = rng.choice([1, 2, 4, 8])
        Hq = Hkv * rng.choice([1, 2, 3, 4])
        B = spread(1, 16)
        room = 300_000_000 // (B * (Hq + Hkv) * D)
        S = spread(1, min(65536, max(1, room // 4)))
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        c = rotary("", B, S, Hq, Hkv, D, R, rng.choice(["half", "interleaved"]), rng.choice([0, 1000, 200000]), rng.choice([True, False]),
                   dtype, scaling, 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]))
    elif op == "attention":
        D = rng.choice([16, 40, 64, 64, 80, 96, 128, 128])
        Hkv = rng.choice([1, 2, 3, 4, 8])
        Hq = Hkv * rng.choice([1, 1, 2, 4, 8])
        B = spread(1, 16)
        train = rng.choice([True, True, False])
        most = (1 << 28) if dtype == "bf16" else (1 << 25)          # scores of all heads
        if not train and rng.random() < 0.5:                        # few queries over a long cache
            Sq = spread(1, 16)
            Sk = spread(max(Sq, 64), max(64, min(65536, most // (B * Hq * Sq), (1 << 29) // (B * Hkv * D))))
        else:
            side = int(math.sqrt(most / (B * Hq)))
            Sq = spread(16, max(16, min(4096, side)))
            Sk = Sq if rng.random() < 0.6 else spread(16, max(16, min(8192, most // (B * Hq * Sq))))
        causal = rng.choice([True, True, False])
        window = rng.choice([0, 0, spread(1, Sk)]) if causal else 0
        mask = "none" if causal else rng.choice(["none", "none", "added" if B * Sq * Sk <= 1 << 26 else "kept", "kept"])
        c = attention("", B, Hq, Hkv, Sq, Sk, D, causal, window, rng.random() < 0.4, mask, train, dtype)
    else:
        V = rng.choice([spread(200, 150000), spread(20000, 150000), 8 * spread(2500, 19000)])
        T = spread(1, max(1, min(16384, (240_000_000 if dtype == "bf16" else 120_000_000) // V)))
        c = distillation("", T, V, spread(1, min(256, V)), rng.choice([1.0, 1.0, 2.0, 0.7]), dtype)
    del c["name"]
    return c


def work(case):
    c, e = case, _TYPES[case["dtype"]].itemsize
    if c["op"] == "rotary":
        values = c["B"] * c["S"] * (c["Hq"] + c["Hkv"]) * c["D"]
        ways = 2 if c["train"] else 1
        return {"bytes": 2 * ways * values * e + 8 * c["B"] * c["S"], "flops": 3 * ways * values}
    if c["op"] == "distillation":
        return {"bytes": 2 * c["T"] * c["V"] * e + c["T"] * (c["K"] * 12 + 4), "flops": 6 * c["T"] * c["V"]}
    B, Hq, Hkv, Sq, Sk, D = (c[k] for k in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
    pairs = keys = 0
    for n in _lengths(c):
        lo = [max(0, i + Sk - Sq + 1 - c["window"]) if c["window"] else 0 for i in range(Sq)]
        hi = [min(n, i + Sk - Sq + 1) if c["causal"] else n for i in range(Sq)]
        pairs += Hq * sum(max(0, h - a) for a, h in zip(lo, hi))
        keys += Hkv * max(0, max(hi) - min(lo))
    rows = B * Hq * Sq
    mask = 0 if c["mask"] == "none" else B * Sq * Sk * (4 if c["mask"] == "added" else 1)
    if not c["train"]:
        return {"bytes": (2 * rows * D + 2 * keys * D) * e + mask, "flops": 4 * pairs * D}
    return {"bytes": (4 * rows * D + 4 * keys * D) * e + mask, "flops": 14 * pairs * D}       # two products forward, five backward


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(c):
    """Number of keys of each batch entry: spread from an eighth to all of them, by the sizes alone."""
    if not c["lengths"]:
        return [c["Sk"]] * c["B"]
    return [max(1, c["Sk"] - (c["Sk"] * 7 * ((5 * b + 2) % c["B"])) // (8 * c["B"])) for b in range(c["B"])]


def _inverse_frequencies(c):
    """(turns in radians per position of each pair, factor on cos and sin), 64 bits, on the host."""
    R, f, base = c["R"], c["factor"], 10000.0
    if c["scaling"] == "ntk" and R > 2:
        base *= f ** (R / (R - 2))
    freq = [base ** (-2.0 * i / R) for i in range(R // 2)]
    if c["scaling"] == "linear":
        return [w / f for w in freq], 1.0
    if c["scaling"] == "yarn":
        # pairs that turn more than 32 times over the original 4096 positions keep their frequency, those that turn less than once are slowed by
        # the factor, a straight line over the pair's number in between
        def number(turns):
            return R * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(number(32.0)), 0), min(math.ceil(number(1.0)), R // 2 - 1)
        slow = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(R // 2)]
        return [w * (1 - s) + w / f * s for w, s in zip(freq, slow)], 0.1 * math.log(f) + 1.0
    return freq, 1.0


def prepare(case, seed):
    c, dt = case, _TYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dt)

    s = {"case": dict(c)}
    if c["op"] == "rotary":
        B, S, D = c["B"], c["S"], c["D"]
        # projections leave (batch, sequence, heads, size); the heads are viewed in front of the sequence
        s["q"], s["k"] = normal(B, S, c["Hq"], D).transpose(1, 2), normal(B, S, c["Hkv"], D).transpose(1, 2)
        first = torch.randint(0, c["far"] + 1, (B, 1), generator=g, device="cuda")
        s["positions"] = first + torch.arange(S, device="cuda")
        if c["train"]:
            s["q"].requires_grad_(), s["k"].requires_grad_()
            s["dq"], s["dk"] = normal(B, S, c["Hq"], D).transpose(1, 2), normal(B, S, c["Hkv"], D).transpose(1, 2)
        if own:
            from axs6_b200 import unified
            s["frequencies"] = unified.rotary_frequencies(c["R"], base=10000.0, scaling=c["scaling"], factor=c["factor"], original_length=4096, device="cuda")
        else:
            inv, s["gain"] = _inverse_frequencies(c)
            s["inverse"] = torch.tensor(inv, dtype=torch.float64, device="cuda")
    elif c["op"] == "attention":
        B, Hq, Hkv, Sq, Sk, D = (c[k] for k in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
        if Sq < Sk:                                   # a cache lies by heads
            s["q"], s["k"], s["v"] = normal(B, Sq, Hq, D).transpose(1, 2), normal(B, Hkv, Sk, D), normal(B, Hkv, Sk, D)
        else:                                         # projections leave (batch, sequence, heads, size)
            s["q"], s["k"], s["v"] = (normal(B, n, h, D).transpose(1, 2) for n, h in ((Sq, Hq), (Sk, Hkv), (Sk, Hkv)))
        s["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda") if c["lengths"] else None
        s["mask"] = None
        if c["mask"] != "none":
            kept = torch.rand((B, 1, Sq, Sk), generator=g, device="cuda") < 0.8
            kept[0, 0, 0] = False                     # a row without any key
            s["mask"] = kept if c["mask"] == "kept" else torch.where(kept, torch.randn((B, 1, Sq, Sk), generator=g, device="cuda"), -math.inf)
        if c["train"]:
            for n in ("q", "k", "v"):
                s[n].requires_grad_()
            s["do"] = normal(B, Sq, Hq, D).transpose(1, 2)
    else:
        T, V, K = c["T"], c["V"], c["K"]
        z = torch.randn((T, V), generator=g, device="cuda") * 2.5
        t = torch.randn((T, V), generator=g, device="cuda").mul_(1.5).add_(z)
        top, index = t.topk(K, dim=-1)
        s["teacher"], s["index"] = top.to(dt), index
        s["logits"] = z.to(dt).requires_grad_()
        # a tenth of the positions are padding: no slot of theirs is used
        s["index"][torch.rand((T,), generator=g, device="cuda") < 0.1] = -1
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"rotary": _rotary, "attention": _attention, "distillation": _distillation}[state["case"]["op"]](state)


def _rotary(s):
    c = s["case"]
    if own:
        from axs6_b200 import unified
        q, k = unified.axs_rotary_unified(s["q"], s["k"], s["positions"], s["frequencies"], layout=c["layout"])
        if not c["train"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    angle = s["positions"].double()[:, None, :, None] * s["inverse"]                        # (B, 1, S, R / 2)
    cos, sin = (angle.cos() * s["gain"]).float(), (angle.sin() * s["gain"]).float()
    out = {"q": _turned(s["q"].detach(), cos, sin, c), "k": _turned(s["k"].detach(), cos, sin, c)}
    if c["train"]:
        out |= {"dq": _turned(s["dq"], cos, -sin, c), "dk": _turned(s["dk"], cos, -sin, c)}
    return out


def _turned(x, cos, sin, c):
    R, y = c["R"], x.float().clone()
    a, b = (slice(0, R // 2), slice(R // 2, R)) if c["layout"] == "half" else (slice(0, R, 2), slice(1, R, 2))
    u, v = x[..., a].float(), x[..., b].float()
    y[..., a], y[..., b] = u * cos - v * sin, u * sin + v * cos
    return y.to(x.dtype)


def _attention(s):
    c = s["case"]
    if own:
        from axs6_b200 import unified
        o = unified.axs_attention_unified(s["q"], s["k"], s["v"], causal=c["causal"], window=c["window"] or None, key_lengths=s["lengths"], mask=s["mask"])
        if not c["train"]:
            return {"o": o}
        dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    B, Hq, Hkv, Sq, Sk, D = (c[k] for k in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
    G, dt, scale = Hq // Hkv, s["q"].dtype, 1.0 / math.sqrt(D)
    q = s["q"].detach().float().reshape(B, Hkv, G * Sq, D)
    k, v = s["k"].detach().float(), s["v"].detach().float()
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).view(B, Hkv, G, Sq, Sk)            # the scores
    i, j = torch.arange(Sq, device=p.device)[:, None] + (Sk - Sq), torch.arange(Sk, device=p.device)
    hidden = torch.zeros((B, 1, 1, Sq, Sk), dtype=torch.bool, device=p.device)
    if c["causal"]:
        hidden |= j > i
    if c["window"]:
        hidden |= j <= i - c["window"]
    if c["lengths"]:
        hidden |= j >= s["lengths"][:, None, None, None, None]
    if c["mask"] == "kept":
        hidden |= ~s["mask"][:, :, None]
    elif c["mask"] == "added":
        p += s["mask"][:, :, None]
    if c["causal"] or c["lengths"] or c["mask"] == "kept":
        p.masked_fill_(hidden, -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(total.masked_fill(total == 0, 1.0))                                               # a row without keys: all zeros
    p = p.view(B, Hkv, G * Sq, Sk)
    o = torch.matmul(p, v)
    out = {"o": o.view(B, Hq, Sq, D).to(dt)}
    if c["train"]:
        do = s["do"].float().reshape(B, Hkv, G * Sq, D)
        out["dv"] = torch.matmul(p.transpose(-1, -2), do).to(dt)
        ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out["dq"] = torch.matmul(ds, k).view(B, Hq, Sq, D).to(dt)
        out["dk"] = torch.matmul(ds.transpose(-1, -2), q).to(dt)
    return out


def _distillation(s):
    c, tau = s["case"], s["case"]["temperature"]
    if own:
        from axs6_b200 import unified
        loss = unified.axs_distillation_unified(s["logits"], s["teacher"], s["index"], temperature=tau, reduction="mean")
        grad, = torch.autograd.grad(loss, s["logits"])
        return {"loss": loss.detach(), "grad": grad}
    z = s["logits"].detach().float() / tau
    used = s["index"] >= 0
    t = (s["teacher"].float() / tau).masked_fill(~used, -math.inf)
    top = t.amax(-1, keepdim=True)
    e = (t - top.masked_fill(top == -math.inf, 0.0)).exp()
    total = e.sum(-1, keepdim=True)
    p = e / total.masked_fill(total == 0, 1.0)
    zt = z.amax(-1, keepdim=True)
    q = (z - zt).exp()
    zsum = q.sum(-1, keepdim=True)
    index = s["index"].clamp_min(0)
    log_q = z.gather(-1, index) - zt - zsum.log()
    rows = torch.where(used & (p > 0), p * (p.log() - log_q), 0.0).sum(-1) * (tau * tau)
    count = used.any(-1)
    n = count.sum().clamp_min(1)
    q.div_(zsum).mul_(count[:, None]).scatter_add_(-1, index, -p)
    return {"loss": rows.sum() / n, "grad": (q * (tau / n)).to(s["logits"].dtype)}


# ------------------------------------------------------------------------------------------------ 64 bits, from the definitions
def exact(case, seed):
    c, s = case, prepare(case, seed)
    s = {n: (v.detach() if torch.is_tensor(v) else v) for n, v in s.items()}
    if c["op"] == "rotary":
        inv, gain = _inverse_frequencies(c)
        theta = s["positions"].double()[..., None] * torch.tensor(inv, dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.full_like(theta, gain), theta)[:, None]                     # (B, 1, S, R / 2) complex
        out, R = {}, c["R"]
        for n in ("q", "k", "dq", "dk"):
            if n not in s:
                continue
            x = s[n].double()
            head = x[..., :R].unflatten(-1, (2, R // 2) if c["layout"] == "half" else (R // 2, 2))
            axis = -2 if c["layout"] == "half" else -1
            z = torch.complex(head.select(axis, 0).contiguous(), head.select(axis, 1).contiguous())
            z = z * (turn if n[0] != "d" else turn.conj())
            out[n] = torch.cat((torch.stack((z.real, z.imag), axis).flatten(-2), x[..., R:]), -1)
        return out
    if c["op"] == "distillation":
        tau, T = c["temperature"], c["T"]
        if T * c["V"] > 1 << 29:
            return None
        teacher, index = s["teacher"].double() / tau, s["index"]
        log_q = torch.log_softmax(s["logits"].double() / tau, -1)
        keep = (index[:, 0] >= 0)
        n = max(1, int(keep.sum()))
        p = torch.softmax(teacher, -1) * keep[:, None]
        full = torch.zeros_like(log_q).scatter_(-1, index.clamp_min(0), p)                   # the top logits' places differ from one another
        loss = (torch.special.xlogy(p, p).sum() - (full * log_q).sum()) * tau * tau / n
        return {"loss": loss, "grad": (log_q.exp_() * keep[:, None] - full) * (tau / n)}
    B, Hq, Hkv, Sq, Sk, D = (c[k] for k in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
    scale = D ** -0.5
    o = torch.zeros((B, Hq, Sq, D), dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(o), torch.zeros((B, Hkv, Sk, D), dtype=torch.float64, device="cuda"), torch.zeros((B, Hkv, Sk, D), dtype=torch.float64, device="cuda")
    row, col = torch.arange(Sq, device="cuda")[:, None], torch.arange(Sk, device="cuda")[None, :]
    for b, n in enumerate(_lengths(c)):
        see = (col < n).expand(Sq, Sk)
        if c["causal"]:
            see = see & (col - row <= Sk - Sq)
        if c["window"]:
            see = see & (col - row > Sk - Sq - c["window"])
        if c["mask"] == "kept":
            see = see & s["mask"][b, 0]
        for h in range(Hq):
            q, k, v = s["q"][b, h].double(), s["k"][b, h * Hkv // Hq].double(), s["v"][b, h * Hkv // Hq].double()
            x = scale * (q @ k.T)
            if c["mask"] == "added":
                x = x + s["mask"][b, 0].double()
            p = torch.softmax(torch.where(see, x, -math.inf), -1).nan_to_num_(0.0)           # 0 / 0 where a row sees nothing
            o[b, h] = p @ v
            if c["train"]:
                g = s["do"][b, h].double()
                dp = g @ v.T
                ds = scale * p * (dp - (dp * p).sum(-1, keepdim=True))
                dq[b, h] = ds @ k
                dk[b, h * Hkv // Hq] += ds.T @ q
                dv[b, h * Hkv // Hq] += p.T @ g
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if c["train"] else {"o": o}
