"""The operators around a served or trained attention layer, as cases that can be prepared, run and compared.

Three kinds of call: the norm of every query and key head with the position rotation in the same pass (a prompt's or a
training batch's tokens, its gradient, one token of each sequence), the decoding step of a batch whose sequences share
prompts (every prompt's keys read once for all of its sequences, then each sequence's own cache, with or without the new
row written first), and the rules a server puts on a step's logits (penalties for tokens that were there, biases, a
grammar's mask).  ``own`` chooses between the plain form - elementary tensor operations in 32 bits, rounded once - and the
framework's calls.  ``exact`` gives the same from the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


def listed():
    return [
        # One token of each of eight sequences: the step of a decoder with norms on its heads, where latency counts.
        dict(name="norm_step", kind="norm", grad=False, dtype="bf16", wdtype="bf16", form="at", b=8, t=1, total=8, hq=32, hkv=8, d=128, dim=128, fused=False, lens_seed=0),
        # A packed training batch of eight sequences, query and key as slices of one projection's output.
        dict(name="norm_packed", kind="norm", grad=False, dtype="bf16", wdtype="bf16", form="packed", b=8, t=4096, total=16384, hq=32, hkv=8, d=128, dim=128, fused=True,
             lens_seed=0),
        # Its gradient, to the weights too, which the optimizer holds in f32.
        dict(name="norm_packed_grad", kind="norm", grad=True, dtype="bf16", wdtype="f32", form="packed", b=8, t=4096, total=16384, hq=32, hkv=8, d=128, dim=128, fused=True,
             lens_seed=0),
        # A small f32 batch of odd sizes, a part of each head rotated, gradients: a test's or a toy model's.
        dict(name="norm_grad_f32", kind="norm", grad=True, dtype="f32", wdtype="f32", form="range", b=3, t=701, total=2103, hq=12, hkv=4, d=96, dim=48, fused=False, lens_seed=0),
        # Four answers to one short question, a few tokens in.
        dict(name="shared_few", kind="shared", dtype="bf16", n=1, each=4, p=1000, plo=1000, s=64, lo=1, hq=16, hkv=4, d=128, window=-1, append=True, lens_seed=2),
        # A full batch behind one long instruction: 64 sequences, 8192 shared tokens, up to 1024 of each sequence's own.
        dict(name="shared_batch", kind="shared", dtype="bf16", n=1, each=64, p=8192, plo=8192, s=1024, lo=1, hq=32, hkv=8, d=128, window=-1, append=False, lens_seed=3),
        # Sampling for training: 32 prompts of different lengths, sixteen answers to each, heads of 64, f16.
        dict(name="shared_samples", kind="shared", dtype="f16", n=32, each=16, p=2048, plo=100, s=512, lo=1, hq=16, hkv=4, d=64, window=-1, append=False, lens_seed=4),
        # Odd sizes in f32, two prompts, a head dimension that no tile divides.
        dict(name="shared_f32", kind="shared", dtype="f32", n=2, each=3, p=777, plo=300, s=33, lo=0, hq=6, hkv=2, d=80, window=-1, append=True, lens_seed=5),
        # One user's logits in f32, a short history.
        dict(name="rules_single", kind="rules", dtype="f32", b=1, v=32768, t=200, bias="none", allowed=False, lens_seed=6),
        # A serving batch with everything: ragged histories, one bias for all, half of the rows under a grammar.
        dict(name="rules_batch", kind="rules", dtype="bf16", b=64, v=151936, t=2048, bias="one", allowed=True, lens_seed=7),
        # A large batch of long histories, a vocabulary that fills no vector.
        dict(name="rules_long", kind="rules", dtype="bf16", b=256, v=100003, t=8192, bias="none", allowed=False, lens_seed=8),
        # Half precision, a bias for each row.
        dict(name="rules_rows", kind="rules", dtype="f16", b=32, v=65536, t=500, bias="rows", allowed=True, lens_seed=9),
    ]


# ------------------------------------------------------------------------------------------------
# More cases of the same ranges
# ------------------------------------------------------------------------------------------------
def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    family = rng.randrange(7)
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    lens_seed = rng.randrange(1000)
    if family < 3:
        d = rng.choice([128, 128, 64, 256, 96, 80])
        dim = rng.choice([d, d, d // 2])
        hq, hkv = rng.choice([(32, 8), (16, 4), (16, 16), (12, 4), (8, 1), (6, 3)])
        form = ("at", "packed", "range")[family]
        grad = form != "at" and rng.random() < 0.6
        if form == "at":
            b, t = _log(rng, 1, 512), 1
            total = b
        elif form == "packed":
            total = _log(rng, 40, 16384 * 40 * 128 // ((hq + hkv) * d) // (2 if dtype == "f32" else 1))
            b = rng.randint(1, max(1, min(12, total // 20)))
            t = total
        else:
            b, t = rng.randint(1, 8), _log(rng, 5, 1500)
            total = b * t
        return dict(kind="norm", grad=grad, dtype=dtype, wdtype=rng.choice([dtype, "f32"]), form=form, b=b, t=t, total=total, hq=hq, hkv=hkv, d=d, dim=dim,
                    fused=rng.random() < 0.5, lens_seed=lens_seed)
    if family < 5:
        d = rng.choice([128, 128, 64, 256, 80]) if dtype != "f32" else rng.choice([64, 80, 128])
        hq, hkv = rng.choice([(32, 8), (16, 4), (8, 8), (8, 1), (6, 2), (24, 4)])
        n = rng.choice([1, 1, 1, 2, 5, 16])
        each = _log(rng, 1, max(1, 128 // n))
        most = min(16384, 8192 * 64 * 32 * 128 // (each * n * hq * d))
        p = _log(rng, 17, max(18, most // (8 if dtype == "f32" else 1)))
        s = _log(rng, 1, 1024 if dtype != "f32" else 200)
        return dict(kind="shared", dtype=dtype, n=n, each=each, p=p, plo=rng.choice([p, p, 0, p // 2]), s=s, lo=rng.choice([0, min(1, s - 1)]), hq=hq, hkv=hkv, d=d,
                    window=rng.choice([-1, -1, -1, p // 2 + 10]), append=rng.random() < 0.5, lens_seed=lens_seed)
    v = _log(rng, 1000, 200000)
    return dict(kind="rules", dtype=dtype, b=_log(rng, 1, 256), v=v, t=_log(rng, 1, 8192), bias=rng.choice(["none", "one", "rows"]) if v < 100000 else "none",
                allowed=rng.random() < 0.5, lens_seed=lens_seed)


# ------------------------------------------------------------------------------------------------
# Sizes
# ------------------------------------------------------------------------------------------------
def _offsets(c):
    """Offsets of the packed sequences: shares of the total, none empty where there is room."""
    raw = np.random.default_rng(c["lens_seed"]).integers(max(1, c["t"] // 8), c["t"] + 1, size=c["b"]).astype(np.float64)
    lens = np.floor(raw * c["total"] / raw.sum()).astype(np.int64)
    lens[: c["total"] - lens.sum()] += 1
    return np.concatenate([[0], np.cumsum(lens)])


def _lengths(c, salt, lo, hi, count):
    """Integers uniform in [lo, hi], made from the case alone."""
    return np.random.default_rng([c["lens_seed"], salt]).integers(lo, max(lo, hi) + 1, size=count)


def _shared_lengths(c):
    """The prompts' lengths, and what each sequence holds of its own (before the step's row)."""
    return _lengths(c, 1, c["plo"], c["p"], c["n"]), _lengths(c, 2, c["lo"], c["s"] - (1 if c["append"] else 0), c["n"] * c["each"])


def _positions_held(c):
    return int(np.max(np.diff(_offsets(c)))) if c["form"] == "packed" else 4096 if c["form"] == "at" else c["t"] + 37


def work(case):
    c, e = case, BYTES[case["dtype"]]
    if c["kind"] == "norm":
        rows = c["total"] * (c["hq"] + c["hkv"])
        at_once = c["total"] if c["form"] == "at" else min(c["total"], _positions_held(c))
        tables, weights = 2 * at_once * c["dim"] * e, 2 * c["d"] * BYTES[c["wdtype"]]
        if c["grad"]:   # in: x and its gradient; out: the inputs' gradient
            return {"bytes": 3 * rows * c["d"] * e + tables + 2 * weights, "flops": rows * (13 * c["d"] + 3 * c["dim"])}
        return {"bytes": 2 * rows * c["d"] * e + tables + weights, "flops": rows * (4 * c["d"] + 3 * c["dim"])}
    if c["kind"] == "shared":
        plens, lens = _shared_lengths(c)
        own_keys = np.minimum(lens + (1 if c["append"] else 0), c["s"])
        w = c["window"]
        in_prefix = np.repeat(plens, c["each"])
        if w >= 0:   # the window reaches over the end of the sequence's own keys
            in_prefix = np.minimum(in_prefix, np.maximum(0, w + 1 - own_keys))
            own_keys = np.minimum(own_keys, w + 1)
        shared = in_prefix.reshape(c["n"], c["each"]).max(axis=1)
        rows = c["n"] * c["each"] * c["d"] * e * (2 * c["hq"] + (2 * c["hkv"] if c["append"] else 0))
        return {"bytes": int(shared.sum() + own_keys.sum()) * c["hkv"] * c["d"] * e * 2 + rows, "flops": 4 * c["d"] * c["hq"] * int(in_prefix.sum() + own_keys.sum())}
    words = c["b"] * ((c["v"] + 31) // 32) if c["allowed"] else 0
    bias = {"none": 0, "one": c["v"], "rows": c["b"] * c["v"]}[c["bias"]]
    return {"bytes": 2 * c["b"] * c["v"] * e + 4 * int(_history(c)[0].sum()) + 4 * words + 4 * bias, "flops": 6 * c["b"] * c["v"]}


def _history(c):
    """How many ids each row's history holds, and how many of them are the prompt's."""
    held = _lengths(c, 3, 0 if c["b"] > 1 else c["t"], c["t"], c["b"])
    return held, held * 2 // 3


# ------------------------------------------------------------------------------------------------
# What a program has in hand
# ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[c["dtype"]]

    def randn(*shape, like=dtype):
        return torch.randn(shape, generator=g, device="cuda", dtype=like)

    def ints(values, kind=torch.int32):
        return torch.tensor(np.asarray(values), dtype=kind, device="cuda")

    s = {"case": c}
    if c["kind"] == "norm":
        lead = (c["b"], c["t"]) if c["form"] == "range" else (c["total"],)
        hq, hkv, d = c["hq"], c["hkv"], c["d"]
        if c["fused"]:
            s["qkv"] = randn(*lead, (hq + 2 * hkv) * d)
        else:
            s.update(q=randn(*lead, hq, d), k=randn(*lead, hkv, d))
        if c["grad"]:
            s.update(gq=randn(*lead, hq, d), gk=randn(*lead, hkv, d))
        s.update(wq=(1 + 0.3 * randn(d, like=torch.float32)).to(DTYPES[c["wdtype"]]), wk=(1 + 0.3 * randn(d, like=torch.float32)).to(DTYPES[c["wdtype"]]))
        held = _positions_held(c)
        angle = torch.arange(held, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * (torch.arange(c["dim"], device="cuda", dtype=torch.float64) % (c["dim"] // 2)) / c["dim"])
        s.update(cos=angle.cos().to(dtype), sin=angle.sin().to(dtype))
        if c["form"] == "packed":
            s["cu"] = ints(_offsets(c))
        elif c["form"] == "at":
            s["positions"] = torch.randint(0, held, (c["b"],), generator=g, device="cuda", dtype=torch.int32)
        else:
            s["start"] = 37
    elif c["kind"] == "shared":
        b, hkv, d = c["n"] * c["each"], c["hkv"], c["d"]
        plens, lens = _shared_lengths(c)
        s.update(q=randn(b, c["hq"], d), pk=randn(c["n"], c["p"], hkv, d), pv=randn(c["n"], c["p"], hkv, d), k=randn(b, c["s"], hkv, d), v=randn(b, c["s"], hkv, d),
                 plens=None if c["plo"] == c["p"] else ints(plens), lens=ints(lens), window=c["window"])
        if c["append"]:
            s.update(k_new=randn(b, hkv, d), v_new=randn(b, hkv, d))
    else:
        b, v, t = c["b"], c["v"], c["t"]
        held, prompt = _history(c)
        # Ids as text has them: a few tokens make up most of it.
        ids = (v ** torch.rand((b, t), generator=g, device="cuda")).to(torch.int32).clamp_(0, v - 1)
        s.update(logits=(3 * randn(b, v, like=torch.float32)).to(dtype), ids=ids, held=ints(held), prompt=ints(prompt),
                 repetition=1 + 0.5 * torch.rand(b, generator=g, device="cuda"), frequency=0.3 * torch.rand(b, generator=g, device="cuda"),
                 presence=0.6 * torch.rand(b, generator=g, device="cuda"))
        s["bias"] = None if c["bias"] == "none" else randn(*((v,) if c["bias"] == "one" else (b, v)), like=torch.float32)
        if c["allowed"]:
            words = torch.randint(-2 ** 31, 2 ** 31, (2, b, (v + 31) // 32), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
            words = words[0] & words[1]
            words[1::2] = -1   # every other row is free
            s["allowed"] = words
    return s


# ------------------------------------------------------------------------------------------------
# The pass
# ------------------------------------------------------------------------------------------------
def run(state):
    return {"norm": _norm, "shared": _shared, "rules": _rules}[state["case"]["kind"]](state)


def _heads(s):
    """The queries' and the keys' heads: views of one projection's output, or tensors of their own."""
    c = s["case"]
    if "qkv" not in s:
        return s["q"], s["k"]
    x, n, m = s["qkv"], c["hq"] * c["d"], (c["hq"] + c["hkv"]) * c["d"]
    return x[..., :n].unflatten(-1, (c["hq"], c["d"])), x[..., n:m].unflatten(-1, (c["hkv"], c["d"]))


def _norm(s):
    c = s["case"]
    q, k = _heads(s)
    if own:
        from dashmag_b200.qk_norm import QkNorm
        from dashmag_b200.rope import Rope
        norm = QkNorm(Rope.from_tables(s["cos"], s["sin"]), s["wq"], s["wk"], EPS)
        if not c["grad"]:
            if c["form"] == "packed":
                return norm.apply_packed(q, k, s["cu"])
            return norm.apply_at(q, k, s["positions"]) if c["form"] == "at" else norm.apply_range(q, k, range(s["start"], s["start"] + c["t"]))
        if c["form"] == "packed":
            return norm.backward_packed(q, k, s["gq"], s["gk"], s["cu"])
        return norm.backward_range(q, k, s["gq"], s["gk"], range(s["start"], s["start"] + c["t"]))
    cos, sin = (x.float()[..., None, :] for x in (s["cos"][_rows_of(s)], s["sin"][_rows_of(s)]))
    if not c["grad"]:
        return _turned(_normed(q.float(), s["wq"].float()), cos, sin).to(q.dtype), _turned(_normed(k.float(), s["wk"].float()), cos, sin).to(q.dtype)
    dq, dwq = _norm_gradient(q.float(), s["wq"].float(), _turned_back(s["gq"].float(), cos, sin))
    dk, dwk = _norm_gradient(k.float(), s["wk"].float(), _turned_back(s["gk"].float(), cos, sin))
    return dq.to(q.dtype), dk.to(q.dtype), dwq.to(s["wq"].dtype), dwk.to(s["wq"].dtype)


def _rows_of(s):
    """The table row of every token."""
    c = s["case"]
    if c["form"] == "at":
        return s["positions"].long()
    if c["form"] == "range":
        return torch.arange(s["start"], s["start"] + c["t"], device="cuda").expand(c["b"], c["t"])
    n, cu = torch.arange(c["total"], device="cuda"), s["cu"].long()
    return n - cu[torch.searchsorted(cu, n, right=True) - 1]


def _normed(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _turned(x, cos, sin):
    dim = cos.shape[-1]
    h, rest = x[..., :dim], x[..., dim:]
    return torch.cat([h * cos + torch.cat([-h[..., dim // 2:], h[..., : dim // 2]], -1) * sin, rest], -1)


def _turned_back(g, cos, sin):
    dim = cos.shape[-1]
    h, rest = g[..., :dim], g[..., dim:]
    z = h * sin
    return torch.cat([h * cos + torch.cat([z[..., dim // 2:], -z[..., : dim // 2]], -1), rest], -1)


def _norm_gradient(x, w, g):
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    n, gw = x * r, g * w
    return r * (gw - n * (n * gw).mean(-1, keepdim=True)), (g * n).sum(tuple(range(x.dim() - 1)))


def _shared(s):
    c = s["case"]
    if own:
        from dashmag_b200.contract import AttentionOptions
        from dashmag_b200.prefix import attention_decode_shared, attention_decode_shared_append
        options = AttentionOptions().with_window(s["window"], 0) if s["window"] >= 0 else AttentionOptions()
        if c["append"]:
            out = attention_decode_shared_append(s["q"], s["k_new"], s["v_new"], s["pk"], s["pv"], s["k"], s["v"], s["lens"], s["plens"], options)
            return {"out": out, "k": s["k"], "v": s["v"]}
        return attention_decode_shared(s["q"], s["pk"], s["pv"], s["k"], s["v"], s["lens"], s["plens"], options)
    b, hq, d = s["q"].shape
    n, p, hkv, _ = s["pk"].shape
    each, group, size = b // n, hq // hkv, s["k"].shape[1]
    lens = s["lens"].long()
    if c["append"]:
        rows = torch.arange(b, device="cuda")
        s["k"][rows, lens] = s["k_new"]
        s["v"][rows, lens] = s["v_new"]
        lens = lens + 1
    plens = torch.full((n,), p, device="cuda") if s["plens"] is None else s["plens"].long()
    first = (plens.repeat_interleave(each) + lens - 1 - s["window"]) if s["window"] >= 0 else torch.zeros_like(lens)
    q = s["q"].float() / math.sqrt(d)
    at_prefix, at_own = torch.arange(p, device="cuda"), torch.arange(size, device="cuda")
    scores = torch.einsum("nihgd,nphd->nihgp", q.view(n, each, hkv, group, d), s["pk"].float()).reshape(b, hkv, group, p)
    seen = (at_prefix < plens.repeat_interleave(each)[:, None]) & (at_prefix >= first[:, None])
    scores = scores.masked_fill(~seen[:, None, None, :], -math.inf)
    tail = torch.einsum("bhgd,bshd->bhgs", q.view(b, hkv, group, d), s["k"].float())
    seen = (at_own < lens[:, None]) & (at_own + plens.repeat_interleave(each)[:, None] >= first[:, None])
    tail = tail.masked_fill(~seen[:, None, None, :], -math.inf)
    top = torch.maximum(scores.amax(-1, keepdim=True), tail.amax(-1, keepdim=True))
    top = top.masked_fill(top == -math.inf, 0.0)
    scores, tail = (scores - top).exp(), (tail - top).exp()
    total = scores.sum(-1, keepdim=True) + tail.sum(-1, keepdim=True)
    out = torch.einsum("nihgp,nphd->nihgd", scores.reshape(n, each, hkv, group, p), s["pv"].float()).reshape(b, hkv, group, d) + torch.einsum("bhgs,bshd->bhgd", tail, s["v"].float())
    out = (out / total.masked_fill(total == 0, 1.0)).reshape(b, hq, d).to(s["q"].dtype)
    return {"out": out, "k": s["k"], "v": s["v"]} if c["append"] else out


def _rules(s):
    if own:
        from dashmag_b200.penalties import Penalties, penalize
        return penalize(s["logits"], Penalties(tokens=s["ids"], lengths=s["held"], prompt_lengths=s["prompt"], repetition=s["repetition"], frequency=s["frequency"],
                                               presence=s["presence"], bias=s["bias"], allowed=s.get("allowed")))
    b, v = s["logits"].shape
    at = torch.arange(s["ids"].shape[1], device="cuda")
    there = (at < s["held"][:, None]).int()
    answered = there * (at >= s["prompt"][:, None]).int()
    ids = s["ids"].long()
    seen = torch.zeros((b, v), dtype=torch.int32, device="cuda").scatter_add_(1, ids, there)
    count = torch.zeros((b, v), dtype=torch.int32, device="cuda").scatter_add_(1, ids, answered)
    z, r = s["logits"].float(), s["repetition"][:, None]
    z = torch.where(seen > 0, torch.where(z > 0, z / r, z * r), z)
    z = z - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        z = z + s["bias"]
    if "allowed" in s:
        token = torch.arange(v, device="cuda")
        z = z.masked_fill((s["allowed"][:, token >> 5] >> (token & 31) & 1) == 0, -math.inf)
    return z.to(s["logits"].dtype)


# ------------------------------------------------------------------------------------------------
# The same from the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] == "norm":
        return _exact_norm(s, c)
    return _exact_shared(s, c) if c["kind"] == "shared" else _exact_rules(s, c)


def _exact_norm(s, c):
    """Pair by pair: features j and j + dim / 2 of a head are one complex number, turned by the table's angle."""
    if c["form"] == "packed":
        starts = _offsets(c)
        pos = torch.cat([torch.arange(int(n), device="cuda") for n in np.diff(starts)])
    elif c["form"] == "at":
        pos = s["positions"].long()
    else:
        pos = (s["start"] + torch.arange(c["t"], device="cuda")).repeat(c["b"])
    half = c["dim"] // 2
    cos, sin = s["cos"].double()[pos][:, None, :], s["sin"].double()[pos][:, None, :]
    c1, c2, s1, s2 = cos[..., :half], cos[..., half:], sin[..., :half], sin[..., half:]
    out = []
    for name, heads, at in (("q", c["hq"], 0), ("k", c["hkv"], c["hq"] * c["d"])):
        if c["fused"]:
            x = s["qkv"].reshape(c["total"], -1)[:, at: at + heads * c["d"]].reshape(c["total"], heads, c["d"]).double()
        else:
            x = s[name].reshape(c["total"], heads, c["d"]).double()
        w = s["w" + name].double()
        size = torch.sqrt(torch.sum(x * x, dim=2, keepdim=True) / c["d"] + EPS)
        unit = x / size
        if not c["grad"]:
            y = unit * w
            lo, hi = y[..., :half].clone(), y[..., half: c["dim"]].clone()
            y[..., :half] = lo * c1 - hi * s1
            y[..., half: c["dim"]] = hi * c2 + lo * s2
            out.append(y.reshape(*_lead(c), heads, c["d"]))
            continue
        g = s["g" + name].reshape(c["total"], heads, c["d"]).double().clone()
        lo, hi = g[..., :half].clone(), g[..., half: c["dim"]].clone()
        g[..., :half] = lo * c1 + hi * s2
        g[..., half: c["dim"]] = hi * c2 - lo * s1
        dw = torch.einsum("thd,thd->d", g, unit)
        g *= w
        along = torch.sum(g * unit, dim=2, keepdim=True) / c["d"]
        out.append(((g - unit * along) / size).reshape(*_lead(c), heads, c["d"]))
        out.append(dw)
    return (out[0], out[1]) if not c["grad"] else (out[0], out[2], out[1], out[3])


def _lead(c):
    return (c["b"], c["t"]) if c["form"] == "range" else (c["total"],)


def _exact_shared(s, c):
    """Sequence by sequence: the prompt's keys and its own behind them, one softmax."""
    plens, lens = _shared_lengths(c)
    group = c["hq"] // c["hkv"]
    if c["append"]:
        for b, n in enumerate(lens):
            s["k"][b, int(n)], s["v"][b, int(n)] = s["k_new"][b], s["v_new"][b]
    out = torch.zeros((len(lens), c["hq"], c["d"]), dtype=torch.float64, device="cuda")
    for b in range(len(lens)):
        n, have = int(plens[b // c["each"]]), int(lens[b]) + (1 if c["append"] else 0)
        keys = torch.cat([s["pk"][b // c["each"], :n], s["k"][b, :have]]).double()
        values = torch.cat([s["pv"][b // c["each"], :n], s["v"][b, :have]]).double()
        if c["window"] >= 0:
            keys, values = keys[max(0, n + have - 1 - c["window"]):], values[max(0, n + have - 1 - c["window"]):]
        if len(keys) == 0:
            continue
        x = s["q"][b].double().reshape(c["hkv"], group, c["d"]) @ keys.permute(1, 2, 0) * c["d"] ** -0.5
        out[b] = (torch.softmax(x, dim=2) @ values.transpose(0, 1)).reshape(c["hq"], c["d"])
    return {"out": out, "k": None, "v": None} if c["append"] else out


def _exact_rules(s, c):
    """Row by row, a histogram of the ids of each."""
    held, prompt = _history(c)
    out = s["logits"].double()
    for b in range(c["b"]):
        z, ids = out[b], s["ids"][b, : int(held[b])].long()
        there = torch.bincount(ids, minlength=c["v"]) > 0
        count = torch.bincount(ids[int(prompt[b]):], minlength=c["v"]).double()
        r = float(s["repetition"][b])
        z[there & (z > 0)] /= r
        z[there & (s["logits"][b].double() <= 0)] *= r
        z -= float(s["frequency"][b]) * count
        z[count > 0] -= float(s["presence"][b])
        if s["bias"] is not None:
            z += (s["bias"] if c["bias"] == "one" else s["bias"][b]).double()
        if c["allowed"]:
            bits = np.unpackbits(s["allowed"][b].cpu().numpy().view(np.uint8), bitorder="little")[: c["v"]]
            z[torch.from_numpy(bits == 0).cuda()] = -math.inf
    return out
