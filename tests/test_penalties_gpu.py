"""Penalties, biases and a grammar's mask on logits against the definition in 64 bits.

Bounds: the quotient or product, the penalties' product and each sum are one f32 rounding of what they are of, at most six u = 2^-24
of the sum of the terms' magnitudes, and the result rounds once to the dtype, h = eps / 2 of it."""
import numpy as np
import pytest
import torch

from dashmag_b200 import _lib
from dashmag_b200.penalties import Penalties, penalize
from dashmag_b200.sample import SampleOptions, sample

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def per_row(x, b):
    return np.asarray(x.cpu().double()) if isinstance(x, torch.Tensor) else np.full(b, float(np.float32(x)))


def definition(z, p: Penalties):
    """The rules in f64 and the magnitudes of what was added up."""
    z = z.double().cpu().numpy().copy()
    b, v = z.shape
    size = np.abs(np.where(np.isfinite(z), z, 0))
    rep, freq, pres = (per_row(x, b) for x in (p.repetition, p.frequency, p.presence))
    for r in range(b):
        if p.tokens is not None:
            ids = p.tokens[r].cpu().numpy().astype(np.int64)
            n = len(ids) if p.lengths is None else min(max(int(p.lengths[r]), 0), len(ids))
            m = 0 if p.prompt_lengths is None else min(max(int(p.prompt_lengths[r]), 0), n)
            there = np.zeros(v, bool)
            count = np.zeros(v)
            for i, t in enumerate(ids[:n]):
                if 0 <= t < v:
                    there[t] = True
                    count[t] += i >= m
            up = there & (z[r] > 0)
            down = there & ~(z[r] > 0)
            z[r, up] /= rep[r]
            z[r, down] *= rep[r]
            size[r] = np.maximum(size[r], np.abs(np.where(np.isfinite(z[r]), z[r], 0))) + np.abs(freq[r]) * count + np.abs(pres[r])
            z[r, count > 0] -= (freq[r] * count + pres[r])[count > 0]
        if p.bias is not None:
            bias = (p.bias if p.bias.dim() == 1 else p.bias[r]).double().cpu().numpy()
            z[r] += bias
            size[r] += np.abs(np.where(np.isfinite(bias), bias, 0))
        if p.allowed is not None:
            words = (p.allowed if p.allowed.dim() == 1 else p.allowed[r]).cpu().numpy().view(np.uint32)
            z[r, (words[np.arange(v) >> 5] >> (np.arange(v) & 31)) & 1 == 0] = -np.inf
    return z, size


def check(got, logits, p):
    want, size = definition(logits, p)
    g = got.double().cpu().numpy()
    h = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    assert got.shape == logits.shape and got.dtype == logits.dtype
    assert np.array_equal(np.isnan(g), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(g[inf], want[inf])
    fine = np.isfinite(want)
    with np.errstate(over="ignore"):
        off = np.abs(g[fine] - want[fine])
    assert np.all(off <= h * np.abs(want[fine]) + 6 * U * size[fine] + tiny), float(np.max(off))


def case(b, v, t, dtype, seed, bias="none", allowed=False, ids=torch.int32):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn((b, v), generator=g) * 3).to(TORCH[dtype]).to(DEV)
    tokens = (v ** torch.rand((b, t), generator=g)).to(ids) - 1
    lengths = torch.randint(0, t + 1, (b,), generator=g)
    kw = {}
    if bias != "none":
        kw["bias"] = torch.randn((v,) if bias == "one" else (b, v), generator=g).to(DEV)
    if allowed:
        kw["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (b, (v + 31) // 32), generator=g).to(torch.int32).to(DEV)
    p = Penalties(tokens=tokens.to(DEV), lengths=lengths.to(ids).to(DEV), prompt_lengths=(lengths // 2).to(torch.int32).to(DEV),
                  repetition=(1 + torch.rand(b, generator=g)).to(DEV), frequency=torch.rand(b, generator=g).to(DEV), presence=torch.rand(b, generator=g).to(DEV), **kw)
    return logits, p


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("b,v,t", [(1, 1, 1), (3, 7, 5), (2, 8, 0), (5, 1000, 300), (4, 4099, 64), (1, 32768, 200), (33, 2048, 17), (3, 50001, 3000), (70, 20011, 500)])
@pytest.mark.parametrize("bias,allowed", [("none", False), ("one", True), ("rows", True)])
def test_against_the_definition(b, v, t, dtype, bias, allowed):
    logits, p = case(b, v, t, dtype, b * 7 + v, bias, allowed, torch.int64 if t % 2 else torch.int32)
    check(penalize(logits, p), logits, p)


@pytest.mark.parametrize("dtype", list(TORCH))
def test_numbers_and_parts_of_the_rules(dtype):
    logits, p = case(4, 3001, 100, dtype, 3, "one", True)
    for q in (Penalties(), Penalties(tokens=p.tokens), Penalties(tokens=p.tokens, repetition=1.3), Penalties(tokens=p.tokens, frequency=0.5, lengths=p.lengths),
              Penalties(tokens=p.tokens, presence=-0.7, prompt_lengths=p.prompt_lengths), Penalties(bias=p.bias), Penalties(bias=p.bias.to(TORCH[dtype])),
              Penalties(allowed=p.allowed), Penalties(allowed=p.allowed[1]), Penalties(tokens=p.tokens, repetition=0.5, frequency=-1.0)):
        check(penalize(logits, q), logits, q)
    assert torch.equal(penalize(logits, Penalties()), logits)


@pytest.mark.parametrize("dtype", list(TORCH))
def test_addresses_strides_and_in_place(dtype):
    """Rows at any address and stride, the result beside them or over them; nothing is written between the rows."""
    t = TORCH[dtype]
    b, v = 5, 1003
    _, p = case(b, v, 60, dtype, 5, "rows", True)
    for shift in range(0, 9):
        for pitch in (v, v + 1, v + 5, 1024):
            flat = torch.randn(b * pitch + 16, device=DEV).to(t)
            logits = torch.as_strided(flat, (b, v), (pitch, 1), shift)
            keep = flat.clone()
            check(penalize(logits, p), logits, p)
            assert torch.equal(flat, keep)
            out = torch.full((b * 1100 + 16,), 7.0, device=DEV, dtype=t)
            view = torch.as_strided(out, (b, v), (1100, 1), (shift * 3) % 8)
            want = penalize(logits, p)
            assert penalize(logits, p, out=view) is view and torch.equal(view, want)
            view.fill_(7.0)
            assert bool((out == 7.0).all())
            penalize(logits, p, out=logits)
            assert torch.equal(logits, want)
            logits.copy_(torch.as_strided(keep, (b, v), (pitch, 1), shift))
            assert torch.equal(flat, keep)
    logits = torch.randn((v, b), device=DEV).to(t).T   # a vocabulary that is not contiguous
    q = Penalties(tokens=p.tokens.T.contiguous().T, bias=p.bias.T.contiguous().T, allowed=p.allowed.T.contiguous().T, repetition=1.5,
                  lengths=torch.stack([p.lengths, p.lengths], 1)[:, 0])
    check(penalize(logits, q), logits, q)


def test_ids_outside_the_vocabulary_and_lengths_out_of_range():
    logits = torch.randn((3, 100), device=DEV)
    tokens = torch.tensor([[-1, 100, 2 ** 31 - 1, 5, 5], [5, -2 ** 31, 99, 0, 0], [1, 2, 3, 4, 5]], device=DEV, dtype=torch.int32)
    for lengths, prompt in (([5, 5, 5], [0, 0, 0]), ([-3, 99, 2], [9, -9, 5])):
        p = Penalties(tokens=tokens, lengths=torch.tensor(lengths, device=DEV), prompt_lengths=torch.tensor(prompt, device=DEV), repetition=2.0, frequency=1.0, presence=0.5)
        check(penalize(logits, p), logits, p)
    far = Penalties(tokens=torch.tensor([[2 ** 40 + 5, -2 ** 40, 2 ** 32, 7]] * 3, device=DEV), repetition=2.0)
    check(penalize(logits, far), logits, far)


def test_infinities_and_nan():
    logits = torch.randn((2, 64), device=DEV)
    logits[0, :6] = torch.tensor([float("inf"), -float("inf"), float("nan"), 0.0, -0.0, 1e38])
    logits[1] = float("nan")
    tokens = torch.arange(6, device=DEV).expand(2, 6)
    p = Penalties(tokens=tokens, repetition=2.0, frequency=1.0)
    check(penalize(logits, p), logits, p)
    shut = Penalties(tokens=tokens, repetition=2.0, allowed=torch.zeros((2, 2), dtype=torch.int32, device=DEV))
    assert bool((penalize(logits, shut) == -float("inf")).all())   # a row that is allowed nothing
    bias = torch.zeros(64, device=DEV)
    bias[10] = -float("inf")
    assert float(penalize(logits, Penalties(bias=bias))[0, 10]) == -float("inf")


def test_many_of_one_token():
    """A token that is there more often than a short integer holds."""
    logits = torch.zeros((1, 50), device=DEV)
    p = Penalties(tokens=torch.full((1, 70000), 7, dtype=torch.int32, device=DEV), frequency=0.5)
    assert float(penalize(logits, p)[0, 7]) == -35000.0


@pytest.mark.parametrize("dtype", list(TORCH))
def test_the_sampler_takes_them(dtype):
    logits, p = case(6, 5003, 80, dtype, 9, "one", True)
    options = SampleOptions(temperature=0.8, top_k=40, top_p=0.9, seed=3, offset=2)
    got, want = sample(logits, options, penalties=p), sample(penalize(logits, p), options)
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.logprob, want.logprob)
    words = p.allowed.cpu().numpy().view(np.uint32)
    for r, t in enumerate(got.tokens.tolist()):
        assert words[r, t >> 5] >> (t & 31) & 1
    one = torch.zeros((6, (5003 + 31) // 32), dtype=torch.int32, device=DEV)
    one[:, 100] = 1 << 9
    assert sample(logits, options, penalties=Penalties(allowed=one)).tokens.tolist() == [3209] * 6


def test_one_launch_captured_and_replayed():
    logits, p = case(3, 3001, 100, "bf16", 4, "one", True)
    before = _lib.probe("kernel_launches")
    penalize(logits, p)
    assert _lib.probe("kernel_launches") == before + 1
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = penalize(logits, p)
    for step in range(3):
        p.lengths.copy_(torch.tensor([10 + step, 0, 100], device=DEV))
        logits.normal_()
        graph.replay()
        check(out, logits, p)


def test_nothing_to_do():
    before = _lib.probe("kernel_launches")
    assert penalize(torch.zeros((0, 10), device=DEV), Penalties()).shape == (0, 10)
    assert penalize(torch.zeros((4, 0), device=DEV), Penalties()).shape == (4, 0)
    assert _lib.probe("kernel_launches") == before


@pytest.mark.parametrize("dtype", list(TORCH))
def test_out_in_other_columns_of_the_logits_tensor(dtype):
    """Logits and result are columns of one larger tensor, side by side, without a token in common."""
    b, v = 4, 333
    logits, p = case(b, v, 50, dtype, 11, "rows", True)
    both = torch.zeros((b, 2 * v + 3), device=DEV, dtype=TORCH[dtype])
    for left in (True, False):
        both.zero_()
        source, out = (both[:, :v], both[:, v + 3:]) if left else (both[:, v + 3:], both[:, :v])
        source.copy_(logits)
        penalize(source, p, out=out)
        assert torch.equal(out, penalize(logits, p)) and torch.equal(source, logits) and not bool(both[:, v:v + 3].any())
