"""Infinities and NaN in features that are not rotated: they reach what the formula says they reach, whichever kernel takes the call.

A feature behind the rotated ones is no partner of another: an infinite one makes the head's mean infinite, every other feature of the head 0 and
itself NaN, and a gradient that is not finite there spoils its head's gradient, but of the weights' gradients that feature's alone.
Bounds as for finite inputs: u = 2^-24, h = eps / 2; 32 u forward, 64 u backward and 300 u for a weight's gradient, of the sum of the terms'
magnitudes, and h of the result."""
import pytest
import torch

from dashmag_b200.qk_norm import QkNorm
from dashmag_b200.rope import Rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24
INF, NAN = float("inf"), float("nan")


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype).to(DEV)


def rope_of(dim, held, dtype):
    angle = torch.arange(held, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * (torch.arange(dim, dtype=torch.float64) % (dim // 2)) / dim)
    return Rope.from_tables(angle.cos().to(dtype).to(DEV), angle.sin().to(dtype).to(DEV))


def turn(x, rope, back=False):
    """x [T, H, D] at the positions 0 .. T - 1; and the sum of the terms' magnitudes."""
    half, dim = rope.dim // 2, rope.dim
    cos, sin = (t.double()[: x.shape[0], None, :] for t in (rope.cos, rope.sin))
    lo, hi = x[..., :half], x[..., half: dim]
    sign = -1.0 if back else 1.0
    s_lo, s_hi = (sin[..., half:], sin[..., :half]) if back else (sin[..., :half], sin[..., half:])
    y, size = x.clone(), x.abs()
    y[..., :half], y[..., half: dim] = lo * cos[..., :half] - sign * hi * s_lo, hi * cos[..., half:] + sign * lo * s_hi
    size[..., :half], size[..., half: dim] = (lo * cos[..., :half]).abs() + (hi * s_lo).abs(), (hi * cos[..., half:]).abs() + (lo * s_hi).abs()
    return y, size


def same(got, want, tol):
    """Finite where the formula is, to the tolerance; infinite and NaN where it is."""
    got, tol = got.double(), tol.nan_to_num(0.0, 0.0, 0.0)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    far = torch.isinf(want)
    assert torch.equal(got[far], want[far])
    fine = torch.isfinite(want)
    assert bool(((got - want).abs()[fine] <= tol[fine]).all())


def inputs(tokens, heads, d, dim, t):
    x, g, w = randn((1, tokens, heads, d), t, 1), randn((1, tokens, heads, d), t, 2), randn((d,), t, 3)
    return x, g, w, QkNorm(rope_of(dim, tokens, t), w, w, 1e-6), range(0, tokens)


# Tokens: few, a warp for each; many, through the rings of the copies.  The address moved by one element: element by element.
CALLS = [(5, 4, 128, 64, 0), (9, 2, 64, 16, 0), (20000, 8, 64, 32, 0), (20000, 4, 128, 64, 0), (12000, 16, 80, 40, 0), (300, 3, 80, 40, 0), (20, 2, 256, 128, 0), (12, 3, 24, 8, 1), (7, 2, 17, 6, 0)]


def moved(x, by):
    return x if by == 0 else torch.cat([x.flatten()[:by], x.flatten()])[by:].view(x.shape)


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("tokens,heads,d,dim,by", CALLS)
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
def test_forward(tokens, heads, d, dim, by, bad, dtype):
    t = TORCH[dtype]
    x, _, w, norm, at = inputs(tokens, heads, d, dim, t)
    for i, c in enumerate(range(dim, d, 5)):   # one feature of one head of one token, here and there
        x[0, (3 * i + 1) % tokens, i % heads, c] = bad
    x = moved(x, by)
    q, k = norm.apply_range(x, x[:, :, :1], at)
    x64 = x[0].double()
    n = x64 / torch.sqrt(x64.square().mean(-1, keepdim=True) + 1e-6) * w.double()
    want, size = turn(n, norm.rope)
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0
    tol = torch.finfo(t).eps / 2 * want.abs() + 32 * U * size + tiny
    same(q[0], want, tol)
    same(k[0], want[:, :1], tol[:, :1])


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("tokens,heads,d,dim,by", CALLS)
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
def test_gradient(tokens, heads, d, dim, by, bad, dtype):
    t = TORCH[dtype]
    x, g, w, norm, at = inputs(tokens, heads, d, dim, t)
    spoilt = list(range(dim, d, 7))[:3]
    for i, c in enumerate(spoilt):
        g[0, (5 * i + 2) % tokens, i % heads, c] = bad
    x, g = moved(x, by), moved(g, by)
    none = x[:, :, :0]
    grads = norm.backward_range(x, none, g, none, at)
    x64, w64 = x[0].double(), w.double()
    r = 1 / torch.sqrt(x64.square().mean(-1, keepdim=True) + 1e-6)
    back, size = turn(g[0].double(), norm.rope, back=True)
    want = r * (w64 * back - x64 * r * r * (x64 * w64 * back).sum(-1, keepdim=True) / d)
    mag = r * w64.abs() * size + x64.abs() * r ** 3 * ((x64 * w64).abs() * size).sum(-1, keepdim=True) / d
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0
    h = torch.finfo(t).eps / 2
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(grads.query[0]), fine)   # (which of an infinity and a NaN goes by the order of the sums)
    assert bool(((grads.query[0].double() - want).abs()[fine] <= (h * want.abs() + 64 * U * mag + tiny)[fine]).all())
    dw, dw_size = (back * x64 * r).sum((0, 1)), (size * (x64 * r).abs()).sum((0, 1))
    kept = torch.ones(d, dtype=torch.bool, device=DEV)
    kept[spoilt] = False
    assert torch.equal(torch.isfinite(grads.query_weight), kept)
    assert bool(((grads.query_weight.double() - dw).abs()[kept] <= (h * dw.abs() + 300 * U * dw_size + tiny)[kept]).all())


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("tokens,heads,d,dim,by", CALLS)
def test_an_infinite_weight(tokens, heads, d, dim, by, dtype):
    """The weight of a feature that is not rotated: that feature alone."""
    t = TORCH[dtype]
    x, _, w, norm, at = inputs(tokens, heads, d, dim, t)
    w[dim + 1] = INF
    x = moved(x, by)
    q, _ = norm.apply_range(x, x[:, :, :1], at)
    x64 = x[0].double()
    want, size = turn(x64 / torch.sqrt(x64.square().mean(-1, keepdim=True) + 1e-6) * w.double(), norm.rope)
    same(q[0], want, torch.finfo(t).eps / 2 * want.abs() + 32 * U * size + (2.0 ** -25 if t == torch.float16 else 0.0))
