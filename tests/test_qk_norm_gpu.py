"""The norm of queries and keys with the rotation in the same pass, and its gradient, against the formulas in 64 bits.

Bounds, u = 2^-24 and h the half step of the dtype (eps / 2): a sum of a head's squares is at most 25 additions deep, its root and the
reciprocal four steps, the products and the sum of the rotation four: 32 u of the sum of the terms' magnitudes, and h of the result for the
rounding.  The gradient has one more such sum: 64 u.  A weight's gradient is a sum
of one lane's tokens and heads (at most 200 of them at these sizes, as twenty thousand tokens are dealt out), of its warps and blocks: 300 u."""
import numpy as np
import pytest
import torch

from dashmag_b200 import _lib
from dashmag_b200.qk_norm import QkNorm
from dashmag_b200.rope import Rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24
# (features rotated, head dimension): whole heads, parts, a lane's columns that fill no warp, shapes too narrow or too ragged for vectors
SHAPES = [(128, 128), (64, 128), (64, 64), (256, 256), (48, 96), (80, 80), (16, 16), (2, 2), (6, 17), (100, 250), (40, 80), (24, 72), (8, 8), (24, 256), (8, 200)]


def smallest(dtype):
    """Half of the dtype's smallest step."""
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def make(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(dtype).to(DEV)


def make_rope(dim, held, dtype):
    angle = torch.arange(held, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * (torch.arange(dim, dtype=torch.float64) % (dim // 2)) / dim)
    return Rope.from_tables(angle.cos().to(dtype).to(DEV), angle.sin().to(dtype).to(DEV))


def turn(x, rope, pos, back=False):
    """x [tokens, H, D] in f64 turned by its tokens' rows, and the sum of the terms' magnitudes."""
    half = rope.dim // 2
    cos, sin = rope.cos.double()[pos][:, None, :], rope.sin.double()[pos][:, None, :]
    lo, hi = x[..., :half], x[..., half: rope.dim]
    c1, c2, s1, s2 = cos[..., :half], cos[..., half:], sin[..., :half], sin[..., half:]
    y, mag = x.clone(), x.abs()
    if back:
        y[..., :half], y[..., half: rope.dim] = lo * c1 + hi * s2, hi * c2 - lo * s1
        mag[..., :half], mag[..., half: rope.dim] = (lo * c1).abs() + (hi * s2).abs(), (hi * c2).abs() + (lo * s1).abs()
    else:
        y[..., :half], y[..., half: rope.dim] = lo * c1 - hi * s1, hi * c2 + lo * s2
        mag[..., :half], mag[..., half: rope.dim] = (lo * c1).abs() + (hi * s1).abs(), (hi * c2).abs() + (lo * s2).abs()
    return y, mag


def check_forward(got, x, w, rope, pos, eps=1e-6):
    x64 = x.double().reshape(-1, *x.shape[-2:])
    r = 1 / torch.sqrt(x64.square().mean(-1, keepdim=True) + eps)
    want, mag = turn(x64 * r * (1.0 if w is None else w.double()), rope, pos)
    h = torch.finfo(x.dtype).eps / 2
    off = (got.double().reshape(want.shape) - want).abs()
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    assert bool((off <= h * want.abs() + 32 * U * mag + smallest(x.dtype)).all()), float((off / (h * want.abs() + 32 * U * mag + 1e-300)).max())


def check_backward(dx, dw, x, w, g, rope, pos, eps=1e-6):
    x64, g64 = x.double().reshape(-1, *x.shape[-2:]), g.double().reshape(-1, *g.shape[-2:])
    w64 = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    d = x.shape[-1]
    r = 1 / torch.sqrt(x64.square().mean(-1, keepdim=True) + eps)
    back, mag = turn(g64, rope, pos, back=True)
    along = (x64 * w64 * back).sum(-1, keepdim=True)
    want = r * w64 * back - x64 * r ** 3 * along / d
    size = r * w64.abs() * mag + x64.abs() * r ** 3 * (x64 * w64).abs().mul(mag).sum(-1, keepdim=True) / d
    h = torch.finfo(x.dtype).eps / 2
    off = (dx.double().reshape(want.shape) - want).abs()
    assert dx.shape == x.shape and dx.dtype == x.dtype and dx.is_contiguous()
    assert bool((off <= h * want.abs() + 64 * U * size + smallest(x.dtype)).all()), float((off / (h * want.abs() + 64 * U * size + 1e-300)).max())
    if w is None:
        assert dw is None
        return
    want, size = (back * x64 * r).sum((0, 1)), (mag * (x64 * r).abs()).sum((0, 1))
    off = (dw.double() - want).abs()
    assert dw.dtype == w.dtype and dw.shape == w.shape
    assert bool((off <= torch.finfo(w.dtype).eps / 2 * want.abs() + 300 * U * size + smallest(w.dtype)).all()), float((off / (size + 1e-300)).max() / U)


def where(form, b, t):
    """The call's extra arguments and every token's position."""
    if form == "range":
        return (range(5, 5 + t),), torch.arange(5, 5 + t).repeat(b)
    if form == "at":
        pos = torch.tensor([(7 * i + 3) % 40 for i in range(b * t)])
        return (pos.to(torch.int32 if b % 2 else torch.int64).to(DEV),), pos
    cu = [0, 1, 1, max(1, b * t // 3), b * t]
    return (torch.tensor(cu, dtype=torch.int64 if t % 2 else torch.int32, device=DEV),), torch.cat([torch.arange(n) for n in np.diff(cu)])


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("dim,d", SHAPES)
@pytest.mark.parametrize("form", ["range", "at", "packed"])
def test_forward_and_gradients(dim, d, dtype, form):
    t = TORCH[dtype]
    b, n = 3, 11
    lead = (b, n) if form == "range" else (b * n,)
    hq, hkv = 5, 2
    q, k, gq, gk = (make((*lead, h, d), t, s) for s, h in enumerate((hq, hkv, hq, hkv)))
    wdtype = torch.float32 if dim % 4 == 0 else t
    wq, wk = (make((d,), wdtype, 10 + s, 0.3) + 1 for s in range(2))
    rope = make_rope(dim, 64, t)
    norm = QkNorm(rope, wq, wk)
    args, pos = where(form, b, n)
    oq, ok = getattr(norm, "apply_" + form)(q, k, *args)
    check_forward(oq, q, wq, rope, pos)
    check_forward(ok, k, wk, rope, pos)
    grads = getattr(norm, "backward_" + form)(q, k, gq, gk, *args)
    check_backward(grads.query, grads.query_weight, q, wq, gq, rope, pos)
    check_backward(grads.key, grads.key_weight, k, wk, gk, rope, pos)


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (16, 16, 64), (1, 1, 256), (7, 1, 96)])
def test_slices_of_one_projection(hq, hkv, d, dtype):
    """Queries and keys that lie side by side in a projection's output are read in place."""
    t = TORCH[dtype]
    qkv = make((2, 300, (hq + 2 * hkv) * d), t, 1)
    q = qkv[..., : hq * d].unflatten(-1, (hq, d))
    k = qkv[..., hq * d: (hq + hkv) * d].unflatten(-1, (hkv, d))
    gq, gk = make((2, 300, hq, d), t, 2), make((2, hkv, 300, d), t, 3).transpose(1, 2)
    rope = make_rope(d, 400, t)
    norm = QkNorm(rope, make((d,), t, 4), make((d,), t, 5), eps=1e-5)
    pos = torch.arange(20, 320).repeat(2)
    oq, ok = norm.apply_range(q, k, range(20, 320))
    check_forward(oq, q, norm.query_weight, rope, pos, 1e-5)
    check_forward(ok, k, norm.key_weight, rope, pos, 1e-5)
    g = norm.backward_range(q, k, gq, gk, range(20, 320))
    check_backward(g[0], g[2], q, norm.query_weight, gq, rope, pos, 1e-5)
    check_backward(g[1], g[3], k, norm.key_weight, gk, rope, pos, 1e-5)
    # a part of the time, every other head, features that are not contiguous, an address off 16 bytes
    views = [(q[:, 3:100], k[:, 3:100]), (q[:, ::3, ::2][:, :97], k[:, ::3][:, :97]),
             (make((2, 97, d, hq), t, 6).transpose(2, 3), make((2, 97, hkv, d + 1), t, 7)[..., 1:])]
    for a, b in views:
        oq, ok = norm.apply_range(a, b, range(0, 97))
        pos = torch.arange(97).repeat(2)
        check_forward(oq, a, norm.query_weight, rope, pos, 1e-5)
        check_forward(ok, b, norm.key_weight, rope, pos, 1e-5)
        g = norm.backward_range(a, b, oq, ok, range(0, 97))
        check_backward(g[0], g[2], a, norm.query_weight, oq, rope, pos, 1e-5)
        check_backward(g[1], g[3], b, norm.key_weight, ok, rope, pos, 1e-5)


def test_without_weights_and_one_weight():
    rope = make_rope(64, 64, torch.bfloat16)
    q, k = make((20, 4, 64), torch.bfloat16, 1), make((20, 4, 64), torch.bfloat16, 2)
    pos = torch.arange(20)
    for wq, wk in ((None, None), (make((64,), torch.float32, 3), None), (None, make((64,), torch.bfloat16, 4))):
        norm = QkNorm(rope, wq, wk)
        oq, ok = norm.apply_at(q, k, pos.to(DEV))
        check_forward(oq, q, wq, rope, pos)
        check_forward(ok, k, wk, rope, pos)
        g = norm.backward_at(q, k, oq, ok, pos.to(DEV))
        check_backward(g.query, g.query_weight, q, wq, oq, rope, pos)
        check_backward(g.key, g.key_weight, k, wk, ok, rope, pos)


@pytest.mark.parametrize("d", [64, 34])
def test_tokens_of_no_sequence_and_positions_outside(d):
    """Tokens before the first offset and behind the last pass unchanged, and so do their gradients; a position outside the tables gives
    NaN in the rotated features and nothing is read there."""
    t = torch.bfloat16
    rope = make_rope(32, 16, t)
    norm = QkNorm(rope, make((d,), t, 1), make((d,), t, 2))
    q, k, gq, gk = make((30, 3, d), t, 3), make((30, 1, d), t, 4), make((30, 3, d), t, 5), make((30, 1, d), t, 6)
    cu = torch.tensor([4, 10, 22], dtype=torch.int32, device=DEV)
    oq, ok = norm.apply_packed(q, k, cu)
    pos = torch.cat([torch.arange(6), torch.arange(12)])
    check_forward(oq[4:22], q[4:22], norm.query_weight, rope, pos)
    g = norm.backward_packed(q, k, gq, gk, cu)
    check_backward(g.query[4:22], g.query_weight, q[4:22], norm.query_weight, gq[4:22], rope, pos)
    check_backward(g.key[4:22], g.key_weight, k[4:22], norm.key_weight, gk[4:22], rope, pos)
    for rows in (slice(0, 4), slice(22, 30)):
        assert torch.equal(oq[rows], q[rows]) and torch.equal(ok[rows], k[rows])
        assert torch.equal(g.query[rows], gq[rows]) and torch.equal(g.key[rows], gk[rows])
    at = torch.tensor([15, 16, -1], device=DEV)
    oq, ok = norm.apply_at(q[:3], k[:3], at)
    check_forward(oq[:1], q[:1], norm.query_weight, rope, torch.tensor([15]))
    assert torch.isnan(oq[1:, :, :32]).all() and torch.isfinite(oq[1:, :, 32:]).all()
    empty = torch.tensor([0], dtype=torch.int64, device=DEV)
    assert torch.equal(norm.apply_packed(q, k, empty)[0], q)


def test_no_tokens():
    t = torch.float16
    rope = make_rope(32, 16, t)
    norm = QkNorm(rope, make((32,), t, 1), make((32,), t, 2))
    q, k = make((0, 3, 32), t, 3), make((0, 1, 32), t, 4)
    at = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert norm.apply_at(q, k, at)[0].shape == (0, 3, 32)
    g = norm.backward_at(q, k, q, k, at)
    assert g.query.shape == (0, 3, 32) and not g.query_weight.any() and not g.key_weight.any()


@pytest.mark.parametrize("d", [64, 34])
def test_a_tensor_without_heads(d):
    """Its weight's gradient is an empty sum."""
    t = torch.bfloat16
    rope = make_rope(32, 64, t)
    norm = QkNorm(rope, make((d,), t, 1), make((d,), t, 2))
    q, none = make((20, 3, d), t, 3), make((20, 0, d), t, 4)
    pos = torch.arange(20)
    for a, b, x in ((q, none, 0), (none, q, 1)):
        out = norm.apply_at(a, b, pos.to(DEV))
        check_forward(out[x], q, (norm.query_weight, norm.key_weight)[x], rope, pos)
        g = norm.backward_at(a, b, a, b, pos.to(DEV))
        check_backward(g[x], g[2 + x], q, (norm.query_weight, norm.key_weight)[x], q, rope, pos)
        assert not g[3 - x].any() and g[1 - x].numel() == 0


@pytest.mark.parametrize("tokens,d", [(5, 64), (5, 34), (9000, 64)])
def test_in_place_through_the_c_abi(tokens, d):
    """Contiguous tensors may be their own results."""
    import ctypes

    t = torch.bfloat16
    rope = make_rope(32, tokens, t)
    q, k = make((1, tokens, 16, d), t, 3), make((1, tokens, 4, d), t, 4)
    norm = QkNorm(rope)
    want = norm.apply_range(q, k, range(tokens))
    p, _, _ = norm._params("qk_norm", q, k, {"start": 0})
    tables = rope.tables()
    assert _lib.lib().dash_rope_norm_apply(ctypes.byref(tables), ctypes.byref(p), q.data_ptr(), k.data_ptr(), None, None, q.data_ptr(), k.data_ptr(),
                                           torch.cuda.current_stream().cuda_stream) == _lib.OK
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("hq,hkv,d,dim", [(32, 8, 128, 128), (16, 4, 64, 64), (8, 1, 64, 32), (5, 3, 96, 96), (70, 2, 32, 32), (12, 12, 256, 128), (16, 4, 80, 40), (3, 1, 40, 24), (9, 2, 248, 8)])
def test_many_tokens(hq, hkv, d, dim, dtype):
    """Long enough that every warp takes tokens one after another, several at a time where their heads are few, in sequences that end anywhere."""
    t = TORCH[dtype]
    n = 6007 if (hq + hkv) * d > 2000 else 20011
    rope = make_rope(dim, n, t)
    norm = QkNorm(rope, make((d,), t, 1), make((d,), t, 2))
    q, k, gq, gk = (make((n, h, d), t, s) for s, h in enumerate((hq, hkv, hq, hkv)))
    cu = [3, 3, 1000, 1001, 2500, n - 5]
    args = torch.tensor(cu, dtype=torch.int32, device=DEV)
    pos = torch.cat([torch.arange(b - a) for a, b in zip(cu, cu[1:])])
    oq, ok = norm.apply_packed(q, k, args)
    rows = slice(cu[0], cu[-1])
    check_forward(oq[rows], q[rows], norm.query_weight, rope, pos)
    check_forward(ok[rows], k[rows], norm.key_weight, rope, pos)
    g = norm.backward_packed(q, k, gq, gk, args)
    check_backward(g.query[rows], g.query_weight, q[rows], norm.query_weight, gq[rows], rope, pos)
    check_backward(g.key[rows], g.key_weight, k[rows], norm.key_weight, gk[rows], rope, pos)
    for rows in (slice(0, cu[0]), slice(cu[-1], n)):
        assert torch.equal(oq[rows], q[rows]) and torch.equal(g.key[rows], gk[rows])
    assert _lib.lib().dash_attn_device_status(0) == 0


def test_zeros_and_large_heads():
    """A head of zeros is zeros (eps keeps its norm finite); one of large values is as good as any."""
    for t in TORCH.values():
        rope = make_rope(64, 8, t)
        norm = QkNorm(rope, make((64,), t, 1), None)
        q = make((8, 4, 64), t, 2)
        q[:, 1] = 0
        q[:, 2] *= 1e4
        q[:, 3] *= 1e-3
        pos = torch.arange(8)
        oq, _ = norm.apply_at(q, q, pos.to(DEV))
        check_forward(oq, q, norm.query_weight, rope, pos)
        g = norm.backward_at(q, q, oq, oq, pos.to(DEV))
        check_backward(g.query, g.query_weight, q, norm.query_weight, oq, rope, pos)


def test_the_gradient_against_differences():
    """In f32, along random directions: the difference quotient of the f64 formula at the same point."""
    t, d = torch.float32, 48
    rope = make_rope(32, 16, t)
    q, k, gq, gk = make((9, 3, d), t, 1), make((9, 2, d), t, 2), make((9, 3, d), t, 3), make((9, 2, d), t, 4)
    wq, wk = make((d,), t, 5), make((d,), t, 6)
    pos = torch.arange(9)
    g = QkNorm(rope, wq, wk).backward_at(q, k, gq, gk, pos.to(DEV))

    def loss(q, k, wq, wk):
        total = 0.0
        for x, w, grad in ((q, wq, gq), (k, wk, gk)):
            y, _ = turn(x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w, rope, pos)
            total = total + (y * grad.double()).sum()
        return float(total)

    point = [x.double() for x in (q, k, wq, wk)]
    step = 1e-5
    for i, got in enumerate(g):
        way = make(got.shape, torch.float64, 20 + i)
        up, down = ([x + s * step * way if j == i else x for j, x in enumerate(point)] for s in (1, -1))
        want = (loss(*up) - loss(*down)) / (2 * step)
        # the quotient's own error is of the order of step^2, the sum's of the results' f32
        assert abs(float((got.double() * way).sum()) - want) <= 1e-6 * float((got.double() * way).abs().sum()) + 1e-6


def test_the_same_bits_and_the_probe():
    t = torch.bfloat16
    rope = make_rope(128, 4096, t)
    norm = QkNorm(rope, make((128,), t, 1), make((128,), t, 2))
    q, k, gq, gk = make((3000, 8, 128), t, 3), make((3000, 2, 128), t, 4), make((3000, 8, 128), t, 5), make((3000, 2, 128), t, 6)
    cu = torch.tensor([0, 1000, 3000], dtype=torch.int32, device=DEV)
    before = _lib.probe("kernel_launches")
    first = norm.backward_packed(q, k, gq, gk, cu)
    assert _lib.probe("kernel_launches") == before + 2
    norm.apply_packed(q, k, cu)
    assert _lib.probe("kernel_launches") == before + 3
    for _ in range(3):
        for a, b in zip(first, norm.backward_packed(q, k, gq, gk, cu)):
            assert torch.equal(a, b)


def test_captured_and_replayed():
    t = torch.bfloat16
    rope = make_rope(64, 64, t)
    norm = QkNorm(rope, make((64,), t, 1), make((64,), t, 2))
    q, k = make((4, 8, 64), t, 3), make((4, 2, 64), t, 4)
    pos = torch.tensor([1, 2, 3, 4], device=DEV)
    norm.apply_at(q, k, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oq, ok = norm.apply_at(q, k, pos)
        grads = norm.backward_at(q, k, oq, ok, pos)
    for step in range(3):
        q.copy_(make((4, 8, 64), t, 50 + step))
        pos.add_(1)
        graph.replay()
        want = norm.apply_at(q, k, pos)
        assert torch.equal(oq, want[0]) and torch.equal(ok, want[1])
        for a, b in zip(grads, norm.backward_at(q, k, oq, ok, pos)):
            assert torch.equal(a, b)


def test_on_another_stream():
    t = torch.bfloat16
    rope = make_rope(64, 64, t)
    norm = QkNorm(rope, make((64,), t, 1), make((64,), t, 2))
    q, k = make((40, 8, 64), t, 3), make((40, 2, 64), t, 4)
    pos = torch.arange(40, device=DEV)
    want = norm.apply_at(q, k, pos)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = norm.apply_at(q, k, pos)
    stream.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
