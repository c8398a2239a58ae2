"""The decoding step over shared prompts against softmax over the joined keys in 64 bits.

Bounds, with h the half step of the dtype (eps / 2), u = 2^-24 and w the exact weights: the tensor-core passes round each probability and the
result to the dtype, h (sum of w |v| + |out|) together; a score's f32 sum is off by at most (D + 16) u of the sum of its
terms' magnitudes A, which its weight feels twice (its own and the total's), and exponentials, sums and the merge by less than 64 u more:
(2 (D + 16) A + 64) u of the sum of w |v|.  An f16 probability below the normal range is off by up to 2^-25 of the largest: 2^-25 of the
largest weight times the sum of |v|.  In f32 nothing is rounded to fewer bits: the second part alone."""
import numpy as np
import pytest
import torch

from dashmag_b200 import _lib
from dashmag_b200 import attention as A
from dashmag_b200.contract import AttentionOptions
from dashmag_b200.prefix import attention_decode_shared, attention_decode_shared_append

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(TORCH[dtype]).to(DEV)


def inputs(dtype, n, each, p, s, hq, hkv, d, seed=1):
    b = n * each
    return dict(q=randn((b, hq, d), dtype, seed), pk=randn((n, p, hkv, d), dtype, seed + 1), pv=randn((n, p, hkv, d), dtype, seed + 2),
                k=randn((b, s, hkv, d), dtype, seed + 3), v=randn((b, s, hkv, d), dtype, seed + 4))


def index(x, kind=torch.int32):
    return torch.tensor(x, dtype=kind, device=DEV)


def check(got, x, plens, lens, left=None, scale=None):
    """`lens` with the step's own row counted, cut to the cache."""
    b, hq, d = x["q"].shape
    n, p, hkv, _ = x["pk"].shape
    s = x["k"].shape[1]
    scale = d ** -0.5 if scale is None else scale
    h = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    assert got.shape == x["q"].shape and got.dtype == x["q"].dtype
    for i in range(b):
        m, have = min(max(plens[i // (b // n)], 0), p), min(max(lens[i], 0), s)
        keys = torch.cat([x["pk"][i // (b // n), :m], x["k"][i, :have]]).double()
        values = torch.cat([x["pv"][i // (b // n), :m], x["v"][i, :have]]).double()
        if left is not None:
            keys, values = keys[max(0, m + have - 1 - left):], values[max(0, m + have - 1 - left):]
        if len(keys) == 0:
            assert not got[i].any(), f"sequence {i} sees no key"
            continue
        q = x["q"][i].double().view(hkv, hq // hkv, d)
        w = torch.softmax(torch.einsum("hgd,shd->hgs", q, keys) * scale, -1)
        want = torch.einsum("hgs,shd->hgd", w, values).reshape(hq, d)
        size = torch.einsum("hgs,shd->hgd", w, values.abs()).reshape(hq, d)
        a = (torch.einsum("hgd,shd->hgs", q.abs(), keys.abs()) * abs(scale)).amax(-1).reshape(hq, 1)
        tol = h * (size + want.abs()) + (2 * (d + 16) * a + 64) * U * size + 1e-30
        if got.dtype == torch.float16:
            tol = tol + 2.0 ** -25 * (1 + w.amax(-1).reshape(hq, 1) * values.abs().sum(0).repeat_interleave(hq // hkv, 0))
        off = (got[i].double() - want).abs()
        assert bool((off <= tol).all()), (i, float((off / tol).max()))


# n, each, p, s, hq, hkv, d
DIMS = [
    (1, 4, 1000, 64, 16, 4, 128),      # a short question's answers
    (1, 64, 700, 40, 32, 8, 128),      # two whole tiles of rows
    (3, 5, 129, 17, 8, 2, 64),         # a key past a tile
    (2, 33, 64, 9, 8, 8, 128),         # no groups, rows past a tile
    (4, 3, 128, 130, 12, 4, 64),       # groups of three
    (1, 40, 515, 33, 8, 1, 128),       # groups of eight, tiles cut
    (5, 1, 1, 1, 4, 2, 128),           # one key each
    (2, 7, 300, 20, 8, 2, 256),
    (1, 70, 65, 600, 4, 1, 256),
    (2, 3, 777, 33, 6, 2, 80),         # features that fill no tile
    (2, 5, 200, 70, 8, 2, 136),
    (3, 4, 150, 300, 4, 4, 24),
    (16, 4, 200, 40, 24, 4, 64),       # groups of six: the rows of a tile that are nobody's
    (2, 50, 150, 20, 20, 4, 128),      # of five
    (1, 9, 300, 20, 14, 2, 256),       # of seven
    (1, 3, 300, 20, 96, 2, 128),       # of forty-eight
    (3, 2, 63, 5, 3, 3, 51),           # on the CUDA cores whatever the dtype
    (1, 100, 200, 3, 10, 2, 32),
    (1, 1, 5000, 100, 32, 8, 128),     # one sequence, its prompt over the whole GPU
]


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("dims", DIMS, ids=str)
def test_lengths(dims, dtype):
    n, each, p, s, hq, hkv, d = dims
    x = inputs(dtype, *dims)
    b = n * each
    g = np.random.default_rng(n * 100 + each)
    for plens, lens in ((None, None), (g.integers(0, p + 1, n), g.integers(0, s + 1, b)), ([0] * n, g.integers(0, s + 1, b)), (g.integers(1, p + 1, n), [0] * b),
                        ([0] * n, [0] * b), ([p + 5] * n, [s + 7] * b), ([-1] * n, [-4] * b)):
        plens_, lens_ = None if plens is None else index(plens, torch.int64), None if lens is None else index(lens)
        got = attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"], lens_, plens_)
        check(got, x, [p] * n if plens is None else list(map(int, plens)), [s] * b if lens is None else list(map(int, lens)))
    assert A._lib.lib().dash_attn_device_status(0) == 0


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("dims", DIMS[:4] + DIMS[7:10], ids=str)
@pytest.mark.parametrize("left", [0, 3, 40, 150, 100000])
def test_windows(dims, left, dtype):
    """A window counts over the sequence's own keys and, past their first, the prompt's."""
    n, each, p, s, hq, hkv, d = dims
    x = inputs(dtype, *dims, seed=20)
    g = np.random.default_rng(left)
    plens, lens = g.integers(0, p + 1, n), g.integers(0, s + 1, n * each)
    got = attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"], index(lens), index(plens), AttentionOptions().with_window(left, 0).with_scale(0.2))
    check(got, x, list(map(int, plens)), list(map(int, lens)), left, 0.2)


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("dims", DIMS[:4] + DIMS[6:10], ids=str)
def test_append(dims, dtype):
    """The new rows land at the lengths, count, and nothing else of the caches changes; a full cache takes none."""
    n, each, p, s, hq, hkv, d = dims
    b = n * each
    x = inputs(dtype, *dims, seed=40)
    kn, vn = randn((b, hkv, d), dtype, 50), randn((b, hkv, d), dtype, 51)
    lens = np.random.default_rng(3).integers(0, s + 1, b)
    lens[0] = s
    k, v = x["k"].clone(), x["v"].clone()
    for i in range(b):
        if lens[i] < s:
            k[i, lens[i]], v[i, lens[i]] = kn[i], vn[i]
    got = attention_decode_shared_append(x["q"], kn, vn, x["pk"], x["pv"], x["k"], x["v"], index(lens))
    assert torch.equal(x["k"], k) and torch.equal(x["v"], v)
    check(got, x, [p] * n, [int(i) + 1 for i in lens])
    plens = [p // 2] * n
    got = attention_decode_shared_append(x["q"], kn, vn, x["pk"], x["pv"], x["k"], x["v"], index(lens), index(plens), AttentionOptions().with_window(30, 0))
    assert torch.equal(x["k"], k) and torch.equal(x["v"], v)
    check(got, x, plens, [int(i) + 1 for i in lens], 30)


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("d", [64, 128, 256, 40])
def test_what_lies_past_the_lengths(dtype, d):
    """NaN and infinities behind a prompt's and a sequence's last key are never seen, wherever in a tile the last key is."""
    n, each, p, s, hq, hkv = 2, 6, 400, 90, 8, 2
    clean = inputs(dtype, n, each, p, s, hq, hkv, d, seed=60)
    for plens in ([1, 63], [64, 65], [127, 128], [129, 200], [399, 321], [0, 256]):
        lens = [(i * 17) % (s + 1) for i in range(n * each)]
        x = {k: t.clone() for k, t in clean.items()}
        for i, m in enumerate(plens):
            x["pk"][i, m:] = float("nan")
            x["pv"][i, m:] = float("inf") if i else float("nan")
        for i, m in enumerate(lens):
            x["k"][i, m:] = float("nan")
            x["v"][i, m:] = float("nan")
        got = attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"], index(lens), index(plens))
        want = attention_decode_shared(clean["q"], clean["pk"], clean["pv"], clean["k"], clean["v"], index(lens), index(plens))
        assert torch.equal(got, want)
        check(got, clean, plens, lens)


@pytest.mark.parametrize("dtype", list(TORCH))
def test_a_nan_that_is_seen_is_seen(dtype):
    x = inputs(dtype, 2, 3, 200, 20, 4, 2, 128, seed=70)
    x["pv"][1, 150, 0, 5] = float("nan")
    x["v"][0, 7, 1, 9] = float("nan")
    got = attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"])
    bad = torch.zeros(got.shape, dtype=torch.bool, device=DEV)
    bad[3:, :2, 5] = True
    bad[0, 2:, 9] = True
    assert torch.equal(torch.isnan(got), bad)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_strides_and_which_kernels(dtype):
    """Slices and layouts the tensor cores read in place, and others, which the CUDA cores take; the result is the same call's."""
    n, each, p, s, hq, hkv, d = 2, 8, 300, 50, 8, 2, 128
    x = inputs(dtype, n, each, p, s, hq, hkv, d, seed=80)
    lens, plens = [(5 * i) % (s + 1) for i in range(n * each)], [300, 123]

    def run(tensor, **other):
        y = {**x, **other}
        runs = _lib.probe("tensor_core_runs")
        got = attention_decode_shared(y["q"], y["pk"], y["pv"], y["k"], y["v"], index(lens), index(plens))
        assert _lib.probe("tensor_core_runs") - runs == int(tensor)
        check(got, y, plens, lens)

    run(True)
    run(True, pk=randn((n, 400, hkv, d), dtype, 90)[:, 50:350], pv=randn((n, p, 3 * hkv, d), dtype, 91)[:, :, hkv: 2 * hkv])          # slices
    run(True, pk=randn((n, hkv, p, d), dtype, 92).transpose(1, 2), q=randn((n * each, 2 * hq, d), dtype, 93)[:, 3: 3 + hq])           # heads first
    run(False, pk=randn((n, p, hkv, d + 1), dtype, 94)[..., 1:])                                                                     # rows off 16 bytes
    run(False, pv=randn((n, p, d, hkv), dtype, 95).transpose(2, 3))                                                                  # features apart
    run(False, pk=randn((1, p, hkv, d), dtype, 96).expand(n, p, hkv, d))                                                             # one for all, stride 0
    run(False, q=randn((1, hq, d), dtype, 97).expand(n * each, hq, d))
    run(False, pv=randn((n, p, 1, d), dtype, 98).expand(n, p, hkv, d))


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales(scale, dtype):
    x = inputs(dtype, 2, 3, 150, 20, 4, 2, 64, seed=100)
    got = attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"], None, None, AttentionOptions().with_scale(scale))
    check(got, x, [150] * 2, [20] * 6, None, scale)


@pytest.mark.parametrize("dtype", list(TORCH))
def test_is_the_step_over_joined_caches(dtype):
    """What ``attention_decode`` gives on caches that hold the prompt's rows and then the sequence's own, to the bound; and without
    prompts its very bits."""
    n, each, p, s, hq, hkv, d = 2, 4, 260, 70, 8, 2, 128
    x = inputs(dtype, n, each, p, s, hq, hkv, d, seed=110)
    lens = index([(9 * i) % (s + 1) for i in range(n * each)])
    joined = [torch.cat([a.repeat_interleave(each, 0), b], 1) for a, b in ((x["pk"], x["k"]), (x["pv"], x["v"]))]
    want = A.attention_decode(x["q"], *joined, lens + p)
    got = attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"], lens)
    check(got, x, [p] * n, lens.tolist())
    check(want, x, [p] * n, lens.tolist())
    none = attention_decode_shared(x["q"], x["pk"][:, :0], x["pv"][:, :0], x["k"], x["v"], lens)
    assert torch.equal(none, A.attention_decode(x["q"], x["k"], x["v"], lens))
    check(attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"][:, :0], x["v"][:, :0]), {**x, "k": x["k"][:, :0], "v": x["v"][:, :0]}, [p] * n, [0] * n * each)


def test_nothing_to_do():
    e = torch.zeros((0, 4, 64), device=DEV)
    none = torch.zeros((0, 5, 2, 64), device=DEV)
    assert attention_decode_shared(e, none, none, none, none).shape == (0, 4, 64)
    q = torch.ones((2, 4, 64), device=DEV)
    empty = torch.zeros((1, 0, 2, 64), device=DEV)
    assert not attention_decode_shared(q, empty, empty, torch.zeros((2, 0, 2, 64), device=DEV), torch.zeros((2, 0, 2, 64), device=DEV)).any()


@pytest.mark.parametrize("dtype", list(TORCH))
def test_launches_bits_and_replay(dtype):
    """Three launches; the same bits on every run, replayed from a graph and with other graphs beside it."""
    x = inputs(dtype, 1, 16, 2000, 64, 8, 2, 128, seed=120)
    lens = index([(3 * i) % 60 for i in range(16)])
    before = _lib.probe("kernel_launches")
    first = attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"], lens)
    assert _lib.probe("kernel_launches") == before + 3
    for _ in range(3):
        assert torch.equal(first, attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"], lens))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graphs.append((torch.cuda.CUDAGraph(),))
        with torch.cuda.graph(graphs[-1][0]):
            graphs[-1] += (attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"], lens),)
    for step in range(3):
        x["q"].copy_(randn(x["q"].shape, dtype, 130 + step))
        lens.add_(1)
        for graph, _ in graphs:
            graph.replay()
        want = attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"], lens)
        assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want)


def test_two_streams_at_once():
    xs = [inputs("bf16", 1, 32, 3001, 200, 16, 4, 128, seed=s) for s in (140, 150)]
    want = [attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"]) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for x, stream in zip(xs, streams):
            with torch.cuda.stream(stream):
                got.append(attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"]))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 2])


def test_far_offsets():
    """Prompts whose rows lie past 2^31 elements from the first."""
    free = torch.cuda.mem_get_info()[0]
    n, p, hkv, d = 3, 70000, 128, 128   # 1.1e9 elements a prompt
    if free < 5 * n * p * hkv * d:
        pytest.skip("not enough memory")
    big = torch.empty((n, p, hkv, d), dtype=torch.bfloat16, device=DEV)
    big.zero_()
    x = inputs("bf16", n, 2, 200, 10, 256, 128, 128, seed=160)
    plens = [200, 3, 150]
    big[:, :200] = x["pk"]
    values = big.clone() if free > 13 * n * p * hkv * d else big
    if values is not big:
        values[:, :200] = x["pv"]
    got = attention_decode_shared(x["q"], big, values, x["k"], x["v"], None, index(plens))
    check(got, {**x, "pk": big[:, :200], "pv": values[:, :200]}, plens, [10] * 6)


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,each,p,hq", [(2, 20, 1500, 32), (1, 2, 5000, 8), (1, 80, 300, 32)])
def test_many_parts(n, each, p, hq, d, dtype):
    """Long own caches and prompts, so that a row has parts for several rounds, by all numbers of rows."""
    s = 3000 if n * each < 80 else 900
    x = inputs(dtype, n, each, p, s, hq, 1, d, seed=170)
    lens = np.random.default_rng(d).integers(0, s + 1, n * each)
    lens[0], lens[1] = s, 0
    check(attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"], index(lens)), x, [p] * n, list(map(int, lens)))
