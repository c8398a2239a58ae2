"""Sequences whose window begins behind their prompt, beside others that still see its end: what lies past the prompt's length reaches neither.

A window of `left` keys hides the whole prompt from a sequence that holds more than `left` of its own.  Rows of the tensor cores' tiles go by
warps of 32; the batches here have warps of such rows alone, of such rows and of nobody's, and of both kinds."""
import pytest
import torch

from dashmag_b200.contract import AttentionOptions
from dashmag_b200.prefix import attention_decode_shared, attention_decode_shared_append

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype).to(DEV)


def expected(q, pk, pv, k, v, plens, lens, left):
    """One sequence at a time in f64."""
    b, hq, d = q.shape
    hkv, each = pk.shape[2], b // pk.shape[0]
    out = torch.zeros(b, hq, d, dtype=torch.float64, device=DEV)
    for i in range(b):
        first = max(0, plens[i // each] + lens[i] - 1 - left)
        keys, values = (torch.cat([x[i // each, : plens[i // each]], y[i, : lens[i]]])[first:].double() for x, y in ((pk, k), (pv, v)))
        w = torch.softmax(torch.einsum("hgd,shd->hgs", q[i].double().view(hkv, -1, d), keys) * d ** -0.5, -1)
        out[i] = torch.einsum("hgs,shd->hgd", w, values).reshape(hq, d)
    return out


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("d", [64, 128, 256, 80, 72])
@pytest.mark.parametrize("n,each,hq,hkv", [(2, 24, 8, 2), (2, 9, 8, 1), (1, 70, 4, 4), (3, 5, 96, 2), (2, 40, 6, 2)])
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_past_the_prompt_under_a_window(n, each, hq, hkv, d, dtype, bad):
    t, b, p, s, left = TORCH[dtype], n * each, 400, 60, 30
    q = randn((b, hq, d), t, 1)
    clean = [randn(shape, t, 2 + i) for i, shape in enumerate([(n, p, hkv, d)] * 2 + [(b, s, hkv, d)] * 2)]
    for plens in ([100] * n, [129] * n, [1] * n, [255] * n, [64] * n):
        for lens in ([3] + [31 + i % 29 for i in range(b - 1)],                     # one sees the prompt's end
                     [3 if i % each < each // 3 else 40 for i in range(b)],          # the first ones do
                     [60 if i % 2 else 8 for i in range(b)]):                        # every other one does
            pk, pv, k, v = (x.clone() for x in clean)
            for i, m in enumerate(plens):
                pk[i, m:], pv[i, m:] = float(bad), float(bad)
            options = AttentionOptions().with_window(left, 0)
            args = torch.tensor(lens, device=DEV), torch.tensor(plens, device=DEV), options
            got = attention_decode_shared(q, pk, pv, k, v, *args)
            assert torch.equal(got, attention_decode_shared(q, *clean, *args))
            want = expected(q, *clean, plens, lens, left)
            # (The arithmetic's own tests are elsewhere: here a step of the dtype on values below four.)
            assert bool(((got.double() - want).abs() <= 4 * torch.finfo(t).eps + 1e-5).all())


@pytest.mark.parametrize("dtype", list(TORCH))
def test_the_step_that_appends(dtype):
    t, n, each, hq, hkv, d, p, s, left = TORCH[dtype], 2, 24, 8, 2, 128, 300, 50, 20
    b = n * each
    q, kn, vn = randn((b, hq, d), t, 1), randn((b, hkv, d), t, 2), randn((b, hkv, d), t, 3)
    clean = [randn(shape, t, 4 + i) for i, shape in enumerate([(n, p, hkv, d)] * 2 + [(b, s, hkv, d)] * 2)]
    plens, lens = [100, 200], [2 if i % each < 8 else 25 + i % 20 for i in range(b)]
    pk, pv = clean[0].clone(), clean[1].clone()
    for i, m in enumerate(plens):
        pk[i, m:], pv[i, m:] = float("nan"), float("nan")
    args = torch.tensor(lens, device=DEV), torch.tensor(plens, device=DEV), AttentionOptions().with_window(left, 0)
    got, want = (attention_decode_shared_append(q, kn, vn, x, y, clean[2].clone(), clean[3].clone(), *args) for x, y in ((pk, pv), clean[:2]))
    assert torch.equal(got, want) and bool(torch.isfinite(got).all())
