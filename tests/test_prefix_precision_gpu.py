"""The probabilities of the step over shared prompts: held as finely as the decoding step holds them.

A probability goes to the tensor cores as the sum of two 16-bit values, so that of one of size p no more than h^2 p is lost, h = eps / 2 of
the dtype; an f16 value below the normal range is off by up to 2^-25 of the largest.  Bounds, u = 2^-24 and w the exact weights: h of the
result for its own rounding; h^2 of the sum of w |v| for the probabilities; (2 (D + 16) A + 64) u of it for scores (A the largest sum of a score's
terms' magnitudes), exponentials, sums and the merge; and n / 4 u of it for the accumulation over n keys, two roundings of up to 2 u for
every sixteen of them and each of the two parts.  Outputs near zero, whose terms cancel, show the difference: one rounding of a
probability is h of a term."""
import pytest
import torch

from dashmag_b200 import attention as A
from dashmag_b200.prefix import attention_decode_shared

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype).to(DEV)


def share_of_bound(got, q, keys, values):
    """The largest error over its bound; `keys` and `values` [B, S, Hkv, D]."""
    b, hq, d = q.shape
    hkv = keys.shape[2]
    q64, k64, v64 = q.double().view(b, hkv, hq // hkv, d), keys.double(), values.double()
    w = torch.softmax(torch.einsum("bhgd,bshd->bhgs", q64, k64) * d ** -0.5, -1)
    want = torch.einsum("bhgs,bshd->bhgd", w, v64).reshape(b, hq, d)
    size = torch.einsum("bhgs,bshd->bhgd", w, v64.abs()).reshape(b, hq, d)
    a = (torch.einsum("bhgd,bshd->bhgs", q64.abs(), k64.abs()) * d ** -0.5).amax(-1).reshape(b, hq, 1)
    h = torch.finfo(got.dtype).eps / 2
    tol = h * want.abs() + (h * h + (2 * (d + 16) * a + 64 + keys.shape[1] / 4) * U) * size
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (1 + w.amax(-1).reshape(b, hq, 1) * v64.abs().sum(1).repeat_interleave(hq // hkv, 1))
    return float(((got.double() - want).abs() / tol).max())


# n, each, p, s, hq, hkv, d
DIMS = [
    (1, 8, 24, 8, 16, 4, 64),
    (3, 40, 70, 5, 8, 2, 64),      # two tiles of rows
    (2, 5, 300, 20, 8, 2, 128),
    (4, 6, 200, 1, 6, 1, 128),
    (2, 5, 130, 30, 8, 2, 256),
    (2, 3, 40, 16, 8, 2, 80),      # own keys swept too
    (2, 4, 33, 90, 4, 4, 136),
    (1, 33, 1500, 40, 8, 8, 128),
]


@pytest.mark.parametrize("dtype", list(TORCH))
@pytest.mark.parametrize("dims", DIMS, ids=str)
def test_probabilities_in_two_parts(dims, dtype):
    n, each, p, s, hq, hkv, d = dims
    t, b = TORCH[dtype], n * each
    q = randn((b, hq, d), t, 1)
    pk, pv, k, v = (randn(shape, t, 2 + i) for i, shape in enumerate([(n, p, hkv, d)] * 2 + [(b, s, hkv, d)] * 2))
    keys, values = (torch.cat([x.repeat_interleave(each, 0), y], 1) for x, y in ((pk, k), (pv, v)))
    assert share_of_bound(attention_decode_shared(q, pk, pv, k, v), q, keys, values) <= 1
    assert share_of_bound(A.attention_decode(q, keys, values), q, keys, values) <= 1   # the step over joined caches keeps the same bound
