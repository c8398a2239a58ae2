"""The repetition penalty's quotient: in f32 the quotient to the bit; in 16 bits, whose result rounds far coarser, within two f32 roundings
before that one; no reciprocal runs out of range, and a row's address changes no bit."""
import numpy as np
import pytest
import torch

from dashmag_b200.penalties import Penalties, penalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("as_tensor", [False, True])
@pytest.mark.parametrize("repetition", [1.1, 1.3, 0.7, 3.0, 1.0 / 3.0, 1e-39, 7e-39, 3.0e38, 1.9e38, 2.0 ** 100, 1e-30])
@pytest.mark.parametrize("t", [40, 40000])
def test_quotients_in_f32(repetition, t, as_tensor):
    """Every token is in the history, of few ids and of more than a 16-bit counter's."""
    b, v = 3, 5001
    g = torch.Generator().manual_seed(int(t))
    logits = torch.randn((b, v), generator=g) * 10.0 ** torch.randint(-6, 6, (b, v), generator=g)
    ids = torch.randint(0, v, (b, t), generator=g, dtype=torch.int32)
    there = torch.zeros((b, v), dtype=torch.bool).scatter_(1, ids.long(), True).numpy()
    r = torch.full((b,), repetition, device=DEV) if as_tensor else repetition
    got = penalize(logits.to(DEV), Penalties(tokens=ids.to(DEV), repetition=r)).cpu().numpy()
    z, r32 = logits.numpy(), np.float32(repetition)
    with np.errstate(all="ignore"):
        want = np.where(there, np.where(z > 0, z / r32, z * r32), z)
    assert want.dtype == np.float32 and there.any() and np.array_equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("repetition", [1.1, 0.7, 3.0, 1e-39, 2e-39, 3.0e38, 2.0 ** 100])
def test_quotients_in_16_bits(repetition, dtype):
    """The quotient is off by at most 2 u = 2^-23 (as f32, or half its smallest step, 2^-150) before the result's own half step."""
    b, v = 3, 5003
    g = torch.Generator().manual_seed(3)
    logits = (torch.randn((b, v), generator=g) * 10.0 ** torch.randint(-4, 4, (b, v), generator=g)).to(dtype)
    logits[:, ::7] *= 1e-3 if dtype == torch.float16 else 1e-36
    ids = torch.randint(0, v, (b, 3000), generator=g, dtype=torch.int32)
    there = torch.zeros((b, v), dtype=torch.bool).scatter_(1, ids.long(), True)
    p = Penalties(tokens=ids.to(DEV), repetition=repetition)
    got = penalize(logits.to(DEV), p).cpu()
    z, r = logits.double(), float(np.float32(repetition))
    want = torch.where(there, torch.where(z > 0, z / r, z * r), z)
    step = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133   # half the smallest step of the dtype, one of f32's 2^-149 before it
    most = torch.finfo(dtype).max * (1 + step)
    over = want.abs() >= most * (1 + 2.0 ** -22)
    assert torch.equal(got[over].double(), torch.sign(want[over]) * float("inf"))
    fine = want.abs() <= torch.finfo(dtype).max
    off = (got.double() - want).abs()[fine]
    assert bool((off <= (step * (1 + 2.0 ** -22) + 2.0 ** -23) * want.abs()[fine] + tiny + 2.0 ** -148).all())
    assert there.any() and torch.equal(got[~there], logits[~there])
    wide = torch.empty((b, v + 1), dtype=dtype, device=DEV)   # rows off 16 bytes, an element at a time
    out = wide[:, 1:]
    assert torch.equal(penalize(logits.to(DEV), p, out).cpu(), got)
