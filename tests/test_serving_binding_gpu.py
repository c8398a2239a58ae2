"""The native host side of the norm with rotation, the step over shared prompts and the rules on logits: the Python side's bits for the calls it makes,
and what it leaves to it."""
import pytest
import torch

from dashmag_b200 import _lib
from dashmag_b200.attention import AttentionError, Unsupported
from dashmag_b200.contract import AttentionOptions
from dashmag_b200.penalties import Penalties, penalize
from dashmag_b200.prefix import attention_decode_shared, attention_decode_shared_append
from dashmag_b200.qk_norm import QkNorm
from dashmag_b200.rope import Rope
from test_binding_gpu import Noted, Nothing, randn

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def calls():
    """Each call, and whether the native side makes it."""
    rope = Rope(64, 10000.0, 200, BF16)
    qkv = randn(2, 40, 8 * 64)
    q, k = qkv[..., :256].unflatten(-1, (4, 64)), qkv[..., 256:384].unflatten(-1, (2, 64))
    gq, gk = randn(2, 40, 4, 64), randn(2, 40, 2, 64)
    cu = torch.tensor([0, 15, 40], dtype=torch.int32, device="cuda")
    pos = torch.tensor([3, 199], device="cuda")
    for wq, wk in ((randn(64), randn(64, seed=1)), (randn(64, dtype=torch.float32), None), (None, None)):
        norm = QkNorm(rope, wq, wk, 1e-5)
        yield True, lambda norm=norm: norm.apply_range(q, k, range(3, 43))
        yield True, lambda norm=norm: norm.backward_range(q, k, gq, gk, range(3, 43))
        yield True, lambda norm=norm: norm.apply_at(q[:, 0], k[:, 0], pos)
        yield True, lambda norm=norm: norm.backward_at(q[:, 0], k[:, 0], gq[:, 0], gk[:, 0], pos.int())
        yield True, lambda norm=norm: norm.apply_packed(q[0], k[0], cu, start=7)
        yield True, lambda norm=norm: norm.backward_packed(q[:1], k[:1], gq[:1], gk[:1], cu.long())
    yield False, lambda: norm.apply_range(q.transpose(2, 3).contiguous().transpose(2, 3), k, range(3, 43))   # copied
    yield False, lambda: norm.backward_range(q, k, gq.sum(-1, keepdim=True).expand(2, 40, 4, 64), gk, range(3, 43))
    n, each, p, s = 2, 3, 150, 20
    dq, pk, pv, ck, cv = randn(6, 4, 64), randn(n, p, 2, 64), randn(n, p, 2, 64, seed=1), randn(6, s, 2, 64), randn(6, s, 2, 64, seed=1)
    nk, nv = randn(6, 2, 64), randn(6, 2, 64, seed=1)
    lens, plens = torch.tensor([0, 19, 20, 3, 4, 5], device="cuda"), torch.tensor([150, 60], dtype=torch.int32, device="cuda")
    for options in (AttentionOptions(), AttentionOptions().with_window(30, 0).with_scale(0.3)):
        yield True, lambda o=options: (attention_decode_shared(dq, pk, pv, ck, cv, lens, plens, o),)
        yield True, lambda o=options: (attention_decode_shared(dq, pk, pv, ck, cv, None, None, o),)

        def append(new_k, o=options):
            kk, vv = ck.clone(), cv.clone()
            return attention_decode_shared_append(dq, new_k, nv, pk, pv, kk, vv, lens.int(), plens, o), kk, vv

        yield True, lambda f=append: f(nk)
        yield False, lambda f=append: f(nk.transpose(1, 2).contiguous().transpose(1, 2))
    z = randn(5, 1003, dtype=torch.float32)
    ids = torch.randint(0, 1003, (5, 30), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    f = torch.rand(5, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) + 0.5
    words = torch.full((5, 32), 0x5555_5555, dtype=torch.int32, device="cuda")
    for rules in (Penalties(), Penalties(tokens=ids, repetition=1.2, frequency=1, presence=0.5), Penalties(tokens=ids.int(), lengths=ids[:, 0] % 31, repetition=f, frequency=f),
                  Penalties(tokens=ids[:, ::1], prompt_lengths=torch.full((5,), 9, dtype=torch.int32, device="cuda"), presence=f, bias=z[0], allowed=words),
                  Penalties(bias=z * 0.1, allowed=words[1])):
        yield True, lambda r=rules: (penalize(z, r),)
        yield True, lambda r=rules: (penalize(z[:, 3:1000].half(), Penalties(tokens=r.tokens, repetition=r.repetition)),)
    yield False, lambda: (penalize(z.t().contiguous().t(), Penalties()),)
    yield False, lambda: (penalize(z, Penalties(tokens=ids[:, ::2], repetition=1.5)),)
    yield False, lambda: (penalize(z, Penalties(), out=torch.empty_like(z)),)


def test_the_same_bits(monkeypatch):
    native = _lib.binding()
    for i, (made, call) in enumerate(calls()):
        noted = Noted(native)
        monkeypatch.setattr(_lib, "_binding", noted)
        got = call()
        assert (noted.made == [True]) == made, f"call {i}"   # (with an output given it is not even asked)
        monkeypatch.setattr(_lib, "_binding", Nothing())
        for a, b in zip(got, call()):
            assert (a is None) == (b is None) and (a is None or torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) and a.dtype == b.dtype), f"call {i}"
            assert a is None or not a.requires_grad


def test_refusals_are_the_c_abi_s():
    q, pk, ck = randn(6, 4, 64), randn(4, 50, 2, 64), randn(6, 9, 2, 64)
    with pytest.raises(AttentionError, match="multiple of the prompts"):
        attention_decode_shared(q, pk, pk, ck, ck)
    with pytest.raises(AttentionError, match="repetition"):
        penalize(randn(2, 30), Penalties(tokens=torch.zeros((2, 3), dtype=torch.int32, device="cuda"), repetition=0.0))
    rope = Rope(64, 10000.0, 20, BF16)
    with pytest.raises(AttentionError, match="Rope"):
        QkNorm(rope).apply_range(randn(1, 30, 2, 64), randn(1, 30, 2, 64), range(0, 30))
    with pytest.raises(AttentionError):
        QkNorm(rope).apply_at(randn(3, 2, 64), randn(3, 2, 64), torch.zeros(3, device="cuda"))
    with pytest.raises(Unsupported, match="CUDA device"):
        penalize(randn(2, 30), Penalties(tokens=torch.zeros((2, 3), dtype=torch.int32), repetition=1.5))
