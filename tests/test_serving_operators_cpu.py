"""What the norm with rotation, the step over shared prompts and the rules on logits refuse, before anything reaches a GPU."""
import ctypes

import pytest
import torch

from dashmag_b200 import _lib
from dashmag_b200.attention import AttentionError, Unsupported
from dashmag_b200.penalties import Penalties, penalize
from dashmag_b200.prefix import attention_decode_shared, attention_decode_shared_append
from dashmag_b200.qk_norm import QkNorm
from dashmag_b200.rope import Rope

BF16, F32 = torch.bfloat16, torch.float32


def rope(dim=8, held=16, dtype=F32):
    return Rope(dim, 10000.0, held, dtype, device="cpu")


def test_tables():
    cos, sin = torch.ones((4, 8)), torch.zeros((4, 8))
    r = Rope.from_tables(cos, sin)
    assert (r.dim, len(r), r.dtype) == (8, 4, F32) and r.cos is cos
    for a, b in ((cos, sin[:3]), (cos, sin.to(BF16)), (cos[0], sin[0]), (cos[:, :7], sin[:, :7]), (cos[:, :0], sin[:, :0]), (cos.double(), sin.double())):
        with pytest.raises(AttentionError, match="Rope"):
            Rope.from_tables(a, b)


def test_norm_refusals():
    with pytest.raises(AttentionError, match="weight is"):
        QkNorm(rope(), torch.ones(8, dtype=BF16))
    with pytest.raises(AttentionError, match="weight is"):
        QkNorm(rope(), torch.ones(1, 8))
    with pytest.raises(AttentionError, match="one dtype for both"):
        QkNorm(rope(dtype=BF16), torch.ones(8), torch.ones(8, dtype=BF16))
    for eps in (-1.0, float("inf"), float("nan")):
        with pytest.raises(AttentionError, match="eps"):
            QkNorm(rope(), eps=eps)
    norm = QkNorm(rope(), torch.ones(8), torch.ones(8))
    q, k = torch.zeros((2, 3, 4, 8)), torch.zeros((2, 3, 1, 8))
    for call in (lambda: norm.apply_range(q, k, range(0, 4)), lambda: norm.apply_range(q, k, range(14, 17)), lambda: norm.apply_range(q, k, range(-1, 2)),
                 lambda: norm.apply_range(q[0], k[0], range(0, 3)), lambda: norm.apply_range(q, k, range(0, 6, 2)), lambda: norm.apply_range(q, k[:1], range(0, 3)),
                 lambda: norm.apply_at(q, k, torch.zeros(2, dtype=torch.int32)), lambda: norm.apply_at(q[0], k[0], torch.zeros(2, dtype=torch.int32)),
                 lambda: norm.apply_at(q[0], k[0], torch.zeros(3)), lambda: norm.apply_at(q[0], k[0, :2], torch.zeros(3, dtype=torch.int64)),
                 lambda: norm.apply_packed(q, k, torch.zeros(2, dtype=torch.int32)), lambda: norm.apply_packed(q[0], k[0], torch.zeros((1, 2), dtype=torch.int32)),
                 lambda: norm.apply_packed(q[0], k[0], torch.zeros(2)), lambda: norm.apply_packed(q[0], k[0, :2], torch.zeros(2, dtype=torch.int32)),
                 lambda: norm.apply_range(q.to(BF16), k, range(0, 3)), lambda: norm.apply_range(q[..., :6], k[..., :6], range(0, 3)),
                 lambda: norm.apply_range(torch.zeros((2, 3, 4, 10)), torch.zeros((2, 3, 1, 10)), range(0, 3)),
                 lambda: norm.apply_range(q, torch.zeros((2, 3, 1, 10)), range(0, 3)),
                 lambda: norm.backward_range(q, k, q[:1], k, range(0, 3)), lambda: norm.backward_range(q, k, q, k.to(BF16), range(0, 3))):
        with pytest.raises(AttentionError):
            call()
    with pytest.raises(Unsupported, match="CUDA"):
        norm.apply_range(q, k, range(0, 3))


def test_norm_refusals_of_the_c_abi():
    lib = _lib.lib()
    t = _lib.RopeTables(0, 8, 16, 1 << 20, 1 << 20)

    def rc(tables=t, **kw):
        p = _lib.QkNormParams(b=1, t=4, d=8, heads_q=2, heads_k=1, weight_dtype=0, eps=1e-6)
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.dash_rope_norm_apply(ctypes.byref(tables), ctypes.byref(p), *[None] * 6, None)

    assert rc() == _lib.INVALID and "null" in _lib.last_error()
    for kw in (dict(b=-1), dict(t=-1), dict(heads_q=-1), dict(weight_dtype=1), dict(eps=-1.0), dict(start=13), dict(start=-1), dict(d=6),
               dict(positions=8, positions_elem_bytes=2), dict(cu_seqlens=8, cu_seqlens_len=2, index_elem_bytes=3), dict(cu_seqlens=8, cu_seqlens_len=0, index_elem_bytes=4),
               dict(cu_seqlens=8, cu_seqlens_len=2, index_elem_bytes=4, b=2)):
        assert rc(**kw) == _lib.INVALID, kw
    assert rc(d=258) == _lib.UNSUPPORTED
    assert rc(t=0) == _lib.OK and rc(heads_q=0, heads_k=0) == _lib.OK
    p = _lib.QkNormParams(b=1, t=4, d=8, heads_q=2, heads_k=1, weight_dtype=0, eps=1e-6)
    need = lib.dash_rope_norm_backward_workspace(ctypes.byref(p))
    assert need > 0
    args = [ctypes.c_void_p(1 << 20)] * 11
    args[10] = None
    assert lib.dash_rope_norm_backward(ctypes.byref(t), ctypes.byref(p), *args, need, None) == _lib.WORKSPACE
    args[10] = ctypes.c_void_p((1 << 20) + 16)
    assert lib.dash_rope_norm_backward(ctypes.byref(t), ctypes.byref(p), *args, need, None) == _lib.WORKSPACE
    args[10] = ctypes.c_void_p(1 << 20)
    assert lib.dash_rope_norm_backward(ctypes.byref(t), ctypes.byref(p), *args, need - 1, None) == _lib.WORKSPACE
    assert lib.dash_rope_norm_apply(ctypes.byref(t), None, *[None] * 6, None) == _lib.INVALID
    assert lib.dash_rope_norm_apply(None, ctypes.byref(p), *[None] * 6, None) == _lib.INVALID


def shared(**kw):
    x = dict(q=torch.zeros((4, 4, 8)), pk=torch.zeros((2, 5, 2, 8)), pv=torch.zeros((2, 5, 2, 8)), k=torch.zeros((4, 3, 2, 8)), v=torch.zeros((4, 3, 2, 8)), lens=None, plens=None)
    x.update(kw)
    return attention_decode_shared(x["q"], x["pk"], x["pv"], x["k"], x["v"], x["lens"], x["plens"])


def test_shared_refusals():
    with pytest.raises(Unsupported, match="CUDA"):
        shared()
    for kw in (dict(q=torch.zeros((4, 8))), dict(pk=torch.zeros((2, 5, 8))), dict(pk=torch.zeros((2, 5, 2, 8), dtype=BF16)), dict(plens=torch.zeros((2, 1), dtype=torch.int32)),
               dict(plens=torch.zeros(2)), dict(lens=torch.zeros(4))):
        with pytest.raises(AttentionError):
            shared(**kw)
    with pytest.raises(AttentionError, match="lengths are needed"):
        attention_decode_shared_append(*[torch.zeros(1)] * 7, None)
    with pytest.raises(AttentionError, match="null"):
        attention_decode_shared_append(torch.zeros(1), None, *[torch.zeros(1)] * 5, torch.zeros(1))


def test_shared_refusals_of_the_c_abi():
    lib = _lib.lib()
    one = ctypes.c_void_p(1 << 20)

    def call(own=None, prompt=None, pointers=(one, one, one, None, None, one, one, one), ws=one, size=1 << 40):
        p = _lib.DecodeParams(dtype=1, b=4, s=3, hq=4, hkv=2, d=8, k_b=4, k_d=8, v_b=4, v_s=3, v_hkv=2, v_d=8)
        x = _lib.PrefixParams(n=2, p=5, hkv=2, d=8, v_n=2, v_p=5, v_hkv=2, v_d=8)
        for target, kw in ((p, own or {}), (x, prompt or {})):
            for k, v in kw.items():
                setattr(target, k, v)
        return lib.dash_attn_decode_shared(ctypes.byref(p), ctypes.byref(x), *pointers, ws, size, None)

    for prompt in (dict(n=3, v_n=3), dict(n=0, v_n=0), dict(n=-1, v_n=-1), dict(p=-1, v_p=-1), dict(v_p=4), dict(v_n=1), dict(hkv=4, v_hkv=4), dict(d=16, v_d=16),
                   dict(lengths=8, lengths_len=4, lengths_elem_bytes=4), dict(lengths=8, lengths_len=2, lengths_elem_bytes=2)):
        assert call(prompt=prompt) == _lib.INVALID, prompt
    assert call(own=dict(dtype=7)) == _lib.INVALID
    assert call(prompt=dict(p=1 << 30, v_p=1 << 30)) == _lib.UNSUPPORTED
    assert call(pointers=(one, one, one, one, one, one, one, one)) == _lib.INVALID and "lengths are needed" in _lib.last_error()
    lens = dict(lengths=8, lengths_len=4, lengths_elem_bytes=4)
    assert call(own=lens, pointers=(one, one, one, one, None, one, one, one)) == _lib.INVALID and "new row" in _lib.last_error()
    for i in (0, 1, 2, 5, 6, 7):
        pointers = [one, one, one, None, None, one, one, one]
        pointers[i] = None
        assert call(pointers=pointers) == _lib.INVALID and "null" in _lib.last_error()
    assert call(size=100) == _lib.WORKSPACE and call(ws=None) == _lib.WORKSPACE and call(ws=ctypes.c_void_p((1 << 20) + 8)) == _lib.WORKSPACE
    assert call(own=dict(b=0, k_b=0, v_b=0), prompt=dict(n=0, v_n=0)) == _lib.OK
    p = _lib.DecodeParams(dtype=1, b=4, s=3, hq=4, hkv=2, d=8, k_b=4, k_d=8, v_b=4, v_s=3, v_hkv=2, v_d=8)
    assert lib.dash_attn_decode_shared(ctypes.byref(p), None, *[one] * 8, one, 1 << 40, None) == _lib.INVALID
    assert lib.dash_attn_decode_shared_workspace(ctypes.byref(p), None) == 0


def test_rules_refusals():
    z = torch.zeros((2, 40))
    ids = torch.zeros((2, 3), dtype=torch.int32)
    for p in (Penalties(tokens=ids[0]), Penalties(tokens=ids[:1]), Penalties(tokens=ids.float()), Penalties(lengths=torch.zeros(2, dtype=torch.int32)),
              Penalties(tokens=ids, lengths=torch.zeros(3, dtype=torch.int32)), Penalties(tokens=ids, lengths=torch.zeros(2)),
              Penalties(tokens=ids, prompt_lengths=torch.zeros((2, 1), dtype=torch.int32)), Penalties(repetition=1.1), Penalties(frequency=0.1), Penalties(presence=0.1),
              Penalties(tokens=ids, repetition=torch.ones(3)), Penalties(tokens=ids, frequency=torch.ones(2, dtype=BF16)), Penalties(bias=torch.zeros(39)),
              Penalties(bias=torch.zeros(40, dtype=BF16)), Penalties(allowed=torch.zeros((2, 1), dtype=torch.int32)), Penalties(allowed=torch.zeros((2, 2), dtype=torch.int64))):
        with pytest.raises(AttentionError, match="penalize"):
            penalize(z, p)
    for bad in (z[0], z.double()):
        with pytest.raises(AttentionError, match="logits must be"):
            penalize(bad, Penalties())
    for out in (z[:1], z.to(BF16), torch.zeros((40, 2)).T, torch.zeros((1, 40)).expand(2, 40)):
        with pytest.raises(AttentionError, match="out"):
            penalize(z, Penalties(), out=out)
    with pytest.raises(Unsupported, match="CUDA"):
        penalize(z, Penalties())


def test_rules_refusals_of_the_c_abi():
    lib = _lib.lib()

    def rc(**kw):
        p = _lib.PenalizeParams(dtype=0, b=2, v=40, row_stride=40, out_stride=40, repetition_all=1.0)
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.dash_sample_penalize(ctypes.byref(p), None, None, None)

    assert rc() == _lib.INVALID and "null" in _lib.last_error()
    for kw in (dict(dtype=3), dict(b=-1), dict(v=-1), dict(ids_len=-1), dict(ids=8, ids_len=2, ids_elem_bytes=2),
               dict(ids=8, ids_len=2, ids_elem_bytes=4, lengths=8, lengths_elem_bytes=1), dict(ids=8, ids_len=2, ids_elem_bytes=4, prompt_lengths=8, prompt_lengths_elem_bytes=1),
               dict(repetition_all=0.0), dict(repetition_all=-1.0), dict(repetition_all=float("nan")), dict(frequency_all=float("inf")), dict(presence_all=float("nan")),
               dict(bias=8, bias_dtype=1)):
        assert rc(**kw) == _lib.INVALID, kw
    assert rc(v=(1 << 30) + 1) == _lib.UNSUPPORTED
    assert rc(b=0) == _lib.OK and rc(v=0) == _lib.OK
    assert lib.dash_sample_penalize(None, None, None, None) == _lib.INVALID
    p = _lib.PenalizeParams(dtype=0, b=2, v=40, row_stride=40, out_stride=39, repetition_all=1.0)
    assert lib.dash_sample_penalize(ctypes.byref(p), 1 << 20, 1 << 20, None) == _lib.INVALID and "overlap" in _lib.last_error()


def test_structs_are_the_headers(tmp_path):
    import pathlib
    import subprocess

    header = pathlib.Path(__file__).resolve().parent.parent / "include" / "dash_attn.h"
    names = {"dash_rope_norm_params": _lib.QkNormParams, "dash_attn_prefix_params": _lib.PrefixParams, "dash_sample_penalize_params": _lib.PenalizeParams}
    lines = [f'printf("%zu ", sizeof({c}));' + "".join(f'printf("%zu ", offsetof({c}, {f[0]}));' for f in s._fields_) for c, s in names.items()]
    source = tmp_path / "sizes.c"
    source.write_text(f'#include "{header}"\n#include <stddef.h>\n#include <stdio.h>\nint main(void){{{"".join(lines)} return 0;}}')
    subprocess.run(["gcc", str(source), "-o", str(tmp_path / "sizes")], check=True)
    got = list(map(int, subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()))
    assert got == [x for s in names.values() for x in (ctypes.sizeof(s), *(getattr(s, f[0]).offset for f in s._fields_))]


def test_rules_refuse_memory_they_would_read_after_writing_it():
    lib = _lib.lib()
    at = 1 << 20

    def rc(out, row=100, out_row=100, b=3, v=40):
        p = _lib.PenalizeParams(dtype=2, b=b, v=v, row_stride=row, out_stride=out_row, repetition_all=1.0)
        return lib.dash_sample_penalize(ctypes.byref(p), at, out, None)

    for out, kw in ((at + 2, {}), (at - 2, {}), (at + 2 * 100 + 2 * 39, {}), (at + 2 * 200 + 2 * 39, {}), (at - 2 * 200 - 2 * 39, {}), (at + 2 * 61, {}),
                    (at, dict(out_row=101)), (at, dict(row=0)), (at + 2 * 239, dict(out_row=50)), (at - 2 * 139, dict(out_row=50)),
                    (at + 2 * 39, dict(b=1)), (at - 2 * 39, dict(b=1))):
        assert rc(out, **kw) == _lib.INVALID and "not them" in _lib.last_error(), (out - at, kw)


def test_rules_want_the_tokens_for_a_tensor_of_penalties():
    z = torch.zeros((2, 40))
    for name in ("repetition", "frequency", "presence"):
        with pytest.raises(AttentionError, match="needs the tokens"):
            penalize(z, Penalties(**{name: torch.ones(2)}))
