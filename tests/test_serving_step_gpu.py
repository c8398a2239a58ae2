"""The operators together, as a layer and a decoder use them: a training step's norm, rotation and attention under automatic
differentiation, and a decoding step of several answers to a prompt, from the projection to the token.

Bounds, u = 2^-24 and h the dtype's half step: where results of one operator feed the next, the next is checked on what it was given, under the
bounds of its own test; gradients in f32 through the chain against f64 under 1e-5 of the largest, the bound the CUDA-core attention is held to."""
import numpy as np
import pytest
import torch

from dashmag_b200 import attention as A
from dashmag_b200 import autodiff
from dashmag_b200.contract import AttentionMask, AttentionOptions
from dashmag_b200.penalties import Penalties, penalize
from dashmag_b200.prefix import attention_decode_shared_append
from dashmag_b200.qk_norm import QkNorm
from dashmag_b200.sample import SampleOptions, sample
from test_penalties_gpu import check as check_rules
from test_prefix_gpu import check as check_step
from test_qk_norm_gpu import check_forward, make, make_rope, turn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def layer(x, wq, wk, heads, norm, cu):
    """One layer's attention from a projection's output, tracked."""
    hq, hkv, d = heads
    q, k, v = (t.unflatten(-1, (h, d)) for t, h in zip(x.split([hq * d, hkv * d, hkv * d], -1), (hq, hkv, hkv)))
    q, k = autodiff.qk_norm_packed(QkNorm(norm.rope, wq, wk), q, k, cu)
    return autodiff.attention(q[None], k[None], v[None], AttentionMask.packed(cu, cu), AttentionOptions.causal_())[0]


def layer64(x, wq, wk, heads, rope, cu):
    hq, hkv, d = heads
    out = []
    for a, b in zip(cu[:-1], cu[1:]):
        y = x[a:b].double()
        q, k, v = (t.unflatten(-1, (h, d)) for t, h in zip(y.split([hq * d, hkv * d, hkv * d], -1), (hq, hkv, hkv)))
        pos = torch.arange(b - a)
        q, k = (turn(t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w.double(), rope, pos)[0] for t, w in ((q, wq), (k, wk)))
        k, v = (t.repeat_interleave(hq // hkv, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) * d ** -0.5
        s = s.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool, device=s.device).triu(1), -float("inf"))
        out.append(torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v))
    return torch.cat(out)


def test_a_training_step():
    heads, cu = (4, 2, 32), [0, 50, 51, 130]
    width = (heads[0] + 2 * heads[1]) * heads[2]
    x, wq, wk = make((130, width), torch.float32, 1), make((32,), torch.float32, 2, 0.3) + 1, make((32,), torch.float32, 3, 0.3) + 1
    g = make((130, heads[0], heads[2]), torch.float32, 4)
    rope = make_rope(32, 128, torch.float32)
    offsets = torch.tensor(cu, dtype=torch.int32, device=DEV)
    leaves = [t.clone().requires_grad_() for t in (x, wq, wk)]
    out = layer(*leaves, heads, QkNorm(rope), offsets)
    got = torch.autograd.grad((out * g).sum(), leaves)
    exact = [t.double().requires_grad_() for t in (x, wq, wk)]

    # (turn() writes into a copy: differentiable)
    want_out = layer64(*exact, heads, rope, cu)
    want = torch.autograd.grad((want_out * g.double()).sum(), exact)
    assert float((out.detach().double() - want_out).abs().max()) <= 1e-5 * max(1.0, float(want_out.abs().max()))
    for a, b in zip(got, want):
        assert a.shape == b.shape and float((a.double() - b).abs().max()) <= 1e-5 * max(1.0, float(b.abs().max()))


@pytest.mark.parametrize("need", [(True, False, False, False), (False, True, False, True), (False, False, True, False), (False, False, False, False)])
def test_only_what_is_tracked_gets_a_gradient(need):
    t = torch.bfloat16
    rope = make_rope(32, 64, t)
    q, k, wq, wk = (x.requires_grad_(n) for x, n in zip((make((20, 4, 32), t, 1), make((20, 2, 32), t, 2), make((32,), t, 3), make((32,), t, 4)), need))
    norm = QkNorm(rope, wq, wk)
    pos = torch.arange(20, device=DEV)
    oq, ok = autodiff.qk_norm_at(norm, q, k, pos)
    want = norm.apply_at(q.detach(), k.detach(), pos)
    assert torch.equal(oq, want[0]) and torch.equal(ok, want[1])
    assert oq.requires_grad == any(need)
    if not any(need):
        return
    (oq.float().sum() + (ok.float() * 2).sum()).backward()
    one = QkNorm(rope, wq.detach(), wk.detach()).backward_at(q.detach(), k.detach(), torch.ones_like(oq), 2 * torch.ones_like(ok), pos)
    for x, n, g in zip((q, k, wq, wk), need, one):
        assert torch.equal(x.grad, g) if n else x.grad is None


def test_forms_under_differentiation_and_a_captured_step():
    t = torch.bfloat16
    rope = make_rope(64, 64, t)
    norm = QkNorm(rope, make((64,), t, 1).requires_grad_(), make((64,), t, 2).requires_grad_())
    q, k = make((2, 16, 4, 64), t, 3), make((2, 16, 2, 64), t, 4)
    leaves = [norm.query_weight, norm.key_weight]

    def step():
        a, b = autodiff.qk_norm_range(norm, q, k, range(3, 19))
        c, d = autodiff.qk_norm_packed(norm, q[:1], k[:1], torch_cu)
        return torch.autograd.grad([a, b, c, d], leaves, [a.detach(), b.detach(), c.detach(), d.detach()])

    torch_cu = torch.tensor([0, 5, 16], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    q.copy_(make(q.shape, t, 9))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):   # the backward itself is not differentiable
        a, b = autodiff.qk_norm_range(norm, q, k, range(3, 19))
        once = torch.autograd.grad(a.float().square().sum(), leaves[0], create_graph=True)[0]
        torch.autograd.grad(once.float().sum(), leaves[0])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_decoding_several_answers_to_a_prompt(dtype):
    """Six steps of eight answers to two prompts: norm and rotation at each sequence's position, the new row appended and attended to behind
    the shared prompt, a projection to logits, the rules, a token."""
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    n, each, p, s, hq, hkv, d, v = 2, 4, 300, 8, 8, 2, 64, 1001
    b = n * each
    rope = make_rope(d, 512, t)
    norm = QkNorm(rope, make((d,), t, 1, 0.3) + 1, make((d,), t, 2, 0.3) + 1)
    prompt_lengths = torch.tensor([300, 171], dtype=torch.int32, device=DEV)
    x = dict(pk=make((n, p, hkv, d), t, 3), pv=make((n, p, hkv, d), t, 4), k=torch.zeros((b, s, hkv, d), dtype=t, device=DEV), v=torch.zeros((b, s, hkv, d), dtype=t, device=DEV))
    lens = torch.zeros(b, dtype=torch.int32, device=DEV)
    embed, project = make((v, (hq + 2 * hkv) * d), t, 5), make((hq * d, v), t, 6, 0.05)
    ids = torch.zeros((b, s + 1), dtype=torch.int64, device=DEV)
    ids[:, 0] = torch.arange(b, device=DEV) * 11
    allowed = torch.full((b, (v + 31) // 32), -1, dtype=torch.int32, device=DEV)
    allowed[:, 0] = 0   # no token under 32
    for step in range(6):
        qkv = embed[ids[:, step]]
        q, new_k, new_v = (y.unflatten(-1, (h, d)) for y, h in zip(qkv.split([hq * d, hkv * d, hkv * d], -1), (hq, hkv, hkv)))
        positions = prompt_lengths.repeat_interleave(each) + lens
        rq, rk = norm.apply_at(q, new_k, positions)
        check_forward(rq, q, norm.query_weight, rope, positions.cpu().long())
        check_forward(rk, new_k, norm.key_weight, rope, positions.cpu().long())
        out = attention_decode_shared_append(rq, rk, new_v, x["pk"], x["pv"], x["k"], x["v"], lens, prompt_lengths)
        assert torch.equal(x["k"][:, step], rk) and torch.equal(x["v"][:, step], new_v)
        lens += 1
        check_step(out, {**x, "q": rq}, prompt_lengths.tolist(), lens.tolist())
        logits = out.reshape(b, -1) @ project
        rules = Penalties(tokens=ids, lengths=lens, prompt_lengths=torch.ones_like(lens), repetition=1.2, frequency=0.4, presence=0.2, allowed=allowed)
        check_rules(penalize(logits, rules), logits, rules)
        drawn = sample(logits, SampleOptions(temperature=0.9, top_k=30, seed=7, offset=step), penalties=rules)
        assert int(drawn.tokens.min()) >= 32
        ids[:, step + 1] = drawn.tokens
    # the same answers over caches that hold prompt and answer together: the last step's output to the bound
    joined = [torch.cat([a.repeat_interleave(each, 0)[:, : 171], c], 1) for a, c in ((x["pk"], x["k"]), (x["pv"], x["v"]))]
    want = A.attention_decode(rq[each:], joined[0][each:], joined[1][each:], lens[each:] + 171)
    assert np.allclose(want.float().cpu(), out[each:].float().cpu(), rtol=0, atol=4 * torch.finfo(t).eps)
