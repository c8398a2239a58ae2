"""What the node of the norm with rotation keeps for its backward: an index buffer or a table that is written again before it is refused."""
import pytest
import torch

from dashmag_b200 import autodiff
from dashmag_b200.qk_norm import QkNorm, QkNormGradients
from dashmag_b200.rope import Rope


class Recorded(QkNorm):
    """The node's calls without a device: the gradients are those of its outputs, and the call's place is kept."""
    places: list = []

    def forward_of(self, query, key, where):
        return query.clone(), key.clone()

    def backward_of(self, query, key, grad_query, grad_key, where):
        Recorded.places.append(where)
        return QkNormGradients(grad_query.clone(), grad_key.clone(), None, None)


@pytest.fixture(autouse=True)
def without_a_device(monkeypatch):
    monkeypatch.setattr(autodiff, "QkNorm", Recorded)
    Recorded.places = []


def inputs(*lead):
    return (torch.randn(*lead, heads, 8, requires_grad=True) for heads in (2, 1))


def norm():
    return Recorded(Rope.from_tables(torch.ones(16, 8), torch.zeros(16, 8)))


def test_an_index_written_again_is_refused():
    q, k = inputs(5)
    for call, index in ((autodiff.qk_norm_at, torch.arange(5)), (autodiff.qk_norm_packed, torch.tensor([0, 2, 5], dtype=torch.int32))):
        a, b = call(norm(), q, k, index)
        index.add_(1)
        with pytest.raises(RuntimeError, match="inplace"):
            (a.sum() + b.sum()).backward()
        assert not Recorded.places


@pytest.mark.parametrize("table", ["cos", "sin"])
def test_a_table_written_again_is_refused(table):
    n = norm()
    q, k = inputs(2, 3)
    a, b = autodiff.qk_norm_range(n, q, k, range(3, 6))
    getattr(n.rope, table).mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        (a.sum() + b.sum()).backward()
    assert not Recorded.places


def test_what_is_left_alone_is_used():
    q, k = inputs(5)
    at, cu = torch.arange(5), torch.tensor([0, 2, 5])
    for call, args, name, index in ((autodiff.qk_norm_at, (at,), "positions", at), (autodiff.qk_norm_packed, (cu, 4), "cu_seqlens", cu)):
        a, b = call(norm(), q, k, *args)
        (a.sum() + b.sum()).backward()
        assert torch.equal(Recorded.places[-1][name], index)
    assert Recorded.places[-1]["start"] == 4
    q, k = inputs(2, 3)
    a, b = autodiff.qk_norm_range(norm(), q, k, range(3, 6))
    (a.sum() + b.sum()).backward()
    assert Recorded.places[-1]["start"] == 3 and Recorded.places[-1]["stop"] == 6


def test_tensors_made_in_inference_mode():
    """Such a tensor has no version to look at: the node keeps a copy."""
    with torch.inference_mode():
        index = torch.arange(5)
        rope = Rope.from_tables(torch.ones(16, 8), torch.zeros(16, 8))
    q, k = inputs(5)
    a, b = autodiff.qk_norm_at(Recorded(rope), q, k, index)
    with torch.inference_mode():
        index.add_(1)
    (a.sum() + b.sum()).backward()
    assert torch.equal(Recorded.places[-1]["positions"], torch.arange(5))
