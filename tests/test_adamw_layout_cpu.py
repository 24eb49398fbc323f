"""What AdamW's tensor table depends on, from host tensors: a tensor that keeps its address can become another one."""
import pytest
import torch


def shorter(t):
    t.data = t.data[:5]


def resized(t):
    t.resize_(20)


def set_to_part(t):
    t.set_(t.untyped_storage(), 0, (3, 2), (2, 1))


def other_type(t):
    t.data = t.data.view(torch.bfloat16)[:, :6]


def twice_as_many(t):
    t.data = t.data.view(torch.bfloat16)


def transposed(t):
    t.data = t.data.t()


@pytest.mark.parametrize("change", [shorter, resized, set_to_part, other_type, twice_as_many, transposed])
@pytest.mark.parametrize("which", [0, 1])
def test_layout_tells_tensors_at_one_address_apart(change, which):
    from dnanet_amd.optim import _layout
    tensors = [torch.zeros(6, 6), torch.zeros(6, 6)]
    before, address = _layout(tensors), tensors[which].data_ptr()
    assert _layout(tensors) == before
    change(tensors[which])
    assert tensors[which].data_ptr() == address and _layout(tensors) != before


def test_layout_of_missing_and_foreign_entries():
    from dnanet_amd.optim import _layout
    a, b = torch.zeros(4), torch.zeros(4)
    assert len({_layout(x) for x in ([a, None], [None, a], [a], [a, b], [b, a], [None, None], [])}) == 7
    with pytest.raises(TypeError, match="tensor or None"):
        _layout([a, 3])
