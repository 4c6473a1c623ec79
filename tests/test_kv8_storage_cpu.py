"""A Kv8Cache's tensors are known to the kernels by address: they can be written
into, not replaced.  (A cache is not constructed without a GPU; its attributes
are set as the constructor sets them.)"""
import importlib

import pytest
import torch

PKG = importlib.import_module("numerics-and-sparse-attn_b200")


@pytest.mark.parametrize("name", ["k_codes", "v_codes", "scales", "page_table", "k_ring", "v_ring", "lens"])
def test_storage_is_written_into_and_not_replaced(name):
    c = PKG.Kv8Cache.__new__(PKG.Kv8Cache)
    mine = torch.zeros(4)
    setattr(c, name, mine)
    with pytest.raises(AttributeError, match=name):
        setattr(c, name, mine.clone())
    with pytest.raises(AttributeError, match=name):
        setattr(c, name, None)
    getattr(c, name)[1] = 3
    getattr(c, name).copy_(getattr(c, name) + 1)
    exec(f"c.{name} += 1", {"c": c})  # in place: the same tensor
    assert getattr(c, name) is mine and mine.tolist() == [2, 5, 2, 2]
    c.anything = 1
    c.anything = 2
