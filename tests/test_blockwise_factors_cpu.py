"""When the exponent bytes beside a cast's factors still count: on hand-made tensors, without a GPU."""
import copy

import pytest
import torch

from float8_experimental_b200.float8_blockwise import Float8BlockTensor

E4 = torch.float8_e4m3fn


def cast_like(rows=256, cols=384):
    """A tensor as the square cast leaves it."""
    exps, exps_t = torch.zeros(4, dtype=torch.uint8), torch.ones(4, dtype=torch.uint8)
    t = Float8BlockTensor._of_cast(torch.zeros(rows, cols).to(E4), torch.ones(rows // 128, cols // 128), (128, 128),
                                   torch.bfloat16, exps, exps_t)
    return t, exps, exps_t


def test_bytes_of_the_matrix_and_its_transpose():
    t, exps, exps_t = cast_like()
    assert t._exponents() is exps and t._exponents(transposed=True) is exps_t
    u = t.t()
    assert u._exponents() is exps_t and u._exponents(transposed=True) is exps
    v = u.t()
    assert v._exponents() is exps and v.block == t.block and v.shape == t.shape
    c = copy.deepcopy(t)
    assert torch.equal(c._exponents(), exps) and c._exponents() is not exps


WRITES = {"assigned": lambda t: setattr(t, "scale_inv", t._scale * 2), "in place": lambda t: t.scale_inv.mul_(2),
          "data": lambda t: t.scale_inv.data.mul_(2), "foreign": lambda t: t.scale_inv.numpy().__imul__(2),
          "through a transpose": lambda t: t.t().scale_inv.data.mul_(2)}


@pytest.mark.parametrize("how", WRITES)
def test_factors_that_may_have_been_written_drop_the_bytes(how):
    t, _, _ = cast_like()
    WRITES[how](t)
    assert bool((t._scale == 2).all())
    assert t._exponents() is None and t._exponents(transposed=True) is None
    assert t.t()._exponents() is None


def test_transposes_made_before_see_a_write():
    t, _, _ = cast_like()
    before = t.t()
    t.scale_inv.data.mul_(2)
    assert bool((before._scale == 2).all()) and before._exponents() is None and before._exponents(transposed=True) is None


def test_an_assignment_leaves_the_transpose_its_factors():
    t, exps, _ = cast_like()
    before = t.t()
    t.scale_inv = torch.full((2, 3), 4.0)
    assert t._exponents() is None and float(t.scale_inv[0, 0]) == 4.0
    assert bool((before._scale == 1).all()) and before._exponents(transposed=True) is exps


def test_assigned_factors_are_checked():
    t, _, _ = cast_like()
    for bad in (torch.ones(3, 2), torch.ones(2, 3).half(), torch.ones(2, 3, device="meta")):
        with pytest.raises(ValueError, match="scale_inv"):
            t.scale_inv = bad
