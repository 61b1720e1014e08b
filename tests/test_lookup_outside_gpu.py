"""Lookups of tokens that have no row, and atoms without one in the expert readout, on the GPU."""

import math

import pytest
import torch

from fsctep_amd import learn_ops as L, train_ops as T
from fsctep_amd.experts import ExpertReadout

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("outside", [0.0, math.nan, -1.5, math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [3, 8, 331])
def test_what_stands_where_a_token_has_no_row(width, dtype, outside):
    g = torch.Generator(device=DEV).manual_seed(1)
    t = torch.randn(5, width, generator=g, device=DEV).to(dtype).requires_grad_(True)
    index = torch.tensor([4, -1, 5, 0, 2 ** 40, 2], device=DEV)
    there = [0, 3, 5]
    y = L.embedding(t, index, 2.0, outside)
    want = torch.full((6, width), outside, device=DEV, dtype=dtype)
    want[there] = 2 * t.detach()[index[there]]
    assert torch.equal(y.nan_to_num(7e9), want.nan_to_num(7e9))
    dt, = torch.autograd.grad(y, t, torch.ones_like(y))
    assert (dt[[4, 0, 2]] == 2).all() and (dt[[1, 3]] == 0).all()
    empty = L.embedding(t.detach()[:0], index, 1.0, outside)
    assert torch.equal(empty.nan_to_num(7e9), torch.full_like(want, outside).nan_to_num(7e9))


@pytest.mark.parametrize("differentiable", [False, True])
def test_an_atom_beyond_a_bound_that_was_believed_becomes_nan(differentiable):
    """As an atom without a row does where the numbers are looked at; the others keep their values to the bit."""
    torch.manual_seed(7)
    m = ExpertReadout(64, 32, 4, k=2, n_species=10).to(DEV)
    with torch.no_grad():
        m.layers[0].w_out.normal_(0, 0.1)
    x = torch.randn(40, 64, device=DEV)
    species = torch.randint(0, 10, (40,), device=DEV)
    species[[3, 20, 39]] = torch.tensor([10, -1, 2 ** 33], device=DEV)
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[[3, 20, 39]] = True
    believed, looked = (m(x, species, differentiable=differentiable, species_below=b) for b in (10, None))
    assert believed[bad].isnan().all() and torch.isfinite(believed[~bad]).all()
    assert torch.equal(believed[~bad], looked[~bad]) and looked[bad].isnan().all()
    ga, gb = (torch.autograd.grad(y[~bad].square().sum(), m.layers[0].gate)[0] for y in (believed, looked))
    assert torch.equal(ga, gb) and torch.isfinite(ga).all()
    if not differentiable:
        q = m.to_8_bits()(x, species, species_below=10)
        assert q[bad].isnan().all() and torch.isfinite(q[~bad]).all()


def test_a_table_of_any_shape():
    t = torch.randn(4, 3, 5, device=DEV)
    y = T.lookup(t, torch.tensor([1, 4, 3], device=DEV), outside=math.nan)
    assert torch.equal(y[[0, 2]], t[[1, 3]]) and y[1].isnan().all()
