"""The lookup's gradient to the bit: rows of small whole numbers, whose sums are exact in 32 bits in any order, so that a row
lost or counted twice shows however many there are."""

import pytest
import torch

from fsctep_amd import learn_ops as L

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def exact(rows, width, table, index, dtype=torch.float32, seed=0):
    """Values of -3 to 3: sums below 2^24 (fp32), rounded once to bfloat16, as the 64-bit sum is."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    dy = torch.randint(-3, 4, (rows, width), generator=g, device=DEV)
    t = torch.zeros(table, width, device=DEV, dtype=dtype, requires_grad=True)
    got, = torch.autograd.grad(L.embedding(t, index), t, dy.to(dtype))
    there = (index >= 0) & (index < table)
    want = torch.zeros(table, width, device=DEV, dtype=torch.int64).index_add_(0, index[there].long(), dy[there])
    assert int(want.abs().max()) < 2 ** 24 if rows else True
    off = (got != want.to(torch.float32).to(dtype)).sum(1)
    assert int(off.sum()) == 0, f"{rows} x {width} into {table}: rows {off.nonzero().flatten().tolist()[:10]}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,width,table", [(2048, 4096, 1600), (2048, 4096, 1601), (2048, 4099, 1600), (256, 4096, 8000), (70, 12288, 10000),
                                              (2048, 2048, 4096), (2048, 1024, 4096), (1000, 8195, 2048)])
def test_wide_rows_where_the_sort_takes_over(rows, width, table, dtype):
    g = torch.Generator(device=DEV).manual_seed(rows + width)
    exact(rows, width, table, torch.randint(0, table, (rows,), generator=g, device=DEV), dtype)
    exact(rows, width, table, torch.full((rows,), table - 1, device=DEV, dtype=torch.int32), dtype)
