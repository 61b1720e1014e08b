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


# sizes that take each way: copies in LDS (up to 24 rows), the sort joined by token (few rows) and by share (many), with
# shares of 32 tokens and of more (above 262,144 tokens), 4 and 16 tokens a thread (above 1,048,576), with and without a scan
WAYS = [(40000, 2, 5000), (70001, 20, 300), (20000, 7, 12), (70001, 20, 24), (600, 64, 9), (4097, 331, 25), (4097, 40, 70000), (9000, 130, 257),
        (2049, 33, 3000), (300007, 5, 700), (300007, 4, 90000), (1100003, 4, 300), (1100003, 3, 66000), (70001, 12, 17000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,width,table", WAYS)
def test_one_token_for_all(rows, width, table, dtype):
    for token in (0, table // 2, table - 1):
        exact(rows, width, table, torch.full((rows,), token, device=DEV), dtype, seed=token)


@pytest.mark.parametrize("rows,width,table", WAYS)
def test_a_few_tokens_with_long_runs(rows, width, table):
    """In order and mixed, beside tokens of one row and tokens outside the table."""
    g = torch.Generator(device=DEV).manual_seed(rows + table)
    few = torch.tensor([0, 1, table // 3, table // 2, table - 1], device=DEV)
    pick = few[torch.randint(0, 5, (rows,), generator=g, device=DEV)]
    rest = torch.randint(-3, table + 3, (rows,), generator=g, device=DEV)
    index = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.01, rest, pick)
    exact(rows, width, table, index)
    exact(rows, width, table, torch.sort(index)[0].to(torch.int32))
    exact(rows, width, table, torch.full((rows,), -1, device=DEV))


@pytest.mark.parametrize("table,by", [(40, "token"), (5000, "share")])
@pytest.mark.parametrize("length", [1, 31, 32, 33, 63, 64, 65, 95, 96, 97, 255, 256, 257, 1000, 8191, 8192, 8193])
def test_runs_that_end_at_a_shares_border(length, table, by):
    """Runs of a length one behind the other, begun 0, 1 and 31 tokens into a share of 32, whatever order they come in."""
    for lead in (0, 1, 31):
        n = lead + length * (table - 1)
        n = max(2100, min(n, 40000))
        index = torch.full((n,), 0, device=DEV)
        index[lead:] = 1 + torch.arange(n - lead, device=DEV) // length
        index = index.clamp(max=table)                    # those behind the last row are outside
        exact(n, 5, table, index)
        exact(n, 36, table, index[torch.randperm(n, device=DEV)])
