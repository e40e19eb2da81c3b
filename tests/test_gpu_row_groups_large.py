"""Row-group calls on arrays of more than 2^31 elements: small whole numbers, whose sums are exact, so that every output is
known.  Row p of a large array holds p % 16 throughout; a wrong address shows as another number."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS, WIDTH = 528000, 4112  # 2.17e9 elements


def numbers(dev, rows=ROWS):
    return torch.arange(rows, device=dev) % 16


def large(dev, dtype=torch.bfloat16, width=WIDTH):
    return torch.empty(ROWS, width, dtype=dtype, device=dev).copy_(numbers(dev)[:, None])


def all_rows_are(x, want):
    """Every element of row i is want[i], a block of rows at a time."""
    want = want.to(x.dtype)[:, None]
    return all(bool((x[i:i + 66000] == want[i:i + 66000]).all()) for i in range(0, len(x), 66000))


def test_rows_there_and_back(mb, dev):
    choices, groups = 8, 100
    tokens = ROWS // choices
    ids = (torch.arange(tokens, device=dev)[:, None] * 7 + torch.arange(choices, device=dev) * 13) % groups
    plan = mb.group_rows(ids, groups)
    x = torch.empty(tokens, WIDTH, dtype=torch.int8, device=dev).copy_((numbers(dev, tokens))[:, None])
    xs = mb.gather_rows_(torch.zeros(ROWS, WIDTH, dtype=torch.int8, device=dev), x, plan)
    assert all_rows_are(xs, (plan.order.long() // choices) % 16)
    del x, xs
    ys, y = large(dev), torch.empty(tokens, WIDTH, dtype=torch.bfloat16, device=dev)
    mb.combine_rows_(y, ys, plan)
    value = (plan.inverse.long() % 16)
    assert all_rows_are(y, value.sum(1))
    w = torch.ones(tokens, choices, device=dev)
    y.copy_(numbers(dev, tokens)[:, None])
    d_ys, d_w = mb.combine_rows_grad_(torch.zeros_like(ys), torch.empty_like(w), y, ys, plan, w)
    assert all_rows_are(d_ys, (plan.order.long() // choices) % 16)
    assert torch.equal(d_w, (value * numbers(dev, tokens)[:, None] * WIDTH).float())
    mb.synchronize_status(dev)


def test_products_of_row_groups(mb, dev):
    offsets = torch.tensor([0, 1, 300001, 300001, ROWS], dtype=torch.int32, device=dev)
    group = torch.searchsorted(offsets.long(), torch.arange(ROWS, device=dev), right=True) - 1
    a = large(dev)
    b = torch.empty(4, 64, WIDTH, dtype=torch.bfloat16, device=dev).copy_(torch.arange(1, 5, device=dev)[:, None, None])
    d = mb.gemm_grouped_(torch.empty(ROWS, 64, device=dev), a, b, offsets)
    assert all_rows_are(d, numbers(dev) * (group + 1) * WIDTH)
    del d
    g = torch.ones(ROWS, 64, dtype=torch.bfloat16, device=dev)
    db = mb.gemm_grouped_grad_(torch.empty(4, 64, WIDTH, device=dev), g, a, offsets)
    sums = torch.zeros(4, dtype=torch.int64, device=dev).index_add_(0, group, numbers(dev))
    assert torch.equal(db, sums[:, None, None].float().expand(4, 64, WIDTH))
    # the large array as the output: the gradient of the rows
    mb.gemm_grouped_(a, g, b.transpose(1, 2), offsets, alpha=0.0625)
    assert all_rows_are(a, (group + 1) * 4)
    mb.synchronize_status(dev)


@pytest.mark.parametrize("requests", [ROWS, 50])
def test_adapters(mb, dev, requests):
    step = ROWS // requests
    which = (torch.arange(requests, device=dev) % 3 - 1).to(torch.int32)
    edge = None if step == 1 else (torch.arange(requests + 1, device=dev) * step).to(torch.int32)
    mine = which.long().repeat_interleave(step)
    scale = torch.tensor([1.0, 2.0], device=dev)
    factor = torch.where(mine >= 0, (mine + 1), 0)
    x = large(dev)
    a, b = torch.ones(2, 8, WIDTH, dtype=torch.bfloat16, device=dev), torch.ones(2, 16, 8, dtype=torch.bfloat16, device=dev)
    d = mb.gemm_lora_(torch.zeros(ROWS, 16, device=dev), x, a, b, which, edge, scale)
    assert all_rows_are(d, numbers(dev) * factor * 8 * WIDTH)
    del d
    small = torch.ones(ROWS, 8, dtype=torch.bfloat16, device=dev)
    a, b = torch.ones(2, 8, 8, dtype=torch.bfloat16, device=dev), torch.ones(2, WIDTH, 8, dtype=torch.bfloat16, device=dev)
    mb.gemm_lora_(x, small, a, b, which, edge, scale)
    assert all_rows_are(x, numbers(dev) + factor * 64)
    mb.synchronize_status(dev)
