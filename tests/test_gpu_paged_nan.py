"""Page selection of rows that hold many NaN or infinite scores, and the calls that lead to them."""
import math

import pytest
import torch

import paged
import paged_plain as plain
import popkv_cuda as pk

pytestmark = pytest.mark.gpu


def check(scores, lengths, kv_heads, budget):
    ln = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = pk.paged_select(scores.cuda(), ln, kv_heads=kv_heads, page_size=16, budget=budget)
    assert plain.list_columns(got, scores.shape[1]) == plain.select(scores, lengths, 16, budget)


def test_two_numbers_and_two_nan():
    row = torch.tensor([-0.4257649, -0.3772625, math.nan, math.nan, 0.0])
    for width in (5, 2000, 5000, 20000, 40000):  # every kernel form; the columns after the newest page are not looked at
        scores = torch.zeros(1, 1, width)
        scores[0, 0, :5] = row
        for budget in (1, 2, 3, 4, 5):
            check(scores, [5 * 16], 1, budget)


@pytest.mark.parametrize("nans", [2, 3, 7, 20, 60])
@pytest.mark.parametrize("width,q_heads,kv_heads", [(200, 8, 2), (1500, 4, 4), (5000, 3, 1), (20000, 2, 1), (40000, 2, 2)])
def test_rows_with_many_nan(nans, width, q_heads, kv_heads):
    g = torch.Generator().manual_seed(width + nans)
    lengths = [width * 16, width * 16 - 37, 16 * 70]
    scores = torch.randn(len(lengths), q_heads, width, generator=g) * 10.0 ** torch.randint(-20, 20, (3, q_heads, 1), generator=g)
    for b in range(len(lengths)):
        for h in range(q_heads):
            at = torch.randperm(min(width, lengths[b] // 16), generator=g)[:nans]
            scores[b, h, at] = math.nan
            scores[b, h, at[0] - 1] = math.inf
            scores[b, h, at[1] - 1] = -math.inf
    for budget in sorted({2, nans, nans + 1, nans + 2, 65}):
        check(scores, lengths, kv_heads, budget)


def test_nan_and_infinite_keys_lead_their_pages_into_the_selection():
    g = torch.Generator().manual_seed(5)
    P, n, D, H, QH = 16, 16 * 60, 64, 2, 6
    cache = paged.new_cache(61, H, D, bounds=True)
    k, v = (torch.randn(n, H, D, generator=g).bfloat16() for _ in range(2))
    for page, value in ((3, math.nan), (11, math.inf), (12, -math.inf), (30, math.nan), (31, math.nan), (40, math.inf)):
        k[page * P + 5, :, 7 + page % 3] = value
    q = torch.randn(1, QH, D, generator=g).bfloat16().cuda()
    table = torch.randperm(60, generator=g).to(torch.int32)[None].cuda()
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    pk.paged_write(cache, k.cuda(), v.cuda(), table, zero, row_offsets=torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    scores = pk.paged_score(q, cache, table, lengths)
    odd = ~torch.isfinite(scores[0])
    assert bool((odd == odd[0]).all()) and torch.nonzero(odd[0])[:, 0].tolist() == [3, 11, 12, 30, 31, 40]
    assert not bool((scores == -math.inf).any())  # NaN or +infinity: above every number
    for budget in (2, 4, 7, 8, 20):
        pages = pk.paged_select(scores, lengths, kv_heads=H, page_size=P, budget=budget)
        chosen = plain.list_columns(pages, QH)
        assert chosen == plain.select(scores, [n], P, budget) and all(59 in c for c in chosen[0])
        got = pk.paged_sparse_attention(q, cache, table, lengths, budget=budget)
        assert bool(torch.isnan(got).any(-1).all())  # every head attends a page whose keys are no numbers
