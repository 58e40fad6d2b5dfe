"""Lengths past the block table, queries and outputs at any address, and the pages that a decoder's step attends."""
import pytest
import torch

import paged_plain as plain
import popkv
import popkv_cuda as pk
from decoder import PagedDecoder
from test_gpu_paged import make
from test_gpu_paged_decoder import ids, tiny_model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("store", ["same", "int8", "fp8"])
@pytest.mark.parametrize("page_size", [16, 48])
def test_lengths_past_the_table_attend_the_whole_table(store, page_size):
    """Every column of the longer sequence is mapped and written: lengths from there on mean the same."""
    full = 5 * page_size
    cache, q, table, _ = make([full, page_size, full], q_heads=6, kv_heads=2, head_dim=64, page_size=page_size, store=store, bounds=True,
                              seed=21)
    over = torch.tensor([2 ** 31 - 1, -5, full + 1], dtype=torch.int32, device="cuda")
    clamped = torch.tensor([full, 0, full], dtype=torch.int32, device="cuda")
    got, lse = pk.paged_attention(q, cache, table, over, with_lse=True)
    plain.check_attention(got, lse, plain.attend(q, cache, table, clamped), q.dtype)
    scores = pk.paged_score(q, cache, table, over)
    assert torch.equal(scores, pk.paged_score(q, cache, table, clamped))
    for budget in (1, 3, 5):
        pages = pk.paged_select(scores, over, kv_heads=2, page_size=page_size, budget=budget)
        chosen = plain.list_columns(pages, 6)
        assert chosen == plain.select(scores, clamped.tolist(), page_size, budget)
        got, lse = pk.paged_sparse_attention(q, cache, table, over, budget=budget, with_lse=True)
        plain.check_attention(got, lse, plain.attend(q, cache, table, clamped, chosen=chosen), q.dtype)


@pytest.mark.parametrize("store", ["same", "int8", "fp8"])
@pytest.mark.parametrize("q_heads", [4, 24])
def test_queries_and_outputs_at_any_address(store, q_heads):
    cache, q, table, lengths = make([200, 33], q_heads=q_heads, kv_heads=2, head_dim=80, store=store, bounds=True, seed=22)
    want = pk.paged_attention(q, cache, table, lengths), pk.paged_sparse_attention(q, cache, table, lengths, budget=3)
    scores = pk.paged_score(q, cache, table, lengths)
    for offset in (1, 2, 4, 7):
        moved = torch.empty(q.numel() + 8, dtype=q.dtype, device="cuda")[offset:offset + q.numel()].view(q.shape).copy_(q)
        out = torch.zeros(q.numel() + 8, dtype=q.dtype, device="cuda")
        at = out[offset:offset + q.numel()].view(q.shape)
        assert torch.equal(pk.paged_score(moved, cache, table, lengths), scores)
        pk.paged_attention(moved, cache, table, lengths, out=at)
        assert torch.equal(at, want[0])
        pk.paged_sparse_attention(moved, cache, table, lengths, budget=3, out=at)
        assert torch.equal(at, want[1])
        assert not bool(out[:offset].any()) and not bool(out[offset + q.numel():].any())


def as_list(chosen, group):
    """Columns per query head as the page list that the attention takes."""
    items = []
    for heads in chosen:
        for k in range(0, len(heads), group):
            columns = sorted(set().union(*heads[k:k + group]))
            items.append([(c, sum((c in h) << g for g, h in enumerate(heads[k:k + group]))) for c in columns])
    room = max(len(x) for x in items)
    pages, masks = (torch.zeros(len(chosen), len(items) // len(chosen), room, dtype=torch.int32) for _ in range(2))
    for i, x in enumerate(items):
        for j, (c, m) in enumerate(x):
            pages.view(-1, room)[i, j], masks.view(-1, room)[i, j] = c, m
    counts = torch.tensor([len(x) for x in items], dtype=torch.int32).view(len(chosen), -1)
    return pages.cuda(), masks.cuda(), counts.cuda()


@pytest.mark.parametrize("store", ["same", "int8"])
def test_quest_steps_attend_the_selected_pages(monkeypatch, store):
    """Prompts around page boundaries: every sparse layer of every step sees the new token's length, and each query head
    the budget's pages, the newest among them."""
    budget, page, prompts = 4, 16, [63, 64, 65, 5, 300]
    dec = PagedDecoder(tiny_model(), popkv.RetrievalConfig(budget=budget * page, full_layers=(0,)), batch=len(prompts), max_tokens=400,
                       page_size=page, store=store, method="quest")
    for b, n in enumerate(prompts):
        dec.prefill(b, ids(n, 40 + b))
    step, calls = [0], [0]
    sparse = pk.paged_sparse_attention

    def watched(q, cache, table, lengths, *, budget, workspace, out):
        want_lengths = [n + 1 + step[0] for n in prompts]
        assert lengths.tolist() == want_lengths
        got = sparse(q, cache, table, lengths, budget=budget, workspace=workspace, out=out)
        chosen = plain.select(pk.paged_score(q, cache, table, lengths), want_lengths, page, budget)
        for b, n in enumerate(want_lengths):
            columns = -(-n // page)
            assert all(len(c) == min(4, columns) and c[-1] == columns - 1 for c in chosen[b])
        assert torch.equal(got, pk.paged_attention(q, cache, table, lengths, pages=as_list(chosen, q.shape[1] // cache.kv_heads)))
        if store == "same":
            plain.check_attention(got, None, plain.attend(q, cache, table, lengths, chosen=chosen), q.dtype)
        calls[0] += 1
        return got

    monkeypatch.setattr(pk, "paged_sparse_attention", watched)
    for _ in range(3):
        dec.step()
        step[0] += 1
    assert calls[0] == 3 * 3  # three layers are sparse
