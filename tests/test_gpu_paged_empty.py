"""Block tables without columns, page lists without room, batches without sequences."""
import math

import pytest
import torch

import paged
import popkv_cuda as pk

pytestmark = pytest.mark.gpu
B, QH, KVH, D = 3, 4, 2, 64


@pytest.fixture
def state():
    cache = paged.new_cache(4, KVH, D, bounds=True)
    q = torch.randn(B, QH, D, dtype=torch.bfloat16, device="cuda")
    return cache, q, torch.zeros(B, 0, dtype=torch.int32, device="cuda"), torch.tensor([0, 7, 100], dtype=torch.int32, device="cuda")


def nothing(out, lse):
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_tables_without_columns(state):
    cache, q, table, lengths = state
    nothing(*pk.paged_attention(q, cache, table, lengths, with_lse=True))
    scores = pk.paged_score(q, cache, table, lengths)
    assert scores.shape == (B, QH, 0)
    pages = pk.paged_select(scores, lengths, kv_heads=KVH, page_size=16, budget=3)
    assert pages[0].shape == (B, KVH, 0) and pages[2].tolist() == [[0, 0]] * B
    nothing(*pk.paged_attention(q, cache, table, lengths, pages=pages, with_lse=True))
    nothing(*pk.paged_sparse_attention(q, cache, table, lengths, budget=3, with_lse=True))
    rows = torch.randn(B, KVH, D, dtype=torch.bfloat16, device="cuda")
    before = cache.keys.clone()
    pk.paged_write(cache, rows, rows, table, lengths)
    assert torch.equal(cache.keys, before)
    k, v = pk.paged_read(cache, table, lengths, rows=B)
    assert not bool(k.any()) and not bool(v.any())


def test_page_lists_without_room(state):
    cache, q, _, lengths = state
    table = torch.zeros(B, 2, dtype=torch.int32, device="cuda")
    none = [torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((B, KVH, 0), (B, KVH, 0), (B, KVH))]
    none[2].fill_(9)  # more than there is room for
    nothing(*pk.paged_attention(q, cache, table, lengths, pages=none, with_lse=True))


def test_no_sequences(state):
    cache, q, _, lengths = state
    table = torch.zeros(0, 2, dtype=torch.int32, device="cuda")
    out, lse = pk.paged_attention(q[:0], cache, table, lengths[:0], with_lse=True)
    assert out.shape == (0, QH, D) and lse.shape == (0, QH)
    scores = pk.paged_score(q[:0], cache, table, lengths[:0])
    pages = pk.paged_select(scores, lengths[:0], kv_heads=KVH, page_size=16, budget=3)
    assert scores.shape == (0, QH, 2) and pages[2].shape == (0, KVH)
    assert pk.paged_sparse_attention(q[:0], cache, table, lengths[:0], budget=3).shape == (0, QH, D)
    rows = torch.zeros(0, KVH, D, dtype=torch.bfloat16, device="cuda")
    pk.paged_write(cache, rows, rows, table, lengths[:0])
