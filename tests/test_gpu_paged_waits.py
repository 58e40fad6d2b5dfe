"""Paged attention whose copies do not count as complete: the waits run out, the call ends, and says so."""
import ctypes
import time

import pytest
import torch

import _native
import popkv
import popkv_cuda as pk
from decoder import PagedDecoder
from test_gpu_paged import make
from test_gpu_paged_decoder import ids, tiny_model

pytestmark = pytest.mark.gpu


class lose_copies:
    """The barriers of block 0 expect an arrival that never comes; waits end after 20 ms."""

    def __enter__(self):
        self.set(0, 20_000_000)

    def __exit__(self, *_):
        self.set(-1, 0)

    def set(self, block, ns):
        _native.c_library().popkv_paged_attention_lose_copies(ctypes.c_int64(block), ctypes.c_uint64(ns))


@pytest.mark.parametrize("store,dtype,q_heads,kv_heads,head_dim,lengths", [
    ("same", torch.bfloat16, 4, 2, 64, [5000]),            # an item over many blocks
    ("int8", torch.bfloat16, 8, 2, 128, [5000, 300]),
    ("fp8", torch.float16, 24, 2, 64, [3000]),             # two groups of 8 heads
    ("same", torch.float16, 4, 2, 256, [2000]),
    ("same", torch.bfloat16, 8, 8, 64, [40] * 130),        # several short items in a block
    ("int8", torch.bfloat16, 32, 8, 64, [40, 0, 17, 200] * 40)])
@pytest.mark.parametrize("sparse", [False, True])
def test_a_lost_copy_ends_the_call_and_is_counted(store, dtype, q_heads, kv_heads, head_dim, lengths, sparse):
    cache, q, table, ln = make(lengths, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, store=store, bounds=True)
    ws = pk.new_paged_workspace(len(lengths), q_heads, kv_heads, head_dim, "cuda", pages=table.shape[1], budget=16)

    def call():
        if sparse:
            return pk.paged_sparse_attention(q, cache, table, ln, budget=16, with_lse=True, workspace=ws)
        return pk.paged_attention(q, cache, table, ln, with_lse=True, workspace=ws)

    want, want_lse = call()
    assert pk.paged_incomplete(ws) == 0
    torch.cuda.synchronize()
    began = time.perf_counter()
    with lose_copies():
        got, lse = call()
    torch.cuda.synchronize()
    assert time.perf_counter() - began < 3.0
    lost = pk.paged_incomplete(ws)
    assert 1 <= lost <= 4  # the block's four warps, once each
    assert not bool(ws[: pk.PAGED_TICKET_BYTES].view(torch.int32)[:-1].any())  # every ticket was taken
    missing = torch.isnan(got).all(-1)
    assert torch.equal(missing, torch.isnan(lse)) and torch.equal(missing, torch.isnan(got).any(-1))
    assert bool(missing[0, 0]) and int(missing.sum()) <= 8 * (q_heads // kv_heads)
    assert torch.equal(got[~missing], want[~missing]) and torch.equal(lse[~missing], want_lse[~missing])
    again, again_lse = call()
    assert torch.equal(again, want) and torch.equal(again_lse, want_lse) and pk.paged_incomplete(ws) == lost


def test_the_decoder_raises():
    dec = PagedDecoder(tiny_model(), popkv.RetrievalConfig(budget=64, full_layers=(0,)), batch=2, max_tokens=200)
    dec.prefill(0, ids(100, 1))
    dec.prefill(1, ids(30, 2))
    good = dec.generate(3)
    with lose_copies():
        with pytest.raises(RuntimeError, match="incomplete"):
            dec.generate(2)
    dec.prefill(0, ids(100, 1))
    dec.prefill(1, ids(30, 2))
    assert torch.equal(dec.generate(3), good)
