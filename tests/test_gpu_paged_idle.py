"""PagedDecoder: sequences that were released or never started take no part in the steps."""
import pytest
import torch

import popkv
from decoder import PagedDecoder
from test_gpu_paged_decoder import ids, tiny_model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("method", ["full", "quest"])
@pytest.mark.parametrize("graphed", [False, True])
def test_idle_sequences_stay_empty(method, graphed):
    dec = PagedDecoder(tiny_model(), popkv.RetrievalConfig(budget=64, full_layers=(0,)), batch=4, max_tokens=200, method=method)
    dec.prefill(0, ids(30, 1))
    dec.prefill(2, ids(50, 2))  # 1 and 3 are never started
    dec.step()
    if graphed:
        dec.capture()
    for _ in range(3):
        dec.step()
    assert dec.starts.tolist() == [34, -1, 54, -1] and dec.lengths.tolist() == [35, 0, 55, 0]
    dec.release(2)
    tokens = dec.generate(40)
    assert tokens.shape == (40, 4)
    assert dec.starts.tolist() == [74, -1, -1, -1] and dec.lengths.tolist() == [75, 0, 0, 0]
    assert dec.host_lengths == [74, 0, 0, 0]
    dec.prefill(3, ids(9, 3))
    dec.step()
    assert dec.starts.tolist() == [75, -1, -1, 10] and dec.lengths.tolist() == [76, 0, 0, 11]


def test_idle_neighbours_do_not_change_a_sequence():
    model = tiny_model()
    out = []
    for others in (False, True):
        dec = PagedDecoder(model, popkv.RetrievalConfig(budget=64, full_layers=(0,)), batch=3, max_tokens=200, method="quest")
        dec.prefill(1, ids(90, 4))
        if others:
            dec.prefill(0, ids(20, 5))
            dec.prefill(2, ids(60, 6))
            dec.release(0)
            dec.release(2)
        out.append(dec.generate(20)[:, 1])
    assert torch.equal(out[0], out[1])
