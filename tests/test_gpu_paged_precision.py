"""Paged attention where little weights or little query channels decide the answer."""
import math

import pytest
import torch

import paged
import paged_plain as plain
import popkv_cuda as pk

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def one_sequence(k, v, dtype, store):
    """k, v [n, D] as the one KV head of one sequence."""
    n, D = k.shape
    pages = -(-n // 16)
    cache = paged.new_cache(pages, 1, D, dtype=dtype, store=store)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32)[None].cuda()
    pk.paged_write(cache, k[:, None].to(dtype).cuda(), v[:, None].to(dtype).cuda(), table,
                   torch.zeros(1, dtype=torch.int32, device="cuda"),
                   row_offsets=torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    return cache, table, torch.tensor([n], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("store,dtype", [("same", HF), ("same", BF), ("int8", BF), ("int8", HF), ("fp8", BF), ("fp8", HF)])
@pytest.mark.parametrize("at", [0, 1777, 3999])
@pytest.mark.parametrize("above", [16, 22])
@pytest.mark.parametrize("alike", [False, True])
def test_a_sink_without_a_value(store, dtype, at, above, alike):
    """One token far above the others whose value is zero: the output is made of the little weights.

    Weights are held to 2^-16 of themselves (bf16 halves; fp16 halves 2^-22) or, where weights are fp16, to 2^-37 of the
    largest (16-bit caches; the half step of fp16 is 2^-25 and the largest weight at least 2^13), with 8-bit caches to
    2^-30 of the largest weight times value scale.  The sequences share their pages: enough of them that a warp sees a
    quarter of a sequence's tokens beside the sink.
    """
    n, D, B = 4000, 64, 640
    g = torch.Generator().manual_seed(above + at)
    k = torch.zeros(n, D) if alike else 0.3 * torch.randn(n, D, generator=g)
    v = 1000.0 * (1 + 0.1 * torch.randn(n, D, generator=g))
    k[at], v[at] = above / D, 0.0
    q = torch.ones(1, 2, D, dtype=dtype, device="cuda")
    cache, table, lengths = one_sequence(k, v, dtype, store)
    got, lse = pk.paged_attention(q.repeat(B, 1, 1), cache, table.repeat(B, 1), lengths.repeat(B), scale=1.0, with_lse=True)
    out, ref_lse, mass, spread = plain.attend(q, cache, table, lengths, scale=1.0)
    keys, values = (plain.pool_values(cache, w)[table[0].cpu().long()].flatten(0, 2)[:n] for w in ("key", "value"))
    p = torch.softmax(q[0].cpu().double() @ keys.T, -1)                # [heads, n]
    if store == "same":
        little = 2.0 ** -37 * p.amax(-1, keepdim=True) * values.abs().sum(0)
    else:
        scale = cache.value_scale[table[0].long()].flatten().cpu().double()[:n]
        codes = torch.where(scale[:, None] > 0, values / scale[:, None].clamp(min=1e-300), torch.zeros_like(values))
        little = 2.0 ** -30 * (p * scale).amax(-1, keepdim=True) * codes.abs().sum(0)
    delta = (D + 16) * 2.0 ** -24 * spread.double()
    tol = plain.UNIT[dtype] * 1.01 * out.abs() + (2.0 ** -16 + 2 * delta)[..., None] * mass + little[None] + 2.0 ** -25
    err = (got.cpu().double() - out).abs()
    assert bool((err <= tol).all()), (float((err / out.abs()).max()), float((tol / out.abs()).min()))
    assert float((tol / out.abs()).max()) < 0.06  # the bound says something
    assert bool(((lse.cpu().double() - ref_lse).abs() <= delta + 2.0 ** -20 * (1 + ref_lse.abs())).all())


@pytest.mark.parametrize("store", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,big,little", [(BF, 2.0 ** 20, 1.0), (BF, 2.0 ** -100, 2.0 ** -120), (BF, 2.0 ** 127, 2.0 ** 106),
                                              (HF, 2.0 ** 15, 2.0 ** -5)])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_a_query_channel_far_above_the_others(store, dtype, big, little, head_dim):
    """Over keys that are zero in that channel, the others decide: 8-bit caches keep them whole."""
    n = 300
    g = torch.Generator().manual_seed(head_dim)
    k = torch.randn(n, head_dim, generator=g)
    v = torch.randn(n, head_dim, generator=g)
    k[:, 5] = 0.0
    q = little * torch.randn(1, 3, head_dim, generator=g)
    q[..., 5] = big * torch.tensor([1.0, -1.0, 1.99])
    q = q.to(dtype).cuda()
    cache, table, lengths = one_sequence(k, v, dtype, store)
    scale = 2.0 * head_dim ** -0.5 / little  # logits of a few units
    if math.isinf(torch.tensor(scale).float().item()) or scale < 1e-37:
        pytest.skip("the scale itself has no 32-bit value")
    got, lse = pk.paged_attention(q, cache, table, lengths, scale=scale, with_lse=True)
    plain.check_attention(got, lse, plain.attend(q, cache, table, lengths, scale=scale), dtype)
