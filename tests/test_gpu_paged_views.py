"""Rows that are views of one buffer: what shares no memory is taken, in place
and beside each other, and gives what rows of their own give."""

from __future__ import annotations

import pytest
import torch

from kiv_amd import HeadNorm, PagedBatch, PagedKVCache, Rotary, norm_rope, paged_append, paged_attention

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def parts(cuda):
    freq = (1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().to(cuda)
    return Rotary(freq), HeadNorm(torch.linspace(0.5, 1.5, 64, device=cuda))


@pytest.mark.parametrize("B,T,hq,hkv", [(1, 1, 4, 1), (1, 7, 4, 2), (3, 5, 1, 4), (2, 1, 8, 8), (2, 600, 4, 1)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_rope_in_place_of_one_buffer(cuda, dtype, B, T, hq, hkv):
    """q and k of a fused projection, each over itself; and into a slice of
    the same buffer beside them."""
    rotary, norm = parts(cuda)
    g = torch.Generator(device=cuda).manual_seed(T)
    pos = torch.arange(T, device=cuda) + 5
    fused = torch.randn(B, T, 2 * hq + hkv, 64, device=cuda, generator=g).to(dtype)
    q, k = fused[:, :, :hq].transpose(1, 2), fused[:, :, hq:hq + hkv].transpose(1, 2)
    want = norm_rope(q.contiguous(), k.contiguous(), pos, rotary, norm, norm)
    rest = fused[:, :, hq + hkv:].transpose(1, 2)
    got = norm_rope(q, k, pos, rotary, norm, norm, q_out=rest)
    assert got[0] is rest and torch.equal(rest, want[0]) and torch.equal(got[1], want[1])
    got = norm_rope(q, k, pos, rotary, norm, norm, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(rest, want[0])


@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("tokens_first", [False, True])
def test_pools_that_share_a_buffer(cuda, T, tokens_first):
    """K and V pages of two layers in one buffer, the queries in place of a
    fused projection; K rows of one head expanded to all."""
    rotary, norm = parts(cuda)
    g = torch.Generator(device=cuda).manual_seed(T)
    pages, ps, hkv, hq = 4, 8, 2, 4
    shape = (pages, 2, 2, ps, hkv, 64) if tokens_first else (pages, 2, 2, hkv, ps, 64)
    pool = torch.zeros(shape, dtype=BF16, device=cuda)
    view = (lambda t: t.transpose(1, 2)) if tokens_first else (lambda t: t)
    layers = [PagedKVCache.from_pages(view(pool[:, i, 0]), view(pool[:, i, 1])) for i in range(2)]
    own = [PagedKVCache(pages, ps, hkv, 64, BF16, cuda, tokens_first) for _ in range(2)]
    for c in own:
        c.k.zero_(), c.v.zero_()
    batch = PagedBatch(torch.tensor([[2, 0, 3]], dtype=torch.int32, device=cuda),
                       torch.tensor([T + 6], dtype=torch.int32, device=cuda),
                       torch.tensor([0, T], dtype=torch.int32, device=cuda))
    for a, b in zip(layers, own):
        qkv = torch.randn(T, hq + 2 * hkv, 64, device=cuda, generator=g).to(BF16)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        want = paged_append(b, batch, k.contiguous(), v.contiguous(), q.contiguous(), None, rotary, norm, norm)
        got = paged_append(a, batch, k, v, q, None, rotary, norm, norm, q_out=q)
        assert got is q and torch.equal(q, want)
        assert torch.equal(paged_attention(q, a, batch, 0.125), paged_attention(want, b, batch, 0.125))
        one = k[:, :1].expand(T, hkv, 64)
        paged_append(a, batch, one, one, None)
        paged_append(b, batch, one.contiguous(), one.contiguous(), None)
    for a, b in zip(layers, own):
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


def test_pages_from_another_pool(cuda):
    """Rows of one layer's pages appended to another's in the same buffer."""
    pool = torch.randn(3, 2, 2, 2, 8, 64, device=cuda).to(F16)
    src, dst = (PagedKVCache.from_pages(pool[:, i, 0], pool[:, i, 1]) for i in range(2))
    batch = PagedBatch(torch.tensor([[1]], dtype=torch.int32, device=cuda),
                       torch.tensor([8], dtype=torch.int32, device=cuda),
                       torch.tensor([0, 8], dtype=torch.int32, device=cuda))
    before = pool.clone()
    paged_append(dst, batch, src.k[2].transpose(0, 1), src.v[2].transpose(0, 1))
    before[1, 1] = before[2, 0]
    assert torch.equal(pool, before)
