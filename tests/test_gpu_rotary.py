"""norm_rope and paged_append against 64-bit references: types, head dims,
partial and interleaved rotations, position axes, far positions, strides,
ragged batches, pages that are not there, streams and graphs."""

from __future__ import annotations

import pytest
import torch

from kiv_amd import HeadNorm, PagedBatch, PagedKVCache, Rotary, norm_rope, paged_append
from tests.paged_ref import (check, make_table, positions_of, ref_angles, ref_norm, ref_rotate, rope_bound)

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def freqs(rot, base=1e4):
    return (base ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))).float()


def expect(x, weight, angle, dtype, eps=1e-6, norm=True, interleaved=False, scale=1.0, offset=0.0):
    """x [B, H, T, D] as its values; (reference, bound)."""
    y = ref_norm(x.double(), weight, eps, offset) if norm else x.double()
    y, mag = ref_rotate(y, angle, interleaved, scale)
    return y, rope_bound(y, mag, dtype)


CASES = [
    # dtype, B, Hq, Hkv, T, D, rot, norm, interleaved, axes
    (BF16, 1, 28, 4, 1, 128, 128, True, False, 0),
    (BF16, 2, 12, 2, 37, 128, 128, True, False, 0),
    (F16, 1, 32, 4, 5, 64, 32, False, True, 3),
    (F32, 2, 8, 8, 19, 128, 64, True, True, 0),
    (F32, 1, 3, 1, 7, 20, 8, True, False, 2),
    (BF16, 1, 32, 32, 11, 96, 96, True, False, 3),
    (F16, 3, 8, 1, 9, 256, 128, True, False, 0),
    (BF16, 1, 4, 2, 3, 512, 512, True, False, 0),
    (BF16, 1, 5, 5, 6, 80, 32, False, False, 0),
    (F16, 1, 1, 1, 2, 8, 0, True, False, 0),
    (F32, 1, 2, 1, 3, 512, 256, False, False, 4),
    (BF16, 1, 16, 4, 700, 128, 128, True, False, 0),  # many tokens: several row groups a wave
    (F32, 1, 9, 3, 900, 64, 64, True, True, 3),
]


@pytest.mark.parametrize("dtype,B,hq,hkv,T,D,rot,norm,inter,axes", CASES)
def test_norm_rope(cuda, dtype, B, hq, hkv, T, D, rot, norm, inter, axes):
    g = torch.Generator().manual_seed(hash((B, hq, T, D, rot)) % 1000)
    qkv = torch.randn(B, T, hq + 2 * hkv, D, generator=g).to(dtype)
    q, k = qkv[:, :, :hq].transpose(1, 2), qkv[:, :, hq:hq + hkv].transpose(1, 2)
    qw, kw = 1 + 0.2 * torch.randn(D, generator=g), 1 + 0.2 * torch.randn(D, generator=g)
    start = 1_000_003
    pos = start + torch.randint(0, 5000, (max(1, axes), B, T), generator=g)
    axis = torch.randint(0, axes, (rot // 2,), generator=g) if axes else None
    dev = qkv.to(cuda)
    dq, dk = dev[:, :, :hq].transpose(1, 2), dev[:, :, hq:hq + hkv].transpose(1, 2)
    rotary = Rotary(freqs(rot).to(cuda), inter, 1.25, None if axis is None else axis.to(cuda)) if rot else None
    dpos = (pos if axes else pos[0]).to(cuda) if rot else None
    qo, ko = norm_rope(dq, dk, dpos, rotary, HeadNorm(qw.to(cuda)) if norm else None,
                       HeadNorm(kw.to(cuda), offset=1.0) if norm else None)
    assert qo.shape == q.shape and ko.shape == k.shape and qo.dtype == dtype
    angle = ref_angles(pos if axes else pos[0], freqs(rot), axis)[:, None] if rot else torch.zeros(1, 1, 1, 0)
    for got, x, w, off in ((qo, q, qw, 0.0), (ko, k, kw, 1.0)):
        check(got, *expect(x, w, angle, dtype, norm=norm, interleaved=inter, scale=1.25, offset=off), f"{dtype} D={D}")


def test_norm_rope_in_place_strides_and_positions(cuda):
    """Outputs over the inputs, q alone, int32 and broadcast positions, head-
    major rows, rows off the 16-byte grid (copied), a norm without a weight."""
    g = torch.Generator().manual_seed(5)
    q = torch.randn(2, 6, 9, 64, generator=g).to(BF16)
    pos = torch.randint(0, 4000, (9,), generator=g)
    angle = ref_angles(pos, freqs(64))
    ref, bound = expect(q, None, angle, BF16)
    rotary, norm = Rotary(freqs(64).to(cuda)), HeadNorm()
    for p in (pos.to(cuda), pos.to(cuda, torch.int32), pos.to(cuda).expand(2, 9), pos.to(cuda)[None]):
        got, none = norm_rope(q.to(cuda), None, p, rotary, norm)
        assert none is None
        check(got, ref, bound)
    dq = q.to(cuda)
    got, _ = norm_rope(dq, None, pos.to(cuda), rotary, norm, q_out=dq)
    assert got is dq
    check(dq, ref, bound)
    off = torch.empty(q.numel() + 3, dtype=BF16, device=cuda)[3:].view(q.shape)
    off.copy_(q)
    assert off.data_ptr() % 16
    check(norm_rope(off, None, pos.to(cuda), rotary, norm)[0], ref, bound)
    wide = torch.zeros(2, 6, 9, 128, dtype=BF16, device=cuda)
    wide[..., ::2] = q.to(cuda)
    check(norm_rope(wide[..., ::2], None, pos.to(cuda), rotary, norm)[0], ref, bound)


def test_norm_rope_edges(cuda):
    """No tokens; all-zero and huge rows; negative positions; no norm and no
    rotation keep every bit, NaNs among them."""
    rotary = Rotary(freqs(64).to(cuda))
    q = torch.randn(1, 4, 0, 64, device=cuda)
    assert norm_rope(q, q, torch.zeros(0, dtype=torch.int64, device=cuda), rotary)[0].shape == q.shape
    z = torch.zeros(1, 2, 3, 64, dtype=F16, device=cuda)
    assert torch.equal(norm_rope(z, None, None, None, HeadNorm(eps=1e-6))[0], z)
    big = torch.full((1, 2, 3, 64), 60000.0, dtype=F16, device=cuda)
    assert torch.equal(norm_rope(big, None, None, None, HeadNorm())[0], torch.ones_like(big))
    x = torch.randn(1, 2, 5, 64)
    pos = torch.tensor([-7, -1, 0, 1, 7])
    check(norm_rope(x.to(cuda), None, pos.to(cuda), rotary)[0], *expect(x, None, ref_angles(pos, freqs(64)), F32,
                                                                        norm=False))
    bits = torch.randint(-2**15, 2**15, (1, 3, 4, 64), dtype=torch.int16).to(cuda)
    got, _ = norm_rope(bits.view(BF16), None, None, None)
    assert torch.equal(got.view(torch.int16), bits)


def test_norm_rope_refusals(cuda):
    q, k = torch.randn(1, 4, 3, 64, device=cuda), torch.randn(1, 2, 3, 64, device=cuda)
    pos = torch.arange(3, device=cuda)
    rotary = Rotary(freqs(64).to(cuda))
    bad = [
        (ValueError, lambda: norm_rope(q[0], None, pos, rotary)),
        (ValueError, lambda: norm_rope(q, k[:, :, :2], pos, rotary)),
        (ValueError, lambda: norm_rope(q, k.half(), pos, rotary)),
        (ValueError, lambda: norm_rope(q, None, None, rotary)),
        (ValueError, lambda: norm_rope(q, None, pos[:2], rotary)),
        (TypeError, lambda: norm_rope(q, None, pos.float(), rotary)),
        (ValueError, lambda: norm_rope(q, None, pos.cpu(), rotary)),
        (ValueError, lambda: norm_rope(q, None, pos, rotary, k_norm=HeadNorm())),
        (ValueError, lambda: norm_rope(q, None, pos, rotary, HeadNorm(torch.ones(32, device=cuda)))),
        (ValueError, lambda: norm_rope(q, None, pos, rotary, q_out=k)),
        (ValueError, lambda: norm_rope(q, None, pos, Rotary(freqs(64).to(cuda), axes=torch.zeros(32, device=cuda,
                                                                                                 dtype=torch.int32)))),
        (RuntimeError, lambda: norm_rope(q, None, pos, Rotary(freqs(128).to(cuda)))),  # wider than the head
        (RuntimeError, lambda: norm_rope(q, None, pos, Rotary(freqs(12).to(cuda)))),   # off the chunks
        (RuntimeError, lambda: norm_rope(torch.randn(1, 1, 3, 516, device=cuda), None, pos, rotary)),
        (RuntimeError, lambda: norm_rope(q.requires_grad_(), None, pos, rotary)),
        (TypeError, lambda: norm_rope(torch.zeros(1, 1, 3, 64, dtype=torch.float64, device=cuda), None, pos, rotary)),
        (TypeError, lambda: Rotary(freqs(64).double().to(cuda))),
        (ValueError, lambda: HeadNorm(torch.ones(2, 2, device=cuda))),
    ]
    for err, f in bad:
        with pytest.raises(err):
            f()
    with torch.no_grad():
        norm_rope(q, None, pos, rotary)


def ragged(g, dtype, qlens, lens, hq, hkv, D, page, tokens_first, cuda, tail=0, pages_extra=3, fill=7.0):
    """A filled pool (every row `fill`), a batch and new rows with `tail`
    rows behind the last sequence."""
    cu = [0]
    for n in qlens:
        cu.append(cu[-1] + n)
    pages = sum(-(-n // page) for n in lens) + pages_extra
    table = make_table(lens, page, pages, g, extra=1)
    cache = PagedKVCache(pages, page, hkv, D, dtype, cuda, tokens_first)
    cache.k.fill_(fill)
    cache.v.fill_(fill)
    batch = PagedBatch(table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                       torch.tensor(cu, dtype=torch.int32, device=cuda))
    qkv = torch.randn(cu[-1] + tail, hq + 2 * hkv, D, generator=g).to(dtype)
    return cache, batch, table, cu, qkv


APPENDS = [
    # dtype, new tokens, lengths, Hq, Hkv, D, page, tokens_first, queries, rot, axes
    (BF16, [1, 1, 1], [1, 300, 129], 28, 4, 128, 128, False, True, 128, 0),
    (F16, [0, 7, 33, 1, 0], [5, 7, 100, 16, 0], 8, 8, 96, 16, True, False, 96, 0),
    (F32, [5, 64], [64, 65], 4, 2, 64, 48, False, True, 32, 3),
    (BF16, [3], [3], 2, 1, 256, 1, True, True, 256, 0),
    (BF16, [1] * 130, list(range(1, 131)), 4, 1, 64, 16, False, True, 64, 0),
    (F16, [600], [1234], 14, 2, 64, 64, False, True, 64, 0),
    (F32, [257, 3], [257, 900], 16, 4, 128, 32, True, True, 0, 0),
]


@pytest.mark.parametrize("dtype,qlens,lens,hq,hkv,D,page,tokens_first,queries,rot,axes", APPENDS)
def test_paged_append(cuda, dtype, qlens, lens, hq, hkv, D, page, tokens_first, queries, rot, axes):
    g = torch.Generator().manual_seed(len(lens) * 31 + D)
    tail = 4
    cache, batch, table, cu, qkv = ragged(g, dtype, qlens, lens, hq, hkv, D, page, tokens_first, cuda, tail)
    dev = qkv.to(cuda)
    total = cu[-1]
    kw, qw = 1 + 0.2 * torch.randn(D, generator=g), 1 + 0.2 * torch.randn(D, generator=g)
    seq, key = positions_of(cu, lens)
    axis = torch.randint(0, axes, (rot // 2,), generator=g) if axes else None
    pos = torch.randint(0, 9000, (axes, total + tail), generator=g) if axes else None
    rotary = Rotary(freqs(rot).to(cuda), axes=None if axis is None else axis.to(cuda)) if rot else None
    q_out = torch.full((total + tail, hq, D), 3.0, dtype=dtype, device=cuda) if queries else None
    got = paged_append(cache, batch, dev[:, hq:hq + hkv], dev[:, hq + hkv:], dev[:, :hq] if queries else None,
                       None if pos is None else pos.to(cuda), rotary, HeadNorm(qw.to(cuda)) if queries else None,
                       HeadNorm(kw.to(cuda)), q_out=q_out)
    assert got is q_out
    at = torch.tensor(key) if pos is None else pos[:, :total]
    angle = ref_angles(at, freqs(rot), axis)[:, None] if rot else torch.zeros(1, 1, 0)
    k, kb = expect(qkv[:total, hq:hq + hkv], kw, angle, dtype)
    want_k = torch.full(cache.k.shape, 7.0, dtype=torch.float64)
    bound_k, want_v = torch.zeros_like(want_k), want_k.clone()
    for r in range(total):
        page_id, slot = int(table[seq[r], key[r] // page]), key[r] % page
        want_k[page_id, :, slot], bound_k[page_id, :, slot] = k[r], kb[r]
        want_v[page_id, :, slot] = qkv[r, hq + hkv:].double()
    check(cache.k, want_k, bound_k, "K pages")
    assert torch.equal(cache.v.cpu().double(), want_v)
    if queries:
        check(q_out[:total], *expect(qkv[:total, :hq], qw, angle, dtype), "q")
        assert (q_out[total:] == 3.0).all()  # rows behind the last sequence


def test_append_pages_that_are_not_there(cuda):
    """Entries outside the pool, lengths past the table, negative key
    indexes, a shrinking cu_q: such rows are dropped, the others written,
    and nothing else changes."""
    g = torch.Generator().manual_seed(9)
    cache, batch, table, cu, qkv = ragged(g, BF16, [4, 4, 4, 4], [20, 20, 20, 20], 2, 1, 64, 8, False, cuda)
    total = cu[-1]
    table[1, 2] = 10_000        # its 4 new tokens' page
    table[2, 2] = -5
    batch.block_table.copy_(table)
    lens = batch.kv_len
    lens[3] = 2                 # rows 0, 1 would be keys -2, -1
    dev = qkv.to(cuda)
    before = cache.k.clone()
    q = paged_append(cache, batch, dev[:, 2:3], dev[:, 3:], dev[:, :2])
    assert torch.equal(q[:total], dev[:total, :2])
    want = before
    for r in range(4):
        want[int(table[0, 2]), :, r] = dev[r, 2:3]
    for r in (14, 15):
        want[int(table[3, 0]), :, r - 14] = dev[r, 2:3]
    assert torch.equal(cache.k, want)
    lens.fill_(2**31 - 1)       # past every table
    batch.cu_q.copy_(torch.tensor([0, 9, 3, 12, 16], dtype=torch.int32))
    paged_append(cache, batch, dev[:, 2:3], dev[:, 3:], dev[:, :2])
    assert torch.equal(cache.k, want)


def test_append_norms_v_and_tokens_to_one_page_table(cuda):
    """v_norm without a weight; no rotation copies K bit for bit."""
    g = torch.Generator().manual_seed(11)
    cache, batch, table, cu, qkv = ragged(g, F16, [5], [5], 1, 2, 64, 8, True, cuda)
    dev = qkv.to(cuda)
    paged_append(cache, batch, dev[:, 1:3], dev[:, 3:], v_norm=HeadNorm(eps=1e-5))
    page = int(table[0, 0])
    assert torch.equal(cache.k[page, :, :5], dev[:, 1:3].transpose(0, 1))
    ref = ref_norm(qkv[:, 3:].double(), None, 1e-5).transpose(0, 1)
    check(cache.v[page, :, :5], ref, rope_bound(ref, ref.abs(), F16))


def test_append_captured_and_on_a_side_stream(cuda):
    """One captured append, replayed for growing lengths, with eager appends
    to another pool between, equals eager ones; also on a side stream."""
    g = torch.Generator().manual_seed(13)
    cache, batch, table, cu, qkv = ragged(g, BF16, [1, 1], [40, 24], 4, 2, 64, 16, False, cuda)
    other = PagedKVCache(cache.num_pages, 16, 2, 64, BF16, cuda)
    other.k.fill_(7.0)
    other.v.fill_(7.0)
    rotary, norm = Rotary(freqs(64).to(cuda)), HeadNorm(torch.ones(64, device=cuda))
    rows = qkv.to(cuda)
    start = torch.tensor([3, 5], dtype=torch.int32, device=cuda)
    batch.kv_len.copy_(start)

    def step(c):
        return paged_append(c, batch, rows[:, 4:6], rows[:, 6:], rows[:, :4], None, rotary, norm, norm)

    step(cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q_graph = step(cache)
    side = torch.cuda.Stream()
    for n in range(4):
        rows.copy_(torch.randn(qkv.shape, generator=g).to(BF16))
        batch.kv_len.copy_(start + n)
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            q = step(other)
        side.synchronize()
        assert torch.equal(q, q_graph)
    assert torch.equal(cache.k[:, :, :], other.k) and torch.equal(cache.v, other.v)


def test_paged_refusals(cuda):
    cache = PagedKVCache(4, 8, 2, 64, BF16, cuda)
    table = torch.zeros(2, 3, dtype=torch.int32, device=cuda)
    lens = torch.ones(2, dtype=torch.int32, device=cuda)
    batch = PagedBatch(table, lens)
    k = torch.zeros(2, 2, 64, dtype=BF16, device=cuda)
    bad = [
        (ValueError, lambda: PagedKVCache(0, 8, 2, 64)),
        (TypeError, lambda: PagedKVCache(1, 8, 2, 64, torch.float64)),
        (ValueError, lambda: PagedKVCache.from_pages(cache.k, cache.v[:2])),
        (ValueError, lambda: PagedKVCache.from_pages(cache.k, cache.v.transpose(1, 2).contiguous().transpose(1, 2))),
        (ValueError, lambda: PagedKVCache.from_pages(cache.k.cpu(), cache.v.cpu())),
        (ValueError, lambda: PagedBatch(table, lens[:1])),
        (TypeError, lambda: PagedBatch(table.long(), lens)),
        (TypeError, lambda: PagedBatch(table, lens.long())),
        (ValueError, lambda: PagedBatch(table, lens.cpu())),
        (ValueError, lambda: PagedBatch(table, lens, lens)),
        (ValueError, lambda: PagedBatch(table, lens, max_q_len=-1)),
        (ValueError, lambda: paged_append(cache, batch, k, k[:1])),
        (ValueError, lambda: paged_append(cache, batch, k[:, :1], k)),
        (TypeError, lambda: paged_append(cache, batch, k.half(), k.half())),
        (ValueError, lambda: paged_append(cache, batch, k, k, q_norm=HeadNorm())),
        (ValueError, lambda: paged_append(cache, batch, k, k, positions=lens)),
        (ValueError, lambda: paged_append(cache, batch, k, k, q=k[:1])),
        (RuntimeError, lambda: paged_append(cache, batch, k.float().requires_grad_().to(BF16), k)),
    ]
    for err, f in bad:
        with pytest.raises(err):
            f()
    paged_append(cache, batch, k, k)
    none = PagedBatch(table[:0], lens[:0])
    assert paged_append(cache, none, k[:0], k[:0]) is None


@pytest.mark.parametrize("dtype,D", [(BF16, 96), (F16, 40), (F32, 20), (BF16, 128), (F16, 8)])
@pytest.mark.parametrize("at", [0, 7])
def test_an_infinity_hides_only_itself(cuda, dtype, D, at):
    """A row with an infinity has an infinite mean: its other entries become
    0, itself NaN, at widths whose lanes do not all hold a chunk too."""
    x = torch.randn(1, 2, 3, D, device=cuda).to(dtype)
    x[0, 1, 2, at] = float("inf")
    got, _ = norm_rope(x, None, None, None, HeadNorm())
    row = got[0, 1, 2]
    assert torch.isnan(row[at]) and (row[torch.arange(D, device=cuda) != at] == 0).all()
    assert torch.isfinite(got[0, 0]).all() and torch.isfinite(got[0, 1, :2]).all()


def test_axes_outside_32_bits_mean_the_nearest(cuda):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(1, 2, 4, 64, generator=g)
    pos = torch.randint(0, 500, (3, 4), generator=g)
    far = torch.tensor([2**32, 2**32 + 1, -2**40, 2**31, -1, 7, 0, 2] * 4)
    got, _ = norm_rope(x.to(cuda), None, pos.to(cuda), Rotary(freqs(64).to(cuda), axes=far.to(cuda)))
    check(got, *expect(x, None, ref_angles(pos, freqs(64), far.clamp(0, 2)), F32, norm=False))
