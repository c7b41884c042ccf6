"""paged_attention against 64-bit attention: types, head shapes, lengths from
none to several shares, windows, pages that end inside a tile or are not
there, stale rows, 64-bit offsets, streams and graphs; and the operators
together as a serving loop runs them."""

from __future__ import annotations

import pytest
import torch

from kiv_amd import HeadNorm, PagedBatch, PagedKVCache, Rotary, norm_rope, paged_append, paged_attention
from tests.paged_ref import attention_bound, check, make_table, ref_attention

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def setup(g, dtype, qlens, lens, hq, hkv, D, page, tokens_first, cuda, tail=0, stale=float("nan"), max_q="exact"):
    """A pool whose rows past each sequence's length, and whose other pages,
    hold `stale`; the batch; packed queries with `tail` rows behind."""
    cu = [0]
    for n in qlens:
        cu.append(cu[-1] + n)
    pages = sum(-(-n // page) for n in lens) + 2
    table = make_table(lens, page, pages, g, extra=1)
    k, v = (torch.full((pages, hkv, page, D), stale, dtype=dtype) for _ in range(2))
    for b, n in enumerate(lens):
        for j in range(-(-n // page)):
            rows = min(page, n - j * page)
            k[int(table[b, j]), :, :rows] = torch.randn(hkv, rows, D, generator=g).to(dtype)
            v[int(table[b, j]), :, :rows] = torch.randn(hkv, rows, D, generator=g).to(dtype)
    dk, dv = k.to(cuda), v.to(cuda)
    if tokens_first:
        dk, dv = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (dk, dv))
    cache = PagedKVCache.from_pages(dk, dv)
    batch = PagedBatch(table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                       torch.tensor(cu, dtype=torch.int32, device=cuda),
                       max_q_len=max([0] + qlens) if max_q == "exact" else max_q,
                       max_kv_len=max([0] + lens) if max_q == "exact" else None)
    q = (1.5 * torch.randn(cu[-1] + tail, hq, D, generator=g)).to(dtype)
    return cache, batch, table, cu, q, k, v


def verify(got, q, k, v, table, lens, cu, scaling, window=0, what=""):
    n = cu[-1]
    ref, mag = ref_attention(q, k, v, table, lens, cu, scaling, window)
    bound = attention_bound(ref, mag, q, k, q.dtype, scaling, max([1] + list(lens)))
    check(got[:n], ref[:n], bound[:n], what)


CASES = [
    # dtype, new tokens, lengths, Hq, Hkv, D, page, tokens_first, window
    (F16, [1], [301], 32, 4, 64, 128, False, 0),
    (BF16, [1, 1, 1, 1], [1, 700, 129, 128], 28, 4, 128, 128, False, 0),
    (F32, [1, 0, 1], [300, 9, 33], 8, 2, 128, 16, True, 0),
    (BF16, [1, 1], [1000, 31], 8, 1, 256, 64, False, 0),
    (F16, [1, 1, 1], [5, 513, 64], 32, 32, 96, 16, True, 0),
    (BF16, [0, 0], [40, 0], 4, 4, 32, 8, False, 0),
    (BF16, [1, 0, 0, 1], [0, 0, 7, 1], 6, 2, 192, 3, False, 0),
    (F32, [1, 3], [77, 260], 20, 1, 256, 7, False, 0),
    (F32, [40], [40], 3, 3, 32, 1, True, 0),
    # chunks
    (BF16, [130], [130], 12, 2, 128, 128, False, 0),
    (BF16, [97, 1, 33], [300, 450, 33], 28, 4, 128, 16, True, 0),
    (F16, [64, 200], [64, 777], 14, 2, 64, 64, False, 0),
    (F16, [70], [200], 32, 32, 96, 32, False, 0),
    (BF16, [150], [400], 8, 1, 256, 48, False, 0),
    (F16, [90, 2], [90, 600], 9, 3, 192, 16, True, 0),
    (BF16, [65], [65], 2, 2, 32, 5, False, 0),
    (F32, [60, 5], [130, 300], 8, 4, 64, 24, False, 0),
    # more heads than a unit's rows
    (BF16, [1, 2], [200, 65], 40, 1, 64, 16, False, 0),
    (BF16, [3], [150], 200, 1, 32, 16, False, 0),
    (F32, [2], [90], 35, 1, 64, 16, False, 0),
    # windows: shorter than a tile, than a page, than the new tokens; longer than all
    (BF16, [1, 1], [900, 50], 16, 4, 128, 64, False, 100),
    (BF16, [300], [700], 8, 2, 64, 32, False, 65),
    (F16, [40, 1], [333, 1029], 8, 8, 128, 16, True, 7),
    (F32, [20, 1], [50, 400], 4, 2, 128, 16, False, 33),
    (BF16, [100], [257], 8, 1, 256, 64, False, 1),
    (BF16, [5, 1], [60, 70], 4, 4, 64, 16, False, 1 << 30),
]


@pytest.mark.parametrize("hint", ["exact", None], ids=["hint", "nohint"])
@pytest.mark.parametrize("dtype,qlens,lens,hq,hkv,D,page,tokens_first,window", CASES)
def test_paged_attention(cuda, dtype, qlens, lens, hq, hkv, D, page, tokens_first, window, hint):
    g = torch.Generator().manual_seed(D * 7 + sum(lens))
    tail = 3
    cache, batch, table, cu, q, k, v = setup(g, dtype, qlens, lens, hq, hkv, D, page, tokens_first, cuda, tail,
                                             max_q=hint)
    out = torch.full(q.shape, 5.0, dtype=dtype, device=cuda)
    got = paged_attention(q.to(cuda), cache, batch, D ** -0.5, window, out=out)
    assert got is out
    verify(out, q, k, v, table, lens, cu, D ** -0.5, window)
    assert (out[cu[-1]:] == 5.0).all()  # rows behind the last sequence


@pytest.mark.parametrize("dtype,lens,qlens", [
    (BF16, [9001], [1]),                                   # one sequence over many shares
    (F16, [5000, 1, 0, 333, 2600], [1, 1, 1, 1, 1]),       # shares across sequences
    (BF16, [1 + 13 * (i % 40) for i in range(300)], [(i % 7 > 0) * 1 for i in range(300)]),  # more than a scan's width
    (F32, [3000, 2000], [1, 2]),
    (BF16, [2100, 1900], [40, 1]),
    (F16, [1500], [700]),
])
def test_many_shares(cuda, dtype, lens, qlens):
    g = torch.Generator().manual_seed(len(lens))
    cache, batch, table, cu, q, k, v = setup(g, dtype, qlens, lens, 8, 2, 64, 32, False, cuda)
    verify(paged_attention(q.to(cuda), cache, batch, 0.125), q, k, v, table, lens, cu, 0.125)


def test_wrong_hints_cost_time_only(cuda):
    """Bounds below the true lengths, and far above them."""
    g = torch.Generator().manual_seed(3)
    for qlens, lens in (([1, 50], [3000, 700]), ([1, 1], [200, 2000])):
        cache, batch, table, cu, q, k, v = setup(g, BF16, qlens, lens, 14, 2, 64, 16, False, cuda)
        for max_q, max_kv in ((1, 1), (0, 0), (10**6, 10**9)):
            b = PagedBatch(batch.block_table, batch.kv_len, batch.cu_q, max_q_len=max_q, max_kv_len=max_kv)
            verify(paged_attention(q.to(cuda), cache, b, 0.125), q, k, v, table, lens, cu, 0.125)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("chunk", [1, 90])
def test_pages_that_are_not_there(cuda, dtype, chunk):
    """Missing pages inside a sequence are keys that no row sees; a sequence
    with none of its pages, or of negative length, gives zeros; a length past
    the table stops at the table."""
    g = torch.Generator().manual_seed(17)
    qlens, lens = [chunk] * 4, [300, 300, 300, 300]
    cache, batch, table, cu, q, k, v = setup(g, dtype, qlens, lens, 4, 2, 64, 16, False, cuda)
    table[0, 3], table[0, 7] = -1, 1 << 20
    table[1, :] = -1
    batch.block_table.copy_(table)
    lens = [300, 300, -4, 2**31 - 1]
    batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
    got = paged_attention(q.to(cuda), cache, batch, 0.2)
    assert (got[cu[1]:cu[3]] == 0).all()
    verify(got, q, k, v, table, [300, 300, 0], cu[:4], 0.2)
    # The last length is past the table, so its rows see the last page's
    # stale rows too: NaN, as the sum over those keys is.
    assert torch.isnan(got[cu[3]:]).all()


@pytest.mark.parametrize("chunk", [1, 90])
def test_length_past_the_table_stops_there(cuda, chunk):
    g = torch.Generator().manual_seed(18)
    cache, batch, table, cu, q, k, v = setup(g, BF16, [chunk], [300], 4, 2, 64, 16, False, cuda, stale=0.5)
    batch.kv_len.fill_(2**31 - 1)
    got = paged_attention(q.to(cuda), cache, batch, 0.2)
    ref, mag = ref_attention(q, k, v, table, [2**31 - 1], cu, 0.2)
    check(got, ref, attention_bound(ref, mag, q, k, BF16, 0.2, table.shape[1] * 16))


def test_lengths_in_disorder_touch_nothing_else(cuda):
    """cu_q that shrinks, starts before 0 or runs past the rows: whatever is
    written lies inside `out`, and rows it does not name keep their value."""
    g = torch.Generator().manual_seed(19)
    cache, batch, table, cu, q, k, v = setup(g, BF16, [4, 4, 4], [50, 60, 70], 4, 2, 64, 16, False, cuda)
    guard = torch.full((q.shape[0] + 64, 4, 64), 5.0, dtype=BF16, device=cuda)
    out = guard[32:32 + q.shape[0]]
    for bad in ([0, 8, 2, 6], [-9, 3, 3, 5], [0, 4, 8, 10_000], [9, 9, 9, 9], [12, 8, 4, 0]):
        guard.fill_(5.0)
        batch.cu_q.copy_(torch.tensor(bad, dtype=torch.int32))
        paged_attention(q.to(cuda), cache, batch, 0.125, out=out)
        assert (guard[:32] == 5.0).all() and (guard[32 + q.shape[0]:] == 5.0).all()
        named = set()
        for a, z in zip(bad[:-1], bad[1:]):
            named |= set(range(max(0, a), min(z, q.shape[0])))
        rest = [r for r in range(q.shape[0]) if r not in named]
        assert (out[rest] == 5.0).all()
        assert torch.isfinite(out).all()


def test_nan_and_infinity_in_keys_no_row_sees(cuda):
    """A later token's K may hold anything: earlier rows' scores for it are
    hidden before they count.  (Its V must be finite.)"""
    g = torch.Generator().manual_seed(23)
    cache, batch, table, cu, q, k, v = setup(g, BF16, [80], [200], 8, 2, 64, 16, False, cuda)
    for j, x in ((199, float("nan")), (198, float("inf"))):
        k[int(table[0, j // 16]), :, j % 16] = x
    cache.k.copy_(k)
    got = paged_attention(q.to(cuda), cache, batch, 0.125)
    clean = k.clone().nan_to_num(0.0, 0.0, 0.0)
    ref, mag = ref_attention(q, clean, v, table, [200], cu, 0.125)
    check(got[:78], ref[:78], attention_bound(ref, mag, q, clean, BF16, 0.125, 200)[:78])


def test_large_scores_and_one_key(cuda):
    """Scores of several hundred, equal scores, and rows with a single key
    (the output is that key's value, to its rounding)."""
    g = torch.Generator().manual_seed(29)
    cache, batch, table, cu, q, k, v = setup(g, F16, [1, 1], [1, 900], 8, 2, 64, 16, False, cuda)
    got = paged_attention(q.to(cuda), cache, batch, 4.0)
    first = v[int(table[0, 0]), :, 0]
    assert torch.equal(got[0].cpu(), first.repeat_interleave(4, 0))
    verify(got, q, k, v, table, [1, 900], cu, 4.0)
    z = torch.zeros_like(q)
    verify(paged_attention(z.to(cuda), cache, batch, 1.0), z, k, v, table, [1, 900], cu, 1.0)


def test_strided_queries_and_copies(cuda):
    g = torch.Generator().manual_seed(31)
    cache, batch, table, cu, q, k, v = setup(g, BF16, [3, 40], [30, 90], 8, 2, 64, 16, True, cuda)
    wide = torch.zeros(q.shape[0], 12, 64, dtype=BF16, device=cuda)
    wide[:, 2:10] = q.to(cuda)
    by_head = q.to(cuda).transpose(0, 1).contiguous().transpose(0, 1)
    off = torch.empty(q.numel() + 1, dtype=BF16, device=cuda)[1:].view(q.shape)
    off.copy_(q)
    want = paged_attention(q.to(cuda), cache, batch, 0.125)
    verify(want, q, k, v, table, [30, 90], cu, 0.125)
    for x in (wide[:, 2:10], by_head, off):
        assert torch.equal(paged_attention(x, cache, batch, 0.125), want)


def test_same_inputs_give_the_same_bits(cuda):
    g = torch.Generator().manual_seed(37)
    cache, batch, table, cu, q, k, v = setup(g, BF16, [1, 60, 1], [4000, 900, 70], 28, 4, 128, 16, False, cuda)
    dq = q.to(cuda)
    want = paged_attention(dq, cache, batch, 0.09)
    for _ in range(5):
        assert torch.equal(paged_attention(dq, cache, batch, 0.09), want)


def test_offsets_past_32_bits(cuda):
    """A pool of over 2^32 bytes and over 2^31 elements of each of K and V;
    the sequences' pages lie at its far end and its start."""
    pages, page, hkv, D = 34_000, 128, 4, 128
    assert pages * page * hkv * D > 2**31
    cache = PagedKVCache(pages, page, hkv, D, BF16, cuda)
    g = torch.Generator().manual_seed(41)
    ids = [pages - 1, 0, pages - 2, 33_000]
    lens, qlens = [300, 100], [1, 30]
    table = torch.full((2, 3), -1, dtype=torch.int32)
    table[0], table[1, 0] = torch.tensor(ids[:3]), ids[3]
    small_k, small_v = (torch.randn(4, hkv, page, D, generator=g).to(BF16) for _ in range(2))
    local = torch.full((2, 3), -1, dtype=torch.int32)
    local[0], local[1, 0] = torch.tensor([0, 1, 2]), 3
    batch = PagedBatch(table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                       torch.tensor([0, 1, 31], dtype=torch.int32, device=cuda))
    q = torch.randn(31, 8, D, generator=g).to(BF16)
    # The rows go there by paged_append: all of both sequences as new tokens.
    every = PagedBatch(batch.block_table, batch.kv_len, torch.tensor([0, 300, 400], dtype=torch.int32, device=cuda))
    def packed(x):
        return torch.cat([x[:3].transpose(1, 2).reshape(-1, hkv, D)[:300], x[3].transpose(0, 1)[:100]]).to(cuda)
    paged_append(cache, every, packed(small_k), packed(small_v))
    verify(paged_attention(q.to(cuda), cache, batch, 0.09), q, small_k, small_v, local, lens, [0, 1, 31], 0.09)


def test_two_captured_calls_and_eager_ones_between(cuda):
    """Two graphs over one cache, replayed in turn with eager calls on the
    same and on another stream between, while the lengths grow."""
    g = torch.Generator().manual_seed(43)
    cache, batch, table, cu, q, k, v = setup(g, BF16, [1, 1], [700, 2000], 28, 4, 128, 16, False, cuda, stale=0.0)
    chunk = PagedBatch(batch.block_table, batch.kv_len, torch.tensor([0, 40, 70], dtype=torch.int32, device=cuda))
    dq, cq = q.to(cuda), torch.randn(70, 28, 128, generator=g).to(BF16).to(cuda)
    paged_attention(dq, cache, batch, 0.09), paged_attention(cq, cache, chunk, 0.09)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x, b in ((dq, batch), (cq, chunk)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_attention(x, cache, b, 0.09))
        graphs.append(graph)
    side = torch.cuda.Stream()
    for lens in ([300, 64], [41, 1999], [700, 2000], [0, 30]):
        batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            here = paged_attention(cq, cache, chunk, 0.09)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], paged_attention(dq, cache, batch, 0.09))
        assert torch.equal(outs[1], here) and torch.equal(here, paged_attention(cq, cache, chunk, 0.09))


def test_serving_loop(cuda):
    """Two requests served as a loop would: a prompt in two chunks beside
    another's decode steps, then both decoding; norms and rotation on the
    way into the cache.  Every step's rows equal attention over the whole
    sequence, whose rows norm_rope makes at once."""
    g = torch.Generator().manual_seed(47)
    hq, hkv, D, page, dtype = 8, 2, 64, 16, BF16
    total = [90, 61]
    qkv = [torch.randn(n, hq + 2 * hkv, D, generator=g).to(dtype).to(cuda) for n in total]
    rotary = Rotary((1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().to(cuda))
    qn, kn = (HeadNorm(1 + 0.1 * torch.randn(D, generator=g).to(cuda)) for _ in range(2))
    cache = PagedKVCache(16, page, hkv, D, dtype, cuda, tokens_first=True)
    table = make_table(total, page, 16, g).to(cuda)
    lens, outs = [0, 0], [[], []]
    steps = [(30, 20), (40, 1), (17, 1)] + [(1, 1)] * 3 + [(0, 36)]
    for new in steps:
        rows = torch.cat([qkv[b][lens[b]:lens[b] + new[b]] for b in range(2)])
        lens = [lens[b] + new[b] for b in range(2)]
        batch = PagedBatch(table, torch.tensor(lens, dtype=torch.int32, device=cuda),
                           torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device=cuda), max_q_len=max(new))
        q = paged_append(cache, batch, rows[:, hq:hq + hkv], rows[:, hq + hkv:], rows[:, :hq], None, rotary, qn, kn)
        out = paged_attention(q, cache, batch, D ** -0.5)
        outs[0].append(out[:new[0]])
        outs[1].append(out[new[0]:])
    assert lens == total
    for b in range(2):
        x = qkv[b].transpose(0, 1)[None]
        pos = torch.arange(total[b], device=cuda)
        q, k = norm_rope(x[:, :hq], x[:, hq:hq + hkv], pos, rotary, qn, kn)
        q, k, v = q[0].transpose(0, 1).cpu(), k[0].cpu(), x[0, hq + hkv:].cpu()
        one = torch.zeros(1, 1, dtype=torch.int32)
        ref, mag = ref_attention(q, k[None], v[None], one, [total[b]], [0, total[b]], D ** -0.5)
        check(torch.cat(outs[b]), ref, attention_bound(ref, mag, q, k, dtype, D ** -0.5, total[b]), f"request {b}")


def test_paged_attention_refusals(cuda):
    g = torch.Generator().manual_seed(53)
    cache, batch, table, cu, q, k, v = setup(g, BF16, [2], [5], 4, 2, 64, 16, False, cuda)
    dq = q.to(cuda)
    bad = [
        (ValueError, lambda: paged_attention(dq[0], cache, batch, 1.0)),
        (ValueError, lambda: paged_attention(dq[..., :32], cache, batch, 1.0)),
        (TypeError, lambda: paged_attention(dq.half(), cache, batch, 1.0)),
        (ValueError, lambda: paged_attention(q, cache, batch, 1.0)),
        (ValueError, lambda: paged_attention(dq, cache, batch, 1.0, window=-1)),
        (ValueError, lambda: paged_attention(dq, cache, batch, 1.0, out=dq.float())),
        (ValueError, lambda: paged_attention(dq, cache, batch, 1.0, out=torch.zeros(2, 8, 64, dtype=BF16,
                                                                                     device=cuda)[:, ::2])),
        (RuntimeError, lambda: paged_attention(dq[:, :3], cache, batch, 1.0)),
        (RuntimeError, lambda: paged_attention(dq, cache, batch, 0.0)),
        (RuntimeError, lambda: paged_attention(dq, cache, batch, -1.0)),
        (RuntimeError, lambda: paged_attention(dq, cache, batch, float("nan"))),
        (RuntimeError, lambda: paged_attention(dq, cache, batch, float("inf"))),
        (RuntimeError, lambda: paged_attention(dq.clone().requires_grad_(), cache, batch, 1.0)),
    ]
    for err, f in bad:
        with pytest.raises(err):
            f()
    odd = PagedKVCache(2, 4, 1, 48, BF16, cuda)
    with pytest.raises(RuntimeError, match="head_dim 48"):
        paged_attention(torch.zeros(2, 2, 48, dtype=BF16, device=cuda), odd, batch, 1.0)
    empty = PagedBatch(batch.block_table[:0], batch.kv_len[:0])
    assert paged_attention(dq[:0], cache, empty, 1.0).shape == (0, 4, 64)
    assert paged_attention(dq[:0], cache, batch, 1.0).shape == (0, 4, 64)


def test_out_over_the_query(cuda):
    """Refused wherever they share memory; next to each other they may lie."""
    g = torch.Generator().manual_seed(73)
    cache, batch, table, cu, q, k, v = setup(g, BF16, [40, 1], [300, 77], 4, 2, 64, 16, False, cuda)
    both = torch.zeros(82, 4, 64, dtype=BF16, device=cuda)
    for at in (0, 1, 40):
        with pytest.raises(RuntimeError, match="overlap"):
            paged_attention(both[:41], cache, batch, 0.125, out=both[at:at + 41])
    with pytest.raises(RuntimeError, match="overlap"):
        paged_attention(both[40:81], cache, batch, 0.125, out=both[:41])
    for lo, hi in ((0, 41), (41, 0)):
        both[lo:lo + 41] = q.to(cuda)
        out = paged_attention(both[lo:lo + 41], cache, batch, 0.125, out=both[hi:hi + 41])
        assert out.data_ptr() == both[hi].data_ptr()
        verify(out, q, k, v, table, [300, 77], cu, 0.125)


def test_handles_keep_their_tensors(cuda):
    """The kernels read through addresses taken at construction: the tensors
    behind them cannot be swapped, and live as long as the handle."""
    g = torch.Generator().manual_seed(59)
    cache, batch, table, cu, q, k, v = setup(g, BF16, [1], [40], 4, 2, 64, 16, False, cuda)
    for obj, name in ((batch, "kv_len"), (batch, "cu_q"), (batch, "block_table"), (cache, "k"), (cache, "v"),
                      (HeadNorm(), "weight"), (Rotary(torch.ones(32, device=cuda)), "inv_freq")):
        with pytest.raises(AttributeError):
            setattr(obj, name, None)
    handle = PagedBatch(table.to(cuda), torch.tensor([40], dtype=torch.int32, device=cuda),
                        torch.tensor([0, 1], dtype=torch.int32, device=cuda))
    junk = [torch.full((n,), 7, dtype=torch.int32, device=cuda) for n in (1, 2, 4) * 20]
    verify(paged_attention(q.to(cuda), cache, handle, 0.125), q, k, v, table, [40], cu, 0.125)
    del junk


def test_many_shapes_in_turn(cuda):
    """Token counts that change from call to call: no shape's arguments serve
    another's."""
    g = torch.Generator().manual_seed(61)
    cache, batch, table, cu, q, k, v = setup(g, BF16, [37], [400], 8, 2, 64, 16, False, cuda)
    dq = q.to(cuda)
    for n in (1, 2, 3, 5, 8, 37, 2, 1):
        b = PagedBatch(batch.block_table, batch.kv_len, torch.tensor([0, n], dtype=torch.int32, device=cuda))
        verify(paged_attention(dq[37 - n:], cache, b, 0.125), q[37 - n:], k, v, table, [400], [0, n], 0.125)


@pytest.mark.parametrize("dtype,max_q", [(F32, 1), (BF16, 1), (BF16, None)])
def test_more_whole_units_than_blocks(cuda, dtype, max_q):
    """Over four thousand units of few keys: blocks take several each."""
    g = torch.Generator().manual_seed(67)
    lens = [1 + 7 * i % 40 for i in range(130)]
    cache, batch, table, cu, q, k, v = setup(g, dtype, [1] * 130, lens, 32, 32, 32, 16, False, cuda)
    b = PagedBatch(batch.block_table, batch.kv_len, batch.cu_q, max_q_len=max_q, max_kv_len=40)
    verify(paged_attention(q.to(cuda), cache, b, 0.2), q, k, v, table, lens, cu, 0.2)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("qlens,lens", [([1], [1]), ([1, 0, 3, 1], [1, 0, 5, 130]), ([30, 1], [30, 300]),
                                        ([1] * 9, [3] * 9), ([200], [4100])])
def test_short_lengths_in_a_wide_table(cuda, dtype, qlens, lens):
    """The table spans far more keys than the lengths reach: shares are dealt
    where there is less work than blocks, some of them a unit's fixed weight
    alone."""
    g = torch.Generator().manual_seed(71)
    cache, batch, table, cu, q, k, v = setup(g, dtype, qlens, lens, 8, 2, 64, 16, False, cuda)
    wide = torch.full((len(lens), 3000), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    for max_q in (max(qlens), None):
        b = PagedBatch(wide.to(cuda), batch.kv_len, batch.cu_q, max_q_len=max_q)
        verify(paged_attention(q.to(cuda), cache, b, 0.125), q, k, v, wide, lens, cu, 0.125)
