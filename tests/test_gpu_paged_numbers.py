"""paged_attention's numbers where a sum is cut or a type is narrow: NaN in
queries and keys, whole and divided units alike, many small weights beside a
large one, and weights that 16 bits do not hold; against references that take
long key ranges at once."""

from __future__ import annotations

import pytest
import torch

from kiv_amd import PagedBatch, PagedKVCache, paged_append, paged_attention
from tests.paged_ref import attention_bound, check

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PAGE = 64


def pool(k, v, dtype, cuda):
    """A cache of one sequence whose pages lie in order, and its table."""
    n, hkv, D = k.shape
    pages = -(-n // PAGE)
    rows = torch.zeros(2, pages * PAGE, hkv, D, dtype=dtype, device=cuda)
    rows[0, :n], rows[1, :n] = k, v
    cache = PagedKVCache.from_pages(*(t.view(pages, PAGE, hkv, D).transpose(1, 2) for t in rows))
    return cache, torch.arange(pages, dtype=torch.int32, device=cuda)[None]


def one_sequence(table, n, T, cuda, hint=True):
    return PagedBatch(table, torch.tensor([n], dtype=torch.int32, device=cuda),
                      torch.tensor([0, T], dtype=torch.int32, device=cuda), max_q_len=T,
                      max_kv_len=n if hint else None)


def reference(q, k, v, scaling):
    """(outputs, sum of p |v|) of the last T tokens over n keys, in 64 bits
    on the inputs' device."""
    T, hq, D = q.shape
    n, hkv, _ = k.shape
    q, k, v = q.double(), k.double(), v.double()
    hidden = torch.arange(n, device=q.device) > torch.arange(n - T, n, device=q.device)[:, None]
    out, mag = torch.empty_like(q), torch.empty_like(q)
    for h in range(hq):
        g = h // (hq // hkv)
        p = torch.softmax((q[:, h] @ k[:, g].T * scaling).masked_fill(hidden, -float("inf")), -1)
        out[:, h], mag[:, h] = p @ v[:, g], p @ v[:, g].abs()
    return out, mag


# Keys of a unit that goes whole, of one that is divided, and of one cut into
# many parts (whose merge splits them over a block).
SHAPES = [(300, 1), (6000, 1), (90_000, 1), (300, 70), (9000, 70)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,T", SHAPES)
@pytest.mark.parametrize("hint", [True, False], ids=["hint", "nohint"])
def test_nan_query_rows_are_nan(cuda, dtype, n, T, hint):
    """A query row of NaN gives a row of NaN however its unit is cut, and no
    other row is touched."""
    g = torch.Generator(device=cuda).manual_seed(n + T)
    k, v = (torch.randn(n, 2, 64, device=cuda, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(T, 8, 64, device=cuda, generator=g).to(dtype)
    cache, table = pool(k, v, dtype, cuda)
    batch = one_sequence(table, n, T, cuda, hint)
    want = paged_attention(q, cache, batch, 0.125)
    assert torch.isfinite(want).all()
    hit = torch.zeros(T, 8, dtype=torch.bool, device=cuda)
    hit[0, 3] = hit[T // 2, 5] = hit[T - 1, 0] = True
    got = paged_attention(torch.where(hit[..., None], float("nan"), q), cache, batch, 0.125)
    assert torch.isnan(got[hit]).all()
    assert torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,T", SHAPES)
@pytest.mark.parametrize("first,share", [(0, 0.4), (0.3, 0.5), (0.5, 0.5)])
def test_nan_keys_reach_the_rows_that_see_them(cuda, dtype, n, T, first, share):
    """A range of NaN keys, longer than some of the parts a unit is cut into:
    every row that sees one is NaN."""
    g = torch.Generator(device=cuda).manual_seed(n + T + 1)
    k, v = (torch.randn(n, 2, 64, device=cuda, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(T, 8, 64, device=cuda, generator=g).to(dtype)
    a = int(first * n)
    k[a:a + int(share * n), 1] = float("nan")
    cache, table = pool(k, v, dtype, cuda)
    got = paged_attention(q, cache, one_sequence(table, n, T, cuda), 0.125)
    sees = torch.arange(n - T, n, device=cuda) >= a
    assert torch.isnan(got[sees][:, 4:]).all()
    assert torch.isfinite(got[:, :4]).all() and torch.isfinite(got[~sees]).all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,T", [(400, 1), (400, 33), (1 << 17, 1), (1 << 20, 1), (1 << 17, 33)])
def test_many_small_weights_beside_a_large_one(cuda, dtype, n, T):
    """One key, worth nothing, 13 to 17.5 nats above all others, each worth 64:
    the output is the others' share, in closed form.  16-bit types round it at
    the store and each probability as an operand, half a step each (all the
    others' probabilities are alike, so theirs does not average out); fp32 sums
    lose at most half a step an addition, of which a lane makes one for each 16
    of the keys (chunks: for each 2), and the exponentials and quotients a few
    more."""
    gaps = torch.tensor([13.0, 14.1875, 15.5, 16.375, 17.0, 17.1875, 17.375, 17.5], dtype=torch.float64)
    k, v = torch.zeros(2, n, 1, 64, device=cuda, dtype=dtype)
    k[5, 0, 0] = 1.0
    v[:] = 64.0
    v[5] = 0.0
    q = torch.zeros(T, len(gaps), 64, device=cuda, dtype=dtype)
    q[:, :, 0] = gaps.to(cuda, dtype)
    gaps = q[0, :, 0].double().cpu()
    cache, table = pool(k, v, dtype, cuda)
    got = paged_attention(q, cache, one_sequence(table, n, T, cuda), 1.0).double().cpu()
    others = (torch.arange(n - T, n, dtype=torch.float64))[:, None]
    want = (64 * others / (others + gaps.exp()))[..., None]
    half = torch.finfo(dtype).eps / 2
    bound = (half + (0 if dtype == F32 else half * (1 + half)) + (n / (16 if T == 1 else 2) + 64) * 2.0 ** -24) * want
    over, off = float(((got - want).abs() - bound).max()), float(((got - want).abs() / want).max())
    assert over <= 0, f"off by up to {off:.2g} of the value"


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("n,T", [(37, 1), (700, 4), (9000, 1)])
def test_tokens_weigh_values_by_more_than_16_bits(cuda, dtype, D, n, T):
    """Units of 16 rows hold a probability to 2^-16 (fp16 2^-22 and, far under
    the maximum, 2^-36) of its value.  Scores are exact products here, so that
    fp32 adds only their scaling's and exponentials' half steps and one an
    addition (a lane adds one in 16 of the keys)."""
    g = torch.Generator(device=cuda).manual_seed(D + n)
    k, v = (torch.randn(n, 2, D, device=cuda, generator=g).to(dtype) for _ in range(2))
    q = torch.zeros(T, 8, D, device=cuda, dtype=dtype)
    q[:, :, 0] = torch.rand(T, 8, device=cuda, generator=g) * 3
    cache, table = pool(k, v, dtype, cuda)
    got = paged_attention(q, cache, one_sequence(table, n, T, cuda), 1.0).double()
    ref, mag = reference(q, k, v, 1.0)
    top = float(q.abs().max() * k[:, :, 0].abs().max())
    rest, gone = (2.0 ** -16, 0.0) if dtype == BF16 else (2.0 ** -22, n * 2.0 ** -36 * float(v.abs().max()) + 2.0 ** -25)
    bound = torch.finfo(dtype).eps / 2 * ref.abs() + (rest + (8 * top + n / 16 + 64) * 2.0 ** -24) * mag + gone
    over = float(((got - ref).abs() - bound).max())
    assert over <= 0, f"{over:.2g} over the bound"


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,T,rows", [(300, 90, 41), (300, 4, 1), (5000, 64, 30)])
def test_a_prefix_of_a_steps_rows(cuda, dtype, n, T, rows):
    """cu_q runs past the rows that a call is given: append and attention
    give each row the key that it has in the whole step."""
    g = torch.Generator(device=cuda).manual_seed(n + T)
    k, v = (torch.randn(n, 2, 64, device=cuda, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(T, 8, 64, device=cuda, generator=g).to(dtype)
    cache, table = pool(k * (torch.arange(n, device=cuda) < n - T)[:, None, None], v, dtype, cuda)
    whole = one_sequence(table, n, T, cuda)
    paged_append(cache, whole, k[n - T:][:rows], v[n - T:][:rows])
    got = paged_attention(q[:rows], cache, whole, 0.125)
    ref, mag = (x[:rows].cpu() for x in reference(q, k, v, 0.125))
    check(got, ref, attention_bound(ref, mag, q.cpu(), k.cpu(), dtype, 0.125, n))
