"""Calls of the paged operators' C entry points whose rows share memory: they
are refused before any device work."""

from __future__ import annotations

import ctypes as C

import pytest

from kiv_amd import _native as nat

MB = 1 << 20


def i64(*x):
    return (C.c_int64 * len(x))(*x)


def refused(entry, args, *words):
    lib = nat.lib()
    assert getattr(lib, entry)(C.byref(args), None) == nat.ERR_INVALID
    text = lib.kiv_last_error().decode()
    assert entry in text and all(w in text for w in words), text


def rope(**over):
    """5 tokens of 4 q heads over 2 k heads of 64 bf16, everything apart."""
    a = nat.NormRopeArgs(batch=2, tokens=5, num_q_heads=4, num_kv_heads=2, head_dim=64, dtype=nat.DTYPE_BF16)
    a.q, a.q_out, a.k, a.k_out = (MB * i for i in range(1, 5))
    a.q_stride = a.q_out_stride = i64(5 * 256, 64, 256)
    a.k_stride = a.k_out_stride = i64(5 * 128, 64, 128)
    for name, value in over.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("words,over", [
    (("q_out", "q"), dict(q_out=MB + 128)),                        # a head further
    (("q_out", "q"), dict(q_out=MB + 16)),
    (("q_out", "q"), dict(q_out=MB, q_out_stride=i64(5 * 256, 5 * 64, 64))),  # in place in another order
    (("k_out", "k"), dict(k_out=3 * MB + 256)),
    (("q_out", "k"), dict(q_out=3 * MB)),
    (("k_out", "q"), dict(k_out=MB + 512)),
    (("q_out", "k_out"), dict(k_out=2 * MB)),
    (("q_out", "k"), dict(q_out=MB, k=MB, k_out=MB)),  # q and k one tensor, both in place
    (("rows of q_out",), dict(q_out_stride=i64(5 * 256, 0, 256))),
    (("rows of k_out",), dict(k_out_stride=i64(0, 64, 128))),
    (("rows of q_out",), dict(q=2 * MB, q_stride=i64(5 * 64, 0, 64), q_out_stride=i64(5 * 64, 0, 64))),  # expanded, in place
    (("q_out", "q"), dict(q_stride=i64(5 * 512, 64, 512), q_out_stride=i64(5 * 512, 64, 512), q_out=MB + 2 * 192)),
])
def test_norm_rope(words, over):
    refused("kiv_norm_rope", rope(**over), *words)


def fill(a):
    """4 pages of 8 tokens of 2 heads of 64 bf16: 16 KiB each of K and V."""
    a.cache = nat.PagedCacheArgs(16 * MB, 32 * MB, i64(1024, 512, 64), 4, 8, 2, 64, nat.DTYPE_BF16, 0)
    a.batch = nat.PagedBatchArgs(MB, MB, MB, 3, 2, 3, 5, 1, 24, 0)


def append(**over):
    a = nat.PagedAppendArgs()
    fill(a)
    a.k, a.v, a.q, a.q_out = 2 * MB, 3 * MB, 4 * MB, 5 * MB
    a.k_stride = a.v_stride = i64(128, 64)
    a.q_stride = a.q_out_stride = i64(256, 64)
    a.num_q_heads = 4
    for name, value in over.items():
        obj, _, field = name.rpartition("__")
        setattr(getattr(a, obj) if obj else a, field, value)
    return a


@pytest.mark.parametrize("words,over", [
    (("q_out", "q"), dict(q_out=4 * MB + 512)),
    (("q_out", "k"), dict(q_out=2 * MB + 128)),
    (("q_out", "v"), dict(q_out=3 * MB)),
    (("rows of q_out",), dict(q_out_stride=i64(256, 0))),
    (("pages", "k"), dict(k=16 * MB + 1024)),
    (("pages", "v"), dict(v=16 * MB + 1024)),
    (("pages", "k"), dict(k=32 * MB)),
    (("pages", "q"), dict(q=32 * MB + 128, q_out=32 * MB + 128)),
    (("pages", "q_out"), dict(q_out=16 * MB - 128)),
    (("K pages", "V pages"), dict(cache__v=16 * MB)),
    (("K pages", "V pages"), dict(cache__v=16 * MB + 2048 * 3)),
    (("rows of the pages",), dict(cache__stride=i64(1024, 0, 64))),
    (("rows of the pages",), dict(cache__stride=i64(512, 512, 64))),
])
def test_paged_append(words, over):
    refused("kiv_paged_append", append(**over), "over" if "rows" not in words[0] else "share", *words)


@pytest.mark.parametrize("out", [16 * MB, 32 * MB + 4 * 2048 - 128, 16 * MB - 5 * 512 + 128])
def test_paged_attention(out):
    a = nat.PagedAttentionArgs()
    fill(a)
    a.q, a.out, a.q_stride = 2 * MB, out, i64(256, 64)
    a.num_q_heads, a.scaling = 4, 0.125
    refused("kiv_paged_attention", a, "out must not overlap the pages")
