"""The paged cache's C entry points without a GPU: struct layouts, and
arguments that are refused before any device work."""

from __future__ import annotations

import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from kiv_amd import _native as nat

HEADER = Path(__file__).resolve().parents[1] / "include" / "kiv_hip.h"
STRUCTS = {
    "kiv_rotary_t": nat.RotaryArgs,
    "kiv_head_norm_t": nat.HeadNormArgs,
    "kiv_norm_rope_args_t": nat.NormRopeArgs,
    "kiv_paged_cache_t": nat.PagedCacheArgs,
    "kiv_paged_batch_t": nat.PagedBatchArgs,
    "kiv_paged_append_args_t": nat.PagedAppendArgs,
    "kiv_paged_attention_args_t": nat.PagedAttentionArgs,
}
AT = 1 << 20  # an aligned address that no refused call follows


def test_struct_layouts_match_c(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for cname, py in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        for field, _ in py._fields_:
            lines.append(f'printf("{cname} {field} %zu\\n", offsetof({cname}, {field}));')
    lines.append("return 0; }")
    (tmp_path / "layout.c").write_text("\n".join(lines))
    subprocess.run([gcc, str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    for line in subprocess.check_output([str(tmp_path / "layout")], text=True).splitlines():
        cname, field, val = line.split()
        py = STRUCTS[cname]
        assert int(val) == (C.sizeof(py) if field == "size" else getattr(py, field).offset), (cname, field)


def rope_args(**over):
    a = nat.NormRopeArgs(batch=1, tokens=2, num_q_heads=2, num_kv_heads=1, head_dim=64, dtype=nat.DTYPE_BF16)
    a.q = a.q_out = a.k = a.k_out = AT
    for f in ("q_stride", "q_out_stride", "k_stride", "k_out_stride"):
        setattr(a, f, (C.c_int64 * 3)(256, 64, 128))
    a.rotary = nat.RotaryArgs(AT, None, AT, (C.c_int64 * 3)(0, 0, 1), 8, 1, 64, 0, 1.0, 0)
    for name, value in over.items():
        obj, _, field = name.rpartition("__")
        setattr(getattr(a, obj) if obj else a, field, value)
    return a


@pytest.mark.parametrize("code,over", [
    (nat.ERR_INVALID, dict(dtype=7)),
    (nat.ERR_UNSUPPORTED, dict(head_dim=60)),
    (nat.ERR_UNSUPPORTED, dict(head_dim=520)),
    (nat.ERR_INVALID, dict(num_q_heads=0)),
    (nat.ERR_INVALID, dict(tokens=-1)),
    (nat.ERR_INVALID, dict(q=None)),
    (nat.ERR_INVALID, dict(k_out=None)),
    (nat.ERR_INVALID, dict(q=AT + 2)),
    (nat.ERR_INVALID, dict(q_stride=(C.c_int64 * 3)(256, 60, 128))),
    (nat.ERR_UNSUPPORTED, dict(rotary__rot_dim=72)),
    (nat.ERR_UNSUPPORTED, dict(rotary__rot_dim=24)),
    (nat.ERR_UNSUPPORTED, dict(rotary__rot_dim=-16)),
    (nat.ERR_INVALID, dict(rotary__inv_freq=None)),
    (nat.ERR_INVALID, dict(rotary__positions=None)),
    (nat.ERR_INVALID, dict(rotary__position_bytes=2)),
    (nat.ERR_INVALID, dict(rotary__num_axes=0)),
    (nat.ERR_INVALID, dict(q_norm=nat.HeadNormArgs(None, -1.0, 1))),
    (nat.ERR_INVALID, dict(q_norm=nat.HeadNormArgs(None, float("nan"), 1))),
    (nat.ERR_INVALID, dict(q_norm=nat.HeadNormArgs(AT + 4, 1e-6, 1))),
])
def test_norm_rope_refusals(code, over):
    lib = nat.lib()
    assert lib.kiv_norm_rope(C.byref(rope_args(**over)), None) == code
    assert b"kiv_norm_rope" in lib.kiv_last_error()


def test_nothing_to_do_is_no_error():
    lib = nat.lib()
    assert lib.kiv_norm_rope(C.byref(rope_args(tokens=0)), None) == 0
    assert lib.kiv_norm_rope(C.byref(rope_args(batch=0)), None) == 0
    assert lib.kiv_paged_append(C.byref(append_args(batch__total_q=0)), None) == 0
    assert lib.kiv_paged_append(C.byref(append_args(batch__num_seqs=0)), None) == 0
    assert lib.kiv_norm_rope(None, None) == nat.ERR_INVALID and lib.kiv_paged_append(None, None) == nat.ERR_INVALID


def fill_cache(a):
    a.cache = nat.PagedCacheArgs(AT, AT, (C.c_int64 * 3)(1024, 512, 64), 4, 8, 2, 64, nat.DTYPE_BF16, 0)
    a.batch = nat.PagedBatchArgs(AT, AT, AT, 3, 2, 3, 2, 1, 24, 0)


def append_args(**over):
    a = nat.PagedAppendArgs()
    fill_cache(a)
    a.k = a.v = a.q = a.q_out = AT
    for f in ("k_stride", "v_stride", "q_stride", "q_out_stride"):
        setattr(a, f, (C.c_int64 * 2)(128, 64))
    a.num_q_heads = 4
    a.rotary = nat.RotaryArgs(AT, None, None, (C.c_int64 * 3)(), 0, 1, 64, 0, 1.0, 0)
    for name, value in over.items():
        obj, _, field = name.rpartition("__")
        setattr(getattr(a, obj) if obj else a, field, value)
    return a


CACHE_REFUSALS = [
    (nat.ERR_INVALID, dict(cache__dtype=3)),
    (nat.ERR_INVALID, dict(cache__k=None)),
    (nat.ERR_INVALID, dict(cache__v=AT + 8)),
    (nat.ERR_INVALID, dict(cache__num_pages=0)),
    (nat.ERR_INVALID, dict(cache__stride=(C.c_int64 * 3)(1024, 512, 60))),
    (nat.ERR_UNSUPPORTED, dict(cache__num_pages=1 << 30)),
    (nat.ERR_INVALID, dict(batch__num_seqs=-1)),
    (nat.ERR_INVALID, dict(batch__cu_q=None)),
    (nat.ERR_INVALID, dict(batch__block_table=None)),
    (nat.ERR_UNSUPPORTED, dict(batch__table_width=1 << 29)),
]


@pytest.mark.parametrize("code,over", CACHE_REFUSALS + [
    (nat.ERR_INVALID, dict(k=None)),
    (nat.ERR_INVALID, dict(v_stride=(C.c_int64 * 2)(128, 4))),
    (nat.ERR_INVALID, dict(q_out=None)),
    (nat.ERR_INVALID, dict(num_q_heads=-1)),
    (nat.ERR_UNSUPPORTED, dict(rotary__rot_dim=80)),
    (nat.ERR_INVALID, dict(rotary__axes=AT)),
    (nat.ERR_INVALID, dict(v_norm=nat.HeadNormArgs(None, -1.0, 1))),
])
def test_paged_append_refusals(code, over):
    lib = nat.lib()
    assert lib.kiv_paged_append(C.byref(append_args(**over)), None) == code
    assert b"kiv_paged_append" in lib.kiv_last_error()


LONG = dict(batch__table_width=1000, batch__max_kv_len=8000)  # keys that several blocks share


def attention_args(**over):
    a = nat.PagedAttentionArgs()
    fill_cache(a)
    a.q = a.out = a.workspace = AT
    a.q_stride = (C.c_int64 * 2)(256, 64)
    a.num_q_heads, a.scaling, a.workspace_bytes = 4, 0.125, 1 << 40
    for name, value in over.items():
        obj, _, field = name.rpartition("__")
        setattr(getattr(a, obj) if obj else a, field, value)
    return a


@pytest.mark.parametrize("code,over", CACHE_REFUSALS + [
    (nat.ERR_INVALID, dict(q=None)),
    (nat.ERR_INVALID, dict(out=AT + 8)),
    (nat.ERR_INVALID, dict(q_stride=(C.c_int64 * 2)(256, 60))),
    (nat.ERR_INVALID, dict(num_q_heads=3)),
    (nat.ERR_INVALID, dict(num_q_heads=0)),
    (nat.ERR_INVALID, dict(window=-1)),
    (nat.ERR_UNSUPPORTED, dict(cache__head_dim=48)),
    (nat.ERR_UNSUPPORTED, dict(cache__head_dim=512)),
    (nat.ERR_UNSUPPORTED, dict(scaling=0.0)),
    (nat.ERR_UNSUPPORTED, dict(scaling=float("nan"))),
    (nat.ERR_UNSUPPORTED, dict(scaling=float("inf"))),
    (nat.ERR_INVALID, dict(LONG, workspace=None)),
    (nat.ERR_INVALID, dict(LONG, workspace=AT + 16)),
    (nat.ERR_INVALID, dict(LONG, workspace_bytes=64)),
    (nat.ERR_UNSUPPORTED, dict(batch__table_width=(1 << 27) + 1)),
    (nat.ERR_UNSUPPORTED, dict(LONG, batch__table_width=1 << 27, batch__total_q=1 << 20)),
])
def test_paged_attention_refusals(code, over):
    lib = nat.lib()
    assert lib.kiv_paged_attention(C.byref(attention_args(**over)), None) == code
    assert b"kiv_paged_attention" in lib.kiv_last_error()


@pytest.mark.parametrize("over", [
    dict(),                                               # the query itself
    dict(out=AT + 512),                                   # a token further
    dict(out=AT + 512, q=AT + 512 * 4),                   # its last rows are the query's first
    dict(out=AT + 512, q_stride=(C.c_int64 * 2)(512, 64)),  # between rows that lie apart
    dict(q=AT + 512 * 8, q_stride=(C.c_int64 * 2)(-256, 64)),
])
def test_paged_attention_out_over_the_query(over):
    lib = nat.lib()
    args = attention_args(batch__total_q=5, **over)
    assert lib.kiv_paged_attention(C.byref(args), None) == nat.ERR_INVALID
    assert b"overlap" in lib.kiv_last_error()


def test_paged_workspace_size():
    lib = nat.lib()
    assert lib.kiv_paged_attention_workspace_size(None) == 0
    assert lib.kiv_paged_attention_workspace_size(C.byref(attention_args(cache__head_dim=48))) == 0
    assert lib.kiv_paged_attention_workspace_size(C.byref(attention_args(batch__total_q=0))) == 0
    assert lib.kiv_paged_attention_workspace_size(C.byref(attention_args())) == 0  # few keys: never divided
    assert lib.kiv_paged_attention_workspace_size(C.byref(attention_args(**LONG))) > 0
    assert lib.kiv_paged_attention(C.byref(attention_args(batch__total_q=0, workspace=None)), None) == 0
    assert lib.kiv_paged_attention(None, None) == nat.ERR_INVALID


def test_cpu_tensors_are_refused():
    from kiv_amd import HeadNorm, PagedKVCache, Rotary, norm_rope

    q = torch.zeros(1, 2, 3, 64)
    with pytest.raises(ValueError):
        norm_rope(q, None, None, None)
    with pytest.raises(ValueError):
        Rotary(torch.ones(32))
    with pytest.raises(ValueError):
        HeadNorm(torch.ones(64))
    with pytest.raises(ValueError):
        PagedKVCache(2, 8, 1, 64, device="cpu")


@pytest.mark.parametrize("scaling", [2.4e38, 3.4e38])
def test_scaling_that_overflows_in_base_2_is_refused(scaling):
    lib = nat.lib()
    assert lib.kiv_paged_attention(C.byref(attention_args(scaling=scaling)), None) == nat.ERR_UNSUPPORTED
    assert b"scaling" in lib.kiv_last_error()


def test_sizes_past_32_bits_are_refused():
    """Before they are cut to 32 bits; on shapes without memory."""
    from types import SimpleNamespace

    from kiv_amd import PagedBatch, PagedKVCache, paged, rotary

    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, device="meta", dtype=dtype)

    n = 2**32 + 1
    cache = SimpleNamespace(head_dim=64, num_kv_heads=1, dtype=torch.bfloat16)
    one = meta(1, 1, 64)
    for f in (
        lambda: rotary._plan(meta(1, 1, n, 8), None),
        lambda: rotary._plan(meta(1, n, 1, 8), meta(1, 1, 1, 8)),
        lambda: rotary._plan(meta(1, 1, 1, 8), meta(1, n, 1, 8)),
        lambda: PagedKVCache.from_pages(meta(n, 1, 1, 8), meta(n, 1, 1, 8)),
        lambda: PagedBatch(meta(n, 1, dtype=torch.int32), meta(n, dtype=torch.int32)),
        lambda: PagedBatch(meta(1, n, dtype=torch.int32), meta(1, dtype=torch.int32)),
        lambda: paged._append_plan(cache, meta(n, 1, 64), meta(n, 1, 64), None),
        lambda: paged._append_plan(cache, one, one, meta(1, n, 64)),
        lambda: paged._attention_plan(meta(n, 1, 64), cache, None, 0),
    ):
        with pytest.raises(ValueError, match="2\\^31"):
            f()
    rotary._plan(meta(1, 1, 2**31 - 1, 8), None)


def test_heads_past_32_bits_are_refused():
    lib = nat.lib()
    assert lib.kiv_norm_rope(C.byref(rope_args(num_q_heads=2**31 - 1)), None) == nat.ERR_UNSUPPORTED
    assert lib.kiv_norm_rope(C.byref(rope_args(num_q_heads=2**30, num_kv_heads=2**30)), None) == nat.ERR_UNSUPPORTED
    assert lib.kiv_paged_append(C.byref(append_args(num_q_heads=2**31 - 1)), None) == nat.ERR_UNSUPPORTED
    assert lib.kiv_paged_append(C.byref(append_args(cache__num_kv_heads=2**30)), None) == nat.ERR_UNSUPPORTED
