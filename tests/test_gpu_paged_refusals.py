"""Calls of the paged cache's operators that would lose something: gradients
of their parameters, pages and outputs, and forward-mode tangents."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from kiv_amd import HeadNorm, PagedBatch, PagedKVCache, Rotary, norm_rope, paged_append, paged_attention

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


class Step:
    """Two tokens of two sequences over four pages."""

    def __init__(self, cuda):
        self.cache = PagedKVCache(4, 8, 2, 64, BF16, cuda)
        self.cache.k.zero_()
        self.cache.v.zero_()
        table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=cuda)
        self.batch = PagedBatch(table, torch.tensor([3, 9], dtype=torch.int32, device=cuda))
        self.q = torch.randn(2, 4, 64, device=cuda).to(BF16)
        self.k, self.v = (torch.randn(2, 2, 64, device=cuda).to(BF16) for _ in range(2))
        self.pos = torch.arange(2, device=cuda)
        self.freq = torch.ones(32, device=cuda)
        self.weight = torch.ones(64, device=cuda)

    def rope(self, **over):
        q, k = self.q.transpose(0, 1)[None], self.k.transpose(0, 1)[None]
        rotary = over.pop("rotary", None) or Rotary(self.freq)
        return norm_rope(q, k, self.pos, rotary, **over)

    def append(self, **over):
        return paged_append(over.pop("cache", self.cache), self.batch, self.k, self.v, self.q, **over)

    def attend(self, **over):
        return paged_attention(self.q, over.pop("cache", self.cache), self.batch, 0.125, **over)


def grad(t):
    return t.detach().clone().requires_grad_()


def trained_pages(s, k, v):
    return PagedKVCache.from_pages(grad(s.cache.k) if k else s.cache.k, grad(s.cache.v) if v else s.cache.v)


CALLS = {
    "rope q_norm": lambda s: s.rope(q_norm=HeadNorm(grad(s.weight))),
    "rope k_norm": lambda s: s.rope(k_norm=HeadNorm(grad(s.weight), offset=1.0)),
    "rope inv_freq": lambda s: s.rope(rotary=Rotary(grad(s.freq))),
    "rope q_out": lambda s: s.rope(q_out=grad(s.q.transpose(0, 1)[None])),
    "rope k_out": lambda s: s.rope(k_out=grad(s.k.transpose(0, 1)[None])),
    "append q_norm": lambda s: s.append(q_norm=HeadNorm(grad(s.weight))),
    "append k_norm": lambda s: s.append(k_norm=HeadNorm(grad(s.weight))),
    "append v_norm": lambda s: s.append(v_norm=HeadNorm(grad(s.weight))),
    "append inv_freq": lambda s: s.append(rotary=Rotary(grad(s.freq))),
    "append q_out": lambda s: s.append(q_out=grad(s.q)),
    "append K pages": lambda s: s.append(cache=trained_pages(s, True, False)),
    "append V pages": lambda s: s.append(cache=trained_pages(s, False, True)),
    "attend K pages": lambda s: s.attend(cache=trained_pages(s, True, False)),
    "attend V pages": lambda s: s.attend(cache=trained_pages(s, False, True)),
    "attend out": lambda s: s.attend(out=grad(s.q)),
}


@pytest.mark.parametrize("name", CALLS)
def test_gradients_are_not_dropped(cuda, name):
    step = Step(cuda)
    with pytest.raises(RuntimeError, match="no backward pass"):
        CALLS[name](step)
    with torch.no_grad():
        CALLS[name](step)


def test_tangents_are_not_dropped(cuda):
    s = Step(cuda)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        k, v, q = s.k, s.v, s.q
        calls = [
            lambda: norm_rope(dual(q)[None], None, None, None, HeadNorm()),
            lambda: norm_rope(q[None], dual(q)[None], None, None, HeadNorm()),
            lambda: paged_append(s.cache, s.batch, dual(k), v),
            lambda: paged_append(s.cache, s.batch, k, dual(v)),
            lambda: paged_append(s.cache, s.batch, k, v, dual(q)),
            lambda: paged_attention(dual(q), s.cache, s.batch, 0.125),
            lambda: HeadNorm(dual(s.weight)),
            lambda: Rotary(dual(s.freq)),
        ]
        for grads in (True, False):
            with torch.set_grad_enabled(grads):
                for f in calls:
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        f()
                s.append()
                s.attend()
