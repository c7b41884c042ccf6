"""Plain 64-bit references of the paged cache's operators, on the CPU, and
the bounds their kernels are held to."""

from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24  # half a step of fp32


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def ref_norm(x, weight, eps, offset=0.0):
    """Rows [..., D] in 64 bits over their root mean square, times weight."""
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    return y if weight is None else y * (weight.double() + offset)


def ref_angles(positions, inv_freq, axes=None):
    """[..., pair] angles of positions [...], or [axis, ...] with axes."""
    p, f = positions.double(), inv_freq.double()
    if axes is None:
        return p[..., None] * f
    return torch.stack([p[int(a)] * f[i] for i, a in enumerate(axes)], -1)


def ref_rotate(x, angle, interleaved=False, scale=1.0):
    """(rotated rows, |a| + |b| of each entry's pair): x [..., D], angle
    [..., rot / 2] broadcastable over x's leading dims."""
    rot = 2 * angle.shape[-1]
    c, s = angle.cos() * scale, angle.sin() * scale
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    u, w, size = a * c - b * s, b * c + a * s, (a.abs() + b.abs()) * abs(scale)
    y, mag = x.clone(), x.abs()
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = u, w
        mag[..., 0:rot:2], mag[..., 1:rot:2] = size, size
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = u, w
        mag[..., :rot // 2], mag[..., rot // 2:rot] = size, size
    return y, mag


def rope_bound(ref, mag, dtype):
    """The store's rounding, and the fp32 steps before it relative to a
    pair's size: the norm's sum (16 products a lane and 6 tree levels, halved
    by the root, about 11 half steps), its root and two products (4), the
    angle's rounding after reduction (pi) and the sine's (2 to 4), products
    and difference (3): under 32 half steps in all."""
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return half_step(dtype) * ref.abs() + 32 * U32 * mag + tiny


def check(got, ref, bound, what=""):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - ref).abs() - bound
    assert (over <= 0).all(), f"{what}: {float(over.max()):.3g} over the bound"


def positions_of(cu, kv_len):
    """Sequence and key index of each packed row."""
    seq, key = [], []
    for b in range(len(kv_len)):
        n = cu[b + 1] - cu[b]
        seq += [b] * n
        key += [kv_len[b] - n + i for i in range(n)]
    return seq, key


def ref_attention(q, k_pages, v_pages, table, kv_len, cu, scaling, window=0):
    """(outputs, sum of p |v|, largest |score|) [rows, Hq, D / 1] in 64 bits
    over the pages that are there; rows of no sequence are zero."""
    hq, D = q.shape[1], q.shape[2]
    pages, hkv, ps, _ = k_pages.shape
    G = hq // hkv
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b in range(len(kv_len)):
        n = cu[b + 1] - cu[b]
        keys = [j for j in range(min(kv_len[b], table.shape[1] * ps)) if 0 <= int(table[b, j // ps]) < pages]
        for i in range(n):
            last = kv_len[b] - n + i
            seen = [j for j in keys if j <= last and (not window or j > last - window)]
            if not seen:
                continue
            at = torch.tensor([int(table[b, j // ps]) for j in seen]), torch.tensor([j % ps for j in seen])
            k, v = k_pages[at[0], :, at[1]].double(), v_pages[at[0], :, at[1]].double()  # [keys, hkv, D]
            qr = q[cu[b] + i].double().view(hkv, G, D)
            s = torch.einsum("hgd,khd->hgk", qr, k) * scaling
            p = torch.softmax(s, -1)
            out[cu[b] + i] = torch.einsum("hgk,khd->hgd", p, v).reshape(hq, D)
            mag[cu[b] + i] = torch.einsum("hgk,khd->hgd", p, v.abs()).reshape(hq, D)
    return out, mag


def make_table(lens, page, pages, g, width=None, extra=0):
    """A block table of scattered pages, -1 past each sequence's last."""
    need = [math.ceil(n / page) for n in lens]
    width = max([1] + need) + extra if width is None else width
    order = torch.randperm(pages, generator=g).tolist()
    t = torch.full((len(lens), width), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for j in range(n):
            t[b, j] = order.pop()
    return t


def attention_bound(ref, mag, q, k_pages, dtype, scaling, n):
    """The store's rounding; the probabilities' rounding to the dtype (16-bit
    types; fp16 also loses those below its smallest number); and fp32 steps:
    a score's D products and sums (relative to the largest sum of |q k|, S),
    which moves a probability by as much and the normalised sum by twice
    that, and n additions of the weighted sum with the exponentials' few."""
    u, D = half_step(dtype), q.shape[-1]
    S = float(q.double().abs().amax() * k_pages.double().abs().nan_to_num(0.0).amax()) * D * scaling
    # |q|_2 |k|_2 bounds sum |q k| far closer where rows are long.
    S = min(S, float(q.double().norm(dim=-1).amax() * k_pages.double().nan_to_num(0.0).norm(dim=-1).amax()) * scaling)
    fp32 = (2 * (D + 8) * S + n + 64) * U32
    bound = u * ref.abs() + (fp32 + (0.0 if dtype == torch.float32 else u)) * mag + 1e-30
    if dtype == torch.float16:
        bound = bound + n * 2.0 ** -25 * mag.amax() + 2.0 ** -25
    return bound
