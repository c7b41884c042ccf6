"""Head norms and position rotation in one pass (kiv_norm_rope).

``norm_rope`` takes the rows a model's q and k projections leave and returns
them normed for each head (optional) and turned by their positions, ready for
the hot window (:class:`kiv_amd.TieredKVCache`), the cold store or the
attention kernels.  :class:`Rotary` and :class:`HeadNorm` also parametrise
:func:`kiv_amd.paged_append`, which does the same on the way into the pages.
No counterpart in the reference, whose models run their own rotation.
"""

from __future__ import annotations

import torch

from . import _native as nat


class HeadNorm:
    """Norm of each head's row: ``x / sqrt(mean(x^2) + eps) * (weight + offset)``.

    ``weight`` ([head_dim], or None for a norm without a scale) is copied in
    fp32 at construction; build another object after changing it.
    """

    def __init__(self, weight: torch.Tensor | None = None, eps: float = 1e-6, offset: float = 0.0) -> None:
        if weight is not None:
            if weight.dim() != 1:
                raise ValueError(f"norm weight must be [head_dim], got {tuple(weight.shape)}")
            if not weight.is_cuda:
                raise ValueError("norm weight must be on a GPU")
            weight = weight.detach().float().clone().contiguous()
            if offset:
                weight += offset
        elif offset:
            raise ValueError("a norm without a weight has no offset")
        if not eps >= 0.0:
            raise ValueError(f"norm epsilon must not be negative, got {eps}")
        self.weight = weight
        self.eps = eps
        self._args = nat.HeadNormArgs(nat.ptr(weight), eps, 1)

    def check(self, head_dim: int, device: torch.device) -> nat.HeadNormArgs:
        w = self.weight
        if w is not None and (w.shape[0] != head_dim or w.device != device):
            raise ValueError(f"norm weight is [{w.shape[0]}] on {w.device}, rows have head_dim {head_dim} on {device}")
        return self._args


class Rotary:
    """Position rotation of the first ``2 * len(inv_freq)`` entries of a row.

    inv_freq     [rot_dim / 2] fp32: pair i turns by position * inv_freq[i];
                 the angle is formed in 64 bits, so far positions keep the
                 precision of near ones.
    interleaved  pairs are neighbours (2 i, 2 i + 1) instead of entries
                 rot_dim / 2 apart.
    scale        factor of the cosines and sines.
    axes         [rot_dim / 2] integers: the position axis each pair follows
                 (images and video: time, height, width); positions then have
                 a leading axis dimension.
    """

    def __init__(self, inv_freq: torch.Tensor, interleaved: bool = False, scale: float = 1.0,
                 axes: torch.Tensor | None = None) -> None:
        if inv_freq.dim() != 1 or inv_freq.numel() == 0:
            raise ValueError(f"inv_freq must be [rot_dim / 2], got {tuple(inv_freq.shape)}")
        if not inv_freq.is_cuda:
            raise ValueError("inv_freq must be on a GPU")
        if inv_freq.dtype != torch.float32:
            raise TypeError(f"inv_freq must be float32, not {inv_freq.dtype}")
        if axes is not None:
            if axes.shape != inv_freq.shape or axes.device != inv_freq.device:
                raise ValueError("axes must have inv_freq's shape and device")
            if axes.is_floating_point() or axes.dtype == torch.bool:
                raise TypeError(f"axes must be integers, not {axes.dtype}")
            axes = axes.to(torch.int32).contiguous()
        self.inv_freq = inv_freq.contiguous()
        self.axes = axes
        self.interleaved = bool(interleaved)
        self.scale = float(scale)
        self.rot_dim = 2 * inv_freq.shape[0]
        self._args = nat.RotaryArgs(self.inv_freq.data_ptr(), nat.ptr(axes), None, nat._I64x3(), 0, 1, self.rot_dim,
                                    int(self.interleaved), self.scale, 0)

    def fill(self, dst: nat.RotaryArgs, positions: torch.Tensor | None, batch: int, tokens: int,
             device: torch.device, batched: bool) -> torch.Tensor | None:
        """Set the rotation in ``dst`` for positions [tokens], [batch, tokens]
        (``batched``) or either behind an axis dimension; returns the tensor
        the launch reads."""
        if self.inv_freq.device != device:
            raise ValueError(f"inv_freq is on {self.inv_freq.device}, rows on {device}")
        if positions is None:
            if self.axes is not None:
                raise ValueError("a rotation with several axes needs positions")
            return None
        if positions.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"positions must be int32 or int64, not {positions.dtype}")
        if positions.device != device:
            raise ValueError(f"positions are on {positions.device}, rows on {device}")
        shape, st = positions.shape, positions.stride()
        lead = 0 if self.axes is None else 1
        if lead:
            if len(shape) < 2 or shape[0] < 1:
                raise ValueError("positions of a rotation with several axes need a leading axis dimension")
            dst.num_axes = shape[0]
            dst.position_stride[0] = st[0]
        rest = shape[lead:]
        if rest == (tokens,):
            sb, stt = 0, st[lead]
        elif batched and len(rest) == 2 and rest[0] in (1, batch) and rest[1] == tokens:
            sb, stt = (0 if rest[0] == 1 else st[lead]), st[lead + 1]
        else:
            raise ValueError(f"positions {tuple(shape)} do not fit {batch} x {tokens} tokens")
        dst.position_stride[1], dst.position_stride[2] = sb, stt
        dst.positions = positions.data_ptr()
        dst.position_bytes = positions.element_size()
        return positions


def no_grad_check(what: str, *tensors: torch.Tensor | None) -> None:
    """These kernels have no backward pass: refuse to drop a gradient."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad()")


def aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """t itself where the kernels can load its rows (unit stride over
    head_dim, 16-byte aligned), else a copy."""
    vec = 16 // t.element_size()
    st = t.stride()
    ok = st[-1] == 1 and t.data_ptr() % 16 == 0
    for n, s in zip(t.shape[:-1], st[:-1]):
        ok = ok and (n == 1 or s % vec == 0)
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def out_rows(out: torch.Tensor, like: torch.Tensor, what: str) -> torch.Tensor:
    """Check a caller's output tensor."""
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{what} must be {tuple(like.shape)} {like.dtype} on {like.device}")
    if aligned_rows(out) is not out:
        raise ValueError(f"{what} rows must be 16-byte aligned, with unit stride over head_dim")
    return out


def norm_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor | None, rotary: Rotary | None,
              q_norm: HeadNorm | None = None, k_norm: HeadNorm | None = None, q_out: torch.Tensor | None = None,
              k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Head norms and position rotation of q [B, Hq, T, D] and k [B, Hkv, T, D]
    (any strides over B, H and T), each row read and written once.

    positions: [T], [B, T] or, with ``rotary.axes``, [axes, T] or
    [axes, B, T]; int32 or int64.  ``q_out`` / ``k_out`` may be the inputs
    themselves; by default they are new tensors in the inputs' memory order.
    fp32, fp16 and bf16; head_dim a multiple of 16 bytes up to 512, the
    rotated width of 32 bytes.  Returns (q_out, k_out).
    """
    no_grad_check("norm_rope", q, k)
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("q and k must be [B, H, T, D]")
    if not q.is_cuda:
        raise ValueError("norm_rope needs GPU tensors")
    B, hq, T, D = q.shape
    if k is not None and ((k.shape[0], k.shape[2], k.shape[3]) != (B, T, D) or k.dtype != q.dtype
                          or k.device != q.device):
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} does not go with q {tuple(q.shape)} {q.dtype}")
    if k is None and (k_norm is not None or k_out is not None):
        raise ValueError("k_norm and k_out need k")
    args = nat.NormRopeArgs()
    dev = q.device
    args.dtype = nat.dtype_code(q.dtype)
    args.batch, args.num_q_heads, args.tokens, args.head_dim = B, hq, T, D
    src = aligned_rows(q)
    q_out = torch.empty_like(src) if q_out is None else out_rows(q_out, q, "q_out")
    args.q, args.q_stride = src.data_ptr(), nat.strides(src, 3)
    args.q_out, args.q_out_stride = q_out.data_ptr(), nat.strides(q_out, 3)
    if q_norm is not None:
        args.q_norm = q_norm.check(D, dev)
    if k is not None:
        ksrc = aligned_rows(k)
        k_out = torch.empty_like(ksrc) if k_out is None else out_rows(k_out, k, "k_out")
        args.num_kv_heads = k.shape[1]
        args.k, args.k_stride = ksrc.data_ptr(), nat.strides(ksrc, 3)
        args.k_out, args.k_out_stride = k_out.data_ptr(), nat.strides(k_out, 3)
        if k_norm is not None:
            args.k_norm = k_norm.check(D, dev)
    if rotary is not None:
        if positions is None:
            raise ValueError("a rotation needs positions")
        args.rotary = rotary._args
        rotary.fill(args.rotary, positions, B, T, dev, batched=True)
    nat.call("kiv_norm_rope", args, dev)
    return q_out, k_out
