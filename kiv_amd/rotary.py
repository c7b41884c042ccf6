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
from torch.autograd import forward_ad

from . import _native as nat


class HeadNorm:
    """Norm of each head's row: ``x / sqrt(mean(x^2) + eps) * (weight + offset)``.

    ``weight`` ([head_dim], or None for a norm without a scale) is copied in
    fp32 at construction; build another object after changing it.  It gets no
    gradient: one that requires it makes calls fail where gradients are
    recorded.
    """

    def __init__(self, weight: torch.Tensor | None = None, eps: float = 1e-6, offset: float = 0.0) -> None:
        no_tangent_check("HeadNorm", weight)
        self.requires_grad = weight is not None and weight.requires_grad
        if weight is not None:
            if weight.dim() != 1:
                raise ValueError(f"norm weight must be [head_dim], got {tuple(weight.shape)}")
            if not weight.is_cuda:
                raise ValueError("norm weight must be on a GPU")
            weight = weight.detach().to(torch.float32, copy=True).contiguous()
            if offset:
                weight += offset
        elif offset:
            raise ValueError("a norm without a weight has no offset")
        if not eps >= 0.0:
            raise ValueError(f"norm epsilon must not be negative, got {eps}")
        self._weight = weight
        self.eps = eps
        self._at = None if weight is None else (weight.shape[0], weight.device)
        self._args = nat.HeadNormArgs(nat.ptr(weight), eps, 1)

    @property
    def weight(self) -> torch.Tensor | None:
        return self._weight

    def check(self, head_dim: int, device: torch.device) -> nat.HeadNormArgs:
        if self.requires_grad:
            no_grad_check("HeadNorm", self)
        at = self._at
        if at is not None and at != (head_dim, device):
            raise ValueError(f"norm weight is [{at[0]}] on {at[1]}, rows have head_dim {head_dim} on {device}")
        return self._args


class Rotary:
    """Position rotation of the first ``2 * len(inv_freq)`` entries of a row.

    inv_freq     [rot_dim / 2] fp32: pair i turns by position * inv_freq[i];
                 the angle is formed in 64 bits, so far positions keep the
                 precision of near ones.  It gets no gradient: one that
                 requires it makes calls fail where gradients are recorded.
    interleaved  pairs are neighbours (2 i, 2 i + 1) instead of entries
                 rot_dim / 2 apart.
    scale        factor of the cosines and sines.
    axes         [rot_dim / 2] integers: the position axis each pair follows
                 (images and video: time, height, width); positions then have
                 a leading axis dimension.  A number outside it means its
                 nearest axis.
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
            if axes.dtype not in (torch.int32, torch.int16, torch.int8, torch.uint8):
                axes = axes.to(torch.int64).clamp(0, 2**31 - 1)  # int32 would wrap round
            axes = axes.to(torch.int32).contiguous()
        no_tangent_check("Rotary", inv_freq)
        self.requires_grad = inv_freq.requires_grad
        self._inv_freq = inv_freq.detach().contiguous()
        self._axes = axes
        self.rot_dim = 2 * inv_freq.shape[0]
        self.device = inv_freq.device
        self._args = nat.RotaryArgs(self._inv_freq.data_ptr(), nat.ptr(axes), None, nat._I64x3(), 0, 1, self.rot_dim,
                                    int(bool(interleaved)), float(scale), 0)

    @property
    def inv_freq(self) -> torch.Tensor:
        return self._inv_freq

    @property
    def axes(self) -> torch.Tensor | None:
        return self._axes

    def fill(self, dst: nat.RotaryArgs, positions: torch.Tensor | None, batch: int, tokens: int,
             device: torch.device, batched: bool) -> None:
        """Set the positions in ``dst``: [tokens], [batch, tokens] (``batched``)
        or either behind an axis dimension."""
        if self.requires_grad:
            no_grad_check("Rotary", self)
        if self.device != device:
            raise ValueError(f"inv_freq is on {self.device}, rows on {device}")
        lead = self._axes is not None
        if positions is None:
            if lead:
                raise ValueError("a rotation with several axes needs positions")
            return
        if positions.device != device:
            raise ValueError(f"positions are on {positions.device}, rows on {device}")
        key = (positions.shape, positions.stride(), positions.dtype, lead, batched, batch, tokens)
        got = _position_layouts.get(key)
        if got is None:
            got = nat.remember(_position_layouts, key, _position_layout(*key))
        dst.position_stride, dst.position_bytes, dst.num_axes = got
        dst.positions = positions.data_ptr()


_position_layouts: dict[tuple, tuple] = {}


def _position_layout(shape, st, dtype, lead: bool, batched: bool, batch: int, tokens: int) -> tuple:
    """(strides over axis, batch and token; bytes; axes) of positions."""
    if dtype not in (torch.int64, torch.int32):
        raise TypeError(f"positions must be int32 or int64, not {dtype}")
    axes, sa, rest = 1, 0, tuple(shape)
    if lead:
        if len(rest) < 2 or rest[0] < 1:
            raise ValueError("positions of a rotation with several axes need a leading axis dimension")
        axes, sa, rest = rest[0], st[0], rest[1:]
    if rest == (tokens,):
        sb, stt = 0, st[lead]
    elif batched and len(rest) == 2 and rest[0] in (1, batch) and rest[1] == tokens:
        sb, stt = (0 if rest[0] == 1 else st[lead]), st[lead + 1]
    else:
        raise ValueError(f"positions {tuple(shape)} do not fit {batch} x {tokens} tokens")
    return nat._I64x3(sa, sb, stt), 8 if dtype == torch.int64 else 4, axes


def no_grad_check(what: str, *inputs: torch.Tensor | HeadNorm | Rotary | None) -> None:
    """These kernels have no derivatives: refuse to drop one, of what a call
    reads or of what it writes over."""
    if torch.is_grad_enabled():
        for x in inputs:
            if x is not None and x.requires_grad:
                raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad()")
    # Tangents exist within a level only; asking each tensor costs 0.3 us.
    if getattr(forward_ad, "_current_level", 0) >= 0:
        no_tangent_check(what, *inputs)


def no_tangent_check(what: str, *inputs: torch.Tensor | HeadNorm | Rotary | None) -> None:
    for x in inputs:
        if isinstance(x, torch.Tensor) and forward_ad.unpack_dual(x).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative")


def aligned_rows(t: torch.Tensor) -> tuple[torch.Tensor, int, nat.Layout]:
    """(tensor, address, layout) of t where the kernels can load its rows (unit
    stride over head_dim, 16-byte aligned), else of a copy."""
    lay, at = nat.layout(t), t.data_ptr()
    if lay.chunked and at & 15 == 0:
        return t, at, lay
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), nat.layout(t)


def out_rows(out: torch.Tensor, like: torch.Tensor, what: str) -> tuple[int, nat.Layout]:
    """Check a caller's output tensor: its address and layout."""
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{what} must be {tuple(like.shape)} {like.dtype} on {like.device}")
    lay, at = nat.layout(out), out.data_ptr()
    if not lay.chunked or at & 15:
        raise ValueError(f"{what} rows must be 16-byte aligned, with unit stride over head_dim")
    return at, lay


def norm_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor | None, rotary: Rotary | None,
              q_norm: HeadNorm | None = None, k_norm: HeadNorm | None = None, q_out: torch.Tensor | None = None,
              k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Head norms and position rotation of q [B, Hq, T, D] and k [B, Hkv, T, D]
    (any strides over B, H and T), each row read and written once.

    positions: [T], [B, T] or, with ``rotary.axes``, [axes, T] or
    [axes, B, T]; int32 or int64.  ``q_out`` / ``k_out`` may be the inputs
    themselves (any other overlap of theirs is refused); by default they are
    new tensors in the inputs' memory order.
    fp32, fp16 and bf16; head_dim a multiple of 16 bytes up to 512, the
    rotated width of 32 bytes.  Returns (q_out, k_out).
    """
    no_grad_check("norm_rope", q, k)
    dev = q.device
    if dev.type != "cuda":
        raise ValueError("norm_rope needs GPU tensors")
    key = (q.shape, q.stride(), q.dtype, None if k is None else (k.shape, k.stride(), k.dtype))
    plan = _plans.get(key)
    if plan is None:
        plan = nat.remember(_plans, key, _plan(q, k))
    template, B, T, D, copy_q, copy_k = plan
    args = nat.NormRopeArgs.from_buffer_copy(template)
    at = q.data_ptr()
    if copy_q or at & 15:
        q, at, lay = aligned_rows(q)
        args.q_stride = args.q_out_stride = lay.strides
    args.q = at
    if q_out is None:
        q_out = torch.empty_like(q)
        args.q_out = q_out.data_ptr()
    else:
        no_grad_check("norm_rope", q_out)
        args.q_out, lay = out_rows(q_out, q, "q_out")
        args.q_out_stride = lay.strides
    if q_norm is not None:
        args.q_norm = q_norm.check(D, dev)
    if k is not None:
        if k.device != dev:
            raise ValueError(f"k is on {k.device}, q on {dev}")
        at = k.data_ptr()
        if copy_k or at & 15:
            k, at, lay = aligned_rows(k)
            args.k_stride = args.k_out_stride = lay.strides
        args.k = at
        if k_out is None:
            k_out = torch.empty_like(k)
            args.k_out = k_out.data_ptr()
        else:
            no_grad_check("norm_rope", k_out)
            args.k_out, lay = out_rows(k_out, k, "k_out")
            args.k_out_stride = lay.strides
        if k_norm is not None:
            args.k_norm = k_norm.check(D, dev)
    elif k_norm is not None or k_out is not None:
        raise ValueError("k_norm and k_out need k")
    if rotary is not None:
        if positions is None:
            raise ValueError("a rotation needs positions")
        args.rotary = rotary._args
        rotary.fill(args.rotary, positions, B, T, dev, True)
    nat.call("kiv_norm_rope", args, dev)
    return q_out, k_out


_plans: dict[tuple, tuple] = {}


def _plan(q: torch.Tensor, k: torch.Tensor | None) -> tuple:
    """What a call's shapes, strides and dtypes give: (its arguments without
    addresses, B, T, D, q must be copied, k must be copied)."""
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("q and k must be [B, H, T, D]")
    nat.check_sizes("norm_rope", *q.shape, *(() if k is None else k.shape))
    B, hq, T, D = q.shape
    if k is not None and ((k.shape[0], k.shape[2], k.shape[3]) != (B, T, D) or k.dtype != q.dtype):
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} does not go with q {tuple(q.shape)} {q.dtype}")
    args = nat.NormRopeArgs(batch=B, tokens=T, num_q_heads=hq, head_dim=D, dtype=nat.dtype_code(q.dtype))
    # The memory order torch gives new tensors like these.
    lay, args.q_out_stride = nat.layout(q), nat.layout(torch.empty_like(q, device="meta")).strides
    args.q_stride = lay.strides
    if k is None:
        return args, B, T, D, not lay.chunked, False
    klay, args.k_out_stride = nat.layout(k), nat.layout(torch.empty_like(k, device="meta")).strides
    args.num_kv_heads, args.k_stride = k.shape[1], klay.strides
    return args, B, T, D, not lay.chunked, not klay.chunked
