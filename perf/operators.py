"""The operators of a paged key/value cache, as cases that can be timed.

A case is a dict of plain values.  Three kinds of call:

  rope     norm_rope: the queries' and keys' norms for each head with the
           position rotation (one or several position axes) in the same pass;
  append   paged_append: the same for a ragged batch of new tokens, the keys
           and values written to their pages of the cache on the way (the
           queries normed and rotated beside them where the case says so);
  attend   paged_attention: a ragged batch of new tokens (single tokens,
           chunks, both together) over the pages of the cache, under the
           causal rule, with or without a sliding window.

Head shapes are those of kiv_amd/synthetic.py, bench.py and the tests.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


def listed() -> list[dict]:
    return [
        # One decode step's token far into a million-token context: all launch and latency.
        dict(name="rope_token_1m", kind="rope", batch=1, hq=28, hkv=4, dim=128, rot=128, dtype="bf16", tokens=1,
             start=1048575, norm=True, interleaved=False, axes=0),
        # One chunk of a long prefill, late in the prompt.
        dict(name="rope_chunk_4096", kind="rope", batch=1, hq=28, hkv=4, dim=128, rot=128, dtype="bf16", tokens=4096,
             start=1040000, norm=True, interleaved=False, axes=0),
        # A batch of two image-and-text prompts: three position axes, half of each head rotated, pairs side by side.
        dict(name="rope_axes_ragged", kind="rope", batch=2, hq=32, hkv=4, dim=64, rot=32, dtype="fp16", tokens=1531,
             start=0, norm=False, interleaved=True, axes=3),
        # A decode step of 64 sequences.
        dict(name="append_tokens_64", kind="append", seqs=64, qlen=1, kv=8192, ragged=True, lens=3, hq=28, hkv=4,
             dim=128, rot=128, dtype="bf16", page=128, tokens_first=False, queries=True, norm=True, axes=0),
        # One prefill chunk onto a cache that holds as much already.
        dict(name="append_chunk_4096", kind="append", seqs=1, qlen=4096, kv=8192, ragged=False, lens=0, hq=12, hkv=2,
             dim=128, rot=128, dtype="bf16", page=128, tokens_first=False, queries=True, norm=True, axes=0),
        # Prompts of many lengths at once, multi-head attention, small pages laid out by token, rotation alone.
        dict(name="append_ragged_mha", kind="append", seqs=13, qlen=1531, kv=2777, ragged=True, lens=5, hq=32, hkv=32,
             dim=96, rot=96, dtype="fp16", page=16, tokens_first=True, queries=False, norm=False, axes=0),
        # The first answer token of a short chat.
        dict(name="attend_token_short", kind="attend", seqs=1, qlen=1, kv=301, ragged=False, lens=0, hq=32, hkv=4,
             dim=64, dtype="fp16", page=128, tokens_first=False, window=0),
        # A decode step of 64 sequences of different lengths.
        dict(name="attend_tokens_64", kind="attend", seqs=64, qlen=1, kv=8192, ragged=True, lens=3, hq=28, hkv=4,
             dim=128, dtype="bf16", page=128, tokens_first=False, window=0),
        # One token over a million keys.
        dict(name="attend_token_1m", kind="attend", seqs=1, qlen=1, kv=1048576, ragged=False, lens=0, hq=28, hkv=4,
             dim=128, dtype="bf16", page=128, tokens_first=False, window=0),
        # One prefill chunk over as many earlier keys and itself.
        dict(name="attend_chunk_4096", kind="attend", seqs=1, qlen=4096, kv=8192, ragged=False, lens=0, hq=12, hkv=2,
             dim=128, dtype="bf16", page=128, tokens_first=False, window=0),
        # Prompt chunks among decode steps, small pages laid out by token, off every tile size.
        dict(name="attend_mixed_ragged", kind="attend", seqs=9, qlen=777, kv=4099, ragged=True, lens=11, hq=32, hkv=8,
             dim=128, dtype="fp16", page=16, tokens_first=True, window=0),
        # Wide heads, one key head, a sliding window.
        dict(name="attend_chunk_window", kind="attend", seqs=2, qlen=1531, kv=6007, ragged=True, lens=4, hq=8, hkv=1,
             dim=256, dtype="bf16", page=64, tokens_first=False, window=1024),
    ]


# ------------------------------------------------------------------ drawing
_HEADS = ((32, 4, 64), (28, 4, 128), (12, 2, 128), (32, 32, 96), (8, 1, 256), (14, 2, 64), (16, 4, 128), (32, 8, 128))


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng) -> dict:
    kind = rng.choice(("rope", "append", "attend", "attend", "attend"))
    hq, hkv, dim = rng.choice(_HEADS)
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    rot = rng.choice((dim, dim, dim // 2))
    if kind == "rope":
        batch = rng.choice((1, 1, 2, 3))
        return dict(kind=kind, batch=batch, hq=hq, hkv=hkv, dim=dim, rot=rot, dtype=dtype,
                    tokens=_log(rng, 1, 4096 // batch // (2 if dtype == "fp32" else 1)),
                    start=_log(rng, 1, 1 << 20), norm=rng.random() < 0.6, interleaved=rng.random() < 0.4,
                    axes=rng.choice((0, 0, 3)))
    shape = rng.choice(("tokens", "tokens", "chunk", "mixed"))
    seqs = {"tokens": _log(rng, 1, 100), "chunk": rng.choice((1, 1, 2)), "mixed": rng.randint(2, 12)}[shape]
    # Keys of all sequences: K and V within 1 GiB in 32 bits.
    kv = _log(rng, 16, max(64, min(1 << 19, (1 << 27) // (seqs * hkv * dim))))
    qlen = 1 if shape == "tokens" else _log(rng, 2, min(kv, 4096))
    if kind == "append":
        return dict(kind=kind, seqs=seqs, qlen=min(qlen, max(1, 4096 // seqs)), kv=kv, ragged=rng.random() < 0.7,
                    lens=rng.randrange(1000), hq=hq, hkv=hkv, dim=dim, rot=rot, dtype=dtype,
                    page=rng.choice((16, 32, 64, 128)), tokens_first=rng.random() < 0.4, queries=rng.random() < 0.7,
                    norm=rng.random() < 0.6, axes=rng.choice((0, 0, 3)))
    # Scores of the padded plain form within those of the listed chunk; fp32 chunks are shorter.
    while seqs * qlen * kv * hq > (1 << 26 if dtype == "fp32" else 1 << 28) and qlen > 1:
        qlen = max(1, qlen // 2)
    return dict(kind=kind, seqs=seqs, qlen=qlen, kv=kv, ragged=rng.random() < 0.7, lens=rng.randrange(1000), hq=hq,
                hkv=hkv, dim=dim, dtype=dtype, page=rng.choice((16, 32, 64, 128)), tokens_first=rng.random() < 0.4,
                window=rng.choice((0, 0, 0, _log(rng, 8, 4096))))


def _lengths(c: dict) -> tuple[list[int], list[int]]:
    """New tokens and keys (the new ones among them) of each sequence: the
    first has the case's; of a ragged batch the others have fewer keys, and
    are idle, decode one token or bring a chunk."""
    r = random.Random(c["lens"])
    q, kv = [c["qlen"]], [c["kv"]]
    for _ in range(c["seqs"] - 1):
        if not c["ragged"]:
            q.append(c["qlen"])
            kv.append(c["kv"])
            continue
        n = r.choice((0, 1, 1, 1, 1, 1, r.randint(1, c["qlen"]), r.randint(1, c["qlen"])))
        q.append(n)
        kv.append(max(n, r.randint(max(1, c["kv"] // 8), c["kv"])))
    return q, kv


# ------------------------------------------------------------------- inputs
def _gen(seed: int, salt: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(1_000_003 * seed + salt)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def _rotary(c: dict, g) -> dict:
    """Inverse frequencies (base 1e6, as long-context models take), the axis
    of each pair (time, height and width in turn) and the norms' weights."""
    half = c["rot"] // 2
    s = {"inv_freq": (1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)).float()}
    s["axis"] = torch.arange(half, device="cuda", dtype=torch.int32) % c["axes"] if c["axes"] else None
    dt = DTYPES[c["dtype"]]
    s["q_weight"] = 1 + _normal(g, (c["dim"],), torch.float32, 0.2).to(dt) if c["norm"] else None
    s["k_weight"] = 1 + _normal(g, (c["dim"],), torch.float32, 0.2).to(dt) if c["norm"] else None
    return s


def _pool(c: dict, g, kv: list[int], filled: bool):
    """Pages of K and V ([page, head, slot, dim], by token in memory where the
    case says so) and a table of pages scattered over the pool."""
    dt, ps = DTYPES[c["dtype"]], c["page"]
    need = [-(-n // ps) for n in kv]
    pages, width = sum(need) + 3, max(1, max(need))
    shape = (pages, ps, c["hkv"], c["dim"]) if c["tokens_first"] else (pages, c["hkv"], ps, c["dim"])
    k, v = (_normal(g, shape, dt) if filled else torch.zeros(shape, device="cuda", dtype=dt) for _ in range(2))
    if c["tokens_first"]:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    first = torch.tensor([0] + need[:-1], device="cuda").cumsum(0)
    col = torch.arange(width, device="cuda")
    at = (first[:, None] + col[None, :]).clamp(max=pages - 1)
    held = col[None, :] < torch.tensor(need, device="cuda")[:, None]
    return k, v, torch.where(held, order[at], -1).to(torch.int32).contiguous()


def prepare(case: dict, seed: int) -> dict:
    c, dt = case, DTYPES[case["dtype"]]
    g = _gen(seed, 17)
    s = dict(case=c)
    if c["kind"] == "rope":
        # The projections' rows side by side, as one product over q, k and v leaves them.
        rows = c["hq"] + 2 * c["hkv"]
        qkv = _normal(g, (c["batch"], c["tokens"], rows, c["dim"]), dt)
        s["q"] = qkv[:, :, :c["hq"]].transpose(1, 2)
        s["k"] = qkv[:, :, c["hq"]:c["hq"] + c["hkv"]].transpose(1, 2)
        pos = c["start"] + torch.arange(c["tokens"], device="cuda").expand(c["batch"], -1)
        # Axes: time, and the row and column of a patch within its image.
        s["positions"] = torch.stack([pos, pos // 16 % 64, pos % 16]) if c["axes"] else pos
        s.update(_rotary(c, g))
        if own:
            from kiv_amd import HeadNorm, Rotary

            s["rotary"] = Rotary(s["inv_freq"], interleaved=c["interleaved"], axes=s["axis"])
            s["q_norm"] = HeadNorm(s["q_weight"], EPS) if c["norm"] else None
            s["k_norm"] = HeadNorm(s["k_weight"], EPS) if c["norm"] else None
        return s
    q, kv = _lengths(c)
    total = sum(q)
    s["cu"] = torch.tensor([0] + q, device="cuda").cumsum(0).to(torch.int32)
    s["lens"] = torch.tensor(kv, device="cuda", dtype=torch.int32)
    s["max_q"], s["max_kv"] = max(q), max(kv)
    s["k_pages"], s["v_pages"], s["table"] = _pool(c, g, kv, filled=c["kind"] == "attend")
    if c["kind"] == "attend":
        s["q"] = _normal(g, (total, c["hq"], c["dim"]), dt)
    else:
        qkv = _normal(g, (total, c["hq"] + 2 * c["hkv"], c["dim"]), dt)
        s["q"] = qkv[:, :c["hq"]]
        s["k"] = qkv[:, c["hq"]:c["hq"] + c["hkv"]]
        s["v"] = qkv[:, c["hq"] + c["hkv"]:]
        s["positions"] = torch.randint(0, 4096, (c["axes"], total), device="cuda", generator=g) if c["axes"] else None
        s.update(_rotary(c, g))
    if own:
        from kiv_amd import HeadNorm, PagedBatch, PagedKVCache, Rotary

        s["cache"] = PagedKVCache.from_pages(s["k_pages"], s["v_pages"])
        s["batch"] = PagedBatch(s["table"], s["lens"], s["cu"], max_q_len=s["max_q"], max_kv_len=s["max_kv"])
        if c["kind"] == "append":
            s["rotary"] = Rotary(s["inv_freq"], axes=s["axis"])
            s["q_norm"] = HeadNorm(s["q_weight"], EPS) if c["norm"] else None
            s["k_norm"] = HeadNorm(s["k_weight"], EPS) if c["norm"] else None
    return s


# -------------------------------------------------------------- plain forms
def _norm(x, weight):
    """Rows over their root mean square, times the weight."""
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _angles(s, positions):
    """Cosines and sines [..., pair] of positions [...] or, with axes,
    [axis, ...]; products of far positions in 64 bits."""
    p = positions.double()
    if s["axis"] is not None:
        p = p[s["axis"].long()].movedim(0, -1)
    else:
        p = p[..., None]
    a = p * s["inv_freq"].double()
    return a.cos().float(), a.sin().float()


def _rotate(x, cos, sin, rot, interleaved):
    """Pairs of the first rot entries turned by their angles; a pair is two
    entries half the rotated width apart, or two neighbours."""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_rope(s):
    c = s["case"]
    cos, sin = _angles(s, s["positions"])
    cos, sin = cos[:, None], sin[:, None]
    return tuple(_rotate(_norm(s[n].float(), s[n + "_weight"]), cos, sin, c["rot"], c["interleaved"]).to(s[n].dtype)
                 for n in ("q", "k"))


def _rows(s):
    """Of each packed token: its sequence, and its key index there."""
    t = torch.arange(s["q"].shape[0], device=s["q"].device)
    b = torch.bucketize(t, s["cu"][1:].long(), right=True)
    return b, s["lens"][b].long() - s["cu"][b + 1].long() + t


def _plain_append(s):
    c = s["case"]
    b, key = _rows(s)
    cos, sin = _angles(s, key if s["positions"] is None else s["positions"])
    cos, sin = cos[:, None], sin[:, None]
    page, slot = s["table"][b, key // c["page"]].long(), key % c["page"]
    k = _rotate(_norm(s["k"].float(), s["k_weight"]), cos, sin, c["rot"], False)
    s["k_pages"][page, :, slot] = k.to(s["k"].dtype)
    s["v_pages"][page, :, slot] = s["v"]
    if not c["queries"]:
        return s["k_pages"], s["v_pages"]
    q = _rotate(_norm(s["q"].float(), s["q_weight"]), cos, sin, c["rot"], False).to(s["q"].dtype)
    return s["k_pages"], s["v_pages"], q


def _plain_attend(s):
    c, q = s["case"], s["q"]
    hq, hkv, dim = c["hq"], c["hkv"], c["dim"]
    dev, n, m = q.device, s["max_q"], s["max_kv"]
    seqs = s["lens"].shape[0]
    table = s["table"].long().clamp(min=0)
    keys, vals = (p[table].transpose(1, 2).reshape(seqs, hkv, -1, dim)[:, :, :m].float()
                  for p in (s["k_pages"], s["v_pages"]))
    cu = s["cu"].long()
    i = torch.arange(n, device=dev)
    qlen = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + i).clamp(max=max(0, q.shape[0] - 1))
    rows = q[at].float().view(seqs, n, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4).reshape(seqs, hkv, -1, dim)
    scores = torch.matmul(rows * dim ** -0.5, keys.transpose(-1, -2)).view(seqs, hkv, hq // hkv, n, -1)
    last = s["lens"].long()[:, None] - qlen[:, None] + i
    j = torch.arange(scores.shape[-1], device=dev)
    seen = (j <= last[..., None]) & (i < qlen[:, None])[..., None]
    if c["window"]:
        seen &= j > last[..., None] - c["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(seqs, hkv, -1, p.shape[-1]), vals).view(*p.shape[:4], dim)
    out = torch.where(total > 0, out / total, 0.0)
    b, _ = _rows(s)
    t = torch.arange(q.shape[0], device=dev)
    return out.permute(0, 3, 1, 2, 4).reshape(seqs, n, hq, dim)[b, t - cu[b]].to(q.dtype)


def run(state: dict):
    s, c = state, state["case"]
    if not own:
        return {"rope": _plain_rope, "append": _plain_append, "attend": _plain_attend}[c["kind"]](s)
    from kiv_amd import norm_rope, paged_append, paged_attention

    if c["kind"] == "rope":
        return norm_rope(s["q"], s["k"], s["positions"], s["rotary"], q_norm=s["q_norm"], k_norm=s["k_norm"])
    if c["kind"] == "attend":
        return paged_attention(s["q"], s["cache"], s["batch"], c["dim"] ** -0.5, window=c["window"])
    q = paged_append(s["cache"], s["batch"], s["k"], s["v"], q=s["q"] if c["queries"] else None,
                     positions=s["positions"], rotary=s["rotary"], q_norm=s["q_norm"], k_norm=s["k_norm"])
    return (s["k_pages"], s["v_pages"], q) if c["queries"] else (s["k_pages"], s["v_pages"])


# --------------------------------------------------------------------- work
def _spans(c: dict):
    """(new tokens, keys that some of them sees, visible pairs) a sequence."""
    got = []
    for q, kv in zip(*_lengths(c)):
        w = c["window"] or kv
        first, base = max(0, kv - q + 1 - w), kv - q
        pairs = sum(min(base + i + 1, w) for i in range(q)) if c["window"] else q * base + q * (q + 1) // 2
        got.append((q, kv - first if q else 0, pairs))
    return got


def work(case: dict) -> dict:
    c, e = case, BYTES[case["dtype"]]
    row = c["dim"] * e
    if c["kind"] == "rope":
        n, rows = c["batch"] * c["tokens"], c["hq"] + c["hkv"]
        per = 3 * c["rot"] + (4 * c["dim"] if c["norm"] else 0)
        return {"bytes": 2 * n * rows * row + 8 * n * max(1, c["axes"]) + 2 * c["rot"], "flops": n * rows * per}
    total = sum(_lengths(c)[0])
    if c["kind"] == "append":
        turned = c["hkv"] + (c["hq"] if c["queries"] else 0)
        per = 3 * c["rot"] + (4 * c["dim"] if c["norm"] else 0)
        moved = 2 * total * (turned + c["hkv"]) * row
        return {"bytes": moved + 8 * total * c["axes"] + 2 * c["rot"] + 12 * c["seqs"], "flops": total * turned * per}
    spans = _spans(c)
    keys, pairs = sum(x[1] for x in spans), sum(x[2] for x in spans)
    return {"bytes": 2 * total * c["hq"] * row + 2 * keys * c["hkv"] * row + 4 * keys // c["page"] + 12 * c["seqs"],
            "flops": 4 * pairs * c["hq"] * c["dim"]}


# -------------------------------------------------------------------- exact
def _exact_rows(x, weight, angle, rot, interleaved):
    """Rows [..., head, dim] in 64 bits: normed, then as complex numbers."""
    x = x.double()
    if weight is not None:
        x = weight.double() * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    z = x[..., :rot]
    z = z.unflatten(-1, (-1, 2)) if interleaved else z.unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_complex(z.contiguous()) * torch.polar(torch.ones_like(angle), angle)[..., None, :]
    z = torch.view_as_real(z)
    z = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
    return torch.cat([z, x[..., rot:]], -1)


def exact(case: dict, seed: int):
    c, s = case, prepare(case, seed)
    if c["kind"] != "attend":
        freq = s["inv_freq"].double()
        pos = s["positions"]
        if pos is None:
            kv, q = torch.tensor(_lengths(c)[1]), torch.tensor(_lengths(c)[0])
            pos = torch.cat([torch.arange(n - m, n) for m, n in zip(q.tolist(), kv.tolist())]).cuda()
        pos = pos.double() if c["axes"] else pos.double()[None]
        angle = torch.stack([pos[f % max(1, c["axes"])] * freq[f] for f in range(freq.numel())], -1)
    if c["kind"] == "rope":
        return tuple(_exact_rows(s[n].transpose(1, 2), s[n + "_weight"], angle, c["rot"], c["interleaved"])
                     .transpose(1, 2) for n in ("q", "k"))
    table, lens = s["table"].cpu(), _lengths(c)
    if c["kind"] == "append":
        k = _exact_rows(s["k"], s["k_weight"], angle, c["rot"], False)
        kp, vp, t = s["k_pages"].double(), s["v_pages"].double(), 0
        for b, (m, n) in enumerate(zip(*lens)):
            key = torch.arange(n - m, n)
            page, slot = table[b][key // c["page"]].long().cuda(), (key % c["page"]).cuda()
            kp.transpose(1, 2)[page, slot] = k[t:t + m]
            vp.transpose(1, 2)[page, slot] = s["v"][t:t + m].double()
            t += m
        q = (_exact_rows(s["q"], s["q_weight"], angle, c["rot"], False),) if c["queries"] else ()
        return (kp, vp) + q
    out, t, group = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0, c["hq"] // c["hkv"]
    for b, (m, n) in enumerate(zip(*lens)):
        pages = table[b][:-(-n // c["page"])].long().cuda()
        last = torch.arange(n - m, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        hidden = key > last
        if c["window"]:
            hidden |= key <= last - c["window"]
        for h in range(c["hq"] if m else 0):
            k, v = (x[pages, h // group].flatten(0, 1)[:n].double() for x in (s["k_pages"], s["v_pages"]))
            w = (s["q"][t:t + m, h].double() @ k.T / math.sqrt(c["dim"])).masked_fill(hidden, -math.inf)
            out[t:t + m, h] = torch.softmax(w, -1) @ v
        t += m
    return out
