"""Keys and values in 4 bits, attention over them, and beam search, in plain 64-bit torch or Python."""
from __future__ import annotations

import math

import torch

D64 = torch.float64


def quantise(x: torch.Tensor):
    """Codes 0 .. 15 (int64), scale and centre (float64 holding bfloat16 values) of rows of values."""
    x = x.to(D64)
    finite = torch.isfinite(x).all(-1, keepdim=True)
    safe = torch.where(finite, x, torch.zeros_like(x))
    low, high = safe.amin(-1, keepdim=True), safe.amax(-1, keepdim=True)
    scale = ((high - low) / 15).float().bfloat16().to(D64)
    centre = (low + 8 * scale).float().bfloat16().to(D64)
    steps = torch.where(scale == 0, torch.zeros_like(x), (safe - centre) / torch.where(scale == 0, torch.ones_like(scale), scale))
    codes = (torch.round(steps) + 8).clamp(0, 15)
    codes = torch.where(finite, codes, torch.full_like(codes, 8)).long()
    centre = torch.where(finite, centre, torch.full_like(centre, math.nan))
    return codes, torch.where(finite, scale, torch.zeros_like(scale))[..., 0], centre[..., 0]


def pack(codes: torch.Tensor) -> torch.Tensor:
    return (codes[..., 0::2] + 16 * codes[..., 1::2]).to(torch.uint8)


def unpack(packed: torch.Tensor) -> torch.Tensor:
    packed = packed.long()
    return torch.stack([packed % 16, packed // 16], -1).flatten(-2)


def values(packed: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    scales = scales.to(D64)
    return scales[..., :1] * (unpack(packed) - 8).to(D64) + scales[..., 1:]


def rotate(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, pairing: int) -> torch.Tensor:
    """x [T, heads, D] (float64)."""
    angle = positions.to(D64)[:, None, None] * inv_freq.to(D64)
    cos, sin = torch.cos(angle), torch.sin(angle)
    half = x.shape[-1] // 2
    out = torch.empty_like(x)
    a, b = (x[..., 0::2], x[..., 1::2]) if pairing == 0 else (x[..., :half], x[..., half:])
    first, second = a * cos - b * sin, a * sin + b * cos
    if pairing == 0:
        out[..., 0::2], out[..., 1::2] = first, second
    else:
        out[..., :half], out[..., half:] = first, second
    return out


def attend(q, keys, vals, position: int, scale: float):
    """One row: q [n_q, D]; keys, vals [n, n_kv, D]; sees keys 0 .. position.  The output [n_q, D] and sum of weight * |value|."""
    n_q, n_kv = q.shape[0], keys.shape[1]
    if position < 0:
        return torch.zeros_like(q, dtype=D64), torch.zeros_like(q, dtype=D64)
    keys, vals = (x[:position + 1].to(D64).repeat_interleave(n_q // n_kv, 1) for x in (keys, vals))
    weights = torch.softmax(torch.einsum("hd,nhd->hn", q.to(D64), keys) * scale, -1)
    return torch.einsum("hn,nhd->hd", weights, vals), torch.einsum("hn,nhd->hd", weights, vals.abs())


def select(logits, scores, ended, end_token: int):
    """Lists of (score, token, parent, ended) per request, from sorting all offers."""
    requests, beams = scores.shape
    out = []
    for r in range(requests):
        offers = []
        for k in range(beams):
            score = float(scores[r, k])
            if score == -math.inf:
                continue
            if int(ended[r, k]):
                offers.append((score, k, end_token))
                continue
            row = logits[r * beams + k].to(D64)
            logs = score + (row - torch.logsumexp(row, 0))
            kept = torch.nonzero(logs > -math.inf)[:, 0]
            offers += [(float(v), k, int(t)) for v, t in zip(logs[kept].tolist(), kept.tolist())]
        offers.sort(key=lambda o: (-o[0], o[1], o[2]))
        rows = [(v, t, k, int(bool(int(ended[r, k])) or t == end_token)) for v, k, t in offers[:beams]]
        rows += [(-math.inf, end_token, i, 1) for i in range(len(rows), beams)]
        out.append(rows)
    return out


def reorder(parents, tables, lengths, page_size: int):
    """New tables and the (from, to) pages that are copied; lists of lists."""
    beams = len(parents[0])
    new, copies = [list(row) for row in tables], []
    for r, (request, length) in enumerate(zip(parents, lengths)):
        full, rest = divmod(length, page_size)
        free = [k for k in range(beams) if k not in request]
        taken = set()
        for i, parent in enumerate(request):
            row, old = new[r * beams + i], tables[r * beams + parent]
            row[:full] = old[:full]
            if rest and full < len(row):
                row[full] = old[full]
                if parent in taken:
                    row[full] = tables[r * beams + free.pop(0)][full]
                    copies.append((old[full], row[full]))
                taken.add(parent)
    return new, copies


def step_tables(first, counts, pages, page_start, page_size: int, tokens: int, width: int):
    start, segments, positions, slots = [0], [], [], []
    tables = []
    for s, (f, n) in enumerate(zip(first, counts)):
        mine = pages[page_start[s]:page_start[s + 1]]
        tables.append((mine + [-1] * width)[:width])
        for j in range(n):
            position = f + j
            page = mine[position // page_size] if position // page_size < len(mine) else -1
            segments.append(s)
            positions.append(position)
            slots.append(page * page_size + position % page_size if page >= 0 else -1)
        start.append(start[-1] + n)
    pad = tokens - len(segments)
    return start, segments + [-1] * pad, positions + [0] * pad, slots + [-1] * pad, [f + n for f, n in zip(first, counts)], tables
