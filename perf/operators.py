"""Timed cases of the operators that serve many beams from a cache held in 4 bits, one call each.

* ``write``: bias, rotation and the write of keys and values into 4-bit pages, read back as the values that they stand for.
* ``rows``: attention of single rows (decoding) over 4-bit pages.
* ``portions``: attention of prompt portions, causal, over 4-bit pages.
* ``select``: beam search's choice of the best continuations over all beams of a request and the vocabulary.
* ``reorder``: block tables (or state slots) after that choice, and the copies of what two beams may no longer share.
* ``tables``: what a step has to know (segments, positions, cache slots, contexts, padded block tables) from its requests' lengths.

A row of D values of a head is held as codes u in 0 .. 15 (uint8, two a byte: byte b holds d = 2b in its low and 2b + 1 in its
high half) with a scale s and a centre c (bfloat16), and stands for s (u - 8) + c.
"""
from __future__ import annotations

import math

import torch

own = False

# (query heads, key/value heads, head size): the benchmark's three models, and small heads without groups
HEADS = {"1.5b": (12, 2, 128), "7b": (28, 4, 128), "14b": (40, 8, 128), "small": (8, 8, 64)}
VOCABULARY = 151936
THETA, PAGE = 1000000.0, 16


def listed() -> list[dict]:
    return [
        # a full batch decoding: a key and a value of 64 requests enter the cache
        {"name": "write_64", "kind": "write", "heads": "7b", "tokens": 64, "context": 2000, "dtype": "bfloat16", "pairing": 1, "page": PAGE},
        # a long prompt's portion of odd length, projections left in float32
        {"name": "write_2001", "kind": "write", "heads": "14b", "tokens": 2001, "context": 8000, "dtype": "float32", "pairing": 0, "page": PAGE},
        # one request that holds a book: few rows, many keys
        {"name": "rows_1x30000", "kind": "rows", "heads": "7b", "requests": 1, "context": 30000, "ragged": False, "page": PAGE},
        # a full batch of chats at different lengths
        {"name": "rows_64x1900", "kind": "rows", "heads": "1.5b", "requests": 64, "context": 1900, "ragged": True, "page": PAGE},
        # prompts in portions beside each other, behind what was cached before
        {"name": "portions_8x200", "kind": "portions", "heads": "1.5b", "requests": 8, "tokens": 200, "context": 500, "ragged": True, "page": PAGE},
        # the last portion of a long prompt
        {"name": "portions_1x2048", "kind": "portions", "heads": "14b", "requests": 1, "tokens": 2048, "context": 6144, "ragged": False, "page": PAGE},
        # one user's four beams
        {"name": "select_1x4", "kind": "select", "requests": 1, "beams": 4, "vocabulary": VOCABULARY},
        # a batch of requests with eight beams each
        {"name": "select_32x8", "kind": "select", "requests": 32, "beams": 8, "vocabulary": VOCABULARY},
        # four beams over the pages of all layers
        {"name": "reorder_1x4", "kind": "reorder", "heads": "1.5b", "layers": 28, "requests": 1, "beams": 4, "context": 1000, "page": PAGE, "states": False},
        # a batch of requests with eight beams each
        {"name": "reorder_16x8", "kind": "reorder", "heads": "7b", "layers": 28, "requests": 16, "beams": 8, "context": 90, "page": PAGE, "states": False},
        # a decoding step of a full batch
        {"name": "tables_64x1", "kind": "tables", "requests": 64, "tokens": 1, "context": 2000, "page": PAGE},
        # prompts side by side, behind long contexts
        {"name": "tables_32x250", "kind": "tables", "requests": 32, "tokens": 250, "context": 12000, "page": PAGE},
    ]


def _log(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    kind = rng.choice(["write", "rows", "rows", "portions", "portions", "select", "reorder", "tables"])
    heads, page = rng.choice(sorted(HEADS)), rng.choice([8, 16, 32, 64])
    if kind == "write":
        return {"kind": kind, "heads": heads, "tokens": _log(rng, 1, 2000), "context": _log(rng, 1, 30000),
                "dtype": rng.choice(["bfloat16", "float32"]), "pairing": rng.choice([0, 1]), "page": page}
    if kind == "rows":
        requests = _log(rng, 1, 64)
        return {"kind": kind, "heads": heads, "requests": requests, "context": _log(rng, 1, min(30000, 120000 // requests)),
                "ragged": rng.choice([True, False]), "page": page}
    if kind == "portions":
        requests = _log(rng, 1, 12)
        return {"kind": kind, "heads": heads, "requests": requests, "tokens": _log(rng, 2, 2000 // requests),
                "context": _log(rng, 1, 6000 // requests), "ragged": rng.choice([True, False]), "page": page}
    if kind == "select":
        beams = rng.randint(1, 16)
        return {"kind": kind, "requests": _log(rng, 1, 256 // beams), "beams": beams, "vocabulary": _log(rng, 1000, VOCABULARY)}
    if kind == "reorder":
        beams = rng.randint(2, 16)
        return {"kind": kind, "heads": heads, "layers": rng.randint(1, 28), "requests": _log(rng, 1, 96 // beams), "beams": beams,
                "context": _log(rng, 1, 1000), "page": rng.choice([8, 16]), "states": rng.choice([True, False])}
    requests = _log(rng, 1, 64)
    return {"kind": kind, "requests": requests, "tokens": _log(rng, 1, 8000 // requests), "context": _log(rng, 1, 12000), "page": page}


# ------------------------------------------------------------------ inputs
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _spread(total: int, requests: int, ragged: bool, g) -> torch.Tensor:
    """Lengths of the requests: all alike, or spread evenly from half to one and a half times the number, in any order."""
    if not ragged:
        return torch.full((requests,), total, dtype=torch.int64, device="cuda")
    factor = 0.5 + (torch.randperm(requests, generator=g, device="cuda").double() + 0.5) / requests
    return (factor * total).round().long().clamp_(min=1)


def _half_steps(x: torch.Tensor):
    """Codes, scales and centres of rows of values (in the type that they come in)."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high - low) / 15).float().bfloat16().to(x.dtype)
    centre = (low + 8 * scale).float().bfloat16().to(x.dtype)
    step = torch.where(scale == 0, torch.zeros_like(x), (x - centre) / torch.where(scale == 0, torch.ones_like(scale), scale))
    return (torch.round(step) + 8).clamp_(0, 15).to(torch.uint8), torch.cat([scale, centre], -1).bfloat16()


def _pack(codes: torch.Tensor) -> torch.Tensor:
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _values(codes: torch.Tensor, scales: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """What packed codes and their scales stand for."""
    wide = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(dtype)
    return (wide - 8) * scales[..., :1].to(dtype) + scales[..., 1:].to(dtype)


def _cache(pages: int, n_kv: int, page: int, dim: int, g):
    """Pages of keys and values as a model leaves them: bell-shaped rows, channels with a level of their own."""
    made = []
    for _ in range(2):
        level = 0.5 * torch.randn((1, n_kv, 1, dim), generator=g, device="cuda")
        codes, scales = _half_steps(torch.randn((pages, n_kv, page, dim), generator=g, device="cuda") + level)
        made += [_pack(codes), scales]
    return made


def _tables(lengths: torch.Tensor, page: int, g):
    """Block tables of requests that hold so many tokens: pages in no order, -1 behind the last one; and how many pages there are."""
    held = (lengths + page - 1) // page
    width, total = int(held.max()), int(held.sum())
    pages = torch.randperm(total, generator=g, device="cuda")
    inside = torch.arange(width, device="cuda")[None, :] < held[:, None]
    tables = torch.full((lengths.shape[0], width), -1, dtype=torch.int64, device="cuda")
    tables[inside] = pages
    return tables.int(), total


def _ints(values) -> torch.Tensor:
    return torch.as_tensor(values, device="cuda").int()


def prepare(case: dict, seed: int) -> dict:
    return globals()["_prepare_" + case["kind"]](case, _generator(seed))


def _prepare_write(case, g):
    n_q, n_kv, dim = HEADS[case["heads"]]
    tokens, page, width = case["tokens"], case["page"], (n_q + 2 * n_kv) * dim
    pages = 2 * (-(-tokens // page)) + 8
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    qkv = torch.randn((tokens, width), generator=g, device="cuda").to(getattr(torch, case["dtype"]))
    positions = torch.randint(0, case["context"] + 1, (1,), generator=g, device="cuda") + torch.arange(tokens, device="cuda")
    k_codes, k_scales, v_codes, v_scales = _cache(pages, n_kv, page, dim, g)
    return {"case": case, "qkv": qkv, "bias": torch.randn(width, generator=g, device="cuda"), "positions": positions.int(),
            "slots": slots.int(), "inv_freq": (THETA ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)).float(),
            "k_codes": k_codes, "k_scales": k_scales, "v_codes": v_codes, "v_scales": v_scales,
            "q": torch.empty((tokens, n_q, dim), dtype=torch.bfloat16, device="cuda"),
            "k": torch.empty((tokens, n_kv, dim), dtype=torch.bfloat16, device="cuda"),
            "v": torch.empty((tokens, n_kv, dim), dtype=torch.bfloat16, device="cuda")}


def _prepare_attention(case, g, counts, contexts):
    n_q, n_kv, dim = HEADS[case["heads"]]
    tables, pages = _tables(contexts, case["page"], g)
    k_codes, k_scales, v_codes, v_scales = _cache(pages, n_kv, case["page"], dim, g)
    tokens = int(counts.sum())
    segments = torch.repeat_interleave(torch.arange(counts.shape[0], device="cuda"), counts)
    start = torch.cat([torch.zeros_like(counts[:1]), counts.cumsum(0)])
    first = contexts - counts
    positions = first[segments] + torch.arange(tokens, device="cuda") - start[segments]
    q = torch.randn((tokens, n_q, dim), generator=g, device="cuda").bfloat16()
    return {"case": case, "q": q, "out": torch.empty_like(q), "k_codes": k_codes, "k_scales": k_scales, "v_codes": v_codes,
            "v_scales": v_scales, "tables": tables, "segments": segments.int(), "positions": positions.int(), "start": start.int(),
            "first": first.int(), "scale": dim ** -0.5, "longest": int(contexts.max()), "keys": int(contexts.sum()),
            "most": int(counts.max())}


def _prepare_rows(case, g):
    contexts = _spread(case["context"], case["requests"], case["ragged"], g)
    return _prepare_attention(case, g, torch.ones_like(contexts), contexts)


def _prepare_portions(case, g):
    counts = _spread(case["tokens"], case["requests"], case["ragged"], g)
    return _prepare_attention(case, g, counts, counts + _spread(case["context"], case["requests"], case["ragged"], g))


def _prepare_select(case, g):
    requests, beams, vocabulary = case["requests"], case["beams"], case["vocabulary"]
    # a model's logits: most tokens far below a few; beams that have lost a few nats on their way, one in ten at its end
    logits = 2.5 * torch.randn((requests * beams, vocabulary), generator=g, device="cuda")
    scores = -5 * torch.rand((requests, beams), generator=g, device="cuda") - 1
    ended = torch.rand((requests, beams), generator=g, device="cuda") < 0.1
    out = (requests, beams)
    return {"case": case, "logits": logits, "scores": scores, "ended": ended.int(), "end_token": 7,
            "out_scores": torch.empty(out, device="cuda"), "out_tokens": torch.empty(out, dtype=torch.int32, device="cuda"),
            "out_parents": torch.empty(out, dtype=torch.int32, device="cuda"), "out_ended": torch.empty(out, dtype=torch.int32, device="cuda")}


def _prepare_reorder(case, g):
    n_q, n_kv, dim = HEADS[case["heads"]]
    requests, beams = case["requests"], case["beams"]
    rows = requests * beams
    # beams of high score have several children, many have none
    parents = (beams * torch.rand((requests, beams), generator=g, device="cuda") ** 2).long().clamp_(max=beams - 1)
    if case["states"]:   # the slots of a fixed-size state: a table of one page of which a part is used
        tables, lengths, page, slots = torch.randperm(rows, generator=g, device="cuda").int()[:, None], torch.ones(requests, device="cuda"), 2, rows
        storage = torch.randn((case["layers"], slots, n_q, dim, 4), generator=g, device="cuda")
    else:
        page = case["page"]
        lengths = _spread(case["context"], requests, True, g)
        # the full pages of the beams are shared already; from the one that is being filled on, every beam has its own
        width = int(lengths.max()) // page + 2
        shared = torch.randint(0, rows, (requests, 1, width), generator=g, device="cuda").expand(requests, beams, width)
        mine = (1 + torch.arange(width, device="cuda"))[None, None, :] % 2 * rows + torch.randperm(rows, generator=g, device="cuda").view(requests, beams, 1)
        at = torch.arange(width, device="cuda")[None, None, :]
        tables = torch.where(at < (lengths // page)[:, None, None], shared, mine).reshape(rows, width).int()
        storage = torch.randn((2 * case["layers"], 2 * rows, n_kv, page, dim), generator=g, device="cuda", dtype=torch.bfloat16)
    return {"case": case, "parents": parents.int(), "tables": tables.contiguous(), "lengths": lengths.int(), "page": page, "storage": storage,
            "new_tables": torch.empty_like(tables)}


def _prepare_tables(case, g):
    requests, page = case["requests"], case["page"]
    counts = _spread(case["tokens"], requests, case["tokens"] > 1, g)
    first = _spread(case["context"], requests, True, g)
    held = (first + counts + page - 1) // page
    tokens, width = int(counts.sum()), -(-(3 * (case["tokens"] + case["context"]) // 2 + 2) // page)     # room for the longest
    start = torch.cat([torch.zeros_like(held[:1]), held.cumsum(0)])
    ints = {"dtype": torch.int32, "device": "cuda"}
    return {"case": case, "first": first.int(), "counts": counts.int(), "page_start": start.int(),
            "pages": torch.randperm(int(held.sum()), generator=g, device="cuda").int(),
            "segment_start": torch.empty(requests + 1, **ints), "segments": torch.empty(tokens, **ints), "positions": torch.empty(tokens, **ints),
            "slots": torch.empty(tokens, **ints), "contexts": torch.empty(requests, **ints), "tables": torch.empty((requests, width), **ints)}


# ------------------------------------------------------------------ one pass
def run(state: dict):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


def _ops():
    from llm_serving_engine_b200.kernels import ops

    return ops


def _own_write(s):
    ops, (n_q, n_kv, dim) = _ops(), HEADS[s["case"]["heads"]]
    cache = (s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])
    ops.rope_kv_write_int4(s["qkv"], s["bias"], s["positions"], s["slots"], s["inv_freq"], s["q"], *cache, n_q, n_kv, dim, s["case"]["pairing"])
    ops.kv_read_int4(*cache, s["slots"], s["k"], s["v"])
    return s["q"], s["k"], s["v"]


def _rotated(x, angles, pairing):
    """Rotates x [T, heads, D] by angles [T, D / 2]: neighbouring pairs (pairing 0) or halves (1)."""
    cos, sin = angles.cos()[:, None, :], angles.sin()[:, None, :]
    a, b = (x[..., 0::2], x[..., 1::2]) if pairing == 0 else x.chunk(2, -1)
    turned = [a * cos - b * sin, b * cos + a * sin]
    return torch.stack(turned, -1).flatten(-2) if pairing == 0 else torch.cat(turned, -1)


def _plain_write(s):
    n_q, n_kv, dim = HEADS[s["case"]["heads"]]
    tokens, page = s["qkv"].shape[0], s["case"]["page"]
    # in 64 bits: angles of far positions, and values next to the border between two codes
    x = (s["qkv"].double() + s["bias"].double()).view(tokens, n_q + 2 * n_kv, dim)
    angles = s["positions"].double()[:, None] * s["inv_freq"].double()[None, :]
    turned = _rotated(x[:, :n_q + n_kv], angles, s["case"]["pairing"])
    s["q"].copy_(turned[:, :n_q])
    at, offset = s["slots"].long() // page, s["slots"].long() % page
    heads = torch.arange(n_kv, device=x.device)[None, :]
    k_codes, k_scales = _half_steps(turned[:, n_q:])
    v_codes, v_scales = _half_steps(x[:, n_q + n_kv:])
    place = (at[:, None], heads, offset[:, None])
    s["k_codes"][place], s["k_scales"][place] = _pack(k_codes), k_scales
    s["v_codes"][place], s["v_scales"][place] = _pack(v_codes), v_scales
    s["k"].copy_(_values(s["k_codes"][place], s["k_scales"][place]))
    s["v"].copy_(_values(s["v_codes"][place], s["v_scales"][place]))
    return s["q"], s["k"], s["v"]


def _own_rows(s):
    return _ops().paged_attention_decode_int4(s["q"], s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"], s["out"], s["tables"],
                                              s["segments"], s["positions"], s["scale"], max_context=s["longest"])


def _own_portions(s):
    return _ops().paged_attention_prefill_int4(s["q"], s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"], s["out"], s["tables"],
                                               s["start"], s["first"], s["scale"], keys=s["keys"])


def _gathered(s, name):
    """Values of every request's pages, [S, n_kv, keys, D]; what lies behind a table's last page belongs to nobody."""
    at = s["tables"].long().clamp(min=0)
    return _values(s[name + "_codes"][at], s[name + "_scales"][at]).transpose(1, 2).flatten(2, 3)


def _attended(q, k, v, positions, scale):
    """q [S, C, n_q, D] at positions [S, C] over k, v [S, n_kv, L, D]; every query head reads the head of its group."""
    requests, rows, n_q, dim = q.shape
    n_kv = k.shape[1]
    q = q.view(requests, rows, n_kv, n_q // n_kv, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = (q @ k.transpose(-1, -2) * scale).view(requests, n_kv, n_q // n_kv, rows, -1)
    hidden = torch.arange(k.shape[2], device=q.device)[None, None, :] > positions[:, :, None]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    weights = (scores - scores.amax(-1, keepdim=True)).exp_()
    weights /= weights.sum(-1, keepdim=True)
    return (weights.flatten(2, 3) @ v).view(requests, n_kv, n_q // n_kv, rows, dim).permute(0, 3, 1, 2, 4).flatten(2, 3)


def _plain_rows(s):
    out = _attended(s["q"].float()[:, None], _gathered(s, "k"), _gathered(s, "v"), s["positions"][:, None], s["scale"])
    return s["out"].copy_(out[:, 0])


def _plain_portions(s):
    segments = s["segments"].long()
    offset = torch.arange(segments.shape[0], device=segments.device) - s["start"].long()[segments]
    requests = s["first"].shape[0]
    q = torch.zeros((requests, s["most"], *s["q"].shape[1:]), device=segments.device)
    q[segments, offset] = s["q"].float()
    positions = s["first"][:, None] + torch.arange(s["most"], device=segments.device)[None, :]
    out = _attended(q, _gathered(s, "k"), _gathered(s, "v"), positions, s["scale"])
    return s["out"].copy_(out[segments, offset])


def _own_select(s):
    out = s["out_scores"], s["out_tokens"], s["out_parents"], s["out_ended"]
    _ops().beam_select(s["logits"], s["scores"], s["ended"], s["end_token"], *out)
    return out


def _plain_select(s):
    requests, beams = s["scores"].shape
    logits = s["logits"].view(requests, beams, -1).double()      # candidates of two beams can lie closer than 32 bits tell apart
    offered = s["scores"].double()[..., None] + logits - torch.logsumexp(logits, -1, keepdim=True)
    ended = s["ended"][..., None] != 0
    offered = offered.masked_fill(ended, -math.inf)
    offered[..., s["end_token"]] = torch.where(ended[..., 0], s["scores"].double(), offered[..., s["end_token"]])
    best, at = torch.sort(offered.flatten(1), dim=-1, descending=True, stable=True)
    best, at = best[:, :beams], at[:, :beams]
    parents, tokens = at // logits.shape[-1], at % logits.shape[-1]
    over = (s["ended"].gather(1, parents) != 0) | (tokens == s["end_token"])
    return best.float(), tokens.int(), parents.int(), over.int()


def _own_reorder(s):
    _ops().beam_reorder(s["parents"], s["tables"], s["lengths"], s["new_tables"], s["page"], [s["storage"]])
    return s["new_tables"], s["storage"]


def _plain_reorder(s):
    requests, beams = s["parents"].shape
    parents, tables = s["parents"].long(), s["tables"].view(requests, beams, -1)
    at, page = torch.arange(tables.shape[-1], device=parents.device), s["page"]
    full, filling = (s["lengths"].long() // page)[:, None], (s["lengths"].long() % page != 0)[:, None]
    inherited = tables.gather(1, parents[..., None].expand_as(tables))
    # a beam's first child goes on in the page that the beam was filling; the others take those of the beams without a child
    same = parents[:, :, None] == parents[:, None, :]
    more = same.tril(-1).any(-1)
    childless = ~(parents[:, :, None] == torch.arange(beams, device=parents.device)).any(1)
    free = torch.sort((~childless).int(), dim=1, stable=True).indices
    taker = torch.where(more, free.gather(1, (more.cumsum(1) - 1).clamp(min=0)), parents)
    here = full[..., None].expand(requests, beams, 1).clamp(max=tables.shape[-1] - 1)
    own_page = torch.where(filling, tables.gather(2, here)[..., 0].gather(1, taker), -1)
    source = torch.where(filling, tables.gather(2, here)[..., 0].gather(1, parents), -1)
    new = torch.where(at < full[..., None], inherited, torch.where((at == full[..., None]) & filling[..., None], own_page[..., None], tables))
    moved = more & filling
    s["storage"][:, own_page[moved].long()] = s["storage"][:, source[moved].long()]
    s["new_tables"].copy_(new.view_as(s["new_tables"]))
    return s["new_tables"], s["storage"]


def _own_tables(s):
    out = s["segment_start"], s["segments"], s["positions"], s["slots"], s["contexts"], s["tables"]
    _ops().step_tables(s["first"], s["counts"], s["pages"], s["page_start"], s["case"]["page"], *out)
    return out


def _plain_tables(s):
    counts, page = s["counts"].long(), s["case"]["page"]
    tokens, device = s["segments"].shape[0], counts.device
    start = torch.cat([torch.zeros_like(counts[:1]), counts.cumsum(0)])
    row = torch.arange(tokens, device=device)
    segments = torch.searchsorted(start[1:].contiguous(), row, right=True)
    positions = s["first"].long()[segments] + row - start[segments]
    held = s["page_start"].long()
    slots = s["pages"].long()[held[segments] + positions // page] * page + positions % page
    at = torch.arange(s["tables"].shape[1], device=device)[None, :] + held[:-1, None]
    tables = torch.where(at < held[1:, None], s["pages"][at.clamp(max=s["pages"].shape[0] - 1)], -1)
    return start.int(), segments.int(), positions.int(), slots.int(), (s["first"] + s["counts"]).int(), tables.int()


# ------------------------------------------------------------------ what a pass cannot do without
def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "select":
        rows = case["requests"] * case["beams"]
        return {"bytes": 4 * rows * (case["vocabulary"] + 6), "flops": 3 * rows * case["vocabulary"]}
    if kind == "tables":
        held = case["requests"] * (-(-(case["context"] + case["tokens"]) // case["page"]))
        return {"bytes": 4 * (3 * case["requests"] * case["tokens"] + 2 * held + 5 * case["requests"]), "flops": 0}
    n_q, n_kv, dim = HEADS[case["heads"]]
    row = 2 * n_kv * (dim // 2 + 4)          # a token's keys and values in the cache
    if kind == "write":
        tokens, size = case["tokens"], 4 if case["dtype"] == "float32" else 2
        return {"bytes": tokens * ((n_q + 2 * n_kv) * dim * size + n_q * dim * 2 + 2 * row + 4 * n_kv * dim), "flops": 6 * tokens * (n_q + 2 * n_kv) * dim}
    if kind == "reorder":
        # of the children of random parents about a third is a second child; tables are read and written
        state = case["layers"] * (n_q * dim * 16 if case["states"] else 4 * n_kv * case["page"] * dim)
        rows = case["requests"] * case["beams"]
        width = 1 if case["states"] else case["context"] // case["page"] + 2
        return {"bytes": 2 * (rows // 3) * state + 8 * rows * width, "flops": 0}
    tokens, requests = case.get("tokens", 1), case["requests"]
    context = case["context"] + (tokens if kind == "portions" else 0)
    pairs = requests * tokens * (context - (tokens - 1) / 2)
    return {"bytes": requests * (context * row + 4 * tokens * n_q * dim), "flops": int(4 * n_q * dim * pairs)}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case: dict, seed: int):
    return globals()["_exact_" + case["kind"]](prepare(case, seed))


def _held(rows: torch.Tensor) -> torch.Tensor:
    """What rows of values (float64) become in the cache."""
    low, high = rows.min(-1).values, rows.max(-1).values
    scale = ((high - low) / 15.0).to(torch.float32).to(torch.bfloat16).to(torch.float64)
    centre = (low + 8.0 * scale).to(torch.float32).to(torch.bfloat16).to(torch.float64)
    steps = torch.nan_to_num((rows - centre[..., None]) / scale[..., None], nan=0.0, posinf=0.0, neginf=0.0)
    return scale[..., None] * torch.clamp(torch.round(steps), -8.0, 7.0) + centre[..., None]


def _exact_write(s):
    n_q, n_kv, dim = HEADS[s["case"]["heads"]]
    x = (s["qkv"].to(torch.float64) + s["bias"].to(torch.float64)).reshape(-1, n_q + 2 * n_kv, dim)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       torch.outer(s["positions"].to(torch.float64), s["inv_freq"].to(torch.float64)))[:, None, :]
    heads = x[:, :n_q + n_kv]
    if s["case"]["pairing"] == 0:
        turned = torch.view_as_real(torch.view_as_complex(heads.reshape(*heads.shape[:-1], dim // 2, 2).contiguous()) * turn).flatten(-2)
    else:
        pairs = torch.complex(heads[..., :dim // 2].contiguous(), heads[..., dim // 2:].contiguous()) * turn
        turned = torch.cat([pairs.real, pairs.imag], dim=-1)
    return turned[:, :n_q], _held(turned[:, n_q:]), _held(x[:, n_q + n_kv:])


def _exact_keys(s, name, request, head, length):
    """Keys (or values) of one request and head, [length, D], float64."""
    page = s["case"]["page"]
    at = s["tables"][request, : -(-length // page)].long()
    codes, scales = s[name + "_codes"][at, head], s[name + "_scales"][at, head].to(torch.float64)
    low, high = torch.remainder(codes, 16), torch.div(codes, 16, rounding_mode="floor")
    u = torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=torch.float64, device=codes.device)
    u[..., 0::2], u[..., 1::2] = low.to(torch.float64), high.to(torch.float64)
    return ((u - 8.0) * scales[..., 0, None] + scales[..., 1, None]).reshape(-1, u.shape[-1])[:length]


def _exact_attention(s):
    n_q, n_kv, dim = HEADS[s["case"]["heads"]]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    starts = s["start"].tolist()
    for request, first in enumerate(s["first"].tolist()):
        low, high = starts[request], starts[request + 1]
        length = first + high - low
        for head in range(n_kv):
            k, v = (_exact_keys(s, name, request, head, length) for name in ("k", "v"))
            mine = slice(head * (n_q // n_kv), (head + 1) * (n_q // n_kv))
            scores = torch.einsum("rhd,ld->rhl", s["q"][low:high, mine].to(torch.float64), k) / math.sqrt(dim)
            seen = torch.arange(length, device=k.device)[None, :] <= torch.arange(first, length, device=k.device)[:, None]
            scores = torch.where(seen[:, None, :], scores, torch.full_like(scores, -math.inf))
            out[low:high, mine] = torch.einsum("rhl,ld->rhd", torch.softmax(scores, -1), v)
    return out


_exact_rows = _exact_portions = _exact_attention


def _exact_select(s):
    """A request's continuations are sorted on the host, after those that cannot be among the best of their own beam are left out."""
    requests, beams = s["scores"].shape
    picked = [[], [], [], []]
    for request in range(requests):
        found = []
        for beam in range(beams):
            score = float(s["scores"][request, beam])
            if int(s["ended"][request, beam]):
                found.append((-score, beam, s["end_token"]))
                continue
            row = s["logits"][request * beams + beam].to(torch.float64)
            logs = torch.log_softmax(row, 0)
            least = torch.topk(row, min(beams, row.shape[0])).values[-1]
            for token in torch.nonzero(row >= least)[:, 0].tolist():
                found.append((-(score + float(logs[token])), beam, token))
        found.sort()
        for value, beam, token in found[:beams]:
            over = bool(int(s["ended"][request, beam])) or token == s["end_token"]
            for column, number in zip(picked, (-value, token, beam, int(over))):
                column.append(number)
    kinds = torch.float64, torch.int32, torch.int32, torch.int32
    return tuple(torch.tensor(column, dtype=kind, device=s["scores"].device).view(requests, beams) for column, kind in zip(picked, kinds))


def _exact_reorder(s):
    requests, beams = s["parents"].shape
    old, page = s["tables"].cpu().tolist(), s["page"]
    new, pairs = [list(row) for row in old], []
    for request, (parents, length) in enumerate(zip(s["parents"].tolist(), s["lengths"].tolist())):
        full, rest = divmod(length, page)
        free = [beam for beam in range(beams) if beam not in parents]
        seen = set()
        for beam, parent in enumerate(parents):
            row, source = new[request * beams + beam], old[request * beams + parent]
            row[:full] = source[:full]
            if rest:
                row[full] = source[full]
                if parent in seen:
                    row[full] = old[request * beams + free.pop(0)][full]
                    pairs.append((source[full], row[full]))
                seen.add(parent)
    storage = s["storage"].clone()
    for source, target in pairs:
        storage[:, target] = s["storage"][:, source]
    return torch.tensor(new, device=storage.device).int(), storage.double() if storage.numel() < 1 << 28 else None


def _exact_tables(s):
    return None
