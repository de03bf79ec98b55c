"""Operators at the end of a decode step, as programs call them: the append to a cache held in 8 bits, attention over that cache,
and sampling.

Kinds of case:
  append     ``cache8.append``: bias and rotation on the fused q|k|v rows, queries out, keys and values into the cache
  attention  ``cache8.attention``: single tokens, a few tokens, and portions of prompts; windows; ragged batches
  sample     ``sampling.sample``: temperature, top-k, top-p and min-p a row, from given random numbers

A cache holds blocks of 64 tokens: e4m3 codes and a power of two for each full block and head, and the FP16 rows of the two newest blocks.
Head layouts and vocabularies are those of ``perf/cases.py`` and generic ones.
"""
from __future__ import annotations

import math
import zlib

import numpy as np
import torch

own = False

DEV = "cuda"
BLOCK = 64                      # tokens
CODE = torch.float8_e4m3fn
MOST_CODE = 448.0
LOGITS = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _case(name, kind, seqs, heads, kv_heads, dim, context, rows=1, ragged=False, window=0):
    return {"name": name, "kind": kind, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim, "context": context, "rows": rows,
            "ragged": ragged, "window": window}


def listed():
    return [
        # one user's token behind 2048 others, 7b heads: latency
        _case("append_1_token", "append", 1, 28, 4, 128, 2048),
        # a batch decoding, every sequence at a place of its own
        _case("append_96_tokens_ragged", "append", 96, 40, 8, 128, 4000, ragged=True),
        # a document's portion into an empty cache
        _case("append_prompt_4000", "append", 1, 28, 4, 128, 0, rows=4000),
        # the same user's token: latency, work split over the keys
        _case("decode_1x2049", "attention", 1, 28, 4, 128, 2048),
        # one long context: the whole cache of the sequence is read by a few heads
        _case("decode_1x100000", "attention", 1, 16, 4, 128, 100000),
        # a serving batch, all lengths
        _case("decode_96x6000_ragged", "attention", 96, 40, 8, 128, 6000, ragged=True),
        # guessed tokens checked four at a time, small heads, a window
        _case("check_4_of_40x3000_window", "attention", 40, 16, 8, 64, 3000, rows=4, ragged=True, window=1024),
        # a document's prompt
        _case("prompt_4000", "attention", 1, 28, 4, 128, 0, rows=4000),
        # portions of prompts behind what their sequences hold, odd lengths
        _case("portions_3x500_on_9000", "attention", 3, 16, 4, 128, 9000, rows=500, ragged=True),
        # one token of one sequence with the usual settings: latency
        {"name": "sample_1x152064", "kind": "sample", "rows": 1, "vocab": 152064, "dtype": "float32", "mode": "all"},
        # a batch with settings of its own a row, half of them greedy or plain
        {"name": "sample_64x32768_mixed", "kind": "sample", "rows": 64, "vocab": 32768, "dtype": "bfloat16", "mode": "mixed"},
        # a large batch on a large vocabulary
        {"name": "sample_250x152064_top_p", "kind": "sample", "rows": 250, "vocab": 152064, "dtype": "float32", "mode": "top_p"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "sample"])
    if kind == "sample":
        rows = _log(rng, 1, 250)
        return {"kind": kind, "rows": rows, "vocab": _log(rng, 100, min(262144, 38000000 // rows)), "dtype": rng.choice(["float32", "float16", "bfloat16"]),
                "mode": rng.choice(["all", "mixed", "top_p", "top_k", "min_p", "plain"])}
    heads, kv_heads = rng.choice([(28, 4), (16, 4), (40, 8), (8, 8), (16, 1), (12, 2), (71, 1)])
    case = {"kind": kind, "seqs": _log(rng, 1, 128), "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([64, 128, 128]), "context": _log(rng, 1, 100000),
            "rows": rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 4000)]), "ragged": rng.random() < 0.7, "window": 0}
    if kind == "attention" and rng.random() < 0.3:
        case["window"] = _log(rng, 16, 4096)
    if kind == "append" and case["rows"] > BLOCK:
        case["context"] = case["context"] // BLOCK * BLOCK
    most = work(next(c for c in listed() if c["name"] == "prompt_4000"))["flops"], work(next(c for c in listed() if c["name"] == "decode_96x6000_ragged"))["bytes"]
    while case["seqs"] > 1 and _costs(case, *most):
        case["seqs"] = case["seqs"] * 2 // 3
    while case["rows"] > 1 and _costs(case, *most):
        case["rows"] = max(1, case["rows"] * 2 // 3)
    return case


def _costs(case, flops, size):
    """Whether a drawn case is over the largest listed ones: work, the cache that it holds, and the plain form's scores."""
    w, lengths = work(case), _lengths(case)
    n, longest = len(lengths), max(a + r for a, r in lengths)
    scores = n * case["heads"] * max(r for _, r in lengths) * longest if case["kind"] == "attention" else 0
    return w["flops"] > flops or w["bytes"] > size or 2 * n * case["kv_heads"] * longest * case["dim"] > 3 * size or scores > 600e6


def _generator(*key):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(key).encode()))


# ------------------------------------------------------------------------------------------------------------ shapes --

def _lengths(case):
    """(tokens in the cache before the call, new tokens) of every sequence."""
    out = []
    for s in range(case["seqs"]):
        part = 0.25 + 0.75 * (0.618 * (s + 1) % 1.0) if case["ragged"] else 1.0
        start, rows = int(case["context"] * part), max(1, int(case["rows"] * (1.25 - part))) if case["rows"] > 1 and case["ragged"] else case["rows"]
        if case["kind"] == "append" and case["rows"] > BLOCK:
            start = start // BLOCK * BLOCK
        out.append((start, rows))
    return out


def _capacity(case):
    return -(-max(a + r for a, r in _lengths(case)) // BLOCK) * BLOCK


def _padding(case):
    return 3 if case["ragged"] else 0               # rows behind the last sequence's


def _pairs(case):
    """Queries times the keys that they see."""
    n = 0
    for start, rows in _lengths(case):
        if case["window"]:
            n += sum(min(p + 1, case["window"]) for p in range(start, start + rows))
        else:
            n += rows * start + rows * (rows + 1) // 2
    return n


def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * LOGITS[case["dtype"]].itemsize + 8 * case["rows"], "flops": 8 * n}
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    lengths = _lengths(case)
    rows = sum(r for _, r in lengths)
    if case["kind"] == "append":
        full = sum((a + r) // BLOCK * BLOCK - a // BLOCK * BLOCK for a, r in lengths if (a + r) // BLOCK > a // BLOCK)
        return {"bytes": rows * (2 * hq + 2 * hk) * d * 2 + full * 2 * hk * d + min(rows, 2 * BLOCK * len(lengths)) * 2 * hk * d * 2,
                "flops": 6 * rows * (hq + 2 * hk) * d}
    seen = sum(a + r - max(0, a + 1 - case["window"]) if case["window"] else a + r for a, r in lengths)
    return {"bytes": seen * 2 * hk * d + 2 * rows * hq * d * 2, "flops": 4 * d * hq * _pairs(case)}


# ------------------------------------------------------------------------------------------------------------- cache --

def _scales(x):
    """x: [..., BLOCK, dim] in 32 bits.  The smallest power of two that brings the largest finite value to at most 448; 1 for zeros."""
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(dim=(-1, -2))
    frac, exp = torch.frexp(top)                    # top = frac * 2^exp, 0.5 <= frac < 1
    return torch.where(top > 0, torch.ldexp(torch.ones_like(top), exp - 9 + (frac > 0.875).int()), 1.0)


def _codes(x, scale):
    y = x / scale[..., None, None]
    return torch.where(torch.isfinite(y), y, math.nan).to(CODE)


def _empty_cache(case):
    s, h, d, cap = case["seqs"], case["kv_heads"], case["dim"], _capacity(case)
    side = lambda: (torch.zeros((s, h, cap, d), device=DEV, dtype=torch.uint8).view(CODE), torch.ones((s, h, cap // BLOCK), device=DEV),  # noqa: E731
                    torch.zeros((s, h, 2, BLOCK, d), device=DEV, dtype=torch.float16))
    (k, ks, kt), (v, vs, vt) = side(), side()
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "k_tail": kt, "v_tail": vt}


def _fill(cache, name, seq, length, x):
    """x: [heads, length, dim] f16 into sequence `seq`."""
    full = length // BLOCK
    if full:
        blocks = x[:, :full * BLOCK].float().unflatten(1, (full, BLOCK))
        scale = _scales(blocks)
        cache[name + "_scale"][seq, :, :full] = scale
        cache[name].view(torch.uint8)[seq, :, :full * BLOCK] = _codes(blocks, scale).view(torch.uint8).flatten(1, 2)
    for b in range(max(0, -(-length // BLOCK) - 2), -(-length // BLOCK)):
        rows = x[:, b * BLOCK:(b + 1) * BLOCK]
        cache[name + "_tail"][seq, :, b % 2, :rows.shape[1]] = rows


def _keys(gen, heads, n, dim):
    """Keys and values as a model has them: some channels are several times larger than the others."""
    x = torch.randn((heads, n, dim), generator=gen, device=DEV)
    channel = torch.randn((heads, 1, dim), generator=gen, device=DEV).mul_(0.6).exp_()
    return (x * channel).half()


def _rope(positions, dim):
    """cos | sin of every position, [positions, dim]."""
    angle = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(dim // 2, device=DEV, dtype=torch.float64) * 2 / dim)
    return torch.cat((angle.cos(), angle.sin()), dim=1).float()


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _prepare_cache(case, seed):
    gen = _generator(case["kind"], seed)
    lengths, hq, hk, d = _lengths(case), case["heads"], case["kv_heads"], case["dim"]
    attention = case["kind"] == "attention"
    rows = sum(r for _, r in lengths)
    row_start = [0]
    for _, r in lengths:
        row_start.append(row_start[-1] + r)
    state = {"case": case, "lengths": lengths, "cache": _empty_cache(case), "start": _int([a for a, _ in lengths]), "row_start": _int(row_start),
             "max_rows": max(r for _, r in lengths)}
    for name in ("k", "v"):
        for s, (a, r) in enumerate(lengths):
            n = a + r if attention else a
            if n:
                _fill(state["cache"], name, s, n, _keys(gen, hk, n, d))
    total = rows + _padding(case)
    if attention:
        state["q"] = (2.0 * torch.randn((total, hq * d), generator=gen, device=DEV)).half()
        state["scale"] = 1.0 / math.sqrt(d)
    else:
        state["qkv"] = torch.randn((total, (hq + 2 * hk) * d), generator=gen, device=DEV).half()
        state["bias"] = 0.5 * torch.randn((hq + 2 * hk) * d, generator=gen, device=DEV)
        state["rope"] = _rope(_capacity(case), d)
    state["out"] = torch.zeros((total, hq * d), dtype=torch.float16, device=DEV)
    # the plain form's places: sequence and position of every row, and every row's place in a batch of equal lengths
    seq = torch.repeat_interleave(torch.arange(len(lengths), device=DEV), state["row_start"].diff().long(), output_size=rows)
    place = torch.arange(rows, device=DEV) - state["row_start"][seq].long()
    state.update(seq=seq, place=place, position=state["start"][seq].long() + place)
    if own:
        from tensorwarp_b200 import cache8
        c = state["cache"]
        state["handle"] = cache8.Cache8(**c)
        if attention:
            state["workspace"] = cache8.Workspace.for_cache(state["handle"], num_heads=hq, max_rows=state["max_rows"])
    return state


def _turned(x, table):
    """Rotate-half of [rows, heads, dim] by [rows, dim] of cos | sin."""
    half = x.shape[-1] // 2
    c, s = table[:, None, :half], table[:, None, half:]
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * c - b * s, a * s + b * c), dim=-1)


def _run_append(state):
    case, cache = state["case"], state["cache"]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if own:
        from tensorwarp_b200 import cache8
        cache8.append(state["handle"], state["qkv"], state["out"], state["start"], num_heads=hq, row_start=state["row_start"], max_rows=state["max_rows"],
                      bias=state["bias"], rope=state["rope"])
        return {"q": state["out"], **cache}
    seq, position = state["seq"], state["position"]
    n = seq.numel()
    x = (state["qkv"][:n].float() + state["bias"]).unflatten(1, (hq + 2 * hk, d))
    turned = _turned(x[:, :hq + hk], state["rope"][position])
    state["out"][:n] = turned[:, :hq].flatten(1).half()
    # all touched blocks of all sequences, whole: what is held in 16 bits, with the new rows put in
    touched = -(-(state["max_rows"] + BLOCK - 1) // BLOCK)
    first = state["start"].long() // BLOCK
    block = first[:, None] + torch.arange(touched, device=DEV)
    length = (state["start"] + state["row_start"].diff()).long()
    full = (block + 1) * BLOCK <= length[:, None]
    here = position // BLOCK - first[seq]
    at = torch.nonzero(full)
    for name, new in (("k", turned[:, hq:].half()), ("v", x[:, hq + hk:].half())):
        tail = cache[name + "_tail"]
        rows = torch.zeros((case["seqs"], touched, BLOCK, hk, d), dtype=torch.float16, device=DEV)
        rows[:, 0] = tail[torch.arange(case["seqs"], device=DEV), :, first % 2].transpose(1, 2)
        rows[seq, here, position % BLOCK] = new
        kept = position >= (-(-length // BLOCK) * BLOCK - 2 * BLOCK)[seq]
        tail[seq[kept], :, (position // BLOCK % 2)[kept], (position % BLOCK)[kept]] = new[kept]
        if at.shape[0]:
            blocks = rows[at[:, 0], at[:, 1]].transpose(1, 2).float()                   # [full blocks, heads, BLOCK, dim]
            scale = _scales(blocks)
            number = block[at[:, 0], at[:, 1]]
            cache[name + "_scale"][at[:, 0], :, number] = scale
            cache[name].view(torch.uint8).unflatten(2, (-1, BLOCK))[at[:, 0], :, number] = _codes(blocks, scale).view(torch.uint8)
    return {"q": state["out"], **cache}


def _values(state, name, dtype):
    """[sequences, heads, capacity, dim] of what the cache stands for."""
    cache, case = state["cache"], state["case"]
    x = cache[name].to(dtype).unflatten(2, (-1, BLOCK)) * cache[name + "_scale"].to(dtype)[..., None, None]
    length = (state["start"] + state["row_start"].diff()).long()
    last = length // BLOCK
    s = torch.nonzero(length % BLOCK)[:, 0]
    x[s, :, last[s]] = cache[name + "_tail"][s, :, last[s] % 2].to(dtype)
    return x.flatten(2, 3)


def _run_attention(state):
    case = state["case"]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if own:
        from tensorwarp_b200 import cache8
        cache8.attention(state["handle"], state["q"], state["out"], state["start"], num_heads=hq, row_start=state["row_start"], max_rows=state["max_rows"],
                         scale=state["scale"], window=case["window"], workspace=state["workspace"])
        return state["out"]
    seq, place, n, most = state["seq"], state["place"], state["seq"].numel(), state["max_rows"]
    q = torch.zeros((case["seqs"], most, hk, hq // hk, d), device=DEV)
    q[seq, place] = state["q"][:n].float().unflatten(1, (hk, hq // hk, d))
    position = torch.full((case["seqs"], most), -1, device=DEV)
    position[seq, place] = state["position"]
    scores = torch.einsum("srhgd,shld->shrgl", q, _values(state, "k", torch.float32)).mul_(state["scale"])
    behind = position[:, :, None] - torch.arange(_capacity(case), device=DEV)
    hidden = behind < 0
    if case["window"]:
        hidden |= behind >= case["window"]
    scores.masked_fill_(hidden[:, None, :, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    weight = scores.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    # what the rows of padding and the hidden keys hold is not looked at
    value = torch.where((torch.arange(_capacity(case), device=DEV) < (state["start"] + state["row_start"].diff())[:, None])[:, None, :, None],
                        _values(state, "v", torch.float32), 0.0)
    out = torch.einsum("shrgl,shld->srhgd", weight, value) / weight.sum(dim=-1).permute(0, 2, 1, 3)[..., None].clamp_min(1e-30)
    state["out"][:n] = out[seq, place].flatten(1).half()
    return state["out"]


# ---------------------------------------------------------------------------------------------------------- sampling --

#: temperature, top-k, top-p, min-p of the rows of a case, in turn
SETTINGS = {
    "all": [(0.7, 50, 0.9, 0.02)],
    "mixed": [(0.0, 0, 1.0, 0.0), (0.7, 50, 0.95, 0.0), (1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.9, 0, 0.92, 0.05), (1.0, 400, 1.0, 0.0), (1.3, 0, 0.99, 0.0),
              (1.0, 0, 1.0, 0.1)],
    "top_p": [(1.0, 0, 0.95, 0.0), (0.6, 0, 0.9, 0.0), (1.5, 0, 0.8, 0.0)],
    "top_k": [(1.0, 40, 1.0, 0.0), (0.8, 1, 1.0, 0.0), (1.0, 5000, 1.0, 0.0)],
    "min_p": [(1.0, 0, 1.0, 0.05), (1.5, 0, 1.0, 0.2)],
    "plain": [(1.0, 0, 1.0, 0.0), (0.5, 0, 1.0, 0.0)],
}


def _prepare_sample(case, seed):
    gen = _generator("sample", seed)
    rows, vocab = case["rows"], case["vocab"]
    # what a head gives: a broad floor and, in most rows, a few tokens far above it
    x = torch.randn((rows, vocab), generator=gen, device=DEV).mul_(2.5)
    few = min(20, vocab)
    at = torch.randint(vocab, (rows, few), generator=gen, device=DEV)
    lift = torch.rand((rows, 1), generator=gen, device=DEV) * 14
    x.scatter_add_(1, at, lift * torch.rand((rows, few), generator=gen, device=DEV))
    settings = SETTINGS[case["mode"]]
    column = lambda i, dtype: torch.tensor([settings[r % len(settings)][i] for r in range(rows)], dtype=dtype, device=DEV)  # noqa: E731
    return {"case": case, "logits": x.to(LOGITS[case["dtype"]]), "random": torch.rand(rows, generator=gen, device=DEV), "temperature": column(0, torch.float32),
            "top_k": column(1, torch.int32), "top_p": column(2, torch.float32), "min_p": column(3, torch.float32),
            "tokens": torch.zeros(rows, dtype=torch.int32, device=DEV), "prob": torch.zeros(rows, dtype=torch.float32, device=DEV)}


def _run_sample(state):
    if own:
        from tensorwarp_b200 import sampling
        sampling.sample(state["logits"], state["random"], state["tokens"], temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
                        min_p=state["min_p"], prob=state["prob"])
        return {"tokens": state["tokens"], "prob": state["prob"]}
    # 64 bits: sums of a whole vocabulary, and values next to a border
    z = state["logits"].double()
    t = state["temperature"].double()[:, None]
    value, index = z.sort(dim=1, descending=True, stable=True)
    w = torch.where(t > 0, (value - value[:, :1]) / t.clamp_min(1e-30), 0.0).exp_()
    rank = torch.arange(z.shape[1], device=DEV)
    top_k = state["top_k"].long()[:, None]
    keep = (rank < torch.where(top_k > 0, top_k, z.shape[1])) & ((t > 0) | (rank == 0))
    w = torch.where(keep, w, 0.0)
    before = w.cumsum(dim=1) - w
    top_p = state["top_p"].double()[:, None]
    keep &= (top_p >= 1) | (before < top_p * w.sum(dim=1, keepdim=True)) | (rank == 0)
    keep &= w >= state["min_p"].double()[:, None]
    w = torch.where(keep, w, 0.0)
    back = torch.zeros_like(w).scatter_(1, index, w)
    run = back.cumsum(dim=1)
    token = (run <= state["random"].double()[:, None] * run[:, -1:]).sum(dim=1, keepdim=True)
    last = torch.where(back > 0, rank, 0).amax(dim=1, keepdim=True)
    token = torch.minimum(token, last)
    return {"tokens": token[:, 0].int(), "prob": (back.gather(1, token) / run[:, -1:])[:, 0].float()}


def prepare(case, seed):
    return _prepare_sample(case, seed) if case["kind"] == "sample" else _prepare_cache(case, seed)


def run(state):
    return {"append": _run_append, "attention": _run_attention, "sample": _run_sample}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------------------- exact --

def exact(case, seed):
    if case["kind"] == "sample":
        return _exact_sample(case, seed)
    if work(case)["flops"] > 3e12:
        return None
    return _exact_attention(case, seed) if case["kind"] == "attention" else _exact_append(case, seed)


def _exact_append(case, seed):
    """The queries; codes and scales come from rounded numbers and have no value in more bits."""
    state = _prepare_cache(case, seed)
    hq, d, half = case["heads"], case["dim"], case["dim"] // 2
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device=DEV)
    table = state["rope"].double()
    row = 0
    for start, rows in state["lengths"]:
        x = (state["qkv"][row:row + rows, :hq * d].double() + state["bias"][:hq * d].double()).view(rows, hq, 2, half)
        turn = torch.complex(table[start:start + rows, :half], table[start:start + rows, half:])[:, None]
        y = torch.complex(x[:, :, 0], x[:, :, 1]) * turn
        out[row:row + rows] = torch.stack((y.real, y.imag), dim=2).reshape(rows, hq * d)
        row += rows
    return {"q": out, **{name: None for name in state["cache"]}}


def _exact_attention(case, seed):
    state = _prepare_cache(case, seed)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    cache = state["cache"]
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device=DEV)

    def held(name, s, h, n):
        full = n // BLOCK
        parts = [cache[name][s, h, :full * BLOCK].double() * cache[name + "_scale"][s, h, :full].double().repeat_interleave(BLOCK)[:, None],
                 cache[name + "_tail"][s, h, full % 2, :n - full * BLOCK].double()]
        return torch.cat(parts)

    row = 0
    for s, (start, rows) in enumerate(state["lengths"]):
        n = start + rows
        q = state["q"][row:row + rows].double().view(rows, hq, d)
        far = torch.arange(start, n, device=DEV)[:, None] - torch.arange(n, device=DEV)
        seen = (far >= 0) & (far < (case["window"] or n + 1))
        for h in range(hk):
            k, v = held("k", s, h, n), held("v", s, h, n)
            for j in range(h * (hq // hk), (h + 1) * (hq // hk)):
                x = torch.where(seen, (q[:, j] @ k.T) * state["scale"], -math.inf)
                out[row:row + rows, j * d:(j + 1) * d] = torch.softmax(x, dim=1) @ v
        row += rows
    return out


def _exact_sample(case, seed):
    state = _prepare_sample(case, seed)
    if case["rows"] * case["vocab"] > 50000000:
        return None
    z = state["logits"].double().cpu().numpy()
    u, t, top_k, top_p, min_p = (state[n].double().cpu().numpy() for n in ("random", "temperature", "top_k", "top_p", "min_p"))
    tokens, prob = np.zeros(len(z), np.int32), np.ones(len(z))
    for r, row in enumerate(z):
        if t[r] <= 0:
            tokens[r] = row.argmax()
            continue
        order = np.lexsort((np.arange(row.size), -row))
        if top_k[r] > 0:
            order = order[:int(top_k[r])]
        p = np.exp((row[order] - row[order[0]]) / t[r])
        if top_p[r] < 1:
            run_ = np.concatenate(([0.0], np.cumsum(p)[:-1]))
            order = order[:max(1, int(np.searchsorted(run_, top_p[r] * p.sum(), side="left")))]
        order = order[p[:order.size] >= min_p[r]]
        order.sort()
        p = np.exp((row[order] - row.max()) / t[r])
        at = min(int(np.searchsorted(np.cumsum(p), u[r] * p.sum(), side="right")), order.size - 1)
        tokens[r], prob[r] = order[at], p[at] / p.sum()
    return {"tokens": torch.from_numpy(tokens), "prob": torch.from_numpy(prob)}
