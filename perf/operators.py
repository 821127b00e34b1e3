"""The attention half of a layer between its input projections and its output projection, as a serving program has it done: head
norms and position rotation, keys and values appended to a paged 8-bit cache, and attention over that cache.

A case is a dict of plain values:
  op          norm / append / attention
  heads, kv_heads, dim    of the layer (queries, keys and values, width of a head)
  page        tokens of a cache page
  sequences, rows, context, spread    the batch: `sequences` sequences with up to `rows` new rows each (exactly that many where
              `spread` is 0, else between one and that many) that end at up to `context` tokens
  window      tokens that a query sees (0: all up to its own)
  rotary      width that is rotated; `still`: how many of its pairs have frequency zero (proportional partial rotation)
Inputs are N(0, 1) activations in a joined Q | K | V layout; page tables are random permutations of the pool's pages.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False
EPSILON = 1e-6
TINY = 2.0 ** -64                # the smallest scale of a page

# (query heads, KV heads, head width): the local and global layers of both models, and other programs' layouts
LAYERS = [(16, 8, 256), (16, 2, 512), (32, 16, 256), (32, 4, 512), (32, 8, 128), (24, 8, 128), (16, 1, 128), (7, 7, 128),
          (12, 4, 256), (8, 8, 512)]


def listed():
    return [
        # queries and keys of a decode step of eight sequences, a local layer of the 31B model: latency
        {"name": "norm decode 8", "op": "norm", "heads": 32, "kv_heads": 16, "dim": 256, "rows": 8, "rotary": 256, "still": 0,
         "interleaved": False, "far": 30000},
        # a prompt chunk of a global layer of the 26B model: a quarter of the pairs turn, positions far into the context
        {"name": "norm prompt 4096", "op": "norm", "heads": 16, "kv_heads": 2, "dim": 512, "rows": 4096, "rotary": 512, "still": 192,
         "interleaved": False, "far": 250000},
        # another program's layout: narrow heads, neighbouring pairs, half of the width turned, ragged row count
        {"name": "norm pairs 1025", "op": "norm", "heads": 24, "kv_heads": 8, "dim": 128, "rows": 1025, "rotary": 64, "still": 0,
         "interleaved": True, "far": 100000},
        # one token each of 64 sequences into pages that are partly full (local layer, 31B)
        {"name": "append decode 64", "op": "append", "heads": 32, "kv_heads": 16, "dim": 256, "page": 64, "sequences": 64, "rows": 1,
         "spread": 0, "context": 4000, "rotary": 256, "still": 0, "interleaved": False, "norm": True},
        # a prompt chunk of one sequence (global layer, 31B)
        {"name": "append prompt 4096", "op": "append", "heads": 32, "kv_heads": 4, "dim": 512, "page": 128, "sequences": 1,
         "rows": 4096, "spread": 0, "context": 20011, "rotary": 512, "still": 192, "interleaved": False, "norm": True},
        # a mixed batch, from one row to hundreds, small pages, keys rotated but not normed
        {"name": "append mixed 9", "op": "append", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "sequences": 9, "rows": 700,
         "spread": 1, "context": 3000, "rotary": 128, "still": 0, "interleaved": False, "norm": False},
        # one long sequence, one token (global layer, 26B): the work of few rows spread over the GPU
        {"name": "attention decode 1 long", "op": "attention", "heads": 16, "kv_heads": 2, "dim": 512, "page": 64, "sequences": 1,
         "rows": 1, "spread": 0, "context": 32749, "window": 0},
        # one token each of 64 sequences in a local layer of the 31B model: windows of 1024 tokens that start inside pages
        {"name": "attention decode 64 window", "op": "attention", "heads": 32, "kv_heads": 16, "dim": 256, "page": 64,
         "sequences": 64, "rows": 1, "spread": 0, "context": 4000, "window": 1024},
        # one token each of 24 sequences of very different lengths (global layer, 31B): memory bound
        {"name": "attention decode 24 ragged", "op": "attention", "heads": 32, "kv_heads": 4, "dim": 512, "page": 128,
         "sequences": 24, "rows": 1, "spread": 0, "context": 32000, "window": 0},
        # drafts of up to five tokens that are verified in one pass, small pages, another program's layout
        {"name": "attention verify 16", "op": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "sequences": 16,
         "rows": 5, "spread": 1, "context": 9000, "window": 0},
        # a prompt chunk in a local layer of the 26B model
        {"name": "attention prompt 2048 window", "op": "attention", "heads": 16, "kv_heads": 8, "dim": 256, "page": 64,
         "sequences": 1, "rows": 2048, "spread": 0, "context": 8123, "window": 1024},
        # a prompt chunk in a global layer of the 26B model behind what is cached already: the largest
        {"name": "attention prompt 4096 long", "op": "attention", "heads": 16, "kv_heads": 2, "dim": 512, "page": 128,
         "sequences": 1, "rows": 4096, "spread": 0, "context": 16384, "window": 0},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choices(["norm", "append", "attention"], [25, 25, 50])[0]
    heads, kv_heads, dim = rng.choice(LAYERS)
    case = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim}
    if op != "attention":
        case["interleaved"] = rng.random() < 0.25
        case["rotary"] = rng.choice([dim, dim, dim // 2, dim // 4 + 16])
        case["still"] = 0 if rng.random() < 0.6 else case["rotary"] * 3 // 8
    if op == "norm":
        case["rows"] = _log_uniform(rng, 1, 4096)
        case["far"] = _log_uniform(rng, 100, 500000)
        return case
    case["page"] = rng.choice([16, 32, 64, 128])
    if rng.random() < 0.55:              # a decode step
        case["sequences"], case["rows"], case["spread"] = _log_uniform(rng, 1, 200), 1, 0
    elif rng.random() < 0.4:             # drafts that are verified
        case["sequences"], case["rows"], case["spread"] = _log_uniform(rng, 1, 64), rng.randint(2, 12), 1
    elif rng.random() < 0.5:             # prompts side by side
        case["sequences"], case["rows"], case["spread"] = rng.randint(2, 8), _log_uniform(rng, 40, 600), 1
    else:                                # a chunk of one prompt
        case["sequences"], case["rows"], case["spread"] = 1, _log_uniform(rng, 100, 4096), 0
    if op == "append":
        case["norm"] = rng.random() < 0.7
        case["context"] = max(case["rows"], _log_uniform(rng, 20, 8000 if case["sequences"] < 16 else 1500))
        return case
    # as many cached elements as the largest listed decode step has at most, and as many operations as the largest prompt
    most = min(40000, 20 * 32000 * 4 * 512 // (case["sequences"] * kv_heads * dim))
    if case["rows"] > 16:
        most = min(most, 4 * 10 ** 11 // (case["sequences"] * case["rows"] * heads * dim), 16384)
    case["context"] = max(case["rows"] + 1, _log_uniform(rng, 16, max(17, most)))
    case["window"] = 0 if rng.random() < 0.6 else rng.choice([128, 500, 1024, 4096])
    return case


# --------------------------------------------------------------------------- what a program has in hand

def _lengths(case):
    """(new rows, tokens with them) of every sequence; a case's own, whatever the seed of its inputs."""
    rng = random.Random("%s %s %s" % (case["sequences"], case["rows"], case["context"]))
    news = [rng.randint(1, case["rows"]) if case["spread"] else case["rows"] for _ in range(case["sequences"])]
    low = 0.15 if case["sequences"] > 1 else 1.0
    return [(n, max(n, int(case["context"] * rng.uniform(low, 1.0)))) for n in news]


def _frequencies(case):
    half = case["rotary"] // 2
    f = [1e6 ** (-i / half) for i in range(half - case["still"])] + [0.0] * case["still"]
    return torch.tensor(f, dtype=torch.float64).float().cuda()


def _batch(case, g):
    lengths = _lengths(case)
    page = case["page"]
    offsets = [0]
    for n, _ in lengths:
        offsets.append(offsets[-1] + n)
    needed = [-(-c // page) for _, c in lengths]
    pages = sum(needed) + 3
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(lengths), max(needed) + 2), -1, dtype=torch.int32)
    place = torch.full_like(table, 0)
    at = 0
    for s, n in enumerate(needed):
        place[s, :n] = torch.arange(at, at + n)
        table[s, :n] = 0
        at += n
    table = torch.where(table.cuda() < 0, table.cuda(), order[place.cuda().long()])
    return {"row_offsets": torch.tensor(offsets, dtype=torch.int32).cuda(), "lengths": torch.tensor([c for _, c in lengths], dtype=torch.int32).cuda(),
            "table": table.contiguous(), "pages": pages, "total": offsets[-1], "most": max(n for n, _ in lengths)}


def _cache(case, pages, g):
    """Codes of N(0, 1) keys and values, louder in some pages than in others, and their scales (powers of two)."""
    heads, page, dim = case["kv_heads"], case["page"], case["dim"]
    made = []
    for _ in range(2):
        loud = torch.rand((pages, heads), generator=g, device="cuda").mul_(1.5).sub_(1.0).exp2_()
        scales = torch.exp2(torch.ceil(torch.log2(loud * 5.0 / 448.0)))
        data = torch.empty((pages, heads, page, dim), dtype=torch.uint8, device="cuda")
        for low in range(0, pages, 512):
            part = torch.randn((min(512, pages - low), heads, page, dim), generator=g, device="cuda")
            part.mul_((loud / scales)[low:low + 512, :, None, None]).clamp_(-448.0, 448.0)
            data[low:low + 512] = part.to(torch.float8_e4m3fn).view(torch.uint8)
        made.append((data, scales.contiguous()))
    return made


def _handles(state, case, batch, made):
    """The cache and the batch as the framework's program keeps them from call to call."""
    import gewell_b200 as gw
    (k_data, k_scales), (v_data, v_scales) = made
    state["cache"] = gw.KvCache(k_data, v_data, k_scales, v_scales)
    state["batch"] = gw.SequenceBatch(batch["row_offsets"], batch["lengths"], batch["table"], batch["total"], batch["most"])


def _joined(case, rows, g):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    x = torch.randn((rows, (heads + 2 * kv_heads) * dim), generator=g, device="cuda").bfloat16()
    q, k, v = x.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1)
    return q.unflatten(1, (heads, dim)), k.unflatten(1, (kv_heads, dim)), v.unflatten(1, (kv_heads, dim))


def _weight(case, g):
    return (1.0 + 0.25 * torch.randn(case["dim"], generator=g, device="cuda")).bfloat16()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "norm":
        state["q"], state["k"], _ = _joined(case, case["rows"], g)
        state["q_weight"], state["k_weight"] = _weight(case, g), _weight(case, g)
        state["positions"] = torch.randint(0, case["far"], (case["rows"],), generator=g, device="cuda", dtype=torch.int32)
        state["frequencies"] = _frequencies(case)
        return state
    batch = _batch(case, g)
    made = _cache(case, batch["pages"], g)
    state |= {"b": batch, "k_cache": made[0], "v_cache": made[1]}
    q, k, v = _joined(case, batch["total"], g)
    if case["op"] == "append":
        state["k"], state["v"] = k, v
        state["k_weight"] = _weight(case, g) if case["norm"] else None
        state["frequencies"] = _frequencies(case)
    else:
        state["q"] = (1.5 * q).contiguous()
        state["scale"] = case["dim"] ** -0.5
    if own:
        _handles(state, case, batch, made)
    return state


# --------------------------------------------------------------------------- one pass

def _turned(x, weight, normed, positions, frequencies, interleaved):
    """Norm of every head and rotation, in 32 bits (angles in 64)."""
    x = x.float()
    if normed:
        x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPSILON)
    if weight is not None:
        x = x * weight.float()
    if frequencies is None:
        return x
    half = frequencies.numel()
    angle = positions.double()[:, None] * frequencies.double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _rows_of(b):
    """Sequence and position of every row."""
    row = torch.arange(b["total"], device="cuda", dtype=torch.int32)
    s = torch.searchsorted(b["row_offsets"], row, right=True).long() - 1
    return s, b["lengths"][s] - (b["row_offsets"][s + 1] - row)


def _append_plain(x, cache, b, sequence, position):
    """x [rows, heads, D] in 32 bits into the pages, in place."""
    data, scales = cache
    page = data.shape[2]
    target = b["table"][sequence, position // page].long()
    slot = (position % page).long()
    high = x.abs().amax(dim=-1)
    loudest = torch.zeros_like(scales).index_reduce_(0, target, high, "amax")
    first = torch.full((scales.shape[0],), page, device="cuda", dtype=torch.long).index_reduce_(0, target, slot, "amin")
    fraction, exponent = torch.frexp(loudest)               # loudest = fraction * 2^exponent, fraction in [1/2, 1)
    needed = torch.ldexp(torch.ones_like(loudest), exponent - 9 + (fraction > 0.875)).clamp_min(TINY)
    needed = torch.where(loudest > 0, needed, TINY)
    touched = (first < page)[:, None]
    new = torch.where(touched, torch.maximum(needed, torch.where((first > 0)[:, None], scales, 0.0)), scales)
    there = torch.arange(page, device="cuda")[None] < first[:, None]
    again = ((new > scales) & touched)[:, :, None, None] & there[:, None, :, None]
    softer = (data.view(torch.float8_e4m3fn).float() * (scales / new)[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    data.copy_(torch.where(again, softer, data))
    scales.copy_(new)
    data[target, :, slot] = (x / new[target][..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)


def _attention_plain(state):
    case, b, q = state["case"], state["b"], state["q"]
    heads, kv_heads, dim = q.shape[1], case["kv_heads"], case["dim"]
    sequence, position = _rows_of(b)
    count = b["table"].shape[0]
    place = torch.arange(b["total"], device="cuda") - b["row_offsets"][sequence]
    padded = torch.zeros((count, b["most"], heads, dim), device="cuda")
    padded[sequence, place] = q.float() * state["scale"]
    at = torch.full((count, b["most"]), -1, device="cuda", dtype=torch.int32)
    at[sequence, place] = position
    pages = b["table"].clamp_min(0).long()
    token = torch.arange(pages.shape[1] * case["page"], device="cuda")
    stored = (token[None] < b["lengths"][:, None])[:, None, :, None]         # [sequence, 1, token, 1]

    def gathered(cache):
        data, scales = cache
        x = data[pages].view(torch.float8_e4m3fn).float() * scales[pages][..., None, None]
        return torch.where(stored, x.transpose(1, 2).flatten(2, 3), 0.0)       # [sequence, head, token, D]

    k = gathered(state["k_cache"])
    group = heads // kv_heads
    folded = padded.unflatten(2, (kv_heads, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)       # [sequence, KV head, group * row, D]
    scores = folded @ k.transpose(-1, -2)
    del k
    seen = token[None, None] <= at[..., None]
    if case["window"]:
        seen &= token[None, None] > at[..., None] - case["window"]
    seen = seen[:, None, None].expand(-1, 1, group, -1, -1).flatten(2, 3)                      # [sequence, 1, group * row, token]
    scores.masked_fill_(~seen, -math.inf)
    scores.sub_(scores.amax(dim=-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    out = (scores @ gathered(state["v_cache"])) / torch.where(total > 0, total, 1.0)
    out = out.unflatten(2, (group, b["most"])).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[sequence, place].bfloat16()


def run(state):
    case = state["case"]
    if own:
        import gewell_b200 as gw
        if case["op"] == "norm":
            return gw.qk_norm_rotary(state["q"], state["k"], state["q_weight"], state["k_weight"], state["positions"],
                                     state["frequencies"], epsilon=EPSILON, interleaved=case["interleaved"])
        if case["op"] == "append":
            gw.kv_cache_append(state["cache"], state["batch"], state["k"], state["v"], key_weight=state["k_weight"],
                               normalize_key=case["norm"], normalize_value=case["norm"], frequencies=state["frequencies"],
                               interleaved=case["interleaved"], epsilon=EPSILON)
            return _stored(state)
        return gw.paged_attention(state["cache"], state["batch"], state["q"], state["scale"], window=case["window"])
    if case["op"] == "norm":
        return tuple(_turned(state[n], state[n + "_weight"], True, state["positions"], state["frequencies"], case["interleaved"]).bfloat16()
                     for n in ("q", "k"))
    if case["op"] == "append":
        sequence, position = _rows_of(state["b"])
        key = _turned(state["k"], state["k_weight"], case["norm"], position, state["frequencies"], case["interleaved"])
        _append_plain(key, state["k_cache"], state["b"], sequence, position)
        _append_plain(_turned(state["v"], None, case["norm"], None, None, False), state["v_cache"], state["b"], sequence, position)
        return _stored(state)
    return _attention_plain(state)


def _stored(state):
    """The whole cache: the values of the codes, and the scales."""
    (k, k_scales), (v, v_scales) = state["k_cache"], state["v_cache"]
    return {"k": k.view(torch.float8_e4m3fn), "v": v.view(torch.float8_e4m3fn), "k_scales": k_scales, "v_scales": v_scales}


# --------------------------------------------------------------------------- the definition in 64 bits

def _head_exact(x, weight, positions, frequencies, interleaved):
    y = x.double()
    y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + EPSILON) if weight is not False else y
    if weight is not None and weight is not False:
        y = y * weight.double()
    if frequencies is None:
        return y
    y = y.clone()
    for i in range(frequencies.numel()):
        p, r = (2 * i, 2 * i + 1) if interleaved else (i, i + frequencies.numel())
        angle = (positions.double() * frequencies[i].double())[:, None]
        first, second = y[..., p].clone(), y[..., r].clone()
        y[..., p] = first * angle.cos() - second * angle.sin()
        y[..., r] = first * angle.sin() + second * angle.cos()
    return y


def _e4m3(x):
    """The nearest value of the format, ties to even, in 64 bits."""
    size = x.abs().clamp_min(2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return tuple(_head_exact(s[n], s[n + "_weight"], s["positions"], s["frequencies"], case["interleaved"]) for n in ("q", "k"))
    lengths, page = _lengths(case), case["page"]
    if case["op"] == "append":
        out, table = {}, s["b"]["table"].cpu().numpy()
        for name, frequencies in (("k", s["frequencies"]), ("v", None)):
            data, scales = s[name + "_cache"]
            codes, scales = data.view(torch.float8_e4m3fn).double(), scales.double()
            positions = torch.cat([torch.arange(c - n, c) for n, c in lengths]).cuda()
            weight = (s["k_weight"] if name == "k" else None) if case["norm"] else False
            x = _head_exact(s[name], weight, positions, frequencies, case["interleaved"])
            low = 0
            for i, (n, c) in enumerate(lengths):
                at = c - n
                while at < c:
                    p, slot = int(table[i, at // page]), at % page
                    many = min(page - slot, c - at)
                    part = x[low:low + many].transpose(0, 1)                       # [head, token, D]
                    needed = torch.exp2(torch.ceil(torch.log2(part.abs().amax(dim=(1, 2)) / 448.0))).clamp_min(TINY)
                    new = torch.maximum(needed, scales[p]) if slot else needed
                    if slot:
                        codes[p, :, :slot] = _e4m3(codes[p, :, :slot] * (scales[p] / new)[:, None, None])
                    codes[p, :, slot:slot + many] = _e4m3(part / new[:, None, None])
                    scales[p] = new
                    low, at = low + many, at + many
            out[name], out[name + "_scales"] = codes, scales
        return out
    group, out = case["heads"] // case["kv_heads"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    low = 0
    for i, (n, c) in enumerate(lengths):
        pages = s["b"]["table"][i, :-(-c // page)].long()
        at = torch.arange(c - n, c, device="cuda")[:, None]
        token = torch.arange(c, device="cuda")[None]
        hidden = token > at
        if case["window"]:
            hidden = hidden | (at - token >= case["window"])
        for h in range(case["kv_heads"]):
            k, v = (((d[pages, h].contiguous().view(torch.float8_e4m3fn).double() * f[pages, h].double()[:, None, None]).flatten(0, 1))[:c]
                    for d, f in (s["k_cache"], s["v_cache"]))
            for j in range(h * group, (h + 1) * group):
                logits = (s["q"][low:low + n, j].double() @ k.T) * s["scale"]
                out[low:low + n, j] = torch.softmax(logits.masked_fill(hidden, -math.inf), dim=-1) @ v
        low += n
    return out


# --------------------------------------------------------------------------- what it cannot do without

def work(case):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "norm":
        elements = case["rows"] * (heads + kv_heads) * dim
        return {"bytes": 4.0 * elements + 4.0 * case["rows"] + 4.0 * dim + 2.0 * case["rotary"], "flops": 8.0 * elements}
    lengths = _lengths(case)
    rows = sum(n for n, _ in lengths)
    if case["op"] == "append":
        elements = 2.0 * rows * kv_heads * dim
        pages = sum(-(-c // case["page"]) - (c - n) // case["page"] for n, c in lengths)
        return {"bytes": 3.0 * elements + 16.0 * pages * kv_heads, "flops": 8.0 * elements}
    window = case["window"] or 1 << 40
    tokens, pairs = 0, 0
    for n, c in lengths:
        tokens += c - max(0, c - n - window + 1)
        seen = np.minimum(np.arange(c - n + 1, c + 1), window)
        pairs += int(seen.sum())
    return {"bytes": 2.0 * tokens * kv_heads * dim + 8.0 * tokens * kv_heads / case["page"] + 4.0 * rows * heads * dim,
            "flops": 4.0 * pairs * heads * dim}
