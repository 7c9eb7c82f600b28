"""The serving operators of compress_zip_b200.ops on measured cases: the 8-bit product with scales for each token and
channel, attention over a cache held in 4 bits with the append that fills it, and eviction from that cache by accumulated
attention weight.

Where ``own`` is false, ``run`` computes the operators with elementary torch operations; where it is true, it makes the
calls that a program makes of compress_zip_b200.ops.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# Sizes: 384 -> 512 is the shipped model's QKV projection; 6 query heads over one key head of 64 are its heads, 8 over one
# the larger model's, with contexts up to 4096 and thousands of streams decoded side by side; the others are generic.
LISTED = [
    # one stream's next token through the shipped model's QKV projection: latency
    {"name": "project_one", "op": "project", "m": 1, "n": 512, "k": 384, "type": "bf16", "out": "bf16", "bias": False},
    # a step of a batch of streams: the weights' bytes
    {"name": "project_step", "op": "project", "m": 48, "n": 4096, "k": 4096, "type": "fp16", "out": "fp16", "bias": False},
    # ragged sizes of a scoring pass, logits kept in 32 bits
    {"name": "project_odd", "op": "project", "m": 1333, "n": 1000, "k": 1100, "type": "bf16", "out": "fp32", "bias": True},
    # a wave of prompts: the tensor cores
    {"name": "project_wave", "op": "project", "m": 8192, "n": 8192, "k": 4096, "type": "bf16", "out": "bf16", "bias": True},
    # one stream's next token early in its context: latency
    {"name": "attend_one", "op": "attend", "b": 1, "t": 1, "hq": 6, "hkv": 1, "d": 64, "len": 77, "cap": 1024, "type": "bf16", "track": False},
    # a batch of long streams whose weights are accumulated for the eviction
    {"name": "attend_track", "op": "attend", "b": 64, "t": 1, "hq": 32, "hkv": 4, "d": 128, "len": 4096, "cap": 4096, "type": "fp16", "track": True},
    # one very long stream: split over its length
    {"name": "attend_long", "op": "attend", "b": 1, "t": 1, "hq": 32, "hkv": 8, "d": 128, "len": 131071, "cap": 131072, "type": "bf16", "track": False},
    # thousands of streams of the shipped model's heads, one token each: append and attend
    {"name": "step_streams", "op": "step", "b": 4096, "t": 1, "hq": 6, "hkv": 1, "d": 64, "len": 512, "cap": 512, "type": "bf16", "track": False},
    # a few streams that take a block of tokens each, some rows of it padding, with weights
    {"name": "step_block", "op": "step", "b": 5, "t": 7, "hq": 8, "hkv": 2, "d": 64, "len": 1500, "cap": 2000, "type": "fp16", "track": True},
    # one stream's slot is full
    {"name": "evict_one", "op": "evict", "b": 1, "hkv": 1, "d": 64, "len": 1024, "cap": 1024, "budget": 700, "recent": 64, "type": "bf16"},
    # the slots of a batch are cut to a quarter
    {"name": "evict_batch", "op": "evict", "b": 48, "hkv": 8, "d": 128, "len": 4096, "cap": 4096, "budget": 1024, "recent": 128, "type": "bf16"},
]


def listed():
    return [dict(c) for c in LISTED]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["project", "project", "attend", "attend", "step", "evict"])
    if op == "project":
        m, n, k = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 32, 8192)
        while m * n * k > 8192 * 8192 * 4096:
            m = m // 2 + 1
        kind = rng.choice(["bf16", "fp16"])
        return {"op": op, "m": m, "n": n, "k": k, "type": kind, "out": rng.choice([kind, kind, "fp32"]), "bias": rng.random() < 0.5}
    d, hkv, kind = rng.choice([64, 128]), rng.choice([1, 2, 4, 8]), rng.choice(["bf16", "fp16"])
    if op == "evict":
        b, length = _log(rng, 1, 64), _log(rng, 16, 16384)
        while b * hkv * d * length > 48 * 8 * 128 * 4096:
            length = length // 2 + 1
        budget = max(1, int(length * rng.uniform(0.1, 0.9)))
        return {"op": op, "b": b, "hkv": hkv, "d": d, "len": length, "cap": length + rng.randrange(0, 65), "budget": budget,
                "recent": rng.randrange(0, max(1, budget // 2)), "type": kind}
    b, t, g = _log(rng, 1, 512), rng.choice([1, 1, 1, rng.randrange(2, 9)]), rng.choice([1, 2, 3, 4, 6, 8])
    length = _log(rng, 1, 65536 if op == "attend" else 8192)
    while b * hkv * d * length > 8 * 131071 * 128 // 2:
        b, length = b // 2 + 1, length // 2 + 1
    return {"op": op, "b": b, "t": t, "hq": g * hkv, "hkv": hkv, "d": d, "len": length, "cap": length + rng.randrange(0, 65),
            "type": kind, "track": rng.random() < 0.4}


def _lengths(case):
    """The sequences' lengths: the longest first, the others spread over (0, len]; from four sequences on, one is empty."""
    b, top = case["b"], case["len"]
    got = [top] + [max(1, math.ceil(top * ((i * 0.6180339887498949) % 1.0))) for i in range(1, b)]
    if b >= 4:
        got[b // 2] = 0
    return got


def _cache(case, gen, dev):
    """A cache as appends and steps before have left it: codes of about normal values, every entry with its own range."""
    shape = (case["b"], case["hkv"], case["cap"])

    def codes():
        c = (torch.randn(*shape, case["d"], generator=gen, device=dev, dtype=torch.float16) * 3 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
        return c[..., 0::2] | (c[..., 1::2] << 4)

    def ranges():
        step = 0.2 + 0.2 * torch.rand(shape, generator=gen, device=dev)
        return step, -step * (6.5 + 2 * torch.rand(shape, generator=gen, device=dev))

    k, v = codes(), codes()
    return k, v, torch.stack([*ranges(), *ranges()], -1).to(torch.bfloat16)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    kind = DTYPES[case["type"]]
    if case["op"] == "project":
        m, n, k = case["m"], case["n"], case["k"]
        x = (randn(m, k) * torch.exp(0.7 * randn(k))).to(kind)
        # the weights' rows begin on 16-byte boundaries, as ops.quantize_rows leaves them
        codes = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device=dev)
        codes[:, :k] = (randn(n, k) * 40).round().clamp(-127, 127).to(torch.int8)
        return {"case": dict(case), "x": x, "codes": codes[:, :k], "scales": (0.5 + torch.rand(n, generator=gen, device=dev)) / (40 * math.sqrt(k)),
                "bias": randn(n) if case["bias"] else None}
    b, hkv, d = case["b"], case["hkv"], case["d"]
    k, v, scales = _cache(case, gen, dev)
    order = torch.randperm(b, generator=gen, device=dev)
    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)[order]
    slots = torch.randperm(b, generator=gen, device=dev).to(torch.int32)
    state = {"case": dict(case), "k": k, "v": v, "scales": scales, "slots": slots, "lengths": lengths, "weights": None}
    if case["op"] == "evict" or case["track"]:  # sums of many steps' weights: a few entries hold most
        state["weights"] = torch.exp(2 * randn(b, hkv, case["cap"]))
    if case["op"] == "evict":
        state["zeros"] = torch.zeros(b, dtype=torch.int32, device=dev)
        return state
    t = case["t"]
    state["q"] = randn(b, t, case["hq"], d).to(kind)
    if case["op"] == "step":
        state["new_k"], state["new_v"] = randn(b, t, hkv, d).to(kind), randn(b, t, hkv, d).to(kind)
        state["starts"] = (lengths - t).clamp_(min=0)
    return state


def work(case):
    if case["op"] == "project":
        m, n, k = case["m"], case["n"], case["k"]
        out = 4 if case["out"] == "fp32" else 2
        return {"bytes": 2 * m * k + n * k + 4 * n + (4 * n if case["bias"] else 0) + out * m * n, "flops": 2 * m * n * k}
    hkv, d, entries = case["hkv"], case["d"], sum(_lengths(case))
    if case["op"] == "evict":
        kept = sum(min(x, case["budget"]) for x in _lengths(case))
        moved = sum(min(x, case["budget"]) for x in _lengths(case) if x > case["budget"])
        # the weights, the entries that move (read and written), and the kept entries given back in 16 bits
        return {"bytes": hkv * (4 * entries + 2 * moved * (d + 12) + 4 * kept + kept * (d + 8 + 4 * d)), "flops": 4 * hkv * kept * d}
    b, t, hq = case["b"], case["t"], case["hq"]
    got = entries * hkv * (d + 8) + 4 * b * t * hq * d
    if case["track"]:
        got += 8 * entries * hkv
    if case["op"] == "step":  # the new rows in, their entries written, and given back in 16 bits
        got += b * t * hkv * (4 * d + d + 8 + 4 * d)
    return {"bytes": got, "flops": 4 * entries * t * hq * d}


# ---- the plain forms ---------------------------------------------------------------------------------------------------


def _unpack(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def _values(codes, step, lo):
    return lo[..., None].float() + step[..., None].float() * _unpack(codes).float()


def _project(s):
    x = s["x"].float()
    top = x.abs().amax(1, keepdim=True)
    codes = torch.where(top > 0, x * 127 / top, 0).round()
    y = (codes @ s["codes"].float().t()) * (top / 127) * s["scales"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(DTYPES[s["case"]["out"]])


def _down(x):
    """The largest bf16 value that is not above x (float64)."""
    y = x.float().to(torch.bfloat16)
    return torch.where(y.double() > x, torch.nextafter(y, torch.full_like(y, -math.inf)), y)


def _up(x):
    y = x.float().to(torch.bfloat16)
    return torch.where(y.double() < x, torch.nextafter(y, torch.full_like(y, math.inf)), y)


def _entry(x):
    """The codes, step and lower end of rows of values."""
    x = x.double()
    lo = _down(x.amin(-1))
    step = _up((x.amax(-1) - lo.double()) / 15)
    c = torch.where(step[..., None] > 0, (x - lo[..., None].double()) / step[..., None].double(), 0).round().clamp(0, 15).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), step, lo


def _append(s):
    """The new rows as entries lengths - t .. lengths - 1 of their slots; rows before entry 0 are padding."""
    t = s["case"]["t"]
    at = s["lengths"].long()[:, None] - t + torch.arange(t, device=s["q"].device)
    src = torch.where(at >= 0, torch.arange(t, device=at.device), t - 1)  # padding repeats the last row
    at = torch.where(at >= 0, at, (s["lengths"].long() - 1).clamp(min=0)[:, None])
    rows = torch.arange(len(at), device=at.device)[:, None]
    kc, ks, kl = _entry(s["new_k"][rows, src])
    vc, vs, vl = _entry(s["new_v"][rows, src])
    slots = s["slots"].long()[:, None]
    some = (s["lengths"] > 0)[:, None, None, None]
    s["k"][slots, :, at] = torch.where(some, kc, s["k"][slots, :, at])
    s["v"][slots, :, at] = torch.where(some, vc, s["v"][slots, :, at])
    s["scales"][slots, :, at] = torch.where(some, torch.stack([ks, kl, vs, vl], -1), s["scales"][slots, :, at])
    if s["weights"] is not None:
        s["weights"][slots, :, at] = torch.where(some[..., 0], 0.0, s["weights"][slots, :, at])


def _attend(s):
    c = s["case"]
    b, t, hq, hkv, d, n = c["b"], c["t"], c["hq"], c["hkv"], c["d"], c["len"]
    slots = s["slots"].long()
    sc = s["scales"][slots, :, :n]
    k = _values(s["k"][slots, :, :n], sc[..., 0], sc[..., 1])
    q = s["q"].float().view(b, t, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)
    score = (q @ k.transpose(-1, -2)) / math.sqrt(d)
    del k
    sees = s["lengths"].long()[:, None] - (t - 1) + torch.arange(t, device=q.device)  # entries that row t sees
    sees = sees.repeat_interleave(hq // hkv, 1)[:, None, :, None] > torch.arange(n, device=q.device)
    score = torch.where(sees, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.where(sees, torch.exp(score - torch.where(top > -math.inf, top, 0.0)), 0.0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    v = _values(s["v"][slots, :, :n], sc[..., 2], sc[..., 3])
    out = (p @ v).view(b, hkv, t, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, t, hq, d)
    if s["weights"] is not None:
        s["weights"][slots, :, :n] += p.sum(2)
    return out.to(s["q"].dtype)


def _read(s, starts, count):
    slots = s["slots"].long()[:, None]
    at = starts.long()[:, None] + torch.arange(count, device=starts.device)
    sc = s["scales"][slots, :, at]
    kind = DTYPES[s["case"]["type"]]
    return _values(s["k"][slots, :, at], sc[..., 0], sc[..., 1]).to(kind), _values(s["v"][slots, :, at], sc[..., 2], sc[..., 3]).to(kind)


def _evict(s):
    c = s["case"]
    n, budget, recent = c["len"], min(c["budget"], c["len"]), c["recent"]
    slots, length = s["slots"].long(), s["lengths"].long()[:, None, None]
    entry = torch.arange(n, device=slots.device)
    w = s["weights"][slots, :, :n]
    rank = torch.where(entry >= length - recent, math.inf, w)
    rank = torch.where(entry < length, rank, -math.inf)
    chosen = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    chosen = torch.where(length > budget, torch.sort(chosen, dim=-1).values, entry[:budget])  # short sequences stay as they are
    there = entry[:budget] < length
    kept = torch.where(there, chosen, -1).to(torch.int32)
    rows, heads = slots[:, None, None], torch.arange(c["hkv"], device=slots.device)[None, :, None]
    for name in ("k", "v", "scales", "weights"):
        moved = s[name][rows, heads, chosen]
        s[name][slots, :, :budget] = moved
    return kept, s["lengths"].clamp(max=budget)


# ---- one pass ----------------------------------------------------------------------------------------------------------


def _ops():
    from __graft_entry__ import load_package

    load_package()
    from compress_zip_b200 import ops

    return ops


def _handle(s):
    """The program's cache object over its buffers, made once."""
    if "handle" not in s:
        s["handle"] = _ops().KV4Cache(s["k"], s["v"], s["scales"], weights=s["weights"])
    return s["handle"]


def run(s):
    c = s["case"]
    if c["op"] == "project":
        if not own:
            return {"y": _project(s)}
        if "weight" not in s:
            s["weight"], s["linear"] = _ops().QRows(s["codes"], s["scales"]), _ops().linear_i8
        return {"y": s["linear"](s["x"], s["weight"], bias=s["bias"], out_dtype=DTYPES[c["out"]])}
    got = {}
    if c["op"] == "evict":
        if own:
            h = _handle(s)
            got["kept"], got["lengths"] = h.evict(s["slots"], s["lengths"], budget=min(c["budget"], c["len"]), recent=c["recent"], max_len=c["len"])
            got["k"], got["v"] = h.read(s["slots"], s["zeros"], min(c["budget"], c["len"]), dtype=DTYPES[c["type"]])
        else:
            got["kept"], got["lengths"] = _evict(s)
            got["k"], got["v"] = _read(s, s["zeros"], min(c["budget"], c["len"]))
        got["weights"] = s["weights"]
        return got
    if c["op"] == "step":
        if own:
            _handle(s).append(s["new_k"], s["new_v"], s["slots"], s["lengths"])
        else:
            _append(s)
    got["out"] = _handle(s).attend(s["q"], s["slots"], s["lengths"], max_len=c["len"]) if own else _attend(s)
    if c["op"] == "step":
        count = min(c["t"], c["cap"])
        got["k"], got["v"] = _handle(s).read(s["slots"], s["starts"], count, dtype=DTYPES[c["type"]]) if own else _read(s, s["starts"], count)
    if s["weights"] is not None:
        got["weights"] = s["weights"]
    return got


# ---- the definitions in 64 bits, sequence by sequence --------------------------------------------------------------------


def _bf16_below(x):
    """x (float64) rounded towards minus infinity to 8 significant bits."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.floor(m * 256), e - 8)


def _exact_rows(x):
    x = x.double()
    lo = _bf16_below(x.min(-1).values)
    step = -_bf16_below(-(x.max(-1).values - lo) / 15)
    q = torch.round((x - lo.unsqueeze(-1)) / torch.where(step > 0, step, 1.0).unsqueeze(-1))
    return lo.unsqueeze(-1) + step.unsqueeze(-1) * q


def _exact_entries(s, name, column, slot, n):
    """Entries 0 .. n-1 of a slot as values: [heads, n, d] in float64."""
    b = s[name][slot, :, :n].to(torch.int32)
    x = torch.empty(*b.shape[:-1], 2 * b.shape[-1], dtype=torch.float64, device=b.device)
    x[..., 0::2], x[..., 1::2] = (b % 16).double(), (b // 16).double()
    sc = s["scales"][slot, :, :n].double()
    return x * sc[..., column:column + 1] + sc[..., column + 1:column + 2]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "project":
        x = s["x"].double()
        top = x.abs().max(1, keepdim=True).values
        q = torch.round(127 * x / torch.where(top == 0, 1.0, top))
        y = torch.mm(q, s["codes"].double().T) * (top / 127) * s["scales"].double().unsqueeze(0)
        return {"y": y if s["bias"] is None else y + s["bias"].double().unsqueeze(0)}
    hkv, d = case["hkv"], case["d"]
    lengths, slots = s["lengths"].tolist(), s["slots"].tolist()
    weights = None if s["weights"] is None else s["weights"].double()
    if case["op"] == "evict":
        budget = min(case["budget"], case["len"])
        kept = torch.full((case["b"], hkv, budget), -1, dtype=torch.int32, device=s["k"].device)
        k = torch.empty(case["b"], budget, hkv, d, dtype=torch.float64, device=s["k"].device)
        v = torch.empty_like(k)
        for i, (slot, n) in enumerate(zip(slots, lengths)):
            ks, vs = (_exact_entries(s, a, c, slot, case["cap"]) for a, c in (("k", 0), ("v", 2)))
            for h in range(hkv):
                if n <= budget:
                    stay = torch.arange(budget, device=k.device)
                    kept[i, h, :n] = stay[:n].int()
                else:
                    old = n - case["recent"]
                    best = torch.argsort(-weights[slot, h, :old], stable=True)[:budget - case["recent"]]
                    stay = torch.cat([best, torch.arange(old, n, device=k.device)]).sort().values
                    kept[i, h] = stay.int()
                    weights[slot, h, :budget] = weights[slot, h, stay].clone()
                k[i, :, h], v[i, :, h] = ks[h, stay], vs[h, stay]
        return {"kept": kept, "lengths": s["lengths"].clamp(max=budget), "k": k, "v": v, "weights": weights}
    b, t, g = case["b"], case["t"], case["hq"] // hkv
    out = torch.zeros(b, t, case["hq"], d, dtype=torch.float64, device=s["k"].device)
    count = min(t, case["cap"])
    back = [torch.zeros(b, count, hkv, d, dtype=torch.float64, device=out.device) for _ in range(2)]
    for i, (slot, n) in enumerate(zip(slots, lengths)):
        top = max(n, count if case["op"] == "step" else 0)
        kv = [_exact_entries(s, a, c, slot, top) for a, c in (("k", 0), ("v", 2))]
        if case["op"] == "step":
            new = min(t, n)
            for x, rows in zip(kv, (s["new_k"], s["new_v"])):
                if new:
                    x[:, n - new:n] = _exact_rows(rows[i, t - new:]).transpose(0, 1)
            if weights is not None:
                weights[slot, :, n - new:n] = 0
            at = max(n - t, 0)
            for x, y in zip(back, kv):
                x[i] = y[:, at:at + count].transpose(0, 1)
        for row in range(t):
            seen = n - (t - 1 - row)
            if seen <= 0:
                continue
            q = s["q"][i, row].double().view(hkv, g, d)
            p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, kv[0][:, :seen]) * d ** -0.5, -1)
            out[i, row] = torch.einsum("hgn,hnd->hgd", p, kv[1][:, :seen]).reshape(-1, d)
            if weights is not None:
                weights[slot, :, :seen] += p.sum(1)
    got = {"out": out}
    if case["op"] == "step":
        got["k"], got["v"] = back
    if weights is not None:
        got["weights"] = weights
    return got
