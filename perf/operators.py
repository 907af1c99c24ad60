"""The operators that serve a causal decoder behind its first prompt, as cases that can be timed:
rotation of positions, keys and values appended to a paged cache, attention over that cache.

A case is one call with its sizes. `run` computes it in plain torch operations, or, where `own` is
true, through the package's calls, prepared once as a serving loop keeps them: the buffers stay where
they are, what they hold and the lengths on the device change.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
LARGEST_FLOPS = 1.2e12     # the long prompt below
LARGEST_BYTES = 6.0e8


def listed() -> list[dict]:
    return [
        # the query and key heads of one token far into a long context: latency alone
        {"name": "rotary_token", "op": "rotary", "tokens": 1, "heads": 40, "head_dim": 128, "rotary_dim": 128,
         "interleaved": False, "scaling": "ramp", "start": 100000, "dtype": "bf16"},
        # all heads of a packed batch of prompts, half of each head rotated
        {"name": "rotary_prompts", "op": "rotary", "tokens": 8192, "heads": 40, "head_dim": 128, "rotary_dim": 64,
         "interleaved": True, "scaling": "none", "start": 0, "dtype": "f16"},
        # one token of each sequence of a decode step; the queries are rotated on the way
        {"name": "append_tokens", "op": "append", "sequences": 64, "new_low": 1, "new_high": 1, "past_low": 100,
         "past_high": 4000, "kv_heads": 8, "q_heads": 32, "head_dim": 128, "rotary_dim": 128, "interleaved": False,
         "scaling": "bands", "page_size": 16, "head_major": False, "dtype": "bf16"},
        # a ragged batch of prompts of a decoder with learned positions: nothing is rotated
        {"name": "append_prompts", "op": "append", "sequences": 7, "new_low": 333, "new_high": 3001, "past_low": 0,
         "past_high": 0, "kv_heads": 32, "q_heads": 0, "head_dim": 64, "rotary_dim": 0, "interleaved": False,
         "scaling": "none", "page_size": 32, "head_major": True, "dtype": "f16"},
        # the next token of one short conversation: latency alone
        {"name": "decode_one", "op": "attention", "sequences": 1, "new_low": 1, "new_high": 1, "past_low": 300,
         "past_high": 300, "kv_heads": 12, "q_heads": 12, "head_dim": 64, "causal": True, "window": 0,
         "page_size": 16, "head_major": False, "dtype": "f16"},
        # a decode step of a server: grouped heads, lengths of all sizes
        {"name": "decode_batch", "op": "attention", "sequences": 32, "new_low": 1, "new_high": 1, "past_low": 500,
         "past_high": 8000, "kv_heads": 8, "q_heads": 32, "head_dim": 128, "causal": True, "window": 0,
         "page_size": 16, "head_major": False, "dtype": "bf16"},
        # the same where each head has keys of its own, as the decoder family of this package
        {"name": "decode_heads", "op": "attention", "sequences": 48, "new_low": 1, "new_high": 1, "past_low": 60,
         "past_high": 2000, "kv_heads": 32, "q_heads": 32, "head_dim": 64, "causal": True, "window": 0,
         "page_size": 32, "head_major": True, "dtype": "f16"},
        # one very long document
        {"name": "decode_long", "op": "attention", "sequences": 1, "new_low": 1, "new_high": 1, "past_low": 150001,
         "past_high": 150001, "kv_heads": 4, "q_heads": 32, "head_dim": 128, "causal": True, "window": 0,
         "page_size": 64, "head_major": False, "dtype": "bf16"},
        # a few drafted tokens of each sequence are checked at once; five heads share keys
        {"name": "draft_tokens", "op": "attention", "sequences": 16, "new_low": 3, "new_high": 8, "past_low": 700,
         "past_high": 6000, "kv_heads": 8, "q_heads": 40, "head_dim": 128, "causal": True, "window": 0,
         "page_size": 16, "head_major": False, "dtype": "bf16"},
        # a piece of a long prompt, behind what is cached of it
        {"name": "chunk_of_prompt", "op": "attention", "sequences": 1, "new_low": 1000, "new_high": 1000,
         "past_low": 30000, "past_high": 30000, "kv_heads": 8, "q_heads": 32, "head_dim": 128, "causal": True,
         "window": 0, "page_size": 16, "head_major": False, "dtype": "bf16"},
        # a ragged batch of prompts, nothing cached before them
        {"name": "prompts", "op": "attention", "sequences": 6, "new_low": 511, "new_high": 4000, "past_low": 0,
         "past_high": 0, "kv_heads": 32, "q_heads": 32, "head_dim": 64, "causal": True, "window": 0,
         "page_size": 32, "head_major": False, "dtype": "f16"},
        # the largest: one long prompt in one piece
        {"name": "long_prompt", "op": "attention", "sequences": 1, "new_low": 12001, "new_high": 12001, "past_low": 0,
         "past_high": 0, "kv_heads": 8, "q_heads": 32, "head_dim": 128, "causal": True, "window": 0,
         "page_size": 128, "head_major": True, "dtype": "bf16"},
    ]


def _log(rng, low: int, high: int) -> int:
    """A whole number between low and high, spread evenly over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def _rotation(rng, head_dim: int) -> dict:
    return {"rotary_dim": rng.choice([head_dim, head_dim, head_dim // 2, 32]), "interleaved": rng.random() < 0.5,
            "scaling": rng.choice(["none", "linear", "base", "ramp", "bands"])}


def draw(rng) -> dict:
    while True:
        dtype = rng.choice(["f16", "bf16"])
        op = rng.choice(["rotary", "append", "attention", "attention", "attention"])
        head_dim = rng.choice([64, 64, 128, 128, 80, 96])
        if op == "rotary":
            case = {"op": op, "tokens": _log(rng, 1, 16000), "heads": rng.choice([1, 8, 12, 32, 40, 71]),
                    "head_dim": head_dim, "start": rng.choice([0, _log(rng, 1, 1000000)]), **_rotation(rng, head_dim)}
        else:
            kv_heads = rng.choice([1, 2, 4, 8, 12, 16, 32])
            group = rng.choice([1, 1, 2, 4, 5, 8]) if kv_heads <= 8 else 1
            case = {"op": op, "kv_heads": kv_heads, "q_heads": kv_heads * group, "head_dim": head_dim,
                    "page_size": rng.choice([8, 16, 32, 64, 128, 48]), "head_major": rng.random() < 0.4}
            kind = rng.choice(["token", "draft", "chunk", "prompt"])
            sequences = _log(rng, 1, {"token": 200, "draft": 60, "chunk": 8, "prompt": 12}[kind])
            past = 0 if kind == "prompt" else _log(rng, 1, 100000 if sequences <= 4 else 6000)
            new = {"token": 1, "draft": rng.randint(2, 16), "chunk": _log(rng, 17, 2000),
                   "prompt": _log(rng, 1, 9000)}[kind]
            case.update(sequences=sequences, new_low=max(1, new - rng.randint(0, new // 2)), new_high=new,
                        past_low=past // rng.choice([1, 2, 10]), past_high=past)
            if op == "append":
                case.update(_rotation(rng, head_dim))
                if rng.random() < 0.3:
                    case.update(rotary_dim=0, q_heads=0, scaling="none")
            else:
                case.update(causal=kind == "token" or rng.random() < 0.85,
                            window=_log(rng, 16, 8000) if rng.random() < 0.2 else 0)
                if not case["causal"]:
                    case["window"] = 0
        case["dtype"] = dtype
        cost = work(case)
        cells = sum(n * (p + n) for n, p in zip(*_lengths(case))) * case["q_heads"] if op == "attention" else 0
        held = 0 if op == "rotary" else sum(map(sum, _lengths(case))) * case["kv_heads"] * head_dim * 4
        if cost["flops"] <= LARGEST_FLOPS and cost["bytes"] <= LARGEST_BYTES and cells <= 5e9 and held <= 6e8:
            return case


# ---------------------------------------------------------------------- sizes
def _spread(low: int, high: int, n: int, stride: int) -> list[int]:
    """n numbers from low to high, in an order of their own."""
    return [low + (high - low) * ((i * stride) % n) // max(1, n - 1) for i in range(n)]


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """New tokens of each sequence, and what is cached before them."""
    n = case["sequences"]
    step = next(s for s in (7, 11, 13, 1) if math.gcd(s, n) == 1)
    return _spread(case["new_low"], case["new_high"], n, step), _spread(case["past_low"], case["past_high"], n, 1)


def _visible(case: dict, new: int, past: int) -> int:
    """Pairs of a query and a key that it sees."""
    if not case["causal"]:
        return new * (new + past)
    w = case["window"] or (new + past)
    return sum(min(w, past + i + 1) for i in range(new))


def work(case: dict) -> dict:
    d = case["head_dim"]
    if case["op"] == "rotary":
        rows = case["tokens"] * case["heads"]
        return {"bytes": 4.0 * rows * d + 4 * case["tokens"], "flops": 3.0 * rows * case["rotary_dim"]}
    news, pasts = _lengths(case)
    tokens = sum(news)
    if case["op"] == "append":
        rows = tokens * (2 * case["kv_heads"] + case["q_heads"])
        return {"bytes": 4.0 * rows * d,
                "flops": 3.0 * tokens * (case["kv_heads"] + case["q_heads"]) * case["rotary_dim"]}
    keys = 0
    for new, past in zip(news, pasts):
        first = max(0, past - case["window"] + 1) if case["window"] else 0
        keys += past + new - first
    return {"bytes": 4.0 * d * (keys * case["kv_heads"] + tokens * case["q_heads"]),
            "flops": 4.0 * d * case["q_heads"] * sum(_visible(case, n, p) for n, p in zip(news, pasts))}


# --------------------------------------------------------------------- inputs
ROTATION = {"theta": 10000.0, "factor": 4.0, "original_length": 8192}
BANDS = {"low": 1.0, "high": 4.0}     # turns within the original length
RAMP = {"low": 1.0, "high": 32.0}


def _rotary_config(case: dict) -> dict:
    c = {"rotary_dim": case["rotary_dim"], "interleaved": case["interleaved"], "scaling": case["scaling"], **ROTATION}
    c.update(BANDS if case["scaling"] == "bands" else RAMP)
    return c


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    dtype, d = DTYPES[case["dtype"]], case["head_dim"]

    def values(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    if case["op"] == "rotary":
        t = case["tokens"]
        # queries and keys of one projection: one row of all heads for each token
        state = {"case": case, "x": values(t, case["heads"], d),
                 "positions": (torch.arange(t, device="cuda") + case["start"]).to(torch.int32)}
        if own:
            from mononn_b200 import Rotary, rotary_runner
            state["out"] = torch.empty_like(state["x"])
            state["call"] = rotary_runner(state["x"], state["positions"], Rotary(**_rotary_config(case)),
                                          out=state["out"])
        return state

    news, pasts = _lengths(case)
    lengths = [a + b for a, b in zip(news, pasts)]
    ps, heads = case["page_size"], case["kv_heads"]
    per = [-(-n // ps) for n in lengths]
    pages = sum(per) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(news), max(per)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    if case["head_major"]:
        k_pages, v_pages = (values(pages, heads, ps, d).transpose(1, 2) for _ in range(2))
    else:
        k_pages, v_pages = (values(pages, ps, heads, d) for _ in range(2))
    indptr = [0]
    for n in news:
        indptr.append(indptr[-1] + n)
    tokens = indptr[-1]
    state = {"case": case, "news": news, "pasts": pasts, "k_pages": k_pages, "v_pages": v_pages, "table": table,
             "indptr": torch.tensor(indptr, dtype=torch.int32, device="cuda"),
             "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
    if case["q_heads"]:
        state["q"] = values(tokens, case["q_heads"], d)
    if case["op"] == "append":
        state["k"], state["v"] = values(tokens, heads, d), values(tokens, heads, d)
    if own:
        from mononn_b200 import PagedCache, Rotary
        cache = PagedCache(k_pages, v_pages, table, state["lengths"])
        if case["op"] == "append":
            rotary = Rotary(**_rotary_config(case)) if case["rotary_dim"] else None
            q = state.get("q")
            state["q_out"] = torch.empty_like(q) if q is not None else None
            state["call"] = cache.append_runner(state["k"], state["v"], state["indptr"], rotary=rotary, q=q,
                                                q_out=state["q_out"])
        else:
            state["out"] = torch.empty_like(state["q"])
            state["call"] = cache.attention_runner(state["q"], state["indptr"], out=state["out"],
                                                   causal=case["causal"], window=case["window"],
                                                   max_new=case["new_high"])
    return state


# ------------------------------------------------------------------ plain form
def _frequencies(c: dict, device) -> tuple[torch.Tensor, float]:
    """Angle of one position for each pair, in 64 bits, and the factor of the rotated values."""
    r, theta, s = c["rotary_dim"], c["theta"], c["factor"]
    i = torch.arange(0, r, 2, dtype=torch.float64, device=device)
    if c["scaling"] == "base" and r > 2:
        theta = theta * s ** (r / (r - 2))
    f = theta ** (-i / r)
    m = 1.0
    if c["scaling"] == "linear":
        f = f / s
    elif c["scaling"] == "bands":
        turns = c["original_length"] * f / (2 * math.pi)
        keep = ((turns - c["low"]) / (c["high"] - c["low"])).clamp(0, 1)
        f = keep * f + (1 - keep) * f / s
    elif c["scaling"] == "ramp":
        def pair(turns):
            return r * math.log(c["original_length"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
        first = max(0, math.floor(pair(c["high"])))
        last = min(r - 1, math.ceil(pair(c["low"])))
        away = ((i / 2 - first) / max(last - first, 0.001)).clamp(0, 1)
        f = (1 - away) * f + away * f / s
        m = 0.1 * math.log(s) + 1.0
    return f, m


def _rotate(x: torch.Tensor, positions: torch.Tensor, c: dict) -> torch.Tensor:
    """x [tokens, heads, head_dim] rotated, in 32 bits (its angles in 64)."""
    r = c["rotary_dim"]
    f, m = _frequencies(c, x.device)
    angle = positions.to(torch.float64)[:, None] * f
    cos, sin = (angle.cos() * m).float()[:, None, :], (angle.sin() * m).float()[:, None, :]
    y = x.float().clone()
    if c["interleaved"]:
        a, b = y[..., 0:r:2].clone(), y[..., 1:r:2].clone()
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = y[..., : r // 2].clone(), y[..., r // 2: r].clone()
        y[..., : r // 2], y[..., r // 2: r] = a * cos - b * sin, b * cos + a * sin
    return y.to(x.dtype)


def _slots(state: dict) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Position, page and row of every new token."""
    ps, table = state["case"]["page_size"], state["table"]
    device = table.device
    new = torch.tensor(state["news"], device=device)
    seq = torch.repeat_interleave(torch.arange(len(state["news"]), device=device), new)
    start = state["indptr"][:-1].long()
    position = torch.arange(seq.numel(), device=device) - start[seq] + (state["lengths"].long() - new)[seq]
    return position, table[seq, position // ps].long(), position % ps


def _plain_append(state: dict):
    case = state["case"]
    position, page, row = _slots(state)
    k, q = state["k"], state.get("q")
    if case["rotary_dim"]:
        c = _rotary_config(case)
        k = _rotate(k, position, c)
        q = _rotate(q, position, c) if q is not None else None
    state["k_pages"][page, row] = k
    state["v_pages"][page, row] = state["v"]
    return [state["k_pages"], state["v_pages"]] + ([q] if q is not None else [])


def _gathered(state: dict, b: int) -> tuple[torch.Tensor, torch.Tensor]:
    n, ps = state["news"][b] + state["pasts"][b], state["case"]["page_size"]
    rows = state["table"][b, : -(-n // ps)].long()
    return (p[rows].flatten(0, 1)[:n] for p in (state["k_pages"], state["v_pages"]))


def _plain_attention(state: dict) -> torch.Tensor:
    case = state["case"]
    heads, d = case["kv_heads"], case["head_dim"]
    group, scale = case["q_heads"] // heads, 1.0 / math.sqrt(d)
    out = torch.empty_like(state["q"])
    at = 0
    for b, (new, past) in enumerate(zip(state["news"], state["pasts"])):
        n = new + past
        k, v = _gathered(state, b)
        q = state["q"][at:at + new].float().view(new, heads, group, d).permute(1, 2, 0, 3)
        # some heads at a time, so that the scores of a long prompt fit
        some = max(1, min(heads, int(2e9 // (group * new * n)) or 1))
        for h in range(0, heads, some):
            kh = k[:, h:h + some].float().permute(1, 2, 0)[:, None]
            vh = v[:, h:h + some].float().permute(1, 0, 2)[:, None]
            s = q[h:h + some] @ kh * scale
            if case["causal"] and (new > 1 or case["window"]):
                pos = torch.arange(past, n, device=s.device)[:, None]
                key = torch.arange(n, device=s.device)[None]
                hidden = key > pos
                if case["window"]:
                    hidden |= key <= pos - case["window"]
                s.masked_fill_(hidden, float("-inf"))
            s -= s.amax(-1, keepdim=True)
            s.exp_()
            o = (s @ vh) / s.sum(-1, keepdim=True)
            out[at:at + new].view(new, heads, group, d)[:, h:h + some] = o.permute(2, 0, 1, 3).to(out.dtype)
        at += new
    return out


def run(state: dict):
    op = state["case"]["op"]
    if own:
        state["call"]()
        if op == "append":
            return [state["k_pages"], state["v_pages"]] + ([state["q_out"]] if "q" in state else [])
        return state["out"]
    if op == "rotary":
        return _rotate(state["x"], state["positions"], _rotary_config(state["case"]))
    return _plain_append(state) if op == "append" else _plain_attention(state)


# ----------------------------------------------------------------- definition
def _turned(x: torch.Tensor, positions: torch.Tensor, c: dict) -> torch.Tensor:
    """The rotation as a product of complex numbers, all of it in 64 bits."""
    r, s = c["rotary_dim"], c["factor"]
    rates = []
    for i in range(r // 2):
        base = c["theta"] * (s ** (r / (r - 2)) if c["scaling"] == "base" and r > 2 else 1.0)
        w = base ** (-2.0 * i / r)
        if c["scaling"] == "linear":
            w /= s
        elif c["scaling"] == "bands":
            share = (c["original_length"] * w / (2 * math.pi) - c["low"]) / (c["high"] - c["low"])
            share = min(1.0, max(0.0, share))
            w *= share + (1 - share) / s
        elif c["scaling"] == "ramp":
            ends = [r * math.log(c["original_length"] / (2 * math.pi * t)) / (2 * math.log(base))
                    for t in (c["high"], c["low"])]
            lo, hi = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), r - 1)
            share = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            w *= (1 - share) + share / s
        rates.append(w)
    size = 1.0 + 0.1 * math.log(s) if c["scaling"] == "ramp" else 1.0
    phase = torch.outer(positions.double(), torch.tensor(rates, dtype=torch.float64, device=x.device))
    turn = torch.polar(torch.full_like(phase, size), phase)[:, None]
    y = x.double()
    part = y[..., :r].unflatten(-1, (r // 2, 2) if c["interleaved"] else (2, r // 2))
    if not c["interleaved"]:
        part = part.transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
    if not c["interleaved"]:
        z = z.transpose(-1, -2)
    return torch.cat([z.flatten(-2), y[..., r:]], -1)


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        return _turned(state["x"], state["positions"], _rotary_config(case))
    heads, d, ps = case["kv_heads"], case["head_dim"], case["page_size"]
    where = state["table"].tolist()
    if case["op"] == "append":
        k, v = state["k"].double(), state["v"].double()
        spot = torch.tensor([p for new, past in zip(state["news"], state["pasts"]) for p in range(past, past + new)],
                            device="cuda")
        q = state["q"].double() if "q" in state else None
        if case["rotary_dim"]:
            c = _rotary_config(case)
            k = _turned(state["k"], spot, c)
            q = _turned(state["q"], spot, c) if q is not None else None
        k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
        at = 0
        for b, (new, past) in enumerate(zip(state["news"], state["pasts"])):
            p = past
            while p < past + new:  # page by page
                n = min(ps - p % ps, past + new - p)
                for pages, src in ((k_pages, k), (v_pages, v)):
                    pages[where[b][p // ps], p % ps: p % ps + n] = src[at:at + n]
                at, p = at + n, p + n
        return [k_pages, v_pages] + ([q] if q is not None else [])
    group = case["q_heads"] // heads
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (new, past) in enumerate(zip(state["news"], state["pasts"])):
        n = new + past
        pages = torch.tensor(where[b][: -(-n // ps)], device="cuda")
        key = torch.arange(n, device="cuda")
        for h in range(heads):
            k = state["k_pages"][pages][:, :, h].reshape(-1, d)[:n].double()
            v = state["v_pages"][pages][:, :, h].reshape(-1, d)[:n].double()
            rows = max(1, int(4e8 // (group * n)))
            for r in range(0, new, rows):
                q = state["q"][first + r:first + min(new, r + rows), h * group:(h + 1) * group].double()
                s = torch.einsum("thd,nd->thn", q, k) / d ** 0.5
                if case["causal"]:
                    p = past + r + torch.arange(q.shape[0], device="cuda")[:, None]
                    sees = key[None] <= p
                    if case["window"]:
                        sees &= p - key[None] < case["window"]
                    s = torch.where(sees[:, None], s, float("-inf"))
                out[first + r:first + r + q.shape[0], h * group:(h + 1) * group] = torch.softmax(s, -1) @ v
        first += new
    return out
