"""Plain 64-bit forms of the operators behind a prompt, and how far a kernel may be from them.

A rounding to type t is off by at most u = finfo(t).eps / 2 of the value. An attention output takes one
for each probability (they are multiplied as values of t) and one at the end; the rest is 32-bit.
"""
import math

import torch


def u(dtype):
    return torch.finfo(dtype).eps / 2


def rotary_rates(r, theta=10000.0, scaling="none", factor=1.0, original_length=0.0, low=None, high=None):
    """Radians per position of every pair, one at a time."""
    rates = []
    for i in range(r // 2):
        base = theta * factor ** (r / (r - 2)) if scaling == "base" and r > 2 else theta
        f = base ** (-2 * i / r)
        if scaling == "linear":
            f /= factor
        if scaling == "bands":
            lo, hi = low or 1.0, high or 4.0
            keep = (original_length / (2 * math.pi / f) - lo) / (hi - lo)
            keep = 0.0 if keep < 0 else 1.0 if keep > 1 else keep
            f = keep * f + (1 - keep) * f / factor
        if scaling == "ramp":
            lo, hi = low or 1.0, high or 32.0
            where = [r * math.log(original_length / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (hi, lo)]
            a, b = max(math.floor(where[0]), 0), min(math.ceil(where[1]), r - 1)
            slow = (i - a) / max(b - a, 0.001)
            slow = 0.0 if slow < 0 else 1.0 if slow > 1 else slow
            f = f * (1 - slow) + f / factor * slow
        rates.append(f)
    return rates


def rotate(x, positions, rates, interleaved, magnitude=1.0):
    """x [tokens, heads, dim] in 64 bits; also the sum of absolute terms behind each element."""
    y, size = x.double().clone(), x.double().abs()
    angle = positions.double()[:, None] * torch.tensor(rates, dtype=torch.float64, device=x.device)
    c, s = angle.cos()[:, None] * magnitude, angle.sin()[:, None] * magnitude
    n = len(rates)
    first = slice(0, 2 * n, 2) if interleaved else slice(0, n)
    second = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
    a, b = x[..., first].double(), x[..., second].double()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = (a.abs() + b.abs()) * magnitude
    size[..., second] = size[..., first]
    return y, size


def assert_rotated(got, want, size, dtype, angle_error=0.0):
    """One rounding to the type; sine, cosine, magnitude, products and sum in 32 bits: 8 half steps of 2^-24 of
    the terms, and what the angle is off by."""
    limit = u(dtype) * want.abs() + (8 * 2.0 ** -24 + angle_error) * (1 + u(dtype)) * size + tiny(dtype)
    off = (got.double() - want).abs()
    assert (off <= limit).all(), f"off by {(off / limit).max().item():.2f} of the limit"


def tiny(dtype):
    """Half the distance between the smallest numbers of the type."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


class Problem:
    """A ragged batch over a paged cache with random pages, and its attention in 64 bits."""

    def __init__(self, news, lengths, kv_heads=2, group=1, dim=64, page=16, dtype=torch.float16, head_major=False,
                 seed=0, spare_rows=0, spread=1.0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def values(*shape):
            return (torch.randn(shape, generator=g, device=device) * spread).to(dtype)

        self.news, self.lens, self.dtype, self.group = list(news), list(lengths), dtype, group
        self.page, self.dim, self.kv_heads = page, dim, kv_heads
        per = [max(1, -(-n // page)) for n in lengths]
        self.pages = sum(per) + 2
        order = torch.randperm(self.pages, generator=g, device=device).to(torch.int32)
        self.table = torch.full((len(per), max(per) + 1), -1, dtype=torch.int32, device=device)
        at = 0
        for b, n in enumerate(per):
            self.table[b, :n] = order[at:at + n]
            at += n
        if head_major:
            self.k, self.v = (values(self.pages, kv_heads, page, dim).transpose(1, 2) for _ in range(2))
        else:
            self.k, self.v = (values(self.pages, page, kv_heads, dim) for _ in range(2))
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        self.starts = starts
        self.indptr = torch.tensor(starts, dtype=torch.int32, device=device)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.q = values(starts[-1] + spare_rows, kv_heads * group, dim)

    def cache(self):
        from mononn_b200 import PagedCache
        return PagedCache(self.k, self.v, self.table, self.lengths)

    def keys(self, b):
        n = self.lens[b]
        rows = self.table[b, : -(-n // self.page)].long()
        return [t[rows].reshape(-1, self.kv_heads, self.dim)[:n].double() for t in (self.k, self.v)]

    def want(self, causal=True, window=0, scale=None):
        """(out, lse, limit of the error of out, of lse) for the tokens of the sequences, in 64 bits."""
        scale = 1 / math.sqrt(self.dim) if scale is None else scale
        device = self.q.device
        outs, lses, limits, lse_limits = [], [], [], []
        for b, n in enumerate(self.news):
            k, v = self.keys(b)
            q = self.q[self.starts[b]:self.starts[b] + n].double()
            kk, vv = (t.repeat_interleave(self.group, 1) for t in (k, v))
            s = torch.einsum("qhd,khd->hqk", q, kk) * scale
            terms = torch.einsum("qhd,khd->hqk", q.abs(), kk.abs()) * scale
            pos = self.lens[b] - n + torch.arange(n, device=device)[:, None]
            key = torch.arange(self.lens[b], device=device)[None]
            see = torch.ones(n, self.lens[b], dtype=torch.bool, device=device)
            if causal:
                see = key <= pos
                if window:
                    see &= key > pos - window
            s = s.masked_fill(~see, -math.inf)
            some = see.any(-1)
            p = torch.where(some[None, :, None], torch.softmax(s, -1), torch.zeros_like(s))
            if self.lens[b] == 0:
                p = p.reshape(q.shape[1], n, 0)
            o = torch.einsum("hqk,khd->qhd", p, vv)
            size = torch.einsum("hqk,khd->qhd", p, vv.abs())
            # a score is a 32-bit sum of dim products, at worst each of them rounded; then scale and exponent. An
            # exponential is off by 2^-22 of itself, or 2.6e-6 + a few 2^-24 < 2^-18 where a polynomial makes it.
            terms = terms.masked_fill(~see, 0.0)
            worst = terms.amax(-1) if self.lens[b] else torch.zeros(q.shape[1], n, device=device, dtype=torch.float64)
            off = worst * (self.dim + 4) * 2.0 ** -24 + 2.0 ** -18
            off_o = off.permute(1, 0)[..., None]
            limit = u(self.dtype) * o.abs() + (u(self.dtype) + 2 * off_o) * (1 + u(self.dtype)) * size + tiny(self.dtype)
            if self.dtype == torch.float16:  # probabilities below the type's normal range
                limit = limit + tiny(self.dtype) * torch.einsum("hqk,khd->qhd", see[None].double().expand_as(p), vv.abs())
            outs.append(o)
            limits.append(limit)
            l = torch.logsumexp(s, -1) if self.lens[b] else torch.full((q.shape[1], n), -math.inf, device=device)
            lses.append(l.permute(1, 0))
            lse_limits.append((off + l.abs().nan_to_num(0, 0, 0) * 2.0 ** -23 + 2.0 ** -20).permute(1, 0))
        return torch.cat(outs), torch.cat(lses), torch.cat(limits), torch.cat(lse_limits)

    def check(self, out, lse=None, **mask):
        o, l, limit, lse_limit = self.want(**mask)
        t = self.starts[-1]
        off = (out[:t].double() - o).abs()
        assert (off <= limit).all(), f"off by {(off / limit).max().item():.2f} of the limit"
        if lse is not None:
            none = torch.isinf(l)
            assert (lse[:t][none] == -math.inf).all()
            assert ((lse[:t].double() - l).abs() <= lse_limit)[~none].all()
