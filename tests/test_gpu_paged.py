"""The operators behind a prompt against their plain 64-bit forms (-m gpu): rotation, append, attention over
pages, and a run of them together."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from mononn_b200 import PagedCache, Rotary, paged_attention_status, rotary  # noqa: E402
from mononn_b200.capi import MononnError, lib  # noqa: E402
from tests.paged_reference import Problem, assert_rotated, rotary_rates, rotate, u  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16
MANY = 10 ** 6  # new tokens of a sequence, as a hint: the kernel for many rows, however small the problem


def attend(p, **kw):
    out = torch.full_like(p.q, 7.0)
    lse = torch.full(p.q.shape[:2], 5.0, device="cuda")
    p.cache().attention(p.q, p.indptr, out=out, lse=lse, **kw)
    paged_attention_status()
    return out, lse


# ------------------------------------------------------------------------------ attention
SINGLE = [1, 1, 1, 1, 1, 1]
LENGTHS = [1, 2, 63, 64, 65, 700]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kv_heads, group, dim, page, head_major", [
    (1, 1, 64, 16, False), (2, 4, 128, 16, False), (3, 5, 80, 8, True), (1, 16, 128, 48, False), (2, 24, 64, 64, True),
    (2, 1, 8, 24, False), (1, 2, 120, 256, True), (4, 3, 72, 32, False)])
def test_single_tokens(dtype, kv_heads, group, dim, page, head_major):
    p = Problem(SINGLE, LENGTHS, kv_heads, group, dim, page, dtype, head_major, seed=dim)
    p.check(*attend(p))


@pytest.mark.parametrize("max_new", [0, 16, MANY])
@pytest.mark.parametrize("dtype, kv_heads, group, dim, page", [
    (F16, 2, 1, 64, 16), (BF16, 1, 4, 128, 32), (F16, 1, 3, 96, 8), (BF16, 2, 8, 64, 128)])
def test_ragged_batch(dtype, kv_heads, group, dim, page, max_new):
    """Sequences without new tokens, without keys, with more new tokens than keys, short and long ones."""
    news = [3, 0, 1, 130, 5, 0, 17, 300, 2]
    lens = [3, 50, 0, 400, 2, 0, 1000, 300, 1]
    p = Problem(news, lens, kv_heads, group, dim, page, dtype, seed=7, spare_rows=5)
    out, lse = attend(p, max_new=max_new)
    p.check(out, lse)
    assert (out[p.starts[-1]:] == 7.0).all() and (lse[p.starts[-1]:] == 5.0).all()
    for b, n in enumerate(news):  # rows before the first key see nothing
        empty = out[p.starts[b]:p.starts[b] + max(0, n - lens[b])]
        assert (empty == 0).all()


@pytest.mark.parametrize("max_new", [0, MANY])
@pytest.mark.parametrize("window", [1, 2, 31, 64, 129, 100000, 2 ** 32 - 1])
def test_window(window, max_new):
    p = Problem([1, 5, 200, 40], [500, 300, 200, 1500], 2, 2, 64, 16, BF16, seed=window % 1000)
    p.check(*attend(p, window=window, max_new=max_new), window=window)


@pytest.mark.parametrize("max_new", [0, MANY])
def test_all_keys(max_new):
    p = Problem([1, 5, 200, 3, 4], [500, 300, 90, 1, 0], 2, 3, 128, 16, F16, seed=3)
    p.check(*attend(p, causal=False, max_new=max_new), causal=False)


@pytest.mark.parametrize("max_new", [1, MANY])
def test_long_split_sequences(max_new):
    """Items that span many CTAs, beside short ones."""
    p = Problem([1, 2, 1, 64], [20001, 70, 9000, 5000], 2, 4, 128, 16, BF16, seed=11)
    p.check(*attend(p, max_new=max_new))


@pytest.mark.parametrize("max_new", [1, MANY])
def test_many_sequences(max_new):
    """More sequences than a CTA has threads, many of them without work."""
    lens = [(37 * i) % 90 for i in range(1500)]
    news = [1 if i % 3 and lens[i] else 0 for i in range(1500)]
    p = Problem(news, lens, 1, 2, 64, 8, F16, seed=5)
    p.check(*attend(p, max_new=max_new))


@pytest.mark.parametrize("max_new", [0, MANY])
def test_what_no_row_sees_may_hold_anything(max_new):
    """NaN and infinities behind the lengths, in pages before the window (their table entries gone) and in
    pages of nobody."""
    for bad in (math.nan, math.inf, -math.inf):
        p = Problem([1, 4, 150], [77, 1005, 330], 2, 2, 64, 16, F16, seed=1)
        window = 100
        seen = torch.zeros(p.pages, p.page, dtype=torch.bool, device="cuda")
        for b, (n, l) in enumerate(zip(p.news, p.lens)):
            first = max(0, l - n + 1 - window)
            for key in range(first, l):
                seen[p.table[b, key // p.page].item(), key % p.page] = True
            p.table[b, : first // p.page] = -1 if b % 2 else 2 ** 30
        keep = seen[:, :, None, None]
        p.k.masked_fill_(~keep, bad)
        p.v.masked_fill_(~keep, bad)
        out, lse = attend(p, window=window, max_new=max_new)
        p.k.masked_fill_(~keep, 0.0)
        p.v.masked_fill_(~keep, 0.0)
        p.table.clamp_(0, p.pages - 1)
        p.check(out, lse, window=window)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("max_new", [1, MANY])
def test_queries_of_no_sequence_may_hold_anything(max_new, dim):
    """They share tiles with the last sequence's, and its results do not change for them."""
    p = Problem([1, 37], [900, 1500], 2, 2, dim, 16, BF16, seed=12, spare_rows=40)
    for bad in (math.nan, math.inf, 3e38):
        p.q[p.starts[-1]:] = bad
        out, lse = attend(p, max_new=max_new)
        p.check(out, lse)


@pytest.mark.parametrize("max_new", [1, MANY])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("jump", [3.0, 40.0, 3000.0])
def test_scores_that_jump(jump, dim, max_new):
    """Rows whose maximum rises little by little, then by a factor that no probability can hold, and falls again;
    others whose highest score comes first."""
    p = Problem([1, 140], [1100, 1400], 1, 2, dim, 16, BF16, seed=13, spread=0.5)
    for b in range(2):
        for i, page in enumerate(range(-(-p.lens[b] // p.page))):
            at = p.table[b, page].item()
            size = jump if i % 17 == 11 else 0.02 * i
            p.k[at] = (torch.sign(p.q[p.starts[b], 0]).float() * size).to(BF16)
    p.check(*attend(p, max_new=max_new))


@pytest.mark.parametrize("max_new", [0, MANY])
def test_pages_out_of_range_read_as_zeros(max_new):
    p = Problem([1, 200], [100, 260], 1, 2, 64, 16, F16, seed=2)
    p.table[0, 2], p.table[1, 0], p.table[1, 5], p.table[1, 9] = -1, p.pages, 2 ** 31 - 1, -2 ** 31
    out, lse = attend(p, max_new=max_new)
    zero = torch.zeros_like(p.k[:1])
    p.k, p.v = torch.cat([p.k, zero]), torch.cat([p.v, zero])
    p.table[(p.table < 0) | (p.table >= p.pages)] = p.pages
    p.check(out, lse)


@pytest.mark.parametrize("max_new", [0, MANY])
def test_lengths_and_indptr_out_of_range_stay_in_bounds(max_new):
    p = Problem([1, 30], [100, 100], 1, 2, 64, 16, F16, seed=2)
    p.lengths.copy_(torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32))
    p.indptr.copy_(torch.tensor([-3, 2, 2 ** 31 - 1], dtype=torch.int32))
    out, _ = attend(p, max_new=max_new)
    assert (out[2:] == 0).all()  # a length below zero: no keys


@pytest.mark.parametrize("max_new", [0, MANY])
def test_strides_of_a_fused_projection(max_new):
    """q as a slice of one projection, out as a slice of a wider buffer, a cache with both in one page."""
    p = Problem([1, 90, 7], [300, 130, 70], 2, 2, 64, 16, BF16, seed=4)
    t = p.starts[-1]
    wide = torch.randn(t, 8, 64, device="cuda").to(BF16)
    wide[:, 2:6] = p.q
    both = torch.empty(p.pages, 2, 16, 2, 64, device="cuda", dtype=BF16)
    both[:, 0], both[:, 1] = p.k, p.v
    result = torch.full((t, 4, 3, 72), 3.0, device="cuda", dtype=BF16)
    cache = PagedCache(both[:, 0], both[:, 1], p.table, p.lengths)
    out = cache.attention(wide[:, 2:6], p.indptr, out=result[:, :, 1, :64], max_new=max_new)
    p.check(out)
    result[:, :, 1, :64] = 3.0
    assert (result == 3.0).all()


@pytest.mark.parametrize("max_new", [0, MANY])
@pytest.mark.parametrize("scale", [1e-6, 0.5, 4.0])
def test_scales(scale, max_new):
    """Nearly even probabilities, and ones that one key takes whole; scores far from zero."""
    p = Problem([1, 140], [900, 300], 1, 2, 64, 16, F16, seed=6, spread=2.0)
    p.check(*attend(p, scale=scale, max_new=max_new), scale=scale)


@pytest.mark.parametrize("max_new", [0, MANY])
def test_rising_scores(max_new):
    """The running maximum goes up at every step."""
    p = Problem([1, 130], [2000, 1500], 1, 1, 64, 16, BF16, seed=8)
    for b in range(2):
        for page in range(-(-p.lens[b] // p.page)):
            at = p.table[b, page].item()
            p.k[at] = (p.q[0, 0].float() * (page + 1) / 40).to(BF16)
    p.q[1:] = p.q[0]
    p.check(*attend(p, max_new=max_new))


@pytest.mark.parametrize("max_new", [1, MANY])
def test_offsets_beyond_32_bits(max_new):
    """A cache of more than 2^32 bytes and 2^31 elements in each of its two buffers."""
    pages, page, heads, dim = 2 ** 31 // (16 * 2 * 128) + 64, 16, 2, 128
    k, v = (torch.empty(pages, page, heads, dim, dtype=F16, device="cuda") for _ in range(2))
    p = Problem([1, 100], [90, 170], heads, 2, dim, page, F16, seed=9)
    far = torch.arange(p.pages, device="cuda", dtype=torch.int32) + (pages - p.pages)
    k[far.long()], v[far.long()] = p.k, p.v
    table = torch.where(p.table >= 0, p.table + (pages - p.pages), p.table)
    out = PagedCache(k, v, table, p.lengths).attention(p.q, p.indptr, max_new=max_new)
    p.check(out)
    # and the append to the far end
    new_k, new_v = (torch.randn(p.starts[-1], heads, dim, device="cuda").to(F16) for _ in range(2))
    PagedCache(k, v, table, p.lengths).append(new_k, new_v, p.indptr)
    spot = p.lens[0] - 1
    at = table[0, spot // page].item()
    assert torch.equal(k[at, spot % page], new_k[0]) and torch.equal(v[at, spot % page], new_v[0])


@pytest.mark.parametrize("max_new", [1, MANY])
def test_same_bits_again_in_a_graph_and_on_another_stream(max_new):
    p = Problem([1, 1, 40, 1], [9000, 31, 700, 2500], 2, 4, 128, 16, BF16, seed=10)
    first, lse = attend(p, max_new=max_new)
    for _ in range(3):
        again, lse2 = attend(p, max_new=max_new)
        assert torch.equal(first, again) and torch.equal(lse, lse2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = p.cache().attention(p.q, p.indptr, max_new=max_new)
    explicit = p.cache().attention(p.q, p.indptr, max_new=max_new, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(first, other) and torch.equal(first, explicit)
    # two graphs at once, each with a workspace of its own; then other contents of the same buffers
    cache = p.cache()
    outs, graphs = [torch.zeros_like(p.q) for _ in range(2)], []
    for out in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache.attention(p.q, p.indptr, out=out, max_new=max_new)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, outs[0]) and torch.equal(first, outs[1])
    p.lens = [8000, 3, 699, 2400]
    p.lengths.copy_(torch.tensor(p.lens, dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    p.check(outs[0])
    paged_attention_status()


def test_refused_on_the_gpu():
    p = Problem([1], [5000], 1, 1, 64, 16, F16)
    with pytest.raises(Exception, match="workspace"):
        p.cache().attention(p.q, p.indptr, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    host = torch.zeros(4, 16, 1, 64, dtype=F16)
    cache = PagedCache(host, host.clone(), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    new = torch.zeros(1, 1, 64, dtype=F16)
    with pytest.raises(Exception, match="device memory"):
        cache.append(new, new, torch.zeros(2, dtype=torch.int32), stream=torch.cuda.current_stream())


# -------------------------------------------------------------------------- rotation, append
ROTATIONS = [dict(rotary_dim=64), dict(rotary_dim=32, interleaved=True), dict(rotary_dim=48, scaling="linear", factor=3.0),
             dict(rotary_dim=20, scaling="base", factor=4.0), dict(rotary_dim=6, interleaved=True),
             dict(rotary_dim=64, interleaved=True, scaling="bands", factor=8.0, original_length=4096),
             dict(rotary_dim=64, scaling="ramp", factor=4.0, original_length=4096), dict(rotary_dim=2, magnitude=0.5)]


def rates_of(c):
    c = dict(c)
    interleaved, magnitude = c.pop("interleaved", False), c.pop("magnitude", None)
    if magnitude is None:
        magnitude = 0.1 * math.log(c["factor"]) + 1 if c.get("scaling") == "ramp" else 1.0
    return rotary_rates(c.pop("rotary_dim"), **c), interleaved, magnitude


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("config", ROTATIONS)
@pytest.mark.parametrize("dim, heads, tokens", [(64, 3, 1), (80, 12, 37), (67, 2, 5), (256, 1, 3), (64, 300, 2)])
def test_rotary(dtype, config, dim, heads, tokens):
    x = torch.randn(tokens, heads, dim, device="cuda").to(dtype)
    pos = torch.randint(0, 5000, (tokens,), device="cuda", dtype=torch.int32)
    want, size = rotate(x, pos, *rates_of(config))
    keep = x.clone()
    out = rotary(x, pos, Rotary(**config), out=torch.full_like(x, 9.0))
    assert torch.equal(x, keep)
    assert_rotated(out, want, size, dtype)
    r = config["rotary_dim"]
    assert torch.equal(out[..., r:], x[..., r:])
    assert rotary(x, pos, Rotary(**config)) is x
    assert torch.equal(x, out)


def test_rotary_far_positions():
    """The angle of any 32-bit position, to what 64 bits of it are worth."""
    pos = torch.tensor([0, 1, -1, 65535, 1000003, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    x = torch.randn(7, 2, 64, device="cuda").to(F16)
    want, size = rotate(x, pos, rotary_rates(64), False)
    # position x rate / 2 pi: both sides round it, and the rate itself, by 2^-53 of up to 2^31 radians, some times over
    assert_rotated(rotary(x, pos, Rotary(64), out=torch.empty_like(x)), want, size, F16, 8 * 2.0 ** (31 - 53))


def test_rotary_strides():
    wide = torch.randn(9, 5, 3, 70, device="cuda").to(BF16)
    x, pos = wide[:, :, 1, 3:67], torch.arange(9, dtype=torch.int32, device="cuda")  # not aligned to 16 bytes
    want, size = rotate(x, pos, rotary_rates(64), False)
    keep = wide.clone()
    rotary(x, pos, Rotary(64))
    assert_rotated(x, want, size, BF16)
    wide[:, :, 1, 3:67] = keep[:, :, 1, 3:67]
    assert torch.equal(wide, keep)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("config", [None, dict(rotary_dim=64), dict(rotary_dim=32, interleaved=True),
                                    dict(rotary_dim=10, scaling="linear", factor=2.0)])
@pytest.mark.parametrize("page, head_major, dim, kv_heads, q_heads", [
    (16, False, 64, 2, 4), (8, True, 80, 1, 0), (1, False, 64, 3, 3), (5, True, 66, 2, 2), (64, False, 128, 32, 32)])
def test_append(dtype, config, page, head_major, dim, kv_heads, q_heads):
    news, lens = [1, 0, 5, 40, 3, 2], [33, 20, 5, 90, 1, 0]  # the last ones have tokens without a place
    p = Problem(news, lens, kv_heads, 1, dim, page, dtype, head_major, seed=1)
    t = p.starts[-1]
    k, v = (torch.randn(t + 2, kv_heads, dim, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn(t + 2, q_heads, dim, device="cuda").to(dtype) if q_heads else None
    at = torch.cat([torch.arange(l - n, l, dtype=torch.int32, device="cuda") for n, l in zip(news, lens)])
    old_k, old_v = p.k.clone(), p.v.clone()
    q_out = torch.full_like(q, 9.0) if q_heads else None
    p.cache().append(k, v, p.indptr, rotary=Rotary(**config) if config else None, q=q, q_out=q_out)
    rates, interleaved, magnitude = rates_of(config) if config else ([], False, 1.0)
    want_k, size_k = rotate(k[:t], at, rates, interleaved, magnitude)
    written = torch.zeros(p.pages, page, dtype=torch.bool, device="cuda")
    i = 0
    for b, n in enumerate(news):
        for j in range(n):
            pos = lens[b] - n + j
            if pos >= 0:
                where = p.table[b, pos // page].item()
                written[where, pos % page] = True
                assert_rotated(p.k[where, pos % page], want_k[i], size_k[i], dtype)
                assert torch.equal(p.v[where, pos % page], v[i])
            i += 1
    assert torch.equal(p.k[~written], old_k[~written]) and torch.equal(p.v[~written], old_v[~written])
    if q_heads:
        want_q, size_q = rotate(q[:t], at, rates, interleaved, magnitude)
        assert_rotated(q_out[:t], want_q, size_q, dtype)
        assert (q_out[t:] == 9.0).all()


def test_append_positions_bad_pages_and_in_place():
    p = Problem([2, 3], [40, 20], 1, 1, 64, 16, F16, seed=2)
    p.table[0, 2], p.table[1, 1] = -1, p.pages  # the places of sequence 0's tokens, of all but one of sequence 1's
    k, v, q = (torch.randn(5, 1, 64, device="cuda").to(F16) for _ in range(3))
    pos = torch.tensor([5, 900, 3, 70000, 8], dtype=torch.int32, device="cuda")
    old = p.k.clone()
    want_q, size_q = rotate(q, pos, rotary_rates(64), False)
    want_k, size_k = rotate(k, pos, rotary_rates(64), False)
    assert p.cache().append(k, v, p.indptr, rotary=Rotary(64), positions=pos, q=q) is q
    assert_rotated(q, want_q, size_q, F16)
    # sequence 1's tokens are at 17, 18, 19: page 1, which is out of range
    assert torch.equal(p.k, old)
    p.table[1, 1] = 3
    p.cache().append(k, v, p.indptr, rotary=Rotary(64), positions=pos)
    assert_rotated(p.k[3, 1:4], want_k[2:], size_k[2:], F16)
    old[3, 1:4] = p.k[3, 1:4]
    assert torch.equal(p.k, old)


def test_append_to_many_sequences():
    lens = [(11 * i) % 40 + 1 for i in range(3000)]
    p = Problem([1] * 3000, lens, 1, 1, 64, 8, F16, seed=2)
    k, v = (torch.randn(3000, 1, 64, device="cuda").to(F16) for _ in range(2))
    p.cache().append(k, v, p.indptr)
    spot = p.lengths.long() - 1
    page = p.table[torch.arange(3000, device="cuda"), spot // 8].long()
    assert torch.equal(p.k[page, spot % 8], k) and torch.equal(p.v[page, spot % 8], v)


# ------------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype, group, dim", [(F16, 1, 64), (BF16, 4, 128)])
def test_prompt_in_pieces_then_tokens(dtype, group, dim):
    """A prompt in one piece, in chunks, and token by token: rotation and append in one launch, then attention,
    captured once for the single tokens and replayed. All agree with attention over the whole in 64 bits."""
    n, heads, page = 200, 2, 16
    config = Rotary(dim, scaling="bands", factor=4.0, original_length=64)
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(n, h, dim, generator=g, device="cuda").to(dtype) for h in (heads * group, heads, heads))
    table = torch.randperm(32, generator=g, device="cuda").to(torch.int32)[None, :16].contiguous()

    def fresh():
        pages = [torch.full((32, page, heads, dim), math.nan, dtype=dtype, device="cuda") for _ in range(2)]
        return PagedCache(*pages, table, torch.zeros(1, dtype=torch.int32, device="cuda"))

    def piece(cache, a, b):
        cache.lengths.fill_(b)
        indptr = torch.tensor([0, b - a], dtype=torch.int32, device="cuda")
        turned = cache.append(k[a:b], v[a:b], indptr, rotary=config, q=q[a:b], q_out=torch.empty_like(q[a:b]))
        return cache.attention(turned, indptr, max_new=b - a)

    whole = fresh()
    full = piece(whole, 0, n)
    # the cache holds the rotated keys; attention over them, exactly
    p = Problem([n], [n], heads, group, dim, page, dtype)
    p.k, p.v, p.table = whole.k_pages, whole.v_pages, table
    p.q = rotary(q, torch.arange(n, dtype=torch.int32, device="cuda"), config, out=torch.empty_like(q))
    p.check(full)
    chunks = fresh()
    p.check(torch.cat([piece(chunks, a, min(n, a + 67)) for a in range(0, n, 67)]))
    assert torch.equal(chunks.k_pages.nan_to_num(9), whole.k_pages.nan_to_num(9))

    single = fresh()
    one_q, one_k, one_v = q[:1].clone(), k[:1].clone(), v[:1].clone()
    indptr = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    turned, out = torch.empty_like(one_q), torch.empty_like(one_q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        single.append(one_k, one_v, indptr, rotary=config, q=one_q, q_out=turned)
        single.attention(turned, indptr, out=out, max_new=1)
    got = []
    for i in range(n):
        single.lengths.fill_(i + 1)
        one_q.copy_(q[i:i + 1]), one_k.copy_(k[i:i + 1]), one_v.copy_(v[i:i + 1])
        graph.replay()
        got.append(out.clone())
    p.check(torch.cat(got))
    assert torch.equal(single.k_pages.nan_to_num(9), whole.k_pages.nan_to_num(9))
    paged_attention_status()


def test_follows_the_prompt_of_the_stand_alone_attention():
    """Keys of a prompt whose attention mononn_attention_noalloc computed go on in a cache: the same rows."""
    from mononn_b200.module import attention_noalloc, attention_noalloc_status
    seq, heads = 100, 3
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = (torch.randn(seq, heads, 64, generator=g, device="cuda").to(F16) for _ in range(3))
    vt = torch.zeros(heads * 64, 104, dtype=F16, device="cuda")
    vt[:, :seq] = v.reshape(seq, heads * 64).T
    old = torch.empty_like(q)
    attention_noalloc(q.data_ptr(), k.data_ptr(), vt.data_ptr(), None, old.data_ptr(), 1, heads, seq, heads * 64, 104,
                      heads * 64, 0.125, causal=True)
    attention_noalloc_status()
    p = Problem([seq], [seq], heads, 1, 64, 16, F16, seed=4)
    p.cache().append(k, v, p.indptr)
    p.q = q
    out, _ = attend(p)
    p.check(out)
    _, _, limit, _ = p.want()
    # the other one rounds its probabilities after the division: two such limits apart at most, by the same count
    assert ((out.double() - old.double()).abs() <= 2 * limit + 2 * u(F16) * out.double().abs()).all()


# ------------------------------------------------------------------------------ further edges
@pytest.mark.parametrize("max_new", [1, MANY])
@pytest.mark.parametrize("group, dim", [(200, 64), (129, 128), (128, 64), (65, 128), (64, 128), (24, 64), (7, 128),
                                        (5, 80), (3, 64)])
def test_wide_and_odd_groups(group, dim, max_new):
    """Groups that leave rows of a tile unused, fill it alone, or are too wide for one."""
    p = Problem([1, 9, 0, 70], [40, 700, 3, 333], 1, group, dim, 16, BF16, seed=group)
    p.check(*attend(p, max_new=max_new))


@pytest.mark.parametrize("mask", [{}, dict(window=200), dict(window=3), dict(causal=False)])
@pytest.mark.parametrize("dtype, group, dim", [(F16, 4, 64), (BF16, 4, 128), (F16, 1, 128), (BF16, 3, 96), (BF16, 5, 48)])
def test_drafts_of_many_sequences(dtype, group, dim, mask):
    """Row tiles that are not full, where both of a CTA take turns with the keys; and sequences beyond the hint, whose
    rows fill one tile, or more than both."""
    g = torch.Generator().manual_seed(dim)
    news = torch.randint(0, 25, (48,), generator=g).tolist()
    lens = (torch.randint(0, 1800, (48,), generator=g) + torch.tensor(news)).tolist()
    news[7], lens[7], news[20], lens[20], news[21], lens[21], news[30], lens[30] = 128 // group, 4000, 300, 700, 33, 40, 25, 1
    p = Problem(news, lens, 2, group, dim, 16, dtype, seed=dim)
    p.check(*attend(p, max_new=24, **mask), **mask)


@pytest.mark.parametrize("max_new", [1, MANY])
@pytest.mark.parametrize("pages", [31, 32, 33, 64, 65])
def test_caches_around_the_size_from_which_items_are_split(pages, max_new):
    p = Problem([1, 40, 2, 0], [pages * 16, pages * 16 - 7, 17, 300], 2, 4, 64, 16, F16, seed=pages)
    p.table = p.table[:, :pages].contiguous()
    p.check(*attend(p, max_new=max_new))


@pytest.mark.parametrize("max_new", [1, MANY])
def test_pages_that_end_inside_a_tile(max_new):
    """Page sizes that share no large factor with a tile of keys."""
    for page in (8, 24, 40, 56, 200, 1000):
        p = Problem([1, 33, 5], [1013, 700, page], 2, 2, 128, page, F16, seed=page)
        p.check(*attend(p, max_new=max_new))


@pytest.mark.parametrize("max_new", [1, MANY])
def test_nothing_new(max_new):
    """No sequence has a new token: nothing is written."""
    p = Problem([0, 0, 0], [5, 900, 0], 2, 2, 64, 16, F16, spare_rows=3)
    out, lse = attend(p, max_new=max_new)
    assert (out == 7.0).all() and (lse == 5.0).all()
    new = torch.ones(3, 2, 64, device="cuda", dtype=F16)
    before = p.k.clone(), p.v.clone()
    q = torch.randn(3, 4, 64, device="cuda").to(F16)
    keep = q.clone()
    p.cache().append(new, new, p.indptr, Rotary(64), q=q)
    assert torch.equal(p.k, before[0]) and torch.equal(p.v, before[1]) and torch.equal(q, keep)


def test_tensors_without_elements():
    p = Problem([0, 0], [5, 9], 2, 2, 64, 16, F16)
    cache, none = p.cache(), torch.empty(0, 2, 64, device="cuda", dtype=F16)
    assert cache.attention(p.q, p.indptr).shape == (0, 4, 64)
    assert cache.append(none, none, p.indptr, Rotary(64), q=p.q).shape == (0, 4, 64)
    assert rotary(p.q, torch.empty(0, device="cuda", dtype=torch.int32), Rotary(64)).shape == (0, 4, 64)
    empty = PagedCache(p.k, p.v, p.table[:0], p.lengths[:0])
    start = torch.zeros(1, device="cuda", dtype=torch.int32)
    out = torch.full((2, 4, 64), 7.0, device="cuda", dtype=F16)
    empty.attention(torch.zeros_like(out), start, out=out)
    assert (out == 7.0).all()


@pytest.mark.parametrize("max_new", [1, MANY])
def test_overlapping_sequences_stay_in_bounds(max_new):
    """An indptr that decreases is not allowed; what it leads to stays within the tensors all the same."""
    p = Problem([31, 0, 0], [200, 90, 900], 2, 2, 64, 16, F16, spare_rows=4)
    p.indptr.copy_(torch.tensor([0, 31, 0, 31], dtype=torch.int32))
    out, lse = attend(p, max_new=max_new)
    assert (out[31:] == 7.0).all() and (lse[31:] == 5.0).all()
    assert torch.isfinite(out[:31]).all()


@pytest.mark.parametrize("max_new", [1, MANY])
def test_a_runner_reads_what_its_buffers_hold(max_new):
    p = Problem([1, 30, 2], [400, 900, 77], 2, 2, 64, 16, BF16, seed=21)
    run = p.cache().attention_runner(p.q, p.indptr, max_new=max_new)
    run()
    p.check(run.out)
    p.q.copy_(torch.randn(p.q.shape, device="cuda"))
    p.news, p.lens, p.starts = [3, 0, 30], [399, 20, 64], [0, 3, 3, 33]
    p.indptr.copy_(torch.tensor(p.starts, dtype=torch.int32))
    p.lengths.copy_(torch.tensor(p.lens, dtype=torch.int32))
    run()
    p.check(run.out)


def test_calls_on_several_streams_at_once():
    """Each with a workspace of its own, over one cache."""
    p = Problem([1, 64, 1], [9000, 5000, 20000], 2, 4, 128, 16, F16, seed=23)
    first, _ = attend(p)
    streams = [torch.cuda.Stream() for _ in range(4)]
    runs = []
    for i, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
        runs.append(p.cache().attention_runner(p.q, p.indptr, max_new=1 if i % 2 else MANY, stream=s))
    for _ in range(20):
        for run in runs:
            run()
    torch.cuda.synchronize()
    paged_attention_status()
    for run in runs[::2]:
        assert torch.equal(run.out, runs[0].out)
    for run in runs[1::2]:
        assert torch.equal(run.out, runs[1].out)
        p.check(run.out)
    p.check(runs[0].out)
    p.check(first)


@pytest.mark.parametrize("dim, heads", [(64, 3), (128, 9), (67, 2), (80, 1), (128, 12), (128, 40), (128, 70)])
@pytest.mark.parametrize("config", [dict(rotary_dim=64), dict(rotary_dim=32, interleaved=True)])
@pytest.mark.parametrize("tokens", [591, 592, 595, 2001])
def test_rotary_of_many_tokens(tokens, config, dim, heads):
    """Enough tokens that a block takes several, and a last block that is not full."""
    x = torch.randn(tokens, heads, dim, device="cuda").to(BF16)
    pos = torch.randint(0, 5000, (tokens,), device="cuda", dtype=torch.int32)
    want, size = rotate(x, pos, *rates_of(config))
    out = rotary(x, pos, Rotary(**config), out=torch.full_like(x, 9.0))
    assert_rotated(out, want, size, BF16)
    assert torch.equal(out[..., config["rotary_dim"]:], x[..., config["rotary_dim"]:])


def test_vectors_and_single_elements_agree():
    """The same rows at addresses that are and are not multiples of 16 bytes."""
    x = torch.randn(700, 5, 128, device="cuda").to(F16)
    pos = torch.arange(700, device="cuda", dtype=torch.int32) * 31
    odd = torch.empty(700 * 5 * 128 + 1, device="cuda", dtype=F16)[1:].view(700, 5, 128)
    for config in (dict(rotary_dim=128), dict(rotary_dim=64, interleaved=True)):
        odd.copy_(x)
        rotary(odd, pos, Rotary(**config))
        assert torch.equal(odd, rotary(x, pos, Rotary(**config), out=torch.empty_like(x)))


@pytest.mark.parametrize("heads, kv_heads, order", [(4, 2, "qkv"), (32, 8, "qkv"), (5, 1, "kvq"), (6, 3, "kqv"), (2, 2, "qkv")])
def test_queries_of_a_fused_projection_turned_in_place(heads, kv_heads, order):
    """Grouped heads as slices of one projection: the queries turn in place beside the keys and values that are stored."""
    p = Problem([1, 40, 7], [300, 130, 7], kv_heads, heads // kv_heads, 64, 16, F16, seed=heads)
    t = p.starts[-1]
    wide = torch.randn(t, heads + 2 * kv_heads, 64, device="cuda").to(F16)
    parts, at = {}, 0
    for name in order:
        n = heads if name == "q" else kv_heads
        parts[name] = wide[:, at:at + n]
        at += n
    config = Rotary(64)
    apart = {name: x.clone() for name, x in parts.items()}
    pages = p.k.clone(), p.v.clone()
    want = PagedCache(*pages, p.table, p.lengths).append(apart["k"], apart["v"], p.indptr, config, q=apart["q"])
    keep = {name: parts[name].clone() for name in "kv"}
    assert p.cache().append(parts["k"], parts["v"], p.indptr, config, q=parts["q"]) is parts["q"]
    assert torch.equal(parts["q"], want)
    assert torch.equal(p.k, pages[0]) and torch.equal(p.v, pages[1])
    assert all(torch.equal(parts[name], keep[name]) for name in "kv")


def test_workspaces_that_overlap_are_refused():
    p = Problem([1], [5000], 1, 1, 64, 16, F16)
    need = p.cache().attention_runner(p.q, p.indptr)
    room = torch.empty(1 << 23, dtype=torch.uint8, device="cuda")
    out = room[4096:4096 + 128].view(F16).view(1, 1, 64)
    with pytest.raises(ValueError, match="workspace overlaps out"):
        p.cache().attention_runner(p.q, p.indptr, out=out, workspace=room)
    assert torch.equal(p.cache().attention(p.q, p.indptr, workspace=room), (need(), need.out)[1])


FEW_BARRIERS, MANY_BARRIERS = [1, 2, 3, 4, 5, 6], [1, 2, 3, 4, 5, 7, 9, 10, 11, 12, 13]


@pytest.mark.parametrize("new, dim, barrier", [(1, 128, b) for b in FEW_BARRIERS] + [(1, 64, 1), (1, 64, 4)]
                         + [(40, 128, b) for b in MANY_BARRIERS] + [(40, 64, b) for b in MANY_BARRIERS + [8]])
def test_waits_that_run_out_are_reported(new, dim, barrier):
    """An arrival that nobody makes: every CTA gives up after its bound, lets its copies land and returns; the status says
    so once, rows of no sequence stay as they were, and the next call is right."""
    news = [new] * 160
    # one sequence so long that items are split, and the join runs over what is there
    p = Problem(news, [new + 150 + i for i in range(159)] + [1300], 6, 2, dim, 16, BF16, seed=barrier, spare_rows=3)
    paged_attention_status()
    assert lib().mononn_debug_paged_skew(barrier) == 0
    out = torch.full_like(p.q, 7.0)
    cache = p.cache()
    cache.attention(p.q, p.indptr, out=out, max_new=new)
    with pytest.raises(MononnError) as e:
        paged_attention_status()
    assert e.value.code == -6
    assert (out[p.starts[-1]:] == 7.0).all()
    paged_attention_status()
    p.check(*attend(p, max_new=new))


@pytest.mark.parametrize("news, lens, kv_heads, group, dim, dtype, max_new", [
    ([1], [300], 12, 1, 64, F16, 1), ([1] * 64, [250] * 64, 2, 4, 128, BF16, 1), ([500], [500], 2, 4, 128, BF16, 500),
    ([16, 1, 0], [2000, 3, 0], 2, 4, 128, BF16, 16), ([1, 40], [129, 40], 2, 2, 80, F16, 0)])
def test_short_sequences_in_a_table_of_a_whole_context(news, lens, kv_heads, group, dim, dtype, max_new):
    """The width of the table decides whether items may be split and which kernel runs; the results are as right."""
    p = Problem(news, lens, kv_heads, group, dim, 16, dtype, seed=dim)
    p.check(*attend(p, max_new=max_new))
    wide = torch.full((len(news), 8192), -1, dtype=torch.int32, device="cuda")
    wide[:, :p.table.shape[1]] = p.table
    p.table = wide
    p.check(*attend(p, max_new=max_new))


def test_tokens_that_fall_on_one_place():
    """Two sequences whose new tokens share a page: equal tokens are there whole, others element by element."""
    p = Problem([1, 1, 3], [20, 20, 40], 2, 1, 64, 16, F16, seed=3)
    p.table[1] = p.table[0]
    k, v = (torch.randn(5, 2, 64, device="cuda").to(F16) for _ in range(2))
    for same in (False, True):
        if same:
            k[1], v[1] = k[0], v[0]
        p.cache().append(k, v, p.indptr)
        for pages, new in ((p.k, k), (p.v, v)):
            got = pages[p.table[0, 1].item(), 3]
            assert ((got == new[0]) | (got == new[1])).all()
            assert torch.equal(pages[p.table[2, 2].item(), 5:8], new[2:])


@pytest.mark.parametrize("max_new", [1, MANY])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("keys", [200, 5000])
def test_scores_that_leave_32_bits_become_nan(keys, dim, max_new):
    """q.k is 2^126 and more, 32-bit, but not when it is scaled: never taken for a row that sees nothing. Rows beside them are
    right, rows without a key are zeros."""
    p = Problem([1, 40, 3], [keys, keys, 2], 1, 2, dim, 16, BF16, seed=dim)
    p.q[0], p.q[11] = 2.0 ** 60, 2.0 ** 60
    for b in (0, 1):
        rows = p.table[b, : -(-keys // 16)].long()
        p.k[rows] = 2.0 ** 60
    p.q[1:11], p.q[12:41] = p.q[1:11] * 2.0 ** -60, p.q[12:41] * 2.0 ** -60
    out, lse = attend(p, scale=4.0, max_new=max_new)
    assert out[[0, 11]].isnan().all() and lse[[0, 11]].isnan().all()
    assert (out[41] == 0).all() and (lse[41] == -math.inf).all()
    keep = torch.ones(44, dtype=torch.bool, device="cuda")
    keep[[0, 11]] = False
    p.q[[0, 11]] = 0
    want, log, limit, log_limit = p.want(scale=4.0)
    off = (out.double() - want).abs()
    assert (off <= limit)[keep].all()
    keep[41] = False
    assert ((lse.double() - log).abs() <= log_limit)[keep].all()
