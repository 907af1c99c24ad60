"""What the operators behind a prompt refuse, and the rates of their rotation: host code, no GPU needed."""
import ctypes as C
import math

import pytest
import torch

from mononn_b200 import PagedCache, Rotary, capi, rotary_runner
from tests.paged_reference import rotary_rates

FAKE = 1 << 20  # an aligned address that is never followed


def cache_args(**change):
    base = dict(k_pages=FAKE, v_pages=2 * FAKE, page_stride=16 * 2 * 64, token_stride=2 * 64, head_stride=64,
                page_table=FAKE, table_stride=4, lengths=FAKE, sequences=2, max_pages=4, num_pages=9, page_size=16,
                kv_heads=2, head_dim=64, dtype=0)
    return capi.PagedCacheArgs(**{**base, **change})


def attention_args(**change):
    base = dict(q=FAKE, out=FAKE, lse=None, q_token_stride=4 * 64, q_head_stride=64, out_token_stride=4 * 64,
                out_head_stride=64, indptr=FAKE, tokens=3, q_heads=4, scale=0.0, causal=1, window=0, max_new=0,
                workspace=None, workspace_bytes=0)
    return capi.PagedAttentionArgs(**{**base, **change})


def append_args(**change):
    base = dict(k=FAKE, v=FAKE, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64, q=None,
                q_out=None, indptr=FAKE, positions=None, tokens=3, q_heads=0)
    return capi.PagedAppendArgs(**{**base, **change})


def rotary_args(**change):
    base = dict(x=FAKE, out=FAKE, x_token_stride=128, x_head_stride=64, out_token_stride=128, out_head_stride=64,
                positions=FAKE, tokens=3, heads=2, head_dim=64, dtype=0)
    return capi.RotaryArgs(**{**base, **change})


def attend(cache=None, args=None):
    return capi.lib().mononn_paged_attention(C.byref(cache or cache_args()), C.byref(args or attention_args()), None)


def append(cache=None, args=None, table=None):
    return capi.lib().mononn_paged_append(C.byref(cache or cache_args()), C.byref(table) if table else None,
                                          C.byref(args or append_args()), None)


# Arguments in order get as far as the device: there is none here, and the address is none of a GPU there.
PASSES = (-5, -1)


@pytest.mark.parametrize("change", [
    dict(k_pages=None), dict(page_table=None), dict(lengths=None), dict(page_size=0), dict(kv_heads=0),
    dict(head_dim=0), dict(num_pages=0), dict(max_pages=0), dict(token_stride=63), dict(head_stride=32),
    dict(page_stride=8), dict(table_stride=3), dict(token_stride=-128), dict(page_table=FAKE + 2),
    dict(page_stride=1 << 39)])
def test_cache_refused(lib_built, change):
    assert attend(cache=cache_args(**change)) == -1
    assert append(cache=cache_args(**change)) == -1


@pytest.mark.parametrize("change, code", [
    (dict(dtype=2), -3), (dict(num_pages=1 << 31), -10), (dict(max_pages=1 << 27, table_stride=1 << 27), -10),
    (dict(head_dim=264, head_stride=264), -10), (dict(sequences=(1 << 24) + 1), -10)])
def test_cache_outside_of_the_supported(lib_built, change, code):
    assert attend(cache=cache_args(**change)) == code
    assert append(cache=cache_args(**change)) == code


@pytest.mark.parametrize("change", [
    dict(q=None), dict(out=None), dict(indptr=None), dict(q_heads=0), dict(q_heads=3), dict(q=FAKE + 2),
    dict(out=FAKE + 8), dict(q_token_stride=4 * 64 + 1), dict(out_head_stride=60), dict(out_head_stride=32),
    dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(causal=0, window=5), dict(lse=FAKE + 1),
    dict(indptr=FAKE + 2), dict(q_token_stride=-64)])
def test_attention_refused(lib_built, change):
    assert attend(args=attention_args(**change)) == -1
    assert b"attention" in capi.lib().mononn_last_error()


@pytest.mark.parametrize("cache, args, code", [
    (dict(head_dim=60), {}, -3), (dict(head_dim=136, head_stride=136, token_stride=272), {}, -3),
    (dict(page_size=12), {}, -3), (dict(page_size=1), {}, -3), (dict(k_pages=FAKE + 8), {}, -1),
    (dict(token_stride=132), {}, -1), ({}, dict(tokens=1 << 31), -10), ({}, dict(q_heads=1 << 17), -10)])
def test_attention_outside_of_the_supported(lib_built, cache, args, code):
    assert attend(cache_args(**cache), attention_args(**args)) == code
    need = C.c_size_t(7)
    assert capi.lib().mononn_paged_attention_workspace(C.byref(cache_args(**cache)), C.byref(attention_args(**args)),
                                                       C.byref(need)) == code
    assert need.value == 0


@pytest.mark.parametrize("change", [
    dict(k=None), dict(v=None), dict(indptr=None), dict(q=FAKE, q_heads=2), dict(q_out=FAKE), dict(k=FAKE + 1),
    dict(q=FAKE, q_out=FAKE, q_heads=0), dict(positions=FAKE + 1), dict(k_token_stride=-1),
    dict(q=FAKE, q_out=FAKE, q_heads=2, q_token_stride=128, q_head_stride=64, q_out_token_stride=256, q_out_head_stride=64),
    dict(q=FAKE, q_out=FAKE + 4096, q_heads=2, q_token_stride=128, q_head_stride=64, q_out_token_stride=128,
         q_out_head_stride=32)])
def test_append_refused(lib_built, change):
    assert append(args=append_args(**change)) == -1
    assert b"append" in capi.lib().mononn_last_error()


@pytest.mark.parametrize("change, code", [
    (dict(x=None), -1), (dict(positions=None), -1), (dict(dtype=3), -3), (dict(head_dim=0), -10),
    (dict(head_dim=257), -10), (dict(out=FAKE + 1), -1), (dict(out_token_stride=256), -1), (dict(positions=FAKE + 2), -1),
    (dict(out=FAKE + (1 << 16), out_head_stride=8), -1), (dict(x_token_stride=-1), -1)])
def test_rotary_refused(lib_built, change, code):
    table = Rotary(64).table()
    assert capi.lib().mononn_rotary_apply(C.byref(table), C.byref(rotary_args(**change)), None) == code


def test_rotary_tables_refused(lib_built):
    for change in (dict(rotary_dim=0), dict(rotary_dim=33), dict(rotary_dim=66), dict(rotary_dim=258), dict(magnitude=math.nan)):
        table = Rotary(64).table()
        for k, v in change.items():
            setattr(table, k, v)
        assert capi.lib().mononn_rotary_apply(C.byref(table), C.byref(rotary_args()), None) == -1
        assert append(table=table) == -1
    table = Rotary(64).table()
    table.turns[31] = math.inf
    assert append(table=table) == -1


def test_arguments_in_order_get_to_the_device(lib_built):
    table = Rotary(64).table()
    assert attend() in PASSES
    assert append(table=table) in PASSES
    assert capi.lib().mononn_rotary_apply(C.byref(table), C.byref(rotary_args()), None) in PASSES
    if not torch.cuda.is_available():
        assert capi.lib().mononn_paged_attention_status(None) == -5


def test_nothing_to_do_is_fine(lib_built):
    assert attend(args=attention_args(tokens=0)) == 0
    assert attend(cache=cache_args(sequences=0)) == 0
    assert append(args=append_args(tokens=0)) == 0
    table = Rotary(64).table()
    assert capi.lib().mononn_rotary_apply(C.byref(table), C.byref(rotary_args(tokens=0)), None) == 0
    # tensors without elements have no addresses
    none = dict.fromkeys(("q", "out", "indptr"))
    assert attend(cache=cache_args(k_pages=None, v_pages=None, num_pages=0), args=attention_args(tokens=0, **none)) == 0
    assert attend(cache=cache_args(sequences=0, page_table=None, lengths=None)) == 0
    assert append(args=append_args(tokens=0, k=None, v=None, indptr=None)) == 0
    assert append(cache=cache_args(sequences=0, page_table=None, lengths=None)) == 0
    lib = capi.lib()
    assert lib.mononn_rotary_apply(C.byref(table), C.byref(rotary_args(tokens=0, x=None, out=None, positions=None)), None) == 0
    assert lib.mononn_rotary_apply(C.byref(table), C.byref(rotary_args(heads=0, x=None, out=None)), None) == 0
    need = C.c_size_t(7)
    rc = lib.mononn_paged_attention_workspace(C.byref(cache_args()), C.byref(attention_args(tokens=0, **none)), C.byref(need))
    assert rc == 0 and need.value == 0
    assert lib.mononn_paged_attention(None, C.byref(attention_args()), None) == -1
    assert lib.mononn_paged_append(C.byref(cache_args()), None, None, None) == -1
    assert lib.mononn_rotary_apply(None, C.byref(rotary_args()), None) == -1
    assert lib.mononn_rotary_init(None, None) == -1


@pytest.mark.parametrize("change", [
    dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=258), dict(theta=1.0), dict(theta=-5.0), dict(theta=math.inf),
    dict(scaling="linear", factor=0.0), dict(scaling="base", factor=-2.0), dict(scaling="ramp", factor=2.0),
    dict(scaling="bands", factor=2.0, original_length=100, low=4.0, high=4.0), dict(magnitude=-1.0),
    dict(scaling="ramp", factor=math.nan, original_length=100)])
def test_rotary_configuration_refused(lib_built, change):
    with pytest.raises(capi.MononnError) as e:
        Rotary(**{"rotary_dim": 64, **change}).table()
    assert e.value.code == -1


@pytest.mark.parametrize("r", [2, 6, 64, 96, 128, 256])
@pytest.mark.parametrize("scaling", ["none", "linear", "base", "ramp", "bands"])
@pytest.mark.parametrize("theta, factor, length", [(10000.0, 4.0, 4096.0), (500000.0, 8.0, 8192.0), (10000.0, 1.0, 2048.0)])
def test_rates(lib_built, r, scaling, theta, factor, length):
    table = Rotary(r, scaling=scaling, theta=theta, factor=factor, original_length=length).table()
    want = rotary_rates(r, theta, scaling, factor if scaling != "none" else 1.0, length)
    for i, f in enumerate(want):  # a few roundings of 64-bit numbers
        assert abs(table.turns[i] * 2 * math.pi - f) <= 64 * 2.0 ** -53 * f
    assert table.magnitude == (0.1 * math.log(factor) + 1.0 if scaling == "ramp" and factor > 1 else 1.0)
    assert table.rotary_dim == r and table.interleaved == 0
    assert Rotary(r, magnitude=0.5).table().magnitude == 0.5


def small_cache(dtype=torch.float16):
    pages = torch.zeros(4, 16, 2, 64, dtype=dtype)
    return pages, torch.zeros_like(pages), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)


def test_tensors_refused(lib_built):
    k, v, table, lengths = small_cache()
    good = PagedCache(k, v, table, lengths)
    for bad in ((k, v[:3], table, lengths), (k, v.transpose(1, 2).contiguous().transpose(1, 2), table, lengths),
                (k, v.bfloat16(), table, lengths), (k, v, table.long(), lengths), (k, v, table, lengths[:1]),
                (k, v, table[0], lengths), (k.transpose(2, 3), v.transpose(2, 3), table, lengths)):
        with pytest.raises((ValueError, TypeError)):
            PagedCache(*bad)
    with pytest.raises(TypeError):
        PagedCache(k.float(), v.float(), table, lengths)
    new = torch.zeros(3, 2, 64, dtype=torch.float16)
    indptr = torch.zeros(3, dtype=torch.int32)
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    for args, kw in (((new, new[:2], indptr), {}), ((new[:, :1], new, indptr), {}), ((new, new, indptr[:2]), {}),
                     ((new, new, indptr.long()), {}), ((new, new, indptr), dict(q_out=q)),
                     ((new, new, indptr), dict(q=q[:2])), ((new, new, indptr), dict(q=q, q_out=q[:, :2])),
                     ((new, new, indptr), dict(q=q, positions=torch.zeros(2, dtype=torch.int32))),
                     ((new.bfloat16(), new, indptr), {}), ((new, new, indptr), dict(q=q[..., ::2]))):
        with pytest.raises(ValueError):
            good.append_runner(*args, **kw)
    flat = torch.zeros(2 * 3 * 4 * 64, dtype=torch.float16)
    over = flat[64:64 + 768].view(3, 4, 64)
    with pytest.raises(ValueError):
        good.append_runner(new, new, indptr, q=flat[:768].view(3, 4, 64), q_out=over)
    for args, kw in (((q[..., :32], indptr), {}), ((q, indptr[:1]), {}), ((q, indptr), dict(out=q[:2])),
                     ((q, indptr), dict(lse=torch.zeros(3, 4, dtype=torch.float16))), ((q, indptr), dict(scale=0.0)),
                     ((q, indptr), dict(out=q)), ((q, indptr), dict(window=-1))):
        with pytest.raises(ValueError):
            good.attention_runner(*args, **kw)
    x = torch.zeros(3, 4, 64, dtype=torch.float16)
    pos = torch.zeros(3, dtype=torch.int32)
    for args, kw in (((x, pos[:2], Rotary(64)), {}), ((x, pos.long(), Rotary(64)), {}),
                     ((x, pos, Rotary(64)), dict(out=x[:2])), ((x[0], pos, Rotary(64)), {}),
                     ((flat[:768].view(3, 4, 64), pos, Rotary(64)), dict(out=over))):
        with pytest.raises(ValueError):
            rotary_runner(*args, **kw)
    with pytest.raises(ValueError):
        Rotary(64, scaling="other").table()


def test_places_written_twice_are_refused(lib_built):
    """Two elements of what is written at one address: strides that are wide enough one by one, but not together."""
    lib, table = capi.lib(), Rotary(64).table()
    assert append(cache=cache_args(v_pages=FAKE)) == -1
    assert append(cache=cache_args(head_stride=128)) == -1
    assert append(cache=cache_args(page_stride=15 * 128 + 64)) == -1
    assert append(cache=cache_args(head_stride=16 * 64, token_stride=64)) in PASSES
    assert append(cache=cache_args(head_stride=9 * 16 * 64, page_stride=16 * 64, token_stride=64)) in PASSES
    q = dict(q=FAKE, q_out=3 * FAKE, q_heads=4, q_token_stride=256, q_head_stride=64)
    assert append(args=append_args(**q, q_out_token_stride=192, q_out_head_stride=64)) == -1
    assert append(args=append_args(**q, q_out_token_stride=64, q_out_head_stride=192)) in PASSES
    assert attend(args=attention_args(out_token_stride=192)) == -1
    assert attend(args=attention_args(out_token_stride=64, out_head_stride=192)) in PASSES
    assert attend(args=attention_args(tokens=1, out_token_stride=0)) in PASSES
    out = dict(out=3 * FAKE, out_token_stride=64, out_head_stride=128)
    assert lib.mononn_rotary_apply(C.byref(table), C.byref(rotary_args(**out)), None) == -1
    out["out_head_stride"] = 192
    assert lib.mononn_rotary_apply(C.byref(table), C.byref(rotary_args(**out)), None) in PASSES


def test_tensors_that_want_gradients_are_refused(lib_built):
    """No gradient is computed, so none may be lost without a word."""
    cache = PagedCache(*small_cache())
    new, q = torch.zeros(3, 2, 64, dtype=torch.float16), torch.zeros(3, 4, 64, dtype=torch.float16)
    indptr, pos = torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    grad = torch.zeros(3, 4, 64, dtype=torch.float16, requires_grad=True)
    for call in (lambda: rotary_runner(grad, pos, Rotary(64)), lambda: cache.attention_runner(grad, indptr),
                 lambda: cache.append_runner(grad[:, :2], new, indptr), lambda: cache.append_runner(new, grad[:, 2:], indptr),
                 lambda: cache.append_runner(new, new, indptr, q=grad), lambda: cache.attention_runner(q, indptr, out=grad)):
        with pytest.raises(ValueError, match="gradient"):
            call()


def test_queries_may_not_overlap_what_is_appended(lib_built):
    cache = PagedCache(*small_cache())
    indptr = torch.zeros(3, dtype=torch.int32)
    wide = torch.zeros(3, 8, 64, dtype=torch.float16)
    q, k, v = wide[:, :4], wide[:, 4:6], wide[:, 6:]
    for q_out in (wide[:, 2:6], wide[:, 4:]):
        with pytest.raises(ValueError, match="overlaps"):
            cache.append_runner(k, v, indptr, q=q, q_out=q_out)


def test_queries_in_place_beside_what_is_appended(lib_built):
    """Slices of one projection: whether q turned in place is taken goes by the elements alone, whichever has more heads
    and comes first. What is taken gets as far as the library call, and is refused there for want of a GPU."""
    cache = PagedCache(*small_cache())
    indptr = torch.zeros(3, dtype=torch.int32)

    class OfHost:
        cuda_stream = 0

    def parts(wide, q, k, v):
        return lambda: cache.append_runner(wide[:, k:k + 2], wide[:, v:v + 2], indptr, q=wide[:, q:q + 4], stream=OfHost)

    wide = torch.zeros(3, 16, 64, dtype=torch.float16)
    for q, k, v in ((0, 4, 6), (4, 0, 2), (2, 0, 6), (12, 10, 8)):
        parts(wide, q, k, v)()
    for q, k, v in ((0, 2, 8), (0, 8, 3), (4, 3, 0), (4, 0, 7), (4, 5, 12)):
        with pytest.raises(ValueError, match="overlaps"):
            parts(wide, q, k, v)()
    heads = torch.zeros(3, 2, 3, 64, dtype=torch.float16)  # the parts of a head side by side
    cache.append_runner(heads[:, :, 1], heads[:, :, 2], indptr, q=heads[:, :, 0], stream=OfHost)
    cache.append_runner(heads[:, :, 0], heads[:, :, 1], indptr, q=heads[:, :, 2], stream=OfHost)
    major = torch.zeros(2, 3, 3, 64, dtype=torch.float16).transpose(0, 1)  # heads apart, then tokens, then parts
    cache.append_runner(major[:, :, 0], major[:, :, 2], indptr, q=major[:, :, 1], stream=OfHost)
    with pytest.raises(ValueError, match="overlaps"):
        cache.append_runner(heads[:, :, 0], heads[:, :, 2], indptr, q=heads[:, :, 0], stream=OfHost)


def test_slices_that_share_an_element_are_never_taken(lib_built):
    """Every two small slices of a buffer that the check takes for disjoint have no element in common."""
    import itertools
    import random

    from mononn_b200.paged import _overlap, _same_grid
    rng = random.Random(5)
    flat = torch.zeros(400, dtype=torch.float16)

    def places(t):
        o = t.storage_offset()
        return {o + sum(i * s for i, s in zip(at, t.stride())) for at in itertools.product(*map(range, t.shape))}

    taken = 0
    for _ in range(6000):
        strides = rng.choice(((8, 2), (12, 4), (2, 9), (6, 3), (24, 6), (4, 2), (0, 2), (3, 3), (5, 2)))
        tokens, dim = rng.randint(1, 3), rng.randint(1, 3)
        a, b = (flat.as_strided((tokens, rng.randint(1, 4), dim), (*strides, 1), rng.randint(0, 30)) for _ in range(2))
        if _same_grid(a, b) or not _overlap(a, b):
            taken += 1
            assert not places(a) & places(b)
    assert taken > 500


@pytest.mark.parametrize("which", [0, 1])
def test_pages_that_want_gradients_are_refused(lib_built, which):
    """A learned prefix among the keys or the values: neither reading nor writing it loses a gradient without a word."""
    tensors = list(small_cache())
    tensors[which].requires_grad_()
    cache = PagedCache(*tensors)
    new, q = torch.zeros(3, 2, 64, dtype=torch.float16), torch.zeros(3, 4, 64, dtype=torch.float16)
    indptr = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: cache.attention_runner(q, indptr), lambda: cache.append_runner(new, new, indptr)):
        with pytest.raises(ValueError, match="_pages requires a gradient"):
            call()

    class OfHost:
        cuda_stream = 0

    with torch.no_grad():
        cache.append_runner(new, new, indptr, stream=OfHost)


def test_forward_gradients_are_refused(lib_built):
    from torch.autograd import forward_ad
    k, v, table, lengths = small_cache()
    new, q = torch.zeros(3, 2, 64, dtype=torch.float16), torch.zeros(3, 4, 64, dtype=torch.float16)
    indptr, pos = torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    cache = PagedCache(k, v, table, lengths)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: rotary_runner(dual(q), pos, Rotary(64)), lambda: cache.attention_runner(dual(q), indptr),
                     lambda: cache.append_runner(dual(new), new, indptr), lambda: cache.append_runner(new, dual(new), indptr),
                     lambda: PagedCache(dual(k), v, table, lengths).attention_runner(q, indptr),
                     lambda: PagedCache(k, dual(v), table, lengths).append_runner(new, new, indptr)):
            with pytest.raises(ValueError, match="forward gradient"):
                call()


def test_status_is_read_on_the_device_of_the_stream(lib_built, monkeypatch):
    """Default streams have the same handle on every device: the one of the stream has to be current."""
    import contextlib

    from mononn_b200 import paged
    current, asked = [0], []

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], d
        yield
        current[0] = before

    class Library:
        @staticmethod
        def mononn_paged_attention_status(handle):
            asked.append((current[0], handle.value))
            return 0

    class DefaultStream:
        device, cuda_stream = 1, 0

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(paged, "lib", Library)
    paged.paged_attention_status(DefaultStream)
    assert asked == [(1, None)] and current == [0]


def test_streams_of_other_devices_are_refused(lib_built):
    from mononn_b200 import paged

    class DefaultStream:
        device, cuda_stream = torch.device("cuda", 1), 0

    with pytest.raises(ValueError, match="stream belongs to cuda:1"):
        paged._stream(torch.device("cuda", 0), DefaultStream)
    assert paged._stream(torch.device("cuda", 1), DefaultStream).value is None


@pytest.mark.parametrize("scaling", ["none", "linear", "base", "ramp", "bands"])
def test_entries_that_a_configuration_leaves_open(lib_built, scaling):
    """None stands for the default, as 0 does."""
    given = dict(scaling=scaling, factor=4.0, original_length=4096.0)
    want = Rotary(64, **given).table()
    got = Rotary(64, **given, theta=None, low=None, high=None, magnitude=None).table()
    assert bytes(got) == bytes(want)
    assert bytes(Rotary(64, factor=None, original_length=None).table()) == bytes(Rotary(64).table())
    if scaling != "none":
        with pytest.raises(capi.MononnError, match="factor"):
            Rotary(64, **{**given, "factor": None}).table()
    if scaling in ("ramp", "bands"):
        with pytest.raises(capi.MononnError, match="original_length"):
            Rotary(64, **{**given, "original_length": None}).table()


@pytest.mark.parametrize("name", ["k_pages", "v_pages", "page_table", "lengths"])
def test_tensors_of_a_cache_are_not_replaced(lib_built, name):
    """Calls would go on with the address of the old one, which may be somebody else's memory by then."""
    tensors = small_cache()
    cache = PagedCache(*tensors)
    before = bytes(cache._args)
    with pytest.raises(AttributeError):
        setattr(cache, name, getattr(cache, name) + 1)
    cache.lengths.add_(1)
    assert bytes(cache._args) == before and cache.lengths is tensors[3] and cache.lengths.tolist() == [1, 1]


def test_scales_that_vanish_in_32_bits_are_refused(lib_built):
    """They would become 0, which stands for 1 / sqrt(head_dim)."""
    cache = PagedCache(*small_cache())
    q, indptr = torch.zeros(3, 4, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int32)
    for scale in (1e-46, 0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="scale must be positive"):
            cache.attention_runner(q, indptr, scale=scale)


def test_rotations_that_leave_the_kernels_numbers_are_refused(lib_built):
    """A magnitude that is infinite in 32 bits, rates whose angle at a far position is infinite: NaN would come out."""
    lib = capi.lib()
    for change in (dict(magnitude=1e39), dict(magnitude=-1e300), dict(turns=1e300), dict(turns=-math.inf), dict(turns=math.nan)):
        table = Rotary(64).table()
        if "turns" in change:
            table.turns[31] = change["turns"]
        else:
            table.magnitude = change["magnitude"]
        assert lib.mononn_rotary_apply(C.byref(table), C.byref(rotary_args()), None) == -1
        assert b"rotary" in lib.mononn_last_error()
        assert append(table=table) == -1
        assert b"rotary" in lib.mononn_last_error()
    for change in (dict(magnitude=1e39), dict(scaling="linear", factor=1e-305),
                   dict(scaling="bands", factor=1e-305, original_length=10.0)):
        with pytest.raises(capi.MononnError, match="rotary"):
            Rotary(64, **change).table()
    table = Rotary(64, magnitude=1e38, scaling="linear", factor=1e-30).table()
    assert append(table=table) in PASSES


def test_sizes_beyond_32_bits_are_refused(lib_built):
    """2^32 tokens would be counted as none, 2^32 + 3 pages as three."""
    cache = PagedCache(*small_cache())
    k, v, table, lengths = small_cache()
    many = torch.zeros(1, 2, 64, dtype=torch.float16).expand(2 ** 32, 2, 64)
    wide = torch.zeros(3, 1, 64, dtype=torch.float16).expand(3, 2 ** 32 + 1, 64)
    indptr, pos = torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: cache.append_runner(many, many, indptr), lambda: cache.attention_runner(wide, indptr, out=wide),
                 lambda: rotary_runner(wide, pos, Rotary(64)),
                 lambda: PagedCache(*[t[:1].expand(2 ** 32 + 3, 16, 2, 64) for t in (k, v)], table, lengths),
                 lambda: PagedCache(k, v, table[:, :1].expand(2, 2 ** 32), lengths)):
        with pytest.raises(ValueError, match="2\\^32 or more"):
            call()


def test_autograd_is_told_what_is_written(lib_built):
    """A graph that saved a tensor does not go on with what a call wrote over it. Without tokens a call needs no GPU."""
    class OfHost:
        cuda_stream = 0

    cache = PagedCache(*small_cache())
    indptr, none = torch.zeros(3, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)

    def rows(heads=2):
        return torch.zeros(0, heads, 64, dtype=torch.float16)

    x, y, q, q2, out, lse = rows(), rows(), rows(4), rows(4), rows(4), torch.zeros(0, 4)
    k, v = rows(), rows()
    for written, kept, call in (
            ((x,), (), lambda: rotary_runner(x, none, Rotary(64), stream=OfHost)()),
            ((y,), (x,), lambda: rotary_runner(x, none, Rotary(64), out=y, stream=OfHost)()),
            ((cache.k_pages, cache.v_pages, q), (k, v), lambda: cache.append(k, v, indptr, q=q, stream=OfHost)),
            ((q2,), (q,), lambda: cache.append(k, v, indptr, q=q, q_out=q2, stream=OfHost)),
            ((out, lse), (q, cache.k_pages), lambda: cache.attention_runner(q, indptr, out=out, lse=lse, stream=OfHost)())):
        weight = torch.ones(1, dtype=torch.float16, requires_grad=True)
        saved = [(weight * t).sum() for t in written]
        fine = [(weight * t).sum() for t in kept]
        call()
        for s in saved:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                s.backward()
        for s in fine:
            s.backward()


def test_what_is_written_may_not_be_read(lib_built):
    """Tensors of any kind that a call writes and reads at one address, or writes twice."""
    halves = torch.zeros(1 << 16, dtype=torch.float16)

    def at(offset, *shape, dtype=torch.float16):
        return halves[offset:].view(dtype).flatten()[:math.prod(shape)].view(*shape)

    def cache(k=0, v=8192, table=16384, lengths=16512):
        return PagedCache(at(k, 4, 16, 2, 64), at(v, 4, 16, 2, 64), at(table, 2, 3, dtype=torch.int32),
                          at(lengths, 2, dtype=torch.int32))

    indptr, pos = at(16640, 3, dtype=torch.int32), at(16768, 3, dtype=torch.int32)
    free = 20480

    class OfHost:
        cuda_stream = 0

    def append(c, q_out=None, **kw):
        q = at(free + 2048, 3, 4, 64)
        given = dict(k=at(free, 3, 2, 64), v=at(free + 1024, 3, 2, 64), indptr=indptr, positions=pos, q=q, stream=OfHost)
        given.update(kw)
        return c.append_runner(q_out=q if q_out is None else q_out, **given)

    append(cache())
    for call, names in ((lambda: append(cache(), q_out=at(4096, 3, 4, 64)), "q_out overlaps k_pages"),
                        (lambda: append(cache(), q_out=at(12288, 3, 4, 64)), "q_out overlaps v_pages"),
                        (lambda: append(cache(), q_out=at(16640 - 64, 3, 4, 64)), "q_out overlaps indptr"),
                        (lambda: append(cache(), q_out=at(16768, 3, 4, 64)), "q_out overlaps positions"),
                        (lambda: append(cache(), k=at(64, 3, 2, 64)), "k_pages overlaps k"),
                        (lambda: append(cache(), v=at(8192, 3, 2, 64)), "v_pages overlaps v"),
                        (lambda: append(cache(table=128)), "k_pages overlaps page_table"),
                        (lambda: append(cache(lengths=8192 + 128)), "v_pages overlaps lengths"),
                        (lambda: rotary_runner(at(16768 - 128, 3, 2, 64), pos, Rotary(64)), "out overlaps positions")):
        with pytest.raises(ValueError, match=names):
            call()

    def attend(c, out, lse):
        return c.attention_runner(at(free, 3, 4, 64), indptr, out=out, lse=lse)

    out, lse = at(free + 1024, 3, 4, 64), at(free + 2048, 3, 4, dtype=torch.float32)
    for call, names in ((lambda: attend(cache(), at(16384, 3, 4, 64), lse), "out overlaps page_table"),
                        (lambda: attend(cache(), at(16512, 3, 4, 64), lse), "out overlaps lengths"),
                        (lambda: attend(cache(), out, at(free + 1024, 3, 4, dtype=torch.float32)), "out overlaps lse"),
                        (lambda: attend(cache(), out, at(free, 3, 4, dtype=torch.float32)), "lse overlaps q"),
                        (lambda: attend(cache(), out, at(0, 3, 4, dtype=torch.float32)), "lse overlaps k_pages"),
                        (lambda: attend(cache(), out, at(16640, 3, 4, dtype=torch.float32)), "lse overlaps indptr")):
        with pytest.raises(ValueError, match=names):
            call()


def test_keys_and_values_of_a_page_share_no_place(lib_built):
    for off in (0, 2, 64, 128, 16 * 128 - 2):  # bytes; a page has 16 tokens x 2 heads x 64 elements
        for change in (dict(v_pages=FAKE + off), dict(k_pages=FAKE + off, v_pages=FAKE)):
            assert append(cache=cache_args(**change)) == -1
            assert b"same places" in capi.lib().mononn_last_error()
    page = 16 * 2 * 64
    assert append(cache=cache_args(v_pages=FAKE + 2 * page, page_stride=2 * page)) in PASSES
    assert append(cache=cache_args(v_pages=FAKE + 2 * 64, head_stride=128, token_stride=256, page_stride=2 * page)) in PASSES
    assert append(cache=cache_args(v_pages=FAKE + 2 * 128, token_stride=256, page_stride=2 * page)) in PASSES
    assert append(cache=cache_args(v_pages=FAKE + 2 * 64, token_stride=256, page_stride=2 * page)) == -1
    assert append(cache=cache_args(v_pages=FAKE + 2 * page, num_pages=4, page_stride=page)) in PASSES  # of other pages


def test_queries_in_place_behind_a_single_head(lib_built):
    """A key or value head directly before the queries is as far away as their heads are from one another."""
    k, v, table, lengths = (t[:, :, :1] if t.dim() == 4 else t for t in small_cache())
    cache = PagedCache(k, v, table, lengths)
    wide, indptr = torch.zeros(3, 7, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int32)

    class OfHost:
        cuda_stream = 0

    for key, value, q in ((0, 1, 2), (1, 0, 2), (5, 6, 0), (0, 6, 1)):
        cache.append_runner(wide[:, key:key + 1], wide[:, value:value + 1], indptr, q=wide[:, q:q + 5], stream=OfHost)
    for key, value, q in ((2, 1, 2), (0, 4, 2), (6, 0, 2)):
        with pytest.raises(ValueError, match="overlaps"):
            cache.append_runner(wide[:, key:key + 1], wide[:, value:value + 1], indptr, q=wide[:, q:q + 5], stream=OfHost)


def test_waits_that_are_to_run_out_are_chosen_from_the_barriers(lib_built):
    lib = capi.lib()
    assert lib.mononn_debug_paged_skew(14) == -1
    for barrier in range(14):
        assert lib.mononn_debug_paged_skew(barrier) == 0
    assert lib.mononn_debug_paged_skew(1) == 0
    assert attend(args=attention_args(tokens=0)) == 0  # the next call, whatever it does, is the one that is meant
    assert lib.mononn_debug_paged_skew(0) == 0
