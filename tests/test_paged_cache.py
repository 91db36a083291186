"""Paged caches without a device: what the entry points and `PagedKVCache` refuse, the partition of the attention kernel
restated, and the 8-bit formats of the restatement."""
import ctypes

import numpy as np
import pytest

from oracle import paged_oracle as orc
from vte_b200.bridge import CudaSafetyError
from vte_b200.bridge.cuda_runtime import PagedAppend, PagedAttention, PagedCache, load_library
from vte_b200.core import PagedKVCache

NOT_INITIALIZED, INVALID, UNSUPPORTED, TOO_LARGE = -2, -1, -3, -7
AT = 1 << 20            # an aligned address: nothing is read from it


@pytest.fixture(scope="module")
def lib(built_library):
    return load_library(str(built_library))


def cache_of(**kw):
    D, H, P = kw.get("head_dim", 128), kw.get("num_kv_heads", 2), kw.get("page_size", 16)
    base = dict(k_pool=AT, v_pool=AT, k_scale=AT, v_scale=AT, page_stride=H * P * D, token_stride=D, head_stride=P * D,
                num_pages=4, page_size=P, num_kv_heads=H, head_dim=D, type=1)
    return PagedCache(**{**base, **kw})


@pytest.mark.parametrize("change,code", [
    ({}, NOT_INITIALIZED), ({"type": 3}, INVALID), ({"type": -1}, INVALID), ({"head_dim": 96}, UNSUPPORTED),
    ({"page_size": 48}, UNSUPPORTED), ({"page_size": 8}, UNSUPPORTED), ({"num_pages": 0}, INVALID), ({"num_kv_heads": 0}, INVALID),
    ({"k_pool": 0}, INVALID), ({"v_pool": AT + 8}, INVALID), ({"k_scale": 0}, INVALID), ({"v_scale": AT + 2}, INVALID),
    ({"type": 0, "k_scale": 0, "v_scale": 0}, NOT_INITIALIZED), ({"token_stride": 64}, INVALID), ({"token_stride": 136}, INVALID),
    ({"head_stride": 1024}, INVALID), ({"page_stride": 4080}, INVALID), ({"page_stride": 1 << 41}, INVALID),
    ({"token_stride": 256, "head_stride": 128}, NOT_INITIALIZED), ({"token_stride": 256, "head_stride": 128, "page_stride": 8192}, NOT_INITIALIZED),
    ({"page_stride": 128, "num_pages": 1}, NOT_INITIALIZED),
])
def test_cache_refusals(lib, change, code):
    c = cache_of(**change)
    assert lib.vteb_paged_cache_init(ctypes.byref(c)) == code and c.ready == 0
    assert lib.vteb_paged_cache_init(None) == INVALID


@pytest.mark.parametrize("change,code", [
    ({}, NOT_INITIALIZED), ({"batch": 0}, INVALID), ({"max_pages": 0}, INVALID), ({"total_tokens": -1}, INVALID),
    ({"max_pages": 1 << 27}, TOO_LARGE), ({"k": 0}, INVALID), ({"v": 0}, INVALID), ({"block_table": 0}, INVALID),
    ({"kv_offsets": 0}, INVALID), ({"k": AT + 8}, INVALID), ({"q_out": AT + 2}, INVALID), ({"q": 0}, INVALID), ({"q_out": 0}, INVALID),
    ({"total_tokens": 5}, INVALID), ({"total_tokens": 5, "token_starts": AT}, NOT_INITIALIZED), ({"k_token_stride": 255}, INVALID),
    ({"v_token_stride": 260}, INVALID), ({"q_token_stride": 1530}, INVALID), ({"q_out_token_stride": 8}, INVALID),
    ({"num_q_heads": 0}, INVALID), ({"q": 0, "q_out": 0, "num_q_heads": 0}, NOT_INITIALIZED), ({"rope_type": 3}, INVALID),
    ({"rope_type": -2}, INVALID), ({"rope_cos": 0}, INVALID), ({"rope_sin": AT + 8}, INVALID), ({"rope_rows": 0}, INVALID),
    ({"rope_type": 2, "rotary_dim": 24}, UNSUPPORTED), ({"rope_type": 2, "rotary_dim": 144}, UNSUPPORTED),
    ({"rope_type": 2, "rotary_dim": 0}, UNSUPPORTED), ({"rope_type": -1, "rope_cos": 0}, NOT_INITIALIZED), ({"total_tokens": 0}, NOT_INITIALIZED),
    ({"total_tokens": 1 << 28, "token_starts": AT}, TOO_LARGE),
])
def test_append_refusals(lib, change, code):
    c = cache_of(ready=1)
    base = dict(k=AT, v=AT, q=AT, q_out=AT, k_token_stride=256, v_token_stride=256, q_token_stride=1536, q_out_token_stride=1536,
                block_table=AT, kv_offsets=AT, rope_cos=AT, rope_sin=AT, batch=4, max_pages=3, total_tokens=4, num_q_heads=12,
                rope_type=0, rotary_dim=128, rope_rows=48)
    a = PagedAppend(**{**base, **change})
    assert lib.vteb_paged_append(ctypes.byref(c), ctypes.byref(a), None) == code, lib.vteb_last_error_string()
    assert lib.vteb_paged_append(ctypes.byref(cache_of()), ctypes.byref(a), None) == INVALID      # not initialised
    assert lib.vteb_paged_append(None, ctypes.byref(a), None) == INVALID
    assert lib.vteb_paged_append(ctypes.byref(c), None, None) == INVALID


@pytest.mark.parametrize("change,code", [
    ({}, NOT_INITIALIZED), ({"q": 0}, INVALID), ({"output": 0}, INVALID), ({"workspace": 0}, INVALID), ({"workspace": AT + 128}, INVALID),
    ({"q": AT + 8}, INVALID), ({"output": AT + 8}, INVALID), ({"block_table": 0}, INVALID), ({"kv_offsets": 0}, INVALID),
    ({"batch": 0}, INVALID), ({"batch": 65536}, INVALID), ({"query_tokens": 0}, INVALID), ({"query_tokens": 17}, INVALID),
    ({"num_q_heads": 11}, INVALID), ({"num_q_heads": 0}, INVALID), ({"num_q_heads": 4098}, INVALID), ({"max_pages": 0}, TOO_LARGE),
    ({"max_pages": 1 << 27}, TOO_LARGE), ({"scale": float("nan")}, INVALID), ({"scale": float("inf")}, INVALID), ({"lse": AT}, NOT_INITIALIZED),
])
def test_attention_refusals(lib, change, code):
    c = cache_of(ready=1)
    base = dict(q=AT, output=AT, block_table=AT, kv_offsets=AT, workspace=AT, workspace_bytes=1 << 30, scale=0.1, batch=2,
                max_pages=4, num_q_heads=12, query_tokens=1)
    a = PagedAttention(**{**base, **change})
    assert lib.vteb_paged_attention(ctypes.byref(c), ctypes.byref(a), None) == code, lib.vteb_last_error_string()
    assert lib.vteb_paged_attention(ctypes.byref(cache_of()), ctypes.byref(a), None) == INVALID
    assert lib.vteb_paged_attention(None, ctypes.byref(a), None) == INVALID
    assert lib.vteb_paged_attention(ctypes.byref(c), None, None) == INVALID


def test_workspace_refusals(lib):
    n = ctypes.c_size_t(0)
    for args, code in (((12, 2, 128, 1, 1), NOT_INITIALIZED), ((12, 5, 128, 1, 1), INVALID), ((12, 2, 80, 1, 1), UNSUPPORTED),
                       ((12, 2, 128, 0, 1), INVALID), ((12, 2, 128, 1, 17), INVALID)):
        assert lib.vteb_paged_attention_workspace(*args, ctypes.byref(n)) == code
    assert lib.vteb_paged_attention_workspace(12, 2, 128, 1, 1, None) == INVALID


class FakeRuntime:
    """The calls that `PagedKVCache` makes, without a device."""

    def __init__(self, fail=False):
        self.live, self.fail, self.calls = {}, fail, []

    def safe_malloc(self, n, tag):
        p = ctypes.c_void_p(AT * (1 + len(self.calls)))
        self.calls.append((tag, n))
        self.live[p.value] = n
        return p

    def safe_free(self, p, tag):
        del self.live[p.value]

    def safe_memset(self, p, n, tag):
        assert self.live[p.value] == n

    def synchronize(self):
        pass

    def paged_cache_init(self, cache):
        if self.fail:
            raise CudaSafetyError("refused")

    def paged_attention_workspace(self, q_heads, kv_heads, head_dim, batch, query_tokens):
        return 1000 * query_tokens

    def paged_append(self, cache, a, stream):
        self.append = {n: getattr(a, n) for n, _ in a._fields_}

    def paged_attention(self, cache, a, stream):
        self.attention = {n: getattr(a, n) for n, _ in a._fields_}


META = {"attention.head_count": 12, "attention.head_count_kv": 2, "attention.key_length": 128}


def test_cache_of_its_own_memory():
    rt = FakeRuntime()
    c = PagedKVCache(rt, META, 10, 16, "e4m3")
    assert [n for _, n in rt.calls] == [10 * 2 * 16 * 128] * 2 + [10 * 2 * 4] * 2
    assert (c._cache.page_stride, c._cache.token_stride, c._cache.head_stride, c._cache.type) == (2 * 16 * 128, 128, 16 * 128, 1)
    c.attend(1, 2, 3, 4, 5, 6)
    first = rt.attention["workspace"]
    assert first % 256 == 0 and rt.attention["workspace_bytes"] == 1000 and rt.attention["query_tokens"] == 1
    assert rt.attention["scale"] == pytest.approx(128 ** -0.5) and not rt.attention["lse"]
    c.attend(1, 2, 3, 4, 5, 6)
    assert rt.attention["workspace"] == first and len(rt.calls) == 5
    c.attend(1, 2, 3, 4, 5, 6, query_tokens=2, scale=0.5, output_f32=True)
    assert rt.attention["workspace"] != first and rt.attention["scale"] == 0.5 and rt.attention["out_is_f32"] == 1
    c.append(1, 2, 3, 4, 5, 6)
    assert rt.append["total_tokens"] == 5 and rt.append["k_token_stride"] == 256 and rt.append["q"] is None and rt.append["rope_type"] == -1
    c.set_rope(7, 8, 99)
    c.append(1, 2, 3, 4, 5, 6, total_tokens=50, token_starts=9, q=16, q_out=16, token_strides=(2048,) * 4)
    assert rt.append["rope_type"] == 0 and rt.append["rope_rows"] == 99 and rt.append["q_out_token_stride"] == 2048
    c.set_rope(0, 0, 0)
    c.append(1, 2, 3, 4, 5, 6)
    assert rt.append["rope_type"] == -1 and rt.append["token_starts"] is None and rt.append["k_token_stride"] == 256
    c.cleanup()
    assert not rt.live
    with pytest.raises(CudaSafetyError):
        PagedKVCache(FakeRuntime(fail=True), META, 4)


def test_a_cache_that_is_refused_frees_what_it_allocated():
    rt = FakeRuntime(fail=True)
    with pytest.raises(CudaSafetyError):
        PagedKVCache(rt, META, 4)
    assert not rt.live and rt.calls


@pytest.mark.parametrize("kw", [{"cache_type": "fp4"}, {"num_pages": 0}, {"page_size": 0}, {"k_pool": AT}, {"k_scale": AT},
                                {"strides": (1, 2, 3)}, {"k_pool": AT, "v_pool": AT, "strides": (1, 2)}])
def test_what_the_cache_refuses(kw):
    rt = FakeRuntime()
    with pytest.raises(CudaSafetyError):
        PagedKVCache(rt, META, **{"num_pages": 4, **kw})
    assert not rt.live


def test_e4m3_grid_and_rounding():
    v = orc.E4M3[np.arange(127)]
    assert v[0] == 0 and v[1] == 2.0 ** -9 and v[126] == 448 and (np.diff(v) > 0).all() and np.isnan(orc.E4M3[[127, 255]]).all()
    assert np.array_equal(orc.to_e4m3(v), np.arange(127)) and np.array_equal(orc.to_e4m3(-v[1:]), np.arange(1, 127) + 128)
    mid = ((v[:-1].astype(np.float64) + v[1:]) / 2).astype(np.float32)
    got = orc.to_e4m3(mid)
    assert (got % 2 == 0).all() and (np.abs(got.astype(int) - np.arange(126)) <= 1).all()      # ties to even
    assert orc.to_e4m3(np.float32(1e9)) == 126 and orc.to_e4m3(np.float32(np.nan)) & 127 == 127


def worker_runs(lengths, head_rows, unit, grid, groups, warps, end=2):
    """The runs that paged_attention_kernel deals to its workers where they are long: equal shares of all units, the end of a
    segment counted as `end` units a warp.  (units of a run, what a segment's end counts, [[(first, end) by segment]])."""
    extra = end * (warps // groups)
    counts = [-(-int(n) // unit) for n in lengths for _ in range(head_rows) if n]
    total = sum(n + extra for n in counts)
    mean = max(-(-sum(counts) // max(len(counts), 1)), 1)
    cuts = -(-mean // extra)
    per = max(-(-total // (grid * groups)), -(-mean // cuts))
    begins = np.cumsum([0] + [n + extra for n in counts])
    return per, begins, counts, -(-total // per)


@pytest.mark.parametrize("groups", [1, 2])
def test_pieces_of_cut_segments_have_places_of_their_own(groups):
    """The kernel's arithmetic for segments that worker borders cut: every unit is one worker's, first and last worker of a
    segment, the piece each one leaves, and the counters of pieces that are merged into one, in two steps where they are many."""
    rng = np.random.default_rng(groups)
    for _ in range(60):
        lengths = rng.integers(0, rng.choice([40, 500, 9000, 200000]), size=rng.integers(1, 40))
        head_rows, unit, warps = int(rng.choice([1, 2, 8])), int(rng.choice([16, 32, 64])), int(rng.choice([6, 8]))
        per, begins, counts, workers = worker_runs(lengths, head_rows, unit, 148, groups, warps)
        assert workers <= 148 * groups
        pieces, counters = set(), [set(), set()]
        for begin, units in zip(begins.tolist(), counts):
            w0, w1 = begin // per, (begin + units - 1) // per
            owned = [(max(w * per, begin), min((w + 1) * per, begin + units)) for w in range(w0, w1 + 1)]
            assert owned[0][0] == begin and owned[-1][1] == begin + units and all(lo < hi for lo, hi in owned)
            assert all(a[1] == b[0] for a, b in zip(owned, owned[1:]))
            n = w1 - w0 + 1
            if n == 1:
                continue
            place = [2 * (w0 + k) if k else 2 * w0 + (0 if w0 * per == begin else 1) for k in range(n)]      # as it is read
            written = [2 * w + (0 if owned[w - w0][0] == w * per else 1) for w in range(w0, w1 + 1)]
            assert place == written and not pieces & set(place)
            pieces |= set(place)
            join = n if n <= 8 else 8 if n <= 64 else -(-n // 8)
            firsts = list(range(0, n, join))
            assert len(firsts) <= 8 and all((k // join * join) in firsts for k in range(n))
            at = [place[k] for k in firsts], [place[0]] if join < n else []
            for level in (0, 1):
                assert not counters[level] & set(at[level])
                counters[level] |= set(at[level])
