"""`PagedKVCache` after its memory is gone, and appends that would drop tokens or race, without a device."""
import ctypes

import pytest

from tests.test_paged_cache import AT, INVALID, META, NOT_INITIALIZED, FakeRuntime, cache_of
from vte_b200.bridge import CudaSafetyError
from vte_b200.bridge.cuda_runtime import PagedAppend, load_library
from vte_b200.core import PagedKVCache

POOLS = {"k_pool": AT, "v_pool": 2 * AT}


class Runtime(FakeRuntime):
    """`FakeRuntime` with the lives of a runtime: what `initialize` makes, and what `cleanup` frees."""

    def __init__(self):
        super().__init__()
        self.launches = 0
        self.initialize()

    def initialize(self):
        self._initialized, self._launch_status = True, ctypes.c_int(0)

    def cleanup(self):
        self.live.clear()
        self._initialized, self._launch_status = False, None

    def paged_append(self, *a):
        self.launches += 1
        super().paged_append(*a)

    def paged_attention(self, *a):
        self.launches += 1
        super().paged_attention(*a)


def calls(cache):
    return [lambda: cache.append(1, 2, 3, 4, 5, 6), lambda: cache.attend(1, 2, 3, 4, 5, 6),
            lambda: cache.attend(1, 2, 3, 4, 5, 6, workspace=AT, workspace_bytes=1000)]


@pytest.mark.parametrize("how", ["cache", "runtime", "runtime_again"])
def test_pools_that_are_gone_are_not_used(how):
    rt = Runtime()
    cache = PagedKVCache(rt, META, 4)
    for call in calls(cache):
        call()
    assert rt.launches == 3
    if how == "cache":
        cache.cleanup()
    else:
        rt.cleanup()
        if how == "runtime_again":
            rt.initialize()
    for call in [*calls(cache), lambda: cache.reserve(1)]:
        with pytest.raises(CudaSafetyError, match="cleaned up"):
            call()
    assert rt.launches == 3 and not rt.live


def test_a_cleanup_after_the_runtimes_own_frees_nothing():
    rt = Runtime()
    cache = PagedKVCache(rt, META, 4)
    held = list(rt.live)
    rt.cleanup()
    rt.initialize()
    for p in held:
        rt.live[p] = 1                                   # the same addresses, in other hands
    cache.cleanup()
    cache.cleanup()
    assert sorted(rt.live) == sorted(held)


def test_pools_of_the_callers_outlive_a_cleanup():
    """Only the workspace was the cache's: it is allocated anew."""
    rt = Runtime()
    cache = PagedKVCache(rt, META, 4, **POOLS)
    for again in (cache.cleanup, lambda: (rt.cleanup(), rt.initialize()), lambda: None):
        for call in calls(cache):
            call()
        assert len(rt.live) == 1 and next(iter(rt.live)) <= cache._workspace < next(iter(rt.live)) + 512
        again()
    cache.cleanup()
    assert not rt.live


def test_ragged_tokens_are_counted():
    """Without their number, rows behind the first `batch` ones would be left out."""
    rt = Runtime()
    cache = PagedKVCache(rt, META, 4, **POOLS)
    with pytest.raises(CudaSafetyError, match="total_tokens"):
        cache.append(1, 2, 3, 4, 5, 6, token_starts=AT)
    assert rt.launches == 0
    cache.append(1, 2, 3, 4, 5, 6, token_starts=AT, total_tokens=0)
    assert rt.append["total_tokens"] == 0


@pytest.mark.parametrize("change,code", [
    ({"q_out_token_stride": 2048}, INVALID), ({"q_token_stride": 2048}, INVALID), ({"q_token_stride": 2048, "q_out_token_stride": 2048}, NOT_INITIALIZED),
    ({"q_out_token_stride": 2048, "q_out": 2 * AT}, NOT_INITIALIZED), ({"q_out_token_stride": 2048, "total_tokens": 1, "batch": 1}, NOT_INITIALIZED),
])
def test_rotating_in_place_takes_one_stride(built_library, change, code):
    """With two, a token's rotated row would lie where another token's row is still to be read."""
    lib = load_library(str(built_library))
    c = cache_of(ready=1)
    base = dict(k=AT, v=AT, q=AT, q_out=AT, k_token_stride=256, v_token_stride=256, q_token_stride=1536, q_out_token_stride=1536,
                block_table=AT, kv_offsets=AT, batch=4, max_pages=3, total_tokens=4, num_q_heads=12, rope_type=-1)
    a = PagedAppend(**{**base, **change})
    assert lib.vteb_paged_append(ctypes.byref(c), ctypes.byref(a), None) == code, lib.vteb_last_error_string()
