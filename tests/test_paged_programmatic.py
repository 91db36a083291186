"""Paged launches may become resident while the launches in front of them run: what those write is read behind the wait only."""
import re

import numpy as np
import pytest

from tests.paged_case import Device, make_cache, metadata, random_pool, table_of
from vte_b200 import build
from vte_b200.workloads import build_rope_cache


@pytest.mark.parametrize("name", ["paged_append.cuh", "paged_attention.cuh"])
def test_no_load_may_be_moved_ahead_of_the_wait(name):
    """Non-coherent loads may: the compiler takes what they read for constant.  Offsets, tables, token starts and Q are written by
    launches in front.  (What the device code promises is checked in the source: a load that comes too early shows by chance.)"""
    source = (build.CSRC / "kernels" / name).read_text()
    code = re.sub(r"//[^\n]*", "", source)
    assert not re.search(r"__ldg|\.nc\b|__restrict__", code)
    kernel = code[code.index("__global__"):]
    before = kernel[:kernel.index("grid_dependency_wait()")]
    assert not re.search(r"[ap]\.(q|k|v|kv_offsets|block_table|token_starts|cos_table|sin_table|k_scale|v_scale|counters|part_\w+|output)\b", before)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "e4m3"])
def test_launches_one_behind_the_other_read_what_was_written_last(cuda_runtime, kind):
    """Steps queued without a wait, each attention's output the next step's Q, which its append rotates in place, against the same
    steps with the device idle in between."""
    rt, dev = cuda_runtime, Device(cuda_runtime)
    rng = np.random.default_rng(7)
    heads, page, steps = (8, 2, 128), 16, 24
    Hq, H, D = heads
    past = np.array([5, 40, 0, 15, 100, 31])
    B = len(past)
    table, pages = table_of(rng, past + steps, page)
    pools, scales = zip(*(random_pool(rng, kind, pages, heads, page) for _ in range(2)))
    cos, sin = build_rope_cache(int(past.max()) + steps, D, 1e4)
    k, v = (rng.standard_normal((steps, B, H, D), dtype=np.float32).astype(np.float16) for _ in range(2))
    q = rng.standard_normal((B, Hq, D), dtype=np.float32).astype(np.float16)
    offsets = np.stack([past + i for i in range(steps)]).astype(np.int32)
    results = []
    try:
        for idle in (True, False, False):
            cache, ptrs, _ = make_cache(dev, metadata(heads), kind, page, pools, scales)
            cache.set_rope(dev.put(cos), dev.put(sin), cos.shape[0])
            cache.reserve(B)
            d_k, d_v, d_off, d_table = dev.put(k), dev.put(v), dev.put(offsets), dev.put(table)
            x = [dev.put(q), dev.put(q)]
            rt.synchronize()
            for i in range(steps):
                row = i * B * H * D * 2
                cache.append(d_k + row, d_v + row, d_table, d_off + i * B * 4, B, table.shape[1], q=x[i % 2], q_out=x[i % 2])
                if idle:
                    rt.synchronize()
                cache.attend(x[i % 2], x[(i + 1) % 2], d_table, d_off + i * B * 4, B, table.shape[1])
                if idle:
                    rt.synchronize()
            rt.synchronize()
            results.append([dev.get(p, q) for p in x] + [dev.get(p, y) for p, y in zip(ptrs, pools)])
            cache.cleanup()
        assert np.isfinite(results[0][0]).all() and results[0][0].any()
        for other in results[1:]:
            assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(results[0], other))
    finally:
        dev.free()
