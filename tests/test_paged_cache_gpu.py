"""Paged caches on the device: the append against its restatement bit for bit, the attention against the definition in 64
bits within the roundings that the kernel makes (tests/paged_case.py, `tolerance`), and a step of the two together."""
import ctypes

import numpy as np
import pytest

from oracle import paged_oracle as orc
from tests.paged_case import (Device, get_pool, make_cache, metadata, poison, put_pool, random_pool, table_of, tolerance,
                              unseen_rows)
from vte_b200.bridge import CudaRuntimeError, CudaSafetyError
from vte_b200.core import PagedKVCache
from vte_b200.workloads import build_rope_cache

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(cuda_runtime):
    d = Device(cuda_runtime)
    yield d
    cuda_runtime.synchronize()
    d.free()


def attend(dev, kind, heads, page, lengths, queries=1, layout="heads", f32=False, seed=0, sigma=1.0, poisoned=True, repeat=1):
    """The kernel's (output, lse) and the definition's (output, lse, bound)."""
    rng = np.random.default_rng([seed, page, len(lengths)])
    lengths = np.asarray(lengths)
    Hq, H, D = heads
    table, pages = table_of(rng, lengths, page)
    pools, scales = zip(*(random_pool(rng, kind, pages, heads, page, sigma) for _ in range(2)))
    if poisoned:
        unseen = unseen_rows(table, lengths, pages, page)
        for x, s in zip(pools, scales):
            poison(x, s, kind, unseen, rng)
    cache, _, _ = make_cache(dev, metadata(heads), kind, page, pools, scales, layout)
    q = rng.standard_normal((len(lengths), queries, Hq, D), dtype=np.float32).astype(np.float16)
    offsets = (lengths - 1).astype(np.int32)
    out = np.full(q.shape, np.nan, dtype=np.float32 if f32 else np.float16)
    lse = np.full(q.shape[:3], np.nan, dtype=np.float32)
    d_out, d_lse = dev.put(out), dev.put(lse)
    args = (dev.put(q), d_out, dev.put(table), dev.put(offsets), len(lengths), table.shape[1])
    got = []
    try:
        for _ in range(repeat):
            cache.attend(*args, query_tokens=queries, output_f32=f32, lse=d_lse)
            dev.rt.synchronize()
            got.append((dev.get(d_out, out), dev.get(d_lse, lse)))
    finally:
        cache.cleanup()
    for again in got[1:]:
        assert np.array_equal(again[0], got[0][0]) and np.array_equal(again[1], got[0][1])
    want = orc.attention(q, pools[0], pools[1], scales[0], scales[1], kind, table, offsets, 1.0 / np.sqrt(D))
    return got[0], want


def check(got, want, D, f32=False):
    (out, lse), (ref, ref_lse, bound) = got, want
    assert np.isfinite(out).all()
    off = np.abs(out.astype(np.float64) - ref)
    allowed = tolerance(bound, ref, D, f32)
    worst = np.unravel_index(np.argmax(off - allowed), off.shape)
    assert (off <= allowed).all(), (worst, off[worst], allowed[worst], out[worst], ref[worst])
    seen = np.isfinite(ref_lse)
    assert np.array_equal(seen, np.isfinite(lse)) and (lse[~seen] == -np.inf).all()
    # a sum of weights each off by at most (D + 8) roundings of `reach` and 2^-20, and the logarithm's own two roundings
    reach = bound[1][seen]
    assert (np.abs(lse[seen] - ref_lse[seen]) <= (D + 8) * 2.0 ** -23 * reach + 2.0 ** -19 + 2.0 ** -22 * np.abs(ref_lse[seen])).all()


HEADS = [(12, 2, 128), (32, 8, 64), (8, 2, 256), (7, 1, 128), (32, 2, 64), (28, 1, 128), (5, 5, 64), (12, 1, 256)]


@pytest.mark.parametrize("kind", ["f16", "e4m3", "int8"])
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
def test_attention_of_short_and_odd_lengths(dev, kind, heads):
    for page in (16, 64):
        lengths = [1, 0, page - 1, page, page + 1, 2, 3 * page + 5, 0, 257, 15, 33, 640]
        got, want = attend(dev, kind, heads, page, lengths, layout="positions" if page == 16 else "heads")
        check(got, want, heads[2])


@pytest.mark.parametrize("kind", ["f16", "e4m3", "int8"])
@pytest.mark.parametrize("heads,page,lengths", [
    ((12, 2, 128), 64, [4999]), ((12, 2, 128), 16, [1]), ((12, 2, 128), 128, [20000]), ((8, 2, 256), 32, [7001, 3]),
    ((32, 8, 64), 128, [3000, 1, 0, 12000, 77]), ((16, 2, 128), 32, [9000, 9001, 8999]),
], ids=["one_4999", "one_1", "one_20000", "two_256wide", "ragged_64wide", "three_even"])
def test_attention_of_sequences_that_are_cut(dev, kind, heads, page, lengths):
    """Segments cut between workers: fp32 outputs, the same bits on every call."""
    got, want = attend(dev, kind, heads, page, lengths, f32=True, repeat=3)
    check(got, want, heads[2], f32=True)


@pytest.mark.parametrize("batch,lo,hi", [(300, 0, 90), (64, 100, 900), (600, 1, 3)])
def test_attention_of_many_sequences(dev, batch, lo, hi):
    lengths = np.random.default_rng(batch).integers(lo, hi, size=batch)
    got, want = attend(dev, "e4m3", (8, 4, 64), 16, lengths, repeat=2)
    check(got, want, 64)


@pytest.mark.parametrize("kind", ["f16", "e4m3", "int8"])
@pytest.mark.parametrize("heads,queries", [((32, 8, 64), 4), ((12, 2, 128), 2), ((8, 2, 256), 5), ((12, 2, 128), 16), ((4, 4, 64), 3)],
                         ids=["4x4", "6x2", "4x5_256wide", "6x16", "1x3"])
def test_attention_of_several_query_tokens(dev, kind, heads, queries):
    """Causal among the newest tokens; sequences shorter than those, whose first rows see nothing."""
    lengths = [queries, 1, 0, 130, queries - 1, 64 + queries, 1000, 63]
    for f32 in (False, True):
        got, want = attend(dev, kind, heads, 32, lengths, queries=queries, f32=f32)
        check(got, want, heads[2], f32)


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
def test_what_a_row_does_not_see_does_not_reach_it(dev, kind):
    """Infinities and NaN in the rows of the newest tokens reach only the query tokens that see them."""
    rng = np.random.default_rng(3)
    heads, page, queries, n = (8, 2, 128), 16, 4, 50
    table, pages = table_of(rng, [n], page)
    pools, scales = zip(*(random_pool(rng, kind, pages, heads, page) for _ in range(2)))
    last = table[0, (n - 2) // page], (n - 2) % page             # position n - 2: seen by the last two query tokens
    bad = np.float16(np.inf) if kind == "f16" else np.uint8(0x7f)
    pools[1][last[0], :, last[1], 7] = bad
    cache, _, _ = make_cache(dev, metadata(heads), kind, page, pools, scales)
    q = rng.standard_normal((1, queries, heads[0], heads[2]), dtype=np.float32).astype(np.float16)
    out = np.zeros(q.shape, dtype=np.float16)
    d_out = dev.put(out)
    cache.attend(dev.put(q), d_out, dev.put(table), dev.put(np.array([n - 1], dtype=np.int32)), 1, table.shape[1], query_tokens=queries)
    dev.rt.synchronize()
    out = dev.get(d_out, out)
    cache.cleanup()
    assert np.isfinite(out[:, :2]).all()
    assert not np.isfinite(out[:, 2:, :, 7]).any()
    assert np.isfinite(np.delete(out[:, 2:], 7, axis=-1)).all()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_scales_of_very_different_size(dev, kind):
    """Scales from 1e-30 to 1e20 beside each other, of both signs, and pages of zeros with a scale of zero; then negative ones alone."""
    rng = np.random.default_rng(9)
    heads, page, n = (8, 2, 64), 16, 400
    table, pages = table_of(rng, [n], page)
    pools, scales = map(list, zip(*(random_pool(rng, kind, pages, heads, page) for _ in range(2))))
    scales[1] = (10.0 ** rng.uniform(-30, 20, size=scales[1].shape)).astype(np.float32)
    scales[1] *= rng.choice(np.array([-1, 1], dtype=np.float32), size=scales[1].shape)
    zero = table[0, 3]
    for x, s in zip(pools, scales):
        x[zero], s[zero] = 0, 0
    q = rng.standard_normal((1, 1, heads[0], heads[2]), dtype=np.float32).astype(np.float16)
    offsets = np.array([n - 1], dtype=np.int32)
    for negative in (False, True):
        if negative:
            scales[1] = -np.abs(scales[1][::-1]).clip(1e-3, 1e3)
            scales[0] = -scales[0]
        cache, _, _ = make_cache(dev, metadata(heads), kind, page, pools, scales)
        out = np.zeros(q.shape, dtype=np.float32)
        d_out = dev.put(out)
        cache.attend(dev.put(q), d_out, dev.put(table), dev.put(offsets), 1, table.shape[1], output_f32=True)
        dev.rt.synchronize()
        out = dev.get(d_out, out)
        cache.cleanup()
        ref, _, bound = orc.attention(q, *pools, *scales, kind, table, offsets, 1.0 / 8)
        assert (np.abs(out - ref) <= tolerance(bound, ref, 64, True)).all()


# ---- append ------------------------------------------------------------------------------------------------------------
def append(dev, kind, heads, page, past, new, rope_type=0, rotary_dim=0, layout="heads", padded=0, seed=1, uniform=False, big=False):
    """Appends on the device and in numpy; returns both sides' (pools, scales, rotated q)."""
    rng = np.random.default_rng([seed, page, len(past)])
    past, new = np.asarray(past), np.asarray(new)
    Hq, H, D = heads
    held = past + new
    table, pages = table_of(rng, held, page)
    pools, scales = map(list, zip(*(random_pool(rng, kind, pages, heads, page) for _ in range(2))))
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    offsets = (held - 1).astype(np.int32)
    if padded:
        offsets[-padded:] = -1
    rows = int(starts[-1])
    k, v, q = (rng.standard_normal((rows, h, D), dtype=np.float32).astype(np.float16) for h in (H, H, Hq))
    if big:                                    # tokens that raise the scale, and tokens that do not
        k[::2] *= np.float16(8)
        v[::3] *= np.float16(0.125)
    width = rotary_dim if rope_type == 2 else D
    cos, sin = build_rope_cache(int(held.max()) + 1, max(width, 2), 1e4)
    cache, ptrs, sc = make_cache(dev, metadata(heads, rope_type, rotary_dim), kind, page, pools, scales, layout)
    if rope_type >= 0:
        cache.set_rope(dev.put(cos), dev.put(sin), cos.shape[0])
    q_out = np.full(q.shape, 7, dtype=np.float16)
    d_q = dev.put(q_out)
    cache.append(dev.put(k), dev.put(v), dev.put(table), dev.put(offsets), len(past), table.shape[1], total_tokens=rows,
                 token_starts=0 if uniform else dev.put(starts), q=dev.put(q), q_out=d_q)
    dev.rt.synchronize()
    got = ([get_pool(dev, p, x, layout) for p, x in zip(ptrs, pools)], [dev.get(p, s) if p else None for p, s in zip(sc, scales)],
           dev.get(d_q, q_out))
    cache.cleanup()
    seq = np.repeat(np.arange(len(past)), new)
    pos = offsets[seq] - (starts[seq + 1] - 1 - np.arange(rows))
    kept = pos >= 0
    rot = lambda x: np.where(kept[:, None, None], orc.rotate(x, np.maximum(pos, 0), cos, sin, rope_type, rotary_dim), x)   # noqa: E731
    orc.append(pools, scales, kind, (rot(k), v), table, offsets, starts, page)
    return got, (pools, scales, np.where(kept[:, None, None], rot(q), q_out))


def same(got, want):
    for x, y in zip(got[0], want[0]):
        assert np.array_equal(x.view(np.uint8 if x.dtype.itemsize == 1 else np.uint16), y.view(np.uint8 if y.dtype.itemsize == 1 else np.uint16))
    for x, y in zip(got[1], want[1]):
        assert x is None or np.array_equal(x, y, equal_nan=True)
    assert np.array_equal(got[2].view(np.uint16), want[2].view(np.uint16))


ROPES = [(0, 0), (1, 0), (2, 32), (-1, 0)]


@pytest.mark.parametrize("kind", ["f16", "e4m3", "int8"])
@pytest.mark.parametrize("rope", ROPES, ids=["split_half", "adjacent", "partial", "none"])
def test_append_of_one_token_each(dev, kind, rope):
    for heads, page, layout in (((12, 2, 128), 16, "heads"), ((32, 8, 64), 64, "positions"), ((8, 2, 256), 128, "heads")):
        past = [0, 1, page - 1, page, page + 1, 700, 5, 0]
        got, want = append(dev, kind, heads, page, past, [1] * len(past), *rope, layout=layout, padded=1, uniform=True, big=True)
        same(got, want)


@pytest.mark.parametrize("kind", ["f16", "e4m3", "int8"])
@pytest.mark.parametrize("rope", ROPES, ids=["split_half", "adjacent", "partial", "none"])
def test_append_of_ragged_prompts(dev, kind, rope):
    for heads, page, layout in (((12, 2, 128), 32, "heads"), ((4, 1, 64), 16, "positions"), ((4, 2, 256), 128, "heads"), ((5, 5, 64), 64, "heads")):
        past = [0, 3, page - 1, 0, 2 * page, 50, 7]
        new = [1, page, page + 1, 0, 3 * page, 2 * page - 1, 333]
        got, want = append(dev, kind, heads, page, past, new, *rope, layout=layout, big=True)
        same(got, want)


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
def test_append_of_the_same_number_each(dev, kind):
    got, want = append(dev, kind, (12, 2, 128), 32, [0, 31, 70, 5], [40] * 4, uniform=True)
    same(got, want)


def test_append_of_padded_tokens(dev):
    """Tokens at negative positions are padding: a prompt whose newest token has position 4 of 9 rows."""
    for kind in ("f16", "int8"):
        rng = np.random.default_rng(2)
        heads, page = (4, 2, 64), 16
        table, pages = table_of(rng, [5], page)
        pools, scales = map(list, zip(*(random_pool(rng, kind, pages, heads, page) for _ in range(2))))
        k, v = (rng.standard_normal((9, 2, 64), dtype=np.float32).astype(np.float16) for _ in range(2))
        cache, ptrs, sc = make_cache(dev, metadata(heads), kind, page, pools, scales)
        starts, offsets = np.array([0, 9], dtype=np.int32), np.array([4], dtype=np.int32)
        cache.append(dev.put(k), dev.put(v), dev.put(table), dev.put(offsets), 1, table.shape[1], total_tokens=9, token_starts=dev.put(starts))
        dev.rt.synchronize()
        got = [dev.get(p, x) for p, x in zip(ptrs, pools)], [dev.get(p, s) if p else None for p, s in zip(sc, scales)], k
        cache.cleanup()
        orc.append(pools, scales, kind, (k, v), table, offsets, starts, page)
        same(got, (pools, scales, k))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_of_what_is_not_finite_and_of_zeros(dev, kind):
    rng = np.random.default_rng(4)
    heads, page, D = (4, 2, 64), 16, 64
    table, pages = table_of(rng, [4, 4, 4], page)
    pools, scales = map(list, zip(*(random_pool(rng, kind, pages, heads, page) for _ in range(2))))
    k, v = (rng.standard_normal((3, 2, D), dtype=np.float32).astype(np.float16) for _ in range(2))
    k[0, 0, 3], k[1, 1, 5], v[2] = np.nan, np.inf, 0
    offsets, starts = np.array([3, 0, 0], dtype=np.int32), np.arange(4, dtype=np.int32)
    cache, ptrs, sc = make_cache(dev, metadata(heads), kind, page, pools, scales)
    cache.append(dev.put(k), dev.put(v), dev.put(table), dev.put(offsets), 3, table.shape[1])
    dev.rt.synchronize()
    got = [dev.get(p, x) for p, x in zip(ptrs, pools)], [dev.get(p, s) for p, s in zip(sc, scales)]
    cache.cleanup()
    orc.append(pools, scales, kind, (k, v), table, offsets, starts, page)
    for x, y in zip(got[1], scales):
        assert np.array_equal(x, y, equal_nan=True)
    assert np.isnan(got[1][0][table[0, 0], 0]) and np.isnan(got[1][0][table[1, 0], 1])
    assert (got[1][1][table[2, 0]] == 0).all() and not got[0][1][table[2, 0], :, 0].any()
    for x, y in zip(got[0], pools):
        assert np.array_equal(orc.widen(x, kind), orc.widen(y, kind), equal_nan=True)


def test_append_from_one_projection_in_place(dev):
    """q, k and v as parts of a projection's rows, q rotated where it lies."""
    rng = np.random.default_rng(6)
    Hq, H, D = heads = (6, 2, 64)
    page, n = 16, 5
    row = (Hq + 2 * H) * D
    x = rng.standard_normal((n, row), dtype=np.float32).astype(np.float16)
    table, pages = table_of(rng, [n], page)
    pools, scales = map(list, zip(*(random_pool(rng, "f16", pages, heads, page) for _ in range(2))))
    cos, sin = build_rope_cache(n, D, 1e4)
    cache, ptrs, _ = make_cache(dev, metadata(heads), "f16", page, pools, scales)
    cache.set_rope(dev.put(cos), dev.put(sin), n)
    at = dev.put(x)
    cache.append(at + Hq * D * 2, at + (Hq + H) * D * 2, dev.put(table), dev.put(np.array([n - 1], dtype=np.int32)), 1, table.shape[1],
                 total_tokens=n, token_starts=dev.put(np.array([0, n], dtype=np.int32)), q=at, q_out=at, token_strides=(row,) * 4)
    dev.rt.synchronize()
    after = dev.get(at, x)
    got = [dev.get(p, y) for p, y in zip(ptrs, pools)]
    cache.cleanup()
    pos = np.arange(n)
    q, k, v = (a.reshape(n, -1, D) for a in (x[:, :Hq * D], x[:, Hq * D:(Hq + H) * D], x[:, (Hq + H) * D:]))
    assert np.array_equal(after[:, :Hq * D].reshape(n, Hq, D), orc.rotate(q, pos, cos, sin, 0, D))
    assert np.array_equal(after[:, Hq * D:], x[:, Hq * D:])
    orc.append(pools, scales, "f16", (orc.rotate(k, pos, cos, sin, 0, D), v), table, [n - 1], [0, n], page)
    assert all(np.array_equal(a.view(np.uint16), b.view(np.uint16)) for a, b in zip(got, pools))


# ---- together ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f16", "e4m3", "int8"])
def test_prompt_then_steps_in_a_graph(dev, kind):
    """Prompts, then decode steps of two layers from one captured graph that reads its offsets from memory; the layers
    share a workspace, and the cache is the runtime's own."""
    rt = dev.rt
    rng = np.random.default_rng(11)
    Hq, H, D = heads = (8, 2, 128)
    page, layers, steps = 16, 2, 20
    prompts = np.array([30, 1, 15, 77])
    B = len(prompts)
    table, pages = table_of(rng, prompts + steps, page)
    cos, sin = build_rope_cache(int(prompts.max()) + steps, D, 1e4)
    meta = metadata(heads)
    d_table, d_cos, d_sin = dev.put(table), dev.put(cos), dev.put(sin)
    caches = [PagedKVCache(rt, meta, pages, page, kind) for _ in range(layers)]
    need = PagedKVCache.workspace_bytes(rt, meta, B)
    scratch = rt.safe_malloc(need, "scratch")
    rt.safe_memset(scratch, need)
    rt.synchronize()
    dtype = np.float16 if kind == "f16" else np.uint8 if kind == "e4m3" else np.int8
    image = [([np.zeros((pages, H, page, D), dtype=dtype) for _ in range(2)], [np.zeros((pages, H), dtype=np.float32) for _ in range(2)]) for _ in range(layers)]
    starts = np.concatenate([[0], np.cumsum(prompts)]).astype(np.int32)
    seq = np.repeat(np.arange(B), prompts)
    pos = np.arange(starts[-1]) - starts[seq]
    new = lambda n, h: rng.standard_normal((n, h, D), dtype=np.float32).astype(np.float16)     # noqa: E731
    d_starts, d_off = dev.put(starts), dev.put((prompts - 1).astype(np.int32))
    for c, (pools, scales) in zip(caches, image):
        c.set_rope(d_cos, d_sin, cos.shape[0])
        k, v = new(starts[-1], H), new(starts[-1], H)
        c.append(dev.put(k), dev.put(v), d_table, d_off, B, table.shape[1], total_tokens=int(starts[-1]), token_starts=d_starts)
        orc.append(pools, scales, kind, (orc.rotate(k, pos, cos, sin, 0, D), v), table, prompts - 1, starts, page)
    bufs = [[dev.put(np.zeros((B, h, D), dtype=np.float16)) for h in (H, H, Hq, Hq, Hq)] for _ in range(layers)]   # k, v, q, rotated q, out
    rt.synchronize()
    rt.stream_begin_capture()
    for c, (k, v, q, qr, out) in zip(caches, bufs):
        c.append(k, v, d_table, d_off, B, table.shape[1], q=q, q_out=qr)
        c.attend(qr, out, d_table, d_off, B, table.shape[1], workspace=scratch, workspace_bytes=need)
    graph = rt.stream_end_capture()
    step = rt.graph_instantiate(graph)
    rt.graph_destroy(graph)
    for i in range(steps):
        offsets = (prompts + i).astype(np.int32)
        rt.safe_memcpy_host_to_device(ctypes.c_void_p(d_off), offsets)
        fresh = [[new(B, h) for h in (H, H, Hq)] for _ in range(layers)]
        for b, f in zip(bufs, fresh):
            for p, x in zip(b, f):
                rt.safe_memcpy_host_to_device(ctypes.c_void_p(p), x)
        rt.graph_launch(step)
        rt.synchronize()
        for (pools, scales), (k, v, q), b in zip(image, fresh, bufs):
            orc.append(pools, scales, kind, (orc.rotate(k, offsets, cos, sin, 0, D), v), table, offsets, np.arange(B + 1), page)
            q = orc.rotate(q, offsets, cos, sin, 0, D)
            assert np.array_equal(dev.get(b[3], q), q)
            out = dev.get(b[4], q).astype(np.float64)
            ref, _, bound = orc.attention(q[:, None], *pools, *scales, kind, table, offsets, 1.0 / np.sqrt(D))
            assert (np.abs(out - ref[:, 0]) <= tolerance(bound, ref, D, False)[:, 0]).all()
    for c, (pools, scales) in zip(caches, image):
        held = unseen_rows(table, prompts + steps, pages, page)
        for p, x in ((c.k_pool, pools[0]), (c.v_pool, pools[1])):
            rows = np.broadcast_to(~held[:, None, :], x.shape[:3])
            assert np.array_equal(dev.get(p, x)[rows].view(np.uint8), x[rows].view(np.uint8))
        c.cleanup()
    rt.graph_exec_destroy(step)
    rt.safe_free(scratch)


def test_bad_pages_and_positions_are_reported(dev):
    """A table entry outside the pool, a position behind the table and one behind the rotation tables: nothing is read or
    written there, the other sequences are served, and the next wait says so."""
    rt = dev.rt
    rng = np.random.default_rng(13)
    heads, page = (8, 2, 64), 16
    lengths = np.array([40, 20, 33])
    for kind in ("f16", "e4m3", "int8"):
        table, pages = table_of(rng, lengths, page)
        pools, scales = map(list, zip(*(random_pool(rng, kind, pages, heads, page) for _ in range(2))))
        cache, ptrs, _ = make_cache(dev, metadata(heads), kind, page, pools, scales)
        q = rng.standard_normal((3, 1, 8, 64), dtype=np.float32).astype(np.float16)
        d_out, d_q = dev.put(q), dev.put(q)
        for entry in (pages, -1):
            wrong = table.copy()
            wrong[1, 1] = entry
            offsets = (lengths - 1).astype(np.int32)
            cache.attend(d_q, d_out, dev.put(wrong), dev.put(offsets), 3, table.shape[1])
            with pytest.raises(CudaRuntimeError, match="page outside the pool"):
                rt.synchronize()
            out = dev.get(d_out, q)
            ref, _, bound = orc.attention(q[[0, 2]], *pools, *scales, kind, table[[0, 2]], offsets[[0, 2]], 1.0 / 8)
            assert np.isnan(out[1]).all() and (np.abs(out[[0, 2]] - ref) <= tolerance(bound, ref, 64, False)).all()
            k = q[:, 0, :2].copy()
            cache.append(dev.put(k), dev.put(k), dev.put(wrong), dev.put(np.array([-1, 16, -1], dtype=np.int32)), 3, table.shape[1])
            with pytest.raises(CudaRuntimeError, match="page outside the pool"):
                rt.synchronize()
            assert all(np.array_equal(dev.get(p, x).view(np.uint8), x.view(np.uint8)) for p, x in zip(ptrs, pools))
        room = table.shape[1] * page
        cache.append(dev.put(k), dev.put(k), dev.put(table), dev.put(np.array([room, -1, -1], dtype=np.int32)), 3, table.shape[1])
        with pytest.raises(CudaRuntimeError, match="beyond its block table"):
            rt.synchronize()
        cos, sin = build_rope_cache(8, 64, 1e4)
        cache.set_rope(dev.put(cos), dev.put(sin), 8)
        cache.append(dev.put(k), dev.put(k), dev.put(table), dev.put(np.array([8, -1, -1], dtype=np.int32)), 3, table.shape[1])
        with pytest.raises(CudaRuntimeError, match="rotation tables"):
            rt.synchronize()
        assert all(np.array_equal(dev.get(p, x).view(np.uint8), x.view(np.uint8)) for p, x in zip(ptrs, pools))
        full = table.copy()
        cache.attend(d_q, d_out, dev.put(np.ascontiguousarray(full[:1])), dev.put(np.array([room + 5], dtype=np.int32)), 1, table.shape[1]) if (full[0] >= 0).all() else None
        if (full[0] >= 0).all():
            with pytest.raises(CudaRuntimeError, match="beyond its block table"):
                rt.synchronize()
        cache.cleanup()


def test_nothing_cached(dev):
    for lengths in ([0], [0, 0, 0]):
        (out, lse), _ = attend(dev, "e4m3", (8, 2, 128), 16, lengths, queries=2)
        assert not out.any() and (lse == -np.inf).all()


def test_pages_far_into_a_large_pool(dev):
    """Pools of more than 2^32 values: the pages that are used lie at their ends."""
    rt = dev.rt
    rng = np.random.default_rng(21)
    heads, page, n = (4, 2, 128), 128, 300
    Hq, H, D = heads
    pages = (1 << 32) // (H * page * D) + 40
    cache = PagedKVCache(rt, metadata(heads), pages, page, "e4m3")
    try:
        table = np.array([[pages - 1, pages - 3, 131072]], dtype=np.int32)       # the last one begins at 2^32
        k, v = (rng.standard_normal((n, H, D), dtype=np.float32).astype(np.float16) for _ in range(2))
        q = rng.standard_normal((1, 1, Hq, D), dtype=np.float32).astype(np.float16)
        offsets = np.array([n - 1], dtype=np.int32)
        d_table, d_off, d_out = dev.put(table), dev.put(offsets), dev.put(q)
        cache.append(dev.put(k), dev.put(v), d_table, d_off, 1, 3, total_tokens=n)
        cache.attend(dev.put(q), d_out, d_table, d_off, 1, 3)
        rt.synchronize()
        small = np.array([[0, 1, 2]], dtype=np.int32)
        pools, scales = [np.zeros((3, H, page, D), dtype=np.uint8) for _ in range(2)], [np.zeros((3, H), dtype=np.float32) for _ in range(2)]
        orc.append(pools, scales, "e4m3", (k, v), small, offsets, [0, n], page)
        for ptr, pool in ((cache.k_pool, pools[0]), (cache.v_pool, pools[1])):
            for i, at in enumerate(table[0]):
                rows = min(page, n - i * page)
                got = dev.get(ptr + int(at) * H * page * D, pool[i])
                assert np.array_equal(got[:, :rows], pool[i][:, :rows])
        ref, _, bound = orc.attention(q, *pools, *scales, "e4m3", small, offsets, 1.0 / np.sqrt(D))
        assert (np.abs(dev.get(d_out, q) - ref) <= tolerance(bound, ref, D, False)).all()
    finally:
        cache.cleanup()


def test_one_pool_for_k_and_v_and_pages_that_sequences_share(dev):
    """K and V of a page side by side in one pool, and a prefix whose pages are two sequences'."""
    rng = np.random.default_rng(22)
    heads, page = (6, 3, 64), 32
    Hq, H, D = heads
    lengths = np.array([70, 90])
    pages = 6
    table = np.array([[4, 2, 0], [4, 2, 5]], dtype=np.int32)
    both = rng.standard_normal((pages, 2, H, page, D), dtype=np.float32).astype(np.float16)
    at = dev.put(both)
    cache = PagedKVCache(dev.rt, metadata(heads), pages, page, "f16", k_pool=at, v_pool=at + H * page * D * 2,
                         strides=(2 * H * page * D, D, page * D))
    q = rng.standard_normal((2, 1, Hq, D), dtype=np.float32).astype(np.float16)
    d_out, offsets = dev.put(q), (lengths - 1).astype(np.int32)
    cache.attend(dev.put(q), d_out, dev.put(table), dev.put(offsets), 2, 3)
    dev.rt.synchronize()
    ref, _, bound = orc.attention(q, both[:, 0], both[:, 1], None, None, "f16", table, offsets, 1.0 / np.sqrt(D))
    assert (np.abs(dev.get(d_out, q) - ref) <= tolerance(bound, ref, D, False)).all()
    cache.cleanup()


def test_another_stream_and_a_workspace_for_all_shapes(dev):
    """Calls of different shapes one behind the other on a stream of the caller's, all with one workspace, which each of them
    leaves ready for the next."""
    rt = dev.rt
    rng = np.random.default_rng(23)
    stream = ctypes.c_void_p()
    assert rt._lib.vteb_stream_create(ctypes.byref(stream)) == 0
    shapes = [((12, 2, 128), 16, [3000]), ((32, 8, 64), 64, [10, 700, 0, 90, 5000]), ((8, 2, 256), 32, [2500, 40]), ((12, 2, 128), 16, [200] * 90)]
    need = max(PagedKVCache.workspace_bytes(rt, metadata(h), len(n), 4) for h, _, n in shapes)
    scratch = rt.safe_malloc(need, "scratch")
    rt.safe_memset(scratch, need)
    rt.synchronize()
    runs = []
    for heads, page, lengths in shapes + shapes[::-1]:
        kind = ("f16", "e4m3", "int8")[len(runs) % 3]
        table, pages = table_of(rng, lengths, page)
        pools, scales = zip(*(random_pool(rng, kind, pages, heads, page) for _ in range(2)))
        cache, _, _ = make_cache(dev, metadata(heads), kind, page, pools, scales)
        queries = 1 + len(runs) % 3
        q = rng.standard_normal((len(lengths), queries, heads[0], heads[2]), dtype=np.float32).astype(np.float16)
        offsets = np.asarray(lengths, dtype=np.int32) - 1
        d_out = dev.put(np.zeros_like(q))
        args = (dev.put(q), d_out, dev.put(table), dev.put(offsets), len(lengths), table.shape[1])
        runs.append((cache, args, queries, q, d_out, (pools, scales, kind, table, offsets), heads))
    for cache, args, queries, *_ in runs:
        cache.attend(*args, query_tokens=queries, workspace=scratch, workspace_bytes=need, stream=stream.value)
    rt.synchronize()
    for cache, _, _, q, d_out, (pools, scales, kind, table, offsets), heads in runs:
        ref, _, bound = orc.attention(q, *pools, *scales, kind, table, offsets, 1.0 / np.sqrt(heads[2]))
        assert (np.abs(dev.get(d_out, q) - ref) <= tolerance(bound, ref, heads[2], False)).all()
        cache.cleanup()
    with pytest.raises(CudaSafetyError, match="workspace holds"):
        runs[0][0].attend(*runs[0][1], workspace=scratch, workspace_bytes=1000)
    rt.safe_free(scratch)
    assert rt._lib.vteb_stream_destroy(stream) == 0


def test_two_graphs_on_two_streams(dev):
    """Two captured steps, each with its cache and its workspace, replayed on two streams at once."""
    rt = dev.rt
    rng = np.random.default_rng(24)
    heads, page = (12, 2, 128), 64
    steps = []
    for n in (9000, 12000):
        table, pages = table_of(rng, [n], page)
        pools, scales = zip(*(random_pool(rng, "e4m3", pages, heads, page) for _ in range(2)))
        cache, _, _ = make_cache(dev, metadata(heads), "e4m3", page, pools, scales)
        cache.reserve(1)
        q = rng.standard_normal((1, 1, heads[0], heads[2]), dtype=np.float32).astype(np.float16)
        offsets = np.array([n - 1], dtype=np.int32)
        d_out = dev.put(np.zeros_like(q))
        args = (dev.put(q), d_out, dev.put(table), dev.put(offsets), 1, table.shape[1])
        rt.synchronize()
        rt.stream_begin_capture()
        for _ in range(8):
            cache.attend(*args)
        graph = rt.stream_end_capture()
        stream = ctypes.c_void_p()
        assert rt._lib.vteb_stream_create(ctypes.byref(stream)) == 0
        steps.append((rt.graph_instantiate(graph), stream, cache, q, d_out, (pools, scales, table, offsets)))
        rt.graph_destroy(graph)
    for _ in range(20):
        for step, stream, *_ in steps:
            assert rt._lib.vteb_graph_launch(step, stream) == 0
    rt.synchronize()
    for step, stream, cache, q, d_out, (pools, scales, table, offsets) in steps:
        ref, _, bound = orc.attention(q, *pools, *scales, "e4m3", table, offsets, 1.0 / np.sqrt(128))
        assert (np.abs(dev.get(d_out, q) - ref) <= tolerance(bound, ref, 128, False)).all()
        rt.graph_exec_destroy(step)
        cache.cleanup()
        assert rt._lib.vteb_stream_destroy(stream) == 0
