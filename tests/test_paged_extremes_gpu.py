"""Paged caches at the ends of what the entry points take: batches, heads and query tokens as many as there may be, rows that lie
apart in memory, and single positions."""
import numpy as np
import pytest

from oracle import paged_oracle as orc
from tests.paged_case import Device, make_cache, metadata, random_pool, table_of, tolerance
from vte_b200.core import PagedKVCache

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(cuda_runtime):
    d = Device(cuda_runtime)
    yield d
    cuda_runtime.synchronize()
    d.free()


def test_the_largest_batch(dev):
    """65,535 sequences of no to three positions, one page for all that have some: each row is the mean of V under its weights."""
    rng = np.random.default_rng(1)
    heads, page, B = (2, 1, 64), 16, 65535
    pools, scales = zip(*(random_pool(rng, "e4m3", 4, heads, page) for _ in range(2)))
    table = rng.integers(0, 4, size=(B, 1)).astype(np.int32)
    lengths = rng.integers(0, 4, size=B)
    q = rng.standard_normal((B, 1, 2, 64), dtype=np.float32).astype(np.float16)
    cache, _, _ = make_cache(dev, metadata(heads), "e4m3", page, pools, scales)
    out = np.full(q.shape, np.nan, dtype=np.float16)
    d_out = dev.put(out)
    cache.attend(dev.put(q), d_out, dev.put(table), dev.put((lengths - 1).astype(np.int32)), B, 1)
    dev.rt.synchronize()
    out = dev.get(d_out, out).astype(np.float64)
    cache.cleanup()
    k, v = (orc.widen(x, "e4m3").astype(np.float64)[:, 0, :3] * s[:, 0, None, None] for x, s in zip(pools, scales))
    seen = np.arange(3)[None] < lengths[:, None]
    s = np.einsum("bhd,btd->bht", q[:, 0].astype(np.float64), k[table[:, 0]]) / 8
    s = np.where(seen[:, None], s, -np.inf)
    p = np.exp(s - np.where(lengths > 0, s.max(axis=2).T, 0).T[:, :, None])
    total = np.where(lengths > 0, p.sum(axis=2).T, 1).T[:, :, None]
    ref, mean = (p @ v[table[:, 0]]) / total, (p @ np.abs(v[table[:, 0]])) / total
    reach = np.abs(s[np.isfinite(s)]).max() + 2.0 ** 5              # sum |q k| / 8 is below 2^5 more than |q k| / 8 (64 products of below 2^2 each)
    assert np.einsum("bhd,btd->bht", np.abs(q[:, 0].astype(np.float64)), np.abs(k[table[:, 0]])).max() / 8 < reach
    assert (np.abs(out[:, 0] - ref) <= tolerance((mean, np.full(ref.shape[:2], reach), 2.0 ** -14 * mean), ref, 64, False)).all()
    assert not out[lengths == 0].any()


@pytest.mark.parametrize("heads,queries,lengths", [((4096, 1, 64), 16, [40, 3, 0]), ((4096, 4096, 64), 1, [5, 1]), ((509, 1, 128), 3, [100, 2]),
                                                   ((2047, 1, 256), 1, [33])], ids=["4096x16_on_1", "4096_on_4096", "509x3_on_1", "2047_on_1"])
def test_the_most_heads(dev, heads, queries, lengths):
    rng = np.random.default_rng([heads[0], queries])
    Hq, H, D = heads
    page = 16
    table, pages = table_of(rng, lengths, page, spare=0)
    pools, scales = zip(*(random_pool(rng, "int8", pages, heads, page) for _ in range(2)))
    q = rng.standard_normal((len(lengths), queries, Hq, D), dtype=np.float32).astype(np.float16)
    cache, _, _ = make_cache(dev, metadata(heads), "int8", page, pools, scales)
    out, lse = np.full(q.shape, np.nan, dtype=np.float16), np.full(q.shape[:3], np.nan, dtype=np.float32)
    d_out, d_lse = dev.put(out), dev.put(lse)
    cache.attend(dev.put(q), d_out, dev.put(table), dev.put(np.asarray(lengths, dtype=np.int32) - 1), len(lengths), table.shape[1],
                 query_tokens=queries, lse=d_lse)
    dev.rt.synchronize()
    out, lse = dev.get(d_out, out).astype(np.float64), dev.get(d_lse, lse)
    cache.cleanup()
    for b, n in enumerate(lengths):
        k, v = (orc.gather(x, s, "int8", table[b, :-(-n // page)], n) for x, s in zip(pools, scales))       # [n, H, D]
        for i in range(queries):
            m = max(n - queries + 1 + i, 0)
            if m == 0:
                assert not out[b, i].any() and (lse[b, i] == -np.inf).all()
                continue
            x = q[b, i].astype(np.float64).reshape(H, Hq // H, D)
            s = np.einsum("hgd,thd->hgt", x, k[:m]) / np.sqrt(D)
            reach = np.einsum("hgd,thd->hgt", np.abs(x), np.abs(k[:m])).max(axis=2) / np.sqrt(D)
            p = np.exp(s - s.max(axis=2, keepdims=True))
            total = p.sum(axis=2, keepdims=True)
            ref, mean = (np.einsum("hgt,thd->hgd", p, y) / total for y in (v[:m], np.abs(v[:m])))
            limit = tolerance((mean, reach, 2.0 ** -14 * np.abs(v[:m]).sum(axis=0)[:, None] + 0 * mean), ref, D, False)
            assert (np.abs(out[b, i].reshape(ref.shape) - ref) <= limit).all(), (b, i)
            assert np.allclose(lse[b, i].reshape(H, -1), s.max(axis=2) + np.log(total[..., 0]), rtol=2.0 ** -22, atol=(D + 8) * 2.0 ** -23 * reach.max() + 2.0 ** -19)


@pytest.mark.parametrize("kind", ["f16", "e4m3", "int8"])
@pytest.mark.parametrize("order", ["heads", "positions"])
def test_rows_that_lie_apart(dev, kind, order):
    """Strides of more than the rows between positions, heads and pages: appended, attended, and nothing written in between."""
    rng = np.random.default_rng(3)
    heads, page, lengths = (6, 3, 64), 32, np.array([70, 1, 33])
    Hq, H, D = heads
    size, dtype = (2, np.float16) if kind == "f16" else (1, np.uint8 if kind == "e4m3" else np.int8)
    pad = 16 // size                                                # values of 16 bytes
    table, pages = table_of(rng, lengths, page)
    inner = (H, page) if order == "heads" else (page, H)
    row, outer = D + pad, (D + pad) * inner[1] + 3 * pad            # of the second and of the first of `inner`
    whole = outer * inner[0] + 5 * pad
    strides = (whole, row, outer) if order == "heads" else (whole, outer, row)
    fill = np.uint8(0x55)
    raw = np.full(pages * whole * size, fill, dtype=np.uint8).view(dtype)
    at = [dev.put(raw) for _ in range(2)]
    scale = np.full((pages, H), 7, dtype=np.float32)
    sc = [dev.put(scale) for _ in range(2)] if kind != "f16" else [0, 0]
    cache = PagedKVCache(dev.rt, metadata(heads), pages, page, kind, k_pool=at[0], v_pool=at[1], k_scale=sc[0], v_scale=sc[1], strides=strides)
    n = int(lengths.sum())
    starts, offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32), (lengths - 1).astype(np.int32)
    k, v = (rng.standard_normal((n, H, D), dtype=np.float32).astype(np.float16) for _ in range(2))
    q = rng.standard_normal((len(lengths), 1, Hq, D), dtype=np.float32).astype(np.float16)
    d_out, d_table, d_off = dev.put(q), dev.put(table), dev.put(offsets)
    cache.append(dev.put(k), dev.put(v), d_table, d_off, len(lengths), table.shape[1], total_tokens=n, token_starts=dev.put(starts))
    cache.attend(dev.put(q), d_out, d_table, d_off, len(lengths), table.shape[1])
    dev.rt.synchronize()
    out, got = dev.get(d_out, q), [dev.get(p, raw) for p in at]
    now = [dev.get(p, scale) if p else None for p in sc]
    cache.cleanup()
    pools = [np.zeros((pages, H, page, D), dtype=dtype) for _ in range(2)]
    scales = [scale.copy() if kind != "f16" else None for _ in range(2)]
    orc.append(pools, scales, kind, (k, v), table, offsets, starts, page)
    held = np.zeros((pages, page), dtype=bool)
    for b, m in enumerate(lengths):
        for t in range(m):
            held[table[b, t // page], t % page] = True
    index = (np.arange(pages)[:, None, None, None] * strides[0] + np.arange(H)[None, :, None, None] * strides[2] +
             np.arange(page)[None, None, :, None] * strides[1] + np.arange(D))
    written = np.zeros(raw.shape, dtype=bool)
    for have, pool, s, s_now in zip(got, pools, scales, now):
        where = np.broadcast_to(held[:, None, :, None], pool.shape)
        assert np.array_equal(have[index][where].view(np.uint8), pool[where].view(np.uint8))
        assert s is None or np.array_equal(s, s_now)
        written[index[where]] = True
        assert (have[~written].view(np.uint8) == fill).all()
    ref, _, bound = orc.attention(q, *pools, *scales, kind, table, offsets, 1.0 / np.sqrt(D))
    assert (np.abs(out - ref) <= tolerance(bound, ref, D, False)).all()
