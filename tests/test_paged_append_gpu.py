"""Paged appends to pages whose scales came from elsewhere, held to what the stored values stand for before and after."""
import numpy as np
import pytest

from oracle import paged_oracle as orc
from tests.paged_case import Device, make_cache, metadata, random_pool, table_of

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(cuda_runtime):
    d = Device(cuda_runtime)
    yield d
    cuda_runtime.synchronize()
    d.free()


def values(stored, scale, kind):
    return orc.widen(stored, kind).astype(np.float64) * scale.astype(np.float64)[:, :, None, None]


def half_step(value, scale, kind):
    """How far a stored value may stand from the `value` that was rounded to it: half a step, and the fp32 roundings of x * (1 / scale)
    and of old / scale, two each, of what is at most 448 or 127 steps."""
    scale = np.abs(scale).astype(np.float64)[..., None]
    own = 0.5 * scale if kind == "int8" else np.maximum(np.abs(value) * 2.0 ** -4, 2.0 ** -10 * scale)
    return own + 2.0 ** -22 * float(orc.LARGEST[kind]) * scale


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("given", [[-0.004, -0.5], [0.0, -0.0], [3.0, -3.0, 1e30], [1e-44, -1e-44, 1e-40]], ids=["negative", "zero", "large", "tiny"])
def test_append_to_pages_with_scales_of_all_kinds(dev, kind, given):
    """Tokens that raise such a scale, tokens that do not, and tokens of zeros."""
    rng = np.random.default_rng([len(given), len(kind)])
    heads, page = (4, 2, 64), 16
    past, new = np.array([3, 9, 15, 1, 7, 12]), np.array([1, 4, 1, 20, 9, 2])
    held = past + new
    table, pages = table_of(rng, held, page)
    pools, scales = map(list, zip(*(random_pool(rng, kind, pages, heads, page) for _ in range(2))))
    for s in scales:
        s[:] = rng.choice(np.array(given, dtype=np.float32), size=s.shape)
    starts, offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32), (held - 1).astype(np.int32)
    x = [rng.standard_normal((int(starts[-1]), 2, 64), dtype=np.float32).astype(np.float16) for _ in range(2)]
    x[0][starts[1]:starts[2]] = 0
    x[1][starts[4]:starts[5]] = 0
    x[1][starts[0]:starts[1]] *= np.float16(0.01)
    cache, ptrs, sc = make_cache(dev, metadata(heads), kind, page, pools, scales)
    cache.append(dev.put(x[0]), dev.put(x[1]), dev.put(table), dev.put(offsets), len(past), table.shape[1], total_tokens=int(starts[-1]),
                 token_starts=dev.put(starts))
    dev.rt.synchronize()
    got = [(dev.get(p, pool), dev.get(s, scale)) for p, pool, s, scale in zip(ptrs, pools, sc, scales)]
    cache.cleanup()
    for rows, pool, scale, (after, now) in zip(x, pools, scales, got):
        assert np.isfinite(now).all()
        before, stands = values(pool, scale, kind), values(after, now, kind)
        for b in range(len(past)):
            for t in range(held[b]):
                p, slot, older = table[b, t // page], t % page, past[b] - t // page * page
                if t < past[b]:
                    value = before[p, :, slot]
                    same = np.abs(now[p]) == np.abs(scale[p])
                    assert np.array_equal(after[p, :, slot][same], pool[p, :, slot][same])
                else:
                    value = rows[starts[b] + t - past[b]].astype(np.float64)
                assert (np.abs(stands[p, :, slot] - value) <= half_step(value, now[p], kind)).all(), (b, t)
                if older > 0:
                    assert ((np.sign(now[p]) == np.sign(scale[p])) | (scale[p] == 0)).all()
    orc.append(pools, scales, kind, x, table, offsets, starts, page)
    for pool, scale, (after, now) in zip(pools, scales, got):
        assert np.array_equal(orc.widen(after, kind), orc.widen(pool, kind)) and np.array_equal(now, scale)


@pytest.mark.parametrize("end", [-1, -2, -2 ** 31])
def test_a_padded_rows_tokens_stay_as_they_were(dev, end):
    """Any negative offset makes all tokens of a row padding, however many there are."""
    rng = np.random.default_rng(5)
    heads, page = (4, 2, 64), 16
    table, pages = table_of(rng, [20, 20], page)
    pools = [random_pool(rng, "f16", pages, heads, page)[0] for _ in range(2)]
    cache, ptrs, _ = make_cache(dev, metadata(heads), "f16", page, pools, (None, None))
    k = rng.standard_normal((10, 2, 64), dtype=np.float32).astype(np.float16)
    q = rng.standard_normal((10, 4, 64), dtype=np.float32).astype(np.float16)
    q_out = np.full_like(q, 7)
    d_q = dev.put(q_out)
    cache.append(dev.put(k), dev.put(k), dev.put(table), dev.put(np.array([end, 4], dtype=np.int32)), 2, table.shape[1], total_tokens=10,
                 q=dev.put(q), q_out=d_q)
    dev.rt.synchronize()
    after, got = dev.get(d_q, q), [dev.get(p, x) for p, x in zip(ptrs, pools)]
    cache.cleanup()
    assert (after[:5] == 7).all() and np.array_equal(after[5:], q[5:])
    orc.append(pools, (None, None), "f16", (k, k), table, [-1, 4], [0, 5, 10], page)
    assert all(np.array_equal(a.view(np.uint16), b.view(np.uint16)) for a, b in zip(got, pools))


def test_older_values_keep_the_whole_range_of_int8(dev):
    """A page that came from elsewhere may hold -128: a scale that grows by less than a half in 128 leaves it so."""
    heads, page, n = (2, 1, 64), 16, 5
    pools = [np.full((1, 1, page, 64), x, dtype=np.int8) for x in (-128, 127)]
    scales = [np.full((1, 1), 1.0, dtype=np.float32) for _ in range(2)]
    x = np.full((1, 1, 64), 127.25, dtype=np.float16)                # 1.00197 of the old scale: 128 / 1.00197 = 127.75
    cache, ptrs, sc = make_cache(dev, metadata(heads), "int8", page, pools, scales)
    cache.append(dev.put(x), dev.put(x), dev.put(np.zeros((1, 1), dtype=np.int32)), dev.put(np.array([n], dtype=np.int32)), 1, 1)
    dev.rt.synchronize()
    got, now = [dev.get(p, y) for p, y in zip(ptrs, pools)], [dev.get(p, y) for p, y in zip(sc, scales)]
    cache.cleanup()
    for after, scale, value in zip(got, now, (-128, 127)):
        assert scale[0, 0] == np.float32(127.25) / np.float32(127)
        assert (after[0, 0, :n] == value).all() and (after[0, 0, n] == 127).all() and (after[0, 0, n + 1:] == value).all()
