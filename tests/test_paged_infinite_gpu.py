"""Paged attention over 16-bit pages with infinite values: a row that sees one is infinite in that channel, whatever the weight's
size, its parts and the pieces that are merged; it is NaN only where infinities of both signs meet.  All other outputs are
held to the definition as if the infinities were zero."""
import numpy as np
import pytest

from oracle import paged_oracle as orc
from tests.paged_case import Device, make_cache, metadata, random_pool, table_of, tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(cuda_runtime):
    d = Device(cuda_runtime)
    yield d
    cuda_runtime.synchronize()
    d.free()


@pytest.mark.parametrize("f32", [False, True], ids=["f16_out", "f32_out"])
@pytest.mark.parametrize("heads,page,lengths,queries", [
    ((4, 2, 64), 16, [1, 2, 17, 64, 33], 1), ((12, 2, 128), 64, [1, 300, 63], 1), ((4, 2, 256), 32, [1, 40, 700], 1),
    ((12, 2, 128), 64, [11003], 1), ((12, 2, 128), 16, [2000], 1), ((8, 2, 256), 32, [7001, 5], 1), ((8, 2, 64), 16, [50, 3, 500], 4),
    ((24, 2, 128), 32, [70, 900], 2),
], ids=["64wide", "128wide", "256wide", "cut_11003", "cut_2000", "cut_256wide", "four_queries", "two_row_tiles"])
def test_an_infinite_value_stays_infinite(dev, f32, heads, page, lengths, queries):
    rng = np.random.default_rng([page, len(lengths), queries, heads[2]])
    Hq, H, D = heads
    table, pages = table_of(rng, lengths, page)
    pools = [random_pool(rng, "f16", pages, heads, page)[0] for _ in range(2)]
    offsets = np.asarray(lengths, dtype=np.int32) - 1
    finite, expected = pools[1].copy(), np.zeros((len(lengths), queries, H, D))
    # channel 0: the first position, 1: the last one, -infinity; 2: both signs; 3: one that weighs 2^-45 of the largest; 5 to 15: anywhere
    spots = []
    for b, n in enumerate(lengths):
        spots += [(b, 0, 0, 1), (b, n - 1, 1, -1), (b, 0, 2, 1), (b, n - 1, 2, -1), (b, n // 2, 3, 1)]
        spots += [(b, int(rng.integers(n)), 5 + i, 1) for i in range(11)]
    for b, t, c, sign in spots:
        p = table[b, t // page]
        pools[1][p, :, t % page, c] = sign * np.inf
        finite[p, :, t % page, c] = 0
    for b, n in enumerate(lengths):
        stored = orc.gather(pools[1], None, "f16", table[b, :-(-n // page)], n)
        for i in range(queries):
            seen = stored[:max(n - queries + 1 + i, 0)]
            with np.errstate(invalid="ignore"):
                expected[b, i] = np.where(np.isinf(seen), seen, 0).sum(axis=0)
    q = rng.standard_normal((len(lengths), queries, Hq, D), dtype=np.float32).astype(np.float16)
    q[..., 0] = 8
    for b, n in enumerate(lengths):                      # channel 0 of Q is 8: the score of position n // 2 falls by 31 and more
        if n > 8:
            pools[0][table[b, n // 2 // page], :, n // 2 % page, 0] = -8 * np.sqrt(D)
    cache, _, _ = make_cache(dev, metadata(heads), "f16", page, pools, (None, None))
    out = np.zeros(q.shape, dtype=np.float32 if f32 else np.float16)
    d_out = dev.put(out)
    cache.attend(dev.put(q), d_out, dev.put(table), dev.put(offsets), len(lengths), table.shape[1], query_tokens=queries, output_f32=f32)
    dev.rt.synchronize()
    out = dev.get(d_out, out)
    cache.cleanup()
    expected = np.repeat(expected, Hq // H, axis=2)
    special = expected != 0
    assert np.array_equal(out[special], expected[special].astype(out.dtype), equal_nan=True)
    ref, _, bound = orc.attention(q, pools[0], finite, None, None, "f16", table, offsets, 1.0 / np.sqrt(D))
    assert (np.abs(out - ref) <= tolerance(bound, ref, D, f32))[~special].all()
