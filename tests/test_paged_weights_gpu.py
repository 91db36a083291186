"""Paged attention where the weights of a row are of very different size: a few positions that outweigh all others, as the first
tokens of a text do, and pages whose scales differ.  What the light positions add up to is held to the definition in 64 bits."""
import numpy as np
import pytest

from oracle import paged_oracle as orc
from tests.paged_case import Device, make_cache, metadata, table_of, tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(cuda_runtime):
    d = Device(cuda_runtime)
    yield d
    cuda_runtime.synchronize()
    d.free()


def attend(dev, kind, heads, page, table, lengths, pools, scales, q, f32):
    cache, _, _ = make_cache(dev, metadata(heads), kind, page, pools, scales)
    offsets = (np.asarray(lengths) - 1).astype(np.int32)
    out = np.full(q.shape, np.nan, dtype=np.float32 if f32 else np.float16)
    lse = np.full(q.shape[:3], np.nan, dtype=np.float32)
    d_out, d_lse = dev.put(out), dev.put(lse)
    try:
        cache.attend(dev.put(q), d_out, dev.put(table), dev.put(offsets), len(lengths), table.shape[1], query_tokens=q.shape[1],
                     output_f32=f32, lse=d_lse)
        dev.rt.synchronize()
    finally:
        cache.cleanup()
    return dev.get(d_out, out), dev.get(d_lse, lse)


def definition(kind, heads, table, lengths, pools, scales, q):
    return orc.attention(q, *pools, *scales, kind, table, np.asarray(lengths) - 1, 1.0 / np.sqrt(heads[2]))


def allowed(bound, ref, f32):
    """`tolerance` for scores that are one product each (8 roundings instead of D + 8), with weights that lose nothing above
    2^-39 of the largest (half a step of fp16 below its normal range, 2^-25, or a whole one, under a factor of 2^15), and up
    to 128 additions to a warp's sums on the tensor cores, each off by 2^-23 at most."""
    mean, reach, floor = bound
    return tolerance((mean, reach, floor * 2.0 ** -14), ref, 0, f32) + 2.0 ** -16 * mean


def stored(x, kind):
    """(stored values [pages, heads, page, D], scales or None) of fp32 values."""
    if kind == "f16":
        return x.astype(np.float16), None
    scale = np.abs(x).max(axis=(2, 3)).astype(np.float32) / orc.LARGEST[kind]
    return orc.narrow(x / np.where(scale > 0, scale, 1)[:, :, None, None], kind), scale


SINKS = {"64x17": ((4, 2, 64), 64, 17.0, 1500, False), "64x17_pages_of_16": ((4, 2, 64), 16, 17.0, 1500, True),
         "64x14": ((4, 2, 64), 64, 14.0, 1500, False), "128x16": ((6, 2, 128), 32, 16.0, 1300, True),
         "256x17": ((4, 2, 256), 128, 17.0, 1000, False), "64x10": ((4, 2, 64), 64, 10.0, 1500, False),
         "64x16_long": ((2, 2, 64), 128, 16.0, 32000, False)}


@pytest.mark.parametrize("kind,case", [(kind, c) for c in SINKS for kind in ("f16", "e4m3", "int8") if not c.endswith("long") or kind == "e4m3"])
def test_a_few_positions_outweigh_all_others(dev, kind, case):
    """Eight positions a sequence score `gap` nats above the mean of the others and have values of zero, so that the output is what the
    others add up to.  `loud`: beside each of them a value of 1000, which gives its page a V scale far above its neighbours'."""
    heads, page, gap, most, loud = SINKS[case]
    rng = np.random.default_rng([int(gap), page, heads[2]])
    Hq, H, D = heads
    lengths = rng.integers(most * 3 // 4, most, size=80 if most < 10000 else 8)
    table, pages = table_of(rng, lengths, page)
    k = np.zeros((pages, H, page, D), dtype=np.float32)
    k[..., 0] = rng.standard_normal((pages, H, page), dtype=np.float32)
    v = 1 + 0.5 * rng.standard_normal((pages, H, page, D), dtype=np.float32)
    for b, n in enumerate(lengths):
        for t in rng.choice(int(n) // page * page, size=8, replace=False):
            p = table[b, t // page]
            k[p, :, t % page, 0] = gap
            v[p, :, t % page] = 0
            if loud:
                v[p, :, (t + 1) % page] *= 1000 * (k[p, :, (t + 1) % page, :1] < gap / 2)
    pools, scales = zip(*(stored(x, kind) for x in (k, v)))
    q = np.zeros((len(lengths), 1, Hq, D), dtype=np.float16)
    q[..., 0] = np.sqrt(D) * (1 - 0.01 * np.arange(Hq))
    ref, ref_lse, bound = definition(kind, heads, table, lengths, pools, scales, q)
    for f32 in (False, True):
        out, lse = attend(dev, kind, heads, page, table, lengths, pools, scales, q, f32)
        off, limit = np.abs(out - ref), allowed(bound, ref, f32)
        assert (off <= limit).all(), (f32, np.unravel_index(np.argmax(off - limit), off.shape), (off / limit).max(), np.linalg.norm(off) / np.linalg.norm(ref))
        # the logarithm's own two roundings, a sum of weights off by 8 roundings of `reach` and 2^-20, and its additions
        assert (np.abs(lse - ref_lse) <= 2.0 ** -20 * bound[1] + 2.0 ** -16 + 2.0 ** -22 * np.abs(ref_lse)).all()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("D,page", [(64, 64), (64, 128), (128, 32), (256, 16), (64, 16)])
def test_v_scales_of_all_kinds_in_units_of_one_page(dev, kind, D, page):
    """Zero, negative, huge and tiny V scales beside ordinary ones, from page to page of a sequence: the unit of the sums
    changes between the quick way and the careful one."""
    rng = np.random.default_rng([D, page])
    heads = Hq, H, _ = (4, 2, D)
    palettes = [[0, 1, -1], [1e31, -1e31, 1e28], [2.0 ** -110, 0, 2.0 ** -105], [1, 1e-13, 0], [1, 1e31, 0, -1, 1e-30], [-1, -2], [0], [1, 1, 1, 0],
                [2.0 ** 101, 2.0 ** 99, 2.0 ** 98]]
    lengths = rng.integers(1, 1500, size=81)
    table, pages = table_of(rng, lengths, page)
    pools, scales = [], []
    for _ in range(2):
        x, s = stored(rng.standard_normal((pages, H, page, D), dtype=np.float32), kind)
        pools.append(x)
        scales.append(s)
    for b, n in enumerate(lengths):
        for p in table[b, :-(-int(n) // page)]:
            scales[1][p] = rng.choice(np.array(palettes[b % len(palettes)], dtype=np.float32), size=H)
    q = rng.standard_normal((len(lengths), 1, Hq, D), dtype=np.float32).astype(np.float16)
    out, _ = attend(dev, kind, heads, page, table, lengths, pools, scales, q, True)
    ref, _, (mean, reach, floor) = definition(kind, heads, table, lengths, pools, scales, q)
    most = tolerance((mean, reach, floor * 2.0 ** -14), ref, D, True) + 2.0 ** -16 * mean
    off = np.abs(out - ref)
    assert (off <= most).all(), (np.unravel_index(np.argmax(off - most), off.shape), (off / np.where(most > 0, most, 1)).max())
