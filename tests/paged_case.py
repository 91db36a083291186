"""A paged cache on the device with its numpy image, for the tests of paged caches."""
import ctypes

import numpy as np

from oracle import paged_oracle as orc
from vte_b200.core import PagedKVCache


class Device:
    """Arrays on the device for the length of a test."""

    def __init__(self, rt):
        self.rt, self.held = rt, []

    def put(self, x):
        x = np.ascontiguousarray(x)
        p = self.rt.safe_malloc(max(x.nbytes, 16), "output of a test")
        self.held.append(p)
        if x.nbytes:
            self.rt.safe_memcpy_host_to_device(p, x.reshape(-1).view(np.uint8))
        return p.value

    def get(self, ptr, like):
        out = np.empty(like.shape, dtype=like.dtype)
        self.rt.safe_memcpy_device_to_host(out.reshape(-1).view(np.uint8), ctypes.c_void_p(ptr), "output of a test")
        return out

    def free(self):
        for p in self.held:
            self.rt.safe_free(p)
        self.held.clear()


def metadata(heads, rope_type=0, rotary_dim=0):
    return {"attention.head_count": heads[0], "attention.head_count_kv": heads[1], "attention.key_length": heads[2],
            "rope_type": rope_type, "rotary_dim": rotary_dim or heads[2]}


def random_pool(rng, kind, pages, heads, page, sigma=1.0):
    """(stored [pages, heads, page, D], scales or None)."""
    x = (rng.standard_normal((pages, heads[1], page, heads[2]), dtype=np.float32) * np.float32(sigma))
    x *= np.exp(rng.uniform(-1.5, 1.5, size=(pages, heads[1], 1, 1))).astype(np.float32)      # pages of different size
    if kind == "f16":
        return x.astype(np.float16), None
    scale = np.abs(x).max(axis=(2, 3)).astype(np.float32) / orc.LARGEST[kind]
    return orc.narrow(x * (np.float32(1) / scale)[:, :, None, None], kind), scale


def poison(stored, scale, kind, unseen, rng):
    """What nothing may read: rows `unseen` [pages, page] of every head, and the scales of pages that are unseen throughout."""
    rows = np.broadcast_to(unseen[:, None, :], stored.shape[:3])
    if kind == "f16":
        bad = np.array([np.nan, np.inf, -np.inf, 65504.0], dtype=np.float16)
        stored[rows] = rng.choice(bad, size=(int(rows.sum()), stored.shape[3]))
    elif kind == "e4m3":
        stored[rows] = rng.choice(np.array([0x7f, 0xff, 0x7e], dtype=np.uint8), size=(int(rows.sum()), stored.shape[3]))
    else:
        stored[rows] = -128
    if scale is not None:
        scale[unseen.all(axis=1)] = np.nan


def table_of(rng, lengths, page, extra=0, spare=3):
    """(block table with -7 behind each sequence's pages, number of pages), pages in random order."""
    used = [-(-max(int(n), 0) // page) for n in lengths]
    pages = sum(used) + spare
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((len(lengths), max(1, max(used)) + extra), -7, dtype=np.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def unseen_rows(table, lengths, pages, page):
    unseen = np.ones((pages, page), dtype=bool)
    for b, n in enumerate(lengths):
        for i in range(-(-max(int(n), 0) // page)):
            unseen[table[b, i], :min(page, int(n) - i * page)] = False
    return unseen


def put_pool(dev, stored, layout):
    """(address, strides) of a pool in one of the two orders."""
    pages, H, P, D = stored.shape
    if layout == "heads":
        return dev.put(stored), (H * P * D, D, P * D)
    return dev.put(stored.transpose(0, 2, 1, 3)), (P * H * D, H * D, D)


def get_pool(dev, ptr, stored, layout):
    if layout == "heads":
        return dev.get(ptr, stored)
    pages, H, P, D = stored.shape
    return dev.get(ptr, np.empty((pages, P, H, D), dtype=stored.dtype)).transpose(0, 2, 1, 3)


def make_cache(dev, meta, kind, page, pools, scales, layout="heads"):
    ptrs = [put_pool(dev, x, layout) for x in pools]
    sc = [dev.put(s) if s is not None else 0 for s in scales]
    cache = PagedKVCache(dev.rt, meta, pools[0].shape[0], page, kind, k_pool=ptrs[0][0], v_pool=ptrs[1][0], k_scale=sc[0],
                         v_scale=sc[1], strides=ptrs[0][1])
    return cache, [p for p, _ in ptrs], sc


def tolerance(bound, out, D, f32):
    """How far an output may be off, element by element; the roundings of the kernel counted:
    a weight: P to fp16 (2^-11; as two parts 2^-21), exp2 and the products with scales (2^-20), and the score's own error, which
    multiplies it: D + 8 fp32 roundings of sums up to `reach`.  It reaches the row twice, in the sum of weights and of values.
    Weights below fp16's normal range are off by half its smallest step, 2^-25, relative to the largest weight and V scale.
    The output's own rounding: 2^-11, or 2^-25 below the normal range of fp16."""
    mean, reach, floor = bound
    weight = (2.0 ** -21 if f32 else 2.0 ** -11) + 2.0 ** -20 + (D + 8) * 2.0 ** -24 * 2 * reach
    return 2 * weight[..., None] * mean + 2.0 ** -25 * floor + (2.0 ** -23 if f32 else 2.0 ** -11) * np.abs(out) + (0 if f32 else 2.0 ** -25)
