"""Paged key/value caches in numpy: 8-bit formats, the append with its rotation and scales, and the attention in 64 bits.

The append is restated with the arithmetic that include/vteb200.h gives it (fp32, one rounding an operation), so that the
kernels can be held to its bits; the attention is the definition in 64 bits."""
import numpy as np

LARGEST = {"e4m3": np.float32(448.0), "int8": np.float32(127.0)}


def _e4m3_values():
    v = np.empty(256, dtype=np.float32)
    for i in range(256):
        e, f = (i >> 3) & 15, i & 7
        x = np.nan if (i & 127) == 127 else (f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7))
        v[i] = -x if i & 128 else x
    return v


E4M3 = _e4m3_values()
_GRID = E4M3[:127].astype(np.float64)          # 0 .. 448, ascending


def to_e4m3(x):
    """fp32 to e4m3 bytes: nearest, ties to the even byte, saturating; NaN stays NaN."""
    x = np.asarray(x, dtype=np.float32)
    a = np.minimum(np.abs(x).astype(np.float64), 448.0)
    hi = np.clip(np.searchsorted(_GRID, np.where(np.isnan(a), 0, a)), 1, 126)
    lo = hi - 1
    down, up = a - _GRID[lo], _GRID[hi] - a
    byte = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    byte = np.where(np.isnan(x), 127, byte)
    return (byte | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def widen(stored, kind):
    """Stored 8-bit values as fp32 (before their scale)."""
    return E4M3[stored.view(np.uint8)] if kind == "e4m3" else stored.astype(np.float32)


def narrow(x, kind):
    if kind == "e4m3":
        return to_e4m3(x)
    with np.errstate(invalid="ignore"):
        return np.where(np.isnan(x), 0, np.clip(np.rint(x), -128, 127)).astype(np.int8)


def rotate(x, pos, cos, sin, rope_type, rotary_dim):
    """fp16 rows [tokens, heads, D] at positions `pos`, in fp32, rounded to fp16."""
    if rope_type < 0:
        return x
    D = x.shape[-1]
    width = rotary_dim if rope_type == 2 else D
    half = width // 2
    f = x.astype(np.float32)
    c, s = (t[pos][:, None, :half].astype(np.float32) for t in (cos, sin))
    out = f.copy()
    one, two = (slice(0, D, 2), slice(1, D, 2)) if rope_type == 1 else (slice(0, half), slice(half, width))
    out[..., one] = f[..., one] * c - f[..., two] * s
    out[..., two] = f[..., one] * s + f[..., two] * c
    return out.astype(np.float16)


def append(pools, scales, kind, new, block_table, kv_offsets, token_starts, page):
    """Appends rotated rows new = (k, v) [tokens, heads, D] in place.  pools [pages, heads, page, D], scales [pages, heads]."""
    f32 = np.float32
    for b, end in enumerate(kv_offsets):
        first, count = int(token_starts[b]), int(token_starts[b + 1] - token_starts[b])
        begin = int(end) - count + 1
        for nth in range(max(begin, 0) // page, int(end) // page + 1) if end >= 0 and count else ():
            lo, hi = max(begin, 0, nth * page), min(int(end), nth * page + page - 1)
            p, slot = int(block_table[b, nth]), lo % page
            for pool, scale, rows in zip(pools, scales, new):
                x = rows[first + lo - begin:first + hi - begin + 1].transpose(1, 0, 2)          # [heads, tokens, D]
                if kind == "f16":
                    pool[p, :, slot:slot + hi - lo + 1] = x
                    continue
                for h in range(x.shape[0]):
                    old = scale[p, h] if slot else f32(0)
                    amax = np.abs(x[h]).max().astype(f32)               # NaN where one is
                    need = amax / LARGEST[kind] if np.isfinite(amax) else f32(np.nan)
                    now = f32(np.nan) if np.isnan(need) or np.isnan(old) else max(old, need) if old >= 0 else min(old, -need)
                    inv = f32(0) if now == 0 or (need == 0 and not np.isnan(now)) else f32(1) / now
                    with np.errstate(invalid="ignore"):
                        if slot and abs(now) > abs(old):
                            pool[p, h, :slot] = narrow(widen(pool[p, h, :slot], kind) * (old / now), kind)
                        pool[p, h, slot:slot + hi - lo + 1] = narrow(x[h].astype(f32) * inv, kind)
                    scale[p, h] = now


def gather(pool, scale, kind, pages, n):
    """The first n rows of a sequence's pages, [n, heads, D] in 64 bits."""
    x = pool[pages]
    x = x.astype(np.float64) if kind == "f16" else widen(x, kind).astype(np.float64) * scale[pages][:, :, None, None].astype(np.float64)
    return x.transpose(0, 2, 1, 3).reshape(-1, pool.shape[1], pool.shape[3])[:n]


def attention(q, k_pool, v_pool, k_scale, v_scale, kind, block_table, kv_offsets, scale):
    """q [batch, queries, heads, D] -> (output, lse, bound) in 64 bits.  `bound` are three arrays like the output from which a
    test derives its tolerance: sum p |v| / sum p, the largest sum |q k| scale of a row, and sum |v| / sum exp(s - max) with
    every |v| taken under the row's largest V scale."""
    B, Q, Hq, D = q.shape
    H, P = k_pool.shape[1], k_pool.shape[2]
    G = Hq // H
    out, lse = np.zeros(q.shape), np.full((B, Q, Hq), -np.inf)
    mean, reach, floor = np.zeros(q.shape), np.zeros((B, Q, Hq)), np.zeros(q.shape)
    for b in range(B):
        n = int(kv_offsets[b]) + 1
        if n <= 0:
            continue
        pages = block_table[b, :-(-n // P)]
        k, v = gather(k_pool, k_scale, kind, pages, n), gather(v_pool, v_scale, kind, pages, n)
        stored = v_pool[pages].astype(np.float64) if kind == "f16" else widen(v_pool[pages], kind).astype(np.float64)
        stored = np.abs(stored.transpose(0, 2, 1, 3).reshape(-1, H, D)[:n])
        for i in range(Q):
            m = n - (Q - 1 - i)
            if m <= 0:
                continue
            for h in range(Hq):
                kv = h // G
                s = (k[:m, kv] @ q[b, i, h].astype(np.float64)) * scale
                top = s.max()
                p = np.exp(s - top)
                out[b, i, h] = p @ v[:m, kv] / p.sum()
                lse[b, i, h] = top + np.log(p.sum())
                mean[b, i, h] = p @ np.abs(v[:m, kv]) / p.sum()
                reach[b, i, h] = (np.abs(k[:m, kv]) @ np.abs(q[b, i, h].astype(np.float64))).max() * abs(scale)
                largest = 1.0 if kind == "f16" else np.abs(v_scale[pages[:-(-m // P)], kv]).max()
                floor[b, i, h] = stored[:m, kv].sum(axis=0) * largest / p.sum()
    return out, lse, (mean, reach, floor)
