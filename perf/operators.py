"""Paged key/value caches, as measurable cases: what a serving program does with them at every layer.

  append   new keys and values into the pages of their sequences, keys rotated to their positions on the way, queries
           rotated beside them; into 16-bit pages, or into 8-bit pages (e4m3 or int8) with one fp32 scale for every
           page and KV head.
  attend   queries of the newest position (or of the newest few, when drafted tokens are verified) over all cached
           positions of their sequences, read from such pages.

A cache is a pool of pages.  A page holds `page` positions of every KV head, [pages, kv_heads, page, head_dim] (layout
"heads") or [pages, page, kv_heads, head_dim] (layout "positions"); a block table int32 [batch, most pages] says which
pages are a sequence's, and kv_offsets int32 [batch] the position of its newest token (-1: a padded row of the batch).

The rules of 8-bit pages: a page's scale is its largest magnitude over 448 (e4m3) or 127 (int8); a value is stored as
round(x * (1 / scale)), ties to even.  Tokens that join a page that already has some only ever raise its scale, and then
the older tokens are stored anew as round(stored * (old scale / new scale)).  The first token of a page starts it afresh.
Keys are rotated in fp32 from fp16 tables, each product rounded, and rounded to fp16 before anything else.
"""
import math

import numpy as np
import torch

own = False


def _append(name, kind, batch, heads, page, new, past, rope=0, rotary=0, empty=0, layout="heads"):
    c = {"op": "append", "kind": kind, "batch": batch, "q_heads": heads[0], "kv_heads": heads[1], "head_dim": heads[2],
         "page": page, "new_min": new[0], "new_max": new[1], "past_min": past[0], "past_max": past[1], "rope": rope,
         "rotary": rotary, "empty": empty, "layout": layout}
    return dict(c, name=name) if name else c


def _attend(name, kind, batch, heads, page, ctx, queries=1, empty=0, outliers=False, layout="heads"):
    c = {"op": "attend", "kind": kind, "batch": batch, "q_heads": heads[0], "kv_heads": heads[1], "head_dim": heads[2],
         "page": page, "ctx_min": ctx[0], "ctx_max": ctx[1], "queries": queries, "empty": empty, "outliers": outliers,
         "layout": layout}
    return dict(c, name=name) if name else c


def listed():
    return [
        # the smallest append there is: the one new token of one sequence, 16-bit pages
        _append("append_f16_one_token", "f16", 1, (12, 2, 128), 16, (1, 1), (511, 511)),
        # a decode step of a serving batch with two padded rows, 8-bit pages, most of them partly filled
        _append("append_e4m3_step_64", "e4m3", 64, (32, 8, 64), 64, (1, 1), (100, 4000), empty=2),
        # ragged prompts, some continuing a cached prefix, a part of each 256-wide head rotated
        _append("append_f16_prompts", "f16", 8, (8, 2, 256), 32, (100, 4000), (0, 1000), rope=2, rotary=64),
        # one long document's prompt at once into 8-bit pages
        _append("append_e4m3_document", "e4m3", 1, (12, 2, 128), 64, (32768, 32768), (0, 0)),
        # chunks of prompts of a batch, odd lengths, adjacent pairs rotated, int8 pages
        _append("append_int8_chunks", "int8", 16, (32, 8, 64), 128, (1, 2048), (0, 8000), rope=1),
        # the smallest attention there is: one sequence of half a thousand positions
        _attend("attend_e4m3_512", "e4m3", 1, (12, 2, 128), 16, (512, 512)),
        # one long sequence
        _attend("attend_e4m3_32k", "e4m3", 1, (12, 2, 128), 64, (32768, 32768)),
        # a serving batch of ragged sequences of 8 x 64-wide heads
        _attend("attend_e4m3_ragged_64", "e4m3", 64, (32, 8, 64), 64, (1024, 16384)),
        # ragged long contexts of 256-wide heads with outliers in the caches
        _attend("attend_int8_ragged_256wide", "int8", 16, (8, 2, 256), 32, (2048, 65536), outliers=True),
        # drafted tokens verified: four queries a sequence
        _attend("attend_e4m3_verify_4", "e4m3", 8, (32, 8, 128), 32, (1000, 6000), queries=4),
        # one sequence of an odd length, 16-bit pages with all heads of a position side by side
        _attend("attend_f16_11003", "f16", 1, (12, 2, 128), 64, (11003, 11003), layout="positions"),
        # the serving batch with 16-bit pages of the smallest size and padded rows
        _attend("attend_f16_ragged_64", "f16", 64, (32, 8, 64), 16, (1024, 16384), empty=3),
    ]


_HEADS = [(12, 2, 128), (32, 8, 64), (8, 2, 256), (28, 4, 128), (32, 8, 128), (16, 2, 128), (32, 2, 128), (8, 8, 128),
          (16, 16, 64), (4, 1, 256)]
_MOST_BYTES = 5.0e8     # cache bytes that one drawn pass may read or write


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads = rng.choice(_HEADS)
    kind = rng.choice(["f16", "e4m3", "int8"])
    page = rng.choice([16, 32, 64, 128])
    layout = rng.choice(["heads", "heads", "positions"])
    position = 2 * heads[1] * heads[2] * (2 if kind == "f16" else 1)
    batch = _log(rng, 1, 128) if rng.random() < 0.7 else 1
    empty = rng.randint(1, 3) if batch > 8 and rng.random() < 0.5 else 0
    if rng.random() < 0.4:
        rope = rng.choice([0, 0, 1, 2, -1])
        rotary = rng.choice([32, 64]) if rope == 2 else 0
        if rng.random() < 0.5:
            new = (1, 1)
        else:
            most = _log(rng, 2, min(32768, max(2, int(3e8 / (batch * 2 * heads[2] * (2 * heads[0] + 3 * heads[1]))))))
            new = (max(1, int(most * rng.uniform(0.0, 1.0))), most)
        past = (0, _log(rng, 1, max(1, min(16384, int(_MOST_BYTES / (batch * position))))))
        return _append(None, kind, batch, heads, page, new, past, rope, rotary, empty, layout)
    longest = _log(rng, 64, max(64, min(524288 if batch == 1 else 65536, int(_MOST_BYTES / (batch * position)))))
    shortest = max(1, int(longest * rng.uniform(0.05, 1.0)))
    queries = rng.choice([1, 1, 1, 2, 3, 4, 8])
    return _attend(None, kind, batch, heads, page, (shortest, longest), queries, empty, rng.random() < 0.3, layout)


def _counts(case):
    """Cached positions and new tokens of each sequence, int64 [batch]; they depend on the case only.  Padded rows come last."""
    rng = np.random.default_rng([case["batch"], case["page"], case["head_dim"]])
    size = case["batch"]
    if case["op"] == "attend":
        past, new = rng.integers(case["ctx_min"], case["ctx_max"] + 1, size=size), np.zeros(size, dtype=np.int64)
    else:
        past = rng.integers(case["past_min"], case["past_max"] + 1, size=size)
        new = rng.integers(case["new_min"], case["new_max"] + 1, size=size)
    if case["empty"]:
        past[-case["empty"]:] = 0
        new[-case["empty"]:] = 0
    return past.astype(np.int64), new.astype(np.int64)


class _State:
    """What a serving program holds for one layer."""


_LARGEST = {"e4m3": 448.0, "int8": 127.0}


def _pool(case, pages, gen):
    """A pool with stale or cached values everywhere, and its scales (None for 16-bit pages)."""
    H, D, P = case["kv_heads"], case["head_dim"], case["page"]
    shape = (pages, H, P, D) if case["layout"] == "heads" else (pages, P, H, D)
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    if case.get("outliers"):
        for part in x.view(-1).split(1 << 26):
            part[torch.rand(part.shape, device="cuda", generator=gen) < 0.01] *= 20.0
    if case["layout"] == "positions":
        x = x.permute(0, 2, 1, 3)
    if case["kind"] == "f16":
        return x.to(torch.float16), None
    scale = x.abs().amax(dim=(2, 3)) / _LARGEST[case["kind"]]
    x = x / scale[:, :, None, None]
    x = x.to(torch.float8_e4m3fn) if case["kind"] == "e4m3" else torch.round(x).to(torch.int8)
    return x, scale.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = _State()
    s.case = case
    B, P, D = case["batch"], case["page"], case["head_dim"]
    past, new = _counts(case)
    held = past + new
    used = -(-held // P)
    s.max_pages = int(max(1, used.max())) + 1
    s.pages = int(used.sum()) + 1 + B // 4
    order = torch.randperm(s.pages, generator=gen, device="cuda").to(torch.int32)
    live = torch.arange(s.max_pages)[None] < torch.from_numpy(used)[:, None]
    table = torch.full((B, s.max_pages), -1, dtype=torch.int32, device="cuda")
    table[live.cuda()] = order[:int(used.sum())]
    s.block_table = table
    s.kv_offsets = torch.from_numpy((held - 1).astype(np.int32)).cuda()
    s.k_pool, s.k_scale = _pool(case, s.pages, gen)
    s.v_pool, s.v_scale = _pool(case, s.pages, gen)
    s.stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "attend":
        shape = (B, case["queries"], case["q_heads"], D)
        s.q = torch.randn(shape, generator=gen, device="cuda").to(torch.float16)
        s.output = torch.zeros(shape, dtype=torch.float16, device="cuda")
        return s
    one_each = case["new_max"] == 1
    rows = B if one_each else int(new.sum())
    s.token_starts = None if one_each else torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
    s.k, s.v, s.q = (torch.randn((rows, h, D), generator=gen, device="cuda").to(torch.float16)
                     for h in (case["kv_heads"], case["kv_heads"], case["q_heads"]))
    s.q_out = torch.zeros_like(s.q)
    s.cos = s.sin = None
    if case["rope"] >= 0:
        width = case["rotary"] if case["rope"] == 2 else D
        at = torch.arange(s.max_pages * P, device="cuda", dtype=torch.float64)
        angle = at[:, None] * (1e6 ** (-torch.arange(width // 2, device="cuda", dtype=torch.float64) * 2 / width))[None]
        s.cos, s.sin = (torch.cat([f(angle), f(angle)], dim=1).to(torch.float16) for f in (torch.cos, torch.sin))
    return s


# ---- the framework's calls -------------------------------------------------------------------------------------------
_program = {}


def _cache(s):
    """The program's runtime, its scratch, and the handle of this layer's cache."""
    from vte_b200.bridge import CudaRuntime
    from vte_b200.core import PagedKVCache
    if not _program:
        _program["rt"] = rt = CudaRuntime(device_index=0)
        rt.initialize()
    rt, c = _program["rt"], s.case
    meta = {"attention.head_count": c["q_heads"], "attention.head_count_kv": c["kv_heads"], "attention.key_length": c["head_dim"]}
    if c["op"] == "append" and c["rope"] >= 0:
        meta.update(rope_type=c["rope"], rotary_dim=c["rotary"])
    need = PagedKVCache.workspace_bytes(rt, meta, c["batch"], c.get("queries", 1))
    if _program.get("bytes", 0) < need:
        _program.update(bytes=need, scratch=torch.zeros(need, dtype=torch.uint8, device="cuda"))
    s.cache = PagedKVCache(rt, meta, s.pages, c["page"], c["kind"], k_pool=s.k_pool.data_ptr(), v_pool=s.v_pool.data_ptr(),
                           k_scale=s.k_scale.data_ptr() if s.k_scale is not None else 0,
                           v_scale=s.v_scale.data_ptr() if s.v_scale is not None else 0,
                           strides=s.k_pool.stride()[:1] + s.k_pool.stride()[2:0:-1])
    if c["op"] == "append" and c["rope"] >= 0:
        s.cache.set_rope(s.cos.data_ptr(), s.sin.data_ptr(), s.cos.shape[0])
    return s.cache


def _call(s):
    cache = getattr(s, "cache", None) or _cache(s)
    c = s.case
    if c["op"] == "attend":
        cache.attend(s.q.data_ptr(), s.output.data_ptr(), s.block_table.data_ptr(), s.kv_offsets.data_ptr(), c["batch"],
                     s.max_pages, query_tokens=c["queries"], workspace=_program["scratch"].data_ptr(),
                     workspace_bytes=_program["bytes"], stream=s.stream)
        return s.output
    cache.append(s.k.data_ptr(), s.v.data_ptr(), s.block_table.data_ptr(), s.kv_offsets.data_ptr(), c["batch"], s.max_pages,
                 total_tokens=s.k.shape[0], token_starts=s.token_starts.data_ptr() if s.token_starts is not None else 0,
                 q=s.q.data_ptr(), q_out=s.q_out.data_ptr(), stream=s.stream)
    return _appended(s)


def _appended(s):
    out = {"k": s.k_pool, "v": s.v_pool, "q": s.q_out}
    if s.k_scale is not None:
        out.update(k_scale=s.k_scale, v_scale=s.v_scale)
    return out


def run(s):
    if own:
        return _call(s)
    return _plain_attend(s) if s.case["op"] == "attend" else _plain_append(s)


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _bits(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _values(x, kind):
    return (x.view(torch.float8_e4m3fn) if kind == "e4m3" else x).float()


def _plain_attend(s):
    """softmax(q k / sqrt(D)) v in fp32 over the pages that hold positions, joined by sequence."""
    c = s.case
    B, Q, Hq, D, P, H = c["batch"], c["queries"], c["q_heads"], c["head_dim"], c["page"], c["kv_heads"]
    G = Hq // H
    length = s.kv_offsets.long() + 1
    seq, nth = (torch.arange(s.max_pages, device="cuda")[None] * P < length[:, None]).nonzero(as_tuple=True)
    page = s.block_table[seq, nth].long()
    k, v = (_values(_bits(x)[page], c["kind"]) for x in (s.k_pool, s.v_pool))                  # [n, H, P, D]
    if s.k_scale is not None:
        k, v = k * s.k_scale[page][:, :, None, None], v * s.v_scale[page][:, :, None, None]
    q = s.q.float().reshape(B, Q, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, Q * G, D)
    score = (q[seq] @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).reshape(-1, H, Q, G, P)
    at = nth[:, None] * P + torch.arange(P, device="cuda")[None]                               # [n, P]
    last = length[seq][:, None] - Q + torch.arange(Q, device="cuda")[None]                     # newest position of query i
    seen = at[:, None, :] <= last[:, :, None]                                                  # [n, Q, P]
    score = torch.where(seen[:, None, :, None, :], score, -math.inf).reshape(-1, H, Q * G, P)
    top = torch.full((B, H, Q * G), -math.inf, device="cuda").index_reduce_(0, seq, score.amax(dim=-1), "amax")
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top)[seq][..., None])
    total = torch.zeros((B, H, Q * G), device="cuda").index_add_(0, seq, p.sum(dim=-1))
    v = torch.where((at < length[seq][:, None])[:, None, :, None], v, 0.0)
    out = torch.zeros((B, H, Q * G, D), device="cuda").index_add_(0, seq, p @ v)
    out = out / torch.where(total == 0, 1.0, total)[..., None]
    s.output.copy_(out.reshape(B, H, Q, G, D).permute(0, 2, 1, 3, 4).reshape(B, Q, Hq, D))
    return s.output


def _plain_rotate(x, cos, sin, rope, rotary):
    """fp16 rows [tokens, heads, D] rotated in fp32 with table rows [tokens, width], rounded to fp16."""
    if rope < 0:
        return x
    f, cos, sin = x.float(), cos.float()[:, None], sin.float()[:, None]
    if rope == 1:
        half = x.shape[-1] // 2
        a, b, cos, sin = f[..., 0::2], f[..., 1::2], cos[..., :half], sin[..., :half]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2).to(torch.float16)
    width = rotary if rope == 2 else x.shape[-1]
    half = width // 2
    a, b, cos, sin = f[..., :half], f[..., half:width], cos[..., :half], sin[..., :half]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, f[..., width:]], dim=-1).to(torch.float16)


def _plain_quantise(x, kind):
    return x.to(torch.float8_e4m3fn).view(torch.uint8) if kind == "e4m3" else torch.round(x).clamp(-127, 127).to(torch.int8)


def _plain_store(pool, scale, x, page, slot, kind):
    """Rows x [tokens, heads, D] into pool[page, :, slot]."""
    if scale is None:
        pool[page, :, slot] = x
        return
    bits, x, P = _bits(pool), x.float(), pool.shape[2]
    need = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(dim=-1), "amax")
    need = need / torch.full_like(need, _LARGEST[kind])
    touched, fresh = (torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda") for _ in range(2))
    touched[page] = True
    fresh[page[slot == 0]] = True
    old = torch.where(fresh[:, None], 0.0, scale)
    now = torch.where(touched[:, None], torch.maximum(old, need), scale)
    # the older tokens of the pages whose scale grows; below the first new slot of the page
    first = torch.full((scale.shape[0],), P, dtype=torch.int64, device="cuda").index_reduce_(0, page, slot, "amin")
    some = (touched & ~fresh).nonzero()[:, 0]
    factor = (old[some] / torch.where(now[some] > 0, now[some], 1.0))[:, :, None, None]
    again = (now[some] > old[some])[:, :, None, None] & (torch.arange(P, device="cuda")[None] < first[some][:, None])[:, None, :, None]
    bits[some] = torch.where(again, _plain_quantise(_values(bits[some], kind) * factor, kind), bits[some])
    scale.copy_(now)
    inverse = torch.where(now > 0, torch.ones_like(now) / now, 0.0)
    bits[page, :, slot] = _plain_quantise(x * inverse[page][:, :, None], kind)


def _plain_append(s):
    c = s.case
    B, P = c["batch"], c["page"]
    end = s.kv_offsets.long()
    if s.token_starts is None:
        seq, row = torch.arange(B, device="cuda"), torch.arange(B, device="cuda")
        at = end.clone()
    else:
        starts = s.token_starts.long()
        seq = torch.repeat_interleave(torch.arange(B, device="cuda"), starts[1:] - starts[:-1])
        row = torch.arange(seq.shape[0], device="cuda")
        at = end[seq] + 1 - (starts[seq + 1] - row)
    kept = at >= 0
    seq, row, at = seq[kept], row[kept], at[kept]
    page, slot = s.block_table[seq, at // P].long(), at % P
    cos, sin = (None, None) if s.cos is None else (s.cos[at], s.sin[at])
    s.q_out[row] = _plain_rotate(s.q[row], cos, sin, c["rope"], c["rotary"])
    _plain_store(s.k_pool, s.k_scale, _plain_rotate(s.k[row], cos, sin, c["rope"], c["rotary"]), page, slot, c["kind"])
    _plain_store(s.v_pool, s.v_scale, s.v[row], page, slot, c["kind"])
    return _appended(s)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attend(s) if case["op"] == "attend" else _exact_append(s)


def _exact_attend(s):
    c = s.case
    H, G, D, P = c["kv_heads"], c["q_heads"] // c["kv_heads"], c["head_dim"], c["page"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    ends, tables = s.kv_offsets.tolist(), s.block_table.tolist()
    for b, end in enumerate(ends):
        if end < 0:
            continue
        pages = torch.tensor(tables[b][:end // P + 1], device="cuda")
        for h in range(H):
            rows = []
            for pool, scale in ((s.k_pool, s.k_scale), (s.v_pool, s.v_scale)):
                x = pool[:, h].view(torch.uint8)[pages].view(pool.dtype) if c["kind"] == "e4m3" else pool[:, h][pages]
                x = x.double()
                if scale is not None:
                    x = x * scale[pages, h].double()[:, None, None]
                rows.append(x.reshape(-1, D)[:end + 1])
            for i in range(c["queries"]):
                n = end + 1 - (c["queries"] - 1 - i)
                if n > 0:
                    z = s.q[b, i, h * G:(h + 1) * G].double() @ rows[0][:n].T / math.sqrt(D)
                    z = torch.exp(z - z.max(dim=-1, keepdim=True).values)
                    out[b, i, h * G:(h + 1) * G] = (z @ rows[1][:n]) / z.sum(dim=-1, keepdim=True)
    return out


def _exact_append(s):
    c = s.case
    kind, P = c["kind"], c["page"]
    past, new = _counts(c)
    pools = [x.double() for x in (s.k_pool, s.v_pool)]
    scales = [None if x is None else x.double() for x in (s.k_scale, s.v_scale)]
    queries = s.q_out.double()
    table, begin = s.block_table.tolist(), 0
    for b in range(c["batch"]):
        n, done, row = int(new[b]), int(past[b]), begin
        begin += 1 if s.token_starts is None else n
        if n == 0:
            continue
        at = torch.arange(done, done + n, device="cuda")
        rows = [x[row:row + n].double() for x in (s.k, s.v, s.q)]
        if c["rope"] >= 0:
            cos, sin = s.cos[at].double()[:, None], s.sin[at].double()[:, None]
            width = c["rotary"] if c["rope"] == 2 else c["head_dim"]
            half = width // 2
            cos, sin = cos[..., :half], sin[..., :half]
            for i in (0, 2):
                x = rows[i].clone()
                one, two = (slice(0, width, 2), slice(1, width, 2)) if c["rope"] == 1 else (slice(0, half), slice(half, width))
                rows[i][..., one] = x[..., one] * cos - x[..., two] * sin
                rows[i][..., two] = x[..., one] * sin + x[..., two] * cos
        queries[row:row + n] = rows[2]
        for x, pool, scale in zip(rows, pools, scales):
            if scale is None:
                pages = torch.tensor([table[b][int(i) // P] for i in at.tolist()], device="cuda")
                pool[pages, :, at % P] = x
                continue
            x = x.to(torch.float16).double()        # rounded to fp16 before it is quantised: a part of the definition
            for first in range(done // P * P, done + n, P):
                page, lo, hi = table[b][first // P], max(first, done), min(first + P, done + n)
                here = x[lo - done:hi - done].transpose(0, 1)                      # [heads, tokens, D]
                old = scale[page].clone() if lo > first else torch.zeros_like(scale[page])
                now = torch.maximum(old, here.abs().amax(dim=(1, 2)) / _LARGEST[kind])
                safe = torch.where(now > 0, now, 1.0)
                pool[page, :, :lo - first] *= (old / safe)[:, None, None]
                pool[page, :, lo - first:hi - first] = here / safe[:, None, None]
                scale[page] = now
    out = {"k": pools[0], "v": pools[1], "q": queries}
    if kind == "int8":
        out.update(k=None, v=None)                  # whole numbers next to a tie have no value in 64 bits
    if scales[0] is not None:
        out.update(k_scale=scales[0], v_scale=scales[1])
    return out


def work(case):
    """Cached rows, scales and table entries that hold positions once; new rows, queries and rotation tables in, results out."""
    past, new = _counts(case)
    B, H, Hq, D, P = case["batch"], case["kv_heads"], case["q_heads"], case["head_dim"], case["page"]
    size = 2 if case["kind"] == "f16" else 1
    if case["op"] == "attend":
        n, pages = int(past.sum()), int((-(-past // P)).sum())
        scales = 0 if case["kind"] == "f16" else 2 * 4 * H * pages
        seen = sum(int(np.maximum(past - i, 0).sum()) for i in range(case["queries"]))
        return {"bytes": 2 * n * H * D * size + scales + 4 * pages + 4 * B + 2 * 2 * B * case["queries"] * Hq * D,
                "flops": 4 * seen * Hq * D}
    n = int(new.sum())
    pages = int(((past + new - 1) // P - past // P + 1)[new > 0].sum())
    scales = 0 if case["kind"] == "f16" else 2 * 4 * H * pages
    width = 0 if case["rope"] < 0 else case["rotary"] if case["rope"] == 2 else D
    return {"bytes": 2 * n * H * D * (2 + size) + 2 * 2 * n * Hq * D + 2 * n * width + 2 * scales + 4 * pages + 4 * B,
            "flops": 3 * n * (H + Hq) * (width or 1)}
