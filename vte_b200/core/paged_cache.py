"""`PagedKVCache`: one layer's key/value cache as a pool of pages, the append that fills it and the attention that reads it.

The contiguous caches of the reference give every sequence room for the longest one (vte/compiler/qwen_mapper.py:321-351);
a server of many ragged sequences hands out pages instead.  Pages hold fp16 values, or 8-bit ones (e4m3 or int8) with an
fp32 scale for every page and KV head, which halves what a decode step has to read.  The rules of the scales, the layout
and what the kernels report are in include/vteb200.h.

A decode step of a layer is two launches, on the runtime's stream or on the caller's:

    cache.append(k, v, block_table, kv_offsets, batch, max_pages, q=q, q_out=q)     # rotates q and k, stores k and v
    cache.attend(q, output, block_table, kv_offsets, batch, max_pages)

Arguments are device addresses (integers, ctypes pointers or `MemoryBlock`s).  Both calls may be captured.  Layers that run
one behind the other may share a workspace (`workspace=`); calls that overlap on the GPU may not.
"""
from __future__ import annotations

import ctypes
import math

from ..bridge.cuda_runtime import LAUNCH_PROGRAMMATIC, PagedAppend, PagedAttention, PagedCache, _ptr_value
from ..bridge.errors import CudaSafetyError
from ..bridge.memory import MemoryRegion

CACHE_TYPES = {"f16": 0, "e4m3": 1, "int8": 2}       # VTEB_PAGED_* (include/vteb200.h)
MAX_QUERY_TOKENS = 16


def _heads(metadata):
    return (int(metadata.get('attention.head_count', 12)), int(metadata.get('attention.head_count_kv', 2)),
            int(metadata.get('attention.key_length', 128)))


class PagedKVCache:
    """`k_pool`, `v_pool` (and `k_scale`, `v_scale`): the caller's memory, with `strides` (page, token, head, in values);
    without pools they are allocated, from `allocator` where one is given, with the positions of a head side by side."""

    def __init__(self, hip, metadata, num_pages: int, page_size: int = 64, cache_type: str = "f16", *, k_pool=0, v_pool=0,
                 k_scale=0, v_scale=0, strides=None, allocator=None):
        if cache_type not in CACHE_TYPES:
            raise CudaSafetyError(f"cache_type {cache_type!r} is none of {', '.join(CACHE_TYPES)}")
        self.hip = hip
        self.num_q_heads, self.num_kv_heads, self.head_dim = _heads(metadata)
        self.rope_type = int(metadata.get('rope_type', 0))
        self.rotary_dim = int(metadata.get('rotary_dim', self.head_dim))
        self.num_pages, self.page_size, self.cache_type = int(num_pages), int(page_size), cache_type
        self._allocator = allocator
        self._owned: list = []
        self._life = self._life_of_runtime()
        self._closed = False
        self._workspace, self._workspace_bytes = 0, 0
        given = [_ptr_value(p) for p in (k_pool, v_pool, k_scale, v_scale)]
        if any(given[:2]) != all(given[:2]) or (any(given[2:]) and not given[0]):
            raise CudaSafetyError("k_pool and v_pool are given together, and scales with them")
        if num_pages <= 0 or page_size <= 0 or self.num_kv_heads <= 0 or self.head_dim <= 0 or self.num_q_heads <= 0:
            raise CudaSafetyError(f"{num_pages} pages of {page_size} positions, {self.num_q_heads} / {self.num_kv_heads} heads of {self.head_dim}")
        if strides is None:
            strides = (self.num_kv_heads * self.page_size * self.head_dim, self.head_dim, self.page_size * self.head_dim)
        elif not given[0]:
            raise CudaSafetyError("strides belong to pools of the caller's")
        if len(strides) != 3:
            raise CudaSafetyError(f"strides are (page, token, head), not {strides!r}")
        self._owns_pools = not given[0]
        if self._owns_pools:
            size = self.num_pages * self.num_kv_heads * self.page_size * self.head_dim * (2 if cache_type == "f16" else 1)
            scales = 0 if cache_type == "f16" else self.num_pages * self.num_kv_heads * 4
            try:
                given = [self._allocate(n, tag) if n else 0 for n, tag in
                         ((size, "paged_k"), (size, "paged_v"), (scales, "paged_k_scale"), (scales, "paged_v_scale"))]
            except Exception:
                self.cleanup()
                raise
        self.k_pool, self.v_pool, self.k_scale, self.v_scale = given
        self._cache = PagedCache(k_pool=given[0], v_pool=given[1], k_scale=given[2], v_scale=given[3], page_stride=int(strides[0]),
                                 token_stride=int(strides[1]), head_stride=int(strides[2]), num_pages=self.num_pages,
                                 page_size=self.page_size, num_kv_heads=self.num_kv_heads, head_dim=self.head_dim,
                                 type=CACHE_TYPES[cache_type])
        try:
            hip.paged_cache_init(self._cache)
        except Exception:
            self.cleanup()
            raise
        kv_row, q_row = self.num_kv_heads * self.head_dim, self.num_q_heads * self.head_dim
        self._append = PagedAppend(num_q_heads=self.num_q_heads, rope_type=-1, k_token_stride=kv_row, v_token_stride=kv_row,
                                   q_token_stride=q_row, q_out_token_stride=q_row)
        self._attention = PagedAttention(num_q_heads=self.num_q_heads)
        self._append.launch_flags = self._attention.launch_flags = 0 if getattr(hip, '_no_pdl', True) else LAUNCH_PROGRAMMATIC
        self._default_strides = (kv_row, kv_row, q_row, q_row)
        self._default_scale = 1.0 / math.sqrt(self.head_dim)

    # ------------------------------------------------------------------ memory
    def _life_of_runtime(self):
        """What a runtime has from one `initialize` to its `cleanup`, at which all that it allocated is freed."""
        return getattr(self.hip, '_launch_status', None)

    def _require_pools(self) -> None:
        if self._owns_pools and (self._closed or self._life is not self._life_of_runtime()):
            raise CudaSafetyError("the cache or its runtime has been cleaned up: its pools are gone")

    def _allocate(self, size: int, tag: str) -> int:
        if self._allocator is not None:
            block = self._allocator.allocate(size, tag, MemoryRegion.SCRATCH if tag == "paged_workspace" else MemoryRegion.KV_CACHE)
            self._owned.append(block)
            ptr = block.ptr
        else:
            handle = self.hip.safe_malloc(size, tag)
            self._owned.append(handle)
            ptr = handle.value
        self.hip.safe_memset(ctypes.c_void_p(ptr), size, tag)
        self.hip.synchronize()                    # calls may come on any stream
        return ptr

    @staticmethod
    def workspace_bytes(hip, metadata, batch_size: int, query_tokens: int = 1) -> int:
        """Bytes of a workspace for `attend`, zeroed by the caller before its first use and 256-byte aligned."""
        q_heads, kv_heads, head_dim = _heads(metadata)
        return hip.paged_attention_workspace(q_heads, kv_heads, head_dim, batch_size, query_tokens)

    def reserve(self, batch_size: int, query_tokens: int = 1) -> None:
        """Allocates the workspace of this cache's own, where the one it has does not do.  Not while the stream is captured."""
        self._require_pools()
        need = self.hip.paged_attention_workspace(self.num_q_heads, self.num_kv_heads, self.head_dim, batch_size, query_tokens)
        if self._life is not self._life_of_runtime():        # went with the runtime's cleanup
            self._owned.clear()
            self._workspace, self._workspace_bytes, self._life = 0, 0, self._life_of_runtime()
        if need > self._workspace_bytes:
            # earlier ones stay until cleanup: a captured step may still name them
            self._workspace = self._allocate(need + 256, "paged_workspace") + 255 & ~255
            self._workspace_bytes = need

    def set_rope(self, cos, sin, rows: int) -> None:
        """Rotation of q and k in `append`: fp16 tables of `rows` positions, with the metadata's `rope_type` and
        `rotary_dim`.  Addresses of 0 turn it off."""
        a = self._append
        if not _ptr_value(cos) and not _ptr_value(sin):
            a.rope_cos, a.rope_sin, a.rope_rows, a.rope_type = None, None, 0, -1
            return
        a.rope_cos, a.rope_sin, a.rope_rows = _ptr_value(cos), _ptr_value(sin), int(rows)
        a.rope_type, a.rotary_dim = self.rope_type, self.rotary_dim

    # ------------------------------------------------------------------ calls
    def append(self, k, v, block_table, kv_offsets, batch: int, max_pages: int, *, total_tokens=None, token_starts=0, q=0, q_out=0,
               token_strides=None, stream=None) -> None:
        """New tokens into the pages of their sequences: one a sequence, or `total_tokens` rows cut by `token_starts`
        (int32[batch + 1]; without it the same number each).  The newest token of sequence b goes to position kv_offsets[b].
        `token_strides`: halves between the tokens of k, v, q and q_out where their rows lie in something wider."""
        self._require_pools()
        a = self._append
        a.k, a.v, a.q, a.q_out = _address(k), _address(v), _address(q), _address(q_out)
        a.block_table, a.kv_offsets, a.token_starts = _address(block_table), _address(kv_offsets), _address(token_starts)
        if total_tokens is None and a.token_starts:
            raise CudaSafetyError("token_starts cuts total_tokens rows: their number is missing")
        a.batch, a.max_pages, a.total_tokens = batch, max_pages, batch if total_tokens is None else total_tokens
        a.k_token_stride, a.v_token_stride, a.q_token_stride, a.q_out_token_stride = token_strides or self._default_strides
        self.hip.paged_append(self._cache, a, stream)

    def attend(self, q, output, block_table, kv_offsets, batch: int, max_pages: int, *, query_tokens: int = 1, scale=None,
               output_f32: bool = False, lse=0, workspace=0, workspace_bytes: int = 0, stream=None) -> None:
        """The newest `query_tokens` tokens of each sequence over its cached positions, causally among themselves.
        `output` like q, fp16 or (`output_f32`) fp32; `lse` optional fp32 [batch, query_tokens, heads]."""
        self._require_pools()
        a = self._attention
        if workspace:
            a.workspace, a.workspace_bytes = _address(workspace), workspace_bytes
        else:
            self.reserve(batch, query_tokens)
            a.workspace, a.workspace_bytes = self._workspace, self._workspace_bytes
        a.q, a.output, a.lse = _address(q), _address(output), _address(lse)
        a.block_table, a.kv_offsets = _address(block_table), _address(kv_offsets)
        a.scale = self._default_scale if scale is None else scale
        a.out_is_f32, a.batch, a.max_pages, a.query_tokens = output_f32, batch, max_pages, query_tokens
        self.hip.paged_attention(self._cache, a, stream)

    def cleanup(self) -> None:
        """Frees what this cache allocated (a runtime that has been cleaned up has done so already).  A cache with pools of its own
        refuses calls from then on."""
        self._closed = True
        if self._life is not self._life_of_runtime() or (self._allocator is None and not getattr(self.hip, "_initialized", True)):
            self._owned.clear()
        for block in self._owned:
            if self._allocator is not None:
                self._allocator.free(block)
            else:
                self.hip.safe_free(block, "paged_cache")
        self._owned.clear()
        self._workspace = self._workspace_bytes = 0


def _address(p):
    return p if type(p) is int else _ptr_value(p)
