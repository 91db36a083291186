"""Paged attention where a lane of a warp gives up on a tile: the kernel ends, the status says so, what is incomplete is NaN and
everything else is right, and the workspace is ready for the next call.

The library's paged unit is built a second time with a wait that one lane of some warps reports as run out, at once, while the
copies are still on their way and the other lanes see them arrive.  Nothing is left out: every copy lands, every wait ends."""
import subprocess

import numpy as np
import pytest

from oracle import paged_oracle as orc
from tests.paged_case import Device, make_cache, metadata, random_pool, table_of, tolerance
from vte_b200 import build
from vte_b200.bridge import CudaRuntimeError
from vte_b200.bridge.cuda_runtime import load_library

pytestmark = pytest.mark.gpu

# One lane of warp 2 of every third block gives up on the second tile that it waits for, all others wait.  Waits with a limit of
# their own are as they were.
HOOKED = r"""
#include "kernels/vteb_common.cuh"
namespace vteb {
__device__ __forceinline__ bool wait_of_a_lane(uint32_t bar, uint32_t parity, volatile int* abort_word, int block, int thread) {
    if (block % 3 == 1 && thread == 2 * 32 + 5 && (bar & 31) == 8) return false;
    return mbar_wait_bounded(bar, parity, abort_word);
}
__device__ __forceinline__ bool wait_of_a_lane(uint32_t bar, uint32_t parity, volatile int* abort_word, long long limit) {
    return mbar_wait_bounded(bar, parity, abort_word, limit);
}
__device__ __forceinline__ bool wait_of_a_lane(uint32_t bar, uint32_t parity, volatile int* abort_word) {
    return wait_of_a_lane(bar, parity, abort_word, (int)blockIdx.x, (int)threadIdx.x);
}
}
#define mbar_wait_bounded wait_of_a_lane
#include "vteb200_paged.cu"
"""


@pytest.fixture(scope="module")
def hooked(built_library, tmp_path_factory):
    d = tmp_path_factory.mktemp("paged_wait")
    (d / "hooked.cu").write_text(HOOKED)
    subprocess.run([build._nvcc(), *build.ARCH_FLAGS, "-O3", "-split-compile", "0", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-diag-suppress", "550",
                    f"-I{build.CSRC}", "-o", str(d / "libhooked.so"), str(d / "hooked.cu"), str(built_library),
                    "-Xlinker", "-Bsymbolic", "-Xlinker", f"-rpath={built_library.parent}"], check=True, capture_output=True, text=True)
    return load_library(str(d / "libhooked.so"))


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
@pytest.mark.parametrize("heads,page,lengths,queries", [
    ((4, 2, 64), 64, [900 + 17 * i for i in range(80)], 1), ((12, 2, 128), 64, [40000], 1), ((8, 2, 128), 16, [20000, 300, 7000], 3),
    ((8, 4, 64), 16, [600] * 100, 1), ((4, 2, 256), 32, [2000 + i for i in range(20)], 1),
], ids=["ragged", "cut", "cut_queries", "two_workers", "256wide"])
def test_a_warp_gives_up_as_one(cuda_runtime, hooked, monkeypatch, kind, heads, page, lengths, queries):
    rt, dev = cuda_runtime, Device(cuda_runtime)
    rng = np.random.default_rng([page, len(lengths)])
    Hq, H, D = heads
    table, pages = table_of(rng, lengths, page)
    pools, scales = zip(*(random_pool(rng, kind, pages, heads, page) for _ in range(2)))
    q = rng.standard_normal((len(lengths), queries, Hq, D), dtype=np.float32).astype(np.float16)
    offsets = np.asarray(lengths, dtype=np.int32) - 1
    cache, _, _ = make_cache(dev, metadata(heads), kind, page, pools, scales)
    out, lse = np.zeros(q.shape, dtype=np.float16), np.zeros(q.shape[:3], dtype=np.float32)
    d_out, d_lse = dev.put(out), dev.put(lse)
    args = (dev.put(q), d_out, dev.put(table), dev.put(offsets), len(lengths), table.shape[1])
    ref, _, bound = orc.attention(q, *pools, *scales, kind, table, offsets, 1.0 / np.sqrt(D))
    most = tolerance(bound, ref, D, False)
    try:
        cache.reserve(len(lengths), queries)
        for again in range(2):
            with monkeypatch.context() as m:
                m.setattr(rt, "_lib", hooked)
                cache.attend(*args, query_tokens=queries, lse=d_lse)
                with pytest.raises(CudaRuntimeError, match=r"bounded wait \(code 1\)"):
                    rt.synchronize()
            out, lse = dev.get(d_out, out), dev.get(d_lse, lse)
            lost = np.isnan(lse)
            assert lost.any() and (lost == np.isnan(out).all(axis=-1)).all() and (lost == np.isnan(out).any(axis=-1)).all()
            assert (np.abs(out - ref) <= most)[~lost].all()
            assert len(lengths) < 50 or not lost.all()                # fewer are cut into pieces of which one is lost each
            cache.attend(*args, query_tokens=queries, lse=d_lse)      # the same workspace, the library's own wait
            rt.synchronize()
            assert (np.abs(dev.get(d_out, out) - ref) <= most).all()
    finally:
        cache.cleanup()
        dev.free()
