"""How paged_attention_kernel deals its units (csrc/paged_partition.h), compiled for the CPU: every unit of every segment is one
worker's, the pieces of cut segments and their counters have places of their own, and readers look where writers wrote."""
import subprocess
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parent.parent / "vte_b200" / "csrc"

HARNESS = r"""
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <tuple>
#include <vector>
#include "paged_partition.h"
using namespace vteb;

struct Lengths {
    const std::vector<int>& n;
    int operator()(int b) const { return n.at(b); }
};
#define CHECK(x) do { if (!(x)) { std::printf("%s (line %d)\n", #x, __LINE__); std::exit(1); } } while (0)

// What one launch deals; `kind` counts aligned runs, two workers a CTA, cut segments and those merged in two steps.
template <int U>
static void deal_out(const std::vector<int>& n, int heads, int row_blocks, int grid, int warps, long long (&kind)[5]) {
    const int batch = (int)n.size(), HR = heads * row_blocks;
    const Lengths lengths{n};
    int units = 0, lives = 0;
    for (int x : n) { units += (x + U - 1) / U; lives += x > 0; }
    units *= HR;
    const PagedDeal d = paged_deal(units, lives, HR, batch, grid, warps);
    CHECK(d.groups >= 1 && d.groups <= kPagedMaxWorkers && d.workers == grid * d.groups && d.per >= 1 && d.gw * d.groups <= warps);
    long long total = 0;
    for (int x : n) total += (long long)d.room_of((x + U - 1) / U) * HR;
    if (batch == 1) CHECK(total == (lives ? (long long)d.room_of(d.mean) * HR : 0));
    CHECK(total < 1 << 30 && (long long)d.workers * d.per >= total);                  // all of it is dealt
    kind[0] += d.aligned; kind[1] += d.groups == 2;
    typedef std::tuple<int, int, int> Segment;
    struct Part { int first, end, units, worker, piece; bool entire; PagedCut cut; };
    std::map<Segment, std::vector<Part>> parts;
    for (int w = 0; w < d.workers; ++w) {
        const int lo = w * d.per;
        if (lo >= total) break;
        int b = 0, rest = lo;
        if (batch > 1)
            for (; ; ++b) {
                const int room = d.room_of((n[b] + U - 1) / U) * HR;
                if (rest < room) break;
                rest -= room;
            }
        PagedCursor at = paged_begin<U>(d, lengths, b, rest, (int)total - lo, batch, row_blocks);
        const int hi = lo + at.left;
        bool any = true;
        if (at.first >= at.units) {
            CHECK(!d.aligned);
            at.end = at.units;
            any = paged_next<U>(lengths, at, batch, heads, row_blocks);
        }
        int segments = 0;
        while (any) {
            CHECK(at.b < batch && at.head < heads && at.rb < row_blocks && at.len == n[at.b] && at.units == (at.len + U - 1) / U);
            CHECK(at.first >= 0 && at.first < at.end && at.end <= at.units && at.left > 0 && at.left <= d.per);
            Part p = {at.first, at.end, at.units, w, paged_piece(w, at.left == hi - lo), at.first == 0 && at.end == at.units, {}};
            if (!p.entire) p.cut = paged_cut(hi - at.left - at.first, at.units, d.per);
            parts[Segment(at.b, at.head, at.rb)].push_back(p);
            ++segments;
            any = paged_next<U>(lengths, at, batch, heads, row_blocks);
        }
        CHECK(!d.aligned || segments == 1);
    }
    std::set<int> pieces, counters[2];
    size_t expected = 0;
    for (int x : n) expected += x > 0 ? HR : 0;
    CHECK(parts.size() == expected);
    for (const auto& s : parts) {
        const std::vector<Part>& v = s.second;
        int next = 0;
        for (const Part& p : v) { CHECK(p.first == next); next = p.end; }
        CHECK(next == v[0].units);                                                    // each unit is one worker's, in order
        if (v.size() == 1) { CHECK(v[0].entire); continue; }
        const PagedCut& c = v[0].cut;
        CHECK(c.n == (int)v.size() && c.w0 == v[0].worker && c.join >= 1 && (c.n + c.join - 1) / c.join <= kPagedJoin);
        ++kind[2]; kind[3] += c.join < c.n;
        int arrivals = 0;
        for (int k = 0; k < c.n; ++k) {
            const Part& p = v[k];
            CHECK(!p.entire && p.worker == c.w0 + k && p.cut.w0 == c.w0 && p.cut.n == c.n && p.cut.p0 == c.p0 && p.cut.join == c.join);
            CHECK(p.piece == c.place(k) && p.piece < 2 * d.workers && pieces.insert(p.piece).second);
            CHECK(c.start(p.worker) == k / c.join * c.join);
            if (k % c.join == 0) {                                                    // a counter each for up to `join` pieces
                CHECK(counters[0].insert(c.place(k)).second && c.count(0, k) <= (c.join > kPagedJoin ? c.join : kPagedJoin));
                arrivals += c.count(0, k);
            }
        }
        CHECK(arrivals == c.n);
        if (c.join < c.n) CHECK(counters[1].insert(c.place(0)).second && c.count(1, 0) == (c.n + c.join - 1) / c.join);
    }
    ++kind[4];
}

int main() {
    int batch, heads, row_blocks, grid, warps, unit;
    long long kind[5] = {};
    while (std::scanf("%d %d %d %d %d %d", &batch, &heads, &row_blocks, &grid, &warps, &unit) == 6) {
        std::vector<int> n(batch);
        for (int& x : n) if (std::scanf("%d", &x) != 1) return 2;
        if (unit == 16) deal_out<16>(n, heads, row_blocks, grid, warps, kind);
        else if (unit == 32) deal_out<32>(n, heads, row_blocks, grid, warps, kind);
        else deal_out<64>(n, heads, row_blocks, grid, warps, kind);
    }
    std::printf("%lld %lld %lld %lld %lld\n", kind[0], kind[1], kind[2], kind[3], kind[4]);
    return 0;
}
"""


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged_partition")
    (d / "harness.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", "-o", str(d / "harness"), str(d / "harness.cpp")], check=True)
    return d / "harness"


@pytest.mark.parametrize("one", [True, False], ids=["one_sequence", "batches"])
def test_every_unit_is_one_workers_and_pieces_have_places_of_their_own(harness, one):
    rng = np.random.default_rng(int(one))
    launches = []
    for _ in range(600):
        batch = 1 if one else int(np.exp(rng.uniform(0, np.log(700))))
        longest = int(np.exp(rng.uniform(0, np.log(1e6 if one else 4e7 / batch if batch < 400 else 2000))))
        lengths = rng.integers(0, longest + 1, size=batch) * (rng.random(batch) > rng.choice([0.0, 0.3, 0.9]))
        shape = (int(rng.choice([1, 2, 3, 4, 8, 16])), int(rng.choice([1, 1, 2, 7])), int(rng.choice([148, 148, 132, 7])), int(rng.choice([6, 8])),
                 int(rng.choice([16, 32, 64])))
        launches.append((batch, *shape, *lengths.tolist()))
    launches += [(1, 2, 1, 148, 8, 32, n) for n in (0, 1, 31, 32, 33, 512, 2000, 11003, 32768)]
    launches += [(8, 8, 2, 148, 8, 32, *rng.integers(1000, 6001, size=8).tolist()), (64, 8, 1, 148, 8, 64, *rng.integers(1024, 16385, size=64).tolist())]
    run = subprocess.run([str(harness)], input="\n".join(" ".join(map(str, x)) for x in launches), capture_output=True, text=True)
    assert run.returncode == 0, run.stdout
    aligned, two_workers, cut, two_steps, all_ = map(int, run.stdout.split())
    assert all_ == len(launches) and aligned > 50 and aligned < all_ and cut > 100 and two_steps > 10 and (two_workers > 50)
