// How paged_attention_kernel deals its work, for the device and for a test on the CPU: units of U positions, segments of
// (sequence, KV head, block of rows), runs of units for the workers, and the pieces that segments leave which a border of two runs cuts.
#pragma once

#if defined(__CUDACC__)
#define VTEB_PAGED_HD __host__ __device__ __forceinline__
#else
#define VTEB_PAGED_HD inline
#endif

namespace vteb {

constexpr int kPagedMaxWorkers = 2;      // of a CTA
// Two workers a CTA from one segment on every fourth SM on (four query tokens of 8 sequences of 8 x 128-wide e4m3 heads 30.3 us, 32.4
// from one an SM on: that case alone); runs begin with a segment each up to so many units a warp (the same 30.3 us, 31.7 up to 4);
// units that a warp of a worker has at least (2,000 positions of 2 x 128-wide heads 10.3 us, 11.7 with 3 and 13.0 with 4).
constexpr int kPagedJoin = 8;            // pieces that are merged at once (sixteen: 8,000 positions of 2 x 256-wide fp16 heads 14.8 us instead of 13.8)
constexpr int kPagedTwoFrom = 4, kPagedTwoBelow = 192, kPagedAligned = 8, kPagedUnitsOfAWarp = 2, kPagedSegmentEnd = 2;

VTEB_PAGED_HD constexpr int paged_min(int x, int y) { return x < y ? x : y; }
VTEB_PAGED_HD constexpr int paged_max(int x, int y) { return x > y ? x : y; }

struct PagedDeal {
    int groups, workers, gw;             // workers of a CTA, of all, warps of one
    int mean, per, extra;                // units of a segment in the mean, of a run; what the end of a segment counts
    bool aligned;
    // What a segment counts.  Aligned runs: `per` units stand for what is left of one, so that no worker has parts of two.
    VTEB_PAGED_HD int room_of(int units) const { return units == 0 ? 0 : aligned ? (units + per - 1) / per * per : units + extra; }
};

// `units`: of all segments; `lives`: sequences that have any, of `batch`; `head_rows`: KV heads times blocks of rows; `grid` CTAs
// of `warps` warps.
VTEB_PAGED_HD PagedDeal paged_deal(int units, int lives, int head_rows, int batch, int grid, int warps) {
    PagedDeal d;
    // Workers of a CTA: two where there are segments for them and these are short, so that one computes while the other merges;
    // one where few segments would be cut more often for that, or where merges are rare beside units (one and two workers: 64
    // sequences of 8 x 64-wide heads, 136 units of e4m3 each, 100.1 and 96.7 us, 272 units of fp16 each, 151 and 155;
    // 100 of 10 to 8,000 positions 94 and 86; one of 32,768 positions 12.8 and 14.9).  Over eight lengths, one token a sequence:
    // 512 e4m3 segments gain by two 7 % at 24 units a segment, 3 at 192 and 2 at 512, 512 fp16 ones 6 % at 24, and lose
    // 1 to 3 from 96 on; 32 to 128 segments mostly lose, 1 to 5 %, at 48 units up to 15.  The limits lie between these.
    const int segments = paged_max(lives * head_rows, 1);         // (1 where nothing is cached: no worker has a unit then)
    d.mean = paged_max((units + segments - 1) / segments, 1);
    d.groups = segments * kPagedTwoFrom >= grid && d.mean < kPagedTwoBelow ? kPagedMaxWorkers : 1;
    d.workers = grid * d.groups;
    d.gw = warps / d.groups;
    // Units of a worker: an equal share, but not so few that a segment is cut where its warps would have little to do each.
    // Short runs begin with a segment each.
    d.aligned = segments * 2 <= d.workers && units < d.workers * d.gw * kPagedAligned;
    const int cuts = (d.mean + kPagedUnitsOfAWarp * d.gw - 1) / (kPagedUnitsOfAWarp * d.gw);
    const int over = !d.aligned ? d.workers : batch == 1 ? d.workers / segments * segments : d.workers - segments;
    // Long runs count the end of a segment, at which a worker's warps wait for one another, as units too, kPagedSegmentEnd a warp:
    // else runs of many short segments take half as long again as runs of one (100 sequences of 10 to 8,000 positions of
    // 8 x 64-wide e4m3 heads 86 us, 124 without; 64 of 1,024 to 16,384 97 and 102).
    d.extra = d.aligned ? 0 : kPagedSegmentEnd * d.gw;
    d.per = paged_max((units + d.extra * lives * head_rows + over - 1) / over, (d.mean + cuts - 1) / cuts);
    return d;
}

// Where a warp is in its worker's run: unit `u` of a segment, of which units [first, end) are this worker's.
struct PagedCursor {
    int b, head, rb, u, first, end, units, len;
    int left;                                               // what is left of the run from `first` on, ends of segments included
    int extra;                                              // what the end of a segment counts
};

template <int U, class Lengths>
VTEB_PAGED_HD void paged_enter(const Lengths& lengths, PagedCursor& c, int batch) {   // first sequence at or behind c.b that has units
    c.len = lengths(c.b);
    c.units = (c.len + U - 1) / U;
    while (c.units == 0 && c.b + 1 < batch) {
        c.len = lengths(++c.b);
        c.units = (c.len + U - 1) / U;
    }
}

// The run of a worker that begins `rest` into the units of sequence `b` and those behind; `behind`: from its begin to the last one's end.
template <int U, class Lengths>
VTEB_PAGED_HD PagedCursor paged_begin(const PagedDeal& d, const Lengths& lengths, int b, int rest, int behind, int batch, int row_blocks) {
    PagedCursor c;
    c.b = b;
    paged_enter<U>(lengths, c, batch);
    const int room = d.room_of(c.units), hr = rest / room;
    c.extra = d.extra;
    c.first = rest - hr * room;
    c.left = paged_min(d.per, d.aligned ? c.units - c.first : behind);
    c.head = row_blocks == 1 ? hr : hr / row_blocks;
    c.rb = row_blocks == 1 ? 0 : hr - c.head * row_blocks;
    c.end = paged_min(c.units, c.first + c.left);
    return c;
}

template <int U, class Lengths>
VTEB_PAGED_HD bool paged_next(const Lengths& lengths, PagedCursor& c, int batch, int num_kv_heads, int row_blocks) {
    c.left -= (c.end == c.units ? c.units + c.extra : c.end) - c.first;
    if (c.left <= 0) return false;
    c.first = 0;
    if (++c.rb == row_blocks) {
        c.rb = 0;
        if (++c.head == num_kv_heads) {
            c.head = 0;
            if (++c.b == batch) return false;               // (the run ends with the last segment's end)
            paged_enter<U>(lengths, c, batch);
        }
    }
    c.end = paged_min(c.units, c.left);
    return c.units > 0;                                     // (no units left: lengths that changed under the launch)
}

// Where a worker's piece of a cut segment goes: two places a worker, as a run has parts of two cut segments at most.
VTEB_PAGED_HD int paged_piece(int worker, bool first_of_run) { return 2 * worker + (first_of_run ? 0 : 1); }

// The workers whose runs hold units of a segment that begins at `begin` of all, and the places of their pieces.  Whoever comes last
// of up to `join` consecutive pieces merges those in place, and whoever comes last of these merges them: the many pieces of
// a long segment are read by several SMs, most of them ahead of the last piece.
struct PagedCut {
    int w0, n, p0, join;
    VTEB_PAGED_HD int place(int k) const { return k == 0 ? p0 : 2 * (w0 + k); }
    VTEB_PAGED_HD int start(int worker) const { return (worker - w0) / join * join; }
    VTEB_PAGED_HD int count(int level, int from) const { return level ? (n + join - 1) / join : paged_min(join, n - from); }
};

VTEB_PAGED_HD PagedCut paged_cut(int begin, int units, int per) {
    PagedCut c;
    c.w0 = begin / per;
    c.n = (begin + units - 1) / per - c.w0 + 1;
    c.p0 = paged_piece(c.w0, c.w0 * per == begin);
    c.join = c.n <= kPagedJoin ? c.n : c.n <= kPagedJoin * kPagedJoin ? kPagedJoin : (c.n + kPagedJoin - 1) / kPagedJoin;
    return c;
}

}  // namespace vteb
