// Decode attention over a paged key/value cache of fp16, e4m3 or int8 values.
//
//   s[r, t] = scale * ks(page of t) * (q[r] . k[t]),  p = exp(s - max),  o[r] = sum_t p vs(page of t) v[t] / sum_t p
//
// for the rows r = (query token, query head of the group) of one (sequence, KV head) and the positions t that the row's
// query token sees.  What has to be moved is the cached rows, once: at 1 byte a value and up to 8 rows a KV head the
// tensor-core work is a third of what mma.sync can do in that time, so the kernel is built to keep loads in flight.
//
// Work.  The positions of a sequence are cut into units of U positions (4 to 8 KB of K and as much of V); (sequence, KV
// head, block of rows) is a segment, and all units of all segments, in that order, are dealt as equal runs to the
// workers.  A worker is all or half of the `W` warps of a CTA, one CTA an SM: the runs are computed on the device from the
// step's own lengths.  Each warp of a worker takes every gw-th unit and has a ring of its own in shared memory, which its own
// lanes fill with tensor-map copies (one box a page) and which only it reads: no warp waits for another between the
// ends of segments, and the loads of the next segment are in flight while one is merged.
//
// Arithmetic.  Positions are the M dimension of both products (S^T = K Q^T, O^T = V^T P^T): a group of up to eight rows is
// one n8 tile, and what is converted from 8 bits to fp16 is the A operand, once for all rows.  ldmatrix on 8-bit rows
// delivers pairs of values; the order of channels inside a 16-channel step is free as long as Q (or the output column)
// follows, so K needs no shuffling at all and V one byte permute per four values.  e4m3 and int8 values are exact in
// fp16.  P is rounded to fp16 where the output is fp16, whose own rounding is as large; for fp32 output it is split into
// two fp16 parts.  Weights are taken relative to the row's maximum less kPagedShift, so that fp16 holds those down to 2^-29 of the
// largest with all its bits and the last ones to 2^-40: relative to the maximum itself, positions 17 above the others took
// 0.8 % of what those add up to, 5 to 14 % beside pages of larger scales.  Page scales never touch the stored values: ks
// multiplies the scores, and O is held in units of the last page's vs, so that P itself is what fp16 has to hold.
//
// Merging.  A segment's warps are merged through shared memory in warp order.  Segments that a worker border cuts leave
// (m, l, o) pieces in the workspace, and the last worker to arrive merges them in worker order: results do not depend on
// who is last, and no block waits for another.
//
// Bound by bytes on long or many sequences (64 ragged ones of 8 x 64-wide heads with start and end: fp16 93 % of the copy
// bandwidth, e4m3 79 to 84 from machine to machine), by latency on short ones: 512 positions take 7.8 us, of which the chain of
// offset, table entry, tile, two units a warp and merge is all but the launch.  With 16 rows a segment a warp's products,
// conversions and softmax wait for one another: two warps a scheduler fill 40 % of its issue slots.
#pragma once

#include <type_traits>

#include "../paged_partition.h"
#include "vteb_common.cuh"

namespace vteb {

constexpr int kPagedF16 = 0, kPagedE4m3 = 1, kPagedInt8 = 2;
constexpr int kStatusBadPage = 5;        // a block table entry outside 0..num_pages-1 for a position that is read or written
constexpr int kStatusBadPosition = 6;    // a position beyond the block table or the rotation tables

struct PagedAttnArgs {
    KvTensorMap k_map, v_map;
    const __half* q;                 // [batch, queries, Hq, D]
    void* output;                    // same shape, fp16 or fp32
    float* lse;                      // [batch, queries, Hq] or null
    const int* block_table;          // [batch, max_pages]
    const int* kv_offsets;           // [batch]
    const float* k_scale;            // [num_pages, Hkv], 8-bit pages
    const float* v_scale;
    int* counters;                   // [2][2 * workers], zero between launches: of the pieces that are merged into one
    float* part_ml;                  // [2 * workers][rows][2]: pieces of cut segments
    float* part_ml2;                 // the same of merged ones
    float* part_o;                   // [2 * workers][rows][D]
    int* status;
    int batch, max_pages, num_pages, page_log2, box_log2;
    int num_q_heads, num_kv_heads, group, queries, row_blocks;
    unsigned group_inv;              // ceil(2^31 / group): r / group = 2 r * group_inv >> 32 for the 2^16 rows r there can be
    float scale_log2e;
};

// Positions of a unit (4 or 8 KB of K, and as much of V) and warps of a CTA, so that the rings (192 KB of an SM's 227) hold at
// least two units a warp.  Few warps with many registers: a warp's own loads, conversions and products overlap, which twelve
// of 168 registers or sixteen of 128 do less well (64 sequences of 8 x 64-wide e4m3 heads, side by side: 103, 114 and 217 us).
__host__ __device__ constexpr int paged_unit(int row_bytes) { return row_bytes >= 256 ? 16 : 4096 / row_bytes; }
__host__ __device__ constexpr int paged_warps(int row_bytes) { return row_bytes == 512 ? 6 : 8; }
constexpr long long kPagedLandingCycles = 4000000000;      // for copies of a warp that gave up: about two seconds a slot
constexpr float kPagedShift = 15.f, kPagedUnshift = 0x1p-15f;     // 2^15 is the largest power of two that fp16 has

template <int D, int KIND, int NT>
struct PagedShape {
    static constexpr int ES = KIND == kPagedF16 ? 2 : 1;
    static constexpr int RB = D * ES;                       // bytes of a row
    static constexpr int CB = RB < 128 ? RB : 128;          // bytes of a column block: the width of a box
    static constexpr int W = paged_warps(RB);
    static constexpr int RING = 192 * 1024 / W;             // bytes of a warp's ring
    static constexpr int U = paged_unit(RB);                           // positions of a unit
    static constexpr int SLOT = 2 * U * RB;                 // K, then V
    static constexpr int NS = RING / SLOT;
    static constexpr int ROWS = 8 * NT;
    static constexpr int PART = 1024;                       // bytes a warp has for the newest tokens' weights
    static constexpr int SMEM = 1024 + W * (RING + PART + ROWS * 8 + 4 * 4 * 8 + 64);
    static_assert(NS >= 2 && NS <= 4, "units in a ring");
    static_assert(ROWS * D * 4 <= SLOT, "a warp's rows fit the slot that it read last");
    static_assert(PART >= 15 * ROWS * 4, "weights of the newest tokens");
};

#if defined(__CUDACC__)

__device__ __forceinline__ void tma_load_pages(uint32_t dst, const void* map, int y, int head, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(dst), "l"(map), "r"(0), "r"(y), "r"(0), "r"(head), "r"(page), "r"(bar)
        : "memory");
}

__device__ __forceinline__ bool elect_one() {               // true in one lane of a warp, always the same one
    uint32_t yes;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
    return yes != 0;
}

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_half2_down(float x, float y) {      // towards zero
    uint32_t r;
    asm("cvt.rz.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(x), "f"(y));
    return r;
}

__device__ __forceinline__ uint32_t above_zero(uint32_t x) {     // both halves, at least 2^-24; NaN stays NaN
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x00010001u));
    return r;
}

// Four 8-bit values to fp16, exactly: lo = values 0 and 1 of the word (2 and 3 with them in hi), or with `PAIRS` 0 and 2
// (1 and 3), which is how ldmatrix.trans leaves two positions of two channels.
template <int KIND, bool PAIRS>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (KIND == kPagedE4m3) {
        if constexpr (PAIRS) w = __byte_perm(w, 0, 0x3120);
        asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
            : "=r"(lo), "=r"(hi) : "r"(w));
    } else {
        // bytes x + 128 under the exponent of 1024: the half 1024 + 128 + x, less 1152
        w ^= 0x80808080u;
        const uint32_t a = __byte_perm(w, 0x64646464u, PAIRS ? 0x4240 : 0x4140);
        const uint32_t b = __byte_perm(w, 0x64646464u, PAIRS ? 0x4341 : 0x4342);
        const uint32_t bias = 0x64806480u;
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&bias));
        const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&bias));
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    }
}

// Byte offset inside a box (column blocks of `block` bytes one after another, swizzled) of 16-byte chunk `chunk` of row `r`.
template <int CB>
__device__ __forceinline__ uint32_t box_offset(int r, int chunk, int block) {
    constexpr int PER = CB / 16;                            // chunks of a column block
    return (uint32_t)((chunk / PER) * block + r * CB + (((chunk % PER) ^ (CB == 128 ? r & 7 : (r >> 1) & 3)) * 16));
}

__device__ __forceinline__ void group_barrier(int gw, int group) {
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(gw * 32) : "memory");
}

struct PagedLengths {                                       // cached positions of sequence b, no more than its table has room for
    const PagedAttnArgs& a;
    __device__ __forceinline__ int operator()(int b) const {
        const int room = a.max_pages << a.page_log2;        // at most 2^30, checked by the host
        const int off = a.kv_offsets[b];
        return off < 0 ? 0 : off >= room ? room : off + 1;
    }
};

template <int D, int KIND, int NT, bool F32>
__global__ void __launch_bounds__(PagedShape<D, KIND, NT>::W * 32, 1) paged_attention_kernel(const __grid_constant__ PagedAttnArgs a)
{
    using S = PagedShape<D, KIND, NT>;
    constexpr int U = S::U, RB = S::RB, CB = S::CB, NS = S::NS, W = S::W, SLABS = U / 16, KSTEPS = D / 16, ROWS = S::ROWS;
    constexpr bool kScaled = KIND != kPagedF16;

    extern __shared__ unsigned char smem_raw[];
    __shared__ int s_scan[W], s_live[W], s_start_b[kPagedMaxWorkers], s_start_rest[kPagedMaxWorkers], s_last[kPagedMaxWorkers], s_slot[W];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    unsigned char* ring = smem + warp * S::RING;
    unsigned char* part_all = smem + W * S::RING;
    float2* ml_all = reinterpret_cast<float2*>(part_all + W * S::PART);
    float2* scales = ml_all + W * ROWS + warp * 16;                                           // [unit % 4][box], of K and V
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(ml_all + W * ROWS + W * 16) + warp * 8;
    const uint32_t ring_u = smem_u32(ring), bars_u = smem_u32(bars), scales_u = smem_u32(scales);

    if (lane == 0) {
        for (int i = 0; i < NS; ++i) mbar_init(bars_u + i * 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (warp == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&a.k_map) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&a.v_map) : "memory");
        }
    }
    // Nothing of the launches in front is touched before this; the launch behind may start when they are complete.  Ordinary loads
    // throughout: a non-coherent one may be moved ahead of the wait, and is not for what is written while the block is there.
    grid_dependency_wait();
    grid_launch_dependents();

    const int box_rows = 1 << a.box_log2;
    const int boxes = U >> a.box_log2;                      // of a unit
    const int HR = a.num_kv_heads * a.row_blocks;

    // ---- all units, and where this CTA's workers begin ------------------------------------------
    const PagedLengths lengths{a};
    auto units_of = [&](int b) { return (lengths(b) + U - 1) / U; };
    const int per_thread = (a.batch + W * 32 - 1) / (W * 32);
    const int b0 = min(tid * per_thread, a.batch), b1 = min(b0 + per_thread, a.batch);
    int total = 0, lives = 0, mine = 0, upto = 0;
    auto scan = [&](auto units) {                           // this thread's sequences, all up to them, all
        mine = 0;
        for (int b = b0; b < b1; ++b) mine += units(b);
        upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int x = __shfl_up_sync(~0u, upto, d);
            if (lane >= d) upto += x;
        }
        if (lane == 31) s_scan[warp] = upto;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w < warp) upto += s_scan[w];
            total += s_scan[w];
        }
    };
    if (a.batch == 1) {
        total = units_of(0);
        lives = total > 0;
        __syncwarp();
    } else {
        int live = 0;
        for (int b = b0; b < b1; ++b) live += units_of(b) > 0;
        live = __reduce_add_sync(~0u, live);
        if (lane == 0) s_live[warp] = live;
        scan(units_of);
#pragma unroll
        for (int w = 0; w < W; ++w) lives += s_live[w];
    }
    total *= HR;
    const int grid = gridDim.x;
    const PagedDeal deal = paged_deal(total, lives, HR, a.batch, grid, W);
    const int groups = deal.groups, gw = deal.gw, per = deal.per;
    const int group = groups == 1 ? 0 : warp / (W / 2), wi = groups == 1 ? warp : warp % (W / 2);
    if (a.batch == 1) total = lives ? deal.room_of(deal.mean) * HR : 0;
    else {
        __syncthreads();                                    // s_scan is written anew
        scan([&](int b) { return deal.room_of(units_of(b)); });
        total *= HR;
    }
    const int worker = blockIdx.x * groups + group;
    const int lo = worker * per;
    if (a.batch > 1) {
        for (int g = 0; g < groups; ++g) {
            const int at = (blockIdx.x * groups + g) * per;
            if (at >= (upto - mine) * HR && at < upto * HR) {
                int rest = at - (upto - mine) * HR, b = b0;
                for (; b < b1; ++b) {
                    const int n = deal.room_of(units_of(b)) * HR;
                    if (rest < n) break;
                    rest -= n;
                }
                s_start_b[g] = b;
                s_start_rest[g] = rest;
            }
        }
        __syncthreads();
    }

    if (lo < total) {
    PagedCursor at = paged_begin<U>(deal, lengths, a.batch > 1 ? s_start_b[group] : 0, a.batch > 1 ? s_start_rest[group] : lo, total - lo,
                                    a.batch, a.row_blocks);         // what this warp computes
    const auto next_segment = [&](PagedCursor& c) { return paged_next<U>(lengths, c, a.batch, a.num_kv_heads, a.row_blocks); };
    const int hi = lo + at.left;
    bool any = true;
    if (at.first >= at.units) {                             // the run begins within the end of a segment
        at.end = at.units;
        any = next_segment(at);
    }
    if (any) {
    // ---- the ring: tables, scales, K and V on their way ----------------------------------------------
    PagedCursor ahead = at;                                 // the unit whose table entries are asked for next
    bool more = true;
    ahead.u = ahead.first + wi;
    // Table entries are read for as many units of a segment at once as the lanes hold, a batch ahead of their use.
    struct Batch { int page = 0, u = 0, n = 0, len = 0, head = 0; } cur, nxt;
    const int box_lanes = 31 - __clz(boxes);                // log2
    int fill_slot = 0, taken = 0, filled = 0;
    auto fill = [&]() {                                     // K and V of the next unit, if there is one
#pragma unroll 1
        for (int i = 0; i < 2 && taken == cur.n; ++i) {     // (twice where nothing has been looked up yet)
            cur = nxt;
            taken = 0;
            nxt.n = 0;
            while (more && ahead.u >= ahead.end) { more = next_segment(ahead); ahead.u = ahead.first + wi; }
            if (!more) continue;
            nxt.n = min(32 >> box_lanes, (ahead.end - ahead.u + gw - 1) / gw);
            nxt.u = ahead.u;
            nxt.len = ahead.len;
            nxt.head = ahead.head;
            const int k = lane >> box_lanes;
            const int pos = (ahead.u + k * gw) * U + ((lane & (boxes - 1)) << a.box_log2);
            nxt.page = k < nxt.n && pos < ahead.len ? a.block_table[(long long)ahead.b * a.max_pages + (pos >> a.page_log2)] : 0;
            ahead.u += nxt.n * gw;
        }
        if (taken < cur.n) {
            const int pos = (cur.u + taken * gw) * U, from = taken << box_lanes;
            const int need = min(boxes, (cur.len - pos + box_rows - 1) >> a.box_log2);
            const uint32_t bar = bars_u + fill_slot * 8;
            uint32_t dst = ring_u + fill_slot * S::SLOT;
            if (elect_one()) mbar_arrive_expect_tx(bar, (uint32_t)(2 * need * box_rows * RB));
#pragma unroll 1
            for (int i = 0; i < need; ++i, dst += box_rows * RB) {
                const int found = __shfl_sync(~0u, cur.page, from + i);
                const bool bad = (unsigned)found >= (unsigned)a.num_pages;
                const int page = bad ? 0 : found, y = (pos + (i << a.box_log2)) & ((1 << a.page_log2) - 1);
                if (elect_one()) {
                    tma_load_pages(dst, &a.k_map, y, cur.head, page, bar);
                    tma_load_pages(dst + U * RB, &a.v_map, y, cur.head, page, bar);
                    const int sc = (filled & 3) * 4 + i;
                    if (bad) {                              // a page that is not there makes its sequence's rows NaN
                        scales[sc] = make_float2(NAN, NAN);
                        if (a.status) *a.status = kStatusBadPage;
                    } else if (kScaled) {
                        const long long at_ = (long long)page * a.num_kv_heads + cur.head;
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(scales_u + sc * 8), "l"(a.k_scale + at_) : "memory");
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(scales_u + sc * 8 + 4), "l"(a.v_scale + at_) : "memory");
                    } else scales[sc] = make_float2(1.f, 1.f);
                }
            }
            ++taken;
            if (++fill_slot == NS) fill_slot = 0;
        }
        ++filled;
        if (kScaled) asm volatile("cp.async.commit_group;" ::: "memory");       // one a call: the scales of a unit are here when NS - 1 are not
    };

    const int g4 = lane >> 2, t4 = lane & 3;
    // Where this lane's row of an ldmatrix begins in a slab, for the first two chunks; the chunks of step 2 i are those xor 2 i
    // (a slab's first row is a multiple of 16, so the swizzle is the same for all slabs).
    const int block = box_rows * CB;                        // bytes of a column block of a box
    const uint32_t k_at = box_offset<CB>((lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4, 0);                    // K, and V of 8-bit pages
    const uint32_t v_at = kScaled ? k_at : box_offset<CB>((lane & 7) + (lane >> 4) * 8, (lane >> 3) & 1, 0);   // V of 16-bit pages
    auto chunk_at = [&](uint32_t first, int chunk) { return (first ^ ((chunk % (CB / 16)) * 16)) + (chunk / (CB / 16)) * block; };
    const int rows_all = a.queries * a.group;
    const int gt = wi * 32 + lane, gthreads = gw * 32;      // thread of the worker
    const float2* ml = ml_all + group * gw * ROWS;

    uint32_t qf[NT][KSTEPS][2];                             // Q of row n (this lane: n = g4) as B operand
    // m is the largest score less kPagedShift; what leaves the warp as l and o is without the factor 2^15 that comes of it
    float m[NT][2], l[NT][2], o[NT][KSTEPS][4], vref = 0.f, vmax = 0.f;
    if (lane == 0) s_slot[warp] = 0;                        // a warp that computes nothing is read, and not used
    int slot = 0, u = 0;
    uint32_t phase = 0;
    bool fresh = true, dead = false;

    // One turn: a unit computed (none while the ring is filled at first, or where the segment has none for this warp), the
    // segment closed where it ends, and a unit asked for into the slot that has come free.  One copy of each in the code, which
    // a short launch spends as much time on fetching as on running.
#pragma unroll 1
    for (;;) {
        if (fresh) {
            fresh = false;
            u = at.first + wi;
            vref = vmax = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                m[nt][0] = m[nt][1] = -INFINITY;
                l[nt][0] = l[nt][1] = dead && u < at.end ? NAN : 0.f;
                const int r = at.rb * ROWS + nt * 8 + g4;
                const int j = __umulhi(2 * r, a.group_inv), g = r - j * a.group;
                const __half* src = a.q + (((long long)at.b * a.queries + j) * a.num_q_heads + at.head * a.group + g) * D;
#pragma unroll
                for (int ks = 0; ks < KSTEPS; ++ks) {
                    o[nt][ks][0] = o[nt][ks][1] = o[nt][ks][2] = o[nt][ks][3] = 0.f;
                    qf[nt][ks][0] = qf[nt][ks][1] = 0;
                    if (r < rows_all) {
                        if (kScaled) {
                            const uint2 x = *reinterpret_cast<const uint2*>(src + ks * 16 + t4 * 4);
                            qf[nt][ks][0] = x.x; qf[nt][ks][1] = x.y;
                        } else {
                            qf[nt][ks][0] = *reinterpret_cast<const uint32_t*>(src + ks * 16 + t4 * 2);
                            qf[nt][ks][1] = *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8 + t4 * 2);
                        }
                    }
                }
            }
        }
        bool room = filled < NS;
        const bool turn = !room;
        if (turn && u < at.end) {
            room = true;
            const int whole = at.len - a.queries + 1;       // positions that every row sees
            const bool ragged = (u + 1) * U > whole;
            int limit[NT][2];                               // positions that the rows of this lane's columns see
            if (ragged) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int r = at.rb * ROWS + nt * 8 + t4 * 2 + e;
                        limit[nt][e] = r < rows_all ? whole + (int)__umulhi(2 * r, a.group_inv) : 0;
                    }
            }
            if (kScaled) asm volatile("cp.async.wait_group %0;" ::"n"(NS - 1) : "memory");
            // Each lane's wait has its own limit: the warp gives up as one, as it has to be whole for what follows.  Rows that it
            // had a part of are NaN then, it asks for nothing more, and the copies under way land before it goes on, as the slots
            // are not its own until then: from this slot up to the one that would be filled next.
            if (!dead && __any_sync(~0u, !mbar_wait_bounded(bars_u + slot * 8, phase, nullptr))) {
                dead = true;
                if (lane == 0 && a.status) *a.status = kStatusFullTimeout;
                asm volatile("cp.async.wait_all;" ::: "memory");
                uint32_t under_way = phase;
                int i = slot;
                do {
                    mbar_wait_bounded(bars_u + i * 8, under_way, nullptr, kPagedLandingCycles);
                    if (++i == NS) { i = 0; under_way ^= 1; }
                } while (i != fill_slot);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) l[nt][0] = l[nt][1] = NAN;
            }
            __syncwarp();

            // ---- scores
            const uint32_t kbase = ring_u + slot * S::SLOT, vbase = kbase + U * RB;
            const float2* sc = scales + ((filled - NS) & 3) * 4;
            float s[SLABS][NT][4], vs[SLABS];
#pragma unroll
            for (int sl = 0; sl < SLABS; ++sl) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[sl][nt][0] = s[sl][nt][1] = s[sl][nt][2] = s[sl][nt][3] = 0.f;
                const int box = (sl * 16) >> a.box_log2;
                const uint32_t from = kbase + box * box_rows * RB + ((sl * 16) & (box_rows - 1)) * CB;
                const float2 x = sc[box];
                const float ks_ = x.x * a.scale_log2e;
                vs[sl] = x.y;
                if constexpr (kScaled) {
#pragma unroll
                    for (int ks = 0; ks < KSTEPS; ks += 2) {
                        uint32_t r0, r1, r2, r3, f0, f1, f2, f3;
                        ldmatrix_x4(from + chunk_at(k_at, ks), r0, r1, r2, r3);
                        widen<KIND, false>(r0, f0, f2);
                        widen<KIND, false>(r1, f1, f3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_16816(s[sl][nt], f0, f1, f2, f3, qf[nt][ks][0], qf[nt][ks][1]);
                        widen<KIND, false>(r2, f0, f2);
                        widen<KIND, false>(r3, f1, f3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_16816(s[sl][nt], f0, f1, f2, f3, qf[nt][ks + 1][0], qf[nt][ks + 1][1]);
                    }
                } else {
#pragma unroll
                    for (int ks = 0; ks < KSTEPS; ++ks) {
                        uint32_t f0, f1, f2, f3;
                        ldmatrix_x4(from + chunk_at(k_at, ks * 2), f0, f1, f2, f3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_16816(s[sl][nt], f0, f1, f2, f3, qf[nt][ks][0], qf[nt][ks][1]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[sl][nt][e] *= ks_;
            }
            if (ragged) {
#pragma unroll
                for (int sl = 0; sl < SLABS; ++sl)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (u * U + sl * 16 + g4 + (e >> 1) * 8 >= limit[nt][e & 1]) s[sl][nt][e] = -INFINITY;
            }

            // ---- running maximum and sum
            float alpha[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = -INFINITY;
#pragma unroll
                    for (int sl = 0; sl < SLABS; ++sl) top = fmaxf(top, fmaxf(s[sl][nt][e], s[sl][nt][e + 2]));
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
                    top = fmaxf(m[nt][e], __fadd_ru(top, -kPagedShift));     // rounded up: no weight is above 2^15, whatever the scores
                    const float ref = top == -INFINITY ? 0.f : top;
                    alpha[nt][e] = fast_exp2(m[nt][e] - ref);
                    m[nt][e] = top;
                    float sum = 0.f;
#pragma unroll
                    for (int sl = 0; sl < SLABS; ++sl) {
                        s[sl][nt][e] = fast_exp2(s[sl][nt][e] - ref);
                        s[sl][nt][e + 2] = fast_exp2(s[sl][nt][e + 2] - ref);
                        sum += s[sl][nt][e] + s[sl][nt][e + 2];
                    }
                    l[nt][e] = l[nt][e] * alpha[nt][e] + sum;
                }

            // O is held in units of `vref`.  A unit of one page makes its scale the unit, which costs nothing beside the
            // rescaling that O has to have; scales that O could overflow under (2^-40 of the largest), that are zero, not
            // finite or of extreme size, and units of several pages have their weights multiplied instead.
            if constexpr (kScaled) {
                float shrink;
                if (boxes == 1 && vs[0] >= vmax * 0x1p-40f && vs[0] > 0x1p-100f && vs[0] < 0x1p100f && vref < 0x1p100f) {
                    shrink = vref == vs[0] ? 1.f : __fdividef(vref, vs[0]);
                    vref = vs[0];
                } else {
                    float top = vref;
#pragma unroll
                    for (int sl = 0; sl < SLABS; ++sl) {
                        if (u * U + sl * 16 >= at.len) vs[sl] = 0.f;             // a page behind the last one
                        if (!(fabsf(vs[sl]) < INFINITY)) vs[sl] = NAN;
                        top = fmaxf(top, fabsf(vs[sl]));
                    }
                    // (steps of 2^64 keep the reciprocal in the normal range)
                    const float step = top > 1.f ? 0x1p-64f : 0x1p64f, inv = top > 0.f ? __fdividef(1.f, top * step) : 0.f;
                    shrink = top > 0.f ? vref * step * inv : 1.f;
#pragma unroll
                    for (int sl = 0; sl < SLABS; ++sl) {
                        const float c = vs[sl] * step * inv;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[sl][nt][e] = ragged && s[sl][nt][e] == 0.f ? 0.f : s[sl][nt][e] * c;
                    }
                    vref = top;
                }
                vmax = fmaxf(vmax, vref);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) { alpha[nt][0] *= shrink; alpha[nt][1] *= shrink; }
            }
            bool same = true;                               // the maxima and the unit of O are mostly what they were
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) same = same && alpha[nt][0] == 1.f && alpha[nt][1] == 1.f;
            if (!__all_sync(~0u, same)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < KSTEPS; ++j) {
                        o[nt][j][0] *= alpha[nt][0]; o[nt][j][1] *= alpha[nt][1];
                        o[nt][j][2] *= alpha[nt][0]; o[nt][j][3] *= alpha[nt][1];
                    }
            }

            // ---- V rows that not every row sees.  They may hold anything, and zero times anything may be NaN: the newest tokens'
            // rows are added one by one to the rows that see them, and then they and what lies behind them are cleared.
            if (ragged) {
                const int from = max(whole - u * U, 0);     // first such position of the unit
                const int till = min(at.len - u * U, U);
                if (a.queries > 1 && from < till) {
                    float* w = reinterpret_cast<float*>(part_all + warp * S::PART) - from * ROWS;
#pragma unroll
                    for (int sl = 0; sl < SLABS; ++sl)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int t = sl * 16 + g4 + (e >> 1) * 8;
                                if (t >= from && t < till) w[t * ROWS + nt * 8 + t4 * 2 + (e & 1)] = s[sl][nt][e];
                                if (t >= from) s[sl][nt][e] = 0.f;
                            }
                    __syncwarp();
#pragma unroll 1
                    for (int t = from; t < till; ++t) {
                        const uint32_t box = vbase + (t >> a.box_log2) * box_rows * RB;
                        const int row = t & (box_rows - 1);
                        const float* wt = w + t * ROWS + t4 * 2;
#pragma unroll
                        for (int j = 0; j < KSTEPS; ++j) {
                            float v0, v1;                   // channels of this lane's accumulators
                            if constexpr (kScaled) {
                                uint32_t x, y;
                                asm volatile("ld.shared.u16 %0, [%1];" : "=r"(x) : "r"(box + box_offset<CB>(row, j, block) + g4 * 2));
                                widen<KIND, false>(x, x, y);
                                const float2 f = unpack_half2(x);
                                v0 = f.x; v1 = f.y;
                            } else {
                                unsigned short x, y;
                                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(box + box_offset<CB>(row, j * 2, block) + g4 * 2));
                                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y) : "r"(box + box_offset<CB>(row, j * 2 + 1, block) + g4 * 2));
                                v0 = __half2float(__ushort_as_half(x)); v1 = __half2float(__ushort_as_half(y));
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 2; ++e)
                                    if (u * U + t < limit[nt][e]) {
                                        o[nt][j][e] += wt[nt * 8 + e] * v0;
                                        o[nt][j][e + 2] += wt[nt * 8 + e] * v1;
                                    }
                        }
                    }
                    __syncwarp();
                }
#pragma unroll 1
                for (int i = lane; i < (U - from) * (RB / 16); i += 32) {
                    const int t = from + i / (RB / 16);
                    const uint32_t to = vbase + (t >> a.box_log2) * box_rows * RB + box_offset<CB>(t & (box_rows - 1), i % (RB / 16), block);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(to), "r"(0) : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // the slot's next copies come behind these stores
                __syncwarp();
            }

            // ---- P V
#pragma unroll
            for (int sl = 0; sl < SLABS; ++sl) {
                uint32_t p[NT][2], pl[NT][2];               // P^T as B operand; its low parts for fp32 output
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float x = s[sl][nt][2 * e], y = s[sl][nt][2 * e + 1];
                        // An infinite V stays infinite only under weights above zero: those of 16-bit pages are no less than fp16's
                        // least, 2^-39 of the largest, and the low part is what a high one rounded down leaves.  (Rows that not all
                        // see are zeros by now.)
                        const uint32_t h = kScaled ? pack_half2(x, y) : above_zero(F32 ? pack_half2_down(x, y) : pack_half2(x, y));
                        p[nt][e] = transpose_8x8(h);
                        if (F32) {
                            const float2 back = unpack_half2(h);
                            const uint32_t low = pack_half2(x - back.x, y - back.y);
                            pl[nt][e] = transpose_8x8(kScaled ? low : above_zero(low));
                        }
                    }
                const int box = (sl * 16) >> a.box_log2;
                const uint32_t from = vbase + box * box_rows * RB + ((sl * 16) & (box_rows - 1)) * CB;
#pragma unroll
                for (int j = 0; j < KSTEPS; j += 2) {
                    uint32_t f[8];                          // two 16-channel steps of V^T
                    if constexpr (kScaled) {
                        uint32_t x0, x1, x2, x3;
                        ldmatrix_x4_trans(from + chunk_at(v_at, j), x0, x1, x2, x3);
                        widen<KIND, true>(x0, f[0], f[1]);
                        widen<KIND, true>(x1, f[2], f[3]);
                        widen<KIND, true>(x2, f[4], f[5]);
                        widen<KIND, true>(x3, f[6], f[7]);
                    } else {
                        ldmatrix_x4_trans(from + chunk_at(v_at, j * 2), f[0], f[1], f[2], f[3]);
                        ldmatrix_x4_trans(from + chunk_at(v_at, j * 2 + 2), f[4], f[5], f[6], f[7]);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_16816(o[nt][j], f[0], f[1], f[2], f[3], p[nt][0], p[nt][1]);
                        mma_16816(o[nt][j + 1], f[4], f[5], f[6], f[7], p[nt][0], p[nt][1]);
                        if (F32) {
                            mma_16816(o[nt][j], f[0], f[1], f[2], f[3], pl[nt][0], pl[nt][1]);
                            mma_16816(o[nt][j + 1], f[4], f[5], f[6], f[7], pl[nt][0], pl[nt][1]);
                        }
                    }
                }
            }
            u += gw;
            if (u >= at.end && lane == 0) s_slot[warp] = slot;
            if (++slot == NS) { slot = 0; phase ^= 1; }
            __syncwarp();                                   // the slot has been read by every lane
        }
        if (turn && u >= at.end) {
        // ---- end of the segment: the warps of the worker are merged ------------------------------------
        const bool entire = at.first == 0 && at.end == at.units;
        const bool has_first = at.left == hi - lo;
        const int rows_here = min(ROWS, rows_all - at.rb * ROWS);
        const int piece = paged_piece(worker, has_first);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = l[nt][e];
                x += __shfl_xor_sync(~0u, x, 4);
                x += __shfl_xor_sync(~0u, x, 8);
                x += __shfl_xor_sync(~0u, x, 16);
                if (g4 == 0) ml_all[warp * ROWS + nt * 8 + t4 * 2 + e] = make_float2(m[nt][e], x * kPagedUnshift);
            }
        auto put = [&](int row, int col, float2 x, float top, float denom) {
            const int r = at.rb * ROWS + row, j = __umulhi(2 * r, a.group_inv);
            const long long to = ((long long)at.b * a.queries + j) * a.num_q_heads + at.head * a.group + r - j * a.group;
            const float inv = __fdividef(1.f, denom);
            x = denom == 0.f ? make_float2(0.f, 0.f) : make_float2(x.x * inv, x.y * inv);
            if (F32) *reinterpret_cast<float2*>(reinterpret_cast<float*>(a.output) + to * D + col) = x;
            else *reinterpret_cast<uint32_t*>(reinterpret_cast<__half*>(a.output) + to * D + col) = pack_half2(x.x, x.y);
            if (a.lse && col == 0) a.lse[to] = denom == 0.f ? -INFINITY : (top + kPagedShift + __log2f(denom)) * kLn2;
        };
        // Through the slots that the warps read last.  Columns of rows 2i, 2i + 1 are xored with 8 i: other banks.  A warp that
        // had no unit of the segment has no such slot, and no weight; one that gave up leaves what is there, under weights of NaN.
        const float gain = kScaled ? vref : 1.f;
        if (at.first + wi < at.end && !dead) {
            float* to = reinterpret_cast<float*>(ring + s_slot[warp] * S::SLOT) + t4 * 2 * D;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < KSTEPS; ++j) {
                    const float (&c)[4] = o[nt][j];
                    if (kScaled) {
                        float* at_ = to + nt * 8 * D + ((j * 16 + 2 * g4) ^ (t4 * 8));
                        *reinterpret_cast<float2*>(at_) = make_float2(c[0] * kPagedUnshift * gain, c[2] * kPagedUnshift * gain);
                        *reinterpret_cast<float2*>(at_ + D) = make_float2(c[1] * kPagedUnshift * gain, c[3] * kPagedUnshift * gain);
                    } else {
                        float* at_ = to + nt * 8 * D + ((j * 16 + g4) ^ (t4 * 8));
                        float* at8 = to + nt * 8 * D + ((j * 16 + 8 + g4) ^ (t4 * 8));
                        at_[0] = c[0] * kPagedUnshift; at8[0] = c[2] * kPagedUnshift;
                        at_[D] = c[1] * kPagedUnshift; at8[D] = c[3] * kPagedUnshift;
                    }
                }
        }
        group_barrier(gw, group);
#pragma unroll 1
        for (int i = gt; i < rows_here * (D / 2); i += gthreads) {
            const int row = i / (D / 2), col = i % (D / 2) * 2;
            float top = -INFINITY, denom = 0.f;
            float2 x = make_float2(0.f, 0.f);
#pragma unroll 1
            for (int w0 = 0; w0 < gw; w0 += 4) {            // four warps at a time, so that their reads are under way together
                float2 y[4];
                float2 v[4];
                float over = top;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int w = min(w0 + q, gw - 1);
                    y[q] = ml[w * ROWS + row];
                    v[q] = *reinterpret_cast<const float2*>(smem + (group * gw + w) * S::RING + s_slot[group * gw + w] * S::SLOT +
                                                            (row * D + (col ^ ((row >> 1 & 3) * 8))) * 4);
                    if (w0 + q >= gw) y[q] = make_float2(-INFINITY, 0.f);
                    over = fmaxf(over, y[q].x);
                }
                const float ref = over == -INFINITY ? 0.f : over, old = fast_exp2(top - ref);
                top = over;
                denom *= old;
                x.x *= old; x.y *= old;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float f = fast_exp2(y[q].x - ref);
                    denom += y[q].y * f;
                    if (y[q].y != 0.f) { x.x += v[q].x * f; x.y += v[q].y * f; }
                }
            }
            if (entire) put(row, col, x, top, denom);
            else {
                *reinterpret_cast<float2*>(a.part_o + (piece * ROWS + row) * D + col) = x;
                if (col == 0) reinterpret_cast<float2*>(a.part_ml)[piece * ROWS + row] = make_float2(top, denom);
            }
        }
        if (!entire) {
            const PagedCut cut = paged_cut(hi - at.left - at.first, at.units, per);
            const int mine_at = cut.start(worker);
#pragma unroll 1
            for (int level = 0; level < 2; ++level) {
                const int step = level ? cut.join : 1, start = level ? 0 : mine_at;
                const int count = cut.count(level, start);
                const bool done = level || cut.join == cut.n;
                int* counter = a.counters + (level ? 2 * kPagedMaxWorkers * grid : 0) + cut.place(start);
                group_barrier(gw, group);
                if (gt == 0) {
                    __threadfence();                        // for the whole worker: its stores are in front of the barrier
                    const bool last = atomicAdd(counter, 1) == count - 1;
                    s_last[group] = last;
                    if (last) *counter = 0;                 // ready for the next launch
                }
                group_barrier(gw, group);
                if (!s_last[group]) break;
                __threadfence();
                const float2* ml_from = reinterpret_cast<const float2*>(level ? a.part_ml2 : a.part_ml);
                // Four columns a thread, the pieces in order: eight reads of each on their way, as they come from L2 (sixteen take
                // registers that the main loop needs: 16 ragged int8 sequences of 256-wide heads 90 and 95 us).
#pragma unroll 1
                for (int i = gt; i < rows_here * (D / 4); i += gthreads) {
                    const int row = i / (D / 4), col = i % (D / 4) * 4;
                    float top = -INFINITY, denom = 0.f;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                    constexpr int AHEAD = 8;
#pragma unroll 1
                    for (int k0 = 0; k0 < count; k0 += AHEAD) {
                        float2 y[AHEAD];
                        float4 v[AHEAD];
#pragma unroll
                        for (int q = 0; q < AHEAD; ++q) {
                            y[q] = make_float2(-INFINITY, 0.f);
                            v[q] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (k0 + q < count) {
                                const int from = cut.place(start + (k0 + q) * step) * ROWS + row;
                                y[q] = __ldcg(ml_from + from);
                                v[q] = __ldcg(reinterpret_cast<const float4*>(a.part_o + from * D + col));
                            }
                        }
                        float over = top;
#pragma unroll
                        for (int q = 0; q < AHEAD; ++q) over = fmaxf(over, y[q].x);
                        const float ref = over == -INFINITY ? 0.f : over, old = fast_exp2(top - ref);
                        top = over;
                        denom *= old;
                        x.x *= old; x.y *= old; x.z *= old; x.w *= old;
#pragma unroll
                        for (int q = 0; q < AHEAD; ++q) {
                            const float f = fast_exp2(y[q].x - ref);
                            denom += y[q].y * f;
                            x.x += v[q].x * f; x.y += v[q].y * f; x.z += v[q].z * f; x.w += v[q].w * f;
                        }
                    }
                    if (done) {
                        put(row, col, make_float2(x.x, x.y), top, denom);
                        put(row, col + 2, make_float2(x.z, x.w), top, denom);
                    } else {                                // only this thread reads what it overwrites
                        const int to = cut.place(start) * ROWS + row;
                        *reinterpret_cast<float4*>(a.part_o + to * D + col) = x;
                        if (col == 0) reinterpret_cast<float2*>(a.part_ml2)[to] = make_float2(top, denom);
                    }
                }
                if (done) break;
            }
        }
        if (!next_segment(at)) break;
        fresh = true;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");             // the slot's next copies come behind these accesses
        group_barrier(gw, group);                           // what was merged has been read
        }
        if (room && !dead) fill();
    }
    }
    }

    // ---- rows of sequences without positions; positions that no table holds -------------------------------
    if (total > 0 && lives == a.batch && a.status == nullptr) return;
    for (int b = blockIdx.x * W + warp; b < a.batch; b += grid * W) {
        const int off = a.kv_offsets[b];
        if (lane == 0 && a.status && off >= (a.max_pages << a.page_log2)) *a.status = kStatusBadPosition;
        if (off >= 0) continue;
        const int rows = a.num_q_heads * a.queries;
        const long long first = (long long)b * rows;
        for (int i = lane; i < rows * (D / 4); i += 32) {
            if (F32) reinterpret_cast<float4*>(a.output)[first * (D / 4) + i] = make_float4(0.f, 0.f, 0.f, 0.f);
            else reinterpret_cast<uint2*>(a.output)[first * (D / 4) + i] = make_uint2(0u, 0u);
        }
        if (a.lse) for (int i = lane; i < rows; i += 32) a.lse[first + i] = -INFINITY;
    }
}

#endif  // __CUDACC__

}  // namespace vteb
