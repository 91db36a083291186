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
// workers.  A worker is `gw` of the eight warps of a CTA: the runs and `gw` are computed on the device from the step's
// own lengths.  Each warp of a worker takes every gw-th unit and has a ring of its own in shared memory, which its own
// lanes fill with tensor-map copies (one box a page) and which only it reads: no warp waits for another between the
// ends of segments, and the loads of the next segment are in flight while one is merged.
//
// Arithmetic.  Positions are the M dimension of both products (S^T = K Q^T, O^T = V^T P^T): a group of up to eight rows is
// one n8 tile, and what is converted from 8 bits to fp16 is the A operand, once for all rows.  ldmatrix on 8-bit rows
// delivers pairs of values; the order of channels inside a 16-channel step is free as long as Q (or the output column)
// follows, so K needs no shuffling at all and V one byte permute per four values.  e4m3 and int8 values are exact in
// fp16.  P is rounded to fp16 where the output is fp16, whose own rounding is as large; for fp32 output it is split into
// two fp16 parts.  Page scales never touch the stored values: ks multiplies the scores, vs (relative to the largest one
// so far, so that fp16 holds the product) the weights.
//
// Merging.  A segment's warps are merged through shared memory in warp order.  Segments that a worker border cuts leave
// (m, l, o) pieces in the workspace, and the last worker to arrive merges them in worker order: results do not depend on
// who is last.
#pragma once

#include "vteb_common.cuh"

namespace vteb {

constexpr int kPagedF16 = 0, kPagedE4m3 = 1, kPagedInt8 = 2;
constexpr int kStatusBadPage = 5;        // a block table entry outside 0..num_pages-1 for a position that is read or written
constexpr int kStatusBadPosition = 6;    // a position beyond the block table or the rotation tables

constexpr int kPagedWarps = 8;
constexpr int kPagedThreads = kPagedWarps * 32;
constexpr int kPagedRing = 24 * 1024;    // bytes of a warp's ring

struct PagedAttnArgs {
    KvTensorMap k_map, v_map;
    const __half* q;                 // [batch, queries, Hq, D]
    void* output;                    // same shape, fp16 or fp32
    float* lse;                      // [batch, queries, Hq] or null
    const int* block_table;          // [batch, max_pages]
    const int* kv_offsets;           // [batch]
    const float* k_scale;            // [num_pages, Hkv], 8-bit pages
    const float* v_scale;
    int* counters;                   // [workers], zero between launches: a cut segment's, at its first worker (no two share one)
    float* part_ml;                  // [2 * workers][rows][2]
    float* part_o;                   // [2 * workers][rows][D]
    int* status;
    int batch, max_pages, num_pages, page_log2, box_log2;
    int num_q_heads, num_kv_heads, group, queries, row_blocks;
    float scale_log2e;
};

template <int D, int KIND>
struct PagedShape {
    static constexpr int ES = KIND == kPagedF16 ? 2 : 1;
    static constexpr int RB = D * ES;                       // bytes of a row
    static constexpr int CB = RB < 128 ? RB : 128;          // bytes of a column block: the width of a box
    static constexpr int NC = RB / CB;
    static constexpr int U = RB == 64 ? 64 : RB <= 256 ? 32 : 16;      // positions of a unit
    static constexpr int SLOT = U * RB;
    static constexpr int NS = kPagedRing / SLOT;            // slots of a ring: K, V, K, V, ...
    static constexpr int MAXBOX = U / 16;
};

template <int NT> struct PagedMerge {                       // cross-warp merge, DC columns at a time
    static constexpr int ROWS = 8 * NT;
    static constexpr int DC = NT == 1 ? 64 : 32;
    static constexpr int LD = DC + 4;                       // rows 2i, 2i+1 of a fragment land on different banks
    static constexpr int WARP_FLOATS = ROWS * LD;
};

template <int NT>
__host__ __device__ constexpr int paged_smem_bytes() {
    // rings, merge buffers, per warp: (m, l) of its rows, scales of its slots, barriers
    return 1024 + kPagedWarps * (kPagedRing + PagedMerge<NT>::WARP_FLOATS * 4 + 8 * NT * 8 + 8 * 16 + 8 * 8);
}

#if defined(__CUDACC__)

__device__ __forceinline__ void tma_load_pages(uint32_t dst, const void* map, int y, int head, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(dst), "l"(map), "r"(0), "r"(y), "r"(0), "r"(head), "r"(page), "r"(bar)
        : "memory");
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

// Four 8-bit values to fp16, exactly: lo = values 0 and 1 of the word (2 and 3 with them in hi), or with `pairs` 0 and 2
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

// Byte offset inside a box of BR rows (column blocks one after another, swizzled) of 16-byte chunk `chunk` of row `r`.
template <int CB>
__device__ __forceinline__ uint32_t box_offset(int r, int chunk, int box_rows) {
    constexpr int PER = CB / 16;                            // chunks of a column block
    const int cb = chunk / PER, c = chunk % PER;
    const int x = CB == 128 ? (c ^ (r & 7)) : (c ^ ((r >> 1) & 3));
    return (uint32_t)(cb * box_rows * CB + r * CB + x * 16);
}

__device__ __forceinline__ void group_barrier(int gw, int group) {
    if (gw == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(gw * 32) : "memory");
}

// Where a warp is in its worker's run: unit `u` of segment (b, hr), of which units [first, end) are this worker's.
struct PagedCursor {
    int b, hr, u, first, end, units, len;
    long long left;                                         // units of the run from `first` on
};

__device__ __forceinline__ int paged_len(const PagedAttnArgs& a, int b) {
    const int room = a.max_pages << a.page_log2;            // at most 2^31 - 1, checked by the host
    const int off = __ldg(a.kv_offsets + b);
    return off < 0 ? 0 : off >= room ? room : off + 1;
}

template <int U>
__device__ __forceinline__ void cursor_enter(const PagedAttnArgs& a, PagedCursor& c) {   // first segment at or behind (b, hr) that has units
    c.len = paged_len(a, c.b);
    c.units = (c.len + U - 1) / U;
    while (c.units == 0 && c.b + 1 < a.batch) {
        c.len = paged_len(a, ++c.b);
        c.units = (c.len + U - 1) / U;
    }
    c.end = (long long)(c.units - c.first) < c.left ? c.units : c.first + (int)c.left;
}

template <int U>
__device__ __forceinline__ bool cursor_next_segment(const PagedAttnArgs& a, PagedCursor& c) {
    c.left -= c.end - c.first;
    if (c.left <= 0) return false;
    c.first = 0;
    if (++c.hr == a.num_kv_heads * a.row_blocks) {
        c.hr = 0;
        ++c.b;
        cursor_enter<U>(a, c);
    } else {
        c.end = (long long)c.units < c.left ? c.units : (int)c.left;
    }
    return true;
}

template <int D, int KIND, int NT, bool F32>
__global__ void __launch_bounds__(kPagedThreads, 1) paged_attention_kernel(const __grid_constant__ PagedAttnArgs a)
{
    using S = PagedShape<D, KIND>;
    using M = PagedMerge<NT>;
    constexpr int U = S::U, RB = S::RB, CB = S::CB, NS = S::NS, SLABS = U / 16, KSTEPS = D / 16, ROWS = 8 * NT;
    constexpr bool kScaled = KIND != kPagedF16;

    extern __shared__ unsigned char smem_raw[];
    __shared__ long long s_scan[kPagedWarps];
    __shared__ int s_live[kPagedWarps];
    __shared__ int s_start_b[kPagedWarps];
    __shared__ long long s_start_rest[kPagedWarps];
    __shared__ int s_last[kPagedWarps];
    __shared__ float s_denom[kPagedWarps][ROWS];            // of the rows of each worker's segment

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    unsigned char* ring = smem + warp * kPagedRing;
    float* merge_all = reinterpret_cast<float*>(smem + kPagedWarps * kPagedRing);
    float2* ml_all = reinterpret_cast<float2*>(merge_all + kPagedWarps * M::WARP_FLOATS);
    float* scales = reinterpret_cast<float*>(ml_all + kPagedWarps * ROWS) + warp * 32;         // [slot][4]
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(reinterpret_cast<float*>(ml_all + kPagedWarps * ROWS) + kPagedWarps * 32) + warp * 8;
    const uint32_t ring_u = smem_u32(ring), bars_u = smem_u32(bars), scales_u = smem_u32(scales);

    const int box_rows = 1 << a.box_log2;
    const int boxes = U >> a.box_log2;                      // of a unit
    if (lane == 0) {
        for (int i = 0; i < NS; ++i) mbar_init(bars_u + i * 8, 1 + (kScaled ? boxes : 0));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }

    // ---- all units, and where this CTA's workers begin ------------------------------------------
    const int HR = a.num_kv_heads * a.row_blocks;
    const int per_thread = (a.batch + kPagedThreads - 1) / kPagedThreads;
    const int b0 = min(tid * per_thread, a.batch), b1 = min(b0 + per_thread, a.batch);
    long long mine = 0;
    int live = 0;
    for (int b = b0; b < b1; ++b) {
        const int units = (paged_len(a, b) + U - 1) / U;
        mine += units;
        live += units > 0;
        if (blockIdx.x == 0 && a.status && __ldg(a.kv_offsets + b) >= (a.max_pages << a.page_log2)) *a.status = kStatusBadPosition;
    }
    long long upto = mine;
    int live_upto = live;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long x = __shfl_up_sync(~0u, upto, d);
        const int y = __shfl_up_sync(~0u, live_upto, d);
        if (lane >= d) { upto += x; live_upto += y; }
    }
    if (lane == 31) { s_scan[warp] = upto; s_live[warp] = live_upto; }
    __syncthreads();
    long long total = 0;
    int lives = 0;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) {
        if (w < warp) upto += s_scan[w];
        total += s_scan[w];
        lives += s_live[w];
    }
    total *= HR;
    // Warps of a worker.
    const long long segments = (long long)lives * HR;
    int gw = kPagedWarps;
    while (gw > 1 && segments * 4 >= (long long)gridDim.x * (kPagedWarps / gw) * 2 &&
           (total >= (long long)gridDim.x * (kPagedWarps / gw) * 2 * 16 || total < segments * gw)) gw >>= 1;
    const int groups = kPagedWarps / gw, group = warp / gw, wi = warp % gw;
    long long workers = (long long)gridDim.x * groups;
    const long long useful = (total + 2 * gw - 1) / (2 * gw);
    if (workers > useful) workers = useful > 0 ? useful : 1;
    const int worker = blockIdx.x * groups + group;
    for (int g = 0; g < groups; ++g) {
        const long long w = (long long)blockIdx.x * groups + g;
        if (w >= workers) break;
        const long long lo = w * total / workers;
        if (lo >= (upto - mine) * HR && lo < upto * HR) {
            long long rest = lo - (upto - mine) * HR;
            int b = b0;
            for (; b < b1; ++b) {
                const long long n = (long long)((paged_len(a, b) + U - 1) / U) * HR;
                if (rest < n) break;
                rest -= n;
            }
            s_start_b[g] = b;
            s_start_rest[g] = rest;
        }
    }
    __syncthreads();

    // ---- sequences without positions: zero rows ---------------------------------------------------
    const int out_row = a.num_q_heads * a.queries;          // rows of a sequence
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        if (paged_len(a, b) > 0) continue;
        const long long base = (long long)b * out_row * D;
        for (int i = tid; i < out_row * D; i += kPagedThreads) {
            if (F32) reinterpret_cast<float*>(a.output)[base + i] = 0.f;
            else reinterpret_cast<__half*>(a.output)[base + i] = __float2half(0.f);
        }
        if (a.lse) for (int i = tid; i < out_row; i += kPagedThreads) a.lse[(long long)b * out_row + i] = -INFINITY;
    }
    if (worker >= workers || total == 0) return;

    const long long lo = (long long)worker * total / workers, hi = (long long)(worker + 1) * total / workers;
    PagedCursor at;                                         // what this warp computes
    at.b = s_start_b[group];
    at.left = hi - lo;
    {
        const long long rest = s_start_rest[group];
        const int units = (paged_len(a, at.b) + U - 1) / U;
        at.hr = (int)(rest / units);
        at.first = (int)(rest % units);
    }
    if (at.left <= 0) return;
    cursor_enter<U>(a, at);
    PagedCursor ahead = at;                                 // the unit whose table entries are asked for
    ahead.u = ahead.first + wi;
    bool more = true;
    while (more && ahead.u >= ahead.end) { more = cursor_next_segment<U>(a, ahead); ahead.u = ahead.first + wi; }

    // ---- the ring -----------------------------------------------------------------------------------
    struct Pending { int page, y, need, head; bool ok; } cur, nxt;
    cur.page = cur.y = cur.need = cur.head = 0; cur.ok = false;
    auto look_up = [&]() {                                  // table entries of `ahead`, one box a lane
        nxt.ok = more;
        if (!more) return;
        const int pos = ahead.u * U + (lane << a.box_log2);
        nxt.need = min(boxes, (ahead.len - ahead.u * U + box_rows - 1) >> a.box_log2);
        nxt.head = ahead.hr / a.row_blocks;
        nxt.y = pos & ((1 << a.page_log2) - 1);
        nxt.page = lane < nxt.need ? __ldg(a.block_table + (long long)ahead.b * a.max_pages + (pos >> a.page_log2)) : 0;
        ahead.u += gw;
        while (more && ahead.u >= ahead.end) { more = cursor_next_segment<U>(a, ahead); ahead.u = ahead.first + wi; }
    };
    int item = 0, fill_slot = 0;                            // next item to ask for: K of a unit, V of it, K of the next ...
    auto fill = [&]() {
        const bool is_v = item & 1;
        ++item;
        if (!is_v) { cur = nxt; look_up(); }
        if (!cur.ok) return;
        const uint32_t bar = bars_u + fill_slot * 8, dst = ring_u + fill_slot * S::SLOT;
        int page = cur.page;
        const bool bad = (unsigned)page >= (unsigned)a.num_pages;
        if (bad) page = 0;
        if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(cur.need * box_rows * RB));
        __syncwarp();
        if (lane < boxes) {
            const uint32_t sc = scales_u + (fill_slot * 4 + lane) * 4;
            if (lane < cur.need) {
                tma_load_pages(dst + lane * box_rows * RB, is_v ? &a.v_map : &a.k_map, cur.y, cur.head, page, bar);
                if (bad && a.status) *a.status = kStatusBadPage;
            }
            if (kScaled && lane < cur.need && !bad) {
                const float* src = (is_v ? a.v_scale : a.k_scale) + (long long)page * a.num_kv_heads + cur.head;
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sc), "l"(src) : "memory");
            } else {                                        // a page that is not there makes its sequence's rows NaN
                scales[fill_slot * 4 + lane] = bad ? NAN : 1.f;
            }
            if (kScaled) async_copy_arrive(bar);
        }
        if (++fill_slot == NS) fill_slot = 0;
    };
    look_up();
#pragma unroll 1
    for (int i = 0; i < NS; ++i) fill();

    int slot = 0;
    uint32_t phase = 0;
    bool dead = false;
    auto wait_slot = [&]() {
        if (!dead && !mbar_wait_bounded(bars_u + slot * 8, phase, nullptr)) {
            dead = true;
            if (a.status) *a.status = kStatusFullTimeout;
        }
        __syncwarp();
    };
    auto release_slot = [&]() {                             // read by every lane; filled anew
        if (++slot == NS) { slot = 0; phase ^= 1; }
        __syncwarp();
        if (!dead) fill();
    };

    const int g4 = lane >> 2, t4 = lane & 3;
    const int mrow = (lane & 7) + ((lane >> 3) & 1) * 8;    // ldmatrix row and chunk of this lane: K, and V of 8-bit pages
    const int mchunk = lane >> 4;
    const int vrow = (lane & 7) + (lane >> 4) * 8;          // V of 16-bit pages
    const int vchunk = (lane >> 3) & 1;

    // ---- segments -------------------------------------------------------------------------------------
    for (;;) {
        const int head = at.hr / a.row_blocks, rb = at.hr - head * a.row_blocks;
        const int rows_all = a.queries * a.group;
        // Q of row n (this lane: n = g4) as B operand
        uint32_t qf[NT][KSTEPS][2];
        int limit[NT][2];                                   // positions that the rows of this lane's columns see
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = rb * ROWS + nt * 8 + g4;
            const int j = r / a.group, g = r - j * a.group;
            const __half* src = a.q + (((long long)at.b * a.queries + j) * a.num_q_heads + head * a.group + g) * D;
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks) {
                if (r < rows_all) {
                    if (kScaled) {
                        const uint2 x = __ldg(reinterpret_cast<const uint2*>(src + ks * 16 + t4 * 4));
                        qf[nt][ks][0] = x.x; qf[nt][ks][1] = x.y;
                    } else {
                        qf[nt][ks][0] = __ldg(reinterpret_cast<const uint32_t*>(src + ks * 16 + t4 * 2));
                        qf[nt][ks][1] = __ldg(reinterpret_cast<const uint32_t*>(src + ks * 16 + 8 + t4 * 2));
                    }
                } else qf[nt][ks][0] = qf[nt][ks][1] = 0;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int rr = rb * ROWS + nt * 8 + t4 * 2 + e;
                limit[nt][e] = rr < rows_all ? at.len - a.queries + 1 + rr / a.group : 0;
            }
        }
        float m[NT][2], l[NT][2], o[NT][KSTEPS][4], vref = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int j = 0; j < KSTEPS; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
        }
        const int whole = at.len - a.queries + 1;           // positions that every row sees

#pragma unroll 1
        for (int u = at.first + wi; u < at.end; u += gw) {
            const bool ragged = (u + 1) * U > whole;
            // scores
            float s[SLABS][NT][4];
#pragma unroll
            for (int sl = 0; sl < SLABS; ++sl)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[sl][nt][0] = s[sl][nt][1] = s[sl][nt][2] = s[sl][nt][3] = 0.f;
            wait_slot();
            {
                const uint32_t base = ring_u + slot * S::SLOT;
                uint32_t slab_at[SLABS];
                int slab_r[SLABS];
                float ks_[SLABS];
#pragma unroll
                for (int sl = 0; sl < SLABS; ++sl) {
                    const int box = (sl * 16) >> a.box_log2;
                    slab_at[sl] = base + box * box_rows * RB;
                    slab_r[sl] = ((sl * 16) & (box_rows - 1)) + mrow;
                    ks_[sl] = scales[slot * 4 + box] * a.scale_log2e;
                }
                if constexpr (kScaled) {
#pragma unroll
                    for (int ks = 0; ks < KSTEPS; ks += 2)
#pragma unroll
                        for (int sl = 0; sl < SLABS; ++sl) {
                            uint32_t r0, r1, r2, r3, f0, f1, f2, f3;
                            ldmatrix_x4(slab_at[sl] + box_offset<CB>(slab_r[sl], ks + mchunk, box_rows), r0, r1, r2, r3);
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
                    for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
                        for (int sl = 0; sl < SLABS; ++sl) {
                            uint32_t f0, f1, f2, f3;
                            ldmatrix_x4(slab_at[sl] + box_offset<CB>(slab_r[sl], ks * 2 + mchunk, box_rows), f0, f1, f2, f3);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma_16816(s[sl][nt], f0, f1, f2, f3, qf[nt][ks][0], qf[nt][ks][1]);
                        }
                }
#pragma unroll
                for (int sl = 0; sl < SLABS; ++sl)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[sl][nt][e] *= ks_[sl];
                            if (ragged && u * U + sl * 16 + g4 + (e >> 1) * 8 >= limit[nt][e & 1]) s[sl][nt][e] = -INFINITY;
                        }
            }
            release_slot();

            // running maximum and sum
            float alpha[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = m[nt][e];
#pragma unroll
                    for (int sl = 0; sl < SLABS; ++sl) top = fmaxf(top, fmaxf(s[sl][nt][e], s[sl][nt][e + 2]));
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
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

            wait_slot();
            {
                const uint32_t base = ring_u + slot * S::SLOT;
                if constexpr (kScaled) {
                    // weights relative to the largest scale so far
                    float vs[SLABS], top = vref;
#pragma unroll
                    for (int sl = 0; sl < SLABS; ++sl) {
                        const int box = (sl * 16) >> a.box_log2;
                        const bool there = u * U + sl * 16 < at.len;
                        vs[sl] = there ? scales[slot * 4 + box] : 0.f;
                        if (!(fabsf(vs[sl]) < INFINITY)) vs[sl] = NAN;
                        top = fmaxf(top, vs[sl]);
                    }
                    const float shrink = top > 0.f ? vref / top : 1.f;
                    const float inv = top > 0.f ? 1.f / top : 0.f;
                    vref = top;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        alpha[nt][0] *= shrink;
                        alpha[nt][1] *= shrink;
#pragma unroll
                        for (int sl = 0; sl < SLABS; ++sl)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                s[sl][nt][e] = (ragged && s[sl][nt][e] == 0.f) ? 0.f : s[sl][nt][e] * (vs[sl] * inv);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < KSTEPS; ++j) {
                        o[nt][j][0] *= alpha[nt][0]; o[nt][j][1] *= alpha[nt][1];
                        o[nt][j][2] *= alpha[nt][0]; o[nt][j][3] *= alpha[nt][1];
                    }
#pragma unroll
                for (int sl = 0; sl < SLABS; ++sl) {
                    uint32_t p[NT][2], pl[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float x = s[sl][nt][2 * e], y = s[sl][nt][2 * e + 1];
                            const uint32_t h = pack_half2(x, y);
                            p[nt][e] = transpose_8x8(h);
                            if (F32) {
                                const float2 back = unpack_half2(h);
                                pl[nt][e] = transpose_8x8(pack_half2(x - back.x, y - back.y));
                            }
                        }
                    const int box = (sl * 16) >> a.box_log2;
                    const uint32_t at_ = base + box * box_rows * RB;
                    const int r0_ = (sl * 16) & (box_rows - 1);
                    // two 16-channel steps of V^T: (f[0..3]) and, of 8-bit pages, (f[4..7])
                    auto load_v = [&](int j, uint32_t (&f)[8]) {
                        if constexpr (kScaled) {
                            uint32_t x0, x1, x2, x3;
                            ldmatrix_x4_trans(at_ + box_offset<CB>(r0_ + mrow, j + mchunk, box_rows), x0, x1, x2, x3);
                            widen<KIND, true>(x0, f[0], f[1]);
                            widen<KIND, true>(x1, f[2], f[3]);
                            widen<KIND, true>(x2, f[4], f[5]);
                            widen<KIND, true>(x3, f[6], f[7]);
                        } else {
                            ldmatrix_x4_trans(at_ + box_offset<CB>(r0_ + vrow, j * 2 + vchunk, box_rows), f[0], f[1], f[2], f[3]);
                            ldmatrix_x4_trans(at_ + box_offset<CB>(r0_ + vrow, j * 2 + 2 + vchunk, box_rows), f[4], f[5], f[6], f[7]);
                        }
                    };
                    if (!ragged) {
#pragma unroll
                        for (int j = 0; j < KSTEPS; j += 2) {
                            uint32_t f[8];
                            load_v(j, f);
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
                    } else {
                        // What a row does not see may be anything: each query token of the block is multiplied with the positions
                        // behind its limit set to zero, and its own columns are kept.
                        const int pos = u * U + sl * 16 + t4 * 2;
                        const int jlo = rb * ROWS / a.group, jhi = min(a.queries - 1, (rb * ROWS + ROWS - 1) / a.group);
#pragma unroll 1
                        for (int qj = jlo; qj <= jhi; ++qj) {
                            const int lim = at.len - a.queries + 1 + qj;
                            if (u * U + sl * 16 >= lim) continue;
                            const uint32_t k0 = (pos < lim ? 0xffffu : 0u) | (pos + 1 < lim ? 0xffff0000u : 0u);
                            const uint32_t k1 = (pos + 8 < lim ? 0xffffu : 0u) | (pos + 9 < lim ? 0xffff0000u : 0u);
#pragma unroll
                            for (int j = 0; j < KSTEPS; j += 2) {
                                uint32_t f[8];
                                load_v(j, f);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                    for (int h = 0; h < 2; ++h) {
                                        float c[4] = {0.f, 0.f, 0.f, 0.f};
                                        mma_16816(c, f[4 * h] & k0, f[4 * h + 1] & k0, f[4 * h + 2] & k1, f[4 * h + 3] & k1, p[nt][0], p[nt][1]);
                                        if (F32) mma_16816(c, f[4 * h] & k0, f[4 * h + 1] & k0, f[4 * h + 2] & k1, f[4 * h + 3] & k1, pl[nt][0], pl[nt][1]);
                                        if (limit[nt][0] == lim) { o[nt][j + h][0] += c[0]; o[nt][j + h][2] += c[2]; }
                                        if (limit[nt][1] == lim) { o[nt][j + h][1] += c[1]; o[nt][j + h][3] += c[3]; }
                                    }
                            }
                        }
                    }
                }
            }
            release_slot();
        }

        // ---- end of the segment: the warps of the worker --------------------------------------------
        const bool entire = at.first == 0 && at.end == at.units;
        float gain[NT][2], big[NT][2], sum_l[NT][2];
        float2* ml = ml_all + warp * ROWS;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = l[nt][e];
                x += __shfl_xor_sync(~0u, x, 4);
                x += __shfl_xor_sync(~0u, x, 8);
                x += __shfl_xor_sync(~0u, x, 16);
                if (g4 == 0) ml[nt * 8 + t4 * 2 + e] = make_float2(m[nt][e], x);
            }
        group_barrier(gw, group);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = nt * 8 + t4 * 2 + e;
                float top = -INFINITY, sum = 0.f;
                for (int w = 0; w < gw; ++w) top = fmaxf(top, ml_all[(group * gw + w) * ROWS + row].x);
                const float ref = top == -INFINITY ? 0.f : top;
                for (int w = 0; w < gw; ++w) {
                    const float2 x = ml_all[(group * gw + w) * ROWS + row];
                    sum += x.y * fast_exp2(x.x - ref);
                }
                gain[nt][e] = fast_exp2(m[nt][e] - ref) * (kScaled ? vref : 1.f);
                big[nt][e] = top;
                sum_l[nt][e] = sum;
            }
        // this worker's piece of a cut segment: slot 0 for the one its run begins with, 1 for the one it ends with
        const bool has_first = at.left == hi - lo;
        const long long piece = 2ll * worker + (has_first ? 0 : 1);
        float* my_o = a.part_o + piece * ROWS * D;
        if (wi == 0 && g4 == 0) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                s_denom[group][nt * 8 + t4 * 2] = sum_l[nt][0];
                s_denom[group][nt * 8 + t4 * 2 + 1] = sum_l[nt][1];
            }
        }
        if (!entire && wi == 0 && g4 == 0) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    reinterpret_cast<float2*>(a.part_ml)[piece * ROWS + nt * 8 + t4 * 2 + e] = make_float2(big[nt][e], sum_l[nt][e]);
        }
        if (entire && a.lse && wi == 0 && g4 == 0) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = rb * ROWS + nt * 8 + t4 * 2 + e;
                    if (r < rows_all) {
                        const int j = r / a.group;
                        a.lse[((long long)at.b * a.queries + j) * a.num_q_heads + head * a.group + r - j * a.group] =
                            sum_l[nt][e] == 0.f ? -INFINITY : (big[nt][e] + log2f(sum_l[nt][e])) * kLn2;
                    }
                }
        }
        float* buf = merge_all + warp * M::WARP_FLOATS;
        const float* buf0 = merge_all + group * gw * M::WARP_FLOATS;
        const int gt = wi * 32 + lane;                      // thread of the worker
        auto put = [&](int row, int col, float x, float y, float denom) {
            const int r = rb * ROWS + row;
            if (r >= rows_all) return;
            const float inv = denom == 0.f ? 0.f : 1.f / denom;
            x = denom == 0.f ? 0.f : x * inv;
            y = denom == 0.f ? 0.f : y * inv;
            const int j = r / a.group;
            const long long to = (((long long)at.b * a.queries + j) * a.num_q_heads + head * a.group + r - j * a.group) * D + col;
            if (F32) *reinterpret_cast<float2*>(reinterpret_cast<float*>(a.output) + to) = make_float2(x, y);
            else *reinterpret_cast<__half2*>(reinterpret_cast<__half*>(a.output) + to) = __floats2half2_rn(x, y);
        };
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += M::DC) {
            if (d0) group_barrier(gw, group);
#pragma unroll
            for (int j = 0; j < M::DC / 16; ++j)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float (&c)[4] = o[nt][d0 / 16 + j];
                    float* to = buf + (nt * 8 + t4 * 2) * M::LD + j * 16;
                    if (kScaled) {
                        *reinterpret_cast<float2*>(to + 2 * g4) = make_float2(c[0] * gain[nt][0], c[2] * gain[nt][0]);
                        *reinterpret_cast<float2*>(to + M::LD + 2 * g4) = make_float2(c[1] * gain[nt][1], c[3] * gain[nt][1]);
                    } else {
                        to[g4] = c[0] * gain[nt][0]; to[g4 + 8] = c[2] * gain[nt][0];
                        to[M::LD + g4] = c[1] * gain[nt][1]; to[M::LD + g4 + 8] = c[3] * gain[nt][1];
                    }
                }
            group_barrier(gw, group);
            for (int i = gt; i < ROWS * M::DC / 2; i += gw * 32) {
                const int row = i / (M::DC / 2), col = i % (M::DC / 2) * 2;
                float x = 0.f, y = 0.f;
                for (int w = 0; w < gw; ++w) {
                    const float2 v = *reinterpret_cast<const float2*>(buf0 + w * M::WARP_FLOATS + row * M::LD + col);
                    x += v.x; y += v.y;
                }
                if (entire) {
                    put(row, d0 + col, x, y, s_denom[group][row]);
                } else {
                    *reinterpret_cast<float2*>(my_o + row * D + d0 + col) = make_float2(x, y);
                }
            }
        }
        if (!entire) {
            // the workers whose runs hold units of this segment
            const long long begin = lo + (hi - lo - at.left) - at.first;       // its first unit, of all
            const long long w0 = ((begin + 1) * workers - 1) / total, w1 = ((begin + at.units) * workers - 1) / total;
            __threadfence();
            group_barrier(gw, group);
            if (gt == 0) {
                const int before = atomicAdd(a.counters + w0, 1);
                s_last[group] = before == (int)(w1 - w0);
                if (before == (int)(w1 - w0)) a.counters[w0] = 0;             // ready for the next launch
            }
            group_barrier(gw, group);
            if (s_last[group]) {
                __threadfence();
                const int n = (int)(w1 - w0) + 1;
                const long long p0 = 2 * w0 + (w0 * total / workers == begin ? 0 : 1);
                auto piece_of = [&](int k) { return k == 0 ? p0 : 2 * (w0 + k); };
                for (int i = gt; i < ROWS * D / 4; i += gw * 32) {
                    const int row = i / (D / 4), col = i % (D / 4) * 4;
                    float top = -INFINITY, denom = 0.f;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                    for (int k = 0; k < n; ++k) top = fmaxf(top, __ldcg(a.part_ml + (piece_of(k) * ROWS + row) * 2));
                    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 4
                    for (int k = 0; k < n; ++k) {
                        const float2 v = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + piece_of(k) * ROWS + row);
                        const float4 c = __ldcg(reinterpret_cast<const float4*>(a.part_o + (piece_of(k) * ROWS + row) * D + col));
                        const float f = fast_exp2(v.x - ref);
                        denom += v.y * f;
                        x.x += c.x * f; x.y += c.y * f; x.z += c.z * f; x.w += c.w * f;
                    }
                    put(row, col, x.x, x.y, denom);
                    put(row, col + 2, x.z, x.w, denom);
                    const int r = rb * ROWS + row;
                    if (a.lse && col == 0 && r < rows_all) {
                        const int j = r / a.group;
                        a.lse[((long long)at.b * a.queries + j) * a.num_q_heads + head * a.group + r - j * a.group] =
                            denom == 0.f ? -INFINITY : (top + log2f(denom)) * kLn2;
                    }
                }
            }
        }
        group_barrier(gw, group);                           // the merge buffers are free again
        if (!cursor_next_segment<U>(a, at)) break;
    }
}

#endif  // __CUDACC__

}  // namespace vteb
