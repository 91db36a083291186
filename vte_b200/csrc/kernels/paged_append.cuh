// Appending keys and values to a paged cache, with the position rotation of K (and of Q beside it) on the way.
//
// A block takes the new tokens of one page of one sequence for one KV head, of K or of V: it reads the fp16 rows, rotates
// them in fp32 (each product rounded, as rope_kernel does) and rounds to fp16, which is what a 16-bit page stores.  For
// 8-bit pages the block then knows the largest magnitude of its tokens, and with the page's scale so far the new scale
//
//   need = amax / 448 (e4m3) or / 127 (int8),  scale = max(older tokens in the page ? |old scale| : 0, need) with the old one's sign,
//   stored = round(x * (1 / scale)),  older tokens, where the scale grew: round(stored * (old / scale)),
//
// all in fp32 with correctly rounded divisions, ties to even.  A value that is not finite makes the scale NaN, and with it
// every result that reads the page.  Blocks behind those of K and V rotate Q.
//
// Bound by bytes on their way for prompts (each value is read once, for 8-bit pages a second time from L1 or L2, and written
// once: a prompt into e4m3 pages fills 61 % of the issue slots, chunks into int8 pages 67 %, and the warps wait for loads), by latency
// for single tokens: 1.9 us in fp16 and 2.4 in e4m3 pages, a launch behind another in a graph.
#pragma once

#include "vteb_common.cuh"

namespace vteb {

struct PagedAppendArgs {
    const __half *k, *v, *q;             // [tokens, heads, D], rows of a token side by side
    __half* q_out;
    void *k_pool, *v_pool;
    float *k_scale, *v_scale;            // [num_pages, Hkv]
    const int *block_table, *kv_offsets, *token_starts;    // token_starts null: the same number of tokens each
    const __half *cos_table, *sin_table;
    int* status;
    long long k_stride, v_stride, q_stride, q_out_stride;  // halves between tokens
    long long page_stride, token_stride, head_stride;      // values
    int batch, max_pages, num_pages, page_log2, total_tokens, each;
    int num_q_heads, num_kv_heads, dim_log2;
    int rope_type, rotary_dim, rope_rows;
    int kv_blocks;                       // blocks of K and V, in front of those of Q
    int q_heads_each;                    // heads of Q a thread, a divisor of num_q_heads
};

#if defined(__CUDACC__)

// 16 channels of a row as 8 + 8: the two halves of eight rotated pairs, or 16 channels side by side.
struct ChannelTask { int a, b, entry; bool rotated, adjacent; };

__device__ __forceinline__ ChannelTask channel_task(int pv, int D, int rope_type, int rotary_dim) {
    ChannelTask t;
    const int rot = rope_type == 2 ? rotary_dim : D;
    t.rotated = rope_type >= 0 && pv * 16 < rot;
    t.adjacent = rope_type == 1;
    if (t.rotated && !t.adjacent) { t.a = pv * 8; t.b = (rot >> 1) + pv * 8; }
    else { t.a = pv * 16; t.b = t.a + 8; }
    t.entry = pv * 8;
    return t;
}

__device__ __forceinline__ void rotate_task(const ChannelTask& t, uint4& xa, uint4& xb, uint4 c4, uint4 s4) {
    uint32_t* a = reinterpret_cast<uint32_t*>(&xa);
    uint32_t* b = reinterpret_cast<uint32_t*>(&xb);
    const uint32_t* cw = reinterpret_cast<const uint32_t*>(&c4);
    const uint32_t* sw = reinterpret_cast<const uint32_t*>(&s4);
    float y[16];
    if (t.adjacent) {                    // pair i: channels 2i, 2i + 1 of the sixteen
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 x = unpack_half2(i < 4 ? a[i] : b[i - 4]);
            const float2 c = unpack_half2(cw[i >> 1]), s = unpack_half2(sw[i >> 1]);
            rope_pair(x.x, x.y, (i & 1) ? c.y : c.x, (i & 1) ? s.y : s.x, y[2 * i], y[2 * i + 1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 lo = unpack_half2(a[i]), hi = unpack_half2(b[i]), c = unpack_half2(cw[i]), s = unpack_half2(sw[i]);
            rope_pair(lo.x, hi.x, c.x, s.x, y[2 * i], y[8 + 2 * i]);
            rope_pair(lo.y, hi.y, c.y, s.y, y[2 * i + 1], y[8 + 2 * i + 1]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) { a[i] = pack_half2(y[2 * i], y[2 * i + 1]); b[i] = pack_half2(y[8 + 2 * i], y[9 + 2 * i]); }
}

// The token range of sequence b, and the position of its first token.
__device__ __forceinline__ void token_range(const PagedAppendArgs& p, int b, int& first, int& count) {
    if (p.token_starts) {
        const int lo = p.token_starts[b], hi = p.token_starts[b + 1];
        first = min(max(lo, 0), p.total_tokens);
        count = max(min(hi, p.total_tokens) - first, 0);
    } else {
        first = b * p.each;
        count = p.each;
    }
}

// Four fp32 values to four 8-bit ones.
template <int KIND>
__device__ __forceinline__ uint32_t narrow4(float x, float y, float z, float w) {
    if constexpr (KIND == 1) {
        uint32_t r;
        asm("{\n .reg .b16 l, h;\n cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n mov.b32 %0, {l, h};\n}"
            : "=r"(r) : "f"(x), "f"(y), "f"(z), "f"(w));
        return r;
    } else {
        // (-128 only where a page that came from elsewhere held it: x * (1 / scale) rounds to 127 at most)
        auto one = [](float v) { return (uint32_t)(min(max(__float2int_rn(v), -128), 127)) & 0xffu; };
        return one(x) | one(y) << 8 | one(z) << 16 | one(w) << 24;
    }
}

template <int KIND>
__device__ __forceinline__ void widen4(uint32_t w, float (&x)[4]) {
    if constexpr (KIND == 1) {
        uint32_t lo, hi;
        asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}" : "=r"(lo), "=r"(hi) : "r"(w));
        const float2 a = unpack_half2(lo), b = unpack_half2(hi);
        x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)(int)(signed char)(w >> (8 * i));
    }
}

template <int KIND>
__device__ __forceinline__ uint2 quantise8(uint4 x, float inv) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
    float2 f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = unpack_half2(w[i]);
        f[i].x = __fmul_rn(f[i].x, inv);
        f[i].y = __fmul_rn(f[i].y, inv);
    }
    return make_uint2(narrow4<KIND>(f[0].x, f[0].y, f[1].x, f[1].y), narrow4<KIND>(f[2].x, f[2].y, f[3].x, f[3].y));
}

// KIND 0: fp16 pages, 1: e4m3, 2: int8.  One 16-channel task of K and V a thread at a time and two of Q, whose position, table rows
// and conversions are then looked up once; 8-bit pages read all but a thread's last task a second time, from L1 or L2, rather than
// hold them.  Registers with next to no spills (8 bytes in the fp16 build) come before more blocks an SM.  A 32,768-token prompt of 12
// query and 2 KV heads of 128 into e4m3 pages: 48.3 us, 52.7 with one task of Q a thread (prompts into fp16 pages 36.9 and 39.7);
// when blocks and tasks were chosen, side by side, 46.5, with seven blocks of spilling threads 54.5 and with four tasks 52.
template <int KIND>
__global__ void __launch_bounds__(256, 5) paged_append_kernel(const __grid_constant__ PagedAppendArgs p)
{
    const int D = 1 << p.dim_log2, tasks_log2 = p.dim_log2 - 4, P = 1 << p.page_log2;
    const int tid = threadIdx.x, T = blockDim.x;
    // Nothing of the launches in front is touched before this; the launch behind may start when they are complete.  Ordinary loads
    // throughout: a non-coherent one may be moved ahead of the wait, and is not for what is written while the block is there.
    grid_dependency_wait();
    grid_launch_dependents();
    if ((int)blockIdx.x >= p.kv_blocks) {                   // ---- Q
        // the same sixteen channels of `q_heads_each` heads of a token: one look at its position and its table rows
        const int groups = p.num_q_heads / p.q_heads_each;
        const long long all = ((long long)p.total_tokens * groups) << tasks_log2;
        const long long at = (long long)(blockIdx.x - p.kv_blocks) * T + tid;
        if (at >= all) return;
        const int pv = (int)at & ((1 << tasks_log2) - 1);
        const unsigned row = (unsigned)(at >> tasks_log2), token = row / (unsigned)groups;
        const int head = (row - token * groups) * p.q_heads_each;
        const ChannelTask t = channel_task(pv, D, p.rope_type, p.rotary_dim);
        const __half* src = p.q + token * p.q_stride + head * D;
        uint4 xa = *reinterpret_cast<const uint4*>(src + t.a), xb = *reinterpret_cast<const uint4*>(src + t.b);   // on their way while the position is looked up
        int b;
        if (p.token_starts) {
            int lo = 0, hi = p.batch;                   // the last sequence that starts at or before the token
            while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (p.token_starts[mid] <= (int)token) lo = mid; else hi = mid; }
            b = lo;
        } else b = p.each == 1 ? token : token / p.each;
        int first, count;
        token_range(p, b, first, count);
        const int end = p.kv_offsets[b], pos = end - (first + count - 1 - (int)token);
        if ((int)token < first || (int)token >= first + count || end < 0 || pos < 0 || (p.rope_type >= 0 && pos >= p.rope_rows)) return;
        uint4 c = make_uint4(0, 0, 0, 0), s = c;
        if (t.rotated) {
            const long long e = (long long)pos * (p.rope_type == 2 ? p.rotary_dim : D) + t.entry;
            c = *reinterpret_cast<const uint4*>(p.cos_table + e);
            s = *reinterpret_cast<const uint4*>(p.sin_table + e);
        }
        __half* dst = p.q_out + token * p.q_out_stride + head * D;
#pragma unroll 1
        for (int h = 0;;) {
            if (t.rotated) rotate_task(t, xa, xb, c, s);
            *reinterpret_cast<uint4*>(dst + t.a) = xa;
            *reinterpret_cast<uint4*>(dst + t.b) = xb;
            if (++h == p.q_heads_each) break;
            src += D;
            dst += D;
            xa = *reinterpret_cast<const uint4*>(src + t.a);
            xb = *reinterpret_cast<const uint4*>(src + t.b);
        }
        return;
    }

    // ---- K or V of one page
    const bool is_v = blockIdx.x & 1;
    const int unit = blockIdx.x >> 1;
    const int h = unit % p.num_kv_heads, x = unit / p.num_kv_heads;
    int b, chunk;
    if (p.token_starts) {
        // pages of sequence b: slots token_starts[b] / P + 2 b on, as n tokens touch at most n / P + 2 pages
        int lo = 0, hi = p.batch;
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if ((max(p.token_starts[mid], 0) >> p.page_log2) + 2 * mid <= x) lo = mid; else hi = mid; }
        b = lo;
        chunk = x - ((max(p.token_starts[b], 0) >> p.page_log2) + 2 * b);
    } else {
        const int per = (p.each >> p.page_log2) + 2;
        b = p.each == 1 ? x : x / per;
        chunk = p.each == 1 ? 0 : x % per;
    }
    int first, count;
    token_range(p, b, first, count);
    const int end = p.kv_offsets[b];
    if (count == 0 || end < 0 || chunk < 0) return;
    const int begin = max(end - count + 1, 0);              // tokens at negative positions are padding
    const int nth = (begin >> p.page_log2) + chunk;
    const int lo = max(begin, nth << p.page_log2);
    int hi = min(end, (nth << p.page_log2) + P - 1);
    if (lo > hi) return;
    if (nth >= p.max_pages || (p.rope_type >= 0 && hi >= p.rope_rows)) {
        if (tid == 0 && p.status) *p.status = 6;
        if (nth >= p.max_pages) return;
        hi = p.rope_rows - 1;
        if (lo > hi) return;
    }
    const int page = p.block_table[(long long)b * p.max_pages + nth];
    if ((unsigned)page >= (unsigned)p.num_pages) {
        if (tid == 0 && p.status) *p.status = 5;
        return;
    }
    const int slot = lo & (P - 1), tokens = hi - lo + 1;
    const int token0 = first + (lo - (end - count + 1));
    const __half* src = is_v ? p.v + token0 * p.v_stride + h * D : p.k + token0 * p.k_stride + h * D;
    const long long src_stride = is_v ? p.v_stride : p.k_stride;
    const int rope = is_v ? -1 : p.rope_type;
    const long long base = (long long)page * p.page_stride + (long long)h * p.head_stride;
    float* scale_at = KIND == 0 ? nullptr : (is_v ? p.v_scale : p.k_scale) + (long long)page * p.num_kv_heads + h;
    const float old = (KIND != 0 && slot > 0) ? *scale_at : 0.f;

    const int tasks = tokens << tasks_log2;
    auto rotated = [&](int at, ChannelTask& t, uint4& xa, uint4& xb) {
        const int tk = at >> tasks_log2;
        t = channel_task(at & ((1 << tasks_log2) - 1), D, rope, p.rotary_dim);
        const __half* row = src + tk * src_stride;
        xa = *reinterpret_cast<const uint4*>(row + t.a);
        xb = *reinterpret_cast<const uint4*>(row + t.b);
        if (t.rotated) {
            const long long e = (long long)(lo + tk) * (rope == 2 ? p.rotary_dim : D) + t.entry;
            rotate_task(t, xa, xb, *reinterpret_cast<const uint4*>(p.cos_table + e), *reinterpret_cast<const uint4*>(p.sin_table + e));
        }
        return tk;
    };
    if constexpr (KIND == 0) {
        __half* pool = (__half*)(is_v ? p.v_pool : p.k_pool) + base;
        for (int at = tid; at < tasks; at += T) {
            ChannelTask t;
            uint4 xa, xb;
            __half* dst = pool + (long long)(slot + rotated(at, t, xa, xb)) * p.token_stride;
            *reinterpret_cast<uint4*>(dst + t.a) = xa;
            *reinterpret_cast<uint4*>(dst + t.b) = xb;
        }
    } else {
        __shared__ uint32_t s_top[8];
        uint32_t top = 0;                                   // of the magnitudes' bits, in both halves: NaN is above infinity
        ChannelTask t;
        uint4 xa = make_uint4(0, 0, 0, 0), xb = xa;
        int tk = 0;
        const int last = tasks - 1 - tid < 0 ? tid : tid + (tasks - 1 - tid) / T * T;        // a thread's last task, whose values it keeps
        for (int at = tid; at < tasks; at += T) {
            tk = rotated(at, t, xa, xb);
            const uint32_t* a = reinterpret_cast<const uint32_t*>(&xa);
            const uint32_t* c = reinterpret_cast<const uint32_t*>(&xb);
#pragma unroll
            for (int k = 0; k < 4; ++k) top = __vmaxu2(top, __vmaxu2(a[k] & 0x7fff7fffu, c[k] & 0x7fff7fffu));
        }
        top = max(top & 0xffffu, top >> 16);
        top = __reduce_max_sync(~0u, top);
        if ((tid & 31) == 0) s_top[tid >> 5] = top;
        __syncthreads();
        for (int w = 0; w < (T >> 5); ++w) top = max(top, s_top[w]);
        const float amax = __half2float(__ushort_as_half((unsigned short)top));
        const float need = top >= 0x7c00u ? NAN : __fdiv_rn(amax, KIND == 1 ? 448.f : 127.f);
        // a scale that another program gave the page may be negative: it keeps its sign, and grows by magnitude
        const float top_scale = fmaxf(fabsf(old), need), now = (isnan(need) || isnan(old)) ? NAN : old < 0.f ? -top_scale : top_scale;
        // tokens of zeros stay zeros: the reciprocal of a scale below 2^-128 is infinite
        const float inv = now == 0.f || (need == 0.f && !isnan(now)) ? 0.f : __fdiv_rn(1.f, now);
        if (tid == 0) *scale_at = now;
        unsigned char* pool = (unsigned char*)(is_v ? p.v_pool : p.k_pool) + base;
        for (int at = last; at >= 0 && at < tasks; at -= T) {
            if (at != last) tk = rotated(at, t, xa, xb);
            unsigned char* dst = pool + (long long)(slot + tk) * p.token_stride;
            *reinterpret_cast<uint2*>(dst + t.a) = quantise8<KIND>(xa, inv);
            *reinterpret_cast<uint2*>(dst + t.b) = quantise8<KIND>(xb, inv);
        }
        if (fabsf(now) > fabsf(old) && slot > 0) {                        // the older tokens of the page under the new scale
            const float factor = __fdiv_rn(old, now);
            for (int at = tid; at < slot << tasks_log2; at += T) {
                uint4* row = reinterpret_cast<uint4*>(pool + (long long)(at >> tasks_log2) * p.token_stride + (at & ((1 << tasks_log2) - 1)) * 16);
                uint4 w = *row;
                uint32_t* q = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float f[4];
                    widen4<KIND>(q[k], f);
                    q[k] = narrow4<KIND>(__fmul_rn(f[0], factor), __fmul_rn(f[1], factor), __fmul_rn(f[2], factor), __fmul_rn(f[3], factor));
                }
                *row = w;
            }
        }
    }
}

#endif  // __CUDACC__

}  // namespace vteb
