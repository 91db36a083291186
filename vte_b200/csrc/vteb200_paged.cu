// Entry points of the paged key/value cache: include/vteb200.h, "paged caches".  A call's arguments are checked before
// anything else, so that a refusal needs no device.
#include <limits.h>
#include <math.h>
#include <string.h>

#include "../../include/vteb200.h"
#include "shim_internal.h"
#include "kernels/paged_attention.cuh"
#include "kernels/paged_append.cuh"

using namespace vteb;
using vteb_shim::report;
using vteb_shim::report_rt;

namespace {

// The library's device for the time of a call: a program may have made another one current.
struct OnDevice {
    int before = -1, rc = 0;
    OnDevice() {
        const int want = vteb_shim::device_index();
        if (want < 0) { rc = report(VTEB_ERR_NOT_INITIALIZED, "vteb_init has not been called"); return; }
        int now = 0;
        if ((rc = report_rt(cudaGetDevice(&now), "cudaGetDevice"))) return;
        if (now != want) {
            if ((rc = report_rt(cudaSetDevice(want), "cudaSetDevice"))) return;
            before = now;
        }
    }
    ~OnDevice() { if (before >= 0) cudaSetDevice(before); }
};

int log2_of(int x) {
    int n = 0;
    while ((1 << n) < x) ++n;
    return n;
}

bool head_dim_ok(int d) { return d == 64 || d == 128 || d == 256; }

int check_cache(const vteb_paged_cache_t* c) {
    if (!c) return report(VTEB_ERR_INVALID_ARGUMENT, "null cache");
    if (c->ready != 1) return report(VTEB_ERR_INVALID_ARGUMENT, "the cache has not been through vteb_paged_cache_init");
    return 0;
}

int row_bytes_of(int head_dim, int type) { return head_dim * (type == kPagedF16 ? 2 : 1); }

// Positions of a box of the tensor maps: as many as a unit of the attention kernel holds.
int box_rows_of(int head_dim, int type, int page_size) {
    const int unit = paged_unit(row_bytes_of(head_dim, type));
    return page_size < unit ? page_size : unit;
}

// Rows (query token, head of the group) that a warp serves at once: 16 where there are more than 8, except with 256-wide
// heads, whose outputs for 16 rows would not fit a thread's registers.
int rows_per_block(int rows, int head_dim) { return rows > 8 && head_dim < 256 ? 16 : 8; }

int sm_count(int* sms) {
    static int known[64];
    const int d = vteb_shim::device_index();
    if (d >= 0 && d < 64 && known[d]) { *sms = known[d]; return 0; }
    const int rc = report_rt(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, d), "sm count");
    if (!rc && d >= 0 && d < 64) known[d] = *sms;
    return rc;
}

struct Workspace { size_t counters, ml, o, bytes; };

// Counters first, at a place and of a size that no shape changes: what one shape leaves in its pieces is never another's counter.
Workspace workspace_of(int rows, int head_dim, int sms) {
    const int block = rows_per_block(rows, head_dim);
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    const size_t workers = (size_t)sms * kPagedMaxWorkers, pieces = 2 * workers;
    Workspace w;
    w.counters = up(2 * pieces * 4);
    w.ml = up(pieces * block * 8);
    w.o = up(pieces * block * (size_t)head_dim * 4);
    w.bytes = w.counters + 2 * w.ml + w.o;
    return w;
}

int check_heads(int q_heads, int kv_heads, int head_dim, int batch, int query_tokens) {
    if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads) return report(VTEB_ERR_INVALID_ARGUMENT, "%d query heads on %d KV heads", q_heads, kv_heads);
    if (!head_dim_ok(head_dim)) return report(VTEB_ERR_UNSUPPORTED, "head_dim %d: 64, 128 or 256", head_dim);
    if (batch <= 0 || batch > 65535) return report(VTEB_ERR_INVALID_ARGUMENT, "batch %d: 1 to 65535", batch);
    if (query_tokens < 1 || query_tokens > VTEB_PAGED_MAX_QUERY_TOKENS)
        return report(VTEB_ERR_INVALID_ARGUMENT, "%d query tokens a sequence: 1 to %d", query_tokens, VTEB_PAGED_MAX_QUERY_TOKENS);
    if (q_heads > 4096) return report(VTEB_ERR_INVALID_ARGUMENT, "%d query heads: at most 4096", q_heads);
    return 0;
}

struct AttnKernel { void (*fn)(const PagedAttnArgs); int threads, smem; };

template <int D, int KIND, int NT>
AttnKernel attention_of(bool f32) {
    using S = PagedShape<D, KIND, NT>;
    return {f32 ? paged_attention_kernel<D, KIND, NT, true> : paged_attention_kernel<D, KIND, NT, false>, S::W * 32, S::SMEM};
}

template <int D, int KIND>
AttnKernel attention_of(int block, bool f32) {
    if constexpr (D < 256) { if (block == 16) return attention_of<D, KIND, 2>(f32); }
    return attention_of<D, KIND, 1>(f32);
}

template <int D>
AttnKernel attention_of(int type, int block, bool f32) {
    return type == kPagedF16 ? attention_of<D, kPagedF16>(block, f32)
         : type == kPagedE4m3 ? attention_of<D, kPagedE4m3>(block, f32) : attention_of<D, kPagedInt8>(block, f32);
}

template <typename Args>
int launch(void (*fn)(const Args), const Args& args, unsigned grid, unsigned threads, int smem, void* stream, bool programmatic, const char* what) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    if (programmatic) { cfg.attrs = &attr; cfg.numAttrs = 1; }
    return report_rt(cudaLaunchKernelEx(&cfg, fn, args), what);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" {

int vteb_paged_cache_init(vteb_paged_cache_t* c) {
    if (!c) return report(VTEB_ERR_INVALID_ARGUMENT, "null cache");
    c->ready = 0;
    if (c->type < VTEB_PAGED_F16 || c->type > VTEB_PAGED_INT8) return report(VTEB_ERR_INVALID_ARGUMENT, "unknown cache type %d", c->type);
    const int size = c->type == VTEB_PAGED_F16 ? 2 : 1;
    if (!head_dim_ok(c->head_dim)) return report(VTEB_ERR_UNSUPPORTED, "head_dim %d: 64, 128 or 256", c->head_dim);
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return report(VTEB_ERR_UNSUPPORTED, "page_size %d: 16, 32, 64 or 128", c->page_size);
    if (c->num_pages <= 0 || c->num_kv_heads <= 0) return report(VTEB_ERR_INVALID_ARGUMENT, "%d pages of %d KV heads", c->num_pages, c->num_kv_heads);
    if (!c->k_pool || !c->v_pool || !aligned16(c->k_pool) || !aligned16(c->v_pool))
        return report(VTEB_ERR_INVALID_ARGUMENT, "the pools are 16-byte aligned device memory (%p, %p)", c->k_pool, c->v_pool);
    if (size == 1 && (!c->k_scale || !c->v_scale)) return report(VTEB_ERR_INVALID_ARGUMENT, "8-bit pages need k_scale and v_scale");
    if (size == 1 && (((uintptr_t)c->k_scale & 3) || ((uintptr_t)c->v_scale & 3))) return report(VTEB_ERR_INVALID_ARGUMENT, "scales are fp32");
    const long long strides[3] = {c->token_stride, c->head_stride, c->page_stride};
    for (long long s : strides)
        if (s < c->head_dim || (s * size) % 16 || s * size >= (1ll << 40))
            return report(VTEB_ERR_INVALID_ARGUMENT, "strides (page %lld, token %lld, head %lld values) are at least head_dim and multiples of 16 bytes",
                          c->page_stride, c->token_stride, c->head_stride);
    // rows must not share memory: one of the two orders inside a page, and pages beyond it
    const long long t = c->token_stride, h = c->head_stride, P = c->page_size, H = c->num_kv_heads;
    const bool by_head = t >= c->head_dim && (H == 1 || h >= t * (P - 1) + c->head_dim);
    const bool by_token = h >= c->head_dim && t >= h * (H - 1) + c->head_dim;
    if ((!by_head && !by_token) || (c->num_pages > 1 && c->page_stride < t * (P - 1) + h * (H - 1) + c->head_dim))
        return report(VTEB_ERR_INVALID_ARGUMENT, "rows of a page overlap (page %lld, token %lld, head %lld values)", c->page_stride, t, h);
    const int row = c->head_dim * size, width = row < 128 ? row : 128;
    const cuuint64_t dims[5] = {(cuuint64_t)(width / size), (cuuint64_t)c->page_size, (cuuint64_t)(row / width), (cuuint64_t)c->num_kv_heads, (cuuint64_t)c->num_pages};
    const cuuint64_t bytes[4] = {(cuuint64_t)(t * size), (cuuint64_t)width, (cuuint64_t)(h * size), (cuuint64_t)(c->page_stride * size)};
    const cuuint32_t box[5] = {(cuuint32_t)(width / size), (cuuint32_t)box_rows_of(c->head_dim, c->type, c->page_size), (cuuint32_t)(row / width), 1u, 1u};
    OnDevice on;
    if (on.rc) return on.rc;
    KvTensorMap maps[2];
    void* const pools[2] = {c->k_pool, c->v_pool};
    for (int i = 0; i < 2; ++i) {
        const int rc = vteb_shim::encode_tiled(reinterpret_cast<CUtensorMap*>(&maps[i]), size == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8,
                                               5, pools[i], dims, bytes, box, width == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
        if (rc) return rc;
    }
    memcpy(c->maps, maps, sizeof(maps));
    c->ready = 1;
    return 0;
}

int vteb_paged_append(const vteb_paged_cache_t* c, const vteb_paged_append_t* a, void* stream) {
    int rc = check_cache(c);
    if (rc) return rc;
    if (!a) return report(VTEB_ERR_INVALID_ARGUMENT, "null arguments");
    if (a->batch <= 0 || a->max_pages <= 0 || a->total_tokens < 0) return report(VTEB_ERR_INVALID_ARGUMENT, "batch %d, %d pages a sequence, %d tokens", a->batch, a->max_pages, a->total_tokens);
    if ((long long)a->max_pages * c->page_size > VTEB_PAGED_MAX_POSITIONS) return report(VTEB_ERR_TOO_LARGE, "%d pages of %d: more than %d positions", a->max_pages, c->page_size, VTEB_PAGED_MAX_POSITIONS);
    if (!a->k || !a->v || !a->block_table || !a->kv_offsets) return report(VTEB_ERR_INVALID_ARGUMENT, "null pointer");
    if (!aligned16(a->k) || !aligned16(a->v) || !aligned16(a->q) || !aligned16(a->q_out)) return report(VTEB_ERR_INVALID_ARGUMENT, "rows are 16-byte aligned");
    if (!a->token_starts && a->total_tokens % a->batch) return report(VTEB_ERR_INVALID_ARGUMENT, "%d tokens of %d sequences without token_starts", a->total_tokens, a->batch);
    if ((a->q != nullptr) != (a->q_out != nullptr)) return report(VTEB_ERR_INVALID_ARGUMENT, "q and q_out go together");
    const int D = c->head_dim;
    const long long kv_row = (long long)c->num_kv_heads * D;
    if (a->k_token_stride < kv_row || a->v_token_stride < kv_row || a->k_token_stride % 8 || a->v_token_stride % 8)
        return report(VTEB_ERR_INVALID_ARGUMENT, "k and v token strides (%lld, %lld): at least %lld halves and multiples of 8", a->k_token_stride, a->v_token_stride, kv_row);
    if (a->q) {
        const long long q_row = (long long)a->num_q_heads * D;
        if (a->num_q_heads <= 0 || a->q_token_stride < q_row || a->q_out_token_stride < q_row || a->q_token_stride % 8 || a->q_out_token_stride % 8)
            return report(VTEB_ERR_INVALID_ARGUMENT, "%d query heads, token strides (%lld, %lld): at least %lld halves and multiples of 8", a->num_q_heads, a->q_token_stride, a->q_out_token_stride, q_row);
        if (a->q == a->q_out && a->q_token_stride != a->q_out_token_stride && a->total_tokens > 1)
            return report(VTEB_ERR_INVALID_ARGUMENT, "q rotated in place with two token strides (%lld, %lld)", a->q_token_stride, a->q_out_token_stride);
        if ((long long)a->total_tokens * a->num_q_heads > INT_MAX) return report(VTEB_ERR_TOO_LARGE, "%d tokens of %d query heads", a->total_tokens, a->num_q_heads);
    }
    if (a->rope_type < -1 || a->rope_type > 2) return report(VTEB_ERR_INVALID_ARGUMENT, "rope_type %d: -1 (none), 0, 1 or 2", a->rope_type);
    if (a->rope_type >= 0) {
        if (!a->rope_cos || !a->rope_sin || !aligned16(a->rope_cos) || !aligned16(a->rope_sin) || a->rope_rows <= 0)
            return report(VTEB_ERR_INVALID_ARGUMENT, "rotation tables: 16-byte aligned, with rows");
        if (a->rope_type == 2 && (a->rotary_dim <= 0 || a->rotary_dim > D || a->rotary_dim % 16))
            return report(VTEB_ERR_UNSUPPORTED, "rotary_dim %d: a multiple of 16 up to head_dim", a->rotary_dim);
    }
    OnDevice on;
    if (on.rc) return on.rc;
    if (a->total_tokens == 0) return 0;
    PagedAppendArgs p;
    memset(&p, 0, sizeof(p));
    p.k = (const __half*)a->k; p.v = (const __half*)a->v; p.q = (const __half*)a->q; p.q_out = (__half*)a->q_out;
    p.k_pool = c->k_pool; p.v_pool = c->v_pool; p.k_scale = c->k_scale; p.v_scale = c->v_scale;
    p.block_table = a->block_table; p.kv_offsets = a->kv_offsets; p.token_starts = a->token_starts;
    p.cos_table = (const __half*)a->rope_cos; p.sin_table = (const __half*)a->rope_sin; p.status = a->status;
    p.k_stride = a->k_token_stride; p.v_stride = a->v_token_stride; p.q_stride = a->q_token_stride; p.q_out_stride = a->q_out_token_stride;
    p.page_stride = c->page_stride; p.token_stride = c->token_stride; p.head_stride = c->head_stride;
    p.batch = a->batch; p.max_pages = a->max_pages; p.num_pages = c->num_pages; p.page_log2 = log2_of(c->page_size);
    p.total_tokens = a->total_tokens; p.each = a->token_starts ? 0 : a->total_tokens / a->batch;
    p.num_q_heads = a->num_q_heads; p.num_kv_heads = c->num_kv_heads; p.dim_log2 = log2_of(D);
    p.rope_type = a->rope_type; p.rotary_dim = a->rope_type == 2 ? a->rotary_dim : D; p.rope_rows = a->rope_rows;
    // Up to two 16-channel tasks of a full page a thread, in blocks of 128 (256 for pages of 16 KB and more); single tokens leave
    // most threads of a block idle: 64.
    const int tasks = c->page_size * D / 16;
    const int threads = p.each == 1 || tasks < 128 ? 64 : tasks > 512 ? 256 : 128;
    const long long slots = a->token_starts ? (long long)a->total_tokens / c->page_size + 2ll * a->batch
                          : p.each == 1 ? a->batch : (long long)a->batch * (p.each / c->page_size + 2);
    const long long kv_blocks = slots * c->num_kv_heads * 2;
    // One head of Q a thread while that leaves SMs without threads, else two.
    p.q_heads_each = a->q && a->num_q_heads % 2 == 0 && (long long)a->total_tokens * a->num_q_heads * (D / 16) > (1ll << 19) ? 2 : 1;
    const int q_groups = a->q ? a->num_q_heads / p.q_heads_each : 1;
    const long long q_tasks = a->q ? (long long)a->total_tokens * q_groups * (D / 16) : 0;
    const long long q_blocks = (q_tasks + threads - 1) / threads;
    if (kv_blocks + q_blocks > INT_MAX || q_tasks > (1ll << 40)) return report(VTEB_ERR_TOO_LARGE, "%d tokens: too many blocks", a->total_tokens);
    p.kv_blocks = (int)kv_blocks;
    auto k = c->type == kPagedF16 ? paged_append_kernel<0> : c->type == kPagedE4m3 ? paged_append_kernel<1> : paged_append_kernel<2>;
    return launch(k, p, (unsigned)(kv_blocks + q_blocks), threads, 0, stream, (a->launch_flags & VTEB_LAUNCH_PROGRAMMATIC) != 0, "paged append launch");
}

int vteb_paged_attention_workspace(int num_q_heads, int num_kv_heads, int head_dim, int batch, int query_tokens, size_t* bytes) {
    if (!bytes) return report(VTEB_ERR_INVALID_ARGUMENT, "null output");
    int rc = check_heads(num_q_heads, num_kv_heads, head_dim, batch, query_tokens), sms = 0;
    if (rc) return rc;
    OnDevice on;
    if (on.rc) return on.rc;
    if ((rc = sm_count(&sms))) return rc;
    *bytes = workspace_of(query_tokens * (num_q_heads / num_kv_heads), head_dim, sms).bytes;
    return 0;
}

int vteb_paged_attention(const vteb_paged_cache_t* c, const vteb_paged_attention_t* a, void* stream) {
    int rc = check_cache(c), sms = 0;
    if (rc) return rc;
    if (!a) return report(VTEB_ERR_INVALID_ARGUMENT, "null arguments");
    if ((rc = check_heads(a->num_q_heads, c->num_kv_heads, c->head_dim, a->batch, a->query_tokens))) return rc;
    if (!a->q || !a->output || !a->block_table || !a->kv_offsets || !a->workspace) return report(VTEB_ERR_INVALID_ARGUMENT, "null pointer");
    if (!aligned16(a->q) || !aligned16(a->output) || ((uintptr_t)a->workspace & 255)) return report(VTEB_ERR_INVALID_ARGUMENT, "q and output are 16-byte, the workspace 256-byte aligned");
    if (a->max_pages <= 0 || (long long)a->max_pages * c->page_size > VTEB_PAGED_MAX_POSITIONS)
        return report(VTEB_ERR_TOO_LARGE, "%d pages of %d a sequence: 1 to %d positions", a->max_pages, c->page_size, VTEB_PAGED_MAX_POSITIONS);
    if (!(a->scale == a->scale) || isinf(a->scale)) return report(VTEB_ERR_INVALID_ARGUMENT, "the scale is not finite");
    OnDevice on;
    if (on.rc) return on.rc;
    if ((rc = sm_count(&sms))) return rc;
    const int group = a->num_q_heads / c->num_kv_heads, rows = a->query_tokens * group;
    const int block = rows_per_block(rows, c->head_dim);
    const int unit = paged_unit(row_bytes_of(c->head_dim, c->type)), blocks = (rows + block - 1) / block;
    if ((long long)a->batch * c->num_kv_heads * blocks * (((long long)a->max_pages * c->page_size + unit - 1) / unit + 16) > INT_MAX / 2)
        return report(VTEB_ERR_TOO_LARGE, "%d sequences of up to %d pages: more work than a launch counts", a->batch, a->max_pages);
    const Workspace w = workspace_of(rows, c->head_dim, sms);
    if (a->workspace_bytes < w.bytes) return report(VTEB_ERR_TOO_LARGE, "the workspace holds %zu of %zu bytes", a->workspace_bytes, w.bytes);
    PagedAttnArgs p;
    memcpy(&p.k_map, c->maps, sizeof(p.k_map));
    memcpy(&p.v_map, c->maps + sizeof(p.k_map), sizeof(p.v_map));
    p.q = (const __half*)a->q; p.output = a->output; p.lse = a->lse;
    p.block_table = a->block_table; p.kv_offsets = a->kv_offsets;
    p.k_scale = c->k_scale; p.v_scale = c->v_scale;
    unsigned char* base = (unsigned char*)a->workspace;
    p.counters = (int*)base;
    p.part_ml = (float*)(base + w.counters);
    p.part_ml2 = (float*)(base + w.counters + w.ml);
    p.part_o = (float*)(base + w.counters + 2 * w.ml);
    p.status = a->status;
    p.batch = a->batch; p.max_pages = a->max_pages; p.num_pages = c->num_pages;
    p.page_log2 = log2_of(c->page_size);
    p.box_log2 = log2_of(box_rows_of(c->head_dim, c->type, c->page_size));
    p.num_q_heads = a->num_q_heads; p.num_kv_heads = c->num_kv_heads; p.group = group; p.queries = a->query_tokens;
    p.row_blocks = (rows + block - 1) / block;
    p.group_inv = ((1u << 31) + group - 1) / group;
    p.scale_log2e = a->scale * kLog2e;
    const bool f32 = a->out_is_f32 != 0;
    AttnKernel k = c->head_dim == 64 ? attention_of<64>(c->type, block, f32)
                 : c->head_dim == 128 ? attention_of<128>(c->type, block, f32) : attention_of<256>(c->type, block, f32);
    static bool raised[64][3][3][2][2];
    const int dev = vteb_shim::device_index(), di = log2_of(c->head_dim) - 6;
    const bool known = dev < 64;
    if (!known || !raised[dev][di][c->type][block == 16][f32]) {
        if ((rc = report_rt(cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem), "cudaFuncSetAttribute(max dynamic shared memory)"))) return rc;
        if (known) raised[dev][di][c->type][block == 16][f32] = true;
    }
    return launch(k.fn, p, sms, k.threads, k.smem, stream, (a->launch_flags & VTEB_LAUNCH_PROGRAMMATIC) != 0, "paged attention launch");
}

}  // extern "C"
