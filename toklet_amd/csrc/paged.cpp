// paged.cpp - host side of the paged cache (include/tokhip.h): the operators'
// checks and launches, and the owner of a pool with its page tables.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "../../include/tokhip.h"
#include "host.hpp"
#include "paged.hpp"

extern "C" hipError_t tkh_launch_paged_decode(const tkh::PagedAttend *p, int dtype, int d, int groups, hipStream_t stream,
                                              hipEvent_t start, hipEvent_t stop);
extern "C" int tkh_paged_chunk_waves(int d);
extern "C" hipError_t tkh_launch_paged_chunk(const tkh::PagedAttend *p, int dtype, int d, int waves, int groups,
                                             hipStream_t stream, hipEvent_t start, hipEvent_t stop);
extern "C" hipError_t tkh_launch_paged_produce(const tkh::PagedProduce *p, int src, int dst, hipStream_t stream);
extern "C" hipError_t tkh_launch_copy_pages(const tkh::CopyPages *c, hipStream_t stream);
extern "C" hipError_t tkh_launch_patch_words(const tkh::PatchWords *w, hipStream_t stream);
extern "C" hipError_t tkh_launch_copy_words(int32_t *dst, const int32_t *src, int32_t n, hipStream_t stream);

using namespace tkh_host;

namespace {

uint32_t unsupported(const char *what, tkh_error *err) {
    return fail(err, TKH_UNSUPPORTED, what, 0, 0, 0, "not supported: %s", what);
}
uint32_t at_least(const char *tensor, uint64_t actual, uint64_t expected, tkh_error *err) {
    if (actual < expected)
        return fail(err, TKH_LENGTH, tensor, 0, expected, actual, "%s length is %llu, expected at least %llu", tensor,
                    (unsigned long long)actual, (unsigned long long)expected);
    return TKH_OK;
}
bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

uint32_t check_layout(const tkh_paged_layout &l, uint64_t *extent, tkh_error *err) {
    TRY(nonzero(l.pages, "pages", err));
    TRY(nonzero(l.kv_heads, "kv_heads", err));
    TRY(nonzero(l.head_dim, "head_dim", err));
    TRY(nonzero(l.page_tokens, "page_tokens", err));
    if (l.head_dim != 64 && l.head_dim != 128 && l.head_dim != 256) return unsupported("paged head_dim", err);
    if (l.page_tokens < 16 || l.page_tokens > 1024 || (l.page_tokens & (l.page_tokens - 1)) != 0)
        return unsupported("page_tokens", err);
    if (l.pages > INT32_MAX || l.kv_heads > 65535) return unsupported("paged cache size", err);
    if (l.page_stride % 8 != 0 || l.head_stride % 8 != 0 || l.row_stride % 8 != 0)
        return invalid("page strides are multiples of 8 elements", err);
    // Rows of one page apart from each other: heads outside rows, or rows outside heads.
    if (l.row_stride < l.head_dim || (l.kv_heads > 1 && l.head_stride < l.head_dim))
        return invalid("page rows overlap", err);
    uint64_t heads, rows, span, n;
    TRY(product(l.kv_heads - 1, l.head_stride, &heads, err));
    TRY(product(l.page_tokens - 1, l.row_stride, &rows, err));
    TRY(add(heads, rows, &span, err));
    TRY(add(span, l.head_dim, &span, err));
    if (l.kv_heads > 1 && l.head_stride < rows + l.head_dim && l.row_stride < heads + l.head_dim)
        return invalid("page rows overlap", err);
    if (l.pages > 1 && l.page_stride < span) return invalid("pages overlap", err);
    TRY(product(l.pages - 1, l.page_stride, &n, err));
    TRY(add(n, span, extent, err));
    if (*extent > (uint64_t)INT64_MAX / 8)
        return fail(err, TKH_SIZE_OVERFLOW, nullptr, 0, 0, 0, "tensor size arithmetic overflow");
    // A page's bytes, and a row's place in it, are 32-bit in the kernels.
    if (l.row_stride > (1u << 17) || (l.pages > 1 && l.page_stride > (1u << 30))) return unsupported("page strides", err);
    return TKH_OK;
}

uint32_t check_batch(const tkh_paged_batch &b, const tkh_paged_layout &l, tkh_error *err) {
    TRY(nonzero(b.sequences, "sequences", err));
    TRY(nonzero(b.max_queries, "max_queries", err));
    TRY(nonzero(b.max_keys, "max_keys", err));
    TRY(nonzero(b.table_rows, "table_rows", err));
    TRY(nonzero(b.table_stride, "table_stride", err));
    uint64_t n;
    TRY(product(b.sequences, b.max_queries, &n, err));
    if (!b.query_start) TRY(length("query rows", b.total_queries, n, err));
    if (!b.slots && b.table_rows < b.sequences) return invalid("table_rows below sequences without slots", err);
    TRY(product(b.table_stride, l.page_tokens, &n, err));
    if (b.max_keys > n) return invalid("max_keys exceeds the page table's rows", err);
    // Positions, rows and table indexes are 32-bit in the kernels.
    if (b.total_queries >= (1u << 24) || b.max_queries > (1u << 24) || b.sequences > 65535 || b.max_keys > (1u << 30) ||
        b.table_rows > INT32_MAX || b.table_stride > INT32_MAX)
        return unsupported("paged batch size", err);
    return TKH_OK;
}

tkh::PagedBatch device_batch(const tkh_paged_batch &b) {
    return tkh::PagedBatch{b.page_table, b.key_lens, b.query_start, b.slots, (int64_t)b.table_stride,
                           (int32_t)b.table_rows, (int32_t)b.sequences, (int32_t)b.max_queries,
                           (int32_t)b.max_keys, (int32_t)b.total_queries, 0};
}
tkh::PagedLayout device_layout(const tkh_paged_layout &l) {
    return tkh::PagedLayout{(int64_t)l.page_stride, (int64_t)l.head_stride, (int64_t)l.row_stride, (int32_t)l.pages,
                            __builtin_ctzll(l.page_tokens)};
}

// The launches of a batch's attention, PAGED_LIST_MAX sequences each.  The kernels count
// the work on the device; a launch has the most workgroups that there can be.  row_blocks:
// blocks of `rows` packed rows that `sequences` sequences can have per KV head; `groups`:
// workgroups to split their keys towards, in parts of `min_blocks` blocks of `block` keys
// at least.
struct Splits {
    int64_t rows, block, min_blocks, groups, groups_short, most, waves;
};
template <class RowBlocks, class Launch>
uint32_t launch_listed(tkh_context *ctx, tkh::PagedAttend p, int D, const Splits &sp, RowBlocks row_blocks, Launch launch, tkh_error *err) {
    // Partials: two slots per group that is split towards, and a counter for each and wave.
    const int64_t slot_bytes = (int64_t)p.rows * (D + 2) * sizeof(float), region = (int64_t)split_region_bytes(ctx) - 64;
    int64_t groups = std::min<int64_t>(sp.groups, std::min<int64_t>(region / slot_bytes, kPagedCounters / sp.waves) / 2);
    p.splits = (int32_t)(groups < 1 ? 1 : sp.most);
    groups = std::max<int64_t>(1, groups);
    p.min_blocks = (int32_t)sp.min_blocks;
    p.groups = (int32_t)groups;
    p.groups_short = (int32_t)std::min(groups, sp.groups_short);
    p.part_ml = reinterpret_cast<float *>(ctx->workspace);
    p.part_o = p.part_ml + (2 * groups * p.rows * 2 + 3) / 4 * 4;
    p.counters = ctx->paged_counters;
    // Keys that a row block sees: window and as many more as it has tokens.
    const int64_t tokens = std::min<int64_t>(p.b.max_queries, (sp.rows - 2) / p.group + 2);
    const int64_t blocks = (std::min<int64_t>(p.b.max_keys, (int64_t)p.window + tokens - 1) + sp.block - 1) / sp.block;
    const int64_t parts = std::min<int64_t>(p.splits, std::max<int64_t>(1, (blocks + sp.min_blocks - 1) / sp.min_blocks));
    const int32_t sequences = p.b.sequences;
    for (p.b.first = 0; p.b.first < sequences; p.b.first += tkh::PAGED_LIST_MAX) {
        p.b.sequences = std::min(sequences - p.b.first, tkh::PAGED_LIST_MAX);
        const int64_t units = p.hkv * row_blocks(p.b.sequences), grid = parts == 1 ? units : std::min(units * parts, units + groups);
        if (grid > INT32_MAX / 512) return unsupported("paged batch size", err);  // threads of a launch are 32-bit
        hipEvent_t *ev = nullptr;
        TRY(profile_events(ctx, false, &ev, err));
        HIP_TRY(launch(p, (int)grid, ev ? ev[0] : nullptr, ev ? ev[1] : nullptr), "paged attention launch");
    }
    return TKH_OK;
}

// paged_decode: sequences of at most 16 packed rows; with FP32 storage, all.
uint32_t launch_decode(tkh_context *ctx, tkh::PagedAttend p, tkh_dtype dtype, int D, tkh_error *err) {
    const int64_t most = std::min<int64_t>((int64_t)p.b.max_queries * p.group, p.decode_rows);
    // Up to 16 rows a block, so that a batch of single tokens stores partials of its own
    // rows only; more rows (FP32 storage) in blocks of 32.
    p.rows = (int32_t)(most <= 16 ? most : 32);
    // Six workgroups a CU, of the two or more that it holds at once, so that sequences of
    // different lengths even out (64 of 512 to 8192 keys: 190 us, 209 at four); four where
    // there are so few sequences and KV heads that each is split evenly (4 of 100,000 keys:
    // 307 us, 322 at six); two of 32 rows, whose partials are larger (4 chunks of 128 FP32
    // tokens: 48 us, 57 at three), where the batch may be all chunks, when idle
    // workgroups only cost time (5 us of 6 a CU), and where six would have fewer than 32
    // blocks each (24 sequences of 203 to 4096 keys, 128 features: 18 us, 23 at six).
    // A split has eight blocks at least: one sequence of 1000 keys 9.6 us, 11 at 16, 17 at 32.
    const bool chunks = dtype != TKH_F32 && (int64_t)p.b.max_queries * p.group > 16;
    int64_t groups = ctx->paged_decode_groups;
    if (p.rows > 16 || chunks) groups = (groups + 2) / 3;
    else if (6 * (int64_t)p.b.sequences * p.hkv < groups) groups = (2 * groups + 2) / 3;
    Splits sp{};
    sp.rows = p.rows > 16 ? 32 : 16;
    sp.block = 16;
    sp.min_blocks = ctx->paged_decode_blocks;
    sp.groups = groups;
    sp.groups_short = (ctx->paged_decode_groups + 2) / 3;
    sp.most = tkh::PAGED_PAIRS_MAX / p.rows;
    sp.waves = 1;
    const int64_t all = (int64_t)p.b.total * p.group / sp.rows;
    auto row_blocks = [&](int64_t sequences) { return p.rows > 16 ? std::min(all + sequences, sequences * ((most + 31) / 32)) : sequences; };
    return launch_listed(ctx, p, D, sp, row_blocks, [&](const tkh::PagedAttend &a, int groups, hipEvent_t start, hipEvent_t stop) {
        return tkh_launch_paged_decode(&a, (int)dtype, D, groups, ctx->stream, start, stop);
    }, err);
}

// Sequences of more: the chunk kernel.
uint32_t launch_chunk(tkh_context *ctx, tkh::PagedAttend p, tkh_dtype dtype, int D, tkh_error *err) {
    // Eight waves where workgroups of 256 rows still fill the CUs.
    int waves = tkh_paged_chunk_waves(D);
    if (waves == 8 && p.hkv * ((int64_t)p.b.total * p.group / 256) < ctx->paged_wide_groups) waves = 4;
    Splits sp{};
    sp.rows = 32 * waves;
    sp.block = 32;
    sp.min_blocks = ctx->paged_chunk_tiles;
    // Workgroups that the CUs hold at once: more would wait for them (24 sequences of 1 to
    // 200 tokens, 256 features: 113 us in 256, 144 in 512).
    sp.groups = sp.groups_short = waves == 8 || D == 256 ? (ctx->paged_chunk_groups + 1) / 2 : ctx->paged_chunk_groups;
    sp.most = 32;
    sp.waves = waves;
    p.rows = (int32_t)sp.rows;
    const int64_t all = (int64_t)p.b.total * p.group / sp.rows, most = ((int64_t)p.b.max_queries * p.group + sp.rows - 1) / sp.rows;
    auto row_blocks = [&](int64_t sequences) { return std::min(all + sequences, sequences * most); };
    return launch_listed(ctx, p, D, sp, row_blocks, [&](const tkh::PagedAttend &a, int groups, hipEvent_t start, hipEvent_t stop) {
        return tkh_launch_paged_chunk(&a, (int)dtype, D, waves, groups, ctx->stream, start, stop);
    }, err);
}

// A captured replay would repeat a launch but not the host's bookkeeping.
uint32_t not_capturing(tkh_context *ctx, tkh_error *err) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    HIP_TRY(hipStreamIsCapturing(ctx->stream, &st), "capture status");
    if (st != hipStreamCaptureStatusNone) return unsupported("a paged cache's changes during stream capture", err);
    return TKH_OK;
}

// Copies in order.  A launch moves its pairs all at once, so it ends before a
// pair that reads or writes a page that the launch writes, or writes one that it
// reads; the stream orders the launches.  Pages of the current launch stand in a
// small open-addressed table.
uint32_t copy_in_order(tkh_context *ctx, tkh::CopyPages &c, const uint64_t *src, const uint64_t *dst, uint64_t count,
                       tkh_error *err) {
    constexpr uint32_t kTable = 2048;  // at most 2 * COPY_PAGES_MAX entries
    static_assert(2 * tkh::COPY_PAGES_MAX < kTable, "open addressing needs free places");
    uint32_t page[kTable];
    uint8_t use[kTable];  // 1: read, 2: written by this launch
    auto place = [&](uint32_t g) {
        uint32_t i = (g * 2654435761u) >> 21;
        while (use[i] && page[i] != g) i = (i + 1) % kTable;
        return i;
    };
    auto flush = [&]() -> uint32_t {
        if (c.count > 0) HIP_TRY(tkh_launch_copy_pages(&c, ctx->stream), "page copy launch");
        c.count = 0;
        std::memset(use, 0, sizeof use);
        return TKH_OK;
    };
    c.count = 0;
    std::memset(use, 0, sizeof use);
    for (uint64_t i = 0; i < count; ++i) {
        if (src[i] == dst[i]) continue;
        const uint32_t s = (uint32_t)src[i], d = (uint32_t)dst[i];
        if (c.count == tkh::COPY_PAGES_MAX || (use[place(s)] & 2) || use[place(d)]) TRY(flush());
        uint32_t at = place(s);
        page[at] = s;
        use[at] |= 1;
        at = place(d);
        page[at] = d;
        use[at] |= 2;
        c.src[c.count] = s;
        c.dst[c.count++] = d;
    }
    return flush();
}

}  // namespace

extern "C" {

uint32_t tkh_paged_attention(tkh_context *ctx, const tkh_paged_batch *batch, const tkh_paged_layout *layout,
                             uint64_t query_heads, tkh_dtype dtype, const void *q, uint64_t q_len, const void *k_pages,
                             uint64_t k_len, const void *v_pages, uint64_t v_len, float scale, uint64_t window,
                             float softcap, void *context, uint64_t context_len, tkh_error *err) {
    if (!batch || !layout) return invalid("paged batch", err);
    if (!valid_dtype(dtype)) return invalid("dtype", err);
    uint64_t extent, rows, n;
    TRY(check_layout(*layout, &extent, err));
    TRY(check_batch(*batch, *layout, err));
    TRY(nonzero(query_heads, "query_heads", err));
    if (query_heads % layout->kv_heads != 0) return invalid("query_heads must be divisible by kv_heads", err);
    if (query_heads > 65535) return unsupported("query_heads", err);
    if (!std::isfinite(scale) || scale <= 0.0f) return invalid("attention scale", err);
    if (!std::isfinite(softcap) || softcap < 0.0f) return invalid("score softcap", err);
    TRY(product(batch->total_queries, query_heads, &rows, err));
    if (rows > (1u << 30)) return unsupported("paged batch size", err);  // packed rows are 32-bit in the kernels
    TRY(product(rows, layout->head_dim, &n, err));
    TRY(length("q", q_len, n, err));
    TRY(length("context", context_len, n, err));
    TRY(at_least("k pages", k_len, extent, err));
    TRY(at_least("v pages", v_len, extent, err));
    if (!ctx) return invalid("context", err);
    if (batch->total_queries == 0) return after_operator(ctx, err);
    if (!q || !k_pages || !v_pages || !context || !batch->page_table || !batch->key_lens)
        return invalid("paged attention buffers", err);
    if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(context))
        return invalid("paged attention buffers start on 16 bytes", err);
    tkh::PagedAttend p{};
    p.b = device_batch(*batch);
    p.l = device_layout(*layout);
    p.q = q;
    p.k = k_pages;
    p.v = v_pages;
    p.out = context;
    p.hq = (int32_t)query_heads;
    p.hkv = (int32_t)layout->kv_heads;
    p.group = p.hq / p.hkv;
    p.by_hkv = tkh::Divisor::of((uint32_t)p.hkv);
    p.by_group = tkh::Divisor::of((uint32_t)p.group);
    p.window = window == 0 || window > (1u << 30) ? 1 << 30 : (int32_t)window;  // no key is further back
    p.scale_log2 = scale * 1.4426950408889634f;
    p.softcap_y = softcap != 0.0f ? scale / softcap : 0.0f;
    p.softcap_log2 = softcap * 1.4426950408889634f;
    p.status = ctx->status_dev;
    HIP_TRY(hipSetDevice(ctx->device), "hipSetDevice");
    const int D = (int)layout->head_dim;
    // A batch may have both kinds of sequences: each kernel passes the other's by.
    p.decode_rows = dtype == TKH_F32 ? INT32_MAX : 16;
    if (dtype == TKH_F32 || p.group <= 16) TRY(launch_decode(ctx, p, dtype, D, err));
    if (dtype != TKH_F32 && (int64_t)p.b.max_queries * p.group > 16) TRY(launch_chunk(ctx, p, dtype, D, err));
    return after_operator(ctx, err);
}

uint32_t tkh_paged_produce(tkh_context *ctx, const tkh_paged_batch *batch, const tkh_paged_layout *layout,
                           const tkh_rope *rope, uint64_t query_heads, tkh_dtype proj_dtype,
                           const tkh_paged_projections *proj, tkh_dtype dtype, void *q_out, uint64_t q_out_len,
                           void *k_pages, uint64_t k_len, void *v_pages, uint64_t v_len, tkh_error *err) {
    if (!batch || !layout || !rope || !proj) return invalid("paged producer", err);
    if (!valid_dtype(dtype) || !valid_dtype(proj_dtype)) return invalid("dtype", err);
    uint64_t extent, n;
    TRY(check_layout(*layout, &extent, err));
    TRY(check_batch(*batch, *layout, err));
    TRY(nonzero(query_heads, "query_heads", err));
    if (query_heads > 65535) return unsupported("query_heads", err);
    const uint64_t D = layout->head_dim, T = batch->total_queries;
    tkh::PagedRotary rot{};
    if (rope->layout > TKH_ROPE_INTERLEAVED) return invalid("rotary layout", err);
    if (rope->layout != TKH_ROPE_NONE) {
        const uint64_t r = rope->rotated_dims ? rope->rotated_dims : D;
        if (r > D) return invalid("rotated_dims exceeds head_dim", err);
        if (r % 8 != 0) return unsupported("rotated_dims is a multiple of 8", err);
        if (!std::isfinite(rope->theta) || rope->theta <= 0.0f) return invalid("rotary theta", err);
        if (!std::isfinite(rope->magnitude) || rope->magnitude <= 0.0f) return invalid("rotary magnitude", err);
        if (rope->scaling > TKH_ROPE_BANDS) return invalid("rotary scaling", err);
        rot.layout = (int32_t)rope->layout;
        rot.rotated = (int32_t)r;
        rot.scaling = (int32_t)rope->scaling;
        rot.step = -2.0 / (double)r * std::log2((double)rope->theta);
        rot.magnitude = rope->magnitude;
        if (rope->scaling != TKH_ROPE_UNSCALED) {
            if (!std::isfinite(rope->factor) || rope->factor < 1.0f) return invalid("rotary factor", err);
            rot.inv_factor = 1.0 / (double)rope->factor;
        }
        if (rope->scaling == TKH_ROPE_BANDS) {
            if (!std::isfinite(rope->low_freq_factor) || rope->low_freq_factor <= 0.0f ||
                !std::isfinite(rope->high_freq_factor) || rope->high_freq_factor <= rope->low_freq_factor)
                return invalid("rotary frequency factors", err);
            if (rope->original_max_positions == 0 || rope->original_max_positions > (uint64_t)1 << 53)
                return invalid("rotary original length", err);
            rot.low = rope->low_freq_factor;
            rot.inv_width = 1.0 / ((double)rope->high_freq_factor - (double)rope->low_freq_factor);
            rot.original = (double)rope->original_max_positions;
        }
    }
    if ((proj->q_norm || proj->k_norm) && (!std::isfinite(proj->norm_epsilon) || proj->norm_epsilon <= 0.0f))
        return invalid("norm epsilon", err);
    TRY(product(T, query_heads, &n, err));
    TRY(product(n, D, &n, err));
    TRY(length("q rows", q_out_len, n, err));
    const struct {
        const char *name;
        const void *at;
        uint64_t stride, len, heads;
    } rows[3] = {{"q projection", proj->q, proj->q_stride, proj->q_len, query_heads},
                 {"k projection", proj->k, proj->k_stride, proj->k_len, layout->kv_heads},
                 {"v projection", proj->v, proj->v_stride, proj->v_len, layout->kv_heads}};
    for (const auto &r : rows) {
        if (r.stride < r.heads * D || r.stride % 4 != 0) return invalid(r.name, err);
        if (T == 0) continue;
        TRY(product(T - 1, r.stride, &n, err));
        TRY(add(n, r.heads * D, &n, err));
        TRY(at_least(r.name, r.len, n, err));
    }
    TRY(at_least("k pages", k_len, extent, err));
    TRY(at_least("v pages", v_len, extent, err));
    if (T * ((query_heads + 2 * layout->kv_heads + 7) / 8) > INT32_MAX) return unsupported("paged producer size", err);
    if (!ctx) return invalid("context", err);
    if (T == 0) return after_operator(ctx, err);
    if (!q_out || !k_pages || !v_pages || !batch->page_table || !batch->key_lens)
        return invalid("paged producer buffers", err);
    for (const auto &r : rows)
        if (!r.at || ((uintptr_t)r.at & (4 * esize(proj_dtype) - 1)) != 0)
            return invalid("projections start on four elements", err);
    if (!aligned16(q_out) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(proj->q_norm) ||
        !aligned16(proj->k_norm))
        return invalid("paged producer buffers start on 16 bytes", err);
    tkh::PagedProduce p{};
    p.b = device_batch(*batch);
    p.l = device_layout(*layout);
    p.rot = rot;
    p.q = proj->q;
    p.k = proj->k;
    p.v = proj->v;
    p.q_stride = (int64_t)proj->q_stride;
    p.k_stride = (int64_t)proj->k_stride;
    p.v_stride = (int64_t)proj->v_stride;
    p.q_norm = proj->q_norm;
    p.k_norm = proj->k_norm;
    p.q_out = q_out;
    p.k_pages = k_pages;
    p.v_pages = v_pages;
    p.hq = (int32_t)query_heads;
    p.hkv = (int32_t)layout->kv_heads;
    p.d = (int32_t)D;
    p.eps = proj->norm_epsilon;
    p.status = ctx->status_dev;
    HIP_TRY(hipSetDevice(ctx->device), "hipSetDevice");
    HIP_TRY(tkh_launch_paged_produce(&p, (int)proj_dtype, (int)dtype, ctx->stream), "paged producer launch");
    return after_operator(ctx, err);
}

uint32_t tkh_copy_pages(tkh_context *ctx, void *pool, uint64_t pool_bytes, uint64_t planes, uint64_t plane_stride,
                        uint64_t pages, uint64_t page_stride, uint64_t page_bytes, const uint64_t *src,
                        const uint64_t *dst, uint64_t count, tkh_error *err) {
    TRY(nonzero(planes, "planes", err));
    TRY(nonzero(pages, "pages", err));
    TRY(nonzero(page_bytes, "page_bytes", err));
    if (planes > 65535 || pages > INT32_MAX || page_bytes > (uint64_t)1 << 31) return unsupported("page copy size", err);
    if (page_bytes % 2 != 0 || page_stride % 2 != 0 || plane_stride % 2 != 0)
        return invalid("pages are whole 16-bit elements", err);
    // Pages and planes apart from each other: pages inside planes, or planes inside pages.
    uint64_t in_plane, in_page, n;
    TRY(product(pages - 1, page_stride, &in_plane, err));
    TRY(product(planes - 1, plane_stride, &in_page, err));
    TRY(add(in_plane, in_page, &n, err));
    TRY(add(n, page_bytes, &n, err));
    const bool pages_inside = (pages == 1 || page_stride >= page_bytes) &&
                              (planes == 1 || plane_stride >= in_plane + page_bytes);
    const bool planes_inside = (planes == 1 || plane_stride >= page_bytes) &&
                               (pages == 1 || page_stride >= in_page + page_bytes);
    if (!pages_inside && !planes_inside) return invalid("pages overlap", err);
    TRY(at_least("pool", pool_bytes, n, err));
    if (count > 0 && (!src || !dst)) return invalid("page lists", err);
    for (uint64_t i = 0; i < count; ++i)
        if (src[i] >= pages || dst[i] >= pages)
            return fail(err, TKH_INVALID_PARAMETER, "page", i, pages, src[i] >= pages ? src[i] : dst[i],
                        "copy %llu names a page past the pool's %llu", (unsigned long long)i, (unsigned long long)pages);
    if (!ctx) return invalid("context", err);
    if (!pool || ((uintptr_t)pool & 1) != 0) return invalid("pool", err);
    HIP_TRY(hipSetDevice(ctx->device), "hipSetDevice");
    tkh::CopyPages c{};
    c.pool = static_cast<uint8_t *>(pool);
    c.plane_stride = (int64_t)plane_stride;
    c.page_stride = (int64_t)page_stride;
    c.page_bytes = (int64_t)page_bytes;
    c.planes = (int32_t)planes;
    TRY(copy_in_order(ctx, c, src, dst, count, err));
    return after_operator(ctx, err);
}

}  // extern "C"

// ---------------------------------------------------------------- owner

struct tkh_paged_kv {
    tkh_context *ctx = nullptr;
    int device = 0;
    tkh_paged_options o{};
    uint64_t page_bytes = 0, allocated = 0, free_pages = 0, lowest = 0;  // no page below `lowest` is free
    void *pool = nullptr;
    int32_t *meta = nullptr;            // page tables, then lengths
    std::vector<uint32_t> refs;         // per page: sequences that hold it
    std::vector<uint32_t> pending;      // per page, 0 between calls
    std::vector<int32_t> table;         // [sequences, sequence_pages]
    std::vector<int64_t> length;        // per sequence; -1: closed
    std::vector<uint8_t> seen;          // per sequence, 0 between calls
    std::vector<uint64_t> from, to;     // page moves of one call
    tkh::PatchWords patch{};
    uint64_t pages_of(uint64_t n) const { return (n + o.page_tokens - 1) / o.page_tokens; }
};

namespace {

// Queues one changed word of the device's tables (or nothing without a device).
uint32_t set_word(tkh_paged_kv *kv, uint64_t index, int32_t value, tkh_error *err);
uint32_t flush_words(tkh_paged_kv *kv, tkh_error *err) {
    if (kv->ctx && kv->patch.count > 0) {
        const hipError_t e = tkh_launch_patch_words(&kv->patch, kv->ctx->stream);
        kv->patch.count = 0;
        HIP_TRY(e, "page table update");
    }
    return TKH_OK;
}
uint32_t set_word(tkh_paged_kv *kv, uint64_t index, int32_t value, tkh_error *err) {
    if (!kv->ctx) return TKH_OK;
    if (kv->patch.count == tkh::PATCH_MAX) TRY(flush_words(kv, err));
    kv->patch.index[kv->patch.count] = (uint32_t)index;
    kv->patch.value[kv->patch.count++] = value;
    return TKH_OK;
}
uint32_t set_entry(tkh_paged_kv *kv, uint64_t s, uint64_t i, int32_t page, tkh_error *err) {
    kv->table[s * kv->o.sequence_pages + i] = page;
    return set_word(kv, s * kv->o.sequence_pages + i, page, err);
}
uint32_t set_length(tkh_paged_kv *kv, uint64_t s, int64_t n, tkh_error *err) {
    kv->length[s] = n;
    return set_word(kv, kv->o.sequences * kv->o.sequence_pages + s, (int32_t)std::max<int64_t>(n, 0), err);
}

uint64_t take_page(tkh_paged_kv *kv) {  // the caller has counted them
    while (kv->refs[kv->lowest]) ++kv->lowest;
    kv->refs[kv->lowest] = 1;
    --kv->free_pages;
    return kv->lowest;
}
void drop_page(tkh_paged_kv *kv, uint64_t page) {
    if (--kv->refs[page] == 0) {
        ++kv->free_pages;
        kv->lowest = std::min(kv->lowest, page);
    }
}

uint32_t move_pages(tkh_paged_kv *kv, tkh_error *err) {
    if (!kv->ctx || kv->from.empty()) return TKH_OK;
    tkh::CopyPages c{};
    c.pool = static_cast<uint8_t *>(kv->pool);
    c.page_bytes = c.page_stride = (int64_t)kv->page_bytes;
    c.plane_stride = (int64_t)(kv->page_bytes * kv->o.pages);
    c.planes = (int32_t)(2 * kv->o.layers);
    return copy_in_order(kv->ctx, c, kv->from.data(), kv->to.data(), kv->from.size(), err);
}

uint32_t changing(tkh_paged_kv *kv, tkh_error *err) {
    if (!kv) return invalid("paged cache", err);
    if (!kv->ctx) return TKH_OK;
    HIP_TRY(hipSetDevice(kv->device), "hipSetDevice");
    return not_capturing(kv->ctx, err);
}
uint32_t open_sequence(const tkh_paged_kv *kv, uint64_t s, tkh_error *err) {
    if (s >= kv->o.sequences || kv->length[s] < 0)
        return fail(err, TKH_INVALID_CONFIG, "sequence", s, 0, 0, "sequence %llu is not open", (unsigned long long)s);
    return TKH_OK;
}
uint32_t changed(tkh_paged_kv *kv, tkh_error *err) {
    TRY(flush_words(kv, err));
    return kv->ctx ? after_operator(kv->ctx, err) : ok(err);
}

uint32_t closed_slot(tkh_paged_kv *kv, uint64_t *s, tkh_error *err) {
    for (*s = 0; *s < kv->o.sequences; ++*s)
        if (kv->length[*s] < 0) return TKH_OK;
    return fail(err, TKH_CAPACITY, "sequences", 0, kv->o.sequences, 0, "all %llu sequences are open",
                (unsigned long long)kv->o.sequences);
}

}  // namespace

extern "C" {

uint32_t tkh_paged_create(tkh_context *ctx, const tkh_paged_options *options, tkh_paged_kv **out, tkh_error *err) {
    if (!options) return invalid("paged options", err);
    if (!out) return invalid("paged cache output", err);
    *out = nullptr;
    const tkh_paged_options &o = *options;
    if (!valid_dtype(o.storage)) return invalid("dtype", err);
    TRY(nonzero(o.layers, "layers", err));
    TRY(nonzero(o.sequences, "sequences", err));
    TRY(nonzero(o.sequence_pages, "sequence_pages", err));
    tkh_paged_layout l{o.pages, o.page_tokens, o.kv_heads, o.head_dim, 0, 0, 0};
    uint64_t extent, bytes, planes, words;
    TRY(product(o.page_tokens, o.head_dim, &l.head_stride, err));
    TRY(product(o.kv_heads, l.head_stride, &l.page_stride, err));
    l.row_stride = o.head_dim;
    TRY(check_layout(l, &extent, err));
    TRY(product(o.layers, 2, &planes, err));
    TRY(product(extent, planes, &bytes, err));
    TRY(product(bytes, (uint64_t)esize(o.storage), &bytes, err));
    TRY(product(o.sequences, o.sequence_pages, &words, err));
    if (planes > 65535 || words + o.sequences > (uint64_t)INT32_MAX || o.sequences > 65535 ||
        o.sequence_pages * o.page_tokens > (1u << 30) || l.page_stride * esize(o.storage) > (uint64_t)1 << 31)
        return unsupported("paged cache size", err);
    if (ctx) TRY(not_capturing(ctx, err));
    auto *kv = new (std::nothrow) tkh_paged_kv();
    if (!kv) return device_error(hipErrorOutOfMemory, "paged cache", err);
    kv->o = o;
    kv->page_bytes = l.page_stride * esize(o.storage);
    kv->free_pages = o.pages;
    try {
        kv->refs.assign(o.pages, 0);
        kv->pending.assign(o.pages, 0);
        kv->table.assign(words, 0);
        kv->length.assign(o.sequences, -1);
        kv->seen.assign(o.sequences, 0);
        kv->from.reserve(std::max(o.pages, o.sequences));
        kv->to.reserve(std::max(o.pages, o.sequences));
    } catch (const std::bad_alloc &) {
        delete kv;
        return device_error(hipErrorOutOfMemory, "paged cache", err);
    }
    if (ctx) {
        kv->ctx = ctx;
        kv->device = ctx->device;
        const size_t meta_bytes = (words + o.sequences) * sizeof(int32_t);
        hipError_t e = hipSetDevice(ctx->device);
        if (e == hipSuccess) e = hipMalloc(&kv->pool, bytes);
        if (e == hipSuccess) e = hipMalloc(&kv->meta, meta_bytes);
        if (e == hipSuccess) e = hipMemsetAsync(kv->pool, 0, bytes, ctx->stream);
        if (e == hipSuccess) e = hipMemsetAsync(kv->meta, 0, meta_bytes, ctx->stream);
        if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
        if (e != hipSuccess) {
            tkh_paged_destroy(kv);
            return device_error(e, "paged cache allocation", err);
        }
        kv->allocated = bytes + meta_bytes;
        kv->patch.base = kv->meta;
    }
    *out = kv;
    return ok(err);
}

void tkh_paged_destroy(tkh_paged_kv *kv) {
    if (!kv) return;
    // As tkh_kv_destroy: the context may be gone, hipFree waits for the device.
    if (kv->pool || kv->meta) hipSetDevice(kv->device);
    if (kv->pool) hipFree(kv->pool);
    if (kv->meta) hipFree(kv->meta);
    delete kv;
}

uint32_t tkh_paged_info_get(const tkh_paged_kv *kv, tkh_paged_info *info) {
    if (!kv || !info) return TKH_INVALID_PARAMETER;
    const tkh_paged_options &o = kv->o;
    *info = tkh_paged_info{o.layers, o.kv_heads, o.head_dim, o.page_tokens, o.pages, o.sequences, o.sequence_pages,
                           kv->free_pages, 0, kv->allocated, kv->pool, kv->meta,
                           kv->meta ? kv->meta + o.sequences * o.sequence_pages : nullptr, o.storage};
    for (int64_t n : kv->length) info->open_sequences += n >= 0;
    return TKH_OK;
}

uint32_t tkh_paged_open(tkh_paged_kv *kv, uint64_t *sequence, tkh_error *err) {
    TRY(changing(kv, err));
    if (!sequence) return invalid("sequence output", err);
    uint64_t s;
    TRY(closed_slot(kv, &s, err));
    TRY(set_length(kv, s, 0, err));
    *sequence = s;
    return changed(kv, err);
}

uint32_t tkh_paged_fork(tkh_paged_kv *kv, uint64_t sequence, uint64_t *forked, tkh_error *err) {
    TRY(changing(kv, err));
    if (!forked) return invalid("sequence output", err);
    TRY(open_sequence(kv, sequence, err));
    uint64_t s;
    TRY(closed_slot(kv, &s, err));
    const uint64_t n = kv->pages_of((uint64_t)kv->length[sequence]), w = kv->o.sequence_pages;
    for (uint64_t i = 0; i < n; ++i) {
        const int32_t page = kv->table[sequence * w + i];
        kv->table[s * w + i] = page;
        ++kv->refs[page];
    }
    TRY(set_length(kv, s, kv->length[sequence], err));
    if (kv->ctx && n > 0)
        HIP_TRY(tkh_launch_copy_words(kv->meta + s * w, kv->meta + sequence * w, (int32_t)n, kv->ctx->stream),
                "page table update");
    *forked = s;
    return changed(kv, err);
}

uint32_t tkh_paged_extend(tkh_paged_kv *kv, const uint64_t *sequences, const uint64_t *tokens, uint64_t count,
                          tkh_error *err) {
    TRY(changing(kv, err));
    if (count > 0 && (!sequences || !tokens)) return invalid("sequences", err);
    const uint64_t P = kv->o.page_tokens, w = kv->o.sequence_pages;
    // What the call takes, before anything changes.  A partly filled last page
    // is copied while more than one sequence holds it; the last of several in
    // this call that share one keeps it.
    uint64_t need = 0, checked = 0, marked = 0;
    uint32_t rc = TKH_OK;
    auto tail = [&](uint64_t s) { return kv->table[s * w + (uint64_t)kv->length[s] / P]; };
    auto grows_partly = [&](uint64_t i) {
        return tokens[i] > 0 && (uint64_t)kv->length[sequences[i]] % P != 0;
    };
    for (; checked < count && rc == TKH_OK; ++checked) {
        const uint64_t s = sequences[checked];
        rc = open_sequence(kv, s, err);
        if (rc != TKH_OK) break;
        if (kv->seen[s]) {
            rc = invalid("a sequence is extended twice", err);
            break;
        }
        kv->seen[s] = 1;
        ++marked;
        const uint64_t old = (uint64_t)kv->length[s];
        if (tokens[checked] > w * P - old) {
            rc = fail(err, TKH_CAPACITY, "sequence", s, w * P, old, "sequence %llu has no room for %llu more keys",
                      (unsigned long long)s, (unsigned long long)tokens[checked]);
            break;
        }
        need += kv->pages_of(old + tokens[checked]) - kv->pages_of(old);
        if (grows_partly(checked) && kv->refs[tail(s)] - kv->pending[tail(s)] > 1) {
            ++kv->pending[tail(s)];
            ++need;
        }
    }
    for (uint64_t i = 0; i < marked; ++i) {
        kv->seen[sequences[i]] = 0;
        if (grows_partly(i)) kv->pending[tail(sequences[i])] = 0;
    }
    if (rc != TKH_OK) return rc;
    if (need > kv->free_pages)
        return fail(err, TKH_CAPACITY, "pages", 0, need, kv->free_pages, "%llu pages are needed, %llu are free",
                    (unsigned long long)need, (unsigned long long)kv->free_pages);
    kv->from.clear();
    kv->to.clear();
    for (uint64_t i = 0; i < count; ++i) {
        const uint64_t s = sequences[i], old = (uint64_t)kv->length[s];
        if (grows_partly(i) && kv->refs[tail(s)] > 1) {
            const uint64_t page = (uint64_t)tail(s), copy = take_page(kv);
            kv->from.push_back(page);
            kv->to.push_back(copy);
            drop_page(kv, page);
            TRY(set_entry(kv, s, old / P, (int32_t)copy, err));
        }
        for (uint64_t j = kv->pages_of(old); j < kv->pages_of(old + tokens[i]); ++j)
            TRY(set_entry(kv, s, j, (int32_t)take_page(kv), err));
        if (tokens[i] > 0) TRY(set_length(kv, s, (int64_t)(old + tokens[i]), err));
    }
    TRY(move_pages(kv, err));
    return changed(kv, err);
}

uint32_t tkh_paged_truncate(tkh_paged_kv *kv, uint64_t sequence, uint64_t length, tkh_error *err) {
    TRY(changing(kv, err));
    TRY(open_sequence(kv, sequence, err));
    const uint64_t old = (uint64_t)kv->length[sequence], w = kv->o.sequence_pages;
    if (length > old) return invalid("truncated length exceeds the sequence", err);
    for (uint64_t i = kv->pages_of(length); i < kv->pages_of(old); ++i) drop_page(kv, (uint64_t)kv->table[sequence * w + i]);
    TRY(set_length(kv, sequence, (int64_t)length, err));
    return changed(kv, err);
}

uint32_t tkh_paged_close(tkh_paged_kv *kv, uint64_t sequence, tkh_error *err) {
    TRY(changing(kv, err));
    TRY(open_sequence(kv, sequence, err));
    const uint64_t w = kv->o.sequence_pages;
    for (uint64_t i = 0; i < kv->pages_of((uint64_t)kv->length[sequence]); ++i)
        drop_page(kv, (uint64_t)kv->table[sequence * w + i]);
    TRY(set_length(kv, sequence, -1, err));
    return changed(kv, err);
}

uint32_t tkh_paged_compact(tkh_paged_kv *kv, uint64_t *moved, tkh_error *err) {
    TRY(changing(kv, err));
    const uint64_t used = kv->o.pages - kv->free_pages, w = kv->o.sequence_pages;
    kv->from.clear();
    kv->to.clear();
    // Every page past the first `used` moves to a free one below; `pending`
    // holds its new number, plus one, until the tables have it.
    for (uint64_t page = used; page < kv->o.pages; ++page) {
        if (!kv->refs[page]) continue;
        const uint32_t holders = kv->refs[page];
        const uint64_t to = take_page(kv);
        kv->refs[to] = holders;
        kv->refs[page] = 0;
        ++kv->free_pages;
        kv->pending[page] = (uint32_t)to + 1;
        kv->from.push_back(page);
        kv->to.push_back(to);
    }
    kv->lowest = std::min(used, kv->o.pages - 1);
    uint32_t rc = TKH_OK;
    for (uint64_t s = 0; s < kv->o.sequences; ++s) {
        if (kv->length[s] < 0) continue;
        for (uint64_t i = 0; i < kv->pages_of((uint64_t)kv->length[s]); ++i) {
            const uint32_t to = kv->pending[kv->table[s * w + i]];
            if (to && rc == TKH_OK) rc = set_entry(kv, s, i, (int32_t)to - 1, err);
        }
    }
    for (uint64_t page : kv->from) kv->pending[page] = 0;
    TRY(rc);
    TRY(move_pages(kv, err));
    if (moved) *moved = kv->from.size();
    return changed(kv, err);
}

uint32_t tkh_paged_sequence_get(const tkh_paged_kv *kv, uint64_t sequence, uint64_t *length, uint64_t *pages,
                                uint64_t capacity) {
    if (!kv || sequence >= kv->o.sequences || kv->length[sequence] < 0) return TKH_INVALID_PARAMETER;
    const uint64_t n = (uint64_t)kv->length[sequence];
    if (length) *length = n;
    if (pages)
        for (uint64_t i = 0; i < std::min(capacity, kv->pages_of(n)); ++i)
            pages[i] = (uint64_t)kv->table[sequence * kv->o.sequence_pages + i];
    return TKH_OK;
}

}  // extern "C"
