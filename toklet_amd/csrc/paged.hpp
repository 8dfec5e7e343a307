// paged.hpp - device-side types of the paged cache's kernels.
//
// K and V of one layer live in pages of `page_tokens` rows: element (head h,
// row r, feature d) of page g at g * page_stride + h * head_stride +
// r * row_stride + d.  Key j of a sequence is row j % page_tokens of page
// table[j / page_tokens].  Tables, lengths and query ranges are device arrays
// that a captured launch reads anew at each replay, so the kernels check every
// value that becomes an address: a value that fails raises ST_BAD_PAGE, and
// nothing is read or written through it.
#pragma once

#include "device.hpp"

namespace tkh {

struct PagedBatch {
    const int32_t *table;        // [table_rows, table_stride]
    const int32_t *key_lens;     // [table_rows]
    const int32_t *query_start;  // [sequences + 1], or null: max_queries rows each
    const int32_t *slots;        // [sequences] table rows, or null: row b
    int64_t table_stride;
    int32_t table_rows, sequences, max_queries, max_keys, total;
    int32_t first;  // the launch's sequences are first .. first + sequences - 1 of the arrays
};
// Sequences that one attention launch lists; a larger batch takes several launches.
constexpr int PAGED_LIST_MAX = 1024;

struct PagedLayout {
    int64_t page_stride, head_stride, row_stride;  // elements
    int32_t pages, page_shift;
};

// Division by d of numbers below 2^31: n m / 2^(31 + l) rounded down, with l = ceil(log2 d)
// and m = ceil(2^(31 + l) / d), is exact, as 2^(31 + l) <= m d <= 2^(31 + l) + 2^l.  A workgroup
// divides some ten times before its first load of keys: one token over 301 keys 8.9 us in
// the kernel, 9.3 with plain divisions.
struct Divisor {
    uint32_t m;
    int32_t shift;
    static Divisor of(uint32_t d) {
        int l = 0;
        while ((1u << l) < d) ++l;
        return {(uint32_t)((((uint64_t)1 << (31 + l)) + d - 1) / d), 31 + l};
    }
    __device__ int operator()(int n) const { return (int)(((uint64_t)(uint32_t)n * m) >> shift); }
};

// Rows x splits whose (maximum, mass) pairs the merging workgroup holds in LDS.
constexpr int PAGED_PAIRS_MAX = 2048;

struct PagedAttend {
    PagedBatch b;
    PagedLayout l;
    const void *q;    // [total, Hq, D]
    const void *k, *v;
    void *out;        // [total, Hq, D] in the storage dtype
    int32_t hq, hkv, group;
    Divisor by_hkv, by_group;
    int32_t window;   // at most 2^30, which hides no key
    float scale_log2;
    float softcap_y, softcap_log2;  // scale / cap and cap * log2(e); 0: no cap
    int32_t splits;      // most key splits of a row block
    int32_t min_blocks;  // key blocks (16 keys; 32 for chunks) of a split at least
    int32_t groups, groups_short;  // workgroups that the batch's key blocks are split towards; if into short parts
    int32_t decode_rows;  // sequences of at most this many packed rows are paged_decode's, others the chunk kernel's
    int32_t rows;         // packed rows (tokens x group) a partial holds
    float *part_ml, *part_o;  // [slot, rows, 2] and [slot, rows, D]
    uint32_t *counters;       // at a row block's first slot: splits that have arrived
    uint32_t *status;
};

struct PagedRotary {
    int32_t layout;   // 0 none, 1 half, 2 interleaved
    int32_t rotated;  // leading features that rotate
    int32_t scaling;  // 0 none, 1 linear, 2 bands
    double step;      // log2 of the ratio of consecutive frequencies (negative)
    double inv_factor, low, inv_width, original;
    float magnitude;
};

struct PagedProduce {
    PagedBatch b;
    PagedLayout l;
    PagedRotary rot;
    const void *q, *k, *v;                // token rows of [H, D]
    int64_t q_stride, k_stride, v_stride;  // elements between tokens
    const float *q_norm, *k_norm;          // [D] or null
    void *q_out;                           // [total, Hq, D]
    void *k_pages, *v_pages;
    int32_t hq, hkv, d;
    float eps;
    uint32_t *status;
};

// Page copies: pairs in the kernel's arguments, so a call uploads nothing.
constexpr int COPY_PAGES_MAX = 480;
struct CopyPages {
    uint8_t *pool;
    int64_t plane_stride, page_stride, page_bytes;  // bytes
    int32_t planes, count;
    uint32_t src[COPY_PAGES_MAX], dst[COPY_PAGES_MAX];
};
static_assert(sizeof(CopyPages) <= 4096, "kernel arguments");

// Changed words of an owner's page tables and lengths, likewise.
constexpr int PATCH_MAX = 500;
struct PatchWords {
    int32_t *base;
    int32_t count;
    uint32_t index[PATCH_MAX];
    int32_t value[PATCH_MAX];
};
static_assert(sizeof(PatchWords) <= 4096, "kernel arguments");

// One sequence of a batch as the kernels use it: query rows [q0, q0 + n), len
// keys.  Anything out of range gives no rows and no keys, and `bad`.
struct PagedSeq {
    int32_t q0, n, len, slot;
    bool bad;
};
// The loads are independent of one another as far as they can be: a workgroup waits
// for them before anything else.
__device__ __forceinline__ PagedSeq paged_sequence(const PagedBatch &b, int in_launch) {
    const int s = b.first + in_launch;
    PagedSeq r;
    int32_t q1;
    if (b.query_start) {
        const_ptr<int32_t> start = (const_ptr<int32_t>)b.query_start + s;
        r.q0 = start[0];
        q1 = start[1];
    } else {
        r.q0 = s * b.max_queries;
        q1 = r.q0 + b.max_queries;
    }
    r.slot = b.slots ? ((const_ptr<int32_t>)b.slots)[s] : s;
    const bool no_slot = (uint32_t)r.slot >= (uint32_t)b.table_rows;
    r.len = ((const_ptr<int32_t>)b.key_lens)[no_slot ? 0 : r.slot];
    r.n = q1 - r.q0;
    r.bad = no_slot || r.q0 < 0 || q1 < r.q0 || q1 > b.total || r.n > b.max_queries || (uint32_t)r.len > (uint32_t)b.max_keys;
    if (r.bad) r.slot = r.q0 = r.n = r.len = 0;
    return r;
}

}  // namespace tkh
