// paged_device.hpp - what the paged attention kernels share.
#pragma once

#include "paged.hpp"

namespace tkh {

namespace {

template <class T> using lds_ptr = __attribute__((address_space(3))) T *;
using s16x4 = short __attribute__((ext_vector_type(4)));
using f16x4 = _Float16 __attribute__((ext_vector_type(4)));
using bf16x4 = __bf16 __attribute__((ext_vector_type(4)));
using u32x2 = uint32_t __attribute__((ext_vector_type(2)));

template <int DT> __device__ __forceinline__ f32x4 mfma_16x16x32(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (DT == BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <int DT> __device__ __forceinline__ f32x4 mfma_16x16x16(u32x2 a, u32x2 b, f32x4 c) {
    if constexpr (DT == BF16)
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
}
// Four FP32 values rounded to 16 bits (to nearest even).
template <int DT> __device__ __forceinline__ u32x2 pack4(f32x4 x) {
    if constexpr (DT == BF16) return __builtin_bit_cast(u32x2, __builtin_convertvector(x, bf16x4));
    else return __builtin_bit_cast(u32x2, __builtin_convertvector(x, f16x4));
}
template <int DT> __device__ __forceinline__ f32x4 unpack4(u32x2 w) {
    if constexpr (DT == BF16) return __builtin_convertvector(__builtin_bit_cast(bf16x4, w), f32x4);
    else return __builtin_convertvector(__builtin_bit_cast(f16x4, w), f32x4);
}

// Four keys of one feature: a 16-lane group reads 4 rows x 16 features of 16 bits
// (lane j the 8 bytes of row j / 4, features 4 (j % 4)) and lane j receives
// feature j's four rows.
__device__ __forceinline__ u32x2 read_tr(lds_ptr<uint8_t> p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<s16x4>)p));
}

// 16 bytes per lane from base + off straight to LDS at m + 16 lane.  Assembly,
// because the compiler would otherwise wait for all of them before any LDS read;
// wait_loads orders them.  No register receives anything.
__device__ __forceinline__ void lds_load16(const void *base, uint32_t off, uint32_t m) {
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(m) : "memory", "m0");
}
// The same for lines that are read once (marked nontemporal).
__device__ __forceinline__ void lds_load16_once(const void *base, uint32_t off, uint32_t m) {
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(base), "s"(m) : "memory", "m0");
}
// Until at most N of this wave's vector memory operations are under way.
template <int N> __device__ __forceinline__ void wait_loads() {
    static_assert(N < 64, "vmcnt field");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Until this wave's LDS reads have returned: their rows may be overwritten.
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ const uint8_t *uniform_ptr(const uint8_t *p) {
    const uint64_t x = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
    return (const uint8_t *)(((uint64_t)hi << 32) | lo);
}

// Reductions over the lanes l, l ^ 16, l ^ 32, l ^ 48 (one query row's four lanes).
__device__ __forceinline__ void swap_pair(float x, bool far, float &a, float &b) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto p = far ? __builtin_amdgcn_permlane32_swap(u, u, false, false) : __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t p0 = p[0], p1 = p[1];
    a = __builtin_bit_cast(float, p0);
    b = __builtin_bit_cast(float, p1);
}
__device__ __forceinline__ float quad_max(float x) {
    float a, b;
    swap_pair(x, false, a, b);
    swap_pair(fmaxf(a, b), true, a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float quad_sum(float x) {
    float a, b;
    swap_pair(x, false, a, b);
    swap_pair(a + b, true, a, b);
    return a + b;
}

template <int DT> __device__ __forceinline__ void store_elem4(void *base, int64_t i, f32x4 x) {
    if constexpr (DT == F32) *gstore_ptr<f32x4>(reinterpret_cast<float *>(base) + i) = x;
    else *gstore_ptr<u32x2>(reinterpret_cast<uint16_t *>(base) + i) = pack4<DT>(x);
}

// Partials pass between workgroups on different XCDs: these go past the L2, so a
// store that has been acknowledged (wait_loads<0>) is there for every other
// workgroup's load.  That orders a partial before its arrival count without an
// agent-scope release and acquire, which write back and invalidate the XCD's
// whole L2: with them each workgroup of a streaming launch took 28 us longer (4
// sessions of 100k..131k keys in 4096 workgroups 512 us, in 2048 399 us).
__device__ __forceinline__ void shared_store(float *p, float x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float shared_load(const float *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

constexpr int CPOL_SC1 = 16;  // a buffer load past the L2, as shared_load
// LDS for that many (maximum, mass) pairs.
__device__ constexpr int pairs_bytes(int pairs) { return (pairs * 8 + 15) / 16 * 16; }

// Of numbers that are not negative.
__device__ __forceinline__ int quotient(int a, int b) { return (int)((uint32_t)a / (uint32_t)b); }

// One workgroup's work: keys of one row block (ROWS packed rows) of a sequence and KV head.
struct PagedWork {
    PagedSeq sq;
    int kvh, rb;
    int part, parts;  // this split, and the most that a row block of the sequence has
    int blocks;       // key blocks for which a row block has one more split
    int slot;         // of the row block's first partial

    // Splits of a row block that sees `n` key blocks.
    __device__ int active(int n) const {
        const int a = quotient(n + blocks - 1, blocks);
        return a < 1 ? 1 : (a < parts ? a : parts);
    }
};
// Workgroup `item`'s work, from the batch's lengths on the device: a ragged batch launches
// few idle workgroups, and its keys are split by their sum, not by the longest sequence's.
// C key blocks over R row blocks are split towards P = groups - R workgroups (half of
// `groups` at least): a row block has a split per C / P of its blocks.  That makes fewer
// than P + R workgroups, so no more than `groups`, which the CUs hold a whole number of times
// (one more, and all wait for it: 4 sequences of 100,000 keys in 1024 workgroups 305 us,
// in 1056 368 us), unless there are more row blocks than half of that; and fewer than 2 P of
// row blocks that are split, which have partials.  Every wave works this out, a lane per
// sequence: 0.3 us for 64.
// Workgroups reach the XCDs in turn.  Neighbours are of different KV heads, so with eight
// heads (or a multiple) a head's row blocks share one L2, and each XCD works on every
// sequence; whole sequences per XCD have 2% less time where all are alike (32 chunks of 128
// tokens) and 30% more where they are not.  With other numbers of heads, each XCD takes
// a contiguous part of the list, head by head, if there are 32 (sequence, KV head) pairs
// to make the parts alike: 8 chunks of 2048 tokens, 8/4 heads of 256, 573 us, 620 by
// neighbours; fewer pairs are dealt out one by one.  Long row blocks come first.
// MANY: the sequences of more than decode_rows packed rows; otherwise those of at most
// that.  False: no work, or a bad batch, of which nothing is worked on.
template <int ROWS, int SHIFT, bool MANY>
__device__ __forceinline__ bool paged_work(const PagedAttend &p, int item, PagedWork &w) {
    static_assert(ROWS >= 2);
    const int lane = threadIdx.x & 63, G = p.group, S = p.b.sequences, each = (S + 63) / 64;
    struct Need {
        int row_blocks, blocks;  // of each KV head; keys of each
    };
    auto need = [&](const PagedSeq &q) {
        const int rows = q.n * G, most = p.by_group(ROWS - 2) + 2, tokens = q.n < most ? q.n : most;
        const int span = p.window + tokens - 1, keys = q.len < span ? q.len : span;
        const bool here = MANY ? rows > p.decode_rows : rows > 0 && rows <= p.decode_rows;
        return Need{here ? (rows + ROWS - 1) / ROWS : 0, keys > 0 ? (keys + (1 << SHIFT) - 1) >> SHIFT : 1};
    };
    PagedSeq mine{};
    float load = 0.0f, units = 0.0f;  // each lane ends with the same sums
    bool bad = false;
    for (int j = 0; j < each; ++j)
        if (lane * each + j < S) {
            const PagedSeq q = paged_sequence(p.b, lane * each + j);
            const Need n = need(q);
            if (j == 0) mine = q;
            bad |= q.bad;
            units += (float)n.row_blocks;
            load += (float)n.row_blocks * (float)n.blocks;
        }
    raise_status(p.status, bad, ST_BAD_PAGE);
    if (__ballot(bad) != 0) return false;
    for (int d = 1; d < 64 && d < S; d *= 2) {
        load += __shfl_xor(load, d);
        units += __shfl_xor(units, d);
    }
    // Rounded sums: P (at most 32768) splits become P (1 + 2^-17) at most, which no count of
    // workgroups or slots, being whole, passes.
    auto split = [&](int groups) {
        const float left = (float)groups - units * (float)p.hkv, half = 0.5f * (float)groups;
        return load * (float)p.hkv / (left > half ? left : half);
    };
    float share = split(p.groups);
    // Parts so short that their start and join would be most of them: fewer.
    if (p.groups_short < p.groups && share < 4.0f * (float)p.min_blocks) share = split(p.groups_short);
    int blocks = uniform(share < 0x1p30f ? (int)share + 1 : 1 << 30);
    blocks = blocks > p.min_blocks ? blocks : p.min_blocks;

    struct Count {
        int parts, items;
    };
    auto count = [&](const Need &n) {
        // A join costs what some min_blocks more do: a split in two is not worth it.
        int parts = n.blocks <= 2 * p.min_blocks ? 1 : quotient(n.blocks + blocks - 1, blocks);
        parts = parts < p.splits ? parts : p.splits;
        return Count{parts, p.hkv * n.row_blocks * parts};
    };
    int items = 0, slots = 0;
    for (int j = 0; j < each; ++j)
        if (lane * each + j < S) {
            const Count c = count(need(j == 0 ? mine : paged_sequence(p.b, lane * each + j)));
            items += c.items;
            slots += c.parts > 1 ? c.items : 0;
        }
    int items_to = items, slots_to = slots;  // up to this lane's and with them
    for (int d = 1; d < 64 && d < S; d *= 2) {
        const int a = __shfl_up(items_to, d), b = __shfl_up(slots_to, d);
        if (lane >= d) {
            items_to += a;
            slots_to += b;
        }
    }
    bool by_xcd = false;
    if (MANY && p.hkv % 8 != 0 && (each > 1 || __builtin_popcountll(__ballot(items > 0)) * p.hkv >= 32)) {
        const int all = __builtin_amdgcn_readlane(items_to, S < 64 ? S - 1 : 63), x = item % 8;
        if (item >= all) return false;
        item = x * (all / 8) + (x < all % 8 ? x : all % 8) + item / 8;
        by_xcd = true;
    }
    const uint64_t owner = __ballot(item >= items_to - items && item < items_to);
    if (owner == 0) return false;
    const int o = __builtin_ctzll(owner);
    int at = item - __builtin_amdgcn_readlane(items_to - items, o), slot = __builtin_amdgcn_readlane(slots_to - slots, o);
    w.sq.q0 = __builtin_amdgcn_readlane(mine.q0, o);
    w.sq.n = __builtin_amdgcn_readlane(mine.n, o);
    w.sq.len = __builtin_amdgcn_readlane(mine.len, o);
    w.sq.slot = __builtin_amdgcn_readlane(mine.slot, o);
    w.sq.bad = false;
    Need n = need(w.sq);
    Count c = count(n);
    for (int s = o * each + 1; at >= c.items && s < S; ++s) {  // the owner's later sequences
        at -= c.items;
        slot += c.parts > 1 ? c.items : 0;
        w.sq = paged_sequence(p.b, uniform(s));
        n = need(w.sq);
        c = count(n);
    }
    at = uniform(at);
    if (at >= c.items) return false;  // only if the lengths change under the launch
    const int row_blocks = uniform(n.row_blocks), of_head = uniform(row_blocks * c.parts);
    const int high = by_xcd ? quotient(at, of_head) : p.by_hkv(at), rest = by_xcd ? at - high * of_head : high;
    w.parts = uniform(c.parts);
    w.blocks = blocks;
    w.kvh = uniform(by_xcd ? high : at - high * p.hkv);
    const int back = w.parts > 1 ? quotient(rest, w.parts) : rest;
    w.part = uniform(rest - back * w.parts);
    w.rb = uniform(row_blocks - 1 - back);
    w.slot = uniform(slot + (w.kvh * row_blocks + w.rb) * w.parts);
    return w.parts == 1 || w.slot + w.parts <= 2 * p.groups;  // likewise
}

// tanh for FP32 scores: a cap multiplies its error, so small arguments (most, where the cap
// is far above the scores) take the Taylor series, whose error is relative, and others
// 1 - 2 / (1 + e^2|y|) with a refined reciprocal: 2^-22 of the result at 1/2, 2^-23 above.
// The form of tanh_fast for all of them loses a factor of 7 (caps of 30 and 50).
__device__ __forceinline__ float tanh_fp32(float y) {
    const float x = y * y;
    float p = -929569.0f / 638512875.0f;
    p = __builtin_fmaf(p, x, 21844.0f / 6081075.0f);
    p = __builtin_fmaf(p, x, -1382.0f / 155925.0f);
    p = __builtin_fmaf(p, x, 62.0f / 2835.0f);
    p = __builtin_fmaf(p, x, -17.0f / 315.0f);
    p = __builtin_fmaf(p, x, 2.0f / 15.0f);
    p = __builtin_fmaf(p, x, -1.0f / 3.0f);
    const float d = __builtin_amdgcn_exp2f(2.0f * LOG2E * __builtin_fabsf(y)) + 1.0f;
    float r = __builtin_amdgcn_rcpf(d);
    if (d < 0x1p126f) r = __builtin_fmaf(r, __builtin_fmaf(-d, r, 1.0f), r);  // beyond, r is 0 beside 1
    const float far = __builtin_copysignf(__builtin_fmaf(-2.0f, r, 1.0f), y);
    return x <= 0.25f ? __builtin_fmaf(y * x, p, y) : far;
}

// How far a score may pass the row's maximum before the maximum moves, in log2.
constexpr float SLACK = 8.0f;

}  // namespace

}  // namespace tkh
