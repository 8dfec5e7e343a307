// paged_chunk.hip - attention of chunks of new tokens over a page table, 16-bit
// storage: many query rows per KV head, bound by the matrix instructions and by what
// feeds them.
//
// A workgroup takes 128 or 256 packed rows (tokens x query heads of one KV head) of one
// sequence, 32 to a wave, and all keys that they see or a split of them.  K and V come in
// tiles of 32 keys through a ring in LDS, filled by direct global->LDS loads whose page
// number is uniform in a wave (a load run lies in one 16-key block, and those never leave
// a page).
//  * S^T = K Q^T on v_mfma_f32_32x32x16, Q in registers as the B operand: lane l
//    holds query row l % 32 and 16 keys, in the order that the B operand of
//    O^T = V^T P^T wants, if V^T's keys are read in that order too (two transposing
//    LDS loads per operand).  P never moves between lanes.
//  * The scores of tile t + 1 are formed while the softmax of tile t runs and the values
//    of tile t - 1 are added: per matrix instruction six vector instructions, about as
//    many as its time holds.
//  * A row's exponent base is a maximum that it has seen; it moves only when a
//    tile's mass against it passes 2^15, which 16-bit weights and FP32 sums hold.
//  * 256 rows (eight waves, two to a SIMD) where they fill the CUs: 32 chunks of 128 tokens
//    after 4096, 32/8 heads of 128, 326 us against 339 of 128 rows; 855 TFLOP/s.  A prompt
//    of 8192 tokens 560 us, 980 TFLOP/s: of its cycles the matrix instructions fill 47%, the
//    vector ones 48%, LDS 23% without a conflict; a wave waits for LDS, loads or the others
//    in 23%.  (64 rows to a wave need half the LDS reads, but leave one wave to a SIMD with
//    nothing to fill its waits: 720 us.)
//  * 256 features fill the registers with one wave to a SIMD: 8 chunks of 2048 tokens of up
//    to 4096 keys 573 us, 720 TFLOP/s.
//  * Sequences of at most 16 packed rows are left to paged_decode.
#include <cstddef>
#include <type_traits>

#include "paged_device.hpp"

namespace tkh {

namespace {

using f32x16 = float __attribute__((ext_vector_type(16)));

template <int DT> __device__ __forceinline__ f32x16 mfma_32x32x16(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (DT == BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <int DT> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 v = {a, b};
    if constexpr (DT == BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
// sum + the two halves of w, one instruction.
template <int DT> __device__ __forceinline__ float add_pair(uint32_t w, float sum) {
    if constexpr (DT == BF16)
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3f803f80u), sum, false);
    else
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), __builtin_bit_cast(f16x2, 0x3c003c00u), sum, false);
}

// x times c, from and to the accumulator registers: if O lived in vector registers on
// this path alone, every step would copy it over and back.
__device__ __forceinline__ void scale_acc(f32x16 &x, float c) {
    f32x16 t = x;
    asm volatile("" : "+v"(t));
    t *= c;
    asm volatile("" : "+a"(t));
    x = t;
}

__device__ __forceinline__ float uniform_float(float x) { return __builtin_bit_cast(float, uniform(__builtin_bit_cast(int, x))); }

constexpr float MASS_LIMIT = 0x1p15f;
// The base of a row that has seen no key: any finite score is far above it, which
// sends the row's first tile to the exact path; a hidden key's -inf still weighs 0.
constexpr float BASE_NONE = -0x1p100f;

}  // namespace

// The rings: NS groups of TG tiles of 32 keys of K, and as many of V, whose tiles are
// read two steps after K's.  The waves meet once per group.  A tile is runs of 1 KiB,
// each RR whole rows as one direct load of a wave leaves them, with a few bytes between
// runs; a row's 16-byte pieces
// are permuted by its place in the run (piece c at c ^ turn).  The two together
// spread over all banks both the 16 rows that a K read takes at one feature and the
// four rows x 64 bytes that a transposing V read takes; and since the permutation
// touches two bits of c only, a read's address is (x ^ constant) + base + constant.
template <int D, int W> struct ChunkRing {
    static constexpr int KT = 32, NS = 4;
    static constexpr int TG = W == 8 ? 2 : 1;  // tiles of a group
    static constexpr int row = 2 * D;
    static constexpr int RR = 1024 / row;
    static constexpr int runs = KT / RR, wave_runs = 8 / RR;  // eight rows of a group per wave
    static_assert(KT * TG == 8 * W, "a group's rows over its waves");
    static constexpr int k_run = 1024 + 16, v_run = D == 256 ? 1024 + 64 : 1024 + 16;
    static constexpr int k_tile = runs * k_run, v_tile = runs * v_run;
    static constexpr int k_group = TG * k_tile, v_group = TG * v_tile;
    static constexpr int v_base = NS * k_group;
    static constexpr int bytes = v_base + NS * v_group;
    __device__ static constexpr int turn(int rr) {
        return D == 64 ? ((rr >> 1) & 1) << 2 | ((rr >> 2) & 1) << 1 : (D == 128 ? rr << 2 : rr << 3);
    }
    __device__ static constexpr int at(int r, int c, int run) { return r / RR * run + r % RR * row + ((c ^ turn(r % RR)) << 4); }
    // The bits of a piece that the permutation touches, as those of K's step i (pieces
    // 2i, 2i + 1) and V's feature block f (pieces 4f .. 4f + 3), and the other bits.
    static constexpr int bits = D == 64 ? 6 : (D == 128 ? 12 : 8);
    static constexpr int k_turned(int i) { return (2 * i & bits) << 4; }
    static constexpr int k_plain(int i) { return (2 * i & ~bits) << 4; }
    static constexpr int v_turned(int f) { return (4 * f & bits) << 4; }
    static constexpr int v_plain(int f) { return (4 * f & ~bits) << 4; }
};

template <int DT, int D, int W, bool CAP>
__global__ __launch_bounds__(64 * W, W == 8 || D <= 128 ? 2 : 1) void paged_chunk(PagedAttend p) {
    using L = ChunkRing<D, W>;
    constexpr int KT = L::KT, NS = L::NS, TG = L::TG, ROWS = 32 * W, QS = D / 16, FB = D / 32;
    __shared__ __attribute__((aligned(1024))) uint8_t lds_mem[L::bytes];
    lds_ptr<uint8_t> lds = (lds_ptr<uint8_t>)lds_mem;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
    const int G = p.group;

    PagedWork work;
    if (!paged_work<ROWS, 5, true>(p, (int)blockIdx.x, work)) return;
    const PagedSeq &sq = work.sq;
    const int kvh = work.kvh, rb = work.rb, split = work.part;
    const int nrows = uniform(sq.n * G), pos0 = uniform(sq.len - sq.n), len = uniform(sq.len);
    // The tiles that a row of the block sees, and this split's share of them.
    int t_lo, t_hi, active;
    {
        const int r1 = (rb * ROWS + ROWS < nrows ? rb * ROWS + ROWS : nrows) - 1;
        const int lo = pos0 + p.by_group(rb * ROWS) - p.window + 1, hi = pos0 + p.by_group(r1) + 1;
        const int t_first = (lo > 0 ? lo : 0) >> 5, t_end = hi > 0 ? (hi + 31) >> 5 : 0;
        const int all = t_end > t_first ? t_end - t_first : 0;
        active = uniform(work.active(all));
        if (split >= active) return;
        const int per = active > 1 ? quotient(all + active - 1, active) : all;
        t_lo = uniform(t_first + split * per);
        t_hi = t_lo + per < t_first + all ? t_lo + per : t_first + all;
    }
    const int tiles = uniform(t_hi > t_lo ? t_hi - t_lo : 0);

    const int groups = (tiles + TG - 1) / TG;

    // Direct loads: this wave's runs of a group, eight rows of one page.
    const_ptr<int32_t> table = (const_ptr<int32_t>)(p.b.table + (int64_t)uniform(sq.slot) * p.b.table_stride);
    const uint8_t *kb = reinterpret_cast<const uint8_t *>(p.k) + (int64_t)kvh * p.l.head_stride * 2;
    const uint8_t *vb = reinterpret_cast<const uint8_t *>(p.v) + (int64_t)kvh * p.l.head_stride * 2;
    const int row_bytes = (int)p.l.row_stride * 2;
    uint32_t off;
    {
        const int rr = lane * 16 / L::row, c = (lane * 16 % L::row) >> 4;
        off = (uint32_t)(rr * row_bytes + ((c ^ L::turn(rr)) << 4));
    }
    const uint32_t lds0 = (uint32_t)uniform((int)(uintptr_t)lds);
    bool bad_page = false;
    // This wave's first key of group u is key_first + 32 TG u.  A group's page number is
    // loaded an iteration before its place is worked out, that one before K's loads, and
    // V's loads, later, take it from there.  Keys behind the last one repeat its page.
    const int key_first = (t_lo << 5) + wave * 8, last_entry = (len > 0 ? len - 1 : 0) >> p.l.page_shift;
    const uint32_t page_bytes = (uint32_t)p.l.page_stride * 2, page_mask = (1u << p.l.page_shift) - 1;
    auto page_of = [&](int u) {
        const int e = (key_first + KT * TG * u) >> p.l.page_shift;
        return table[e < last_entry ? e : last_entry];
    };
    auto place_of = [&](int u, int page) {
        const bool in = (uint32_t)page < (uint32_t)p.l.pages;
        bad_page |= !in;
        return (uint64_t)(in ? (uint32_t)page : 0u) * page_bytes + (((uint32_t)(key_first + KT * TG * u) & page_mask) * (uint32_t)row_bytes);
    };
    const uint32_t lds_k = lds0 + (uint32_t)wave * (L::wave_runs * L::k_run), lds_v = lds0 + L::v_base + (uint32_t)wave * (L::wave_runs * L::v_run);
    auto issue = [&](auto value, int u, uint64_t at) {
        constexpr bool V = decltype(value)::value;
        const uint8_t *a = uniform_ptr((V ? vb : kb) + at);
        const uint32_t m = V ? lds_v + (uint32_t)(u & (NS - 1)) * L::v_group : lds_k + (uint32_t)(u & (NS - 1)) * L::k_group;
        for (int i = 0; i < L::wave_runs; ++i) lds_load16(a + (uint32_t)(i * L::RR * row_bytes), off, (uint32_t)uniform((int)m) + i * (V ? L::v_run : L::k_run));
    };
    using K = std::false_type;
    using V = std::true_type;

    // This wave's rows: lane row n.  Their loads come first, and are waited for here:
    // the compiler, which does not count the direct loads, would otherwise wait for Q
    // inside the loop, and with it for all of them.
    const int wave_row = rb * ROWS + wave * 32;
    const bool works = wave_row < nrows;  // uniform
    u32x4 q[QS];
    int pos;  // -2^30 - 1: a row past the last, which sees nothing
    {
        const int r = wave_row + n, rr = r < nrows ? r : nrows - 1;
        const int tok = p.by_group(rr), head = kvh * G + rr - tok * G;
        pos = r < nrows ? pos0 + tok : -(1 << 30) - 1;
        for (int s = 0; s < QS; ++s)
            q[s] = *gload_ptr<u32x4>(reinterpret_cast<const uint16_t *>(p.q) + ((int64_t)(sq.q0 + tok) * p.hq + head) * D + 16 * s + 8 * h);
    }
    // Iteration u starts the loads of K of group u + KA and V of group u + VA; the first
    // ones here, in that order: iterations -KA .. -1.
    constexpr int KA = TG == 2 ? 3 : 4, VA = 2;
    uint64_t at_k, at_v[KA - VA];
    int page_next;
    {
        int pages[KA + 1];
        uint64_t at[KA + 1];
        for (int u = 0; u <= KA; ++u) pages[u] = page_of(u);
        page_next = page_of(KA + 1);
        for (int u = 0; u <= KA; ++u) at[u] = place_of(u, pages[u]);
        at_k = at[KA];
        for (int i = 0; i < KA - VA; ++i) at_v[i] = at[VA + i];
        for (int s = 0; s < QS; ++s) asm volatile("" : "+v"(q[s]));
        for (int u = 0; u < KA; ++u) {
            if (u < groups) issue(K{}, u, at[u]);
            const int uv = u - KA + VA;
            if (uv >= 0 && uv < groups) issue(V{}, uv, at[uv]);
        }
    }

    const int wave_last = wave_row + 31 < nrows ? wave_row + 31 : nrows - 1;
    // Keys that every row of the wave sees: [full_lo, full_hi).
    const int full_lo = uniform(pos0 + p.by_group(wave_last) - p.window + 1), full_hi = uniform(pos0 + p.by_group(wave_row) + 1);
    const int first_key = pos0 - p.window + 1 > 0 ? pos0 - p.window + 1 : 0;

    f32x16 o[FB] = {};
    float base = BASE_NONE, l = 0.0f;
    bool bad = false;

    // A cap's tanh(y) = 1 - 2 / (1 + e^2y) goes into one multiply-add with what follows.
    const float cap_k = uniform_float(2.0f * LOG2E * p.softcap_y), cap_2 = uniform_float(-2.0f * p.softcap_log2);
    auto capped = [&](float s, float add) {
        return __builtin_fmaf(__builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s * cap_k) + 1.0f), cap_2, add);
    };
    auto in_log2 = [&](float s) { return CAP ? capped(s, p.softcap_log2) : s * p.scale_log2; };
    // A score's weight against a base; a hidden key's score is -inf.
    auto weight = [&](float s, float from) {
        float x;
        if constexpr (CAP) {
            x = capped(s, p.softcap_log2 - from);
            asm("" : "+v"(x));  // formed always: a branch per weight would cut the steps to pieces
            x = s == NEG_INF ? NEG_INF : x;
        } else x = __builtin_fmaf(s, p.scale_log2, -from);
        return __builtin_amdgcn_exp2f(x);
    };
    // LDS addresses of this lane's operands: a base and the row's permutation.
    uint32_t k_base, k_turn, v_base, v_turn;
    {
        const int j = lane & 15, r = 4 * h + (j >> 2), c = 2 * ((lane >> 4) & 1) + ((j & 3) >> 1), x = L::turn(r % L::RR);
        k_turn = (uint32_t)L::turn(n % L::RR) << 4;
        k_base = lds0 + n / L::RR * L::k_run + n % L::RR * L::row + h * 16;
        v_turn = (uint32_t)(x & ~3) << 4;
        v_base = lds0 + L::v_base + r / L::RR * L::v_run + r % L::RR * L::row + ((c ^ (x & 3)) << 4) + (j & 1) * 8;
    }
    // An operand's address; opaque, so that the constants after it stay in the loads.
    auto turned = [&](uint32_t base, uint32_t turn, int bits) {
        uint32_t x = (turn ^ (uint32_t)bits) + base;
        asm("" : "+v"(x));
        return x;
    };
    auto k_operand = [&](uint32_t base, uint32_t turn, int i) {
        return *(lds_ptr<u32x4>)((lds_ptr<uint8_t>)(uintptr_t)turned(base, turn, L::k_turned(i)) + L::k_plain(i));
    };
    // V^T operand i: feature block i % FB, keys 16 (i / FB) .. + 15.
    auto v_operand = [&](uint32_t base, uint32_t turn, int i) {
        const int first = 16 * (i / FB) / L::RR * L::v_run + L::v_plain(i % FB);
        lds_ptr<uint8_t> x = (lds_ptr<uint8_t>)(uintptr_t)turned(base, turn, L::v_turned(i % FB));
        const u32x2 a = read_tr(x + first), b = read_tr(x + first + 8 / L::RR * L::v_run);
        return u32x4{a[0], a[1], b[0], b[1]};
    };
    // Places of a tile in the rings.
    auto k_place = [&](int t) { return (uint32_t)(t & (NS * TG - 1)) * L::k_tile; };
    auto v_place = [&](int t) { return (uint32_t)(t & (NS * TG - 1)) * L::v_tile; };
    auto meet = [&]() {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // Until the groups that iteration u reads have arrived, and every wave has left
    // iteration u - 1, whose groups the next loads overwrite.  What the last iteration
    // (TG 2) or the last two (TG 1) have started may be under way.
    auto arrive = [&](int u) {
        const int left = groups - u;
        if constexpr (TG == 2) {
            if (left >= 3) wait_loads<2 * L::wave_runs>();
            else if (left == 2) wait_loads<L::wave_runs>();
            else wait_loads<0>();
        } else {
            if (left >= 4) wait_loads<4 * L::wave_runs>();
            else if (left == 3) wait_loads<3 * L::wave_runs>();
            else if (left == 2) wait_loads<2 * L::wave_runs>();
            else if (left == 1) wait_loads<L::wave_runs>();
            else wait_loads<0>();
        }
        meet();
    };
    // Keys of tile t that no row of the sequence sees are whatever the page holds there,
    // NaN too: their V rows become zeros before any wave reads them.
    auto clear_dead = [&](int t) {
        const int key0 = (t_lo + t) << 5;
        if (t < 0 || t >= tiles || (key0 >= first_key && key0 + KT <= len)) return;
        lds_ptr<uint8_t> vt = lds + L::v_base + v_place(t);
        for (int i = threadIdx.x; i < KT * L::row / 16; i += 64 * W) {
            const int r = i * 16 / L::row, key = key0 + r;
            if (key < first_key || key >= len) *(lds_ptr<u32x4>)(vt + L::at(r, i % (L::row / 16), L::v_run)) = u32x4{};
        }
        wait_lds();
        meet();
    };
    // What iteration u starts with: its tiles are there, the next ones' loads begin.
    auto next_loads = [&](int u) {
        arrive(u);
        if (u + KA < groups) issue(K{}, u + KA, at_k);
        if (u + VA < groups) issue(V{}, u + VA, at_v[0]);
        for (int i = 0; i + 1 < KA - VA; ++i) at_v[i] = at_v[i + 1];
        at_v[KA - VA - 1] = at_k;
        at_k = place_of(u + KA + 1, page_next);
        page_next = page_of(u + KA + 2);
        if constexpr (TG == 2) {
            clear_dead(2 * u);
            clear_dead(2 * u + 1);
        } else {
            clear_dead(u - 1);
        }
    };
    // Whether every row of the wave sees every key of tile t.
    auto is_full = [&](int t) {
        const int key0 = (t_lo + t) << 5;
        return key0 >= full_lo && key0 + KT <= full_hi;
    };
    auto hide = [&](int t, f32x16 &s) {
        const int key0 = ((t_lo + t) << 5) + 4 * h;
        for (int i = 0; i < 16; ++i) {
            const int key = key0 + 8 * (i >> 2) + (i & 3);
            const bool seen = key <= pos && key > pos - p.window;
            bad |= seen && !is_finite_f(s[i]);
            s[i] = seen ? s[i] : NEG_INF;
        }
    };
    // A row's base moves up to the tile's maximum, and the tile's weights are formed again.
    // (Seldom: kept apart into small pieces, so that it takes few registers.)
    auto move_base = [&](const f32x16 &s, u32x4 (&w)[2]) {
        float mx = NEG_INF;
        for (int i = 0; i < 16; ++i) {
            float x = in_log2(s[i]);
            if constexpr (CAP) {
                asm("" : "+v"(x));
                x = s[i] == NEG_INF ? NEG_INF : x;
            }
            mx = fmaxf(mx, x);
            __builtin_amdgcn_sched_barrier(0);
        }
        float a0, a1;
        swap_pair(mx, true, a0, a1);
        const float above = fmaxf(base, fmaxf(a0, a1)), c = __builtin_amdgcn_exp2f(base - above);
        l *= c;
        for (int f = 0; f < FB; ++f) {
            if constexpr (D == 256) scale_acc(o[f], c);
            else o[f] *= c;
            __builtin_amdgcn_sched_barrier(0);
        }
        base = above;
        float mass = 0.0f;
        for (int j = 0; j < 8; ++j) {
            const uint32_t both = pack2<DT>(weight(s[2 * j], above), weight(s[2 * j + 1], above));
            w[j >> 2][j & 3] = both;
            mass = add_pair<DT>(both, mass);
            __builtin_amdgcn_sched_barrier(0);
        }
        bad |= !is_finite_f(mass);
        return mass;
    };
    // Scores of tile t + 1, weights of tile t and values of tile t - 1 together, in eight
    // slots of QS / 4 matrix instructions and the weights of one pair of keys, which the
    // scheduler keeps in this order: the vector instructions fill the matrix
    // instructions' time, half of a slot's behind each half of its matrix instructions (a
    // prompt of 8192: 571 us with all behind the last).  The first step adds values and the last forms scores of a tile
    // that is not there: weights of zero against a cleared tile, and scores that nobody
    // uses.
    auto step = [&](int t, f32x16 &now, f32x16 &next, u32x4 (&w)[2], const u32x4 (&before)[2]) {
        const uint32_t ka = k_base + k_place(t + 1), va = v_base + v_place(t - 1);
        const bool full = is_full(t);
        if (!full) hide(t, now);
        // Not the same from step to step, as far as the compiler knows: it would keep a
        // register for each operand's address.
        uint32_t kx = k_turn, vx = v_turn;
        asm volatile("" : "+v"(kx), "+v"(vx));
        asm volatile("" : "+v"(now));  // in vector registers, not among the accumulators
        u32x4 k = k_operand(ka, kx, 0), v = v_operand(va, vx, 0);
        float mass = 0.0f, top = 0.0f, x0 = 0.0f, x1 = 0.0f;
        auto pack = [&](int j) {  // the pair that the slot before weighed
            const uint32_t both = pack2<DT>(x0, x1);
            w[j >> 2][j & 3] = both;
            mass = add_pair<DT>(both, mass);
        };
        auto vector_work = [&](int u, int part) {  // of slot u, in two parts
            if (part == 0) {
                if (u > 0) pack(u - 1);
                x0 = weight(now[2 * u], base);
            } else {
                top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, __builtin_fabsf(now[2 * u])), __builtin_fabsf(now[2 * u + 1]));
                x1 = weight(now[2 * u + 1], base);
            }
        };
        // A cap's longer chains want more room to be spread in: slots of two pairs (24 chunks of
        // 1024 tokens, 128 features, 540 us; 590 with one).
        constexpr int PAIRS = CAP && D == 128 ? 2 : 1, MS = PAIRS * QS / 4;
#pragma unroll
        for (int u = 0; u < 8; u += PAIRS) {
#pragma unroll
            for (int z = 0; z < MS; ++z) {
                if (PAIRS == 1 || z == 0) __builtin_amdgcn_sched_barrier(0);
                const int m = u * (QS / 4) + z, i = m / 2;
                if (m % 2 == 0) {
                    o[i % FB] = mfma_32x32x16<DT>(v, before[i / FB], o[i % FB]);
                    if (i + 1 < QS) v = v_operand(va, vx, i + 1);
                } else {
                    next = mfma_32x32x16<DT>(k, q[i], i == 0 ? f32x16{} : next);
                    if (i + 1 < QS) k = k_operand(ka, kx, i + 1);
                }
                if (PAIRS == 1 && (MS == 1 || z == MS / 2 - 1)) vector_work(u, 0);
                if (PAIRS == 1 && z == MS - 1) vector_work(u, 1);
            }
            for (int w = 0; PAIRS == 2 && w < 4; ++w) vector_work(u + w / 2, w % 2);
        }
        __builtin_amdgcn_sched_barrier(0);
        pack(7);
        bad |= full && !(top < __builtin_inff());
        if (__builtin_expect(__ballot(!(mass <= MASS_LIMIT)) != 0, 0)) mass = move_base(now, w);
        l += mass;
    };

    for (int i = threadIdx.x; i < L::v_group / 16; i += 64 * W) *(lds_ptr<u32x4>)(lds + L::v_base + (NS - 1) * L::v_group + i * 16) = u32x4{};
    wait_lds();
    if (tiles > 0) {
        f32x16 sa, sb;
        u32x4 wa[2] = {}, wb[2] = {};
        arrive(0);
        for (int i = 0; i < QS; ++i) sa = mfma_32x32x16<DT>(k_operand(k_base, k_turn, i), q[i], i == 0 ? f32x16{} : sa);
        wait_lds();
        auto last_values = [&](const u32x4 (&w)[2]) {
            if constexpr (TG == 1) {
                arrive(tiles);
                clear_dead(tiles - 1);
            }
            if (!works) return;
            const uint32_t va = v_base + v_place(tiles - 1);
            for (int i = 0; i < QS; ++i) o[i % FB] = mfma_32x32x16<DT>(v_operand(va, v_turn, i), w[i / FB], o[i % FB]);
        };
        for (int t = 0;;) {
            next_loads(t / TG);
            if (works) step(t, sa, sb, wa, wb);
            if (++t == tiles) {
                last_values(wa);
                break;
            }
            if constexpr (TG == 1) {
                wait_lds();
                next_loads(t);
            }
            if (works) step(t, sb, sa, wb, wa);
            if (++t == tiles) {
                last_values(wb);
                break;
            }
            wait_lds();
        }
    }

    raise_status(p.status, bad_page, ST_BAD_PAGE);
    raise_status(p.status, bad, ST_NONFINITE_INPUT);
    if (!works) return;
    float a0, a1;
    swap_pair(l, true, a0, a1);
    float mass = a0 + a1;
    int r = wave * 32 + n;  // row in the block
    asm volatile("" : "+v"(r));  // formed again here: nothing of it lives through the loop
    // Splits: a wave's partial as its registers have it, so that a lane reads back what the
    // same lane of another split stored.  Each wave counts the splits that have arrived;
    // the last one adds all of them up in split order, so the result does not depend on
    // who is last, and leaves the counter at 0.
    if (active > 1) {
        const int64_t slot0 = work.slot, wave_floats = 32 * D;
        auto part = [&](int s) { return __builtin_amdgcn_make_buffer_rsrc(p.part_o + ((slot0 + s) * W + wave) * wave_floats, 0, 0x7FFFFFFF, 0x00020000); };
        auto pair = [&](int s) { return p.part_ml + (((slot0 + s) * W + wave) * 32 + n) * 2; };
        {
            const __amdgpu_buffer_rsrc_t to = part(split);
            for (int f = 0; f < FB; ++f)
                for (int i = 0; i < 4; ++i)
                    __builtin_amdgcn_raw_buffer_store_b128(
                        __builtin_bit_cast(u32x4, f32x4{o[f][4 * i], o[f][4 * i + 1], o[f][4 * i + 2], o[f][4 * i + 3]}), to,
                        (uint32_t)lane * 16u + (uint32_t)(4 * f + i) * 1024u, 0, CPOL_SC1);
        }
        if (h == 0) {
            shared_store(pair(split), base);
            shared_store(pair(split) + 1, mass);
        }
        wait_loads<0>();
        uint32_t *const counter = p.counters + slot0 * W + wave;
        uint32_t old = 0;
        if (lane == 0) old = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (uniform((int)old) != active - 1) return;
        asm volatile("" ::: "memory");  // the loads come after the count
        if (lane == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        float top = BASE_NONE;
        for (int s = 0; s < active; ++s) top = fmaxf(top, shared_load(pair(s)));
        mass = 0.0f;
        for (int f = 0; f < FB; ++f) o[f] = f32x16{};
        for (int s = 0; s < active; ++s) {
            const float c = __builtin_amdgcn_exp2f(shared_load(pair(s)) - top);
            mass = __builtin_fmaf(c, shared_load(pair(s) + 1), mass);
            const __amdgpu_buffer_rsrc_t from = part(s);
            for (int f = 0; f < FB; ++f) {
                f32x4 x[4];
                for (int i = 0; i < 4; ++i)
                    x[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, (uint32_t)lane * 16u + (uint32_t)(4 * f + i) * 1024u, 0, CPOL_SC1));
                for (int i = 0; i < 16; ++i) o[f][i] = __builtin_fmaf(c, x[i >> 2][i & 3], o[f][i]);
            }
        }
    }
    bool bad_out = false;
    if (rb * ROWS + r < nrows) {
        const int tok = p.by_group(rb * ROWS + r), head = kvh * G + rb * ROWS + r - tok * G;
        const float inv = 1.0f / mass;
        for (int f = 0; f < FB; ++f)
            for (int i = 0; i < 4; ++i) {
                f32x4 y = {};
                if (pos0 + tok >= 0)
                    for (int j = 0; j < 4; ++j) {
                        y[j] = o[f][4 * i + j] * inv;
                        bad_out |= !is_finite_f(y[j]);
                    }
                store_elem4<DT>(p.out, ((int64_t)(sq.q0 + tok) * p.hq + head) * D + 32 * f + 8 * i + 4 * h, y);
            }
    }
    raise_status(p.status, bad_out, ST_NONFINITE_OUTPUT);
}

}  // namespace tkh

namespace {

template <class F> hipError_t chunk_build(int dtype, int d, int waves, bool cap, F f) {
    using namespace tkh;
    auto caps = [&](auto dt, auto dims, auto w) {
        return cap ? f(dt, dims, w, std::true_type{}) : f(dt, dims, w, std::false_type{});
    };
    auto rows = [&](auto dt, auto dims) {
        if constexpr (decltype(dims)::value <= 128) {
            if (waves == 8) return caps(dt, dims, std::integral_constant<int, 8>{});
        }
        return caps(dt, dims, std::integral_constant<int, 4>{});
    };
    auto heads = [&](auto dt) {
        if (d == 64) return rows(dt, std::integral_constant<int, 64>{});
        if (d == 128) return rows(dt, std::integral_constant<int, 128>{});
        return rows(dt, std::integral_constant<int, 256>{});
    };
    if (dtype == F16) return heads(std::integral_constant<int, F16>{});
    if (dtype == BF16) return heads(std::integral_constant<int, BF16>{});
    return hipErrorInvalidValue;
}

}  // namespace

// Most waves of a chunk workgroup, 32 rows each (it has these or 4).
extern "C" int tkh_paged_chunk_waves(int d) { return d <= 128 ? 8 : 4; }

extern "C" hipError_t tkh_launch_paged_chunk(const tkh::PagedAttend *p, int dtype, int d, int waves, int groups,
                                             hipStream_t stream, hipEvent_t start, hipEvent_t stop) {
    return chunk_build(dtype, d, waves, p->softcap_y != 0.0f, [&](auto dt, auto dims, auto w, auto cap) {
        constexpr int W = decltype(w)::value;
        hipExtLaunchKernelGGL((tkh::paged_chunk<decltype(dt)::value, decltype(dims)::value, W, decltype(cap)::value>),
                              dim3((unsigned)groups), dim3(64 * W), 0, stream, start, stop, 0, *p);
        return hipGetLastError();
    });
}
