// paged_attend.hip - attention over a page table.
//
// Query i of a sequence's n new tokens, at position p = L - n + i of L keys, sees
// keys j <= p with p - j < window; s_j = scale q.k_j (capped: c tanh(s_j / c)),
// o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), in one pass with a running
// maximum m and mass.  Scores live in units of log2.
//
// paged_decode: blocks of 16 NR packed rows (tokens x query heads of one KV head); for
// 16-bit storage one block of 16, and more rows are the chunk kernel's, for FP32
// storage any number.  Bound by the bytes of K and V with few rows (4 sequences of 100,000
// to 131,000 keys 307 us, 6.5 TB/s; 64 of 512 to 8192 keys 190 us, 5.9 TB/s; a copy of
// 2 GiB reads and writes 4.85), by the FP32 matrix instructions (1/16 of the 16-bit
// ones' rate) with many (4 chunks of 128 tokens, 14/2 heads of 64, 49 us, 53 TFLOP/s).
//  * The keys are cut into blocks of 16, which never leave a page, and a
//    workgroup takes one split of them.  Its waves take blocks in turn, each
//    through a ring of its own in LDS filled by direct global->LDS loads: no
//    barrier, no register waits for memory, and the page number of a block is
//    wave-uniform, so its address is one scalar base.
//  * S^T = K Q^T on v_mfma_f32_16x16x32 (FP32: 16x16x4), K rows as the A operand
//    straight from LDS, which leaves lane l with query row l % 16 and keys
//    4 (l / 16) + 0..3: the B operand of O^T = V^T P^T on 16x16x16 (FP32: four
//    16x16x4, one key of each lane group at a time), so P never moves between
//    lanes.  16-bit V^T is read by the transposing LDS load.
//  * Rows' maxima move only when a score passes them by 8 (a factor of 256,
//    which FP32 sums and 16-bit weights hold).
//  * Splits store their partial and count up an arrival counter; the last one
//    to arrive merges all of them in split order, so the result does not depend
//    on who is last, and leaves the counter at 0.
#include <cstddef>
#include <type_traits>

#include "paged_device.hpp"

namespace tkh {

namespace {

__device__ __forceinline__ f32x4 mfma_16x16x4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

}  // namespace

// The ring of one wave: NS stages of one 16-key block, K rows then V rows.  Rows hold
// their 16-byte pieces permuted (piece c of row r at c ^ turn(r)), so that the rows
// read at one feature fall on different bank groups.
template <int DT, int D> struct DecodeRing {
    static constexpr int ES = ElemSize<DT>::value;
    static constexpr int row = ES * D;
    static constexpr int W = row >= 512 ? 2 : 4;         // waves per workgroup
    static constexpr int NS = row == 128 ? 4 : 2;        // stages per wave
    static constexpr int tile = 16 * row;
    static constexpr int stage = 2 * tile;
    static constexpr int wave_bytes = NS * stage;
    static constexpr int bytes = W * wave_bytes;         // 64 KiB (two workgroups per CU); FP32 256-wide 128
    static constexpr int loads = tile / 1024;            // direct loads per tile
    __device__ static constexpr int turn(int r) { return row == 128 ? (r >> 1) & 7 : r & 15; }
    __device__ static constexpr int at(int r, int c) { return r * row + ((c ^ turn(r)) << 4); }
};

template <int DT, int D, int NR, bool CAP>
__global__ __launch_bounds__((64 * DecodeRing<DT, D>::W)) void paged_decode(PagedAttend p) {
    using L = DecodeRing<DT, D>;
    constexpr bool HALF = DT != F32;
    constexpr int W = L::W, NS = L::NS, FT = D / 16, QP = HALF ? D / 32 : D / 16, ROWS = 16 * NR;  // QP: 16-byte pieces of a row per lane
    __shared__ __attribute__((aligned(1024))) uint8_t lds_mem[L::bytes];
    __shared__ float lds_ml[W][ROWS][2];
    __shared__ float lds_mass[64 * W];
    __shared__ uint32_t lds_last;
    lds_ptr<uint8_t> lds = (lds_ptr<uint8_t>)lds_mem;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, n = lane & 15;
    const int G = p.group;
    PagedWork work;
    if (!paged_work<ROWS, 4, false>(p, (int)blockIdx.x, work)) return;
    const PagedSeq &sq = work.sq;
    const int kvh = work.kvh, split = work.part;
    const int all_rows = uniform(sq.n * G), pos0 = uniform(sq.len - sq.n), len = uniform(sq.len);
    const int row0 = work.rb * ROWS;
    const int nrows = all_rows - row0 < ROWS ? all_rows - row0 : ROWS;
    const int tok0 = p.by_group(row0), tok1 = p.by_group(row0 + nrows - 1);  // tokens of the first and the last row

    // The blocks that some row sees, and this split's share of them.
    const int first_key = pos0 - p.window + 1 > 0 ? pos0 - p.window + 1 : 0;  // of the sequence
    const int see_lo = pos0 + tok0 - p.window + 1 > 0 ? pos0 + tok0 - p.window + 1 : 0, see_hi = pos0 + tok1 + 1;
    const int b_first = see_lo >> 4, b_end = see_hi > 0 ? (see_hi + 15) >> 4 : 0;
    const int blocks = b_end > b_first ? b_end - b_first : 0;
    const int active = work.active(blocks);
    if (split >= active) return;
    const int per = active > 1 ? quotient(blocks + active - 1, active) : blocks;
    const int b_lo = uniform(b_first + split * per);
    const int b_hi = b_lo + per < b_end ? b_lo + per : b_end;
    const int mine = uniform(b_hi - b_lo > wave ? (b_hi - b_lo - wave + W - 1) / W : 0);

    const_ptr<int32_t> table = (const_ptr<int32_t>)(p.b.table + (int64_t)uniform(sq.slot) * p.b.table_stride);
    const uint8_t *kb = reinterpret_cast<const uint8_t *>(p.k) + (int64_t)kvh * p.l.head_stride * L::ES;
    const uint8_t *vb = reinterpret_cast<const uint8_t *>(p.v) + (int64_t)kvh * p.l.head_stride * L::ES;
    const uint32_t row_bytes = (uint32_t)p.l.row_stride * L::ES, page_mask = (1u << p.l.page_shift) - 1;
    const uint64_t page_bytes = (uint64_t)p.l.page_stride * L::ES;
    uint32_t off[L::loads];
    for (int i = 0; i < L::loads; ++i) {
        const int at = i * 1024 + lane * 16, r = at / L::row, c = (at % L::row) >> 4;
        off[i] = (uint32_t)r * row_bytes + (uint32_t)((c ^ L::turn(r)) << 4);
    }
    const uint32_t ring = (uint32_t)uniform((int)(uintptr_t)(lds + wave * L::wave_bytes));
    bool bad_page = false;
    auto page_of = [&](int t) { return table[((b_lo + wave + t * W) << 4) >> p.l.page_shift]; };
    auto issue = [&](int t, int page) {
        const int key = (b_lo + wave + t * W) << 4;
        if ((uint32_t)page >= (uint32_t)p.l.pages) {
            page = 0;
            bad_page = true;
        }
        const uint64_t at = (uint64_t)page * page_bytes + ((uint32_t)key & page_mask) * row_bytes;
        const uint8_t *ka = uniform_ptr(kb + at), *va = uniform_ptr(vb + at);
        const uint32_t m = ring + (uint32_t)(t % NS) * L::stage;
        for (int i = 0; i < L::loads; ++i) lds_load16_once(ka, off[i], m + i * 1024);
        for (int i = 0; i < L::loads; ++i) lds_load16_once(va, off[i], m + L::tile + i * 1024);
    };

    {
        int pages[NS];
        for (int t = 0; t < NS; ++t) pages[t] = t < mine ? page_of(t) : 0;
        for (int t = 0; t < NS; ++t)
            if (t < mine) issue(t, pages[t]);
    }
    // This lane's query rows (rows past the last repeat it and see nothing).  16-bit
    // storage: the features of the matrix instruction's B operand; FP32: a lane group's
    // quarter of the features, one at a time, as K's reads have them.
    u32x4 q[NR][QP];
    int lo[NR], hi[NR];  // visible keys [lo, hi)
    for (int a = 0; a < NR; ++a) {
        const int rr = row0 + (16 * a + n < nrows ? 16 * a + n : nrows - 1), tok = p.by_group(rr), head = kvh * G + rr - tok * G;
        const uint8_t *at = reinterpret_cast<const uint8_t *>(p.q) + ((int64_t)(sq.q0 + tok) * p.hq + head) * L::row;
        for (int s = 0; s < QP; ++s) q[a][s] = *gload_ptr<u32x4>(at + 16 * (HALF ? 4 * s + g : QP * g + s));
        lo[a] = pos0 + tok - p.window + 1;
        hi[a] = 16 * a + n < nrows ? pos0 + tok + 1 : INT32_MIN;
    }
    const int all_lo = pos0 + tok1 - p.window + 1, all_hi = nrows == ROWS ? pos0 + tok0 + 1 : INT32_MIN;  // keys that every row sees
    // Q is loaded behind the first stages and waited for at its first use: waiting for it
    // here, and so for all the first stages, costs 6% (4 sequences of 100,000 keys: 342
    // instead of 322 us).

    f32x4 acc[NR][FT] = {};
    float m[NR], l[NR];
    for (int a = 0; a < NR; ++a) {
        m[a] = NEG_INF;
        l[a] = 0.0f;
    }
    bool bad = false;
    for (int t = 0; t < mine; ++t) {
        // The next block's page number arrives while this one is waited for.
        const int page_next = t + NS < mine ? page_of(t + NS) : 0;
        // Loads of later stages may stay under way.
        const int ahead = mine - 1 - t < NS - 1 ? mine - 1 - t : NS - 1;
        if (NS == 4 && ahead >= 3) wait_loads<NS == 4 ? 3 * 2 * L::loads : 0>();
        else if (NS == 4 && ahead == 2) wait_loads<NS == 4 ? 2 * 2 * L::loads : 0>();
        else if (ahead >= 1) wait_loads<2 * L::loads < 64 ? 2 * L::loads : 63>();
        else wait_loads<0>();
        lds_ptr<uint8_t> kt = lds + (wave * L::wave_bytes + (t % NS) * L::stage), vt = kt + L::tile;
        const int key0 = (b_lo + wave + t * W) << 4;
        f32x4 s[NR] = {};
        for (int i = 0; i < QP; ++i) {
            const u32x4 k = *(lds_ptr<u32x4>)(kt + L::at(n, HALF ? 4 * i + g : QP * g + i));
            for (int a = 0; a < NR; ++a) {
                if constexpr (HALF) {
                    s[a] = mfma_16x16x32<DT>(k, q[a][i], s[a]);
                } else {
                    const f32x4 kf = __builtin_bit_cast(f32x4, k), qf = __builtin_bit_cast(f32x4, q[a][i]);
                    for (int e = 0; e < 4; ++e) s[a] = mfma_16x16x4(kf[e], qf[e], s[a]);
                }
            }
        }
        // V^T operands: this lane's feature of each 16, keys 4g .. 4g + 3.
        u32x2 v[HALF ? FT : 1];
        if constexpr (HALF)
            for (int f = 0; f < FT; ++f) v[f] = read_tr(vt + L::at(4 * g + (n >> 2), 2 * f + ((n & 3) >> 1)) + (n & 1) * 8);
        const bool inside = key0 >= all_lo && key0 + 16 <= all_hi;
        // Whether the page's rows hold keys that no row of the sequence sees: whatever is
        // there, NaN too, must weigh nothing.
        const bool dead = key0 < first_key || key0 + 16 > len;
        if (HALF && dead) {
            uint32_t keep[2];
            for (int i = 0; i < 2; ++i) {
                const int key = key0 + 4 * g + 2 * i;
                keep[i] = (key >= first_key && key < len ? 0xffffu : 0u) | (key + 1 >= first_key && key + 1 < len ? 0xffff0000u : 0u);
            }
            for (int f = 0; f < (HALF ? FT : 1); ++f) v[f] = u32x2{v[f][0] & keep[0], v[f][1] & keep[1]};
        }
        f32x4 w[NR];
        u32x2 pw[NR];
        for (int a = 0; a < NR; ++a) {
            float x[4];
            for (int i = 0; i < 4; ++i) x[i] = CAP ? (HALF ? tanh_fast(s[a][i] * p.softcap_y) : tanh_fp32(s[a][i] * p.softcap_y)) * p.softcap_log2 : s[a][i] * p.scale_log2;
            if (inside) {
                for (int i = 0; i < 4; ++i) bad |= !is_finite_f(s[a][i]);
            } else {
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 4 * g + i;
                    const bool seen = key >= lo[a] && key < hi[a];
                    bad |= seen && !is_finite_f(s[a][i]);
                    x[i] = seen ? x[i] : NEG_INF;
                }
            }
            const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            if (__ballot(top > m[a] + SLACK) != 0) {
                const float mn = fmaxf(m[a], quad_max(top));
                const float c = mn == NEG_INF ? 1.0f : __builtin_amdgcn_exp2f(m[a] - mn);
                m[a] = mn;
                l[a] *= c;
                for (int f = 0; f < FT; ++f) acc[a][f] *= c;
            }
            const float base = m[a] == NEG_INF ? 0.0f : m[a];
            for (int i = 0; i < 4; ++i) w[a][i] = __builtin_amdgcn_exp2f(x[i] - base);
            if constexpr (HALF) {
                pw[a] = pack4<DT>(w[a]);  // the mass is summed from the weights as rounded
                w[a] = unpack4<DT>(pw[a]);
            }
            l[a] += (w[a][0] + w[a][1]) + (w[a][2] + w[a][3]);
        }
        for (int f = 0; f < FT; ++f) {
            if constexpr (HALF) {
                for (int a = 0; a < NR; ++a) acc[a][f] = mfma_16x16x16<DT>(v[f], pw[a], acc[a][f]);
            } else {
                float vf[4];
                for (int i = 0; i < 4; ++i) vf[i] = *(lds_ptr<float>)(vt + L::at(4 * g + i, 4 * f + (n >> 2)) + (n & 3) * 4);
                if (dead)
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + 4 * g + i;
                        vf[i] = key >= first_key && key < len ? vf[i] : 0.0f;
                    }
                for (int i = 0; i < 4; ++i)
                    for (int a = 0; a < NR; ++a) acc[a][f] = mfma_16x16x4(vf[i], w[a][i], acc[a][f]);
            }
        }
        if (t + NS < mine) {
            wait_lds();
            issue(t + NS, page_next);
        }
    }
    for (int a = 0; a < NR; ++a) l[a] = quad_sum(l[a]);

    // The waves' results through LDS (each in its own ring), then one thread per
    // four features of a row.
    constexpr int OS = D + 4;  // floats between rows
    static_assert(ROWS * OS * 4 <= L::wave_bytes, "a wave's context fits its ring");
    static_assert(pairs_bytes(PAGED_PAIRS_MAX) + 64 * W * 16 <= L::bytes, "the merge's pairs and sums");
    wait_lds();
    {
        lds_ptr<float> o = (lds_ptr<float>)(lds + wave * L::wave_bytes);
        for (int a = 0; a < NR; ++a) {
            for (int f = 0; f < FT; ++f) *(lds_ptr<f32x4>)(o + (16 * a + n) * OS + 16 * f + 4 * g) = acc[a][f];
            if (g == 0) {
                lds_ml[wave][16 * a + n][0] = m[a];
                lds_ml[wave][16 * a + n][1] = l[a];
            }
        }
    }
    raise_status(p.status, bad_page, ST_BAD_PAGE);
    raise_status(p.status, bad, ST_NONFINITE_INPUT);
    __syncthreads();
    const int64_t slot0 = work.slot, slot = slot0 + split;
    const __amdgpu_buffer_rsrc_t to = __builtin_amdgcn_make_buffer_rsrc(p.part_o + slot * p.rows * D, 0, 0x7FFFFFFF, 0x00020000);
    bool bad_out = false;
    auto finish = [&](int r, int d, f32x4 o, float mass) {
        const int tok = p.by_group(row0 + r), head = kvh * G + row0 + r - tok * G;
        f32x4 y = {};
        if (pos0 + tok >= 0)
            for (int i = 0; i < 4; ++i) {
                y[i] = o[i] / mass;
                bad_out |= !is_finite_f(y[i]);
            }
        store_elem4<DT>(p.out, ((int64_t)(sq.q0 + tok) * p.hq + head) * D + d, y);
    };
    for (int i = threadIdx.x; i < nrows * (D / 4); i += 64 * W) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float M = NEG_INF, mass = 0.0f;
        for (int w = 0; w < W; ++w) M = fmaxf(M, lds_ml[w][r][0]);
        const float base = M == NEG_INF ? 0.0f : M;
        f32x4 o = {};
        for (int w = 0; w < W; ++w) {
            const float c = __builtin_amdgcn_exp2f(lds_ml[w][r][0] - base);
            mass += c * lds_ml[w][r][1];
            const f32x4 ow = *(lds_ptr<f32x4>)((lds_ptr<float>)(lds + w * L::wave_bytes) + r * OS + d);
            for (int j = 0; j < 4; ++j) o[j] = __builtin_fmaf(c, ow[j], o[j]);
        }
        if (active == 1) {
            finish(r, d, o, mass);
        } else {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), to, (uint32_t)(r * D + d) * 4u, 0, CPOL_SC1);
            if (d == 0) {
                shared_store(p.part_ml + (slot * p.rows + r) * 2, M);
                shared_store(p.part_ml + (slot * p.rows + r) * 2 + 1, mass);
            }
        }
    }
    if (active > 1) {
        wait_loads<0>();
        __syncthreads();  // every thread's stores come before the count
        if (threadIdx.x == 0) {
            const uint32_t old = __hip_atomic_fetch_add(p.counters + slot0, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            lds_last = old == (uint32_t)active - 1 ? 1u : 0u;
            if (lds_last) __hip_atomic_store(p.counters + slot0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!lds_last) return;
        // Every (maximum, mass) pair at once, into LDS; then each thread sums four
        // features of a row over its share of the splits, several loads under way.
        lds_ptr<f32x2> ml = (lds_ptr<f32x2>)lds;
        const int pairs = nrows * active, items = nrows * (D / 4);
        const float *part_ml = p.part_ml + slot0 * p.rows * 2, *part_o = p.part_o + slot0 * p.rows * D;
        for (int i = threadIdx.x; i < pairs; i += 64 * W) {
            const int s = i / nrows, r = i % nrows;
            ml[i] = f32x2{shared_load(part_ml + (s * p.rows + r) * 2), shared_load(part_ml + (s * p.rows + r) * 2 + 1)};
        }
        __syncthreads();
        const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(part_o), 0, 0x7FFFFFFF, 0x00020000);
        // Threads share an item's splits when there are fewer items than threads.
        const int shares = items >= 64 * W ? 1 : 64 * W / items;
        lds_ptr<f32x4> sums = (lds_ptr<f32x4>)(lds + pairs_bytes(pairs));
        for (int i0 = threadIdx.x; i0 < items * shares; i0 += 64 * W) {
            const int i = i0 % items, share = i0 / items, r = i / (D / 4), d = i % (D / 4) * 4;
            float M = NEG_INF, mass = 0.0f;
            for (int s = 0; s < active; ++s) M = fmaxf(M, ml[s * nrows + r][0]);
            const float base = M == NEG_INF ? 0.0f : M;
            f32x4 o = {};
            constexpr int U = 8;
            for (int s0 = share; s0 < active; s0 += U * shares) {
                f32x4 part[U];
                for (int u = 0; u < U; ++u) {
                    const int s = s0 + u * shares;
                    // Past the last split: out of the buffer's range, which reads as 0.
                    const uint32_t at = s < active ? (uint32_t)((s * p.rows + r) * D + d) * 4u : 0x80000000u;
                    part[u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, CPOL_SC1));
                }
                for (int u = 0; u < U; ++u) {
                    const int s = s0 + u * shares;
                    const float c = s < active ? __builtin_amdgcn_exp2f(ml[s * nrows + r][0] - base) : 0.0f;
                    for (int j = 0; j < 4; ++j) o[j] = __builtin_fmaf(c, part[u][j], o[j]);
                }
            }
            for (int s = 0; s < active; ++s) mass = __builtin_fmaf(__builtin_amdgcn_exp2f(ml[s * nrows + r][0] - base), ml[s * nrows + r][1], mass);
            if (shares == 1) {
                finish(r, d, o, mass);
            } else {
                sums[i0] = o;
                lds_mass[i0] = mass;
            }
        }
        if (shares > 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < items; i += 64 * W) {
                f32x4 o = sums[i];
                for (int share = 1; share < shares; ++share) o += sums[share * items + i];
                finish(i / (D / 4), i % (D / 4) * 4, o, lds_mass[i]);
            }
        }
    }
    raise_status(p.status, bad_out, ST_NONFINITE_OUTPUT);
}

}  // namespace tkh

extern "C" hipError_t tkh_launch_paged_decode(const tkh::PagedAttend *p, int dtype, int d, int groups, hipStream_t stream,
                                              hipEvent_t start, hipEvent_t stop) {
    using namespace tkh;
    const dim3 grid((unsigned)groups);
    auto go = [&](auto kernel, int waves) {
        hipExtLaunchKernelGGL(kernel, grid, dim3(64 * waves), 0, stream, start, stop, 0, *p);
        return hipGetLastError();
    };
    auto rows = [&](auto dt, auto dims, auto cap) {
        constexpr int DT = decltype(dt)::value, D = decltype(dims)::value;
        constexpr bool CAP = decltype(cap)::value;
        if constexpr (DT == F32) {
            if (p->rows > 16) return go(paged_decode<DT, D, 2, CAP>, DecodeRing<DT, D>::W);
        }
        return go(paged_decode<DT, D, 1, CAP>, DecodeRing<DT, D>::W);
    };
    auto dims = [&](auto dt, auto cap) {
        if (d == 64) return rows(dt, std::integral_constant<int, 64>{}, cap);
        if (d == 128) return rows(dt, std::integral_constant<int, 128>{}, cap);
        return rows(dt, std::integral_constant<int, 256>{}, cap);
    };
    auto caps = [&](auto dt) { return p->softcap_y != 0.0f ? dims(dt, std::true_type{}) : dims(dt, std::false_type{}); };
    if (dtype == F32) return caps(std::integral_constant<int, F32>{});
    if (dtype == F16) return caps(std::integral_constant<int, F16>{});
    if (dtype == BF16) return caps(std::integral_constant<int, BF16>{});
    return hipErrorInvalidValue;
}
