// paged_attend.hip - attention over a page table.
//
// Query i of a sequence's n new tokens, at position p = L - n + i of L keys, sees
// keys j <= p with p - j < window; s_j = scale q.k_j (capped: c tanh(s_j / c)),
// o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), in one pass with a running
// maximum m and mass.  Scores live in units of log2.
//
// paged_decode: up to 16 packed rows (tokens x query heads of one KV head) per
// (sequence, KV head), 16-bit storage; bound by the bytes of K and V.
//  * The keys are cut into blocks of 16, which never leave a page, and a
//    workgroup takes one split of them.  Its waves take blocks in turn, each
//    through a ring of its own in LDS filled by direct global->LDS loads: no
//    barrier, no register waits for memory, and the page number of a block is
//    wave-uniform, so its address is one scalar base.
//  * S^T = K Q^T on v_mfma_f32_16x16x32 (K rows as the A operand straight from
//    LDS), which leaves lane l with query row l % 16 and keys 4 (l / 16) + 0..3:
//    the B operand of O^T = V^T P^T on v_mfma_f32_16x16x16, so P never moves
//    between lanes.  V^T is read by the transposing LDS load.
//  * Rows' maxima move only when a score passes them by 8 (a factor of 256,
//    which FP32 sums and 16-bit weights hold).
//  * Splits store their partial and count up an arrival counter; the last one
//    to arrive merges all of them in split order, so the result does not depend
//    on who is last, and leaves the counter at 0.
//
// paged_rows: one wave per (query row, head), FP32 throughout.
#include <cstddef>
#include <type_traits>

#include "paged_device.hpp"

namespace tkh {

// The ring of one wave: NS stages of one 16-key block, K rows then V rows of 2D
// bytes.  Rows hold their 16-byte pieces permuted (piece c of row r at c ^ turn(r)),
// so that 16 rows read at one feature fall on 16 different bank groups.
template <int D> struct DecodeRing {
    static constexpr int W = D == 256 ? 2 : 4;          // waves per workgroup
    static constexpr int NS = D == 64 ? 4 : 2;          // stages per wave
    static constexpr int row = 2 * D;
    static constexpr int tile = 16 * row;
    static constexpr int stage = 2 * tile;
    static constexpr int wave_bytes = NS * stage;
    static constexpr int bytes = W * wave_bytes;         // 64 KiB: two workgroups per CU
    static constexpr int loads = tile / 1024;            // direct loads per tile
    __device__ static constexpr int turn(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
    __device__ static constexpr int at(int r, int c) { return r * row + ((c ^ turn(r)) << 4); }
};

template <int DT, int D, bool CAP>
__global__ __launch_bounds__(64 * DecodeRing<D>::W) void paged_decode(PagedAttend p) {
    using L = DecodeRing<D>;
    constexpr int W = L::W, NS = L::NS, FT = D / 16, KS = D / 32;
    __shared__ __attribute__((aligned(1024))) uint8_t lds_mem[L::bytes];
    __shared__ float lds_ml[W][16][2];
    __shared__ float lds_mass[64 * W];
    __shared__ uint32_t lds_last;
    lds_ptr<uint8_t> lds = (lds_ptr<uint8_t>)lds_mem;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, n = lane & 15;
    const int kvh = (int)(blockIdx.x % (uint32_t)p.hkv), split = (int)(blockIdx.x / (uint32_t)p.hkv), G = p.group;
    const PagedSeq sq = paged_sequence(p.b, blockIdx.y);
    if (sq.bad) {
        raise_status(p.status, true, ST_BAD_PAGE);
        return;
    }
    const int nrows = uniform(sq.n * G), pos0 = uniform(sq.len - sq.n), len = uniform(sq.len);
    if (nrows == 0 || nrows > p.decode_rows) return;

    // The blocks that some row sees, and this split's share of them.
    const int first_key = pos0 - p.window + 1 > 0 ? pos0 - p.window + 1 : 0;
    const int b_first = first_key >> 4, b_end = (len + 15) >> 4;
    const int blocks = b_end > b_first ? b_end - b_first : 0;
    int active = (blocks + p.split_blocks - 1) / p.split_blocks;
    active = active < 1 ? 1 : (active > p.splits ? p.splits : active);
    if (split >= active) return;
    const int per = (blocks + active - 1) / active;
    const int b_lo = b_first + split * per;
    const int b_hi = b_lo + per < b_end ? b_lo + per : b_end;
    const int mine = b_hi - b_lo > wave ? (b_hi - b_lo - wave + W - 1) / W : 0;

    const_ptr<int32_t> table = (const_ptr<int32_t>)(p.b.table + (int64_t)uniform(sq.slot) * p.b.table_stride);
    const uint8_t *kb = reinterpret_cast<const uint8_t *>(p.k) + (int64_t)kvh * p.l.head_stride * 2;
    const uint8_t *vb = reinterpret_cast<const uint8_t *>(p.v) + (int64_t)kvh * p.l.head_stride * 2;
    const int row_bytes = (int)p.l.row_stride * 2;
    uint32_t off[L::loads];
    for (int i = 0; i < L::loads; ++i) {
        const int at = i * 1024 + lane * 16, r = at / L::row, c = (at % L::row) >> 4;
        off[i] = (uint32_t)(r * row_bytes + ((c ^ L::turn(r)) << 4));
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
        const int64_t at = ((int64_t)page * p.l.page_stride + (int64_t)(key & ((1 << p.l.page_shift) - 1)) * p.l.row_stride) * 2;
        const uint8_t *ka = uniform_ptr(kb + at), *va = uniform_ptr(vb + at);
        const uint32_t m = ring + (uint32_t)(t % NS) * L::stage;
        for (int i = 0; i < L::loads; ++i) lds_load16_once(ka, off[i], m + i * 1024);
        for (int i = 0; i < L::loads; ++i) lds_load16_once(va, off[i], m + L::tile + i * 1024);
    };
    int pages[NS];
    for (int t = 0; t < NS; ++t) pages[t] = t < mine ? page_of(t) : 0;
    for (int t = 0; t < NS; ++t)
        if (t < mine) issue(t, pages[t]);

    // This lane's query row (rows past the last repeat it and see nothing).
    const int row = n < nrows ? n : nrows - 1;
    const int tok = row / G, head = kvh * G + row % G;
    u32x4 q[KS];
    for (int s = 0; s < KS; ++s)
        q[s] = *gload_ptr<u32x4>(reinterpret_cast<const uint16_t *>(p.q) + ((int64_t)(sq.q0 + tok) * p.hq + head) * D + 32 * s + 8 * g);
    const int pos = pos0 + tok;
    const int lo = pos - p.window + 1, hi = n < nrows ? pos + 1 : INT32_MIN;  // visible keys [lo, hi)
    const int all_lo = pos0 + (nrows - 1) / G - p.window + 1, all_hi = pos0 + 1;  // keys that every row sees

    f32x4 acc[FT] = {};
    float m = NEG_INF, l = 0.0f;
    bool bad = false;
    for (int t = 0; t < mine; ++t) {
        // The next block's page number arrives while this one is waited for.
        const int page_next = t + NS < mine ? page_of(t + NS) : 0;
        // Loads of later stages may stay under way.
        const int ahead = mine - 1 - t < NS - 1 ? mine - 1 - t : NS - 1;
        if (NS == 4 && ahead >= 3) wait_loads<3 * 2 * L::loads>();
        else if (NS == 4 && ahead == 2) wait_loads<2 * 2 * L::loads>();
        else if (ahead >= 1) wait_loads<2 * L::loads>();
        else wait_loads<0>();
        lds_ptr<uint8_t> kt = lds + (wave * L::wave_bytes + (t % NS) * L::stage), vt = kt + L::tile;
        const int key0 = (b_lo + wave + t * W) << 4;
        f32x4 s = {};
        for (int i = 0; i < KS; ++i) s = mfma_16x16x32<DT>(*(lds_ptr<u32x4>)(kt + L::at(n, g + 4 * i)), q[i], s);
        u32x2 v[FT];
        for (int f = 0; f < FT; ++f) {
            const int r = 4 * g + (n >> 2);
            v[f] = read_tr(vt + L::at(r, 2 * f + ((n & 3) >> 1)) + (n & 1) * 8);
        }
        float x[4];
        for (int i = 0; i < 4; ++i) x[i] = CAP ? tanh_fast(s[i] * p.softcap_y) * p.softcap_log2 : s[i] * p.scale_log2;
        if (key0 >= all_lo && key0 + 16 <= all_hi) {
            for (int i = 0; i < 4; ++i) bad |= !is_finite_f(s[i]);
        } else {
            // Keys that this row does not see weigh nothing; the values of keys that
            // no row sees are whatever the page holds, NaN too, and become zeros.
            for (int i = 0; i < 4; ++i) {
                const int key = key0 + 4 * g + i;
                const bool seen = key >= lo && key < hi;
                bad |= seen && !is_finite_f(s[i]);
                x[i] = seen ? x[i] : NEG_INF;
            }
            uint32_t keep[2];
            for (int i = 0; i < 2; ++i) {
                const int key = key0 + 4 * g + 2 * i;
                keep[i] = (key >= first_key && key < len ? 0xffffu : 0u) | (key + 1 >= first_key && key + 1 < len ? 0xffff0000u : 0u);
            }
            for (int f = 0; f < FT; ++f) v[f] = u32x2{v[f][0] & keep[0], v[f][1] & keep[1]};
        }
        const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        if (__ballot(top > m + SLACK) != 0) {
            const float mn = fmaxf(m, quad_max(top));
            const float c = mn == NEG_INF ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= c;
            for (int f = 0; f < FT; ++f) acc[f] *= c;
        }
        const float base = m == NEG_INF ? 0.0f : m;
        f32x4 w;
        for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_exp2f(x[i] - base);
        const u32x2 pw = pack4<DT>(w);  // the mass is summed from the weights as rounded
        w = unpack4<DT>(pw);
        l += (w[0] + w[1]) + (w[2] + w[3]);
        for (int f = 0; f < FT; ++f) acc[f] = mfma_16x16x16<DT>(v[f], pw, acc[f]);
        if (t + NS < mine) {
            wait_lds();
            issue(t + NS, page_next);
        }
    }
    l = quad_sum(l);

    // The waves' results through LDS (each in its own ring), then one thread per
    // four features of a row.
    constexpr int OS = D + 4;  // floats between rows
    static_assert(16 * OS * 4 <= L::wave_bytes, "a wave's context fits its ring");
    wait_lds();
    {
        lds_ptr<float> o = (lds_ptr<float>)(lds + wave * L::wave_bytes);
        for (int f = 0; f < FT; ++f) *(lds_ptr<f32x4>)(o + n * OS + 16 * f + 4 * g) = acc[f];
        if (g == 0) {
            lds_ml[wave][n][0] = m;
            lds_ml[wave][n][1] = l;
        }
    }
    raise_status(p.status, bad_page, ST_BAD_PAGE);
    raise_status(p.status, bad, ST_NONFINITE_INPUT);
    __syncthreads();
    const int64_t unit = (int64_t)blockIdx.y * p.hkv + kvh, slot = unit * p.splits + split;
    const __amdgpu_buffer_rsrc_t to = __builtin_amdgcn_make_buffer_rsrc(p.part_o + slot * p.rows * D, 0, 0x7FFFFFFF, 0x00020000);
    bool bad_out = false;
    auto finish = [&](int r, int d, f32x4 o, float mass) {
        f32x4 y = {};
        if (pos0 + r / G >= 0)
            for (int i = 0; i < 4; ++i) {
                y[i] = o[i] / mass;
                bad_out |= !is_finite_f(y[i]);
            }
        store_elem4<DT>(p.out, ((int64_t)(sq.q0 + r / G) * p.hq + kvh * G + r % G) * D + d, y);
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
            const uint32_t old = __hip_atomic_fetch_add(p.counters + unit, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            lds_last = old == (uint32_t)active - 1 ? 1u : 0u;
            if (lds_last) __hip_atomic_store(p.counters + unit, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!lds_last) return;
        // Every (maximum, mass) pair at once, into LDS; then each thread sums four
        // features of a row over its share of the splits, several loads under way.
        lds_ptr<f32x2> ml = (lds_ptr<f32x2>)lds;
        const int pairs = nrows * active, items = nrows * (D / 4);
        const float *part_ml = p.part_ml + unit * p.splits * p.rows * 2, *part_o = p.part_o + unit * p.splits * p.rows * D;
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

template <int DT, int D>
__global__ __launch_bounds__(64) void paged_rows(PagedAttend p) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x, s = blockIdx.z, h = blockIdx.y, kvh = h / p.group;
    const PagedSeq q = paged_sequence(p.b, s);
    if (q.bad) {
        raise_status(p.status, true, ST_BAD_PAGE);
        return;
    }
    const int i = blockIdx.x;
    if (i >= q.n) return;
    const int pos = q.len - q.n + i;
    const int64_t at = ((int64_t)(q.q0 + i) * p.hq + h) * D;
    float x[E], o[E] = {}, m = NEG_INF, l = 0.0f;
    for (int e = 0; e < E; ++e) x[e] = load_elem<DT>(p.q, at + lane + 64 * e);
    const int lo = pos >= p.window ? pos - p.window + 1 : 0;
    bool bad = false, bad_page = false;
    for (int j = lo; j <= pos; ++j) {
        const int page = gload_ptr<int32_t>(p.b.table)[(int64_t)q.slot * p.b.table_stride + (j >> p.l.page_shift)];
        if ((uint32_t)page >= (uint32_t)p.l.pages) {
            bad_page = true;
            break;
        }
        const int64_t row = (int64_t)page * p.l.page_stride + (int64_t)kvh * p.l.head_stride +
                            (int64_t)(j & ((1 << p.l.page_shift) - 1)) * p.l.row_stride;
        float dot = 0.0f;
        for (int e = 0; e < E; ++e) dot = __builtin_fmaf(x[e], load_elem<DT>(p.k, row + lane + 64 * e), dot);
        dot = wave_sum(dot);
        const float sc = p.softcap_y != 0.0f ? tanh_fast(dot * p.softcap_y) * p.softcap_log2 : dot * p.scale_log2;
        bad |= !is_finite_f(dot);
        const float mn = fmaxf(m, sc), c = __builtin_amdgcn_exp2f(m - mn), w = __builtin_amdgcn_exp2f(sc - mn);
        m = mn;
        l = l * c + w;
        for (int e = 0; e < E; ++e) o[e] = o[e] * c + w * load_elem<DT>(p.v, row + lane + 64 * e);
    }
    for (int e = 0; e < E; ++e) {
        const float y = pos < 0 ? 0.0f : o[e] / l;
        bad |= !is_finite_f(y);
        store_elem<DT>(p.out, at + lane + 64 * e, y);
    }
    raise_status(p.status, bad_page, ST_BAD_PAGE);
    raise_status(p.status, bad, ST_NONFINITE_INPUT);
}

}  // namespace tkh

extern "C" hipError_t tkh_launch_paged_decode(const tkh::PagedAttend *p, int dtype, int d, hipStream_t stream,
                                              hipEvent_t start, hipEvent_t stop) {
    using namespace tkh;
    const dim3 grid((unsigned)(p->hkv * p->splits), (unsigned)p->b.sequences);
    auto go = [&](auto kernel, int waves) {
        hipExtLaunchKernelGGL(kernel, grid, dim3(64 * waves), 0, stream, start, stop, 0, *p);
        return hipGetLastError();
    };
    auto dims = [&](auto dt, auto cap) {
        constexpr int DT = decltype(dt)::value;
        constexpr bool CAP = decltype(cap)::value;
        if (d == 64) return go(paged_decode<DT, 64, CAP>, DecodeRing<64>::W);
        if (d == 128) return go(paged_decode<DT, 128, CAP>, DecodeRing<128>::W);
        return go(paged_decode<DT, 256, CAP>, DecodeRing<256>::W);
    };
    auto caps = [&](auto dt) { return p->softcap_y != 0.0f ? dims(dt, std::true_type{}) : dims(dt, std::false_type{}); };
    if (dtype == F16) return caps(std::integral_constant<int, F16>{});
    if (dtype == BF16) return caps(std::integral_constant<int, BF16>{});
    return hipErrorInvalidValue;
}

extern "C" hipError_t tkh_launch_paged_rows(const tkh::PagedAttend *p, int dtype, int d, hipStream_t stream,
                                            hipEvent_t start, hipEvent_t stop) {
    const dim3 grid((unsigned)p->b.max_queries, (unsigned)p->hq, (unsigned)p->b.sequences), block(64);
    auto go = [&](auto kernel) {
        hipExtLaunchKernelGGL(kernel, grid, block, 0, stream, start, stop, 0, *p);
        return hipGetLastError();
    };
    using namespace tkh;
    if (dtype == F32) return d == 64 ? go(paged_rows<F32, 64>) : d == 128 ? go(paged_rows<F32, 128>) : go(paged_rows<F32, 256>);
    if (dtype == F16) return d == 64 ? go(paged_rows<F16, 64>) : d == 128 ? go(paged_rows<F16, 128>) : go(paged_rows<F16, 256>);
    return d == 64 ? go(paged_rows<BF16, 64>) : d == 128 ? go(paged_rows<BF16, 128>) : go(paged_rows<BF16, 256>);
}
