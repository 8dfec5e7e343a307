// paged_chunk.hip - attention of chunks of new tokens over a page table, 16-bit
// storage: many query rows per KV head, bound by the matrix cores.
//
// A workgroup takes 128 NB packed rows (tokens x query heads of one KV head) of one
// sequence: four waves of NB blocks of 32 rows.  K and V come in tiles of 32 keys
// through a ring in LDS, filled by direct global->LDS loads whose page number is
// uniform in a wave (a load run lies in one 16-key block, and those never leave a
// page).
//  * S^T = K Q^T on v_mfma_f32_32x32x16, Q in registers as the B operand: lane l
//    holds query row l % 32 and 16 keys, in the order that the B operand of
//    O^T = V^T P^T wants, if V^T's keys are read in that order too (two transposing
//    LDS loads per operand).  P never moves between lanes.
//  * The scores of tile t + 1 are formed while the softmax of tile t runs.
//  * A row's exponent base is a maximum that it has seen; it moves only when a
//    tile's mass against it passes 2^15, which 16-bit weights and FP32 sums hold.
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

constexpr float MASS_LIMIT = 0x1p15f;
// The base of a row that has seen no key: any finite score is far above it, which
// sends the row's first tile to the exact path; a hidden key's -inf still weighs 0.
constexpr float BASE_NONE = -0x1p100f;

}  // namespace

// The ring: NS tiles of 32 keys, K rows then V rows.  Rows hold their 16-byte
// pieces permuted by the row, so that rows read at one feature spread over the banks.
template <int D> struct ChunkRing {
    static constexpr int KT = 32, NS = 4;
    static constexpr int row = 2 * D;
    static constexpr int tile = KT * row;
    static constexpr int stage = 2 * tile;
    static constexpr int bytes = NS * stage;
    static constexpr int runs = tile / 4096;  // 1 KiB runs of a tile per wave
    __device__ static constexpr int turn(int r) { return D >= 128 ? (5 * r) & 15 : (2 * r + (r >> 2)) & 7; }
    __device__ static constexpr int at(int r, int c) { return r * row + ((c ^ turn(r)) << 4); }
};

// The tiles of row block `rb` that one of its rows sees, and how many splits share them.
struct ChunkSpan {
    int t_first, t_end, active;
};
template <int ROWS> __device__ __forceinline__ ChunkSpan chunk_span(const PagedAttend &p, const PagedSeq &sq, int rb) {
    const int G = p.group, pos0 = sq.len - sq.n, nrows = sq.n * G;
    const int r0 = rb * ROWS, r1 = (r0 + ROWS < nrows ? r0 + ROWS : nrows) - 1;
    const int lo = pos0 + r0 / G - p.window + 1, hi = pos0 + r1 / G + 1;
    ChunkSpan s;
    s.t_first = (lo > 0 ? lo : 0) >> 5;
    s.t_end = hi > 0 ? (hi + 31) >> 5 : 0;
    if (s.t_end < s.t_first) s.t_end = s.t_first;
    s.active = (s.t_end - s.t_first + p.split_blocks - 1) / p.split_blocks;
    s.active = s.active < 1 ? 1 : (s.active > p.splits ? p.splits : s.active);
    return s;
}

template <int DT, int D, int NB, bool CAP>
__global__ __launch_bounds__(256, NB == 1 && D <= 128 ? 2 : 1) void paged_chunk(PagedAttend p, int row_blocks) {
    using L = ChunkRing<D>;
    constexpr int KT = L::KT, NS = L::NS, ROWS = 128 * NB, QS = D / 16, FB = D / 32;
    __shared__ __attribute__((aligned(1024))) uint8_t lds_mem[L::bytes];
    lds_ptr<uint8_t> lds = (lds_ptr<uint8_t>)lds_mem;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
    const int G = p.group;

    // Workgroups reach the XCDs in turn; each XCD takes a contiguous range of the
    // (sequence, KV head) units, whose row blocks share K and V in its L2.  Within a
    // unit the longest row blocks and the shortest alternate.
    int unit, rb, split;
    {
        const uint32_t nb = gridDim.x, b = blockIdx.x, x = b % 8, k = b / 8;
        const uint32_t per = (nb + 7) / 8, full = nb % 8 == 0 ? 8 : nb % 8;
        const uint32_t t = x < full ? x * per + k : full * per + (x - full) * (per - 1) + k;
        split = (int)(t % (uint32_t)p.splits);
        const uint32_t i = t / (uint32_t)p.splits % (uint32_t)row_blocks;
        unit = (int)(t / (uint32_t)p.splits / (uint32_t)row_blocks);
        rb = i % 2 == 0 ? row_blocks - 1 - (int)(i / 2) : (int)(i / 2);
    }
    const int kvh = unit % p.hkv;
    const PagedSeq sq = paged_sequence(p.b, unit / p.hkv);
    if (sq.bad) {
        raise_status(p.status, true, ST_BAD_PAGE);
        return;
    }
    const int nrows = uniform(sq.n * G), pos0 = uniform(sq.len - sq.n), len = uniform(sq.len);
    if (nrows <= p.decode_rows || rb * ROWS >= nrows) return;
    const ChunkSpan span = chunk_span<ROWS>(p, sq, rb);
    if (split >= span.active) return;
    const int per = (span.t_end - span.t_first + span.active - 1) / span.active;
    const int t_lo = span.t_first + split * per;
    const int t_hi = t_lo + per < span.t_end ? t_lo + per : span.t_end;
    const int tiles = uniform(t_hi > t_lo ? t_hi - t_lo : 0);

    // Direct loads: run i of this wave covers rows 16-byte pieces of 1 KiB.
    const_ptr<int32_t> table = (const_ptr<int32_t>)(p.b.table + (int64_t)sq.slot * p.b.table_stride);
    const uint8_t *kb = reinterpret_cast<const uint8_t *>(p.k) + (int64_t)kvh * p.l.head_stride * 2;
    const uint8_t *vb = reinterpret_cast<const uint8_t *>(p.v) + (int64_t)kvh * p.l.head_stride * 2;
    const int row_bytes = (int)p.l.row_stride * 2;
    constexpr int RUN_ROWS = 1024 / L::row;             // rows of one run
    constexpr int WAVE_ROWS = RUN_ROWS * L::runs;        // 8: rows of this wave's share of a tile
    uint32_t off[L::runs];
    for (int i = 0; i < L::runs; ++i) {
        const int r = wave * WAVE_ROWS + i * RUN_ROWS + lane * 16 / L::row, c = (lane * 16 % L::row) >> 4;
        off[i] = (uint32_t)((r - wave * WAVE_ROWS) * row_bytes + ((c ^ L::turn(r)) << 4));
    }
    const uint32_t lds0 = (uint32_t)uniform((int)(uintptr_t)lds) + (uint32_t)wave * (L::runs * 1024);
    bool bad_page = false;
    const int last_entry = (len > 0 ? len - 1 : 0) >> p.l.page_shift;
    // This wave's first key of tile t; keys behind the last one repeat its page.
    auto key_of = [&](int t) { return ((t_lo + t) << 5) + wave * WAVE_ROWS; };
    auto page_of = [&](int t) {
        const int e = key_of(t) >> p.l.page_shift;
        return table[e < last_entry ? e : last_entry];
    };
    auto issue = [&](int t, int page) {
        if ((uint32_t)page >= (uint32_t)p.l.pages) {
            page = 0;
            bad_page = true;
        }
        const int64_t at = ((int64_t)page * p.l.page_stride + (int64_t)(key_of(t) & ((1 << p.l.page_shift) - 1)) * p.l.row_stride) * 2;
        const uint8_t *ka = uniform_ptr(kb + at), *va = uniform_ptr(vb + at);
        const uint32_t m = lds0 + (uint32_t)(t % NS) * L::stage;
        for (int i = 0; i < L::runs; ++i) lds_load16(ka, off[i], m + i * 1024);
        for (int i = 0; i < L::runs; ++i) lds_load16(va, off[i], m + L::tile + i * 1024);
    };
    {
        int pages[NS - 1];
        for (int t = 0; t < NS - 1; ++t) pages[t] = t < tiles ? page_of(t) : 0;
        for (int t = 0; t < NS - 1; ++t)
            if (t < tiles) issue(t, pages[t]);
    }

    // This wave's rows: lane row n of block nb.
    const int wave_row = rb * ROWS + wave * 32 * NB;
    const bool works = wave_row < nrows;  // uniform
    u32x4 q[NB][QS];
    int pos[NB], tok[NB], head[NB];
    bool real[NB];
    for (int b = 0; b < NB; ++b) {
        const int r = wave_row + 32 * b + n;
        real[b] = r < nrows;
        const int rr = real[b] ? r : nrows - 1;
        tok[b] = rr / G;
        head[b] = kvh * G + rr % G;
        pos[b] = pos0 + tok[b];
        for (int s = 0; s < QS; ++s)
            q[b][s] = *gload_ptr<u32x4>(reinterpret_cast<const uint16_t *>(p.q) + ((int64_t)(sq.q0 + tok[b]) * p.hq + head[b]) * D + 16 * s + 8 * h);
    }
    const int wave_last = wave_row + 32 * NB - 1 < nrows ? wave_row + 32 * NB - 1 : nrows - 1;
    // Keys that every row of the wave sees: [full_lo, full_hi).
    const int full_lo = uniform(pos0 + wave_last / G - p.window + 1), full_hi = uniform(pos0 + wave_row / G + 1);
    const int first_key = pos0 - p.window + 1 > 0 ? pos0 - p.window + 1 : 0;

    f32x16 o[NB][FB] = {};
    float base[NB], l[NB];
    for (int b = 0; b < NB; ++b) {
        base[b] = BASE_NONE;
        l[b] = 0.0f;
    }
    bool bad = false;

    // Scores of tile t for every block.
    auto scores = [&](int t, f32x16 (&s)[NB]) {
        lds_ptr<uint8_t> kt = lds + (t % NS) * L::stage;
        for (int b = 0; b < NB; ++b) s[b] = f32x16{};
        for (int i = 0; i < QS; ++i) {
            const u32x4 k = *(lds_ptr<u32x4>)(kt + L::at(n, 2 * i + h));
            for (int b = 0; b < NB; ++b) s[b] = mfma_32x32x16<DT>(k, q[b][i], s[b]);
        }
    };
    auto in_log2 = [&](float s) { return CAP ? tanh_fast(s * p.softcap_y) * p.softcap_log2 : s * p.scale_log2; };
    // Weights of tile t from its scores, the rows' masses and bases.
    auto softmax = [&](int t, f32x16 (&s)[NB], u32x4 (&w)[NB][2]) {
        const int key0 = (t_lo + t) << 5;
        const bool full = key0 >= full_lo && key0 + KT <= full_hi;
        if (!full) {
            for (int b = 0; b < NB; ++b)
                for (int i = 0; i < 16; ++i) {
                    const int key = key0 + 8 * (i >> 2) + 4 * h + (i & 3);
                    const bool seen = real[b] && key <= pos[b] && key > pos[b] - p.window;
                    bad |= seen && !is_finite_f(s[b][i]);
                    s[b][i] = seen ? s[b][i] : NEG_INF;
                }
        }
        for (int b = 0; b < NB; ++b) {
            float x[16];
            float top = 0.0f;
            for (int i = 0; i < 16; ++i) top = fmaxf(top, __builtin_fabsf(s[b][i]));
            bad |= full && !(top < __builtin_inff());
            auto weights = [&]() {
                float mass = 0.0f;
                for (int i = 0; i < 16; ++i) {
                    if constexpr (CAP) x[i] = (full || s[b][i] != NEG_INF) ? in_log2(s[b][i]) - base[b] : NEG_INF;
                    else x[i] = __builtin_fmaf(s[b][i], p.scale_log2, -base[b]);
                    x[i] = __builtin_amdgcn_exp2f(x[i]);
                }
                for (int j = 0; j < 8; ++j) {
                    const uint32_t v = pack2<DT>(x[2 * j], x[2 * j + 1]);
                    w[b][j >> 2][j & 3] = v;
                    mass = add_pair<DT>(v, mass);
                }
                return mass;
            };
            float mass = weights();
            if (__ballot(!(mass <= MASS_LIMIT)) != 0) {
                float mx = NEG_INF;
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, (CAP && s[b][i] == NEG_INF) ? NEG_INF : in_log2(s[b][i]));
                float a0, a1;
                swap_pair(mx, true, a0, a1);
                mx = fmaxf(a0, a1);
                const float next = fmaxf(base[b], mx);
                const float c = __builtin_amdgcn_exp2f(base[b] - next);
                base[b] = next;
                l[b] *= c;
                for (int f = 0; f < FB; ++f) o[b][f] *= c;
                mass = weights();
                bad |= !is_finite_f(mass);
            }
            l[b] += mass;
        }
    };
    // O^T += V^T P^T of tile t.
    auto values = [&](int t, const u32x4 (&w)[NB][2]) {
        lds_ptr<uint8_t> vt = lds + (t % NS) * L::stage + L::tile;
        const int key0 = (t_lo + t) << 5, g = (lane >> 4) & 1, j = lane & 15;
        const bool dead = key0 < first_key || key0 + KT > len;
        for (int f = 0; f < FB; ++f)
            for (int s = 0; s < 2; ++s) {
                u32x2 v[2];
                for (int e = 0; e < 2; ++e) {
                    const int r = 16 * s + 8 * e + 4 * h + (j >> 2);
                    v[e] = read_tr(vt + L::at(r, 4 * f + 2 * g + ((j & 3) >> 1)) + (j & 1) * 8);
                    if (dead) {  // whatever the page holds there, NaN too
                        for (int i = 0; i < 2; ++i) {
                            const int key = key0 + 16 * s + 8 * e + 4 * h + 2 * i;
                            v[e][i] &= (key >= first_key && key < len ? 0xffffu : 0u) | (key + 1 >= first_key && key + 1 < len ? 0xffff0000u : 0u);
                        }
                    }
                }
                const u32x4 a = {v[0][0], v[0][1], v[1][0], v[1][1]};
                for (int b = 0; b < NB; ++b) o[b][f] = mfma_32x32x16<DT>(a, w[b][s], o[b][f]);
            }
    };

    // Tile t + 1 has arrived (this wave's loads of tile t + 2 may be under way), and
    // no wave still reads tile t - 1, whose place tile t + 3 takes.
    auto next_tile = [&](int t) {
        const int page = t + NS - 1 < tiles ? page_of(t + NS - 1) : 0;
        if (t + 2 < tiles) wait_loads<2 * L::runs>();
        else wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (t + NS - 1 < tiles) issue(t + NS - 1, page);
    };
    f32x16 sa[NB], sb[NB];
    u32x4 w[NB][2];
    if (tiles > 0) {
        // Tile 0 before the loop.
        if (tiles > 2) wait_loads<4 * L::runs>();
        else if (tiles > 1) wait_loads<2 * L::runs>();
        else wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (works) scores(0, sa);
        for (int t = 0; t < tiles; t += 2) {
            next_tile(t);
            if (works) {
                if (t + 1 < tiles) scores(t + 1, sb);
                softmax(t, sa, w);
                values(t, w);
            }
            wait_lds();
            if (t + 1 >= tiles) break;
            next_tile(t + 1);
            if (works) {
                if (t + 2 < tiles) scores(t + 2, sa);
                softmax(t + 1, sb, w);
                values(t + 1, w);
            }
            wait_lds();
        }
    }

    bool bad_out = false;
    const int64_t slot = ((int64_t)unit * row_blocks + rb) * p.splits + split;
    if (works)
        for (int b = 0; b < NB; ++b) {
            float a0, a1;
            swap_pair(l[b], true, a0, a1);
            const float mass = a0 + a1;
            const int r = wave * 32 * NB + 32 * b + n;  // row in the block
            if (!real[b]) continue;
            if (span.active == 1) {
                const float inv = 1.0f / mass;
                for (int f = 0; f < FB; ++f)
                    for (int i = 0; i < 4; ++i) {
                        f32x4 y = {};
                        if (pos[b] >= 0)
                            for (int j = 0; j < 4; ++j) {
                                y[j] = o[b][f][4 * i + j] * inv;
                                bad_out |= !is_finite_f(y[j]);
                            }
                        store_elem4<DT>(p.out, ((int64_t)(sq.q0 + tok[b]) * p.hq + head[b]) * D + 32 * f + 8 * i + 4 * h, y);
                    }
            } else {
                for (int f = 0; f < FB; ++f)
                    for (int i = 0; i < 4; ++i) {
                        const f32x4 y = {o[b][f][4 * i], o[b][f][4 * i + 1], o[b][f][4 * i + 2], o[b][f][4 * i + 3]};
                        *gstore_ptr<f32x4>(p.part_o + (slot * ROWS + r) * D + 32 * f + 8 * i + 4 * h) = y;
                    }
                if (h == 0) *gstore_ptr<f32x2>(p.part_ml + (slot * ROWS + r) * 2) = f32x2{base[b], mass};
            }
        }
    raise_status(p.status, bad_page, ST_BAD_PAGE);
    raise_status(p.status, bad, ST_NONFINITE_INPUT);
    raise_status(p.status, bad_out, ST_NONFINITE_OUTPUT);
}

// The splits of every row block joined: a thread per four features of a row.
template <int DT, int D, int ROWS>
__global__ __launch_bounds__(256) void paged_chunk_merge(PagedAttend p, int row_blocks) {
    constexpr int PER = 256 / (D / 4);
    const int piece = blockIdx.x % (ROWS / PER), rb = blockIdx.x / (ROWS / PER) % row_blocks, unit = blockIdx.x / (ROWS / PER) / row_blocks;
    const int kvh = unit % p.hkv, G = p.group;
    const PagedSeq sq = paged_sequence(p.b, unit / p.hkv);
    const int nrows = sq.n * G, r = piece * PER + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
    if (sq.bad || nrows <= p.decode_rows || rb * ROWS + r >= nrows) return;
    const ChunkSpan span = chunk_span<ROWS>(p, sq, rb);
    if (span.active == 1) return;
    const int64_t slot = ((int64_t)unit * row_blocks + rb) * p.splits;
    float M = BASE_NONE, mass = 0.0f;
    f32x4 o = {};
    constexpr int U = 4;
    for (int s0 = 0; s0 < span.active; s0 += U) {
        f32x2 ml[U];
        f32x4 part[U];
        for (int u = 0; u < U; ++u) {
            const int s = s0 + u < span.active ? s0 + u : span.active - 1;
            ml[u] = *gload_ptr<f32x2>(p.part_ml + ((slot + s) * ROWS + r) * 2);
            part[u] = *gload_ptr<f32x4>(p.part_o + ((slot + s) * ROWS + r) * D + d);
        }
        for (int u = 0; u < U; ++u)
            if (s0 + u < span.active) {
                const float m = fmaxf(M, ml[u][0]), c0 = __builtin_amdgcn_exp2f(M - m), c1 = __builtin_amdgcn_exp2f(ml[u][0] - m);
                M = m;
                mass = c0 * mass + c1 * ml[u][1];
                for (int j = 0; j < 4; ++j) o[j] = c0 * o[j] + c1 * part[u][j];
            }
    }
    const int tok = (rb * ROWS + r) / G, head = kvh * G + (rb * ROWS + r) % G;
    bool bad = false;
    f32x4 y = {};
    if (sq.len - sq.n + tok >= 0)
        for (int j = 0; j < 4; ++j) {
            y[j] = o[j] / mass;
            bad |= !is_finite_f(y[j]);
        }
    store_elem4<DT>(p.out, ((int64_t)(sq.q0 + tok) * p.hq + head) * D + d, y);
    raise_status(p.status, bad, ST_NONFINITE_OUTPUT);
}

}  // namespace tkh

namespace {

template <class F> hipError_t chunk_build(int dtype, int d, int blocks, bool cap, F f) {
    using namespace tkh;
    auto caps = [&](auto dt, auto dims, auto nb) {
        return cap ? f(dt, dims, nb, std::true_type{}) : f(dt, dims, nb, std::false_type{});
    };
    auto rows = [&](auto dt, auto dims) {
        if constexpr (decltype(dims)::value <= 128) {
            if (blocks == 2) return caps(dt, dims, std::integral_constant<int, 2>{});
        }
        return caps(dt, dims, std::integral_constant<int, 1>{});
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

// Blocks of 32 rows a wave of the chunk kernel may take.
extern "C" int tkh_paged_chunk_blocks(int d) { return d <= 128 ? 2 : 1; }

extern "C" hipError_t tkh_launch_paged_chunk(const tkh::PagedAttend *p, int dtype, int d, int blocks, int row_blocks,
                                             hipStream_t stream, hipEvent_t start, hipEvent_t stop) {
    const int64_t groups = (int64_t)p->b.sequences * p->hkv * row_blocks * p->splits;
    return chunk_build(dtype, d, blocks, p->softcap_y != 0.0f, [&](auto dt, auto dims, auto nb, auto cap) {
        hipExtLaunchKernelGGL((tkh::paged_chunk<decltype(dt)::value, decltype(dims)::value, decltype(nb)::value, decltype(cap)::value>),
                              dim3((unsigned)groups), dim3(256), 0, stream, start, stop, 0, *p, row_blocks);
        return hipGetLastError();
    });
}

extern "C" hipError_t tkh_launch_paged_chunk_merge(const tkh::PagedAttend *p, int dtype, int d, int blocks, int row_blocks,
                                                   hipStream_t stream, hipEvent_t start, hipEvent_t stop) {
    return chunk_build(dtype, d, blocks, false, [&](auto dt, auto dims, auto nb, auto) {
        constexpr int D = decltype(dims)::value, ROWS = 128 * decltype(nb)::value, PER = 256 / (D / 4);
        const int64_t groups = (int64_t)p->b.sequences * p->hkv * row_blocks * (ROWS / PER);
        hipExtLaunchKernelGGL((tkh::paged_chunk_merge<decltype(dt)::value, D, ROWS>), dim3((unsigned)groups), dim3(256), 0, stream,
                              start, stop, 0, *p, row_blocks);
        return hipGetLastError();
    });
}
