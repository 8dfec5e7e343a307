// paged_produce.hip - what writes a paged cache: the producer of a batch's new
// rows, copies of pages, and the owner's table updates.
//
// paged_produce: per head row x of D features,
//   y = x * w / sqrt(mean(x^2) + eps)          (Q and K, with norm weights; FP64)
//   (u, v) -> m (u cos a - v sin a, v cos a + u sin a),  a = p f_j
// over the pairs of the first `rotated` features, (j, j + rotated/2) or
// (2j, 2j + 1), with f_j = theta^(-2j/rotated), divided by a factor (linear) or
// by wavelength band; then one rounding to the storage dtype.  Q rows go to
// q_out, K and V rows to their page.  The angle is formed in FP64 as turns,
// t = p f_j / 2 pi, and reduced by t - rint(t), so a far position costs no
// precision; sine and cosine are FP32 of the reduced turns, corrected by what
// the rounding of the turns left out.
// Bound by the bytes of the rows: 6000 tokens of 8/4 heads of 256, norms and interleaved
// pairs, FP32 to bf16, 14.5 us, 4.7 TB/s (a copy of 2 GiB: 4.85).  One token 3.5 us, 64
// single ones 4.4: a launch and the trips to the lengths, the table and the rows.
#include <cstddef>
#include <type_traits>

#include "paged.hpp"

namespace tkh {

namespace {

template <int DT> struct Elem4;  // four elements as stored
template <> struct Elem4<F32> { using type = f32x4; };
template <> struct Elem4<F16> { using type = _Float16 __attribute__((ext_vector_type(4))); };
template <> struct Elem4<BF16> { using type = __bf16 __attribute__((ext_vector_type(4))); };

template <int DT> __device__ __forceinline__ f32x4 load4(const void *base, int64_t i) {
    using T = typename Elem4<DT>::type;
    const T v = *gload_ptr<T>(reinterpret_cast<const uint8_t *>(base) + i * ElemSize<DT>::value);
    return __builtin_convertvector(v, f32x4);
}
template <int DT> __device__ __forceinline__ void store4(void *base, int64_t i, f32x4 x) {
    using T = typename Elem4<DT>::type;
    *gstore_ptr<T>(reinterpret_cast<uint8_t *>(base) + i * ElemSize<DT>::value) = __builtin_convertvector(x, T);
}

// cos and sin of 2 pi t for pair j's turns t at position p, times the magnitude.
__device__ __forceinline__ f32x2 rotation(const PagedRotary &r, int j, int pos) {
    double f = exp2((double)j * r.step);
    if (r.scaling == 1) {
        f *= r.inv_factor;
    } else if (r.scaling == 2) {
        // original * f / 2 pi rotations over the original length: kept from
        // `high` on, divided up to `low`, blended between.
        double keep = (r.original * f * 0.15915494309189535 - r.low) * r.inv_width;
        keep = keep < 0.0 ? 0.0 : (keep > 1.0 ? 1.0 : keep);
        f *= keep + (1.0 - keep) * r.inv_factor;
    }
    const double t = (double)pos * f * 0.15915494309189535;
    const double frac = t - rint(t);  // [-1/2, 1/2]
    const float hi = (float)frac, lo = (float)(frac - (double)hi);
    float s, c;
    sincospif(2.0f * hi, &s, &c);
    const float e = lo * 6.2831855f;
    return f32x2{r.magnitude * __builtin_fmaf(-e, s, c), r.magnitude * __builtin_fmaf(e, c, s)};
}

}  // namespace

// One workgroup covers `rows` head slots of one token (slots [0, Hq) query
// heads, then key heads, then value heads).  A lane holds eight elements of a
// row, the two halves of four pairs, so D/8 lanes make a row and a pair never
// leaves its lane.  The token's rotations are the same for every head: evaluated
// once per workgroup, into LDS, while the rows are on their way.
template <int SRC, int DST, int D>
__global__ __launch_bounds__(256) void paged_produce(PagedProduce p, int rows, int blocks_per_token) {
    constexpr int LPR = D / 8, RPI = 256 / LPR;  // lanes per row, rows per pass
    __shared__ f32x2 rot[D / 2];
    const int t = (int)(blockIdx.x / (uint32_t)blocks_per_token);
    const int first = (int)(blockIdx.x % (uint32_t)blocks_per_token) * rows;
    const int slots = p.hq + 2 * p.hkv;
    const int end = first + rows < slots ? first + rows : slots;
    const int tid = threadIdx.x, sub = tid % LPR;

    // The token's sequence: the last that starts at or before it.
    int s = 0;
    if (p.b.query_start) {
        int lo = 0, n = p.b.sequences;
        while (n > 1) {
            const int half = n >> 1;
            if (gload_ptr<int32_t>(p.b.query_start)[lo + half] <= t) {
                lo += half;
                n -= half;
            } else {
                n = half;
            }
        }
        s = __builtin_amdgcn_readfirstlane(lo);
    } else {
        s = t / p.b.max_queries;
    }
    const PagedSeq q = paged_sequence(p.b, s);
    const int pos = q.len - q.n + (t - q.q0);
    const bool mine = !q.bad && t >= q.q0 && t < q.q0 + q.n;
    bool bad = q.bad || (mine && pos < 0);
    int page = 0;
    if (mine && !bad) {
        page = gload_ptr<int32_t>(p.b.table)[(int64_t)q.slot * p.b.table_stride + (pos >> p.l.page_shift)];
        bad = (uint32_t)page >= (uint32_t)p.l.pages;
    }
    if (bad || !mine) {  // a row of no sequence stays as it is
        raise_status(p.status, bad, ST_BAD_PAGE);
        return;
    }
    const int64_t row_at = (int64_t)page * p.l.page_stride + (int64_t)(pos & ((1 << p.l.page_shift) - 1)) * p.l.row_stride;

    // This lane's elements a .. a + 3 and b .. b + 3, and its first pair.
    const int r = p.rot.layout ? p.rot.rotated : 0;
    const bool turns = sub * 8 < r;
    const int pair = sub * 4;
    const int a = turns && p.rot.layout == 1 ? pair : sub * 8;
    const int b = turns && p.rot.layout == 1 ? pair + r / 2 : sub * 8 + 4;

    f32x4 xa = {}, xb = {};
    auto load = [&](int slot) {
        const int64_t T = t;
        if (slot < p.hq) {
            xa = load4<SRC>(p.q, T * p.q_stride + slot * D + a);
            xb = load4<SRC>(p.q, T * p.q_stride + slot * D + b);
        } else if (slot < p.hq + p.hkv) {
            xa = load4<SRC>(p.k, T * p.k_stride + (slot - p.hq) * D + a);
            xb = load4<SRC>(p.k, T * p.k_stride + (slot - p.hq) * D + b);
        } else {
            xa = load4<SRC>(p.v, T * p.v_stride + (slot - p.hq - p.hkv) * D + a);
            xb = load4<SRC>(p.v, T * p.v_stride + (slot - p.hq - p.hkv) * D + b);
        }
    };
    int slot = first + tid / LPR;
    if (slot < end) load(slot);
    for (int j = tid; j < r / 2; j += 256) rot[j] = rotation(p.rot, j, pos);
    __syncthreads();

    bool nonfinite = false;
    for (; slot < end; slot += RPI) {
        if (slot >= first + RPI) load(slot);
        const bool is_q = slot < p.hq, is_v = slot >= p.hq + p.hkv;
        const float *w = is_v ? nullptr : (is_q ? p.q_norm : p.k_norm);
        if (w) {
            double ss = 0.0;
            for (int i = 0; i < 4; ++i) ss += (double)xa[i] * (double)xa[i] + (double)xb[i] * (double)xb[i];
            for (int m = 1; m < LPR; m <<= 1) ss += __shfl_xor(ss, m, 64);
            const double inv = 1.0 / sqrt(ss / (double)D + (double)p.eps);
            const f32x4 wa = *gload_ptr<f32x4>(w + a), wb = *gload_ptr<f32x4>(w + b);
            for (int i = 0; i < 4; ++i) {
                xa[i] = (float)((double)xa[i] * inv * (double)wa[i]);
                xb[i] = (float)((double)xb[i] * inv * (double)wb[i]);
            }
        }
        if (!is_v && turns) {
            if (p.rot.layout == 1) {
                for (int i = 0; i < 4; ++i) {
                    const f32x2 cs = rot[pair + i];
                    const float u = xa[i], v = xb[i];
                    xa[i] = u * cs[0] - v * cs[1];
                    xb[i] = v * cs[0] + u * cs[1];
                }
            } else {
                for (int i = 0; i < 2; ++i) {
                    const f32x2 ca = rot[pair + i], cb = rot[pair + 2 + i];
                    const float ua = xa[2 * i], va = xa[2 * i + 1], ub = xb[2 * i], vb = xb[2 * i + 1];
                    xa[2 * i] = ua * ca[0] - va * ca[1];
                    xa[2 * i + 1] = va * ca[0] + ua * ca[1];
                    xb[2 * i] = ub * cb[0] - vb * cb[1];
                    xb[2 * i + 1] = vb * cb[0] + ub * cb[1];
                }
            }
        }
        for (int i = 0; i < 4; ++i) nonfinite |= !is_finite_f(xa[i]) || !is_finite_f(xb[i]);
        if (is_q) {
            const int64_t at = ((int64_t)t * p.hq + slot) * D;
            store4<DST>(p.q_out, at + a, xa);
            store4<DST>(p.q_out, at + b, xb);
        } else {
            void *out = is_v ? p.v_pages : p.k_pages;
            const int64_t at = row_at + (int64_t)(slot - p.hq - (is_v ? p.hkv : 0)) * p.l.head_stride;
            store4<DST>(out, at + a, xa);
            store4<DST>(out, at + b, xb);
        }
    }
    raise_status(p.status, nonfinite, ST_NONFINITE_INPUT);
}

// Page copies: workgroup (chunk, pair, plane) moves four units per thread of one page,
// all loads before the stores.  1.6 GB in three launches 327 us, 4.95 TB/s; 24 pages of
// 32 KiB in 56 planes 18 us, 4.8.
constexpr int COPY_UNITS = 4;  // units per thread
template <class T>
__global__ __launch_bounds__(256) void copy_pages(CopyPages c) {
    const uint32_t s = c.src[blockIdx.y], d = c.dst[blockIdx.y];
    uint8_t *plane = c.pool + (int64_t)blockIdx.z * c.plane_stride;
    global_cptr<T> src = gload_ptr<T>(plane + (int64_t)s * c.page_stride);
    global_ptr<T> dst = gstore_ptr<T>(plane + (int64_t)d * c.page_stride);
    const int64_t n = c.page_bytes / (int64_t)sizeof(T);
    const int64_t i0 = (int64_t)blockIdx.x * (256 * COPY_UNITS) + threadIdx.x;
    T x[COPY_UNITS];
    for (int u = 0; u < COPY_UNITS; ++u)
        if (i0 + u * 256 < n) x[u] = src[i0 + u * 256];
    for (int u = 0; u < COPY_UNITS; ++u)
        if (i0 + u * 256 < n) dst[i0 + u * 256] = x[u];
}

// A word's later values come later in the list: the last one stays.
__global__ __launch_bounds__(256) void patch_words(PatchWords w) {
    for (int i = threadIdx.x; i < w.count; i += 256) {
        bool last = true;
        for (int j = i + 1; j < w.count && last; ++j) last = w.index[j] != w.index[i];
        if (last) w.base[w.index[i]] = w.value[i];
    }
}
__global__ __launch_bounds__(256) void copy_words(int32_t *dst, const int32_t *src, int32_t n) {
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) dst[i] = src[i];
}

}  // namespace tkh

namespace {

template <int SRC, int DST, int D> hipError_t launch_produce(const tkh::PagedProduce *p, hipStream_t stream) {
    constexpr int RPI = 256 / (D / 8);
    const int slots = p->hq + 2 * p->hkv;
    // Few tokens: one pass per workgroup, for latency.  Many: a workgroup takes
    // its token whole and evaluates the rotation once.
    const int passes = (slots + RPI - 1) / RPI;
    const int rows = (int64_t)p->b.total * passes <= 1024 ? RPI : slots;
    const int bpt = (slots + rows - 1) / rows;
    hipLaunchKernelGGL((tkh::paged_produce<SRC, DST, D>), dim3((unsigned)(p->b.total * bpt)), dim3(256), 0, stream, *p, rows, bpt);
    return hipGetLastError();
}
template <int SRC, int DST> hipError_t produce_dims(const tkh::PagedProduce *p, hipStream_t stream) {
    if (p->d == 64) return launch_produce<SRC, DST, 64>(p, stream);
    if (p->d == 128) return launch_produce<SRC, DST, 128>(p, stream);
    if (p->d == 256) return launch_produce<SRC, DST, 256>(p, stream);
    return hipErrorInvalidValue;
}
template <int SRC> hipError_t produce_dst(const tkh::PagedProduce *p, int dst, hipStream_t stream) {
    if (dst == tkh::F32) return produce_dims<SRC, tkh::F32>(p, stream);
    if (dst == tkh::F16) return produce_dims<SRC, tkh::F16>(p, stream);
    return produce_dims<SRC, tkh::BF16>(p, stream);
}

template <class T> void launch_copy(const tkh::CopyPages *c, hipStream_t stream) {
    const int64_t n = c->page_bytes / (int64_t)sizeof(T), per = 256 * tkh::COPY_UNITS;
    hipLaunchKernelGGL((tkh::copy_pages<T>), dim3((unsigned)((n + per - 1) / per), (unsigned)c->count, (unsigned)c->planes), dim3(256), 0, stream, *c);
}

}  // namespace

extern "C" hipError_t tkh_launch_paged_produce(const tkh::PagedProduce *p, int src, int dst, hipStream_t stream) {
    if (src == tkh::F32) return produce_dst<tkh::F32>(p, dst, stream);
    if (src == tkh::F16) return produce_dst<tkh::F16>(p, dst, stream);
    return produce_dst<tkh::BF16>(p, dst, stream);
}

// Units of 16 bytes where every page starts and ends on one, else of the 16-bit
// elements that any storage dtype is made of.
extern "C" hipError_t tkh_launch_copy_pages(const tkh::CopyPages *c, hipStream_t stream) {
    if ((((uintptr_t)c->pool | (uintptr_t)c->plane_stride | (uintptr_t)c->page_stride | (uintptr_t)c->page_bytes) & 15) == 0)
        launch_copy<tkh::u32x4>(c, stream);
    else
        launch_copy<uint16_t>(c, stream);
    return hipGetLastError();
}

extern "C" hipError_t tkh_launch_patch_words(const tkh::PatchWords *w, hipStream_t stream) {
    hipLaunchKernelGGL(tkh::patch_words, dim3(1), dim3(256), 0, stream, *w);
    return hipGetLastError();
}
extern "C" hipError_t tkh_launch_copy_words(int32_t *dst, const int32_t *src, int32_t n, hipStream_t stream) {
    hipLaunchKernelGGL(tkh::copy_words, dim3((unsigned)((n + 255) / 256 > 64 ? 64 : (n + 255) / 256)), dim3(256), 0, stream, dst, src, n);
    return hipGetLastError();
}
