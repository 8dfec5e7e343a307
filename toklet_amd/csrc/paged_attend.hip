// paged_attend.hip - attention over a page table.
//
// paged_rows: one wave per (query row, head), FP32 throughout.
#include "paged.hpp"

namespace tkh {

template <int DT> __device__ __forceinline__ void store_row(void *base, int64_t i, float x);
template <> __device__ __forceinline__ void store_row<F32>(void *base, int64_t i, float x) { reinterpret_cast<float *>(base)[i] = x; }
template <> __device__ __forceinline__ void store_row<F16>(void *base, int64_t i, float x) { reinterpret_cast<_Float16 *>(base)[i] = (_Float16)x; }
template <> __device__ __forceinline__ void store_row<BF16>(void *base, int64_t i, float x) { reinterpret_cast<__bf16 *>(base)[i] = (__bf16)x; }

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
        store_row<DT>(p.out, at + lane + 64 * e, y);
    }
    raise_status(p.status, bad_page, ST_BAD_PAGE);
    raise_status(p.status, bad, ST_NONFINITE_INPUT);
}

}  // namespace tkh

extern "C" hipError_t tkh_launch_paged_attend(const tkh::PagedAttend *p, int dtype, int d, hipStream_t stream) {
    const dim3 grid((unsigned)p->b.max_queries, (unsigned)p->hq, (unsigned)p->b.sequences), block(64);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, block, 0, stream, *p);
        return hipGetLastError();
    };
    using namespace tkh;
    if (dtype == F32) return d == 64 ? go(paged_rows<F32, 64>) : d == 128 ? go(paged_rows<F32, 128>) : go(paged_rows<F32, 256>);
    if (dtype == F16) return d == 64 ? go(paged_rows<F16, 64>) : d == 128 ? go(paged_rows<F16, 128>) : go(paged_rows<F16, 256>);
    return d == 64 ? go(paged_rows<BF16, 64>) : d == 128 ? go(paged_rows<BF16, 128>) : go(paged_rows<BF16, 256>);
}
