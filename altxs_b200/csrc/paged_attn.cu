// Attention of new tokens over a paged key/value cache.
//
// One warp per (token, head): the lanes share the channels, keys one at a time
// with a running maximum and sum (o = o 2^(m - m') + p v), fp32 throughout.
#include "paged.cuh"
#include "prof.cuh"

namespace altxs {
namespace {

template <typename T, int HD>
__global__ void __launch_bounds__(128) k_paged_rows(PagedAttnArgs a) {
    constexpr int E = HD / 32;
    const Seq s = load_seq_report(a.c, blockIdx.x);
    const int h = blockIdx.y, g = h / (a.H / a.kv.n_kv_heads), lane = threadIdx.x & 31;
    const float c2 = __fmul_rn(a.scale, kLog2e);
    for (int i = blockIdx.z * 4 + (threadIdx.x >> 5); i < s.n; i += gridDim.z * 4) {
        const T *q = static_cast<const T *>(a.q) + (int64_t)(s.q0 + i) * a.ldq + (int64_t)h * HD + lane * E;
        float x[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = __fmul_rn(to_f(q[e]), c2), o[e] = 0.0f;
        const int pos = s.L - s.n + i;
        for (int j = a.window > 0 ? max(0, pos - a.window + 1) : 0; j <= pos; ++j) {
            const int page = a.c.page_table[blockIdx.x * a.c.table_stride + j / a.kv.page_size];
            if (page < 0 || page >= a.kv.n_pages) {
                if (lane == 0) set_status(a.c.status, ALTXS_ST_BAD_POS);
                continue;
            }
            const int64_t at = page * a.kv.page_stride + (int64_t)(j % a.kv.page_size) * a.kv.token_stride +
                               g * a.kv.head_stride + lane * E;
            float d = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) d = __fmaf_rn(x[e], to_f(static_cast<const T *>(a.kv.k)[at + e]), d);
            d = warp_sum(d);
            const float mn = fmaxf(m, d), f = m == -INFINITY ? 0.0f : exp2f(__fsub_rn(m, mn));
            const float p = d == -INFINITY ? 0.0f : exp2f(__fsub_rn(d, mn));
            l = __fmaf_rn(l, f, p);
            m = mn;
#pragma unroll
            for (int e = 0; e < E; ++e)
                o[e] = __fmaf_rn(o[e], f, __fmul_rn(p, to_f(static_cast<const T *>(a.kv.v)[at + e])));
        }
        T *y = static_cast<T *>(a.out) + (int64_t)(s.q0 + i) * a.ldo + (int64_t)h * HD + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = from_f<T>(m == -INFINITY ? 0.0f : __fdiv_rn(o[e], l));
        if (a.lse && lane == 0)
            a.lse[(int64_t)h * a.c.n_tokens + s.q0 + i] = m == -INFINITY ? -INFINITY : __fadd_rn(m, log2f(l));
    }
}

template <typename T>
void go(const PagedAttnArgs &a, cudaStream_t st) {
    const dim3 grid(a.c.n_seqs, a.H, (unsigned)min(256, (a.c.max_new + 3) / 4));
    if (a.kv.head_dim == 32) k_paged_rows<T, 32><<<grid, 128, 0, st>>>(a);
    else if (a.kv.head_dim == 64) k_paged_rows<T, 64><<<grid, 128, 0, st>>>(a);
    else k_paged_rows<T, 128><<<grid, 128, 0, st>>>(a);
}

}  // namespace

int64_t paged_attention_ws(const altxs_paged_kv &, const altxs_chunks &, int, int) { return 0; }

int launch_paged_attention(const PagedAttnArgs &a, cudaStream_t st) {
    if (a.c.max_new == 0) return ALTXS_OK;
    if (a.kv.dtype == ALTXS_F32) ALTXS_LAUNCH(kKPaged, st, go<float>(a, st));
    else if (a.kv.dtype == ALTXS_BF16) ALTXS_LAUNCH(kKPaged, st, go<__nv_bfloat16>(a, st));
    else ALTXS_LAUNCH(kKPaged, st, go<__half>(a, st));
    return ALTXS_OK;
}

}  // namespace altxs
