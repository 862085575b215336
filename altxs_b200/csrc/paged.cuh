// Paged key/value cache: what its kernels share (types, sequences, page
// look-up) and the launchers behind the C entry points.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace altxs {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// N consecutive elements as one aligned access
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
    T e[N];
};

__device__ __forceinline__ void set_status(uint32_t *status, uint32_t bit) {
    if (status) atomicOr(status, bit);
}

// The rows of one sequence of a call: tokens q0 .. q0 + n, cache positions
// L - n .. L of them; n = 0 when the sequence is empty or outside its bounds.
struct Seq {
    int q0, n, L;
};
__device__ __forceinline__ Seq load_seq(const altxs_chunks &c, int s) {
    Seq q;
    q.q0 = c.q_start[s];
    const int q1 = c.q_start[s + 1];
    q.L = c.kv_len[s];
    q.n = q1 - q.q0;
    if (q.q0 < 0 || q1 > c.n_tokens || q1 < q.q0 || q.n > c.max_new || q.L < 0 || q.L > c.max_kv) q.n = -1;
    return q;
}
// as load_seq, with a bad sequence reported and made empty
__device__ __forceinline__ Seq load_seq_report(const altxs_chunks &c, int s) {
    Seq q = load_seq(c, s);
    if (q.n < 0) {
        set_status(c.status, ALTXS_ST_BAD_POS);
        q.n = 0;
    }
    return q;
}
// first cache position that any of the sequence's rows sees
__host__ __device__ __forceinline__ int first_seen(int n, int L, int window) {
    const int f = window > 0 ? L - n - window + 1 : 0;
    return f > 0 ? f : 0;
}

struct PagedAttnArgs {
    altxs_paged_kv kv;
    altxs_chunks c;
    int H, window;
    float scale;
    const void *q;
    int64_t ldq;
    void *out;
    int64_t ldo;
    float *lse;
    void *ws;
    int64_t ws_bytes;
};
int64_t paged_attention_ws(const altxs_paged_kv &kv, const altxs_chunks &c, int H, int window);
// The tensor-core kernel for many rows: bounds on its items and
// partial slots from the host's bounds on the lengths.
struct ManyPlan {
    int64_t items, slots, slot_bytes;
    int rows;  // rows of a slot
};
ManyPlan paged_many_plan(const altxs_paged_kv &kv, const altxs_chunks &c, int H, int window);
int launch_paged_many(const PagedAttnArgs &a, const ManyPlan &p, int min_rows, uint32_t *spoilt, uint32_t *cnt,
                      float *part, int sms, cudaStream_t stream);
int set_wait_limit_paged(uint32_t limit);
int launch_paged_attention(const PagedAttnArgs &a, cudaStream_t stream);

}  // namespace altxs
