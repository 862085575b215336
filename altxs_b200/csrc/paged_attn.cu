// Attention of a few new tokens over a paged key/value cache: at most 16 rows
// (the query heads of one key/value head times the sequence's new tokens), and
// the launch of all paged attention (paged_tc.cu has the kernel for more rows).
//
// o = sum_j p_j v_j / sum_j p_j with p_j = 2^(x_j - m), x = scale log2(e) q . k:
// one pass over the keys with the running maximum m and sum.  Every cached key
// and value is read once and serves at most 16 rows, so HBM bounds it (16 flops
// a byte at 16 rows in 16 bits against the card's 260).
//
// A sequence's visible keys are cut into splits (split_keys: a function of the
// sequence's own lengths, so a row's bits do not depend on the batch); an item
// is one split of one key/value head.  A split's rows go to the workspace as
// (m, l, o); the block that finishes the last split of a (sequence, head) joins
// them in split order.
//
// 16-bit types (k_paged_few): a block of four warps per item.  Each warp
// streams 8 KB chunks (keys and values of CK positions) through its own three
// slots with 16-byte asynchronous copies, gathering rows through the page table
// (a page may end anywhere in a chunk; rows past the end are filled with
// zeros), two chunks in flight while one is computed; there is no block-wide
// barrier until the four warps' partial rows meet.  Per chunk a warp forms
// S = Q K^T, the online softmax and O += P V as m16n8k16 fragments with fp32
// sums.  p is rounded to the type for P V (the fragments take no other), its sum
// from the unrounded p: the error against 64 bits is 1.0 to 1.2 times that of the
// plain form, which keeps p in fp32 and rounds the output once.  The tcgen05 tile
// is 128 rows for at most 16 real ones.  More rows in groups of 16 read the keys
// again and lose to it: 256 streams of up to 2048 keys, 20 rows a head, took
// 251 us against 137.
// Measured: three contexts of 60000 to 100000 keys, 32 heads over 8, hd 128 in
// bf16: 1.12 GB in 205 us (5.5 TB/s).
// fp32 (k_paged_vec, below): 256 streams of up to 2048 keys, 8 heads of 64:
// 1.10 GB in 190 us (5.8 TB/s); one stream of 2049 keys 13 us.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "paged.cuh"
#include "prof.cuh"

namespace altxs {
namespace {

constexpr int kWarps = 4;
constexpr int kSlots = 3;
constexpr int kChunkBytes = 8192;  // keys and values of one chunk
constexpr int kMaxRows = 16;
constexpr int kSplitUnit = 512;  // keys of a split at least
constexpr int kSplitItems = 296;  // items of a sequence at most, about: two blocks on each of 148 SMs
constexpr unsigned kAll = 0xffffffffu;

// Keys of a split of a sequence that shows `keys` of them to `width` (head, row group) pairs: a long one by
// itself fills the card once.  (An item costs some microseconds besides its keys' time: 100000 keys x 8 heads
// in 98 splits of 1024 took 286 us next to two like it, in 37 of 2752 205 us.)
__host__ __device__ inline int split_keys(int keys, int width) {
    const int most = width < kSplitItems ? kSplitItems / width : 1;
    const int each = (keys + most - 1) / most;
    return each > kSplitUnit ? (each + 63) / 64 * 64 : kSplitUnit;
}
__host__ __device__ inline int split_count(int keys, int width) {
    const int k = split_keys(keys, width);
    return keys > k ? (keys + k - 1) / k : 1;
}

struct FewArgs {
    PagedAttnArgs a;
    int G, min_rows, max_rows;  // sequences with rows in this range are the kernel's
    int group;                  // rows of an item at most
    int64_t max_items;  // partial slots in the workspace
    uint32_t *cnt;      // [n_seqs * Hkv * groups], zero between calls
    int groups;         // row groups of a sequence at most
    float *part;        // [max_items][rows][HD + 4]: o, m, l (two words keep the rows on 16 bytes)
    int part_rows;
};

// Items of the sequences before each run of `per` sequences; the sequences themselves while they fit.
constexpr int kScan = 128;
struct ItemScan {
    int before[kScan + 1];
    int per;
    Seq seq[kScan];
};

// items of a split: a (key/value head, row group) each
__device__ __forceinline__ int few_width(const FewArgs &f, const Seq &q) {
    return f.a.kv.n_kv_heads * ((q.n * f.G + f.group - 1) / f.group);
}
__device__ __forceinline__ int few_splits(const FewArgs &f, const Seq &q) {
    if (q.n <= 0 || q.n * f.G < f.min_rows || q.n * f.G > f.max_rows) return 0;
    return split_count(max(0, q.L - first_seen(q.n, q.L, f.a.window)), few_width(f, q));
}

// The kernel for many rows, where the call has one, is just ahead in the stream and need not have ended (they share no
// sequence): this one ends after it.
__device__ __forceinline__ void end_after_many() {
    if (blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ void scan_items(const FewArgs &f, ItemScan &sc) {
    __shared__ int wsum[kScan / 32];
    const int n = f.a.c.n_seqs, per = (n + kScan - 1) / kScan;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int inc = 0;
    if (tid < kScan) {
        for (int s = tid * per; s < min(n, (tid + 1) * per); ++s) {
            const Seq q = blockIdx.x == 0 ? load_seq_report(f.a.c, s) : load_seq(f.a.c, s);
            inc += few_splits(f, q) * few_width(f, q);
            if (per == 1) sc.seq[s] = q;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(kAll, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) wsum[warp] = inc;
    }
    __syncthreads();
    if (tid < kScan) {
        for (int w = 0; w < warp; ++w) inc += wsum[w];
        sc.before[tid + 1] = inc;
        if (tid == 0) sc.before[0] = 0, sc.per = per;
    }
    __syncthreads();
}

// item -> sequence, split, head (heads fastest: they share the rows' DRAM pages), row group
struct Where {
    Seq q;
    int s, split, g, grp, width;  // width: items from one split to the next
};
__device__ __forceinline__ Where locate(const FewArgs &f, const ItemScan &sc, int item) {
    int lo = 0, hi = kScan;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (sc.before[m] <= item) lo = m; else hi = m;
    }
    Where w;
    w.s = lo * sc.per;
    int local = item - sc.before[lo];
    w.q = sc.per == 1 ? sc.seq[lo] : load_seq(f.a.c, w.s);
    for (int n; sc.per > 1 && w.s < f.a.c.n_seqs - 1 && local >= (n = few_splits(f, w.q) * few_width(f, w.q)); w.q = load_seq(f.a.c, ++w.s))
        local -= n;
    w.width = few_width(f, w.q);
    w.split = local / w.width;
    const int x = local - w.split * w.width;
    w.grp = x / f.a.kv.n_kv_heads;
    w.g = x - w.grp * f.a.kv.n_kv_heads;
    return w;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int TRANS>
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t *r) {
    if (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void lds128(uint32_t addr, uint32_t *r) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ float4 ldg_stream(const float *p) {  // read once
    float4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
    return v;
}
template <typename T>
__device__ __forceinline__ void mma16(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

template <typename T, int HD>
struct Few {
    static constexpr int ES = sizeof(T), RB = HD * ES;        // bytes of a row
    static constexpr int CK = kChunkBytes / (2 * RB);         // positions of a chunk
    static constexpr int NC = RB / 16;                        // 16-byte pieces of a row
    static constexpr int NK = CK / 8, NO = HD / 8;            // score and output column tiles
    // piece c of position k in shared memory: conflict-free for the reads below
    static __device__ __forceinline__ uint32_t at(int k, int c) {
        const int sw = NC >= 8 ? k & 7 : (k >> 1) & 3;
        return k * RB + ((c ^ sw) << 4);
    }
};

// The keys that only some of a sequence's rows see: positions of [k0, k1) outside [all0, all1).
struct OddKeys {
    int k0, k1, all0, all1;
};

// The end of an item: `sets` partial rows (m, l in ml, o in rows, [set][stride][HD], shared memory) are joined
// in order; a sequence of one split is finished, else the rows go to the workspace and the block that brings
// the last split joins them.  odd: values that are not finite were kept out of o; they are added to the rows
// that see them.
template <typename T, int HD>
__device__ __forceinline__ void finish_item(const FewArgs &f, int item, const Where &w0, int nsplit, int R, int sets, int stride,
                                            float *rows, const float *ml, int *last_sh, const OddKeys *odd) {
    const PagedAttnArgs &a = f.a;
    const Seq &q = w0.q;
    const int G = f.G, s = w0.s, g = w0.g, r0 = w0.grp * f.group;  // row r of the item is row r0 + r of the sequence
    for (int i = threadIdx.x; i < R * (HD / 4); i += blockDim.x) {
        const int r = i / (HD / 4), c = (i % (HD / 4)) * 4;
        float M = -INFINITY, lt = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int w = 0; w < sets; ++w) M = fmaxf(M, ml[2 * (w * stride + r)]);
#pragma unroll 4
        for (int w = 0; w < sets; ++w) {
            const float2 v = *reinterpret_cast<const float2 *>(ml + 2 * (w * stride + r));
            const float sc2 = M == -INFINITY ? 0.0f : ex2(__fsub_rn(v.x, M));
            const float4 x = *reinterpret_cast<const float4 *>(rows + (w * stride + r) * HD + c);
            lt = __fmaf_rn(v.y, sc2, lt);
            y[0] = __fmaf_rn(x.x, sc2, y[0]), y[1] = __fmaf_rn(x.y, sc2, y[1]);
            y[2] = __fmaf_rn(x.z, sc2, y[2]), y[3] = __fmaf_rn(x.w, sc2, y[3]);
        }
        if (odd) {
            const int pos = q.L - q.n + (r0 + r) / G;
            for (int k = odd->k0; k < odd->k1; ++k) {
                if (k >= odd->all0 && k < odd->all1) continue;
                if (k > pos || (a.window > 0 && k <= pos - a.window)) continue;
                const int b = k / a.kv.page_size, page = __ldg(a.c.page_table + s * a.c.table_stride + b);
                if (page < 0 || page >= a.kv.n_pages) continue;
                const T *v = static_cast<const T *>(a.kv.v) + (int64_t)page * a.kv.page_stride +
                             (int64_t)(k - b * a.kv.page_size) * a.kv.token_stride + (int64_t)g * a.kv.head_stride + c;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!isfinite(to_f(v[e]))) y[e] = __fadd_rn(y[e], to_f(v[e]));
            }
        }
        if (nsplit == 1) {
            const int tok = q.q0 + (r0 + r) / G, h = g * G + (r0 + r) % G;
            const float inv = M == -INFINITY ? 0.0f : __frcp_rn(lt);
            Vec<T, 4> out;
#pragma unroll
            for (int e = 0; e < 4; ++e) out.e[e] = from_f<T>(__fmul_rn(y[e], inv));
            *reinterpret_cast<Vec<T, 4> *>(static_cast<T *>(a.out) + (int64_t)tok * a.ldo + (int64_t)h * HD + c) = out;
            if (a.lse && c == 0)
                a.lse[(int64_t)h * a.c.n_tokens + tok] = lt == 0.0f ? -INFINITY : __fadd_rn(M, log2f(lt));
        } else if (item < f.max_items) {
            float *p = f.part + ((int64_t)item * f.part_rows + r) * (HD + 4);
            __stcg(reinterpret_cast<float4 *>(p + c), make_float4(y[0], y[1], y[2], y[3]));
            if (c == 0) __stcg(reinterpret_cast<float2 *>(p + HD), make_float2(M, lt));
        } else if (i == 0) {  // the lengths' sum is above its bound
            set_status(a.c.status, ALTXS_ST_BAD_POS);
        }
    }
    if (nsplit == 1) return;
    __syncthreads();
    const int64_t first = item - (int64_t)w0.split * w0.width;  // the rows' split 0
    if (threadIdx.x == 0) {
        __threadfence();  // the block's rows are ordered before its arrival
        uint32_t *cnt = f.cnt + ((int64_t)s * a.kv.n_kv_heads + g) * f.groups + w0.grp;
        const bool last = atomicAdd(cnt, 1u) == (uint32_t)nsplit - 1;
        if (last) *cnt = 0;
        __threadfence();
        *last_sh = last;
    }
    __syncthreads();
    if (!*last_sh || first + (int64_t)(nsplit - 1) * w0.width >= f.max_items) return;
    // all (m, l) first, then the rows' weights, in shared memory
    float *ms = rows;                                                  // [nsplit][R], then [R] 1 / sum
    float2 *in = reinterpret_cast<float2 *>(rows + ((nsplit + 1) * R + 1 & ~1));  // [nsplit][R]
    const float *p0 = f.part + first * f.part_rows * (HD + 4);
    const int64_t ps = (int64_t)w0.width * f.part_rows * (HD + 4);
    for (int i = threadIdx.x; i < nsplit * R; i += blockDim.x)
        in[i] = __ldcg(reinterpret_cast<const float2 *>(p0 + i / R * ps + i % R * (HD + 4) + HD));
    __syncthreads();
    for (int r = threadIdx.x; r < R; r += blockDim.x) {
        float M = -INFINITY, lt = 0.0f;
        for (int t = 0; t < nsplit; ++t) M = fmaxf(M, in[t * R + r].x);
        for (int t = 0; t < nsplit; ++t) {
            const float2 x = in[t * R + r];
            const float w = M == -INFINITY ? 0.0f : ex2(__fsub_rn(x.x, M));
            ms[t * R + r] = w;
            lt = __fmaf_rn(x.y, w, lt);
        }
        ms[nsplit * R + r] = M == -INFINITY ? 0.0f : __frcp_rn(lt);
        if (a.lse)
            a.lse[(int64_t)(g * G + (r0 + r) % G) * a.c.n_tokens + q.q0 + (r0 + r) / G] =
                lt == 0.0f ? -INFINITY : __fadd_rn(M, log2f(lt));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * (HD / 4); i += blockDim.x) {
        const int r = i / (HD / 4), c = (i % (HD / 4)) * 4;
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
        for (int t = 0; t < nsplit; ++t) {
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(p0 + t * ps + r * (HD + 4) + c));
            const float w = ms[t * R + r];
            y[0] = __fmaf_rn(x.x, w, y[0]), y[1] = __fmaf_rn(x.y, w, y[1]);
            y[2] = __fmaf_rn(x.z, w, y[2]), y[3] = __fmaf_rn(x.w, w, y[3]);
        }
        const float inv = ms[nsplit * R + r];
        Vec<T, 4> out;
#pragma unroll
        for (int e = 0; e < 4; ++e) out.e[e] = from_f<T>(__fmul_rn(y[e], inv));
        *reinterpret_cast<Vec<T, 4> *>(static_cast<T *>(a.out) + (int64_t)(q.q0 + (r0 + r) / G) * a.ldo + (int64_t)(g * G + (r0 + r) % G) * HD + c) = out;
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kWarps * 32, 2) k_paged_few(const __grid_constant__ FewArgs f) {
    using F = Few<T, HD>;
    constexpr int CK = F::CK, NC = F::NC, NK = F::NK, NO = F::NO;
    extern __shared__ __align__(1024) unsigned char few_smem[];
    __shared__ ItemScan sc;
    __shared__ uint64_t seen_sh[kWarps][kSlots];  // positions of a slot's chunk that exist
    __shared__ float ml_sh[kWarps][kMaxRows][2];
    __shared__ int last_sh, odd_sh;
    const PagedAttnArgs &a = f.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, j = lane & 3;
    const int G = f.G, P = a.kv.page_size;
    const int pshift = (P & (P - 1)) == 0 ? 31 - __clz(P) : -1;
    const float c2 = __fmul_rn(a.scale, kLog2e);
    // fp16 ends at 2^-24: p carries 2^14 (and is at most that), so that what a dominant key leaves to each of many
    // others is not rounded to 0 while the row's sum has it
    constexpr float kBias = std::is_same<T, __half>::value ? 14.0f : 0.0f, unbias = std::is_same<T, __half>::value ? 1.0f / 16384.0f : 1.0f;
    const uint32_t ring = smem_u32(few_smem) + warp * kSlots * kChunkBytes;
    scan_items(f, sc);
    const int total = sc.before[kScan];

    for (int item = blockIdx.x; item < total; item += gridDim.x) {
        const Where at = locate(f, sc, item);
        const Seq q = at.q;
        const int s = at.s, g = at.g, split = at.split;
        const int R = q.n * G, kfirst = first_seen(q.n, q.L, a.window), keys = max(0, q.L - kfirst);
        const int nsplit = split_count(keys, at.width), slen = split_keys(keys, at.width);
        const int k0 = kfirst + split * slen, k1 = min(q.L, k0 + slen);
        const int nchunk = k1 > k0 ? (k1 - k0 + CK - 1) / CK : 0;
        const int p0 = q.L - q.n;  // position of the first new token
        // positions [all0, all1) are seen by every row
        const int all1 = p0 + 1, all0 = a.window > 0 ? q.L - a.window : 0;
        const char *kb = static_cast<const char *>(a.kv.k) + (int64_t)g * a.kv.head_stride * F::ES;
        const char *vb = static_cast<const char *>(a.kv.v) + (int64_t)g * a.kv.head_stride * F::ES;
        const int32_t *table = a.c.page_table + s * a.c.table_stride;
        if (threadIdx.x == 0) odd_sh = 0;

        auto block_of = [&](int k) { return pshift >= 0 ? k >> pshift : k / P; };
        constexpr int KL = (CK + 31) / 32;  // positions a lane looks up per chunk
        int pg[KL];
        auto fetch_pages = [&](int ci) {
#pragma unroll
            for (int r = 0; r < KL; ++r) {
                const int kc = r * 32 + lane, k = k0 + ci * CK + kc;
                pg[r] = kc < CK && k < k1 && ci < nchunk ? __ldg(table + block_of(k)) : -1;
            }
        };
        auto issue = [&](int ci, int slot) {  // chunk ci into a slot; pg holds its pages
            uint64_t seen = 0;
            int64_t off[KL];
#pragma unroll
            for (int r = 0; r < KL; ++r) {
                const int k = k0 + ci * CK + r * 32 + lane;
                const bool in = pg[r] >= 0 && pg[r] < a.kv.n_pages;
                if (!in && k < k1 && r * 32 + lane < CK) set_status(a.c.status, ALTXS_ST_BAD_POS);
                const int b = block_of(k);
                off[r] = in ? ((int64_t)pg[r] * a.kv.page_stride + (int64_t)(k - b * P) * a.kv.token_stride) * F::ES : -1;
                seen |= (uint64_t)__ballot_sync(kAll, in) << (32 * r);
            }
            if (lane == 0) seen_sh[warp][slot] = seen;
            const uint32_t dst = ring + slot * kChunkBytes;
#pragma unroll
            for (int i = 0; i < CK * NC / 32; ++i) {
                const int p = i * 32 + lane, k = p / NC, c = p % NC;
                const int64_t o = __shfl_sync(kAll, off[CK > 32 ? (i * 32 / NC) / 32 : 0], k & 31);
                const int64_t src = (o < 0 ? 0 : o) + c * 16;
                const uint32_t bytes = o < 0 ? 0u : 16u, d = dst + F::at(k, c);
                cp_async16(d, kb + src, bytes);
                cp_async16(d + kChunkBytes / 2, vb + src, bytes);
            }
        };

        // the first chunks are on their way before the queries are read
        int next = warp;
        fetch_pages(next);
#pragma unroll
        for (int i = 0; i < kSlots - 1; ++i) {
            if (next < nchunk) issue(next, i);
            cp_commit();
            next += kWarps;
            fetch_pages(next);
        }
        // Q fragments: rows quad, quad + 8 (row r = token r / G, head r % G of the group)
        uint32_t qa[HD / 16][4];
        int rpos[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            const int r = quad + 8 * hh, i = r / G, h = g * G + r - i * G;
            rpos[hh] = r < R ? p0 + i : -1;
            const T *qp = static_cast<const T *>(a.q) + (int64_t)(q.q0 + i) * a.ldq + (int64_t)h * HD;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
                qa[kk][hh] = r < R ? *reinterpret_cast<const uint32_t *>(qp + 16 * kk + 2 * j) : 0u;
                qa[kk][2 + hh] = r < R ? *reinterpret_cast<const uint32_t *>(qp + 16 * kk + 8 + 2 * j) : 0u;
            }
        }
        float o[NO][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < NO; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
        __syncthreads();  // odd_sh is clear

        int slot = 0;
        for (int ci = warp; ci < nchunk; ci += kWarps) {
            cp_wait<kSlots - 2>();
            __syncwarp();  // the chunk has landed for every lane, and the slot before it has been read
            if (next < nchunk) issue(next, slot == 0 ? kSlots - 1 : slot - 1);
            cp_commit();
            next += kWarps;
            fetch_pages(next);
            const uint32_t kt = ring + slot * kChunkBytes, vt = kt + kChunkBytes / 2;
            const uint64_t have = seen_sh[warp][slot];
            // S = Q K^T
            float sacc[NK][4];
#pragma unroll
            for (int t = 0; t < NK; ++t) sacc[t][0] = sacc[t][1] = sacc[t][2] = sacc[t][3] = 0.0f;
#pragma unroll
            for (int t = 0; t < NK; t += 2)
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    uint32_t b[4];
                    ldsm4<0>(kt + F::at(8 * t + (lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)), b);
                    mma16<T>(sacc[t], qa[kk], b[0], b[1]);
                    mma16<T>(sacc[t + 1], qa[kk], b[2], b[3]);
                }
            // scale, mask, running maximum
            const int kc = k0 + ci * CK;
            const bool whole = kc >= all0 && kc + CK <= min(all1, k1) &&
                               have == (CK == 64 ? ~0ull : (1ull << (CK & 63)) - 1);
            float mx[2] = {m[0], m[1]};
#pragma unroll
            for (int t = 0; t < NK; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int kl = 8 * t + 2 * j + (e & 1), k = kc + kl, hh = e >> 1;
                    float x = __fmul_rn(sacc[t][e], c2);
                    if (!whole)
                        x = k <= rpos[hh] && (a.window == 0 || k > rpos[hh] - a.window) && ((have >> kl) & 1) ? x : -INFINITY;
                    sacc[t][e] = x;
                    mx[hh] = fmaxf(mx[hh], x);
                }
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                if (hh == 1 && R <= 8) break;  // rows 8 .. are empty
                mx[hh] = fmaxf(mx[hh], __shfl_xor_sync(kAll, mx[hh], 1));
                mx[hh] = fmaxf(mx[hh], __shfl_xor_sync(kAll, mx[hh], 2));
                const float base = mx[hh] == -INFINITY ? 0.0f : mx[hh];  // nothing seen yet: every p is 2^-inf = 0
                const float fold = ex2(__fsub_rn(m[hh], base));
                m[hh] = mx[hh];
                mx[hh] = __fsub_rn(base, kBias);
                l[hh] = __fmul_rn(l[hh], fold);
#pragma unroll
                for (int t = 0; t < NO; ++t) {
                    o[t][2 * hh] = __fmul_rn(o[t][2 * hh], fold);
                    o[t][2 * hh + 1] = __fmul_rn(o[t][2 * hh + 1], fold);
                }
            }
#pragma unroll
            for (int t = 0; t < NK; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (e >= 2 && R <= 8) break;  // (their p is whatever the scores are: finite, and not stored)
                    sacc[t][e] = ex2(__fsub_rn(sacc[t][e], mx[e >> 1]));
                    sum[e >> 1] = __fadd_rn(sum[e >> 1], sacc[t][e]);
                }
            l[0] = __fadd_rn(l[0], sum[0]);
            l[1] = __fadd_rn(l[1], sum[1]);
            // Some rows do not see some of these values: one of those that is not finite must not
            // meet their p = 0.  It becomes 0 here and is added to the rows that see it at the end.
            if (!whole && q.n > 1) {
                bool odd = false;
#pragma unroll
                for (int i = 0; i < CK * NC / 32; ++i) {
                    const uint32_t d = vt + (i * 32 + lane) * 16;
                    const int k = kc + (i * 32 + lane) / NC;
                    if (k >= all0 && k < all1) continue;  // every row sees it
                    uint32_t w[4];
                    lds128(d, w);
                    bool bad = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        constexpr uint32_t X = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
                        if ((w[e] & X) == X) w[e] &= 0xffff0000u, bad = true;
                        if (((w[e] >> 16) & X) == X) w[e] &= 0xffffu, bad = true;
                    }
                    if (bad) {
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(d), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                        odd = true;
                    }
                }
                if (odd) odd_sh = 1;
                __syncwarp();
            }
            // O += P V
#pragma unroll
            for (int t = 0; t < NK; t += 2) {
                const uint32_t pa[4] = {pack2<T>(sacc[t][0], sacc[t][1]), pack2<T>(sacc[t][2], sacc[t][3]),
                                        pack2<T>(sacc[t + 1][0], sacc[t + 1][1]), pack2<T>(sacc[t + 1][2], sacc[t + 1][3])};
#pragma unroll
                for (int n = 0; n < NO; n += 2) {
                    uint32_t b[4];
                    ldsm4<1>(vt + F::at(8 * t + (lane & 15), n + (lane >> 4)), b);
                    mma16<T>(o[n], pa, b[0], b[1]);
                    mma16<T>(o[n + 1], pa, b[2], b[3]);
                }
            }
            slot = slot == kSlots - 1 ? 0 : slot + 1;
        }
        cp_wait<0>();
        __syncthreads();  // every warp is done with its slots: they take the warps' rows [warp][row][HD]
        float *rows = reinterpret_cast<float *>(few_smem);
        const OddKeys odd{k0, k1, all0, all1};
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            l[hh] = __fadd_rn(l[hh], __shfl_xor_sync(kAll, l[hh], 1));
            l[hh] = __fadd_rn(l[hh], __shfl_xor_sync(kAll, l[hh], 2));
            const int r = quad + 8 * hh;
            if (r >= R) continue;
            if (j == 0) ml_sh[warp][r][0] = m[hh], ml_sh[warp][r][1] = __fmul_rn(l[hh], unbias);
            float *y = rows + (warp * kMaxRows + r) * HD;
#pragma unroll
            for (int t = 0; t < NO; ++t)
                *reinterpret_cast<float2 *>(y + 8 * t + 2 * j) = make_float2(__fmul_rn(o[t][2 * hh], unbias), __fmul_rn(o[t][2 * hh + 1], unbias));
        }
        __syncthreads();
        finish_item<T, HD>(f, item, at, nsplit, R, kWarps, kMaxRows, rows, &ml_sh[0][0][0], &last_sh,
                           odd_sh ? &odd : nullptr);
        __syncthreads();  // before the slots and the shared words are used again
    }
    end_after_many();
}

// fp32: half a flop a byte and row, so plain fp32 arithmetic keeps up with HBM for a few rows.  HD / 8 lanes
// share a position, each with eight channels of its key and value straight from global memory (two 16-byte
// loads each, the row contiguous over the lanes); at one row a head a warp has 4 KB in flight and an SM 32 warps.
// Every group of lanes keeps its own (m, l, o) over its positions, joined at the end.  More than eight rows are two
// items that read the same keys.  (As 16-row MMA tiles of three tf32 products, with a dozen instructions to split
// each pair of values, 256 streams took 471 us where this takes 190.  Four warps a block: 185 us, but one stream
// 15.4 us where eight take 13.)
constexpr int kVecRows = 8, kVecWarps = 8;
template <int HD, int R>
__global__ void __launch_bounds__(kVecWarps * 32, R == 1 ? 4 : R < 4 ? 2 : 1) k_paged_vec(const __grid_constant__ FewArgs f) {
    constexpr int LPK = HD / 8, KS = 32 / LPK, U = 2, B = U * KS, Sets = kVecWarps;  // lanes a position, positions a step
    __shared__ ItemScan sc;
    // (the join of the splits keeps three words for each of them there)
    constexpr int Words = Sets * HD > 3 * kSplitItems + 4 ? Sets * HD : 3 * kSplitItems + 4;
    __shared__ __align__(16) float rows[Words * R];
    __shared__ __align__(8) float ml[Sets * R * 2];
    __shared__ int last_sh;
    const PagedAttnArgs &a = f.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kg = lane / LPK, li = lane % LPK;
    const int G = f.G, P = a.kv.page_size, pshift = (P & (P - 1)) == 0 ? 31 - __clz(P) : -1;
    const float c2 = __fmul_rn(a.scale, kLog2e);
    scan_items(f, sc);
    const int total = sc.before[kScan];
    for (int item = blockIdx.x; item < total; item += gridDim.x) {
        const Where at = locate(f, sc, item);
        const Seq q = at.q;
        const int s = at.s, g = at.g, split = at.split;
        const int r0 = at.grp * f.group, n = min(f.group, q.n * G - r0), kfirst = first_seen(q.n, q.L, a.window), keys = max(0, q.L - kfirst);
        const int nsplit = split_count(keys, at.width), slen = split_keys(keys, at.width);
        const int k0 = kfirst + split * slen, k1 = min(q.L, k0 + slen), p0 = q.L - q.n;
        const float *kb = static_cast<const float *>(a.kv.k) + (int64_t)g * a.kv.head_stride + 4 * li;
        const float *vb = static_cast<const float *>(a.kv.v) + (int64_t)g * a.kv.head_stride + 4 * li;
        const int32_t *table = a.c.page_table + s * a.c.table_stride;
        float qr[R][8], o[R][8], m[R], l[R];
        int pos[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = (r0 + r) / G;
            pos[r] = r < n ? p0 + i : -1;
            m[r] = -INFINITY, l[r] = 0.0f;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
            if (r < n) {
                const float *qp = static_cast<const float *>(a.q) + (int64_t)(q.q0 + i) * a.ldq + (int64_t)(g * G + r0 + r - i * G) * HD + 4 * li;
                x = __ldg(reinterpret_cast<const float4 *>(qp)), y = __ldg(reinterpret_cast<const float4 *>(qp + HD / 2));
            }
            const float t[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) qr[r][e] = __fmul_rn(t[e], c2), o[r][e] = 0.0f;
        }
        auto block_of = [&](int k) { return pshift >= 0 ? k >> pshift : k / P; };
        int page[U];
        auto fetch = [&](int kb0) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = kb0 + u * KS + kg;
                page[u] = k < k1 ? __ldg(table + block_of(k)) : INT32_MIN;
            }
        };
        fetch(k0 + warp * B);
        for (int kc = k0 + warp * B; kc < k1; kc += kVecWarps * B) {
            float kr[U][8], vr[U][8];
            bool in[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = kc + u * KS + kg;
                in[u] = page[u] >= 0 && page[u] < a.kv.n_pages;
                if (!in[u] && page[u] != INT32_MIN) set_status(a.c.status, ALTXS_ST_BAD_POS);
                const int64_t off = (int64_t)page[u] * a.kv.page_stride + (int64_t)(k - block_of(k) * P) * a.kv.token_stride;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x, z = x, w = x;
                if (in[u]) {
                    x = ldg_stream(kb + off), y = ldg_stream(kb + off + HD / 2);
                    z = ldg_stream(vb + off), w = ldg_stream(vb + off + HD / 2);
                }
                kr[u][0] = x.x, kr[u][1] = x.y, kr[u][2] = x.z, kr[u][3] = x.w, kr[u][4] = y.x, kr[u][5] = y.y, kr[u][6] = y.z, kr[u][7] = y.w;
                vr[u][0] = z.x, vr[u][1] = z.y, vr[u][2] = z.z, vr[u][3] = z.w, vr[u][4] = w.x, vr[u][5] = w.y, vr[u][6] = w.z, vr[u][7] = w.w;
            }
            fetch(kc + kVecWarps * B);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float sco[U], mx = m[r];
                bool see[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float d = __fmul_rn(qr[r][0], kr[u][0]);
#pragma unroll
                    for (int e = 1; e < 8; ++e) d = __fmaf_rn(qr[r][e], kr[u][e], d);
                    sco[u] = d;
                }
#pragma unroll
                for (int w = 1; w < LPK; w <<= 1)
#pragma unroll
                    for (int u = 0; u < U; ++u) sco[u] = __fadd_rn(sco[u], __shfl_xor_sync(kAll, sco[u], w));
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int k = kc + u * KS + kg;
                    see[u] = in[u] && k <= pos[r] && (a.window == 0 || k > pos[r] - a.window);
                    if (see[u]) mx = fmaxf(mx, sco[u]);
                }
                const float fold = mx == -INFINITY ? 0.0f : ex2(__fsub_rn(m[r], mx)), base = mx == -INFINITY ? 0.0f : mx;
                m[r] = mx;
                l[r] = __fmul_rn(l[r], fold);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[r][e] = __fmul_rn(o[r][e], fold);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (see[u]) {
                        const float p = ex2(__fsub_rn(sco[u], base));
                        l[r] = __fadd_rn(l[r], p);
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[r][e] = __fmaf_rn(p, vr[u][e], o[r][e]);
                    }
            }
        }
#pragma unroll
        for (int w = LPK; w < 32; w <<= 1)  // the warp's groups of lanes, in a fixed tree
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float m1 = __shfl_xor_sync(kAll, m[r], w), l1 = __shfl_xor_sync(kAll, l[r], w), M = fmaxf(m[r], m1);
                const float f0 = m[r] == -INFINITY ? 0.0f : ex2(__fsub_rn(m[r], M)), f1 = m1 == -INFINITY ? 0.0f : ex2(__fsub_rn(m1, M));
                // the two sides add the same two products, so they agree
                l[r] = __fadd_rn(__fmul_rn(l[r], f0), __fmul_rn(l1, f1));
                m[r] = M;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    o[r][e] = __fadd_rn(__fmul_rn(o[r][e], f0), __fmul_rn(__shfl_xor_sync(kAll, o[r][e], w), f1));
            }
        if (kg == 0)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float *y = rows + (warp * R + r) * HD + 4 * li;
                *reinterpret_cast<float4 *>(y) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
                *reinterpret_cast<float4 *>(y + HD / 2) = make_float4(o[r][4], o[r][5], o[r][6], o[r][7]);
                if (li == 0) ml[2 * (warp * R + r)] = m[r], ml[2 * (warp * R + r) + 1] = l[r];
            }
        __syncthreads();
        finish_item<float, HD>(f, item, at, nsplit, n, Sets, R, rows, ml, &last_sh, nullptr);
        __syncthreads();  // before the shared rows are used again
    }
    end_after_many();
}

// Workspace: a word that a call which gave up sets, arrival counters (zero between calls: a call's last arrivals
// reset them), then partial rows.
constexpr int64_t kHead = 4;  // words ahead of the counters
constexpr int64_t kCounters = 65536;  // more than these of a kind are cleared by the call that needs them
static_assert(2 * 4 * kCounters == ALTXS_PAGED_COUNTER_BYTES, "what the caller zeroes");

struct Plan {
    bool few, many;       // which kernels the host's bounds allow work for
    int group, groups;    // few: rows of an item, items of a (split, head) at most
    int64_t items;        // few: bound on the items
    int part_rows;
    ManyPlan mp;
    int64_t few_cnt, many_cnt, few_part, bytes;  // both lists of counters, then both kernels' partial rows
};
Plan plan_of(const altxs_paged_kv &kv, const altxs_chunks &c, int H, int window) {
    Plan p{};
    const int G = H / kv.n_kv_heads;
    const int64_t n = c.n_seqs;
    if (n == 0) return p;
    const int64_t max_new = std::max(c.max_new, 1);  // (sequences above a bound of 0 are the kernels' to report)
    // The lengths are the device's: n_tokens = n max_new does not say that every sequence has max_new (rows may belong
    // to none), so the kernel for few rows is left out only where a single token has too many of them.
    const int64_t most = max_new * G;  // rows of a sequence
    p.many = most > kMaxRows;
    p.few = G <= kMaxRows;
    p.group = kv.dtype == ALTXS_F32 ? kVecRows : kMaxRows;
    p.groups = (int)((std::min<int64_t>(kMaxRows, most) + p.group - 1) / p.group);
    const int64_t keys = window > 0 ? std::min<int64_t>(c.max_kv, (int64_t)window + c.max_new - 1) : c.max_kv;
    int64_t total = n * keys;
    if (c.total_kv > 0) total = std::min(total, c.total_kv);
    const bool split = keys > kSplitUnit;
    p.items = (split ? total / kSplitUnit + n : n) * kv.n_kv_heads * std::max(p.groups, 1);
    p.part_rows = (int)std::min<int64_t>(p.group, most);
    if (p.few && split) p.few_part = align_up(p.items * p.part_rows * (kv.head_dim + 4) * 4, 256);
    if (p.many) p.mp = paged_many_plan(kv, c, H, window);
    const int64_t part = p.few_part + p.mp.slots * p.mp.slot_bytes;
    p.few_cnt = align_up(4 * std::max(kCounters, kHead + n * kv.n_kv_heads * std::max(p.groups, 1)), 256);
    p.many_cnt = align_up(4 * std::max(kCounters, p.mp.slots + 1), 256);  // its first word: the item tickets
    if (part > 0 || p.many) p.bytes = p.few_cnt + p.many_cnt + part;
    return p;
}

int sm_count() {
    static int sms[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (!sms[dev]) cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
    return sms[dev] > 0 ? sms[dev] : 148;
}

// beside: the kernel for many rows is just ahead in the stream and need not have ended
int launch_few(void (*k)(FewArgs), const FewArgs &f, unsigned grid, int threads, int smem, bool beside, cudaStream_t st) {
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = threads;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &early;
    cfg.numAttrs = beside ? 1 : 0;
    ALTXS_LAUNCH(kKPaged, st, cudaLaunchKernelEx(&cfg, k, f));
    return ALTXS_OK;
}

template <typename T, int HD>
int launch(const PagedAttnArgs &a, const Plan &p, cudaStream_t st) {
    unsigned char *ws = static_cast<unsigned char *>(a.ws);
    uint32_t *spoilt = nullptr, *few_cnt = nullptr, *many_cnt = nullptr;
    float *part = nullptr, *many_part = nullptr;
    if (p.bytes > 0) {
        spoilt = reinterpret_cast<uint32_t *>(ws);
        few_cnt = spoilt + kHead;
        many_cnt = reinterpret_cast<uint32_t *>(ws + p.few_cnt);
        part = reinterpret_cast<float *>(ws + p.few_cnt + p.many_cnt);
        many_part = reinterpret_cast<float *>(ws + p.few_cnt + p.many_cnt + p.few_part);
        if ((p.few_cnt > 4 * kCounters || p.many_cnt > 4 * kCounters) &&
            cudaMemsetAsync(ws, 0, p.few_cnt + p.many_cnt, st) != cudaSuccess)
            return ALTXS_ECUDA;
    }
    const FewArgs f{a, a.H / a.kv.n_kv_heads, 1, kMaxRows, p.group, p.bytes > 0 ? p.items : 0, few_cnt, p.groups, part, p.part_rows};
    const int64_t sms = sm_count();
    if (p.many)
        if (const int rc = launch_paged_many(a, p.mp, kMaxRows + 1, spoilt, many_cnt, many_part, (int)sms, st)) return rc;
    if (!p.few) return ALTXS_OK;
    if constexpr (std::is_same<T, float>::value) {
        const int64_t most = (int64_t)a.c.max_new * f.G;  // rows
        const unsigned grid = (unsigned)std::min<int64_t>(p.items, (most == 1 ? 4 : most <= 2 ? 2 : 1) * sms);
        constexpr int n = kVecWarps * 32;
        return most == 1 ? launch_few(k_paged_vec<HD, 1>, f, grid, n, 0, p.many, st) : most == 2 ? launch_few(k_paged_vec<HD, 2>, f, grid, n, 0, p.many, st)
               : most <= 4 ? launch_few(k_paged_vec<HD, 4>, f, grid, n, 0, p.many, st) : launch_few(k_paged_vec<HD, 8>, f, grid, n, 0, p.many, st);
    } else {
        constexpr int smem = kWarps * kSlots * kChunkBytes;
        static std::atomic<uint64_t> set{0};  // devices whose shared-memory limit is raised
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess) return ALTXS_ECUDA;
        if (dev >= 64 || !((set.load() >> dev) & 1)) {
            if (cudaFuncSetAttribute(k_paged_few<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
                return ALTXS_ECUDA;
            if (dev < 64) set.fetch_or(1ull << dev);
        }
        return launch_few(k_paged_few<T, HD>, f, (unsigned)std::min<int64_t>(p.items, 2 * sms), kWarps * 32, smem, p.many, st);
    }
}
template <typename T>
int launch(const PagedAttnArgs &a, const Plan &p, cudaStream_t st) {
    return a.kv.head_dim == 32 ? launch<T, 32>(a, p, st) : a.kv.head_dim == 64 ? launch<T, 64>(a, p, st) : launch<T, 128>(a, p, st);
}

}  // namespace

int64_t paged_attention_ws(const altxs_paged_kv &kv, const altxs_chunks &c, int H, int window) {
    return plan_of(kv, c, H, window).bytes;
}

int launch_paged_attention(const PagedAttnArgs &a, cudaStream_t st) {
    const Plan p = plan_of(a.kv, a.c, a.H, a.window);
    if (a.kv.dtype == ALTXS_F32) return launch<float>(a, p, st);
    return a.kv.dtype == ALTXS_BF16 ? launch<__nv_bfloat16>(a, p, st) : launch<__half>(a, p, st);
}

}  // namespace altxs
