// Rotary positions and the append of new tokens to a paged key/value cache,
// and the C entry points of the paged cache (the attention's kernels are in
// paged_attn.cu).
//
// Both kernels move every byte once and compute six flops per rotated pair, so
// HBM bounds them (latency, for a few tokens).  A thread handles a unit of 2 V
// channels: for the half layout V channels of each half of the rotated part,
// for the interleaved layout V neighbouring pairs, two V-wide vector accesses
// either way.  It takes that unit of all heads that its lane has of one token, two at
// a time, so that the token's cos and sin are read once for them, and the next
// two (or the next token's first) are on their way while two are rotated and
// stored.  Two heads keep three blocks of 256 threads on an SM: four took
// 126 us, one 121 us where two take 114 us.
//
// Measured: 32768 tokens of 40 heads of 128 in bf16 rotated in 114 us (671 MB,
// 5.9 TB/s); 16384 tokens of 32 query and 8 + 8 key and value heads of 128 in
// fp16 rotated and appended in 219 us (1.28 GB, 5.9 TB/s); one token of 64
// streams in 3.9 us (a launch and two dependent rounds of loads).
#include <algorithm>
#include <cmath>

#include "paged.cuh"
#include "prof.cuh"

namespace altxs {
namespace {

constexpr int kThreads = 256;
constexpr int kHeads = 2;  // heads per thread and pass

// Threads of a token: `upr` units x `hl` head lanes; `tokens` tokens a block.
struct Shape {
    int upr, hl, tokens;
    unsigned threads, grid;
};
Shape shape_of(int64_t n_tokens, int heads, int hd, int v) {
    Shape s;
    s.upr = hd / (2 * v);
    s.hl = std::min((heads + kHeads - 1) / kHeads, std::max(1, kThreads / s.upr));
    const int tpt = s.upr * s.hl;
    s.tokens = std::max(1, kThreads / tpt);
    s.threads = (unsigned)align_up(s.tokens * tpt, 32);
    s.grid = (unsigned)((n_tokens + s.tokens - 1) / s.tokens);
    return s;
}

struct RopeArgs {
    altxs_rotary r;
    int upr, hl, tokens;
    int T, H, hd;
    const int64_t *pos;
    const void *x;
    void *y;
    int64_t ldx, ldy;
    float dir;  // +1 forward, -1 backward: the sense of the rotation
    uint32_t *status;
};

// the two vectors of unit u of a head: channel offsets o0, o1
template <int V, bool IL>
__device__ __forceinline__ void unit_at(int u, int dims, int &o0, int &o1, bool &rot) {
    rot = u < dims / (2 * V);
    if (!IL && rot) {
        o0 = u * V;
        o1 = dims / 2 + u * V;
    } else {
        o0 = u * 2 * V;
        o1 = o0 + V;
    }
}

template <int V>
__device__ __forceinline__ void load_table(const float *p, float *w) {
    if constexpr (V >= 4) {
#pragma unroll
        for (int i = 0; i < V; i += 4) *reinterpret_cast<float4 *>(w + i) = __ldg(reinterpret_cast<const float4 *>(p + i));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = __ldg(p + i);
    }
}

// (a, b) -> (a cos + b sin, b cos - a sin) on the unit's V pairs, in fp32
template <typename T, int V, bool IL>
__device__ __forceinline__ void rotate(Vec<T, V> &x0, Vec<T, V> &x1, const float *cs, const float *sn, float dir) {
    float x[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = to_f(x0.e[i]), x[V + i] = to_f(x1.e[i]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int ia = IL ? 2 * i : i, ib = IL ? 2 * i + 1 : V + i;
        const float a = x[ia], b = x[ib], s = __fmul_rn(dir, sn[i]);
        x[ia] = __fmaf_rn(a, cs[i], __fmul_rn(b, s));
        x[ib] = __fmaf_rn(b, cs[i], -__fmul_rn(a, s));
    }
#pragma unroll
    for (int i = 0; i < V; ++i) x0.e[i] = from_f<T>(x[i]), x1.e[i] = from_f<T>(x[V + i]);
}

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> nan_vec() {
    Vec<T, V> v;
#pragma unroll
    for (int i = 0; i < V; ++i) v.e[i] = from_f<T>(__int_as_float(0x7fffffff));
    return v;
}

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_once(const T *p) {
    Vec<T, V> v;
    if constexpr (sizeof(T) * V == 16) {
        uint4 w;
        asm volatile("ld.global.cs.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "l"(p));
        v = *reinterpret_cast<Vec<T, V> *>(&w);
    } else {
        v = *reinterpret_cast<const Vec<T, V> *>(p);
    }
    return v;
}

// streaming: the written lines are the first to leave the L2 (a plain store cost 144 and 292 us where this costs
// 129 and 227 us, rotary prefill and append of prompts)
template <typename T, int V>
__device__ __forceinline__ void store_once(T *p, const Vec<T, V> &v) {
    if constexpr (sizeof(T) * V == 16) {
        const uint4 w = *reinterpret_cast<const uint4 *>(&v);
        asm volatile("st.global.cs.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
    } else {
        *reinterpret_cast<Vec<T, V> *>(p) = v;
    }
}

template <typename T, int V, bool IL>
__global__ void __launch_bounds__(kThreads, 3) k_rope(RopeArgs a) {
    const int tpt = a.upr * a.hl, ts = threadIdx.x / tpt, w = threadIdx.x - ts * tpt, hl = w / a.upr, u = w - hl * a.upr;
    if (ts >= a.tokens) return;
    int o0, o1;
    bool rot;
    unit_at<V, IL>(u, a.r.dims, o0, o1, rot);
    Vec<T, V> x0[kHeads], x1[kHeads];
    auto load = [&](int64_t t, int h0) {
#pragma unroll
        for (int k = 0; k < kHeads; ++k) {
            const int h = h0 + k * a.hl;
            if (h >= a.H || t >= a.T) break;
            const T *x = static_cast<const T *>(a.x) + t * a.ldx + (int64_t)h * a.hd;
            x0[k] = load_once<T, V>(x + o0);
            x1[k] = load_once<T, V>(x + o1);
        }
    };
    const int64_t step = (int64_t)gridDim.x * a.tokens;
    int64_t t = (int64_t)blockIdx.x * a.tokens + ts, pos = t < a.T ? __ldg(a.pos + t) : 0;
    load(t, hl);
    while (t < a.T) {
        const bool bad = pos < 0 || pos >= a.r.positions;
        if (bad && w == 0) set_status(a.status, ALTXS_ST_BAD_POS);
        float cs[V], sn[V];
        if (rot && !bad) {
            const int64_t at = pos * (a.r.dims / 2) + u * V;
            load_table<V>(a.r.cos + at, cs);
            load_table<V>(a.r.sin + at, sn);
        }
        const int64_t tn = t + step;
        if (tn < a.T) pos = __ldg(a.pos + tn);
        for (int h0 = hl; h0 < a.H; h0 += kHeads * a.hl) {
#pragma unroll
            for (int k = 0; k < kHeads; ++k) {
                const int h = h0 + k * a.hl;
                if (h >= a.H) break;
                if (bad) x0[k] = x1[k] = nan_vec<T, V>();
                else if (rot) rotate<T, V, IL>(x0[k], x1[k], cs, sn, a.dir);
                T *y = static_cast<T *>(a.y) + t * a.ldy + (int64_t)h * a.hd;
                store_once<T, V>(y + o0, x0[k]);
                store_once<T, V>(y + o1, x1[k]);
            }
            const bool next = h0 + kHeads * a.hl >= a.H;  // the next token's
            load(next ? tn : t, next ? hl : h0 + kHeads * a.hl);
        }
        t = tn;
    }
}

struct AppendArgs {
    altxs_paged_kv kv;
    altxs_chunks c;
    altxs_rotary r;  // dims 0: no rotation
    const int64_t *pos;
    const void *q, *k, *v;
    void *q_out;
    int64_t ldq, ldk, ldv, ldqo;
    int Hq;  // 0: no queries
    int upr, hl, tokens, passes;
};

constexpr int kStaged = 512;  // sequence starts kept in shared memory

// Where a token goes: element offset of its cache row (head 0; -1 = not stored) and its rotary position (-1 =
// none, -2 = a row of no sequence).
__device__ __forceinline__ void place_token(const AppendArgs &a, const int32_t *starts, int t, int64_t &off, int64_t &rp) {
    off = -1;
    rp = a.pos ? a.pos[t] : -1;
    int lo = 0, hi = a.c.n_seqs;  // the sequence with q_start[s] <= t < q_start[s + 1]
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (starts[m] <= t) lo = m; else hi = m;
    }
    const Seq q = load_seq(a.c, lo);
    if (q.n >= 0 && (t < q.q0 || t >= q.q0 + q.n)) {  // a row of no sequence
        rp = -2;
        return;
    }
    bool bad = q.n < 0;
    const int p = q.L - q.n + (t - q.q0);
    if (!bad && p >= 0) {
        const int page = a.c.page_table[lo * a.c.table_stride + p / a.kv.page_size];
        if (page >= 0 && page < a.kv.n_pages)
            off = page * a.kv.page_stride + (int64_t)(p % a.kv.page_size) * a.kv.token_stride;
    }
    if (!a.pos) rp = bad ? -1 : p;
    if (!a.r.dims) rp = 0;  // nothing to look up
    else if (rp < 0 || rp >= a.r.positions) rp = -1, off = -1;
    if (off < 0) set_status(a.c.status, ALTXS_ST_BAD_POS);
}

template <typename T, int V, bool IL>
__global__ void __launch_bounds__(kThreads, 3) k_paged_append(AppendArgs a) {
    // A block takes `passes` runs of `tokens` tokens: it finds all their places at once (a chain of four loads),
    // then streams.
    __shared__ int64_t off_sh[kThreads], pos_sh[kThreads];
    __shared__ int32_t start_sh[kStaged];
    const int hd = a.kv.head_dim, Hkv = a.kv.n_kv_heads, nh = a.Hq + 2 * Hkv;
    const int tpt = a.upr * a.hl, ts = threadIdx.x / tpt, w = threadIdx.x - ts * tpt, hl = w / a.upr, u = w - hl * a.upr;
    const int first = blockIdx.x * a.tokens * a.passes, here = min(a.tokens * a.passes, a.c.n_tokens - first);
    int o0, o1;
    bool rot;
    unit_at<V, IL>(u, a.r.dims, o0, o1, rot);
    Vec<T, V> x0[kHeads], x1[kHeads];
    auto load = [&](int t, int h0) {
#pragma unroll
        for (int k = 0; k < kHeads; ++k) {
            const int h = h0 + k * a.hl;
            if (h >= nh) break;
            const T *x = h < a.Hq ? static_cast<const T *>(a.q) + t * a.ldq + (int64_t)h * hd
                         : h < a.Hq + Hkv ? static_cast<const T *>(a.k) + t * a.ldk + (int64_t)(h - a.Hq) * hd
                                          : static_cast<const T *>(a.v) + t * a.ldv + (int64_t)(h - a.Hq - Hkv) * hd;
            x0[k] = load_once<T, V>(x + o0);
            x1[k] = load_once<T, V>(x + o1);
        }
    };
    const bool active = ts < a.tokens;
    if (active && ts < here) load(first + ts, hl);  // on its way while the tokens are placed
    const bool staged = a.c.n_seqs <= kStaged;
    if (staged)
        for (int i = threadIdx.x; i < a.c.n_seqs; i += blockDim.x) start_sh[i] = a.c.q_start[i];
    __syncthreads();
    for (int i = threadIdx.x; i < here; i += blockDim.x) place_token(a, staged ? start_sh : a.c.q_start, first + i, off_sh[i], pos_sh[i]);
    __syncthreads();
    for (int i = ts; active && i < here; i += a.tokens) {
        const int t = first + i;
        const int64_t off = off_sh[i], p = pos_sh[i];
        float cs[V], sn[V];
        if (rot && p >= 0) {
            const int64_t at = p * (a.r.dims / 2) + u * V;
            load_table<V>(a.r.cos + at, cs);
            load_table<V>(a.r.sin + at, sn);
        }
        for (int h0 = hl; h0 < nh; h0 += kHeads * a.hl) {
#pragma unroll
            for (int k = 0; k < kHeads; ++k) {
                const int h = h0 + k * a.hl;
                if (h >= nh) break;
                const bool is_q = h < a.Hq, is_v = h >= a.Hq + Hkv;
                if (p == -2 || (!is_q && off < 0)) continue;
                if (!is_v && a.r.dims) {
                    if (p < 0) x0[k] = x1[k] = nan_vec<T, V>();
                    else if (rot) rotate<T, V, IL>(x0[k], x1[k], cs, sn, 1.0f);
                }
                T *y = is_q ? static_cast<T *>(a.q_out) + t * a.ldqo + (int64_t)h * hd
                            : static_cast<T *>(is_v ? a.kv.v : a.kv.k) + off + (h - a.Hq - (is_v ? Hkv : 0)) * a.kv.head_stride;
                store_once<T, V>(y + o0, x0[k]);
                store_once<T, V>(y + o1, x1[k]);
            }
            if (h0 + kHeads * a.hl < nh) load(t, h0 + kHeads * a.hl);
            else if (i + a.tokens < here) load(t + a.tokens, hl);  // the next token's
        }
    }
}

int es_of(int dtype) { return dtype == ALTXS_F32 ? 4 : 2; }
bool dtype_ok(int dtype) { return dtype == ALTXS_F32 || dtype == ALTXS_BF16 || dtype == ALTXS_F16; }
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_rotary(const altxs_rotary &r, int hd) {
    if ((r.dims && (!r.cos || !r.sin)) || r.positions < 0 || r.dims < 0 || r.dims > hd || (r.dims & 1)) return ALTXS_EINVAL;
    return aligned16(r.cos) && aligned16(r.sin) ? ALTXS_OK : ALTXS_EINVAL;
}

// The widest unit that head size, rotated part, row strides and bases allow:
// 16-byte vectors, 8-byte ones, or single elements.
int unit_width(int dtype, int hd, int dims, std::initializer_list<const void *> bases,
               std::initializer_list<int64_t> lds) {
    const int es = es_of(dtype);
    for (int v = 16 / es; v >= 8 / es; v /= 2) {
        bool ok = hd % (2 * v) == 0 && dims % (2 * v) == 0;
        for (const void *b : bases) ok = ok && reinterpret_cast<uintptr_t>(b) % (v * es) == 0;
        for (int64_t l : lds) ok = ok && l % v == 0;
        if (ok) return v;
    }
    return 1;
}

// F<T, V, interleaved>::go(args...) for run-time dtype, width (full, half, 1) and layout
template <template <typename, int, bool> class F, typename... A>
void dispatch(int dtype, int v, bool il, A... args) {
#define ALTXS_V(T, N)                                   \
    if (v == N) {                                       \
        if (il) F<T, N, true>::go(args...);             \
        else F<T, N, false>::go(args...);               \
        return;                                         \
    }
    if (dtype == ALTXS_F32) {
        ALTXS_V(float, 4) ALTXS_V(float, 2) ALTXS_V(float, 1)
    } else if (dtype == ALTXS_BF16) {
        ALTXS_V(__nv_bfloat16, 8) ALTXS_V(__nv_bfloat16, 4) ALTXS_V(__nv_bfloat16, 1)
    } else {
        ALTXS_V(__half, 8) ALTXS_V(__half, 4) ALTXS_V(__half, 1)
    }
#undef ALTXS_V
}
template <typename T, int V, bool IL>
struct GoRope {
    static void go(const RopeArgs &a, Shape s, cudaStream_t st) { k_rope<T, V, IL><<<s.grid, s.threads, 0, st>>>(a); }
};
template <typename T, int V, bool IL>
struct GoAppend {
    static void go(const AppendArgs &a, Shape s, cudaStream_t st) { k_paged_append<T, V, IL><<<s.grid, s.threads, 0, st>>>(a); }
};

int check_kv(const altxs_paged_kv &kv) {
    if (!dtype_ok(kv.dtype) || kv.page_size < 1 || kv.n_pages < 0 || kv.n_kv_heads < 1) return ALTXS_EINVAL;
    if (kv.head_dim != 32 && kv.head_dim != 64 && kv.head_dim != 128) return ALTXS_ENOTSUP;
    const int64_t u = 16 / es_of(kv.dtype);
    if (!aligned16(kv.k) || !aligned16(kv.v) || kv.page_stride % u || kv.token_stride % u || kv.head_stride % u)
        return ALTXS_EINVAL;
    if (kv.page_stride < 0 || kv.token_stride < kv.head_dim || kv.head_stride < kv.head_dim) return ALTXS_EINVAL;
    return ALTXS_OK;
}
constexpr int kMaxLength = 1 << 30;  // positions of a sequence: their sums with windows and tiles stay in 32 bits
// a window that covers every position is none
int window_of(const altxs_chunks &c, int window) { return window >= c.max_kv ? 0 : window; }
int check_chunks(const altxs_paged_kv &kv, const altxs_chunks &c) {
    if (c.n_seqs < 0 || c.n_tokens < 0 || c.max_new < 0 || c.max_kv < 0 || c.table_stride < 0 || c.total_kv < 0)
        return ALTXS_EINVAL;
    if (c.table_stride * kv.page_size < c.max_kv) return ALTXS_EINVAL;
    return c.max_kv > kMaxLength || c.max_new > kMaxLength ? ALTXS_ENOTSUP : ALTXS_OK;
}

}  // namespace
}  // namespace altxs

using namespace altxs;

extern "C" {

int altxs_rope(int dtype, int n_tokens, int n_heads, int head_dim, const altxs_rotary *r, const int64_t *pos,
               int backward, const void *x, int64_t ldx, void *y, int64_t ldy, uint32_t *status,
               altxs_stream_t stream) {
    if (!dtype_ok(dtype) || !r || n_tokens < 0 || n_heads < 0 || head_dim < 2 || (head_dim & 1)) return ALTXS_EINVAL;
    if (head_dim > 512) return ALTXS_ENOTSUP;
    const int64_t width = (int64_t)n_heads * head_dim;
    if (ldx < width || ldy < width) return ALTXS_EINVAL;
    if (n_tokens == 0 || n_heads == 0) return ALTXS_OK;
    if (const int rc = check_rotary(*r, head_dim)) return rc;
    const uintptr_t em = (uintptr_t)es_of(dtype) - 1;
    if (!pos || !x || !y || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & em) ||
        (x == y && ldx != ldy))
        return ALTXS_EINVAL;
    const int v = unit_width(dtype, head_dim, r->dims, {x, y}, {ldx, ldy});
    Shape sh = shape_of(n_tokens, n_heads, head_dim, v);
    sh.grid = std::min(sh.grid, 148u * 24u);
    const RopeArgs a{*r, sh.upr, sh.hl, sh.tokens, n_tokens, n_heads, head_dim, pos, x, y, ldx, ldy, backward ? -1.0f : 1.0f, status};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    ALTXS_LAUNCH(kKRope, st, dispatch<GoRope>(dtype, v, r->interleaved != 0, a, sh, st));
    return ALTXS_OK;
}

int altxs_paged_append(const altxs_paged_kv *kv, const altxs_chunks *c, const altxs_rotary *r, const int64_t *pos,
                       const void *k, int64_t ldk, const void *v, int64_t ldv, int n_heads, const void *q,
                       int64_t ldq, void *q_out, int64_t ldqo, altxs_stream_t stream) {
    if (!kv || !c) return ALTXS_EINVAL;
    if (const int rc = check_kv(*kv)) return rc;
    if (const int rc = check_chunks(*kv, *c)) return rc;
    const int hd = kv->head_dim;
    const int64_t kvw = (int64_t)kv->n_kv_heads * hd;
    if (ldk < kvw || ldv < kvw || n_heads < 0) return ALTXS_EINVAL;
    if (q && (!q_out || ldq < (int64_t)n_heads * hd || ldqo < (int64_t)n_heads * hd || (q == q_out && ldq != ldqo)))
        return ALTXS_EINVAL;
    if (c->n_seqs == 0 || c->n_tokens == 0) return ALTXS_OK;
    if (r)
        if (const int rc = check_rotary(*r, hd)) return rc;
    if (!k || !v || !kv->k || !kv->v || !c->q_start || !c->kv_len || !c->page_table) return ALTXS_EINVAL;
    const int Hq = q ? n_heads : 0;
    AppendArgs a{*kv, *c, r ? *r : altxs_rotary{}, pos, q, k, v, q_out, ldq, ldk, ldv, ldqo, Hq, 0, 0, 0, 1};
    const uintptr_t em = (uintptr_t)es_of(kv->dtype) - 1;
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(q) |
         reinterpret_cast<uintptr_t>(q_out)) & em)
        return ALTXS_EINVAL;
    const int w = q ? unit_width(kv->dtype, hd, a.r.dims, {k, v, q, q_out}, {ldk, ldv, ldq, ldqo})
                    : unit_width(kv->dtype, hd, a.r.dims, {k, v}, {ldk, ldv});
    Shape sh = shape_of(c->n_tokens, Hq + 2 * kv->n_kv_heads, hd, w);
    // runs per block: as many as leave every SM eight blocks
    a.passes = std::max(1, std::min({c->n_tokens / (sh.tokens * 148 * 8), kThreads / sh.tokens, 32}));
    sh.grid = (unsigned)((c->n_tokens + (int64_t)sh.tokens * a.passes - 1) / ((int64_t)sh.tokens * a.passes));
    a.upr = sh.upr, a.hl = sh.hl, a.tokens = sh.tokens;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    ALTXS_LAUNCH(kKRope, st, dispatch<GoAppend>(kv->dtype, w, a.r.interleaved != 0, a, sh, st));
    return ALTXS_OK;
}

int64_t altxs_paged_attention_workspace_bytes(const altxs_paged_kv *kv, const altxs_chunks *c, int n_heads,
                                              int window) {
    if (!kv || !c || check_kv(*kv) || check_chunks(*kv, *c) || n_heads < 1 || n_heads % kv->n_kv_heads || window < 0)
        return -1;
    return paged_attention_ws(*kv, *c, n_heads, window_of(*c, window));
}

int altxs_paged_attention(const altxs_paged_kv *kv, const altxs_chunks *c, int n_heads, float scale, int window,
                          const void *q, int64_t ldq, void *out, int64_t ldo, float *lse, void *workspace,
                          int64_t workspace_bytes, altxs_stream_t stream) {
    if (!kv || !c) return ALTXS_EINVAL;
    if (const int rc = check_kv(*kv)) return rc;
    if (const int rc = check_chunks(*kv, *c)) return rc;
    if (n_heads < 1 || n_heads % kv->n_kv_heads || window < 0 || !std::isfinite(scale)) return ALTXS_EINVAL;
    const int64_t width = (int64_t)n_heads * kv->head_dim, u = 16 / es_of(kv->dtype);
    if (ldq < width || ldo < width || ldq % u || ldo % u || !aligned16(q) || !aligned16(out)) return ALTXS_EINVAL;
    if (c->n_seqs == 0 || c->n_tokens == 0) return ALTXS_OK;
    if (!q || !out || !kv->k || !kv->v || !c->q_start || !c->kv_len || !c->page_table) return ALTXS_EINVAL;
    window = window_of(*c, window);
    const int64_t need = paged_attention_ws(*kv, *c, n_heads, window);
    if (workspace_bytes < need || (need > 0 && !workspace) || !aligned16(workspace)) return ALTXS_ENOSPC;
    return launch_paged_attention(PagedAttnArgs{*kv, *c, n_heads, window, scale, q, ldq, out, ldo, lse, workspace,
                                                workspace_bytes},
                                  reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
