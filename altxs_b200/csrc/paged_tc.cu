// Attention of many new tokens over a paged key/value cache on the tensor
// cores, the scores never leaving the SM.
//
// The rows of one key/value head (its G query heads x the sequence's new
// tokens, row = token * G + head) are cut into blocks of 256 (fp32 with 128
// channels: 128); an item is one split of one block's visible key tiles (128
// positions each; there: 64), taken by a persistent block of warps:
//   warps 0-3, 4-7  softmax groups 0 and 1, one score row per thread;
//   warp 8          issues the MMAs: S = Q K^T into a group's tensor-memory
//                   score columns, then (P written over S) O += P V, P read
//                   from tensor memory, V as it lies (MN-major);
//   the rest        fetch key and value rows through the page table into a
//                   ring of tiles by tensor copies, one for each run of
//                   positions within a page (16 bits: and 64-channel half);
//                   runs that no row of the block needs are filled with zeros.
// With more than 128 rows each group owns 128 of them and every key tile
// serves both; with at most 128 the two groups share the rows and take even
// and odd key tiles, and both outputs are joined at the end.  Either way the
// MMA warp alternates between the groups, so one group's softmax runs under
// the other's MMAs.  At most 64 (32) rows are held 2 (4) times, each copy with
// its share of a tile's columns.
//
// Softmax: x = s scale log2(e) in fp32, p = 2^(x - m), the sum from the
// unrounded p.  m follows the running maximum only when that grows by more
// than 2^8: until then p <= 256 is as exact, and O (fp32, in tensor memory) is
// not touched.
//
// 16-bit types: the tiles are the cache's own rows, p is rounded to the type for
// P V (a second plane of p would double that product): the error against 64 bits
// is 1.2 to 1.3 times the plain form's, which keeps p in fp32 and rounds the
// output once (bf16 0.0022 and 0.0017, fp16 0.00026 and 0.00021 relative).
// Warps 9 and 11 fetch every other tile, warp 10 draws and announces the items
// and clears what must not meet a p = 0 in tiles that not every row sees whole.
// fp32: every operand is a pair of fp16 planes, hi = fp16(v 2^a) and lo = fp16(v
// 2^a - hi), the power of two chosen per query row and per 2 KB of keys and of
// values (per position in tiles that not every row sees whole) so that the
// largest magnitude is at 2^14: hi + lo keeps 22 significant bits of everything
// within 2^-18 of that magnitude, and 2^-40 of it below.  p carries the values'
// powers, O their running largest per row.  A product is hi hi + hi lo + lo hi
// with fp32 sums: three fp16 products instead of six with bf16 planes or three
// at half the rate with tf32.  (An infinity has no low plane: one among the keys
// or values that a row sees leaves it NaN.)  Warp 9 fetches raw rows to a stage
// each for keys and values (and announces the items), warps 10 to 15 write the
// planes.
//
// Bounds: at full tiles the softmax group's own chain (wait for S and the P V
// before it, load and maximum, exponentials, store: about 4000 clocks for two
// jobs of 128 x 128 x 128, of which the MMAs are 2050); otherwise an item's
// start and end (mostly cold code; with 64 channels about 4000 clocks to find
// the first item, 2000 for the queries, 1500 for the last products and 7000 for
// the outputs).  Items are drawn by ticket, longest first, one ahead: two or
// three ahead the long piece took 743 us where it took 651.  (Found by every
// role for itself instead of by one ahead of all: 5 tokens of 48 streams 35 us
// where they took 31.)  A sequence is cut as if it were alone, so 16 streams of
// 8 pairs are 256 items for 148 SMs, where uncut they are 128.  Pages whose size
// is not a multiple of 4 are fetched position by position: 5 tokens of 48
// streams 105 us with pages of 1 to 3, 47 with 4, 40 with 8, 36 with 16 and
// more.
// Measured per call: 4096 new tokens over 20000 positions, 16 heads over 8, hd
// 128 in fp16: 647 us at 1965 MHz (931 TFLOP/s), 708 us back to back, where the
// power limit holds the SMs at 1765 MHz; nine ragged sequences of up to 1999 new
// tokens, 16 heads over 4, bf16: 204 us (648 TFLOP/s); 5 new tokens of 48
// streams in windows of 1024, 16-token pages, fp16: 35 us; 64 new tokens of 16
// streams over windows of 2048, 8 heads of 64, fp32: 97 us.  (Of the last two 1
// us is the empty kernel for few rows behind this one, and in fp32 5 us more the
// code that it drives out of the instruction cache, where nothing runs between
// two calls.)
//
// Splits of a block go to the workspace as (m, l, O); the item that arrives
// last joins them in split order.  Tiles, blocks and splits are functions of
// the sequence's own lengths, so a row's bits do not depend on the batch.
//
// Every wait is bounded: one that gives up stops the block's roles, which let
// their copies and MMAs finish, and sets ALTXS_ST_TIMEOUT.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "paged.cuh"
#include "prof.cuh"
#include "tcgen05.cuh"

namespace altxs {
namespace {

constexpr int kMmaWarp = 8;
constexpr int kScan = 64;        // sequences are counted in this many groups
constexpr int kMostItems = 1184;  // splits of one sequence
constexpr int kSms = 148;
constexpr int kMostSplits = 16;
constexpr int kNext = 4;           // items announced to a block's roles ahead
constexpr unsigned kAll = 0xffffffffu;
constexpr float kLazy = 8.0f;

template <typename T, int HD>
struct Tc {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int KT = F32 && HD > 64 ? 64 : 128;     // positions per key tile
    static constexpr int Rows = F32 && HD > 64 ? 128 : 256;  // rows per item
    static constexpr int Planes = F32 ? 2 : 1;
    static constexpr int Halves = HD > 64 ? 2 : 1;           // 64-channel halves of a plane
    static constexpr int PlaneB = Halves * KT * 128;         // HD 32 leaves half of each 128-byte row unused
    static constexpr int TileB = Planes * PlaneB;
    static constexpr int QPlaneB = Halves * 128 * 128, QTileB = Planes * QPlaneB;  // 128 rows
    static constexpr int Loaders = F32 ? 7 : 3;  // warps from 9 on
    static constexpr int Converters = 6;         // fp32: of them, warps 10 to 15
    static constexpr int Threads = (kMmaWarp + 1 + Loaders) * 32;
    // registers: (8 warps x RegS + the others x RegP) x 32 = Threads x 168 (16 bits) or 128 (fp32)
    static constexpr int RegS = F32 ? 176 : 208, RegP = F32 ? 80 : 88;
    static_assert(256 * RegS + (Threads - 256) * RegP == Threads * (F32 ? 128 : 168), "register split");
    static constexpr int Slots = F32 ? 3 : HD > 64 ? 5 : 11;
    static constexpr int UnitRows = F32 ? 512 / HD : KT, Units = KT / UnitRows;  // fp32: rows that share an exponent
    static constexpr int StageB = F32 ? KT * HD * 4 : 0;  // fp32: a tile's raw rows, one stage for keys and one for values
    // Key tiles (and items) the producers are ahead of the softmax, at most.  fp32: while the oldest tile's values
    // keep their slot, the next tile is in the slots, one more in the stages and the masks of the one after it known.
    static constexpr int Ring = F32 ? 4 : Slots > 8 ? 16 : 8;
    static constexpr int QB = Rows / 128 * QTileB;
    static constexpr int MlAt = QB > 32768 ? 32768 : QB + Slots * TileB;  // 256 (m, l): see the softmax warps
    static constexpr int Smem = QB + Slots * TileB + 2 * StageB + (QB > 32768 ? 0 : 2048) + 1024;
    // Tensor memory of group i: S at KT i, O at 256 + HD i.  fp32 up to 64 channels keeps the small products
    // (hi lo + lo hi) apart at 256 + HD (2 + i): a sum loses least when it meets O's magnitude least often.
    static constexpr bool Apart = F32 && HD <= 64;
    static constexpr uint32_t ColS = 0, ColO = 2 * 128;
    static_assert(Smem + 2048 <= 227 * 1024, "shared memory (with the static part)");
};
// the same two numbers for the host and the item arithmetic
__host__ __device__ inline int tile_keys(int dtype, int hd) { return dtype == ALTXS_F32 && hd > 64 ? 64 : 128; }
__host__ __device__ inline int block_rows(int dtype, int hd) { return dtype == ALTXS_F32 && hd > 64 ? 128 : 256; }

// One sequence's share of the work: its (block, head) pairs, longest blocks
// first; the first `whole` of them are one item each, the others nsplit items.
struct Shape {
    int pairs, whole, nsplit;
    __host__ __device__ int items() const { return whole + (pairs - whole) * nsplit; }
};
__host__ __device__ inline int tiles_of(int keys, int kt) { return (keys + kt - 1) / kt; }
// A sequence by itself fills the 148 SMs in whole waves; the pairs of the last,
// partly filled wave are cut so that they spread over all SMs, at least 8 key
// tiles to a split (a split costs about 4.5 tiles' time, a whole item 1.5) and
// only for a twentieth or more of the sequence's time.
__host__ __device__ inline void split_rule(Shape &w, int nt) {
    const int waves = w.pairs / kSms, rest = w.pairs - waves * kSms, most = nt / 8;
    w.whole = w.pairs;
    w.nsplit = 1;
    if (rest == 0 || most < 2) return;
    float cost = (float)nt + 1.5f;
    const float gain = 0.05f * cost * (float)(waves + 1);
    cost -= gain;
#pragma unroll
    for (int ns = 2; ns <= kMostSplits; ++ns) {  // unrolled: the divisors are constants
        const float c = (float)((rest * ns + kSms - 1) / kSms) * ((float)nt * (1.0f / (float)ns) + 4.5f);
        if (ns <= most && rest * ns <= kMostItems && c < cost) cost = c, w.nsplit = ns;
    }
    if (w.nsplit > 1) w.whole = waves * kSms;
}

// Waves that the cut pairs of a sequence of nt tiles take at most: the least tiles for which the rule chooses 2, 3, ..
// waves for any number of pairs (less one, for sums that round otherwise on the device).
inline int most_waves(int64_t nt) {
    constexpr int from[] = {16, 26, 60, 110, 180, 275, 401, 565};
    int w = 0;
    while (w < 8 && nt >= from[w]) ++w;
    return w;
}

struct ManyArgs {
    PagedAttnArgs a;
    int G, min_rows;    // sequences with at least min_rows rows are this kernel's
    int run;            // positions that lie within a page
    int64_t max_slots;  // partial slots in the workspace (one per item of a split sequence)
    uint32_t *spoilt;   // set by a call that gave up: its counters may still be counting
    uint32_t *cnt;      // [max_slots], zero between calls
    uint32_t *ticket;   // items handed out beyond the first of each block, zero between calls
    float *part;        // [max_slots][part_rows * (HD + 2)]
    int part_rows;
};

template <class C>
__device__ __forceinline__ Shape shape_of(const ManyArgs &f, const Seq &q) {
    Shape w{0, 0, 1};
    if (q.n <= 0 || q.n * f.G < f.min_rows) return w;
    const int R = q.n * f.G;
    w.pairs = (R + C::Rows - 1) / C::Rows * f.a.kv.n_kv_heads;
    // the longest block: the last rows' keys
    const int toks = (min(R, C::Rows) + f.G - 1) / f.G;
    const int keys = f.a.window > 0 ? min(q.L, f.a.window + toks - 1) : q.L;
    split_rule(w, tiles_of(max(keys, 0), C::KT));
    return w;
}

struct Scan {
    int before[kScan + 1], slots[kScan + 1];  // items, and partial slots, before each group of sequences
    int per;
    uint32_t share[kScan];  // groups of one sequence: whole << 5 | nsplit of its shape
};

struct Item {
    Seq q;
    int s, g, nsplit, split;
    int r0, rows;        // rows of the block
    int lo, hi, base, t0, t1;  // the block sees [lo, hi); positions base + KT t of key tiles t0 .. t1 of this split
    bool two;            // two row tiles (both groups over every key tile)
    int slot;            // partial slot of the block's split 0
};

template <class C>
__device__ __forceinline__ Item locate(const ManyArgs &f, const Scan &sc, int item) {
    int lo = 0, hi = kScan;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (sc.before[m] <= item) lo = m; else hi = m;
    }
    Item it;
    const int Hkv = f.a.kv.n_kv_heads;
    it.s = lo * sc.per;
    int local = item - sc.before[lo], slot = sc.slots[lo];
    Shape w;
    it.q = load_seq(f.a.c, it.s);
    if (sc.per == 1) {
        w.whole = sc.share[lo] >> 5, w.nsplit = sc.share[lo] & 31;
    } else {
        w = shape_of<C>(f, it.q);
        for (int n; it.s < f.a.c.n_seqs - 1 && local >= (n = w.items()); w = shape_of<C>(f, it.q)) {
            local -= n;
            slot += n - w.whole;
            it.q = load_seq(f.a.c, ++it.s);
        }
    }
    const int R = it.q.n * f.G;
    it.nsplit = 1, it.split = 0, it.slot = 0;
    if (local >= w.whole && w.nsplit > 1) {
        const int r = local - w.whole, pr = r / w.nsplit;
        it.nsplit = w.nsplit;
        it.split = r - pr * w.nsplit;
        it.slot = slot + r - it.split;
        local = w.whole + pr;
    }
    const int bd = local / Hkv, blk = (R + C::Rows - 1) / C::Rows - 1 - bd;  // the longest blocks first
    it.g = local - bd * Hkv;
    it.r0 = blk * C::Rows;
    it.rows = min(R - it.r0, C::Rows);
    it.two = it.rows > 128;
    const int p0 = it.q.L - it.q.n, i0 = it.r0 / f.G, i1 = (it.r0 + it.rows - 1) / f.G;
    it.hi = max(0, p0 + i1 + 1);
    it.lo = f.a.window > 0 ? max(0, p0 + i0 - f.a.window + 1) : 0;
    it.base = it.lo / C::KT * C::KT;  // tiles start at multiples of KT: no run of a page crosses a tile
    const int nt = tiles_of(max(0, it.hi - it.base), C::KT), per = (nt + it.nsplit - 1) / it.nsplit;
    it.t0 = min(nt, it.split * per);
    it.t1 = min(nt, it.t0 + per);
    return it;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void sts16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void sts8(uint32_t addr, uint2 v) {
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
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
template <typename T>
constexpr uint32_t idesc(int n, int bmn) {  // kind::f16 (bf16, or fp16: fp32's planes too), fp32 sums, M = 128, A K-major
    const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)bmn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// whether a phase is complete, without waiting (mbar_try_wait may sleep for a while first)
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
// Matrix descriptors of 128-byte-swizzled tiles: the upper word is the same for
// all of them (8-row groups every 1024 bytes), the lower one holds the address
// and, for MN-major tiles, the distance of 64-channel halves; offsets are added
// in units of 16 bytes.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | (lbo >> 4) << 16; }
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %5, 0;\n mov.b64 a, {%1, %3};\n mov.b64 b, {%2, %3};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(kDescHi), "r"(id), "r"(accumulate)
        : "memory");
}
// D += A B with A (rows = lanes, two 16-bit values per column) in tensor memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.b32 p, %5, 0;\n mov.b64 b, {%2, %3};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(kDescHi), "r"(id), "r"(accumulate)
        : "memory");
}
#define ALTXS_R32(v) \
    "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), \
    "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), \
    "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), \
    "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        ALTXS_R32(v)
        : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 columns without waiting; tc_wait_ld, then tc_tie32 before the values are used
__device__ __forceinline__ void tc_ld32_nowait(uint32_t taddr, float *f) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tc_ld16(uint32_t taddr, float *f) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_tie32(float *f) {
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        asm volatile("" : "+f"(f[i]), "+f"(f[i + 1]), "+f"(f[i + 2]), "+f"(f[i + 3]), "+f"(f[i + 4]), "+f"(f[i + 5]),
                          "+f"(f[i + 6]), "+f"(f[i + 7])::"memory");
}

// 8 consecutive values to dst (16- or 32-byte aligned)
template <typename T>
__device__ __forceinline__ void store8(T *dst, const float *v) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4 *>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4 *>(dst) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
}
// fp16 planes of two values
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(__fsub_rn(a, f.x), __fsub_rn(b, f.y));
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
// Exponent e of the largest finite magnitude (its bits), -100 at least: 2^(14 - e) scales it to 2^14 ..
__device__ __forceinline__ int exp_of(uint32_t bits) { return max((int)(bits >> 23) - 127, -100); }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ uint32_t finite_abs(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}

// Exponents travel as the bytes of fp32's exponent field: keys' of 2^(e - 14), values' of 2^(e - kVal).
constexpr int kVal = 12;
__device__ __forceinline__ float pow2_byte(uint32_t word, int i) {  // of byte i
    return __uint_as_float((i == 0 ? word << 23 : i == 1 ? word << 15 : i == 2 ? word << 7 : word >> 1) & 0x7f800000u);
}

// two fp32 operations per instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
        " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}\n"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
        " add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}\n"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
        " mul.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}\n"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// The values of channel `dim` that are not finite, over the positions [lo, hi) that a
// row at `pos` sees (the tiles that only some rows see hold 0 in their place).
template <typename T>
__device__ __noinline__ float odd_term(const PagedAttnArgs &a, int s, int g, int pos, int lo, int hi, int dim) {
    float y = 0.0f;
    for (int k = max(lo, a.window > 0 ? pos - a.window + 1 : 0); k < min(hi, pos + 1); ++k) {
        const int b = k / a.kv.page_size, page = __ldg(a.c.page_table + s * a.c.table_stride + b);
        if (page < 0 || page >= a.kv.n_pages) continue;
        const float v = to_f(static_cast<const T *>(a.kv.v)[page * a.kv.page_stride +
                                                           (int64_t)(k - b * a.kv.page_size) * a.kv.token_stride +
                                                           g * a.kv.head_stride + dim]);
        if (!isfinite(v)) y = __fadd_rn(y, v);
    }
    return y;
}

template <typename T, int HD>
__global__ void __launch_bounds__(Tc<T, HD>::Threads, 1) k_paged_many(const __grid_constant__ ManyArgs f, const __grid_constant__ CUtensorMap tk,
                                                                        const __grid_constant__ CUtensorMap tv) {
    using C = Tc<T, HD>;
    constexpr int KT = C::KT;
    constexpr bool F32 = C::F32, Half = std::is_same<T, __half>::value;
    extern __shared__ unsigned char pm_smem_raw[];
    __shared__ __align__(8) uint64_t full[C::Slots], empty[C::Slots], landed[F32 ? 1 : C::Slots], s_full[2], p_full[2], o_done[2], q_full, drainb,
        raw_full[2], raw_empty[2], next_full[kNext], next_empty[kNext], want;
    __shared__ Scan sc;
    // by key tile: which positions exist (4 to a byte), and (fp32) the exponents of its positions' keys and values.
    // Two tiles of those do: a tile's are written once the values' slot of the tile two before is free.
    __shared__ __align__(16) uint8_t kmask[C::Ring][KT / 4];
    __shared__ __align__(16) uint8_t kv_exp[F32 ? 2 : 1][2][F32 ? KT : 16];
    static_assert(!F32 || C::Slots <= 3, "exponents of two tiles");
    __shared__ uint32_t tmem_sh;
    __shared__ __align__(8) uint8_t odd8_sh[F32 ? C::Ring : 1][8];  // by item: values that are not finite were set to 0 (fp32: per warp)
    __shared__ uint32_t odd_sh[F32 ? 1 : C::Ring];
    __shared__ int2 wsum[kScan / 32];
    __shared__ int last_sh, item_sh;
    __shared__ __align__(16) Item next_sh[kNext];
    __shared__ volatile int abort_sh;
    const PagedAttnArgs &a = f.a;
    const uint32_t raw_s = smem_u32(pm_smem_raw);
    const uint32_t sq = raw_s + ((1024u - (raw_s & 1023u)) & 1023u), ring = sq + C::QB;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t limit = wait_limit();
    // the kernel for few rows (it shares no sequence with this one) may start as these blocks leave
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int s = 0; s < C::Slots; ++s) {
            mbar_init(&full[s], F32 ? C::Converters : 1);
            mbar_init(&empty[s], 1);
            if (!F32) mbar_init(&landed[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_done[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&raw_full[i], 1);
            mbar_init(&raw_empty[i], C::Converters);
        }
        for (int i = 0; i < kNext; ++i) {
            mbar_init(&next_full[i], 1);
            mbar_init(&next_empty[i], C::Loaders + 1);  // the other loaders, the MMA warp, softmax warp 0
        }
        mbar_init(&q_full, 8);
        mbar_init(&drainb, 1);
        mbar_init(&want, 1);
        abort_sh = 0;
        for (int i = 0; i < (F32 ? 1 : C::Ring); ++i) odd_sh[i] = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_sh)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp < kScan / 32) {  // items of the sequences before each thread's group of them
        const int n = a.c.n_seqs, per = (n + kScan - 1) / kScan;
        int sum = 0, cut = 0;
        for (int s = tid * per; s < min(n, (tid + 1) * per); ++s) {
            const Seq q = blockIdx.x == 0 ? load_seq_report(a.c, s) : load_seq(a.c, s);
            const Shape w = shape_of<C>(f, q);
            sum += w.items();
            if (w.nsplit > 1) cut += w.items() - w.whole;
            if (per == 1) sc.share[s] = w.whole << 5 | w.nsplit;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(kAll, sum, o), u = __shfl_up_sync(kAll, cut, o);
            if (lane >= o) sum += v, cut += u;
        }
        if (lane == 31) wsum[warp] = make_int2(sum, cut);
        asm volatile("bar.sync 1, %0;" ::"n"(kScan) : "memory");
        for (int w = 0; w < warp; ++w) sum += wsum[w].x, cut += wsum[w].y;
        sc.before[tid + 1] = sum, sc.slots[tid + 1] = cut;
        if (tid == 0) sc.before[0] = sc.slots[0] = 0, sc.per = per;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_sh;
    const int total = sc.before[kScan];
    // Items go to whoever is free (they differ in length several times over): one warp (the one with the least to do)
    // draws a ticket per item, finds what it is and announces it, an item ahead; s = -1: there is none.
    constexpr int kAnnouncer = F32 ? 0 : 1;  // of the producers
    auto announced = [&](int r, Item &it) {  // a warp's r-th item
        const bool got = __all_sync(kAll, mbar_wait_bounded(&next_full[r % kNext], (r / kNext) & 1, limit));
        if (got) it = next_sh[r % kNext];
        else it.s = -1, abort_sh = 1;
        __syncwarp();
        if (got && lane == 0) mbar_arrive(&next_empty[r % kNext]);
    };

    if (warp > kMmaWarp) {
        // ---- producers ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::RegP));
        const int pw = warp - kMmaWarp - 1;
        const int P = a.kv.page_size, pshift = (P & (P - 1)) == 0 ? 31 - __clz(P) : -1;
        auto block_of = [&](int k) { return pshift >= 0 ? k >> pshift : k / P; };
        uint32_t n = 0, kt = 0, live = 0;  // slots, key tiles and items with tiles so far
        bool ok = true;
        // The tile whose copies come next: found (and its page numbers on their way) one tile ahead.
        int round = 0, t = 0, drawn = blockIdx.x, told = 0;  // items taken, tile, last item drawn, items announced
        Item it;
        it.t1 = 0;
        bool fresh = false, more = true, none = false;
        auto announce = [&]() {
            // not before the loads have come to the item ahead of it: an item drawn early is one that a free block misses
            if (!F32 && told > 0 && !__all_sync(kAll, !abort_sh && mbar_wait_bounded(&want, (told - 1) & 1, limit))) {
                ok = more = false;
                return;
            }
            if (told > 0 && lane == 0) drawn = (int)gridDim.x + (int)atomicAdd(f.ticket, 1u);
            const int item = __shfl_sync(kAll, drawn, 0), slot = told % kNext;
            if (told >= kNext && !__all_sync(kAll, mbar_wait_bounded(&next_empty[slot], (told / kNext - 1) & 1, limit))) {
                ok = more = false;
                return;
            }
            Item next;
            next.s = -1;
            if (item < total) next = locate<C>(f, sc, item);
            if (lane == 0) {
                next_sh[slot] = next;
                mbar_arrive(&next_full[slot]);
            }
            __syncwarp();
            ++told;
        };
        // To the next tile, or past one item that has none: a warp issues the copies it holds back before it goes past
        // more items, whose announcements may wait for the softmax to take one that waits for those copies.
        auto advance = [&]() {
            ++t;
            fresh = none = false;
            if (t < it.t1) return;
            if (pw == kAnnouncer) {
                if (told == round) announce();
                if (!ok) return;
                it = next_sh[round++ % kNext];
            } else {
                announced(round++, it);
                if (pw == 0 && lane == 0) mbar_arrive(&want);
            }
            if (it.s < 0) {
                more = false;
                return;
            }
            t = it.t0;
            fresh = true;
            none = t >= it.t1;
        };
        // Positions [all0, all1) are seen by every row of the block.
        int all0 = 0, all1 = 0;
        auto bounds = [&]() {
            const int p0 = it.q.L - it.q.n;
            all1 = p0 + it.r0 / f.G + 1;
            all0 = a.window > 0 ? p0 + (it.r0 + it.rows - 1) / f.G - a.window + 1 : 0;
        };
        if constexpr (!F32) {
            // Runs of `run` positions (the largest power of two up to KT that divides the page size) lie within a
            // page: one tensor copy per run and 64-channel half.  Runs of no page or outside [lo, hi) take a
            // page number past the pool, which fills zeros.
            const int run = f.run, runs = KT / run, mine = runs < 32 ? runs : 32;
            // A values tile whose rows are not all seen by every row of the block goes to landed[] first, and
            // warp 10 clears what must not meet a p = 0: rows outside [lo, hi), and values that are not finite
            // in rows that only some see (the latter reach those in the epilogue).
            auto mixed = [&]() {
                const int kb = it.base + t * KT;
                return kb < max(all0, it.lo) || kb + KT > min(all1, it.hi);
            };
            uint32_t lph = 0;  // landed[]'s parities, by slot
            if (pw != 1) {
                // Warp 9 fetches the even tiles, warp 11 the odd ones: a warp issues one copy in about 100 clocks, and
                // finding a tile's pages takes as long as eight of them.  (With all keys to one and all values to the
                // other it was no faster or slower.)
                const uint32_t odd = pw >> 1;
                uint32_t issued = 0, was_look = 0;  // copies up to this warp's last; slots whose last copy went to landed[]
                int page[KT / 32];
                auto fetch = [&]() {
#pragma unroll
                    for (int e = 0; e < KT / 32; ++e) {
                        const int u = e * 32 + lane, k = it.base + t * KT + u * run;
                        page[e] = more && !none && u < runs && k < it.hi && k + run > it.lo
                                      ? __ldg(a.c.page_table + it.s * a.c.table_stride + block_of(k)) : INT32_MIN;
                        if (e * 32 + 32 >= runs) break;
                    }
                };
                bool have = false, look = false;
                uint32_t cur = 0;  // the tile whose copies come next
                int g = 0, pos_in[KT / 32], pg[KT / 32];
                while (ok) {
                    uint32_t at = 0;
                    bool mix = false, flush = false;
                    do {  // on to this warp's next tile; not to an item that is not announced before what is held back is issued
                        flush = have && t + 1 >= it.t1 && !__all_sync(kAll, mbar_test(&next_full[round % kNext], (round / kNext) & 1));
                        if (flush) break;
                        advance();
                        if (!more || none) break;
                        if (fresh) bounds();
                        at = kt++;
                        mix = mixed();
                        const uint32_t bit = 1u << (2 * at + 1) % C::Slots;
                        if (mix) lph ^= bit;
                        was_look = (was_look & ~bit) | (mix ? bit : 0u);
                    } while ((at & 1) != odd);
                    if (!flush) fetch();
                    if (have) {
#pragma unroll
                        for (int kv = 0; kv < 2; ++kv) {
                            const uint32_t n = 2 * cur + kv, s = n % C::Slots;
                            if (n >= C::Slots)
                                ok = ok && __all_sync(kAll, !abort_sh && mbar_wait_bounded(&empty[s], ((n / C::Slots) - 1) & 1, limit));
                            if (!ok) continue;
                            uint64_t *bar = kv && look ? &landed[s] : &full[s];
                            if (lane == 0) mbar_expect_tx(bar, C::TileB);
                            __syncwarp();
#pragma unroll
                            for (int e = 0; e < KT / 32; ++e) {
                                if (e * 32 >= runs) break;
                                if (lane < mine) {
                                    const uint32_t d = ring + s * C::TileB + (e * 32 + lane) * run * 128;
#pragma unroll
                                    for (int h = 0; h < C::Halves; ++h)
                                        tma_load_4d(d + h * (KT * 128), kv ? &tv : &tk, 64 * h, pos_in[e], g, pg[e], bar);
                                }
                            }
                            issued = n + 1;
                        }
                    }
                    have = more && !none && !flush;
                    if (!more || !ok) break;
                    if (none || flush) continue;
                    const int kb = it.base + t * KT;
                    cur = at, look = mix, g = it.g;
#pragma unroll
                    for (int e = 0; e < KT / 32; ++e) {
                        if (e * 32 >= runs) break;
                        const int k = kb + (e * 32 + lane) * run;
                        const bool in = page[e] >= 0 && page[e] < a.kv.n_pages;
                        if (!in && page[e] != INT32_MIN) set_status(a.c.status, ALTXS_ST_BAD_POS);
                        pos_in[e] = k - block_of(k) * P;
                        pg[e] = in ? page[e] : max(a.kv.n_pages, 1);
                        // which positions exist, for the softmax (what is outside [lo, hi) no row sees)
                        const uint32_t seen = __ballot_sync(kAll, in);
                        if (run >= 4) {
                            if (lane < mine)
                                for (int i = 0; i < run / 4; ++i) kmask[cur % C::Ring][(e * 32 + lane) * (run / 4) + i] = in ? 15 : 0;
                        } else if (lane % 4 == 0) {
                            kmask[cur % C::Ring][e * 8 + lane / 4] = (uint8_t)((seen >> lane) & 15);
                        }
                    }
                    __syncwarp();
                }
                // every copy of this warp has landed before the block can exit: those that are the last in their slots
                const uint32_t end = ok ? 2 * kt : issued;
                for (uint32_t i = end > C::Slots ? end - C::Slots : 0; i < issued; ++i) {
                    const uint32_t s = i % C::Slots;
                    if ((i >> 1 & 1) != odd) continue;
                    if ((i & 1) && ((was_look >> s) & 1)) mbar_wait_bounded(&landed[s], ((lph >> s) & 1) ^ 1, kWaitLimit);
                    else mbar_wait_bounded(&full[s], (i / C::Slots) & 1, kWaitLimit);
                }
            } else if (pw == 1) {
                uint32_t me = 0;
                while (ok) {
                    advance();
                    if (!more) break;
                    if (none) continue;
                    const bool ahead = fresh && told == round;  // the next item, once the first tile is on its way
                    if (fresh) {
                        bounds();
                        me = live++ % C::Ring;  // the softmax clears it when the item is done
                    }
                    const uint32_t s = (n + 1) % C::Slots;
                    n += 2;
                    if (mixed()) {
                        ok = __all_sync(kAll, !abort_sh && mbar_wait_bounded(&landed[s], (lph >> s) & 1, limit));
                        if (!ok) break;
                        lph ^= 1u << s;
                        const int kb = it.base + t * KT;
                        bool odd = false;
                        constexpr int NC = HD / 8;
                        for (int i = lane; i < KT * NC; i += 32) {
                            const int r = i / NC, c = i % NC, k = kb + r;
                            if (k >= max(all0, it.lo) && k < min(all1, it.hi)) continue;
                            const uint32_t d = ring + s * C::TileB + (c >> 3) * (KT * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                            uint4 v = make_uint4(0, 0, 0, 0);
                            if (k >= it.lo && k < it.hi) {
                                v = lds16(d);
                                uint32_t *w = reinterpret_cast<uint32_t *>(&v);
                                bool bad = false;
                                constexpr uint32_t X = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
#pragma unroll
                                for (int u = 0; u < 4; ++u) {
                                    if ((w[u] & X) == X) w[u] &= 0xffff0000u, bad = true;
                                    if (((w[u] >> 16) & X) == X) w[u] &= 0xffffu, bad = true;
                                }
                                odd = odd || bad;
                                if (!bad) continue;
                            }
                            sts16(d, v);
                        }
                        if (__any_sync(kAll, odd) && lane == 0) odd_sh[me] = 1;
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&full[s]);
                    }
                    if (ahead) announce();
                }
            }
        } else {
            const int run = f.run, runs = KT / run, issue = runs < 32 ? runs : 32;
            const uint32_t raw = ring + C::Slots * C::TileB;
            if (pw == 0) {  // warp 9: a tile's raw rows, keys to one stage and values to the other, run by run
                int page[KT / 32];
                auto fetch = [&]() {
#pragma unroll
                    for (int e = 0; e < KT / 32; ++e) {
                        const int u = e * 32 + lane, k = it.base + t * KT + u * run;
                        page[e] = more && !none && u < runs && k < it.hi && k + run > it.lo
                                      ? __ldg(a.c.page_table + it.s * a.c.table_stride + block_of(k)) : INT32_MIN;
                        if (e * 32 + 32 >= runs) break;
                    }
                };
                bool have = false;
                int g = 0, pos_in[KT / 32], pg[KT / 32];
                uint32_t sent[2] = {0, 0};
                while (ok) {
                    advance();
                    fetch();
                    if (have) {
#pragma unroll
                        for (int kv = 0; kv < 2; ++kv) {
                            if (ok && sent[kv] > 0)
                                ok = __all_sync(kAll, !abort_sh && mbar_wait_bounded(&raw_empty[kv], (sent[kv] - 1) & 1, limit));
                            if (!ok) continue;
                            ++sent[kv];
                            if (lane == 0) mbar_expect_tx(&raw_full[kv], C::StageB);
                            __syncwarp();
                            const CUtensorMap *map = kv ? &tv : &tk;
#pragma unroll
                            for (int e = 0; e < KT / 32; ++e) {
                                if (e * 32 >= runs) break;
                                if (lane < issue)
                                    tma_load_4d(raw + kv * C::StageB + (e * 32 + lane) * run * HD * 4, map, 0, pos_in[e], g, pg[e], &raw_full[kv]);
                            }
                        }
                        if (!ok) break;
                    }
                    have = more && !none;
                    if (!more) break;
                    if (none) continue;
                    const int kb = it.base + t * KT;
                    g = it.g;
                    const bool ahead = fresh && told == round;
#pragma unroll
                    for (int e = 0; e < KT / 32; ++e) {
                        if (e * 32 >= runs) break;
                        const int k = kb + (e * 32 + lane) * run;
                        const bool in = page[e] >= 0 && page[e] < a.kv.n_pages;
                        if (!in && page[e] != INT32_MIN) set_status(a.c.status, ALTXS_ST_BAD_POS);
                        pos_in[e] = k - block_of(k) * P;
                        pg[e] = in ? page[e] : max(a.kv.n_pages, 1);
                        const uint32_t seen = __ballot_sync(kAll, in);
                        if (run >= 4) {
                            if (lane < issue)
                                for (int i = 0; i < run / 4; ++i) kmask[kt % C::Ring][(e * 32 + lane) * (run / 4) + i] = in ? 15 : 0;
                        } else if (lane % 4 == 0) {
                            kmask[kt % C::Ring][e * 8 + lane / 4] = (uint8_t)((seen >> lane) & 15);
                        }
                    }
                    __syncwarp();
                    ++kt;
                    if (ahead) announce();
                }
                // every copy has landed before the block can exit
#pragma unroll
                for (int kv = 0; kv < 2; ++kv)
                    if (sent[kv] > 0) mbar_wait_bounded(&raw_full[kv], (sent[kv] - 1) & 1, kWaitLimit);
            } else {
                // Units of 2 KB (UR rows), 16-byte pieces; warp cw takes units cw, cw + 6, ..: find the unit's
                // largest magnitude, write the scaled planes.  Where some rows of the block do not see the whole
                // tile, every position has its own exponent: what a row does not see must not set the scale of
                // what it sees.  (Loops are left rolled: with everything unrolled the block's roles miss the
                // instruction cache.)
                constexpr int CR = HD / 4, UR = C::UnitRows, Units = C::Units;
                const int cw = pw - 1;
                uint32_t me = 0;
                while (ok) {
                    advance();
                    if (!more) break;
                    if (none) continue;
                    if (fresh) {
                        bounds();
                        me = live++ % C::Ring;
                        if (lane == 0) odd8_sh[me][cw] = 0;
                    }
                    const int kb = it.base + t * KT;
                    const bool look = kb < all0 || kb + KT > all1, edge = kb < it.lo || kb + KT > it.hi;
#pragma unroll 1
                    for (int kv = 0; kv < 2; ++kv, ++n) {
                        const uint32_t s = n % C::Slots;
                        ok = mbar_wait_bounded(&raw_full[kv], kt & 1, limit);
                        if (n >= C::Slots) ok = ok && mbar_wait_bounded(&empty[s], ((n / C::Slots) - 1) & 1, limit);
                        ok = __all_sync(kAll, ok && !abort_sh);
                        if (!ok) break;
                        const uint32_t stage = raw + kv * C::StageB + lane * 16, dst = ring + s * C::TileB;
#pragma unroll 1
                        for (int un = cw; un < Units; un += C::Converters) {
                            float4 x[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[e] = lds_f4(stage + un * 2048 + e * 512);
                            if (edge) {  // rows outside [lo, hi): whatever the page holds there
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int k = kb + un * UR + (e * 32 + lane) / CR;
                                    if (k < it.lo || k >= it.hi) x[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                                }
                            }
                            float mf = 0.0f;
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                mf = fmaxf(mf, fmaxf(fmaxf(fabsf(x[e].x), fabsf(x[e].y)), fmaxf(fabsf(x[e].z), fabsf(x[e].w))));
                            uint32_t mx = __reduce_max_sync(kAll, __float_as_uint(mf));
                            uint8_t *exps = kv_exp[kt & 1][kv] + un * UR;
                            const int bias = 127 - (kv ? kVal : 14);
                            float scale[4];
                            if (look || mx == 0x7f800000u) {  // finite magnitudes alone; odd values; by row
                                bool odd = false;
                                uint32_t me4[4] = {};
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    float *w = reinterpret_cast<float *>(&x[e]);
#pragma unroll
                                    for (int u = 0; u < 4; ++u) {
                                        me4[e] = max(me4[e], finite_abs(w[u]));
                                        if (kv && look && !isfinite(w[u])) w[u] = 0.0f, odd = true;
                                    }
                                }
                                if (!look) me4[0] = me4[1] = me4[2] = me4[3] = __reduce_max_sync(kAll, max(max(me4[0], me4[1]), max(me4[2], me4[3])));
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
#pragma unroll
                                    for (int d = 1; d < CR; d <<= 1) me4[e] = max(me4[e], __shfl_xor_sync(kAll, me4[e], d));
                                    const int ex = exp_of(me4[e]);
                                    scale[e] = pow2(14 - ex);
                                    if (lane % CR == 0) exps[(e * 32 + lane) / CR] = (uint8_t)(ex + bias);
                                }
                                if (__any_sync(kAll, odd) && lane == 0) odd8_sh[me][cw] = 1;
                            } else {
                                const int ex = exp_of(mx);
                                scale[0] = scale[1] = scale[2] = scale[3] = pow2(14 - ex);
                                if (lane < UR) exps[lane] = (uint8_t)(ex + bias);
                            }
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int q = e * 32 + lane, r = un * UR + q / CR, c4 = q % CR, c = c4 >> 1;
                                uint2 hi, lo;
                                split2(x[e].x * scale[e], x[e].y * scale[e], hi.x, lo.x);
                                split2(x[e].z * scale[e], x[e].w * scale[e], hi.y, lo.y);
                                const uint32_t d = dst + (c >> 3) * (KT * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4) + (c4 & 1) * 8;
                                sts8(d, hi);
                                sts8(d + C::PlaneB, lo);
                            }
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(&raw_empty[kv]);
                            mbar_arrive(&full[s]);
                        }
                    }
                    ++kt;
                }
            }
        }
        if (!ok) abort_sh = 1;
        if (pw == kAnnouncer && lane == 0) {
            // every block draws until it is past the end (after a wait that gave up, here): the last of them resets the count
            while (drawn < total) drawn = (int)gridDim.x + (int)atomicAdd(f.ticket, 1u);
            if (blockIdx.x < total && drawn - (int)gridDim.x == total - 1) *f.ticket = 0;
        }
    } else if (warp == kMmaWarp) {
        // ---- MMA issuer ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::RegP));
        {
            // The whole warp runs the loop and one lane issues, so that the operands stay in uniform
            // registers: an issue from one lane's own control flow costs about 100 clocks each.
            const uint32_t tm = __shfl_sync(kAll, tmem, 0);
            const bool leader = elect_one();
            uint32_t items = 0, pph0 = 0, pph1 = 0;  // items so far; p_full's parity per group
            // keys take slots 0, 2, 4, .. and values 1, 3, 5, .. of the ring's sequence
            uint32_t ks = 0, kph = 0, vs = 1, vph = 0;
            auto step = [](uint32_t &s, uint32_t &ph) {
                s += 2;
                if (s >= C::Slots) s -= C::Slots, ph ^= 1;
            };
            constexpr uint32_t kTileD = C::TileB >> 4, kPlaneD = C::PlaneB >> 4, kQPlaneD = C::QPlaneB >> 4;
            const uint32_t ringk = desc_lo(ring, 16), ringv = desc_lo(ring, KT * 128), q0d = desc_lo(sq, 16);
            bool ok = true;
            for (int round = 0; ok; ++round) {
                Item it;
                announced(round, it);
                if (__shfl_sync(kAll, it.s, 0) < 0) break;
                const int nt = __shfl_sync(kAll, it.t1 - it.t0, 0);
                const bool two = __shfl_sync(kAll, (int)it.two, 0) != 0;
                if (nt == 0) continue;
                ok = __all_sync(kAll, mbar_wait_bounded(&q_full, items & 1, limit));
                ++items;
                const int T2 = two ? 2 * nt : nt;  // jobs: (group t & 1, tile t / 2 or t)
                auto issue_pv = [&](int i, uint32_t more) {  // O_i += P V
                    const uint32_t vb = ringv + vs * kTileD, d = tm + C::ColO + HD * i, p = tm + C::ColS + KT * i;
                    if constexpr (F32) {
                        const uint32_t dl = d + (C::Apart ? 2 * HD : 0);
#pragma unroll
                        for (int kk = 0; kk < KT / 16; ++kk) {
                            mma_ts(dl, p + 8 * kk, vb + kPlaneD + kk * 128, idesc<T>(HD, 1), kk ? 1u : more);
                            mma_ts(dl, p + KT / 2 + 8 * kk, vb + kk * 128, idesc<T>(HD, 1), 1u);
                        }
                    }
#pragma unroll
                    for (int kk = 0; kk < KT / 16; ++kk)
                        mma_ts(d, p + 8 * kk, vb + kk * 128, idesc<T>(HD, 1), kk || (F32 && !C::Apart) ? 1u : more);
                };
                auto issue_s = [&](int i) {  // S_i = Q K^T
                    const uint32_t kb = ringk + ks * kTileD, qb = q0d + (two && i ? C::QTileB >> 4 : 0), d = tm + C::ColS + KT * i;
                    // channels 16 kk ..: 32 bytes along a row, 64 channels to a half
                    auto at = [](int kk, int half) { return (uint32_t)((kk >> 2) * (half >> 4) + (kk & 3) * 2); };
                    if constexpr (F32) {  // the small products first, while the sum is small
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk) {
                            mma_ss(d, qb + at(kk, 128 * 128), kb + kPlaneD + at(kk, KT * 128), idesc<T>(KT, 0), kk != 0);
                            mma_ss(d, qb + kQPlaneD + at(kk, 128 * 128), kb + at(kk, KT * 128), idesc<T>(KT, 0), 1u);
                        }
                    }
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk)
                        mma_ss(d, qb + at(kk, 128 * 128), kb + at(kk, KT * 128), idesc<T>(KT, 0), F32 || kk != 0);
                };
                for (int t = 0; t < T2 + 2; ++t) {
                    const int i = t & 1;
                    const bool last = !two || i == 1;  // the tile's last use
                    // The keys of job t are usually there: then its S follows the P V of job t - 2 in one go.
                    // (Where they wait for that P V's slot, it goes first.)
                    bool keys = t < T2 && __all_sync(kAll, mbar_test(&full[ks], kph));
                    if (t >= 2) {
                        ok = mbar_wait_bounded(&full[vs], vph, limit) && mbar_wait_bounded(&p_full[i], i ? pph1 : pph0, limit);
                        ok = __all_sync(kAll, ok && !abort_sh);
                        if (!ok) break;
                        if (i) pph1 ^= 1; else pph0 ^= 1;
                        tc_fence_after();
                        if (leader) {
                            issue_pv(i, t >= 4);
                            if (keys) {
                                issue_s(i);
                                tc_commit(&s_full[i]);
                            }
                            if (t >= T2) tc_commit(&o_done[i]);  // the group's last; before, its next S says as much
                            if (last) tc_commit(&empty[vs]);
                            if (last && keys) tc_commit(&empty[ks]);
                        }
                        if (last) step(vs, vph);
                        if (keys) {
                            if (last) step(ks, kph);
                            continue;
                        }
                    }
                    if (t < T2) {
                        ok = __all_sync(kAll, mbar_wait_bounded(&full[ks], kph, limit));
                        if (!ok) break;
                        tc_fence_after();
                        if (leader) {
                            issue_s(i);
                            tc_commit(&s_full[i]);
                            if (last) tc_commit(&empty[ks]);
                        }
                        if (last) step(ks, kph);
                    }
                }
                ok = __all_sync(kAll, ok && !abort_sh);
            }
            if (!ok) abort_sh = 1;
            if (leader) {
                tc_commit(&drainb);  // every MMA has completed before the block can exit
                mbar_wait_bounded(&drainb, 0, kWaitLimit);
            }
        }
        __syncwarp();
    } else {
        // ---- softmax ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::RegS));
        const int grp = warp >> 2, wq = warp & 3, row = wq * 32 + lane;  // tensor-memory lane `row`
        const uint32_t lanes = (uint32_t)(wq * 32) << 16;
        const uint32_t ts = tmem + lanes + C::ColS + KT * grp, to = tmem + lanes + C::ColO + HD * grp;
        // a negative scale turns the queries round instead; a scale of 0 stays above it (-inf marks the unseen)
        const float c2 = fmaxf(__fmul_rn(fabsf(a.scale), kLog2e), 1.17549435e-38f);
        // fp16 ends at 2^-24.  p carries a power of two (with the lag of m it is 2^15 at most, fp32's with its values'
        // powers 2^14), so that what it loses there is far from the sum: at 2^-32 of the maximum a key, a million
        // keys lose half an fp16 rounding.  (A lag of 2^4 and 2^11 for fp16: long piece 653 us against 648, ragged
        // prompts 278 against 273.)
        constexpr float kBias = F32 ? 6.0f : Half ? 7.0f : 0.0f;
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
        unsigned char *qsm = pm_smem_raw + (sq - raw_s);
        // between an item's last S and the next item's queries their place holds 32 KB of outputs, then 256 (m, l)
        float *stage = reinterpret_cast<float *>(qsm);
        float2 *ml = reinterpret_cast<float2 *>(qsm + C::MlAt);
        uint32_t job = 0, kt = 0, live = 0, done = 0;
        bool ok = true;
        // the item is warp 0's to ask for: the groups meet at barriers, so all of them end at the same one
        int round = 0;
        auto ask = [&]() {
            if (warp == 0) {
                if (round > 0 && lane == 0) mbar_arrive(&next_empty[(round - 1) % kNext]);  // all warps have read it
                const bool got = __all_sync(kAll, mbar_wait_bounded(&next_full[round % kNext], (round / kNext) & 1, limit));
                if (!got) abort_sh = 1;
                if (lane == 0) item_sh = got && !abort_sh;
            }
            ++round;
        };
        ask();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        for (;;) {
            if (!item_sh) break;
            const Item it = next_sh[(round - 1) % kNext];
            if (it.s < 0) break;
            const int nt = it.t1 - it.t0, p0 = it.q.L - it.q.n;
            // At most 64 (32) rows are held 2 (4) times, each copy with its share of a tile's columns, its own
            // (m, l) and O: a thread's chain of exponentials is 2 (4) times shorter.
            const int rep = it.two ? 1 : it.rows > 64 ? 1 : it.rows > 32 || KT < 128 ? 2 : 4, rrows = it.two ? 256 : 128 / rep;
            // this thread's row of the block (rows past the end follow the last one and are not stored) and its part
            const int r_own = it.two ? grp * 128 + row : row & (rrows - 1), part = it.two ? 0 : row / rrows;
            const int r = it.r0 + min(r_own, it.rows - 1), tok = r / f.G, h = it.g * f.G + r - tok * f.G;
            const int pos = p0 + tok;
            float m = -INFINITY, l = 0.0f;
            int qe = 0, ve = -100;                   // fp32: exponents of the row's query and of O's values
            uint32_t njob = 0;                       // jobs of this group in this item
            if (nt > 0) {
                // queries: the lanes share rows (16 bytes each); with shared rows each group takes half of a warp's
                constexpr int NC = HD * (int)sizeof(T) / 16, RPI = 32 / NC;  // pieces of a row, rows per load
                const int64_t qoff = ((int64_t)(it.q.q0 + tok) * a.ldq + (int64_t)h * HD) * (int)sizeof(T);
                const uint32_t qd = sq + (it.two ? grp * C::QTileB : 0);
                // (fp32: both look at all of them, for their exponents)
                const int e0 = it.two ? 0 : grp * 16, e1 = it.two ? 32 : e0 + 16;
                auto query = [&](int e) {  // rows e ..
                    const int64_t o = __shfl_sync(kAll, qoff, e + lane / NC);
                    return __ldg(reinterpret_cast<const uint4 *>(static_cast<const char *>(a.q) + o) + lane % NC);
                };
                if constexpr (F32) {
                    constexpr int B = 8;  // loads in flight
#pragma unroll 1
                    for (int eb = 0; eb < 32; eb += B * RPI) {
                        uint4 v[B];
#pragma unroll
                        for (int i = 0; i < B; ++i) v[i] = query(min(eb + i * RPI, 32 - RPI));
#pragma unroll
                        for (int i = 0; i < B; ++i) {
                            const int e = eb + i * RPI, rr = wq * 32 + e + lane / NC, c = lane % NC;
                            const float x[4] = {__uint_as_float(v[i].x), __uint_as_float(v[i].y), __uint_as_float(v[i].z), __uint_as_float(v[i].w)};
                            uint32_t mq = max(max(finite_abs(x[0]), finite_abs(x[1])), max(finite_abs(x[2]), finite_abs(x[3])));
#pragma unroll
                            for (int d = 1; d < NC; d <<= 1) mq = max(mq, __shfl_xor_sync(kAll, mq, d));
                            const int ex = exp_of(mq);
                            const int own = __shfl_sync(kAll, ex, (lane - e) * NC & 31);
                            if (lane >= e && lane < e + RPI) qe = own;
                            if (e >= e0 && e < e1) {
                                const float s1 = a.scale < 0.0f ? -pow2(14 - ex) : pow2(14 - ex);
                                uint2 hi, lo;
                                split2(x[0] * s1, x[1] * s1, hi.x, lo.x);
                                split2(x[2] * s1, x[3] * s1, hi.y, lo.y);
                                const int c8 = c >> 1;
                                const uint32_t dd = qd + (c8 >> 3) * (128 * 128) + rr * 128 + (((c8 & 7) ^ (rr & 7)) << 4) + (c & 1) * 8;
                                sts8(dd, hi);
                                sts8(dd + C::QPlaneB, lo);
                            }
                        }
                    }
                } else {
#pragma unroll 8
                    for (int e = e0; e < e1; e += RPI) {
                        const int rr = wq * 32 + e + lane / NC, c = lane % NC;
                        uint4 v = query(e);
                        v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
                        sts16(qd + (c >> 3) * (128 * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4), v);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full);
                // positions that all of this warp's rows see: from its first row's and its last row's
                const int ra = it.r0 + min(r_own - lane, it.rows - 1), rb = it.r0 + min(r_own - lane + 31, it.rows - 1);
                int pa = p0 + ra / f.G, pb = p0 + rb / f.G;
                // fp32: from the block's, whose other tiles have an exponent for every position
                if (F32) pa = p0 + it.r0 / f.G, pb = p0 + (it.r0 + it.rows - 1) / f.G;

                auto tile = [&](auto rep_c, int j) -> bool {
                    constexpr int REP = decltype(rep_c)::value, W = KT / REP;  // columns of this thread's share
                    const int c0 = REP > 1 ? part * W : 0;
                    const int kb = it.base + (it.t0 + j) * KT + c0;
                    if (!__all_sync(kAll, !abort_sh && mbar_wait_bounded(&s_full[grp], job & 1, limit))) return false;
                    tc_fence_after();
                    // positions that exist, 4 to a byte; what all the warp's rows see
                    const uint32_t *km = reinterpret_cast<const uint32_t *>(kmask[(kt + j) % C::Ring]) + c0 / 16;
                    uint32_t have = 0x0f0f0f0fu;
#pragma unroll
                    for (int c = 0; c < W / 16; ++c) have &= km[c];
                    const int ka = F32 ? kb - c0 : kb, kw = F32 ? KT : W;  // fp32: the whole tile
                    const bool whole = ka + kw <= pa + 1 && (a.window == 0 || ka > pb - a.window) && have == 0x0f0f0f0fu;
                    const uint8_t *ke = kv_exp[F32 ? (kt + j) & 1 : 0][0] + (F32 ? c0 : 0), *vx = kv_exp[F32 ? (kt + j) & 1 : 0][1] + (F32 ? c0 : 0);
                    const float cq = F32 ? __fmul_rn(c2, pow2(qe - 14)) : c2;
                    uint32_t top = 0;  // fp32: byte of the largest exponent of the values that the row sees
                    if constexpr (F32) {
                        const uint32_t v = 2 * (kt + j) + 1;  // the values' slot: their exponents come with them
                        if (!__all_sync(kAll, mbar_wait_bounded(&full[v % C::Slots], (v / C::Slots) & 1, limit))) return false;
                    }
                    const int first = a.window > 0 ? max(0, pos - a.window + 1 - kb) : 0, last = pos - kb;
                    if (F32 && !whole) {
                        // Scaled, every position by its own, and masked where they lie, 16 columns at a time: such
                        // tiles are few, and unrolled over the registers this came from beyond the instruction
                        // cache each time (encoder windows 98 us where this takes 89).
#pragma unroll 1
                        for (int c = 0; c < W; c += 16) {
                            float y[16];
                            tc_ld16(ts + c0 + c, y);
                            const uint32_t k = km[c / 16];
                            uint32_t see = (k & 15) | (k >> 4 & 0xf0) | (k >> 8 & 0xf00) | (k >> 12 & 0xf000);
                            const int f0 = first - c, l0 = last - c;  // of [0, 15]
                            see &= f0 >= 16 ? 0u : f0 <= 0 ? kAll : kAll << f0;
                            see &= l0 < 0 ? 0u : l0 >= 15 ? kAll : kAll >> (31 - l0);
#pragma unroll
                            for (int u = 0; u < 16; u += 4) {
                                const uint32_t kx = *reinterpret_cast<const uint32_t *>(ke + c + u);
#pragma unroll
                                for (int d = 0; d < 4; ++d) y[u + d] = __fmul_rn(y[u + d], __fmul_rn(cq, pow2_byte(kx, d)));
                                const uint32_t vw = *reinterpret_cast<const uint32_t *>(vx + c + u) &
                                                    (((see >> u & 15) * 0x00204081u & 0x01010101u) * 255u);
                                top = __vmaxu2(top, __vmaxu2(vw & 0x00ff00ffu, vw >> 8 & 0x00ff00ffu));
                            }
                            uint32_t w[16];
#pragma unroll
                            for (int u = 0; u < 16; ++u) w[u] = see & (1u << u) ? __float_as_uint(y[u]) : 0xff800000u;
                            tc_st16(ts + c0 + c, w);
                        }
                        tc_wait_st();
                        top = max(top & 0xffffu, top >> 16);
                    }
                    float x[W];
#pragma unroll
                    for (int c = 0; c < W; c += 32) tc_ld32_nowait(ts + c0 + c, x + c);
                    // columns that share a scale, and their factors to log2 units (fp32: times the row's and the unit's)
                    constexpr int UC = F32 ? C::UnitRows : W, NU = W / UC;
                    float cf[NU];
#pragma unroll
                    for (int i = 0; i < NU; ++i) cf[i] = !F32 ? c2 : whole ? fmaxf(__fmul_rn(cq, pow2_byte(ke[i * UC], 0)), 1.17549435e-38f) : 1.0f;
                    int vt = -100;  // fp32: the values' exponent
                    if constexpr (F32) {
                        if (whole)
#pragma unroll
                            for (int i = 0; i < NU; ++i) top = max(top, (uint32_t)vx[i * UC]);
                        vt = max(vt, (int)top - (127 - kVal));
                        vt = njob == 0 ? vt : max(ve, vt);
                        if (njob == 0) ve = vt;
                    }
                    tc_wait_ld();
#pragma unroll
                    for (int c = 0; c < W; c += 32) tc_tie32(x + c);
                    if (!F32 && !whole) {
#pragma unroll
                        for (int c = 0; c < W; c += 32) {  // bit u: column c + u is seen
                            uint32_t bits = 0;
#pragma unroll
                            for (int d = 0; d < 2; ++d) {
                                const uint32_t k = km[c / 16 + d];
                                bits |= ((k & 15) | (k >> 4 & 0xf0) | (k >> 8 & 0xf00) | (k >> 12 & 0xf000)) << (16 * d);
                            }
                            const int f0 = first - c, l0 = last - c;  // of [0, 31]
                            bits &= f0 >= 32 ? 0u : f0 <= 0 ? kAll : kAll << f0;
                            bits &= l0 < 0 ? 0u : l0 >= 31 ? kAll : kAll >> (31 - l0);
#pragma unroll
                            for (int u = 0; u < 32; ++u)
                                if (!(bits & (1u << u))) x[c + u] = -INFINITY;
                        }
                    }
                    float mx = -INFINITY;
                    if constexpr (F32) {
                        float mu[NU];
#pragma unroll
                        for (int i = 0; i < NU; ++i) {
                            mu[i] = x[i * UC];
#pragma unroll
                            for (int u = 1; u < UC; ++u) mu[i] = fmaxf(mu[i], x[i * UC + u]);
                            mu[i] = mu[i] == -INFINITY ? mu[i] : __fmul_rn(mu[i], cf[i]);
                        }
#pragma unroll
                        for (int i = 0; i < NU; ++i) mx = fmaxf(mx, mu[i]);
                    } else {
                        float mu[8];  // short chains: few warps are there to hide their latency
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            mu[i] = x[i];
#pragma unroll
                            for (int u = i + 8; u < W; u += 8) mu[i] = fmaxf(mu[i], x[u]);
                        }
                        mx = fmaxf(fmaxf(fmaxf(mu[0], mu[1]), fmaxf(mu[2], mu[3])), fmaxf(fmaxf(mu[4], mu[5]), fmaxf(mu[6], mu[7])));
                        mx = mx == -INFINITY ? mx : __fmul_rn(mx, c2);
                    }
                    const bool grow = mx > __fadd_rn(m, kLazy) || (m == -INFINITY && mx > m);
                    if (__any_sync(kAll, grow || (F32 && vt != ve))) {
                        const float mn = grow ? mx : m;
                        float fold = m == -INFINITY ? 0.0f : grow ? ex2(__fsub_rn(m, mn)) : 1.0f;
                        l = __fmul_rn(l, fold);
                        m = mn;
                        if constexpr (F32) {  // O in the units of the larger values
                            fold = __fmul_rn(fold, pow2(max(ve - vt, -126)));
                            ve = vt;
                        }
                        if (njob > 0) {  // this job's S came after the products of the jobs before: O is at rest
#pragma unroll
                            for (int c = 0; c < HD * (C::Apart ? 2 : 1); c += 32) {
                                const uint32_t at = to + (c < HD ? c : c + HD);
                                float v[32];
                                tc_ld32(at, v);
                                uint32_t w[32];
#pragma unroll
                                for (int u = 0; u < 32; ++u) w[u] = __float_as_uint(__fmul_rn(v[u], fold));
                                tc_st32(at, w);
                            }
                        }
                    }
                    const float base = m == -INFINITY ? 0.0f : __fsub_rn(m, kBias);
                    const float2 nb2 = make_float2(-base, -base);
                    const float rs = F32 ? pow2(kVal - vt) : 1.0f;  // fp32: p in the units of its row's values
                    float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                    for (int c = 0; c < W; c += 32) {
                        uint32_t w[16], wl[F32 ? 16 : 1], vw = 0;
#pragma unroll
                        for (int u = 0; u < 32; u += 2) {
                            const int un = (c + u) / UC;
                            const float2 t = fma2(make_float2(x[c + u], x[c + u + 1]), make_float2(cf[un], cf[un]), nb2);
                            float2 e = make_float2(ex2(t.x), ex2(t.y));
                            sum[u / 2 & 1] = add2(sum[u / 2 & 1], e);
                            if constexpr (F32) {
                                if (u % 4 == 0) vw = *reinterpret_cast<const uint32_t *>(vx + c + u);
                                e = mul2(mul2(e, make_float2(rs, rs)), make_float2(pow2_byte(vw, u % 4), pow2_byte(vw, u % 4 + 1)));
                                split2(e.x, e.y, w[u / 2], wl[u / 2]);
                            } else {
                                w[u / 2] = pack2<T>(e.x, e.y);
                            }
                        }
                        tc_st16(ts + (c0 + c) / 2, w);
                        if constexpr (F32) tc_st16(ts + KT / 2 + (c0 + c) / 2, wl);
                    }
                    if constexpr (REP > 1) {  // the other copies' columns
                        const uint32_t z[16] = {};
#pragma unroll
                        for (int d = W; d < KT; d += 32) {
                            const uint32_t at = ts + ((c0 + d) & (KT - 1)) / 2;
                            tc_st16(at, z);
                            if constexpr (F32) tc_st16(at + KT / 2, z);
                        }
                    }
                    const float2 s2 = add2(sum[0], sum[1]);
                    l = __fadd_rn(l, __fadd_rn(s2.x, s2.y));
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[grp]);
                    ++job;
                    ++njob;
                    return true;
                };
                const int j0 = it.two ? 0 : grp, dj = it.two ? 1 : 2;
                if (rep == 1)
                    for (int j = j0; j < nt && ok; j += dj) ok = tile(std::integral_constant<int, 1>{}, j);
                else if (rep == 2)
                    for (int j = j0; j < nt && ok; j += dj) ok = tile(std::integral_constant<int, 2>{}, j);
                else if constexpr (KT == 128)
                    for (int j = j0; j < nt && ok; j += dj) ok = tile(std::integral_constant<int, 4>{}, j);
                kt += nt;
                if (ok && njob > 0) {  // the group's last products
                    ok = __all_sync(kAll, mbar_wait_bounded(&o_done[grp], done & 1, limit));
                    ++done;
                    tc_fence_after();
                }
            }
            if (!ok) abort_sh = 1;
            // ---- the item's rows: the sets that share a row (its copies, both groups) are joined in order ----
            const int sets = it.two ? 1 : 2 * rep, set = it.two ? 0 : grp * rep + part;
            const int slot = set * rrows + r_own;  // 0 .. 255
            asm volatile("bar.sync 1, 256;" ::: "memory");  // no S is left to read the queries
            ml[slot] = make_float2(m, l);
            asm volatile("bar.sync 1, 256;" ::: "memory");
            float M = m, lt = l;
            if (sets > 1) {
                M = -INFINITY, lt = 0.0f;
                for (int s = 0; s < sets; ++s) M = fmaxf(M, ml[s * rrows + r_own].x);
                for (int s = 0; s < sets; ++s) {
                    const float2 v = ml[s * rrows + r_own];
                    lt = __fmaf_rn(v.y, v.x == -INFINITY ? 0.0f : ex2(__fsub_rn(v.x, M)), lt);
                }
            }
            const bool fin = it.nsplit == 1, room = it.slot + it.nsplit <= f.max_slots;
            float wgt = m == -INFINITY ? 0.0f : ex2(__fsub_rn(m, M));
            if (m == M) wgt = m == -INFINITY ? 0.0f : 1.0f;
            if (fin) wgt = __fmul_rn(wgt, M == -INFINITY ? 0.0f : __frcp_rn(lt));
            if constexpr (F32) wgt = __fmul_rn(__fmul_rn(wgt, pow2(ve)), pow2(-14));
            bool odd = false;
            if (nt > 0) {
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < C::Converters; ++e) odd = odd || odd8_sh[live % C::Ring][e] != 0;
                } else {
                    odd = odd_sh[live % C::Ring] != 0;
                }
            }
            const bool whole_ok = !abort_sh;
            float *pp = f.part + (int64_t)(it.slot + it.split) * f.part_rows * (HD + 2);
            const int64_t ooff = (int64_t)(it.q.q0 + tok) * a.ldo + (int64_t)h * HD;
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                float v[32];
                if (njob > 0) {
                    tc_ld32(to + c, v);
                    if constexpr (C::Apart) {  // large and small products
                        float u[32];
                        tc_ld32(to + 2 * HD + c, u);
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __fadd_rn(v[i], u[i]);
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __fmul_rn(v[i], wgt);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)  // 128-byte rows, swizzled like the tiles
                    *reinterpret_cast<float4 *>(stage + slot * 32 + ((i ^ (slot & 7)) << 2)) =
                        make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                // Rows of one set are the warp's own; shared ones meet in the block.  Then four lanes a row, eight
                // channels each.
                if (it.two) __syncwarp();
                else asm volatile("bar.sync 1, 256;" ::: "memory");
                const int rend = it.two ? min(it.rows, (warp + 1) * 32) : min(rrows, it.rows), step = it.two ? 8 : 64;
#pragma unroll 1
                for (int rq = it.two ? warp * 32 : warp * 8; rq < rend; rq += step) {
                    const int ro = rq + (lane >> 2), q = (lane & 3) * 2, ch = c + 4 * q;
                    float y[8] = {};
#pragma unroll 2
                    for (int s = 0; s < sets; ++s) {
                        const int at = s * rrows + ro;
#pragma unroll
                        for (int d = 0; d < 2; ++d) {
                            const float4 u = *reinterpret_cast<const float4 *>(stage + (at & 255) * 32 + (((q + d) ^ (at & 7)) << 2));
                            y[4 * d] = __fadd_rn(y[4 * d], u.x), y[4 * d + 1] = __fadd_rn(y[4 * d + 1], u.y);
                            y[4 * d + 2] = __fadd_rn(y[4 * d + 2], u.z), y[4 * d + 3] = __fadd_rn(y[4 * d + 3], u.w);
                        }
                    }
                    // the row's output: this warp's lanes hold its rows' places, else it is worked out again
                    int64_t o = __shfl_sync(kAll, ooff, ro & 31);
                    if (!it.two) {
                        const int rr = it.r0 + ro, tk = rr / f.G;
                        o = (int64_t)(it.q.q0 + tk) * a.ldo + (int64_t)(it.g * f.G + rr - tk * f.G) * HD;
                    }
                    if (ro >= rend || !whole_ok) continue;
                    if (odd) {  // what is not finite replaces the sum that it was kept out of
#pragma unroll 1
                        for (int e = 0; e < 8; ++e) {
                            const float t = odd_term<T>(a, it.s, it.g, p0 + (it.r0 + ro) / f.G, max(it.lo, it.base + it.t0 * KT), it.base + it.t1 * KT, ch + e);
#pragma unroll
                            for (int d = 0; d < 8; ++d)
                                if (d == e && t != 0.0f) y[d] = t;
                        }
                    }
                    if (fin) {
                        store8<T>(static_cast<T *>(a.out) + o + ch, y);
                    } else if (room) {
                        __stcg(reinterpret_cast<float4 *>(pp + (int64_t)ro * HD + ch), make_float4(y[0], y[1], y[2], y[3]));
                        __stcg(reinterpret_cast<float4 *>(pp + (int64_t)ro * HD + ch + 4), make_float4(y[4], y[5], y[6], y[7]));
                    }
                }
                if (it.two) __syncwarp();
                else asm volatile("bar.sync 1, 256;" ::: "memory");
            }
            if (set == 0 && r_own < it.rows && whole_ok) {
                if (fin) {
                    if (a.lse) a.lse[(int64_t)h * a.c.n_tokens + it.q.q0 + tok] = lt == 0.0f ? -INFINITY : __fadd_rn(M, __fsub_rn(log2f(lt), kBias));
                } else if (room) {
                    __stcg(reinterpret_cast<float2 *>(pp + (int64_t)HD * f.part_rows) + r_own, make_float2(M, lt));
                } else if (r_own == 0) {  // the lengths are above their bounds
                    set_status(a.c.status, ALTXS_ST_BAD_POS);
                }
            }
            if (it.nsplit > 1) {  // the same barriers on every path
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (tid == 0) {
                    __threadfence();  // the block's rows are ordered before its arrival
                    last_sh = 0;
                    if (room) {
                        uint32_t *cnt = f.cnt + it.slot;
                        last_sh = atomicAdd(cnt, 1u) == (uint32_t)it.nsplit - 1;
                        if (last_sh) *cnt = 0;
                    }
                    __threadfence();
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (last_sh) {  // join the splits in order: their weights by row, then four channels a thread
                    const int64_t ps = (int64_t)f.part_rows * (HD + 2);
                    const float *p = f.part + it.slot * ps;
                    const int n4 = (it.nsplit + 3) & ~3;
                    float *wt = stage;  // [n4][256]
                    if (tid < it.rows) {
                        const float *q = p + (int64_t)HD * f.part_rows + 2 * tid;
                        float Mr = -INFINITY, ls = 0.0f;
#pragma unroll 4
                        for (int t = 0; t < it.nsplit; ++t) Mr = fmaxf(Mr, __ldcg(q + t * ps));
#pragma unroll 4
                        for (int t = 0; t < it.nsplit; ++t) {
                            const float2 v = __ldcg(reinterpret_cast<const float2 *>(q + t * ps));
                            const float w = v.x == -INFINITY ? 0.0f : ex2(__fsub_rn(v.x, Mr));
                            ls = __fmaf_rn(v.y, w, ls);
                            wt[t * 256 + tid] = w;
                        }
                        const float inv = Mr == -INFINITY ? 0.0f : __frcp_rn(ls);
                        for (int t = 0; t < n4; ++t) wt[t * 256 + tid] = t < it.nsplit ? __fmul_rn(wt[t * 256 + tid], inv) : 0.0f;
                        const int rr = it.r0 + tid, tk = rr / f.G;
                        if (a.lse)
                            a.lse[(int64_t)(it.g * f.G + rr - tk * f.G) * a.c.n_tokens + it.q.q0 + tk] =
                                ls == 0.0f ? -INFINITY : __fadd_rn(Mr, __fsub_rn(log2f(ls), kBias));
                    }
                    asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll 2
                    for (int i = tid; i < it.rows * (HD / 4); i += 256) {
                        const int ro = i / (HD / 4), c = i % (HD / 4) * 4;
                        const float *q = p + (int64_t)ro * HD + c;
                        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        for (int t = 0; t < n4; t += 4) {
                            float4 u[4];
#pragma unroll
                            for (int d = 0; d < 4; ++d) u[d] = __ldcg(reinterpret_cast<const float4 *>(q + min(t + d, it.nsplit - 1) * ps));
#pragma unroll
                            for (int d = 0; d < 4; ++d) {
                                const float w = wt[(t + d) * 256 + ro];
                                y.x = __fmaf_rn(u[d].x, w, y.x), y.y = __fmaf_rn(u[d].y, w, y.y);
                                y.z = __fmaf_rn(u[d].z, w, y.z), y.w = __fmaf_rn(u[d].w, w, y.w);
                            }
                        }
                        const int rr = it.r0 + ro, tk = rr / f.G;
                        T *yp = static_cast<T *>(a.out) + (int64_t)(it.q.q0 + tk) * a.ldo + (int64_t)(it.g * f.G + rr - tk * f.G) * HD + c;
                        if constexpr (F32) *reinterpret_cast<float4 *>(yp) = y;
                        else *reinterpret_cast<uint2 *>(yp) = make_uint2(pack2<T>(y.x, y.y), pack2<T>(y.z, y.w));
                    }
                }
            }
            // the next item's queries overwrite the staged outputs, and its first products O
            ask();
            tc_fence_before();
            asm volatile("bar.sync 1, 256;" ::: "memory");
            tc_fence_after();
            if (nt > 0) {
                if (!F32 && tid == 0) odd_sh[live % C::Ring] = 0;
                ++live;
            }
        }
        if (tid == 0) {  // in a workspace left by a call that gave up, splits may have been joined early
            if (abort_sh) *f.spoilt = 1;
            if (abort_sh || (blockIdx.x == 0 && __ldcg(f.spoilt) != 0)) set_status(a.c.status, ALTXS_ST_TIMEOUT);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// [pages][heads][positions][channels] of a pool as it lies, boxes of `run` positions x 64 channels (fp32: all)
bool pool_map(CUtensorMap *m, const altxs_paged_kv &kv, void *pool, int run) {
    const auto enc = encoder();
    if (!enc) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)kv.head_dim, (cuuint64_t)kv.page_size, (cuuint64_t)kv.n_kv_heads,
                                (cuuint64_t)std::max(kv.n_pages, 1)};
    const bool f32 = kv.dtype == ALTXS_F32;
    const cuuint64_t b = f32 ? 4 : 2;
    // the stride over a single page is never taken: any valid one will do
    const cuuint64_t strides[3] = {(cuuint64_t)kv.token_stride * b, (cuuint64_t)kv.head_stride * b,
                                   kv.n_pages > 1 ? (cuuint64_t)kv.page_stride * b : 16};
    const cuuint32_t box[4] = {f32 ? (cuuint32_t)kv.head_dim : 64, (cuuint32_t)run, 1, 1}, es[4] = {1, 1, 1, 1};
    return enc(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : kv.dtype == ALTXS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
               4, pool, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, f32 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD>
int launch(const ManyArgs &f, unsigned grid, cudaStream_t st) {
    CUtensorMap tk{}, tv{};
    if ((!pool_map(&tk, f.a.kv, f.a.kv.k, f.run) || !pool_map(&tv, f.a.kv, f.a.kv.v, f.run))) return ALTXS_ECUDA;
    static std::atomic<uint64_t> set{0};  // devices whose shared-memory limit is raised
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return ALTXS_ECUDA;
    if (dev >= 64 || !((set.load() >> dev) & 1)) {
        if (cudaFuncSetAttribute(k_paged_many<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tc<T, HD>::Smem) != cudaSuccess)
            return ALTXS_ECUDA;
        if (dev < 64) set.fetch_or(1ull << dev);
    }
    ALTXS_LAUNCH(kKPaged, st, k_paged_many<T, HD><<<grid, Tc<T, HD>::Threads, Tc<T, HD>::Smem, st>>>(f, tk, tv));
    return ALTXS_OK;
}
template <typename T>
int launch(const ManyArgs &f, unsigned grid, cudaStream_t st) {
    const int hd = f.a.kv.head_dim;
    return hd == 32 ? launch<T, 32>(f, grid, st) : hd == 64 ? launch<T, 64>(f, grid, st) : launch<T, 128>(f, grid, st);
}

}  // namespace

ManyPlan paged_many_plan(const altxs_paged_kv &kv, const altxs_chunks &c, int H, int window) {
    ManyPlan p{};
    const int G = H / kv.n_kv_heads;
    const int rows = block_rows(kv.dtype, kv.head_dim);
    const int64_t blocks = (int64_t)c.n_tokens * G / rows + c.n_seqs;
    const int64_t keys = window > 0 ? std::min<int64_t>(c.max_kv, (int64_t)window + rows) : c.max_kv;
    const int kt = tile_keys(kv.dtype, kv.head_dim);
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kMostSplits, tiles_of((int)keys, kt) / 8));
    p.items = blocks * kv.n_kv_heads * most;
    p.rows = (int64_t)c.max_new * G <= 128 ? 128 : rows;
    if (most > 1) {  // one per item of the last, partly filled wave of a sequence that is cut
        const int64_t nt = tiles_of((int)keys, kt), pairs = ((int64_t)std::max(c.max_new, 1) * G + rows - 1) / rows * kv.n_kv_heads;
        const int64_t each = std::min<int64_t>({(int64_t)most_waves(nt) * kSms, std::min<int64_t>(pairs, kSms - 1) * most, kMostItems});
        // a sequence is cut from 16 tiles on
        const int64_t seqs = c.total_kv > 0 ? std::min<int64_t>(c.n_seqs, c.total_kv / (15 * kt)) : c.n_seqs;
        p.slots = std::min(p.items, seqs * each);
    }
    p.slot_bytes = (int64_t)p.rows * (kv.head_dim + 2) * 4;
    return p;
}

int launch_paged_many(const PagedAttnArgs &a, const ManyPlan &p, int min_rows, uint32_t *spoilt, uint32_t *cnt,
                      float *part, int sms, cudaStream_t st) {
    const int run = std::min(tile_keys(a.kv.dtype, a.kv.head_dim), a.kv.page_size & -a.kv.page_size);
    const ManyArgs f{a, a.H / a.kv.n_kv_heads, min_rows, run < 4 ? 1 : run, p.slots, spoilt, cnt + 1, cnt, part, p.rows};
    const unsigned grid = (unsigned)std::min<int64_t>(p.items, sms);
    if (a.kv.dtype == ALTXS_F32) return launch<float>(f, grid, st);
    return a.kv.dtype == ALTXS_BF16 ? launch<__nv_bfloat16>(f, grid, st) : launch<__half>(f, grid, st);
}

int set_wait_limit_paged(uint32_t limit) {
    return cudaMemcpyToSymbol(g_wait_limit, &limit, sizeof(limit)) == cudaSuccess ? ALTXS_OK : ALTXS_ECUDA;
}

}  // namespace altxs
