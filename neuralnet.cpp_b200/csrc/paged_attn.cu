// paged_attn.cu — attention of one new token per sequence over a paged key-value cache.
#include <cooperative_groups.h>
#include <math.h>

#include "device_math.cuh"
#include "paged.cuh"

namespace nnb {

struct DecodeArgs {
    const void* q;
    long long q_stride;
    int n_head, group;
    float scale;
    void* out;
    float* lse;
};

__device__ __forceinline__ float2 load_pair(const float* p) { return make_float2(p[0], p[1]); }
__device__ __forceinline__ float2 load_pair(const __nv_bfloat16* p) { return make_float2(__bfloat162float(p[0]), __bfloat162float(p[1])); }
__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ float load_one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_one(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_one(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// ------------------------------------------------------------------------------------------------ division of the work
// A CTA's four warps take wh (1 or 2) KV heads at a time, wp = 4 / wh warps each: with two, fewer warps have to be joined at
// an item's end.  An item is (sequence, wh KV heads, slab of query heads); its positions form units of 16 wp (8 wp for wide
// f32 rows), a tile for each warp.  The work is cut evenly whatever the lengths: an item costs its units and ITEM_COST more
// for its beginning and end (measured with 0 / 1 / 2 / 4: 86 / 73 / 67 / 67 us for 128 sequences of 0..640 positions), and
// each worker (one CTA; at most as many as the whole cost) takes an even share of the batch in order.  A worker finishes the
// items that lie inside its range; of an item that several workers share each leaves a partial softmax (maximum, sum,
// weighted values) that paged_join_kernel folds in order.  A worker has at most two partial items: slot 0 is one that began
// in an earlier worker, slot 1 one that begins here and goes on in the next.
//
// A short call (few items over a short table) is dealt out differently, to a cluster of CLUSTER CTAs per item, which share its
// tiles evenly and join through distributed shared memory: one launch less, and no way through global memory.  Measured with
// clusters / with workers and a join, 20 query heads on 5 KV heads of 128: 6.8 / 9.7 us at 300 positions, 7.8 / 10.1 at 700,
// 10.5 / 12.3 at 2000; 16 KV heads without groups meet at 2000 (14.2 us).
constexpr int CLUSTER = 8, SHORT_CALL = 2048;  // the longest table of a short call, in positions
constexpr int LONG_CALL = 96;  // units per worker from which on a call has a second set of workers
constexpr int MAX_CTAS_PER_SM = 4, MAX_WORKERS = MAX_CTAS_PER_SM * 3 / 2 /* per SM, both sets */, MAX_UNIT = 64, ITEM_COST = 2;

struct DecodeWs {
    int2* desc;      // (workers): the split item that begins in a worker and its last worker; item -1: none
    float* ml;       // (workers, 2, wh, rows, 2): maximum (log2 domain) and sum of a partial softmax
    float* o;        // (workers, 2, wh, rows, dkm): its weighted values
    float* lse2;     // (n_seq, n_head): log2 of the sum of exp, for the weights; or NULL
    float* scores;   // (n_seq, n_head, score_stride): scores in the log2 domain, for the weights; or NULL
    long long score_stride;
    int wh, wide;    // wide: workers of the first set
    int clusters;    // a short call
    int rows, dkm;   // query heads of an item per KV head, and the pitch of the partial results
    int slab_groups; // items per (sequence, wh KV heads): larger groups of query heads than a pass serves are cut
};

// an item's place in the batch and a tile of it
struct UnitIter {
    int seq, hs, tile, n, tiles;
};

__device__ __forceinline__ void load_seq(UnitIter& it, const PagedView& c, const SeqView& s, int unit, int* flags)
{
    it.n = paged_len(c, s, it.seq, flags);
    it.tiles = (it.n + unit - 1) / unit;
}
// to the first tile of the next item
__device__ __forceinline__ void next_item(UnitIter& it, const PagedView& c, const SeqView& s, int unit, int items_per_seq, int* flags)
{
    it.tile = 0;
    if (++it.hs < items_per_seq) return;
    it.hs = 0;
    do {
        ++it.seq;
        load_seq(it, c, s, unit, flags);
    } while (it.tiles == 0 && it.seq + 1 < s.n_seq);
}

// How the cost is dealt out.  The SMs of some GPCs get up to a fifth less of the memory's rate than others, so a long call's
// last tenth goes to a second set of workers, half as many, which start wherever one of the first set ends (64 sequences of
// 1000..8192 positions: 213 us without, 198 us with; with as many as the first set 200 us, with the last 15 % 203 us).
struct Deal {
    long long units, head;  // the whole, and what the first `wide` workers share evenly
    int wide, rest;         // the other `rest` workers share what is left
    __device__ __forceinline__ long long start(int w) const
    {
        return w <= wide ? head * w / wide : head + (units - head) * (w - wide) / rest;
    }
    // the worker that has position u: the last that starts at u or before
    __device__ __forceinline__ int worker_of(long long u) const
    {
        return u < head ? (int)(((u + 1) * wide - 1) / head) : wide + (int)(((u - head + 1) * rest - 1) / (units - head));
    }
};

// the same for a short call: this CTA's tiles of its cluster's item
__device__ __forceinline__ bool find_tiles(const PagedView& c, const SeqView& s, int unit, int items_per_seq, UnitIter& it, long long& left, int* flags)
{
    const int item = blockIdx.x / CLUSTER, rank = blockIdx.x % CLUSTER;
    it.seq = item / items_per_seq;
    it.hs = item % items_per_seq;
    load_seq(it, c, s, unit, flags);
    it.tile = it.tiles * rank / CLUSTER;
    left = it.tiles * (rank + 1) / CLUSTER - it.tile;
    return left > 0;
}

// Called by all 128 threads: this worker's range of the cost and the place of its first unit; false if it has none.
__device__ __forceinline__ bool find_work(const PagedView& c, const SeqView& s, int unit, int items_per_seq, const DecodeWs& ws, UnitIter& it, long long& u0, long long& u1,
                                          Deal& deal, int* flags)
{
    __shared__ long long warp_sum[4], place;
    __shared__ int place_seq, place_n;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (s.n_seq + 127) / 128, first = min(s.n_seq, tid * per), last = min(s.n_seq, first + per);
    int n_seen = 0;  // the length that was read last: the only one where each thread has one sequence
    auto cost = [&](int i) {
        n_seen = paged_len(c, s, i, flags);
        return n_seen ? (n_seen + unit - 1) / unit + ITEM_COST : 0;
    };
    long long mine = 0;
    for (int i = first; i < last; ++i) mine += cost(i);
    mine *= items_per_seq;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    long long base = 0;
    deal.units = 0;
    for (int i = 0; i < 4; ++i) {
        if (i < warp) base += warp_sum[i];
        deal.units += warp_sum[i];
    }
    deal.wide = (int)min((long long)ws.wide, deal.units);
    deal.rest = deal.units >= (long long)LONG_CALL * ws.wide ? gridDim.x - ws.wide : 0;
    deal.head = deal.rest ? deal.units * 9 / 10 : deal.units;
    if ((int)blockIdx.x >= deal.wide + deal.rest) return false;
    u0 = deal.start(blockIdx.x);
    u1 = deal.start(blockIdx.x + 1);
    base += incl - mine;
    if (u0 >= base && u0 < base + mine) {
        int i = first;
        long long left = u0 - base;
        if (per > 1)
            for (;; ++i) {
                const long long n = (long long)cost(i) * items_per_seq;
                if (left < n || i + 1 == last) break;
                left -= n;
            }
        place_seq = i;
        place_n = n_seen;
        place = left;
    }
    __syncthreads();
    it.seq = place_seq;
    it.n = place_n;
    it.tiles = (it.n + unit - 1) / unit;
    it.hs = (int)(place / (it.tiles + ITEM_COST));
    it.tile = (int)(place % (it.tiles + ITEM_COST));
    if (it.tile >= it.tiles) {  // the range begins in what the end of an item costs
        u0 += it.tiles + ITEM_COST - it.tile;
        if (u0 >= u1) return false;
        next_item(it, c, s, unit, items_per_seq, flags);
    }
    return true;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void* p)
{
    const uint32_t a = (uint32_t)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], const void* p)
{
    const uint32_t a = (uint32_t)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with nothing to add to
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// two f32 operations in one instruction
__device__ __forceinline__ unsigned long long two(float x, float y)
{
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b)
{
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(two(x, y)), "l"(two(a, b)));
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(x), "=f"(y) : "l"(r));
}
// (x, y) += (a, b) * (p, q)
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float p, float q)
{
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(two(a, b)), "l"(two(p, q)), "l"(two(x, y)));
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(x), "=f"(y) : "l"(r));
}
__device__ __forceinline__ uint32_t pack_rn(float lo, float hi)
{
    const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&x);
}
// the leading 8 bits of two non-negative numbers as a bf16 pair; what is left of them stays in x, y (exactly)
__device__ __forceinline__ uint32_t take_top(float& x, float& y)
{
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    x = __fsub_rn(x, __uint_as_float(a & 0xffff0000u));
    y = __fsub_rn(y, __uint_as_float(b & 0xffff0000u));
    return __byte_perm(a, b, 0x7632);
}
// 2^x for x <= 0 (results below the normal range are 0)
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp16_zfill(void* smem, const void* gmem, bool valid)
{
    const uint32_t sa = (uint32_t)__cvta_generic_to_shared(smem);
    const int sz = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(sa), "l"(gmem), "r"(sz) : "memory");
}

// the queries of the item that the issuing side has come to, into L1: they are read NST units later
template <typename TQ>
__device__ __forceinline__ void prefetch_queries(const PagedView& c, const DecodeArgs& a, const DecodeWs& ws, int seq, int hk, int row0)
{
    const TQ* q = (const TQ*)a.q + (long long)seq * a.q_stride + (long long)(hk * a.group + row0) * c.dk;
    const int bytes = min(ws.rows, a.group - row0) * c.dk * (int)sizeof(TQ);
    for (int b = (threadIdx.x & 31) * 128; b < bytes; b += 32 * 128) asm volatile("prefetch.global.L1 [%0];\n" ::"l"((const char*)q + b));
}

// Folds the results that the wp warps of a KV head have parked (rows of STRIDE floats, then maximum and sum per row; warps
// warp_stride floats apart) and writes them: outputs if the item is whole, a partial result (to part, part_ml) otherwise.
template <int DKM, int STRIDE, int ROWS, typename TQ>
__device__ __forceinline__ void fold_warps(const float* parked, int warp_stride, int wp, const PagedView& c, const DecodeArgs& a, const DecodeWs& ws,
                                           int seq, int hk, int row0, bool whole, float* part, float* part_ml)
{
    const int rows = min(min(ROWS, ws.rows), a.group - row0), threads = 32 * wp, in_head = (threadIdx.x >> 5) / wp;
    for (int p = threadIdx.x & (threads - 1); p < rows * (DKM / 4); p += threads) {
        const int r = p / (DKM / 4), f = p % (DKM / 4) * 4;
        float top = -INFINITY, sum = 0.0f;
        for (int w = 0; w < wp; ++w) top = fmaxf(top, parked[w * warp_stride + ROWS * STRIDE + 2 * r]);
        const float base = top == -INFINITY ? 0.0f : top;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w = 0; w < wp; ++w) {
            const float2 ml = *reinterpret_cast<const float2*>(parked + w * warp_stride + ROWS * STRIDE + 2 * r);
            const float k = exp2f(ml.x - base);
            const float4 y = *reinterpret_cast<const float4*>(parked + w * warp_stride + r * STRIDE + f);
            sum = fmaf(ml.y, k, sum);
            x.x = fmaf(y.x, k, x.x);
            x.y = fmaf(y.y, k, x.y);
            x.z = fmaf(y.z, k, x.z);
            x.w = fmaf(y.w, k, x.w);
        }
        if (whole) {
            const long long hq = (long long)seq * a.n_head + hk * a.group + row0 + r;
            const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum), v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (f + i < c.dk) store_one((TQ*)a.out + hq * c.dk + f + i, v[i] * inv);
            if (f == 0) {
                const float z = sum == 0.0f ? -INFINITY : top + log2f(sum);
                if (a.lse) a.lse[hq] = z * 0.693147180559945309f;
                if (ws.lse2) ws.lse2[hq] = z;
            }
        } else {
            const int pr = in_head * ws.rows + r;
            *reinterpret_cast<float4*>(part + pr * ws.dkm + f) = x;
            if (f == 0) *reinterpret_cast<float2*>(part_ml + pr * 2) = make_float2(top, sum);
        }
    }
}

// Short calls: a CTA's partial result of its item in shared memory, empty at first: (wh, rows, dkm) values, then (wh, rows)
// maximum and sum.
__device__ __forceinline__ void clear_partial(float* part, const DecodeWs& ws)
{
    float2* ml = reinterpret_cast<float2*>(part + ws.wh * ws.rows * ws.dkm);
    for (int i = threadIdx.x; i < ws.wh * ws.rows; i += 128) ml[i] = make_float2(-INFINITY, 0.0f);
}
// The CTAs of the cluster fold their partial results, each for its share of the values, in the order of their ranks.
template <typename TQ>
__device__ void join_cluster(float* part, const PagedView& c, const DecodeArgs& a, const DecodeWs& ws, int seq, int hs)
{
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int rank = (int)cluster.block_rank(), vecs = ws.dkm / 4;
    float* ml = part + ws.wh * ws.rows * ws.dkm;
    for (int p = rank * 128 + threadIdx.x; p < ws.wh * ws.rows * vecs; p += CLUSTER * 128) {
        const int row = p / vecs, f = (p - row * vecs) * 4;
        const int gi = hs % ws.slab_groups * ws.rows + row % ws.rows, hk = hs / ws.slab_groups * ws.wh + row / ws.rows;
        if (gi >= a.group) continue;
        float2 m[CLUSTER];
        float4 y[CLUSTER];
#pragma unroll
        for (int r = 0; r < CLUSTER; ++r) m[r] = *reinterpret_cast<const float2*>(cluster.map_shared_rank(ml + 2 * row, r));
#pragma unroll
        for (int r = 0; r < CLUSTER; ++r)  // (the values of a CTA without any tile were never written)
            y[r] = m[r].x == -INFINITY ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : *reinterpret_cast<const float4*>(cluster.map_shared_rank(part + row * ws.dkm + f, r));
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int r = 0; r < CLUSTER; ++r) top = fmaxf(top, m[r].x);
        const float base = top == -INFINITY ? 0.0f : top;
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < CLUSTER; ++r) {
            const float k = exp2f(m[r].x - base);
            sum = fmaf(m[r].y, k, sum);
            x[0] = fmaf(y[r].x, k, x[0]);
            x[1] = fmaf(y[r].y, k, x[1]);
            x[2] = fmaf(y[r].z, k, x[2]);
            x[3] = fmaf(y[r].w, k, x[3]);
        }
        const long long hq = (long long)seq * a.n_head + hk * a.group + gi;
        const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (f + i < c.dk) store_one((TQ*)a.out + hq * c.dk + f + i, x[i] * inv);
        if (f == 0) {
            const float z = sum == 0.0f ? -INFINITY : top + log2f(sum);
            if (a.lse) a.lse[hq] = z * 0.693147180559945309f;
            if (ws.lse2) ws.lse2[hq] = z;
        }
    }
    cluster.sync();  // nobody leaves while its shared memory is read
}

// ------------------------------------------------------------------------------------------------ bf16 caches
// Tensor cores multiply bf16, so queries and probabilities enter as bf16 pieces whose sum is the f32 value: two pieces keep 16
// bits (bf16 queries are one), three keep 24 (PREC: f32 queries and outputs).  An m16 tile has room for the pieces of several
// heads, so most come at no further multiplication: the thread that holds row g of an accumulator also holds row g + 8.
//   HEADS 4:  leading pieces in rows 0-3, second in 8-11, third in 4-7 (the lanes 16 away)
//   HEADS 8:  leading in rows 0-7, second in 8-15, third (if any) by a second multiplication
//   HEADS 16: two slabs of the last kind that share the loaded tiles
// KS: 16-feature steps of a row (dk padded with zeros, in shared memory only).
template <int KS, int HEADS, bool PREC>
struct MmaCfg {
    static constexpr int NSLAB = HEADS == 16 ? 2 : 1, DKM = KS * 16, LD = DKM + 8, TK = 16;
    static constexpr bool THIRD = PREC && HEADS > 4;                        // a second multiplication for the third pieces
    static constexpr bool REGQ = KS * NSLAB * (THIRD ? 6 : 4) <= 64;        // query fragments in registers, else in shared memory
    static constexpr int QS = NSLAB * (THIRD ? 24 : 16), QROWS = REGQ ? 0 : QS;
    static constexpr int STAGE = 2 * TK * LD;                               // elements of a warp's key and value tile
    static constexpr int NST = KS <= 8 && HEADS < 16 ? 3 : 2;             // 3 CTAs of 2 stages instead of 2 of 3: 139 us for 96
    static constexpr int CTAS = KS == 4 ? (HEADS == 16 ? 2 : 4) : KS <= 8 ? 2 : 1;
    // a warp's result of an item is parked over the tile that it has just used: rows of PARK floats, then maximum and sum
    static constexpr int ROWS = 8 * NSLAB, PARK = DKM + (NSLAB == 1 ? 8 : 4);
    static_assert((ROWS * PARK + 2 * ROWS) * 4 <= STAGE * 2, "a parked result fits in a stage");
    static constexpr size_t SMEM = (size_t)4 * NST * STAGE * 2 + (size_t)(HEADS == 16 ? 1 : 2) * QROWS * LD * 2;  // queries: for each KV head of the CTA
};

template <int KS, int HEADS, typename TQ>
__global__ void __launch_bounds__(128, MmaCfg<KS, HEADS, sizeof(TQ) == 4>::CTAS)
paged_decode_mma_kernel(const PagedView c, const SeqView s, const DecodeArgs a, const DecodeWs ws, int* flags)
{
    constexpr bool PREC = sizeof(TQ) == 4;
    using C = MmaCfg<KS, HEADS, PREC>;
    constexpr int LD = C::LD, TK = C::TK, NST = C::NST, NSLAB = C::NSLAB, NT = 2 * KS;
    constexpr bool SPREAD = PREC && HEADS == 4;  // the lanes 16 away hold the third pieces of the same head
    // a load instruction covers RPI rows with CHP lanes each (2 KS of them with a 16-byte chunk of the padded row)
    constexpr int CH = 2 * KS, CHP = KS <= 4 ? 8 : KS <= 8 ? 16 : 32, RPI = 32 / CHP;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    __nv_bfloat16* ring = reinterpret_cast<__nv_bfloat16*>(smem_raw) + (size_t)warp * NST * C::STAGE;
    __nv_bfloat16* qs = reinterpret_cast<__nv_bfloat16*>(smem_raw) + (size_t)4 * NST * C::STAGE + (size_t)(warp / (4 / ws.wh)) * C::QROWS * LD;
    float* shared_part = reinterpret_cast<float*>(smem_raw + C::SMEM);  // of a short call
    pdl_wait();
    pdl_launch();
    const int wp = 4 / ws.wh, unit = TK * wp, in_head = warp / wp, items_per_seq = c.heads / ws.wh * ws.slab_groups;
    UnitIter ct;
    long long u_begin, u_end, left;  // left: cost for the computing side
    Deal deal;
    if (ws.clusters) {
        clear_partial(shared_part, ws);
        if (!find_tiles(c, s, unit, items_per_seq, ct, left, flags)) {
            join_cluster<TQ>(shared_part, c, a, ws, ct.seq, ct.hs);
            return;
        }
    } else {
        const bool work = find_work(c, s, unit, items_per_seq, ws, ct, u_begin, u_end, deal, flags);
        if (tid == 0) ws.desc[blockIdx.x] = make_int2(-1, -1);
        if (!work) return;
        left = u_end - u_begin;
    }
    long long to_issue = left;  // for the issuing side, which runs NST units ahead

    const char* kbase = (const char*)c.k;
    const char* vbase = (const char*)c.v;
    const unsigned row_bytes = (unsigned)c.pitch * 2;
    const int my_row = lane / CHP, my_ch = lane % CHP;
    const bool my_live = my_ch < c.pitch / 8;
    const unsigned my_off = my_row * row_bytes + min(my_ch, c.pitch / 8 - 1) * 16;
    // Pages of a multiple of 16 positions: a tile lies in one page and its rows follow one another.  Otherwise each lane
    // looks up the row of one position of the tile.
    const bool whole_tiles = c.page % TK == 0;
    const int my_pos = warp % wp * TK + (whole_tiles ? 0 : lane & 15);
    const int col_step = unit / c.page, slot_step = unit % c.page;
    UnitIter it = ct;
    int col = (it.tile * unit + my_pos) / c.page, slot_in_page = (it.tile * unit + my_pos) % c.page, page_id = -1;
    int head = it.hs / ws.slab_groups * ws.wh + in_head;
    if (warp % wp == 0) prefetch_queries<TQ>(c, a, ws, it.seq, head, it.hs % ws.slab_groups * ws.rows);
    const int32_t* table_row = s.table + (long long)it.seq * s.stride;
    int ahead = it.n - it.tile * unit - my_pos;  // positions of the item from this lane's on
    unsigned long long exist = 0;  // which of the 16 positions of each tile under way exist (a bit each, the oldest tile lowest)
    if (ahead > 0) page_id = table_row[col];
    // The tile's keys are requested as soon as the scores of the one before in this stage are formed, its values (and the
    // commit) after that one's products.
    const char* next_kp = kbase;  // whole tiles: this lane's first chunk; otherwise the row of its position is in next_row
    int next_row = -1, next_lim = 0;
    auto issue_tile = [&](__nv_bfloat16* dst, const char* base, const char* first) {
        if (whole_tiles) {
            if (CH == CHP || my_ch < CH)
#pragma unroll
                for (int i = 0; i < TK / RPI; ++i) {
                    cp16_zfill(dst + i * RPI * LD, first, i * RPI < next_lim);
                    first += RPI * row_bytes;
                }
        } else {
#pragma unroll
            for (int i = 0; i < TK / RPI; ++i) {
                const int src = __shfl_sync(0xffffffffu, next_row, i * RPI + my_row);
                const bool ok = src >= 0 && my_live;
                if (CH == CHP || my_ch < CH) cp16_zfill(dst + i * RPI * LD, base + (ok ? (size_t)(unsigned)src * row_bytes + my_ch * 16 : 0), ok);
            }
        }
    };
    auto issue_keys = [&](int stage, int age) {
        if (to_issue <= 0) return;
        unsigned mask = 0;
        int row = -1;
        if (ahead > 0) {
            if ((unsigned)page_id < (unsigned)c.n_pages)
                row = (page_id * c.heads + head) * c.page + slot_in_page;
            else
                paged_flag(flags, PAGED_BAD_PAGE);
        }
        if (whole_tiles) {
            const int n = row >= 0 ? min(ahead, TK) : 0;
            mask = (1u << n) - 1u;
            // (all 16 rows lie in the page, or in the pool's first for a tile without any: every address is in the pool)
            next_kp = kbase + ((size_t)(unsigned)(n ? row : 0) * row_bytes + my_off);
            next_lim = my_live ? n - my_row : 0;  // row i * RPI + my_row exists: i * RPI < next_lim
        } else {
            mask = __ballot_sync(0xffffffffu, row >= 0) & 0xffffu;
            next_row = row;
        }
        issue_tile(ring + stage * C::STAGE + my_row * LD + my_ch * 8, kbase, next_kp);
        exist |= (unsigned long long)mask << (16 * age);
    };
    auto issue_values = [&](int stage) {
        if (to_issue > 0) {
            issue_tile(ring + stage * C::STAGE + (TK + my_row) * LD + my_ch * 8, vbase, next_kp + (vbase - kbase));
            --to_issue;
            if (++it.tile == it.tiles) to_issue -= ITEM_COST;
            if (to_issue > 0) {
                if (it.tile < it.tiles) {
                    ahead -= unit;
                    col += col_step;
                    slot_in_page += slot_step;
                    if (slot_in_page >= c.page) {
                        slot_in_page -= c.page;
                        ++col;
                    }
                } else {
                    next_item(it, c, s, unit, items_per_seq, flags);
                    head = it.hs / ws.slab_groups * ws.wh + in_head;
                    if (warp % wp == 0) prefetch_queries<TQ>(c, a, ws, it.seq, head, it.hs % ws.slab_groups * ws.rows);
                    table_row = s.table + (long long)it.seq * s.stride;
                    ahead = it.n - my_pos;
                    col = my_pos / c.page;
                    slot_in_page = my_pos % c.page;
                }
                if (ahead > 0) page_id = table_row[col];  // used by the next call
            }
        }
        asm volatile("cp.async.commit_group;\n" ::);
    };
#pragma unroll
    for (int i = 0; i < NST; ++i) {
        issue_keys(i, i);
        issue_values(i);
    }

    const float scale2 = a.scale * 1.44269504088896341f;
    uint32_t qa[C::REGQ ? NSLAB : 1][C::REGQ ? KS : 1][4], qb[C::REGQ && C::THIRD ? NSLAB : 1][C::REGQ && C::THIRD ? KS : 1][2];
    // o[..][0..1]: row g, o[..][2..3]: row g + 8.  With f32 outputs they are added in f32 after every tile: tensor cores truncate
    // their sums, which f32 results cannot afford over a long context.
    float o[NSLAB][NT][4], m[NSLAB], l[NSLAB];
    bool fresh = true, starts_here = false;
    int stage = 0;
    for (;; ) {
        // this warp's KV head and the first query head of its group here
        const int hk = ct.hs / ws.slab_groups * ws.wh + in_head, row0 = (ct.hs % ws.slab_groups) * HEADS;
        if (fresh) {  // a new item: its queries
            fresh = false;
            starts_here = ct.tile == 0;
            if (!C::REGQ) __syncthreads();
#pragma unroll
            for (int sl = 0; sl < NSLAB; ++sl) {
                m[sl] = -INFINITY;
                l[sl] = 0.0f;
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[sl][i][j] = 0.0f;
                const int gi = row0 + (HEADS == 4 ? g & 3 : sl * 8 + g);
                const TQ* q = (const TQ*)a.q + (long long)ct.seq * a.q_stride + (long long)(hk * a.group + gi) * c.dk;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    if (!C::REGQ && (ks & (wp - 1)) != warp % wp) continue;
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const int f = ks * 16 + hf * 8 + 2 * t4;
                        const float2 x = gi < a.group && f < c.dk ? load_pair(q + f) : make_float2(0.0f, 0.0f);
                        uint32_t hi = pack_rn(x.x, x.y), lo = 0, lo2 = 0;
                        if (PREC) {
                            const float r0 = __fsub_rn(x.x, __uint_as_float(hi << 16)), r1 = __fsub_rn(x.y, __uint_as_float(hi & 0xffff0000u));
                            lo = pack_rn(r0, r1);
                            lo2 = pack_rn(__fsub_rn(r0, __uint_as_float(lo << 16)), __fsub_rn(r1, __uint_as_float(lo & 0xffff0000u)));
                        }
                        if (HEADS == 4 && g >= 4) {
                            hi = lo2;
                            lo = 0;
                        }
                        if constexpr (C::REGQ) {
                            qa[sl][ks][2 * hf] = hi;
                            qa[sl][ks][2 * hf + 1] = lo;
                            if constexpr (C::THIRD) qb[sl][ks][hf] = lo2;
                        } else {
                            __nv_bfloat16* dst = qs + (size_t)sl * (C::QS / NSLAB) * LD + f;
                            *reinterpret_cast<uint32_t*>(dst + g * LD) = hi;
                            *reinterpret_cast<uint32_t*>(dst + (8 + g) * LD) = lo;
                            if (C::THIRD) *reinterpret_cast<uint32_t*>(dst + (16 + g) * LD) = lo2;
                        }
                    }
                }
            }
            if (!C::REGQ) __syncthreads();
        }
        asm volatile("cp.async.wait_group %0;\n" ::"n"(NST - 1) : "memory");
        __syncwarp();
        const __nv_bfloat16* kt = ring + stage * C::STAGE;
        const __nv_bfloat16* vt = kt + TK * LD;
        const unsigned live = (unsigned)exist & 0xffffu;
        exist >>= 16;
        // scores of 16 positions: n-tile j holds positions 8 j + 2 t4 + {0, 1} of the tile, of the thread's head
        float x[NSLAB][2][2];
        {
            float acc[NSLAB][2][2][4];  // two sums per n-tile (even and odd steps) halve the chain of dependent multiplications
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t b[4];
                ldsm4(b, kt + ((lane & 7) + 8 * (lane >> 4)) * LD + ks * 16 + 8 * ((lane >> 3) & 1));
#pragma unroll
                for (int sl = 0; sl < NSLAB; ++sl) {
                    uint32_t f[4], f2[2] = {0u, 0u};
                    if constexpr (C::REGQ) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) f[i] = qa[sl][ks][i];
                        if constexpr (C::THIRD) {
                            f2[0] = qb[sl][ks][0];
                            f2[1] = qb[sl][ks][1];
                        }
                    } else {
                        const __nv_bfloat16* src = qs + (size_t)sl * (C::QS / NSLAB) * LD + ks * 16;
                        ldsm4(f, src + ((lane & 7) + 8 * ((lane >> 3) & 1)) * LD + 8 * (lane >> 4));
                        if constexpr (C::THIRD) {
                            f2[0] = *reinterpret_cast<const uint32_t*>(src + (16 + g) * LD + 2 * t4);
                            f2[1] = *reinterpret_cast<const uint32_t*>(src + (16 + g) * LD + 8 + 2 * t4);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float(&d)[4] = acc[sl][j][ks & 1];
                        if (ks < 2)
                            mma16816_first(d, f[0], f[1], f[2], f[3], b[2 * j], b[2 * j + 1]);
                        else
                            mma16816(d, f[0], f[1], f[2], f[3], b[2 * j], b[2 * j + 1]);
                        if constexpr (C::THIRD) mma16816(d, f2[0], 0u, f2[1], 0u, b[2 * j], b[2 * j + 1]);
                    }
                }
            }
#pragma unroll
            for (int sl = 0; sl < NSLAB; ++sl)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float y = __fadd_rn(acc[sl][j][0][i], acc[sl][j][1][i]);
                        if (PREC) y = __fadd_rn(y, __fadd_rn(acc[sl][j][0][2 + i], acc[sl][j][1][2 + i]));
                        if (SPREAD) y = __fadd_rn(y, __shfl_xor_sync(0xffffffffu, y, 16));
                        x[sl][j][i] = __fmul_rn(y, scale2);
                    }
            if (live != 0xffffu)
#pragma unroll
                for (int sl = 0; sl < NSLAB; ++sl)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            if (!((live >> (8 * j + 2 * t4 + i)) & 1u)) x[sl][j][i] = -INFINITY;
        }
        const bool ends = ct.tile + 1 == ct.tiles;
        left -= ends ? 1 + ITEM_COST : 1;
        const bool last = left <= 0, closing = ends || last;  // a closing tile's stage is needed once more
        __syncwarp();
        if (!closing) issue_keys(stage, NST - 1);
        float corr[NSLAB];
        bool moved = false;
#pragma unroll
        for (int sl = 0; sl < NSLAB; ++sl) {
            const int gi = row0 + (HEADS == 4 ? g : sl * 8 + g);
            if (ws.scores && gi < a.group && (HEADS != 4 || g < 4)) {
                float* dst = ws.scores + ((long long)ct.seq * a.n_head + hk * a.group + gi) * ws.score_stride + ct.tile * unit + warp % wp * TK + 2 * t4;
                *reinterpret_cast<float2*>(dst) = make_float2(x[sl][0][0], x[sl][0][1]);
                *reinterpret_cast<float2*>(dst + 8) = make_float2(x[sl][1][0], x[sl][1][1]);
            }
            float top = fmaxf(fmaxf(x[sl][0][0], x[sl][0][1]), fmaxf(x[sl][1][0], x[sl][1][1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(m[sl], fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)));
            const float base = top == -INFINITY ? 0.0f : top;  // nothing seen yet: every exponential is 0
            corr[sl] = exp2_fast(m[sl] - base);
            moved |= top != m[sl];
            m[sl] = top;
            l[sl] *= corr[sl];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    x[sl][j][i] = exp2_fast(x[sl][j][i] - base);
                    l[sl] += x[sl][j][i];
                }
        }
        // o = o * corr + p . v; the sums that stay in the tensor cores are rescaled when a maximum has moved
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int sl = 0; sl < NSLAB; ++sl)
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[sl][i][j] *= corr[sl];
        }
        uint32_t pa[NSLAB][4], pb[NSLAB][2];
#pragma unroll
        for (int sl = 0; sl < NSLAB; ++sl)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float p0 = x[sl][j][0], p1 = x[sl][j][1];
                pa[sl][2 * j] = take_top(p0, p1);
                if constexpr (PREC) {
                    pa[sl][2 * j + 1] = take_top(p0, p1);
                    pb[sl][j] = pack_rn(p0, p1);
                    if (SPREAD && g >= 4) {
                        pa[sl][2 * j] = pb[sl][j];
                        pa[sl][2 * j + 1] = 0u;
                    }
                } else {
                    pa[sl][2 * j + 1] = pack_rn(p0, p1);
                }
            }
#pragma unroll
        for (int np = 0; np < KS; ++np) {
            uint32_t b[4];
            ldsm4_t(b, vt + ((lane & 7) + 8 * ((lane >> 3) & 1)) * LD + np * 16 + 8 * (lane >> 4));
#pragma unroll
            for (int sl = 0; sl < NSLAB; ++sl)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float(&d)[4] = o[sl][2 * np + j];
                    if constexpr (PREC) {
                        float y[4];
                        mma16816_first(y, pa[sl][0], pa[sl][1], pa[sl][2], pa[sl][3], b[2 * j], b[2 * j + 1]);
                        if constexpr (C::THIRD) mma16816(y, pb[sl][0], 0u, pb[sl][1], 0u, b[2 * j], b[2 * j + 1]);
                        add2(d[0], d[1], y[0], y[1]);
                        add2(d[2], d[3], y[2], y[3]);
                    } else {
                        mma16816(d, pa[sl][0], pa[sl][1], pa[sl][2], pa[sl][3], b[2 * j], b[2 * j + 1]);
                    }
                }
        }
        __syncwarp();
        if (closing) {  // fold the four warps' results
            const bool whole = starts_here && ends && !ws.clusters;
            if (tid == 0 && starts_here && !ends && !ws.clusters)
                ws.desc[blockIdx.x] = make_int2(ct.seq * items_per_seq + ct.hs, deal.worker_of(u_end - 1 + (ct.tiles - 1 - ct.tile)));
            float* park = reinterpret_cast<float*>(ring + stage * C::STAGE);
#pragma unroll
            for (int sl = 0; sl < NSLAB; ++sl) {
                float ls = l[sl];
                ls += __shfl_xor_sync(0xffffffffu, ls, 1);
                ls += __shfl_xor_sync(0xffffffffu, ls, 2);
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        o[sl][i][j] += o[sl][i][2 + j];
                        if (SPREAD) o[sl][i][j] += __shfl_xor_sync(0xffffffffu, o[sl][i][j], 16);
                    }
                if (row0 + sl * 8 + g >= a.group || (HEADS == 4 && g >= 4)) continue;
                float* dst = park + (sl * 8 + g) * C::PARK + 2 * t4;
#pragma unroll
                for (int i = 0; i < NT; ++i) *reinterpret_cast<float2*>(dst + i * 8) = make_float2(o[sl][i][0], o[sl][i][1]);
                if (t4 == 0) *reinterpret_cast<float2*>(park + C::ROWS * C::PARK + (sl * 8 + g) * 2) = make_float2(m[sl], ls);
            }
            __syncthreads();
            const long long part_row = ((long long)blockIdx.x * 2 + (starts_here ? 1 : 0)) * ws.wh * ws.rows;
            float* part = ws.clusters ? shared_part : ws.o + part_row * ws.dkm;
            float* part_ml = ws.clusters ? shared_part + ws.wh * ws.rows * ws.dkm : ws.ml + part_row * 2;
            fold_warps<C::DKM, C::PARK, C::ROWS, TQ>(reinterpret_cast<const float*>(smem_raw) + (in_head * wp * NST + stage) * (C::STAGE / 2),
                                                     NST * (C::STAGE / 2), wp, c, a, ws, ct.seq, hk, row0, whole, part, part_ml);
            __syncthreads();
            fresh = true;
        }
        if (last) break;
        if (closing) issue_keys(stage, NST - 1);
        issue_values(stage);
        stage = stage + 1 == NST ? 0 : stage + 1;
        if (++ct.tile == ct.tiles) next_item(ct, c, s, unit, items_per_seq, flags);
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    if (ws.clusters) join_cluster<TQ>(shared_part, c, a, ws, ct.seq, ct.hs);
}

// ------------------------------------------------------------------------------------------------ f32 caches
// The same division of the work with f32 multiply-adds: tensor cores would round the cache.  FL lanes cover a row of V with
// NFI vectors of four features each; ROWS query heads (at most 8) share a pass.
template <int FL, int NFI, int ROWS>
struct FmaCfg {
    static constexpr int TK = NFI == 2 ? 8 : 16, LPK = 32 / TK, NST = NFI == 2 || (FL == 16 && ROWS >= 4) ? 2 : 3, DKM = FL * 4 * NFI;
    // pitch of a row in shared memory: 4 * LPK floats beyond a multiple of 32, so that the keys of a quarter warp, LPK lanes
    // each, fall on different banks
    static __host__ __device__ constexpr int ld(int pitch)
    {
        // (rows of 8 floats are spread out further: a stage also has to hold a parked result)
        return pitch == 8 ? 40 : pitch + (4 * LPK + 32 - pitch % 32) % 32;
    }
    static_assert(2 * TK * ld(FL == 16 ? 8 : NFI == 1 ? 72 : 136) >= ROWS * (DKM + 2), "a parked result fits in a stage, whatever the pitch");
    static __host__ __device__ constexpr size_t smem(int pitch)
    {
        return ((size_t)4 * NST * 2 * TK * ld(pitch) + (size_t)2 * ROWS * ld(pitch) + 4 * TK * ROWS) * sizeof(float);
    }
};

template <int FL, int NFI, int ROWS, typename TQ>
__global__ void __launch_bounds__(128, 2)
paged_decode_fma_kernel(const PagedView c, const SeqView s, const DecodeArgs a, const DecodeWs ws, int* flags)
{
    using C = FmaCfg<FL, NFI, ROWS>;
    constexpr int TK = C::TK, LPK = C::LPK, NST = C::NST, RPI = 32 / FL;  // RPI: rows that one load instruction covers
    extern __shared__ __align__(16) float smem_f[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, ld = C::ld(c.pitch), stage_len = 2 * TK * ld;
    float* ring = smem_f + (size_t)warp * NST * stage_len;
    float* shared_part = smem_f + C::smem(C::DKM) / sizeof(float);  // of a short call
    pdl_wait();
    pdl_launch();
    const int wp = 4 / ws.wh, unit = TK * wp, in_head = warp / wp, items_per_seq = c.heads / ws.wh * ws.slab_groups;
    float* qs = smem_f + (size_t)4 * NST * stage_len + (size_t)in_head * ROWS * ld;  // one copy per KV head of the CTA
    float* ps = smem_f + (size_t)4 * NST * stage_len + (size_t)ws.wh * ROWS * ld + warp * TK * ROWS;  // this warp's probabilities, (position, row)
    UnitIter ct;
    long long u_begin, u_end, left;
    Deal deal;
    if (ws.clusters) {
        clear_partial(shared_part, ws);
        if (!find_tiles(c, s, unit, items_per_seq, ct, left, flags)) {
            join_cluster<TQ>(shared_part, c, a, ws, ct.seq, ct.hs);
            return;
        }
    } else {
        const bool work = find_work(c, s, unit, items_per_seq, ws, ct, u_begin, u_end, deal, flags);
        if (tid == 0) ws.desc[blockIdx.x] = make_int2(-1, -1);
        if (!work) return;
        left = u_end - u_begin;
    }
    long long to_issue = left;

    const int chunks = c.pitch / 4, key = lane / LPK, sub = lane % LPK;
    const float* kbase = (const float*)c.k;
    const float* vbase = (const float*)c.v;
    // as in the bf16 kernel; each lane looks up the row of one position of the tile
    const int my_pos = warp % wp * TK + lane % TK, col_step = unit / c.page, slot_step = unit % c.page;
    UnitIter it = ct;
    int col = (it.tile * unit + my_pos) / c.page, slot_in_page = (it.tile * unit + my_pos) % c.page, page_id = -1;
    int head = it.hs / ws.slab_groups * ws.wh + in_head;
    if (warp % wp == 0) prefetch_queries<TQ>(c, a, ws, it.seq, head, it.hs % ws.slab_groups * ws.rows);
    const int32_t* table_row = s.table + (long long)it.seq * s.stride;
    int ahead = it.n - it.tile * unit - my_pos;
    unsigned long long exist = 0;
    if (ahead > 0) page_id = table_row[col];
    auto issue = [&](int stage, int age) {
        if (to_issue > 0) {
            int row = -1;
            if (ahead > 0) {
                if ((unsigned)page_id < (unsigned)c.n_pages)
                    row = (page_id * c.heads + head) * c.page + slot_in_page;
                else
                    paged_flag(flags, PAGED_BAD_PAGE);
            }
            const unsigned mask = __ballot_sync(0xffffffffu, row >= 0) & ((1u << TK) - 1u);
            float* kt = ring + stage * stage_len;
            float* vt = kt + TK * ld;
#pragma unroll
            for (int i = 0; i < TK / RPI; ++i) {
                const int r = i * RPI + lane / FL;
                const int src = __shfl_sync(0xffffffffu, row, r);
                const size_t off = src >= 0 ? (size_t)(unsigned)src * c.pitch + lane % FL * 4 : 0;
#pragma unroll
                for (int j = 0; j < NFI; ++j) {
                    const int ch = lane % FL + FL * j;
                    if (ch < chunks) {
                        cp16_zfill(kt + r * ld + ch * 4, src >= 0 ? kbase + off + FL * 4 * j : kbase, src >= 0);
                        cp16_zfill(vt + r * ld + ch * 4, src >= 0 ? vbase + off + FL * 4 * j : vbase, src >= 0);
                    }
                }
            }
            exist |= (unsigned long long)mask << (16 * age);
            --to_issue;
            if (++it.tile == it.tiles) to_issue -= ITEM_COST;
            if (to_issue > 0) {
                if (it.tile < it.tiles) {
                    ahead -= unit;
                    col += col_step;
                    slot_in_page += slot_step;
                    if (slot_in_page >= c.page) {
                        slot_in_page -= c.page;
                        ++col;
                    }
                } else {
                    next_item(it, c, s, unit, items_per_seq, flags);
                    head = it.hs / ws.slab_groups * ws.wh + in_head;
                    if (warp % wp == 0) prefetch_queries<TQ>(c, a, ws, it.seq, head, it.hs % ws.slab_groups * ws.rows);
                    table_row = s.table + (long long)it.seq * s.stride;
                    ahead = it.n - my_pos;
                    col = my_pos / c.page;
                    slot_in_page = my_pos % c.page;
                }
                if (ahead > 0) page_id = table_row[col];
            }
        }
        asm volatile("cp.async.commit_group;\n" ::);
    };
#pragma unroll
    for (int i = 0; i < NST; ++i) issue(i, i);

    const float scale2 = a.scale * 1.44269504088896341f;
    float4 o[ROWS][NFI];
    float m[ROWS], l[ROWS];  // l: this lane's share
    bool fresh = true, starts_here = false;
    int stage = 0;
    for (;;) {
        const int hk = ct.hs / ws.slab_groups * ws.wh + in_head, row0 = (ct.hs % ws.slab_groups) * ROWS;
        if (fresh) {
            fresh = false;
            starts_here = ct.tile == 0;
            const TQ* q = (const TQ*)a.q + (long long)ct.seq * a.q_stride + (long long)(hk * a.group + row0) * c.dk;
            __syncthreads();
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                for (int f = tid & (32 * wp - 1); f < c.pitch; f += 32 * wp)
                    qs[r * ld + f] = row0 + r < a.group && f < c.dk ? load_one(q + r * c.dk + f) : 0.0f;
            __syncthreads();
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                m[r] = -INFINITY;
                l[r] = 0.0f;
#pragma unroll
                for (int j = 0; j < NFI; ++j) o[r][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
        asm volatile("cp.async.wait_group %0;\n" ::"n"(NST - 1) : "memory");
        __syncwarp();
        const float* kt = ring + stage * stage_len;
        const float* vt = kt + TK * ld;
        const int t0 = ct.tile * unit + warp % wp * TK;
        const unsigned live = (unsigned)exist & 0xffffu;
        exist >>= 16;
        // scores: LPK lanes per position, every LPK-th vector of the row each
        float x[ROWS], x_odd[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) x[r] = x_odd[r] = 0.0f;
#pragma unroll 4
        for (int ch = sub; ch < chunks; ch += LPK) {
            const float4 kf = *reinterpret_cast<const float4*>(kt + key * ld + ch * 4);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const float4 qf = *reinterpret_cast<const float4*>(qs + r * ld + ch * 4);
                fma2(x[r], x_odd[r], qf.x, qf.y, kf.x, kf.y);
                fma2(x[r], x_odd[r], qf.z, qf.w, kf.z, kf.w);
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) x[r] += x_odd[r];
        const bool on = (live >> key) & 1u;
        float corr[ROWS];
        bool moved = false;  // the same for the whole warp
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
#pragma unroll
            for (int d = 1; d < LPK; d <<= 1) x[r] += __shfl_xor_sync(0xffffffffu, x[r], d);
            x[r] = on ? __fmul_rn(x[r], scale2) : -INFINITY;
            if (ws.scores && sub == 0 && row0 + r < a.group)
                ws.scores[((long long)ct.seq * a.n_head + hk * a.group + row0 + r) * ws.score_stride + t0 + key] = x[r];
            float top = x[r];
#pragma unroll
            for (int d = LPK; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            top = fmaxf(top, m[r]);
            const float base = top == -INFINITY ? 0.0f : top;
            corr[r] = exp2_fast(m[r] - base);
            moved |= top != m[r];
            m[r] = top;
            x[r] = exp2_fast(x[r] - base);
            l[r] = fmaf(l[r], corr[r], x[r]);  // the LPK lanes of a position hold the same share: divided out at the end
            if (sub == 0) ps[key * ROWS + r] = x[r];
        }
        __syncwarp();
        if (moved)
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
#pragma unroll
                for (int j = 0; j < NFI; ++j) {
                    o[r][j].x *= corr[r];
                    o[r][j].y *= corr[r];
                    o[r][j].z *= corr[r];
                    o[r][j].w *= corr[r];
                }
#pragma unroll
        for (int i = 0; i < TK / RPI; ++i) {
            const int t = i * RPI + lane / FL;
#pragma unroll
            for (int j = 0; j < NFI; ++j) {
                const int ch = lane % FL + FL * j;
                if (ch < chunks) {
                    const float4 vf = *reinterpret_cast<const float4*>(vt + t * ld + ch * 4);
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) {
                        const float p = ps[t * ROWS + r];
                        fma2(o[r][j].x, o[r][j].y, p, p, vf.x, vf.y);
                        fma2(o[r][j].z, o[r][j].w, p, p, vf.z, vf.w);
                    }
                }
            }
        }
        __syncwarp();
        const bool ends = ct.tile + 1 == ct.tiles;
        left -= ends ? 1 + ITEM_COST : 1;
        const bool last = left <= 0;
        if (ends || last) {  // fold the lanes' and the warps' results
            const bool whole = starts_here && ends && !ws.clusters;
            if (tid == 0 && starts_here && !ends && !ws.clusters)
                ws.desc[blockIdx.x] = make_int2(ct.seq * items_per_seq + ct.hs, deal.worker_of(u_end - 1 + (ct.tiles - 1 - ct.tile)));
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                l[r] = warp_sum(l[r]) * (1.0f / LPK);
#pragma unroll
                for (int j = 0; j < NFI; ++j)
#pragma unroll
                    for (int d = FL; d < 32; d <<= 1) {
                        o[r][j].x += __shfl_xor_sync(0xffffffffu, o[r][j].x, d);
                        o[r][j].y += __shfl_xor_sync(0xffffffffu, o[r][j].y, d);
                        o[r][j].z += __shfl_xor_sync(0xffffffffu, o[r][j].z, d);
                        o[r][j].w += __shfl_xor_sync(0xffffffffu, o[r][j].w, d);
                    }
            }
            float* park = ring + stage * stage_len;  // over the tile that was just used
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                if (lane < FL)
#pragma unroll
                    for (int j = 0; j < NFI; ++j) *reinterpret_cast<float4*>(park + r * C::DKM + (lane + FL * j) * 4) = o[r][j];
                if (lane == 0) {
                    park[ROWS * C::DKM + 2 * r] = m[r];
                    park[ROWS * C::DKM + 2 * r + 1] = l[r];
                }
            }
            __syncthreads();
            const long long part_row = ((long long)blockIdx.x * 2 + (starts_here ? 1 : 0)) * ws.wh * ws.rows;
            float* part = ws.clusters ? shared_part : ws.o + part_row * ws.dkm;
            float* part_ml = ws.clusters ? shared_part + ws.wh * ws.rows * ws.dkm : ws.ml + part_row * 2;
            fold_warps<C::DKM, C::DKM, ROWS, TQ>(smem_f + (in_head * wp * NST + stage) * stage_len, NST * stage_len, wp, c, a, ws, ct.seq, hk, row0, whole, part,
                                                 part_ml);
            __syncthreads();
            fresh = true;
        }
        if (last) break;
        issue(stage, NST - 1);
        stage = stage + 1 == NST ? 0 : stage + 1;
        if (++ct.tile == ct.tiles) next_item(ct, c, s, unit, items_per_seq, flags);
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    if (ws.clusters) join_cluster<TQ>(shared_part, c, a, ws, ct.seq, ct.hs);
}

// ------------------------------------------------------------------------------------------------ joining
// One CTA per (worker whose last item goes on, row of the item): folds the partial results of workers w .. last.  Also
// answers for the sequences without any position.
template <typename TQ>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedView c, const SeqView s, const DecodeArgs a, const DecodeWs ws, int* flags)
{
    extern __shared__ float wgt[];  // the partial results' factors, then the threads' sums
    __shared__ float red[4];
    pdl_wait();
    pdl_launch();
    const int w0 = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
    if (row == 0)
        for (int i = w0; i < s.n_seq; i += gridDim.x)
            if (paged_len(c, s, i, flags) == 0) {
                for (int f = tid; f < a.n_head * c.dk; f += 128) store_one((TQ*)a.out + (long long)i * a.n_head * c.dk + f, 0.0f);
                for (int h = tid; a.lse && h < a.n_head; h += 128) a.lse[(long long)i * a.n_head + h] = -INFINITY;
            }
    const int2 d = ws.desc[w0];
    if (d.x < 0) return;
    const int items_per_seq = c.heads / ws.wh * ws.slab_groups, seq = d.x / items_per_seq, hs = d.x % items_per_seq;
    const int gi = hs % ws.slab_groups * ws.rows + row % ws.rows, hk = hs / ws.slab_groups * ws.wh + row / ws.rows, n = d.y - w0 + 1;
    if (gi >= a.group) return;
    // the first worker's partial result is in its slot 1, the others' in slot 0
    auto at = [&](int i) { return ((long long)(w0 + i) * 2 + (i == 0 ? 1 : 0)) * ws.wh * ws.rows + row; };
    float top = -INFINITY;
    for (int i = tid; i < n; i += 128) top = fmaxf(top, ws.ml[at(i) * 2]);
    top = warp_max(top);
    if ((tid & 31) == 0) red[tid >> 5] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    for (int i = tid; i < n; i += 128) {
        const float2 ml = *reinterpret_cast<const float2*>(ws.ml + at(i) * 2);
        const float f = exp2f(ml.x - base);
        wgt[i] = f;
        sum = fmaf(ml.y, f, sum);
    }
    __syncthreads();
    sum = warp_sum(sum);
    if ((tid & 31) == 0) red[tid >> 5] = sum;
    __syncthreads();
    sum = (red[0] + red[1]) + (red[2] + red[3]);
    // four features per thread, the remaining factor of the CTA over the partial results
    const int lanes = ws.dkm / 4, parts = 128 / lanes, f = tid % lanes, part = tid / lanes;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (part < parts)
        for (int i = part; i < n; i += parts) {
            const float4 y = *reinterpret_cast<const float4*>(ws.o + at(i) * ws.dkm + 4 * f);
            const float k = wgt[i];
            acc.x = fmaf(y.x, k, acc.x);
            acc.y = fmaf(y.y, k, acc.y);
            acc.z = fmaf(y.z, k, acc.z);
            acc.w = fmaf(y.w, k, acc.w);
        }
    __syncthreads();
    float4* sums = reinterpret_cast<float4*>(wgt);
    sums[tid] = acc;
    __syncthreads();
    const long long hq = (long long)seq * a.n_head + hk * a.group + gi;
    if (part == 0) {
        for (int p = 1; p < parts; ++p) {
            const float4 y = sums[p * lanes + f];
            acc.x += y.x;
            acc.y += y.y;
            acc.z += y.z;
            acc.w += y.w;
        }
        const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
        const float v[4] = {acc.x, acc.y, acc.z, acc.w};
        for (int i = 0; i < 4; ++i)
            if (4 * f + i < c.dk) store_one((TQ*)a.out + hq * c.dk + 4 * f + i, v[i] * inv);
    }
    if (tid == 0) {
        const float z = sum == 0.0f ? -INFINITY : top + log2f(sum);
        if (a.lse) a.lse[hq] = z * 0.693147180559945309f;
        if (ws.lse2) ws.lse2[hq] = z;
    }
}

// weight[t] += sum over the group of 2^(score_t - lse): one thread per position of a (sequence, KV head)
__global__ void __launch_bounds__(256) paged_add_weights_kernel(const PagedView c, const SeqView s, const DecodeArgs a, const DecodeWs ws, int* flags)
{
    pdl_wait();
    const int seq = blockIdx.x / c.heads, hk = blockIdx.x % c.heads, n = paged_len(c, s, seq, flags);
    const long long hq = (long long)seq * a.n_head + hk * a.group;
    for (int t = blockIdx.y * 256 + threadIdx.x; t < n; t += gridDim.y * 256) {
        const long long row = paged_row(s.table[(long long)seq * s.stride + t / c.page], c.n_pages, c.heads, c.page, hk, t % c.page);
        if (row < 0) continue;
        float sum = 0.0f;
        for (int i = 0; i < a.group; ++i) {
            const float z = ws.lse2[hq + i];
            sum += z == -INFINITY ? 0.0f : exp2f(ws.scores[(hq + i) * ws.score_stride + t] - z);
        }
        // added atomically: a page listed by several sequences loses nothing (elsewhere there is one addition, in no need of order)
        atomicAdd(c.w + row, sum);
    }
}

// how a call lays out its workspace; rows and dkm follow the kernel that takes it
struct WsPlan {
    size_t desc, ml, o, lse2, scores, total;
    int wh, rows, dkm, slab_groups;
    long long score_stride;
};
static WsPlan plan_ws(int sm_count, bool f32_cache, const PagedView& c, const SeqView& s, size_t n_head, bool accumulate)
{
    const int group = (int)(n_head / c.heads);
    WsPlan p{};
    if (f32_cache) {
        p.rows = group == 1 ? 1 : group == 2 ? 2 : group <= 4 ? 4 : 8;
        p.dkm = c.dk <= 64 ? 64 : c.dk <= 128 ? 128 : 256;
    } else {
        p.rows = group > 8 ? 16 : group > 4 ? 8 : 4;
        p.dkm = c.dk <= 64 ? 64 : c.dk <= 112 ? 112 : c.dk <= 128 ? 128 : c.dk <= 192 ? 192 : 256;
    }
    p.slab_groups = (group + p.rows - 1) / p.rows;
    // Measured with 1 / 2 / 4 heads: 128 sequences of 0..640 positions with 16 KV heads of 128 73.7 / 65.8 / 70.6 us, 32 of
    // 256..2048 with 32 of 100 97.5 / 98.7 / 105 us, 64 of 1000..8192 with 8 of 128 206.6 / 206.8 / 210 us.
    p.wh = p.rows == 16 || c.heads % 2 != 0 ? 1 : 2;
    const size_t g = (size_t)sm_count * MAX_WORKERS;
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    p.desc = 0;
    p.ml = up(g * sizeof(int2));
    p.o = p.ml + up(g * 2 * p.wh * p.rows * 2 * sizeof(float));
    p.lse2 = p.o + up(g * 2 * p.wh * p.rows * p.dkm * sizeof(float));
    p.scores = p.lse2 + (accumulate ? up(s.n_seq * n_head * sizeof(float)) : 0);
    p.score_stride = (paged_capacity(c, s) + MAX_UNIT - 1) / MAX_UNIT * MAX_UNIT;
    p.total = p.scores + (accumulate ? s.n_seq * n_head * (size_t)p.score_stride * sizeof(float) : 0);
    return p;
}

template <typename... K>
static nnb_status launch_workers(nnb_engine* e, void (*kern)(K...), size_t smem, int (&per_sm)[64], const PagedView& c, const SeqView& s, const DecodeArgs& a,
                                 DecodeWs ws, int* workers)
{
    const size_t part = (size_t)ws.wh * ws.rows * (ws.dkm + 2) * sizeof(float);
    int& n = per_sm[e->device & 63];  // resident CTAs per SM, by device
    if (n == 0) {  // (a short call's parts: at most 16 rows)
        NNB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(smem + 16 * (ws.dkm + 2) * sizeof(float))));
        NNB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, 128, smem));
        n = n < 1 ? 1 : n > MAX_CTAS_PER_SM ? MAX_CTAS_PER_SM : n;
    }
    ws.wide = e->sm_count * n;
    const size_t items = (size_t)s.n_seq * (c.heads / ws.wh) * ws.slab_groups, cap = (size_t)paged_capacity(c, s);
    // One CTA per SM at most, so that the clusters of a short call find room at once.
    if (cap <= SHORT_CALL && items * CLUSTER <= (size_t)e->sm_count) {
        ws.clusters = 1;
        *workers = 0;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)items * CLUSTER);
        cfg.blockDim = dim3(128);
        cfg.dynamicSmemBytes = smem + part;
        cfg.stream = e->stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {CLUSTER, 1, 1};
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        NNB_CUDA(cudaLaunchKernelEx(&cfg, kern, c, s, a, ws, e->dev_flags));
        e->launches++;
        return NNB_OK;
    }
    // (the lengths are on the device: the table's capacity bounds the cost from above)
    const size_t most = items * (ceil_div(cap, (size_t)16 * (4 / ws.wh)) + ITEM_COST);
    *workers = most >= (size_t)LONG_CALL * ws.wide ? ws.wide + ws.wide / 2 : ws.wide;
    NNB_CUDA(launch_ex(e, kern, dim3((unsigned)*workers), dim3(128), smem, c, s, a, ws, e->dev_flags));
    e->launches++;
    return NNB_OK;
}
template <int KS, typename TQ>
static nnb_status launch_mma(nnb_engine* e, const PagedView& c, const SeqView& s, const DecodeArgs& a, const DecodeWs& ws, int* workers)
{
    constexpr bool PREC = sizeof(TQ) == 4;
    static int n4[64] = {}, n8[64] = {}, n16[64] = {};
    if (ws.rows == 16) return launch_workers(e, paged_decode_mma_kernel<KS, 16, TQ>, MmaCfg<KS, 16, PREC>::SMEM, n16, c, s, a, ws, workers);
    if constexpr (PREC) {
        if (ws.rows == 4) return launch_workers(e, paged_decode_mma_kernel<KS, 4, TQ>, MmaCfg<KS, 4, PREC>::SMEM, n4, c, s, a, ws, workers);
    }
    return launch_workers(e, paged_decode_mma_kernel<KS, 8, TQ>, MmaCfg<KS, 8, PREC>::SMEM, n8, c, s, a, ws, workers);
}
template <int FL, int NFI, int ROWS, typename TQ>
static nnb_status launch_fma_rows(nnb_engine* e, const PagedView& c, const SeqView& s, const DecodeArgs& a, const DecodeWs& ws, int* workers)
{
    static int per_sm[64] = {};
    // one size for all rows that these lanes cover, so that residency is a property of the kernel
    return launch_workers(e, paged_decode_fma_kernel<FL, NFI, ROWS, TQ>, FmaCfg<FL, NFI, ROWS>::smem(FL * 4 * NFI), per_sm, c, s, a, ws, workers);
}
template <int FL, int NFI, typename TQ>
static nnb_status launch_fma(nnb_engine* e, const PagedView& c, const SeqView& s, const DecodeArgs& a, const DecodeWs& ws, int* workers)
{
    switch (ws.rows) {
        case 1: return launch_fma_rows<FL, NFI, 1, TQ>(e, c, s, a, ws, workers);
        case 2: return launch_fma_rows<FL, NFI, 2, TQ>(e, c, s, a, ws, workers);
        case 4: return launch_fma_rows<FL, NFI, 4, TQ>(e, c, s, a, ws, workers);
        default: return launch_fma_rows<FL, NFI, 8, TQ>(e, c, s, a, ws, workers);
    }
}
template <typename TQ>
static nnb_status launch_decode(nnb_engine* e, bool f32_cache, const PagedView& c, const SeqView& s, const DecodeArgs& a, bool accumulate, char* base)
{
    const WsPlan p = plan_ws(e->sm_count, f32_cache, c, s, (size_t)a.n_head, accumulate);
    DecodeWs ws{(int2*)(base + p.desc), (float*)(base + p.ml), (float*)(base + p.o), accumulate ? (float*)(base + p.lse2) : nullptr,
                      accumulate ? (float*)(base + p.scores) : nullptr, p.score_stride, p.wh, 0, 0, p.rows, p.dkm, p.slab_groups};
    PdlOn pdl(e);
    int workers = 0;
    if (f32_cache) {
        if (p.dkm == 64)
            NNB_TRY((launch_fma<16, 1, TQ>(e, c, s, a, ws, &workers)));
        else if (p.dkm == 128)
            NNB_TRY((launch_fma<32, 1, TQ>(e, c, s, a, ws, &workers)));
        else
            NNB_TRY((launch_fma<32, 2, TQ>(e, c, s, a, ws, &workers)));
    } else {
        switch (p.dkm) {
            case 64: NNB_TRY((launch_mma<4, TQ>(e, c, s, a, ws, &workers))); break;
            case 112: NNB_TRY((launch_mma<7, TQ>(e, c, s, a, ws, &workers))); break;
            case 128: NNB_TRY((launch_mma<8, TQ>(e, c, s, a, ws, &workers))); break;
            case 192: NNB_TRY((launch_mma<12, TQ>(e, c, s, a, ws, &workers))); break;
            default: NNB_TRY((launch_mma<16, TQ>(e, c, s, a, ws, &workers))); break;
        }
    }
    if (workers > 0) {  // (a short call has joined its parts itself)
        const size_t smem = (size_t)(workers > 512 ? workers : 512) * sizeof(float);
        NNB_CUDA(launch_ex(e, paged_join_kernel<TQ>, dim3((unsigned)workers, (unsigned)(p.wh * p.rows)), dim3(128), smem, c, s, a, ws, e->dev_flags));
        e->launches++;
    }
    if (accumulate) {
        const unsigned items = (unsigned)(s.n_seq * c.heads);
        const size_t want = ceil_div((size_t)e->sm_count * 8, items), most = ceil_div((size_t)paged_capacity(c, s), 256);
        NNB_CUDA(launch_ex(e, paged_add_weights_kernel, dim3(items, (unsigned)(want < most ? want : most)), dim3(256), 0, c, s, a, ws, e->dev_flags));
        e->launches++;
    }
    return NNB_OK;
}

}  // namespace nnb

using namespace nnb;

extern "C" {

size_t nnb_paged_attention_workspace(nnb_engine* e, const nnb_paged_cache* c, const nnb_paged_seqs* s, size_t n_head, int accumulate)
{
    PagedView cv;
    SeqView sv;
    if (!e || paged_check_cache("paged_attention_decode", c, &cv) != NNB_OK || paged_check_seqs("paged_attention_decode", c, s, &sv) != NNB_OK ||
        n_head == 0 || n_head % cv.heads != 0)
        return 0;
    return plan_ws(e->sm_count, c->dtype == NNB_F32, cv, sv, n_head, accumulate != 0).total;
}

nnb_status nnb_paged_attention_decode(nnb_engine* e, const nnb_paged_cache* c, const nnb_paged_seqs* s, const void* d_q, int dtype,
                                      size_t q_stride, size_t n_head, float scale, void* d_out, float* d_lse, int accumulate, void* d_ws,
                                      size_t ws_bytes)
{
    const char* who = "paged_attention_decode";
    PagedView cv;
    SeqView sv;
    NNB_TRY(paged_check_cache(who, c, &cv));
    NNB_TRY(paged_check_seqs(who, c, s, &sv));
    NNB_REQUIRE(dtype == NNB_F32 || dtype == NNB_BF16, "%s: dtype %d is neither f32 nor bf16", who, dtype);
    NNB_REQUIRE(n_head > 0 && n_head % cv.heads == 0, "%s: %zu query heads do not share %d key / value heads", who, n_head, cv.heads);
    NNB_REQUIRE((unsigned long long)n_head * s->n_seq <= INT32_MAX, "%s: more than 2^31 - 1 (sequence, head) pairs", who);
    NNB_REQUIRE(s->n_seq == 0 || (d_q && d_out), "%s: queries or output are NULL", who);
    NNB_REQUIRE(s->n_seq <= 1 || q_stride >= n_head * cv.dk, "%s: rows of the queries overlap", who);
    const size_t item = dtype == NNB_F32 ? 4 : 2;
    NNB_REQUIRE(((uintptr_t)d_q | (uintptr_t)d_out) % item == 0, "%s: misaligned queries or output", who);
    NNB_REQUIRE(isfinite(scale), "%s: the scale is not finite", who);
    NNB_REQUIRE(!accumulate || c->d_weight, "%s: the cache has no weights to add to", who);
    NNB_REQUIRE(e, "%s: engine is NULL", who);
    if (s->n_seq == 0) return NNB_OK;
    NNB_REQUIRE(d_ws && (uintptr_t)d_ws % 16 == 0 && ws_bytes >= nnb_paged_attention_workspace(e, c, s, n_head, accumulate),
                "%s: the workspace is too small", who);
    DeviceScope dev(e->device);
    const DecodeArgs a{d_q, (long long)q_stride, (int)n_head, (int)(n_head / cv.heads), scale != 0.0f ? scale : 1.0f / sqrtf((float)cv.dk), d_out, d_lse};
    if (dtype == NNB_F32) return launch_decode<float>(e, c->dtype == NNB_F32, cv, sv, a, accumulate != 0, (char*)d_ws);
    return launch_decode<__nv_bfloat16>(e, c->dtype == NNB_F32, cv, sv, a, accumulate != 0, (char*)d_ws);
}

}  // extern "C"
