// paged_attn.cu — attention of one new token per sequence over a paged key-value cache.
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
// The work is cut evenly whatever the lengths: the positions of every (sequence, KV head) form units of 64 (32 for wide f32
// rows), a tile of each unit for each of the CTA's four warps, and worker w of G
// (one CTA each; G at most U, so that every worker has some) takes the units [U w / G, U (w + 1) / G) of the batch in order.  A worker finishes the
// (sequence, KV head) items that lie inside its range; of an item that several workers share each leaves a partial softmax
// (maximum, sum, weighted values) that paged_join_kernel folds in order.  A worker has at most two partial items: slot 0 is
// one that began in an earlier worker, slot 1 one that begins here and goes on in the next.
constexpr int MAX_CTAS_PER_SM = 4, MAX_UNIT = 64;

struct DecodeWs {
    int2* desc;      // (G): the split item that begins in worker w and its last worker; item -1: none
    float* ml;       // (G, 2, rows, 2): maximum (log2 domain) and sum of a partial softmax
    float* o;        // (G, 2, rows, dkm): its weighted values
    float* lse2;     // (n_seq, n_head): log2 of the sum of exp, for the weights; or NULL
    float* scores;   // (n_seq, n_head, score_stride): scores in the log2 domain, for the weights; or NULL
    long long score_stride;
    int rows, dkm;   // rows of an item and their pitch in the partial results
    int slab_groups; // items per (sequence, KV head): larger groups of query heads than a pass serves are cut
};

// position in the batch's order of units
struct UnitIter {
    int seq, hs, tile, n, tiles;
};

template <int UNIT>
__device__ __forceinline__ void advance(UnitIter& it, const PagedView& c, const SeqView& s, int items_per_seq, int* flags)
{
    if (++it.tile < it.tiles) return;
    it.tile = 0;
    if (++it.hs < items_per_seq) return;
    it.hs = 0;
    do {
        it.n = paged_len(c, s, ++it.seq, flags);
        it.tiles = (it.n + UNIT - 1) / UNIT;
    } while (it.tiles == 0 && it.seq + 1 < s.n_seq);
}

// Called by all 128 threads: this worker's units and the place of the first one.
template <int UNIT>
__device__ __forceinline__ bool find_work(const PagedView& c, const SeqView& s, int items_per_seq, UnitIter& it, long long& u0, long long& u1,
                                          long long& units, int& workers, int* flags)
{
    __shared__ long long warp_sum[4], place;
    __shared__ int place_seq;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (s.n_seq + 127) / 128, first = min(s.n_seq, tid * per), last = min(s.n_seq, first + per);
    long long mine = 0;
    for (int i = first; i < last; ++i) mine += (paged_len(c, s, i, flags) + UNIT - 1) / UNIT;
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
    units = 0;
    for (int i = 0; i < 4; ++i) {
        if (i < warp) base += warp_sum[i];
        units += warp_sum[i];
    }
    workers = (int)min((long long)gridDim.x, units);
    if ((int)blockIdx.x >= workers) return false;
    u0 = units * blockIdx.x / workers;
    u1 = units * (blockIdx.x + 1) / workers;
    base += incl - mine;
    if (u0 >= base && u0 < base + mine) {
        int i = first;
        long long left = u0 - base;
        for (; i + 1 < last; ++i) {
            const long long n = (long long)((paged_len(c, s, i, flags) + UNIT - 1) / UNIT) * items_per_seq;
            if (left < n) break;
            left -= n;
        }
        place_seq = i;
        place = left;
    }
    __syncthreads();
    it.seq = place_seq;
    it.n = paged_len(c, s, it.seq, flags);
    it.tiles = (it.n + UNIT - 1) / UNIT;
    it.hs = (int)(place / it.tiles);
    it.tile = (int)(place % it.tiles);
    return true;
}
// the worker that has unit u: the largest w with floor(units w / G) <= u
__device__ __forceinline__ int worker_of(long long u, long long units, int g) { return (int)(((u + 1) * g - 1) / units); }

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
__device__ __forceinline__ void cp16_zfill(void* smem, const void* gmem, bool valid)
{
    const uint32_t sa = (uint32_t)__cvta_generic_to_shared(smem);
    const int sz = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(sa), "l"(gmem), "r"(sz) : "memory");
}

// ------------------------------------------------------------------------------------------------ bf16 caches
// What a configuration of the kernel needs.  KS: 16-feature steps of a row (dk padded with zeros in shared memory only);
// NSLAB: slabs of 8 query heads that share one pass over the cache; PREC: f32 queries and outputs.
template <int KS, int NSLAB, bool PREC>
struct MmaCfg {
    static constexpr int DKM = KS * 16, LD = DKM + 8, TK = 16, UNIT = 4 * TK;
    static constexpr bool REGQ = KS * NSLAB * (PREC ? 6 : 4) <= 64;  // query fragments in registers, else in shared memory
    static constexpr int QROWS = REGQ ? 0 : NSLAB * (PREC ? 24 : 16);
    static constexpr int STAGE = 2 * TK * LD;                        // elements of a warp's key and value tile
    static constexpr int NST = KS > 8 || NSLAB == 2 ? 2 : 3;
    static constexpr int MB_LD = DKM + 8;
    static constexpr size_t SMEM = (size_t)4 * NST * STAGE * 2 + (size_t)QROWS * LD * 2 + 2 * 8 * MB_LD * 4 + 2 * 8 * 2 * 4;
    static constexpr int CTAS = KS <= 8 ? 2 : 1;
};

template <int KS, int NSLAB, typename TQ>
__global__ void __launch_bounds__(128, MmaCfg<KS, NSLAB, sizeof(TQ) == 4>::CTAS)
paged_decode_mma_kernel(const PagedView c, const SeqView s, const DecodeArgs a, const DecodeWs ws, int* flags)
{
    constexpr bool PREC = sizeof(TQ) == 4;
    using C = MmaCfg<KS, NSLAB, PREC>;
    constexpr int LD = C::LD, TK = C::TK, NST = C::NST, CH = 2 * KS, NT = 2 * KS;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    __nv_bfloat16* ring = reinterpret_cast<__nv_bfloat16*>(smem_raw) + (size_t)warp * NST * C::STAGE;
    __nv_bfloat16* qs = reinterpret_cast<__nv_bfloat16*>(smem_raw) + (size_t)4 * NST * C::STAGE;
    float* mb = reinterpret_cast<float*>(qs + (size_t)C::QROWS * LD);  // two parked partial results
    float* mb_ml = mb + 2 * 8 * C::MB_LD;
    pdl_wait();
    pdl_launch();
    const int items_per_seq = c.heads * ws.slab_groups;
    UnitIter ct;
    long long u, u1, units;
    int workers;
    const bool work = find_work<C::UNIT>(c, s, items_per_seq, ct, u, u1, units, workers, flags);
    if (tid == 0) ws.desc[blockIdx.x] = make_int2(-1, -1);
    if (!work) return;

    const int chunks = c.pitch / 8;
    const char* kbase = (const char*)c.k;
    const char* vbase = (const char*)c.v;
    const size_t row_bytes = (size_t)c.pitch * 2;
    // the issuing side runs NST units ahead of the computing side; the page of its lane's row is loaded one unit ahead
    UnitIter it = ct;
    long long iu = u;
    int page_id = -1;
    auto fetch_page = [&]() {
        const int pos = it.tile * C::UNIT + warp * TK + (lane & 15);
        if (iu < u1) page_id = pos < it.n ? s.table[(long long)it.seq * s.stride + pos / c.page] : -1;
    };
    fetch_page();
    // which of the 16 positions of each tile under way exist (bit per position, the oldest tile lowest)
    unsigned long long exist = 0;
    auto issue = [&](int stage, int age) {
        unsigned mask = 0;
        if (iu < u1) {
            const int pos = it.tile * C::UNIT + warp * TK + (lane & 15);
            int row = -1;
            if (pos < it.n) {
                row = (int)paged_row(page_id, c.n_pages, c.heads, c.page, it.hs / ws.slab_groups, pos % c.page);
                if (row < 0) paged_flag(flags, PAGED_BAD_PAGE);
            }
            mask = __ballot_sync(0xffffffffu, row >= 0) & 0xffffu;
            __nv_bfloat16* kt = ring + stage * C::STAGE;
            __nv_bfloat16* vt = kt + TK * LD;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const int idx = i * 32 + lane, r = idx / CH, ch = idx % CH;
                const int src = __shfl_sync(0xffffffffu, row, r);
                const bool ok = src >= 0 && ch < chunks;
                const size_t off = ok ? (size_t)src * row_bytes + ch * 16 : 0;
                cp16_zfill(kt + r * LD + ch * 8, kbase + off, ok);
                cp16_zfill(vt + r * LD + ch * 8, vbase + off, ok);
            }
            if (++iu < u1) advance<C::UNIT>(it, c, s, items_per_seq, flags);
            fetch_page();
        }
        exist |= (unsigned long long)mask << (16 * age);
        asm volatile("cp.async.commit_group;\n" ::);
    };
#pragma unroll
    for (int i = 0; i < NST; ++i) issue(i, i);

    const float scale2 = a.scale * 1.44269504088896341f;
    uint32_t qa[C::REGQ ? NSLAB : 1][C::REGQ ? KS : 1][4], qb[C::REGQ && PREC ? NSLAB : 1][C::REGQ && PREC ? KS : 1][2];
    float o[NSLAB][NT][2], m[NSLAB], l[NSLAB];
    bool fresh = true, starts_here = false;
    int stage = 0, slot = 0;
    for (; u < u1; ++u) {
        const int hk = ct.hs / ws.slab_groups, row0 = (ct.hs % ws.slab_groups) * (8 * NSLAB);  // first query head of the group here
        if (fresh) {  // a new item: its queries, as bf16 pieces whose sum is the f32 value; row g the leading, row g + 8 the second
            fresh = false;
            starts_here = ct.tile == 0;
            slot = starts_here ? 1 : 0;
            if (!C::REGQ) __syncthreads();
#pragma unroll
            for (int sl = 0; sl < NSLAB; ++sl) {
                m[sl] = -INFINITY;
                l[sl] = 0.0f;
#pragma unroll
                for (int i = 0; i < NT; ++i) o[sl][i][0] = o[sl][i][1] = 0.0f;
                const int gi = row0 + sl * 8 + g;
                const TQ* q = (const TQ*)a.q + (long long)ct.seq * a.q_stride + (long long)(hk * a.group + gi) * c.dk;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    if (!C::REGQ && (ks & 3) != warp) continue;
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const int col = ks * 16 + hf * 8 + 2 * t4;
                        const float2 x = gi < a.group && col < c.dk ? load_pair(q + col) : make_float2(0.0f, 0.0f);
                        const uint32_t hi = pack_rn(x.x, x.y);
                        uint32_t lo = 0, lo2 = 0;
                        if (PREC) {
                            const float r0 = __fsub_rn(x.x, __uint_as_float(hi << 16)), r1 = __fsub_rn(x.y, __uint_as_float(hi & 0xffff0000u));
                            lo = pack_rn(r0, r1);
                            lo2 = pack_rn(__fsub_rn(r0, __uint_as_float(lo << 16)), __fsub_rn(r1, __uint_as_float(lo & 0xffff0000u)));
                        }
                        if constexpr (C::REGQ) {
                            qa[sl][ks][2 * hf] = hi;
                            qa[sl][ks][2 * hf + 1] = lo;
                            if constexpr (PREC) qb[sl][ks][hf] = lo2;
                        } else {
                            __nv_bfloat16* dst = qs + (size_t)sl * (PREC ? 24 : 16) * LD + col;
                            *reinterpret_cast<uint32_t*>(dst + g * LD) = hi;
                            *reinterpret_cast<uint32_t*>(dst + (8 + g) * LD) = lo;
                            if (PREC) *reinterpret_cast<uint32_t*>(dst + (16 + g) * LD) = lo2;
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
        const int t0 = ct.tile * C::UNIT + warp * TK;
        const unsigned live = (unsigned)exist & 0xffffu;
        exist >>= 16;
        // scores of 16 positions: n-tile j holds positions t0 + 8 j + 2 t4 + {0, 1} of head g
        float x[NSLAB][2][2];
        {
            float acc[NSLAB][2][4], acc2[NSLAB][2][4];
#pragma unroll
            for (int sl = 0; sl < NSLAB; ++sl)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[sl][j][i] = acc2[sl][j][i] = 0.0f;
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
                        if constexpr (PREC) {
                            f2[0] = qb[sl][ks][0];
                            f2[1] = qb[sl][ks][1];
                        }
                    } else {
                        const __nv_bfloat16* src = qs + (size_t)sl * (PREC ? 24 : 16) * LD + ks * 16;
                        ldsm4(f, src + ((lane & 7) + 8 * ((lane >> 3) & 1)) * LD + 8 * (lane >> 4));
                        if constexpr (PREC) {
                            f2[0] = *reinterpret_cast<const uint32_t*>(src + (16 + g) * LD + 2 * t4);
                            f2[1] = *reinterpret_cast<const uint32_t*>(src + (16 + g) * LD + 8 + 2 * t4);
                        }
                    }
                    mma16816(acc[sl][0], f[0], f[1], f[2], f[3], b[0], b[1]);
                    mma16816(acc[sl][1], f[0], f[1], f[2], f[3], b[2], b[3]);
                    if constexpr (PREC) {
                        mma16816(acc2[sl][0], f2[0], 0u, f2[1], 0u, b[0], b[1]);
                        mma16816(acc2[sl][1], f2[0], 0u, f2[1], 0u, b[2], b[3]);
                    }
                }
            }
#pragma unroll
            for (int sl = 0; sl < NSLAB; ++sl)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float y = __fadd_rn(acc[sl][j][i], acc[sl][j][2 + i]);
                        if constexpr (PREC) y = __fadd_rn(y, acc2[sl][j][i]);
                        x[sl][j][i] = (live >> (8 * j + 2 * t4 + i)) & 1u ? __fmul_rn(y, scale2) : -INFINITY;
                    }
        }
        float corr[NSLAB];
#pragma unroll
        for (int sl = 0; sl < NSLAB; ++sl) {
            if (ws.scores && row0 + sl * 8 + g < a.group) {
                float* dst = ws.scores + ((long long)ct.seq * a.n_head + hk * a.group + row0 + sl * 8 + g) * ws.score_stride + t0 + 2 * t4;
                *reinterpret_cast<float2*>(dst) = make_float2(x[sl][0][0], x[sl][0][1]);
                *reinterpret_cast<float2*>(dst + 8) = make_float2(x[sl][1][0], x[sl][1][1]);
            }
            float top = fmaxf(fmaxf(x[sl][0][0], x[sl][0][1]), fmaxf(x[sl][1][0], x[sl][1][1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(m[sl], fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)));
            const float base = top == -INFINITY ? 0.0f : top;  // nothing seen yet: every exponential is 0
            corr[sl] = exp2f(m[sl] - base);
            m[sl] = top;
            l[sl] *= corr[sl];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    x[sl][j][i] = exp2f(x[sl][j][i] - base);
                    l[sl] += x[sl][j][i];
                }
        }
        // o = o * corr + p . v, p as bf16 pieces (16 bits of it, 24 for f32 outputs) in rows g and g + 8
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
                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma16816(acc, pa[sl][0], pa[sl][1], pa[sl][2], pa[sl][3], b[2 * j], b[2 * j + 1]);
                    if constexpr (PREC) mma16816(acc, pb[sl][0], 0u, pb[sl][1], 0u, b[2 * j], b[2 * j + 1]);
                    o[sl][2 * np + j][0] = fmaf(o[sl][2 * np + j][0], corr[sl], __fadd_rn(acc[0], acc[2]));
                    o[sl][2 * np + j][1] = fmaf(o[sl][2 * np + j][1], corr[sl], __fadd_rn(acc[1], acc[3]));
                }
        }
        __syncwarp();
        issue(stage, NST - 1);
        stage = stage + 1 == NST ? 0 : stage + 1;

        const bool ends = ct.tile + 1 == ct.tiles;
        if (ends || u + 1 == u1) {  // fold the four warps' results; warp 0 writes
            const bool whole = starts_here && ends;
            if (tid == 0 && starts_here && !ends)
                ws.desc[blockIdx.x] = make_int2(ct.seq * items_per_seq + ct.hs, worker_of(u + (ct.tiles - 1 - ct.tile), units, workers));
#pragma unroll
            for (int sl = 0; sl < NSLAB; ++sl) {
                float ls = l[sl], ms = m[sl];
                ls += __shfl_xor_sync(0xffffffffu, ls, 1);
                ls += __shfl_xor_sync(0xffffffffu, ls, 2);
                auto park = [&](int buf) {
                    float* dst = mb + (buf * 8 + g) * C::MB_LD + 2 * t4;
#pragma unroll
                    for (int i = 0; i < NT; ++i) *reinterpret_cast<float2*>(dst + i * 8) = make_float2(o[sl][i][0], o[sl][i][1]);
                    if (t4 == 0) *reinterpret_cast<float2*>(mb_ml + (buf * 8 + g) * 2) = make_float2(ms, ls);
                };
                auto fold = [&](int buf) {
                    const float* src = mb + (buf * 8 + g) * C::MB_LD + 2 * t4;
                    const float2 ml = *reinterpret_cast<const float2*>(mb_ml + (buf * 8 + g) * 2);
                    const float top = fmaxf(ms, ml.x), base = top == -INFINITY ? 0.0f : top;
                    const float ca = exp2f(ms - base), cb = exp2f(ml.x - base);
                    ms = top;
                    ls = fmaf(ls, ca, ml.y * cb);
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        const float2 y = *reinterpret_cast<const float2*>(src + i * 8);
                        o[sl][i][0] = fmaf(o[sl][i][0], ca, y.x * cb);
                        o[sl][i][1] = fmaf(o[sl][i][1], ca, y.y * cb);
                    }
                };
                __syncthreads();
                if (warp >= 2) park(warp - 2);
                __syncthreads();
                if (warp < 2) fold(warp);
                __syncthreads();
                if (warp == 1) park(0);
                __syncthreads();
                if (warp == 0) {
                    fold(0);
                    const int gi = row0 + sl * 8 + g;
                    if (whole && gi < a.group) {
                        const long long hq = (long long)ct.seq * a.n_head + hk * a.group + gi;
                        const float inv = ls == 0.0f ? 0.0f : __fdiv_rn(1.0f, ls);
                        TQ* dst = (TQ*)a.out + hq * c.dk + 2 * t4;
#pragma unroll
                        for (int i = 0; i < NT; ++i)
                            if (i * 8 + 2 * t4 < c.dk) {
                                store_one(dst + i * 8, o[sl][i][0] * inv);
                                store_one(dst + i * 8 + 1, o[sl][i][1] * inv);
                            }
                        if (t4 == 0) {
                            const float z = ls == 0.0f ? -INFINITY : ms + log2f(ls);
                            if (a.lse) a.lse[hq] = z * 0.693147180559945309f;
                            if (ws.lse2) ws.lse2[hq] = z;
                        }
                    } else if (!whole) {
                        const long long r = ((long long)blockIdx.x * 2 + slot) * ws.rows + sl * 8 + g;
                        float* dst = ws.o + r * ws.dkm + 2 * t4;
#pragma unroll
                        for (int i = 0; i < NT; ++i) *reinterpret_cast<float2*>(dst + i * 8) = make_float2(o[sl][i][0], o[sl][i][1]);
                        if (t4 == 0) *reinterpret_cast<float2*>(ws.ml + r * 2) = make_float2(ms, ls);
                    }
                }
            }
            fresh = true;
        }
        if (u + 1 < u1) advance<C::UNIT>(ct, c, s, items_per_seq, flags);
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
}

// ------------------------------------------------------------------------------------------------ f32 caches
// The same division of the work with f32 multiply-adds: tensor cores would round the cache.  FL lanes cover a row of V with
// NFI vectors of four features each; ROWS query heads (at most 8) share a pass.
template <int FL, int NFI, int ROWS>
struct FmaCfg {
    static constexpr int TK = NFI == 2 ? 8 : 16, UNIT = 4 * TK, LPK = 32 / TK, NST = NFI == 2 ? 2 : 3, DKM = FL * 4 * NFI;
    static constexpr int MB = ROWS * DKM + (2 * ROWS + 3) / 4 * 4;  // a parked partial result: values, then maximum and sum per row
    // pitch of a row in shared memory: 4 * LPK floats beyond a multiple of 32, so that the keys of a quarter warp, LPK lanes
    // each, fall on different banks
    static __host__ __device__ constexpr int ld(int pitch) { return pitch + (4 * LPK + 32 - pitch % 32) % 32; }
    static __host__ __device__ constexpr size_t smem(int pitch)
    {
        return ((size_t)4 * NST * 2 * TK * ld(pitch) + (size_t)ROWS * ld(pitch) + 4 * TK * ROWS + (size_t)2 * MB) * sizeof(float);
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
    float* qs = smem_f + (size_t)4 * NST * stage_len;
    float* ps = qs + (size_t)ROWS * ld + warp * TK * ROWS;  // this warp's probabilities, (position, row)
    float* mb = qs + (size_t)ROWS * ld + 4 * TK * ROWS;     // two parked partial results
    pdl_wait();
    pdl_launch();
    const int items_per_seq = c.heads * ws.slab_groups;
    UnitIter ct;
    long long u, u1, units;
    int workers;
    const bool work = find_work<C::UNIT>(c, s, items_per_seq, ct, u, u1, units, workers, flags);
    if (tid == 0) ws.desc[blockIdx.x] = make_int2(-1, -1);
    if (!work) return;

    const int chunks = c.pitch / 4, key = lane / LPK, sub = lane % LPK;
    const float* kbase = (const float*)c.k;
    const float* vbase = (const float*)c.v;
    UnitIter it = ct;
    long long iu = u;
    int page_id = -1;
    auto fetch_page = [&]() {
        const int pos = it.tile * C::UNIT + warp * TK + lane % TK;
        if (iu < u1) page_id = pos < it.n ? s.table[(long long)it.seq * s.stride + pos / c.page] : -1;
    };
    fetch_page();
    unsigned long long exist = 0;  // as in the bf16 kernel
    auto issue = [&](int stage, int age) {
        unsigned mask = 0;
        if (iu < u1) {
            const int pos = it.tile * C::UNIT + warp * TK + lane % TK;
            int row = -1;
            if (pos < it.n) {
                row = (int)paged_row(page_id, c.n_pages, c.heads, c.page, it.hs / ws.slab_groups, pos % c.page);
                if (row < 0) paged_flag(flags, PAGED_BAD_PAGE);
            }
            mask = __ballot_sync(0xffffffffu, row >= 0) & ((1u << TK) - 1u);
            float* kt = ring + stage * stage_len;
            float* vt = kt + TK * ld;
#pragma unroll
            for (int i = 0; i < TK / RPI; ++i) {
                const int r = i * RPI + lane / FL;
                const int src = __shfl_sync(0xffffffffu, row, r);
#pragma unroll
                for (int j = 0; j < NFI; ++j) {
                    const int ch = lane % FL + FL * j;
                    if (ch < chunks) {
                        const size_t off = src >= 0 ? (size_t)src * c.pitch + ch * 4 : 0;
                        cp16_zfill(kt + r * ld + ch * 4, kbase + off, src >= 0);
                        cp16_zfill(vt + r * ld + ch * 4, vbase + off, src >= 0);
                    }
                }
            }
            if (++iu < u1) advance<C::UNIT>(it, c, s, items_per_seq, flags);
            fetch_page();
        }
        exist |= (unsigned long long)mask << (16 * age);
        asm volatile("cp.async.commit_group;\n" ::);
    };
#pragma unroll
    for (int i = 0; i < NST; ++i) issue(i, i);

    const float scale2 = a.scale * 1.44269504088896341f;
    float4 o[ROWS][NFI];
    float m[ROWS], l[ROWS];  // l: this lane's share
    bool fresh = true, starts_here = false;
    int stage = 0, slot = 0;
    for (; u < u1; ++u) {
        const int hk = ct.hs / ws.slab_groups, row0 = (ct.hs % ws.slab_groups) * ROWS;
        if (fresh) {
            fresh = false;
            starts_here = ct.tile == 0;
            slot = starts_here ? 1 : 0;
            const TQ* q = (const TQ*)a.q + (long long)ct.seq * a.q_stride + (long long)(hk * a.group + row0) * c.dk;
            __syncthreads();
            for (int i = tid; i < ROWS * c.pitch; i += 128) {
                const int r = i / c.pitch, f = i % c.pitch;
                qs[r * ld + f] = row0 + r < a.group && f < c.dk ? load_one(q + r * c.dk + f) : 0.0f;
            }
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
        const int t0 = ct.tile * C::UNIT + warp * TK;
        const unsigned live = (unsigned)exist & 0xffffu;
        exist >>= 16;
        // scores: LPK lanes per position, every LPK-th vector of the row each
        float x[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) x[r] = 0.0f;
        for (int ch = sub; ch < chunks; ch += LPK) {
            const float4 kf = *reinterpret_cast<const float4*>(kt + key * ld + ch * 4);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const float4 qf = *reinterpret_cast<const float4*>(qs + r * ld + ch * 4);
                x[r] = fmaf(qf.x, kf.x, fmaf(qf.y, kf.y, fmaf(qf.z, kf.z, fmaf(qf.w, kf.w, x[r]))));
            }
        }
        const bool on = (live >> key) & 1u;
        float corr[ROWS];
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
            corr[r] = exp2f(m[r] - base);
            m[r] = top;
            x[r] = exp2f(x[r] - base);
            l[r] = fmaf(l[r], corr[r], x[r]);  // the LPK lanes of a position hold the same share: divided out at the end
            if (sub == 0) ps[key * ROWS + r] = x[r];
        }
        __syncwarp();
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
                        o[r][j].x = fmaf(p, vf.x, o[r][j].x);
                        o[r][j].y = fmaf(p, vf.y, o[r][j].y);
                        o[r][j].z = fmaf(p, vf.z, o[r][j].z);
                        o[r][j].w = fmaf(p, vf.w, o[r][j].w);
                    }
                }
            }
        }
        __syncwarp();
        issue(stage, NST - 1);
        stage = stage + 1 == NST ? 0 : stage + 1;

        const bool ends = ct.tile + 1 == ct.tiles;
        if (ends || u + 1 == u1) {  // fold the lanes' and the warps' results; warp 0 writes
            const bool whole = starts_here && ends;
            if (tid == 0 && starts_here && !ends)
                ws.desc[blockIdx.x] = make_int2(ct.seq * items_per_seq + ct.hs, worker_of(u + (ct.tiles - 1 - ct.tile), units, workers));
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
            auto park = [&](float* buf) {
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    if (lane < FL)
#pragma unroll
                        for (int j = 0; j < NFI; ++j) *reinterpret_cast<float4*>(buf + r * C::DKM + (lane + FL * j) * 4) = o[r][j];
                    if (lane == 0) {
                        buf[ROWS * C::DKM + 2 * r] = m[r];
                        buf[ROWS * C::DKM + 2 * r + 1] = l[r];
                    }
                }
            };
            auto fold = [&](const float* buf) {
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    const float mo = buf[ROWS * C::DKM + 2 * r], lo = buf[ROWS * C::DKM + 2 * r + 1];
                    const float top = fmaxf(m[r], mo), base = top == -INFINITY ? 0.0f : top;
                    const float ca = exp2f(m[r] - base), cb = exp2f(mo - base);
                    m[r] = top;
                    l[r] = fmaf(l[r], ca, lo * cb);
#pragma unroll
                    for (int j = 0; j < NFI; ++j) {
                        const float4 y = *reinterpret_cast<const float4*>(buf + r * C::DKM + (lane % FL + FL * j) * 4);
                        o[r][j].x = fmaf(o[r][j].x, ca, y.x * cb);
                        o[r][j].y = fmaf(o[r][j].y, ca, y.y * cb);
                        o[r][j].z = fmaf(o[r][j].z, ca, y.z * cb);
                        o[r][j].w = fmaf(o[r][j].w, ca, y.w * cb);
                    }
                }
            };
            __syncthreads();
            if (warp >= 2) park(mb + (warp - 2) * C::MB);
            __syncthreads();
            if (warp < 2) fold(mb + warp * C::MB);
            __syncthreads();
            if (warp == 1) park(mb);
            __syncthreads();
            if (warp == 0) {
                fold(mb);
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    if (row0 + r >= a.group) continue;
                    const long long hq = (long long)ct.seq * a.n_head + hk * a.group + row0 + r;
                    const long long pr = ((long long)blockIdx.x * 2 + slot) * ws.rows + r;
                    const float inv = l[r] == 0.0f ? 0.0f : __fdiv_rn(1.0f, l[r]);
#pragma unroll
                    for (int j = 0; j < NFI; ++j) {
                        const int f = (lane + FL * j) * 4;
                        if (lane >= FL) continue;
                        if (!whole) {
                            *reinterpret_cast<float4*>(ws.o + pr * ws.dkm + f) = o[r][j];
                        } else {
                            const float v[4] = {o[r][j].x, o[r][j].y, o[r][j].z, o[r][j].w};
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (f + i < c.dk) store_one((TQ*)a.out + hq * c.dk + f + i, v[i] * inv);
                        }
                    }
                    if (lane == 0) {
                        if (!whole) {
                            ws.ml[pr * 2] = m[r];
                            ws.ml[pr * 2 + 1] = l[r];
                        } else {
                            const float z = l[r] == 0.0f ? -INFINITY : m[r] + log2f(l[r]);
                            if (a.lse) a.lse[hq] = z * 0.693147180559945309f;
                            if (ws.lse2) ws.lse2[hq] = z;
                        }
                    }
                }
            }
            fresh = true;
        }
        if (u + 1 < u1) advance<C::UNIT>(ct, c, s, items_per_seq, flags);
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
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
    const int items_per_seq = c.heads * ws.slab_groups, seq = d.x / items_per_seq, hs = d.x % items_per_seq;
    const int gi = hs % ws.slab_groups * ws.rows + row, n = d.y - w0 + 1;
    if (gi >= a.group) return;
    // the first worker's partial result is in its slot 1, the others' in slot 0
    auto at = [&](int i) { return ((long long)(w0 + i) * 2 + (i == 0 ? 1 : 0)) * ws.rows + row; };
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
    const long long hq = (long long)seq * a.n_head + hs / ws.slab_groups * a.group + gi;
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
    int rows, dkm, slab_groups;
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
        p.rows = group > 8 ? 16 : 8;
        p.dkm = c.dk <= 64 ? 64 : c.dk <= 112 ? 112 : c.dk <= 128 ? 128 : c.dk <= 192 ? 192 : 256;
    }
    p.slab_groups = (group + p.rows - 1) / p.rows;
    const size_t g = (size_t)sm_count * MAX_CTAS_PER_SM;
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    p.desc = 0;
    p.ml = up(g * sizeof(int2));
    p.o = p.ml + up(g * 2 * p.rows * 2 * sizeof(float));
    p.lse2 = p.o + up(g * 2 * p.rows * p.dkm * sizeof(float));
    p.scores = p.lse2 + (accumulate ? up(s.n_seq * n_head * sizeof(float)) : 0);
    p.score_stride = (paged_capacity(c, s) + MAX_UNIT - 1) / MAX_UNIT * MAX_UNIT;
    p.total = p.scores + (accumulate ? s.n_seq * n_head * (size_t)p.score_stride * sizeof(float) : 0);
    return p;
}

// launches with the programmatic attribute: the kernel waits for its predecessor itself (pdl_wait before its first access)
struct PdlOn {
    nnb_engine* e;
    bool prev;
    explicit PdlOn(nnb_engine* en) : e(en), prev(en->pdl) { e->pdl = true; }
    ~PdlOn() { e->pdl = prev; }
};

template <typename... K>
static nnb_status launch_workers(nnb_engine* e, void (*kern)(K...), size_t smem, int (&per_sm)[64], const PagedView& c, const SeqView& s, const DecodeArgs& a,
                                 const DecodeWs& ws, int* workers)
{
    int& n = per_sm[e->device & 63];  // resident CTAs per SM, by device
    if (n == 0) {
        NNB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        NNB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, 128, smem));
        n = n < 1 ? 1 : n > MAX_CTAS_PER_SM ? MAX_CTAS_PER_SM : n;
    }
    *workers = e->sm_count * n;
    NNB_CUDA(launch_ex(e, kern, dim3((unsigned)*workers), dim3(128), smem, c, s, a, ws, e->dev_flags));
    e->launches++;
    return NNB_OK;
}
template <int KS, typename TQ>
static nnb_status launch_mma(nnb_engine* e, const PagedView& c, const SeqView& s, const DecodeArgs& a, const DecodeWs& ws, int* workers)
{
    static int one[64] = {}, two[64] = {};
    if (ws.rows == 16)
        return launch_workers(e, paged_decode_mma_kernel<KS, 2, TQ>, MmaCfg<KS, 2, sizeof(TQ) == 4>::SMEM, two, c, s, a, ws, workers);
    return launch_workers(e, paged_decode_mma_kernel<KS, 1, TQ>, MmaCfg<KS, 1, sizeof(TQ) == 4>::SMEM, one, c, s, a, ws, workers);
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
    const DecodeWs ws{(int2*)(base + p.desc), (float*)(base + p.ml), (float*)(base + p.o), accumulate ? (float*)(base + p.lse2) : nullptr,
                      accumulate ? (float*)(base + p.scores) : nullptr, p.score_stride, p.rows, p.dkm, p.slab_groups};
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
    const size_t smem = (size_t)(workers > 512 ? workers : 512) * sizeof(float);
    NNB_CUDA(launch_ex(e, paged_join_kernel<TQ>, dim3((unsigned)workers, (unsigned)(a.group < p.rows ? a.group : p.rows)), dim3(128), smem, c, s, a, ws,
                       e->dev_flags));
    e->launches++;
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
