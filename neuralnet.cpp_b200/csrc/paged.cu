// paged.cu — the paged key-value cache: argument checks, appending new tokens, eviction by accumulated attention.
#include <cooperative_groups.h>
#include <math.h>

#include "device_math.cuh"
#include "paged.cuh"

namespace nnb {

nnb_status paged_check_cache(const char* who, const nnb_paged_cache* c, PagedView* out)
{
    NNB_REQUIRE(c && c->d_k && c->d_v, "%s: the cache has no keys or values", who);
    NNB_REQUIRE(c->dtype == NNB_F32 || c->dtype == NNB_BF16, "%s: cache dtype %d is neither f32 nor bf16", who, c->dtype);
    NNB_REQUIRE(c->n_pages > 0 && c->page_size > 0 && c->n_head_kv > 0, "%s: the cache has no pages, positions or heads", who);
    NNB_REQUIRE(c->dk > 0 && c->dk <= 256 && c->dk % 2 == 0, "%s: head size %d is not an even number up to 256", who, c->dk);
    NNB_REQUIRE((long long)c->n_pages * c->page_size <= INT32_MAX / c->n_head_kv, "%s: the pool has more than 2^31 - 1 rows", who);
    NNB_REQUIRE(((uintptr_t)c->d_k | (uintptr_t)c->d_v) % 16 == 0 && (uintptr_t)c->d_weight % 4 == 0,
                "%s: keys and values must be 16-byte aligned", who);
    *out = PagedView{c->d_k, c->d_v, c->d_weight, c->n_pages, c->page_size, c->n_head_kv, c->dk, (int)nnb_paged_pitch((size_t)c->dk)};
    return NNB_OK;
}

nnb_status paged_check_seqs(const char* who, const nnb_paged_cache* c, const nnb_paged_seqs* s, SeqView* out)
{
    NNB_REQUIRE(s && s->n_seq >= 0 && s->max_pages > 0, "%s: bad number of sequences or pages", who);
    NNB_REQUIRE(s->n_seq == 0 || (s->d_table && s->d_len), "%s: page table or lengths are NULL", who);
    NNB_REQUIRE(s->table_stride >= (size_t)s->max_pages, "%s: rows of the page table overlap", who);
    NNB_REQUIRE((long long)s->max_pages * c->page_size <= (1ll << 30), "%s: more than 2^30 positions per sequence", who);
    *out = SeqView{s->d_table, s->d_len, (long long)s->table_stride, s->n_seq, s->max_pages};
    return NNB_OK;
}

nnb_status paged_check_errors(nnb_engine* e)
{
    int h = 0;
    NNB_CUDA(cudaMemcpyAsync(&h, e->dev_flags + 1, sizeof(int), cudaMemcpyDeviceToHost, e->stream));
    NNB_CUDA(cudaStreamSynchronize(e->stream));
    if (h) {
        NNB_CUDA(cudaMemsetAsync(e->dev_flags + 1, 0, sizeof(int), e->stream));
        NNB_FAIL(NNB_ERR_INVALID, "a paged-cache operator met%s%s%s%s", h & PAGED_BAD_PAGE ? " a page id outside the pool;" : "",
                 h & PAGED_BAD_LEN ? " a length outside the page table;" : "",
                 h & PAGED_NO_ROOM ? " a token behind the end of its page table;" : "",
                 h & PAGED_BAD_POS ? " a position outside the rotary tables;" : "");
    }
    return NNB_OK;
}

// ------------------------------------------------------------------------------------------------ append
struct AppendArgs {
    const void *q, *k, *v;
    void* q_out;
    long long q_stride, k_stride, v_stride, q_out_stride;
    int n_head, ctx, n_rows;
    const int32_t *row_start, *pos;
    const float *cos, *sin;
    int32_t* len_out;
};

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// VEC elements at p (aligned to VEC elements, 16 bytes at most) as f32, and back with one rounding
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC > 16 ? 16 : sizeof(T) * VEC) Pack {
    T x[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[VEC])
{
    const Pack<T, VEC> r = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = to_f32<T>(r.x[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[VEC])
{
    Pack<T, VEC> r;
    if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) *reinterpret_cast<__nv_bfloat162*>(r.x + i) = __floats2bfloat162_rn(x[i], x[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.x[i] = from_f32<T>(x[i]);
    }
    *reinterpret_cast<Pack<T, VEC>*>(p) = r;
}

// the sequence that row r belongs to: the last s with start[s] <= r, if r is in front of start[s + 1]; -1: none
__device__ __forceinline__ int find_sequence(const int32_t* __restrict__ start, int n_seq, int r)
{
    int lo = 0, hi = n_seq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (start[mid] <= r)
            lo = mid;
        else
            hi = mid;
    }
    return start[lo] <= r && r < start[lo + 1] ? lo : -1;
}

// the new length of ragged sequence i
__device__ __forceinline__ void advance_length(const PagedView& c, const SeqView& s, const int32_t* row_start, int32_t* len_out, int i, int* flags)
{
    const int len = paged_len(c, s, i, flags), cap = paged_capacity(c, s);
    const long long n = (long long)row_start[i + 1] - row_start[i];
    len_out[i] = (int)min((long long)cap, len + (n > 0 ? n : 0));
}

// A CTA takes `tokens` new tokens (at most 4).  All of their features are requested at once, into shared memory (STAGED);
// meanwhile a thread each looks up where they go (sequence, length, page) and the CTA brings their angles.  Then every thread
// turns VEC pairs (j, j + dk/2) of a head of q or k, or copies the same features of v.  Pure traffic, each input read once
// and each output written once; the asynchronous copies hide the chain of lookups (1.8 us) and angles (0.9 us), which with
// loads into registers cost as much again as the features (8400 tokens of 20 + 2 x 5 heads of 128: 41 us).
// Features that are not 16-byte aligned are loaded directly.
// (Room for eight tokens' angles although four are taken: what it leaves, five CTAs per SM, is better than six by 31 to 34 us
// for the tokens above.)
constexpr int APPEND_TOKENS = 8, APPEND_MANY = 4;
constexpr size_t APPEND_SMEM = 64 * 1024;
template <typename TI, typename TC, int VEC, bool STAGED>
__global__ void __launch_bounds__(512) paged_append_kernel(const PagedView c, const SeqView s, const AppendArgs a, int tokens, int* flags)
{
    __shared__ long long place[APPEND_TOKENS];  // row of the token's first KV head, -1: it is not written
    __shared__ int angle[APPEND_TOKENS];
    __shared__ __align__(16) float turn[APPEND_TOKENS][2][128];  // cos and sin of the token's position
    extern __shared__ __align__(16) unsigned char staged[];      // (tokens, q | k | v)
    pdl_wait();
    pdl_launch();
    const int tid = threadIdx.x, half = c.dk / 2, per = half / VEC, heads = a.n_head + 2 * c.heads;
    if ((int)blockIdx.x * tokens >= a.n_rows) {  // the CTA behind the last token: new lengths of ragged sequences
        for (int i = tid; i < s.n_seq; i += blockDim.x) advance_length(c, s, a.row_start, a.len_out, i, flags);
        return;
    }
    const int r0 = blockIdx.x * tokens, n = min(tokens, a.n_rows - r0);
    const TI* q0 = (const TI*)a.q + r0 * a.q_stride;
    const TI* k0 = (const TI*)a.k + r0 * a.k_stride;
    const TI* v0 = (const TI*)a.v + r0 * a.v_stride;
    if (STAGED) {
        const int qc = a.n_head * c.dk * (int)sizeof(TI) / 16, kc = c.heads * c.dk * (int)sizeof(TI) / 16;
        for (int t = 0; t < n; ++t) {
            unsigned char* dst = staged + (size_t)t * (qc + 2 * kc) * 16;
            for (int i = tid; i < qc + 2 * kc; i += blockDim.x) {
                const char* src = i < qc        ? (const char*)(q0 + t * a.q_stride) + i * 16
                                  : i < qc + kc ? (const char*)(k0 + t * a.k_stride) + (i - qc) * 16
                                                : (const char*)(v0 + t * a.v_stride) + (i - qc - kc) * 16;
                const uint32_t sa = (uint32_t)__cvta_generic_to_shared(dst + i * 16);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(sa), "l"(src) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;\n" ::);
    }
    if (tid < n) {
        const int r = r0 + tid;
        int seq = r, index = 0;
        if (a.row_start) {
            seq = find_sequence(a.row_start, s.n_seq, r);
            index = seq < 0 ? 0 : r - a.row_start[seq];
        }
        long long at = -1;
        if (seq >= 0) {
            const int cap = paged_capacity(c, s), len = paged_len(c, s, seq, flags);
            const bool idle = !a.row_start && a.pos && a.pos[r] < 0;
            const bool room = index < cap - len;  // no sum that could pass 2^31
            const int slot = room ? len + index : 0, pos = a.pos ? a.pos[r] : slot;
            if (!a.row_start && a.len_out) a.len_out[seq] = idle || !room ? len : len + 1;
            if (!idle) {
                const bool bad_pos = a.cos && (pos < 0 || pos >= a.ctx);
                if (room && !bad_pos) at = paged_row(s.table[(long long)seq * s.stride + slot / c.page], c.n_pages, c.heads, c.page, 0, slot % c.page);
                if (at < 0) paged_flag(flags, !room ? PAGED_NO_ROOM : bad_pos ? PAGED_BAD_POS : PAGED_BAD_PAGE);
            }
            angle[tid] = pos;
        }
        place[tid] = at;
    }
    __syncthreads();
    if (a.cos) {
        for (int i = tid; i < n * half; i += blockDim.x) {
            const int t = i / half, f = i - t * half;
            if (place[t] >= 0) {
                turn[t][0][f] = a.cos[(long long)angle[t] * half + f];
                turn[t][1][f] = a.sin[(long long)angle[t] * half + f];
            }
        }
    }
    if (STAGED) asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    __syncthreads();
    TC* kc = reinterpret_cast<TC*>(c.k);
    TC* vc = reinterpret_cast<TC*>(c.v);
    for (int i = tid; i < heads * per; i += blockDim.x) {
        const int h = i / per, j = (i - h * per) * VEC;
        for (int t = 0; t < n; ++t) {
            const long long row0 = place[t];
            if (row0 < 0) continue;
            const TI* src;
            if (STAGED)
                src = reinterpret_cast<const TI*>(staged) + (t * heads + h) * c.dk + j;
            else if (h < a.n_head)
                src = q0 + t * a.q_stride + (long long)h * c.dk + j;
            else if (h < a.n_head + c.heads)
                src = k0 + t * a.k_stride + (long long)(h - a.n_head) * c.dk + j;
            else
                src = v0 + t * a.v_stride + (long long)(h - a.n_head - c.heads) * c.dk + j;
            float x[VEC], y[VEC];
            load_vec<TI, VEC>(src, x);
            load_vec<TI, VEC>(src + half, y);
            if (a.cos && h < a.n_head + c.heads) {
                float cs[VEC], sn[VEC];
                load_vec<float, VEC>(turn[t][0] + j, cs);
                load_vec<float, VEC>(turn[t][1] + j, sn);
#pragma unroll
                for (int u = 0; u < VEC; ++u) {
                    const float p = x[u], q = y[u];
                    x[u] = fmaf(p, cs[u], -__fmul_rn(q, sn[u]));
                    y[u] = fmaf(q, cs[u], __fmul_rn(p, sn[u]));
                }
            }
            if (h < a.n_head) {
                TI* dst = (TI*)a.q_out + (r0 + t) * a.q_out_stride + (long long)h * c.dk + j;
                store_vec<TI, VEC>(dst, x);
                store_vec<TI, VEC>(dst + half, y);
            } else {
                const int hk = h - a.n_head;
                TC* dst = (hk < c.heads ? kc + (row0 + (long long)hk * c.page) * c.pitch : vc + (row0 + (long long)(hk - c.heads) * c.page) * c.pitch) + j;
                store_vec<TC, VEC>(dst, x);
                store_vec<TC, VEC>(dst + half, y);
            }
        }
    }
    const int pad = c.pitch - c.dk;
    for (int i = tid; i < n * c.heads; i += blockDim.x) {
        const int t = i / c.heads;
        if (place[t] < 0) continue;
        const long long row = place[t] + (long long)(i - t * c.heads) * c.page;
        for (int f = 0; f < pad; ++f) kc[row * c.pitch + c.dk + f] = vc[row * c.pitch + c.dk + f] = from_f32<TC>(0.0f);
        if (c.w) c.w[row] = 0.0f;
    }
}

// the same as a launch of its own, after the rows, which read the old lengths: for d_len_out = d_len
__global__ void paged_advance_kernel(const PagedView c, const SeqView s, const int32_t* __restrict__ row_start, int32_t* len_out, int* flags)
{
    pdl_wait();
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < s.n_seq) advance_length(c, s, row_start, len_out, i, flags);
}

template <typename TI, typename TC>
static nnb_status launch_append(nnb_engine* e, const PagedView& c, const SeqView& s, const AppendArgs& a, size_t n_rows)
{
    const int half = c.dk / 2;
    const uintptr_t io = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v;
    const unsigned long long st = a.q_stride | a.k_stride | a.v_stride;
    const size_t q_bytes = (size_t)a.n_head * c.dk * sizeof(TI), kv_bytes = (size_t)c.heads * c.dk * sizeof(TI), row = q_bytes + 2 * kv_bytes;
    const bool staged = io % 16 == 0 && st * sizeof(TI) % 16 == 0 && q_bytes % 16 == 0 && kv_bytes % 16 == 0 && row <= APPEND_SMEM;
    // the widest vector that head size, strides and addresses allow
    auto fits = [&](int v) {
        const uintptr_t bytes = sizeof(TI) * v > 16 ? 16 : sizeof(TI) * v;
        return half % v == 0 && (uintptr_t)a.q_out % bytes == 0 && a.q_out_stride % v == 0 && (staged || (io % bytes == 0 && st % v == 0));
    };
    const int vec = fits(8) ? 8 : fits(2) ? 2 : 1, items = (a.n_head + 2 * c.heads) * (half / vec);
    // Few tokens: one per CTA, a thread for every vector.  Many: four, whose lookups are done side by side (8400 tokens of 20 + 2 x 5
    // heads of 128 take 44 / 34 / 31 / 36 us with 1 / 2 / 4 / 8 per CTA of 256 threads).
    const bool few = n_rows <= 4 * (size_t)e->sm_count;
    size_t tokens = few ? 1 : APPEND_MANY;
    if (staged && tokens > APPEND_SMEM / row) tokens = APPEND_SMEM / row;
    const unsigned threads = !few ? 256 : items >= 512 ? 512 : (unsigned)(items + 31) / 32 * 32;
    const bool lengths = a.row_start && a.len_out && a.len_out != s.len;
    void (*kern)(PagedView, SeqView, AppendArgs, int, int*);
    if (staged) {
        kern = vec == 8 ? paged_append_kernel<TI, TC, 8, true> : vec == 2 ? paged_append_kernel<TI, TC, 2, true> : paged_append_kernel<TI, TC, 1, true>;
        static bool raised[64][3] = {};  // the attribute is per device
        bool& done = raised[e->device & 63][vec == 8 ? 0 : vec == 2 ? 1 : 2];
        if (!done) NNB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)APPEND_SMEM));
        done = true;
    } else {
        kern = vec == 8 ? paged_append_kernel<TI, TC, 8, false> : vec == 2 ? paged_append_kernel<TI, TC, 2, false> : paged_append_kernel<TI, TC, 1, false>;
    }
    NNB_CUDA(launch_ex(e, kern, dim3((unsigned)ceil_div(n_rows, tokens) + lengths), dim3(threads), staged ? tokens * row : 0, c, s, a, (int)tokens, e->dev_flags));
    e->launches++;
    return NNB_OK;
}

// ------------------------------------------------------------------------------------------------ eviction
// A weight as an unsigned key of the same order; -0 is 0 and a NaN is below every number.
__device__ __forceinline__ uint32_t weight_key(float w)
{
    if (w != w) return 0u;
    const uint32_t b = __float_as_uint(__fadd_rn(w, 0.0f));
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int SEL_NT = 512, SEL_BITS = 11, SEL_BINS = 1 << SEL_BITS;
static_assert(SEL_BINS == 4 * SEL_NT && 3 * SEL_BITS >= 32, "a thread holds four digits, three rounds see every bit");
constexpr int SEL_KEYS = 40 * 1024;  // keys that a CTA can hold (160 KB)

// A cluster of CTAs per (sequence, KV head), each with a stretch of its positions: the positions to keep, in order, into
// kept[item][0..budget).  Of the middle positions the `need` heaviest are wanted: rounds of a radix histogram over the
// weights' ordered bits (11, 11 and 10 of them), summed over the cluster through distributed shared memory, find the key of
// the last one taken and how many positions with that key are taken, the lowest positions first; then every warp counts and
// compacts a stretch with ballots.  The rounds end as soon as all positions with the prefix are taken, mostly after two.  The
// weights are read once, into shared memory, if a CTA's share fits there.  Bound by the latency of its rounds, 2 us each
// (8-bit digits take three or four of them, 1.7 us each).
__global__ void __launch_bounds__(SEL_NT)
paged_select_kernel(const PagedView c, const SeqView s, int budget, int sinks, int recent, int32_t* __restrict__ kept, int kept_stride, int cached, int* flags)
{
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ __align__(16) uint32_t keys[];
    __shared__ __align__(16) int hist[SEL_BINS], sum[SEL_BINS];
    __shared__ int n_sure[32], n_tie[32], total[2], pick[3];
    pdl_wait();
    pdl_launch();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int item = blockIdx.x / ranks, seq = item / c.heads, head = item % c.heads;
    constexpr int WARPS = SEL_NT / 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = paged_len(c, s, seq, flags);
    if (n <= budget) return;  // the whole cluster: everything is kept
    const int32_t* table = s.table + (long long)seq * s.stride;
    auto key_at = [&](int t) {
        const long long row = paged_row(table[t / c.page], c.n_pages, c.heads, c.page, head, t % c.page);
        if (row < 0) paged_flag(flags, PAGED_BAD_PAGE);
        return row < 0 ? weight_key(0.0f) : weight_key(c.w[row]);
    };
    const int part = (n + ranks - 1) / ranks, t0 = min(n, rank * part), t1 = min(n, t0 + part);
    const int lo = max(t0, sinks), hi = min(t1, n - recent);  // the middle positions of this CTA
    const bool hold = part <= cached;
    reinterpret_cast<int4*>(hist)[tid] = make_int4(0, 0, 0, 0);
    if (hold) {
        int col = (lo + tid) / c.page, slot = (lo + tid) % c.page;
        const int col_step = SEL_NT / c.page, slot_step = SEL_NT % c.page;
        bool bad = false;  // (raised at the end: a flag between the loads would keep them in order)
        for (int t = lo + tid; t < hi; t += 8 * SEL_NT) {
            long long row[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const bool in = t + u * SEL_NT < hi;
                row[u] = in ? paged_row(table[col], c.n_pages, c.heads, c.page, head, slot) : -2;
                col += col_step;
                slot += slot_step;
                if (slot >= c.page) {
                    slot -= c.page;
                    ++col;
                }
            }
            float w[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                w[u] = row[u] >= 0 ? c.w[row[u]] : 0.0f;
                bad |= row[u] == -1;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (t + u * SEL_NT < hi) keys[t + u * SEL_NT - t0] = weight_key(w[u]);
        }
        if (bad) paged_flag(flags, PAGED_BAD_PAGE);
    }
    __syncthreads();
    auto key = [&](int t) { return hold ? keys[t - t0] : key_at(t); };
    int need = budget - sinks - recent, shift = 32;
    uint32_t prefix = 0;  // the key of the last position taken, down to bit `shift`
    if (need > 0) {
        for (int round = 0; round < 3; ++round) {
            const int above = shift;  // the bits from here on are known
            shift = max(32 - (round + 1) * SEL_BITS, 0);
            for (int t = lo + tid; t < hi; t += SEL_NT) {
                const uint32_t k = key(t);
                if (round == 0 || k >> above == prefix) atomicAdd(&hist[(k >> shift) & (SEL_BINS - 1) & ((1u << (above - shift)) - 1u)], 1);
            }
            cluster.sync();
            if (ranks > 1) {
                // each CTA adds up its share of the digits and gives the sums to all
                const int share = SEL_BINS / ranks;
                for (int i = rank * share + tid * 4; i < (rank + 1) * share; i += SEL_NT * 4) {
                    int4 part_of[8], all = make_int4(0, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 8; ++r) part_of[r] = r < ranks ? *reinterpret_cast<const int4*>(cluster.map_shared_rank(hist + i, r)) : all;
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        all.x += part_of[r].x;
                        all.y += part_of[r].y;
                        all.z += part_of[r].z;
                        all.w += part_of[r].w;
                    }
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (r < ranks) *reinterpret_cast<int4*>(cluster.map_shared_rank(sum + i, r)) = all;
                }
                cluster.sync();
            }
            // thread i: digit SEL_BINS - 1 - 4 i and the three below
            const int4 own = *reinterpret_cast<const int4*>((ranks > 1 ? sum : hist) + SEL_BINS - 4 - 4 * tid);
            const int mine = own.x + own.y + own.z + own.w;
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            if (lane == 31) n_sure[warp] = upto;
            __syncthreads();
            upto += warp_sum_i(lane < warp ? n_sure[lane] : 0);
            if (upto >= need && upto - mine < need) {
                int left = need - (upto - mine), digit = SEL_BINS - 1 - 4 * tid, count = own.w;
                if (count < left) { left -= count; --digit; count = own.z; }
                if (digit == SEL_BINS - 2 - 4 * tid && count < left) { left -= count; --digit; count = own.y; }
                if (digit == SEL_BINS - 3 - 4 * tid && count < left) { left -= count; --digit; count = own.x; }
                pick[0] = digit;
                pick[1] = left;
                pick[2] = count;
            }
            __syncthreads();
            prefix = prefix << (above - shift) | (uint32_t)pick[0];
            need = pick[1];
            if (pick[2] == need) break;  // every position with this prefix is taken
            // for the next round (with a cluster, everybody has read the counts before the second sync)
            reinterpret_cast<int4*>(hist)[tid] = make_int4(0, 0, 0, 0);
            __syncthreads();
        }
    }
    // kept for sure / one of the equal ones of which the first `need` are kept
    const bool any = budget > sinks + recent;  // (otherwise need is 0 and no middle position is kept)
    auto sort_out = [&](int t, bool& sure, bool& tie) {
        sure = t < t1 && (t < sinks || t >= n - recent);
        tie = false;
        if (any && t >= lo && t < hi) {
            const uint32_t k = key(t) >> shift;
            sure = k > prefix;
            tie = k == prefix;
        }
    };
    const int stretch = ((t1 - t0 + WARPS - 1) / WARPS + 31) / 32 * 32, w0 = t0 + warp * stretch, w1 = min(t1, w0 + stretch);
    int sures = 0, ties = 0;
    for (int t = w0; t < w1; t += 32) {
        bool sure, tie;
        sort_out(t + lane < w1 ? t + lane : t1, sure, tie);
        sures += __popc(__ballot_sync(0xffffffffu, sure));
        ties += __popc(__ballot_sync(0xffffffffu, tie));
    }
    if (lane == 0) {
        n_sure[warp] = sures;
        n_tie[warp] = ties;
    }
    __syncthreads();
    if (warp == 0) {
        const int a = warp_sum_i(lane < WARPS ? n_sure[lane] : 0), b = warp_sum_i(lane < WARPS ? n_tie[lane] : 0);
        if (lane == 0) {
            total[0] = a;
            total[1] = b;
        }
    }
    cluster.sync();
    // what lies before this warp's stretch
    sures = warp_sum_i((lane < warp ? n_sure[lane] : 0) + (lane < rank ? *cluster.map_shared_rank(&total[0], min(lane, ranks - 1)) : 0));
    ties = warp_sum_i((lane < warp ? n_tie[lane] : 0) + (lane < rank ? *cluster.map_shared_rank(&total[1], min(lane, ranks - 1)) : 0));
    int32_t* out = kept + (long long)item * kept_stride;
    const unsigned below = (1u << lane) - 1u;
    for (int t = w0; t < w1; t += 32) {
        bool sure, tie;
        sort_out(t + lane < w1 ? t + lane : t1, sure, tie);
        const unsigned ms = __ballot_sync(0xffffffffu, sure), mt = __ballot_sync(0xffffffffu, tie);
        const int tb = ties + __popc(mt & below);
        if (sure || (tie && tb < need)) out[sures + __popc(ms & below) + min(tb, need)] = t + lane;
        sures += __popc(ms);
        ties += __popc(mt);
    }
    cluster.sync();  // nobody leaves while its shared memory is read
}

// Copies the kept rows.  A CTA looks up 64 rows of a (sequence, KV head) at once, then moves them with 16-byte loads, eight
// under way per thread.
constexpr int MOVE_ROWS = 64;
__global__ void __launch_bounds__(256)
paged_move_kernel(const PagedView c, const SeqView s, const int32_t* __restrict__ kept, int kept_stride, int budget, int first, const PagedView d,
                  const int32_t* __restrict__ dst_table, long long dst_stride, int row_bytes, int32_t* __restrict__ len_out, int* flags)
{
    __shared__ long long from[MOVE_ROWS], to[MOVE_ROWS];
    pdl_wait();
    pdl_launch();
    const int item = blockIdx.x, seq = item / c.heads, head = item % c.heads, tid = threadIdx.x;
    const int n = paged_len(c, s, seq, flags), left = min(n, budget), r0 = first + blockIdx.y * MOVE_ROWS, rows = min(MOVE_ROWS, left - r0);
    if (r0 == 0 && head == 0 && tid == 0) len_out[seq] = left;
    if (rows <= 0) return;
    if (tid < rows) {
        const int r = r0 + tid, t = n > budget ? kept[(long long)item * kept_stride + r] : r;
        const long long f = paged_row(s.table[(long long)seq * s.stride + t / c.page], c.n_pages, c.heads, c.page, head, t % c.page);
        const long long g = paged_row(dst_table[(long long)seq * dst_stride + r / d.page], d.n_pages, d.heads, d.page, head, r % d.page);
        if (f < 0 || g < 0) paged_flag(flags, PAGED_BAD_PAGE);
        if (g >= 0) d.w[g] = f >= 0 ? c.w[f] : 0.0f;
        from[tid] = f;
        to[tid] = g;
    }
    __syncthreads();
    const int chunks = row_bytes / 16;
    for (int i0 = tid; i0 < rows * chunks; i0 += 4 * 256) {
        uint4 x[4], y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * 256, r = i / chunks;
            x[u] = y[u] = make_uint4(0u, 0u, 0u, 0u);
            if (i < rows * chunks && from[r] >= 0) {
                const long long at = from[r] * row_bytes + (i - r * chunks) * 16;
                x[u] = *reinterpret_cast<const uint4*>((const char*)c.k + at);
                y[u] = *reinterpret_cast<const uint4*>((const char*)c.v + at);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * 256, r = i / chunks;
            if (i < rows * chunks && to[r] >= 0) {
                const long long at = to[r] * row_bytes + (i - r * chunks) * 16;
                *reinterpret_cast<uint4*>((char*)d.k + at) = x[u];
                *reinterpret_cast<uint4*>((char*)d.v + at) = y[u];
            }
        }
    }
}

}  // namespace nnb

using namespace nnb;

extern "C" {

size_t nnb_paged_pitch(size_t dk) { return (dk + 7) / 8 * 8; }

int64_t nnb_paged_row(const nnb_paged_cache* c, const int32_t* h_table_row, int32_t max_pages, int32_t head, int64_t pos)
{
    if (!c || !h_table_row || c->page_size <= 0 || head < 0 || head >= c->n_head_kv || pos < 0 || pos / c->page_size >= max_pages) return -1;
    return paged_row(h_table_row[pos / c->page_size], c->n_pages, c->n_head_kv, c->page_size, head, (int)(pos % c->page_size));
}

nnb_status nnb_paged_append(nnb_engine* e, const nnb_paged_cache* c, const nnb_paged_seqs* s, const nnb_paged_tokens* t, int32_t* d_len_out)
{
    const char* who = "paged_append";
    PagedView cv;
    SeqView sv;
    NNB_TRY(paged_check_cache(who, c, &cv));
    NNB_TRY(paged_check_seqs(who, c, s, &sv));
    NNB_REQUIRE(t, "%s: tokens are NULL", who);
    NNB_REQUIRE(t->dtype == NNB_F32 || t->dtype == NNB_BF16, "%s: dtype %d is neither f32 nor bf16", who, t->dtype);
    NNB_REQUIRE(t->n_rows <= (1u << 30), "%s: more than 2^30 tokens", who);
    NNB_REQUIRE(t->d_row_start || t->n_rows == (size_t)s->n_seq, "%s: %zu tokens for %d sequences need d_row_start", who, t->n_rows, s->n_seq);
    const size_t kv_row = (size_t)c->n_head_kv * c->dk, q_row = t->n_head > 0 ? (size_t)t->n_head * c->dk : 0;
    NNB_REQUIRE(t->n_rows == 0 || (t->d_k && t->d_v), "%s: keys or values are NULL", who);
    NNB_REQUIRE(t->n_head >= 0 && (t->n_rows == 0 || ((t->n_head > 0) == (t->d_q != nullptr) && (t->d_q != nullptr) == (t->d_q_out != nullptr))),
                "%s: n_head, d_q and d_q_out go together", who);
    NNB_REQUIRE(t->n_rows <= 1 || (t->k_stride >= kv_row && t->v_stride >= kv_row && (!t->d_q || (t->q_stride >= q_row && t->q_out_stride >= q_row))),
                "%s: rows of the new tokens overlap", who);
    NNB_REQUIRE(t->d_q != t->d_q_out || t->q_stride == t->q_out_stride, "%s: rotating in place needs one stride", who);
    const size_t item = t->dtype == NNB_F32 ? 4 : 2;
    NNB_REQUIRE(((uintptr_t)t->d_q | (uintptr_t)t->d_k | (uintptr_t)t->d_v | (uintptr_t)t->d_q_out) % item == 0, "%s: misaligned tokens", who);
    NNB_REQUIRE((t->d_rope_cos == nullptr) == (t->d_rope_sin == nullptr), "%s: rope tables go together", who);
    NNB_REQUIRE(!t->d_rope_cos || t->rope_ctx > 0, "%s: empty rope tables", who);
    NNB_REQUIRE(e, "%s: engine is NULL", who);
    if (s->n_seq == 0) return NNB_OK;
    DeviceScope dev(e->device);
    const AppendArgs a{t->d_q, t->d_k, t->d_v, t->d_q_out, (long long)t->q_stride, (long long)t->k_stride, (long long)t->v_stride,
                       (long long)t->q_out_stride, t->n_head, t->rope_ctx, (int)t->n_rows, t->d_row_start, t->d_pos, t->d_rope_cos, t->d_rope_sin, d_len_out};
    PdlOn pdl(e);
    if (t->n_rows > 0) {
        if (t->dtype == NNB_F32) {
            if (c->dtype == NNB_F32)
                NNB_TRY((launch_append<float, float>(e, cv, sv, a, t->n_rows)));
            else
                NNB_TRY((launch_append<float, __nv_bfloat16>(e, cv, sv, a, t->n_rows)));
        } else {
            if (c->dtype == NNB_F32)
                NNB_TRY((launch_append<__nv_bfloat16, float>(e, cv, sv, a, t->n_rows)));
            else
                NNB_TRY((launch_append<__nv_bfloat16, __nv_bfloat16>(e, cv, sv, a, t->n_rows)));
        }
    }
    if (t->d_row_start && d_len_out && (d_len_out == s->d_len || t->n_rows == 0)) {
        NNB_CUDA(launch_ex(e, paged_advance_kernel, dim3((unsigned)ceil_div((size_t)s->n_seq, 256)), dim3(256), 0, cv, sv, t->d_row_start, d_len_out,
                           e->dev_flags));
        e->launches++;
    }
    return NNB_OK;
}

size_t nnb_paged_evict_workspace(nnb_engine* e, const nnb_paged_cache* src, const nnb_paged_seqs* s, size_t budget)
{
    PagedView cv;
    SeqView sv;
    if (!e || paged_check_cache("paged_evict", src, &cv) != NNB_OK || paged_check_seqs("paged_evict", src, s, &sv) != NNB_OK) return 0;
    const size_t cap = (size_t)paged_capacity(cv, sv), keep = budget < cap ? budget : cap;
    return (size_t)s->n_seq * cv.heads * keep * sizeof(int32_t) + 16;
}

nnb_status nnb_paged_evict(nnb_engine* e, const nnb_paged_cache* src, const nnb_paged_seqs* s, size_t budget, size_t sinks, size_t recent,
                           const nnb_paged_cache* dst, const int32_t* d_dst_table, size_t dst_max_pages, size_t dst_table_stride,
                           int32_t* d_len_out, void* d_ws, size_t ws_bytes)
{
    const char* who = "paged_evict";
    PagedView cv, dv;
    SeqView sv;
    NNB_TRY(paged_check_cache(who, src, &cv));
    NNB_TRY(paged_check_cache(who, dst, &dv));
    NNB_TRY(paged_check_seqs(who, src, s, &sv));
    NNB_REQUIRE(src->d_weight && dst->d_weight, "%s: both caches need weights", who);
    NNB_REQUIRE(src->dtype == dst->dtype && src->n_head_kv == dst->n_head_kv && src->dk == dst->dk,
                "%s: the caches differ in dtype, heads or head size", who);
    NNB_REQUIRE(budget > 0 && budget <= (1u << 30) && sinks <= budget && recent <= budget - sinks,
                "%s: a budget of %zu does not hold %zu sinks and %zu recent positions", who, budget, sinks, recent);
    NNB_REQUIRE(s->n_seq == 0 || (d_dst_table && d_len_out), "%s: destination table or lengths are NULL", who);
    NNB_REQUIRE(dst_max_pages > 0 && dst_table_stride >= dst_max_pages, "%s: rows of the destination table overlap", who);
    NNB_REQUIRE((long long)s->n_seq * cv.heads <= INT32_MAX, "%s: more than 2^31 - 1 (sequence, head) pairs", who);
    const size_t cap = (size_t)paged_capacity(cv, sv), keep = budget < cap ? budget : cap;
    NNB_REQUIRE(dst_max_pages >= ceil_div(keep, (size_t)dst->page_size), "%s: the destination table holds fewer than %zu positions", who, keep);
    NNB_REQUIRE(d_len_out != s->d_len, "%s: the new lengths need their own array", who);
    NNB_REQUIRE(e, "%s: engine is NULL", who);
    if (s->n_seq == 0) return NNB_OK;
    NNB_REQUIRE(d_ws && (uintptr_t)d_ws % 16 == 0 && ws_bytes >= nnb_paged_evict_workspace(e, src, s, budget), "%s: the workspace is too small", who);
    DeviceScope dev(e->device);
    int32_t* kept = (int32_t*)d_ws;
    const unsigned items = (unsigned)(s->n_seq * cv.heads);
    PdlOn pdl(e);
    if (cap > budget) {
        // CTAs per (sequence, KV head): as many as the GPU has room for, each with at least 2048 positions
        unsigned ranks = 1;
        while (ranks < 8 && (size_t)items * ranks * 2 <= (size_t)e->sm_count && cap / (ranks * 2) >= 2048) ranks *= 2;
        const size_t part = ceil_div(cap, ranks), cached = part < SEL_KEYS ? part : SEL_KEYS;
        static bool raised[64] = {};  // the attribute is per device
        if (!raised[e->device & 63]) {
            NNB_CUDA(cudaFuncSetAttribute(paged_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_KEYS * 4));
            raised[e->device & 63] = true;
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(items * ranks);
        cfg.blockDim = dim3(SEL_NT);
        cfg.dynamicSmemBytes = cached * 4;
        cfg.stream = e->stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {ranks, 1, 1};
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        NNB_CUDA(cudaLaunchKernelEx(&cfg, paged_select_kernel, cv, sv, (int)budget, (int)sinks, (int)recent, kept, (int)keep, (int)cached, e->dev_flags));
        e->launches++;
    }
    const int row_bytes = cv.pitch * (src->dtype == NNB_F32 ? 4 : 2);
    for (size_t done = 0; done < keep; done += (size_t)MOVE_ROWS * 65535) {  // (a grid has at most 65535 rows of CTAs)
        const size_t blocks = ceil_div(keep - done, MOVE_ROWS);
        NNB_CUDA(launch_ex(e, paged_move_kernel, dim3(items, (unsigned)(blocks < 65535 ? blocks : 65535)), dim3(256), 0, cv, sv, kept, (int)keep, (int)budget,
                           (int)done, dv,
                           d_dst_table, (long long)dst_table_stride, row_bytes, d_len_out, e->dev_flags));
        e->launches++;
    }
    return NNB_OK;
}

}  // extern "C"
