// paged.cu — the paged key-value cache: argument checks, appending new tokens, eviction by accumulated attention.
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
    int n_head, ctx;
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
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.x[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Pack<T, VEC>*>(p) = r;
}

// the sequence that row r belongs to (the last s with start[s] <= r), by a 32-way search of the whole warp; -1: none
__device__ __forceinline__ int find_sequence(const int32_t* __restrict__ start, int n_seq, int r)
{
    const int lane = threadIdx.x & 31;
    int lo = 0, len = n_seq;
    for (;;) {
        const int step = (len + 31) / 32, i = lane * step;
        const unsigned below = __ballot_sync(0xffffffffu, i < len && start[lo + (i < len ? i : 0)] <= r);
        const int n = __popc(below);
        if (n == 0) return -1;
        lo += (n - 1) * step;
        len = min(step, len - (n - 1) * step);
        if (len <= 1) break;
    }
    return r < start[lo + 1] ? lo : -1;
}

// One CTA per new token.  Every thread turns VEC pairs (j, j + dk/2) of a head of q or k, or copies the same features of v;
// all of a token is written by its CTA, so with one token per sequence the CTA also advances the length.  Pure traffic:
// each input is read once and each output written once.
template <typename TI, typename TC, int VEC>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedView c, const SeqView s, const AppendArgs a, int* flags)
{
    const int r = blockIdx.x, tid = threadIdx.x, half = c.dk / 2, per = half / VEC;
    int seq = r, index = 0;
    if (a.row_start) {
        seq = find_sequence(a.row_start, s.n_seq, r);
        if (seq < 0) return;
        index = r - a.row_start[seq];
    }
    const int cap = paged_capacity(c, s), len = paged_len(c, s, seq, flags);
    const bool idle = !a.row_start && a.pos && a.pos[r] < 0;
    const bool room = index < cap - len;  // no sum that could pass 2^31
    const int slot = room ? len + index : 0;
    const int pos = a.pos ? a.pos[r] : slot;
    if (!a.row_start) {
        __syncthreads();  // the length may be overwritten in place: everyone has read it
        if (a.len_out && tid == 0) a.len_out[seq] = idle || !room ? len : len + 1;
    }
    if (idle) return;
    const bool bad_pos = a.cos && (pos < 0 || pos >= a.ctx);
    const int page = room ? s.table[(long long)seq * s.stride + slot / c.page] : -1;
    const bool bad_page = room && paged_row(page, c.n_pages, c.heads, c.page, 0, 0) < 0;
    if (!room || bad_pos || bad_page) {
        if (tid == 0) paged_flag(flags, !room ? PAGED_NO_ROOM : bad_pos ? PAGED_BAD_POS : PAGED_BAD_PAGE);
        return;
    }
    const long long row0 = paged_row(page, c.n_pages, c.heads, c.page, 0, slot % c.page);
    TC* kc = reinterpret_cast<TC*>(c.k);
    TC* vc = reinterpret_cast<TC*>(c.v);
    for (int i = tid; i < (a.n_head + 2 * c.heads) * per; i += blockDim.x) {
        int h = i / per;
        const int j = (i - h * per) * VEC;
        float x[VEC], y[VEC];
        if (h < a.n_head + c.heads) {
            const bool is_q = h < a.n_head;
            const TI* src = is_q ? (const TI*)a.q + (long long)r * a.q_stride + (long long)h * c.dk
                                 : (const TI*)a.k + (long long)r * a.k_stride + (long long)(h - a.n_head) * c.dk;
            load_vec<TI, VEC>(src + j, x);
            load_vec<TI, VEC>(src + j + half, y);
            if (a.cos) {
                float cs[VEC], sn[VEC];
                load_vec<float, VEC>(a.cos + (long long)pos * half + j, cs);
                load_vec<float, VEC>(a.sin + (long long)pos * half + j, sn);
#pragma unroll
                for (int u = 0; u < VEC; ++u) {
                    const float p = x[u], q = y[u];
                    x[u] = __fadd_rn(__fmul_rn(p, cs[u]), __fmul_rn(-q, sn[u]));
                    y[u] = __fadd_rn(__fmul_rn(q, cs[u]), __fmul_rn(p, sn[u]));
                }
            }
            if (is_q) {
                TI* dst = (TI*)a.q_out + (long long)r * a.q_out_stride + (long long)h * c.dk;
                store_vec<TI, VEC>(dst + j, x);
                store_vec<TI, VEC>(dst + j + half, y);
            } else {
                TC* dst = kc + (row0 + (long long)(h - a.n_head) * c.page) * c.pitch;
                store_vec<TC, VEC>(dst + j, x);
                store_vec<TC, VEC>(dst + j + half, y);
            }
        } else {
            h -= a.n_head + c.heads;
            const TI* src = (const TI*)a.v + (long long)r * a.v_stride + (long long)h * c.dk;
            load_vec<TI, VEC>(src + j, x);
            load_vec<TI, VEC>(src + j + half, y);
            TC* dst = vc + (row0 + (long long)h * c.page) * c.pitch;
            store_vec<TC, VEC>(dst + j, x);
            store_vec<TC, VEC>(dst + j + half, y);
        }
    }
    const int pad = c.pitch - c.dk;
    for (int i = tid; i < c.heads * pad; i += blockDim.x) {
        const long long at = (row0 + (long long)(i / pad) * c.page) * c.pitch + c.dk + i % pad;
        kc[at] = from_f32<TC>(0.0f);
        vc[at] = from_f32<TC>(0.0f);
    }
    if (c.w)
        for (int h = tid; h < c.heads; h += blockDim.x) c.w[row0 + (long long)h * c.page] = 0.0f;
}

// lengths of ragged appends: after the rows, which read the old lengths (d_len_out may be d_len)
__global__ void paged_advance_kernel(const PagedView c, const SeqView s, const int32_t* __restrict__ row_start, int32_t* len_out, int* flags)
{
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= s.n_seq) return;
    const int len = paged_len(c, s, i, flags), cap = paged_capacity(c, s);
    const long long n = (long long)row_start[i + 1] - row_start[i];
    len_out[i] = (int)min((long long)cap, len + (n > 0 ? n : 0));
}

template <typename TI, typename TC>
static nnb_status launch_append(nnb_engine* e, const PagedView& c, const SeqView& s, const AppendArgs& a, size_t n_rows)
{
    const int half = c.dk / 2;
    // the widest vector that head size, strides and addresses allow; tables have rows of half floats
    auto fits = [&](int v) {
        const uintptr_t bi = sizeof(TI) * v > 16 ? 16 : sizeof(TI) * v, bt = 4 * v > 16 ? 16 : 4 * v;
        const uintptr_t io = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out;
        const unsigned long long st = a.q_stride | a.k_stride | a.v_stride | a.q_out_stride;
        return half % v == 0 && io % bi == 0 && st % v == 0 && ((uintptr_t)a.cos | (uintptr_t)a.sin) % bt == 0;
    };
    const int vec = fits(8) ? 8 : fits(2) ? 2 : 1;
    const int items = (a.n_head + 2 * c.heads) * (half / vec);
    const unsigned threads = items >= 256 ? 256 : items > 64 ? 128 : 64;
    auto kern = vec == 8 ? paged_append_kernel<TI, TC, 8> : vec == 2 ? paged_append_kernel<TI, TC, 2> : paged_append_kernel<TI, TC, 1>;
    kern<<<(unsigned)n_rows, threads, 0, e->stream>>>(c, s, a, e->dev_flags);
    e->launches++;
    NNB_CHECK_LAUNCH("paged_append_kernel");
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

constexpr int SEL_NT = 1024;

// exclusive prefix sum of x over the CTA; *total receives the sum.  Uses 33 ints of shared memory.
__device__ __forceinline__ int block_scan(int x, int* sh, int* total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int v = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) sh[warp] = v;
    __syncthreads();
    if (warp == 0) {
        int t = lane < nw ? sh[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += u;
        }
        sh[lane] = t;
    }
    __syncthreads();
    const int base = warp ? sh[warp - 1] : 0;
    *total = sh[31];
    __syncthreads();
    return base + v - x;
}

// One CTA per (sequence, KV head): the positions to keep, in order, into kept[item][0..min(len, budget)).  Of the middle
// positions the `need` heaviest are wanted: four rounds of a radix histogram over the weights' ordered bits give the key T
// of the last one taken and how many positions with exactly that key are taken, lowest positions first; a second pass over
// the positions compacts them.
__global__ void __launch_bounds__(SEL_NT)
paged_select_kernel(const PagedView c, const SeqView s, int budget, int sinks, int recent, int32_t* __restrict__ kept, int kept_stride,
                    int* flags)
{
    __shared__ int hist[256], sh[33], pick[2];
    const int seq = blockIdx.x / c.heads, head = blockIdx.x % c.heads, tid = threadIdx.x;
    const int n = paged_len(c, s, seq, flags);
    int32_t* out = kept + (long long)blockIdx.x * kept_stride;
    if (n <= budget) {
        for (int t = tid; t < n; t += SEL_NT) out[t] = t;
        return;
    }
    const int32_t* table = s.table + (long long)seq * s.stride;
    auto key_at = [&](int t) {
        const long long row = paged_row(table[t / c.page], c.n_pages, c.heads, c.page, head, t % c.page);
        if (row < 0) paged_flag(flags, PAGED_BAD_PAGE);
        return row < 0 ? weight_key(0.0f) : weight_key(c.w[row]);
    };
    const int lo = sinks, hi = n - recent;
    int need = budget - sinks - recent;
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int t = lo + tid; t < hi; t += SEL_NT) {
            const uint32_t key = key_at(t);
            if (shift == 24 || key >> (shift + 8) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int left = need, d = 255;
            while (d > 0 && hist[d] < left) left -= hist[d--];
            pick[0] = d;
            pick[1] = left;
        }
        __syncthreads();
        prefix = prefix << 8 | (uint32_t)pick[0];
        need = pick[1];
        __syncthreads();
    }
    // need == 0 from the start: no middle position is kept
    const bool any = budget > sinks + recent;
    int done = 0, ties = 0;
    for (int t0 = 0; t0 < n; t0 += SEL_NT) {
        const int t = t0 + tid;
        bool keep = t < n && (t < lo || t >= hi), tie = false;
        if (any && t >= lo && t < hi) {
            const uint32_t key = key_at(t);
            keep = key > prefix;
            tie = key == prefix;
        }
        int n_tie = 0, n_keep = 0;
        const int before = block_scan(tie ? 1 : 0, sh, &n_tie);
        if (tie && ties + before < need) keep = true;
        const int at = block_scan(keep ? 1 : 0, sh, &n_keep);
        if (keep) out[done + at] = t;
        done += n_keep;
        ties += n_tie;
    }
}

// Copies the kept rows: one warp per row of a (sequence, KV head), 16 bytes per lane of keys, then of values.
__global__ void __launch_bounds__(256)
paged_move_kernel(const PagedView c, const SeqView s, const int32_t* __restrict__ kept, int kept_stride, int budget, const PagedView d,
                  const int32_t* __restrict__ dst_table, long long dst_stride, int row_bytes, int32_t* __restrict__ len_out, int* flags)
{
    const int item = blockIdx.x, seq = item / c.heads, head = item % c.heads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int left = min(paged_len(c, s, seq, flags), budget);
    if (blockIdx.y == 0 && head == 0 && threadIdx.x == 0) len_out[seq] = left;
    for (int r = blockIdx.y * 8 + warp; r < left; r += gridDim.y * 8) {
        const int t = kept[(long long)item * kept_stride + r];
        const long long from = paged_row(s.table[(long long)seq * s.stride + t / c.page], c.n_pages, c.heads, c.page, head, t % c.page);
        const long long to = paged_row(dst_table[(long long)seq * dst_stride + r / d.page], d.n_pages, d.heads, d.page, head, r % d.page);
        if (from < 0 || to < 0) {
            if (lane == 0) paged_flag(flags, PAGED_BAD_PAGE);
            if (to < 0) continue;
        }
        for (int b = lane * 16; b < row_bytes; b += 512) {
            uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
            if (from >= 0) {
                x = *reinterpret_cast<const uint4*>((const char*)c.k + from * row_bytes + b);
                y = *reinterpret_cast<const uint4*>((const char*)c.v + from * row_bytes + b);
            }
            *reinterpret_cast<uint4*>((char*)d.k + to * row_bytes + b) = x;
            *reinterpret_cast<uint4*>((char*)d.v + to * row_bytes + b) = y;
        }
        if (lane == 0) d.w[to] = from >= 0 ? c.w[from] : 0.0f;
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
    NNB_REQUIRE(t->n_rows <= (size_t)INT32_MAX, "%s: more than 2^31 - 1 tokens", who);
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
                       (long long)t->q_out_stride, t->n_head, t->rope_ctx, t->d_row_start, t->d_pos, t->d_rope_cos, t->d_rope_sin, d_len_out};
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
    if (t->d_row_start && d_len_out) {
        paged_advance_kernel<<<(unsigned)ceil_div((size_t)s->n_seq, 256), 256, 0, e->stream>>>(cv, sv, t->d_row_start, d_len_out, e->dev_flags);
        e->launches++;
        NNB_CHECK_LAUNCH("paged_advance_kernel");
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
    paged_select_kernel<<<items, SEL_NT, 0, e->stream>>>(cv, sv, (int)budget, (int)sinks, (int)recent, kept, (int)keep, e->dev_flags);
    e->launches++;
    NNB_CHECK_LAUNCH("paged_select_kernel");
    const size_t want = ceil_div((size_t)e->sm_count * 8, items), most = ceil_div(keep, 8);
    const int row_bytes = cv.pitch * (src->dtype == NNB_F32 ? 4 : 2);
    paged_move_kernel<<<dim3(items, (unsigned)(want < most ? want : most)), 256, 0, e->stream>>>(
        cv, sv, kept, (int)keep, (int)budget, dv, d_dst_table, (long long)dst_table_stride, row_bytes, d_len_out, e->dev_flags);
    e->launches++;
    NNB_CHECK_LAUNCH("paged_move_kernel");
    return NNB_OK;
}

}  // extern "C"
