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
__device__ __forceinline__ void store_one(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_one(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// One CTA per (sequence, query head), its four warps on every fourth position each; a lane holds pairs of features.
template <typename TQ, typename TC>
__global__ void __launch_bounds__(128) paged_decode_kernel(const PagedView c, const SeqView s, const DecodeArgs a, float* __restrict__ lse_out, int* flags)
{
    __shared__ float part[4][258];
    const int seq = blockIdx.x / a.n_head, h = blockIdx.x % a.n_head, hk = h / a.group;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = paged_len(c, s, seq, flags);
    const TQ* q = (const TQ*)a.q + (long long)seq * a.q_stride + (long long)h * c.dk;
    float2 qf[4], o[4];
    for (int i = 0; i < 4; ++i) {
        const int f = 2 * lane + 64 * i;
        qf[i] = f < c.dk ? load_pair(q + f) : make_float2(0.0f, 0.0f);
        o[i] = make_float2(0.0f, 0.0f);
    }
    float m = -INFINITY, l = 0.0f;
    for (int t = warp; t < n; t += 4) {
        const long long row = paged_row(s.table[(long long)seq * s.stride + t / c.page], c.n_pages, c.heads, c.page, hk, t % c.page);
        if (row < 0) {
            if (lane == 0) paged_flag(flags, PAGED_BAD_PAGE);
            continue;
        }
        const TC* k = (const TC*)c.k + row * c.pitch;
        const TC* v = (const TC*)c.v + row * c.pitch;
        float x = 0.0f;
        for (int i = 0; i < 4; ++i)
            if (2 * lane + 64 * i < c.dk) {
                const float2 kf = load_pair(k + 2 * lane + 64 * i);
                x = fmaf(qf[i].x, kf.x, fmaf(qf[i].y, kf.y, x));
            }
        x = warp_sum(x) * a.scale;
        const float top = fmaxf(m, x), base = top == -INFINITY ? 0.0f : top;
        const float old = expf(m - base), p = expf(x - base);
        l = fmaf(l, old, p);
        for (int i = 0; i < 4; ++i)
            if (2 * lane + 64 * i < c.dk) {
                const float2 vf = load_pair(v + 2 * lane + 64 * i);
                o[i].x = fmaf(o[i].x, old, p * vf.x);
                o[i].y = fmaf(o[i].y, old, p * vf.y);
            }
        m = top;
    }
    for (int i = 0; i < 4; ++i)
        if (2 * lane + 64 * i < c.dk) {
            part[warp][2 * lane + 64 * i] = o[i].x;
            part[warp][2 * lane + 64 * i + 1] = o[i].y;
        }
    if (lane == 0) {
        part[warp][256] = m;
        part[warp][257] = l;
    }
    __syncthreads();
    float top = -INFINITY, total = 0.0f;
    for (int w = 0; w < 4; ++w) top = fmaxf(top, part[w][256]);
    const float base = top == -INFINITY ? 0.0f : top;
    for (int w = 0; w < 4; ++w) total = fmaf(part[w][257], expf(part[w][256] - base), total);
    for (int f = threadIdx.x; f < c.dk; f += 128) {
        float x = 0.0f;
        for (int w = 0; w < 4; ++w) x = fmaf(part[w][f], expf(part[w][256] - base), x);
        store_one((TQ*)a.out + (long long)blockIdx.x * c.dk + f, total == 0.0f ? 0.0f : x / total);
    }
    if (threadIdx.x == 0) lse_out[blockIdx.x] = total == 0.0f ? -INFINITY : base + logf(total);
}

// weight[t] += sum over the group of exp(x_t - lse): one CTA per (sequence, KV head), a warp per position
template <typename TQ, typename TC>
__global__ void __launch_bounds__(256) paged_weight_kernel(const PagedView c, const SeqView s, const DecodeArgs a, const float* __restrict__ lse, int* flags)
{
    const int seq = blockIdx.x / c.heads, hk = blockIdx.x % c.heads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = paged_len(c, s, seq, flags);
    for (int t = warp; t < n; t += 8) {
        const long long row = paged_row(s.table[(long long)seq * s.stride + t / c.page], c.n_pages, c.heads, c.page, hk, t % c.page);
        if (row < 0) continue;
        const TC* k = (const TC*)c.k + row * c.pitch;
        float sum = 0.0f;
        for (int g = 0; g < a.group; ++g) {
            const int h = hk * a.group + g;
            const TQ* q = (const TQ*)a.q + (long long)seq * a.q_stride + (long long)h * c.dk;
            float x = 0.0f;
            for (int f = 2 * lane; f < c.dk; f += 64) {
                const float2 kf = load_pair(k + f), qf = load_pair(q + f);
                x = fmaf(qf.x, kf.x, fmaf(qf.y, kf.y, x));
            }
            x = warp_sum(x) * a.scale;
            const float z = lse[(long long)seq * a.n_head + h];
            sum += z == -INFINITY ? 0.0f : expf(x - z);
        }
        if (lane == 0) atomicAdd(c.w + row, sum);
    }
}

template <typename TQ, typename TC>
static nnb_status launch_decode(nnb_engine* e, const PagedView& c, const SeqView& s, const DecodeArgs& a, bool accumulate, float* ws)
{
    float* lse = a.lse ? a.lse : ws;
    paged_decode_kernel<TQ, TC><<<(unsigned)(s.n_seq * a.n_head), 128, 0, e->stream>>>(c, s, a, lse, e->dev_flags);
    e->launches++;
    NNB_CHECK_LAUNCH("paged_decode_kernel");
    if (accumulate) {
        paged_weight_kernel<TQ, TC><<<(unsigned)(s.n_seq * c.heads), 256, 0, e->stream>>>(c, s, a, lse, e->dev_flags);
        e->launches++;
        NNB_CHECK_LAUNCH("paged_weight_kernel");
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
    (void)accumulate;
    if (!e || paged_check_cache("paged_attention_decode", c, &cv) != NNB_OK || paged_check_seqs("paged_attention_decode", c, s, &sv) != NNB_OK ||
        n_head == 0 || n_head % cv.heads != 0)
        return 0;
    return (size_t)sv.n_seq * n_head * sizeof(float) + 16;
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
    const bool acc = accumulate != 0;
    if (dtype == NNB_F32) {
        if (c->dtype == NNB_F32) return launch_decode<float, float>(e, cv, sv, a, acc, (float*)d_ws);
        return launch_decode<float, __nv_bfloat16>(e, cv, sv, a, acc, (float*)d_ws);
    }
    if (c->dtype == NNB_F32) return launch_decode<__nv_bfloat16, float>(e, cv, sv, a, acc, (float*)d_ws);
    return launch_decode<__nv_bfloat16, __nv_bfloat16>(e, cv, sv, a, acc, (float*)d_ws);
}

}  // extern "C"
