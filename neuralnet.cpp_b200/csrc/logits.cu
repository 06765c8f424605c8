// logits.cu — adjustment of a batch of logits before sampling: bias, penalties for repeated tokens, allowed-token masks.
#include <math.h>

#include "device_math.cuh"
#include "paged.cuh"

namespace nnb {

struct LogitsArgs {
    const int32_t *history, *history_len, *prompt_len;
    long long history_stride;
    int max_history, window;
    const float *repeat, *presence, *frequency, *bias;
    long long bias_stride;
    const uint32_t* allowed;
    long long allowed_stride;
};

__device__ __forceinline__ float logit_f32(float x) { return x; }
__device__ __forceinline__ float logit_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void logit_put(float* p, float x) { *p = x; }
__device__ __forceinline__ void logit_put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

constexpr uint32_t SEEN = 0x80000000u;

// One CTA per (slice of SLICE token ids, sequence).  Every load that depends on nothing is requested first: the thread's
// logits, their bias and mask, and the first ids of the history.  Then the CTA walks the sequence's history once and counts,
// in shared memory, the ids that fall into its slice (low bits: occurrences from the prompt's end on; top bit: inside the
// repeat window).  Integer counts do not depend on the order of the atomics.  Bound by reading and writing the logits; the
// history is read once per slice, from L2.  Slices begin where the row is 16-byte aligned, whatever the vocabulary.  With
// penalties alone and in place (SPARSE) only what the history touches is read and written.
template <typename T, int SLICE, int NT, bool SPARSE>
__global__ void __launch_bounds__(NT) adjust_logits_kernel(const T* in, T* out, int vocab, long long stride, long long out_stride, const LogitsArgs a)
{
    constexpr int VEC = 16 / sizeof(T), PER = SLICE / (NT * VEC), IDS = 2048 / NT;
    __shared__ __align__(16) uint32_t count[SLICE];
    pdl_wait();
    pdl_launch();
    const int s = blockIdx.x, tid = threadIdx.x;
    const T* src = in + (long long)s * stride;
    T* dst = out + (long long)s * out_stride;
    const int first = (int)(blockIdx.y * SLICE) - (int)((uintptr_t)src / sizeof(T) % VEC);  // id of the slice's first place
    const float* bias = a.bias ? a.bias + (long long)s * a.bias_stride : nullptr;
    const uint32_t* allowed = a.allowed ? a.allowed + (long long)s * a.allowed_stride : nullptr;
    const int32_t* ids = a.history + (long long)s * a.history_stride;
    const int words = (vocab + 31) / 32;
    auto id_of = [&](int j) { return first + (j * NT + tid) * VEC; };
    auto whole = [&](int id) { return id >= 0 && id + VEC <= vocab; };
    auto bias_vec = [&](int id) { return bias && whole(id) && (uintptr_t)(bias + id) % 16 == 0; };
    // what the thread's vectors need; vectors that are not whole are read where they are used
    uint4 raw[PER];
    float4 b4[SPARSE ? 1 : PER][VEC / 4];
    uint32_t word0[PER], word1[PER];  // the mask words of the vector's first and last id (mostly the same)
    if (!SPARSE) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int id = id_of(j);
            if (whole(id)) raw[j] = *reinterpret_cast<const uint4*>(src + id);
            if (bias_vec(id))
#pragma unroll
                for (int i = 0; i < VEC / 4; ++i) b4[j][i] = *reinterpret_cast<const float4*>(bias + id + 4 * i);
            if (allowed) {
                word0[j] = allowed[min(max(id, 0) >> 5, words - 1)];
                word1[j] = allowed[min(max(id + VEC - 1, 0) >> 5, words - 1)];
            }
        }
    }
    const float r = a.repeat ? a.repeat[s] : 1.0f, pres = a.presence ? a.presence[s] : 0.0f, freq = a.frequency ? a.frequency[s] : 0.0f;
    const bool rep = r > 0.0f && r != 1.0f;
    if (a.history) {
        int early[IDS];
#pragma unroll
        for (int u = 0; u < IDS; ++u) early[u] = u * NT + tid < a.max_history ? ids[u * NT + tid] : -1;
        const int n = min(max(a.history_len[s], 0), a.max_history);
        const int prompt = a.prompt_len ? a.prompt_len[s] : 0, from = a.window > 0 ? n - a.window : 0;
        for (int i = tid * 4; i < SLICE; i += 4 * NT) *reinterpret_cast<uint4*>(count + i) = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
        auto note = [&](int t, int id) {
            if ((unsigned)(id - first) >= (unsigned)SLICE || (unsigned)id >= (unsigned)vocab || t >= n) return;
            if (t >= from && !(count[id - first] & SEEN)) atomicOr(&count[id - first], SEEN);
            if (t >= prompt) atomicAdd(&count[id - first], 1u);
        };
#pragma unroll
        for (int u = 0; u < IDS; ++u) note(u * NT + tid, early[u]);
#pragma unroll 4
        for (int t = IDS * NT + tid; t < n; t += NT) note(t, ids[t]);
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int at = (j * NT + tid) * VEC, id = first + at;
        if (id >= vocab || id + VEC <= 0) continue;
        uint32_t c[VEC], any = 0;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            c[i] = a.history ? count[at + i] : 0u;
            any |= c[i];
        }
        if (SPARSE && !any) continue;
        float x[VEC];
        if (whole(id)) {
            if (SPARSE) raw[j] = *reinterpret_cast<const uint4*>(src + id);
            const T* e = reinterpret_cast<const T*>(&raw[j]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] = logit_f32(e[i]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] = id + i >= 0 && id + i < vocab ? logit_f32(src[id + i]) : 0.0f;
        }
        if (!SPARSE && bias) {
            if (bias_vec(id)) {
                const float* b = reinterpret_cast<const float*>(b4[j]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[i] = __fadd_rn(x[i], b[i]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (id + i >= 0 && id + i < vocab) x[i] = __fadd_rn(x[i], bias[id + i]);
            }
        }
        if (any) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (c[i] == 0) continue;  // few ids occur: a warp mostly has one of its lanes' four here
                const uint32_t k = c[i] & ~SEEN;
                if (rep && (c[i] & SEEN)) x[i] = x[i] > 0.0f ? __fdiv_rn(x[i], r) : __fmul_rn(x[i], r);
                if (k) x[i] = __fsub_rn(x[i], __fadd_rn(__fmul_rn(freq, (float)k), pres));
            }
        }
        if (!SPARSE && allowed) {
            // (ids in front of the row have no bits; where both words are the same one, the second is not reached)
            const uint32_t bits = id < 0 ? word0[j] << -id : __funnelshift_r(word0[j], word1[j], id & 31);
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (!(bits >> i & 1u)) x[i] = -INFINITY;
        }
        if (whole(id) && (uintptr_t)(dst + id) % 16 == 0) {
            uint4 packed;
            T* e = reinterpret_cast<T*>(&packed);
#pragma unroll
            for (int i = 0; i < VEC; ++i) logit_put(e + i, x[i]);
            *reinterpret_cast<uint4*>(dst + id) = packed;
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (id + i >= 0 && id + i < vocab) logit_put(dst + id + i, x[i]);
        }
    }
}

template <typename T, int SLICE, int NT>
static nnb_status launch_adjust_slice(nnb_engine* e, const T* in, T* out, size_t n_seq, size_t vocab, size_t stride, size_t out_stride, const LogitsArgs& a)
{
    constexpr int VEC = 16 / sizeof(T);
    const bool sparse = in == out && !a.bias && !a.allowed;
    if (sparse && !a.history) return NNB_OK;  // nothing to change
    auto kern = sparse ? adjust_logits_kernel<T, SLICE, NT, true> : adjust_logits_kernel<T, SLICE, NT, false>;
    // (a row may begin VEC - 1 places behind its slices)
    PdlOn pdl(e);
    NNB_CUDA(launch_ex(e, kern, dim3((unsigned)n_seq, (unsigned)ceil_div(vocab + VEC - 1, SLICE)), dim3(NT), 0, in, out, (int)vocab, (long long)stride,
                       (long long)out_stride, a));
    e->launches++;
    return NNB_OK;
}
template <typename T>
static nnb_status launch_adjust(nnb_engine* e, const T* in, T* out, size_t n_seq, size_t vocab, size_t stride, size_t out_stride, const LogitsArgs& a)
{
    // Long slices read the history less often, short ones fill the GPU when there are few rows.  Slices of 4096 by 512 threads
    // and of 2048 by 256 take 33.4 and 39.1 us for 128 x 128256 f32 logits, 3.4 and 3.2 us for 4 x 32000 bf16.
    if (n_seq * ceil_div(vocab, 4096) >= 2 * (size_t)e->sm_count) return launch_adjust_slice<T, 4096, 512>(e, in, out, n_seq, vocab, stride, out_stride, a);
    return launch_adjust_slice<T, 2048, 256>(e, in, out, n_seq, vocab, stride, out_stride, a);
}

}  // namespace nnb

using namespace nnb;

extern "C" nnb_status nnb_adjust_logits(nnb_engine* e, const void* d_logits, int dtype, size_t n_seq, size_t vocab, size_t stride,
                                        const nnb_logits_config* cfg, void* d_out, size_t out_stride)
{
    const char* who = "adjust_logits";
    NNB_REQUIRE(cfg && (n_seq == 0 || (d_logits && d_out)), "%s: NULL argument", who);
    NNB_REQUIRE(dtype == NNB_F32 || dtype == NNB_BF16, "%s: dtype %d is neither f32 nor bf16", who, dtype);
    NNB_REQUIRE(vocab > 0 && vocab <= (1u << 26) && n_seq <= (size_t)INT32_MAX, "%s: bad shape (%zu sequences, %zu tokens)", who, n_seq, vocab);
    NNB_REQUIRE(n_seq <= 1 || (stride >= vocab && out_stride >= vocab), "%s: rows overlap", who);
    NNB_REQUIRE(d_logits != d_out || stride == out_stride, "%s: in place needs one stride", who);
    const size_t item = dtype == NNB_F32 ? 4 : 2;
    NNB_REQUIRE(((uintptr_t)d_logits | (uintptr_t)d_out) % item == 0, "%s: misaligned logits", who);
    NNB_REQUIRE((cfg->d_history == nullptr) == (cfg->d_history_len == nullptr), "%s: history and its lengths go together", who);
    NNB_REQUIRE(cfg->d_history || !(cfg->d_repeat || cfg->d_presence || cfg->d_frequency), "%s: penalties need a history", who);
    NNB_REQUIRE(cfg->max_history <= (size_t)INT32_MAX && (n_seq <= 1 || cfg->history_stride >= cfg->max_history), "%s: rows of the history overlap", who);
    NNB_REQUIRE(cfg->repeat_window >= 0, "%s: negative repeat window", who);
    NNB_REQUIRE(!cfg->d_bias || n_seq <= 1 || cfg->bias_stride == 0 || cfg->bias_stride >= vocab, "%s: rows of the bias overlap", who);
    NNB_REQUIRE(!cfg->d_allowed || n_seq <= 1 || cfg->allowed_stride == 0 || cfg->allowed_stride >= ceil_div(vocab, 32), "%s: rows of the mask overlap", who);
    NNB_REQUIRE(e, "%s: engine is NULL", who);
    if (n_seq == 0) return NNB_OK;
    DeviceScope dev(e->device);
    const bool penalties = cfg->d_repeat || cfg->d_presence || cfg->d_frequency;
    const LogitsArgs a{penalties ? cfg->d_history : nullptr, cfg->d_history_len, cfg->d_prompt_len, (long long)cfg->history_stride, (int)cfg->max_history,
                       cfg->repeat_window, cfg->d_repeat, cfg->d_presence, cfg->d_frequency, cfg->d_bias, (long long)cfg->bias_stride, cfg->d_allowed,
                       (long long)cfg->allowed_stride};
    if (dtype == NNB_F32) return launch_adjust<float>(e, (const float*)d_logits, (float*)d_out, n_seq, vocab, stride, out_stride, a);
    return launch_adjust<__nv_bfloat16>(e, (const __nv_bfloat16*)d_logits, (__nv_bfloat16*)d_out, n_seq, vocab, stride, out_stride, a);
}
