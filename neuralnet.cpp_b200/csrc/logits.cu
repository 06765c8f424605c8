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

// One CTA per (slice of SLICE token ids, sequence).  The CTA walks the sequence's history once and counts, in shared
// memory, the ids that fall into its slice (low bits: occurrences from the prompt's end on; top bit: inside the repeat
// window); integer counts do not depend on the order of the atomics.  Then it streams its logits through once.
template <typename T, int SLICE>
__global__ void __launch_bounds__(256) adjust_logits_kernel(const T* in, T* out, int vocab, long long stride, long long out_stride, const LogitsArgs a)
{
    __shared__ uint32_t count[SLICE];
    const int s = blockIdx.y, first = blockIdx.x * SLICE, tid = threadIdx.x;
    const int n_ids = min(SLICE, vocab - first);
    for (int i = tid; i < SLICE; i += 256) count[i] = 0;
    __syncthreads();
    if (a.history) {
        const int n = min(max(a.history_len[s], 0), a.max_history);
        const int prompt = a.prompt_len ? a.prompt_len[s] : 0, from = a.window > 0 ? n - a.window : 0;
        const int32_t* ids = a.history + (long long)s * a.history_stride;
        for (int t = tid; t < n; t += 256) {
            const int id = ids[t] - (ids[t] >= first ? first : 0);
            if (ids[t] < first || id >= n_ids) continue;
            if (t >= from) atomicOr(&count[id], SEEN);
            if (t >= prompt) atomicAdd(&count[id], 1u);
        }
    }
    __syncthreads();
    const float r = a.repeat ? a.repeat[s] : 1.0f, pres = a.presence ? a.presence[s] : 0.0f, freq = a.frequency ? a.frequency[s] : 0.0f;
    const bool rep = r > 0.0f && r != 1.0f;
    for (int i = tid; i < n_ids; i += 256) {
        const int id = first + i;
        float x = logit_f32(in[(long long)s * stride + id]);
        if (a.bias) x = __fadd_rn(x, a.bias[(long long)s * a.bias_stride + id]);
        const uint32_t c = count[i];
        if (rep && (c & SEEN)) x = x > 0.0f ? __fdiv_rn(x, r) : __fmul_rn(x, r);
        if (c & ~SEEN) x = __fsub_rn(x, __fadd_rn(__fmul_rn(freq, (float)(c & ~SEEN)), pres));
        if (a.allowed && !(a.allowed[(long long)s * a.allowed_stride + id / 32] >> (id % 32) & 1u)) x = -INFINITY;
        logit_put(out + (long long)s * out_stride + id, x);
    }
}

template <typename T>
static nnb_status launch_adjust(nnb_engine* e, const T* in, T* out, size_t n_seq, size_t vocab, size_t stride, size_t out_stride, const LogitsArgs& a)
{
    constexpr int SLICE = 4096;
    adjust_logits_kernel<T, SLICE><<<dim3((unsigned)ceil_div(vocab, SLICE), (unsigned)n_seq), 256, 0, e->stream>>>(in, out, (int)vocab, (long long)stride,
                                                                                                   (long long)out_stride, a);
    e->launches++;
    NNB_CHECK_LAUNCH("adjust_logits_kernel");
    return NNB_OK;
}

}  // namespace nnb

using namespace nnb;

extern "C" nnb_status nnb_adjust_logits(nnb_engine* e, const void* d_logits, int dtype, size_t n_seq, size_t vocab, size_t stride,
                                        const nnb_logits_config* cfg, void* d_out, size_t out_stride)
{
    const char* who = "adjust_logits";
    NNB_REQUIRE(cfg && (n_seq == 0 || (d_logits && d_out)), "%s: NULL argument", who);
    NNB_REQUIRE(dtype == NNB_F32 || dtype == NNB_BF16, "%s: dtype %d is neither f32 nor bf16", who, dtype);
    NNB_REQUIRE(vocab > 0 && vocab <= (1u << 30) && n_seq <= 65535, "%s: bad shape (%zu sequences, %zu tokens)", who, n_seq, vocab);
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
