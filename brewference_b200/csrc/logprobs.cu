// logprobs.cu — log probabilities of given tokens, the entropy of each row
// of logits and its top alternatives:
//   lse = log sum_i e^{x_i},  log p_i = x_i - lse,  H = -sum_i p_i log p_i
#include "brew_internal.cuh"
#include "logprobs.cuh"

namespace brew {
namespace {

constexpr int LP_THREADS = 512;

__device__ __forceinline__ float cta_max(float v, float* red) {
    v = warp_max(v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = red[0];
    for (int w = 1; w < LP_THREADS / 32; ++w) t = fmaxf(t, red[w]);
    __syncthreads();
    return t;
}

__device__ __forceinline__ float cta_add(float v, float* red) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
    for (int w = 0; w < LP_THREADS / 32; ++w) t += red[w];
    __syncthreads();
    return t;
}

// Order of the alternatives: larger logits first, equal ones by index; a NaN
// counts as -inf.
__device__ __forceinline__ unsigned long long order_key(float v, int i) {
    if (v != v) v = -INFINITY;
    v += 0.0f;   // -0 equals 0
    uint32_t b = __float_as_uint(v);
    b = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (unsigned long long)b << 32 | (0xFFFFFFFFu - (uint32_t)i);
}

__device__ __forceinline__ float key_value(unsigned long long k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

// One CTA per row, one pass for each statistic and each alternative.
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(const __grid_constant__ LogprobsParams p) {
    __shared__ float red[LP_THREADS / 32];
    __shared__ unsigned long long kred[LP_THREADS / 32];
    const int64_t r = blockIdx.x;
    const float* x = p.logits + r * p.ld;
    float m = -INFINITY, nan = 0.0f;
    for (int i = threadIdx.x; i < p.vocab; i += LP_THREADS) {
        m = fmaxf(m, x[i]);
        if (x[i] != x[i]) nan = x[i];
    }
    m = cta_max(m, red);
    nan = cta_add(nan, red);
    float z = 0.0f, zy = 0.0f;
    for (int i = threadIdx.x; i < p.vocab; i += LP_THREADS) {
        const float y = x[i] - m, e = expf(y);
        z += e;
        if (e > 0.0f) zy += e * y;
    }
    z = cta_add(z, red) + nan;
    zy = cta_add(zy, red);
    const bool none = m == -INFINITY && nan == 0.0f;   // no token has a probability
    const float lz = logf(z);
    auto logp = [&](float v) { return none ? -INFINITY : (v - m) - lz; };
    if (threadIdx.x == 0) {
        if (p.logprob) {
            const int t = p.tokens[r];
            p.logprob[r] = t >= 0 && t < p.vocab ? logp(x[t]) : __uint_as_float(0x7fffffffu);
        }
        if (p.entropy) p.entropy[r] = none ? 0.0f : lz - zy / z;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top; ++k) {
        unsigned long long best = 0;
        for (int i = threadIdx.x; i < p.vocab; i += LP_THREADS) {
            const unsigned long long key = order_key(x[i], i);
            if (key < last && key > best) best = key;
        }
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if ((threadIdx.x & 31) == 0) kred[threadIdx.x >> 5] = best;
        __syncthreads();
        for (int w = 0; w < LP_THREADS / 32; ++w) best = max(best, kred[w]);
        __syncthreads();
        last = best;
        if (threadIdx.x == 0) {
            if (p.top_ids) p.top_ids[r * p.top + k] = (int32_t)(0xFFFFFFFFu - (uint32_t)best);
            if (p.top_logprobs) p.top_logprobs[r * p.top + k] = logp(key_value(best));
        }
    }
}

}  // namespace

int logprobs_launch(const LogprobsParams& p, cudaStream_t s) {
    logprobs_kernel<<<p.rows, LP_THREADS, 0, s>>>(p);
    BREW_CUDA(cudaGetLastError());
    count_launch();
    return BREW_OK;
}

}  // namespace brew

using namespace brew;

extern "C" int brew_logprobs_dev(const float* logits, int64_t ld, int32_t vocab, int32_t rows, const int32_t* tokens,
                                 float* logprob, float* entropy, int32_t top, int32_t* top_ids, float* top_logprobs,
                                 void* stream) {
    BREW_CHECK(logits, BREW_ERR_INVALID_ARG, "logits is null");
    BREW_CHECK(vocab > 0 && rows >= 0, BREW_ERR_INVALID_ARG, "vocab %d, rows %d", vocab, rows);
    BREW_CHECK(ld >= vocab, BREW_ERR_INVALID_ARG, "row stride %lld under the vocabulary of %d", (long long)ld, vocab);
    BREW_CHECK((tokens != nullptr) == (logprob != nullptr), BREW_ERR_INVALID_ARG, "tokens and logprob are given together");
    BREW_CHECK(top >= 0 && top <= BREW_MAX_TOP && top <= vocab, BREW_ERR_INVALID_ARG,
               "%d alternatives of %d tokens (at most %d)", top, vocab, BREW_MAX_TOP);
    BREW_CHECK(top == 0 || (top_ids && top_logprobs), BREW_ERR_INVALID_ARG, "top_ids and top_logprobs must be given");
    BREW_CHECK((((uintptr_t)logits | (uintptr_t)tokens | (uintptr_t)logprob | (uintptr_t)entropy | (uintptr_t)top_ids |
                 (uintptr_t)top_logprobs) & 3) == 0, BREW_ERR_INVALID_ARG, "unaligned arrays");
    BREW_CHECK(logprob || entropy || top > 0, BREW_ERR_INVALID_ARG, "nothing is asked");
    if (rows == 0) return BREW_OK;
    DeviceScope ds;
    if (ds.rc) return ds.rc;
    const LogprobsParams p = {logits, ld, vocab, rows, tokens, logprob, entropy, top, top_ids, top_logprobs};
    return logprobs_launch(p, static_cast<cudaStream_t>(stream));
}
