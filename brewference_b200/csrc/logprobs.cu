// logprobs.cu — log probabilities of given tokens, the entropy of each row
// of logits and its top alternatives, in one pass over the logits:
//   lse = r + log z,  log p_i = (x_i - r) - log z,
//   H = -sum_i p_i log p_i = log z - (sum_i (x_i - r) e^{x_i - r}) / z,
//   z = sum_i e^{x_i - r},  for any reference r near the maximum.
//
// Bound by the read of 4 bytes a logit (about 8 instructions each beside
// it).  A row is read by a cluster of 1 to 8 CTAs in 16-byte loads.  Each
// thread sums relative to a reference that it moves only when a logit is
// LP_LAZY above it; threads, warps, CTAs and the cluster (through
// distributed shared memory) join in a fixed order.
//
// Top alternatives: every warp keeps the 32 largest of its logits as sorted
// 64-bit keys (the logit's order, then the lower index), one a lane.  A logit
// is a candidate only when it beats the warp's own `top`-th and reaches the
// CTA's floor, which the warps make together three times a row; 32 candidates
// are sorted and joined with the list at a time (an exchange and five steps).
// In rising rows every logit is a candidate.
//
// 1777 rows of 151936: 222 us with 20 alternatives (0.74 of a copy's rate), 171
// without (0.96).  (An insertion per candidate 508; a floor of each warp's own
// 357; of the CTA's, from sorted lists 310, from the lanes' largest 222.)
#include <algorithm>

#include "brew_internal.cuh"
#include "logprobs.cuh"

namespace brew {
namespace {

constexpr int LP_THREADS = 256;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_VEC = 4;               // float4s of a lane in flight
constexpr int LP_MAX_CLUSTER = 8;
constexpr int LP_FIRST = 8;             // keys of a warp that go into the CTA's floor
constexpr float LP_LAZY = 10.0f;
constexpr float LP_LOW = -110.0f;       // e^-110 is 0 in fp32: differences (-inf among them) stop here
constexpr float LOG2E = 1.44269504088896341f;

static_assert(LP_WARPS * LP_FIRST == 64, "the floor is made of two lists of 32");

using Key = unsigned long long;

// Larger logits first; a NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t order_bits(float v) {
    if (v != v) v = -INFINITY;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t b) {
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ Key order_key(float v, int i) {
    return (Key)order_bits(v) << 32 | (0xFFFFFFFFu - (uint32_t)i);
}

__device__ __forceinline__ float lp_exp(float y) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y * LOG2E));
    return e;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// z and zy = sum (x - r) e^(x - r) relative to r (-inf: nothing yet).
struct LpStat {
    float r, z, zy;
};

__device__ __forceinline__ void lp_move(LpStat& s, float r) {   // to the reference r
    const float d = s.r - r, e = expf(d);
    s.zy = e == 0.0f ? 0.0f : e * (s.zy + d * s.z);
    s.z *= e;
    s.r = r;
}
__device__ __forceinline__ LpStat lp_join(LpStat a, LpStat b) {
    if (a.r == -INFINITY || b.r == -INFINITY) {   // one side has no logit over -inf: its z is 0, or NaN
        LpStat s = a.r == -INFINITY ? b : a;
        const float other = a.r == -INFINITY ? a.z : b.z;
        s.z += other;
        s.zy += other;
        return s;
    }
    const float r = fmaxf(a.r, b.r);
    lp_move(a, r);
    lp_move(b, r);
    return {r, a.z + b.z, a.zy + b.zy};
}

// The 32 largest of two lists of 32 (a lane holds a key of each, largest in
// lane 0), sorted.
template <class T>
__device__ __forceinline__ T lp_merge(T a, T b, int lane) {
    const T o = __shfl_sync(0xffffffffu, b, 31 - lane);
    T k = a > o ? a : o;   // the larger half of both, rising and then falling
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) {
        const T v = __shfl_xor_sync(0xffffffffu, k, w);
        k = ((lane & w) == 0) == (k > v) ? k : v;
    }
    return k;
}

// The lanes' values sorted, the largest in lane 0.
template <class T>
__device__ __forceinline__ T lp_sort(T k, int lane) {
#pragma unroll
    for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
        for (int w = n >> 1; w > 0; w >>= 1) {
            const T v = __shfl_xor_sync(0xffffffffu, k, w);
            const bool down = n == 32 || (lane & n) == 0;   // this run falls
            k = ((lane & w) == 0) == ((k > v) == down) ? k : v;
        }
    return k;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
// The address of `p` (in this CTA's shared memory) in the cluster's CTA r.
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t r) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(r));
    return a;
}

template <bool TOP>
__global__ void __launch_bounds__(LP_THREADS, 4) logprobs_kernel(const __grid_constant__ LogprobsParams p, int cluster) {
    __shared__ LpStat stat[LP_WARPS], cstat[LP_MAX_CLUSTER];   // the warps'; the CTAs' (in rank 0)
    __shared__ Key best[TOP ? LP_WARPS : 1][32], cbest[TOP ? LP_MAX_CLUSTER : 1][32];
    __shared__ Key waiting[TOP ? LP_WARPS : 1][TOP ? 32 + 128 : 1];
    __shared__ int s_wait[LP_WARPS];
    __shared__ uint32_t s_first[LP_WARPS * LP_FIRST], s_floor;   // order bits: the warps' first keys; `top` are at or above
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = cluster > 1 ? cluster_rank() : 0;
    const int64_t row = blockIdx.x / cluster;
    const float* x = p.logits + row * p.ld;
    // float4s from the row's first 16-byte boundary on: this CTA's are [q0, q1)
    const int head = min(p.vocab, (int)((0 - ((uintptr_t)x >> 2)) & 3));
    const int quads = (p.vocab - head) / 4;
    const int q0 = (int)((int64_t)quads * rank / cluster), q1 = (int)((int64_t)quads * (rank + 1) / cluster);
    if (cluster > 1) cluster_arrive();   // every CTA runs before rank 0's memory is written
    if (TOP) {
        if (tid == 0) s_floor = 0;
        for (int k = tid; k < LP_WARPS * 160; k += LP_THREADS) (&waiting[0][0])[k] = 0;
        if (tid < LP_WARPS) s_wait[tid] = 0;
        __syncthreads();
    }

    LpStat s = {-INFINITY, 0.0f, 0.0f};
    Key mine = 0;                 // the lane's key of the warp's list
    uint32_t own = 0;             // order bits of its `top`-th key (0: it has fewer)
    auto raise = [&](float v) {   // v: a maximum that the sums are to hold
        if (v > s.r + LP_LAZY) {
            if (s.r == -INFINITY) s.r = v;   // z and zy are 0 (or NaN) so far
            else lp_move(s, v);
        }
    };
    auto add = [&](float v) {
        const float y = max_nan(v - s.r, LP_LOW), e = lp_exp(y);
        s.z += e;
        s.zy += e * y;
    };
    Key* wait = waiting[TOP ? warp : 0];
    auto settle = [&]() {         // after the list has changed
        own = (uint32_t)(__shfl_sync(0xffffffffu, mine, p.top - 1) >> 32);
    };
    auto take = [&]() {           // all that wait, 32 at a time, into the list
        __syncwarp();
        int n = s_wait[warp];
        __syncwarp();
        for (; n > 10; n -= 32) {
            const int at = max(n, 32) - 32 + lane;
            const Key k = at < n ? wait[at] : 0;
            mine = lp_merge(mine, lp_sort(k, lane), lane);
        }
        for (; n > 0; --n) {      // a few are quicker one by one
            const Key c = wait[n - 1];
            const int at = __popc(__ballot_sync(0xffffffffu, mine > c));
            const Key up = __shfl_up_sync(0xffffffffu, mine, 1);
            mine = lane < at ? mine : lane == at ? c : up;
        }
        __syncwarp();
        if (lane == 0) s_wait[warp] = 0;
        __syncwarp();
        settle();
    };
    // a lane's candidates (c[j] where bit j of `is`), indexes i, i + 1, ...; their order does not matter
    auto append = [&](const float (&c)[4], uint32_t is, int i) {
        int at = atomicAdd(&s_wait[warp], __popc(is));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (is >> j & 1) wait[at++] = order_key(c[j], i + j);
    };
    // the CTA's floor: the `top`-th of the first keys of its warps' lists (sorted, a lane each; 0: none)
    auto make_floor = [&](uint32_t k) {
        if (lane < LP_FIRST) s_first[lane * LP_WARPS + warp] = k;
        __syncthreads();
        if (warp == 0) {
            const uint32_t f = lp_merge(lp_sort(s_first[lane], lane), lp_sort(s_first[lane + 32], lane), lane);
            if (lane == p.top - 1) s_floor = max(s_floor, f);
        }
        __syncthreads();
    };
    // the few logits before the first float4 and behind the last one; those behind it have the row's highest indexes, so
    // they become candidates last (the list drops a later equal of its `top`-th)
    if (warp == 0 && (rank == 0 || rank == (uint32_t)cluster - 1)) {
        const int i = lane < 4 ? lane : head + 4 * quads + lane - 4;
        const bool is = lane < 8 && (lane < 4 ? rank == 0 && lane < head : rank == (uint32_t)cluster - 1 && i < p.vocab);
        const float v = is ? x[i] : -INFINITY;
        raise(v);
        if (is && s.r == -INFINITY) s.z += v - v == 0.0f || v == -INFINITY ? 0.0f : v - v;   // a NaN alone
        else if (is) add(v);
        if (TOP && is && lane < 4) {
            const float c[4] = {v, 0, 0, 0};
            append(c, 1, i);
        }
    }
    const float4* xq = reinterpret_cast<const float4*>(x + head);
    const int rounds = (q1 - q0 + LP_THREADS * LP_VEC - 1) / (LP_THREADS * LP_VEC);
    for (int round = 0; round < rounds; ++round) {
        const int b = q0 + (round * LP_WARPS + warp) * 32 * LP_VEC;
        float4 v[LP_VEC];
#pragma unroll
        for (int k = 0; k < LP_VEC; ++k) {
            const int q = b + 32 * k + lane;
            v[k] = q < q1 ? __ldcs(xq + q) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        }
        float mx[LP_VEC];
#pragma unroll
        for (int k = 0; k < LP_VEC; ++k) mx[k] = fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w));
        const float top4 = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        raise(top4);
        if (s.r != -INFINITY) {
#pragma unroll
            for (int k = 0; k < LP_VEC; ++k) {
                add(v[k].x); add(v[k].y); add(v[k].z); add(v[k].w);
            }
        } else {   // -inf or NaN all of them
#pragma unroll
            for (int k = 0; k < LP_VEC; ++k) {
                const bool nan = v[k].x != v[k].x || v[k].y != v[k].y || v[k].z != v[k].z || v[k].w != v[k].w;
                if (nan) s.z = s.zy = __uint_as_float(0x7fffffffu);
            }
        }
        if (TOP) {
            // before the first candidates: a floor from the lanes' largest
            if (round == 0) make_floor(lp_sort(top4 > -INFINITY ? order_bits(top4) : 0u, lane));
            // Candidates lie above the warp's own `top`-th (an equal one that comes later has a higher index) and not
            // below the CTA's floor; without either every logit is one.
            const uint32_t least = max(own + (own != 0), s_floor);
            const float floor = order_value(least);
            uint32_t any = 0;   // bit k: v[k] has one
#pragma unroll
            for (int k = 0; k < LP_VEC; ++k) any |= least == 0 || mx[k] >= floor ? 1u << k : 0u;
            any = __reduce_or_sync(0xffffffffu, any);
            for (int k = 0; any; ++k, any >>= 1) {
                if (any & 1) {
                    const float c[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
                    const int q = b + 32 * k + lane;
                    uint32_t is = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) is |= least == 0 || c[j] >= floor ? 1u << j : 0;
                    if (is && q < q1) append(c, is, head + 4 * q);
                    __syncwarp();
                    if (s_wait[warp] >= 32) take();
                }
#pragma unroll
                for (int n = 0; n + 1 < LP_VEC; ++n) v[n] = v[n + 1];
            }
            // after 4 and 13 rounds: a floor from the warps' lists
            if ((round == 3 || round == 12) && round + 1 < rounds) {
                take();
                make_floor((uint32_t)(mine >> 32));
            }
        }
    }
    if (TOP) {
        const int i = head + 4 * quads + lane;
        if (warp == 0 && rank == (uint32_t)cluster - 1 && lane < 4 && i < p.vocab) {
            const float c[4] = {x[i], 0, 0, 0};
            append(c, 1, i);
        }
        take();
    }

    // ---- joins: lanes, warps, CTAs
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) {
        LpStat o;
        o.r = __shfl_xor_sync(0xffffffffu, s.r, w);
        o.z = __shfl_xor_sync(0xffffffffu, s.z, w);
        o.zy = __shfl_xor_sync(0xffffffffu, s.zy, w);
        s = lane & w ? lp_join(o, s) : lp_join(s, o);
    }
    if (lane == 0) stat[warp] = s;
    if (TOP) best[warp][lane] = mine;
    __syncthreads();
    if (TOP) {
        for (int h = LP_WARPS / 2; h > 0; h >>= 1) {
            if (warp < h) best[warp][lane] = lp_merge(best[warp][lane], best[warp + h][lane], lane);
            __syncthreads();
        }
    }
    if (tid == 0) {
        s = stat[0];
        for (int w = 1; w < LP_WARPS; ++w) s = lp_join(s, stat[w]);
        stat[0] = s;
    }
    if (cluster > 1) {   // to rank 0
        cluster_wait();
        __syncthreads();
        if (warp == 0) {
            if (lane == 0) {
                const uint32_t a = cluster_addr(&cstat[rank], 0);
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(stat[0].r) : "memory");
                asm volatile("st.shared::cluster.f32 [%0 + 4], %1;" ::"r"(a), "f"(stat[0].z) : "memory");
                asm volatile("st.shared::cluster.f32 [%0 + 8], %1;" ::"r"(a), "f"(stat[0].zy) : "memory");
            }
            if (TOP)
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_addr(&cbest[rank][lane], 0)), "l"(best[0][lane])
                             : "memory");
        }
        cluster_arrive();   // releases the stores
        cluster_wait();     // and acquires them
        if (rank != 0) return;
    }
    if (warp != 0) return;
    if (cluster > 1) {
        s = cstat[0];
        for (int c = 1; c < cluster; ++c) s = lp_join(s, cstat[c]);
    } else {
        s = stat[0];
    }
    const bool none = s.r == -INFINITY && s.z == s.z;   // no token has a probability
    const float lz = logf(s.z);
    auto logp = [&](float v) { return none ? -INFINITY : (v - s.r) - lz; };
    if (lane == 0) {
        if (p.logprob) {
            const int t = p.tokens[row];
            p.logprob[row] = t >= 0 && t < p.vocab ? logp(x[t]) : __uint_as_float(0x7fffffffu);
        }
        if (p.entropy) p.entropy[row] = none ? 0.0f : lz - s.zy / s.z;
    }
    if (TOP) {
        Key k = cluster > 1 ? cbest[0][lane] : best[0][lane];
        for (int c = 1; c < cluster; ++c) k = lp_merge(k, cbest[c][lane], lane);
        if (lane < p.top) {
            p.top_ids[row * p.top + lane] = (int32_t)(0xFFFFFFFFu - (uint32_t)k);
            p.top_logprobs[row * p.top + lane] = logp(order_value((uint32_t)(k >> 32)));
        }
    }
}

}  // namespace

int logprobs_launch(const LogprobsParams& p, cudaStream_t s) {
    // four CTAs an SM: few rows are shared by a cluster each (no less than 2048 logits a CTA)
    int cluster = 1;
    while (cluster < LP_MAX_CLUSTER && (int64_t)p.rows * cluster * 2 <= 4 * 148 && p.vocab / (cluster * 2) >= 2048)
        cluster *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.rows * cluster);
    cfg.blockDim = dim3(LP_THREADS);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    if (p.top > 0) BREW_CUDA(cudaLaunchKernelEx(&cfg, logprobs_kernel<true>, p, cluster));
    else BREW_CUDA(cudaLaunchKernelEx(&cfg, logprobs_kernel<false>, p, cluster));
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
