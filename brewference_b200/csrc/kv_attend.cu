// kv_attend.cu — attention over the paged 4-bit K/V cache:
//   o = sum_t softmax_t(scale * q . k_t) v_t
// over the positions t <= the row's own (and > own - window).
//
// Arithmetic.  A cached value is (c - 8) d with a 4-bit code c and an fp16
// scale d of its block of 32.  Both products run on mma.m16n8k16 with the
// codes' exact c - 8 as one operand.  fp32 accuracy comes from the other
// operand, carried as two fp16 numbers (hi = fp16(x), lo = fp16(x - hi), 22
// bits together) in rows g and g + 8 of the tile, summed in fp32; 8 (row,
// head) pairs fill a tile.
//   scores   S = sum_b d_K[t][b] (sum_{i in b} q_i (c_ti - 8))
//   output   O = sum_t (p_t d_V[t][b]) (c_ti - 8)
// q, p and d_V are scaled by powers of two (q below 2^14, p and p d_V to 2^15
// at most), so that no part leaves fp16's range and little falls among its
// subnormals (2^-24 beside 2^13).  The softmax is online; its running maximum
// moves only when exceeded by 2^2, so O is rarely rescaled.
//
// Work split.  Units of 128 positions of one (sequence, kv head, 8 pairs),
// laid end to end over all sequences of the call; every CTA takes an equal
// run of units, whatever the lengths (read on the device: a captured graph
// follows them).  A run's first and last item may be shared with other CTAs:
// their partial results (max, sum, O) go to the workspace and the last CTA to
// arrive joins them in order.  Within a unit each warp streams its own
// 32-position tiles through a ring of shared-memory stages (bulk copies: the
// tile's K, V and scales are one run per page).
#include <algorithm>

#include "brew_internal.cuh"
#include "decode.cuh"
#include "kv.cuh"

namespace brew {
namespace {

constexpr int AT_WARPS = 4;
constexpr int AT_THREADS = 32 * AT_WARPS;
constexpr int AT_TILE = 32;                       // positions a warp handles at once
constexpr int AT_UNIT = AT_TILE * AT_WARPS;
constexpr int AT_PAIRS = 8;                       // (row, head) pairs of a tile
constexpr int AT_MAX_CTAS = 3 * 148;
constexpr float AT_LAZY = 2.0f;                   // log2 of how far p may exceed 1

template <int R>
struct AtShape {
    static constexpr int HD = 32 * R;
    static constexpr int TILE_BYTES = 2 * kv_group_bytes(R);
    static constexpr int STAGES = R <= 2 ? 6 : R == 3 ? 5 : R == 4 ? 4 : 3;
    static constexpr int RING = STAGES * TILE_BYTES;               // of a warp
    static constexpr int QFRAG = R == 8 ? R * 2 * 32 * 16 : 0;     // q fragments in shared memory
    static constexpr int BARS = AT_WARPS * RING + QFRAG;
    static constexpr int PREFIX = BARS + AT_WARPS * STAGES * 8;
    static constexpr int CTAS_PER_SM = R == 8 ? 2 : 3;
    static_assert(AT_PAIRS * (HD + 2) * 4 <= RING, "a warp's result fits its ring");
};

// ---- mma.m16n8k16 --------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                        const float (&c)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// x0, x1 as two pairs of fp16: the rounded values and what they leave.
__device__ __forceinline__ void split_half2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack_half2(x0 - f.x, x1 - f.y);
}

// The values c - 8 of the codes c in nibbles 0 and 4, 1 and 5, 2 and 6, 3 and
// 7 of w, as fp16 pairs: a nibble below the exponent of 1024 is 1024 + c (one
// place up 1024 + 16 c); one exact operation takes the rest off.  (A nibble
// alone, the subnormal c 2^-24, would save that operation, but mma aligns its
// products by their exponent fields and loses 7 bits of a subnormal's.)
__device__ __forceinline__ uint32_t code_bits(uint32_t w, uint32_t mask, uint32_t base) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(mask), "r"(base));   // w & mask | base
    return d;
}
// `base`: 0x64006400, a launch parameter so that it stays in a register and
// each step is one instruction (as a constant it took two: 64 more of 478 per
// 16 positions, and 6 % of the time).
__device__ __forceinline__ void unpack(uint32_t (&x)[4], uint32_t w, uint32_t base) {
    const uint32_t y = w >> 8;
    const uint32_t e0 = code_bits(w, 0x000F000Fu, base), e1 = code_bits(w, 0x00F000F0u, base);
    const uint32_t e2 = code_bits(y, 0x000F000Fu, base), e3 = code_bits(y, 0x00F000F0u, base);
    asm("sub.f16x2 %0, %1, %2;" : "=r"(x[0]) : "r"(e0), "r"(0x64086408u));                            // - 1032
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(x[1]) : "r"(e1), "r"(0x2C002C00u), "r"(0xD480D480u));   // / 16 - 72
    asm("sub.f16x2 %0, %1, %2;" : "=r"(x[2]) : "r"(e2), "r"(0x64086408u));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(x[3]) : "r"(e3), "r"(0x2C002C00u), "r"(0xD480D480u));
}

__device__ __forceinline__ float2 half2_bits(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Two fp32 numbers at a time.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\t"
        "mov.b64 {%0, %1}, x;}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// fp16 pairs.
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t fma_h2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t neg_h2(uint32_t a) {
    uint32_t d;
    asm("neg.f16x2 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// The larger magnitude, with some sign.
__device__ __forceinline__ uint32_t maxabs_h2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Words (u, 0 .. R - 1, lane) of a group's K or V quants.
template <int R>
__device__ __forceinline__ void load_words(uint32_t (&w)[R], const uint8_t* q, int u, int lane) {
    if constexpr (R % 4 == 0) {
#pragma unroll
        for (int c = 0; c < R / 4; ++c) {
            const uint4 v = *reinterpret_cast<const uint4*>(q + 4 * kv_word(R, u, 4 * c, lane));
            w[4 * c] = v.x; w[4 * c + 1] = v.y; w[4 * c + 2] = v.z; w[4 * c + 3] = v.w;
        }
    } else if constexpr (R == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(q + 4 * kv_word(R, u, 0, lane));
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int b = 0; b < R; ++b) w[b] = *reinterpret_cast<const uint32_t*>(q + 4 * kv_word(R, u, b, lane));
    }
}

// Scales of positions 8 u + 2 i and + 1, blocks 0 .. R - 1 (fp16 pairs).
template <int R>
__device__ __forceinline__ void load_scales(uint32_t (&w)[R], const uint8_t* s, int u, int i) {
    const uint8_t* p = s + 4 * R * (4 * u + i);
    if constexpr (R % 4 == 0) {
#pragma unroll
        for (int c = 0; c < R / 4; ++c) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 16 * c);
            w[4 * c] = v.x; w[4 * c + 1] = v.y; w[4 * c + 2] = v.z; w[4 * c + 3] = v.w;
        }
    } else if constexpr (R == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int b = 0; b < R; ++b) w[b] = *reinterpret_cast<const uint32_t*>(p + 4 * b);
    }
}

// The power of two that d_V is carried with, from the exponent over every
// |d_V| so far (|d_V| < 2^(ve - 15)): scales all under 2^-6, and those that
// reach 1, are brought to about 1, so that p d_V times both factors stays
// under 2^15 and its small terms off fp16's subnormals.
constexpr float AT_PSCALE = 8192.0f;   // p's factor: p may be 2^AT_LAZY
struct AtScale {
    uint32_t ve;     // 1 .. 32
    uint32_t dmul;   // factor of d_V, an fp16 pair
    float total;     // both factors
    __device__ explicit AtScale(uint32_t e) : ve(e) {
        const int up = e < 10 || e > 15 ? 15 - (int)e : 0;
        // 2^-15 and less (d_V at fp16's end) are subnormals
        const uint32_t h = up > -15 ? (uint32_t)(15 + up) << 10 : 1u << (25 + up - 1);
        dmul = h | h << 16;
        total = AT_PSCALE * __uint_as_float((uint32_t)(127 + up) << 23);
    }
};

// ---- the units of a call ---------------------------------------------------
struct AtSpan {
    int base;     // first position, rounded down to a tile
    int units;    // of AT_UNIT positions
    int groups;   // of AT_PAIRS (row, head) pairs
};

__device__ __forceinline__ AtSpan at_span(const KvEntry& e, int window, int G) {
    const int first = window > 0 ? max(0, e.pos0 - window + 1) : 0;
    AtSpan s;
    s.base = first & ~(AT_TILE - 1);
    s.units = (e.pos0 + e.rows - 1 - s.base) / AT_UNIT + 1;
    s.groups = (int)(((int64_t)e.rows * G + AT_PAIRS - 1) / AT_PAIRS);
    return s;
}

// First CTA whose run reaches past unit u: CTA c has units floor(U c / C) ..
__device__ __forceinline__ int cta_of(int64_t u, int64_t U, int C) { return (int)(((u + 1) * C + U - 1) / U) - 1; }

template <int R>
__global__ void __launch_bounds__(AT_THREADS, AtShape<R>::CTAS_PER_SM)
    kv_attend_kernel(const __grid_constant__ KvAttendParams p) {
    using S = AtShape<R>;
    constexpr int HD = S::HD;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, i = lane & 3;
    uint8_t* ring = smem + warp * S::RING;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BARS) + warp * S::STAGES;
    int64_t* prefix = reinterpret_cast<int64_t*>(smem + S::PREFIX);   // [n_seqs + 1]
    __shared__ int64_t s_warp[AT_WARPS];
    __shared__ int s_last, s_fail;
    const KvView& kv = p.kv;
    const uint32_t base = p.code_base;
    const int n_kv = kv.n_kv, G = kv.n_heads / n_kv, n_seqs = p.rows.n_seqs;

    if (lane == 0) {
        for (int k = 0; k < S::STAGES; ++k) mbar_init(&bars[k], 1);
        fence_mbar_init();
    }
    // units before each entry
    int64_t carry = 0;
    for (int b0 = 0; b0 < n_seqs; b0 += AT_THREADS) {
        const int k = b0 + tid;
        int64_t n = 0;
        if (k < n_seqs) {
            const KvEntry e = kv_entry(kv, p.rows, k, blockIdx.x == 0);
            if (e.rows > 0) {
                const AtSpan sp = at_span(e, p.window, G);
                n = (int64_t)sp.units * sp.groups * n_kv;
            }
        }
        int64_t inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        if (lane == 31) s_warp[warp] = inc;
        __syncthreads();
        int64_t before = carry;
        for (int w = 0; w < warp; ++w) before += s_warp[w];
        if (k < n_seqs) prefix[k] = before + inc - n;
        for (int w = 0; w < AT_WARPS; ++w) carry += s_warp[w];
        __syncthreads();
    }
    const int64_t U = carry;
    if (tid == 0) {
        prefix[n_seqs] = U;
        s_fail = 0;
    }
    __syncthreads();
    if (U == 0) return;
    const int C = (int)min((int64_t)gridDim.x, U), cta = blockIdx.x;
    if (cta >= C) return;
    const int64_t u_begin = U * cta / C, u_end = U * (cta + 1) / C;

    int* counters = reinterpret_cast<int*>(p.workspace);
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + 4096);   // [CTA][2][pairs][HD + 2]
    constexpr int PART = AT_PAIRS * (HD + 2);
    uint32_t it = 0;   // tiles this warp has taken from its ring

    for (int64_t u = u_begin; u < u_end;) {
        int lo = 0, hi = n_seqs;   // the entry of unit u: prefix[lo] <= u < prefix[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (prefix[mid] <= u) lo = mid;
            else hi = mid;
        }
        const KvEntry e = kv_check_entry(kv, p.rows, lo);
        if (e.rows == 0) break;   // its arrays changed under the kernel
        const AtSpan sp = at_span(e, p.window, G);
        const int64_t rel = u - prefix[lo];
        const int item = (int)(rel / sp.units), ua = (int)(rel - (int64_t)item * sp.units);
        const int ub = (int)min((int64_t)sp.units, ua + (u_end - u));
        const int hk = item / sp.groups, pr0 = (item - hk * sp.groups) * AT_PAIRS;
        const int npairs = min(AT_PAIRS, (int)min((int64_t)e.rows * G - pr0, (int64_t)AT_PAIRS));
        const int jmin = pr0 / G, jmax = (pr0 + npairs - 1) / G;
        // positions that some pair sees, and those that all pairs see
        const int kmax = e.pos0 + jmax, kall_hi = e.pos0 + jmin;
        const int kmin = p.window > 0 ? max(0, kall_hi - p.window + 1) : 0;
        const int kall_lo = p.window > 0 ? max(0, kmax - p.window + 1) : 0;
        const int t0 = max(sp.base / AT_TILE + ua * AT_WARPS, kmin / AT_TILE);
        const int t1 = min(sp.base / AT_TILE + ub * AT_WARPS, kmax / AT_TILE + 1);
        const int nt = t0 + warp < t1 ? (t1 - t0 - warp + AT_WARPS - 1) / AT_WARPS : 0;
        // this lane's pair (a missing one computes the last one's again)
        const int pi = pr0 + min(g, npairs - 1), jr = pi / G;
        const int qpos = e.pos0 + jr, qlo = p.window > 0 ? qpos - p.window + 1 : 0;

        // ---- copies: page ids of 32 of this warp's tiles at a time, one a lane
        const int32_t* pages = kv.table + (int64_t)e.seq * kv.max_pages;
        const int per = 1 << (kv.page_shift - 4);
        int id0 = 0, id1 = 0;
        auto lookup = [&](int k0) {
            const int pos = (t0 + warp + (k0 + lane) * AT_WARPS) * AT_TILE;
            if (k0 + lane < nt) {
                id0 = pages[pos >> kv.page_shift];
                if (kv.page_shift == 4 && pos + 16 <= kmax) id1 = pages[(pos >> 4) + 1];
            }
        };
        auto issue = [&](int k) {   // the warp's tile k into its next stage
            const int pos = (t0 + warp + k * AT_WARPS) * AT_TILE;
            const int p0 = __shfl_sync(0xffffffffu, id0, k & 31), p1 = __shfl_sync(0xffffffffu, id1, k & 31);
            if (lane == 0) {
                const uint32_t slot = (it + k) % S::STAGES;   // `it` is the segment's first
                uint8_t* dst = ring + slot * S::TILE_BYTES;
                const bool two = pos + 16 <= kmax;   // the second group holds a position that is seen
                const uint32_t bytes = kv_group_bytes(R) * (two ? 2 : 1);
                mbar_arrive_expect_tx(&bars[slot], bytes);
                const int64_t g0 = ((int64_t)p0 * n_kv + hk) * per + ((pos >> 4) & (per - 1));
                if (kv.page_shift > 4) {
                    bulk_g2s(dst, kv.pages + g0 * kv_group_bytes(R), bytes, &bars[slot]);
                } else {
                    bulk_g2s(dst, kv.pages + g0 * kv_group_bytes(R), kv_group_bytes(R), &bars[slot]);
                    if (two)
                        bulk_g2s(dst + kv_group_bytes(R), kv.pages + ((int64_t)p1 * n_kv + hk) * kv_group_bytes(R),
                                 kv_group_bytes(R), &bars[slot]);
                }
            }
        };
        lookup(0);
        for (int k = 0; k < min(nt, S::STAGES); ++k) issue(k);

        // ---- q: two fp16 parts of the pair's vector times a power of two
        float sfac;                       // score = sfac * (sum of the products)
        uint32_t qf[R == 8 ? 1 : R][2][4];
        uint4* qs = reinterpret_cast<uint4*>(smem + AT_WARPS * S::RING);
        {
            const float* qr = p.q + (int64_t)(e.row0 + jr) * p.ldq + (int64_t)(hk * G + pi - jr * G) * HD + 8 * i;
            float amax = 0.0f;
#pragma unroll
            for (int b = 0; b < R; ++b)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float4 x = *reinterpret_cast<const float4*>(qr + 32 * b + 4 * c);
                    amax = fmaxf(amax, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
                }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // amax * f in [2^13, 2^14)
            const int fe = min(253, max(1, 267 - (int)(__float_as_uint(amax) >> 23)));
            const float f = __uint_as_float((uint32_t)fe << 23);
            sfac = p.scale * 1.44269504088896341f * __uint_as_float((uint32_t)(254 - fe) << 23);
#pragma unroll
            for (int b = 0; b < R; ++b) {
                const float4 x = *reinterpret_cast<const float4*>(qr + 32 * b);
                const float4 y = *reinterpret_cast<const float4*>(qr + 32 * b + 4);
                const float v[8] = {x.x * f, x.y * f, x.z * f, x.w * f, y.x * f, y.y * f, y.z * f, y.w * f};
                // k order of the two products: nibbles (0, 4 | 1, 5) and (2, 6 | 3, 7)
                uint32_t a[2][4];
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    split_half2(v[2 * s], v[2 * s + 4], a[s][0], a[s][1]);
                    split_half2(v[2 * s + 1], v[2 * s + 5], a[s][2], a[s][3]);
                    if constexpr (R == 8) {
                        if (warp == 0) qs[(b * 2 + s) * 32 + lane] = make_uint4(a[s][0], a[s][1], a[s][2], a[s][3]);
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c) qf[b][s][c] = a[s][c];
                    }
                }
            }
            if constexpr (R == 8) __syncthreads();
        }

        float o[R][4][4];
#pragma unroll
        for (int b = 0; b < R; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[b][j][c] = 0.0f;
        float m = -INFINITY;
        float2 l2 = make_float2(0.0f, 0.0f);
        AtScale sv(1);

        for (int k = 0; k < nt; ++k) {
            const uint32_t n = it + k, slot = n % S::STAGES;
            if (!mbar_wait_bounded(&bars[slot], (n / S::STAGES) & 1, kv.err, BREW_DEVERR_TIMEOUT_FULL)) {
                s_fail = 1;   // recorded; the CTA stops after this item
                break;
            }
            const uint8_t* tile = ring + slot * S::TILE_BYTES;
            const int tpos = (t0 + warp + k * AT_WARPS) * AT_TILE;
            const bool full = tpos >= kall_lo && tpos + AT_TILE - 1 <= kall_hi;   // no position is masked

            // ---- scores of positions 8 u + 2 i + e (u = 0 .. 3), log2 units
            float2 s[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) s[u] = make_float2(0.0f, 0.0f);
            if constexpr (R == 8) {
                uint32_t kw[4][8];
                uint32_t sc[4][8];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    load_words<R>(kw[u], tile + (u >> 1) * kv_group_bytes(R), u & 1, lane);
                    load_scales<R>(sc[u], tile + (u >> 1) * kv_group_bytes(R) + 512 * R, u & 1, i);
                }
#pragma unroll
                for (int b = 0; b < R; ++b) {
                    uint32_t a[2][4];
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const uint4 v = qs[(b * 2 + t) * 32 + lane];
                        a[t][0] = v.x; a[t][1] = v.y; a[t][2] = v.z; a[t][3] = v.w;
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        uint32_t x[4];
                        unpack(x, kw[u][b], base);
                        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma_f16(c, a[0], x[0], x[1], c);
                        mma_f16(c, a[1], x[2], x[3], c);
                        s[u] = fma2(half2_bits(sc[u][b]), add2(make_float2(c[0], c[1]), make_float2(c[2], c[3])), s[u]);
                    }
                }
            } else {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    uint32_t kw[R], sc[R];
                    load_words<R>(kw, tile + (u >> 1) * kv_group_bytes(R), u & 1, lane);
                    load_scales<R>(sc, tile + (u >> 1) * kv_group_bytes(R) + 512 * R, u & 1, i);
#pragma unroll
                    for (int b = 0; b < R; ++b) {
                        uint32_t x[4];
                        unpack(x, kw[b], base);
                        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma_f16(c, qf[b][0], x[0], x[1], c);
                        mma_f16(c, qf[b][1], x[2], x[3], c);
                        s[u] = fma2(half2_bits(sc[b]), add2(make_float2(c[0], c[1]), make_float2(c[2], c[3])), s[u]);
                    }
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < 4; ++u) s[u] = make_float2(s[u].x * sfac, s[u].y * sfac);
            uint32_t dead = 0;   // bit 2 u + e: masked for this lane's pair
            if (!full) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int pos = tpos + 8 * u + 2 * i;
                    if (pos > qpos || pos < qlo) {
                        dead |= 1u << (2 * u);
                        s[u].x = -INFINITY;
                    }
                    if (pos + 1 > qpos || pos + 1 < qlo) {
                        dead |= 2u << (2 * u);
                        s[u].y = -INFINITY;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) mx = fmaxf(mx, fmaxf(s[u].x, s[u].y));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            if (__any_sync(0xffffffffu, mx > m + AT_LAZY)) {
                const float mn = mx > m + AT_LAZY ? mx : m;
                const float corr = mn == m ? 1.0f : ex2(m - mn);   // m = -inf: 0
                m = mn;
                l2 = make_float2(l2.x * corr, l2.y * corr);
#pragma unroll
                for (int b = 0; b < R; ++b)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int c = 0; c < 4; ++c) o[b][j][c] *= corr;
            }
            const float mref = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                s[u].x = ex2(s[u].x - mref);
                s[u].y = ex2(s[u].y - mref);
                l2 = add2(l2, s[u]);
            }

            // ---- O += (p d_V) (c - 8), a group of 16 positions at a time
            uint32_t vsc[4][R];
            uint32_t dm = 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                load_scales<R>(vsc[u], tile + (u >> 1) * kv_group_bytes(R) + 544 * R, u & 1, i);
                if (!full) {   // what lies behind a mask may be anything: no NaN of it gets into a product
                    const uint32_t d2 = dead >> (2 * u);
                    const uint32_t keep = (d2 & 1 ? 0u : 0xFFFFu) | (d2 & 2 ? 0u : 0xFFFF0000u);
#pragma unroll
                    for (int b = 0; b < R; ++b) vsc[u][b] &= keep;
                }
#pragma unroll
                for (int b = 0; b < R; ++b) dm = maxabs_h2(dm, vsc[u][b]);
            }
            {
                const uint32_t top = max(dm & 0x7FFFu, dm >> 16 & 0x7FFFu) >> 10;   // fp16's exponent field
                if (__any_sync(0xffffffffu, top >= sv.ve)) {
                    const AtScale next(__reduce_max_sync(0xffffffffu, top) + 1);
                    const float corr = next.total * (1.0f / sv.total);
                    sv = next;
#pragma unroll
                    for (int b = 0; b < R; ++b)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int c = 0; c < 4; ++c) o[b][j][c] *= corr;
                }
                if (sv.dmul != 0x3C003C00u) {
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int b = 0; b < R; ++b) vsc[u][b] = mul_h2(vsc[u][b], sv.dmul);
                }
            }
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
                const uint8_t* grp = tile + gr * kv_group_bytes(R);
                uint32_t vw[2][R], ph[2], pl[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    load_words<R>(vw[c], grp + 256 * R, c, lane);
                    split_half2(s[2 * gr + c].x * AT_PSCALE, s[2 * gr + c].y * AT_PSCALE, ph[c], pl[c]);
                }
#pragma unroll
                for (int b = 0; b < R; ++b) {
                    // p d as two fp16 numbers: the rounded ph d, and its exact rest plus pl d
                    uint32_t a[4];
                    a[0] = mul_h2(ph[0], vsc[2 * gr][b]);
                    a[1] = fma_h2(pl[0], vsc[2 * gr][b], fma_h2(ph[0], vsc[2 * gr][b], neg_h2(a[0])));
                    a[2] = mul_h2(ph[1], vsc[2 * gr + 1][b]);
                    a[3] = fma_h2(pl[1], vsc[2 * gr + 1][b], fma_h2(ph[1], vsc[2 * gr + 1][b], neg_h2(a[2])));
                    uint32_t x0[4], x1[4];
                    unpack(x0, vw[0][b], base);
                    unpack(x1, vw[1][b], base);
#pragma unroll
                    for (int j = 0; j < 4; ++j) mma_f16(o[b][j], a, x0[j], x1[j], o[b][j]);
                }
            }
            __syncwarp();   // every lane has read the stage
            if (((k + S::STAGES) & 31) == 0 && k + S::STAGES < nt) lookup(k + S::STAGES);
            if (k + S::STAGES < nt) issue(k + S::STAGES);
        }
        it += nt;

        // ---- the warps' results meet in shared memory (each in its own ring)
        float l = l2.x + l2.y;
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        float* mine = reinterpret_cast<float*>(ring);   // [pairs][HD], then [pairs][2]
        {
            const float un = 1.0f / sv.total;
#pragma unroll
            for (int b = 0; b < R; ++b)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float4 x = make_float4((o[b][0][c] + o[b][0][c + 2]) * un,
                                                 (o[b][1][c] + o[b][1][c + 2]) * un,
                                                 (o[b][2][c] + o[b][2][c + 2]) * un,
                                                 (o[b][3][c] + o[b][3][c + 2]) * un);
                    *reinterpret_cast<float4*>(mine + g * HD + 32 * b + 8 * i + 4 * c) = x;
                }
            if (i == 0) {
                mine[AT_PAIRS * HD + 2 * g] = m;
                mine[AT_PAIRS * HD + 2 * g + 1] = l;
            }
        }
        __syncthreads();
        const bool whole = ua == 0 && ub == sp.units;
        float* slot = parts + (int64_t)(cta * 2 + (u == u_begin ? 0 : 1)) * PART;
        for (int x = tid; x < npairs * (HD / 4); x += AT_THREADS) {
            const int r = x / (HD / 4), d = x % (HD / 4) * 4;
            float M = -INFINITY, L = 0.0f, wt[AT_WARPS];
#pragma unroll
            for (int w = 0; w < AT_WARPS; ++w)
                M = fmaxf(M, reinterpret_cast<float*>(smem + w * S::RING)[AT_PAIRS * HD + 2 * r]);
            float4 a = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < AT_WARPS; ++w) {
                const float* sw = reinterpret_cast<float*>(smem + w * S::RING);
                const float mw = sw[AT_PAIRS * HD + 2 * r];
                wt[w] = mw == -INFINITY ? 0.0f : ex2(mw - M);
                L += wt[w] * sw[AT_PAIRS * HD + 2 * r + 1];
                const float4 v = *reinterpret_cast<const float4*>(sw + r * HD + d);
                a.x += wt[w] * v.x; a.y += wt[w] * v.y; a.z += wt[w] * v.z; a.w += wt[w] * v.w;
            }
            if (whole) {
                const int pr = pr0 + r, j = pr / G;
                const float inv = 1.0f / L;
                *reinterpret_cast<float4*>(p.out + (int64_t)(e.row0 + j) * p.ldo + (int64_t)(hk * G + pr - j * G) * HD + d) =
                    make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
            } else {
                __stcg(reinterpret_cast<float4*>(slot + r * HD + d), a);
                if (d == 0) __stcg(reinterpret_cast<float2*>(slot + AT_PAIRS * HD + 2 * r), make_float2(M, L));
            }
        }
        if (!whole) {
            // the item's CTAs; the last one to arrive joins their parts
            const int64_t v0 = prefix[lo] + (int64_t)item * sp.units;
            const int c0 = cta_of(v0, U, C), c1 = cta_of(v0 + sp.units - 1, U, C), np = c1 - c0 + 1;
            const bool c0_first = U * c0 / C >= v0;   // the item is the first of CTA c0's run
            __syncthreads();
            if (tid == 0) {
                __threadfence();
                s_last = atomicAdd(&counters[c0], 1) == np - 1;
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                auto part = [&](int c) { return parts + (int64_t)((c0 + c) * 2 + (c == 0 && !c0_first)) * PART; };
                // weights [part][pair] into shared memory
                float* wt = reinterpret_cast<float*>(smem);
                float* tot = wt + AT_MAX_CTAS * AT_PAIRS;   // [pair] sum, then the warps' sums [warp][pairs][HD]
                for (int r = warp; r < npairs; r += AT_WARPS) {
                    float M = -INFINITY, L = 0.0f;
                    for (int c = lane; c < np; c += 32) M = fmaxf(M, __ldcg(part(c) + AT_PAIRS * HD + 2 * r));
                    M = warp_max(M);
                    for (int c = lane; c < np; c += 32) {
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(part(c) + AT_PAIRS * HD + 2 * r));
                        const float w = ml.x == -INFINITY ? 0.0f : ex2(ml.x - M);
                        wt[c * AT_PAIRS + r] = w;
                        L += w * ml.y;
                    }
                    L = warp_sum(L);
                    if (lane == 0) tot[r] = 1.0f / L;
                }
                __syncthreads();
                for (int x = tid; x < npairs * (HD / 4); x += AT_THREADS) {
                    const int r = x / (HD / 4), d = x % (HD / 4) * 4;
                    float4 a = make_float4(0, 0, 0, 0);
#pragma unroll 8
                    for (int c = 0; c < np; ++c) {
                        const float w = wt[c * AT_PAIRS + r];
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(part(c) + r * HD + d));
                        a.x += w * v.x; a.y += w * v.y; a.z += w * v.z; a.w += w * v.w;
                    }
                    const int pr = pr0 + r, j = pr / G;
                    const float inv = tot[r];
                    *reinterpret_cast<float4*>(p.out + (int64_t)(e.row0 + j) * p.ldo + (int64_t)(hk * G + pr - j * G) * HD + d) =
                        make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
                }
                if (tid == 0) counters[c0] = 0;
            }
        }
        fence_proxy_async();   // these plain accesses come before the next item's bulk copies
        __syncthreads();
        if (s_fail) return;
        u += ub - ua;
    }
}

template <int R>
int attend_r(const KvAttendParams& p, cudaStream_t s) {
    using S = AtShape<R>;
    static std::mutex mu;
    static unsigned long long done = 0;
    const int smem = S::PREFIX + 8 * (p.rows.n_seqs + 1);
    {
        std::lock_guard<std::mutex> lk(mu);
        BREW_CUDA(smem_attr_per_device((const void*)kv_attend_kernel<R>, S::PREFIX + 8 * (KV_MAX_SEQS + 1), &done));
    }
    const int ctas = std::min(AT_MAX_CTAS, S::CTAS_PER_SM * num_sms());
    KvAttendParams q = p;
    q.code_base = 0x64006400u;
    kv_attend_kernel<R><<<ctas, AT_THREADS, smem, s>>>(q);
    BREW_CUDA(cudaGetLastError());
    count_launch();
    return BREW_OK;
}

}  // namespace

int64_t kv_attend_workspace(int head_size) {
    return 4096 + (int64_t)AT_MAX_CTAS * 2 * AT_PAIRS * (head_size + 2) * 4;
}

int kv_attend_launch(int hd, const KvAttendParams& p, cudaStream_t s) {
    switch (hd / 32) {
        case 1: return attend_r<1>(p, s);
        case 2: return attend_r<2>(p, s);
        case 3: return attend_r<3>(p, s);
        case 4: return attend_r<4>(p, s);
        default: return attend_r<8>(p, s);
    }
}

}  // namespace brew
