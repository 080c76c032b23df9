// kv_attend.cu — attention over the paged 4-bit K/V cache:
//   o = sum_t softmax_t(scale * q . k_t) v_t
// over the positions t <= the row's own (and > own - window).
//
// Arithmetic.  A cached value is (c - 8) d with a 4-bit code c and an fp16
// scale d of its block of 32.  Both products run on mma.m16n8k16 with the
// codes' exact c - 8 as the 16-row operand (16 positions, or 16 dims) and 8
// (row, head) pairs as the 8 columns.  fp32 accuracy comes from carrying the
// other operand as two fp16 numbers (hi = fp16(x), lo = fp16(x - hi), 22 bits
// together), one product each.
//   scores   S = sum_b d_K[t][b] (sum_{i in b} q_i (c_ti - 8))
//   output   O = sum_t (p_t d_V[t][b]) (c_ti - 8)
// q, p and d_V are scaled by powers of two (q below 2^14, p and p d_V to 2^15
// at most), so that no part leaves fp16's range and little falls among its
// subnormals (2^-24 beside 2^13): each block of V has a power of its own, at
// least 1, so that no d_V is rounded for another block or another tile; where p
// d_V would pass 2^15 all the same (values over 32 that carry the weight), the
// tile's p are taken down instead.  The softmax is online; its running maximum
// moves only when exceeded by 2^2, so O is rarely rescaled.
//
// Work split.  Units of a tile for each warp of one (sequence, kv head, 8 pairs),
// laid end to end over all sequences of the call, each item's behind a weight;
// every CTA takes an equal run, whatever the lengths (read on the device: a captured graph
// follows them).  A run's first and last item may be shared with other CTAs:
// their partial results (max, sum, O) go to the workspace and the last CTA to
// arrive joins them in order.  Within an item each warp streams its own
// 32-position tiles through a ring of shared-memory stages (bulk copies: the
// tile's K, V and scales are one run per page); the next item's first tiles
// are under way while an item's warps meet.
//
// Bound: the steps between the copies and the products (unpacking the codes, the
// split of q, p and p d_V), of which 4 warps a scheduler have too few under way:
// 54 % of the issue slots are taken, the tensor pipe 32 %, and the largest stalls
// are an instruction's own latency (1.5 an issue), the math pipe and another
// warp's turn (1.1 each).  128 sequences of 8192 positions, 28/4 heads of 128: 178
// us on the device for 608 MB, 3.4 TB/s or 0.52 of a copy's rate; one of 131071,
// 16/8 heads: 53 us, 2.8 TB/s.  (4 warps a CTA and 3 or 4 CTAs 182 to 184 us; 5
// and 3 190; a kernel of its own for the join 4.6 us more on small calls.)
#include <algorithm>

#include "brew_internal.cuh"
#include "decode.cuh"
#include "kv_device.cuh"

namespace brew {
namespace {

constexpr int AT_TILE = 32;                       // positions a warp handles at once
constexpr int AT_PAIRS = 8;                       // (row, head) pairs of a tile
constexpr int AT_MAX_CTAS = 4 * 148;
// mma truncates as it accumulates: after this many tiles its sums are added,
// rounded, to others (128 x 8192 positions: error 3.0e-6 without).
constexpr int AT_FLUSH = 8;
// From this many (row, head) pairs of an entry and kv head on, the prompt
// kernel takes it: its tiles of 128 pairs cost the same however few there are,
// but no more than this kernel's 8 tiles of 8.  32 sequences of 1000 positions
// with 64 pairs each, 16/8 heads of 128: 77 us there, 121 here; with 16 pairs
// 71 and 43.  In a call of few rows, where neither fills the device, this
// kernel starts faster: one sequence of 300 positions with 256 pairs, 30 us
// there, 23 here; of 4096 positions with 256 pairs 41 and 57, with 64 39 and 30.
constexpr int64_t AT_PROMPT_PAIRS = 64, AT_PROMPT_PAIRS_FEW = 256, AT_MANY_PAIRS = 2048;
// Units that an item weighs beside its own, for its start and end: without, the
// CTAs that short sequences fall to are the last (32 sequences of 38 to 32768
// positions, 28/4 heads of 128: 91 us, 80 with it).
constexpr int AT_ITEM = 1;
constexpr float AT_LAZY = 2.0f;                   // log2 of how far p may exceed 1

template <int R>
struct AtShape {
    static constexpr int HD = 32 * R;
    // 16 warps an SM (8 with heads of 256)
    static constexpr int WARPS = R == 8 || R == 4 ? 8 : 4;
    static constexpr int CTAS_PER_SM = R == 8 ? 1 : R == 4 ? 2 : 4;
    static constexpr int THREADS = 32 * WARPS;
    static constexpr int UNIT = AT_TILE * WARPS;
    static constexpr int TILE_BYTES = 2 * kv_group_bytes(R);
    static constexpr int STAGES = R <= 2 ? 4 : 2;
    static constexpr int RING = STAGES * TILE_BYTES;   // of a warp
    static constexpr int PITCH = HD + 4;               // floats of a pair's result (conflict-free stores)
    static constexpr int SUMS = (AT_PAIRS * PITCH + 2 * AT_PAIRS) * 4;   // of a warp: its sums, later its result
    static constexpr int Q = WARPS * (RING + SUMS);
    static constexpr int QBYTES = R * 2 * 32 * 16 + AT_PAIRS * 4;        // q's fragments, the pairs' factors
    static constexpr int BARS = Q + QBYTES;
    static constexpr int PREFIX = BARS + WARPS * STAGES * 8;
    static_assert(SUMS % 16 == 0 && RING % 128 == 0, "alignment");
    static_assert(AT_MAX_CTAS * 4 <= RING, "a join's weights fit a warp's ring");
};

// ---- mma.m16n8k16 --------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                        const float (&c)[4]) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// The first product of a sum.
__device__ __forceinline__ void mma_f16_new(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{0f00000000,0f00000000,0f00000000,0f00000000};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr float AT_PLOG2 = 13.0f;   // p is carried times 2^13, sums and all: p may be 2^AT_LAZY
// A block's d_V are carried times 2^up, up >= 0, which brings the largest of them
// under 1, and over 2^-6 or so: above, p d_V might pass fp16; below, its second
// part would lie among the subnormals.  It moves when a tile's scales leave
// [2^-8, 1]: they differ little from tile to tile, so that is rare.  The blocks'
// ups are the nibbles of a register.  (One power for all blocks, from the largest
// so far, rounded d_V themselves: 60 % off in a block 10^7 below another.  The
// check costs 1.5 % of a batch, 178 us against 176 for 128 sequences of 8192
// positions; values over 8 cost 14 %, under 0.03 6 %.)
constexpr int AT_UP_MAX = 14;       // 2^14 is about where fp16 ends
__device__ __forceinline__ int up_of(uint32_t ups, int b) { return (int)(ups >> 4 * b & 15u); }
__device__ __forceinline__ uint32_t up_h2(uint32_t ups, int b) {
    const uint32_t h = (uint32_t)(15 + up_of(ups, b)) << 10;
    return h | h << 16;
}
__device__ __forceinline__ float pow2f(int k) { return __uint_as_float((uint32_t)(127 + k) << 23); }

// An 8 x 8 matrix of fp16, row g in lanes 4 g .. 4 g + 3, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// ---- the units of a call ---------------------------------------------------
struct AtSpan {
    int base;     // first position, rounded down to a tile
    int units;    // of AtShape::UNIT positions
    int groups;   // of AT_PAIRS (row, head) pairs
};

template <int R>
__device__ __forceinline__ AtSpan at_span(const KvEntry& e, int window, int G) {
    const int first = window > 0 ? max(0, e.pos0 - window + 1) : 0;
    AtSpan s;
    s.base = first & ~(AT_TILE - 1);
    s.units = (e.pos0 + e.rows - 1 - s.base) / AtShape<R>::UNIT + 1;
    s.groups = (int)(((int64_t)e.rows * G + AT_PAIRS - 1) / AT_PAIRS);
    return s;
}

// The CTA of unit u: CTA c has units U c / C up to U (c + 1) / C
__device__ __forceinline__ int cta_of(int64_t u, int64_t U, int C) { return (int)(((u + 1) * C + U - 1) / U) - 1; }

__host__ __device__ constexpr int at_part_floats(int HD) { return AT_PAIRS * (HD + 2); }   // O, then (max, sum)
static_assert(AT_MAX_CTAS * 4 <= KV_COUNTER_BYTES, "counters");

// A CTA's run through one item.
struct AtSeg {
    int seq, pos0, row0;
    int hk, pr0, npairs;
    int ua, ub, units;        // units [ua, ub) of the item's
    int64_t item0;            // the item's first unit
    int t0, nt;               // first tile of this warp (tiles of a unit are dealt to the warps), and how many
    int kmax;                 // last position that a pair sees
    int all_lo, all_hi;       // positions that all pairs see
};

template <int R>
__global__ void __launch_bounds__(AtShape<R>::THREADS, AtShape<R>::CTAS_PER_SM)
    kv_attend_kernel(const __grid_constant__ KvAttendParams p) {
    using S = AtShape<R>;
    constexpr int HD = S::HD;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, i = lane & 3;
    if (p.prompts) pdl_launch_dependents();   // it shares nothing with this kernel's work: other entries, another workspace
    uint8_t* ring = smem + warp * S::RING;
    float* mine = reinterpret_cast<float*>(smem + S::WARPS * S::RING + warp * S::SUMS);
    uint4* qs = reinterpret_cast<uint4*>(smem + S::Q);                 // [block][hi, lo][lane]
    float* qfac = reinterpret_cast<float*>(smem + S::Q + R * 2 * 32 * 16);   // [pair]
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BARS) + warp * S::STAGES;
    int64_t* prefix = reinterpret_cast<int64_t*>(smem + S::PREFIX);   // [a thread's entries]
    __shared__ int64_t s_warp[S::WARPS];
    __shared__ AtSeg s_seg[S::WARPS], s_done;   // the warps' present item, and the one whose result is made
    __shared__ AtSeg s_ends[2];            // the run's first and last item, where shared with other CTAs
    __shared__ int s_fail, s_join[2];
    const KvView& kv = p.kv;
    const uint32_t base = p.code_base;
    const int n_kv = kv.n_kv, G = kv.n_heads / n_kv, n_seqs = p.rows.n_seqs;

    if (lane == 0) {
        for (int k = 0; k < S::STAGES; ++k) mbar_init(&bars[k], 1);
        fence_mbar_init();
    }
    if (tid == 0) s_fail = 0;
    // units before each thread's entries (one for up to 256 of them)
    auto entry_units = [&](const KvEntry& e) -> int64_t {
        if (e.rows <= 0 || (int64_t)e.rows * G >= p.pairs_min) return 0;
        const AtSpan sp = at_span<R>(e, p.window, G);
        return (int64_t)(sp.units + AT_ITEM) * sp.groups * n_kv;
    };
    const int step = (n_seqs + S::THREADS - 1) / S::THREADS, nsteps = (n_seqs + step - 1) / step;
    int64_t U = 0;
    {
        int64_t n = 0;
        for (int k = tid * step; k < min(n_seqs, (tid + 1) * step); ++k)
            n += entry_units(kv_entry(kv, p.rows, k, blockIdx.x == 0));
        int64_t inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        if (lane == 31) s_warp[warp] = inc;
        __syncthreads();
        int64_t before = 0;
#pragma unroll
        for (int w = 0; w < S::WARPS; ++w) {
            if (w < warp) before += s_warp[w];
            U += s_warp[w];
        }
        if (tid < nsteps) prefix[tid] = before + inc - n;
        __syncthreads();
    }
    const int C = (int)min((int64_t)gridDim.x, U), cta = blockIdx.x;
    if (cta >= C) return;
    const int64_t u_begin = U * cta / C, u_end = U * (cta + 1) / C;

    auto locate = [&](int64_t u, AtSeg& to) {
        int lo = 0, hi = nsteps;   // the entries of unit u: prefix[lo] <= u, the next one's is more
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (prefix[mid] <= u) lo = mid;
            else hi = mid;
        }
        AtSeg s;
        int64_t rel = u - prefix[lo];
        int k = lo * step;
        KvEntry e = kv_check_entry(kv, p.rows, k);
        for (int64_t n; k + 1 < n_seqs && rel >= (n = entry_units(e)); rel -= n) e = kv_check_entry(kv, p.rows, ++k);
        AtSpan sp = {0, 1, 1};
        if (e.rows > 0) sp = at_span<R>(e, p.window, G);
        const int width = sp.units + AT_ITEM;
        const int item = rel < (1ll << 31) ? (int)rel / width : (int)(rel / width);
        s.seq = e.seq;
        s.pos0 = e.pos0;
        s.row0 = e.row0;
        s.units = sp.units;
        const int in = (int)(rel - (int64_t)item * width);   // below AT_ITEM: before the item's first unit
        s.item0 = u - in + AT_ITEM;
        s.ua = max(in - AT_ITEM, 0);
        s.ub = (int)min((int64_t)sp.units, u_end - s.item0);
        s.hk = item / sp.groups;
        s.pr0 = (item - s.hk * sp.groups) * AT_PAIRS;
        s.npairs = (int)min((int64_t)e.rows * G - s.pr0, (int64_t)AT_PAIRS);
        s.all_hi = e.pos0 + s.pr0 / G;                       // the first pair's position
        s.kmax = e.pos0 + (s.pr0 + s.npairs - 1) / G;        // the last one's
        s.all_lo = p.window > 0 ? max(0, s.kmax - p.window + 1) : 0;
        const int kmin = p.window > 0 ? max(0, s.all_hi - p.window + 1) : 0;
        const int a = max(sp.base / AT_TILE + s.ua * S::WARPS, kmin / AT_TILE) + warp;
        const int b = min(sp.base / AT_TILE + s.ub * S::WARPS, s.kmax / AT_TILE + 1);
        s.t0 = a;
        s.nt = e.rows > 0 && a < b ? (b - a + S::WARPS - 1) / S::WARPS : 0;
        if (lane == 0) to = s;
    };

    // ---- copies: the sources of 32 of this warp's tiles at a time, one a
    // lane, which issues them itself when their turn comes
    const int per = 1 << (kv.page_shift - 4);   // groups of a page and head
    const uint8_t *src0 = nullptr, *src1 = nullptr;
    uint32_t nbytes = 0;
    auto lookup = [&](const AtSeg& s, int k0) {
        const int pos = (s.t0 + (k0 + lane) * S::WARPS) * AT_TILE;
        if (k0 + lane < s.nt) {
            const int32_t* pages = kv.table + (int64_t)s.seq * kv.max_pages;
            const int id = pages[pos >> kv.page_shift];
            src0 = kv.pages + (((int64_t)id * n_kv + s.hk) * per + ((pos >> 4) & (per - 1))) * kv_group_bytes(R);
            const bool two = pos + 16 <= s.kmax;   // the second group holds a position that is seen
            nbytes = kv_group_bytes(R) * (two ? 2 : 1);
            if (per == 1 && two)
                src1 = kv.pages + ((int64_t)pages[(pos >> 4) + 1] * n_kv + s.hk) * kv_group_bytes(R);
        }
    };
    auto issue = [&](int k, uint32_t n) {   // tile k, the warp's n-th, into its stage
        if (lane == (k & 31)) {
            const uint32_t slot = n % S::STAGES;
            uint8_t* dst = ring + slot * S::TILE_BYTES;
            mbar_arrive_expect_tx(&bars[slot], nbytes);
            bulk_g2s(dst, src0, per > 1 ? nbytes : kv_group_bytes(R), &bars[slot]);
            if (per == 1 && nbytes > kv_group_bytes(R))
                bulk_g2s(dst + kv_group_bytes(R), src1, kv_group_bytes(R), &bars[slot]);
        }
    };
    uint32_t nth = 0;   // tiles this warp has taken
    // the copies of its next n tiles, which are under way: a CTA that gives up ends behind them
    auto drain = [&](int n) {
        for (uint32_t k = nth; k < nth + n; ++k)
            mbar_wait_bounded(&bars[k % S::STAGES], k / S::STAGES & 1, kv.err, BREW_DEVERR_TIMEOUT_FULL);
    };
    auto fill = [&](const AtSeg& s) {
        lookup(s, 0);
        for (int k = 0; k < min(s.nt, S::STAGES); ++k) issue(k, nth + k);
    };

    int* counters = reinterpret_cast<int*>(p.workspace);                                             // [CTA]
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + KV_COUNTER_BYTES);   // [CTA][2][part]
    AtSeg& seg = s_seg[warp];
    const AtSeg& done = s_done;
    locate(u_begin, seg);
    __syncwarp();
    if (seg.ub <= seg.ua) return;   // nothing but an item's weight
    fill(seg);
    bool split_first = false, split_last = false;   // the run's first and last item is shared

    for (int64_t u = u_begin;;) {
        // ---- q: a warp makes a pair's two fp16 parts, times a power of two
        for (int pair = warp; pair < AT_PAIRS; pair += S::WARPS) {
            const int pi = seg.pr0 + min(pair, seg.npairs - 1), j = pi / G;   // missing pairs repeat the last one
            const float* qr = p.q + (int64_t)(seg.row0 + j) * p.ldq + (int64_t)(seg.hk * G + pi - j * G) * HD;
            constexpr int NV = R == 8 ? 2 : 1;
            float4 x[NV];
            float amax = 0.0f;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                x[n] = 4 * lane < HD ? *reinterpret_cast<const float4*>(qr + 128 * n + 4 * lane) : make_float4(0, 0, 0, 0);
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(x[n].x), fabsf(x[n].y)), fmaxf(fabsf(x[n].z), fabsf(x[n].w))));
            }
            amax = warp_max(amax);
            // amax * f in [2^13, 2^14)
            const int fe = min(253, max(1, 267 - (int)(__float_as_uint(amax) >> 23)));
            const float f = copysignf(__uint_as_float((uint32_t)fe << 23), p.scale);   // a negative scale turns q
            // (never 0: a masked score is -inf times it)
            if (lane == 0)
                qfac[pair] = fmaxf(fabsf(p.scale) * 1.44269504088896341f * __uint_as_float((uint32_t)(254 - fe) << 23), 1e-37f);
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                // dims 8 i + 0 .. 3 (even lanes) and 8 i + 4 .. 7 (odd) of block b; k order of the products: dims
                // (0, 4 | 1, 5) and (2, 6 | 3, 7); the even lane stores the high parts, the odd one the low ones
                const float v[4] = {x[n].x * f, x[n].y * f, x[n].z * f, x[n].w * f};
                uint32_t w[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float other = __shfl_xor_sync(0xffffffffu, v[c], 1);
                    uint32_t hi, lo;
                    split_half2(lane & 1 ? other : v[c], lane & 1 ? v[c] : other, hi, lo);
                    w[c] = lane & 1 ? lo : hi;
                }
                if (4 * lane < HD)
                    qs[((4 * n + lane / 8) * 2 + (lane & 1)) * 32 + pair * 4 + (lane & 7) / 2] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        __syncthreads();
        // this lane's pairs: g as the products' operand, 2 i and 2 i + 1 in their results
        const int gpos = seg.pos0 + (seg.pr0 + min(g, seg.npairs - 1)) / G;
        // the warp's tiles full0 .. full0 + nfull - 1 have no masked position
        int full0 = 0, nfull = 0;
        if (seg.all_hi >= AT_TILE - 1) {
            const int a = (seg.all_lo + AT_TILE - 1) / AT_TILE - seg.t0, b = (seg.all_hi - AT_TILE + 1) / AT_TILE - seg.t0;
            full0 = max(0, a + S::WARPS - 1) / S::WARPS;
            nfull = b < 0 ? 0 : max(0, b / S::WARPS + 1 - full0);
        }
        const float sfac[2] = {qfac[2 * i], qfac[2 * i + 1]};   // score = sfac * (sum of the products)

        float o[R][2][4];   // (b, t): dims 32 b + 4 g + 2 t (0, 1) and + 1 (2, 3) of pairs 2 i (0, 2) and 2 i + 1 (1, 3)
#pragma unroll
        for (int b = 0; b < R; ++b)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[b][t][c] = 0.0f;
        // O of the tiles before the last few (see AT_FLUSH), in shared memory: a lane's own values
        bool kept = false;
        auto keep = [&](float (&k)[2]) {   // sums = sums * k (+ o, which starts again)
            float4* sm = reinterpret_cast<float4*>(mine);
#pragma unroll
            for (int b = 0; b < R; ++b)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    float4 v = kept ? sm[(2 * b + t) * 32 + lane] : make_float4(0, 0, 0, 0);
                    v.x = v.x * k[0] + o[b][t][0]; v.y = v.y * k[1] + o[b][t][1];
                    v.z = v.z * k[0] + o[b][t][2]; v.w = v.w * k[1] + o[b][t][3];
                    sm[(2 * b + t) * 32 + lane] = v;
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[b][t][c] = 0.0f;
                }
            kept = true;
        };
        auto rescale = [&](float (&k)[2]) {
#pragma unroll
            for (int b = 0; b < R; ++b)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[b][t][c] *= k[c & 1];
            if (kept) keep(k);
        };
        auto lower = [&](int sign, int k) {   // o = o * 2^(sign * k), k of the pair's own lanes
            float f[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) f[c] = pow2f(sign * __shfl_sync(0xffffffffu, k, 8 * i + 4 * c));
#pragma unroll
            for (int b = 0; b < R; ++b)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[b][t][c] *= f[c & 1];
        };
        float m[2] = {-INFINITY, -INFINITY};
        float2 l2 = make_float2(0.0f, 0.0f);
        uint32_t ups = 0;

        int k = 0;
        for (; k < seg.nt; ++k) {
            const uint32_t slot = nth % S::STAGES;
            if (!mbar_wait_bounded(&bars[slot], nth / S::STAGES & 1, kv.err, BREW_DEVERR_TIMEOUT_FULL)) {
                s_fail = 1;   // recorded; the CTA stops after this item
                drain(min(seg.nt - k, S::STAGES));
                break;
            }
            const uint8_t* tile = ring + slot * S::TILE_BYTES;
            // ---- scores (log2 units) of positions 16 gr + g (0, 1) and + 8 (2, 3), pairs 2 i and 2 i + 1
            float s[2][4];
            {
                uint32_t kw[2][2][R];
                __half d[2][2][R];
#pragma unroll
                for (int gr = 0; gr < 2; ++gr)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        load_words<R>(kw[gr][h], tile + gr * kv_group_bytes(R), h, lane);
                        load_kscales<R>(d[gr][h], tile + gr * kv_group_bytes(R) + 512 * R, g + 8 * h);
                        s[gr][2 * h] = s[gr][2 * h + 1] = 0.0f;
                    }
#pragma unroll
                for (int b = 0; b < R; ++b) {
                    const uint4 qh = qs[2 * b * 32 + lane], ql = qs[(2 * b + 1) * 32 + lane];
#pragma unroll
                    for (int gr = 0; gr < 2; ++gr) {
                        uint32_t x0[4], x1[4];
                        unpack(x0, kw[gr][0][b], base);
                        unpack(x1, kw[gr][1][b], base);
                        const uint32_t a0[4] = {x0[0], x1[0], x0[1], x1[1]}, a1[4] = {x0[2], x1[2], x0[3], x1[3]};
                        float c[4];
                        mma_f16_new(c, a0, ql.x, ql.y);
                        mma_f16(c, a1, ql.z, ql.w, c);
                        mma_f16(c, a0, qh.x, qh.y, c);
                        mma_f16(c, a1, qh.z, qh.w, c);
                        const float f0 = __half2float(d[gr][0][b]), f1 = __half2float(d[gr][1][b]);
                        s[gr][0] = fmaf(f0, c[0], s[gr][0]);
                        s[gr][1] = fmaf(f0, c[1], s[gr][1]);
                        s[gr][2] = fmaf(f1, c[2], s[gr][2]);
                        s[gr][3] = fmaf(f1, c[3], s[gr][3]);
                    }
                }
            }
            uint32_t vsc[4][R];   // V's scales of positions 8 u + 2 i, + 1
#pragma unroll
            for (int u4 = 0; u4 < 4; ++u4)
                load_scales<R>(vsc[u4], tile + (u4 >> 1) * kv_group_bytes(R) + 544 * R, u4 & 1, i);
            if ((uint32_t)(k - full0) >= (uint32_t)nfull) {   // some position is masked
                const int tpos = (seg.t0 + k * S::WARPS) * AT_TILE;
                int qpos[2], qlo[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    qpos[c] = __shfl_sync(0xffffffffu, gpos, 8 * i + 4 * c);
                    qlo[c] = p.window > 0 ? qpos[c] - p.window + 1 : 0;
                }
#pragma unroll
                for (int gr = 0; gr < 2; ++gr)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int pos = tpos + 16 * gr + 4 * (c & 2) + g;
                        if (pos > qpos[c & 1] || pos < qlo[c & 1]) s[gr][c] = -INFINITY;
                    }
                // what lies behind a mask may be anything: no NaN of it gets into a product
                const int glo = p.window > 0 ? gpos - p.window + 1 : 0;
#pragma unroll
                for (int u4 = 0; u4 < 4; ++u4) {
                    const int pos = tpos + 8 * u4 + 2 * i;
                    const uint32_t live = (pos > gpos || pos < glo ? 0u : 0xFFFFu) |
                                          (pos + 1 > gpos || pos + 1 < glo ? 0u : 0xFFFF0000u);
#pragma unroll
                    for (int b = 0; b < R; ++b) vsc[u4][b] &= live;
                }
            }
            float mx[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) mx[c] = fmaxf(fmaxf(s[0][c], s[0][c + 2]), fmaxf(s[1][c], s[1][c + 2])) * sfac[c];
            if (__any_sync(0xffffffffu, mx[0] > m[0] + AT_LAZY || mx[1] > m[1] + AT_LAZY)) {
                float corr[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], w));
                    const float mn = mx[c] > m[c] + AT_LAZY ? mx[c] : m[c];
                    corr[c] = mn == m[c] ? 1.0f : ex2(m[c] - mn);   // m = -inf: 0
                    m[c] = mn;
                }
                l2 = make_float2(l2.x * corr[0], l2.y * corr[1]);
                rescale(corr);
            }
            const float mref[2] = {m[0] == -INFINITY ? 0.0f : AT_PLOG2 - m[0], m[1] == -INFINITY ? 0.0f : AT_PLOG2 - m[1]};
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
#pragma unroll
                for (int c = 0; c < 4; ++c) s[gr][c] = ex2(fmaf(s[gr][c], sfac[c & 1], mref[c & 1]));
                l2 = add2(l2, make_float2(s[gr][0], s[gr][1]));
                l2 = add2(l2, make_float2(s[gr][2], s[gr][3]));
            }

            // ---- O += (p d_V) (c - 8), a group of 16 positions at a time
            int down = 0;          // log2 of what this lane's pair's p are divided by for this tile
            bool lowered = false;  // some pair's are
            {
                uint32_t hi = 0, lo = 0x7C007C00u;   // the blocks' largest scales: the largest and the smallest
#pragma unroll
                for (int b = 0; b < R; ++b) {
                    const uint32_t d = maxabs_h2(maxabs_h2(vsc[0][b], vsc[1][b]), maxabs_h2(vsc[2][b], vsc[3][b]));
                    hi = maxabs_h2(hi, d);
                    lo = minabs_h2(lo, d);
                }
                if (__builtin_expect(ups != 0, 0)) {
                    hi = 0;
                    lo = 0x7C007C00u;
#pragma unroll
                    for (int b = 0; b < R; ++b) {
                        const uint32_t d = mul_h2(maxabs_h2(maxabs_h2(vsc[0][b], vsc[1][b]), maxabs_h2(vsc[2][b], vsc[3][b])), up_h2(ups, b));
                        hi = maxabs_h2(hi, d);
                        lo = minabs_h2(lo, d);
                    }
                }
                // in either half: hi over 1 (0x3C00, to which 0x43FF carries) or lo under 2^-8 (0x1C00, 0x6400)
                const uint32_t over = ((hi & 0x7FFF7FFFu) + 0x43FF43FFu) & 0x80008000u;
                const uint32_t under = ~((lo & 0x7FFF7FFFu) + 0x64006400u) & 0x80008000u;
                auto raise = [&] {
#pragma unroll
                    for (int b = 0; b < R; ++b) {
                        const uint32_t f = up_h2(ups, b);
#pragma unroll
                        for (int u4 = 0; u4 < 4; ++u4) vsc[u4][b] = mul_h2(vsc[u4][b], f);
                    }
                };
                if (__builtin_expect(__any_sync(0xffffffffu, over | under), 0)) {
                    const bool move = ups != 0 || __any_sync(0xffffffffu, under);
                    if (move) {
#pragma unroll
                        for (int b = 0; b < R; ++b) {
                            const uint32_t d = maxabs_h2(maxabs_h2(vsc[0][b], vsc[1][b]), maxabs_h2(vsc[2][b], vsc[3][b])) & 0x7FFF7FFFu;
                            const uint32_t d0 = d & 0xFFFFu, d1 = d >> 16;   // (NaN: no size)
                            const uint32_t top = __reduce_max_sync(0xffffffffu, max(d0 < 0x7C00u ? d0 : 0u, d1 < 0x7C00u ? d1 : 0u));
                            const int k = up_of(ups, b), e = (int)(top >> 10) - 14 + k;   // top * 2^up < 2^e
                            const int next = top != 0 && (e > 0 || e < -5) ? min(AT_UP_MAX, max(0, k - e)) : k;
                            if (next == k) continue;
                            const float f = pow2f(next - k);
#pragma unroll
                            for (int t = 0; t < 2; ++t)
#pragma unroll
                                for (int c = 0; c < 4; ++c) o[b][t][c] *= f;
                            if (kept) {
                                float4* sm = reinterpret_cast<float4*>(mine);
#pragma unroll
                                for (int t = 0; t < 2; ++t) {
                                    float4 v = sm[(2 * b + t) * 32 + lane];
                                    v.x *= f; v.y *= f; v.z *= f; v.w *= f;
                                    sm[(2 * b + t) * 32 + lane] = v;
                                }
                            }
                            ups ^= (uint32_t)(k ^ next) << 4 * b;
                        }
                    }
                    if (ups != 0) raise();
                    // p d_V of a pair: 2^15 at most
                    uint32_t pd = 0, x[4], d[4];
#pragma unroll
                    for (int u4 = 0; u4 < 4; ++u4) {
                        x[u4] = transpose8(pack_half2(s[u4 >> 1][2 * (u4 & 1)], s[u4 >> 1][2 * (u4 & 1) + 1]));
                        d[u4] = 0;
#pragma unroll
                        for (int b = 0; b < R; ++b) d[u4] = maxabs_h2(d[u4], vsc[u4][b]);
                        pd = maxabs_h2(pd, mul_h2(x[u4], d[u4]));
                    }
                    if (__any_sync(0xffffffffu, ((pd & 0x7FFF7FFFu) + 0x07FF07FFu) & 0x80008000u)) {   // over 2^15: 0x7800
                        float most = 0.0f;
#pragma unroll
                        for (int u4 = 0; u4 < 4; ++u4) {
                            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&x[u4]));
                            const float2 z = __half22float2(*reinterpret_cast<const __half2*>(&d[u4]));
                            most = fmaxf(most, fmaxf(fabsf(y.x * z.x), fabsf(y.y * z.y)));
                        }
#pragma unroll
                        for (int w = 1; w < 4; w <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, w));
                        if (most > 32768.0f) down = (int)(__float_as_uint(most) >> 23) - 127 - 14;
                        lowered = true;
                        const float f[2] = {pow2f(-__shfl_sync(0xffffffffu, down, 8 * i)), pow2f(-__shfl_sync(0xffffffffu, down, 8 * i + 4))};
#pragma unroll
                        for (int gr = 0; gr < 2; ++gr)
#pragma unroll
                            for (int c = 0; c < 4; ++c) s[gr][c] *= f[c & 1];
                        lower(-1, down);
                    }
                } else if (__builtin_expect(ups != 0, 0)) {
                    raise();
                }
            }
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
                uint32_t vw[2][R], ph[2], pl[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    load_words<R>(vw[c], tile + gr * kv_group_bytes(R) + 256 * R, c, lane);
                    // p of (position g, pairs 2 i and + 1), transposed to (pair g, positions 2 i and + 1)
                    split_half2(s[gr][2 * c], s[gr][2 * c + 1], ph[c], pl[c]);
                    ph[c] = transpose8(ph[c]);
                    pl[c] = transpose8(pl[c]);
                }
#pragma unroll
                for (int b = 0; b < R; ++b) {
                    // p d as two fp16 numbers: the rounded ph d, and its exact rest plus pl d
                    const uint32_t v0 = vsc[2 * gr][b], v1 = vsc[2 * gr + 1][b];
                    const uint32_t h0 = mul_h2(ph[0], v0), h1 = mul_h2(ph[1], v1);
                    const uint32_t r0 = fma_h2(pl[0], v0, fma_h2(ph[0], v0, neg_h2(h0)));
                    const uint32_t r1 = fma_h2(pl[1], v1, fma_h2(ph[1], v1, neg_h2(h1)));
                    uint32_t x0[4], x1[4];
                    unpack(x0, vw[0][b], base);
                    unpack(x1, vw[1][b], base);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const uint32_t a[4] = {x0[2 * t], x0[2 * t + 1], x1[2 * t], x1[2 * t + 1]};
                        mma_f16(o[b][t], a, r0, r1, o[b][t]);
                        mma_f16(o[b][t], a, h0, h1, o[b][t]);
                    }
                }
            }
            if (__builtin_expect(lowered, 0)) lower(1, down);
            __syncwarp();   // every lane has read the stage
            if (k + S::STAGES < seg.nt) {
                if (((k + S::STAGES) & 31) == 0) lookup(seg, k + S::STAGES);
                issue(k + S::STAGES, nth);
            }
            ++nth;
            if ((k & (AT_FLUSH - 1)) == AT_FLUSH - 1) {
                float one[2] = {1.0f, 1.0f};
                keep(one);
            }
        }

        // ---- the next item's first tiles, then this one's result
        const int64_t at = u;
        const bool cut = k < seg.nt;   // this warp gave up
        u = seg.item0 + seg.ub;
        if (tid == 0) s_done = seg;
        __syncwarp();
        const bool more = !cut && u + AT_ITEM < u_end;
        if (more) {
            locate(u, seg);
            __syncwarp();
            fill(seg);
        }
        float l[2] = {l2.x, l2.y};
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) l[c] += __shfl_xor_sync(0xffffffffu, l[c], w);
        {
            if (kept) {
                const float4* sm = reinterpret_cast<const float4*>(mine);
#pragma unroll
                for (int b = 0; b < R; ++b)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const float4 v = sm[(2 * b + t) * 32 + lane];
                        o[b][t][0] += v.x; o[b][t][1] += v.y; o[b][t][2] += v.z; o[b][t][3] += v.w;
                    }
                __syncwarp();
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int b = 0; b < R; ++b) {
                    const float un = pow2f(-up_of(ups, b));
                    *reinterpret_cast<float4*>(mine + (2 * i + c) * S::PITCH + 32 * b + 4 * g) =
                        make_float4(o[b][0][c] * un, o[b][0][c + 2] * un, o[b][1][c] * un, o[b][1][c + 2] * un);
                }
                if (g == 0) {
                    mine[AT_PAIRS * S::PITCH + 2 * (2 * i + c)] = m[c];
                    mine[AT_PAIRS * S::PITCH + 2 * (2 * i + c) + 1] = l[c];
                }
            }
        }
        __syncthreads();
        const bool whole = done.ua == 0 && done.ub == done.units;
        float* slot = parts + (int64_t)(cta * 2 + (at == u_begin ? 0 : 1)) * at_part_floats(HD);
        for (int x = tid; x < done.npairs * (HD / 4); x += S::THREADS) {
            const int r = x / (HD / 4), d = x % (HD / 4) * 4;
            const float* res = reinterpret_cast<const float*>(smem + S::WARPS * S::RING);
            constexpr int ML = AT_PAIRS * S::PITCH, WARP = S::SUMS / 4;
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < S::WARPS; ++w) M = fmaxf(M, res[w * WARP + ML + 2 * r]);
            float4 a = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < S::WARPS; ++w) {
                const float mw = res[w * WARP + ML + 2 * r];
                const float wt = mw == -INFINITY ? 0.0f : ex2(mw - M);
                L += wt * res[w * WARP + ML + 2 * r + 1];
                const float4 v = *reinterpret_cast<const float4*>(res + w * WARP + r * S::PITCH + d);
                a.x += wt * v.x; a.y += wt * v.y; a.z += wt * v.z; a.w += wt * v.w;
            }
            if (whole) {
                const int pr = done.pr0 + r, j = pr / G;
                const float inv = 1.0f / L;
                *reinterpret_cast<float4*>(p.out + (int64_t)(done.row0 + j) * p.ldo + (int64_t)(done.hk * G + pr - j * G) * HD + d) =
                    make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
            } else {
                __stcg(reinterpret_cast<float4*>(slot + r * HD + d), a);
                if (d == 0) __stcg(reinterpret_cast<float2*>(slot + AT_PAIRS * HD + 2 * r), make_float2(M, L));
            }
        }
        if (!whole) {
            if (at == u_begin) split_first = true;
            else split_last = true;
            if (tid == 0) s_ends[at != u_begin] = done;
        }
        __syncthreads();   // the results are read, the next q may be written
        if (s_fail) {
            if (more) drain(min(seg.nt, S::STAGES));
            return;
        }
        if (!more) break;
    }

    // ---- shared items: the last of an item's CTAs to get here joins its parts
    if (!split_first && !split_last) return;
    int np[2] = {0, 0}, c0[2] = {0, 0};
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        if (!(x == 0 ? split_first : split_last)) continue;
        c0[x] = cta_of(s_ends[x].item0, U, C);
        np[x] = cta_of(s_ends[x].item0 + s_ends[x].units - 1, U, C) - c0[x] + 1;
    }
    if (tid == 0) {
        __threadfence();
#pragma unroll
        for (int x = 0; x < 2; ++x) s_join[x] = np[x] > 0 && atomicAdd(&counters[c0[x]], 1) == np[x] - 1;
        __threadfence();
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        if (!s_join[x]) continue;
        const AtSeg& e = s_ends[x];
        const bool first = U * c0[x] / C >= e.item0 - AT_ITEM;   // the item is the first of CTA c0's run
        auto part = [&](int c) { return parts + (int64_t)((c0[x] + c) * 2 + (c == 0 && !first)) * at_part_floats(HD); };
        for (int r = warp; r < e.npairs; r += S::WARPS) {   // a warp for a pair
            float* wt = reinterpret_cast<float*>(ring);
            const float* ml = parts + AT_PAIRS * HD + 2 * r;
            float M = -INFINITY, L = 0.0f;
            for (int c = lane; c < np[x]; c += 32) {
                wt[c] = __ldcg(ml + (part(c) - parts));
                M = fmaxf(M, wt[c]);
            }
            M = warp_max(M);
            for (int c = lane; c < np[x]; c += 32) {
                wt[c] = wt[c] == -INFINITY ? 0.0f : ex2(wt[c] - M);
                L += wt[c] * __ldcg(ml + (part(c) - parts) + 1);
            }
            L = warp_sum(L);
            __syncwarp();
            const int pr = e.pr0 + r, j = pr / G;
            float* dst = p.out + (int64_t)(e.row0 + j) * p.ldo + (int64_t)(e.hk * G + pr - j * G) * HD;
            const float inv = 1.0f / L;
            for (int d = 4 * lane; d < HD; d += 128) {
                float4 a = make_float4(0, 0, 0, 0);
                constexpr int AHEAD = 16;   // loads in flight
                for (int c = 0; c < np[x]; c += AHEAD) {
                    float4 v[AHEAD];
#pragma unroll
                    for (int y = 0; y < AHEAD; ++y)
                        v[y] = __ldcg(reinterpret_cast<const float4*>(part(min(c + y, np[x] - 1)) + r * HD + d));
#pragma unroll
                    for (int y = 0; y < AHEAD; ++y) {
                        const float w = c + y < np[x] ? wt[c + y] : 0.0f;
                        a.x += w * v[y].x; a.y += w * v[y].y; a.z += w * v[y].z; a.w += w * v[y].w;
                    }
                }
                *reinterpret_cast<float4*>(dst + d) = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
            }
            __syncwarp();   // wt is the next pair's
        }
        if (tid == 0) counters[c0[x]] = 0;
    }
}

template <int R>
int attend_r(const KvAttendParams& p, cudaStream_t s) {
    using S = AtShape<R>;
    static std::mutex mu;
    static unsigned long long done = 0;
    constexpr int smem = S::PREFIX + 8 * S::THREADS;
    {
        std::lock_guard<std::mutex> lk(mu);
        BREW_CUDA(smem_attr_per_device((const void*)kv_attend_kernel<R>, smem, &done));
    }
    const int ctas = std::min(AT_MAX_CTAS, S::CTAS_PER_SM * num_sms());
    KvAttendParams q = p;
    q.code_base = 0x64006400u;
    kv_attend_kernel<R><<<ctas, S::THREADS, smem, s>>>(q);
    BREW_CUDA(cudaGetLastError());
    count_launch();
    return BREW_OK;
}

}  // namespace

// The single-token kernel's part of the workspace; the prompt kernel's lies behind it.
static int64_t at_workspace(int head_size) {
    return KV_COUNTER_BYTES + ((int64_t)AT_MAX_CTAS * 2 * at_part_floats(head_size) * 4 + 255) / 256 * 256;
}
int64_t kv_attend_workspace(int head_size) { return at_workspace(head_size) + kv_prefill_workspace(head_size); }

int kv_attend_counters(int hd, void* workspace, int value, cudaStream_t s) {
    uint8_t* w = static_cast<uint8_t*>(workspace);
    BREW_CUDA(cudaMemsetAsync(w, value, KV_COUNTER_BYTES, s));
    if (kv_prefill_supported(hd)) BREW_CUDA(cudaMemsetAsync(w + at_workspace(hd), value, KV_COUNTER_BYTES, s));
    return BREW_OK;
}

int kv_attend_launch(int hd, const KvAttendParams& p0, cudaStream_t s) {
    KvAttendParams p = p0;
    const int64_t most = (int64_t)p.rows.max_rows * (p.kv.n_heads / p.kv.n_kv);
    p.pairs_min = !kv_prefill_supported(hd) ? INT64_MAX
                  : (int64_t)p.rows.n_rows * p.kv.n_heads >= AT_MANY_PAIRS ? AT_PROMPT_PAIRS : AT_PROMPT_PAIRS_FEW;
    p.prompts = most >= p.pairs_min;
    int rc;
    switch (hd / 32) {
        case 1: rc = attend_r<1>(p, s); break;
        case 2: rc = attend_r<2>(p, s); break;
        case 3: rc = attend_r<3>(p, s); break;
        case 4: rc = attend_r<4>(p, s); break;
        default: rc = attend_r<8>(p, s); break;
    }
    if (rc || !p.prompts) return rc;
    p.workspace = static_cast<uint8_t*>(p.workspace) + at_workspace(hd);
    return kv_prefill_launch(hd, p, s);
}

}  // namespace brew
