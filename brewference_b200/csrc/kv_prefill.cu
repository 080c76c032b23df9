// kv_prefill.cu — attention over the paged 4-bit K/V cache for prompt
// chunks, on the tcgen05 tensor cores.
//
// An item is 128 (row, head) pairs of one (sequence, kv head): the 128 lanes
// of tensor memory.  Keys go by in tiles of 64.  fp32 accuracy comes from
// fp16 operands in two parts: q and p (hi = fp16(x), lo = fp16(x - hi): 22
// bits) and the cached values, for which two parts are exact: d (c - 8) has
// 11 + 4 bits (in tiles with values past fp16 the scales under 2^-10 are rounded).  Three of the four products are made (lo lo is below 2^-22):
//   S = q_hi k_hi + q_hi k_lo + q_lo k_hi,   O = p_hi v_hi + p_hi v_lo + p_lo v_hi
// so nothing of the blocks' scales is left to the softmax.  q and p are the
// products' operands in tensor memory (as shared-memory operands they would be
// read again for every 64 keys, and shared memory would bound the kernel), k
// and v in shared memory in the K-major core-matrix layout, and each tile's O
// starts at 0 and is added in fp32 registers with the softmax's correction,
// because accumulation in tensor memory truncates.
//
// The tiles of all items, end to end, are cut into one equal run a CTA, an
// item's beginning and end (q, the output, a pipeline that empties) weighing 6
// tiles (2: 156 us, 4: 126, 6: 117, 9: 118 for ragged prompts of up to 700
// rows, before the registers were divided as they are).  Items that a cut divides leave parts (O, maximum, sum) in the
// workspace, which the last of their CTAs joins.
//
// 28 warps, the registers divided among them:
//   0        walks the run's items (a ring of descriptions in shared memory that
//            the others read) and copies their packed tiles (bulk copies)
//   1        issues q k, 24 MMAs of 64 columns a tile
//   2, 3     issue p v, a warp for each half of the dims: one half of O is read
//            while the other is made
//   4 .. 11  softmax: two warpgroups, every other tile; a thread is a row.  The
//            running maximum passes from one tile to the next in shared memory.
//   12 .. 19 add up O: a thread is half a row
//   20 .. 27 unpack: a warpgroup for K, which brings q too, one for V
// K, V, S, P and the packed tiles have two buffers or more, and the rings go on
// from item to item.
//
// Measured: a tile of 64 keys takes 1.4 us a CTA, where its 48 MMAs of 37
// cycles take 1.0 (a chunk of 512 rows at 4096 positions, 16/8 heads of 128:
// 63 us, of which 12 until the first product and 8 from the last to the joined
// output).  What bounds it is the other warps' work beside them: 7800 warp
// instructions a tile at 45% of the issue slots, in loops that have to stay in
// the instruction cache together (the waits as a dozen instructions each, not
// forty, took 15% off).
#include <algorithm>

#include "brew_internal.cuh"
#include "decode.cuh"
#include "kv_device.cuh"
#include "tc_device.cuh"

namespace brew {
namespace {

constexpr int PF_M = 128;              // pairs of an item
constexpr int PF_KT = 64;              // keys of a tile
constexpr int PF_GROUPS = PF_KT / KV_GROUP;
constexpr int PF_RAW = 4;              // packed tiles in flight
constexpr int PF_MAX_CTAS = 148;
constexpr int PF_RUN = 4;              // tiles of a run, at least
constexpr int PF_ITEM = 6;             // what an item costs beside its tiles, in tiles
constexpr float PF_PLOG2 = 9.0f;       // p is carried times 2^9 (2^13 in tiles whose values are taken 2^-4)
constexpr int PF_QS = 36, PF_OS = 20;  // floats from row to row where q and the output are turned: no bank twice

// Seven warpgroups; the first warp of each kind, and the registers of its
// threads (the sum over the warpgroups is what the block is launched with; 80
// for the softmax and 64 for the unpacking: 64.5 us for the chunk below against
// 61.7, 117 for the ragged prompts against 111).
constexpr int PF_W_SOFT = 4, PF_W_SUM = 12, PF_W_UNPACK = 20, PF_THREADS = 896;
constexpr int PF_ITEM_USERS = 3 + 24;   // warps that walk the run's items
constexpr int PF_REGS = 72, PF_REGS_ISSUE = 40, PF_REGS_SOFT = 72, PF_REGS_SUM = 88, PF_REGS_UNPACK = 72;
static_assert(PF_RAW <= 4, "rings of 4");
static_assert(PF_REGS_ISSUE + 2 * (PF_REGS_SOFT + PF_REGS_SUM + PF_REGS_UNPACK) <= 7 * PF_REGS, "registers");
static_assert(PF_REGS_ISSUE <= PF_REGS && PF_REGS_UNPACK <= PF_REGS && PF_REGS_SOFT >= PF_REGS && PF_REGS_SUM >= PF_REGS,
              "the first two kinds give registers up, the others take some");

// Tensor memory: S twice, O, q's parts, p's parts twice.
constexpr uint32_t PF_T_S = 0, PF_T_O = 128, PF_T_QH = 256, PF_T_QL = 320, PF_T_P = 384;

template <int R>
struct PfShape {
    static constexpr int HD = 32 * R;
    static constexpr int RAW_BYTES = PF_GROUPS * kv_group_bytes(R);
    // K: [dims / 8][key][16 B], the 8-dim pieces 32 bytes further apart than their 64 keys take, V: [keys / 8][dim][16 B],
    // groups of 8 dims 16 bytes further apart: the unpacking warps' stores fall into different banks
    static constexpr int K_PIECE = PF_KT * 16 + 32, K_PART = HD / 8 * K_PIECE;
    static constexpr int V_GROUP = 144, V_PIECE = HD / 8 * V_GROUP, V_PART = PF_KT / 8 * V_PIECE;
    static constexpr int K = PF_RAW * RAW_BYTES, V = K + 4 * K_PART, QSTAGE = V + 4 * V_PART;
    static constexpr int OSTAGE = QSTAGE + 4 * 32 * PF_QS * 4, REST = OSTAGE + 8 * 32 * PF_OS * 4;
};

// The (row, head) pairs of one (entry, kv head), 128 at a time, and the part
// of their keys that this CTA's run of tiles covers.
struct PfItem {
    KvEntry e;
    int b, hk, mt;       // entry, kv head, which 128 pairs
    int off;             // the item's first tile, counted from the run's beginning (negative: others have its beginning)
    int cnt;             // its tiles
    int pr0, npairs;
    int kmin, kmax;      // the keys that some pair sees
    int all_lo, all_hi;  // the keys that every pair sees
    int ta, n;           // the run's tiles of it
};

struct PfRest {
    uint64_t raw_full[PF_RAW], raw_empty[PF_RAW], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], s_empty[2];
    uint64_t p_full[2], p_empty[2], meta_full[4], ml_full[2], ml_empty[2], m_full[2][4], item_full[8], item_empty[8], part_full, last_full, q_full, q_empty[4], o_full[2], o_empty[2];
    uint64_t poison[4];         // of tile i & 3: its V rows with a NaN scale, a bit each
    int64_t all;                // the call's tiles and items' costs
    int ctas, len;              // CTAs that have some; this one's part
    PfItem item[8];             // of item j & 7
    uint32_t tmem;
    int last;
    float unscale[4];           // of tile i & 3: 16 where its values are taken times 2^-4
    float corr[4][PF_M];        // of tile i & 3: what O so far is multiplied by
    float m[2][PF_M];           // the running maximum behind tile i & 1
    float qmax[PF_M];           // the largest magnitudes of the item's q rows
    float sfac[4][PF_M];        // of item j & 3: scores are the products times this (log2)
    float2 ml[2][2][PF_M];      // of item j & 1 and a softmax warpgroup: maximum and sum of its tiles
};

// True in one lane.  In a branch on it 37 cycles go by from one M128 N64 K16 to
// the next, 56 in a branch on the lane's number.
__device__ __forceinline__ bool elect_one() {
    uint32_t p = 0;
    asm volatile(
        "{\n\t.reg .b32 r;\n\t.reg .pred q;\n\telect.sync r|q, 0xffffffff;\n\t@q mov.u32 %0, 1;\n\t}" : "+r"(p));
    return p != 0;
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
        "r"(accumulate)
        : "memory");
}
// kind::f16: D fp32, A and B fp16, K-major.
constexpr uint32_t umma_idesc_f16(int M, int N) {
    return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ float2 f2_float2(uint64_t x) {
    float2 d;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(x));
    return d;
}
template <int N>
__device__ __forceinline__ void regs_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Waits for a phase, some 4 million tries of at most a microsecond in which the
// warp sleeps (polling warps would take issue slots and shared-memory cycles
// from the working ones); false, in all lanes and recorded, if it does not
// come: the warp then leaves, and so, one after the other, do those that wait
// for it.  (Few instructions: the kernel's loops have to stay in the
// instruction cache together, and what follows a wait waits for its fetch.)
constexpr uint32_t PF_TRIES = 1u << 22;
__device__ __forceinline__ bool pf_wait_warp(uint64_t* bar, uint32_t parity, unsigned int* err) {
#pragma unroll 1
    for (uint32_t it = 0; it < PF_TRIES; ++it) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(1000u)
            : "memory");
        if (__all_sync(0xffffffffu, ok)) return true;
    }
    atomicOr(err, BREW_DEVERR_TIMEOUT_FULL);
    return false;
}

__device__ __forceinline__ void pf_range(const KvAttendParams& p, const KvEntry& e, int G, int mt, int& all_hi, int& kmin,
                                         int& kmax) {
    const int pr0 = mt * PF_M;
    all_hi = e.pos0 + pr0 / G;
    kmax = e.pos0 + (min(e.rows * G, pr0 + PF_M) - 1) / G;
    kmin = p.window > 0 ? max(0, all_hi - p.window + 1) : 0;
}
__device__ __forceinline__ void pf_set(const KvAttendParams& p, int G, int len, PfItem& x) {
    pf_range(p, x.e, G, x.mt, x.all_hi, x.kmin, x.kmax);
    x.pr0 = x.mt * PF_M;
    x.npairs = min(x.e.rows * G - x.pr0, PF_M);
    x.all_lo = p.window > 0 ? max(0, x.kmax - p.window + 1) : 0;
    x.cnt = x.kmax / PF_KT + 1 - x.kmin / PF_KT;
    const int first = max(0, -x.off);
    x.ta = x.kmin / PF_KT + first;
    x.n = min(x.cnt, len - x.off) - first;
}
// False behind the run's last item.
__device__ __forceinline__ bool pf_next(const KvAttendParams& p, int G, int len, PfItem& x) {
    x.off += x.cnt + PF_ITEM;
    if (x.off >= len) return false;
    if (++x.mt >= (x.e.rows * G + PF_M - 1) / PF_M) {
        x.mt = 0;
        if (++x.hk >= p.kv.n_kv) {
            x.hk = 0;
            do {
                if (++x.b >= p.rows.n_seqs) return false;
                x.e = kv_check_entry(p.kv, p.rows, x.b);
            } while ((int64_t)x.e.rows * G < p.pairs_min);
        }
    }
    pf_set(p, G, len, x);
    return true;
}

// Item j of the run (n = 0: behind the last), and giving its slot back.
__device__ __forceinline__ bool pf_item(PfRest& sh, int j, PfItem& x, unsigned int* err) {
    if (!pf_wait_warp(&sh.item_full[j & 7], j >> 3 & 1, err)) return false;
    x = sh.item[j & 7];
    return x.n > 0;
}
__device__ __forceinline__ void pf_item_done(PfRest& sh, int j, int lane) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.item_empty[j & 7]);
}

// The item's q rows to tensor memory: two fp16 parts times a power of two,
// amax * f in [2^13, 2^14).  A warp brings 32 rows, 32 dims of 4 rows a load,
// and turns them (lane = row) in shared memory: with a row a lane, a warp's
// loads would touch 32 lines each (4.6 us an item).
template <int R>
__device__ __forceinline__ void pf_q_at(const KvAttendParams& p, const PfItem& x, int G, int r, int64_t& at) {
    const int pi = x.pr0 + min(r, x.npairs - 1), qr = pi / G;   // missing pairs repeat the last one
    at = (int64_t)(x.e.row0 + qr) * p.ldq + (int64_t)(x.hk * G + pi - qr * G) * (32 * R);
}
// To L2, before it is wanted.
template <int R>
__device__ __forceinline__ void pf_q_ahead(const KvAttendParams& p, const PfItem& x, int G, int lane) {
#pragma unroll 1
    for (int r = lane; r < x.npairs; r += 32) {
        int64_t at;
        pf_q_at<R>(p, x, G, r, at);
#pragma unroll
        for (int d = 0; d < 32 * R; d += 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.q + at + d));
    }
}
__device__ __forceinline__ void pf_q_load(const KvAttendParams& p, int64_t row_at, int d, int lane, float4 (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k)   // dims d .. d + 31 of rows 4 k + lane / 8
        v[k] = *reinterpret_cast<const float4*>(p.q + __shfl_sync(0xffffffffu, row_at, 4 * k + (lane >> 3)) + d + 4 * (lane & 7));
}
// The rows' largest magnitudes, before the last item's products are made.
template <int R>
__device__ __forceinline__ void pf_q_max(const KvAttendParams& p, PfRest& sh, const PfItem& x, int G, int w, int lane) {
    int64_t row_at;
    pf_q_at<R>(p, x, G, 32 * w + lane, row_at);
    float amax[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) amax[k] = 0.0f;
#pragma unroll 1
    for (int d = 0; d < 32 * R; d += 32) {
        float4 v[8];
        pf_q_load(p, row_at, d, lane, v);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            amax[k] = fmaxf(amax[k], fmaxf(fmaxf(fabsf(v[k].x), fabsf(v[k].y)), fmaxf(fabsf(v[k].z), fabsf(v[k].w))));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) amax[k] = fmaxf(amax[k], __shfl_xor_sync(0xffffffffu, amax[k], o));
        if ((lane & 7) == k) sh.qmax[32 * w + 4 * k + (lane >> 3)] = amax[k];
    }
    __syncwarp();
}
template <int R>
__device__ __forceinline__ bool pf_q_store(const KvAttendParams& p, PfRest& sh, float* stage, uint32_t tmem, const PfItem& x, int G,
                                           int j, int w, int lane) {
    const int r = 32 * w + lane;
    int64_t row_at;
    pf_q_at<R>(p, x, G, r, row_at);
    stage += w * 32 * PF_QS;
    float4 v[8];
    pf_q_load(p, row_at, 0, lane, v);
    const int fe = min(253, max(1, 267 - (int)(__float_as_uint(sh.qmax[r]) >> 23)));
    const float f = copysignf(__uint_as_float((uint32_t)fe << 23), p.scale);
    // the last item's products are made, and sfac of four items before is read: the products of its tiles' successors
    // waited for that
    if (j > 0 && !pf_wait_warp(&sh.q_empty[(j - 1) & 3], (j - 1) >> 2 & 1, p.kv.err)) return false;
    tc_fence_after();
    // (never 0: a masked score is -inf times it)
    sh.sfac[j & 3][r] = fmaxf(fabsf(p.scale) * 1.44269504088896341f * __uint_as_float((uint32_t)(254 - fe) << 23), 1e-36f);
    const uint32_t tq = tmem + ((uint32_t)(32 * w) << 16);
#pragma unroll 1
    for (int d = 0; d < 32 * R; d += 32) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            *reinterpret_cast<float4*>(stage + (4 * k + (lane >> 3)) * PF_QS + 4 * (lane & 7)) = v[k];
        __syncwarp();
        if (d + 32 < 32 * R) pf_q_load(p, row_at, d + 32, lane, v);
#pragma unroll 1
        for (int c = 0; c < 32; c += 16) {   // dims (0, 4 | 1, 5 | 2, 6 | 3, 7) of each 8, as K's are unpacked
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 y = *reinterpret_cast<const float4*>(stage + lane * PF_QS + c + 8 * h);
                const float4 z = *reinterpret_cast<const float4*>(stage + lane * PF_QS + c + 8 * h + 4);
                split_half2(y.x * f, z.x * f, hi[4 * h], lo[4 * h]);
                split_half2(y.y * f, z.y * f, hi[4 * h + 1], lo[4 * h + 1]);
                split_half2(y.z * f, z.z * f, hi[4 * h + 2], lo[4 * h + 2]);
                split_half2(y.w * f, z.w * f, hi[4 * h + 3], lo[4 * h + 3]);
            }
            tmem_st8(tq + PF_T_QH + (d + c) / 2, hi);
            tmem_st8(tq + PF_T_QL + (d + c) / 2, lo);
        }
        __syncwarp();
    }
    tmem_st_wait();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.q_full);
    return true;
}

// What a copying or issuing warp (0 .. 3) has under way when it leaves: the last
// copies have landed, and the last commits (and with them the products) have
// arrived, before the CTA ends, also where some wait gave up.
__device__ __noinline__ void pf_drain(PfRest& sh, int warp, int tiles, int items, unsigned int* err) {
    if (warp == 0) {
#pragma unroll 1
        for (int n = max(0, tiles - PF_RAW); n < tiles; ++n) pf_wait_warp(&sh.raw_full[n % PF_RAW], n / PF_RAW & 1, err);
        return;
    }
    const int n = tiles - 1;
    if (n < 0) return;
    if (warp == 1) {
        pf_wait_warp(&sh.k_empty[n & 1], n >> 1 & 1, err);
        if (items > 0) pf_wait_warp(&sh.q_empty[(items - 1) & 3], (items - 1) >> 2 & 1, err);
    } else {
        pf_wait_warp(&sh.o_full[warp - 2], n & 1, err);
        pf_wait_warp(&sh.p_empty[n & 1], n >> 1 & 1, err);
    }
}

// A tile with a scale over 8188, or a NaN: bit 16, whether it is one that some
// row sees, and a number; below, the positions of group w with a NaN among V's.
template <int R>
__device__ __noinline__ uint32_t pf_rare(const uint8_t* tile, int k0, int kmin, int kmax, int w, int lane) {
    uint32_t seen = 0;
#pragma unroll 1
    for (int z = lane; z < PF_GROUPS * 16 * R; z += 32) {
        const int y = z / (16 * R), n = z % (16 * R);   // words of a group: 8 R of K's, 8 R of V's
        const uint32_t d = reinterpret_cast<const uint32_t*>(tile + y * kv_group_bytes(R) + 512 * R)[n] & 0x7FFF7FFFu;
        const int p0 = k0 + 16 * y + (n < 8 * R ? 2 * n / R : (n - 8 * R) / R * 2), p1 = n < 8 * R ? p0 : p0 + 1;
        const uint32_t d0 = d & 0xFFFFu, d1 = d >> 16;
        if (p0 >= kmin && p0 <= kmax && d0 < 0x7C00u) seen = max(seen, d0);
        if (p1 >= kmin && p1 <= kmax && d1 < 0x7C00u) seen = max(seen, d1);
    }
    bool nan = false;   // lane = position
#pragma unroll 1
    for (int y = 0; y < R && k0 + 16 * w <= kmax; ++y)
        nan |= (reinterpret_cast<const uint16_t*>(tile + w * kv_group_bytes(R) + 544 * R)[kv_vscale(R, lane & 15, y)] & 0x7FFFu) > 0x7C00u;
    return (__reduce_max_sync(0xffffffffu, seen) > 0x6FFFu ? 0x10000u : 0u) | (__ballot_sync(0xffffffffu, nan) & 0xFFFFu);
}

template <int R>
__global__ void __launch_bounds__(PF_THREADS, 1) kv_prefill_kernel(const __grid_constant__ KvAttendParams p) {
    using S = PfShape<R>;
    constexpr int HD = S::HD;
    extern __shared__ __align__(128) uint8_t smem[];
    PfRest& sh = *reinterpret_cast<PfRest*>(smem + S::REST);
    const KvView& kv = p.kv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n_kv = kv.n_kv, G = kv.n_heads / n_kv;

    if (warp == 0) {
        // ---- the run: the tiles of all items end to end (entries, kv heads, pairs, keys), before each item's what it
        // costs besides, cut into equal parts
        auto entry_tiles = [&](int b) -> int64_t {   // of one kv head; 0: the other kernel's (which records bad entries)
            KvEntry e = {};
            if (b < p.rows.n_seqs) e = kv_check_entry(kv, p.rows, b);
            const int mts = (int64_t)e.rows * G >= p.pairs_min ? (e.rows * G + PF_M - 1) / PF_M : 0;
            auto cost = [&](const KvEntry& y, int mt) {
                int hi, kmin, kmax;
                pf_range(p, y, G, mt, hi, kmin, kmax);
                return PF_ITEM + kmax / PF_KT + 1 - kmin / PF_KT;
            };
            int64_t t = 0;
            if (__reduce_max_sync(0xffffffffu, mts) <= 4) {
#pragma unroll 1
                for (int mt = 0; mt < mts; ++mt) t += cost(e, mt);
                return t;
            }
#pragma unroll 1
            for (uint32_t some = __ballot_sync(0xffffffffu, mts > 0); some; some &= some - 1) {   // long ones: a lane an item
                const int at = __ffs(some) - 1, its = __shfl_sync(0xffffffffu, mts, at);
                KvEntry y = {};
                y.pos0 = __shfl_sync(0xffffffffu, e.pos0, at);
                y.rows = __shfl_sync(0xffffffffu, e.rows, at);
                int64_t u = 0;
#pragma unroll 1
                for (int mt = lane; mt < its; mt += 32) u += cost(y, mt);
#pragma unroll
                for (int o = 16; o; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
                if (lane == at) t = u;
            }
            return t;
        };
        auto scan = [&](int64_t x) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t t = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += t;
            }
            return x;
        };
        int64_t all = 0, mine = 0, inc = 0;
        int items = 0;
#pragma unroll 1
        for (int b0 = 0; b0 < p.rows.n_seqs; b0 += 32) {
            mine = entry_tiles(b0 + lane);
            inc = scan(mine);
            all += __shfl_sync(0xffffffffu, inc, 31) * n_kv;
            items += __popc(__ballot_sync(0xffffffffu, mine > 0));
        }
        // fewer CTAs for little work: a cut item costs its join
        const int ctas = (int)min((int64_t)gridDim.x, max((int64_t)items * n_kv, (all + PF_RUN - 1) / PF_RUN));
        const int64_t t0 = all * blockIdx.x / max(ctas, 1), t1 = all * (blockIdx.x + 1) / max(ctas, 1);
        int len = blockIdx.x < ctas ? (int)(t1 - t0) : 0;
        if (len > 0) {
            int64_t rel = t0;
#pragma unroll 1
            for (int b0 = 0; b0 < p.rows.n_seqs; b0 += 32) {
                if (p.rows.n_seqs > 32) {
                    mine = entry_tiles(b0 + lane);
                    inc = scan(mine);
                }
                const int64_t here = __shfl_sync(0xffffffffu, inc, 31) * n_kv;
                if (rel >= here) {
                    rel -= here;
                    continue;
                }
                const int at = __ffs(__ballot_sync(0xffffffffu, inc * n_kv > rel)) - 1;
                rel -= __shfl_sync(0xffffffffu, inc - mine, at) * n_kv;
                const int64_t head = __shfl_sync(0xffffffffu, mine, at);
                const KvEntry e = kv_check_entry(kv, p.rows, b0 + at);
                const int hk = (int)(rel / head);
                rel -= hk * head;
#pragma unroll 1
                for (int m0 = 0;; m0 += 32) {
                    int cnt = 0;
                    if ((m0 + lane) * PF_M < e.rows * G) {
                        int hi, kmin, kmax;
                        pf_range(p, e, G, m0 + lane, hi, kmin, kmax);
                        cnt = PF_ITEM + kmax / PF_KT + 1 - kmin / PF_KT;
                    }
                    const int64_t up = scan(cnt), last = __shfl_sync(0xffffffffu, up, 31);
                    if (rel >= last) {
                        rel -= last;
                        continue;
                    }
                    const int w = __ffs(__ballot_sync(0xffffffffu, up > rel)) - 1;
                    if (lane == w) {
                        PfItem x;
                        x.e = e; x.b = b0 + at; x.hk = hk; x.mt = m0 + w;
                        x.off = PF_ITEM - (int)(rel - (up - cnt));
                        pf_set(p, G, len, x);
                        sh.item[0] = x;
                        if (x.off >= len) len = 0;   // nothing but the beginning of an item's cost
                    }
                    break;
                }
                break;
            }
        }
        len = __reduce_min_sync(0xffffffffu, len);
        if (lane == 0) {
            sh.all = all;
            sh.ctas = ctas;
            sh.len = len;
        }
    } else if (warp == 2 && lane == 0) {
        for (int i = 0; i < PF_RAW; ++i) {
            mbar_init(&sh.raw_full[i], 1);
            mbar_init(&sh.raw_empty[i], 8);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.k_full[i], 4);
            mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.v_full[i], 4);
            mbar_init(&sh.v_empty[i], 2);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.s_empty[i], 4);
            mbar_init(&sh.p_full[i], 4);
            mbar_init(&sh.p_empty[i], 2);
            mbar_init(&sh.o_full[i], 1);
            mbar_init(&sh.o_empty[i], 4);
            mbar_init(&sh.ml_full[i], 8);
            mbar_init(&sh.ml_empty[i], 8);
#pragma unroll 1
            for (int q = 0; q < 4; ++q) mbar_init(&sh.m_full[i][q], 1);
        }
        mbar_init(&sh.part_full, 8);
        mbar_init(&sh.last_full, 1);
        mbar_init(&sh.q_full, 4);
        for (int i = 0; i < 8; ++i) {
            mbar_init(&sh.item_full[i], 1);
            mbar_init(&sh.item_empty[i], PF_ITEM_USERS);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&sh.q_empty[i], 1);
            mbar_init(&sh.meta_full[i], 4);
        }
        fence_mbar_init();
    } else if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int len = sh.len;

    // i counts the run's tiles, j its items; a ring's slot and phase follow from them
    if (warp < PF_W_SOFT) {
        regs_dec<PF_REGS_ISSUE>();
        int i = 0, items = 0;   // tiles that this warp has copied or issued, items that it has issued whole
        if (warp == 0 && len > 0) {
            // ---------------- the run's items, and their copies: a group of 16 positions a lane ----------------
            const int per = 1 << (kv.page_shift - 4);
            PfItem x = sh.item[0];
            bool ok = true;
#pragma unroll 1
            for (int j = 0; ok; ++j) {
                if (j > 0) {
                    if (!pf_next(p, G, len, x)) x.n = 0;
                    if (!pf_wait_warp(&sh.item_empty[j & 7], (j >> 3 & 1) ^ 1, kv.err)) break;
                    if (lane == 0) sh.item[j & 7] = x;
                }
                if (lane == 0) mbar_arrive(&sh.item_full[j & 7]);
                if (x.n == 0) break;
                if (j > 0) pf_q_ahead<R>(p, x, G, lane);
                const int32_t* pages = kv.table + (int64_t)x.e.seq * kv.max_pages;
                auto page_of = [&](int t) {
                    const int pos = (x.ta + t) * PF_KT + 16 * lane;
                    return lane < PF_GROUPS && t < x.n && pos <= x.kmax ? pages[pos >> kv.page_shift] : -1;
                };
                int id = page_of(0);
#pragma unroll 1
                for (int t = 0; t < x.n && ok; ++t, ++i) {
                    const int st = i % PF_RAW;
                    ok = pf_wait_warp(&sh.raw_empty[st], (i / PF_RAW & 1) ^ 1, kv.err);
                    if (!ok) break;
                    const uint32_t have = __popc(__ballot_sync(0xffffffffu, id >= 0));
                    if (lane == 0) mbar_arrive_expect_tx(&sh.raw_full[st], have * kv_group_bytes(R));
                    __syncwarp();
                    if (id >= 0) {
                        const int grp = ((x.ta + t) * PF_KT + 16 * lane) >> 4 & (per - 1);
                        bulk_g2s(smem + st * S::RAW_BYTES + lane * kv_group_bytes(R),
                                 kv.pages + (((int64_t)id * n_kv + x.hk) * per + grp) * kv_group_bytes(R),
                                 kv_group_bytes(R), &sh.raw_full[st]);
                    }
                    id = page_of(t + 1);
                }
            }
        } else if (warp == 1 && len > 0) {
            // ---------------- MMA issue: S = q k ----------------
            constexpr uint32_t idesc = umma_idesc_f16(PF_M, PF_KT);
            const uint64_t kdesc = umma_desc_k(smem_u32(smem + S::K), S::K_PIECE, 128);
            PfItem x;
            bool ok = true;
#pragma unroll 1
            for (int j = 0; ok && pf_item(sh, j, x, kv.err); ++j) {
                ok = pf_wait_warp(&sh.q_full, j & 1, kv.err);
#pragma unroll 1
                for (int t = 0; t < x.n && ok; ++t, ++i) {
                    const int b = i & 1;
                    ok = pf_wait_warp(&sh.k_full[b], i >> 1 & 1, kv.err) &&
                         pf_wait_warp(&sh.s_empty[b], (i >> 1 & 1) ^ 1, kv.err);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t hi = kdesc + b * (2 * S::K_PART / 16);
                        const uint32_t d = tmem + PF_T_S + b * PF_KT;
#pragma unroll
                        for (int pass = 0; pass < 3; ++pass)
#pragma unroll
                            for (int s = 0; s < HD / 16; ++s)
                                umma_f16_ts(d, tmem + (pass == 0 ? PF_T_QL : PF_T_QH) + 8 * s,
                                            hi + ((pass == 1 ? S::K_PART : 0) + s * 2 * S::K_PIECE) / 16, idesc, pass + s > 0);
                        umma_commit(&sh.s_full[b]);
                        umma_commit(&sh.k_empty[b]);
                        if (t == x.n - 1) umma_commit(&sh.q_empty[j & 3]);
                    }
                    __syncwarp();
                }
                pf_item_done(sh, j, lane);
                items += ok;
            }
        } else if (warp >= 2 && len > 0) {
            // ---------------- MMA issue: O = p v, a warp for each half of the dims ----------------
            constexpr uint32_t idesc = umma_idesc_f16(PF_M, HD / 2);
            const int h = warp - 2;
            if (h == 1)   // the first item's q rows to L2
                pf_q_ahead<R>(p, sh.item[0], G, lane);
            const uint32_t to = tmem + PF_T_O + h * (HD / 2);
            const uint64_t vdesc = umma_desc_k(smem_u32(smem + S::V), S::V_PIECE, S::V_GROUP) + h * (HD / 16 * S::V_GROUP / 16);
            PfItem x;
            int j = 0, tiles = 0;
            bool ok = true;
#pragma unroll 1
            for (;; ++i) {
                if (i == tiles) {
                    if (!pf_item(sh, j, x, kv.err)) break;
                    tiles += x.n;
                    pf_item_done(sh, j++, lane);
                }
                const int b = i & 1;
                ok = pf_wait_warp(&sh.v_full[b], i >> 1 & 1, kv.err) && pf_wait_warp(&sh.o_empty[h], (i & 1) ^ 1, kv.err) &&
                     pf_wait_warp(&sh.p_full[b], i >> 1 & 1, kv.err);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t hi = vdesc + b * (2 * S::V_PART / 16);
                    const uint32_t tp = tmem + PF_T_P + b * PF_KT;
#pragma unroll
                    for (int pass = 0; pass < 3; ++pass)
#pragma unroll
                        for (int s = 0; s < PF_KT / 16; ++s)
                            umma_f16_ts(to, tp + (pass == 0 ? PF_KT / 2 : 0) + 8 * s,
                                        hi + ((pass == 1 ? S::V_PART : 0) + s * 2 * S::V_PIECE) / 16, idesc, pass + s > 0);
                    umma_commit(&sh.o_full[h]);
                    umma_commit(&sh.v_empty[b]);
                    umma_commit(&sh.p_empty[b]);
                }
                __syncwarp();
            }
        }
        __syncwarp();
        pf_drain(sh, warp, i, items, kv.err);
    } else if (warp < PF_W_SUM) {
        // ---------------- softmax: thread = row, a warpgroup every other tile ----------------
        regs_inc<PF_REGS_SOFT>();
        const int w = warp & 3, r = 32 * w + lane, b = (warp - PF_W_SOFT) / 4;
        const uint32_t tq = tmem + ((uint32_t)(32 * w) << 16), ts = tq + PF_T_S + b * PF_KT, tp = tq + PF_T_P + b * PF_KT;
        if (len > 0) {
            PfItem x;
            int i = 0;
            bool ok = true;
#pragma unroll 1
            for (int j = 0; ok && pf_item(sh, j, x, kv.err); ++j) {
                const int pi = x.pr0 + min(r, x.npairs - 1);   // missing pairs repeat the last one
                const int qpos = x.e.pos0 + pi / G, qlo = p.window > 0 ? qpos - p.window + 1 : 0;
                float m = -INFINITY, l = 0.0f, sfac = 0.0f;   // of this warpgroup's tiles
                bool fresh = true;
#pragma unroll 1
                for (int t = 0; t < x.n && ok; ++t, ++i) {
                    if ((i & 1) != b) continue;
                    ok = pf_wait_warp(&sh.s_full[b], i >> 1 & 1, kv.err);
                    if (!ok) break;
                    tc_fence_after();
                    if (fresh) sfac = sh.sfac[j & 3][r];
                    fresh = false;
                    const float up = sh.unscale[i & 3], f = sfac * up;
                    const int k0 = (x.ta + t) * PF_KT;
                    const bool full = k0 >= x.all_lo && k0 + PF_KT - 1 <= x.all_hi;   // no key is masked for any row
                    // the row's keys, as bits from k0 on
                    const uint64_t see = full ? ~0ull
                                              : (~0ull >> (63 - min(63, max(0, qpos - k0)))) & (~0ull << min(63, max(0, qlo - k0))) &
                                                    (qpos < k0 || qlo > k0 + 63 ? 0 : ~0ull);
                    // a NaN among V's scales: the rows that see its key become NaN, the others do not (the unpacked value is 0)
                    const uint64_t bad = sh.poison[i & 3];
                    if (bad & see) l = __uint_as_float(0x7fffffffu);
                    float mx = -INFINITY;
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        float v[32];
                        tmem_ld32(ts + 32 * h, v);
                        tmem_ld_wait();
                        if (!full) {
                            const uint32_t s32 = (uint32_t)(see >> 32 * h);
#pragma unroll
                            for (int c = 0; c < 32; ++c)
                                if (!(s32 >> c & 1)) v[c] = -INFINITY;
                        }
                        float a0 = v[0], a1 = v[1];
#pragma unroll
                        for (int c = 2; c < 32; c += 2) {
                            a0 = fmaxf(a0, v[c]);
                            a1 = fmaxf(a1, v[c + 1]);
                        }
                        mx = fmaxf(mx, fmaxf(a0, a1));
                    }
                    // the running maximum passes from one warpgroup's tile to the other's
                    if (i > 0) ok = pf_wait_warp(&sh.m_full[b ^ 1][w], (i - 1) >> 1 & 1, kv.err);
                    const float before = t == 0 ? -INFINITY : sh.m[b ^ 1][r];
                    const float mn = fmaxf(before, mx * f);
                    sh.m[b][r] = mn;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.m_full[b][w]);
                    const float corr = mn == before ? 1.0f : ex2(before - mn);   // before = -inf: 0
                    l *= mn == m ? 1.0f : ex2(m - mn);
                    m = mn;
                    // p times 2^9, and 2^4 more where the values are taken times 2^-4
                    const float mref = m == -INFINITY ? 0.0f : PF_PLOG2 + (up == 1.0f ? 0.0f : 4.0f) - m;
                    const uint64_t f2 = f2_packf(f, f), mref2 = f2_packf(mref, mref), minus = f2_packf(-1.0f, -1.0f);
                    ok = ok && pf_wait_warp(&sh.p_empty[b], (i >> 1 & 1) ^ 1, kv.err);   // and corr of four tiles before is read
                    if (!ok) break;
                    tc_fence_after();
                    uint64_t sum = f2_packf(0.0f, 0.0f);
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        float v[32];
                        tmem_ld32(ts + 32 * h, v);
                        tmem_ld_wait();
                        if (h == 1) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&sh.s_empty[b]);
                        }
                        if (!full) {
                            const uint32_t s32 = (uint32_t)(see >> 32 * h);
#pragma unroll
                            for (int c = 0; c < 32; ++c)
                                if (!(s32 >> c & 1)) v[c] = -INFINITY;
                        }
#pragma unroll
                        for (int c = 0; c < 32; c += 16) {
                            uint32_t hi[8], lo[8];
#pragma unroll
                            for (int y = 0; y < 16; y += 2) {
                                const float2 a = f2_float2(f2_fma(f2_packf(v[c + y], v[c + y + 1]), f2, mref2));
                                const float p0 = ex2(a.x), p1 = ex2(a.y);
                                const uint64_t pp = f2_packf(p0, p1);
                                sum = f2_add(sum, pp);
                                const __half2 ph = __floats2half2_rn(p0, p1);
                                const float2 pf = __half22float2(ph);
                                hi[y / 2] = *reinterpret_cast<const uint32_t*>(&ph);
                                const float2 rest = f2_float2(f2_fma(f2_packf(pf.x, pf.y), minus, pp));
                                lo[y / 2] = pack_half2(rest.x, rest.y);
                            }
                            tmem_st8(tp + 16 * h + c / 2, hi);
                            tmem_st8(tp + PF_KT / 2 + 16 * h + c / 2, lo);
                        }
                    }
                    const float2 sf = f2_float2(sum);
                    l = fmaf(sf.x + sf.y, up == 1.0f ? 1.0f : 0.0625f, l);
                    sh.corr[i & 3][r] = corr;
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.p_full[b]);
                }
                ok = ok && pf_wait_warp(&sh.ml_empty[j & 1], (j >> 1 & 1) ^ 1, kv.err);
                sh.ml[j & 1][b][r] = make_float2(m, l);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.ml_full[j & 1]);
                pf_item_done(sh, j, lane);
            }
        }
    } else if (warp < PF_W_UNPACK) {
        // ---------------- O: thread = row, half of its dims ----------------
        regs_inc<PF_REGS_SUM>();
        constexpr int NC = HD / 2;
        const int w8 = warp - PF_W_SUM, w = warp & 3, r = 32 * w + lane, c0 = w8 / 4 * NC;
        const uint32_t to = tmem + ((uint32_t)(32 * w) << 16) + PF_T_O + c0;
        float* stage = reinterpret_cast<float*>(smem + S::OSTAGE) + w8 * 32 * PF_OS;
        if (len > 0) {
            PfItem x;
            int i = 0, cuts = 0;
            bool ok = true;
#pragma unroll 1
            for (int j = 0; ok && pf_item(sh, j, x, kv.err); ++j) {
                uint64_t o[NC / 2];
#pragma unroll
                for (int c = 0; c < NC / 2; ++c) o[c] = 0;
#pragma unroll 1
                for (int t = 0; t < x.n && ok; ++t, ++i) {
                    ok = pf_wait_warp(&sh.o_full[w8 / 4], i & 1, kv.err);
                    if (!ok) break;
                    tc_fence_after();
                    const float corr = sh.corr[i & 3][r];
                    const uint64_t corr2 = f2_packf(corr, corr);
#pragma unroll
                    for (int h = 0; h < NC; h += 16) {
                        float v[16];
                        tmem_ld16(to + h, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 16; c += 2) o[(h + c) / 2] = f2_fma(o[(h + c) / 2], corr2, f2_packf(v[c], v[c + 1]));
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.o_empty[w8 / 4]);
                }
                // the item's end
                ok = ok && pf_wait_warp(&sh.ml_full[j & 1], j >> 1 & 1, kv.err);
                if (!ok) break;
                const float2 ml0 = sh.ml[j & 1][0][r], ml1 = sh.ml[j & 1][1][r];
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.ml_empty[j & 1]);
                const float m = fmaxf(ml0.x, ml1.x);
                const float l = ml0.y * (ml0.x == -INFINITY ? 0.0f : ex2(ml0.x - m)) +
                                ml1.y * (ml1.x == -INFINITY ? 0.0f : ex2(ml1.x - m));
                const int pi = x.pr0 + min(r, x.npairs - 1), qr = pi / G;
                const int64_t row_at = (int64_t)(x.e.row0 + qr) * p.ldo + (int64_t)(x.hk * G + pi - qr * G) * HD + c0;
                // 16 dims of the warp's rows go to `out` by way of shared memory: 64 bytes of 8 rows at a time
                auto write = [&](int c, const float (&v)[16]) {
#pragma unroll
                    for (int k = 0; k < 16; k += 4)
                        *reinterpret_cast<float4*>(stage + lane * PF_OS + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 32; k += 8) {
                        const int row = k + (lane >> 2);
                        const int64_t at = __shfl_sync(0xffffffffu, row_at, row);
                        const float4 y = *reinterpret_cast<const float4*>(stage + row * PF_OS + 4 * (lane & 3));
                        if (32 * w + row < x.npairs) *reinterpret_cast<float4*>(p.out + at + c + 4 * (lane & 3)) = y;
                    }
                    __syncwarp();
                };
                if (x.off >= 0 && x.off + x.cnt <= len) {
                    const float f = 1.0f / l;
#pragma unroll
                    for (int c = 0; c < NC; c += 16) {
                        float v[16];
#pragma unroll
                        for (int k = 0; k < 16; k += 2) {
                            const float2 y = f2_float2(o[(c + k) / 2]);
                            v[k] = y.x * f;
                            v[k + 1] = y.y * f;
                        }
                        write(c, v);
                    }
                } else {
                    // others have parts of it: the last of its CTAs to arrive joins them.  A CTA keeps at most two: of an
                    // item that begins before its run, and of one that ends behind it.
                    const int64_t begin = sh.all * blockIdx.x / sh.ctas + x.off;
                    const int cta0 = (int)(((begin + 1) * sh.ctas - 1) / sh.all);
                    const int parts = (int)(((begin + x.cnt) * sh.ctas - 1) / sh.all) - cta0 + 1;
                    int* counter = reinterpret_cast<int*>(p.workspace) + cta0;
                    float* ws = reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + KV_COUNTER_BYTES);
                    auto part = [&](int k) { return ws + (int64_t)(2 * (cta0 + k) + (k == 0)) * (PF_M * (HD + 4)); };
                    float* mine = part(blockIdx.x - cta0);
#pragma unroll
                    for (int c = 0; c < NC; c += 4) {
                        const float2 y0 = f2_float2(o[c / 2]), y1 = f2_float2(o[c / 2 + 1]);
                        __stcg(reinterpret_cast<float4*>(mine) + (w8 * (NC / 4) + c / 4) * 32 + lane,
                               make_float4(y0.x, y0.y, y1.x, y1.y));
                    }
                    if (c0 == 0) __stcg(reinterpret_cast<float2*>(mine + PF_M * HD) + r, make_float2(m, l));
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.part_full);
                    if (w8 == 0) {
                        ok = pf_wait_warp(&sh.part_full, cuts & 1, kv.err);
                        if (!ok) break;
                        if (lane == 0) {
                            __threadfence();
                            const int last = atomicAdd(counter, 1) == parts - 1;
                            __threadfence();
                            sh.last = last;
                            if (last) *counter = 0;
                            mbar_arrive(&sh.last_full);
                        }
                        __syncwarp();
                    }
                    ok = pf_wait_warp(&sh.last_full, cuts & 1, kv.err);
                    if (!ok) break;
                    ++cuts;
                    if (sh.last) {
                        float M = -INFINITY, L = 0.0f;
#pragma unroll 4
                        for (int k = 0; k < parts; ++k) {
                            const float2 y = __ldcg(reinterpret_cast<const float2*>(part(k) + PF_M * HD) + r);
                            const float n = fmaxf(M, y.x);
                            L = L * (M == n ? 1.0f : ex2(M - n)) + y.y * (y.x == -INFINITY ? 0.0f : ex2(y.x - n));
                            M = n;
                        }
                        const float inv = 1.0f / L;
#pragma unroll 1
                        for (int c = 0; c < NC; c += 16) {
                            float v[16];
#pragma unroll
                            for (int k = 0; k < 16; ++k) v[k] = 0.0f;
                            const float4* at = reinterpret_cast<const float4*>(part(0)) + (w8 * (NC / 4) + c / 4) * 32 + lane;
                            const float2* ml = reinterpret_cast<const float2*>(part(0) + PF_M * HD) + r;
                            // (the first part is the second of its CTA's, the others are the first of theirs)
                            constexpr int64_t STEP = PF_M * (HD + 4) / 4;
#pragma unroll 4
                            for (int k = 0; k < parts; ++k) {
                                const float my = __ldcg(ml).x;
                                float4 z[4];
#pragma unroll
                                for (int y = 0; y < 4; ++y) z[y] = __ldcg(at + 32 * y);
                                const float a = my == -INFINITY ? 0.0f : ex2(my - M) * inv;
#pragma unroll
                                for (int y = 0; y < 4; ++y) {
                                    v[4 * y] += a * z[y].x;
                                    v[4 * y + 1] += a * z[y].y;
                                    v[4 * y + 2] += a * z[y].z;
                                    v[4 * y + 3] += a * z[y].w;
                                }
                                at += k == 0 ? STEP : 2 * STEP;
                                ml += k == 0 ? 2 * STEP : 4 * STEP;
                            }
                            write(c, v);
                        }
                    }
                }
                pf_item_done(sh, j, lane);
            }
        }
    } else {
        // ---------------- unpacking: warp = group of the tile, a warpgroup for K and q, one for V ----------------
        regs_dec<PF_REGS_UNPACK>();
        const int w = warp & 3, g = lane >> 2, q = lane & 3;
        const bool is_k = warp < PF_W_UNPACK + 4;
        const uint32_t base = p.code_base;
        if (len > 0) {
            PfItem x;
            int i = 0;
            bool ok = true;
#pragma unroll 1
            for (int j = 0; ok && pf_item(sh, j, x, kv.err); ++j) {
                if (is_k) pf_q_max<R>(p, sh, x, G, w, lane);
#pragma unroll 1
                for (int t = 0; t < x.n; ++t, ++i) {
                    const int b = i & 1, st = i % PF_RAW;
                    const uint8_t* tile = smem + st * S::RAW_BYTES;
                    const uint8_t* raw = tile + w * kv_group_bytes(R);
                    const int k0 = (x.ta + t) * PF_KT;
                    ok = pf_wait_warp(&sh.raw_full[st], i / PF_RAW & 1, kv.err);
                    if (!ok) break;
                    if (is_k) {
                        // The largest scale of the tile's live groups (as fp16 bits): above 8188 its values are taken times
                        // 2^-4, so that d (c - 8) stays in fp16's range; above infinity some are NaN.  (2^-4 rounds scales
                        // under 2^-10 to multiples of 2^-20: beside a value past 65504 that some row of the item sees.)
                        uint32_t top = 0;
#pragma unroll
                        for (int y = 0; y < PF_GROUPS; ++y)
                            if (k0 + 16 * y <= x.kmax)
#pragma unroll
                                for (int z = lane; z < 16 * R; z += 32)
                                    top = __vmaxu2(top, reinterpret_cast<const uint32_t*>(tile + y * kv_group_bytes(R) + 512 * R)[z] &
                                                            0x7FFF7FFFu);
                        top = __reduce_max_sync(0xffffffffu, max(top & 0xFFFFu, top >> 16));
                        uint32_t rare = 0;   // bit 16: some value is past fp16; below: V's positions with a NaN
                        if (top > 0x6FFFu) rare = pf_rare<R>(tile, k0, x.kmin, x.kmax, w, lane);
                        const bool big = rare >> 16;
                        const uint32_t nan = rare & 0xFFFFu;
                        ok = pf_wait_warp(&sh.k_empty[b], (i >> 1 & 1) ^ 1, kv.err);
                        if (!ok) break;
                        if (lane == 0) {
                            reinterpret_cast<uint16_t*>(&sh.poison[i & 3])[w] = (uint16_t)nan;
                            if (w == 0) sh.unscale[i & 3] = big ? 16.0f : 1.0f;
                            mbar_arrive(&sh.meta_full[i & 3]);
                        }
                        const uint32_t shrink = big ? 0x2C002C00u : 0x3C003C00u;   // 2^-4 or 1
                        uint8_t* kd = smem + S::K + b * 2 * S::K_PART;
#pragma unroll 1
                        for (int u = 0; u < 2; ++u) {   // key 8 u + g, dims 32 y + 8 q .. + 7
                            uint32_t c4[R];
                            __half d[R];
                            load_words<R>(c4, raw, u, lane);
                            load_kscales<R>(d, raw + 512 * R, 8 * u + g);
#pragma unroll
                            for (int y = 0; y < R; ++y) {
                                __half2 dd = __half2half2(d[y]);
                                uint32_t d2 = *reinterpret_cast<uint32_t*>(&dd), c[4];
                                d2 = mul_h2(d2, shrink);
                                unpack(c, c4[y], base);
                                uint4 hi, lo;
                                hi.x = mul_h2(c[0], d2); lo.x = fma_h2(c[0], d2, neg_h2(hi.x));
                                hi.y = mul_h2(c[1], d2); lo.y = fma_h2(c[1], d2, neg_h2(hi.y));
                                hi.z = mul_h2(c[2], d2); lo.z = fma_h2(c[2], d2, neg_h2(hi.z));
                                hi.w = mul_h2(c[3], d2); lo.w = fma_h2(c[3], d2, neg_h2(hi.w));
                                uint8_t* at = kd + (4 * y + q) * S::K_PIECE + (16 * w + 8 * u + g) * 16;
                                *reinterpret_cast<uint4*>(at) = hi;
                                *reinterpret_cast<uint4*>(at + S::K_PART) = lo;
                            }
                        }
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(&sh.k_full[b]);
                            mbar_arrive(&sh.raw_empty[st]);
                        }
                        if (t == 0)   // behind the first tile's K, which does not wait for the last item's products
                            ok = pf_q_store<R>(p, sh, reinterpret_cast<float*>(smem + S::QSTAGE), tmem, x, G, j, w, lane);
                        if (!ok) break;
                    } else {
                        // (K's warps are at most the packed tiles in flight ahead: unscale and poison are still this tile's)
                        ok = pf_wait_warp(&sh.meta_full[i & 3], i >> 2 & 1, kv.err) &&
                             pf_wait_warp(&sh.v_empty[b], (i >> 1 & 1) ^ 1, kv.err);
                        if (!ok) break;
                        const uint32_t shrink = sh.unscale[i & 3] != 1.0f ? 0x2C002C00u : 0x3C003C00u;   // 2^-4 or 1
                        const uint32_t nan = reinterpret_cast<const uint16_t*>(&sh.poison[i & 3])[w];
                        uint8_t* vd = smem + S::V + b * 2 * S::V_PART;
#pragma unroll 1
                        for (int u = 0; u < 2; ++u) {   // keys 8 u + 2 q, + 1, dims 32 y + 4 g .. + 3
                            uint32_t c4[R], d[R];
                            load_words<R>(c4, raw + 256 * R, u, lane);
                            load_scales<R>(d, raw + 544 * R, u, q);
                            // keys that no row sees may hold anything: 0
                            const int key = 8 * u + 2 * q, pos = k0 + 16 * w + key;
                            const uint32_t live = (pos > x.kmax || pos < x.kmin || (nan >> key & 1) ? 0u : 0xFFFFu) |
                                                  (pos + 1 > x.kmax || pos + 1 < x.kmin || (nan >> key & 2) ? 0u : 0xFFFF0000u);
#pragma unroll
                            for (int y = 0; y < R; ++y) {
                                uint32_t d2 = d[y] & live, c[4];
                                d2 = mul_h2(d2, shrink);
                                unpack(c, c4[y], base);
#pragma unroll
                                for (int z = 0; z < 4; ++z) {
                                    const uint32_t hi = mul_h2(c[z], d2), lo = fma_h2(c[z], d2, neg_h2(hi));
                                    uint8_t* at = vd + (2 * w + u) * S::V_PIECE + (4 * y + (g >> 1)) * S::V_GROUP +
                                                  (4 * (g & 1) + z) * 16 + 4 * q;
                                    *reinterpret_cast<uint32_t*>(at) = hi;
                                    *reinterpret_cast<uint32_t*>(at + S::V_PART) = lo;
                                }
                            }
                        }
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(&sh.v_full[b]);
                            mbar_arrive(&sh.raw_empty[st]);
                        }
                    }
                }
                pf_item_done(sh, j, lane);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    pdl_wait();   // the single-token kernel: what comes after this one on the stream comes after both
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <int R>
int prefill_r(const KvAttendParams& p, cudaStream_t s) {
    using S = PfShape<R>;
    static std::mutex mu;
    static unsigned long long done = 0;
    constexpr int smem = S::REST + (int)sizeof(PfRest);
    static_assert(smem <= 227 * 1024, "shared memory");
    {
        std::lock_guard<std::mutex> lk(mu);
        BREW_CUDA(smem_attr_per_device((const void*)kv_prefill_kernel<R>, smem, &done));
        static bool checked = false;
        // the warpgroups' shares of the registers come out of what the block is launched with
        if (!checked) {
            cudaFuncAttributes a;
            BREW_CUDA(cudaFuncGetAttributes(&a, (const void*)kv_prefill_kernel<R>));
            BREW_CHECK(a.numRegs >= PF_REGS, BREW_ERR_CUDA, "the prompt attention kernel has %d registers a thread",
                       a.numRegs);
            checked = true;
        }
    }
    KvAttendParams q = p;
    q.code_base = 0x64006400u;
    // starts beside the single-token kernel of the call, which has nothing to do where all entries are prompts
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(std::min(PF_MAX_CTAS, num_sms()));
    cfg.blockDim = dim3(PF_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    BREW_CUDA(cudaLaunchKernelEx(&cfg, kv_prefill_kernel<R>, q));
    count_launch();
    return BREW_OK;
}

}  // namespace

bool kv_prefill_supported(int hd) { return hd == 64 || hd == 128; }

int64_t kv_prefill_workspace(int hd) {
    return kv_prefill_supported(hd) ? KV_COUNTER_BYTES + (int64_t)2 * PF_MAX_CTAS * PF_M * (hd + 4) * 4 : 0;
}

int kv_prefill_launch(int hd, const KvAttendParams& p, cudaStream_t s) {
    return hd == 64 ? prefill_r<2>(p, s) : prefill_r<4>(p, s);
}

}  // namespace brew
