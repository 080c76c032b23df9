// kv_prefill.cu — attention over the paged 4-bit K/V cache for prompt
// chunks, on the tcgen05 tensor cores.
//
// An item is 128 (row, head) pairs of one (sequence, kv head): the 128 lanes
// of tensor memory.  Keys go by in tiles of 64.  fp32 accuracy comes from
// fp16 operands in two parts: q and p (hi = fp16(x), lo = fp16(x - hi): 22
// bits) and the cached values, for which two parts are exact: d (c - 8) has
// 11 + 4 bits.  Three of the four products are made (lo lo is below 2^-22):
//   S = q_hi k_hi + q_hi k_lo + q_lo k_hi,   O = p_hi v_hi + p_hi v_lo + p_lo v_hi
// so nothing of the blocks' scales is left to the softmax.  q and p are the
// products' operands in tensor memory (as shared-memory operands they would be
// read again for every 64 keys, and shared memory would bound the kernel), k
// and v in shared memory in the K-major core-matrix layout, and each tile's O
// starts at 0 and is added in fp32 registers with the softmax's correction,
// because accumulation in tensor memory truncates.
//
// Warps: one copies the tiles' packed groups (bulk copies), one thread issues
// the MMAs, four make the softmax (a thread is a row), eight add up O (a
// thread is half a row), four unpack K and V.  K, V, S and the packed tiles
// are buffered twice or more; QK of the next tile is issued before PV of the
// present one, so the tensor cores work while the softmax does.
//
// Bound: the tensor cores, 1536 cycles a tile of 64 keys x 128 pairs x 128
// dims (3 + 3 products), beside about 3400 instructions of the 16 warps.
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
constexpr int PF_RAW = 3;              // packed tiles in flight
constexpr int PF_WARPS = 18;
constexpr int PF_THREADS = 32 * PF_WARPS;
constexpr int PF_W_SUM = 6, PF_W_UNPACK = 14;   // first warps of the sums and the unpacking (0 copies, 1 issues)
constexpr float PF_PLOG2 = 9.0f;       // p is carried times 2^9 (2^13 in tiles whose values are taken 2^-4)
constexpr int PF_MAX_PARTS = 148;      // parts of split items

// Tensor memory: S twice, O, q's parts, p's parts.
constexpr uint32_t PF_T_S = 0, PF_T_O = 128, PF_T_QH = 256, PF_T_QL = 320, PF_T_PH = 384, PF_T_PL = 416;

template <int R>
struct PfShape {
    static constexpr int HD = 32 * R;
    static constexpr int RAW_BYTES = PF_GROUPS * kv_group_bytes(R);
    // K: [dims / 8][key][16 B], the 8-dim pieces 32 bytes further apart than their 64 keys take, V: [keys / 8][dim][16 B],
    // groups of 8 dims 16 bytes further apart: the unpacking warps' stores fall into different banks
    static constexpr int K_PIECE = PF_KT * 16 + 32, K_PART = HD / 8 * K_PIECE;
    static constexpr int V_GROUP = 144, V_PIECE = HD / 8 * V_GROUP, V_PART = PF_KT / 8 * V_PIECE;
    static constexpr int K = PF_RAW * RAW_BYTES, V = K + 4 * K_PART, REST = V + 4 * V_PART;
};

struct PfRest {
    uint64_t raw_full[PF_RAW], raw_empty[PF_RAW], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], s_empty[2];
    uint64_t q_full, p_full, p_empty, o_full, o_empty, fin;
    uint32_t tmem;
    int last;
    int abort;
    float corr[2][PF_M], m[PF_M], l[PF_M];
    float unscale[4];           // of tile i & 3: 16 where its values are taken times 2^-4
    uint32_t poison[4][PF_GROUPS];   // its V rows with a NaN scale, a bit each
};

// True in one lane.  In a branch on it the compiler keeps an MMA's operands in
// uniform registers: 37 cycles from one M128 N64 K16 to the next, 56 in a
// branch on the lane's number.
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

// One try of at most about 0.1 ms in which the thread sleeps: polling warps
// would take issue slots and shared-memory cycles from the working ones.
__device__ __forceinline__ bool pf_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(100000u)
        : "memory");
    return ok != 0;
}

// Waits for a phase, at most a second, or until another warp of the CTA has
// given up (which is recorded).
__device__ __forceinline__ bool pf_wait(uint64_t* bar, uint32_t parity, PfRest& s, unsigned int* err) {
    if (pf_try(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    for (uint32_t it = 0; it < BREW_SPIN_LIMIT; ++it) {
        if (pf_try(bar, parity)) return true;
        if (ld_volatile_int(&s.abort) || global_ns() - t0 > 1000000000ull) break;
    }
    s.abort = 1;
    atomicOr(err, BREW_DEVERR_TIMEOUT_FULL);
    return false;
}
__device__ __forceinline__ bool pf_wait_warp(uint64_t* bar, uint32_t parity, PfRest& s, unsigned int* err) {
    return __all_sync(0xffffffffu, pf_wait(bar, parity, s, err));
}

template <int R>
__global__ void __launch_bounds__(PF_THREADS, 1) kv_prefill_kernel(const __grid_constant__ KvAttendParams p, int splits) {
    using S = PfShape<R>;
    constexpr int HD = S::HD;
    extern __shared__ __align__(128) uint8_t smem[];
    PfRest& sh = *reinterpret_cast<PfRest*>(smem + S::REST);
    const KvView& kv = p.kv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n_kv = kv.n_kv, G = kv.n_heads / n_kv;

    // ---- this CTA's item: the entries' items end to end, the long ones of each first
    const int split = blockIdx.x % splits;
    int64_t rel = blockIdx.x / splits;
    const int64_t item = rel;
    KvEntry e = {};
    int tiles_m = 0;
    for (int b0 = 0; b0 < p.rows.n_seqs; b0 += 32) {   // every warp for itself, 32 entries at a time
        int mine = 0;
        if (b0 + lane < p.rows.n_seqs) {
            const KvEntry x = kv_check_entry(kv, p.rows, b0 + lane);   // (the other kernel of the call records bad ones)
            if ((int64_t)x.rows * G >= p.pairs_min) mine = (int)(((int64_t)x.rows * G + PF_M - 1) / PF_M);
        }
        int inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        const int64_t all = (int64_t)__shfl_sync(0xffffffffu, inc, 31) * n_kv;
        if (rel >= all) {
            rel -= all;
            continue;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, (int64_t)inc * n_kv > rel);
        const int at = __ffs(past) - 1;
        rel -= (int64_t)(__shfl_sync(0xffffffffu, inc - mine, at)) * n_kv;
        tiles_m = __shfl_sync(0xffffffffu, mine, at);
        e = kv_check_entry(kv, p.rows, b0 + at);
        break;
    }
    if (tiles_m == 0) return;
    const int hk = (int)(rel / tiles_m), pr0 = (tiles_m - 1 - (int)(rel % tiles_m)) * PF_M;
    const int npairs = (int)min((int64_t)e.rows * G - pr0, (int64_t)PF_M);
    const int all_hi = e.pos0 + pr0 / G, kmax = e.pos0 + (pr0 + npairs - 1) / G;   // the first and last pair's positions
    const int kmin = p.window > 0 ? max(0, all_hi - p.window + 1) : 0;
    const int all_lo = p.window > 0 ? max(0, kmax - p.window + 1) : 0;
    const int tiles = kmax / PF_KT + 1 - kmin / PF_KT;
    const int ta = kmin / PF_KT + (int)((int64_t)tiles * split / splits);
    const int n = kmin / PF_KT + (int)((int64_t)tiles * (split + 1) / splits) - ta;   // this CTA's tiles

    if (tid == 0) {
        for (int i = 0; i < PF_RAW; ++i) {
            mbar_init(&sh.raw_full[i], 1);
            mbar_init(&sh.raw_empty[i], 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.k_full[i], 4);
            mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.v_full[i], 4);
            mbar_init(&sh.v_empty[i], 1);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.s_empty[i], 4);
        }
        mbar_init(&sh.q_full, 4);
        mbar_init(&sh.p_full, 4);
        mbar_init(&sh.p_empty, 1);
        mbar_init(&sh.o_full, 1);
        mbar_init(&sh.o_empty, 8);
        mbar_init(&sh.fin, 4);
        sh.abort = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;

    if (warp == 0) {
        // ---------------- copies: a group of 16 positions a lane ----------------
        const int32_t* pages = kv.table + (int64_t)e.seq * kv.max_pages;
        const int per = 1 << (kv.page_shift - 4);
        auto page_of = [&](int i) {
            const int pos = (ta + i) * PF_KT + 16 * lane;
            return lane < PF_GROUPS && i < n && pos <= kmax ? pages[pos >> kv.page_shift] : -1;
        };
        int id = page_of(0);
        for (int i = 0; i < n; ++i) {
            const int st = i % PF_RAW;
            if (!pf_wait_warp(&sh.raw_empty[st], (i / PF_RAW & 1) ^ 1, sh, kv.err)) break;
            const uint32_t have = __popc(__ballot_sync(0xffffffffu, id >= 0));
            if (lane == 0) mbar_arrive_expect_tx(&sh.raw_full[st], have * kv_group_bytes(R));
            __syncwarp();
            if (id >= 0) {
                const int grp = ((ta + i) * PF_KT + 16 * lane) >> 4 & (per - 1);
                bulk_g2s(smem + st * S::RAW_BYTES + lane * kv_group_bytes(R),
                         kv.pages + (((int64_t)id * n_kv + hk) * per + grp) * kv_group_bytes(R), kv_group_bytes(R),
                         &sh.raw_full[st]);
            }
            id = page_of(i + 1);
        }
    } else if (warp == 1) {
        // ---------------- MMA issue ----------------
        if (n > 0) {
            constexpr uint32_t iqk = umma_idesc_f16(PF_M, PF_KT), ipv = umma_idesc_f16(PF_M, HD);
            const uint64_t kdesc = umma_desc_k(smem_u32(smem + S::K), S::K_PIECE, 128);
            const uint64_t vdesc = umma_desc_k(smem_u32(smem + S::V), S::V_PIECE, S::V_GROUP);
            auto qk = [&](int i) -> bool {
                const int b = i & 1;
                if (!pf_wait_warp(&sh.k_full[b], i >> 1 & 1, sh, kv.err) ||
                    !pf_wait_warp(&sh.s_empty[b], (i >> 1 & 1) ^ 1, sh, kv.err))
                    return false;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t hi = kdesc + b * (2 * S::K_PART / 16);
                    const uint32_t d = tmem + PF_T_S + b * PF_KT;
#pragma unroll
                    for (int pass = 0; pass < 3; ++pass)
#pragma unroll
                        for (int s = 0; s < HD / 16; ++s)
                            umma_f16_ts(d, tmem + (pass == 0 ? PF_T_QL : PF_T_QH) + 8 * s,
                                        hi + ((pass == 1 ? S::K_PART : 0) + s * 2 * S::K_PIECE) / 16, iqk, pass + s > 0);
                    umma_commit(&sh.s_full[b]);
                    umma_commit(&sh.k_empty[b]);
                }
                __syncwarp();
                return true;
            };
            auto pv = [&](int i) -> bool {
                const int b = i & 1;
                if (!pf_wait_warp(&sh.p_full, i & 1, sh, kv.err) || !pf_wait_warp(&sh.v_full[b], i >> 1 & 1, sh, kv.err) ||
                    !pf_wait_warp(&sh.o_empty, (i & 1) ^ 1, sh, kv.err))
                    return false;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t hi = vdesc + b * (2 * S::V_PART / 16);
#pragma unroll
                    for (int pass = 0; pass < 3; ++pass)
#pragma unroll
                        for (int s = 0; s < PF_KT / 16; ++s)
                            umma_f16_ts(tmem + PF_T_O, tmem + (pass == 0 ? PF_T_PL : PF_T_PH) + 8 * s,
                                        hi + ((pass == 1 ? S::V_PART : 0) + s * 2 * S::V_PIECE) / 16, ipv, pass + s > 0);
                    umma_commit(&sh.o_full);
                    umma_commit(&sh.v_empty[b]);
                    umma_commit(&sh.p_empty);
                }
                __syncwarp();
                return true;
            };
            bool ok = pf_wait_warp(&sh.q_full, 0, sh, kv.err) && qk(0);
            for (int i = 0; i < n && ok; ++i) ok = (i + 1 >= n || qk(i + 1)) && pv(i);
        }
        __syncwarp();
    } else if (warp < PF_W_SUM) {
        // ---------------- softmax: thread = row 32 (warp % 4) + lane ----------------
        const int r = 32 * (warp & 3) + lane;
        const uint32_t tq = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const int pi = pr0 + min(r, npairs - 1), j = pi / G;   // missing pairs repeat the last one
        const int qpos = e.pos0 + j, qlo = p.window > 0 ? qpos - p.window + 1 : 0;
        float sfac;
        {   // q: two fp16 parts times a power of two, amax * f in [2^13, 2^14)
            const float* qr = p.q + (int64_t)(e.row0 + j) * p.ldq + (int64_t)(hk * G + pi - j * G) * HD;
            float amax = 0.0f;
            for (int d = 0; d < HD; d += 4) {
                const float4 x = *reinterpret_cast<const float4*>(qr + d);
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
            }
            const int fe = min(253, max(1, 267 - (int)(__float_as_uint(amax) >> 23)));
            const float f = copysignf(__uint_as_float((uint32_t)fe << 23), p.scale);
            // (never 0: a masked score is -inf times it)
            sfac = fmaxf(fabsf(p.scale) * 1.44269504088896341f * __uint_as_float((uint32_t)(254 - fe) << 23), 1e-36f);
            for (int d = 0; d < HD; d += 16) {   // dims (0, 4 | 1, 5 | 2, 6 | 3, 7) of each 8, as K's are unpacked
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float4 x = *reinterpret_cast<const float4*>(qr + d + 8 * h);
                    const float4 y = *reinterpret_cast<const float4*>(qr + d + 8 * h + 4);
                    split_half2(x.x * f, y.x * f, hi[4 * h], lo[4 * h]);
                    split_half2(x.y * f, y.y * f, hi[4 * h + 1], lo[4 * h + 1]);
                    split_half2(x.z * f, y.z * f, hi[4 * h + 2], lo[4 * h + 2]);
                    split_half2(x.w * f, y.w * f, hi[4 * h + 3], lo[4 * h + 3]);
                }
                tmem_st8(tq + PF_T_QH + d / 2, hi);
                tmem_st8(tq + PF_T_QL + d / 2, lo);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full);
        }
        float m = -INFINITY, l = 0.0f;
        for (int i = 0; i < n; ++i) {
            const int b = i & 1;
            if (!pf_wait_warp(&sh.s_full[b], i >> 1 & 1, sh, kv.err)) break;
            tc_fence_after();
            float v[2][32];
            tmem_ld32(tq + PF_T_S + b * PF_KT, v[0]);
            tmem_ld32(tq + PF_T_S + b * PF_KT + 32, v[1]);
            tmem_ld_wait();
            tc_fence_before();
            const float up = sh.unscale[i & 3], f = sfac * up;
            const int k0 = (ta + i) * PF_KT;
            const bool full = k0 >= all_lo && k0 + PF_KT - 1 <= all_hi;   // no key is masked for any row
            if (!full) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (k0 + 32 * h + c > qpos || k0 + 32 * h + c < qlo) v[h][c] = -INFINITY;
            }
            // a NaN among V's scales: the rows that see its key become NaN, the others do not (the unpacked value is 0)
#pragma unroll
            for (int g = 0; g < PF_GROUPS; ++g) {
                uint32_t bad = sh.poison[i & 3][g];
                for (; bad; bad &= bad - 1) {
                    const int key = k0 + 16 * g + __ffs(bad) - 1;
                    if (key <= qpos && key >= qlo) l = __uint_as_float(0x7fffffffu);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.s_empty[b]);
            float mx[4] = {v[0][0], v[0][1], v[0][2], v[0][3]};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < 32; ++c) mx[c & 3] = fmaxf(mx[c & 3], v[h][c]);
            const float mn = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * f);
            const float corr = mn == m ? 1.0f : ex2(m - mn);   // m = -inf: 0
            m = mn;
            const float mref = m == -INFINITY ? 0.0f : PF_PLOG2 - m;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (!pf_wait_warp(&sh.p_empty, (i & 1) ^ 1, sh, kv.err)) break;   // and corr of two tiles before is read
            tc_fence_after();
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < 32; c += 16) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int x = 0; x < 16; x += 2) {
                        const float p0 = ex2(fmaf(v[h][c + x], f, mref)), p1 = ex2(fmaf(v[h][c + x + 1], f, mref));
                        sum[x & 2] += p0;
                        sum[(x & 2) + 1] += p1;
                        split_half2(p0 * up, p1 * up, hi[x / 2], lo[x / 2]);
                    }
                    tmem_st8(tq + PF_T_PH + 16 * h + c / 2, hi);
                    tmem_st8(tq + PF_T_PL + 16 * h + c / 2, lo);
                }
            l = l * corr + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
            sh.corr[b][r] = corr;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.p_full);
        }
        sh.m[r] = m;
        sh.l[r] = l;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.fin);
    } else if (warp < PF_W_UNPACK) {
        // ---------------- O: thread = row, half of its dims ----------------
        constexpr int NC = HD / 2;
        const int r = 32 * (warp & 3) + lane, c0 = (warp - PF_W_SUM) / 4 * NC;
        const uint32_t to = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + PF_T_O + c0;
        float o[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) o[c] = 0.0f;
        bool ok = true;
        for (int i = 0; i < n && ok; ++i) {
            ok = pf_wait_warp(&sh.o_full, i & 1, sh, kv.err);
            if (!ok) break;
            tc_fence_after();
            const float corr = sh.corr[i & 1][r];
#pragma unroll
            for (int h = 0; h < NC; h += 32) {
                float t[32];
                tmem_ld32(to + h, t);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 32; ++c) o[h + c] = fmaf(o[h + c], corr, t[c]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.o_empty);
        }
        ok = ok && pf_wait_warp(&sh.fin, 0, sh, kv.err);
        if (ok && r < npairs) {
            const int pi = pr0 + r, j = pi / G;
            float* dst = splits == 1 ? p.out + (int64_t)(e.row0 + j) * p.ldo + (int64_t)(hk * G + pi - j * G) * HD + c0
                                     : reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + KV_COUNTER_BYTES) +
                                           ((item * splits + split) * PF_M + r) * (HD + 4) + c0;
            const float f = splits == 1 ? 1.0f / sh.l[r] : 1.0f;
#pragma unroll
            for (int c = 0; c < NC; c += 4)
                __stcg(reinterpret_cast<float4*>(dst + c), make_float4(o[c] * f, o[c + 1] * f, o[c + 2] * f, o[c + 3] * f));
            if (splits > 1 && c0 == 0) __stcg(reinterpret_cast<float2*>(dst + HD), make_float2(sh.m[r], sh.l[r]));
        }
    } else {
        // ---------------- unpacking: warp = group of the tile ----------------
        const int grp = warp - PF_W_UNPACK, g = lane >> 2, q = lane & 3;
        const uint32_t base = p.code_base;
        for (int i = 0; i < n; ++i) {
            const int b = i & 1, st = i % PF_RAW;
            const uint8_t* tile = smem + st * S::RAW_BYTES;
            const uint8_t* raw = tile + grp * kv_group_bytes(R);
            const int k0 = (ta + i) * PF_KT;
            if (!pf_wait_warp(&sh.raw_full[st], i / PF_RAW & 1, sh, kv.err)) break;
            if (!pf_wait_warp(&sh.k_empty[b], (i >> 1 & 1) ^ 1, sh, kv.err)) break;
            // the largest scale of the tile's live groups (as fp16 bits): above 8188 its values are taken times 2^-4,
            // so that d (c - 8) stays in fp16's range; above infinity some are NaN
            uint32_t top = 0;
#pragma unroll
            for (int x = 0; x < PF_GROUPS; ++x)
                if (k0 + 16 * x <= kmax)
#pragma unroll
                    for (int w = lane; w < 16 * R; w += 32)
                        top = __vmaxu2(top, reinterpret_cast<const uint32_t*>(tile + x * kv_group_bytes(R) + 512 * R)[w] & 0x7FFF7FFFu);
            top = __reduce_max_sync(0xffffffffu, max(top & 0xFFFFu, top >> 16));
            const bool big = top > 0x6FFFu;
            uint32_t nan = 0;
            if (top > 0x7C00u && k0 + 16 * grp <= kmax) {
                bool mine = false;   // lane = position
#pragma unroll
                for (int x = 0; x < R; ++x)
                    mine |= (reinterpret_cast<const uint16_t*>(raw + 544 * R)[kv_vscale(R, lane & 15, x)] & 0x7FFFu) > 0x7C00u;
                nan = __ballot_sync(0xffffffffu, mine) & 0xFFFFu;
            }
            if (lane == 0) {
                sh.poison[i & 3][grp] = nan;
                if (grp == 0) sh.unscale[i & 3] = big ? 16.0f : 1.0f;
            }
            uint8_t* kd = smem + S::K + b * 2 * S::K_PART;
#pragma unroll
            for (int u = 0; u < 2; ++u) {   // key 8 u + g, dims 32 x + 8 q .. + 7
                uint32_t w[R];
                __half d[R];
                load_words<R>(w, raw, u, lane);
                load_kscales<R>(d, raw + 512 * R, 8 * u + g);
#pragma unroll
                for (int x = 0; x < R; ++x) {
                    __half2 dd = __half2half2(d[x]);
                    uint32_t d2 = *reinterpret_cast<uint32_t*>(&dd), c[4];
                    if (big) d2 = mul_h2(d2, 0x2C002C00u);
                    unpack(c, w[x], base);
                    uint4 hi, lo;
                    hi.x = mul_h2(c[0], d2); lo.x = fma_h2(c[0], d2, neg_h2(hi.x));
                    hi.y = mul_h2(c[1], d2); lo.y = fma_h2(c[1], d2, neg_h2(hi.y));
                    hi.z = mul_h2(c[2], d2); lo.z = fma_h2(c[2], d2, neg_h2(hi.z));
                    hi.w = mul_h2(c[3], d2); lo.w = fma_h2(c[3], d2, neg_h2(hi.w));
                    uint8_t* at = kd + (4 * x + q) * S::K_PIECE + (16 * grp + 8 * u + g) * 16;
                    *reinterpret_cast<uint4*>(at) = hi;
                    *reinterpret_cast<uint4*>(at + S::K_PART) = lo;
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.k_full[b]);
            if (!pf_wait_warp(&sh.v_empty[b], (i >> 1 & 1) ^ 1, sh, kv.err)) break;
            uint8_t* vd = smem + S::V + b * 2 * S::V_PART;
#pragma unroll
            for (int u = 0; u < 2; ++u) {   // keys 8 u + 2 q, + 1, dims 32 x + 4 g .. + 3
                uint32_t w[R], d[R];
                load_words<R>(w, raw + 256 * R, u, lane);
                load_scales<R>(d, raw + 544 * R, u, q);
                // keys that no row sees may hold anything: 0
                const int key = 8 * u + 2 * q, pos = k0 + 16 * grp + key;
                uint32_t live = (pos > kmax || pos < kmin || (nan >> key & 1) ? 0u : 0xFFFFu) |
                                (pos + 1 > kmax || pos + 1 < kmin || (nan >> key & 2) ? 0u : 0xFFFF0000u);
#pragma unroll
                for (int x = 0; x < R; ++x) {
                    uint32_t d2 = d[x] & live, c[4];
                    if (big) d2 = mul_h2(d2, 0x2C002C00u);
                    unpack(c, w[x], base);
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const uint32_t hi = mul_h2(c[y], d2), lo = fma_h2(c[y], d2, neg_h2(hi));
                        uint8_t* at = vd + (2 * grp + u) * S::V_PIECE + (4 * x + (g >> 1)) * S::V_GROUP + (4 * (g & 1) + y) * 16 + 4 * q;
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
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (splits == 1 || sh.abort) return;

    // ---- a split item: the last CTA to arrive joins its parts
    int* counters = reinterpret_cast<int*>(p.workspace);
    if (tid == 0) {
        __threadfence();
        sh.last = atomicAdd(&counters[item], 1) == splits - 1;
        __threadfence();
    }
    __syncthreads();
    if (!sh.last) return;
    const float* parts = reinterpret_cast<const float*>(static_cast<const uint8_t*>(p.workspace) + KV_COUNTER_BYTES) +
                         item * splits * PF_M * (HD + 4);
    for (int x = tid; x < npairs * (HD / 4); x += PF_THREADS) {
        const int r = x / (HD / 4), d = x % (HD / 4) * 4;
        auto part = [&](int s) { return parts + ((int64_t)s * PF_M + r) * (HD + 4); };
        float M = -INFINITY, L = 0.0f;
        for (int s = 0; s < splits; ++s) M = fmaxf(M, __ldcg(part(s) + HD));
        float4 a = make_float4(0, 0, 0, 0);
        for (int s = 0; s < splits; ++s) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(part(s) + HD));
            const float4 v = __ldcg(reinterpret_cast<const float4*>(part(s) + d));
            const float w = ml.x == -INFINITY ? 0.0f : ex2(ml.x - M);
            L += w * ml.y;
            a.x += w * v.x; a.y += w * v.y; a.z += w * v.z; a.w += w * v.w;
        }
        const int pi = pr0 + r, j = pi / G;
        const float inv = 1.0f / L;
        *reinterpret_cast<float4*>(p.out + (int64_t)(e.row0 + j) * p.ldo + (int64_t)(hk * G + pi - j * G) * HD + d) =
            make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
    }
    if (tid == 0) counters[item] = 0;
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
    }
    const int G = p.kv.n_heads / p.kv.n_kv;
    // at most this many items; fewer than the SMs: each item's keys are split
    const int64_t items = ((int64_t)p.rows.n_rows * G / PF_M + p.rows.n_seqs) * p.kv.n_kv;
    const int splits = items < PF_MAX_PARTS ? (int)(PF_MAX_PARTS / items) : 1;
    BREW_CHECK(items * splits <= 0x7fffffff, BREW_ERR_INVALID_ARG, "attention of %d rows", p.rows.n_rows);
    KvAttendParams q = p;
    q.code_base = 0x64006400u;
    kv_prefill_kernel<R><<<(unsigned)(items * splits), PF_THREADS, smem, s>>>(q, splits);
    BREW_CUDA(cudaGetLastError());
    count_launch();
    return BREW_OK;
}

}  // namespace

bool kv_prefill_supported(int hd) { return hd == 64 || hd == 128; }

int64_t kv_prefill_workspace(int hd) {
    return kv_prefill_supported(hd) ? KV_COUNTER_BYTES + (int64_t)PF_MAX_PARTS * PF_M * (hd + 4) * 4 : 0;
}

int kv_prefill_launch(int hd, const KvAttendParams& p, cudaStream_t s) {
    return hd == 64 ? prefill_r<2>(p, s) : prefill_r<4>(p, s);
}

}  // namespace brew
