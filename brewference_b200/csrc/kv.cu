// kv.cu — the paged 4-bit K/V cache: its handle (pages, reservations), the
// append and read kernels and the C ABI of both and of the attention.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "brew_internal.cuh"
#include "kv_device.cuh"

struct brew_kv_s {
    brew_kv_config c = {};
    int max_pages = 0;              // pages of one sequence
    int page_shift = 0;
    int64_t layer_bytes = 0;
    uint8_t* pool = nullptr;
    int32_t* table = nullptr;       // [max_seqs][max_pages]
    int32_t* reserved = nullptr;    // [max_seqs]
    unsigned int* err = nullptr;
    int device = 0;
    std::mutex mu;
    std::vector<int32_t> free_pages;             // the last one is handed out next
    std::vector<std::vector<int32_t>> seq_pages;
};

namespace brew {
namespace {

// Page ids of a sequence, and then its reserved positions: launch parameters,
// so that the call stays asynchronous and needs no staging buffer.
struct KvIds {
    int32_t id[KV_PUT_PAGES];
};

__global__ void kv_table_kernel(int32_t* row, int first, int n, KvIds ids, int32_t* reserved, int tokens) {
    if ((int)threadIdx.x < n) row[first + threadIdx.x] = ids.id[threadIdx.x];
    if (threadIdx.x == 0 && tokens >= 0) *reserved = tokens;
}

int set_pages(brew_kv_s* kv, int seq, int first, int end, int tokens, cudaStream_t s) {
    const std::vector<int32_t>& pages = kv->seq_pages[seq];
    int32_t* row = kv->table + (int64_t)seq * kv->max_pages;
    do {
        const KvPut p = kv_put(first, end, tokens);
        KvIds ids;
        for (int i = 0; i < p.n; ++i) ids.id[i] = pages[first + i];
        kv_table_kernel<<<1, 128, 0, s>>>(row, first, p.n, ids, kv->reserved + seq, p.tokens);
        BREW_CUDA(cudaGetLastError());
        count_launch();
        first += p.n;
    } while (first < end);
    return BREW_OK;
}

// Pages change hands once, on the host: a replayed graph would do it again.
int not_captured(cudaStream_t s) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    BREW_CUDA(cudaStreamIsCapturing(s, &st));
    BREW_CHECK(st == cudaStreamCaptureStatusNone, BREW_ERR_INVALID_ARG,
               "pages cannot be reserved or released while the stream is captured");
    return BREW_OK;
}

// ---- append -------------------------------------------------------------
// The 4-bit code of a value next to a rounding border depends on its last
// bit (and a position of 10^5 leaves 32 bits no digit of the angle), so
// angles, norm and rotation run in 64 bits and are rounded once.
//
// A CTA takes up to AP_ROWS rows of an entry; their sines and the norm's
// weights are made once and shared by all heads.  A lane holds 16 dims of a
// vector (a head of q, k or v) in two pieces of 8, the second half a head
// after the first where blocks of 32 allow it (heads of 64, 128, 256): then
// the pairs of either rotation are the lane's own, a piece is a word of K's
// codes, and no value is converted twice.  (4 dims a lane, partners loaded
// and converted again: 102 us for 5194 rows of 16 + 16 heads of 128; the same
// in pairs of fp32 numbers instead of 64 bits: 69 us.)  Now 47 us with norms,
// 170 MB at 3.6 TB/s; half the issue slots are taken, the 64-bit steps and the
// sines' chains in between bound it.
constexpr int AP_THREADS = 256;
constexpr int AP_ROWS = 4;

template <int R, bool NORM, int ROPE>
__global__ void __launch_bounds__(AP_THREADS) kv_append_kernel(const __grid_constant__ KvAppendParams p) {
    constexpr int HD = 32 * R, HALF = HD / 2;
    constexpr bool OWN = R % 2 == 0;          // pieces half a head apart (else side by side)
    constexpr int LPV = R == 3 ? 8 : 2 * R;   // lanes a vector (R = 3: 6 of them hold values)
    constexpr int VPW = 32 / LPV;             // vectors of a warp
    constexpr int SL = HALF / 8;              // sines lie [i % 8][i / 8]: a step's are side by side over the lanes
    __shared__ double2 cs[AP_ROWS][HALF];     // cosine, sine
    __shared__ double wq[NORM ? HD : 1], wk[NORM ? HD : 1];   // [d % 8][d / 8]
    const KvEntry e = kv_entry(p.kv, p.rows, blockIdx.y, threadIdx.x == 0 && blockIdx.x == 0);
    const int j0 = blockIdx.x * AP_ROWS, nr = min(AP_ROWS, e.rows - j0);
    if (nr <= 0) return;
    auto wat = [](int d) { return d % 8 * (HD / 8) + d / 8; };
    auto sat = [](int i) { return i % 8 * SL + i / 8; };
    if (ROPE != BREW_KV_ROPE_NONE) {
        for (int x = threadIdx.x; x < nr * HALF; x += AP_THREADS) {
            const int r = x / HALF, i = x % HALF;
            double c, s;
            sincos((double)(e.pos0 + j0 + r) * p.rope_scale * exp2(-2.0 * i * p.log2_base_hd), &s, &c);
            cs[r][sat(i)] = make_double2(c, s);
        }
    }
    if (NORM) {
        for (int d = threadIdx.x; d < HD; d += AP_THREADS) {
            wq[wat(d)] = p.qnorm ? (double)p.qnorm[d] : 1.0;
            wk[wat(d)] = p.knorm ? (double)p.knorm[d] : 1.0;
        }
    }
    if (NORM || ROPE != BREW_KV_ROPE_NONE) __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int l = lane % LPV;
    const int dim[2] = {OWN ? 8 * l : 16 * l, OWN ? 8 * l + HALF : 16 * l + 8};   // the pieces
    const bool act = R != 3 || l < 6;
    const int hq = p.q ? p.kv.n_heads : 0, hk = p.kv.n_kv;
    const int nvec = hq + 2 * hk;
    for (int r = 0; r < nr; ++r) {
        const int pos = e.pos0 + j0 + r;
        const int64_t row = (int64_t)e.row0 + j0 + r;
        const int64_t grp0 = kv_group_at<R>(p.kv, e.seq, pos, 0);   // kv head 0's; the next ones' follow a page's groups apart
        const int pg = pos & 15, u = pg >> 3;
        for (int v0 = warp * VPW; v0 < nvec; v0 += AP_THREADS / 32 * VPW) {   // uniform over the warp
            const int v = v0 + lane / LPV;
            const bool on = act && v < nvec;
            const bool isq = v < hq, isk = !isq && v < hq + hk;
            const bool qk = on && (isq || isk);
            const int head = isq ? v : isk ? v - hq : v - hq - hk;
            const float* src = (isq ? p.q + row * p.ldq : (isk ? p.k : p.v) + row * p.ldkv) + (int64_t)head * HD;
            float x[2][8], y[2][8];   // the pieces, and (!OWN) their dims' partners half a head away
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < 8; c += 4) {
                    const float4 t = on ? *reinterpret_cast<const float4*>(src + dim[h] + c) : make_float4(0, 0, 0, 0);
                    x[h][c] = t.x; x[h][c + 1] = t.y; x[h][c + 2] = t.z; x[h][c + 3] = t.w;
                    if (!OWN && ROPE == BREW_KV_ROPE_HALF) {
                        const int m = dim[h] < HALF ? dim[h] + HALF : dim[h] - HALF;
                        const float4 o = qk ? *reinterpret_cast<const float4*>(src + m + c) : make_float4(0, 0, 0, 0);
                        y[h][c] = o.x; y[h][c + 1] = o.y; y[h][c + 2] = o.z; y[h][c + 3] = o.w;
                    }
                }
            double inv = 1.0;
            if (NORM && v0 < hq + hk) {   // uniform over the warp: the shuffles are every lane's
                double ss = 0.0;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int c = 0; c < 8; ++c) ss = fma((double)x[h][c], (double)x[h][c], ss);
#pragma unroll
                for (int o = LPV / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const bool has = isq ? p.qnorm != nullptr : p.knorm != nullptr;
                inv = has ? rsqrt(ss * (1.0 / HD) + p.eps) : 1.0;
            }
            __syncwarp();   // q_out may be q: every lane has read before one writes
            if ((NORM || ROPE != BREW_KV_ROPE_NONE) && qk) {
                const double* w = isq ? wq : wk;
                // a dim with its norm
                auto in = [&](float t, int d) { return NORM ? (double)t * inv * w[wat(d)] : (double)t; };
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    if (ROPE == BREW_KV_ROPE_HALF && OWN) {   // the pieces are each other's partners
                        const double2 t = cs[r][c * SL + l];
                        const double a = in(x[0][c], dim[0] + c), b = in(x[1][c], dim[1] + c);
                        x[0][c] = (float)(a * t.x - b * t.y);
                        x[1][c] = (float)(a * t.y + b * t.x);
                    } else if (ROPE == BREW_KV_ROPE_HALF) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int d = dim[h] + c;
                            const bool low = d < HALF;
                            const double2 t = cs[r][sat(low ? d : d - HALF)];
                            const double a = in(x[h][c], d), b = in(y[h][c], low ? d + HALF : d - HALF);
                            x[h][c] = (float)(low ? a * t.x - b * t.y : b * t.y + a * t.x);
                        }
                    } else if (ROPE == BREW_KV_ROPE_INTERLEAVED) {
                        if (c % 2) continue;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const double2 t = cs[r][sat((dim[h] + c) / 2)];
                            const double a = in(x[h][c], dim[h] + c), b = in(x[h][c + 1], dim[h] + c + 1);
                            x[h][c] = (float)(a * t.x - b * t.y);
                            x[h][c + 1] = (float)(a * t.y + b * t.x);
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) x[h][c] = (float)in(x[h][c], dim[h] + c);
                    }
                }
            }
            if (on && isq) {
                float* dst = p.q_out + row * p.ldq + (int64_t)head * HD;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int c = 0; c < 8; c += 4)
                        *reinterpret_cast<float4*>(dst + dim[h] + c) =
                            make_float4(x[h][c], x[h][c + 1], x[h][c + 2], x[h][c + 3]);
            }
            if (v0 + VPW <= hq) continue;   // a warp of q alone
            // a block's scale: -1/8 of its first value of largest magnitude, of a piece, then of the block's lanes
            float top[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                top[h] = x[h][0];
#pragma unroll
                for (int c = 1; c < 8; ++c) top[h] = fabsf(x[h][c]) > fabsf(top[h]) || x[h][c] != x[h][c] ? x[h][c] : top[h];
            }
            if (!OWN && (fabsf(top[1]) > fabsf(top[0]) || top[1] != top[1])) top[0] = top[1];   // one block
#pragma unroll
            for (int h = 0; h < (OWN ? 2 : 1); ++h)
#pragma unroll
                for (int o = 1; o < (OWN ? 4 : 2); o <<= 1) {
                    const float other = __shfl_xor_sync(0xffffffffu, top[h], o);
                    const bool take = lane & o ? !(fabsf(top[h]) > fabsf(other)) : fabsf(other) > fabsf(top[h]);
                    if ((take && top[h] == top[h]) || other != other) top[h] = other;
                }
            if (!OWN) top[1] = top[0];
            if (!on || isq) continue;
            uint8_t* grp = p.kv.pages + grp0 + ((int64_t)head << (p.kv.page_shift - 4)) * kv_group_bytes(R);
            uint16_t* sc = reinterpret_cast<uint16_t*>(grp + 512 * R);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float d = top[h] * -0.125f;
                // fp16 ends at 65504: larger blocks saturate (a NaN stays one)
                if (fabsf(d) > 65504.0f) d = copysignf(65504.0f, d);
                const float id = d == 0.0f ? 0.0f : __frcp_rn(d);
                uint32_t q = 0;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    // 0 .. 15: the integer part, as the last bits of 2^23 + it
                    const float t = fminf(fmaxf(__fadd_rn(__fmul_rn(x[h][c], id), 8.5f), 0.0f), 15.5f);
                    q |= (__float_as_uint(__fadd_rd(t, 8388608.0f)) & 15u) << (4 * c);
                }
                const int b = dim[h] / 32, i = dim[h] % 32 / 8;
                const uint16_t dh = __half_as_ushort(__float2half_rn(d));
                if (isk) {
                    reinterpret_cast<uint32_t*>(grp)[kv_word(R, u, b, (pg & 7) * 4 + i)] = q;
                    if (i == 0) sc[kv_kscale(R, pg, b)] = dh;
                } else {
                    uint16_t* vq = reinterpret_cast<uint16_t*>(grp + 256 * R);
                    vq[2 * kv_word(R, u, b, 8 * i + ((pg & 7) >> 1)) + (pg & 1)] = (uint16_t)q;
                    vq[2 * kv_word(R, u, b, 8 * i + 4 + ((pg & 7) >> 1)) + (pg & 1)] = (uint16_t)(q >> 16);
                    if (i == 0) sc[16 * R + kv_vscale(R, pg, b)] = dh;
                }
            }
        }
    }
}

template <int R>
int append_r(const KvAppendParams& p, cudaStream_t s) {
    // (a call of no rows too checks its entries)
    const dim3 grid((unsigned)((std::max<int64_t>(p.rows.max_rows, 1) + AP_ROWS - 1) / AP_ROWS), p.rows.n_seqs);
    auto go = [&](auto kernel) { kernel<<<grid, AP_THREADS, 0, s>>>(p); };
    if (p.qnorm || p.knorm) {
        if (p.rope == BREW_KV_ROPE_HALF) go(kv_append_kernel<R, true, BREW_KV_ROPE_HALF>);
        else if (p.rope == BREW_KV_ROPE_INTERLEAVED) go(kv_append_kernel<R, true, BREW_KV_ROPE_INTERLEAVED>);
        else go(kv_append_kernel<R, true, BREW_KV_ROPE_NONE>);
    } else {
        if (p.rope == BREW_KV_ROPE_HALF) go(kv_append_kernel<R, false, BREW_KV_ROPE_HALF>);
        else if (p.rope == BREW_KV_ROPE_INTERLEAVED) go(kv_append_kernel<R, false, BREW_KV_ROPE_INTERLEAVED>);
        else go(kv_append_kernel<R, false, BREW_KV_ROPE_NONE>);
    }
    BREW_CUDA(cudaGetLastError());
    count_launch();
    return BREW_OK;
}

// ---- read: the values that stored rows stand for --------------------------
// 2^23 + code as the bits of a float, less 2^23 + 8, times d.
__device__ __forceinline__ float4 kv_values4(uint32_t w, float d) {
    float v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = (__uint_as_float((w >> 4 * c & 15u) | 0x4B000000u) - 8388616.0f) * d;
    return make_float4(v[0], v[1], v[2], v[3]);
}

// A warp is 8 positions of a kv head, half a group, whose words it reads as
// they lie: K's words are 8 dims of a position, V's 4 dims of two.  Bound by
// the latency of entry, page and words one after the other: 16 us for 5194 rows
// of 8 heads of 128 (42.6 MB written; 20 with 8 dims of a row a thread, which
// gathers V's and the scales in 16-bit pieces).
template <int R>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvView kv,
                                                      const __grid_constant__ KvRowsDev rows, float* k_out,
                                                      float* v_out, int64_t ld) {
    const KvEntry e = kv_entry(kv, rows, blockIdx.y, threadIdx.x == 0 && blockIdx.x == 0);
    if (e.rows <= 0) return;
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int first = e.pos0 >> 3, n = (((e.pos0 + e.rows - 1) >> 3) - first + 1) * kv.n_kv;
    for (int x = blockIdx.x * 8 + (threadIdx.x >> 5); x < n; x += gridDim.x * 8) {
        const int hk = x % kv.n_kv, base = (first + x / kv.n_kv) * 8, u = base >> 3 & 1;
        const uint8_t* grp = kv_group<R>(kv, e.seq, base, hk);
        const int64_t o = (int64_t)hk * 32 * R;
        auto row = [&](int pos) { return (int64_t)(e.row0 + pos - e.pos0) * ld + o; };
        auto in = [&](int pos) { return pos >= e.pos0 && pos < e.pos0 + e.rows; };
        uint32_t wk[R], wv[R], dv[R];
        __half dk[R];
        if (k_out) load_words<R>(wk, grp, u, lane);
        if (v_out) load_words<R>(wv, grp + 256 * R, u, lane);
        if (k_out) load_kscales<R>(dk, grp + 512 * R, 8 * u + g);
        if (v_out) load_scales<R>(dv, grp + 544 * R, u, q);
        if (k_out && in(base + g)) {
            float* at = k_out + row(base + g) + 8 * q;
#pragma unroll
            for (int b = 0; b < R; ++b) {
                const float d = __half2float(dk[b]);
                *reinterpret_cast<float4*>(at + 32 * b) = kv_values4(wk[b], d);
                *reinterpret_cast<float4*>(at + 32 * b + 4) = kv_values4(wk[b] >> 16, d);
            }
        }
        if (v_out) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int pos = base + 2 * q + h;
                if (!in(pos)) continue;
                float* at = v_out + row(pos) + 4 * g;
#pragma unroll
                for (int b = 0; b < R; ++b)
                    *reinterpret_cast<float4*>(at + 32 * b) =
                        kv_values4(wv[b] >> 16 * h, half_bits_to_float((uint16_t)(dv[b] >> 16 * h)));
            }
        }
    }
}

template <int R>
int read_r(const KvView& kv, const KvRowsDev& rows, float* k, float* v, int64_t ld, cudaStream_t s) {
    // positions of an entry begin anywhere in 8
    const int64_t warps = ((int64_t)rows.max_rows + 14) / 8 * kv.n_kv;
    const dim3 grid((unsigned)std::min<int64_t>((warps + 7) / 8, 1 << 16), rows.n_seqs);
    kv_read_kernel<R><<<grid, 256, 0, s>>>(kv, rows, k, v, ld);
    BREW_CUDA(cudaGetLastError());
    count_launch();
    return BREW_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_rows(const brew_kv_s* kv, int layer, const brew_kv_rows* r) {
    BREW_CHECK(kv, BREW_ERR_INVALID_ARG, "null K/V cache");
    BREW_CHECK(r, BREW_ERR_INVALID_ARG, "rows is null");
    BREW_CHECK(layer >= 0 && layer < kv->c.n_layers, BREW_ERR_INVALID_ARG, "layer %d of %d", layer, kv->c.n_layers);
    BREW_CHECK(r->n_seqs >= 0 && r->n_seqs <= KV_MAX_SEQS, BREW_ERR_INVALID_ARG, "n_seqs %d (at most %d)", r->n_seqs,
               KV_MAX_SEQS);
    BREW_CHECK(r->n_rows >= 0 && r->max_rows >= 0, BREW_ERR_INVALID_ARG, "n_rows %d, max_rows %d", r->n_rows,
               r->max_rows);
    if (r->n_seqs == 0) return BREW_OK;
    BREW_CHECK(r->seq && r->pos, BREW_ERR_INVALID_ARG, "rows: seq and pos must be given");
    BREW_CHECK(r->row_start || (r->n_rows == r->n_seqs && r->max_rows <= 1), BREW_ERR_INVALID_ARG,
               "rows without row_start: one row for each sequence (n_rows %d, n_seqs %d, max_rows %d)", r->n_rows,
               r->n_seqs, r->max_rows);
    BREW_CHECK(((uintptr_t)r->seq & 3) == 0 && ((uintptr_t)r->pos & 3) == 0 && ((uintptr_t)r->row_start & 3) == 0,
               BREW_ERR_INVALID_ARG, "rows: unaligned int32 arrays");
    return BREW_OK;
}

int check_matrix(const char* what, const void* p, int64_t ld, int64_t width) {
    BREW_CHECK(p, BREW_ERR_INVALID_ARG, "%s is null", what);
    BREW_CHECK(aligned16(p) && ld % 4 == 0, BREW_ERR_INVALID_ARG, "%s: rows must start on 16-byte boundaries", what);
    BREW_CHECK(ld >= width, BREW_ERR_INVALID_ARG, "%s: row stride %lld under its width %lld", what, (long long)ld,
               (long long)width);
    return BREW_OK;
}

// (an entry has no more rows than the buffers: grids do not grow with a bound far above them)
KvRowsDev rows_dev(const brew_kv_rows* r) {
    return {r->seq, r->pos, r->row_start, r->n_seqs, r->n_rows, std::min(r->max_rows, r->n_rows)};
}

}  // namespace

KvView kv_view(const brew_kv_s* kv, int layer) {
    KvView v;
    v.pages = kv->pool + layer * kv->layer_bytes;
    v.table = kv->table;
    v.reserved = kv->reserved;
    v.max_seqs = kv->c.max_seqs;
    v.max_pages = kv->max_pages;
    v.page_shift = kv->page_shift;
    v.n_heads = kv->c.n_heads;
    v.n_kv = kv->c.n_kv_heads;
    v.err = kv->err;
    return v;
}

int kv_clear(brew_kv_s* kv, cudaStream_t s) {
    BREW_CUDA(cudaMemsetAsync(kv->pool, 0, (size_t)kv->layer_bytes * kv->c.n_layers, s));
    BREW_CUDA(cudaStreamSynchronize(s));
    return BREW_OK;
}

bool kv_head_supported(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 256; }

int kv_append_launch(int hd, const KvAppendParams& p, cudaStream_t s) {
    switch (hd / 32) {
        case 1: return append_r<1>(p, s);
        case 2: return append_r<2>(p, s);
        case 3: return append_r<3>(p, s);
        case 4: return append_r<4>(p, s);
        default: return append_r<8>(p, s);
    }
}

}  // namespace brew

using namespace brew;

extern "C" {

int brew_kv_create(const brew_kv_config* cfg, brew_kv* out) {
    BREW_CHECK(cfg && out, BREW_ERR_INVALID_ARG, "null argument");
    *out = nullptr;
    const brew_kv_config& c = *cfg;
    BREW_CHECK(kv_head_supported(c.head_size), BREW_ERR_UNSUPPORTED, "K/V cache: head size %d (32, 64, 96, 128 or 256)",
               c.head_size);
    BREW_CHECK(c.n_layers > 0 && c.n_kv_heads > 0 && c.n_heads > 0 && c.n_heads % c.n_kv_heads == 0,
               BREW_ERR_INVALID_ARG, "K/V cache: %d layers, %d heads, %d kv heads", c.n_layers, c.n_heads, c.n_kv_heads);
    BREW_CHECK(c.n_heads <= 1024, BREW_ERR_UNSUPPORTED, "K/V cache: %d heads", c.n_heads);
    BREW_CHECK(c.max_seqs > 0 && c.max_seqs <= KV_MAX_SEQS, BREW_ERR_INVALID_ARG, "K/V cache: %d sequences (1 .. %d)",
               c.max_seqs, KV_MAX_SEQS);
    BREW_CHECK(c.max_tokens > 0 && c.max_tokens <= (1 << 30), BREW_ERR_INVALID_ARG, "K/V cache: %d positions a sequence",
               c.max_tokens);
    BREW_CHECK(c.page_tokens == 16 || c.page_tokens == 32 || c.page_tokens == 64 || c.page_tokens == 128,
               BREW_ERR_INVALID_ARG, "K/V cache: pages of %d positions (16, 32, 64 or 128)", c.page_tokens);
    const int64_t max_pages = ((int64_t)c.max_tokens + c.page_tokens - 1) / c.page_tokens;
    const int64_t pages = c.n_pages > 0 ? c.n_pages : max_pages * c.max_seqs;
    BREW_CHECK(c.n_pages >= 0 && pages <= (1 << 30), BREW_ERR_INVALID_ARG, "K/V cache: %lld pages", (long long)pages);
    const int64_t page_bytes = (int64_t)c.n_kv_heads * (c.page_tokens / KV_GROUP) * kv_group_bytes(c.head_size / 32);
    BREW_CHECK(pages <= (int64_t)1 << 40 >> 6 && page_bytes * pages <= ((int64_t)1 << 50) / c.n_layers,
               BREW_ERR_INVALID_ARG, "K/V cache: %lld pages of %lld bytes in %d layers", (long long)pages,
               (long long)page_bytes, c.n_layers);
    DeviceScope ds;
    if (ds.rc) return ds.rc;
    brew_kv_s* kv = nullptr;
    try {
        kv = new brew_kv_s();
        kv->c = c;
        kv->c.n_pages = (int32_t)pages;
        kv->max_pages = (int)max_pages;
        while ((1 << kv->page_shift) < c.page_tokens) ++kv->page_shift;
        kv->layer_bytes = page_bytes * pages;
        kv->device = ctx().device;
        kv->seq_pages.resize(c.max_seqs);
        kv->free_pages.resize((size_t)pages);
        for (int64_t i = 0; i < pages; ++i) kv->free_pages[i] = (int32_t)(pages - 1 - i);
    } catch (const std::bad_alloc&) {
        delete kv;
        return set_error(BREW_ERR_CUDA, "K/V cache: out of host memory");
    }
    const size_t tb = sizeof(int32_t) * (size_t)c.max_seqs * max_pages;
    cudaError_t e = cudaMalloc(&kv->pool, (size_t)kv->layer_bytes * c.n_layers);
    if (e == cudaSuccess) e = cudaMalloc(&kv->table, tb);
    if (e == cudaSuccess) e = cudaMalloc(&kv->reserved, sizeof(int32_t) * (c.max_seqs + 1));
    if (e == cudaSuccess) {
        kv->err = reinterpret_cast<unsigned int*>(kv->reserved + c.max_seqs);
        e = cudaMemset(kv->table, 0, tb);
    }
    if (e == cudaSuccess) e = cudaMemset(kv->reserved, 0, sizeof(int32_t) * (c.max_seqs + 1));
    // positions that are reserved and never appended read as zeros
    if (e == cudaSuccess) e = cudaMemset(kv->pool, 0, (size_t)kv->layer_bytes * c.n_layers);
    if (e == cudaSuccess) e = cudaStreamSynchronize(0);
    if (e != cudaSuccess) {
        cudaGetLastError();
        brew_kv_free(kv);
        return cuda_error(e, "K/V cache allocation");
    }
    *out = kv;
    return BREW_OK;
}

int brew_kv_free(brew_kv kv) {
    if (!kv) return BREW_OK;
    {
        DeviceScope ds;
        cudaDeviceSynchronize();
        cudaFree(kv->pool);
        cudaFree(kv->table);
        cudaFree(kv->reserved);
    }
    delete kv;
    return BREW_OK;
}

int brew_kv_info(brew_kv kv, int64_t* bytes, int32_t* free_pages) {
    BREW_CHECK(kv, BREW_ERR_INVALID_ARG, "null K/V cache");
    std::lock_guard<std::mutex> lk(kv->mu);
    if (bytes) *bytes = kv->layer_bytes * kv->c.n_layers;
    if (free_pages) *free_pages = (int32_t)kv->free_pages.size();
    return BREW_OK;
}

int brew_kv_reserve(brew_kv kv, int32_t seq, int32_t n_tokens, void* stream) {
    BREW_CHECK(kv, BREW_ERR_INVALID_ARG, "null K/V cache");
    BREW_CHECK(seq >= 0 && seq < kv->c.max_seqs, BREW_ERR_INVALID_ARG, "sequence %d of %d", seq, kv->c.max_seqs);
    BREW_CHECK(n_tokens >= 0, BREW_ERR_INVALID_ARG, "%d positions", n_tokens);
    BREW_CHECK(n_tokens <= kv->c.max_tokens, BREW_ERR_CONTEXT_FULL, "The session has reached its context limit of %d tokens.",
               kv->c.max_tokens);
    DeviceScope ds;
    if (ds.rc) return ds.rc;
    std::lock_guard<std::mutex> lk(kv->mu);
    std::vector<int32_t>& have = kv->seq_pages[seq];
    const size_t need = ((size_t)n_tokens + kv->c.page_tokens - 1) >> kv->page_shift, first = have.size();
    if (need <= first) return BREW_OK;
    int rc = not_captured(static_cast<cudaStream_t>(stream));
    if (rc) return rc;
    BREW_CHECK(need - first <= kv->free_pages.size(), BREW_ERR_CONTEXT_FULL,
               "K/V cache: %zu pages needed, %zu free", need - first, kv->free_pages.size());
    try {
        have.reserve(need);
    } catch (const std::bad_alloc&) {
        return set_error(BREW_ERR_CUDA, "K/V cache: out of host memory");
    }
    for (size_t i = first; i < need; ++i) {
        have.push_back(kv->free_pages.back());
        kv->free_pages.pop_back();
    }
    // the last page may reach past max_tokens: the sequence does not
    const int tokens = (int)std::min<size_t>(need << kv->page_shift, kv->c.max_tokens);
    rc = set_pages(kv, seq, (int)first, (int)need, tokens, static_cast<cudaStream_t>(stream));
    for (; rc && have.size() > first; have.pop_back()) kv->free_pages.push_back(have.back());
    return rc;
}

int brew_kv_release(brew_kv kv, int32_t seq, void* stream) {
    BREW_CHECK(kv, BREW_ERR_INVALID_ARG, "null K/V cache");
    BREW_CHECK(seq >= 0 && seq < kv->c.max_seqs, BREW_ERR_INVALID_ARG, "sequence %d of %d", seq, kv->c.max_seqs);
    DeviceScope ds;
    if (ds.rc) return ds.rc;
    std::lock_guard<std::mutex> lk(kv->mu);
    std::vector<int32_t>& have = kv->seq_pages[seq];
    int rc = not_captured(static_cast<cudaStream_t>(stream));
    if (rc || (rc = set_pages(kv, seq, 0, 0, 0, static_cast<cudaStream_t>(stream)))) return rc;
    // free_pages was sized for every page: no allocation here
    for (size_t i = have.size(); i-- > 0;) kv->free_pages.push_back(have[i]);
    have.clear();
    return BREW_OK;
}

int brew_kv_append_dev(brew_kv kv, int32_t layer, float* q_out, const float* q, int64_t ldq, const float* k,
                       const float* v, int64_t ldkv, const brew_kv_rows* rows, const brew_kv_rope* rope, void* stream) {
    int rc = check_rows(kv, layer, rows);
    if (rc) return rc;
    const brew_kv_config& c = kv->c;
    if ((rc = check_matrix("k", k, ldkv, (int64_t)c.n_kv_heads * c.head_size)) ||
        (rc = check_matrix("v", v, ldkv, (int64_t)c.n_kv_heads * c.head_size)))
        return rc;
    BREW_CHECK((q != nullptr) == (q_out != nullptr), BREW_ERR_INVALID_ARG, "q and q_out are given together");
    if (q && ((rc = check_matrix("q", q, ldq, (int64_t)c.n_heads * c.head_size)) ||
              (rc = check_matrix("q_out", q_out, ldq, (int64_t)c.n_heads * c.head_size))))
        return rc;
    KvAppendParams p = {};
    p.rope = BREW_KV_ROPE_NONE;
    if (rope) {
        BREW_CHECK(rope->mode == BREW_KV_ROPE_NONE || rope->mode == BREW_KV_ROPE_HALF ||
                       rope->mode == BREW_KV_ROPE_INTERLEAVED,
                   BREW_ERR_INVALID_ARG, "rope mode %d", rope->mode);
        BREW_CHECK(rope->mode == BREW_KV_ROPE_NONE ||
                       (rope->base > 0.0 && std::isfinite(rope->base) && std::isfinite(rope->scale)),
                   BREW_ERR_INVALID_ARG, "rope base %g, scale %g", rope->base, rope->scale);
        const bool norm = rope->qnorm || rope->knorm;
        BREW_CHECK(!norm || (rope->eps >= 0.0 && std::isfinite(rope->eps)), BREW_ERR_INVALID_ARG, "norm eps %g", rope->eps);
        BREW_CHECK(((uintptr_t)rope->qnorm & 3) == 0 && ((uintptr_t)rope->knorm & 3) == 0, BREW_ERR_INVALID_ARG,
                   "unaligned norm weights");
        p.rope = rope->mode;
        p.rope_scale = rope->scale;
        p.log2_base_hd = p.rope == BREW_KV_ROPE_NONE ? 0.0 : std::log2(rope->base) / c.head_size;
        p.qnorm = rope->qnorm;
        p.knorm = rope->knorm;
        p.eps = rope->eps;
    }
    if (rows->n_seqs == 0) return BREW_OK;
    DeviceScope ds;
    if (ds.rc) return ds.rc;
    p.kv = kv_view(kv, layer);
    p.rows = rows_dev(rows);
    p.q = q;
    p.q_out = q_out;
    p.k = k;
    p.v = v;
    p.ldq = ldq;
    p.ldkv = ldkv;
    return kv_append_launch(c.head_size, p, static_cast<cudaStream_t>(stream));
}

int brew_kv_read_dev(brew_kv kv, int32_t layer, float* k_out, float* v_out, int64_t ld, const brew_kv_rows* rows,
                     void* stream) {
    int rc = check_rows(kv, layer, rows);
    if (rc) return rc;
    const brew_kv_config& c = kv->c;
    BREW_CHECK(k_out || v_out, BREW_ERR_INVALID_ARG, "k_out and v_out are null");
    if ((k_out && (rc = check_matrix("k_out", k_out, ld, (int64_t)c.n_kv_heads * c.head_size))) ||
        (v_out && (rc = check_matrix("v_out", v_out, ld, (int64_t)c.n_kv_heads * c.head_size))))
        return rc;
    if (rows->n_seqs == 0) return BREW_OK;
    DeviceScope ds;
    if (ds.rc) return ds.rc;
    const KvView view = kv_view(kv, layer);
    const KvRowsDev rd = rows_dev(rows);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (c.head_size / 32) {
        case 1: return read_r<1>(view, rd, k_out, v_out, ld, s);
        case 2: return read_r<2>(view, rd, k_out, v_out, ld, s);
        case 3: return read_r<3>(view, rd, k_out, v_out, ld, s);
        case 4: return read_r<4>(view, rd, k_out, v_out, ld, s);
        default: return read_r<8>(view, rd, k_out, v_out, ld, s);
    }
}

int64_t brew_kv_workspace_bytes(brew_kv kv) { return kv ? kv_attend_workspace(kv->c.head_size) : -1; }

int brew_kv_attend_dev(brew_kv kv, int32_t layer, float* out, int64_t ldo, const float* q, int64_t ldq,
                       const brew_kv_rows* rows, int32_t window, float scale, void* workspace, void* stream) {
    int rc = check_rows(kv, layer, rows);
    if (rc) return rc;
    const brew_kv_config& c = kv->c;
    if ((rc = check_matrix("out", out, ldo, (int64_t)c.n_heads * c.head_size)) ||
        (rc = check_matrix("q", q, ldq, (int64_t)c.n_heads * c.head_size)))
        return rc;
    BREW_CHECK(window >= 0, BREW_ERR_INVALID_ARG, "window %d", window);
    BREW_CHECK(std::isfinite(scale), BREW_ERR_INVALID_ARG, "scale %g", (double)scale);
    BREW_CHECK(workspace && ((uintptr_t)workspace & 255) == 0, BREW_ERR_INVALID_ARG,
               "the workspace must be given, on a 256-byte boundary");
    if (rows->n_seqs == 0) return BREW_OK;
    DeviceScope ds;
    if (ds.rc) return ds.rc;
    KvAttendParams p = {};
    p.kv = kv_view(kv, layer);
    p.rows = rows_dev(rows);
    p.q = q;
    p.out = out;
    p.ldq = ldq;
    p.ldo = ldo;
    p.window = window;
    p.scale = scale != 0.0f ? scale : 1.0f / (float)std::sqrt((double)c.head_size);   // AttentionEngine.java:18-19
    p.workspace = workspace;
    return kv_attend_launch(c.head_size, p, static_cast<cudaStream_t>(stream));
}

int brew_kv_check(brew_kv kv) {
    BREW_CHECK(kv, BREW_ERR_INVALID_ARG, "null K/V cache");
    DeviceScope ds;
    if (ds.rc) return ds.rc;
    BREW_CUDA(cudaDeviceSynchronize());
    unsigned int v = 0;
    BREW_CUDA(cudaMemcpy(&v, kv->err, sizeof(v), cudaMemcpyDeviceToHost));
    if (v == 0) return BREW_OK;
    BREW_CUDA(cudaMemset(kv->err, 0, sizeof(v)));
    BREW_CUDA(cudaStreamSynchronize(0));
    if (v & (BREW_DEVERR_TIMEOUT_FULL | BREW_DEVERR_TIMEOUT_EMPTY))
        return set_error(BREW_ERR_TIMEOUT, "K/V cache: a bounded device wait timed out (flags 0x%x)", v);
    return set_error(BREW_ERR_OUT_OF_BOUNDS,
                     "K/V cache: a sequence, position or row outside the cache or its reserved pages was skipped");
}

}  // extern "C"
