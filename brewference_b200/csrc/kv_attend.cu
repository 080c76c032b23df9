// kv_attend.cu — attention over the paged 4-bit K/V cache:
//   o = sum_t softmax_t(scale * q . k_t) v_t
// over the positions t <= the row's own (and > own - window).
#include "brew_internal.cuh"
#include "kv.cuh"

namespace brew {
namespace {

constexpr int AT_WARPS = 4;

// One CTA per (row, head, sequence); each warp walks every fourth position
// with a running maximum and sum, and the warps join in shared memory.
template <int R>
__global__ void __launch_bounds__(32 * AT_WARPS) kv_attend_kernel(const __grid_constant__ KvAttendParams p) {
    constexpr int HD = 32 * R;
    constexpr int NV = R == 8 ? 2 : 1;
    __shared__ float sm[AT_WARPS][HD], sml[AT_WARPS][2];
    const KvEntry e = kv_entry(p.kv, p.rows, blockIdx.z, threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0);
    const int j = blockIdx.x, h = blockIdx.y;
    if (j >= e.rows) return;
    const int hk = h / (p.kv.n_heads / p.kv.n_kv);
    const int pos = e.pos0 + j;
    const int first = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool act = 4 * lane < HD;
    const float* qr = p.q + (e.row0 + j) * p.ldq + (int64_t)h * HD;
    float q[NV][4], o[NV][4];
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            q[n][c] = act ? qr[128 * n + 4 * lane + c] : 0.0f;
            o[n][c] = 0.0f;
        }
    float m = -INFINITY, l = 0.0f;
    for (int t = first + warp; t <= pos; t += AT_WARPS) {
        const uint8_t* grp = kv_group<R>(p.kv, e.seq, t, hk);
        const uint16_t* kq = reinterpret_cast<const uint16_t*>(grp);
        const uint16_t* sc = reinterpret_cast<const uint16_t*>(grp + 512 * R);
        const int pg = t & 15, u = pg >> 3, li = lane & 7;
        float s = 0.0f, v[NV][4];
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            if (!act) break;
            const int b = 4 * n + lane / 8, si = kv_scale(R, pg, b);
            const uint32_t qk = kq[2 * kv_word(R, u, b, (pg & 7) * 4 + li / 2) + (li & 1)];
            const uint32_t qv = kq[128 * R + 2 * kv_word(R, u, b, li * 4 + ((pg & 7) >> 1)) + (pg & 1)];
            const float dk = half_bits_to_float(sc[si]), dv = half_bits_to_float(sc[16 * R + si]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s += q[n][c] * ((float)((int)(qk >> 4 * c & 15) - 8) * dk);
                v[n][c] = (float)((int)(qv >> 4 * c & 15) - 8) * dv;
            }
        }
        s = warp_sum(s) * p.scale;
        const float mn = fmaxf(m, s);
        const float corr = expf(m - mn), w = expf(s - mn);
        l = l * corr + w;
        m = mn;
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[n][c] = act ? o[n][c] * corr + w * v[n][c] : 0.0f;
    }
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (act) sm[warp][128 * n + 4 * lane + c] = o[n][c];
    if (lane == 0) {
        sml[warp][0] = m;
        sml[warp][1] = l;
    }
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
    for (int w = 0; w < AT_WARPS; ++w) M = fmaxf(M, sml[w][0]);
    for (int w = 0; w < AT_WARPS; ++w) L += sml[w][0] == -INFINITY ? 0.0f : sml[w][1] * expf(sml[w][0] - M);
    for (int d = threadIdx.x; d < HD; d += 32 * AT_WARPS) {
        float a = 0.0f;
        for (int w = 0; w < AT_WARPS; ++w) a += sml[w][0] == -INFINITY ? 0.0f : sm[w][d] * expf(sml[w][0] - M);
        p.out[(e.row0 + j) * p.ldo + (int64_t)h * HD + d] = a / L;
    }
}

template <int R>
int attend_r(const KvAttendParams& p, cudaStream_t s) {
    const dim3 grid(p.rows.max_rows, p.kv.n_heads, p.rows.n_seqs);
    kv_attend_kernel<R><<<grid, 32 * AT_WARPS, 0, s>>>(p);
    BREW_CUDA(cudaGetLastError());
    count_launch();
    return BREW_OK;
}

}  // namespace

int64_t kv_attend_workspace(int head_size) { return 256; }

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
