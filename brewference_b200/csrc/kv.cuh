// kv.cuh — the paged 4-bit K/V cache: layout, kernel parameters, launches.
//
// A page holds page_tokens consecutive positions of one sequence, for every
// kv head.  Its unit is the group: 16 positions of one kv head, 576 R bytes
// (R = head_size / 32 blocks a row), contiguous:
//
//   K quants  256 R bytes   V quants  256 R bytes
//   K scales   32 R bytes   V scales   32 R bytes
//
// The quants of a group are words in the order in which the lanes of a warp
// feed them to mma.m16n8k16, so that a lane reads its share with 16-byte
// loads and unpacks it with masks alone.  With lane = 4 g + i, u = 0, 1 the
// half of the group and b the block:
//
//   K word (u, b, lane)   position 8 u + g, dims 32 b + 8 i + n in nibble n
//   V word (u, b, lane)   positions 8 u + 2 i + e in 16-bit half e, dims
//                         32 b + 4 g + j in the half's nibble j
//   K scales              fp16, p R + b: a position's side by side
//   V scales              fp16, ((p / 2) R + b) 2 + p % 2: a position pair's
//                         scales of one block side by side
//
// A nibble q stands for (q - 8) * scale: the values of GGML's Q4_0 blocks.
#pragma once

#include "brew_common.cuh"

namespace brew {

constexpr int KV_GROUP = 16;          // positions of a group
constexpr int KV_MAX_SEQS = 2048;     // sequences of a cache, and of a call
constexpr int KV_MAX_HEAD = 256;

__host__ __device__ constexpr int kv_group_bytes(int R) { return 576 * R; }

// Index of K or V word (u, b, lane) of a group: vectors of W words per lane.
__host__ __device__ constexpr int kv_word(int R, int u, int b, int lane) {
    const int W = R % 2 == 0 ? 4 : 2, m = u * R + b;
    return ((m / W) * 32 + lane) * W + m % W;
}

__host__ __device__ constexpr int kv_kscale(int R, int p, int b) { return p * R + b; }
__host__ __device__ constexpr int kv_vscale(int R, int p, int b) { return ((p >> 1) * R + b) * 2 + (p & 1); }

// One launch of a reservation: page ids first .. first + n - 1 of a sequence,
// and its reserved positions, or -1 where more launches follow: the length is
// published behind its last page id, so that one whose launches fail midway
// leaves the old one in force (its pages may be another sequence's by then).
constexpr int KV_PUT_PAGES = 120;
struct KvPut {
    int first, n, tokens;
};
inline KvPut kv_put(int first, int end, int tokens) {
    const int n = end - first < KV_PUT_PAGES ? end - first : KV_PUT_PAGES;
    return {first, n, first + n == end ? tokens : -1};
}

// The cache as the kernels see it, one layer.
struct KvView {
    uint8_t* pages;            // [n_pages][n_kv][page_tokens / 16] groups
    const int32_t* table;      // [max_seqs][max_pages] page ids
    const int32_t* reserved;   // [max_seqs] positions that have a page
    int max_seqs, max_pages;
    int page_shift;            // log2(page_tokens)
    int n_heads, n_kv;
    unsigned int* err;
};

// The rows of a call: entry i of n_seqs has rows row_start[i] ..
// row_start[i + 1] - 1 (without row_start: row i) of sequence seq[i], at
// positions pos[i], pos[i] + 1, ...
struct KvRowsDev {
    const int32_t* seq;
    const int32_t* pos;
    const int32_t* row_start;
    int n_seqs, n_rows, max_rows;
};

struct KvAppendParams {
    KvView kv;
    KvRowsDev rows;
    const float *q, *k, *v;
    float* q_out;
    int64_t ldq, ldkv;
    int rope;                  // BREW_KV_ROPE_*
    double rope_scale, log2_base_hd;   // angle = pos * rope_scale * 2^(-2 i log2(base) / hd)
    const float *qnorm, *knorm;
    double eps;
};

struct KvAttendParams {
    KvView kv;
    KvRowsDev rows;
    const float* q;
    float* out;
    int64_t ldq, ldo;
    int window;
    float scale;
    void* workspace;
    uint32_t code_base;        // set by the launch
    int prompts;               // the prompt kernel follows
    int64_t pairs_min;         // entries of fewer (row, head) pairs a kv head are the single-token kernel's, the others
                               // the prompt kernel's
};

// The kernels' view of a cache's layer (kernels record bad rows in its own error word unless the caller sets another),
// and every page zeroed in stream order.
KvView kv_view(const brew_kv_s* kv, int layer);
int kv_clear(brew_kv_s* kv, cudaStream_t s);
int kv_append_launch(int head_size, const KvAppendParams& p, cudaStream_t s);
int kv_attend_launch(int head_size, const KvAttendParams& p, cudaStream_t s);
int64_t kv_attend_workspace(int head_size);
// The workspace's arrival counters set to `value` bytes in stream order: 0 makes it ready again after a call that a
// bounded wait ended.
int kv_attend_counters(int head_size, void* workspace, int value, cudaStream_t s);
bool kv_head_supported(int head_size);
// The prompt kernel (tcgen05), its part of the workspace: kv_attend_launch's.
constexpr int KV_COUNTER_BYTES = 4096;
bool kv_prefill_supported(int head_size);
int64_t kv_prefill_workspace(int head_size);
int kv_prefill_launch(int head_size, const KvAttendParams& p, cudaStream_t s);

// Entry i of a call, checked: its rows lie in the buffers, its sequence in
// the cache and its positions in reserved pages.  A bad entry has no rows.
struct KvEntry {
    int seq, pos0, row0, rows;
    bool bad;
};

__host__ __device__ inline KvEntry kv_check_entry(const KvView& kv, const KvRowsDev& r, int i) {
    KvEntry e;
    e.seq = r.seq[i];
    e.pos0 = r.pos[i];
    e.row0 = r.row_start ? r.row_start[i] : i;
    const int64_t end = r.row_start ? r.row_start[i + 1] : i + 1;
    const int64_t n = end - e.row0;
    bool ok = e.row0 >= 0 && n >= 0 && end <= r.n_rows && n <= r.max_rows;
    if (ok && n > 0)
        ok = e.seq >= 0 && e.seq < kv.max_seqs && e.pos0 >= 0 && (int64_t)e.pos0 + n <= kv.reserved[e.seq];
    e.rows = ok ? (int)n : 0;
    e.bad = !ok;
    return e;
}

// Byte offset in a layer of the group of position `pos` (reserved) of
// sequence `seq`, kv head hk.
template <int R>
__host__ __device__ inline int64_t kv_group_at(const KvView& kv, int seq, int pos, int hk) {
    const int page = kv.table[(int64_t)seq * kv.max_pages + (pos >> kv.page_shift)];
    const int per = 1 << (kv.page_shift - 4);   // groups of a page and head
    return (((int64_t)page * kv.n_kv + hk) * per + ((pos >> 4) & (per - 1))) * kv_group_bytes(R);
}

#ifdef __CUDACC__

// kv_check_entry, a bad entry recorded by the caller's thread `rec`.
__device__ __forceinline__ KvEntry kv_entry(const KvView& kv, const KvRowsDev& r, int i, bool rec) {
    const KvEntry e = kv_check_entry(kv, r, i);
    if (e.bad && rec) atomicOr(kv.err, BREW_DEVERR_BAD_INDEX);
    return e;
}

template <int R>
__device__ __forceinline__ uint8_t* kv_group(const KvView& kv, int seq, int pos, int hk) {
    return kv.pages + kv_group_at<R>(kv, seq, pos, hk);
}

#endif

}  // namespace brew
