// A paged key-value cache as kernels see it: which rows belong to which sequence, and where its positions lie.
#pragma once
#include "fh_internal.h"

typedef _Float16 fh_half;
typedef __bf16 fh_bf;

enum { FH_PAGED_BF16 = FH_DECODER_BF16, FH_PAGED_MAX = 1 << 29 /* positions of a sequence */ };

// From a maximum m of this size on, in the log2 domain, a weight's exponent is (score rounded as m was - m) + 14 next to f16, without the 14 next to
// other types; below it one fma: score + (14 - m).  What m and 14 - m are rounded by is in the latter, and 14 - m is rounded by more than m where it lies above a power
// of two that |m| is below: below 2^22 by 2^-3 and 2^-2 at most, so weights that start at 2^14, or 2^15.5 in prompts, stay below f16's 2^16.
#define PAGED_FAR 0x1p22f

struct PagedKv {
    const char *k, *v;
    int64_t page, head, slot; // strides in bytes, K and V alike
    int pages, shift;         // page_size = 1 << shift, 16 .. 4096
};
struct PagedRows {
    const int *starts, *lens, *table; // starts NULL: one row a sequence
    int cols, seqs, tokens, max_new;
};
struct PagedSeq {
    int row, rows; // rows of q and out: row .. row + rows - 1, all of them inside the tensors whatever `starts` holds
    int first;     // position of the first of them (below 0 where the sequence is said to be shorter than its new rows)
    int len;       // positions that can be read: no further than the table's row reaches
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedRows &r, int shift, int len, int from, int to) {
    PagedSeq s;
    len = len < 0 ? 0 : len > FH_PAGED_MAX ? FH_PAGED_MAX : len;
    from = from < 0 ? 0 : from > r.tokens ? r.tokens : from;
    to = to < from ? from : to > r.tokens ? r.tokens : to;
    s.row = from;
    s.first = len - (to - from);
    s.rows = to - from < r.max_new ? to - from : r.max_new;
    const int64_t reach = (int64_t)r.cols << shift;
    s.len = len < reach ? len : (int)reach;
    return s;
}
__device__ __forceinline__ PagedSeq paged_seq(const PagedRows &r, int shift, int i) {
    return r.starts ? paged_seq(r, shift, r.lens[i], r.starts[i], r.starts[i + 1]) : paged_seq(r, shift, r.lens[i], i, i + 1);
}
// The same for an index that is the wavefront's, by scalar loads: their waits leave the vector loads that are on their way alone.
typedef const __attribute__((address_space(4))) int *PagedScalars;
__device__ __forceinline__ int paged_scalar(const int *p, int64_t i) { return ((PagedScalars)(uintptr_t)p)[i]; }
__device__ __forceinline__ PagedSeq paged_seq_scalar(const PagedRows &r, int shift, int i) {
    const int len = paged_scalar(r.lens, i);
    return r.starts ? paged_seq(r, shift, len, paged_scalar(r.starts, i), paged_scalar(r.starts, i + 1)) : paged_seq(r, shift, len, i, i + 1);
}

// The first of an f32 value's terms, what is left is the next ones': rounded, but to bf16's largest value what would be rounded to infinity (infinities and NaN stay in
// what is left).
template <typename T> __device__ __forceinline__ T paged_first(float x) {
    if constexpr (__is_same(T, fh_bf)) x = fminf(fmaxf(x, -0x1.fep127f), 0x1.fep127f);
    return (T)x;
}

// The scale of scores whose row is taken 2^ex times as large.  It stays a normal number - ex is no larger than that allows, and scores of smaller rows do not tell
// positions apart: they are below 2^(15 + 16 + 8 - 126) - and finite: where it would not be, scores are 0 or, of the smallest key, 2^(14 - 24 + 128) apart.
__device__ __forceinline__ float paged_brought(float scale, int &ex) {
    const int most = __builtin_amdgcn_frexp_expf(scale) + 125;
    ex = ex < most ? ex : most;
    return fminf(ldexpf(scale, -ex), 0x1.fffffep127f);
}

// One row and head by a wavefront, over the positions from .. to: what the tiles are checked against where they end up infinite or NaN (an infinity or a NaN
// among values that a neighbour sees and this row does not, terms of an infinite f32).  A key a lane for the scores; o[e]: value lane + 64 e.  m is in
// the log2 domain, weights are 2^shift times what they are.
template <typename TX, typename TP>
__device__ __forceinline__ void paged_again(const TX *q, int d, float sc2, float shift, const PagedKv &kv, const int *table, int kh, int from, int to, float &m, float &l,
                                            float (&o)[4]) {
    constexpr float SMALLER = __is_same(TP, fh_half) ? 0x1p-24f : 1.f; // (f32 rows times f16 keys: 2^127 * 2^16 * 256; keys of the other types can be as large as rows are small)
    const int lane = threadIdx.x & 63;
    m = -INFINITY, l = 0.f;
    for (int e = 0; e < 4; e++) o[e] = 0.f;
    for (int t = from; t <= to; t += 64) {
        const int key = t + lane;
        float y = -INFINITY;
        int64_t at = -1;
        if (key <= to) {
            const int page = table[key >> kv.shift];
            if ((unsigned)page < (unsigned)kv.pages) {
                at = page * kv.page + kh * kv.head + (key & ((1 << kv.shift) - 1)) * kv.slot;
                y = 0.f;
#pragma unroll 1 // (few registers: it stands behind loops that have none left)
                for (int e = 0; e < d; e += 8) { // (multiples of 8 at multiples of 16 bytes)
                    TP x[8];
                    uint4 w[sizeof(TP) / 2];
                    for (int i = 0; i < (int)sizeof(TP) / 2; i++) w[i] = ((const uint4 *)(kv.k + at + e * (int)sizeof(TP)))[i];
                    __builtin_memcpy(x, w, sizeof(x));
                    for (int i = 0; i < 8; i++) y = fmaf((float)q[e + i] * SMALLER, (float)x[i], y);
                }
                y *= sc2 / SMALLER;
            }
        }
        float mx = y;
        for (int w = 32; w; w >>= 1) mx = fmaxf(mx, __shfl_xor(mx, w));
        mx = fmaxf(mx, m);
        const float ref = mx == -INFINITY ? 0.f : mx, alpha = __builtin_amdgcn_exp2f(m - ref), pr = at < 0 ? 0.f : __builtin_amdgcn_exp2f(y - ref + shift);
        m = mx;
        float sum = pr;
        for (int w = 32; w; w >>= 1) sum += __shfl_xor(sum, w);
        l = l * alpha + sum;
        for (int e = 0; e < 4; e++) o[e] *= alpha;
#pragma unroll 4
        for (int j = 0; j < 64; j++) {
            const int64_t v = __shfl(at, j);
            const float p = __shfl(pr, j);
            if (v >= 0)
                for (int e = 0; e < 4; e++)
                    if (lane + 64 * e < d) o[e] = fmaf(p, (float)((const TP *)(kv.v + v))[lane + 64 * e], o[e]);
        }
        bool lost = true; // nothing that comes makes any of it finite again
        for (int e = 0; e < 4; e++) lost &= lane + 64 * e >= d || !(0.f * o[e] == 0.f);
        if (__all(lost || !(0.f * l == 0.f))) return;
    }
}

// Arguments both entry points check, without touching a device: FH_OK, or an error with its message.  `kv` and `rows` are filled in.
fh_status fh_paged_arguments(int dtype, int kv_dtype, int hq, int hkv, int d, const void *k_pages, const void *v_pages, int64_t page_stride,
                             int64_t head_stride, int64_t slot_stride, int pages, int page_size, const int32_t *starts, const int32_t *lens,
                             const int32_t *table, int cols, int seqs, int tokens, PagedKv *kv, PagedRows *rows);
// Arguments of fh_paged_attention that its kernels share.
struct PagedCall {
    const void *q;
    void *out;
    int64_t q_st, q_sh; // elements
    PagedKv kv;
    PagedRows rows;
    float scale;
    int window, hq, hkv, d;
};
// rows.max_new rows of a KV head's heads: one row, or up to 16 in all where fh_paged_step_whole.
fh_status fh_paged_step(fh_device *dev, int dtype, int kv_dtype, const PagedCall &call, int max_len);
bool fh_paged_step_whole(const fh_device *dev, int kv_dtype, const PagedCall &call, int max_len); // caches so short that a pair is one workgroup's
fh_status fh_paged_prompt(fh_device *dev, int dtype, int kv_dtype, const PagedCall &call, int max_len);
// The GPU of `dev` is the calling thread's current one while this lives.
struct PagedGpu {
    int before = -1;
    fh_status enter(const fh_device *dev);
    ~PagedGpu();
};
