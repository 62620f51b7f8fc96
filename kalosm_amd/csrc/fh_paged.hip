// Paged key-value cache: entry points, argument checks, rotary positions with the append to the pages.
//
// The reference keeps one dense cache a sequence (fusor-ml/fusor/src/cache/kv_cache.rs:24-63) and rotates q and k by one
// position a token (composite/rope.rs:284-329), or by three of them where pictures are among the tokens
// (models/kalosm-llama/src/raw/rope.rs); pages have no counterpart there.
#include "fh_paged.h"

fh_status PagedGpu::enter(const fh_device *dev) {
    int now = -1;
    FH_HIP(hipGetDevice(&now));
    if (now != dev->ordinal) {
        FH_HIP(hipSetDevice(dev->ordinal));
        before = now;
    }
    return FH_OK;
}
PagedGpu::~PagedGpu() {
    if (before >= 0) (void)hipSetDevice(before);
}

fh_status fh_paged_arguments(int dtype, int kv_dtype, int hq, int hkv, int d, const void *k_pages, const void *v_pages, int64_t page_stride,
                             int64_t head_stride, int64_t slot_stride, int pages, int page_size, const int32_t *starts, const int32_t *lens,
                             const int32_t *table, int cols, int seqs, int tokens, PagedKv *kv, PagedRows *rows) {
    FH_REQUIRE(k_pages && v_pages && lens && table, "NULL argument");
    FH_REQUIRE(dtype == FH_F32 || dtype == FH_F16 || dtype == FH_PAGED_BF16, "rows are f32, f16 or bf16, not type %d", dtype);
    FH_REQUIRE(kv_dtype == FH_F32 || kv_dtype == FH_F16 || kv_dtype == FH_PAGED_BF16, "pages are f32, f16 or bf16, not type %d", kv_dtype);
    if (dtype != kv_dtype && dtype != FH_F32)
        FH_FAIL(FH_ERR_UNSUPPORTED, "rows of type %d over pages of type %d: the same type, or f32 rows", dtype, kv_dtype);
    FH_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0, "%d query heads do not share %d KV heads evenly", hq, hkv);
    FH_REQUIRE(d > 0 && seqs >= 0 && tokens >= 0 && pages > 0 && cols > 0, "bad shape");
    if (d % 8 || d > 256) FH_FAIL(FH_ERR_UNSUPPORTED, "head_dim %d: paged attention takes multiples of 8 up to 256", d);
    if (page_size < 16 || page_size > 4096 || (page_size & (page_size - 1)))
        FH_FAIL(FH_ERR_UNSUPPORTED, "pages of %d positions: powers of two from 16 to 4096 are supported", page_size);
    FH_REQUIRE(hq <= 65535 && seqs <= 65535 && pages <= FH_PAGED_MAX, "at most 65535 heads and sequences and 2^29 pages");
    FH_REQUIRE((int64_t)cols * page_size <= FH_PAGED_MAX, "a table row of %d pages of %d positions reaches past 2^29", cols, page_size);
    FH_REQUIRE(starts || tokens == seqs, "%d rows of %d sequences need their starts", tokens, seqs);
    const int size = kv_dtype == FH_F32 ? 4 : 2;
    const int64_t lim = INT64_MAX / 8 / pages / size;
    FH_REQUIRE(slot_stride >= d && head_stride >= d && page_stride >= d && slot_stride <= (1 << 24) && head_stride <= INT64_MAX / 8 / hkv / size && page_stride <= lim,
               "page strides (%lld, %lld, %lld)", (long long)page_stride, (long long)head_stride, (long long)slot_stride);
    // [page][head][slot] or [page][slot][head]; rows that overlap would be written by two
    const bool by_head = head_stride >= page_size * slot_stride && page_stride >= hkv * head_stride;
    const bool by_slot = slot_stride >= hkv * head_stride && page_stride >= page_size * slot_stride;
    FH_REQUIRE(by_head || by_slot || (hkv == 1 && page_stride >= page_size * slot_stride), "pages of strides (%lld, %lld, %lld) overlap", (long long)page_stride,
               (long long)head_stride, (long long)slot_stride);
    if ((((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) || (slot_stride * size) % 16 || (head_stride * size) % 16 || (page_stride * size) % 16)
        FH_FAIL(FH_ERR_UNSUPPORTED, "rows of pages begin at multiples of 16 bytes");
    int shift = 4;
    while (1 << shift < page_size) shift++;
    *kv = PagedKv{(const char *)k_pages, (const char *)v_pages, page_stride * size, head_stride * size, slot_stride * size, pages, shift};
    *rows = PagedRows{starts, lens, table, cols, seqs, tokens, 1};
    return FH_OK;
}

// ---------------------------------------------------------------- rotation and append
enum { PAGED_AXES = 4 };
struct PagedTurn {
    const float *cos, *sin; // [table_rows][pairs of the tables' rows]
    const int *positions;   // [axes][tokens], NULL: the position in the cache
    int table_rows, table_pairs, pairs, axes, end[PAGED_AXES]; // pairs that turn (the first 2 * pairs of a head's values); the axis' last pair + 1
};

// One workgroup a row; a thread takes the pairs and the values of all heads in turn.
template <typename TX, typename TP, bool TANGLED>
__global__ __launch_bounds__(256) void k_paged_append(const TX *q, int64_t q_st, int64_t q_sh, const TX *__restrict__ k, const TX *__restrict__ v,
                                                      int64_t kv_st, int64_t kv_sh, int hq, int hkv, int d, PagedTurn turn, PagedKv kv, PagedRows rows,
                                                      TX *q_out) { // (q_out may be q)
    const int row = blockIdx.x, tid = threadIdx.x;
    int lo = 0, hi = rows.seqs; // the sequence whose rows this one is among: the last that begins at or before it
    if (rows.starts)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (rows.starts[mid] <= row) lo = mid;
            else hi = mid;
        }
    else
        lo = row;
    if (rows.starts && (row < rows.starts[lo] || row >= rows.starts[lo + 1])) return; // before the first or behind the last sequence
    const int len = rows.lens[lo], p = rows.starts ? len - (rows.starts[lo + 1] - row) : len - 1;
    if (len > FH_PAGED_MAX || p < 0 || p >> kv.shift >= rows.cols) return;
    const int page = rows.table[(int64_t)lo * rows.cols + (p >> kv.shift)];
    if ((unsigned)page >= (unsigned)kv.pages) return;
    const int64_t at = (int64_t)page * kv.page + (int64_t)(p & ((1 << kv.shift) - 1)) * kv.slot;
    int where[PAGED_AXES] = {p, p, p, p};
    if (turn.pairs) {
        for (int a = 0; a < turn.axes; a++) {
            if (turn.positions) where[a] = turn.positions[(int64_t)a * rows.tokens + row];
            if ((unsigned)where[a] >= (unsigned)turn.table_rows) return;
        }
    }
    const int units = d / 2, turned = (q ? hq : 0) + hkv;
    for (int i = tid; i < turned * units; i += 256) {
        const int h = i / units, j = i % units;
        const bool is_q = q && h < hq;
        const int kh = h - (q ? hq : 0);
        const TX *from = is_q ? q + row * q_st + h * q_sh : k + row * kv_st + kh * kv_sh;
        int a = 2 * j, b = 2 * j + 1; // behind the turned pairs: neighbours, as they are
        float c = 1.f, s = 0.f;
        if (j < turn.pairs) {
            if (!TANGLED) a = j, b = j + turn.pairs;
            int pos = where[0];
#pragma unroll
            for (int e = 0; e + 1 < PAGED_AXES; e++)
                if (j >= turn.end[e]) pos = where[e + 1];
            c = turn.cos[(int64_t)pos * turn.table_pairs + j];
            s = turn.sin[(int64_t)pos * turn.table_pairs + j];
        }
        const float x = (float)from[a], y = (float)from[b];
        const float u = j < turn.pairs ? x * c - y * s : x, w = j < turn.pairs ? x * s + y * c : y;
        if (is_q) {
            TX *to = q_out + ((int64_t)row * hq + h) * d;
            to[a] = (TX)u, to[b] = (TX)w;
        } else {
            TP *to = (TP *)((char *)kv.k + at + kh * kv.head);
            to[a] = (TP)u, to[b] = (TP)w;
        }
    }
    for (int i = tid; i < hkv * d; i += 256) {
        const int h = i / d, e = i % d;
        ((TP *)((char *)kv.v + at + h * kv.head))[e] = (TP)v[row * kv_st + h * kv_sh + e];
    }
}

extern "C" fh_status fh_paged_rope_append(fh_device *dev, int32_t dtype, int32_t kv_dtype, const void *q_dev, int64_t q_st, int64_t q_sh,
                                          const void *k_dev, const void *v_dev, int64_t kv_st, int64_t kv_sh, int32_t hq, int32_t hkv, int32_t d,
                                          const float *cos_dev, const float *sin_dev, int32_t table_rows, int32_t table_pairs,
                                          const int32_t *positions_dev, const int32_t *sections_host, int32_t axes, int32_t interleaved,
                                          void *k_pages_dev, void *v_pages_dev, int64_t page_stride, int64_t head_stride, int64_t slot_stride,
                                          int32_t pages, int32_t page_size, const int32_t *starts_dev, const int32_t *lens_dev,
                                          const int32_t *table_dev, int32_t table_cols, int32_t seqs, int32_t tokens, void *q_out_dev) {
    PagedKv kv;
    PagedRows rows;
    FH_TRY(fh_paged_arguments(dtype, kv_dtype, hq, hkv, d, k_pages_dev, v_pages_dev, page_stride, head_stride, slot_stride, pages, page_size,
                              starts_dev, lens_dev, table_dev, table_cols, seqs, tokens, &kv, &rows));
    FH_REQUIRE(k_dev && v_dev, "NULL argument");
    FH_REQUIRE(!q_dev == !q_out_dev, "q and its output come together");
    FH_REQUIRE((cos_dev != nullptr) == (sin_dev != nullptr), "cos and sin come together");
    PagedTurn turn = {};
    if (cos_dev) {
        FH_REQUIRE(axes >= 1 && axes <= PAGED_AXES, "%d axes: 1 .. %d are supported", axes, (int)PAGED_AXES);
        FH_REQUIRE(axes == 1 || (positions_dev && sections_host), "several axes need their positions and sections");
        FH_REQUIRE(table_rows > 0 && table_pairs > 0, "bad tables");
        int64_t n = 0;
        for (int a = 0; a < PAGED_AXES; a++) {
            if (a < axes) {
                const int s = sections_host ? sections_host[a] : table_pairs;
                FH_REQUIRE(s >= 0, "section %d has %d pairs", a, s);
                n += s;
            }
            FH_REQUIRE(n <= table_pairs && 2 * n <= d, "sections of %lld pairs in a head of %d values and tables of %d", (long long)n, d, table_pairs);
            turn.end[a] = a + 1 < axes ? (int)n : d; // (the last axis has whatever follows)
        }
        FH_REQUIRE(n > 0, "sections without a pair");
        turn.cos = cos_dev, turn.sin = sin_dev, turn.positions = positions_dev;
        turn.table_rows = table_rows, turn.table_pairs = table_pairs, turn.pairs = (int)n, turn.axes = axes;
    } else
        FH_REQUIRE(!positions_dev && !sections_host, "positions without tables");
    FH_REQUIRE(dev, "NULL device");
    if (!tokens || !seqs) return FH_OK;
    PagedGpu gpu;
    FH_TRY(gpu.enter(dev));
#define FH_PA(TX, TP)                                                                                                                            \
    (interleaved ? k_paged_append<TX, TP, true> : k_paged_append<TX, TP, false>)<<<dim3((unsigned)tokens), dim3(256), 0, dev->stream>>>(            \
        (const TX *)q_dev, q_st, q_sh, (const TX *)k_dev, (const TX *)v_dev, kv_st, kv_sh, hq, hkv, d, turn, kv, rows, (TX *)q_out_dev)
    if (dtype == FH_F16) FH_PA(fh_half, fh_half);
    else if (dtype == FH_PAGED_BF16) FH_PA(fh_bf, fh_bf);
    else if (kv_dtype == FH_F32) FH_PA(float, float);
    else if (kv_dtype == FH_F16) FH_PA(float, fh_half);
    else FH_PA(float, fh_bf);
#undef FH_PA
    FH_HIP(hipGetLastError());
    return FH_OK;
}

// ---------------------------------------------------------------- attention
extern "C" fh_status fh_paged_attention(fh_device *dev, int32_t dtype, int32_t kv_dtype, const void *q_dev, int64_t q_st, int64_t q_sh, int32_t hq,
                                        int32_t hkv, int32_t d, float scale, int32_t window, const void *k_pages_dev, const void *v_pages_dev,
                                        int64_t page_stride, int64_t head_stride, int64_t slot_stride, int32_t pages, int32_t page_size,
                                        const int32_t *starts_dev, const int32_t *lens_dev, const int32_t *table_dev, int32_t table_cols, int32_t seqs,
                                        int32_t tokens, int32_t max_new, int32_t max_len, void *out_dev) {
    PagedKv kv;
    PagedRows rows;
    FH_TRY(fh_paged_arguments(dtype, kv_dtype, hq, hkv, d, k_pages_dev, v_pages_dev, page_stride, head_stride, slot_stride, pages, page_size,
                              starts_dev, lens_dev, table_dev, table_cols, seqs, tokens, &kv, &rows));
    FH_REQUIRE(q_dev && out_dev, "NULL argument");
    FH_REQUIRE(scale >= 0x1p-60f && scale < INFINITY, "scale %g", (double)scale);
    FH_REQUIRE(window >= 0 && max_new >= 0 && max_len >= 0, "window %d, max_new %d, max_len %d", window, max_new, max_len);
    FH_REQUIRE(dev, "NULL device");
    if (!tokens || !seqs || !max_new) return FH_OK;
    rows.max_new = max_new < tokens ? max_new : tokens;
    PagedGpu gpu;
    FH_TRY(gpu.enter(dev));
    const PagedCall call = {q_dev, out_dev, q_st, q_sh, kv, rows, scale, window, hq, hkv, d};
    if (rows.max_new == 1) return fh_paged_step(dev, dtype, kv_dtype, call, max_len);
    return fh_paged_prompt(dev, dtype, kv_dtype, call, max_len);
}
