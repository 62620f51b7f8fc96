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
    FH_REQUIRE(hq <= 65535 && seqs <= 65535 && pages <= FH_PAGED_MAX && tokens <= FH_PAGED_MAX, "at most 65535 heads and sequences and 2^29 pages and rows");
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
    int table_rows, table_pairs, pairs, axes, aligned, end[PAGED_AXES]; // aligned: four of a row's pairs are 16 bytes; pairs that turn (the first 2 * pairs of a head's values); the axis' last pair + 1
};

// Where a row goes: its sequence's page and slot, and its positions on the axes; at < 0: nowhere.  By scalar loads: a search through the starts
// (of few sequences: all in one cache line), the length and the axes' positions, the table.
struct PagedPlace {
    int64_t at; // bytes into the pages of head 0
    int where0, where1, where2, where3;
};
__device__ __forceinline__ PagedPlace paged_place(int row, const PagedRows &rows, const PagedKv &kv, const PagedTurn &turn) {
    PagedPlace x = {-1, 0, 0, 0, 0};
    const int *given = turn.positions ? turn.positions + row : rows.lens; // (axes that there are not: the first one's again)
    const int t = rows.tokens, g0 = paged_scalar(given, 0), g1 = paged_scalar(given, turn.positions && turn.axes > 1 ? t : 0),
              g2 = paged_scalar(given, turn.positions && turn.axes > 2 ? 2 * (int64_t)t : 0), g3 = paged_scalar(given, turn.positions && turn.axes > 3 ? 3 * (int64_t)t : 0);
    int seq = row, p;
    if (!rows.starts) p = paged_scalar(rows.lens, row) - 1;
    else {
        int lo = 0, hi = rows.seqs; // the last sequence that begins at or before the row
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (paged_scalar(rows.starts, mid) <= row) lo = mid;
            else hi = mid;
        }
        const int begin = paged_scalar(rows.starts, lo), end = paged_scalar(rows.starts, lo + 1), len = paged_scalar(rows.lens, lo);
        if (row < begin || row >= end) return x; // before the first or behind the last sequence
        seq = lo, p = len > FH_PAGED_MAX ? -1 : len - (end - row);
    }
    if (p < 0 || p >> kv.shift >= rows.cols) return x;
    const int page = paged_scalar(rows.table, (int64_t)seq * rows.cols + (p >> kv.shift));
    x.where0 = x.where1 = x.where2 = x.where3 = p;
    if (turn.positions) x.where0 = g0, x.where1 = g1, x.where2 = g2, x.where3 = g3;
    const unsigned end = (unsigned)turn.table_rows;
    const bool fits = !turn.pairs || ((unsigned)x.where0 < end && (unsigned)x.where1 < end && (unsigned)x.where2 < end && (unsigned)x.where3 < end);
    if (fits && (unsigned)page < (unsigned)kv.pages) x.at = page * kv.page + (p & ((1 << kv.shift) - 1)) * kv.slot;
    return x;
}
__device__ __forceinline__ int paged_axis_position(const PagedTurn &turn, const PagedPlace &x, int pair) {
    const int p0 = x.where0, p1 = x.where1, p2 = x.where2, p3 = x.where3; // (values: a choice among a structure's fields would put it into LDS)
    const int p = pair >= turn.end[0] ? p1 : p0, r = pair >= turn.end[1] ? p2 : p;
    return pair >= turn.end[2] ? p3 : r;
}

// Eight values of a row in memory.
template <typename T> struct Paged8 {
    T v[8];
};
template <typename T> __device__ __forceinline__ Paged8<T> paged_load8(const T *p) { // at a multiple of 16 bytes
    Paged8<T> x;
    const uint4 *u = (const uint4 *)p;
    uint4 w[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) w[i] = u[i];
    __builtin_memcpy(&x, w, sizeof(x));
    return x;
}
template <typename T> __device__ __forceinline__ void paged_store8(T *p, const float (&y)[8]) {
    T v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (T)y[e];
    uint4 w[sizeof(T) / 2];
    __builtin_memcpy(w, v, sizeof(v));
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) ((uint4 *)p)[i] = w[i];
}

// A thread takes eight pairs of a head, or eight values that are copied (V, what the sections leave): moves 4 to 6 bytes an operation, so it is bound by the
// memory for many rows, and by the chain of requests for few: the values are asked for before the row's place is looked up.
// (32 / 8 heads of 128: 1 row of f32 2.8 us, 64 of bf16 3.7, 22 thousand of f16 by three axes 97 to 106, 5.2 to 5.7 TB/s.)
// grid (rows, units of a row / 256)
template <typename TX, typename TP, bool TANGLED>
__global__ __launch_bounds__(256) void k_paged_append8(const TX *q, const TX *__restrict__ k, const TX *__restrict__ v, int hq, int hkv, int d, int n,
                                                       const int *__restrict__ starts, const int *__restrict__ lens, int seqs, int cols, int64_t q_st, int64_t q_sh,
                                                       int64_t kv_st, int64_t kv_sh, const int *__restrict__ table, int tokens, PagedKv kv, PagedTurn turn,
                                                       TX *q_out) { // (q_out may be q)
    const PagedRows rows = {starts, lens, table, cols, seqs, tokens, 0};
    const int row = blockIdx.x;
    int u = (int)blockIdx.y * 256 + threadIdx.x;
    const int heads = hq + hkv, turns = n / 8, copies = (d - 2 * n) / 8; // of a head (hq: 0 without q)
    // which of the row's units: pairs of q and k, then what is copied of them, then V (threads behind the last: that one, and they store nothing)
    const int all = heads * (turns + copies) + hkv * (d / 8);
    const bool mine = u < all;
    u = mine ? u : all - 1;
    int h, a, b; // head of q and k together (V: heads ..), its values a .. and b ..
    const bool turned = u < heads * turns;
    if (turned) {
        h = u / turns, a = (u - h * turns) * 8;
        if (TANGLED) a *= 2, b = a + 8;
        else b = a + n;
    } else if ((u -= heads * turns) < heads * copies) h = u / copies, a = b = 2 * n + (u - h * copies) * 8;
    else u -= heads * copies, h = u / (d / 8), a = b = (u - h * (d / 8)) * 8, h += heads;
    const TX *base = h < hq ? q : h < heads ? k : v;
    const int64_t st = h < hq ? q_st : kv_st, off = h < hq ? h * q_sh : (h - (h < heads ? hq : heads)) * kv_sh;
    const Paged8<TX> x = paged_load8(base + row * st + off + a), y = paged_load8(base + row * st + off + b);
    const PagedPlace to = paged_place(row, rows, kv, turn);
    if (to.at < 0 || !mine) return;
    float p[8], r[8];
#pragma unroll
    for (int e = 0; e < 8; e++) p[e] = (float)x.v[e], r[e] = (float)y.v[e];
    if (turned) {
        const int j = TANGLED ? a / 2 : a; // first pair
        bool one = turn.aligned; // axis for all eight
#pragma unroll
        for (int e = 0; e + 1 < PAGED_AXES; e++) one &= j >= turn.end[e] || j + 7 < turn.end[e];
        float c[8], s[8];
        if (one) {
            const int64_t at = (int64_t)paged_axis_position(turn, to, j) * turn.table_pairs + j;
            const float4 c0 = *(const float4 *)(turn.cos + at), c1 = *(const float4 *)(turn.cos + at + 4), s0 = *(const float4 *)(turn.sin + at), s1 = *(const float4 *)(turn.sin + at + 4);
            c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w, c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
            s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w, s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
        } else
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int64_t at = (int64_t)paged_axis_position(turn, to, j + e) * turn.table_pairs + j + e;
                c[e] = turn.cos[at], s[e] = turn.sin[at];
            }
        if (TANGLED) {
            float z[16];
#pragma unroll
            for (int e = 0; e < 8; e++) z[e] = p[e], z[8 + e] = r[e];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float f = z[2 * e], g = z[2 * e + 1];
                z[2 * e] = f * c[e] - g * s[e], z[2 * e + 1] = f * s[e] + g * c[e];
            }
#pragma unroll
            for (int e = 0; e < 8; e++) p[e] = z[e], r[e] = z[8 + e];
        } else
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float f = p[e], g = r[e];
                p[e] = f * c[e] - g * s[e], r[e] = f * s[e] + g * c[e];
            }
    }
    if (h < hq) {
        TX *o = q_out + ((int64_t)row * hq + h) * d;
        paged_store8(o + a, p);
        if (turned) paged_store8(o + b, r);
    } else {
        TP *o = (TP *)((char *)(h < heads ? kv.k : kv.v) + to.at + (h < heads ? h - hq : h - heads) * kv.head);
        paged_store8(o + a, p);
        if (turned) paged_store8(o + b, r);
    }
}

// The same a value or pair at a time, for rows that do not begin at multiples of 16 bytes and pairs that are no multiple of eight.  One workgroup a row.
template <typename TX, typename TP, bool TANGLED>
__global__ __launch_bounds__(256) void k_paged_append(const TX *q, int64_t q_st, int64_t q_sh, const TX *__restrict__ k, const TX *__restrict__ v,
                                                      int64_t kv_st, int64_t kv_sh, int hq, int hkv, int d, PagedTurn turn, PagedKv kv, PagedRows rows,
                                                      TX *q_out) { // (q_out may be q)
    const int row = blockIdx.x, tid = threadIdx.x;
    const PagedPlace place = paged_place(row, rows, kv, turn);
    if (place.at < 0) return;
    const int units = d / 2;
    for (int i = tid; i < (hq + hkv) * units; i += 256) {
        const int h = i / units, j = i % units, kh = h - hq;
        const bool is_q = h < hq;
        const TX *from = is_q ? q + row * q_st + h * q_sh : k + row * kv_st + kh * kv_sh;
        int a = 2 * j, b = 2 * j + 1; // behind the turned pairs: neighbours, as they are
        float c = 1.f, s = 0.f;
        if (j < turn.pairs) {
            if (!TANGLED) a = j, b = j + turn.pairs;
            const int64_t at = (int64_t)paged_axis_position(turn, place, j) * turn.table_pairs + j;
            c = turn.cos[at], s = turn.sin[at];
        }
        const float x = (float)from[a], y = (float)from[b];
        const float u = j < turn.pairs ? x * c - y * s : x, w = j < turn.pairs ? x * s + y * c : y;
        if (is_q) {
            TX *to = q_out + ((int64_t)row * hq + h) * d;
            to[a] = (TX)u, to[b] = (TX)w;
        } else {
            TP *to = (TP *)((char *)kv.k + place.at + kh * kv.head);
            to[a] = (TP)u, to[b] = (TP)w;
        }
    }
    for (int i = tid; i < hkv * d; i += 256) {
        const int h = i / d, e = i % d;
        ((TP *)((char *)kv.v + place.at + h * kv.head))[e] = (TP)v[row * kv_st + h * kv_sh + e];
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
    FH_REQUIRE(!q_dev || q_dev != q_out_dev || ((hq == 1 || q_sh == d) && (tokens <= 1 || q_st == (int64_t)hq * d)), "q with strides cannot be its own output");
    FH_REQUIRE(tokens < 1 << 24, "%d rows: a launch takes fewer than 2^24", tokens); // (of 256 threads each, 2^32 in all)
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
        turn.aligned = !(((uintptr_t)cos_dev | (uintptr_t)sin_dev) & 15) && table_pairs % 4 == 0;
    } else
        FH_REQUIRE(!positions_dev && !sections_host, "positions without tables");
    FH_REQUIRE(dev, "NULL device");
    if (!tokens || !seqs) return FH_OK;
    PagedGpu gpu;
    FH_TRY(gpu.enter(dev));
    const int size = dtype == FH_F32 ? 4 : 2, heads = q_dev ? hq : 0;
    auto odd = [&](const void *p, int64_t st, int64_t sh) { return ((uintptr_t)p | (uintptr_t)(st * size) | (uintptr_t)(sh * size)) & 15; };
    const bool eights = turn.pairs % 8 == 0 && !(q_dev && (odd(q_dev, q_st, q_sh) || odd(q_out_dev, 0, 0))) && !odd(k_dev, kv_st, kv_sh) && !odd(v_dev, kv_st, kv_sh);
    const int64_t units = (int64_t)(heads + hkv) * (turn.pairs / 8 + (d - 2 * turn.pairs) / 8) + (int64_t)hkv * (d / 8);
    const dim3 grid((unsigned)tokens, eights ? (unsigned)((units + 255) / 256) : 1u), block(256);
#define FH_PA(TX, TP)                                                                                                                              \
    do {                                                                                                                                           \
        const TX *q = (const TX *)q_dev, *k = (const TX *)k_dev, *v = (const TX *)v_dev;                                                           \
        if (eights)                                                                                                                                \
            (interleaved ? k_paged_append8<TX, TP, true> : k_paged_append8<TX, TP, false>)<<<grid, block, 0, dev->stream>>>(                       \
                q, k, v, heads, hkv, d, turn.pairs, starts_dev, lens_dev, seqs, table_cols, q_st, q_sh, kv_st, kv_sh, table_dev, tokens, kv, turn, \
                (TX *)q_out_dev);                                                                                                                  \
        else                                                                                                                                       \
            (interleaved ? k_paged_append<TX, TP, true> : k_paged_append<TX, TP, false>)<<<grid, block, 0, dev->stream>>>(                         \
                q, q_st, q_sh, k, v, kv_st, kv_sh, heads, hkv, d, turn, kv, rows, (TX *)q_out_dev);                                                \
    } while (0)
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
    FH_REQUIRE(q_dev != out_dev, "q cannot be the output"); // (a row may be read again after it was written)
    FH_REQUIRE((int64_t)seqs * hkv * ((hq / hkv + 15) / 16) * ((int64_t)table_cols * page_size) <= (int64_t)1 << 38,
               "%d sequences of %d heads and %d pages of %d positions: more than 2^38 in all", seqs, hkv, table_cols, page_size);
    FH_REQUIRE(scale >= 0x1p-60f && scale <= 0x1p60f, "scale %g", (double)scale);
    FH_REQUIRE(window >= 0 && max_new >= 0 && max_len >= 0, "window %d, max_new %d, max_len %d", window, max_new, max_len);
    FH_REQUIRE(dev, "NULL device");
    if (!tokens || !seqs || !max_new) return FH_OK;
    rows.max_new = max_new < tokens ? max_new : tokens;
    PagedGpu gpu;
    FH_TRY(gpu.enter(dev));
    const PagedCall call = {q_dev, out_dev, q_st, q_sh, kv, rows, scale, window < FH_PAGED_MAX ? window : FH_PAGED_MAX, hq, hkv, d};
    // A few rows behind a short cache: as single tokens, the rows' heads as columns (32 / 8 heads of 128, f16, us, 2 rows behind 300 positions 8.5, by the tiles of a
    // prompt 14.1; 4 behind 1000 of 8 sequences 16.3 / 25.3).  Longer caches are cut into parts for either, and the tiles' are joined sooner (4 rows
    // behind 2000 25.1 / 23.1, 65536 73.8 / 60.2).
    if (rows.max_new == 1 || ((int64_t)rows.max_new * (hq / hkv) <= 16 && fh_paged_step_whole(dev, kv_dtype, call, max_len)))
        return fh_paged_step(dev, dtype, kv_dtype, call, max_len);
    return fh_paged_prompt(dev, dtype, kv_dtype, call, max_len);
}
