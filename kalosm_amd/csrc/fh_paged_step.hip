// Attention of one new token of every sequence over its pages: softmax(scale q . K^T) . V for the query heads that share a KV
// head, every key and value read once.
//
// What it has to do is a stream of cache rows: 4 d flops a query head and key against 4 d bytes a KV head and key (16-bit
// pages), so the arithmetic goes to the matrix cores and has to stay out of the loads' way.  A wavefront takes tiles of 32
// positions (f32 pages: 16), 8 KB of K and 8 KB of V at head_dim 128, straight into registers; nothing goes through LDS.
//   scores  S^T (keys x heads) = K . Q^T    A: K rows as they were loaded (lane (n, g): key n of 16, values 8 g ..), B: Q^T
//   output  O^T (d x heads)   += V^T . P^T  B: the scores' accumulators, exponentiated, as they sit in the registers: slot (g, j)
//           of the product is key 4 g + j of the tile's first half (j < 4) or second.  A lane loads 16 bytes of the eight rows of
//           its slots, d = 8 n ..; operand e takes element e of each of them - row n of that product is d = 8 n + e - so the
//           transposition of V is 32 byte permutations a tile and no exchange between lanes.  A lane ends up with one head's
//           outputs d = 32 g .. 32 g + 31.
// Both halves of a tile (16 positions) lie in one page each: a page's address is scalar, a lane's offset within it constant.
// f32 pages use v_mfma_f32_16x16x4_f32 the same way, in full f32.  f32 rows over 16-bit pages: Q and P are taken as sums of
// 16-bit terms, two of f16 (22 bits; Q's rows brought to 2^14 first), three of bf16 (24 bits).  Weights of bf16 rows have two
// terms, which cost nothing here, weights of f16 rows one, 2^14 times what they are, so that those below 2^-24 of the largest count.
//
// The tiles of all (sequence, KV head) pairs are one line, cut into equal stretches, one a workgroup, whatever the lengths: a
// workgroup has the end of one pair, whole pairs, and the beginning of another.  Its wavefronts take a pair's tiles in turn,
// each with its own running maximum and sum, and are joined through LDS where the pair (or the stretch) ends.  What is not a
// whole pair goes to scratch memory, two places a workgroup, and whoever of the pair's workgroups counts itself in last adds
// them up, in their order: the same bits in every run.  Pairs of few tiles are a workgroup each, and nothing is joined.
// Measured (32 / 8 heads of 128; a copy: 4.6 TB/s): 1 sequence of 131072, bf16, 98 to 101 us, 5.3 to 5.5 TB/s; 64 of 8192, f32 rows over f16, 64 / 8 heads, 235 to 245 us, 5.5 to 5.7;
// 32 of 2048, f16, a pair a workgroup, 38 us, 4.5.  1 of 300, f32: 12 us, by eight workgroups, each through its
// products and requests one behind the other; the dense cache's kernel, over more compute units and with a second launch, takes 6.8.
#include "fh_paged.h"
#include <type_traits>

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float ps_rows_max(float a) { // over the four 16-lane rows of the wavefront
    const uint32_t u = __float_as_uint(a);
    auto s16 = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    a = fmaxf(__uint_as_float(s16[0]), __uint_as_float(s16[1]));
    const uint32_t w = __float_as_uint(a);
    auto s32 = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__uint_as_float(s32[0]), __uint_as_float(s32[1]));
}
__device__ __forceinline__ float ps_rows_sum(float a) {
    const uint32_t u = __float_as_uint(a);
    auto s16 = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    a = __uint_as_float(s16[0]) + __uint_as_float(s16[1]);
    const uint32_t w = __float_as_uint(a);
    auto s32 = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return __uint_as_float(s32[0]) + __uint_as_float(s32[1]);
}
__device__ __forceinline__ floatx4 ps_mfma(half8 a, half8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ floatx4 ps_mfma(bf8 a, bf8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ int ps_uniform(int a) { return __builtin_amdgcn_readfirstlane(a); }

__device__ __forceinline__ uint32_t ps_scan(uint32_t x) { // inclusive prefix sums over the lanes
#define PS_ADD(CTRL, ROWS) x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false)
    PS_ADD(0x111, 0xf); // within 16 lanes: from 1, 2, 4, 8 before
    PS_ADD(0x112, 0xf);
    PS_ADD(0x114, 0xf);
    PS_ADD(0x118, 0xf);
    PS_ADD(0x142, 0xa); // rows 1 and 3: the last lane of the row before
    PS_ADD(0x143, 0xc); // rows 2 and 3: lane 31
#undef PS_ADD
    return x;
}

template <typename TP> struct PsVec { typedef half8 type; };
template <> struct PsVec<fh_bf> { typedef bf8 type; };

// A pair's tiles: positions first * TK .. (first + tiles) * TK - 1, of which begin .. end - 1 are seen by one of its rows, the first of which has position p.
struct PsSpan {
    int row, rows, p, begin, end, first, tiles;
};
template <int TK> __device__ __forceinline__ PsSpan ps_span(const PagedSeq &s, int window) {
    PsSpan r;
    r.row = s.row, r.rows = s.rows, r.p = s.first;
    r.end = r.p + r.rows < s.len ? r.p + r.rows : s.len;
    r.end = r.end < 0 ? 0 : r.end;
    r.begin = window && r.p - window + 1 > 0 ? r.p - window + 1 : 0;
    r.begin = r.begin < r.end ? r.begin : r.end;
    r.first = r.begin / TK;
    r.tiles = (r.end + TK - 1) / TK - r.first;
    r.tiles = s.rows < 1 ? 0 : r.tiles < 1 ? 1 : r.tiles; // (a row that sees nothing has one tile, all masked: it writes zeros)
    return r;
}

// The arguments that the first requests need come first: they are in registers when the kernel starts.
//   blocks of up to 16 query heads a KV head; whole: a pair a workgroup; least: tiles a stretch has at least; place: floats of a part
template <typename TX, typename TP, int DP, int NWV>
__global__ __launch_bounds__(64 * NWV) void k_paged_step(const int *__restrict__ table, const int *__restrict__ lens, const int *__restrict__ starts, int cols, int shift,
                                                         int whole, int hkv, int blocks, int window, int pages, const char *__restrict__ k_pages,
                                                         const char *__restrict__ v_pages, int64_t page_stride, int64_t head_stride, int64_t slot_stride,
                                                         const TX *__restrict__ q, int64_t q_st, int64_t q_sh, int group, int d, float scale, int seqs, int tokens, int max_new, int least,
                                                         int place, float *__restrict__ sums, uint32_t *__restrict__ arrived, TX *__restrict__ out) {
    constexpr bool F32 = sizeof(TP) == 4, F16 = __is_same(TP, fh_half), MIXED = sizeof(TX) != sizeof(TP);
    constexpr int TK = F32 ? 16 : 32, HALVES = TK / 16;
    constexpr int QT = F32 ? 1 : !MIXED ? 1 : F16 ? 2 : 3, PT = F32 ? 1 : MIXED ? (F16 ? 2 : 3) : F16 ? 1 : 2; // terms
    constexpr int KL = DP * (int)sizeof(TP) / 64;                     // 16-byte pieces of a row of K in a lane
    constexpr int VB = DP * (int)sizeof(TP) / 16 < 16 ? 8 : 16, VL = DP * (int)sizeof(TP) / 16 / VB; // pieces of a row of V: their bytes, and how many
    constexpr int VE = VB / (int)sizeof(TP), NA = VL * VE;            // values of a piece; output tiles: d = 16 VE c + VE (4 g + i) + e
    constexpr int THREADS = 64 * NWV;
    typedef typename PsVec<TP>::type vec8;
    extern __shared__ __attribute__((aligned(16))) float ps_lds[];
    __shared__ float s_st[NWV * 16 * 2];
    __shared__ uint32_t s_last, s_bad[16];
    const int tid = threadIdx.x, wave = ps_uniform(tid >> 6), lane = tid & 63, n = lane & 15, g = lane >> 4;
    const PagedRows rows = {starts, lens, table, cols, seqs, tokens, max_new};
    const int H = hkv * blocks, page_mask = (1 << shift) - 1;

    // ---- this workgroup's stretch of the line: `step` tiles.  Places on the line are counted from the stretch's beginning.
    struct Cursor { // a pair on the line: sequence b, block hh of its query heads
        PsSpan s;
        int b, hh, kh, at;  // at: where it begins (below 0: in an earlier stretch)
        int from, to;       // tiles from .. to - 1 of the pair lie in the stretch
    };
    Cursor cur;
    int step = 0, stretch = 0; // stretch: its length where it is not the line's last
    int early_page[HALVES]; // of this wavefront's first tile, if that is tile `wave` of the sequence
    if (whole) {
        cur.b = ps_uniform((int)blockIdx.x / H), cur.hh = (int)blockIdx.x - cur.b * H, cur.at = 0;
#pragma unroll
        for (int h = 0; h < HALVES; h++) {
            const int col = (wave * TK + 16 * h) >> shift;
            early_page[h] = paged_scalar(table, (int64_t)cur.b * cols + (col < cols ? col : cols - 1));
        }
        cur.s = ps_span<TK>(paged_seq_scalar(rows, shift, cur.b), window);
        if (cur.s.tiles == 0) return;
        step = cur.s.tiles;
    } else {
        // Prefix sums over 64 sequences at a time; a sequence has fewer than 2^26 tiles.
        PsSpan mine = {};
        auto tiles_of = [&](int i) {
            if (i >= seqs) return 0u;
            mine = ps_span<TK>(paged_seq(rows, shift, i), window);
            return (uint32_t)mine.tiles;
        };
        uint32_t upto = ps_scan(tiles_of(lane)), here = ps_uniform(__builtin_amdgcn_readlane(upto, 63));
        int64_t total = here;
        for (int c = 64; c < seqs; c += 64) total += (uint32_t)__builtin_amdgcn_readlane(ps_scan(tiles_of(c + lane)), 63);
        total *= H;
        int64_t each = (total + gridDim.x - 1) / gridDim.x;
        each = each < least ? least : each;
        const int64_t lo = each * blockIdx.x;
        if (lo >= total) return;
        step = (int)(each < total - lo ? each : total - lo), stretch = (int)each;
        int64_t before = 0;
        int c = 0;
        if (seqs > 64) // (lo < total: it ends)
            for (;; c += 64) {
                upto = ps_scan(tiles_of(c + lane)), here = __builtin_amdgcn_readlane(upto, 63);
                if ((before + here) * H > lo) break;
                before += here;
            }
        const int in = __popcll(__ballot((before + upto) * H <= lo)); // sequences of these 64 that end before
        cur.b = ps_uniform(c + in);
        cur.s.row = __builtin_amdgcn_readlane(mine.row, in), cur.s.rows = __builtin_amdgcn_readlane(mine.rows, in), cur.s.p = __builtin_amdgcn_readlane(mine.p, in);
        cur.s.begin = __builtin_amdgcn_readlane(mine.begin, in), cur.s.end = __builtin_amdgcn_readlane(mine.end, in);
        cur.s.first = __builtin_amdgcn_readlane(mine.first, in), cur.s.tiles = __builtin_amdgcn_readlane(mine.tiles, in);
        const int64_t at = (before + (in ? (uint32_t)__builtin_amdgcn_readlane(upto, in - 1) : 0u)) * H - lo;
        cur.hh = (int)(-at / cur.s.tiles);
        cur.at = (int)(at + (int64_t)cur.hh * cur.s.tiles);
        early_page[0] = 0;
    }
    auto enter = [&](Cursor &c) { // the part of the pair that lies in the stretch
        c.from = c.at < 0 ? -c.at : 0;
        c.to = step - c.at < c.s.tiles ? step - c.at : c.s.tiles;
        c.kh = blocks == 1 ? c.hh : c.hh / blocks;
    };
    auto next_pair = [&](Cursor &c) { // false at the stretch's end
        if (c.at + c.s.tiles >= step) return false;
        c.at += c.s.tiles;
        if (++c.hh == H) {
            c.hh = 0;
            do c.s = ps_span<TK>(paged_seq_scalar(rows, shift, ++c.b), window);
            while (c.s.tiles == 0); // (the line goes on, so there is one)
        }
        enter(c);
        return true;
    };
    enter(cur);

    // ---- requests.  `ahead` is two tiles ahead of the products: the pages of its tile are asked for while the tile before is requested.
    u32x4 kr[HALVES][KL];
    typedef typename std::conditional<VB == 16, u32x4, u32x2>::type vpiece;
    vpiece vr[HALVES][4][VL]; // [half][row 4 g + j][piece]
    uint32_t k_off[KL], v_off[4], v_piece[VL];
    {
        const uint32_t slot = (uint32_t)slot_stride, row_bytes = (uint32_t)d * sizeof(TP);
#pragma unroll
        for (int s = 0; s < KL; s++) { // pieces behind the head's end: its first one again (Q is zero there)
            const uint32_t piece = 64 * s + 16 * g;
            k_off[s] = n * slot + (piece < row_bytes ? piece : 0);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) v_off[j] = (4 * g + j) * slot;
#pragma unroll
        for (int c = 0; c < VL; c++) {
            const uint32_t piece = 16 * VB * c + VB * n;
            v_piece[c] = piece < row_bytes ? piece : 0; // (outputs that are not stored)
        }
    }
    Cursor ahead = cur;
    int t = cur.from + wave; // tile of `ahead`
    bool more = true;
    int next_key = 0, next_kh = 0, next_page[HALVES]; // the tile whose pages have been asked for
    const char *kb[HALVES], *vb[HALVES];              // the tile that is requested,
    int key0 = 0;                                     // its first position
    uint32_t holes = 0;                               // and its halves without a page
    auto look_up = [&]() {
        while (more && t >= ahead.to) {
            more = next_pair(ahead);
            if (more) t = ahead.from + wave;
        }
        next_key = more ? (ahead.s.first + t) * TK : 0; // (behind the end: something that is there, and dropped)
        next_kh = ahead.kh;
#pragma unroll
        for (int h = 0; h < HALVES; h++) {
            const int col = (next_key + 16 * h) >> shift;
            next_page[h] = paged_scalar(table, (int64_t)ahead.b * cols + (col < cols ? col : cols - 1));
        }
        t += NWV;
    };
    auto move = [&]() {
        key0 = next_key, holes = 0;
#pragma unroll
        for (int h = 0; h < HALVES; h++) {
            int page = next_page[h];
            if ((unsigned)page >= (unsigned)pages) page = 0, holes |= 1u << h;
            const int64_t o = page * page_stride + next_kh * head_stride + ((key0 + 16 * h) & page_mask) * slot_stride;
            kb[h] = k_pages + o, vb[h] = v_pages + o;
        }
    };
    auto ask_k = [&]() {
#pragma unroll
        for (int h = 0; h < HALVES; h++)
#pragma unroll
            for (int s = 0; s < KL; s++) kr[h][s] = *(const u32x4 *)(kb[h] + k_off[s]);
    };
    auto ask_v = [&]() {
#pragma unroll
        for (int h = 0; h < HALVES; h++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int c = 0; c < VL; c++) vr[h][j][c] = *(const vpiece *)(vb[h] + (v_off[j] + v_piece[c]));
    };
    // A pair's columns are its rows' heads: column c of a sequence is head c % group of row c / group (one row: of head c).  Places 16 columns at a time.
    auto columns = [&](const Cursor &c) { // of this block
        const int n = c.s.rows * group - (c.hh - c.kh * blocks) * 16;
        return n < 16 ? n : 16;
    };
    auto row_of = [&](int column) { return max_new == 1 ? 0 : column / group; };
    // Q's values of a pair as they lie: lane (column n, g) has those of K's pieces; zeros for columns that there are not and behind the head's end
    constexpr int E = 16 / (int)sizeof(TP); // values of a piece
    TX rq[KL][E];
    auto ask_q = [&](const Cursor &c) {
        const int column = (c.hh - c.kh * blocks) * 16 + n, r = row_of(column);
        const TX *p = q + (c.s.row + r) * q_st + (c.kh * group + column - r * group) * q_sh;
        const bool there = n < columns(c);
#pragma unroll
        for (int s = 0; s < KL; s++) {
            const int at = 4 * E * s + E * g;
#pragma unroll
            for (int e = 0; e < E; e++) rq[s][e] = (TX)0.f;
            if (there && at < d) __builtin_memcpy(rq[s], p + at, sizeof(rq[s])); // (any address)
        }
    };
    ask_q(cur);
    if (whole && cur.s.first == 0 && wave < cur.s.tiles) {
        next_key = wave * TK, next_kh = cur.kh;
#pragma unroll
        for (int h = 0; h < HALVES; h++) next_page[h] = early_page[h];
        t += NWV;
    } else
        look_up();
    move();
    ask_k();
    ask_v();
    look_up();

    // ---- pair after pair
    bool go = true;
    while (go) {
        const int skip = (cur.hh - cur.kh * blocks) * 16, heads = columns(cur); // (columns `skip` and up)
        // what this lane's column sees, and what all of them see
        const int my_p = cur.s.p + (row_of(skip + n) < cur.s.rows ? row_of(skip + n) : cur.s.rows - 1), last_p = cur.s.p + cur.s.rows - 1;
        const int high = my_p < cur.s.end - 1 ? my_p : cur.s.end - 1, low = window && my_p - window + 1 > 0 ? my_p - window + 1 : 0;
        const int all_high = cur.s.p < cur.s.end - 1 ? cur.s.p : cur.s.end - 1, all_low = window && last_p - window + 1 > 0 ? last_p - window + 1 : 0;
        vec8 qf[QT][F32 ? 1 : KL];
        floatx4 qx[F32 ? KL : 1];
        float sc2 = scale * 1.4426950408889634f; // scores in the log2 domain
        {
            float x[KL][E], most = 0.f;
#pragma unroll
            for (int s = 0; s < KL; s++)
#pragma unroll
                for (int e = 0; e < E; e++) {
                    x[s][e] = (float)rq[s][e];
                    most = fmaxf(most, fabsf(x[s][e]));
                }
            if constexpr (MIXED && F16) { // brought to 2^14 .. 2^15
                most = ps_rows_max(most);
                int ex = 0;
                if (most > 0.f && most < INFINITY) ex = 15 - __builtin_amdgcn_frexp_expf(most);
                sc2 = paged_brought(sc2, ex);
#pragma unroll
                for (int s = 0; s < KL; s++)
#pragma unroll
                    for (int e = 0; e < E; e++) x[s][e] = ldexpf(x[s][e], ex);
            }
#pragma unroll
            for (int s = 0; s < KL; s++) {
                if constexpr (F32) qx[s] = floatx4{x[s][0], x[s][1], x[s][2], x[s][3]};
                else
#pragma unroll
                    for (int u = 0; u < QT; u++)
#pragma unroll
                        for (int e = 0; e < E; e++) {
                            const TP v = u == 0 && QT > 1 ? paged_first<TP>(x[s][e]) : (TP)x[s][e];
                            qf[u][s][e] = v;
                            x[s][e] -= (float)v;
                        }
            }
        }
        float m_run = -INFINITY, l_run = 0.f;
        floatx4 acc[NA];
#pragma unroll
        for (int e = 0; e < NA; e++) acc[e] = floatx4{0.f, 0.f, 0.f, 0.f};

        for (int u = cur.from + wave; u < cur.to; u += NWV) {
            const int first = key0;
            const uint32_t hole = holes;
            floatx4 st[HALVES];
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                floatx4 other = {0.f, 0.f, 0.f, 0.f}; // (two chains: a product of f32 takes 32 cycles)
                st[h] = other;
#pragma unroll
                for (int s = 0; s < KL; s++) {
                    if constexpr (F32) {
                        const floatx4 kx = __builtin_bit_cast(floatx4, kr[h][s]);
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            st[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[e], qx[s][e], st[h], 0, 0, 0);
                            other = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[e + 1], qx[s][e + 1], other, 0, 0, 0);
                        }
                    } else
#pragma unroll
                        for (int w = QT - 1; w >= 0; w--) st[h] = ps_mfma(__builtin_bit_cast(vec8, kr[h][s]), qf[w][s], st[h]);
                }
                if constexpr (F32) st[h] += other;
            }
            move();
            __builtin_amdgcn_sched_barrier(0);
            ask_k();
            look_up();
            __builtin_amdgcn_sched_barrier(0);
            // ---- positions that are not seen: scores -inf, values 0 (they may be anything)
            const bool edge = first < all_low || first + TK - 1 > all_high || hole;
            if (edge) {
#pragma unroll
                for (int h = 0; h < HALVES; h++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int key = first + 16 * h + 4 * g + i;
                        const bool there = !(hole >> h & 1), seen = key >= cur.s.begin && key < cur.s.end && there;
                        st[h][i] = key >= low && key <= high && there ? st[h][i] : -INFINITY;
#pragma unroll
                        for (int c = 0; c < VL; c++)
#pragma unroll
                            for (int w = 0; w < VB / 4; w++) vr[h][i][c][w] = seen ? vr[h][i][c][w] : 0u;
                    }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int h = 0; h < HALVES; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) mx = fmaxf(mx, st[h][i]);
            mx = ps_rows_max(mx) * sc2;
            const float m_new = fmaxf(m_run, mx);
            const float ref = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = __builtin_amdgcn_exp2f(m_run - ref);
            const float sub = F16 ? 14.f - ref : -ref;
            float p[HALVES][4], ps = 0.f;
#pragma unroll
            for (int h = 0; h < HALVES; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) p[h][i] = F32 ? st[h][i] * sc2 + sub : fmaf(st[h][i], sc2, sub);
            // Scores rounded as the maximum was, as those of f32 pages always are.
            if (!F32 && __any(fabsf(ref) >= PAGED_FAR))
#pragma unroll
                for (int h = 0; h < HALVES; h++)
#pragma unroll
                    for (int i = 0; i < 4; i++) p[h][i] = st[h][i] * sc2 - ref + (F16 ? 14.f : 0.f);
#pragma unroll
            for (int h = 0; h < HALVES; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    p[h][i] = __builtin_amdgcn_exp2f(p[h][i]);
                    ps += p[h][i];
                }
            l_run = l_run * alpha + ps; // of this lane's keys: the four rows of a column are added at the end
            m_run = m_new;
            if (__any(alpha != 1.f)) {
#pragma unroll
                for (int e = 0; e < NA; e++) acc[e] *= alpha;
            }
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int c = 0; c < VL; c++) {
                        const floatx4 vx = __builtin_bit_cast(floatx4, vr[0][i][c]);
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[c * VE + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vx[e], p[0][i], acc[c * VE + e], 0, 0, 0);
                    }
            } else {
                vec8 pb[PT];
#pragma unroll
                for (int w = 0; w < PT; w++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const TP x = (TP)p[j >> 2][j & 3];
                        pb[w][j] = x;
                        p[j >> 2][j & 3] -= (float)x;
                    }
#pragma unroll
                for (int c = 0; c < VL; c++)
#pragma unroll
                    for (int e = 0; e < VE; e++) { // element e of the eight rows
                        u32x4 x;
                        const uint32_t pick = e & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            x[j] = __builtin_amdgcn_perm(vr[j >> 1][2 * (j & 1) + 1][c][e >> 1], vr[j >> 1][2 * (j & 1)][c][e >> 1], pick);
#pragma unroll
                        for (int w = PT - 1; w >= 0; w--) acc[c * VE + e] = ps_mfma(__builtin_bit_cast(vec8, x), pb[w], acc[c * VE + e]);
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
            ask_v();
            __builtin_amdgcn_sched_barrier(0);
        }

        // ---- the wavefronts' results together: thread (head, four values); the next pair's Q is on its way
        Cursor next = cur;
        go = next_pair(next);
        if (go && !MIXED) ask_q(next); // (f32 rows over 16-bit pages: behind the merge, for want of registers)
        l_run = ps_rows_sum(l_run);
        if (n < heads) {
            float *to = ps_lds + (wave * heads + n) * DP;
#pragma unroll
            for (int c = 0; c < VL; c++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < VE; e += 4)
                        *(floatx4 *)(to + 16 * VE * c + VE * (4 * g + i) + e) =
                            floatx4{acc[c * VE + e][i], acc[c * VE + e + 1][i], acc[c * VE + e + 2][i], acc[c * VE + e + 3][i]};
            if (g == 0) s_st[(wave * 16 + n) * 2] = m_run, s_st[(wave * 16 + n) * 2 + 1] = l_run;
        }
        if (tid < 16) s_bad[tid] = 0;
        __syncthreads();
        const bool all = cur.from == 0 && cur.to == cur.s.tiles;
        constexpr int PITCH = DP + 4, QUADS = DP / 4; // PITCH: of a part's head: values, maximum, sum
        float *own = sums + ((int64_t)blockIdx.x * 2 + (cur.from ? 0 : 1)) * place;
        auto put = [&](float *p, float x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        auto get = [&](const float *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        auto place_of = [&](int h) { // of column h in `out`
            const int r = row_of(skip + h);
            return ((int64_t)(cur.s.row + r) * hkv * group + cur.kh * group + skip + h - r * group) * d;
        };
        auto store = [&](int h, int at, floatx4 x, float den) {
            if (at >= d) return;
            const float inv = den == 0.f ? 0.f : 1.f / den; // (a row that sees nothing: zeros)
            TX y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = (TX)(x[i] * inv);
            __builtin_memcpy(out + place_of(h) + at, y, sizeof(y));
        };
        for (int i = tid; i < heads * QUADS; i += THREADS) {
            const int h = i / QUADS, at = i % QUADS * 4;
            float mx = -INFINITY, den = 0.f;
#pragma unroll
            for (int w = 0; w < NWV; w++) mx = fmaxf(mx, s_st[(w * 16 + h) * 2]);
            const float ref = mx == -INFINITY ? 0.f : mx;
            floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NWV; w++) {
                const float f = __builtin_amdgcn_exp2f(s_st[(w * 16 + h) * 2] - ref);
                x += *(const floatx4 *)(ps_lds + (w * heads + h) * DP + at) * f;
                den = fmaf(s_st[(w * 16 + h) * 2 + 1], f, den);
            }
            if (max_new > 1 && !(0.f * x[0] + 0.f * x[1] + 0.f * x[2] + 0.f * x[3] + 0.f * den == 0.f)) s_bad[h] = 1;
            if (all) store(h, at, x, den);
            else {
#pragma unroll
                for (int e = 0; e < 4; e++) put(own + h * PITCH + at + e, x[e]);
                if (at == 0) put(own + h * PITCH + DP, mx), put(own + h * PITCH + DP + 1, den);
            }
        }
        if (max_new > 1) { // several rows, and so a whole pair (of one row: what it does not see was set to zeros)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // what was stored before
            __syncthreads();
            for (int h = wave; h < heads; h += NWV)
                if (s_bad[h]) {
                    const int r = row_of(skip + h), p = cur.s.p + r;
                    const PagedKv kv = {k_pages, v_pages, page_stride, head_stride, slot_stride, pages, shift};
                    float m, l, o[4];
                    paged_again<TX, TP>(q + (cur.s.row + r) * q_st + (cur.kh * group + skip + h - r * group) * q_sh, d, scale * 1.4426950408889634f, F16 ? 14.f : 0.f, kv,
                                        table + (int64_t)cur.b * cols, cur.kh, window && p - window + 1 > 0 ? p - window + 1 : 0, p < cur.s.end - 1 ? p : cur.s.end - 1, m, l, o);
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    for (int e = 0; e < 4; e++)
                        if (lane + 64 * e < d) out[place_of(h) + lane + 64 * e] = (TX)(o[e] * inv);
                }
        }
        if (!all) {
            // the pair's workgroups (all stretches before the line's last are as long as this one, or this is the last)
            const int w0 = (int)blockIdx.x - (cur.from ? (cur.from + stretch - 1) / stretch : 0);
            const int parts = (int)blockIdx.x - w0 + 1 + (cur.s.tiles - cur.to + stretch - 1) / stretch;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // written before this workgroup counts itself in
            __syncthreads();
            if (tid == 0) s_last = __hip_atomic_fetch_add(arrived + w0, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            if (s_last == (uint32_t)parts - 1) {
                if (tid == 0) __hip_atomic_store(arrived + w0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); // as it was found
                auto part = [&](int i) { return sums + ((int64_t)(w0 + i) * 2 + (i ? 0 : 1)) * place; };
                float *s_w = ps_lds, *s_l = ps_lds + parts * heads; // [head][part]: maxima, then weights; sums
                // Groups of threads take parts in turn, the first EARLY of each along with the statistics.
                const int items = heads * QUADS, groups = items < THREADS ? THREADS / items : 1, pg = groups > 1 ? tid / items : 0;
                constexpr int EARLY = MIXED ? 4 : 8;
                floatx4 first[EARLY];
                auto ask = [&](int i, int k) {
                    const float *p = part(k) + i / QUADS * PITCH + i % QUADS * 4;
                    return floatx4{get(p), get(p + 1), get(p + 2), get(p + 3)};
                };
                {
                    const int i = groups > 1 ? tid % items : tid;
#pragma unroll
                    for (int k = 0; k < EARLY; k++)
                        if (pg + k * groups < parts && i < items && pg < groups) first[k] = ask(i, pg + k * groups);
                }
                for (int i = tid; i < parts * heads; i += THREADS) {
                    const float *p = part(i % parts) + i / parts * PITCH + DP;
                    s_w[i] = get(p), s_l[i] = get(p + 1);
                }
                __syncthreads();
                for (int h = wave; h < heads; h += NWV) { // a wavefront a head
                    float mx = -INFINITY, sum = 0.f;
                    for (int i = lane; i < parts; i += 64) mx = fmaxf(mx, s_w[h * parts + i]);
#pragma unroll
                    for (int w = 32; w; w >>= 1) mx = fmaxf(mx, __shfl_xor(mx, w));
                    const float ref = mx == -INFINITY ? 0.f : mx;
                    for (int i = lane; i < parts; i += 64) {
                        const float f = __builtin_amdgcn_exp2f(s_w[h * parts + i] - ref);
                        s_w[h * parts + i] = f;
                        sum = fmaf(s_l[h * parts + i], f, sum);
                    }
#pragma unroll
                    for (int w = 32; w; w >>= 1) sum += __shfl_xor(sum, w);
                    if (lane == 0) s_st[h] = sum;
                }
                __syncthreads();
                float *s_x = ps_lds + 2 * parts * heads + (2 * parts * heads & 2 ? 2 : 0); // (16-byte places)
                for (int base = 0; base < items; base += THREADS) {
                    const int i = base + (groups > 1 ? tid % items : tid);
                    floatx4 x = {0.f, 0.f, 0.f, 0.f};
                    if (i < items && pg < groups) {
                        const float *w = s_w + i / QUADS * parts;
#pragma unroll
                        for (int k = 0; k < EARLY; k++)
                            if (pg + k * groups < parts) x += (base ? ask(i, pg + k * groups) : first[k]) * w[pg + k * groups];
#pragma unroll 8
                        for (int k = pg + EARLY * groups; k < parts; k += groups) x += ask(i, k) * w[k];
                    }
                    if (groups > 1) {
                        if (pg < groups) *(floatx4 *)(s_x + (pg * items + i) * 4) = x;
                        __syncthreads();
                        if (pg == 0)
                            for (int k = 1; k < groups; k++) x += *(const floatx4 *)(s_x + (k * items + i) * 4);
                    }
                    if (i < items && pg == 0) store(i / QUADS, i % QUADS * 4, x, s_st[i / QUADS]);
                }
            }
        }
        __syncthreads(); // the next pair's results go to the same places
        if (go && MIXED) ask_q(next);
        cur = next;
    }
}

template <typename TX, typename TP, int DP, int NWV>
static fh_status ps_launch(fh_device *dev, const PagedCall &call, int whole) {
    const int group = call.hq / call.hkv, wide = call.rows.max_new * group, heads = wide < 16 ? wide : 16;
    const int blocks = (wide + 15) / 16, place = heads * (DP + 4);
    unsigned grid = (unsigned)((int64_t)call.rows.seqs * call.hkv * blocks);
    if (!whole) {
        grid = (unsigned)dev->compute_units;
        FH_TRY(fh_dev_scratch(dev, (void **)&dev->part_buf, &dev->part_cap, (size_t)grid * 2 * place * 4));
    }
    // results of the wavefronts; where parts are joined, two words a part and head and 16 bytes a thread
    size_t lds = (size_t)NWV * heads * DP * 4;
    const size_t join = (size_t)grid * heads * 8 + 16 + 64 * NWV * 16;
    if (!whole && lds < join) lds = join;
    const auto kern = k_paged_step<TX, TP, DP, NWV>;
    FH_TRY(fh_kernel_lds(dev, (const void *)kern, lds));
    kern<<<dim3(grid), dim3(64 * NWV), lds, dev->stream>>>(call.rows.table, call.rows.lens, call.rows.starts, call.rows.cols, call.kv.shift, whole, call.hkv, blocks, call.window,
                                                           call.kv.pages, call.kv.k, call.kv.v, call.kv.page, call.kv.head, call.kv.slot, (const TX *)call.q, call.q_st, call.q_sh,
                                                           group, call.d, call.scale, call.rows.seqs, call.rows.tokens, call.rows.max_new, NWV, place, dev->part_buf, dev->arrived, (TX *)call.out);
    FH_HIP(hipGetLastError());
    return FH_OK;
}
// A pair a workgroup of four wavefronts (two of them a compute unit), or the line's stretches of eight.  Few tiles are not worth the join; with a pair for every
// compute unit there is less to balance (32 / 8 heads of 128, f16, us, a pair / stretches: 1 sequence of 700 positions 11.3 / 17.5, 2000 22.8 / 16.6; 16 of 1500
// 20.7 / 24.0, 2000 28.5 / 25.8; 32 of 2048 38.1 / 41.7, 4096 70.8 / 70.1).  Pairs by eight wavefronts: 64 sequences of 100 12.7 / 8.5, 1 of 1000 14.6 / 13.6;
// stretches of four, two a compute unit: 1 of 131072 102 / 115.
bool fh_paged_step_whole(const fh_device *dev, int kv_dtype, const PagedCall &call, int max_len) {
    const int TK = kv_dtype == FH_F32 ? 16 : 32, wide = call.rows.max_new * (call.hq / call.hkv);
    int64_t longest = (int64_t)call.rows.cols << call.kv.shift;
    if (max_len > 0 && max_len < longest) longest = max_len;
    const int64_t most = (int64_t)call.window + call.rows.max_new + TK;
    if (call.window > 0 && most < longest) longest = most;
    const int64_t tiles = (longest + TK - 1) / TK * (call.d > 128 ? 2 : 1), pairs = (int64_t)call.rows.seqs * call.hkv * ((wide + 15) / 16);
    if (pairs >= 1 << 24) return false; // (workgroups of 256 threads: fewer than 2^32 in all)
    return tiles <= 32 || (tiles <= 48 && 2 * pairs >= dev->compute_units) || (tiles <= 64 && pairs >= dev->compute_units);
}
template <typename TX, typename TP>
static fh_status ps_dim(fh_device *dev, const PagedCall &call, bool whole) {
    if (call.d > 128) return ps_launch<TX, TP, 256, 4>(dev, call, whole);
    if (call.d > 64) return whole ? ps_launch<TX, TP, 128, 4>(dev, call, true) : ps_launch<TX, TP, 128, 8>(dev, call, false);
    return whole ? ps_launch<TX, TP, 64, 4>(dev, call, true) : ps_launch<TX, TP, 64, 8>(dev, call, false);
}
fh_status fh_paged_step(fh_device *dev, int dtype, int kv_dtype, const PagedCall &call, int max_len) {
    const bool whole = fh_paged_step_whole(dev, kv_dtype, call, max_len);
    if (dtype == FH_F16) return ps_dim<fh_half, fh_half>(dev, call, whole);
    if (dtype == FH_PAGED_BF16) return ps_dim<fh_bf, fh_bf>(dev, call, whole);
    if (kv_dtype == FH_F32) return ps_dim<float, float>(dev, call, whole);
    if (kv_dtype == FH_F16) return ps_dim<float, fh_half>(dev, call, whole);
    return ps_dim<float, fh_bf>(dev, call, whole);
}
