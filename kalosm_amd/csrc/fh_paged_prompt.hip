// Attention of several new tokens of every sequence over its pages (a prompt, or a part of one behind a filled cache), causal.
//
// 4 d flops a query head and key: bound by the matrix cores and the softmax between the two products.  The query heads of a KV head are
// rows of one tile: row r of a sequence is token r / group, head r % group, so a tile of 128 rows reads K and V once for 128 / group
// tokens of all heads, few tokens fill a tile as well as many, and the causal edge is 128 / group tokens wide.
// As in fh_attention_prefill.hip both products are computed transposed, S^T = K . Q^T and O^T = V^T . P^T, with 32 x 32 x 16 products:
// a lane stands for one query, the statistics are its own, and P^T is the second product's operand as it sits in the registers.
// A page's 16 positions are one scalar address: requests add a lane's constant offset.
// grid (KV heads, blocks of rows - the last, longest ones first -, sequences x parts).  With fewer workgroups than compute units the
// positions are split over `parts` workgroups, whose sums go to scratch memory in f32 and are added up by a second launch.
// Measured (32 / 8 heads of 128): 8192 tokens of f16 605 to 651 us by the card, 845 to 910 TFLOP/s, the matrix cores busy 45 % of the cycles; 8 sequences of
// 184 to 512 behind up to 4001, bf16, 174 to 185 us, 715 to 760; 33 behind 65536, f16, 90 us, 3.0 TB/s (a workgroup has one step of 64 KB on its way, which takes 2.3 us
// whatever the number of rows).  2 x 2049, window 1024, 16 / 4 heads of 64, f32: 104 us, 110 TFLOP/s.
//
// Positions that a row does not see have weight 0, whatever lies there: scores are replaced, and where a row's sums end up infinite or NaN and a position in its
// tiles that some row does not see has an infinity or a NaN - 0 times that is NaN - the row is worked out again in f32 over what it sees (pp_mend): one at a
// time by a wavefront, until nothing of it can be finite.  (Looked for in the tiles as they come, by the sums before and behind them, 8192 tokens take 660 us for 626.)
#include "fh_attention_tiles.h"
#include "fh_paged.h"
#include <type_traits>

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct PpVec { typedef half8 type; };
template <> struct PpVec<fh_bf> { typedef bf8 type; };
__device__ __forceinline__ floatx16 pp_mfma(half8 a, half8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ floatx16 pp_mfma(bf8 a, bf8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

enum { PP_PARTS = 256 }; // at most
// m_run, what the exponents of a row are taken relative to, moves where a tile's maximum is further than this ahead of it (in the log2 domain), each row's by
// its own scores: mostly in the first tiles.  (With every new maximum some row of a wavefront's 32 moves in more than half of a long row's tiles, and all sums
// with it: 8 prompts of 184 to 512 rows, bf16, 184 us for 176, 8192 rows of f16 610 for 605.)  Weights of f16 are 2^14 times what they are next to m_run,
// so that the small ones count: 2^15.5 is what they can take.
template <bool F16> constexpr float pp_ahead = F16 ? 1.5f : 8.f;
struct PpArgs {
    PagedCall c;
    int parts, sorted; // sorted: the longest sequences first
    float *sums, *stats; // [part][row][head][d], [part][row][head][maximum, sum]
};

// The sequence that the z-th place of the grid has: with more workgroups than run at once, and up to 64 sequences, the z-th longest, so that the short ones
// fill what the long ones leave (8 sequences of 1.4 to 4.5 thousand positions, 184 to 512 new ones, bf16, 32 / 8 heads of 128: 202 us as they come, 188 so).
__device__ __forceinline__ int pp_sequence(const PpArgs &a, int z) {
    const int n = a.c.rows.seqs, lane = threadIdx.x & 63;
    if (!a.sorted || n == 1 || n > 64) return z;
    const int len = lane < n ? a.c.rows.lens[lane] : 0;
    int rank = lane < n ? 0 : 64;
    for (int j = 0; j < n; j++) {
        const int other = __builtin_amdgcn_readlane(len, j);
        rank += other > len || (other == len && j < lane);
    }
    return __builtin_amdgcn_readfirstlane(__ffsll(__ballot(rank == z)) - 1);
}

// A lane's query and what it sees: positions low .. high, if any.
struct PpRow {
    int token, head, low, high;
};
__device__ __forceinline__ PpRow pp_row(const PagedSeq &s, int r, int group, int window) {
    PpRow x;
    const int token = r / group;
    x.head = r - token * group;
    x.token = token < s.rows ? token : s.rows - 1; // (rows behind the last are computed and not stored)
    const int p = s.first + x.token;
    x.high = p < s.len - 1 ? p : s.len - 1;
    x.low = window && p - window + 1 > 0 ? p - window + 1 : 0;
    return x;
}
// The positions that the rows of a block see, from a multiple of 64 on, cut into steps of STEP for `parts` workgroups.
struct PpSpan {
    int base, end, steps; // of this part
};
template <int STEP> __device__ __forceinline__ PpSpan pp_span(const PagedSeq &s, int r0, int r1, int group, int window, int part, int parts) {
    const int t0 = r0 / group, t1 = r1 / group < s.rows ? r1 / group : s.rows - 1;
    int end = s.first + t1 + 1, from = window ? s.first + t0 - window + 1 : 0;
    end = end < s.len ? end : s.len;
    from = from > 0 ? from & ~63 : 0;
    const int steps = end > from ? (end - from + STEP - 1) / STEP : 0;
    const int a = (int)((int64_t)steps * part / parts), b = (int)((int64_t)steps * (part + 1) / parts);
    return PpSpan{from + a * STEP, end, b - a};
}

// A part's sums, or the result where there is one part.
template <typename TX, int D>
__device__ __forceinline__ void pp_store(const PpArgs &a, int part, const PagedSeq &s, const PpRow &x, int kh, int group, int g, float m, float l, const floatx16 (&acc)[D / 32]) {
    const int64_t row = (int64_t)(s.row + x.token) * a.c.hq + kh * group + x.head;
    auto put = [&](auto *to, float f) {
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
            for (int r4 = 0; r4 < 4; r4++)
                if (32 * dt + 8 * r4 + 4 * g < a.c.d)
                    ap_store4(to + 32 * dt + 8 * r4 + 4 * g, acc[dt][4 * r4] * f, acc[dt][4 * r4 + 1] * f, acc[dt][4 * r4 + 2] * f, acc[dt][4 * r4 + 3] * f);
    };
    if (a.parts == 1) put((TX *)a.c.out + row * a.c.d, l == 0.f ? 0.f : 1.f / l); // (a row that sees nothing: zeros)
    else {
        const int64_t at = (int64_t)part * a.c.rows.tokens * a.c.hq + row;
        put(a.sums + at * a.c.d, 1.f);
        if (g == 0) a.stats[2 * at] = m, a.stats[2 * at + 1] = l;
    }
}

// Row r of a sequence again, positions from .. to of those that it sees.
template <typename TX, typename TP>
__device__ __forceinline__ void pp_again(const PpArgs &a, int part, int seq, const PagedSeq &s, int r, int kh, int group, int from, int to) {
    const int lane = threadIdx.x & 63, d = a.c.d;
    const PpRow x = pp_row(s, r, group, a.c.window);
    const TX *q = (const TX *)a.c.q + (s.row + x.token) * a.c.q_st + (kh * group + x.head) * a.c.q_sh;
    float m, l, o[4];
    paged_again<TX, TP>(q, d, a.c.scale * 1.4426950408889634f, __is_same(TP, fh_half) ? 14.f : 0.f, a.c.kv, a.c.rows.table + (int64_t)seq * a.c.rows.cols, kh,
                        from > x.low ? from : x.low, to < x.high ? to : x.high, m, l, o);
    const int64_t row = (int64_t)(s.row + x.token) * a.c.hq + kh * group + x.head, where = (int64_t)part * a.c.rows.tokens * a.c.hq + row;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int e = 0; e < 4; e++)
        if (lane + 64 * e < d) {
            if (a.parts == 1) ((TX *)a.c.out)[row * d + lane + 64 * e] = (TX)(o[e] * inv);
            else a.sums[where * d + lane + 64 * e] = o[e];
        }
    if (a.parts > 1 && lane == 0) a.stats[2 * where] = m, a.stats[2 * where + 1] = l;
}
// The rows of a wavefront, first .. first + 31 of the sequence's `rows`, whose sums are not finite, again, where positions from .. to have an infinity or a NaN
// among the values that not all of them see.
template <typename TX, typename TP, int D>
__device__ __forceinline__ void pp_mend(const PpArgs &a, int part, int seq, const PagedSeq &s, const PpRow &x, int first, int rows, int kh, int group, int from, int to, bool holed,
                                        float l, const floatx16 (&acc)[D / 32]) {
    float sum = 0.f * l; // (of 0 times everything)
#pragma unroll
    for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
        for (int r = 0; r < 16; r++) sum = fmaf(0.f, acc[dt][r], sum);
    uint64_t bad = __ballot(!(sum == 0.f));
    bad = (bad | bad >> 32) & 0xFFFFFFFFu;
    if (!bad) return;
    // what lies behind the first row's end, and in front of the last one's beginning
    const PagedKv &kv = a.c.kv;
    const int lane = threadIdx.x & 63, pieces = a.c.d * (int)sizeof(TP) / 16;
    int high = x.high, low = x.low;
    for (int w = 32; w; w >>= 1) {
        const int h = __shfl_xor(high, w), y = __shfl_xor(low, w);
        high = h < high ? h : high, low = y > low ? y : low;
    }
    to = to < s.len - 1 ? to : s.len - 1;
    const int begin = high + 1 > from ? high + 1 : from, behind = to >= begin ? to - begin + 1 : 0, ahead = low <= to ? (low > from ? low - from : 0) : to - from + 1;
    bool wild = holed; // (what was read for a hole may be anything)
    for (int i = lane; i < (behind + ahead) * pieces; i += 64) {
        const int n = i / pieces, p = n < behind ? begin + n : from + n - behind, page = a.c.rows.table[(int64_t)seq * a.c.rows.cols + (p >> kv.shift)];
        if ((unsigned)page >= (unsigned)kv.pages) wild = true;
        else {
            const uint4 w = *(const uint4 *)(kv.v + page * kv.page + kh * kv.head + (p & ((1 << kv.shift) - 1)) * kv.slot + (i - n * pieces) * 16);
            TP v[16 / sizeof(TP)];
            __builtin_memcpy(v, &w, 16);
            for (int e = 0; e < 16 / (int)sizeof(TP); e++) wild |= !(0.f * (float)v[e] == 0.f);
        }
    }
    if (!__any(wild)) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // what was stored before
    for (int i = 0; i < 32; i++)
        if (bad >> i & 1 && first + i < rows) pp_again<TX, TP>(a, part, seq, s, first + i, kh, group, from, to);
}

// ---------------------------------------------------------------- rows and pages of one 16-bit type, head_dim up to 128 (in tiles of 64 or 128 values)
// k_attn_ahead's loop (fh_attention_prefill.hip): the scores of the next tile beside the softmax of this one, K a tile ahead of V, both straight
// into LDS with their 16-byte pieces swapped on the memory side.
template <typename T, int D, int KS>
__global__ __launch_bounds__(256 * KS) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_paged_tiles(PpArgs a) {
    constexpr int QW = 4, NB = 2; // wavefronts of rows; buffers: step `it` asks for K of step it + NB and V of step it + NB - 1
    constexpr int BN = 64, DT = D / 32, KSTEPS = D / 16, CH = D / 8, TILE = BN * D, NW = QW * KS, NP = TILE * KS * 2 / 1024 / NW; // NP: 1 KB pieces of K a wavefront
    constexpr bool F16 = __is_same(T, fh_half);
    typedef typename PpVec<T>::type vec8;
    extern __shared__ __attribute__((aligned(16))) fh_half pp_lds[]; // [NB buffers][KS tiles of K, KS of V]
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, li = lane & 31, g = lane >> 5;
    const int kset = KS == 2 ? wave / QW : 0;
    const PagedKv &kv = a.c.kv;
    const PagedRows &rows = a.c.rows;
    const int kh = blockIdx.x, group = a.c.hq / a.c.hkv, seq = pp_sequence(a, (int)blockIdx.z / a.parts), part = (int)blockIdx.z % a.parts;
    const PagedSeq s = paged_seq_scalar(rows, kv.shift, seq);
    const int r0 = (int)(gridDim.y - 1 - blockIdx.y) * 32 * QW;
    if (r0 >= s.rows * group) return;
    const PpSpan span = pp_span<KS * BN>(s, r0, r0 + 32 * QW - 1, group, a.c.window, part, a.parts);
    const int steps = span.steps;
    const bool alive = r0 + (wave % QW) * 32 < s.rows * group; // (wavefronts without a row bring tiles and keep the barriers)
    const int r = r0 + (wave % QW) * 32 + li;
    const PpRow x = pp_row(s, r, group, a.c.window);

    // Piece i of this wavefront: rows row + i RSTEP of a step's KS tiles, within 16 positions of one page; a lane brings 16 bytes of a row.
    constexpr int RSTEP = NW * 64 / CH;
    static_assert(RSTEP % 16 == 0 && 64 / CH <= 16, "the same swap in all of a lane's rows, one page a piece");
    const int row = (wave * 64 + lane) / CH, piece = lane % CH, slot = (int)kv.slot;
    // (pieces behind the head's end: its first one again.  Q is zero there, and V's outputs are not stored)
    auto in_head = [&](int c) { return c < a.c.d * 2 ? c : 0; };
    const int kc = in_head((piece ^ (D == 128 ? row & 15 : (row >> 1) & 7)) * 16), vc = in_head((piece ^ (D == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2)) * 16);
    const int last16 = (s.len - 1) & ~15; // the last 16 positions there are
    auto begin16 = [&](int it, int i) __attribute__((always_inline)) {
        const int p = span.base + it * KS * BN + ((i * RSTEP + wave * (64 / CH)) & ~15);
        return p < last16 ? p : last16;
    };
    auto column = [&](int p) __attribute__((always_inline)) { return paged_scalar(rows.table, (int64_t)seq * rows.cols + (p >> kv.shift)); };
    auto look = [&](int it, int (&page)[NP]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NP; i++) page[i] = column(begin16(it, i));
    };
    auto place = [&](int it, const int (&page)[NP], int64_t (&at)[NP]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NP; i++) { // (a hole: any page, none of whose positions is seen)
            const int p = begin16(it, i), o = (unsigned)page[i] < (unsigned)kv.pages ? page[i] : 0;
            at[i] = o * kv.page + kh * kv.head + (p & ((1 << kv.shift) - 1)) * kv.slot;
        }
    };
    auto fetch = [&](const char *base, int c, int it, int plane, const int64_t (&at)[NP]) __attribute__((always_inline)) { // step `it` of K (plane 0) or V (1) into its buffer
        fh_half *to = pp_lds + (it % NB * 2 + plane) * KS * TILE + wave * 512;
        if (span.base + (it + 1) * KS * BN <= s.len) {
#pragma unroll
            for (int i = 0; i < NP; i++) fh_buffer_to_lds(base + at[i], 0x7FFFFFFF, to + NW * i * 512, (row & 15) * slot + c, 0);
        } else {
#pragma unroll
            for (int i = 0; i < NP; i++) { // rows past the last position repeat it
                const int end = s.len - 1 - begin16(it, i), y = (row & 15) < end ? row & 15 : end;
                fh_buffer_to_lds(base + at[i], 0x7FFFFFFF, to + NW * i * 512, y * slot + c, 0);
            }
        }
    };
    // This wavefront's pieces but the LATER last requests' are there, and everybody's behind the barrier; where no more are asked for, all of them.
    auto landed = [&](auto later, bool asking) {
        if (decltype(later)::value > 0 && asking) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(decltype(later)::value) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    constexpr std::integral_constant<int, (2 * NB - 2) * NP> but_first = {};
    constexpr std::integral_constant<int, (2 * NB - 4) * NP> but_two = {}; // K of the first two steps and V of the first, or a step's requests of NB - 2 steps
    static_assert((2 * NB - 2) * NP < 64, "a counter of six bits");
    // Whether any entry of the table that this part reads is no page; only then are they looked at again where scores are masked.
    bool holed = false;
    if (steps > 0) {
        const int c0 = span.base >> kv.shift, p1 = span.base + steps * KS * BN - 1, c1 = (p1 < s.len - 1 ? p1 : s.len - 1) >> kv.shift;
        for (int c = c0 + lane; c <= c1; c += 64) holed |= (unsigned)rows.table[(int64_t)seq * rows.cols + c] >= (unsigned)kv.pages;
        holed = __any(holed);
    }
    int page[NP];
    int64_t now[NP], then[NP]; // of the step whose V is requested next, and of the one whose K is
    if (steps > 0) look(0, page);
#pragma unroll
    for (int j = 0; j < NB; j++)
        if (j < steps) {
            place(j, page, then);
            if (j + 1 < steps) look(j + 1, page);
            fetch(kv.k, kc, j, 0, then);
            if (j > 0) fetch(kv.v, vc, j - 1, 1, now);
#pragma unroll
            for (int i = 0; i < NP; i++) now[i] = then[i];
        }
    if (steps < NB && steps > 0) fetch(kv.v, vc, steps - 1, 1, now);
    vec8 qf[KSTEPS];
    {
        const T *qp = (const T *)a.c.q + (s.row + x.token) * a.c.q_st + (kh * group + x.head) * a.c.q_sh + 8 * g;
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ks++) {
            qf[ks] = vec8{};
            if (16 * ks + 8 * g < a.c.d) __builtin_memcpy(&qf[ks], qp + 16 * ks, 16); // (any address)
        }
    }
    const int prow = 16 * (li >> 4) + 8 * ((li >> 2) & 1) + 4 * ((li >> 3) & 1) + (li & 3); // key read by MFMA row li
    const uint32_t k_at = kset * TILE * 2 + prow * D * 2 + (g ^ (D == 128 ? prow & 15 : (prow >> 1) & 7)) * 16; // bytes
    // keys 8 g + s / 4 (and 4 more) of a step of 16, dims 16 (lane / 16 % 2) + 4 (s % 4) .. of a tile of 32
    const int vrow = 8 * g + ((lane & 15) >> 2), vpiece = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
    const uint32_t v_at = (KS + kset) * TILE * 2 + vrow * D * 2 + (vpiece ^ (D == 128 ? (vrow & 3) << 2 : ((vrow >> 1) & 1) << 2)) * 16 + 8 * (lane & 1);
    const float sc2 = a.c.scale * 1.4426950408889634f; // scores in the log2 domain
    float m_run = -INFINITY, l_run = 0.f; // l_run: of this lane's keys
    floatx16 acc[DT], sa[2], sb[2];
    const floatx16 zero = {0.f};
#pragma unroll
    for (int dt = 0; dt < DT; dt++) acc[dt] = zero;
    auto scores = [&](int it, floatx16 (&to)[2]) __attribute__((always_inline)) { // S^T of step `it`
        uint32_t at = k_at + (uint32_t)(it % NB) * (4 * KS * TILE); // (swapped pieces are an exclusive or on the address, one instruction where it is used)
        asm volatile("" : "+v"(at));
        constexpr int NI = 2 * KSTEPS, AHEAD = 4;
        vec8 ka[AHEAD];
        auto read = [&](int i) { ka[i % AHEAD] = *(const vec8 *)((const uint8_t *)pp_lds + (at ^ (uint32_t)((i >> 1) * 32)) + (i & 1) * 64 * D); };
#pragma unroll
        for (int i = 0; i < AHEAD; i++) read(i);
#pragma unroll
        for (int i = 0; i < NI; i++) {
            to[i & 1] = pp_mfma(ka[i % AHEAD], qf[i >> 1], i < 2 ? zero : to[i & 1]);
            if (i + AHEAD < NI) read(i + AHEAD);
        }
    };
    // Register r of half kt is key t0 + 32 kt + 16 (r / 8) + 8 g + r % 8.
    auto mask = [&](int it, floatx16 (&to)[2]) __attribute__((always_inline)) {
        const int t0 = span.base + (it * KS + kset) * BN;
        uint32_t holes = 0; // its 16s without a page
        if (holed)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int p = t0 + 16 * i;
                if ((unsigned)column(p < last16 ? p : last16) >= (unsigned)kv.pages) holes |= 1u << i;
            }
        if (__any(t0 + BN - 1 > x.high || t0 < x.low) || holes) // some row does not see the whole tile
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int key = t0 + 32 * kt + 16 * (r >> 3) + 8 * g + (r & 7);
                    const bool seen = key >= x.low && key <= x.high && !(holes >> (2 * kt + (r >> 3)) & 1);
                    to[kt][r] = seen ? to[kt][r] : -INFINITY;
                }
    };
    auto requests = [&](int it) __attribute__((always_inline)) {
        if (it + NB < steps) {
            place(it + NB, page, then);
            fetch(kv.k, kc, it + NB, 0, then);
            if (it + NB + 1 < steps) look(it + NB + 1, page);
        }
        if (it + NB - 1 < steps) {
            fetch(kv.v, vc, it + NB - 1, 1, now);
#pragma unroll
            for (int i = 0; i < NP; i++) now[i] = then[i];
        }
    };
    auto step = [&](int it, floatx16 (&st)[2], floatx16 (&next)[2], bool last) __attribute__((always_inline)) {
        float mx = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int r = 0; r < 16; r++) mx = fmaxf(mx, st[kt][r]);
        mx = ap_swap32_max(mx) * sc2;
        const bool moves = mx - m_run > pp_ahead<F16>;
        if (__any(moves)) {
            const float alpha = moves ? __builtin_amdgcn_exp2f(m_run - mx) : 1.f;
            m_run = moves ? mx : m_run, l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int r = 0; r < 16; r++) acc[dt][r] *= alpha;
        }
        const float ref = m_run == -INFINITY ? 0.f : m_run;
        float by = sc2, m_sub = (F16 ? 14.f : 0.f) - ref; // weights of f16 are 2^14 times what they are: 2^-39 of the largest still counts
        if (__any(fabsf(ref) >= PAGED_FAR)) {
            by = 1.f, m_sub = F16 ? 14.f : 0.f;
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int r = 0; r < 16; r++) st[kt][r] = st[kt][r] * sc2 - ref;
        }
        requests(it);
        __builtin_amdgcn_sched_barrier(0);
        if (!last) scores(it + 1, next);
        vec8 pb[2][2];
        float ps = 0.f;
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int s2 = 0; s2 < 2; s2++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(st[kt][8 * s2 + e], by, m_sub));
                    ps += p;
                    pb[kt][s2][e] = (T)p;
                }
        l_run += ps;
#pragma unroll
        for (int kt = 0; kt < 2; kt++) // (here, beside the scores, and not behind the branch that follows)
#pragma unroll
            for (int s2 = 0; s2 < 2; s2++) asm volatile("" : "+v"(pb[kt][s2]));
        if (!last) {
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int i = 0; i < 2 * KSTEPS; i++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if (i < 2 * KSTEPS - 4) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 80 / (2 * KSTEPS), 0);
                __builtin_amdgcn_sched_group_barrier(0x400, 32 / (2 * KSTEPS), 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (!last) mask(it + 1, next);
        __builtin_amdgcn_sched_barrier(0);
        uint32_t at = v_at + (uint32_t)(it % NB) * (4 * KS * TILE);
        asm volatile("" : "+v"(at));
        constexpr int NJ = 4 * DT, AHEAD = 8;
        half8 va[AHEAD];
        auto read = [&](int j) { va[j % AHEAD] = ap_vt8((const fh_half *)((const uint8_t *)pp_lds + (at ^ (uint32_t)(j % DT * 64))) + 16 * (j / DT) * D, D); };
#pragma unroll
        for (int j = 0; j < AHEAD; j++) read(j);
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int c = j / DT;
            acc[j % DT] = pp_mfma(__builtin_bit_cast(vec8, va[j % AHEAD]), pb[c >> 1][c & 1], acc[j % DT]);
            if (j + AHEAD < NJ) read(j + AHEAD);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * AHEAD, 0);
#pragma unroll
        for (int j = 0; j < NJ - AHEAD; j++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
        landed(but_two, it + NB < steps);
    };
    if (steps > 0) {
        landed(but_first, steps >= NB);
        if (alive) {
            scores(0, sa);
            mask(0, sa);
            landed(but_two, steps >= NB);
            int t = 0;
            for (; t + 2 < steps; t += 2) {
                step(t, sa, sb, false);
                step(t + 1, sb, sa, false);
            }
            if (t + 2 == steps) {
                step(t, sa, sb, false);
                step(t + 1, sb, sa, true);
            } else
                step(t, sa, sb, true);
        } else {
            landed(but_two, steps >= NB);
            for (int t = 0; t < steps; t++) {
                requests(t);
                landed(but_two, t + NB < steps);
            }
        }
    }
    if constexpr (KS == 2) ap_merge<D, QW>((float *)pp_lds, wave, lane, kset, m_run, l_run, acc);
    if (KS == 2 && kset == 1) return;
    l_run = ap_swap32_sum(l_run);
    if (r < s.rows * group) pp_store<T, D>(a, part, s, x, kh, group, g, m_run, l_run, acc);
    pp_mend<T, T, D>(a, part, seq, s, x, r0 + (wave % QW) * 32, s.rows * group, kh, group, span.base, span.base + steps * KS * BN - 1, holed, l_run, acc);
}

// ---------------------------------------------------------------- every other type and head_dim
// Tiles of 32 positions through registers into LDS, f32 pages as three bf16 planes that add up to their values (24 bits, the whole range); f32 rows
// as three terms of bf16, or two of f16 brought to 2^14 first (22 bits).  Products of terms beyond the third order are below 2^-24 and left out:
// six where both operands have three, three or two where pages are of 16 bits.  Weights have as many terms as Q.
// One buffer, two barriers a tile: products, softmax and splitting follow each other (2048 rows, us, 32 / 8 heads of 128: f32 231, f32 over f16 130, over bf16 133; 16 / 4 heads
// of 256: f16 147, bf16 129, f32 523, over f16 185, over bf16 297).
template <typename TX, typename TP, int DP>
__global__ __launch_bounds__(256) void k_paged_planes(PpArgs a) {
    constexpr bool F32 = sizeof(TP) == 4, F16 = __is_same(TP, fh_half), MIXED = sizeof(TX) != sizeof(TP);
    typedef typename std::conditional<F16, fh_half, fh_bf>::type T; // of the products
    typedef typename PpVec<T>::type vec8;
    constexpr int BN = 32, DT = DP / 32, KSTEPS = DP / 16, CH = DP / 8, KR = DP + 8, VR = DP + 32; // halfs of a row of K and V in LDS
    constexpr int KP = F32 ? 3 : 1, QT = F32 ? 3 : !MIXED ? 1 : F16 ? 2 : 3, N = BN * CH / 256;    // planes, terms; pieces of 8 values a thread
    extern __shared__ __attribute__((aligned(16))) fh_half pp_lds[]; // [KP][BN][KR], [KP][BN][VR]
    fh_half *sk = pp_lds, *sv = pp_lds + KP * BN * KR;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, li = lane & 31, g = lane >> 5;
    const PagedKv &kv = a.c.kv;
    const PagedRows &rows = a.c.rows;
    const int kh = blockIdx.x, group = a.c.hq / a.c.hkv, seq = pp_sequence(a, (int)blockIdx.z / a.parts), part = (int)blockIdx.z % a.parts;
    const PagedSeq s = paged_seq_scalar(rows, kv.shift, seq);
    const int r0 = (int)(gridDim.y - 1 - blockIdx.y) * 128;
    if (r0 >= s.rows * group) return;
    const PpSpan span = pp_span<BN>(s, r0, r0 + 127, group, a.c.window, part, a.parts);
    const bool alive = r0 + wave * 32 < s.rows * group;
    const int r = r0 + wave * 32 + li;
    const PpRow x = pp_row(s, r, group, a.c.window);

    vec8 qf[QT][KSTEPS];
    float sc2 = a.c.scale * 1.4426950408889634f; // scores in the log2 domain
    {
        const TX *qp = (const TX *)a.c.q + (s.row + x.token) * a.c.q_st + (kh * group + x.head) * a.c.q_sh + 8 * g;
        int ex = 0;
        if constexpr (MIXED && F16) { // brought to 2^14 .. 2^15
            float most = 0.f;
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ks++)
                if (16 * ks + 8 * g < a.c.d)
#pragma unroll
                    for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf((float)qp[16 * ks + e]));
            most = ap_swap32_max(most);
            if (most > 0.f && most < INFINITY) ex = 15 - __builtin_amdgcn_frexp_expf(most);
            sc2 = paged_brought(sc2, ex);
        }
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ks++) {
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (16 * ks + 8 * g < a.c.d) {
                TX t[8];
                __builtin_memcpy(t, qp + 16 * ks, sizeof(t)); // (any address)
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = MIXED && F16 ? ldexpf((float)t[e], ex) : (float)t[e];
            }
#pragma unroll
            for (int u = 0; u < QT; u++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const T y = u == 0 && QT > 1 ? paged_first<T>(v[e]) : (T)v[e];
                    qf[u][ks][e] = y;
                    v[e] -= (float)y;
                }
        }
    }
    const int prow = 16 * (li >> 4) + 8 * ((li >> 2) & 1) + 4 * ((li >> 3) & 1) + (li & 3); // key read by MFMA row li
    const int vrow = 8 * g + ((lane & 15) >> 2), vcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    float m_run = -INFINITY, l_run = 0.f; // l_run: of this lane's keys
    floatx16 acc[DT];
    const floatx16 zero = {0.f};
#pragma unroll
    for (int dt = 0; dt < DT; dt++) acc[dt] = zero;

    const int last16 = (s.len - 1) & ~15;
    uint4 kraw[N][KP == 3 ? 2 : 1], vraw[N][KP == 3 ? 2 : 1];
    uint32_t holes = 0, next_holes = 0;
    bool holed = false;
    int page[2];
    auto look = [&](int t0) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int p = t0 + 16 * h < last16 ? t0 + 16 * h : last16;
            page[h] = paged_scalar(rows.table, (int64_t)seq * rows.cols + (p >> kv.shift));
        }
    };
    auto ask = [&](int t0) { // a tile into registers; rows past the last position repeat it, values behind the head's end are zeros
        next_holes = 0;
        int64_t at[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int p = t0 + 16 * h < last16 ? t0 + 16 * h : last16;
            if ((unsigned)page[h] >= (unsigned)kv.pages) page[h] = 0, next_holes |= 1u << h;
            at[h] = page[h] * kv.page + kh * kv.head + (p & ((1 << kv.shift) - 1)) * kv.slot;
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int c = tid + 256 * i, y = c / CH, e = c % CH * 8, h = y >> 4;
            int key = t0 + (y & ~15) < last16 ? y & 15 : s.len - 1 - last16; // slot of its 16
            if (t0 + (y & ~15) == last16) key = (y & 15) < s.len - 1 - last16 ? y & 15 : s.len - 1 - last16;
            const int64_t o = (h ? at[1] : at[0]) + key * kv.slot + e * (int)sizeof(TP);
#pragma unroll
            for (int w = 0; w < (KP == 3 ? 2 : 1); w++) {
                kraw[i][w] = vraw[i][w] = make_uint4(0, 0, 0, 0);
                if (e < a.c.d) kraw[i][w] = *(const uint4 *)(kv.k + o + 16 * w), vraw[i][w] = *(const uint4 *)(kv.v + o + 16 * w);
            }
        }
    };
    auto keep = [&](const uint4 (&raw)[KP == 3 ? 2 : 1], fh_half *to, int plane) { // eight values to LDS
        if constexpr (KP == 1) *(uint4 *)to = raw[0];
        else {
            uint32_t v[8];
            __builtin_memcpy(v, raw, 32);
            uint32_t w[3][4];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                uint32_t p0 = v[e], p1 = v[e + 1];
#pragma unroll
                for (int u = 0; u < 3; u++) { // the upper 16 bits, and what they leave (8 + 8 + 8 bits)
                    w[u][e / 2] = __builtin_amdgcn_perm(p1, p0, 0x07060302u);
                    p0 = __float_as_uint(__uint_as_float(p0) - __uint_as_float(p0 & 0xFFFF0000u));
                    p1 = __float_as_uint(__uint_as_float(p1) - __uint_as_float(p1 & 0xFFFF0000u));
                }
            }
#pragma unroll
            for (int u = 0; u < 3; u++) *(uint4 *)(to + u * plane) = make_uint4(w[u][0], w[u][1], w[u][2], w[u][3]);
        }
    };
    if (span.steps > 0) {
        look(span.base);
        ask(span.base);
        if (span.steps > 1) look(span.base + BN);
    }
    for (int it = 0; it < span.steps; it++) {
        const int t0 = span.base + it * BN;
        __syncthreads(); // nobody reads the tile before any more
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int c = tid + 256 * i, y = c / CH, e = c % CH * 8;
            keep(kraw[i], sk + y * KR + e, BN * KR);
            keep(vraw[i], sv + y * VR + e, BN * VR);
        }
        holes = next_holes, holed |= holes != 0;
        __syncthreads();
        if (it + 1 < span.steps) {
            ask(t0 + BN);
            if (it + 2 < span.steps) look(t0 + 2 * BN);
        }
        if (!alive) continue;
        floatx16 st = zero;
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ks++) {
            vec8 k[KP];
#pragma unroll
            for (int u = 0; u < KP; u++) k[u] = *(const vec8 *)(sk + u * BN * KR + prow * KR + 16 * ks + 8 * g);
#pragma unroll
            for (int o = (KP > QT ? KP : QT) - 1; o >= 0; o--) // the smallest first
#pragma unroll
                for (int u = 0; u < KP; u++)
                    if (o - u >= 0 && o - u < QT) st = pp_mfma(k[u], qf[o - u][ks], st);
        }
        // register r is key t0 + 16 (r / 8) + 8 g + r % 8
        if (__any(t0 + BN - 1 > x.high || t0 < x.low) || holes)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int key = t0 + 16 * (r >> 3) + 8 * g + (r & 7);
                const bool seen = key >= x.low && key <= x.high && !(holes >> (r >> 3) & 1);
                st[r] = seen ? st[r] : -INFINITY;
            }
        float mx = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; r++) mx = fmaxf(mx, st[r]);
        mx = ap_swap32_max(mx) * sc2;
        const bool moves = mx - m_run > pp_ahead<F16>;
        if (__any(moves)) {
            const float alpha = moves ? __builtin_amdgcn_exp2f(m_run - mx) : 1.f;
            m_run = moves ? mx : m_run, l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int r = 0; r < 16; r++) acc[dt][r] *= alpha;
        }
        const float ref = m_run == -INFINITY ? 0.f : m_run;
        float by = sc2, m_sub = (F16 ? 14.f : 0.f) - ref; // (weights of f16: 2^14 times what they are)
        if (__any(fabsf(ref) >= PAGED_FAR)) {
            by = 1.f, m_sub = F16 ? 14.f : 0.f;
#pragma unroll
            for (int r = 0; r < 16; r++) st[r] = st[r] * sc2 - ref;
        }
        vec8 pb[QT][2];
#pragma unroll
        for (int r = 0; r < 16; r++) {
            float p = __builtin_amdgcn_exp2f(fmaf(st[r], by, m_sub));
            l_run += p;
#pragma unroll
            for (int u = 0; u < QT; u++) {
                const T y = (T)p;
                pb[u][r >> 3][r & 7] = y;
                p -= (float)y;
            }
        }
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                half8 v[KP];
#pragma unroll
                for (int u = 0; u < KP; u++) v[u] = ap_vt8(sv + u * BN * VR + (16 * c + vrow) * VR + 32 * dt + vcol, VR);
#pragma unroll
                for (int o = (KP > QT ? KP : QT) - 1; o >= 0; o--)
#pragma unroll
                    for (int u = 0; u < KP; u++)
                        if (o - u >= 0 && o - u < QT) acc[dt] = pp_mfma(__builtin_bit_cast(vec8, v[u]), pb[o - u][c], acc[dt]);
            }
    }
    l_run = ap_swap32_sum(l_run);
    if (r < s.rows * group) pp_store<TX, DP>(a, part, s, x, kh, group, g, m_run, l_run, acc);
    pp_mend<TX, TP, DP>(a, part, seq, s, x, r0 + wave * 32, s.rows * group, kh, group, span.base, span.base + span.steps * BN - 1, holed, l_run, acc);
}

// ---------------------------------------------------------------- the parts together
// A wavefront a row and head: lanes weigh a part each, then groups of them take parts in turn, four values a lane, eight parts on their way.
template <typename TX>
__global__ __launch_bounds__(256) void k_paged_join(PpArgs a) {
    __shared__ float s_w[4][PP_PARTS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = (int)blockIdx.x * 4 + wave, d = a.c.d, parts = a.parts;
    const PagedSeq s = paged_seq(a.c.rows, a.c.kv.shift, blockIdx.y);
    if (i >= s.rows * a.c.hq) return;
    const int64_t row = (int64_t)s.row * a.c.hq + i, all = (int64_t)a.c.rows.tokens * a.c.hq;
    float m[PP_PARTS / 64], l[PP_PARTS / 64], mx = -INFINITY, den = 0.f;
#pragma unroll
    for (int k = 0; k < PP_PARTS / 64; k++) {
        const int p = lane + 64 * k;
        m[k] = -INFINITY, l[k] = 0.f;
        if (p < parts) m[k] = a.stats[2 * (p * all + row)], l[k] = a.stats[2 * (p * all + row) + 1];
        mx = fmaxf(mx, m[k]);
    }
#pragma unroll
    for (int w = 32; w; w >>= 1) mx = fmaxf(mx, __shfl_xor(mx, w));
    const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int k = 0; k < PP_PARTS / 64; k++) {
        const float f = __builtin_amdgcn_exp2f(m[k] - ref);
        s_w[wave][lane + 64 * k] = f; // (read by this wavefront alone: its LDS operations are in order)
        den = fmaf(l[k], f, den);
    }
#pragma unroll
    for (int w = 32; w; w >>= 1) den += __shfl_xor(den, w);
    int wide = 2; // lanes of a group: a power of two that has all of the row
    while (4 * wide < d) wide *= 2;
    const int at = lane % wide * 4, first = lane / wide, groups = 64 / wide;
    const bool mine = at < d;
    const float *from = a.sums + row * d + (mine ? at : 0);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int p = first; p < parts; p += groups) {
        const float4 y = *(const float4 *)(from + p * all * d);
        const float f = s_w[wave][p];
        x.x = fmaf(y.x, f, x.x), x.y = fmaf(y.y, f, x.y), x.z = fmaf(y.z, f, x.z), x.w = fmaf(y.w, f, x.w);
    }
    for (int w = wide; w < 64; w *= 2) x.x += __shfl_xor(x.x, w), x.y += __shfl_xor(x.y, w), x.z += __shfl_xor(x.z, w), x.w += __shfl_xor(x.w, w);
    const float inv = den == 0.f ? 0.f : 1.f / den; // (a row that sees nothing: zeros)
    if (mine && first == 0) ap_store4((TX *)a.c.out + row * d + at, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
}

// ---------------------------------------------------------------- which form
// Parts: as many as compute units have a workgroup each, of at least a step of positions; one where that saves a workgroup fewer than `saves` steps, which is what
// the second launch takes (32 / 8 heads of 128, f16, us, with parts / without: 16 rows behind 500 positions 14.2 / 19.4, 8 behind 2000 16.3 / 39.6, a prompt of 300
// 20.5 / 16.0, of 512 24.0 / 18.8; f32 10 behind 500 18.9 / 57), and where scratch memory cannot be had.
static int pp_parts(fh_device *dev, const PagedCall &call, int64_t wgs, int64_t longest, int step, int saves, PpArgs *a) {
    const int64_t steps = (longest + step - 1) / step;
    int parts = (int)(dev->compute_units / wgs < steps ? dev->compute_units / wgs : steps);
    parts = parts < 1 ? 1 : parts > PP_PARTS ? PP_PARTS : parts;
    if (steps - (steps + parts - 1) / parts < saves) parts = 1;
    a->parts = parts;
    if (parts == 1) return 1;
    const size_t n = (size_t)parts * call.rows.tokens * call.hq;
    if (call.rows.seqs * parts > 65535 || !fh_dev_scratch_try(dev, (void **)&dev->part_buf, &dev->part_cap, n * (call.d + 2) * 4)) return a->parts = 1;
    a->sums = dev->part_buf, a->stats = dev->part_buf + n * call.d;
    return parts;
}
template <typename TX> static fh_status pp_join(fh_device *dev, const PpArgs &a) {
    if (a.parts > 1) {
        k_paged_join<TX><<<dim3((unsigned)(((int64_t)a.c.rows.max_new * a.c.hq + 3) / 4), (unsigned)a.c.rows.seqs), dim3(256), 0, dev->stream>>>(a);
        FH_HIP(hipGetLastError());
    }
    return FH_OK;
}

template <typename T, int D, int KS>
static fh_status pp_tiles(fh_device *dev, PpArgs a) {
    constexpr int LDS = 4 * KS * 64 * D * 2, MERGE = KS == 2 ? (2 + D / 2) * 256 * 4 : 0, BYTES = LDS > MERGE ? LDS : MERGE;
    const auto kern = k_paged_tiles<T, D, KS>;
    FH_TRY(fh_kernel_lds(dev, (const void *)kern, BYTES));
    const unsigned blocks = (unsigned)(((int64_t)a.c.rows.max_new * (a.c.hq / a.c.hkv) + 127) / 128);
    kern<<<dim3((unsigned)a.c.hkv, blocks, (unsigned)(a.c.rows.seqs * a.parts)), dim3(256 * KS), BYTES, dev->stream>>>(a);
    FH_HIP(hipGetLastError());
    return pp_join<T>(dev, a);
}
template <typename TX, typename TP, int DP>
static fh_status pp_planes(fh_device *dev, PpArgs a, int64_t longest) {
    constexpr int KP = sizeof(TP) == 4 ? 3 : 1, LDS = KP * 32 * (DP + 8 + DP + 32) * 2;
    const int64_t blocks = ((int64_t)a.c.rows.max_new * (a.c.hq / a.c.hkv) + 127) / 128;
    a.sorted = blocks * a.c.hkv * a.c.rows.seqs > dev->compute_units;
    pp_parts(dev, a.c, blocks * a.c.hkv * a.c.rows.seqs, longest, 64, 1, &a);
    const auto kern = k_paged_planes<TX, TP, DP>;
    FH_TRY(fh_kernel_lds(dev, (const void *)kern, LDS));
    kern<<<dim3((unsigned)a.c.hkv, (unsigned)blocks, (unsigned)(a.c.rows.seqs * a.parts)), dim3(256), LDS, dev->stream>>>(a);
    FH_HIP(hipGetLastError());
    return pp_join<TX>(dev, a);
}
template <typename TX, typename TP> static fh_status pp_dim(fh_device *dev, const PpArgs &a, int64_t longest) {
    if (a.c.d <= 64) return pp_planes<TX, TP, 64>(dev, a, longest);
    if (a.c.d <= 128) return pp_planes<TX, TP, 128>(dev, a, longest);
    return pp_planes<TX, TP, 256>(dev, a, longest);
}
template <typename T> static fh_status pp_same(fh_device *dev, PpArgs a, int64_t longest) {
    if (a.c.d > 128) return pp_planes<T, T, 256>(dev, a, longest);
    const int64_t rows = (int64_t)a.c.rows.max_new * (a.c.hq / a.c.hkv), pairs = (int64_t)a.c.hkv * a.c.rows.seqs;
    const int64_t wgs = pairs * ((rows + 127) / 128);
    // Two groups of four wavefronts share a workgroup's positions while no more than two workgroups of four would have come to a compute unit (32 / 8 heads of 128, us,
    // two groups / one: 1024 behind 4000 101 / 131, 33 behind 65536 91 / 117, 2048 alone 58 / 62, behind 4000 193 / 186; 4096 alone 187 / 176, 8192 670 / 604,
    // 8 of 512 behind 4001 211 / 173).
    const bool halves = wgs <= 2 * dev->compute_units && longest > 128;
    a.sorted = wgs > dev->compute_units;
    pp_parts(dev, a.c, wgs, longest, 128, 3, &a);
    if (a.c.d > 64) return halves ? pp_tiles<T, 128, 2>(dev, a) : pp_tiles<T, 128, 1>(dev, a);
    return halves ? pp_tiles<T, 64, 2>(dev, a) : pp_tiles<T, 64, 1>(dev, a);
}
fh_status fh_paged_prompt(fh_device *dev, int dtype, int kv_dtype, const PagedCall &call, int max_len) {
    FH_REQUIRE((int64_t)call.rows.max_new * (call.hq / call.hkv) <= 65535LL * 64, "%d new rows of a sequence with %d heads a KV head", call.rows.max_new,
               call.hq / call.hkv);
    PpArgs a = {};
    a.c = call;
    int64_t longest = (int64_t)call.rows.cols << call.kv.shift;
    if (max_len > 0 && max_len < longest) longest = max_len;
    if (call.window > 0 && (int64_t)call.window + call.rows.max_new < longest) longest = (int64_t)call.window + call.rows.max_new;
    if (dtype == FH_F16) return pp_same<fh_half>(dev, a, longest);
    if (dtype == FH_PAGED_BF16) return pp_same<fh_bf>(dev, a, longest);
    if (kv_dtype == FH_F32) return pp_dim<float, float>(dev, a, longest);
    if (kv_dtype == FH_F16) return pp_dim<float, fh_half>(dev, a, longest);
    return pp_dim<float, fh_bf>(dev, a, longest);
}
