// Kernels of the serving operators on paged K/V caches: appending new tokens
// with their position rotation, and attention behind shared prefixes.
#pragma once
#include "fav4_serving.h"
#include "bshd_kernel.hpp"

namespace fav4 {

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Division of 0 <= n < 2^31 by a divisor d >= 1 that the host knows: with l =
// ceil(log2 d) and m = floor(2^(31 + l) / d) + 1 (below 2^32), n / d is
// floor(n m / 2^(31 + l)).
struct FastDiv {
    uint32_t m;
    int l;
    __device__ __forceinline__ int operator()(int n) const { return int(__umulhi(uint32_t(n) * 2, m) >> l); }
};
inline FastDiv fast_div(int d) {
    int l = 0;
    while ((int64_t(1) << l) < d) ++l;
    return {uint32_t((uint64_t(1) << (31 + l)) / uint32_t(d) + 1), l};
}

// Of values that are the same in every lane.
__device__ __forceinline__ int udiv(int n, int d) { return uniform(int(uint32_t(n) / uint32_t(d))); }
__device__ __forceinline__ int udiv_up(int n, int d) { return udiv(n + d - 1, d); }

// How many of the non-decreasing cu[1..n] are <= x, found by the whole wave: 64
// entries at a time, so two rounds of loads up to 4096 entries.  For x >=
// cu[0] that is the index of the range [cu[i], cu[i + 1]) that holds x, or n
// behind the last one.
__device__ __forceinline__ int wave_find(const int* cu, int n, int x, int lane) {
    int lo = 0, left = n;
    while (left > 64) {
        const int stride = (left + 63) >> 6;
        const int at = lo + min((lane + 1) * stride, left);        // last entry of this lane's stretch
        const uint64_t below = __builtin_amdgcn_ballot_w64(cu[at] <= x);
        const int c = below == ~0ull ? 64 : __builtin_ctzll(~below);
        const int next = min(c * stride, left);
        lo += next;
        left = min(stride, left - next);
    }
    const uint64_t below = __builtin_amdgcn_ballot_w64(lane < left && cu[lo + min(lane, left - 1) + 1] <= x);
    return left > 0 ? lo + __builtin_popcountll(below) : lo;
}

// ---------------------------------------------------------------------------
// Append.  One wave takes 8 of a token's heads + 2 * kv_heads rows (Q, then K,
// then V): 8 lanes a row, each with the two 16-byte granules whose dims are
// rotated together (both lie in this lane: granules j and j + rotary_dim / 16,
// or neighbours).  Bound by memory, for few tokens by the chain of dependent
// loads: offsets -> sequence and rows -> key count, table entry and angles ->
// store.  Rows are loaded behind the check that a sequence has them, for a
// caller's buffers may end with the last sequence.
// ---------------------------------------------------------------------------
template <bool INTERLEAVED>
__global__ __launch_bounds__(256) void append_kernel(Fav4AppendArgs a, int units, int64_t total, FastDiv by_units, FastDiv by_page) {
    const int lane = threadIdx.x & 63, j = lane & 7;
    const int64_t stride = int64_t(gridDim.x) * 4;
    const int qheads = a.q ? a.heads : 0, rows = qheads + 2 * a.kv_heads;
    const int half = a.rotary_dim >> 4;                    // granules of half the rotated dims
    const int first = a.cu_seqlens_q[0], end = a.cu_seqlens_q[a.batch];
    for (int64_t id = int64_t(blockIdx.x) * 4 + uniform(threadIdx.x >> 6); id < total; id += stride) {
        const int t = uniform(by_units(int(id))), unit = uniform(int(id) - t * units);
        if (t < first || t >= end) continue;               // in no sequence
        const int row = unit * 8 + (lane >> 3);
        const bool live = row < rows, is_q = row < qheads, is_v = row >= qheads + a.kv_heads;
        const int head = is_q ? row : is_v ? row - qheads - a.kv_heads : row - qheads;
        const char* src = static_cast<const char*>(is_q ? a.q : is_v ? a.v : a.k);
        src += (int64_t(t) * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride) + int64_t(head) * D) * 2;
        // This lane's granules of the row.
        const bool turn = j < half;
        const int g0 = INTERLEAVED || !turn ? 2 * j : j;
        const int g1 = INTERLEAVED || !turn ? g0 + 1 : j + half;
        bf16x8 x{}, y{};
        if (live) {
            x = *reinterpret_cast<const bf16x8*>(src + g0 * 16);
            y = *reinterpret_cast<const bf16x8*>(src + g1 * 16);
        }
        const int b = wave_find(a.cu_seqlens_q, a.batch, t, lane);     // below batch: the last offset is above t
        const int64_t slot = int64_t(a.seqlens_k[b]) - a.cu_seqlens_q[b + 1] + t;
        int page = -1, in_page = 0;
        if (slot >= 0 && slot < int64_t(a.max_pages_per_seq) * a.page_size && slot <= INT_MAX) {
            const int at = by_page(int(slot));
            in_page = int(slot) - at * a.page_size;
            page = a.block_table[int64_t(b) * a.max_pages_per_seq + at];
        }
        const bool stored = page >= 0 && page < a.num_pages;
        if (turn && !is_v && live) {
            const int64_t pos = a.positions ? int64_t(a.positions[t]) : slot;
            const int64_t r = min(max(pos, int64_t(0)), int64_t(a.rotary_rows - 1));
            const int64_t at = r * (half * 8) + j * 8;
            const f32x4* cp = reinterpret_cast<const f32x4*>(a.cos + at);
            const f32x4* sp = reinterpret_cast<const f32x4*>(a.sin + at);
            const f32x4 c[2] = {cp[0], cp[1]}, s[2] = {sp[0], sp[1]};
            bf16x8 u, w;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float ci = c[i >> 2][i & 3], si = s[i >> 2][i & 3];
                if constexpr (INTERLEAVED) {
                    const bf16x8& z = i < 4 ? x : y;
                    const float p = float(z[2 * (i & 3)]), q = float(z[2 * (i & 3) + 1]);
                    bf16x8& o = i < 4 ? u : w;
                    o[2 * (i & 3)] = __bf16(p * ci - q * si);
                    o[2 * (i & 3) + 1] = __bf16(q * ci + p * si);
                } else {
                    const float p = float(x[i]), q = float(y[i]);
                    u[i] = __bf16(p * ci - q * si);
                    w[i] = __bf16(q * ci + p * si);
                }
            }
            x = u;
            y = w;
        }
        if (!live || (!is_q && !stored)) continue;
        char* dst;
        if (is_q) {
            dst = static_cast<char*>(a.q_out) + (int64_t(t) * a.q_out_stride + int64_t(head) * D) * 2;
        } else {
            dst = static_cast<char*>(is_v ? a.v_cache : a.k_cache);
            dst += ((int64_t(page) * a.page_size + in_page) * a.kv_heads + head) * ROW_BYTES;
        }
        *reinterpret_cast<bf16x8*>(dst + g0 * 16) = x;
        *reinterpret_cast<bf16x8*>(dst + g1 * 16) = y;
    }
}

// ---------------------------------------------------------------------------
// Attention behind shared prefixes.  Rows are (token, query head of the K/V
// head's group), r = token * group + head: the rows of all sequences of a
// prefix are neighbours, and so are those of one sequence.  A segment is a row
// tile of one prefix against the prefix's keys (BM rows), or of one sequence
// against the sequence's own keys; it costs its key tiles and some more (SEG_TILES),
// laid before them, for what its start and end cost (without keys, one tile).
// The segments of a K/V head are laid end to end, the prefixes' on one line,
// the sequences' own on another, and each line is cut into ranges of one
// length, whatever segments they cross.
//
// A prefix range is a workgroup's: its eight waves take 32 rows each of the row
// tile and share the K/V tiles (attend_shared), or, where the prefixes have few
// rows, all take the same 32 rows, each every eighth key tile (attend_split).  An
// own range is a workgroup's too, or a single wave's where the sequences have few
// rows (attend_wave): the wave streams 32-key tiles through 16 KiB of LDS of its
// own, with no barrier, and the eight such waves of a CU hide each other's
// latency.
//
// A segment's part that lies in range w writes its O (normalised, FP32) and two
// log-sums (log2: of the BF16 weights, and of the FP32 ones) to partial block
// (segment + w) of its line: segments and ranges both only grow along the line,
// so no two parts have the same sum, and the blocks number segments + ranges.
// Weights are rounded to BF16 for the product with V, whose matrix instruction
// takes no wider operand beside a BF16 V, and summed as rounded, as in the forward:
// 0.0023 of O against 64 bits, 0.0017 with FP32 weights; everything else is FP32.
// The part that holds a segment's first key tile also notes for each of its rows
// where its partials start and how many there are; prefix_merge_kernel goes by
// those notes.
// ---------------------------------------------------------------------------
struct PrefixPlan {
    float *o_part, *lse_part;         // prefix blocks of all K/V heads (BM rows each), then own blocks (own_rows each)
    int2* notes;                      // [total_q * group][2]: first partial row and parts, prefix and own
    int group;                        // query heads of a K/V head
    int ranges;                       // workgroups of a K/V head
    FastDiv by_kv_heads, by_group, by_page, by_heads, by_bm, by_own_rows;
    int prefix_blocks, own_blocks;    // partial blocks of a K/V head
    int own_rows;                     // rows of an own block
    int most_prefix_keys;             // of a prefix, whole pages: its table's, and those that max_seqlen_k reaches into
    int br;                           // bottom-right causal
};

// Of a shared segment (the eight waves' key tiles), a wave's, and a split one.
constexpr int SEG_TILES = 4, OWN_SEG_TILES = 2, SPLIT_SEG_TILES = 8;
constexpr int MIN_PREFIX_TILES = 2, MIN_OWN_TILES = 1, MIN_SPLIT_TILES = 4;  // shortest ranges
// What a prefix's key tile costs, in own key tiles of a wave (its share of the
// workgroups follows): 64 keys against 256 rows, and 32 keys against 32 rows split
// over the waves (at 2: 32.4 -> 33.6 us over 53 calls).
constexpr float PREFIX_COST = 4.f, SPLIT_COST = 1.f;

// A prefix or a sequence: its tokens and the keys [k0, k1) that they read here.
// A sequence of no prefix has k0 = -1 for 0.
struct Family {
    int t0, tokens, k0, k1;
};

// The families of a batch of up to so many sequences and prefixes are worked out
// once and kept in LDS; of larger ones they are read from memory where they are
// needed.  (What comes before the first tile is some 300 instructions that every
// workgroup runs once, at about 10 ns each: their code has to be fetched.)
constexpr int PLAN_SEQS = 512, PLAN_PREFIXES = 256;
struct PlanLds {
    int4 own[PLAN_SEQS + 1], prefix[PLAN_PREFIXES];
    int first_seq[PLAN_PREFIXES + 1], prefix_keys[PLAN_PREFIXES];
};

// The batch as read on the device, clamped: tokens to [0, total_q], keys to
// [0, max_seqlen_k], a prefix's keys to whole pages of its table (of those that a
// sequence of max_seqlen_k keys reaches into).
template <bool CACHED>
struct PrefixBatch {
    const Fav4PrefixArgs& a;
    const PrefixPlan& pl;
    const PlanLds& lds;
    bool hidden;                      // a sequence may not see all of its prefix

    __device__ __forceinline__ int load_cu(int b) const {
        return min(max(a.paged.cu_seqlens_q[b], 0), a.paged.total_q);
    }
    __device__ __forceinline__ int load_keys(int b) const {
        return min(max(a.paged.seqlens_k[b], 0), a.paged.max_seqlen_k);
    }
    __device__ __forceinline__ int load_first_seq(int p) const {
        return min(max(a.cu_prefix_seqs[p], 0), a.paged.batch);
    }
    __device__ __forceinline__ int load_prefix_keys(int p) const {
        return pl.by_page(min(max(a.prefix_lens[p], 0), pl.most_prefix_keys)) * a.paged.page_size;
    }
    __device__ __forceinline__ int cu(int b) const { return CACHED ? lds.own[b].x : load_cu(b); }
    __device__ __forceinline__ int keys(int b) const { return CACHED ? lds.own[b].w : load_keys(b); }
    __device__ __forceinline__ int first_seq(int p) const { return CACHED ? lds.first_seq[p] : load_first_seq(p); }
    __device__ __forceinline__ int prefix_keys(int p) const { return CACHED ? lds.prefix_keys[p] : load_prefix_keys(p); }
    // Shared keys of sequence b: of the last prefix that starts at or before it.
    __device__ __forceinline__ int find_shared(int b) const {
        int lo = 0, hi = a.num_prefixes;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first_seq(mid) <= b) lo = mid;
            else hi = mid;
        }
        return first_seq(lo) <= b && b < first_seq(lo + 1) ? prefix_keys(lo) : 0;
    }
    __device__ __forceinline__ Family make_prefix(int p) const {
        const int s0 = first_seq(p), s1 = max(first_seq(p + 1), s0), t0 = cu(s0), keys = prefix_keys(p);
        return {t0, keys > 0 ? max(0, cu(s1) - t0) : 0, 0, keys};
    }
    __device__ __forceinline__ Family make_own(int t0, int t1, int sk, int shared) const {
        return {t0, min(max(t1 - t0, 0), a.paged.max_seqlen_q), shared > 0 ? min(shared, sk) : -1, sk};
    }
    __device__ __forceinline__ Family prefix_family(int p) const {
        if constexpr (CACHED) return __builtin_bit_cast(Family, lds.prefix[p]);
        return make_prefix(p);
    }
    __device__ __forceinline__ Family own_family(int b) const {
        if constexpr (CACHED) return __builtin_bit_cast(Family, lds.own[b]);
        return make_own(load_cu(b), load_cu(b + 1), load_keys(b), find_shared(b));
    }
};

// A line of families' segments: row tiles of ROWS rows, key tiles of BN keys,
// LEAD units before each segment's key tiles.
template <class B, bool OWN, int ROWS, int BN, int LEAD>
struct Line {
    const B& x;
    int count, group;
    __device__ __forceinline__ Family family(int i) const { return OWN ? x.own_family(i) : x.prefix_family(i); }
    __device__ __forceinline__ int tiles(const Family& f) const { return int(uint32_t(f.tokens * group + ROWS - 1) / ROWS); }
    __device__ __forceinline__ int key_tiles(const Family& f) const { return int(uint32_t(f.k1 - max(f.k0, 0) + BN - 1) / BN); }
    __device__ __forceinline__ int seg_cost(const Family& f) const { return max(1, key_tiles(f)) + LEAD; }

    // Up to 64 families from i on in the wave's lanes: the units and segments up to and with each.
    struct Sums {
        int cost, segs, cost_end, segs_end;
    };
    __device__ __forceinline__ Sums sums(int i, int lane) const {
        Family f{};
        if (i + lane < count) f = family(i + lane);
        const int s = tiles(f), c = s * seg_cost(f);
        return {c, s, wave_scan(c), wave_scan(s)};
    }
    // The line's length; `head` gets the first families' sums.
    __device__ __forceinline__ int length(int lane, Sums& head) const {
        head = sums(0, lane);
        int total = __builtin_amdgcn_readlane(head.cost_end, 63);
        for (int i = 64; i < count; i += 64) total += __builtin_amdgcn_readlane(sums(i, lane).cost_end, 63);
        return total;
    }
    // The family that holds unit `at`, the unit where it starts and the segments before it.
    struct Place {
        int idx, base, seg;
    };
    __device__ __forceinline__ Place find(int at, int lane, const Sums& head) const {
        Sums v = head;
        Place p{0, 0, 0};
        for (;;) {
            const uint64_t hit = __builtin_amdgcn_ballot_w64(p.base + v.cost_end > at);
            if (hit) {
                const int l = __builtin_ctzll(hit);
                return {uniform(p.idx + l), uniform(p.base + __builtin_amdgcn_readlane(v.cost_end - v.cost, l)),
                        uniform(p.seg + __builtin_amdgcn_readlane(v.segs_end - v.segs, l))};
            }
            p.base += __builtin_amdgcn_readlane(v.cost_end, 63);
            p.seg += __builtin_amdgcn_readlane(v.segs_end, 63);
            p.idx += 64;
            if (p.idx >= count) return {count, 0, 0};
            v = sums(p.idx, lane);
        }
    }
};

// Number of a page table's entries, 64 of them in the wave's lanes; key tiles
// are taken in ascending order.
struct PageWalk {
    const int* table;
    int entries, page_size, num_pages, pages, slot0, slot, in_page;
    __device__ __forceinline__ void load(int lane) {
        slot0 = slot;
        pages = min(max(table[min(slot + lane, entries - 1)], 0), num_pages - 1);
    }
    __device__ __forceinline__ void start(const int* t, int n, int key, const FastDiv& by_page, int lane) {
        table = t;
        entries = n;
        slot = by_page(key);
        in_page = key - slot * page_size;
        load(lane);
    }
    // The cache row of the present key; then on by `step` keys.
    __device__ __forceinline__ int64_t row(int step, int lane) {
        if (slot - slot0 >= 64) load(lane);
        const int64_t r = int64_t(__builtin_amdgcn_readlane(pages, slot - slot0)) * page_size + in_page;
        in_page += step;
        while (in_page >= page_size) in_page -= page_size, ++slot;
        return r;
    }
};

__device__ __forceinline__ void load_q(const Fav4PagedArgs& pg, int tok, int head, int half, bf16x8 (&qr)[8]) {
    const char* qp = static_cast<const char*>(pg.q) + (int64_t(tok) * pg.heads + head) * ROW_BYTES + half * 16;
#pragma unroll
    for (int c = 0; c < 8; ++c) qr[c] = *reinterpret_cast<const bf16x8*>(qp + c * 32);
}

__device__ __forceinline__ void clear(RowState& st) {
#pragma unroll
    for (int db = 0; db < 4; ++db) st.o[db] = f32x16{};
    st.m = -__builtin_inff();
    st.lb = 0.f;
    st.l = 0.f;
}

// The keys that rows [first, last] of a family see: the last one of the row of
// token `tok` (a lane's own); all rows see those of the family's keys below
// `plain`, and none sees any from `end` on.
struct Visible {
    int lim, plain, end;
};
template <bool OWN, class B>
__device__ __forceinline__ Visible visible(const B& x, const PrefixPlan& pl, const Family& f, int idx, int first,
                                           int last, int tok) {
    if constexpr (OWN) {
        if (!pl.br) return {f.k1 - 1, uniform(f.k1), uniform(f.k1)};
        const int shift = f.k1 - f.tokens;                             // last visible key of query 0
        const int i0 = pl.by_group(first), i1 = pl.by_group(last);
        const int k0 = max(f.k0, 0);
        return {shift + tok - f.t0, uniform(max(k0, min(f.k1, shift + i0 + 1))),
                uniform(max(k0, min(f.k1, shift + i1 + 1)))};
    } else {
        if (!x.hidden) return {INT_MAX, uniform(f.k1), uniform(f.k1)};
        // The last of the prefix's sequences that starts at or before tok.
        int lo = x.first_seq(idx), hi = max(x.first_seq(idx + 1), lo + 1);
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (x.cu(mid) <= tok) lo = mid;
            else hi = mid;
        }
        return {x.keys(lo) - (pl.br ? x.cu(lo + 1) - tok : 1), 0, uniform(f.k1)};
    }
}

// The partial rows of one wave's 32 rows (`live` of them exist), to partial row prow on.
template <bool LSE, int TILE_BYTES>
__device__ __forceinline__ void store_parts(const RowState& st, const PrefixPlan& pl, int64_t prow, int live,
                                            unsigned char* smem, uint32_t slot, int lane) {
    if (live <= 0) return;
    const rsrc_t rp = make_rsrc(pl.o_part + prow * D, uint32_t(live) * D * 4);
    const float inv = st.lb > 0.f ? 1.f / st.lb : 0.f;
    store_part_rows<TILE_BYTES, true>(st, inv, smem, slot, rp, 0, live, lane);
    if (lane < 32 && lane < live) {
        const float sb = st.m + __builtin_amdgcn_logf(st.lb);
        reinterpret_cast<float2*>(pl.lse_part)[prow + lane] =
            float2{sb, LSE ? st.m + __builtin_amdgcn_logf(st.l) : sb};
    }
}

// The segments of the range [g0, g0 + per) of a line, each by WAVES waves that
// share its key tiles: prefixes (OWN false) or sequences.  aligned: the units
// of a segment of the line's only family, a multiple of per (0: seg_cost).
template <bool LSE, int WAVES, bool OWN, int BN, int STAGES, class B, class L>
__device__ __forceinline__ void attend_shared(const B& x, const PrefixPlan& pl, const L& line,
                                              const typename L::Sums& head, int range, int per, int aligned, int kvh,
                                              unsigned char* smem) {
    constexpr int BM = WAVES * 32, AHEAD = STAGES - 1;         // prefetch distance in tiles
    constexpr int TILE_BYTES = BN * ROW_BYTES, STAGE_BYTES = 2 * TILE_BYTES;
    constexpr int DMA = BN / 4 / WAVES, SLAB = DMA * 4;        // this wave's key rows of a tile
    static_assert(DMA >= 2, "a wave's DMA slots hold 2 KiB per matrix (O staging)");
    static_assert(32 % SLAB == 0, "a wave's rows of a tile lie in one page");
    const Fav4PrefixArgs& a = x.a;
    const Fav4PagedArgs& pg = a.paged;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5, group = line.group;
    const uint32_t kv_row_bytes = uint32_t(pg.kv_heads) * ROW_BYTES;
    const float scale2 = pg.scale * LOG2E;
    const uint32_t smem_base = lds_addr(smem);
    const int g0 = range * per, g1 = g0 + per;

    const LdsOffsets off = lds_offsets(lane);
    DmaOffsets<DMA> dofs;
#pragma unroll
    for (int i = 0; i < DMA; ++i) {
        const int in_slab = i * 4 + (lane >> 4), r = wave * SLAB + in_slab, p = lane & 15;
        dofs.k[i] = in_slab * kv_row_bytes + ((p ^ k_swz(r)) << 4);
        dofs.v[i] = in_slab * kv_row_bytes + ((p ^ v_swz(r)) << 4);
    }
    typename L::Place at = aligned ? typename L::Place{0, 0, 0} : line.find(g0, lane, head);
    for (; at.idx < line.count && at.base < g1; ++at.idx) {
        const Family f = line.family(at.idx);
        const int t0 = uniform(f.t0), tokens = uniform(f.tokens), k0 = uniform(max(f.k0, 0)), k1 = uniform(f.k1);
        const int tiles = uniform(line.tiles(f)), ktiles = uniform(line.key_tiles(f)),
                  seg_cost = aligned ? aligned : uniform(line.seg_cost(f));
        const int rows = tokens * group;
        // The first row tile whose units reach past g0 (bad offsets may overlap the
        // families and overflow the line: every index stays in bounds all the same).
        for (int rt = at.base < g0 && tiles > 1 ? udiv(max(0, g0 - at.base), seg_cost) : 0; rt < tiles; ++rt) {
            const int first = at.base + (rt + 1) * seg_cost - max(ktiles, 1);     // unit of its first key tile
            if (first >= g1) break;
            if (first + max(ktiles, 1) <= g0) continue;
            const int a0 = max(0, g0 - first), a1 = min(ktiles, g1 - first);
            const int q0 = rt * BM, qw = q0 + wave * 32, row = qw + col;
            const int srow = min(row, rows - 1);
            const int trow = pl.by_group(srow), tok = t0 + trow, qhead = kvh * group + srow - trow * group;

            const Visible see = visible<OWN>(x, pl, f, at.idx, q0, min(rows, q0 + BM) - 1, tok);
            const int plain = see.plain, end = see.end, lim = see.lim;
            const int nfull = max(0, plain - k0) / BN;
            const int e1 = min(a1, (end - k0 + BN - 1) / BN);          // past what any row sees: nothing to do

            RowState st;
            clear(st);
            if (a0 < e1) {
                PageWalk walk{nullptr, 0, pg.page_size, pg.num_pages};
                const int key0 = k0 + a0 * BN + wave * SLAB;           // this wave's first key row
                if constexpr (OWN)
                    walk.start(pg.block_table + int64_t(at.idx) * pg.max_pages_per_seq, pg.max_pages_per_seq, key0,
                               pl.by_page, lane);
                else
                    walk.start(a.prefix_table + int64_t(at.idx) * a.max_pages_per_prefix, a.max_pages_per_prefix,
                               key0, pl.by_page, lane);
                bf16x8 qr[8];
                load_q(pg, tok, qhead, half, qr);
                // Q and the pages have landed before the first tile is asked for, so that
                // the loop's only outstanding loads are its tiles.  (Q through LDS, between
                // the first two tiles, was 1.7% slower over 32 cases.)
#pragma unroll
                for (int c = 0; c < 8; ++c) asm volatile("" ::"v"(qr[c]));
                asm volatile("" ::"v"(walk.pages));
                // Tiles past the last one read nothing (the descriptors' bound is 0) and land
                // in a stage that no later step reads, which keeps the vmcnt count uniform.
                auto issue = [&](int t, int stage) {
                    const int left = t < e1 ? min(k1 - (k0 + t * BN + wave * SLAB), SLAB) : 0;
                    const uint32_t bytes = left > 0 ? uint32_t(left - 1) * kv_row_bytes + ROW_BYTES : 0u;
                    const int64_t byte = t < e1 ? (walk.row(BN, lane) * pg.kv_heads + kvh) * ROW_BYTES : 0;
                    const u32x4 rk = make_desc(static_cast<const char*>(pg.k_cache) + byte, bytes);
                    const u32x4 rv = make_desc(static_cast<const char*>(pg.v_cache) + byte, bytes);
                    dma_tile<DMA, TILE_BYTES>(rk, rv, smem_base + stage * STAGE_BYTES, wave, dofs);
                };
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) issue(a0 + i, i);
                const bool idle = qw >= rows;                          // all of this wave's rows are past the family's
                int t = a0, stage = 0;
                auto steps = [&](auto masked_c, int to) {
                    for (; t < to; ++t) {
                        const unsigned char* cur = smem + stage * STAGE_BYTES;
                        wait_vmem_keep<2 * DMA * (AHEAD - 1)>();
                        __syncthreads();
                        issue(t + AHEAD, stage == 0 ? AHEAD : stage - 1);
                        if (!idle)
                            attend_fused<BN, decltype(masked_c)::value, true, LSE, true>(
                                cur, cur + TILE_BYTES, off, qr, st, t == a0, k0 + t * BN, k1, lim, half, scale2);
                        stage = stage == STAGES - 1 ? 0 : stage + 1;
                    }
                };
                steps(std::integral_constant<bool, false>{}, min(e1, nfull));
                steps(std::integral_constant<bool, true>{}, e1);
                // The prefetches past the end have landed, and every wave has read its last
                // tile, before any stages O or loads the next segment's first one.
                wait_vmem();
                __syncthreads();
            }
            // The part's partial rows, and the segment's notes.
            const int block = at.seg + rt + range;
            const int stride = OWN ? pl.own_rows : BM, blocks = OWN ? pl.own_blocks : pl.prefix_blocks;
            const int live = min(min(32, stride - wave * 32), rows - qw);      // of this wave's rows
            if (ktiles > 0 && uint32_t(block) < uint32_t(blocks)) {
                const int64_t prow = (OWN ? int64_t(pg.kv_heads) * pl.prefix_blocks * BM : 0) +
                                     (int64_t(kvh) * blocks + block) * stride + wave * 32;
                store_parts<LSE, TILE_BYTES>(st, pl, prow, live, smem, wave * DMA * 1024, lane);
            }
            if (kvh == 0 && first >= g0 && lane < 32 && lane < live) {
                const int parts = ktiles > 0 ? udiv(first + ktiles - 1, per) - range + 1 : 0;
                int2* note = pl.notes + (int64_t(t0) * group + row) * 2;
                note[OWN] = int2{block * stride + wave * 32 + lane, parts};
                if (OWN && uniform(f.k0) < 0) note[0] = int2{0, 0};
            }
            // The staging has been read (its values were stored) before this wave's
            // next copy into its slots.
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        at.base += tiles * seg_cost;
        at.seg += tiles;
    }
}

// A part of a segment of up to 32 rows, by single waves: wave `turn` of every
// `step` waves takes the part's key tiles a0 + turn, a0 + turn + step, ... below
// e1, 32 keys each, through 16 KiB of LDS of its own at `slot`, with no barrier.
template <bool LSE>
__device__ __forceinline__ void attend_tiles(const Fav4PagedArgs& pg, const int* table, int entries,
                                             const FastDiv& by_page, int t, int step, int e1, int nfull, int k0, int k1,
                                             int lim, int tok, int qhead, int kvh, uint32_t kv_row_bytes, float scale2,
                                             const LdsOffsets& off, const DmaOffsets<8>& dofs, unsigned char* smem,
                                             uint32_t slot, RowState& st, int lane) {
    constexpr int BN = 32, TILE_BYTES = BN * ROW_BYTES, DMA = BN / 4;
    const int half = lane >> 5;
    PageWalk walk{nullptr, 0, pg.page_size, pg.num_pages};
    walk.start(table, entries, k0 + t * BN, by_page, lane);
    bf16x8 qr[8];
    load_q(pg, tok, qhead, half, qr);
#pragma unroll
    for (int c = 0; c < 8; ++c) asm volatile("" ::"v"(qr[c]));
    const uint32_t stage = lds_addr(smem) + slot;
    auto issue = [&](int at) {
        const int left = min(k1 - (k0 + at * BN), BN);
        const uint32_t bytes = uint32_t(left - 1) * kv_row_bytes + ROW_BYTES;
        const int64_t byte = (walk.row(BN * step, lane) * pg.kv_heads + kvh) * ROW_BYTES;
        const u32x4 rk = make_desc(static_cast<const char*>(pg.k_cache) + byte, bytes);
        const u32x4 rv = make_desc(static_cast<const char*>(pg.v_cache) + byte, bytes);
        dma_tile<DMA, TILE_BYTES, true>(rk, rv, stage, 0, dofs);
    };
    issue(t);
    const unsigned char* ks = smem + slot;
    bool first = true;
    auto tile = [&](auto masked_c) {
        wait_vmem();
        attend_fused<BN, decltype(masked_c)::value, true, LSE, true>(ks, ks + TILE_BYTES, off, qr, st, first,
                                                                     k0 + t * BN, k1, lim, half, scale2);
        // The tile has been read: the next one may land in its place.
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        first = false;
        t += step;
        if (t < e1) issue(t);
    };
    while (t < min(e1, nfull)) tile(std::integral_constant<bool, false>{});
    while (t < e1) tile(std::integral_constant<bool, true>{});
    wait_vmem();                                                       // (the last tile left none in flight)
}

// The segments of the range [g0, g0 + per) of the sequences' line by one wave.
// Neighbouring families are taken with neighbouring K/V heads: a wave that stays
// with one head reads one eighth of the memory channels, and some of them are
// slower (128 sequences of 64..4096 own keys behind 32768, H32 KVH8: the slowest
// head's tiles took 3.48 us, the fastest's 2.75; 159 -> 146 us for the call).
template <bool LSE, class B, class L>
__device__ __forceinline__ void attend_wave(const B& x, const PrefixPlan& pl, const L& line,
                                            const typename L::Sums& head, int range, int per, int turn,
                                            unsigned char* smem, uint32_t slot, int64_t part0) {
    constexpr int BN = 32, BM = 32, TILE_BYTES = BN * ROW_BYTES;
    const Fav4PagedArgs& pg = x.a.paged;
    const int lane = threadIdx.x & 63, col = lane & 31, group = line.group;
    const uint32_t kv_row_bytes = uint32_t(pg.kv_heads) * ROW_BYTES;
    const float scale2 = pg.scale * LOG2E;
    const int g0 = range * per, g1 = g0 + per, blocks = pl.own_blocks, stride = pl.own_rows;

    const LdsOffsets off = lds_offsets(lane);
    const DmaOffsets<8> dofs = dma_offsets<8>(0, lane, kv_row_bytes, kv_row_bytes);
    for (typename L::Place at = line.find(g0, lane, head); at.idx < line.count && at.base < g1; ++at.idx) {
        const Family f = line.family(at.idx);
        const int t0 = uniform(f.t0), tokens = uniform(f.tokens), k0 = uniform(max(f.k0, 0)), k1 = uniform(f.k1);
        const int tiles = uniform(line.tiles(f)), ktiles = uniform(line.key_tiles(f)), seg_cost = uniform(line.seg_cost(f));
        const int rows = tokens * group;
        const int kvh = uniform(turn + at.idx - pl.by_kv_heads(turn + at.idx) * pg.kv_heads);
        for (int rt = at.base < g0 && tiles > 1 ? udiv(max(0, g0 - at.base), seg_cost) : 0; rt < tiles; ++rt) {
            const int first = at.base + (rt + 1) * seg_cost - max(ktiles, 1);
            if (first >= g1) break;
            if (first + max(ktiles, 1) <= g0) continue;
            const int a0 = max(0, g0 - first), a1 = min(ktiles, g1 - first);
            const int q0 = rt * BM, row = q0 + col, srow = min(row, rows - 1);
            const int trow = pl.by_group(srow), tok = t0 + trow, qhead = kvh * group + srow - trow * group;
            const Visible see = visible<true>(x, pl, f, at.idx, q0, min(rows, q0 + BM) - 1, tok);
            const int nfull = max(0, see.plain - k0) / BN, e1 = min(a1, (see.end - k0 + BN - 1) / BN);

            RowState st;
            clear(st);
            if (a0 < e1)
                attend_tiles<LSE>(pg, pg.block_table + int64_t(at.idx) * pg.max_pages_per_seq, pg.max_pages_per_seq,
                                  pl.by_page, a0, 1, e1, nfull, k0, k1, see.lim, tok, qhead, kvh, kv_row_bytes, scale2,
                                  off, dofs, smem, slot, st, lane);
            const int block = at.seg + rt + range, live = min(min(32, stride), rows - q0);
            if (ktiles > 0 && uint32_t(block) < uint32_t(blocks))
                store_parts<LSE, TILE_BYTES>(st, pl, part0 + (int64_t(kvh) * blocks + block) * stride, live, smem, slot,
                                             lane);
            if (kvh == 0 && first >= g0 && lane < 32 && lane < live) {
                const int parts = ktiles > 0 ? udiv(first + ktiles - 1, per) - range + 1 : 0;
                int2* note = pl.notes + (int64_t(t0) * group + row) * 2;
                note[1] = int2{block * stride + lane, parts};
                if (uniform(f.k0) < 0) note[0] = int2{0, 0};
            }
            // The staging has been read (its values were stored) before the next copy.
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        at.base += tiles * seg_cost;
        at.seg += tiles;
    }
}

// The segments of the range [g0, g0 + per) of the prefixes' line where they have
// 32 rows: the workgroup's eight waves take the range's key tiles in turn, and join
// their parts in LDS (by the largest maximum of each row) before one is written.
// One wave a range writes eight times the parts, and a 64-key tile shared by
// eight waves, seven of them idle, takes 1.9 us where eight 32-key tiles take
// 2.7 (H32 KVH8, 4 rows a prefix: 64 sequences each behind its own 2048 keys
// 103 us by single waves, 132 shared, 97 split; 2 behind 8192 21.3, 18.8, 17.5).
template <bool LSE, class B, class L>
__device__ __forceinline__ void attend_split(const B& x, const PrefixPlan& pl, const L& line,
                                             const typename L::Sums& head, int range, int per, int turn,
                                             unsigned char* smem, float4 (&stats)[8][32]) {
    constexpr int WAVES = 8, BN = 32, BM = 32, SLOT = 2 * BN * ROW_BYTES;
    const Fav4PrefixArgs& a = x.a;
    const Fav4PagedArgs& pg = a.paged;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const int group = line.group;
    const uint32_t kv_row_bytes = uint32_t(pg.kv_heads) * ROW_BYTES;
    const float scale2 = pg.scale * LOG2E;
    const int g0 = range * per, g1 = g0 + per, blocks = pl.prefix_blocks;

    const LdsOffsets off = lds_offsets(lane);
    const DmaOffsets<8> dofs = dma_offsets<8>(0, lane, kv_row_bytes, kv_row_bytes);
    for (typename L::Place at = line.find(g0, lane, head); at.idx < line.count && at.base < g1; ++at.idx) {
        const Family f = line.family(at.idx);
        const int t0 = uniform(f.t0), tokens = uniform(f.tokens), k1 = uniform(f.k1);
        const int tiles = uniform(line.tiles(f)), ktiles = uniform(line.key_tiles(f)), seg_cost = uniform(line.seg_cost(f));
        const int rows = tokens * group;
        const int kvh = uniform(turn + at.idx - pl.by_kv_heads(turn + at.idx) * pg.kv_heads);
        for (int rt = at.base < g0 && tiles > 1 ? udiv(max(0, g0 - at.base), seg_cost) : 0; rt < tiles; ++rt) {
            const int first = at.base + (rt + 1) * seg_cost - max(ktiles, 1);
            if (first >= g1) break;
            if (first + max(ktiles, 1) <= g0) continue;
            const int a0 = max(0, g0 - first), a1 = min(ktiles, g1 - first);
            const int q0 = rt * BM, row = q0 + col, srow = min(row, rows - 1);
            const int trow = pl.by_group(srow), tok = t0 + trow, qhead = kvh * group + srow - trow * group;
            const Visible see = visible<false>(x, pl, f, at.idx, q0, min(rows, q0 + BM) - 1, tok);
            const int block = at.seg + rt + range, live = min(32, rows - q0);

            RowState st;
            clear(st);
            if (a0 + wave < a1)
                attend_tiles<LSE>(pg, a.prefix_table + int64_t(at.idx) * a.max_pages_per_prefix, a.max_pages_per_prefix,
                                  pl.by_page, a0 + wave, WAVES, a1, see.plain / BN, 0, k1, see.lim, tok, qhead, kvh,
                                  kv_row_bytes, scale2, off, dofs, smem, wave * SLOT, st, lane);
            // O by quads of 4 dims: quad q of a lane holds dims 32 (q / 4) + 8 (q % 4) +
            // 4 half of row col.  Wave w sums quads 2w and 2w + 1 of all waves.
            if (half == 0) stats[wave][col] = float4{st.m, st.lb, st.l, 0.f};
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                const f32x16& o = st.o[q >> 2];
                const int i = (q & 3) * 4;
                *reinterpret_cast<FAV4_LDS f32x4*>((FAV4_LDS void*)(smem + wave * SLOT + q * 1024 + lane * 16)) =
                    f32x4{o[i], o[i + 1], o[i + 2], o[i + 3]};
            }
            __syncthreads();
            float m = -__builtin_inff(), lb = 0.f, l = 0.f, weight[WAVES];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) m = fmaxf(m, weight[w] = stats[w][col].x);
            const float base = m == -__builtin_inff() ? 0.f : m;       // rows that see no key of the part
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                weight[w] = exp2_native(weight[w] - base);
                lb += weight[w] * stats[w][col].y;
                if constexpr (LSE) l += weight[w] * stats[w][col].z;
            }
            const float inv = lb > 0.f ? 1.f / lb : 0.f;
            if (ktiles > 0 && uint32_t(block) < uint32_t(blocks)) {
                const int64_t prow = (int64_t(kvh) * blocks + block) * BM;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int q = wave * 2 + i;
                    f32x4 sum{};
#pragma unroll
                    for (int w = 0; w < WAVES; ++w)
                        sum += weight[w] * *reinterpret_cast<const FAV4_LDS f32x4*>(
                                               (FAV4_LDS const void*)(smem + w * SLOT + q * 1024 + lane * 16));
                    if (col < live)
                        *reinterpret_cast<f32x4*>(pl.o_part + (prow + col) * D + (q >> 2) * 32 + (q & 3) * 8 + half * 4) =
                            sum * inv;
                }
                if (wave == 0 && lane < live) {
                    const float sb = base + __builtin_amdgcn_logf(lb);
                    reinterpret_cast<float2*>(pl.lse_part)[prow + lane] =
                        float2{sb, LSE ? base + __builtin_amdgcn_logf(l) : sb};
                }
            }
            if (wave == 0 && kvh == 0 && first >= g0 && lane < live) {
                const int parts = ktiles > 0 ? udiv(first + ktiles - 1, per) - range + 1 : 0;
                pl.notes[(int64_t(t0) * group + row) * 2] = int2{block * BM + lane, parts};
            }
            // Every wave has read the sums before the next segment's copies and statistics.
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __syncthreads();
        }
        at.base += tiles * seg_cost;
        at.seg += tiles;
    }
}

// How a call's lines are cut (by the host, from the sizes): MANY rows per
// sequence, both lines by whole workgroups; FEW, the prefixes' by workgroups
// and the sequences' own by waves; FEWEST (a prefix's rows, too, few), the same,
// with a prefix's keys split over the workgroup's waves.
enum Cut { MANY, FEW, FEWEST };

template <bool LSE, Cut CUT, bool CACHED>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))
void prefix_kernel(Fav4PrefixArgs a, PrefixPlan pl) {
    constexpr int WAVES = 8, BN = 64, STAGES = 4;                      // three tiles in flight
    constexpr bool OWN_WAVES = CUT != MANY, SPLIT = CUT == FEWEST;
    constexpr int BM = SPLIT ? 32 : WAVES * 32;                        // rows of a prefix segment
    constexpr int OWN_RANGES = OWN_WAVES ? WAVES : 1;                  // of a workgroup
    __shared__ __attribute__((aligned(1024))) unsigned char smem[STAGES * 2 * BN * ROW_BYTES];
    __shared__ PlanLds lds;
    static_assert(sizeof(smem) >= WAVES * 64 * ROW_BYTES, "a 32-key tile of K and V for each wave");
    const Fav4PagedArgs& pg = a.paged;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int w = uniform(pl.by_kv_heads(blockIdx.x)), kvh = uniform(int(blockIdx.x) - w * pg.kv_heads);
    const int group = pl.group;

    PrefixBatch<CACHED> x{a, pl, lds, true};
    if constexpr (CACHED) {
        // One round of loads for as many sequences as the workgroup has lanes.
        for (int i = threadIdx.x; i <= max(pg.batch, a.num_prefixes); i += WAVES * 64) {
            const int t0 = x.load_cu(min(i, pg.batch)), t1 = x.load_cu(min(i + 1, pg.batch));
            const int sk = x.load_keys(min(i, pg.batch - 1));
            const int first = x.load_first_seq(min(i, a.num_prefixes));
            const int prefix_keys = x.load_prefix_keys(min(i, a.num_prefixes - 1));
            if (i <= pg.batch) lds.own[i] = __builtin_bit_cast(int4, x.make_own(t0, t1, sk, 0));
            if (i <= a.num_prefixes) lds.first_seq[i] = first;
            if (i < a.num_prefixes) lds.prefix_keys[i] = prefix_keys;
        }
        __syncthreads();
        int hidden = 0;
        for (int i = threadIdx.x; i < max(pg.batch, a.num_prefixes); i += WAVES * 64) {
            if (i < pg.batch) {
                const int shared = x.find_shared(i), sk = lds.own[i].w, n = lds.own[i + 1].x - lds.own[i].x;
                if (shared > 0) lds.own[i].z = min(shared, sk);
                hidden |= shared > 0 && n > 0 && sk - (pl.br ? n : 1) < shared - 1;
            }
            if (i < a.num_prefixes) lds.prefix[i] = __builtin_bit_cast(int4, x.make_prefix(i));
        }
        x.hidden = __syncthreads_or(hidden);
    }
    using B = PrefixBatch<CACHED>;
    const Line<B, false, BM, SPLIT ? 32 : BN, SPLIT ? SPLIT_SEG_TILES : SEG_TILES> prefixes{x, a.num_prefixes, group};
    const Line<B, true, OWN_WAVES ? 32 : BM, OWN_WAVES ? 32 : BN, OWN_WAVES ? OWN_SEG_TILES : SEG_TILES> own{
        x, pg.batch, group};
    typename decltype(prefixes)::Sums prefix_head;
    typename decltype(own)::Sums own_head;
    const int prefix_units = prefixes.length(lane, prefix_head), own_units = own.length(lane, own_head);

    // The workgroups of either line, by what its tiles cost; the two kinds alternate,
    // so that the XCDs have both.
    const float cost = prefix_units * (SPLIT ? SPLIT_COST : OWN_WAVES ? PREFIX_COST : 1.f);
    int pw = min(max(int(cost / (cost + own_units) * pl.ranges + 0.5f), 1), pl.ranges - 1);
    if (prefix_units <= 0) pw = 0;
    // One prefix, a range or more for each row tile: the tiles are cut at the same
    // keys (the lead units take up the rest), so that they read them at the same time
    // and share them in L2, unless that leaves over a quarter of the workgroups idle
    // (H32 KVH8: 256 sequences behind 1024 keys 42.6 us alike, 45.8 not; 40 x 16 queries
    // behind 8192 114 not alike, 130 alike).
    int tiles = 0;
    if (a.num_prefixes == 1 && pw > 0) {
        tiles = uniform(prefixes.tiles(prefixes.family(0)));
        if (udiv(pw, tiles) * tiles * 4 < pw * 3) tiles = 0;
    }
    // w pw / ranges, exact: both factors are at most 1024.
    const float step = 1.f / pl.ranges;
    const int before = int((w * pw + 0.5f) * step);
    if (int(((w + 1) * pw + 0.5f) * step) > before) {
        if constexpr (SPLIT) {
            __shared__ float4 stats[WAVES][32];
            const int per = max(udiv_up(prefix_units, pw), MIN_SPLIT_TILES);
            attend_split<LSE>(x, pl, prefixes, prefix_head, before, per, kvh, smem, stats);
        } else {
            int per = max(udiv_up(prefix_units, pw), MIN_PREFIX_TILES), aligned = 0;
            if (tiles) {
                const int cost = uniform(prefixes.seg_cost(prefixes.family(0)));
                per = max(udiv_up(cost, udiv(pw, tiles)), MIN_PREFIX_TILES);
                aligned = udiv_up(cost, per) * per;
            }
            attend_shared<LSE, WAVES, false, BN, STAGES>(x, pl, prefixes, prefix_head, before, per, aligned, kvh, smem);
        }
    } else {
        const int ranges = (pl.ranges - pw) * OWN_RANGES, range = w - before;
        const int per = max(udiv_up(own_units, ranges), MIN_OWN_TILES);
        if constexpr (OWN_WAVES)
            attend_wave<LSE>(x, pl, own, own_head, range * WAVES + wave, per, kvh, smem, wave * 64 * ROW_BYTES,
                             int64_t(pg.kv_heads) * pl.prefix_blocks * BM);
        else
            attend_shared<LSE, WAVES, true, BN, STAGES>(x, pl, own, own_head, range, per, 0, kvh, smem);
    }
}

// Merge of a row's parts.  PER teams of 16 lanes share one row of one head, 8
// dims a lane; a team takes every PER-th part, NS at a time with all their loads
// in flight, and keeps the running maximum and sums of a softmax over the
// parts' log-sums.  Bound by the chain notes -> parts -> output, and by the rate
// at which waves start: few teams with many loads each, and rather than 32
// lanes a row.
template <int PER>
__global__ __launch_bounds__(256) void prefix_merge_kernel(Fav4PrefixArgs a, PrefixPlan pl, int bm) {
    constexpr int RPB = 16 / PER, NS = PER == 1 ? 4 : 8;
    __shared__ float4 red[16];
    __shared__ f32x4 red_o[16][32];
    const Fav4PagedArgs& pg = a.paged;
    const int grp = threadIdx.x >> 4, l16 = threadIdx.x & 15;
    const int slot = grp / PER, part = grp - slot * PER;
    const int group = pl.group;
    const uint32_t rows = uint32_t(pg.total_q) * uint32_t(pg.heads), blocks = (rows + RPB - 1) / RPB;
    for (uint32_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
        const uint32_t r = blk * RPB + slot;                   // token * heads + head
        const int tok = pl.by_heads(r), head = int(r - uint32_t(tok) * uint32_t(pg.heads));
        const int kvh = pl.by_group(head), hg = head - kvh * group;
        int first[2] = {}, n[2] = {};
        bool live = r < rows;
        if (live) {
            const int4 note = *reinterpret_cast<const int4*>(pl.notes + (int64_t(tok) * group + hg) * 2);
            live = tok >= pg.cu_seqlens_q[0] && tok < pg.cu_seqlens_q[pg.batch];
            // Clamped: bad offsets leave notes unwritten.
            first[0] = min(max(note.x, 0), pl.prefix_blocks * bm - 1);
            first[1] = min(max(note.z, 0), pl.own_blocks * pl.own_rows - 1);
            if (live) {
                n[0] = min(max(note.y, 0), pl.prefix_blocks - pl.by_bm(first[0]));
                n[1] = min(max(note.w, 0), pl.own_blocks - pl.by_own_rows(first[1]));
            }
        }
        const int total = n[0] + n[1];
        const int64_t at_p = int64_t(kvh) * pl.prefix_blocks * bm + first[0];
        const int64_t at_o = int64_t(pg.kv_heads) * pl.prefix_blocks * bm + int64_t(kvh) * pl.own_blocks * pl.own_rows +
                             first[1];
        float mb = -__builtin_inff(), ml = mb, den = 0.f, suml = 0.f;
        f32x4 acc[2] = {};
        for (int c0 = part; c0 < total; c0 += PER * NS) {
            // Loads past the last part repeat it, with weight 0: no branch between the loads.
            float2 v[NS];
            f32x4 xo[NS][2];
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const int c = min(c0 + i * PER, total - 1);
                const int64_t row = c < n[0] ? at_p + int64_t(c) * bm : at_o + int64_t(c - n[0]) * pl.own_rows;
                v[i] = reinterpret_cast<const float2*>(pl.lse_part)[row];
                const f32x4* o = reinterpret_cast<const f32x4*>(pl.o_part + row * D + l16 * 8);
                xo[i][0] = o[0], xo[i][1] = o[1];
            }
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (c0 + i * PER >= total) v[i] = float2{-__builtin_inff(), -__builtin_inff()};
            float nb = mb, nl = ml;
#pragma unroll
            for (int i = 0; i < NS; ++i) nb = fmaxf(nb, v[i].x), nl = fmaxf(nl, v[i].y);
            if (nb == -__builtin_inff()) {
                // Parts without a visible key, or of a query that is no number: its log-sums
                // are none either (maxima pass over them), and so are then O and the LSE.
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    if (v[i].x != v[i].x) den = suml = __builtin_nanf("");
                continue;
            }
            const float keep = exp2_native(mb - nb);
            acc[0] *= keep, acc[1] *= keep;
            den *= keep;
            suml *= exp2_native(ml - nl);
            mb = nb, ml = nl;
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const float wgt = exp2_native(v[i].x - mb);
                if (wgt != 0.f) acc[0] += wgt * xo[i][0], acc[1] += wgt * xo[i][1];
                den += wgt;
                suml += exp2_native(v[i].y - ml);
            }
        }
        if constexpr (PER > 1) {
            if (l16 == 0) red[grp] = float4{mb, ml, den, suml};
            red_o[grp][l16 * 2] = acc[0], red_o[grp][l16 * 2 + 1] = acc[1];
            __syncthreads();
#pragma unroll
            for (int p = 0; p < PER; ++p) mb = fmaxf(mb, red[slot * PER + p].x), ml = fmaxf(ml, red[slot * PER + p].y);
            den = suml = 0.f;
            acc[0] = acc[1] = f32x4{};
#pragma unroll
            for (int p = 0; p < PER; ++p) {
                const float4 o = red[slot * PER + p];
                if (o.z == 0.f) continue;                      // no part with a visible key
                const float wgt = exp2_native(o.x - mb);
                den += wgt * o.z;
                suml += exp2_native(o.y - ml) * o.w;
                acc[0] += wgt * red_o[slot * PER + p][l16 * 2], acc[1] += wgt * red_o[slot * PER + p][l16 * 2 + 1];
            }
            __syncthreads();
        }
        if (!live || part != 0) continue;
        // No key in any part: O = 0, LSE = -inf.
        const float rden = den == 0.f ? 0.f : 1.f / den;
        bf16x8 y;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __bf16(acc[i >> 2][i & 3] * rden);
        *reinterpret_cast<bf16x8*>(static_cast<char*>(pg.o) + int64_t(r) * ROW_BYTES + l16 * 16) = y;
        if (pg.lse && l16 == 0) pg.lse[int64_t(head) * pg.total_q + tok] =
            den == 0.f ? -__builtin_inff() : (ml + __builtin_amdgcn_logf(suml)) * LN2;
    }
}

}  // namespace fav4
