// Kernels of the serving operators on paged K/V caches: appending new tokens
// with their position rotation, and attention behind shared prefixes.
#pragma once
#include "fav4_serving.h"
#include "bshd_kernel.hpp"

namespace fav4 {

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

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
// loads: offsets -> key count and table entry -> angles -> store; the rows
// themselves are loaded ahead of it.
// ---------------------------------------------------------------------------
template <bool INTERLEAVED>
__global__ __launch_bounds__(256) void append_kernel(Fav4AppendArgs a, int units, int64_t total) {
    const int lane = threadIdx.x & 63, j = lane & 7;
    const int64_t stride = int64_t(gridDim.x) * 4;
    const int qheads = a.q ? a.heads : 0, rows = qheads + 2 * a.kv_heads;
    const int half = a.rotary_dim >> 4;                    // granules of half the rotated dims
    for (int64_t id = int64_t(blockIdx.x) * 4 + uniform(threadIdx.x >> 6); id < total; id += stride) {
        const int t = uniform(int(id / units)), unit = uniform(int(id - int64_t(t) * units));
        const int row = unit * 8 + (lane >> 3);
        const bool live = row < rows, is_q = row < qheads, is_v = row >= qheads + a.kv_heads;
        const int head = is_q ? row : is_v ? row - qheads - a.kv_heads : row - qheads;
        const char* src = static_cast<const char*>(is_q ? a.q : is_v ? a.v : a.k);
        src += (int64_t(t) * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride) + int64_t(head) * D) * 2;
        // This lane's granules of the row.
        const bool turn = INTERLEAVED ? j < half : j < half;
        const int g0 = INTERLEAVED ? 2 * j : turn ? j : 2 * half + 2 * (j - half);
        const int g1 = INTERLEAVED ? g0 + 1 : turn ? j + half : g0 + 1;
        bf16x8 x{}, y{};
        if (live) {
            x = *reinterpret_cast<const bf16x8*>(src + g0 * 16);
            y = *reinterpret_cast<const bf16x8*>(src + g1 * 16);
        }
        const int b = wave_find(a.cu_seqlens_q, a.batch, t, lane);
        if (b >= a.batch || t < a.cu_seqlens_q[0]) continue;           // behind the last sequence
        const int64_t slot = int64_t(a.seqlens_k[b]) - a.cu_seqlens_q[b + 1] + t;
        const int64_t slots = int64_t(a.max_pages_per_seq) * a.page_size;
        int page = -1, in_page = 0;
        if (slot >= 0 && slot < slots) {
            const int at = int(slot / a.page_size);
            in_page = int(slot - int64_t(at) * a.page_size);
            page = a.block_table[int64_t(b) * a.max_pages_per_seq + at];
        }
        const bool stored = page >= 0 && page < a.num_pages;
        if (half > 0 && turn && !is_v && live) {
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
// tile of BM rows of one prefix against the prefix's keys, or of one sequence
// against the sequence's own keys; it costs its key tiles and SEG_TILES more,
// laid before them, for what its start and end cost.  The segments of a K/V
// head, prefixes first, are laid end to end and cut into ranges of one length,
// one per workgroup, whatever segments they cross.
//
// A segment's part that lies in range w writes its O (normalised, FP32) and two
// log-sums (log2: of the BF16 weights, and of the FP32 ones) to partial block
// (segment + w) of its kind: segments and ranges both only grow along the line,
// so no two parts have the same sum, and the blocks number segments + ranges.
// The part that holds a segment's first key tile also notes for each of its rows
// where its partials start and how many there are; prefix_merge_kernel goes by
// those notes.
// ---------------------------------------------------------------------------
struct PrefixPlan {
    float *o_part, *lse_part;         // prefix blocks of all K/V heads (BM rows each), then own blocks (own_rows each)
    int2* notes;                      // [total_q * group][2]: first partial row and parts, prefix and own
    int ranges, min_tiles;            // ranges of a K/V head; shortest range
    int prefix_blocks, own_blocks;    // partial blocks of a K/V head
    int own_rows;                     // rows of an own block
    int br;                           // bottom-right causal
};

// Tokens, rows and key tiles of one segment family: a prefix or a sequence.
struct Family {
    int t0, tokens;                   // first token, tokens
    int k0, k1;                       // keys [k0, k1)
};

// Prefix p's sequences [s0, s1) and keys.
struct PrefixSpan {
    int s0, s1, keys;
};
__device__ __forceinline__ PrefixSpan prefix_span(const Fav4PrefixArgs& a, int p) {
    const int n = a.paged.batch, page = a.paged.page_size;
    const int s0 = min(max(a.cu_prefix_seqs[p], 0), n), s1 = min(max(a.cu_prefix_seqs[p + 1], s0), n);
    const int most = int(min(int64_t(a.max_pages_per_prefix) * page, int64_t(a.paged.max_seqlen_k)));
    return {s0, s1, min(max(a.prefix_lens[p], 0), most) / page * page};
}
__device__ __forceinline__ int clamp_token(const Fav4PrefixArgs& a, int x) { return min(max(x, 0), a.paged.total_q); }

__device__ __forceinline__ Family prefix_family(const Fav4PrefixArgs& a, int p) {
    const PrefixSpan s = prefix_span(a, p);
    const int t0 = clamp_token(a, a.paged.cu_seqlens_q[s.s0]), t1 = max(t0, clamp_token(a, a.paged.cu_seqlens_q[s.s1]));
    return {t0, s.keys > 0 ? t1 - t0 : 0, 0, s.keys};
}
// Shared keys of sequence b.
__device__ __forceinline__ int shared_keys(const Fav4PrefixArgs& a, int b) {
    int lo = 0, hi = a.num_prefixes;                           // the last prefix that starts at or before b
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu_prefix_seqs[mid] <= b) lo = mid;
        else hi = mid;
    }
    const PrefixSpan s = prefix_span(a, lo);
    return s.s0 <= b && b < s.s1 ? s.keys : 0;
}
struct OwnFamily {
    Family f;
    int sq, sk, shared;
};
__device__ __forceinline__ OwnFamily own_family(const Fav4PrefixArgs& a, int b) {
    const int t0 = clamp_token(a, a.paged.cu_seqlens_q[b]);
    const int t1 = min(max(clamp_token(a, a.paged.cu_seqlens_q[b + 1]), t0), t0 + a.paged.max_seqlen_q);
    const int sk = min(max(a.paged.seqlens_k[b], 0), a.paged.max_seqlen_k), shared = shared_keys(a, b);
    return {{t0, t1 - t0, min(shared, sk), sk}, t1 - t0, sk, shared};
}

constexpr int SEG_TILES = 4;

template <bool LSE, int WAVES>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void prefix_kernel(Fav4PrefixArgs a, PrefixPlan pl) {
    constexpr int BN = 64, BM = WAVES * 32;
    constexpr int TILE_BYTES = BN * ROW_BYTES, STAGE_BYTES = 2 * TILE_BYTES;
    constexpr int DMA = BN / 4 / WAVES, SLAB = DMA * 4;        // this wave's key rows of a tile
    static_assert(DMA >= 2, "a wave's DMA slots hold 2 KiB per matrix (O staging)");
    static_assert(32 % SLAB == 0, "a wave's rows of a tile lie in one page");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * STAGE_BYTES];

    const Fav4PagedArgs& pg = a.paged;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int group = pg.heads / pg.kv_heads;
    const uint32_t kv_row_bytes = uint32_t(pg.kv_heads) * ROW_BYTES;
    const float scale2 = pg.scale * LOG2E;
    const uint32_t smem_base = lds_addr(smem);
    const int kvh = uniform(int(blockIdx.x) % pg.kv_heads), w = uniform(int(blockIdx.x) / pg.kv_heads);

    auto row_tiles = [&](int tokens) { return int((int64_t(tokens) * group + BM - 1) / BM); };
    auto cost = [&](const Family& f) { return row_tiles(f.tokens) * (max(1, (f.k1 - f.k0 + BN - 1) / BN) + SEG_TILES); };

    // The line: its length, and where the prefixes' part ends.
    int prefix_end = 0, prefix_segs = 0, total = 0;
    for (int p0 = 0; p0 < a.num_prefixes; p0 += 64) {
        Family f{};
        if (p0 + lane < a.num_prefixes) f = prefix_family(a, p0 + lane);
        prefix_end += wave_total(cost(f));
        prefix_segs += wave_total(row_tiles(f.tokens));
    }
    total = prefix_end;
    for (int b0 = 0; b0 < pg.batch; b0 += 64) {
        Family f{};
        if (b0 + lane < pg.batch) f = own_family(a, b0 + lane).f;
        total += wave_total(cost(f));
    }
    const int per = max((total + pl.ranges - 1) / pl.ranges, pl.min_tiles);
    if (int64_t(w) * per >= total) return;
    const int g0 = w * per, g1 = g0 + per;

    // The family that holds unit g0, the unit that it starts at and the
    // segments of its kind before it.
    bool own = g0 >= prefix_end;
    int idx = 0, base = own ? prefix_end : 0, seg0 = 0;
    {
        const int count = own ? pg.batch : a.num_prefixes;
        for (int i0 = 0; i0 < count; i0 += 64) {
            Family f{};
            if (i0 + lane < count) f = own ? own_family(a, i0 + lane).f : prefix_family(a, i0 + lane);
            const int c = cost(f), s = row_tiles(f.tokens), end = wave_scan(c), segs = wave_scan(s);
            const uint64_t hit = __builtin_amdgcn_ballot_w64(base + end > g0);
            if (hit) {
                const int l = __builtin_ctzll(hit);
                idx = i0 + l;
                base += __builtin_amdgcn_readlane(end - c, l);
                seg0 += __builtin_amdgcn_readlane(segs - s, l);
                break;
            }
            base += __builtin_amdgcn_readlane(end, 63);
            seg0 += __builtin_amdgcn_readlane(segs, 63);
        }
    }
    base = uniform(base), seg0 = uniform(seg0), idx = uniform(idx);

    const LdsOffsets off = lds_offsets(lane);
    DmaOffsets<DMA> dofs;
#pragma unroll
    for (int i = 0; i < DMA; ++i) {
        const int in_slab = i * 4 + (lane >> 4), r = wave * SLAB + in_slab, p = lane & 15;
        dofs.k[i] = in_slab * kv_row_bytes + ((p ^ k_swz(r)) << 4);
        dofs.v[i] = in_slab * kv_row_bytes + ((p ^ v_swz(r)) << 4);
    }

    for (;;) {
        // The next family that has rows, from idx on.
        const int count = own ? pg.batch : a.num_prefixes;
        if (idx >= count) {
            if (own) break;
            own = true, idx = 0, seg0 = 0, base = prefix_end;
            continue;
        }
        OwnFamily o{};
        if (own) o = own_family(a, idx);
        else o.f = prefix_family(a, idx);
        const int t0 = uniform(o.f.t0), tokens = uniform(o.f.tokens), k0 = uniform(o.f.k0), k1 = uniform(o.f.k1);
        const int sq = uniform(o.sq), sk = uniform(o.sk), shared = uniform(o.shared);
        const int tiles = row_tiles(tokens), ktiles = (k1 - k0 + BN - 1) / BN;
        const int seg_cost = max(1, ktiles) + SEG_TILES;
        const int rows = tokens * group;
        // The first row tile whose units reach past g0 (bad offsets may overlap the
        // families and overflow the line: every index stays in bounds all the same).
        int rt = base < g0 ? max(0, (g0 - base) / seg_cost) : 0;
        const PrefixSpan ps = own ? PrefixSpan{} : prefix_span(a, idx);
        const int s0 = uniform(ps.s0), s1 = uniform(ps.s1);
        for (; rt < tiles; ++rt) {
            const int first = base + rt * seg_cost + SEG_TILES;        // unit of its first key tile
            if (first >= g1) break;
            if (first + max(ktiles, 1) <= g0) continue;
            const int a0 = max(0, g0 - first), a1 = min(ktiles, g1 - first);
            const bool starts = first >= g0;
            const int q0 = rt * BM, qw = q0 + wave * 32, row = qw + col;
            const int srow = min(row, rows - 1);
            const int tok = t0 + srow / group, hg = srow - (srow / group) * group;

            // Visible keys: the last one of this lane's row; all rows of the tile see
            // those below `plain`, and none sees any from `end` on.
            int lim, plain, end = k1;
            if (own) {
                const int shift = pl.br ? sk - sq : sk - 1;            // last visible key of query 0
                const int i0 = q0 / group, i1 = min(rows - 1, q0 + BM - 1) / group;
                lim = pl.br ? shift + tok - t0 : shift;
                plain = min(k1, (pl.br ? shift + i0 : shift) + 1);
                end = min(k1, (pl.br ? shift + i1 : shift) + 1);
            } else {
                int low = INT_MAX;
                for (int b0 = s0; b0 < s1; b0 += 64) {
                    const int b = min(b0 + lane, s1 - 1);
                    const int n = max(0, pg.cu_seqlens_q[b + 1] - pg.cu_seqlens_q[b]);
                    const int keys = min(max(pg.seqlens_k[b], 0), pg.max_seqlen_k);
                    if (n > 0) low = min(low, pl.br ? keys - n : keys - 1);
                }
#pragma unroll
                for (int m = 32; m >= 1; m >>= 1) low = min(low, __shfl_xor(low, m));
                low = uniform(low);
                plain = min(k1, max(-1, low) + 1);
                lim = INT_MAX;
                if (plain < k1) {
                    // Some sequence has fewer keys than its prefix: each row's own limit.
                    int lo = s0, hi = s1;                              // the last sequence that starts at or before tok
                    while (hi - lo > 1) {
                        const int mid = (lo + hi) >> 1;
                        if (pg.cu_seqlens_q[mid] <= tok) lo = mid;
                        else hi = mid;
                    }
                    const int keys = min(max(pg.seqlens_k[lo], 0), pg.max_seqlen_k);
                    lim = pl.br ? keys - (pg.cu_seqlens_q[lo + 1] - tok) : keys - 1;
                }
            }
            plain = uniform(max(plain, k0)), end = uniform(max(end, k0));
            const int nfull = (plain - k0) / BN;
            const int e1 = min(a1, (end - k0 + BN - 1) / BN);          // past what any row sees: nothing to do

            RowState st;
#pragma unroll
            for (int db = 0; db < 4; ++db) st.o[db] = f32x16{};
            st.m = -__builtin_inff();
            st.lb = 0.f;
            st.l = 0.f;
            if (a0 < e1) {
                const int* table = own ? pg.block_table + int64_t(idx) * pg.max_pages_per_seq
                                       : a.prefix_table + int64_t(idx) * a.max_pages_per_prefix;
                const int entries = own ? pg.max_pages_per_seq : a.max_pages_per_prefix;
                int pages = 0, page0 = 0;                              // lane l holds the page of slot page0 + l
                auto load_pages = [&](int slot) {
                    page0 = slot;
                    pages = min(max(table[min(slot + lane, entries - 1)], 0), pg.num_pages - 1);
                };
                load_pages((k0 + a0 * BN + wave * SLAB) / pg.page_size);
                auto issue = [&](int t) {
                    const int key = k0 + t * BN + wave * SLAB;         // this wave's first key row of the tile
                    const int slot = key / pg.page_size, in_page = key - slot * pg.page_size;
                    if (slot - page0 >= 64) load_pages(slot);
                    const int64_t r0 =
                        int64_t(__builtin_amdgcn_readlane(pages, slot - page0)) * pg.page_size + in_page;
                    const int left = min(k1 - key, SLAB);
                    const uint32_t bytes = left > 0 ? uint32_t(left - 1) * kv_row_bytes + ROW_BYTES : 0u;
                    const int64_t at = (r0 * pg.kv_heads + kvh) * ROW_BYTES;
                    const u32x4 rk = make_desc(static_cast<const char*>(pg.k_cache) + at, bytes);
                    const u32x4 rv = make_desc(static_cast<const char*>(pg.v_cache) + at, bytes);
                    dma_tile<DMA, TILE_BYTES>(rk, rv, smem_base + ((t - a0) & 1) * STAGE_BYTES, wave, dofs);
                };
                issue(a0);
                bf16x8 qr[8];
                {
                    const char* qp = static_cast<const char*>(pg.q) +
                                     (int64_t(tok) * pg.heads + kvh * group + hg) * ROW_BYTES + half * 16;
#pragma unroll
                    for (int c = 0; c < 8; ++c) qr[c] = *reinterpret_cast<const bf16x8*>(qp + c * 32);
#pragma unroll
                    for (int c = 0; c < 8; ++c) asm volatile("" ::"v"(qr[c]));
                }
                const bool idle = qw >= rows;                          // all of this wave's rows are past the family's
                auto step = [&](auto stage_c, auto masked_c, int t) {
                    constexpr int STAGE = decltype(stage_c)::value;
                    constexpr bool MASKED = decltype(masked_c)::value;
                    const unsigned char* cur = smem + STAGE * STAGE_BYTES;
                    wait_vmem();
                    __syncthreads();
                    if (t + 1 < e1) issue(t + 1);
                    if (!idle)
                        attend_fused<BN, MASKED, true, LSE, true>(cur, cur + TILE_BYTES, off, qr, st, t == a0,
                                                                  k0 + t * BN, k1, lim, half, scale2);
                };
                using S0 = std::integral_constant<int, 0>;
                using S1 = std::integral_constant<int, 1>;
                using Plain = std::integral_constant<bool, false>;
                using Masked = std::integral_constant<bool, true>;
                int t = a0;
                for (; t + 1 < min(e1, nfull); t += 2) {
                    step(S0{}, Plain{}, t);
                    step(S1{}, Plain{}, t + 1);
                }
                for (; t + 1 < e1; t += 2) {
                    step(S0{}, Masked{}, t);
                    step(S1{}, Masked{}, t + 1);
                }
                if (t < e1) step(S0{}, Masked{}, t);
                // Every wave has read its last tile before any stages O or loads the
                // next segment's first one.
                __syncthreads();
            }
            // The part's partial rows, and the segment's notes.
            const int seg = seg0 + rt, block = seg + w;
            const int stride = own ? pl.own_rows : BM, blocks = own ? pl.own_blocks : pl.prefix_blocks;
            const int live = min(min(BM, stride), rows - q0);          // rows of the tile
            if (ktiles > 0 && uint32_t(block) < uint32_t(blocks)) {
                const int64_t prow0 = (own ? int64_t(pg.kv_heads) * pl.prefix_blocks * BM : 0) +
                                      (int64_t(kvh) * blocks + block) * stride;
                const rsrc_t rp = make_rsrc(pl.o_part + prow0 * D, uint32_t(live) * D * 4);
                const float inv = st.lb > 0.f ? 1.f / st.lb : 0.f;
                store_part_rows<TILE_BYTES, true>(st, inv, smem, wave * DMA * 1024, rp, wave * 32, live - wave * 32,
                                                  lane);
                if (half == 0 && wave * 32 + col < live) {
                    float* lp = pl.lse_part + (prow0 + wave * 32 + col) * 2;
                    const float sb = st.m + __builtin_amdgcn_logf(st.lb);
                    lp[0] = sb;
                    lp[1] = LSE ? st.m + __builtin_amdgcn_logf(st.l) : sb;
                }
            }
            if (kvh == 0 && starts && half == 0 && wave * 32 + col < live) {
                const int parts = ktiles > 0 ? (first + ktiles - 1) / per - first / per + 1 : 0;
                const int64_t r = int64_t(t0) * group + row;
                pl.notes[r * 2 + own] = int2{block * stride + wave * 32 + col, parts};
                if (own && shared == 0) pl.notes[r * 2] = int2{0, 0};
            }
            // The staging has been read (its values were stored) before this wave's
            // next copy into its slots.
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        base += tiles * seg_cost;
        seg0 += tiles;
        ++idx;
        if (base >= g1) break;
    }
}

// Merge: PER groups of 32 lanes share one (row, K/V head), 4 dims a lane.
template <int PER>
__global__ __launch_bounds__(256) void prefix_merge_kernel(Fav4PrefixArgs a, PrefixPlan pl, int bm) {
    constexpr int RPB = 8 / PER;
    __shared__ float2 red[8];
    __shared__ f32x4 red_o[8][32];
    const Fav4PagedArgs& pg = a.paged;
    const int grp = threadIdx.x >> 5, q4 = threadIdx.x & 31;
    const int slot = grp / PER, part = grp - slot * PER, team = part * 32 + q4;
    const int group = pg.heads / pg.kv_heads;
    const uint32_t rows = uint32_t(pg.total_q) * uint32_t(pg.heads), blocks = (rows + RPB - 1) / RPB;
    for (uint32_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
        const uint32_t r = blk * RPB + slot;                   // token * heads + head
        const int tok = int(r / uint32_t(pg.heads)), head = int(r - uint32_t(tok) * uint32_t(pg.heads));
        const int kvh = head / group, hg = head - kvh * group;
        const bool live = r < rows && tok >= pg.cu_seqlens_q[0] && tok < pg.cu_seqlens_q[pg.batch];
        int first[2] = {}, n[2] = {};
        if (live) {
            const int2* note = pl.notes + (int64_t(tok) * group + hg) * 2;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // Clamped: bad offsets leave notes unwritten.
                const int stride = i ? pl.own_rows : bm, last = (i ? pl.own_blocks : pl.prefix_blocks) * stride - 1;
                first[i] = min(max(note[i].x, 0), last);
                n[i] = min(max(note[i].y, 0), (last - first[i]) / stride + 1);
            }
        }
        const int total = n[0] + n[1];
        const int64_t at[2] = {int64_t(kvh) * pl.prefix_blocks * bm + first[0],
                               int64_t(pg.kv_heads) * pl.prefix_blocks * bm +
                                   int64_t(kvh) * pl.own_blocks * pl.own_rows + first[1]};
        auto row_of = [&](int c) {
            return c < n[0] ? at[0] + int64_t(c) * bm : at[1] + int64_t(c - n[0]) * pl.own_rows;
        };
        auto sums = [&](int c) { return *reinterpret_cast<const float2*>(pl.lse_part + row_of(c) * 2); };
        float mb = -__builtin_inff(), ml = mb;
        for (int c = team; c < total; c += PER * 32) {
            const float2 v = sums(c);
            mb = fmaxf(mb, v.x), ml = fmaxf(ml, v.y);
        }
        mb = max32(mb), ml = max32(ml);
        if constexpr (PER > 1) {
            if (q4 == 0) red[grp] = float2{mb, ml};
            __syncthreads();
#pragma unroll
            for (int p = 0; p < PER; ++p) mb = fmaxf(mb, red[slot * PER + p].x), ml = fmaxf(ml, red[slot * PER + p].y);
            __syncthreads();
        }
        // No key in any part: weights 2^-inf = 0, so O = 0 and LSE = -inf.
        if (mb == -__builtin_inff()) mb = ml = 0.f;
        float den = 0.f, suml = 0.f;
        for (int c = team; c < total; c += PER * 32) {
            const float2 v = sums(c);
            den += exp2_native(v.x - mb), suml += exp2_native(v.y - ml);
        }
        den = sum32(den), suml = sum32(suml);
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int c = part; c < total; c += PER) {
            const float wgt = exp2_native(sums(c).x - mb);
            const f32x4 x = *reinterpret_cast<const f32x4*>(pl.o_part + row_of(c) * D + q4 * 4);
            if (wgt > 0.f) acc += wgt * x;
        }
        if constexpr (PER > 1) {
            if (q4 == 0) red[grp] = float2{den, suml};
            red_o[grp][q4] = acc;
            __syncthreads();
            den = suml = 0.f;
            acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = 0; p < PER; ++p) {
                den += red[slot * PER + p].x, suml += red[slot * PER + p].y;
                acc += red_o[slot * PER + p][q4];
            }
            __syncthreads();
        }
        if (!live || part != 0) continue;
        const float rden = den > 0.f ? 1.f / den : 0.f;
        const f32x4 y = acc * rden;
        const f32x2 y0 = {y[0], y[1]}, y1 = {y[2], y[3]};
        const bf16x2 b0 = __builtin_convertvector(y0, bf16x2), b1 = __builtin_convertvector(y1, bf16x2);
        *reinterpret_cast<bf16x4*>(static_cast<char*>(pg.o) + int64_t(r) * ROW_BYTES + q4 * 8) =
            bf16x4{b0[0], b0[1], b1[0], b1[1]};
        if (pg.lse && q4 == 0) pg.lse[int64_t(head) * pg.total_q + tok] = (ml + __builtin_amdgcn_logf(suml)) * LN2;
    }
}

}  // namespace fav4
