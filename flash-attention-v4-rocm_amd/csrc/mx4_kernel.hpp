// Kernels of the operators of 4-bit (MXFP4) paged K/V caches: storing new tokens,
// reading rows back, and attention.
#pragma once
#include "fav4_mx4.h"
#include "serving_kernel.hpp"

namespace fav4 {

constexpr int MX4_CODES = D / 2, MX4_SCALES = D / 32;      // bytes of a cache row

// A scale byte's power of two; 255 makes NaN of whatever it scales.
__device__ __forceinline__ float mx4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }
constexpr uint32_t MX4_MOST = 252;                         // the largest scale of numbers

// Eight numbers (one dword of codes) times their block's scale: exact in BF16.
__device__ __forceinline__ bf16x8 mx4_values(uint32_t codes, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Whether one of four scales is above 252.  (Adding 3 to a byte's low seven bits carries
// into its top bit from 125 on.)
__device__ __forceinline__ bool mx4_no_numbers(uint32_t x) {
    return (((x & 0x7f7f7f7fu) + 0x03030303u) & x & 0x80808080u) != 0;
}

// ---------------------------------------------------------------------------
// Append.  The layout of append_kernel: one wave takes 8 of a token's heads + 2 *
// kv_heads rows (Q, then K, then V), 8 lanes a row, each with the two 16-byte
// granules whose dims are rotated together.  The four granules of a block of 32 dims
// then lie in up to four lanes, so the granules' largest magnitudes go through LDS
// (as bits, whose order is that of the magnitudes, infinities and NaN above them) and
// each lane reads its blocks' four.  Bound by memory (16 prompts of 500..4096, H32 KVH8,
// 626 MB: 128 us, 4.9 TB/s; 123 with all rows of a token a wave and streaming Q stores, but
// then 4 tokens take 3.6 in place of 3.2; 126 to 164 with one head of eight tokens a wave),
// for few tokens by the chain offsets -> table -> store.
// ---------------------------------------------------------------------------
// The block's scale byte (255: not all numbers are finite) from its largest
// magnitude's bits: the smallest e with max <= 1.75 * 2^(e + 2), i.e. the exponent,
// one more where the mantissa is above 0.75.
__device__ __forceinline__ int mx4_block_scale(u32x4 most) {
    const uint32_t m = max(max(most[0], most[1]), max(most[2], most[3]));
    return m >= 0x7f800000u ? 255 : min(max(int((m + 0x1fffffu) >> 23) - 2, 2), 252);
}
__device__ __forceinline__ uint32_t mx4_codes(const float (&x)[8], int scale) {
    const float inv = __uint_as_float(uint32_t(254 - scale) << 23);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0] * inv, x[1] * inv, 1.f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2] * inv, x[3] * inv, 1.f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4] * inv, x[5] * inv, 1.f, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6] * inv, x[7] * inv, 1.f, 3);
    return scale == 255 ? 0 : c;
}

// Products and sums rounded one by one: what is quantised does not depend on which of
// them the compiler would fuse.
__device__ __forceinline__ void mx4_turn(float& p, float& q, float c, float s) {
#pragma clang fp contract(off)
    const float u = p * c - q * s, w = q * c + p * s;
    p = u;
    q = w;
}

template <bool INTERLEAVED>
__global__ __launch_bounds__(256) void mx4_store_kernel(Fav4Mx4AppendArgs args, int units, int total,
                                                        FastDiv by_units, FastDiv by_page) {
    __shared__ __attribute__((aligned(16))) uint32_t most[4][8][16];
    const Fav4AppendArgs& a = args.append;
    const int lane = threadIdx.x & 63, j = lane & 7, wave = uniform(threadIdx.x >> 6);
    const int qheads = a.q ? a.heads : 0, rows = qheads + 2 * a.kv_heads;
    const int half = a.rotary_dim >> 4;                    // granules of half the rotated dims
    const int first = a.cu_seqlens_q[0], end = min(a.cu_seqlens_q[a.batch], a.total_q);
    for (int id = blockIdx.x; id < total; id += gridDim.x) {
        const int four = uniform(by_units(id)), unit = uniform(id - four * units), t = four * 4 + wave;
        if (t < first || t >= end) continue;               // in no sequence
        const int row = unit * 8 + (lane >> 3);
        const bool live = row < rows, is_q = row < qheads, is_v = row >= qheads + a.kv_heads;
        const int head = is_q ? row : is_v ? row - qheads - a.kv_heads : row - qheads;
        const char* src = static_cast<const char*>(is_q ? a.q : is_v ? a.v : a.k);
        src += (int64_t(t) * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride) + int64_t(head) * D) * 2;
        // This lane's granules of the row.
        const bool turn = j < half && !is_v;
        const int g0 = INTERLEAVED || !turn ? 2 * j : j;
        const int g1 = INTERLEAVED || !turn ? g0 + 1 : j + half;
        bf16x8 bx{}, by{};
        if (live) {
            bx = *reinterpret_cast<const bf16x8*>(src + g0 * 16);
            by = *reinterpret_cast<const bf16x8*>(src + g1 * 16);
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
        float x[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = float(bx[i]), y[i] = float(by[i]);
        if (turn && live) {
            const int64_t pos = a.positions ? int64_t(a.positions[t]) : slot;
            const int64_t r = min(max(pos, int64_t(0)), int64_t(a.rotary_rows - 1));
            const int64_t at = r * (half * 8) + j * 8;
            const f32x4* cp = reinterpret_cast<const f32x4*>(a.cos + at);
            const f32x4* sp = reinterpret_cast<const f32x4*>(a.sin + at);
            const f32x4 c[2] = {cp[0], cp[1]}, s[2] = {sp[0], sp[1]};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float ci = c[i >> 2][i & 3], si = s[i >> 2][i & 3];
                float& p = INTERLEAVED ? (i < 4 ? x : y)[2 * (i & 3)] : x[i];
                float& q = INTERLEAVED ? (i < 4 ? x : y)[2 * (i & 3) + 1] : y[i];
                mx4_turn(p, q, ci, si);
            }
        }
        if (is_q && live) {
            char* dst = static_cast<char*>(a.q_out) + (int64_t(t) * a.q_out_stride + int64_t(head) * D) * 2;
            bf16x8 u, w;
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = __bf16(x[i]), w[i] = __bf16(y[i]);
            *reinterpret_cast<bf16x8*>(dst + g0 * 16) = u;
            *reinterpret_cast<bf16x8*>(dst + g1 * 16) = w;
        }
        if (is_q || !live || !stored) continue;
        // The granules' largest magnitudes; the blocks' scales.  (A row's eight lanes
        // are here together; LDS takes a wave's accesses in order.)
        uint32_t m0 = 0, m1 = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m0 = max(m0, __float_as_uint(x[i]) & 0x7fffffffu);
            m1 = max(m1, __float_as_uint(y[i]) & 0x7fffffffu);
        }
        uint32_t* mine = most[wave][lane >> 3];
        mine[g0] = m0;
        mine[g1] = m1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const u32x4* blocks = reinterpret_cast<const u32x4*>(mine);
        const int s0 = mx4_block_scale(blocks[g0 >> 2]), s1 = mx4_block_scale(blocks[g1 >> 2]);
        const int own = mx4_block_scale(blocks[j & 3]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int64_t at = (int64_t(page) * a.kv_heads + head) * a.page_size + in_page;
        char* codes = static_cast<char*>(is_v ? a.v_cache : a.k_cache) + at * MX4_CODES;
        *reinterpret_cast<uint32_t*>(codes + g0 * 4) = mx4_codes(x, s0);
        *reinterpret_cast<uint32_t*>(codes + g1 * 4) = mx4_codes(y, s1);
        if (j < 4) static_cast<uint8_t*>(is_v ? args.v_scales : args.k_scales)[at * MX4_SCALES + j] = uint8_t(own);
    }
}

// ---------------------------------------------------------------------------
// Reading back.  One wave takes two neighbouring rows (tokens), or one where there are
// few: their sequences by one search and one look at the offsets behind it, their places
// in the caches in the wave's lanes, then K and V, 16 lanes a head's row (4 bytes of
// codes, 16 of BF16), 16 heads' rows with all their loads in flight.  Bound by memory:
// 256 of 324 bytes are written, past the caches (12 histories of up to 16384 keys H32/8,
// 268 MB: 44.4 us, 6.0 TB/s; 73.5 with ordinary stores; 45.1 with one row a wave, 45.3
// with four, 48.0 with eight); for few rows by the chain offsets -> table -> codes ->
// store (4 rows 3.1 us).
// ---------------------------------------------------------------------------
constexpr int MX4_READ_ROWS = 2;
__global__ __launch_bounds__(256) void mx4_read_kernel(Fav4Mx4GatherArgs a, FastDiv by_page, int each) {
    constexpr int U = 4;
    const int lane = threadIdx.x & 63, sub = lane >> 4, l16 = lane & 15;
    const int first = max(a.cu_seqlens_k[0], 0), end = min(a.cu_seqlens_k[a.batch], a.total_k);
    const int64_t step = int64_t(gridDim.x) * 4 * each;
    for (int64_t at = (int64_t(blockIdx.x) * 4 + uniform(threadIdx.x >> 6)) * each; at < end; at += step) {
        const int t0 = max(int(at), first), n = uniform(min(int(at) + each, end) - t0);
        if (n <= 0) continue;
        // Lane i: the sequence of row t0 + i, and its row of the caches (-1: in no page).
        const int b0 = wave_find(a.cu_seqlens_k, a.batch, t0, lane);
        const int next = a.cu_seqlens_k[min(b0 + 1 + lane, a.batch)];
        int b = b0;
        for (int i = 1; i < n; ++i) {
            const uint64_t past = __builtin_amdgcn_ballot_w64(b0 + 1 + lane <= a.batch && next <= t0 + i);
            const int here = past == ~0ull ? wave_find(a.cu_seqlens_k, a.batch, t0 + i, lane)
                                           : b0 + __builtin_popcountll(past);
            if (lane == i) b = here;
        }
        int64_t place = -1;
        if (lane < n && b < a.batch) {
            const int64_t slot = int64_t(t0) + lane - a.cu_seqlens_k[b] + (a.starts ? a.starts[b] : 0);
            if (slot >= 0 && slot < int64_t(a.max_pages_per_seq) * a.page_size && slot <= INT_MAX) {
                const int entry = by_page(int(slot));
                const int page = a.block_table[int64_t(b) * a.max_pages_per_seq + entry];
                if (page >= 0 && page < a.num_pages)
                    place = int64_t(page) * a.kv_heads * a.page_size + (int(slot) - entry * a.page_size);
            }
        }
        const int lo = int(place), hi = int(place >> 32);
        const int rows = 2 * a.kv_heads;
        for (int i = 0; i < n; ++i) {
            const int64_t base = int64_t(uint32_t(__builtin_amdgcn_readlane(lo, i))) |
                                 int64_t(__builtin_amdgcn_readlane(hi, i)) << 32;
            for (int row0 = 0; row0 < rows; row0 += 4 * U) {
                uint32_t codes[U] = {}, scale[U] = {};
                if (base >= 0) {
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int row = min(row0 + u * 4 + sub, rows - 1);         // past the last: it again
                        const bool is_v = row >= a.kv_heads;
                        const int64_t r = base + int64_t(is_v ? row - a.kv_heads : row) * a.page_size;
                        codes[u] = reinterpret_cast<const uint32_t*>(
                            static_cast<const char*>(is_v ? a.v_cache : a.k_cache) + r * MX4_CODES)[l16];
                        scale[u] = static_cast<const uint8_t*>(is_v ? a.v_scales : a.k_scales)[r * MX4_SCALES + (l16 >> 2)];
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int row = row0 + u * 4 + sub;
                    if (row >= rows) continue;
                    const bool is_v = row >= a.kv_heads;
                    char* dst = static_cast<char*>(is_v ? a.v : a.k) +
                                (int64_t(t0 + i) * (is_v ? a.v_stride : a.k_stride) +
                                 int64_t(is_v ? row - a.kv_heads : row) * D) * 2;
                    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, mx4_values(codes[u], mx4_scale(scale[u] > MX4_MOST ? 255u : scale[u]))),
                                                reinterpret_cast<u32x4*>(dst + l16 * 16));
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Attention.  Rows are (token, query head of the K/V head's group), r = token *
// group + head.  Sequences of up to 64 rows (decode, drafts), and of more where the call
// does not fill the GPU, go by mx4_decode_kernel, others by mx4_prefill_kernel.
// ---------------------------------------------------------------------------
// Sequences' row tiles and their key tiles lie end to end on a line, a few units more
// before each row tile for what its start and end cost, and the line is cut into equal
// ranges, one a workgroup of each K/V head.  A row tile whole in a range is finished
// there.  Of the others a range has at most two: one that began before it, whose part
// goes to the range's partial block 0, and one that ends behind it (block 1); they are
// merged by mx4_merge_kernel.
struct Mx4Plan {
    float *o_part, *lse_part;         // partial blocks of all K/V heads: two a range, of `stride` rows each
    int4* notes;                      // [ranges]: first row (token * group + head), rows and parts of the row tile whose
                                      // first part is the range's block 1 (no parts: there is none)
    int group;                        // query heads of a K/V head
    int ranges;                       // of a K/V head
    FastDiv by_kv_heads, by_group, by_page, by_merge;
    int stride, merge_chunks;         // rows of a partial block; workgroups of the merge for those that can be live
    int tiles;                        // row tiles that a sequence of few rows can have
    int br;                           // bottom-right causal
};
// The partial block of a row tile's part in range w.
__device__ __forceinline__ int mx4_block(int w, bool began_before) { return 2 * w + (began_before ? 0 : 1); }
// How far behind a row's first partial block its part c lies.
__device__ __forceinline__ int mx4_part(int c) { return c > 0 ? 2 * c - 1 : 0; }

// A sequence as read on the device, clamped.
struct Mx4Seq {
    int t0, tokens, keys;
};
__device__ __forceinline__ Mx4Seq mx4_seq(const Fav4PagedArgs& pg, int b) {
    const int t0 = min(max(pg.cu_seqlens_q[b], 0), pg.total_q), t1 = min(max(pg.cu_seqlens_q[b + 1], 0), pg.total_q);
    return {t0, min(max(t1 - t0, 0), pg.max_seqlen_q), min(max(pg.seqlens_k[b], 0), pg.max_seqlen_k)};
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// Over the four lanes that hold one row (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float quad_max(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return xhalf_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quad_sum(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return xhalf_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// ---- Few rows ---------------------------------------------------------------------
// A workgroup's waves all take the same NT * 16 rows, and every WAVES-th tile of SUB * 16
// keys of a part of the keys; they join in LDS.  Codes and scales are loaded straight into
// registers, each as soon as the one before has been used.
//  * S^T = K Q^T on 16x16x32 MFMAs: lane l has key l % 16 of a subtile and the block
//    of 32 dims l / 16, 16 bytes of codes and one scale; the four dwords of codes are
//    the four k-steps, whose order over the dims is free as long as Q's is the same.
//  * O^T += V^T P^T: P leaves the accumulators as the B operand, lane l / 16 = g
//    holding keys 4g + e of both subtiles of 32 keys.  V is converted as K is and goes
//    through LDS of the wave's own, from where ds_read_b64_tr_b16 reads it turned.  The
//    sums of the weights come from one more MFMA, against ones.
//  * The weights are rounded to BF16 for that product, as the forward's are, because FP32
//    MFMAs take 16 times as long and a second BF16 part of the weights twice: O is off by
//    0.0020 to 0.0023 of its size against 64 bits, with FP32 weights by 0.0017 (its own
//    rounding alone).  O is divided by the sum of the rounded ones; that, the LSE's sum and
//    all parts stay FP32.
//  * Keys are hidden by their scores, so V needs no other care than to be finite: a block
//    with a scale above 252 becomes 0 there, and its key's scores NaN by way of its K
//    scale.
// Bound by memory where the GPU is full (32 sequences of 4096..32768, H32 KVH8: 76 us, 6.4
// TB/s over the whole kernel), else by a wave's chain of conversions, products, softmax and
// LDS, 1.8 us for 64 keys.  Two or three tiles ahead, four waves a SIMD, V converted before
// the scores or read ahead of the softmax, rows of LDS padded by 32 bytes: no quicker.
template <int NT>
struct Mx4State {
    f32x4 o[NT][8], lb[NT];           // lb: sums of the BF16 weights, over all lanes
    float m[NT], l[NT];               // base (log2), sums of the FP32 weights of this lane's keys
};
template <int SUB>
struct Mx4Tile {
    u32x4 k[SUB], v[SUB];
    uint32_t ks[SUB], vs[SUB];
};

// P64: pages of a multiple of 64 keys, so that a tile lies in one.
template <int NT, int WAVES, int SUB, bool LSE, bool P64>
struct Mx4Decode {
    static constexpr int VROW = ROW_BYTES + 16, SLOT = 32 * VROW, BM = NT * 16, BN = SUB * 16;
    static_assert(BN == 64 || BN == 32, "tiles lie in a page of a multiple of 64 keys");
    const Fav4Mx4PagedArgs& a;
    const Mx4Plan& pl;
    unsigned char* smem;              // WAVES slots
    float4 (*stats)[16];              // [WAVES][16]
    int lane, wave;

    // Where this wave's tiles lie: the cache rows of the next 64 (with small pages: of the
    // subtiles of the next 64 / SUB) in the lanes.
    static constexpr int PIECES = P64 ? 1 : SUB, HELD = 64 / PIECES;
    struct Places {
        const int* table;
        int64_t head_row;             // of the head within a page
        int first, lo, hi;            // tile of lane 0; this lane's cache row
    };
    __device__ __forceinline__ void hold(Places& p, int t) const {
        const Fav4PagedArgs& pg = a.paged;
        p.first = t;
        const int key = min(t + lane / PIECES * WAVES, pg.max_seqlen_k / BN) * BN + lane % PIECES * 16;
        const int slot = pl.by_page(key), entry = p.table[min(slot, pg.max_pages_per_seq - 1)];
        const int page = min(max(entry, 0), pg.num_pages - 1);
        const int64_t row = int64_t(page) * pg.kv_heads * pg.page_size + p.head_row + (key - slot * pg.page_size);
        p.lo = int(row), p.hi = int(row >> 32);
    }
    // Of sequence b with head kvh, this wave's tiles from t on.
    __device__ __forceinline__ Places places(int b, int kvh, int t) const {
        Places p{a.paged.block_table + int64_t(b) * a.paged.max_pages_per_seq, int64_t(kvh) * a.paged.page_size, t};
        hold(p, t);
        return p;
    }
    struct Rows {
        int64_t at[PIECES];
    };
    __device__ __forceinline__ Rows rows(int t, Places& p) const {
        int e = uniform((t - p.first) / WAVES);
        if (e >= HELD) hold(p, t), e = 0;
        Rows r;
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
            r.at[i] = int64_t(uint32_t(__builtin_amdgcn_readlane(p.lo, e * PIECES + i))) |
                      int64_t(__builtin_amdgcn_readlane(p.hi, e * PIECES + i)) << 32;
        return r;
    }
    // Subtile i's first byte of a cache with `bytes` a row.
    __device__ __forceinline__ const char* at(const void* cache, const Rows& r, int i, int bytes) const {
        return static_cast<const char*>(cache) + (P64 ? r.at[0] * bytes + i * 16 * bytes : r.at[P64 ? 0 : i] * bytes);
    }
    __device__ __forceinline__ void load_k(Mx4Tile<SUB>& x, const Rows& r) const {
        const uint32_t code = uint32_t(lane & 15) * MX4_CODES + uint32_t(lane >> 4) * 16;
        const uint32_t scale = uint32_t(lane & 15) * MX4_SCALES + uint32_t(lane >> 4);
#pragma unroll
        for (int i = 0; i < SUB; ++i) {
            x.k[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at(a.paged.k_cache, r, i, MX4_CODES) + code));
            x.ks[i] = *reinterpret_cast<const uint8_t*>(at(a.k_scales, r, i, MX4_SCALES) + scale);
            x.vs[i] = *reinterpret_cast<const uint8_t*>(at(a.v_scales, r, i, MX4_SCALES) + scale);
        }
    }
    __device__ __forceinline__ void load_v(Mx4Tile<SUB>& x, const Rows& r, int i) const {
        const uint32_t code = uint32_t(lane & 15) * MX4_CODES + uint32_t(lane >> 4) * 16;
        x.v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at(a.paged.v_cache, r, i, MX4_CODES) + code));
    }

    // Tile t, in x; this wave's next tile is loaded in its place (behind the last one that
    // again: with the loads behind a branch the compiler could no longer tell how
    // many are under way, and would wait for the newest where it needs the oldest).
    __device__ __forceinline__ void tile(Mx4Tile<SUB>& x, const bf16x8 (&q)[NT][4], Mx4State<NT>& st, int t, int last, bool masked,
                                         const int (&lim)[NT], float scale2, Places& where) const {
        const int col = lane & 15, g = lane >> 4;
        const Rows r = rows(min(t + WAVES, last), where);
        uint32_t most = max(x.ks[0], x.vs[0]);
#pragma unroll
        for (int i = 1; i < SUB; ++i) most = max(most, max(x.ks[i], x.vs[i]));
        if (__builtin_amdgcn_ballot_w64(most > MX4_MOST)) {
#pragma unroll
            for (int i = 0; i < SUB; ++i) {
                const bool none = x.vs[i] > MX4_MOST;
                uint64_t keys_of = __builtin_amdgcn_ballot_w64(none);
                keys_of |= keys_of >> 32;
                keys_of |= keys_of >> 16;
                x.ks[i] = x.ks[i] > MX4_MOST || keys_of >> col & 1 ? 255u : x.ks[i];
                x.vs[i] = none ? 127u : x.vs[i];
                x.v[i] = none ? u32x4{} : x.v[i];
            }
        }
        uint32_t vb[SUB];
        f32x4 s[NT][SUB];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < SUB; ++i) {
                const bf16x8 kop = mx4_values(x.k[i][c], mx4_scale(x.ks[i]));
#pragma unroll
                for (int n = 0; n < NT; ++n) s[n][i] = mfma16(kop, q[n][c], c ? s[n][i] : f32x4{});
            }
#pragma unroll
        for (int i = 0; i < SUB; ++i) vb[i] = x.vs[i];
        load_k(x, r);
        bf16x8 p[NT][SUB / 2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (masked) {
                const int d = lim[n] - t * BN - 4 * g;
#pragma unroll
                for (int i = 0; i < SUB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][i][e] = i * 16 + e > d ? -__builtin_inff() : s[n][i][e];
            }
            float mx = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < SUB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[n][i][e]);
            // The base moves where a maximum passes it by more than the threshold.
            const float cand = fmaxf(st.m[n], quad_max(mx) * scale2);
            const bool update = cand > st.m[n] + RESCALE_THRESHOLD;
            if (__builtin_amdgcn_ballot_w64(update)) {
                const float now = update ? cand : st.m[n], alpha = update ? exp2_native(st.m[n] - now) : 1.f;
#pragma unroll
                for (int db = 0; db < 8; ++db) st.o[n][db] *= alpha;
                st.lb[n] *= alpha;
                st.l[n] *= alpha;
                st.m[n] = now;
            }
            const float base = st.m[n] == -__builtin_inff() ? 0.f : st.m[n];        // rows that have seen no key
#pragma unroll
            for (int h = 0; h < SUB / 2; ++h)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float w = exp2_native(fmaf(s[n][2 * h + (j >> 2)][j & 3], scale2, -base));
                    if constexpr (LSE) st.l[n] += w;
                    p[n][h][j] = __bf16(w);
                }
        }
        // V, 32 keys at a time.  Rows lie further apart than they are long: the 16 rows that
        // an access touches then start in different banks, and the offsets within a row are
        // constants.
        unsigned char* slot = smem + wave * SLOT;
        const __bf16 one(1.f);
        const bf16x8 ones{one, one, one, one, one, one, one, one};
#pragma unroll
        for (int h = 0; h < SUB / 2; ++h) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float scale = mx4_scale(vb[2 * h + i]);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    *reinterpret_cast<FAV4_LDS bf16x8*>((FAV4_LDS void*)(slot + (i * 16 + col) * VROW + (4 * g + c) * 16)) =
                        mx4_values(x.v[2 * h + i][c], scale);
            }
            load_v(x, r, 2 * h), load_v(x, r, 2 * h + 1);
#pragma unroll
            for (int n = 0; n < NT; ++n) st.lb[n] = mfma16(ones, p[n][h], st.lb[n]);
#pragma unroll
            for (int db = 0; db < 8; ++db) {
                const unsigned char* from = slot + (4 * g + (lane >> 2 & 3)) * VROW + (lane & 3) * 8 + db * 32;
                const bf16x4 lo = lds_read_tr(from), hi = lds_read_tr(from + 16 * VROW);
                const bf16x8 vop{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
                for (int n = 0; n < NT; ++n) st.o[n][db] = mfma16(vop, p[n][h], st.o[n][db]);
            }
        }
    }

    // Key tiles [a0, a1) of the rows from r0 on of sequence f with head kvh; this wave's, from a0 + wave on, lie
    // `where`.  split: the part is not all of the sequence's keys, and goes to partial block `block`.
    __device__ __forceinline__ void attend(const Mx4Seq& f, int r0, int kvh, Places& where, int a0, int a1, bool split,
                                           int block) const {
        const Fav4PagedArgs& pg = a.paged;
        const int col = lane & 15, g = lane >> 4, group = pl.group, live = f.tokens * group;
        const float scale2 = pg.scale * LOG2E;
        int lim[NT];
        bf16x8 q[NT][4];
        Mx4State<NT> st;
        const int shift = f.keys - f.tokens;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = min(r0 + n * 16 + col, live - 1), token = pl.by_group(row), head = kvh * group + row - token * group;
            lim[n] = pl.br ? min(shift + token, f.keys - 1) : f.keys - 1;
            const char* qp = static_cast<const char*>(pg.q) + (int64_t(f.t0 + token) * pg.heads + head) * ROW_BYTES + g * 64;
#pragma unroll
            for (int c = 0; c < 4; ++c) q[n][c] = *reinterpret_cast<const bf16x8*>(qp + c * 16);
#pragma unroll
            for (int db = 0; db < 8; ++db) st.o[n][db] = f32x4{};
            st.lb[n] = f32x4{};
            st.m[n] = -__builtin_inff();
            st.l[n] = 0.f;
        }
        // Tiles whose keys all rows see, and the end of those that some row sees.
        const int i0 = pl.by_group(r0), i1 = pl.by_group(min(live, r0 + BM) - 1);
        const int plain = pl.br ? max(0, min(f.keys, shift + i0 + 1)) : f.keys;
        const int seen = pl.br ? max(0, min(f.keys, shift + i1 + 1)) : f.keys;
        const int nfull = uniform(plain / BN), e1 = uniform(min(a1, (seen + BN - 1) / BN));
        int t = a0 + wave;
        if (t < e1) {
            const int last = t + (e1 - 1 - t) / WAVES * WAVES;             // of this wave
            Mx4Tile<SUB> x;
            const Rows r = rows(t, where);
            load_k(x, r);
#pragma unroll
            for (int i = 0; i < SUB; ++i) load_v(x, r, i);
            for (; t < e1; t += WAVES) tile(x, q, st, t, last, t >= nfull, lim, scale2, where);
        }
        // Join: row n's quad of dims 4u at u ^ n of its 512 bytes.
        unsigned char* slot = smem + wave * SLOT;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float lb = st.lb[n][0], l = LSE ? quad_sum(st.l[n]) : 0.f;
            if (n > 0) __syncthreads();
#pragma unroll
            for (int db = 0; db < 8; ++db)
                *reinterpret_cast<FAV4_LDS f32x4*>((FAV4_LDS void*)(slot + col * 512 + (((db * 4 + g) ^ col) << 4))) = st.o[n][db];
            if (g == 0) stats[wave][col] = float4{st.m[n], lb, l, 0.f};
            __syncthreads();
            for (int id = threadIdx.x; id < 512; id += WAVES * 64) {
                const int r = id >> 5, u = id & 31, row = r0 + n * 16 + r;
                if (row >= live) continue;
                float m = -__builtin_inff(), sb = 0.f, sl = 0.f;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) m = fmaxf(m, stats[w][r].x);
                const float base = m == -__builtin_inff() ? 0.f : m;
                f32x4 o{};
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
                    const float4 v = stats[w][r];
                    const float weight = exp2_native(v.x - base);
                    sb += weight * v.y;
                    sl += weight * v.z;
                    o += weight * *reinterpret_cast<const FAV4_LDS f32x4*>((FAV4_LDS const void*)(smem + w * SLOT + r * 512 + ((u ^ r) << 4)));
                }
                // (No key: 0; sums that are no numbers stay so.)
                o *= sb == 0.f ? 0.f : 1.f / sb;
                const int token = pl.by_group(row), head = kvh * group + row - token * group;
                if (!split) {
                    const bf16x4 y{__bf16(o[0]), __bf16(o[1]), __bf16(o[2]), __bf16(o[3])};
                    *reinterpret_cast<bf16x4*>(static_cast<char*>(pg.o) + (int64_t(f.t0 + token) * pg.heads + head) * ROW_BYTES + u * 8) = y;
                    if (LSE && u == 0)
                        pg.lse[int64_t(head) * pg.total_q + f.t0 + token] = (base + __builtin_amdgcn_logf(sl)) * LN2;
                } else {
                    const int64_t prow = (int64_t(kvh) * 2 * pl.ranges + block) * BM + n * 16 + r;
                    *reinterpret_cast<f32x4*>(pl.o_part + prow * D + u * 4) = o;
                    if (u == 0)
                        reinterpret_cast<float2*>(pl.lse_part)[prow] =
                            float2{base + __builtin_amdgcn_logf(sb), base + __builtin_amdgcn_logf(LSE ? sl : sb)};
                }
            }
        }
        __syncthreads();               // read: the next part may use the slots
    }
};

// What a row tile's start and end cost, in key tiles of 32 (64 with 32 rows): 64 sequences of
// 500..8192, H32 KVH8, 43.3 us, with 8 and 12 43.5; 4 of 100..2000 10.5, 10.6 and 10.8.
constexpr int MX4_LEAD = 10;

// One row tile of a sequence and one K/V head a workgroup (SPLIT false), or a range of
// the line.
template <int NT, int WAVES, int SUB, int EU, bool SPLIT, bool LSE, bool P64>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(EU, EU)))
void mx4_decode_kernel(Fav4Mx4PagedArgs a, Mx4Plan pl) {
    constexpr int BM = NT * 16, BN = SUB * 16;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[WAVES * Mx4Decode<NT, WAVES, SUB, LSE, P64>::SLOT];
    __shared__ float4 stats[WAVES][16];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const Fav4PagedArgs& pg = a.paged;
    const int w = uniform(pl.by_kv_heads(blockIdx.x)), turn = uniform(int(blockIdx.x) - w * pg.kv_heads);
    if constexpr (!SPLIT) {
        const int b = pl.tiles > 1 ? udiv(w, pl.tiles) : w, r0 = (w - b * pl.tiles) * BM;
        const Mx4Decode<NT, WAVES, SUB, LSE, P64> decode{a, pl, smem, stats, lane, wave};
        // (The table and the lengths load side by side.)
        auto where = decode.places(b, turn, wave);
        Mx4Seq f = mx4_seq(pg, b);
        f = {uniform(f.t0), uniform(f.tokens), uniform(f.keys)};
        if (r0 < f.tokens * pl.group) decode.attend(f, r0, turn, where, 0, (f.keys + BN - 1) / BN, false, 0);
    } else {
        auto tiles_of = [&](const Mx4Seq& f) { return int(uint32_t(f.tokens * pl.group + BM - 1) / BM); };
        auto cost_of = [&](const Mx4Seq& f) { return max(1, (f.keys + BN - 1) / BN) + MX4_LEAD; };
        // The units of 64 sequences from i on, in the lanes: of each, and up to and with it.
        auto sums = [&](int i) {
            Mx4Seq f{};
            if (i + lane < pg.batch) f = mx4_seq(pg, i + lane);
            const int c = tiles_of(f) * cost_of(f);
            return int2{c, wave_scan(c)};
        };
        const int2 head = sums(0);
        int units = __builtin_amdgcn_readlane(head.y, 63);
        for (int i = 64; i < pg.batch; i += 64) units += __builtin_amdgcn_readlane(sums(i).y, 63);
        const int per = max(udiv_up(units, pl.ranges), 1), g0 = w * per, g1 = g0 + per;
        // The sequence that holds unit g0, and the unit where it starts.
        int idx = 0, base = 0;
        for (int2 v = head;; v = sums(idx)) {
            const uint64_t hit = __builtin_amdgcn_ballot_w64(base + v.y > g0);
            if (hit) {
                const int l = __builtin_ctzll(hit);
                idx = uniform(idx + l);
                base = uniform(base + __builtin_amdgcn_readlane(v.y - v.x, l));
                break;
            }
            base += __builtin_amdgcn_readlane(v.y, 63);
            idx += 64;
            if (idx >= pg.batch) break;
        }
        int4 note{};
        for (; idx < pg.batch && base < g1; ++idx) {
            Mx4Seq f = mx4_seq(pg, idx);
            f = {uniform(f.t0), uniform(f.tokens), uniform(f.keys)};
            const int n = tiles_of(f), cost = cost_of(f), tiles = (f.keys + BN - 1) / BN;
            // Neighbouring sequences are taken with neighbouring heads, as in attend_wave.
            const int kvh = uniform(turn + idx - pl.by_kv_heads(turn + idx) * pg.kv_heads);
            for (int rt = 0; rt < n; ++rt, base += cost) {
                const int end = base + cost, first = end - max(tiles, 1);      // unit of the first key tile
                if (first >= g1 || end <= g0) continue;
                const bool before = first < g0, split = before || end > g1;
                const int block = mx4_block(w, before);
                const int a0 = max(0, g0 - first);
                // An opaque lane number, so that what follows from it is not kept from one row tile to the next.
                int own_lane = lane;
                asm volatile("" : "+v"(own_lane));
                const Mx4Decode<NT, WAVES, SUB, LSE, P64> decode{a, pl, smem, stats, own_lane, wave};
                auto where = decode.places(idx, kvh, a0 + wave);
                decode.attend(f, rt * BM, kvh, where, a0, min(tiles, g1 - first), split, block);
                if (split && !before)
                    note = int4{f.t0 * pl.group + rt * BM, min(BM, f.tokens * pl.group - rt * BM),
                                udiv(end - 1, per) - w + 1, 0};
            }
        }
        if (turn == 0 && threadIdx.x == 0) pl.notes[w] = note;
    }
}

// ---- Many rows --------------------------------------------------------------------
// Eight waves (or four) of 32 rows each share 64-key tiles of K and V, which they convert
// to BF16 on the way into LDS (two stages): the loop of the forward, attend_fused, behind
// another source.  A thread has 16 (32) dims of one key: 8 (16) bytes of codes and the key's
// four scales, loaded two tiles ahead.  Of the two waves of a SIMD that eight make one
// converts the next tile before its products and the other behind them, so that one's
// conversion runs beside the other's products; two workgroups of four do that unasked.
// Bound by the MFMAs and what the loop issues beside them: dense 8 x 2048 queries x 8192
// keys, H32 KVH8, 1104 to 1138 TFLOP/s by the card (BF16 caches 1158 to 1189).
constexpr int MX4_MANY_LEAD = 3;       // a row tile's start and end, in key tiles of 64
constexpr int MX4_LINE_TILES = 1024, MX4_LINE_SEQS = 512;      // of a batch that is cut into ranges

template <int WAVES, bool LSE>
struct Mx4Prefill {
    static constexpr int BM = WAVES * 32, BN = 64, TILE_BYTES = BN * ROW_BYTES;
    static constexpr int DWORDS = 16 / WAVES, KEYS = 64 / WAVES;       // of codes a thread, and of a wave
    const Fav4Mx4PagedArgs& a;
    const Mx4Plan& pl;
    unsigned char* smem;              // two stages of a K and a V tile
    int lane, wave;

    __device__ __forceinline__ int tiles_of(const Mx4Seq& f) const {
        return int(uint32_t(f.tokens * pl.group + BM - 1) / BM);
    }
    // Key tiles that some row of row tile rt sees.
    __device__ __forceinline__ int key_tiles(const Mx4Seq& f, int rt) const {
        const int last = pl.by_group(min(f.tokens * pl.group, (rt + 1) * BM) - 1);
        const int seen = pl.br ? max(0, min(f.keys, f.keys - f.tokens + last + 1)) : f.keys;
        return (seen + BN - 1) / BN;
    }

    // Key tiles [t, e1) of row tile rt of sequence b with head kvh; split as in Mx4Decode::attend.
    __device__ __forceinline__ void attend(int b, const Mx4Seq& f, int rt, int kvh, int t, int e1, bool split,
                                           int block) const {
        const Fav4PagedArgs& pg = a.paged;
        const int col = lane & 31, half = lane >> 5, group = pl.group, rows = f.tokens * group;
        const int q0 = rt * BM, qw = q0 + wave * 32, row = qw + col, srow = min(row, rows - 1);
        const int token = pl.by_group(srow), head = kvh * group + srow - token * group;
        const int shift = f.keys - f.tokens;
        const int plain = uniform(pl.br ? max(0, min(f.keys, shift + pl.by_group(q0) + 1)) : f.keys);
        const int lim = pl.br ? shift + token : f.keys - 1;
        const float scale2 = pg.scale * LOG2E;
        RowState st;
        clear(st);
        if (t < e1) {
            // This thread's key, and which of its stretches of DWORDS * 8 dims.
            const int kr = wave * KEYS + lane / WAVES, j = lane % WAVES, block = j * DWORDS / 4;
            typedef uint32_t codes_t __attribute__((ext_vector_type(DWORDS)));
            codes_t ck, cv;
            uint32_t ks, vs;
            // The cache rows of this wave's keys of 64 tiles from `held` on, in the lanes.  (Keys past the sequence's are
            // masked, and lie in whatever pages the table has there, clamped into the pool.)
            int held = t, lo = 0, hi = 0;
            auto hold = [&](int from) {
                held = from;
                const int key = min(from + lane, e1 - 1) * BN + wave * KEYS, slot_of = pl.by_page(key);
                const int entry = pg.block_table[int64_t(b) * pg.max_pages_per_seq + min(slot_of, pg.max_pages_per_seq - 1)];
                const int64_t r = (int64_t(min(max(entry, 0), pg.num_pages - 1)) * pg.kv_heads + kvh) * pg.page_size +
                                  (key - slot_of * pg.page_size);
                lo = int(r), hi = int(r >> 32);
            };
            hold(t);
            const LdsOffsets off = lds_offsets(lane);
            bf16x8 qr[8];
            load_q(pg, f.t0 + token, head, half, qr);
            auto load = [&](int at) {
                // Behind the last tile that again, into the stage that no step reads: no branch around the loads.
                int e = min(at, e1 - 1) - held;
                if (e >= 64) hold(held + e), e = 0;
                const int64_t r = int64_t(uint32_t(__builtin_amdgcn_readlane(lo, e))) |
                                  int64_t(__builtin_amdgcn_readlane(hi, e)) << 32;
                const uint32_t code = lane * DWORDS * 4, scale = lane / WAVES * MX4_SCALES;
                ck = *reinterpret_cast<const codes_t*>(static_cast<const char*>(pg.k_cache) + r * MX4_CODES + code);
                cv = *reinterpret_cast<const codes_t*>(static_cast<const char*>(pg.v_cache) + r * MX4_CODES + code);
                ks = *reinterpret_cast<const uint32_t*>(static_cast<const char*>(a.k_scales) + r * MX4_SCALES + scale);
                vs = *reinterpret_cast<const uint32_t*>(static_cast<const char*>(a.v_scales) + r * MX4_SCALES + scale);
            };
            auto store = [&](int stage) {
                const uint32_t kbyte = ks >> (8 * block) & 255u, vbyte = vs >> (8 * block) & 255u;
                const bool none = vbyte > MX4_MOST;
                const float sk = mx4_scale(mx4_no_numbers(vs) || kbyte > MX4_MOST ? 255u : kbyte);
                const float sv = mx4_scale(none ? 0u : vbyte);
                unsigned char* k = smem + stage * 2 * TILE_BYTES + kr * ROW_BYTES;
                unsigned char* v = k + TILE_BYTES;
                auto put = [](unsigned char* p, bf16x8 x) { *reinterpret_cast<FAV4_LDS bf16x8*>((FAV4_LDS void*)p) = x; };
#pragma unroll
                for (int i = 0; i < DWORDS; ++i) {
                    put(k + (((DWORDS * j + i) ^ k_swz(kr)) << 4), mx4_values(ck[i], sk));
                    put(v + (((DWORDS * j + i) ^ v_swz(kr)) << 4), mx4_values(none ? 0u : cv[i], sv));
                }
            };
            const bool idle = qw >= rows, early = WAVES == 4 || wave < 4;
            const int t0 = t;
            load(t);
            store(0);
            load(t + 1);
            int stage = 0;
            auto steps = [&](auto masked, int to) {
                for (; t < to; ++t) {
                    __syncthreads();
                    if (early) {
                        store(stage ^ 1);
                        load(t + 2);
                    }
                    const unsigned char* cur = smem + stage * 2 * TILE_BYTES;
                    if (!idle)
                        attend_fused<BN, decltype(masked)::value, true, LSE, true>(cur, cur + TILE_BYTES, off, qr, st, t == t0,
                                                                                   t * BN, f.keys, lim, half, scale2);
                    if (!early) {
                        store(stage ^ 1);
                        load(t + 2);
                    }
                    stage ^= 1;
                }
            };
            steps(std::integral_constant<bool, false>{}, min(e1, plain / BN));
            steps(std::integral_constant<bool, true>{}, e1);
            __syncthreads();               // every wave has read its last tile: the stages may hold O
        }
        const int live = min(32, rows - qw);
        const float inv = st.lb == 0.f ? 0.f : 1.f / st.lb;
        const uint32_t slot = wave * 2048;
        if (live <= 0) return;
        if (split) {
            const int64_t prow = (int64_t(kvh) * 2 * pl.ranges + block) * BM + wave * 32;
            store_part_rows<TILE_BYTES, true>(st, inv, smem, slot, make_rsrc(pl.o_part + prow * D, uint32_t(live) * D * 4),
                                              0, live, lane);
            if (lane < live) {
                const float sb = st.m + __builtin_amdgcn_logf(st.lb);
                reinterpret_cast<float2*>(pl.lse_part)[prow + lane] =
                    float2{sb, LSE ? st.m + __builtin_amdgcn_logf(st.l) : sb};
            }
            return;
        }
        // Through LDS, 32 rows x 128 bytes at a time, so that a store writes whole lines: as store_o_rows, for rows
        // that lie at any multiple of 256 bytes.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int dl = 0; dl < 2; ++dl)
#pragma unroll
                for (int vg = 0; vg < 4; ++vg) {
                    const f32x16& o = st.o[2 * h + dl];
                    const bf16x4 y{__bf16(o[vg * 4] * inv), __bf16(o[vg * 4 + 1] * inv), __bf16(o[vg * 4 + 2] * inv),
                                   __bf16(o[vg * 4 + 3] * inv)};
                    const uint32_t at = slot + (col >> 4) * TILE_BYTES + (col & 15) * 128 +
                                        (((4 * dl + vg) ^ (col & 7)) << 4) + half * 8;
                    *reinterpret_cast<FAV4_LDS bf16x4*>((FAV4_LDS void*)(smem + at)) = y;
                }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 8 * i + (lane >> 3), c = lane & 7;
                const uint32_t at = slot + (r >> 4) * TILE_BYTES + (r & 15) * 128 + ((c ^ (r & 7)) << 4);
                const bf16x8 y = *reinterpret_cast<const FAV4_LDS bf16x8*>((FAV4_LDS const void*)(smem + at));
                if (r < live) {
                    const int tk = pl.by_group(qw + r), hd = kvh * group + qw + r - tk * group;
                    *reinterpret_cast<bf16x8*>(static_cast<char*>(pg.o) + (int64_t(f.t0 + tk) * pg.heads + hd) * ROW_BYTES +
                                               h * 128 + c * 16) = y;
                }
            }
        }
        if (LSE && lane < live)
            pg.lse[int64_t(head) * pg.total_q + f.t0 + token] =
                st.lb == 0.f ? -__builtin_inff() : (st.m + __builtin_amdgcn_logf(st.l)) * LN2;
    }
};

// One row tile of the batch and one K/V head a workgroup, those with the most key tiles first,
// so that the last ones to start are short (8 prompts of 500..2500, H32 KVH8: 134 us, 139
// where only a sequence's own were in that order).  How many row tiles have more than u key
// tiles is, for each sequence, a division (their last token's number grows with the tile's);
// the sequences lie in the lanes, and u is found by halving.  More sequences than lanes go
// one behind the other, each its longest first.
template <int WAVES, bool LSE>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void mx4_prefill_kernel(Fav4Mx4PagedArgs a, Mx4Plan pl) {
    constexpr int BM = WAVES * 32;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * Mx4Prefill<WAVES, LSE>::TILE_BYTES];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const Mx4Prefill<WAVES, LSE> x{a, pl, smem, lane, wave};
    const Fav4PagedArgs& pg = a.paged;
    const int id = uniform(pl.by_kv_heads(blockIdx.x)), kvh = uniform(int(blockIdx.x) - id * pg.kv_heads);
    auto in_lane = [](const Mx4Seq& f, int l) {
        return Mx4Seq{__builtin_amdgcn_readlane(f.t0, l), __builtin_amdgcn_readlane(f.tokens, l),
                      __builtin_amdgcn_readlane(f.keys, l)};
    };
    Mx4Seq f{};
    int b = 0, rt;
    if (pg.batch <= 64) {
        Mx4Seq own{};
        if (lane < pg.batch) own = mx4_seq(pg, lane);
        const int n = x.tiles_of(own), shift = own.keys - own.tokens;
        auto above = [&](int u) {      // of the lane's sequence
            if (!pl.br) return own.keys > int64_t(u) * 64 ? n : 0;
            const int64_t token = int64_t(u) * 64 - shift;         // the first that sees more
            return token >= own.tokens ? 0 : token <= 0 ? n : n - int(uint32_t(token) * uint32_t(pl.group) / BM);
        };
        auto sum = [](int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); };
        if (id >= sum(n)) return;
        int lo = 0, hi = (pg.max_seqlen_k + 63) >> 6;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (sum(above(mid)) <= id) hi = mid;
            else lo = mid + 1;
        }
        const int more = above(lo), equal = (lo > 0 ? above(lo - 1) : n) - more, end = wave_scan(equal);
        const int at = id - sum(more);
        b = __builtin_ctzll(__builtin_amdgcn_ballot_w64(end > at));
        f = in_lane(own, b);
        rt = __builtin_amdgcn_readlane(n - 1 - more - (at - (end - equal)), b);
    } else {
        int before = 0;
        for (;;) {
            if (b + lane < pg.batch) f = mx4_seq(pg, b + lane);
            const int n = b + lane < pg.batch ? x.tiles_of(f) : 0, end = wave_scan(n);
            const uint64_t hit = __builtin_amdgcn_ballot_w64(before + end > id);
            if (hit) {
                const int l = __builtin_ctzll(hit);
                rt = __builtin_amdgcn_readlane(before + end - 1 - id, l);
                f = in_lane(f, l);
                b = uniform(b + l);
                break;
            }
            before += __builtin_amdgcn_readlane(end, 63);
            b += 64;
            if (b >= pg.batch) return;
        }
    }
    x.attend(b, f, rt, kvh, 0, uniform(x.key_tiles(f, rt)), false, 0);
}

// A range of the line.  The workgroup first lays out the line in LDS: the sequences'
// row tiles by a sum over the sequences, then each row tile's units by one over those.
// (Of tiles past MX4_LINE_TILES, which only bad offsets can make, nothing is attended.)
template <int WAVES, bool LSE>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void mx4_prefill_line_kernel(Fav4Mx4PagedArgs a, Mx4Plan pl) {
    __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * Mx4Prefill<WAVES, LSE>::TILE_BYTES];
    constexpr int BM = WAVES * 32, THREADS = WAVES * 64;
    __shared__ int seq_end[MX4_LINE_SEQS], unit_end[MX4_LINE_TILES], waves[WAVES];
    __shared__ uint16_t seq_of[MX4_LINE_TILES];
    __shared__ Mx4Seq seqs[MX4_LINE_SEQS];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const Mx4Prefill<WAVES, LSE> x{a, pl, smem, lane, wave};
    const Fav4PagedArgs& pg = a.paged;
    const int w = uniform(pl.by_kv_heads(blockIdx.x)), kvh = uniform(int(blockIdx.x) - w * pg.kv_heads);
    // The sum of x over threads 0..tid; `all` gets that over the workgroup.
    auto scan = [&](int v, int& all) {
        const int mine = wave_scan(v);
        __syncthreads();
        if (lane == 63) waves[wave] = mine;
        __syncthreads();
        int before = 0;
        all = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            if (i < wave) before += waves[i];
            all += waves[i];
        }
        return before + mine;
    };
    int tiles = 0;
    for (int b0 = 0; b0 < pg.batch; b0 += THREADS) {
        const int b = b0 + tid;
        Mx4Seq f{};
        if (b < pg.batch) seqs[b] = f = mx4_seq(pg, b);
        const int n = x.tiles_of(f);
        int all;
        const int end = tiles + scan(n, all);
        if (b < pg.batch) seq_end[b] = end;
        for (int i = end - n; i < min(end, MX4_LINE_TILES); ++i) seq_of[i] = uint16_t(b);
        tiles += all;
    }
    tiles = min(uniform(tiles), MX4_LINE_TILES);
    __syncthreads();
    int units = 0;
    for (int i0 = 0; i0 < tiles; i0 += THREADS) {
        const int i = i0 + tid;
        int c = 0;
        if (i < tiles) {
            const int b = seq_of[i];
            c = max(1, x.key_tiles(seqs[b], i - (b > 0 ? seq_end[b - 1] : 0))) + MX4_MANY_LEAD;
        }
        int all;
        const int end = units + scan(c, all);
        if (i < tiles) unit_end[i] = end;
        units += all;
    }
    __syncthreads();
    units = uniform(units);
    const int per = max(udiv_up(units, pl.ranges), 1), g0 = w * per, g1 = min(g0 + per, units);
    // The first row tile that ends behind unit g0.
    int lo = 0, hi = tiles;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (unit_end[mid] > g0) hi = mid;
        else lo = mid + 1;
    }
    int4 note{};
    for (int i = uniform(lo); i < tiles; ++i) {
        const int base = uniform(i > 0 ? unit_end[i - 1] : 0), end = uniform(unit_end[i]);
        if (base >= g1) break;
        const int b = uniform(seq_of[i]), rt = i - uniform(b > 0 ? seq_end[b - 1] : 0);
        Mx4Seq f = seqs[b];
        f = {uniform(f.t0), uniform(f.tokens), uniform(f.keys)};
        const int n = uniform(x.key_tiles(f, rt)), first = end - max(n, 1);
        if (first >= g1) break;
        const bool before = first < g0, split = before || end > g1;
        const int block = mx4_block(w, before);
        x.attend(b, f, rt, kvh, max(0, g0 - first), min(n, g1 - first), split, block);
        if (split && !before)
            note = int4{f.t0 * pl.group + rt * BM, min(BM, f.tokens * pl.group - rt * BM),
                        udiv(end - 1, per) - w + 1, 0};
        __syncthreads();               // O has left the stages
    }
    if (kvh == 0 && tid == 0) pl.notes[w] = note;
}

// ---- Merge --------------------------------------------------------------------------
// The row tiles that were cut: workgroup by workgroup 16 / PER rows of a range's, with one
// K/V head.  PER teams of 16 lanes share a row, 8 dims a lane; a team takes every PER-th
// part, NS at a time with all their loads in flight, with the running maximum and sums of a
// softmax over the parts' log-sums.  Bound by latency (3.6 to 5 us, as little as a kernel
// that follows another and reads what it wrote can take): the first parts are loaded beside
// the note that says how many there are.
template <int PER, int NS>
__global__ __launch_bounds__(256) void mx4_merge_kernel(Fav4Mx4PagedArgs a, Mx4Plan pl) {
    constexpr int RPB = 16 / PER;
    __shared__ float4 red[16];
    __shared__ f32x4 red_o[16][32];
    const Fav4PagedArgs& pg = a.paged;
    const int grp = threadIdx.x >> 4, l16 = threadIdx.x & 15;
    const int slot = grp / PER, part = grp - slot * PER;
    const int piece = pl.by_merge(blockIdx.x), r = (int(blockIdx.x) - piece * pl.merge_chunks) * RPB + slot;
    const int w = pl.by_kv_heads(piece), kvh = piece - w * pg.kv_heads;
    const int64_t at = int64_t(kvh) * 2 * pl.ranges * pl.stride + r;
    const int block = mx4_block(w, false), last = 2 * pl.ranges - 1;
    float2 v[NS];
    f32x4 xo[NS][2];
    // Parts c0, c0 + PER, ...; blocks past the last are it again, and get weight 0.
    auto load = [&](int c0) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int64_t row = at + int64_t(min(block + mx4_part(c0 + i * PER), last)) * pl.stride;
            v[i] = reinterpret_cast<const float2*>(pl.lse_part)[row];
            const f32x4* o = reinterpret_cast<const f32x4*>(pl.o_part + row * D + l16 * 8);
            xo[i][0] = o[0], xo[i][1] = o[1];
        }
    };
    load(part);
    const int4 note = pl.notes[w];
    // (Rows of the call, whatever another one that was given the same workspace has written there.)
    const int rows = min(note.y, pg.total_q * pl.group - note.x);
    if (note.x < 0 || r - slot >= rows || note.z <= 0) return;
    const int total = min(note.z, pl.ranges - w);
    const bool live = r < rows;
    const int tok = pl.by_group(note.x + min(r, rows - 1)), head = kvh * pl.group + note.x + r - tok * pl.group;
    float mb = -__builtin_inff(), ml = mb, den = 0.f, suml = 0.f;
    f32x4 acc[2] = {};
    for (int c0 = part; c0 < total; c0 += PER * NS) {
        if (c0 != part) load(c0);
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (c0 + i * PER >= total) v[i] = float2{-__builtin_inff(), -__builtin_inff()};
        float nb = mb, nl = ml;
#pragma unroll
        for (int i = 0; i < NS; ++i) nb = fmaxf(nb, v[i].x), nl = fmaxf(nl, v[i].y);
        if (nb == -__builtin_inff()) {
            // Parts without a visible key, or with sums that are no numbers (which maxima
            // pass over): so are then O and the LSE.
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
    if (!live || part != 0) return;
    const float rden = den == 0.f ? 0.f : 1.f / den;
    bf16x8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __bf16(acc[i >> 2][i & 3] * rden);
    *reinterpret_cast<bf16x8*>(static_cast<char*>(pg.o) + (int64_t(tok) * pg.heads + head) * ROW_BYTES + l16 * 16) = y;
    if (pg.lse && l16 == 0) pg.lse[int64_t(head) * pg.total_q + tok] =
        den == 0.f ? -__builtin_inff() : (ml + __builtin_amdgcn_logf(suml)) * LN2;
}

}  // namespace fav4
