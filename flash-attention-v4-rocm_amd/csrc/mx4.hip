// C-ABI host dispatch of the operators of 4-bit paged K/V caches
// (include/fav4_mx4.h): the argument checks, before any HIP call, and the launches.
#include "fav4_mx4.h"
#include "mx4_kernel.hpp"

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>

namespace {

constexpr int64_t MAX_GRID = int64_t(1) << 22;
constexpr int64_t MAX_BYTES = int64_t(1) << 48;
constexpr int MAX_BATCH = INT_MAX - 63;       // wave_find's 64 steps through the offsets fit an int
constexpr int BOTTOM_RIGHT = 2;
constexpr int MAX_KEYS = INT_MAX - 255;       // in whole pages: a position and a tile's width fit an int
constexpr int MAX_HEADS = 1 << 15;            // the documented limit; indexes need total_q * heads < 2^31 alone
constexpr int MAX_ROW_TILES = 1 << 22;
constexpr int MAX_KEY_TILES = 1'000'000'000;

// CU count of the current device (256 if it cannot be read), cached per
// device after the first query.
int device_cus() {
    static std::atomic<int> cache[64];
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess) return 256;
    const bool slot = dev >= 0 && dev < 64;
    if (slot && (cus = cache[dev].load(std::memory_order_relaxed)) > 0) return cus;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) cus = 256;
    if (slot) cache[dev].store(cus, std::memory_order_relaxed);
    return cus;
}

template <class... P>
bool aligned(uintptr_t to, P... p) {
    return ((... | reinterpret_cast<uintptr_t>(p)) & (to - 1)) == 0;
}

bool caches_fit(int num_pages, int page_size, int kv_heads) {
    return static_cast<__int128>(num_pages) * page_size * kv_heads * fav4::MX4_CODES < MAX_BYTES;
}
bool stride_ok(long long stride, int heads, int rows) {
    return stride >= int64_t(heads) * fav4::D && (stride & 7) == 0 && static_cast<__int128>(stride) * rows * 2 < MAX_BYTES;
}

bool append_ok(const Fav4Mx4AppendArgs* args) {
    if (!args || !args->k_scales || !args->v_scales || !aligned(16, args->k_scales, args->v_scales)) return false;
    const Fav4AppendArgs* a = &args->append;
    if (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->cu_seqlens_q || !a->seqlens_k || !a->block_table ||
        !a->q != !a->q_out)
        return false;
    if (a->batch < 1 || a->batch > MAX_BATCH || a->heads < 1 || a->kv_heads < 1 || a->total_q < 1 ||
        a->num_pages < 1 || a->page_size < 1 || a->max_pages_per_seq < 1 || a->rotary_dim < 0 ||
        a->rotary_dim > fav4::D || a->rotary_dim % 16 || (a->interleaved != 0 && a->interleaved != 1))
        return false;
    if (a->rotary_dim > 0 ? !a->cos || !a->sin || a->rotary_rows < 1 : a->cos || a->sin) return false;
    const int64_t rows = (a->q ? int64_t(a->heads) : 0) + 2 * int64_t(a->kv_heads);
    if (rows > INT_MAX || rows * a->total_q > INT_MAX) return false;
    if (!stride_ok(a->k_stride, a->kv_heads, a->total_q) || !stride_ok(a->v_stride, a->kv_heads, a->total_q)) return false;
    if (a->q && (!stride_ok(a->q_stride, a->heads, a->total_q) || !stride_ok(a->q_out_stride, a->heads, a->total_q) ||
                 (a->q == a->q_out && a->q_stride != a->q_out_stride)))
        return false;
    return caches_fit(a->num_pages, a->page_size, a->kv_heads) &&
           aligned(16, a->q, a->k, a->v, a->q_out, a->k_cache, a->v_cache, a->cos, a->sin) &&
           aligned(4, a->cu_seqlens_q, a->seqlens_k, a->block_table, a->positions);
}

bool gather_ok(const Fav4Mx4GatherArgs* a) {
    if (!a || !a->k_cache || !a->k_scales || !a->v_cache || !a->v_scales || !a->k || !a->v || !a->cu_seqlens_k ||
        !a->block_table)
        return false;
    if (a->batch < 1 || a->batch > MAX_BATCH || a->kv_heads < 1 || a->total_k < 1 || a->num_pages < 1 ||
        a->page_size < 1 || a->max_pages_per_seq < 1 || 2 * int64_t(a->kv_heads) * a->total_k > INT_MAX)
        return false;
    return stride_ok(a->k_stride, a->kv_heads, a->total_k) && stride_ok(a->v_stride, a->kv_heads, a->total_k) &&
           caches_fit(a->num_pages, a->page_size, a->kv_heads) &&
           aligned(16, a->k_cache, a->k_scales, a->v_cache, a->v_scales, a->k, a->v) &&
           aligned(4, a->cu_seqlens_k, a->starts, a->block_table);
}

// ---- attention -------------------------------------------------------------------
bool paged_shape_ok(const Fav4Mx4PagedArgs* args, int causal) {
    if (!args) return false;
    const Fav4PagedArgs& a = args->paged;
    if (a.batch < 1 || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads || a.max_seqlen_q < 1 ||
        a.max_seqlen_k < 1 || a.total_q < 1 || a.total_k < 0 || a.num_pages < 1 || a.page_size < 1 ||
        a.max_pages_per_seq < 1 || (causal != 0 && causal != BOTTOM_RIGHT) || !std::isfinite(a.scale) || a.scale <= 0)
        return false;
    return a.page_size % 16 == 0 && a.max_seqlen_k <= int64_t(a.max_pages_per_seq) * a.page_size &&
           (int64_t(a.max_seqlen_k) + a.page_size - 1) / a.page_size <= MAX_KEYS / a.page_size && a.heads <= MAX_HEADS &&
           int64_t(a.total_q) * a.heads <= INT_MAX && caches_fit(a.num_pages, a.page_size, a.kv_heads);
}

// The decode kernel's workgroups on a line (cut): four waves of 32-key tiles, three a CU,
// with up to 16 rows; of 64-key tiles, two a CU, with 32.  Whole sequences: eight waves of
// 32-key tiles, one a CU, or twelve with up to 16 rows and more than LONG_KEYS keys: 1
// sequence of 800, H32 KVH8, 6.8 and 7.2 us (8.0 with eight of 64-key tiles), 16 of 500..2500
// 14.5 and 13.6 (14.8), 32 x 4 queries of 200..4096 21.2 and 19.6 (21.3).
constexpr int LINE_WAVES = 4, WHOLE_WAVES = 8, LONG_WAVES = 12, LONG_KEYS = 2048;
constexpr int line_per_cu(int row_tiles) { return row_tiles == 1 ? 3 : 2; }
constexpr int line_subtiles(int row_tiles) { return row_tiles == 1 ? 2 : 4; }
// Keys that a workgroup of a line should have at least: what it takes grows with them, what
// the merge takes with the longest sequence's parts; their sum is least near the root of its
// keys.  With 4, 5, 3 times that and with 384: 4 sequences of 100..2000, H32 KVH8, 9.0, 9.5,
// 9.8 and 10.4 us; 24 of 1000..16384, H8 KVH1, 15.4, 15.1, 15.5 and 15.5; 3 x 6 queries
// behind 540..8641, H16 KVH2, 15.6, 17.3, 16.0 and 15.6.
double line_keys(int max_keys) { return std::max(128.0, 4 * std::sqrt(double(max_keys))); }
// Up to this many parts of the longest sequence's rows four teams of a merge take two parts
// each at once, above eight teams four: 24 of 1000..16384, H8 KVH1, 15.5 so and 16.5 with
// four, 48 of 100..4096, H32 KVH8, 19.4 and with eight 20.2 (20.6 with four of eight parts
// each, many of whose loads find no part).  Of many rows one team takes four, or four two:
// 5 x 329 queries behind 329..1216 keys, H16 KVH1, 31.1 with one and 34.3 with four; 2 x
// 30..99 behind 4503, H40 KVH8, 36.1 and 39.6; 3 x 7..15 behind 29006..77731, H32 KVH1, 61.5
// and 47.7; one of 30 behind 26965, H32 KVH8, 45.4 and 41.1.  Over 40 such batches the limit
// costs 6% less than one team for all, and 1% less than four.
constexpr int MERGE_PARTS = 16;
// Whether a call goes by the decode kernel: with up to FEW_ROWS rows a sequence, and with
// more where its row tiles of 32 are no more than the CUs and read so few keys in all (and
// what their starts and ends cost) that the GPU is not full.  Decode / prefill kernels: H8
// KVH1, 64 x 8 queries behind 1000..4000 25.3 / 28.5; H32 KVH8, 32 x 16 behind 2000..8000
// 78.6 / 90.7, 32 x 20 109 / 94, 8 x 20 behind 500..2000 16.7 / 26.1; prompts, one of 128
// 6.6 / 7.8, 13 of 26 26.7 / 6.8.  The two limits are what parts such measurements, and have
// no other reason.  Over 60 batches of 100 to 800 pairs of a row tile of 32 and a K/V head,
// drawn apart from those (19 of them go by the decode kernel), the choice costs 0.9% more than
// the quicker kernel; at the worst, one of 1022 behind 2730, H8 KVH1, 20.2 / 32.8.
constexpr int FEW_ROWS = 64;
bool few_rows(int64_t seq_rows, double rows, double keys, int64_t batch, int kv_heads, int cus) {
    if (seq_rows <= FEW_ROWS) return true;
    const int64_t tiles = (seq_rows + 31) / 32;
    return double(tiles) * double(batch) * kv_heads <= cus &&
           (keys + 640. * double(batch)) * kv_heads * std::min(double(tiles), rows / 32 / double(batch) + 0.5) <= 750e3;
}

// Whether every sequence and K/V head (`pairs`) has a workgroup of its own, and no merge.
// Measured, as graphs: such workgroups start and end in 4.2 us, read 290 keys a us (175 with
// 32 rows) and wait for 0.3 of the time that all bytes take at 6.3 TB/s; a line takes 9.1,
// 0.05 to 0.3 for each row up to 16 (by how many pairs write parts), and the bytes' time.  H32
// KVH8 and one query where not said, whole / cut: 1 sequence of 2500, 4 queries, 13.6 / 10.9;
// 4 of 500..2000, H16 KVH2, 2 queries, 12.3 / 10.7; 16 of 500..2500, 4 queries, 14.2 / 17.7;
// 32 of 200..4096, 4 queries, 19.6 / 21.5; 32 of 3500..4000, 8 queries, 28.5 / 41.5.  With
// more pairs than CUs whole sequences wait for one another: 48 of 100..4096 23.3 whole, 20.2
// cut; 64 of 500..8192 55.8 and 44.5.
bool whole_sequences(int64_t pairs, int64_t rows, int64_t max_keys, double all_keys, int cus) {
    const double rate = rows <= 16 ? 290 : 175;
    const double row = 0.05 + 0.25 * double(pairs) / cus;
    return pairs <= cus &&
           double(max_keys) < rate * (4.9 + row * double(std::min<int64_t>(rows, 16)) + 0.7 * all_keys * 136 / 6.3e6);
}

// Key tiles of many rows that a range should have at least: with a half, 0.3, 0.8 times the
// longest's root, and one, 3 sequences of 14 queries behind 28774..109665, H8 KVH1, 48.4, 54.4,
// 60.2 and 54.8 us; 3 of 18..42 behind 14379..85937, H8 KVH1, 59.4, 52.0, 78.5 and 52.1; one of
// 30 behind 26965, H32 KVH8, 41.1, 35.9, 38.1 and 35.9.  Over 40 batches whose ranges it
// decides 0.3 and one cost 1% less than a half, 0.8 costs 10% more.
double range_tiles(double most) { return std::max(1.0, 0.5 * std::sqrt(most)); }

// Sequences of many rows: row tiles of eight waves (256 rows, one workgroup a CU) or four
// (128, two), each whole, the longest first, or on a line.  By an estimate in us of each,
// from the sizes (of unequal lengths their means and the longest), its constants fitted to
// 120 batches timed all four ways, among them some that few_rows has since sent to the decode
// kernel; over 60 others that come here its choice costs 1.2% more than the best (at the
// worst 16%: one of 797 behind 1059, dense, H16 KVH16, 36.3 / 27.8 / 33.2 / 32.2).  A
// 64-key tile takes a workgroup of eight waves 1.9, one of four 2.06 in a full GPU (2.15 on
// a line) and 1.3 alone; a row tile starts and ends in 4 (2.2), on a line in 6.8; a line's own
// start, the second launch and its merge take 15.  Measured, H32 KVH8 where not said, whole 8
// / whole 4 / line 8 / line 4: 8 x 64..512 queries behind 1024..8192 keys 227 / 188 / 156 /
// 172; prompts of 500..2500 134 / 137 / 148 / 162; 2 prompts of 146 and 134 behind 224, H40,
// 13.7 / 10.9 / 20.5 / 17.9; 5 x 144..316 behind 1590..11482 319 / 249 / 136 / 146; 4 x 84
// behind 3328..14065, dense, 390 / 290 / 83.9 / 80.6.
struct Cut {
    int waves, ranges;                // ranges of a K/V head, 0: whole
    double parts;                     // of the longest row tile on a line, about
};
template <class F>
Cut many_rows_cut(const Fav4PagedArgs& a, int causal, int cus, F&& row_tiles) {
    double mean_q = double(a.total_q) / a.batch;
    double mean_k = a.total_k > 0 ? double(a.total_k) / a.batch : double(a.max_seqlen_k);
    const bool br = causal == BOTTOM_RIGHT, even = !br && mean_k > 0.95 * a.max_seqlen_k;
    const bool prompts = a.max_seqlen_k < 2.0 * a.max_seqlen_q;
    if (prompts) {                    // the long ones' row tiles are the most
        mean_q += 0.4 * (a.max_seqlen_q - mean_q);
        mean_k += 0.4 * (a.max_seqlen_k - mean_k);
    }
    const double units = std::max(1.0, (mean_k - (br ? 0.5 * mean_q : 0.0)) / 64);
    const double most = std::max(units, a.max_seqlen_k / 64.0);
    Cut best{};
    double least = 1e30;
    for (int waves : {8, 4}) {
        const double tiles = row_tiles(waves), n = tiles * a.kv_heads, slots = double(cus) * (8 / waves), turns = n / slots;
        const double unit = waves == 8 ? 1.9 : n <= cus ? 1.3 : n <= slots && br && prompts ? 1.45 : 2.06;
        const double ends = waves == 8 ? 4 : 2.2;
        const double tail = even ? (std::ceil(turns) - turns) * (unit * units + ends) : 0.24 * unit * most;
        const double whole = 3 + (turns <= 1 ? unit * most + ends : turns * (unit * units + ends) + tail);
        const int ranges = int(std::min(std::max(1.0, std::floor(slots / a.kv_heads)), 1 + tiles * units / range_tiles(most)));
        const double groups = double(ranges) * a.kv_heads, line_unit = waves == 8 ? 1.9 : groups <= cus ? 1.3 : 2.15;
        const double line = 15 + (line_unit * units + 6.8) * n / groups;
        if (whole < least) least = whole, best = {waves, 0, 1};
        if (line < least) least = line, best = {waves, ranges, most * ranges / (tiles * units)};
    }
    return best;
}

struct Sizes {
    fav4::Mx4Plan plan;
    int64_t bytes, part_rows, grid, merge_grid;
    int merge_teams, waves;
    bool few, split;
    bool ok;
    double parts;                     // of the longest sequence's rows, about
};
Sizes paged_sizes(const Fav4Mx4PagedArgs& args, int causal) {
    const Fav4PagedArgs& a = args.paged;
    const int64_t group = a.heads / a.kv_heads, rows = a.total_q * group;
    const int64_t seq_rows = std::min<int64_t>(a.max_seqlen_q * group, rows);
    const int cus = device_cus();
    Sizes s{};
    fav4::Mx4Plan& p = s.plan;
    p.group = int(group);
    p.br = causal == BOTTOM_RIGHT;
    const int64_t keys = a.total_k > 0 ? a.total_k : int64_t(a.batch) * a.max_seqlen_k;
    s.few = few_rows(seq_rows, double(rows), double(keys), a.batch, a.kv_heads, cus);
    // Workgroups of a K/V head that are resident at once, at most: with few rows, and with many.
    const int few_ranges = std::max(1, line_per_cu(1) * cus / a.kv_heads);
    auto many_ranges = [&](int waves) { return std::max(1, 8 / waves * cus / a.kv_heads); };
    int64_t segs;
    if (s.few) {
        p.stride = seq_rows <= 16 ? 16 : 32;
        p.tiles = int((seq_rows + p.stride - 1) / p.stride);
        segs = int64_t(a.batch) * p.tiles;
        const int resident = std::max(1, line_per_cu(p.stride / 16) * cus / a.kv_heads);
        s.split = !whole_sequences(segs * a.kv_heads, seq_rows, a.max_seqlen_k, double(keys) * p.tiles * a.kv_heads, cus);
        p.ranges = s.split ? int(std::min(double(resident), 1 + double(keys) * p.tiles / line_keys(a.max_seqlen_k))) : 1;
        s.parts = a.max_seqlen_k * double(p.ranges) / (double(keys) * p.tiles);
    } else {
        auto row_tiles = [&](int bm) {
            return std::min<int64_t>(a.batch * ((seq_rows + bm - 1) / bm), (rows + int64_t(a.batch) * (bm - 1)) / bm);
        };
        const bool equal = double(a.max_seqlen_q) * a.batch < 1.05 * a.total_q;
        const Cut cut = many_rows_cut(a, causal, cus, [&](int waves) {
            const double most = double(row_tiles(waves * 32));
            return equal ? most : std::min(most, double(rows) / (waves * 32) + 0.5 * a.batch);
        });
        s.waves = cut.waves;
        p.stride = s.waves * 32;
        segs = row_tiles(p.stride);
        s.split = cut.ranges && segs <= fav4::MX4_LINE_TILES && a.batch <= fav4::MX4_LINE_SEQS;
        p.ranges = s.split ? std::min(cut.ranges, many_ranges(s.waves)) : 1;
        s.parts = cut.parts;
    }
    s.grid = a.kv_heads * (s.split ? int64_t(p.ranges) : segs);
    // A grid has less than 2^32 threads, and the units of a line (of 32 keys) end below 2^31.
    s.ok = segs <= MAX_ROW_TILES && s.grid < (int64_t(1) << 23) &&
           segs * (int64_t(a.max_seqlen_k) / 64 + 1 + std::max(fav4::MX4_LEAD, fav4::MX4_MANY_LEAD)) < MAX_KEY_TILES;
    p.by_kv_heads = fav4::fast_div(a.kv_heads);
    p.by_group = fav4::fast_div(int(group));
    p.by_page = fav4::fast_div(a.page_size);
    // Teams per merged row.
    s.merge_teams = s.few ? s.parts <= MERGE_PARTS ? 4 : 8 : s.parts <= MERGE_PARTS ? 1 : 4;
    p.merge_chunks = int((std::min<int64_t>(p.stride, seq_rows) * s.merge_teams + 15) / 16);
    s.merge_grid = int64_t(p.ranges) * a.kv_heads * p.merge_chunks;
    p.by_merge = fav4::fast_div(p.merge_chunks);
    // What a call of either kind could need: more queries or sequences never need less.
    // (With more K/V heads than CUs a range of 128-row tiles holds less than one of 256.)
    const int few_part = few_ranges * 32, many_part = std::max(many_ranges(8) * 256, many_ranges(4) * 128);
    s.part_rows = int64_t(a.kv_heads) * 2 * (seq_rows <= FEW_ROWS ? few_part : std::max(few_part, many_part));
    s.bytes = s.part_rows * (fav4::D * 4 + 8) + int64_t(few_ranges) * 16;
    return s;
}

template <int NT>
void launch_few(const Fav4Mx4PagedArgs& a, const Sizes& s, hipStream_t stream) {
    auto go = [&](auto kernel, int waves) {
        hipLaunchKernelGGL(kernel, dim3(unsigned(s.grid)), dim3(waves * 64), 0, stream, a, s.plan);
    };
    auto with = [&](auto lse, auto p64) {
        constexpr bool L = decltype(lse)::value, P = decltype(p64)::value;
        if (s.split)
            go(fav4::mx4_decode_kernel<NT, LINE_WAVES, line_subtiles(NT), line_per_cu(NT), true, L, P>, LINE_WAVES);
        else if (NT == 1 && a.paged.max_seqlen_k > LONG_KEYS)
            go(fav4::mx4_decode_kernel<1, LONG_WAVES, 2, 3, false, L, P>, LONG_WAVES);
        else
            go(fav4::mx4_decode_kernel<NT, WHOLE_WAVES, 2, 2, false, L, P>, WHOLE_WAVES);
    };
    const bool p64 = a.paged.page_size % 64 == 0;
    if (a.paged.lse) p64 ? with(std::true_type{}, std::true_type{}) : with(std::true_type{}, std::false_type{});
    else p64 ? with(std::false_type{}, std::true_type{}) : with(std::false_type{}, std::false_type{});
}

template <int WAVES, bool LSE>
void launch_many(const Fav4Mx4PagedArgs& a, const Sizes& s, hipStream_t stream) {
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(unsigned(s.grid)), dim3(WAVES * 64), 0, stream, a, s.plan);
    };
    if (s.split) go(fav4::mx4_prefill_line_kernel<WAVES, LSE>);
    else go(fav4::mx4_prefill_kernel<WAVES, LSE>);
}

}  // namespace

extern "C" __attribute__((visibility("default"))) int fav4_bshd_append_paged_mx4(const Fav4Mx4AppendArgs* args,
                                                                                hipStream_t stream) {
    if (!append_ok(args)) return hipErrorInvalidValue;
    const Fav4AppendArgs& a = args->append;
    const int rows = (a.q ? a.heads : 0) + 2 * a.kv_heads, units = (rows + 7) / 8;
    const int64_t total = int64_t(units) * ((int64_t(a.total_q) + 3) / 4), blocks = std::min(total, MAX_GRID);
    const fav4::FastDiv by_units = fav4::fast_div(units), by_page = fav4::fast_div(a.page_size);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(256), 0, stream, *args, units, int(total), by_units, by_page);
    };
    if (a.interleaved) go(fav4::mx4_store_kernel<true>);
    else go(fav4::mx4_store_kernel<false>);
    return hipGetLastError();
}

extern "C" __attribute__((visibility("default"))) int fav4_bshd_gather_paged_mx4(const Fav4Mx4GatherArgs* a,
                                                                                hipStream_t stream) {
    if (!gather_ok(a)) return hipErrorInvalidValue;
    // Rows a wave: one each until the waves fill the GPU.
    const int each = int(std::min<int64_t>(std::max<int64_t>(a->total_k / (int64_t(16) * device_cus()), 1), fav4::MX4_READ_ROWS));
    const int64_t per = 4 * each, blocks = std::min((a->total_k + per - 1) / per, MAX_GRID);
    hipLaunchKernelGGL(fav4::mx4_read_kernel, dim3(unsigned(blocks)), dim3(256), 0, stream, *a, fav4::fast_div(a->page_size),
                       each);
    return hipGetLastError();
}

extern "C" __attribute__((visibility("default"))) long long fav4_bshd_paged_mx4_workspace_size(
    const Fav4Mx4PagedArgs* args, int causal) {
    if (!paged_shape_ok(args, causal)) return -1;
    const Sizes s = paged_sizes(*args, causal);
    return s.ok ? s.bytes : -1;
}

extern "C" __attribute__((visibility("default"))) int fav4_bshd_forward_paged_mx4(const Fav4Mx4PagedArgs* args,
                                                                                 int causal, void* workspace,
                                                                                 size_t workspace_bytes,
                                                                                 hipStream_t stream) {
    if (!paged_shape_ok(args, causal)) return hipErrorInvalidValue;
    const Fav4PagedArgs& a = args->paged;
    if (!a.q || !a.k_cache || !a.v_cache || !a.o || !a.cu_seqlens_q || !a.seqlens_k || !a.block_table ||
        !args->k_scales || !args->v_scales ||
        !aligned(16, a.q, a.k_cache, a.v_cache, a.o, args->k_scales, args->v_scales) ||
        !aligned(4, a.lse, a.cu_seqlens_q, a.seqlens_k, a.block_table))
        return hipErrorInvalidValue;
    Sizes s = paged_sizes(*args, causal);
    if (!s.ok || !workspace || !aligned(256, workspace) || uint64_t(s.bytes) > workspace_bytes)
        return hipErrorInvalidValue;
    fav4::Mx4Plan& p = s.plan;
    p.o_part = static_cast<float*>(workspace);
    p.lse_part = p.o_part + s.part_rows * fav4::D;
    p.notes = reinterpret_cast<int4*>(p.lse_part + s.part_rows * 2);
    if (s.few) {
        if (p.stride == 16) launch_few<1>(*args, s, stream);
        else launch_few<2>(*args, s, stream);
    } else {
        if (a.lse) s.waves == 4 ? launch_many<4, true>(*args, s, stream) : launch_many<8, true>(*args, s, stream);
        else s.waves == 4 ? launch_many<4, false>(*args, s, stream) : launch_many<8, false>(*args, s, stream);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !s.split) return e;
    auto merge = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(unsigned(s.merge_grid)), dim3(256), 0, stream, *args, p);
    };
    if (s.merge_teams == 8) merge(fav4::mx4_merge_kernel<8, 4>);
    else if (s.merge_teams == 4) merge(fav4::mx4_merge_kernel<4, 2>);
    else merge(fav4::mx4_merge_kernel<1, 4>);
    return hipGetLastError();
}
