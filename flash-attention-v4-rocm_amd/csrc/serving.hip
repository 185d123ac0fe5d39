// C-ABI host dispatch of the serving operators (include/fav4_serving.h): the
// argument checks, before any HIP call, and the launches.
#include "fav4_serving.h"
#include "serving_kernel.hpp"

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>

namespace {

constexpr int64_t MAX_GRID = int64_t(1) << 22;
constexpr int64_t MAX_BYTES = int64_t(1) << 48;

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

// ---- append ------------------------------------------------------------------
constexpr int MAX_BATCH = INT_MAX - 63;      // wave_find's 64 steps through the offsets fit an int
bool append_ok(const Fav4AppendArgs* a) {
    if (!a || !a->k || !a->v || !a->k_cache || !a->v_cache || !a->cu_seqlens_q || !a->seqlens_k || !a->block_table ||
        !a->q != !a->q_out)
        return false;
    if (a->batch < 1 || a->batch > MAX_BATCH || a->heads < 1 || a->kv_heads < 1 || a->total_q < 1 ||
        a->num_pages < 1 || a->page_size < 1 || a->max_pages_per_seq < 1 || a->rotary_dim < 0 ||
        a->rotary_dim > fav4::D || a->rotary_dim % 16 || (a->interleaved != 0 && a->interleaved != 1))
        return false;
    if (a->rotary_dim > 0 ? !a->cos || !a->sin || a->rotary_rows < 1 : a->cos || a->sin) return false;
    const int64_t rows = (a->q ? int64_t(a->heads) : 0) + 2 * int64_t(a->kv_heads);
    if (rows > INT_MAX || rows * a->total_q > INT_MAX) return false;
    auto stride_ok = [&](long long stride, int heads) {
        return stride >= int64_t(heads) * fav4::D && (stride & 7) == 0 &&
               static_cast<__int128>(stride) * a->total_q * 2 < MAX_BYTES;
    };
    if (!stride_ok(a->k_stride, a->kv_heads) || !stride_ok(a->v_stride, a->kv_heads)) return false;
    if (a->q && (!stride_ok(a->q_stride, a->heads) || !stride_ok(a->q_out_stride, a->heads) ||
                 (a->q == a->q_out && a->q_stride != a->q_out_stride)))
        return false;
    if (static_cast<__int128>(a->num_pages) * a->page_size * a->kv_heads * fav4::ROW_BYTES >= MAX_BYTES) return false;
    return aligned(16, a->q, a->k, a->v, a->q_out, a->k_cache, a->v_cache, a->cos, a->sin) &&
           aligned(4, a->cu_seqlens_q, a->seqlens_k, a->block_table, a->positions);
}

// ---- attention behind shared prefixes ------------------------------------------
constexpr int BOTTOM_RIGHT = 2;
// Up to this many rows of a prefix (the mean) its keys are split over a workgroup's
// waves (H32 KVH8, 16 prefixes of 4096 keys: at 24..32 rows 73 us split, 82 shared; at
// 48 rows 122 and 84).
constexpr int SPLIT_ROWS = 32;
// Up to this many rows of a sequence its own keys are read by single waves (32 rows,
// 64 sequences behind 4096 H32 KVH8: 60 us by waves, 70 by workgroups; 48 rows, 48
// sequences of 1000..4000 own keys: 203, two row tiles each, and 151).
constexpr int WAVE_ROWS = 32;

// Keys of a sequence and of a prefix, whole pages: a position and a tile's width fit an int.
constexpr int MAX_KEYS = INT_MAX - 255;
constexpr int MAX_HEADS = 1 << 15;    // the documented limit; indexes need total_q * heads < 2^31 alone

// Pages that max_seqlen_k keys take.
int64_t whole_pages(const Fav4PagedArgs& a) { return (int64_t(a.max_seqlen_k) + a.page_size - 1) / a.page_size; }

bool prefix_shape_ok(const Fav4PrefixArgs* args, int causal) {
    if (!args) return false;
    const Fav4PagedArgs& a = args->paged;
    if (a.batch < 1 || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads || a.max_seqlen_q < 1 ||
        a.max_seqlen_k < 1 || a.total_q < 1 || a.total_k < 0 || a.num_pages < 1 || a.page_size < 1 ||
        a.max_pages_per_seq < 1 || args->num_prefixes < 1 || args->max_pages_per_prefix < 1 ||
        (causal != 0 && causal != BOTTOM_RIGHT) || !std::isfinite(a.scale) || a.scale <= 0)
        return false;
    if (a.page_size % 32 || a.max_seqlen_k > int64_t(a.max_pages_per_seq) * a.page_size ||
        whole_pages(a) > MAX_KEYS / a.page_size || a.heads > MAX_HEADS || int64_t(a.total_q) * a.heads > INT_MAX ||
        int64_t(a.kv_heads) * fav4::ROW_BYTES * 32 > INT_MAX ||
        static_cast<__int128>(a.num_pages) * a.page_size * a.kv_heads * fav4::ROW_BYTES >= MAX_BYTES)
        return false;
    return true;
}

struct PrefixSizes {
    fav4::PrefixPlan plan;
    int64_t part_rows, bytes;
    int64_t parts;             // that a row can have of its prefix and of its own, on average
    int prefix_rows;           // of a prefix block
    fav4::Cut cut;
    bool ok;
};
PrefixSizes prefix_sizes(const Fav4PrefixArgs& args, int causal) {
    const Fav4PagedArgs& a = args.paged;
    const int64_t group = a.heads / a.kv_heads, rows = a.total_q * group;
    const int64_t seq_rows = std::min<int64_t>(a.max_seqlen_q * group, rows);
    PrefixSizes s{};
    s.plan.br = causal == BOTTOM_RIGHT;
    s.cut = a.max_seqlen_q * group > WAVE_ROWS                     ? fav4::MANY
            : rows <= int64_t(args.num_prefixes) * SPLIT_ROWS ? fav4::FEWEST
                                                                    : fav4::FEW;
    const int WAVES = 8, BM = s.prefix_rows = s.cut == fav4::FEWEST ? 32 : WAVES * 32;
    const bool own_waves = s.cut != fav4::MANY;
    // As many workgroups as are resident at once; at least one for each line.
    s.plan.ranges = std::min(1024, std::max(2, device_cus() / a.kv_heads));
    // Row tiles that the rows of n families can have.
    auto tiles = [&](int64_t n, int64_t most, int bm) {
        return std::min(n * ((most + bm - 1) / bm), (rows + n * (bm - 1)) / bm);
    };
    const int own_bm = own_waves ? 32 : BM;
    const int64_t own_rows = std::min<int64_t>(own_bm, seq_rows);
    const int64_t prefix_segs = tiles(args.num_prefixes, rows, BM);
    const int64_t own_segs = tiles(a.batch, seq_rows, own_bm);
    // Whole pages of a prefix, the one too that the longest sequence ends in (a sequence
    // may have fewer keys than its prefix, and reads none of those in its own table).
    const int64_t prefix_keys = std::min<int64_t>(args.max_pages_per_prefix, whole_pages(a)) * a.page_size;
    s.plan.most_prefix_keys = int(prefix_keys);
    const int64_t lead = 1 + std::max(fav4::SEG_TILES, fav4::SPLIT_SEG_TILES);
    const int64_t units = prefix_segs * (prefix_keys / 32 + lead) + own_segs * (a.max_seqlen_k / 32 + lead);
    const int64_t prefix_ranges = s.plan.ranges;
    const int64_t own_ranges = s.plan.ranges * (own_waves ? WAVES : 1);
    const int64_t prefix_blocks = prefix_segs + prefix_ranges, own_blocks = own_segs + own_ranges;
    s.parts = std::min(prefix_ranges / std::max<int64_t>(1, prefix_segs),
                       prefix_keys / (s.cut == fav4::FEWEST ? 32 * fav4::MIN_SPLIT_TILES : 64 * fav4::MIN_PREFIX_TILES)) +
              std::min(own_ranges / std::max<int64_t>(1, own_segs),
                       std::max<int64_t>(0, a.max_seqlen_k - prefix_keys) / ((own_waves ? 32 : 64) * fav4::MIN_OWN_TILES));
    s.part_rows = (a.kv_heads * (prefix_blocks * BM + own_blocks * own_rows) + 1) & ~int64_t(1);   // notes 16-byte aligned
    s.ok = units < (1 << 30) && prefix_blocks * BM <= INT_MAX && own_blocks * own_rows <= INT_MAX;
    s.plan.prefix_blocks = int(prefix_blocks);
    s.plan.own_blocks = int(own_blocks);
    s.plan.own_rows = int(own_rows);
    s.plan.group = int(group);
    s.plan.by_kv_heads = fav4::fast_div(a.kv_heads);
    s.plan.by_group = fav4::fast_div(int(group));
    s.plan.by_page = fav4::fast_div(a.page_size);
    s.plan.by_heads = fav4::fast_div(a.heads);
    s.plan.by_bm = fav4::fast_div(BM);
    s.plan.by_own_rows = fav4::fast_div(int(own_rows));
    // What a call of any cut needs at most: a larger batch, more queries or prefixes
    // never need less, so that one workspace serves a serving loop's smaller steps.
    const int64_t range_rows = std::max<int64_t>(512, int64_t(2) * device_cus() * 128 / a.kv_heads);
    const int64_t own_pad = a.max_seqlen_q * group > WAVE_ROWS ? 255 : 31;
    const int64_t most = a.kv_heads * (2 * (rows + range_rows) + int64_t(args.num_prefixes) * 255 + a.batch * own_pad);
    s.ok = s.ok && s.part_rows <= most + 1 && most < (int64_t(1) << 40);
    if (!s.ok) return s;
    s.bytes = (most + 1) * (fav4::D * 4 + 8) + rows * 16;
    return s;
}

void launch_prefix(const Fav4PrefixArgs& args, const PrefixSizes& s, hipStream_t stream) {
    const dim3 grid(unsigned(args.paged.kv_heads) * unsigned(s.plan.ranges));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(512), 0, stream, args, s.plan); };
    auto with_lse = [&](auto cut, auto cached) {
        constexpr fav4::Cut CUT = decltype(cut)::value;
        constexpr bool C = decltype(cached)::value;
        if (args.paged.lse) go(fav4::prefix_kernel<true, CUT, C>);
        else go(fav4::prefix_kernel<false, CUT, C>);
    };
    auto with_cut = [&](auto cached) {
        if (s.cut == fav4::MANY) with_lse(std::integral_constant<fav4::Cut, fav4::MANY>{}, cached);
        else if (s.cut == fav4::FEW) with_lse(std::integral_constant<fav4::Cut, fav4::FEW>{}, cached);
        else with_lse(std::integral_constant<fav4::Cut, fav4::FEWEST>{}, cached);
    };
    if (args.paged.batch <= fav4::PLAN_SEQS && args.num_prefixes <= fav4::PLAN_PREFIXES) with_cut(std::true_type{});
    else with_cut(std::false_type{});
}

}  // namespace

extern "C" __attribute__((visibility("default"))) int fav4_bshd_append_paged(const Fav4AppendArgs* a,
                                                                            hipStream_t stream) {
    if (!append_ok(a)) return hipErrorInvalidValue;
    const int rows = (a->q ? a->heads : 0) + 2 * a->kv_heads, units = (rows + 7) / 8;
    const int64_t total = int64_t(units) * a->total_q, blocks = std::min((total + 3) / 4, MAX_GRID);
    const fav4::FastDiv by_units = fav4::fast_div(units), by_page = fav4::fast_div(a->page_size);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(256), 0, stream, *a, units, total, by_units, by_page);
    };
    if (a->interleaved) go(fav4::append_kernel<true>);
    else go(fav4::append_kernel<false>);
    return hipGetLastError();
}

extern "C" __attribute__((visibility("default"))) long long fav4_bshd_prefix_paged_workspace_size(
    const Fav4PrefixArgs* args, int causal) {
    if (!prefix_shape_ok(args, causal)) return -1;
    const PrefixSizes s = prefix_sizes(*args, causal);
    return s.ok ? s.bytes : -1;
}

extern "C" __attribute__((visibility("default"))) int fav4_bshd_forward_prefix_paged(const Fav4PrefixArgs* args,
                                                                                    int causal, void* workspace,
                                                                                    size_t workspace_bytes,
                                                                                    hipStream_t stream) {
    if (!prefix_shape_ok(args, causal)) return hipErrorInvalidValue;
    const Fav4PagedArgs& a = args->paged;
    if (!a.q || !a.k_cache || !a.v_cache || !a.o || !a.cu_seqlens_q || !a.seqlens_k || !a.block_table ||
        !args->prefix_table || !args->prefix_lens || !args->cu_prefix_seqs ||
        !aligned(16, a.q, a.k_cache, a.v_cache, a.o) ||
        !aligned(4, a.lse, a.cu_seqlens_q, a.seqlens_k, a.block_table, args->prefix_table, args->prefix_lens,
                 args->cu_prefix_seqs))
        return hipErrorInvalidValue;
    PrefixSizes s = prefix_sizes(*args, causal);
    if (!s.ok || !workspace || !aligned(256, workspace) || uint64_t(s.bytes) > workspace_bytes)
        return hipErrorInvalidValue;
    s.plan.o_part = static_cast<float*>(workspace);
    s.plan.lse_part = s.plan.o_part + s.part_rows * fav4::D;
    s.plan.notes = reinterpret_cast<int2*>(s.plan.lse_part + s.part_rows * 2);
    launch_prefix(*args, s, stream);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // Teams per merged row: many where a row can have many parts (24 sequences behind
    // 16384 keys H8 KVH1, 132 parts: 24.6 us on 4, 21.6 on 16), one where it has few or
    // the rows alone fill the GPU (384 sequences behind 1024 keys H32 KVH8: 66.5 on 4,
    // 57.3 on one; 64 behind 8192, 36 parts: 35.8 and 37.7).  The steps lie where 44 such
    // calls changed sides; between those points they are a guess.
    const int64_t rows = int64_t(a.total_q) * a.heads;
    const bool many = (s.parts > 44 && rows <= 256) || (s.parts > 96 && rows <= 1024);
    const bool few = rows > 4096 || s.parts <= 5 || (s.parts <= 18 && rows > 2048);
    const int per = many ? 16 : few ? 1 : 4;
    const unsigned blocks = unsigned(std::min((rows * per + 15) / 16, MAX_GRID));
    auto merge = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream, *args, s.plan, s.prefix_rows);
    };
    if (per == 16) merge(fav4::prefix_merge_kernel<16>);
    else if (per == 4) merge(fav4::prefix_merge_kernel<4>);
    else merge(fav4::prefix_merge_kernel<1>);
    return hipGetLastError();
}
