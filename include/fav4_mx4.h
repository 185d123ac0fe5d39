#pragma once
// C ABI of the operators of 4-bit paged K/V caches (build/libfav4_mx4.so, MI355X /
// gfx950): storing, reading back, attending.  No counterpart in the reference.
// Sequences, block tables and the rules of a call are those of fav4_serving.h:
//  * every pointer is device memory of the calling thread's current device;
//    a call only enqueues work on `stream`, allocates nothing and never
//    synchronizes, so it can be captured in a HIP graph;
//  * sizes and pointers are checked before any HIP call (hipErrorInvalidValue
//    = 1); lengths, offsets and page numbers are read on the device and
//    clamped or skipped, so bad ones give undefined values but no access
//    outside the buffers.
//
// A cache row (the 128 dims of one key and K/V head) is MXFP4: 64 bytes of E2M1
// codes, dims 2i and 2i + 1 in the low and the high half of byte i, and four E8M0
// scales: the number in a dim of block j (dims 32j to 32j + 31) is
// +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}[code & 7] * 2^(scale[j] - 127), negative where
// code & 8.  Scales of 253 to 255 make their block no numbers (NaN; an append writes 255
// alone).  All others are exact in BF16; with scales of 0 and 1 numbers below 2^-126 may
// count as 0.
// The caches of K and of V are each two tensors, contiguous, head before slot, so
// that the keys of a page and head that a workgroup reads lie side by side:
//   codes   uint8 [num_pages, kv_heads, page_size, 64]
//   scales  uint8 [num_pages, kv_heads, page_size, 4]
#include "fav4_serving.h"

// ---- Appending -----------------------------------------------------------------
// fav4_bshd_append_paged (fav4_serving.h) for such caches: the same tokens, slots,
// rotation and outputs, with append.k_cache and append.v_cache the codes.
//  * K is rotated in FP32, each product and the sum rounded once, and that number
//    quantised, not one rounded to BF16 before.  Q is rounded to BF16.
//  * A block's scale is the smallest power of two 2^e with max |x| <= 7 * 2^e, e in
//    [-125, 125]: numbers between 6 and 7 times the scale become 6, which is nearer
//    to them than the grid of the next scale is on average (relative error of normal
//    numbers 0.112; 0.115 with 6 or with 8 in place of 7).  Each number goes to the
//    nearest value of the grid, ties to the even code; numbers below 2^-126 count as 0.
//  * A block that holds an infinity or a NaN gets scale 255 and codes 0.
struct Fav4Mx4AppendArgs {
    Fav4AppendArgs append;             // k_cache, v_cache: codes
    void *k_scales, *v_scales;
};
// Checks: those of fav4_bshd_append_paged, 16-byte aligned scales.
extern "C" int fav4_bshd_append_paged_mx4(const Fav4Mx4AppendArgs* args, hipStream_t stream);

// ---- Reading back ----------------------------------------------------------------
// The numbers that the caches hold, as BF16 rows of a packed batch (what
// fav4_bshd_forward_varlen takes as K and V): rows [cu_seqlens_k[b],
// cu_seqlens_k[b + 1]) of k and v get keys starts[b], starts[b] + 1, ... of sequence
// b (0, 1, ... where starts is NULL).
//  * A row whose slot is negative or past the table, or whose page number is not in
//    [0, num_pages), becomes 0.  Blocks of scales above 252 become NaN.
//  * Rows in no sequence (behind the last one) are not written.
struct Fav4Mx4GatherArgs {
    const void *k_cache, *k_scales, *v_cache, *v_scales;
    void *k, *v;                       // BF16 rows [total_k, kv_heads, 128]
    const int *cu_seqlens_k;           // device int32 [batch + 1], non-decreasing
    const int *starts;                 // optional device int32 [batch]
    const int *block_table;            // device int32 [batch, max_pages_per_seq]
    long long k_stride, v_stride;      // elements from row to row
    int batch, kv_heads, total_k;
    int num_pages, page_size, max_pages_per_seq;
};
// Checks: the pointers, sizes >= 1, strides of at least kv_heads * 128 elements that
// are multiples of 8, 16-byte aligned rows and caches, 4-byte aligned int arrays,
// 2 kv_heads * total_k < 2^31, batch <= 2^31 - 64, tensors of less than 2^48 bytes.
extern "C" int fav4_bshd_gather_paged_mx4(const Fav4Mx4GatherArgs* args, hipStream_t stream);

// ---- Attention -------------------------------------------------------------------
// The paged call (fav4_bshd_forward_splitkv_paged, fav4_bshd.h) over such caches: new
// queries of each sequence, any number of them, dense (causal 0) or bottom-right causal
// (2), against its keys.  A sequence without keys, and rows that see no key, get O = 0
// and LSE = -inf; a sequence without queries writes nothing, nor do rows in no sequence.
//  * A key with a scale above 252 in any block of its K or V is no number: a row that sees
//    it gets O and LSE of NaN in all dims, and so does one whose query holds a NaN; rows
//    that do not see the key are not touched by it, nor by what slots behind seqlens_k
//    and hidden keys hold.
//  * A query that holds an infinity has no finite score: its row's O and LSE are NaN, or as
//    without keys where all its scores are -inf.
//  * Scores and sums are FP32.  Where one passes 3.4e38 (with queries of about 1 that takes
//    keys of some 1e36, and an append stores numbers of up to 2.6e38), O and LSE of the rows
//    that see the key are infinite or NaN, and of no others.
//  * K and V enter the matrix products as BF16, which holds their numbers exactly;
//    weights are rounded to BF16 and O is divided by the sum of the rounded ones, as in
//    the forward.  Results are the same from call to call.
//  * total_k, the sum of seqlens_k, steers how the call is cut and nothing else, by a rule
//    that is not fav4_bshd.h's: 0 says that the sum is not known, and every sequence is then
//    taken for max_seqlen_k long, as with batch * max_seqlen_k; one less than that is a sum
//    like any other.  The cut is chosen on the host, so a captured call keeps it.  Where
//    all sequences are taken for long and there are no more pairs of one and a K/V head than
//    CUs, each pair gets a workgroup: 32 x 1 queries, 32 / 8 heads, max_seqlen_k 32768, with
//    the sum and without: one of 32768 keys and 31 of 300 19 and 116 us, all of 300 18 and 6,
//    all of 32768 169 both.
struct Fav4Mx4PagedArgs {
    Fav4PagedArgs paged;               // k_cache, v_cache: codes
    const void *k_scales, *v_scales;
};
// Checks: those of Fav4PagedArgs with causal 0 or 2, page_size a multiple of 16,
// max_seqlen_k <= max_pages_per_seq * page_size and in whole pages < 2^31 - 255, heads
// <= 2^15, total_q * heads < 2^31, 16-byte aligned scales, caches of less than 2^48
// bytes, and a plan of fewer than 10^9 key tiles, at most 2^22 row tiles, and fewer than
// 2^23 row tiles over all K/V heads.  The workspace is caller-owned device memory,
// 256-byte aligned, of at least fav4_bshd_paged_mx4_workspace_size() bytes and not shared
// with a concurrent call (two captured graphs that may run at once included); its
// contents do not matter.  The size query reads only the sizes (pointers may be NULL),
// returns -1 for rejected arguments, and never less for a larger batch or more queries:
// the size follows from kv_heads and from whether a sequence may have more than 64 rows.
extern "C" int fav4_bshd_forward_paged_mx4(const Fav4Mx4PagedArgs* args, int causal, void* workspace,
                                           size_t workspace_bytes, hipStream_t stream);
extern "C" long long fav4_bshd_paged_mx4_workspace_size(const Fav4Mx4PagedArgs* args, int causal);
