#pragma once
// C ABI of the serving operators on paged K/V caches (build/libfav4_serving.so,
// MI355X / gfx950).  No counterpart in the reference.  BF16 at head dimension
// 128, with the caches, block tables and packed sequences of
// fav4_bshd_forward_splitkv_paged (fav4_bshd.h), whose contract they share:
//  * every pointer is device memory of the calling thread's current device;
//    a call only enqueues work on `stream`, allocates nothing and never
//    synchronizes, so it can be captured in a HIP graph;
//  * sizes and pointers are checked before any HIP call (hipErrorInvalidValue
//    = 1); lengths, offsets and page numbers are read on the device and
//    clamped or skipped, so bad ones give undefined values but no access
//    outside the buffers.
#include "fav4_bshd.h"

// ---- Appending to paged K/V caches ------------------------------------------
// Stores the new tokens' K and V rows in the caches, K and Q rotated by
// position on the way.  Sequence b's tokens are rows [cu_seqlens_q[b],
// cu_seqlens_q[b + 1]) of q, k and v; seqlens_k[b] counts its keys with the new
// ones (the value that the attention call after it takes), so the i-th of its
// sq tokens goes to slot seqlens_k[b] - sq + i, in page
// block_table[b * max_pages_per_seq + slot / page_size].
//  * Rotation of the first rotary_dim dims of each head by the angles of row p
//    of cos / sin, p = positions[token], or the token's slot where positions is
//    NULL: (x, y) -> (x cos - y sin, y cos + x sin) in FP32, rounded once.  The
//    pairs are dims (j, j + rotary_dim / 2), or neighbours (2j, 2j + 1) where
//    interleaved; angle j of the row belongs to pair j.  Other dims, and V, are
//    copied.  rotary_dim 0 (cos and sin NULL): nothing is rotated.
//  * A token whose slot is negative or past the table, or whose page number is
//    not in [0, num_pages) (an idle slot's -1), is not stored.  Its q_out row
//    is written all the same.  p is clamped to [0, rotary_rows).
//  * Tokens in no sequence (behind the last one) are neither read nor written.
//  * Two tokens of one call must not have the same slot (undefined which stays).
struct Fav4AppendArgs {
    const void *q, *k, *v;             // BF16 rows [total_q, heads | kv_heads, 128]; q may be NULL (with q_out)
    void *q_out;                       // BF16 [total_q, heads, 128]: rotated Q; may be q (in place, same stride)
    void *k_cache, *v_cache;           // BF16 [num_pages, page_size, kv_heads, 128], contiguous
    const float *cos, *sin;            // FP32 [rotary_rows, rotary_dim / 2], contiguous
    const int *cu_seqlens_q;           // device int32 [batch + 1], non-decreasing
    const int *seqlens_k;              // device int32 [batch]: keys per sequence, the new ones included
    const int *block_table;            // device int32 [batch, max_pages_per_seq]
    const int *positions;              // optional device int32 [total_q]
    long long q_stride, k_stride, v_stride, q_out_stride;   // elements from token to token
    int batch, heads, kv_heads, total_q;
    int num_pages, page_size, max_pages_per_seq;
    int rotary_dim, rotary_rows, interleaved;
};
// Checks: the pointers (q and q_out both or neither; cos and sin with
// rotary_dim > 0), sizes >= 1, rotary_dim a multiple of 16 up to 128,
// rotary_rows >= 1 where it is not 0, interleaved 0 or 1, strides of at least
// heads * 128 (kv_heads * 128) elements that are multiples of 8, q_out_stride =
// q_stride where q_out is q, 16-byte aligned rows and tables of angles, 4-byte
// aligned int arrays, (heads + 2 kv_heads) * total_q < 2^31, batch <= 2^31 - 64
// and tensors of less than 2^48 bytes.
extern "C" int fav4_bshd_append_paged(const Fav4AppendArgs* args, hipStream_t stream);

// ---- Attention behind shared prefixes ----------------------------------------
// fav4_bshd_forward_splitkv_paged for batches whose sequences share leading
// pages: one system prompt, several samples of a prompt, beams.  Prefix p is
// shared by the sequences [cu_prefix_seqs[p], cu_prefix_seqs[p + 1]); its keys
// are the pages prefix_table[p * max_pages_per_prefix + ...], prefix_lens[p]
// keys in whole pages (a rest is left to the sequences' own pages).  Key j of a
// sequence of prefix p lies in prefix_table[p] for j < prefix_lens[p] and in
// its own row of block_table, entry j / page_size as ever, from there on; the
// entries of block_table before that are not read.  seqlens_k counts all keys.
// The rows of all sequences of a prefix read its keys together; each sequence
// then reads its own, and the parts are merged by their log-sum-exp.
//  * Any number of new queries per sequence, dense (causal 0) or bottom-right
//    causal (2).  Sequences in no prefix, or of a prefix without keys, are
//    attended over their own pages alone.  A sequence with fewer keys than its
//    prefix sees those alone (max_seqlen_k bounds the sequences' keys, and may
//    lie inside a prefix); one without keys gets O = 0 and LSE = -inf, one
//    without queries writes nothing.
//  * K and V of every key in [0, seqlens_k) and of every shared key must be
//    finite, also for rows that do not see it: hidden keys have weight 0, and 0
//    times a NaN is one.  Slots behind seqlens_k may hold anything.  A row whose
//    query holds a NaN and that sees a key gets O and LSE of NaN; no query changes
//    another row.
//  * Results meet the tolerances of the paged call (not bitwise its results:
//    the parts are cut elsewhere), and are the same from call to call.
struct Fav4PrefixArgs {
    Fav4PagedArgs paged;               // as for fav4_bshd_forward_splitkv_paged (total_k is not used)
    const int *prefix_table;           // device int32 [num_prefixes, max_pages_per_prefix]: page numbers
    const int *prefix_lens;            // device int32 [num_prefixes]: shared keys
    const int *cu_prefix_seqs;         // device int32 [num_prefixes + 1], non-decreasing: sequences of each prefix
    int num_prefixes, max_pages_per_prefix;
};
// Checks: those of Fav4PagedArgs with causal 0 or 2, page_size a multiple of 32,
// max_seqlen_k <= max_pages_per_seq * page_size and in whole pages < 2^31 - 255,
// num_prefixes and max_pages_per_prefix >= 1, heads <= 2^15, total_q * heads <
// 2^31, and a plan of fewer than 2^30 key tiles.  The workspace is caller-owned
// device memory, 256-byte aligned, of at least
// fav4_bshd_prefix_paged_workspace_size() bytes and not shared with a concurrent
// call (two captured graphs that may run at once included); its contents do not
// matter.  The size query reads only the sizes (pointers may be NULL), returns
// -1 for rejected arguments, and never less for a larger batch, more queries,
// prefixes or pages: it counts what any cut of the call could need, about twice
// what a decode step lays out (80 MB for 64 sequences, 32 heads on 8).
//
// Sizes that steer the speed: up to 32 * num_prefixes rows (total_q * heads /
// kv_heads) are taken for few rows a prefix, slots without sequences counted, so
// num_prefixes should be near the number in use.  A sequence with fewer keys
// than its prefix (an idle slot inside its range) makes the prefix tiles of the
// whole call masked ones, as more than 512 sequences or 256 prefixes do: idle
// slots are better behind the last prefix.
extern "C" int fav4_bshd_forward_prefix_paged(const Fav4PrefixArgs* args, int causal, void* workspace,
                                              size_t workspace_bytes, hipStream_t stream);
extern "C" long long fav4_bshd_prefix_paged_workspace_size(const Fav4PrefixArgs* args, int causal);
