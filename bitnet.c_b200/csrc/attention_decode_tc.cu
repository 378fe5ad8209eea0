// Entries of the decode attention of attention_decode_tc.cuh, in which one kernel does all.
#include "attention_decode_tc.cuh"

// qkv: [n_seqs, q_stride] bfloat16 rows with the raw query heads first, the key heads at element
// k_off and the value heads at v_off (all multiples of 8 elements).  The kernel rotates queries and
// the new key (rotary_dims = 0: none), writes the new key and value into the cache at tok_pos[b],
// attends and combines.  A block walks pages_per_block pages of 64 positions; n_splits blocks cover
// a sequence, so n_splits * pages_per_block * 64 must cover the longest sequence.  part_o / part_ml:
// scratch of n_seqs * n_heads * n_splits * head_dim and n_seqs * n_heads * n_splits * 2 floats (unused
// when n_splits is 1); tickets: n_seqs * n_kv_heads * ceil(group / 16) ints, zero before and after.
// The caches are [n_cache_pages, n_kv_heads, 64, head_dim], contiguous and 16-byte aligned.  status:
// one int on the device, left as it is unless a page load never completed (then 4, and the output
// of that launch is not valid).
//
// With items (n_items ints on the device, a multiple of group; group 1 to 8): block x of the grid
// works on what items[x] names, sequence | split << 16 | splits << 24, or on nothing (-1).  Clusters
// of `group` blocks run along x; a cluster must hold either the `group` splits of one sequence, in
// order, or sequences that are not split (splits = 1) and padding.  n_splits and pages_per_block
// are not used then.  This is how a batch of unequal lengths gets more blocks for its long
// sequences than for its short ones, and its long ones started first.
extern "C" int bn_attention_decode_tc(const void* qkv, int q_stride, int k_off, int v_off, void* out, int out_stride,
                                      int n_seqs, int n_heads, int n_kv_heads, int head_dim, float scale, int window,
                                      int rotary_dims, float theta_scale, const int* tok_pos, const int* slots,
                                      const int* page_table, int pt_stride, void* k_cache, void* v_cache,
                                      int n_cache_pages, int* status, float* part_o, float* part_ml, int n_splits, int pages_per_block, int* tickets,
                                      int n_tickets, cudaStream_t stream) {
  return dt_run<false>(qkv, q_stride, k_off, v_off, out, out_stride, n_seqs, n_heads, n_kv_heads, head_dim, scale, window, rotary_dims,
                       theta_scale, tok_pos, slots, page_table, pt_stride, k_cache, v_cache, n_cache_pages, status, part_o, part_ml,
                       n_splits, pages_per_block, tickets, n_tickets, nullptr, 0, 0, nullptr, nullptr, nullptr, 0, stream);
}
extern "C" int bn_attention_decode_tc_items(const void* qkv, int q_stride, int k_off, int v_off, void* out, int out_stride,
                                            int n_seqs, int n_heads, int n_kv_heads, int head_dim, float scale, int window,
                                            int rotary_dims, float theta_scale, const int* tok_pos, const int* slots,
                                            const int* page_table, int pt_stride, void* k_cache, void* v_cache,
                                            int n_cache_pages, int* status, float* part_o, float* part_ml, int* tickets,
                                            int n_tickets, const int* items, int n_items, int item_group, cudaStream_t stream) {
  if (!items) return BN_ERR_BAD_ARG;
  return dt_run<false>(qkv, q_stride, k_off, v_off, out, out_stride, n_seqs, n_heads, n_kv_heads, head_dim, scale, window, rotary_dims,
                       theta_scale, tok_pos, slots, page_table, pt_stride, k_cache, v_cache, n_cache_pages, status, part_o, part_ml,
                       1, 1, tickets, n_tickets, items, n_items, item_group, nullptr, nullptr, nullptr, 0, stream);
}
