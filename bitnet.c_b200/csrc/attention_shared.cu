// Attention of one new token for each of several sequences over pages that they share, in bfloat16 on the 5th-generation tensor
// cores: the part of a decode step's attention that sequences forked from one prompt have in common.
//
// A run of shared pages is read once for all its sequences: the query heads that read one key/value head, of up to 128 / (heads per key/value head)
// sequences, are the 128 rows of the products
//     S = Q K^T  (per page: M=128, N=64, K=head size),   P = exp2(S * scale * log2(e) - m),   O += P V
// and every row leaves its maximum m, its sum of P and its unnormalised O in float32.  The kernel that attends over a sequence's own
// pages (attention_decode_tc.cuh) reads them and joins them with its own.  All keys of a run are visible to all its rows (a run ends in front of
// every new token), so nothing is masked.
//
// Which block works on what is a list made on the host: (first member, members and the first one's sequence, first page, pages) per item, members as (sequence, where its
// results go).  Copies bring it to the device, which no kernel overlaps, so it is read in front of the wait; all else is read behind it.  Blocks and roles as in attention_prefill_tc.cu: warp 0 requests pages (TMA, 128-byte swizzle), warp 1 issues the MMAs,
// S of the next page ahead of P V of this one, warps 2 to 5 copy the queries into shared memory and do the softmax, one row per thread.
// P goes back to tensor memory over the columns S came from.  Every wait is bounded; a block whose wait gave up records it and stores nothing.
//
// The bytes bound it, the list of work spreads the pages over five blocks on four SMs, beside which the blocks of the sequences' own pages run: a page takes a
// block about 0.9 us, the tensor cores' part of which is a sixth.  Both kernels together, 32 heads on 8 of 128: 64 sequences behind 8,192 tokens with 500 of
// their own 31.9 us (231 where each reads all its pages), 8 prompts of 2,048 by 8 with 300 of their own 27.0 us.
#include "attention_decode_tc.cuh"
#include "umma.cuh"

#define AS_ROWS 128
#define AS_KEYS BN_PAGE
#define AS_THREADS 192
#define AS_RESCALE 8.0f  // raise a row's reference maximum only beyond this (log2 domain)
#define AS_ERR_WAIT 9

struct AsArgs {
  const __nv_bfloat16* q;  // [n_seqs, q_stride], rotated
  int q_stride, n_seqs, n_heads, n_kv_heads, head_dim, per_group;
  float scale_log2e;
  const int4* items;       // first member, members + 256 * the first one's sequence, first page, pages; no members: nothing to do
  const int2* members;     // sequence, where its results go
  int n_members, n_parts;
  const int* slots;
  const int* page_table;
  int pt_stride;
  float* part_o;           // [n_parts][n_heads][head_dim]
  float* part_ml;          // [n_parts][n_heads][2]
  int* status;
};

__device__ __forceinline__ bool as_wait(unsigned bar, unsigned parity, volatile int* failed, int* status) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = global_timer();
  for (;;) {
    if (mbar_try_wait_for(bar, parity, TMA_SUSPEND_NS)) return true;
    if (*failed) return false;
    if (global_timer() - t0 > TMA_WAIT_NS) {
      *failed = 1;
      atomicExch(status, AS_ERR_WAIT);
      return false;
    }
  }
}

template <int HD, int KS, int VS>
__global__ void __launch_bounds__(AS_THREADS)
attention_shared_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AsArgs a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  constexpr int BOXES = HD / 64, Q_BOX = AS_ROWS * 128, KV_BOX = AS_KEYS * 128, PAGE_BYTES = BOXES * KV_BOX;
  constexpr unsigned TMEM_COLS = 256, O_COL = 128;  // S0 at 0, S1 at 64, O at 128
  constexpr unsigned IDESC_S = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(AS_KEYS >> 3) << 17) | ((AS_ROWS >> 4) << 24);
  constexpr unsigned IDESC_O = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((unsigned)(HD >> 3) << 17) | ((AS_ROWS >> 4) << 24);
  unsigned char* q_smem = smem_raw;  // (no static shared memory: the base is 1024-byte aligned, and the swizzle a function of the address)
  unsigned char* k_smem = q_smem + BOXES * Q_BOX;
  unsigned char* v_smem = k_smem + KS * PAGE_BYTES;
  unsigned long long* bars = (unsigned long long*)(v_smem + VS * PAGE_BYTES);
  const unsigned q_full = smem_u32(bars), k_full0 = q_full + 8, k_empty0 = k_full0 + 8 * KS, v_full0 = k_empty0 + 8 * KS,
                 v_empty0 = v_full0 + 8 * VS, s_full0 = v_empty0 + 8 * VS, p_full0 = s_full0 + 16, pv_done0 = p_full0 + 16;
  unsigned* tmem_slot = (unsigned*)(bars + 2 * KS + 2 * VS + 7);
  volatile int* failed = (volatile int*)(tmem_slot + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.x;
  const int4 item = a.items[blockIdx.y];
  const int n_tiles = item.w, n_members = item.y & 255;
  if (n_members <= 0 || n_tiles <= 0 || item.x < 0 || item.x + n_members > a.n_members || (item.y >> 8) >= a.n_seqs || item.z < 0 || item.z + n_tiles > a.pt_stride) {
    pdl_wait();
    return;
  }
  const int rows = min(AS_ROWS, n_members * a.per_group);
  const int2* members = a.members + item.x;

  if (tid == 0) {
    *failed = 0;
    if (smem_u32(smem_raw) & 1023u) {
      *failed = 1;
      atomicExch(a.status, AS_ERR_WAIT);
    }
    tma_prefetch_map(&map_k);
    tma_prefetch_map(&map_v);
    mbar_init(q_full, 4);
    for (int s = 0; s < KS; ++s) { mbar_init(k_full0 + 8 * s, 1); mbar_init(k_empty0 + 8 * s, 1); }
    for (int s = 0; s < VS; ++s) { mbar_init(v_full0 + 8 * s, 1); mbar_init(v_empty0 + 8 * s, 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(s_full0 + 8 * b, 1); mbar_init(p_full0 + 8 * b, 4); mbar_init(pv_done0 + 8 * b, 1); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem_base = *tmem_slot;

  if (warp == 0) {
    // (whatever filled the pages, or chose the slots, may still run before that: asking in front of it was worth 0.5 us of 27 for 64 sequences, less for others)
    pdl_wait();
    if (lane == 0) {
      const int* pt = a.page_table + (size_t)a.slots[item.y >> 8] * a.pt_stride + item.z;
      auto request = [&](int j, bool values) -> bool {
        const int n = values ? VS : KS, s = j % n, round = j / n;
        const unsigned empty = (values ? v_empty0 : k_empty0) + 8 * s, bar = (values ? v_full0 : k_full0) + 8 * s;
        const int page = __ldg(pt + j);
        if (round > 0 && !as_wait(empty, (unsigned)(round - 1) & 1u, failed, a.status)) return false;
        const unsigned dst = smem_u32(values ? v_smem + s * PAGE_BYTES : k_smem + s * PAGE_BYTES);
        mbar_expect_tx(bar, PAGE_BYTES);
#pragma unroll
        for (int bx = 0; bx < BOXES; ++bx) tma_load_3d(dst + bx * KV_BOX, values ? &map_v : &map_k, bar, bx * 64, kvh * BN_PAGE, page);
        return true;
      };
      bool ok = !*failed;
      for (int j = 0; ok && j < min(KS - 1, n_tiles); ++j) ok = request(j, false);
      for (int t = 0; ok && t < n_tiles; ++t) {
        if (t + KS - 1 < n_tiles) ok = request(t + KS - 1, false);
        if (ok) ok = request(t, true);
      }
    }
  } else if (warp == 1) {
    pdl_wait();
    // the whole warp walks the loop, one elected lane issues
    const bool issuer = elect_one();
    const unsigned tbase = __shfl_sync(0xffffffffu, tmem_base, 0);
    bool ok = __all_sync(0xffffffffu, as_wait(q_full, 0, failed, a.status));
    const unsigned sq = smem_u32(q_smem);
    for (int j = 0; ok && j <= n_tiles; ++j) {
      if (j < n_tiles) {
        const int s = j % KS, b = j & 1;
        ok = __all_sync(0xffffffffu, as_wait(k_full0 + 8 * s, (unsigned)(j / KS) & 1u, failed, a.status));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const unsigned sk = smem_u32(k_smem + s * PAGE_BYTES);
        if (issuer) {
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks)
            umma_mma(tbase + b * AS_KEYS, umma_desc_k(sq + (ks >> 2) * Q_BOX + (ks & 3) * 32), umma_desc_k(sk + (ks >> 2) * KV_BOX + (ks & 3) * 32),
                     IDESC_S, ks ? 1u : 0u);
          umma_commit(k_empty0 + 8 * s);
          umma_commit(s_full0 + 8 * b);
        }
        __syncwarp();
      }
      if (j >= 1) {
        const int i = j - 1, s = i % VS, b = i & 1;
        ok = __all_sync(0xffffffffu, as_wait(p_full0 + 8 * b, (unsigned)(i >> 1) & 1u, failed, a.status) &&
                                         as_wait(v_full0 + 8 * s, (unsigned)(i / VS) & 1u, failed, a.status));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const unsigned sv = smem_u32(v_smem + s * PAGE_BYTES);
        if (issuer) {
#pragma unroll
          for (int kk = 0; kk < AS_KEYS / 16; ++kk)
            umma_mma_ts(tbase + O_COL, tbase + b * AS_KEYS + kk * 8, umma_desc_mn(sv + kk * 2048, KV_BOX), IDESC_O, (i | kk) ? 1u : 0u);
          umma_commit(v_empty0 + 8 * s);
          umma_commit(pv_done0 + 8 * b);
        }
        __syncwarp();
      }
    }
  } else {
    // ---- the queries, into the layout that TMA would leave: boxes of 128 rows x 64 numbers, 16-byte pieces XORed with the row.  A thread copies one piece
    // of every eighth (or sixteenth) row, all of its loads in flight before the first store; whose rows they are is known before the wait.
    {
      constexpr int PIECES = HD / 8, EACH = PIECES, APART = 128 / PIECES;
      const int t = tid - 64, c = t % PIECES, row0 = t / PIECES;
      int from[EACH];
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int row = row0 + e * APART, member = row / a.per_group;
        from[e] = -1;
        if (row < rows && c * 8 < a.head_dim) from[e] = members[member].x * a.q_stride + (kvh * a.per_group + row - member * a.per_group) * a.head_dim + c * 8;
      }
      pdl_wait();
      uint4 v[EACH];
#pragma unroll
      for (int e = 0; e < EACH; ++e) v[e] = from[e] >= 0 ? *reinterpret_cast<const uint4*>(a.q + from[e]) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int row = row0 + e * APART;
        *reinterpret_cast<uint4*>(q_smem + (c >> 3) * Q_BOX + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = v[e];
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
    // behind the wait, so that what the next kernel reads of this one's predecessor is there; and behind the queries, so that they do not queue
    // behind the pages that it asks for
    pdl_launch_dependents();
    // ---- softmax: thread <-> row <-> lane of tensor memory
    const int quad = warp & 3, r = quad * 32 + lane;
    const unsigned lane_addr = tmem_base + ((unsigned)(quad * 32) << 16);
    const bool active = quad * 32 < rows;  // a warp without a row only keeps the barriers going: its lanes' results are not read
    float m_ref = -INFINITY, l_run = 0.f;
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      const int b = j & 1;
      if (!as_wait(s_full0 + 8 * b, (unsigned)(j >> 1) & 1u, failed, a.status)) { ok = false; break; }
      // (each phase of both barriers is waited for in turn, so that a parity always means the phase that is asked for)
      if (j >= 2 && !as_wait(pv_done0 + 8 * b, (unsigned)((j >> 1) - 1) & 1u, failed, a.status)) { ok = false; break; }
      if (active) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        float s[AS_KEYS];
        tmem_ld64(lane_addr + b * AS_KEYS, s);
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int k = 4; k < AS_KEYS; ++k) mx[k & 3] = fmaxf(mx[k & 3], s[k]);
        const float m_tile = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2e;
        bool need = false;
        if (m_ref == -INFINITY) m_ref = m_tile;  // nothing accumulated yet: O and the sum are zero
        else need = m_tile > m_ref + AS_RESCALE;
        if (__any_sync(0xffffffffu, need)) {
          if (!as_wait(pv_done0 + 8 * ((j - 1) & 1), (unsigned)((j - 1) >> 1) & 1u, failed, a.status)) { ok = false; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const float alpha = need ? exp2f(m_ref - m_tile) : 1.0f;
          if (need) { m_ref = m_tile; l_run *= alpha; }
#pragma unroll
          for (int c = 0; c < HD; c += 32) {
            float o[32];
            tmem_ld32(lane_addr + O_COL + c, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= alpha;
            tmem_st32(lane_addr + O_COL + c, o);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        const float neg_m = (m_ref == -INFINITY) ? 0.f : -m_ref;
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < AS_KEYS; ++k) {
          s[k] = ex2_approx(fmaf(s[k], a.scale_log2e, neg_m));
          ls[k & 3] += s[k];
        }
        l_run += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        float pk[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) pk[c] = __uint_as_float(pack_bf16x2(s[2 * c], s[2 * c + 1]));
        tmem_st32(lane_addr + b * AS_KEYS, pk);
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full0 + 8 * b);
    }
    // ---- maximum, sum and O of every row
    if (ok && n_tiles > 1) ok = as_wait(pv_done0 + 8 * ((n_tiles - 2) & 1), (unsigned)((n_tiles - 2) >> 1) & 1u, failed, a.status);
    if (ok && as_wait(pv_done0 + 8 * ((n_tiles - 1) & 1), (unsigned)((n_tiles - 1) >> 1) & 1u, failed, a.status) && active) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int part = r < rows ? members[r / a.per_group].y : -1, h = kvh * a.per_group + r % a.per_group;
      const bool store = part >= 0 && part < a.n_parts;
      const size_t at = (size_t)part * a.n_heads + h;
      if (store) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m_ref, l_run);
      // A row of O lies in one lane: by way of shared memory (the queries and pages are done with), where rows of OSTRIDE bytes keep the lanes of a store
      // on different banks, it goes out as one copy of the row
      constexpr int OSTRIDE = HD * 4 + 16;
      static_assert(AS_ROWS * OSTRIDE <= BOXES * Q_BOX + (KS + VS) * PAGE_BYTES, "the rows of O reuse the queries' and pages' room");
      unsigned char* orow = q_smem + r * OSTRIDE;
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        float o[32];
        tmem_ld32(lane_addr + O_COL + c, o);
#pragma unroll
        for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(orow + (c + i) * 4) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (store) {
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(a.part_o + at * a.head_dim), "r"(smem_u32(orow)), "r"(a.head_dim * 4)
                     : "memory");
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*failed) {  // loads that were requested may still be landing in this block's shared memory
    const unsigned long long t0 = global_timer();
    while (global_timer() - t0 < 200000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

template <int HD, int KS, int VS>
static int as_launch(const CUtensorMap& mk, const CUtensorMap& mv, const AsArgs& a, int n_items, cudaStream_t stream) {
  const size_t smem = (size_t)AS_ROWS * HD * 2 + (size_t)(KS + VS) * AS_KEYS * HD * 2 + (2 * KS + 2 * VS + 7) * 8 + 16;
  static BnGrant grant;
  const cudaError_t e = grant.ask((const void*)attention_shared_kernel<HD, KS, VS>, smem, 0);
  if (e != cudaSuccess) return BN_ERR_LAUNCH + (int)e;
  BN_LAUNCH((attention_shared_kernel<HD, KS, VS>), dim3(a.n_kv_heads, n_items), AS_THREADS, smem, stream, mk, mv, a);
  return BN_OK;
}

// The kernel above and directly behind it the joining form of attention_decode_tc.cuh (one call from the host: two take it 3 us more; and that form relies on what is in front).  qkv: [n_seqs, q_stride] bfloat16 rows, rotated, query head h at
// element h * head_dim, key heads at k_off, value heads at v_off, 16-byte aligned, q_stride a multiple of 8.  items [n_items], members [n_parts] and
// sequences [n_seqs] (pages, first result, results, which sequence; those with the most pages of their own first) as above and there; part_o [n_parts, n_heads, head_dim] and part_ml [n_parts, n_heads, 2] are written where members say.  n_splits blocks, 8 at
// most, share each sequence's own pages evenly.  The caches are
// [n_cache_pages, n_kv_heads, 64, head_dim], contiguous and 16-byte aligned.  head_dim: a multiple of 16 up to 128; n_heads / n_kv_heads at
// most 128.  status: one int, left as it is unless a wait gave up (then 9, or the other kernel's).
extern "C" int bn_attention_shared(const void* qkv, int q_stride, int k_off, int v_off, void* out, int out_stride, int n_seqs, int n_heads,
                                   int n_kv_heads, int head_dim, float scale, const int* items, int n_items, const int* members, int n_parts,
                                   const int* sequences, const int* tok_pos, const int* slots, const int* page_table, int pt_stride, void* k_cache,
                                   void* v_cache, int n_cache_pages, float* part_o, float* part_ml, int n_splits,
                                   int* status, cudaStream_t stream) {
  if (n_seqs <= 0) return BN_OK;
  if (n_items <= 0 || head_dim <= 0 || head_dim % 16 || head_dim > 128 || n_kv_heads <= 0 || n_heads % n_kv_heads || n_heads / n_kv_heads > AS_ROWS || !(scale > 0.f) ||
      q_stride % 8 || (long long)n_seqs * q_stride > 0x7fffffffll || n_items > 65535 || n_cache_pages <= 0 || n_parts <= 0 || !items || !members || !sequences || !part_o || !part_ml || !status ||
      (((uintptr_t)qkv | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)items | (uintptr_t)part_o) & 15) || ((uintptr_t)sequences & 15) || (((uintptr_t)members | (uintptr_t)part_ml) & 7))
    return BN_ERR_BAD_ARG;
  CUtensorMap mk, mv;
  if (!tma_map_bf16_pages(&mk, k_cache, n_cache_pages, (unsigned long long)n_kv_heads * BN_PAGE, head_dim, BN_PAGE) ||
      !tma_map_bf16_pages(&mv, v_cache, n_cache_pages, (unsigned long long)n_kv_heads * BN_PAGE, head_dim, BN_PAGE))
    return BN_ERR_BAD_ARG;
  AsArgs a = {};
  a.q = (const __nv_bfloat16*)qkv; a.q_stride = q_stride; a.n_seqs = n_seqs; a.n_heads = n_heads; a.n_kv_heads = n_kv_heads; a.head_dim = head_dim;
  a.per_group = n_heads / n_kv_heads; a.scale_log2e = scale * 1.4426950408889634f; a.items = (const int4*)items; a.members = (const int2*)members;
  a.n_members = n_parts; a.n_parts = n_parts; a.slots = slots; a.page_table = page_table; a.pt_stride = pt_stride; a.part_o = part_o;
  a.part_ml = part_ml; a.status = status;
  // 64 KB and 112 KB: room for blocks of the sequences' own pages on the same SM, or for a second one of these (64 behind 8,192 and 8 by 8: 31.9 and 27.0 us; 128 KB
  // with rings of three and three: 32.4 and 36.0; 96 KB with two and two: 32.2 and 27.2)
  const int rc = head_dim <= 64 ? as_launch<64, 3, 3>(mk, mv, a, n_items, stream) : as_launch<128, 3, 2>(mk, mv, a, n_items, stream);
  if (rc != BN_OK) return rc;
  return dt_run<true>(qkv, q_stride, k_off, v_off, out, out_stride, n_seqs, n_heads, n_kv_heads, head_dim, scale, 0, 0, 1.0f, tok_pos, slots, page_table, pt_stride,
                      k_cache, v_cache, n_cache_pages, status, nullptr, nullptr, n_splits, 1, nullptr, 0, nullptr, 0, 0, sequences, part_o, part_ml, n_parts,
                      stream);
}
