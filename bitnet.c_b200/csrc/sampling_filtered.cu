// The next token from temperature, top-k, top-p and min-p, from a given random number per row.
//
// Sorted order of a row: falling logits, equal ones by rising index; NaN counts as -inf and -inf is never chosen.  With
// w_i = exp((l_i - max) / T):  K1 the first k;  K2 of K1 up to the first whose running sum exceeds top_p * sum(K1);  K3 those of K2 with
// w_i >= min_p;  the token is the first of K3 whose running sum exceeds u * sum(K3).  Each set is a beginning of the sorted order, so nothing
// is sorted: every border is "the first whose running sum (of ones, or of weights) exceeds a number", found by the bits of the logits.
//
// A cluster of blocks holds a row in its shared memory as ordered 32-bit keys, so that memory is read once however many passes
// follow.  A pass over a level of 11, 11 or 10 bits adds the ones or weights of the keys that agree with the bits found
// so far into a histogram per block; the blocks then add up a share of the bins each, over the cluster, and the one
// whose bins hold the border tells the others.
// Weights are numbers of 64 bits in fixed point: sums do not depend on the order of additions, and a running sum that lies next to a
// border falls on the same side as in a sum of doubles (rounding to 2^-45 a token at a vocabulary of 2^17; a float sum would move a token in
// a thousand).
#include "common.cuh"

#define SF_THREADS 512
#define SF_BINS 2048
#define SF_MAX_CLUSTER 8

struct SfArgs {
  const void* logits;
  long long ld;
  int vocab, per;  // per: numbers of a row that each block of the cluster holds, a multiple of 8
  float temperature, top_p, min_p;
  int top_k;
  const float* temperatures;  // per row, or null: the numbers above
  const int* top_ks;
  const float* top_ps;
  const float* min_ps;
  const float* u;             // per row, or null: drawn from rng
  unsigned long long* rng;
  const int* index;           // row -> its generator, or null
  int* out;
  int scale_bits;             // weights are multiples of 2^-scale_bits
};

__device__ __forceinline__ unsigned sf_key(float v) {
  if (!(v > -INFINITY)) return 0u;  // -inf and NaN
  const unsigned b = __float_as_uint(v + 0.f);  // -0 is 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sf_value(unsigned key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

__device__ __forceinline__ unsigned sf_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned sf_size() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void sf_sync() {  // all threads of the cluster; what they wrote to shared memory is seen by all
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned sf_remote(const void* p, unsigned rank) {
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ unsigned long long sf_load(const unsigned long long* p, unsigned rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(sf_remote(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void sf_store(unsigned long long* p, unsigned rank, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(sf_remote(p, rank)), "l"(v) : "memory");
}

struct SfShared {
  unsigned long long hist[SF_BINS];
  unsigned long long warp[SF_THREADS / 32];
  // one entry per block of the cluster, written by that block; two sets in turn, so that one barrier per exchange is enough
  unsigned long long part[2][SF_MAX_CLUSTER];
  unsigned long long found[2];  // what the block that found a border tells the others
};

template <typename T, bool RESIDENT>
struct SfRow {
  SfArgs a;
  SfShared& s;
  const unsigned* keys;  // shared memory, RESIDENT
  const T* row;          // this block's part of the row
  int n;                 // numbers of it
  unsigned rank, blocks;
  int turn = 0;
  double top, per_t;     // the largest logit, 1 / temperature
  bool infinite;         // the largest logit is +inf: those share everything

  __device__ __forceinline__ unsigned key(int i) const { return RESIDENT ? keys[i] : sf_key(to_f32<T>(row[i])); }
  __device__ __forceinline__ double weight(unsigned k) const {
    const double v = (double)sf_value(k);
    return infinite ? (v == top ? 1.0 : 0.0) : exp((v - top) * per_t);
  }
  __device__ __forceinline__ unsigned long long fixed(double w) const { return (unsigned long long)__double2ll_rn(ldexp(w, a.scale_bits)); }

  __device__ unsigned long long block_sum64(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned long long all = 0;
#pragma unroll
    for (int w = 0; w < SF_THREADS / 32; ++w) all += s.warp[w];
    return all;
  }
  // Every block's number to every block; *before: the sum over the blocks with a lower rank.
  __device__ unsigned long long exchange_sum(unsigned long long v, unsigned long long* before) {
    const int t = turn++ & 1;
    if (threadIdx.x < blocks) sf_store(&s.part[t][rank], threadIdx.x, v);
    sf_sync();
    unsigned long long all = 0, low = 0;
    for (unsigned r = 0; r < blocks; ++r) {
      if (r < rank) low += s.part[t][r];
      all += s.part[t][r];
    }
    *before = low;
    return all;
  }
  __device__ unsigned exchange_max(unsigned v) {
    const int t = turn++ & 1;
    if (threadIdx.x < blocks) sf_store(&s.part[t][rank], threadIdx.x, v);
    sf_sync();
    unsigned m = 0;
    for (unsigned r = 0; r < blocks; ++r) m = max(m, (unsigned)s.part[t][r]);
    return m;
  }

  // The first key, from the largest on, where the running sum of the weights (ones, if ONES) exceeds thr; *above: the sum over larger keys.
  // thr is less than the sum over all keys.
  template <bool ONES>
  __device__ unsigned first_exceeding(unsigned long long thr, unsigned long long* above) {
    unsigned prefix = 0, mask = 0;
    unsigned long long over = 0;
    const int shifts[3] = {21, 10, 0};
#pragma unroll 1
    for (int level = 0; level < 3; ++level) {
      const int shift = shifts[level];
      const unsigned low_bits = level == 2 ? 0x3ffu : 0x7ffu;
      for (int b = threadIdx.x; b < SF_BINS; b += SF_THREADS) s.hist[b] = 0ull;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += SF_THREADS) {
        const unsigned k = key(i);
        if (k != 0u && (k & mask) == prefix) {
          const unsigned long long w = ONES ? 1ull : fixed(weight(k));
          if (w) atomicAdd(&s.hist[(k >> shift) & low_bits], w);
        }
      }
      sf_sync();
      // this block's share of the bins, higher ranks the higher bins; thread t the t-th of them
      const int share = SF_BINS / (int)blocks, b0 = (int)rank * share;
      constexpr int MOST = SF_BINS / SF_THREADS;  // bins of a thread when one block has them all
      const int each = (share + SF_THREADS - 1) / SF_THREADS;
      unsigned long long mine[MOST], sum = 0;
#pragma unroll
      for (int e = 0; e < MOST; ++e) {
        mine[e] = 0;
        const int b = (int)threadIdx.x * each + e;
        if (e < each && b < share)
          for (unsigned r = 0; r < blocks; ++r) mine[e] += sf_load(&s.hist[b0 + b], r);
        sum += mine[e];
      }
      // sums behind this thread within the block
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
      unsigned long long behind = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_down_sync(0xffffffffu, behind, o);
        if (lane + o < 32) behind += t;
      }
      __syncthreads();
      if (lane == 0) s.warp[warp] = behind;
      __syncthreads();
      unsigned long long total = 0;
      behind -= sum;
      for (int w = 0; w < SF_THREADS / 32; ++w) {
        if (w > warp) behind += s.warp[w];
        total += s.warp[w];
      }
      unsigned long long before;
      const unsigned long long all = exchange_sum(total, &before);
      unsigned long long run = over + (all - before - total) + behind;
#pragma unroll
      for (int e = MOST - 1; e >= 0; --e) {
        if (e < each && run <= thr && run + mine[e] > thr) {  // one thread of the cluster
          const unsigned long long bin = (unsigned long long)(b0 + (int)threadIdx.x * each + e);
          for (unsigned r = 0; r < blocks; ++r) {
            sf_store(&s.found[0], r, bin);
            sf_store(&s.found[1], r, run);
          }
        }
        if (e < each) run += mine[e];
      }
      sf_sync();
      prefix |= (unsigned)s.found[0] << shift;
      mask |= low_bits << shift;
      over = s.found[1];
    }
    *above = over;
    return prefix;
  }

  // The index of the j-th (from 0) of the row's numbers with key k, in the block that has it; -1 elsewhere.
  __device__ int nth(unsigned k, unsigned long long j) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = SF_THREADS / 32;
    const int run = (((n + nw - 1) / nw) + 31) & ~31, lo = min(n, warp * run), hi = min(n, lo + run);
    unsigned mine = 0;
    for (int i = lo; i < hi; i += 32) mine += __popc(__ballot_sync(0xffffffffu, i + lane < hi && key(i + lane) == k));
    __syncthreads();
    if (lane == 0) s.warp[warp] = mine;
    __syncthreads();
    unsigned long long total = 0, at = 0;
    for (int w = 0; w < nw; ++w) {
      if (w < warp) at += s.warp[w];
      total += s.warp[w];
    }
    unsigned long long before;
    exchange_sum(total, &before);
    at += before;
    if (j < at || j >= at + mine) return -1;
    int got = -1;
    for (int i = lo; i < hi; i += 32) {
      const bool is = i + lane < hi && key(i + lane) == k;
      const unsigned all = __ballot_sync(0xffffffffu, is);
      if (is && at + __popc(all & ((1u << lane) - 1)) == j) got = i + lane;
      at += __popc(all);
    }
    return got;
  }
};

template <typename T, bool RESIDENT>
__global__ void __launch_bounds__(SF_THREADS) sample_filtered_kernel(SfArgs a) {
  pdl_launch_dependents();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  SfShared& s = *reinterpret_cast<SfShared*>(smem_raw);
  unsigned* keys = reinterpret_cast<unsigned*>(smem_raw + sizeof(SfShared));
  const unsigned rank = sf_rank(), blocks = sf_size();
  const int r = blockIdx.x / blocks;
  const int first = min(a.vocab, (int)rank * a.per);
  SfRow<T, RESIDENT> row{a, s, keys, (const T*)a.logits + (size_t)r * a.ld + first, min(a.vocab, first + a.per) - first, rank, blocks};
  pdl_wait();
  const float temperature = a.temperatures ? a.temperatures[r] : a.temperature;
  const float top_p = a.top_ps ? a.top_ps[r] : a.top_p, asked = a.min_ps ? a.min_ps[r] : a.min_p;
  const float min_p = asked > 0.f ? fminf(asked, 1.f) : 0.f;  // the most probable token always stays
  const int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
  unsigned high = 0;
  unsigned long long valid = 0;
  for (int i = threadIdx.x; i < row.n; i += SF_THREADS) {
    const unsigned k = sf_key(to_f32<T>(row.row[i]));
    if (RESIDENT) keys[i] = k;
    high = max(high, k);
    valid += k != 0u;
  }
  sf_sync();  // every block of the cluster runs: its shared memory may be written
  // the random number, drawn once for the whole cluster
  if (rank == 0 && threadIdx.x == 0) {
    float u;
    if (a.u) {
      u = a.u[r];
    } else {  // xorshift64*, as in sampling.cu
      unsigned long long* state = a.rng + (a.index ? a.index[r] : r);
      unsigned long long x = *state;
      x ^= x >> 12; x ^= x << 25; x ^= x >> 27;
      *state = x;
      u = (float)((unsigned)((x * 0x2545F4914F6CDD1DULL) >> 32) >> 8) / 16777216.0f;
    }
    for (unsigned b = 0; b < blocks; ++b) sf_store(&s.found[0], b, __float_as_uint(u));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) high = max(high, __shfl_xor_sync(0xffffffffu, high, o));
  if ((threadIdx.x & 31) == 0) s.warp[threadIdx.x >> 5] = high;
  __syncthreads();
  for (int w = 0; w < SF_THREADS / 32; ++w) high = max(high, (unsigned)s.warp[w]);
  high = row.exchange_max(high);
  const float u = __uint_as_float((unsigned)s.found[0]);
  unsigned chosen = high;
  unsigned long long tie = 0;
  if (high != 0u && temperature > 0.f) {
    unsigned long long before;
    valid = row.exchange_sum(row.block_sum64(valid), &before);
    row.top = (double)sf_value(high);
    row.infinite = row.top == INFINITY;
    row.per_t = 1.0 / (double)temperature;
    // kept: all larger than `cut`, and `ties` of those equal to it
    unsigned cut = 1u;
    unsigned long long ties = 0;
    if (top_k > 0 && (unsigned long long)top_k < valid) {
      unsigned long long above;
      cut = row.template first_exceeding<true>((unsigned long long)top_k - 1, &above);
      ties = (unsigned long long)top_k - above;
    }
    auto kept_mass = [&](float least) {
      unsigned long long m = 0;
      for (int i = threadIdx.x; i < row.n; i += SF_THREADS) {
        const unsigned k = row.key(i);
        if (k > cut) {
          const double w = row.weight(k);
          if (w >= (double)least) m += row.fixed(w);
        }
      }
      m = row.block_sum64(m);
      unsigned long long low, all = row.exchange_sum(m, &low);
      if (ties) {
        const double w = row.weight(cut);
        if (w >= (double)least) all += ties * row.fixed(w);
      }
      return all;
    };
    if (top_p > 0.f && top_p < 1.f) {
      const unsigned long long all = kept_mass(0.f);
      const unsigned long long thr = min((unsigned long long)((double)top_p * (double)all), all - 1);
      unsigned long long above;
      const unsigned k = row.template first_exceeding<false>(thr, &above);
      const unsigned long long w = row.fixed(row.weight(k)), j = (thr - above) / w + 1;
      ties = k == cut ? min(ties, j) : j;
      cut = k;
    }
    const unsigned long long all = kept_mass(min_p);
    const float share = u > 0.f ? u : 0.f;
    const unsigned long long thr = min((unsigned long long)((double)share * (double)all), all - 1);
    unsigned long long above;
    chosen = row.template first_exceeding<false>(thr, &above);
    tie = (thr - above) / row.fixed(row.weight(chosen));
  }
  if (high == 0u) {
    if (rank == 0 && threadIdx.x == 0) a.out[r] = -1;
  } else {
    const int at = row.nth(chosen, tie);
    if (at >= 0) a.out[r] = first + at;
  }
  sf_sync();  // no block leaves while another may still read from it or write to it
}

template <typename T, bool RESIDENT>
static int sf_launch(const SfArgs& a, int n_rows, int blocks, size_t smem, cudaStream_t stream) {
  static BnGrant grant;
  const cudaError_t g = grant.ask((const void*)sample_filtered_kernel<T, RESIDENT>, smem, 0);
  if (g != cudaSuccess) return BN_ERR_LAUNCH + (int)g;
  const cudaError_t e = bn_launch_cluster(sample_filtered_kernel<T, RESIDENT>, dim3((unsigned)(n_rows * blocks)), dim3(SF_THREADS), smem, stream,
                                          dim3((unsigned)blocks, 1, 1), a);
  return e == cudaSuccess ? BN_OK : BN_ERR_LAUNCH + (int)e;
}

#define SF_KEYS_MAX 51200  // keys that a block holds beside its histogram

// logits [n_rows, vocab] of `dtype`, rows ld numbers apart.  The four parameters hold for all rows where their array is null.  u: a number in
// [0, 1) per row, or null: drawn from the generator rng[index ? index[r] : r], which is advanced.  out: the tokens, -1 for a row
// without a number above -inf.
extern "C" int bn_sample_filtered(const void* logits, int dtype, long long ld, int n_rows, int vocab, float temperature, const float* temperatures,
                                  int top_k, const int* top_ks, float top_p, const float* top_ps, float min_p, const float* min_ps, const float* u,
                                  unsigned long long* rng, const int* index, int* out, cudaStream_t stream) {
  if (n_rows <= 0) return BN_OK;
  if (!logits || !out || vocab <= 0 || ld < vocab || (!u && !rng) || (dtype != BN_F32 && dtype != BN_BF16) || n_rows > 0x7fffffff / SF_MAX_CLUSTER)
    return BN_ERR_BAD_ARG;
  SfArgs a = {};
  a.logits = logits; a.ld = ld; a.vocab = vocab;
  a.temperature = temperature; a.top_p = top_p; a.min_p = min_p; a.top_k = top_k;
  a.temperatures = temperatures; a.top_ks = top_ks; a.top_ps = top_ps; a.min_ps = min_ps;
  a.u = u; a.rng = rng; a.index = index; a.out = out;
  int bits = 0;
  while ((1ll << bits) < vocab) ++bits;
  a.scale_bits = 62 - bits;  // the sum of all weights stays below 2^62
  int blocks = SF_MAX_CLUSTER;
  while (blocks > 1 && vocab <= (blocks / 2) * 2048) blocks /= 2;
  a.per = (((vocab + blocks - 1) / blocks) + 7) & ~7;
  const bool resident = a.per <= SF_KEYS_MAX;
  const size_t smem = sizeof(SfShared) + (resident ? (size_t)a.per * 4 : 0);
  if (dtype == BN_F32) return resident ? sf_launch<float, true>(a, n_rows, blocks, smem, stream) : sf_launch<float, false>(a, n_rows, blocks, smem, stream);
  return resident ? sf_launch<__nv_bfloat16, true>(a, n_rows, blocks, smem, stream) : sf_launch<__nv_bfloat16, false>(a, n_rows, blocks, smem, stream);
}
