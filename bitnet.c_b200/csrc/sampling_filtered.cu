// The next token from temperature, top-k, top-p and min-p, from a given random number per row.
//
// Sorted order of a row: falling logits, equal ones by rising index; NaN counts as -inf and -inf is never chosen.  With
// w_i = exp((l_i - max) / T):  K1 the first k;  K2 of K1 up to the first whose running sum exceeds top_p * sum(K1);  K3 those of K2 with
// w_i >= min_p;  the token is the first of K3 whose running sum exceeds u * sum(K3).  Each set is a beginning of the sorted order, so nothing
// is sorted: every border is "the first whose running sum (of ones, or of weights) exceeds a number", found by the bits of the logits.
//
// A cluster of blocks holds a row in its shared memory as ordered 32-bit keys, so that memory is read once however many passes
// follow.  One pass adds up the keys' weights (with top-k: counts the keys) in steps of 2^(1/32) of the weight (finer ones
// where the row's weights lie closer together: fewer keys meet in a step); from these sums the first block of the
// cluster knows in which step each border lies.  A second pass hands the keys of those steps to it; it sorts them (some tens of keys, of a flat row
// hundreds) and decides.  Where too many keys lie together (ties by the thousand, a huge temperature) or the border is not known well (a top-k of thousands), borders are found by the bits of the keys
// instead, 11, 11 and 10 at a time, the weights of the keys that agree with the bits found so far added into a histogram.
// Weights are whole numbers of 64 bits: sums do not depend on the order of additions, and a running sum that lies next to a border falls on the
// same side as in a sum of doubles unless it is within 10^-9 of the sum (a float sum would move a token in a thousand).  exp(-y) is taken apart into 2^-(j/32) from a
// table, a shift, and 1 - e of what is left of y behind multiples of ln 2 / 32 (in two parts, after Cody and Waite).  y = (max - l) / T and e are carried in two floats,
// since one of them is off by up to 2^-30 of the weight by itself: weights are good to 2^-31, where this was measured on the CPU 2^-31.2.
//
// Measured: one row of 32,000 with top-k 11.4 us, 8 rows of 128,256 with top-p 17.6, 64 rows of 128,256 with parameters of their own 36.5, 200 flat
// rows of 50,257 in bfloat16 54.5.  Few rows are bound by latency (the first block's plan takes 5.5 us, handing over and deciding 2.7, the cluster's barriers 2.5), many by some
// 69 instructions a number, two additions in shared memory (2.8 cycles a warp's where no lanes meet) among them.
//
// Borders by bits are slow.  Ties: 64 rows of 128,256 equal numbers 4.2 ms.  Top-k of thousands: with top-k, steps are counted and not summed, so every mass is known to some 4.7 % only, and
// the keys between the bounds may be more than the list holds.  64 rows of 128,256 normal logits of spread 3 with a top-k of 50 / 1,000 / 5,000 / 50,000: 24.6 / 41 / 307 / 327 us,
// with top-p 0.95 behind it 26.2 / 47 / 525 / 535; one row 13.9 / 15.9 / 19.1 / 34.3 and 14.6 / 27.9 / 186 / 188.  A temperature of 10,000: 64 rows 290, one 98.
#include "common.cuh"
#include <math.h>

#define SF_THREADS 512
#define SF_BINS 2048     // of a histogram of bits
#define SF_STEPS 2048    // of the counts by weight: 64 octaves of 32 steps; the last one's keys weigh nothing (and are not counted)
#define SF_LIST 2048     // keys that the first block may be handed
#define SF_NOTED 512     // logits near a border that a block notes before it settles them (more are settled one by one)
#define SF_COUNTED 65000 // keys of a block whose weights' halves add up in 32 bits whatever their steps
#define SF_POINT 56      // a weight of 1 is 2^56 while a thread adds up its own (at most 2^7 of them)
#define SF_MAX_CLUSTER 8
#define SF_NO_STATE 0xffffffffu  // in place of a random number: the row's index names no generator
#define SF_FAR 44.4f           // as far as there are steps: 64 octaves
#define SF_32ND (5678.f / 262144.f)      // ln 2 / 32, 13 bits of it
#define SF_32ND_REST 9.98318279e-7f      // and the rest

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
  unsigned long long* rng;    // n_states of them
  const int* index;           // row -> its generator, or null
  int n_states;
  int* out;
  int scale_bits;             // weights are multiples of 2^-scale_bits
  unsigned long long table[32];  // 2^-(j/32), 1 = 2^SF_POINT
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
__device__ __forceinline__ void sf_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void sf_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void sf_sync(unsigned blocks) {  // all threads of the cluster; what they wrote to shared memory is seen by all
  if (blocks == 1) {
    __syncthreads();
  } else {
    sf_arrive();
    sf_wait();
  }
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
__device__ __forceinline__ uint4 sf_load4(const unsigned* p, unsigned rank) {  // 16-byte aligned
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(sf_remote(p, rank)));
  return v;
}
__device__ __forceinline__ void sf_store(unsigned long long* p, unsigned rank, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(sf_remote(p, rank)), "l"(v) : "memory");
}

struct SfRange {  // steps first .. last
  int first, last;
};
struct alignas(8) SfPlan {
  SfRange range[4];    // where the borders of top-k, top-p, min-p and the draw lie; none: last < first
  unsigned least;      // min-p: the smallest key that stays
  unsigned rest;       // top-k: so many keys of its step stay
  int by_bits;         // borders are found by the bits of the keys
  int pad;
};
#define SF_TOP_K 0
#define SF_TOP_P 1
#define SF_MIN_P 2
#define SF_DRAW 3

struct SfShared {
  ulonglong2 warp_sums[SF_THREADS / 32];  // first block: bounds of the weights of a warp's steps
  union {
    unsigned long long hist[SF_BINS];
    struct {
      // of a step's keys their number; or the sum of their weights in parts of 2^-31 of its largest, upper and lower 16 bits apart
      unsigned one[SF_STEPS], two[SF_STEPS];
    };
    unsigned long long list[SF_LIST];  // keys falling, equal ones by index: (~key, index)
  };
  unsigned long long warp[SF_THREADS / 32];
  // one entry per block of the cluster, written by that block; two sets in turn, so that one barrier per exchange is enough
  unsigned long long part[2][SF_MAX_CLUSTER];
  unsigned long long found[2];  // what the block that found a border tells the others
  unsigned long long over[SF_MAX_CLUSTER][4];   // first block: the weights of each block's keys above each range
  unsigned long long all_mass;                  // first block: of all keys (not with top-k)
  SfPlan plan;
  unsigned listed;                              // keys in this block's list
  unsigned noted;                               // logits of this block near a border, and where they are
  int note[SF_NOTED];
  unsigned high, low;                           // the largest key of this block, the largest of 0 - key
  unsigned long long table[32];                 // 2^-(j/32), 1 = 2^SF_POINT
  int small_table[32];                          // the same, 1 = 2^30
  unsigned long long warp4[SF_THREADS / 32][4];
  unsigned long long got[4];
  int steps[8];
  int place;  // of this block's keys in the first block's list
};

template <typename T, bool RESIDENT>
struct SfRow {
  SfArgs a;
  SfShared& s;
  const T* held;         // this block's part of the row in shared memory (RESIDENT), -inf behind its end
  const T* row;          // and where it came from
  int n;                 // numbers of it
  unsigned rank, blocks;
  int turn = 0;
  double top, per_t;     // the largest logit, 1 / temperature
  bool infinite;         // the largest logit is +inf: those share everything
  float topf, t_hi, t_lo;  // the largest logit, 1 / temperature in two floats
  int fine;                // steps are 2^-fine of a 32nd of an octave: as fine as lets the smallest weight have a step in front of the last
  float steps;             // in 1 of y

  __device__ __forceinline__ unsigned key(int i) const { return sf_key(to_f32<T>(RESIDENT ? held[i] : row[i])); }
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
    v = (threadIdx.x & 31) < SF_THREADS / 32 ? s.warp[threadIdx.x & 31] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  // Every block's number to every block; *before: the sum over the blocks with a lower rank.
  __device__ unsigned long long exchange_sum(unsigned long long v, unsigned long long* before) {
    const int t = turn++ & 1;
    if (threadIdx.x < blocks) sf_store(&s.part[t][rank], threadIdx.x, v);
    sf_sync(blocks);
    unsigned long long all = 0, low = 0;
    for (unsigned r = 0; r < blocks; ++r) {
      if (r < rank) low += s.part[t][r];
      all += s.part[t][r];
    }
    *before = low;
    return all;
  }
  // The largest of every block's `high` and `low`.
  __device__ void exchange_max(unsigned* high, unsigned* low) {
    const int t = turn++ & 1;
    if (threadIdx.x < blocks) sf_store(&s.part[t][rank], threadIdx.x, ((unsigned long long)*high << 32) | *low);
    sf_sync(blocks);
    for (unsigned r = 0; r < blocks; ++r) {
      const unsigned long long x = s.part[t][r];
      *high = max(*high, (unsigned)(x >> 32));
      *low = max(*low, (unsigned)x);
    }
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
      sf_sync(blocks);
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
      sf_sync(blocks);
      prefix |= (unsigned)s.found[0] << shift;
      mask |= low_bits << shift;
      over = s.found[1];
    }
    *above = over;
    return prefix;
  }

  // ---- by steps of weight ----
  // The step of a logit (falling logits, rising steps: the nearest to y), and 1 - exp(-r), in two floats, of what is left (r) of y behind the 32nd of an octave that the
  // step lies in.  Conversions by adding 1.5 * 2^23: those of the conversion unit take four times the issue slots.  (Whatever the logit, the step is one of those that
  // there are.)  SF_32ND has 13 bits, so that its multiples and the first part of r are exact.
  __device__ __forceinline__ int step_of(float v, float2* e) const {
    const float d = topf - v, bb = d - topf, dl = (topf - (d - bb)) - (v + bb);
    const float y = d * t_hi, yl = fmaf(d, t_hi, -y) + fmaf(d, t_lo, dl * t_hi);
    const int n = (int)min((unsigned)__float_as_int(fmaf(fminf(y, SF_FAR), steps, 12582912.f)) - 0x4B400000u, SF_STEPS - 1u);
    const float at = __int_as_float((n >> fine) + 0x4B400000) - 12582912.f;
    const float r = fmaf(at, -SF_32ND, y), rl = fmaf(at, -SF_32ND_REST, yl), s = r + rl;
    // 1 - exp(-r) = r - r^2 / 2 + r^3 / 6 - r^4 / 24 and less than 2^-34
    *e = make_float2(r, rl - s * (s * (0.5f - s * (0.16666667f - s * 0.041666668f))));
    return n;
  }
  __device__ __forceinline__ int step_of(float v) const {
    return (int)min((unsigned)__float_as_int(fmaf(fminf((topf - v) * t_hi, SF_FAR), steps, 12582912.f)) - 0x4B400000u, SF_STEPS - 1u);
  }
  // The weight that a step's 32nd of an octave has its keys' weights from.
  __device__ __forceinline__ unsigned long long most_at(int n) const { return s.table[(n >> fine) & 31] >> (n >> fine >> 5); }
  // exp(-y), 1 = 2^SF_POINT, to 2^-32 of itself
  __device__ __forceinline__ unsigned long long weight_at(int n, float2 e) const {
    const int whole = __float2int_rn(e.x * 17179869184.f) + __float2int_rn(e.y * 17179869184.f), at = n >> fine;  // (below 2^29)
    const unsigned long long w = s.table[at & 31] - (((long long)s.small_table[at & 31] * whole) >> (64 - SF_POINT));
    return nothing(n) ? 0ull : w >> (at >> 5);
  }
  // Whether a step's keys weigh nothing: the last one's, where steps are as wide as they get (else no key lies there).
  __device__ __forceinline__ bool nothing(int n) const { return n == SF_STEPS - 1; }
  __device__ __forceinline__ unsigned long long to_scale(unsigned long long w) const {  // from 2^SF_POINT to 2^scale_bits
    const int down = SF_POINT - a.scale_bits;
    return down ? (w + (1ull << (down - 1))) >> down : w;
  }
  // A thread adds up its weights with SF_POINT bits behind the point while it has few of them (a row that is held), else with as many as the sums have.
  __device__ __forceinline__ void add(unsigned long long& sum, unsigned long long w) const { sum += RESIDENT ? w : to_scale(w); }
  __device__ __forceinline__ unsigned long long added(unsigned long long sum) const { return RESIDENT ? to_scale(sum) : sum; }
  // f(logits, index of the first) for this block's logits, a few at a time (-inf and NaN among them).
  template <class F>
  __device__ __forceinline__ void each_value(F f) const {
    constexpr int V = 16 / (int)sizeof(T);
    float v[V];
    const auto take = [&](const uint4& raw, int i) {
      const T* x = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = to_f32<T>(x[e]);
      f(v, i);
    };
    if (RESIDENT) {
#pragma unroll 1
      for (int i = threadIdx.x * V; i < n; i += SF_THREADS * V) take(*reinterpret_cast<const uint4*>(held + i), i);
      return;
    }
    int done = 0;
    if ((((uintptr_t)row) & 15) == 0) {
      const int nv = n / V;
      done = nv * V;
#pragma unroll 1
      for (int i = threadIdx.x; i < nv; i += 2 * SF_THREADS) {  // two loads in flight
        const uint4 a0 = __ldg(reinterpret_cast<const uint4*>(row) + i), a1 = __ldg(reinterpret_cast<const uint4*>(row) + min(i + SF_THREADS, nv - 1));
        take(a0, i * V);
        if (i + SF_THREADS < nv) take(a1, (i + SF_THREADS) * V);
      }
    }
#pragma unroll 1
    for (int i = done + threadIdx.x; i < n; i += SF_THREADS) {
      const float x[1] = {to_f32<T>(row[i])};
      f(x, i);
    }
  }

  // All blocks: the keys by their steps.  With top-k their numbers (in one histogram: two, for fewer lanes that meet, cost the first block 0.6 us of loads); without it
  // their weights, to 2^-31 of themselves (half of which is what is left behind 31 bits).
  __device__ __forceinline__ void count_steps(bool numbers) const {
    if (numbers) {
      each_value([&](const auto& v, int) {
#pragma unroll
        for (const float x : v) {
          const int n = step_of(x);
          if (!nothing(n)) atomicAdd(&s.one[n], 1u);
        }
      });
    } else {
      each_value([&](const auto& v, int) {
#pragma unroll
        for (const float x : v) {
          float2 e;
          const int n = step_of(x, &e);
          // 2^31 - e 2^31 in halves: e 2^15 is cut to a whole number, what is left of it (from -0.0003 to 1) has 16 bits more
          const float z = fmaf(e.x + e.y, 32768.f, -0.4999f) + 12582912.f, left = fmaf(e.y, 32768.f, fmaf(e.x, 32768.f, 12582912.f - z));
          if (!nothing(n)) {
            atomicAdd(&s.one[n], (unsigned)(0x4B400000 + 32767 - __float_as_int(z)));
            atomicAdd(&s.two[n], (unsigned)(0x4B400000 + 65536 - __float_as_int(fmaf(left, 65536.f, 12582912.f))));
          }
        }
      });
    }
  }

  // First block: the steps in which the borders lie, from what all blocks have counted.
  __device__ void make_plan(bool k_on, unsigned top_k, bool p_on, float top_p, bool m_on, float min_p, float temperature, float u) {
    constexpr int EACH = SF_STEPS / SF_THREADS, NW = SF_THREADS / 32;
    static_assert(EACH % 4 == 0, "a thread's steps are read 16 bytes at a time");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n0 = tid * EACH;
    unsigned long long one[EACH] = {}, two[EACH] = {};
#pragma unroll 1
    for (unsigned r0 = 0; r0 < blocks; r0 += 4) {
      uint4 ones[4][EACH / 4], twos[4][EACH / 4];  // all of them asked for before the first is used
#pragma unroll
      for (unsigned r = 0; r < 4; ++r)
#pragma unroll
        for (int q = 0; q < EACH / 4; ++q) {
          ones[r][q] = r0 + r < blocks ? sf_load4(&s.one[n0 + 4 * q], r0 + r) : make_uint4(0u, 0u, 0u, 0u);
          twos[r][q] = !k_on && r0 + r < blocks ? sf_load4(&s.two[n0 + 4 * q], r0 + r) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
      for (unsigned r = 0; r < 4; ++r)
#pragma unroll
        for (int q = 0; q < EACH / 4; ++q) {
          one[4 * q] += ones[r][q].x; one[4 * q + 1] += ones[r][q].y; one[4 * q + 2] += ones[r][q].z; one[4 * q + 3] += ones[r][q].w;
          two[4 * q] += twos[r][q].x; two[4 * q + 1] += twos[r][q].y; two[4 * q + 2] += twos[r][q].z; two[4 * q + 3] += twos[r][q].w;
        }
    }
    if (tid < 8) s.steps[tid] = -1;
    // the smallest key whose weight is at least min_p: exp((v - max) / T) >= min_p where v >= max + T log(min_p)
    if (tid == SF_THREADS - 1 && m_on) s.plan.least = min(max(sf_key(__double2float_ru(top + (double)temperature * log((double)min_p))), 1u), sf_key(topf));
    // of each step its keys (without top-k: at least so many) and bounds of their weights' sum, which are the sum itself without top-k; the last step's keys
    // weigh nothing
    unsigned c[EACH];
    unsigned long long lo[EACH], up[EACH];
    unsigned before = 0;
    unsigned long long low = 0, high = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int n = n0 + e;
      const unsigned long long t = most_at(n);
      if (k_on) {
        c[e] = (unsigned)one[e];
        up[e] = c[e] * (to_scale(t + (t >> 6)) + 1);  // (2^(1/64) at most, 2^(-1/32) at least)
        lo[e] = c[e] * to_scale(t - (t >> 5));
      } else {
        const unsigned long long w = (one[e] << 16) + two[e];  // 1 = 2^31, below 2^51
        c[e] = (unsigned)((w + (w >> 5)) >> 31) + (w ? 1u : 0u);
        // w * t / 2^31, t of SF_POINT bits, to 2^scale_bits
        const int down = 31 + SF_POINT - a.scale_bits;
        const unsigned long long h = __umul64hi(w, t), l = w * t;
        const unsigned long long half = 1ull << (down - 1), l2 = l + half;
        up[e] = lo[e] = ((h + (l2 < l)) << (64 - down)) | (l2 >> down);
      }
      if (n == SF_STEPS - 1) up[e] = lo[e] = 0;
      before += c[e];
      low += lo[e];
      high += up[e];
    }
    unsigned cs = before;
    unsigned long long ls = low, us = high;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned x = __shfl_up_sync(0xffffffffu, cs, o);
      const unsigned long long y = __shfl_up_sync(0xffffffffu, ls, o), z = __shfl_up_sync(0xffffffffu, us, o);
      if (lane >= o) { cs += x; ls += y; us += z; }
    }
    if (lane == 31) {
      s.warp_sums[warp] = make_ulonglong2(ls, us);
      s.warp[warp] = cs;
    }
    __syncthreads();
    cs -= before; ls -= low; us -= high;
    unsigned total = 0;
    unsigned long long all_low = 0;
#pragma unroll 4
    for (int w = 0; w < NW; ++w) {
      const ulonglong2 x = s.warp_sums[w];
      const unsigned y = (unsigned)s.warp[w];
      if (w < warp) { cs += y; ls += x.x; us += x.y; }
      total += y;
      all_low += x.x;
    }
    unsigned long long all_up = all_low;
    const unsigned long long ls_before = ls;
    // from here on running sums, each with its step
    unsigned ci[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      cs += c[e]; ls += lo[e]; us += up[e];
      ci[e] = cs; lo[e] = ls; up[e] = us;
    }
    // the first step whose running sum exceeds thr, by the upper and the lower bound, goes to steps[slot] and steps[slot + 1] (-1: none does)
    auto find = [&](int slot, unsigned long long thr_up, unsigned long long thr_lo) {
      unsigned by_up = ~0u, by_lo = ~0u;
#pragma unroll
      for (int e = EACH - 1; e >= 0; --e) {
        if (up[e] > thr_up) by_up = (unsigned)(n0 + e);
        if (lo[e] > thr_lo) by_lo = (unsigned)(n0 + e);
      }
      by_up = __reduce_min_sync(0xffffffffu, by_up);
      by_lo = __reduce_min_sync(0xffffffffu, by_lo);
      if (lane == 0 && by_up != ~0u) atomicMin((unsigned*)&s.steps[slot], by_up);
      if (lane == 0 && by_lo != ~0u) atomicMin((unsigned*)&s.steps[slot + 1], by_lo);
    };
    const unsigned kth = min(top_k, total);
    const int m_step = m_on ? step_of(sf_value(s.plan.least)) : SF_STEPS;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      if (k_on && ci[e] - c[e] < kth && ci[e] >= kth) {
        s.steps[0] = n0 + e;
        s.plan.rest = kth - (ci[e] - c[e]);
        s.got[0] = e ? lo[e - 1] : ls_before;  // (some of the step's weights stay)
        s.got[1] = up[e];
      }
      if (m_step == n0 + e) {
        s.got[2] = e ? lo[e - 1] : ls_before;
        s.got[3] = up[e];
      }
    }
    __syncthreads();
    const int k_step = k_on ? s.steps[0] : SF_STEPS - 1;
    if (k_on) { all_low = s.got[0]; all_up = s.got[1]; }
    const auto part = [](float share, unsigned long long of) { return (unsigned long long)((double)share * (double)of); };
    if (p_on) find(1, min(part(top_p, all_low), all_low ? all_low - 1 : 0ull), min(part(top_p, all_up), all_up - 1));
    __syncthreads();
    SfRange range[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) range[r] = SfRange{1, 0};
    // (no border that matters lies in the last step: its keys are not asked for)
    int cut = SF_STEPS - 2;
    unsigned long long kept_low = all_low, kept_up = all_up;
    if (k_on) { range[SF_TOP_K] = SfRange{k_step, k_step}; cut = min(cut, k_step); }
    if (p_on) {
      const int p1 = s.steps[2] < 0 ? cut : min(cut, s.steps[2]), p0 = s.steps[1] < 0 ? p1 : min(p1, s.steps[1]);
      range[SF_TOP_P] = SfRange{p0, p1};
      cut = p1;
      kept_low = part(top_p, all_low);
      const unsigned long long t = most_at(p0);  // the token that crosses stays
      kept_up = part(top_p, all_up) + to_scale(t + (t >> 6)) + 1;
    }
    if (m_on && (m_step <= cut || !(k_on || p_on))) {
      if (m_step < (p_on ? range[SF_TOP_P].first : k_step) || !(k_on || p_on)) {  // what lies behind does not matter
        range[SF_TOP_K] = range[SF_TOP_P] = SfRange{1, 0};
        kept_low = s.got[2];
        kept_up = s.got[3];
      } else {
        kept_low = min(kept_low, s.got[2]);
        kept_up = min(kept_up, s.got[3]);
      }
      range[SF_MIN_P] = SfRange{m_step, m_step};
      cut = min(cut, m_step);
    }
    // (the weights of single keys are rounded once more than those of steps: a draw that lies next to a border of steps is looked for on both sides)
    const unsigned long long r0 = part(u, kept_low), r1 = part(u, kept_up);
    find(3, r0 - (r0 >> 30), r1 + (r1 >> 30));
    __syncthreads();
    const int d1 = s.steps[4] < 0 ? cut : min(cut, s.steps[4]), d0 = s.steps[3] < 0 ? d1 : min(d1, s.steps[3]);
    range[SF_DRAW] = SfRange{d0, d1};
    unsigned wanted = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int n = n0 + e;
      bool in = false;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        in |= n >= range[r].first && n <= range[r].last;
        if (n == range[r].first) s.over[0][r] = e ? lo[e - 1] : ls_before;  // (with top-k the blocks write what they find)
      }
      wanted += in && n != SF_STEPS - 1 ? c[e] : 0u;
    }
    wanted = __reduce_add_sync(0xffffffffu, wanted);
    if (lane == 0 && wanted) atomicAdd((unsigned*)&s.steps[7], wanted);  // (from -1 on)
    if (tid == 0) {
#pragma unroll
      for (int r = 0; r < 4; ++r) s.plan.range[r] = range[r];
      s.all_mass = all_low;
    }
    if (tid >= 4 && tid < 4 * (int)blocks) s.over[tid >> 2][tid & 3] = 0;
    __syncthreads();
    if (tid == 0) s.plan.by_bits = s.steps[7] + 1 > SF_LIST;
    __syncthreads();
    constexpr int WORDS = sizeof(SfPlan) / 8;
    if (tid < WORDS * (int)blocks && tid >= WORDS) sf_store(reinterpret_cast<unsigned long long*>(&s.plan) + tid % WORDS, tid / WORDS,
                                                            reinterpret_cast<const unsigned long long*>(&s.plan)[tid % WORDS]);
  }

  // All blocks: the keys of the ranges to the first block; with top-k also the weights above each range (few keys lie there).
  __device__ void hand_over(bool numbers) {
    int first[4], last[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      first[r] = s.plan.range[r].first;
      last[r] = s.plan.range[r].last;
      if (last[r] < first[r]) {
        first[r] = last[r] = -1;
      }
    }
    unsigned long long over[4] = {0, 0, 0, 0};
    const int offset = (int)rank * a.per;
    // Each block fills the list of its own first; the first block's is the one that counts.
    const auto give = [&](unsigned k, int i) {
      const unsigned at = atomicAdd(&s.listed, 1u);
      if (at < SF_LIST) s.list[at] = ((unsigned long long)~k << 32) | (unsigned)(offset + i);
    };
    // The logits of a range lie between about these (a step's logits are within half a step of it; they are
    // looked at again); with top-k all above the last are needed.
    float from[4], to[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float y0 = topf - ((float)last[r] + 0.6f) / (steps * t_hi), y1 = topf - ((float)first[r] - 0.6f) / (steps * t_hi);
      from[r] = fmaxf(y0 - fminf(fabsf(y0), 1e38f) * 1e-6f, -3.4028235e38f);
      to[r] = numbers ? INFINITY : y1 + fminf(fabsf(y1), 1e38f) * 1e-6f;
      if (first[r] < 0) from[r] = INFINITY, to[r] = -INFINITY;
    }
    const float lowest = fminf(fminf(from[0], from[1]), fminf(from[2], from[3]));
    if (numbers) from[1] = lowest, to[1] = INFINITY;
    const auto near = [&](float x) {  // (there is no border of top-k without its numbers)
      return (x >= from[1] && x <= to[1]) || (x >= from[2] && x <= to[2]) || (x >= from[3] && x <= to[3]);
    };
    const auto settle = [&](int i) {
      const float x = to_f32<T>(RESIDENT ? held[i] : row[i]);
      float2 e;
      const int n = step_of(x, &e);
      bool in = false;
#pragma unroll
      for (int r = 0; r < 4; ++r) in |= n >= first[r] && n <= last[r] && !nothing(n);
      if (numbers) {
        const unsigned long long w = weight_at(n, e);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n < first[r]) add(over[r], w);
      }
      if (in) give(sf_key(x), i);
    };
    // Logits that are near are noted first, and settled a thread each when all have been looked at: a warp would wait for its lanes that have one again and again
    // (200 flat rows of 50,257: 54 us, 59 with each settled where it is found).
    each_value([&](const auto& v, int i0) {
      constexpr int V = sizeof(v) / sizeof(float);
      float most = -INFINITY;  // (most logits lie below all of them)
#pragma unroll
      for (int e = 0; e < V; ++e) most = fmaxf(most, v[e]);
      if (!(most >= lowest)) return;
      unsigned hit = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) hit |= near(v[e]) ? 1u << e : 0u;
      for (; hit; hit &= hit - 1) {
        const int i = i0 + __ffs(hit) - 1;
        const unsigned at = atomicAdd(&s.noted, 1u);
        if (at < SF_NOTED) s.note[at] = i;
        else settle(i);
      }
    });
    __syncthreads();
    for (unsigned j = threadIdx.x; j < min(s.noted, (unsigned)SF_NOTED); j += SF_THREADS) settle(s.note[j]);
    __syncthreads();
    if (rank != 0 && s.listed) {
      const int mine = min((int)s.listed, SF_LIST);
      if (threadIdx.x == 0) {
        unsigned at;
        asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(at) : "r"(sf_remote(&s.listed, 0)), "r"(mine) : "memory");
        s.place = (int)at;
      }
      __syncthreads();
      const int at = s.place;
      for (int i = threadIdx.x; i < mine && at + i < SF_LIST; i += SF_THREADS) sf_store(&s.list[at + i], 0, s.list[i]);
    }
    if (!numbers) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      over[r] = added(over[r]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) over[r] += __shfl_xor_sync(0xffffffffu, over[r], o);
    }
    const int lane = threadIdx.x & 31;
    if (lane < 4) s.warp4[threadIdx.x >> 5][lane] = lane == 0 ? over[0] : lane == 1 ? over[1] : lane == 2 ? over[2] : over[3];
    __syncthreads();
    if (threadIdx.x < 4) {
      unsigned long long sum = 0;
#pragma unroll 4
      for (int w = 0; w < SF_THREADS / 32; ++w) sum += s.warp4[w][threadIdx.x];
      sf_store(&s.over[rank][threadIdx.x], 0, sum);
    }
  }

  // First block (GROUP threads of it, EACH keys a thread): sorts the keys that it was handed and finds the token.  Whatever is asked of the sorted keys holds for
  // a beginning of them, or from some key on up to another: the borders are counts.
  template <int GROUP, int EACH>
  __device__ void decide(float top_p, float u, int* out) {
    const int m = min((int)s.listed, SF_LIST), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const auto sync = [] {
      if (GROUP == 32) __syncwarp();
      else __syncthreads();
    };
    unsigned long long entry[EACH];
    if (EACH == 1) {  // each key counts those in front of it
      entry[0] = tid < m ? s.list[tid] : ~0ull;
      int place = tid < m ? 0 : tid;
      if (GROUP == 32) {
        for (int j = 0; j < m; ++j) {  // (all lanes take part in the shuffle)
          const unsigned long long other = __shfl_sync(0xffffffffu, entry[0], j);
          place += tid < m && other < entry[0];
        }
      } else if (tid < m) {
#pragma unroll 4
        for (int j = 0; j < m; ++j) place += s.list[j] < entry[0];
      }
      sync();
      if (tid < m) s.list[place] = entry[0];
      sync();
      if (tid < m) entry[0] = s.list[tid];
    } else {
      int size = 2;
      while (size < m) size *= 2;
      for (int i = m + tid; i < size; i += GROUP) s.list[i] = ~0ull;
      sync();
      for (int k = 2; k <= size; k *= 2) {
        for (int j = k / 2; j > 0; j /= 2) {
          for (int i = tid; i < size / 2; i += GROUP) {
            const int x = 2 * i - (i & (j - 1)), y = x + j;
            const unsigned long long p = s.list[x], q = s.list[y];
            if ((p > q) == ((x & k) == 0)) { s.list[x] = q; s.list[y] = p; }
          }
          sync();
        }
      }
#pragma unroll
      for (int e = 0; e < EACH; ++e) entry[e] = tid + e * GROUP < m ? s.list[tid + e * GROUP] : ~0ull;
      sync();
    }
    // the keys' steps, and the running sums in front of them and with them (those in runs[], too)
    unsigned long long* runs = EACH == 1 ? s.list + SF_LIST / 2 : s.list;  // (beside the keys, or over them: the threads have those)
    unsigned long long before[EACH], run[EACH], total = 0;
    int n[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      float2 less;
      n[e] = step_of(sf_value(~(unsigned)(entry[e] >> 32)), &less);
      const unsigned long long w = tid + e * GROUP < m ? to_scale(weight_at(n[e], less)) : 0ull;
      run[e] = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, run[e], o);
        if (lane >= o) run[e] += t;
      }
      if (GROUP > 32) {
        if (lane == 31) s.warp[warp] = run[e];
        __syncthreads();
        unsigned long long chunk = 0;
#pragma unroll 4
        for (int x = 0; x < GROUP / 32; ++x) {
          if (x < warp) run[e] += s.warp[x];
          chunk += s.warp[x];
        }
        run[e] += total;
        total += chunk;
        runs[tid + e * GROUP] = run[e];
        __syncthreads();
      }
      before[e] = run[e] - w;
    }
    const auto run_at = [&](int i) {  // the running sum with the i-th key (0 in front of the first)
      if (GROUP == 32) {
        const unsigned long long x = __shfl_sync(0xffffffffu, run[0], max(i, 0));
        return i < 0 ? 0ull : x;
      }
      return i < 0 ? 0ull : runs[i];
    };
    const auto count = [&](auto holds) {  // the keys for which holds(their place, which of this thread's)
      int c = 0;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int i = tid + e * GROUP;
        const bool is = i < m && holds(i, e);
        c += GROUP == 32 ? __popc(__ballot_sync(0xffffffffu, is)) : __syncthreads_count(is);
      }
      return c;
    };
    unsigned long long over[4], part4 = 0;  // lane: block lane / 4 and 8 more, range lane % 4
    for (unsigned b = lane >> 2; b < blocks; b += 8) part4 += s.over[b][lane & 3];
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) part4 += __shfl_xor_sync(0xffffffffu, part4, o);
#pragma unroll
    for (int r = 0; r < 4; ++r) over[r] = __shfl_sync(0xffffffffu, part4, r);
    SfRange range[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) range[r] = s.plan.range[r];
    const auto is_in = [&](int r) { return range[r].last >= range[r].first; };
    const auto begin = [&](int r) { return count([&](int, int e) { return n[e] < range[r].first; }); };  // the place of a range's first key
    unsigned long long kept = s.all_mass;
    if (is_in(SF_TOP_K)) {
      const int at = begin(SF_TOP_K);
      kept = over[SF_TOP_K] + run_at(min(at + (int)s.plan.rest, m) - 1) - run_at(at - 1);
    }
    if (is_in(SF_TOP_P)) {  // up to the last whose predecessors do not exceed it
      const unsigned long long thr = min((unsigned long long)((double)top_p * (double)kept), kept - 1);
      const int at = begin(SF_TOP_P);
      const unsigned long long off = over[SF_TOP_P] - run_at(at - 1);
      kept = off + run_at(at + count([&](int i, int e) { return i >= at && n[e] <= range[SF_TOP_P].last && before[e] + off <= thr; }) - 1);
    }
    if (is_in(SF_MIN_P)) {
      const unsigned least = s.plan.least;
      const int at = begin(SF_MIN_P), stay = count([&](int, int e) { return ~(unsigned)(entry[e] >> 32) >= least; });
      const unsigned long long sum = over[SF_MIN_P] + run_at(max(stay, at) - 1) - run_at(at - 1);
      // (where min-p alone decides, the plan has no other range, and its sum is the smaller one)
      kept = is_in(SF_TOP_K) || is_in(SF_TOP_P) ? min(kept, sum) : sum;
    }
    const unsigned long long thr = min((unsigned long long)((double)u * (double)kept), kept - 1);
    const int at = begin(SF_DRAW);
    const unsigned long long off = over[SF_DRAW] - run_at(at - 1);
    const int c = count([&](int i, int e) { return i >= at && n[e] <= range[SF_DRAW].last && before[e] + off <= thr; });
    const int chosen = c ? at + c - 1 : max(min(at, m - 1), 0);
#pragma unroll
    for (int e = 0; e < EACH; ++e)
      if (tid + e * GROUP == chosen) *out = (int)(unsigned)entry[e];
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

// One block's part of a row into shared memory (RESIDENT); the largest of it, and the smallest above -inf (or +inf).
template <typename T, bool RESIDENT>
__device__ __forceinline__ float sf_read(const T* row, int n, int per, T* held, float* smallest) {
  float high = -INFINITY, low = INFINITY;
  constexpr int V = 16 / (int)sizeof(T);
  int done = 0;
  if ((((uintptr_t)row) & 15) == 0) {
    const int nv = n / V;
#pragma unroll 8
    for (int i = threadIdx.x; i < nv; i += SF_THREADS) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row) + i);
      const T* x = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float v = to_f32<T>(x[e]);
        high = fmaxf(high, v);
        low = fminf(low, v > -INFINITY ? v : INFINITY);
      }
      if (RESIDENT) reinterpret_cast<uint4*>(held)[i] = raw;
    }
    done = nv * V;
  }
#pragma unroll 8
  for (int i = done + threadIdx.x; i < (RESIDENT ? per : n); i += SF_THREADS) {
    const T x = i < n ? row[i] : from_f32<T>(-INFINITY);
    const float v = to_f32<T>(x);
    high = fmaxf(high, v);
    low = fminf(low, v > -INFINITY ? v : INFINITY);
    if (RESIDENT) held[i] = x;
  }
  *smallest = low;
  return high;
}

template <typename T, bool RESIDENT>
__global__ void __launch_bounds__(SF_THREADS, 1024 / SF_THREADS) sample_filtered_kernel(const __grid_constant__ SfArgs a) {
  pdl_launch_dependents();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  SfShared& s = *reinterpret_cast<SfShared*>(smem_raw);
  T* held = reinterpret_cast<T*>(smem_raw + ((sizeof(SfShared) + 15) & ~(size_t)15));
  const unsigned rank = sf_rank(), blocks = sf_size();
  const int r = blockIdx.x / blocks;
  const int first = min(a.vocab, (int)rank * a.per);
  SfRow<T, RESIDENT> row{a, s, held, (const T*)a.logits + (size_t)r * a.ld + first, min(a.vocab, first + a.per) - first, rank, blocks};
  for (int b = threadIdx.x; b < SF_STEPS; b += SF_THREADS) s.one[b] = s.two[b] = 0;
  if (threadIdx.x < 32) {
    const unsigned long long x = a.table[threadIdx.x];
    s.table[threadIdx.x] = x;
    s.small_table[threadIdx.x] = (int)((x + (1ull << (SF_POINT - 31))) >> (SF_POINT - 30));
  }
  if (threadIdx.x == 0) s.high = s.low = s.listed = s.noted = 0;
  if (blocks > 1) sf_arrive();  // behind what this thread has set: whoever has waited finds it, in this block too
  pdl_wait();
  const float temperature = a.temperatures ? a.temperatures[r] : a.temperature;
  const float top_p = a.top_ps ? a.top_ps[r] : a.top_p, asked = a.min_ps ? a.min_ps[r] : a.min_p;
  const float min_p = asked > 0.f ? fminf(asked, 1.f) : 0.f;  // the most probable token always stays
  const int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
  float smallest;
  unsigned high = sf_key(sf_read<T, RESIDENT>(row.row, row.n, a.per, held, &smallest)), low = 0u - sf_key(smallest);
  if (blocks > 1) sf_wait();
  else __syncthreads();  // every block of the cluster runs: its shared memory may be written
  // the random number, drawn once for the whole cluster
  if (rank == 0 && threadIdx.x == 0) {
    const int i = a.index ? a.index[r] : r;
    float u;
    if (a.u) {
      u = a.u[r];
    } else if (i < 0 || i >= a.n_states) {
      u = __uint_as_float(SF_NO_STATE);
    } else {  // xorshift64*, as in sampling.cu
      unsigned long long* state = a.rng + i;
      unsigned long long x = *state;
      x ^= x >> 12; x ^= x << 25; x ^= x >> 27;
      *state = x;
      u = (float)((unsigned)((x * 0x2545F4914F6CDD1DULL) >> 32) >> 8) / 16777216.0f;
    }
    for (unsigned b = 0; b < blocks; ++b) sf_store(&s.found[0], b, __float_as_uint(u));
  }
  high = __reduce_max_sync(0xffffffffu, high);
  low = __reduce_max_sync(0xffffffffu, low);
  if ((threadIdx.x & 31) == 0) { atomicMax(&s.high, high); atomicMax(&s.low, low); }
  __syncthreads();
  high = s.high;
  low = s.low;
  row.exchange_max(&high, &low);
  const float asked_u = __uint_as_float((unsigned)s.found[0]), u = asked_u > 0.f ? asked_u : 0.f;
  if (a.u == nullptr && (unsigned)s.found[0] == SF_NO_STATE) high = 0u;  // as a row without a number above -inf
  unsigned chosen = high;
  unsigned long long tie = 0;
  if (high != 0u && temperature > 0.f) {
    row.topf = sf_value(high);
    row.top = (double)row.topf;
    row.infinite = row.topf == INFINITY;
    row.per_t = 1.0 / (double)temperature;
    const double c = 1.4426950408889634 * row.per_t;
    row.t_hi = (float)row.per_t;
    row.t_lo = (float)(row.per_t - (double)row.t_hi);
    const float octaves = (row.topf - sf_value(0u - low)) * (float)c;
    row.fine = 0;
    while (row.fine < 5 && octaves * (float)(64 << row.fine) < (float)(SF_STEPS - 2)) ++row.fine;
    row.steps = (float)(32 << row.fine) * 1.442695f;
    const bool k_on = top_k > 0 && top_k < a.vocab, p_on = top_p > 0.f && top_p < 1.f, m_on = min_p > 0.f;
    bool by_bits = row.infinite || !(c > 1e-30 && c < 1e30) || a.per > SF_COUNTED;
    if (!by_bits) {
      row.count_steps(k_on);
      sf_sync(blocks);
      if (rank == 0) row.make_plan(k_on, (unsigned)top_k, p_on, top_p, m_on, min_p, temperature, u);
      sf_sync(blocks);
      by_bits = s.plan.by_bits;
      if (!by_bits) {
        row.hand_over(k_on);
        sf_sync(blocks);  // the last time that another block is needed
        if (rank == 0) {
          if (s.listed > SF_THREADS) row.template decide<SF_THREADS, SF_LIST / SF_THREADS>(top_p, u, a.out + r);
          else if (s.listed > 32) row.template decide<SF_THREADS, 1>(top_p, u, a.out + r);
          else if (threadIdx.x < 32) row.template decide<32, 1>(top_p, u, a.out + r);
        }
        return;
      }
    }
    unsigned long long valid = 0, before;
    for (int i = threadIdx.x; i < row.n; i += SF_THREADS) valid += row.key(i) != 0u;
    valid = row.exchange_sum(row.block_sum64(valid), &before);
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
    if (p_on) {
      const unsigned long long all = kept_mass(0.f);
      const unsigned long long thr = min((unsigned long long)((double)top_p * (double)all), all - 1);
      unsigned long long above;
      const unsigned k = row.template first_exceeding<false>(thr, &above);
      const unsigned long long w = row.fixed(row.weight(k)), j = (thr - above) / w + 1;
      ties = k == cut ? min(ties, j) : j;
      cut = k;
    }
    const unsigned long long all = kept_mass(min_p);
    const unsigned long long thr = min((unsigned long long)((double)u * (double)all), all - 1);
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
  sf_sync(blocks);  // no block leaves while another may still read from it or write to it
}

template <typename T, bool RESIDENT>
static int sf_launch(const SfArgs& a, int n_rows, int blocks, size_t smem, cudaStream_t stream) {
  static BnGrant grant;
  cudaError_t e = grant.ask((const void*)sample_filtered_kernel<T, RESIDENT>, smem, 0);
  if (e != cudaSuccess) return BN_ERR_LAUNCH + (int)e;
  e = bn_launch_cluster(sample_filtered_kernel<T, RESIDENT>, dim3((unsigned)(n_rows * blocks)), dim3(SF_THREADS), smem, stream,
                        dim3((unsigned)blocks, 1, 1), a);
  return e == cudaSuccess ? BN_OK : BN_ERR_LAUNCH + (int)e;
}
template <typename T>
static int sf_run(SfArgs& a, int n_rows, cudaStream_t stream) {
  int device = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (e != cudaSuccess) return BN_ERR_LAUNCH + (int)e;
  // Blocks of a row: so many that each has 4,096 numbers (one row of 32,000: 14.9 us with one block, 13.2 with two, 11.3 with eight), but not
  // more than 2.75 an SM in all, of which two run at once (64 rows of 128,256: 36.7 us with four blocks a row, 49.6 with eight; 200 of 50,257: 54 with two, 65 with
  // four).  Clusters of eight only for some ten rows: more of them do not find their place at once (12 rows of 128,256: 22.6 us with eight, 19.8 with four; 10: 20.0 and 19.8;
  // 40: 37.4 and 32.6).  No fewer blocks than add up a row's numbers.
  int blocks = SF_MAX_CLUSTER;
  while (blocks > 1 && a.vocab <= blocks / 2 * 4096) blocks /= 2;
  if (blocks == 8 && 64ll * n_rows > 5ll * sms && (a.vocab + 3) / 4 <= SF_COUNTED - 8) blocks = 4;
  while (blocks > 1 && 4ll * n_rows * blocks > 11ll * sms && (a.vocab + blocks / 2 - 1) / (blocks / 2) <= SF_COUNTED - 8) blocks /= 2;
  a.per = (((a.vocab + blocks - 1) / blocks) + 7) & ~7;
  // The row stays in shared memory where two blocks an SM still fit, or where there is one at most; else later passes find it in the L2 (256 rows of 32,000 in float32,
  // one block each: 31.9 us from the L2, 39.9 held).
  const size_t base = (sizeof(SfShared) + 15) & ~(size_t)15, held = (((size_t)a.per * sizeof(T)) + 15) & ~(size_t)15;
  const bool resident = base + held <= ((long long)n_rows * blocks <= sms ? 220 : 112) * 1024 && a.per <= 128 * SF_THREADS;
  return resident ? sf_launch<T, true>(a, n_rows, blocks, base + held, stream) : sf_launch<T, false>(a, n_rows, blocks, base, stream);
}

// logits [n_rows, vocab] of `dtype`, rows ld numbers apart.  The four parameters hold for all rows where their array is null.  u: a number in
// [0, 1) per row, or null: drawn from the generator rng[index ? index[r] : r] (of n_states), which is advanced.  out: the tokens, -1 for a row
// without a number above -inf, or without a generator.
extern "C" int bn_sample_filtered(const void* logits, int dtype, long long ld, int n_rows, int vocab, float temperature, const float* temperatures,
                                  int top_k, const int* top_ks, float top_p, const float* top_ps, float min_p, const float* min_ps, const float* u,
                                  unsigned long long* rng, int n_states, const int* index, int* out, cudaStream_t stream) {
  if (n_rows <= 0) return BN_OK;
  if (!logits || !out || vocab <= 0 || ld < vocab || (!u && !rng) || (dtype != BN_F32 && dtype != BN_BF16) || n_rows > 0x7fffffff / SF_MAX_CLUSTER)
    return BN_ERR_BAD_ARG;
  SfArgs a = {};
  a.logits = logits; a.ld = ld; a.vocab = vocab;
  a.temperature = temperature; a.top_p = top_p; a.min_p = min_p; a.top_k = top_k;
  a.temperatures = temperatures; a.top_ks = top_ks; a.top_ps = top_ps; a.min_ps = min_ps;
  a.u = u; a.rng = rng; a.n_states = n_states; a.index = index; a.out = out;
  int bits = 0;
  while ((1ll << bits) < vocab) ++bits;
  a.scale_bits = 62 - bits < SF_POINT ? 62 - bits : SF_POINT;  // the sum of all weights stays below 2^62
  for (int j = 0; j < 32; ++j) a.table[j] = (unsigned long long)llround(ldexp(exp2(-j / 32.0), SF_POINT));
  return dtype == BN_F32 ? sf_run<float>(a, n_rows, stream) : sf_run<__nv_bfloat16>(a, n_rows, stream);
}
