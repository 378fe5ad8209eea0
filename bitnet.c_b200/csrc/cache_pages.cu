// Pages of a cache copied to other pages, in all planes at once, and the states of one sequence copied to other slots.
//
// A sequence that is forked shares its full pages with its forks; what has to be copied is the page that is only partly filled
// (its first `rows` rows of every head) and the fixed-size states.  The same copies move whole pages when a pool is compacted.
// Nothing is computed: the bytes bound it.  Which pages go where travels as an argument of the launch (no copy to the device, and
// the host's lists may change as soon as the call returns).  Moves with one source are one group: what they copy is read once
// and stored to every destination, so that n forks take n + 1 times the page's bytes and not 2 n.
//
// A block takes pieces of CP_THREADS x CP_UNROLL units, all loads of a thread in flight before its first store.  Units are 16 bytes where
// rows and addresses allow it, else the largest power of two that they allow.  Measured: 64 whole pages of 32 planes with 8 heads of 128 (1.07 GB read
// and written) 178 us, 6.0 TB/s; 51 rows of one page to 16 pages of such a cache 21.5 us (5.3 TB/s); a page of 16 planes to two 2.4 us, the launch.
#include "common.cuh"

#define CP_THREADS 256
#define CP_UNROLL 4
#define CP_MOVES 256    // destinations of one launch: the argument stays within 4 KB
#define CP_TENSORS 128  // state tensors of one launch

struct CpMoves {
  int src[CP_MOVES];
  int dst[CP_MOVES];
  unsigned short first[CP_MOVES + 1];  // group g goes to dst[first[g]] .. dst[first[g + 1] - 1]
  unsigned char rows[CP_MOVES];
};
struct CpPlanes {
  unsigned char* base[2];          // keys, values
  long long plane[2];              // bytes from plane to plane
  int head[2];                     // bytes of one head of a page
  int row[2];                      // bytes of a row of a head
  int heads, planes;
};

// `n` units of T at offsets that `at` gives, from `from` to every one of the destinations.
template <typename T, class At, class To>
__device__ __forceinline__ void copy_units(const unsigned char* from, unsigned n, unsigned first, unsigned step, At at, int to0, int to1, To to) {
  for (unsigned i0 = first; i0 < n; i0 += CP_UNROLL * step) {
    T v[CP_UNROLL];
    size_t off[CP_UNROLL];
#pragma unroll
    for (int u = 0; u < CP_UNROLL; ++u) {
      const unsigned i = i0 + u * step;
      if (i < n) {
        off[u] = at(i) * sizeof(T);
        v[u] = *reinterpret_cast<const T*>(from + off[u]);
      }
    }
    for (int t = to0; t < to1; ++t) {
      unsigned char* p = to(t);
#pragma unroll
      for (int u = 0; u < CP_UNROLL; ++u)
        if (i0 + u * step < n) *reinterpret_cast<T*>(p + off[u]) = v[u];
    }
  }
}

// grid: (pieces of a page, planes x {keys, values}, groups)
template <typename T>
__global__ void __launch_bounds__(CP_THREADS) copy_pages_kernel(const __grid_constant__ CpPlanes a, const __grid_constant__ CpMoves m) {
  pdl_wait();
  const int which = blockIdx.y / a.planes, plane = blockIdx.y % a.planes, g = blockIdx.z;
  unsigned char* base = a.base[which] + (size_t)plane * a.plane[which];
  const size_t page = (size_t)a.heads * a.head[which];
  const unsigned head = (unsigned)(a.head[which] / sizeof(T)), taken = (unsigned)(m.rows[g] * a.row[which] / sizeof(T));
  const unsigned char* from = base + (size_t)m.src[g] * page;
  const auto to = [&](int t) { return base + (size_t)m.dst[t] * page; };
  const unsigned first = blockIdx.x * CP_THREADS + threadIdx.x, step = gridDim.x * CP_THREADS;
  if (taken == head) {  // whole pages: the heads lie one behind the other
    copy_units<T>(from, head * a.heads, first, step, [&](unsigned i) { return (size_t)i; }, m.first[g], m.first[g + 1], to);
  } else {
    copy_units<T>(from, taken * a.heads, first, step, [&](unsigned i) { return (size_t)(i / taken) * head + i % taken; }, m.first[g], m.first[g + 1], to);
  }
  // the kernel behind this one may start as soon as all blocks have ended, and may ask for pages before it waits: they are in the L2 by then
  __threadfence();
}

// groups: n_groups times (source page, rows, number of destinations), then their n_dst destinations, group by group.  A destination is no
// group's source and no other's destination.  k (and v, or null): [planes, pages, heads, 64, row bytes].
extern "C" int bn_copy_pages(void* k, void* v, int planes, int pages, int heads, int k_row, int v_row, const int* groups, int n_groups,
                             int n_dst, cudaStream_t stream) {
  if (n_groups <= 0) return BN_OK;
  const int* dst = groups ? groups + 3 * (size_t)n_groups : nullptr;
  if (!k || !groups || planes <= 0 || pages <= 0 || heads <= 0 || k_row <= 0 || (v && v_row <= 0)) return BN_ERR_BAD_ARG;
  const int sides = v ? 2 : 1;
  if ((long long)planes * sides > 65535 || (long long)heads * BN_PAGE * (k_row > v_row ? k_row : v_row) > 0x7fffffffll) return BN_ERR_BAD_ARG;
  long long all = 0;
  for (int g = 0; g < n_groups; ++g) {
    if (groups[3 * g] < 0 || groups[3 * g] >= pages || groups[3 * g + 1] <= 0 || groups[3 * g + 1] > BN_PAGE || groups[3 * g + 2] <= 0) return BN_ERR_BAD_ARG;
    all += groups[3 * g + 2];
  }
  if (all != n_dst) return BN_ERR_BAD_ARG;
  for (int i = 0; i < n_dst; ++i)
    if (dst[i] < 0 || dst[i] >= pages) return BN_ERR_BAD_ARG;
  CpPlanes a = {};
  a.base[0] = (unsigned char*)k; a.base[1] = (unsigned char*)v;
  a.row[0] = k_row; a.row[1] = v ? v_row : 0;
  a.heads = heads; a.planes = planes;
  uintptr_t align = (uintptr_t)k | (uintptr_t)k_row | (v ? (uintptr_t)v | (uintptr_t)v_row : 0);
  for (int i = 0; i < 2; ++i) {
    a.head[i] = BN_PAGE * a.row[i];
    a.plane[i] = (long long)pages * heads * a.head[i];
  }
  CpMoves m;
  int g = 0, done = 0, at = 0;  // the next group, how many of its destinations went before, the next destination
  while (g < n_groups) {
    int n = 0, to = 0, most = 0;
    while (g < n_groups && to < CP_MOVES) {
      const int left = groups[3 * g + 2] - done, take = left < CP_MOVES - to ? left : CP_MOVES - to;
      m.src[n] = groups[3 * g]; m.rows[n] = (unsigned char)groups[3 * g + 1]; m.first[n] = (unsigned short)to;
      if (groups[3 * g + 1] > most) most = groups[3 * g + 1];
      for (int i = 0; i < take; ++i) m.dst[to + i] = dst[at + i];
      to += take; at += take; ++n;
      if (take == left) { ++g; done = 0; } else { done += take; }
    }
    m.first[n] = (unsigned short)to;
    const int row = k_row > a.row[1] ? k_row : a.row[1];
    const int unit = (align & 15) == 0 ? 16 : (align & 7) == 0 ? 8 : (align & 3) == 0 ? 4 : (align & 1) == 0 ? 2 : 1;
    const long long units = (long long)heads * most * row / unit;
    long long pieces = (units + CP_THREADS * CP_UNROLL - 1) / (CP_THREADS * CP_UNROLL);
    if (pieces > 65535) pieces = 65535;
    const dim3 grid((unsigned)pieces, (unsigned)(planes * sides), (unsigned)n);
    switch (unit) {
      case 16: BN_LAUNCH(copy_pages_kernel<uint4>, grid, CP_THREADS, 0, stream, a, m); break;
      case 8: BN_LAUNCH(copy_pages_kernel<uint2>, grid, CP_THREADS, 0, stream, a, m); break;
      case 4: BN_LAUNCH(copy_pages_kernel<unsigned>, grid, CP_THREADS, 0, stream, a, m); break;
      case 2: BN_LAUNCH(copy_pages_kernel<unsigned short>, grid, CP_THREADS, 0, stream, a, m); break;
      default: BN_LAUNCH(copy_pages_kernel<unsigned char>, grid, CP_THREADS, 0, stream, a, m); break;
    }
    BN_CHECK_LAUNCH();
  }
  return BN_OK;
}

// ---- states ------------------------------------------------------------------------------------
struct CpStates {
  unsigned char* base[CP_TENSORS];
  long long bytes[CP_TENSORS];  // of one slot
};
struct CpSlots {
  int n, src;
  int dst[CP_MOVES];
};

// grid: (pieces of the largest state, tensors)
__global__ void __launch_bounds__(CP_THREADS) copy_slots_kernel(const __grid_constant__ CpStates a, const __grid_constant__ CpSlots s) {
  pdl_wait();
  unsigned char* base = a.base[blockIdx.y];
  const size_t bytes = (size_t)a.bytes[blockIdx.y];
  const unsigned char* from = base + (size_t)s.src * bytes;
  const auto to = [&](int t) { return base + (size_t)s.dst[t] * bytes; };
  const auto same = [](unsigned i) { return (size_t)i; };
  const unsigned first = blockIdx.x * CP_THREADS + threadIdx.x, step = gridDim.x * CP_THREADS;
  const uintptr_t align = (uintptr_t)base | bytes;
  if ((align & 15) == 0) copy_units<uint4>(from, (unsigned)(bytes / 16), first, step, same, 0, s.n, to);
  else if ((align & 3) == 0) copy_units<unsigned>(from, (unsigned)(bytes / 4), first, step, same, 0, s.n, to);
  else copy_units<unsigned char>(from, (unsigned)bytes, first, step, same, 0, s.n, to);
  __threadfence();
}

// where: n_tensors times (address, bytes of one slot), on the host; slot `src` of each tensor goes to the slots dst, none of which is src or
// named twice.
extern "C" int bn_copy_slots(const long long* where, int n_tensors, int n_slots, int src, const int* dst, int n_dst, cudaStream_t stream) {
  if (n_tensors <= 0 || n_dst <= 0) return BN_OK;
  if (!where || !dst || src < 0 || src >= n_slots) return BN_ERR_BAD_ARG;
  for (int i = 0; i < n_dst; ++i)
    if (dst[i] < 0 || dst[i] >= n_slots || dst[i] == src) return BN_ERR_BAD_ARG;
  for (int t0 = 0; t0 < n_tensors; t0 += CP_TENSORS) {
    CpStates a = {};
    const int n = n_tensors - t0 < CP_TENSORS ? n_tensors - t0 : CP_TENSORS;
    long long pieces = 1;
    for (int t = 0; t < n; ++t) {
      a.base[t] = (unsigned char*)where[2 * (t0 + t)];
      a.bytes[t] = where[2 * (t0 + t) + 1];
      if (a.bytes[t] < 0 || a.bytes[t] > 0x7fffffffll) return BN_ERR_BAD_ARG;
      const uintptr_t align = (uintptr_t)a.base[t] | (uintptr_t)a.bytes[t];
      const int unit = (align & 15) == 0 ? 16 : (align & 3) == 0 ? 4 : 1;
      const long long p = (a.bytes[t] / unit + CP_THREADS * CP_UNROLL - 1) / (CP_THREADS * CP_UNROLL);
      if (p > pieces) pieces = p;
    }
    if (pieces > 65535) pieces = 65535;
    for (int i0 = 0; i0 < n_dst; i0 += CP_MOVES) {
      CpSlots s = {};
      s.src = src;
      s.n = n_dst - i0 < CP_MOVES ? n_dst - i0 : CP_MOVES;
      for (int i = 0; i < s.n; ++i) s.dst[i] = dst[i0 + i];
      BN_LAUNCH(copy_slots_kernel, dim3((unsigned)pieces, (unsigned)n), CP_THREADS, 0, stream, a, s);
      BN_CHECK_LAUNCH();
    }
  }
  return BN_OK;
}
