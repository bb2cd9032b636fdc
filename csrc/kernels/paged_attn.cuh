// What the kernels of the paged attention share: the work list, how its tiles are
// dealt to CTAs, and where partial results lie.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"

namespace nk {
namespace pa {

// One item, eight int32 (laid out by the host): (row, query head) pairs that lie
// one after another, against a run of keys.
struct Item {
  int shared;  // 1: the shared pages of a group, 0: the rest of a sequence
  int first;   // shared: first sequence of the group; else the slot
  int count;   // shared: sequences of the group
  int row0;    // first pair: row * share + head
  int rows;    // pairs
  int key0;    // first key
  int keys;    // shared: number of keys; else the tokens that follow the item's last row
  int alone;   // its pairs have no other run of keys
};

// The items of one kernel. Their units are numbered one after another, head by head,
// and every worker (a warp, or a CTA) takes an equal contiguous share of the numbers.
// An item with keys has `over` units for what a worker spends on any item (look-ups,
// Q, write-out), then one for each tile of its keys.
struct Work {
  const Item* items;
  int n;           // items of one head
  int workers;
  int over;
  int* unit0;      // n + 1: first unit of each item, of one head (written by CTA 0)
  long continued;  // partial slots of the workers' pieces that continue an earlier worker's
  int item_rows;   // slots of each
  int least;       // units of a share, at least
};
constexpr int kSmallRows = 16;
constexpr int kBig = 1 << 30;  // marks an item of work[1] in the join's lists

struct Args {
  const void* q;
  long q_row, q_head;
  const int *table, *lens;
  int width, page, pages;
  const int *slot_of_seq, *row_slot, *row_back;
  int rows, share, hk;
  float sl2;         // scale * log2(e)
  float* part_o;     // a partial output (D, unnormalised) a slot: (2, hk, rows * share), then the continued ones
  float2* part_ml;   // its maximum in base-2 units, and its sum
  Work work[2];      // on mma.sync, on tcgen05
  void* out;
  long out_row, out_head;
  float* lse;        // may be null
  int* err;
  const void *k, *v;     // the pages, beside the tensor maps of them
  long k_page, v_page;   // elements
};

// mbar_wait that polls for a while before it first reads the timer, which would
// otherwise stand in the path of every wait that has to wait at all. By a whole warp,
// with one answer for all its lanes: a warp that gives up leaves its role as a whole,
// so that none of its lanes stands at a barrier, shuffle or tensor-memory access that
// the others no longer reach.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int code, int* err) {
#pragma unroll 1
  for (int i = 0; i < 64; ++i)
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, code, err));
}

// 1 / sum; 0 for a row without keys, NaN where the sum is.
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

__device__ __forceinline__ int length_of(const Args& a, int slot) {
  return min(max(a.lens[slot], 0), a.width * a.page);
}

template <int TK>
__device__ __forceinline__ int units_of(const Args& a, const Work& w, const Item& it) {
  const int keys = it.shared ? it.keys : length_of(a, it.first) - it.keys - it.key0;
  return keys > 0 ? w.over + (keys + TK - 1) / TK : 0;
}

// Units are dealt in shares of equal size (the last one may be shorter): worker c
// takes [c * size, (c + 1) * size) of `total`.
__device__ __forceinline__ int share_size(int workers, int total, int least) {
  return max((total + workers - 1) / workers, least);
}

__device__ __forceinline__ long base_slot(const Args& a, int shared, int head, int pair) {
  return (long(shared) * a.hk + head) * a.rows * a.share + pair;
}
// An item's pairs are consecutive and at most item_rows (a power of two), so their
// low bits tell them apart.
__device__ __forceinline__ long continued_slot(const Work& w, int worker, int pair) {
  return w.continued + long(worker) * w.item_rows + (pair & (w.item_rows - 1));
}

// The first unit of every item, in shared memory while there are few items; of more,
// only of each thread's run [t * per, (t + 1) * per).
constexpr int kFirsts = 512;
template <int THREADS>
struct Deal {
  int run[THREADS + 1];  // units before each thread's run; the last entry: units of one head
  int first[kFirsts + 1];
};

// Numbers the items' units; CTA 0 leaves every item's first one for the joining
// kernel. All THREADS threads of the CTA take part. Returns the units of one head.
template <int TK, int THREADS>
__device__ __forceinline__ int deal(const Args& a, const Work& w, Deal<THREADS>& d) {
  const int tid = threadIdx.x, per = (w.n + THREADS - 1) / THREADS;
  const int i0 = min(w.n, tid * per), i1 = min(w.n, i0 + per);
  int mine = 0;
  for (int i = i0; i < i1; ++i) mine += units_of<TK>(a, w, w.items[i]);
  d.run[tid] = mine;
  __syncthreads();
  if (tid < 32) {
    int run = 0;
    for (int b = 0; b < THREADS; b += 32) {
      const int v = d.run[b + tid];
      int x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (tid >= o) x += y;
      }
      d.run[b + tid] = run + x - v;
      run += __shfl_sync(0xffffffffu, x, 31);
    }
    if (tid == 0) d.run[THREADS] = run;
  }
  __syncthreads();
  if (blockIdx.x == 0 || w.n <= kFirsts) {
    int t = d.run[tid];
    for (int i = i0; i < i1; ++i) {
      if (w.n <= kFirsts) d.first[i] = t;
      if (blockIdx.x == 0) w.unit0[i] = t;
      t += per == 1 ? mine : units_of<TK>(a, w, w.items[i]);
    }
    if (tid == 0) {
      if (w.n <= kFirsts) d.first[w.n] = d.run[THREADS];
      if (blockIdx.x == 0) w.unit0[w.n] = d.run[THREADS];
    }
  }
  __syncthreads();
  return d.run[THREADS];
}

// The item that holds unit t of a head; `at` becomes its first unit, `n` its units.
template <int TK, int THREADS>
__device__ __forceinline__ int item_of(const Args& a, const Work& w, const Deal<THREADS>& d, int t, int& at, int& n) {
  const bool few = w.n <= kFirsts;
  const int* first = few ? d.first : d.run;
  int lo = 0, hi = (few ? w.n : THREADS) - 1;  // the last whose first unit is not past t
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (first[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  at = first[lo];
  if (few) {
    n = first[lo + 1] - at;
    return lo;
  }
  int i = lo * ((w.n + THREADS - 1) / THREADS);
  n = units_of<TK>(a, w, w.items[i]);
  while (at + n <= t) {
    at += n;
    n = units_of<TK>(a, w, w.items[++i]);
  }
  return i;
}

// A worker's piece of an item: the units [u0, u0 + units) of the item's n are its.
struct Span {
  int units, tile0, tiles;
  bool whole;  // all tiles of the item
};
__device__ __forceinline__ Span span_of(const Work& w, int u0, int n, int left) {
  Span s;
  s.units = min(n - u0, left);
  s.tile0 = max(0, u0 - w.over);
  s.tiles = max(0, u0 + s.units - w.over) - s.tile0;
  s.whole = s.tiles == n - w.over;
  return s;
}

// The table row that an item's keys are read through, and the end of those that
// exist; by a whole warp. Shared pages are read through the first sequence that
// holds all of them, else through the longest (idle slots hold none).
__device__ __forceinline__ void run_end(const Args& a, const Item& item, int& slot, int& end) {
  const int lane = threadIdx.x % 32;
  slot = item.first;
  if (!item.shared) {
    end = length_of(a, slot) - item.keys;
    return;
  }
  const int all = item.key0 + item.keys;
  int best = -1;
  for (int s = item.first; s < item.first + item.count && best < all; s += 32) {
    const bool there = s + lane < item.first + item.count;
    const int c = there ? a.slot_of_seq[s + lane] : 0, len = there ? length_of(a, c) : -1;
    const unsigned full = __ballot_sync(0xffffffffu, len >= all);
    int most = len;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    const unsigned longest = __ballot_sync(0xffffffffu, len == most);
    const int from = __ffs(full ? full : longest) - 1;
    if (full || most > best) {
      best = __shfl_sync(0xffffffffu, len, from);
      slot = __shfl_sync(0xffffffffu, c, from);
    }
  }
  end = min(best, all);
}

template <typename T>
__device__ __forceinline__ uint32_t pack(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float x, float y) { return pack_bf16x2(x, y); }
template <>
__device__ __forceinline__ uint32_t pack<__half>(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) { return unpack_bf16x2(w); }
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Items of many rows, on tcgen05 (paged_attn_tc.cu). The map's boxes are
// min(page, kBigKeys) rows of 64 columns.
constexpr int kBigKeys = 128, kBigRows = 256;
template <typename T, int D>
void launch_big(const CUtensorMap& k, const CUtensorMap& v, const Args& a, cudaStream_t stream);

}  // namespace pa
}  // namespace nk
