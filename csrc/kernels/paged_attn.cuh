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
  int small;   // keys are split over the warps
};

// The items of one kernel. Their tiles are numbered one after another, head by
// head, and every CTA takes an equal contiguous share of the numbers.
struct Work {
  const Item* items;
  int n;           // items of one head
  int ctas;
  int* tile0;      // n + 1: first tile of each item, of one head (written by CTA 0)
  long continued;  // partial slots of the CTAs' pieces that continue an earlier CTA's
  int item_rows;   // slots of each
};
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
  int* err;
};

__device__ __forceinline__ int length_of(const Args& a, int slot) {
  return min(max(a.lens[slot], 0), a.width * a.page);
}

template <int TK>
__device__ __forceinline__ int tiles_of(const Args& a, const Item& it) {
  const int keys = it.shared ? it.keys : length_of(a, it.first) - it.keys - it.key0;
  return keys > 0 ? (keys + TK - 1) / TK : 0;
}

// CTA c's share of `total` tiles is [begin(c), begin(c + 1)); there are at most
// as many shares as tiles.
__device__ __forceinline__ int shares(int ctas, long total) { return int(total < ctas ? total : ctas); }
__device__ __forceinline__ long share_begin(long c, int n, long total) { return c * total / n; }
__device__ __forceinline__ int share_of(long t, int n, long total) { return int(((t + 1) * n - 1) / total); }

__device__ __forceinline__ long base_slot(const Args& a, int shared, int head, int pair) {
  return (long(shared) * a.hk + head) * a.rows * a.share + pair;
}
__device__ __forceinline__ long cta_slot(const Work& w, int cta, int r) {
  return w.continued + long(cta) * w.item_rows + r;
}

// Thread t's run of items is [t * per, (t + 1) * per); sums[t] becomes the tiles
// before it. Returns the tiles of one head; CTA 0 leaves every item's first tile
// for the joining kernel. All THREADS threads of the CTA take part; sums has one
// entry more.
template <int TK, int THREADS>
__device__ __forceinline__ int deal(const Args& a, const Work& w, int* sums) {
  const int tid = threadIdx.x, per = (w.n + THREADS - 1) / THREADS;
  const int i0 = min(w.n, tid * per), i1 = min(w.n, i0 + per);
  int mine = 0;
  for (int i = i0; i < i1; ++i) mine += tiles_of<TK>(a, w.items[i]);
  sums[tid] = mine;
  __syncthreads();
  if (tid < 32) {
    int run = 0;
    for (int b = 0; b < THREADS; b += 32) {
      const int v = sums[b + tid];
      int x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (tid >= o) x += y;
      }
      sums[b + tid] = run + x - v;
      run += __shfl_sync(0xffffffffu, x, 31);
    }
    if (tid == 0) sums[THREADS] = run;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    int t = sums[tid];
    for (int i = i0; i < i1; ++i) {
      w.tile0[i] = t;
      t += tiles_of<TK>(a, w.items[i]);
    }
    if (tid == 0) w.tile0[w.n] = sums[THREADS];
  }
  return sums[THREADS];
}

// The item that holds tile t of a head; `at` becomes its first tile, `n` its tiles.
template <int TK, int THREADS>
__device__ __forceinline__ int item_of(const Args& a, const Work& w, const int* sums, int t, int& at, int& n) {
  int lo = 0, hi = THREADS - 1;  // the last run whose first tile is not past t
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (sums[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  int i = lo * ((w.n + THREADS - 1) / THREADS);
  at = sums[lo];
  n = tiles_of<TK>(a, w.items[i]);
  while (at + n <= t) {
    at += n;
    n = tiles_of<TK>(a, w.items[++i]);
  }
  return i;
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

// Items of many rows, on tcgen05 (paged_attn_tc.cu). The map's boxes are
// min(page, kBigKeys) rows of 64 columns.
constexpr int kBigKeys = 128, kBigRows = 256;
template <typename T, int D>
void launch_big(const CUtensorMap& k, const CUtensorMap& v, const Args& a, cudaStream_t stream);

}  // namespace pa
}  // namespace nk
