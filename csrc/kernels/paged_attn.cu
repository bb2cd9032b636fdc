// Attention of new tokens over a paged KV cache, with the pages that a group of
// sequences shares read once for all of them.
//
//   out[r, hq] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q_r . k_j - max)
//
// over the keys j < limit(r) = lens[slot(r)] - back(r) of the row's sequence: the
// row sees every token up to its own. A row without keys gives 0 (LSE -inf).
//
// The work of one kv head is a list of items, made once for a plan: an item is up
// to 64 (row, query head) pairs against a run of keys, either the shared pages of
// a group (rows of all its sequences) or the rest of one sequence. Tiles of 64
// keys of all items are numbered one after another and the CTAs take equal
// contiguous shares, whatever the lengths are; they are read on the device, so a
// captured graph follows them. Where a share ends inside an item, both CTAs leave
// a partial (max, sum, unnormalised output, fp32); a second kernel joins a row's
// partials from the shared keys and from its own.
//
// CTA: a producer warp works out 32 tiles at a time (one a lane), then one thread
// issues the TMA loads of a tile's pages; four warps compute on mma.sync, with the
// running maximum and sum in registers. Items of up to 16 pairs (single tokens)
// split a tile's keys over the warps, larger ones their rows. Tensor-core work is
// far below what the loads take for few rows.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <climits>

#include "flash_common.cuh"
#include "message.h"
#include "paged_attn.cuh"
#include "status.h"
#include "tma_host.h"

namespace nk {
namespace pa {

constexpr int TK = 64;            // keys of a tile
constexpr int kConsumers = 128;   // four warps
constexpr int kThreads = kConsumers + 32;
constexpr int kStages = 3;
constexpr int kRing = 64;         // tile records, two batches of 32
constexpr int kMaxBoxes = 8;      // pages of a tile (page of 8 rows)
constexpr int kSmallRows = 16;    // items up to here split the keys over the warps
constexpr int kItemRows = 64;

struct Tile {
  int item, head, key0, valid;  // valid: keys of the tile that are loaded
  int flags, row0, rows, small;
  int box[kMaxBoxes];           // page of each box
};
constexpr int kFirst = 1, kLast = 2, kContinued = 4;  // of the CTA's piece of the item

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
  mma16816(d, x, b0, b1);
}
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}
template <int D>
struct Smem {
  static constexpr int kSub = TK * 128;             // 64 columns of a tile's rows, 128-byte swizzled
  static constexpr int kTile = kSub * (D / 64);     // K or V of a tile
  static constexpr int kMerge = kSmallRows * D * 4;
  static constexpr int kBytes = 1024 + kStages * 2 * kTile + kMerge;
};

// Barrier of the four computing warps; like every wait it ends after a limit.
__device__ __forceinline__ bool consumers_sync(uint64_t* bar, uint32_t& phase, int* err) {
  __syncwarp();
  if (threadIdx.x % 32 == 0) mbar_arrive(bar);
  const bool ok = mbar_wait(bar, phase, kErrTimeoutOther, err);
  phase ^= 1;
  return ok;
}

// The state of a warp's 16 rows; thread (g, t4) holds rows g and g + 8.
template <int D>
struct Acc {
  float o[D / 8][4];
  float m[2], l[2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }
};

// Scores, softmax step and P V of one warp's 16 rows against NK keys of a tile,
// from key k0 of it on. lim: keys of the tile that each of the two rows sees.
template <typename T, int D, int NK>
__device__ __forceinline__ void step(Acc<D>& acc, const uint32_t (&qf)[D / 16][4], uint32_t sK, uint32_t sV, int k0,
                                     const int (&lim)[2], float sl2) {
  constexpr int kSub = Smem<D>::kSub;
  const int t4 = threadIdx.x & 3;
  float s[NK / 8][4];
#pragma unroll
  for (int n = 0; n < NK / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
    for (int np = 0; np < NK / 16; ++np) {
      uint32_t b[4];
      load_b_nk<64>(sK + (kk / 4) * kSub, k0 + np * 16, (kk % 4) * 16, b);
      mma<T>(s[2 * np], qf[kk], b[0], b[1]);
      mma<T>(s[2 * np + 1], qf[kk], b[2], b[3]);
    }
  const bool masked = k0 + NK > min(lim[0], lim[1]);
  float mx[2] = {acc.m[0], acc.m[1]};
#pragma unroll
  for (int n = 0; n < NK / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // A hidden score is replaced, whatever stood in its place.
      const bool hide = masked && k0 + n * 8 + t4 * 2 + (e & 1) >= lim[e >> 1];
      s[n][e] = hide ? -INFINITY : s[n][e] * sl2;
      mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
    }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
    mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
  }
  float ref[2], sum[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    ref[i] = mx[i] == -INFINITY ? 0.f : mx[i];  // a row that has seen no key yet
    const float alpha = ex2_approx(acc.m[i] - ref[i]);
    acc.l[i] *= alpha;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      acc.o[n][2 * i] *= alpha;
      acc.o[n][2 * i + 1] *= alpha;
    }
    acc.m[i] = mx[i];
  }
#pragma unroll
  for (int n = 0; n < NK / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[n][e] = ex2_approx(s[n][e] - ref[e >> 1]);
      sum[e >> 1] += s[n][e];
    }
  acc.l[0] += sum[0];  // this thread's columns; the quad's sums meet at the end of the item
  acc.l[1] += sum[1];
#pragma unroll
  for (int ks = 0; ks < NK / 16; ++ks) {
    // P is rounded to the values' type for the tensor core; the sum keeps fp32.
    const uint32_t p[4] = {pack<T>(s[2 * ks][0], s[2 * ks][1]), pack<T>(s[2 * ks][2], s[2 * ks][3]),
                           pack<T>(s[2 * ks + 1][0], s[2 * ks + 1][1]), pack<T>(s[2 * ks + 1][2], s[2 * ks + 1][3])};
#pragma unroll
    for (int n = 0; n < D / 16; ++n) {
      uint32_t b[4];
      load_b_kn<64>(sV + (n / 4) * kSub, (n % 4) * 16, k0 + ks * 16, b);
      mma<T>(acc.o[2 * n], p, b[0], b[1]);
      mma<T>(acc.o[2 * n + 1], p, b[2], b[3]);
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const Args a) {
  using S = Smem<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_merge = reinterpret_cast<float*>(smem + kStages * 2 * S::kTile);
  __shared__ Tile ring[kRing];
  __shared__ int s_sum[kThreads + 1];
  __shared__ float s_ml[2][kSmallRows];
  __shared__ uint64_t full[kStages], empty[kStages], together;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kConsumers / 32);
    }
    mbar_init(&together, kConsumers / 32);
    fence_barrier_init();
  }
  const Work& work = a.work[0];
  const int head_tiles = deal<TK, kThreads>(a, work, s_sum);
  const long total = long(head_tiles) * a.hk;
  const int n_shares = shares(work.ctas, total);
  if (int(blockIdx.x) >= n_shares) return;
  const long t_begin = share_begin(blockIdx.x, n_shares, total);
  const int n_tiles = int(share_begin(blockIdx.x + 1, n_shares, total) - t_begin);
  const int box_rows = min(a.page, TK);

  if (warp == kConsumers / 32) {
    for (int base = 0; base < n_tiles; base += 32) {
      if (base + lane < n_tiles) {
        const long t = t_begin + base + lane;
        Tile r;
        r.head = int(t / head_tiles);
        const int tt = int(t % head_tiles);
        int at, n;
        const int i = item_of<TK, kThreads>(a, work, s_sum, tt, at, n);
        const Item it = work.items[i];
        r.item = i;
        r.key0 = it.key0 + (tt - at) * TK;
        r.row0 = it.row0;
        r.rows = it.rows;
        r.small = it.small;
        r.flags = (tt == at || base + lane == 0 ? kFirst : 0) |
                  (tt == at + n - 1 || base + lane == n_tiles - 1 ? kLast : 0) |
                  (tt != at && base + lane == 0 ? kContinued : 0);
        int slot = it.first, end;
        if (it.shared) {
          // The shared pages are read through the first sequence that holds all of
          // them, else through the longest (idle slots hold none).
          int best = -1;
          for (int s = it.first; s < it.first + it.count; ++s) {
            const int c = a.slot_of_seq[s], len = length_of(a, c);
            if (len > best) {
              best = len;
              slot = c;
            }
            if (len >= it.key0 + it.keys) break;
          }
          end = min(best, it.key0 + it.keys);
        } else {
          end = length_of(a, slot) - it.keys;
        }
        r.valid = min(TK, max(0, end - r.key0));
#pragma unroll
        for (int b = 0; b < kMaxBoxes; ++b) {
          const int key = r.key0 + b * box_rows;
          int page = 0;
          if (b * box_rows < r.valid) {
            page = a.table[long(slot) * a.width + key / a.page];
            if (page < 0 || page >= a.pages) {
              atomicCAS(a.err, 0, kErrBounds);
              page = 0;
            }
          }
          r.box[b] = page;
        }
        ring[(base + lane) % kRing] = r;
      }
      __syncwarp();
      if (lane == 0) {
        for (int i = base; i < min(n_tiles, base + 32); ++i) {
          const int st = i % kStages;
          if (!mbar_wait(&empty[st], ((i / kStages) & 1) ^ 1, kErrTimeoutProducer, a.err)) {
            base = n_tiles;
            break;
          }
          const Tile& r = ring[i % kRing];
          const int boxes = (r.valid + box_rows - 1) / box_rows;
          if (boxes == 0) {
            mbar_arrive(&full[st]);
            continue;
          }
          mbar_arrive_expect_tx(&full[st], boxes * box_rows * D * 2 * 2);
          uint8_t* sK = smem + st * 2 * S::kTile;
          for (int b = 0; b < boxes; ++b) {
            const int row = r.head * a.page + (r.key0 + b * box_rows) % a.page;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              tma_load_3d(sK + c * S::kSub + b * box_rows * 128, &tm_k, &full[st], c * 64, row, r.box[b]);
              tma_load_3d(sK + S::kTile + c * S::kSub + b * box_rows * 128, &tm_v, &full[st], c * 64, row, r.box[b]);
            }
          }
        }
      }
      base = __shfl_sync(0xffffffffu, base, 0);
    }
    return;
  }

  const int g = lane >> 2, t4 = lane & 3;
  const T* Q = static_cast<const T*>(a.q);
  Acc<D> acc;
  uint32_t qf[D / 16][4];
  int lim[2];
  uint32_t phase = 0;
  bool continued = false;  // the piece at hand began in an earlier CTA
  for (int i = 0; i < n_tiles; ++i) {
    const int st = i % kStages;
    if (!mbar_wait(&full[st], (i / kStages) & 1, kErrTimeoutMma, a.err)) break;
    const Tile& r = ring[i % kRing];
    const int flags = r.flags, rows = r.rows, row0 = r.row0, head = r.head, valid = r.valid, key0 = r.key0;
    const bool small = r.small;
    const int wr = small ? 0 : warp * 16;  // first row of this warp
    if (flags & kFirst) {
      acc.clear();
      continued = flags & kContinued;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int rr = wr + g + 8 * e;
        lim[e] = INT_MAX / 2;  // rows past the item's: computed on zeros, never written
        const T* src = nullptr;
        if (rr < rows) {
          const int row = (row0 + rr) / a.share, h = (row0 + rr) % a.share;
          lim[e] = length_of(a, a.row_slot[row]) - a.row_back[row];
          src = Q + row * a.q_row + (head * a.share + h) * a.q_head;
        }
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          qf[kk][e] = src ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + t4 * 2) : 0u;
          qf[kk][e + 2] = src ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8 + t4 * 2) : 0u;
        }
      }
    }
    const uint32_t sK = smem_u32(smem + st * 2 * S::kTile), sV = sK + S::kTile;
    if (valid < TK) {
      // Rows past the last key hold what the page or an earlier tile held, which
      // may be anything: values are cleared, so that 0 * v is 0.
      for (int c = tid; c < (TK - valid) * (D / 8); c += kConsumers) {
        const int row = valid + c / (D / 8), ch = c % (D / 8);
        uint8_t* at = smem + (st * 2 + 1) * S::kTile + (ch / 8) * S::kSub + row * 128 + (ch % 8) * 16;
        *reinterpret_cast<uint4*>(at) = make_uint4(0, 0, 0, 0);
      }
      if (!consumers_sync(&together, phase, a.err)) return;
    }
    const int tl[2] = {min(lim[0] - key0, valid), min(lim[1] - key0, valid)};
    if (small) {
      step<T, D, 16>(acc, qf, sK, sV, warp * 16, tl, a.sl2);
    } else if (wr < rows) {
      step<T, D, TK>(acc, qf, sK, sV, 0, tl, a.sl2);
    }
    if (valid < TK) fence_proxy_async();  // the clearing stores come before the next load into this stage
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[st]);
    if (!(flags & kLast)) continue;

#pragma unroll
    for (int e = 0; e < 2; ++e) {
      acc.l[e] += __shfl_xor_sync(0xffffffffu, acc.l[e], 1);
      acc.l[e] += __shfl_xor_sync(0xffffffffu, acc.l[e], 2);
    }
    if (small) {
      // Warps 3, 2, 1 hand their rows down; warp 0 ends with all of them.
#pragma unroll 1
      for (int w = kConsumers / 32 - 1; w > 0; --w) {
        if (warp == w) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int rr = g + 8 * e;
            if (rr >= rows) continue;
            if (t4 == 0) {
              s_ml[0][rr] = acc.m[e];
              s_ml[1][rr] = acc.l[e];
            }
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
              *reinterpret_cast<float2*>(s_merge + rr * D + n * 8 + t4 * 2) =
                  make_float2(acc.o[n][2 * e], acc.o[n][2 * e + 1]);
          }
        }
        if (!consumers_sync(&together, phase, a.err)) return;
        if (warp == w - 1) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int rr = g + 8 * e;
            if (rr >= rows) continue;
            const float m2 = s_ml[0][rr], m = fmaxf(acc.m[e], m2), ref = m == -INFINITY ? 0.f : m;
            const float x = exp2f(acc.m[e] - ref), y = exp2f(m2 - ref);
            acc.m[e] = m;
            acc.l[e] = acc.l[e] * x + s_ml[1][rr] * y;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
              const float2 o = *reinterpret_cast<const float2*>(s_merge + rr * D + n * 8 + t4 * 2);
              acc.o[n][2 * e] = acc.o[n][2 * e] * x + o.x * y;
              acc.o[n][2 * e + 1] = acc.o[n][2 * e + 1] * x + o.y * y;
            }
          }
        }
        if (!consumers_sync(&together, phase, a.err)) return;
      }
    }
    if (small && warp > 0) continue;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int rr = wr + g + 8 * e;
      if (rr >= rows) continue;
      const int shared = work.items[r.item].shared;
      const long slot = continued ? cta_slot(work, blockIdx.x, rr) : base_slot(a, shared, head, row0 + rr);
      if (t4 == 0) a.part_ml[slot] = make_float2(acc.m[e], acc.l[e]);
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        *reinterpret_cast<float2*>(a.part_o + slot * D + n * 8 + t4 * 2) =
            make_float2(acc.o[n][2 * e], acc.o[n][2 * e + 1]);
    }
  }
}

// Joins the partials of every (row, query head): a warp each. A lane looks up one
// partial, so their loads are in flight together, and the outputs are added with
// the weights known.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_join_kernel(const Args a, const int* __restrict__ shared_item,
                                                         const int* __restrict__ own_item, T* __restrict__ out,
                                                         long out_row, long out_head, float* __restrict__ lse) {
  constexpr int E = D / 32, U = 4;
  const int wi = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
  const int hq = a.hk * a.share;
  if (wi >= a.rows * hq) return;
  const int row = wi / hq, head = (wi % hq) / a.share, pair = row * a.share + wi % a.share;
  const int item[2] = {own_item[pair], shared_item[pair]};  // the plan's: no kernel before this one writes them
  pdl_wait();
  // Partials of either run: the first at its base slot, the others CTA by CTA.
  int count[2] = {0, 0}, c0[2], r0[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (item[s] < 0) continue;
    const Work& w = a.work[item[s] >= kBig];
    const int i = item[s] % kBig, head_tiles = w.tile0[w.n];
    const int first = w.tile0[i], n = w.tile0[i + 1] - first;
    r0[s] = pair - w.items[i].row0;
    if (n == 0) continue;
    const long total = long(head_tiles) * a.hk, t = long(head) * head_tiles + first;
    const int n_shares = shares(w.ctas, total);
    c0[s] = share_of(t, n_shares, total);
    count[s] = share_of(t + n - 1, n_shares, total) - c0[s] + 1;
  }
  float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  const int parts = count[0] + count[1];
  for (int base = 0; base < parts; base += 32) {
    float2 ml = make_float2(-INFINITY, 0.f);
    long slot = 0;
    if (base + lane < parts) {
      const int s = base + lane < count[0] ? 0 : 1, i = base + lane - (s ? count[0] : 0);
      slot = i == 0 ? base_slot(a, s, head, pair) : cta_slot(a.work[item[s] >= kBig], c0[s] + i, r0[s]);
      ml = a.part_ml[slot];
    }
    float mx = ml.x;
#pragma unroll
    for (int b = 16; b > 0; b >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, b));
    mx = fmaxf(mx, m);
    const float ref = mx == -INFINITY ? 0.f : mx;
    // A partial that saw no key adds nothing, whatever its output holds.
    const bool none = ml.x == -INFINITY && ml.y == 0.f;
    const float weight = none ? 0.f : exp2f(ml.x - ref), before = exp2f(m - ref);
    float sum = none ? 0.f : ml.y * weight;
#pragma unroll
    for (int b = 16; b > 0; b >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, b);
    l = l * before + sum;
    m = mx;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= before;
    unsigned todo = __ballot_sync(0xffffffffu, !none);
    while (todo) {
      float x[U][E], wt[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int from = todo ? __ffs(todo) - 1 : 0;
        wt[u] = __shfl_sync(0xffffffffu, weight, from);
        const float* p = a.part_o + __shfl_sync(0xffffffffu, slot, from) * D + lane * E;
        if (todo) {
          if constexpr (E == 4) {
            const float4 v = *reinterpret_cast<const float4*>(p);
            x[u][0] = v.x; x[u][1] = v.y; x[u][2] = v.z; x[u][3] = v.w;
          } else {
            const float2 v = *reinterpret_cast<const float2*>(p);
            x[u][0] = v.x; x[u][1] = v.y;
          }
        } else {
          wt[u] = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) x[u][e] = 0.f;
        }
        todo &= todo - 1;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(x[u][e], wt[u], o[e]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a NaN sum stays one
  T* dst = out + row * out_row + (wi % hq) * out_head + lane * E;
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack<T>(o[e] * inv, o[e + 1] * inv);
  if (lse && lane == 0)
    lse[long(row) * hq + wi % hq] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

CUtensorMap page_map(const torch::Tensor& t, int most_rows, const char* name) {
  const int64_t pages = t.size(0), heads = t.size(1), page = t.size(2), d = t.size(3);
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && t.stride(0) * 2 % 16 == 0, name,
              ": pages must be 16-byte aligned");
  CUtensorMap m;
  const cuuint64_t dims[3] = {cuuint64_t(d), cuuint64_t(heads * page), cuuint64_t(pages)};
  const cuuint64_t strides[2] = {cuuint64_t(d * 2), cuuint64_t((pages > 1 ? t.stride(0) : heads * page * d) * 2)};
  const cuuint32_t box[3] = {64, cuuint32_t(std::min<int64_t>(page, most_rows)), 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const auto type = t.scalar_type() == at::kHalf ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult r = encode_tiled_fn()(&m, type, 3, t.data_ptr(), dims, strides, box, estr,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, name, ": cuTensorMapEncodeTiled failed with code ", num(r));
  return m;
}

template <typename T, int D>
void launch(const torch::Tensor& k, const torch::Tensor& v, Args& a, const int* shared_item, const int* own_item,
            torch::Tensor& out, float* lse) {
  constexpr int smem = Smem<D>::kBytes;
  static const bool configured = [] {
    TORCH_CHECK(cudaFuncSetAttribute(paged_attn_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) ==
                    cudaSuccess, "paged_attention: shared memory");
    return true;
  }();
  (void)configured;
  auto stream = at::cuda::getCurrentCUDAStream();
  if (a.work[1].n)
    launch_big<T, D>(page_map(k, kBigKeys, "paged_attention: k"), page_map(v, kBigKeys, "paged_attention: v"), a,
                     stream);
  if (a.work[0].n) {
    paged_attn_kernel<T, D><<<a.work[0].ctas, kThreads, smem, stream>>>(page_map(k, TK, "paged_attention: k"),
                                                                       page_map(v, TK, "paged_attention: v"), a);
    TORCH_CHECK(cudaGetLastError() == cudaSuccess, "paged_attention launch failed");
  }
  // The joining kernel is launched early and waits for the first one's results.
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned((int64_t(a.rows) * a.hk * a.share + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  TORCH_CHECK(cudaLaunchKernelEx(&cfg, paged_join_kernel<T, D>, a, shared_item, own_item,
                                 reinterpret_cast<T*>(out.data_ptr()), long(out.stride(0)), long(out.stride(1)), lse) ==
                  cudaSuccess, "paged_attention: join launch failed");
}

}  // namespace pa

// q, out: (rows, query heads, head_dim); k, v: one layer's pages (pages, kv heads,
// rows of a page, head_dim). items, big_items: (n, 8) int32; shared_item, own_item:
// item of each (row, query head of a kv head), plus kBig for big items, -1 where
// there is none.
void paged_attention(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor table, torch::Tensor lens,
                     torch::Tensor items, torch::Tensor big_items, torch::Tensor slot_of_seq, torch::Tensor row_slot,
                     torch::Tensor row_back,                    torch::Tensor shared_item, torch::Tensor own_item, int64_t max_slot, double scale,
                     torch::Tensor out, c10::optional<torch::Tensor> lse) {
  using namespace pa;
  const auto type = q.scalar_type();
  TORCH_CHECK(q.is_cuda(), "paged_attention: q must be on a GPU");
  TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf, "paged_attention: bf16 or fp16, got ", type_name(q));
  TORCH_CHECK(q.dim() == 3 && out.sizes() == q.sizes() && out.scalar_type() == type && out.device() == q.device(),
              "paged_attention: q and out must be (rows, heads, head_dim) alike");
  const int64_t rows = q.size(0), hq = q.size(1), d = q.size(2);
  TORCH_CHECK(d == 64 || d == 128, "paged_attention: head_dim must be 64 or 128, got ", num(d));
  for (const auto* t : {&q, &out})
    TORCH_CHECK(t->stride(2) == 1 && t->stride(0) % 2 == 0 && t->stride(1) % 2 == 0 &&
                    reinterpret_cast<uintptr_t>(t->data_ptr()) % 4 == 0,
                "paged_attention: rows and heads of q and out must be 4-byte aligned, elements contiguous");
  TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes(),
              "paged_attention: pages must be (pages, kv heads, rows, head_dim)");
  for (const auto* t : {&k, &v}) {
    TORCH_CHECK(t->device() == q.device() && t->scalar_type() == type && t->size(3) == d,
                "paged_attention: pages must be of q's device, dtype and head_dim");
    TORCH_CHECK(t->stride(3) == 1 && t->stride(2) == d && t->stride(1) == d * t->size(2),
                "paged_attention: a page must be contiguous");
  }
  const int64_t hk = k.size(1), page = k.size(2);
  TORCH_CHECK(hk > 0 && hq % hk == 0, "paged_attention: ", num(hq), " query heads on ", num(hk), " kv heads");
  TORCH_CHECK(page >= 8 && (page & (page - 1)) == 0 && page <= 4096,
              "paged_attention: rows of a page must be a power of two from 8 to 4096, got ", num(page));
  for (const auto* t : {&table, &lens, &items, &big_items, &slot_of_seq, &row_slot, &row_back, &shared_item, &own_item})
    TORCH_CHECK(t->device() == q.device() && t->scalar_type() == at::kInt && t->is_contiguous(),
                "paged_attention: table, lens and the plan must be contiguous int32 on ", place(q));
  TORCH_CHECK(table.dim() == 2 && lens.dim() == 1 && table.size(0) == lens.size(0) && max_slot < table.size(0),
              "paged_attention: table and lens must have a row for each of the plan's slots");
  TORCH_CHECK(row_slot.numel() == rows, "paged_attention: the plan has ", num(row_slot.numel()),
              " rows, q has ", num(rows));
  const int64_t share = hq / hk;
  TORCH_CHECK(shared_item.numel() == rows * share, "paged_attention: the plan is for ",
              num(rows ? shared_item.numel() / rows : 0), " query heads a kv head, q has ", num(share));
  TORCH_CHECK(scale > 0, "paged_attention: scale must be positive");
  TORCH_CHECK(rows * hq <= (int64_t(1) << 30) && table.size(1) * page <= INT32_MAX, "paged_attention: sizes");
  float* lse_p = nullptr;
  if (lse.has_value()) {
    TORCH_CHECK(lse->device() == q.device() && lse->scalar_type() == at::kFloat && lse->is_contiguous() &&
                    lse->dim() == 2 && lse->size(0) == rows && lse->size(1) == hq,
                "paged_attention: lse must be contiguous fp32 (rows, heads)");
    lse_p = lse->data_ptr<float>();
  }
  if (rows == 0) return;
  const at::cuda::CUDAGuard guard(q.device());
  Args a{};
  a.q = q.data_ptr();
  a.q_row = q.stride(0);
  a.q_head = q.stride(1);
  a.table = table.data_ptr<int>();
  a.lens = lens.data_ptr<int>();
  a.width = int(table.size(1));
  a.page = int(page);
  a.pages = int(k.size(0));
  a.slot_of_seq = slot_of_seq.data_ptr<int>();
  a.row_slot = row_slot.data_ptr<int>();
  a.row_back = row_back.data_ptr<int>();
  a.rows = int(rows);
  a.share = int(share);
  a.hk = int(hk);
  a.sl2 = float(scale * 1.4426950408889634);
  a.err = error_word();
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  // Partials and the items' first tiles, from the caching allocator: calls on
  // different streams do not share them.
  int64_t slots = 2 * rows * hq, firsts = 0;
  for (int i = 0; i < 2; ++i) {
    const auto& list = i ? big_items : items;
    Work& w = a.work[i];
    w.items = reinterpret_cast<const Item*>(list.data_ptr<int>());
    w.n = int(list.size(0));
    w.ctas = i ? sms : 2 * sms;
    w.item_rows = i ? kBigRows : kItemRows;
    w.continued = slots;
    if (w.n == 0) continue;
    slots += int64_t(w.ctas) * w.item_rows;
    firsts += w.n + 1;
  }
  auto ws = torch::empty({slots * (d + 2) + firsts}, q.options().dtype(at::kFloat));
  a.part_o = ws.data_ptr<float>();
  a.part_ml = reinterpret_cast<float2*>(a.part_o + slots * d);
  a.work[0].tile0 = reinterpret_cast<int*>(a.part_ml + slots);
  a.work[1].tile0 = a.work[0].tile0 + (a.work[0].n ? a.work[0].n + 1 : 0);
  const int *si = shared_item.data_ptr<int>(), *oi = own_item.data_ptr<int>();
  if (type == at::kBFloat16 && d == 128) launch<__nv_bfloat16, 128>(k, v, a, si, oi, out, lse_p);
  else if (type == at::kBFloat16) launch<__nv_bfloat16, 64>(k, v, a, si, oi, out, lse_p);
  else if (d == 128) launch<__half, 128>(k, v, a, si, oi, out, lse_p);
  else launch<__half, 64>(k, v, a, si, oi, out, lse_p);
}

}  // namespace nk
