// Attention of new tokens over a paged KV cache, with the pages that a group of
// sequences shares read once for all of them.
//
//   out[r, hq] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q_r . k_j - max)
//
// over the keys j < limit(r) = lens[slot(r)] - back(r) of the row's sequence: the
// row sees every token up to its own. A row without keys gives 0 (LSE -inf).
//
// The work of one kv head is a list of items, made once for a plan: an item is some
// (row, query head) pairs against a run of keys, either the shared pages of a group
// (rows of all its sequences) or the rest of one sequence. The items' tiles of keys
// are numbered one after another and the workers take equal contiguous shares,
// whatever the lengths are; they are read on the device, so a captured graph follows
// them. Where a share ends inside an item, both workers leave a partial (max, sum,
// unnormalised output, fp32); a last kernel joins a row's partials from the shared
// keys and from its own.
//
// Here: items of up to 16 pairs (single tokens) on mma.sync, which is far from the
// bound for so few rows; what counts is to keep loads in flight. A warp is a worker
// of its own: it takes a share of the tiles, brings them into a two-stage ring of
// its own by TMA and keeps the running maximum and sum in registers. No warp waits
// for another, so the look-ups, first loads and write-outs of one run under the
// loads of the others on its SM. Items of more pairs: paged_attn_tc.cu.
//
// Measured (one B200): the own keys of 256 requests, 268 MB, in 58 us (4.6 TB/s); 64
// samples of one prompt of 1984 tokens, ten heads of 128, in 23 us with the join,
// where look-ups and partials, not bytes (7 us), are the time. CTAs whose four warps
// shared tiles and met at barriers took 27 us for that call's first kernel, these 21.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <climits>

#include "flash_common.cuh"
#include "launch.h"
#include "message.h"
#include "overlap.h"
#include "paged_attn.cuh"
#include "status.h"
#include "tma_host.h"

namespace nk {
namespace pa {

constexpr int kWarps = 3;   // of a CTA; two CTAs an SM by shared memory
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 2;

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
// A stage holds the K and V of TK keys, 16 KB: boxes of 32 or 64 rows by 128 bytes.
template <int D>
struct Ring {
  static constexpr int TK = 4096 / D;
  static constexpr int kSub = TK * 128;          // 64 columns of the rows, 128-byte swizzled
  static constexpr int kTile = kSub * (D / 64);  // K or V
  static constexpr int kWarp = kStages * 2 * kTile;
  static constexpr int kBytes = 1024 + kWarps * kWarp;
};

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

// Scores, softmax step and P V of 16 rows against the TK keys of a stage. lim: keys
// of the tile that each of the thread's two rows sees.
template <typename T, int D>
__device__ __forceinline__ void step(Acc<D>& acc, const uint32_t (&qf)[D / 16][4], uint32_t sK, uint32_t sV,
                                     const int (&lim)[2], float sl2) {
  constexpr int TK = Ring<D>::TK, kSub = Ring<D>::kSub;
  const int t4 = threadIdx.x & 3;
  float s[TK / 8][4];
#pragma unroll
  for (int n = 0; n < TK / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
    for (int np = 0; np < TK / 16; ++np) {
      uint32_t b[4];
      load_b_nk<64>(sK + (kk / 4) * kSub, np * 16, (kk % 4) * 16, b);
      mma<T>(s[2 * np], qf[kk], b[0], b[1]);
      mma<T>(s[2 * np + 1], qf[kk], b[2], b[3]);
    }
  const bool masked = TK > min(lim[0], lim[1]);
  float mx[2] = {acc.m[0], acc.m[1]};
#pragma unroll
  for (int n = 0; n < TK / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // A hidden score is replaced, whatever stood in its place.
      const bool hide = masked && n * 8 + t4 * 2 + (e & 1) >= lim[e >> 1];
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
  for (int n = 0; n < TK / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[n][e] = ex2_approx(s[n][e] - ref[e >> 1]);
      sum[e >> 1] += s[n][e];
    }
  acc.l[0] += sum[0];  // this thread's columns; the quad's sums meet at the end of the piece
  acc.l[1] += sum[1];
#pragma unroll
  for (int ks = 0; ks < TK / 16; ++ks) {
    // P is rounded to the values' type for the tensor core; the sum keeps fp32.
    const uint32_t p[4] = {pack<T>(s[2 * ks][0], s[2 * ks][1]), pack<T>(s[2 * ks][2], s[2 * ks][3]),
                           pack<T>(s[2 * ks + 1][0], s[2 * ks + 1][1]), pack<T>(s[2 * ks + 1][2], s[2 * ks + 1][3])};
#pragma unroll
    for (int n = 0; n < D / 16; ++n) {
      uint32_t b[4];
      load_b_kn<64>(sV + (n / 4) * kSub, (n % 4) * 16, ks * 16, b);
      mma<T>(acc.o[2 * n], p, b[0], b[1]);
      mma<T>(acc.o[2 * n + 1], p, b[2], b[3]);
    }
  }
}

// The part of an item that lies in a worker's share.
struct Piece {
  int head, units, tiles, key0, end, slot;  // end: keys of the item's run that exist
  bool continued, whole;
  Item item;
};

// The piece that begins at unit u, `left` before the share's end; by a whole warp.
template <int TK>
__device__ __forceinline__ Piece piece_at(const Args& a, const Work& w, const Deal<kThreads>& d, int head_units, int u,
                                          int left) {
  Piece p;
  p.head = u / head_units;
  int at, n;
  const int i = item_of<TK, kThreads>(a, w, d, u % head_units, at, n);
  const Span s = span_of(w, u % head_units - at, n, left);
  p.item = w.items[i];
  p.units = s.units;
  p.tiles = s.tiles;
  p.key0 = p.item.key0 + s.tile0 * TK;
  p.continued = s.tile0 > 0;
  p.whole = s.whole;
  if (p.tiles) run_end(a, p.item, p.slot, p.end);
  return p;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const Args a) {
  using R = Ring<D>;
  constexpr int TK = R::TK;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ Deal<kThreads> dealt;
  __shared__ uint64_t s_full[kWarps][kStages];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023)) +
                  warp * R::kWarp;
  uint64_t* full = s_full[warp];
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  pdl_trigger();
  const Work& work = a.work[0];
  const int head_units = deal<TK, kThreads>(a, work, dealt);
  const int total = head_units * a.hk, size = share_size(work.workers, total, work.least);
  const int worker = warp * gridDim.x + blockIdx.x;  // few shares: spread over the SMs
  const int u0 = worker * size, units = min(total - u0, size);
  if (units <= 0) {
    pdl_wait();
    return;
  }

  // The loads run ahead of the computation by the ring's stages, with a cursor of
  // their own (in, in_j); it holds the pages of up to 32 boxes of its piece, one a lane.
  const int box_rows = min(a.page, TK), boxes_of_tile = TK / box_rows;
  Piece in;
  in.tiles = 0;
  int in_j = 0, in_units = 0, loaded = 0;  // tiles loaded of the piece; units up to its end, tiles loaded of the share
  int page = 0, page_from = 0;             // boxes [page_from, page_from + 32) of the piece are in `page`
  auto look_up = [&](int box) {
    page_from = box;
    const int key = in.key0 + (box + lane) * box_rows;
    page = 0;
    if (key < in.end && box + lane < in.tiles * boxes_of_tile) {
      page = a.table[long(in.slot) * a.width + key / a.page];
      if (page < 0 || page >= a.pages) {
        atomicCAS(a.err, 0, kErrBounds);
        page = 0;
      }
    }
  };
  auto load_next = [&]() {
    while (in_j == in.tiles) {
      if (in_units == units) return;
      in = piece_at<TK>(a, work, dealt, head_units, u0 + in_units, units - in_units);
      in_units += in.units;
      in_j = 0;
      if (in.tiles) look_up(0);
    }
    const int box0 = in_j * boxes_of_tile, k0 = in.key0 + in_j * TK;
    if (box0 + boxes_of_tile > page_from + 32) look_up(box0);
    const int boxes = k0 < in.end ? (min(in.end - k0, TK) + box_rows - 1) / box_rows : 0;
    const int st = loaded % kStages;
    if (lane == 0) mbar_arrive_expect_tx(&full[st], boxes * box_rows * D * 2 * 2);
    __syncwarp();
    // One lane a box: its page comes from the lane that looked it up.
    const int pg = __shfl_sync(0xffffffffu, page, (box0 - page_from + lane) & 31);
    if (lane < boxes) {
      uint8_t* sK = ring + st * 2 * R::kTile + lane * box_rows * 128;
      const int row = in.head * a.page + (k0 + lane * box_rows) % a.page;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        tma_load_3d(sK + c * R::kSub, &tm_k, &full[st], c * 64, row, pg);
        tma_load_3d(sK + R::kTile + c * R::kSub, &tm_v, &full[st], c * 64, row, pg);
      }
    }
    ++in_j;
    ++loaded;
  };
  const int g = lane >> 2, t4 = lane & 3;
  const T* Q = static_cast<const T*>(a.q);
  Acc<D> acc;
  uint32_t qf[D / 16][4];
  int lim[2];
  auto begin = [&](const Piece& p) {
    acc.clear();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int rr = g + 8 * e;
      lim[e] = INT_MAX / 2;  // rows past the item's: computed on zeros, never written
      const T* src = nullptr;
      if (rr < p.item.rows) {
        const int row = (p.item.row0 + rr) / a.share, h = (p.item.row0 + rr) % a.share;
        lim[e] = length_of(a, a.row_slot[row]) - a.row_back[row];
        src = Q + row * a.q_row + (p.head * a.share + h) * a.q_head;
      }
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[kk][e] = src ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + t4 * 2) : 0u;
        qf[kk][e + 2] = src ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8 + t4 * 2) : 0u;
      }
    }
  };
  // The first piece is known from its first load; its Q comes while the tiles do.
  load_next();
  Piece now = in;
  int j = 0, now_units = in_units;
  if (now.tiles) begin(now);
#pragma unroll
  for (int i = 1; i < kStages; ++i) load_next();
  bool more = true;
  for (int i = 0;; ++i) {
    if (j == now.tiles) {
      do {
        if (!(more = now_units < units)) break;
        now = piece_at<TK>(a, work, dealt, head_units, u0 + now_units, units - now_units);
        now_units += now.units;
      } while (now.tiles == 0);
      if (!more) break;
      j = 0;
      begin(now);
    }
    const int st = i % kStages, k0 = now.key0 + j * TK, valid = min(TK, max(0, now.end - k0));
    if (!wait(&full[st], (i / kStages) & 1, kErrTimeoutMma, a.err)) {
      // The other stage's copies may still be on their way into this CTA's memory.
      if (loaded > i + 1) wait(&full[(i + 1) % kStages], ((i + 1) / kStages) & 1, kErrTimeoutMma, a.err);
      break;
    }
    uint8_t* tile = ring + st * 2 * R::kTile;
    if (valid < TK) {
      // Rows past the last key hold what the page or an earlier tile held, which
      // may be anything: values are cleared, so that 0 * v is 0.
      for (int c = lane; c < (TK - valid) * (D / 8); c += 32) {
        const int row = valid + c / (D / 8), ch = c % (D / 8);
        *reinterpret_cast<uint4*>(tile + R::kTile + (ch / 8) * R::kSub + row * 128 + (ch % 8) * 16) =
            make_uint4(0, 0, 0, 0);
      }
      __syncwarp();
    }
    const int see[2] = {min(lim[0] - k0, valid), min(lim[1] - k0, valid)};
    step<T, D>(acc, qf, smem_u32(tile), smem_u32(tile + R::kTile), see, a.sl2);
    if (valid < TK) fence_proxy_async();  // the clearing stores come before the next load into this stage
    __syncwarp();
    load_next();
    if (++j < now.tiles) continue;

#pragma unroll
    for (int e = 0; e < 2; ++e) {
      acc.l[e] += __shfl_xor_sync(0xffffffffu, acc.l[e], 1);
      acc.l[e] += __shfl_xor_sync(0xffffffffu, acc.l[e], 2);
      const int rr = g + 8 * e;
      if (rr >= now.item.rows) continue;
      if (now.item.alone && now.whole) {  // nothing to join
        const int row = (now.item.row0 + rr) / a.share, h = now.head * a.share + (now.item.row0 + rr) % a.share;
        const float inv = inverse(acc.l[e]);
        T* dst = static_cast<T*>(a.out) + row * a.out_row + h * a.out_head + t4 * 2;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<uint32_t*>(dst + n * 8) = pack<T>(acc.o[n][2 * e] * inv, acc.o[n][2 * e + 1] * inv);
        if (a.lse && t4 == 0) a.lse[long(row) * a.hk * a.share + h] = lse_of(acc.m[e], acc.l[e]);
        continue;
      }
      const long slot = now.continued ? continued_slot(work, worker, now.item.row0 + rr)
                                      : base_slot(a, now.item.shared, now.head, now.item.row0 + rr);
      if (t4 == 0) a.part_ml[slot] = make_float2(acc.m[e], acc.l[e]);
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        *reinterpret_cast<float2*>(a.part_o + slot * D + n * 8 + t4 * 2) =
            make_float2(acc.o[n][2 * e], acc.o[n][2 * e + 1]);
    }
  }
  pdl_wait();  // started beside the kernel of the big items: it ends, and the join begins, after that one
}

// The output of one (row, query head) from the keys that it sees and no others, key by
// key in fp32; by L lanes. The tensor cores multiply the probabilities of a tile with
// the values of all its keys, so a NaN or an infinite value of a key that other rows of
// the tile see comes out as 0 * inf = NaN in rows that do not see it. Those rows are
// done again here; no call comes here where values are finite, and no row whose runs
// hold no key that it does not see.
template <typename T, int D, int L>
__device__ __noinline__ void attend_alone(const Args& a, const int* shared_item, const int* own_item, int id) {
  const unsigned lanes = (L == 32 ? 0xffffffffu : (1u << (L % 32)) - 1) << (threadIdx.x % 32 / L * L);
  const int hq = a.hk * a.share, row = id / hq, h = id % hq, pair = row * a.share + h % a.share;
  const int slot = a.row_slot[row], len = length_of(a, slot), keys = len - a.row_back[row];
  const int own = own_item[pair], shared = shared_item[pair];
  auto item = [&](int i) -> const Item& { return (i >= kBig ? a.work[1] : a.work[0]).items[i & (kBig - 1)]; };
  if (keys >= len - item(own).keys && (shared < 0 || keys >= item(shared).key0 + item(shared).keys)) return;
  constexpr int E = D / L, U = 4, W = E < 4 ? E : 4;  // element e of a lane: as in the join
  const int c0 = threadIdx.x % L * W, head = h / a.share;
  auto load = [](const T* p, float(&x)[E]) {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 w = unpack<T>(*reinterpret_cast<const uint32_t*>(p + (e / W) * W * L + e % W));
      x[e] = w.x;
      x[e + 1] = w.y;
    }
  };
  float q[E], o[E], m = -INFINITY, l = 0.f;
  load(static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head + c0, q);
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 1
  for (int j = 0; j < keys; j += U) {
    float s[U], v[U][E], mx = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = min(j + u, keys - 1), page = a.table[long(slot) * a.width + key / a.page];
      const int pg = page < 0 || page >= a.pages ? 0 : page;  // as the other kernels, which report it
      const long at = long(head * a.page + key % a.page) * D + c0;
      float k[E];
      load(static_cast<const T*>(a.k) + pg * a.k_page + at, k);
      load(static_cast<const T*>(a.v) + pg * a.v_page + at, v[u]);
      s[u] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s[u] = fmaf(q[e], k[e], s[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int b = L / 2; b > 0; b >>= 1) s[u] += __shfl_xor_sync(lanes, s[u], b);
      s[u] *= a.sl2;
      mx = fmaxf(mx, s[u]);
    }
    const float ref = mx == -INFINITY ? 0.f : mx, alpha = exp2f(m - ref);
    m = mx;
    l *= alpha;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= alpha;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j + u >= keys) break;
      const float p = exp2f(s[u] - ref);
      l += p;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(p, v[u][e], o[e]);
    }
  }
  const float inv = inverse(l);
  T* dst = static_cast<T*>(a.out) + row * a.out_row + h * a.out_head + c0;
#pragma unroll
  for (int e = 0; e < E; e += 2)
    *reinterpret_cast<uint32_t*>(dst + (e / W) * W * L + e % W) = pack<T>(o[e] * inv, o[e + 1] * inv);
}

// Joins the partials of every (row, query head) that the kernels above left in
// several pieces: L lanes each. A lane looks up one partial, so their loads are in
// flight together, and the outputs are added with the weights known. All 32 lanes
// where there are few pairs and so many partials of each (latency counts), eight
// where there are many pairs of few partials (loads in flight count).
constexpr int kJoinThreads = 128;
// With eight lanes a pair there are many CTAs, and the registers are held at what the
// join itself needs (attend_alone, which hardly any call reaches, may spill): 99 us
// instead of 101 for a call of 33 prompts. With 32 there are few, and the bound would
// cost 1 us of 15.
template <typename T, int D, int L>
__global__ void __launch_bounds__(kJoinThreads, L == 32 ? 1 : (D == 128 ? 7 : 9))
    paged_join_kernel(const __grid_constant__ Args a, const int* __restrict__ shared_item,
                      const int* __restrict__ own_item) {
  constexpr int E = D / L, U = 4 * L / 32 + 1, W = E < 4 ? E : 4;  // W: floats of a load
  const int id = (blockIdx.x * kJoinThreads + threadIdx.x) / L, lane = threadIdx.x % L;
  const unsigned lanes = (L == 32 ? 0xffffffffu : (1u << (L % 32)) - 1) << (threadIdx.x % 32 / L * L);
  const int hq = a.hk * a.share;
  if (id >= a.rows * hq) return;  // by whole groups of lanes
  const int row = id / hq, h = id % hq, head = h / a.share, pair = row * a.share + h % a.share;
  const int item[2] = {own_item[pair], shared_item[pair]};  // the plan's: no kernel before this one writes them
  pdl_wait();
  // The output that a pair's only piece may have written, on its way with the look-ups.
  T* dst = static_cast<T*>(a.out) + row * a.out_row + h * a.out_head + lane * W;
  uint32_t* word[E / 2];
  uint32_t written[E / 2];
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    word[e / 2] = reinterpret_cast<uint32_t*>(dst + (e / W) * W * L + e % W);
    if (item[1] < 0) written[e / 2] = *word[e / 2];
  }
  // Partials of either run: the first at its base slot, the others worker by worker.
  int count[2] = {0, 0}, c0[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (item[s] < 0) continue;
    const Work& w = item[s] >= kBig ? a.work[1] : a.work[0];
    const int i = item[s] & (kBig - 1), all = w.unit0[w.n], first = w.unit0[i], n = w.unit0[i + 1] - first;
    if (n == 0) continue;
    const int size = share_size(w.workers, all * a.hk, w.least), u = head * all + first;
    c0[s] = (u + w.over) / size;
    count[s] = (u + n - 1) / size - c0[s] + 1;
  }
  const int parts = count[0] + count[1];
  bool nan = false;
  if (parts == 1 && (item[0] < 0 || item[1] < 0)) {  // its only piece wrote the output
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      const float2 x = unpack<T>(written[e]);
      nan |= isnan(x.x) || isnan(x.y);
    }
    if (__any_sync(lanes, nan)) attend_alone<T, D, L>(a, shared_item, own_item, id);
    return;
  }
  float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int base = 0; base < parts; base += L) {
    float2 ml = make_float2(-INFINITY, 0.f);
    long slot = 0;
    if (base + lane < parts) {
      const int s = base + lane < count[0] ? 0 : 1, i = base + lane - (s ? count[0] : 0);
      slot = i == 0 ? base_slot(a, s, head, pair)
                    : continued_slot(item[s] >= kBig ? a.work[1] : a.work[0], c0[s] + i, pair);
      ml = a.part_ml[slot];
    }
    float mx = ml.x;
#pragma unroll
    for (int b = L / 2; b > 0; b >>= 1) mx = fmaxf(mx, __shfl_xor_sync(lanes, mx, b));
    mx = fmaxf(mx, m);
    const float ref = mx == -INFINITY ? 0.f : mx;
    // A partial that saw no key adds nothing, whatever its output holds.
    const bool none = ml.x == -INFINITY && ml.y == 0.f;
    const float weight = none ? 0.f : exp2f(ml.x - ref), before = exp2f(m - ref);
    float sum = none ? 0.f : ml.y * weight;
#pragma unroll
    for (int b = L / 2; b > 0; b >>= 1) sum += __shfl_xor_sync(lanes, sum, b);
    l = l * before + sum;
    m = mx;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= before;
    const int n = min(L, parts - base);
    for (int i = 0; i < n; i += U) {
      float x[U][E], wt[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int from = min(i + u, n - 1);
        wt[u] = __shfl_sync(lanes, i + u < n ? weight : 0.f, from, L);
        if (i + u >= n) wt[u] = 0.f;
        const float* p = a.part_o + __shfl_sync(lanes, slot, from, L) * D + lane * W;
        if (wt[u] != 0.f) {
#pragma unroll
          for (int e = 0; e < E; e += W) {
            if constexpr (W == 4) {
              const float4 v = *reinterpret_cast<const float4*>(p + e * L);
              x[u][e] = v.x;
              x[u][e + 1] = v.y;
              x[u][e + 2] = v.z;
              x[u][e + 3] = v.w;
            } else {
              const float2 v = *reinterpret_cast<const float2*>(p + e * L);
              x[u][e] = v.x;
              x[u][e + 1] = v.y;
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) x[u][e] = 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(x[u][e], wt[u], o[e]);
    }
  }
  const float inv = inverse(l);
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    nan |= isnan(o[e]) || isnan(o[e + 1]);
    *word[e / 2] = pack<T>(o[e] * inv, o[e + 1] * inv);
  }
  if (a.lse && lane == 0) a.lse[long(row) * hq + h] = lse_of(m, l);
  if (__any_sync(lanes, nan) && !isnan(l)) attend_alone<T, D, L>(a, shared_item, own_item, id);
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
void launch(const torch::Tensor& k, const torch::Tensor& v, const Args& a, const int* shared_item,
            const int* own_item) {
  constexpr int smem = Ring<D>::kBytes, TK = Ring<D>::TK;
  static const bool configured = [] {
    TORCH_CHECK(cudaFuncSetAttribute(paged_attn_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) ==
                    cudaSuccess, "paged_attention: shared memory");
    return true;
  }();
  (void)configured;
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool big = a.work[1].n, small = a.work[0].n;
  if (big)
    launch_big<T, D>(page_map(k, kBigKeys, "paged_attention: k"), page_map(v, kBigKeys, "paged_attention: v"), a,
                     stream);
  if (small) {
    const dim3 grid(unsigned(a.work[0].workers / kWarps));
    const CUtensorMap tk = page_map(k, TK, "paged_attention: k"), tv = page_map(v, TK, "paged_attention: v");
    if (big) {  // reads nothing of the big items' kernel, so it may fill the SMs that one leaves free
      TORCH_CHECK(launch_early(paged_attn_kernel<T, D>, grid, dim3(kThreads), smem, stream, tk, tv, a) == cudaSuccess,
                  "paged_attention launch failed");
    } else {
      paged_attn_kernel<T, D><<<grid, kThreads, smem, stream>>>(tk, tv, a);
      TORCH_CHECK(cudaGetLastError() == cudaSuccess, "paged_attention launch failed");
    }
  }
  const int64_t pairs = int64_t(a.rows) * a.hk * a.share;
  const bool few = pairs <= 148 * 64;
  const int64_t per = kJoinThreads / (few ? 32 : 8);
  const auto join = few ? paged_join_kernel<T, D, 32> : paged_join_kernel<T, D, 8>;
  TORCH_CHECK(launch_early(join, dim3(unsigned((pairs + per - 1) / per)), dim3(kJoinThreads), 0, stream, a, shared_item,
                           own_item) == cudaSuccess, "paged_attention: join launch failed");
}

}  // namespace pa

// q, out: (rows, query heads, head_dim); k, v: one layer's pages (pages, kv heads,
// rows of a page, head_dim). items, big_items: (n, 8) int32; shared_item, own_item:
// item of each (row, query head of a kv head), plus kBig for big items, -1 where
// there is none. plan_page: rows of the pages that the items were made for;
// plan_keys: keys of the longest shared run.
void paged_attention(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor table, torch::Tensor lens,
                     torch::Tensor items, torch::Tensor big_items, torch::Tensor slot_of_seq, torch::Tensor row_slot,
                     torch::Tensor row_back, torch::Tensor shared_item, torch::Tensor own_item, int64_t max_slot,
                     int64_t plan_page, int64_t plan_keys, double scale, torch::Tensor out,
                     c10::optional<torch::Tensor> lse) {
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
  check_result(Operand(q, "paged_attention: q"), Operand(out, "paged_attention: out"));
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
  // Runs begin where a page of the plan does; inside one of another size a box of
  // keys would run on into the next head.
  TORCH_CHECK(page == plan_page, "paged_attention: the plan is for pages of ", num(plan_page), " rows, these have ",
              num(page));
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
  // A shared run is as long as the plan says, whatever the table holds. The room below
  // the limit is for the last worker's share, which may end past the last unit.
  const int64_t most_keys = std::max(table.size(1) * page, plan_keys);
  TORCH_CHECK(rows * hq <= (int64_t(1) << 28) && most_keys <= INT32_MAX &&
                  (items.size(0) + big_items.size(0)) * hk * (4 + most_keys / 32) <= INT32_MAX - (1 << 16),
              "paged_attention: more rows or tiles than 32-bit numbers count");
  if (lse.has_value()) {
    TORCH_CHECK(lse->device() == q.device() && lse->scalar_type() == at::kFloat && lse->is_contiguous() &&
                    lse->dim() == 2 && lse->size(0) == rows && lse->size(1) == hq,
                "paged_attention: lse must be contiguous fp32 (rows, heads)");
  }
  if (rows == 0) return;
  const at::cuda::CUDAGuard guard(q.device());
  if (out.data_ptr() == q.data_ptr()) q = q.clone();  // the join may need q again when out is written
  Args a{};
  a.q = q.data_ptr();
  a.q_row = q.stride(0);
  a.q_head = q.stride(1);
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_page = k.stride(0);
  a.v_page = v.stride(0);
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
  a.out = out.data_ptr();
  a.out_row = out.stride(0);
  a.out_head = out.stride(1);
  a.lse = lse.has_value() ? lse->data_ptr<float>() : nullptr;
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
    w.workers = i ? sms : 2 * kWarps * sms;
    w.item_rows = i ? kBigRows : kSmallRows;
    w.continued = slots;
    // Swept from 0 to 4 on calls of 4 to 300 sequences: a worker's time for a piece
    // without its tiles is that of about three tiles in both kernels (none counted: 5
    // to 25 % slower where pieces are short). Shares of fewer than four units leave
    // more to join than they save.
    w.over = 3;
    w.least = i ? 1 : 4;
    if (w.n == 0) continue;
    slots += int64_t(w.workers) * w.item_rows;
    firsts += w.n + 1;
  }
  auto ws = torch::empty({slots * (d + 2) + firsts}, q.options().dtype(at::kFloat));
  a.part_o = ws.data_ptr<float>();
  a.part_ml = reinterpret_cast<float2*>(a.part_o + slots * d);
  a.work[0].unit0 = reinterpret_cast<int*>(a.part_ml + slots);
  a.work[1].unit0 = a.work[0].unit0 + (a.work[0].n ? a.work[0].n + 1 : 0);
  const int *si = shared_item.data_ptr<int>(), *oi = own_item.data_ptr<int>();
  if (type == at::kBFloat16 && d == 128) launch<__nv_bfloat16, 128>(k, v, a, si, oi);
  else if (type == at::kBFloat16) launch<__nv_bfloat16, 64>(k, v, a, si, oi);
  else if (d == 128) launch<__half, 128>(k, v, a, si, oi);
  else launch<__half, 64>(k, v, a, si, oi);
}

}  // namespace nk
