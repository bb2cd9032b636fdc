// Paged attention, items of many rows (prompts of many tokens, or many single
// tokens behind one prefix): the same sums as paged_attn.cu on the 5th-generation
// tensor cores.
//
// One CTA an SM takes an equal share of all items' units and walks
// it piece by piece (a piece: the part of an item that lies in its share). An item
// is up to 256 (row, query head) pairs: two tiles of 128, so that one tile's MMAs
// run under the other's softmax. Tensor memory holds S0, S1 and O0, O1. Roles:
//   warp 0      finds the pieces, writes their records, loads K and V: a lane a page
//   warp 1      issues the MMAs, S_t = Q_t K^T and O_t += P_t V (P_t in tensor
//               memory over the columns of S_t)
//   warps 2-9   softmax of tile 0, warps 10-17 of tile 1. Two threads have a row, each
//               half of the tile's keys; they exchange their maxima by shared memory.
//               (Exponentials are the bound; two warps a tile and scheduler hide each
//               other's loads and barriers.) They bring their row of Q to shared memory
//               at the start of a piece and write its partial at the end. O is rescaled
//               only when a row's maximum grew by 2^8 or more since the last time; the
//               stale maximum scales P and O alike.
// Keys past the end of an item's run are hidden by the mask; their values are
// cleared in shared memory first, since 0 * NaN is not 0. Rows that a NaN of a key
// which only other rows see has reached are done again by the join (paged_attn.cu).
//
// Measured (one B200): 1024 rows against 32768 keys on 4 kv heads of 128 (69 GFLOP) in
// 81 us, 849 TFLOP/s; a tile of 256 rows and 128 keys takes about 3600 cycles, of which
// the MMAs need 2048 and the exponentials as many: what is left is the way between the
// two (scores ready, maximum, P stored, MMA issued), which two tiles do not quite hide.
#include <ATen/cuda/CUDAContext.h>
#include <torch/extension.h>

#include <climits>
#include <type_traits>

#include "paged_attn.cuh"
#include "status.h"

namespace nk {
namespace pa {

namespace {

constexpr int kThreads = 576;
constexpr int kSoftWarps = 8;  // of one tile
constexpr int kPieces = 8;  // records; the producer is at most five pieces ahead of the slowest role
constexpr float kRescale = 8.f;

struct Piece {
  int row0, rows, head, shared;
  int key0, tiles;   // first key and tiles of the piece (none: it ends the share)
  int end;           // keys of the item's run that exist
  int continued;
  int final;         // nothing to join: the piece writes the output
};

template <int D>
struct Big {
  static constexpr int kSub = 128 * 128;            // 64 columns of 128 rows, 128-byte swizzled
  static constexpr int kTile = kSub * (D / 64);     // Q, K or V tile
  static constexpr int kSmem = 1024 + 6 * kTile;    // Q0, Q1, two K, two V
};

// One lane of a warp that is whole, and a value that is the same in all its lanes:
// in forms that the compiler knows as such.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return reinterpret_cast<float2&>(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return reinterpret_cast<float2&>(d);
}

// bf16 operands have format 1 in bits 7 and 10 of the descriptor, fp16 format 0.
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int m, int n, bool b_mn) {
  return idesc_bf16(m, n, false, b_mn) & (std::is_same<T, __half>::value ? ~((1u << 7) | (1u << 10)) : ~0u);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    paged_attn_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                         const Args a) {
  using S = Big<D>;
  constexpr int BK = kBigKeys;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem, *sK = smem + 2 * S::kTile, *sV = smem + 4 * S::kTile;
  __shared__ Deal<kThreads> dealt;
  __shared__ Piece pieces[kPieces];
  __shared__ uint64_t piece_full[kPieces], q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], v_clear, s_full[2],
      p_full[2], o_done[2], both[2][4];  // both: the two warps that share 32 rows
  __shared__ float s_row[2][2][2][128];  // exchanged between a row's threads: [parity][tile][half][row]
  __shared__ uint32_t tmem_slot;
  const int warp = uniform(threadIdx.x / 32), lane = threadIdx.x % 32;
  const Work& w = a.work[1];
  if (threadIdx.x == 0) {
    for (int i = 0; i < kPieces; ++i) mbar_init(&piece_full[i], 1);
    mbar_init(&q_full, 2 * kSoftWarps);
    mbar_init(&v_clear, kSoftWarps);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kSoftWarps);
      for (int q = 0; q < 4; ++q) mbar_init(&both[i][q], 2);
      mbar_init(&o_done[i], 1);
    }
    fence_barrier_init();
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  if (warp == 1) tmem_alloc(&tmem_slot, 512);
  pdl_trigger();
  const int head_units = deal<BK, kThreads>(a, w, dealt);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(tmem_slot);  // S0 @0, S1 @128, O0 @256, O1 @256 + D
  const int total = head_units * a.hk, size = share_size(w.workers, total, w.least);
  const int u_begin = blockIdx.x * size, n_units = uniform(min(total - u_begin, size));  // none: n_units <= 0

  if (warp == 0) {
    const int box_rows = min(a.page, BK);
    int it = 0, units = 0, p = 0;  // tiles loaded, units up to the end of the piece found last, pieces
    bool ok = true;
    Piece pc;
    int slot = 0;
    // Finds the share's next piece with tiles and leaves its record; after the last
    // one, a record without.
    auto find = [&]() {
      pc = Piece{};
      while (pc.tiles == 0 && units < n_units) {
        const int u = u_begin + units;
        int at, n;
        const int i = item_of<BK, kThreads>(a, w, dealt, u % head_units, at, n);
        const Item item = w.items[i];
        const Span s = span_of(w, u % head_units - at, n, n_units - units);
        units += s.units;
        if (s.tiles == 0) continue;
        int end;
        run_end(a, item, slot, end);
        pc = Piece{item.row0, item.rows, u / head_units, item.shared, item.key0 + s.tile0 * BK, s.tiles, end,
                   s.tile0 > 0, item.alone && s.whole};
      }
      if (lane == 0) {
        pieces[p % kPieces] = pc;
        mbar_arrive(&piece_full[p % kPieces]);
      }
      ++p;
    };
    find();
    while (pc.tiles && ok) {
      const int key0 = pc.key0, tiles = pc.tiles, head = pc.head, end = pc.end, row_slot = slot;
      auto page_of = [&](int j) {  // of this lane's box of tile j of the piece
        const int key = key0 + j * BK + lane * box_rows;
        if (lane * box_rows >= BK || key >= end || j >= tiles) return 0;
        int page = a.table[long(row_slot) * a.width + key / a.page];
        if (page < 0 || page >= a.pages) {
          atomicCAS(a.err, 0, kErrBounds);
          page = 0;
        }
        return page;
      };
      int page = page_of(0);
      for (int j = 0; j < tiles && ok; ++j, ++it) {
        const int next = page_of(j + 1);  // on its way while this tile waits for room
        const int b = it & 1, k0 = key0 + j * BK;
        const int boxes = k0 < end ? (min(end - k0, BK) + box_rows - 1) / box_rows : 0;
        const int row = head * a.page + (k0 + lane * box_rows) % a.page;
        ok = wait(&k_empty[b], ((it >> 1) & 1) ^ 1, kErrTimeoutProducer, a.err);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&k_full[b], boxes * box_rows * D * 2);
        __syncwarp();
        if (lane < boxes)
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_load_3d(sK + b * S::kTile + c * S::kSub + lane * box_rows * 128, &tm_k, &k_full[b], c * 64, row, page);
        ok = wait(&v_empty[b], ((it >> 1) & 1) ^ 1, kErrTimeoutProducer, a.err);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&v_full[b], boxes * box_rows * D * 2);
        __syncwarp();
        if (lane < boxes)
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_load_3d(sV + b * S::kTile + c * S::kSub + lane * box_rows * 128, &tm_v, &v_full[b], c * 64, row, page);
        page = next;
        // The next piece is found while this one's tiles are at work.
        if (j == min(1, tiles - 1)) find();
      }
    }
    // After a wait that ran out: copies may still be on their way into this CTA's memory.
    for (int x = max(0, it - 2); !ok && x <= it; ++x) {
      wait(&k_full[x & 1], (x >> 1) & 1, kErrTimeoutProducer, a.err);
      wait(&v_full[x & 1], (x >> 1) & 1, kErrTimeoutProducer, a.err);
    }
  } else if (warp == 1) {
    // The whole warp walks the loop and one lane issues: descriptors and phases stay
    // in uniform registers, which the MMA instruction reads. With the loop itself
    // on one lane every operand was moved there first, 80 cycles an MMA, and the
    // issue was the bound.
    constexpr uint32_t id_s = idesc<T>(128, BK, false), id_o = idesc<T>(128, D, true);
    const bool leader = elect_one();
    const uint64_t d_q = sw128_desc(smem_u32(sQ), 16, 1024), d_k = sw128_desc(smem_u32(sK), 16, 1024),
                   d_v = sw128_desc(smem_u32(sV), S::kSub, 1024);
    uint32_t c_p0 = 0, c_p1 = 0, c_clear = 0;  // phases of p_full and v_clear
    int it = 0;
    bool ok = true;
    auto issue_s = [&](int t, int b) {
      const uint64_t q = desc_advance(d_q, t * S::kTile), k = desc_advance(d_k, b * S::kTile);
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * S::kSub + (kk & 3) * 32;
          umma_bf16(tmem + t * BK, desc_advance(q, off), desc_advance(k, off), id_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[t]);
      }
      __syncwarp();
    };
    auto issue_pv = [&](int t, int b, bool first) {
      const uint64_t v = desc_advance(d_v, b * S::kTile);
      const uint32_t more = first ? 0u : 1u;
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk)
          umma_bf16_ts(tmem + 256 + t * D, tmem + t * BK + 8 * kk, desc_advance(v, kk * 2048), id_o,
                       kk > 0 ? 1u : more);
        umma_commit(&o_done[t]);
      }
      __syncwarp();
    };
    auto release = [&](uint64_t* bar) {
      if (leader) umma_commit(bar);
      __syncwarp();
    };
    for (int p = 0; ok; ++p) {
      if (!(ok = wait(&piece_full[p % kPieces], (p / kPieces) & 1, kErrTimeoutMma, a.err))) break;
      const int rows = uniform(pieces[p % kPieces].rows), tiles = uniform(pieces[p % kPieces].tiles);
      if (tiles == 0) break;
      const int keys = uniform(pieces[p % kPieces].end - pieces[p % kPieces].key0);
      const bool two = rows > 128;
      if (!(ok = wait(&q_full, p & 1, kErrTimeoutMma, a.err))) break;
      if (!(ok = wait(&k_full[it & 1], (it >> 1) & 1, kErrTimeoutMma, a.err))) break;
      tc_fence_after();
      issue_s(0, it & 1);
      if (two) issue_s(1, it & 1);
      release(&k_empty[it & 1]);
      for (int j = 0; j < tiles; ++j, ++it) {
        const bool next = j + 1 < tiles;
        const int b = it & 1, nb = b ^ 1;
        if (!(ok = wait(&v_full[b], (it >> 1) & 1, kErrTimeoutMma, a.err))) break;
        if (keys - j * BK < BK) {
          if (!(ok = wait(&v_clear, c_clear, kErrTimeoutMma, a.err))) break;
          c_clear ^= 1;
        }
        if (!(ok = wait(&p_full[0], c_p0, kErrTimeoutMma, a.err))) break;
        c_p0 ^= 1;
        tc_fence_after();
        issue_pv(0, b, j == 0);
        if (next) {
          if (!(ok = wait(&k_full[nb], ((it + 1) >> 1) & 1, kErrTimeoutMma, a.err))) break;
          tc_fence_after();
          issue_s(0, nb);
        }
        if (two) {
          if (!(ok = wait(&p_full[1], c_p1, kErrTimeoutMma, a.err))) break;
          c_p1 ^= 1;
          tc_fence_after();
          issue_pv(1, b, j == 0);
        }
        release(&v_empty[b]);
        if (next) {
          if (two) issue_s(1, nb);
          release(&k_empty[nb]);
        }
      }
    }
  } else {
    constexpr int HK = BK / 2, HD = D / 2;  // of a thread: keys of a tile, columns of O
    const int t = (warp - 2) / kSoftWarps, half = (warp - 2) / 4 % 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const uint32_t t_s = tmem + lanes + t * BK, t_o = tmem + lanes + 256 + t * D + half * HD;
    uint32_t c_s = 0, c_o = 0, c_b = 0;  // phases of s_full, o_done and both
    int it = 0;
    bool ok = true;
    // The other thread's value of this row.
    auto exchange = [&](float x, float& other) {
      float(&slot)[2][128] = s_row[c_b][t];
      slot[half][r] = x;
      __syncwarp();
      if (lane == 0) mbar_arrive(&both[t][quarter]);
      const bool done = wait(&both[t][quarter], c_b, kErrTimeoutEpilogue, a.err);
      c_b ^= 1;
      other = slot[half ^ 1][r];
      return done;
    };
    for (int p = 0; ok; ++p) {
      if (!wait(&piece_full[p % kPieces], (p / kPieces) & 1, kErrTimeoutEpilogue, a.err)) break;
      const Piece pc = pieces[p % kPieces];
      if (pc.tiles == 0) break;
      const int pair = pc.row0 + t * 128 + r;
      const bool active = pc.rows > t * 128, mine = t * 128 + r < pc.rows;
      int lim = INT_MAX / 2;  // rows past the item's: computed on zeros, never written
      if (active) {
        const T* src = nullptr;
        if (mine) {
          const int row = pair / a.share, h = pair % a.share;
          lim = length_of(a, a.row_slot[row]) - a.row_back[row];
          src = static_cast<const T*>(a.q) + row * a.q_row + (pc.head * a.share + h) * a.q_head;
        }
        // Chunk c of row r lies at c ^ (r & 7), the swizzle that the tensor core reads.
        // All of the row's loads are issued before the first store waits for one.
        const int c0 = half * (HD / 8);
        uint4 x[HD / 8];
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) x[i] = make_uint4(0, 0, 0, 0);
        if (mine && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) x[i] = reinterpret_cast<const uint4*>(src)[c0 + i];
        } else if (mine) {
          const uint32_t* s = reinterpret_cast<const uint32_t*>(src) + c0 * 4;
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) x[i] = make_uint4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
        }
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
          const int c = c0 + i;
          uint8_t* sub = sQ + t * S::kTile + (c / 8) * S::kSub;
          *reinterpret_cast<uint4*>(sub + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = x[i];
        }
        fence_proxy_async();
      }
      // All warps arrive for every piece, each once the last piece's arrivals are
      // complete: nobody is counted twice and nobody falls a piece behind.
      if (p > 0 && !wait(&q_full, (p - 1) & 1, kErrTimeoutEpilogue, a.err)) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
      if (!active) {
        it += pc.tiles;
        continue;
      }
      float m_used = -INFINITY, l = 0.f;  // l: of this thread's keys
      for (int j = 0; j < pc.tiles && ok; ++j, ++it) {
        const int k0 = pc.key0 + j * BK, valid = pc.end - k0;
        if (t == 0 && valid < BK) {
          // Thread = key: clear the values of keys that do not exist.
          if (!(ok = wait(&v_full[it & 1], (it >> 1) & 1, kErrTimeoutEpilogue, a.err))) break;
          if (r >= valid)
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
              const int c = half * (HD / 8) + i;
              *reinterpret_cast<uint4*>(sV + (it & 1) * S::kTile + (c / 8) * S::kSub + r * 128 + (c & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
            }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_clear);
        }
        if (!(ok = wait(&s_full[t], c_s, kErrTimeoutEpilogue, a.err))) break;
        c_s ^= 1;
        tc_fence_after();
        float2 sv[HK / 2];
        tmem_ld_32x64(t_s + half * HK, *reinterpret_cast<float(*)[64]>(sv));
        const int see = min(lim - k0, valid) - half * HK;
        if (__any_sync(0xffffffffu, see < HK)) {
#pragma unroll
          for (int i = 0; i < HK / 2; ++i) {
            if (2 * i >= see) sv[i].x = -INFINITY;
            if (2 * i + 1 >= see) sv[i].y = -INFINITY;
          }
        }
        float mx4[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) mx4[k] = fmaxf(sv[k].x, sv[k].y);
#pragma unroll
        for (int i = 4; i < HK / 2; i += 4)
#pragma unroll
          for (int k = 0; k < 4; ++k) mx4[k] = fmaxf(mx4[k], fmaxf(sv[i + k].x, sv[i + k].y));
        float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), mx_other;
        // Both threads have read their scores once this is done, so either may store P over them.
        tc_fence_before();
        if (!(ok = exchange(mx, mx_other))) break;
        tc_fence_after();
        mx = a.sl2 * fmaxf(mx, mx_other);
        const bool grow = mx > m_used + kRescale || (m_used == -INFINITY && mx > -INFINITY);
        // The P V before this one must be done before P is rewritten or O rescaled.
        if (j > 0) {
          if (!(ok = wait(&o_done[t], c_o, kErrTimeoutEpilogue, a.err))) break;
          c_o ^= 1;
          tc_fence_after();
        }
        if (__any_sync(0xffffffffu, grow)) {
          const float m_new = grow ? mx : m_used;
          const float alpha = grow ? ex2_approx(m_used - m_new) : 1.f;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < HD / 16; ++c) {
              uint32_t o[16];
              tmem_ld_32x16_issue(t_o + c * 16, o);
              tmem_ld_wait16(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_32x16(t_o + c * 16, o);
            }
          }
          l *= alpha;
          m_used = m_new;
        }
        const float ref = m_used == -INFINITY ? 0.f : m_used;  // a row that has seen no key yet
        const float2 scale2 = make_float2(a.sl2, a.sl2), ref2 = make_float2(-ref, -ref);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < HK / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 x = fma2(sv[c * 16 + i], scale2, ref2);
            const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
            sum[i & 1] = add2(sum[i & 1], e);
            // P is rounded to the values' type for the tensor core; the sum keeps fp32.
            pk[i] = pack<T>(e.x, e.y);
          }
          tmem_st_32x16_issue(t_s + half * (HK / 2) + 16 * c, pk);
        }
        sum[0] = add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      float l_other;
      if (!ok || !exchange(l, l_other) || !wait(&o_done[t], c_o, kErrTimeoutEpilogue, a.err)) break;
      c_o ^= 1;
      l += l_other;
      tc_fence_after();
      // A warp's 32 rows go out through its own part of the Q tile (which no MMA
      // reads any more), C columns at a time: written a row a thread, read as runs of
      // a row, so that the stores to memory are whole lines. Row by row from the
      // registers, a piece's write-out took 6 us.
      constexpr int C = D / 4, V = C / 4;  // V: 16-byte vectors of a row's run
      uint8_t* stage = sQ + t * S::kTile + (D == 128 ? half * S::kSub + quarter * 4096 : quarter * 4096 + half * 2048);
      const float inv = inverse(l);
      const int hq = a.hk * a.share;
      if (mine && half == 0) {
        if (!pc.final)
          a.part_ml[pc.continued ? continued_slot(w, blockIdx.x, pair) : base_slot(a, pc.shared, pc.head, pair)] =
              make_float2(m_used, l);
        else if (a.lse)
          a.lse[long(pair / a.share) * hq + pc.head * a.share + pair % a.share] = lse_of(m_used, l);
      }
#pragma unroll 1
      for (int c = 0; c < HD / C; ++c) {
#pragma unroll
        for (int e = 0; e < C / 16; ++e) {
          uint32_t o[16];
          tmem_ld_32x16_issue(t_o + c * C + e * 16, o);
          tmem_ld_wait16(o);
          const float f = pc.final ? inv : 1.f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4*>(stage + lane * (C * 4) + (((e * 4 + i) ^ (lane % V)) << 4)) =
                make_float4(__uint_as_float(o[4 * i]) * f, __uint_as_float(o[4 * i + 1]) * f,
                            __uint_as_float(o[4 * i + 2]) * f, __uint_as_float(o[4 * i + 3]) * f);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int rr = i * (32 / V) + lane / V, v = lane % V;  // row of the warp, vector of its run
          const int row_of = t * 128 + quarter * 32 + rr, pr = pc.row0 + row_of, col = half * HD + c * C + v * 4;
          if (row_of >= pc.rows) continue;
          const float4 x = *reinterpret_cast<const float4*>(stage + rr * (C * 4) + ((v ^ (rr % V)) << 4));
          if (pc.final) {
            T* dst = static_cast<T*>(a.out) + (pr / a.share) * a.out_row +
                     (pc.head * a.share + pr % a.share) * a.out_head + col;
            reinterpret_cast<uint32_t*>(dst)[0] = pack<T>(x.x, x.y);
            reinterpret_cast<uint32_t*>(dst)[1] = pack<T>(x.z, x.w);
          } else {
            const long slot = pc.continued ? continued_slot(w, blockIdx.x, pr) : base_slot(a, pc.shared, pc.head, pr);
            *reinterpret_cast<float4*>(a.part_o + slot * D + col) = x;
          }
        }
        __syncwarp();
      }
      // The other warp of these rows has left the Q tile's part, too, before either
      // brings new rows of Q there.
      if (!(ok = exchange(0.f, l_other))) break;
      tc_fence_before();  // O is read before the next piece's first P V overwrites it
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

template <typename T, int D>
void launch_big(const CUtensorMap& k, const CUtensorMap& v, const Args& a, cudaStream_t stream) {
  constexpr int smem = Big<D>::kSmem;
  static const bool configured = [] {
    TORCH_CHECK(cudaFuncSetAttribute(paged_attn_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) ==
                    cudaSuccess, "paged_attention: shared memory");
    return true;
  }();
  (void)configured;
  paged_attn_tc_kernel<T, D><<<a.work[1].workers, kThreads, smem, stream>>>(k, v, a);
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "paged_attention launch failed");
}

template void launch_big<__nv_bfloat16, 64>(const CUtensorMap&, const CUtensorMap&, const Args&, cudaStream_t);
template void launch_big<__nv_bfloat16, 128>(const CUtensorMap&, const CUtensorMap&, const Args&, cudaStream_t);
template void launch_big<__half, 64>(const CUtensorMap&, const CUtensorMap&, const Args&, cudaStream_t);
template void launch_big<__half, 128>(const CUtensorMap&, const CUtensorMap&, const Args&, cudaStream_t);

}  // namespace pa
}  // namespace nk
