// Paged attention, items of many rows (prompts of many tokens, or many single
// tokens behind one prefix): the same sums as paged_attn.cu on the 5th-generation
// tensor cores.
//
// One CTA an SM takes an equal share of all (item, 128-key tile) numbers and walks
// it piece by piece (a piece: the part of an item that lies in its share). An item
// is up to 256 (row, query head) pairs: two tiles of 128, so that one tile's MMAs
// run under the other's softmax. Tensor memory holds S0, S1 and O0, O1. Roles:
//   warp 0      finds the pieces, writes their records, loads K and V: a lane a page
//   warp 1      issues the MMAs, S_t = Q_t K^T and O_t += P_t V (P_t in tensor
//               memory over the columns of S_t)
//   warps 2-5   softmax of tile 0, warps 6-9 of tile 1: thread = row. They bring
//               their row of Q to shared memory at the start of a piece and write its
//               partial at the end. O is rescaled only when a row's maximum grew by
//               2^8 or more since the last time; the stale maximum scales P and O alike.
// Keys past the end of an item's run are hidden by the mask; their values are
// cleared in shared memory first, since 0 * NaN is not 0.
#include <ATen/cuda/CUDAContext.h>
#include <torch/extension.h>

#include <climits>
#include <type_traits>

#include "paged_attn.cuh"
#include "status.h"

namespace nk {
namespace pa {

namespace {

constexpr int kThreads = 320;
constexpr int kPieces = 8;  // records; the producer is at most four pieces ahead of the slowest role
constexpr float kRescale = 8.f;

struct Piece {
  int row0, rows, head, shared;
  int key0, tiles;   // first key and tiles of the piece
  int end;           // keys of the item's run that exist
  int continued;
};

template <int D>
struct Big {
  static constexpr int kSub = 128 * 128;            // 64 columns of 128 rows, 128-byte swizzled
  static constexpr int kTile = kSub * (D / 64);     // Q, K or V tile
  static constexpr int kSmem = 1024 + 6 * kTile;    // Q0, Q1, two K, two V
};

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
  __shared__ int s_sum[kThreads + 1];
  __shared__ Piece pieces[kPieces];
  __shared__ uint64_t piece_full[kPieces], q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], v_clear, s_full[2],
      p_full[2], o_done[2];
  __shared__ uint32_t tmem_slot;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const Work& w = a.work[1];
  if (threadIdx.x == 0) {
    for (int i = 0; i < kPieces; ++i) mbar_init(&piece_full[i], 1);
    mbar_init(&q_full, 8);
    mbar_init(&v_clear, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    fence_barrier_init();
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  if (warp == 1) tmem_alloc(&tmem_slot, 512);
  const int head_tiles = deal<BK, kThreads>(a, w, s_sum);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;  // S0 @0, S1 @128, O0 @256, O1 @256 + D
  const long total = long(head_tiles) * a.hk;
  const int n_shares = shares(w.ctas, total);
  const bool busy = int(blockIdx.x) < n_shares;
  const long t_begin = busy ? share_begin(blockIdx.x, n_shares, total) : 0;
  const int n_tiles = busy ? int(share_begin(blockIdx.x + 1, n_shares, total) - t_begin) : 0;

  if (warp == 0) {
    const int box_rows = min(a.page, BK);
    int it = 0;  // tiles loaded
    bool ok = true;
    for (int p = 0; it < n_tiles && ok; ++p) {
      const long t = t_begin + it;
      int at, n;
      const int tt = int(t % head_tiles);
      const int i = item_of<BK, kThreads>(a, w, s_sum, tt, at, n);
      const Item item = w.items[i];
      int slot = item.first, end;
      if (item.shared) {
        // Read through the first sequence that holds all of the shared tokens, else
        // through the longest (idle slots hold none).
        int best = -1;
        for (int s = item.first; s < item.first + item.count && best < item.key0 + item.keys; s += 32) {
          const bool there = s + lane < item.first + item.count;
          const int c = there ? a.slot_of_seq[s + lane] : 0, len = there ? length_of(a, c) : -1;
          const unsigned full = __ballot_sync(0xffffffffu, len >= item.key0 + item.keys);
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
        end = min(best, item.key0 + item.keys);
      } else {
        end = length_of(a, slot) - item.keys;
      }
      const int tiles = min(n - (tt - at), n_tiles - it), key0 = item.key0 + (tt - at) * BK, head = int(t / head_tiles);
      if (lane == 0) {
        pieces[p % kPieces] = Piece{item.row0, item.rows, head, item.shared, key0, tiles, end, tt != at};
        mbar_arrive(&piece_full[p % kPieces]);
      }
      auto page_of = [&](int j) {  // of this lane's box of tile j of the piece
        const int key = key0 + j * BK + lane * box_rows;
        if (lane * box_rows >= BK || key >= end || j >= tiles) return 0;
        int page = a.table[long(slot) * a.width + key / a.page];
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
        ok = mbar_wait(&k_empty[b], ((it >> 1) & 1) ^ 1, kErrTimeoutProducer, a.err);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) mbar_arrive_expect_tx(&k_full[b], boxes * box_rows * D * 2);
        __syncwarp();
        if (lane < boxes)
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_load_3d(sK + b * S::kTile + c * S::kSub + lane * box_rows * 128, &tm_k, &k_full[b], c * 64, row, page);
        ok = mbar_wait(&v_empty[b], ((it >> 1) & 1) ^ 1, kErrTimeoutProducer, a.err);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) mbar_arrive_expect_tx(&v_full[b], boxes * box_rows * D * 2);
        __syncwarp();
        if (lane < boxes)
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_load_3d(sV + b * S::kTile + c * S::kSub + lane * box_rows * 128, &tm_v, &v_full[b], c * 64, row, page);
        page = next;
      }
      ok = __all_sync(0xffffffffu, ok);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t id_s = idesc<T>(128, BK, false), id_o = idesc<T>(128, D, true);
      uint32_t c_p[2] = {0, 0}, c_clear = 0;  // phases of p_full and v_clear
      int it = 0;
      bool ok = true;
      auto issue_s = [&](int t, int b) {
        const uint32_t q = smem_u32(sQ + t * S::kTile), k = smem_u32(sK + b * S::kTile);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * S::kSub + (kk & 3) * 32;
          umma_bf16(tmem + t * BK, sw128_desc(q + off, 16, 1024), sw128_desc(k + off, 16, 1024), id_s,
                    kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[t]);
      };
      auto issue_pv = [&](int t, int b, bool first) {
        const uint32_t v = smem_u32(sV + b * S::kTile);
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk)
          umma_bf16_ts(tmem + 256 + t * D, tmem + t * BK + 8 * kk, sw128_desc(v + kk * 2048, S::kSub, 1024), id_o,
                       (!first || kk > 0) ? 1u : 0u);
        umma_commit(&o_done[t]);
      };
      auto wait_p = [&](int t) {
        const bool r = mbar_wait(&p_full[t], c_p[t], kErrTimeoutMma, a.err);
        c_p[t] ^= 1;
        tc_fence_after();
        return r;
      };
      for (int p = 0; it < n_tiles && ok; ++p) {
        if (!mbar_wait(&piece_full[p % kPieces], (p / kPieces) & 1, kErrTimeoutMma, a.err)) break;
        const Piece pc = pieces[p % kPieces];
        const bool two = pc.rows > 128;
        if (!mbar_wait(&q_full, p & 1, kErrTimeoutMma, a.err)) break;
        if (!mbar_wait(&k_full[it & 1], (it >> 1) & 1, kErrTimeoutMma, a.err)) break;
        tc_fence_after();
        issue_s(0, it & 1);
        if (two) issue_s(1, it & 1);
        umma_commit(&k_empty[it & 1]);
        for (int j = 0; j < pc.tiles && ok; ++j, ++it) {
          const bool next = j + 1 < pc.tiles;
          const int b = it & 1, nb = b ^ 1;
          ok = mbar_wait(&v_full[b], (it >> 1) & 1, kErrTimeoutMma, a.err);
          if (pc.end - pc.key0 - j * BK < BK && ok) {
            ok = mbar_wait(&v_clear, c_clear, kErrTimeoutMma, a.err);
            c_clear ^= 1;
          }
          if (!ok || !(ok = wait_p(0))) break;
          issue_pv(0, b, j == 0);
          if (next) {
            if (!(ok = mbar_wait(&k_full[nb], ((it + 1) >> 1) & 1, kErrTimeoutMma, a.err))) break;
            tc_fence_after();
            issue_s(0, nb);
          }
          if (two) {
            if (!(ok = wait_p(1))) break;
            issue_pv(1, b, j == 0);
          }
          umma_commit(&v_empty[b]);
          if (next) {
            if (two) issue_s(1, nb);
            umma_commit(&k_empty[nb]);
          }
        }
      }
    }
  } else {
    const int t = (warp - 2) / 4, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const uint32_t t_s = tmem + lanes + t * BK, t_o = tmem + lanes + 256 + t * D;
    uint32_t c_s = 0, c_o = 0;  // phases of s_full and o_done
    int it = 0;
    bool ok = true;
    for (int p = 0; it < n_tiles && ok; ++p) {
      if (!mbar_wait(&piece_full[p % kPieces], (p / kPieces) & 1, kErrTimeoutEpilogue, a.err)) break;
      const Piece pc = pieces[p % kPieces];
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
        const bool wide = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (mine && wide) {
            x = *reinterpret_cast<const uint4*>(src + c * 8);
          } else if (mine) {
            const uint32_t* s = reinterpret_cast<const uint32_t*>(src + c * 8);
            x = make_uint4(s[0], s[1], s[2], s[3]);
          }
          *reinterpret_cast<uint4*>(sQ + t * S::kTile + (c / 8) * S::kSub + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = x;
        }
        fence_proxy_async();
      }
      // All eight warps arrive for every piece, each once the last piece's arrivals
      // are complete: nobody is counted twice and nobody falls a piece behind.
      if (p > 0 && !mbar_wait(&q_full, (p - 1) & 1, kErrTimeoutEpilogue, a.err)) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
      if (!active) {
        it += pc.tiles;
        continue;
      }
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < pc.tiles && ok; ++j, ++it) {
        const int k0 = pc.key0 + j * BK, valid = pc.end - k0;
        if (t == 0 && valid < BK) {
          // Thread = key: clear the values of keys that do not exist.
          if (!(ok = mbar_wait(&v_full[it & 1], (it >> 1) & 1, kErrTimeoutEpilogue, a.err))) break;
          if (r >= valid)
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
              *reinterpret_cast<uint4*>(sV + (it & 1) * S::kTile + (c / 8) * S::kSub + r * 128 + (c & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_clear);
        }
        if (!(ok = mbar_wait(&s_full[t], c_s, kErrTimeoutEpilogue, a.err))) break;
        c_s ^= 1;
        tc_fence_after();
        float sv[BK];
        tmem_ld_32x64(t_s, *reinterpret_cast<float(*)[64]>(sv));
        tmem_ld_32x64(t_s + 64, *reinterpret_cast<float(*)[64]>(sv + 64));
        const int see = min(lim - k0, valid);
        if (__any_sync(0xffffffffu, see < BK)) {
#pragma unroll
          for (int i = 0; i < BK; ++i)
            if (i >= see) sv[i] = -INFINITY;
        }
        float mx8[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) mx8[k] = sv[k];
#pragma unroll
        for (int i = 8; i < BK; i += 8)
#pragma unroll
          for (int k = 0; k < 8; ++k) mx8[k] = fmaxf(mx8[k], sv[i + k]);
        const float mx = a.sl2 * fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])),
                                       fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
        // The P V before this one must be done before P is rewritten or O rescaled.
        if (j > 0) {
          if (!(ok = mbar_wait(&o_done[t], c_o, kErrTimeoutEpilogue, a.err))) break;
          c_o ^= 1;
          tc_fence_after();
        }
        const bool grow = mx > m_used + kRescale || (m_used == -INFINITY && mx > -INFINITY);
        if (__any_sync(0xffffffffu, grow)) {
          const float m_new = grow ? mx : m_used;
          const float alpha = grow ? ex2_approx(m_used - m_new) : 1.f;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
              tmem_ld_32x32(t_o + c * 32, o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= alpha;
              tmem_st_32x32(t_o + c * 32, o);
            }
          }
          l *= alpha;
          m_used = m_new;
        }
        const float ref = m_used == -INFINITY ? 0.f : m_used;  // a row that has seen no key yet
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < BK / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float p0 = ex2_approx(fmaf(sv[c * 32 + i], a.sl2, -ref));
            const float p1 = ex2_approx(fmaf(sv[c * 32 + i + 1], a.sl2, -ref));
            sum[(i >> 1) & 3] += p0 + p1;
            // P is rounded to the values' type for the tensor core; the sum keeps fp32.
            pk[i / 2] = pack<T>(p0, p1);
          }
          tmem_st_32x16_issue(t_s + 16 * c, pk);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (!ok || !mbar_wait(&o_done[t], c_o, kErrTimeoutEpilogue, a.err)) break;
      c_o ^= 1;
      tc_fence_after();
      const long slot = pc.continued ? cta_slot(w, blockIdx.x, t * 128 + r) : base_slot(a, pc.shared, pc.head, pair);
      if (mine) a.part_ml[slot] = make_float2(m_used, l);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        tmem_ld_32x32(t_o + c * 32, o);
        if (mine)
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(a.part_o + slot * D + c * 32 + i) =
                make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
      }
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
  paged_attn_tc_kernel<T, D><<<a.work[1].ctas, kThreads, smem, stream>>>(k, v, a);
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "paged_attention launch failed");
}

template void launch_big<__nv_bfloat16, 64>(const CUtensorMap&, const CUtensorMap&, const Args&, cudaStream_t);
template void launch_big<__nv_bfloat16, 128>(const CUtensorMap&, const CUtensorMap&, const Args&, cudaStream_t);
template void launch_big<__half, 64>(const CUtensorMap&, const CUtensorMap&, const Args&, cudaStream_t);
template void launch_big<__half, 128>(const CUtensorMap&, const CUtensorMap&, const Args&, cudaStream_t);

}  // namespace pa
}  // namespace nk
