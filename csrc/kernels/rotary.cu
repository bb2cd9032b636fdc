// Rotary positions, alone (forward and backward, out of place or in place) and
// fused with the write of new keys and values into the pages of a cache.
//
// Pair i of a head's first `rot` elements turns by the angle of its row's
// position, in this framework's sign convention (rs-nanogpt src/model/rope.rs:48-72):
//     y1 = x1 cos + x2 sin,   y2 = x2 cos - x1 sin
// with (x1, x2) = (x[i], x[i + rot/2]) in the half layout and (x[2i], x[2i+1])
// in the interleaved one; elements past `rot` pass through. The gradient is the
// transposed turn, sin -> -sin. cos and sin come from tables of one row a
// position (fp32, computed in 64 bits on the host side), so an angle of a far
// position costs no precision. All arithmetic is fp32, rounded once on the store.
//
// Bound by memory: a row-head is read and written once and the few operations a
// value hide under it.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>
#include <torch/extension.h>

#include "common.cuh"
#include "message.h"
#include "overlap.h"
#include "status.h"

namespace nk {
namespace {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half(v); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

// One item: V pairs. In the half layout its two vectors lie rot/2 apart, in the
// interleaved one side by side; items past the rotated part are two vectors
// side by side that pass through. There are d / (2 V) items a row-head.
template <int V>
__device__ __forceinline__ void item_offsets(int j, int half, bool interleaved, int& a, int& b) {
  if (!interleaved && j * V < half) {
    a = j * V;
    b = half + j * V;
  } else {
    a = 2 * j * V;
    b = a + V;
  }
}

template <int V>
__device__ __forceinline__ void load_angles(const float* __restrict__ cos_t, const float* __restrict__ sin_t, long at,
                                            float sign, float (&c)[V], float (&s)[V]) {
  const Vec<float, (V < 4 ? V : 4)>* pc = reinterpret_cast<const Vec<float, (V < 4 ? V : 4)>*>(cos_t + at);
  const Vec<float, (V < 4 ? V : 4)>* ps = reinterpret_cast<const Vec<float, (V < 4 ? V : 4)>*>(sin_t + at);
#pragma unroll
  for (int i = 0; i < (V + 3) / 4; ++i) {
    const auto vc = pc[i], vs = ps[i];
#pragma unroll
    for (int e = 0; e < (V < 4 ? V : 4); ++e) {
      c[4 * i + e] = vc.e[e];
      s[4 * i + e] = sign * vs.e[e];
    }
  }
}

// Turns one item held in fp32 (two vectors of V).
template <int V>
__device__ __forceinline__ void turn(float (&x)[2 * V], const float (&c)[V], const float (&s)[V], bool interleaved) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    // Index arithmetic on constants only, so x stays in registers in both layouts.
    if (interleaved) {
      const float x1 = x[2 * i], x2 = x[2 * i + 1];
      x[2 * i] = x1 * c[i] + x2 * s[i];
      x[2 * i + 1] = x2 * c[i] - x1 * s[i];
    } else {
      const float x1 = x[i], x2 = x[V + i];
      x[i] = x1 * c[i] + x2 * s[i];
      x[V + i] = x2 * c[i] - x1 * s[i];
    }
  }
}

struct Heads {  // one tensor (rows, heads, d): read at src, written at dst
  const void* src;
  void* dst;
  long src_row, src_head, dst_row, dst_head;
};

struct RotateArgs {
  Heads q, k;
  const int* pos;
  const float *cos_t, *sin_t;
  int rows, hq, heads, half, items, positions, abreast;  // abreast: heads of a row that threads hold side by side
  float sign;
  bool interleaved;
  int* err;
};

constexpr int kRotThreads = 256;

// Thread = (row, one of `abreast` neighbouring heads, item): it reads the row's
// angles once and walks the heads `abreast` apart. With a warp on one row, its loads
// are runs of 512 bytes and more. One head's loads a thread and five CTAs an SM
// (48 registers) keep more in flight than several heads a thread: 65536 rows of 20
// heads of 128 in bf16 (672 MB) take 111 us, 6.1 TB/s; with 2, 3 and 5 heads' loads
// at once 150, 196 and 190 us, with four or six CTAs 118 us each.
template <typename T, int V>
__global__ void __launch_bounds__(kRotThreads, 5) rotate_kernel(const RotateArgs a) {
  const long id = long(blockIdx.x) * kRotThreads + threadIdx.x;
  const int of_row = a.items * a.abreast;
  if (id >= long(a.rows) * of_row) return;
  const int row = int(id / of_row), in_row = int(id - long(row) * of_row), j = in_row % a.items;
  const int p = a.pos[row];
  if (p < 0 || p >= a.positions) {  // reported; the row is left as it was
    if (in_row == 0) atomicCAS(a.err, 0, kErrBounds);
    return;
  }
  int oa, ob;
  item_offsets<V>(j, a.half, a.interleaved, oa, ob);
  const bool turned = j * V < a.half;
  float c[V], s[V];
  if (turned) load_angles<V>(a.cos_t, a.sin_t, long(p) * a.half + j * V, a.sign, c, s);
#pragma unroll 1
  for (int h = in_row / a.items; h < a.heads; h += a.abreast) {
    const bool is_q = h < a.hq;
    const Heads& t = is_q ? a.q : a.k;
    const int i = is_q ? h : h - a.hq;
    const T* src = static_cast<const T*>(t.src) + row * t.src_row + i * t.src_head;
    T* dst = static_cast<T*>(t.dst) + row * t.dst_row + i * t.dst_head;
    Vec<T, V> va = *reinterpret_cast<const Vec<T, V>*>(src + oa), vb = *reinterpret_cast<const Vec<T, V>*>(src + ob);
    if (turned) {
      float x[2 * V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x[e] = to_f32<T>(va.e[e]);
        x[V + e] = to_f32<T>(vb.e[e]);
      }
      turn<V>(x, c, s, a.interleaved);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        va.e[e] = from_f32<T>(x[e]);
        vb.e[e] = from_f32<T>(x[V + e]);
      }
    }
    *reinterpret_cast<Vec<T, V>*>(dst + oa) = va;
    *reinterpret_cast<Vec<T, V>*>(dst + ob) = vb;
  }
}

struct AppendArgs {
  Heads q, k, v;  // k.dst, v.dst: the layer's pages; *_row: elements a page, *_head: elements a head of a page
  const int *table, *lens, *row_slot, *row_back;
  const int* room;             // tokens of a slot that were granted and not yet written; null: nothing is known
  const float *cos_t, *sin_t;  // null: no turn
  int rows, hq, hk, half, positions, page, width, pages, slots;
  float eps;
  bool norm, interleaved;
  int* err;
};

// D / 16 lanes a (row, head), each with 8 / V items; heads are q's, then k's,
// then v's. The norm's sum of squares is a shuffle over those lanes. 11000 rows of
// 24 heads of 64 (67 MB): 18.5 us from memory, 12.8 us from L2; one decode step of
// 32 rows: 2.6 us, launch included.
template <typename T, int V, int D>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
  constexpr int L = D / 16, NI = 8 / V;
  const int group = (blockIdx.x * 256 + threadIdx.x) / L, lane = threadIdx.x % L;
  const int heads = a.hq + 2 * a.hk;
  if (group >= a.rows * heads) return;  // whole groups leave; the shuffles name only their own lanes
  const int row = group / heads, h = group % heads;
  const bool is_q = h < a.hq, is_v = h >= a.hq + a.hk;
  const Heads& t = is_q ? a.q : (is_v ? a.v : a.k);
  const int i = is_q ? h : (is_v ? h - a.hq - a.hk : h - a.hq);
  const int slot = __ldg(a.row_slot + row), back = __ldg(a.row_back + row);
  // The values are on their way while the row's place is looked up.
  const T* src = static_cast<const T*>(t.src) + row * t.src_row + i * t.src_head;
  Vec<T, V> va[NI], vb[NI];
  int oa[NI], ob[NI];
#pragma unroll
  for (int n = 0; n < NI; ++n) {
    item_offsets<V>(lane + n * L, a.half, a.interleaved, oa[n], ob[n]);
    va[n] = *reinterpret_cast<const Vec<T, V>*>(src + oa[n]);
    vb[n] = *reinterpret_cast<const Vec<T, V>*>(src + ob[n]);
  }
  // A row that stands nowhere: 0 in q's output, not what its memory held.
  auto nowhere = [&](int code) {
    if (code && lane == 0) atomicCAS(a.err, 0, code);
    if (!is_q) return;
    T* dst = static_cast<T*>(t.dst) + row * t.dst_row + i * t.dst_head;
#pragma unroll
    for (int n = 0; n < NI; ++n)
      *reinterpret_cast<Vec<T, V>*>(dst + oa[n]) = *reinterpret_cast<Vec<T, V>*>(dst + ob[n]) = Vec<T, V>{};
  };
  if (slot < 0 || slot >= a.slots) return nowhere(kErrBounds);
  const int p = __ldg(a.lens + slot) - 1 - back;
  if (p < 0) return nowhere(kErrNone);  // a slot that holds fewer tokens than its rows: nothing to write
  if (a.room && back >= a.room[slot]) return nowhere(kErrNoPages);  // the place of a token that the cache holds
  if (p >= a.positions || p >= a.width * a.page) return nowhere(kErrBounds);
  T* dst;
  if (is_q) {
    dst = static_cast<T*>(t.dst) + row * t.dst_row + i * t.dst_head;
  } else {
    const int page = __ldg(a.table + long(slot) * a.width + p / a.page);
    if (page < 0 || page >= a.pages) {
      if (lane == 0) atomicCAS(a.err, 0, kErrBounds);
      return;
    }
    dst = static_cast<T*>(t.dst) + page * t.dst_row + i * t.dst_head + long(p % a.page) * D;
  }
  if (!is_v) {
    float x[NI][2 * V], sq = 0.f;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x[n][e] = to_f32<T>(va[n].e[e]);
        x[n][V + e] = to_f32<T>(vb[n].e[e]);
      }
      const int j = lane + n * L;
      if (j * V < a.half) {
        float c[V], s[V];
        load_angles<V>(a.cos_t, a.sin_t, long(p) * a.half + j * V, 1.f, c, s);
        turn<V>(x[n], c, s, a.interleaved);
      }
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) sq = fmaf(x[n][e], x[n][e], sq);
    }
    float r = 1.f;
    if (a.norm) {
      const unsigned lanes = ((1ull << L) - 1) << (threadIdx.x % 32 / L * L);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(lanes, sq, o);
      r = 1.f / sqrtf(sq / D + a.eps);
    }
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        va[n].e[e] = from_f32<T>(x[n][e] * r);
        vb[n].e[e] = from_f32<T>(x[n][V + e] * r);
      }
  }
#pragma unroll
  for (int n = 0; n < NI; ++n) {
    *reinterpret_cast<Vec<T, V>*>(dst + oa[n]) = va[n];
    *reinterpret_cast<Vec<T, V>*>(dst + ob[n]) = vb[n];
  }
}

// ---- host ---------------------------------------------------------------------

void check_heads(const torch::Tensor& t, const char* name, const torch::Tensor& like, int64_t rows, int64_t d) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, ": must be on ", place(like));
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, ": dtype ", type_name(t), ", expected ", type_name(like));
  TORCH_CHECK(t.dim() == 3 && t.size(0) == rows && t.size(2) == d, name, ": expected (", num(rows), ", heads, ", num(d),
              "), got ", dims(t));
  TORCH_CHECK(t.size(2) == 1 || t.stride(2) == 1, name, ": the last dimension must be contiguous");
}

void check_tables(const torch::Tensor& cos_t, const torch::Tensor& sin_t, const torch::Tensor& like, int64_t d) {
  TORCH_CHECK(cos_t.is_cuda() && cos_t.device() == like.device() && cos_t.scalar_type() == at::kFloat &&
                  cos_t.dim() == 2 && cos_t.is_contiguous() && sin_t.device() == cos_t.device() &&
                  sin_t.scalar_type() == at::kFloat && sin_t.sizes() == cos_t.sizes() && sin_t.is_contiguous(),
              "rotary: cos and sin must be contiguous fp32 (positions, rot / 2) on ", place(like));
  TORCH_CHECK(cos_t.size(1) >= 1 && 2 * cos_t.size(1) <= d, "rotary: tables turn ", num(2 * cos_t.size(1)),
              " elements of heads of ", num(d));
}

void check_ints(const torch::Tensor& t, const char* name, const torch::Tensor& like) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt && t.is_contiguous(), name,
              ": must be contiguous int32 on ", place(like));
}

// Elements a vector access may hold so that every row, head and item start is aligned to it.
struct Width {
  int64_t v;
  explicit Width(int64_t most) : v(most) {}
  void fit(int64_t n) { while (v > 1 && n % v) v /= 2; }
  void fit(const torch::Tensor& cos_t, const torch::Tensor& sin_t) {  // rows are a multiple of v long already
    for (const auto* t : {&cos_t, &sin_t}) fit(int64_t(reinterpret_cast<uintptr_t>(t->data_ptr()) / 4));
  }
  void fit(const torch::Tensor& t) {
    fit(int64_t(reinterpret_cast<uintptr_t>(t.data_ptr()) / t.element_size()));
    for (int i = 0; i + 1 < t.dim(); ++i)
      if (t.size(i) > 1) fit(t.stride(i));
  }
};

Heads heads_of(const torch::Tensor& src, const torch::Tensor& dst) {
  return Heads{src.data_ptr(), dst.data_ptr(), src.stride(0), src.stride(1), dst.stride(0), dst.stride(1)};
}

template <typename T>
void launch_rotate(const RotateArgs& a, int64_t v, unsigned grid, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (v == 8) {
      rotate_kernel<T, 8><<<grid, kRotThreads, 0, stream>>>(a);
      return;
    }
  }
  if (v == 4) rotate_kernel<T, 4><<<grid, kRotThreads, 0, stream>>>(a);
  else if (v == 2) rotate_kernel<T, 2><<<grid, kRotThreads, 0, stream>>>(a);
  else rotate_kernel<T, 1><<<grid, kRotThreads, 0, stream>>>(a);
}

template <typename T, int D>
void launch_append(const AppendArgs& a, int64_t v, unsigned grid, cudaStream_t stream) {
  if (v == 8) append_kernel<T, 8, D><<<grid, 256, 0, stream>>>(a);
  else if (v == 4) append_kernel<T, 4, D><<<grid, 256, 0, stream>>>(a);
  else if (v == 2) append_kernel<T, 2, D><<<grid, 256, 0, stream>>>(a);
  else append_kernel<T, 1, D><<<grid, 256, 0, stream>>>(a);
}

}  // namespace

// q_out = turn(q), k_out = turn(k) with the angles of row r's position pos[r];
// back: the transposed turn, for gradients.
void rotate(torch::Tensor q, c10::optional<torch::Tensor> k, torch::Tensor pos, torch::Tensor cos_t,
            torch::Tensor sin_t, bool interleaved, bool back, torch::Tensor q_out, c10::optional<torch::Tensor> k_out) {
  const auto type = q.scalar_type();
  TORCH_CHECK(q.is_cuda(), "rotate: q must be on a GPU");
  TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat, "rotate: bf16, fp16 or fp32, got ",
              type_name(q));
  TORCH_CHECK(q.dim() == 3, "rotate: q must be (rows, heads, head_dim), got ", dims(q));
  const int64_t rows = q.size(0), d = q.size(2);
  TORCH_CHECK(d % 2 == 0 && d > 0, "rotate: head_dim must be even, got ", num(d));
  check_heads(q, "rotate: q", q, rows, d);
  check_heads(q_out, "rotate: q_out", q, rows, d);
  TORCH_CHECK(q_out.sizes() == q.sizes(), "rotate: q_out shape");
  TORCH_CHECK(k.has_value() == k_out.has_value(), "rotate: k and k_out come together");
  if (k.has_value()) {
    check_heads(*k, "rotate: k", q, rows, d);
    check_heads(*k_out, "rotate: k_out", q, rows, d);
    TORCH_CHECK(k_out->sizes() == k->sizes(), "rotate: k_out shape");
  }
  check_tables(cos_t, sin_t, q, d);
  check_ints(pos, "rotate: pos", q);
  TORCH_CHECK(pos.dim() == 1 && pos.size(0) == rows, "rotate: pos must have ", num(rows), " entries");
  const Operand oq(q, "rotate: q"), oq_out(q_out, "rotate: q_out");
  check_result(oq, oq_out);
  if (k.has_value()) {
    const Operand ok(*k, "rotate: k"), ok_out(*k_out, "rotate: k_out");
    check_result(ok, ok_out);
    check_disjoint(oq_out, ok);
    check_disjoint(ok_out, oq);
    check_disjoint(oq_out, ok_out);
  }
  RotateArgs a{};
  a.hq = int(q.size(1));
  a.heads = a.hq + (k.has_value() ? int(k->size(1)) : 0);
  if (rows == 0 || a.heads == 0) return;
  TORCH_CHECK(rows <= INT32_MAX && cos_t.size(0) <= INT32_MAX, "rotate: too many rows");
  const int64_t half = cos_t.size(1);
  Width w(16 / q.element_size());
  w.fit(half);
  w.fit(cos_t, sin_t);
  w.fit(d / 2);
  w.fit(q);
  w.fit(q_out);
  if (k.has_value()) {
    w.fit(*k);
    w.fit(*k_out);
  }
  a.q = heads_of(q, q_out);
  if (k.has_value()) a.k = heads_of(*k, *k_out);
  a.pos = pos.data_ptr<int>();
  a.cos_t = cos_t.data_ptr<float>();
  a.sin_t = sin_t.data_ptr<float>();
  a.rows = int(rows);
  a.half = int(half);
  a.items = int(d / (2 * w.v));
  a.positions = int(cos_t.size(0));
  a.sign = back ? -1.f : 1.f;
  a.interleaved = interleaved;
  a.err = error_word();
  const at::cuda::CUDAGuard guard(q.device());
  // A warp's worth of a row's items side by side; all heads side by side while that
  // leaves a thread for every item (few rows: no thread walks over heads).
  a.abreast = std::min(a.heads, std::max(1, 32 / a.items));
  if (rows * a.items * a.heads <= 148 * 2048) a.abreast = a.heads;
  const int64_t blocks = (rows * a.items * a.abreast + kRotThreads - 1) / kRotThreads;
  TORCH_CHECK(blocks <= INT32_MAX, "rotate: too many rows");
  const unsigned grid = unsigned(blocks);
  auto stream = at::cuda::getCurrentCUDAStream();
  if (type == at::kBFloat16) launch_rotate<__nv_bfloat16>(a, w.v, grid, stream);
  else if (type == at::kHalf) launch_rotate<__half>(a, w.v, grid, stream);
  else launch_rotate<float>(a, w.v, grid, stream);
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "rotate launch failed");
}

// q_out = norm(turn(q)); k's and v's rows go to the pages of their sequences
// (k turned and normed as q is).
void paged_append(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor k_pages, torch::Tensor v_pages,
                  torch::Tensor table, torch::Tensor lens, torch::Tensor row_slot, torch::Tensor row_back,
                  c10::optional<torch::Tensor> cos_t, c10::optional<torch::Tensor> sin_t, bool interleaved, double eps,
                  bool norm, torch::Tensor q_out, c10::optional<torch::Tensor> room) {
  const auto type = q.scalar_type();
  TORCH_CHECK(q.is_cuda(), "append: q must be on a GPU");
  TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf, "append: bf16 or fp16, got ", type_name(q));
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "append: q, k and v must be (rows, heads, head_dim)");
  const int64_t rows = q.size(0), d = q.size(2), hk = k.size(1);
  TORCH_CHECK(d == 64 || d == 128, "append: head_dim must be 64 or 128, got ", num(d));
  check_heads(q, "append: q", q, rows, d);
  check_heads(k, "append: k", q, rows, d);
  check_heads(v, "append: v", q, rows, d);
  check_heads(q_out, "append: q_out", q, rows, d);
  TORCH_CHECK(v.size(1) == hk && q_out.size(1) == q.size(1), "append: head counts of k and v, q and q_out differ");
  const Operand oq_out(q_out, "append: q_out");
  check_result(Operand(q, "append: q"), oq_out);
  check_disjoint(oq_out, Operand(k, "append: k"));
  check_disjoint(oq_out, Operand(v, "append: v"));
  for (const auto* p : {&k_pages, &v_pages}) {
    TORCH_CHECK(p->device() == q.device() && p->scalar_type() == type && p->dim() == 4 && p->size(1) == hk &&
                    p->size(3) == d && p->sizes() == k_pages.sizes(),
                "append: pages must be (pages, ", num(hk), ", rows of a page, ", num(d), ") of q's dtype, got ",
                dims(*p));
    TORCH_CHECK(p->stride(3) == 1 && p->stride(2) == d && p->stride(1) == d * p->size(2),
                "append: a page must be contiguous");
  }
  check_ints(table, "append: table", q);
  check_ints(lens, "append: lens", q);
  check_ints(row_slot, "append: row_slot", q);
  check_ints(row_back, "append: row_back", q);
  TORCH_CHECK(table.dim() == 2 && lens.dim() == 1 && table.size(0) == lens.size(0),
              "append: table and lens slots differ");
  TORCH_CHECK(row_slot.numel() == rows && row_back.numel() == rows, "append: the plan has ", num(row_slot.numel()),
              " rows, q has ", num(rows));
  if (room.has_value()) {
    check_ints(*room, "append: room", q);
    TORCH_CHECK(room->sizes() == lens.sizes(), "append: room must have one entry for each slot");
  }
  AppendArgs a{};
  Width w(8);
  if (cos_t.has_value()) {
    TORCH_CHECK(sin_t.has_value(), "append: cos and sin come together");
    check_tables(*cos_t, *sin_t, q, d);
    a.cos_t = cos_t->data_ptr<float>();
    a.sin_t = sin_t->data_ptr<float>();
    a.half = int(cos_t->size(1));
    a.positions = int(cos_t->size(0));
    w.fit(a.half);
    w.fit(*cos_t, *sin_t);
  } else {
    a.positions = INT32_MAX;
  }
  if (rows == 0) return;
  for (const auto* t : {&q, &k, &v, &q_out, &k_pages, &v_pages}) w.fit(*t);
  a.q = heads_of(q, q_out);
  a.k = heads_of(k, k_pages);
  a.v = heads_of(v, v_pages);
  a.table = table.data_ptr<int>();
  a.lens = lens.data_ptr<int>();
  a.row_slot = row_slot.data_ptr<int>();
  a.row_back = row_back.data_ptr<int>();
  a.room = room.has_value() ? room->data_ptr<int>() : nullptr;
  a.rows = int(rows);
  a.hq = int(q.size(1));
  a.hk = int(hk);
  a.page = int(k_pages.size(2));
  a.width = int(table.size(1));
  a.pages = int(k_pages.size(0));
  a.slots = int(table.size(0));
  a.eps = float(eps);
  a.norm = norm;
  a.interleaved = interleaved;
  a.err = error_word();
  const int64_t threads = rows * (a.hq + 2 * hk) * (d / 16);
  TORCH_CHECK(threads <= INT32_MAX - 256, "append: too many rows");
  const at::cuda::CUDAGuard guard(q.device());
  const unsigned grid = unsigned((threads + 255) / 256);
  auto stream = at::cuda::getCurrentCUDAStream();
  if (type == at::kBFloat16 && d == 128) launch_append<__nv_bfloat16, 128>(a, w.v, grid, stream);
  else if (type == at::kBFloat16) launch_append<__nv_bfloat16, 64>(a, w.v, grid, stream);
  else if (d == 128) launch_append<__half, 128>(a, w.v, grid, stream);
  else launch_append<__half, 64>(a, w.v, grid, stream);
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "paged_append launch failed");
}

}  // namespace nk
