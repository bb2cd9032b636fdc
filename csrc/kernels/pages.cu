// Pages of a KV cache: forking sequences (copy of the last, partly filled page),
// making room for new tokens, freeing sequences, compacting the pool, and plain
// page copies. All state lives on the device and no call reads it back, so the
// operators can be queued (or captured in a CUDA graph) without a host wait.
//
//   k, v    (layers, pages, kv heads, rows of a page, head dim)
//   table   (slots, width) int32: a sequence's pages in order, -1 past the last
//   lens    (slots) int32: tokens of a sequence (0: the slot is empty)
//   refs    (pages) int32: table entries that name the page (0: the page is free)
//   room    (slots) int32, optional: tokens that grow granted and that are not written
//           yet, so that the append can tell them from those the cache holds
//
// Full pages are shared between forks and never written again; a partly filled
// page belongs to one sequence. New pages are the lowest free ones, handed out in
// the order of the call's list, so every result is defined exactly.
//
// Each operator is one launch that rewrites table, lens and refs (into fresh
// tensors or in place) in phases separated by barriers, and, where rows move, a
// second launch that copies them from a list of pairs that the first one left in
// the workspace. The first is bound by its chain of barriers and look-ups: one CTA
// runs it while the state is small, a cluster of eight when there is much to read.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <climits>
#include <utility>

#include "common.cuh"
#include "launch.h"
#include "message.h"
#include "status.h"

namespace nk {
namespace {

constexpr int kMetaThreads = 1024;
constexpr int kMetaCtas = 8;  // one portable cluster

// The threads that work on the state: a CTA, or a cluster of C.
template <int C>
struct Team {
  static constexpr int kAll = C * kMetaThreads, kWarps = kAll / 32;
  __device__ static int cta() { return C == 1 ? 0 : int(cluster_rank()); }
  __device__ static int gid() { return cta() * kMetaThreads + int(threadIdx.x); }
  __device__ static void sync() {
    if constexpr (C == 1) __syncthreads();
    else cluster_sync();
  }
};

struct PageState {
  const int *table_in, *lens_in, *refs_in;
  int *table, *lens, *refs;
  int slots, width, pages, page;  // page: rows of one
  bool fresh;                     // the outputs are other tensors than the inputs
  int* err;
};

// Workspace of the metadata kernels (int32): per-CTA counts and totals, then the
// lists. kListAt is where the first list starts.
constexpr int kWsCounts = 0, kWsPairs = 8, kListAt = 16;

__device__ __forceinline__ void report(int* err, int code) { atomicCAS(err, 0, code); }

// table, lens and refs into the outputs, by the whole team.
template <int C>
__device__ __forceinline__ void copy_state(const PageState& s) {
  if (!s.fresh) return;
  constexpr int all = Team<C>::kAll, U = 4;
  const int gid = Team<C>::gid();
  const long n = long(s.slots) * s.width;
  for (long i = gid; i < n; i += long(U) * all) {
    int x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + long(u) * all < n) x[u] = s.table_in[i + long(u) * all];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + long(u) * all < n) s.table[i + long(u) * all] = x[u];
  }
  for (int i = gid; i < s.slots; i += all) s.lens[i] = s.lens_in[i];
  for (int i = gid; i < s.pages; i += all) s.refs[i] = s.refs_in[i];
}

// Exclusive sum over a CTA's threads; every thread also gets the total. Sums stop at
// kMany, which is more than there can be pages or list entries, and are not exact there.
constexpr int kMany = (1 << 30) - 1;
__device__ __forceinline__ int cta_scan(int v, int* sm, int& total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x = min(x + y, kMany);
  }
  __syncthreads();  // sm may still be read from an earlier call
  if (lane == 31) sm[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = sm[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w = min(w + y, kMany);
    }
    sm[lane] = w;
  }
  __syncthreads();
  total = sm[31];
  return (warp ? sm[warp - 1] : 0) + x - v;
}

// Each thread of the team owns pages [lo, hi). Returns how many pages before lo
// have refs > 0, and the number of all such pages. One barrier of the team.
template <int C>
__device__ __forceinline__ int live_before(const int* refs, int pages, int* sm, int* ws, int& lo, int& hi, int& live) {
  const int span = (pages + Team<C>::kAll - 1) / Team<C>::kAll;
  lo = min(pages, Team<C>::gid() * span);
  hi = min(pages, lo + span);
  int mine = 0;
  for (int p = lo; p < hi; ++p) mine += refs[p] > 0;
  int total;
  int before = cta_scan(mine, sm, total);
  if (C > 1 && threadIdx.x == 0) ws[kWsCounts + Team<C>::cta()] = total;
  Team<C>::sync();
  live = total;
  if constexpr (C > 1) {
    live = 0;
    for (int c = 0; c < C; ++c) {
      const int n = __ldcg(ws + kWsCounts + c);
      if (c < Team<C>::cta()) before += n;
      live += n;
    }
  }
  return before;
}

// ---- fork ----------------------------------------------------------------------

// ws lists: owner (slots); then n each of: free pages, pair sources, pair
// targets, pair rows, lengths of the children to make (-1: none).
template <int C>
__global__ void __launch_bounds__(kMetaThreads)
    fork_meta_kernel(const PageState s, const int* __restrict__ parents, const int* __restrict__ children, int n,
                     int* ws) {
  __shared__ int sm[32];
  using team = Team<C>;
  const int gid = team::gid();
  pdl_trigger();
  int *owner = ws + kListAt, *spare = owner + s.slots, *src = spare + n, *dst = src + n, *rows = dst + n,
      *length = rows + n;
  copy_state<C>(s);
  for (int i = gid; i < s.slots; i += team::kAll) owner[i] = INT_MAX;
  int lo, hi, live;
  const int before = live_before<C>(s.refs_in, s.pages, sm, ws, lo, hi, live);
  for (int p = lo, f = lo - before; p < hi && f < n; ++p)
    if (s.refs_in[p] <= 0) spare[f++] = p;
  // A slot that the list names twice goes to its first mention.
  for (int i = gid; i < n; i += team::kAll) {
    const int c = children[i];
    if (c >= 0 && c < s.slots) atomicMin(owner + c, i);
  }
  team::sync();
  if (team::cta() == 0) {
    // Which children are made, and the page of each that needs one: by one CTA,
    // in the list's order.
    const int span = (n + kMetaThreads - 1) / kMetaThreads;
    const int i0 = min(n, int(threadIdx.x) * span), i1 = min(n, i0 + span);
    int mine = 0, total;
    for (int i = i0; i < i1; ++i) {
      const int p = parents[i], c = children[i];
      const bool ok = p >= 0 && p < s.slots && c >= 0 && c < s.slots && __ldcg(owner + c) == i && s.lens_in[c] == 0 &&
                      s.lens_in[p] >= 0 && s.lens_in[p] <= s.width * s.page;
      if (!ok) report(s.err, kErrBounds);
      length[i] = ok ? s.lens_in[p] : -1;
      mine += ok && length[i] % s.page;
    }
    int rank = cta_scan(mine, sm, total);
    for (int i = i0; i < i1; ++i) {
      const int len = length[i];
      const bool part = len >= 0 && len % s.page;
      src[i] = dst[i] = -1;
      rows[i] = 0;
      if (part && rank++ < s.pages - live) {
        src[i] = s.table_in[long(parents[i]) * s.width + len / s.page];
        dst[i] = __ldcg(spare + rank - 1);
        rows[i] = len % s.page;
      } else if (part) {
        report(s.err, kErrNoPages);
        length[i] = -1;
      }
    }
  }
  team::sync();
  for (int i = gid / 32; i < n; i += team::kWarps) {
    const int len = __ldcg(length + i), lane = threadIdx.x % 32;
    if (len < 0) continue;
    const int* from = s.table_in + long(parents[i]) * s.width;
    int* to = s.table + long(children[i]) * s.width;
    for (int e = lane; e < len / s.page; e += 32) {
      const int q = from[e];
      to[e] = q;
      if (q >= 0 && q < s.pages) atomicAdd(s.refs + q, 1);
    }
    if (lane == 0) {
      s.lens[children[i]] = len;
      if (len % s.page) {
        const int q = __ldcg(dst + i);
        to[len / s.page] = q;
        s.refs[q] = 1;
      }
    }
  }
}

// ---- grow ----------------------------------------------------------------------

// ws lists: free pages (pages); of each slot, the first of its pages in that list
// (slots; -1: refused), written only where there are too few pages for all.
template <int C>
__global__ void __launch_bounds__(kMetaThreads)
    grow_meta_kernel(const PageState s, const int* __restrict__ add, int* room, int* ws) {
  __shared__ int sm[32];
  using team = Team<C>;
  const int gid = team::gid();
  pdl_trigger();
  int *spare = ws + kListAt, *served = spare + s.pages;
  copy_state<C>(s);
  int lo, hi, live;
  const int before = live_before<C>(s.refs_in, s.pages, sm, ws, lo, hi, live);
  for (int p = lo, f = lo - before; p < hi; ++p)
    if (s.refs_in[p] <= 0) spare[f++] = p;
  team::sync();
  if (team::cta() != 0) return;
  const int span = (s.slots + kMetaThreads - 1) / kMetaThreads, avail = s.pages - live;
  const int i0 = min(s.slots, int(threadIdx.x) * span), i1 = min(s.slots, i0 + span);
  auto pages_for = [&](int tokens) { return int((unsigned(tokens) + s.page - 1) / s.page); };
  auto need = [&](int i, int& len, int& have) {  // pages that slot i lacks; -1: it cannot be grown
    const int more = add[i];
    len = s.lens_in[i];
    have = pages_for(len);
    if (more < 0 || len < 0 || long(len) + more > long(s.width) * s.page) return -1;
    return pages_for(len + more) - have;
  };
  int len, have, mine = 0, total;
  for (int i = i0; i < i1; ++i) mine = int(min(mine + unsigned(max(0, need(i, len, have))), unsigned(kMany)));
  const int rank = cta_scan(mine, sm, total);
  const bool enough = total <= avail;
  if (!enough) {
    // Served in order; a slot that wants more than is left takes nothing. A warp
    // looks at 32 slots together and deals them their pages one by one.
    if (threadIdx.x < 32) {
      int used = 0;
      for (int b = 0; b < s.slots; b += 32) {
        const int i = b + int(threadIdx.x), m = i < s.slots ? max(0, need(i, len, have)) : 0;
        int at = m ? -1 : 0;
        for (unsigned left = __ballot_sync(0xffffffffu, m > 0); left; left &= left - 1) {
          const int from = __ffs(left) - 1, want = __shfl_sync(0xffffffffu, m, from);
          if (want > avail - used) continue;
          if (int(threadIdx.x) == from) at = used;
          used += want;
        }
        if (i < s.slots) served[i] = at;
      }
    }
    __syncthreads();
  }
  int next = enough ? rank : 0;
  for (int i = i0; i < i1; ++i) {
    const int m = need(i, len, have), at = enough ? next : served[i];
    next += max(0, m);
    if (m < 0) {
      report(s.err, kErrBounds);
    } else if (at < 0) {
      report(s.err, kErrNoPages);  // this slot keeps its length
    } else {
      for (int e = 0; e < m; ++e) {
        const int q = __ldcg(spare + at + e);
        s.table[long(i) * s.width + have + e] = q;
        s.refs[q] = 1;
      }
      if (add[i]) {
        s.lens[i] = len + add[i];
        if (room) room[i] += add[i];
      }
    }
  }
}

// ---- free ----------------------------------------------------------------------

template <int C>
__global__ void __launch_bounds__(kMetaThreads)
    free_meta_kernel(const PageState s, const int* __restrict__ seqs, int n, int* room) {
  using team = Team<C>;
  const int gid = team::gid();
  copy_state<C>(s);
  team::sync();
  for (int i = gid / 32; i < n; i += team::kWarps) {
    const int slot = seqs[i], lane = threadIdx.x % 32;
    if (slot < 0 || slot >= s.slots) {
      if (lane == 0) report(s.err, kErrBounds);
      continue;
    }
    if (room && lane == 0) room[slot] = 0;
    // A slot that the list names twice is freed once.
    const int had = __shfl_sync(0xffffffffu, lane == 0 ? atomicExch(s.lens + slot, 0) : 0, 0);
    if (had <= 0) continue;
    int* row = s.table + long(slot) * s.width;
    for (int e = lane; e < s.width; e += 32) {
      const int q = __ldcg(row + e);
      if (q >= 0 && q < s.pages) atomicSub(s.refs + q, 1);
      row[e] = -1;
    }
  }
}

// ---- compact -------------------------------------------------------------------

// The L pages in use get the numbers below L: those that have one keep it, the
// i-th of the others (ascending) moves to the i-th free page below L.
// ws lists (pages each): pair sources, pair targets, sources from the last one
// down, new number of each page.
template <int C>
__global__ void __launch_bounds__(kMetaThreads)
    compact_meta_kernel(const PageState s, int* ws) {
  __shared__ int sm[32];
  using team = Team<C>;
  const int gid = team::gid();
  pdl_trigger();
  int *src = ws + kListAt, *dst = src + s.pages, *down = dst + s.pages, *to = down + s.pages;
  copy_state<C>(s);
  int lo, hi, live;
  int r = live_before<C>(s.refs_in, s.pages, sm, ws, lo, hi, live);
  if (gid == 0 && live == s.pages) ws[kWsPairs] = 0;
  for (int p = lo; p < hi; ++p) {
    const bool used = s.refs_in[p] > 0;
    to[p] = p;
    if (p == live) ws[kWsPairs] = live - r;
    if (!used && p < live) dst[p - r] = p;
    if (used && p >= live) down[live - 1 - r] = p;
    r += used;
  }
  team::sync();
  const int pairs = __ldcg(ws + kWsPairs);
  for (int i = gid; i < pairs; i += team::kAll) {
    const int from = __ldcg(down + pairs - 1 - i), t = __ldcg(dst + i);
    src[i] = from;
    to[from] = t;
    s.refs[t] = s.refs_in[from];
    s.refs[from] = 0;
  }
  team::sync();
  for (long i = gid; i < long(s.slots) * s.width; i += team::kAll) {
    const int q = s.table_in[i];
    if (q >= 0 && q < s.pages) s.table[i] = __ldcg(to + q);
  }
}

// ---- copies of pages -------------------------------------------------------------

struct CopyArgs {
  char *k, *v;
  long k_layer, k_page, v_layer, v_page;  // bytes
  const int *src, *dst, *rows;            // rows null: whole pages
  const int* count;                       // null: n pairs
  int n, layers, heads, page, row_bytes, pages;
  int* err;
};

constexpr int kCopyThreads = 256;

// A warp copies the rows of one (pair, layer, k or v, head): up to 2 KB of
// loads in flight, neighbouring warps on neighbouring heads of a page. Bound by
// memory: pages of 3.2 MB over 20 layers move at 6.3 TB/s (1.57 GB in 251 us).
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const CopyArgs a) {
  pdl_wait();  // the list may be the state kernel's
  const int lane = threadIdx.x % 32;
  const long warps = long(gridDim.x) * (kCopyThreads / 32);
  const int n = a.count ? min(*a.count, a.n) : a.n;
  const long units = long(n) * a.layers * 2 * a.heads;
  for (long u = long(blockIdx.x) * (kCopyThreads / 32) + threadIdx.x / 32; u < units; u += warps) {
    // All pairs of one layer's k or v, then the next: what is written at a time lies
    // in a few slices of the pool instead of all over it.
    const int head = int(u % a.heads);
    const long w = u / a.heads;
    const int pair = int(w % n), slice = int(w / n), layer = slice / 2;
    const bool is_v = slice & 1;
    const int from = a.src[pair], to = a.dst[pair];
    if (from < 0) continue;
    if (from >= a.pages || to < 0 || to >= a.pages) {
      if (lane == 0) report(a.err, kErrBounds);
      continue;
    }
    char* base = (is_v ? a.v + layer * a.v_layer : a.k + layer * a.k_layer) + long(head) * a.page * a.row_bytes;
    const long stride = is_v ? a.v_page : a.k_page;
    const uint4* in = reinterpret_cast<const uint4*>(base + from * stride);
    uint4* out = reinterpret_cast<uint4*>(base + to * stride);
    const int vecs = (a.rows ? a.rows[pair] : a.page) * (a.row_bytes / 16);
    for (int i = lane; i < vecs; i += 128) {
      uint4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + 32 * j < vecs) x[j] = in[i + 32 * j];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + 32 * j < vecs) out[i + 32 * j] = x[j];
    }
  }
}

// ---- host ----------------------------------------------------------------------

void check_int_vec(const torch::Tensor& t, const char* name, const torch::Tensor& like) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt && t.is_contiguous(), name,
              ": must be contiguous int32 on ", place(like));
}

PageState state_of(const torch::Tensor& table, const torch::Tensor& lens, const torch::Tensor& refs,
                   const torch::Tensor& table_out, const torch::Tensor& lens_out, const torch::Tensor& refs_out,
                   int64_t page, const char* op) {
  TORCH_CHECK(table.is_cuda(), op, ": table must be on a GPU");
  TORCH_CHECK(table.dim() == 2 && lens.dim() == 1 && refs.dim() == 1 && lens.size(0) == table.size(0), op,
              ": expected table (slots, width), lens (slots), refs (pages), got ", dims(table), ", ", dims(lens),
              ", ", dims(refs));
  for (const auto* t : {&table, &lens, &refs, &table_out, &lens_out, &refs_out}) check_int_vec(*t, op, table);
  TORCH_CHECK(table_out.sizes() == table.sizes() && lens_out.sizes() == lens.sizes() &&
                  refs_out.sizes() == refs.sizes(), op, ": shapes of the outputs");
  // Tensors without entries have no place of their own: they go with the others.
  int same = 0, other = 0;
  for (const auto& [in, to] : {std::pair(&table, &table_out), std::pair(&lens, &lens_out), std::pair(&refs, &refs_out)})
    if (in->numel()) (in->data_ptr() == to->data_ptr() ? same : other)++;
  TORCH_CHECK(!same || !other, op, ": table, lens and refs are written all in place or all out of place");
  TORCH_CHECK(page >= 1 && table.size(0) <= INT32_MAX / 8 && refs.size(0) <= INT32_MAX / 8 &&
                  table.size(1) * page <= INT32_MAX, op, ": sizes");
  return PageState{table.data_ptr<int>(), lens.data_ptr<int>(), refs.data_ptr<int>(), table_out.data_ptr<int>(),
                   lens_out.data_ptr<int>(), refs_out.data_ptr<int>(), int(table.size(0)), int(table.size(1)),
                   int(refs.size(0)), int(page), other > 0, error_word()};
}

int* room_of(const c10::optional<torch::Tensor>& room, const torch::Tensor& lens, const char* op) {
  if (!room.has_value()) return nullptr;
  check_int_vec(*room, op, lens);
  TORCH_CHECK(room->sizes() == lens.sizes(), op, ": room must have one entry for each slot");
  return room->data_ptr<int>();
}

CopyArgs pools_of(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& like, const char* op) {
  for (const auto* t : {&k, &v}) {
    TORCH_CHECK(t->is_cuda() && t->device() == like.device(), op, ": pages must be on ", place(like));
    TORCH_CHECK(t->dim() == 5 && t->sizes() == k.sizes() && t->scalar_type() == k.scalar_type(), op,
                ": pages must be (layers, pages, kv heads, rows, head_dim), k and v alike, got ", dims(*t));
    TORCH_CHECK(t->stride(4) == 1 && t->stride(3) == t->size(4) && t->stride(2) == t->size(3) * t->size(4), op,
                ": a page must be contiguous");
    const int64_t es = t->element_size();
    TORCH_CHECK(t->size(4) * es % 16 == 0 && t->stride(0) * es % 16 == 0 && t->stride(1) * es % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                op, ": rows of a page must be 16-byte aligned multiples of 16 bytes");
  }
  CopyArgs a{};
  const int64_t es = k.element_size();
  a.k = static_cast<char*>(k.data_ptr());
  a.v = static_cast<char*>(v.data_ptr());
  a.k_layer = k.stride(0) * es;
  a.k_page = k.stride(1) * es;
  a.v_layer = v.stride(0) * es;
  a.v_page = v.stride(1) * es;
  a.layers = int(k.size(0));
  a.pages = int(k.size(1));
  a.heads = int(k.size(2));
  a.page = int(k.size(3));
  a.row_bytes = int(k.size(4) * es);
  a.err = error_word();
  return a;
}

void launch_copy(const CopyArgs& a) {
  const int64_t units = int64_t(a.n) * a.layers * 2 * a.heads;
  if (units == 0) return;
  // Four rounds of CTAs, so that one that starts late (its SM still held by the state
  // kernel) does not end late: with one round of longer CTAs, 252 forks took 185 us
  // instead of 133.
  const int64_t blocks = std::min<int64_t>((units + kCopyThreads / 32 - 1) / (kCopyThreads / 32), 148 * 32);
  TORCH_CHECK(launch_early(copy_pages_kernel, dim3(unsigned(blocks)), dim3(kCopyThreads), 0,
                           at::cuda::getCurrentCUDAStream(), a) == cudaSuccess, "copy_pages launch failed");
}

// One CTA while each of its threads has a few entries of the state to read (up to 32
// of table, lens and refs), else a cluster: a cluster's barriers cost more than it
// reads faster. 7 forks and the room for their next token take 11.8 us of GPU time in
// three launches with one CTA, and took 16.7 us with eight (12 slots of 32 pages).
template <typename... KArgs, typename... Args>
void launch_team(const PageState& s, const char* op, void (*one)(KArgs...), void (*eight)(KArgs...), Args... args) {
  const bool small = int64_t(s.slots) * s.width + s.slots + s.pages <= 32 * kMetaThreads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(small ? 1 : kMetaCtas);
  cfg.blockDim = dim3(kMetaThreads);
  cfg.stream = at::cuda::getCurrentCUDAStream();
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = small ? 1 : kMetaCtas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  TORCH_CHECK(cudaLaunchKernelEx(&cfg, small ? one : eight, s, args...) == cudaSuccess, op, " launch failed");
}

torch::Tensor workspace(const torch::Tensor& like, int64_t ints) {
  return torch::empty({kListAt + ints}, like.options());
}

}  // namespace

void pages_fork(torch::Tensor k, torch::Tensor v, torch::Tensor table, torch::Tensor lens, torch::Tensor refs,
                torch::Tensor parents, torch::Tensor children, torch::Tensor table_out, torch::Tensor lens_out,
                torch::Tensor refs_out) {
  CopyArgs c = pools_of(k, v, table, "fork_pages");
  const PageState s = state_of(table, lens, refs, table_out, lens_out, refs_out, c.page, "fork_pages");
  TORCH_CHECK(c.pages == s.pages, "fork_pages: refs counts ", num(s.pages), " pages, the pool has ", num(c.pages));
  check_int_vec(parents, "fork_pages: parents", table);
  check_int_vec(children, "fork_pages: children", table);
  TORCH_CHECK(parents.dim() == 1 && parents.sizes() == children.sizes(), "fork_pages: one parent for each child");
  const int n = int(parents.size(0));
  const at::cuda::CUDAGuard guard(table.device());
  auto ws = workspace(table, s.slots + 5 * int64_t(n));
  int* w = ws.data_ptr<int>();
  launch_team(s, "fork_pages", fork_meta_kernel<1>, fork_meta_kernel<kMetaCtas>, parents.data_ptr<int>(),
              children.data_ptr<int>(), n, w);
  c.src = w + kListAt + s.slots + n;
  c.dst = c.src + n;
  c.rows = c.dst + n;
  c.n = n;
  launch_copy(c);
}

void pages_grow(torch::Tensor table, torch::Tensor lens, torch::Tensor refs, torch::Tensor add, int64_t page,
                torch::Tensor table_out, torch::Tensor lens_out, torch::Tensor refs_out,
                c10::optional<torch::Tensor> room) {
  const PageState s = state_of(table, lens, refs, table_out, lens_out, refs_out, page, "grow_pages");
  check_int_vec(add, "grow_pages: add", table);
  TORCH_CHECK(add.sizes() == lens.sizes(), "grow_pages: add must have one entry for each slot");
  const at::cuda::CUDAGuard guard(table.device());
  auto ws = workspace(table, int64_t(s.pages) + s.slots);
  launch_team(s, "grow_pages", grow_meta_kernel<1>, grow_meta_kernel<kMetaCtas>, add.data_ptr<int>(),
              room_of(room, lens, "grow_pages"), ws.data_ptr<int>());
}

void pages_free(torch::Tensor table, torch::Tensor lens, torch::Tensor refs, torch::Tensor seqs,
                torch::Tensor table_out, torch::Tensor lens_out, torch::Tensor refs_out,
                c10::optional<torch::Tensor> room) {
  const PageState s = state_of(table, lens, refs, table_out, lens_out, refs_out, 1, "free_pages");
  check_int_vec(seqs, "free_pages: seqs", table);
  TORCH_CHECK(seqs.dim() == 1, "free_pages: seqs must be a vector");
  const at::cuda::CUDAGuard guard(table.device());
  launch_team(s, "free_pages", free_meta_kernel<1>, free_meta_kernel<kMetaCtas>, seqs.data_ptr<int>(),
              int(seqs.size(0)), room_of(room, lens, "free_pages"));
}

void pages_compact(torch::Tensor k, torch::Tensor v, torch::Tensor table, torch::Tensor lens, torch::Tensor refs,
                   torch::Tensor table_out, torch::Tensor lens_out, torch::Tensor refs_out) {
  CopyArgs c = pools_of(k, v, table, "compact_pages");
  const PageState s = state_of(table, lens, refs, table_out, lens_out, refs_out, c.page, "compact_pages");
  TORCH_CHECK(c.pages == s.pages, "compact_pages: refs counts ", num(s.pages), " pages, the pool has ", num(c.pages));
  const at::cuda::CUDAGuard guard(table.device());
  auto ws = workspace(table, 4 * int64_t(s.pages));
  int* w = ws.data_ptr<int>();
  launch_team(s, "compact_pages", compact_meta_kernel<1>, compact_meta_kernel<kMetaCtas>, w);
  c.src = w + kListAt;
  c.dst = c.src + s.pages;
  c.count = w + kWsPairs;
  c.n = s.pages / 2;  // a move needs a page in use above and a free one below
  launch_copy(c);
}

// Pages dst[i] = pages src[i] of every layer, k and v; pairs with a negative
// source are skipped. No page may be both a source and a target.
void pages_copy(torch::Tensor k, torch::Tensor v, torch::Tensor src, torch::Tensor dst) {
  TORCH_CHECK(src.is_cuda(), "copy_pages: src must be on a GPU");
  CopyArgs c = pools_of(k, v, src, "copy_pages");
  check_int_vec(src, "copy_pages: src", src);
  check_int_vec(dst, "copy_pages: dst", src);
  TORCH_CHECK(src.dim() == 1 && src.sizes() == dst.sizes(), "copy_pages: one target for each source");
  const at::cuda::CUDAGuard guard(src.device());
  c.src = src.data_ptr<int>();
  c.dst = dst.data_ptr<int>();
  c.n = int(src.size(0));
  launch_copy(c);
}

}  // namespace nk
