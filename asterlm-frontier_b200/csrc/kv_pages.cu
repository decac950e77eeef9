// The content of paged key/value pools moved, in all layers of a stack by one launch (64 layers each):
//   keep   accepted rows of a draft closed up behind the cached tokens: place length + kept[i] to length + i
//   copy   whole pages to others (a forked sequence's last page, pages moved together)
// Bytes in and bytes out are all there is to it: both move 16-byte vectors, several loads of a thread under way.
// Measured: 60 pages of 64 tokens, 8 heads of 128 f16 dims and 24 layers, 755 MB in and out: 113 us, 6.6 TB/s, the measured copy
// bandwidth; 48 trees' accepted rows in 16 layers, 25 MB: 8.3 us.
#include "asterq_internal.h"
#include "common.cuh"

namespace asterq {
namespace kvp {

constexpr int kLayers = 64;  // of one launch: their addresses are in its parameters
constexpr int kThreads = 256;

struct Pools {
  uint4* k[kLayers];
  uint4* v[kLayers];
};

struct Keep {
  const int* page_table;
  const int* lengths;
  const int* row_offsets;
  const int* kept;
  const int* n_kept;
  int* status;
  long long n_rows, n_pages;
  int page_tokens, max_pages, n_kv_heads, vecs;  // vecs: 16-byte vectors of a head
};

// One CTA moves a sequence's rows in one layer; a thread its vectors of a head of keys or values, rows in
// their order.  kept ascends, so row i goes to a place that no later row comes from: kept[j] >= j > i.
constexpr int kBatch = 8, kList = 128;
__global__ void __launch_bounds__(kThreads) keep_kernel(const __grid_constant__ Pools pools, const Keep a) {
  const int s = blockIdx.y, layer = blockIdx.x, tid = threadIdx.x;
  __shared__ long long from_s[kList], to_s[kList];  // of a run of rows: page * heads * page_tokens + place in the page; -1: not moved
  const int begin = __ldg(a.row_offsets + s), end = __ldg(a.row_offsets + s + 1), length = __ldg(a.lengths + s);
  const int n = __ldg(a.n_kept + s);
  if (length < 0 || n <= 0) return;
  bool bad = begin < 0 || end < begin || end > a.n_rows || n > end - begin;
  if (!bad)
    for (int i = tid; i < n; i += kThreads) {
      const int k = __ldg(a.kept + begin + i), before = i > 0 ? __ldg(a.kept + begin + i - 1) : -1;
      bad = bad || k <= before || k >= end - begin;
    }
  if (__syncthreads_or(bad)) {
    if (tid == 0 && a.status) atomicMax(a.status, 1);
    return;
  }
  const long long head_step = (long long)a.page_tokens * a.vecs;
  const int per_pool = a.n_kv_heads * a.vecs;
  for (int first = 0; first < n; first += kList) {
    const int count = min(kList, n - first);
    __syncthreads();
    for (int i = tid; i < count; i += kThreads) {
      const int k = __ldg(a.kept + begin + first + i);
      long long place[2] = {(long long)length + k, (long long)length + first + i}, at[2];
      bool fine = true;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const long long column = place[e] / a.page_tokens;
        int page = -1;
        if (column < a.max_pages) page = __ldg(a.page_table + (long long)s * a.max_pages + column);
        fine = fine && page >= 0 && page < a.n_pages;
        at[e] = (long long)page * a.n_kv_heads * a.page_tokens + (place[e] - column * a.page_tokens);
      }
      if (!fine && a.status) atomicMax(a.status, 1);
      from_s[i] = fine && k != first + i ? at[0] : -1;
      to_s[i] = at[1];
    }
    __syncthreads();
    for (int item = tid; item < 2 * per_pool; item += kThreads) {
      const int in_pool = item % per_pool, head = in_pool / a.vecs;
      uint4* pool = (item < per_pool ? pools.k[layer] : pools.v[layer]) + head * head_step + (in_pool - head * a.vecs);
      for (int i0 = 0; i0 < count; i0 += kBatch) {
        uint4 w[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
          if (i0 + b < count && from_s[i0 + b] >= 0) w[b] = pool[from_s[i0 + b] * a.vecs];
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
          if (i0 + b < count && from_s[i0 + b] >= 0) pool[to_s[i0 + b] * a.vecs] = w[b];
      }
    }
  }
}

// One CTA copies kChunk vectors of a page of keys or values in one layer.
constexpr int kChunk = 2048;  // 32 KB
__global__ void __launch_bounds__(kThreads)
    copy_kernel(const __grid_constant__ Pools pools, const int2* __restrict__ pairs, int n_pairs, long long n_pages,
                long long page_vecs, int* status) {
  const int2 me = __ldg(pairs + blockIdx.x);
  if (me.x < 0 || me.y < 0) return;  // left out
  // a page that two pairs write, or that one writes and another reads, would depend on the order: left out
  bool bad = me.x >= n_pages || me.y >= n_pages;
  for (int i = threadIdx.x; i < n_pairs; i += kThreads) {
    const int2 o = __ldg(pairs + i);
    if (i != (int)blockIdx.x && o.x >= 0 && o.y >= 0) bad = bad || o.y == me.y || o.x == me.y || o.y == me.x;
  }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0 && status) atomicMax(status, 1);
    return;
  }
  if (me.x == me.y) return;
  uint4* pool = blockIdx.y & 1 ? pools.v[blockIdx.y / 2] : pools.k[blockIdx.y / 2];
  const uint4* from = pool + me.x * page_vecs;
  uint4* to = pool + me.y * page_vecs;
  const long long first = (long long)blockIdx.z * kChunk + threadIdx.x;
  uint4 w[kChunk / kThreads];
#pragma unroll
  for (int k = 0; k < kChunk / kThreads; ++k)
    if (first + k * kThreads < page_vecs) w[k] = ldg_nc_v4(from + first + k * kThreads);
#pragma unroll
  for (int k = 0; k < kChunk / kThreads; ++k)
    if (first + k * kThreads < page_vecs) to[first + k * kThreads] = w[k];
}

static int check_pools(const char* what, int dtype, int n_layers, int n_kv_heads, int head_dim, int page_tokens,
                       int64_t n_pages, void* const* k, void* const* v) {
  if (n_layers < 0 || n_kv_heads <= 0 || page_tokens <= 0 || n_pages < 0)
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "%s: bad sizes", what);
  if (dtype != ASTERQ_DTYPE_BF16 && dtype != ASTERQ_DTYPE_F16)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "%s: dtype %d: bf16 or f16", what, dtype);
  if (head_dim <= 0 || head_dim % 8) return set_error(ASTERQ_ERR_UNSUPPORTED, "%s: head_dim %d must be a multiple of 8", what, head_dim);
  if (n_layers > 0 && (!k || !v)) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  for (int i = 0; i < n_layers; ++i) {
    if (!k[i] || !v[i]) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "%s: null pool of layer %d", what, i);
    if ((reinterpret_cast<uintptr_t>(k[i]) | reinterpret_cast<uintptr_t>(v[i])) & 15)
      return set_error(ASTERQ_ERR_MISALIGNED, "%s: pools must be 16-byte aligned", what);
  }
  return ASTERQ_OK;
}

static Pools some_layers(void* const* k, void* const* v, int first, int count) {
  Pools p = {};
  for (int i = 0; i < count; ++i) {
    p.k[i] = static_cast<uint4*>(k[first + i]);
    p.v[i] = static_cast<uint4*>(v[first + i]);
  }
  return p;
}

}  // namespace kvp
}  // namespace asterq

using namespace asterq;

extern "C" int asterq_kv_keep(const asterq_kv_keep_params* p, void* stream) {
  clear_error();
  if (!p) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_keep: null parameters");
  const int st = kvp::check_pools("kv_keep", p->dtype, p->n_layers, p->n_kv_heads, p->head_dim, p->page_tokens, p->n_pages,
                                  p->k_pools, p->v_pools);
  if (st != ASTERQ_OK) return st;
  if (p->n_seqs < 0 || p->n_rows < 0 || p->max_pages < 0)
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_keep: bad sizes");
  if (p->n_seqs > 65535) return set_error(ASTERQ_ERR_UNSUPPORTED, "kv_keep: more than 65535 sequences");
  if (p->n_seqs == 0 || p->n_layers == 0 || p->n_rows == 0) return ASTERQ_OK;
  if (!p->lengths || !p->row_offsets || !p->kept || !p->n_kept || (p->max_pages > 0 && !p->page_table))
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_keep: null pointer");
  kvp::Keep a;
  a.page_table = p->page_table;
  a.lengths = p->lengths;
  a.row_offsets = p->row_offsets;
  a.kept = p->kept;
  a.n_kept = p->n_kept;
  a.status = p->status;
  a.n_rows = p->n_rows;
  a.n_pages = p->n_pages;
  a.page_tokens = p->page_tokens;
  a.max_pages = p->max_pages;
  a.n_kv_heads = p->n_kv_heads;
  a.vecs = p->head_dim / 8;
  for (int first = 0; first < p->n_layers; first += kvp::kLayers) {
    const int count = p->n_layers - first < kvp::kLayers ? p->n_layers - first : kvp::kLayers;
    kvp::keep_kernel<<<dim3(count, p->n_seqs), kvp::kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
        kvp::some_layers(p->k_pools, p->v_pools, first, count), a);
  }
  return check_launch("kv_keep");
}

extern "C" int asterq_kv_copy_pages(const asterq_kv_copy_params* p, void* stream) {
  clear_error();
  if (!p) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_copy_pages: null parameters");
  const int st = kvp::check_pools("kv_copy_pages", p->dtype, p->n_layers, p->n_kv_heads, p->head_dim, p->page_tokens,
                                  p->n_pages, p->k_pools, p->v_pools);
  if (st != ASTERQ_OK) return st;
  if (p->n_pairs < 0) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_copy_pages: bad sizes");
  if (p->n_pairs == 0 || p->n_layers == 0) return ASTERQ_OK;
  if (!p->pairs) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_copy_pages: null pointer");
  if (reinterpret_cast<uintptr_t>(p->pairs) & 7)
    return set_error(ASTERQ_ERR_MISALIGNED, "kv_copy_pages: pairs must be 8-byte aligned");
  const long long vecs = (long long)p->n_kv_heads * p->page_tokens * (p->head_dim / 8);
  const long long chunks = (vecs + kvp::kChunk - 1) / kvp::kChunk;
  if (chunks > 65535) return set_error(ASTERQ_ERR_UNSUPPORTED, "kv_copy_pages: a page of more than 2 GB");
  for (int first = 0; first < p->n_layers; first += kvp::kLayers) {
    const int count = p->n_layers - first < kvp::kLayers ? p->n_layers - first : kvp::kLayers;
    kvp::copy_kernel<<<dim3(p->n_pairs, 2 * count, (unsigned)chunks), kvp::kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
        kvp::some_layers(p->k_pools, p->v_pools, first, count), reinterpret_cast<const int2*>(p->pairs), p->n_pairs,
        p->n_pages, vecs, p->status);
  }
  return check_launch("kv_copy_pages");
}
