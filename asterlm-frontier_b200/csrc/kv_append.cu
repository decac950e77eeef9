// Append of new keys and values to a paged grouped-query cache, keys and queries rotated by
// their position on the way (the cache that csrc/paged_attention.cu reads).
//
// Row r of sequence s (row_offsets[s] <= r < row_offsets[s + 1]) has position
// p = lengths[s] + r - row_offsets[s].  The first rotary_dim dims of each head of q and k turn
// in pairs (x, y): x' = x c - y s, y' = y c + x s with c = cos[p][j], s = sin[p][j], computed in
// fp32 and rounded once; pair j is dims (j, j + rotary_dim / 2), or (2j, 2j + 1) interleaved.
//
// Measured: 16411 prompt rows of 32 query and 2 x 8 kv heads of 128 dims in 72 us, 5.7 TB/s; 256 single tokens 3.9 us
// and 8 of them 3.0, which is the latency of a launch and four dependent loads.
#include "asterq_internal.h"
#include "common.cuh"

namespace asterq {
namespace kva {

constexpr int kThreads = 256;

template <bool kF16>
ASTERQ_DEVICE float2 unpack2(uint32_t w) {
  return kF16 ? unpack_half2(w) : unpack_bf162(w);
}
template <bool kF16>
ASTERQ_DEVICE uint32_t pack2(float lo, float hi) {
  return kF16 ? pack_half2(lo, hi) : pack_bf162(lo, hi);
}

// The last s in [0, n) with off[s] <= row (off[0] <= row), by all lanes of a warp: 32 probes a
// round, so two dependent loads find a row among a thousand sequences.
ASTERQ_DEVICE int find_sequence(const int* __restrict__ off, int n, long long row) {
  const int lane = threadIdx.x & 31;
  int lo = 0, len = n;
  while (len > 1) {
    const int step = (len + 31) / 32;
    const int at = lo + lane * step;
    const bool below = lane * step < len && (long long)__ldg(off + at) <= row;
    // off[lo] <= row holds throughout, so the count is at least one
    const int k = max(__popc(__ballot_sync(0xffffffffu, below)), 1) - 1;
    const int skip = k * step;
    lo += skip;
    len = min(step, len - skip);
  }
  return lo;
}

// One thread holds one rotation unit of 16 dims (two 16-byte vectors, whose pairs share eight
// cos and sin values) of one row and walks over heads, so the cos and sin values are read once
// for all heads.  The kernel moves 2 bytes in and 2 out for each value and a few multiplies: it
// is bound by memory, or for a few rows by the chain row -> sequence -> position -> cos, during
// which the first head's values are already on their way.
template <bool kF16>
__global__ void __launch_bounds__(kThreads) append_kernel(const asterq_kv_append_params p, int rows_per_block) {
  const int D = p.head_dim, units = D / 16, turn = p.rotary_dim / 16;
  const int per_row = kThreads / rows_per_block;  // threads of one row: whole warps
  const int sub = threadIdx.x / per_row, r = threadIdx.x % per_row;
  const int groups = per_row / units;  // heads side by side
  const int u = r % units, g = r / units;
  const long long row = (long long)blockIdx.x * rows_per_block + sub;
  if (row >= p.n_rows) return;  // whole warps
  const int n_q = p.q ? p.n_heads : 0, n_all = n_q + 2 * p.n_kv_heads;

  const bool half = !p.interleaved && u < turn;
  const int d0 = half ? 8 * u : 16 * u, d1 = half ? p.rotary_dim / 2 + 8 * u : 16 * u + 8;
  auto source = [&](int h) -> const uint16_t* {
    if (h < n_q) return (const uint16_t*)p.q + row * p.q_row_stride + (long long)h * p.q_head_stride;
    h -= n_q;
    if (h < p.n_kv_heads) return (const uint16_t*)p.k + row * p.k_row_stride + (long long)h * p.k_head_stride;
    return (const uint16_t*)p.v + row * p.v_row_stride + (long long)(h - p.n_kv_heads) * p.v_head_stride;
  };
  uint4 a = make_uint4(0, 0, 0, 0), b = a;
  const bool works = g < groups;
  if (works && g < n_all) {
    const uint16_t* src = source(g);
    a = ldg_nc_v4(src + d0);
    b = ldg_nc_v4(src + d1);
  }

  // where the row belongs; every warp looks it up for itself
  if ((long long)__ldg(p.row_offsets) > row || row >= (long long)__ldg(p.row_offsets + p.n_seqs)) return;
  const int s = find_sequence(p.row_offsets, p.n_seqs, row);
  const int length = __ldg(p.lengths + s);
  if (length < 0) return;  // an empty slot
  const long long begin = __ldg(p.row_offsets + s), pos = (long long)length + (row - begin);
  const long long col = pos / p.page_tokens;
  const int at = (int)(pos - col * p.page_tokens);
  int page = -1;
  // the search finds a sequence that the row is not of where offsets are out of order
  if (row >= begin && row < (long long)__ldg(p.row_offsets + s + 1) && col < p.max_pages)
    page = __ldg(p.page_table + (long long)s * p.max_pages + col);
  if (page < 0 || page >= p.n_pages || (turn && pos >= p.n_positions)) {
    if (p.status && (threadIdx.x & 31) == 0) atomicMax(p.status, 1);
    return;
  }
  if (!works) return;

  float c[8], sn[8];
  if (u < turn) {
    const float4* cp = reinterpret_cast<const float4*>(p.cos + pos * (p.rotary_dim / 2) + 8 * u);
    const float4* sp = reinterpret_cast<const float4*>(p.sin + pos * (p.rotary_dim / 2) + 8 * u);
    *reinterpret_cast<float4*>(c) = __ldg(cp);
    *reinterpret_cast<float4*>(c + 4) = __ldg(cp + 1);
    *reinterpret_cast<float4*>(sn) = __ldg(sp);
    *reinterpret_cast<float4*>(sn + 4) = __ldg(sp + 1);
  }
  const long long page0 = (long long)page * p.n_kv_heads;
  for (int h = g; h < n_all; h += groups) {
    // the next head's values are loaded before this one's are turned and stored
    uint4 na = a, nb = b;
    if (h + groups < n_all) {
      const uint16_t* src = source(h + groups);
      na = ldg_nc_v4(src + d0);
      nb = ldg_nc_v4(src + d1);
    }
    if (u < turn && h < n_q + p.n_kv_heads) {
      uint32_t* x = reinterpret_cast<uint32_t*>(&a);
      uint32_t* y = reinterpret_cast<uint32_t*>(&b);
      if (half) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 xf = unpack2<kF16>(x[i]), yf = unpack2<kF16>(y[i]);
          x[i] = pack2<kF16>(xf.x * c[2 * i] - yf.x * sn[2 * i], xf.y * c[2 * i + 1] - yf.y * sn[2 * i + 1]);
          y[i] = pack2<kF16>(yf.x * c[2 * i] + xf.x * sn[2 * i], yf.y * c[2 * i + 1] + xf.y * sn[2 * i + 1]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 xf = unpack2<kF16>(x[i]), yf = unpack2<kF16>(y[i]);
          x[i] = pack2<kF16>(xf.x * c[i] - xf.y * sn[i], xf.y * c[i] + xf.x * sn[i]);
          y[i] = pack2<kF16>(yf.x * c[4 + i] - yf.y * sn[4 + i], yf.y * c[4 + i] + yf.x * sn[4 + i]);
        }
      }
    }
    uint16_t* dst;
    if (h < n_q) {
      dst = (uint16_t*)p.q_out + (row * n_q + h) * D;
    } else {
      const int kv = h - n_q, hk = kv < p.n_kv_heads ? kv : kv - p.n_kv_heads;
      dst = (uint16_t*)(kv < p.n_kv_heads ? p.k_pool : p.v_pool) + ((page0 + hk) * p.page_tokens + at) * D;
    }
    *reinterpret_cast<uint4*>(dst + d0) = a;
    *reinterpret_cast<uint4*>(dst + d1) = b;
    a = na;
    b = nb;
  }
}

}  // namespace kva
}  // namespace asterq

using namespace asterq;

extern "C" int asterq_kv_append(const asterq_kv_append_params* p, void* stream) {
  clear_error();
  if (!p) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_append: null parameters");
  if (p->n_seqs < 0 || p->n_rows < 0 || p->n_pages < 0 || p->max_pages < 0 || p->n_kv_heads <= 0 || p->n_heads < 0 ||
      p->n_positions < 0 || p->page_tokens <= 0)
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_append: bad sizes");
  if (p->dtype != ASTERQ_DTYPE_BF16 && p->dtype != ASTERQ_DTYPE_F16)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "kv_append: dtype %d: bf16 or f16", p->dtype);
  if (p->head_dim <= 0 || p->head_dim % 16 || p->head_dim > 512)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "kv_append: head_dim %d must be a multiple of 16 up to 512", p->head_dim);
  if (p->rotary_dim < 0 || p->rotary_dim > p->head_dim || p->rotary_dim % 16)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "kv_append: rotary_dim %d must be a multiple of 16 up to head_dim",
                     p->rotary_dim);
  if (p->n_rows == 0 || p->n_seqs == 0) return ASTERQ_OK;
  if (p->n_rows > 0x7fffffffLL) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_append: more than 2^31 - 1 rows");
  if (!p->k || !p->v || !p->k_pool || !p->v_pool || !p->lengths || !p->row_offsets ||
      (p->max_pages > 0 && !p->page_table) || (p->q && (!p->q_out || p->n_heads <= 0)) ||
      (p->rotary_dim > 0 && (!p->cos || !p->sin)))
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_append: null pointer");
  const void* vec[] = {p->q, p->k, p->v, p->cos, p->sin, p->q_out, p->k_pool, p->v_pool};
  for (const void* ptr : vec)
    if (reinterpret_cast<uintptr_t>(ptr) & 15)
      return set_error(ASTERQ_ERR_MISALIGNED, "kv_append: arrays must be 16-byte aligned");
  const int64_t strides[] = {p->q ? p->q_row_stride : 0, p->q ? p->q_head_stride : 0, p->k_row_stride,
                             p->k_head_stride, p->v_row_stride, p->v_head_stride};
  for (int64_t st : strides)
    if (st % 8) return set_error(ASTERQ_ERR_MISALIGNED, "kv_append: row and head strides must be multiples of 8");
  // Threads of a row: enough for all its heads at once while rows are few (a decode step's latency is one
  // pass of each thread), 64 from 600 rows on, where the cos and sin values are then shared by several heads
  // of a thread and a warp's loads stay in one row.  Measured at 32 + 2 x 8 heads of 128, 64 threads against
  // all: 400 rows 5.1 against 4.5 us, 600 rows 5.7 against 6.2, 2000 rows 9.3 against 13.3, 16411 rows 73
  // against 93; at heads of 64, 512 rows 5.5 against 4.8, 1024 rows 6.1 against 7.5.
  const int units = p->head_dim / 16;
  const int64_t items = (int64_t)units * ((p->q ? p->n_heads : 0) + 2 * p->n_kv_heads);
  int per_row = kva::kThreads;
  while (per_row > 64 && per_row / 2 >= units && (per_row / 2 >= items || p->n_rows >= 600)) per_row /= 2;
  const int rows_per_block = kva::kThreads / per_row;
  const unsigned grid = (unsigned)((p->n_rows + rows_per_block - 1) / rows_per_block);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (p->dtype == ASTERQ_DTYPE_F16)
    kva::append_kernel<true><<<grid, kva::kThreads, 0, s>>>(*p, rows_per_block);
  else
    kva::append_kernel<false><<<grid, kva::kThreads, 0, s>>>(*p, rows_per_block);
  return check_launch("kv_append");
}
