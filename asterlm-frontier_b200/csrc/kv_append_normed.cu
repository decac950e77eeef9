// Append of new keys and values to a paged grouped-query cache with the norms of queries and keys: each head is
// divided by its root mean square and weighted, then rotated by its position, in one pass from a projection's rows to
// the pages (csrc/kv_append.cu is the append without norms).
//
//   y = x / sqrt(mean(x^2) + eps) w  for each head of q and of k (where weights are given), fp32;
//   the first rotary_dim dims of y turn in pairs by cos[p][j], sin[p][j]; one rounding at the end.
// p is the row's place behind the sequence's cached tokens, or positions[row] (a drafted node's place in the
// pages goes by its number, its position by its depth).
//
// 2 bytes in and 2 out a value, and some ten operations.  A head is held by the lanes of one
// group, 16 dims each (two 16-byte vectors whose pairs share eight cos and sin values), so its sum of squares
// is a few shuffles; a group walks over heads, and CTAs over rows with the weights in shared memory (in registers, 112
// of them a thread, 16,387 rows took 107 us instead of 84).
// Measured: 16,387 rows of 32 + 8 + 8 heads of 128 dims (64 of them turned, interleaved), 407 MB in and out: 84 us, 4.84 TB/s (0.74 of
// the measured copy bandwidth; the append without norms takes 72).  What bounds it is the pipe of shared memory and loads, busy 133,000 of an SM's
// 157,000 cycles: lanes of a head read weights 32 or 64 bytes apart, and of 10.8 million accesses to shared memory 8.2 million are repeats for
// bank conflicts.  32 rows 6.2 us, a launch.
#include "asterq_internal.h"
#include "common.cuh"
#include "launch.cuh"

namespace asterq {
namespace kvn {

constexpr int kThreads = 256;

template <bool kF16>
ASTERQ_DEVICE float2 unpack2(uint32_t w) {
  return kF16 ? unpack_half2(w) : unpack_bf162(w);
}
template <bool kF16>
ASTERQ_DEVICE uint32_t pack2(float lo, float hi) {
  return kF16 ? pack_half2(lo, hi) : pack_bf162(lo, hi);
}

// The last s in [0, n) with off[s] <= row (off[0] <= row), by all lanes of a warp.
ASTERQ_DEVICE int find_sequence(const int* __restrict__ off, int n, long long row) {
  const int lane = threadIdx.x & 31;
  int lo = 0, len = n;
  while (len > 1) {
    const int step = (len + 31) / 32;
    const bool below = lane * step < len && (long long)__ldg(off + lo + lane * step) <= row;
    const int skip = (max(__popc(__ballot_sync(0xffffffffu, below)), 1) - 1) * step;
    lo += skip;
    len = min(step, len - skip);
  }
  return lo;
}

template <bool kF16>
__global__ void __launch_bounds__(kThreads) append_kernel(const asterq_kv_append_normed_params p, int rows_per_block, int lanes) {
  const int D = p.head_dim, units = D / 16, turn = p.rotary_dim / 16;
  const int per_row = kThreads / rows_per_block;  // threads of one row: whole warps
  const int sub = threadIdx.x / per_row, r = threadIdx.x % per_row;
  const int u = r % lanes, g = r / lanes, groups = per_row / lanes;  // a head's lanes: a power of two
  const bool works = u < units;
  const int n_q = p.q ? p.n_heads : 0, n_all = n_q + 2 * p.n_kv_heads;
  const bool half = !p.interleaved && u < turn;
  const float per_dim = 1.0f / (float)D;
  const int d0 = !works ? 0 : half ? 8 * u : 16 * u, d1 = !works ? 8 : half ? p.rotary_dim / 2 + 8 * u : 16 * u + 8;
  // the weights in shared memory: 32 registers of them cost half of the CTAs that an SM holds
  __shared__ __align__(16) float weight_s[2][512];
  for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
    const int of = i >= D, d = i - of * D;
    const void* w = of ? p.k_norm : p.q_norm;
    if (w)
      weight_s[of][d] = p.norm_dtype == ASTERQ_DTYPE_F32 ? __ldg(static_cast<const float*>(w) + d)
                                                         : unpack2<kF16>(__ldg(static_cast<const uint16_t*>(w) + d)).x;
  }
  __syncthreads();

  for (long long row = (long long)blockIdx.x * rows_per_block + sub; row < p.n_rows; row += (long long)gridDim.x * rows_per_block) {
    auto source = [&](int h) -> const uint16_t* {
      if (h < n_q) return (const uint16_t*)p.q + row * p.q_row_stride + (long long)h * p.q_head_stride;
      h -= n_q;
      if (h < p.n_kv_heads) return (const uint16_t*)p.k + row * p.k_row_stride + (long long)h * p.k_head_stride;
      return (const uint16_t*)p.v + row * p.v_row_stride + (long long)(h - p.n_kv_heads) * p.v_head_stride;
    };
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (works && g < n_all) {
      const uint16_t* src = source(g);
      a = ldg_nc_v4(src + d0);
      b = ldg_nc_v4(src + d1);
    }
    // where the row belongs; every warp looks it up for itself
    if ((long long)__ldg(p.row_offsets) > row || row >= (long long)__ldg(p.row_offsets + p.n_seqs)) continue;
    const int s = find_sequence(p.row_offsets, p.n_seqs, row);
    const int length = __ldg(p.lengths + s);
    if (length < 0) continue;  // an empty slot
    const long long begin = __ldg(p.row_offsets + s), place = (long long)length + (row - begin);
    const long long col = place / p.page_tokens;
    const int inside = (int)(place - col * p.page_tokens);
    const long long pos = p.positions ? (long long)__ldg(p.positions + row) : place;
    int page = -1;
    // the search finds a sequence that the row is not of where offsets are out of order
    if (row >= begin && row < (long long)__ldg(p.row_offsets + s + 1) && col < p.max_pages)
      page = __ldg(p.page_table + (long long)s * p.max_pages + col);
    if (page < 0 || page >= p.n_pages || (turn && (pos < 0 || pos >= p.n_positions))) {
      if (p.status && (threadIdx.x & 31) == 0) atomicMax(p.status, 1);
      continue;
    }
    float c[8], sn[8];
    if (works && u < turn) {
      const float4* cp = reinterpret_cast<const float4*>(p.cos + pos * (p.rotary_dim / 2) + 8 * u);
      const float4* sp = reinterpret_cast<const float4*>(p.sin + pos * (p.rotary_dim / 2) + 8 * u);
      *reinterpret_cast<float4*>(c) = __ldg(cp);
      *reinterpret_cast<float4*>(c + 4) = __ldg(cp + 1);
      *reinterpret_cast<float4*>(sn) = __ldg(sp);
      *reinterpret_cast<float4*>(sn + 4) = __ldg(sp + 1);
    }
    const long long page0 = (long long)page * p.n_kv_heads;
    for (int h0 = 0; h0 < n_all; h0 += groups) {  // every lane all rounds: a head's lanes meet in shuffles
      const int h = h0 + g;
      uint4 na = a, nb = b;
      if (works && h + groups < n_all) {
        const uint16_t* src = source(h + groups);
        na = ldg_nc_v4(src + d0);
        nb = ldg_nc_v4(src + d1);
      }
      const bool is_q = h < n_q, is_k = !is_q && h < n_q + p.n_kv_heads;
      const bool normed = (is_q && p.q_norm) || (is_k && p.k_norm);
      uint32_t* x = reinterpret_cast<uint32_t*>(&a);
      uint32_t* y = reinterpret_cast<uint32_t*>(&b);
      float scale = 1.0f;
      if (__any_sync(0xffffffffu, normed)) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 xf = unpack2<kF16>(x[i]), yf = unpack2<kF16>(y[i]);
          sum = fmaf(xf.x, xf.x, fmaf(xf.y, xf.y, fmaf(yf.x, yf.x, fmaf(yf.y, yf.y, sum))));
        }
        if (!works) sum = 0.0f;
        for (int d = 1; d < lanes; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        scale = rsqrtf(sum * per_dim + p.norm_eps);
      }
      if (works && h < n_all) {
        const bool turns = u < turn && (is_q || is_k);
        if (normed || turns) {  // values go as they came
          const float2* wx = reinterpret_cast<const float2*>(weight_s[is_q ? 0 : 1] + d0);
          const float2* wy = reinterpret_cast<const float2*>(weight_s[is_q ? 0 : 1] + d1);
          // two pairs at a time, so that few are held in 32 bits
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float2 xf = unpack2<kF16>(x[i]), yf = unpack2<kF16>(y[i]);
            if (normed) {
              const float2 wa = wx[i], wb = wy[i];
              xf = make_float2(xf.x * scale * wa.x, xf.y * scale * wa.y);
              yf = make_float2(yf.x * scale * wb.x, yf.y * scale * wb.y);
            }
            if (turns && half) {
              x[i] = pack2<kF16>(xf.x * c[2 * i] - yf.x * sn[2 * i], xf.y * c[2 * i + 1] - yf.y * sn[2 * i + 1]);
              y[i] = pack2<kF16>(yf.x * c[2 * i] + xf.x * sn[2 * i], yf.y * c[2 * i + 1] + xf.y * sn[2 * i + 1]);
            } else if (turns) {
              x[i] = pack2<kF16>(xf.x * c[i] - xf.y * sn[i], xf.y * c[i] + xf.x * sn[i]);
              y[i] = pack2<kF16>(yf.x * c[4 + i] - yf.y * sn[4 + i], yf.y * c[4 + i] + yf.x * sn[4 + i]);
            } else {
              x[i] = pack2<kF16>(xf.x, xf.y);
              y[i] = pack2<kF16>(yf.x, yf.y);
            }
          }
        }
        uint16_t* dst;
        if (is_q) {
          dst = (uint16_t*)p.q_out + (row * n_q + h) * D;
        } else {
          const int kv = h - n_q, hk = is_k ? kv : kv - p.n_kv_heads;
          dst = (uint16_t*)(is_k ? p.k_pool : p.v_pool) + ((page0 + hk) * p.page_tokens + inside) * D;
        }
        *reinterpret_cast<uint4*>(dst + d0) = a;
        *reinterpret_cast<uint4*>(dst + d1) = b;
      }
      a = na;
      b = nb;
    }
  }
}

}  // namespace kvn
}  // namespace asterq

using namespace asterq;

extern "C" int asterq_kv_append_normed(const asterq_kv_append_normed_params* p, void* stream) {
  clear_error();
  if (!p) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_append_normed: null parameters");
  if (p->n_seqs < 0 || p->n_rows < 0 || p->n_pages < 0 || p->max_pages < 0 || p->n_kv_heads <= 0 || p->n_heads < 0 ||
      p->n_positions < 0 || p->page_tokens <= 0)
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_append_normed: bad sizes");
  if (p->dtype != ASTERQ_DTYPE_BF16 && p->dtype != ASTERQ_DTYPE_F16)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "kv_append_normed: dtype %d: bf16 or f16", p->dtype);
  if ((p->q_norm || p->k_norm) && p->norm_dtype != p->dtype && p->norm_dtype != ASTERQ_DTYPE_F32)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "kv_append_normed: weights are of the rows' type or f32");
  if (p->head_dim <= 0 || p->head_dim % 16 || p->head_dim > 512)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "kv_append_normed: head_dim %d must be a multiple of 16 up to 512", p->head_dim);
  if (p->rotary_dim < 0 || p->rotary_dim > p->head_dim || p->rotary_dim % 16)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "kv_append_normed: rotary_dim %d must be a multiple of 16 up to head_dim",
                     p->rotary_dim);
  if (!(p->norm_eps >= 0.0f)) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_append_normed: negative norm_eps");
  if (p->n_rows == 0 || p->n_seqs == 0) return ASTERQ_OK;
  if (p->n_rows > 0x7fffffffLL) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_append_normed: more than 2^31 - 1 rows");
  if (!p->k || !p->v || !p->k_pool || !p->v_pool || !p->lengths || !p->row_offsets ||
      (p->max_pages > 0 && !p->page_table) || (p->q && (!p->q_out || p->n_heads <= 0)) ||
      (p->rotary_dim > 0 && (!p->cos || !p->sin)))
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "kv_append_normed: null pointer");
  const void* vec[] = {p->q, p->k, p->v, p->cos, p->sin, p->q_out, p->k_pool, p->v_pool};
  for (const void* ptr : vec)
    if (reinterpret_cast<uintptr_t>(ptr) & 15)
      return set_error(ASTERQ_ERR_MISALIGNED, "kv_append_normed: arrays must be 16-byte aligned");
  const int64_t strides[] = {p->q ? p->q_row_stride : 0, p->q ? p->q_head_stride : 0, p->k_row_stride,
                             p->k_head_stride, p->v_row_stride, p->v_head_stride};
  for (int64_t st : strides)
    if (st % 8) return set_error(ASTERQ_ERR_MISALIGNED, "kv_append_normed: row and head strides must be multiples of 8");
  int dev = 0;
  const int sms = current_sms(&dev);
  if (sms <= 0) return set_error(ASTERQ_ERR_CUDA, "kv_append_normed: no CUDA device");
  int lanes = 1;
  while (lanes < p->head_dim / 16) lanes *= 2;
  // Threads of a row: for all its heads at once while rows are few, 64 for many.  With 32 + 8 + 8 heads of 128 dims, at
  // once and by 64: 300 rows 6.2 and 8.3 us, 600 8.4 and 10.3, 1200 12.4 and 10.3, 4800 33 and 26.
  // CTAs an SM: 4 84.3 us, 8 86.0, 16 88.1 (16,387 rows); one for each four rows 90.5.
  const int64_t items = (int64_t)lanes * ((p->q ? p->n_heads : 0) + 2 * p->n_kv_heads);
  int per_row = kvn::kThreads;
  while (per_row > 64 && (per_row / 2 >= items || p->n_rows >= 1000)) per_row /= 2;
  const int rows_per_block = kvn::kThreads / per_row;
  const int64_t blocks = (p->n_rows + rows_per_block - 1) / rows_per_block, most = (int64_t)sms * 4;
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (p->dtype == ASTERQ_DTYPE_F16)
    kvn::append_kernel<true><<<grid, kvn::kThreads, 0, s>>>(*p, rows_per_block, lanes);
  else
    kvn::append_kernel<false><<<grid, kvn::kThreads, 0, s>>>(*p, rows_per_block, lanes);
  return check_launch("kv_append_normed");
}
