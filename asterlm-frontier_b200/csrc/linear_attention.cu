// Linear attention with a decay for each head, state held in fp32 (sm_100a).
//
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   S [Dk][Dv] per (slot, head)
//
// scan_kernel walks the recurrence token by token: the form for single tokens, for prompts too short
// for the chunked form (csrc/linear_chunk.cu) and for the types that it does not take.
#include "linear.cuh"

namespace asterq {
namespace lin {

template <int kType>
ASTERQ_DEVICE float load1(const void* p, long long i) {
  if constexpr (kType == ASTERQ_DTYPE_F32) return __ldg(static_cast<const float*>(p) + i);
  if constexpr (kType == ASTERQ_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
template <int kType>
ASTERQ_DEVICE void store1(void* p, long long i, float x) {
  if constexpr (kType == ASTERQ_DTYPE_F32) static_cast<float*>(p)[i] = x;
  else if constexpr (kType == ASTERQ_DTYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(x);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}
template <int kType>
ASTERQ_DEVICE float4 load4(const void* p, long long i) {
  if constexpr (kType == ASTERQ_DTYPE_F32) return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
  const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i));
  const float2 a = kType == ASTERQ_DTYPE_F16 ? unpack_half2(w.x) : unpack_bf162(w.x);
  const float2 b = kType == ASTERQ_DTYPE_F16 ? unpack_half2(w.y) : unpack_bf162(w.y);
  return make_float4(a.x, a.y, b.x, b.y);
}

constexpr int kThreads = 256;

// One CTA: kCols columns of one (sequence, head)'s state, in registers from the first token to the
// last.  A single token reads and writes 8 Dk Dv bytes of state for 5 Dk Dv operations: bound by
// memory.  Each thread has four columns of Dk kCols / 1024 rows, all of whose loads are in flight at
// once, and kCols / 4 lanes read a row's columns together.  Measured: 256 rows of 32 heads of 128 x 128, one
// token each, 164 us, 6.5 TB/s; 4 rows of 16 heads 2.9 us.  Several tokens add about 0.45 us each, the latency of
// the next token's loads and of the sum over the key dims.  e^g is rounded to fp32 at every token, as in any fp32 form
// of the recurrence: a constant decay near one adds that up (g = -1e-4: 1.7e-4 of the state after 10,000 tokens, where
// the chunked form, which sums decays in 64 bits, keeps 2e-7).
template <int kType, int kDk, int kDv, int kCols>
__global__ void __launch_bounds__(kThreads) scan_kernel(const __grid_constant__ Args a) {
  constexpr int kLanes = kCols / 4;              // threads of a row
  constexpr int kGroups = kThreads / kLanes;     // rows side by side
  constexpr int kRows = kDk / kGroups;           // rows of a thread
  constexpr int kWarps = kThreads / 32;
  __shared__ float qk[2][2][kDk];
  __shared__ float part[2][kWarps][kCols];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seq = blockIdx.x, head = blockIdx.y, col0 = blockIdx.z * kCols;
  const int slot = __ldg(a.slots + seq);
  long long row = seq, end = seq + 1;
  if (a.row_offsets) {
    row = __ldg(a.row_offsets + seq);
    end = __ldg(a.row_offsets + seq + 1);
  }
  if (row < 0 || end > a.n_rows || row >= end) {
    if (tid == 0 && (row < 0 || end > a.n_rows || row > end) && a.status) atomicMax(a.status, 1);
    return;
  }
  if (slot < 0 || slot >= a.n_slots) {
    // an empty slot: its rows are zeros
    if (tid == 0 && slot >= a.n_slots && a.status) atomicMax(a.status, 1);
    for (; row < end; ++row)
      for (int i = tid; i < kCols; i += kThreads) store1<kType>(a.out, (row * a.n_heads + head) * kDv + col0 + i, 0.0f);
    return;
  }
  const bool fresh = a.lengths && __ldg(a.lengths + seq) <= 0;
  const int c4 = (tid % kLanes) * 4, r0 = tid / kLanes;
  float* s_ptr = a.state + ((long long)slot * a.n_heads + head) * kDk * kDv + col0 + c4;
  float4 s[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    s[i] = fresh ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                 : __ldcs(reinterpret_cast<const float4*>(s_ptr + (long long)(r0 + i * kGroups) * kDv));
  int buf = 0;
  for (; row < end; ++row, buf ^= 1) {
    for (int i = tid; i < 2 * kDk; i += kThreads) {
      const int d = i % kDk;
      qk[buf][i / kDk][d] = i < kDk ? load1<kType>(a.q, row * a.q_row + head * a.q_head + d)
                                    : load1<kType>(a.k, row * a.k_row + head * a.k_head + d);
    }
    const float4 v = load4<kType>(a.v, row * a.v_row + head * a.v_head + col0 + c4);
    const float decay = expf(__ldg(a.log_decay + row * a.decay_row + head));
    __syncthreads();
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const float q = qk[buf][0][r0 + i * kGroups], k = qk[buf][1][r0 + i * kGroups];
      s[i].x = fmaf(decay, s[i].x, k * v.x);
      s[i].y = fmaf(decay, s[i].y, k * v.y);
      s[i].z = fmaf(decay, s[i].z, k * v.z);
      s[i].w = fmaf(decay, s[i].w, k * v.w);
      o.x = fmaf(q, s[i].x, o.x);
      o.y = fmaf(q, s[i].y, o.y);
      o.z = fmaf(q, s[i].z, o.z);
      o.w = fmaf(q, s[i].w, o.w);
    }
#pragma unroll
    for (int d = kLanes; d < 32; d *= 2) {
      o.x += __shfl_xor_sync(0xffffffffu, o.x, d);
      o.y += __shfl_xor_sync(0xffffffffu, o.y, d);
      o.z += __shfl_xor_sync(0xffffffffu, o.z, d);
      o.w += __shfl_xor_sync(0xffffffffu, o.w, d);
    }
    if (lane < kLanes) *reinterpret_cast<float4*>(&part[buf][warp][c4]) = o;
    __syncthreads();
    if (tid < kCols) {
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += part[buf][w][tid];
      store1<kType>(a.out, (row * a.n_heads + head) * kDv + col0 + tid, sum * a.scale);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    __stcs(reinterpret_cast<float4*>(s_ptr + (long long)(r0 + i * kGroups) * kDv), s[i]);
}

template <int kType, int kDk, int kDv>
static void scan(const Args& a, int sms, cudaStream_t s) {
  // Columns of a CTA: the whole width, whose loads are the longest runs, but 32 of 128 while the (sequence,
  // head) pairs do not fill the SMs twice over.  Measured at 128 x 128 dims, 32 columns against all 128:
  // one token, 64 pairs 2.9 against 3.5 us, 288 pairs 6.2 against 5.9, 8192 pairs 173 against 164; 24 tokens,
  // 64 pairs 14.7 against 17.2, 512 pairs 72 against 58.  Of 64 columns the whole is as good or better
  // throughout: 64 pairs of 2 tokens 3.3 against 3.4 us, 4096 of 24 tokens 156 against 238.
  const dim3 grid(a.n_seqs, a.n_heads, 1);
  if constexpr (kDv == 128) {
    if ((long long)a.n_seqs * a.n_heads < 2ll * sms) {
      scan_kernel<kType, kDk, kDv, 32><<<dim3(a.n_seqs, a.n_heads, kDv / 32), kThreads, 0, s>>>(a);
      return;
    }
  }
  scan_kernel<kType, kDk, kDv, kDv><<<grid, kThreads, 0, s>>>(a);
}
template <int kType>
static void scan_by_dims(const Args& a, int dk, int dv, int sms, cudaStream_t s) {
  if (dk == 64 && dv == 64) scan<kType, 64, 64>(a, sms, s);
  else if (dk == 64) scan<kType, 64, 128>(a, sms, s);
  else if (dv == 64) scan<kType, 128, 64>(a, sms, s);
  else scan<kType, 128, 128>(a, sms, s);
}

// SMs of the current device, read once per device
static int sm_count(int* device) {
  static int counts[64] = {0};
  int n = 0;
  if (cudaGetDevice(device) != cudaSuccess) return 0;
  if (*device < 64 && counts[*device]) return counts[*device];
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *device) != cudaSuccess) return 0;
  if (*device < 64) counts[*device] = n;
  return n;
}

// The chunked form takes bf16 prompts of 24 tokens a sequence or more on average.  Measured at 128 x 128
// dims, chunked against the scan: one sequence of 16 heads, 24 tokens 14.2 against 12.5 us, 32 tokens 14.4
// against 15.8, 128 tokens 16.5 against 57; 4 of 32 heads, 24 tokens 15.0 against 22.8; 64 of 64 heads, 24 tokens
// 232 against 451, 128 tokens 296 against 2147.  At 64 x 64 dims: one sequence of 16 heads, 24 tokens 9.8
// against 12.6; 64 of 64 heads, 24 tokens 130 against 155, 128 tokens 135 against 753.  These are sequences of one
// length, and the host sees no other: a long prompt among many idle slots or single rows has a small average and goes
// token by token, where it would take a fraction of the time by itself.
static bool in_chunks(const asterq_linear_params* p) {
  return p->dtype == ASTERQ_DTYPE_BF16 && p->row_offsets && p->n_rows >= 24ll * p->n_seqs;
}

static int check(const asterq_linear_params* p) {
  if (!p) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "linear_attention: null parameters");
  if (p->n_seqs < 0 || p->n_heads <= 0 || p->n_slots < 0 || p->n_rows < 0)
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "linear_attention: bad sizes");
  if (p->dtype != ASTERQ_DTYPE_BF16 && p->dtype != ASTERQ_DTYPE_F16 && p->dtype != ASTERQ_DTYPE_F32)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "linear_attention: dtype %d: bf16, f16 or f32", p->dtype);
  if ((p->dk != 64 && p->dk != 128) || (p->dv != 64 && p->dv != 128))
    return set_error(ASTERQ_ERR_UNSUPPORTED, "linear_attention: head dims %d and %d: 64 or 128", p->dk, p->dv);
  if (p->n_heads > 65535) return set_error(ASTERQ_ERR_UNSUPPORTED, "linear_attention: more than 65535 heads");
  if (p->n_rows > 0x7fffffffLL) return set_error(ASTERQ_ERR_UNSUPPORTED, "linear_attention: more than 2^31 - 1 rows");
  return ASTERQ_OK;
}

}  // namespace lin
}  // namespace asterq

using namespace asterq;

extern "C" int64_t asterq_linear_workspace_bytes(const asterq_linear_params* p) {
  clear_error();
  if (lin::check(p) != ASTERQ_OK || !lin::in_chunks(p)) return 0;
  int device = 0;
  return lin::chunk_workspace_bytes(p->dk, p->dv, lin::sm_count(&device));
}

extern "C" int asterq_linear_attention(const asterq_linear_params* p, void* stream) {
  clear_error();
  const int st = lin::check(p);
  if (st != ASTERQ_OK) return st;
  if (p->n_seqs == 0 || p->n_rows == 0) return ASTERQ_OK;
  if (!p->q || !p->k || !p->v || !p->log_decay || !p->state || !p->slots || !p->out)
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "linear_attention: null pointer");
  if (!p->row_offsets && p->n_rows != p->n_seqs)
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "linear_attention: %lld rows for %d sequences of one token each",
                     (long long)p->n_rows, p->n_seqs);
  const void* vec[] = {p->q, p->k, p->v, p->state, p->out, p->workspace};
  for (const void* ptr : vec)
    if (reinterpret_cast<uintptr_t>(ptr) & 15)
      return set_error(ASTERQ_ERR_MISALIGNED, "linear_attention: arrays must be 16-byte aligned");
  const int64_t strides[] = {p->q_row_stride, p->q_head_stride, p->k_row_stride, p->k_head_stride, p->v_row_stride,
                             p->v_head_stride};
  for (int64_t s : strides)
    if (s % 8) return set_error(ASTERQ_ERR_MISALIGNED, "linear_attention: row and head strides must be multiples of 8");
  int device = 0;
  const int sms = lin::sm_count(&device);
  if (sms <= 0) return set_error(ASTERQ_ERR_CUDA, "linear_attention: no CUDA device");
  lin::Args a;
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.log_decay = p->log_decay;
  a.state = p->state;
  a.slots = p->slots;
  a.lengths = p->lengths;
  a.row_offsets = p->row_offsets;
  a.out = p->out;
  a.status = p->status;
  a.q_row = p->q_row_stride;
  a.q_head = p->q_head_stride;
  a.k_row = p->k_row_stride;
  a.k_head = p->k_head_stride;
  a.v_row = p->v_row_stride;
  a.v_head = p->v_head_stride;
  a.decay_row = p->decay_row_stride;
  a.n_rows = p->n_rows;
  a.n_seqs = p->n_seqs;
  a.n_heads = p->n_heads;
  a.n_slots = p->n_slots;
  a.scale = p->scale;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (lin::in_chunks(p)) {
    const int64_t need = lin::chunk_workspace_bytes(p->dk, p->dv, sms);
    if (!p->workspace || p->workspace_bytes < need)
      return set_error(ASTERQ_ERR_WORKSPACE, "linear_attention: workspace of %lld bytes, %lld needed",
                       (long long)p->workspace_bytes, (long long)need);
    const int done = lin::chunk_launch(a, p->dk, p->dv, sms, device, p->workspace, s);
    if (done != ASTERQ_ERR_UNSUPPORTED) return done;  // else strides that the copy engine cannot follow
  }
  switch (p->dtype) {
    case ASTERQ_DTYPE_F32: lin::scan_by_dims<ASTERQ_DTYPE_F32>(a, p->dk, p->dv, sms, s); break;
    case ASTERQ_DTYPE_F16: lin::scan_by_dims<ASTERQ_DTYPE_F16>(a, p->dk, p->dv, sms, s); break;
    default: lin::scan_by_dims<ASTERQ_DTYPE_BF16>(a, p->dk, p->dv, sms, s); break;
  }
  return check_launch("linear_attention");
}
