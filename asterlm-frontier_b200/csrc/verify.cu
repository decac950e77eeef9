// Verification of drafted tokens against the target's probabilities, by given random numbers.
//
// A sequence's drafted tokens are the nodes of a tree (or a chain); node 0 is the root, its token is accepted
// already.  target[i] is the target's distribution behind node i, draft[i] the one that i's children were drawn from.
// The walk is at cur = 0 with r = target[cur], m = 1.  Nodes i = 1, 2, ..: where parent(i) = cur, x its token,
//   accepted if accept[i] draft[cur][x] m < r(x): cur = i, r = target[i], m = 1;
//   rejected: r = max(r - m draft[cur], 0), m = sum r; if nothing is left (m = 0), r = target[cur], m = 1 again.
// At the end the next token is the least t with r(0) + .. + r(t) > sample sum r.  This draws from the target's
// distribution whatever the draft's was.  Without draft probabilities drafts are taken as certain: accepted if
// accept[i] m < r(x), rejected r(x) = 0 and m = m - r(x).
//
// What bounds it: one row of the target's probabilities a sequence, and one of the draft's, are read for each
// rejection behind which something follows, and to draw; the nodes' own values are gathered at once.  A cluster of CTAs shares a
// sequence's vocabulary while sequences are few.  Sums are in 64 bits: a border between two tokens among 10^5 is hit
// by the rounding of a 32-bit sum once in some hundred draws.
// Measured: 96 trees of 12 over 128,256 tokens (float32) 62 to 77 us over machines, 80 to 87 a call on new inputs each time: passes of 1 MB a
// sequence, each of which waits for the decision before it, by 384 CTAs on 296 places; 4 chains of 6 over 32,000 8.3 to 10.5 us, a launch and reads
// that wait for one another.
#include <cooperative_groups.h>

#include "asterq_internal.h"
#include "common.cuh"
#include "launch.cuh"

namespace asterq {
namespace ver {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = 16, kMaxNodes = 1024, kMaxCluster = 8;

struct Args {
  const void* target;
  const void* draft;
  const int* tokens;
  const int* parents;
  const int* row_offsets;
  const float* accept;
  const float* sample;
  int* kept;
  int* n_kept;
  int* next_token;
  int* status;
  long long target_stride, draft_stride, n_rows;
  int vocab;
};

template <int kType>
ASTERQ_DEVICE float value_at(const void* x, long long i) {
  if constexpr (kType == ASTERQ_DTYPE_F32) return __ldg(static_cast<const float*>(x) + i);
  const uint32_t w = __ldg(static_cast<const uint16_t*>(x) + i);
  return kType == ASTERQ_DTYPE_F16 ? unpack_half2(w).x : unpack_bf162(w).x;
}

ASTERQ_DEVICE double warp_sum(double x) {
#pragma unroll
  for (int d = 1; d < 32; d *= 2) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}

// The offsets name no nodes that can be walked: out of order, out of range, or too many.
ASTERQ_DEVICE bool refused(long long begin, long long end, long long n_rows) {
  return begin < 0 || end < begin || end > n_rows || end - begin > kMaxNodes;
}

// Rows between the least and the greatest offset that no walked sequence has become -1, by the CTA of the first refused sequence;
// the others' rows are written by their own CTAs, so none is written twice.  Taken = a bit a row of a window of 32 n_words rows.
__device__ __noinline__ void clear_refused(const int* row_offsets, int* kept, long long n_rows, int s, int n_seqs, uint32_t* taken,
                                           int n_words) {
  const int tid = threadIdx.x;
  bool later = false;
  int least = 0x7fffffff, most = -0x7fffffff;
  for (int t = tid; t < n_seqs; t += kThreads) {
    const int begin = __ldg(row_offsets + t), end = __ldg(row_offsets + t + 1);
    later = later || (t < s && refused(begin, end, n_rows));
    least = min(least, min(begin, end));
    most = max(most, max(begin, end));
  }
  if (__syncthreads_or(later)) return;
  int* range = reinterpret_cast<int*>(taken);
  if (tid == 0) {
    range[0] = 0x7fffffff;
    range[1] = -0x7fffffff;
  }
  __syncthreads();
  atomicMin(range, least);
  atomicMax(range + 1, most);
  __syncthreads();
  const long long from = max(0, range[0]), to = min(n_rows, (long long)range[1]);
  for (long long w0 = from; w0 < to; w0 += 32ll * n_words) {
    const long long w1 = min(to, w0 + 32ll * n_words);
    __syncthreads();
    for (int i = tid; i < n_words; i += kThreads) taken[i] = 0;
    __syncthreads();
    for (int t = tid; t < n_seqs; t += kThreads) {
      const long long begin = __ldg(row_offsets + t), end = __ldg(row_offsets + t + 1);
      if (refused(begin, end, n_rows)) continue;
      for (long long r = max(begin, w0); r < min(end, w1); ++r) atomicOr(taken + (r - w0) / 32, 1u << ((r - w0) & 31));
    }
    __syncthreads();
    for (long long r = w0 + tid; r < w1; r += kThreads)
      if (!(taken[(r - w0) / 32] >> ((r - w0) & 31) & 1u)) kept[r] = -1;
  }
}

template <int kType>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const Args a) {
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), s = blockIdx.x / ranks;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ int parent_s[kMaxNodes], token_s[kMaxNodes];
  __shared__ double p_s[kMaxNodes], q_s[kMaxNodes];
  __shared__ float u_s[kMaxNodes];
  __shared__ double mass_s[kMaxNodes];     // m before each rejection at cur
  __shared__ int gone_s[kMaxNodes];        // tokens rejected at cur, of drafts without probabilities
  __shared__ double warp_sums[kWarps], rank_sums[2][kMaxCluster];
  const long long begin = __ldg(a.row_offsets + s), end = __ldg(a.row_offsets + s + 1);
  const bool bad = refused(begin, end, a.n_rows);
  const int n = bad ? 0 : (int)(end - begin);
  if (n == 0) {  // the whole cluster
    if (rank == 0 && tid == 0) {
      a.n_kept[s] = 0;
      a.next_token[s] = -1;
      if (bad && a.status) atomicMax(a.status, 1);
    }
    if (bad && rank == 0) clear_refused(a.row_offsets, a.kept, a.n_rows, s, gridDim.x / ranks, reinterpret_cast<uint32_t*>(mass_s), 2 * kMaxNodes);
    return;
  }
  // a CTA's shared memory may be written by others once it has begun: arrived at here, waited for before the first sum
  if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;");
  bool odd = false;
  for (int i = tid; i < n; i += kThreads) {
    int up = a.parents ? __ldg(a.parents + begin + i) : i - 1;
    const bool root = i == 0;
    if (root ? up != -1 : (up < -1 || up >= i)) {
      odd = true;
      up = -1;
    }
    if (root) up = -1;
    const int x = __ldg(a.tokens + begin + i);
    const bool in = x >= 0 && x < a.vocab;
    odd = odd || (!root && !in);
    const bool use = !root && up >= 0 && in;
    parent_s[i] = up;
    token_s[i] = in ? x : -1;
    u_s[i] = __ldg(a.accept + begin + i);
    p_s[i] = use ? value_at<kType>(a.target, (begin + up) * a.target_stride + x) : 0.0;
    q_s[i] = use && a.draft ? value_at<kType>(a.draft, (begin + up) * a.draft_stride + x) : use ? 1.0 : 0.0;
  }
  if (odd && rank == 0 && a.status) atomicMax(a.status, 1);
  __syncthreads();

  // this CTA's part of the vocabulary, and its warps' parts
  const int chunk = (a.vocab + ranks - 1) / ranks;
  const int v0 = min(rank * chunk, a.vocab), v1 = min(v0 + chunk, a.vocab);
  int cur = 0, rejected = 0, count = 1, round = 0;
  double m = 1.0;
  // what is left of the target at t after the rejections so far
  auto left_at = [&](int t) {
    double r = (double)value_at<kType>(a.target, (begin + cur) * a.target_stride + t);
    const double q = a.draft && rejected > 0 ? (double)value_at<kType>(a.draft, (begin + cur) * a.draft_stride + t) : 0.0;
#pragma unroll 1
    for (int j = 0; j < rejected; ++j) {
      if (a.draft) {
        const double d = __dsub_rn(r, __dmul_rn(mass_s[j], q));
        r = d > 0.0 ? d : 0.0;
      } else {
        r = gone_s[j] == t ? 0.0 : r;
      }
    }
    return r;
  };
  // The sum of what is left over [from, to) by this warp, lanes side by side: the loads of kAhead rounds (4, 6, 8: 70, 62,
  // 64 us) are under way before the first is used.
  auto sum_of = [&](int from, int to) {
    double sum = 0.0;
    constexpr int kAhead = 6;
    const long long p0 = (begin + cur) * a.target_stride, q0 = (begin + cur) * a.draft_stride;
    const bool drafted = a.draft && rejected > 0;
#pragma unroll 1
    for (int t = from + lane; t < to; t += 32 * kAhead) {
      float p[kAhead], q[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) p[k] = t + 32 * k < to ? value_at<kType>(a.target, p0 + t + 32 * k) : 0.0f;
      if (drafted) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) q[k] = t + 32 * k < to ? value_at<kType>(a.draft, q0 + t + 32 * k) : 0.0f;
      }
      double r[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) r[k] = (double)p[k];
      if (drafted) {
#pragma unroll 1
        for (int j = 0; j < rejected; ++j) {
          const double mj = mass_s[j];
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            const double d = __dsub_rn(r[k], __dmul_rn(mj, (double)q[k]));
            r[k] = d > 0.0 ? d : 0.0;
          }
        }
      } else if (!a.draft) {
#pragma unroll 1
        for (int j = 0; j < rejected; ++j) {
          const int gone = gone_s[j] - t;
#pragma unroll
          for (int k = 0; k < kAhead; ++k) r[k] = gone == 32 * k ? 0.0 : r[k];
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) sum += r[k];
    }
    return warp_sum(sum);
  };
  auto part_of = [](int from, int to, int w, int& a0, int& a1) {
    const int each = ((to - from + kWarps - 1) / kWarps + 31) / 32 * 32;
    a0 = min(from + w * each, to);
    a1 = min(a0 + each, to);
  };
  // the sum over the vocabulary, the same in every thread of the cluster; warps' and CTAs' sums stay in shared memory
  auto total_left = [&]() {
    int a0, a1;
    part_of(v0, v1, warp, a0, a1);
    const double mine = sum_of(a0, a1);
    __syncthreads();
    if (lane == 0) warp_sums[warp] = mine;
    __syncthreads();
    if (round == 0 && ranks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    double* sums = rank_sums[round & 1];
    ++round;
    if (tid < ranks) {
      double sum = 0.0;
      for (int w = 0; w < kWarps; ++w) sum += warp_sums[w];
      *cluster.map_shared_rank(sums + rank, tid) = sum;
    }
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    double all = 0.0;
    for (int k = 0; k < ranks; ++k) all += sums[k];
    return all;
  };
  if (rank == 0 && tid == 0) a.kept[begin] = 0;
  int at = 0;  // every warp walks for itself: no barrier until sums are needed
  double total = -1.0;  // of what is left, once known
  while (true) {
    // the next node whose parent is cur
    int next = n;
    for (int base = (at + 1) & ~31; base < n && next == n; base += 32) {
      const int i = base + lane;
      const uint32_t hit = __ballot_sync(0xffffffffu, i > at && i < n && parent_s[i] == cur);
      if (hit) next = base + __ffs(hit) - 1;
    }
    if (next == n) break;
    at = next;
    const int x = token_s[next];
    double r = p_s[next];
    if (a.draft) {
      for (int k = 0; k < rejected; ++k) {
        const double d = __dsub_rn(r, __dmul_rn(mass_s[k], q_s[next]));
        r = d > 0.0 ? d : 0.0;
      }
    } else {
      for (int k = 0; k < rejected; ++k) r = gone_s[k] == x ? 0.0 : r;
    }
    if (__dmul_rn(__dmul_rn((double)u_s[next], q_s[next]), m) < r) {
      cur = next;
      if (rank == 0 && tid == 0) a.kept[begin + count] = next;
      ++count;
      rejected = 0;
      m = 1.0;
      total = -1.0;
      continue;
    }
    __syncthreads();  // no warp still reads the lists
    if (tid == 0) {
      mass_s[rejected] = m;
      gone_s[rejected] = x;
    }
    __syncthreads();
    ++rejected;
    if (a.draft) {
      total = total_left();
      m = total;
      if (total == 0.0) {
        rejected = 0;
        m = 1.0;
        total = -1.0;
      }
    } else {
      m = __dsub_rn(m, r);
    }
  }
  __syncthreads();
  if (total < 0.0) total = total_left();
  if (total == 0.0 && rejected > 0) {
    rejected = 0;
    total = total_left();
  }
  for (int i = count + rank * kThreads + tid; i < n; i += ranks * kThreads) a.kept[begin + i] = -1;
  if (rank == 0 && tid == 0) {
    a.n_kept[s] = count;
    if (!(total > 0.0)) {  // no distribution
      a.next_token[s] = -1;
      if (a.status) atomicMax(a.status, 1);
    }
  }
  if (total > 0.0) {
    // The CTA, then the warp's part, then parts of it, in which the running sum passes `rest`.
    const double* sums = rank_sums[(round - 1) & 1];
    double rest = __dmul_rn((double)__ldg(a.sample + s), total);
    if (rest < 0.0) rest = 0.0;
    int owner = -1, last = 0;
    for (int k = 0; k < ranks; ++k) {
      if (sums[k] > 0.0) last = k;
      if (owner < 0) {
        if (rest < sums[k]) owner = k;
        else rest -= sums[k];
      }
    }
    bool over = owner < 0;  // by rounding, or a random number of 1: the last token that has a probability
    if (over) owner = last;
    if (rank == owner) {
      int from = v0, to = v1;
      bool known = true;  // this CTA's warps' sums
      while (to - from > 32) {
        int a0, a1;
        part_of(from, to, warp, a0, a1);
        if (!known) {
          const double mine = sum_of(a0, a1);
          if (lane == 0) warp_sums[warp] = mine;
          __syncthreads();
        }
        known = false;
        int pick = -1, final = 0;
        double left = rest;
        for (int w = 0; w < kWarps; ++w) {
          if (warp_sums[w] > 0.0) final = w;
          if (pick < 0 && !over) {
            if (left < warp_sums[w]) pick = w;
            else left -= warp_sums[w];
          }
        }
        if (pick < 0) {
          over = true;
          pick = final;
        } else {
          rest = left;
        }
        __syncthreads();
        part_of(from, to, pick, a0, a1);
        from = a0;
        to = a1;
      }
      if (warp == 0) {
        const double r = from + lane < to ? left_at(from + lane) : 0.0;
        double scan = r;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
          const double up = __shfl_up_sync(0xffffffffu, scan, d);
          if (lane >= d) scan += up;
        }
        const uint32_t above = __ballot_sync(0xffffffffu, scan > rest && r > 0.0), some = __ballot_sync(0xffffffffu, r > 0.0);
        const int hit = !over && above ? __ffs(above) - 1 : 31 - __clz(some);
        if (lane == 0) a.next_token[s] = from + hit;
      }
    }
  }
  if (ranks > 1) cluster.sync();  // no CTA leaves while another may still write into it
}

template <int kType>
static cudaError_t launch(const Args& a, int n_seqs, int ranks, cudaStream_t s) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(n_seqs * ranks);
  c.blockDim = kThreads;
  c.stream = s;
  c.attrs = attr;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, verify_kernel<kType>, a);
}

}  // namespace ver
}  // namespace asterq

using namespace asterq;

extern "C" int asterq_verify_drafts(const asterq_verify_params* p, void* stream) {
  clear_error();
  if (!p) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "verify_drafts: null parameters");
  if (p->n_seqs < 0 || p->n_rows < 0 || p->vocab <= 0)
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "verify_drafts: bad sizes");
  if (p->dtype != ASTERQ_DTYPE_F32 && p->dtype != ASTERQ_DTYPE_BF16 && p->dtype != ASTERQ_DTYPE_F16)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "verify_drafts: dtype %d: f32, bf16 or f16", p->dtype);
  if (p->vocab > 0x7fff0000 || p->n_seqs > (1 << 27))
    return set_error(ASTERQ_ERR_UNSUPPORTED, "verify_drafts: more than 2^31 tokens or 2^27 sequences");
  if (p->n_seqs == 0) return ASTERQ_OK;
  if (!p->row_offsets || !p->n_kept || !p->next_token || !p->sample ||
      (p->n_rows > 0 && (!p->target || !p->tokens || !p->accept || !p->kept)))
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "verify_drafts: null pointer");
  if (p->target_stride < 0 || p->draft_stride < 0)
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "verify_drafts: negative strides");
  int dev = 0;
  const int sms = current_sms(&dev);
  if (sms <= 0) return set_error(ASTERQ_ERR_CUDA, "verify_drafts: no CUDA device");
  ver::Args a;
  a.target = p->target;
  a.draft = p->draft;
  a.tokens = p->tokens;
  a.parents = p->parents;
  a.row_offsets = p->row_offsets;
  a.accept = p->accept;
  a.sample = p->sample;
  a.kept = p->kept;
  a.n_kept = p->n_kept;
  a.next_token = p->next_token;
  a.status = p->status;
  a.target_stride = p->target_stride;
  a.draft_stride = p->draft_stride;
  a.n_rows = p->n_rows;
  a.vocab = p->vocab;
  // CTAs of a sequence: 8, where that leaves two a SM to each; more sequences have 4, as the passes of one wait for one another
  // and the others' fill the SMs, and from twice the SMs on 2; each has a part of 2048 tokens or more.  Trees of 12 over 128,256
  // tokens, 1, 2, 4 and 8 CTAs: 16 sequences 153, 86, 52, 37 us; 74: 157, 89, 63, 59; 96: 161, 89, 64, 75; 160: 242, 133,
  // 95, 118; 240: 263, 152, 130, 173; 320: 227, 157, 162, 218; 480: 282, 228, 234, 321.  Parts from 512 or from 8192 tokens on make no
  // difference above 2 us for vocabularies of 2,048 to 32,768.
  const int most = p->n_seqs <= sms / 2 ? ver::kMaxCluster : p->n_seqs <= 2 * sms ? 4 : 2;
  int ranks = 1;
  while (ranks < most && p->vocab / (ranks * 2) >= 2048) ranks *= 2;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = p->dtype == ASTERQ_DTYPE_F32    ? ver::launch<ASTERQ_DTYPE_F32>(a, p->n_seqs, ranks, s)
                        : p->dtype == ASTERQ_DTYPE_BF16 ? ver::launch<ASTERQ_DTYPE_BF16>(a, p->n_seqs, ranks, s)
                                                        : ver::launch<ASTERQ_DTYPE_F16>(a, p->n_seqs, ranks, s);
  if (e != cudaSuccess) return set_error(ASTERQ_ERR_CUDA, "verify_drafts: launch failed: %s", cudaGetErrorString(e));
  return check_launch("verify_drafts");
}
