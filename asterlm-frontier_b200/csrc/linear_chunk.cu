// Linear attention of prompts in chunks of 128 tokens on the fifth-generation tensor cores.
//
// With G_ij = g_{j+1} + ... + g_i the decay between two tokens of a chunk (all in log2), G_i0 the
// decay from the chunk's start through token i and w_j that from token j to the chunk's end:
//   A_ij = (q_i . k_j) 2^{G_ij}  (j <= i),   o_i = scale (2^{G_i0} q_i S + sum_j A_ij v_j),
//   S <- 2^{G} S + sum_j (w_j k_j) v_j^T.
// Four products of 128 x 128 x 128 a chunk and head of 128 dims; q, k, v are read once and o written
// once (128 KB a chunk and head).  At one head-chunk a CTA, an SM's share of the memory bandwidth
// takes 5,700 cycles for them; the products below take 3,600 to 4,100 on the tensor core.
//
// Rounding.  Products take bf16 operands and sum in fp32.  A and S enter as two bf16 parts (16 bits:
// beside the output's own rounding they vanish).  The state is an fp32 output, so its update must not
// round w_j k_j to less: it enters as three bf16 parts (24 bits), smallest first, each chunk's sum is
// formed from zero on the tensor core and added to S in fp32 registers.
//
// Work.  One persistent CTA an SM takes an equal, contiguous share of all (sequence, head, chunk)s.
// Where a share ends inside a (sequence, head), the state there has to come from the chunks before:
// a first pass computes what each such piece adds to a state of zeros (keys and values only), a small
// kernel chains the pieces of a (sequence, head), and the main pass starts each piece from its state.
//
// Roles in a CTA (448 threads): warps 0-3 turn Q K^T into A (row i = thread i) and write the output;
// warps 4-11 hold S in registers (thread = key dim, half of the value dims), scale and split the keys
// and update S; warp 12 loads by TMA; one thread of warp 13 issues all products.
#include <cuda.h>

#include "linear.cuh"
#include "tcgen05.cuh"

namespace asterq {
namespace lin {
namespace {

constexpr int kChunk = 128;
constexpr int kSlots = 5;       // tiles of 128 tokens in flight or in use
constexpr int kThreads = 448;
constexpr int kWarps = kThreads / 32;
constexpr int kBoxBytes = kChunk * 128;
constexpr int kMinShare = 4;    // chunks: below that the first pass costs more than another SM saves
constexpr float kLog2e = 1.44269504088896340736f;
// tensor memory columns
constexpr uint32_t kColA = 0, kColO = 128, kColU = 256, kColK = 384;

// what the first pass leaves of each worker's last piece, when that ends inside a (sequence, head)
struct Header {
  double decay;  // log2 of the piece's whole decay
  int kind;      // 0: no such piece, 1: the (sequence, head)'s first piece, 2: a later one
  int slot, head, fresh;
};

struct Work {
  Header* headers;  // [workers]
  float* pieces;    // [workers][Dk][Dv]: the pieces' own sums, then the states after them
  float* starts;    // [workers][Dk][Dv]: first pieces' initial states (their slot may be rewritten meanwhile)
};

struct Seq {
  long long row0;
  int rows, slot, chunks, fresh;
};
ASTERQ_DEVICE Seq seq_of(const Args& a, int s) {
  Seq q;
  const int begin = __ldg(a.row_offsets + s), end = __ldg(a.row_offsets + s + 1);
  q.slot = __ldg(a.slots + s);
  q.row0 = begin;
  const bool ok = begin >= 0 && end <= a.n_rows && begin < end;
  q.rows = ok ? end - begin : 0;
  q.chunks = ok && q.slot >= 0 && q.slot < a.n_slots ? (q.rows + kChunk - 1) / kChunk : 0;
  q.fresh = a.lengths && __ldg(a.lengths + s) <= 0;
  return q;
}

struct Walk {
  long long x, end, seq_start;
  int s;
  Seq seq;
  int head, k0, n;  // the current piece: chunks [k0, k0 + n) of (sequence s, head)
  ASTERQ_DEVICE bool next(const Args& a) {
    if (x >= end) return false;
    while (x >= seq_start + (long long)seq.chunks * a.n_heads) {
      seq_start += (long long)seq.chunks * a.n_heads;
      seq = seq_of(a, ++s);
    }
    const long long in = x - seq_start;
    head = (int)(in / seq.chunks);
    k0 = (int)(in - (long long)head * seq.chunks);
    n = (int)min((long long)(seq.chunks - k0), end - x);
    x += n;
    return true;
  }
};

template <int kDk, int kDv, bool kStateOnly>
struct Cfg {
  static constexpr int kTiles = kStateOnly ? 2 : 3;  // tiles of a chunk: K, (Q,) V
  static constexpr int kMaxD = kDk > kDv ? kDk : kDv;
  static constexpr int kSlotBytes = kMaxD / 64 * kBoxBytes;
  static constexpr int kStateBytes = kStateOnly ? 0 : kDk * kDv * 2;  // one bf16 part
  // barriers
  static constexpr int kFull = 0, kEmpty = kSlots, kQk = 2 * kSlots, kQs = kQk + 1, kULo = kQk + 2, kU = kQk + 3,
                       kO = kQk + 4, kDecay = kQk + 5, kKeys = kQk + 6, kKeysHi = kQk + 7, kS = kQk + 8,
                       kA = kQk + 9, kOFree = kQk + 10, kDrain = kQk + 11, kBars = kQk + 12;
  static constexpr int kMiscBytes = 2 * kChunk * 4 + kChunk * 4 + 16 + kBars * 8 + 16 * 8 + 32 + 32;
  static constexpr int kSmem = kSlots * kSlotBytes + 2 * kStateBytes + kMiscBytes;
};

ASTERQ_DEVICE void tma_rows(uint32_t dst, const CUtensorMap* map, int x, int head, int row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(head), "r"(row), "r"(bar)
      : "memory");
}

// x as a sum of bf16 parts, two values at a time
ASTERQ_DEVICE uint32_t split_part(float& x, float& y) {
  const uint32_t p = pack_bf162(x, y);
  x -= bf16lo_to_f32(p);
  y -= bf16hi_to_f32(p);
  return p;
}

template <int kDk, int kDv, bool kStateOnly>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                 const __grid_constant__ CUtensorMap v_map, const __grid_constant__ Args a,
                 const __grid_constant__ Work work) {
  using C = Cfg<kDk, kDv, kStateOnly>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t s_hi = base + kSlots * C::kSlotBytes, s_lo = s_hi + C::kStateBytes;
  float* g_s = reinterpret_cast<float*>(smem + kSlots * C::kSlotBytes + 2 * C::kStateBytes);  // [2][kChunk]
  float* w_s = g_s + 2 * kChunk;
  float* tot_s = w_s + kChunk;  // [4]
  uint64_t* bars_s = reinterpret_cast<uint64_t*>(tot_s + 4);
  long long* scan_s = reinterpret_cast<long long*>(bars_s + C::kBars);  // [16]
  long long* start_s = scan_s + 16;                                     // sequence, its first chunk
  int* abort_s = reinterpret_cast<int*>(start_s + 2);
  uint32_t* tmem_s = reinterpret_cast<uint32_t*>(abort_s + 1);
  const uint32_t bars = smem_u32(bars_s);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto bar = [&](int i) { return bars + 8 * i; };
  // A wait that runs into its limit raises the abort flag and every other wait returns at once: the
  // walk goes on to its end over whatever is there, within bounds, and nothing hangs.
  auto wait = [&](int i, int phase) { (void)mbar_wait(bar(i), phase & 1, abort_s); };

  if (tid == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(bar(C::kFull + i), 1);
      mbar_init(bar(C::kEmpty + i), 1);
    }
    for (int i : {C::kQk, C::kQs, C::kULo, C::kU, C::kO, C::kDecay, C::kDrain}) mbar_init(bar(i), 1);
    for (int i : {C::kKeys, C::kKeysHi, C::kS}) mbar_init(bar(i), 8);
    for (int i : {C::kA, C::kOFree}) mbar_init(bar(i), 4);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *abort_s = 0;
  }

  // this CTA's share: a prefix sum over the sequences' chunks, thread t summing a strip of them
  const int strip = (a.n_seqs + kThreads - 1) / kThreads;
  const int s0 = min(tid * strip, a.n_seqs), s1 = min(s0 + strip, a.n_seqs);
  long long sum = 0;
  for (int s = s0; s < s1; ++s) sum += seq_of(a, s).chunks;
  sum *= a.n_heads;
  long long scan = sum;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long up = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += up;
  }
  if (lane == 31) scan_s[warp] = scan;
  __syncthreads();
  long long before = scan - sum, total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += scan_s[w];
    total += scan_s[w];
  }
  const int me = blockIdx.x;
  const int W = (int)max(1ll, min((long long)gridDim.x, (total + kMinShare - 1) / kMinShare));
  Walk walk;
  walk.x = me < W ? total * me / W : total;
  walk.end = me < W ? total * (me + 1) / W : total;
  if (walk.x < walk.end && before <= walk.x && walk.x < before + sum) {
    int s = s0;
    long long at = before;
    while (true) {
      const long long here = (long long)seq_of(a, s).chunks * a.n_heads;
      if (walk.x < at + here) break;
      at += here;
      ++s;
    }
    start_s[0] = s;
    start_s[1] = at;
  }
  if (!kStateOnly) {
    // rows of empty slots are zeros; ranges out of bounds are reported
    for (int s = me; s < a.n_seqs; s += gridDim.x) {
      const Seq q = seq_of(a, s);
      if (q.chunks > 0) continue;
      const int begin = __ldg(a.row_offsets + s), end = __ldg(a.row_offsets + s + 1);
      if (tid == 0 && a.status && (begin < 0 || end > a.n_rows || (q.rows > 0 && q.slot >= a.n_slots)))
        atomicMax(a.status, 1);
      uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + q.row0 * a.n_heads * kDv);
      for (long long i = tid; i < (long long)q.rows * a.n_heads * (kDv / 8); i += kThreads)
        dst[i] = make_uint4(0, 0, 0, 0);
    }
  }
  __syncthreads();
  if (walk.x < walk.end) {
    walk.s = (int)start_s[0];
    walk.seq_start = start_s[1];
    walk.seq = seq_of(a, walk.s);
  }
  if (kStateOnly) {
    // only the share's last piece, when its (sequence, head) goes on in the next share
    bool cut = false;
    if (walk.x < walk.end) {
      Walk last = walk;
      while (true) {
        Walk step = last;
        if (!step.next(a)) break;
        walk = last;
        last = step;
        cut = step.k0 + step.n < step.seq.chunks;
      }
    }
    if (!cut) {
      if (tid == 0) work.headers[me].kind = 0;
      return;
    }
  } else if (walk.x >= walk.end) {
    return;
  }

  if (warp == 13) tc::alloc512(smem_u32(tmem_s));
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_s;

  if (warp == 12) {
    // ---------------------------------------------------------------- loads
    if (lane == 0) {
      int n = 0;
      auto load = [&](const CUtensorMap* map, int boxes, int row, int head) {
        const int slot = n % kSlots;
        if (n >= kSlots) wait(C::kEmpty + slot, n / kSlots - 1);
        mbar_expect_tx(bar(C::kFull + slot), boxes * kBoxBytes);
        for (int b = 0; b < boxes; ++b)
          tma_rows(base + slot * C::kSlotBytes + b * kBoxBytes, map, b * 64, head, row, bar(C::kFull + slot));
        ++n;
      };
      while (walk.next(a))
        for (int j = 0; j < walk.n; ++j) {
          const int row = (int)walk.seq.row0 + (walk.k0 + j) * kChunk;
          load(&k_map, kDk / 64, row, walk.head);
          if (!kStateOnly) load(&q_map, kDk / 64, row, walk.head);
          load(&v_map, kDv / 64, row, walk.head);
        }
      // after a wait ran out nobody may have waited for the last copies: they land before the exit
      if (ld_shared_volatile(abort_s)) {
        int none = 0;
        for (int t = max(0, n - kSlots); t < n; ++t)
          (void)mbar_wait(bar(C::kFull + t % kSlots), (t / kSlots) & 1, &none, 20000000);
      }
    }
    __syncwarp();
  } else if (warp == 13) {
    // ---------------------------------------------------------------- products
    if (lane == 0) {
      constexpr uint32_t kQkDesc = tc::idesc_bf16(kChunk, false), kVDesc = tc::idesc_bf16(kDv, true);
      int c = 0;
      while (walk.next(a))
        for (int j = 0; j < walk.n; ++j, ++c) {
          const int rows = min(kChunk, walk.seq.rows - (walk.k0 + j) * kChunk), steps = (rows + 15) / 16;
          const int t = c * C::kTiles, tv = t + C::kTiles - 1;
          const uint32_t k_at = base + (t % kSlots) * C::kSlotBytes, v_at = base + (tv % kSlots) * C::kSlotBytes;
          const bool carried = walk.k0 + j > 0 || !walk.seq.fresh;  // S is not zero by construction
          if constexpr (!kStateOnly) {
            const int tq = t + 1;
            const uint32_t q_at = base + (tq % kSlots) * C::kSlotBytes;
            wait(C::kFull + t % kSlots, t / kSlots);
            wait(C::kFull + tq % kSlots, tq / kSlots);
#pragma unroll
            for (int s = 0; s < kDk / 16; ++s) {
              const uint32_t at = (s / 4) * kBoxBytes + (s % 4) * 32;
              tc::mma_ss(tmem + kColA, tc::desc_k_major(q_at + at), tc::desc_k_major(k_at + at), kQkDesc, s > 0);
            }
            tc::commit(bar(C::kQk));
            wait(C::kS, c);
            if (c > 0) wait(C::kOFree, c - 1);
            tc::fence_after();
            if (carried) {
#pragma unroll
              for (int s = 0; s < kDk / 16; ++s) {
                const uint64_t q_desc = tc::desc_k_major(q_at + (s / 4) * kBoxBytes + (s % 4) * 32);
                tc::mma_ss(tmem + kColO, q_desc, tc::desc_mn_major(s_hi + s * 2048, kDk * 128), kVDesc, s > 0);
                tc::mma_ss(tmem + kColO, q_desc, tc::desc_mn_major(s_lo + s * 2048, kDk * 128), kVDesc, true);
              }
            }
            tc::commit(bar(C::kQs));
            tc::commit(bar(C::kEmpty + tq % kSlots));
          } else {
            wait(C::kS, c);
            tc::fence_after();
          }
          wait(C::kFull + tv % kSlots, tv / kSlots);
          wait(C::kKeys, c);
          tc::fence_after();
          for (int s = 0; s < steps; ++s)
            tc::mma_ts(tmem + kColU, tmem + kColK + 8 * s, tc::desc_mn_major(v_at + s * 2048, kBoxBytes), kVDesc, s > 0);
          tc::commit(bar(C::kULo));
          for (int s = 0; s < steps; ++s)
            tc::mma_ts(tmem + kColU, tmem + kColK + 64 + 8 * s, tc::desc_mn_major(v_at + s * 2048, kBoxBytes), kVDesc, true);
          wait(C::kKeysHi, c);
          tc::fence_after();
          for (int s = 0; s < steps; ++s)
            tc::mma_ts(tmem + kColU, tmem + kColK + 8 * s, tc::desc_mn_major(v_at + s * 2048, kBoxBytes), kVDesc, true);
          tc::commit(bar(C::kU));
          tc::commit(bar(C::kEmpty + t % kSlots));
          if constexpr (!kStateOnly) {
            wait(C::kA, c);
            tc::fence_after();
            for (int s = 0; s < steps; ++s) {
              const uint32_t at = tmem + kColA + 32 * (s / 2) + 8 * (s % 2);
              const uint64_t v_desc = tc::desc_mn_major(v_at + s * 2048, kBoxBytes);
              tc::mma_ts(tmem + kColO, at, v_desc, kVDesc, carried || s > 0);
              tc::mma_ts(tmem + kColO, at + 16, v_desc, kVDesc, true);
            }
            tc::commit(bar(C::kO));
          }
          tc::commit(bar(C::kEmpty + tv % kSlots));
        }
      // every product and every arrival above is done before the tensor memory goes back
      tc::commit(bar(C::kDrain));
      int none = 0;
      (void)mbar_wait(bar(C::kDrain), 0, &none);
    }
    __syncwarp();
  } else if (warp < 4) {
    // ---------------------------------------------------------------- A and the output
    if constexpr (!kStateOnly) {
      const uint32_t lanes = tmem + ((uint32_t)warp << 21);  // this warp's 32 lanes
      const int i = warp * 32 + lane;                        // row of the chunk
      int c = 0;
      while (walk.next(a))
        for (int j = 0; j < walk.n; ++j, ++c) {
          const int rows = min(kChunk, walk.seq.rows - (walk.k0 + j) * kChunk);
          const bool carried = walk.k0 + j > 0 || !walk.seq.fresh;
          const float* g = g_s + (c & 1) * kChunk;
          if (c == 0) wait(C::kDecay, 0);
          wait(C::kQk, c);
          tc::fence_after();
          // From the row's own token back: sum = G_ij, exact where it matters, whatever came before.
          float sum = 0.0f;
#pragma unroll 1
          for (int group = 3; group >= 0; --group) {
            uint32_t r[32];
            if (group > warp) {
              if (32 * group >= rows) continue;  // no product reads these columns
#pragma unroll
              for (int e = 0; e < 32; ++e) r[e] = 0;
              tc::st32(lanes + kColA + 32 * group, r);
              continue;
            }
            tc::ld32(r, lanes + kColA + 32 * group);
            tc::wait_ld();
            uint32_t out[32];
            if (group == warp) {
#pragma unroll
              for (int e = 15; e >= 0; --e) {
                float x[2];
#pragma unroll
                for (int h = 1; h >= 0; --h) {
                  const int col = 2 * e + h;
                  if (col < lane) sum += g[32 * group + col + 1];
                  x[h] = col <= lane ? __uint_as_float(r[col]) * ex2_ftz(sum) : 0.0f;
                }
                out[e] = split_part(x[0], x[1]);
                out[16 + e] = pack_bf162(x[0], x[1]);
              }
            } else {
#pragma unroll
              for (int e = 15; e >= 0; --e) {
                sum += g[32 * group + 2 * e + 2];
                float x1 = __uint_as_float(r[2 * e + 1]) * ex2_ftz(sum);
                sum += g[32 * group + 2 * e + 1];
                float x0 = __uint_as_float(r[2 * e]) * ex2_ftz(sum);
                out[e] = split_part(x0, x1);
                out[16 + e] = pack_bf162(x0, x1);
              }
            }
            tc::st32(lanes + kColA + 32 * group, out);
          }
          const float from_start = exp2f(sum + g[0]);
          wait(C::kQs, c);
          tc::fence_after();
          if (carried) {
#pragma unroll 1
            for (int d = 0; d < kDv; d += 32) {
              uint32_t r[32];
              tc::ld32(r, lanes + kColO + d);
              tc::wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * from_start);
              tc::st32(lanes + kColO + d, r);
            }
          }
          tc::wait_st();
          tc::fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::kA));
          wait(C::kO, c);
          tc::fence_after();
          const long long row = walk.seq.row0 + (walk.k0 + j) * kChunk + i;
          uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (row * a.n_heads + walk.head) * kDv);
#pragma unroll 1
          for (int d = 0; d < kDv; d += 32) {
            uint32_t r[32];
            tc::ld32(r, lanes + kColO + d);
            tc::wait_ld();
            if (d + 32 == kDv) {
              // The next chunk's decays are waited for before the products may go on: the warps that
              // write them could otherwise run two chunks ahead of this barrier's phase.
              if (j + 1 < walk.n || walk.x < walk.end) wait(C::kDecay, c + 1);
              tc::fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(C::kOFree));
            }
            if (i < rows) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                uint32_t p[4];
#pragma unroll
                for (int h = 0; h < 4; ++h)
                  p[h] = pack_bf162(__uint_as_float(r[8 * e + 2 * h]) * a.scale,
                                    __uint_as_float(r[8 * e + 2 * h + 1]) * a.scale);
                dst[d / 8 + e] = make_uint4(p[0], p[1], p[2], p[3]);
              }
            }
          }
        }
    }
  } else {
    // ---------------------------------------------------------------- keys and state
    constexpr int kCols = kDv / 2;
    const int part = (warp - 4) >> 2;               // tokens 64 part .., value dims kCols part ..
    const int dk = (warp & 3) * 32 + lane;          // key dim
    const bool has = kDk == 128 || (warp & 3) < 2;  // whole warps
    const int t = (warp & 3) * 32 + lane;           // token whose decay a thread of the first part reads
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    const uint32_t k_col = (dk / 64) * kBoxBytes + (dk & 7) * 2;
    const int k_unit = (dk % 64) >> 3;
    float s[kCols];
    int c = 0;
    while (walk.next(a)) {
      const Seq q = walk.seq;
      const bool ends = walk.k0 + walk.n == q.chunks;
      const long long slot_at = (((long long)q.slot * a.n_heads + walk.head) * kDk + dk) * kDv + part * kCols;
      const long long piece_at = (long long)dk * kDv + part * kCols;
      // the state at the piece's start
      const float* from = nullptr;
      if (!kStateOnly) {
        if (walk.k0 > 0) from = work.pieces + (long long)(me - 1) * kDk * kDv + piece_at;
        else if (q.fresh) from = nullptr;
        else from = ends ? a.state + slot_at : work.starts + (long long)me * kDk * kDv + piece_at;
      }
#pragma unroll
      for (int e = 0; e < kCols; e += 4) {
        const float4 x = from && has ? *reinterpret_cast<const float4*>(from + e) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        s[e] = x.x;
        s[e + 1] = x.y;
        s[e + 2] = x.z;
        s[e + 3] = x.w;
      }
      double decay = 0.0;
      auto read_decay = [&](int j) {
        const int at = (walk.k0 + j) * kChunk + t;
        return part == 0 && j < walk.n && at < q.rows ? __ldg(a.log_decay + (q.row0 + at) * a.decay_row + walk.head) : 0.0f;
      };
      float g_next = read_decay(0);
      for (int j = 0; j < walk.n; ++j, ++c) {
        const int rows = min(kChunk, q.rows - (walk.k0 + j) * kChunk), steps = (rows + 15) / 16;
        // S for this chunk's outputs; the products of the last chunk that read the old one are done
        // (they were issued before the update that was waited for)
        if (!kStateOnly && has) {
          const uint32_t row_at = ((part * kCols) / 64) * (kDk * 128) + dk * 128;
          const int unit0 = ((part * kCols) % 64) / 8;
#pragma unroll
          for (int e = 0; e < kCols / 8; ++e) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              float x = s[8 * e + 2 * h], y = s[8 * e + 2 * h + 1];
              hi[h] = split_part(x, y);
              lo[h] = pack_bf162(x, y);
            }
            const uint32_t at = row_at + (((unit0 + e) ^ (dk & 7)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(s_hi + at), "r"(hi[0]), "r"(hi[1]), "r"(hi[2]),
                         "r"(hi[3])
                         : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(s_lo + at), "r"(lo[0]), "r"(lo[1]), "r"(lo[2]),
                         "r"(lo[3])
                         : "memory");
          }
          fence_async_shared();
        }
        tc::fence_before();  // after the reads of U
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kS));

        // decays: this token's, and the weight from it to the chunk's end
        const float g = g_next * kLog2e;
        g_next = read_decay(j + 1);
        float after = g;  // inclusive from this token on, within the warp
        if (part == 0) {
          g_s[(c & 1) * kChunk + t] = g;
#pragma unroll
          for (int d = 1; d < 32; d *= 2) {
            const float down = __shfl_down_sync(0xffffffffu, after, d);
            if (lane + d < 32) after += down;
          }
          if (lane == 0) tot_s[warp & 3] = after;
          after = __shfl_down_sync(0xffffffffu, after, 1);
          if (lane == 31) after = 0.0f;
        }
        named_sync(2, 256);
        if (tid == 128) mbar_arrive(bar(C::kDecay));
        if (part == 0) {
#pragma unroll
          for (int w = 3; w > 0; --w)
            if (w > (warp & 3)) after += tot_s[w];
          w_s[t] = exp2f(after);
        }
        const double chunk_decay = ((double)tot_s[0] + tot_s[1]) + ((double)tot_s[2] + tot_s[3]);
        decay += chunk_decay;
        // in 64 bits: a constant decay's error would add up over all the chunks it acts on
        const float whole = (float)exp2(chunk_decay);
        named_sync(2, 256);

        // the keys, weighted and split
        const int tk = c * C::kTiles, tv = tk + C::kTiles - 1;
        const uint32_t k_at = base + (tk % kSlots) * C::kSlotBytes + k_col;
        uint32_t hi[32];
        wait(C::kFull + tk % kSlots, tk / kSlots);
        if (has) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int t0 = part * 64 + u * 16;
            if (t0 >= rows) continue;
            uint32_t mid[8], lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float x[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int tok = t0 + 2 * e + h;
                uint16_t raw;
                asm volatile("ld.shared.u16 %0, [%1];"
                             : "=h"(raw)
                             : "r"(k_at + tok * 128 + ((k_unit ^ (tok & 7)) << 4)));
                x[h] = __uint_as_float((uint32_t)raw << 16) * w_s[tok];
                if (tok >= rows) x[h] = 0.0f;
              }
              hi[u * 8 + e] = split_part(x[0], x[1]);
              mid[e] = split_part(x[0], x[1]);
              lo[e] = pack_bf162(x[0], x[1]);
            }
            tc::st8(lanes + kColK + t0 / 2, lo);
            tc::st8(lanes + kColK + 64 + t0 / 2, mid);
          }
        }
        wait(C::kFull + tv % kSlots, tv / kSlots);
        if (rows < steps * 16) {
          // the last chunk's products run over whole steps of 16 tokens: values past the end are zeros
          const uint32_t v_at = base + (tv % kSlots) * C::kSlotBytes;
          for (int e = tid - 128; e < (steps * 16 - rows) * (kDv / 8); e += 256) {
            const int row = rows + e / (kDv / 8), unit = e % (kDv / 8);
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v_at + (unit / 8) * kBoxBytes + row * 128 +
                                                                          (unit % 8) * 16),
                         "r"(0)
                         : "memory");
          }
          fence_async_shared();
        }
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kKeys));
        wait(C::kULo, c);
        tc::fence_after();
        if (has) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int t0 = part * 64 + u * 16;
            if (t0 >= rows) continue;
            uint32_t r[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) r[e] = hi[u * 8 + e];
            tc::st8(lanes + kColK + t0 / 2, r);
          }
        }
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kKeysHi));

        wait(C::kU, c);
        tc::fence_after();
        if (has) {
#pragma unroll
          for (int d = 0; d < kCols; d += 32) {
            uint32_t r[32];
            tc::ld32(r, lanes + kColU + part * kCols + d);
            tc::wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) s[d + e] = fmaf(whole, s[d + e], __uint_as_float(r[e]));
          }
        }
      }
      float* to = nullptr;
      if (kStateOnly) {
        to = work.pieces + (long long)me * kDk * kDv + piece_at;
        if (tid == 128) {
          Header h;
          h.decay = decay;
          h.kind = walk.k0 == 0 ? 1 : 2;
          h.slot = q.slot;
          h.head = walk.head;
          h.fresh = q.fresh;
          work.headers[me] = h;
        }
      } else if (ends) {
        to = a.state + slot_at;
      }
      if (to && has) {
#pragma unroll
        for (int e = 0; e < kCols; e += 4)
          *reinterpret_cast<float4*>(to + e) = make_float4(s[e], s[e + 1], s[e + 2], s[e + 3]);
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 13) {
    tc::fence_after();
    tc::dealloc512(tmem);
  }
  if (tid == 0 && *abort_s && a.status) atomicMax(a.status, 2);
}

// The states between the pieces of a (sequence, head), one thread for four values: worker w's piece
// becomes the state after it.  A chain is as long as the (sequence, head) has shares.
template <int kDk, int kDv>
__global__ void __launch_bounds__(256) chain_kernel(const __grid_constant__ Args a, const __grid_constant__ Work work,
                                                    int workers) {
  int w = blockIdx.x;
  Header h = work.headers[w];
  if (h.kind != 1) return;
  const long long at = ((long long)blockIdx.y * 256 + threadIdx.x) * 4;
  if (at >= kDk * kDv) return;
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (!h.fresh) s = *reinterpret_cast<const float4*>(a.state + ((long long)h.slot * a.n_heads + h.head) * kDk * kDv + at);
  *reinterpret_cast<float4*>(work.starts + (long long)w * kDk * kDv + at) = s;
  while (true) {
    float4* p = reinterpret_cast<float4*>(work.pieces + (long long)w * kDk * kDv + at);
    const float f = (float)exp2(h.decay);
    const float4 u = *p;
    s.x = fmaf(f, s.x, u.x);
    s.y = fmaf(f, s.y, u.y);
    s.z = fmaf(f, s.z, u.z);
    s.w = fmaf(f, s.w, u.w);
    *p = s;
    if (++w >= workers) break;
    h = work.headers[w];
    if (h.kind != 2) break;
  }
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  }
  return fn;
}

// rows of bf16 heads [n_rows][n_heads][dim] with any strides, read in boxes of 128 rows x 64 dims
bool make_map(CUtensorMap* map, const void* base, const Args& a, int dim, long long row_stride, long long head_stride) {
  EncodeTiledFn fn = encode_fn();
  if (!fn || row_stride <= 0 || head_stride <= 0) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)a.n_heads, (cuuint64_t)a.n_rows};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)row_stride * 2};
  const cuuint32_t box[3] = {64u, 1u, (cuuint32_t)kChunk}, step[3] = {1u, 1u, 1u};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kDk, int kDv>
int launch(const Args& a, int workers, int device, void* workspace, cudaStream_t s) {
  using First = Cfg<kDk, kDv, true>;
  using Main = Cfg<kDk, kDv, false>;
  CUtensorMap q_map, k_map, v_map;
  if (!make_map(&q_map, a.q, a, kDk, a.q_row, a.q_head) || !make_map(&k_map, a.k, a, kDk, a.k_row, a.k_head) ||
      !make_map(&v_map, a.v, a, kDv, a.v_row, a.v_head))
    return ASTERQ_ERR_UNSUPPORTED;
  static unsigned long long configured = 0;  // one bit per device ordinal
  if (device >= 64 || !(configured & (1ull << device))) {
    cudaError_t e = cudaFuncSetAttribute(chunk_kernel<kDk, kDv, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         First::kSmem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(chunk_kernel<kDk, kDv, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Main::kSmem);
    if (e != cudaSuccess)
      return set_error(ASTERQ_ERR_CUDA, "linear_attention: shared memory opt-in: %s", cudaGetErrorString(e));
    if (device < 64) configured |= 1ull << device;
  }
  Work work;
  work.headers = static_cast<Header*>(workspace);
  work.pieces = reinterpret_cast<float*>(static_cast<char*>(workspace) + (workers * sizeof(Header) + 255) / 256 * 256);
  work.starts = work.pieces + (long long)workers * kDk * kDv;
  chunk_kernel<kDk, kDv, true><<<workers, kThreads, First::kSmem, s>>>(q_map, k_map, v_map, a, work);
  chain_kernel<kDk, kDv><<<dim3(workers, kDk * kDv / 1024), 256, 0, s>>>(a, work, workers);
  chunk_kernel<kDk, kDv, false><<<workers, kThreads, Main::kSmem, s>>>(q_map, k_map, v_map, a, work);
  return check_launch("linear_attention");
}

}  // namespace

int64_t chunk_workspace_bytes(int dk, int dv, int workers) {
  return (workers * (int64_t)sizeof(Header) + 255) / 256 * 256 + 2ll * workers * dk * dv * 4;
}

int chunk_launch(const Args& a, int dk, int dv, int workers, int device, void* workspace, cudaStream_t s) {
  if (dk == 64 && dv == 64) return launch<64, 64>(a, workers, device, workspace, s);
  if (dk == 64) return launch<64, 128>(a, workers, device, workspace, s);
  if (dv == 64) return launch<128, 64>(a, workers, device, workspace, s);
  return launch<128, 128>(a, workers, device, workspace, s);
}

}  // namespace lin
}  // namespace asterq
