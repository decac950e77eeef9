// Linear attention of prompts in chunks of 128 tokens on the fifth-generation tensor cores.
//
// With G_ij = g_{j+1} + ... + g_i the decay between two tokens of a chunk (all in log2), G_i0 the
// decay from the chunk's start through token i and w_j that from token j to the chunk's end:
//   A_ij = (q_i . k_j) 2^{G_ij}  (j <= i),   o_i = scale (2^{G_i0} q_i S + sum_j A_ij v_j),
//   S <- 2^{G} S + sum_j (w_j k_j) v_j^T.
// Four products of 128 x 128 x 128 a chunk and head of 128 dims; q, k, v are read once and o written
// once (128 KB a chunk and head).  At one head-chunk a CTA, an SM's share of the memory bandwidth
// takes 5,700 cycles for them; the products below take 4,600 on the tensor core.
//
// Measured (128 x 128 dims): 32777 tokens of 12 sequences and 32 heads 425 us, 2.6 TB/s (the bytes alone: 170 us); call
// after call its power takes the clock from 1965 to some 1650 MHz, and the time, which is all cycles, goes to 480 us.
// A CTA's 56 chunks take some 9,400 cycles each: the warp that issues the products is busy for 5,500 of them and
// goes from one role's barrier to the next for the rest, since a chunk's state, its outputs and the next
// chunk's keys wait for one another.  8192 tokens of one sequence and 16 heads: 94 us, some 35 of them the first pass
// and the chain of states.  One chunk of 16 heads: 15 us, a launch and the latency of one chunk.
//
// Rounding.  Products take bf16 operands and sum in fp32.  A and S enter as two bf16 parts (16 bits:
// beside the output's own rounding they vanish).  The state is an fp32 output, so its update must not
// round w_j k_j to less.  The weight is split into bf16 parts w = w1 + w2 + w3 and the key's bf16 products
// with them, exact in two parts each by one multiplication and one fused one, give four operands,
//   k w1 = p1 + p2,   k w2 = m + r,   l = k w3 + r:   p1, p2, m and l,
// for five packed operations a pair of values (splitting the fp32 product instead took twenty).  They are
// summed smallest first; each chunk's sum is formed from zero on the tensor core and added to S in fp32
// registers.
//
// Work.  One persistent CTA an SM takes an equal, contiguous share of all (sequence, head, chunk)s.
// Where a share ends inside a (sequence, head), the state there has to come from the chunks before:
// a first pass computes what these chunks add to a state of zeros (keys and values only), itself cut into
// equal shares, a small kernel chains the parts of each (sequence, head), and the main pass starts each of
// its pieces from its state.
//
// Roles in a CTA (512 threads): warps 0-3 turn Q K^T into A (row i = thread i) and write the output;
// warps 4-11 hold S in registers (thread = key dim, half of the value dims), scale and split the keys
// and update S; warp 12 loads by TMA; warp 13 issues all products; warp 14 sums the decays, a chunk
// ahead; warp 15 looks for values that are not finite (2% of the time: an answer must not depend on what comes after
// it).  Warps 4-11 take registers from the other groups (at
// 128 a thread S would spill to local memory).
#include <cuda.h>

#include "launch.cuh"
#include "linear.cuh"
#include "tcgen05.cuh"

namespace asterq {
namespace lin {
namespace {

constexpr int kChunk = 128;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kRegsA = 96, kRegsS = 168, kRegsIssue = 80;
static_assert(kRegsA + 2 * kRegsS + kRegsIssue <= 4 * 128, "the split draws on the block's registers at launch");
constexpr int kBoxBytes = kChunk * 128;
constexpr float kLog2e = 1.44269504088896340736f;

// A part of the first pass: some chunks of one (sequence, head), from a state of zeros.
struct Part {
  float decay;   // over all of them
  int slot, head, fresh;
  int next;      // the (sequence, head)'s next part, or -1
  int border;    // the border of shares that the part reaches, or -1
};

// Border w is between the main pass's shares w - 1 and w.
struct Work {
  Part* parts;     // [2 workers]
  int* first;      // [workers] the first part of the (sequence, head) whose first cut is border w, or -1
  float* sums;     // [2 workers][Dk][Dv]: what the parts add
  float* borders;  // [workers][Dk][Dv]: the state at border w
  float* starts;   // [workers][Dk][Dv]: the initial state of the (sequence, head) whose first cut is border w (its
                   // slot may be rewritten while the main pass still wants it)
  uint32_t* bad;   // [workers][4][Dv]: the first row of chunk c % 4 whose value is not finite
};

struct Seq {
  int row0, rows, slot, chunks, fresh;
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

// The launch sees to it that all chunks of a call count up to less than 2^31.
struct Walk {
  int x, end, seq_start;
  int s;
  Seq seq;
  int head, k0, n;  // the current piece: chunks [k0, k0 + n) of (sequence s, head)
  ASTERQ_DEVICE bool next(const Args& a) {
    if (x >= end) return false;
    while (x >= seq_start + seq.chunks * a.n_heads) {
      seq_start += seq.chunks * a.n_heads;
      seq = seq_of(a, ++s);
    }
    head = (x - seq_start) / seq.chunks;
    k0 = x - seq_start - head * seq.chunks;
    n = min(seq.chunks - k0, end - x);
    x += n;
    return true;
  }
};

// The same for the first pass: the chunks before each border that is inside a (sequence, head), back to the
// border before or the (sequence, head)'s start, laid end to end.
struct FirstWalk {
  int x, end;  // this CTA's share
  const int* before;     // [W + 1] chunks in front of those of border w
  const int* position;   // [W] the borders themselves
  const int* sequence;   // [W] the sequence that border w is in, and its first chunk
  const int* seq_start;
  int w;       // the border that the current piece belongs to
  Seq seq;
  int head, k0, n;
  ASTERQ_DEVICE bool next(const Args& a) {
    if (x >= end) return false;
    while (x >= before[w + 1]) ++w;
    seq = seq_of(a, sequence[w]);
    const int at = position[w] - (before[w + 1] - x) - seq_start[w];
    head = at / seq.chunks;
    k0 = at - head * seq.chunks;
    n = min(before[w + 1], end) - x;
    x += n;
    return true;
  }
};
template <bool kStateOnly>
struct WalkOf {
  using type = Walk;
};
template <>
struct WalkOf<true> {
  using type = FirstWalk;
};

template <int kDk, int kDv, bool kStateOnly>
struct Cfg {
  // Tiles of 128 tokens in shared memory.  Main pass: keys, values and queries of all chunks, in this order, take
  // five slots in turn.  Values, which are held longest (until A V of their chunk, during the next one) and have to
  // be checked, then follow queries into a slot and are asked for a whole chunk ahead; with two slots of
  // their own the products waited 2,000 of a chunk's 10,400 cycles for them.  First pass: three chunks' keys and values.
  static constexpr int kSlots = kStateOnly ? 6 : 5;
  // A chunk's tile: its slot, how many tiles that held before, and the barrier and phase of its arrival.  In the main
  // pass barriers belong to a kind of tile and not to a slot: whoever waits for a tile has seen the one before it on
  // the same barrier, and none has its barrier used again before all have seen it.
  struct Place {
    int slot, use, full, phase;
  };
  ASTERQ_DEVICE static Place keys_of(int c) {
    if (kStateOnly) return {2 * (c % 3), c / 3, kFull + 2 * (c % 3), c / 3};
    return {3 * c % 5, 3 * c / 5, kFull + (c & 1), c / 2};
  }
  ASTERQ_DEVICE static Place values_of(int c) {
    if (kStateOnly) return {2 * (c % 3) + 1, c / 3, kFull + 2 * (c % 3) + 1, c / 3};
    return {(3 * c + 1) % 5, (3 * c + 1) / 5, kFull + 2 + (c & 1), c / 2};
  }
  ASTERQ_DEVICE static Place queries_of(int c) { return {(3 * c + 2) % 5, (3 * c + 2) / 5, kFull + 4, c}; }
  static constexpr int kWBufs = kStateOnly ? 2 : 1;  // chunks' weights held (the main pass has no room for two)
  static constexpr int kMaxD = kDk > kDv ? kDk : kDv;
  static constexpr int kSlotBytes = kMaxD / 64 * kBoxBytes;
  // Tensor memory columns: A, the output, U (what a chunk adds to the state), and the keys' smaller and larger
  // parts.  Where there is room (the first pass has no outputs, and 64 value dims take half) the larger parts
  // have a place of their own and need not wait for the smaller parts' products, and the first pass adds a
  // chunk's U to the state while the next chunk's products run: 32768 tokens of 16 heads 276 -> 254 us, of 12 heads
  // of 64 x 64 dims 168 -> 158.
  static constexpr bool kTwoKeys = kStateOnly || kDv == 64;
  static constexpr uint32_t kColA = 0, kColO = 128, kColU = kStateOnly ? 0 : 128 + kDv, kColU1 = kStateOnly ? 128 : kColU,
                            kColK = kTwoKeys ? 256 : 384, kColL = 384;
  static constexpr int kStateBytes = kStateOnly ? 0 : kDk * kDv * 2;  // one bf16 part
  // barriers
  static constexpr int kFull = 0, kEmpty = kSlots, kQk = 2 * kSlots, kQs = kQk + 1, kULo = kQk + 2, kU = kQk + 3,
                       kO = kQk + 4, kKeys = kQk + 5, kKeysHi = kQk + 6, kS = kQk + 7, kA = kQk + 8,
                       kOFree = kQk + 9, kDrain = kQk + 10, kW = kQk + 11, kWFree = kQk + 13, kDecay = kQk + 15,
                       kDecayFree = kQk + 17, kChecked = kQk + 19, kBars = kQk + 23;
  static constexpr int kMiscBytes = 2 * (kChunk + 96) * 4 + 4 * 4 * 4 + kWBufs * 3 * kChunk * 2 + 16 + kBars * 8 + 28 * 4;
  static_assert(kWarps <= 16, "scan_s");
  static constexpr int kTableBytes = kStateOnly ? (4 * kThreads + 2) * 4 : 0;  // FirstWalk's arrays
  static constexpr int kSmem = kSlots * kSlotBytes + 2 * kStateBytes + kMiscBytes + kTableBytes;
};

ASTERQ_DEVICE void tma_rows(uint32_t dst, const CUtensorMap* map, int x, int head, int row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(head), "r"(row), "r"(bar)
      : "memory");
}

// A wait of a whole warp in as few instructions as its limit allows: the roles' loops together have to fit
// the instruction cache (unrolled, and with longer waits, they did not, and half of all issue slots went
// by without an instruction).  A round suspends for up to 20 us, so the limit is some seconds.
ASTERQ_DEVICE bool wait_for(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  uint32_t done;
  int rounds = 0;
  while ((done = mbar_try_sleep(bar, parity, 20000u)) == 0) {
    if (++rounds > (1 << 18)) *abort_flag = 1;
    if (ld_shared_volatile(abort_flag)) break;
  }
  return __all_sync(0xffffffffu, (int)done) != 0;
}

// x as a sum of bf16 parts, two values at a time, by cutting off: the next eight bits of each, packed, and
// the rest, which is exact.  Rounding instead would take cvt, a quarter-rate conversion of which this
// kernel would need 67,000 a chunk: it was what bound it.  Three parts leave less than 2^-24 of x, two
// less than 2^-16, towards zero.
ASTERQ_DEVICE uint32_t last_part(float x, float y) { return prmt(__float_as_uint(x), __float_as_uint(y), 0x7632); }
ASTERQ_DEVICE uint32_t split_part(float& x, float& y) {
  const uint32_t p = last_part(x, y);
  x -= __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  y -= __uint_as_float(__float_as_uint(y) & 0xffff0000u);
  return p;
}

// per bf16: the larger magnitude (its sign means nothing), or NaN
ASTERQ_DEVICE uint32_t max_abs_bf162(uint32_t x, uint32_t y) {
  uint32_t r;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}

ASTERQ_DEVICE void st_global_32(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

ASTERQ_DEVICE void ld_global_32(float* r, const float* p) {
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
               : "l"(p)
               : "memory");
}

// 2^x of a whole chunk's decay to fp32's last bit: a constant decay's error would add up over all the chunks
// it acts on.  x = n + r with |r| <= 1/2, 2^r by the series of e^(r ln 2), whose tenth term is below 2^-36.
ASTERQ_DEVICE float exp2_once(double x) {
  if (x < -160.0) return 0.0f;
  const double n = rint(x), r = (x - n) * 0.69314718055994530942;
  double y = 1.0;
#pragma unroll
  for (int i = 9; i > 0; --i) y = fma(y, r * (1.0 / i), 1.0);
  return ldexpf((float)y, (int)n);
}

template <int kDk, int kDv, bool kStateOnly>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                 const __grid_constant__ CUtensorMap v_map, const __grid_constant__ Args a,
                 const __grid_constant__ Work work) {
  using C = Cfg<kDk, kDv, kStateOnly>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t s_hi = base + C::kSlots * C::kSlotBytes, s_lo = s_hi + C::kStateBytes;
  // decays of a chunk (log2 of a token's, and what follows from them), by warp 14
  float* g_s = reinterpret_cast<float*>(smem + C::kSlots * C::kSlotBytes + 2 * C::kStateBytes);  // [2][kChunk], of the token after
  float* f_s = g_s + 2 * kChunk;  // [2][96]: 2^(from a token of the first three 32s to the end of its 32)
  float* p32_s = f_s + 2 * 96;    // [2][4]: 2^(each 32's decay)
  float* first_s = p32_s + 8;     // [2][4]: decays (log2) of each 32's first token
  uint16_t* w_s = reinterpret_cast<uint16_t*>(first_s + 8);      // [kWBufs][3][kChunk]: bf16 parts of the weight to the chunk's end
  float* whole_s = reinterpret_cast<float*>(w_s + C::kWBufs * 3 * kChunk);  // [4], kWBufs used: 2^(the chunk's decay)
  uint64_t* bars_s = reinterpret_cast<uint64_t*>(whole_s + 4);
  int* scan_s = reinterpret_cast<int*>(bars_s + C::kBars);  // [16]
  int* start_s = scan_s + 16;                               // sequence, its first chunk
  int* abort_s = start_s + 2;
  int* never_s = abort_s + 1;  // stays 0: the flag of waits that an abort must not cut short
  uint32_t* tmem_s = reinterpret_cast<uint32_t*>(abort_s + 2);
  int* bad_s = abort_s + 3;  // [4]: whether chunk c % 4 has values that are not finite
  [[maybe_unused]] int* table_s = abort_s + 10;
  const uint32_t bars = smem_u32(bars_s);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto bar = [&](int i) { return bars + 8 * i; };
  // A wait that runs into its limit raises the abort flag, every other wait then returns at once, and
  // each warp leaves its work as a whole and waits (again with a limit) for what it has in flight.
  auto wait = [&](int i, int phase) { return wait_for(bar(i), phase & 1, abort_s); };
  bool ok = true;
  // The chain's CTAs and then the main pass's are set up as SMs become free; they wait for what they read.
  if constexpr (kStateOnly) asm volatile("griddepcontrol.launch_dependents;");

  if (tid == 0) {
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(bar(C::kFull + i), 1);
      mbar_init(bar(C::kEmpty + i), 1);
    }
    for (int i : {C::kQk, C::kQs, C::kULo, C::kU, C::kO, C::kDrain, C::kDecay, C::kDecay + 1, C::kW, C::kW + 1})
      mbar_init(bar(i), 1);
    for (int i = 0; i < 4; ++i) mbar_init(bar(C::kChecked + i), 1);
    for (int i : {C::kKeys, C::kKeysHi, C::kS, C::kWFree, C::kWFree + 1}) mbar_init(bar(i), 8);
    for (int i : {C::kA, C::kOFree}) mbar_init(bar(i), 4);
    for (int i : {C::kDecayFree, C::kDecayFree + 1}) mbar_init(bar(i), 4);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *abort_s = 0;
    *never_s = 0;
  }

  // this CTA's share: a prefix sum over the sequences' chunks, thread t summing a strip of them
  const int strip = (a.n_seqs + kThreads - 1) / kThreads;
  const int s0 = min(tid * strip, a.n_seqs), s1 = min(s0 + strip, a.n_seqs);
  int sum = 0, disorder = 0;
  for (int s = s0; s < s1; ++s) {
    sum += seq_of(a, s).chunks;
    disorder |= __ldg(a.row_offsets + s + 1) < __ldg(a.row_offsets + s);
  }
  sum *= a.n_heads;
  int scan = sum;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int up = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += up;
  }
  if (lane == 31) scan_s[warp] = scan;
  // Sequences that share rows could count up to any number of chunks: offsets out of order leave the call undone.
  disorder = __syncthreads_or(disorder);
  int before = scan - sum, total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += scan_s[w];
    total += scan_s[w];
  }
  const int me = blockIdx.x;
  if (disorder) {
    total = 0;
    if (!kStateOnly && me == 0 && tid == 0 && a.status) atomicMax(a.status, 1);
  }
  // As many shares as the longest needs: fewer cuts inside a (sequence, head).
  const int longest = max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x);
  const int W = max(1, (total + longest - 1) / longest);
  auto border = [&](int w) { return (int)((long long)total * w / W); };
  typename WalkOf<kStateOnly>::type walk;
  if constexpr (!kStateOnly) {
    walk.x = me < W ? border(me) : total;
    walk.end = me < W ? border(me + 1) : total;
    if (walk.x < walk.end && before <= walk.x && walk.x < before + sum) {
      int s = s0, at = before;
      while (true) {
        const int here = seq_of(a, s).chunks * a.n_heads;
        if (walk.x < at + here) break;
        at += here;
        ++s;
      }
      start_s[0] = s;
      start_s[1] = at;
    }
    // rows of empty slots are zeros; ranges out of bounds are reported
    for (int s = me; s < a.n_seqs; s += gridDim.x) {
      const Seq q = seq_of(a, s);
      if (q.chunks > 0) continue;
      const int begin = __ldg(a.row_offsets + s), end = __ldg(a.row_offsets + s + 1);
      if (tid == 0 && a.status && (begin < 0 || end > a.n_rows || (q.rows > 0 && q.slot >= a.n_slots)))
        atomicMax(a.status, 1);
      uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (long long)q.row0 * a.n_heads * kDv);
      for (long long i = tid; i < (long long)q.rows * a.n_heads * (kDv / 8); i += kThreads)
        dst[i] = make_uint4(0, 0, 0, 0);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // every thread, also of a CTA without a share
    __syncthreads();
    if (walk.x >= walk.end) return;
    walk.s = start_s[0];
    walk.seq_start = start_s[1];
    walk.seq = seq_of(a, walk.s);
  } else {
    // Thread w looks where border w is and how many chunks before it the first pass needs.
    int* strips = reinterpret_cast<int*>(smem);  // the tiles' place, not used yet: [kThreads]
    int* tables = table_s;                       // 4 arrays of kThreads + 1
    strips[tid] = before;
    __syncthreads();
    const int w = tid;
    int need = 0, s = 0, at = 0, unit = 0;
    if (w > 0 && w < W) {
      const int pos = border(w);
      int lo = 0, hi = kThreads - 1;
      while (lo < hi) {  // the last strip that starts at pos or before
        const int mid = (lo + hi + 1) / 2;
        if (strips[mid] <= pos) lo = mid;
        else hi = mid - 1;
      }
      s = lo * strip;
      at = strips[lo];
      int chunks;
      while (true) {
        chunks = seq_of(a, s).chunks;
        if (pos < at + chunks * a.n_heads) break;
        at += chunks * a.n_heads;
        ++s;
      }
      unit = pos - (pos - at) % chunks;
      if (unit < pos) need = pos - max(border(w - 1), unit);
    }
    scan = need;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int up = __shfl_up_sync(0xffffffffu, scan, d);
      if (lane >= d) scan += up;
    }
    if (lane == 31) scan_s[warp] = scan;
    __syncthreads();
    int ahead = scan - need, all = 0;
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) ahead += scan_s[i];
      all += scan_s[i];
    }
    tables[w] = ahead;
    if (w == kThreads - 1) tables[kThreads] = all;
    tables[kThreads + 1 + w] = border(min(w, W));
    tables[2 * kThreads + 1 + w] = s;
    tables[3 * kThreads + 1 + w] = at;
    // part i of worker m at border w is number w + m: both go up together along the chunks
    if (w == me && w < (int)gridDim.x) {
      const bool starts = need > 0 && unit >= border(w - 1);
      work.first[w] = starts ? w + (int)(((long long)(ahead + 1) * W - 1) / all) : -1;
    }
    fence_async_shared();  // the copy engine writes tiles over `strips`
    __syncthreads();
    walk.x = me < W ? (int)((long long)all * me / W) : all;
    walk.end = me < W ? (int)((long long)all * (me + 1) / W) : all;
    if (walk.x >= walk.end) return;
    walk.before = tables;
    walk.position = tables + kThreads + 1;
    walk.sequence = tables + 2 * kThreads + 1;
    walk.seq_start = tables + 3 * kThreads + 1;
    walk.w = 0;
  }

  if (warp == 13) tc::alloc512(smem_u32(tmem_s));
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_s;

  // Registers of a thread by role: 128 (kRegsA + 2 kRegsS + kRegsIssue) of the 512 x 128 that the block was
  // launched with.
  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
    if (warp == 12) {
      // -------------------------------------------------------------- loads
      int c = 0;
      while (ok && walk.next(a)) {
        // the state that the piece starts from, for the warps that will want it about a chunk later
        if (!kStateOnly && walk.k0 == 0 && !walk.seq.fresh && lane == 0)
          asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(
                           a.state + ((long long)walk.seq.slot * a.n_heads + walk.head) * kDk * kDv),
                       "r"(kDk * kDv * 4)
                       : "memory");
        for (int j = 0; j < walk.n && ok; ++j, ++c) {
          const int row = walk.seq.row0 + (walk.k0 + j) * kChunk;
          // values first: their slot is the first to be free (but the very first chunk starts with its keys)
#pragma unroll 1
          for (int i = 0; i < (kStateOnly ? 2 : 3); ++i) {
            const int tile = i == 2 ? 2 : (i + (c > 0 && !kStateOnly)) & 1;
            const typename C::Place at = tile == 0 ? C::keys_of(c) : tile == 1 ? C::values_of(c) : C::queries_of(c);
            const CUtensorMap* map = tile == 0 ? &k_map : tile == 1 ? &v_map : &q_map;
            const int boxes = tile == 1 ? kDv / 64 : kDk / 64;
            if (at.use > 0) ok = wait(C::kEmpty + at.slot, at.use - 1);
            if (!ok) break;
            if (lane == 0) {
              mbar_expect_tx(bar(at.full), boxes * kBoxBytes);
#pragma unroll 1
              for (int b = 0; b < boxes; ++b)
                tma_rows(base + at.slot * C::kSlotBytes + b * kBoxBytes, map, b * 64, walk.head, row,
                         bar(at.full));
            }
          }
        }
      }
      // the last copies have landed before the exit, also when nobody waits for them any more (the slots'
      // last uses: of the chunk before this one, whichever was reached)
      if (!ok) {
        for (int last = max(0, c - 2); last <= c; ++last) {
          (void)mbar_wait(bar(C::keys_of(last).full), C::keys_of(last).phase & 1, never_s, 200000000);
          (void)mbar_wait(bar(C::values_of(last).full), C::values_of(last).phase & 1, never_s, 200000000);
          if (!kStateOnly)
            (void)mbar_wait(bar(C::queries_of(last).full), C::queries_of(last).phase & 1, never_s, 200000000);
        }
      }
    } else if (warp == 13) {
      // -------------------------------------------------------------- products
      constexpr uint32_t kQkDesc = tc::idesc_bf16(kChunk, false), kVDesc = tc::idesc_bf16(kDv, true);
      // steps of 16 tokens: eight of them but in a sequence's last chunk.  Rolled: under elect an unrolled loop
      // issues no faster, and the instruction cache is short.
      auto over_tokens = [&](int steps, auto step) {
#pragma unroll 1
        for (int s = 0; s < steps; ++s) step(s);
      };
      // The order of a chunk's products follows the state warps, on whose loop everything waits: the smaller
      // parts of the keys; A V of the chunk before (its A is made by now) while they make the larger parts;
      // those; and Q K^T and Q S while they update S and weigh the next keys.
      int last_steps = 0, last_carried = 0;
      auto a_times_v = [&](int c) {
        ok = wait(C::kA, c);
        if (!ok) return;
        tc::fence_after();
        if (tc::elect()) {
          const uint32_t v_desc = tc::desc_mn_major(base + C::values_of(c).slot * C::kSlotBytes, kBoxBytes);
          over_tokens(last_steps, [&](int s) {
            const uint32_t at = tmem + C::kColA + 16 * s;
            tc::mma_ts(tmem + C::kColO, at, v_desc + s * 128, kVDesc, last_carried || s > 0);
            tc::mma_ts(tmem + C::kColO, at + 8, v_desc + s * 128, kVDesc, true);
          });
          tc::commit(bar(C::kO));
          tc::commit(bar(C::kEmpty + C::values_of(c).slot));
        }
      };
      int c = 0;
      while (ok && walk.next(a))
        for (int j = 0; j < walk.n; ++j, ++c) {
          const int rows = min(kChunk, walk.seq.rows - (walk.k0 + j) * kChunk), steps = (rows + 15) / 16;
          const typename C::Place kp = C::keys_of(c), vp = C::values_of(c);
          const uint32_t v_desc = tc::desc_mn_major(base + vp.slot * C::kSlotBytes, kBoxBytes);
          const uint32_t u = tmem + (c & 1 ? C::kColU1 : C::kColU);
          ok = wait(vp.full, vp.phase) && (kStateOnly || wait(C::kChecked + (c & 3), c / 4)) && wait(C::kKeys, c);
          if (!ok) break;
          tc::fence_after();
          if (tc::elect()) {
            over_tokens(steps, [&](int s) { tc::mma_ts(u, tmem + C::kColK + 8 * s, v_desc + s * 128, kVDesc, s > 0); });
            over_tokens(steps, [&](int s) { tc::mma_ts(u, tmem + C::kColK + 64 + 8 * s, v_desc + s * 128, kVDesc, true); });
            tc::commit(bar(C::kULo));
          }
          if (!kStateOnly && c > 0) a_times_v(c - 1);
          ok = ok && wait(C::kKeysHi, c);
          if (!ok) break;
          tc::fence_after();
          if (tc::elect()) {
            over_tokens(steps, [&](int s) { tc::mma_ts(u, tmem + C::kColL + 8 * s, v_desc + s * 128, kVDesc, true); });
            over_tokens(steps, [&](int s) { tc::mma_ts(u, tmem + C::kColL + 64 + 8 * s, v_desc + s * 128, kVDesc, true); });
            tc::commit(bar(C::kU));
            if (kStateOnly) {
              tc::commit(bar(C::kEmpty + kp.slot));
              tc::commit(bar(C::kEmpty + vp.slot));
            }
          }
          const typename C::Place qp = C::queries_of(c);
          const uint32_t q_desc = tc::desc_k_major(base + qp.slot * C::kSlotBytes);
          if constexpr (!kStateOnly) {
            // the columns that Q K^T goes to are free when the last chunk's A has been read
            ok = wait(kp.full, kp.phase) && wait(qp.full, qp.phase) && (c == 0 || wait(C::kO, c - 1));
            if (!ok) break;
            if (tc::elect()) {
              const uint32_t k_desc = tc::desc_k_major(base + kp.slot * C::kSlotBytes);
#pragma unroll 1
              for (int s = 0; s < kDk / 16; ++s) {
                const uint32_t at = ((s / 4) * kBoxBytes + (s % 4) * 32) >> 4;
                tc::mma_ss(tmem + C::kColA, q_desc + at, k_desc + at, kQkDesc, s > 0);
              }
              tc::commit(bar(C::kQk));
              tc::commit(bar(C::kEmpty + kp.slot));
            }
          }
          if constexpr (!kStateOnly) {
            const bool carried = walk.k0 + j > 0 || !walk.seq.fresh;  // S is not zero by construction
            ok = wait(C::kS, c) && (c == 0 || wait(C::kOFree, c - 1));
            if (!ok) break;
            tc::fence_after();
            if (tc::elect()) {
              if (carried) {
                const uint32_t hi_desc = tc::desc_mn_major(s_hi, kDk * 128), lo_desc = tc::desc_mn_major(s_lo, kDk * 128);
#pragma unroll 1
                for (int s = 0; s < kDk / 16; ++s) {
                  const uint32_t at = ((s / 4) * kBoxBytes + (s % 4) * 32) >> 4;
                  tc::mma_ss(tmem + C::kColO, q_desc + at, hi_desc + s * 128, kVDesc, s > 0);
                  tc::mma_ss(tmem + C::kColO, q_desc + at, lo_desc + s * 128, kVDesc, true);
                }
              }
              tc::commit(bar(C::kQs));
              tc::commit(bar(C::kEmpty + qp.slot));
            }
            last_steps = steps;
            last_carried = carried;
          }
        }
      if (!kStateOnly && ok) a_times_v(c - 1);
      // every product and every arrival above is done before the tensor memory goes back
      if (tc::elect()) tc::commit(bar(C::kDrain));
      (void)mbar_wait(bar(C::kDrain), 0, never_s);
    } else if (warp == 14) {
      // -------------------------------------------------------------- decays
      // Lane i has tokens 4 i .. 4 i + 3, eight lanes a 32.  Everything is a sum of what follows, never a
      // difference: a decay of -inf, or one that outweighs the others, costs the tokens after it nothing.
      double decay = 0.0;
      int c = 0;
      while (ok && walk.next(a)) {
        float next[4];
        auto read = [&](int j) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = (walk.k0 + j) * kChunk + 4 * lane + e;
            next[e] = j < walk.n && at < walk.seq.rows
                          ? __ldg(a.log_decay + (long long)(walk.seq.row0 + at) * a.decay_row + walk.head) : 0.0f;
          }
        };
        read(0);
        for (int j = 0; j < walk.n; ++j, ++c) {
          float g[4], after[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) g[e] = next[e] * kLog2e;
          read(j + 1);
          after[3] = 0.0f;
#pragma unroll
          for (int e = 2; e >= 0; --e) after[e] = after[e + 1] + g[e + 1];
          float sum = after[0] + g[0];  // from this lane's first token to the end of its 32
#pragma unroll
          for (int d = 1; d < 8; d *= 2) {
            const float down = __shfl_down_sync(0xffffffffu, sum, d);
            if ((lane & 7) + d < 8) sum += down;
          }
          float later = __shfl_down_sync(0xffffffffu, sum, 1);
          if ((lane & 7) == 7) later = 0.0f;
          const float all = __shfl_sync(0xffffffffu, sum, 8 * (lane & 3));  // the decay of 32 number lane % 4
          float beyond = 0.0f;                                              // of the 32s after it
#pragma unroll
          for (int e = 1; e < 4; ++e) {
            const float x = __shfl_sync(0xffffffffu, all, (lane & 3) + e < 4 ? (lane & 3) + e : 0);
            if ((lane & 3) + e < 4) beyond += x;
          }
          double whole = ((double)g[0] + g[1]) + ((double)g[2] + g[3]);
#pragma unroll
          for (int d = 16; d > 0; d /= 2) whole += __shfl_xor_sync(0xffffffffu, whole, d);
          decay += whole;
          if constexpr (!kStateOnly) {
            const int buf = c & 1;
            if (c >= 2) {
              ok = wait(C::kDecayFree + buf, c / 2 - 1);
              if (!ok) break;
            }
            const float after_lane = __shfl_down_sync(0xffffffffu, g[0], 1);
            reinterpret_cast<float4*>(g_s + buf * kChunk)[lane] = make_float4(g[1], g[2], g[3], after_lane);
            if (lane % 8 == 0) first_s[buf * 4 + lane / 8] = g[0];
            if (lane < 24)
              reinterpret_cast<float4*>(f_s + buf * 96)[lane] = make_float4(
                  ex2_ftz(after[0] + later), ex2_ftz(after[1] + later), ex2_ftz(after[2] + later),
                  ex2_ftz(after[3] + later));
            if (lane < 4) p32_s[buf * 4 + lane] = ex2_ftz(all);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(C::kDecay + buf));
          }
          later += __shfl_sync(0xffffffffu, beyond, lane / 8);
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = ex2_ftz(after[e] + later);
          const int wb = c % C::kWBufs;
          if (c >= C::kWBufs) {
            ok = wait(C::kWFree + wb, c / C::kWBufs - 1);
            if (!ok) break;
          }
#pragma unroll
          for (int part = 0; part < 3; ++part) {
            const uint32_t w01 = split_part(w[0], w[1]), w23 = split_part(w[2], w[3]);
            reinterpret_cast<uint2*>(w_s + (wb * 3 + part) * kChunk)[lane] = make_uint2(w01, w23);
          }
          if (lane == 0) whole_s[wb] = exp2_once(whole);
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::kW + wb));
        }
        if constexpr (kStateOnly) {
          if (lane == 0) {
            const int w = walk.w, at_border = walk.x == walk.before[w + 1];
            Part p;
            p.decay = exp2_once(decay);
            p.slot = walk.seq.slot;
            p.head = walk.head;
            p.fresh = walk.seq.fresh;
            p.border = at_border ? w : -1;
            const int all = walk.before[kThreads];
            auto worker_of = [&](int x) { return (int)(((long long)(x + 1) * W - 1) / all); };
            p.next = at_border ? -1 : w + worker_of(walk.x);
            if (at_border) {
              // the (sequence, head) goes on to the next border, or ends before it
              const int unit = walk.position[w] - walk.k0 - walk.n;
              const bool more = w + 1 < W && walk.before[w + 2] > walk.before[w + 1] &&
                                walk.position[w + 1] < unit + walk.seq.chunks;
              p.next = more ? w + 1 + worker_of(walk.x) : -1;
            }
            work.parts[w + me] = p;
          }
          decay = 0.0;
        }
      }
    } else if (!kStateOnly) {
      // -------------------------------------------------------------- values that are not finite
      // A's zeros above the diagonal do not cancel them, so rows before them would become NaN.  They are
      // taken out here; the warps of the output and of the state write NaN in their column from their row on.
      int c = 0;
      while (ok && walk.next(a))
        for (int j = 0; j < walk.n; ++j, ++c) {
          const int rows = min(kChunk, walk.seq.rows - (walk.k0 + j) * kChunk);
          const typename C::Place vp = C::values_of(c);
          uint8_t* tile = smem + vp.slot * C::kSlotBytes;
          ok = wait(vp.full, vp.phase);
          if (!ok) break;
          uint32_t most = 0;
#pragma unroll 1
          for (int at = lane * 16; at < kDv / 64 * kBoxBytes; at += 4 * 512) {
            uint4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
              x[u] = (at + u * 512) % kBoxBytes < rows * 128 ? *reinterpret_cast<const uint4*>(tile + at + u * 512)
                                                             : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int u = 0; u < 4; ++u)
              most = max_abs_bf162(max_abs_bf162(max_abs_bf162(max_abs_bf162(most, x[u].x), x[u].y), x[u].z), x[u].w);
          }
          const bool any = __any_sync(0xffffffffu, (most & 0x7fffu) >= 0x7f80u || (most >> 16 & 0x7fffu) >= 0x7f80u);
          if (any) {
#pragma unroll 1
            for (int d = lane; d < kDv; d += 32) {
              uint32_t first = 0;  // or NaN with the column's first row in its last bits
#pragma unroll 1
              for (int row = rows - 1; row >= 0; --row) {
                uint16_t* x = reinterpret_cast<uint16_t*>(tile + d / 64 * kBoxBytes + row * 128 +
                                                          (((d % 64 / 8) ^ (row & 7)) << 4)) + d % 8;
                if ((*x & 0x7f80) != 0x7f80) continue;
                *x = 0;
                first = 0x7fc00000u | row;
              }
              work.bad[(me * 4 + (c & 3)) * kDv + d] = first;
            }
            fence_async_shared();
          }
          if (lane == 0) bad_s[c & 3] = any;
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::kChecked + (c & 3)));
        }
    }
  } else if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsA));
    // ---------------------------------------------------------------- A and the output
    if constexpr (!kStateOnly) {
      const uint32_t lanes = tmem + ((uint32_t)warp << 21);  // this warp's 32 lanes
      const int i = warp * 32 + lane;                        // row of the chunk
      int c = 0;
      while (ok && walk.next(a))
        for (int j = 0; j < walk.n; ++j, ++c) {
          const int rows = min(kChunk, walk.seq.rows - (walk.k0 + j) * kChunk), steps = (rows + 15) / 16;
          const bool carried = walk.k0 + j > 0 || !walk.seq.fresh;
          uint32_t r[32];
          const float* g = g_s + (c & 1) * kChunk;
          const float* f = f_s + (c & 1) * 96;
          const float* p32 = p32_s + (c & 1) * 4;
          ok = wait(C::kDecay + (c & 1), c / 2) && wait(C::kQk, c);
          if (!ok) break;
          tc::fence_after();
          // A step of 16 columns at a time, in place: eight columns of leading parts, eight of the rest.
          // The row's own 32 columns: 2^G_ij from the diagonal back, sums that are exact where they matter.
          uint32_t x[16];
          float sum = 0.0f;
#pragma unroll 1
          for (int half = 1; half >= 0; --half) {
            const uint32_t at = lanes + C::kColA + 32 * warp + 16 * half;
            const float4* next = reinterpret_cast<const float4*>(g + 32 * warp + 16 * half);
            const int left = lane - 16 * half;  // columns of this step before the row's own
            tc::ld16(x, at);
            uint32_t out[16];
            tc::wait_ld();
#pragma unroll
            for (int e = 3; e >= 0; --e) {
              const float4 w = next[e];
              float y[4];
              const float step[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int h = 3; h >= 0; --h) {
                const int col = 4 * e + h;
                sum += col < left ? step[h] : 0.0f;
                const float product = __uint_as_float(x[col]) * (ex2_ftz(sum) * a.scale);
                y[h] = col <= left ? product : 0.0f;
              }
              out[2 * e] = split_part(y[0], y[1]);
              out[8 + 2 * e] = last_part(y[0], y[1]);
              out[2 * e + 1] = split_part(y[2], y[3]);
              out[8 + 2 * e + 1] = last_part(y[2], y[3]);
            }
            tc::st16(at, out);
          }
          // The 32s before it: 2^(from the 32's end to the row) times 2^(from the column to the 32's end).
          float far = ex2_ftz(sum + first_s[(c & 1) * 4 + warp]) * a.scale;
#pragma unroll 1
          for (int step = 2 * warp - 1; step >= 0; --step) {
            tc::ld16(x, lanes + C::kColA + 16 * step);
            const float4* fg = reinterpret_cast<const float4*>(f + 16 * step);
            tc::wait_ld();
            uint32_t out[16];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 w = fg[e];
              float x0 = __uint_as_float(x[4 * e]) * far * w.x, x1 = __uint_as_float(x[4 * e + 1]) * far * w.y;
              float x2 = __uint_as_float(x[4 * e + 2]) * far * w.z, x3 = __uint_as_float(x[4 * e + 3]) * far * w.w;
              out[2 * e] = split_part(x0, x1);
              out[8 + 2 * e] = last_part(x0, x1);
              out[2 * e + 1] = split_part(x2, x3);
              out[8 + 2 * e + 1] = last_part(x2, x3);
            }
            tc::st16(lanes + C::kColA + 16 * step, out);
            if (step % 2 == 0) far *= p32[step / 2];
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = 0;
#pragma unroll 1
          for (int step = 2 * warp + 2; step < steps; ++step) tc::st16(lanes + C::kColA + 16 * step, x);
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::kDecayFree + (c & 1)));
          ok = wait(C::kQs, c) && wait(C::kChecked + (c & 3), c / 4);
          if (!ok) break;
          tc::fence_after();
          if (carried) {
#pragma unroll 1
            for (int d = 0; d < kDv; d += 32) {
              tc::ld32(r, lanes + C::kColO + d);
              tc::wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * far);
              tc::st32(lanes + C::kColO + d, r);
            }
          }
          tc::wait_st();
          tc::fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::kA));
          ok = wait(C::kO, c);
          if (!ok) break;
          tc::fence_after();
          const long long row = walk.seq.row0 + (walk.k0 + j) * kChunk + i;
          uint16_t* dst = static_cast<uint16_t*>(a.out) + (row * a.n_heads + walk.head) * kDv;
#pragma unroll 1
          for (int d = 0; d < kDv; d += 32) {
            tc::ld32(r, lanes + C::kColO + d);
            tc::wait_ld();
            if (d + 32 == kDv) {
              tc::fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(C::kOFree));
            }
            if (i >= rows) continue;
            // whole sectors of a row at a time
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t p[8];
#pragma unroll
              for (int h = 0; h < 8; ++h)
                p[h] = pack_bf162(__uint_as_float(r[16 * e + 2 * h]), __uint_as_float(r[16 * e + 2 * h + 1]));
              st_global_32(dst + d + 16 * e, p);
            }
          }
          if (bad_s[c & 3] && i < rows) {
            const uint32_t* bad = work.bad + (me * 4 + (c & 3)) * kDv;
#pragma unroll 1
            for (int d = 0; d < kDv; ++d)
              if (bad[d] && (int)(bad[d] & (kChunk - 1)) <= i) dst[d] = 0x7fff;
          }
        }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsS));
    // ---------------------------------------------------------------- keys and state
    constexpr int kCols = kDv / 2;
    const int part = (warp - 4) >> 2;               // tokens 64 part .., value dims kCols part ..
    const int dk = (warp & 3) * 32 + lane;          // key dim
    const bool has = kDk == 128 || (warp & 3) < 2;  // whole warps
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    // ldmatrix rows: lane -> token lane % 8 of an 8-token block, 8 key dims lane / 8 of the warp's 32
    const uint32_t k_row = ((warp & 3) / 2) * kBoxBytes + (part * 64 + (lane & 7)) * 128 +
                           (((((warp & 3) % 2) * 4 + (lane >> 3)) ^ (lane & 7)) << 4);
    float s[kCols];
    // s <- f s + what chunk c has added
    auto add = [&](int c, float f) {
      tc::fence_after();
      if (has) {
#pragma unroll
        for (int d = 0; d < kCols; d += 32) {
          uint32_t r[32];
          tc::ld32(r, lanes + (c & 1 ? C::kColU1 : C::kColU) + part * kCols + d);
          tc::wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) s[d + e] = fmaf(f, s[d + e], __uint_as_float(r[e]));
        }
      }
    };
    float last_whole = 0.0f;
    int c = 0;
    while (ok && walk.next(a)) {
      const Seq q = walk.seq;
      const bool ends = walk.k0 + walk.n == q.chunks;
      const long long slot_at = (((long long)q.slot * a.n_heads + walk.head) * kDk + dk) * kDv + part * kCols;
      const long long piece_at = (long long)dk * kDv + part * kCols;
      // the state at the piece's start
      const float* from = nullptr;
      if (!kStateOnly) {
        if (walk.k0 > 0) from = work.borders + (long long)me * kDk * kDv + piece_at;
        else if (q.fresh) from = nullptr;
        else from = ends ? a.state + slot_at : work.starts + (long long)(me + 1) * kDk * kDv + piece_at;
      }
      if (from && has) {
#pragma unroll
        for (int e = 0; e < kCols; e += 8) ld_global_32(s + e, from + e);
      } else {
#pragma unroll
        for (int e = 0; e < kCols; ++e) s[e] = 0.0f;
      }
      for (int j = 0; j < walk.n; ++j, ++c) {
        const int rows = min(kChunk, q.rows - (walk.k0 + j) * kChunk), steps = (rows + 15) / 16;
        // the keys, weighted and split: thread t has key dims t / 4 + 8 m and tokens 2 (t % 4), + 1 of each block
        const typename C::Place kp = C::keys_of(c), vp = C::values_of(c);
        const uint32_t k_at = base + kp.slot * C::kSlotBytes + k_row;
        const int wb = c % C::kWBufs;
        const uint32_t* weight = reinterpret_cast<const uint32_t*>(w_s) + wb * 192 + part * 32 + (lane & 3);
        ok = wait(C::kW + wb, c / C::kWBufs) && wait(kp.full, kp.phase) && (!C::kTwoKeys || c == 0 || wait(C::kULo, c - 1));
        if (!ok) break;
        tc::fence_after();
        const float whole = whole_s[wb];
        // 32 tokens of the warp's 32 key dims: values 4 h + m are key dims 8 m .. of tokens 8 h ..
        auto put = [&](uint32_t to, const uint32_t (&p)[16]) {
          tc::st_16x128b_x4(to, p[0], p[1], p[4], p[5], p[8], p[9], p[12], p[13]);
          tc::st_16x128b_x4(to + (16u << 16), p[2], p[3], p[6], p[7], p[10], p[11], p[14], p[15]);
        };
        const int units = has ? min(2, (rows - part * 64 + 31) / 32) : 0;  // 32s of tokens here; may be < 0
        if (rows < kChunk && has) {
          // keys past the sequence's end, where this warp would read them: zeros (a weight of zero would
          // not clear a NaN)
          for (int e = lane + 4 * max(0, rows - part * 64); e < 4 * 64; e += 32) {
            const int tok = part * 64 + e / 4, unit = ((warp & 3) % 2) * 4 + e % 4;
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                             base + kp.slot * C::kSlotBytes + ((warp & 3) / 2) * kBoxBytes + tok * 128 +
                             ((unit ^ (tok & 7)) << 4)),
                         "r"(0)
                         : "memory");
          }
          fence_async_shared();  // the slot's next tile is written by the copy engine
          __syncwarp();
        }
        {
#pragma unroll 1
          for (int u = 0; u < units; ++u) {
            uint32_t m[16], l[16];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              uint32_t k[4];
              ldmatrix_x4_trans(k, k_at + (4 * u + h) * 1024);
              const uint32_t w2 = weight[64 + (4 * u + h) * 4], w3 = weight[128 + (4 * u + h) * 4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                m[h * 4 + e] = tc::mul_bf162(k[e], w2);
                l[h * 4 + e] = tc::fma_bf162(k[e], w3, tc::fma_bf162(k[e], w2, tc::neg_bf162(m[h * 4 + e])));
              }
            }
            put(lanes + C::kColK + part * 32 + u * 16, l);
            put(lanes + C::kColK + 64 + part * 32 + u * 16, m);
          }
        }
        ok = wait(vp.full, vp.phase);
        if (!ok) break;
        if (rows < steps * 16) {
          // the last chunk's products run over whole steps of 16 tokens: values past the end are zeros
          const uint32_t v_at = base + vp.slot * C::kSlotBytes;
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
        if (C::kTwoKeys) ok = !kStateOnly || c == 0 || wait(C::kU, c - 1);
        else ok = wait(C::kULo, c);
        ok = ok && (kStateOnly || wait(C::kChecked + (c & 3), c / 4));
        if (!ok) break;
        tc::fence_after();
        // the larger parts in their place
#pragma unroll 1
        for (int u = 0; u < units; ++u) {
          uint32_t p1[16], p2[16];
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            uint32_t k[4];
            ldmatrix_x4_trans(k, k_at + (4 * u + h) * 1024);
            const uint32_t w1 = weight[(4 * u + h) * 4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              p1[h * 4 + e] = tc::mul_bf162(k[e], w1);
              p2[h * 4 + e] = tc::fma_bf162(k[e], w1, tc::neg_bf162(p1[h * 4 + e]));
            }
          }
          put(lanes + C::kColL + part * 32 + u * 16, p2);
          put(lanes + C::kColL + 64 + part * 32 + u * 16, p1);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kWFree + wb));
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kKeysHi));

        // S for this chunk's outputs, over the one that the last chunk's have read
        if (!kStateOnly) {
          if (c > 0) ok = wait(C::kQs, c - 1);
          if (!ok) break;
        }
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
              lo[h] = last_part(x, y);
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
        if (!kStateOnly) {
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::kS));
        }

        if (kStateOnly) {
          if (j > 0) add(c - 1, last_whole);
          last_whole = whole;
          if (j + 1 < walk.n) continue;
        }
        ok = wait(C::kU, c);
        if (!ok) break;
        add(c, whole);
        if (has) {
          if (!kStateOnly && bad_s[c & 3]) {
            const uint32_t* bad = work.bad + (me * 4 + (c & 3)) * kDv + part * kCols;
#pragma unroll
            for (int d = 0; d < kCols; d += 4) {
              const uint4 x = *reinterpret_cast<const uint4*>(bad + d);
              s[d] += __uint_as_float(x.x);
              s[d + 1] += __uint_as_float(x.y);
              s[d + 2] += __uint_as_float(x.z);
              s[d + 3] += __uint_as_float(x.w);
            }
          }
        }
      }
      if (!ok) break;
      float* to = nullptr;
      if constexpr (kStateOnly) to = work.sums + (long long)(walk.w + me) * kDk * kDv + piece_at;
      else if (ends) to = a.state + slot_at;
      if (to && has) {
#pragma unroll
        for (int e = 0; e < kCols; e += 8) {
          uint32_t p[8];
#pragma unroll
          for (int h = 0; h < 8; ++h) p[h] = __float_as_uint(s[e + h]);
          st_global_32(to + e, p);
        }
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

// The states at the borders inside a (sequence, head), one thread for four values: block b follows the
// parts of the one whose first cut is border b.
template <int kDk, int kDv>
__global__ void __launch_bounds__(256) chain_kernel(const __grid_constant__ Args a, const __grid_constant__ Work work) {
  __shared__ Part parts[2 * kThreads];
  __shared__ int list[2 * kThreads], count;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");  // all CTAs: the next grid takes this one's end for both
  const int first = work.first[blockIdx.x];
  if (first < 0) return;
  // the parts that may belong to it, then their order: a chain of loads from memory would take longer than
  // all the rest
  for (int i = first + threadIdx.x; i < 2 * (int)gridDim.x; i += 256) parts[i] = work.parts[i];
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0;
    for (int i = first; i >= 0 && n < 2 * (int)gridDim.x; i = parts[i].next) list[n++] = i;
    count = n;
  }
  __syncthreads();
  const long long at = ((long long)blockIdx.y * 256 + threadIdx.x) * 4;
  const Part p0 = parts[first];
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (!p0.fresh)
    s = *reinterpret_cast<const float4*>(a.state + ((long long)p0.slot * a.n_heads + p0.head) * kDk * kDv + at);
  *reinterpret_cast<float4*>(work.starts + (long long)blockIdx.x * kDk * kDv + at) = s;
  const int n = count;
#pragma unroll 4
  for (int k = 0; k < n; ++k) {
    const int i = list[k];
    const float4 u = __ldcg(reinterpret_cast<const float4*>(work.sums + (long long)i * kDk * kDv + at));
    const float f = parts[i].decay;
    s.x = fmaf(f, s.x, u.x);
    s.y = fmaf(f, s.y, u.y);
    s.z = fmaf(f, s.z, u.z);
    s.w = fmaf(f, s.w, u.w);
    if (parts[i].border >= 0)
      *reinterpret_cast<float4*>(work.borders + (long long)parts[i].border * kDk * kDv + at) = s;
  }
}

// rows of bf16 heads [n_rows][n_heads][dim] with any strides, read in boxes of 128 rows x 64 dims
bool make_map(CUtensorMap* map, const void* base, const Args& a, int dim, long long row_stride, long long head_stride) {
  const EncodeTiled fn = encode_tiled();
  // outputs and states are read and written 32 bytes at a time
  if ((reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.state)) & 31) return false;
  if ((a.n_rows / kChunk + a.n_seqs) * a.n_heads > 0x7fffffff) return false;  // Walk counts in 32 bits
  if (!fn || row_stride <= 0 || head_stride <= 0) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)a.n_heads, (cuuint64_t)a.n_rows};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)row_stride * 2};
  const cuuint32_t box[3] = {64u, 1u, (cuuint32_t)kChunk}, step[3] = {1u, 1u, 1u};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t table_bytes(int workers) {
  return (2 * workers * (int64_t)sizeof(Part) + workers * (int64_t)sizeof(int) + 255) / 256 * 256;
}

template <int kDk, int kDv>
int launch(const Args& a, int workers, int device, void* workspace, cudaStream_t s) {
  using First = Cfg<kDk, kDv, true>;
  using Main = Cfg<kDk, kDv, false>;
  CUtensorMap q_map, k_map, v_map;
  if (!make_map(&q_map, a.q, a, kDk, a.q_row, a.q_head) || !make_map(&k_map, a.k, a, kDk, a.k_row, a.k_head) ||
      !make_map(&v_map, a.v, a, kDv, a.v_row, a.v_head) || (reinterpret_cast<uintptr_t>(workspace) & 31))
    return ASTERQ_ERR_UNSUPPORTED;
  const std::lock_guard<std::mutex> guard(launch_lock());
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
  char* at = static_cast<char*>(workspace);
  work.parts = reinterpret_cast<Part*>(at);
  work.first = reinterpret_cast<int*>(at + 2 * workers * sizeof(Part));
  work.sums = reinterpret_cast<float*>(at + table_bytes(workers));
  work.borders = work.sums + 2ll * workers * kDk * kDv;
  work.starts = work.borders + (long long)workers * kDk * kDv;
  work.bad = reinterpret_cast<uint32_t*>(work.starts + (long long)workers * kDk * kDv);
  // Rows of one chunk cannot be a sequence of two: no cut is inside a (sequence, head).  128 tokens of
  // 16 heads in one launch 14.9 us, in three 21.1.
  const bool single = a.n_rows <= kChunk;
  if (!single) chunk_kernel<kDk, kDv, true><<<workers, kThreads, First::kSmem, s>>>(q_map, k_map, v_map, a, work);
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t chain = {}, main = {};
  chain.gridDim = dim3(workers, kDk * kDv / 1024);
  chain.blockDim = 256;
  main.gridDim = workers;
  main.blockDim = kThreads;
  main.dynamicSmemBytes = Main::kSmem;
  chain.stream = main.stream = s;
  chain.attrs = main.attrs = early;
  chain.numAttrs = 1;
  main.numAttrs = single ? 0 : 1;
  cudaError_t e = single ? cudaSuccess : cudaLaunchKernelEx(&chain, chain_kernel<kDk, kDv>, a, work);
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&main, chunk_kernel<kDk, kDv, false>, q_map, k_map, v_map, a, work);
  if (e != cudaSuccess)
    return set_error(ASTERQ_ERR_CUDA, "linear_attention: launch failed: %s", cudaGetErrorString(e));
  return check_launch("linear_attention");
}

}  // namespace

int64_t chunk_workspace_bytes(int dk, int dv, int workers) {
  return table_bytes(min(workers, kThreads)) + 4ll * min(workers, kThreads) * (dk * dv + dv) * 4;
}

int chunk_launch(const Args& a, int dk, int dv, int workers, int device, void* workspace, cudaStream_t s) {
  workers = min(workers, kThreads);  // the first pass looks each share's border up with a thread
  if (dk == 64 && dv == 64) return launch<64, 64>(a, workers, device, workspace, s);
  if (dk == 64) return launch<64, 128>(a, workers, device, workspace, s);
  if (dv == 64) return launch<128, 64>(a, workers, device, workspace, s);
  return launch<128, 128>(a, workers, device, workspace, s);
}

}  // namespace lin
}  // namespace asterq
