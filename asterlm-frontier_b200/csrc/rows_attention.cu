// Attention of many new tokens a sequence over a paged grouped-query cache (sm_100a): prompt chunks, causal
// among themselves, and trees of drafted tokens, which see their ancestors.
//
//   out[i, h] = sum_j softmax_j(score) v_j,  score = scale q[i, h] . k_j, softcapped where asked,
//   over the keys j <= p_i with (j < sink or j > p_i - (window - sink)),  p_i = length + i       (prompts)
//   over the cached keys under the same rule with p_i = length + depth_i, and the keys of i's ancestors and
//   its own, their positions under the same rule                                                 (trees)
//   lse[i, h] = log sum_j exp(score).
//
// What bounds it: 4 D operations a visible pair and head.  For prompts these outweigh the bytes by far, and of them
// the exponentials do: 16 a clock and SM are 1024 cycles for 128 x 128 scores, the two products of 128 dims 512.  Trees of a few
// nodes over long caches are bound by reading keys and values once.
//
// Rows.  The g = n_heads / n_kv_heads query heads of one kv head share its keys, so a tile of 128 rows is 128 / g
// tokens times g heads.  A unit of work is two such tiles of one (sequence, kv head), which share the tiles of keys
// and values that TMA brings; a warpgroup takes each, thread t row t, so that maxima and sums need no shuffles, and one's
// exponentials run under the other's products.  A unit of at most 128 rows has both warpgroups on the same rows and alternate
// tiles of keys; they join at its end, through tensor memory.
// S = Q K^T (128 x 128, fp32) lies in tensor memory, its weights as 16-bit values over it, O beside it.  Weights are rounded once for
// their product (csrc/paged_attention.cu takes them in two parts): a second part would double these products, which with the scores' set the
// pace of long prompts.  Against 64 bits the outputs are 2.1e-3 to 2.3e-3 of their norm off in bf16,
// where exact sums rounded to bf16 are 1.7e-3, and 2.7e-4 to 2.9e-4 in f16, where those are 2.1e-4.  The chain of a tile
// (softmax, then product and next scores, 1,024 cycles of the tensor cores, and two waits of some 300 until one side sees
// the other) is what sets the pace; the weights are handed over in halves to shorten it.  (Tried and slower: a third place for
// scores of 64 dims, tiles of 64 keys, sixteen softmax warps, a warp of products for each row tile, and a quarter of the
// exponentials by a polynomial: 5 to 8 % longer, although the softmax alone is 8 % faster so.)
// Measured, one sequence of 8,192 rows over 24,576 cached, 32 over 8 heads of 128 dims, bf16: 3.1 ms in the first calls, 3.55 to 3.65
// call after call at the clock that the power limit leaves: 1.05 to 1.24 PFLOP/s, 0.63 to 0.74 of the measured burst of matrix products.  9 prompts
// of 16,393 rows with a window of 1,024 (16 over 8 heads of 64 dims, f16): 161 us, whose 268 million exponentials in whole tiles are 74.  32
// trees of 16 nodes: 90 to 104 us over machines, 3.6 to 4.1 TB/s; 24 trees of 61 nodes 290 to 335.  One tree of 8 nodes 19 to 25 us, a prompt of
// 150 tokens 25 to 27: one pass through code that no SM has run before, some 5,000 cycles of it until the first copies, and the join.
//
// Split.  The key tiles of all units laid end to end (with kUnitCost in front of each) are cut into equal contiguous
// shares, one for each CTA, by sums over lengths and offsets that every CTA does for itself: no planning launch, no
// copy of lengths to the host.  A cut unit leaves (o, m, l) records in the workspace, and a second small grid joins
// them in the order of the shares.
#include "asterq_internal.h"
#include "common.cuh"
#include "launch.cuh"
#include "shares.h"
#include "tcgen05.cuh"

namespace asterq {
namespace rat {

constexpr int kMaxWorkers = 256;
// Warps 0 to 7: softmax, a warpgroup a row tile; then loads, products, and two that look values over.  (With eight warps beside
// the softmax the waiting ones alone slow the others: a wait reads shared memory, which the products keep busy.)
constexpr int kThreads = 384, kWarps = 12, kLoads = 8, kProducts = 9, kLook = 10;
constexpr int kRowsTile = 128;
constexpr int kMaxNodes = 128;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
// registers of a thread: 256 x 216 + 128 x 72 = 384 x 168 of the launch
constexpr int kRegsLaunch = 168, kRegsSoftmax = 216, kRegsHelp = 72;
static_assert(256 * kRegsSoftmax + 128 * kRegsHelp <= kThreads * kRegsLaunch, "more registers than launched with");
// What a unit costs beside its tiles, and the least that a CTA takes, in tiles.  (kUnitCost, kMinShare): a prompt of 150 tokens,
// 9 windowed prompts, one tree of 8, 32 of 16, 24 of 61 in us.  (1, 2): 26.8, 171, 18.8, 93, 294; (3, 2): 26.8, 174, 19.1, 95, 287;
// (1, 6): 32.9, 171, 24.9, 93, 294; (1, 3): 24.9, 171, 23.6, 93, 293.
constexpr int kUnitCost = 1;
constexpr int kMinShare = 2;

struct Desc {  // of a cut unit, by the CTA that has its first tile
  int pieces, row0, tokens, head;
};

struct Args {
  const void* q;
  const int* page_table;
  const int* lengths;
  const int* row_offsets;
  const int* parents;
  const void* v_pool;
  void* out;
  float* lse;
  float* records;  // o [2 W][D / 4][rows][4], then m [2 W][rows], then l [2 W][rows]
  Desc* desc;      // [W]
  int* status;
  long long n_rows, n_pages, capacity;  // capacity: tokens a row of the table can hold
  int n_seqs, n_heads, n_kv_heads, group, tile_tokens, unit_tokens;
  int page_tokens, max_pages, box_rows;
  int window, sink, reach;  // reach: newest tokens that a window shows, window - sink
  int out_f32;
  float scale, scale2, softcap, cap_in;
};

// kPre: scores are changed before their maximum is taken (a softcap, or a scale that is not positive)
// kOne: no unit has more than one row tile, and the second one's queries leave their room to keys and values
template <bool kF16_, int D_, bool kPre_, bool kOne_>
struct Cfg {
  static constexpr bool kF16 = kF16_, kPre = kPre_, kOne = kOne_;
  static constexpr int D = D_;
  static constexpr int kTiles = D == 256 ? 1 : 2;  // row tiles of a unit: two accumulators of 256 dims leave no room for scores
  static constexpr int kRows = kTiles * kRowsTile, kKeys = D == 256 ? 64 : 128;
  static constexpr int kQBytes = kRowsTile * D * 2, kSlotBytes = kKeys * D * 2;  // a slot holds a tile of keys or of values
  static constexpr int kQTiles = kOne ? 1 : kTiles, kSlots = D == 64 ? (kOne ? 13 : 12) : D == 128 && kOne ? 6 : 5;
  // columns of tensor memory: two places for scores and the weights over them (one for each row tile, or for every other
  // tile of keys), then the accumulators
  static constexpr int kColO = 2 * kKeys, kStepO = D;
  static_assert(kColO + kTiles * D <= 512, "tensor memory");
  // barriers: full, empty and looked over of each slot, the others by name; of scores one for each place, of weights for
  // each place and half, so that whoever waits sees all phases of one
  static constexpr int kEmpty = kSlots, kClean = 2 * kSlots, kQFull = 3 * kSlots, kQEmpty = kQFull + 1, kWFull = kQEmpty + 1,
                       kWEmpty = kWFull + 2, kSFull = kWEmpty + 2, kPReady = kSFull + 2, kDone = kPReady + 4,
                       kDrain = kDone + 2, kMeet = kDrain + 1, kBars = kMeet + 1;
  // behind the slots: barriers, two work entries, what threads exchange
  static constexpr int kAtWork = (kBars * 8 + 15) / 16 * 16, kAtFlags = kAtWork + 160, kAtUp = kAtFlags + 16,
                       kAtSwap = kAtUp + 2 * kMaxNodes, kSmall = kAtSwap + 2 * kRowsTile * 4;
  static constexpr int kSmem = kQTiles * kQBytes + kSlots * kSlotBytes + kSmall;
  static_assert(kSmem <= 232448, "more shared memory than a CTA has");
};

ASTERQ_DEVICE void tma_kv(uint32_t dst, const CUtensorMap* map, int token, int half, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(map), "r"(0), "r"(token), "r"(half), "r"(z), "r"(bar)
      : "memory");
}
ASTERQ_DEVICE void tma_q(uint32_t dst, const CUtensorMap* map, int dim, int head, int row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(dim), "r"(head), "r"(row), "r"(bar)
      : "memory");
}
// whether the predicate holds for all of `count` threads
ASTERQ_DEVICE bool named_all(int id, int count, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n barrier.cta.red.and.pred q, %1, %2, p;\n selp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"(id), "r"(count), "r"((uint32_t)pred)
      : "memory");
  return r != 0;
}

// a value that all lanes have, known as such to the compiler: what comes of it stays in uniform registers, where the
// tensor cores' instructions have their operands (otherwise each takes some 110 cycles to issue instead of 64)
ASTERQ_DEVICE int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

constexpr uint32_t idesc(bool f16, int n, bool b_mn_major) {
  return (1u << 4) | ((f16 ? 0u : 1u) << 7) | ((f16 ? 0u : 1u) << 10) | ((b_mn_major ? 1u : 0u) << 16) |
         ((uint32_t)(n / 8) << 17) | ((128u / 16) << 24);
}

// A sequence's new rows that are answered: none of an empty slot, and none that the page table has no place for.
struct Seq {
  int row0, n, length;
};
ASTERQ_DEVICE Seq seq_of(const Args& a, int s, bool& bad, int& dead) {
  const int begin = __ldg(a.row_offsets + s), end = __ldg(a.row_offsets + s + 1), length = __ldg(a.lengths + s);
  Seq q;
  bad = begin < 0 || end < begin || end > a.n_rows || (a.parents && end - begin > kMaxNodes);
  q.row0 = begin;
  q.length = length;
  const int rows = bad ? 0 : end - begin;
  q.n = length < 0 ? 0 : (int)max(0ll, min((long long)rows, a.capacity - length));
  dead = rows - q.n;
  return q;
}

// The key tiles of a unit: tile k of its list is keys [kKeys j, kKeys (j + 1)) with j = k below sink_tiles and
// first + k - sink_tiles from there on.  A node's key is at its number's place while it is seen by its position: where a window is
// all sink, nodes at positions in the sink may have theirs behind its last tile.
struct Span {
  int tok0, tokens, from, end, sink_tiles, first, tiles;
};
template <int kKeys>
ASTERQ_DEVICE Span span_of(const Args& a, const Seq& q, int block) {
  Span s;
  s.tok0 = block * a.unit_tokens;
  s.tokens = min(q.n - s.tok0, a.unit_tokens);
  s.end = q.length + s.tok0 + s.tokens;
  const int last = (s.end + kKeys - 1) / kKeys;
  s.from = 0;
  s.sink_tiles = 0;
  s.first = 0;
  if (a.window > 0) {
    const int from = q.length + (a.parents ? min(1 - a.reach, 0) : s.tok0 - a.reach + 1);
    if (from > 0) {
      s.from = from;
      s.sink_tiles = min((a.sink + kKeys - 1) / kKeys, last);
      s.first = a.reach == 0 && (!a.parents || q.length >= a.sink) ? last : max(from / kKeys, s.sink_tiles);
    }
  }
  s.tiles = s.sink_tiles + last - s.first;
  return s;
}

// What the load warp tells the others about a piece of a unit.
struct Work {
  int n;            // tiles here; 0: the end
  int k0, sink_tiles, first;
  int row0, tokens, head;      // row of its first token, tokens, kv head
  int length, tok0, from;      // cached tokens, index of its first token in the sequence, first key of its window
  int seq_row0, nodes;         // row of the sequence's first token, rows of the sequence up to the unit's end
  int seq;                     // the sequence, its row of the page table
  int pair, cut, slot, poison;  // poison: a value that is not finite was taken out of a tile that not all rows see
  int pad[3];
  ASTERQ_DEVICE int tile(int k) const { return k < sink_tiles ? k : first + (k - sink_tiles); }
};

// bits i of keys c + i in [lo, hi)
ASTERQ_DEVICE uint32_t bits_between(int c, int lo, int hi) {
  const int l = min(max(lo - c, 0), 32), h = min(max(hi - c, 0), 32);
  const uint32_t below_h = h >= 32 ? 0xffffffffu : (1u << h) - 1u, below_l = l >= 32 ? 0xffffffffu : (1u << l) - 1u;
  return below_h & ~below_l;
}

// What one row sees.
struct View {
  int lo, hi, sink;             // keys [lo, hi) and [0, sink), sink <= hi
  int length;                   // of the nodes' first key
  uint32_t node[kMaxNodes / 32];  // nodes, of trees
  template <bool kTree>
  ASTERQ_DEVICE uint32_t bits(int c) const {
    uint32_t w = bits_between(c, lo, hi) | bits_between(c, 0, sink);
    if (kTree) {
      const int at = c - length;
      if (at > -32 && at < kMaxNodes) {
        const int i = at >> 5, sh = at & 31;  // at may be negative: i = -1
        auto word = [&](int k) { return k == 0 ? node[0] : k == 1 ? node[1] : k == 2 ? node[2] : k == 3 ? node[3] : 0u; };
        w |= __funnelshift_r(word(i), word(i + 1), sh);
      }
    }
    return w;
  }
};

struct Start {
  int s, head, block, at;
};

// tanh x to a few 2^-23 of itself: below 0.9 Lambert's continued fraction x / (1 + x^2 / (3 + x^2 / (5 + x^2 / (7 + x^2 / 9))))
// as a quotient, its error x^10 / 9.8e6 < 2^-24; from there on (e^2x - 1) / (e^2x + 1).
ASTERQ_DEVICE float tanh_of(float x) {
  const float x2 = x * x;
  const float e2x = ex2_ftz(fminf(fmaxf(x * (2.0f * kLog2e), -64.0f), 64.0f));
  const bool large = fabsf(x) >= 0.9f;  // not of a NaN
  const float num = large ? e2x - 1.0f : x * fmaf(x2, x2 + 105.0f, 945.0f);
  const float den = large ? e2x + 1.0f : fmaf(x2, fmaf(x2, 15.0f, 420.0f), 945.0f);
  return __fdividef(num, den);
}

template <bool kF16>
ASTERQ_DEVICE uint32_t pack2(float lo, float hi) {
  return kF16 ? pack_half2(lo, hi) : pack_bf162(lo, hi);
}
// the halves of w that are infinities or NaN, as a mask
template <bool kF16>
ASTERQ_DEVICE uint32_t not_finite2(uint32_t w) {
  constexpr uint32_t e = kF16 ? 0x7c00u : 0x7f80u;
  return ((w & e) == e ? 0xffffu : 0u) | ((w & (e << 16)) == (e << 16) ? 0xffff0000u : 0u);
}

template <bool kF16>
ASTERQ_DEVICE bool all_finite(uint4 x) {
  uint32_t s;
  if constexpr (kF16) s = hfma2_u32(x.w, 0u, hfma2_u32(x.z, 0u, hfma2_u32(x.y, 0u, hmul2_u32(x.x, 0u))));
  else s = tc::fma_bf162(x.w, 0u, tc::fma_bf162(x.z, 0u, tc::fma_bf162(x.y, 0u, tc::mul_bf162(x.x, 0u))));
  return (s & 0x7fff7fffu) == 0;  // zeros of either sign
}
ASTERQ_DEVICE float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// the end of loads from tensor memory whose values are in r: nothing reads r before it
ASTERQ_DEVICE void wait_ld32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// A wait of a whole warp in few instructions, since the roles' loops together have to fit the instruction cache.  A round
// suspends for up to 20 us, so the limit is some seconds.
ASTERQ_DEVICE void wait_quietly(uint32_t bar, uint32_t parity, volatile int* abort_flag, int rounds = 1 << 18) {
  if (mbar_try(bar, parity)) return;
#pragma unroll 1
  while (mbar_try_sleep(bar, parity, 20000u) == 0) {
    if (--rounds < 0) *abort_flag = 1;
    if (ld_shared_volatile(abort_flag)) break;
  }
}
// false where a wait has run out
ASTERQ_DEVICE bool wait_for(uint32_t bar, uint32_t parity, volatile int* abort_flag, int rounds = 1 << 18) {
  uint32_t done = mbar_try(bar, parity);
#pragma unroll 1
  while (done == 0 && (done = mbar_try_sleep(bar, parity, 20000u)) == 0) {
    if (--rounds < 0) *abort_flag = 1;
    if (ld_shared_volatile(abort_flag)) break;
  }
  return __all_sync(0xffffffffu, (int)done) != 0;
}

template <class C>
__global__ void __launch_bounds__(kThreads, 1)
    rows_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                const __grid_constant__ CUtensorMap v_map, const __grid_constant__ Args a) {
  constexpr int D = C::D, kKeys = C::kKeys;
  constexpr bool kF16 = C::kF16;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t q_base = smem_u32(smem), ring = q_base + C::kQTiles * C::kQBytes;
  uint8_t* small = smem + C::kQTiles * C::kQBytes + C::kSlots * C::kSlotBytes;
  const uint32_t bars = smem_u32(small);
  auto bar = [&](int i) { return bars + 8 * i; };
  Work* work = reinterpret_cast<Work*>(small + C::kAtWork);  // [2]
  uint32_t* tmem_s = reinterpret_cast<uint32_t*>(small + C::kAtFlags);
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_s + 1);
  volatile int* never_s = reinterpret_cast<volatile int*>(tmem_s + 2);
  int8_t* up_s = reinterpret_cast<int8_t*>(small + C::kAtUp);     // [2][kMaxNodes]: parents, for each row tile
  float* swap_s = reinterpret_cast<float*>(small + C::kAtSwap);   // [2][kRowsTile]: m and l of a joined unit's second warpgroup
  long long* scan_s = reinterpret_cast<long long*>(swap_s);       // [kWarps], and the share's start, before all that
  Start* start_s = reinterpret_cast<Start*>(swap_s + kRowsTile);
  static_assert(sizeof(Work) == 80 && sizeof(Start) <= kRowsTile * 4 && kWarps * 8 <= kRowsTile * 4, "small");
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31, me = blockIdx.x;

  asm volatile("griddepcontrol.launch_dependents;");
  if (tid < C::kBars) {
    const int i = tid;
    int count = 1;
    if (i >= C::kEmpty && i < C::kClean) count = 3;  // the products', and two warps that look values over
    else if (i >= C::kClean && i < C::kQFull) count = 2;
    else if (i >= C::kWEmpty && i < C::kSFull) count = 11;
    else if (i >= C::kPReady && i < C::kDone) count = 4;  // a warp each
    else if (i == C::kMeet) count = 8;
    mbar_init(bar(i), count);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 0) {
    // boxes lie in patterns of 1024 bytes
    *abort_s = (q_base & 1023) != 0;
    *never_s = 0;
  }
  if (warp == kProducts) tc::alloc512(smem_u32(tmem_s));
  if (warp == kLoads && lane < 3) {
    const CUtensorMap* map = lane == 0 ? &q_map : lane == 1 ? &k_map : &v_map;
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  }

  // ---------------------------------------------------------------------------------- the share
  // Warp w sums the costs of sequences [w strip, (w + 1) strip), 32 at a time; the sums of a sequence of many
  // units by all lanes.
  const int strip = (a.n_seqs + kWarps - 1) / kWarps;
  const int s_begin = min(warp * strip, a.n_seqs), s_end = min(s_begin + strip, a.n_seqs);
  bool any_bad = false;
  auto costs_of = [&](int base, Seq& q) {
    bool bad = false;
    int dead = 0;
    q.n = 0;
    if (base + lane < s_end) q = seq_of(a, base + lane, bad, dead);
    any_bad = any_bad || bad;
    const int blocks = (q.n + a.unit_tokens - 1) / a.unit_tokens;
    long long cost = 0;
    if (blocks == 1) cost = span_of<kKeys>(a, q, 0).tiles + kUnitCost;
    uint32_t many = __ballot_sync(0xffffffffu, blocks > 1);
#pragma unroll 1
    while (many) {
      const int from = __ffs(many) - 1;
      many &= many - 1;
      Seq o;
      o.n = __shfl_sync(0xffffffffu, q.n, from);
      o.length = __shfl_sync(0xffffffffu, q.length, from);
      const int n = __shfl_sync(0xffffffffu, blocks, from);
      long long all = 0;
#pragma unroll 1
      for (int b = lane; b < n; b += 32) all += span_of<kKeys>(a, o, b).tiles + kUnitCost;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) all += __shfl_xor_sync(0xffffffffu, all, d);
      if (lane == from) cost = all;
    }
    return cost * a.n_kv_heads;
  };
  long long sum = 0, cost = 0;
  Seq q;
  q.n = 0;
#pragma unroll 1
  for (int base = s_begin; base < s_end; base += 32) {
    cost = costs_of(base, q);
    sum += cost;
  }
#pragma unroll
  for (int d = 1; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) scan_s[warp] = sum;
  // offsets out of order or out of range: which rows are whose is not known, and the call is left undone
  tc::fence_before();
  if (__syncthreads_or(any_bad)) {
    tc::fence_after();
    if (warp == kProducts) tc::dealloc512(*tmem_s);
    if (tid == 0) {
      a.desc[me].pieces = 0;
      if (a.status) atomicMax(a.status, 1);
    }
    return;
  }
  long long before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const long long x = scan_s[w];
    before += w < warp ? x : 0;
    total += x;
  }
  // CTAs that take part: each has kMinShare tiles or more
  const int W = (int)max(1ll, min((long long)gridDim.x, total / kMinShare));
  const long long x0 = share_of(total, min(me, W), W), x1 = share_of(total, min(me + 1, W), W);
  if (x0 < x1 && before <= x0 && x0 < before + sum) {
    long long at = before;
#pragma unroll 1
    for (int base = s_begin; base < s_end; base += 32) {
      if (strip > 32) cost = costs_of(base, q);
      long long scan = cost;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const long long up = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += up;
      }
      const uint32_t beyond = __ballot_sync(0xffffffffu, x0 < at + scan);
      if (beyond == 0) {
        at += __shfl_sync(0xffffffffu, scan, 31);
        continue;
      }
      const int here = __ffs(beyond) - 1;
      at += __shfl_sync(0xffffffffu, scan - cost, here);
      const long long head_cost = share_of(__shfl_sync(0xffffffffu, cost, here), 1, a.n_kv_heads);
      Seq o;
      o.n = __shfl_sync(0xffffffffu, q.n, here);
      o.length = __shfl_sync(0xffffffffu, q.length, here);
      const int head = (int)share_of(x0 - at, 1, head_cost);
      long long rest = x0 - at - head * head_cost;
      const int blocks = (o.n + a.unit_tokens - 1) / a.unit_tokens;
#pragma unroll 1
      for (int b0 = 0; b0 < blocks; b0 += 32) {
        const int c = b0 + lane < blocks ? span_of<kKeys>(a, o, b0 + lane).tiles + kUnitCost : 0;
        long long up_to = c;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
          const long long up = __shfl_up_sync(0xffffffffu, up_to, d);
          if (lane >= d) up_to += up;
        }
        const uint32_t in = __ballot_sync(0xffffffffu, rest < up_to);
        if (in == 0) {
          rest -= __shfl_sync(0xffffffffu, up_to, 31);
          continue;
        }
        if (lane == __ffs(in) - 1) *start_s = {base + here, head, b0 + lane, (int)(rest - (up_to - c))};
        break;
      }
      break;
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = uniform(*tmem_s);
  if (warp >= kLook) {
    // rows that are not answered: zeros, and a log-sum of -inf
#pragma unroll 1
    for (int base = (me * 2 + warp - kLook) * 32; base < a.n_seqs; base += gridDim.x * 64) {
      bool bad = false;
      int dead = 0;
      Seq o;
      o.n = 0;
      if (base + lane < a.n_seqs) o = seq_of(a, base + lane, bad, dead);
      if (dead > 0 && o.length >= 0 && a.status) atomicMax(a.status, 1);
      uint32_t some = __ballot_sync(0xffffffffu, dead > 0);
#pragma unroll 1
      while (some) {
        const int from = __ffs(some) - 1;
        some &= some - 1;
        const long long row = __shfl_sync(0xffffffffu, o.row0 + o.n, from);
        const long long n = (long long)__shfl_sync(0xffffffffu, dead, from) * a.n_heads;
        uint4* dst = reinterpret_cast<uint4*>(static_cast<char*>(a.out) + row * a.n_heads * D * (a.out_f32 ? 4 : 2));
#pragma unroll 1
        for (long long i = lane; i < n * (a.out_f32 ? D / 4 : D / 8); i += 32) dst[i] = make_uint4(0, 0, 0, 0);
#pragma unroll 1
        for (long long i = lane; a.lse && i < n; i += 32) a.lse[row * a.n_heads + i] = -INFINITY;
      }
    }
  }
  if (x0 >= x1 || *abort_s) {
    if (tid == 0) {
      a.desc[me].pieces = 0;
      if (*abort_s && a.status) atomicMax(a.status, 2);
    }
    if (warp == kProducts) tc::dealloc512(tmem);
    return;
  }

  // the keys that all rows of a unit see: below hi, and from lo on or in the sink
  struct Seen {
    int hi, lo;
    ASTERQ_DEVICE bool all(int key, int sink) const { return key < hi && (key >= lo || key < sink); }
    ASTERQ_DEVICE bool all_of_tile(int c, int sink) const { return c + kKeys <= hi && (c >= lo || c + kKeys <= sink); }
  };
  auto seen_of = [&](const Work& u) {
    Seen s;
    s.hi = a.parents ? u.length : u.length + u.tok0 + 1;
    const long long newest = (long long)u.length + (a.parents ? u.nodes : u.tok0 + u.tokens) - 1;
    s.lo = a.window == 0 ? 0 : (int)max(0ll, newest - a.reach + 1);
    return s;
  };
  if (warp >= kLoads) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsHelp));
    bool ok = true;
    // each role follows the ring by itself
    int slot = 0, phase = 0;
    auto step = [&]() {
      if (++slot == C::kSlots) {
        slot = 0;
        phase ^= 1;
      }
    };
    if (warp == kLoads) {
      // ------------------------------------------------------------------------------ loads
      Desc desc;
      desc.pieces = 0;
      int s = start_s->s, head = start_s->head, block = start_s->block, at = start_s->at;
      long long x = x0;
      bool bad;
      int dead;
      Seq q = seq_of(a, s, bad, dead);
      Span span = span_of<kKeys>(a, q, block);
      int pieces = 0;
      bool round = false;  // the slots have been used before
      // one lane a box: box_rows keys (a divisor of the page and of the tile) of 64 dims
      constexpr int halves = D / 64;
      const int my_key = lane / halves * a.box_rows, my_half = lane % halves;
      const bool works = my_key < kKeys;
      const uint32_t box_bytes = a.box_rows * 128;
      const uint32_t box_at = ring + my_half * (kKeys * 128) + my_key * 128;
      const int columns = kKeys / a.page_tokens, rest = kKeys - columns * a.page_tokens;  // from a tile to the next
#pragma unroll 1
      while (ok && x < x1) {
        const int cost = (int)min((long long)(span.tiles + kUnitCost - at), x1 - x);
        const int k0 = max(at - kUnitCost, 0), n = max(at + cost - kUnitCost, 0) - k0;
        if (n > 0) {
          // A tile's pages are looked up two tiles before it is wanted.
          struct Box {
            int page, offset;
            bool want;
          };
          int k_at = k0, key = 0, column = 0, offset = 0;
          const int* table = a.page_table + (long long)s * a.max_pages;
          auto look_up = [&]() {
            Box box = {0, 0, false};
            if (k_at < k0 + n) {
              if (k_at == k0 || k_at == span.sink_tiles) {
                key = (k_at < span.sink_tiles ? k_at : span.first + (k_at - span.sink_tiles)) * kKeys + my_key;
                column = key / a.page_tokens;
                offset = key - column * a.page_tokens;
              }
              box.offset = offset;
              box.want = works && key < span.end && (key < a.sink || key + a.box_rows > span.from);
              if (box.want) box.page = __ldg(table + column);
              key += kKeys;
              column += columns;
              offset += rest;
              if (offset >= a.page_tokens) {
                offset -= a.page_tokens;
                ++column;
              }
              ++k_at;
            }
            return box;
          };
          Box now = look_up(), ahead = look_up();
          // queries
          if (pieces > 0 && !(ok = wait_for(bar(C::kQEmpty), (pieces - 1) & 1, abort_s))) break;
          const int q_tiles = span.tokens > a.tile_tokens ? 2 : 1;
          if (lane == 0) mbar_expect_tx(bar(C::kQFull), q_tiles * halves * a.tile_tokens * a.group * 128);
          __syncwarp();
          if (lane < q_tiles * halves) {
            const int t = lane / halves, h = lane % halves;
            tma_q(q_base + t * C::kQBytes + h * (kRowsTile * 128), &q_map, h * 64, head * a.group,
                  q.row0 + span.tok0 + t * a.tile_tokens, bar(C::kQFull));
          }
          const int e = pieces & 1;
          if (pieces >= 2 && !(ok = wait_for(bar(C::kWEmpty + e), ((pieces >> 1) - 1) & 1, abort_s))) break;
          if (lane == 0) {
            const bool cut = n < span.tiles;
            Work u;
            u.n = n;
            u.k0 = k0;
            u.sink_tiles = span.sink_tiles;
            u.first = span.first;
            u.row0 = q.row0 + span.tok0;
            u.tokens = span.tokens;
            u.head = head;
            u.length = q.length;
            u.tok0 = span.tok0;
            u.from = span.from;
            u.seq_row0 = q.row0;
            u.nodes = span.tok0 + span.tokens;
            u.seq = s;
            u.pair = C::kTiles == 2 && span.tokens <= a.tile_tokens;
            u.cut = cut;
            u.slot = 2 * me + (k0 == 0);
            u.poison = 0;
            work[e] = u;
            mbar_arrive(bar(C::kWFull + e));
            if (cut && k0 == 0) {
              // the pieces after this one are in the next CTAs' first slots
              desc.pieces = shares_up_to(x - at + kUnitCost + span.tiles, W, total, me);
              desc.row0 = u.row0;
              desc.tokens = u.tokens;
              desc.head = head;
            }
          }
          __syncwarp();
          ++pieces;
          // keys and values
#pragma unroll 1
          for (int i = 0; i < n; ++i) {
            const Box later = look_up();
            const uint32_t wanted = __ballot_sync(0xffffffffu, now.want);
            int page = now.page;
            if (now.want && (page < 0 || page >= a.n_pages)) {
              if (a.status) atomicMax(a.status, 1);
              page = 0;
            }
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              if (round && !(ok = wait_for(bar(C::kEmpty + slot), phase ^ 1, abort_s))) break;
              if (lane == 0) mbar_expect_tx(bar(slot), __popc(wanted) * box_bytes);
              __syncwarp();
              if (now.want)
                tma_kv(box_at + slot * C::kSlotBytes, v ? &v_map : &k_map, now.offset, my_half, page * a.n_kv_heads + head, bar(slot));
              step();
              if (slot == 0) round = true;
            }
            if (!ok) break;
            now = ahead;
            ahead = later;
          }
          if (!ok) break;
        }
        x += cost;
        at += cost;
        if (at == span.tiles + kUnitCost && x < x1) {
          at = 0;
          ++block;
          if (block * a.unit_tokens >= q.n) {
            block = 0;
            if (++head == a.n_kv_heads) {
              head = 0;
#pragma unroll 1
              do q = seq_of(a, ++s, bad, dead);
              while (q.n == 0);
            }
          }
          span = span_of<kKeys>(a, q, block);
        }
      }
      if (ok) {
        const int e = pieces & 1;
        if (pieces >= 2) ok = wait_for(bar(C::kWEmpty + e), ((pieces >> 1) - 1) & 1, abort_s);
        if (ok && lane == 0) {
          work[e].n = 0;
          mbar_arrive(bar(C::kWFull + e));
        }
      }
      if (!ok) {
        // the last copies have landed before the exit, also when nobody waits for them any more: each barrier
        // ends the phase that it is in within the limit, or has ended the ones begun
#pragma unroll 1
        for (int i = 0; i < 2 * (C::kSlots + 1); ++i)
          (void)wait_for(bar(i / 2 == C::kSlots ? C::kQFull : i / 2), i & 1, never_s, 1000);
      }
      if (lane == 0) a.desc[me] = desc;
    } else if (warp == kProducts) {
      // ------------------------------------------------------------------------------ products
      // Job i of a unit: a row tile's scores with a tile of keys, and its weights' product.  The scores of job i + 2, which take
      // the place of job i's weights, are asked for right behind that product.
      constexpr uint32_t kQk = idesc(kF16, kKeys, false), kPv = idesc(kF16, D, true);
      uint32_t weights = 0;            // phases of kPReady, a bit a place
      int v_slot = 0, v_phase = 0;     // of the next values; slot and phase: of the next keys
      auto next_tile = [&](int& s, int& ph) {  // keys and values take the slots in turn
        s += 2;
        if (s >= C::kSlots) {
          s -= C::kSlots;
          ph ^= 1;
        }
      };
      v_slot = 1;
#pragma unroll 1
      for (int piece = 0;; ++piece) {
        const int e = piece & 1;
        if (!(ok = wait_for(bar(C::kWFull + e), (piece >> 1) & 1, abort_s))) break;
        const int n = uniform(work[e].n), pair = uniform(work[e].pair);
        const int k0 = uniform(work[e].k0), sink_tiles = uniform(work[e].sink_tiles), first = uniform(work[e].first);
        Seen seen_all = seen_of(work[e]);
        seen_all.hi = uniform(seen_all.hi);
        seen_all.lo = uniform(seen_all.lo);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kWEmpty + e));
        if (n == 0) break;
        if (!(ok = wait_for(bar(C::kQFull), piece & 1, abort_s))) break;
        const bool both = C::kQTiles == 2 && !pair;  // two row tiles to each tile of keys
        const int jobs = both ? 2 * n : n;
        int j = 0;  // tile of keys of job i
#pragma unroll 1
        for (int i = -2; i < jobs; ++i) {
          const int b = i & 1;
          const bool last = !both || b == 1;  // the last job of its tile of keys
          const uint32_t s_at = uniform(tmem + b * kKeys);
          if (i >= 0) {
            if (!both || b == 0) {
              const int k = k0 + j, c = (k < sink_tiles ? k : first + (k - sink_tiles)) * kKeys;
              if (!(ok = wait_for(bar((seen_all.all_of_tile(c, a.sink) ? 0 : C::kClean) + v_slot), v_phase, abort_s))) break;
            }
            const uint32_t v0 = uniform(tc::desc_mn_major(ring + v_slot * C::kSlotBytes, kKeys * 128));
            const uint32_t d = tmem + C::kColO + (C::kTiles == 2 ? b : 0) * C::kStepO;
            const bool add = i >= C::kTiles;
            if (!(ok = wait_for(bar(C::kPReady + 2 * b), weights >> b & 1, abort_s))) break;
            tc::fence_after();
            if (tc::elect()) {
#pragma unroll
              for (int s = 0; s < kKeys / 32; ++s) tc::mma_ts(d, s_at + 8 * s, v0 + s * 128, kPv, add || s > 0);
            }
            __syncwarp();
            if (i + 2 < jobs && (!both || b == 0) && !(ok = wait_for(bar(slot), phase, abort_s))) break;
            if (!(ok = wait_for(bar(C::kPReady + 2 * b + 1), weights >> b & 1, abort_s))) break;
            weights ^= 1u << b;
            tc::fence_after();
            if (tc::elect()) {
#pragma unroll
              for (int s = kKeys / 32; s < kKeys / 16; ++s) tc::mma_ts(d, s_at + 8 * s, v0 + s * 128, kPv, true);
              if (last) tc::commit(bar(C::kEmpty + v_slot));
              if (i + C::kTiles >= jobs) tc::commit(bar(C::kDone + (C::kTiles == 2 ? b : 0)));
              if (C::kTiles == 1) tc::commit(bar(C::kDone + 1));  // of each job
            }
            __syncwarp();
            if (last) {
              next_tile(v_slot, v_phase);
              ++j;
            }
          } else if (i + 2 < jobs && (!both || b == 0) && !(ok = wait_for(bar(slot), phase, abort_s))) {
            break;
          }
          if (i + 2 < jobs) {
            const uint32_t q0 = uniform(tc::desc_k_major(q_base + (both ? b : 0) * C::kQBytes));
            const uint32_t kd = uniform(tc::desc_k_major(ring + slot * C::kSlotBytes));
            if (tc::elect()) {
#pragma unroll
              for (int s = 0; s < D / 16; ++s)
                tc::mma_ss(s_at, q0 + s / 4 * (kRowsTile * 8) + s % 4 * 2, kd + s / 4 * (kKeys * 8) + s % 4 * 2, kQk, s > 0);
              tc::commit(bar(C::kSFull + b));
              if (last) tc::commit(bar(C::kEmpty + slot));
              if (i + 3 == jobs) tc::commit(bar(C::kQEmpty));
            }
            __syncwarp();
            if (last) next_tile(slot, phase);
          }
        }
        if (!ok) break;
      }
      if (!ok) {  // products under way end before tensor memory goes
        if (tc::elect()) tc::commit(bar(C::kDrain));
        __syncwarp();
        (void)wait_for(bar(C::kDrain), 0, never_s, 10000);
      }
    } else {
      // ------------------------------------------------------------------------------ values looked over
      // In a tile that not every row sees all of, a weight of zero meets values that the row does not see, and zero
      // times an infinity or NaN is not zero.  Values that no row sees become zeros; of the others those that are not
      // finite do, and the rows' threads add them where they are seen (poison).
      const int part = warp - kLook;
#pragma unroll 1
      for (int piece = 0;; ++piece) {
        const int e = piece & 1;
        if (!(ok = wait_for(bar(C::kWFull + e), (piece >> 1) & 1, abort_s))) break;
        const int n = work[e].n, k0 = work[e].k0, sink_tiles = work[e].sink_tiles, first = work[e].first;
        const int end = work[e].length + work[e].nodes, from = work[e].from;
        const Seen seen_all = seen_of(work[e]);
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
          if (!(ok = wait_for(bar(slot), phase, abort_s))) break;
          if (lane == 0) {  // keys
            mbar_arrive(bar(C::kClean + slot));
            mbar_arrive(bar(C::kEmpty + slot));
          }
          step();
          if (!(ok = wait_for(bar(slot), phase, abort_s))) break;
          const int k = k0 + i, c = (k < sink_tiles ? k : first + (k - sink_tiles)) * kKeys;
          if (!seen_all.all_of_tile(c, a.sink)) {
            uint4* v = reinterpret_cast<uint4*>(smem + C::kQTiles * C::kQBytes + slot * C::kSlotBytes);
            constexpr int kAll = C::kSlotBytes / 16 / 64;  // vectors a lane
            uint4* mine = v + part * 32 + lane;
            if (c + kKeys > end || (c < from && c + kKeys > a.sink)) {
#pragma unroll 1
              for (int x = 0; x < kAll; ++x) {
                const int key = c + (x * 8 + part * 4 + lane / 8) % kKeys;
                if (key >= end || (key < from && key >= a.sink)) mine[64 * x] = make_uint4(0, 0, 0, 0);
              }
            }
            // A sum of zero times each value is zero, or a NaN where one of them is not finite.
            bool found = false;
            constexpr int kBatch = 8;
#pragma unroll 1
            for (int x0 = 0; x0 < kAll; x0 += kBatch) {
              uint4 w[kBatch];
#pragma unroll
              for (int x = 0; x < kBatch; ++x) w[x] = mine[64 * (x0 + x)];
              bool fine = true;
#pragma unroll
              for (int x = 0; x < kBatch; ++x) fine = all_finite<kF16>(w[x]) && fine;
              if (__all_sync(0xffffffffu, fine)) continue;
#pragma unroll 1
              for (int x = x0; x < x0 + kBatch; ++x) {
                uint4 o = mine[64 * x];
                if (all_finite<kF16>(o)) continue;
                o.x &= ~not_finite2<kF16>(o.x);
                o.y &= ~not_finite2<kF16>(o.y);
                o.z &= ~not_finite2<kF16>(o.z);
                o.w &= ~not_finite2<kF16>(o.w);
                mine[64 * x] = o;
                found = true;
              }
            }
            if (found) *reinterpret_cast<volatile int*>(&work[e].poison) = 1;
            fence_async_shared();
          }
          __syncwarp();
          if (lane == 0) {  // for every use, so that no phase is left out
            mbar_arrive(bar(C::kClean + slot));
            mbar_arrive(bar(C::kEmpty + slot));
          }
          step();
        }
        if (!ok) break;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kWEmpty + e));
        if (n == 0) break;
      }
    }
  } else {
    // -------------------------------------------------------------------------------- softmax, one row a thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int tile = warp >> 2, r = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    const uint32_t col_o = lanes + C::kColO + tile * C::kStepO;
    const int token_in = r / a.group, head_in = r - token_in * a.group;
    const bool in_tile = token_in < a.tile_tokens;
    const float scale2 = C::kPre ? 1.0f : a.scale2;
    uint32_t full = 0, done = 0, met = 0, rests = 0;  // phases: of kSFull (a bit a place), kDone and kMeet; jobs so far
    // Both warpgroups of a unit that they share.  With others each goes its own way, and one's outputs are written under the
    // other's products.
    auto meet = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::kMeet));
      wait_quietly(bar(C::kMeet), met, abort_s);
      met ^= 1;
      __syncwarp();
    };
    View view;
    int view_row = -1, view_tok0 = 0;
    bool view_pair = false;
#pragma unroll 1
    for (int piece = 0;; ++piece) {
      const int e = piece & 1;
      const bool got = wait_for(bar(C::kWFull + e), (piece >> 1) & 1, abort_s);
      // a warpgroup goes on or does not: its warps meet at barriers (after a wait has run out, waits return at once)
      if (!named_all(2 + tile, 128, got)) break;
      const Work* u = work + e;
      const int n = u->n, k0 = u->k0;
      if (n == 0) break;
      if (C::kTiles == 1 && tile == 1) {  // one row tile: these have nothing to do
        if (lane == 0) mbar_arrive(bar(C::kWEmpty + e));
        continue;
      }
      const bool pair = u->pair;
      const int token = token_in + (pair ? 0 : tile * a.tile_tokens);  // of the unit
      const bool valid = in_tile && token < u->tokens;
      // heads of one tree's rows in turn: what they see is the same
      if (!(a.parents && view_row == u->seq_row0 && view_tok0 == u->tok0 && view_pair == pair)) {
        view_row = u->seq_row0;
        view_tok0 = u->tok0;
        view_pair = pair;
        view.length = u->length;
        int position = u->length + u->tok0 + token;
        view.hi = position + 1;
        if (a.parents) {
          // the sequence's nodes up to the unit's end, then a walk up from the row's own
          int8_t* up = up_s + tile * kMaxNodes;
          const int me_in = tid & 127;
          if (me_in < u->nodes) {
            const int p = __ldg(a.parents + u->seq_row0 + me_in);
            const bool fine = p >= -1 && p < me_in;
            if (!fine && a.status) atomicMax(a.status, 1);
            up[me_in] = (int8_t)(fine ? p : -1);
          }
          named_sync(2 + tile, 128);
          const int own = u->tok0 + token;
#pragma unroll
          for (int i = 0; i < kMaxNodes / 32; ++i) view.node[i] = 0;
          if (valid) {
            position = u->length;
#pragma unroll 1
            for (int i = up[own]; i >= 0; i = up[i]) ++position;
            int at = position;
#pragma unroll 1
            for (int i = own; i >= 0; i = up[i], --at) {
              const bool seen = a.window == 0 || at > position - a.reach || at < a.sink;
#pragma unroll
              for (int k = 0; k < kMaxNodes / 32; ++k) view.node[k] |= seen && (i >> 5) == k ? 1u << (i & 31) : 0u;
            }
          }
          named_sync(2 + tile, 128);
          view.hi = u->length;
        }
        view.lo = a.window == 0 ? 0 : max(0, position - a.reach + 1);
        view.sink = a.window == 0 ? 0 : min(a.sink, view.hi);
      }
      float m = -INFINITY, l = 0.0f;  // m: what exponents are taken from (log2 units), at most 8 below the maximum
      const bool rows_here = __any_sync(0xffffffffu, valid);
      const Seen seen_all = seen_of(*u);
      const int sink_tiles = u->sink_tiles, gap = (u->first - sink_tiles) * kKeys;
      const int jobs = C::kTiles == 2 && !pair ? 2 * n : n;
#pragma unroll 1
      for (int i = C::kTiles == 2 ? tile : 0; i < jobs; i += C::kTiles) {
        const int k_at = k0 + (C::kTiles == 2 && !pair ? i >> 1 : i), c = k_at * kKeys + (k_at < sink_tiles ? 0 : gap);
        const int b = i & 1;
        const uint32_t s_at = lanes + b * kKeys, p_ready = bar(C::kPReady + 2 * b);
        wait_quietly(bar(C::kSFull + b), full >> b & 1, abort_s);
        full ^= 1u << b;
        __syncwarp();
        tc::fence_after();
        auto ready = [&](int half) {
          tc::wait_st();
          tc::fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_ready + 8 * half);
        };
        // A row's new maximum (in log2 units): O keeps its scale while maxima go up by less than 2^8, l and O stay exact
        // multiples, far from overflow.  A row's own maximum alone decides for it, so that it does not depend on the rows
        // beside it.  Weights are up to 2^7 in f16 (and, with the eight, 2^15): under 2^-14 a 16-bit weight would be
        // subnormal.  O is at rest: these scores were asked for behind the product before.
        auto raise = [&](float top) {
          const float high = top * scale2 - (kF16 ? 7.0f : 0.0f);
          const bool higher = high > m + 8.0f || (m == -INFINITY && high > m);
          if (__any_sync(0xffffffffu, higher)) {
            const float turn = higher ? ex2_ftz(m - high) : 1.0f;
            m = higher ? high : m;
            l *= turn;
            if (i >= C::kTiles) {
              if (C::kTiles == 1) {  // of the other place: its product may still be under way
                wait_quietly(bar(C::kDone + 1), (rests - 1) & 1, abort_s);
                __syncwarp();
                tc::fence_after();
              }
#pragma unroll 1
              for (int d = 0; d < D; d += 32) {
                uint32_t o[32];
                tc::ld32(o, col_o + d);
                wait_ld32(o);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * turn);
                tc::st32(col_o + d, o);
              }
            }
          }
        };
        constexpr int kParts = kKeys / 32;
        const bool whole = seen_all.all_of_tile(c, a.sink);
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        auto weigh = [&](uint32_t (&p)[16], const uint32_t (&s)[32], float2 scale_2, float2 minus_2) {
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            float2 y = fma2(make_float2(__uint_as_float(s[2 * x]), __uint_as_float(s[2 * x + 1])), scale_2, minus_2);
            y.x = ex2_ftz(y.x);
            y.y = ex2_ftz(y.y);
            sum[x & 1] = add2(sum[x & 1], y);
            p[x] = pack2<kF16>(y.x, y.y);
          }
        };
        if (!rows_here) {  // what is in these rows' weights and sums, nobody reads
          if (lane == 0) {
            mbar_arrive(p_ready);
            mbar_arrive(p_ready + 8);
          }
        } else if (!C::kPre && (whole || !a.parents)) {
          uint32_t s[kParts][32];
#pragma unroll
          for (int k = 0; k < kParts; ++k) tc::ld32(s[k], s_at + 32 * k);
#pragma unroll
          for (int k = 0; k < kParts; ++k) wait_ld32(s[k]);
          if (!whole) {
            uint32_t w[kParts];
#pragma unroll
            for (int k = 0; k < kParts; ++k) w[k] = view.template bits<false>(c + 32 * k);
#pragma unroll
            for (int k = 0; k < kParts; ++k) {
              if (__all_sync(0xffffffffu, w[k] == 0xffffffffu)) continue;
#pragma unroll
              for (int x = 0; x < 32; ++x) s[k][x] = w[k] >> x & 1u ? s[k][x] : 0xff800000u;
            }
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int k = 0; k < kParts; ++k)
#pragma unroll
            for (int x = 0; x < 32; x += 8)
#pragma unroll
              for (int y = 0; y < 4; ++y)
                top[y] = max3(top[y], __uint_as_float(s[k][x + 2 * y]), __uint_as_float(s[k][x + 2 * y + 1]));
          raise(fmaxf(max3(top[0], top[1], top[2]), top[3]));
          const float minus = m == -INFINITY ? 0.0f : -m;  // a row that has seen nothing keeps weights of exp2(-inf) = 0
          const float2 scale_2 = make_float2(scale2, scale2), minus_2 = make_float2(minus, minus);
#pragma unroll
          for (int k = 0; k < kParts; ++k) {
            uint32_t p[16];
            weigh(p, s[k], scale_2, minus_2);
            tc::st16(s_at + 16 * k, p);
            if (k == kParts / 2 - 1) ready(0);
          }
          ready(1);
        } else {
          // Trees' tiles that some row does not see all of, and scores that are changed: 32 keys at a time, the scores as they
          // are meant put back by a first round.  Keys that none of the warp's rows sees cost nothing more.  (Prompts of 16,393
          // tokens with a window of 1,024, four tiles of ten: 170 us so, 161 by masks in registers as above.  For trees, with
          // one such tile or two, it makes no difference.)
          uint32_t live = 0;
          float top = -INFINITY;
#pragma unroll 1
          for (int k = 0; k < kParts; ++k) {
            uint32_t w = 0xffffffffu;
            if (!whole) w = a.parents ? view.template bits<true>(c + 32 * k) : view.template bits<false>(c + 32 * k);
            if (!__any_sync(0xffffffffu, valid && w != 0)) continue;
            live |= 1u << k;
            uint32_t s[32];
            tc::ld32(s, s_at + 32 * k);
            wait_ld32(s);
#pragma unroll
            for (int x = 0; x < 32; ++x) {
              float y = __uint_as_float(s[x]);
              if constexpr (C::kPre) y = a.softcap > 0.0f ? a.softcap * kLog2e * tanh_of(y * a.cap_in) : y * a.scale2;
              y = w >> x & 1u ? y : -INFINITY;
              top = fmaxf(top, y);
              s[x] = __float_as_uint(y);
            }
            tc::st32(s_at + 32 * k, s);
          }
          tc::wait_st();
          raise(top);
          const float minus = m == -INFINITY ? 0.0f : -m;
          const float2 scale_2 = make_float2(scale2, scale2), minus_2 = make_float2(minus, minus);
#pragma unroll 1
          for (int k = 0; k < kParts; ++k) {
            uint32_t p[16];
            if (live >> k & 1u) {
              uint32_t s[32];
              tc::ld32(s, s_at + 32 * k);
              wait_ld32(s);
              weigh(p, s, scale_2, minus_2);
            } else {
#pragma unroll
              for (int x = 0; x < 16; ++x) p[x] = 0;
            }
            tc::st16(s_at + 16 * k, p);  // over scores that have been read
            if (k == kParts / 2 - 1) ready(0);
          }
          ready(1);
        }
        sum[0] = add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
        ++rests;
      }

      // ------------------------------------------------------------------------------ the unit's rows
      if (jobs > (C::kTiles == 2 ? tile : 0)) {
        wait_quietly(bar(C::kDone + tile), done, abort_s);
        done ^= 1;
        __syncwarp();
      }
      tc::fence_after();
      // Values that were taken out of tiles come back, to the rows that see them (32 dims from d on of this row): rare,
      // and one by one.
      auto put_back = [&](uint32_t (&o)[32], int d) {
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
          const int c = u->tile(k0 + i) * kKeys;
          if (seen_all.all_of_tile(c, a.sink)) continue;
#pragma unroll 1
          for (int k = 0; k < kKeys; k += 32) {
            uint32_t w = valid ? (a.parents ? view.template bits<true>(c + k) : view.template bits<false>(c + k)) : 0u;
#pragma unroll 1
            while (w) {
              const int key = c + k + __ffs(w) - 1;
              w &= w - 1;
              const int column = key / a.page_tokens;
              int page = __ldg(a.page_table + (long long)u->seq * a.max_pages + column);
              if (page < 0 || page >= a.n_pages) page = 0;
              const uint32_t* v = static_cast<const uint32_t*>(a.v_pool) +
                                  ((((long long)page * a.n_kv_heads + u->head) * a.page_tokens + key - column * a.page_tokens) * D + d) / 2;
#pragma unroll
              for (int x = 0; x < 16; ++x) {
                const uint32_t two = __ldg(v + x), odd = not_finite2<kF16>(two);
                const float2 f = kF16 ? unpack_half2(two) : unpack_bf162(two);
                if (odd & 0xffffu) o[2 * x] = __float_as_uint(__uint_as_float(o[2 * x]) + f.x);
                if (odd >> 16) o[2 * x + 1] = __float_as_uint(__uint_as_float(o[2 * x + 1]) + f.y);
              }
            }
          }
        }
      };
      float f0 = 1.0f, f1 = 0.0f;
      const bool second = pair && n > 1;  // the other accumulator has a part
      if (pair) {
        if (tile == 1) {
          swap_s[r] = m;
          swap_s[kRowsTile + r] = l;
        }
        tc::fence_before();
        meet();
        tc::fence_after();
        if (second && tile == 0) {
          const float m1 = swap_s[r], l1 = swap_s[kRowsTile + r], now = fmaxf(m, m1);
          f0 = now == -INFINITY ? 1.0f : ex2_ftz(m - now);
          f1 = now == -INFINITY ? 1.0f : ex2_ftz(m1 - now);
          l = l * f0 + l1 * f1;
          m = now;
        }
      }
      // behind the barrier: the other row tile's last values may be looked over after this one's products are done
      const bool poison = *reinterpret_cast<volatile const int*>(&u->poison) != 0;
      if (rows_here && (!pair || tile == 0)) {
        const int row_in = (pair ? 0 : tile * kRowsTile) + r;
        const long long row = u->row0 + token, at_head = row * a.n_heads + (long long)u->head * a.group + head_in;
        const float inverse = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // nothing seen: zeros
        const long long n_slots = 2ll * gridDim.x;
        const bool cut = u->cut;
        if (valid) {
          if (cut) {
            float* rm = a.records + n_slots * C::kRows * D + (long long)u->slot * C::kRows + row_in;
            rm[0] = m;
            rm[n_slots * C::kRows] = l;
          } else if (a.lse) {
            a.lse[at_head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
          }
        }
#pragma unroll 1
        for (int d = 0; d < D; d += 32) {
          uint32_t o[32];
          tc::ld32(o, col_o + d);
          if (second) {
            uint32_t o1[32];
            tc::ld32(o1, col_o + C::kStepO + d);
            wait_ld32(o1);
            wait_ld32(o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f0 + __uint_as_float(o1[k]) * f1);
          } else {
            wait_ld32(o);
          }
          if (__builtin_expect(poison, 0)) put_back(o, d);
          if (cut && valid) {
            float4* rec = reinterpret_cast<float4*>(a.records) + ((long long)u->slot * (D / 4) + d / 4) * C::kRows + row_in;
#pragma unroll
            for (int k = 0; k < 8; ++k)
              rec[(long long)k * C::kRows] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                                         __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
          } else if (valid) {
            // a row that saw nothing has an accumulator of zero weights' products
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = inverse == 0.0f ? 0u : __float_as_uint(__uint_as_float(o[k]) * inverse);
            if (a.out_f32) {
              uint4* dst = reinterpret_cast<uint4*>(static_cast<float*>(a.out) + at_head * D + d);
#pragma unroll
              for (int k = 0; k < 8; ++k) dst[k] = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
            } else {
              uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at_head * D + d);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                auto two = [&](int i) {
                  return pack2<kF16>(__uint_as_float(o[8 * k + 2 * i]), __uint_as_float(o[8 * k + 2 * i + 1]));
                };
                dst[k] = make_uint4(two(0), two(1), two(2), two(3));
              }
            }
          }
          __syncwarp();
        }
        tc::fence_before();
      }
      // the sums, and the second accumulator, have been read
      if (pair) meet();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::kWEmpty + e));
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == kProducts) tc::dealloc512(tmem);
  // a wait that ran into its limit (some seconds): the outputs are not valid
  if (tid == 0 && *abort_s && a.status) atomicMax(a.status, 2);
}

// The records of the cut units become their rows.  A place is four dims of a row; rows lie side by side, as the records have
// them.  A CTA lists the units (one descriptor a thread) and takes every gridDim.x-th strip of places: 256 with a
// thread each, or 64 of a unit of many pieces, whose pieces four threads take in turn and join in shared memory.  What it takes
// is latency: two rounds of loads for up to eight pieces, and enough CTAs beside one another.  (Strips of 64 throughout and
// 2.4 times fewer CTAs: 50 to 150 us a call.  So, on a cold cache: 8 us for one tree of 8, 16 for the cut units of 9 windowed
// prompts of 64 dims, 26 for those of 24 trees of 61 nodes and 128 dims.)
constexpr int kJoinThreads = 256, kJoinFew = 8, kJoinLoads = 4, kJoinCtas = 5;
template <class C>
__global__ void __launch_bounds__(kJoinThreads, kJoinCtas) join_kernel(const __grid_constant__ Args a, int workers) {
  constexpr int D = C::D;
  __shared__ Desc desc_s[kMaxWorkers];
  __shared__ int first_s[kMaxWorkers + 1], sums_s[kJoinThreads / 32];
  __shared__ float part_s[3][6][kJoinThreads / 4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Desc mine;
  mine.pieces = 0;
  if (tid < workers) mine = a.desc[tid];
  const int wide = mine.pieces > kJoinFew ? kJoinThreads / 4 : kJoinThreads;  // places of a strip
  const int strips = mine.pieces > 0 ? (mine.tokens * a.group * (D / 4) + wide - 1) / wide : 0;
  int scan = strips;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int up = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += up;
  }
  if (lane == 31) sums_s[warp] = scan;
  __syncthreads();
  int total = 0;
  for (int w = 0; w < kJoinThreads / 32; ++w) {
    if (w < warp) scan += sums_s[w];
    total += sums_s[w];
  }
  desc_s[tid] = mine;
  first_s[tid] = scan - strips;
  __syncthreads();
  const long long n_slots = 2ll * workers;
  const float4* o = reinterpret_cast<const float4*>(a.records);
  const float* rm = a.records + n_slots * C::kRows * D;
  const float* rl = rm + n_slots * C::kRows;
#pragma unroll 1
  for (int strip = blockIdx.x; strip < total; strip += gridDim.x) {
    int lo = 0, hi = kJoinThreads - 1;  // the last unit that starts at the strip or before
#pragma unroll 1
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (first_s[mid] <= strip) lo = mid;
      else hi = mid - 1;
    }
    const Desc u = desc_s[lo];
    const bool many = u.pieces > kJoinFew;
    const int ways = many ? 4 : 1, way = many ? tid / (kJoinThreads / 4) : 0, at_strip = many ? tid % (kJoinThreads / 4) : tid;
    const int rows = u.tokens * a.group, place = (strip - first_s[lo]) * (kJoinThreads / ways) + at_strip;
    const int d4 = place / rows, r = place - d4 * rows, token = r / a.group;
    const int tile = token / a.tile_tokens, row_in = tile * kRowsTile + r - tile * a.tile_tokens * a.group;
    const bool real = d4 < D / 4;
    float m = -INFINITY, l = 0.0f;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // another part with maximum mk and sum lk: of none nothing is taken
    auto join = [&](float mk, float lk, float4 v) {
      if (lk == 0.0f) return;
      const float top = fmaxf(m, mk), f0 = m == top ? 1.0f : ex2_ftz(m - top), f1 = mk == top ? 1.0f : ex2_ftz(mk - top);
      m = top;
      l = l * f0 + lk * f1;
      sum.x = sum.x * f0 + v.x * f1;
      sum.y = sum.y * f0 + v.y * f1;
      sum.z = sum.z * f0 + v.z * f1;
      sum.w = sum.w * f0 + v.w * f1;
    };
    if (real) {
#pragma unroll 1
      for (int k0 = way; k0 < u.pieces; k0 += ways * kJoinLoads) {
        float mk[kJoinLoads], lk[kJoinLoads];
        float4 v[kJoinLoads];
#pragma unroll
        for (int i = 0; i < kJoinLoads; ++i) {
          const int k = k0 + ways * i;
          mk[i] = lk[i] = 0.0f;
          v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (k < u.pieces) {
            const long long slot = k == 0 ? 2ll * lo + 1 : 2ll * (lo + k);  // the CTA's of the first piece, then the next ones'
            mk[i] = __ldcg(rm + slot * C::kRows + row_in);
            lk[i] = __ldcg(rl + slot * C::kRows + row_in);
            v[i] = __ldcg(o + (slot * (D / 4) + d4) * C::kRows + row_in);
          }
        }
#pragma unroll
        for (int i = 0; i < kJoinLoads; ++i) join(mk[i], lk[i], v[i]);
      }
    }
    if (many) {
      if (way > 0) {
        float* p = &part_s[way - 1][0][at_strip];
        p[0] = m;
        p[kJoinThreads / 4] = l;
        p[2 * kJoinThreads / 4] = sum.x;
        p[3 * kJoinThreads / 4] = sum.y;
        p[4 * kJoinThreads / 4] = sum.z;
        p[5 * kJoinThreads / 4] = sum.w;
      }
      __syncthreads();
      if (way == 0) {
#pragma unroll 1
        for (int i = 0; i < 3; ++i) {
          const float* p = &part_s[i][0][at_strip];
          join(p[0], p[kJoinThreads / 4], make_float4(p[2 * kJoinThreads / 4], p[3 * kJoinThreads / 4], p[4 * kJoinThreads / 4],
                                                      p[5 * kJoinThreads / 4]));
        }
      }
    }
    if (way == 0 && real) {
      const float inverse = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      if (inverse == 0.0f) sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const long long at_head = (long long)(u.row0 + token) * a.n_heads + (long long)u.head * a.group + r - token * a.group;
      const long long at = at_head * D + 4 * d4;
      if (a.out_f32) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) =
            make_float4(sum.x * inverse, sum.y * inverse, sum.z * inverse, sum.w * inverse);
      } else {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
            make_uint2(pack2<C::kF16>(sum.x * inverse, sum.y * inverse), pack2<C::kF16>(sum.z * inverse, sum.w * inverse));
      }
      if (a.lse && d4 == 0) a.lse[at_head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
    }
    if (many) __syncthreads();
  }
}

static int64_t desc_bytes(int workers) { return (workers * (int64_t)sizeof(Desc) + 255) / 256 * 256; }
static int64_t workspace_bytes(int workers, int head_dim) {
  const int rows = head_dim == 256 ? kRowsTile : 2 * kRowsTile;
  return desc_bytes(workers) + 2ll * workers * rows * (head_dim + 2) * 4;
}

template <class C>
static int launch(const asterq_rows_attention_params* p, Args& a, int workers, int dev, cudaStream_t s) {
  // a box of keys lies in one page: the largest of the tile, its half, .. down to 16 tokens that divides the page
  a.box_rows = C::kKeys;
  while (a.page_tokens % a.box_rows) a.box_rows /= 2;
  a.tile_tokens = kRowsTile / a.group;
  a.unit_tokens = C::kQTiles * a.tile_tokens;
  CUtensorMap q_map, k_map, v_map;
  const cuuint64_t q_dims[3] = {(cuuint64_t)C::D, (cuuint64_t)a.n_heads, (cuuint64_t)a.n_rows};
  const cuuint64_t q_strides[2] = {(cuuint64_t)p->q_head_stride * 2, (cuuint64_t)p->q_row_stride * 2};
  const cuuint32_t q_box[3] = {64u, (cuuint32_t)a.group, (cuuint32_t)a.tile_tokens};
  const bool pools = a.capacity > 0;  // with none, no row is answered and the maps are never read
  const cuuint64_t dims[4] = {64u, (cuuint64_t)a.page_tokens, (cuuint64_t)C::D / 64,
                              (cuuint64_t)(pools ? a.n_pages * a.n_kv_heads : 1)};
  const cuuint64_t strides[3] = {(cuuint64_t)C::D * 2, 128u, (cuuint64_t)C::D * 2 * a.page_tokens};
  const cuuint32_t box[4] = {64u, (cuuint32_t)a.box_rows, 1u, 1u};
  if (!map_of_16bit(&q_map, p->q, 3, q_dims, q_strides, q_box) ||
      !map_of_16bit(&k_map, pools ? p->k_pool : p->workspace, 4, dims, strides, box) ||
      !map_of_16bit(&v_map, pools ? p->v_pool : p->workspace, 4, dims, strides, box))
    return set_error(ASTERQ_ERR_CUDA, "rows_attention: tensor map encoding failed");
  const std::lock_guard<std::mutex> guard(launch_lock());
  static unsigned long long configured = 0;  // one bit per device ordinal
  if (dev >= 64 || !(configured & (1ull << dev))) {
    cudaFuncAttributes f;
    cudaError_t e = cudaFuncGetAttributes(&f, rows_kernel<C>);
    if (e == cudaSuccess && f.numRegs != kRegsLaunch)  // a split over what was launched with would wait for good
      return set_error(ASTERQ_ERR_UNSUPPORTED, "rows_attention: built with %d registers, not %d", f.numRegs, kRegsLaunch);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(rows_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess)
      return set_error(ASTERQ_ERR_CUDA, "rows_attention: shared memory opt-in: %s", cudaGetErrorString(e));
    if (dev < 64) configured |= 1ull << dev;
  }
  rows_kernel<C><<<workers, kThreads, C::kSmem, s>>>(q_map, k_map, v_map, a);
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t join = {};
  join.gridDim = kJoinCtas * workers;
  join.blockDim = kJoinThreads;
  join.stream = s;
  join.attrs = early;
  join.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&join, join_kernel<C>, a, workers);
  if (e != cudaSuccess) return set_error(ASTERQ_ERR_CUDA, "rows_attention: launch failed: %s", cudaGetErrorString(e));
  return check_launch("rows_attention");
}

// Units of one row tile where sequences have no more rows than that on average, and where there are units enough to be bound
// by memory; the sixth slot of 32 KB has more loads under way then.  One and two row tiles a unit, 32 heads of 128 dims over 8 kv heads:
// 32 trees of 16 nodes 123 and 130 us, 512 of them 636 and 718, 64 decode rows over 16,384 cached tokens 669 and 777, a chunk of
// 1,900 tokens beside 63 decode rows over 4,096 each 329 and 430, 2,000 beside 255 860 and 1,263.  The average misses long rows among many
// short ones over little cache (7,900 tokens beside 255 rows over 500: 895 and 711), as each tile of keys and values of the long one is then
// read by twice as many units.
// Idle sequences are left out of the average from four row tiles an SM on: one prompt beside 255 of them 43 and 47 us for 1,000
// tokens, 83 and 82 for 2,000, 211 and 186 for 4,000, 642 and 551 for 8,000.
template <bool kF16, int D, bool kPre>
static int by_rows(const asterq_rows_attention_params* p, Args& a, int workers, int dev, cudaStream_t s) {
  if constexpr (D != 256) {
    const bool many = p->n_rows * p->n_heads > (int64_t)workers * 4 * kRowsTile;
    const int64_t seqs = many && p->n_active > 0 && p->n_active < p->n_seqs ? p->n_active : p->n_seqs;
    if (seqs * p->n_kv_heads >= workers && p->n_rows <= seqs * (kRowsTile / a.group))
      return launch<Cfg<kF16, D, kPre, true>>(p, a, workers, dev, s);
  }
  return launch<Cfg<kF16, D, kPre, false>>(p, a, workers, dev, s);
}
template <bool kF16, int D>
static int by_scale(const asterq_rows_attention_params* p, Args& a, bool pre, int workers, int dev, cudaStream_t s) {
  return pre ? by_rows<kF16, D, true>(p, a, workers, dev, s) : by_rows<kF16, D, false>(p, a, workers, dev, s);
}

static int check(const asterq_rows_attention_params* p) {
  if (!p) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "rows_attention: null parameters");
  if (p->n_seqs < 0 || p->n_rows < 0 || p->n_heads <= 0 || p->n_kv_heads <= 0 || p->n_heads % p->n_kv_heads ||
      p->page_tokens <= 0 || p->max_pages < 0 || p->n_pages < 0 || p->window < 0 || p->sink < 0 || p->n_active < 0)
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "rows_attention: bad sizes");
  if (p->dtype != ASTERQ_DTYPE_BF16 && p->dtype != ASTERQ_DTYPE_F16)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "rows_attention: dtype %d: bf16 or f16", p->dtype);
  if (p->out_dtype != p->dtype && p->out_dtype != ASTERQ_DTYPE_F32)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "rows_attention: the output is of the queries' type or f32");
  if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "rows_attention: head_dim %d: 64, 128 or 256", p->head_dim);
  if (p->n_heads / p->n_kv_heads > kRowsTile)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "rows_attention: %d query heads a kv head: at most %d",
                     p->n_heads / p->n_kv_heads, kRowsTile);
  if (p->page_tokens % 16)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "rows_attention: page_tokens %d must be a multiple of 16", p->page_tokens);
  if (p->n_pages * p->n_kv_heads > 0x7fffffffLL || (int64_t)p->max_pages * p->page_tokens > 0x7fff0000LL ||
      p->n_rows > 0x7fff0000LL)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "rows_attention: more than 2^31 pages, rows or tokens of a sequence");
  return ASTERQ_OK;
}

}  // namespace rat
}  // namespace asterq

using namespace asterq;

extern "C" int64_t asterq_rows_attention_workspace_bytes(const asterq_rows_attention_params* p) {
  clear_error();
  if (rat::check(p) != ASTERQ_OK) return 0;
  int dev = 0;
  const int workers = current_sms(&dev);
  return rat::workspace_bytes(workers > 0 && workers < rat::kMaxWorkers ? workers : rat::kMaxWorkers, p->head_dim);
}

extern "C" int asterq_rows_attention(const asterq_rows_attention_params* p, void* stream) {
  clear_error();
  int st = rat::check(p);
  if (st != ASTERQ_OK) return st;
  if (p->n_rows == 0 || p->n_seqs == 0) return ASTERQ_OK;
  if (!p->q || !p->lengths || !p->row_offsets || !p->out || !p->workspace ||
      (p->max_pages > 0 && p->n_pages > 0 && (!p->k_pool || !p->v_pool)) || (p->max_pages > 0 && !p->page_table))
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "rows_attention: null pointer");
  const void* vec[] = {p->q, p->k_pool, p->v_pool, p->out, p->workspace};
  for (const void* ptr : vec)
    if (reinterpret_cast<uintptr_t>(ptr) & 15)
      return set_error(ASTERQ_ERR_MISALIGNED, "rows_attention: arrays must be 16-byte aligned");
  if (p->q_row_stride % 8 || p->q_head_stride % 8)
    return set_error(ASTERQ_ERR_MISALIGNED, "rows_attention: the queries' strides must be multiples of 8");
  if (p->q_row_stride <= 0 || p->q_head_stride <= 0)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "rows_attention: the queries' strides must be positive");
  int dev = 0;
  int workers = current_sms(&dev);
  if (workers <= 0) return set_error(ASTERQ_ERR_CUDA, "rows_attention: no CUDA device");
  workers = workers < rat::kMaxWorkers ? workers : rat::kMaxWorkers;
  if (p->workspace_bytes < rat::workspace_bytes(workers, p->head_dim))
    return set_error(ASTERQ_ERR_WORKSPACE, "rows_attention: workspace of %lld bytes, %lld needed",
                     (long long)p->workspace_bytes, (long long)rat::workspace_bytes(workers, p->head_dim));
  rat::Args a = {};
  a.q = p->q;
  a.page_table = p->page_table;
  a.lengths = p->lengths;
  a.row_offsets = p->row_offsets;
  a.parents = p->parents;
  a.v_pool = p->v_pool;
  a.out = p->out;
  a.lse = p->lse;
  a.desc = static_cast<rat::Desc*>(p->workspace);
  a.records = reinterpret_cast<float*>(static_cast<char*>(p->workspace) + rat::desc_bytes(workers));
  a.status = p->status;
  a.n_rows = p->n_rows;
  a.n_pages = p->n_pages;
  a.capacity = p->n_pages > 0 ? (long long)p->max_pages * p->page_tokens : 0;
  a.n_seqs = p->n_seqs;
  a.n_heads = p->n_heads;
  a.n_kv_heads = p->n_kv_heads;
  a.group = p->n_heads / p->n_kv_heads;
  a.page_tokens = p->page_tokens;
  a.max_pages = p->max_pages;
  a.window = p->window;
  a.sink = p->window > 0 ? (p->sink < p->window ? p->sink : p->window) : 0;
  a.reach = p->window - a.sink;
  a.out_f32 = p->out_dtype == ASTERQ_DTYPE_F32;
  a.scale = p->softmax_scale;
  a.scale2 = a.scale * rat::kLog2e;
  a.softcap = p->logit_softcap > 0.0f ? p->logit_softcap : 0.0f;
  a.cap_in = a.softcap > 0.0f ? a.scale / a.softcap : 0.0f;
  // the maximum is taken of what the tensor cores give, before the scale, where that keeps the order
  const bool pre = a.softcap > 0.0f || !(a.scale > 0.0f);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool f16 = p->dtype == ASTERQ_DTYPE_F16;
  switch (p->head_dim) {
    case 64: return f16 ? rat::by_scale<true, 64>(p, a, pre, workers, dev, s) : rat::by_scale<false, 64>(p, a, pre, workers, dev, s);
    case 128: return f16 ? rat::by_scale<true, 128>(p, a, pre, workers, dev, s)
                         : rat::by_scale<false, 128>(p, a, pre, workers, dev, s);
    default: return f16 ? rat::by_scale<true, 256>(p, a, pre, workers, dev, s)
                        : rat::by_scale<false, 256>(p, a, pre, workers, dev, s);
  }
}
