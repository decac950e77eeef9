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
// and values that TMA brings; two warpgroups take a tile each, thread t row t, so that maxima and sums need no
// shuffles, and one's exponentials run under the other's products.  A unit of at most 128 rows has both warpgroups on
// the same rows and alternate tiles of keys; they join at its end, through tensor memory.
// S = Q K^T (128 x 128) lies in tensor memory, its weights as 16-bit values over it, O beside it.
//
// Split.  The key tiles of all units laid end to end (with kUnitCost in front of each) are cut into equal contiguous
// shares, one for each CTA, by sums over lengths and offsets that every CTA does for itself: no planning launch, no
// copy of lengths to the host.  A cut unit leaves (o, m, l) records in the workspace, and a second small grid joins
// them in the order of the shares.
#include "asterq_internal.h"
#include "common.cuh"
#include "launch.cuh"
#include "tcgen05.cuh"

namespace asterq {
namespace rat {

constexpr int kMaxWorkers = 256;
constexpr int kThreads = 384, kWarps = 12;
constexpr int kRowsTile = 128;
constexpr int kMaxNodes = 128;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
// registers of a thread: 256 x 216 + 128 x 72 = 384 x 168 of the launch
constexpr int kRegsLaunch = 168, kRegsSoftmax = 216, kRegsHelp = 72;
static_assert(256 * kRegsSoftmax + 128 * kRegsHelp <= kThreads * kRegsLaunch, "more registers than launched with");
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
  int out_f32, premultiply;
  float scale, scale2, softcap, cap_in;
};

template <bool kF16_, int D_>
struct Cfg {
  static constexpr bool kF16 = kF16_;
  static constexpr int D = D_;
  static constexpr int kTiles = D == 256 ? 1 : 2;  // row tiles of a unit: two accumulators of 256 dims leave no room for scores
  static constexpr int kKeys = D == 256 ? 64 : 128;
  static constexpr int kRows = kTiles * kRowsTile;
  static constexpr int kQBytes = kRowsTile * D * 2, kSlotBytes = kKeys * D * 2;
  static constexpr int kSlots = D == 64 ? 12 : 5;
  static constexpr int kColS = 0, kColO = 256, kStepS = 128, kStepO = D;
  static constexpr int kSmall = 2048;  // barriers, work entries, parents, the sums of a joined pair
  static constexpr int kSmem = 1024 + kTiles * kQBytes + kSlots * kSlotBytes + kSmall;
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
// first + k - sink_tiles from there on.
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
    const int from = q.length + (a.parents ? 0 : s.tok0) - a.reach + 1;
    if (from > 0) {
      s.from = from;
      s.sink_tiles = min((a.sink + kKeys - 1) / kKeys, last);
      s.first = a.reach == 0 ? last : max(from / kKeys, s.sink_tiles);
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
  long long x;
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

template <class C>
__global__ void __launch_bounds__(kThreads, 1)
    rows_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                const __grid_constant__ CUtensorMap v_map, const __grid_constant__ Args a) {
  constexpr int D = C::D, kKeys = C::kKeys;
  constexpr bool kF16 = C::kF16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t q_base = smem_u32(smem), ring = q_base + C::kTiles * C::kQBytes;
  uint8_t* small = smem + C::kTiles * C::kQBytes + C::kSlots * C::kSlotBytes;
  // barriers: full and empty of each slot, the others by name, and at the end whether a slot's values were looked over
  const uint32_t bars = smem_u32(small);
  constexpr int kEmpty = C::kSlots, kQFull = 2 * C::kSlots, kQEmpty = kQFull + 1, kWFull = kQEmpty + 1, kWEmpty = kWFull + 2,
                kSFull = kWEmpty + 2, kPReady = kSFull + 2, kOFull = kPReady + 2, kClean = kOFull + 2, kDrain = kClean + C::kSlots,
                kBars = kDrain + 1;
  static_assert(kBars * 8 <= 448, "barriers");
  auto bar = [&](int i) { return bars + 8 * i; };
  Work* work = reinterpret_cast<Work*>(small + 448);                   // [2]
  int8_t* up_s = reinterpret_cast<int8_t*>(small + 448 + 160);      // [2][kMaxNodes]
  float* pair_s = reinterpret_cast<float*>(small + 448 + 160 + 256);   // [2][kRowsTile]: m and l of the second warpgroup
  long long* scan_s = reinterpret_cast<long long*>(small + 448 + 160 + 256 + 1024);  // [kWarps]
  Start* start_s = reinterpret_cast<Start*>(small + 448 + 160 + 256 + 1024 + 96);
  uint32_t* tmem_s = reinterpret_cast<uint32_t*>(small + 448 + 160 + 256 + 1024 + 96 + 32);
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_s + 1);
  volatile int* never_s = reinterpret_cast<volatile int*>(tmem_s + 2);
  static_assert(sizeof(Work) == 80 && sizeof(Start) <= 32 && 448 + 160 + 256 + 1024 + 96 + 32 + 12 <= C::kSmall, "small");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, me = blockIdx.x;

  asm volatile("griddepcontrol.launch_dependents;");
  if (tid == 0) {
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(bar(i), 1);
      mbar_init(bar(kEmpty + i), 3);  // the products', and two warps that look values over
      mbar_init(bar(kClean + i), 2);
    }
    mbar_init(bar(kQFull), 1);
    mbar_init(bar(kQEmpty), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kWFull + i), 1);
      mbar_init(bar(kWEmpty + i), 11);
      mbar_init(bar(kSFull + i), 1);
      mbar_init(bar(kPReady + i), 4);
      mbar_init(bar(kOFull + i), 1);
    }
    mbar_init(bar(kDrain), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *abort_s = 0;
    *never_s = 0;
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
    if (blocks <= 4)
      for (int b = 0; b < blocks; ++b) cost += span_of<kKeys>(a, q, b).tiles + kUnitCost;
    uint32_t many = __ballot_sync(0xffffffffu, blocks > 4);
    while (many) {
      const int from = __ffs(many) - 1;
      many &= many - 1;
      Seq o;
      o.n = __shfl_sync(0xffffffffu, q.n, from);
      o.length = __shfl_sync(0xffffffffu, q.length, from);
      const int n = __shfl_sync(0xffffffffu, blocks, from);
      long long sum = 0;
      for (int b = lane; b < n; b += 32) sum += span_of<kKeys>(a, o, b).tiles + kUnitCost;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (lane == from) cost = sum;
    }
    return cost * a.n_kv_heads;
  };
  long long sum = 0;
  for (int base = s_begin; base < s_end; base += 32) {
    Seq q;
    sum += costs_of(base, q);
  }
#pragma unroll
  for (int d = 1; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) scan_s[warp] = sum;
  // offsets out of order or out of range: which rows are whose is not known, and the call is left undone
  if (__syncthreads_or(any_bad)) {
    if (tid == 0) {
      a.desc[me].pieces = 0;
      if (a.status) atomicMax(a.status, 1);
    }
    return;
  }
  long long before = 0, total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += scan_s[w];
    total += scan_s[w];
  }
  // CTAs that take part: each has kMinShare tiles or more
  const int W = (int)max(1ll, min((long long)gridDim.x, total / kMinShare));
  const long long x0 = total * min(me, W) / W, x1 = total * min(me + 1, W) / W;
  if (x0 < x1 && before <= x0 && x0 < before + sum) {
    long long at = before;
    for (int base = s_begin; base < s_end; base += 32) {
      Seq q;
      const long long cost = costs_of(base, q);
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
      const long long head_cost = __shfl_sync(0xffffffffu, cost, here) / a.n_kv_heads;
      Seq o;
      o.n = __shfl_sync(0xffffffffu, q.n, here);
      o.length = __shfl_sync(0xffffffffu, q.length, here);
      const int head = (int)((x0 - at) / head_cost);
      long long rest = x0 - at - head * head_cost;
      const int blocks = (o.n + a.unit_tokens - 1) / a.unit_tokens;
      for (int b0 = 0; b0 < blocks; b0 += 32) {
        long long c = b0 + lane < blocks ? span_of<kKeys>(a, o, b0 + lane).tiles + kUnitCost : 0, up_to = c;
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
        const int l = __ffs(in) - 1;
        if (lane == l) {
          start_s->s = base + here;
          start_s->head = head;
          start_s->block = b0 + l;
          start_s->at = (int)(rest - (up_to - c));
        }
        break;
      }
      break;
    }
  }
  // rows that are not answered: zeros, and a log-sum of -inf
  for (int base = (me * kWarps + warp) * 32; base < a.n_seqs; base += gridDim.x * kWarps * 32) {
    bool bad = false;
    int dead = 0;
    Seq q;
    q.n = 0;
    if (base + lane < a.n_seqs) q = seq_of(a, base + lane, bad, dead);
    if (dead > 0 && q.length >= 0 && a.status) atomicMax(a.status, 1);
    uint32_t some = __ballot_sync(0xffffffffu, dead > 0);
    while (some) {
      const int from = __ffs(some) - 1;
      some &= some - 1;
      const long long row = __shfl_sync(0xffffffffu, q.row0 + q.n, from), rows = __shfl_sync(0xffffffffu, dead, from);
      const long long w0 = row * a.n_heads * D, n = rows * a.n_heads * D;
      for (long long i = lane * 8; i < n; i += 256) {
        if (a.out_f32) {
          float4* o = reinterpret_cast<float4*>(static_cast<float*>(a.out) + w0 + i);
          o[0] = o[1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        } else {
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + w0 + i) = make_uint4(0, 0, 0, 0);
        }
      }
      if (a.lse)
        for (long long i = lane; i < rows * a.n_heads; i += 32) a.lse[row * a.n_heads + i] = -INFINITY;
    }
  }
  __syncthreads();
  if (x0 >= x1) {
    if (tid == 0) a.desc[me].pieces = 0;
    return;
  }
  if (warp == 9) tc::alloc512(smem_u32(tmem_s));
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_s;

  // tiles that some row of the unit does not see all of
  auto partial = [&](const Work& u, int c) {
    const bool seen = c + kKeys <= (a.parents ? u.length : u.length + u.tok0 + 1);
    if (!seen) return true;
    if (a.window == 0 || c + kKeys <= a.sink) return false;
    const long long newest = (long long)u.length + (a.parents ? u.nodes : u.tok0 + u.tokens) - 1;
    return c <= newest - a.reach;
  };
  // where a piece's tiles lie in the ring: K0 K1 V0 K2 V1 .., behind `base` uses of it
  auto place_k = [](int j) { return j == 0 ? 0 : 2 * j - 1; };
  auto place_v = [](int j, int n) { return j + 1 < n ? 2 * j + 2 : 2 * n - 1; };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsHelp));
    if (warp == 8) {
      // ------------------------------------------------------------------------------ loads
      Desc desc;
      desc.pieces = 0;
      bool ok = true;
      int s = start_s->s, head = start_s->head, block = start_s->block, at = start_s->at;
      long long x = x0;
      bool bad;
      int dead;
      Seq q = seq_of(a, s, bad, dead);
      Span span = span_of<kKeys>(a, q, block);
      uint32_t base = 0;  // uses of the ring's slots
      uint32_t q_bytes = 0;
      int pieces = 0;
      const int boxes = kKeys / a.box_rows, halves = D / 64;
      const uint32_t box_bytes = a.box_rows * 128;
      const int my_box = lane / halves, my_half = lane % halves;  // one lane a box
      while (ok && x < x1) {
        const int cost = (int)min((long long)(span.tiles + kUnitCost - at), x1 - x);
        const int k0 = max(at - kUnitCost, 0), n = max(at + cost - kUnitCost, 0) - k0;
        if (n > 0) {
          const int e = pieces & 1;
          if (pieces >= 2) ok = mbar_wait(bar(kWEmpty + e), ((pieces >> 1) - 1) & 1, abort_s);
          ok = __all_sync(0xffffffffu, (int)ok) != 0;
          if (!ok) break;
          const bool cut = n < span.tiles;
          if (lane == 0) {
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
            u.seq = s;
            u.nodes = span.tok0 + span.tokens;
            u.pair = C::kTiles == 2 && span.tokens <= a.tile_tokens;
            u.cut = cut;
            u.slot = 2 * me + (k0 == 0);
            u.poison = 0;
            work[e] = u;
            mbar_arrive(bar(kWFull + e));
            if (cut && k0 == 0) {
              // the pieces after this one are in the next CTAs' first slots
              const long long u1 = x - at + kUnitCost + span.tiles;
              desc.pieces = (int)((u1 * W - 1) / total) - me + 1;
              desc.row0 = u.row0;
              desc.tokens = u.tokens;
              desc.head = head;
            }
          }
          __syncwarp();
          // queries
          if (pieces > 0) ok = mbar_wait(bar(kQEmpty), (pieces - 1) & 1, abort_s);
          ok = __all_sync(0xffffffffu, (int)ok) != 0;
          if (!ok) break;
          const int q_tiles = span.tokens > a.tile_tokens ? 2 : 1;
          q_bytes = q_tiles * halves * a.tile_tokens * a.group * 128;
          if (lane == 0) mbar_expect_tx(bar(kQFull), q_bytes);
          __syncwarp();
          if (lane < q_tiles * halves) {
            const int t = lane / halves, h = lane % halves;
            tma_q(q_base + t * C::kQBytes + h * (kRowsTile * 128), &q_map, h * 64, head * a.group,
                  q.row0 + span.tok0 + t * a.tile_tokens, bar(kQFull));
          }
          ++pieces;
          // keys and values
          for (int i = 0; i < 2 * n && ok; ++i) {
            // position i of K0 K1 V0 K2 V1 .. K(n-1) V(n-2) V(n-1)
            const bool is_v = i == 2 * n - 1 || (i > 0 && (i & 1) == 0);
            const int j = i == 2 * n - 1 ? n - 1 : i == 0 ? 0 : is_v ? i / 2 - 1 : (i + 1) / 2;
            const uint32_t use = base + i, slot = use % C::kSlots, round = use / C::kSlots;
            const int k = k0 + j, tile = k < span.sink_tiles ? k : span.first + (k - span.sink_tiles);
            const int token = tile * kKeys + my_box * a.box_rows;
            const bool want = lane < boxes * halves && token < span.end &&
                              (token < a.sink || token + a.box_rows > span.from);
            int page = 0, column = 0;
            if (want) {
              column = token / a.page_tokens;
              page = __ldg(a.page_table + (long long)s * a.max_pages + column);
            }
            if (round > 0) ok = mbar_wait(bar(kEmpty + slot), (round - 1) & 1, abort_s);
            ok = __all_sync(0xffffffffu, (int)ok) != 0;
            if (!ok) break;
            const uint32_t wanted = __ballot_sync(0xffffffffu, want);
            if (lane == 0) mbar_expect_tx(bar(slot), __popc(wanted) * box_bytes);
            __syncwarp();
            if (want) {
              if (page < 0 || page >= a.n_pages) {
                if (a.status) atomicMax(a.status, 1);
                page = 0;
              }
              tma_kv(ring + slot * C::kSlotBytes + my_half * (kKeys * 128) + my_box * box_bytes, is_v ? &v_map : &k_map,
                     token - column * a.page_tokens, my_half, page * a.n_kv_heads + head, bar(slot));
            }
          }
          if (!ok) break;
          base += 2 * n;
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
              do q = seq_of(a, ++s, bad, dead);
              while (q.n == 0);
            }
          }
          span = span_of<kKeys>(a, q, block);
        }
      }
      if (ok) {
        const int e = pieces & 1;
        if (pieces >= 2) ok = mbar_wait(bar(kWEmpty + e), ((pieces >> 1) - 1) & 1, abort_s);
        ok = __all_sync(0xffffffffu, (int)ok) != 0;
        if (ok && lane == 0) {
          work[e].n = 0;
          mbar_arrive(bar(kWFull + e));
        }
      }
      if (!ok) {
        // the last copies have landed before the exit, also when nobody waits for them any more: each slot's barrier
        // ends a phase that it is in within the limit, or has ended the ones begun
        __syncwarp();
        for (int i = 0; i <= kQFull; i = i + 1 == C::kSlots ? kQFull : i + 1)
          for (int parity = 0; parity < 2; ++parity) (void)mbar_wait(bar(i), parity, never_s, 50000000);
      }
      if (lane == 0) a.desc[me] = desc;
    } else if (warp == 9) {
      // ------------------------------------------------------------------------------ products
      constexpr uint32_t kQk = idesc(kF16, kKeys, false), kPv = idesc(kF16, D, true);
      bool ok = true;
      uint32_t base = 0, s_ready[2] = {0, 0};
      for (int piece = 0; ok; ++piece) {
        const int e = piece & 1;
        ok = mbar_wait(bar(kWFull + e), (piece >> 1) & 1, abort_s);
        ok = __all_sync(0xffffffffu, (int)ok) != 0;
        if (!ok) break;
        const Work u = work[e];
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kWEmpty + e));
        if (u.n == 0) break;
        ok = mbar_wait(bar(kQFull), piece & 1, abort_s);
        auto slot_of = [&](int place) { return (base + place) % C::kSlots; };
        auto wait_slot = [&](int place) {
          const uint32_t use = base + place;
          ok = ok && mbar_wait(bar(use % C::kSlots), (use / C::kSlots) & 1, abort_s);
        };
        auto qk = [&](int stream, int row_tile, int j) {
          const uint32_t q0 = tc::desc_k_major(q_base + row_tile * C::kQBytes);
          const uint32_t k0 = tc::desc_k_major(ring + slot_of(place_k(j)) * C::kSlotBytes);
          if (tc::elect()) {
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
              tc::mma_ss(tmem + C::kColS + stream * C::kStepS, q0 + s / 4 * (kRowsTile * 8) + s % 4 * 2,
                         k0 + s / 4 * (kKeys * 8) + s % 4 * 2, kQk, s > 0);
            tc::commit(bar(kSFull + stream));
          }
          __syncwarp();
        };
        auto pv = [&](int stream, int j, bool first) {
          const uint32_t v0 = tc::desc_mn_major(ring + slot_of(place_v(j, u.n)) * C::kSlotBytes, kKeys * 128);
          ok = ok && mbar_wait(bar(kPReady + stream), s_ready[stream] & 1, abort_s);
          ++s_ready[stream];
          ok = __all_sync(0xffffffffu, (int)ok) != 0;
          if (!ok) return;
          tc::fence_after();
          if (tc::elect()) {
#pragma unroll
            for (int s = 0; s < kKeys / 16; ++s)
              tc::mma_ts(tmem + C::kColO + stream * C::kStepO, tmem + C::kColS + stream * C::kStepS + 8 * s, v0 + s * 128,
                         kPv, !first || s > 0);
          }
          __syncwarp();
        };
        auto wait_values = [&](int j) {
          wait_slot(place_v(j, u.n));
          if (partial(u, u.tile(u.k0 + j) * kKeys)) {
            const uint32_t use = base + place_v(j, u.n);
            ok = ok && mbar_wait(bar(kClean + use % C::kSlots), (use / C::kSlots) & 1, abort_s);
          }
        };
        auto signal = [&](int b) {
          if (tc::elect()) tc::commit(bar(b));
          __syncwarp();
        };
        const int streams = C::kTiles == 2 ? 2 : 1;
        wait_slot(place_k(0));
        ok = __all_sync(0xffffffffu, (int)ok) != 0;
        if (!ok) break;
        if (u.pair) {
          qk(0, 0, 0);
          signal(kEmpty + slot_of(place_k(0)));
          if (u.n > 1) {
            wait_slot(place_k(1));
            ok = __all_sync(0xffffffffu, (int)ok) != 0;
            if (!ok) break;
            qk(1, 0, 1);
            signal(kEmpty + slot_of(place_k(1)));
          }
          if (u.n <= 2) signal(kQEmpty);
          for (int j = 0; j < u.n && ok; ++j) {
            wait_values(j);
            pv(j & 1, j, j < 2);
            if (!ok) break;
            signal(kEmpty + slot_of(place_v(j, u.n)));
            if (j + 2 < u.n) {
              wait_slot(place_k(j + 2));
              ok = __all_sync(0xffffffffu, (int)ok) != 0;
              if (!ok) break;
              qk(j & 1, 0, j + 2);
              signal(kEmpty + slot_of(place_k(j + 2)));
              if (j + 3 == u.n) signal(kQEmpty);
            }
          }
          if (!ok) break;
          signal(kOFull);
          signal(kOFull + 1);
        } else {
          for (int t = 0; t < streams; ++t) qk(t, t, 0);
          signal(kEmpty + slot_of(place_k(0)));
          if (u.n == 1) signal(kQEmpty);
          for (int j = 0; j < u.n && ok; ++j) {
            wait_values(j);
            for (int t = 0; t < streams && ok; ++t) {
              pv(t, j, j == 0);
              if (!ok) break;
              if (t + 1 == streams) signal(kEmpty + slot_of(place_v(j, u.n)));
              if (j + 1 == u.n) signal(kOFull + t);
              if (j + 1 < u.n) {
                if (t == 0) wait_slot(place_k(j + 1));
                ok = __all_sync(0xffffffffu, (int)ok) != 0;
                if (!ok) break;
                qk(t, t, j + 1);
                if (t + 1 == streams) {
                  signal(kEmpty + slot_of(place_k(j + 1)));
                  if (j + 2 == u.n) signal(kQEmpty);
                }
              }
            }
          }
          if (!ok) break;
        }
        base += 2 * u.n;
      }
      if (!ok) {  // products under way end before tensor memory goes
        __syncwarp();
        if (tc::elect()) tc::commit(bar(kDrain));
        __syncwarp();
        (void)mbar_wait(bar(kDrain), 0, never_s, 200000000);
      }
    } else {
      // ------------------------------------------------------------------------------ values looked over
      // In a tile that not every row sees all of, a weight of zero meets values that the row does not see, and zero
      // times an infinity or NaN is not zero.  Values that no row sees become zeros; of the others those that are not
      // finite do, and the rows' threads add them where they are seen (poison).
      bool ok = true;
      uint32_t base = 0;
      const int part = warp - 10;
      for (int piece = 0; ok; ++piece) {
        const int e = piece & 1;
        ok = mbar_wait(bar(kWFull + e), (piece >> 1) & 1, abort_s);
        ok = __all_sync(0xffffffffu, (int)ok) != 0;
        if (!ok) break;
        const Work u = work[e];
        const int end = u.length + u.nodes;
        if (u.n > 0) {
          for (int i = 0; i < 2 * u.n && ok; ++i) {
            const bool is_v = i == 2 * u.n - 1 || (i > 0 && (i & 1) == 0);
            const int j = i == 2 * u.n - 1 ? u.n - 1 : i / 2 - 1;
            const uint32_t use = base + i, slot = use % C::kSlots;
            ok = mbar_wait(bar(slot), (use / C::kSlots) & 1, abort_s);
            ok = __all_sync(0xffffffffu, (int)ok) != 0;
            if (!ok) break;
            const int c = is_v ? u.tile(u.k0 + j) * kKeys : 0;
            if (is_v && partial(u, c)) {
              uint4* v = reinterpret_cast<uint4*>(smem + C::kTiles * C::kQBytes + slot * C::kSlotBytes);
              bool found = false;
              constexpr int kAll = C::kSlotBytes / 16, kEach = kAll / 64, kBatch = 8;
#pragma unroll 1
              for (int r = 0; r < kEach; r += kBatch) {
                uint4 w[kBatch];
#pragma unroll
                for (int b = 0; b < kBatch; ++b) w[b] = v[(r + b) * 64 + part * 32 + lane];
#pragma unroll
                for (int b = 0; b < kBatch; ++b) {
                  const int at = (r + b) * 64 + part * 32 + lane, token = c + (at / 8) % kKeys;
                  const bool seen = token < end && (token >= u.from || token < a.sink);
                  uint4 mask;
                  mask.x = not_finite2<kF16>(w[b].x);
                  mask.y = not_finite2<kF16>(w[b].y);
                  mask.z = not_finite2<kF16>(w[b].z);
                  mask.w = not_finite2<kF16>(w[b].w);
                  const bool odd = (mask.x | mask.y | mask.z | mask.w) != 0;
                  if (!seen || odd) {
                    found = found || seen;
                    v[at] = seen ? make_uint4(w[b].x & ~mask.x, w[b].y & ~mask.y, w[b].z & ~mask.z, w[b].w & ~mask.w)
                                 : make_uint4(0, 0, 0, 0);
                  }
                }
              }
              if (found) *reinterpret_cast<volatile int*>(&work[e].poison) = 1;
              fence_async_shared();
            }
            __syncwarp();
            if (lane == 0) {  // for every use, so that no phase is left out
              mbar_arrive(bar(kClean + slot));
              mbar_arrive(bar(kEmpty + slot));
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kWEmpty + e));
        if (u.n == 0) break;
        base += 2 * u.n;
      }
    }
  } else {
    // -------------------------------------------------------------------------------- softmax, one row a thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int stream = warp >> 2, r = tid & 127, wg = stream;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    const uint32_t col_s = lanes + C::kColS + stream * C::kStepS, col_o = lanes + C::kColO + stream * C::kStepO;
    const int token_in = r / a.group, head_in = r - token_in * a.group;
    const bool in_tile = token_in < a.tile_tokens;
    const float scale2 = a.premultiply ? 1.0f : a.scale2;
    uint32_t tiles_done = 0, units_done = 0;
    for (int piece = 0;; ++piece) {
      const int e = piece & 1;
      bool got = mbar_wait(bar(kWFull + e), (piece >> 1) & 1, abort_s);
      // all warps go on or none does: they meet at barriers (after a wait has run out, waits return at once)
      if (!named_all(1, 256, got)) break;
      const Work* u = work + e;
      const int n = u->n, k0 = u->k0;
      if (n == 0) break;
      if (C::kTiles == 1 && stream == 1) {  // one row tile: the second warpgroup has nothing to do
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kWEmpty + e));
        continue;
      }
      const bool pair = u->pair;
      const int token = token_in + (pair ? 0 : stream * a.tile_tokens);  // of the unit
      const bool valid = in_tile && token < u->tokens;
      View view;
      view.length = u->length;
      {
        int position = u->length + u->tok0 + token;
        if (a.parents) {
          // the sequence's nodes up to the unit's end, then a walk up from the row's own
          const int nodes = u->nodes;
          int8_t* up = up_s + wg * kMaxNodes;
          const int me_in = tid & 127;
          if (me_in < nodes) {
            const int p = __ldg(a.parents + u->seq_row0 + me_in);
            const bool fine = p >= -1 && p < me_in;
            if (!fine && a.status) atomicMax(a.status, 1);
            up[me_in] = (int8_t)(fine ? p : -1);
          }
          named_sync(2 + wg, 128);
          const int own = u->tok0 + token;
          int depth = 0;
#pragma unroll
          for (int i = 0; i < kMaxNodes / 32; ++i) view.node[i] = 0;
          if (valid) {
            for (int i = up[own]; i >= 0; i = up[i]) ++depth;
            position = u->length + depth;
            int at = position;
            for (int i = own; i >= 0; i = up[i], --at) {
              const bool seen = a.window == 0 || at > position - a.reach || at < a.sink;
#pragma unroll
              for (int k = 0; k < kMaxNodes / 32; ++k) view.node[k] |= seen && (i >> 5) == k ? 1u << (i & 31) : 0u;
            }
          }
          named_sync(2 + wg, 128);
          view.hi = u->length;
        } else {
          view.hi = position + 1;
        }
        view.lo = a.window == 0 ? 0 : max(0, position - a.reach + 1);
        view.sink = a.window == 0 ? 0 : min(a.sink, view.hi);
      }
      float m = -INFINITY, l = 0.0f;  // m: what exponents are taken from (log2 units), at most 8 below the maximum
      const int step = pair ? 2 : 1, mine = pair ? (n - stream + 1) / 2 : n;
      for (int i = 0; i < mine; ++i) {
        const int c = u->tile(k0 + (pair ? stream + step * i : i)) * kKeys;
        (void)mbar_wait(bar(kSFull + stream), tiles_done & 1, abort_s);
        ++tiles_done;
        __syncwarp();
        tc::fence_after();
        uint32_t raw[kKeys / 32][32];
#pragma unroll
        for (int k = 0; k < kKeys / 32; ++k) tc::ld32(raw[k], col_s + 32 * k);
        tc::wait_ld();
        float s[kKeys];
#pragma unroll
        for (int k = 0; k < kKeys; ++k) s[k] = __uint_as_float(raw[k / 32][k % 32]);
        if (a.premultiply) {
          if (a.softcap > 0.0f) {
#pragma unroll
            for (int k = 0; k < kKeys; ++k) s[k] = a.softcap * kLog2e * tanh_of(s[k] * a.cap_in);
          } else {
#pragma unroll
            for (int k = 0; k < kKeys; ++k) s[k] *= a.scale2;
          }
        }
        if (partial(*u, c)) {
#pragma unroll
          for (int k = 0; k < kKeys / 32; ++k) {
            const uint32_t w = a.parents ? view.bits<true>(c + 32 * k) : view.bits<false>(c + 32 * k);
#pragma unroll
            for (int b = 0; b < 32; ++b) s[32 * k + b] = w >> b & 1u ? s[32 * k + b] : -INFINITY;
          }
        }
        float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int k = 4; k < kKeys; k += 4) {
          top[0] = fmaxf(top[0], s[k]);
          top[1] = fmaxf(top[1], s[k + 1]);
          top[2] = fmaxf(top[2], s[k + 2]);
          top[3] = fmaxf(top[3], s[k + 3]);
        }
        // Weights are up to 2^7 in f16 (and, with the eight below, 2^15): under 2^-14 a 16-bit weight would be subnormal.
        const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale2 - (kF16 ? 7.0f : 0.0f);
        // O keeps its scale while maxima go up by less than 2^8: l and O stay exact multiples, far from overflow
        const bool higher = high > m + 8.0f || (m == -INFINITY && high > m);
        if (__any_sync(0xffffffffu, higher)) {
          const float now = fmaxf(m, high);
          const float turn = now == -INFINITY ? 1.0f : ex2_ftz(m - now);
          m = now;
          l *= turn;
          if (i > 0) {
#pragma unroll 1
            for (int d = 0; d < D; d += 32) {
              uint32_t o[32];
              tc::ld32(o, col_o + d);
              tc::wait_ld();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * turn);
              tc::st32(col_o + d, o);
            }
            tc::wait_st();
          }
        }
        const float minus = m == -INFINITY ? 0.0f : -m;  // a row that has seen nothing keeps weights of exp2(-inf) = 0
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < kKeys / 64; ++k) {
          uint32_t p[32];
#pragma unroll
          for (int b = 0; b < 32; ++b) {
            const float e0 = ex2_ftz(fmaf(s[64 * k + 2 * b], scale2, minus));
            const float e1 = ex2_ftz(fmaf(s[64 * k + 2 * b + 1], scale2, minus));
            part[b & 1] += e0;
            part[2 + (b & 1)] += e1;
            p[b] = pack2<kF16>(e0, e1);
          }
          tc::st32(col_s + 32 * k, p);
        }
        l += (part[0] + part[1]) + (part[2] + part[3]);
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kPReady + stream));
      }

      // ------------------------------------------------------------------------------ the unit's rows
      (void)mbar_wait(bar(kOFull + stream), units_done & 1, abort_s);
      ++units_done;
      __syncwarp();
      tc::fence_after();
      const bool poison = *reinterpret_cast<volatile const int*>(&u->poison) != 0;
      // Values that were taken out of tiles come back, to the rows that see them (32 dims from d on of this row): rare,
      // and one by one.
      auto put_back = [&](uint32_t (&o)[32], int d) {
        for (int i = 0; i < n; ++i) {
          const int c = u->tile(k0 + i) * kKeys;
          if (!partial(*u, c)) continue;
          for (int k = 0; k < kKeys; k += 32) {
            uint32_t w = valid ? (a.parents ? view.bits<true>(c + k) : view.bits<false>(c + k)) : 0u;
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
      bool second = false;  // this thread's row has a part in the other warpgroup's accumulator
      if (pair) {
        if (stream == 1) {
          pair_s[r] = m;
          pair_s[kRowsTile + r] = l;
        }
        tc::fence_before();
        named_sync(1, 256);
        tc::fence_after();
        if (stream == 0) {
          const float m1 = pair_s[r], l1 = pair_s[kRowsTile + r];
          second = n > 1;
          const float now = fmaxf(m, m1);
          f0 = now == -INFINITY ? 1.0f : ex2_ftz(m - now);
          f1 = now == -INFINITY ? 1.0f : ex2_ftz(m1 - now);
          l = second ? l * f0 + l1 * f1 : l;
          if (!second) f0 = 1.0f;
          else m = now;
        }
      }
      if (!pair || stream == 0) {
        const int row_in = (pair ? 0 : stream * kRowsTile) + r;
        const long long row = u->row0 + token, at_head = row * a.n_heads + (long long)u->head * a.group + head_in;
        const float inverse = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // nothing seen: zeros
        const long long n_slots = 2ll * gridDim.x;
        if (u->cut && valid) {
          float* rm = a.records + n_slots * C::kRows * D + (long long)u->slot * C::kRows + row_in;
          rm[0] = m;
          rm[n_slots * C::kRows] = l;
        } else if (a.lse && valid) {  // not cut
          a.lse[at_head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
        }
#pragma unroll 1
        for (int d = 0; d < D; d += 32) {
          uint32_t o[32];
          tc::ld32(o, col_o + d);
          if (second) {
            uint32_t o1[32];
            tc::ld32(o1, lanes + C::kColO + C::kStepO + d);
            tc::wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k)
              o[k] = __float_as_uint(__uint_as_float(o[k]) * f0 + __uint_as_float(o1[k]) * f1);
          } else {
            tc::wait_ld();
          }
          if (poison) put_back(o, d);
          if (u->cut) {
            if (!valid) continue;
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
        }
        tc::fence_before();
      }
      if (pair) named_sync(1, 256);  // the second accumulator and its sums have been read
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kWEmpty + e));
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 9) tc::dealloc512(tmem);
  // a wait that ran into its limit (about two seconds): the outputs are not valid
  if (tid == 0 && *abort_s && a.status) atomicMax(a.status, 2);
}

// The records of a cut unit become its rows: thread by thread a row's four dims, rows side by side, so that loads and
// the records' layout agree.  blockIdx.x: the CTA that has the unit's first piece; blockIdx.y takes a part of the rows and dims.
constexpr int kJoinParts = 8;
template <class C>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Args a) {
  constexpr int D = C::D;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Desc u = a.desc[blockIdx.x];
  if (u.pieces == 0) return;
  const long long n_slots = 2ll * gridDim.x;
  const float4* o = reinterpret_cast<const float4*>(a.records);
  const float* rm = a.records + n_slots * C::kRows * D;
  const float* rl = rm + n_slots * C::kRows;
  auto slot_of = [&](int k) { return k == 0 ? 2ll * blockIdx.x + 1 : 2ll * (blockIdx.x + k); };
  for (int i = blockIdx.y * 256 + threadIdx.x; i < C::kRows * (D / 4); i += kJoinParts * 256) {
    const int row_in = i % C::kRows, d4 = i / C::kRows, r = row_in % kRowsTile;
    const int token_in = r / a.group, token = row_in / kRowsTile * a.tile_tokens + token_in;
    if (token_in >= a.tile_tokens || token >= u.tokens) continue;
    float m = -INFINITY;
#pragma unroll 4
    for (int k = 0; k < u.pieces; ++k) m = fmaxf(m, __ldcg(rm + slot_of(k) * C::kRows + row_in));
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
#pragma unroll 4
    for (int k = 0; k < u.pieces; ++k) {
      const long long slot = slot_of(k);
      const float mk = __ldcg(rm + slot * C::kRows + row_in), lk = __ldcg(rl + slot * C::kRows + row_in);
      const float4 v = __ldcg(o + (slot * (D / 4) + d4) * C::kRows + row_in);
      const bool none = lk == 0.0f;  // nothing seen in this piece, and nothing to be taken from it
      const float f = mk == m ? 1.0f : ex2_ftz(mk - m);
      if (!none) {
        l += f * lk;
        sum.x += f * v.x;
        sum.y += f * v.y;
        sum.z += f * v.z;
        sum.w += f * v.w;
      }
    }
    const float inverse = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    if (inverse == 0.0f) sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const long long at_head = (long long)(u.row0 + token) * a.n_heads + (long long)u.head * a.group + r - token_in * a.group;
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
  a.unit_tokens = C::kTiles * a.tile_tokens;
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
  join.gridDim = dim3(workers, kJoinParts);
  join.blockDim = 256;
  join.stream = s;
  join.attrs = early;
  join.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&join, join_kernel<C>, a);
  if (e != cudaSuccess) return set_error(ASTERQ_ERR_CUDA, "rows_attention: launch failed: %s", cudaGetErrorString(e));
  return check_launch("rows_attention");
}

static int check(const asterq_rows_attention_params* p) {
  if (!p) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "rows_attention: null parameters");
  if (p->n_seqs < 0 || p->n_rows < 0 || p->n_heads <= 0 || p->n_kv_heads <= 0 || p->n_heads % p->n_kv_heads ||
      p->page_tokens <= 0 || p->max_pages < 0 || p->n_pages < 0 || p->window < 0 || p->sink < 0)
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
  a.premultiply = a.softcap > 0.0f || !(a.scale > 0.0f);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool f16 = p->dtype == ASTERQ_DTYPE_F16;
  switch (p->head_dim) {
    case 64: return f16 ? rat::launch<rat::Cfg<true, 64>>(p, a, workers, dev, s)
                        : rat::launch<rat::Cfg<false, 64>>(p, a, workers, dev, s);
    case 128: return f16 ? rat::launch<rat::Cfg<true, 128>>(p, a, workers, dev, s)
                         : rat::launch<rat::Cfg<false, 128>>(p, a, workers, dev, s);
    default: return f16 ? rat::launch<rat::Cfg<true, 256>>(p, a, workers, dev, s)
                        : rat::launch<rat::Cfg<false, 256>>(p, a, workers, dev, s);
  }
}
