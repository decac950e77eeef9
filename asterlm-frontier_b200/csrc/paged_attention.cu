// Attention of one new token a sequence over a paged grouped-query cache (sm_100a).
//
//   out[b, h] = sum_t softmax_t(score) v_t,  score = scale q[b, h] . k_t, softcapped where asked,
//   over the visible tokens t < L and (t < sink or t >= L - (window - sink)),
//   with L = lengths[b] + n_new; lse[b, h] = log sum_t exp(score).
//
// What bounds it: the visible keys and values are read once (4 Hkv D bytes a token) for 4 H D
// operations, so H / Hkv operations a byte: memory.  Everything below serves keeping bytes in
// flight: one persistent CTA per SM, a producer warp that streams 64-token tiles of keys and values
// into a ring of shared memory by TMA, across the borders of its work, and consumer warps that never
// wait for one another inside a sequence.
//
// Split.  The tiles of all (sequence, kv head, row block) units, laid end to end with a few tiles' worth
// in front of each unit for what it costs by itself, are cut into equal contiguous shares, one per CTA,
// by a prefix sum over `lengths` that every CTA computes for itself: no planning launch, no host copy of
// the lengths, and a long sequence and a ragged batch are both even to a tile.  A unit that lies in one
// share is finished there; a short one by half of the CTA's warps, while the other half has the next.  A
// cut unit leaves (o, m, l) records in the workspace, and the CTA that stores its last one joins them, in
// the order of the shares, so results do not depend on which CTA came last; of many records groups are
// joined first, each by the CTA that stores its last one.  No CTA waits for another.
//
// Measured (bf16, 128 dims, 8 kv heads, pages of 64): 64 sequences of 1k to 32k tokens 362 us, 6.6 TB/s of keys
// and values.  One sequence of 8192 tokens of 4 kv heads takes 12.8 us, of which the bytes are 2.6: launch, lengths,
// table, first tiles (5 us), the warps' join (1.2), records and their count (1.5) and the join of 37 pieces a head
// (3) are chains of latencies.  256 sequences of at most 512 visible tokens, 16 kv heads of 64, with a softcap: 93 us
// against 25 of bytes, since a unit of six tiles keeps a team's warps busy for some 1,450 cycles a tile and 1,700 more.
#include <cuda.h>

#include "asterq_internal.h"
#include "common.cuh"

namespace asterq {
namespace pat {

constexpr int kMaxWorkers = 256;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;

struct Args {
  const void* q;
  const int* page_table;
  const int* lengths;
  void* out;
  float* lse;
  float* records;  // o [2 W][NR][D], then m [2 W][NR], then l [2 W][NR]
  int* counters;   // [4 W], zero between calls: records stored of a unit or of a group, groups joined of a unit
  int* status;
  long long q_row_stride, q_head_stride, n_pages, capacity;  // capacity: tokens a row of the table can hold
  int n_rows, n_heads, n_kv_heads, group, row_blocks;
  int page_tokens, max_pages, box_rows, n_new, window, sink, out_f32;
  float scale, softcap, cap_in;  // cap_in: scale / softcap
};

// D: head dim.  NR: query rows of a block (the query heads of one kv head, in eights).
template <bool kF16_, int D_, int NR_>
struct Cfg {
  static constexpr bool kF16 = kF16_;
  static constexpr int D = D_, NR = NR_, NT = NR_ / 8;
  // Tiles of 32 KB.  A warp takes kSub times 16 tokens of a tile.  Two teams of warps take alternate tiles,
  // so one team's softmax runs beside the other's products.
  static constexpr int kTile = 8192 / D, kSub = D == 64 ? 2 : 1;
  static constexpr int kTeamWarps = kTile / 16 / kSub, kWarps = 2 * kTeamWarps, kThreads = 32 * kWarps + 32;
  static constexpr int kSubTokens = 16 * kTeamWarps;  // from one of a warp's 16 tokens to its next
  static constexpr int kHalfBytes = kTile * D * 2, kStageBytes = 2 * kHalfBytes;
  static constexpr int kStages = 6;
  // queries of the next units, rows padded against conflicts
  static constexpr int kQSlots = NR * D >= 2048 ? 2 : 4, kQPitch = D * 2 + 16;
  static constexpr int kQBytes = NR * kQPitch;
  // dims joined at a time, in two buffers taken in turn; their count is even, so a unit ends with the second
  static constexpr int kSlice = NR == 16 ? 16 : 32, kPad = kSlice + 4;
  static constexpr int kBufFloats = kWarps * NR * kPad, kMergeFloats = 2 * kBufFloats;
  static_assert(D / kSlice % 2 == 0, "the two buffers alternate across units that the same warps join");
  static_assert(kMergeFloats >= 48 * NR, "weights of the records that are joined at once");
  // kUnitCost: what a unit costs beside its tiles, in tiles.  Measured with 0, 1 and 2: 64 rows of 1 to 2048 tokens,
  // 8 kv heads of 128, 39.2, 30.1 and 27.9 us; of 1 to 512 tokens 20.3, 19.9 and 20.7; of 1k to 32k tokens 366, 364 and
  // 362; 256 rows of at most 512 visible tokens, 16 kv heads of 64, 111, 93 and 103.
  // kSoloTiles: units up to this long are taken by one team.  Measured with 0, 4 and 8: the same four 34.7, 30.1 and
  // 30.1 us; 21.0, 19.9 and 20.7; 364, 364 and 364; 108, 93 and 92.
  static constexpr int kUnitCost = 1;
  static constexpr int kSoloTiles = 4;
  static constexpr int kSmem =
      1024 + kStages * kStageBytes + kQSlots * kQBytes + (kMergeFloats + 2 * kWarps * NR) * 4 + (3 * kStages + 2 * kQSlots) * 8;
};

ASTERQ_DEVICE void tma_box(uint32_t dst, const CUtensorMap* map, int token, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %2, %4}], "
      "[%5];" ::"r"(dst),
      "l"(map), "r"(0), "r"(token), "r"(z), "r"(bar)
      : "memory");
}
// the transpose of an 8 x 8 matrix of 16-bit values held as MMA fragments
ASTERQ_DEVICE uint32_t transpose8(uint32_t x) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}

// Two 16-bit values: an infinity as the largest finite value, a NaN as any finite one.  With b positive, xorsign gives
// min(|x|, |b|) the sign of x; of a number and a NaN it takes the number.
template <bool kF16>
ASTERQ_DEVICE uint32_t finite2(uint32_t x) {
  uint32_t r;
  if constexpr (kF16) asm("min.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x7bff7bffu));
  else asm("min.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x7f7f7f7fu));
  return r;
}

// tanh x to a few 2^-23 of itself (of 1 it is not enough: under a cap far above the scores that is the scores' whole size).
// Below 0.9 Lambert's continued fraction x / (1 + x^2 / (3 + x^2 / (5 + x^2 / (7 + x^2 / 9)))) as a quotient, its error
// x^10 / 9.8e6 < 2^-24; from there on (e^2x - 1) / (e^2x + 1), the exponent held within what 2^x and the quotient take.
ASTERQ_DEVICE float tanh_of(float x) {
  const float x2 = x * x;
  const float e2x = ex2_ftz(fminf(fmaxf(x * (2.0f * kLog2e), -64.0f), 64.0f));
  const bool large = fabsf(x) >= 0.9f;  // not of a NaN
  const float num = large ? e2x - 1.0f : x * fmaf(x2, x2 + 105.0f, 945.0f);
  const float den = large ? e2x + 1.0f : fmaf(x2, fmaf(x2, 15.0f, 420.0f), 945.0f);
  return __fdividef(num, den);
}

// The visible tiles of one sequence.  Tile k of its list is tokens [kTile j, kTile (j + 1)) with
// j = k below sink_tiles and first + k - sink_tiles from there on.
struct Span {
  int length, sink, from, sink_tiles, first, tiles;
  ASTERQ_DEVICE int tile(int k) const { return k < sink_tiles ? k : first + (k - sink_tiles); }
  ASTERQ_DEVICE bool visible(int t) const { return t < length && (t < sink || t >= from); }
};
template <int kTile>
ASTERQ_DEVICE Span span_of(const Args& a, int row) {
  Span s;
  const int n = __ldg(a.lengths + row);
  long long want = n < 0 ? 0 : (long long)n + a.n_new;
  s.length = (int)min(want, a.capacity);
  s.sink = 0;
  s.from = 0;
  s.sink_tiles = 0;
  s.first = 0;
  const int last = (s.length + kTile - 1) / kTile;
  if (a.window > 0 && s.length > a.window) {
    s.sink = min(a.sink, a.window);
    s.from = s.length - (a.window - s.sink);
    s.sink_tiles = (s.sink + kTile - 1) / kTile;
    s.first = s.from >= s.length ? last : max(s.from / kTile, s.sink_tiles);
  }
  s.tiles = s.sink_tiles + max(0, last - s.first);
  return s;
}

// One CTA's share [x, end) of all units' costs, walked piece by piece; every warp walks it for itself.
template <int kTile, int kUnitCost>
struct Walk {
  long long x, end, unit_start;  // unit_start: of the unit that x is in, or has just passed
  int row;
  Span span;
  // of the current piece
  int unit, k0, n;        // unit within the row, its first tile here, tiles here
  long long first_tile;   // where the unit's first tile is
  template <class A>
  ASTERQ_DEVICE void start(const A& a, int at_row, long long row_start) {
    row = at_row;
    span = span_of<kTile>(a, row);
    unit = (int)((x - row_start) / (span.tiles + kUnitCost));
    unit_start = row_start + (long long)unit * (span.tiles + kUnitCost);
  }
  template <class A>
  ASTERQ_DEVICE bool next(const A& a, int units_per_row) {
    while (x < end) {
      int per_unit = span.tiles + kUnitCost;
      if (x >= unit_start + per_unit) {
        unit_start += per_unit;
        if (++unit == units_per_row) {
          unit = 0;
          do span = span_of<kTile>(a, ++row);
          while (span.tiles == 0);
          per_unit = span.tiles + kUnitCost;
        }
      }
      const int at = (int)(x - unit_start), cost = (int)min((long long)(per_unit - at), end - x);
      first_tile = unit_start + kUnitCost;
      k0 = max(at - kUnitCost, 0);
      n = max(at + cost - kUnitCost, 0) - k0;
      x += cost;
      if (n > 0) return true;
    }
    return false;
  }
};

struct Start {
  long long row_start, total;
  int row;
};

template <class C>
__global__ void __launch_bounds__(C::kThreads, 1)
    attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                     const __grid_constant__ Args a) {
  constexpr int D = C::D, NR = C::NR, NT = C::NT, kTile = C::kTile;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t q_ring = smem_u32(smem) + C::kStages * C::kStageBytes;
  float* merge = reinterpret_cast<float*>(smem + C::kStages * C::kStageBytes + C::kQSlots * C::kQBytes);
  float* warp_m = merge + C::kMergeFloats;
  float* warp_l = warp_m + C::kWarps * NR;
  uint64_t* bars = reinterpret_cast<uint64_t*>(warp_l + C::kWarps * NR);
  __shared__ Start start_s;
  __shared__ long long scan_s[32];
  __shared__ int abort_s, never_s, last_s;  // never_s stays 0: for waits that an abort must not cut short
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // a full barrier for each stage and the team that its tile is for: a barrier's waiters see each of its phases
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 16 * C::kStages, q_full0 = empty0 + 8 * C::kStages,
                 q_empty0 = q_full0 + 8 * C::kQSlots;
  const int units_per_row = a.n_kv_heads * a.row_blocks;

  if (tid == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(full0 + 16 * i, 1);
      mbar_init(full0 + 16 * i + 8, 1);
      mbar_init(empty0 + 8 * i, C::kTeamWarps);
    }
    for (int i = 0; i < C::kQSlots; ++i) {
      mbar_init(q_full0 + 8 * i, 1);
      mbar_init(q_empty0 + 8 * i, C::kWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    abort_s = never_s = 0;
  }

  // The share: thread t sums the costs of rows [t R, (t + 1) R), the block scans the sums.
  const int strip = (a.n_rows + C::kThreads - 1) / C::kThreads;
  const int r0 = min(tid * strip, a.n_rows), r1 = min(r0 + strip, a.n_rows);
  long long sum = 0;
  auto cost_of = [&](int row) {
    const int tiles = span_of<kTile>(a, row).tiles;
    return tiles > 0 ? (long long)(tiles + C::kUnitCost) * units_per_row : 0ll;
  };
  for (int r = r0; r < r1; ++r) sum += cost_of(r);
  long long scan = sum;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long up = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += up;
  }
  if (lane == 31) scan_s[warp] = scan;
  __syncthreads();
  long long before = scan - sum, total = 0;
  for (int w = 0; w <= C::kWarps; ++w) {
    if (w < warp) before += scan_s[w];
    total += scan_s[w];
  }
  const int W = (int)min((long long)gridDim.x, max(total, 1ll)), me = blockIdx.x;
  Walk<kTile, C::kUnitCost> walk;
  walk.x = total * me / W;
  walk.end = me < W ? total * (me + 1) / W : walk.x;
  if (walk.x < walk.end && before <= walk.x && walk.x < before + sum) {
    Start s;
    s.row = r0;
    s.row_start = before;
    while (true) {
      const long long here = cost_of(s.row);
      if (walk.x < s.row_start + here) break;
      s.row_start += here;
      ++s.row;
    }
    start_s = s;
  }
  // rows that see nothing: zeros, and a log-sum of -inf
  for (int r = me; r < a.n_rows; r += gridDim.x) {
    if (span_of<kTile>(a, r).tiles > 0) continue;
    for (int i = tid; i < a.n_heads * D; i += C::kThreads) {
      const long long at = (long long)r * a.n_heads * D + i;
      if (a.out_f32) static_cast<float*>(a.out)[at] = 0.0f;
      else static_cast<uint16_t*>(a.out)[at] = 0;
    }
    if (a.lse)
      for (int i = tid; i < a.n_heads; i += C::kThreads) a.lse[(long long)r * a.n_heads + i] = -INFINITY;
  }
  __syncthreads();
  if (walk.x >= walk.end) return;
  const long long my_start = walk.x;
  walk.start(a, start_s.row, start_s.row_start);

  if (warp == C::kWarps) {
    // ------------------------------------------------------------------ producer
    // A tile comes in boxes of box_rows tokens (a divisor of the page and of the tile), one lane a box of keys
    // or values: it looks its page up and issues its copy.
    const int box = lane / 2, is_v = lane & 1;
    const CUtensorMap* map = is_v ? &v_map : &k_map;
    const uint32_t box_bytes = a.box_rows * D * 2;
    const uint32_t box_at = is_v * C::kHalfBytes + box * box_bytes;
    // Lookups run ahead of the copies, by a tile within a unit and by a unit's first tile across units: this
    // warp by itself has to stay below the time that a tile takes to arrive.
    struct Piece {
      int k0, n, row, head, block, solo;
      Span span;
      int token, column, offset, page;  // this lane's box of the next tile: its page's place in the table, and id
      bool use;
    };
    auto look_up = [&](Piece& p, bool same_page) {
      p.use = box * a.box_rows < kTile && p.token < p.span.length &&
              (p.token < p.span.sink || p.token + a.box_rows > p.span.from);
      if (p.use && !same_page) p.page = __ldg(a.page_table + (long long)p.row * a.max_pages + p.column);
    };
    auto place = [&](Piece& p, int k) {
      p.token = p.span.tile(k) * kTile + box * a.box_rows;
      p.column = p.token / a.page_tokens;
      p.offset = p.token - p.column * a.page_tokens;
      p.page = 0;
      look_up(p, false);
    };
    auto next_piece = [&](Piece& p) {
      if (!walk.next(a, units_per_row)) return false;
      p.k0 = walk.k0;
      p.n = walk.n;
      p.row = walk.row;
      p.head = walk.unit / a.row_blocks;
      p.block = walk.unit - p.head * a.row_blocks;
      p.span = walk.span;
      p.solo = walk.n == walk.span.tiles && walk.n <= C::kSoloTiles;
      place(p, p.k0);
      return true;
    };
    uint32_t used[2] = {0, 0};  // uses of each stage by each team, modulo 2
    bool ok = true;
    int stage = 0, round = 0, piece = 0;
    Piece p, ahead;
    bool more = next_piece(ahead);
    for (; ok && more; ++piece) {
      p = ahead;
      more = next_piece(ahead);
      const int q_slot = piece % C::kQSlots, rows = min(NR, a.group - p.block * NR);
      if (piece >= C::kQSlots) {
        ok = __all_sync(0xffffffffu, (int)mbar_wait(q_empty0 + 8 * q_slot, ((piece / C::kQSlots) - 1) & 1, &abort_s)) != 0;
        if (!ok) break;
      }
      if (lane == 0) mbar_expect_tx(q_full0 + 8 * q_slot, rows * D * 2);
      __syncwarp();
      if (lane < rows)
        bulk_1d(q_ring + q_slot * C::kQBytes + lane * C::kQPitch,
                static_cast<const uint16_t*>(a.q) + p.row * a.q_row_stride +
                    ((long long)p.head * a.group + p.block * NR + lane) * a.q_head_stride,
                D * 2, q_full0 + 8 * q_slot);
      for (int j = 0; j < p.n; ++j) {
        const int team = (p.solo ? piece : j) & 1;
        int page = p.page;
        const int offset = p.offset;
        const bool use = p.use;
        if (j + 1 < p.n) {
          if (p.k0 + j + 1 == p.span.sink_tiles) {
            place(p, p.k0 + j + 1);
          } else {
            const int column = p.column;
            const bool had = p.use;
            p.token += kTile;
            for (p.offset += kTile; p.offset >= a.page_tokens; p.offset -= a.page_tokens) ++p.column;
            look_up(p, had && p.column == column);
          }
        }
        if (round > 0) {
          ok = __all_sync(0xffffffffu, (int)mbar_wait(empty0 + 8 * stage, (round - 1) & 1, &abort_s)) != 0;
          if (!ok) break;
        }
        const uint32_t bar = full0 + 16 * stage + 8 * team;
        const uint32_t wanted = __ballot_sync(0xffffffffu, use);
        if (lane == 0) mbar_expect_tx(bar, __popc(wanted) * box_bytes);
        __syncwarp();
        if (use) {
          if (page < 0 || page >= a.n_pages) {
            if (a.status) atomicMax(a.status, 1);
            page = 0;
          }
          tma_box(smem_u32(smem) + stage * C::kStageBytes + box_at, map, offset, page * a.n_kv_heads + p.head, bar);
        }
        used[0] ^= (uint32_t)(team == 0) << stage;
        used[1] ^= (uint32_t)team << stage;
        if (++stage == C::kStages) {
          stage = 0;
          ++round;
        }
      }
    }
    // the last copies have landed before the exit, also when a wait ran out and nobody waits for them
    if (!ok) {
      for (int i = 0; i < 2 * C::kStages; ++i)
        (void)mbar_wait(full0 + 8 * i, (used[i & 1] >> (i / 2) & 1) ^ 1, &never_s, 200000000);
      for (int i = max(0, piece - C::kQSlots); i <= piece; ++i)
        (void)mbar_wait(q_full0 + 8 * (i % C::kQSlots), (i / C::kQSlots) & 1, &never_s, 200000000);
    }
    return;
  }

  // -------------------------------------------------------------------- consumers
  // Scores are computed transposed, S^T = K Q^T with tokens as the MMA's 16 rows and query heads as
  // its 8 columns, so a group of 8 heads or fewer wastes nothing; then O^T += V^T P^T with dims as
  // rows.  Each warp keeps its own running maximum and sum over the tokens it saw; the warps join
  // once a unit.
  const int team = warp / C::kTeamWarps, g = lane >> 2, qd = lane & 3;
  const int row16 = (warp % C::kTeamWarps) * 16;
  const int k_row = row16 + (lane & 15), k_chunk = lane >> 4;
  const int v_row = row16 + (lane & 7) + ((lane >> 4) << 3), v_chunk = (lane >> 3) & 1;
  // a box's rows of 64 dims, then the same rows of the next 64
  const uint32_t col_bytes = a.box_rows * 128;
  uint32_t k_at[C::kSub], v_at[C::kSub];
#pragma unroll
  for (int u = 0; u < C::kSub; ++u) {
    const int k = k_row + u * C::kSubTokens, v = v_row + u * C::kSubTokens;
    k_at[u] = k / a.box_rows * (a.box_rows * D * 2) + k % a.box_rows * 128;
    v_at[u] = v / a.box_rows * (a.box_rows * D * 2) + v % a.box_rows * 128;
  }
  const float scale2 = a.scale * kLog2e;
  const long long n_slots = 2ll * gridDim.x;
  int it = 0;
  uint32_t phase = 0;  // of each stage's barrier of this team
  bool all_joined = false;  // the unit before was joined by all warps
  for (int piece = 0; walk.next(a, units_per_row); ++piece) {
    const int head = walk.unit / a.row_blocks, block = walk.unit - head * a.row_blocks;
    const int rows = min(NR, a.group - block * NR);
    const long long h0 = (long long)head * a.group + block * NR;  // query head of the block's row 0
    const bool cut = walk.n < walk.span.tiles, solo = !cut && walk.n <= C::kSoloTiles;
    const int q_slot = piece % C::kQSlots;
    // All warps' join ends with reads of one another's sums that nothing orders.  The first barrier of another such
    // join does, a team's own does not: its second slice would overwrite what the other team may still read.
    if (solo && all_joined) named_sync(3, 32 * C::kWarps);
    all_joined = !solo;
    // Every warp follows the queries of every unit, so that none falls a phase behind.  (After a wait has run
    // out all go on to the end, waits returning at once, since they still meet at barriers.)
    (void)mbar_wait(q_full0 + 8 * q_slot, (piece / C::kQSlots) & 1, &abort_s);
    __syncwarp();
    if (solo && (piece & 1) != team) {
      it += walk.n;
      if (lane == 0) mbar_arrive(q_empty0 + 8 * q_slot);
      continue;
    }
    uint32_t qf[D / 16][NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int s = 0; s < D / 16; s += 2) {
        uint32_t f[4];
        ldmatrix_x4(f, q_ring + q_slot * C::kQBytes + (t * 8 + (lane & 7)) * C::kQPitch + s * 32 + (lane >> 3) * 16);
        qf[s][t][0] = f[0];
        qf[s][t][1] = f[1];
        qf[s + 1][t][0] = f[2];
        qf[s + 1][t][1] = f[3];
      }
    __syncwarp();
    if (lane == 0) mbar_arrive(q_empty0 + 8 * q_slot);
    float acc[D / 16][NT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][t][e] = 0.0f;
    }

    for (int j = 0; j < walk.n; ++j, ++it) {
      if (!solo && (j & 1) != team) continue;
      const int stage = it % C::kStages;
      const uint32_t k_base = smem_u32(smem) + stage * C::kStageBytes, v_base = k_base + C::kHalfBytes;
      if (!__all_sync(0xffffffffu, (int)mbar_wait(full0 + 16 * stage + 8 * team, phase >> stage & 1, &abort_s))) break;
      phase ^= 1u << stage;
      const int token0 = walk.span.tile(walk.k0 + j) * kTile + row16;
      // all of the warp's tokens are seen / some are
      bool whole = true, any = false;
#pragma unroll
      for (int u = 0; u < C::kSub; ++u) {
        const int first = token0 + u * C::kSubTokens, last = first + 15;
        whole = whole && last < walk.span.length && (first >= walk.span.from || last < walk.span.sink);
        any = any || (first < walk.span.length && (first < walk.span.sink || last >= walk.span.from));
      }
      if (any) {
        float sc[C::kSub][NT][4];
#pragma unroll
        for (int u = 0; u < C::kSub; ++u)
#pragma unroll
          for (int t = 0; t < NT; ++t) sc[u][t][0] = sc[u][t][1] = sc[u][t][2] = sc[u][t][3] = 0.0f;
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
#pragma unroll
          for (int u = 0; u < C::kSub; ++u) {
            uint32_t f[4];
            ldmatrix_x4(f, k_base + k_at[u] + (s / 4) * col_bytes + ((((s % 4) * 2 + k_chunk) ^ (k_row & 7)) << 4));
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              if constexpr (C::kF16) mma_f16(sc[u][t], f, qf[s][t][0], qf[s][t][1]);
              else mma_bf16(sc[u][t], f, qf[s][t][0], qf[s][t][1]);
            }
          }
        // this thread's tokens: g and g + 8 of each 16; its query rows: 8 t + 2 qd + {0, 1}
        bool see[C::kSub][2];
#pragma unroll
        for (int u = 0; u < C::kSub; ++u) {
          see[u][0] = whole || walk.span.visible(token0 + u * C::kSubTokens + g);
          see[u][1] = whole || walk.span.visible(token0 + u * C::kSubTokens + g + 8);
        }
        uint32_t ph[C::kSub][NT][2], pl[C::kSub][NT][2];
        float hi[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          hi[t][0] = hi[t][1] = -INFINITY;
#pragma unroll
          for (int u = 0; u < C::kSub; ++u) {
            if (a.softcap > 0.0f) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                sc[u][t][e] = a.softcap * kLog2e * tanh_of(sc[u][t][e] * a.cap_in);
              }
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) sc[u][t][e] *= scale2;
            }
            if (!see[u][0]) sc[u][t][0] = sc[u][t][1] = -INFINITY;
            if (!see[u][1]) sc[u][t][2] = sc[u][t][3] = -INFINITY;
            hi[t][0] = fmaxf(hi[t][0], fmaxf(sc[u][t][0], sc[u][t][2]));
            hi[t][1] = fmaxf(hi[t][1], fmaxf(sc[u][t][1], sc[u][t][3]));
          }
        }
#pragma unroll
        for (int d = 4; d < 32; d *= 2)
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            hi[t][0] = fmaxf(hi[t][0], __shfl_xor_sync(0xffffffffu, hi[t][0], d));
            hi[t][1] = fmaxf(hi[t][1], __shfl_xor_sync(0xffffffffu, hi[t][1], d));
          }
        if constexpr (C::kF16) {
          // Weights are up to 2^15 and not 1: below 2^-14 a 16-bit part of them would be subnormal, and of many small
          // weights beside a large one (a sink's, say) little was left, up to all of an eighth of them.
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            hi[t][0] -= 15.0f;
            hi[t][1] -= 15.0f;
          }
        }
        bool higher = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) higher = higher || hi[t][0] > m[t][0] || hi[t][1] > m[t][1];
        if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            float turn[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float now = fmaxf(m[t][e], hi[t][e]);
              turn[e] = now == -INFINITY ? 1.0f : ex2_ftz(m[t][e] - now);
              m[t][e] = now;
              l[t][e] *= turn[e];
            }
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              acc[i][t][0] *= turn[0];
              acc[i][t][1] *= turn[1];
              acc[i][t][2] *= turn[0];
              acc[i][t][3] *= turn[1];
            }
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          // a row whose scores so far are all -inf keeps weights exp2(-inf - 0) = 0
          const float m0 = m[t][0] == -INFINITY ? 0.0f : m[t][0], m1 = m[t][1] == -INFINITY ? 0.0f : m[t][1];
#pragma unroll
          for (int u = 0; u < C::kSub; ++u) {
            const float p0 = see[u][0] ? ex2_ftz(sc[u][t][0] - m0) : 0.0f, p1 = see[u][0] ? ex2_ftz(sc[u][t][1] - m1) : 0.0f;
            const float p2 = see[u][1] ? ex2_ftz(sc[u][t][2] - m0) : 0.0f, p3 = see[u][1] ? ex2_ftz(sc[u][t][3] - m1) : 0.0f;
            l[t][0] += p0 + p2;
            l[t][1] += p1 + p3;
            // The weights go to the second product as two 16-bit parts: one rounding would cost the output as
            // much as its own type does, and the second product's time is hidden behind the loads.
            uint32_t h01, h23;
            float2 b01, b23;
            if constexpr (C::kF16) {
              h01 = pack_half2(p0, p1), h23 = pack_half2(p2, p3);
              b01 = unpack_half2(h01), b23 = unpack_half2(h23);
              pl[u][t][0] = transpose8(pack_half2(p0 - b01.x, p1 - b01.y));
              pl[u][t][1] = transpose8(pack_half2(p2 - b23.x, p3 - b23.y));
            } else {
              h01 = pack_bf162(p0, p1), h23 = pack_bf162(p2, p3);
              b01 = unpack_bf162(h01), b23 = unpack_bf162(h23);
              pl[u][t][0] = transpose8(pack_bf162(p0 - b01.x, p1 - b01.y));
              pl[u][t][1] = transpose8(pack_bf162(p2 - b23.x, p3 - b23.y));
            }
            ph[u][t][0] = transpose8(h01);
            ph[u][t][1] = transpose8(h23);
          }
        }
        // In a tile with tokens that are not seen, their values are cleared as well: 0 times an
        // infinity or NaN that a page happens to hold past a sequence's end is not 0.
        uint32_t keep[C::kSub][2];
#pragma unroll
        for (int u = 0; u < C::kSub; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = token0 + u * C::kSubTokens + 2 * qd + 8 * h;
            keep[u][h] = whole ? 0xffffffffu
                               : (walk.span.visible(at) ? 0xffffu : 0u) | (walk.span.visible(at + 1) ? 0xffff0000u : 0u);
          }
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int u = 0; u < C::kSub; ++u) {
            uint32_t f[4];
            ldmatrix_x4_trans(f, v_base + v_at[u] + (i / 4) * col_bytes + ((((i % 4) * 2 + v_chunk) ^ (v_row & 7)) << 4));
            if (!whole) {
              f[0] &= keep[u][0];
              f[1] &= keep[u][0];
              f[2] &= keep[u][1];
              f[3] &= keep[u][1];
            }
            // The weights' smaller parts are zero or negative at times: an infinity times them is not what the
            // formula has, and the larger parts bring it in.
            uint32_t fl[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) fl[e] = finite2<C::kF16>(f[e]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              if constexpr (C::kF16) {
                mma_f16(acc[i][t], f, ph[u][t][0], ph[u][t][1]);
                mma_f16(acc[i][t], fl, pl[u][t][0], pl[u][t][1]);
              } else {
                mma_bf16(acc[i][t], f, ph[u][t][0], ph[u][t][1]);
                mma_bf16(acc[i][t], fl, pl[u][t][0], pl[u][t][1]);
              }
            }
          }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty0 + 8 * stage);
    }

    // ------------------------------------------------------------------ the warps join
    // What the joins compute from these must not be kept in registers over the loop above, which has none to
    // spare: the compiler is not told that they are still the same.
    int tid_j = tid;
    float *merge_j = merge, *records = a.records;
    asm volatile("" : "+r"(tid_j), "+l"(merge_j), "+l"(records));
    const int lane_j = tid_j & 31, warp_j = tid_j >> 5;
    float *m_j = merge_j + C::kMergeFloats, *l_j = m_j + C::kWarps * NR;
    // the team's, or all; either way with barriers that only they use
    const int wa = solo ? team * C::kTeamWarps : 0, wn = solo ? C::kTeamWarps : C::kWarps;
    const int me_in = tid_j - wa * 32, threads = wn * 32;
    auto sync = [&]() { named_sync(solo ? 1 + team : 3, threads); };
    // slot of this piece: a share's first piece may be the tail or middle of a unit, its last the head
    const long long slot = 2ll * me + (walk.first_tile > my_start ? 1 : 0);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d *= 2) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], d);
        if ((lane_j >> 2) == 0) {
          m_j[warp_j * NR + t * 8 + 2 * (lane_j & 3) + e] = m[t][e];
          l_j[warp_j * NR + t * 8 + 2 * (lane_j & 3) + e] = l[t][e];
        }
      }
    // Each thread sums the same rows of every slice, so the warps' factors are looked up once, behind the
    // first barrier; with the second slice's barrier passed nobody reads m_j and l_j any more.
    constexpr int kOwn = NR * C::kSlice / (C::kTeamWarps * 32);  // of a team; half as many with all warps
    float factor[kOwn][C::kWarps], inverse[kOwn];
#pragma unroll
    for (int part = 0; part < D / C::kSlice; ++part) {
      float* buf = merge_j + (part & 1) * C::kBufFloats;
#pragma unroll
      for (int i = 0; i < C::kSlice / 16; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            buf[(warp_j * NR + t * 8 + 2 * (lane_j & 3) + (e & 1)) * C::kPad + i * 16 + (lane_j >> 2) + (e >> 1) * 8] =
                acc[part * (C::kSlice / 16) + i][t][e];
      sync();
#pragma unroll
      for (int k = 0; k < kOwn; ++k) {
        if (!solo && k >= kOwn / 2) continue;
        const int i = me_in + k * threads, r = i / C::kSlice, d = i % C::kSlice, dim = part * C::kSlice + d;
        if (part == 0) {
          // A row's weights, by kWarps lanes of its warp: every thread for itself took 850 cycles of a
          // unit's 3,000.
          const int w = lane_j % C::kWarps;
          const float mw = w < wn ? m_j[(wa + w) * NR + r] : -INFINITY;
          const float lw = w < wn ? l_j[(wa + w) * NR + r] : 0.0f;  // not 0 although mw is -inf: NaN scores
          float top = mw;
#pragma unroll
          for (int e = 1; e < C::kWarps; e *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, e));
          const float f = mw == -INFINITY ? 0.0f : ex2_ftz(mw - top);
          float total_l = mw == -INFINITY ? lw : lw * f;
#pragma unroll
          for (int e = 1; e < C::kWarps; e *= 2) total_l += __shfl_xor_sync(0xffffffffu, total_l, e);
#pragma unroll
          for (int e = 0; e < C::kWarps; ++e) factor[k][e] = __shfl_sync(0xffffffffu, f, (lane_j & ~(C::kWarps - 1)) + e);
          if (d == 0 && r < rows) {
            if (cut) {
              records[n_slots * NR * D + slot * NR + r] = top;
              records[n_slots * NR * (D + 1) + slot * NR + r] = total_l;
            } else if (a.lse) {
              a.lse[(long long)walk.row * a.n_heads + h0 + r] = (top + log2f(total_l)) * kLn2;
            }
          }
          inverse[k] = 1.0f / total_l;
        }
        if (r >= rows) continue;
        float sum = 0.0f;
        const float* from = buf + (wa * NR + r) * C::kPad + d;
#pragma unroll
        for (int w = 0; w < C::kTeamWarps; ++w) sum = fmaf(factor[k][w], from[w * NR * C::kPad], sum);
        if (!solo) {
#pragma unroll
          for (int w = C::kTeamWarps; w < C::kWarps; ++w) sum = fmaf(factor[k][w], from[w * NR * C::kPad], sum);
        }
        if (cut) {
          records[(slot * NR + r) * D + dim] = sum;
        } else {
          const long long at = ((long long)walk.row * a.n_heads + h0 + r) * D + dim;
          const float o = sum * inverse[k];
          if (a.out_f32) static_cast<float*>(a.out)[at] = o;
          else if constexpr (C::kF16) static_cast<__half*>(a.out)[at] = __float2half_rn(o);
          else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(o);
        }
      }
    }
    if (!cut) continue;

    // ------------------------------------------------------------------ the pieces of a cut unit join
    const long long u0 = walk.first_tile, u1 = u0 + walk.span.tiles;
    const int w0 = (int)(((u0 + 1) * W - 1) / total), w1 = (int)((u1 * W - 1) / total);
    const int pieces = w1 - w0 + 1;
    const int slot0 = 2 * w0 + (u0 > total * w0 / W ? 1 : 0);  // pieces after the first are at 2 w
    auto slot_of = [&](int i) { return i == 0 ? slot0 : 2 * (w0 + i); };
    // Beyond 24 records (48 of 8 rows), groups of about their square root are joined first.  37 records of 4 rows
    // at once 12.8 us, in groups 13.8; of 8 rows 13.6 and 14.2 (one sequence of 8192 tokens, 4 kv heads of 128).
    const int size = pieces <= 24 || (pieces <= 48 && NR == 8) ? pieces : pieces <= 64 ? 8 : pieces <= 160 ? 12 : 16;
    const int groups = (pieces + size - 1) / size, group = (me - w0) / size;
    float* rec_m = records + n_slots * NR * D;
    float* rec_l = rec_m + n_slots * NR;
    // Records first, first + step, .. (n of them) become the output, or take the first one's place.  This runs once or
    // twice a launch, so what it takes is the latency of its loads (all that fit are on their way before the
    // first is needed) and of fetching its instructions: one copy of them for both levels.
    int first = group * size, n = min(size, pieces - first), step = 1;
    int* counter = a.counters + slot_of(first);
    bool whole = groups == 1;
#pragma unroll 1
    while (true) {
      sync();
      if (tid_j == 0) {
        __threadfence();
        last_s = atomicAdd(counter, 1) == n - 1;
        if (last_s) *counter = 0;
        __threadfence();
      }
      sync();
      if (!last_s) break;
      constexpr int kAhead = 16;
      auto record = [&](int k) { return slot_of(first + k * step) * NR; };
      bool weighed = false;
#pragma unroll 1
      for (int i0 = 0; i0 < rows * (D / 4); i0 += C::kWarps * 32) {
        const int i = i0 + tid_j, r = i / (D / 4), d = (i % (D / 4)) * 4;
        const bool mine = r < rows;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
        for (int k0 = 0; k0 < n; k0 += kAhead) {
          float4 v[kAhead];
#pragma unroll
          for (int k = 0; k < kAhead; ++k)
            v[k] = mine && k0 + k < n
                       ? __ldcg(reinterpret_cast<const float4*>(records + (long long)(record(k0 + k) + r) * D + d))
                       : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (!weighed) {
            weighed = true;
#pragma unroll 1
            for (int q = warp_j; q < rows; q += C::kWarps) {
              float top = -INFINITY, sum = 0.0f, m2[2], l2[2];  // n is at most 48
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int k = lane_j + 32 * h;
                m2[h] = k < n ? __ldcg(rec_m + record(k) + q) : -INFINITY;
                l2[h] = k < n ? __ldcg(rec_l + record(k) + q) : 0.0f;
                top = fmaxf(top, m2[h]);
              }
#pragma unroll
              for (int e = 1; e < 32; e *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, e));
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float f = m2[h] == -INFINITY ? 1.0f : ex2_ftz(m2[h] - top);
                if (lane_j + 32 * h < n) merge_j[(lane_j + 32 * h) * NR + q] = f;
                sum += f * l2[h];
              }
#pragma unroll
              for (int e = 1; e < 32; e *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, e);
              if (lane_j == 0) {
                l_j[q] = sum;
                if (!whole) {
                  m_j[q] = top;
                } else if (a.lse) {
                  a.lse[(long long)walk.row * a.n_heads + h0 + q] = (top + log2f(sum)) * kLn2;
                }
              }
            }
            sync();
          }
#pragma unroll
          for (int k = 0; k < kAhead; ++k)
          {
            const float f = mine && k0 + k < n ? merge_j[(k0 + k) * NR + r] : 0.0f;
            o.x += f * v[k].x;
            o.y += f * v[k].y;
            o.z += f * v[k].z;
            o.w += f * v[k].w;
          }
        }
        if (!mine) continue;
        if (!whole) {
          *reinterpret_cast<float4*>(records + (long long)(record(0) + r) * D + d) = o;
          continue;
        }
        const float inv = 1.0f / l_j[r];
        const long long at = ((long long)walk.row * a.n_heads + h0 + r) * D + d;
        if (a.out_f32) {
          *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) =
              make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        } else {
          uint2 w;
          if constexpr (C::kF16) w = make_uint2(pack_half2(o.x * inv, o.y * inv), pack_half2(o.z * inv, o.w * inv));
          else w = make_uint2(pack_bf162(o.x * inv, o.y * inv), pack_bf162(o.z * inv, o.w * inv));
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = w;
        }
      }
      if (whole) {
        sync();  // the buffers are the next unit's
        break;
      }
      if (tid_j < rows) {
        rec_m[record(0) + tid_j] = m_j[tid_j];
        rec_l[record(0) + tid_j] = l_j[tid_j];
      }
      first = 0;
      n = groups;
      step = size;
      whole = true;
      counter = a.counters + n_slots + slot0;
    }
  }
  // a wait that ran into its limit (about two seconds): the outputs are not valid
  if (tid == 0 && ld_shared_volatile(&abort_s) && a.status) atomicMax(a.status, 2);
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
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

// [n_pages * n_kv_heads][page_tokens][D] 16-bit values, read in boxes of [D / 64][box_rows][64 dims] with the
// 128-byte swizzle
static int make_map(CUtensorMap* map, const void* base, const asterq_paged_attention_params* p, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return set_error(ASTERQ_ERR_CUDA, "paged_attention: cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[4] = {64u, (cuuint64_t)p->page_tokens, (cuuint64_t)p->head_dim / 64,
                              (cuuint64_t)(p->n_pages > 0 ? p->n_pages * p->n_kv_heads : 1)};
  const cuuint64_t strides[3] = {(cuuint64_t)p->head_dim * 2, 128u, (cuuint64_t)p->head_dim * 2 * p->page_tokens};
  const cuuint32_t box[4] = {64u, (cuuint32_t)box_rows, (cuuint32_t)p->head_dim / 64, 1u}, step[4] = {1u, 1u, 1u, 1u};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void*>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(ASTERQ_ERR_CUDA, "paged_attention: tensor map encoding failed (%d)", (int)r);
  return ASTERQ_OK;
}

// SMs of the current device, read once per device
static int sm_count(int* dev) {
  static int counts[64] = {0};
  if (cudaGetDevice(dev) != cudaSuccess) return 0;
  if (*dev < 64 && counts[*dev]) return counts[*dev];
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev) != cudaSuccess) return 0;
  n = n < kMaxWorkers ? n : kMaxWorkers;
  if (*dev < 64) counts[*dev] = n;
  return n;
}

static int rows_of_block(int group) { return group <= 8 ? 8 : 16; }

static int64_t workspace_bytes(int workers, int rows, int head_dim) {
  return 2ll * workers * rows * (head_dim + 2) * 4 + (4ll * workers * 4 + 15) / 16 * 16;
}

template <class C>
static int launch(const CUtensorMap& k_map, const CUtensorMap& v_map, const Args& a, int workers, int dev,
                  cudaStream_t s) {
  static unsigned long long configured = 0;  // one bit per device ordinal
  if (dev >= 64 || !(configured & (1ull << dev))) {
    const cudaError_t e = cudaFuncSetAttribute(attention_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess)
      return set_error(ASTERQ_ERR_CUDA, "paged_attention: shared memory opt-in: %s", cudaGetErrorString(e));
    if (dev < 64) configured |= 1ull << dev;
  }
  attention_kernel<C><<<workers, C::kThreads, C::kSmem, s>>>(k_map, v_map, a);
  return check_launch("paged_attention");
}

template <bool kF16, int D>
static int by_rows(const CUtensorMap& k_map, const CUtensorMap& v_map, const Args& a, int workers, int dev,
                   cudaStream_t s) {
  if (rows_of_block(a.group) == 8) return launch<Cfg<kF16, D, 8>>(k_map, v_map, a, workers, dev, s);
  return launch<Cfg<kF16, D, 16>>(k_map, v_map, a, workers, dev, s);
}

static int check(const asterq_paged_attention_params* p) {
  if (!p) return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "paged_attention: null parameters");
  if (p->n_rows < 0 || p->n_heads <= 0 || p->n_kv_heads <= 0 || p->n_heads % p->n_kv_heads || p->page_tokens <= 0 ||
      p->max_pages < 0 || p->n_pages < 0 || p->n_new < 0 || p->window < 0 || p->sink < 0)
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "paged_attention: bad sizes");
  if (p->dtype != ASTERQ_DTYPE_BF16 && p->dtype != ASTERQ_DTYPE_F16)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "paged_attention: dtype %d: bf16 or f16", p->dtype);
  if (p->out_dtype != p->dtype && p->out_dtype != ASTERQ_DTYPE_F32)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "paged_attention: the output is of the queries' type or f32");
  if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "paged_attention: head_dim %d: 64, 128 or 256", p->head_dim);
  if (p->page_tokens % 16)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "paged_attention: page_tokens %d must be a multiple of 16", p->page_tokens);
  if (p->n_pages * p->n_kv_heads > 0x7fffffffLL || (int64_t)p->max_pages * p->page_tokens > 0x7fff0000LL)
    return set_error(ASTERQ_ERR_UNSUPPORTED, "paged_attention: more than 2^31 pages or tokens of a sequence");
  return ASTERQ_OK;
}

}  // namespace pat
}  // namespace asterq

using namespace asterq;

extern "C" int64_t asterq_paged_attention_workspace_bytes(const asterq_paged_attention_params* p) {
  clear_error();
  if (pat::check(p) != ASTERQ_OK) return 0;
  int dev = 0;
  const int workers = pat::sm_count(&dev);
  return pat::workspace_bytes(workers > 0 ? workers : pat::kMaxWorkers, pat::rows_of_block(p->n_heads / p->n_kv_heads),
                              p->head_dim);
}

extern "C" int asterq_paged_attention(const asterq_paged_attention_params* p, void* stream) {
  clear_error();
  int st = pat::check(p);
  if (st != ASTERQ_OK) return st;
  if (p->n_rows == 0) return ASTERQ_OK;
  if (!p->q || !p->lengths || !p->out || (p->max_pages > 0 && p->n_pages > 0 && (!p->k_pool || !p->v_pool)) ||
      (p->max_pages > 0 && !p->page_table))
    return set_error(ASTERQ_ERR_INVALID_ARGUMENT, "paged_attention: null pointer");
  const void* vec[] = {p->q, p->k_pool, p->v_pool, p->out, p->workspace};
  for (const void* ptr : vec)
    if (reinterpret_cast<uintptr_t>(ptr) & 15)
      return set_error(ASTERQ_ERR_MISALIGNED, "paged_attention: arrays must be 16-byte aligned");
  if (p->q_row_stride % 8 || p->q_head_stride % 8)
    return set_error(ASTERQ_ERR_MISALIGNED, "paged_attention: the queries' strides must be multiples of 8");
  int dev = 0;
  const int workers = pat::sm_count(&dev);
  if (workers <= 0) return set_error(ASTERQ_ERR_CUDA, "paged_attention: no CUDA device");
  pat::Args a;
  a.group = p->n_heads / p->n_kv_heads;
  const int rows = pat::rows_of_block(a.group);
  if (!p->workspace || p->workspace_bytes < pat::workspace_bytes(workers, rows, p->head_dim))
    return set_error(ASTERQ_ERR_WORKSPACE, "paged_attention: workspace of %lld bytes, %lld needed",
                     (long long)p->workspace_bytes, (long long)pat::workspace_bytes(workers, rows, p->head_dim));
  a.row_blocks = (a.group + rows - 1) / rows;
  a.q = p->q;
  a.page_table = p->page_table;
  a.lengths = p->lengths;
  a.out = p->out;
  a.lse = p->lse;
  // counters first: their place does not depend on the call's geometry, so one workspace serves calls
  // of different heads in turn
  a.counters = static_cast<int*>(p->workspace);
  a.records = reinterpret_cast<float*>(static_cast<char*>(p->workspace) + (4ll * workers * 4 + 15) / 16 * 16);
  a.status = p->status;
  a.q_row_stride = p->q_row_stride;
  a.q_head_stride = p->q_head_stride;
  a.n_pages = p->n_pages;
  a.capacity = p->n_pages > 0 ? (long long)p->max_pages * p->page_tokens : 0;
  a.n_rows = p->n_rows;
  a.n_heads = p->n_heads;
  a.n_kv_heads = p->n_kv_heads;
  a.page_tokens = p->page_tokens;
  a.max_pages = p->max_pages;
  a.n_new = p->n_new;
  a.window = p->window;
  a.sink = p->sink;
  a.out_f32 = p->out_dtype == ASTERQ_DTYPE_F32;
  a.scale = p->softmax_scale;
  a.softcap = p->logit_softcap > 0.0f ? p->logit_softcap : 0.0f;
  a.cap_in = a.softcap > 0.0f ? a.scale / a.softcap : 0.0f;
  // a box of a tile lies in one page: the largest of the tile, its half, .. down to 16 tokens that divides the page
  a.box_rows = 8192 / p->head_dim;
  while (p->page_tokens % a.box_rows) a.box_rows /= 2;
  CUtensorMap k_map, v_map;
  const bool pools = a.capacity > 0;  // with none, nothing is visible and the maps are never read
  if ((st = pat::make_map(&k_map, pools ? p->k_pool : p->workspace, p, a.box_rows)) != ASTERQ_OK) return st;
  if ((st = pat::make_map(&v_map, pools ? p->v_pool : p->workspace, p, a.box_rows)) != ASTERQ_OK) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool f16 = p->dtype == ASTERQ_DTYPE_F16;
  switch (p->head_dim) {
    case 64: return f16 ? pat::by_rows<true, 64>(k_map, v_map, a, workers, dev, s)
                        : pat::by_rows<false, 64>(k_map, v_map, a, workers, dev, s);
    case 128: return f16 ? pat::by_rows<true, 128>(k_map, v_map, a, workers, dev, s)
                         : pat::by_rows<false, 128>(k_map, v_map, a, workers, dev, s);
    default: return f16 ? pat::by_rows<true, 256>(k_map, v_map, a, workers, dev, s)
                        : pat::by_rows<false, 256>(k_map, v_map, a, workers, dev, s);
  }
}
