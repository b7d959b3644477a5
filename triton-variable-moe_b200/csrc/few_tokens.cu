// The MoE layer for a few tokens (decode), in two kernels (four above 8 tokens; the router
// kernel also runs for an fp32 router beside 16-bit x), and
// the products of 4-bit expert weights with rows grouped by expert, in two.
//
// Mathematics, for token t and its k experts S(t):
//   l[t,e] = sum_h x[t,h] Wr[e,h]     S(t) = the k largest l[t,:]
//   p[t,e] = sigmoid(l[t,e])          g[t,e] = p / (sum_S p + 1e-20), or p
//   u = x[t] W1_e                     h = act(u)
//   out[t] = sum_{e in S(t)} g[t,e] (h W2_e)
// Every sum is fp32 and the output is rounded once.
//
// What bounds it: the weights of the experts that the tokens reach are read
// once from HBM; nothing else is large.  At one token of a small layer the
// bytes take about a microsecond and the chain launch -> router -> up -> down
// -> sum is what costs, so there are two launches up to 8 tokens, each able to start
// while the one before it ends, no host step and no memset:
//   up kernel    Every cluster of 2 to 8 CTAs computes the routing for itself (each
//                CTA its part of the hidden size, the sums exchanged over
//                distributed shared memory): it costs one or two microseconds of
//                L2 reads and needs no launch and no grid-wide wait of its own.
//                Then the grid's teams of four warps share the items (expert, tile of
//                64 or 128 columns, 8 or 16 of its tokens).  Items that do not make
//                a whole wave are cut into slices of the reduction, all in one
//                cluster; the team that finishes an item's last slice (a counter in
//                shared memory) adds them in order.  Then the activation, and h.
//                (More than 8 tokens: a router kernel runs first.)
//   down kernel  The units (slice of an expert's width, tile of the hidden size).  The team that finishes a column tile's last unit
//                (a counter per tile, zeroed by the up kernel) adds the tile's
//                partial sums in a fixed order, weights them and writes the
//                output: results do not depend on timing.  (More than 8 tokens: a
//                sum kernel after it.)
// Measured: one token of 768 on 16 experts 18.5 us, all latency; 5 tokens on 64 experts of
// 2048 x 1024 69.5 us (3.8 TB/s over the call, 5.2 while it streams); 64 tokens of 4096 on
// 128 experts 423 us, 5.6 TB/s where a copy reaches 6.6.  (Prefetching the down weights to
// L2 as the up kernel ends: 69.3 to 69.9 us at 16 MB, 73 at 64 MB, as other teams still
// stream theirs.)
// No block waits for another but at hardware barriers and the grid dependency
// between the two launches; a warp's wait for its own copies is bounded.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <mutex>
#include <type_traits>

#include "few_tokens.cuh"
#include "moe_internal.h"
#include "sm100_ptx.cuh"

namespace moe {
namespace {

namespace cg = cooperative_groups;
using namespace few;

constexpr int kMaxTokens = 64;    // one 64-bit mask of tokens an expert
constexpr int kMaxExperts = 256;  // (a byte names one)
constexpr int kMaxTopK = 32;
constexpr int kMaxCluster = 8;
constexpr int kThreads = 512;     // 16 warps: at 128 registers a thread the SM is full
constexpr int kWarps = kThreads / 32;
constexpr int kTeam = 4;          // warps that share a unit (they split its reduction)
constexpr int kTeams = kWarps / kTeam;
constexpr int kTeamThreads = kTeam * 32;
constexpr int kMaxLocal = kMaxCluster * kTeams;  // sliced items of a cluster: under a wave
constexpr int kMinTile = 64;      // columns of a unit: L::kTile, 64 or 128
constexpr int kMaxTile = 128;
template <typename L>
constexpr int kRedLd = L::kTile + 4;
constexpr int kMaxSlices = 16;
constexpr int kMaxDepth = 4;
constexpr int kAddTokens = 8;     // up to this many, the down kernel writes the output
constexpr int kMaxWidth = 32768;  // hidden size and expert width: item counts stay 32-bit

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }
// log2 of the outputs of a tile: a gated activation's is half gate and half up columns.
template <typename L>
__device__ __forceinline__ int outputs_log2(int act) {
  constexpr int n = L::kTile == 128 ? 7 : 6;
  static_assert(1 << n == L::kTile, "tiles of 64 or 128 columns");
  return act == ACT_SWIGLU ? n - 1 : n;
}
__host__ __device__ inline int group_count(int rows, int shift) {
  return (rows + (1 << shift) - 1) >> shift;
}

// ---- what both kernels of the layer know -----------------------------------
// The experts that have rows, in order (built by the up kernel).
struct Active {
  int n[kMaxExperts];      // rows
  int base[kMaxExperts];   // first row in expert-sorted order
  int first[kMaxExperts];  // first column of w1 (grouped: of the offsets)
  int width[kMaxExperts];  // intermediate width
  int kb[kMaxExperts];     // packed w2: first block row, first group
  int sg[kMaxExperts];
  int item[kMaxExperts];   // first work item
};
constexpr int kActiveArrays = 7;
// The same numbers for the down kernel, in the workspace.
enum PlanWord : int { PLAN_ACTIVE = 0, PLAN_LENGTH = 1, PLAN_ITEMS = 2, PLAN_WORDS = 32 };

struct LayerParams {
  CUtensorMap map1, map2;    // dense w1, w2
  const void* x;
  long long ldx;
  const void* router;
  int router_fp32;  // the router is fp32 beside 16-bit x (4-bit experts only)
  const void* w1;
  const void* s1;  // 4-bit weights: group scales
  const void* w2;
  const void* s2;
  const int* off;  // [E + 1] columns of w1
  int T, H, E, k, norm, act, total, max_width;
  int shift;                 // log2 of the group
  int blocks2, groups2;      // block rows and groups of the packed w2
  int down_teams;            // teams of the down kernel's grid
  int smem_work;             // up kernel: bytes before its UpSmem
  int cluster;               // its CTAs a cluster (1: the router kernel ran)
  void* out;
  long long ldo;
  // workspace
  int* sel;                  // [T * k] from the router kernel, or null
  int* plan;                 // [PLAN_WORDS], then an Active
  int* slot;                 // [T * k] active expert of an assignment (-1: none)
  int* row;                  // [T * k] its expert-sorted row
  float* wgt;                // [T * k]
  int* ticket;               // [tiles of the hidden size]
  float* u;                  // [slices][T * k][ldu]: partial sums of sliced items
  long long ldu;
  void* h;                   // [T * k][ldh]: see HiddenSource
  long long ldh;
  float* y;                  // [slices][T * k][H]
  int max_slices;
  int* status;
  unsigned long long wait_ns;  // limit of a wait for copies
};

// The rows of a packed w2's segments, an expert each: segment e is rows row[e] ..
// row[e + 1] - 1 (n = 0: not known, and taken from the call's offsets).
struct PackedRows {
  int n;
  int row[kMaxExperts + 1];
};
struct NoRows {};
template <typename L>
using RowsOf = std::conditional_t<L::kPacked, PackedRows, NoRows>;

// Exclusive prefix sum over a warp; `total` gets the sum.
__device__ __forceinline__ int warp_scan(int v, int* total) {
  const int lane = threadIdx.x & 31;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int q = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += q;
  }
  *total = __shfl_sync(0xffffffffu, s, 31);
  return s - v;
}

// The active expert whose items hold index i.
__device__ __forceinline__ int find_item(const int* item, int n, int i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (item[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Counts up; releases what the thread has seen written and acquires what others
// released, within the cluster (a counter in shared memory) or the GPU.
__device__ __forceinline__ int count_cluster(int* counter) {
  int old;
  asm volatile("atom.acq_rel.cluster.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
  return old;
}
__device__ __forceinline__ int count_gpu(int* counter) {
  int old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
  return old;
}

__device__ __forceinline__ void team_sync(int team) {
  asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(kTeamThreads) : "memory");
}

// One unit of a team.  The first units of every team are worked out once, a thread each,
// into a table in shared memory: by the warps themselves, twice (for the copies and for
// the products), that is a few thousand cycles before the first byte.
struct alignas(16) Unit {
  Strip strip;
  int begin;           // first reduction row
  int count;           // vectors
  int row;             // first of them in expert-sorted order
  int e, tile, slice;  // active expert, column tile, slice of the reduction
  int local;           // up kernel: the cluster's item that this is a slice of, or -1
};
static_assert(sizeof(Unit) == 64, "four vectors");
constexpr int kTable = 64;  // units a team

// What every kernel here keeps in shared memory (16-byte vectors follow it).
struct alignas(16) Common {
  Active act;
  unsigned long long bar[kWarps][kMaxDepth];
  int plan[4];  // number of active experts, items, rounds of a slice
  int last[kTeams];
  int abort;
  Unit table[kTeams][kTable];
};

// The strip of an up product's tile.
template <typename L>
__device__ __forceinline__ void up_strip(Strip& s, int first, int width, int act, int tile, int H,
                                         int shift) {
  constexpr int half = L::kTile / 2;
  s.row = 0;
  s.kb = s.sg = 0;
  s.groups = group_count(H, shift);
  if (act == ACT_SWIGLU) {
    s.col = first + tile * half;
    s.lo = s.hi = min(half, width - tile * half);
    s.jump = width;
  } else {
    s.col = first + tile * L::kTile;
    s.lo = min(half, width - tile * L::kTile);
    s.hi = min(half, max(0, width - tile * L::kTile - half));
    s.jump = half;
  }
}
template <typename L>
__device__ __forceinline__ void down_strip(Strip& s, const Active& a, int e, int row, int tile,
                                           int H, int shift) {
  s.row = row;
  constexpr int half = L::kTile / 2;
  s.col = tile * L::kTile;
  s.lo = min(half, H - s.col);
  s.hi = min(half, max(0, H - s.col - half));
  s.jump = half;
  s.kb = a.kb[e];
  s.sg = a.sg[e];
  s.groups = group_count(a.width[e], shift);
}

// Bounded wait of a warp for a phase of a copy barrier.  false, for all lanes: it ran
// out, here or in another warp (abort).  A poll may suspend the warp, for longer than a
// copy takes: not with a limit below a millisecond.  (The part after the first poll is
// hardly ever run, and kept out of the loops.)
__device__ __noinline__ bool ring_wait_on(uint32_t bar, uint32_t parity, volatile int* abort,
                                          uint64_t limit) {
  const bool brief = limit < 1000000;
  if (brief && __all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
  const uint64_t t0 = global_timer_ns();
  do {
    // (+ 1: the timer may stand still for longer than a small limit)
    if (__any_sync(0xffffffffu, *abort || global_timer_ns() - t0 + 1 >= limit)) {
      *abort = 1;
      return false;
    }
  } while (!__all_sync(0xffffffffu,
                       brief ? mbar_test_wait(bar, parity) : mbar_try_wait(bar, parity)));
  return true;
}
__device__ __forceinline__ bool ring_wait(uint32_t bar, uint32_t parity, volatile int* abort,
                                          uint64_t limit) {
  return (limit >= 1000000 && __all_sync(0xffffffffu, mbar_try_wait(bar, parity))) ||
         ring_wait_on(bar, parity, abort, limit);
}

// Runs the `total` units of a team.  Every warp copies its steps (begin + (wr + 4 j)
// kStep) into its ring as far ahead as it is deep, on into its next units, so the
// loads go on during the reduction and the output of a unit.  unit(n) works out the
// team's n-th unit, source(unit) gives its vectors, and finish(unit) finds the unit's
// sums in red (see unit_sum) between team barriers.
template <int N>
using Int = std::integral_constant<int, N>;

template <typename L, int NG, typename MakeUnit, typename MakeSource, typename Finish>
__device__ __forceinline__ void run_units(int total, const Matrix& m,
                                          unsigned char* work, float* red, Common& c,
                                          uint64_t limit, MakeUnit unit, MakeSource source,
                                          Finish finish) {
  constexpr int kRows = kTeam * L::kStep, TOK = L::template kTokens<NG>;
  constexpr int D = L::template kDepth<NG>;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int team = wid / kTeam, wr = wid % kTeam;
  const uint32_t ring = smem_u32(work) + wid * (D * L::kStage);
  const uint32_t bars = smem_u32(&c.bar[wid][0]);
  const typename L::Lane at(lane, m.gated);
  using Src = decltype(source(unit(0)));
  const int tt = threadIdx.x % kTeamThreads;
  if (tt < min(total, kTable)) c.table[team][tt] = unit(tt);
  team_sync(team);
  auto nth = [&](int n) { return n < kTable ? c.table[team][n] : unit(n); };

  int copied = 0, used = 0;  // steps
  uint32_t copy_slot = 0, use_slot = 0, phase = 0;
  // the copying side: the team's cn-th unit, next step at row ck
  int cn = -1, ck = 0, cend = 0;
  bool more = true;
  typename L::Cursor cursor;
  auto top_up = [&]() {
    while (more && copied - used < D) {
      if (ck >= cend) {
        more = ++cn < total;
        if (more) {
          const Unit cu = nth(cn);
          ck = cu.begin + wr * L::kStep;
          cend = cu.strip.end;
          if (ck < cend) cursor.set(m, cu.strip, ck);
        }
      } else {
        if (lane == 0) cursor.issue(m, ring + copy_slot * L::kStage, bars + 8 * copy_slot);
        copy_slot = copy_slot + 1 == D ? 0 : copy_slot + 1;
        ++copied;
        ck += kRows;
        cursor.template next<kRows>(m);
      }
    }
  };
  top_up();
  float acc[L::kSums][NG][4];
  for (int n = 0; n < total; ++n) {
    const Unit u = nth(n);
    const Src src = source(u);
    // with only the groups of columns, and parts, that the unit has
    auto sums = [&](auto groups, auto parts) {
      constexpr int G = decltype(groups)::value, P = decltype(parts)::value;
#pragma unroll
      for (int a = 0; a < L::kSums; ++a)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[a][g][j] = 0.f;
      const int k = u.begin + wr * L::kStep;
      int left = u.strip.end - k;
      typename L::template Vectors<NG, Src> v;
      if (left > 0) {
        v.template rows<G, P>(src, u.count, k, lane);
        v.template load<G, P>(0, src, left, lane);
      }
      for (; left > 0; left -= kRows) {  // the vectors of each half load during the half before
        const uint32_t stage = ring + use_slot * L::kStage;
        v.template load<G, P>(1, src, left, lane);
        if (used < copied && !ring_wait(bars + 8 * use_slot, phase, &c.abort, limit))
          more = false;  // (its place may still be written: no further copies of this warp)
        L::template half<G, P, NG, Src>(0, acc, at, m, u.strip, left, stage, lane, v);
        v.template advance<G>(kRows);
        v.template load<G, P>(0, src, left - kRows, lane);
        L::template half<G, P, NG, Src>(1, acc, at, m, u.strip, left, stage, lane, v);
        __syncwarp();  // the step has been read by every lane: its place is free
        ++used;
        if (++use_slot == D) {
          use_slot = 0;
          phase ^= 1;
        }
        top_up();
      }
      // warps 2 and 3 leave their sums, 0 and 1 add theirs to them
      float* mine = red + (wr & 1) * TOK * kRedLd<L>;
      if (wr >= 2) L::template store<G, NG, kRedLd<L>, false>(acc, lane, mine);
      team_sync(team);
      if (wr < 2) L::template store<G, NG, kRedLd<L>, true>(acc, lane, mine);
      team_sync(team);
    };
    if constexpr (!L::kGroups)
      sums(Int<NG>(), Int<1>());
    else if (NG > 1 && u.count > 8)
      sums(Int<NG>(), Int<Src::kParts>());
    else if (Src::kParts == 2 && u.count > 4)
      sums(Int<1>(), Int<2>());
    else
      sums(Int<1>(), Int<1>());
    finish(u);
    team_sync(team);
  }
  // After a wait that ran out: the warp's last copies (the ones before them were waited
  // for) land before the block ends and its shared memory is another's.
  if (*static_cast<volatile int*>(&c.abort)) {
    for (int j = max(0, copied - D); j < copied; ++j) {
      const uint64_t t0 = global_timer_ns();
      while (!mbar_try_wait(bars + 8 * (j % D), (j / D) & 1) &&
             global_timer_ns() - t0 <= MOE_WAIT_NS) {
      }
    }
  }
}

// Before a kernel's first copies: the warp's barriers, each for one arrival (its
// own lane's) a phase.
template <int D>
__device__ __forceinline__ void ring_init(Common& c) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  if (lane < D) {
    mbar_init(reinterpret_cast<uint64_t*>(&c.bar[wid][lane]), 1);
    fence_barrier_init();
  }
  __syncwarp();
  if (threadIdx.x == 0) c.abort = 0;  // (seen by all after the next block barrier)
}

// The unit's sums of vector `tok`, columns c .. c + 3.
template <typename L, int NG>
__device__ __forceinline__ float4 unit_sum(const float* red, int tok, int c) {
  constexpr int TOK = L::template kTokens<NG>, LD = kRedLd<L>;
  const float4 a = *reinterpret_cast<const float4*>(red + tok * LD + c);
  const float4 b = *reinterpret_cast<const float4*>(red + (TOK + tok) * LD + c);
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}
__device__ __forceinline__ void add4(float4& a, const float4& b) {
  a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
}
template <typename T>
__device__ __forceinline__ void store4(T* d, float4 v, bool vec) {
  if (vec) {
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint2*>(d) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
    else
      *reinterpret_cast<float4*>(d) = v;
  } else {
    d[0] = from_f<T>(v.x);
    d[1] = from_f<T>(v.y);
    d[2] = from_f<T>(v.z);
    d[3] = from_f<T>(v.w);
  }
}

// Shared memory of the teams: rings (1 KB aligned for the swizzle), then two sum
// buffers a team.
template <typename L, int NG>
constexpr int kRingBytes = kWarps * L::template kDepth<NG> * L::kStage;
template <typename L, int NG>
constexpr int kRedFloats = 2 * L::template kTokens<NG> * kRedLd<L>;  // a team
template <typename L, int NG>
constexpr int kWorkBytes = kRingBytes<L, NG> + 4 * kTeams * kRedFloats<L, NG>;

// Length of a slice, in rounds (a step by each warp of a team), that finishes
// first for items of `rounds` rounds each and `passes` each: whole waves of units
// over the teams, a unit's own cost being `own` and a round's four quarter rounds;
// what a slice adds to the final sum counts a quarter.  One warp; lane 0's result
// is everyone's.
__device__ __forceinline__ int slice_length(int i) {  // 1 2 3 4 6 8 12 16 .. 512
  return i == 0 ? 1 : i % 2 ? 2 << (i - 1) / 2 : 3 << (i - 2) / 2;
}
constexpr int kLengths = 18;
static_assert(kMaxWidth <= 512 * 64, "the last length is the rounds of the longest reduction");
template <typename Units>
__device__ __forceinline__ int plan_length(int most, int teams, int max_slices, int own,
                                           Units units) {
  long long best = 0x7fffffffffffffffll;
  int best_len = 0;
#pragma unroll 1
  for (int i = 0; i < kLengths; ++i) {
    const int len = slice_length(i);
    const int parts = ceil_div(most, len);
    if (parts <= max_slices) {
      const long long waves = (units(len) + teams - 1) / teams;
      const long long cost = waves * (4 * min(len, most) + own) + parts;
      if (cost < best) {
        best = cost;
        best_len = len;
      }
    }
    if (len >= most) break;
  }
  return best_len;
}

// ---- routing --------------------------------------------------------------
// This CTA's partial logits of up to 8 tokens over reduction range [k_lo, k_hi):
// log[t][E16].
template <typename T>
__device__ __forceinline__ void partial_logits(const LayerParams& p, const T* x, int count,
                                               int k_lo, int k_hi, float* part, float* log,
                                               int lde) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const T* wr = static_cast<const T*>(p.router);
  const int tiles = lde / 16, ksub = max(1, kWarps / tiles);
  // 16 experts an item; ksub warps split its reduction
  for (int item = wid; item < tiles * ksub; item += kWarps) {
    const int et = item % tiles, ks = item / tiles;
    const int e0 = et * 16 + g, e1 = e0 + 8;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    constexpr int kBatch = 4;  // steps whose loads are issued together
    for (int k0 = k_lo + 32 * ks; k0 < k_hi; k0 += 32 * ksub * kBatch) {
      uint4 a[kBatch][2], b[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int k = k0 + 32 * ksub * j + 8 * t4;
        const bool in = k0 + 32 * ksub * j < k_hi && k < p.H;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        a[j][0] = in && e0 < p.E
                      ? *reinterpret_cast<const uint4*>(wr + static_cast<long long>(e0) * p.H + k)
                      : zero;
        a[j][1] = in && e1 < p.E
                      ? *reinterpret_cast<const uint4*>(wr + static_cast<long long>(e1) * p.H + k)
                      : zero;
        b[j] = in && g < count
                   ? *reinterpret_cast<const uint4*>(x + static_cast<long long>(g) * p.ldx + k)
                   : zero;
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const uint32_t a0[4] = {a[j][0].x, a[j][1].x, a[j][0].y, a[j][1].y};
        const uint32_t a1[4] = {a[j][0].z, a[j][1].z, a[j][0].w, a[j][1].w};
        mma<T>(acc, a0, b[j].x, b[j].y);
        mma<T>(acc, a1, b[j].z, b[j].w);
      }
    }
    // rows of the result are experts, columns tokens
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = 2 * t4 + j;
      if (t < count) {
        part[(ks * count + t) * lde + e0] = acc[j];
        part[(ks * count + t) * lde + e1] = acc[j + 2];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count * lde; i += kThreads) {
    float s = part[i];
    for (int q = 1; q < ksub; ++q) s += part[q * count * lde + i];
    log[i] = s;
  }
}

// Four neighbouring values as floats.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    const float2 a = unpack2<T>(v.x), b = unpack2<T>(v.y);
    return make_float4(a.x, a.y, b.x, b.y);
  }
}

// The same with an fp32 router (the layer's own type, or that of a layer whose experts
// alone were quantised): plain FMAs, as the tensor pipe would round the weight.
template <typename T>
__device__ __forceinline__ void partial_logits_fp32(const LayerParams& p, const T* x, int count,
                                                    int k_lo, int k_hi, float* log, int lde) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const float* wr = static_cast<const float*>(p.router);
  const int hi = min(k_hi, p.H);
  for (int e = wid; e < p.E; e += kWarps) {
    const float* row = wr + static_cast<long long>(e) * p.H;
    for (int t0 = 0; t0 < count; t0 += 8) {
      float acc[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = 0.f;
      for (int k = k_lo + 4 * lane; k < hi; k += 128) {
        const float4 w = *reinterpret_cast<const float4*>(row + k);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (t0 + j < count) {
            const float4 v = load4<T>(x + static_cast<long long>(t0 + j) * p.ldx + k);
            acc[j] = fmaf(v.x, w.x, acc[j]);
            acc[j] = fmaf(v.y, w.y, acc[j]);
            acc[j] = fmaf(v.z, w.z, acc[j]);
            acc[j] = fmaf(v.w, w.w, acc[j]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
        if (lane == 0 && t0 + j < count) log[(t0 + j) * lde + e] = acc[j];
      }
    }
  }
}
template <>
__device__ __forceinline__ void partial_logits<float>(const LayerParams& p, const float* x,
                                                      int count, int k_lo, int k_hi, float*,
                                                      float* log, int lde) {
  partial_logits_fp32<float>(p, x, count, k_lo, k_hi, log, lde);
}

// Unsigned order of floats; NaN above all (torch.topk's order).  Never 0.
__device__ __forceinline__ unsigned order_key(float v) {
  if (isnan(v)) return 0xffffffffu;
  const unsigned b = __float_as_uint(v + 0.f);  // -0 equals 0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// One warp chooses the k experts of row t of the cluster's partial logits (value j of
// lane l is expert 32 j + l): lane s < k gets the s-th and its weight.
template <int J>
__device__ __forceinline__ void choose(const LayerParams& p, cg::cluster_group& cluster, float* log,
                                       int lde, int t, int* sel_out, float* wgt_out) {
  const int lane = threadIdx.x & 31;
  float v[J];
  unsigned key[J];
#pragma unroll
  for (int j = 0; j < J; ++j) v[j] = 0.f;
  const int ctas = static_cast<int>(cluster.num_blocks());
#pragma unroll
  for (int c0 = 0; c0 < kMaxCluster; c0 += 4) {  // four CTAs' parts in flight
    if (c0 >= ctas) break;
    float a[4][J];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float* q = cluster.map_shared_rank(log, min(c0 + c, ctas - 1)) + t * lde;
#pragma unroll
      for (int j = 0; j < J; ++j) a[c][j] = q[min(32 * j + lane, p.E - 1)];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int j = 0; j < J; ++j) v[j] += c0 + c < ctas ? a[c][j] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < J; ++j) key[j] = 32 * j + lane < p.E ? order_key(v[j]) : 0u;
  float mine = 0.f;
  int sel = 0;
  for (int s = 0; s < p.k; ++s) {
    unsigned best = key[0];
#pragma unroll
    for (int j = 1; j < J; ++j) best = max(best, key[j]);
    best = __reduce_max_sync(0xffffffffu, best);
    unsigned at = 0xffffffffu;
    float val = 0.f;
#pragma unroll
    for (int j = J - 1; j >= 0; --j)
      if (key[j] == best) {
        at = 32 * j + lane;
        val = v[j];
      }
    const unsigned e = __reduce_min_sync(0xffffffffu, at);  // ties: the lower index
    val = __shfl_sync(0xffffffffu, val, e & 31);
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (e == 32u * j + lane) key[j] = 0u;
    if (lane == s) {
      mine = val;
      sel = static_cast<int>(e);
    }
  }
  float w = lane < p.k ? 1.f / (1.f + expf(-mine)) : 0.f;
  if (p.norm) {
    float sum = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    w = w / (sum + 1e-20f);
  }
  *sel_out = sel;
  *wgt_out = w;
}
__device__ __forceinline__ void choose(const LayerParams& p, cg::cluster_group& cluster, float* log,
                                       int lde, int t, int* sel, float* wgt) {
  if (p.E <= 32)
    choose<1>(p, cluster, log, lde, t, sel, wgt);
  else if (p.E <= 64)
    choose<2>(p, cluster, log, lde, t, sel, wgt);
  else if (p.E <= 128)
    choose<4>(p, cluster, log, lde, t, sel, wgt);
  else
    choose<8>(p, cluster, log, lde, t, sel, wgt);
}

// ---- router kernel (more than 8 tokens, or an fp32 router beside 16-bit x) ---------
// Every cluster of the up kernel would route all tokens (33 tokens, 64 experts: 7 us);
// here a cluster of 8 CTAs has 8 of them, each CTA an eighth of the hidden size and
// then one token to choose for.  The up kernel then needs no clusters and runs on all
// SMs.
// R: type of the router, T's or fp32 (an instance of its own: as a branch it cost 17 tokens
// of 1104 0.2 us).
template <typename T, typename R>
__global__ void __launch_bounds__(kThreads, 1) few_router_kernel(const __grid_constant__ LayerParams p) {
  extern __shared__ __align__(1024) unsigned char raw[];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), lane = threadIdx.x & 31;
  const int t0 = blockIdx.x / kMaxCluster * kMaxCluster, count = min(kMaxCluster, p.T - t0);
  const int lde = ceil_div(p.E, 16) * 16;
  float* log = reinterpret_cast<float*>(raw);
  float* part = log + count * lde;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int per = ceil_div(ceil_div(p.H, 32), kMaxCluster) * 32;
  const T* x = static_cast<const T*>(p.x) + t0 * p.ldx;
  const int k_lo = min(rank * per, p.H), k_hi = min((rank + 1) * per, p.H);
  if constexpr (!std::is_same_v<R, T>)
    partial_logits_fp32<T>(p, x, count, k_lo, k_hi, log, lde);
  else
    partial_logits<T>(p, x, count, k_lo, k_hi, part, log, lde);
  cluster.sync();
  if (rank < count && threadIdx.x < 32) {
    int sel;
    float wgt;
    choose(p, cluster, log, lde, rank, &sel, &wgt);
    if (lane < p.k) {
      p.sel[(t0 + rank) * p.k + lane] = sel;
      p.wgt[(t0 + rank) * p.k + lane] = wgt;
    }
  }
  cluster.sync();  // the parts stay until they have been read
}

// ---- the layer's active experts ----------------------------------------------
struct alignas(16) UpSmem {
  Common c;
  unsigned long long mask[kMaxExperts];      // tokens of each expert
  int off[kMaxExperts + 1];
  int slot[kMaxExperts];  // active expert of an expert (-1: none)
  int base[kMaxExperts];  // first expert-sorted row of an expert
  int ticket[kMaxLocal];  // slices done of the cluster's items (rank 0's is used)
  int kb[kMaxExperts];    // packed w2 (otherwise 0): first block row, first group,
  int sg[kMaxExperts];
  int fits[kMaxExperts];  // and whether the expert lies in it
  int row[kMaxExperts + 1];  // its row offsets, where they are known
};
static_assert(sizeof(UpSmem) % 16 == 0, "16-byte vectors follow");

// Whether an expert's offsets [a, b) are columns of the matrix, and whether the width
// that they give is one that the call allows.
__device__ __forceinline__ bool expert_columns(int a, int b, int total, int act) {
  const int step = (act == ACT_SWIGLU ? 32 : 16) - 1;
  return a >= 0 && b >= a && b <= total && ((a | b) & step) == 0;
}
__device__ __forceinline__ bool expert_width(int a, int b, int total, int max_width, int act,
                                             int* width) {
  const int gated = act == ACT_SWIGLU ? 1 : 0;  // log2
  const bool ok = expert_columns(a, b, total, act) && (b - a) >> gated <= max_width;
  *width = ok ? (b - a) >> gated : 0;
  return ok;
}

// One warp: where each expert's rows of a packed w2 start, and whether they are the
// call's.  Known rows (in shared memory: read from the arguments here, a lane each, they
// cost the down product of 192 rows 0.6 us): the expert's offsets have to be its
// segment's.  Otherwise the segments are those of the offsets, as far as these are columns
// of w1: nothing says where the experts after others start, and they are refused.
__device__ __forceinline__ void find_packed(bool known, const int* row, const int* off, int E,
                                            int total, int act, int shift, int blocks2, int groups2,
                                            int* kb_s, int* sg_s, int* fits) {
  const int lane = threadIdx.x & 31, gated = act == ACT_SWIGLU ? 1 : 0;
  int kb = 0, sg = 0;
  bool lost = false;
#pragma unroll 1
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int e = e0 + lane;
    int a = 0, b = 0, n;
    if (e < E) {
      a = off[e];
      b = off[e + 1];
    }
    bool ok;
    int w;
    if (known) {
      const int lo = e < E ? row[e] : 0, hi = e < E ? row[e + 1] : 0;
      ok = a == lo << gated && b == hi << gated;
      w = hi - lo;
    } else {
      const unsigned bad = __ballot_sync(0xffffffffu, !expert_columns(a, b, total, act));
      ok = !lost && (bad & ((2u << lane) - 1)) == 0;
      w = ok ? (b - a) >> gated : 0;
      lost = lost || bad != 0;
    }
    const int blocks = ceil_div(w, 64), groups = group_count(w, shift);
    const int my_kb = kb + warp_scan(blocks, &n);
    kb += n;
    const int my_sg = sg + warp_scan(groups, &n);
    sg += n;
    if (e < E) {
      kb_s[e] = my_kb;
      sg_s[e] = my_sg;
      fits[e] = ok && my_kb + blocks <= blocks2 && my_sg + groups <= groups2;
    }
  }
}

// One warp: from the token masks and the offsets, the experts that have rows and
// columns, and their (pass, tile) items.  Offsets that leave the matrices, or are
// not in steps of 16, empty the expert and set the status word.
template <typename L, int TOK>
__device__ __forceinline__ void find_active(const LayerParams& p, UpSmem& s) {
  const int lane = threadIdx.x & 31, outputs = outputs_log2<L>(p.act);
  static_assert((kMaxTokens / 4 * kMaxTopK + kMaxExperts) * (kMaxWidth / 32) <= 1 << 20,
                "20 bits of items, 12 of rows");
  unsigned sums = 0;
  int active = 0;
#pragma unroll 1
  for (int e0 = 0; e0 < p.E; e0 += 32) {
    const int e = e0 + lane;
    int n = 0, a = 0, w = 0;
    bool ok = true;
    unsigned long long mask = 0;
    if (e < p.E) {
      mask = s.mask[e];
      n = __popcll(mask);
      a = s.off[e];
      ok = expert_width(a, s.off[e + 1], p.total, p.max_width, p.act, &w) && s.fits[e];
    }
    if (!ok && p.status && blockIdx.x == 0) *p.status = kStatusBadArg;
    const bool here = ok && n > 0 && w > 0;
    const int items = here ? ceil_div(n, TOK) * ((w + (1 << outputs) - 1) >> outputs) : 0;
    int total;
    const unsigned mine =
        sums + static_cast<unsigned>(warp_scan(static_cast<int>(items | static_cast<unsigned>(n) << 20), &total));
    sums += static_cast<unsigned>(total);
    const unsigned who = __ballot_sync(0xffffffffu, here);
    const int at = active + __popc(who & ((1u << lane) - 1));
    active += __popc(who);
    const int base = static_cast<int>(mine >> 20);
    if (e < p.E) {
      s.slot[e] = here ? at : -1;
      s.base[e] = base;
    }
    if (here) {
      s.c.act.n[at] = n;
      s.c.act.base[at] = base;
      s.c.act.first[at] = a;
      s.c.act.width[at] = w;
      s.c.act.kb[at] = s.kb[e];
      s.c.act.sg[at] = s.sg[e];
      s.c.act.item[at] = static_cast<int>(mine & 0xfffffu);
    }
  }
  if (lane == 0) {
    s.c.plan[0] = active;
    s.c.plan[1] = static_cast<int>(sums & 0xfffffu);
  }
}

// One warp: the down kernel's slice length and items, into the workspace.
template <typename L, int TOK, int ROUND>
__device__ __forceinline__ void plan_down(const LayerParams& p, const Active& act, int active) {
  const int lane = threadIdx.x & 31, tiles = ceil_div(p.H, L::kTile);
  int widest = 0;
  for (int j = lane; j < active; j += 32) widest = max(widest, act.width[j]);
  widest = __reduce_max_sync(0xffffffffu, widest);
  // a unit's own cost in quarter rounds (4, 8, 12 where no final sum follows: 64 tokens,
  // 435, 426, 427 us; 9 for 5, 9, 14 with it: 69.5, 68.9, 69.4 at 5 tokens)
  const int own = p.T <= kAddTokens ? 9 : 8;
  const int len = plan_length(max(1, ceil_div(widest, ROUND)), p.down_teams, p.max_slices, own,
                              [&](int length) {
    int n = 0;
    for (int j = lane; j < active; j += 32)
      n += ceil_div(act.n[j], TOK) * ceil_div(ceil_div(act.width[j], ROUND), length);
    return static_cast<long long>(__reduce_add_sync(0xffffffffu, n)) * tiles;
  });
  int items = 0;
  for (int j0 = 0; j0 < active; j0 += 32) {
    const int j = j0 + lane;
    int n = 0, total;
    if (j < active) n = ceil_div(act.n[j], TOK) * ceil_div(ceil_div(act.width[j], ROUND), len);
    const int before = items + warp_scan(n, &total);
    items += total;
    if (j < active) p.plan[PLAN_WORDS + 6 * kMaxExperts + j] = before;
  }
  if (lane == 0) {
    p.plan[PLAN_ACTIVE] = active;
    p.plan[PLAN_LENGTH] = len;
    p.plan[PLAN_ITEMS] = items;
  }
}

// ---- up kernel ---------------------------------------------------------------
template <typename L, int NG>
__global__ void __launch_bounds__(kThreads, 1)
    few_up_kernel(const __grid_constant__ LayerParams p, const __grid_constant__ RowsOf<L> rows2) {
  using T = typename L::Elem;
  constexpr int TOK = L::template kTokens<NG>, kRound = kTeam * L::kStep;
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* work = raw;  // rings first: 1 KB aligned
  const int lde = ceil_div(p.E, 16) * 16, A = p.T * p.k;
  float* log = reinterpret_cast<float*>(work);  // the routing's sums, before the rings
  float* part = log + p.T * lde;
  UpSmem& s = *reinterpret_cast<UpSmem*>(raw + p.smem_work);
  float* wgt_s = reinterpret_cast<float*>(raw + p.smem_work + sizeof(UpSmem));
  uint8_t* sel_s = reinterpret_cast<uint8_t*>(wgt_s + A);
  uint8_t* list = sel_s + A;  // token of each expert-sorted row
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;

  // (the router kernel, if it ran, waited for the inputs)
  if (!p.sel) asm volatile("griddepcontrol.wait;" ::: "memory");
  // every block of this grid runs by the time the last one gets here
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int e = tid; e <= p.E; e += kThreads) {
    s.off[e] = p.off[e];
    if constexpr (L::kPacked) s.row[e] = rows2.row[e];
  }
  for (int e = tid; e < p.E; e += kThreads) {
    s.mask[e] = 0;
    s.kb[e] = s.sg[e] = 0;
    s.fits[e] = 1;
  }
  for (int i = tid; i < kMaxLocal; i += kThreads) s.ticket[i] = 0;
  ring_init<L::template kDepth<NG>>(s.c);

  unsigned* mask32 = reinterpret_cast<unsigned*>(s.mask);
  auto packed = [&]() {  // (one warp, while others route)
    if constexpr (L::kPacked)
      if (wid == kWarps - 1)
        find_packed(rows2.n > 0, s.row, s.off, p.E, p.total, p.act, p.shift, p.blocks2, p.groups2,
                    s.kb, s.sg, s.fits);
  };
  if (p.sel) {
    __syncthreads();
    packed();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int a = tid; a < A; a += kThreads) {
      const int sel = p.sel[a], t = a / p.k;
      sel_s[a] = static_cast<uint8_t>(sel);
      wgt_s[a] = p.wgt[a];
      atomicOr(mask32 + 2 * sel + (t >> 5), 1u << (t & 31));
    }
    __syncthreads();
  } else {
    // routing: this CTA's part of the hidden size, then tokens rank, rank + cluster, ...
    const int per = ceil_div(ceil_div(p.H, 32), p.cluster) * 32;
    partial_logits<T>(p, static_cast<const T*>(p.x), p.T, min(rank * per, p.H),
                      min((rank + 1) * per, p.H), part, log, lde);
    cluster.sync();
    packed();
    for (int t = rank + p.cluster * wid; t < p.T; t += p.cluster * kWarps) {
      int sel;
      float wgt;
      choose(p, cluster, log, lde, t, &sel, &wgt);
      if (lane < p.k) {
        for (int c = 0; c < p.cluster; ++c) {
          cluster.map_shared_rank(sel_s, c)[t * p.k + lane] = static_cast<uint8_t>(sel);
          cluster.map_shared_rank(wgt_s, c)[t * p.k + lane] = wgt;
          // (32-bit words: in clusters of 2 to 8 CTAs 64-bit ORs through these addresses
          // lost bits in every word of 512,000, 32-bit ones in none; why is not known)
          atomicOr(cluster.map_shared_rank(mask32, c) + 2 * sel + (t >> 5), 1u << (t & 31));
        }
      }
    }
    cluster.sync();
  }

  const int clusters = gridDim.x / p.cluster, teams = gridDim.x * kTeams;
  const int rounds = ceil_div(p.H, kRound);
  if (wid == 0) {
    find_active<L, TOK>(p, s);
    __syncwarp();
    // Whole items, a wave of them over all teams at a time; the rest whole too, or in
    // slices of a cluster's items over its teams.  Lane l weighs l + 1 slices, in
    // quarter rounds: a unit's own cost is a round, a slice's, with the joining, two.
    const int rest = s.c.plan[1] % teams;
    const int local = ceil_div(rest, clusters), cut = lane + 1;
    int cost = 0x7fffffff;
    if (cut == 1)
      cost = 4 * rounds + 4;
    else if (cut <= min(p.max_slices, rounds))
      cost = ceil_div(local * cut, p.cluster * kTeams) * (4 * ceil_div(rounds, cut) + 9);
    const int best = __reduce_min_sync(0xffffffffu, cost);
    const int at = __ffs(__ballot_sync(0xffffffffu, cost == best));
    if (lane == 0) s.c.plan[2] = ceil_div(rounds, at);
  }
  fence_proxy_async_smem();  // the routing's use of the rings, before copies into them
  __syncthreads();
  const int active = s.c.plan[0], U = s.c.plan[1], q = s.c.plan[2];
  const int slices = ceil_div(rounds, q);

  for (int a = tid; a < A; a += kThreads) {
    const int e = sel_s[a], t = a / p.k;
    list[s.base[e] + __popcll(s.mask[e] & ((1ull << t) - 1))] = static_cast<uint8_t>(t);
  }
  __syncthreads();
  if (blockIdx.x == gridDim.x - 1) {  // (the block that units come to last)
    for (int a = tid; a < A; a += kThreads) {
      const int e = sel_s[a], t = a / p.k;
      p.slot[a] = s.slot[e];
      p.row[a] = s.base[e] + __popcll(s.mask[e] & ((1ull << t) - 1));
      if (!p.sel) p.wgt[a] = wgt_s[a];
    }
    for (int i = tid; i < ceil_div(p.H, L::kTile); i += kThreads) p.ticket[i] = 0;
    for (int j = tid; j < active; j += kThreads) {
      int* d = p.plan + PLAN_WORDS + j;
      d[0 * kMaxExperts] = s.c.act.n[j];
      d[1 * kMaxExperts] = s.c.act.base[j];
      d[2 * kMaxExperts] = s.c.act.first[j];
      d[3 * kMaxExperts] = s.c.act.width[j];
      d[4 * kMaxExperts] = s.c.act.kb[j];
      d[5 * kMaxExperts] = s.c.act.sg[j];
    }
    if (wid == kWarps - 1) plan_down<L, TOK, kRound>(p, s.c.act, active);
  }

  // the team's units: its items of the whole waves, then its slices of the cluster's
  // items (every `clusters`-th of the rest; neighbouring slices on different CTAs)
  const int team = wid / kTeam, tt = tid % kTeamThreads;
  const int me = blockIdx.x * kTeams + team, waves = U / teams, rest = U % teams;
  const int mine = blockIdx.x / p.cluster, start = team * p.cluster + rank;
  const int group = p.cluster * kTeams;
  int total = waves;
  if (slices == 1) {
    total += me < rest;
  } else {
    const int units = rest > mine ? ceil_div(rest - mine, clusters) * slices : 0;
    if (units > start) total += ceil_div(units - start, group);
  }
  const Active& act = s.c.act;
  auto unit = [&](int n) {
    Unit u;
    int item = n * teams + me;
    u.slice = 0;
    u.local = -1;
    if (n >= waves && slices > 1) {
      const int i = start + (n - waves) * group;
      u.local = i / slices;
      u.slice = i - u.local * slices;
      item = waves * teams + mine + clusters * u.local;
    }
    u.e = find_item(act.item, active, item);
    const int width = act.width[u.e], outputs = outputs_log2<L>(p.act);
    const int tiles = (width + (1 << outputs) - 1) >> outputs, r = item - act.item[u.e];
    const int pass = r / tiles;
    u.tile = r - pass * tiles;
    u.count = min(act.n[u.e] - pass * TOK, TOK);
    u.row = act.base[u.e] + pass * TOK;
    u.begin = u.slice * q * kRound;
    u.strip.end = u.local < 0 ? p.H : min(p.H, u.begin + q * kRound);
    up_strip<L>(u.strip, act.first[u.e], width, p.act, u.tile, p.H, p.shift);
    return u;
  };
  auto source = [&](const Unit& u) {
    return RowSource<T>{static_cast<const T*>(p.x), p.ldx, list, u.row};
  };
  float* red = reinterpret_cast<float*>(work + kRingBytes<L, NG>) + team * kRedFloats<L, NG>;
  // activated sums of vector tok, from get(tok, column)
  auto emit = [&](const Unit& u, int tok, int c, auto get) {
    const float4 a = get(tok, c);
    float v[4];
    const int col = (u.tile << outputs_log2<L>(p.act)) + c;
    if (p.act == ACT_SWIGLU) {
      const float4 b = get(tok, c + L::kTile / 2);
      v[0] = act_gated(a.x, b.x); v[1] = act_gated(a.y, b.y);
      v[2] = act_gated(a.z, b.z); v[3] = act_gated(a.w, b.w);
    } else {
      v[0] = act_plain(a.x, p.act); v[1] = act_plain(a.y, p.act);
      v[2] = act_plain(a.z, p.act); v[3] = act_plain(a.w, p.act);
    }
    if (col < act.width[u.e])
      hidden_store4<T>(static_cast<T*>(p.h) + (u.row + tok) * p.ldh, p.max_width, col, v);
  };
  const int vecs = 1 << (outputs_log2<L>(p.act) - 2);
  const Matrix m{&p.map1, p.w1, p.s1, p.total, p.shift, p.act == ACT_SWIGLU};
  run_units<L, NG>(total, m, work, red, s.c, p.wait_ns, unit, source, [&](const Unit& u) {
    if (u.local < 0) {
      for (int j = tt; j < u.count * vecs; j += kTeamThreads)
        emit(u, j / vecs, 4 * (j % vecs),
             [&](int tok, int c) { return unit_sum<L, NG>(red, tok, c); });
      return;
    }
    float* dst = p.u + u.row * p.ldu + u.tile * L::kTile;
    const long long slice = static_cast<long long>(A) * p.ldu;
    for (int j = tt; j < u.count * (L::kTile / 4); j += kTeamThreads) {
      const int tok = j / (L::kTile / 4), c = 4 * (j % (L::kTile / 4));
      *reinterpret_cast<float4*>(dst + u.slice * slice + tok * p.ldu + c) =
          unit_sum<L, NG>(red, tok, c);
    }
    team_sync(team);
    if (tt == 0) {
      // (after the team's sums, and before reading the other teams')
      s.c.last[team] =
          count_cluster(cluster.map_shared_rank(s.ticket, 0) + u.local) == slices - 1;
    }
    team_sync(team);
    if (s.c.last[team]) {
      for (int j = tt; j < u.count * vecs; j += kTeamThreads)
        emit(u, j / vecs, 4 * (j % vecs), [&](int tok, int c) {
          const float* src = dst + tok * p.ldu + c;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int z = 0; z < slices; ++z)
            add4(v, __ldcg(reinterpret_cast<const float4*>(src + z * slice)));
          return v;
        });
    }
  });
  if (s.c.abort && lane == 0 && p.status) *p.status = kStatusTimeout;
  if (slices > 1) cluster.sync();  // rank 0's counters stay until the last team is done
}

// ---- down kernel -------------------------------------------------------------
template <typename L, int NG>
__global__ void __launch_bounds__(kThreads, 1)
    few_down_kernel(const __grid_constant__ LayerParams p) {
  using T = typename L::Elem;
  constexpr int TOK = L::template kTokens<NG>, kRound = kTeam * L::kStep;
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* work = raw;
  Common& s = *reinterpret_cast<Common*>(raw + kWorkBytes<L, NG>);
  const int A = p.T * p.k, gated = p.act == ACT_SWIGLU ? 2 : 1;
  int* slot_s = reinterpret_cast<int*>(raw + kWorkBytes<L, NG> + sizeof(Common));
  int* row_s = slot_s + A;
  float* wgt_s = reinterpret_cast<float*>(row_s + A);
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  ring_init<L::template kDepth<NG>>(s);
  if (tid == 0 && p.shift == 0) tma_prefetch_desc(&p.map2);

  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (tid < 3) s.plan[tid] = p.plan[tid];
  static_assert(sizeof(Active) == 4 * kActiveArrays * kMaxExperts && kThreads == 2 * kMaxExperts,
                "two arrays a pass");
  if (tid % kMaxExperts < p.E) {
#pragma unroll
    for (int i = tid; i < kActiveArrays * kMaxExperts; i += kThreads)
      reinterpret_cast<int*>(&s.act)[i] = p.plan[PLAN_WORDS + i];
  }
  for (int a = tid; a < A; a += kThreads) {
    slot_s[a] = p.slot[a];
    row_s[a] = p.row[a];
    wgt_s[a] = p.wgt[a];
  }
  __syncthreads();
  const int active = s.plan[PLAN_ACTIVE], q = s.plan[PLAN_LENGTH], items = s.plan[PLAN_ITEMS];
  const int tiles = ceil_div(p.H, L::kTile);
  const Active& act = s.act;

  T* out = static_cast<T*>(p.out);
  const bool add = p.T <= kAddTokens;  // this kernel also adds the parts up
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (items == 0) {  // no expert has a column (or all were refused): the sum is empty
    if (!add) return;
    for (long long i = blockIdx.x * static_cast<long long>(kThreads) + tid;
         i < static_cast<long long>(p.T) * p.H; i += static_cast<long long>(gridDim.x) * kThreads)
      out[i / p.H * p.ldo + i % p.H] = from_f<T>(0.f);
    return;
  }

  const int team = wid / kTeam, tt = tid % kTeamThreads;
  // Eight column tiles (1 KB of a row) at a time: neighbouring teams read
  // neighbouring pieces, and the tiles finish one block after another, so that
  // only the last block's final sums have nothing to overlap.
  const int me = blockIdx.x * kTeams + team, teams = gridDim.x * kTeams;
  auto unit = [&](int n) {
    const int i = me + n * teams;
    const int block = i / (8 * items), r = i - block * 8 * items;
    const int nb = min(8, tiles - 8 * block), it = r / nb;
    Unit u;
    u.e = find_item(act.item, active, it);
    const int width = act.width[u.e], j = it - act.item[u.e];
    const int ns = ceil_div(ceil_div(width, kRound), q), pass = j / ns;
    u.tile = 8 * block + r - it * nb;
    u.slice = j - pass * ns;
    u.local = -1;
    u.count = min(act.n[u.e] - pass * TOK, TOK);
    u.row = act.base[u.e] + pass * TOK;
    u.begin = u.slice * q * kRound;
    u.strip.end = min(width, u.begin + q * kRound);
    down_strip<L>(u.strip, act, u.e, act.first[u.e] / gated, u.tile, p.H, p.shift);
    return u;
  };
  auto source = [&](const Unit& u) {
    return HiddenSource<T>{static_cast<const T*>(p.h), p.ldh, p.max_width, u.row};
  };
  float* red = reinterpret_cast<float*>(work + kRingBytes<L, NG>) + team * kRedFloats<L, NG>;
  const long long slice = static_cast<long long>(A) * p.H;
  const bool vec = (p.ldo & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  // threads that share a (token, column vector) of the final sum
  // (one pass over them then: they meet in shared memory)
  constexpr int kVecs = L::kTile / 4;
  const int share = p.T * kVecs > kTeamThreads / 2 ? 1
                    : kTeamThreads / (kVecs * (p.T == 1 ? 1 : p.T == 2 ? 2 : 4));
  const Matrix m{&p.map2, p.w2, p.s2, p.H, p.shift, 0};
  run_units<L, NG>(
      items * tiles > me ? ceil_div(items * tiles - me, teams) : 0, m, work, red, s, p.wait_ns, unit,
      source,
      [&](const Unit& u) {
        const int cols = p.H - u.tile * L::kTile;
        float* y = p.y + u.tile * L::kTile;
        // (with the remainders' columns, see HiddenSource)
        const bool split = sizeof(T) == 2 && u.count <= 4;
        auto down_sum = [&](int tok, int c) {
          float4 v = unit_sum<L, NG>(red, tok, c);
          if (split) add4(v, unit_sum<L, NG>(red, tok + 4, c));
          return v;
        };
        for (int j = tt; j < u.count * (L::kTile / 4); j += kTeamThreads) {
          const int tok = j / (L::kTile / 4), c = 4 * (j % (L::kTile / 4));
          if (c < cols)
            *reinterpret_cast<float4*>(y + u.slice * slice +
                                       static_cast<long long>(u.row + tok) * p.H + c) =
                down_sum(tok, c);
        }
        if (!add) return;
        team_sync(team);
        if (tt == 0) {
          // (after the team's sums, and before reading the other teams')
          s.last[team] = count_gpu(&p.ticket[u.tile]) == items - 1;
        }
        team_sync(team);
        if (!s.last[team]) return;
        // each thread's slots in order, two at a time, their parts in order (four or eight,
        // or several parts at once, are more loads in flight but more code to fetch: one token
        // 18.4 us with two, 18.9, 20.1; 5 tokens 69.2, 68.8, 72.2)
        const int lanes = kTeamThreads / share, part = tt / lanes;
        for (int j0 = 0; j0 < p.T * (L::kTile / 4); j0 += lanes) {  // (barriers inside)
          const int j = j0 + tt % lanes, t = j / (L::kTile / 4), c = 4 * (j % (L::kTile / 4));
          const bool in = t < p.T && c < cols;
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
          if (in) {
            for (int a0 = part; a0 < p.k; a0 += 2 * share) {
              const float* src[2];
              int parts[2];
              float4 v[2];
              int longest = 0;
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const int a = t * p.k + a0 + n * share;
                v[n] = make_float4(0.f, 0.f, 0.f, 0.f);
                parts[n] = 0;
                src[n] = y;
                if (a0 + n * share < p.k && slot_s[a] >= 0) {
                  parts[n] = ceil_div(ceil_div(act.width[slot_s[a]], kRound), q);
                  src[n] = y + static_cast<long long>(row_s[a]) * p.H + c;
                }
                longest = max(longest, parts[n]);
              }
#pragma unroll 1
              for (int z = 0; z < longest; ++z)
#pragma unroll
                for (int n = 0; n < 2; ++n)
                  if (z < parts[n])
                    add4(v[n], __ldcg(reinterpret_cast<const float4*>(src[n] + z * slice)));
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                // (an expert without columns adds nothing, whatever its weight)
                const float g = parts[n] ? wgt_s[t * p.k + a0 + n * share] : 0.f;
                o.x = fmaf(g, v[n].x, o.x);
                o.y = fmaf(g, v[n].y, o.y);
                o.z = fmaf(g, v[n].z, o.z);
                o.w = fmaf(g, v[n].w, o.w);
              }
            }
          }
          if (share > 1) {
            float4* sums = reinterpret_cast<float4*>(red);  // read above, before a barrier
            sums[tt] = o;
            team_sync(team);
            if (part == 0)
              for (int g = 1; g < share; ++g) add4(o, sums[tt + g * lanes]);
          }
          if (part == 0 && in) store4<T>(out + t * p.ldo + u.tile * L::kTile + c, o, vec);
        }
      });
  if (s.abort && lane == 0 && p.status) *p.status = kStatusTimeout;
}

// More than 8 tokens: the final sum as a kernel of its own.  (In the down kernel a
// team adds the tile that it finishes; at 64 tokens that is 40,000 cycles of it at
// the end, with the other teams idle.)  A block is a token's 1024 columns; slots in
// order, their parts in order.
constexpr int kSumThreads = 256;
template <typename L>
__global__ void __launch_bounds__(kSumThreads) few_sum_kernel(const __grid_constant__ LayerParams p) {
  using T = typename L::Elem;
  constexpr int kRound = kTeam * L::kStep;
  __shared__ int row_s[kMaxTopK], parts_s[kMaxTopK];
  __shared__ float wgt_s[kMaxTopK];
  const int t = blockIdx.y, tid = threadIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid < p.k) {
    const int a = t * p.k + tid, slot = p.slot[a];
    row_s[tid] = p.row[a];
    wgt_s[tid] = p.wgt[a];
    parts_s[tid] = 0;
    if (slot >= 0)
      parts_s[tid] = ceil_div(ceil_div(p.plan[PLAN_WORDS + 3 * kMaxExperts + slot], kRound),
                              p.plan[PLAN_LENGTH]);
  }
  __syncthreads();
  const int c = 4 * (blockIdx.x * kSumThreads + tid);
  if (c >= p.H) return;
  T* out = static_cast<T*>(p.out);
  const bool vec = (p.ldo & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  const long long slice = static_cast<long long>(p.T) * p.k * p.H;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int a = 0; a < p.k; ++a) {
    const float* y = p.y + static_cast<long long>(row_s[a]) * p.H + c;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int z = 0; z < parts_s[a]; ++z)
      add4(v, __ldcg(reinterpret_cast<const float4*>(y + z * slice)));
    // (an expert without columns adds nothing, whatever its weight)
    const float g = parts_s[a] ? wgt_s[a] : 0.f;
    o.x = fmaf(g, v.x, o.x);
    o.y = fmaf(g, v.y, o.y);
    o.z = fmaf(g, v.z, o.z);
    o.w = fmaf(g, v.w, o.w);
  }
  store4<T>(out + t * p.ldo + c, o, vec);
}

// ---- 4-bit products of rows grouped by expert --------------------------------
// The up or down product by itself: its units are (expert, 8 rows, tile, slice), the
// slices meet in the sum kernel, which also applies the activation and writes the zeros.
// Bound by the work a code, as the layer's 4-bit products: 192 rows on 64 experts of
// 1024 x 2048 take 37.2 us (1.8 TB/s); 6 rows on 16 small experts 10.3, two launches.
struct GroupParams {
  const void* x;
  long long ldx;
  long long rows;     // rows of x and of the output
  const void* w;
  const void* s;
  const int* tok_off;  // [E + 1]
  const int* tok_cnt;  // [E] or null
  const int* off;      // [E + 1]: columns of w (up) or rows of w (down)
  int E, H, total, max_width, act, down;
  int shift, blocks, groups;
  int* plan;           // [PLAN_WORDS], then n, base, width [E] of the active experts
  float* part;         // [slices][rows][ldp]: whole tiles
  long long ldp;
  int max_slices;
  void* out;
  long long ldo;
  int* status;
  unsigned long long wait_ns;
};

struct alignas(16) GroupSmem {
  Common c;
  int off[kMaxExperts + 1];
  int tok[kMaxExperts + 1];
  int cnt[kMaxExperts];
  int kb[kMaxExperts];  // as UpSmem's
  int sg[kMaxExperts];
  int fits[kMaxExperts];
  int row[kMaxExperts + 1];
};
static_assert(sizeof(GroupSmem) % 16 == 0, "16-byte vectors follow");

// ROWS: PackedRows for the down product, NoRows for up (a kilobyte of arguments is 0.7 us a
// launch on the host).
template <typename L, int NG, typename ROWS>
__global__ void __launch_bounds__(kThreads, 1)
    few_group_kernel(const __grid_constant__ GroupParams p, const __grid_constant__ ROWS rows) {
  using T = typename L::Elem;
  constexpr int TOK = L::template kTokens<NG>, kRound = kTeam * L::kStep;
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* work = raw;
  GroupSmem& s = *reinterpret_cast<GroupSmem*>(raw + kWorkBytes<L, NG>);
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int e = tid; e <= p.E; e += kThreads) {
    s.off[e] = p.off[e];
    s.tok[e] = p.tok_off[e];
    if constexpr (std::is_same_v<ROWS, PackedRows>) s.row[e] = rows.row[e];
    if (e < p.E) {
      s.cnt[e] = p.tok_cnt ? p.tok_cnt[e] : 0x7fffffff;
      s.kb[e] = s.sg[e] = 0;
      s.fits[e] = 1;
    }
  }
  ring_init<L::template kDepth<NG>>(s.c);
  __syncthreads();
  const int outputs = 1 << outputs_log2<L>(p.act), teams = gridDim.x * kTeams;
  if (wid == 0) {  // as find_active
    if constexpr (std::is_same_v<ROWS, PackedRows>) {
      find_packed(rows.n > 0, s.row, s.off, p.E, p.total, p.act, p.shift, p.blocks, p.groups, s.kb,
                  s.sg, s.fits);
      __syncwarp();
    }
    int active = 0;
#pragma unroll 1
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      int n = 0, a = 0, w = 0, lo = 0;
      bool ok = true;
      if (e < p.E) {
        a = s.off[e];
        lo = s.tok[e];
        const int hi = s.tok[e + 1];
        ok = expert_width(a, s.off[e + 1], p.total, p.max_width, p.act, &w) && s.fits[e] && lo >= 0 &&
             hi >= lo && hi <= p.rows && s.cnt[e] >= 0;
        n = ok ? min(hi - lo, s.cnt[e]) : 0;
      }
      if (!ok && p.status && blockIdx.x == 0) *p.status = kStatusBadArg;
      const bool here = ok && n > 0 && w > 0;
      const unsigned who = __ballot_sync(0xffffffffu, here);
      const int at = active + __popc(who & ((1u << lane) - 1));
      active += __popc(who);
      if (here) {
        s.c.act.n[at] = n;
        s.c.act.base[at] = lo;
        s.c.act.first[at] = a;
        s.c.act.width[at] = w;
        s.c.act.kb[at] = s.kb[e];
        s.c.act.sg[at] = s.sg[e];
      }
    }
    __syncwarp();
    auto units = [&](int j, int len) {
      return ceil_div(s.c.act.n[j], TOK) *
             (p.down ? ceil_div(p.H, L::kTile) * ceil_div(ceil_div(s.c.act.width[j], kRound), len)
                     : ceil_div(s.c.act.width[j], outputs) * ceil_div(ceil_div(p.H, kRound), len));
    };
    int widest = 0;
    for (int j = lane; j < active; j += 32) widest = max(widest, s.c.act.width[j]);
    widest = __reduce_max_sync(0xffffffffu, widest);
    const int most = max(1, ceil_div(p.down ? widest : p.H, kRound));
    const int len = plan_length(most, teams, p.max_slices, 4, [&](int length) {
      int n = 0;
      for (int j = lane; j < active; j += 32) n += units(j, length);
      return static_cast<long long>(__reduce_add_sync(0xffffffffu, n));
    });
    int items = 0;
    for (int j0 = 0; j0 < active; j0 += 32) {
      const int j = j0 + lane;
      int total;
      const int before = items + warp_scan(j < active ? units(j, len) : 0, &total);
      items += total;
      if (j < active) s.c.act.item[j] = before;
    }
    if (lane == 0) {
      s.c.plan[0] = active;
      s.c.plan[1] = items;
      s.c.plan[2] = len;
    }
  }
  __syncthreads();
  const int active = s.c.plan[0], q = s.c.plan[2];
  const Active& act = s.c.act;
  if (blockIdx.x == gridDim.x - 1) {
    for (int j = tid; j < active; j += kThreads) {
      int* d = p.plan + PLAN_WORDS + j;
      d[0 * p.E] = act.n[j];
      d[1 * p.E] = act.base[j];
      d[2 * p.E] = act.width[j];
    }
    if (tid == 0) {
      p.plan[PLAN_ACTIVE] = active;
      p.plan[PLAN_LENGTH] = q;
    }
  }

  const int team = wid / kTeam, tt = tid % kTeamThreads;
  const int me = blockIdx.x * kTeams + team, units = s.c.plan[1];
  auto unit = [&](int n) {
    const int i = me + n * teams;
    Unit u;
    u.e = find_item(act.item, active, i);
    const int width = act.width[u.e], k_rows = p.down ? width : p.H;
    const int tiles = p.down ? ceil_div(p.H, L::kTile) : ceil_div(width, outputs);
    const int ns = ceil_div(ceil_div(k_rows, kRound), q), r = i - act.item[u.e];
    const int j = r / tiles, pass = j / ns;
    u.tile = r - j * tiles;
    u.slice = j - pass * ns;
    u.local = -1;
    u.count = min(act.n[u.e] - pass * TOK, TOK);
    u.row = act.base[u.e] + pass * TOK;
    u.begin = u.slice * q * kRound;
    u.strip.end = min(k_rows, u.begin + q * kRound);
    if (p.down)
      down_strip<L>(u.strip, act, u.e, act.first[u.e], u.tile, p.H, p.shift);
    else
      up_strip<L>(u.strip, act.first[u.e], width, p.act, u.tile, p.H, p.shift);
    return u;
  };
  auto source = [&](const Unit& u) {
    return RowSource<T>{static_cast<const T*>(p.x), p.ldx, nullptr, u.row};
  };
  float* red = reinterpret_cast<float*>(work + kRingBytes<L, NG>) + team * kRedFloats<L, NG>;
  const Matrix m{nullptr, p.w, p.s, p.down ? p.H : p.total, p.shift, p.act == ACT_SWIGLU};
  run_units<L, NG>(units > me ? ceil_div(units - me, teams) : 0, m, work, red, s.c, p.wait_ns, unit,
                   source,
                   [&](const Unit& u) {
                     float* dst = p.part +
                                  (static_cast<long long>(u.slice) * p.rows + u.row) * p.ldp +
                                  u.tile * L::kTile;
                     const int cols = static_cast<int>(p.ldp) - u.tile * L::kTile;
                     for (int j = tt; j < u.count * (L::kTile / 4); j += kTeamThreads) {
                       const int tok = j / (L::kTile / 4), c = 4 * (j % (L::kTile / 4));
                       if (c < cols)
                         *reinterpret_cast<float4*>(dst + tok * p.ldp + c) =
                             unit_sum<L, NG>(red, tok, c);
                     }
                   });
  if (s.c.abort && lane == 0 && p.status) *p.status = kStatusTimeout;
}

// Adds the slices, applies the activation, writes every element of the output:
// zero in rows and columns that belong to no expert.
template <typename L>
__global__ void __launch_bounds__(kThreads)
    few_group_sum_kernel(const __grid_constant__ GroupParams p) {
  using T = typename L::Elem;
  constexpr int kRound = kTeam * L::kStep;
  __shared__ int n_s[kMaxExperts], base_s[kMaxExperts], width_s[kMaxExperts], head[2];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int j = threadIdx.x; j < p.E; j += kThreads) {
    n_s[j] = p.plan[PLAN_WORDS + j];
    base_s[j] = p.plan[PLAN_WORDS + p.E + j];
    width_s[j] = p.plan[PLAN_WORDS + 2 * p.E + j];
  }
  if (threadIdx.x < 2) head[threadIdx.x] = p.plan[threadIdx.x];
  __syncthreads();
  const int active = head[PLAN_ACTIVE], q = head[PLAN_LENGTH];
  const int out_cols = p.down ? p.H : p.max_width, vecs = out_cols / 4;
  const long long slice = p.rows * p.ldp;
  const bool vec = (p.ldo & 3) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
  const bool gated = p.act == ACT_SWIGLU;
  for (long long i = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; i < p.rows * vecs;
       i += static_cast<long long>(gridDim.x) * kThreads) {
    const int row = static_cast<int>(i / vecs), c = 4 * static_cast<int>(i % vecs);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (active > 0) {
      const int e = find_item(base_s, active, row);
      if (row >= base_s[e] && row - base_s[e] < n_s[e] && (p.down || c < width_s[e])) {
        const int ns = ceil_div(ceil_div(p.down ? width_s[e] : p.H, kRound), q);
        const float* src = p.part + row * p.ldp +
                           (gated ? c / (L::kTile / 2) * L::kTile + c % (L::kTile / 2) : c);
        float4 b = v;
#pragma unroll 4
        for (int z = 0; z < ns; ++z) {
          add4(v, __ldcg(reinterpret_cast<const float4*>(src + z * slice)));
          if (gated) add4(b, __ldcg(reinterpret_cast<const float4*>(src + z * slice + L::kTile / 2)));
        }
        if (gated)
          v = make_float4(act_gated(v.x, b.x), act_gated(v.y, b.y), act_gated(v.z, b.z),
                          act_gated(v.w, b.w));
        else
          v = make_float4(act_plain(v.x, p.act), act_plain(v.y, p.act), act_plain(v.z, p.act),
                          act_plain(v.w, p.act));
      }
    }
    store4<T>(static_cast<T*>(p.out) + row * p.ldo + c, v, vec);
  }
}

// ---- host ---------------------------------------------------------------------
long long align_up(long long v, long long a) { return (v + a - 1) / a * a; }

struct LayerPlan {
  long long plan, slot, row, wgt, ticket, sel, u, h, y, bytes;
  long long ldu;
  int slices;
};

// Columns of a product's partial sums: whole tiles of either size.
long long padded_columns(long long width, int act) {
  const int n = act == ACT_SWIGLU ? kMaxTile / 2 : kMaxTile;
  return (width + n - 1) / n * kMaxTile;
}

// Slices of a reduction the workspace holds: 64 MB of partial sums, or one slice.
int slice_limit(long long floats) {
  const long long n = (64ll << 20) / (4 * (floats > 0 ? floats : 1));
  return static_cast<int>(n < 1 ? 1 : n > kMaxSlices ? kMaxSlices : n);
}

LayerPlan layer_plan(int T, int H, int k, int max_width, int act) {
  LayerPlan p{};
  const long long A = static_cast<long long>(T) * k;
  p.ldu = padded_columns(max_width, act);
  p.slices = slice_limit(A * (p.ldu > H ? p.ldu : H));
  long long at = 0;
  auto take = [&](long long bytes) {
    const long long here = at;
    at = align_up(at + bytes, 128);
    return here;
  };
  p.plan = take(4ll * PLAN_WORDS + static_cast<long long>(sizeof(Active)));
  p.slot = take(4 * A);
  p.row = take(4 * A);
  p.wgt = take(4 * A);
  p.ticket = take(4ll * ceil_div(H, kMinTile));
  p.sel = take(4 * A);
  p.u = take(4 * p.slices * A * p.ldu);
  p.h = take(4 * A * max_width);  // two 16-bit values or one fp32
  p.y = take(4 * p.slices * A * H);
  p.bytes = at;
  return p;
}

int current_device() {
  int d = 0;
  return cudaGetDevice(&d) == cudaSuccess && d >= 0 && d < 64 ? d : -1;
}

// Shared memory above 48 KB has to be allowed once per kernel and device.
constexpr int kSmemMax = 227 * 1024;
template <typename K>
bool allow_smem(K* kernel, std::atomic<unsigned long long>& done, int device) {
  const unsigned long long bit = 1ull << device;
  if (done.load(std::memory_order_acquire) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax) !=
      cudaSuccess)
    return false;
  done.fetch_or(bit, std::memory_order_release);
  return true;
}

// CTAs of clusters of `size` that are resident together at one CTA an SM.
template <typename K>
int resident_ctas(K* kernel, std::atomic<int>* known, int size) {
  int n = known->load(std::memory_order_acquire);
  if (n > 0) return n;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(num_sms() / size * size));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemMax;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) return -1;
  if (n > num_sms() / size) n = num_sms() / size;
  known->store(n * size, std::memory_order_release);
  return n * size;
}

// CTAs a cluster of the up kernel.  Every cluster reads the whole router weight, so
// larger clusters read less of it; but 8 CTAs fit together on only 120 of 148 SMs
// (4: 132, 2: all).
int cluster_size(long long router_bytes) {
  // (5 tokens, 256 KB: 68.8, 71.4, 71.5 us with 2, 4, 8; one token on 4-bit experts, 1 MB:
  // 52.3, 44.2, 42.7)
  return router_bytes <= (256 << 10) ? 2 : router_bytes <= (512 << 10) ? 4 : 8;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  return fn;
}

// Boxes of 4 KB (gated: two of 2 KB side by side) of a contiguous weight.
bool weight_map(CUtensorMap* map, const void* w, int dtype, long long rows, long long cols,
                bool gated) {
  const auto fn = encode_tiled();
  if (!fn) return false;
  const int es = dtype == 2 ? 4 : 2;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols * es)};
  const cuuint32_t box[2] = {gated ? 32u : 64u, dtype == 2 ? 16u : 32u};
  const cuuint32_t step[2] = {1, 1};
  return fn(map,
            dtype == 2   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
            : dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                         : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            2, const_cast<void*>(w), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            dtype == 2 ? CU_TENSOR_MAP_SWIZZLE_NONE
            : gated    ? CU_TENSOR_MAP_SWIZZLE_64B
                       : CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// 4-bit products in tiles of 128 columns rather than 64: cheaper a weight, but a step
// takes twice as long, which shows where every team has one or two.  (64 / 128 columns:
// 33 tokens, 64 experts of 1024, 94 / 85 us; one token, 8 of up to 2048, 42.7 / 41.1; 6
// tokens, 11 of up to 336, 22.8 / 26.5.)
bool wide_tiles(long long experts, long long rows, long long cols) {
  return (rows < experts ? rows : experts) * cols >= 100 * 128;
}

template <typename L, int NG>
int launch_layer(LayerParams& p, const RowsOf<L>& rows2, cudaStream_t st) {
  static std::atomic<unsigned long long> up_ok{0}, down_ok{0};
  static std::atomic<int> resident[64][kMaxCluster + 1];
  const int dev = current_device();
  if (dev < 0) return kStatusCuda;
  auto* up = few_up_kernel<L, NG>;
  auto* down = few_down_kernel<L, NG>;
  if (!allow_smem(up, up_ok, dev) || !allow_smem(down, down_ok, dev)) return kStatusCuda;
  const int lde = ceil_div(p.E, 16) * 16, tiles = lde / 16, A = p.T * p.k;
  const int ksub = kWarps / tiles > 1 ? kWarps / tiles : 1;
  const size_t route = p.T > kAddTokens ? 0 : sizeof(float) * (1 + ksub) * p.T * lde;
  const size_t work = kWorkBytes<L, NG>;
  p.smem_work = static_cast<int>(route > work ? route : work);
  const size_t up_smem = p.smem_work + sizeof(UpSmem) + 6 * A;
  const size_t down_smem = work + sizeof(Common) + 12 * A;
  if (up_smem > kSmemMax || down_smem > kSmemMax) return kStatusUnsupported;
  using T = typename L::Elem;
  // (an fp32 router beside 16-bit x has its own kernel for any number of tokens: in the up
  // kernel the second form of the logits cost 33 tokens of 2048 84.6 -> 86.0 us unused)
  const bool router = p.T > kAddTokens || p.router_fp32;
  if (!router) p.sel = nullptr;
  p.cluster = router ? 1 : cluster_size(static_cast<long long>(p.E) * p.H * sizeof(T));
  const int n = resident_ctas(up, &resident[dev][p.cluster], p.cluster), sms = num_sms();
  if (n < 1) return kStatusCuda;
  p.down_teams = sms * kTeams;

  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cfg.attrs = attr;
  if (router) {
    static std::atomic<unsigned long long> router_ok[2];
    auto* kernel = p.router_fp32 ? few_router_kernel<T, float> : few_router_kernel<T, T>;
    if (!allow_smem(kernel, router_ok[p.router_fp32], dev)) return kStatusCuda;
    attr[1].val.clusterDim.x = kMaxCluster;
    cfg.gridDim = dim3(static_cast<unsigned>(ceil_div(p.T, kMaxCluster) * kMaxCluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(float) * (1 + ksub) * kMaxCluster * lde;
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) return kStatusCuda;
    attr[1].val.clusterDim.x = 1;
  }
  cfg.gridDim = dim3(static_cast<unsigned>(n));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = up_smem;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, up, p, rows2) != cudaSuccess) return kStatusCuda;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(sms));
  cfg.dynamicSmemBytes = down_smem;
  if (cudaLaunchKernelEx(&cfg, down, p) != cudaSuccess) return kStatusCuda;
  if (p.T > kAddTokens) {
    cfg.gridDim = dim3(static_cast<unsigned>(ceil_div(p.H, 4 * kSumThreads)),
                       static_cast<unsigned>(p.T));
    cfg.blockDim = dim3(kSumThreads);
    cfg.dynamicSmemBytes = 0;
    if (cudaLaunchKernelEx(&cfg, few_sum_kernel<L>, p) != cudaSuccess) return kStatusCuda;
  }
  return cudaPeekAtLastError() == cudaSuccess ? kStatusOk : kStatusCuda;
}

// 8 or 16 vectors a unit: 16 when an expert has more than about 6 rows on average (each
// further pass over an expert's weights reads them again, from L2).  4-bit products have 8:
// 128 columns of 16 vectors do not fit the registers.  fp32 has 4 (8 took 26 instead of 22 us
// at one token of 768, 161 instead of 152 at 6 rows each for 16 experts of 2048 x 1024).
template <typename L>
int layer_for_tokens(LayerParams& p, cudaStream_t st) {
  return p.T <= 8 || p.T * p.k <= 6 * p.E ? launch_layer<L, 1>(p, {}, st)
                                          : launch_layer<L, 2>(p, {}, st);
}

template <typename L, int NG, typename ROWS>
int launch_group(const GroupParams& p, const ROWS& rows, cudaStream_t st) {
  static std::atomic<unsigned long long> ok{0};
  const int dev = current_device();
  if (dev < 0) return kStatusCuda;
  auto* kernel = few_group_kernel<L, NG, ROWS>;
  auto* sum = few_group_sum_kernel<L>;
  if (!allow_smem(kernel, ok, dev)) return kStatusCuda;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(num_sms()));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kWorkBytes<L, NG> + sizeof(GroupSmem);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p, rows) != cudaSuccess) return kStatusCuda;
  const long long vecs = p.rows * ((p.down ? p.H : p.max_width) / 4);
  long long blocks = (vecs + kThreads - 1) / kThreads;
  if (blocks > 4ll * num_sms()) blocks = 4ll * num_sms();
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.dynamicSmemBytes = 0;
  if (cudaLaunchKernelEx(&cfg, sum, p) != cudaSuccess) return kStatusCuda;
  return cudaPeekAtLastError() == cudaSuccess ? kStatusOk : kStatusCuda;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int group_shift(int group) { return group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : 0; }

bool layer_sizes_ok(long long T, long long H, int E, int k, long long max_width, int act) {
  return T >= 0 && T <= kMaxTokens && H >= 16 && H % 16 == 0 && H <= kMaxWidth && E >= 1 &&
         E <= kMaxExperts && k >= 1 && k <= E && k <= kMaxTopK && max_width >= 16 &&
         max_width % 16 == 0 && max_width <= kMaxWidth && act >= 0 && act <= 2;
}

// A packed w2's segments from its row offsets (host; null: one segment of all rows), and
// its block rows and groups.
int packed_rows(const int32_t* off, int E, long long rows, int group, PackedRows* r,
                long long* blocks, long long* groups) {
  if (off == nullptr && E != 1) return kStatusBadArg;
  if (E < 1 || E > kMaxExperts) return kStatusBadArg;
  const int rc = int4_rows(rows, group, off, E, blocks, groups);
  if (rc != kStatusOk) return rc;
  r->n = E;
  for (int e = 0; e <= E; ++e) r->row[e] = off ? off[e] : e * static_cast<int>(rows);
  return kStatusOk;
}

constexpr long long kGroupHeader = 4 * (PLAN_WORDS + 3 * kMaxExperts);
static_assert(kGroupHeader % 128 == 0, "partial sums follow");

}  // namespace

long long few_tokens_workspace(long long T, long long H, int E, int k, long long max_width,
                               int act) {
  if (!layer_sizes_ok(T, H, E, k, max_width, act)) return -1;
  return layer_plan(static_cast<int>(T), static_cast<int>(H), k, static_cast<int>(max_width), act)
      .bytes;
}

namespace {

int run_layer(const void* x, long long T, long long ldx, long long H, const void* router,
              int router_dtype, int E, const void* w1, const void* s1, const void* w2,
              const void* s2, int group, long long blocks2, long long groups2,
              const PackedRows& rows2, long long total, const int* off, long long max_width, int k,
              int norm, int act, void* out, long long ldo, void* ws, long long ws_bytes, int dtype,
              int* status, cudaStream_t st) {
  if (!layer_sizes_ok(T, H, E, k, max_width, act)) return kStatusBadArg;
  if (T == 0) return kStatusOk;
  const int shift = group_shift(group);
  if (router_dtype != dtype && (shift == 0 || router_dtype != 2)) return kStatusUnsupported;
  const int per16 = dtype == 2 ? 4 : 8;  // elements of a 16-byte vector
  if (!x || !router || !w1 || !w2 || !off || !out || !ws || total < 16 || total % 16 != 0 ||
      total > (1ll << 30) || ldx < H || ldx % per16 != 0 || ldo < H || !aligned16(x) ||
      !aligned16(router) || !aligned16(w1) || !aligned16(w2) || (group != 0 && shift == 0) ||
      (shift && (!s1 || !s2 || !aligned16(s1) || !aligned16(s2) || blocks2 < 0 || groups2 < 0 ||
                 blocks2 > (1 << 30) || groups2 > (1 << 30))))
    return kStatusBadArg;
  const LayerPlan plan = layer_plan(static_cast<int>(T), static_cast<int>(H), k,
                                    static_cast<int>(max_width), act);
  if (ws_bytes < plan.bytes || !aligned16(ws)) return kStatusBadArg;
  unsigned char* b = static_cast<unsigned char*>(ws);
  LayerParams p{};
  p.x = x; p.ldx = ldx; p.router = router; p.router_fp32 = router_dtype == 2 && dtype != 2;
  p.w1 = w1; p.s1 = s1; p.w2 = w2; p.s2 = s2; p.off = off;
  p.T = static_cast<int>(T); p.H = static_cast<int>(H); p.E = E; p.k = k; p.norm = norm; p.act = act;
  p.total = static_cast<int>(total); p.max_width = static_cast<int>(max_width);
  p.shift = shift;
  p.blocks2 = static_cast<int>(blocks2); p.groups2 = static_cast<int>(groups2);
  p.out = out; p.ldo = ldo;
  p.sel = reinterpret_cast<int*>(b + plan.sel);
  p.plan = reinterpret_cast<int*>(b + plan.plan);
  p.slot = reinterpret_cast<int*>(b + plan.slot);
  p.row = reinterpret_cast<int*>(b + plan.row);
  p.wgt = reinterpret_cast<float*>(b + plan.wgt);
  p.ticket = reinterpret_cast<int*>(b + plan.ticket);
  p.u = reinterpret_cast<float*>(b + plan.u);
  p.ldu = plan.ldu;
  p.h = b + plan.h;
  p.ldh = dtype == 2 ? max_width : 2 * max_width;
  p.y = reinterpret_cast<float*>(b + plan.y);
  p.max_slices = plan.slices;
  p.status = status;
  p.wait_ns = wait_ns();
  if (shift) {
    const bool wide = wide_tiles(E, T * k, act == ACT_SWIGLU ? 2 * max_width : max_width);
    if (dtype == 0)
      return wide ? launch_layer<Int4<__nv_bfloat16, 128>, 1>(p, rows2, st)
                  : launch_layer<Int4<__nv_bfloat16, 64>, 1>(p, rows2, st);
    if (dtype == 1)
      return wide ? launch_layer<Int4<__half, 128>, 1>(p, rows2, st)
                  : launch_layer<Int4<__half, 64>, 1>(p, rows2, st);
    return kStatusUnsupported;
  }
  if (dtype < 0 || dtype > 2) return kStatusUnsupported;
  const bool gated = act == ACT_SWIGLU;
  if (!weight_map(&p.map1, w1, dtype, H, total, gated) ||
      !weight_map(&p.map2, w2, dtype, total / (gated ? 2 : 1), H, false))
    return kStatusCuda;
  if (dtype == 0) return layer_for_tokens<Dense16<__nv_bfloat16>>(p, st);
  if (dtype == 1) return layer_for_tokens<Dense16<__half>>(p, st);
  return launch_layer<Dense32, 1>(p, {}, st);
}

}  // namespace

int few_tokens(const void* x, long long T, long long ldx, long long H, const void* router, int E,
               const void* w1, const void* s1, const void* w2, const void* s2, int group,
               long long blocks2, long long groups2, long long total, const int* off,
               long long max_width, int k, int norm, int act, void* out, long long ldo, void* ws,
               long long ws_bytes, int dtype, int* status, cudaStream_t st) {
  const PackedRows unknown{};
  return run_layer(x, T, ldx, H, router, dtype, E, w1, s1, w2, s2, group, blocks2, groups2, unknown,
                   total, off, max_width, k, norm, act, out, ldo, ws, ws_bytes, dtype, status, st);
}

int few_tokens_int4(const void* x, long long T, long long ldx, long long H, const void* router,
                    int router_dtype, int E, const void* w1, const void* s1, const void* w2,
                    const void* s2, int group, const int32_t* rows2, long long total, const int* off,
                    long long max_width, int k, int norm, int act, void* out, long long ldo,
                    void* ws, long long ws_bytes, int dtype, int* status, cudaStream_t st) {
  PackedRows rows{};
  long long blocks = 0, groups = 0;
  if (act < 0 || act > 2 || total % (act == ACT_SWIGLU ? 32 : 16) != 0) return kStatusBadArg;
  const int rc = packed_rows(rows2, E, act == ACT_SWIGLU ? total / 2 : total, group, &rows, &blocks,
                             &groups);
  if (rc != kStatusOk) return rc;
  return run_layer(x, T, ldx, H, router, router_dtype, E, w1, s1, w2, s2, group, blocks, groups, rows,
                   total, off, max_width, k, norm, act, out, ldo, ws, ws_bytes, dtype, status, st);
}

long long grouped_int4_workspace(long long rows, long long H, long long max_width, int act,
                                 int down) {
  if (rows < 0 || rows > 65536 || H < 16 || H % 16 != 0 || H > kMaxWidth || max_width < 16 ||
      max_width % 16 != 0 || max_width > kMaxWidth || act < 0 || act > 2 || (down && act != 0))
    return -1;
  const long long cols = padded_columns(down ? H : max_width, act);
  return kGroupHeader + 4ll * slice_limit(rows * cols) * rows * cols;
}

namespace {

template <typename ROWS>
int group_for_type(const GroupParams& p, const ROWS& rows, bool wide, int dtype, cudaStream_t st) {
  if (dtype == 0)
    return wide ? launch_group<Int4<__nv_bfloat16, 128>, 1>(p, rows, st)
                : launch_group<Int4<__nv_bfloat16, 64>, 1>(p, rows, st);
  if (dtype == 1)
    return wide ? launch_group<Int4<__half, 128>, 1>(p, rows, st)
                : launch_group<Int4<__half, 64>, 1>(p, rows, st);
  return kStatusUnsupported;
}

int run_group(const void* x, long long rows, long long ldx, const void* w, const void* s,
              int group, long long blocks, long long groups, const PackedRows& rows_w, long long H,
              long long total, const int* tok_off, const int* off, const int* tok_cnt, int E,
              long long max_width, int act, int down, void* out, long long ldo, void* ws,
              long long ws_bytes, int dtype, int* status, cudaStream_t st) {
  const int shift = group_shift(group);
  const long long need = grouped_int4_workspace(rows, H, max_width, act, down);
  if (need < 0 || total < 16 || total % 16 != 0 || total > (1ll << 30) || E < 1 ||
      E > kMaxExperts || shift == 0 || blocks < 0 || groups < 0 || blocks > (1 << 30) ||
      groups > (1 << 30))
    return kStatusBadArg;
  if (rows == 0) return kStatusOk;
  if (!x || !w || !s || !tok_off || !off || !out || !ws || ldx < (down ? max_width : H) ||
      ldx % 8 != 0 || ldo < (down ? H : max_width) || !aligned16(x) || !aligned16(w) || !aligned16(s) ||
      !aligned16(ws) || ws_bytes < need)
    return kStatusBadArg;
  if (!down && (blocks < (H + 63) / 64 || groups < (H + group - 1) / group)) return kStatusBadArg;
  GroupParams p{};
  p.x = x; p.ldx = ldx; p.rows = rows; p.w = w; p.s = s;
  p.tok_off = tok_off; p.tok_cnt = tok_cnt; p.off = off;
  p.E = E; p.H = static_cast<int>(H); p.total = static_cast<int>(total);
  p.max_width = static_cast<int>(max_width); p.act = act; p.down = down;
  p.shift = shift; p.blocks = static_cast<int>(blocks); p.groups = static_cast<int>(groups);
  p.plan = static_cast<int*>(ws);
  p.part = reinterpret_cast<float*>(static_cast<unsigned char*>(ws) + kGroupHeader);
  p.ldp = padded_columns(down ? H : max_width, act);
  p.max_slices = slice_limit(rows * p.ldp);
  p.out = out; p.ldo = ldo; p.status = status; p.wait_ns = wait_ns();
  const bool wide = wide_tiles(E, rows, down ? H : act == ACT_SWIGLU ? 2 * max_width : max_width);
  return down ? group_for_type(p, rows_w, wide, dtype, st)
              : group_for_type(p, NoRows{}, wide, dtype, st);
}

}  // namespace

int grouped_int4(const void* x, long long rows, long long ldx, const void* w, const void* s,
                 int group, long long blocks, long long groups, long long H, long long total,
                 const int* tok_off, const int* off, const int* tok_cnt, int E,
                 long long max_width, int act, int down, void* out, long long ldo, void* ws,
                 long long ws_bytes, int dtype, int* status, cudaStream_t st) {
  const PackedRows unknown{};
  return run_group(x, rows, ldx, w, s, group, blocks, groups, unknown, H, total, tok_off, off,
                   tok_cnt, E, max_width, act, down, out, ldo, ws, ws_bytes, dtype, status, st);
}

int grouped_down_int4(const void* x, long long rows, long long ldx, const void* w, const void* s,
                      int group, const int32_t* rows_w, long long H, long long total,
                      const int* tok_off, const int* off, const int* tok_cnt, int E,
                      long long max_width, void* out, long long ldo, void* ws, long long ws_bytes,
                      int dtype, int* status, cudaStream_t st) {
  PackedRows r{};
  long long blocks = 0, groups = 0;
  const int rc = packed_rows(rows_w, E, total, group, &r, &blocks, &groups);
  if (rc != kStatusOk) return rc;
  return run_group(x, rows, ldx, w, s, group, blocks, groups, r, H, total, tok_off, off, tok_cnt, E,
                   max_width, ACT_NONE, 1, out, ldo, ws, ws_bytes, dtype, status, st);
}

}  // namespace moe
