// The MoE layer for a few tokens (decode), in two kernels, and the products of
// 4-bit expert weights with rows grouped by expert.
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
// -> sum is what costs, so there are two launches, no host step and no memset:
//   up kernel    Every 8-CTA cluster computes the routing for itself (each CTA
//                an eighth of the hidden size, the sums exchanged over
//                distributed shared memory): it costs one or two microseconds of
//                L2 reads and needs no launch and no grid-wide wait of its own.
//                Then the grid's teams of four warps share the units (expert,
//                64-column tile, slice of the reduction) and write fp32 partial
//                sums of u.
//   down kernel  The units (expert, slice of its width, 64-column tile of the
//                hidden size); the partial sums of u are added and activated as
//                they are loaded.  The team that finishes a column tile's last
//                unit (a counter per tile, zeroed by the up kernel) adds the
//                tile's partial sums in a fixed order, weights them and writes
//                the output: results do not depend on timing.
// Nothing waits in a loop: the only waits are hardware barriers and the grid
// dependency between the two launches.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "few_tokens.cuh"
#include "moe_internal.h"

namespace moe {
namespace {

namespace cg = cooperative_groups;
using namespace few;

constexpr int kMaxTokens = 64;    // one 64-bit mask of tokens an expert
constexpr int kMaxExperts = 256;
constexpr int kMaxTopK = 32;
constexpr int kCluster = 8;
constexpr int kThreads = 512;     // 16 warps: at 128 registers a thread the SM is full
constexpr int kWarps = kThreads / 32;
constexpr int kTeam = 4;          // warps that share a unit (they split its reduction)
constexpr int kTeams = kWarps / kTeam;
constexpr int kTile = 64;         // columns of a unit
constexpr int kRedLd = kTile + 4;
constexpr int kMaxSlices = 16;
constexpr int kMaxWidth = 32768;  // hidden size and expert width: item counts stay 32-bit

template <typename L, int NG>
struct Shape {
  static constexpr int kTok = 8 * NG;
};
template <int NG>
struct Shape<Dense32, NG> {
  static constexpr int kTok = 4 * NG;
};

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// ---- what both kernels of the layer know -----------------------------------
struct LayerParams {
  const void* x;
  long long ldx;
  const void* router;
  const void* w1;
  const void* s1;  // 4-bit weights: group scales
  const void* w2;
  const void* s2;
  const int* off;  // [E + 1] columns of w1
  int T, H, E, k, norm, act, total, max_width;
  int shift;                 // log2 of the group
  int blocks2, groups2;      // block rows and groups of the packed w2
  void* out;
  long long ldo;
  // workspace
  unsigned long long* mask;  // [E] tokens of each expert
  int* sel;                  // [T * k]
  float* wgt;                // [T * k]
  int* info;                 // [0]: slices of u
  int* ticket;               // [tiles of the hidden size]
  float* u;                  // [slices][T * k][ldu]
  long long ldu;
  float* y;                  // [slices][T * k][H]
  int max_slices;
  int* status;
};

// Per-expert numbers, in shared memory (16-byte vectors of floats follow them).
struct alignas(16) Meta {
  int n[kMaxExperts];      // rows (0 when the expert's offsets are refused)
  int base[kMaxExperts];   // first row in expert-sorted order
  int first[kMaxExperts];  // first column of w1 (layer: the offsets' own units)
  int width[kMaxExperts];  // intermediate width
  int item[kMaxExperts + 1];  // prefix of the work items
  int kb[kMaxExperts];     // packed w2: first block row, first group
  int sg[kMaxExperts];
  int scan[kWarps + 1];
};

// Exclusive prefix sum over the block's threads; every thread also gets the total.
__device__ __forceinline__ int block_scan(int v, int* buf, int* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int q = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += q;
  }
  __syncthreads();  // buf may still be read from a call before
  if (lane == 31) buf[w] = s;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    const int q = buf[i];
    before += i < w ? q : 0;
    all += q;
  }
  *total = all;
  return before + s - v;
}

// The expert whose items hold index i (item is an exclusive prefix, E + 1 long).
__device__ __forceinline__ int find_item(const int* item, int E, int i) {
  int lo = 0, hi = E - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (item[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void team_sync(int team) {
  asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(kTeam * 32) : "memory");
}

// Rounds (a step by each warp of a team) of a slice: enough slices that every
// team of the grid has a few units, and no more (a slice costs its partial
// sums); never more than the workspace holds.
__device__ __forceinline__ int slice_rounds(long long all_rounds, int most, int teams,
                                            int max_slices) {
  const int want = static_cast<int>(min(all_rounds / (4ll * teams), 1ll << 20));
  return max(max(want, 1), ceil_div(most, max_slices));
}

// Adds the team's partial sums and writes rows [0, count) x cols of the unit.
template <int TOK>
__device__ __forceinline__ void team_store(const float* red, int count, int cols, float* dst,
                                           long long ldd) {
  const int i0 = threadIdx.x % (kTeam * 32);
  for (int i = i0; i < TOK * (kTile / 4); i += kTeam * 32) {
    const int tok = i / (kTile / 4), c = 4 * (i % (kTile / 4));
    if (tok < count && c < cols) {
      const float* p = red + tok * kRedLd + c;
      float4 v = *reinterpret_cast<const float4*>(p);
#pragma unroll
      for (int w = 1; w < kTeam; ++w) {
        const float4 q = *reinterpret_cast<const float4*>(p + w * TOK * kRedLd);
        v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w;
      }
      *reinterpret_cast<float4*>(dst + static_cast<long long>(tok) * ldd + c) = v;
    }
  }
}

// Expert e's strip of 64 columns from `col` of a matrix whose reduction rows of
// this expert start at `row`, up to reduction row `end`.
template <typename L>
struct Strips;
template <typename T>
struct Strips<Dense16<T>> {
  static __device__ __forceinline__ typename Dense16<T>::Strip make(
      const void* w, const void*, long long ld, long long row, int, int, int, int col, int end,
      int cols, int) {
    return {static_cast<const T*>(w) + row * ld + col, ld, end, cols};
  }
};
template <>
struct Strips<Dense32> {
  static __device__ __forceinline__ Dense32::Strip make(const void* w, const void*, long long ld,
                                                        long long row, int, int, int, int col,
                                                        int end, int cols, int) {
    return {static_cast<const float*>(w) + row * ld + col, ld, end, cols};
  }
};
template <typename T>
struct Strips<Int4<T>> {
  static __device__ __forceinline__ typename Int4<T>::Strip make(
      const void* w, const void* sc, long long ld, long long, int kb, int sg, int groups, int col,
      int end, int cols, int shift) {
    const long long nb = ld / 16;
    return {static_cast<const uint4*>(w) + (kb * nb + col / 16) * 32, nb,
            static_cast<const T*>(sc) + static_cast<long long>(sg) * ld + col, ld, end, cols,
            shift, groups};
  }
};

// ---- routing --------------------------------------------------------------
// This CTA's partial logits over reduction range [k_lo, k_hi): log[t][E16].
template <typename T>
__device__ __forceinline__ void partial_logits(const LayerParams& p, int k_lo, int k_hi,
                                               float* part, float* log, int lde) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const T* x = static_cast<const T*>(p.x);
  const T* wr = static_cast<const T*>(p.router);
  const int tiles = lde / 16, ksub = max(1, kWarps / tiles);
  // 16 experts x all tokens an item; ksub warps split its reduction
  for (int item = wid; item < tiles * ksub; item += kWarps) {
    const int et = item % tiles, ks = item / tiles;
    const int e0 = et * 16 + g, e1 = e0 + 8;
    for (int tg0 = 0; tg0 < p.T; tg0 += 32) {
      float acc[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[n][c] = 0.f;
      constexpr int kBatch = 2;  // steps whose loads are issued together
      for (int k0 = k_lo + 32 * ks; k0 < k_hi; k0 += 32 * ksub * kBatch) {
        uint4 a[kBatch][2], b[kBatch][4];
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
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int t = tg0 + 8 * n + g;
            b[j][n] = in && t < p.T
                          ? *reinterpret_cast<const uint4*>(x + static_cast<long long>(t) * p.ldx + k)
                          : zero;
          }
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const uint32_t a0[4] = {a[j][0].x, a[j][1].x, a[j][0].y, a[j][1].y};
          const uint32_t a1[4] = {a[j][0].z, a[j][1].z, a[j][0].w, a[j][1].w};
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            if (tg0 + 8 * n < p.T) {
              mma<T>(acc[n], a0, b[j][n].x, b[j][n].y);
              mma<T>(acc[n], a1, b[j][n].z, b[j][n].w);
            }
          }
        }
      }
      // rows of the result are experts, columns tokens
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int t = tg0 + 8 * n + 2 * t4 + j;
          if (t < p.T) {
            part[(ks * p.T + t) * lde + e0] = acc[n][j];
            part[(ks * p.T + t) * lde + e1] = acc[n][j + 2];
          }
        }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.T * lde; i += kThreads) {
    float s = part[i];
    for (int q = 1; q < ksub; ++q) s += part[q * p.T * lde + i];
    log[i] = s;
  }
}

template <>
__device__ __forceinline__ void partial_logits<float>(const LayerParams& p, int k_lo, int k_hi,
                                                      float*, float* log, int lde) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const float* x = static_cast<const float*>(p.x);
  const float* wr = static_cast<const float*>(p.router);
  const int hi = min(k_hi, p.H);
  for (int e = wid; e < p.E; e += kWarps) {
    const float* row = wr + static_cast<long long>(e) * p.H;
    for (int t0 = 0; t0 < p.T; t0 += 8) {
      float acc[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = 0.f;
      for (int k = k_lo + 4 * lane; k < hi; k += 128) {
        const float4 w = *reinterpret_cast<const float4*>(row + k);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (t0 + j < p.T) {
            const float4 v =
                *reinterpret_cast<const float4*>(x + static_cast<long long>(t0 + j) * p.ldx + k);
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
        if (lane == 0 && t0 + j < p.T) log[(t0 + j) * lde + e] = acc[j];
      }
    }
  }
}

// Unsigned order of floats; NaN above all (torch.topk's order).  Never 0.
__device__ __forceinline__ unsigned order_key(float v) {
  if (isnan(v)) return 0xffffffffu;
  const unsigned b = __float_as_uint(v + 0.f);  // -0 equals 0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// One warp chooses the k experts of a token from its logits (value j of lane l
// is expert 32 j + l).  Lane s < k gets the s-th expert and its weight.
__device__ __forceinline__ void choose(const float (&v)[kMaxExperts / 32], int E, int k, int norm,
                                       int* sel, float* wgt) {
  const int lane = threadIdx.x & 31;
  unsigned key[kMaxExperts / 32];
#pragma unroll
  for (int j = 0; j < kMaxExperts / 32; ++j) key[j] = 32 * j + lane < E ? order_key(v[j]) : 0u;
  float mine = 0.f;
  int idx = 0;
  for (int s = 0; s < k; ++s) {
    unsigned best = 0;
#pragma unroll
    for (int j = 0; j < kMaxExperts / 32; ++j) best = max(best, key[j]);
    best = __reduce_max_sync(0xffffffffu, best);
    unsigned at = 0xffffffffu;
    float val = 0.f;
#pragma unroll
    for (int j = kMaxExperts / 32 - 1; j >= 0; --j)
      if (key[j] == best) {
        at = 32 * j + lane;
        val = v[j];
      }
    const unsigned e = __reduce_min_sync(0xffffffffu, at);  // ties: the lower index
    val = __shfl_sync(0xffffffffu, val, e & 31);
#pragma unroll
    for (int j = 0; j < kMaxExperts / 32; ++j)
      if (e == 32u * j + lane) key[j] = 0u;
    if (lane == s) {
      mine = val;
      idx = static_cast<int>(e);
    }
  }
  float w = 1.f / (1.f + expf(-mine));
  if (norm) {
    float sum = 0.f;  // in rank order
    for (int s = 0; s < k; ++s) sum += __shfl_sync(0xffffffffu, w, s);
    w = w / (sum + 1e-20f);
  }
  *sel = idx;
  *wgt = w;
}

// ---- the layer's per-expert numbers ----------------------------------------
// From the token masks (shared) and the offsets (global): rows, first rows,
// widths.  Offsets that leave the matrices, or are not in steps of 16, empty the
// expert and set the status word.
__device__ __forceinline__ void layer_meta(const LayerParams& p, const unsigned long long* mask,
                                           Meta& m) {
  const int e = threadIdx.x;
  const int gated = p.act == ACT_SWIGLU ? 2 : 1;
  int n = 0, a = 0, w = 0;
  bool ok = true;
  if (e < p.E) {
    n = __popcll(mask[e]);
    a = p.off[e];
    const int b = p.off[e + 1];
    ok = a >= 0 && b >= a && b <= p.total && a % (16 * gated) == 0 &&
         (b - a) % (16 * gated) == 0 && (b - a) / gated <= p.max_width;
    w = ok ? (b - a) / gated : 0;
  }
  int all;
  const int base = block_scan(n, m.scan, &all);
  int kb = 0, sg = 0;
  if (p.shift) {
    kb = block_scan(ceil_div(w, 64), m.scan, &all);
    sg = block_scan((w + (1 << p.shift) - 1) >> p.shift, m.scan, &all);
  }
  if (e < p.E) {
    // a packed w2 quantised for other offsets
    if (p.shift && (kb + ceil_div(w, 64) > p.blocks2 ||
                    sg + ((w + (1 << p.shift) - 1) >> p.shift) > p.groups2))
      ok = false;
    if (!ok && p.status && blockIdx.x == 0) *p.status = kStatusBadArg;
    m.n[e] = ok ? n : 0;
    m.base[e] = base;
    m.first[e] = a;
    m.width[e] = ok ? w : 0;
    m.kb[e] = kb;
    m.sg[e] = sg;
  }
}

// ---- up kernel ---------------------------------------------------------------
struct alignas(16) UpSmem {
  Meta m;
  unsigned long long mask[kMaxExperts];
  int sel[kMaxTokens * kMaxTopK];
  float wgt[kMaxTokens * kMaxTopK];
  int list[kMaxTokens * kMaxTopK];  // token of each expert-sorted row
};

static_assert(sizeof(Meta) % 16 == 0 && sizeof(UpSmem) % 16 == 0, "16-byte vectors follow");

template <typename L, int NG>
__global__ void __launch_bounds__(kThreads, 1) few_up_kernel(const LayerParams p) {
  using T = typename L::Elem;
  constexpr int TOK = Shape<L, NG>::kTok;
  extern __shared__ __align__(16) unsigned char raw[];
  UpSmem& s = *reinterpret_cast<UpSmem*>(raw);
  const int lde = ceil_div(p.E, 16) * 16;
  float* log = reinterpret_cast<float*>(raw + sizeof(UpSmem));
  float* part = log + p.T * lde;  // the routing's partial sums, then the teams'
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;

  asm volatile("griddepcontrol.wait;" ::: "memory");
  // every block of this grid runs by the time the last one gets here
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // routing: an eighth of the hidden size, then tokens rank, rank + 8, ...
  const int per = ceil_div(ceil_div(p.H, 32), kCluster) * 32;
  partial_logits<T>(p, min(rank * per, p.H), min((rank + 1) * per, p.H), part, log, lde);
  for (int e = tid; e < p.E; e += kThreads) s.mask[e] = 0;
  cluster.sync();
  for (int t = rank + kCluster * wid; t < p.T; t += kCluster * kWarps) {
    float v[kMaxExperts / 32];
#pragma unroll
    for (int j = 0; j < kMaxExperts / 32; ++j) {
      const int e = 32 * j + lane;
      v[j] = 0.f;
      if (e < p.E) {
#pragma unroll
        for (int c = 0; c < kCluster; ++c)
          v[j] += cluster.map_shared_rank(log, c)[t * lde + e];
      }
    }
    int sel;
    float wgt;
    choose(v, p.E, p.k, p.norm, &sel, &wgt);
    if (lane < p.k) {
#pragma unroll
      for (int c = 0; c < kCluster; ++c) {
        cluster.map_shared_rank(s.sel, c)[t * p.k + lane] = sel;
        cluster.map_shared_rank(s.wgt, c)[t * p.k + lane] = wgt;
      }
    }
  }
  cluster.sync();

  const int A = p.T * p.k;
  for (int a = tid; a < A; a += kThreads) atomicOr(&s.mask[s.sel[a]], 1ull << (a / p.k));
  __syncthreads();
  layer_meta(p, s.mask, s.m);
  const int gated = p.act == ACT_SWIGLU ? 2 : 1;
  int items = 0;  // (pass, tile) pairs of this thread's expert
  if (tid < p.E)
    items = ceil_div(s.m.n[tid], TOK) * ceil_div(gated * s.m.width[tid], kTile);
  int U;
  const int before = block_scan(items, s.m.scan, &U);
  if (tid < p.E) s.m.item[tid] = before;
  for (int a = tid; a < A; a += kThreads) {
    const int e = s.sel[a], t = a / p.k;
    s.list[s.m.base[e] + __popcll(s.mask[e] & ((1ull << t) - 1))] = t;
  }
  const int teams = gridDim.x * kTeams;
  constexpr int kRound = kTeam * L::kStep;
  const int rounds = ceil_div(p.H, kRound);
  const int q = slice_rounds(static_cast<long long>(U) * rounds, rounds, teams, p.max_slices);
  const int slices = ceil_div(rounds, q);
  if (blockIdx.x == 0) {
    for (int e = tid; e < p.E; e += kThreads) p.mask[e] = s.mask[e];
    for (int a = tid; a < A; a += kThreads) {
      p.sel[a] = s.sel[a];
      p.wgt[a] = s.wgt[a];
    }
    for (int i = tid; i < ceil_div(p.H, kTile); i += kThreads) p.ticket[i] = 0;
    if (tid == 0) p.info[0] = slices;
  }
  __syncthreads();

  const int team = wid / kTeam, wr = wid % kTeam;
  float* red = part + team * (kTeam * TOK * kRedLd);
  for (int i = blockIdx.x * kTeams + team; i < U * slices; i += teams) {
    const int sl = i / U, r = i % U;
    const int e = find_item(s.m.item, p.E, r);
    const int cols = gated * s.m.width[e], tiles = ceil_div(cols, kTile);
    const int pass = (r - s.m.item[e]) / tiles, tile = (r - s.m.item[e]) % tiles;
    const int begin = sl * q * kRound, end = min(p.H, begin + q * kRound);
    const int count = min(s.m.n[e] - pass * TOK, TOK);
    const int row = s.m.base[e] + pass * TOK;
    const auto strip =
        Strips<L>::make(p.w1, p.s1, p.total, 0, 0, 0, (p.H + (1 << p.shift) - 1) >> p.shift,
                        s.m.first[e] + tile * kTile, end, cols - tile * kTile, p.shift);
    const RowSource<T> src{static_cast<const T*>(p.x), p.ldx, s.list, row};
    product<L, NG, kRound, kRedLd>(strip, src, count, begin + wr * L::kStep, lane,
                                   red + wr * TOK * kRedLd);
    team_sync(team);
    team_store<TOK>(red, count, cols - tile * kTile,
                    p.u + (static_cast<long long>(sl) * A + row) * p.ldu + tile * kTile, p.ldu);
    team_sync(team);
  }
}

// ---- down kernel -------------------------------------------------------------
struct alignas(16) DownSmem {
  Meta m;
  unsigned long long mask[kMaxExperts];
  int sel[kMaxTokens * kMaxTopK];
  float wgt[kMaxTokens * kMaxTopK];
  int last[kTeams];
};

static_assert(sizeof(DownSmem) % 16 == 0, "16-byte vectors follow");

template <typename L, int NG>
__global__ void __launch_bounds__(kThreads, 1) few_down_kernel(const LayerParams p) {
  using T = typename L::Elem;
  constexpr int TOK = Shape<L, NG>::kTok;
  extern __shared__ __align__(16) unsigned char raw[];
  DownSmem& s = *reinterpret_cast<DownSmem*>(raw);
  float* part = reinterpret_cast<float*>(raw + sizeof(DownSmem));
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int A = p.T * p.k, gated = p.act == ACT_SWIGLU ? 2 : 1;

  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int e = tid; e < p.E; e += kThreads) s.mask[e] = p.mask[e];
  for (int a = tid; a < A; a += kThreads) {
    s.sel[a] = p.sel[a];
    s.wgt[a] = p.wgt[a];
  }
  const int u_slices = p.info[0];
  __syncthreads();
  layer_meta(p, s.mask, s.m);
  constexpr int kRound = kTeam * L::kStep;
  int mine = 0, passes = 0, all_rounds, most;
  if (tid < p.E) {
    passes = ceil_div(s.m.n[tid], TOK);
    mine = ceil_div(s.m.width[tid], kRound);
  }
  block_scan(passes * mine, s.m.scan, &all_rounds);
  most = ceil_div(p.max_width, kRound);
  const int tiles = ceil_div(p.H, kTile), teams = gridDim.x * kTeams;
  const int q = slice_rounds(static_cast<long long>(all_rounds) * tiles, most, teams, p.max_slices);
  int items;
  const int before = block_scan(passes * ceil_div(mine, q), s.m.scan, &items);
  if (tid < p.E) s.m.item[tid] = before;
  __syncthreads();

  T* out = static_cast<T*>(p.out);
  if (items == 0) {  // no expert has a column (or all were refused): the sum is empty
    for (long long i = blockIdx.x * static_cast<long long>(kThreads) + tid;
         i < static_cast<long long>(p.T) * p.H; i += static_cast<long long>(gridDim.x) * kThreads)
      out[i / p.H * p.ldo + i % p.H] = from_f<T>(0.f);
    return;
  }

  const int team = wid / kTeam, wr = wid % kTeam;
  float* red = part + team * (kTeam * TOK * kRedLd);
  for (int i = blockIdx.x * kTeams + team; i < items * tiles; i += teams) {
    const int it = i / tiles, tile = i % tiles;
    const int e = find_item(s.m.item, p.E, it);
    const int width = s.m.width[e], ns = ceil_div(ceil_div(width, kRound), q);
    const int pass = (it - s.m.item[e]) / ns, sl = (it - s.m.item[e]) % ns;
    const int begin = sl * q * kRound, end = min(width, begin + q * kRound);
    const int count = min(s.m.n[e] - pass * TOK, TOK);
    const int row = s.m.base[e] + pass * TOK, cols = p.H - tile * kTile;
    const auto strip =
        Strips<L>::make(p.w2, p.s2, p.H, s.m.first[e] / gated, s.m.kb[e], s.m.sg[e],
                        (width + (1 << p.shift) - 1) >> p.shift, tile * kTile, end, cols, p.shift);
    const PartialSource<T> src{p.u, p.ldu, static_cast<long long>(A) * p.ldu, u_slices, row,
                               p.act, width};
    product<L, NG, kRound, kRedLd>(strip, src, count, begin + wr * L::kStep, lane,
                                   red + wr * TOK * kRedLd);
    team_sync(team);
    team_store<TOK>(red, count, cols,
                    p.y + (static_cast<long long>(sl) * A + row) * p.H + tile * kTile, p.H);
    team_sync(team);
    if (tid % (kTeam * 32) == 0) {
      __threadfence();  // the team's stores, before the count
      s.last[team] = atomicAdd(&p.ticket[tile], 1) == items - 1;
      __threadfence();  // and the other teams' stores, after it
    }
    team_sync(team);
    if (s.last[team]) {
      // token by token: slots in order, slices in order
      for (int j = tid % (kTeam * 32); j < p.T * (kTile / 4); j += kTeam * 32) {
        const int t = j / (kTile / 4), c = 4 * (j % (kTile / 4));
        if (c >= cols) continue;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int a = t * p.k; a < (t + 1) * p.k; ++a) {
          const int ex = s.sel[a];
          if (s.m.n[ex] == 0) continue;
          const int parts = ceil_div(ceil_div(s.m.width[ex], kRound), q);
          const int r = s.m.base[ex] + __popcll(s.mask[ex] & ((1ull << t) - 1));
          const float* y = p.y + static_cast<long long>(r) * p.H + tile * kTile + c;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int z = 0; z < parts; ++z) {
            const float4 d = __ldcg(
                reinterpret_cast<const float4*>(y + static_cast<long long>(z) * A * p.H));
            v.x += d.x; v.y += d.y; v.z += d.z; v.w += d.w;
          }
          const float w = s.wgt[a];
          o.x = fmaf(w, v.x, o.x);
          o.y = fmaf(w, v.y, o.y);
          o.z = fmaf(w, v.z, o.z);
          o.w = fmaf(w, v.w, o.w);
        }
        T* d = out + t * p.ldo + tile * kTile + c;
        d[0] = from_f<T>(o.x);
        d[1] = from_f<T>(o.y);
        d[2] = from_f<T>(o.z);
        d[3] = from_f<T>(o.w);
      }
    }
    team_sync(team);  // s.last and the partial sums are free again
  }
}

// ---- 4-bit products of rows grouped by expert --------------------------------
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
  int* info;           // [0]: rounds of a slice
  float* part;         // [slices][rows][ldp]
  long long ldp;
  int max_slices;
  void* out;
  long long ldo;
  int* status;
};

// Rows, widths and work items; the same numbers in both kernels.
__device__ __forceinline__ void group_meta(const GroupParams& p, Meta& m) {
  const int e = threadIdx.x;
  const int gated = p.act == ACT_SWIGLU ? 2 : 1;
  int n = 0, a = 0, w = 0, lo = 0;
  bool ok = true;
  if (e < p.E) {
    a = p.off[e];
    const int b = p.off[e + 1];
    lo = p.tok_off[e];
    const int hi = p.tok_off[e + 1];
    n = hi - lo;
    if (p.tok_cnt) n = min(n, p.tok_cnt[e]);
    ok = a >= 0 && b >= a && b <= p.total && a % (16 * gated) == 0 &&
         (b - a) % (16 * gated) == 0 && (b - a) / gated <= p.max_width && lo >= 0 && hi >= lo &&
         hi <= p.rows && n >= 0;
    w = ok ? (b - a) / gated : 0;
  }
  int kb = 0, sg = 0, all;
  if (p.down) {
    kb = block_scan(ceil_div(w, 64), m.scan, &all);
    sg = block_scan((w + (1 << p.shift) - 1) >> p.shift, m.scan, &all);
  }
  if (e < p.E) {
    if (p.down && (kb + ceil_div(w, 64) > p.blocks ||
                   sg + ((w + (1 << p.shift) - 1) >> p.shift) > p.groups))
      ok = false;
    if (!ok && p.status && blockIdx.x == 0) *p.status = kStatusBadArg;
    m.n[e] = ok ? n : 0;
    m.base[e] = lo;
    m.first[e] = a;
    m.width[e] = ok ? w : 0;
    m.kb[e] = kb;
    m.sg[e] = sg;
  }
  __syncthreads();
}

template <typename L, int NG>
__global__ void __launch_bounds__(kThreads, 1) few_group_kernel(const GroupParams p) {
  using T = typename L::Elem;
  constexpr int TOK = Shape<L, NG>::kTok;
  constexpr int kRound = kTeam * L::kStep;
  extern __shared__ __align__(16) unsigned char raw[];
  Meta& m = *reinterpret_cast<Meta*>(raw);
  float* part = reinterpret_cast<float*>(raw + sizeof(Meta));
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  group_meta(p, m);
  const int gated = p.act == ACT_SWIGLU ? 2 : 1;
  int passes = 0, mine = 0, tiles_e = 0, all;
  if (tid < p.E) {
    passes = ceil_div(m.n[tid], TOK);
    tiles_e = ceil_div(p.down ? p.H : gated * m.width[tid], kTile);
    mine = ceil_div(p.down ? m.width[tid] : p.H, kRound);
  }
  block_scan(passes * tiles_e * mine, m.scan, &all);
  const int teams = gridDim.x * kTeams;
  const int q = slice_rounds(all, ceil_div(p.down ? p.max_width : p.H, kRound), teams, p.max_slices);
  int U;
  const int before = block_scan(passes * tiles_e * ceil_div(mine, q), m.scan, &U);
  if (tid < p.E) m.item[tid] = before;
  if (blockIdx.x == 0 && tid == 0) p.info[0] = q;
  __syncthreads();

  const int team = wid / kTeam, wr = wid % kTeam;
  float* red = part + team * (kTeam * TOK * kRedLd);
  for (int i = blockIdx.x * kTeams + team; i < U; i += teams) {
    const int e = find_item(m.item, p.E, i);
    const int width = m.width[e];
    const int n_cols = p.down ? p.H : gated * width, k_rows = p.down ? width : p.H;
    const int tiles = ceil_div(n_cols, kTile), ns = ceil_div(ceil_div(k_rows, kRound), q);
    const int r = i - m.item[e];
    const int tile = r % tiles, pass = r / tiles / ns, sl = r / tiles % ns;
    const int begin = sl * q * kRound, end = min(k_rows, begin + q * kRound);
    const int count = min(m.n[e] - pass * TOK, TOK);
    const int row = m.base[e] + pass * TOK, cols = n_cols - tile * kTile;
    const auto strip = p.down
        ? Strips<L>::make(p.w, p.s, p.H, m.first[e], m.kb[e], m.sg[e],
                          (width + (1 << p.shift) - 1) >> p.shift, tile * kTile, end, cols, p.shift)
        : Strips<L>::make(p.w, p.s, p.total, 0, 0, 0, (p.H + (1 << p.shift) - 1) >> p.shift,
                          m.first[e] + tile * kTile, end, cols, p.shift);
    const RowSource<T> src{static_cast<const T*>(p.x), p.ldx, nullptr, row};
    product<L, NG, kRound, kRedLd>(strip, src, count, begin + wr * L::kStep, lane,
                                   red + wr * TOK * kRedLd);
    team_sync(team);
    team_store<TOK>(red, count, cols,
                    p.part + (static_cast<long long>(sl) * p.rows + row) * p.ldp + tile * kTile,
                    p.ldp);
    team_sync(team);
  }
}

// Adds the slices, applies the activation, writes every element of the output:
// zero in rows and columns that belong to no expert.
template <typename L>
__global__ void __launch_bounds__(kThreads) few_group_sum_kernel(const GroupParams p) {
  using T = typename L::Elem;
  constexpr int kRound = kTeam * L::kStep;
  __shared__ Meta m;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  group_meta(p, m);
  const int q = p.info[0];
  const int out_cols = p.down ? p.H : p.max_width, vec = out_cols / 4;
  const long long stride = static_cast<long long>(p.rows) * p.ldp;
  for (long long i = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; i < p.rows * vec;
       i += static_cast<long long>(gridDim.x) * kThreads) {
    const long long row = i / vec;
    const int c = 4 * static_cast<int>(i % vec);
    // the last expert that starts at or before this row (empty ones share a start)
    int e = 0;
    for (int step = kMaxExperts / 2; step > 0; step >>= 1)
      if (e + step < p.E && m.base[e + step] <= row) e += step;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    const int cols = p.down ? p.H : m.width[e];
    if (row >= m.base[e] && row < static_cast<long long>(m.base[e]) + m.n[e] && c < cols) {
      const int ns = ceil_div(ceil_div(p.down ? m.width[e] : p.H, kRound), q);
      const float* src = p.part + row * p.ldp + c;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
      for (int z = 0; z < ns; ++z) {
        const float4 d = __ldcg(reinterpret_cast<const float4*>(src + z * stride));
        a.x += d.x; a.y += d.y; a.z += d.z; a.w += d.w;
        if (p.act == ACT_SWIGLU) {
          const float4 f = __ldcg(reinterpret_cast<const float4*>(src + z * stride + m.width[e]));
          b.x += f.x; b.y += f.y; b.z += f.z; b.w += f.w;
        }
      }
      if (p.act == ACT_SWIGLU) {
        v[0] = act_gated(a.x, b.x); v[1] = act_gated(a.y, b.y);
        v[2] = act_gated(a.z, b.z); v[3] = act_gated(a.w, b.w);
      } else {
        v[0] = act_plain(a.x, p.act); v[1] = act_plain(a.y, p.act);
        v[2] = act_plain(a.z, p.act); v[3] = act_plain(a.w, p.act);
      }
    }
    T* d = static_cast<T*>(p.out) + row * p.ldo + c;
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j] = from_f<T>(v[j]);
  }
}

// ---- host ---------------------------------------------------------------------
long long align_up(long long v, long long a) { return (v + a - 1) / a * a; }

struct LayerPlan {
  long long mask, sel, wgt, info, ticket, u, y, bytes;
  long long ldu;
  int slices;
};

// Slices of a reduction the workspace holds: 64 MB of partial sums, or one slice.
int slice_limit(long long floats) {
  const long long n = (64ll << 20) / (4 * (floats > 0 ? floats : 1));
  return static_cast<int>(n < 1 ? 1 : n > kMaxSlices ? kMaxSlices : n);
}

LayerPlan layer_plan(int T, int H, int E, int k, int max_width, int act) {
  LayerPlan p{};
  const long long A = static_cast<long long>(T) * k;
  p.ldu = static_cast<long long>(act == ACT_SWIGLU ? 2 : 1) * max_width;
  p.slices = slice_limit(A * (p.ldu > H ? p.ldu : H));
  long long at = 0;
  auto take = [&](long long bytes) {
    const long long here = at;
    at = align_up(at + bytes, 128);
    return here;
  };
  p.mask = take(8ll * E);
  p.sel = take(4 * A);
  p.wgt = take(4 * A);
  p.info = take(16);
  p.ticket = take(4ll * ceil_div(H, kTile));
  p.u = take(4 * p.slices * A * p.ldu);
  p.y = take(4 * p.slices * A * H);
  p.bytes = at;
  return p;
}

int current_device() {
  int d = 0;
  return cudaGetDevice(&d) == cudaSuccess && d >= 0 && d < 64 ? d : -1;
}

// Shared memory above 48 KB has to be allowed once per kernel and device.
template <typename K>
bool allow_smem(K* kernel, std::atomic<unsigned long long>& done, int device) {
  const unsigned long long bit = 1ull << device;
  if (done.load(std::memory_order_acquire) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) !=
      cudaSuccess)
    return false;
  done.fetch_or(bit, std::memory_order_release);
  return true;
}

// 8-CTA clusters that are resident together at one CTA an SM.
template <typename K>
int resident_clusters(K* kernel, std::atomic<int>* known, int device, size_t smem) {
  int n = known[device].load(std::memory_order_acquire);
  if (n > 0) return n;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(num_sms() / kCluster * kCluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) return -1;
  if (n > num_sms() / kCluster) n = num_sms() / kCluster;
  known[device].store(n, std::memory_order_release);
  return n;
}

template <typename L, int NG>
int launch_layer(const LayerParams& p, cudaStream_t st) {
  static std::atomic<unsigned long long> up_ok{0}, down_ok{0};
  static std::atomic<int> clusters[64];
  constexpr int TOK = Shape<L, NG>::kTok;
  const int dev = current_device();
  if (dev < 0) return kStatusCuda;
  auto* up = few_up_kernel<L, NG>;
  auto* down = few_down_kernel<L, NG>;
  if (!allow_smem(up, up_ok, dev) || !allow_smem(down, down_ok, dev)) return kStatusCuda;
  const int lde = ceil_div(p.E, 16) * 16, tiles = lde / 16;
  const int ksub = kWarps / tiles > 1 ? kWarps / tiles : 1;
  const size_t red = sizeof(float) * kWarps * TOK * kRedLd;
  const size_t part = sizeof(float) * ksub * p.T * lde;
  const size_t up_smem = sizeof(UpSmem) + sizeof(float) * p.T * lde + (red > part ? red : part);
  const size_t down_smem = sizeof(DownSmem) + red;
  const int n = resident_clusters(up, clusters, dev, 227 * 1024);
  if (n < 1) return kStatusCuda;

  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(n * kCluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = up_smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, up, p) != cudaSuccess) return kStatusCuda;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(num_sms()));
  cfg.dynamicSmemBytes = down_smem;
  if (cudaLaunchKernelEx(&cfg, down, p) != cudaSuccess) return kStatusCuda;
  return cudaPeekAtLastError() == cudaSuccess ? kStatusOk : kStatusCuda;
}

template <typename L>
int layer_for_tokens(const LayerParams& p, cudaStream_t st) {
  return p.T <= 8 ? launch_layer<L, 1>(p, st) : launch_layer<L, 2>(p, st);
}

template <typename L, int NG>
int launch_group(const GroupParams& p, cudaStream_t st) {
  static std::atomic<unsigned long long> ok{0};
  const int dev = current_device();
  if (dev < 0) return kStatusCuda;
  auto* kernel = few_group_kernel<L, NG>;
  auto* sum = few_group_sum_kernel<L>;
  if (!allow_smem(kernel, ok, dev)) return kStatusCuda;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(num_sms()));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Meta) + sizeof(float) * kWarps * Shape<L, NG>::kTok * kRedLd;
  cfg.stream = st;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) return kStatusCuda;
  const long long vecs = p.rows * ((p.down ? p.H : p.max_width) / 4);
  long long blocks = (vecs + kThreads - 1) / kThreads;
  if (blocks > 4ll * num_sms()) blocks = 4ll * num_sms();
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.dynamicSmemBytes = 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
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

}  // namespace

long long few_tokens_workspace(long long T, long long H, int E, int k, long long max_width,
                               int act) {
  if (!layer_sizes_ok(T, H, E, k, max_width, act)) return -1;
  return layer_plan(static_cast<int>(T), static_cast<int>(H), E, k, static_cast<int>(max_width), act)
      .bytes;
}

int few_tokens(const void* x, long long T, long long ldx, long long H, const void* router, int E,
               const void* w1, const void* s1, const void* w2, const void* s2, int group,
               long long blocks2, long long groups2, long long total, const int* off,
               long long max_width, int k, int norm, int act, void* out, long long ldo, void* ws,
               long long ws_bytes, int dtype, int* status, cudaStream_t st) {
  if (!layer_sizes_ok(T, H, E, k, max_width, act)) return kStatusBadArg;
  if (T == 0) return kStatusOk;
  const int shift = group_shift(group);
  const int per16 = dtype == 2 ? 4 : 8;  // elements of a 16-byte vector
  if (!x || !router || !w1 || !w2 || !off || !out || !ws || total < 16 || total % 16 != 0 ||
      total > (1ll << 30) || ldx < H || ldx % per16 != 0 || ldo < H || !aligned16(x) ||
      !aligned16(router) || !aligned16(w1) || !aligned16(w2) || (group != 0 && shift == 0) ||
      (shift && (!s1 || !s2 || !aligned16(s1) || !aligned16(s2) || blocks2 < 0 || groups2 < 0 ||
                 blocks2 > (1 << 30) || groups2 > (1 << 30))))
    return kStatusBadArg;
  const LayerPlan plan = layer_plan(static_cast<int>(T), static_cast<int>(H), E, k,
                                    static_cast<int>(max_width), act);
  if (ws_bytes < plan.bytes || !aligned16(ws)) return kStatusBadArg;
  unsigned char* b = static_cast<unsigned char*>(ws);
  LayerParams p{};
  p.x = x; p.ldx = ldx; p.router = router;
  p.w1 = w1; p.s1 = s1; p.w2 = w2; p.s2 = s2; p.off = off;
  p.T = static_cast<int>(T); p.H = static_cast<int>(H); p.E = E; p.k = k; p.norm = norm; p.act = act;
  p.total = static_cast<int>(total); p.max_width = static_cast<int>(max_width);
  p.shift = shift;
  p.blocks2 = static_cast<int>(blocks2); p.groups2 = static_cast<int>(groups2);
  p.out = out; p.ldo = ldo;
  p.mask = reinterpret_cast<unsigned long long*>(b + plan.mask);
  p.sel = reinterpret_cast<int*>(b + plan.sel);
  p.wgt = reinterpret_cast<float*>(b + plan.wgt);
  p.info = reinterpret_cast<int*>(b + plan.info);
  p.ticket = reinterpret_cast<int*>(b + plan.ticket);
  p.u = reinterpret_cast<float*>(b + plan.u);
  p.ldu = plan.ldu;
  p.y = reinterpret_cast<float*>(b + plan.y);
  p.max_slices = plan.slices;
  p.status = status;
  if (shift) {
    if (dtype == 0) return layer_for_tokens<Int4<__nv_bfloat16>>(p, st);
    if (dtype == 1) return layer_for_tokens<Int4<__half>>(p, st);
    return kStatusUnsupported;
  }
  if (dtype == 0) return layer_for_tokens<Dense16<__nv_bfloat16>>(p, st);
  if (dtype == 1) return layer_for_tokens<Dense16<__half>>(p, st);
  if (dtype == 2) return launch_layer<Dense32, 2>(p, st);
  return kStatusUnsupported;
}

long long grouped_int4_workspace(long long rows, long long cols) {
  if (rows < 0 || rows > 65536 || cols < 16 || cols % 16 != 0 || cols > 2 * kMaxWidth) return -1;
  return 128 + 4ll * slice_limit(rows * cols) * rows * cols;
}

int grouped_int4(const void* x, long long rows, long long ldx, const void* w, const void* s,
                 int group, long long blocks, long long groups, long long H, long long total,
                 const int* tok_off, const int* off, const int* tok_cnt, int E,
                 long long max_width, int act, int down, void* out, long long ldo, void* ws,
                 long long ws_bytes, int dtype, int* status, cudaStream_t st) {
  const int shift = group_shift(group);
  const int gated = act == ACT_SWIGLU ? 2 : 1;
  const long long cols = down ? H : gated * max_width, in = down ? max_width : H;
  if (rows < 0 || rows > 65536 || H < 16 || H % 16 != 0 || H > kMaxWidth || total < 16 ||
      total % 16 != 0 || total > (1ll << 30) || E < 1 || E > kMaxExperts || max_width < 16 ||
      max_width % 16 != 0 || max_width > kMaxWidth || act < 0 || act > 2 || (down && act != 0) ||
      shift == 0 || blocks < 0 || groups < 0 || blocks > (1 << 30) || groups > (1 << 30))
    return kStatusBadArg;
  if (rows == 0) return kStatusOk;
  if (!x || !w || !s || !tok_off || !off || !out || !ws || ldx < in || ldx % 8 != 0 ||
      ldo < (down ? H : max_width) || !aligned16(x) || !aligned16(w) || !aligned16(s) ||
      !aligned16(ws) || ws_bytes < grouped_int4_workspace(rows, cols))
    return kStatusBadArg;
  GroupParams p{};
  p.x = x; p.ldx = ldx; p.rows = rows; p.w = w; p.s = s;
  p.tok_off = tok_off; p.tok_cnt = tok_cnt; p.off = off;
  p.E = E; p.H = static_cast<int>(H); p.total = static_cast<int>(total);
  p.max_width = static_cast<int>(max_width); p.act = act; p.down = down;
  p.shift = shift; p.blocks = static_cast<int>(blocks); p.groups = static_cast<int>(groups);
  p.info = static_cast<int*>(ws);
  p.part = reinterpret_cast<float*>(static_cast<unsigned char*>(ws) + 128);
  p.ldp = cols;
  p.max_slices = slice_limit(rows * cols);
  p.out = out; p.ldo = ldo; p.status = status;
  if (dtype == 0)
    return rows <= 8 ? launch_group<Int4<__nv_bfloat16>, 1>(p, st)
                     : launch_group<Int4<__nv_bfloat16>, 2>(p, st);
  if (dtype == 1)
    return rows <= 8 ? launch_group<Int4<__half>, 1>(p, st) : launch_group<Int4<__half>, 2>(p, st);
  return kStatusUnsupported;
}

}  // namespace moe
