// 4-bit weights with group scales: quantising, packing given codes, and back.
//
// A weight [K, N] is cut into groups of G rows (32, 64 or 128) in each column;
// w is held as (q - 8) s with q in 0..15:
//   s = round(amax / 7) to the storage type,  q = 8 + clamp(rint(w / s), -8, 7).
// Groups start anew in each segment of rows (an expert's rows of w2), so none
// spans two experts; the last group of a segment may be shorter.  A group whose
// amax is 0 (or whose scale rounds to 0) is all q = 8; one that holds a NaN or an
// infinity gets a NaN or infinite scale and reads back as NaN.
//
// Packed layout: blocks of 64 rows x 16 columns in 512 bytes, block rows of N / 16
// blocks, every segment starting a new block row.  Lane l = 4 g + t of a warp
// owns 16 bytes of a block; bits 3 + 4 j (and 19 + 4 j, around the end) of its word s
// are rows 32 (s / 2) + 8 t + 4 (s % 2) + 2 (j / 2) and the next, column 2 g + j % 2: a
// product loads its fragments as they lie, 512 contiguous bytes a warp, and gets the
// codes to the top of 16-bit mantissas by rotating (few_tokens.cuh).
//
// All three are one pass over memory (2.5 bytes a weight at 16 bits).
// A CTA takes 128 rows x 64 columns.  Quantising, a thread holds 4 rows x 8 columns
// (four 16-byte loads, 16 KB in flight a CTA), which are exactly four words of the
// packed layout; only the group maxima and the finished words go through shared memory.
// A 2048 x 65536 bf16 weight: quantising 81 us (4.2 TB/s; four fifths of the issue slots:
// a maximum, a conversion and a rounding a weight), back 65 us (5.2 TB/s, four fifths of it
// writes: filling the output alone takes 72 us with the library's fill), codes packed in
// 58 us.
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "few_tokens.cuh"
#include "moe_internal.h"

namespace moe {
namespace {

using few::from_f;
using few::to_f;

constexpr int kMaxSegments = 256;
constexpr int kRows = 128, kCols = 64, kThreadsQ = 256;
constexpr int kLd = kCols + 2;

// Segments by value: first row, first 128-row chunk, first block row, first group.
struct Segments {
  int n;
  int row[kMaxSegments + 1];
  int chunk[kMaxSegments + 1];
  int block[kMaxSegments + 1];
  int group[kMaxSegments + 1];
};

struct Where {
  int row, rows;   // this chunk's rows
  int block, group;  // its first block row and group
};

__device__ __forceinline__ Where locate(const Segments& s, int chunk, int shift) {
  int lo = 0, hi = s.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s.chunk[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  const int c = chunk - s.chunk[lo];
  const int row = s.row[lo] + c * kRows;
  return {row, min(kRows, s.row[lo + 1] - row), s.block[lo] + c * (kRows / 64),
          s.group[lo] + (c * kRows >> shift)};
}

// Where a word holds the code of its row i (0..3) and column c (0, 1).
__device__ __forceinline__ int bit(int i, int c) {
  return 3 + 4 * (c + 2 * (i >> 1)) + 16 * (i & 1);
}
__device__ __forceinline__ uint32_t place(uint32_t code, int i, int c) {
  return __funnelshift_l(code, code, bit(i, c));
}

// The integer nearest to w / s, ties to even, exactly: the quotient's own rounding (w / s,
// or w times the rounded reciprocal: off by less than one either way) is undone by the
// remainder, which fp32 holds without error.
constexpr float kMagic = 12582912.f;  // 1.5 x 2^23: adding it rounds to integers
__device__ __forceinline__ float exact_nearest(float w, float s, float quotient) {
  const float q = (quotient + kMagic) - kMagic;
  const float r = fmaf(-q, s, w), half = 0.5f * s;
  const bool odd = (__float_as_uint(q + kMagic) & 1u) != 0;
  const bool move = fabsf(r) > half || (fabsf(r) == half && odd);
  return move ? q + (r < 0.f ? -1.f : 1.f) : q;
}

// The same for weights and scales of 16 bits, from the reciprocal of the scale.  Both
// have at most 11 significant bits, so a quotient is either halfway between integers
// or at least 2^-12 from it; w * inv is within 2^-19 of the quotient; rounding it to
// steps of 2^-13 first therefore gives halfway exactly when it is, and the second
// rounding sends that to even.
//
// The result is the bits of kMagic + the integer: its low bits are the integer's, in two's
// complement.
__device__ __forceinline__ uint32_t nearest(float w, float inv) {
  const float step = 1536.f;  // 1.5 x 2^10: the sum's last place is 2^-13
  return __float_as_uint(fmaf(w, inv, step) + (kMagic - step));
}

// Maxima of two pairs of magnitudes of 16 bits, a NaN above all.
template <typename T>
__device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t pair_max<__nv_bfloat16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                       *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
template <>
__device__ __forceinline__ uint32_t pair_max<__half>(uint32_t a, uint32_t b) {
  const __half2 m =
      __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}

// rows x 64 columns of a row-major matrix into shared memory, zeros beyond.
template <typename T>
__device__ __forceinline__ void load_tile(const T* w, long long ld, int row, int rows, int col,
                                          int cols, T* tile) {
  constexpr int V = 16 / sizeof(T), PER = kCols / V, N = kRows * PER / kThreadsQ;
  uint4 v[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int i = threadIdx.x + j * kThreadsQ, r = i / PER, c = V * (i % PER);
    v[j] = r < rows && c < cols
               ? few::ld_stream(w + static_cast<long long>(row + r) * ld + col + c)
               : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int i = threadIdx.x + j * kThreadsQ, r = i / PER, c = V * (i % PER);
    const T* e = reinterpret_cast<const T*>(&v[j]);
#pragma unroll
    for (int x = 0; x < V; ++x) tile[r * kLd + c + x] = e[x];
  }
}

// 8 values of a row as floats.
template <typename T>
struct Eight {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p, bool ok) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
      v[i] = ok ? few::ld_stream(p + 16 / sizeof(T) * i) : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    const float2 f = few::unpack2<std::conditional_t<sizeof(T) == 4, __half, T>>(w[i / 2]);
    return i & 1 ? f.y : f.x;
  }
  __device__ __forceinline__ uint32_t pair(int j) const {  // 16-bit types
    return reinterpret_cast<const uint32_t*>(v)[j];
  }
};

// T: type of the weights, S: type of the scales.
template <typename T, typename S>
__global__ void __launch_bounds__(kThreadsQ)
    quantize_kernel(const T* __restrict__ w, long long ld, int N, const Segments seg, int shift,
                    uint4* __restrict__ packed, S* __restrict__ scales) {
  __shared__ __align__(16) uint32_t words[2 * 4 * 32 * 4];
  __shared__ unsigned amax[4][kCols];  // of 32 rows each
  __shared__ __align__(16) float scale[4][kCols], inverse[4][kCols];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const Where at = locate(seg, blockIdx.x, shift);
  const int col = blockIdx.y * kCols, cols = min(kCols, N - col);
  // warp: 32 rows (part) x 32 columns; lane: rows 4 r .. + 3, columns c .. c + 7
  const int part = wid & 3, r = lane >> 2, c = 32 * (wid >> 2) + 8 * (lane & 3);
  Eight<T> v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 32 * part + 4 * r + i;
    v[i].load(w + static_cast<long long>(at.row + row) * ld + col + c, row < at.rows && c < cols);
  }
  if constexpr (sizeof(T) == 4) {
    unsigned m[8];  // order of the bits of |w|: a NaN above all
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) m[j] = max(m[j], __float_as_uint(v[i].get(j)) & 0x7fffffffu);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) m[j] = max(m[j], __shfl_xor_sync(0xffffffffu, m[j], o));
    }
    unsigned mine = m[0];  // lane r keeps column c + r
#pragma unroll
    for (int j = 1; j < 8; ++j) mine = r == j ? m[j] : mine;
    amax[part][c + r] = mine;
  } else {
    uint32_t m[4];  // pairs of columns
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = v[0].pair(j) & 0x7fff7fffu;
#pragma unroll
      for (int i = 1; i < 4; ++i) m[j] = pair_max<T>(m[j], v[i].pair(j) & 0x7fff7fffu);
    }
    // each exchange halves the columns that a lane keeps: in the end 2 (r / 2) and the
    // next, of which it writes column r
    const bool up = r & 4, right = r & 2;
    uint32_t keep[2], one;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      keep[j] = up ? m[j + 2] : m[j];
      keep[j] = pair_max<T>(keep[j], __shfl_xor_sync(0xffffffffu, up ? m[j] : m[j + 2], 16));
    }
    one = right ? keep[1] : keep[0];
    one = pair_max<T>(one, __shfl_xor_sync(0xffffffffu, right ? keep[0] : keep[1], 8));
    one = pair_max<T>(one, __shfl_xor_sync(0xffffffffu, one, 4));
    const float2 f = few::unpack2<T>(one);
    amax[part][c + r] = __float_as_uint(r & 1 ? f.y : f.x);
  }
  __syncthreads();
  {
    const int cc = tid % kCols, pt = tid / kCols, per = 1 << (shift - 5);
    const int first = pt / per * per;
    unsigned m = amax[first][cc];
    for (int i = 1; i < per; ++i) m = max(m, amax[first + i][cc]);
    const S s = from_f<S>(__uint_as_float(m) / 7.f);
    const float f = to_f<S>(s);
    scale[pt][cc] = f;
    // 0: not finite, zero, below 2^-100, or so small in S that its rounding lets a
    // quotient past 7
    constexpr float kLeast = few::kIsBf16<S> ? 7.8886091e-31f : 6.1035156e-05f;
    inverse[pt][cc] = f >= kLeast && f <= 3.4028234e38f ? 1.f / f : 0.f;
    if (pt == first && 32 * first < at.rows && cc < cols)
      scales[static_cast<long long>(at.group + pt / per) * N + col + cc] = s;
  }
  __syncthreads();
  float inv[8];
  *reinterpret_cast<float4*>(inv) = *reinterpret_cast<const float4*>(&inverse[part][c]);
  *reinterpret_cast<float4*>(inv + 4) = *reinterpret_cast<const float4*>(&inverse[part][c + 4]);
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // columns c + 2 j, + 1: lane (g, t) of a block
    // Rows 0 and 2 (of both columns) make the low 16 bits, rows 1 and 3 the high ones:
    // four numbers -7..7 with weights 1, 16, 256, 4096, and 8 of each, modulo 2^16.
    uint32_t half[2];
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      uint32_t sum = 0x8888u;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int i = o + 2 * (n >> 1), x = n & 1;
        const float value = v[i].get(2 * j + x), f = inv[2 * j + x];
        uint32_t q;
        if constexpr (sizeof(T) == 4)
          q = __float_as_uint(exact_nearest(value, scale[part][c + 2 * j + x], value * f) + kMagic);
        else
          q = nearest(value, f);
        sum += q << 4 * n;
      }
      half[o] = sum;
    }
    uint32_t word = __byte_perm(half[0], half[1], 0x5410);
    word = __funnelshift_l(word, word, 3);
    if (inv[2 * j] == 0.f || inv[2 * j + 1] == 0.f) {  // a scale without its reciprocal
      word = 0;
#pragma unroll 1
      for (int k = 0; k < 8; ++k) {
        const float f = scale[part][c + 2 * j + (k & 1)];
        float value = 0.f;
#pragma unroll
        for (int n = 0; n < 8; ++n)
          if (n == k) value = v[n >> 1].get(2 * j + (n & 1));
        float q = 0.f;
        if (f > 0.f && f <= 3.4028234e38f)
          q = fminf(fmaxf(exact_nearest(value, f, value / f), -8.f), 7.f);
        word |= place(__float_as_uint(q + (kMagic + 8.f)) & 15u, k >> 1, k & 1);
      }
    }
    const int nb = c / 16, g = c % 16 / 2 + j, t = r >> 1, h = part & 1, kb = part >> 1;
    words[((kb * 4 + nb) * 32 + 4 * g + t) * 4 + 2 * h + (r & 1)] = word;
  }
  __syncthreads();
  // thread = (block row, block column, lane)
  const int nb = wid & 3, kb = wid >> 2;
  if (16 * nb >= cols || 64 * kb >= at.rows) return;
  packed[(static_cast<long long>(at.block + kb) * (N / 16) + col / 16 + nb) * 32 + lane] =
      reinterpret_cast<const uint4*>(words)[tid];
}

// Codes 0..15, one a byte, to the packed layout (rows beyond a segment: 8).
__global__ void __launch_bounds__(kThreadsQ)
    pack_kernel(const uint8_t* __restrict__ codes, long long ld, int N, const Segments seg,
                int shift, uint4* __restrict__ packed) {
  __shared__ __align__(16) uint8_t tile[kRows * kLd];
  const int tid = threadIdx.x;
  const Where at = locate(seg, blockIdx.x, shift);
  const int col = blockIdx.y * kCols, cols = min(kCols, N - col);
  load_tile(codes, ld, at.row, at.rows, col, cols, tile);
  __syncthreads();
  const int lane = tid & 31, nb = (tid >> 5) & 3, kb = tid >> 7;
  const int g = lane >> 2, t = lane & 3;
  if (16 * nb >= cols || 64 * kb >= at.rows) return;
  uint4 out;
  uint32_t* word = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int r0 = 64 * kb + 32 * (s >> 1) + 8 * t + 4 * (s & 1);
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t code = r0 + i < at.rows ? tile[(r0 + i) * kLd + 16 * nb + 2 * g + c] & 15u : 8u;
        v |= place(code, i, c);
      }
    word[s] = v;
  }
  packed[(static_cast<long long>(at.block + kb) * (N / 16) + col / 16 + nb) * 32 + lane] = out;
}

// (q - 8) s of two codes, `shift` bits up from bits 3..6 and 19..22 of the word, and two
// scales.  The codes become the mantissas of B + 8 q (B = 128 in bf16, 1024 in fp16); an
// eighth of that less B / 8 + 8 is q - 8 exactly, and the product with the scale is
// rounded once.
template <typename S>
__device__ __forceinline__ uint32_t two_values(uint32_t word, int shift, uint32_t s) {
  const uint32_t codes = __funnelshift_r(word, word, shift) & 0x00780078u;
  if constexpr (few::kIsBf16<S>) {
    const uint32_t b = codes | 0x43004300u;
    const __nv_bfloat162 q =
        __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&b), __float2bfloat162_rn(0.125f),
                __float2bfloat162_rn(-24.f));
    const __nv_bfloat162 r = __hmul2_rn(q, *reinterpret_cast<const __nv_bfloat162*>(&s));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const uint32_t b = codes | 0x64006400u;
    const __half2 q = __hfma2(*reinterpret_cast<const __half2*>(&b), __float2half2_rn(0.125f),
                              __float2half2_rn(-136.f));
    const __half2 r = __hmul2_rn(q, *reinterpret_cast<const __half2*>(&s));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

template <typename S>
__global__ void __launch_bounds__(kThreadsQ)
    dequantize_kernel(const uint4* __restrict__ packed, const S* __restrict__ scales, int N,
                      const Segments seg, int shift, S* __restrict__ out, long long ld) {
  // rows of 128 bytes, 16-byte chunks exchanged by row so that neither side conflicts
  __shared__ __align__(16) uint32_t tile[kRows * kCols / 2];
  const int tid = threadIdx.x;
  const Where at = locate(seg, blockIdx.x, shift);
  const int col = blockIdx.y * kCols, cols = min(kCols, N - col);
  const int lane = tid & 31, nb = (tid >> 5) & 3, kb = tid >> 7;
  const int g = lane >> 2, t = lane & 3;
  auto chunk = [](int row, int c) { return c ^ ((row >> 3 & 3) << 1); };
  if (16 * nb < cols && 64 * kb < at.rows) {
    const uint4 v = few::ld_stream(
        packed + (static_cast<long long>(at.block + kb) * (N / 16) + col / 16 + nb) * 32 + lane);
    const uint32_t* word = reinterpret_cast<const uint32_t*>(&v);
    uint32_t s2[2];  // two columns' scales of each 32-row half
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 64 * kb + 32 * h;
      const uint32_t two =
          r < at.rows ? *reinterpret_cast<const uint32_t*>(
                            scales + static_cast<long long>(at.group + (r >> shift)) * N + col +
                            16 * nb + 2 * g)
                      : 0u;
      s2[h] = two;
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int r0 = 64 * kb + 32 * (s >> 1) + 8 * t + 4 * (s & 1);
#pragma unroll
      for (int i = 0; i < 4; i += 2) {  // two rows of two columns
        uint32_t v[2];
#pragma unroll
        for (int c = 0; c < 2; ++c)
          v[c] = two_values<S>(word[s], 4 * (i + c),
                               __byte_perm(s2[s >> 1], 0, c ? 0x3232 : 0x1010));
#pragma unroll
        for (int n = 0; n < 2; ++n)
          tile[(r0 + i + n) * 32 + 4 * chunk(r0 + i + n, 2 * nb + (g >> 2)) + (g & 3)] =
              __byte_perm(v[0], v[1], n ? 0x7632 : 0x5410);
      }
    }
  }
  __syncthreads();
  constexpr int PER = kCols / 8;
#pragma unroll
  for (int j = 0; j < kRows * PER / kThreadsQ; ++j) {
    const int i = tid + j * kThreadsQ, r = i / PER, c = i % PER;
    if (r < at.rows && 8 * c < cols)
      __stcs(reinterpret_cast<uint4*>(out + static_cast<long long>(at.row + r) * ld + col + 8 * c),
             reinterpret_cast<const uint4*>(tile)[r * PER + chunk(r, c)]);
  }
}

int shift_of(int group) { return group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : 0; }

// false: not ascending multiples of 16 from 0 to K
bool make_segments(const int32_t* off, int n, long long K, int group, Segments& s) {
  if (K < 16 || K % 16 != 0 || K > (1ll << 30)) return false;
  if (off == nullptr) n = 1;
  if (n < 1 || n > kMaxSegments) return false;
  s.n = n;
  s.row[0] = s.chunk[0] = s.block[0] = s.group[0] = 0;
  for (int i = 0; i < n; ++i) {
    const long long a = off ? off[i] : 0, b = off ? off[i + 1] : K;
    if (a != s.row[i] || b < a || b > K || b % 16 != 0) return false;
    const int len = static_cast<int>(b - a);
    s.row[i + 1] = static_cast<int>(b);
    s.chunk[i + 1] = s.chunk[i] + (len + kRows - 1) / kRows;
    s.block[i + 1] = s.block[i] + (len + 63) / 64;
    s.group[i + 1] = s.group[i] + (len + group - 1) / group;
  }
  return s.row[n] == K;
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool sizes_ok(const Segments& s, long long N) {
  return N >= 16 && N % 16 == 0 && (N + kCols - 1) / kCols <= 65535 && s.chunk[s.n] >= 1;
}

}  // namespace

// Block rows and groups of a weight of K rows: negative on bad arguments.
int int4_rows(long long K, int group, const int32_t* off, int n, long long* blocks,
              long long* groups) {
  Segments s;
  if (shift_of(group) == 0 || !make_segments(off, n, K, group, s)) return kStatusBadArg;
  *blocks = s.block[s.n];
  *groups = s.group[s.n];
  return kStatusOk;
}

int int4_quantize(const void* w, long long K, long long N, long long ld, int w_dtype, int group,
                  const int32_t* off, int n, void* packed, void* scales, int s_dtype,
                  cudaStream_t st) {
  Segments s;
  const int shift = shift_of(group);
  if (!w || !packed || !scales || shift == 0 || !make_segments(off, n, K, group, s) ||
      !sizes_ok(s, N) || ld < N || ld % (w_dtype == 2 ? 4 : 8) != 0 || !aligned(w) ||
      !aligned(packed))
    return kStatusBadArg;
  const dim3 grid(static_cast<unsigned>(s.chunk[s.n]), static_cast<unsigned>((N + kCols - 1) / kCols));
  uint4* out = static_cast<uint4*>(packed);
  const int cols = static_cast<int>(N);
#define MOE_QUANTIZE(T, S)                                                        \
  quantize_kernel<T, S><<<grid, kThreadsQ, 0, st>>>(static_cast<const T*>(w), ld, cols, s, shift, \
                                                    out, static_cast<S*>(scales))
  if (w_dtype == 0 && s_dtype == 0)
    MOE_QUANTIZE(__nv_bfloat16, __nv_bfloat16);
  else if (w_dtype == 1 && s_dtype == 1)
    MOE_QUANTIZE(__half, __half);
  else if (w_dtype == 2 && s_dtype == 0)
    MOE_QUANTIZE(float, __nv_bfloat16);
  else if (w_dtype == 2 && s_dtype == 1)
    MOE_QUANTIZE(float, __half);
  else
    return kStatusUnsupported;
#undef MOE_QUANTIZE
  return cudaPeekAtLastError() == cudaSuccess ? kStatusOk : kStatusCuda;
}

int int4_pack(const uint8_t* codes, long long K, long long N, long long ld, int group,
              const int32_t* off, int n, void* packed, cudaStream_t st) {
  Segments s;
  const int shift = shift_of(group);
  if (!codes || !packed || shift == 0 || !make_segments(off, n, K, group, s) || !sizes_ok(s, N) ||
      ld < N || ld % 16 != 0 || !aligned(codes) || !aligned(packed))
    return kStatusBadArg;
  const dim3 grid(static_cast<unsigned>(s.chunk[s.n]), static_cast<unsigned>((N + kCols - 1) / kCols));
  pack_kernel<<<grid, kThreadsQ, 0, st>>>(codes, ld, static_cast<int>(N), s, shift,
                                          static_cast<uint4*>(packed));
  return cudaPeekAtLastError() == cudaSuccess ? kStatusOk : kStatusCuda;
}

int int4_dequantize(const void* packed, const void* scales, long long K, long long N, int group,
                    const int32_t* off, int n, void* out, long long ld, int dtype,
                    cudaStream_t st) {
  Segments s;
  const int shift = shift_of(group);
  if (!packed || !scales || !out || shift == 0 || !make_segments(off, n, K, group, s) ||
      !sizes_ok(s, N) || ld < N || ld % 8 != 0 || !aligned(packed) || !aligned(scales) ||
      !aligned(out))
    return kStatusBadArg;
  const dim3 grid(static_cast<unsigned>(s.chunk[s.n]), static_cast<unsigned>((N + kCols - 1) / kCols));
  const uint4* in = static_cast<const uint4*>(packed);
  const int cols = static_cast<int>(N);
  if (dtype == 0)
    dequantize_kernel<<<grid, kThreadsQ, 0, st>>>(in, static_cast<const __nv_bfloat16*>(scales),
                                                  cols, s, shift,
                                                  static_cast<__nv_bfloat16*>(out), ld);
  else if (dtype == 1)
    dequantize_kernel<<<grid, kThreadsQ, 0, st>>>(in, static_cast<const __half*>(scales), cols, s,
                                                  shift, static_cast<__half*>(out), ld);
  else
    return kStatusUnsupported;
  return cudaPeekAtLastError() == cudaSuccess ? kStatusOk : kStatusCuda;
}

}  // namespace moe
