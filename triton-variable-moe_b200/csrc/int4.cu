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
// All three are one pass over memory (2.5 bytes a weight at 16 bits) and HBM
// bound: a CTA takes 128 rows x 64 columns, 16 KB in flight in four vectors a
// thread, transposes through shared memory (row stride 33 words: conflict free)
// and writes one 16-byte vector a thread.
#include <cuda_runtime.h>

#include <cstdint>

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

// The integer nearest to w / s, ties to even, exactly: the quotient's own
// rounding is undone by the remainder, which fp32 holds without error.
__device__ __forceinline__ int nearest(float w, float s) {
  float q = rintf(w / s);
  const float r = fmaf(-q, s, w), half = 0.5f * s;
  const bool odd = (static_cast<int>(q) & 1) != 0;
  if (r > half || (r == half && odd)) q += 1.f;
  if (r < -half || (r == -half && odd)) q -= 1.f;
  return static_cast<int>(fminf(fmaxf(q, -8.f), 7.f));
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

// T: type of the weights, S: type of the scales.
template <typename T, typename S>
__global__ void __launch_bounds__(kThreadsQ)
    quantize_kernel(const T* __restrict__ w, long long ld, int N, const Segments seg, int shift,
                    uint4* __restrict__ packed, S* __restrict__ scales) {
  __shared__ __align__(16) T tile[kRows * kLd];
  __shared__ unsigned amax[4][kCols];  // of 32 rows each
  __shared__ float sc[4][kCols];
  const int tid = threadIdx.x;
  const Where at = locate(seg, blockIdx.x, shift);
  const int col = blockIdx.y * kCols, cols = min(kCols, N - col);
  load_tile(w, ld, at.row, at.rows, col, cols, tile);
  __syncthreads();
  {
    const int c = tid % kCols, part = tid / kCols;
    unsigned m = 0;  // order of the bits of |w|: a NaN above all
    for (int r = 0; r < 32; ++r)
      m = max(m, __float_as_uint(to_f<T>(tile[(32 * part + r) * kLd + c])) & 0x7fffffffu);
    amax[part][c] = m;
  }
  __syncthreads();
  {
    const int c = tid % kCols, part = tid / kCols, per = 1 << (shift - 5);
    const int first = part / per * per;
    unsigned m = amax[first][c];
    for (int i = 1; i < per; ++i) m = max(m, amax[first + i][c]);
    const S s = from_f<S>(__uint_as_float(m) / 7.f);
    sc[part][c] = to_f<S>(s);
    if (part == first && 32 * first < at.rows && c < cols)
      scales[static_cast<long long>(at.group + part / per) * N + col + c] = s;
  }
  __syncthreads();
  // thread = (block row, block column, lane)
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
        const int cc = 16 * nb + 2 * g + c;
        const float x = to_f<T>(tile[(r0 + i) * kLd + cc]), q = sc[(r0 + i) >> 5][cc];
        const int code = q > 0.f && q <= 3.4028234e38f ? nearest(x, q) + 8 : 8;
        v |= place(code, i, c);
      }
    word[s] = v;
  }
  packed[(static_cast<long long>(at.block + kb) * (N / 16) + col / 16 + nb) * 32 + lane] = out;
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

template <typename S>
__global__ void __launch_bounds__(kThreadsQ)
    dequantize_kernel(const uint4* __restrict__ packed, const S* __restrict__ scales, int N,
                      const Segments seg, int shift, S* __restrict__ out, long long ld) {
  __shared__ __align__(16) S tile[kRows * kLd];
  const int tid = threadIdx.x;
  const Where at = locate(seg, blockIdx.x, shift);
  const int col = blockIdx.y * kCols, cols = min(kCols, N - col);
  const int lane = tid & 31, nb = (tid >> 5) & 3, kb = tid >> 7;
  const int g = lane >> 2, t = lane & 3;
  if (16 * nb < cols && 64 * kb < at.rows) {
    const uint4 v = few::ld_stream(
        packed + (static_cast<long long>(at.block + kb) * (N / 16) + col / 16 + nb) * 32 + lane);
    const uint32_t* word = reinterpret_cast<const uint32_t*>(&v);
    float s2[2][2];  // of each 32-row half, each column
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = 64 * kb + 32 * h;
        s2[h][c] = r < at.rows ? to_f<S>(scales[static_cast<long long>(at.group + (r >> shift)) * N +
                                               col + 16 * nb + 2 * g + c])
                               : 0.f;
      }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int r0 = 64 * kb + 32 * (s >> 1) + 8 * t + 4 * (s & 1);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int q = static_cast<int>(__funnelshift_r(word[s], word[s], bit(i, c)) & 15u) - 8;
          tile[(r0 + i) * kLd + 16 * nb + 2 * g + c] =
              from_f<S>(static_cast<float>(q) * s2[s >> 1][c]);
        }
    }
  }
  __syncthreads();
  constexpr int V = 8, PER = kCols / V;
#pragma unroll
  for (int j = 0; j < kRows * PER / kThreadsQ; ++j) {
    const int i = tid + j * kThreadsQ, r = i / PER, c = V * (i % PER);
    if (r < at.rows && c < cols) {
      uint4 v;
      S* e = reinterpret_cast<S*>(&v);
#pragma unroll
      for (int x = 0; x < V; ++x) e[x] = tile[r * kLd + c + x];
      *reinterpret_cast<uint4*>(out + static_cast<long long>(at.row + r) * ld + col + c) = v;
    }
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
      !sizes_ok(s, N) || ld < N || ld % 8 != 0 || !aligned(packed) || !aligned(out))
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
