// Device pieces of the few-token kernels: a warp's product of a strip of weights (64 or
// 128 columns) with up to 8 * NG token vectors.
//
// With few rows per expert the products are bound by reading the weights once
// (at 8 tokens: 16 flops per 2-byte weight against the ~250 that would balance
// HBM and the tensor pipe), so what counts is bytes in flight and instructions a
// byte.  Every warp streams its own rows of a strip through a ring in shared
// memory, one bulk copy (4 KB: 32 rows x 64 columns of 16-bit weights) a step,
// issued by one lane; no other warp touches the ring, so the loop has no block
// barrier and the ring runs on into the warp's next strip.  The multiply is
// m16n8k16 with the weights as the 16-row operand and the tokens as its 8
// columns.  (Register double buffering instead of the ring held half the bytes in
// flight; per-lane asynchronous copies took five times the instructions: the
// 128-expert layer at 64 tokens ran 722 and 1580 us a call.)
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace moe {
namespace few {

// ------------------------------------------------------------------ numbers
template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f<__half>(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f<float>(float v) {
  return v;
}
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ float from_f<float>(float v) {
  return v;
}

template <typename T>
constexpr bool kIsBf16 = false;
template <>
constexpr bool kIsBf16<__nv_bfloat16> = true;

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// d = a (16 x 16) * b (16 x 8) + c, fp32 accumulation.
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1, const float (&c)[4]) {
  if constexpr (kIsBf16<T>)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]),
          "f"(c[2]), "f"(c[3]));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]),
          "f"(c[2]), "f"(c[3]));
}
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
  mma<T>(d, a, b0, b1, d);
}

// 16 bytes that are read once: past L1.
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// ------------------------------------------------------------- bulk copies
// Contiguous bytes to shared memory (addresses and size in multiples of 16).
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void box_load(uint32_t dst, const void* tmap, int c0, int c1,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(tmap), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("{ .reg .b64 st; mbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1; }" ::"r"(bar),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void ldsm_trans(uint32_t (&a)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
               : "r"(addr)
               : "memory");
}

// -------------------------------------------------------------- activations
enum Act : int { ACT_NONE = 0, ACT_RELU2 = 1, ACT_SWIGLU = 2 };

__device__ __forceinline__ float act_plain(float u, int act) {
  if (act == ACT_RELU2) {
    // relu keeps a NaN (fmaxf would drop it)
    const float r = u < 0.f ? 0.f : u;
    return r * r;
  }
  return u;
}
__device__ __forceinline__ float act_gated(float gate, float up) {
  return gate / (1.f + expf(-gate)) * up;
}

// ------------------------------------------------------------ token vectors
// The multiplied vectors.  A warp's lane g = lane / 4 holds rows g, g + 8, ..;
// lanes past the count repeat the last row (their columns of the product are not
// used), and elements past the reduction's end are zero (never read), so nothing
// beyond a vector enters a sum.

// Rows of a matrix of the storage type: the layer's tokens (through the list of the
// tokens of the expert-sorted rows), or the rows of a grouped product.
template <typename T>
struct RowSource {
  static constexpr int kParts = 1;  // 16-bit operands per value
  static constexpr int half = 0;
  const T* x;
  long long ld;
  const uint8_t* list;  // null: rows first, first + 1, ..
  int first;
  __device__ __forceinline__ const T* row(int i) const {
    return x + static_cast<long long>(list ? list[first + i] : first + i) * ld;
  }
};

// The layer's intermediate, already activated.  For 16-bit weights each fp32
// value is held as two 16-bit operands (value and remainder), multiplied one after
// the other: the intermediate is not rounded to the storage type's digits, and the
// second multiply is free beside the weight loads.  bf16 keeps 2^-16 of a value.
// fp16 keeps 2^-22 of it or 2^-25, whichever is more, as its smallest step is 2^-24:
// values below 2^-3 have fewer digits and those below 2^-25 are zero (the forward, one
// fp16 number, keeps 2^-11 or 2^-25; a scale a row would keep more, but its maximum is
// known only when the whole grid is done: a launch more).  In fp16 a value above 65504
// is infinite, as it is in the layer's forward, which stores it (and times 4-bit
// weights a NaN: see Int4).  A row: [values | remainders].
//
// A unit of up to 4 vectors holds their remainders in the instruction's other four
// columns (one multiply for both; `split`), and the sums of columns j and j + 4 are
// added at the end.
template <typename T>
struct HiddenSource {
  static constexpr int kParts = 2;
  const T* h;
  long long ld;
  int half;  // remainders this far behind the values
  int first;
  __device__ __forceinline__ const T* row(int i) const {
    return h + static_cast<long long>(first + i) * ld;
  }
};
template <typename T>
__device__ __forceinline__ void hidden_store4(T* row, int half, int c, const float (&v)[4]) {
  uint32_t hi[2], lo[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    hi[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    const float2 h = unpack2<T>(hi[i]);
    // an infinite or NaN value has no remainder
    lo[i] = pack2<T>(fabsf(h.x) <= 3.4e38f ? v[2 * i] - h.x : 0.f,
                     fabsf(h.y) <= 3.4e38f ? v[2 * i + 1] - h.y : 0.f);
  }
  *reinterpret_cast<uint2*>(row + c) = make_uint2(hi[0], hi[1]);
  *reinterpret_cast<uint2*>(row + half + c) = make_uint2(lo[0], lo[1]);
}
template <>
__device__ __forceinline__ void hidden_store4<float>(float* row, int, int c, const float (&v)[4]) {
  *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
}

// ------------------------------------------------------------------ weights
// A strip: reduction rows up to `end` of one expert's weights and a tile of its
// columns, in two halves: side by side, or (a gated activation) gate columns and the
// up columns they go with, `jump` further right.  `lo` and `hi` of each half's columns
// exist, in multiples of 16; the sums of others are meaningless and nobody reads them.
struct Strip {
  int row, col;        // matrix row of reduction row 0; first column
  int end;             // reduction rows
  int lo, hi, jump;
  int kb, sg, groups;  // 4-bit: first block row; first group, number of groups
};

// What a matrix is to the copies.
struct Matrix {
  const void* map;     // dense: tensor map (boxes of 64, gated 32, columns)
  const void* w;       // 4-bit: packed blocks, scales
  const void* scales;
  int cols;
  int shift;           // log2 of the group
  int gated;
};

// Where the copies of a dense strip are: the step at row k, then every `rows` further.
template <int STAGE>
struct BoxCursor {
  int col, jump, row;
  __device__ __forceinline__ void set(const Matrix&, const Strip& s, int k) {
    col = s.col;
    jump = s.jump;
    row = s.row + k;
  }
  template <int ROWS>
  __device__ __forceinline__ void next(const Matrix&) {
    row += ROWS;
  }
  __device__ __forceinline__ void issue(const Matrix& m, uint32_t stage, uint32_t bar) const {
    expect_bytes(bar, STAGE);
    box_load(stage, m.map, col, row, bar);
    if (m.gated) box_load(stage + STAGE / 2, m.map, col + jump, row, bar);
  }
};

// 16-bit weights, row-major.  One step is a box of 32 rows x 64 columns, 128-byte
// swizzled (gated: two of 32 columns, 64-byte swizzled).  Lane t = lane % 4 has
// reduction rows 16 s + 4 t .. + 3 as its k slots of multiply s: for t < 2 the
// first two as the instruction's slots 2t, 2t + 1 and the others as 2t + 8, 2t + 9,
// for t >= 2 the other way round, which makes the eight rows of each transposed
// 8 x 8 load different modulo 8 (no bank conflict) and a lane's token elements four
// in a row.
template <typename T>
struct Dense16 {
  using Elem = T;
  static constexpr int kTile = 64;  // columns of a strip
  static constexpr int kSums = 4;   // a lane's multiplies of 16 columns
  static constexpr int kStep = 32;
  static constexpr bool kPacked = false;
  static constexpr bool kGroups = true;  // vectors in groups of 8 columns, of which a unit
                                         // may have fewer
  static constexpr int kStage = 4096;  // bytes of a step in the ring
  template <int NG>
  static constexpr int kDepth = 2;     // steps in the ring
  template <int NG>
  static constexpr int kTokens = 8 * NG;
  // per-lane offsets into a stage
  struct Lane {
    uint32_t off[4];  // of multiply i's 16 columns
    uint32_t half;    // bytes of 16 rows
    __device__ __forceinline__ Lane(int lane, int gated) {
      const int mi = lane >> 3, j = lane & 7, t = j >> 1;
      const int row = 4 * t + 2 * ((mi >> 1) ^ (t >> 1)) + (j & 1);
      half = gated ? 1024 : 2048;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = 2 * i + (mi & 1);  // 8-column chunk
        off[i] = gated ? (c >> 2) * 2048 + row * 64 + (((c & 3) ^ (row >> 1 & 3)) << 4)
                       : row * 128 + ((c ^ (row & 7)) << 4);
      }
    }
  };
  using Cursor = BoxCursor<kStage>;
  // The vectors' elements of half h (16 rows) of a step.
  template <int NG, typename Src>
  struct Vectors {
    const T* r[NG];  // at the step's first row
    uint2 b[2][NG][Src::kParts];
    template <int G, int P>
    __device__ __forceinline__ void rows(const Src& src, int count, int k, int lane) {
      const int g = lane >> 2;
#pragma unroll
      for (int n = 0; n < G; ++n) r[n] = src.row(min(8 * n + g, count - 1)) + 4 * (lane & 3) + k;
      if (Src::kParts == 2 && P == 1)
        r[0] = src.row(min(g & 3, count - 1)) + (g & 4 ? src.half : 0) + 4 * (lane & 3) + k;
    }
    template <int G, int P>
    __device__ __forceinline__ void load(int h, const Src& src, int left, int lane) {
      if (16 * h >= left) return;
#pragma unroll
      for (int n = 0; n < G; ++n)
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const uint2 v = *reinterpret_cast<const uint2*>(r[n] + p * src.half + 16 * h);
          b[h][n][p] = (lane & 2) ? make_uint2(v.y, v.x) : v;
        }
    }
    template <int G>
    __device__ __forceinline__ void advance(int rows) {
#pragma unroll
      for (int n = 0; n < G; ++n) r[n] += rows;
    }
  };
  // One half of a step for the first G groups of vectors and P of their parts.
  template <int G, int P, int NG, typename Src>
  static __device__ __forceinline__ void half(int h, float (&acc)[4][NG][4], const Lane& l,
                                              const Matrix&, const Strip&, int left,
                                              uint32_t stage, int,
                                              const Vectors<NG, Src>& v) {
    if (16 * h >= left) return;  // rows beyond are another expert's
    uint32_t a[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ldsm_trans(a[i], stage + h * l.half + l.off[i]);
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int n = 0; n < G; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) mma<T>(acc[i][n], a[i], v.b[h][n][p].x, v.b[h][n][p].y);
  }
  // The lane's sums to (ADD: added to) red[token][64 columns], row stride LD.
  template <int G, int NG, int LD, bool ADD>
  static __device__ __forceinline__ void store(const float (&acc)[4][NG][4], int lane, float* red) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < G; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float* p = red + (8 * n + 2 * t + (c & 1)) * LD + 16 * i + 8 * (c >> 1) + g;
          *p = ADD ? *p + acc[i][n][c] : acc[i][n][c];
        }
  }
};

// 4-bit weights in the packed layout (see int4.cu): blocks of 64 rows x 16
// columns, 16 bytes a lane.  Word s of a lane's vector feeds the multiply of
// the block's rows 32 (s / 2) + 8t + 4 (s % 2) .. + 3; rotated right by 4 j, its bits
// 3..6 and 19..22 are the two codes of operand register j (columns 2g, 2g + 1 as the
// instruction's rows g and g + 8).
//
// With those bits as the top of a mantissa and a constant exponent, a code q is the
// 16-bit number B + 8 q (B = 128 in bf16, 1024 in fp16) after one rotation and one
// logic instruction for two codes.  What is wanted, 8 (q - 8), is that less
// B + 64, and the sum of (B + 64) x over the rows is the same for every column: one
// product with a constant operand gives it, and the sums start from its negative.
// (Subtracting in the operands instead is exact to the bit but costs another
// instruction for two codes, where the 1.7 codes a cycle and lane that HBM delivers
// leave 4 or 5.)  The fp32 sums carry terms of up to 31 + 24 = 55 (fp16: 143 + 136 =
// 279) scales times |x| whatever the code, so their error is a few 2^-22 of
// 55 (279) scale sum |x| and does not shrink with the weights: a column of codes 8 comes
// out at that error, not at zero (unless its scale is zero, as a quantised column of
// zeros has it).  An infinite vector element makes a NaN of every column it meets, and
// so can bf16 ones from 2^115 on: 192 of them times 32 rows reach fp32's end.  The
// sums of each
// group are scaled as they are added up, so the scales are never rounded into the
// weights.  One step is 64 rows of 128 columns: the work beside the codes themselves
// (copies, vectors, the constant product) is that of 64 columns, and was half of all;
// 64 columns where there are few units (see wide_tiles in few_tokens.cu).  33 tokens on
// 64 experts of 2048 x 1024 take 84 us, 1.7 TB/s: not the bytes, and no pipe is full
// either (ALU 50 to 58 %, issue slots 37 to 45 %); a warp's chain of load, rotate, mask,
// multiply and scale, with four warps a scheduler, and 10 us before the first product.
template <typename T, int TILE>
struct Int4 {
  using Elem = T;
  static constexpr int kTile = TILE;
  static constexpr int kSums = TILE / 16;
  static constexpr int kStep = 64;
  static constexpr bool kPacked = true;
  static constexpr bool kGroups = true;
  static constexpr int kScales = 32 * TILE;  // a step in the ring: weights, then the
  static constexpr int kStage = kScales + 4 * TILE;  // scales of two groups
  template <int NG>
  static constexpr int kDepth = 256 / TILE;
  template <int NG>
  static constexpr int kTokens = 8 * NG;
  struct Lane {
    __device__ __forceinline__ Lane(int, int) {}
  };
  struct Cursor {
    const char* w;
    const T* sc;
    int lo, hi, jump;
    int left;  // groups after this step's first
    __device__ __forceinline__ void set(const Matrix& m, const Strip& s, int k) {
      const long long nb = m.cols / 16;
      const int g = k >> m.shift;
      w = static_cast<const char*>(m.w) + ((s.kb + (k >> 6)) * nb + s.col / 16) * 512;
      sc = static_cast<const T*>(m.scales) + static_cast<long long>(s.sg + g) * m.cols + s.col;
      lo = s.lo;
      hi = s.hi;
      jump = s.jump;
      left = s.groups - g - 1;
    }
    template <int ROWS>
    __device__ __forceinline__ void next(const Matrix& m) {
      static_assert(ROWS % 128 == 0, "whole groups");
      const int g = ROWS >> m.shift;
      w += static_cast<long long>(m.cols) * (ROWS / 64 * 32);
      sc += static_cast<long long>(m.cols) * g;
      left -= g;
    }
    __device__ __forceinline__ void issue(const Matrix& m, uint32_t stage, uint32_t bar) const {
      // a second group in the step, unless the weight ends before it
      const bool two = m.shift == 5;
      const T* sd = left > 0 ? sc + m.cols : sc;
      const int n = lo + hi;
      expect_bytes(bar, (two ? 36 : 34) * n);
      if (m.gated) {
        bulk_load(stage, w, 32 * lo, bar);
        bulk_load(stage + kScales / 2, w + 32ll * jump, 32 * hi, bar);
        bulk_load(stage + kScales, sc, 2 * lo, bar);
        bulk_load(stage + kScales + TILE, sc + jump, 2 * hi, bar);
        if (two) {
          bulk_load(stage + kScales + 2 * TILE, sd, 2 * lo, bar);
          bulk_load(stage + kScales + 3 * TILE, sd + jump, 2 * hi, bar);
        }
      } else {
        bulk_load(stage, w, 32 * n, bar);
        bulk_load(stage + kScales, sc, 2 * n, bar);
        if (two) bulk_load(stage + kScales + 2 * TILE, sd, 2 * n, bar);
      }
    }
  };
  // The vectors' elements of half h (32 rows) of a step.
  template <int NG, typename Src>
  struct Vectors {
    const T* r[NG];  // at the step's first row
    uint4 b[2][NG][Src::kParts];
    template <int G, int P>
    __device__ __forceinline__ void rows(const Src& src, int count, int k, int lane) {
      const int g = lane >> 2;
#pragma unroll
      for (int n = 0; n < G; ++n) r[n] = src.row(min(8 * n + g, count - 1)) + 8 * (lane & 3) + k;
      if (Src::kParts == 2 && P == 1)
        r[0] = src.row(min(g & 3, count - 1)) + (g & 4 ? src.half : 0) + 8 * (lane & 3) + k;
    }
    template <int G, int P>
    __device__ __forceinline__ void load(int h, const Src& src, int left, int lane) {
      const bool whole = 32 * h + 32 <= left;  // else the weights end inside: 16 rows
      if (32 * h >= left) return;
#pragma unroll
      for (int n = 0; n < G; ++n)
#pragma unroll
        for (int p = 0; p < P; ++p) {
          b[h][n][p] = make_uint4(0, 0, 0, 0);
          if (whole || 32 * h + 8 * (lane & 3) < left)
            b[h][n][p] = *reinterpret_cast<const uint4*>(r[n] + p * src.half + 32 * h);
        }
    }
    template <int G>
    __device__ __forceinline__ void advance(int rows) {
#pragma unroll
      for (int n = 0; n < G; ++n) r[n] += rows;
    }
  };
  // codes j of w as B + 8 q, and the operand of -(B + 64)
  static constexpr uint32_t kBase = kIsBf16<T> ? 0x43004300u : 0x64006400u;
  static constexpr uint32_t kMinus = kIsBf16<T> ? 0xc340c340u : 0xe440e440u;
  static __device__ __forceinline__ void operands(uint32_t (&a)[4], uint32_t w) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      a[j] = ((j ? __funnelshift_r(w, w, 4 * j) : w) & 0x00780078u) | kBase;
  }
  // One half of a step for the first G groups of vectors and P of their parts.
  template <int G, int P, int NG, typename Src>
  static __device__ __forceinline__ void half(int h, float (&acc)[kSums][NG][4], const Lane&,
                                              const Matrix& m, const Strip& s, int left,
                                              uint32_t stage, int lane,
                                              const Vectors<NG, Src>& v) {
    if (32 * h >= left) return;
    float minus[G][4] = {};
    const uint32_t minus_op[4] = {kMinus, kMinus, kMinus, kMinus};
    const uint32_t scales =
        stage + kScales + 4 * (lane >> 2) + (h && m.shift == 5 ? 2 * TILE : 0);
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int n = 0; n < G; ++n)
          mma<T>(minus[n], minus_op, q ? v.b[h][n][p].z : v.b[h][n][p].x,
                 q ? v.b[h][n][p].w : v.b[h][n][p].y);
#pragma unroll
    for (int i0 = 0; i0 < kSums; i0 += 4) {  // four blocks interleaved
      if (TILE > 64 && i0 >= kSums / 2 && s.hi == 0) break;
      uint2 w[4];
      float part[4][G][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = lds8(stage + 512 * (i0 + i) + 16 * lane + 8 * h);
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t a[4];
          operands(a, q ? w[i].y : w[i].x);
#pragma unroll
          for (int p = 0; p < P; ++p)
#pragma unroll
            for (int n = 0; n < G; ++n) {
              if (q == 0 && p == 0)
                mma<T>(part[i][n], a, v.b[h][n][p].x, v.b[h][n][p].y, minus[n]);
              else
                mma<T>(part[i][n], a, q ? v.b[h][n][p].z : v.b[h][n][p].x,
                       q ? v.b[h][n][p].w : v.b[h][n][p].y);
            }
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 sc = unpack2<T>(lds4(scales + 32 * (i0 + i)));
#pragma unroll
        for (int n = 0; n < G; ++n) {
          float(&d)[4] = acc[i0 + i][n];
          d[0] += sc.x * part[i][n][0];
          d[1] += sc.x * part[i][n][1];
          d[2] += sc.y * part[i][n][2];
          d[3] += sc.y * part[i][n][3];
        }
      }
    }
  }
  template <int G, int NG, int LD, bool ADD>
  static __device__ __forceinline__ void store(const float (&acc)[kSums][NG][4], int lane, float* red) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < G; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float* p = red + (8 * n + 2 * t + j) * LD + 2 * g;
#pragma unroll
        for (int i = 0; i < kSums; ++i) {
          float2* d = reinterpret_cast<float2*>(p + 16 * i);
          float2 a = make_float2(0.125f * acc[i][n][j], 0.125f * acc[i][n][j + 2]);
          if (ADD) {
            const float2 x = *d;
            a.x += x.x;
            a.y += x.y;
          }
          *d = a;
        }
      }
  }
};

// fp32 weights: plain FMAs (the tensor pipe's tf32 would drop 13 bits of both
// operands).  One step is a box of 16 rows x 64 columns (gated: two of 32): half-warp
// p takes columns 4c..4c+3 (c = lane % 16) of rows 8p..8p+7; the token values are
// the same for all lanes of a half-warp (broadcast loads).  The halves are added
// at the end.
struct Dense32 {
  using Elem = float;
  static constexpr int kTile = 64;
  static constexpr int kSums = 4;
  static constexpr int kStep = 16;
  static constexpr bool kPacked = false;
  static constexpr bool kGroups = false;
  static constexpr int kStage = 4096;
  template <int NG>
  static constexpr int kDepth = 2;
  template <int NG>
  static constexpr int kTokens = 4 * NG;  // acc[4][NG][4]: 4 NG tokens x 4 columns
  struct Lane {
    uint32_t off, ld;
    __device__ __forceinline__ Lane(int lane, int gated) {
      const int p = lane >> 4, c = lane & 15;
      ld = gated ? 128 : 256;
      off = gated ? (c >> 3) * 2048 + p * 1024 + (c & 7) * 16 : p * 2048 + c * 16;
    }
  };
  using Cursor = BoxCursor<kStage>;
  template <int NG, typename Src>
  struct Vectors {
    const float* r[4 * NG];  // at this half-warp's first row
    template <int G, int P>
    __device__ __forceinline__ void rows(const Src& src, int count, int k, int lane) {
#pragma unroll
      for (int t = 0; t < 4 * NG; ++t) r[t] = t < count ? src.row(t) + k + 8 * (lane >> 4) : nullptr;
    }
    template <int G, int P>
    __device__ __forceinline__ void load(int, const Src&, int, int) {}
    template <int G>
    __device__ __forceinline__ void advance(int rows) {
#pragma unroll
      for (int t = 0; t < 4 * NG; ++t)
        if (r[t]) r[t] += rows;
    }
  };
  // One half of a step for the first G groups of vectors and P of their parts.
  template <int G, int P, int NG, typename Src>
  static __device__ __forceinline__ void half(int h, float (&acc)[4][NG][4], const Lane& l,
                                              const Matrix&, const Strip&, int left,
                                              uint32_t stage, int lane,
                                              const Vectors<NG, Src>& v) {
    if (h || 8 * (lane >> 4) >= left) return;  // (one part: all 16 rows)
    float4 w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 f = lds16(stage + l.off + i * l.ld);
      w[i] = *reinterpret_cast<const float4*>(&f);
    }
#pragma unroll
    for (int t = 0; t < 4 * NG; ++t) {
      if (v.r[t]) {
        const float* x = v.r[t];
        const float4 x0 = *reinterpret_cast<const float4*>(x);
        const float4 x1 = *reinterpret_cast<const float4*>(x + 4);
        const float xs[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
        float(&a)[4] = acc[t / NG][t % NG];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          a[0] = fmaf(xs[i], w[i].x, a[0]);
          a[1] = fmaf(xs[i], w[i].y, a[1]);
          a[2] = fmaf(xs[i], w[i].z, a[2]);
          a[3] = fmaf(xs[i], w[i].w, a[3]);
        }
      }
    }
  }
  template <int G, int NG, int LD, bool ADD>
  static __device__ __forceinline__ void store(const float (&acc)[4][NG][4], int lane, float* red) {
#pragma unroll
    for (int t = 0; t < 4 * NG; ++t) {
      const float(&a)[4] = acc[t / NG][t % NG];
      float v[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = a[c] + __shfl_xor_sync(0xffffffffu, a[c], 16);
      if (lane < 16) {
        float4* d = reinterpret_cast<float4*>(red + t * LD + 4 * lane);
        if (ADD) {
          const float4 x = *d;
          v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
        }
        *d = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
  }
};

}  // namespace few
}  // namespace moe
