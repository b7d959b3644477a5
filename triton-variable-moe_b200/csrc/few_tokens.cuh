// Device pieces of the few-token kernels: a warp's product of a 64-column
// strip of weights with up to 8 * NG token vectors.
//
// With few rows per expert the products are bound by reading the weights once
// (at 8 tokens: 16 flops per 2-byte weight against the ~250 that would balance
// HBM and the tensor pipe), so the layout is chosen for the loads: a lane takes
// 16-byte vectors straight from global memory into registers (no shared
// memory, no barrier in the loop), a warp-wide load covers four 128-byte row
// pieces, and the next step's vectors are in flight while the current ones are
// multiplied.  The multiply is m16n8k16 with the weights as the 16-row operand
// and the tokens as its 8 columns: any assignment of reduction rows to the
// instruction's k slots is right as long as both operands share it, so the
// lane's registers become fragments with one byte permute per weight pair.
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

// d += a (16 x 16) * b (16 x 8), fp32 accumulation.
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4],
                                                   uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                            uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Weights are read once: past L1, first to leave L2 (what is read again, the
// token vectors and partial sums, stays).
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
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
// Where the multiplied vectors come from.  A lane asks for 8 consecutive
// reduction elements of one row; rows past the count and elements past the end
// are zero (never read), so nothing beyond a vector enters a sum.

// Rows of a matrix of the storage type (the layer's tokens, through an index
// list, or the rows of a grouped product).
template <typename T>
struct RowSource {
  static constexpr int kParts = 1;  // 16-bit operands per value
  const T* x;
  long long ld;
  const int* list;  // row of the k-th vector (null: first + k)
  int first;
  __device__ __forceinline__ const T* row(int i) const {
    return x + static_cast<long long>(list ? list[first + i] : first + i) * ld;
  }
  __device__ __forceinline__ void load8(const T* r, int k, uint4 (&b)[1]) const {
    b[0] = *reinterpret_cast<const uint4*>(r + k);
  }
  __device__ __forceinline__ void load8f(const T* r, int k, float (&v)[8]) const {
    const float4 a = *reinterpret_cast<const float4*>(r + k);
    const float4 c = *reinterpret_cast<const float4*>(r + k + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = c.x; v[5] = c.y; v[6] = c.z; v[7] = c.w;
  }
};

// The activated intermediate, from the partial sums of the up product: the
// slices are added in order and the activation applied on the way in.  For
// 16-bit weights the fp32 value is split in two 16-bit operands (value and
// remainder, about 2^-17 relative), multiplied one after the other: the
// intermediate is never rounded to the storage type, and the second multiply
// is free beside the weight loads.  In fp16 a value above 65504 is infinite, as
// it is in the layer's forward, which stores it.
template <typename T>
struct PartialSource {
  static constexpr int kParts = 2;
  const float* u;  // [slices][rows][ld]
  long long ld, slice_stride;
  int slices, first, act, width;  // width: the gated activation's second operand
  __device__ __forceinline__ const float* row(int i) const {
    return u + static_cast<long long>(first + i) * ld;
  }
  __device__ __forceinline__ void sum8(const float* r, float (&v)[8]) const {
    float4 a = *reinterpret_cast<const float4*>(r);
    float4 c = *reinterpret_cast<const float4*>(r + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = c.x; v[5] = c.y; v[6] = c.z; v[7] = c.w;
#pragma unroll 4
    for (int s = 1; s < slices; ++s) {
      r += slice_stride;
      a = *reinterpret_cast<const float4*>(r);
      c = *reinterpret_cast<const float4*>(r + 4);
      v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
      v[4] += c.x; v[5] += c.y; v[6] += c.z; v[7] += c.w;
    }
  }
  __device__ __forceinline__ void load8f(const float* r, int k, float (&v)[8]) const {
    sum8(r + k, v);
    if (act == ACT_SWIGLU) {
      float up[8];
      sum8(r + k + width, up);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_gated(v[i], up[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_plain(v[i], act);
    }
  }
  __device__ __forceinline__ void load8(const float* r, int k, uint4 (&b)[2]) const {
    float v[8];
    load8f(r, k, v);
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hi[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
      const float2 h = unpack2<T>(hi[i]);
      // an infinite or NaN value has no remainder
      const float l0 = v[2 * i] - h.x, l1 = v[2 * i + 1] - h.y;
      lo[i] = pack2<T>(fabsf(h.x) <= 3.4e38f ? l0 : 0.f, fabsf(h.y) <= 3.4e38f ? l1 : 0.f);
    }
    b[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    b[1] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
};

// ------------------------------------------------------------------ weights
// A strip: the reduction rows [0, rows) of one expert's weights and 64 of its
// columns (fewer at the right edge; a multiple of 16 always).

// 16-bit weights, row-major.  One step is 32 rows: lane (g = lane / 4,
// t = lane % 4) loads columns 8g..8g+7 of rows 8t..8t+7.  Multiply (i, s), i < 4,
// s < 2, takes columns 8g + 2i and 8g + 2i + 1 as its rows g and g + 8 and
// reduction rows 8t + 4s .. 8t + 4s + 3 as lane t's k slots.
template <typename T>
struct Dense16 {
  using Elem = T;
  static constexpr int kStep = 32;
  struct Strip {
    const T* w;  // first row, first column of the strip
    long long ld;
    int rows, cols;
  };
  struct Frag {
    uint4 v[8];
  };
  static __device__ __forceinline__ void load(const Strip& s, int k0, int lane, Frag& f) {
    const int g = lane >> 2, k = k0 + 8 * (lane & 3);
    const bool ok = 8 * g < s.cols && k < s.rows;  // rows and columns come in 8s
    const T* p = s.w + static_cast<long long>(k) * s.ld + 8 * g;
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = ok ? ld_stream(p + i * s.ld) : make_uint4(0, 0, 0, 0);
  }
  template <int NG, typename Src>
  static __device__ __forceinline__ void step(float (&acc)[4][NG][4], const Frag& f,
                                              const Strip& s, int k0, int lane, const Src& src,
                                              int count) {
    const int g = lane >> 2, k = k0 + 8 * (lane & 3);
    uint4 b[NG][Src::kParts];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
#pragma unroll
      for (int p = 0; p < Src::kParts; ++p) b[n][p] = make_uint4(0, 0, 0, 0);
      if (8 * n + g < count && k < s.rows) src.load8(src.row(8 * n + g), k, b[n]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t* r0 = reinterpret_cast<const uint32_t*>(&f.v[4 * h]);
      const uint32_t* r1 = reinterpret_cast<const uint32_t*>(&f.v[4 * h + 1]);
      const uint32_t* r2 = reinterpret_cast<const uint32_t*>(&f.v[4 * h + 2]);
      const uint32_t* r3 = reinterpret_cast<const uint32_t*>(&f.v[4 * h + 3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a[4] = {__byte_perm(r0[i], r1[i], 0x5410), __byte_perm(r0[i], r1[i], 0x7632),
                               __byte_perm(r2[i], r3[i], 0x5410), __byte_perm(r2[i], r3[i], 0x7632)};
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int p = 0; p < Src::kParts; ++p)
            mma<T>(acc[i][n], a, h ? b[n][p].z : b[n][p].x, h ? b[n][p].w : b[n][p].y);
      }
    }
  }
  // red[token][64 columns] (row stride kRedLd) of this warp's sums
  template <int NG, int LD>
  static __device__ __forceinline__ void store(const float (&acc)[4][NG][4], int lane, float* red) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float* p = red + (8 * n + 2 * t + j) * LD + 8 * g;
        *reinterpret_cast<float4*>(p) =
            make_float4(acc[0][n][j], acc[0][n][j + 2], acc[1][n][j], acc[1][n][j + 2]);
        *reinterpret_cast<float4*>(p + 4) =
            make_float4(acc[2][n][j], acc[2][n][j + 2], acc[3][n][j], acc[3][n][j + 2]);
      }
  }
};

// 4-bit weights in the packed layout (see int4.cu): blocks of 64 rows x 16
// columns, 16 bytes a lane.  Word s of a lane's vector feeds the multiply of
// the block's rows 32 (s / 2) + 8t + 4 (s % 2) .. + 3; its nibbles j and j + 4
// are operand register j (columns 2g, 2g + 1 as the instruction's rows g and
// g + 8).  A nibble q is held as the exact 16-bit number q - 8 and multiplied
// unscaled; the fp32 sums of each group are scaled as they are added up, so the
// scales are never rounded into the weights.  One step is 64 rows.
template <typename T>
struct Int4 {
  using Elem = T;
  static constexpr int kStep = 64;
  struct Strip {
    const uint4* w;   // first block row, first column block of the strip
    long long ld;     // blocks a block row
    const T* scales;  // first group, first column
    long long lds;
    int rows, cols, shift, groups;  // 2^shift rows a group
  };
  struct Frag {
    uint4 v[4];
    uint32_t sc[2][4];
  };
  static __device__ __forceinline__ void load(const Strip& s, int k0, int lane, Frag& f) {
    const uint4* p = s.w + (static_cast<long long>(k0 >> 6) * s.ld) * 32 + lane;
    const bool in = k0 < s.rows;
    const int g0 = min(k0 >> s.shift, s.groups - 1);
    const T* sp = s.scales + static_cast<long long>(g0) * s.lds + 2 * (lane >> 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool ok = in && 16 * i < s.cols;
      f.v[i] = ok ? ld_stream(p + 32 * i) : make_uint4(0, 0, 0, 0);
      f.sc[0][i] = ok ? __ldg(reinterpret_cast<const uint32_t*>(sp + 16 * i)) : 0u;
    }
    if (s.shift == 5) {
      const int g1 = min(g0 + 1, s.groups - 1);
      const T* sq = s.scales + static_cast<long long>(g1) * s.lds + 2 * (lane >> 2);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        f.sc[1][i] = in && 16 * i < s.cols ? __ldg(reinterpret_cast<const uint32_t*>(sq + 16 * i)) : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) f.sc[1][i] = f.sc[0][i];
    }
  }
  // nibbles j and j + 4 of w as two 16-bit numbers q - 8 (exact: 128 + q, or
  // 1024 + q, is the number whose low mantissa bits are q)
  static __device__ __forceinline__ uint32_t nibbles(uint32_t w, int j);
  template <int NG, typename Src>
  static __device__ __forceinline__ void step(float (&acc)[4][NG][4], const Frag& f,
                                              const Strip& s, int k0, int lane, const Src& src,
                                              int count) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // 32 rows each
      const int g = lane >> 2, k = k0 + 32 * h + 8 * (lane & 3);
      uint4 b[NG][Src::kParts];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
#pragma unroll
        for (int p = 0; p < Src::kParts; ++p) b[n][p] = make_uint4(0, 0, 0, 0);
        if (8 * n + g < count && k < s.rows) src.load8(src.row(8 * n + g), k, b[n]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float part[NG][4];
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) part[n][c] = 0.f;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t w = reinterpret_cast<const uint32_t*>(&f.v[i])[2 * h + q];
          const uint32_t a[4] = {nibbles(w, 0), nibbles(w, 1), nibbles(w, 2), nibbles(w, 3)};
#pragma unroll
          for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int p = 0; p < Src::kParts; ++p)
              mma<T>(part[n], a, q ? b[n][p].z : b[n][p].x, q ? b[n][p].w : b[n][p].y);
        }
        const float2 sc = unpack2<T>(f.sc[h][i]);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          acc[i][n][0] += sc.x * part[n][0];
          acc[i][n][1] += sc.x * part[n][1];
          acc[i][n][2] += sc.y * part[n][2];
          acc[i][n][3] += sc.y * part[n][3];
        }
      }
    }
  }
  template <int NG, int LD>
  static __device__ __forceinline__ void store(const float (&acc)[4][NG][4], int lane, float* red) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float* p = red + (8 * n + 2 * t + j) * LD + 2 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float2*>(p + 16 * i) = make_float2(acc[i][n][j], acc[i][n][j + 2]);
      }
  }
};
template <>
__device__ __forceinline__ uint32_t Int4<__nv_bfloat16>::nibbles(uint32_t w, int j) {
  uint32_t v = ((w >> (4 * j)) & 0x000f000fu) | 0x43004300u;
  const uint32_t off = 0x43084308u;  // 136
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v),
                                   *reinterpret_cast<const __nv_bfloat162*>(&off));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t Int4<__half>::nibbles(uint32_t w, int j) {
  uint32_t v = ((w >> (4 * j)) & 0x000f000fu) | 0x64006400u;
  const uint32_t off = 0x64086408u;  // 1032
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v),
                            *reinterpret_cast<const __half2*>(&off));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// fp32 weights: plain FMAs (the tensor pipe's tf32 would drop 13 bits of both
// operands).  One step is 16 rows: half-warp p loads columns 4c..4c+3 (c =
// lane % 16) of rows 8p..8p+7; the token values are the same for all lanes of a
// half-warp (one broadcast load each).  The halves are added at the end.
struct Dense32 {
  using Elem = float;
  static constexpr int kStep = 16;
  struct Strip {
    const float* w;
    long long ld;
    int rows, cols;
  };
  struct Frag {
    uint4 v[8];
  };
  static __device__ __forceinline__ void load(const Strip& s, int k0, int lane, Frag& f) {
    const int c = 4 * (lane & 15), k = k0 + 8 * (lane >> 4);
    const bool ok = c < s.cols && k < s.rows;
    const float* p = s.w + static_cast<long long>(k) * s.ld + c;
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = ok ? ld_stream(p + i * s.ld) : make_uint4(0, 0, 0, 0);
  }
  // acc[token][column]: NG is 2 here for 8 tokens of 4 columns (32 sums)
  template <int NG, typename Src>
  static __device__ __forceinline__ void step(float (&acc)[4][NG][4], const Frag& f,
                                              const Strip& s, int k0, int lane, const Src& src,
                                              int count) {
    const int k = k0 + 8 * (lane >> 4);
    if (k >= s.rows) return;
#pragma unroll
    for (int t = 0; t < 4 * NG; ++t) {
      if (t >= count) break;
      float v[8];
      src.load8f(src.row(t), k, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 w = *reinterpret_cast<const float4*>(&f.v[i]);
        float(&a)[4] = acc[t / NG][t % NG];
        a[0] = fmaf(v[i], w.x, a[0]);
        a[1] = fmaf(v[i], w.y, a[1]);
        a[2] = fmaf(v[i], w.z, a[2]);
        a[3] = fmaf(v[i], w.w, a[3]);
      }
    }
  }
  template <int NG, int LD>
  static __device__ __forceinline__ void store(const float (&acc)[4][NG][4], int lane, float* red) {
#pragma unroll
    for (int t = 0; t < 4 * NG; ++t) {
      const float(&a)[4] = acc[t / NG][t % NG];
      float v[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = a[c] + __shfl_xor_sync(0xffffffffu, a[c], 16);
      if (lane < 16)
        *reinterpret_cast<float4*>(red + t * LD + 4 * lane) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
};

// One warp's share of a strip: steps begin + wr * kStep, + stride, ... below
// s.rows, the next step's weights loading while one is multiplied; its sums go
// to red[token][column].
template <typename L, int NG, int STRIDE, int LD, typename Src>
__device__ __forceinline__ void product(const typename L::Strip& s, const Src& src, int count,
                                        int k, int lane, float* red) {
  float acc[4][NG][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][n][c] = 0.f;
  typename L::Frag f0, f1;
  if (k < s.rows) {
    L::load(s, k, lane, f0);
    while (true) {
      if (k + STRIDE < s.rows) L::load(s, k + STRIDE, lane, f1);
      L::template step<NG>(acc, f0, s, k, lane, src, count);
      k += STRIDE;
      if (k >= s.rows) break;
      if (k + STRIDE < s.rows) L::load(s, k + STRIDE, lane, f0);
      L::template step<NG>(acc, f1, s, k, lane, src, count);
      k += STRIDE;
      if (k >= s.rows) break;
    }
  }
  L::template store<NG, LD>(acc, lane, red);
}

}  // namespace few
}  // namespace moe
