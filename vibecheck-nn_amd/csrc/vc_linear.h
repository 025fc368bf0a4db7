// The fc layer's kernels share this: types, activations, what a product is and how
// its sums are finished (bias, activation, residual, rounding, stores).
#pragma once
#include <type_traits>

#include "vc_gemm_core.h"
#include "vc_split.h"

namespace vcl {

using namespace vcs;

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

typedef uint32_t u4at4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u2at4 __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u2at2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float v4fat4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u1at2 __attribute__((aligned(2)));

// Sixteen bytes at any alignment of the type.
__device__ __forceinline__ u4 load16(const float* p) { return *reinterpret_cast<const u4at4*>(p); }
__device__ __forceinline__ u4 load16(const uint16_t* p) { return *reinterpret_cast<const u4at2*>(p); }

enum Act { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3 };

__device__ __forceinline__ float bf_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) {
  return __builtin_bit_cast(float, w & 0xffff0000u);
}
// Two values rounded to nearest, the first in the low half.
__device__ __forceinline__ uint32_t bf_pack(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2bf));
}

// Two values' parts, the first cut: h + m + l is the value.  A NaN is made quiet first: one
// whose upper sixteen bits are an infinity's would be cut to that.
__device__ __forceinline__ void cut2(float x0, float x1, uint32_t& h, uint32_t& m, uint32_t& l) {
  x0 = __builtin_canonicalizef(x0);
  x1 = __builtin_canonicalizef(x1);
  const uint32_t b0 = __builtin_bit_cast(uint32_t, x0), b1 = __builtin_bit_cast(uint32_t, x1);
  h = __builtin_amdgcn_perm(b1, b0, 0x07060302);
  const float a0 = x0 - __builtin_bit_cast(float, b0 & 0xffff0000u);
  const float a1 = x1 - __builtin_bit_cast(float, b1 & 0xffff0000u);
  m = bf_pack(a0, a1);
  l = bf_pack(a0 - bf_lo(m), a1 - bf_hi(m));
}

template <class T>
__device__ __forceinline__ float get(const T* p) {
  if constexpr (sizeof(T) == 4) return *p;
  else return bf_lo(*p);
}
template <class T>
__device__ __forceinline__ void put(T* p, float v) {
  if constexpr (sizeof(T) == 4) *p = v;
  else *p = (uint16_t)bf_pack(v, 0.f);
}

constexpr float kLog2e = 1.44269504088896341f;
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// bf16: the normal distribution's integral up to z, and e = exp(-z^2 / 2) on the way
// (Abramowitz and Stegun 7.1.26, off by at most 7.5e-8): twenty instructions,
// where the library's erff takes twice as many and the 134 million values of an
// 8192 x 16384 output showed it (150 us of 1140).
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.f));
  e = __builtin_amdgcn_exp2f(z * z * (-0.5f * kLog2e));
  float p = __builtin_fmaf(1.061405429f, t, -1.453152027f);
  p = __builtin_fmaf(p, t, 1.421413741f);
  p = __builtin_fmaf(p, t, -0.284496736f);
  p = __builtin_fmaf(p, t, 0.254829592f);
  const float q = 0.5f * p * t * e;  // of -|z|
  return z < 0.f ? q : 1.f - q;
}

// In fp32 the forms that lose nothing: erfc keeps the small values of a negative z, and
// exp(-|z|) both of a sigmoid's sides.
template <class T>
__device__ __forceinline__ float activate(float z, int act) {
  if (act == kRelu) return z > 0.f ? z : (z != z ? z : 0.f);
  if constexpr (sizeof(T) == 4) {
    if (act == kGelu) return 0.5f * z * erfcf(z * -0.70710678118654752f);
    if (act == kSilu) {
      const float e = expf(-fabsf(z));
      return (z < 0.f ? z * e : z) / (1.f + e);
    }
  } else {
    float e;
    if (act == kGelu) return z * normal_cdf(z, e);
    if (act == kSilu) return z * __builtin_amdgcn_rcpf(1.f + exp_of(-z));
  }
  return z;
}

// dy act'(z).  ReLU's is a choice: an infinite or NaN dy where it is closed adds nothing.
template <class T>
__device__ __forceinline__ float dz_of(float dy, float z, int act) {
  if (act == kRelu) return z > 0.f ? dy : 0.f;
  if constexpr (sizeof(T) == 4) {
    if (act == kGelu)
      return dy * __builtin_fmaf(z * expf(-0.5f * z * z), 0.39894228040143268f,
                                 0.5f * erfcf(z * -0.70710678118654752f));
    const float e = expf(-fabsf(z)), u = 1.f / (1.f + e), v = e * u;
    return dy * __builtin_fmaf(z * u, v, z < 0.f ? v : u);
  } else {
    if (act == kGelu) {
      float e;
      const float c = normal_cdf(z, e);
      return dy * __builtin_fmaf(z * e, 0.39894228040143268f, c);
    }
    const float s = __builtin_amdgcn_rcpf(1.f + exp_of(-z));
    return dy * (s * (1.f + z * (1.f - s)));
  }
}

// An operand: `rows` of its free axis; (row, k) at p[row ld + k], across at
// p[k ld + row].
template <class T>
struct Operand {
  const T* p;
  int64_t ld;
  int rows;
};

template <class T>
struct Product {
  Operand<T> A, B;
  int I, J, K;
  int slices, steps;  // steps of a slice
  float* part;        // slices > 1: (slices, I, part_line(J))
  const T *bias, *res;
  int64_t ldr;
  T *out, *z;
  int act;
  int64_t tiles;
  vcg::FastDiv f_nj;
  // as bf16 parts (an fp32 value is three): plane p of an operand starts p planes
  // after the first
  const uint16_t *pa, *pb;
  int64_t lda, ldb, planeA, planeB;
};

// The tiled products of vc_linear_tile.hip, shapes 0, 1, 2: 256 x 256 (fp32 256 x
// 128), 128 x 128, 64 x 64; 3, bf16 forward alone: 64 x 64, loaded three steps ahead.
// Rows (across: k) lie lda, ldb values apart.  The caller has seen to it that every operand's base and ld are
// multiples of 16 bytes, that K is a multiple of eight (an operand whose k is
// contiguous) or its lines are padded to one (read across), and that 256 of them
// span less than 2^31 bytes.
struct TileShape {
  int bi, bj, bk;
};
TileShape tile_shape(int type, int shape);

// The blocks' sums of dz's columns, joined: 32 columns a workgroup at a time.
template <class T>
struct Columns {
  const float* sums;  // (blocks, N)
  int blocks, N;
  T* db;
  int groups;         // workgroups
};

// The forward's product of fp32 rows as they are: bases, lds and K multiples of 16
// bytes, 64 rows within 2^31.
void run_raw(const Product<float>& a, hipStream_t st);
// The forward's product.
template <class T>
void run_tile(const Product<T>& a, int shape, hipStream_t st);
// The backward's two and the columns' sums, in one launch of `grid` workgroups.
template <class T>
void run_tiles(const Product<T>& w, const Product<T>& x, const Columns<T>& c, int shape,
               unsigned grid, hipStream_t st);

// A line of a slice's sums.
__host__ __device__ __forceinline__ int part_line(int J) { return (J + 3) & ~3; }

// Four values at any alignment of the type.
__device__ __forceinline__ v4f load4(const float* p) { return *reinterpret_cast<const v4fat4*>(p); }
__device__ __forceinline__ v4f load4(const uint16_t* p) {
  const u2 w = *reinterpret_cast<const u2at2*>(p);
  return v4f{bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y)};
}
__device__ __forceinline__ void store4(float* p, const v4f& v) { *reinterpret_cast<v4fat4*>(p) = v; }
__device__ __forceinline__ void store4(uint16_t* p, const v4f& v) {
  *reinterpret_cast<u2at2*>(p) = u2{bf_pack(v[0], v[1]), bf_pack(v[2], v[3])};
}

// Columns j .. j + 3 (all within J) of rows i, i + step, .. as far as they go: bias,
// activation, residual, stores.  Every row's loads come before the first that is
// worked on, one branch chooses the activation of all.  bias: zeros where there is
// none.  BARE: a product with none of them, as the backward's are.
template <class T, bool BARE, int U>
__device__ __forceinline__ void finish_rows(const Product<T>& a, int i, int step, int j,
                                            const v4f& bias, const v4f (&s)[U]) {
  const int64_t o = (int64_t)i * a.J + j;
  if (BARE) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * step < a.I) store4(a.out + o + (int64_t)u * step * a.J, s[u]);
    return;
  }
  v4f z[U], v[U], r[U];
  if (a.res) {
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = load4(a.res + min(i + u * step, a.I - 1) * a.ldr + j);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) v[u] = z[u] = a.bias ? s[u] + bias : s[u];
  const auto each = [&](auto act) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[u][q] = activate<T>(z[u][q], act);
  };
  if (a.act == kRelu) each(std::integral_constant<int, kRelu>{});
  else if (a.act == kGelu) each(std::integral_constant<int, kGelu>{});
  else if (a.act == kSilu) each(std::integral_constant<int, kSilu>{});
  if (a.res) {
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] += r[u];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (i + u * step >= a.I) continue;
    store4(a.out + o + (int64_t)u * step * a.J, v[u]);
    if (a.z) store4(a.z + o + (int64_t)u * step * a.J, z[u]);
  }
}

template <class T>
__device__ __forceinline__ v4f bias_of(const Product<T>& a, int j) {
  v4f b = v4f{0.f, 0.f, 0.f, 0.f};
  if (a.bias) {
#pragma unroll
    for (int q = 0; q < 4; ++q) b[q] = get(a.bias + min(j + q, a.J - 1));
  }
  return b;
}

// Four columns j .. j + 3 of row i, the last of them past J perhaps.
template <class T, bool BARE>
__device__ __forceinline__ void finish(const Product<T>& a, int i, int j, const v4f& s) {
  if (j + 4 <= a.J) {
    const v4f one[1] = {s};
    finish_rows<T, BARE>(a, i, 0, j, BARE ? v4f{} : bias_of(a, j), one);
    return;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (j + q >= a.J) continue;
    const int64_t o = (int64_t)i * a.J + j + q;
    if (BARE) {
      put(a.out + o, s[q]);
      continue;
    }
    const float z = a.bias ? s[q] + get(a.bias + j + q) : s[q];
    float v = activate<T>(z, a.act);
    if (a.res) v += get(a.res + i * a.ldr + j + q);
    put(a.out + o, v);
    if (a.z) put(a.z + o, z);
  }
}

// Four columns of row i of a slice: finished, or left for the join.
template <class T, bool BARE>
__device__ __forceinline__ void deliver(const Product<T>& a, int64_t slice, int i, int j,
                                        const v4f& s) {
  if (a.slices == 1) finish<T, BARE>(a, i, j, s);
  else *reinterpret_cast<v4f*>(a.part + (slice * a.I + i) * part_line(a.J) + j) = s;
}

// lds: 32 floats for every 32 threads.
template <class T>
__device__ __forceinline__ void add_columns(const Columns<T>& a, int block, float* lds) {
  const int c = threadIdx.x & 31, y = threadIdx.x >> 5, ny = blockDim.x >> 5;
#pragma unroll 1
  for (int at = block * 32; at < a.N; at += a.groups * 32) {
    const int j = at + c;
    const float* const p = a.sums + min(j, a.N - 1);
    float s = 0.f;
    for (int b = y; b < a.blocks; b += 8 * ny) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = p[(int64_t)min(b + u * ny, a.blocks - 1) * a.N];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += b + u * ny < a.blocks ? v[u] : 0.f;
    }
    __syncthreads();  // the turn before has read
    lds[y * 32 + c] = s;
    __syncthreads();
    if (y || j >= a.N) continue;
    for (int i = 1; i < ny; ++i) s += lds[i * 32 + c];
    put(a.db + j, s);
  }
}

}  // namespace vcl
