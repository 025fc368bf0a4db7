// The fc layer itself, forward and backward, in fp32 and bf16:
//   z = x W^T + b, y = act(z) + r;
//   dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum over rows of dz.
//
// Every product is C[i][j] = sum_k A(i, k) B(j, k) on the bf16 matrix cores,
// summed in fp32; an operand's k may be its contiguous axis or its other one
// (dx reads W, dW reads dz and x across).  An fp32 value is three bf16 parts,
// here cut rather than rounded at the first (h = the value's upper 16 bits), so
// that a finite value never becomes an infinity; six of the nine part products
// are formed (vc_split.h).  The five small ones run on in the accumulator, the
// largest starts from zero each step of 32 and is added in fp32.  Where the sum
// is not finite the largest products' sum stands alone: with an infinity or NaN
// among the values it is what the fp32 product gives, and the small ones are not.
#include "vc_gemm_core.h"
#include "vc_split.h"

namespace {

using namespace vcs;

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

constexpr int LNT = 256;  // threads: four waves, 2 x 2 over the tile

enum Act { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3 };

__device__ __forceinline__ float bf_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) {
  return __builtin_bit_cast(float, w & 0xffff0000u);
}
// Two values rounded to nearest, the first in the low half.
__device__ __forceinline__ uint32_t bf_pack(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2bf));
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

__device__ __forceinline__ float activate(float z, int act) {
  if (act == kRelu) return z > 0.f ? z : (z != z ? z : 0.f);
  if (act == kGelu) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  if (act == kSilu) return z / (1.f + expf(-z));
  return z;
}

__device__ __forceinline__ float slope(float z, int act) {
  if (act == kRelu) return z > 0.f ? 1.f : 0.f;
  if (act == kGelu)
    return 0.5f * (1.f + erff(z * 0.70710678118654752f)) +
           z * expf(-0.5f * z * z) * 0.39894228040143268f;
  const float s = 1.f / (1.f + expf(-z));
  return s * (1.f + z * (1.f - s));
}

// An operand: `rows` of its free axis; (row, k) at p[row ld + k], across at
// p[k ld + row].  vec: two rows' eight k may be read by its wide loads.
template <class T>
struct Operand {
  const T* p;
  int64_t ld;
  int rows, vec;
};

template <class T>
struct Product {
  Operand<T> A, B;
  int I, J, K;
  int slices, steps;  // steps of a slice
  float* part;        // slices > 1: (slices, I, J)
  const T *bias, *res;
  int64_t ldr;
  T *out, *z;
  int act, wide;      // wide: four columns of out, z, res and bias by one access
  int64_t tiles;
  vcg::FastDiv f_nj;
};

// Eight k of two rows, as loaded: of bf16 [row][k pair] or across [k] (both
// rows), of fp32 [row][k] or across [k][row].
template <class T>
struct Raw {
  uint32_t d[sizeof(T) == 4 ? 16 : 8];
};

template <class T, bool ACROSS>
__device__ __forceinline__ void load_unit(const Operand<T>& o, int row, int k, int K, Raw<T>& v) {
  constexpr bool F = sizeof(T) == 4;
  const int r0 = min(row, o.rows - 1), r1 = min(row + 1, o.rows - 1);
  if (!ACROSS) {
    const T* const p0 = o.p + (int64_t)r0 * o.ld + k;
    const T* const p1 = o.p + (int64_t)r1 * o.ld + k;
    if (o.vec) {  // K a multiple of eight
      u4 a[F ? 4 : 2];
      const u4 zero = u4{0, 0, 0, 0};
      const bool in = k < K;
      const u4* const q0 = reinterpret_cast<const u4*>(in ? p0 : p0 - k);
      const u4* const q1 = reinterpret_cast<const u4*>(in ? p1 : p1 - k);
      a[0] = q0[0];
      if (F) a[1] = q0[1];
      a[F ? 2 : 1] = q1[0];
      if (F) a[F ? 3 : 1] = q1[1];
#pragma unroll
      for (int i = 0; i < (F ? 4 : 2); ++i) {
        a[i] = in ? a[i] : zero;
#pragma unroll
        for (int j = 0; j < 4; ++j) v.d[4 * i + j] = a[i][j];
      }
      return;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const T* const p = r ? p1 : p0;
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = 0;
        if (k + j < K) {
          if (F) w[j] = __builtin_bit_cast(uint32_t, (float)get(p + j));
          else w[j] = (uint32_t)p[j];
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (F) v.d[8 * r + j] = w[j];
        else if (j & 1) v.d[4 * r + j / 2] = w[j - 1] | w[j] << 16;
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool in = k + j < K;
    const T* const p = o.p + (int64_t)(in ? k + j : 0) * o.ld;
    if (o.vec) {  // rows and ld even
      if (F) {
        const u2 w = *reinterpret_cast<const u2*>(p + min(row, o.rows - 2));
        v.d[2 * j] = in ? w.x : 0;
        v.d[(2 * j + 1) % (F ? 16 : 8)] = in ? w.y : 0;
      } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p + min(row, o.rows - 2));
        v.d[j] = in ? w : 0;
      }
    } else if (F) {
      v.d[(2 * j) % (F ? 16 : 8)] = in ? __builtin_bit_cast(uint32_t, (float)get(p + r0)) : 0;
      v.d[(2 * j + 1) % (F ? 16 : 8)] = in ? __builtin_bit_cast(uint32_t, (float)get(p + r1)) : 0;
    } else {
      v.d[j] = in ? (uint32_t)p[r0] | (uint32_t)p[r1] << 16 : 0;
    }
  }
}

// Two values' parts, the first cut: h + m + l is the value.
__device__ __forceinline__ void cut2(float x0, float x1, uint32_t& h, uint32_t& m, uint32_t& l) {
  const uint32_t b0 = __builtin_bit_cast(uint32_t, x0), b1 = __builtin_bit_cast(uint32_t, x1);
  h = __builtin_amdgcn_perm(b1, b0, 0x07060302);
  const float a0 = x0 - __builtin_bit_cast(float, b0 & 0xffff0000u);
  const float a1 = x1 - __builtin_bit_cast(float, b1 & 0xffff0000u);
  m = bf_pack(a0, a1);
  l = bf_pack(a0 - bf_lo(m), a1 - bf_hi(m));
}

// The 16-byte operands of row r (0, 1) of a unit, one per part.
template <class T, bool ACROSS>
__device__ __forceinline__ void unit_row(const Raw<T>& v, int r, u4* o) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x0 = __builtin_bit_cast(float, v.d[ACROSS ? 4 * j + r : 8 * r + 2 * j]);
      const float x1 = __builtin_bit_cast(float, v.d[ACROSS ? 4 * j + 2 + r : 8 * r + 2 * j + 1]);
      uint32_t h, m, l;
      cut2(x0, x1, h, m, l);
      o[0][j] = h;
      o[1][j] = m;
      o[2][j] = l;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[0][j] = ACROSS ? __builtin_amdgcn_perm(v.d[2 * j + 1], v.d[2 * j],
                                               r ? 0x07060302 : 0x05040100)
                       : v.d[4 * r + j];
  }
}

// Four columns j .. j + 3 of row i: bias, activation, residual, stores.
template <class T>
__device__ __forceinline__ void finish(const Product<T>& a, int64_t i, int j, const float* s) {
  const int n = min(4, a.J - j);
  float v[4], b[4] = {0.f, 0.f, 0.f, 0.f}, r[4] = {0.f, 0.f, 0.f, 0.f};
  T* const o = a.out + i * a.J + j;
  if (a.wide) {  // J a multiple of four
    if (a.bias) {
#pragma unroll
      for (int q = 0; q < 4; ++q) b[q] = get(a.bias + j + q);
    }
    if (a.res) {
      const T* const p = a.res + i * a.ldr + j;
      if constexpr (sizeof(T) == 4) {
        const v4f w = *reinterpret_cast<const v4f*>(p);
#pragma unroll
        for (int q = 0; q < 4; ++q) r[q] = w[q];
      } else {
        const u2 w = *reinterpret_cast<const u2*>(p);
        r[0] = bf_lo(w.x), r[1] = bf_hi(w.x), r[2] = bf_lo(w.y), r[3] = bf_hi(w.y);
      }
    }
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q >= n) continue;
      if (a.bias) b[q] = get(a.bias + j + q);
      if (a.res) r[q] = get(a.res + i * a.ldr + j + q);
    }
  }
  float z[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    z[q] = a.bias ? s[q] + b[q] : s[q];
    v[q] = activate(z[q], a.act);
    if (a.res) v[q] += r[q];
  }
  if (a.wide) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<v4f*>(o) = v4f{v[0], v[1], v[2], v[3]};
      if (a.z) *reinterpret_cast<v4f*>(a.z + i * a.J + j) = v4f{z[0], z[1], z[2], z[3]};
    } else {
      *reinterpret_cast<u2*>(o) = u2{bf_pack(v[0], v[1]), bf_pack(v[2], v[3])};
      if (a.z)
        *reinterpret_cast<u2*>(a.z + i * a.J + j) = u2{bf_pack(z[0], z[1]), bf_pack(z[2], z[3])};
    }
    return;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (q >= n) continue;
    put(o + q, v[q]);
    if (a.z) put(a.z + i * a.J + j + q, z[q]);
  }
}

// BI x BJ tiles, steps of 32 KS.  A unit is eight k of two rows, read into
// registers while the step before is multiplied, then laid into the other of
// two LDS buffers: [k step][part][row][four 16-byte chunks], chunk c of row r at
// c ^ (r / 2 mod 4), so that a fragment read meets every bank evenly.  The
// columns' fragment is the matrix step's first operand: a lane holds four
// consecutive columns of one row.
template <class T, bool XA, bool XB, int BI, int BJ>
__global__ __launch_bounds__(LNT, 2) void k_product(Product<T> a) {
  constexpr bool F = sizeof(T) == 4;
  constexpr int NP = F ? 3 : 1, KS = F ? 1 : 2, MI = BI / 32, MJ = BJ / 32;
  constexpr int UA = BI / 2 * 4 * KS, UB = BJ / 2 * 4 * KS, NU = (UA + UB) / LNT;
  constexpr int SA = KS * NP * BI * 4, SB = KS * NP * BJ * 4;  // 16-byte units of a buffer
  static_assert((UA + UB) % LNT == 0 && UA % LNT % 64 == 0, "units are dealt by whole waves");
  __shared__ __align__(16) u4 lds[2][SA + SB];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int64_t w = vcg::xcd_tile(blockIdx.x, a.tiles);
  const int ti = (int)a.f_nj.div((uint32_t)w), tj = (int)(w - (int64_t)ti * a.f_nj.d);
  const int i0 = ti * BI, j0 = tj * BJ, s0 = blockIdx.y * a.steps;
  const int steps = min(a.steps, (a.K + 32 * KS - 1) / (32 * KS) - s0);
  const int wi = wv >> 1, wj = wv & 1;

  v4f acc[MI][MJ], small[F ? MI : 1][F ? MJ : 1];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j) {
      acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
      if (F) small[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    }

  Raw<T> raw[NU];
  const auto place = [&](int n, bool& isA, int& row, int& c) {
    const int u0 = tid + n * LNT;
    isA = __builtin_amdgcn_readfirstlane(u0) < UA;
    const int u = isA ? u0 : u0 - UA, pairs = (isA ? BI : BJ) / 2;
    const bool across = isA ? XA : XB;
    row = 2 * (across ? u % pairs : u / (4 * KS));
    c = across ? u / pairs : u % (4 * KS);
  };
  const auto load = [&](int s) {
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      bool isA;
      int row, c;
      place(n, isA, row, c);
      const int k = (s0 + s) * 32 * KS + 8 * c;
      if (isA) load_unit<T, XA>(a.A, i0 + row, k, a.K, raw[n]);
      else load_unit<T, XB>(a.B, j0 + row, k, a.K, raw[n]);
    }
  };
  const auto store = [&](int buf) {
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      bool isA;
      int row, c;
      place(n, isA, row, c);
      const int R = isA ? BI : BJ;
      u4* const at = lds[buf] + (isA ? 0 : SA) + (c >> 2) * NP * R * 4;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u4 o[NP];
        if (isA) unit_row<T, XA>(raw[n], h, o);
        else unit_row<T, XB>(raw[n], h, o);
        const int q = (row + h) * 4 + ((c & 3) ^ ((row >> 1) & 3));
#pragma unroll
        for (int p = 0; p < NP; ++p) at[p * R * 4 + q] = o[p];
      }
    }
  };
  if (steps > 0) {
    load(0);
    store(0);
  }
#pragma unroll 1
  for (int s = 0; s < steps; ++s) {
    __syncthreads();  // this step is laid down, the buffer of the one before is read
    if (s + 1 < steps) load(s + 1);
    const u4* const base = lds[s & 1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      u4 fa[MI][NP];
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int row = (wi * MI + i) * 16 + r;
#pragma unroll
        for (int p = 0; p < NP; ++p)
          fa[i][p] = base[(ks * NP + p) * BI * 4 + row * 4 + (g ^ ((row >> 1) & 3))];
      }
#pragma unroll
      for (int j = 0; j < MJ; ++j) {
        const int row = (wj * MJ + j) * 16 + r;
        u4 fb[NP];
#pragma unroll
        for (int p = 0; p < NP; ++p)
          fb[p] = base[SA + (ks * NP + p) * BJ * 4 + row * 4 + (g ^ ((row >> 1) & 3))];
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          if constexpr (F) {
#pragma unroll
            for (int p = 0; p < 5; ++p)
              small[i][j] = mfma_bf16(fb[kPartA[p]], fa[i][kPartB[p]], small[i][j]);
            acc[i][j] += mfma_bf16(fb[0], fa[i][0], v4f{0.f, 0.f, 0.f, 0.f});
          } else {
            acc[i][j] = mfma_bf16(fb[0], fa[i][0], acc[i][j]);
          }
        }
      }
    }
    if (s + 1 < steps) store((s + 1) & 1);
  }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t row = i0 + (wi * MI + i) * 16 + r;
    if (row >= a.I) continue;
#pragma unroll
    for (int j = 0; j < MJ; ++j) {
      const int col = j0 + (wj * MJ + j) * 16 + 4 * g;
      if (col >= a.J) continue;
      float v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        v[q] = acc[i][j][q];
        if (F) {
          const float t = v[q] + small[i][j][q];
          v[q] = finite(t) ? t : v[q];
        }
      }
      if (a.slices == 1) {
        finish(a, row, col, v);
      } else {
        float* const o = a.part + ((int64_t)blockIdx.y * a.I + row) * a.J + col;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (col + q < a.J) o[q] = v[q];
      }
    }
  }
}

// The slices' sums joined in their order.
template <class T>
__global__ __launch_bounds__(LNT) void k_join(Product<T> a) {
  const int nq = (a.J + 3) / 4;
  for (int64_t t = blockIdx.x * (int64_t)LNT + threadIdx.x; t < (int64_t)a.I * nq;
       t += (int64_t)gridDim.x * LNT) {
    const int64_t i = t / nq;
    const int j = (int)(t - i * nq) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.slices; ++s) {
      const float* const p = a.part + ((int64_t)s * a.I + i) * a.J + j;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (j + q < a.J) v[q] = s ? v[q] + p[q] : p[q];
    }
    finish(a, i, j, v);
  }
}

// dz = dy act'(z), and the columns' sums of each block of rows.
template <class T>
struct Slope {
  const T *dy, *z;
  int64_t ldy, ldz;
  T* dz;        // null: sums only
  float* sums;  // (blocks of rows, N), or null
  int64_t M;
  int N, act, rows;
};

constexpr int kSlopeCols = 64;  // columns of a workgroup, its four waves take every fourth row

template <class T>
__global__ __launch_bounds__(LNT) void k_slope(Slope<T> a) {
  __shared__ float part[4][kSlopeCols];
  const int c = threadIdx.x & 63, y = threadIdx.x >> 6;
  const int j = blockIdx.x * kSlopeCols + c;
  const int64_t m0 = (int64_t)blockIdx.y * a.rows;
  const int64_t m1 = m0 + a.rows < a.M ? m0 + a.rows : a.M;
  float sum = 0.f;
  if (j < a.N)
    for (int64_t m = m0 + y; m < m1; m += 4) {
      float d = get(a.dy + m * a.ldy + j);
      if (a.act != kNone) d *= slope(get(a.z + m * a.ldz + j), a.act);
      if (a.dz) put(a.dz + m * a.N + j, d);
      sum += d;
    }
  part[y][c] = sum;
  __syncthreads();
  if (a.sums && y == 0 && j < a.N)
    a.sums[(int64_t)blockIdx.y * a.N + j] = (part[0][c] + part[1][c]) + (part[2][c] + part[3][c]);
}

template <class T>
__global__ __launch_bounds__(LNT) void k_slope_join(const float* sums, int blocks, int N, T* db) {
  const int j = blockIdx.x * LNT + threadIdx.x;
  if (j >= N) return;
  float s = 0.f;
  for (int b = 0; b < blocks; ++b) s += sums[(int64_t)b * N + j];
  put(db + j, s);
}

int cu_count() {
  static int n[16];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 256;
  const int at = dev & 15;
  if (!n[at]) {
    int v = 0;
    if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || v < 1)
      v = 256;
    n[at] = v;
  }
  return n[at];
}

// How a product is cut: tiles of 128 where they fill the chip, else of 64, and
// slices of k where those do not either.
struct Cut {
  int tile, slices, steps;
  int64_t tiles, nj;
};

Cut cut(int type, int64_t I, int64_t J, int64_t K) {
  const int kstep = type == VC_FP32 ? 32 : 64;
  const int64_t all = (K + kstep - 1) / kstep, cus = 256;
  Cut c;
  const int64_t t128 = ((I + 127) / 128) * ((J + 127) / 128);
  c.tile = t128 >= cus ? 128 : 64;
  c.nj = (J + c.tile - 1) / c.tile;
  c.tiles = ((I + c.tile - 1) / c.tile) * c.nj;
  int64_t s = 1;
  if (c.tiles < cus && all >= 16) {
    s = cus / c.tiles;
    if (s > all / 8) s = all / 8;
    if (s > 64) s = 64;
  }
  c.steps = (int)((all + s - 1) / s);
  if (c.steps < 1) c.steps = 1;
  c.slices = (int)((all + c.steps - 1) / c.steps);
  if (c.slices < 1) c.slices = 1;
  return c;
}

int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

int64_t part_bytes(const Cut& c, int64_t I, int64_t J) {
  return c.slices > 1 ? up256(4 * c.slices * I * J) : 0;
}

template <class T>
bool wide_rows(const T* p, int64_t ld, int64_t K) {
  return aligned16(p) && ld % (16 / (int)sizeof(T)) == 0 && K % 8 == 0;
}
template <class T>
bool wide_across(const T* p, int64_t ld, int64_t rows) {
  return ((uintptr_t)p & (2 * sizeof(T) - 1)) == 0 && ld % 2 == 0 && rows % 2 == 0;
}
template <class T>
bool quads(const void* p, int64_t ld) {
  return !p || (((uintptr_t)p & (4 * sizeof(T) - 1)) == 0 && ld % 4 == 0);
}

template <class T, bool XA, bool XB>
int run_product(Product<T> a, void* work, int64_t work_bytes, hipStream_t st) {
  constexpr int type = sizeof(T) == 4 ? VC_FP32 : VC_BF16;
  if (a.I == 0 || a.J == 0) return VC_OK;
  const Cut c = cut(type, a.I, a.J, a.K);
  if (c.tiles > (1ll << 23)) return VC_ERR_UNSUPPORTED;  // threads of a grid axis: below 2^32
  if (part_bytes(c, a.I, a.J) > work_bytes) return VC_ERR_OOM;
  a.A.vec = XA ? wide_across(a.A.p, a.A.ld, a.A.rows) : wide_rows(a.A.p, a.A.ld, a.K);
  a.B.vec = XB ? wide_across(a.B.p, a.B.ld, a.B.rows) : wide_rows(a.B.p, a.B.ld, a.K);
  a.wide = a.J % 4 == 0 && quads<T>(a.out, a.J) && quads<T>(a.z, a.J) && quads<T>(a.res, a.ldr);
  a.slices = c.slices;
  a.steps = c.steps;
  a.part = (float*)work;
  a.tiles = c.tiles;
  a.f_nj = vcg::FastDiv::make((uint32_t)c.nj);
  const dim3 grid((unsigned)c.tiles, (unsigned)c.slices);
  if (c.tile == 128) k_product<T, XA, XB, 128, 128><<<grid, LNT, 0, st>>>(a);
  else k_product<T, XA, XB, 64, 64><<<grid, LNT, 0, st>>>(a);
  if (c.slices > 1) {
    const int64_t n = (int64_t)a.I * ((a.J + 3) / 4);
    int64_t blocks = (n + LNT - 1) / LNT;
    if (blocks > 4096) blocks = 4096;
    k_join<T><<<(unsigned)blocks, LNT, 0, st>>>(a);
  }
  VC_LAUNCH_CHECK();
  return VC_OK;
}

bool sizes_ok(int64_t M, int K, int N) {
  return M >= 0 && M <= 0x7fffff00 && K >= 0 && K <= 0x7fffff00 && N >= 0 && N <= 0x7fffff00;
}

template <class T>
int forward(const void* x, int64_t M, int K, int64_t ldx, const void* W, int N, const void* bias,
            int act, const void* res, int64_t ldr, void* y, void* z, void* work,
            int64_t work_bytes, hipStream_t st) {
  Product<T> a = {};
  a.A = {(const T*)x, ldx, (int)M, 0};
  a.B = {(const T*)W, K, N, 0};
  a.I = (int)M;
  a.J = N;
  a.K = K;
  a.bias = (const T*)bias;
  a.res = (const T*)res;
  a.ldr = ldr;
  a.out = (T*)y;
  a.z = (T*)z;
  a.act = act;
  return run_product<T, false, false>(a, work, work_bytes, st);
}

// Rows of a block of k_slope: at most 256 blocks.
int slope_rows(int64_t M) {
  int64_t r = (M + 255) / 256;
  return (int)(r < 64 ? 64 : r);
}

struct BackwardPlan {
  int rows, blocks;
  int64_t dz, sums, part, bytes;  // offsets in the workspace, and its size
};

BackwardPlan plan_backward(int type, int64_t M, int K, int N, int act, int need) {
  BackwardPlan p;
  const int64_t e = type == VC_FP32 ? 4 : 2;
  p.rows = slope_rows(M);
  p.blocks = (int)((M + p.rows - 1) / p.rows);
  p.dz = 0;
  p.sums = act != kNone && (need & 3) ? up256(e * M * N) : 0;
  p.part = p.sums + (need & 4 ? up256(4ll * p.blocks * N) : 0);
  int64_t most = 0;
  if (need & 1) most = part_bytes(cut(type, M, K, N), M, K);
  if (need & 2) {
    const int64_t b = part_bytes(cut(type, N, K, M), N, K);
    if (b > most) most = b;
  }
  p.bytes = p.part + most;
  return p;
}

template <class T>
int backward(const void* dy, int64_t ldy, const void* x, int64_t ldx, const void* W, const void* z,
             int64_t ldz, int act, int64_t M, int K, int N, void* dx, void* dW, void* db,
             void* work, int64_t work_bytes, hipStream_t st) {
  constexpr int type = sizeof(T) == 4 ? VC_FP32 : VC_BF16;
  const int need = (dx ? 1 : 0) | (dW ? 2 : 0) | (db ? 4 : 0);
  const BackwardPlan p = plan_backward(type, M, K, N, act, need);
  if (p.bytes > work_bytes || (p.bytes && !work)) return VC_ERR_OOM;
  char* const base = (char*)work;
  const T* dz = (const T*)dy;
  int64_t ldd = ldy;
  const bool write = act != kNone && (need & 3);
  if (N > 0 && M > 0 && (write || db)) {
    Slope<T> s = {(const T*)dy, (const T*)z, ldy, ldz, write ? (T*)(base + p.dz) : nullptr,
                  db ? (float*)(base + p.sums) : nullptr, M, N, act, p.rows};
    k_slope<T><<<dim3((unsigned)((N + kSlopeCols - 1) / kSlopeCols), (unsigned)p.blocks), LNT, 0, st>>>(s);
  }
  if (db && N > 0)
    k_slope_join<T><<<(unsigned)((N + LNT - 1) / LNT), LNT, 0, st>>>((float*)(base + p.sums), p.blocks,
                                                                   N, (T*)db);
  VC_LAUNCH_CHECK();
  if (write) {
    dz = (const T*)(base + p.dz);
    ldd = N;
  }
  const int64_t left = work_bytes - p.part;
  if (dx) {
    Product<T> a = {};
    a.A = {dz, ldd, (int)M, 0};
    a.B = {(const T*)W, K, K, 0};
    a.I = (int)M;
    a.J = K;
    a.K = N;
    a.out = (T*)dx;
    const int rc = run_product<T, false, true>(a, base + p.part, left, st);
    if (rc != VC_OK) return rc;
  }
  if (dW) {
    Product<T> a = {};
    a.A = {dz, ldd, N, 0};
    a.B = {(const T*)x, ldx, K, 0};
    a.I = N;
    a.J = K;
    a.K = (int)M;
    a.out = (T*)dW;
    return run_product<T, true, true>(a, base + p.part, left, st);
  }
  return VC_OK;
}

bool known(int type, int act) {
  return (type == VC_FP32 || type == VC_BF16) && act >= kNone && act <= kSilu;
}

}  // namespace

extern "C" int64_t vc_linear_workspace(int type, int64_t M, int K, int N) {
  if (!known(type, kNone) || !sizes_ok(M, K, N)) return -1;
  if (M == 0 || N == 0) return 0;
  return part_bytes(cut(type, M, N, K), M, N);
}

extern "C" int vc_linear(int type, const void* x, int64_t M, int K, int64_t ldx, const void* W,
                         int N, const void* bias, int act, const void* res, int64_t ldr, void* y,
                         void* z, void* work, int64_t work_bytes, vc_stream_t stream) {
  if (!known(type, act) || !sizes_ok(M, K, N) || ldx < K || (res && ldr < N)) return VC_ERR_ARG;
  if (M == 0 || N == 0) return VC_OK;
  if (!y || (K > 0 && (!x || !W))) return VC_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  return type == VC_FP32 ? forward<float>(x, M, K, ldx, W, N, bias, act, res, ldr, y, z, work,
                                          work_bytes, st)
                         : forward<uint16_t>(x, M, K, ldx, W, N, bias, act, res, ldr, y, z, work,
                                             work_bytes, st);
}

extern "C" int64_t vc_linear_backward_workspace(int type, int64_t M, int K, int N, int act,
                                                int need) {
  if (!known(type, act) || !sizes_ok(M, K, N)) return -1;
  return plan_backward(type, M, K, N, act, need).bytes;
}

extern "C" int vc_linear_backward(int type, const void* dy, int64_t ldy, const void* x,
                                  int64_t ldx, const void* W, const void* z, int64_t ldz, int act,
                                  int64_t M, int K, int N, void* dx, void* dW, void* db,
                                  void* work, int64_t work_bytes, vc_stream_t stream) {
  if (!known(type, act) || !sizes_ok(M, K, N)) return VC_ERR_ARG;
  const bool some = M > 0 && N > 0;
  if (some && (!dy || ldy < N || (act != kNone && (!z || ldz < N)))) return VC_ERR_ARG;
  if (some && K > 0 && ((dx && !W) || (dW && (!x || ldx < K)))) return VC_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  return type == VC_FP32 ? backward<float>(dy, ldy, x, ldx, W, z, ldz, act, M, K, N, dx, dW, db,
                                           work, work_bytes, st)
                         : backward<uint16_t>(dy, ldy, x, ldx, W, z, ldz, act, M, K, N, dx, dW,
                                              db, work, work_bytes, st);
}
