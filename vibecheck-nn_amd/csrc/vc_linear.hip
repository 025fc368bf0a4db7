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
#include "vc_linear.h"

namespace {

using namespace vcl;

constexpr int LNT = 256;  // threads: four waves, 2 x 2 over the tile

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

// Eight values j .. j + 7 of a row of n, as floats; past the end zero.
template <class T>
__device__ __forceinline__ void load8(const T* p, int j, int n, bool wide, float* o) {
  if (wide && j + 8 <= n) {
    if constexpr (sizeof(T) == 4) {
      const v4f a = *reinterpret_cast<const v4f*>(p + j), b = *reinterpret_cast<const v4f*>(p + j + 4);
#pragma unroll
      for (int q = 0; q < 4; ++q) o[q] = a[q], o[4 + q] = b[q];
    } else {
      const u4 a = *reinterpret_cast<const u4*>(p + j);
#pragma unroll
      for (int q = 0; q < 4; ++q) o[2 * q] = bf_lo(a[q]), o[2 * q + 1] = bf_hi(a[q]);
    }
    return;
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) o[q] = j + q < n ? get(p + j + q) : 0.f;
}

// Eight values as 16 bytes of each part, part p at p planes.
template <class T>
__device__ __forceinline__ void store_parts(const float* v, uint16_t* to, int64_t plane) {
  u4 h, m, l;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (sizeof(T) == 4) {
      uint32_t a, b, c;
      cut2(v[2 * q], v[2 * q + 1], a, b, c);
      h[q] = a, m[q] = b, l[q] = c;
    } else {
      h[q] = bf_pack(v[2 * q], v[2 * q + 1]);
    }
  }
  *reinterpret_cast<u4*>(to) = h;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<u4*>(to + plane) = m;
    *reinterpret_cast<u4*>(to + 2 * plane) = l;
  }
}

// Up to two matrices as parts for the tiled products, their lines padded with
// zeros to a multiple of eight.
template <class T>
struct Pack {
  const T* p;
  int64_t ld, rows;
  int n, np, wide;  // values of a line, and with its padding
  uint16_t* to;
};

template <class T>
__global__ __launch_bounds__(LNT) void k_pack(Pack<T> a, Pack<T> b, int64_t split) {
  const bool second = blockIdx.x >= split;
  const Pack<T> m = second ? b : a;
  const int64_t t = (blockIdx.x - (second ? split : 0)) * (int64_t)LNT + threadIdx.x;
  const int c = m.np / 8;
  const int64_t row = t / c;
  if (row >= m.rows) return;
  const int j = (int)(t - row * c) * 8;
  float v[8];
  load8(m.p + row * m.ld, j, m.n, m.wide, v);
  store_parts<T>(v, m.to + row * m.np + j, m.rows * m.np);
}

// dz = dy act'(z), and the columns' sums of each block of rows.  dz as values, or
// as parts for the tiled products (lines of np values, zeros past N).
template <class T>
struct Slope {
  const T *dy, *z;
  int64_t ldy, ldz;
  T* dz;           // lines of N, or null
  uint16_t* parts; // or null
  float* sums;     // (blocks of rows, N), or null
  int64_t M;
  int N, np, act, rows, wide;
};

constexpr int kSlopeCols = 256;  // of a workgroup: eight a thread, eight rows at a time

template <class T>
__global__ __launch_bounds__(LNT) void k_slope(Slope<T> a) {
  __shared__ float part[8][kSlopeCols + 8];
  const int c = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int j = blockIdx.x * kSlopeCols + 8 * c;
  const int64_t m0 = (int64_t)blockIdx.y * a.rows;
  const int64_t m1 = m0 + a.rows < a.M ? m0 + a.rows : a.M;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (j < a.N) {
    for (int64_t m = m0 + y; m < m1; m += 32) {  // four rows' loads before the first is used
      float d[4][8], z[4][8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t r = m + 8 * q < m1 ? m + 8 * q : m;
        load8(a.dy + r * a.ldy, j, a.N, a.wide, d[q]);
        if (a.act != kNone) load8(a.z + r * a.ldz, j, a.N, a.wide, z[q]);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t r = m + 8 * q;
        if (r >= m1) break;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (a.act != kNone) d[q][i] *= slope(z[q][i], a.act);
          sum[i] += d[q][i];
        }
        if (a.parts) store_parts<T>(d[q], a.parts + r * a.np + j, a.M * a.np);
        if (a.dz) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (j + i < a.N) put(a.dz + r * a.N + j + i, d[q][i]);
        }
      }
    }
  }
  if (!a.sums) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) part[y][8 * c + i] = sum[i];
  __syncthreads();
  const int k = blockIdx.x * kSlopeCols + threadIdx.x;
  if (k >= a.N) return;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += part[i][threadIdx.x];
  a.sums[(int64_t)blockIdx.y * a.N + k] = s;
}

// The blocks' sums joined: 32 columns a workgroup, eight threads a column.
template <class T>
__global__ __launch_bounds__(LNT) void k_slope_join(const float* sums, int blocks, int N, T* db) {
  __shared__ float part[8][32];
  const int c = threadIdx.x & 31, y = threadIdx.x >> 5, j = blockIdx.x * 32 + c;
  float s = 0.f;
  if (j < N)
    for (int b = y; b < blocks; b += 8) s += sums[(int64_t)b * N + j];
  part[y][c] = s;
  __syncthreads();
  if (y || j >= N) return;
  for (int i = 1; i < 8; ++i) s += part[i][c];
  put(db + j, s);
}

int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }
int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }
constexpr int64_t kCus = 256;

// How a product is cut: the kernel (shape -1: k_product, else k_tile's) and the
// slices of k, by the time that they are expected to take.
struct Cut {
  int shape, slices, steps;
  int64_t tiles, nj;
};

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

Cut cut_general(int type, int64_t I, int64_t J, int64_t K) {
  const int64_t all = div_up(K, type == VC_FP32 ? 32 : 64);
  Cut c;
  c.shape = -1;
  c.nj = div_up(J, 64);
  c.tiles = div_up(I, 64) * c.nj;
  int64_t s = 1;
  if (c.tiles < kCus && all >= 16) {
    s = kCus / c.tiles;
    if (s > all / 8) s = all / 8;
    if (s > 64) s = 64;
  }
  c.steps = (int)div_up(all, s);
  if (c.steps < 1) c.steps = 1;
  c.slices = (int)div_up(all, c.steps);
  if (c.slices < 1) c.slices = 1;
  return c;
}

// Of the tiled kernels: a step of one tile alone on a CU, and of each of several
// that share one (us, measured on 264 x 328 and 8192 x 16384 outputs).
constexpr float kStepAlone[2][3] = {{2.0f, 1.5f, 0.50f}, {2.1f, 1.0f, 0.45f}};
constexpr float kStepShared[2][3] = {{2.7f, 1.54f, 0.46f}, {2.2f, 0.55f, 0.21f}};
constexpr int kShare[2][3] = {{1, 1, 3}, {1, 2, 4}};

Cut cut_tiles(int type, int64_t I, int64_t J, int64_t K) {
  Cut best = {};
  float least = 1e30f;
  for (int shape = 0; shape < 3; ++shape) {
    const TileShape t = tile_shape(type, shape);
    const int b = type == VC_FP32 ? 0 : 1;
    const int64_t all = div_up(K, t.bk), nj = div_up(J, t.bj), tiles = div_up(I, t.bi) * nj;
    for (int64_t want = 1; want <= 16 && want <= all; want *= 2) {
      const int64_t steps = div_up(all, want), slices = div_up(all, steps);
      const int64_t load = div_up(tiles * slices, kCus);
      const float alone = kStepAlone[b][shape] * div_up(load, kShare[b][shape]);
      const float shared = kStepShared[b][shape] * load;
      float us = steps * (alone > shared ? alone : shared);
      // the slices' sums written, read again and joined by a launch
      if (slices > 1) us += 4.f + 8.f * slices * I * J / 4e6f;
      if (us < least) {
        least = us;
        best = {shape, (int)slices, (int)steps, tiles, nj};
      }
    }
  }
  return best;
}

// Which products are tiled: those whose time the tiles cut by more than their
// parts' pass and its launch cost.
bool tiled(int type, int64_t M, int64_t K, int64_t N) {
  return K > 0 && (double)M * K * N >= (type == VC_FP32 ? 3e8 : 1.5e8) && K < (1 << 21) &&
         N < (1 << 21);
}

Cut cut(int type, int64_t I, int64_t J, int64_t K, bool tiles) {
  return tiles ? cut_tiles(type, I, J, K) : cut_general(type, I, J, K);
}

int64_t part_bytes(const Cut& c, int64_t I, int64_t J) {
  return c.slices > 1 ? up256(4 * c.slices * I * J) : 0;
}

// A matrix of `rows` lines as parts, and whether it has to be made into them.
template <class T>
bool as_it_is(const T* p, int64_t ld, int64_t n) {
  return sizeof(T) == 2 && aligned16(p) && ld % 8 == 0 && n % 8 == 0 && ld < (1 << 21);
}
int64_t parts_bytes(int type, int64_t rows, int64_t n) {
  return up256((type == VC_FP32 ? 6 : 2) * rows * up8(n));
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
int run_product(Product<T> a, const Cut& c, void* work, int64_t work_bytes, hipStream_t st) {
  if (a.I == 0 || a.J == 0) return VC_OK;
  if (c.tiles > (1ll << 23)) return VC_ERR_UNSUPPORTED;  // threads of a grid axis: below 2^32
  if (part_bytes(c, a.I, a.J) > work_bytes) return VC_ERR_OOM;
  a.wide = a.J % 4 == 0 && quads<T>(a.out, a.J) && quads<T>(a.z, a.J) && quads<T>(a.res, a.ldr);
  a.slices = c.slices;
  a.steps = c.steps;
  a.part = (float*)work;
  a.tiles = c.tiles;
  a.f_nj = vcg::FastDiv::make((uint32_t)c.nj);
  if (c.shape >= 0) {
    run_tiles<T>(a, c.shape, XA, XB, st);
  } else {
    a.A.vec = XA ? wide_across(a.A.p, a.A.ld, a.A.rows) : wide_rows(a.A.p, a.A.ld, a.K);
    a.B.vec = XB ? wide_across(a.B.p, a.B.ld, a.B.rows) : wide_rows(a.B.p, a.B.ld, a.K);
    k_product<T, XA, XB, 64, 64><<<dim3((unsigned)c.tiles, (unsigned)c.slices), LNT, 0, st>>>(a);
  }
  if (c.slices > 1) {
    const int64_t n = (int64_t)a.I * ((a.J + 3) / 4);
    const int64_t blocks = div_up(n, LNT);
    k_join<T><<<(unsigned)(blocks < 4096 ? blocks : 4096), LNT, 0, st>>>(a);
  }
  VC_LAUNCH_CHECK();
  return VC_OK;
}

template <class T>
void run_pack(Pack<T> a, Pack<T> b, hipStream_t st) {
  const int64_t na = a.to ? div_up(a.rows * (a.np / 8), LNT) : 0;
  const int64_t nb = b.to ? div_up(b.rows * (b.np / 8), LNT) : 0;
  a.wide = aligned16(a.p) && a.ld % (16 / (int)sizeof(T)) == 0;
  b.wide = aligned16(b.p) && b.ld % (16 / (int)sizeof(T)) == 0;
  if (na + nb > 0) k_pack<T><<<(unsigned)(na + nb), LNT, 0, st>>>(a, b, na);
}

bool sizes_ok(int64_t M, int K, int N) {
  return M >= 0 && M <= 0x7fffff00 && K >= 0 && K <= 0x7fffff00 && N >= 0 && N <= 0x7fffff00;
}

struct ForwardPlan {
  bool tiles;
  Cut c;
  int64_t x, W, part, bytes;  // offsets in the workspace, and its size
};

ForwardPlan plan_forward(int type, int64_t M, int K, int N) {
  ForwardPlan p;
  p.tiles = tiled(type, M, K, N);
  p.c = cut(type, M, N, K, p.tiles);
  p.x = 0;
  p.W = p.tiles ? parts_bytes(type, M, K) : 0;
  p.part = p.W + (p.tiles ? parts_bytes(type, N, K) : 0);
  p.bytes = p.part + part_bytes(p.c, M, N);
  return p;
}

template <class T>
int forward(const void* x, int64_t M, int K, int64_t ldx, const void* W, int N, const void* bias,
            int act, const void* res, int64_t ldr, void* y, void* z, void* work,
            int64_t work_bytes, hipStream_t st) {
  constexpr int type = sizeof(T) == 4 ? VC_FP32 : VC_BF16;
  const ForwardPlan p = plan_forward(type, M, K, N);
  if (p.bytes > work_bytes || (p.bytes && !work)) return VC_ERR_OOM;
  char* const base = (char*)work;
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
  if (p.tiles) {
    const int kp = (int)up8(K);
    Pack<T> px = {}, pw = {};
    if (!as_it_is((const T*)x, ldx, K)) px = {(const T*)x, ldx, M, K, kp, 0, (uint16_t*)(base + p.x)};
    if (!as_it_is((const T*)W, K, K)) pw = {(const T*)W, K, N, K, kp, 0, (uint16_t*)(base + p.W)};
    run_pack(px, pw, st);
    a.pa = px.to ? px.to : (const uint16_t*)x;
    a.lda = px.to ? kp : ldx;
    a.planeA = M * kp;
    a.pb = pw.to ? pw.to : (const uint16_t*)W;
    a.ldb = kp;
    a.planeB = (int64_t)N * kp;
    a.K = kp;
  }
  return run_product<T, false, false>(a, p.c, base + p.part, work_bytes - p.part, st);
}

// Rows of a block of k_slope: at most 256 blocks.
int slope_rows(int64_t M) {
  const int64_t r = (M + 255) / 256;
  return (int)(r < 64 ? 64 : r);
}

struct BackwardPlan {
  bool tiles;
  Cut cx, cw;
  int rows, blocks;
  int64_t dz, W, x, sums, part, bytes;  // offsets in the workspace, and its size
};

BackwardPlan plan_backward(int type, int64_t M, int K, int N, int act, int need) {
  BackwardPlan p;
  const int64_t e = type == VC_FP32 ? 4 : 2;
  p.tiles = tiled(type, M, K, N);
  p.cx = cut(type, M, K, N, p.tiles);
  p.cw = cut(type, N, K, M, p.tiles);
  p.rows = slope_rows(M);
  p.blocks = (int)div_up(M, p.rows);
  p.dz = 0;
  int64_t at = 0;
  if (need & 3) at += p.tiles ? parts_bytes(type, M, N) : act != kNone ? up256(e * M * N) : 0;
  p.W = at;
  if ((need & 1) && p.tiles) at += parts_bytes(type, N, K);
  p.x = at;
  if ((need & 2) && p.tiles) at += parts_bytes(type, M, K);
  p.sums = at;
  if (need & 4) at += up256(4ll * p.blocks * N);
  p.part = at;
  int64_t most = need & 1 ? part_bytes(p.cx, M, K) : 0;
  const int64_t b = need & 2 ? part_bytes(p.cw, N, K) : 0;
  p.bytes = at + (b > most ? b : most);
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
  const int np = (int)up8(N), kp = (int)up8(K);
  // dy itself is dz where nothing is between them and the products can read it
  const bool made = (need & 3) && (act != kNone || (p.tiles && !as_it_is((const T*)dy, ldy, N)));
  if (N > 0 && M > 0 && (made || db)) {
    Slope<T> s = {};
    s.dy = (const T*)dy;
    s.z = (const T*)z;
    s.ldy = ldy;
    s.ldz = ldz;
    if (made && p.tiles) s.parts = (uint16_t*)(base + p.dz);
    else if (made) s.dz = (T*)(base + p.dz);
    s.sums = db ? (float*)(base + p.sums) : nullptr;
    s.M = M;
    s.N = N;
    s.np = np;
    s.act = act;
    s.rows = p.rows;
    const int per = 16 / (int)sizeof(T);
    s.wide = aligned16(dy) && ldy % per == 0 && (act == kNone || (aligned16(z) && ldz % per == 0));
    k_slope<T><<<dim3((unsigned)div_up(N, kSlopeCols), (unsigned)p.blocks), LNT, 0, st>>>(s);
  }
  if (db && N > 0)
    k_slope_join<T><<<(unsigned)div_up(N, 32), LNT, 0, st>>>((float*)(base + p.sums), p.blocks, N,
                                                             (T*)db);
  VC_LAUNCH_CHECK();
  Product<T> a = {};
  if (p.tiles && (need & 3)) {
    Pack<T> pw = {}, px = {};
    if (dx && !as_it_is((const T*)W, K, K)) pw = {(const T*)W, K, N, K, kp, 0, (uint16_t*)(base + p.W)};
    if (dW && !as_it_is((const T*)x, ldx, K)) px = {(const T*)x, ldx, M, K, kp, 0, (uint16_t*)(base + p.x)};
    run_pack(pw, px, st);
    a.pa = made ? (const uint16_t*)(base + p.dz) : (const uint16_t*)dy;
    a.lda = made ? np : ldy;
    a.planeA = M * np;
    if (dx) {
      a.pb = pw.to ? pw.to : (const uint16_t*)W;
      a.ldb = kp;
      a.planeB = (int64_t)N * kp;
    }
    if (dx) {
      a.I = (int)M;
      a.J = K;
      a.K = N;
      a.out = (T*)dx;
      const int rc = run_product<T, false, true>(a, p.cx, base + p.part, work_bytes - p.part, st);
      if (rc != VC_OK) return rc;
    }
    if (dW) {
      a.pb = px.to ? px.to : (const uint16_t*)x;
      a.ldb = px.to ? kp : ldx;
      a.planeB = M * kp;
      a.I = N;
      a.J = K;
      a.K = (int)M;
      a.out = (T*)dW;
      return run_product<T, true, true>(a, p.cw, base + p.part, work_bytes - p.part, st);
    }
    return VC_OK;
  }
  const T* const dz = made ? (const T*)(base + p.dz) : (const T*)dy;
  const int64_t ldd = made ? N : ldy;
  if (dx) {
    a.A = {dz, ldd, (int)M, 0};
    a.B = {(const T*)W, K, K, 0};
    a.I = (int)M;
    a.J = K;
    a.K = N;
    a.out = (T*)dx;
    const int rc = run_product<T, false, true>(a, p.cx, base + p.part, work_bytes - p.part, st);
    if (rc != VC_OK) return rc;
  }
  if (dW) {
    a.A = {dz, ldd, N, 0};
    a.B = {(const T*)x, ldx, K, 0};
    a.I = N;
    a.J = K;
    a.K = (int)M;
    a.out = (T*)dW;
    return run_product<T, true, true>(a, p.cw, base + p.part, work_bytes - p.part, st);
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
  return plan_forward(type, M, K, N).bytes;
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
