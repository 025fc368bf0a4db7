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
#include <type_traits>

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

// Values k .. k + 7 of a row of K; past the end zero.
template <class T>
__device__ __forceinline__ void load_k8(const T* p, int k, int K, uint32_t* d) {
  constexpr bool F = sizeof(T) == 4;
  if (k + 8 <= K) {
    const u4 a = load16(p + k);
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j] = a[j];
    if (F) {
      const u4 b = load16(p + k + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) d[(4 + j) % (F ? 8 : 4)] = b[j];
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < (F ? 8 : 4); ++j) d[j] = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (k + j >= K) continue;
    if constexpr (F) d[j] = __builtin_bit_cast(uint32_t, p[k + j]);
    else d[j / 2] |= (uint32_t)p[k + j] << 16 * (j & 1);
  }
}

template <class T, bool ACROSS>
__device__ __forceinline__ void load_unit(const Operand<T>& o, int row, int k, int K, Raw<T>& v) {
  constexpr bool F = sizeof(T) == 4;
  const int r0 = min(row, o.rows - 1), r1 = min(row + 1, o.rows - 1);
  if (!ACROSS) {
    load_k8(o.p + (int64_t)r0 * o.ld, k, K, v.d);
    load_k8(o.p + (int64_t)r1 * o.ld, k, K, v.d + (F ? 8 : 4));
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool in = k + j < K;
    const T* const p = o.p + (int64_t)(in ? k + j : 0) * o.ld;
    if (row + 1 < o.rows) {
      if constexpr (F) {
        const u2 w = *reinterpret_cast<const u2at4*>(p + row);
        v.d[2 * j] = in ? w.x : 0;
        v.d[2 * j + 1] = in ? w.y : 0;
      } else {
        const uint32_t w = *reinterpret_cast<const u1at2*>(p + row);
        v.d[j] = in ? w : 0;
      }
    } else if constexpr (F) {
      v.d[2 * j] = in ? __builtin_bit_cast(uint32_t, p[r0]) : 0;
      v.d[2 * j + 1] = v.d[2 * j];
    } else {
      v.d[j] = in ? (uint32_t)p[r0] * 0x10001u : 0;
    }
  }
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

// Few rows, or few steps: 16 MB rows x 16 NB columns by eight waves that share the
// k, each reading its fragments straight from memory (64 of k at a time, UN of
// these requested together) and, in fp32, taking its values apart itself: no LDS,
// no barrier until the waves' sums are joined, in their order.  One token through
// 4096 x 4096 bf16 is 256 workgroups with 64 KB on its way to each CU.
constexpr int kDirectWaves = 8;

template <class T>
__device__ __forceinline__ void parts_of(const uint32_t* d, u4* o) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 4) {
      uint32_t h, m, l;
      cut2(__builtin_bit_cast(float, d[2 * j]), __builtin_bit_cast(float, d[2 * j + 1]), h, m, l);
      o[0][j] = h, o[1][j] = m, o[2][j] = l;
    } else {
      o[0][j] = d[j];
    }
  }
}

template <class T, int NB, int MB, int UN>
__global__ __launch_bounds__(64 * kDirectWaves, 2) void k_direct(Product<T> a) {
  constexpr bool F = sizeof(T) == 4;
  constexpr int NP = F ? 3 : 1, D = F ? 8 : 4, NW = kDirectWaves;
  __shared__ __align__(16) v4f part[NW][NB * MB][64];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int64_t w = vcg::xcd_tile(blockIdx.x, a.tiles);
  const int ti = (int)a.f_nj.div((uint32_t)w), tj = (int)(w - (int64_t)ti * a.f_nj.d);
  const int i0 = ti * 16 * MB, j0 = tj * 16 * NB;
  const T *pa[MB], *pb[NB];
#pragma unroll
  for (int i = 0; i < MB; ++i) pa[i] = a.A.p + (int64_t)min(i0 + 16 * i + r, a.I - 1) * a.A.ld;
#pragma unroll
  for (int j = 0; j < NB; ++j) pb[j] = a.B.p + (int64_t)min(j0 + 16 * j + r, a.J - 1) * a.B.ld;
  v4f acc[MB][NB], small[F ? MB : 1][F ? NB : 1];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
      if (F) small[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    }
  // slices: workgroups, then waves, take every 64-deep piece in turn
  const int each = NW * gridDim.y;
  const auto pieces = [&](int c, auto whole) {
    uint32_t da[UN][2][MB][D], db[UN][2][NB][D];
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = (c + u * each) * 64 + 32 * h + 8 * g, K = whole ? 0x7fffffff : a.K;
#pragma unroll
        for (int j = 0; j < NB; ++j) load_k8(pb[j], k, K, db[u][h][j]);
#pragma unroll
        for (int i = 0; i < MB; ++i) load_k8(pa[i], k, K, da[u][h][i]);
      }
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u4 fb[NB][NP];
#pragma unroll
        for (int j = 0; j < NB; ++j) parts_of<T>(db[u][h][j], fb[j]);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          u4 fa[NP];
          parts_of<T>(da[u][h][i], fa);
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            if constexpr (F) {
#pragma unroll
              for (int p = 0; p < 5; ++p)
                small[i][j] = mfma_bf16(fb[j][kPartA[p]], fa[kPartB[p]], small[i][j]);
              acc[i][j] += mfma_bf16(fb[j][0], fa[0], v4f{0.f, 0.f, 0.f, 0.f});
            } else {
              acc[i][j] = mfma_bf16(fb[j][0], fa[0], acc[i][j]);
            }
          }
        }
      }
  };
  for (int c = blockIdx.y * NW + wv; c * 64 < a.K; c += UN * each) {
    if ((c + (UN - 1) * each) * 64 + 64 <= a.K) pieces(c, std::true_type{});
    else pieces(c, std::false_type{});
  }
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      v4f s = acc[i][j];
      if (F) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float t = s[q] + small[i][j][q];
          s[q] = finite(t) ? t : s[q];
        }
      }
      part[wv][i * NB + j][lane] = s;
    }
  __syncthreads();
  for (int b = wv; b < NB * MB; b += NW) {
    v4f s = part[0][b][lane];
#pragma unroll
    for (int k = 1; k < NW; ++k) s += part[k][b][lane];
    const int64_t row = i0 + 16 * (b / NB) + r;
    const int col = j0 + 16 * (b % NB) + 4 * g;
    if (row >= a.I || col >= a.J) continue;
    const float v[4] = {s[0], s[1], s[2], s[3]};
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

// The slices' sums joined in their order.
template <class T>
__global__ __launch_bounds__(LNT) void k_join(Product<T> a) {
  const int nq = (a.J + 3) / 4;
  for (int64_t t = blockIdx.x * (int64_t)LNT + threadIdx.x; t < (int64_t)a.I * nq;
       t += (int64_t)gridDim.x * LNT) {
    const int64_t i = t / nq;
    const int j = (int)(t - i * nq) * 4;
    float v[4] = {-0.f, -0.f, -0.f, -0.f};  // adds nothing, not even a sign
    const int64_t step = (int64_t)a.I * a.J;
    const float* p = a.part + (int64_t)i * a.J + j;
    if (a.J % 4 == 0) {
#pragma unroll 8
      for (int s = 0; s < a.slices; ++s, p += step) {
        const v4f w = *reinterpret_cast<const v4f*>(p);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] += w[q];
      }
    } else {
#pragma unroll 4
      for (int s = 0; s < a.slices; ++s, p += step)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (j + q < a.J) v[q] += p[q];
    }
    finish(a, i, j, v);
  }
}

// Eight values j .. j + 7 of a row of n, as floats; past the end zero.
template <class T>
__device__ __forceinline__ void load8(const T* p, int j, int n, float* o) {
  uint32_t d[sizeof(T) == 4 ? 8 : 4];
  load_k8(p, j, n, d);
#pragma unroll
  for (int q = 0; q < 8; ++q)
    o[q] = sizeof(T) == 4 ? __builtin_bit_cast(float, d[q % (sizeof(T) * 2)])
                          : q & 1 ? bf_hi(d[q / 2]) : bf_lo(d[q / 2]);
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
  int n, np;  // values of a line, and with its padding
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
  load8(m.p + row * m.ld, j, m.n, v);
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
  int N, np, act, rows;
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
        load8(a.dy + r * a.ldy, j, a.N, d[q]);
        if (a.act != kNone) load8(a.z + r * a.ldz, j, a.N, z[q]);
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

// How a product is cut: the kernel, its shape, and the slices of k, by the time
// that they are expected to take (us).
enum Kernel { kProduct, kDirect, kTile };
struct Cut {
  Kernel kernel;
  int shape, slices, steps;
  int64_t tiles, nj;
  float us;
};

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The slices' sums written, read again and joined by a launch.
float join_us(int64_t slices, int64_t I, int64_t J) {
  return slices > 1 ? 4.f + 0.1f * slices + 8.f * slices * I * J / 4e6f : 0.f;
}

// A grid of `tiles` workgroups of `all` steps, cut into more slices while that
// helps: `alone` us a step for as many workgroups as share a CU, `shared` us for
// each of them.
void slice(Cut& best, Kernel kernel, int shape, int type, int64_t I, int64_t J, int64_t K, int bi,
           int bj, int bk, float alone, float shared, int share) {
  const int64_t all = div_up(K, bk);
  const float hbm = (type == VC_FP32 ? 6.f : 2.f) * (I + J) * K / 4.5e6f;
  const int64_t nj = div_up(J, bj), tiles = div_up(I, bi) * nj;
  for (int64_t want = 1; want <= 32 && (want == 1 || 4 * want <= all); want *= 2) {
    const int64_t steps = div_up(all, want) > 0 ? div_up(all, want) : 1;
    const int64_t slices = div_up(all, steps) > 0 ? div_up(all, steps) : 1;
    const int64_t load = div_up(tiles * slices, kCus);
    const float a = steps * alone * div_up(load, share), s = steps * shared * load;
    const float work = a > s ? a : s;
    const float us = 4.f + (work > hbm ? work : hbm) + join_us(slices, I, J);
    if (us < best.us) best = {kernel, shape, (int)slices, (int)steps, tiles, nj, us};
  }
}

// The kernel of 64 x 64 tiles by registers: steps of 32 (bf16: 64).
Cut cut_product(int type, int64_t I, int64_t J, int64_t K) {
  Cut c = {};
  c.us = 1e30f;
  const bool f = type == VC_FP32;
  slice(c, kProduct, 0, type, I, J, K, 64, 64, f ? 32 : 64, f ? 1.0f : 0.9f, f ? 0.9f : 0.5f, 2);
  return c;
}

// The tiled kernels: a step of one tile alone on a CU, and of each of several that
// share one (measured on 264 x 328 and 512 x 512 outputs, and on 8192 x 16384 and
// 4096 x 4096).
constexpr float kStepAlone[2][3] = {{1.15f, 0.50f, 0.f}, {1.45f, 1.0f, 0.45f}};
constexpr float kStepShared[2][3] = {{1.39f, 0.46f, 0.f}, {1.95f, 0.55f, 0.21f}};
constexpr int kShare[2][3] = {{1, 3, 1}, {1, 2, 4}};

Cut cut_tiles(int type, int64_t I, int64_t J, int64_t K) {
  Cut c = {};
  c.us = 1e30f;
  const int b = type == VC_FP32 ? 0 : 1;
  for (int shape = 0; shape < (b ? 3 : 2); ++shape) {
    const TileShape t = tile_shape(type, shape);
    slice(c, kTile, shape, type, I, J, K, t.bi, t.bj, t.bk, kStepAlone[b][shape],
          kStepShared[b][shape], kShare[b][shape]);
  }
  return c;
}

// The direct kernel: 16 rows by 16 columns, 32 by 16, 64 by 16, 64 by 32.  A
// workgroup's operands come at about 25 GB/s a CU (sixteen rows a load, 16 bytes a
// lane), all of them together at no
// more than the memory's rate.
constexpr int kDirectRows[4] = {16, 32, 64, 64}, kDirectCols[4] = {16, 16, 16, 32};

Cut cut_direct(int type, int64_t I, int64_t J, int64_t K) {
  Cut c = {};
  c.us = 1e30f;
  const float e = type == VC_FP32 ? 4.f : 2.f;
  for (int shape = 0; shape < 4; ++shape) {
    const int bi = kDirectRows[shape], bj = kDirectCols[shape];
    const int64_t nj = div_up(J, bj), tiles = div_up(I, bi) * nj;
    int64_t s = 1;
    while (tiles * s < kCus && 1024 * s < K && s < 16) s *= 2;
    const float own = e * ((I < bi ? I : bi) + bj) * (float)K / s;
    const float l2 = div_up(tiles * s, kCus) * own / 25e3f;
    const float hbm = e * (I + J) * (float)K / 4.5e6f;
    const float us = 3.f + (l2 > hbm ? l2 : hbm) + join_us(s, I, J);
    if (us < c.us) c = {kDirect, shape, (int)s, 0, tiles, nj, us};
  }
  return c;
}

// Whether tiles can be made of matrices with lines of this length at all.
bool tile_lines(int64_t n) { return n > 0 && n < (1 << 21); }

// The pass that makes `n` values into parts.
float pack_us(int type, int64_t n) { return 4.f + n * (type == VC_FP32 ? 10.f : 4.f) / 4e6f; }

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
  const dim3 grid((unsigned)c.tiles, (unsigned)c.slices);
  if (c.kernel == kTile) {
    run_tiles<T>(a, c.shape, XA, XB, st);
  } else if constexpr (XB) {
    k_product<T, XA, XB, 64, 64><<<grid, LNT, 0, st>>>(a);
  } else {
    constexpr bool F = sizeof(T) == 4;
    const int threads = 64 * kDirectWaves;
    if (c.shape == 0) k_direct<T, 1, 1, F ? 2 : 8><<<grid, threads, 0, st>>>(a);
    else if (c.shape == 1) k_direct<T, 1, 2, F ? 2 : 4><<<grid, threads, 0, st>>>(a);
    else if (c.shape == 2) k_direct<T, 1, 4, F ? 1 : 2><<<grid, threads, 0, st>>>(a);
    else k_direct<T, 2, 4, F ? 1 : 2><<<grid, threads, 0, st>>>(a);
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
  if (na + nb > 0) k_pack<T><<<(unsigned)(na + nb), LNT, 0, st>>>(a, b, na);
}

bool sizes_ok(int64_t M, int K, int N) {
  return M >= 0 && M <= 0x7fffff00 && K >= 0 && K <= (1 << 30) && N >= 0 && N <= (1 << 30);
}

struct ForwardPlan {
  Cut c;
  int64_t x, W, part, bytes;  // offsets in the workspace, and its size
};

ForwardPlan plan_forward(int type, int64_t M, int K, int N) {
  ForwardPlan p;
  p.c = cut_direct(type, M, N, K);
  if (tile_lines(K)) {
    const Cut t = cut_tiles(type, M, N, K);
    const float pack = type == VC_FP32 || K % 8 ? pack_us(type, (M + N) * K) : 0.f;
    if (t.us + pack < p.c.us) p.c = t;
  }
  const bool tiles = p.c.kernel == kTile;
  p.x = 0;
  p.W = tiles ? parts_bytes(type, M, K) : 0;
  p.part = p.W + (tiles ? parts_bytes(type, N, K) : 0);
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
  a.A = {(const T*)x, ldx, (int)M};
  a.B = {(const T*)W, K, N};
  a.I = (int)M;
  a.J = N;
  a.K = K;
  a.bias = (const T*)bias;
  a.res = (const T*)res;
  a.ldr = ldr;
  a.out = (T*)y;
  a.z = (T*)z;
  a.act = act;
  if (p.c.kernel == kTile) {
    const int kp = (int)up8(K);
    Pack<T> px = {}, pw = {};
    if (!as_it_is((const T*)x, ldx, K)) px = {(const T*)x, ldx, M, K, kp, (uint16_t*)(base + p.x)};
    if (!as_it_is((const T*)W, K, K)) pw = {(const T*)W, K, N, K, kp, (uint16_t*)(base + p.W)};
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
  p.cx = cut_product(type, M, K, N);
  p.cw = cut_product(type, N, K, M);
  p.tiles = false;
  if (tile_lines(K) && tile_lines(N)) {
    const Cut x = cut_tiles(type, M, K, N), w = cut_tiles(type, N, K, M);
    const float pack = type == VC_FP32 || K % 8 ? pack_us(type, (M + N) * K) : 0.f;
    p.tiles = (need & 1 ? x.us : 0.f) + (need & 2 ? w.us : 0.f) + pack <
              (need & 1 ? p.cx.us : 0.f) + (need & 2 ? p.cw.us : 0.f);
    if (p.tiles) p.cx = x, p.cw = w;
  }
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
    k_slope<T><<<dim3((unsigned)div_up(N, kSlopeCols), (unsigned)p.blocks), LNT, 0, st>>>(s);
  }
  if (db && N > 0)
    k_slope_join<T><<<(unsigned)div_up(N, 32), LNT, 0, st>>>((float*)(base + p.sums), p.blocks, N,
                                                             (T*)db);
  VC_LAUNCH_CHECK();
  Product<T> a = {};
  if (p.tiles && (need & 3)) {
    Pack<T> pw = {}, px = {};
    if (dx && !as_it_is((const T*)W, K, K)) pw = {(const T*)W, K, N, K, kp, (uint16_t*)(base + p.W)};
    if (dW && !as_it_is((const T*)x, ldx, K)) px = {(const T*)x, ldx, M, K, kp, (uint16_t*)(base + p.x)};
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
    a.A = {dz, ldd, (int)M};
    a.B = {(const T*)W, K, K};
    a.I = (int)M;
    a.J = K;
    a.K = N;
    a.out = (T*)dx;
    const int rc = run_product<T, false, true>(a, p.cx, base + p.part, work_bytes - p.part, st);
    if (rc != VC_OK) return rc;
  }
  if (dW) {
    a.A = {dz, ldd, N};
    a.B = {(const T*)x, ldx, K};
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
