// The fc layer itself, forward and backward, in fp32 and bf16:
//   z = x W^T + b, y = act(z) + r;
//   dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum over rows of dz.
//
// Every product is C[i][j] = sum_k A(i, k) B(j, k) on the matrix cores, summed in
// fp32; an operand's k may be its contiguous axis or its other one (dx reads W, dW
// reads dz and x across).  An fp32 value is three bf16 parts, here cut rather than
// rounded at the first (h = the value's upper 16 bits), so that a finite value never
// becomes an infinity; six of the nine part products are formed (vc_split.h), what
// is left out is under 2^-22 of |x| |w|.  Where a sum is not finite it is taken from
// the largest parts' products (here) or summed again from the values
// (vc_linear_tile.hip): the small parts of an infinity are not numbers.
//
// Four kernels, by the time that each is expected to take (choose, cut_direct):
//   k_direct      few rows or short sums, no LDS: 1 x 4096 x 4096 bf16 7.7 us;
//   k_tile(s)     vc_linear_tile.hip, 64 to 256 square from bf16 parts in memory:
//                 8192 x 4096 x 16384 bf16 900 us (1222 TFLOP/s);
//   k_raw         the same file, fp32 forward without parts: 512 x 784 x 1024 12.2 us
//                 (by tiles, with the pass that makes the parts, 16.6);
//   k_product(s)  64 x 64 through registers, from the values as they are: what is
//                 too small for the parts' pass, or not aligned.
// Backward is a launch for dz with its columns' sums, parts and copies (none where dy is
// dz and all is aligned), one for both products (one each where they differ in shape or
// each fills the chip) and, where k went in slices, one that joins the slices' and the
// columns' sums.
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

// Values k .. k + 7 of a row of K; past the end zero.  whole (the same in all
// lanes): none is.  Every lane loads, and moves and masks what it has afterwards: a
// branch that lanes do not share would have each load waited for before the next.
template <class T>
__device__ __forceinline__ void load_k8(const T* p, int k, int K, bool whole, uint32_t* d) {
  constexpr bool F = sizeof(T) == 4;
  constexpr int D = F ? 8 : 4;
  if (whole || K >= 8) {
    const int at = whole ? k : min(k, K - 8);
    const u4 a = load16(p + at);
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j] = a[j];
    if (F) {
      const u4 b = load16(p + at + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) d[(4 + j) % D] = b[j];
    }
    if (whole) return;
    const int over = min(k - at, 8);  // values to drop from the front, zeros behind
#pragma unroll
    for (int step = 4; step >= 1; step /= 2) {
      const bool on = over & step;
      if (F || step > 1) {
        const int n = F ? step : step / 2;
#pragma unroll
        for (int j = 0; j < D; ++j) d[j] = on ? (j + n < D ? d[(j + n) % D] : 0) : d[j];
      } else {
#pragma unroll
        for (int j = 0; j < D; ++j)
          d[j] = on ? d[j] >> 16 | (j + 1 < D ? d[(j + 1) % D] << 16 : 0) : d[j];
      }
    }
#pragma unroll
    for (int j = 0; j < D; ++j) d[j] = over >= 8 ? 0 : d[j];
    return;
  }
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const T v = p[min(k + j, K - 1)];
    if constexpr (F) w[j] = __builtin_bit_cast(uint32_t, v);
    else w[j] = v;
    w[j] = k + j < K ? w[j] : 0;
  }
#pragma unroll
  for (int j = 0; j < D; ++j) d[j] = F ? w[j] : w[2 * j % 8] | w[(2 * j + 1) % 8] << 16;
}

template <class T, bool ACROSS>
__device__ __forceinline__ void load_unit(const Operand<T>& o, int row, int k, int K, bool whole,
                                          Raw<T>& v) {
  constexpr bool F = sizeof(T) == 4;
  if (!ACROSS) {
    const int r0 = min(row, o.rows - 1), r1 = min(row + 1, o.rows - 1);
    load_k8(o.p + (int64_t)r0 * o.ld, k, K, whole, v.d);
    load_k8(o.p + (int64_t)r1 * o.ld, k, K, whole, v.d + (F ? 8 : 4));
    return;
  }
  // past the last row the last two (mend_unit)
  const int r0 = max(min(row, o.rows - 2), 0);
  if (o.rows > 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const T* const p = o.p + (int64_t)(whole ? k + j : min(k + j, K - 1)) * o.ld + r0;
      if constexpr (F) {
        const u2 w = *reinterpret_cast<const u2at4*>(p);
        v.d[2 * j] = w.x;
        v.d[2 * j + 1] = w.y;
      } else {
        v.d[j] = *reinterpret_cast<const u1at2*>(p);
      }
    }
    if (whole) return;  // loads alone: nothing here waits for them
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const T w = o.p[(int64_t)min(k + j, K - 1) * o.ld];
      if constexpr (F) v.d[2 * j] = v.d[2 * j + 1] = __builtin_bit_cast(uint32_t, w);
      else v.d[j] = (uint32_t)w | (uint32_t)w << 16;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool in = k + j < K;
    if constexpr (F) {
      v.d[2 * j] = in ? v.d[2 * j] : 0;
      v.d[2 * j + 1] = in ? v.d[2 * j + 1] : 0;
    } else {
      v.d[j] = in ? v.d[j] : 0;
    }
  }
}

// An operand of an odd number of rows, read across: its last row is the second of
// the pair that was read for it, and goes to the first's place.
template <class T>
__device__ __forceinline__ void mend_unit(bool last, Raw<T>& v) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (sizeof(T) == 4) v.d[2 * j] = last ? v.d[2 * j + 1] : v.d[2 * j];
    else v.d[j] = last ? v.d[j] >> 16 : v.d[j];
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

// 64 x 64 tiles, steps of 32 KS, by G groups of four waves that take the steps in
// turn (few tiles: a CU's waves on one of them) and join their sums in order.  A
// unit is eight k of two rows, read into registers while the step before is
// multiplied, then laid into the other of the group's two LDS buffers: [k
// step][part][row][four 16-byte chunks], chunk c of row r at c ^ (r / 2 mod 4), so
// that a fragment read meets every bank evenly.  The columns' fragment is the
// matrix step's first operand: a lane holds four consecutive columns of one row.  fp32:
// the five small part products run on in an accumulator of their own, the largest
// starts from zero each step and is added in fp32.
constexpr int kTileSide = 64;
template <class T>
constexpr int product_lds(int groups) {  // bytes
  return groups * 2 * (sizeof(T) == 4 ? 3 : 2) * 2 * kTileSide * 64;
}

template <class T, bool XA, bool XB, int G>
__device__ __forceinline__ void product_tile(const Product<T>& a, uint32_t block, u4* shared) {
  constexpr bool F = sizeof(T) == 4;
  constexpr int NP = F ? 3 : 1, KS = F ? 1 : 2, B = kTileSide, M2 = 2;
  constexpr int U = B / 2 * 4 * KS, NU = 2 * U / LNT;  // units of an operand, of a thread
  constexpr int S = KS * NP * B * 4;                   // 16-byte pieces of an operand's buffer
  const int tid = threadIdx.x & (LNT - 1), lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = G == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int g = lane >> 4, r = lane & 15;
  const int slice = __builtin_amdgcn_readfirstlane(block / (uint32_t)a.tiles);
  const uint32_t w = (uint32_t)vcg::xcd_tile(block - slice * (uint32_t)a.tiles, a.tiles);
  const int ti = (int)a.f_nj.div(w), tj = (int)w - ti * (int)a.f_nj.d;
  const int i0 = ti * B, j0 = tj * B, s0 = slice * a.steps;
  const int steps = min(a.steps, (a.K + 32 * KS - 1) / (32 * KS) - s0);
  const int wi = wv >> 1, wj = wv & 1;
  u4* const lds = shared + grp * 4 * S;

  v4f acc[M2][M2], small[F ? M2 : 1][F ? M2 : 1];
#pragma unroll
  for (int i = 0; i < M2; ++i)
#pragma unroll
    for (int j = 0; j < M2; ++j) {
      acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
      if (F) small[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    }

  Raw<T> raw[NU];
  const auto place = [&](int n, bool& isA, int& row, int& c) {
    const int u0 = tid + n * LNT;
    isA = __builtin_amdgcn_readfirstlane(u0) < U;
    const int u = isA ? u0 : u0 - U;
    const bool across = isA ? XA : XB;
    row = 2 * (across ? u % (B / 2) : u / (4 * KS));
    c = across ? u / (B / 2) : u % (4 * KS);
  };
  const auto load = [&](int s) {
    const bool whole = (s0 + s + 1) * 32 * KS <= a.K;
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      bool isA;
      int row, c;
      place(n, isA, row, c);
      const int k = (s0 + s) * 32 * KS + 8 * c;
      if (isA) load_unit<T, XA>(a.A, i0 + row, k, a.K, whole, raw[n]);
      else load_unit<T, XB>(a.B, j0 + row, k, a.K, whole, raw[n]);
    }
  };
  const auto store = [&](int buf) {
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      bool isA;
      int row, c;
      place(n, isA, row, c);
      u4* const at = lds + buf * 2 * S + (isA ? 0 : S) + (c >> 2) * NP * B * 4;
      const int rows = isA ? a.A.rows : a.B.rows, at0 = isA ? i0 : j0;
      if ((isA ? XA : XB) && (rows & 1) && at0 + B >= rows) mend_unit(at0 + row >= rows - 1, raw[n]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u4 o[NP];
        if (isA) unit_row<T, XA>(raw[n], h, o);
        else unit_row<T, XB>(raw[n], h, o);
        const int q = (row + h) * 4 + ((c & 3) ^ ((row >> 1) & 3));
#pragma unroll
        for (int p = 0; p < NP; ++p) at[p * B * 4 + q] = o[p];
      }
    }
  };
  if (grp < steps) {
    load(grp);
    store(0);
  }
  int buf = 0;
#pragma unroll 1
  for (int s = grp; s - grp < steps; s += G, buf ^= 1) {
    __syncthreads();  // this step is laid down, the buffer of the one before is read
    if (s + G < steps) load(s + G);
    const u4* const base = lds + buf * 2 * S;
    if (G == 1 || s < steps) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        u4 fa[M2][NP];
#pragma unroll
        for (int i = 0; i < M2; ++i) {
          const int row = (wi * M2 + i) * 16 + r;
#pragma unroll
          for (int p = 0; p < NP; ++p)
            fa[i][p] = base[(ks * NP + p) * B * 4 + row * 4 + (g ^ ((row >> 1) & 3))];
        }
#pragma unroll
        for (int j = 0; j < M2; ++j) {
          const int row = (wj * M2 + j) * 16 + r;
          u4 fb[NP];
#pragma unroll
          for (int p = 0; p < NP; ++p)
            fb[p] = base[S + (ks * NP + p) * B * 4 + row * 4 + (g ^ ((row >> 1) & 3))];
#pragma unroll
          for (int i = 0; i < M2; ++i) {
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
    }
    if (s + G < steps) store(buf ^ 1);
  }
  v4f sum[M2][M2];
#pragma unroll
  for (int i = 0; i < M2; ++i)
#pragma unroll
    for (int j = 0; j < M2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float v = acc[i][j][q], t = F ? v + small[F ? i : 0][F ? j : 0][q] : v;
        sum[i][j][q] = finite(t) ? t : v;
      }
  if (G > 1) {
    v4f* const part = reinterpret_cast<v4f*>(shared);  // of group k: [block][thread]
    __syncthreads();
    if (grp > 0) {
#pragma unroll
      for (int b = 0; b < M2 * M2; ++b) part[((grp - 1) * M2 * M2 + b) * LNT + tid] = sum[b / M2][b % M2];
    }
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int k = 1; k < G; ++k)
#pragma unroll
      for (int b = 0; b < M2 * M2; ++b) sum[b / M2][b % M2] += part[((k - 1) * M2 * M2 + b) * LNT + tid];
  }
#pragma unroll
  for (int i = 0; i < M2; ++i) {
    const int64_t row = i0 + (wi * M2 + i) * 16 + r;
    if (row >= a.I) continue;
#pragma unroll
    for (int j = 0; j < M2; ++j) {
      const int col = j0 + (wj * M2 + j) * 16 + 4 * g;
      if (col >= a.J) continue;
      deliver<T, XB>(a, slice, row, col, sum[i][j]);
    }
  }
}

template <class T, int G>
__global__ __launch_bounds__(LNT* G, G == 1 ? 2 : 4) void k_product(Product<T> a) {
  __shared__ __align__(16) u4 lds[product_lds<T>(G) / 16];
  product_tile<T, false, false, G>(a, blockIdx.x, lds);
}

// The backward's two products and the bias's gradient: workgroups of dW (the
// longer sums), then of dx, then of the columns' sums.
template <class T, int G>
__global__ __launch_bounds__(LNT* G, G == 1 ? 2 : 4) void k_products(Product<T> w, Product<T> x, Columns<T> c) {
  __shared__ __align__(16) u4 lds[product_lds<T>(G) / 16];
  const uint32_t nw = w.tiles * w.slices, nx = x.tiles * x.slices, b = blockIdx.x;
  if (b < nw) product_tile<T, true, true, G>(w, b, lds);
  else if (b < nw + nx) product_tile<T, false, true, G>(x, b - nw, lds);
  else add_columns(c, (int)(b - nw - nx), reinterpret_cast<float*>(lds));
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
  const auto pieces = [&](int c, bool whole, auto count) {
    constexpr int N = decltype(count)::value;
    uint32_t da[N][2][MB][D], db[N][2][NB][D];
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = (c + u * each) * 64 + 32 * h + 8 * g;
#pragma unroll
        for (int j = 0; j < NB; ++j) load_k8(pb[j], k, a.K, whole, db[u][h][j]);
#pragma unroll
        for (int i = 0; i < MB; ++i) load_k8(pa[i], k, a.K, whole, da[u][h][i]);
      }
#pragma unroll
    for (int u = 0; u < N; ++u)
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
  int c = blockIdx.y * NW + wv;
  for (; (c + (UN - 1) * each) * 64 + 64 <= a.K; c += UN * each)
    pieces(c, true, std::integral_constant<int, UN>{});
  for (; c * 64 < a.K; c += each) pieces(c, c * 64 + 64 <= a.K, std::integral_constant<int, 1>{});
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
    const int row = i0 + 16 * (b / NB) + r, col = j0 + 16 * (b % NB) + 4 * g;
    if (row < a.I && col < a.J) deliver<T, false>(a, blockIdx.y, row, col, s);
  }
}

// The slices' sums joined in their order, of up to two products; eight slices' (or
// four, or two) loads before the first is added, the last again past the last.
template <class T>
__device__ __forceinline__ void join_quad(const Product<T>& a, uint32_t t, vcg::FastDiv line) {
  const int i = (int)line.div(t), j = (int)(t - i * line.d) * 4;
  const int64_t step = (int64_t)a.I * part_line(a.J);
  const float* const p = a.part + (int64_t)t * 4;
  v4f v = v4f{-0.f, -0.f, -0.f, -0.f};  // adds nothing, not even a sign
  const auto some = [&](int s, auto count) {
    constexpr int N = decltype(count)::value;
    v4f w[N];
#pragma unroll
    for (int u = 0; u < N; ++u)
      w[u] = *reinterpret_cast<const v4f*>(p + min(s + u, a.slices - 1) * step);
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (s + u < a.slices) v += w[u];
  };
  if (a.slices == 2) some(0, std::integral_constant<int, 2>{});
  else if (a.slices <= 4) some(0, std::integral_constant<int, 4>{});
  else
    for (int s = 0; s < a.slices; s += 8) some(s, std::integral_constant<int, 8>{});
  finish<T, false>(a, i, j, v);
}

// Workgroups of the columns' sums first, where dz has any left to join.
template <class T>
__global__ __launch_bounds__(LNT) void k_join(Product<T> a, uint32_t na, vcg::FastDiv la,
                                              Product<T> b, uint32_t nb, vcg::FastDiv lb,
                                              Columns<T> c, uint32_t nc) {
  __shared__ float lds[LNT];
  if (blockIdx.x < nc) {
    add_columns(c, (int)blockIdx.x, lds);
    return;
  }
  const uint32_t t = (blockIdx.x - nc) * LNT + threadIdx.x;
  if (t < na) join_quad(a, t, la);
  else if (t - na < nb) join_quad(b, t - na, lb);
}

// Eight values j .. j + 7 of a row of n, as floats; past the end zero.
template <class T>
__device__ __forceinline__ void load8(const T* p, int j, int n, bool whole, float* o) {
  uint32_t d[sizeof(T) == 4 ? 8 : 4];
  load_k8(p, j, n, whole, d);
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

// Eight fp32 values as 16 bytes of each of two bf16 parts, the first cut (store_parts
// has three): 2^-16 of a value is lost.  An infinity or NaN stands in the first alone.
__device__ __forceinline__ void store_two(const float* v, uint16_t* to, int64_t plane) {
  u4 h, l;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t b0 = __builtin_bit_cast(uint32_t, v[2 * q]), b1 = __builtin_bit_cast(uint32_t, v[2 * q + 1]);
    h[q] = __builtin_amdgcn_perm(b1, b0, 0x07060302);
    l[q] = bf_pack(finite(v[2 * q]) ? v[2 * q] - bf_hi(b0) : 0.f,
                   finite(v[2 * q + 1]) ? v[2 * q + 1] - bf_hi(b1) : 0.f);
  }
  *reinterpret_cast<u4*>(to) = h;
  *reinterpret_cast<u4*>(to + plane) = l;
}

// Up to two matrices as parts for the tiled products, their lines padded with
// zeros to a multiple of eight.
template <class T>
struct Pack {
  const T* p;
  int64_t ld, rows;
  int n, np;      // values of a line, and with its padding
  uint16_t* to;
  int64_t line;   // from one line written to the next
  int64_t lines;  // with those of zeros behind the rows
  int64_t again;  // bf16: from a line to its second copy, zeros for what is not finite, or 0
};
template <class T>
Pack<T> pack_of(const void* p, int64_t ld, int64_t rows, int n, int np, void* to) {
  return {(const T*)p, ld, rows, n, np, (uint16_t*)to, np, rows, 0};
}

template <class T>
__device__ __forceinline__ void pack_block(const Pack<T>& m, int64_t block, int64_t blocks) {
  const int c = m.np / 8;
#pragma unroll 1
  for (int64_t t = block * LNT + threadIdx.x; t < m.lines * c; t += blocks * LNT) {
    const int64_t row = t / c;
    const int j = (int)(t - row * c) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row < m.rows) load8(m.p + row * m.ld, j, m.n, j + 8 <= m.n, v);
    uint16_t* const to = m.to + row * m.line + j;
    store_parts<T>(v, to, m.rows * m.np);
    if constexpr (sizeof(T) == 2) {
      if (!m.again) continue;
      // dz's second parts meet this copy: they add nothing to an infinity or NaN
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = finite(v[q]) ? v[q] : 0.f;
      store_parts<T>(v, to + m.again, 0);
    }
  }
}

// dz = dy act'(z), and the columns' sums of each block of rows, from dz in fp32.  dz as
// values, or as parts for the tiled products (lines of np values, zeros past N).
//
// The matrix cores multiply bf16 with nothing wider, and in bf16 the dz of GELU and SiLU
// has more bits than that (ReLU's and none's are dy's own).  So it is two parts, and
// the products are those of a sum twice as long: a row of dz is its h and then its l,
//   dx[m] = [h_m l_m] [W; W],   dW = sum over lines h_0, l_0, h_1, .. times x_0, x_0, x_1, ..
// with W and x copied so by the pass before.  Twice the products' work for dx and dW 1.7e-3 of
// their norm off, which is the rounding of the result, instead of 2.3e-3 with dz rounded
// (8192 x 4096 x 4096 GELU 996 us and 495, 1021 x 333 x 777 SiLU 24.5 and 19.6); a caller
// who prefers the time asks for that (VC_DZ_ROUNDED).
template <class T>
struct Slope {
  const T *dy, *z;
  int64_t ldy, ldz;
  T* dz;           // lines of N, or null
  uint16_t* parts; // or null
  int64_t line, plane;  // of the parts: from a row to the next, from a part to the next
  float* sums;     // (blocks of rows, N), or null
  int64_t M;
  int N, act, rows, lanes;
  bool two;        // bf16 in two parts
};

// Lanes across a row, eight columns each; the workgroup's others take more rows.
int slope_lanes(int N) { return N <= 64 ? 8 : N <= 128 ? 16 : 32; }

template <class T>
__device__ __forceinline__ void slope_block(const Slope<T>& a, int bx, int by) {
  __shared__ float part[LNT / 8 * 72];
  const int cols = 8 * a.lanes, per = LNT / a.lanes, line = cols + 8;  // per: rows at a time
  const int c = threadIdx.x & (a.lanes - 1), y = threadIdx.x / (unsigned)a.lanes;
  const int j = bx * cols + 8 * c;
  const bool whole = (bx + 1) * cols <= a.N;
  const int64_t m0 = (int64_t)by * a.rows;
  const int64_t m1 = m0 + a.rows < a.M ? m0 + a.rows : a.M;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  // R rows of this thread's: all their loads before the first is used
  const auto take = [&](int64_t m, auto count) {
    constexpr int R = decltype(count)::value;
    float d[R][8], z[R][8];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const int64_t r = m + per * q < m1 ? m + per * q : m;
      load8(a.dy + r * a.ldy, j, a.N, whole, d[q]);
      if (a.act != kNone) load8(a.z + r * a.ldz, j, a.N, whole, z[q]);
    }
    const auto each = [&](auto act) {  // one branch chooses the slope of all
#pragma unroll
      for (int q = 0; q < R; ++q) {
        const int64_t r = m + per * q;
        if (r >= m1) break;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (act != kNone) d[q][i] = dz_of<T>(d[q][i], z[q][i], act);
          sum[i] += d[q][i];
        }
        if (a.parts) {
          uint16_t* const to = a.parts + r * a.line + j;
          if (sizeof(T) == 2 && a.two) store_two(d[q], to, a.plane);
          else store_parts<T>(d[q], to, a.plane);
        }
        if (a.dz) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (j + i < a.N) put(a.dz + r * a.N + j + i, d[q][i]);
        }
        __builtin_amdgcn_sched_barrier(0);  // one row's temporaries at a time
      }
    };
    if (a.act == kNone) each(std::integral_constant<int, kNone>{});
    else if (a.act == kRelu) each(std::integral_constant<int, kRelu>{});
    else if (a.act == kGelu) each(std::integral_constant<int, kGelu>{});
    else each(std::integral_constant<int, kSilu>{});
  };
  if (j < a.N) {
    if (a.rows <= per) {
      if (m0 + y < m1) take(m0 + y, std::integral_constant<int, 1>{});
    } else {
      for (int64_t m = m0 + y; m < m1; m += 4 * per) take(m, std::integral_constant<int, 4>{});
    }
  }
  if (!a.sums) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) part[y * line + 8 * c + i] = sum[i];
  __syncthreads();
  const int k = bx * cols + threadIdx.x;
  if ((int)threadIdx.x >= cols || k >= a.N) return;
  float s = 0.f;
#pragma unroll 8
  for (int i = 0; i < per; ++i) s += part[i * line + threadIdx.x];
  a.sums[(int64_t)by * a.N + k] = s;
}

// What has to be there before the products: workgroups of dz, then of up to two
// matrices' parts.
template <class T>
__global__ __launch_bounds__(LNT) void k_before(Slope<T> s, int ns, int cols, Pack<T> a, int64_t na,
                                                Pack<T> b) {
  const int64_t w = blockIdx.x;
  if (w < ns) slope_block(s, (int)w % cols, (int)w / cols);
  else if (w < ns + na) pack_block(a, w - ns, na);
  else pack_block(b, w - ns - na, gridDim.x - ns - na);
}

int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }
int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }
constexpr int64_t kCus = 256;

// How a product is cut: the kernel, its shape, and the slices of k, by the time
// that they are expected to take (us).
enum Kernel { kProduct, kDirect, kTile, kRaw };
struct Cut {
  Kernel kernel;
  int shape, slices, steps;
  int64_t tiles, nj;
  float us;
};

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A launch has fewer than 2^32 threads.  A product's workgroups, of so many threads at most, have
// fewer than 2^30 of them: two of these go together, with the columns' sums (2^18
// workgroups at most, that take more columns each beyond).
bool fits(int64_t tiles, int64_t slices, int threads) {
  return tiles < (1 << 30) && tiles * slices * threads < (1 << 30);
}
constexpr int64_t kMostGroups = 1 << 18;
constexpr int64_t kMostPacks = 1 << 20;  // workgroups of a matrix's parts
constexpr int64_t kMostSlopes = (1 << 24) - 2 * kMostPacks - 1;  // of dz, beside them

// The slices' sums written, read again and joined by a launch.
float join_us(int64_t slices, int64_t I, int64_t J) {
  return slices > 1 ? 4.f + 0.1f * slices + 8.f * slices * I * J / 4e6f : 0.f;
}

// One product's grid of bi x bj tiles, its k in about `want` slices.
struct Grid {
  int64_t tiles, nj, slices, steps;
};
Grid grid_of(int64_t I, int64_t J, int64_t K, int bi, int bj, int bk, int64_t want) {
  Grid g;
  const int64_t all = div_up(K, bk) > 0 ? div_up(K, bk) : 1;
  g.nj = div_up(J, bj);
  g.tiles = div_up(I, bi) * g.nj;
  g.steps = div_up(all, want);
  g.slices = div_up(all, g.steps);
  return g;
}

// What a kernel's tiles cost: `alone` us a step for as many workgroups as share a
// CU, `shared` us for each of them, `end` us for a tile's output.
struct Cost {
  int bi, bj, bk, threads, share;
  float alone, shared, end;
};

// The expected time of up to two products in one launch, and of joining them.
struct Job {
  int64_t I, J, K;
};
float expect(int type, const Cost& c, const Job* job, const Grid* g, int n) {
  int64_t wgs = 0, longest = 0;
  double steps = 0.0, bytes = 0.0;
  float join = 0.f;
  for (int i = 0; i < n; ++i) {
    wgs += g[i].tiles * g[i].slices;
    steps += (double)g[i].tiles * g[i].slices * g[i].steps;
    if (g[i].steps > longest) longest = g[i].steps;
    bytes += (type == VC_FP32 ? 6.0 : 2.0) * (job[i].I + job[i].J) * job[i].K;
    const float j = join_us(g[i].slices, job[i].I, job[i].J);
    join = join > 0.f && j > 0.f ? join + j - 4.f : join + j;
  }
  const int64_t rounds = div_up(wgs, kCus * c.share), load = div_up(wgs, kCus);
  // of a CU: the busiest where several share one, else the mean
  const float even = (float)(steps / kCus) * (c.share > 1 ? (float)load * kCus / wgs : 1.f);
  const float a = (c.alone * longest + c.end) * rounds, s = c.shared * even + c.end * load;
  const float m = (float)(bytes / 4.5e6);
  const float work = a > s ? a : s;
  return 4.f + (work > m ? work : m) + join;
}

// The slices that are expected to be fastest, of up to two products.
float best_slices(int type, const Cost& c, const Job* job, int n, Grid* best) {
  constexpr int kWant[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 32}, kN = 15;
  float least = 1e30f;
  for (int p = 0; p < kN; ++p)
    for (int q = 0; q < (n > 1 ? kN : 1); ++q) {
      Grid g[2];
      bool sane = true;
      for (int i = 0; i < n; ++i) {
        const int64_t want = kWant[i ? q : p];
        sane = sane && (want == 1 || (4 * want * c.bk <= job[i].K && job[i].I * job[i].J < (1ll << 31)));
        g[i] = grid_of(job[i].I, job[i].J, job[i].K, c.bi, c.bj, c.bk, want);
        sane = sane && fits(g[i].tiles, g[i].slices, c.threads);
      }
      const float us = sane ? expect(type, c, job, g, n) : 1e30f;
      if (us < least) {
        least = us;
        for (int i = 0; i < n; ++i) best[i] = g[i];
      }
    }
  return least;
}

// The tiles by registers, shape 0 by one group of waves, 1 by several: steps of 32
// (bf16: 64) times the groups (measured on 64 x 64, 512 x 1024 and 2048 x 2048
// outputs).  Backward with the passes before and after, by the one, by the other and by
// the best tiles: fp32 265 x 352 x 461 16.4, 16.9 and 18.6 us, 512 x 784 x 1024 36.9, 38.7
// and 27.2, 5171 x 896 x 64 33, 42 and 31; bf16 1021 x 333 x 777 22.5, 18.1 and 19.1, 2050 x
// 512 x 1030 47, 50 and 36, 17 x 256 x 64 7.2, 9.2 and 7.8.
constexpr int kGroups32 = 3, kGroups16 = 4;
Cost product_cost(int type, int shape) {
  if (type == VC_FP32)
    return shape ? Cost{64, 64, 96, LNT * kGroups32, 1, 2.0f, 1.75f, 1.f}
                 : Cost{64, 64, 32, LNT, 3, 1.12f, 0.6f, 0.5f};
  return shape ? Cost{64, 64, 256, LNT * kGroups16, 1, 2.9f, 2.2f, 1.f}
               : Cost{64, 64, 64, LNT, 4, 1.3f, 0.4f, 0.5f};
}

// The tiles that go straight into LDS: a step of as many as share a CU while others
// stand idle, a step of each with all of them busy (random operands: the card's power
// then sets the pace), and a tile's output (8192 x 8192, fp32 4096 x 4096, of one step:
// 41, 37 and 41 us, fp32 22, 24 and 19).  8192 x 4096 x 4096 bf16 212, 255 and 383 us,
// 1024 x 1024 x 1024 27, 13 and 7.5; fp32 8192 x 1024 x 4096 331, 348 and 485, 2048
// x 2048 x 2048 134, 87 and 151, 1024 x 1024 x 1024 64, 36 and 24.
// far: the operands come from beyond the last-level cache and are used by few tiles
// (103 x 10768 x 12758 bf16, 277 MB: 64 x 64 in one slice 124 us, 128 x 128 in five 69;
// fp32 64 x 8192 x 8192 in four slices 169, 104 and 103).
Cost tile_cost(int type, int shape, bool far) {
  constexpr float alone[2][2][4] = {{{2.0f, 1.06f, 0.8f}, {1.15f, 0.6f, 0.4f, 0.25f}},
                                    {{2.0f, 1.06f, 0.88f}, {1.3f, 0.83f, 0.7f, 0.65f}}};
  constexpr float shared[2][2][4] = {{{2.3f, 1.19f, 0.5f}, {1.6f, 0.47f, 0.17f, 0.3f}},
                                     {{2.6f, 1.65f, 0.8f}, {2.0f, 0.95f, 0.38f, 0.38f}}};
  constexpr int share[2][4] = {{1, 1, 2}, {1, 2, 4, 2}};
  constexpr float end[2][4] = {{6.8f, 3.8f, 0.5f}, {7.5f, 1.5f, 0.4f, 0.4f}};
  const TileShape t = tile_shape(type, shape);
  const int b = type == VC_FP32 ? 0 : 1;
  return {t.bi, t.bj, t.bk, 512, share[b][shape], alone[far][b][shape], shared[far][b][shape],
          end[b][shape]};
}

// Up to two products by the kernel and shape expected to be fastest, of so many shapes
// of tiles (0: tiles cannot be made).  extra: what
// the tiles' parts cost before.
float choose(int type, const Job* job, int n, bool products, int tiles, float extra, Cut* out) {
  float least = 1e30f;
  const auto take = [&](Kernel k, int shape, const Cost& c, float more) {
    Grid g[2];
    const float us = best_slices(type, c, job, n, g) + more;
    if (us >= least) return;
    least = us;
    for (int i = 0; i < n; ++i) {
      const int per = k == kProduct && shape ? (type == VC_FP32 ? kGroups32 : kGroups16) : 1;
      out[i] = {k, shape, (int)g[i].slices, (int)g[i].steps * per, g[i].tiles, g[i].nj, us};
    }
  };
  bool far = true;
  int64_t bytes = 0;
  for (int i = 0; i < n; ++i) {
    bytes += (type == VC_FP32 ? 6 : 2) * (job[i].I + job[i].J) * job[i].K;
    far = far && job[i].I * job[i].J < 256 * (job[i].I + job[i].J);
  }
  far = far && bytes > (100 << 20);
  for (int shape = 0; shape < (products ? 2 : 0); ++shape) take(kProduct, shape, product_cost(type, shape), 0.f);
  for (int shape = 0; shape < tiles; ++shape) take(kTile, shape, tile_cost(type, shape, far), extra);
  return least;
}

// The direct kernel: 16 rows by 16 columns, 32 by 16, 64 by 16, 64 by 32.  A
// workgroup's operands come at about 40 GB/s a CU (sixteen rows a load, 16 bytes a
// lane; 5 x 15872 x 788 fp32 18.7 us, the tiles of 64 x 32 30), all of them together
// at no more than the memory's rate.
constexpr int kDirectRows[4] = {16, 32, 64, 64}, kDirectCols[4] = {16, 16, 16, 32};

Cut cut_direct(int type, int64_t I, int64_t J, int64_t K) {
  Cut c = {};
  c.us = 1e30f;
  const float e = type == VC_FP32 ? 4.f : 2.f;
  // fp32 has no 64 by 32: its parts do not fit into the registers
  for (int shape = 0; shape < (type == VC_FP32 ? 3 : 4); ++shape) {
    const int bi = kDirectRows[shape], bj = kDirectCols[shape];
    const int64_t nj = div_up(J, bj), tiles = div_up(I, bi) * nj;
    if (!fits(tiles, 1, 64 * kDirectWaves)) continue;
    int64_t s = 1;
    while (tiles * s < kCus && 1024 * s < K && s < 16) s *= 2;
    const float own = e * (bi + bj) * (float)K / s;  // rows past the last are read as the last
    const float l2 = div_up(tiles * s, kCus) * own / 40e3f;
    const float hbm = e * (I + J) * (float)K / 4.5e6f;
    const float us = 4.f + (l2 > hbm ? l2 : hbm) + join_us(s, I, J);
    if (us < c.us) c = {kDirect, shape, (int)s, 0, tiles, nj, us};
  }
  return c;
}

// Whether tiles can be made of matrices with lines of this length at all.
bool tile_lines(int64_t n) { return n > 0 && n < (1 << 21); }

// The pass that makes `n` values into parts.
float pack_us(int type, int64_t n) { return 4.f + n * (type == VC_FP32 ? 10.f : 4.f) / 4e6f; }

int64_t part_bytes(const Cut& c, int64_t I, int64_t J) {
  return c.slices > 1 ? up256(4 * c.slices * I * part_line((int)J)) : 0;
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
void set_cut(Product<T>& a, const Cut& c, void* part) {
  a.slices = c.slices;
  a.steps = c.steps;
  a.part = (float*)part;
  a.tiles = c.tiles;
  a.f_nj = vcg::FastDiv::make((uint32_t)c.nj);
}
template <class T>
void run_join(const Product<T>& a, const Product<T>& b, const Columns<T>& c, hipStream_t st) {
  const auto quads = [](const Product<T>& p) {
    return p.slices > 1 ? (uint32_t)p.I * (uint32_t)(part_line(p.J) / 4) : 0u;
  };
  const auto line = [](const Product<T>& p) {
    return vcg::FastDiv::make((uint32_t)(p.slices > 1 ? part_line(p.J) / 4 : 1));
  };
  const uint32_t na = quads(a), nb = quads(b);
  const uint32_t nc = c.db ? (uint32_t)c.groups : 0u;
  const unsigned grid = nc + (unsigned)div_up((int64_t)na + nb, LNT);
  if (grid > 0) k_join<T><<<grid, LNT, 0, st>>>(a, na, line(a), b, nb, line(b), c, nc);
}

template <class T>
void run_before(Slope<T> s, Pack<T> a, Pack<T> b, hipStream_t st) {
  const auto packs = [](const Pack<T>& m) {
    const int64_t all = m.to ? div_up(m.lines * (m.np / 8), LNT) : 0;
    return all < kMostPacks ? all : kMostPacks;
  };
  const int64_t na = packs(a), nb = packs(b);
  const int cols = s.dy ? (int)div_up(s.N, 8 * s.lanes) : 0, ns = s.dy ? cols * (int)div_up(s.M, s.rows) : 0;
  if (ns + na + nb > 0) k_before<T><<<(unsigned)(ns + na + nb), LNT, 0, st>>>(s, ns, cols, a, na, b);
}

bool sizes_ok(int64_t M, int K, int N) {
  return M >= 0 && M <= 0x7fffff00 && K >= 0 && K <= (1 << 30) && N >= 0 && N <= (1 << 30);
}

struct ForwardPlan {
  Cut c;
  int64_t x, W, part, bytes;  // offsets in the workspace, and its size (-1: no cut fits a launch)
};

// A thread's latest plans, by their sizes: the search takes up to 50 us.
template <class Plan>
struct Plans {
  struct Entry {
    int64_t key[6];
    bool set;
    Plan plan;
  } all[64];
  template <class Make>
  const Plan& get(const int64_t (&key)[6], const Make& make) {
    uint64_t h = 0;
    for (const int64_t k : key) h = (h ^ (uint64_t)k) * 0x9e3779b97f4a7c15ull;
    Entry& e = all[h >> 58];
    bool same = e.set;
    for (int i = 0; i < 6; ++i) same = same && e.key[i] == key[i];
    if (!same) {
      e.plan = make();
      for (int i = 0; i < 6; ++i) e.key[i] = key[i];
      e.set = true;
    }
    return e.plan;
  }
};

// raw: fp32 rows that the loads into LDS can take as they are.
ForwardPlan make_forward(int type, int64_t M, int K, int N, bool raw) {
  ForwardPlan p;
  const Job job = {M, N, K};
  const float pack = type == VC_FP32 || K % 8 ? pack_us(type, (M + N) * K) : 0.f;
  p.c = cut_direct(type, M, N, K);
  Cut c = {};
  // bf16 goes by the tiles or directly: between them the other products gain nothing
  choose(type, &job, 1, type == VC_FP32, !tile_lines(K) ? 0 : type == VC_FP32 ? 3 : 4, pack, &c);
  if (c.us > 0.f && c.us < p.c.us) p.c = c;
  if (raw) {
    // two steps of 32 alone on a CU, and of each of two that share one (512 x 784 x
    // 1024 12.2 us, 64 x 8192 x 1024 in eight slices 14.9, 1024 x 784 x 1024 23)
    const Cost c = {64, 32, 64, 512, 2, 0.68f, 0.68f, 0.5f};
    Grid g;
    const float us = best_slices(type, c, &job, 1, &g);
    if (us < p.c.us) p.c = {kRaw, 0, (int)g.slices, (int)g.steps * 2, g.tiles, g.nj, us};
  }
  if (p.c.us >= 1e30f) {
    p.bytes = -1;
    return p;
  }
  const bool tiles = p.c.kernel == kTile;
  p.x = 0;
  p.W = tiles ? parts_bytes(type, M, K) : 0;
  p.part = p.W + (tiles ? parts_bytes(type, N, K) : 0);
  p.bytes = p.part + part_bytes(p.c, M, N);
  return p;
}
ForwardPlan plan_forward(int type, int64_t M, int K, int N, bool raw) {
  static thread_local Plans<ForwardPlan> plans;
  return plans.get({type, M, K, N, raw, 0}, [&] { return make_forward(type, M, K, N, raw); });
}

template <class T>
int forward(const void* x, int64_t M, int K, int64_t ldx, const void* W, int N, const void* bias,
            int act, const void* res, int64_t ldr, void* y, void* z, void* work,
            int64_t work_bytes, hipStream_t st) {
  constexpr int type = sizeof(T) == 4 ? VC_FP32 : VC_BF16;
  const bool raw = type == VC_FP32 && K % 4 == 0 && K > 0 && ldx % 4 == 0 && aligned16(x) &&
                   aligned16(W) && K < (1 << 21) && ldx < (1 << 21);
  const ForwardPlan p = plan_forward(type, M, K, N, raw);
  if (p.bytes < 0) return VC_ERR_UNSUPPORTED;
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
    if (!as_it_is((const T*)x, ldx, K)) px = pack_of<T>(x, ldx, M, K, kp, base + p.x);
    if (!as_it_is((const T*)W, K, K)) pw = pack_of<T>(W, K, N, K, kp, base + p.W);
    run_before<T>({}, px, pw, st);
    a.pa = px.to ? px.to : (const uint16_t*)x;
    a.lda = px.to ? kp : ldx;
    a.planeA = M * kp;
    a.pb = pw.to ? pw.to : (const uint16_t*)W;
    a.ldb = kp;
    a.planeB = (int64_t)N * kp;
    a.K = kp;
  }
  set_cut(a, p.c, base + p.part);
  constexpr bool F = sizeof(T) == 4;
  const dim3 grid((unsigned)p.c.tiles, (unsigned)p.c.slices);
  const unsigned flat = (unsigned)(p.c.tiles * p.c.slices);
  constexpr int threads = 64 * kDirectWaves;
  if (p.c.kernel == kTile) {
    run_tile<T>(a, p.c.shape, st);
  } else if (p.c.kernel == kRaw) {
    if constexpr (F) run_raw(a, st);
  } else if (p.c.kernel == kProduct) {
    if constexpr (F) {
      if (p.c.shape == 0) k_product<T, 1><<<flat, LNT, 0, st>>>(a);
      else k_product<T, kGroups32><<<flat, LNT * kGroups32, 0, st>>>(a);
    }
  }
  else if (p.c.shape == 0) k_direct<T, 1, 1, F ? 2 : 8><<<grid, threads, 0, st>>>(a);
  else if (p.c.shape == 1) k_direct<T, 1, 2, F ? 2 : 4><<<grid, threads, 0, st>>>(a);
  else if (p.c.shape == 2) k_direct<T, 1, 4, F ? 1 : 2><<<grid, threads, 0, st>>>(a);
  else if constexpr (!F) k_direct<T, 2, 4, 2><<<grid, threads, 0, st>>>(a);
  run_join<T>(a, {}, {}, st);
  VC_LAUNCH_CHECK();
  return VC_OK;
}

// Rows of a block of dz: as many as its threads take at a time while 256 blocks hold M
// (265 x 461 with silu: four a thread 8.6 us, one 3.8), beyond that what 256 need (4096
// x 1024 by 512 blocks 18.5 us, by 256 15.9).
int slope_rows(int64_t M, int N) {
  const int64_t r = (M + 255) / 256, per = LNT / slope_lanes(N);
  return (int)(r <= per ? per : r < 4 * per ? 4 * per : r);
}

// Whether the products take dz in two parts (slope_block), by act as the caller gave it.
constexpr int kRounded = VC_DZ_ROUNDED;
bool two_parts(int type, int act, int need) {
  return type == VC_BF16 && (act == kGelu || act == kSilu) && (need & 3);
}

struct BackwardPlan {
  bool tiles, two;
  Cut x, w;
  int rows, blocks;
  int64_t dz, W, in, sums, px, pw, bytes;  // offsets in the workspace, and its size (-1: as above)
};

BackwardPlan make_backward(int type, int64_t M, int K, int N, int act, int need) {
  BackwardPlan p = {};
  const int64_t e = type == VC_FP32 ? 4 : 2;
  p.two = two_parts(type, act, need);
  act &= ~kRounded;
  const int64_t np = up8(N), times = p.two ? 2 : 1;
  Job job[2];
  Cut c[2] = {};
  // for both products, whichever are asked for: the same bits either way.  M and N are
  // rows of a product: below 2^29 where a cut fits, so sums twice as long stay within 32 bits
  job[0] = {N, K, times * M};
  job[1] = {M, K, p.two ? 2 * np : N};
  if (need & 3) {
    // the parts of W and x, and of dz beyond its values, in dz's own pass; with dz in two
    // parts both are copied for any kernel
    const float pack = type == VC_FP32   ? pack_us(type, (M + N) * K + M * N / 5) - (act != kNone ? 4.f : 0.f)
                       : K % 8 && !p.two ? pack_us(type, (M + N) * K) - (act != kNone ? 4.f : 0.f)
                                         : 0.f;
    const int can = tile_lines(K) && tile_lines(times * np) ? 3 : 0;
    const float one = choose(type, job, 2, true, can, pack, c);
    if (one >= 1e30f) {
      p.bytes = -1;
      return p;
    }
    p.tiles = c[0].kernel == kTile;
    // or a launch each, in a shape of its own
    Cut w = {}, x = {};
    const float two = choose(type, job, 1, false, can, pack, &w) + choose(type, job + 1, 1, false, can, 0.f, &x);
    if (p.tiles && w.kernel == kTile && x.kernel == kTile && two < one) c[0] = w, c[1] = x;
  }
  if (need & 2) p.w = c[0];
  if (need & 1) p.x = c[1];
  p.rows = slope_rows(M, N);
  p.blocks = (int)div_up(M, p.rows);
  if (div_up(N, 8 * slope_lanes(N)) * p.blocks > kMostSlopes) {
    p.bytes = -1;
    return p;
  }
  int64_t at = 0;
  const bool parts = p.tiles || p.two;
  if (need & 3) at += parts ? parts_bytes(type, times * M, N) : act != kNone ? up256(e * M * N) : 0;
  p.W = at;
  if ((need & 1) && parts) at += parts_bytes(type, p.two ? 2 * np : N, K);
  p.in = at;
  if ((need & 2) && parts) at += parts_bytes(type, times * M, K);
  p.sums = at;
  if (need & 4) at += up256(4ll * p.blocks * N);
  p.px = at;
  if (need & 1) at += part_bytes(p.x, M, K);
  p.pw = at;
  if (need & 2) at += part_bytes(p.w, N, K);
  p.bytes = at;
  return p;
}
BackwardPlan plan_backward(int type, int64_t M, int K, int N, int act, int need) {
  static thread_local Plans<BackwardPlan> plans;
  return plans.get({type, M, K, N, act, need},
                   [&] { return make_backward(type, M, K, N, act, need); });
}

template <class T>
int backward(const void* dy, int64_t ldy, const void* x, int64_t ldx, const void* W, const void* z,
             int64_t ldz, int act, int64_t M, int K, int N, void* dx, void* dW, void* db,
             void* work, int64_t work_bytes, hipStream_t st) {
  constexpr int type = sizeof(T) == 4 ? VC_FP32 : VC_BF16;
  // nothing to write, and what that leaves of the others
  if (K == 0 || N == 0) dW = nullptr;
  if (K == 0 || M == 0) dx = nullptr;
  if (N == 0 || M == 0) db = nullptr;
  const int need = (dx ? 1 : 0) | (dW ? 2 : 0) | (db ? 4 : 0);
  if (!need) return VC_OK;
  const BackwardPlan p = plan_backward(type, M, K, N, act, need);
  act &= ~kRounded;
  if (p.bytes < 0) return VC_ERR_UNSUPPORTED;
  if (p.bytes > work_bytes || (p.bytes && !work)) return VC_ERR_OOM;
  char* const base = (char*)work;
  const int np = (int)up8(N), kp = (int)up8(K);
  // dy itself is dz where nothing is between them and the products can read it
  const bool made = (need & 3) && (act != kNone || (p.tiles && !as_it_is((const T*)dy, ldy, N)));
  const bool parts = p.tiles || p.two;
  Slope<T> s = {};
  if (N > 0 && M > 0 && (made || db)) {
    s.dy = (const T*)dy;
    s.z = (const T*)z;
    s.ldy = ldy;
    s.ldz = ldz;
    if (made && parts) s.parts = (uint16_t*)(base + p.dz);
    else if (made) s.dz = (T*)(base + p.dz);
    s.sums = db ? (float*)(base + p.sums) : nullptr;
    s.act = act;
  }
  s.M = M;
  s.N = N;
  s.two = p.two;
  s.line = p.two ? 2 * np : np;
  s.plane = p.two ? np : M * np;
  s.rows = p.rows;
  s.lanes = slope_lanes(N);
  Pack<T> mw = {}, mx = {};
  if (dx && (p.two || (p.tiles && !as_it_is((const T*)W, K, K))))
    mw = pack_of<T>(W, K, N, K, kp, base + p.W);
  if (dW && (p.two || (p.tiles && !as_it_is((const T*)x, ldx, K))))
    mx = pack_of<T>(x, ldx, M, K, kp, base + p.in);
  if (p.two) {
    mw.lines = np;
    mw.again = (int64_t)np * kp;
    mx.line = 2 * kp;
    mx.again = kp;
  }
  run_before<T>(s, mw, mx, st);

  Product<T> px = {}, pw = {};
  const T* const dz = made ? (const T*)(base + p.dz) : (const T*)dy;
  const int64_t ldd = !made ? ldy : parts ? np : N;
  if (dx) {
    px.I = (int)M;
    px.J = K;
    px.K = p.two ? 2 * np : N;
    px.out = (T*)dx;
    px.A = {dz, p.two ? 2 * np : ldd, (int)M};
    px.B = {(const T*)(p.two ? (const void*)mw.to : W), p.two ? kp : K, K};
    px.pb = mw.to ? mw.to : (const uint16_t*)W;
    px.ldb = kp;
    px.planeB = (int64_t)N * kp;
    set_cut(px, p.x, base + p.px);
  }
  if (dW) {
    pw.I = N;
    pw.J = K;
    pw.K = p.two ? 2 * (int)M : (int)M;
    pw.out = (T*)dW;
    pw.A = {dz, ldd, N};
    pw.B = {(const T*)(p.two ? (const void*)mx.to : x), p.two ? kp : ldx, K};
    pw.pb = mx.to ? mx.to : (const uint16_t*)x;
    pw.ldb = mx.to ? kp : ldx;
    pw.planeB = M * kp;
    set_cut(pw, p.w, base + p.pw);
  }
  px.pa = pw.pa = (const uint16_t*)dz;
  px.lda = px.A.ld;
  pw.lda = pw.A.ld;
  px.planeA = pw.planeA = M * np;
  // the columns' sums: in the join's launch where there is one (beside the products they
  // would wait for a CU's whole LDS), else in the products'
  const int64_t each = div_up(N, 32);
  const Columns<T> sums = {(const float*)(base + p.sums), p.blocks, N, db ? (T*)db : nullptr,
                           (int)(each < kMostGroups ? each : kMostGroups)};
  const bool late = p.w.slices > 1 || p.x.slices > 1;
  const Columns<T> c = late ? Columns<T>{} : sums;
  const unsigned grid = (unsigned)(p.w.tiles * p.w.slices + p.x.tiles * p.x.slices + (c.db ? c.groups : 0));
  constexpr int G = sizeof(T) == 4 ? kGroups32 : kGroups16;
  const Cut& any = dW ? p.w : p.x;
  // two of different shapes, or that each fill the chip, go one after the other: their
  // tiles share what they read while they run in step (8192 x 4096 x 4096 bf16, dz
  // rounded: 495 us, together 567)
  const int64_t nw = p.w.tiles * p.w.slices, nx = p.x.tiles * p.x.slices;
  if (p.tiles && dW && dx && (p.w.shape != p.x.shape || (nw >= kCus && nx >= kCus))) {
    Product<T> none = {};
    run_tiles<T>(pw, none, c, p.w.shape, (unsigned)nw, st);
    run_tiles<T>(none, px, c, p.x.shape, grid - (unsigned)nw, st);
  } else if (grid == 0) {
  } else if (p.tiles) run_tiles<T>(pw, px, c, any.shape, grid, st);
  else if (any.shape == 0 || !(need & 3)) k_products<T, 1><<<grid, LNT, 0, st>>>(pw, px, c);
  else k_products<T, G><<<grid, LNT * G, 0, st>>>(pw, px, c);
  run_join<T>(pw, px, late ? sums : Columns<T>{}, st);
  VC_LAUNCH_CHECK();
  return VC_OK;
}

bool known(int type, int act) {
  return (type == VC_FP32 || type == VC_BF16) && act >= kNone && act <= kSilu;
}
bool backward_ok(int type, int64_t M, int K, int N, int act) {
  return known(type, act & ~kRounded) && sizes_ok(M, K, N);
}

}  // namespace

extern "C" int64_t vc_linear_workspace(int type, int64_t M, int K, int N) {
  if (!known(type, kNone) || !sizes_ok(M, K, N)) return -1;
  if (M == 0 || N == 0) return 0;
  const int64_t a = plan_forward(type, M, K, N, false).bytes;
  const int64_t b = plan_forward(type, M, K, N, type == VC_FP32).bytes;
  return a < 0 || b < 0 ? -1 : a > b ? a : b;
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
  if (!backward_ok(type, M, K, N, act)) return -1;
  return plan_backward(type, M, K, N, act, need).bytes;
}

extern "C" int vc_linear_backward(int type, const void* dy, int64_t ldy, const void* x,
                                  int64_t ldx, const void* W, const void* z, int64_t ldz, int act,
                                  int64_t M, int K, int N, void* dx, void* dW, void* db,
                                  void* work, int64_t work_bytes, vc_stream_t stream) {
  if (!backward_ok(type, M, K, N, act)) return VC_ERR_ARG;
  const bool some = M > 0 && N > 0, slopes = (act & ~kRounded) != kNone;
  if (some && (!dy || ldy < N || (slopes && (!z || ldz < N)))) return VC_ERR_ARG;
  if (some && K > 0 && ((dx && !W) || (dW && (!x || ldx < K)))) return VC_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  return type == VC_FP32 ? backward<float>(dy, ldy, x, ldx, W, z, ldz, act, M, K, N, dx, dW, db,
                                           work, work_bytes, st)
                         : backward<uint16_t>(dy, ldy, x, ldx, W, z, ldz, act, M, K, N, dx, dW,
                                              db, work, work_bytes, st);
}
