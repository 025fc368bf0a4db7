// The fc layer's large products: tiles of 64 x 64 to 256 x 256 (fp32 256 x 128), both
// operands as bf16 (an fp32 value as three parts, vc_linear.hip) brought into LDS by
// loads that pass no register.
//
// A step of BK goes into one of two to four LDS buffers while another is
// multiplied.  A load instruction writes 1 KB of LDS in lane order, so the order
// that spreads a fragment's reads over the banks is made by which address each
// lane reads from:
//   k contiguous: [row][BK], 16-byte chunk c of row r at c ^ (r mod 8) (BK 64) or
//     c ^ (r / 2 mod 4) (BK 32); a lane's fragment is one 16-byte read;
//   read across: [k][row], 32-byte chunk c of line k at c ^ f(k), f = k mod 4 + 4
//     (k / 8 mod 2); two 8-byte transposing reads give a lane its eight k.
//
// Shapes of eight waves take turns: while four multiply, the other four, one on
// each SIMD, read their next fragments; a barrier ends each turn.  256 x 256 by
// waves of 128 x 64: a turn of 32 products deep is 512 cycles of matrix
// instructions on each SIMD beside 48 KB of fragment reads and 16 KB of loads into
// LDS, at 128 bytes a cycle 512 as well.  8192 x 4096 x 16384 bf16 with gelu: 900 us,
// 1222 TFLOP/s, the matrix units busy in 58% of the cycles at the 2.0 GHz that the
// card's power leaves of 2.4; constant operands, which switch less, 770 us.  fp32
// 4096 x 4096 x 4096 572 to 659 us (random operands), 209 to 240 TFLOP/s.
#include "vc_linear.h"

namespace {

using namespace vcl;

typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint32_t u8w __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char LdsChar;
typedef __attribute__((address_space(3))) v4s LdsV4s;

// Tile w of ni x nj, eight tile rows at a time, so that tiles close in time share
// both operands in an XCD's L2.
__device__ __forceinline__ void tile_of(int64_t w, int ni, int nj, int& ti, int& tj) {
  const int64_t per = 8ll * nj;
  const int band = (int)(w / per), r = (int)(w - band * per), rows = min(8, ni - 8 * band);
  tj = r / rows;
  ti = 8 * band + r - tj * rows;
}

// One operand's side of a tile: R rows, NW waves.
template <bool X, int R, int BK, int NW>
struct Side {
  static constexpr int kGroups = R * BK * 2 / 1024;  // load instructions of one plane's step
  static constexpr int kOwn = kGroups / NW;
  static constexpr int kBytes = R * BK * 2;
  static_assert(kGroups % NW == 0, "every wave issues as many loads");
  const uint16_t* base;  // of the tile's first row and k
  uint32_t off[kOwn];    // bytes

  static __device__ __forceinline__ int fold(int k) { return ((k & 3) | ((k >> 3) & 1) << 2) & (R / 16 - 1); }

  // Which chunk of which row (across: of which line k) the lane brings in by its i-th load.
  static __device__ __forceinline__ void at(int i, int wv, int lane, int& line, int& chunk) {
    const int n = i * NW + wv;
    if (X) {
      constexpr int CR = R / 8;
      line = n * (64 / CR) + lane / CR;
      const int pos = lane % CR;
      chunk = ((pos >> 1) ^ fold(line)) * 2 + (pos & 1);
    } else {
      constexpr int CR = BK / 8;
      line = n * (64 / CR) + lane / CR;
      const int pos = lane % CR;
      chunk = pos ^ (BK == 64 ? line & 7 : (line >> 1) & 3);
    }
  }

  __device__ __forceinline__ void init(const uint16_t* p, int64_t ld, int rows, int r0, int64_t k0,
                                       int wv, int lane) {
    base = X ? p + k0 * ld + r0 : p + (int64_t)r0 * ld + k0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      int line, chunk;
      at(i, wv, lane, line, chunk);
      // past the last row the last again: its products are not stored
      if (X) off[i] = (uint32_t)(line * ld * 2) + min(chunk * 8, rows - 8 - r0) * 2;
      else off[i] = (uint32_t)(min(line, rows - 1 - r0) * ld * 2) + chunk * 16;
    }
  }

  // Whole steps: straight into LDS.
  __device__ __forceinline__ void issue(const uint16_t* from, char* lds, int wv) const {
    const Buf b = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(from), 0, 0x7fffffff,
                                                    0x00027000);
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          b, (__attribute__((address_space(3))) void*)(lds + (i * NW + wv) * 1024), 16, (int)off[i],
          0, 0, 0);
  }

  // The last step where K does not fill it (left < BK of it): zeros past the end.
  __device__ __forceinline__ void tail(const uint16_t* from, char* lds, int wv, int lane,
                                       int left) const {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      int line, chunk;
      at(i, wv, lane, line, chunk);
      const bool in = X ? line < left : chunk * 8 < left;
      const u4 v = *reinterpret_cast<const u4*>(reinterpret_cast<const char*>(from) + (in ? off[i] : 0));
      *reinterpret_cast<u4*>(lds + (i * NW + wv) * 1024 + lane * 16) = in ? v : u4{0, 0, 0, 0};
    }
  }

  // The fragment of 16 rows from row0 (a multiple of 16), k = 32 ks + 8 g + 0 .. 7.
  static __device__ __forceinline__ v8bf frag(const char* lds, int row0, int ks, int lane) {
    const int g = lane >> 4, r = lane & 15;
    if (X) {
      const int k = ks * 32 + 8 * g + (r >> 2);
      const char* const p = lds + k * (R * 2) + ((row0 >> 4) ^ fold(k)) * 32 + (r & 3) * 8;
      const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsV4s*)(LdsChar*)p);
      const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsV4s*)(LdsChar*)(p + 4 * R * 2));
      return __builtin_bit_cast(v8bf, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    const int c = (ks * 4 + g) ^ (BK == 64 ? r & 7 : (r >> 1) & 3);
    return *reinterpret_cast<const v8bf*>(lds + (row0 + r) * (BK * 2) + c * 16);
  }
};

// Up to n vector memory operations of this wave may still run (and any LDS ones,
// with lds none).
template <int N, bool LDS>
__device__ __forceinline__ void wait_for() {
  __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | (LDS ? 0 : 15) << 8 | (N >> 4) << 14);
}
// A workgroup barrier that waits for nothing else, and that nothing is moved over.
__device__ __forceinline__ void turn() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// A value put together from its three parts; an infinity or NaN stands in the first.
__device__ __forceinline__ float whole_value(const uint16_t* p, int64_t plane) {
  const float h = bf_lo(p[0]);
  return finite(h) ? (bf_lo(p[2 * plane]) + bf_lo(p[plane])) + h : h;
}

// The plain sum of the products k0 .. k1, where an infinity or NaN among the values
// (or a sum past the largest) has made what the parts' products cannot say.
template <bool XA, bool XB, class T>
__device__ float plain_sum(const Product<T>& a, int64_t i, int64_t j, int64_t k0, int64_t k1) {
  float s = 0.f;
#pragma unroll 1
  for (int64_t k = k0; k < k1 && s == s; ++k)  // NaN stays
    s += whole_value(a.pa + (XA ? k * a.lda + i : i * a.lda + k), a.planeA) *
         whole_value(a.pb + (XB ? k * a.ldb + j : j * a.ldb + k), a.planeB);
  return s;
}

// NBUF: LDS buffers.  TURNS: the waves take turns, one for each 32 of k.
template <class T, int NP, bool XA, bool XB, int BI, int BJ, int WI, int WJ, int BK, int NBUF,
          bool TURNS>
__device__ __forceinline__ void tile(const Product<T>& a, uint32_t block, char* lds) {
  constexpr int NW = WI * WJ, MI = BI / WI / 16, MJ = BJ / WJ / 16;
  typedef Side<XA, BI, BK, NW> SA;
  typedef Side<XB, BJ, BK, NW> SB;
  constexpr int kStage = NP * (SA::kBytes + SB::kBytes);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ni = (a.I + BI - 1) / BI, nj = (a.J + BJ - 1) / BJ;
  int ti, tj;
  // in scalar registers, as the bases of the loads into LDS have to be
  const int slice = __builtin_amdgcn_readfirstlane(block / (uint32_t)a.tiles);
  tile_of(vcg::xcd_tile(block - slice * (uint32_t)a.tiles, a.tiles), ni, nj, ti, tj);
  ti = __builtin_amdgcn_readfirstlane(ti);
  tj = __builtin_amdgcn_readfirstlane(tj);
  const int i0 = ti * BI, j0 = tj * BJ;
  const int64_t k0 = (int64_t)slice * a.steps * BK;
  const int left = (int)min((int64_t)a.steps * BK, a.K - k0);
  const int full = left / BK;
  const int wi = wv / WJ, wj = wv % WJ;

  SA sa;
  SB sb;
  // a line that is read across is padded to whole chunks
  sa.init(a.pa, a.lda, XA ? (a.I + 7) & ~7 : a.I, i0, k0, wv, lane);
  sb.init(a.pb, a.ldb, XB ? (a.J + 7) & ~7 : a.J, j0, k0, wv, lane);

  v4f acc[MI][MJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

  // A step of an operand whose k is contiguous is 64 or 128 bytes of each of its
  // rows, and rows a power of two apart lie in one channel of the L2: with two such
  // operands the tiles of an XCD start at eight places 256 bytes apart and wrap
  // (8192 x 16384 x 4096 1137 -> 1007 us; with one, 262 -> 283, the tiles then no
  // longer share what they read).
  const int first = XA || XB || full == 0 ? 0 : (int)(block >> 3) % 8 * (128 / BK) % full;
  const auto load = [&](int step, char* to) {
    const int s = step + first < full ? step + first : step + first - full;
    const uint16_t* const fa = sa.base + (XA ? (int64_t)s * BK * a.lda : (int64_t)s * BK);
    const uint16_t* const fb = sb.base + (XB ? (int64_t)s * BK * a.ldb : (int64_t)s * BK);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      sa.issue(fa + p * a.planeA, to + p * SA::kBytes, wv);
      sb.issue(fb + p * a.planeB, to + NP * SA::kBytes + p * SB::kBytes, wv);
    }
  };
  v8bf fb[MJ][NP], fa[MI][NP];
  const auto read = [&](const char* from, int ks) {
#pragma unroll
    for (int j = 0; j < MJ; ++j)
#pragma unroll
      for (int p = 0; p < NP; ++p)
        fb[j][p] = SB::frag(from + NP * SA::kBytes + p * SB::kBytes, (wj * MJ + j) * 16, ks, lane);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int p = 0; p < NP; ++p)
        fa[i][p] = SA::frag(from + p * SA::kBytes, (wi * MI + i) * 16, ks, lane);
  };
  const auto multiply = [&]() {
    if constexpr (NP == 1) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < MJ; ++j) acc[i][j] = mfma_bf16(fb[j][0], fa[i][0], acc[i][j]);
    } else {
      // a step's six products from zero, smallest first, added in fp32 while the
      // next rows' run
      v4f t[2][MJ];
#pragma unroll
      for (int i = 0; i <= MI; ++i) {
        if (i < MI) {
#pragma unroll
          for (int p = 0; p < 6; ++p)
#pragma unroll
            for (int j = 0; j < MJ; ++j)
              t[i & 1][j] = mfma_bf16(fb[j][kPartA[p]], fa[i][kPartB[p]],
                                      p ? t[i & 1][j] : v4f{0.f, 0.f, 0.f, 0.f});
        }
        if (i > 0) {
#pragma unroll
          for (int j = 0; j < MJ; ++j) acc[i - 1][j] += t[(i - 1) & 1][j];
        }
      }
    }
  };
  constexpr int kLoads = NP * (SA::kOwn + SB::kOwn), AHEAD = NBUF - 1;
  if (full > 0) {
    if constexpr (!TURNS) {
#pragma unroll
      for (int s = 0; s < AHEAD; ++s)
        if (s < full) load(s, lds + s * kStage);
      int at = 0;  // this step's buffer
#pragma unroll 1
      for (int s = 0; s < full; ++s) {
        // this step has arrived, the buffer of the one before is read
        if (s + AHEAD <= full) wait_for<(AHEAD - 1) * kLoads, true>();
        else wait_for<0, true>();
        turn();
        if (s + AHEAD < full) load(s + AHEAD, lds + (at == 0 ? NBUF - 1 : at - 1) * kStage);
#pragma unroll
        for (int ks = 0; ks < BK / 32; ++ks) {
          read(lds + at * kStage, ks);
          multiply();
        }
        at = at == NBUF - 1 ? 0 : at + 1;
      }
    } else {
      // Waves wv and wv + 4 share a SIMD; the later ones run a turn behind.  A
      // step's loads are issued in its wave's first reading turn, into the buffer
      // whose last reader was waited for at the turn's barrier, and waited for at
      // the barrier before the turn that reads them first.
      static_assert(NW == 8);
      constexpr int PH = BK / 32;
      const bool late = wv >= 4;
#pragma unroll
      for (int s = 0; s < AHEAD; ++s)
        if (s < full) load(s, lds + s * kStage);
      if (full >= AHEAD) wait_for<(AHEAD - 1) * kLoads, false>();
      else wait_for<0, false>();
      turn();
      if (late) turn();
      int at = 0;  // this step's buffer
#pragma unroll 1
      for (int s = 0; s < full; ++s) {
        const char* const from = lds + at * kStage;
        const int before = at == 0 ? NBUF - 1 : at - 1;
#pragma unroll
        for (int ph = 0; ph < PH; ++ph) {
          read(from, ph);
          if (ph == 0 && s + AHEAD < full) load(s + AHEAD, lds + before * kStage);
          if (ph == PH - 1 && late) {
            if (s + AHEAD < full) wait_for<(AHEAD - 1) * kLoads, true>();
            else wait_for<0, true>();
          } else {
            __builtin_amdgcn_s_waitcnt(15 | 7 << 4 | 3 << 14);  // fragments only
          }
          turn();
          __builtin_amdgcn_s_setprio(1);
          multiply();
          __builtin_amdgcn_s_setprio(0);
          if (ph == PH - 1 && !late) {
            if (s + AHEAD < full) wait_for<(AHEAD - 1) * kLoads, false>();
            else wait_for<0, false>();
          }
          turn();
        }
        at = at == NBUF - 1 ? 0 : at + 1;
      }
      if (!late) turn();
    }
  }
  if (left > full * BK) {
    const uint16_t* const fa = sa.base + (XA ? (int64_t)full * BK * a.lda : (int64_t)full * BK);
    const uint16_t* const fb = sb.base + (XB ? (int64_t)full * BK * a.ldb : (int64_t)full * BK);
    __syncthreads();
#pragma unroll 1
    for (int p = 0; p < NP; ++p) {
      sa.tail(fa + p * a.planeA, lds + p * SA::kBytes, wv, lane, left - full * BK);
      sb.tail(fb + p * a.planeB, lds + NP * SA::kBytes + p * SB::kBytes, wv, lane, left - full * BK);
    }
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < BK / 32; ++ks) {
      read(lds, ks);
      multiply();
    }
  }

  // The sums go through LDS, as many rows as fit: what follows them (bias,
  // activation, residual, stores of whole lines) is one short loop, eight rows of a
  // thread's four columns at a time (four where half of the sums stay in registers
  // meanwhile).  One after another, each waiting for its own loads, took 14 us of a 256
  // x 256 tile, this takes 5.  Four columns c of row i at c ^ (i mod 16).
  constexpr int Q = BJ / 4, kFit = NBUF * kStage / (BJ * 4), ROWS = kFit < BI ? BI / WI : BI;
  static_assert(ROWS <= kFit && Q >= 16);
  constexpr int STEP = 64 * NW / Q, U = ROWS < BI ? 4 : ROWS / STEP < 8 ? ROWS / STEP : 8;
  static_assert(64 * NW % Q == 0 && ROWS % (STEP * U) == 0);
  v4f* const sums = reinterpret_cast<v4f*>(lds);
  const int g = lane >> 4, r = lane & 15;
  const int q = tid % Q, row0 = tid / Q, j = j0 + 4 * q;
  const v4f bias = XB ? v4f{} : bias_of(a, j);
#pragma unroll 1
  for (int p = 0; p < BI / ROWS; ++p) {
    __syncthreads();
    if (ROWS == BI || p == wi) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < MJ; ++j) {
          const int row = ((ROWS == BI ? wi * MI : 0) + i) * 16 + r;
          sums[row * Q + (((wj * MJ + j) * 4 + g) ^ (row & 15))] = acc[i][j];
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int t = row0; t < ROWS; t += U * STEP) {
      const int i = i0 + p * ROWS + t;
      if (i >= a.I || j >= a.J) break;
      v4f w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = sums[(t + u * STEP) * Q + (q ^ ((t + u * STEP) & 15))];
      bool apart = a.slices == 1 && j + 4 > a.J;
      if constexpr (NP == 3) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int k = 0; k < 4; ++k) apart |= !finite(w[u][k]);
      }
      if (!apart && a.slices == 1) {
        finish_rows<T, XB>(a, i, STEP, j, bias, w);
      } else if (!apart) {
        const int line = part_line(a.J);
        float* const o = a.part + (slice * (int64_t)a.I + i) * line + j;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (i + u * STEP < a.I) *reinterpret_cast<v4f*>(o + (int64_t)u * STEP * line) = w[u];
      } else {
#pragma unroll 1
        for (int u = t; u < t + U * STEP && i0 + p * ROWS + u < a.I; u += STEP) {
          const int iu = i0 + p * ROWS + u;
          v4f x = sums[u * Q + (q ^ (u & 15))];
          if constexpr (NP == 3) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float v = x[k];
              if (!finite(v) && j + k < a.J)
                x[k] = plain_sum<XA, XB>(a, iu, j + k, k0, k0 + left);
            }
          }
          deliver<T, XB>(a, slice, iu, j, x);
        }
      }
    }
  }
}

template <class T, int SHAPE>
struct Form {
  static constexpr bool F = sizeof(T) == 4;
  static constexpr int NP = F ? 3 : 1;
  static constexpr int BI = SHAPE == 0 ? 256 : SHAPE == 1 ? 128 : 64;
  static constexpr int BJ = F && SHAPE == 0 ? 128 : BI;
  static constexpr bool TURNS = SHAPE == 0 || (F && SHAPE == 1);
  static constexpr int WI = F && SHAPE == 0 ? 4 : 2, WJ = (TURNS ? 8 : 4) / WI;
  static constexpr int BK = F ? 32 : 64;
  // 64 x 64 in bf16 has two buffers, so that four workgroups share a CU (2048 cubed,
  // backward's dW, 27 us; with four buffers and two workgroups 44), or as shape 3 four of
  // them for few workgroups whose operands come from far (20 x 12480 x 2624 14 us; with two
  // 20); fp32 has three (1024 cubed 22 us; with two 24)
  static constexpr int NBUF = F && SHAPE > 0 ? 3 : SHAPE == 3 ? 4 : 2;
  static constexpr int kThreads = 64 * WI * WJ;
  static constexpr int kLds = NBUF * NP * (BI + BJ) * BK * 2;
  template <bool XA, bool XB>
  static __device__ __forceinline__ void run(const Product<T>& a, uint32_t block, char* lds) {
    tile<T, NP, XA, XB, BI, BJ, WI, WJ, BK, NBUF, TURNS>(a, block, lds);
  }
};

template <class T, int SHAPE>
__global__ __launch_bounds__((Form<T, SHAPE>::kThreads), 2) void k_tile(Product<T> a) {
  extern __shared__ __align__(1024) char lds[];
  Form<T, SHAPE>::template run<false, false>(a, blockIdx.x, lds);
}

// Workgroups of dW (the longer sums), then of dx, then of the columns' sums.
template <class T, int SHAPE>
__global__ __launch_bounds__((Form<T, SHAPE>::kThreads), 2) void k_tiles(Product<T> w, Product<T> x,
                                                                      Columns<T> c) {
  extern __shared__ __align__(1024) char lds[];
  const uint32_t nw = w.tiles * w.slices, nx = x.tiles * x.slices, b = blockIdx.x;
  if (b < nw) Form<T, SHAPE>::template run<true, true>(w, b, lds);
  else if (b < nw + nx) Form<T, SHAPE>::template run<false, true>(x, b - nw, lds);
  else add_columns(c, (int)(b - nw - nx), reinterpret_cast<float*>(lds));
}

// fp32 forward products too small for the parts' pass: 64 x 32 tiles straight from
// x and W, on the fp32 matrix steps.  A row's 32 values of a step are 128 bytes, as
// 64 of bf16 are: the same loads and order of LDS.  A lane's 16 bytes are four k;
// matrix step q takes the q-th of every lane, the columns' operand alike.  Two
// groups of four waves take the steps in turn, each with three buffers of its own,
// and add their sums.
constexpr int kRawI = 64, kRawJ = 32, kRawBuf = 3;

__global__ __launch_bounds__(512, 2) void k_raw(Product<float> a) {
  typedef Side<false, kRawI, 64, 4> SA;
  typedef Side<false, kRawJ, 64, 4> SB;
  constexpr int kStage = SA::kBytes + SB::kBytes, kLoads = SA::kOwn + SB::kOwn, AHEAD = kRawBuf - 1;
  constexpr int Q = kRawJ / 4;
  __shared__ __align__(1024) char all[2 * kRawBuf * kStage];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6) & 3;
  const int grp = __builtin_amdgcn_readfirstlane(tid >> 8);
  const int slice = __builtin_amdgcn_readfirstlane(blockIdx.x / (uint32_t)a.tiles);
  const uint32_t w = (uint32_t)vcg::xcd_tile(blockIdx.x - slice * (uint32_t)a.tiles, a.tiles);
  const int ti = __builtin_amdgcn_readfirstlane(a.f_nj.div(w));
  const int i0 = ti * kRawI, j0 = ((int)w - ti * (int)a.f_nj.d) * kRawJ;
  const int k0 = slice * a.steps * 32, left = min(a.steps * 32, a.K - k0);
  const int steps = (left + 31) / 32, full = left / 32;
  const int wi = wv >> 1, wj = wv & 1, g = lane >> 4, r = lane & 15;
  char* const lds = all + grp * kRawBuf * kStage;
  SA sa;
  SB sb;
  // lengths and strides in bf16's: two to a value
  sa.init(reinterpret_cast<const uint16_t*>(a.A.p), 2 * a.A.ld, a.I, i0, 2 * (int64_t)k0, wv, lane);
  sb.init(reinterpret_cast<const uint16_t*>(a.B.p), 2 * a.B.ld, a.J, j0, 2 * (int64_t)k0, wv, lane);
  const auto load = [&](int s, int buf) {
    char* const to = lds + buf * kStage;
    if (s < full) {
      sa.issue(sa.base + s * 64, to, wv);
      sb.issue(sb.base + s * 64, to + SA::kBytes, wv);
    } else {
      sa.tail(sa.base + s * 64, to, wv, lane, 2 * (left - full * 32));
      sb.tail(sb.base + s * 64, to + SA::kBytes, wv, lane, 2 * (left - full * 32));
    }
  };
  v4f acc[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
  // the group's own steps: grp, grp + 2, ..; both groups pass as many barriers
  const int turns = (steps + 1) / 2;
#pragma unroll
  for (int t = 0; t < AHEAD; ++t)
    if (2 * t + grp < steps) load(2 * t + grp, t);
  int at = 0;
#pragma unroll 1
  for (int t = 0; t < turns; ++t) {
    // in flight beyond this step: the next one, when it is a whole one
    if (2 * (t + 1) + grp < full) wait_for<kLoads, true>();
    else wait_for<0, true>();
    turn();
    const int before = at == 0 ? kRawBuf - 1 : at - 1;
    if (2 * (t + AHEAD) + grp < steps) load(2 * (t + AHEAD) + grp, before);
    if (2 * t + grp < steps) {
      const char* const from = lds + at * kStage;
      v4f fa[2][2], fb[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = ((4 * h + g) ^ (r & 7)) * 16;
        fb[h] = *reinterpret_cast<const v4f*>(from + SA::kBytes + (wj * 16 + r) * 128 + c);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          fa[i][h] = *reinterpret_cast<const v4f*>(from + (wi * 32 + i * 16 + r) * 128 + c);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int i = 0; i < 2; ++i) acc[i] = mfma16x16x4(fb[h][q], fa[i][h][q], acc[i]);
    }
    at = at == kRawBuf - 1 ? 0 : at + 1;
  }
  // row, four columns c: at c ^ (row mod 8)
  v4f* const sums = reinterpret_cast<v4f*>(all);
  __syncthreads();
#pragma unroll
  for (int k = 1; k >= 0; --k) {
    if (grp == k) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = wi * 32 + i * 16 + r;
        v4f& s = sums[row * Q + ((wj * 4 + g) ^ (row & 7))];
        s = k ? acc[i] : s + acc[i];
      }
    }
    __syncthreads();
  }
  const int row = tid / Q, q = tid % Q, j = j0 + 4 * q;
  if (i0 + row >= a.I || j >= a.J) return;
  deliver<float, false>(a, slice, i0 + row, j, sums[row * Q + (q ^ (row & 7))]);
}

// A kernel's LDS limit, set once per device.
template <class K>
void allow_lds(K k, int bytes, bool* set) {
  int dev = 0;
  (void)hipGetDevice(&dev);
  if (set[dev & 15]) return;
  (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k),
                            hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  set[dev & 15] = true;
}

template <class T, int SHAPE>
void one(const Product<T>& a, hipStream_t st) {
  typedef Form<T, SHAPE> Fm;
  static bool set[16];
  allow_lds(k_tile<T, SHAPE>, Fm::kLds, set);
  k_tile<T, SHAPE><<<(unsigned)(a.tiles * a.slices), Fm::kThreads, Fm::kLds, st>>>(a);
}

template <class T, int SHAPE>
void both(const Product<T>& w, const Product<T>& x, const Columns<T>& c, unsigned grid, hipStream_t st) {
  typedef Form<T, SHAPE> Fm;
  static bool set[16];
  allow_lds(k_tiles<T, SHAPE>, Fm::kLds, set);
  k_tiles<T, SHAPE><<<grid, Fm::kThreads, Fm::kLds, st>>>(w, x, c);
}

}  // namespace

namespace vcl {

TileShape tile_shape(int type, int shape) {
  const int bk = type == VC_FP32 ? 32 : 64;
  if (shape == 0) return {256, type == VC_FP32 ? 128 : 256, bk};
  return shape == 1 ? TileShape{128, 128, bk} : TileShape{64, 64, bk};
}

void run_raw(const Product<float>& a, hipStream_t st) {
  k_raw<<<(unsigned)(a.tiles * a.slices), 512, 0, st>>>(a);
}

template <class T>
void run_tile(const Product<T>& a, int shape, hipStream_t st) {
  if (shape == 0) one<T, 0>(a, st);
  else if (shape == 1) one<T, 1>(a, st);
  else if (sizeof(T) == 4 || shape == 2) one<T, 2>(a, st);
  else if constexpr (sizeof(T) == 2) one<T, 3>(a, st);
}
template <class T>
void run_tiles(const Product<T>& w, const Product<T>& x, const Columns<T>& c, int shape,
               unsigned grid, hipStream_t st) {
  if (shape == 0) both<T, 0>(w, x, c, grid, st);
  else if (shape == 1) both<T, 1>(w, x, c, grid, st);
  else both<T, 2>(w, x, c, grid, st);
}
template void run_tile<float>(const Product<float>&, int, hipStream_t);
template void run_tile<uint16_t>(const Product<uint16_t>&, int, hipStream_t);
template void run_tiles<float>(const Product<float>&, const Product<float>&, const Columns<float>&,
                               int, unsigned, hipStream_t);
template void run_tiles<uint16_t>(const Product<uint16_t>&, const Product<uint16_t>&,
                                  const Columns<uint16_t>&, int, unsigned, hipStream_t);

}  // namespace vcl
