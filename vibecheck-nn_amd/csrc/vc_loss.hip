// Softmax cross-entropy of rows of logits, and its gradient:
//   lse = log sum_j exp(z_j),  loss = lse - (1 - e) z_t - (e / V) sum_j z_j,
//   dz_j = s (exp(z_j - lse) - (1 - e) [j = t] - e / V),
// s = 1, or one over the number of rows that count (mean).  A row whose target
// is `ignore` adds nothing; one whose target is no class gives NaN.  A row
// without any logit above -inf has an infinite loss and no gradient.
//
// With m the largest logit and S = sum over j != t of exp(z_j - m), the target's
// gradient is -S / (S + exp(z_t - m)) + e - e / V and the loss log(S + exp(z_t -
// m)) + (m - z_t): nothing cancels where the target's probability is near one,
// or where the logits are large beside their differences.
#include <type_traits>
#include <utility>

#include "vc_common.h"

namespace {

struct Rows {
  const void* z;
  int64_t R, V, ld;
  const int64_t* t;
  int64_t ignore;
  float smooth;
  int mean;            // the gradient is of the mean over the rows that count
  const float* scale;  // mean: one over their number; null: counted here
  float* loss;         // (R)
  void* dz;            // null: no gradient
  int64_t ldd;
  float* joined;       // k_loss_few: the sum or mean, or null
};

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const uint16_t* p) {
  return __builtin_bit_cast(float, (uint32_t)*p << 16);
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(uint16_t* p, float v) {
  *p = __builtin_bit_cast(uint16_t, (__bf16)v);
}

typedef uint32_t u4at4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4at2 __attribute__((ext_vector_type(4), aligned(2)));

// Sixteen bytes of a row, at any alignment of its type.
template <class T>
struct Chunk {
  static constexpr int kN = 16 / sizeof(T);
  static constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : 0xff80u;  // -inf
  typedef std::conditional_t<sizeof(T) == 4, u4at4, u4at2> Any;
  static __device__ __forceinline__ u4 load(const T* p) { return *reinterpret_cast<const Any*>(p); }
  static __device__ __forceinline__ void store(T* p, u4 v) { *reinterpret_cast<Any*>(p) = v; }
  static __device__ __forceinline__ float value(u4 w, int i) {
    const uint32_t u = sizeof(T) == 4 ? w[i % 4] : i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16;
    return __builtin_bit_cast(float, u);
  }
  static __device__ __forceinline__ u4 pack(const float* v) {
    u4 w;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, v[i]);
    } else {
      typedef float v2f __attribute__((ext_vector_type(2)));
      typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{v[2 * i], v[2 * i + 1]}, v2bf));
    }
    return w;
  }
  static __device__ __forceinline__ u4 none_at(u4 w, int i) {  // -inf in place i
    if constexpr (sizeof(T) == 4) {
      return u4{i == 0 ? kNone : w[0], i == 1 ? kNone : w[1], i == 2 ? kNone : w[2],
                i == 3 ? kNone : w[3]};
    } else {
      const uint32_t m = i & 1 ? 0xffffu : 0xffff0000u, v = i & 1 ? kNone << 16 : kNone;
      return u4{i / 2 == 0 ? (w[0] & m) | v : w[0], i / 2 == 1 ? (w[1] & m) | v : w[1],
                i / 2 == 2 ? (w[2] & m) | v : w[2], i / 2 == 3 ? (w[3] & m) | v : w[3]};
    }
  }
  // The first n values dropped, -inf behind the others.
  static __device__ __forceinline__ u4 drop(u4 w, int n) {
    constexpr uint32_t f = sizeof(T) == 4 ? kNone : kNone | kNone << 16;
    if constexpr (sizeof(T) == 4) {
      w = n & 2 ? u4{w[2], w[3], f, f} : w;
      w = n & 1 ? u4{w[1], w[2], w[3], f} : w;
    } else {
      w = n & 4 ? u4{w[2], w[3], f, f} : w;
      w = n & 2 ? u4{w[1], w[2], w[3], f} : w;
      w = n & 1 ? u4{w[0] >> 16 | w[1] << 16, w[1] >> 16 | w[2] << 16, w[2] >> 16 | w[3] << 16,
                     w[3] >> 16 | f << 16} : w;
    }
    return n >= kN ? u4{f, f, f, f} : w;
  }
};

// f(0), f(1), .., each with a constant: an array indexed by them is in registers
// from the start.
template <class F, int... K>
__device__ __forceinline__ void each(std::integer_sequence<int, K...>, F f) {
  (f(std::integral_constant<int, K>{}), ...);
}

constexpr float kLog2e = 1.44269504088896341f;
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// The running maximum and sum of exponentials of two parts of a row joined.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  if (top == -INFINITY) {  // nothing yet, or NaN sums
    s += s2;
    return;
  }
  s = s * exp_of(m - top) + s2 * exp_of(m2 - top);
  m = top;
}

// others: the sum without the target's term et, in units of em, the largest
// logit's own term; half: half the logits' mean, which rounding cannot take past
// the largest value.
__device__ __forceinline__ float row_loss(float m, float others, float et, float em, float zt,
                                          float half, float e) {
  const float v = log1pf((others + (et - em)) / em);
  if (e == 0.f) return v + (m - zt);
  return v + ((1.f - e) * (m - zt) + e * (2.f * (0.5f * m - half)));
}

// Rows that one wavefront or a workgroup of W waves takes: sums and maxima over
// its threads, each wave's part through LDS where there are several.
template <int W>
struct Team {
  float (*sh)[W];
  int lane, wv;
  __device__ __forceinline__ float max_of(float v) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    if (W == 1) return v;
    if (lane == 0) sh[0][wv] = v;
    __syncthreads();
    v = sh[0][0];
#pragma unroll
    for (int i = 1; i < W; ++i) v = fmaxf(v, sh[0][i]);
    return v;
  }
  __device__ __forceinline__ void sums(float& a, float& b, bool two) {
    a = wave_sum(a);
    if (two) b = wave_sum(b);
    if (W == 1) return;
    if (lane == 0) {
      sh[1][wv] = a;
      sh[2][wv] = b;
    }
    __syncthreads();
    a = sh[1][0];
    b = sh[2][0];
#pragma unroll
    for (int i = 1; i < W; ++i) a += sh[1][i], b += sh[2][i];
  }
};

// One over the rows that count, by every wave for itself (few rows, one launch).
__device__ __forceinline__ float scale_of(const Rows& a, int lane) {
  if (!a.mean) return 1.f;
  if (a.scale) return *a.scale;
  int n = 0;
  for (int64_t i = lane; i < a.R; i += 64) n += a.t[i] != a.ignore;
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  return 1.f / (float)n;
}

// A row's largest logit within kFar of zero: its product with log2 e is off by at most
// a quarter, and the whole number above it is exact.  Further out (half a last place of the
// product is 128 from 3e9 on) the difference has to come before the product: plain_row.
// A thread's reference starts at kLowest, below any that such a row can end with, so that
// logits far below (masks such as -1e10 or -1e30) add zeros, alone in a thread too.
constexpr float kFar = 0x1p22f, kLowest = -0x1p23f;
static_assert(-kLowest > kFar * kLog2e + 1.f, "what a thread starts with lies below");

// A row of any values, two passes over memory: rows without a finite largest
// logit, or one too far from zero.
template <class T, int W>
__device__ void plain_row(const Rows& a, const T* z, T* dz, int64_t t, float zt, int tid, float w,
                          float* loss, Team<W> team) {
  const float iv = 0.5f / (float)a.V;
  const bool valid = t >= 0 && t < a.V;
  float m = -INFINITY, s = 0.f, half = 0.f;
  for (int64_t j = tid; j < a.V; j += 64 * W) {
    const float v = load1(z + j);
    // a NaN is no maximum: it is kept in the sum, before there is a maximum too
    join(m, s, v, v != v ? v : v == -INFINITY || j == t ? 0.f : 1.f);
    half += v * iv;
  }
  if (W > 1) __syncthreads();
  const float top = team.max_of(m);
  s = top == -INFINITY ? s : s * exp_of(m - top);
  m = top;
  team.sums(s, half, true);  // after its barrier the target's logit may be overwritten
  const bool none = m == -INFINITY && s == 0.f;
  const float et = exp_of(zt - m);
  if (tid == 0) *loss = !valid ? NAN : none ? INFINITY : row_loss(m, s, et, 1.f, zt, half, a.smooth);
  if (!dz) return;
  const float inv = 1.f / (s + et), ev = a.smooth / (float)a.V;
  for (int64_t j = tid; j < a.V; j += 64 * W) {
    const float p = j == t ? a.smooth - s * inv : exp_of(load1(z + j) - m) * inv;
    store1(dz + j, !valid ? NAN : none ? 0.f : (p - ev) * w);
  }
}

// A row is read once: its chunks stay in the team's registers, NV a thread (the row
// ends within the last ENDS of them), or (NV 0, rows that do not fit) are read again
// for the gradient.
//
// While chunks arrive a thread keeps r, a whole number not below its largest
// logit times log2 e, and the sum of 2^(z log2 e - r): one fma and one
// exponential a value, and moving to another r multiplies by a power of two,
// which rounds nothing.  What the rounding of log2 e does to large logits is in
// every term, the largest's own (em) too, and cancels; a thread that meets one beyond
// kFar may end with any sum, its row goes to plain_row.  The target's term is kept
// apart (its place holds -inf meanwhile).
//
// Memory bounds it: 8,192 x 131,072 bf16, logits read and gradient written, 760 us
// (5.6 TB/s), x 50,021 343 (4.8); read twice, as the first kernel did, 2,726.  1000 x 50,021
// fp32 rows that no 16 bytes divide, 91 us (4.4).  A team is as small as holds its row in at most 16
// chunks a thread: what a smaller one saves is the joins across waves, what a larger
// one saves is registers: of sixteen waves with up to 4 chunks a thread (58 to 60
// registers) a CU has two teams, with 6 (68 to 72) to 16 (110 to 124) one.
template <class T, int W, int NV, int ENDS, bool SMOOTH>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void k_loss_rows(Rows a) {
  typedef Chunk<T> C;
  typedef std::conditional_t<NV != 0, int, int64_t> Index;  // held rows: 32 bits beside the row's base
  constexpr int N = C::kN, TH = 64 * W, NB = NV ? NV : 4;
  __shared__ float sh[3][W];
  const int tid = W == 1 ? threadIdx.x & 63 : threadIdx.x, lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = W == 1 ? blockIdx.x * 4ll + wv : blockIdx.x;
  if (row >= a.R) return;
  Team<W> team{sh, lane, wv};
  const T* const z = (const T*)a.z + row * a.ld;
  T* const dz = a.dz ? (T*)a.dz + row * a.ldd : nullptr;
  const int64_t t = a.t[row];
  // a bf16 row at an odd place: its first value goes by itself, the chunks start at a
  // multiple of four bytes (8192 x 50021 498 us without, 343 with)
  const int h = sizeof(T) == 2 && ((uintptr_t)z & 2) ? 1 : 0;
  const T* const zh = z + h;
  T* const dzh = dz + h;
  const int64_t V = a.V - h;
  // chunks; what is left over belongs to chunk `whole`
  const Index whole = (Index)(V / N), chunks = (Index)((V + N - 1) / N);
  if (t == a.ignore) {
    if (tid == 0) a.loss[row] = 0.f;
    if (dz) {
      for (int64_t c = tid; c < whole; c += TH) C::store(dzh + c * N, u4{0, 0, 0, 0});
      for (int64_t j = whole * N + tid; j < V; j += TH) store1(dzh + j, 0.f);
      if (h && tid == 0) store1(dz, 0.f);
    }
    return;
  }
  const bool valid = t >= 0 && t < a.V;
  const float zt = load1(z + (valid ? t : 0)), z0 = load1(z), iv = 0.5f / (float)a.V;
  const Index ct = valid && t >= h ? (Index)((t - h) / N) : -1;
  const auto at = [](auto* p, Index c) {
    typedef std::remove_pointer_t<decltype(p)> P;
    if constexpr (NV != 0) return p + (uint32_t)c * (uint32_t)N;
    else return (P*)p + c * N;
  };
  // Every lane loads a whole chunk, one that would pass the row's end the row's
  // last: a branch that lanes do not share would have each load waited for before
  // the next.  What is not the chunk's own is masked when it is taken.
  const Index last = (Index)(V - N);
  const auto fetch = [&](Index c) {
    const Index e = c < whole ? c * N : last;
    if constexpr (NV != 0) return C::load(zh + (uint32_t)e);
    else return C::load(zh + e);
  };
  // Of chunks first .. first + TH - 1, that of this lane: a part of one is moved to
  // its front, the rest is -inf.
  const auto mask = [&](u4 w, Index c, Index first) {
    if (first + TH <= whole) return w;  // the same in all lanes
    return C::drop(w, c < whole ? 0 : c == whole ? (int)((int64_t)c * N - last) : N);
  };
  float m = -INFINITY, r = kLowest, s = 0.f, half = 0.f;
  const auto take = [&](u4 w, Index c, Index first, bool end) {
    if (end) w = mask(w, c, first);
    asm volatile("" : "+v"(w));  // one chunk's values at a time
    if (SMOOTH) {
      if (!end || first + TH <= whole) {
#pragma unroll
        for (int i = 0; i < N; ++i) half += C::value(w, i) * iv;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) half += (int64_t)c * N + i < V ? C::value(w, i) * iv : 0.f;
      }
      // the values are unpacked again for the sum below, not kept beside these: with three
      // times the registers chunks would spill
      asm volatile("" : "+v"(half));
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" : "+v"(w));
    }
    if (c == ct) w = C::none_at(w, (int)(t - h - (int64_t)ct * N));
    float top = C::value(w, 0);
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, C::value(w, i));
    if (top > m) {
      m = top;
      const float to = fmaxf(ceilf(m * kLog2e), r);
      s *= __builtin_amdgcn_exp2f(r - to);
      r = to;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      s += __builtin_amdgcn_exp2f(__builtin_fmaf(C::value(w, i), kLog2e, -r));
    return w;
  };
  u4 v[NB];
  constexpr std::make_integer_sequence<int, NB> held{};
  if (NV) {
    each(held, [&](auto k) { v[k] = fetch(tid + k * TH); });
    each(held, [&](auto k) {
      v[k] = take(v[k], tid + k * TH, k * TH, k >= NV - ENDS);
      __builtin_amdgcn_sched_barrier(0);  // one chunk's floats at a time
    });
  } else {
    for (Index c = 0; c < chunks; c += NB * TH) {
      each(held, [&](auto k) { v[k] = fetch(c + tid + k * TH); });
      each(held, [&](auto k) { take(v[k], c + tid + k * TH, c + k * TH, true); });
    }
  }
  if (h && tid == 0) {
    if (SMOOTH) half += z0 * iv;
    if (t != 0) {
      if (z0 > m) {
        m = z0;
        const float to = fmaxf(ceilf(m * kLog2e), r);
        s *= __builtin_amdgcn_exp2f(r - to);
        r = to;
      }
      s += __builtin_amdgcn_exp2f(__builtin_fmaf(z0, kLog2e, -r));
    }
  }
  const float w = scale_of(a, lane);
  const float top = team.max_of(fmaxf(m, zt));
  if (!(fabsf(top) < kFar)) {  // the same in every thread of the row
    plain_row<T, W>(a, z, dz, t, zt, tid, w, a.loss + row, team);
    return;
  }
  const float to = ceilf(top * kLog2e);
  s *= __builtin_amdgcn_exp2f(r - to);
  r = to;
  team.sums(s, half, SMOOTH);
  const float em = __builtin_amdgcn_exp2f(__builtin_fmaf(top, kLog2e, -r));
  const float et = __builtin_amdgcn_exp2f(__builtin_fmaf(zt, kLog2e, -r));
  if (tid == 0) a.loss[row] = valid ? row_loss(top, s, et, em, zt, half, a.smooth) : NAN;
  if (!dz) return;
  const float inv = valid ? w / (s + et) : NAN, ev = a.smooth / (float)a.V * w;
  const float at_t = a.smooth * w - s * inv - ev;
  const auto grad = [&](float x) {
    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x, kLog2e, -r));
    return SMOOTH ? __builtin_fmaf(p, inv, -ev) : p * inv;
  };
  const auto give = [&](u4 x, Index c, bool end) {
    asm volatile("" : "+v"(x));  // unpacked again here, not kept from before: twice the registers
    float g[N];
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = grad(C::value(x, i));
    if (!end || c < whole) {
      C::store(at(dzh, c), C::pack(g));
    } else if (c == whole) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if ((int64_t)c * N + i < V) store1(dzh + (int64_t)c * N + i, g[i]);
    }
  };
  if (NV) {
    each(held, [&](auto k) {
      give(v[k], tid + k * TH, k >= NV - ENDS);
      __builtin_amdgcn_sched_barrier(0);
    });
  } else {
    // dz may be z: a lane reads its chunk's own values before it writes them (what
    // else a chunk at the row's end brings is masked)
    for (Index c = 0; c < chunks; c += NB * TH) {
      each(held, [&](auto k) { v[k] = fetch(c + tid + k * TH); });
      each(held, [&](auto k) {
        give(mask(v[k], c + tid + k * TH, c + k * TH), c + tid + k * TH, true);
      });
    }
  }
  if (h && tid == 0) store1(dz, valid && t == 0 ? at_t : grad(z0));
  // its own place, over what the chunk left there, by the same thread
  if (ct >= 0 && tid == (int)(ct % TH)) store1(dz + t, at_t);
}

// Few classes: a thread a row, its values from the caches for each of its passes.
// With ONE the whole call is this workgroup: the rows are counted and their
// losses added here too: 512 x 10 fp32 takes one launch instead of three (10.6 us a call
// with the caller's host time, 19.8 before).
constexpr int kFew = 32;

template <class T, int TH, bool ONE>
__global__ __launch_bounds__(TH) void k_loss_few(Rows a) {
  __shared__ double sums[TH / 64];
  __shared__ int counts[TH / 64];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x * (int64_t)TH + tid;
  const bool in = row < a.R;
  const int64_t t = in ? a.t[row] : 0;
  const bool on = in && t != a.ignore, valid = t >= 0 && t < a.V;
  float w = 1.f;
  int count = 0;
  if (ONE) {
    const int n = __popcll(__ballot(on));
    if ((tid & 63) == 0) counts[tid >> 6] = n;
    __syncthreads();
    for (int i = 0; i < TH / 64; ++i) count += counts[i];
    if (a.mean) w = 1.f / (float)count;
  } else if (a.mean) {
    w = *a.scale;
  }
  float loss = 0.f;
  const int V = (int)a.V;
  if (on) {
    const T* const z = (const T*)a.z + row * a.ld;
    T* const dz = a.dz ? (T*)a.dz + row * a.ldd : nullptr;
    const float zt = load1(z + (valid ? t : 0)), iv = 0.5f / (float)V;
    float m = -INFINITY, s = 0.f, half = 0.f;
    for (int j = 0; j < V; ++j) m = fmaxf(m, load1(z + j));
    const bool none = m == -INFINITY;
    for (int j = 0; j < V; ++j) {
      const float v = load1(z + j);
      half += v * iv;
      if (j != t) s += none && v == m ? 0.f : exp_of(v - m);
    }
    const float et = exp_of(zt - m);
    const bool empty = none && s == 0.f;
    loss = !valid ? NAN : empty ? INFINITY : row_loss(m, s, et, 1.f, zt, half, a.smooth);
    if (dz) {
      const float inv = 1.f / (s + et), ev = a.smooth / (float)V;
      for (int j = 0; j < V; ++j) {
        const float p = j == t ? a.smooth - s * inv : exp_of(load1(z + j) - m) * inv;
        store1(dz + j, !valid ? NAN : empty ? 0.f : (p - ev) * w);
      }
    }
  } else if (in && a.dz) {
    for (int j = 0; j < V; ++j) store1((T*)a.dz + row * a.ldd + j, 0.f);
  }
  if (!ONE || !a.joined) {
    if (in) a.loss[row] = loss;
    return;
  }
  const double sum = wave_sum_f64((double)loss);
  if ((tid & 63) == 0) sums[tid >> 6] = sum;
  __syncthreads();
  if (tid) return;
  double all = 0.0;
  for (int i = 0; i < TH / 64; ++i) all += sums[i];
  *a.joined = (float)(a.mean ? all / (double)count : all);
}

// scale[0] = one over the number of rows that count.
__global__ __launch_bounds__(1024) void k_loss_count(const int64_t* t, int64_t R, int64_t ignore,
                                                     float* scale) {
  __shared__ int sh[16];
  int n = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < R; i += 1024) n += t[i] != ignore;
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) n += sh[i];
    *scale = 1.f / (float)n;
  }
}

// The rows' losses added in a fixed order, in 64 bits; averaged over the rows
// that count.
__global__ __launch_bounds__(1024) void k_loss_sum(const float* loss, int64_t R, const int64_t* t,
                                                   int64_t ignore, int mean, float* out) {
  __shared__ double sh[16];
  __shared__ int shn[16];
  double s = 0.0;
  int n = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < R; i += 1024) {
    s += (double)loss[i];
    if (mean) n += t[i] != ignore;
  }
  for (int o = 32; o > 0; o >>= 1) {
    s += __shfl_xor(s, o, 64);
    n += __shfl_xor(n, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    sh[threadIdx.x >> 6] = s;
    shn[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) s += sh[i], n += shn[i];
    *out = (float)(mean ? s / (double)n : s);
  }
}

// A launch has fewer than 2^32 threads: more rows than 2^31 threads take (33 million by a
// wave each, 2 million by sixteen) go by several.
template <class T, int W, int NV, int ENDS>
void run_rows(const Rows& a, hipStream_t st) {
  const int64_t most = (1ll << 31) / (64 * W);
  const int threads = W == 1 ? 256 : 64 * W;
  for (int64_t at = 0; at < a.R; at += most) {
    Rows b = a;
    b.R = a.R - at < most ? a.R - at : most;
    b.z = (const T*)a.z + at * a.ld;
    b.t = a.t + at;
    b.loss = a.loss + at;
    if (a.dz) b.dz = (T*)a.dz + at * a.ldd;
    const unsigned grid = (unsigned)(W == 1 ? (b.R + 3) / 4 : b.R);
    if (a.smooth != 0.f) k_loss_rows<T, W, NV, ENDS, true><<<grid, threads, 0, st>>>(b);
    else k_loss_rows<T, W, NV, ENDS, false><<<grid, threads, 0, st>>>(b);
  }
}

constexpr int64_t kOneRows = 1024;    // of k_loss_few by one workgroup
constexpr int64_t kCountRows = 1024;  // that every wave counts by itself
static_assert(kCountRows <= (1ll << 31) / 1024, "one launch has them all");

// The team of a row: as many waves as hold it in at most 16 chunks a thread; the
// row's end lies in the last chunks of a thread, those past the limit before.
template <class T>
void run_loss(const Rows& a, hipStream_t st) {
  const auto fits = [&](int waves, int held) { return a.V <= 64ll * waves * held * Chunk<T>::kN; };
  if (a.V <= kFew) {
    if (a.R <= kOneRows) k_loss_few<T, kOneRows, true><<<1, kOneRows, 0, st>>>(a);
    else k_loss_few<T, 256, false><<<(unsigned)((a.R + 255) / 256), 256, 0, st>>>(a);
  } else if (fits(1, 1)) run_rows<T, 1, 1, 1>(a, st);
  else if (fits(1, 2)) run_rows<T, 1, 2, 1>(a, st);
  else if (fits(1, 4)) run_rows<T, 1, 4, 2>(a, st);
  else if (fits(4, 2)) run_rows<T, 4, 2, 1>(a, st);
  else if (fits(4, 3)) run_rows<T, 4, 3, 1>(a, st);
  else if (fits(4, 4)) run_rows<T, 4, 4, 1>(a, st);
  else if (fits(4, 6)) run_rows<T, 4, 6, 2>(a, st);
  else if (fits(4, 8)) run_rows<T, 4, 8, 2>(a, st);
  else if (fits(16, 3)) run_rows<T, 16, 3, 1>(a, st);
  else if (fits(16, 4)) run_rows<T, 16, 4, 1>(a, st);
  else if (fits(16, 6)) run_rows<T, 16, 6, 2>(a, st);
  else if (fits(16, 8)) run_rows<T, 16, 8, 2>(a, st);
  else if (fits(16, 10)) run_rows<T, 16, 10, 2>(a, st);
  else if (fits(16, 13)) run_rows<T, 16, 13, 3>(a, st);
  else if (fits(16, 16)) run_rows<T, 16, 16, 3>(a, st);
  else run_rows<T, 16, 0, 0>(a, st);
}

}  // namespace

extern "C" int64_t vc_cross_entropy_workspace(int64_t R, int reduction) {
  if (R < 0) return -1;
  return reduction == VC_REDUCE_NONE ? 0 : 256 + (4 * R + 255) / 256 * 256;
}

extern "C" int vc_cross_entropy(int type, const void* logits, int64_t R, int64_t V, int64_t ld,
                                const int64_t* target, int64_t ignore, float smoothing,
                                int reduction, float* loss, void* dlogits, int64_t ldd, void* work,
                                int64_t work_bytes, vc_stream_t stream) {
  if ((type != VC_FP32 && type != VC_BF16) || R < 0 || R > 0x7fffffff || V < 1 || ld < V ||
      !(smoothing >= 0.f && smoothing <= 1.f) || reduction < VC_REDUCE_NONE ||
      reduction > VC_REDUCE_MEAN || (dlogits && ldd < V))
    return VC_ERR_ARG;
  if (R == 0 && reduction == VC_REDUCE_NONE) return VC_OK;
  if (!loss || (R > 0 && (!logits || !target))) return VC_ERR_ARG;
  const int64_t need = vc_cross_entropy_workspace(R, reduction);
  if (need > work_bytes || (need && !work)) return VC_ERR_OOM;
  hipStream_t st = (hipStream_t)stream;
  const bool mean = reduction == VC_REDUCE_MEAN, joined = reduction != VC_REDUCE_NONE;
  // with few rows of few classes one workgroup is the whole call; with few rows
  // their number is counted by every wave, which spares a launch
  const bool one = V <= kFew && R <= kOneRows;
  float* const scale = mean && !one && (R > kCountRows || V <= kFew) ? (float*)work : nullptr;
  Rows a = {logits, R,  V,    ld, target, ignore, smoothing, mean && (one || dlogits), scale,
            joined ? (float*)work + 64 : loss, dlogits, ldd, one && joined ? loss : nullptr};
  if (scale && dlogits) k_loss_count<<<1, 1024, 0, st>>>(target, R, ignore, scale);
  if (R > 0 || one) {
    if (type == VC_FP32) run_loss<float>(a, st);
    else run_loss<uint16_t>(a, st);
  }
  if (joined && !one)
    k_loss_sum<<<1, 1024, 0, st>>>(a.loss, R, target, ignore, mean, loss);
  VC_LAUNCH_CHECK();
  return VC_OK;
}
