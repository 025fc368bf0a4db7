// One AdamW step over many tensors:
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps),
// the update in adam_update's order.  A launch takes up to
// kTensors tensors, described in its arguments, so that nothing is copied to the
// device or kept between calls.
//
// The state of all tensors is two arrays, each tensor padded to whole blocks of
// 256 values: a wavefront takes one block, four values a lane.  Memory bounds it: 16
// blocks a workgroup keep enough loads on their way (403 million values in 32 bits,
// 28 bytes each, 1.87 to 2.15 ms, 5.2 to 6.0 TB/s; 200 million in 8 bits, 16 bytes each,
// 669 us, 4.8), and small tensors cost a share of one launch.  In 32 bits it
// holds m and v.  In 8 bits it holds m and u = sqrt(v) as e4m3 values with one
// fp32 scale a block, the block's largest / 448, and each is rounded up or down
// with the probability of what is cut, by a hash of its place and the step.
// Rounded to nearest instead, v would stand still after a few steps: with b2 =
// 0.999 one changes u by at most 1/2000 of it in the long run, the grid's step
// is 1/8 to 1/16.  u has half of v's octaves, and one that is positive is never
// stored as zero, so that m / (u + eps) stays bounded (a block that is all below 2^-100
// is: the square of such a gradient is below fp32's smallest value).
#include "vc_common.h"

namespace {

constexpr int ANT = 256;
constexpr int kBlock = 256;       // values that share a scale
constexpr int kBlocksPerWg = 16;  // of one tensor
constexpr int kTensors = 88;
constexpr int64_t kMostWgs = 1 << 23;  // threads of a grid: below 2^32

struct Tensor {
  void* p;
  const void* g;
  uint16_t* c;  // bf16 copy of p, or null
  int64_t n;
  int64_t b0;   // its first block in the state
};

struct Step {
  Tensor t[kTensors];
  int w0[kTensors];  // its first workgroup
  int n;
  uint32_t seed;
  float decay, b1;
  AdamConst c;
  void *m, *v;
  float *ms, *vs;
  const float* scale;  // of the gradients, or null
};
static_assert(sizeof(Step) <= 4096, "a launch's arguments");

__device__ __forceinline__ float up(uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2bf));
}

// At any alignment of the type.
typedef float v4fat4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u2at2 __attribute__((ext_vector_type(2), aligned(2)));

// Values i .. i + 3 of n; past the end zero (WHOLE: none is).
template <bool WHOLE>
__device__ __forceinline__ void load4(const float* p, int64_t i, int64_t n, float* o) {
  if (WHOLE) {
    const v4fat4 w = *reinterpret_cast<const v4fat4*>(p + i);
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = w[q];
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = i + q < n ? p[i + q] : 0.f;
  }
}
template <bool WHOLE>
__device__ __forceinline__ void load4(const uint16_t* p, int64_t i, int64_t n, float* o) {
  if (WHOLE) {
    const u2at2 w = *reinterpret_cast<const u2at2*>(p + i);
    o[0] = up((uint16_t)w.x);
    o[1] = __builtin_bit_cast(float, w.x & 0xffff0000u);
    o[2] = up((uint16_t)w.y);
    o[3] = __builtin_bit_cast(float, w.y & 0xffff0000u);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = i + q < n ? up(p[i + q]) : 0.f;
  }
}
template <bool WHOLE>
__device__ __forceinline__ void store4(float* p, int64_t i, int64_t n, const float* v) {
  if (WHOLE) {
    *reinterpret_cast<v4fat4*>(p + i) = v4fat4{v[0], v[1], v[2], v[3]};
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (i + q < n) p[i + q] = v[q];
  }
}
template <bool WHOLE>
__device__ __forceinline__ void store4(uint16_t* p, int64_t i, int64_t n, const float* v) {
  if (WHOLE) {
    *reinterpret_cast<u2at2*>(p + i) = u2at2{pack2(v[0], v[1]), pack2(v[2], v[3])};
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (i + q < n) p[i + q] = (uint16_t)pack2(v[q], 0.f);
  }
}

// The largest magnitude of a block, as bits: NaN is above everything.
__device__ __forceinline__ float block_max(const float* x) {
  uint32_t t = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) t = max(t, __builtin_bit_cast(uint32_t, x[q]) & 0x7fffffffu);
  for (int o = 32; o > 0; o >>= 1) t = max(t, (uint32_t)__shfl_xor((int)t, o, 64));
  return __builtin_bit_cast(float, t);
}

// Four values as e4m3 bytes, and the block's scale (0: the block is zeros).
// From the smallest normal, 2^-6, up the byte is cut from the float's bits after
// the dither is added, below it is a count of 2^-9.
template <bool POSITIVE>
__device__ __forceinline__ uint32_t encode(const float* x, const uint32_t* dither, float& scale) {
  const float top = block_max(x);
  const bool none = top < 0x1p-100f;
  const float inv = none ? 0.f : __fdiv_rn(1.f, top) * 448.f;
  scale = none ? 0.f : top * (1.f / 448.f);
  uint32_t out = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float t = fabsf(x[q]) * inv;
    int code = (int)((__builtin_bit_cast(uint32_t, t) + dither[q]) >> 20) - 960;
    if (t < 0x1p-6f) code = (int)(t * 512.f + (float)dither[q] * 0x1p-20f);
    code = min(code, 126);
    if (POSITIVE) code = t > 0.f ? max(code, 1) : code;
    else code |= (int)(__builtin_bit_cast(uint32_t, x[q]) >> 24 & 0x80);
    out |= (uint32_t)code << 8 * q;
  }
  return out;
}

__device__ __forceinline__ void decode(uint32_t w, float scale, float* o) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const v2f b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  o[0] = a.x * scale;
  o[1] = a.y * scale;
  o[2] = b.x * scale;
  o[3] = b.y * scale;
}

// Twenty bits for the rounding of the value at place i (a multiplicative hash
// with the fractions of the golden ratio and of the square roots of 2 and 3).
__device__ __forceinline__ uint32_t dither_of(uint32_t i, uint32_t seed) {
  uint32_t h = i * 0x9E3779B9u + seed;
  h = (h ^ h >> 15) * 0xBB67AE85u;
  return (h ^ h >> 15) >> 12;
}

// One value's update, every operation rounded by itself; v becomes its root.  What is
// stored follows from m and the root by a cut, so their last bits decide: they are those
// of the plain sequence of operations (__fsqrt_rn can be off by one).  The parameter's are
// too: with a product by a reciprocal it is off by some 2^-22 of the step (200 million
// values 652 us, so 669).
__device__ __forceinline__ float update8(float p, float g, float& m, float& v, const Step& a) {
  m = a.b1 * m + a.c.w1 * g;
  v = __builtin_sqrtf(a.c.b2 * v + a.c.w2 * g * g);
  return p + __fdiv_rn(a.c.neg_step * m, __fdiv_rn(v, a.c.bc2) + a.c.eps);
}

template <class P, class G, int BITS, bool WHOLE>
__device__ __forceinline__ void step_block(const Step& a, const Tensor& t, int64_t blk, int lane,
                                           float gs) {
  const int64_t i = blk * kBlock + 4 * lane, at = (t.b0 + blk) * kBlock + 4 * lane;
  float p[4], g[4], m[4], v[4];
  load4<WHOLE>((const P*)t.p, i, t.n, p);
  load4<WHOLE>((const G*)t.g, i, t.n, g);
  if (BITS == 32) {
    load4<true>((const float*)a.m, at, 0, m);
    load4<true>((const float*)a.v, at, 0, v);
  } else {
    decode(((const uint32_t*)a.m)[at >> 2], a.ms[t.b0 + blk], m);
    decode(((const uint32_t*)a.v)[at >> 2], a.vs[t.b0 + blk], v);
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] *= v[q];
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (a.scale) g[q] *= gs;
    if (BITS == 32) p[q] = adam_update(p[q] * a.decay, g[q], m[q], v[q], a.c);
    else p[q] = update8(p[q] * a.decay, g[q], m[q], v[q], a);
  }
  store4<WHOLE>((P*)t.p, i, t.n, p);
  if (t.c) store4<WHOLE>(t.c, i, t.n, p);
  if (BITS == 32) {
    store4<true>((float*)a.m, at, 0, m);
    store4<true>((float*)a.v, at, 0, v);
  } else {
    uint32_t d[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) d[q] = dither_of((uint32_t)at + q, a.seed);
    float sm, sv;
    const uint32_t cm = encode<false>(m, d, sm), cv = encode<true>(v, d, sv);
    ((uint32_t*)a.m)[at >> 2] = cm;
    ((uint32_t*)a.v)[at >> 2] = cv;
    if (lane == 0) {
      a.ms[t.b0 + blk] = sm;
      a.vs[t.b0 + blk] = sv;
    }
  }
}

template <class P, class G, int BITS>
__global__ __launch_bounds__(ANT) void k_adamw(Step a) {
  float gs = 1.f;
  if (a.scale) {
    gs = *a.scale;
    if (!(fabsf(gs) <= 3.402823466e38f)) return;  // an overflow somewhere: no step
  }
  const int w = blockIdx.x, lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lo = 0, hi = a.n;  // w0[lo] <= w < w0[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.w0[mid] <= w) lo = mid;
    else hi = mid;
  }
  const Tensor t = a.t[lo];
  const int64_t blocks = (t.n + kBlock - 1) / kBlock;
  const int64_t b = (int64_t)(w - a.w0[lo]) * kBlocksPerWg;
  for (int k = wv; k < kBlocksPerWg; k += ANT / 64) {
    const int64_t blk = b + k;
    if (blk >= blocks) break;
    if ((blk + 1) * kBlock <= t.n) step_block<P, G, BITS, true>(a, t, blk, lane, gs);
    else step_block<P, G, BITS, false>(a, t, blk, lane, gs);
  }
}

template <class P, class G>
void launch(const Step& a, int bits, int grid, hipStream_t st) {
  if (bits == 8) k_adamw<P, G, 8><<<grid, ANT, 0, st>>>(a);
  else k_adamw<P, G, 32><<<grid, ANT, 0, st>>>(a);
}

}  // namespace

extern "C" int vc_adamw_step(const void* const* p, const void* const* g, const void* const* copy,
                             const int64_t* n, int count, int ptype, int gtype, int bits, void* m,
                             void* v, float* m_scale, float* v_scale, double lr, double b1,
                             double b2, double eps, double weight_decay, int64_t step,
                             const float* scale, vc_stream_t stream) {
  if (count < 0 || (ptype != VC_FP32 && ptype != VC_BF16) || (gtype != VC_FP32 && gtype != VC_BF16) ||
      (bits != 8 && bits != 32) || step < 1 || !(b1 >= 0 && b1 < 1) || !(b2 >= 0 && b2 < 1) ||
      !(eps >= 0) || (count > 0 && (!p || !g || !n)))
    return VC_ERR_ARG;
  int64_t total = 0;
  for (int i = 0; i < count; ++i) {
    if (n[i] < 0 || (n[i] > 0 && (!p[i] || !g[i]))) return VC_ERR_ARG;
    total += n[i];
  }
  if (total == 0) return VC_OK;
  for (int i = 0; i < count; ++i)  // all of them before the first is changed
    if (n[i] > kMostWgs * kBlocksPerWg * kBlock) return VC_ERR_UNSUPPORTED;
  if (!m || !v || !aligned16(m) || !aligned16(v) || (bits == 8 && (!m_scale || !v_scale)))
    return VC_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  Step a;
  a.seed = (uint32_t)step * 0x6A09E667u;
  a.decay = (float)(1.0 - lr * weight_decay);
  a.b1 = (float)b1;
  a.c = adam_const(b1, b2, eps, lr / (1.0 - pow(b1, (double)step)),
                   sqrt(1.0 - pow(b2, (double)step)));
  a.m = m;
  a.v = v;
  a.ms = m_scale;
  a.vs = v_scale;
  a.scale = scale;
  int64_t block = 0, wgs = 0;
  a.n = 0;
  const auto flush = [&]() {
    if (a.n == 0) return;
    const int grid = (int)wgs;
    if (ptype == VC_FP32) {
      if (gtype == VC_FP32) launch<float, float>(a, bits, grid, st);
      else launch<float, uint16_t>(a, bits, grid, st);
    } else {
      if (gtype == VC_FP32) launch<uint16_t, float>(a, bits, grid, st);
      else launch<uint16_t, uint16_t>(a, bits, grid, st);
    }
    a.n = 0;
    wgs = 0;
  };
  for (int i = 0; i < count; ++i) {
    const int64_t blocks = (n[i] + kBlock - 1) / kBlock;
    const int64_t w = (blocks + kBlocksPerWg - 1) / kBlocksPerWg;
    if (w == 0) continue;
    if (a.n == kTensors || wgs + w > kMostWgs) flush();
    a.t[a.n] = Tensor{const_cast<void*>(p[i]), g[i], copy ? (uint16_t*)copy[i] : nullptr, n[i], block};
    a.w0[a.n++] = (int)wgs;
    wgs += w;
    block += blocks;
  }
  flush();
  VC_LAUNCH_CHECK();
  return VC_OK;
}
