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
#include "vc_common.h"

namespace {

constexpr int CNT = 256;  // threads of a row

struct Rows {
  const void* z;
  int64_t R, V, ld;
  const int64_t* t;
  int64_t ignore;
  float smooth;
  int mean;
  const float* scale;  // mean: one over the rows that count
  float* loss;         // (R)
  void* dz;            // null: no gradient
  int64_t ldd;
};

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const uint16_t* p) {
  return __builtin_bit_cast(float, (uint32_t)*p << 16);
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(uint16_t* p, float v) {
  *p = __builtin_bit_cast(uint16_t, (__bf16)v);
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

// others: the sum without the target's term et; half: half the logits' mean, which
// rounding cannot take past the largest value.
__device__ __forceinline__ float row_loss(float m, float others, float et, float zt, float half,
                                          float e) {
  if (m == -INFINITY && others == 0.f) return INFINITY;
  float v = log1pf(others + (et - 1.f));
  if (e == 0.f) return v + (m - zt);
  return v + ((1.f - e) * (m - zt) + e * (2.f * (0.5f * m - half)));
}

// One workgroup a row: a pass for the running maximum and sum, one for the
// gradient.
template <class T>
__global__ __launch_bounds__(CNT) void k_loss_rows(Rows a) {
  __shared__ float sh[3][CNT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t row = blockIdx.x;
  const T* const z = (const T*)a.z + row * a.ld;
  T* const dz = a.dz ? (T*)a.dz + row * a.ldd : nullptr;
  const int64_t t = a.t[row];
  if (t == a.ignore) {
    if (tid == 0) a.loss[row] = 0.f;
    if (dz)
      for (int64_t j = tid; j < a.V; j += CNT) store1(dz + j, 0.f);
    return;
  }
  const bool valid = t >= 0 && t < a.V;
  const float zt = load1(z + (valid ? t : 0)), iv = 0.5f / (float)a.V;
  float m = -INFINITY, s = 0.f, half = 0.f;
  for (int64_t j = tid; j < a.V; j += CNT) {
    const float v = load1(z + j);
    join(m, s, v, v == -INFINITY || j == t ? 0.f : 1.f);
    half += v * iv;
  }
  for (int o = 32; o > 0; o >>= 1) {
    join(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64));
    half += __shfl_xor(half, o, 64);
  }
  if (lane == 0) {
    sh[0][wv] = m;
    sh[1][wv] = s;
    sh[2][wv] = half;
  }
  __syncthreads();  // and dz may be z: the target's logit is read
  m = sh[0][0];
  s = sh[1][0];
  half = sh[2][0];
  for (int i = 1; i < CNT / 64; ++i) {
    join(m, s, sh[0][i], sh[1][i]);
    half += sh[2][i];
  }
  const float et = exp_of(zt - m);
  if (tid == 0) a.loss[row] = valid ? row_loss(m, s, et, zt, half, a.smooth) : NAN;
  if (!dz) return;
  const bool none = m == -INFINITY && s == 0.f;
  const float w = a.mean ? *a.scale : 1.f;
  const float inv = 1.f / (s + et), ev = a.smooth / (float)a.V;
  for (int64_t j = tid; j < a.V; j += CNT) {
    const float p = j == t ? a.smooth - s * inv : exp_of(load1(z + j) - m) * inv;
    store1(dz + j, !valid ? NAN : none ? 0.f : (p - ev) * w);
  }
}

// scale[0] = one over the number of rows that count.
__global__ __launch_bounds__(1024) void k_loss_count(const int64_t* t, int64_t R, int64_t ignore,
                                                     float* scale) {
  __shared__ int sh[16];
  int n = 0;
  for (int64_t i = threadIdx.x; i < R; i += 1024) n += t[i] != ignore;
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) n += sh[i];
    *scale = n ? 1.f / (float)n : NAN;
  }
}

// The rows' losses added in a fixed order, in 64 bits.
__global__ __launch_bounds__(1024) void k_loss_sum(const float* loss, int64_t R, const float* scale,
                                                   float* out) {
  __shared__ double sh[16];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < R; i += 1024) s += (double)loss[i];
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) s += sh[i];
    *out = (float)(scale ? s * (double)*scale : s);
  }
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
  float* const scale = (float*)work;
  const bool mean = reduction == VC_REDUCE_MEAN, joined = reduction != VC_REDUCE_NONE;
  Rows a = {logits, R,    V,     ld, target, ignore, smoothing, mean, scale,
            joined ? (float*)work + 64 : loss, dlogits, ldd};
  if (mean) k_loss_count<<<1, 1024, 0, st>>>(target, R, ignore, scale);
  if (R > 0) {
    if (type == VC_FP32) k_loss_rows<float><<<(unsigned)R, CNT, 0, st>>>(a);
    else k_loss_rows<uint16_t><<<(unsigned)R, CNT, 0, st>>>(a);
  }
  if (joined) k_loss_sum<<<1, 1024, 0, st>>>(a.loss, R, mean ? scale : nullptr, loss);
  VC_LAUNCH_CHECK();
  return VC_OK;
}
