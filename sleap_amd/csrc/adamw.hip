// One AdamW step over many tensors:
//     m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2          [w = max(w, v)]
//     p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(w or v) / sqrt(1 - b2^t) + eps)
// in 32 bits per value whatever the parameter's type; a 16-bit parameter is rounded once, to nearest.
//
// Memory bound: 28 bytes a value with float32 parameters (36 with the running maximum). A launch carries the addresses of up to
// SLOTS tensors in its arguments -- no table in device memory to fill, nothing kept between calls, and a captured launch holds its
// own copy -- and as many workgroups as the tensors have pieces of CHUNK values; a workgroup finds its tensor with one ballot.
#include "sa_common.h"
#include "token_types.h"

namespace {

using namespace sa;

constexpr int SLOTS = 64;      // 64 x 48 bytes + the piece table: within the 4 KB of kernel arguments
constexpr int CHUNK = 4096;    // values of a workgroup: 256 threads x 4 pieces of 4

struct Slot {
  void* p;
  const void* g;
  float *m, *v, *w;
  int64_t n;
};

struct AdamwParams {
  Slot slot[SLOTS];
  uint32_t first[SLOTS];      // first workgroup of each tensor
  int n;
  float lr, decay, b1, b2, eps;
  float c1, c2;               // 1 - b1^t, sqrt(1 - b2^t) of a step counted on the host
  const float* lr_dev;        // a learning rate in device memory (or NULL)
  const int64_t* step_dev;    // a step counter in device memory (or NULL)
  double b1d, b2d;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

struct Rates {
  float b1, a1, b2, a2, eps, keep, rate, root;
};

template <bool AMS>
__device__ __forceinline__ void one(float& p, float g, float& m, float& v, float& w, const Rates& r) {
  m = r.b1 * m + r.a1 * g;
  v = r.b2 * v + r.a2 * (g * g);
  float u = v;
  if constexpr (AMS) u = w = (v > w || v != v) ? v : w;  // a NaN stays
  p = p * r.keep - r.rate * (m / (sqrtf(u) * r.root + r.eps));
}

template <typename T, bool AMS, int V>
__device__ __forceinline__ void chunk(const Slot& s, int64_t at, const Rates& r) {
  T* p = static_cast<T*>(s.p);
  const T* g = static_cast<const T*>(s.g);
  const int64_t end = min(at + CHUNK, s.n);
  constexpr int K = CHUNK / (256 * V);
  if (V > 1 && end - at == CHUNK) {  // a whole piece: every load is issued before the first use
    using VT = Vec<T, V>;
    using VF = Vec<float, V>;
    VT pp[K], gg[K];
    VF mm[K], vv[K], ww[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t i = at + (k * 256 + threadIdx.x) * V;
      pp[k] = *reinterpret_cast<const VT*>(p + i);
      gg[k] = *reinterpret_cast<const VT*>(g + i);
      mm[k] = *reinterpret_cast<const VF*>(s.m + i);
      vv[k] = *reinterpret_cast<const VF*>(s.v + i);
      if constexpr (AMS) ww[k] = *reinterpret_cast<const VF*>(s.w + i);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t i = at + (k * 256 + threadIdx.x) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float x = to_f32(pp[k].e[e]);
        one<AMS>(x, to_f32(gg[k].e[e]), mm[k].e[e], vv[k].e[e], ww[k].e[e], r);
        pp[k].e[e] = from_f32<T>(x);
      }
      *reinterpret_cast<VT*>(p + i) = pp[k];
      *reinterpret_cast<VF*>(s.m + i) = mm[k];
      *reinterpret_cast<VF*>(s.v + i) = vv[k];
      if constexpr (AMS) *reinterpret_cast<VF*>(s.w + i) = ww[k];
    }
    return;
  }
  for (int64_t i = at + threadIdx.x; i < end; i += 256) {
    float x = to_f32(p[i]), m = s.m[i], v = s.v[i], w = AMS ? s.w[i] : 0.0f;
    one<AMS>(x, to_f32(g[i]), m, v, w, r);
    p[i] = from_f32<T>(x);
    s.m[i] = m;
    s.v[i] = v;
    if constexpr (AMS) s.w[i] = w;
  }
}

template <typename T, bool AMS>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamwParams a) {
  // the last tensor that begins at or before this workgroup: one read and a ballot (SLOTS == lanes of a wave)
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t begun = __ballot((int)lane < a.n && a.first[lane] <= blockIdx.x);
  const int lo = __builtin_amdgcn_readfirstlane(63 - __clzll(begun));
  float c1 = a.c1, c2 = a.c2;
  if (a.step_dev) {
    const double t = (double)*a.step_dev;
    c1 = (float)(1.0 - pow(a.b1d, t));
    c2 = (float)sqrt(1.0 - pow(a.b2d, t));
  }
  const float lr = a.lr_dev ? *a.lr_dev : a.lr;
  const Rates r = {a.b1, (float)(1.0 - a.b1d), a.b2, (float)(1.0 - a.b2d), a.eps, 1.0f - lr * a.decay, lr / c1, 1.0f / c2};
  const Slot s = a.slot[lo];
  const uint64_t any = (uint64_t)s.m | (uint64_t)s.v | (AMS ? (uint64_t)s.w : 0);
  const bool wide = any % 16 == 0 && ((uint64_t)s.p | (uint64_t)s.g) % (4 * sizeof(T)) == 0;
  const int64_t at = (int64_t)(blockIdx.x - a.first[lo]) * CHUNK;
  if (wide) chunk<T, AMS, 4>(s, at, r);
  else chunk<T, AMS, 1>(s, at, r);
}

template <typename T>
void launch(const AdamwParams& a, bool ams, uint32_t blocks, hipStream_t s) {
  if (ams) adamw_kernel<T, true><<<dim3(blocks), dim3(256), 0, s>>>(a);
  else adamw_kernel<T, false><<<dim3(blocks), dim3(256), 0, s>>>(a);
}

}  // namespace

extern "C" int sa_adamw_step(const sa_adamw_tensor* tensors, int n, int dtype, int amsgrad, double lr, const float* lr_dev, double beta1,
                             double beta2, double eps, double weight_decay, int64_t step, const int64_t* step_dev, sa_stream_t stream) {
  SA_REQUIRE(n >= 0 && (n == 0 || tensors), "sa_adamw_step: bad tensor list");
  SA_REQUIRE(dtype == SA_F32 || dtype == SA_F16 || dtype == SA_BF16, "sa_adamw_step: bad dtype %d", dtype);
  SA_REQUIRE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "sa_adamw_step: betas must lie in [0, 1)");
  SA_REQUIRE(eps >= 0 && weight_decay >= 0 && (lr_dev || lr >= 0), "sa_adamw_step: lr, eps and weight_decay must not be negative");
  SA_REQUIRE(step_dev || step >= 1, "sa_adamw_step: the first step is 1");
  for (int i = 0; i < n; ++i) {
    const sa_adamw_tensor& t = tensors[i];
    SA_REQUIRE(t.n >= 0 && (t.n == 0 || (t.param && t.grad && t.exp_avg && t.exp_avg_sq && (!amsgrad || t.max_exp_avg_sq))),
               "sa_adamw_step: tensor %d has a negative size or a null address", i);
    SA_REQUIRE((t.n + CHUNK - 1) / CHUNK < (1ll << 24), "sa_adamw_step: tensor %d has more than 2^36 values", i);
  }
  AdamwParams a;
  a.lr = (float)lr;
  a.decay = (float)weight_decay;
  a.b1 = (float)beta1;
  a.b2 = (float)beta2;
  a.eps = (float)eps;
  a.b1d = beta1;
  a.b2d = beta2;
  a.c1 = (float)(1.0 - pow(beta1, (double)step));
  a.c2 = (float)sqrt(1.0 - pow(beta2, (double)step));
  a.lr_dev = lr_dev;
  a.step_dev = step_dev;
  for (int at = 0; at < n;) {
    a.n = 0;
    uint32_t blocks = 0;
    for (; at < n && a.n < SLOTS; ++at) {
      const sa_adamw_tensor& t = tensors[at];
      if (t.n == 0) continue;
      a.slot[a.n] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.max_exp_avg_sq, t.n};
      a.first[a.n++] = blocks;
      blocks += (uint32_t)((t.n + CHUNK - 1) / CHUNK);
    }
    if (a.n == 0) break;
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == SA_F32) launch<float>(a, amsgrad, blocks, s);
    else if (dtype == SA_F16) launch<_Float16>(a, amsgrad, blocks, s);
    else launch<__bf16>(a, amsgrad, blocks, s);
    SA_LAUNCH_CHECK();
  }
  return SA_OK;
}
