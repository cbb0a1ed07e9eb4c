// One AdamW step over many tensors:
//     m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2          [w = max(w, v)]
//     p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(w or v) / sqrt(1 - b2^t) + eps)
// in 32 bits per value whatever the parameter's type; a 16-bit parameter is rounded once, to nearest.
//
// Memory bound: 28 bytes a value with float32 parameters (36 with the running maximum). A launch carries the addresses of up to
// 128 tensors in its arguments -- no table in device memory to fill, nothing kept between calls, and a captured launch holds its
// own copy -- and as many workgroups as the tensors have pieces of CHUNK values; a workgroup finds its tensor with two ballots. 66 M values in 448
// tensors, with the running maximum: 483 us = 4.9 TB/s (a large copy: 5.1).
#include "sa_common.h"
#include "token_types.h"

namespace {

using namespace sa;

constexpr int CHUNK = 4096;  // values of a workgroup: 256 threads x 4 pieces of 4

// What a workgroup has of its tensor
struct Slot {
  void* p;
  const void* g;
  float *m, *v, *w;
  int n;
};

// As many tensors as the 4 KB of kernel arguments hold (448 tensors of four addresses: 4 launches; as plain structures of 48 bytes 7): 48-bit
// addresses in two parts, and of the size only what the workgroups' numbers do not say already.
template <bool AMS>
struct AdamwParams {
  static constexpr int ADDRESSES = AMS ? 5 : 4, SLOTS = AMS ? 108 : 128;
  uint32_t low[ADDRESSES][SLOTS];
  uint16_t high[ADDRESSES][SLOTS];
  uint16_t tail[SLOTS];     // values of a tensor's last workgroup
  uint32_t first[SLOTS];    // first workgroup of each tensor
  uint32_t blocks;
  int n;
  float lr, decay, b1, b2, eps;
  float c1, c2;             // 1 - b1^t, sqrt(1 - b2^t) of a step counted on the host
  const float* lr_dev;      // a learning rate in device memory (or NULL)
  const int64_t* step_dev;  // a step counter in device memory (or NULL)
  double b1d, b2d;
};
static_assert(sizeof(AdamwParams<false>) <= 4096 && sizeof(AdamwParams<true>) <= 4096, "kernel arguments");

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
__device__ __forceinline__ void chunk(const Slot& s, const Rates& r) {
  T* p = static_cast<T*>(s.p);
  const T* g = static_cast<const T*>(s.g);
  constexpr int K = CHUNK / (256 * V);
  if (V > 1 && s.n == CHUNK) {  // a whole piece: every load is issued before the first use
    using VT = Vec<T, V>;
    using VF = Vec<float, V>;
    VT pp[K], gg[K];
    VF mm[K], vv[K], ww[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = (k * 256 + threadIdx.x) * V;
      pp[k] = *reinterpret_cast<const VT*>(p + i);
      gg[k] = *reinterpret_cast<const VT*>(g + i);
      mm[k] = *reinterpret_cast<const VF*>(s.m + i);
      vv[k] = *reinterpret_cast<const VF*>(s.v + i);
      if constexpr (AMS) ww[k] = *reinterpret_cast<const VF*>(s.w + i);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = (k * 256 + threadIdx.x) * V;
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
  for (int i = threadIdx.x; i < s.n; i += 256) {
    float x = to_f32(p[i]), m = s.m[i], v = s.v[i], w = AMS ? s.w[i] : 0.0f;
    one<AMS>(x, to_f32(g[i]), m, v, w, r);
    p[i] = from_f32<T>(x);
    s.m[i] = m;
    s.v[i] = v;
    if constexpr (AMS) s.w[i] = w;
  }
}

template <typename T, bool AMS>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamwParams<AMS> a) {
  // the last tensor that begins at or before this workgroup: two reads and ballots for up to 128
  const int lane = threadIdx.x & 63;
  const uint64_t one_ = __ballot(lane < a.n && a.first[lane] <= blockIdx.x);
  const uint64_t two = __ballot(lane + 64 < a.n && a.first[min(lane + 64, a.SLOTS - 1)] <= blockIdx.x);
  const int slot = __builtin_amdgcn_readfirstlane(two ? 127 - __clzll(two) : 63 - __clzll(one_));
  const uint32_t begin = a.first[slot], end = slot + 1 < a.n ? a.first[slot + 1] : a.blocks;
  const int64_t at = (int64_t)(blockIdx.x - begin) * CHUNK;
  auto address = [&](int k) { return (uint64_t)a.high[k][slot] << 32 | a.low[k][slot]; };
  float c1 = a.c1, c2 = a.c2;
  if (a.step_dev) {
    const double t = (double)*a.step_dev;
    c1 = (float)(1.0 - pow(a.b1d, t));
    c2 = (float)sqrt(1.0 - pow(a.b2d, t));
  }
  const float lr = a.lr_dev ? *a.lr_dev : a.lr;
  const Rates r = {a.b1, (float)(1.0 - a.b1d), a.b2, (float)(1.0 - a.b2d), a.eps, 1.0f - lr * a.decay, lr / c1, 1.0f / c2};
  Slot s;
  s.p = reinterpret_cast<T*>(address(0)) + at;
  s.g = reinterpret_cast<const T*>(address(1)) + at;
  s.m = reinterpret_cast<float*>(address(2)) + at;
  s.v = reinterpret_cast<float*>(address(3)) + at;
  s.w = AMS ? reinterpret_cast<float*>(address(AMS ? 4 : 0)) + at : nullptr;
  s.n = blockIdx.x + 1 == end ? a.tail[slot] : CHUNK;
  const uint64_t any = (uint64_t)s.m | (uint64_t)s.v | (AMS ? (uint64_t)s.w : 0);
  const bool wide = any % 16 == 0 && ((uint64_t)s.p | (uint64_t)s.g) % (4 * sizeof(T)) == 0;
  if (wide) chunk<T, AMS, 4>(s, r);
  else chunk<T, AMS, 1>(s, r);
}

template <bool AMS>
int step_all(AdamwParams<AMS>& a, const sa_adamw_tensor* tensors, int n, int dtype, hipStream_t s) {
  for (int at = 0; at < n;) {
    a.n = 0;
    a.blocks = 0;
    for (; at < n && a.n < a.SLOTS; ++at) {
      const sa_adamw_tensor& t = tensors[at];
      if (t.n == 0) continue;
      const void* address[5] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.max_exp_avg_sq};
      for (int k = 0; k < a.ADDRESSES; ++k) {
        a.low[k][a.n] = (uint32_t)(uintptr_t)address[k];
        a.high[k][a.n] = (uint16_t)((uintptr_t)address[k] >> 32);
      }
      const uint32_t pieces = (uint32_t)((t.n + CHUNK - 1) / CHUNK);
      if (a.n && (uint64_t)a.blocks + pieces >= (1ull << 24)) break;  // a launch has less than 2^32 threads
      a.tail[a.n] = (uint16_t)(t.n - (int64_t)(pieces - 1) * CHUNK);
      a.first[a.n++] = a.blocks;
      a.blocks += pieces;
    }
    if (a.n == 0) break;
    const dim3 grid(a.blocks), block(256);
    if (dtype == SA_F32) adamw_kernel<float, AMS><<<grid, block, 0, s>>>(a);
    else if (dtype == SA_F16) adamw_kernel<_Float16, AMS><<<grid, block, 0, s>>>(a);
    else adamw_kernel<__bf16, AMS><<<grid, block, 0, s>>>(a);
    SA_LAUNCH_CHECK();
  }
  return SA_OK;
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
    SA_REQUIRE((((uintptr_t)t.param | (uintptr_t)t.grad | (uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq | (uintptr_t)(amsgrad ? t.max_exp_avg_sq : nullptr)) >> 48) == 0,
               "sa_adamw_step: tensor %d: addresses have 48 bits", i);
    SA_REQUIRE(t.n <= (1ll << 36) - CHUNK, "sa_adamw_step: tensor %d has more than 2^36 values", i);
  }
  auto go = [&](auto& a) {
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
    return step_all(a, tensors, n, dtype, (hipStream_t)stream);
  };
  if (amsgrad) {
    AdamwParams<true> a;
    return go(a);
  }
  AdamwParams<false> a;
  return go(a);
}
