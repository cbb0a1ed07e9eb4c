// Rotary positions with several axes: every pair of a head's values belongs to one axis of the token's position (time, row,
// column of a clip, or x, y of a keypoint) and is turned by  angle = position[axis] * frequency:
//     (a, b) -> (a cos - b sin, b cos + a sin)        gradient: the same with -angle (the inverse turn)
// Angles are held in TURNS in 64 bits, their whole part is taken off there, and only the fraction goes to 32 bits: the frame index
// of a long video (1e6) times a frequency of 1 leaves 4 bits of a float's 24 for the fraction of a turn.
//
// Memory bound: one read and one write of x. All heads of a token share its angles, so a workgroup takes a run of tokens, puts
// their cosines and sines in LDS once (tokens x pairs x 8 bytes), and then walks the run's values in memory order, 16 bytes a
// lane and load where sizes and addresses allow it. 2 x 32768 tokens x 8 x 64 bf16: 27 us with cold inputs = 4.9 TB/s (a large copy: 5.1).
#include "sa_common.h"
#include "token_types.h"

namespace {

using namespace sa;

constexpr int MAX_PAIRS = 128, MAX_AXES = 8;

struct RotaryParams {
  const void* x;
  void* y;
  const void* pos;
  int pos_type;
  int64_t xb, xt, xh;      // strides of x, in elements
  int64_t pb, pt, pa;      // strides of the positions
  int T, H, D, P, tok;     // tokens, heads, head size, pairs, tokens of a workgroup
  uint32_t tiles, blocks;  // workgroups of a batch entry, of the launch
  FastDiv div_tiles, div_g, div_h, div_p;
  int G;                   // pieces of a head: P / V (or 2P / V) rotated ones, then the ones that pass
  int rot;                 // how many of them are rotated
  float sign;
  double freq[MAX_PAIRS];  // in turns per unit of position
  uint8_t axis[MAX_PAIRS];
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Piece {
  T e[V];
};

__device__ __forceinline__ double position(const RotaryParams& p, int64_t i) {
  if (p.pos_type == SA_POS_F32) return static_cast<const float*>(p.pos)[i];
  if (p.pos_type == SA_POS_I32) return static_cast<const int32_t*>(p.pos)[i];
  return (double)static_cast<const int64_t*>(p.pos)[i];
}

template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p) {
  extern __shared__ float2 cs[];  // [tok][P]
  const uint32_t block = workgroup();
  if (block >= p.blocks) return;
  const uint32_t b = div_by(block, p.div_tiles);
  const int t0 = (int)(block - b * p.tiles) * p.tok;
  const int nt = min(p.tok, p.T - t0);
  for (uint32_t i = threadIdx.x; i < (uint32_t)(nt * p.P); i += 256) {
    const uint32_t t = div_by(i, p.div_p), j = i - t * p.P;
    const double turns = position(p, (int64_t)b * p.pb + (int64_t)(t0 + t) * p.pt + (int64_t)p.axis[j] * p.pa) * p.freq[j];
    const float r = (float)(turns - rint(turns));
    float s, c;
    sincospif(2.0f * r, &s, &c);
    cs[i] = make_float2(c, p.sign * s);
  }
  __syncthreads();
  using Pc = Piece<T, V>;
  const T* xb = static_cast<const T*>(p.x) + (int64_t)b * p.xb;
  T* yb = static_cast<T*>(p.y) + (int64_t)b * p.T * p.H * p.D;
  const uint32_t items = (uint32_t)nt * p.H * p.G;
  for (uint32_t i = threadIdx.x; i < items; i += 256) {  // (two or four pieces a lane and turn: the same time)
    const uint32_t row = div_by(i, p.div_g), g = i - row * p.G;
    const uint32_t t = div_by(row, p.div_h), h = row - t * p.H;
    const bool turned = g < (uint32_t)p.rot;  // values behind the pairs pass
    const int e = (INTERLEAVED || turned ? 0 : p.P) + (int)g * V;
    const T* src = xb + (int64_t)(t0 + t) * p.xt + (int64_t)h * p.xh + e;
    T* dst = yb + ((int64_t)(t0 + t) * p.H + h) * p.D + e;
    Pc a = *reinterpret_cast<const Pc*>(src);
    if (turned) {
      const float2* w = cs + t * p.P + (INTERLEAVED ? g * (V / 2) : g * V);
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int k = 0; k < V; k += 2) {
          const float2 q = w[k >> 1];
          const float x = to_f32(a.e[k]), y = to_f32(a.e[k + 1]);
          a.e[k] = from_f32<T>(x * q.x - y * q.y);
          a.e[k + 1] = from_f32<T>(y * q.x + x * q.y);
        }
      } else {
        Pc c = *reinterpret_cast<const Pc*>(src + p.P);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float2 q = w[k];
          const float x = to_f32(a.e[k]), y = to_f32(c.e[k]);
          a.e[k] = from_f32<T>(x * q.x - y * q.y);
          c.e[k] = from_f32<T>(y * q.x + x * q.y);
        }
        *reinterpret_cast<Pc*>(dst + p.P) = c;
      }
    }
    *reinterpret_cast<Pc*>(dst) = a;
  }
}

template <typename T, int V>
void launch_v(const RotaryParams& p, bool interleaved, size_t lds, hipStream_t s) {
  if (!interleaved) rotary_kernel<T, V, false><<<grid_of(p.blocks), dim3(256), lds, s>>>(p);
  else if constexpr (V > 1) rotary_kernel<T, V, true><<<grid_of(p.blocks), dim3(256), lds, s>>>(p);
}

template <typename T>
void launch(const RotaryParams& p, int V, bool interleaved, size_t lds, hipStream_t s) {
  if (V * sizeof(T) == 16) return launch_v<T, 16 / sizeof(T)>(p, interleaved, lds, s);
  if constexpr (sizeof(T) == 2) {
    if (V == 4) return launch_v<T, 4>(p, interleaved, lds, s);
  }
  if (V == 2) return launch_v<T, 2>(p, interleaved, lds, s);
  launch_v<T, 1>(p, interleaved, lds, s);
}

}  // namespace

extern "C" int sa_rotary_axes(const void* x, int dtype, int B, int T, int H, int D, const int64_t* x_strides, const void* positions,
                              int pos_type, const int64_t* pos_strides, int n_axes, const int* sections, double theta, int shared_ladder,
                              int interleaved, int inverse, void* y, sa_stream_t stream) {
  SA_REQUIRE(B >= 0 && T >= 0 && H >= 1 && D >= 2 && D % 2 == 0, "sa_rotary_axes: bad shape B=%d T=%d H=%d D=%d", B, T, H, D);
  SA_REQUIRE(H <= 4096 && D <= 4096, "sa_rotary_axes: at most 4096 heads of 4096 values");
  SA_REQUIRE(dtype == SA_F32 || dtype == SA_F16 || dtype == SA_BF16, "sa_rotary_axes: bad dtype %d", dtype);
  SA_REQUIRE(pos_type == SA_POS_I32 || pos_type == SA_POS_I64 || pos_type == SA_POS_F32, "sa_rotary_axes: bad position type %d", pos_type);
  SA_REQUIRE(n_axes >= 1 && n_axes <= MAX_AXES, "sa_rotary_axes: 1 to %d axes", MAX_AXES);
  SA_REQUIRE(theta > 0 && theta < 1e30, "sa_rotary_axes: theta must be positive and finite");
  SA_REQUIRE(x_strides && pos_strides && sections, "sa_rotary_axes: null address of strides or sections");
  int P = 0;
  for (int a = 0; a < n_axes; ++a) {
    SA_REQUIRE(sections[a] >= 0 && sections[a] <= MAX_PAIRS, "sa_rotary_axes: bad section %d", sections[a]);
    P += sections[a];
  }
  SA_REQUIRE(P >= 1 && P <= MAX_PAIRS && 2 * P <= D, "sa_rotary_axes: %d pairs in heads of %d (1 to %d, two values each)", P, D, MAX_PAIRS);
  if (B == 0 || T == 0) return SA_OK;
  SA_REQUIRE(x && positions && y, "sa_rotary_axes: null address");
  RotaryParams p;
  p.x = x;
  p.y = y;
  p.pos = positions;
  p.pos_type = pos_type;
  p.xb = x_strides[0];
  p.xt = x_strides[1];
  p.xh = x_strides[2];
  p.pb = pos_strides[0];
  p.pt = pos_strides[1];
  p.pa = pos_strides[2];
  p.T = T;
  p.H = H;
  p.D = D;
  p.P = P;
  p.sign = inverse ? -1.0f : 1.0f;
  int j = 0;
  for (int a = 0; a < n_axes; ++a)
    for (int i = 0; i < sections[a]; ++i, ++j) {
      p.freq[j] = pow(theta, -(shared_ladder ? (double)j / P : (double)i / sections[a])) / 6.283185307179586476925286766559;
      p.axis[j] = (uint8_t)a;
    }
  // the widest piece that the head's parts, the strides and both addresses are multiples of
  const int size = dtype == SA_F32 ? 4 : 2;
  int V = 16 / size;
  auto fits = [&](int v) {
    if ((interleaved ? 2 * P : P) % v || D % v) return false;
    if (((uintptr_t)x | (uintptr_t)y) % (uintptr_t)(v * size)) return false;
    return !((B > 1 && p.xb % v) || (T > 1 && p.xt % v) || (H > 1 && p.xh % v));
  };
  while (V > 1 && !fits(V)) V >>= 1;
  SA_REQUIRE(!interleaved || V > 1, "sa_rotary_axes: interleaved pairs need even strides and an address of whole pairs");
  p.rot = (interleaved ? 2 * P : P) / V;
  p.G = p.rot + (D - 2 * P) / V;
  // tokens of a workgroup: enough values to make the angles cheap, few enough for four workgroups a CU
  const int64_t tokens = (int64_t)B * T;
  int tok = (int)((tokens + 1023) / 1024);
  tok = tok < 1 ? 1 : tok > 16 ? 16 : tok;
  while (tok > 1 && tok * P > 2048) tok >>= 1;
  p.tok = tok;
  p.tiles = (uint32_t)((T + tok - 1) / tok);
  const uint64_t blocks = (uint64_t)p.tiles * B;
  SA_REQUIRE(blocks < (1ull << 31), "sa_rotary_axes: too many tokens");
  p.div_tiles = fast_div(p.tiles);
  p.div_g = fast_div(p.G);
  p.div_h = fast_div(H);
  p.div_p = fast_div(P);
  p.blocks = (uint32_t)blocks;
  const size_t lds = sizeof(float2) * tok * P;
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == SA_F32) launch<float>(p, V, interleaved, lds, s);
  else if (dtype == SA_F16) launch<_Float16>(p, V, interleaved, lds, s);
  else launch<__bf16>(p, V, interleaved, lds, s);
  SA_LAUNCH_CHECK();
  return SA_OK;
}
