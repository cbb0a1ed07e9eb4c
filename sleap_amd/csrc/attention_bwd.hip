// Gradients of cross attention. With w = softmax (from the stored logarithms of its denominators, not kept), dw = do v^T,
// ds = w (dw - rowsum(do * out)):
//     dv = w^T do        dk = scale ds^T q        dq = scale ds k
// Two sides, both without atomics, so that sums have one order: one whose waves own keys and walk the rows (dk, dv: four products), one
// whose waves own rows and walk the keys (dq: three). One that does both would save two of the seven products and need
// atomics or a float32 dq read and written once per tile of keys. Shared heads are rows like any others (attention.h): dk and dv sum
// over them by themselves. Where one side owns little, runs of what it walks go to several workgroups, and a last
// kernel adds their float32 sums in order. A side whose gradients nobody asks for (a frozen map, given queries) is not run: forward and
// backward of 4096 x 8192 x 8 x 128 take 574 us, for dq alone 335, for dk and dv alone 387.
//
// Measured: 8 heads x 4096 x 8192 x 128 bf16 430 us for both sides = 1.12 PFLOP/s of seven products (the rate of a large library product);
// 8 x 8 heads x 192 x 4096 x 64 68 us, 0.66 PFLOP/s: three tiles of rows a workgroup, so that what it reads first and writes last weighs.
#include "attention.h"

namespace {

using namespace sa;

struct Side {
  uint32_t blocks, tiles, splits;  // workgroups; of them along the owned side, along the walked side
  int run;                         // rows (keys) of a run: a multiple of TILE
  FastDiv div_tiles, div_pieces;
};

struct BwdParams {
  AttnShape a;
  const void *out, *low, *dout;  // low: what the rounding of out left, or NULL
  int64_t ob, ot, oh;       // strides of dout
  const float* lse;         // [B, Hq, Tq]
  float *lse2, *delta;      // [B * Hkv][R]: log2 of the denominator less LIFT; rowsum(do * out)
  void *dq, *dk, *dv;       // contiguous
  float *part_dq, *part_dk, *part_dv;  // [splits] of the whole gradient each, or NULL
  Side kv, rows;            // who owns keys and walks rows (dk, dv); who owns rows and walks keys (dq)
  uint32_t heads;           // B * Hkv
  FastDiv div_heads, div_hq;
};

// w is rounded to 16 bits for w^T do, ds for the other two. bf16 has the range of float32. fp16 has not: w moves up by 2^14 (held down to
// 2^-38), and ds by a power of two of each column that follows its largest value so far (Range16 below).
template <typename E>
struct Lift {
  static constexpr float LOG = 0.0f, BACK = 1.0f;
};
template <>
struct Lift<_Float16> {
  static constexpr float LOG = 14.0f, BACK = 1.0f / 16384.0f;
};

// power of two that a column's ds is multiplied with before it is rounded; never grows, so sums are rescaled a few times at most
template <typename E>
struct Range16 {
  __device__ __forceinline__ void follow(f32x16&, f32x16*, int) {}
  __device__ __forceinline__ float back() const { return 1.0f; }
};
template <>
struct Range16<_Float16> {
  float up = 0x1p100f;
  __device__ __forceinline__ void follow(f32x16& ds, f32x16* acc, int n) {
    float top = fabsf(ds[0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) top = larger(top, fabsf(ds[i]));
    top = max_halves(top);
    if (__any(top * up > 0x1p15f)) {
      const int e = __builtin_amdgcn_frexp_expf(top);  // top < 2^e
      const float to = top * up > 0x1p15f ? __builtin_amdgcn_ldexpf(1.0f, min(13 - e, 100)) : up;
      const float r = to / up;
      up = to;
      for (int db = 0; db < n; ++db) acc[db] *= r;
    }
    ds *= up;
  }
  __device__ __forceinline__ float back() const { return 1.0f / up; }
};

// TWICE: w and ds are multiplied in two terms, rounded and what that left. Their rounding alone makes gradients 1.41 times as inexact as
// their own rounding does where sums are long, up to 2.8 times where a few weights make them up, and dq of heads of up to 32 values 1.5 to 1.7
// times at any size. So dq of such heads is multiplied twice always (2 x 2048 x 4096 x 8 x 16 bf16, both sides: 99 us with neither, 109 with dq,
// 135 with all three), and all three are where it costs next to nothing: up to FREE multiply-adds a product, 30 us of kernel at most
// beside the 40 to 75 that torch's engine takes on the host (3 x 417 x 1531 x 8 on 2 x 40 fp16, 0.9 FREE: 25.8 us of kernel, 22.6 without). 4096 x 8192 x 8
// x 128 bf16 would take 629 us instead of 442.
constexpr double FREE = 1024.0 * 1024 * 1024;

template <typename E>
__global__ __launch_bounds__(256) void attention_stats_kernel(const BwdParams p, uint32_t total) {
  const AttnShape& a = p.a;
  const uint32_t i = workgroup() * 16 + (threadIdx.x >> 4);  // 16 lanes of 8 values a row
  const uint32_t ic = min(i, total - 1);
  const uint32_t bt = div_by(ic, p.div_hq), hh = ic - bt * a.Hq;
  const uint32_t b = bt / a.Tq, t = bt - b * a.Tq;
  const int d = (threadIdx.x & 15) * 8;
  float sum = 0.0f;
  if (d < a.D) {
    union {
      s16x8 v;
      E e[8];
    } x, y;
    x.v = *reinterpret_cast<const s16x8*>(static_cast<const E*>(p.out) + (int64_t)ic * a.D + d);
    y.v = *reinterpret_cast<const s16x8*>(static_cast<const E*>(p.dout) + (int64_t)b * p.ob + (int64_t)t * p.ot + (int64_t)hh * p.oh + d);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += to_f32(x.e[e]) * to_f32(y.e[e]);
    if (p.low) {
      x.v = *reinterpret_cast<const s16x8*>(static_cast<const E*>(p.low) + (int64_t)ic * a.D + d);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += to_f32(x.e[e]) * to_f32(y.e[e]);
    }
  }
#pragma unroll
  for (int w = 8; w; w >>= 1) sum += __shfl_xor(sum, w);
  if (i < total && (threadIdx.x & 15) == 0) {
    const float l = p.lse[((int64_t)b * a.Hq + hh) * a.Tq + t];
    const int64_t at = ((int64_t)b * a.Hkv + hh / a.G) * a.R + (int64_t)t * a.G + hh % a.G;
    p.lse2[at] = l == -INFINITY ? INFINITY : l * LOG2E - Lift<E>::LOG;
    p.delta[at] = sum;
  }
}

// rows r0 .. r0 + 63 of q and dout into two tiles
template <int DP, int NW, typename E>
__device__ __forceinline__ void copy_rows(char* lds, const Pieces<DP, NW>& at, const BwdParams& p, const E* q, const E* dout, uint32_t r0, uint32_t end, int wave) {
  const AttnShape& a = p.a;
  const uint32_t t0 = __builtin_amdgcn_readfirstlane(div_by(r0, a.div_g));
  const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc(const_cast<E*>(q + (int64_t)t0 * a.qt), 0, 0x7FFFFFFF, 0x00020000);
  const __amdgpu_buffer_rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc(const_cast<E*>(dout + (int64_t)t0 * p.ot), 0, 0x7FFFFFFF, 0x00020000);
#pragma unroll
  for (int j = 0; j < at.N; ++j) {
    if (!at.any(wave, j)) break;
    const int c = at.piece(j);
    const uint32_t r = r0 + at.row(j), t = div_by(r, a.div_g), g = r - t * a.G;
    const bool in = r < end && c * 8 < a.D;
    const uint32_t oq = in ? 2 * ((t - t0) * (uint32_t)a.qt + g * (uint32_t)a.qh) + c * 16 : OUT_OF_RANGE;
    const uint32_t oo = in ? 2 * ((t - t0) * (uint32_t)p.ot + g * (uint32_t)p.oh) + c * 16 : OUT_OF_RANGE;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rq, (lds_ptr)(lds + (wave + j * NW) * 1024), 16, oq, 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(ro, (lds_ptr)(lds + Tile<DP>::BYTES + (wave + j * NW) * 1024), 16, oo, 0, 0, 0);
  }
}

// dk, dv: a wave owns 32 keys (k and v in registers) and walks rows in tiles of 64
template <typename E, int DB, int NW, bool TWICE>
__device__ __forceinline__ void keys_side(const BwdParams& p, uint32_t block, char* lds) {
  constexpr int DP = DB == 3 ? 128 : DB * 32, KS = DB * 2;
  using T = Tile<DP>;
  constexpr int STAGE = 2 * T::BYTES + 2 * TILE * 4;  // q, dout, lse2, delta
  // When do v^T is multiplied: beside the exponentials of w, or, where the registers do not hold both (fp16 at 128 values, which also
  // follows the range of ds), after w has been used. 8 x 4096 x 8192 x 128: fp16 588 us early, 526 late; bf16 514 early, 528 late.
  constexpr bool LATE = DB == 4 && Lift<E>::LOG != 0.0f;
  const AttnShape& a = p.a;
  const Side& side = p.kv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
  const Piece piece = piece_of(block, p.heads, side.tiles * side.splits, side.div_pieces);
  const uint32_t bh = piece.head, split = div_by(piece.at, side.div_tiles), tile = piece.at - split * side.tiles;
  const uint32_t b = div_by(bh, p.div_heads), hk = bh - b * a.Hkv;

  int length = a.Tk;
  if (a.lengths) length = min(max(a.lengths[b], 0), a.Tk);
  const int key0 = (int)tile * (NW * 32), key = key0 + wave * 32 + n;
  bool seen = key < length;
  if (seen && a.mask) seen = a.mask[(int64_t)b * a.mb + (int64_t)key * a.mt] != 0;
  s16x8 kf[KS], vf[KS];
  {
    const E* ks_ = static_cast<const E*>(a.k) + (int64_t)b * a.kb + (int64_t)hk * a.kh + (int64_t)key * a.kt;
    const E* vs_ = static_cast<const E*>(a.v) + (int64_t)b * a.vb + (int64_t)hk * a.vh + (int64_t)key * a.vt;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = ks * 16 + h * 8;
      const bool in = seen && d < a.D;
      kf[ks] = in ? *reinterpret_cast<const s16x8*>(ks_ + d) : s16x8{};
      vf[ks] = in ? *reinterpret_cast<const s16x8*>(vs_ + d) : s16x8{};
    }
  }
  const uint32_t first = split * (uint32_t)side.run, end = min(first + (uint32_t)side.run, a.R);
  const int tiles = key0 < length && first < end ? (int)((end - first + TILE - 1) / TILE) : 0;  // no visible key in this tile: nothing to walk
  const E* qbase = static_cast<const E*>(a.q) + (int64_t)b * a.qb + (int64_t)(hk * a.G) * a.qh;
  const E* obase = static_cast<const E*>(p.dout) + (int64_t)b * p.ob + (int64_t)(hk * a.G) * p.oh;
  Pieces<DP, NW> pieces;
  pieces.init(wave, lane);
  auto copy = [&](int i) {
    char* s = lds + (i & 1) * STAGE;
    const uint32_t r0 = first + (uint32_t)i * TILE;
    copy_rows<DP, NW, E>(s, pieces, p, qbase, obase, r0, end, wave);
    if (wave == 0) {
      const int64_t at = (int64_t)bh * a.R + r0;
      const uint32_t o = r0 + lane < end ? lane * 4 : OUT_OF_RANGE;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(p.lse2 + at, 0, 0x7FFFFFFF, 0x00020000), (lds_ptr)(s + 2 * T::BYTES), 4, o, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(p.delta + at, 0, 0x7FFFFFFF, 0x00020000), (lds_ptr)(s + 2 * T::BYTES + TILE * 4), 4, o, 0, 0, 0);
    }
  };
  const int aa = T::at_a(n, h), at_ = T::at_t(lane);
  f32x16 dk[DB] = {}, dv[DB] = {};
  Range16<E> range;
  if (tiles) copy(0);
  for (int i = 0; i < tiles; ++i) {
    tile_barrier();
    if (i + 1 < tiles) copy(i + 1);
    // one block of 32 rows after the other, not unrolled: its scores are out of the registers before the next one's come in, which
    // leaves room for a second wave on each SIMD
#pragma unroll 1
    for (int blk = 0; blk < 2; ++blk) {
      const char* qt = lds + (i & 1) * STAGE + blk * 32 * T::ROW;
      const char* dt = qt + T::BYTES;
      const float* stat = reinterpret_cast<const float*>(lds + (i & 1) * STAGE + 2 * T::BYTES) + 4 * h + blk * 32;
      f32x16 s = {}, dp = {};
      auto multiply_dp = [&] {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) dp = Mfma<E>::run(read_a(dt, aa ^ (ks << 5)), vf[ks], dp);
      };
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = Mfma<E>::run(read_a(qt, aa ^ (ks << 5)), kf[ks], s);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 l = *reinterpret_cast<const f32x4*>(stat + 8 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * j + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * j + e], a.c, -l[e]));
      }
      if (!LATE) multiply_dp();
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const s16x8 w = pack8<E>(s, s2);
        s16x8 rest;
        if constexpr (TWICE) rest = pack8_rest<E>(s, s2, w);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const s16x8 f = read_t(dt, (at_ ^ (db << 6)) + s2 * 16 * T::ROW, 8 * T::ROW);
          dv[db] = Mfma<E>::run(f, w, dv[db]);
          if constexpr (TWICE) dv[db] = Mfma<E>::run(f, rest, dv[db]);
        }
      }
      if (LATE) multiply_dp();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 l = *reinterpret_cast<const f32x4*>(stat + TILE + 8 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * j + e] = s[4 * j + e] * (dp[4 * j + e] - l[e]);
      }
      range.follow(dp, dk, DB);
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const s16x8 w = pack8<E>(dp, s2);
        s16x8 rest;
        if constexpr (TWICE) rest = pack8_rest<E>(dp, s2, w);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const s16x8 f = read_t(qt, (at_ ^ (db << 6)) + s2 * 16 * T::ROW, 8 * T::ROW);
          dk[db] = Mfma<E>::run(f, w, dk[db]);
          if constexpr (TWICE) dk[db] = Mfma<E>::run(f, rest, dk[db]);
        }
      }
    }
  }
  if (!seen) {
#pragma unroll
    for (int db = 0; db < DB; ++db) dk[db] = dv[db] = f32x16{};
  }
  const float by_k = a.scale * Lift<E>::BACK * range.back(), by_v = Lift<E>::BACK;
  auto place = [&](int64_t k) { return (((int64_t)b * a.Tk + k) * a.Hkv + hk) * a.D; };
  if (p.part_dk) {
    if (key >= a.Tk) return;
    const int64_t at = split * ((int64_t)p.heads * a.Tk * a.D) + place(key);
    store_part(p.part_dk + at, dk, a.D, h, by_k);
    store_part(p.part_dv + at, dv, a.D, h, by_v);
    return;
  }
  tile_barrier();  // the last tile has been read
  auto row_of = [&](void* base) {
    return [=](int i) -> E* { return key - n + i < a.Tk ? static_cast<E*>(base) + place(key - n + i) : nullptr; };
  };
  char* own = lds + wave * 32 * T::ROW;
  store_rows<E, DP>(own, dk, lane, a.D, by_k, row_of(p.dk));
  store_rows<E, DP>(own, dv, lane, a.D, by_v, row_of(p.dv));
}

// dq: a wave owns 32 rows (q and dout in registers) and walks keys in tiles of 64
template <typename E, int DB, int NW, bool TWICE>
__device__ __forceinline__ void rows_side(const BwdParams& p, uint32_t block, char* lds) {
  constexpr int DP = DB == 3 ? 128 : DB * 32, KS = DB * 2;
  using T = Tile<DP>;
  const AttnShape& a = p.a;
  const Side& side = p.rows;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
  const Piece piece = piece_of(block, p.heads, side.tiles * side.splits, side.div_pieces);
  const uint32_t bh = piece.head, split = div_by(piece.at, side.div_tiles), tile = piece.at - split * side.tiles;
  const uint32_t b = div_by(bh, p.div_heads), hk = bh - b * a.Hkv;

  const uint32_t row = tile * (NW * 32) + wave * 32 + n;
  const bool real = row < a.R;
  const uint32_t rr = real ? row : a.R - 1, t = div_by(rr, a.div_g), g = rr - t * a.G;
  s16x8 qf[KS], df[KS];
  {
    const E* q = static_cast<const E*>(a.q) + (int64_t)b * a.qb + (int64_t)t * a.qt + (int64_t)(hk * a.G + g) * a.qh;
    const E* o = static_cast<const E*>(p.dout) + (int64_t)b * p.ob + (int64_t)t * p.ot + (int64_t)(hk * a.G + g) * p.oh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = ks * 16 + h * 8;
      qf[ks] = d < a.D ? *reinterpret_cast<const s16x8*>(q + d) : s16x8{};
      df[ks] = d < a.D ? *reinterpret_cast<const s16x8*>(o + d) : s16x8{};
    }
  }
  const float lse2 = p.lse2[(int64_t)bh * a.R + rr], delta = p.delta[(int64_t)bh * a.R + rr];
  int length = a.Tk;
  if (a.lengths) length = min(max(a.lengths[b], 0), a.Tk);
  const int first = (int)split * side.run, end = min(first + side.run, length);
  const int tiles = end > first ? (end - first + TILE - 1) / TILE : 0;
  const E* kbase = static_cast<const E*>(a.k) + (int64_t)b * a.kb + (int64_t)hk * a.kh;
  const E* vbase = static_cast<const E*>(a.v) + (int64_t)b * a.vb + (int64_t)hk * a.vh;
  const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.mb : nullptr;
  TileCopy<DP, NW> ck, cv;
  ck.init(wave, lane, a.kt * 2, a.D);
  cv.init(wave, lane, a.vt * 2, a.D);
  auto load_mask = [&](int i) -> uint8_t {
    const int key = first + i * TILE + lane;
    return mask && key < end ? mask[(int64_t)key * a.mt] : 1;
  };
  auto seen_of = [&](int i, uint8_t m) { return __ballot(first + i * TILE + lane < end && m); };
  auto copy = [&](int i, uint64_t seen) {
    char* s = lds + (i & 1) * 2 * T::BYTES;
    const int64_t key = first + (int64_t)i * TILE;
    ck.issue(s, kbase + key * a.kt, seen, wave);
    cv.issue(s + T::BYTES, vbase + key * a.vt, seen, wave);
  };
  int oa[KS], ot[DB];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) oa[ks] = T::at_a(n, h) ^ (ks << 5);
#pragma unroll
  for (int db = 0; db < DB; ++db) ot[db] = T::at_t(lane) ^ (db << 6);

  f32x16 dq[DB] = {};
  Range16<E> range;
  uint64_t seen = 0;
  uint8_t next_mask = 1;
  if (tiles) {
    seen = seen_of(0, load_mask(0));
    copy(0, seen);
    next_mask = load_mask(1);
  }
  for (int i = 0; i < tiles; ++i) {
    tile_barrier();
    const uint64_t now = seen;
    if (i + 1 < tiles) {
      seen = seen_of(i + 1, next_mask);
      copy(i + 1, seen);
      next_mask = load_mask(i + 2);
    }
    if (now == 0) continue;
    const char* kt = lds + (i & 1) * 2 * T::BYTES;
    const char* vt = kt + T::BYTES;
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = Mfma<E>::run(read_a(kt, oa[ks] + blk * 32 * T::ROW), qf[ks], s);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) dp = Mfma<E>::run(read_a(vt, oa[ks] + blk * 32 * T::ROW), df[ks], dp);
      if (now != ~0ull) hide(s, (uint32_t)(now >> (32 * blk)), h);
#pragma unroll
      for (int e = 0; e < 16; ++e) dp[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], a.c, -lse2)) * (dp[e] - delta);
      range.follow(dp, dq, DB);
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const s16x8 w = pack8<E>(dp, s2);
        s16x8 rest;
        if constexpr (TWICE) rest = pack8_rest<E>(dp, s2, w);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const s16x8 f = read_t(kt, ot[db] + (blk * 2 + s2) * 16 * T::ROW, 8 * T::ROW);
          dq[db] = Mfma<E>::run(f, w, dq[db]);
          if constexpr (TWICE) dq[db] = Mfma<E>::run(f, rest, dq[db]);
        }
      }
    }
  }
  const float by = a.scale * Lift<E>::BACK * range.back();
  if (p.part_dq) {
    if (real) store_part(p.part_dq + split * ((int64_t)p.heads * a.R * a.D) + (((int64_t)b * a.Tq + t) * a.Hq + hk * a.G + g) * a.D, dq, a.D, h, by);
    return;
  }
  tile_barrier();  // the last tile has been read
  store_rows<E, DP>(lds + wave * 32 * T::ROW, dq, lane, a.D, by, [&](int i) -> E* {
    const uint32_t r = row - n + i, t = div_by(r, a.div_g), g = r - t * a.G;
    return r < a.R ? static_cast<E*>(p.dq) + (((int64_t)b * a.Tq + t) * a.Hq + hk * a.G + g) * a.D : nullptr;
  });
}

// Both sides in one launch: neither needs the other, and one's last workgroups fill up with the other's. Rows come first, their
// walks are the longer ones where keys are many.
template <typename E, int DB, int NW, bool TWICE>
__global__ __launch_bounds__(NW * 64, 2) void attention_bwd_kernel(const BwdParams p) {
  extern __shared__ __align__(1024) char lds[];
  const uint32_t block = workgroup();
  if (block < p.rows.blocks) rows_side<E, DB, NW, TWICE || DB == 1>(p, block, lds);
  else if (block < p.rows.blocks + p.kv.blocks) keys_side<E, DB, NW, TWICE>(p, block - p.rows.blocks, lds);
}

// Adds the runs' gradients, in their order, of up to three tensors; a thread has 8 values of one.
struct AddParams {
  const float* part[3];
  void* dst[3];
  int64_t n[3];
  int splits[3];
  uint32_t first[3];  // first workgroup of each
  uint32_t blocks;
};
template <typename E>
__global__ __launch_bounds__(256) void attention_add_kernel(const AddParams p) {
  const uint32_t block = workgroup();
  if (block >= p.blocks) return;
  const int k = block >= p.first[2] ? 2 : block >= p.first[1] ? 1 : 0;
  const int64_t i = ((int64_t)(block - p.first[k]) * 256 + threadIdx.x) * 8, n = p.n[k];
  if (i >= n) return;
  f32x4 x = {}, y = {};
#pragma unroll 4
  for (int s = 0; s < p.splits[k]; ++s) {
    const f32x4* src = reinterpret_cast<const f32x4*>(p.part[k] + s * n + i);
    x += src[0];
    y += src[1];
  }
  *reinterpret_cast<u32x4*>(static_cast<E*>(p.dst[k]) + i) = u32x4{pack2<E>(x[0], x[1]), pack2<E>(x[2], x[3]), pack2<E>(y[0], y[1]), pack2<E>(y[2], y[3])};
}

// How a side is cut: what it owns among waves of 32, what it walks among `splits` runs.
Side cut(int waves, uint64_t heads, uint64_t own, uint64_t walk, double splits_) {
  Side c;
  c.tiles = (uint32_t)((own + waves * 32 - 1) / (waves * 32));
  const uint64_t walked = (walk + TILE - 1) / TILE, most = std::max<uint64_t>(1, walked / 4);  // a run of at least four tiles
  const uint64_t splits = std::max<uint64_t>(1, std::min<uint64_t>(most, (uint64_t)(splits_ + 0.5)));
  const uint64_t per = std::max<uint64_t>(1, (walked + splits - 1) / splits);
  c.run = (int)(per * TILE);
  c.splits = (uint32_t)std::max<uint64_t>(1, (walked + per - 1) / per);
  c.blocks = (uint32_t)std::min<uint64_t>(c.tiles * heads * c.splits, 0xFFFFFFFFu);
  c.div_tiles = fast_div(std::max(1u, c.tiles));
  c.div_pieces = fast_div(std::max(1u, c.tiles * c.splits));
  return c;
}

struct Layout {
  int waves;
  Side kv = {}, rows = {};  // one whose gradients are not asked for has no workgroups
  size_t stats, dq, dkv;  // floats of each part of the workspace
  size_t total() const { return 2 * stats + dq + 2 * dkv; }
};
Layout layout(int B, int Tq, int Tk, int Hq, int Hkv, int D, bool want_q, bool want_kv) {
  Layout l;
  const uint64_t R = (uint64_t)Tq * (Hq / Hkv), heads = (uint64_t)B * Hkv, most = std::max<uint64_t>(want_q ? R : 0, want_kv ? Tk : 0);
  l.waves = most <= 32 ? 1 : most <= 64 ? 2 : 4;
  // Work of a workgroup of each side in products of a tile, and what falls to one of the eight-waves-a-CU places. Fewer workgroups than
  // places: runs of that length. More: of half of it, so that the last ones are short (8 x 4096 x 8192 x 128: 424 us, runs of the
  // whole length 464; 3 x 2 x 1668 x 1531 x 40: 20 us, runs of half of it 24).
  auto tiles = [](uint64_t n, uint64_t of) { return (n + of - 1) / of; };
  const double places = 2048.0 / l.waves, nk = want_kv ? (double)(heads * tiles(Tk, l.waves * 32)) : 0, nr = want_q ? (double)(heads * tiles(R, l.waves * 32)) : 0;
  const double wk = 4.0 * tiles(R, TILE), wr = 3.0 * tiles(Tk, TILE);
  const double each = (nk * wk + nr * wr) / places * (nk + nr <= places ? 1.0 : 0.5);
  if (want_kv) l.kv = cut(l.waves, heads, Tk, R, each > 0 ? wk / each : 1);
  if (want_q) l.rows = cut(l.waves, heads, R, Tk, each > 0 ? wr / each : 1);
  l.stats = ((size_t)B * Hq * Tq + 3) / 4 * 4;
  l.dq = l.rows.splits > 1 ? (size_t)l.rows.splits * B * Hq * Tq * D : 0;
  l.dkv = l.kv.splits > 1 ? (size_t)l.kv.splits * B * Hkv * Tk * D : 0;
  return l;
}

template <typename E, int DB, bool TWICE>
void launch_sides(const BwdParams& p, int waves, hipStream_t s) {
  constexpr size_t lds = 2 * (2 * Tile<DB == 3 ? 128 : DB * 32>::BYTES + 2 * TILE * 4);  // the keys' side, which has the rows' numbers beside its tiles
  auto go = [&](auto kernel) {
    if (lds > 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    kernel<<<grid_of((uint64_t)p.rows.blocks + p.kv.blocks), dim3(waves * 64), lds, s>>>(p);
  };
  if (waves == 1) go(attention_bwd_kernel<E, DB, 1, TWICE>);
  else if (waves == 2) go(attention_bwd_kernel<E, DB, 2, TWICE>);
  else go(attention_bwd_kernel<E, DB, 4, TWICE>);
}

template <typename E>
int launch(const BwdParams& p, int waves, hipStream_t s) {
  const AttnShape& a = p.a;
  const int db = (a.D + 31) / 32;
  if (a.R) {
    const uint32_t rows = p.heads * a.R;
    attention_stats_kernel<E><<<grid_of(((uint64_t)rows + 15) / 16), dim3(256), 0, s>>>(p, rows);
    SA_LAUNCH_CHECK();
  }
  if (p.rows.blocks + p.kv.blocks == 0) return SA_OK;
  auto sides = [&](auto twice) {
    if (db == 1) launch_sides<E, 1, twice>(p, waves, s);
    else if (db == 2) launch_sides<E, 2, twice>(p, waves, s);
    else if (db == 3) launch_sides<E, 3, twice>(p, waves, s);
    else launch_sides<E, 4, twice>(p, waves, s);
  };
  if ((double)p.heads * a.R * a.Tk * (db * 32) <= FREE) sides(std::true_type{});
  else sides(std::false_type{});
  SA_LAUNCH_CHECK();
  AddParams add = {};
  uint32_t blocks = 0;
  auto sum = [&](int k, const float* part, void* dst, uint64_t tokens, uint32_t splits) {
    add.first[k] = blocks;
    if (!part) return;
    add.part[k] = part;
    add.dst[k] = dst;
    add.n[k] = (int64_t)(p.heads * tokens * a.D);
    add.splits[k] = (int)splits;
    blocks += (uint32_t)((add.n[k] / 8 + 255) / 256);
  };
  sum(0, p.part_dk, p.dk, a.Tk, p.kv.splits);
  sum(1, p.part_dv, p.dv, a.Tk, p.kv.splits);
  sum(2, p.part_dq, p.dq, a.R, p.rows.splits);
  if (blocks) {
    add.blocks = blocks;
    attention_add_kernel<E><<<grid_of(blocks), dim3(256), 0, s>>>(add);
    SA_LAUNCH_CHECK();
  }
  return SA_OK;
}

}  // namespace

extern "C" size_t sa_cross_attention_backward_workspace(int B, int Tq, int Tk, int Hq, int Hkv, int D) {
  if (B < 1 || Tq < 0 || Tk < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || D < 1) return 0;
  size_t most = 0;  // whichever gradients are asked for: a side alone is cut into other runs
  for (int want = 1; want <= 3; ++want) most = std::max(most, layout(B, Tq, Tk, Hq, Hkv, D, want & 1, want & 2).total());
  return most * sizeof(float);
}

extern "C" int sa_cross_attention_backward(const void* q, const void* k, const void* v, int dtype, int B, int Tq, int Tk, int Hq, int Hkv,
                                           int D, const int64_t* strides, const int32_t* key_lengths, const uint8_t* key_mask,
                                           const int64_t* mask_strides, float scale, const void* out, const void* out_low, const float* lse, const void* dout,
                                           const int64_t* dout_strides, void* dq, void* dk, void* dv, void* workspace,
                                           size_t workspace_bytes, sa_stream_t stream) {
  const char* who = "sa_cross_attention_backward";
  BwdParams p;
  if (int rc = attention_shape(who, &p.a, q, k, v, dtype, B, Tq, Tk, Hq, Hkv, D, strides, key_lengths, key_mask, mask_strides, scale)) return rc;
  if (B == 0 || (Tq == 0 && Tk == 0)) return SA_OK;
  SA_REQUIRE((Tq == 0 || (out && lse && dout)) && (Tk == 0 || !dk == !dv), "%s: null address", who);
  if (!dq && !dk) return SA_OK;
  SA_REQUIRE((((uintptr_t)out | (uintptr_t)out_low | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)workspace) & 15) == 0, "%s: addresses are multiples of 16", who);
  SA_REQUIRE(dout_strides, "%s: null address of strides", who);
  for (int i = 0; i < 3; ++i) SA_REQUIRE(dout_strides[i] >= 0 && dout_strides[i] % 8 == 0, "%s: strides are multiples of 8 elements", who);
  const int64_t G = Hq / Hkv, far = 1ll << 30;
  auto near = [&](const int64_t* s) { return s[1] < far && s[2] < far && TILE * s[1] + G * s[2] < far; };
  SA_REQUIRE(near(strides) && near(dout_strides),
             "%s: 64 tokens and the heads on one key head span less than 2^30 elements of q and of dout", who);
  const Layout l = layout(B, Tq, Tk, Hq, Hkv, D, dq, dk);
  SA_REQUIRE((uint64_t)l.kv.blocks + l.rows.blocks < (1ull << 31) && (uint64_t)B * Hq * Tq < (1ull << 31) - 1024 && (uint64_t)B * Hkv < (1ull << 31), "%s: too many rows", who);
  if (l.total() && (!workspace || workspace_bytes < l.total() * sizeof(float))) return fail(SA_ERR_WORKSPACE, "%s: workspace of %zu bytes is too small", who, workspace_bytes);
  p.out = out;
  p.low = out_low;
  p.dout = dout;
  p.ob = dout_strides[0];
  p.ot = dout_strides[1];
  p.oh = dout_strides[2];
  p.lse = lse;
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  float* w = static_cast<float*>(workspace);
  p.lse2 = w;
  p.delta = w + l.stats;
  p.part_dq = l.dq ? w + 2 * l.stats : nullptr;
  p.part_dk = l.dkv ? w + 2 * l.stats + l.dq : nullptr;
  p.part_dv = l.dkv ? w + 2 * l.stats + l.dq + l.dkv : nullptr;
  p.kv = l.kv;
  p.rows = l.rows;
  p.heads = (uint32_t)B * Hkv;
  p.div_heads = fast_div(Hkv);
  p.div_hq = fast_div(Hq);
  return dtype == SA_F16 ? launch<_Float16>(p, l.waves, (hipStream_t)stream) : launch<__bf16>(p, l.waves, (hipStream_t)stream);
}
