// Cross attention to an encoder's states: out = softmax(scale q k^T over the visible keys) v, rows without a visible key are zero.
// One pass over the keys with a running maximum and sum per row (in 32 bits); the layout of the products is in attention.h:
//     S^T [keys x rows] = k q^T        P^T = exp2(c S^T - m)        O^T [d x rows] += v^T P^T
//
// A wave has 32 rows, a workgroup of one, two or four waves a tile of 64 keys and values in LDS, the next one on its way. At 128 values
// a head two workgroups a CU overlap one's products with the other's exponentials: 2 x 8 heads x 4096 x 16384 bf16 in 523 us = 1.05
// PFLOP/s (a library product of 8192^3: 1.19), matrix pipes busy 0.53 of the time at the 1.85 GHz that the chip holds under that load. At 64
// values the vector units are the limit (32 exponentials of 16 cycles a tile and lane beside 512 cycles of products): 0.70 to 0.77
// PFLOP/s. Where rows are few, waves share the keys (52 queries x 8 heads x 32 on 1024 keys: 6.1 us) or the keys are cut
// into runs: 32 single tokens on 16384 keys x 2 heads x 128 read theirs at 4.7 TB/s.
#include "attention.h"

namespace {

using namespace sa;

struct FwdParams {
  AttnShape a;
  void* out;              // [B, Tq, Hq, D] contiguous
  float* lse;             // [B, Hq, Tq] natural logarithm of the softmax's denominator, or NULL
  void* low;              // like out, what its rounding left, rounded: out + low has twice the bits; or NULL
  float* part;            // splits > 1: [B * Hkv][splits][R][D] of each run of keys, normalised
  float* part_lse;        // and their base-2 logarithms [B * Hkv][splits][R]
  uint32_t blocks, heads, row_tiles, splits;  // heads: B * Hkv; blocks: heads * row_tiles * splits
  FastDiv div_tiles, div_pieces, div_heads;
  int split_keys;         // keys of a run: a multiple of TILE
};

// P is rounded to 16 bits. Its maximum is 2^GROW at most (the running maximum is only followed when it has grown by 2^GROW: most tiles
// then skip the rescaling of O). fp16 moves all of P up by a power of two, so that weights down to 2^-31 of the largest are held.
template <typename E>
struct Range {
  static constexpr float LIFT = 0.0f;
};
template <>
struct Range<_Float16> {
  static constexpr float LIFT = 7.0f;
};
constexpr float GROW = 8.0f;

// A sum of zero has two causes: no visible key (the row is zeros), or visible keys that all score -inf (it is NaN: their softmax is
// undefined). The logarithm of the first is -inf and of the second the lowest finite number, which no run of a finite score goes below.
constexpr float LOWEST = -3.4028234663852886e38f;
__device__ __forceinline__ float of_sum(float sum, float log, float value) {
  return sum != 0.0f ? value : log == LOWEST ? __builtin_nanf("") : 0.0f;
}
__device__ __forceinline__ float lse_of_sum(float sum, float log) {
  return sum != 0.0f ? (log + __log2f(sum)) * LN2 : log == LOWEST ? __builtin_nanf("") : -INFINITY;
}

// LOW: weights are multiplied in two terms, rounded and what that left, and `low` is written. For gradients over few keys: rowsum(do * out)
// has to cancel against w^T (do v^T) there, and the roundings of w and out alone made dq and dk over 3 keys 2.2 times as inexact as
// their own rounding (600 keys: 1.5 times; from 4096 on it no longer shows). What counts are visible keys: FEW by the length, or, under
// a mask, the first FEW of each run, since they may all lie in one (a share of FEW each is 4 to 15 % faster where runs are long, 125 us instead of 140
// for 8 x 8 heads x 192 x 16384 x 64, but then 2000 visible keys that lie together are 1.36 times as far off); further ones are multiplied once.
constexpr int FEW = 2048;

// KW: waves along the keys, each with the same 32 rows, a run of keys and tiles of its own, so that they need no barrier before their sums meet
// in LDS: for few rows on few keys, where a second launch would join the runs otherwise.
template <typename E, int DB, int NW, bool LOW, int KW>
__global__ __launch_bounds__(NW * KW * 64, 2) void attention_kernel(const FwdParams p) {
  static_assert(NW == 1 || KW == 1, "");
  constexpr int DP = DB == 3 ? 128 : DB * 32, KS = DB * 2;
  using T = Tile<DP>;
  extern __shared__ __align__(1024) char lds_all[];  // [KW][2 stages][k tile, v tile]
  const AttnShape& a = p.a;
  const int id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = KW > 1 ? 0 : id, part = KW > 1 ? id : 0;
  const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
  char* lds = lds_all + part * 4 * T::BYTES;
  const uint32_t block = workgroup();
  if (block >= p.blocks) return;
  const Piece piece = piece_of(block, p.heads, p.row_tiles * p.splits, p.div_pieces);
  const uint32_t bh = piece.head, split = div_by(piece.at, p.div_tiles), tile = piece.at - split * p.row_tiles;
  const uint32_t b = div_by(bh, p.div_heads), hk = bh - b * a.Hkv;

  const uint32_t row = tile * (NW * 32) + wave * 32 + n;
  const bool real = row < a.R;
  const uint32_t rr = real ? row : a.R - 1, t = div_by(rr, a.div_g), g = rr - t * a.G;
  s16x8 q[KS];
  {
    const E* src = static_cast<const E*>(a.q) + (int64_t)b * a.qb + (int64_t)t * a.qt + (int64_t)(hk * a.G + g) * a.qh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = ks * 16 + h * 8;
      q[ks] = d < a.D ? *reinterpret_cast<const s16x8*>(src + d) : s16x8{};
    }
  }
  int length = a.Tk;
  if (a.lengths) length = min(max(a.lengths[b], 0), a.Tk);
  const int first = (int)(split * KW + part) * p.split_keys, end = min(first + p.split_keys, length);
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

  f32x16 o[DB] = {};
  int few = length <= FEW ? 0x7FFFFFFF : mask ? FEW : 0;  // LOW: visible keys still to be multiplied twice
  float m = -INFINITY, l = 0.0f, shift = -Range<E>::LIFT;  // shift = c m - LIFT, of a maximum that is not -inf
  // A tile is copied while the one before is multiplied; the mask's bytes come one tile earlier still. (Three stages: slower by 5 to 15 %
  // at every head size, and workgroups of eight waves gain nothing either.)
  uint64_t seen = 0, any = 0;
  uint8_t next_mask = 1;
  if (tiles) {
    seen = seen_of(0, load_mask(0));
    copy(0, seen);
    next_mask = load_mask(1);
  }
  for (int i = 0; i < tiles; ++i) {
    if constexpr (KW > 1) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the tiles are this wave's alone
    else tile_barrier();
    const uint64_t now = seen;
    if (i + 1 < tiles) {
      seen = seen_of(i + 1, next_mask);
      copy(i + 1, seen);
      next_mask = load_mask(i + 2);
    }
    if (now == 0) continue;
    any |= now;
    const char* kt = lds + (i & 1) * 2 * T::BYTES;
    const char* vt = kt + T::BYTES;
    f32x16 s0 = {}, s1 = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s0 = Mfma<E>::run(read_a(kt, oa[ks]), q[ks], s0);
      s1 = Mfma<E>::run(read_a(kt, oa[ks] + 32 * T::ROW), q[ks], s1);
    }
    if (now != ~0ull) {
      hide(s0, (uint32_t)now, h);
      hide(s1, (uint32_t)(now >> 32), h);
    }
    float top = larger(s0[0], s1[0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) top = larger(larger(top, s0[i]), s1[i]);
    top = max_halves(top);
    if (__any((top - m) * a.c > GROW)) {
      const float grown = larger(m, top), at = grown == -INFINITY ? 0.0f : grown;
      const float keep = __builtin_amdgcn_exp2f((m - at) * a.c);
      m = grown;
      shift = at * a.c - Range<E>::LIFT;
      l *= keep;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= keep;
    }
    float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s0[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s0[i], a.c, -shift));
      s1[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s1[i], a.c, -shift));
      l0 += s0[i];
      l1 += s1[i];
    }
    l += l0 + l1;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const f32x16& s = kk < 2 ? s0 : s1;
      const s16x8 w = pack8<E>(s, kk & 1);
      s16x8 v[DB];
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        v[db] = read_t(vt, ot[db] + kk * 16 * T::ROW, 8 * T::ROW);
        o[db] = Mfma<E>::run(v[db], w, o[db]);
      }
      if (LOW && few > 0) {
        const s16x8 rest = pack8_rest<E>(s, kk & 1, w);
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] = Mfma<E>::run(v[db], rest, o[db]);
      }
    }
    if (LOW) few -= __popcll(now);
  }

  l = sum_halves(l);
  if (l == 0.0f) shift = any ? LOWEST : -INFINITY;
  if constexpr (KW > 1) {
    constexpr int STATS = DB * 4 * 1024;
    if (part) {
#pragma unroll
      for (int j = 0; j < DB * 4; ++j)
        *reinterpret_cast<f32x4*>(lds + (j * 64 + lane) * 16) = f32x4{o[j >> 2][4 * (j & 3)], o[j >> 2][4 * (j & 3) + 1], o[j >> 2][4 * (j & 3) + 2], o[j >> 2][4 * (j & 3) + 3]};
      reinterpret_cast<float*>(lds + STATS)[lane] = shift;
      reinterpret_cast<float*>(lds + STATS)[64 + lane] = l;
    }
    __syncthreads();
    if (part) return;
    float shifts[KW], sums[KW], top = shift;
    shifts[0] = shift;
    sums[0] = l;
#pragma unroll
    for (int w = 1; w < KW; ++w) {
      const float* stats = reinterpret_cast<const float*>(lds + w * 4 * T::BYTES + STATS);
      shifts[w] = stats[lane];
      sums[w] = stats[64 + lane];
      top = larger(top, shifts[w]);
    }
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const float by = sums[w] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(shifts[w] - top);  // a run without weight: nothing
      l += sums[w] * by;
#pragma unroll
      for (int j = 0; j < DB * 4; ++j) {
        if (w == 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j >> 2][4 * (j & 3) + e] *= by;
        } else {
          const f32x4 x = *reinterpret_cast<const f32x4*>(lds + w * 4 * T::BYTES + (j * 64 + lane) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j >> 2][4 * (j & 3) + e] += x[e] * by;
        }
      }
    }
    shift = top;
  }
  if (p.splits > 1) {
    if (!real) return;
    const int64_t at = ((int64_t)bh * p.splits + split) * a.R + row;
    if (h == 0) p.part_lse[at] = l == 0.0f ? shift : shift + __log2f(l);
    store_part(p.part + at * a.D, o, a.D, h, l == 0.0f ? 0.0f : 1.0f / l);
    return;
  }
  const float inv = of_sum(l, shift, 1.0f / l);
  if (p.lse && real && h == 0) p.lse[((int64_t)b * a.Hq + hk * a.G + g) * a.Tq + t] = lse_of_sum(l, shift);
  if constexpr (KW == 1) tile_barrier();  // the last tile has been read
  auto row_of = [&](void* base) {
    return [=](int i) -> E* {
      const uint32_t r = row - n + i, t = div_by(r, a.div_g), g = r - t * a.G;
      return r < a.R ? static_cast<E*>(base) + (((int64_t)b * a.Tq + t) * a.Hq + hk * a.G + g) * a.D : nullptr;
    };
  };
  store_rows<E, DP>(lds + wave * 32 * T::ROW, o, lane, a.D, inv, row_of(p.out));
  if constexpr (LOW) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[db][e] = rest_of<E>(o[db][e] * inv);
    store_rows<E, DP>(lds + wave * 32 * T::ROW, o, lane, a.D, 1.0f, row_of(p.low));
  }
}

// Joins the runs of keys: out = sum_s 2^(lse_s - max) part_s / sum_s 2^(lse_s - max). A row has 16 lanes of 8 values and `groups` of
// them: group j takes runs j, j + groups, ..., four loads of both kinds in flight, and the groups' sums meet in LDS. (One group that
// walks all 32 runs of a single token: 14 us of latency where the attention itself takes 82.)
template <typename E>
__global__ __launch_bounds__(256) void attention_join_kernel(const FwdParams p, FastDiv div_rows, uint32_t groups_log2, uint32_t rows) {
  __shared__ float sums[256][10];
  const AttnShape& a = p.a;
  const uint32_t groups = 1u << groups_log2, lane = threadIdx.x & 15, unit = threadIdx.x >> 4, group = unit & (groups - 1);
  const uint32_t br = workgroup() * (16 >> groups_log2) + (unit >> groups_log2), d = lane * 8;
  const bool real = br < rows && d < (uint32_t)a.D;
  const uint32_t bh = div_by(min(br, rows - 1), div_rows), row = min(br, rows - 1) - bh * a.R;
  const float* lse = p.part_lse + (int64_t)bh * p.splits * a.R + row;
  const float* part = p.part + ((int64_t)bh * p.splits * a.R + row) * a.D + (real ? d : 0);
  const int64_t step = (int64_t)a.R * a.D;
  float m = -INFINITY, sum = 0.0f, acc[8] = {};
  for (uint32_t s0 = group; s0 < p.splits; s0 += 4 * groups) {
    float l[4];
    f32x4 x[4], y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t s = min(s0 + k * groups, p.splits - 1);
      l[k] = lse[(int64_t)s * a.R];
      x[k] = *reinterpret_cast<const f32x4*>(part + s * step);
      y[k] = *reinterpret_cast<const f32x4*>(part + s * step + 4);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (s0 + k * groups >= p.splits || l[k] == -INFINITY) continue;  // a run without a visible key
      const float top = larger(m, l[k]), keep = __builtin_amdgcn_exp2f(m - top), w = __builtin_amdgcn_exp2f(l[k] - top);
      m = top;
      sum = sum * keep + w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[e] = acc[e] * keep + w * x[k][e];
        acc[4 + e] = acc[4 + e] * keep + w * y[k][e];
      }
    }
  }
  if (groups > 1) {
    float* mine = sums[threadIdx.x];
    mine[0] = m;
    mine[1] = sum;
#pragma unroll
    for (int e = 0; e < 8; ++e) mine[2 + e] = acc[e];
    __syncthreads();
    if (group) return;
    for (uint32_t g = 1; g < groups; ++g) {
      const float* other = sums[threadIdx.x + 16 * g];
      const float top = larger(m, other[0]);
      if (other[1] == 0.0f) continue;
      const float keep = __builtin_amdgcn_exp2f(m - top), w = __builtin_amdgcn_exp2f(other[0] - top);
      m = top;
      sum = sum * keep + w * other[1];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = acc[e] * keep + w * other[2 + e];
    }
  }
  if (!real) return;
  const uint32_t b = div_by(bh, p.div_heads), hk = bh - b * a.Hkv, t = div_by(row, a.div_g), g = row - t * a.G;
  if (m == LOWEST) sum = 0.0f;
  const float inv = of_sum(sum, m, 1.0f / sum);
  if (p.lse && d == 0) p.lse[((int64_t)b * a.Hq + hk * a.G + g) * a.Tq + t] = lse_of_sum(sum, m);
  const int64_t at = (((int64_t)b * a.Tq + t) * a.Hq + hk * a.G + g) * a.D + d;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] *= inv;
  *reinterpret_cast<u32x4*>(static_cast<E*>(p.out) + at) = u32x4{pack2<E>(acc[0], acc[1]), pack2<E>(acc[2], acc[3]), pack2<E>(acc[4], acc[5]), pack2<E>(acc[6], acc[7])};
  if (!p.low) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = rest_of<E>(acc[e]);
  *reinterpret_cast<u32x4*>(static_cast<E*>(p.low) + at) = u32x4{pack2<E>(acc[0], acc[1]), pack2<E>(acc[2], acc[3]), pack2<E>(acc[4], acc[5]), pack2<E>(acc[6], acc[7])};
}

// How a call is cut: waves of a workgroup (32 rows each, or along the keys) and runs of keys.
struct Cut {
  int waves, key_waves;
  uint32_t row_tiles, splits;
  int split_keys;
};
Cut cut(int B, int Tq, int Tk, int Hq, int Hkv, int D) {
  const uint64_t R = (uint64_t)Tq * (Hq / Hkv);
  Cut c;
  c.waves = R <= 32 ? 1 : R <= 64 ? 2 : 4;
  c.row_tiles = (uint32_t)((R + c.waves * 32 - 1) / (c.waves * 32));
  const uint64_t blocks = (uint64_t)c.row_tiles * B * Hkv;
  const uint64_t want = 2048 / c.waves;  // eight waves a CU
  const uint32_t key_tiles = (uint32_t)(((int64_t)Tk + TILE - 1) / TILE);
  uint64_t splits = blocks ? want / blocks : 1;
  const uint64_t most = key_tiles / 4;   // a run of at least four tiles
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  if (c.waves == 4 && blocks > want) {
    // More workgroups than places: the last round may be nearly empty. Runs even it out and cost a float32 result written and read
    // for each; in microseconds, a tile at two workgroups a CU 0.45 + 0.005 D, 4 bytes a value twice at 4 TB/s, 6 for the launch that joins.
    // (17 heads x 4096 x 8192 x 128, 544 workgroups: 402 us whole, 337 in the runs chosen here; 1024 of them, 16 heads x 4096 x 16384 x 128, stay whole.)
    double best = 0;
    for (uint64_t s = 1; s <= 8 && (s == 1 || s <= most); ++s) {
      const double rounds = (double)((blocks * s + want - 1) / want), run = (double)((key_tiles + s - 1) / s);
      const double cost = rounds * run * (0.45 + 0.005 * D) + (s > 1 ? 6 + (double)s * R * B * Hkv * D * 8 / 4e6 : 0);
      if (s == 1 || cost < best) {
        best = cost;
        splits = s;
      }
    }
  }
  // Few rows on few keys: four waves of a workgroup along the keys and one launch, as long as every workgroup has a place (64 KB of
  // tiles at up to 32 values a head, 128 KB above) and the longer runs cost less than a second launch and the runs' results, written
  // and read: in microseconds, a tile of a lone wave 0.45 + 0.01 D, 1.5 for the launch, 4 bytes a value twice at 4 TB/s. (52 queries x 8 heads x 32 on
  // 640 keys: 5.3 us, 8.5 in two launches; on 1024: 6.1 and 7.9; on 2048, in two launches: 8.4, 9.0 in one. 2 x 416 x 8 x 32 on 1536: 7.8 and 13.1.)
  c.key_waves = 1;
  const uint64_t narrow = (R + 31) / 32 * B * Hkv, along = (key_tiles + 3) / 4;
  if (key_tiles >= 3 && D <= 64 && narrow <= (D <= 32 ? 512 : 256)) {
    const double longer = (double)along - (double)((key_tiles + splits - 1) / splits);
    if (splits == 1 || longer * (0.45 + 0.01 * D) <= 1.5 + (double)splits * R * B * Hkv * D * 8 / 4e6) {
      c.waves = 1;
      c.key_waves = 4;
      c.row_tiles = (uint32_t)((R + 31) / 32);
      c.splits = 1;
      c.split_keys = (int)along * TILE;
      return c;
    }
  }
  const uint32_t per = key_tiles ? (uint32_t)((key_tiles + splits - 1) / splits) : 1;
  c.split_keys = (int)per * TILE;
  c.splits = key_tiles ? (key_tiles + per - 1) / per : 1;
  return c;
}

template <typename E, int DB, bool LOW>
void launch_low(const FwdParams& p, const Cut& c, hipStream_t s) {
  constexpr size_t lds = 4 * Tile<DB == 3 ? 128 : DB * 32>::BYTES;
  if constexpr (DB <= 2) {
    if (c.key_waves > 1) {
      const auto kernel = attention_kernel<E, DB, 1, LOW, 4>;
      if (4 * lds > 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)(4 * lds));
      kernel<<<grid_of(p.blocks), dim3(256), 4 * lds, s>>>(p);
      return;
    }
  }
  if (c.waves == 1) attention_kernel<E, DB, 1, LOW, 1><<<grid_of(p.blocks), dim3(64), lds, s>>>(p);
  else if (c.waves == 2) attention_kernel<E, DB, 2, LOW, 1><<<grid_of(p.blocks), dim3(128), lds, s>>>(p);
  else attention_kernel<E, DB, 4, LOW, 1><<<grid_of(p.blocks), dim3(256), lds, s>>>(p);
}

template <typename E, int DB>
void launch(const FwdParams& p, const Cut& c, hipStream_t s) {
  if (p.low) launch_low<E, DB, true>(p, c, s);
  else launch_low<E, DB, false>(p, c, s);
}

template <typename E>
void launch_e(const FwdParams& p, const Cut& c, hipStream_t s) {
  const int db = (p.a.D + 31) / 32;
  if (db == 1) launch<E, 1>(p, c, s);
  else if (db == 2) launch<E, 2>(p, c, s);
  else if (db == 3) launch<E, 3>(p, c, s);
  else launch<E, 4>(p, c, s);
  if (p.splits > 1) {
    const uint32_t rows = p.heads * p.a.R;
    uint32_t log2 = 0;
    while (log2 < 4 && (4u << log2) < p.splits) ++log2;  // four runs a group
    const uint32_t per = 16 >> log2;
    attention_join_kernel<E><<<grid_of((rows + per - 1) / per), dim3(256), 0, s>>>(p, fast_div(p.a.R), log2, rows);
  }
}

}  // namespace

namespace sa {

int attention_shape(const char* who, AttnShape* a, const void* q, const void* k, const void* v, int dtype, int B, int Tq, int Tk, int Hq,
                    int Hkv, int D, const int64_t* strides, const int32_t* lengths, const uint8_t* mask, const int64_t* mask_strides, float scale) {
  SA_REQUIRE(B >= 0 && Tq >= 0 && Tk >= 0 && Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0, "%s: bad shape B=%d Tq=%d Tk=%d Hq=%d Hkv=%d", who, B, Tq, Tk, Hq, Hkv);
  SA_REQUIRE(D >= 8 && D <= 128 && D % 8 == 0, "%s: head size %d (a multiple of 8, at most 128)", who, D);
  SA_REQUIRE(dtype == SA_F16 || dtype == SA_BF16, "%s: 16-bit types only (%d)", who, dtype);
  SA_REQUIRE(scale > 0 && scale <= 1e30f, "%s: scale must be positive and finite", who);
  SA_REQUIRE(Tk <= (1 << 30) && (uint64_t)Tq * (Hq / Hkv) < (1ull << 31) - 1024 && (uint64_t)B * Hq < (1ull << 31), "%s: too many rows", who);
  SA_REQUIRE(strides, "%s: null address of strides", who);
  for (int i = 0; i < 9; ++i) SA_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0, "%s: strides are multiples of 8 elements", who);
  for (int i = 3; i < 9; i += 3) SA_REQUIRE(strides[i + 1] < (1ll << 23), "%s: token strides of keys and values are below 2^23 elements", who);
  SA_REQUIRE(!mask || mask_strides, "%s: a mask needs its strides", who);
  const uint64_t rows = (uint64_t)B * Tq, keys = (uint64_t)B * Tk;
  SA_REQUIRE((q || !rows) && ((k && v) || !keys), "%s: null address", who);
  SA_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) == 0, "%s: addresses are multiples of 16", who);
  a->q = q;
  a->k = k;
  a->v = v;
  a->qb = strides[0]; a->qt = strides[1]; a->qh = strides[2];
  a->kb = strides[3]; a->kt = strides[4]; a->kh = strides[5];
  a->vb = strides[6]; a->vt = strides[7]; a->vh = strides[8];
  a->Tq = Tq;
  a->Tk = Tk;
  a->Hq = Hq;
  a->Hkv = Hkv;
  a->G = Hq / Hkv;
  a->D = D;
  a->R = (uint32_t)Tq * a->G;
  a->div_g = fast_div(a->G);
  a->lengths = lengths;
  a->mask = mask;
  a->mb = mask ? mask_strides[0] : 0;
  a->mt = mask ? mask_strides[1] : 0;
  a->scale = scale;
  a->c = scale * LOG2E;
  return SA_OK;
}

}  // namespace sa

extern "C" size_t sa_cross_attention_workspace(int B, int Tq, int Tk, int Hq, int Hkv, int D) {
  if (B < 1 || Tq < 1 || Tk < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || D < 1) return 0;
  const Cut c = cut(B, Tq, Tk, Hq, Hkv, D);
  return c.splits > 1 ? (size_t)B * Hq * Tq * c.splits * (D + 1) * sizeof(float) : 0;
}

extern "C" int sa_cross_attention(const void* q, const void* k, const void* v, int dtype, int B, int Tq, int Tk, int Hq, int Hkv, int D,
                                  const int64_t* strides, const int32_t* key_lengths, const uint8_t* key_mask, const int64_t* mask_strides,
                                  float scale, void* out, float* lse, void* out_low, void* workspace, size_t workspace_bytes, sa_stream_t stream) {
  FwdParams p;
  if (int rc = attention_shape("sa_cross_attention", &p.a, q, k, v, dtype, B, Tq, Tk, Hq, Hkv, D, strides, key_lengths, key_mask, mask_strides, scale)) return rc;
  if (B == 0 || Tq == 0) return SA_OK;
  SA_REQUIRE(out, "sa_cross_attention: null address");
  SA_REQUIRE((((uintptr_t)out | (uintptr_t)out_low | (uintptr_t)workspace) & 15) == 0, "sa_cross_attention: addresses are multiples of 16");
  const Cut c = cut(B, Tq, Tk, Hq, Hkv, D);
  const uint64_t blocks = (uint64_t)c.row_tiles * c.splits * B * Hkv;
  SA_REQUIRE(blocks < (1ull << 31) && (uint64_t)B * Hq * Tq < (1ull << 31) - 1024, "sa_cross_attention: too many rows");
  if (c.splits > 1 && (!workspace || workspace_bytes < sa_cross_attention_workspace(B, Tq, Tk, Hq, Hkv, D)))
    return fail(SA_ERR_WORKSPACE, "sa_cross_attention: workspace of %zu bytes is too small", workspace_bytes);
  p.out = out;
  p.lse = lse;
  p.low = out_low;
  p.part = static_cast<float*>(workspace);
  p.part_lse = p.part + (size_t)B * Hq * Tq * c.splits * D;
  p.blocks = (uint32_t)blocks;
  p.row_tiles = c.row_tiles;
  p.splits = c.splits;
  p.split_keys = c.split_keys;
  p.div_tiles = fast_div(c.row_tiles);
  p.heads = (uint32_t)B * Hkv;
  p.div_pieces = fast_div(c.row_tiles * c.splits);
  p.div_heads = fast_div(Hkv);
  if (dtype == SA_F16) launch_e<_Float16>(p, c, (hipStream_t)stream);
  else launch_e<__bf16>(p, c, (hipStream_t)stream);
  SA_LAUNCH_CHECK();
  return SA_OK;
}
