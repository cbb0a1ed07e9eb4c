// Pieces that the cross attention kernels (attention.hip, attention_bwd.hip) share.
//
// Layout of the work. All query heads that share a key head are one matrix: row r = t * G + g is token t of the g-th of those heads,
// so a single token of 8 heads on 2 key heads is a tile of 4 rows and shared heads sum their gradients by themselves.
//
// Matrix products are v_mfma_f32_32x32x16 (fp16 / bf16 operands, float32 sums): A [32 x 16] gives lane l the eight k-values
// 8 (l >> 5) .. + 7 of row l & 31, B [16 x 32] the same of column l & 31, and C [32 x 32] holds column l & 31 in lane l, its
// register i being row 8 (i >> 2) + 4 (l >> 5) + (i & 3). Every product here is arranged so that the 32 columns are rows r of the
// softmax (or keys, for the gradients of k and v): one lane then owns one softmax row (shared with lane ^ 32), maxima and sums need one
// exchange, and registers 8s .. 8s + 7 of a C are, rounded to 16 bits, the B operand of the next product -- for the k order
// {4h .. 4h + 3, 8 + 4h .. 8 + 4h + 3}, h = l >> 5. The A operand in that order is two transposed reads from LDS
// (ds_read_b64_tr_b16: 16 lanes read four rows of 16 values and lane i gets column i), so no value of a softmax passes through LDS.
//
// Tiles in LDS are rows of DP 16-bit values (DP = 32, 64 or 128), the 16-byte pieces of a row exchanged against bank conflicts (swizzle
// below). They come by buffer_load ... lds: the exchange is applied to the source offset, and a lane whose key is hidden or whose
// piece lies behind D gets an offset out of range, which writes zeros: what hidden keys hold (NaN, infinities) never enters a product.
#pragma once
#include "sa_common.h"
#include "token_types.h"

#include <algorithm>

namespace sa {

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int TILE = 64;                   // rows of a tile in LDS
constexpr uint32_t OUT_OF_RANGE = 0xFFFFFFF0u;

template <typename E>
struct Mfma;
template <>
struct Mfma<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  __device__ static __forceinline__ f32x16 run(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};
template <>
struct Mfma<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  __device__ static __forceinline__ f32x16 run(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};

template <typename E>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const f32x2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, typename Mfma<E>::v2));
}
// registers 8s .. 8s + 7 of a C as a B operand
template <typename E>
__device__ __forceinline__ s16x8 pack8(const f32x16& c, int s) {
  const u32x4 v = {pack2<E>(c[8 * s], c[8 * s + 1]), pack2<E>(c[8 * s + 2], c[8 * s + 3]), pack2<E>(c[8 * s + 4], c[8 * s + 5]),
                   pack2<E>(c[8 * s + 6], c[8 * s + 7])};
  return __builtin_bit_cast(s16x8, v);
}

// what rounding to 16 bits takes from a value
template <typename E>
__device__ __forceinline__ float rest_of(float v) {
  return v - static_cast<float>(static_cast<E>(v));
}
// and from registers 8s .. 8s + 7 of a C, given what they were rounded to
template <typename E>
__device__ __forceinline__ s16x8 pack8_rest(const f32x16& c, int s, s16x8 rounded) {
  const typename Mfma<E>::v8 r = __builtin_bit_cast(typename Mfma<E>::v8, rounded);
  f32x16 x;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = c[8 * s + e] - static_cast<float>(r[e]);
  return pack8<E>(x, 0);
}

// The larger of two, NaN if one of them is: v_maximum3_f32, two of them in one instruction. (fmaxf would need another for each operand that
// an arithmetic instruction did not write, to quiet a signalling NaN.)
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// the two half-waves' values of the same column
__device__ __forceinline__ float max_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return larger(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Which piece of 16 bytes of its row a piece is exchanged with. LDS serves 256 bytes a cycle, 32 lanes of a transposed read: their four rows
// (64 bytes each) have to fall into different quarters of a 256-byte line, so those of the row's low two bits that do not choose the
// place in the line already (128-byte rows: one, 64-byte rows: both) exchange whole 64 bytes; the third bit parts eight rows read at one
// piece. (16 lanes read an A operand in a cycle, two rows a bank: taking the fourth bit in as well frees that too, but then rows r and
// r + 8 are not a fixed distance apart and the second address costs more registers than the conflicts cost time: backward 425 -> 489 us.)
// Linear: swizzle(a ^ b) = swizzle(a) ^ swizzle(b).
template <int DP>
__device__ __host__ constexpr int swizzle(int row) {
  constexpr int PER_LINE = 128 / DP;
  return (((row & 3) / PER_LINE) << 2) | ((row >> 2) & 1);
}

// one 16-bit [TILE][DP] tile in LDS
template <int DP>
struct Tile {
  static constexpr int ROW = DP * 2, BYTES = TILE * ROW, PIECES = BYTES / 1024;
  // A operand: eight values of k-step ks of row m of a 32-row block at (at_a(m, h) ^ (ks << 5)) + block * 32 * ROW
  __device__ static __forceinline__ int at_a(int m, int h) { return m * ROW + ((h ^ swizzle<DP>(m)) << 4); }
  // transposed read: rows 16 kk + 8 u + 4 h .. + 3, columns of block db at (at_t(lane) ^ (db << 6)) + (16 kk + 8 u) * ROW
  __device__ static __forceinline__ int at_t(int lane) {
    const int row = 4 * (lane >> 5) + ((lane & 15) >> 2), c = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    return row * ROW + ((c ^ swizzle<DP>(row)) << 4) + (lane & 1) * 8;
  }
};

// A wave's transposed result (C registers: 32 columns, N blocks of 32 rows d) times `by` as 32 rows of D values.
// float32, to rows of a workspace: 16 bytes a lane and store.
template <int N>
__device__ __forceinline__ void store_part(float* row, const f32x16 (&acc)[N], int D, int h, float by) {
#pragma unroll
  for (int db = 0; db < N; ++db)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = db * 32 + j * 8 + h * 4;
      if (d < D) *reinterpret_cast<f32x4*>(row + d) = f32x4{acc[db][4 * j] * by, acc[db][4 * j + 1] * by, acc[db][4 * j + 2] * by, acc[db][4 * j + 3] * by};
    }
}
// 16-bit, by way of LDS (32 * ROW bytes of the wave's own): a lane has four values of each eight and its partner in the other half-wave the
// other four, one exchange of two dwords makes 16 bytes of them, and rows are read back whole, so that stores fill lines.
// `row_of(i)`: where row i begins, or NULL. (8-byte stores straight from the registers: 84 us for the gradients of 8 x 8 x 192 x 4096 x
// 64, 16-byte ones 70.)
template <typename E, int DP, int N, typename F>
__device__ __forceinline__ void store_rows(char* lds, const f32x16 (&acc)[N], int lane, int D, float by, F row_of) {
  using T = Tile<DP>;
  const int n = lane & 31, h = lane >> 5;
#pragma unroll
  for (int db = 0; db < N; ++db)
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const f32x16& x = acc[db];
      const int i = 4 * j;
      const auto lo = __builtin_amdgcn_permlane32_swap(pack2<E>(x[i] * by, x[i + 1] * by), pack2<E>(x[i + 4] * by, x[i + 5] * by), false, false);
      const auto hi = __builtin_amdgcn_permlane32_swap(pack2<E>(x[i + 2] * by, x[i + 3] * by), pack2<E>(x[i + 6] * by, x[i + 7] * by), false, false);
      *reinterpret_cast<u32x4*>(lds + n * T::ROW + (((db * 4 + j + h) ^ swizzle<DP>(n)) << 4)) = u32x4{lo[0], hi[0], lo[1], hi[1]};
    }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // of this wave alone
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    const int at = k * 64 + lane, row = at / (DP / 8), c = at & (DP / 8 - 1);
    E* dst = row_of(row);
    if (dst && c * 8 < D) *reinterpret_cast<u32x4*>(dst + c * 8) = *reinterpret_cast<const u32x4*>(lds + row * T::ROW + ((c ^ swizzle<DP>(row)) << 4));
  }
}

__device__ __forceinline__ s16x8 read_a(const char* lds, int off) { return *reinterpret_cast<const s16x8*>(lds + off); }
__device__ __forceinline__ s16x8 read_t(const char* lds, int off, int step) {
  typedef __attribute__((address_space(3))) s16x4* p4;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(lds + off)), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(lds + off + step));
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// every wave's copies have landed, every wave's reads are done
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Which 16 bytes of a tile each lane copies: piece (wave + j NW) of 1 KB holds rows row0 + j STEP. A lane's place in its row is the same
// for every j (swizzle(row) repeats with STEP), but for a single wave on rows of 256 bytes, where odd j differ in one bit.
template <int DP, int NW>
struct Pieces {
  static constexpr int N = (Tile<DP>::PIECES + NW - 1) / NW, STEP = NW * 1024 / Tile<DP>::ROW;
  int row0, c0;
  __device__ __forceinline__ void init(int wave, int lane) {
    const int at = wave * 1024 + lane * 16;
    row0 = at / Tile<DP>::ROW;
    c0 = ((at >> 4) & (DP / 8 - 1)) ^ swizzle<DP>(row0);
  }
  __device__ __forceinline__ int row(int j) const { return row0 + j * STEP; }
  __device__ __forceinline__ int piece(int j) const { return c0 ^ swizzle<DP>(j * STEP); }
  __device__ static __forceinline__ bool any(int wave, int j) { return Tile<DP>::PIECES % NW == 0 || wave + j * NW < Tile<DP>::PIECES; }
};

// Copies of a tile's rows into LDS by NW waves. `rows` is the 64-bit word of the rows that exist (all others become zeros).
template <int DP, int NW>
struct TileCopy {
  Pieces<DP, NW> at;
  uint32_t off[Pieces<DP, NW>::N];  // kept: computing them in every tile costs the forward kernel 5 %
  __device__ __forceinline__ void init(int wave, int lane, int64_t stride_bytes, int D) {
    at.init(wave, lane);
#pragma unroll
    for (int j = 0; j < at.N; ++j) off[j] = at.piece(j) * 8 < D ? at.row(j) * (uint32_t)stride_bytes + at.piece(j) * 16 : OUT_OF_RANGE;
  }
  __device__ __forceinline__ void issue(char* lds, const void* base, uint64_t rows, int wave) const {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7FFFFFFF, 0x00020000);
#pragma unroll
    for (int j = 0; j < at.N; ++j) {
      if (!at.any(wave, j)) break;
      const uint32_t o = rows == ~0ull || ((rows >> at.row(j)) & 1) ? off[j] : OUT_OF_RANGE;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(lds + (wave + j * NW) * 1024), 16, o, 0, 0, 0);
    }
  }
};

// Hides the scores of keys whose bit in `seen` (32 keys of a block) is not set: minus infinity in two instructions a score. Behind a
// branch: the barrier keeps the compiler from doing this in every tile (it would take the select for cheaper than the jump).
__device__ __forceinline__ void hide(f32x16& s, uint32_t seen, int h) {
  __builtin_amdgcn_sched_barrier(0);
  const int w = (int)(seen >> (4 * h));
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int bit = 8 * (i >> 2) + (i & 3);
    const uint32_t keep = (uint32_t)((w << (31 - bit)) >> 31);
    s[i] = __uint_as_float((__float_as_uint(s[i]) & keep) | (0xFF800000u & ~keep));
  }
}

// Which head and which of its `per` pieces of work a workgroup has. Workgroups go round the eight XCDs, each with its own L2: all pieces
// of a head, which read the same keys (rows), go to one XCD, and heads go round the XCDs, so that images with few keys or none, whose
// heads are neighbours, leave no XCD idle. What is left of the heads after whole rounds is cut into eight runs of pieces.
struct Piece {
  uint32_t head, at;
};
__device__ __forceinline__ Piece piece_of(uint32_t block, uint32_t heads, uint32_t per, const FastDiv& div_per) {
  const uint32_t whole = (heads & ~7u) * per, x = block & 7;
  if (block < whole) {
    const uint32_t slot = block >> 3, round = div_by(slot, div_per);
    return {round * 8 + x, slot - round * per};
  }
  const uint32_t n = (heads & 7) * per, q = n >> 3, r = n & 7;
  const uint32_t id = x * q + min(x, r) + ((block - whole) >> 3), head = div_by(id, div_per);
  return {(heads & ~7u) + head, id - head * per};
}

// what forward and backward know of a call
struct AttnShape {
  const void *q, *k, *v;
  int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh;  // strides in elements
  int Tq, Tk, G, Hq, Hkv, D;
  uint32_t R;                                  // rows of a key head: Tq * G
  FastDiv div_g;
  const int32_t* lengths;                      // keys of each batch entry, or NULL
  const uint8_t* mask;                         // [B, Tk], 0 hides a key, or NULL
  int64_t mb, mt;
  float c;                                     // scale * log2(e)
  float scale;
};

// checks a call's shape and fills `a` (attention.hip)
int attention_shape(const char* who, AttnShape* a, const void* q, const void* k, const void* v, int dtype, int B, int Tq, int Tk, int Hq,
                    int Hkv, int D, const int64_t* strides, const int32_t* lengths, const uint8_t* mask, const int64_t* mask_strides, float scale);

}  // namespace sa
