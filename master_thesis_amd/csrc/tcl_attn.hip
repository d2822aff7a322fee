// Attention of a target's tokens over chosen blocks of reference keys: tcl_block_attention_fwd / _bwd.
//
//   out_q = sum_n softmax_n(scale <q, k_n>) v_n   over the visible keys n of the blocks chosen for q's group
//   (0, and lse = -inf, where nothing is visible).
//
// All products run on the matrix pipe, 16 x 16 with 32 k-elements per step (one v_mfma_f32_16x16x32 for 16-bit operands, eight
// v_mfma_f32_16x16x4_f32 for fp32): lane l holds row (column) l % 16 of an operand and 8 k-elements of the quarter l / 16; the result
// has column l % 16 and rows 4 (l / 16) .. + 3 (32 x 32 with 16 k-elements where a wave's tile allows: half the instructions, and one
// softmax row per lane instead of two).  The order of the k-elements is free as long as both operands share it, and that is what keeps the probabilities in registers: S^T = K Q^T leaves a lane 4 + 4 probabilities of ITS query (two
// 16-key tiles), which are, as they are, the second operand of O^T = V^T P^T once V^T is read in the same key order: for 16-bit
// types with the transposing LDS read, for fp32 element by element.  So every tensor has ONE image in LDS, rows as they lie in
// memory, for contractions over channels and over tokens alike.
//
// Tiles go from memory to LDS without passing registers (16-byte pieces, global_load_lds), one tile ahead of the products: an image
// is a run of 1 KiB pieces that a wave's 64 lanes fill in lane order, so the order of the 16-byte chunks within a row is turned
// (an exclusive or with bits of the row) on the SOURCE side, such that both ways of reading hit every bank once.  Rows that are not to be
// seen are read from 16 zero bytes instead: what lies in a hole never reaches a product.
//
// Statistics (running maximum, sum, lse, rowsum(dout o out)) and all accumulators are fp32.  16-bit inputs: the probabilities and the
// score gradients are rounded to the inputs' type as operands of the second product (half a step of it relative to each
// term, the size of the rounding of the result itself; fp16, whose steps are absolute below 2^-14, after scaling: PScale, GradRange);
// nothing else is rounded before the end.
#include "tcl_common.h"
#include <math.h>

namespace tcl {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8), aligned(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Vec8;
template <> struct Vec8<float> { typedef f32x8 type; };
template <> struct Vec8<__bf16> { typedef bf16x8 type; };
template <> struct Vec8<_Float16> { typedef f16x8 type; };
template <typename T> struct Vec4 { typedef T type __attribute__((ext_vector_type(4))); };

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// 16 k-elements, 4 per lane (element 4 (l / 16) + e)
__device__ __forceinline__ f32x4 mma4(bf16x4 a, bf16x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma4(f16x4 a, f16x4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma4(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// the same 32 x 32 with 16 k-elements: lane l holds row (column) l % 32 and 8 k-elements of the half l / 32, and gets column l % 32, rows
// 8 j + 4 (l / 32) .. + 3
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// c + a b, where c is a long sum: fp32 products, whose k-elements go into an accumulator one after another, are summed for themselves first and added whole.
// A serial sum of n random terms is off by about 0.4 sqrt(n / 2) 2^-24 of its size: outputs over 16,384 keys by 37 2^-24, 9 so (forward 101 -> 102 us, query
// gradient 133 -> 133 for 16,384 keys of 64 channels; 128 channels 178 -> 183 and 274 -> 278).  16-bit results have no use for it.
template <typename F, typename A> __device__ __forceinline__ A mma_whole(F a, F b, A c) { return mma(a, b, c); }
__device__ __forceinline__ f32x4 mma_whole(f32x8 a, f32x8 b, f32x4 c) { return c + mma(a, b, f32x4{0.f, 0.f, 0.f, 0.f}); }
template <typename F> __device__ __forceinline__ f32x4 mma4_whole(F a, F b, f32x4 c) { return mma4(a, b, c); }
__device__ __forceinline__ f32x4 mma4_whole(f32x4 a, f32x4 b, f32x4 c) { return c + mma4(a, b, f32x4{0.f, 0.f, 0.f, 0.f}); }

// The two shapes: S x S products of KS k-elements, AE results per lane.  Result e of a lane in quarter (half) q = lane / S is row
// row(e) + 4 q of the tile.
template <int S> struct Shape;
template <> struct Shape<16> {
  typedef f32x4 acc;
  static constexpr int KS = 32, AE = 4;
  static constexpr int row(int e) { return e; }
};
template <> struct Shape<32> {
  typedef f32x16 acc;
  static constexpr int KS = 16, AE = 16;
  static constexpr int row(int e) { return e / 4 * 8 + e % 4; }
};

constexpr float kNegInf = -__builtin_inff();
constexpr float kPosInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

constexpr int64_t kMaxTop = 2048;         // a group's list in LDS: 8 KB
constexpr int64_t kMaxKeyBlocks = 65536;  // a bit per block in LDS: 8 KB
constexpr int64_t kMaxRows = 1 << 20;     // query rows of one group

struct Str { int64_t b, n, h; };   // element strides of a (B, N, H, D) tensor with dense channels

struct AttnArgs {
  const void *q, *k, *v, *dout;
  const float *vis;
  const int32_t *blocks;
  void *out, *lo, *dq, *dk, *dv;   // lo: what rounding took from out, laid out like it
  float *lse;                      // (B, Hq, Nq), natural logarithm
  float *ref, *weight;             // (B, Hq, Nq): what the backward pass takes the probabilities from, or null: from lse (row_statistics)
  float *delta;                    // (B, Hq, Nq)
  uint32_t *inv;                   // (B, Hkv, nb, words): which groups chose the block
  uint32_t *chosen;                // (B, Hkv, nb): by how many entries, directly behind inv
  int32_t *order;                  // (B, Hkv, nb): the blocks, often chosen ones first
  int64_t plan_words;              // of inv and chosen
  float *part;                     // partial results of split work: of the forward's keys, or [dk, dv][split][item, key head][key][D]
  Str sq, sk, sv, so, sdo, sdq, sdk, sdv;
  int B, Nq, Nk, Hq, Hkv, G, D, S, top, nb, lb, q_block, rows, chunks, splits, words, cap;   // splits: of the forward's keys, or of the rows of the key / value gradients
  float c;                         // scale * log2(e)
  float scale;
  FastDiv by_g, by_rows, by_d4;
};

// LDS image of token rows of DP channels: NCH chunks of 16 bytes per row (a power of two)
template <typename T, int DP> struct Img {
  static constexpr int VE = 16 / sizeof(T);
  static constexpr int NCH = DP / VE <= 4 ? 4 : DP / VE <= 8 ? 8 : DP / VE <= 16 ? 16 : 32;
  static constexpr int RB = NCH * 16;
  // chunk c of row r lies at c ^ swz(r): 16 rows reading one chunk, and 8 rows reading two neighbouring ones, hit different banks
  __device__ __forceinline__ static int swz(int r) {
    if (NCH == 4) return ((r >> 2) & 1) << 1 | ((r >> 3) & 1);
    if (NCH == 8) return ((r >> 1) & 3) << 1 | ((r >> 3) & 1);
    return (r & 7) << 1 | ((r >> 3) & 1);
  }
};

typedef __attribute__((address_space(3))) void *lds_vptr;
typedef const __attribute__((address_space(1))) void *glb_cvptr;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

static __device__ __attribute__((aligned(16))) const uint32_t g_zero_chunk[4] = {0, 0, 0, 0};

__device__ __forceinline__ void dma16(const char *src, char *lds) {   // lds: of the wave's first lane
  __builtin_amdgcn_global_load_lds((glb_cvptr)src, (lds_vptr)lds, 16, 0, 0);
}
// Maxima that hand on a NaN (one instruction for three operands; fmaxf, which does not, takes two for two): a row that sees a NaN is NaN
__device__ __forceinline__ float max2(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// maximum over the lanes that hold the same column of an S x S result: the swaps leave rows (halves) of both halves in both operands
template <int S> __device__ __forceinline__ float column_max(float x) {
  if constexpr (S == 16) {
    const unsigned u = __float_as_uint(x);
    const u32x2 a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = max2(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  const unsigned w = __float_as_uint(x);
  const u32x2 b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return max2(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// Bit `row` + 4 (lane / S) of a uniform mask.  S = 32: as a lane mask that the scalar unit makes, which leaves one vector instruction per
// masked score of three (four bits instead of two would cost the scalar unit more than that: fp32 backward 138 -> 144 us).
template <int S> __device__ __forceinline__ bool key_seen(unsigned part, int row) {
  if constexpr (S == 32) {
    const unsigned lo = (unsigned)((int)(part << (31 - row)) >> 31), hi = (unsigned)((int)(part << (27 - row)) >> 31);
    return __builtin_amdgcn_inverse_ballot_w64((uint64_t)hi << 32 | lo);
  } else return (part >> (threadIdx.x % 64 / 16 * 4 + row)) & 1;
}
// fp16 steps are absolute below 2^-14, so a probability is scaled up as an operand: in the forward, where those of a row are exp2(score - reference), by
// 2^10 (unscaled, the tail of a long row is lost: 131,068 keys with 2^-25.2 of the largest each are 0.4 % of its weight and came out as zeros; scaled,
// each loses 2^-35 of the largest at most), in the backward, where P <= 1, by 2^14.
template <typename T> struct PScale { static constexpr float room = 8.f, fwd = 0.f, up = 1.f, inv = 1.f; };
template <> struct PScale<_Float16> { static constexpr float room = 4.f, fwd = 10.f, up = 0x1p14f, inv = 0x1p-14f; };

// The running maximum need not be the maximum: any reference r with the scores at most `room` above it (in log2 units) keeps exp2(score - r) <= 256
// (fp16: 16, scaled 2^14) far from every type's limits, and it costs no accuracy, since all sums are of floating-point numbers.  So the sums and outputs so
// far are scaled only where a score passes the reference by more (64 tiles of random scores, 32 rows a wave: in 1 or 2 tiles instead of about 45).
// A NaN becomes the reference, and with it the whole row.
template <int S, typename T, typename O> __device__ __forceinline__ void raise_reference(float mx, float &m, float &l, float &lr, O &o) {
  if (__any(!(mx <= m + PScale<T>::room))) {
    const float mn = max2(m, mx), f = __builtin_amdgcn_exp2f(m - (mn == kNegInf ? 0.f : mn));
    m = mn;
    l *= f;
    lr *= f;
#pragma unroll
    for (int d = 0; d < (int)(sizeof(O) / sizeof(o[0])); ++d) o[d] *= f;
  }
}
// c + the sum of rounded probabilities (a training step divides by it what it keeps of the output for rowsum(dout o out): the roundings' errors are then those of
// the values' differences from the output, where over the unrounded sum they are those of the values, which may have a large common part: with values of
// mean 5 and deviation 1 dq was off by twice its own rounding, of mean 50 by 17 times, now by 1.05).  Forward of the training step of 63,600 keys 215 -> 222 us.
__device__ __forceinline__ float add_rounded(float c, bf16x4 p) {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  const pair one = {(__bf16)1.f, (__bf16)1.f};
  c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 0, 1), one, c, false);
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 2, 3), one, c, false);
}
__device__ __forceinline__ float add_rounded(float c, f16x4 p) {
  typedef _Float16 pair __attribute__((ext_vector_type(2)));
  const pair one = {(_Float16)1.f, (_Float16)1.f};
  c = __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 0, 1), one, c, false);
  return __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 2, 3), one, c, false);
}
__device__ __forceinline__ float add_rounded(float c, bf16x8 p) {
  return add_rounded(add_rounded(c, __builtin_shufflevector(p, p, 0, 1, 2, 3)), __builtin_shufflevector(p, p, 4, 5, 6, 7));
}
__device__ __forceinline__ float add_rounded(float c, f16x8 p) {
  return add_rounded(add_rounded(c, __builtin_shufflevector(p, p, 0, 1, 2, 3)), __builtin_shufflevector(p, p, 4, 5, 6, 7));
}
// all but the last N LDS-DMAs of this wave have landed and every LDS read of it has been served; then the workgroup meets
// (by the builtin: a wait in inline assembly is unknown to the compiler, which then waits again, for the tile that is on its way)
template <int N> __device__ __forceinline__ void tile_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | (N >> 4) << 14);   // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// Lanes of one wave exchange values through LDS: the hardware keeps a wave's LDS operations in order, and this tells the compiler to (it costs no instruction)
__device__ __forceinline__ void wave_exchange() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Where the pieces of this thread lie: piece u of an image of ROWS rows is row u * RPU + threadIdx.x / NCH, chunk `ch` of it (the
// same for every u, or one of two in turn where a step is 8 rows)
template <typename T, int DP, int ROWS> struct Pieces {
  typedef Img<T, DP> I;
  static constexpr int RPU = 256 / I::NCH, NU = (ROWS * I::NCH + 255) / 256;
  static constexpr bool whole = ROWS * I::NCH % 256 == 0;
  __device__ __forceinline__ static int row(int u) { return u * RPU + (int)threadIdx.x / I::NCH; }
  __device__ __forceinline__ static int chunk(int u) { return ((int)threadIdx.x % I::NCH) ^ I::swz(row(u)); }
  __device__ __forceinline__ static bool any(int u, int wave) { return whole || u * 256 + wave * 64 < ROWS * I::NCH; }   // wave-uniform
  __device__ __forceinline__ static char *dst(char *img, int u, int wave) { return img + (u * 256 + wave * 64) * 16; }
};

// Chunks beyond the head's channels (a head size that is not a multiple of 32) are zeroed once, by `images` images of ROWS rows, and
// left alone by the loads, whose lanes for them stay idle.
template <typename T, int DP, int ROWS> __device__ __forceinline__ void zero_pads(char *img, int images, int chunks, int wave) {
  typedef Pieces<T, DP, ROWS> P;
  if (chunks == P::I::NCH) return;
  const uint4 zero = {0, 0, 0, 0};
  for (int i = 0; i < images; ++i)
#pragma unroll
    for (int u = 0; u < P::NU; ++u)
      if (P::any(u, wave) && P::chunk(u) >= chunks)
        *reinterpret_cast<uint4 *>(img + (size_t)i * ROWS * P::I::RB + (u * 256 + (int)threadIdx.x) * 16) = zero;
}

// ROWS rows that lie `st` bytes apart, from row `off` of the 64 that `mask` speaks of -> image; rows the mask leaves out are zeros.
// `base`, `st`, `mask`, `off` are uniform: a tile without holes costs no vector instruction but the loads.
template <typename T, int DP, int ROWS> __device__ __forceinline__ void dma_segment(char *img, const char *base, unsigned st, uint64_t mask, int off, int chunks, int wave) {
  typedef Pieces<T, DP, ROWS> P;
  base += (size_t)((unsigned)off * st);
  mask >>= off;
  const uint64_t need = ROWS >= 64 ? ~0ull : (1ull << ROWS) - 1;
  if ((mask & need) == need) {
#pragma unroll
    for (int u = 0; u < P::NU; ++u)
      if (P::any(u, wave) && P::chunk(u) < chunks) dma16(base + ((unsigned)P::row(u) * st + (unsigned)P::chunk(u) * 16), P::dst(img, u, wave));
  } else {
    const char *zero = reinterpret_cast<const char *>(g_zero_chunk);
#pragma unroll
    for (int u = 0; u < P::NU; ++u)
      if (P::any(u, wave) && P::chunk(u) < chunks) {
        const uint32_t half = P::RPU > 32 ? (P::row(u) < 32 ? (uint32_t)mask : (uint32_t)(mask >> 32)) : u * P::RPU < 32 ? (uint32_t)mask : (uint32_t)(mask >> 32);
        const bool in = (half >> (P::row(u) & 31)) & 1;
        const char *p = base + ((unsigned)P::row(u) * st + (unsigned)P::chunk(u) * 16);
        dma16(in ? p : zero, P::dst(img, u, wave));
      }
  }
}

// the 8 k-elements (channels ch .. ch + 7) of a lane for a contraction over channels; row: a multiple of 16 + the lane's column
template <typename T, int DP> __device__ __forceinline__ typename Vec8<T>::type row_frag(const char *img, int row, int ch) {
  typedef Img<T, DP> I;
  const int s = I::swz(row), c = ch / I::VE;
  const char *p = img + row * I::RB;
  if constexpr (sizeof(T) == 2) return *reinterpret_cast<const typename Vec8<T>::type *>(p + ((c ^ s) << 4));
  else {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(p + ((c ^ s) << 4)), b = *reinterpret_cast<const f32x4 *>(p + (((c + 1) ^ s) << 4));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}
// ... for a contraction over tokens, in the order in which a lane holds the results of an S x S product: channel d0 + lane % S, and
//   S = 16: of the 32 tokens from t0, tokens t0 + 4 q .. + 3 and t0 + 16 + 4 q .. + 3
//   S = 32: of the 16 tokens from t0, tokens t0 + 4 q .. + 3 and t0 + 8 + 4 q .. + 3
// with q = lane / S; t0 is a multiple of 16.  col_frag4: the first four alone.
template <typename T, int DP, int S = 16> __device__ __forceinline__ typename Vec4<T>::type col_frag4(const char *img, int d0, int lane) {
  typedef Img<T, DP> I;
  const int q = lane / S, col = lane % 16;
  if constexpr (sizeof(T) == 2) {
    // transposing read: lane 4 r + p of a group of 16 points at row r, elements 4 p .. + 3 of a 4 x 16 block and gets column lane % 16 of it
    const int row = 4 * q + col / 4, p = col % 4, ch = (d0 + (S == 32 ? lane / 16 % 2 * 16 : 0)) / 8 + p / 2;
    return __builtin_bit_cast(typename Vec4<T>::type, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(img + row * I::RB + ((ch ^ I::swz(row)) << 4) + (p % 2) * 8)));
  } else {
    static_assert(S == 16, "fp32 products are 16 x 16");
    f32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = 4 * q + e;
      r[e] = *reinterpret_cast<const float *>(img + row * I::RB + (((d0 / 4 + col / 4) ^ I::swz(row)) << 4) + (col % 4) * 4);
    }
    return r;
  }
}
template <typename T, int DP, int S = 16> __device__ __forceinline__ typename Vec8<T>::type col_frag(const char *img, int t0, int d0, int lane) {
  typedef Img<T, DP> I;
  if constexpr (sizeof(T) == 2) {
    const int q = lane / S, col = lane % 16;
    constexpr int SECOND = S == 16 ? 16 : 8;
    const int row = 4 * q + col / 4, p = col % 4, ch = (d0 + (S == 32 ? lane / 16 % 2 * 16 : 0)) / 8 + p / 2;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(img + (t0 + row) * I::RB + ((ch ^ I::swz(row)) << 4) + (p % 2) * 8));
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(img + (t0 + row + SECOND) * I::RB + ((ch ^ I::swz(row + SECOND)) << 4) + (p % 2) * 8));
    const s16x8 both = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename Vec8<T>::type, both);
  } else {
    const f32x4 x = col_frag4<T, DP, S>(img + t0 * I::RB, d0, lane), y = col_frag4<T, DP, S>(img + (t0 + 16) * I::RB, d0, lane);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// ------------------------------------------------------------------------------------------ the blocks of one group
// blocks[0 .. top) of one group -> list[]: the valid indices, each once (an index outside [0, nb) is no block).  A list that is
// ascending with its invalid entries last, as select_blocks writes it, is taken as it is; any other goes through a bit per block.
// Returns their number.  Called by the whole workgroup.
__device__ __forceinline__ int group_blocks(const int32_t *blocks, int top, int nb, uint32_t *bits, int *list, int *n_out) {
  int good = 1, mine = 0;
  for (int i0 = 0; i0 < top; i0 += 256) {
    const int i = i0 + (int)threadIdx.x;
    const int j = i < top ? blocks[i] : -1, before = i < top && i > 0 ? blocks[i - 1] : -1;
    const bool valid = j >= 0 && j < nb;
    if (valid) {
      good &= i == 0 || (before >= 0 && before < j);
      if (i < min(top, nb)) list[i] = j;
      ++mine;
    }
  }
  if (threadIdx.x == 0) *n_out = 0;
  if (__syncthreads_and(good)) {
    if (mine) atomicAdd(n_out, mine);
    __syncthreads();
    return *n_out;
  }
  const int words = (nb + 31) / 32;
  for (int i = threadIdx.x; i < words; i += 256) bits[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < top; i += 256) {
    const int j = blocks[i];
    if (j >= 0 && j < nb) atomicOr(&bits[j >> 5], 1u << (j & 31));
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    int base = 0;
    for (int w0 = 0; w0 < words; w0 += 64) {
      const int w = w0 + (int)threadIdx.x;
      uint32_t m = w < words ? bits[w] : 0;
      int incl = __popc(m);
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(incl, o, 64);
        if ((int)threadIdx.x >= o) incl += t;
      }
      int at = base + incl - __popc(m);
      base += __shfl(incl, 63, 64);
      while (m) {
        list[at++] = w * 32 + __builtin_ctz(m);
        m &= m - 1;
      }
    }
    if (threadIdx.x == 0) *n_out = base;
  }
  __syncthreads();
  return *n_out;
}

// ------------------------------------------------------------------------------------------ forward
// The keys of a group pass in segments of 64 (a block is one or two of them).
struct Segment {
  int key0;                                                      // first key, or -1: none
  uint64_t mask;                                                 // bit r: key0 + r exists and is seen
  __device__ __forceinline__ uint64_t there(int nk) const {      // bit r: key0 + r exists (a block of 128 may end in its first segment)
    return key0 < 0 || key0 >= nk ? 0ull : key0 + 64 <= nk ? ~0ull : (1ull << (nk - key0)) - 1;
  }
};
// The raw parts of a segment are asked for a tile before they are needed.  The load is unconditional (clamped): a load behind a
// condition would be waited for where the paths meet, and with it the tile that is on its way.
struct SegmentLoad { int key0; float seen; };
static __device__ const float g_one = 1.f;
struct KeySource {
  const int *list;
  const float *vis;
  int vis_step, n, lb, nk;                                       // segments, log2 of the block, keys
  __device__ __forceinline__ SegmentLoad load(int i) const {     // n > 0
    const int per = lb - 6, j = min(i, n - 1);
    const int key0 = __builtin_amdgcn_readfirstlane((list[j >> per] << lb) + ((j & ((1 << per) - 1)) << 6));
    const int key = min(key0 + (int)(threadIdx.x & 63), nk - 1);
    return SegmentLoad{i < n ? key0 : -1, *(const __attribute__((address_space(1))) float *)(vis + (int64_t)key * vis_step)};
  }
  // segment 0, which has to be waited for: without a mask nothing is loaded
  __device__ __forceinline__ Segment first() const {
    if (vis_step) return finish(load(0));
    Segment s{__builtin_amdgcn_readfirstlane(list[0] << lb), 0};
    s.mask = s.there(nk);
    return s;
  }
  __device__ __forceinline__ Segment finish(const SegmentLoad &l) const {
    return Segment{l.key0, l.key0 < 0 ? 0ull : __ballot(l.seen > 0.5f && l.key0 + (int)(threadIdx.x & 63) < nk)};
  }
};

// of a sum: nothing seen gives zero; NaN stays NaN
__device__ __forceinline__ float inverse(float sum) { return sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum); }

// The statistics of a row, from its reference (log2 units; +inf for a row that sees nothing), the sum under it and one over that.  lse holds the
// probabilities of the backward pass only to |lse| 2^-24 each (scores of 10^4: value gradients off by 8 10^-4; of 10^8: 10^8 times too large), so P is taken as
// the forward has it: exp2(score - ref) weight, the one exact where the other is not small (a factor more per score of dk and dv: training step of 63,600
// keys 398 -> 403 us, fp32 186 -> 189; dq has it once a row).
template <typename T> __device__ __forceinline__ void put_statistics(const AttnArgs &a, int64_t at, float mx, float sum, float inv) {
  a.lse[at] = sum == 0.f ? kNegInf : (mx - PScale<T>::fwd + __builtin_log2f(sum)) * kLn2;
  if (a.ref) {
    a.ref[at] = sum == 0.f ? kPosInf : mx - PScale<T>::fwd;
    a.weight[at] = inv;
  }
}
__device__ __forceinline__ void row_statistics(const AttnArgs &a, int64_t at, float &ref, float &weight) {
  if (a.ref) {
    ref = a.ref[at];
    weight = a.weight[at];
  } else {
    const float x = a.lse[at];
    ref = x == kNegInf ? kPosInf : x * kLog2e;
    weight = 1.f;
  }
}

// x, as a number that the compiler knows nothing about: where one value's rounding to 16 bits is used twice (the output, and what is missing from it), it has rounded
// the product once for one use and twice for the other, and the two were a step apart
__device__ __forceinline__ float settled(float x) {
  asm("" : "+v"(x));
  return x;
}

// Joins the WN key sets of a workgroup's M = S WM rows and writes them: every wave leaves its output, maximum and sums, and a thread adds
// them up under the common maximum.  `o`, `m`, `l`, `lr` as the forward's loops leave them; `part`: where a split's partial rows go, or null.
template <typename T, int DP, int S, int WM, int WN, typename Rows>
__device__ __forceinline__ void join_sets(const AttnArgs &a, char *smem, const typename Shape<S>::acc (&o)[DP / S], float m, float l, float lr, const Rows &row_of, float *pm, int b, int wm, int wn) {
  typedef Shape<S> H;
  constexpr int M = S * WM, LO = DP + 4, DT = DP / S;
  const int tid = threadIdx.x, lane = tid % 64, col = lane % S, g = lane / S;
  float *jo = reinterpret_cast<float *>(smem);                   // [WN][M][LO]
  float *jm = jo + WN * M * LO, *jl = jm + WN * M, *jr = jl + WN * M;   // [WN][M] each
  __syncthreads();
  {
    const int r = wn * M + wm * S + col;
    if (S == 16) {
      l += __shfl_xor(l, 16, 64);
      lr += __shfl_xor(lr, 16, 64);
    }
    l += __shfl_xor(l, 32, 64);
    lr += __shfl_xor(lr, 32, 64);
    if (g == 0) {
      jm[r] = m;
      jl[r] = l;
      jr[r] = lr;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < H::AE; e += 4)
        *reinterpret_cast<f32x4 *>(jo + r * LO + d * S + H::row(e) + g * 4) = f32x4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
  }
  __syncthreads();
  // write out: rows of D channels, 4 per thread
  for (int id = tid; id < M * (a.D / 4); id += 256) {
    const int r = (int)a.by_d4.div((unsigned)id), ch = (id - r * (a.D / 4)) * 4;
    int token, head;
    if (!row_of(r, token, head)) continue;
    float mx = kNegInf, sum = 0.f, rounded = 0.f;
#pragma unroll
    for (int x = 0; x < WN; ++x) mx = max2(mx, jm[x * M + r]);
    f32x4 x4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < WN; ++x) {
      const float f = mx == kNegInf ? 0.f : __builtin_amdgcn_exp2f(jm[x * M + r] - mx);
      sum += mx == kNegInf ? 0.f : jl[x * M + r] * f;
      rounded += mx == kNegInf ? 0.f : jr[x * M + r] * f;
      x4 += *reinterpret_cast<const f32x4 *>(jo + (x * M + r) * LO + ch) * f;
    }
    if (pm) {
      *reinterpret_cast<f32x4 *>(pm + (int64_t)r * a.D + ch) = x4;
      if (ch == 0) {
        pm[(int64_t)M * a.D + r] = mx;
        pm[(int64_t)M * a.D + M + r] = sum;
        pm[(int64_t)M * a.D + 2 * M + r] = rounded;
      }
      continue;
    }
    const float inv = inverse(sum), inv_rounded = inverse(rounded);
    const int64_t at = (int64_t)b * a.so.b + (int64_t)token * a.so.n + (int64_t)head * a.so.h + ch;
    typename Vec4<T>::type y, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float z = settled(x4[e] * inv);
      y[e] = (T)z;
      lo[e] = (T)(x4[e] * inv_rounded - (float)y[e]);
    }
    *reinterpret_cast<typename Vec4<T>::type *>(reinterpret_cast<T *>(a.out) + at) = y;
    if (sizeof(T) == 2 && a.lo) *reinterpret_cast<typename Vec4<T>::type *>(reinterpret_cast<T *>(a.lo) + at) = lo;
    if (ch == 0 && a.lse) put_statistics<T>(a, ((int64_t)b * a.Hq + head) * a.Nq + token, mx, sum, inv);
  }
}

// One workgroup: M = S WM query rows of one group (a row = one query token and one head of the key head's group), 4 waves as WM row
// sets x WN key sets.  The group's keys pass as one stream in tiles of TK = S KU WN (up to a segment); every wave keeps its own
// running maximum, sum and output for its S KU keys of each tile, joined at the end, so the only meeting of the waves in the loop is
// the hand-over of the tile.
// Measured: 32 x 1,590 tokens x 2 heads against 2,048 of 15,900 keys of 64 bf16 channels 115 us (464 TFLOP/s; a large product reaches
// 1,261), 4 x 6,360 x 2 against 4,096 of 63,600 of 128 channels 222 us (481, a training step's), 2 x 4,096 x 4 against 1,024 of 16,384 of 64 fp32 channels 101
// us (85 of 154).  By counters (128 channels) the vector unit is busy 32 % of the time, the matrix pipe 21 %, with 1.35 of the 2 waves that a
// SIMD has room for: equal pieces of work do not fill the last round of the GPU (800 workgroups on 512 places).  Idle lanes for hidden
// rows, in place of a choice of addresses, save a tenth of the vector instructions and lose 3 %.
template <typename T, int DP, int S, int WM, int WN, int KU> struct FwdTile {
  static constexpr int M = S * WM, TK = S * KU * WN, LO = DP + 4;
  static constexpr size_t img = (size_t)TK * Img<T, DP>::RB, tiles = 4 * img;          // K and V, twice
  static constexpr size_t join = (size_t)WN * M * (LO + 3) * 4;                        // outputs, maxima and sums of the key sets
  static constexpr size_t body = tiles > join ? tiles : join;
};
// LO: for a training step of 16-bit types (add_rounded).
template <typename T, int DP, int S, int WM, int WN, int KU, bool LO>
__global__ __launch_bounds__(256, 2) void attend_fwd_kernel(AttnArgs a) {
  typedef FwdTile<T, DP, S, WM, WN, KU> F;
  typedef Shape<S> H;
  constexpr int M = F::M, TK = F::TK, KC = DP / H::KS, DT = DP / S, E = H::AE * KU, PF = E / 8;   // E: scores per lane
  static_assert(TK <= 64 && S * KU == 32, "one segment per tile, 32 keys a wave");
  typedef typename H::acc acc;
  typedef typename Vec8<T>::type frag;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  int *list = reinterpret_cast<int *>(smem + F::body);
  uint32_t *bits = reinterpret_cast<uint32_t *>(list + a.cap);
  __shared__ int n_list;

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, col = lane % S, g = lane / S;
  const int wm = wave / WN, wn = wave % WN;
  unsigned item = xcd_remap(blockIdx.x, gridDim.x);
  const int split = (int)(item % a.splits);
  item /= a.splits;
  const unsigned work = item;
  const int chunk = (int)(item % a.chunks);
  item /= a.chunks;
  const int gr = (int)(item % a.S);
  const int bh = (int)(item / a.S), hk = bh % a.Hkv, b = bh / a.Hkv;

  // row r of the group: token q_block * s + r / G, head hk * G + r % G
  auto row_of = [&](int m, int &token, int &head) {
    const int r = chunk * M + m;
    const int t = (int)a.by_g.div((unsigned)r);
    token = gr * a.q_block + t;
    head = hk * a.G + (r - t * a.G);
    return r < a.rows && token < a.Nq;
  };
  // the queries, as columns (asked for first, so that they arrive while the list is made)
  frag qf[KC];
  {
    int token, head;
    const bool ok = row_of(wm * S + col, token, head);
    const T *p = reinterpret_cast<const T *>(a.q) + (int64_t)b * a.sq.b + (int64_t)token * a.sq.n + (int64_t)head * a.sq.h;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int ch = c * H::KS + g * 8;
      frag t = {};
      if (ok && ch < a.D) t = *reinterpret_cast<const frag *>(p + ch);
      qf[c] = t;
    }
  }
  const int chunks = a.D / Img<T, DP>::VE;
  zero_pads<T, DP, TK>(smem, 4, chunks, wave);
  const int n = group_blocks(a.blocks + ((int64_t)bh * a.S + gr) * a.top, a.top, a.nb, bits, list, &n_list);
  const int e0 = (int)((int64_t)n * split / a.splits), e1 = (int)((int64_t)n * (split + 1) / a.splits);
  const KeySource keys{list + e0, a.vis ? a.vis + (int64_t)b * a.Nk : &g_one, a.vis != nullptr, (e1 - e0) << (a.lb - 6), a.lb, a.Nk};
  const int nt = keys.n * 64 / TK;
  const char *kb = reinterpret_cast<const char *>(reinterpret_cast<const T *>(a.k) + (int64_t)b * a.sk.b + (int64_t)hk * a.sk.h);
  const char *vb = reinterpret_cast<const char *>(reinterpret_cast<const T *>(a.v) + (int64_t)b * a.sv.b + (int64_t)hk * a.sv.h);
  const unsigned kst = (unsigned)(a.sk.n * sizeof(T)), vst = (unsigned)(a.sv.n * sizeof(T));   // host: 128 rows stay below 2^31
  auto issue = [&](int t, const Segment &x) {
    char *kd = smem + (t & 1) * 2 * F::img, *vd = kd + F::img;
    const int off = (t * TK) & 63;                               // within the segment
    // a hidden key's score is overwritten, so its row may be anything; its value row is multiplied by a probability of 0
    dma_segment<T, DP, TK>(kd, kb + (int64_t)x.key0 * a.sk.n * (int64_t)sizeof(T), kst, x.there(a.Nk), off, chunks, wave);
    dma_segment<T, DP, TK>(vd, vb + (int64_t)x.key0 * a.sv.n * (int64_t)sizeof(T), vst, x.mask, off, chunks, wave);
  };
  Segment cur = {}, nxt = {};
  SegmentLoad raw = {};
  if (nt > 0) {
    cur = keys.first();
    issue(0, cur);
    raw = keys.load(TK / 64);
  }
  // a negative scale turns the queries' sign, so that the largest product is the largest score
  const float sc2 = fmaxf(fabsf(a.c), 1e-30f);                   // not 0: -inf times it has to stay -inf
  if (a.c < 0.f) {
#pragma unroll
    for (int c = 0; c < KC; ++c) qf[c] = -qf[c];
  }
  acc o[DT];
  float m = kNegInf, l = 0.f, lr = 0.f;                          // reference in log2 units, sums of exp2(score - reference), scaled as P is, and rounded as P is
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = acc(0.f);
  if (nt > 0) nxt = keys.finish(raw);
  for (int t = 0; t < nt; ++t) {
    tile_barrier<0>();                                           // tile t is there, tile t - 1 has been read
    const char *krows = smem + (t & 1) * 2 * F::img, *vrows = krows + F::img;
    // all fragments of a product are asked for before its first step, those of the second product before the softmax: an LDS read
    // takes longer than a product, and there are only a few waves to hide it behind
    frag kf[KU][KC];
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int c = 0; c < KC; ++c) kf[u][c] = row_frag<T, DP>(krows, (wn * KU + u) * S + col, c * H::KS + g * 8);
    __builtin_amdgcn_sched_barrier(0);
    acc sc[KU];
#pragma unroll
    for (int u = 0; u < KU; ++u) {
      sc[u] = acc(0.f);
#pragma unroll
      for (int c = 0; c < KC; ++c) sc[u] = mma(kf[u][c], qf[c], sc[u]);
    }
    constexpr int NV = DT * PF, AH = sizeof(T) == 2 ? NV : NV / 2;   // fp32 fragments are twice as large, and their products 16 times as long
    frag vf[AH];
    auto v_frag = [&](int i) { return col_frag<T, DP, S>(vrows, wn * 32 + i % PF * 16, i / PF * S, lane); };
#pragma unroll
    for (int i = 0; i < AH; ++i) vf[i] = v_frag(i);
    __builtin_amdgcn_sched_barrier(0);
    // The next tile sets out once this one's fragments have been asked for: a transposing read behind it would be held back until it
    // has landed (the compiler cannot tell the two halves of the LDS apart).
    if (t + 1 < nt) issue(t + 1, nxt);
    raw = keys.load((t + 2) * TK / 64);
    // this wave's keys of the mask
    const unsigned part = (unsigned)(cur.mask >> (((t * TK) & 63) + wn * 32));
    if (part != ~0u) {
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int e = 0; e < H::AE; ++e) sc[u][e] = key_seen<S>(part, u * S + H::row(e)) ? sc[u][e] : kNegInf;
    }
    float mx = max2(sc[0][0], sc[0][1]);
#pragma unroll
    for (int e = 2; e < E; ++e) mx = max2(mx, sc[e / H::AE][e % H::AE]);
    mx = column_max<S>(mx);
    raise_reference<S, T>(mx * sc2, m, l, lr, o);
    const float ms = (m == kNegInf ? 0.f : m) - PScale<T>::fwd;  // nothing seen yet: exp2(-inf - 0) = 0
    float sum = 0.f;
    frag pf[PF];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float p = __builtin_amdgcn_exp2f(fmaf(sc[e / H::AE][e % H::AE], sc2, -ms));
      sum += p;
      pf[e / 8][e % 8] = (T)p;
    }
    l += sum;
    if constexpr (LO) {
#pragma unroll
      for (int i = 0; i < PF; ++i) lr = add_rounded(lr, pf[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) o[i / PF] = mma_whole(i < AH ? vf[i % AH] : v_frag(i), pf[i % PF], o[i / PF]);
    __builtin_amdgcn_sched_barrier(0);                           // the mask of the tile after next is not waited for before the products
    cur = nxt;
    nxt = keys.finish(raw);
  }

  join_sets<T, DP, S, WM, WN>(a, smem, o, m, l, lr, row_of, a.splits > 1 ? a.part + ((int64_t)work * a.splits + split) * M * (a.D + 3) : nullptr, b, wm, wn);
}

// Few rows (a group of up to 16: one token of some heads): one workgroup holds all of them, and no element of a key is used twice.  The four
// waves take 16 keys of a segment each and go their own ways: keys come to registers in the operand's order, values pass through 16 rows
// of LDS of the wave's own (for the transposing read alone), one segment ahead, and no wave waits for another before the join.  What counts is
// the number of loads in flight, so registers are kept to four workgroups per CU; two or three segments ahead at two or three
// workgroups are slower (1,590 tokens x 2 key heads, each with 12 blocks of 64 keys of 72 bf16 channels: 69 us; two ahead 78, three ahead
// 82; the tiles shared through LDS that the larger groups use: 109).  That is 10 TB/s of keys and values, out of the caches; the
// vector instructions of the softmax take about half the time.  A single token of 4 items against 64 blocks of 128 (34 MB): 14 us, 5 of them
// the launch and the list, and 4 for the join.
template <typename T, int DP> struct FewTile {
  static constexpr size_t img = (size_t)16 * Img<T, DP>::RB, tiles = 4 * img, join = (size_t)4 * 16 * (DP + 7) * 4;
  static constexpr size_t body = tiles > join ? tiles : join;
};
template <typename T, int DP, int OCC, bool LO>
__global__ __launch_bounds__(256, OCC) void attend_few_kernel(AttnArgs a) {
  typedef FewTile<T, DP> F;
  typedef Img<T, DP> I;
  constexpr int KC = DP / 32, DT = DP / 16;
  typedef typename Vec8<T>::type frag;
  typedef typename Vec4<T>::type frag4;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  int *list = reinterpret_cast<int *>(smem + F::body);
  uint32_t *bits = reinterpret_cast<uint32_t *>(list + a.cap);
  __shared__ int n_list;

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, col = lane % 16, g = lane / 16;
  unsigned item = xcd_remap(blockIdx.x, gridDim.x);
  const int split = (int)(item % a.splits);
  const unsigned work = item / a.splits;
  const int gr = (int)(work % a.S), bh = (int)(work / a.S), hk = bh % a.Hkv, b = bh / a.Hkv;
  auto row_of = [&](int r, int &token, int &head) {
    const int t = (int)a.by_g.div((unsigned)r);
    token = gr * a.q_block + t;
    head = hk * a.G + (r - t * a.G);
    return r < a.rows && token < a.Nq;
  };
  frag qf[KC];
  {
    int token, head;
    const bool ok = row_of(col, token, head);
    const T *p = reinterpret_cast<const T *>(a.q) + (int64_t)b * a.sq.b + (int64_t)token * a.sq.n + (int64_t)head * a.sq.h;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int ch = c * 32 + g * 8;
      frag t = {};
      if (ok && ch < a.D) t = *reinterpret_cast<const frag *>(p + ch);
      qf[c] = a.c < 0.f ? -t : t;                                // a negative scale turns the queries' sign, as in the other forward
    }
  }
  const int n = group_blocks(a.blocks + ((int64_t)bh * a.S + gr) * a.top, a.top, a.nb, bits, list, &n_list);
  const int e0 = (int)((int64_t)n * split / a.splits), e1 = (int)((int64_t)n * (split + 1) / a.splits);
  const int per = a.lb - 6, nt = (e1 - e0) << per;
  const char *kb = reinterpret_cast<const char *>(reinterpret_cast<const T *>(a.k) + (int64_t)b * a.sk.b + (int64_t)hk * a.sk.h);
  const char *vb = reinterpret_cast<const char *>(reinterpret_cast<const T *>(a.v) + (int64_t)b * a.sv.b + (int64_t)hk * a.sv.h);
  const float *vis = a.vis ? a.vis + (int64_t)b * a.Nk : &g_one;
  const int vis_step = a.vis != nullptr;
  const int64_t kst = a.sk.n * (int64_t)sizeof(T), vst = a.sv.n * (int64_t)sizeof(T);
  // channels from D on are read as the last ones (a product's are zeroed, an output's not written)
  const unsigned ch0 = (unsigned)(g * 8 * sizeof(T)), ch1 = (unsigned)(min((KC - 1) * 32 + g * 8, a.D - 8) * sizeof(T));
  char *img = smem + wave * F::img;

  frag kf[KC], vf[KC];
  float see = 0.f;
  int left = 0;                                                  // keys from this wave's first one on
  auto key_of = [&](int i) { return (list[e0 + (i >> per)] << a.lb) + ((i & ((1 << per) - 1)) << 6) + wave * 16; };
  // A key behind the last one is read as the last (a wave that has none: as the head's first); its score is overwritten.
  auto load = [&](int key0) {
    left = a.Nk - key0;
    const bool live = left > 0;
    const int first = live ? key0 : 0;
    const unsigned row = live ? (unsigned)min(col, left - 1) : 0u;
    const char *kp = kb + first * kst, *vp = vb + first * vst;
    const unsigned kr = row * (unsigned)kst, vr = row * (unsigned)vst;
#pragma unroll
    for (int c = 0; c < KC; ++c) kf[c] = *(const __attribute__((address_space(1))) frag *)(kp + (kr + (c + 1 < KC ? c * 32 * (unsigned)sizeof(T) + ch0 : ch1)));
#pragma unroll
    for (int c = 0; c < KC; ++c) vf[c] = *(const __attribute__((address_space(1))) frag *)(vp + (vr + (c + 1 < KC ? c * 32 * (unsigned)sizeof(T) + ch0 : ch1)));
    see = *(const __attribute__((address_space(1))) float *)(vis + first * vis_step + row * (unsigned)vis_step);
  };
  const float sc2 = fmaxf(fabsf(a.c), 1e-30f);                   // not 0: -inf times it has to stay -inf
  f32x4 o[DT];
  float m = kNegInf, l = 0.f, lr = 0.f;
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (nt > 0) load(__builtin_amdgcn_readfirstlane(key_of(0)));
  for (int t = 0; t < nt; ++t) {
    const int next = key_of(min(t + 1, nt - 1));
    const bool in = col < left && see > 0.5f;
    const unsigned part = (unsigned)__ballot(in);                // the four quarters say the same
    f32x4 sc = f32x4{0.f, 0.f, 0.f, 0.f};
    if (part != 0) {
      if (a.D < DP && (KC - 1) * 32 + g * 8 >= a.D) kf[KC - 1] = frag{};
#pragma unroll
      for (int c = 0; c < KC; ++c) sc = mma(kf[c], qf[c], sc);
      if (part != ~0u) {                                         // a hidden value is multiplied by a probability of 0: it has to be a number
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          typedef unsigned words __attribute__((ext_vector_type(sizeof(frag) / 4)));
          words w = __builtin_bit_cast(words, vf[c]);
#pragma unroll
          for (int e = 0; e < (int)sizeof(frag) / 4; ++e) w[e] = in ? w[e] : 0u;
          vf[c] = __builtin_bit_cast(frag, w);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[e] = key_seen<16>(part, e) ? sc[e] : kNegInf;
      }
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        char *row = img + col * I::RB;
        if constexpr (sizeof(T) == 2) *reinterpret_cast<frag *>(row + (((c * 4 + g) ^ I::swz(col)) << 4)) = vf[c];
        else {
          *reinterpret_cast<f32x4 *>(row + (((c * 8 + g * 2) ^ I::swz(col)) << 4)) = __builtin_shufflevector(vf[c], vf[c], 0, 1, 2, 3);
          *reinterpret_cast<f32x4 *>(row + (((c * 8 + g * 2 + 1) ^ I::swz(col)) << 4)) = __builtin_shufflevector(vf[c], vf[c], 4, 5, 6, 7);
        }
      }
      wave_exchange();                                           // the rows are there
    }
    if (t + 1 < nt) load(__builtin_amdgcn_readfirstlane(next));
    if (part == 0) continue;
    frag4 vt[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) vt[d] = col_frag4<T, DP>(img, d * 16, lane);
    wave_exchange();                                             // the rows have been read
    const float mx = column_max<16>(max2(max2(sc[0], sc[1]), max2(sc[2], sc[3])));
    raise_reference<16, T>(mx * sc2, m, l, lr, o);
    const float ms = (m == kNegInf ? 0.f : m) - PScale<T>::fwd;
    f32x4 p;
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], sc2, -ms));
    l += (p[0] + p[1]) + (p[2] + p[3]);
    const frag4 pf = __builtin_convertvector(p, frag4);
    if constexpr (LO) lr = add_rounded(lr, pf);
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = mma4_whole(vt[d], pf, o[d]);
  }
  join_sets<T, DP, 16, 1, 4>(a, smem, o, m, l, lr, row_of, a.splits > 1 ? a.part + ((int64_t)work * a.splits + split) * 16 * (a.D + 3) : nullptr, b, 0, wave);
}
// Joins the splits (at most kMaxSplits) of a row: one workgroup per row.  Lane x of every wave holds split x's factor; the waves take
// the splits in turn, a lane two channels of them, and are added up in wave order.  Everything is asked for at once: the time is that
// of one trip to memory.
constexpr int kMaxSplits = 64;
template <typename T>
__global__ __launch_bounds__(256) void attend_join_kernel(AttnArgs a, int M) {
  __shared__ float2 sums[4][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int64_t work = blockIdx.x / (unsigned)M;
  const int r = (int)(blockIdx.x - (unsigned)work * (unsigned)M);
  const int chunk = (int)(work % a.chunks), s = (int)(work / a.chunks % a.S);
  const int bh = (int)(work / a.chunks / a.S), hk = bh % a.Hkv, b = bh / a.Hkv;
  const int row = chunk * M + r, t = (int)a.by_g.div((unsigned)row), token = s * a.q_block + t, head = hk * a.G + (row - t * a.G);
  if (row >= a.rows || token >= a.Nq) return;
  const int64_t step = (int64_t)M * (a.D + 3);
  const float *p = a.part + work * a.splits * step;
  const int x = min(lane, a.splits - 1);
  const float m = lane < a.splits ? p[x * step + (int64_t)M * a.D + r] : kNegInf;
  const float l = p[x * step + (int64_t)M * a.D + M + r], lr = p[x * step + (int64_t)M * a.D + 2 * M + r];
  const int ch = min(lane * 2, a.D - 2);
  float2 v[kMaxSplits / 4];
#pragma unroll
  for (int i = 0; i < kMaxSplits / 4; ++i) v[i] = *reinterpret_cast<const float2 *>(p + min(i * 4 + wave, a.splits - 1) * step + (int64_t)r * a.D + ch);
  const float mx = wave_max(m);
  const float w = m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m - mx);
  const float sum = wave_sum(m == kNegInf ? 0.f : l * w), rounded = wave_sum(m == kNegInf ? 0.f : lr * w);
  float2 o = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kMaxSplits / 4; ++i) {                     // a split that is not there has a factor of 0
    const float f = __shfl(w, i * 4 + wave, 64);
    o.x += f == 0.f ? 0.f : v[i].x * f;
    o.y += f == 0.f ? 0.f : v[i].y * f;
  }
  sums[wave][lane] = o;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    o.x += sums[i][lane].x;
    o.y += sums[i][lane].y;
  }
  const float inv = inverse(sum), inv_rounded = inverse(rounded);
  if (lane * 2 < a.D) {
    const int64_t at = (int64_t)b * a.so.b + (int64_t)token * a.so.n + (int64_t)head * a.so.h + ch;
    T *y = reinterpret_cast<T *>(a.out) + at, *lo = reinterpret_cast<T *>(a.lo) + at;
    const float z0 = settled(o.x * inv), z1 = settled(o.y * inv);
    const T y0 = (T)z0, y1 = (T)z1;
    y[0] = y0;
    y[1] = y1;
    if (sizeof(T) == 2 && a.lo) {
      lo[0] = (T)(o.x * inv_rounded - (float)y0);
      lo[1] = (T)(o.y * inv_rounded - (float)y1);
    }
  }
  if (lane == 0 && a.lse) put_statistics<T>(a, ((int64_t)b * a.Hq + head) * a.Nq + token, mx, sum, inv);
}

// ------------------------------------------------------------------------------------------ backward
// With P = exp(scale S - lse) (row_statistics) and dP = dout V^T:  dV = P^T dout,  dS = scale P o (dP - delta),  delta = rowsum(dout o out),
// dQ = dS K,  dK = dS^T Q.  dQ is summed per query tile (like the forward), dK and dV per key tile: two kernels that both recompute
// S and dP, and no atomics, so a gradient does not depend on the order of the workgroups.

// fp16: a score gradient lies anywhere between the cotangent's size and that over the number of keys, and fp16 steps are absolute below 2^-14 (a
// cotangent of 10^-3 and 4,096 keys, as they are: dq and dk off by 2 %).  So the gradients of a row (dq) or a key (dk) are multiplied by a power of
// two of their own, which the sums are divided by at the end.  It starts high (a result of 2^-25 needs no term below 2^-60) and falls, like the
// reference of a softmax, whenever one of the gradients passes 2^15; the largest of those is then just above 2^10, so what rounding takes from a term is half
// a step of it or 2^-35 of the largest.  Nothing but the row's (key's) own terms decides it.  Measured: fp16 training step of 63,600 keys, dq 254 -> 267 us,
// dk and dv 422 -> 428.
template <typename T> struct GradRange { static constexpr bool on = false; };
template <> struct GradRange<_Float16> { static constexpr bool on = true; static constexpr float start = 0x1p60f, limit = 0x1p15f; };
// ds: a lane's gradients, times f; o: its column's sums, times f
template <int S, typename V, int N, typename O, int DT> __device__ __forceinline__ void fit_range(V (&ds)[N], float &f, O (&o)[DT]) {
  typedef GradRange<_Float16> R;
  constexpr int E = sizeof(V) / 4;
  float mx = 0.f;
#pragma unroll
  for (int e = 0; e < N * E; ++e) mx = fmaxf(mx, fabsf(ds[e / E][e % E]));
  if (__any(mx > R::limit)) {
    const float top = column_max<S>(mx);
    const float g = top > R::limit && top < kPosInf ? __builtin_ldexpf(1.f, 11 - __builtin_amdgcn_frexp_expf(top)) : 1.f;
    f *= g;
#pragma unroll
    for (int u = 0; u < N; ++u) ds[u] *= g;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] *= g;
  }
}

// TWO: what rounding takes from a 16-bit operand (a score gradient; for dV a probability) is multiplied too.  Rounded once, it adds an error of the size of the
// result's own rounding: together 1.46 times that.  Where a sum has few terms, or a tensor few sums, the roundings do not average out
// (items of 8 queries up to 2.3, of 300 up to 1.58), and below 64 channels they lie along the sum: there both parts are taken (1.00 to 1.06).  The rule looks at the sums of one item: whatever shares a call with it does not matter.
// Two parts throughout would cost dq 248 -> 299 us, dk and dv 415 -> 487 (training step of 63,600 bf16 keys).
constexpr int64_t kFewKeys = 512, kFewQueries = 2048;
template <typename T> static bool two_parts(const AttnArgs &a) {
  const int64_t keys = (int64_t)a.cap << a.lb;
  return sizeof(T) == 2 && (a.D < 64 || (keys < a.Nk ? keys : a.Nk) <= kFewKeys || (int64_t)a.Nq * a.G <= kFewQueries);
}

// delta of every row: 16 lanes per row, 8 channels each.  The output is taken as it was before its rounding (out + lo): delta is
// subtracted from products of its own size, and with few keys a rounded output's error is the largest of the gradient (2 to 16
// keys: error of dq and dk 1.6 to 2.9 times that of their own rounding, 1.4 to 1.5 so; the smaller part of it is left, that of the
// score gradients as operands).  And the plan of the key / value gradients (inv, chosen) is cleared
template <typename T>
__global__ __launch_bounds__(256) void attend_delta_kernel(AttnArgs a) {
  const int64_t id = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
  const int ch = threadIdx.x % 16 * 8;
  const bool live = id < (int64_t)a.B * a.Nq * a.Hq;
  const int64_t w = live ? id : 0;
  const int head = (int)(w % a.Hq);
  const int64_t bt = w / a.Hq;
  const int token = (int)(bt % a.Nq), b = (int)(bt / a.Nq);
  float sum = 0.f;
  if (live && ch < a.D) {
    typedef typename Vec8<T>::type frag;
    const frag x = *reinterpret_cast<const frag *>(reinterpret_cast<const T *>(a.dout) + (int64_t)b * a.sdo.b + (int64_t)token * a.sdo.n + (int64_t)head * a.sdo.h + ch);
    const frag y = *reinterpret_cast<const frag *>(reinterpret_cast<const T *>(a.out) + (int64_t)b * a.so.b + (int64_t)token * a.so.n + (int64_t)head * a.so.h + ch);
    frag z = {};
    if (sizeof(T) == 2 && a.lo) z = *reinterpret_cast<const frag *>(reinterpret_cast<const T *>(a.lo) + (int64_t)b * a.so.b + (int64_t)token * a.so.n + (int64_t)head * a.so.h + ch);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf((float)x[e], (float)y[e] + (float)z[e], sum);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (live && ch == 0) a.delta[((int64_t)b * a.Hq + head) * a.Nq + token] = sum;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.plan_words; i += (int64_t)gridDim.x * 256) a.inv[i] = 0;
}

// which groups chose each block: one bit per (block, group), and (for the order of the work only) how many entries named it
__global__ __launch_bounds__(256) void attend_invert_kernel(AttnArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.B * a.Hkv * a.S * a.top) return;
  const int j = a.blocks[i];
  const int64_t row = i / a.top;
  const int s = (int)(row % a.S);
  const int64_t bh = row / a.S;
  if (j < 0 || j >= a.nb) return;
  atomicOr(&a.inv[(bh * a.nb + j) * a.words + (s >> 5)], 1u << (s & 31));
  atomicAdd(&a.chosen[bh * a.nb + j], 1u);
}
// The blocks of one (item, key head), often chosen ones first: the work per block differs by a factor of four and more, and a long one
// that starts last keeps the GPU waiting (key and value gradients of the training step of 63,600 keys: 517 -> 445 us then).  Counting sort into 256 classes; the
// order within a class does not matter.  One workgroup per (item, key head).
__global__ __launch_bounds__(1024) void attend_order_kernel(AttnArgs a) {
  __shared__ unsigned start[256], most;
  const uint32_t *cnt = a.chosen + (int64_t)blockIdx.x * a.nb;
  int32_t *order = a.order + (int64_t)blockIdx.x * a.nb;
  if (threadIdx.x < 256) start[threadIdx.x] = 0;
  if (threadIdx.x == 0) most = 0;
  __syncthreads();
  for (int j = threadIdx.x; j < a.nb; j += 1024) atomicMax(&most, cnt[j]);
  __syncthreads();
  const unsigned top = most + 1;
  auto cls = [&](unsigned c) { return 255 - (unsigned)((uint64_t)c * 256 / top); };
  for (int j = threadIdx.x; j < a.nb; j += 1024) atomicAdd(&start[cls(cnt[j])], 1u);
  __syncthreads();
  if (threadIdx.x < 64) {                                        // exclusive prefix sums, 4 classes a lane
    unsigned v[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = sum; sum += start[threadIdx.x * 4 + i]; }
    unsigned incl = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned t = __shfl_up(incl, o, 64);
      if ((int)threadIdx.x >= o) incl += t;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) start[threadIdx.x * 4 + i] = incl - sum + v[i];
  }
  __syncthreads();
  for (int j = threadIdx.x; j < a.nb; j += 1024) order[atomicAdd(&start[cls(cnt[j])], 1u)] = j;
}

// The forward's tiles with two products for one: 244 us (656 TFLOP/s) for the training step of 63,600 keys, fp32 133 us (97).
template <typename T, int DP, int S, int WM, int WN> struct DqTile {
  static constexpr int KU = 32 / S, M = S * WM, TK = 32 * WN, LO = DP + 4;             // 32 keys a wave
  static constexpr size_t img = (size_t)TK * Img<T, DP>::RB, tiles = 4 * img;          // K and V, twice
  static constexpr size_t join = (size_t)WN * M * LO * 4;
  static constexpr size_t body = tiles > join ? tiles : join;
};
template <typename T, int DP, int S, int WM, int WN, int OCC, bool TWO>
__global__ __launch_bounds__(256, OCC) void attend_dq_kernel(AttnArgs a) {
  typedef DqTile<T, DP, S, WM, WN> F;
  typedef Shape<S> H;
  typedef typename H::acc acc;
  constexpr int M = F::M, TK = F::TK, KU = F::KU, KC = DP / H::KS, DT = DP / S, PF = 2 * KU * H::AE / 16;
  static_assert(TK <= 64, "one segment per tile");
  typedef typename Vec8<T>::type frag;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  int *list = reinterpret_cast<int *>(smem + F::body);
  uint32_t *bits = reinterpret_cast<uint32_t *>(list + a.cap);
  __shared__ int n_list;

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, col = lane % S, g = lane / S;
  const int wm = wave / WN, wn = wave % WN;
  unsigned item = xcd_remap(blockIdx.x, gridDim.x);
  const int chunk = (int)(item % a.chunks);
  item /= a.chunks;
  const int gr = (int)(item % a.S);
  const int bh = (int)(item / a.S), hk = bh % a.Hkv, b = bh / a.Hkv;
  auto row_of = [&](int m, int &token, int &head) {
    const int r = chunk * M + m;
    const int t = (int)a.by_g.div((unsigned)r);
    token = gr * a.q_block + t;
    head = hk * a.G + (r - t * a.G);
    return r < a.rows && token < a.Nq;
  };
  frag qf[KC], df[KC];
  float ref = kPosInf, weight = 0.f, delta = 0.f;                // exp2(x - inf) = 0: no row, or a row that sees nothing
  {
    int token, head;
    const bool ok = row_of(wm * S + col, token, head);
    const T *p = reinterpret_cast<const T *>(a.q) + (int64_t)b * a.sq.b + (int64_t)token * a.sq.n + (int64_t)head * a.sq.h;
    const T *d = reinterpret_cast<const T *>(a.dout) + (int64_t)b * a.sdo.b + (int64_t)token * a.sdo.n + (int64_t)head * a.sdo.h;
    if (ok) {
      const int64_t at = ((int64_t)b * a.Hq + head) * a.Nq + token;
      row_statistics(a, at, ref, weight);
      delta = a.delta[at];
    }
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int ch = c * H::KS + g * 8;
      frag t = {}, u = {};
      if (ok && ch < a.D) {
        t = *reinterpret_cast<const frag *>(p + ch);
        u = *reinterpret_cast<const frag *>(d + ch);
      }
      qf[c] = t;
      df[c] = u;
    }
  }
  const int chunks = a.D / Img<T, DP>::VE;
  zero_pads<T, DP, TK>(smem, 4, chunks, wave);
  const int n = group_blocks(a.blocks + ((int64_t)bh * a.S + gr) * a.top, a.top, a.nb, bits, list, &n_list);
  const KeySource keys{list, a.vis ? a.vis + (int64_t)b * a.Nk : &g_one, a.vis != nullptr, n << (a.lb - 6), a.lb, a.Nk};
  const int nt = keys.n * 64 / TK;
  const char *kb = reinterpret_cast<const char *>(reinterpret_cast<const T *>(a.k) + (int64_t)b * a.sk.b + (int64_t)hk * a.sk.h);
  const char *vb = reinterpret_cast<const char *>(reinterpret_cast<const T *>(a.v) + (int64_t)b * a.sv.b + (int64_t)hk * a.sv.h);
  const unsigned kst = (unsigned)(a.sk.n * sizeof(T)), vst = (unsigned)(a.sv.n * sizeof(T));
  auto issue = [&](int t, const Segment &x) {
    char *kd = smem + (t & 1) * 2 * F::img, *vd = kd + F::img;
    const int off = (t * TK) & 63;
    dma_segment<T, DP, TK>(kd, kb + (int64_t)x.key0 * a.sk.n * (int64_t)sizeof(T), kst, x.mask, off, chunks, wave);
    dma_segment<T, DP, TK>(vd, vb + (int64_t)x.key0 * a.sv.n * (int64_t)sizeof(T), vst, x.mask, off, chunks, wave);
  };
  Segment cur = {}, nxt = {};
  SegmentLoad raw = {};
  if (nt > 0) {
    cur = keys.first();
    issue(0, cur);
    raw = keys.load(TK / 64);
  }
  const float c2 = a.c == 0.f ? 1e-30f : a.c, hidden = c2 < 0.f ? kPosInf : kNegInf;   // their product has to be -inf
  acc o[DT];
  float range = 1.f;
  if constexpr (GradRange<T>::on) range = GradRange<T>::start;
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = acc(0.f);
  if (nt > 0) nxt = keys.finish(raw);
  for (int t = 0; t < nt; ++t) {
    tile_barrier<0>();
    const char *krows = smem + (t & 1) * 2 * F::img, *vrows = krows + F::img;
    acc sc[KU], dp[KU];
#pragma unroll
    for (int u = 0; u < KU; ++u) sc[u] = dp[u] = acc(0.f);
    // the fragments of a quarter of the products (S = 32: half of them) at a time, always one batch ahead
    constexpr int NB = 2, CB = KU * KC / NB;                     // (u, c) pairs of a batch
    frag kf[NB][CB], vf[NB][CB];
    auto rows = [&](int x) {
#pragma unroll
      for (int i = 0; i < CB; ++i) {
        const int u = (x * CB + i) / KC, c = (x * CB + i) % KC;
        kf[x][i] = row_frag<T, DP>(krows, wn * 32 + u * S + col, c * H::KS + g * 8);
        vf[x][i] = row_frag<T, DP>(vrows, wn * 32 + u * S + col, c * H::KS + g * 8);
      }
    };
    rows(0);
#pragma unroll
    for (int x = 0; x < NB; ++x) {
      __builtin_amdgcn_sched_barrier(0);
      if (x + 1 < NB) rows(x + 1);
#pragma unroll
      for (int i = 0; i < CB; ++i) {
        const int u = (x * CB + i) / KC, c = (x * CB + i) % KC;
        sc[u] = mma(kf[x][i], qf[c], sc[u]);
        dp[u] = mma(vf[x][i], df[c], dp[u]);
      }
    }
    constexpr int NV = DT * PF, AH = sizeof(T) == 2 ? NV : NV / 2;
    frag ka[AH];
    auto k_frag = [&](int i) { return col_frag<T, DP, S>(krows, wn * 32 + i % PF * 16, i / PF * S, lane); };
#pragma unroll
    for (int i = 0; i < AH; ++i) ka[i] = k_frag(i);
    __builtin_amdgcn_sched_barrier(0);
    if (t + 1 < nt) issue(t + 1, nxt);                           // behind the transposing reads, as in the forward
    raw = keys.load((t + 2) * TK / 64);
    frag gf[PF], gl[TWO ? PF : 1];
    const unsigned part = (unsigned)(cur.mask >> (((t * TK) & 63) + wn * 32));
    if (part != ~0u) {                                           // an unseen key's products are those of zeros: its probability has to become 0
#pragma unroll
      for (int e = 0; e < KU * H::AE; ++e) sc[e / H::AE][e % H::AE] = key_seen<S>(part, e / H::AE * S + H::row(e % H::AE)) ? sc[e / H::AE][e % H::AE] : hidden;
    }
#pragma unroll
    for (int e = 0; e < KU * H::AE; ++e) {
      const int u = e / H::AE, x = e % H::AE;
      const float p = __builtin_amdgcn_exp2f(fmaf(sc[u][x], c2, -ref));
      sc[u][x] = p * (dp[u][x] - delta);
      if constexpr (GradRange<T>::on) sc[u][x] *= range;
    }
    if constexpr (GradRange<T>::on) fit_range<S>(sc, range, o);
#pragma unroll
    for (int e = 0; e < KU * H::AE; ++e) {
      const float ds = sc[e / H::AE][e % H::AE];
      gf[e / 8][e % 8] = (T)ds;
      if constexpr (TWO) gl[e / 8][e % 8] = (T)(ds - (float)gf[e / 8][e % 8]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const frag k = i < AH ? ka[i % AH] : k_frag(i);
      o[i / PF] = mma_whole(k, gf[i % PF], o[i / PF]);
      if constexpr (TWO) o[i / PF] = mma(k, gl[i % PF], o[i / PF]);
    }
    __builtin_amdgcn_sched_barrier(0);                           // the mask of the tile after next is not waited for before the products
    cur = nxt;
    nxt = keys.finish(raw);
  }
  float *jo = reinterpret_cast<float *>(smem);                   // [WN][M][LO]
  __syncthreads();
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    o[d] *= GradRange<T>::on ? weight / range : weight;          // every key set has a range of its own
#pragma unroll
    for (int e = 0; e < H::AE; e += 4)
      *reinterpret_cast<f32x4 *>(jo + (wn * M + wm * S + col) * F::LO + d * S + H::row(e) + g * 4) = f32x4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
  }
  __syncthreads();
  for (int id = tid; id < M * (a.D / 4); id += 256) {
    const int r = (int)a.by_d4.div((unsigned)id), ch = (id - r * (a.D / 4)) * 4;
    int token, head;
    if (!row_of(r, token, head)) continue;
    f32x4 x = *reinterpret_cast<const f32x4 *>(jo + r * F::LO + ch);
#pragma unroll
    for (int w = 1; w < WN; ++w) x += *reinterpret_cast<const f32x4 *>(jo + (w * M + r) * F::LO + ch);
    x *= a.scale;
    typename Vec4<T>::type y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)x[e];
    *reinterpret_cast<typename Vec4<T>::type *>(reinterpret_cast<T *>(a.dq) + (int64_t)b * a.sdq.b + (int64_t)token * a.sdq.n + (int64_t)head * a.sdq.h + ch) = y;
  }
}

// One workgroup: 64 keys (a tile of one block), 16 per wave, against all query rows of the groups that chose the block.  The rows pass
// as a stream (group after group, in ascending order) in tiles of 32; rows and keys have changed places with the forward:
// S = Q K^T leaves a lane the probabilities of ITS key, the operand of dV^T = dout^T P and, as dS, of dK^T = Q^T dS.
// 16 keys a wave: with 32 (half the LDS reads per product) the two accumulators take 350 registers, one wave per SIMD, and
// every wait shows (802 against 594 us then for the training step of 63,600 keys, 416 now: 513 TFLOP/s; fp32 as in the forward 189 us, 91).
// LDS is busy 41 % of the time, the vector unit 32 %, the matrix pipe 23 %.  Rows lie scattered, so their tiles come from a ring
// of four, three tiles ahead; where the rows lie is worked out for 512 of them at a time, not in the loop.
constexpr int kWindow = 32;    // words of group bits taken at a time: up to 1024 groups in the list
constexpr int kBatch = 512;    // rows located at a time
// Rows after which an fp32 accumulator is added to the others: a serial sum of n random terms is off by about 0.4 sqrt(n / 2) 2^-24 of its size (measured:
// 38 2^-24 for 16,000 rows, 10 so).  2,000 queries x 16 heads x 32 items, 512 keys of 2 heads of 64 channels: training step 5,262 -> 5,327 us.  16-bit
// results have no use for it.
constexpr unsigned kSerial = 512;

template <typename T, int DP> struct DkvTile {
  static constexpr int M = 64, TR = 32, NB = sizeof(T) == 4 && DP > 64 ? 2 : 4;
  static constexpr size_t img = (size_t)TR * Img<T, DP>::RB, tiles = NB * 2 * img;     // Q and dout
  static constexpr size_t body = tiles;
  // behind the tiles: where a row lies in q and dout (in 16 bytes), statistics and delta, the list of groups
  static constexpr size_t bytes = body + kBatch * 20 + 32 * kWindow * 4;
};
template <typename T, int DP, bool TWO>
__global__ __launch_bounds__(256, 2) void attend_dkv_kernel(AttnArgs a) {
  typedef DkvTile<T, DP> F;
  typedef Pieces<T, DP, F::TR> P;
  constexpr int M = F::M, TR = F::TR, NB = F::NB, KC = DP / 32, DT = DP / 16, PER = 2 * P::NU;
  typedef typename Vec8<T>::type frag;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  u32x2 *tab = reinterpret_cast<u32x2 *>(smem + F::body);                              // [kBatch], x = ~0: no row
  float *refs = reinterpret_cast<float *>(tab + kBatch), *weights = refs + kBatch, *delta = weights + kBatch;   // [kBatch] each
  int *list = reinterpret_cast<int *>(delta + kBatch);                                 // [32 kWindow]
  __shared__ int n_list;

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, col = lane % 16, g = lane / 16;
  const int per_block = 1 << (a.lb - 6), tiles_of = a.nb * per_block;
  unsigned item = xcd_remap(blockIdx.x, gridDim.x);
  const int split = (int)(item % a.splits);
  item /= a.splits;
  const int bh = (int)(item / tiles_of), hk = bh % a.Hkv, b = bh / a.Hkv, at_ = (int)(item % tiles_of);
  const int block = __builtin_amdgcn_readfirstlane(a.order[(int64_t)bh * a.nb + at_ / per_block]), kt = block * per_block + at_ % per_block;
  if (kt * M >= a.Nk) return;                                    // the second half of a block that ends in its first
  const uint32_t *inv = a.inv + ((int64_t)bh * a.nb + block) * a.words;

  // this lane's key.  A hidden key's row is taken as zeros: whatever its probabilities come to stays in its own column, which is
  // not written.  Its loads are unconditional and not waited for before the first rows are on their way.
  const uint32_t first_word = tid < kWindow && tid < a.words ? inv[tid] : 0;
  frag kf[KC], vf[KC];
  const int key = kt * M + wave * 16 + col;
  const float see = a.vis ? a.vis[(int64_t)b * a.Nk + min(key, a.Nk - 1)] : 1.f;
  {
    const int row = min(key, a.Nk - 1);
    const T *p = reinterpret_cast<const T *>(a.k) + (int64_t)b * a.sk.b + (int64_t)row * a.sk.n + (int64_t)hk * a.sk.h;
    const T *q = reinterpret_cast<const T *>(a.v) + (int64_t)b * a.sv.b + (int64_t)row * a.sv.n + (int64_t)hk * a.sv.h;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int ch = min(c * 32 + g * 8, a.D - 8);
      kf[c] = *reinterpret_cast<const frag *>(p + ch);
      vf[c] = *reinterpret_cast<const frag *>(q + ch);
    }
  }
  bool fresh = true;                                             // kf, vf as loaded
  bool seen = false;
  const char *qb = reinterpret_cast<const char *>(reinterpret_cast<const T *>(a.q) + (int64_t)b * a.sq.b);
  const char *db = reinterpret_cast<const char *>(reinterpret_cast<const T *>(a.dout) + (int64_t)b * a.sdo.b);
  const int chunks = a.D / P::I::VE;
  float range = 1.f;                                             // of this lane's key; P's own factor is part of it
  if constexpr (GradRange<T>::on) range = GradRange<T>::start * PScale<T>::inv;
  f32x4 gk[DT], gv[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) gk[d] = gv[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  zero_pads<T, DP, TR>(smem, 2 * NB, chunks, wave);

  // The sums to their rows (of a split: to its part).  A lane holds 4 channels of its key per 16: the 4 quarters together write 32 (fp32: 64) bytes of 16
  // rows at a time.  fp32 sums go there every kSerial rows and are added to what lies there.
  bool begun = false;
  unsigned summed = 0;
  auto put = [&]() {
    if (key < a.Nk) {
      const float k_scale = GradRange<T>::on ? a.scale * PScale<T>::inv / range : a.scale;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        T *out = reinterpret_cast<T *>(which ? a.dv : a.dk);
        if (out == nullptr) continue;
        const Str st = which ? a.sdv : a.sdk;
        const float f = which ? PScale<T>::inv : k_scale;
        float *part = a.splits > 1 ? a.part + ((((int64_t)which * a.splits + split) * a.B * a.Hkv + bh) * a.Nk + key) * a.D + g * 4 : nullptr;
        T *row = out + (int64_t)b * st.b + (int64_t)key * st.n + (int64_t)hk * st.h + g * 4;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          if (d * 16 + g * 4 >= a.D) continue;
          f32x4 y = seen ? (which ? gv[d] : gk[d]) * f : f32x4{0.f, 0.f, 0.f, 0.f};
          if (part) {
            f32x4 *to = reinterpret_cast<f32x4 *>(part + d * 16);
            if (sizeof(T) == 4 && begun) y += *to;
            *to = y;
          } else {
            typename Vec4<T>::type *to = reinterpret_cast<typename Vec4<T>::type *>(row + d * 16), z;
            if constexpr (sizeof(T) == 4) {
              if (begun) y += *to;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = (T)y[e];
            *to = z;
          }
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) gk[d] = gv[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    begun = true;
    summed = 0;
  };
  for (int w0 = 0; w0 < a.words; w0 += kWindow) {
    __syncthreads();                                             // the last window's list has been read
    if (tid < 64) {
      uint32_t m = w0 == 0 ? first_word : tid < kWindow && w0 + tid < a.words ? inv[w0 + tid] : 0;
      int incl = __popc(m);
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(incl, o, 64);
        if (tid >= o) incl += t;
      }
      int at = incl - __popc(m);
      if (tid == 63) n_list = incl;
      while (m) {
        list[at++] = (w0 + tid) * 32 + __builtin_ctz(m);
        m &= m - 1;
      }
    }
    __syncthreads();
    const unsigned all = (unsigned)n_list * (unsigned)a.rows;    // < 2^31
    const unsigned total = (unsigned)((uint64_t)all * (split + 1) / a.splits);
    for (unsigned r0 = (unsigned)((uint64_t)all * split / a.splits); r0 < total; r0 += kBatch) {
      if (sizeof(T) == 4 && summed >= kSerial) put();
      __syncthreads();                                           // the last batch's tables and tiles have been read
      const int in_batch = (int)min((unsigned)kBatch, total - r0), nt = (in_batch + TR - 1) / TR;
      summed += in_batch;
#pragma unroll
      for (int u = 0; u < kBatch / 256; ++u) {
        const int r = u * 256 + tid;
        u32x2 where = {~0u, ~0u};
        float ref = kPosInf, weight = 0.f, de = 0.f;             // exp2(x - inf) = 0
        if (r < in_batch) {
          const unsigned e = a.by_rows.div(r0 + r), rr = r0 + r - e * (unsigned)a.rows;
          const unsigned tk = a.by_g.div(rr);
          const int token = list[e] * a.q_block + (int)tk;
          const int head = hk * a.G + (int)(rr - tk * (unsigned)a.G);
          if (token < a.Nq) {
            constexpr int64_t u16 = 16 / sizeof(T);              // strides are multiples of 16 bytes
            where.x = (unsigned)(((int64_t)token * a.sq.n + (int64_t)head * a.sq.h) / u16);
            where.y = (unsigned)(((int64_t)token * a.sdo.n + (int64_t)head * a.sdo.h) / u16);
            const int64_t at = ((int64_t)b * a.Hq + head) * a.Nq + token;
            row_statistics(a, at, ref, weight);
            de = a.delta[at];
          }
        }
        tab[r] = where;
        refs[r] = ref;
        weights[r] = weight * PScale<T>::up;                     // not into ref, which may be too large to take it
        delta[r] = de;
      }
      __syncthreads();
      u32x2 x[P::NU];                                            // where the rows of the next tile lie, read a tile before they are asked for
      auto locate = [&](int t) {
#pragma unroll
        for (int u = 0; u < P::NU; ++u) x[u] = tab[min(t, kBatch / TR - 1) * TR + (P::whole ? P::row(u) : min(P::row(u), TR - 1))];
      };
      auto issue = [&](int t) {
        char *qd = smem + (t % NB) * 2 * F::img, *dd = qd + F::img;
        const char *zero = reinterpret_cast<const char *>(g_zero_chunk);
#pragma unroll
        for (int u = 0; u < P::NU; ++u)
          if (P::any(u, wave)) {
            const bool in = x[u].x != ~0u;
            const char *p = in ? qb + ((uint64_t)x[u].x + P::chunk(u)) * 16 : zero, *q = in ? db + ((uint64_t)x[u].y + P::chunk(u)) * 16 : zero;
            if (P::chunk(u) < chunks) {
              dma16(p, P::dst(qd, u, wave));
              dma16(q, P::dst(dd, u, wave));
            }
          }
      };
#pragma unroll
      for (int t = 0; t < NB - 1; ++t)
        if (t < nt) {
          locate(t);
          issue(t);
        }
      locate(NB - 1);
      if (fresh) {
        fresh = false;
        seen = key < a.Nk && see > 0.5f;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool in = seen && c * 32 + g * 8 < a.D;
            kf[c][e] = in ? kf[c][e] : (T)0.f;
            vf[c][e] = in ? vf[c][e] : (T)0.f;
          }
      }
      for (int t = 0; t < nt; ++t) {
        // tile t is there (the NB - 2 behind it may be on their way) and tile t - 1, whose place tile t + NB - 1 takes, has been read
        if (NB == 4 && t + 2 < nt) tile_barrier<NB == 4 ? 2 * PER : 0>();
        else if (NB == 4 && t + 1 < nt) tile_barrier<NB == 4 ? PER : 0>();
        else tile_barrier<0>();
        const char *qrows = smem + (t % NB) * 2 * F::img, *drows = qrows + F::img;
        constexpr bool ahead = sizeof(T) == 2 || DP <= 64;        // all fragments before the first product (fp32: registers for 64 channels)
        frag qf[2][KC], df[2][KC];
        if constexpr (ahead) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int c = 0; c < KC; ++c) {
              qf[u][c] = row_frag<T, DP>(qrows, u * 16 + col, c * 32 + g * 8);
              df[u][c] = row_frag<T, DP>(drows, u * 16 + col, c * 32 + g * 8);
            }
        }
        f32x4 ref[2], we[2], de[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          ref[u] = *reinterpret_cast<const f32x4 *>(refs + t * TR + u * 16 + g * 4);
          we[u] = *reinterpret_cast<const f32x4 *>(weights + t * TR + u * 16 + g * 4);
          de[u] = *reinterpret_cast<const f32x4 *>(delta + t * TR + u * 16 + g * 4);
        }
        if constexpr (ahead) __builtin_amdgcn_sched_barrier(0);
        f32x4 sc[2], dp[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          sc[u] = dp[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            sc[u] = mma(ahead ? qf[u][c] : row_frag<T, DP>(qrows, u * 16 + col, c * 32 + g * 8), kf[c], sc[u]);
            dp[u] = mma(ahead ? df[u][c] : row_frag<T, DP>(drows, u * 16 + col, c * 32 + g * 8), vf[c], dp[u]);
          }
        }
        constexpr int AH = ahead ? DT / 2 : 1;
        frag da[AH], qa[AH];
#pragma unroll
        for (int d = 0; d < AH; ++d) {
          da[d] = col_frag<T, DP>(drows, 0, d * 16, lane);
          qa[d] = col_frag<T, DP>(qrows, 0, d * 16, lane);
        }
        __builtin_amdgcn_sched_barrier(0);
        frag pf, gf, pl, gl;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f(fmaf(sc[u][e], a.c, -ref[u][e])) * we[u][e];
            dp[u][e] = p * (dp[u][e] - de[u][e]);
            if constexpr (GradRange<T>::on) dp[u][e] *= range;
            pf[u * 4 + e] = (T)p;
            if constexpr (TWO) pl[u * 4 + e] = (T)(p - (float)pf[u * 4 + e]);
          }
        if constexpr (GradRange<T>::on) fit_range<16>(dp, range, gk);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            gf[u * 4 + e] = (T)dp[u][e];
            if constexpr (TWO) gl[u * 4 + e] = (T)(dp[u][e] - (float)gf[u * 4 + e]);
          }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const frag x = da[d % AH], y = qa[d % AH];
          if (d + AH < DT) {
            da[d % AH] = col_frag<T, DP>(drows, 0, (d + AH) * 16, lane);
            qa[d % AH] = col_frag<T, DP>(qrows, 0, (d + AH) * 16, lane);
          } else if (d + AH == DT) {                             // behind the transposing reads, as in the forward
            if (t + NB - 1 < nt) issue(t + NB - 1);
            locate(t + NB);
          }
          gv[d] = mma(x, pf, gv[d]);
          gk[d] = mma(y, gf, gk[d]);
          if constexpr (TWO) {
            gv[d] = mma(x, pl, gv[d]);
            gk[d] = mma(y, gl, gk[d]);
          }
        }
      }
    }
  }
  put();
}

// Adds the parts of split rows up, in the order of the rows: a thread has 4 channels of one key.
template <typename T>
__global__ __launch_bounds__(256) void attend_add_kernel(AttnArgs a) {
  const int64_t per = (int64_t)a.B * a.Hkv * a.Nk * (a.D / 4), id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= 2 * per) return;
  const int which = id >= per;
  const int64_t at = id - which * per;
  T *out = reinterpret_cast<T *>(which ? a.dv : a.dk);
  if (out == nullptr) return;
  const float *p = a.part + (int64_t)which * a.splits * per * 4 + at * 4;
  f32x4 sum = *reinterpret_cast<const f32x4 *>(p);
  for (int i = 1; i < a.splits; ++i) sum += *reinterpret_cast<const f32x4 *>(p + i * per * 4);
  const int64_t row = at / (a.D / 4);
  const int ch = (int)(at - row * (a.D / 4)) * 4, key = (int)(row % a.Nk), bh = (int)(row / a.Nk);
  const Str st = which ? a.sdv : a.sdk;
  typename Vec4<T>::type y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (T)sum[e];
  *reinterpret_cast<typename Vec4<T>::type *>(out + (int64_t)(bh / a.Hkv) * st.b + (int64_t)key * st.n + (int64_t)(bh % a.Hkv) * st.h + ch) = y;
}

// ------------------------------------------------------------------------------------------ host
// Tile shapes.  16-bit: 64 rows x 64 keys as 2 x 2 waves of 32 x 32 (every LDS fragment feeds two products); fp32, whose products take 16
// times as long per fragment: 64 rows x 32 keys as 4 x 1 waves of 16 x 32.  Groups of up to 16 rows (one token of a few heads) have a
// kernel of their own: half of the second product's k-elements stay empty there, but such calls wait for memory.
constexpr int kFewRows = 16;
static int fwd_rows(const AttnArgs &a) { return a.rows <= kFewRows ? 16 : 64; }
static int fwd_keys(const AttnArgs &a, bool f32) { return a.rows > kFewRows && f32 ? 32 : 64; }

static size_t list_bytes(const AttnArgs &a) { return (size_t)a.cap * 4 + (size_t)(a.nb + 31) / 32 * 4; }

template <typename K> static int launch(K kernel, size_t lds, int64_t blocks, const AttnArgs &a, hipStream_t s, const char *what) {
  TCL_REQUIRE(blocks < (1LL << 31), TCL_ERR_SHAPE, "%s: grid of %ld blocks", what, (long)blocks);
  TCL_REQUIRE(lds_ready((const void *)kernel, lds), TCL_ERR_LAUNCH, "%s: the device refuses %zu bytes of LDS", what, lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), lds, s, a);
  return check_launch(what);
}
template <typename T, int DP, bool LO> static int launch_fwd(const AttnArgs &a, int64_t blocks, hipStream_t s) {
  const char *what = "block_attention";
  if (a.rows <= kFewRows) return launch(attend_few_kernel<T, DP, (sizeof(T) == 4 && DP > 64 ? 2 : 4), LO>, FewTile<T, DP>::body + list_bytes(a), blocks, a, s, what);
  if constexpr (sizeof(T) == 4) return launch(attend_fwd_kernel<T, DP, 16, 4, 1, 2, LO>, FwdTile<T, DP, 16, 4, 1, 2>::body + list_bytes(a), blocks, a, s, what);
  else return launch(attend_fwd_kernel<T, DP, 32, 2, 2, 1, LO>, FwdTile<T, DP, 32, 2, 2, 1>::body + list_bytes(a), blocks, a, s, what);
}
template <typename T, int DP, bool TWO> static int launch_dq(AttnArgs a, hipStream_t s) {
  const char *what = "block_attention backward (queries)";
  const bool few = a.rows <= 32;
  a.chunks = (int)cdiv(a.rows, few ? 32 : 64);
  const int64_t blocks = (int64_t)a.B * a.Hkv * a.S * a.chunks;
  if (few) return launch(attend_dq_kernel<T, DP, 16, 2, 2, 1, TWO>, DqTile<T, DP, 16, 2, 2>::body + list_bytes(a), blocks, a, s, what);
  if constexpr (sizeof(T) == 4) return launch(attend_dq_kernel<T, DP, 16, 4, 1, 1, TWO>, DqTile<T, DP, 16, 4, 1>::body + list_bytes(a), blocks, a, s, what);
  else return launch(attend_dq_kernel<T, DP, 32, 2, 2, 2, TWO>, DqTile<T, DP, 32, 2, 2>::body + list_bytes(a), blocks, a, s, what);
}
// Key tiles, and the splits of the rows each of them sums where there are too few tiles for the GPU: a batch of rows each at least.  The rows are
// those of all groups (a key can be chosen by every one).  A training step of 2,000
// queries x 16 heads against 200 keys of 2 heads of 64 fp32 channels 1,350 -> 141 us, bf16 350 -> 95 (the host's time).
static int64_t dkv_tiles(const AttnArgs &a) { return ((int64_t)a.nb << (a.lb - 6)) * a.B * a.Hkv; }
static int dkv_splits(const AttnArgs &a) {
  const int64_t tiles = dkv_tiles(a), rows = (int64_t)a.S * a.rows;
  int64_t n = cdiv(2 * kNumCU, tiles > 0 ? tiles : 1);
  if (n > rows / kBatch) n = rows / kBatch;
  return (int)(n < 1 ? 1 : n > 32 ? 32 : n);
}
static size_t dkv_part(const AttnArgs &a) {
  const int n = dkv_splits(a);
  return n > 1 ? round_up((size_t)2 * n * a.B * a.Hkv * a.Nk * a.D * 4, 256) : 0;
}
template <typename T, int DP, bool TWO> static int launch_dkv(const AttnArgs &a, hipStream_t s) {
  const char *what = "block_attention backward (keys)";
  const int64_t blocks = dkv_tiles(a) * a.splits;
  const int r = launch(attend_dkv_kernel<T, DP, TWO>, DkvTile<T, DP>::bytes, blocks, a, s, what);
  if (r != TCL_OK || a.splits == 1) return r;
  const int64_t adds = cdiv((int64_t)a.B * a.Hkv * a.Nk * (a.D / 4) * 2, 256);
  hipLaunchKernelGGL((attend_add_kernel<T>), dim3((unsigned)adds), dim3(256), 0, s, a);   // few keys: far below 2^31
  return check_launch(what);
}

// head sizes are padded to a multiple of 32 in LDS and registers
#define TCL_BY_DIM(T, CALL)                                       \
  switch ((a.D + 31) / 32) {                                      \
    case 1: return CALL(T, 32);                                   \
    case 2: return CALL(T, 64);                                   \
    case 3: return CALL(T, 96);                                   \
    default: return CALL(T, 128);                                 \
  }
template <typename T> static int fwd_by_dim(const AttnArgs &a, int64_t blocks, hipStream_t s) {
#define CALL(T, DP) (sizeof(T) == 2 && a.lo ? launch_fwd<T, DP, sizeof(T) == 2>(a, blocks, s) : launch_fwd<T, DP, false>(a, blocks, s))
  TCL_BY_DIM(T, CALL)
#undef CALL
}
// a head of up to 32 channels is always taken in two parts, fp32 never
template <typename T> static int dq_by_dim(const AttnArgs &a, hipStream_t s) {
#define CALL(T, DP) (DP == 32 || two_parts<T>(a) ? launch_dq<T, DP, sizeof(T) == 2>(a, s) : launch_dq<T, DP, sizeof(T) == 2 && DP == 32>(a, s))
  TCL_BY_DIM(T, CALL)
#undef CALL
}
template <typename T> static int dkv_by_dim(const AttnArgs &a, hipStream_t s) {
#define CALL(T, DP) (DP == 32 || two_parts<T>(a) ? launch_dkv<T, DP, sizeof(T) == 2>(a, s) : launch_dkv<T, DP, sizeof(T) == 2 && DP == 32>(a, s))
  TCL_BY_DIM(T, CALL)
#undef CALL
}

// shapes, limits and derived sizes shared by both directions
static int attn_setup(AttnArgs &a, int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D, int64_t top_k, int64_t block, int64_t q_block,
                      double scale, int dtype) {
  TCL_REQUIRE(B >= 0 && Nq >= 0 && Nk >= 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && top_k > 0 && q_block > 0, TCL_ERR_SHAPE, "block_attention: bad shape");
  TCL_REQUIRE(B < (1LL << 24) && Nq < (1LL << 30) && Hq < (1LL << 16), TCL_ERR_SHAPE, "block_attention: bad shape");
  TCL_REQUIRE(D > 0 && D % 8 == 0 && D <= 128, TCL_ERR_UNSUPPORTED, "block_attention: head size %ld (a multiple of 8 up to 128)", (long)D);
  TCL_REQUIRE(block == 64 || block == 128, TCL_ERR_UNSUPPORTED, "block_attention: blocks of 64 or 128 keys (got %ld)", (long)block);
  TCL_REQUIRE(top_k <= kMaxTop, TCL_ERR_UNSUPPORTED, "block_attention: %ld blocks per group (at most %ld)", (long)top_k, (long)kMaxTop);
  TCL_REQUIRE(cdiv(Nk, block) <= kMaxKeyBlocks, TCL_ERR_UNSUPPORTED, "block_attention: %ld keys (at most %ld blocks)", (long)Nk, (long)kMaxKeyBlocks);
  TCL_REQUIRE(dtype == TCL_DT_F32 || dtype == TCL_DT_BF16 || dtype == TCL_DT_F16, TCL_ERR_UNSUPPORTED, "block_attention: unknown dtype %d", dtype);
  TCL_REQUIRE(isfinite((float)(scale * 1.4426950408889634074)), TCL_ERR_ARG, "block_attention: scale %g", scale);
  if (q_block > Nq) q_block = Nq > 0 ? Nq : 1;
  TCL_REQUIRE(q_block * (Hq / Hkv) <= kMaxRows, TCL_ERR_UNSUPPORTED, "block_attention: groups of %ld query rows (at most %ld)", (long)(q_block * (Hq / Hkv)), (long)kMaxRows);
  a.B = (int)B; a.Nq = (int)Nq; a.Nk = (int)Nk; a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.G = (int)(Hq / Hkv); a.D = (int)D;
  a.top = (int)top_k; a.nb = (int)cdiv(Nk, block); a.lb = block == 64 ? 6 : 7; a.q_block = (int)q_block;
  a.S = (int)cdiv(Nq, q_block);
  a.rows = (int)(q_block * a.G);
  a.cap = a.top < a.nb ? a.top : a.nb;
  a.words = (int)cdiv(a.S, 32);
  a.by_g = make_fastdiv((uint32_t)a.G);
  a.by_rows = make_fastdiv((uint32_t)a.rows);
  a.by_d4 = make_fastdiv((uint32_t)(a.D / 4));
  a.scale = (float)scale;
  a.c = (float)(scale * 1.4426950408889634074);
  a.chunks = 1;
  a.splits = 1;
  return TCL_OK;
}

// Splits of the keys of a forward work item: enough workgroups for two per CU, two tiles each at least.
struct FwdPlan { int chunks, splits; int64_t works; size_t part; };
static FwdPlan fwd_plan(const AttnArgs &a, bool f32) {
  FwdPlan p;
  p.chunks = (int)cdiv(a.rows, fwd_rows(a));
  p.works = (int64_t)a.B * a.Hkv * a.S * p.chunks;
  const int64_t tiles = cdiv((int64_t)a.cap << a.lb, fwd_keys(a, f32));
  int64_t n = cdiv(2 * kNumCU, p.works > 0 ? p.works : 1);
  if (n > tiles / 2) n = tiles / 2;
  p.splits = (int)(n < 1 ? 1 : n > kMaxSplits ? kMaxSplits : n);
  p.part = p.splits > 1 ? round_up((size_t)p.works * p.splits * fwd_rows(a) * (a.D + 3) * 4, 256) : 0;
  return p;
}
static bool rows16(const void *p, const Str &s, int dtype) {
  const int64_t ve = dtype == TCL_DT_F32 ? 4 : 8;
  return aligned(p, 16) && s.b % ve == 0 && s.n % ve == 0 && s.h % ve == 0;
}
static void statistics_behind(AttnArgs &a) {
  const int64_t rows = (int64_t)a.B * a.Hq * a.Nq;
  a.ref = a.lse + rows;
  a.weight = a.ref + rows;
}
// the rows of a block are addressed by 32-bit byte offsets from its first
static bool near_rows(const Str &s) { return s.n >= 0 && s.n < (1LL << 22); }
// the query rows of a batch item by 32-bit counts of 16 bytes
static bool near_batch(const Str &s, const AttnArgs &a, int dtype) {
  const int64_t last = (int64_t)(a.Nq - 1) * s.n + (int64_t)(a.Hq - 1) * s.h;
  return s.n >= 0 && s.h >= 0 && s.n < (1LL << 31) && s.h < (1LL << 31) && last / (dtype == TCL_DT_F32 ? 4 : 8) < (1LL << 32) - 64;
}

}  // namespace tcl

using namespace tcl;

extern "C" size_t tcl_block_attention_fwd_workspace_bytes(int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D, int64_t top_k, int64_t block,
                                                          int64_t q_block) {
  AttnArgs a{};
  if (attn_setup(a, B, Nq, Nk, Hq, Hkv, D, top_k, block, q_block, 1.0, TCL_DT_F32) != TCL_OK) return 0;
  const FwdPlan p = fwd_plan(a, true), q = fwd_plan(a, false);   // either type's
  return p.part > q.part ? p.part : q.part;
}

extern "C" int tcl_block_attention_fwd(const void *q, int64_t q_sb, int64_t q_sn, int64_t q_sh, const void *k, int64_t k_sb, int64_t k_sn, int64_t k_sh,
                                       const void *v, int64_t v_sb, int64_t v_sn, int64_t v_sh, const float *visible, const int32_t *blocks,
                                       void *out, int64_t o_sb, int64_t o_sn, int64_t o_sh, void *out_lo, float *lse,
                                       int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D, int64_t top_k, int64_t block, int64_t q_block,
                                       double scale, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  AttnArgs a{};
  const bool statistics = dtype & TCL_DT_STATISTICS;
  dtype &= ~TCL_DT_STATISTICS;
  const int rc = attn_setup(a, B, Nq, Nk, Hq, Hkv, D, top_k, block, q_block, scale, dtype);
  if (rc != TCL_OK) return rc;
  if (B == 0 || Nq == 0) return TCL_OK;
  TCL_REQUIRE(q && out && blocks && (Nk == 0 || (k && v)), TCL_ERR_ARG, "block_attention: null pointer");
  a.q = q; a.k = k; a.v = v; a.vis = visible; a.blocks = blocks; a.out = out; a.lo = out_lo; a.lse = lse;
  if (statistics && lse) statistics_behind(a);
  a.sq = Str{q_sb, q_sn, q_sh}; a.sk = Str{k_sb, k_sn, k_sh}; a.sv = Str{v_sb, v_sn, v_sh}; a.so = Str{o_sb, o_sn, o_sh};
  TCL_REQUIRE(rows16(q, a.sq, dtype) && (Nk == 0 || (rows16(k, a.sk, dtype) && rows16(v, a.sv, dtype))) && rows16(out, a.so, dtype) && aligned(out_lo, 16), TCL_ERR_ARG,
              "block_attention: rows must start on 16 bytes");
  TCL_REQUIRE(near_rows(a.sk) && near_rows(a.sv), TCL_ERR_UNSUPPORTED, "block_attention: keys lie more than 2^22 elements apart");
  const bool f32 = dtype == TCL_DT_F32;
  const FwdPlan plan = fwd_plan(a, f32);
  a.chunks = plan.chunks;
  a.splits = plan.splits;
  const int64_t blocks_n = plan.works * a.splits;
  TCL_REQUIRE(plan.part == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= plan.part), TCL_ERR_WORKSPACE, "block_attention: workspace of %zu bytes needed", plan.part);
  a.part = (float *)workspace;
  const hipStream_t s = (hipStream_t)stream;
  const int r = dtype == TCL_DT_F32 ? fwd_by_dim<float>(a, blocks_n, s) : dtype == TCL_DT_BF16 ? fwd_by_dim<__bf16>(a, blocks_n, s) : fwd_by_dim<_Float16>(a, blocks_n, s);
  if (r != TCL_OK || a.splits == 1) return r;
  const int M = fwd_rows(a);
  TCL_REQUIRE(plan.works * M < (1LL << 31), TCL_ERR_SHAPE, "block_attention: too many rows for one call");
  const dim3 grid((unsigned)(plan.works * M));
  if (dtype == TCL_DT_F32) hipLaunchKernelGGL((attend_join_kernel<float>), grid, dim3(256), 0, s, a, M);
  else if (dtype == TCL_DT_BF16) hipLaunchKernelGGL((attend_join_kernel<__bf16>), grid, dim3(256), 0, s, a, M);
  else hipLaunchKernelGGL((attend_join_kernel<_Float16>), grid, dim3(256), 0, s, a, M);
  return check_launch("block_attention (join)");
}

extern "C" size_t tcl_block_attention_bwd_workspace_bytes(int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D, int64_t top_k, int64_t block,
                                                          int64_t q_block) {
  AttnArgs a{};
  if (attn_setup(a, B, Nq, Nk, Hq, Hkv, D, top_k, block, q_block, 1.0, TCL_DT_F32) != TCL_OK) return 256;
  return round_up((size_t)B * Hq * Nq * 4, 256) + round_up((size_t)B * Hkv * a.nb * (a.words + 1) * 4, 256) + round_up((size_t)B * Hkv * a.nb * 4, 256) + 256 +
         dkv_part(a);
}

extern "C" int tcl_block_attention_bwd(const void *grad_out, int64_t g_sb, int64_t g_sn, int64_t g_sh, const void *q, int64_t q_sb, int64_t q_sn, int64_t q_sh,
                                       const void *k, int64_t k_sb, int64_t k_sn, int64_t k_sh, const void *v, int64_t v_sb, int64_t v_sn, int64_t v_sh,
                                       const float *visible, const int32_t *blocks, const void *out, int64_t o_sb, int64_t o_sn, int64_t o_sh, const void *out_lo,
                                       const float *lse,
                                       void *g_q, int64_t gq_sb, int64_t gq_sn, int64_t gq_sh, void *g_k, int64_t gk_sb, int64_t gk_sn, int64_t gk_sh,
                                       void *g_v, int64_t gv_sb, int64_t gv_sn, int64_t gv_sh,
                                       int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D, int64_t top_k, int64_t block, int64_t q_block,
                                       double scale, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  AttnArgs a{};
  const bool statistics = dtype & TCL_DT_STATISTICS;
  dtype &= ~TCL_DT_STATISTICS;
  const int rc = attn_setup(a, B, Nq, Nk, Hq, Hkv, D, top_k, block, q_block, scale, dtype);
  if (rc != TCL_OK) return rc;
  if (B == 0 || Nq == 0 || Nk == 0) return TCL_OK;             // the caller zeroes gradients of an empty attention
  TCL_REQUIRE(grad_out && q && k && v && out && blocks && lse, TCL_ERR_ARG, "block_attention backward: null pointer");
  a.q = q; a.k = k; a.v = v; a.dout = grad_out; a.vis = visible; a.blocks = blocks; a.out = const_cast<void *>(out); a.lo = const_cast<void *>(out_lo); a.lse = const_cast<float *>(lse);
  if (statistics) statistics_behind(a);
  a.dq = g_q; a.dk = g_k; a.dv = g_v;
  a.sq = Str{q_sb, q_sn, q_sh}; a.sk = Str{k_sb, k_sn, k_sh}; a.sv = Str{v_sb, v_sn, v_sh}; a.so = Str{o_sb, o_sn, o_sh}; a.sdo = Str{g_sb, g_sn, g_sh};
  a.sdq = Str{gq_sb, gq_sn, gq_sh}; a.sdk = Str{gk_sb, gk_sn, gk_sh}; a.sdv = Str{gv_sb, gv_sn, gv_sh};
  TCL_REQUIRE(rows16(q, a.sq, dtype) && rows16(k, a.sk, dtype) && rows16(v, a.sv, dtype) && rows16(out, a.so, dtype) && rows16(grad_out, a.sdo, dtype) && aligned(out_lo, 16) &&
              (!g_q || rows16(g_q, a.sdq, dtype)) && (!g_k || rows16(g_k, a.sdk, dtype)) && (!g_v || rows16(g_v, a.sdv, dtype)), TCL_ERR_ARG,
              "block_attention backward: rows must start on 16 bytes");
  TCL_REQUIRE(near_rows(a.sk) && near_rows(a.sv), TCL_ERR_UNSUPPORTED, "block_attention backward: keys lie more than 2^22 elements apart");
  TCL_REQUIRE(near_batch(a.sq, a, dtype) && near_batch(a.sdo, a, dtype), TCL_ERR_UNSUPPORTED, "block_attention backward: the query rows of a batch item span more than 64 GB");
  const size_t need = tcl_block_attention_bwd_workspace_bytes(B, Nq, Nk, Hq, Hkv, D, top_k, block, q_block);
  TCL_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= need, TCL_ERR_WORKSPACE, "block_attention backward: workspace of %zu bytes needed", need);
  a.delta = (float *)workspace;
  a.inv = (uint32_t *)((char *)workspace + round_up((size_t)B * Hq * Nq * 4, 256));
  const hipStream_t s = (hipStream_t)stream;
  const int64_t bh = B * Hkv, dblocks = cdiv(B * Nq * Hq, 16), sel_n = bh * a.S * a.top;
  a.plan_words = g_k || g_v ? bh * a.nb * (a.words + 1) : 0;
  a.chosen = a.inv + bh * a.nb * a.words;
  a.order = (int32_t *)((char *)a.inv + round_up((size_t)bh * a.nb * (a.words + 1) * 4, 256));
  a.part = (float *)((char *)a.order + round_up((size_t)bh * a.nb * 4, 256));
  TCL_REQUIRE(dblocks < (1LL << 31) && cdiv(sel_n, 256) < (1LL << 31) && bh < (1LL << 31), TCL_ERR_SHAPE, "block_attention backward: too many rows for one call");
  if (dtype == TCL_DT_F32) hipLaunchKernelGGL((attend_delta_kernel<float>), dim3((unsigned)dblocks), dim3(256), 0, s, a);
  else if (dtype == TCL_DT_BF16) hipLaunchKernelGGL((attend_delta_kernel<__bf16>), dim3((unsigned)dblocks), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((attend_delta_kernel<_Float16>), dim3((unsigned)dblocks), dim3(256), 0, s, a);
  if (g_q) {
    const int r = dtype == TCL_DT_F32 ? dq_by_dim<float>(a, s) : dtype == TCL_DT_BF16 ? dq_by_dim<__bf16>(a, s) : dq_by_dim<_Float16>(a, s);
    if (r != TCL_OK) return r;
  }
  if (!g_k && !g_v) return check_launch("block_attention backward");
  hipLaunchKernelGGL(attend_invert_kernel, dim3((unsigned)cdiv(sel_n, 256)), dim3(256), 0, s, a);
  hipLaunchKernelGGL(attend_order_kernel, dim3((unsigned)bh), dim3(1024), 0, s, a);
  a.splits = dkv_splits(a);
  return dtype == TCL_DT_F32 ? dkv_by_dim<float>(a, s) : dtype == TCL_DT_BF16 ? dkv_by_dim<__bf16>(a, s) : dkv_by_dim<_Float16>(a, s);
}
