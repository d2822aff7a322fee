// Rotary positions over several axes (time, height, width, ...): tcl_rotate_positions.
//
// The channels of a head are cut into one section per axis.  Pair i of a section of d channels turns by the angle
// p_axis * base^(-2 i / d):  (a, b) -> (a cos - b sin, b cos + a sin).  The backward pass is the same with the angle negated.
//
// Bound: memory (each element is read and written once, 3 flops each): 32 x 15,900 tokens of 128 bf16 channels 54 us, 4.9 TB/s, the rate of
// a copy.  A thread owns V pairs of one token and walks the
// heads, so the angle, its reduction and the sine / cosine are paid once per token and pair, not once per head.
//
// Angles: the position times the frequency in TURNS is formed in 64 bits and reduced to [-1/2, 1/2] there (fp32 would be off by
// 0.006 rad at position 100,000 and frequency 1); the fraction goes on in fp32.  fp32 outputs take sincospi (correct to an ulp);
// 16-bit outputs take the hardware's sine / cosine of a fraction of a turn, whose error (about 2^-20 absolute) is far below
// half a step of the result.
#include "tcl_common.h"
#include <math.h>

namespace tcl {

constexpr int kRopeMaxPairs = 128;   // dim <= 256
constexpr int kRopeMaxAxes = 4;
constexpr int kRopeBlocks = kNumCU * 16;   // workgroups of a large call

struct RotateArgs {   // passed by value
  const void *x;
  void *y;
  const void *pos;
  int64_t x_sb, x_sn, x_sh, y_sb, y_sn, y_sh, p_sb;
  int N, H, chunks, heads_per_thread, axes, pos_int, interleaved;
  unsigned rows, threads, step;        // B * N; threads at work: step tokens x chunks
  FastDiv by_chunks, by_n;
  float sign;
  // per pair: frequency in turns (0 = the channels pass through), axis, channel of the first and the second half
  double turns[kRopeMaxPairs];
  uint8_t axis[kRopeMaxPairs];
  uint8_t first[kRopeMaxPairs], second[kRopeMaxPairs];
};

template <typename T, int V> struct RopeVec { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T> struct RopeVec<T, 1> { typedef T type; };

template <typename T, int V> __device__ __forceinline__ void rope_ld(const T *p, float *o) {
  typedef typename RopeVec<T, V>::type vec;
  const vec t = *reinterpret_cast<const vec *>(p);
  if constexpr (V == 1) o[0] = (float)t;
  else {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = (float)t[i];
  }
}
template <typename T, int V> __device__ __forceinline__ void rope_st(T *p, const float *o) {
  typedef typename RopeVec<T, V>::type vec;
  vec t;
  if constexpr (V == 1) t = (T)o[0];
  else {
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = (T)o[i];
  }
  *reinterpret_cast<vec *>(p) = t;
}

// V pairs per thread.  IL: a pair is two neighbouring channels (2 V consecutive elements: one access, two where they pass 16
// bytes or nothing is known of their alignment, V = 1); otherwise the two halves of a section (V elements in each).
// A thread keeps its pairs and walks tokens `step` apart, so frequencies and channel numbers are read once.
template <typename T, int V, bool IL>
__global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a) {
  const unsigned id = blockIdx.x * 256 + threadIdx.x;
  if (id >= a.threads) return;
  const unsigned row0 = a.by_chunks.div(id);                     // item * N + token (host: < 2^31)
  const int c = (int)(id - row0 * (unsigned)a.chunks);
  double f[V];
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = a.turns[c * V + i];
  const bool turn = f[0] != 0.0;                                 // a chunk lies within one section
  const int axis = a.axis[c * V], o0 = a.first[c * V], o1 = a.second[c * V];
  const int h0 = blockIdx.y * a.heads_per_thread, h1 = min(a.H, h0 + a.heads_per_thread);
  constexpr int W = IL && V > 1 && 2 * V * sizeof(T) <= 16 ? 2 * V : V;   // elements of one access
  for (unsigned row = row0; row < a.rows; row += a.step) {
    const unsigned b = a.by_n.div(row), n = row - b * (unsigned)a.N;
    const int64_t at = (int64_t)b * a.p_sb + (int64_t)n * a.axes + axis;
    const double p = a.pos_int ? (double)reinterpret_cast<const int32_t *>(a.pos)[at] : (double)reinterpret_cast<const float *>(a.pos)[at];
    const T *x = reinterpret_cast<const T *>(a.x) + (int64_t)b * a.x_sb + (int64_t)n * a.x_sn;
    T *y = reinterpret_cast<T *>(a.y) + (int64_t)b * a.y_sb + (int64_t)n * a.y_sn;
    float cs[V], sn[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const double w = p * f[i];
      const float r = (float)(w - rint(w));                       // fraction of a turn
      if (sizeof(T) == 4) sincospif(2.f * r, &sn[i], &cs[i]);
      else { sn[i] = __builtin_amdgcn_sinf(r); cs[i] = __builtin_amdgcn_cosf(r); }
      sn[i] *= a.sign;
    }
    for (int h = h0; h < h1; ++h) {
      float u[2 * V], r[2 * V];
      const T *xp = x + (int64_t)h * a.x_sh;
      T *yp = y + (int64_t)h * a.y_sh;
      rope_ld<T, W>(xp + o0, u);
      if (W == V) rope_ld<T, V>(xp + (IL ? o0 + V : o1), u + V);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int ia = IL ? 2 * i : i, ib = IL ? 2 * i + 1 : V + i;
        const float p = u[ia], q = u[ib];
        r[ia] = turn ? p * cs[i] - q * sn[i] : p;
        r[ib] = turn ? q * cs[i] + p * sn[i] : q;
      }
      rope_st<T, W>(yp + o0, r);
      if (W == V) rope_st<T, V>(yp + (IL ? o0 + V : o1), r + V);
    }
  }
}

template <typename T, int V> static void rotate_launch_v(const RotateArgs &a, dim3 grid, hipStream_t s) {
  if (a.interleaved) hipLaunchKernelGGL((rotate_kernel<T, V, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((rotate_kernel<T, V, false>), grid, dim3(256), 0, s, a);
}

template <typename T> static int rotate_launch(RotateArgs &a, int64_t B, int pairs, int64_t unit, hipStream_t s) {
  // pairs per thread: the widest power of two (up to a 16-byte access) whose elements divide `unit`
  int V = sizeof(T) == 4 ? 4 : 8;
  while (V > 1 && unit % (a.interleaved ? 2 * V : V)) V /= 2;
  a.chunks = pairs / V;
  TCL_REQUIRE(B * a.N < (1LL << 31), TCL_ERR_SHAPE, "rotate_positions: %ld tokens are too many for one call", (long)(B * a.N));
  a.rows = (unsigned)(B * a.N);
  a.by_chunks = make_fastdiv((uint32_t)a.chunks);
  a.by_n = make_fastdiv((uint32_t)a.N);
  // All heads of a token share the angles, but a small call is split over the heads until it fills the CUs; a large one gives every
  // thread several tokens (the frequencies are then read once for them)
  const int64_t all = cdiv((int64_t)a.rows * a.chunks, 256);
  int groups = (int)(all >= kNumCU * 4 ? 1 : cdiv(kNumCU * 4, all));
  if (groups > a.H) groups = a.H;
  a.heads_per_thread = (int)cdiv(a.H, groups);
  const int64_t blocks = all < kRopeBlocks ? all : kRopeBlocks;
  a.step = (unsigned)(blocks * 256 / a.chunks);
  a.threads = a.step * (unsigned)a.chunks;
  const dim3 grid((unsigned)blocks, (unsigned)cdiv(a.H, a.heads_per_thread));
  switch (V) {
    case 8: if constexpr (sizeof(T) == 2) rotate_launch_v<T, 8>(a, grid, s); break;
    case 4: rotate_launch_v<T, 4>(a, grid, s); break;
    case 2: rotate_launch_v<T, 2>(a, grid, s); break;
    default: rotate_launch_v<T, 1>(a, grid, s); break;
  }
  return check_launch("rotate_positions");
}

static int64_t gcd64(int64_t a, int64_t b) { while (b) { const int64_t t = a % b; a = b; b = t; } return a < 0 ? -a : a; }

}  // namespace tcl

using namespace tcl;

extern "C" int tcl_rotate_positions(const void *x, int64_t x_sb, int64_t x_sn, int64_t x_sh, const void *positions, int positions_int32, int64_t p_sb,
                                    void *y, int64_t y_sb, int64_t y_sn, int64_t y_sh, int64_t B, int64_t N, int64_t H, int64_t D,
                                    const int32_t *sections, int64_t n_sections, double base, int interleaved, int inverse, int dtype, void *stream) {
  TCL_REQUIRE(B >= 0 && N >= 0 && H > 0 && D > 0 && B < (1LL << 31) && N < (1LL << 31) && H < (1LL << 31), TCL_ERR_SHAPE, "rotate_positions: bad shape");
  TCL_REQUIRE(D % 2 == 0 && D <= 2 * kRopeMaxPairs, TCL_ERR_UNSUPPORTED, "rotate_positions: head size %ld (even, up to %d)", (long)D, 2 * kRopeMaxPairs);
  TCL_REQUIRE(sections && n_sections >= 1 && n_sections <= kRopeMaxAxes, TCL_ERR_ARG, "rotate_positions: 1 to %d axes", kRopeMaxAxes);
  TCL_REQUIRE(base > 0.0 && isfinite(base), TCL_ERR_ARG, "rotate_positions: base must be positive");
  TCL_REQUIRE(dtype == TCL_DT_F32 || dtype == TCL_DT_BF16 || dtype == TCL_DT_F16, TCL_ERR_UNSUPPORTED, "rotate_positions: unknown dtype %d", dtype);
  RotateArgs a;
  int64_t at = 0, unit = 0;   // unit: what section offsets, halves, strides and addresses (in elements) are all multiples of
  int pairs = 0;
  for (int64_t s = 0; s < n_sections; ++s) {
    const int64_t d = sections[s];
    TCL_REQUIRE(d >= 0 && d % 2 == 0 && at + d <= D, TCL_ERR_SHAPE, "rotate_positions: section %ld has %ld channels (even, in all at most %ld)", (long)s, (long)d, (long)D);
    for (int64_t i = 0; i < d / 2; ++i, ++pairs) {
      a.turns[pairs] = pow(base, -2.0 * (double)i / (double)d) / 6.283185307179586476925286766559;
      a.axis[pairs] = (uint8_t)s;
      a.first[pairs] = (uint8_t)(interleaved ? at + 2 * i : at + i);
      a.second[pairs] = (uint8_t)(interleaved ? at + 2 * i + 1 : at + d / 2 + i);
    }
    unit = gcd64(unit, interleaved ? d : gcd64(at, d / 2));
    at += d;
  }
  // channels behind the last section pass through: two halves that a frequency of zero leaves alone
  const int64_t rest = D - at;
  for (int64_t i = 0; i < rest / 2; ++i, ++pairs) {
    a.turns[pairs] = 0.0;
    a.axis[pairs] = 0;
    a.first[pairs] = (uint8_t)(interleaved ? at + 2 * i : at + i);
    a.second[pairs] = (uint8_t)(interleaved ? at + 2 * i + 1 : at + rest / 2 + i);
  }
  unit = gcd64(unit, interleaved ? rest : gcd64(rest ? at : 0, rest / 2));
  if (B == 0 || N == 0) return TCL_OK;
  TCL_REQUIRE(x && y && positions, TCL_ERR_ARG, "rotate_positions: null pointer");
  const size_t size = dtype == TCL_DT_F32 ? 4 : 2;
  TCL_REQUIRE(aligned(x, size) && aligned(y, size) && aligned(positions, 4), TCL_ERR_ARG, "rotate_positions: misaligned pointer");
  for (int64_t st : {x_sb, x_sn, x_sh, y_sb, y_sn, y_sh}) unit = gcd64(unit, st);
  for (const void *p : {x, (const void *)y}) unit = gcd64(unit, gcd64((int64_t)(reinterpret_cast<uintptr_t>(p) / size % 16), 16));
  a.x = x; a.y = y; a.pos = positions;
  a.x_sb = x_sb; a.x_sn = x_sn; a.x_sh = x_sh;
  a.y_sb = y_sb; a.y_sn = y_sn; a.y_sh = y_sh;
  a.p_sb = p_sb;
  a.N = (int)N; a.H = (int)H; a.axes = (int)n_sections;
  a.pos_int = positions_int32 != 0;
  a.interleaved = interleaved != 0;
  a.sign = inverse ? -1.f : 1.f;
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == TCL_DT_F32) return rotate_launch<float>(a, B, pairs, unit, s);
  if (dtype == TCL_DT_BF16) return rotate_launch<__bf16>(a, B, pairs, unit, s);
  return rotate_launch<_Float16>(a, B, pairs, unit, s);
}
