// Attention of a target's tokens over chosen blocks of reference keys: tcl_block_attention_fwd / _bwd.
//
//   out_q = sum_n softmax_n(scale <q, k_n>) v_n   over the visible keys n of the blocks chosen for q's group
//   (0, and lse = -inf, where nothing is visible).
//
// All products run on the matrix pipe in one shape, 16 x 16 with 32 k-elements per step (one v_mfma_f32_16x16x32 for 16-bit
// operands, eight v_mfma_f32_16x16x4_f32 for fp32): lane l holds row (column) l % 16 of an operand and 8 consecutive
// k-elements of the quarter l / 16; the result has column l % 16 and rows 4 (l / 16) .. + 3.  The order of the k-elements is free
// as long as both operands share it, and that is what keeps the probabilities in registers: S^T = K Q^T leaves a lane 4 + 4
// probabilities of ITS query (two 16-key tiles), which are, as they are, the second operand of O^T = V^T P^T once V^T is read
// in the same key order.  For that V lies in LDS in quads of 4 keys, [key / 4][channel][key % 4].  The backward products use the same
// two forms (rows as they are for contractions over channels, quads for contractions over tokens).
//
// Statistics (running maximum, sum, lse, rowsum(dout o out)) and all accumulators are fp32.  16-bit inputs: the probabilities and the
// score gradients are rounded to the inputs' type as operands of the second product (half a step of it relative to each
// term, the size of the rounding of the result itself); nothing else is rounded before the end.
#include "tcl_common.h"

namespace tcl {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8), aligned(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

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
  void *out, *dq, *dk, *dv;
  float *lse;                      // (B, Hq, Nq), natural logarithm
  float *delta;                    // (B, Hq, Nq)
  uint32_t *inv;                   // (B, Hkv, nb, words): which groups chose the block
  float *part;                     // partial results of split work
  Str sq, sk, sv, so, sdo, sdq, sdk, sdv;
  int B, Nq, Nk, Hq, Hkv, G, D, S, top, nb, lb, q_block, rows, chunks, splits, words, cap;
  float c;                         // scale * log2(e)
  float scale;
  FastDiv by_g, by_rows;
};

// LDS images of a tile of TK token rows x DP channels
template <typename T, int DP> struct Lay {
  static constexpr int VE = 16 / sizeof(T);
  static constexpr int LD = DP + VE;                                  // rows, + 16 bytes: 16 lanes reading 16 bytes each of 16 rows hit every bank once
  static constexpr int QD = 4 * (DP + (sizeof(T) == 2 ? 16 : 0));     // quads of 4 tokens (16-bit: + 128 bytes, so that the two quads of a half wave use different banks)
  static constexpr size_t rows(int tk) { return (size_t)tk * LD * sizeof(T); }
  static constexpr size_t quads(int tk) { return (size_t)tk / 4 * QD * sizeof(T); }
};

// the 8 k-elements of a lane for a contraction over channels
template <typename T, int DP> __device__ __forceinline__ typename Vec8<T>::type row_frag(const T *rows, int row, int ch) {
  return *reinterpret_cast<const typename Vec8<T>::type *>(rows + row * Lay<T, DP>::LD + ch);
}
// ... over the 32 tokens that start at t0: tokens t0 + 4 g .. + 3 and t0 + 16 + 4 g .. + 3 of channel d
template <typename T, int DP> __device__ __forceinline__ typename Vec8<T>::type quad_frag(const T *quads, int t0, int g, int d) {
  typedef typename Vec4<T>::type v4;
  const T *p = quads + (t0 / 4 + g) * Lay<T, DP>::QD + d * 4;
  const v4 a = *reinterpret_cast<const v4 *>(p), b = *reinterpret_cast<const v4 *>(p + 4 * Lay<T, DP>::QD);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A tile's global loads, kept in registers until the barrier that frees the LDS tile: 16-byte pieces of rows
template <typename T, int DP, int TK> struct RowStage {
  typedef T vec __attribute__((ext_vector_type(Lay<T, DP>::VE)));
  static constexpr int VE = Lay<T, DP>::VE, PER = DP / VE, NU = TK * PER / 256;
  static_assert(TK * PER % 256 == 0, "whole pieces per thread");
  vec r[NU];
  // at(row) -> pointer to the row's first channel, or null for a row of zeros
  template <typename F> __device__ __forceinline__ void load(F at, int D) {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int id = threadIdx.x + u * 256, row = id / PER, ch = id % PER * VE;
      const T *p = at(row);
      const bool in = p != nullptr && ch < D;
      vec t = {};
      if (in) t = *reinterpret_cast<const vec *>(p + ch);
      r[u] = t;
    }
  }
  __device__ __forceinline__ void store(T *lds) const {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int id = threadIdx.x + u * 256, row = id / PER, ch = id % PER * VE;
      *reinterpret_cast<vec *>(lds + row * Lay<T, DP>::LD + ch) = r[u];
    }
  }
};
// ... 4 x 4 pieces (4 tokens x 4 channels) that are turned into quads on their way to LDS
template <typename T, int DP, int TK> struct QuadStage {
  typedef typename Vec4<T>::type vec;
  static constexpr int PER = DP / 4, N = TK / 4 * PER, NU = (N + 255) / 256;
  vec r[NU][4];
  template <typename F> __device__ __forceinline__ void load(F at, int D) {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int id = threadIdx.x + u * 256, quad = id / PER, ch = id % PER * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        vec t = {};
        if (id < N) {
          const T *p = at(quad * 4 + i);
          if (p != nullptr && ch < D) t = *reinterpret_cast<const vec *>(p + ch);
        }
        r[u][i] = t;
      }
    }
  }
  __device__ __forceinline__ void store(T *lds) const {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int id = threadIdx.x + u * 256, quad = id / PER, ch = id % PER * 4;
      if (id >= N) continue;
      T *p = lds + quad * Lay<T, DP>::QD + ch * 4;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const vec t = {r[u][0][d], r[u][1][d], r[u][2][d], r[u][3][d]};
        *reinterpret_cast<vec *>(p + d * 4) = t;
      }
    }
  }
};

// ------------------------------------------------------------------------------------------ the blocks of one group
// blocks[0 .. top) of one group -> list[]: the valid indices, ascending, each once (a repeated index counts once, an index outside
// [0, nb) is no block).  Through a bit per block; returns their number.  Called by the whole workgroup.
__device__ __forceinline__ int group_blocks(const int32_t *blocks, int top, int nb, uint32_t *bits, int *list, int *n_out) {
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
// One workgroup: M = 16 NQ WM query rows of one group (a row = one query token and one head of the key head's group), 4 waves as WM
// row sets x WN key sets.  The group's keys pass as one stream in tiles of TK = 32 WN; every wave keeps its own running maximum, sum
// and output for its 32 keys of each tile, joined at the end, so the only meeting of the waves in the loop is the staging of the tile.
template <typename T, int DP, int NQ, int WM, int WN>
__global__ __launch_bounds__(256) void attend_fwd_kernel(AttnArgs a) {
  constexpr int M = 16 * NQ * WM, TK = 32 * WN, KC = DP / 32, DT = DP / 16;
  typedef Lay<T, DP> L;
  typedef typename Vec8<T>::type frag;
  extern __shared__ char smem[];
  T *krows = reinterpret_cast<T *>(smem);
  T *vquads = reinterpret_cast<T *>(smem + L::rows(TK));
  constexpr size_t tiles = L::rows(TK) + L::quads(TK);
  constexpr size_t join = (size_t)M * (DP + 4) * 4 + (size_t)WN * M * 8;
  constexpr size_t body = tiles > join ? tiles : join;
  float *lim = reinterpret_cast<float *>(smem + body);           // per key of the tile: +inf, or -inf where it is not seen
  int *list = reinterpret_cast<int *>(lim + TK);
  uint32_t *bits = reinterpret_cast<uint32_t *>(list + a.cap);
  __shared__ int n_list;

  const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64, col = lane % 16, g = lane / 16;
  const int wm = wave / WN, wn = wave % WN;
  unsigned item = xcd_remap(blockIdx.x, gridDim.x);
  const int split = (int)(item % a.splits);
  item /= a.splits;
  const unsigned work = item;
  const int chunk = (int)(item % a.chunks);
  item /= a.chunks;
  const int s = (int)(item % a.S);
  const int bh = (int)(item / a.S), hk = bh % a.Hkv, b = bh / a.Hkv;

  const int n = group_blocks(a.blocks + ((int64_t)bh * a.S + s) * a.top, a.top, a.nb, bits, list, &n_list);
  const int e0 = (int)((int64_t)n * split / a.splits), e1 = (int)((int64_t)n * (split + 1) / a.splits);
  const int total = (e1 - e0) << a.lb, nt = (total + TK - 1) / TK;

  // row r of the group: token q_block * s + r / G, head hk * G + r % G
  auto row_of = [&](int m, int &token, int &head) {
    const int r = chunk * M + m;
    const int t = (int)a.by_g.div((unsigned)r);
    token = s * a.q_block + t;
    head = hk * a.G + (r - t * a.G);
    return r < a.rows && token < a.Nq;
  };
  frag qf[NQ][KC];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    int token, head;
    const bool ok = row_of((wm * NQ + i) * 16 + col, token, head);
    const T *p = reinterpret_cast<const T *>(a.q) + (int64_t)b * a.sq.b + (int64_t)token * a.sq.n + (int64_t)head * a.sq.h;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int ch = c * 32 + g * 8;
      frag t = {};
      if (ok && ch < a.D) t = *reinterpret_cast<const frag *>(p + ch);
      qf[i][c] = t;
    }
  }

  const T *kb = reinterpret_cast<const T *>(a.k) + (int64_t)b * a.sk.b + (int64_t)hk * a.sk.h;
  const T *vb = reinterpret_cast<const T *>(a.v) + (int64_t)b * a.sv.b + (int64_t)hk * a.sv.h;
  const float *vis = a.vis ? a.vis + (int64_t)b * a.Nk : nullptr;
  // key of row r of the tile at t0, or -1
  auto key_of = [&](int t0, int r) {
    const int at = t0 + r;
    if (at >= total) return -1;
    const int key = (list[e0 + (at >> a.lb)] << a.lb) + (at & ((1 << a.lb) - 1));
    if (key >= a.Nk) return -1;
    if (vis && !(vis[key] > 0.5f)) return -1;
    return key;
  };
  RowStage<T, DP, TK> ks;
  QuadStage<T, DP, TK> vs;
  float lim_r = kNegInf;
  auto load = [&](int t0) {
    ks.load([&](int r) { const int key = key_of(t0, r); return key < 0 ? nullptr : kb + (int64_t)key * a.sk.n; }, a.D);
    vs.load([&](int r) { const int key = key_of(t0, r); return key < 0 ? nullptr : vb + (int64_t)key * a.sv.n; }, a.D);
    if (tid < TK) lim_r = key_of(t0, tid) < 0 ? kNegInf : kPosInf;
  };

  f32x4 o[NQ][DT];
  float m[NQ], l[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    m[i] = kNegInf;
    l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (nt > 0) load(0);
  for (int t = 0; t < nt; ++t) {
    __syncthreads();                                             // the last tile has been read
    ks.store(krows);
    vs.store(vquads);
    if (tid < TK) lim[tid] = lim_r;
    __syncthreads();
    if (t + 1 < nt) load((t + 1) * TK);
    f32x4 sc[2][NQ];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < NQ; ++i) sc[u][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const frag kf = row_frag<T, DP>(krows, wn * 32 + u * 16 + col, c * 32 + g * 8);
#pragma unroll
        for (int i = 0; i < NQ; ++i) sc[u][i] = mma(kf, qf[i][c], sc[u][i]);
      }
    }
    frag pf[NQ];
    f32x4 lm[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) lm[u] = *reinterpret_cast<const f32x4 *>(lim + wn * 32 + u * 16 + g * 4);
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      float mx = kNegInf;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[u][i][e] = fminf(sc[u][i][e] * a.c, lm[u][e]);      // log2 units; an unseen key's score becomes -inf
          mx = fmaxf(mx, sc[u][i][e]);
        }
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float mn = fmaxf(m[i], mx);
      const float ms = mn == kNegInf ? 0.f : mn;                 // nothing seen yet: exp2(-inf - 0) = 0
      const float f = __builtin_amdgcn_exp2f(m[i] - ms);
      m[i] = mn;
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(sc[u][i][e] - ms);
          sum += p;
          pf[i][u * 4 + e] = (T)p;
        }
      l[i] = l[i] * f + sum;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[i][d] *= f;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const frag vf = quad_frag<T, DP>(vquads, wn * 32, g, d * 16 + col);
#pragma unroll
      for (int i = 0; i < NQ; ++i) o[i][d] = mma(vf, pf[i], o[i][d]);
    }
  }

  // join the key sets: common maximum, then the outputs added up in LDS in wave order
  float *jo = reinterpret_cast<float *>(smem);                   // [M][DP + 4]
  float *jm = jo + M * (DP + 4), *jl = jm + WN * M;              // [WN][M] each
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    l[i] += __shfl_xor(l[i], 16, 64);
    l[i] += __shfl_xor(l[i], 32, 64);
    if (g == 0) {
      jm[wn * M + (wm * NQ + i) * 16 + col] = m[i];
      jl[wn * M + (wm * NQ + i) * 16 + col] = l[i];
    }
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WN; ++w) {
    if (wn == w) {
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        const int r = (wm * NQ + i) * 16 + col;
        float mx = kNegInf;
#pragma unroll
        for (int x = 0; x < WN; ++x) mx = fmaxf(mx, jm[x * M + r]);
        const float f = mx == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m[i] - mx);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          f32x4 *p = reinterpret_cast<f32x4 *>(jo + r * (DP + 4) + d * 16 + g * 4);
          const f32x4 x = o[i][d] * f;
          *p = w == 0 ? x : *p + x;
        }
      }
    }
    __syncthreads();
  }
  // write out: rows of D channels, 4 per thread
  float *pm = a.splits > 1 ? a.part + ((int64_t)work * a.splits + split) * M * (a.D + 2) : nullptr;
  const int per = a.D / 4;
  for (int id = tid; id < M * per; id += 256) {
    const int r = id / per, ch = (id - r * per) * 4;
    int token, head;
    if (!row_of(r, token, head)) continue;
    float mx = kNegInf, sum = 0.f;
#pragma unroll
    for (int x = 0; x < WN; ++x) mx = fmaxf(mx, jm[x * M + r]);
#pragma unroll
    for (int x = 0; x < WN; ++x) sum += mx == kNegInf ? 0.f : jl[x * M + r] * __builtin_amdgcn_exp2f(jm[x * M + r] - mx);
    const f32x4 x = *reinterpret_cast<const f32x4 *>(jo + r * (DP + 4) + ch);
    if (pm) {
      *reinterpret_cast<f32x4 *>(pm + (int64_t)r * a.D + ch) = x;
      if (ch == 0) {
        pm[(int64_t)M * a.D + r] = mx;
        pm[(int64_t)M * a.D + M + r] = sum;
      }
      continue;
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);   // nothing seen: zero; NaN stays NaN
    typename Vec4<T>::type y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)(x[e] * inv);
    *reinterpret_cast<typename Vec4<T>::type *>(reinterpret_cast<T *>(a.out) + (int64_t)b * a.so.b + (int64_t)token * a.so.n + (int64_t)head * a.so.h + ch) = y;
    if (ch == 0 && a.lse) a.lse[((int64_t)b * a.Hq + head) * a.Nq + token] = sum == 0.f ? kNegInf : (mx + __builtin_log2f(sum)) * kLn2;
  }
}

// Joins the splits of a row: one wave per row, 4 rows per workgroup.
template <typename T>
__global__ __launch_bounds__(256) void attend_join_kernel(AttnArgs a, int M) {
  const int64_t id = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  const int lane = threadIdx.x % 64;
  const int64_t works = (int64_t)a.B * a.Hkv * a.S * a.chunks;
  const int64_t work = id / M;
  const int r = (int)(id - work * M);
  if (work >= works) return;
  const int chunk = (int)(work % a.chunks), s = (int)(work / a.chunks % a.S);
  const int bh = (int)(work / a.chunks / a.S), hk = bh % a.Hkv, b = bh / a.Hkv;
  const int row = chunk * M + r, t = (int)a.by_g.div((unsigned)row), token = s * a.q_block + t, head = hk * a.G + (row - t * a.G);
  if (row >= a.rows || token >= a.Nq) return;
  const int64_t step = (int64_t)M * (a.D + 2);
  const float *p = a.part + work * a.splits * step;
  float mx = kNegInf, sum = 0.f;
  for (int x = 0; x < a.splits; ++x) mx = fmaxf(mx, p[x * step + (int64_t)M * a.D + r]);
  for (int x = 0; x < a.splits; ++x) {
    const float mi = p[x * step + (int64_t)M * a.D + r];
    if (mi != kNegInf) sum += p[x * step + (int64_t)M * a.D + M + r] * __builtin_amdgcn_exp2f(mi - mx);
  }
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  for (int ch = lane; ch < a.D; ch += 64) {
    float o = 0.f;
    for (int x = 0; x < a.splits; ++x) {
      const float mi = p[x * step + (int64_t)M * a.D + r];
      if (mi != kNegInf) o += p[x * step + (int64_t)r * a.D + ch] * __builtin_amdgcn_exp2f(mi - mx);
    }
    reinterpret_cast<T *>(a.out)[(int64_t)b * a.so.b + (int64_t)token * a.so.n + (int64_t)head * a.so.h + ch] = (T)(o * inv);
  }
  if (lane == 0 && a.lse) a.lse[((int64_t)b * a.Hq + head) * a.Nq + token] = sum == 0.f ? kNegInf : (mx + __builtin_log2f(sum)) * kLn2;
}

// ------------------------------------------------------------------------------------------ backward
// With P = exp(scale S - lse) and dP = dout V^T:  dV = P^T dout,  dS = scale P o (dP - delta),  delta = rowsum(dout o out),
// dQ = dS K,  dK = dS^T Q.  dQ is summed per query tile (like the forward), dK and dV per key tile: two kernels that both recompute
// S and dP, and no atomics, so a gradient does not depend on the order of the workgroups.
//
// fp16: P is scaled up by 2^10 as an operand (P <= 1; of 4096 equal keys each has 2^-12, and below 2^-14 fp16 loses bits).
template <typename T> struct PScale { static constexpr float bits = 0.f, inv = 1.f; };
template <> struct PScale<_Float16> { static constexpr float bits = 10.f, inv = 0x1p-10f; };

// delta of every row: 16 lanes per row, 8 channels each
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
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf((float)x[e], (float)y[e], sum);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (live && ch == 0) a.delta[((int64_t)b * a.Hq + head) * a.Nq + token] = sum;
}

// which groups chose each block: one bit per (block, group)
__global__ __launch_bounds__(256) void attend_clear_kernel(uint32_t *p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = 0;
}
__global__ __launch_bounds__(256) void attend_invert_kernel(AttnArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.B * a.Hkv * a.S * a.top) return;
  const int j = a.blocks[i];
  const int64_t row = i / a.top;
  const int s = (int)(row % a.S);
  const int64_t bh = row / a.S;
  if (j >= 0 && j < a.nb) atomicOr(&a.inv[(bh * a.nb + j) * a.words + (s >> 5)], 1u << (s & 31));
}

template <typename T, int DP, int NQ, int WM, int WN>
__global__ __launch_bounds__(256) void attend_dq_kernel(AttnArgs a) {
  constexpr int M = 16 * NQ * WM, TK = 32 * WN, KC = DP / 32, DT = DP / 16;
  typedef Lay<T, DP> L;
  typedef typename Vec8<T>::type frag;
  extern __shared__ char smem[];
  T *krows = reinterpret_cast<T *>(smem);
  T *vrows = reinterpret_cast<T *>(smem + L::rows(TK));
  T *kquads = reinterpret_cast<T *>(smem + 2 * L::rows(TK));
  constexpr size_t tiles = 2 * L::rows(TK) + L::quads(TK);
  constexpr size_t join = (size_t)M * (DP + 4) * 4;
  constexpr size_t body = tiles > join ? tiles : join;
  float *lim = reinterpret_cast<float *>(smem + body);
  int *list = reinterpret_cast<int *>(lim + TK);
  uint32_t *bits = reinterpret_cast<uint32_t *>(list + a.cap);
  __shared__ int n_list;

  const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64, col = lane % 16, g = lane / 16;
  const int wm = wave / WN, wn = wave % WN;
  unsigned item = xcd_remap(blockIdx.x, gridDim.x);
  const int chunk = (int)(item % a.chunks);
  item /= a.chunks;
  const int s = (int)(item % a.S);
  const int bh = (int)(item / a.S), hk = bh % a.Hkv, b = bh / a.Hkv;
  const int n = group_blocks(a.blocks + ((int64_t)bh * a.S + s) * a.top, a.top, a.nb, bits, list, &n_list);
  const int total = n << a.lb, nt = (total + TK - 1) / TK;
  auto row_of = [&](int m, int &token, int &head) {
    const int r = chunk * M + m;
    const int t = (int)a.by_g.div((unsigned)r);
    token = s * a.q_block + t;
    head = hk * a.G + (r - t * a.G);
    return r < a.rows && token < a.Nq;
  };
  frag qf[NQ][KC], df[NQ][KC];
  float lse2[NQ], delta[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    int token, head;
    const bool ok = row_of((wm * NQ + i) * 16 + col, token, head);
    const T *p = reinterpret_cast<const T *>(a.q) + (int64_t)b * a.sq.b + (int64_t)token * a.sq.n + (int64_t)head * a.sq.h;
    const T *d = reinterpret_cast<const T *>(a.dout) + (int64_t)b * a.sdo.b + (int64_t)token * a.sdo.n + (int64_t)head * a.sdo.h;
    lse2[i] = kPosInf;                                           // exp2(x - inf) = 0: no row, or a row that sees nothing
    delta[i] = 0.f;
    if (ok) {
      const int64_t at = ((int64_t)b * a.Hq + head) * a.Nq + token;
      const float x = a.lse[at];
      lse2[i] = x == kNegInf ? kPosInf : x * kLog2e;
      delta[i] = a.delta[at];
    }
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int ch = c * 32 + g * 8;
      frag t = {}, u = {};
      if (ok && ch < a.D) {
        t = *reinterpret_cast<const frag *>(p + ch);
        u = *reinterpret_cast<const frag *>(d + ch);
      }
      qf[i][c] = t;
      df[i][c] = u;
    }
  }
  const T *kb = reinterpret_cast<const T *>(a.k) + (int64_t)b * a.sk.b + (int64_t)hk * a.sk.h;
  const T *vb = reinterpret_cast<const T *>(a.v) + (int64_t)b * a.sv.b + (int64_t)hk * a.sv.h;
  const float *vis = a.vis ? a.vis + (int64_t)b * a.Nk : nullptr;
  auto key_of = [&](int t0, int r) {
    const int at = t0 + r;
    if (at >= total) return -1;
    const int key = (list[at >> a.lb] << a.lb) + (at & ((1 << a.lb) - 1));
    if (key >= a.Nk) return -1;
    if (vis && !(vis[key] > 0.5f)) return -1;
    return key;
  };
  RowStage<T, DP, TK> ks, vs;
  QuadStage<T, DP, TK> kq;
  float lim_r = kNegInf;
  auto load = [&](int t0) {
    ks.load([&](int r) { const int key = key_of(t0, r); return key < 0 ? nullptr : kb + (int64_t)key * a.sk.n; }, a.D);
    vs.load([&](int r) { const int key = key_of(t0, r); return key < 0 ? nullptr : vb + (int64_t)key * a.sv.n; }, a.D);
    kq.load([&](int r) { const int key = key_of(t0, r); return key < 0 ? nullptr : kb + (int64_t)key * a.sk.n; }, a.D);
    if (tid < TK) lim_r = key_of(t0, tid) < 0 ? kNegInf : kPosInf;
  };
  f32x4 o[NQ][DT];
#pragma unroll
  for (int i = 0; i < NQ; ++i)
#pragma unroll
    for (int d = 0; d < DT; ++d) o[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (nt > 0) load(0);
  for (int t = 0; t < nt; ++t) {
    __syncthreads();
    ks.store(krows);
    vs.store(vrows);
    kq.store(kquads);
    if (tid < TK) lim[tid] = lim_r;
    __syncthreads();
    if (t + 1 < nt) load((t + 1) * TK);
    f32x4 sc[2][NQ], dp[2][NQ];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < NQ; ++i) sc[u][i] = dp[u][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const frag kf = row_frag<T, DP>(krows, wn * 32 + u * 16 + col, c * 32 + g * 8);
        const frag vf = row_frag<T, DP>(vrows, wn * 32 + u * 16 + col, c * 32 + g * 8);
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          sc[u][i] = mma(kf, qf[i][c], sc[u][i]);
          dp[u][i] = mma(vf, df[i][c], dp[u][i]);
        }
      }
    }
    frag gf[NQ];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const f32x4 lm = *reinterpret_cast<const f32x4 *>(lim + wn * 32 + u * 16 + g * 4);
#pragma unroll
      for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(fminf(sc[u][i][e] * a.c, lm[e]) - lse2[i]);
          gf[i][u * 4 + e] = (T)(p * (dp[u][i][e] - delta[i]) * a.scale);
        }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const frag kf = quad_frag<T, DP>(kquads, wn * 32, g, d * 16 + col);
#pragma unroll
      for (int i = 0; i < NQ; ++i) o[i][d] = mma(kf, gf[i], o[i][d]);
    }
  }
  float *jo = reinterpret_cast<float *>(smem);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WN; ++w) {
    if (wn == w) {
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        const int r = (wm * NQ + i) * 16 + col;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          f32x4 *p = reinterpret_cast<f32x4 *>(jo + r * (DP + 4) + d * 16 + g * 4);
          *p = w == 0 ? o[i][d] : *p + o[i][d];
        }
      }
    }
    __syncthreads();
  }
  const int per = a.D / 4;
  for (int id = tid; id < M * per; id += 256) {
    const int r = id / per, ch = (id - r * per) * 4;
    int token, head;
    if (!row_of(r, token, head)) continue;
    const f32x4 x = *reinterpret_cast<const f32x4 *>(jo + r * (DP + 4) + ch);
    typename Vec4<T>::type y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)x[e];
    *reinterpret_cast<typename Vec4<T>::type *>(reinterpret_cast<T *>(a.dq) + (int64_t)b * a.sdq.b + (int64_t)token * a.sdq.n + (int64_t)head * a.sdq.h + ch) = y;
  }
}

// One workgroup: 16 NK WM keys (a tile of one block) against all query rows of the groups that chose the block.  The rows pass as a
// stream (group after group, in ascending order) in tiles of TR = 32 WN; rows and keys have changed places with the forward:
// S = Q K^T leaves a lane the probabilities of ITS key, the operand of dV^T = dout^T P and, as dS, of dK^T = Q^T dS.
constexpr int kWindow = 32;   // words of group bits taken at a time: up to 1024 groups in the list

template <typename T, int DP, int NK, int WM, int WN>
__global__ __launch_bounds__(256) void attend_dkv_kernel(AttnArgs a) {
  constexpr int M = 16 * NK * WM, TR = 32 * WN, KC = DP / 32, DT = DP / 16;
  typedef Lay<T, DP> L;
  typedef typename Vec8<T>::type frag;
  extern __shared__ char smem[];
  T *qrows = reinterpret_cast<T *>(smem);
  T *drows = reinterpret_cast<T *>(smem + L::rows(TR));
  T *qquads = reinterpret_cast<T *>(smem + 2 * L::rows(TR));
  T *dquads = reinterpret_cast<T *>(smem + 2 * L::rows(TR) + L::quads(TR));
  constexpr size_t tiles = 2 * (L::rows(TR) + L::quads(TR));
  constexpr size_t join = (size_t)M * (DP + 4) * 4;
  constexpr size_t body = tiles > join ? tiles : join;
  float *lse2 = reinterpret_cast<float *>(smem + body), *delta = lse2 + TR;
  int *list = reinterpret_cast<int *>(delta + TR);               // [32 kWindow]
  __shared__ int n_list;

  const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64, col = lane % 16, g = lane / 16;
  const int wm = wave / WN, wn = wave % WN;
  const int tiles_of = (a.Nk + M - 1) / M;
  unsigned item = xcd_remap(blockIdx.x, gridDim.x);
  const int kt = (int)(item % tiles_of);
  const int bh = (int)(item / tiles_of), hk = bh % a.Hkv, b = bh / a.Hkv;
  const uint32_t *inv = a.inv + ((int64_t)bh * a.nb + (((int64_t)kt * M) >> a.lb)) * a.words;

  frag kf[NK][KC], vf[NK][KC];
  float lim[NK];
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int key = kt * M + (wm * NK + i) * 16 + col;
    const bool ok = key < a.Nk && (!a.vis || a.vis[(int64_t)b * a.Nk + key] > 0.5f);
    lim[i] = ok ? kPosInf : kNegInf;
    const T *p = reinterpret_cast<const T *>(a.k) + (int64_t)b * a.sk.b + (int64_t)key * a.sk.n + (int64_t)hk * a.sk.h;
    const T *q = reinterpret_cast<const T *>(a.v) + (int64_t)b * a.sv.b + (int64_t)key * a.sv.n + (int64_t)hk * a.sv.h;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int ch = c * 32 + g * 8;
      frag t = {}, u = {};
      if (ok && ch < a.D) {
        t = *reinterpret_cast<const frag *>(p + ch);
        u = *reinterpret_cast<const frag *>(q + ch);
      }
      kf[i][c] = t;
      vf[i][c] = u;
    }
  }
  const T *qb = reinterpret_cast<const T *>(a.q) + (int64_t)b * a.sq.b;
  const T *db = reinterpret_cast<const T *>(a.dout) + (int64_t)b * a.sdo.b;
  f32x4 gk[NK][DT], gv[NK][DT];
#pragma unroll
  for (int i = 0; i < NK; ++i)
#pragma unroll
    for (int d = 0; d < DT; ++d) gk[i][d] = gv[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int w0 = 0; w0 < a.words; w0 += kWindow) {
    __syncthreads();                                             // the last window's list has been read
    if (tid < 64) {
      const uint32_t bitsw = tid < kWindow && w0 + tid < a.words ? inv[w0 + tid] : 0;
      uint32_t m = bitsw;
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
    const int64_t total = (int64_t)n_list * a.rows;
    const int64_t nt = (total + TR - 1) / TR;
    // row r of the tile at t0: (token, head), or none
    auto row_of = [&](int64_t t0, int r, int &token, int &head) {
      const int64_t at = t0 + r;
      if (at >= total) return false;
      const unsigned e = a.by_rows.div((unsigned)at), rr = (unsigned)at - e * (unsigned)a.rows;
      const unsigned t = a.by_g.div(rr);
      token = list[e] * a.q_block + (int)t;
      head = hk * a.G + (int)(rr - t * (unsigned)a.G);
      return token < a.Nq;
    };
    auto q_at = [&](int64_t t0, int r) -> const T * {
      int token, head;
      return row_of(t0, r, token, head) ? qb + (int64_t)token * a.sq.n + (int64_t)head * a.sq.h : nullptr;
    };
    auto d_at = [&](int64_t t0, int r) -> const T * {
      int token, head;
      return row_of(t0, r, token, head) ? db + (int64_t)token * a.sdo.n + (int64_t)head * a.sdo.h : nullptr;
    };
    RowStage<T, DP, TR> qs, ds;
    QuadStage<T, DP, TR> qq, dq;
    float lse_r = kPosInf, delta_r = 0.f;
    auto load = [&](int64_t t0) {
      qs.load([&](int r) { return q_at(t0, r); }, a.D);
      ds.load([&](int r) { return d_at(t0, r); }, a.D);
      qq.load([&](int r) { return q_at(t0, r); }, a.D);
      dq.load([&](int r) { return d_at(t0, r); }, a.D);
      if (tid < TR) {
        int token, head;
        lse_r = kPosInf;
        delta_r = 0.f;
        if (row_of(t0, tid, token, head)) {
          const int64_t at = ((int64_t)b * a.Hq + head) * a.Nq + token;
          const float x = a.lse[at];
          lse_r = x == kNegInf ? kPosInf : x * kLog2e - PScale<T>::bits;
          delta_r = a.delta[at];
        }
      }
    };
    if (nt > 0) load(0);
    for (int64_t t = 0; t < nt; ++t) {
      __syncthreads();
      qs.store(qrows);
      ds.store(drows);
      qq.store(qquads);
      dq.store(dquads);
      if (tid < TR) { lse2[tid] = lse_r; delta[tid] = delta_r; }
      __syncthreads();
      if (t + 1 < nt) load((t + 1) * TR);
      f32x4 sc[2][NK], dp[2][NK];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int i = 0; i < NK; ++i) sc[u][i] = dp[u][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const frag qf = row_frag<T, DP>(qrows, wn * 32 + u * 16 + col, c * 32 + g * 8);
          const frag df = row_frag<T, DP>(drows, wn * 32 + u * 16 + col, c * 32 + g * 8);
#pragma unroll
          for (int i = 0; i < NK; ++i) {
            sc[u][i] = mma(qf, kf[i][c], sc[u][i]);
            dp[u][i] = mma(df, vf[i][c], dp[u][i]);
          }
        }
      }
      frag pf[NK], gf[NK];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f32x4 ls = *reinterpret_cast<const f32x4 *>(lse2 + wn * 32 + u * 16 + g * 4);
        const f32x4 de = *reinterpret_cast<const f32x4 *>(delta + wn * 32 + u * 16 + g * 4);
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f(fminf(sc[u][i][e] * a.c, lim[i]) - ls[e]);
            pf[i][u * 4 + e] = (T)p;
            gf[i][u * 4 + e] = (T)(p * (dp[u][i][e] - de[e]) * (a.scale * PScale<T>::inv));
          }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const frag df = quad_frag<T, DP>(dquads, wn * 32, g, d * 16 + col);
        const frag qf = quad_frag<T, DP>(qquads, wn * 32, g, d * 16 + col);
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          gv[i][d] = mma(df, pf[i], gv[i][d]);
          gk[i][d] = mma(qf, gf[i], gk[i][d]);
        }
      }
    }
  }
  float *jo = reinterpret_cast<float *>(smem);
  const int per = a.D / 4;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    T *out = reinterpret_cast<T *>(which ? a.dv : a.dk);
    if (out == nullptr) continue;
    const Str st = which ? a.sdv : a.sdk;
    const float f = which ? PScale<T>::inv : 1.f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WN; ++w) {
      if (wn == w) {
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            f32x4 *p = reinterpret_cast<f32x4 *>(jo + ((wm * NK + i) * 16 + col) * (DP + 4) + d * 16 + g * 4);
            const f32x4 x = (which ? gv[i][d] : gk[i][d]) * f;
            *p = w == 0 ? x : *p + x;
          }
      }
      __syncthreads();
    }
    for (int id = tid; id < M * per; id += 256) {
      const int r = id / per, ch = (id - r * per) * 4, key = kt * M + r;
      if (key >= a.Nk) continue;
      const f32x4 x = *reinterpret_cast<const f32x4 *>(jo + r * (DP + 4) + ch);
      typename Vec4<T>::type y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (T)x[e];
      *reinterpret_cast<typename Vec4<T>::type *>(out + (int64_t)b * st.b + (int64_t)key * st.n + (int64_t)hk * st.h + ch) = y;
    }
  }
}

// ------------------------------------------------------------------------------------------ host
template <typename T, int DP, int NQ, int WM, int WN> static size_t fwd_lds(const AttnArgs &a) {
  constexpr int M = 16 * NQ * WM, TK = 32 * WN;
  const size_t tiles = Lay<T, DP>::rows(TK) + Lay<T, DP>::quads(TK), join = (size_t)M * (DP + 4) * 4 + (size_t)WN * M * 8;
  return (tiles > join ? tiles : join) + TK * 4 + (size_t)a.cap * 4 + (size_t)(a.nb + 31) / 32 * 4;
}

constexpr int kFewRows = 16;       // up to 16 rows in a group: the kernel whose four waves share the keys of 16 rows
static int fwd_rows(const AttnArgs &a) { return a.rows <= kFewRows ? 16 : 64; }

template <typename T, int DP, int NQ, int WM, int WN> static int launch_fwd_tile(const AttnArgs &a, int64_t blocks, hipStream_t s) {
  const auto kernel = attend_fwd_kernel<T, DP, NQ, WM, WN>;
  const size_t lds = fwd_lds<T, DP, NQ, WM, WN>(a);
  TCL_REQUIRE(lds_ready((const void *)kernel, lds), TCL_ERR_LAUNCH, "block_attention: the device refuses %zu bytes of LDS", lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), lds, s, a);
  return check_launch("block_attention");
}
template <typename T, int DP> static int launch_fwd(const AttnArgs &a, int64_t blocks, hipStream_t s) {
  return fwd_rows(a) == 16 ? launch_fwd_tile<T, DP, 1, 1, 4>(a, blocks, s) : launch_fwd_tile<T, DP, 2, 2, 2>(a, blocks, s);
}

template <typename T, int DP, int NQ, int WM, int WN> static int launch_dq_tile(const AttnArgs &a, int64_t blocks, hipStream_t s) {
  constexpr int M = 16 * NQ * WM, TK = 32 * WN;
  const size_t tiles = 2 * Lay<T, DP>::rows(TK) + Lay<T, DP>::quads(TK), join = (size_t)M * (DP + 4) * 4;
  const size_t lds = (tiles > join ? tiles : join) + TK * 4 + (size_t)a.cap * 4 + (size_t)(a.nb + 31) / 32 * 4;
  const auto kernel = attend_dq_kernel<T, DP, NQ, WM, WN>;
  TCL_REQUIRE(lds_ready((const void *)kernel, lds), TCL_ERR_LAUNCH, "block_attention: the device refuses %zu bytes of LDS", lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), lds, s, a);
  return check_launch("block_attention backward (queries)");
}
constexpr int kDqFewRows = 32;     // the same for the query gradient (three tile images: 64 keys at a time, 32 rows)
template <typename T, int DP> static int launch_dq(AttnArgs a, hipStream_t s) {
  const bool few = a.rows <= kDqFewRows;
  a.chunks = (int)cdiv(a.rows, few ? 32 : 64);
  const int64_t blocks = (int64_t)a.B * a.Hkv * a.S * a.chunks;
  TCL_REQUIRE(blocks < (1LL << 31), TCL_ERR_SHAPE, "block_attention backward: grid of %ld blocks", (long)blocks);
  return few ? launch_dq_tile<T, DP, 1, 2, 2>(a, blocks, s) : launch_dq_tile<T, DP, 2, 2, 2>(a, blocks, s);
}
template <typename T, int DP> static int launch_dkv(const AttnArgs &a, hipStream_t s) {
  typedef Lay<T, DP> L;
  constexpr int M = 64, TR = 64;
  const size_t tiles = 2 * (L::rows(TR) + L::quads(TR)), join = (size_t)M * (DP + 4) * 4;
  const size_t lds = (tiles > join ? tiles : join) + 2 * TR * 4 + 32 * kWindow * 4;
  const int64_t blocks = cdiv(a.Nk, M) * a.B * a.Hkv;
  TCL_REQUIRE(blocks < (1LL << 31), TCL_ERR_SHAPE, "block_attention backward: grid of %ld blocks", (long)blocks);
  const auto kernel = attend_dkv_kernel<T, DP, 2, 2, 2>;
  TCL_REQUIRE(lds_ready((const void *)kernel, lds), TCL_ERR_LAUNCH, "block_attention: the device refuses %zu bytes of LDS", lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), lds, s, a);
  return check_launch("block_attention backward (keys)");
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
#define CALL(T, DP) (launch_fwd<T, DP>(a, blocks, s))
  TCL_BY_DIM(T, CALL)
#undef CALL
}
template <typename T> static int dq_by_dim(const AttnArgs &a, hipStream_t s) {
#define CALL(T, DP) (launch_dq<T, DP>(a, s))
  TCL_BY_DIM(T, CALL)
#undef CALL
}
template <typename T> static int dkv_by_dim(const AttnArgs &a, hipStream_t s) {
#define CALL(T, DP) (launch_dkv<T, DP>(a, s))
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
  a.scale = (float)scale;
  a.c = (float)(scale * 1.4426950408889634074);
  a.chunks = 1;
  a.splits = 1;
  return TCL_OK;
}

// Splits of the keys of a forward work item: enough workgroups for two per CU, two tiles each at least.
static int fwd_splits(const AttnArgs &a, int64_t works) {
  const int tk = fwd_rows(a) == 16 ? 128 : 64;
  const int64_t tiles = cdiv((int64_t)a.cap << a.lb, tk);
  int64_t n = cdiv(2 * kNumCU, works > 0 ? works : 1);
  if (n > tiles / 2) n = tiles / 2;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}
static size_t fwd_part_bytes(const AttnArgs &a, int64_t works, int splits) {
  return splits > 1 ? round_up((size_t)works * splits * fwd_rows(a) * (a.D + 2) * 4, 256) : 256;
}
static bool rows16(const void *p, const Str &s, int dtype) {
  const int64_t ve = dtype == TCL_DT_F32 ? 4 : 8;
  return aligned(p, 16) && s.b % ve == 0 && s.n % ve == 0 && s.h % ve == 0;
}

}  // namespace tcl

using namespace tcl;

extern "C" size_t tcl_block_attention_fwd_workspace_bytes(int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D, int64_t top_k, int64_t block,
                                                          int64_t q_block) {
  AttnArgs a{};
  if (attn_setup(a, B, Nq, Nk, Hq, Hkv, D, top_k, block, q_block, 1.0, TCL_DT_F32) != TCL_OK) return 256;
  const int64_t works = B * Hkv * a.S * cdiv(a.rows, fwd_rows(a));
  return fwd_part_bytes(a, works, fwd_splits(a, works));
}

extern "C" int tcl_block_attention_fwd(const void *q, int64_t q_sb, int64_t q_sn, int64_t q_sh, const void *k, int64_t k_sb, int64_t k_sn, int64_t k_sh,
                                       const void *v, int64_t v_sb, int64_t v_sn, int64_t v_sh, const float *visible, const int32_t *blocks,
                                       void *out, int64_t o_sb, int64_t o_sn, int64_t o_sh, float *lse,
                                       int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D, int64_t top_k, int64_t block, int64_t q_block,
                                       double scale, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  AttnArgs a{};
  const int rc = attn_setup(a, B, Nq, Nk, Hq, Hkv, D, top_k, block, q_block, scale, dtype);
  if (rc != TCL_OK) return rc;
  if (B == 0 || Nq == 0) return TCL_OK;
  TCL_REQUIRE(q && out && blocks && (Nk == 0 || (k && v)), TCL_ERR_ARG, "block_attention: null pointer");
  a.q = q; a.k = k; a.v = v; a.vis = visible; a.blocks = blocks; a.out = out; a.lse = lse;
  a.sq = Str{q_sb, q_sn, q_sh}; a.sk = Str{k_sb, k_sn, k_sh}; a.sv = Str{v_sb, v_sn, v_sh}; a.so = Str{o_sb, o_sn, o_sh};
  TCL_REQUIRE(rows16(q, a.sq, dtype) && (Nk == 0 || (rows16(k, a.sk, dtype) && rows16(v, a.sv, dtype))) && rows16(out, a.so, dtype), TCL_ERR_ARG,
              "block_attention: rows must start on 16 bytes");
  a.chunks = (int)cdiv(a.rows, fwd_rows(a));
  const int64_t works = B * Hkv * a.S * a.chunks;
  a.splits = fwd_splits(a, works);
  const int64_t blocks_n = works * a.splits;
  TCL_REQUIRE(blocks_n < (1LL << 31), TCL_ERR_SHAPE, "block_attention: grid of %ld blocks", (long)blocks_n);
  const size_t need = fwd_part_bytes(a, works, a.splits);
  TCL_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= need, TCL_ERR_WORKSPACE, "block_attention: workspace of %zu bytes needed", need);
  a.part = (float *)workspace;
  const hipStream_t s = (hipStream_t)stream;
  const int r = dtype == TCL_DT_F32 ? fwd_by_dim<float>(a, blocks_n, s) : dtype == TCL_DT_BF16 ? fwd_by_dim<__bf16>(a, blocks_n, s) : fwd_by_dim<_Float16>(a, blocks_n, s);
  if (r != TCL_OK || a.splits == 1) return r;
  const int M = fwd_rows(a);
  const dim3 grid((unsigned)cdiv(works * M, 4));
  if (dtype == TCL_DT_F32) hipLaunchKernelGGL((attend_join_kernel<float>), grid, dim3(256), 0, s, a, M);
  else if (dtype == TCL_DT_BF16) hipLaunchKernelGGL((attend_join_kernel<__bf16>), grid, dim3(256), 0, s, a, M);
  else hipLaunchKernelGGL((attend_join_kernel<_Float16>), grid, dim3(256), 0, s, a, M);
  return check_launch("block_attention (join)");
}

extern "C" size_t tcl_block_attention_bwd_workspace_bytes(int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D, int64_t top_k, int64_t block,
                                                          int64_t q_block) {
  AttnArgs a{};
  if (attn_setup(a, B, Nq, Nk, Hq, Hkv, D, top_k, block, q_block, 1.0, TCL_DT_F32) != TCL_OK) return 256;
  return round_up((size_t)B * Hq * Nq * 4, 256) + round_up((size_t)B * Hkv * a.nb * a.words * 4, 256) + 256;
}

extern "C" int tcl_block_attention_bwd(const void *grad_out, int64_t g_sb, int64_t g_sn, int64_t g_sh, const void *q, int64_t q_sb, int64_t q_sn, int64_t q_sh,
                                       const void *k, int64_t k_sb, int64_t k_sn, int64_t k_sh, const void *v, int64_t v_sb, int64_t v_sn, int64_t v_sh,
                                       const float *visible, const int32_t *blocks, const void *out, int64_t o_sb, int64_t o_sn, int64_t o_sh, const float *lse,
                                       void *g_q, int64_t gq_sb, int64_t gq_sn, int64_t gq_sh, void *g_k, int64_t gk_sb, int64_t gk_sn, int64_t gk_sh,
                                       void *g_v, int64_t gv_sb, int64_t gv_sn, int64_t gv_sh,
                                       int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D, int64_t top_k, int64_t block, int64_t q_block,
                                       double scale, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  AttnArgs a{};
  const int rc = attn_setup(a, B, Nq, Nk, Hq, Hkv, D, top_k, block, q_block, scale, dtype);
  if (rc != TCL_OK) return rc;
  if (B == 0 || Nq == 0 || Nk == 0) return TCL_OK;             // the caller zeroes gradients of an empty attention
  TCL_REQUIRE(grad_out && q && k && v && out && blocks && lse, TCL_ERR_ARG, "block_attention backward: null pointer");
  a.q = q; a.k = k; a.v = v; a.dout = grad_out; a.vis = visible; a.blocks = blocks; a.out = const_cast<void *>(out); a.lse = const_cast<float *>(lse);
  a.dq = g_q; a.dk = g_k; a.dv = g_v;
  a.sq = Str{q_sb, q_sn, q_sh}; a.sk = Str{k_sb, k_sn, k_sh}; a.sv = Str{v_sb, v_sn, v_sh}; a.so = Str{o_sb, o_sn, o_sh}; a.sdo = Str{g_sb, g_sn, g_sh};
  a.sdq = Str{gq_sb, gq_sn, gq_sh}; a.sdk = Str{gk_sb, gk_sn, gk_sh}; a.sdv = Str{gv_sb, gv_sn, gv_sh};
  TCL_REQUIRE(rows16(q, a.sq, dtype) && rows16(k, a.sk, dtype) && rows16(v, a.sv, dtype) && rows16(out, a.so, dtype) && rows16(grad_out, a.sdo, dtype) &&
              (!g_q || rows16(g_q, a.sdq, dtype)) && (!g_k || rows16(g_k, a.sdk, dtype)) && (!g_v || rows16(g_v, a.sdv, dtype)), TCL_ERR_ARG,
              "block_attention backward: rows must start on 16 bytes");
  const size_t need = tcl_block_attention_bwd_workspace_bytes(B, Nq, Nk, Hq, Hkv, D, top_k, block, q_block);
  TCL_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= need, TCL_ERR_WORKSPACE, "block_attention backward: workspace of %zu bytes needed", need);
  a.delta = (float *)workspace;
  a.inv = (uint32_t *)((char *)workspace + round_up((size_t)B * Hq * Nq * 4, 256));
  const hipStream_t s = (hipStream_t)stream;
  const int64_t dblocks = cdiv(B * Nq * Hq, 16), inv_n = (int64_t)B * Hkv * a.nb * a.words, sel_n = (int64_t)B * Hkv * a.S * a.top;
  TCL_REQUIRE(dblocks < (1LL << 31) && cdiv(inv_n, 256) < (1LL << 31) && cdiv(sel_n, 256) < (1LL << 31), TCL_ERR_SHAPE, "block_attention backward: too many rows for one call");
  if (dtype == TCL_DT_F32) hipLaunchKernelGGL((attend_delta_kernel<float>), dim3((unsigned)dblocks), dim3(256), 0, s, a);
  else if (dtype == TCL_DT_BF16) hipLaunchKernelGGL((attend_delta_kernel<__bf16>), dim3((unsigned)dblocks), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((attend_delta_kernel<_Float16>), dim3((unsigned)dblocks), dim3(256), 0, s, a);
  if (g_q) {
    const int r = dtype == TCL_DT_F32 ? dq_by_dim<float>(a, s) : dtype == TCL_DT_BF16 ? dq_by_dim<__bf16>(a, s) : dq_by_dim<_Float16>(a, s);
    if (r != TCL_OK) return r;
  }
  if (!g_k && !g_v) return check_launch("block_attention backward");
  hipLaunchKernelGGL(attend_clear_kernel, dim3((unsigned)cdiv(inv_n, 256)), dim3(256), 0, s, a.inv, inv_n);
  hipLaunchKernelGGL(attend_invert_kernel, dim3((unsigned)cdiv(sel_n, 256)), dim3(256), 0, s, a);
  return dtype == TCL_DT_F32 ? dkv_by_dim<float>(a, s) : dtype == TCL_DT_BF16 ? dkv_by_dim<__bf16>(a, s) : dkv_by_dim<_Float16>(a, s);
}
