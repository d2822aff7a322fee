// Block summaries and block selection of the frame attention: tcl_block_means, tcl_select_blocks.
//
// Keys lie in blocks of 64 or 128 consecutive tokens.  A block is summarised by the mean of its visible keys; a group of queries
// (q_block consecutive tokens with all query heads of one key head) scores block j by <sum of its queries, mean_j> and takes the
// top_k best blocks that have a visible key.  A choice is a comparison of values that can lie arbitrarily close, so sums, products
// and comparisons are all carried in 64 bits: a result of fp32 scores would depend on the order of summation.
#include "tcl_common.h"

namespace tcl {

typedef double f64x4 __attribute__((ext_vector_type(4)));

template <typename T, int V> struct SelVec { typedef T type __attribute__((ext_vector_type(V))); };

// ------------------------------------------------------------------------------------------ block means
struct MeansArgs {
  const void *k;
  const float *vis;
  float *means;
  int32_t *counts;
  int64_t sb, sn, sh;
  int B, N, H, D, block, nb;
};

// One wave per (item, head, block).  A row takes D / VE lanes (16-byte loads), so 64 / (D / VE) rows are read per step, four steps in
// flight; every lane sums its channels of its rows in 64 bits, the row groups are joined through LDS.
// Bound: memory (K once): 32 x 15,900 keys x 2 heads of 64 bf16 channels 24 us, 5.5 TB/s; one frame of 1,590 keys 5 us, a launch.
template <typename T>
__global__ __launch_bounds__(256) void block_means_kernel(MeansArgs a) {
  constexpr int VE = 16 / sizeof(T);
  typedef typename SelVec<T, VE>::type vec;
  __shared__ double part[4][64 * VE];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int64_t items = (int64_t)a.B * a.H * a.nb;
  const int64_t id = (int64_t)blockIdx.x * 4 + wave;
  const bool live = id < items;
  const int64_t w = live ? id : items - 1;
  // heads innermost: the waves of one workgroup read neighbouring rows of the same tokens
  const int h = (int)(w % a.H);
  const int64_t bj = w / a.H;
  const int j = (int)(bj % a.nb), b = (int)(bj / a.nb);
  const int n0 = j * a.block;
  uint64_t seen[2];
  int count = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = i * 64 + lane, n = n0 + r;
    bool ok = r < a.block && n < a.N;
    if (ok && a.vis) ok = a.vis[(int64_t)b * a.N + n] > 0.5f;
    seen[i] = __ballot(ok);
    count += __popcll(seen[i]);
  }
  const int lr = a.D / VE, rp = 64 / lr;             // lanes of a row, rows of a step
  const int rg = lane / lr, ch = (lane - rg * lr) * VE;
  const bool in = rg < rp;
  double acc[VE] = {};
  const T *base = reinterpret_cast<const T *>(a.k) + (int64_t)b * a.sb + (int64_t)h * a.sh + ch;
  const int last = min(a.block, a.N - n0) - 1;
  for (int r0 = 0; r0 <= last; r0 += 4 * rp) {
    vec t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = min(r0 + u * rp + (in ? rg : 0), last);
      t[u] = *reinterpret_cast<const vec *>(base + (int64_t)(n0 + r) * a.sn);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = r0 + u * rp + rg;
      const bool use = in && r <= last && ((seen[r >= 64] >> (r & 63)) & 1);
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] += use ? (double)(float)t[u][e] : 0.0;
    }
  }
  if (in) {
#pragma unroll
    for (int e = 0; e < VE; ++e) part[wave][rg * a.D + ch + e] = acc[e];
  }
  __syncthreads();
  if (!live) return;
  const int64_t row = ((int64_t)b * a.H + h) * a.nb + j;
  for (int c = lane; c < a.D; c += 64) {
    double sum = 0.0;
    for (int g = 0; g < rp; ++g) sum += part[wave][g * a.D + c];
    a.means[row * a.D + c] = (float)(sum / (double)max(count, 1));
  }
  if (h == 0 && lane == 0) a.counts[(int64_t)b * a.nb + j] = count;
}

// ------------------------------------------------------------------------------------------ selection
struct SelectArgs {
  const void *q;
  const float *means;
  const int32_t *counts;
  int32_t *blocks;
  double *pooled;      // (B, Hkv, S, D)
  uint64_t *keys;      // (B, Hkv, S, nb)
  int64_t sb, sn, sh;
  int B, N, H, Hkv, G, D, nb, top, q_block, S;
  FastDiv by_g;
};

// sum of the queries of one group, 64 bits.  One wave per (item, key head, group): a row takes D / VE lanes, the wave's 64 / (D / VE) row
// sets are joined through LDS.
template <typename T>
__global__ __launch_bounds__(256) void select_pool_kernel(SelectArgs a) {
  constexpr int VE = 4;
  typedef typename SelVec<T, VE>::type vec;
  __shared__ double part[4][64 * VE];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int64_t rows = (int64_t)a.B * a.Hkv * a.S, id = (int64_t)blockIdx.x * 4 + wave;
  const bool live = id < rows;
  const int64_t w = live ? id : rows - 1;
  const int s = (int)(w % a.S);
  const int64_t bh = w / a.S;
  const int hk = (int)(bh % a.Hkv), b = (int)(bh / a.Hkv);
  const T *q = reinterpret_cast<const T *>(a.q) + (int64_t)b * a.sb + (int64_t)hk * a.G * a.sh;
  const int n0 = (int)((int64_t)s * a.q_block), n = (int)(min((int64_t)a.N, (int64_t)n0 + a.q_block) - n0) * a.G;   // (token, head) rows
  const int lr = a.D / VE, rp = 64 / lr, rg = lane / lr, ch = (lane - rg * lr) * VE;
  const bool in = rg < rp;
  double acc[VE] = {};
  for (int r0 = 0; r0 < n; r0 += 4 * rp) {
    vec t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = min(r0 + u * rp + (in ? rg : 0), n - 1), tk = (int)a.by_g.div((unsigned)r);
      t[u] = *reinterpret_cast<const vec *>(q + (int64_t)(n0 + tk) * a.sn + (int64_t)(r - tk * a.G) * a.sh + ch);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool use = in && r0 + u * rp + rg < n;
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] += use ? (double)(float)t[u][e] : 0.0;
    }
  }
  if (in) {
#pragma unroll
    for (int e = 0; e < VE; ++e) part[wave][rg * a.D + ch + e] = acc[e];
  }
  __syncthreads();
  if (!live) return;
  for (int c = lane; c < a.D; c += 64) {
    double sum = 0.0;
    for (int g = 0; g < rp; ++g) sum += part[wave][g * a.D + c];
    a.pooled[id * a.D + c] = sum;
  }
}

// Order-preserving map of a score to 64 bits; 0 is reserved for "cannot be chosen" (no visible key, a score of -inf or NaN).
__device__ __forceinline__ uint64_t score_key(double s, bool can) {
  s += 0.0;                                                     // -0 and +0 tie
  const uint64_t u = (uint64_t)__double_as_longlong(s);
  const uint64_t m = (u >> 63) ? ~u : (u | (1ull << 63));
  return can && s > -__builtin_inf() ? m : 0ull;
}

// scores of 16 groups x 64 blocks per wave with v_mfma_f64_16x16x4: lane l holds row (column) l % 16 of both operands and, in a
// slice of 16 channels, channels 4 (l / 16) .. + 3, one of them per instruction.
constexpr int kScoreTiles = 4;
__global__ __launch_bounds__(256) void select_score_kernel(SelectArgs a) {
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int r = lane % 16, g = lane / 16;
  const int64_t bh = blockIdx.z;
  const int s0 = blockIdx.y * 16, j0 = (blockIdx.x * 4 + wave) * 16 * kScoreTiles;
  if (j0 >= a.nb) return;
  const int b = (int)(bh / a.Hkv);
  const int s = min(s0 + r, a.S - 1);
  const double *qp = a.pooled + (bh * a.S + s) * a.D;
  f64x4 acc[kScoreTiles] = {};
  for (int c0 = 0; c0 < a.D; c0 += 16) {
    const int c = c0 + 4 * g;
    const bool in = c < a.D;                                    // D is a multiple of 8
    double qv[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) qv[e] = in ? qp[c + e] : 0.0;
#pragma unroll
    for (int t = 0; t < kScoreTiles; ++t) {
      const float *mp = a.means + (bh * a.nb + min(j0 + t * 16 + r, a.nb - 1)) * a.D;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t] = __builtin_amdgcn_mfma_f64_16x16x4f64(qv[e], in ? (double)mp[c + e] : 0.0, acc[t], 0, 0, 0);
    }
  }
  // result: column l % 16, rows l / 16 + 4 i
#pragma unroll
  for (int t = 0; t < kScoreTiles; ++t) {
    const int col = j0 + t * 16 + r;
    const bool can = col < a.nb && a.counts[(int64_t)b * a.nb + col] > 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = s0 + g + 4 * i;
      if (row < a.S && col < a.nb) a.keys[(bh * a.S + row) * a.nb + col] = score_key(acc[t][i], can);
    }
  }
}

// maximum over the wave of an unsigned value
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#define TCL_DPP(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, false))
  TCL_DPP(0x111, 0xf);   // row_shr:1, 2, 4, 8: lane 15 of each row of 16 has the row's maximum
  TCL_DPP(0x112, 0xf);
  TCL_DPP(0x114, 0xf);
  TCL_DPP(0x118, 0xf);
  TCL_DPP(0x142, 0xa);   // row_bcast:15 into rows 1 and 3
  TCL_DPP(0x143, 0xc);   // row_bcast:31 into rows 2 and 3
#undef TCL_DPP
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// The top_k largest of the keys a wave holds (R per lane, key i of a lane has index 64 i + lane): ties to the lower index, ascending,
// -1 behind the last.  The threshold is found bit by bit (how many keys are >= the candidate?), and the search ends as soon as
// exactly the wanted number passes.  The sign and exponent come from the largest key downwards (the threshold is seldom more than
// a few binades below it; if it is, the search starts at the top bit), then the upper half's other 20 bits; the lower half is looked at
// only if keys share the threshold's upper half.
template <int R> __device__ __forceinline__ void choose(const uint64_t (&key)[R], int top, int32_t *out) {
  const int lane = threadIdx.x % 64;
  uint32_t hi[R], most = 0;
  int valid = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    hi[i] = (uint32_t)(key[i] >> 32);
    most = max(most, hi[i]);
    valid += __popcll(__ballot(key[i] != 0));
  }
  const int want = min(top, valid);
  auto reach = [&](uint32_t c) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) n += __popcll(__ballot(hi[i] >= c));
    return n;
  };
  uint64_t t = 1;                                               // everything that can be chosen
  int have = valid;
  if (have > want) {
    uint32_t th = (wave_umax(most) >> 20) << 20, bit = 1u << 31;
    for (int tries = 0; tries < 4 && th >= 1u << 20; ++tries, th -= 1u << 20) {
      have = reach(th);
      if (have >= want) { bit = 1u << 19; break; }
    }
    if (bit != 1u << 19) { th = 0; have = -1; }
    while (have != want && bit) {
      const int n = reach(th | bit);
      if (n >= want) { th |= bit; have = n; }
      bit >>= 1;
    }
    t = (uint64_t)th << 32;
    if (have != want) {
      for (int low = 31; low >= 0 && have != want; --low) {
        const uint64_t cand = t | (1ull << low);
        int n = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) n += __popcll(__ballot(key[i] >= cand));
        if (n >= want) { t = cand; have = n; }
      }
    }
  }
  int at = 0;
  if (have == want) {
    if (want > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const bool in = key[i] >= t;
        const uint64_t m = __ballot(in);
        if (in) out[__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, at))] = i * 64 + lane;
        at += __popcll(m);
      }
    }
  } else {                                                      // keys equal to t, some of which have to stay out: the last ones
    int stay = want - have, eq = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) stay += __popcll(__ballot(key[i] == t));
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const bool same = key[i] == t;
      const uint64_t sm = __ballot(same);
      const bool in = key[i] >= t && (!same || eq + __popcll(sm & below) < stay);
      const uint64_t m = __ballot(in);
      if (in) out[at + __popcll(m & below)] = i * 64 + lane;
      at += __popcll(m);
      eq += __popcll(sm);
    }
  }
  for (int i = at + lane; i < top; i += 64) out[i] = -1;
}

// Scores and choice of 16 groups by one workgroup, up to 64 R blocks: the four waves share out the products' block tiles, the keys meet
// in LDS, and every wave chooses for four of the groups.  DIRECT: the groups' few queries are summed here; otherwise the sums come
// from the workspace.  DS: slices of 16 channels.
// Against scores written out and read back by a second kernel 330 -> 111 us (65,536 groups x 256 blocks, one wave per 16 groups with the keys
// in registers), -> 89 us with the waves sharing the products, -> 80 with
// the sums of the queries shared out too; two or four choices of a wave side by side are slower (93, 96);
// the products alone take 29 at the rate of a large 64-bit product, the comparisons the rest.
template <typename T, bool DIRECT, int R, int DS>
__global__ __launch_bounds__(256) void select_fused_kernel(SelectArgs a) {
  constexpr int LD = R * 64 + 16;
  extern __shared__ uint64_t lkey[];                            // [16][LD]
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int r = lane % 16, g = lane / 16;
  const int stiles = (a.S + 15) / 16;
  const int64_t bh = blockIdx.x / (unsigned)stiles;
  const int s0 = (int)(blockIdx.x - (unsigned)bh * (unsigned)stiles) * 16, hk = (int)(bh % a.Hkv), b = (int)(bh / a.Hkv);
  // the groups' query sums: this lane's row r, channels 16 c + 4 g .. + 3
  double q[DS][4];
  const int s = min(s0 + r, a.S - 1);
  if (DIRECT) {
    typedef typename SelVec<T, 4>::type vec;
    const T *qp = reinterpret_cast<const T *>(a.q) + (int64_t)b * a.sb + (int64_t)hk * a.G * a.sh;
    const int n0 = (int)((int64_t)s * a.q_block), n1 = (int)min((int64_t)a.N, (int64_t)n0 + a.q_block);
    // a quarter of the channels per wave (summed by all four, the sums cost as much as the products); they meet where the keys come later
    constexpr int LQ = DS * 16 + 2, MY = DS / 4;
    double *lq = reinterpret_cast<double *>(lkey), sum[MY][4];
#pragma unroll
    for (int c = 0; c < MY; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[c][e] = 0.0;
    for (int n = n0; n < n1; ++n)
      for (int h = 0; h < a.G; ++h)
#pragma unroll
        for (int c = 0; c < MY; ++c) {
          const int ch = (wave * MY + c) * 16 + g * 4;
          const vec t = *reinterpret_cast<const vec *>(qp + (int64_t)n * a.sn + (int64_t)h * a.sh + min(ch, a.D - 4));
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[c][e] += ch < a.D ? (double)(float)t[e] : 0.0;
        }
#pragma unroll
    for (int c = 0; c < MY; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) lq[r * LQ + (wave * MY + c) * 16 + g * 4 + e] = sum[c][e];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < DS; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) q[c][e] = lq[r * LQ + c * 16 + g * 4 + e];
    __syncthreads();
  } else {
#pragma unroll
    for (int c = 0; c < DS; ++c) {
      const int ch = c * 16 + g * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) q[c][e] = ch < a.D ? a.pooled[(bh * a.S + s) * a.D + ch + e] : 0.0;
    }
  }
  typedef float f4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int t = 0; t < R; ++t) {
    const int j = (t * 4 + wave) * 16 + r;
    const float *mp = a.means + (bh * a.nb + min(j, a.nb - 1)) * a.D;
    f4 mv[DS];
#pragma unroll
    for (int c = 0; c < DS; ++c) mv[c] = *reinterpret_cast<const f4 *>(mp + min(c * 16 + g * 4, a.D - 4));
    const bool can = a.counts[(int64_t)b * a.nb + min(j, a.nb - 1)] > 0 && j < a.nb;
    f64x4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int c = 0; c < DS; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(q[c][e], c * 16 + g * 4 < a.D ? (double)mv[c][e] : 0.0, acc, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) lkey[(g + 4 * i) * LD + j] = score_key(acc[i], can);
  }
  __syncthreads();
#pragma unroll 1
  for (int x = 0; x < 4; ++x) {
    const int row = wave * 4 + x;
    if (s0 + row >= a.S) break;
    uint64_t key[R];
#pragma unroll
    for (int i = 0; i < R; ++i) key[i] = lkey[row * LD + i * 64 + lane];
    choose<R>(key, a.top, a.blocks + (bh * a.S + s0 + row) * a.top);
  }
}

// The choice for long rows: one workgroup per row, its keys in LDS.
__global__ __launch_bounds__(256) void select_topk_block_kernel(SelectArgs a) {
  extern __shared__ uint64_t lkey[];
  __shared__ int lsum[2][4];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int64_t row = blockIdx.x;
  const int padded = (a.nb + 255) / 256 * 256;
  int flip = 0;
  auto total = [&](int n) {                                     // n is wave-uniform
    if (lane == 0) lsum[flip][wave] = n;
    __syncthreads();
    const int t = lsum[flip][0] + lsum[flip][1] + lsum[flip][2] + lsum[flip][3];
    flip ^= 1;                                                  // the other half: no second barrier needed before the next write
    return t;
  };
  auto count = [&](uint64_t c) {
    int n = 0;
    for (int j = threadIdx.x; j < padded; j += 256) n += __popcll(__ballot(lkey[j] >= c));
    return total(n);
  };
  for (int j = threadIdx.x; j < padded; j += 256) lkey[j] = j < a.nb ? a.keys[row * a.nb + j] : 0ull;
  __syncthreads();
  const int valid = count(1);
  const int want = min(a.top, valid);
  uint64_t t = 1;
  int have = valid;
  if (have > want) {
    t = 0;
    for (int bit = 63; bit >= 0 && have != want; --bit) {
      const uint64_t cand = t | (1ull << bit);
      const int n = count(cand);
      if (n >= want) { t = cand; have = n; }
    }
  }
  const int spare = have - want;
  int equal = 0;
  if (spare > 0) {
    int n = 0;
    for (int j = threadIdx.x; j < padded; j += 256) n += __popcll(__ballot(lkey[j] == t));
    equal = total(n) - spare;
  }
  int32_t *out = a.blocks + row * a.top;
  if (wave != 0) return;
  const uint64_t below = (1ull << lane) - 1;
  int at = 0, eq = 0;
  for (int j = lane; j < padded; j += 64) {
    const uint64_t key = lkey[j];
    const bool same = spare > 0 && key == t;
    const uint64_t sm = __ballot(same);
    const bool in = key >= t && want > 0 && (!same || eq + __popcll(sm & below) < equal);
    const uint64_t m = __ballot(in);
    if (in) out[at + __popcll(m & below)] = j;
    at += __popcll(m);
    eq += __popcll(sm);
  }
  for (int i = at + lane; i < a.top; i += 64) out[i] = -1;
}

constexpr int64_t kMaxBlocks = 16384;   // keys of one row in LDS: 128 KB
constexpr int kFusedBlocks = 512;       // up to 512 blocks the keys of 16 groups stay in LDS (68 KB)
constexpr int kDirectRows = 8;          // groups of up to 8 query rows are summed where they are used

static size_t pooled_bytes(int64_t B, int64_t Hkv, int64_t S, int64_t D) { return round_up((size_t)(B * Hkv * S * D) * sizeof(double), 256); }

template <typename T, bool DIRECT, int R> static int launch_fused_r(const SelectArgs &a, dim3 wg, hipStream_t s) {
  // a row's keys, or its queries' sum before them
  const int keys = R * 64 + 16, sums = DIRECT ? (a.D <= 64 ? 4 : 8) * 16 + 2 : 0;
  const size_t lds = (size_t)16 * (keys > sums ? keys : sums) * sizeof(uint64_t);
  const auto kernel = a.D <= 64 ? select_fused_kernel<T, DIRECT, R, 4> : select_fused_kernel<T, DIRECT, R, 8>;
  TCL_REQUIRE(lds_ready((const void *)kernel, lds), TCL_ERR_LAUNCH, "select_blocks: the device refuses %zu bytes of LDS", lds);
  hipLaunchKernelGGL(kernel, wg, dim3(256), lds, s, a);
  return check_launch("select_blocks");
}
template <typename T, bool DIRECT> static int launch_fused(const SelectArgs &a, dim3 wg, hipStream_t s) {
  if (a.nb <= 64) return launch_fused_r<T, DIRECT, 1>(a, wg, s);
  if (a.nb <= 256) return launch_fused_r<T, DIRECT, 4>(a, wg, s);
  return launch_fused_r<T, DIRECT, 8>(a, wg, s);
}

}  // namespace tcl

using namespace tcl;

extern "C" int tcl_block_means(const void *k, int64_t k_sb, int64_t k_sn, int64_t k_sh, const float *visible, float *means, int32_t *counts,
                               int64_t B, int64_t N, int64_t H, int64_t D, int64_t block, int dtype, void *stream) {
  TCL_REQUIRE(B >= 0 && N >= 0 && H > 0 && B < (1LL << 31) && N < (1LL << 31) && H < (1LL << 31), TCL_ERR_SHAPE, "block_means: bad shape");
  TCL_REQUIRE(D > 0 && D % 8 == 0 && D <= 128, TCL_ERR_UNSUPPORTED, "block_means: head size %ld (a multiple of 8 up to 128)", (long)D);
  TCL_REQUIRE(block == 64 || block == 128, TCL_ERR_UNSUPPORTED, "block_means: blocks of 64 or 128 keys (got %ld)", (long)block);
  TCL_REQUIRE(dtype == TCL_DT_F32 || dtype == TCL_DT_BF16 || dtype == TCL_DT_F16, TCL_ERR_UNSUPPORTED, "block_means: unknown dtype %d", dtype);
  if (B == 0 || N == 0) return TCL_OK;
  TCL_REQUIRE(k && means && counts, TCL_ERR_ARG, "block_means: null pointer");
  const int64_t ve = dtype == TCL_DT_F32 ? 4 : 8;
  TCL_REQUIRE(aligned(k, 16) && k_sb % ve == 0 && k_sn % ve == 0 && k_sh % ve == 0, TCL_ERR_ARG, "block_means: key rows must start on 16 bytes");
  MeansArgs a{k, visible, means, counts, k_sb, k_sn, k_sh, (int)B, (int)N, (int)H, (int)D, (int)block, (int)cdiv(N, block)};
  const int64_t blocks = cdiv(B * H * a.nb, 4);
  TCL_REQUIRE(blocks < (1LL << 31), TCL_ERR_SHAPE, "block_means: grid of %ld blocks", (long)blocks);
  const dim3 grid((unsigned)blocks);
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == TCL_DT_F32) hipLaunchKernelGGL((block_means_kernel<float>), grid, dim3(256), 0, s, a);
  else if (dtype == TCL_DT_BF16) hipLaunchKernelGGL((block_means_kernel<__bf16>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((block_means_kernel<_Float16>), grid, dim3(256), 0, s, a);
  return check_launch("block_means");
}

// the choice without a score in memory, and its groups' sums formed where they are used
static bool select_is_fused(int64_t nb) { return nb > 0 && nb <= kFusedBlocks; }
static bool select_is_direct(int64_t N, int64_t H, int64_t Hkv, int64_t nb, int64_t q_block) {
  return select_is_fused(nb) && (q_block < N ? q_block : N) * (H / Hkv) <= kDirectRows;
}

extern "C" size_t tcl_select_blocks_workspace_bytes(int64_t B, int64_t N, int64_t H, int64_t Hkv, int64_t D, int64_t nb, int64_t q_block) {
  if (B <= 0 || N <= 0 || H <= 0 || Hkv <= 0 || D <= 0 || nb <= 0 || q_block <= 0) return 0;
  const int64_t S = cdiv(N, q_block);
  if (select_is_direct(N, H, Hkv, nb, q_block)) return 0;
  return pooled_bytes(B, Hkv, S, D) + (select_is_fused(nb) ? 0 : round_up((size_t)(B * Hkv * S * nb) * sizeof(uint64_t), 256));
}

extern "C" int tcl_select_blocks(const void *q, int64_t q_sb, int64_t q_sn, int64_t q_sh, const float *means, const int32_t *counts, int32_t *blocks,
                                 int64_t B, int64_t N, int64_t H, int64_t Hkv, int64_t D, int64_t nb, int64_t top_k, int64_t q_block, int dtype,
                                 void *workspace, size_t workspace_bytes, void *stream) {
  TCL_REQUIRE(B >= 0 && N >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && nb >= 0 && top_k > 0 && q_block > 0, TCL_ERR_SHAPE, "select_blocks: bad shape");
  TCL_REQUIRE(B < (1LL << 31) && N < (1LL << 31) && H < (1LL << 31) && top_k < (1LL << 31) && q_block < (1LL << 31), TCL_ERR_SHAPE, "select_blocks: bad shape");
  TCL_REQUIRE(D > 0 && D % 8 == 0 && D <= 128, TCL_ERR_UNSUPPORTED, "select_blocks: head size %ld (a multiple of 8 up to 128)", (long)D);
  TCL_REQUIRE(nb <= kMaxBlocks, TCL_ERR_UNSUPPORTED, "select_blocks: %ld blocks (at most %ld)", (long)nb, (long)kMaxBlocks);
  TCL_REQUIRE(dtype == TCL_DT_F32 || dtype == TCL_DT_BF16 || dtype == TCL_DT_F16, TCL_ERR_UNSUPPORTED, "select_blocks: unknown dtype %d", dtype);
  const int64_t S = cdiv(N, q_block), rows = B * Hkv * S;
  if (rows == 0) return TCL_OK;
  TCL_REQUIRE(q && blocks && (nb == 0 || (means && counts)), TCL_ERR_ARG, "select_blocks: null pointer");
  const size_t size = dtype == TCL_DT_F32 ? 4 : 2;
  TCL_REQUIRE(aligned(q, 4 * size) && q_sb % 4 == 0 && q_sn % 4 == 0 && q_sh % 4 == 0 && aligned(means, 16), TCL_ERR_ARG,
              "select_blocks: query rows must start on 4 elements, means on 16 bytes");
  const bool fused = select_is_fused(nb), direct = select_is_direct(N, H, Hkv, nb, q_block);
  // the scores' kernel has a grid of three dimensions, which only a choice from many blocks needs
  TCL_REQUIRE(rows < (1LL << 31) && (fused || nb == 0 || (B * Hkv < 65536 && cdiv(S, 16) < 65536)), TCL_ERR_SHAPE, "select_blocks: %ld groups are too many for one call", (long)rows);
  const size_t need = tcl_select_blocks_workspace_bytes(B, N, H, Hkv, D, nb, q_block);
  TCL_REQUIRE(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need), TCL_ERR_WORKSPACE, "select_blocks: workspace of %zu bytes needed", need);
  SelectArgs a{q, means, counts, blocks, (double *)workspace, nullptr, q_sb, q_sn, q_sh, (int)B, (int)N, (int)H, (int)Hkv, (int)(H / Hkv), (int)D, (int)nb,
               (int)top_k, (int)q_block, (int)S};
  a.keys = (uint64_t *)((char *)workspace + pooled_bytes(B, Hkv, S, D));
  const hipStream_t s = (hipStream_t)stream;
  a.by_g = make_fastdiv((uint32_t)a.G);
  const int64_t per_group = (q_block < N ? q_block : N) * a.G;
  TCL_REQUIRE(per_group < (1LL << 31), TCL_ERR_SHAPE, "select_blocks: groups of %ld query rows", (long)per_group);
  if (nb > 0 && !direct) {
    const dim3 pool((unsigned)cdiv(rows, 4));
    if (dtype == TCL_DT_F32) hipLaunchKernelGGL((select_pool_kernel<float>), pool, dim3(256), 0, s, a);
    else if (dtype == TCL_DT_BF16) hipLaunchKernelGGL((select_pool_kernel<__bf16>), pool, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((select_pool_kernel<_Float16>), pool, dim3(256), 0, s, a);
  }
  if (fused) {
    TCL_REQUIRE(B * Hkv * cdiv(S, 16) < (1LL << 31), TCL_ERR_SHAPE, "select_blocks: %ld groups are too many for one call", (long)rows);
    const dim3 wg((unsigned)(B * Hkv * cdiv(S, 16)));
    if (!direct) return launch_fused<double, false>(a, wg, s);
    if (dtype == TCL_DT_F32) return launch_fused<float, true>(a, wg, s);
    if (dtype == TCL_DT_BF16) return launch_fused<__bf16, true>(a, wg, s);
    return launch_fused<_Float16, true>(a, wg, s);
  }
  if (nb > 0) hipLaunchKernelGGL(select_score_kernel, dim3((unsigned)cdiv(nb, 64 * kScoreTiles), (unsigned)cdiv(S, 16), (unsigned)(B * Hkv)), dim3(256), 0, s, a);
  const size_t lds = (size_t)(nb + 255) / 256 * 256 * sizeof(uint64_t);
  TCL_REQUIRE(lds_ready((const void *)select_topk_block_kernel, lds), TCL_ERR_LAUNCH, "select_blocks: the device refuses %zu bytes of LDS", lds);
  hipLaunchKernelGGL(select_topk_block_kernel, dim3((unsigned)rows), dim3(256), lds, s, a);
  return check_launch("select_blocks");
}
