// Attention of query tokens over the tokens of another sequence, forward.
//
//   S = scale Q K^T,  P = softmax(S) over the allowed keys,  O = P V,  lse2 = log2 sum exp2(S log2 e)
//
// One pass over the keys with the running maximum m and sum l of the softmax.  The rows of a work item are the query
// tokens of all heads that share a key head (row m = token m / G, head m % G), so that a tile of keys and values is
// staged once for the group.  Both products run transposed: S^T = K Q^T leaves a query in each lane with its scores in
// registers (maximum and sum need one exchange between the wave's halves), and is, exponentiated and rounded, the right
// operand of O^T = V^T P^T as it stands -- probabilities never touch LDS.
//
// What bounds it, and what it reaches (kernel times, medians of 300 launches; the library's large bf16 product: 1217 TFLOP/s,
// a large copy 4.8 TB/s):
//   many rows, wide heads: the matrix and the vector pipe together; 8 x 2047 x 4095, 16/4 heads of 128, bf16, a mask with
//     holes: 575 us, 957 TFLOP/s; the matrix pipe is busy 45 % of the time, the vector pipe 44 %
//   rows of an image: latency, as a sequence is only a few tiles long; 768 x 312 x 312, a head of 256, fp16: 159 us,
//     3.1 TB/s and 480 TFLOP/s (matrix pipe 21 %, vector pipe 22 %, LDS 10 %); 640 x 180 x 180, 8 heads of 32, bf16, with
//     what the backward pass needs: 78 us, 3.8 TB/s, 270 TFLOP/s
//   few rows: memory; 16 x 1 x 8192 ragged keys, 32/8 heads of 128, bf16: 75 us, 4.5 TB/s, and 4.8 of join
//   a token over 1000 keys: one workgroup a head goes through its eight tiles, 11 us
#include "attention.h"

#include <initializer_list>

namespace {

// Scores are compared and exponentiated in units of log2: p = exp2(s c - m), c = scale log2 e.  The accumulators are
// rescaled only when a maximum grows by more than AT_SLACK.  In fp16, p is rounded to numbers that end at 2^-24, and a long
// row's small probabilities, each lost, would be missed together (8192 of 2^-26 are 1.2e-4 of the row): m lies AT_LIFT below
// the maximum, so that p ends at 2^-31 of it and stays under 2^15.
constexpr float AT_SLACK = 8.0f;
template <typename T> constexpr float AT_LIFT = at_fit<T>::ON ? 7.0f : 0.0f;

struct at_split {
  float* o;     // [item][split][rows][D]: unnormalised sums
  float* ml;    // [item][split][2][rows]: maxima (in fp16 AT_LIFT below), sums
  int32_t n;    // splits of the keys
  int32_t keys; // of one split, a multiple of the tile
};

template <typename T, int DC, int NWQ, int NWK, int NKB> struct at_fwd_cfg {
  using R = at_row<T, DC>;
  static constexpr int WAVES = NWQ * NWK;
  static constexpr int ROWS = 32 * NWQ;       // query rows of a work item
  static constexpr int KT = 32 * NKB * NWK;   // keys of a tile
  static constexpr int TILE = R::tile(KT);
  static constexpr int LDS = 4 * TILE;        // keys and values, two tiles each
};

// NWQ waves side by side own 32 rows each; NWK waves share the same rows and take 32 NKB keys each of every tile.
template <typename T, int DC, int NWQ, int NWK, int NKB, bool AHEAD, int OCC>
__global__ __launch_bounds__(64 * NWQ * NWK, OCC) void at_fwd_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                                     const T* __restrict__ v, T* __restrict__ out,
                                                                     T* __restrict__ rest_out, float* __restrict__ lse, at_split sp, at_args a,
                                                                     at_order order, at_div by_tiles, at_div by_splits) {
  using C = at_fwd_cfg<T, DC, NWQ, NWK, NKB>;
  using R = at_row<T, DC>;
  constexpr int NDB = DC / 32;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  int item = order.item();
  if (item < 0) return;
  int rt = 0, split, n, hk;
  if constexpr (NWK > 1) {
    // few rows: heads fastest, then splits, then sequences
    const int rest = a.by_Hk.of(item);
    hk = item - rest * a.Hk;
    n = by_splits.of(rest);
    split = rest - n * (int)by_splits.d;
    item = (n * a.Hk + hk) * (int)by_splits.d + split;
  } else {
    // rows fastest, then splits, then heads and sequences
    const int rest = by_tiles.of(item), nh = by_splits.of(rest);
    rt = item - rest * (int)by_tiles.d;
    split = rest - nh * (int)by_splits.d;
    n = a.by_Hk.of(nh);
    hk = nh - n * a.Hk;
  }

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wq = wave % NWQ, wk = wave / NWQ;
  const int c = lane & 31, h = lane >> 5;
  const int rows = a.Tq * a.G, row0 = (rt * NWQ + wq) * 32, row = row0 + c;
  const bool live = row < rows;
  const int first = min(a.by_G.of(row0), a.Tq - 1);  // the wave's first token
  const int t = live ? a.by_G.of(row) : first, g = live ? row - t * a.G : 0;

  const int len = at_length(a, n);
  const int k_begin = split * sp.keys, k_end = min(len, k_begin + sp.keys);
  const int tiles = k_end > k_begin ? (k_end - k_begin + C::KT - 1) / C::KT : 0;

  at_key_tiles<T, DC, C::KT, C::WAVES> kv;
  kv.init(a, k, v, n, hk, k_begin, k_end, wave, lane);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(at_lds)smem;
  if (tiles > 0) kv.template fetch<true, true>(a, lds0, lds0 + 2 * C::TILE, wave, lane);

  at_u4 qf[R::STEPS];
  at_rows_of(q + (int64_t)n * a.qs[0] + (int64_t)first * a.qs[1] + (int64_t)hk * a.G * a.qs[2])
      .row<T, DC>(live ? (uint32_t)(t - first) * (uint32_t)(a.qs[1] * sizeof(T)) + (uint32_t)g * (uint32_t)(a.qs[2] * sizeof(T))
                       : AT_OUTSIDE,
                  a.D, lane, qf);

  at_places<T, DC> at;
  at.init(lane);
  at_f16 acc[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i) acc[i] = (at_f16)(0.0f);
  float m = -INFINITY, l = 0.0f;
  uint32_t any = 0;

  const int kr = 32 * NKB * wk;  // this wave's first key of a tile
  const bool idle = row0 >= rows;  // this wave only helps with the loads
  // While a wave multiplies, its partner on the SIMD exponentiates; the matrix pipe is the scarcer one for wide heads
  // (2 % at 4095 keys and D 128; heads of 64 and less lose as much)
  auto priority = [](int on) {
    if constexpr (DC > 64) {
      if (on) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
    }
  };
  // the scores of a tile
  auto start = [&](at_f16 (&s)[NKB], int j) {
#pragma unroll
    for (int b = 0; b < NKB; ++b) {
      const uint32_t take = at_key_bits(a, n, k_end, k_begin + j * C::KT + kr + 32 * b);
      any |= take;
      s[b] = at_start<T>(take, lane);
    }
  };
  auto scores = [&](at_f16 (&s)[NKB], int j, const unsigned char* kt) {
    start(s, j);
#pragma unroll
    for (int st = 0; st < R::STEPS; ++st)
#pragma unroll
      for (int b = 0; b < NKB; ++b) s[b] = at_mma(T(), at.rows(kt, kr + 32 * b, st), qf[st], s[b]);
  };
  auto largest = [&](const at_f16 (&s)[NKB]) {
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < NKB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
    return at_half_max(mx) * a.scale_log2 - AT_LIFT<T>;
  };
  auto raise = [&](float mx) {
    if (__any(mx > m + AT_SLACK)) {
      const float mn = fmaxf(m, mx);
      const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int i = 0; i < NDB; ++i) acc[i] *= f;
    }
  };
  auto probabilities = [&](at_f16 (&s)[NKB]) {
    const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int b = 0; b < NKB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[b][i] = __builtin_amdgcn_exp2f(s[b][i] * a.scale_log2 - mu);
        l += s[b][i];
      }
  };
  auto values = [&](const at_f16 (&s)[NKB], const unsigned char* vt) {
#pragma unroll
    for (int b = 0; b < NKB; ++b) at_mma_cols<T, DC>(at, vt, kr + 32 * b, s[b], acc);
  };

  if constexpr (AHEAD) {
    // The scores of the next tile are multiplied while this one's are exponentiated, so that the matrix and the vector
    // pipe of a SIMD have work at the same time: the keys are fetched a tile ahead of the values.
    at_f16 s0[NKB], s1[NKB];
    if (tiles > 0) {
      at_landed();
      if (tiles > 1) kv.template fetch<true, false>(a, lds0 + C::TILE, 0u, wave, lane);
      if (!idle) {
        scores(s0, 0, smem);
        raise(largest(s0));
      }
    }
    // (behind the last tile, scores of whatever lies in LDS are multiplied; nothing looks at them)
    auto step = [&](at_f16 (&s)[NKB], at_f16 (&next)[NKB], int j, int odd) {
      at_landed();
      if (j + 2 < tiles) kv.template fetch<true, false>(a, lds0 + odd * C::TILE, 0u, wave, lane);
      if (j + 1 < tiles) kv.template fetch<false, true>(a, 0u, lds0 + (2 + (odd ^ 1)) * C::TILE, wave, lane);
      if (idle) return;
      const unsigned char* kt = smem + (odd ^ 1) * C::TILE;
      const unsigned char* vt = smem + (2 + odd) * C::TILE;
      start(next, j + 1);
      const float mu = m == -INFINITY ? 0.0f : m;
      at_u4 kf[2][NKB];
#pragma unroll
      for (int b = 0; b < NKB; ++b) kf[0][b] = at.rows(kt, kr + 32 * b, 0);
#pragma unroll
      for (int st = 0; st < R::STEPS; ++st) {
#pragma unroll
        for (int b = 0; b < NKB; ++b) {
          if (st + 1 < R::STEPS) kf[(st + 1) & 1][b] = at.rows(kt, kr + 32 * b, st + 1);
          next[b] = at_mma(T(), kf[st & 1][b], qf[st], next[b]);
#pragma unroll
          for (int i = 16 * st / R::STEPS; i < 16 * (st + 1) / R::STEPS; ++i) {
            s[b][i] = __builtin_amdgcn_exp2f(s[b][i] * a.scale_log2 - mu);
            l += s[b][i];
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      priority(1);
      constexpr int U = NKB * 2 * NDB;  // products of the values: 16 keys by 32 elements each
      float mx = next[0][0];
      at_u4 vf[2];
      at_u4 pf;
      vf[0] = at.cols(vt, kr, 0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int b = u / (2 * NDB), hf = u / NDB % 2, db = u % NDB;
        if (u + 1 < U) vf[(u + 1) & 1] = at.cols(vt, kr + 16 * ((u + 1) / NDB), (u + 1) % NDB);
        if (db == 0) {
#pragma unroll
          for (int x = 0; x < 4; ++x) pf[x] = at_pack(T(), s[b][8 * hf + 2 * x], s[b][8 * hf + 2 * x + 1]);
        }
        acc[db] = at_mma(T(), vf[u & 1], pf, acc[db]);
#pragma unroll
        for (int i = 16 * NKB * u / U; i < 16 * NKB * (u + 1) / U; ++i) mx = fmaxf(mx, next[i / 16][i % 16]);
        __builtin_amdgcn_sched_barrier(0);
      }
      priority(0);
      mx = at_half_max(mx) * a.scale_log2 - AT_LIFT<T>;
      raise(mx);
    };
    for (int j = 0; j < tiles; j += 2) {
      step(s0, s1, j, 0);
      if (j + 1 < tiles) step(s1, s0, j + 1, 1);
    }
  } else {
    for (int j = 0; j < tiles; ++j) {
      at_landed();
      if (j + 1 < tiles)
        kv.template fetch<true, true>(a, lds0 + ((j + 1) & 1) * C::TILE, lds0 + (2 + ((j + 1) & 1)) * C::TILE, wave, lane);
      if (idle) continue;
      at_f16 s[NKB];
      priority(1);
      scores(s, j, smem + (j & 1) * C::TILE);
      priority(0);
      raise(largest(s));
      probabilities(s);
      priority(1);
      values(s, smem + (2 + (j & 1)) * C::TILE);
      priority(0);
    }
  }
  l = at_half_sum(l);

  if constexpr (NWK > 1) {
    // the waves that share rows meet in LDS: each writes its maximum and sums, and takes a share of the elements
    at_sync();
    float* mbuf = reinterpret_cast<float*>(smem);                          // [WAVES][2][32]
    float* obuf = mbuf + C::WAVES * 64;                                    // [WAVES][NDB * 16][64]
    if (h == 0) {
      mbuf[wave * 64 + c] = m;
      mbuf[wave * 64 + 32 + c] = l;
    }
    reinterpret_cast<uint32_t*>(obuf + C::WAVES * NDB * 1024)[wave] = any;
#pragma unroll
    for (int i = 0; i < NDB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) obuf[((wave * NDB + i) * 16 + r) * 64 + lane] = acc[i][r];
    at_sync();
    float ms[NWK], top = -INFINITY;
    l = 0.0f;
    any = 0;
#pragma unroll
    for (int x = 0; x < NWK; ++x) {
      ms[x] = mbuf[(x * NWQ + wq) * 64 + c];
      top = fmaxf(top, ms[x]);
      any |= reinterpret_cast<const uint32_t*>(obuf + C::WAVES * NDB * 1024)[x * NWQ + wq];
    }
#pragma unroll
    for (int x = 0; x < NWK; ++x) {
      ms[x] = ms[x] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms[x] - top);
      l += ms[x] * mbuf[(x * NWQ + wq) * 64 + 32 + c];
    }
    m = top;
#pragma unroll
    for (int i = 0; i < NDB; ++i) {
      if (i % NWK != wk) continue;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float sum = 0.0f;
#pragma unroll
        for (int x = 0; x < NWK; ++x) sum += ms[x] * obuf[(((x * NWQ + wq) * NDB + i) * 16 + r) * 64 + lane];
        acc[i][r] = sum;
      }
    }
  }
  any = __builtin_amdgcn_readfirstlane(any);

  if (sp.n > 1) {
    // no key at all: sum 0; keys, but every score -inf: sum -1, which the join counts as nothing (a sum is positive or NaN)
    l = any ? (l == 0.0f ? -1.0f : l) : 0.0f;
    float* ml = sp.ml + (int64_t)item * 2 * C::ROWS + wq * 32;
    if (wk == 0 && h == 0) {
      ml[c] = m;
      ml[C::ROWS + c] = l;
    }
    float* o = sp.o + ((int64_t)item * C::ROWS + wq * 32 + c) * a.D;
#pragma unroll
    for (int i = 0; i < NDB; ++i) {
      if (NWK > 1 && i % NWK != wk) continue;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int d = 32 * i + 8 * b + 4 * h;
        const at_f4 w = {acc[i][4 * b], acc[i][4 * b + 1], acc[i][4 * b + 2], acc[i][4 * b + 3]};
        if (live && d < a.D) *reinterpret_cast<at_f4*>(o + d) = w;
      }
    }
    return;
  }
  const float f = 1.0f / l;
  const int hq = hk * a.G + g;
  T* o = out + ((int64_t)((int64_t)n * a.Tq + t) * a.Hq + hq) * a.D;
  T* r = rest_out + (o - out);
#pragma unroll
  for (int i = 0; i < NDB; ++i) {
    if (NWK > 1 && i % NWK != wk) continue;
    if (sizeof(T) == 2 && rest_out != nullptr) at_store_rows<T, 32, true>(o + 32 * i, live, any != 0, acc + i, f, a.D - 32 * i, lane, r + 32 * i);
    else at_store_rows<T, 32>(o + 32 * i, live, any != 0, acc + i, f, a.D - 32 * i, lane);
  }
  if (lse != nullptr && live && h == 0 && wk == 0)
    lse[((int64_t)n * a.Hq + hq) * a.Tq + t] = any ? m + __builtin_amdgcn_logf(l) : INFINITY;
}

// Joins the splits: a wave per row, or four.  The lanes take a split's maximum and sum each, the weights exp2(m_i - max) go to LDS;
// then a group of D / 4 lanes takes four elements each of every (64 / group)th split, many loads in flight.
// Bound by latency: 512 rows of 128 in 4 splits take 4.8 us.
constexpr int AT_MOST_SPLITS = 512;

template <typename T, int WAVES>
__global__ __launch_bounds__(256) void at_join_kernel(T* __restrict__ out, T* __restrict__ rest, float* __restrict__ lse, at_split sp, at_args a,
                                                      at_div by_rows, at_div by_tile_rows, int row_tiles, int64_t all_rows) {
  __shared__ float weights[4][AT_MOST_SPLITS];
  __shared__ at_f4 sums[4][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * (4 / WAVES) + wave / WAVES;
  if (WAVES == 1 && i >= all_rows) return;  // (a wave joins its row alone; four share a workgroup's)
  const int nh = by_rows.of((int)i), row = (int)i - nh * (int)by_rows.d;
  const int tile_rows = (int)by_tile_rows.d, rt = by_tile_rows.of(row), r = row - rt * tile_rows;
  const int64_t item0 = (int64_t)nh * sp.n * row_tiles + rt;  // + split * row_tiles
  float top = -INFINITY;
  for (int s = lane; s < sp.n; s += 64) top = fmaxf(top, sp.ml[(item0 + (int64_t)s * row_tiles) * 2 * tile_rows + r]);
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
  float l = 0.0f;
  bool keys = false;
  for (int s = lane; s < sp.n; s += 64) {
    const float* ml = sp.ml + (item0 + (int64_t)s * row_tiles) * 2 * tile_rows + r;
    const float mi = ml[0], li = ml[tile_rows];
    // a weight of -1: no key in this split.  A split of -inf alone has the weight 0: its values count if they are not finite
    const float w = li == 0.0f ? -1.0f : mi == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mi - top);
    weights[wave][s] = w;
    keys |= li != 0.0f;
    l += li == 0.0f ? 0.0f : mi == -INFINITY ? (li < 0.0f ? 0.0f : li) : w * li;  // (a NaN stays one)
  }
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) l += __shfl_xor(l, x);
  const bool none = !__any(keys);  // (keys, but a sum of 0: 0 / 0)
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  int group = 2;  // lanes of a group: D / 4 rounded up to a power of two
  while (group * 4 < a.D) group *= 2;
  const int e = (lane & (group - 1)) * 4, part = lane / group, parts = 64 / group, share = wave % WAVES;
  at_f4 acc = (at_f4)(0.0f);
  if (e < a.D && !none) {
    const float* o = sp.o + (item0 * tile_rows + r) * a.D + e;
    const int64_t step = (int64_t)row_tiles * tile_rows * a.D;
#pragma unroll 8
    for (int s = share * parts + part; s < sp.n; s += parts * WAVES) {
      const float w = weights[wave][s];
      if (!(w < 0.0f)) acc += w * *reinterpret_cast<const at_f4*>(o + s * step);
    }
  }
  for (int x = group; x < 64; x <<= 1)
#pragma unroll
    for (int y = 0; y < 4; ++y) acc[y] += __shfl_xor(acc[y], x);
  if constexpr (WAVES > 1) {
    sums[wave][lane] = acc;
    __syncthreads();
    if (share > 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) acc += sums[w][lane];
  }
  const int n = a.by_Hk.of(nh), hk = nh - n * a.Hk, t = a.by_G.of(row), hq = hk * a.G + row - t * a.G;
  if (e < a.D && part == 0) {
    const float f = none ? 0.0f : 1.0f / l;
    const int64_t at = (((int64_t)n * a.Tq + t) * a.Hq + hq) * a.D + e;
    if constexpr (sizeof(T) == 2) {
      const at_u2 w = {at_pack(T(), acc[0] * f, acc[1] * f), at_pack(T(), acc[2] * f, acc[3] * f)};
      *reinterpret_cast<at_u2*>(out + at) = w;
      if (rest != nullptr) {
        const at_f2 x = at_unpack(T(), w[0]), y = at_unpack(T(), w[1]);
        *reinterpret_cast<at_u2*>(rest + at) = at_u2{at_pack(T(), acc[0] * f - x[0], acc[1] * f - x[1]),
                                                     at_pack(T(), acc[2] * f - y[0], acc[3] * f - y[1])};
      }
    } else {
      *reinterpret_cast<at_f4*>(out + at) = acc * f;
    }
  }
  if (lse != nullptr && lane == 0) lse[((int64_t)n * a.Hq + hq) * a.Tq + t] = none ? INFINITY : top + __builtin_amdgcn_logf(l);
}

// The mask as one bit per key: a scalar load tells a tile which keys take part.  (Nothing is skipped for it in this pass or
// for dq: tiles go by the lengths, and one whose keys are all masked is multiplied with zeros.  Only the kernel of dk and dv
// leaves out keys of which a whole workgroup has none.)  8 x 4095 keys: 4.8 us, most of it the launch.
__global__ __launch_bounds__(256) void at_bits_kernel(const unsigned char* __restrict__ mask, int64_t stride,
                                                      uint64_t* __restrict__ bits, int64_t words, int Tk, int64_t total) {
  const int64_t w = (int64_t)at_block() * 4 + (threadIdx.x >> 6);  // a wave per word
  if (w >= total) return;
  const int64_t n = w / words, key = (w - n * words) * 64 + (threadIdx.x & 63);
  const bool on = key < Tk && mask[n * stride + key] != 0;
  const unsigned long long b = __ballot(on);
  if ((threadIdx.x & 63) == 0) bits[w] = b;
}

template <typename T, int DC, int NWQ, int NWK, int NKB, bool AHEAD, int OCC>
int at_launch(const rc_attn* a, const at_args& d, const void* q, const void* k, const void* v, void* out, void* rest, float* lse,
              at_split sp, hipStream_t st) {
  using C = at_fwd_cfg<T, DC, NWQ, NWK, NKB>;
  constexpr int lds = NWK > 1 && C::WAVES * (64 + DC / 32 * 1024 + 4) * 4 > C::LDS ? C::WAVES * (64 + DC / 32 * 1024 + 4) * 4 : C::LDS;
  static_assert(lds <= 160 * 1024, "LDS");
  constexpr auto kernel = at_fwd_kernel<T, DC, NWQ, NWK, NKB, AHEAD, OCC>;
  int rc = at_allow_lds<kernel>(lds);
  if (rc) return rc;
  const int64_t rows = a->Tq * d.G, row_tiles = (rows + C::ROWS - 1) / C::ROWS;
  // few rows: nothing is read twice, and the heads of a split, which may share cache lines, are all that stays together
  const at_order order = NWK > 1 ? at_order(a->N * sp.n, a->Hk) : at_order(a->N, a->Hk, sp.n * row_tiles);
  kernel<<<order.grid(), 64 * C::WAVES, lds, st>>>((const T*)q, (const T*)k, (const T*)v, (T*)out, (T*)rest, lse, sp, d,
                                                order, at_div((uint32_t)row_tiles), at_div((uint32_t)sp.n));
  rc = rc_check_launch("rc_cross_attn_fwd");
  if (rc || sp.n == 1) return rc;
  const int64_t all = a->N * a->Hk * rows;
  // many splits: four waves to a row (8 rows of 128 in 64 splits: a call 21.3 -> 18.6 us)
  auto join = [&](auto kernel, int64_t blocks) {
    kernel<<<(uint32_t)blocks, 256, 0, st>>>((T*)out, (T*)rest, lse, sp, d, at_div((uint32_t)rows), at_div(C::ROWS), (int)row_tiles, all);
  };
  if (sp.n > 8) join(at_join_kernel<T, 4>, all);
  else join(at_join_kernel<T, 1>, (all + 3) / 4);
  return rc_check_launch("rc_cross_attn_fwd (join)");
}

int at_padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : D <= 192 ? 192 : 256; }

// How the work is cut: rows of an item, and splits of the keys.
struct at_plan {
  int few;            // rows fit one wave: four (two) waves share them and divide the keys
  int tile_rows;
  int64_t row_tiles, items;
  at_split sp;
};

at_plan at_make_plan(const rc_attn* a) {
  at_plan p = {};
  const int64_t rows = a->Tq * (a->Hq / a->Hk);
  p.few = rows <= 32;
  p.tile_rows = p.few ? 32 : 128;
  p.row_tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  p.items = a->N * a->Hk * p.row_tiles;
  // Fewer work items than fill the card twice: the keys are divided too, into as many parts as it has room for (one more
  // is a second turn: 33 x 1 x 1100, 8/8 heads of 128 in bf16, 264 items: 39 us, in two parts each 58).  A part has 256 keys
  // at least, or 128 where there are rows enough (one token over 3426 keys, 4 heads of 192: 22 us, with 128 27); in fp32,
  // whose products take sixteen times as long, 64 (128 for narrow heads, where that is the tile; 4 x 1124 keys, 4/2 heads
  // of 256: 38 us, 90 with 256).  (One token in each of 16 sequences, 8192 ragged keys, 32/8 heads of 128: 84 us; one over
  // 16384 keys, 8/1 heads: 19 us, in splits of 1024 keys 29.)
  const bool f32 = a->dtype == RC_F32;
  const int64_t unit = !f32 ? (p.few ? 256 : 128) : a->D > 32 ? 64 : 128;
  // (many rows of narrow 16-bit heads: three workgroups a CU; 300 items of 100 rows and 4000 keys, heads of 64: 90 us, 102
  // undivided; 64 such items, in eight parts: 26, in twelve 31)
  const int64_t places = !f32 && !p.few && a->D <= 64 && p.items > 128 ? 768 : 512;
  int64_t n = 1;
  if (p.items > 0 && p.items < 512) {
    n = places / p.items;
    // (fp32 keeps the matrix pipe busy with one workgroup a CU: the second turn is half as long; 3 x 1000 x 2000, 16/16 heads
    // of 64: 246 us, 285 undivided)
    if (n == 1 && f32) n = 2;
    // Joining is a launch more, and the parts of many rows are many bytes.  Up to so many keys an item goes through all of
    // them.  Few rows: 4 units (1000 keys in bf16: 14.7 against 18.9 us a call); fp32 heads beyond 128, which one wave goes
    // through alone, one.  Many rows, by the number of items (us, undivided and divided; heads of 64, 128 and 256 in 16
    // bits): 64 items of 300 keys 13, 13, 24 and 18, 19, 25; of 1000 20, 28, 61 and 18, 23, 38; 130 items of 1000 keys 21,
    // 28, 75 and 23, 31, 58; 256 items of 1000 keys 22, 36, 85 and 31, 47, 85, of 4000 92, 130, 293 and 75, 120, 225.  fp32,
    // heads of 128: 40 items of 200 keys 37 and 25; heads of 64: 64 items of 300 keys 27 and 23, 130 items 28 and 34, of
    // 1000 keys 80 and 67; 256 items of 1000 keys 88 and 92, 300 items 146 and 130.
    int64_t alone = (f32 && a->D > 128 ? 1 : 4) * unit;
    if (!p.few) {
      if (f32) alone = p.items <= 64 && a->D > 64 ? 128 : p.items <= 170 ? 256 : p.items <= 256 ? 1024 : 768;
      else if (a->D > 128) alone = p.items <= 170 ? 512 : 1024;
      else alone = p.items <= 64 ? 512 : p.items <= 170 ? 1024 : 2048;
    }
    if (a->Tk <= alone) n = 1;
    const int64_t most = (a->Tk + unit - 1) / unit;
    n = n < most ? n : most;
    n = n < AT_MOST_SPLITS ? n : AT_MOST_SPLITS;
    n = n < 1 ? 1 : n;
  }
  const int64_t keys = ((a->Tk + n - 1) / n + unit - 1) / unit * unit;
  p.sp.n = (int)(keys ? (a->Tk + keys - 1) / keys : 1);
  if (p.sp.n < 1) p.sp.n = 1;
  p.sp.keys = (int)(keys ? keys : unit);
  return p;
}

template <typename T, int DC>
int at_run(const rc_attn* a, const at_args& d, const void* q, const void* k, const void* v, void* out, void* rest, float* lse,
           const at_plan& p, hipStream_t st) {
  // waves of an item's keys, blocks of keys of a wave in a tile, resident workgroups: what registers and 160 KiB of LDS
  // allow.  Few rows: two workgroups per CU, so that one streams while the other starts or ends (D 128: two waves a
  // workgroup; with four, and one workgroup, 8192 ragged keys took 110 instead of 84 us)
  constexpr int RB = at_row<T, DC>::RB;
  constexpr int NWK = RB >= 1024 ? 1 : RB >= 256 ? 2 : 4;
  constexpr int NKB = RB >= 512 ? 1 : 2;
  constexpr int OCC = RB >= 1024 ? 1 : DC * (int)sizeof(T) >= 192 ? 2 : 3;
  // AHEAD: 16-bit heads of 96 and 128 (8 x 2047 x 4095, 16/4 heads of 128: 620 against 680 us, 800 x 800: 122 against
  // 138).  Narrower heads are held up by the exponentials either way and have four waves per SIMD to hide them with
  // (D 64: 332 against 328 us, 312 x 312: 167 against 148); wider ones have no registers for a second tile of scores.
  constexpr bool AHEAD = sizeof(T) == 2 && DC > 64 && DC <= 128;
  if (p.few) return at_launch<T, DC, 1, NWK, 1, false, 1>(a, d, q, k, v, out, rest, lse, p.sp, st);
  return at_launch<T, DC, 4, 1, NKB, AHEAD, (AHEAD ? 2 : OCC)>(a, d, q, k, v, out, rest, lse, p.sp, st);
}

template <typename T>
int at_run_d(const rc_attn* a, const at_args& d, const void* q, const void* k, const void* v, void* out, void* rest, float* lse,
             const at_plan& p, hipStream_t st) {
  switch (at_padded(a->D)) {
    case 32: return at_run<T, 32>(a, d, q, k, v, out, rest, lse, p, st);
    case 64: return at_run<T, 64>(a, d, q, k, v, out, rest, lse, p, st);
    case 96: return at_run<T, 96>(a, d, q, k, v, out, rest, lse, p, st);
    case 128: return at_run<T, 128>(a, d, q, k, v, out, rest, lse, p, st);
    case 192: return at_run<T, 192>(a, d, q, k, v, out, rest, lse, p, st);
    default: return at_run<T, 256>(a, d, q, k, v, out, rest, lse, p, st);
  }
}

}  // namespace

int at_check(const rc_attn* a) {
  RC_REQUIRE(a != nullptr, RC_EINVAL, "rc_cross_attn: null description");
  RC_REQUIRE(a->dtype == RC_F32 || a->dtype == RC_F16 || a->dtype == RC_BF16, RC_EUNSUPPORTED, "unknown dtype %d", a->dtype);
  RC_REQUIRE(a->D >= 8 && a->D <= RC_HEAD_DIM_MAX && a->D % 8 == 0, RC_EUNSUPPORTED,
             "head dimension %d is no multiple of 8 in 8..%d", a->D, RC_HEAD_DIM_MAX);
  RC_REQUIRE(a->N >= 0 && a->N < (1ll << 31) && a->Tq >= 0 && a->Tk >= 0 && a->Hq >= 1 && a->Hk >= 1, RC_EINVAL,
             "rc_cross_attn: negative size, or no head");
  RC_REQUIRE(a->Hq % a->Hk == 0, RC_EINVAL, "rc_cross_attn: %d query heads are no multiple of %d key heads", a->Hq, a->Hk);
  RC_REQUIRE(a->Tq < (1ll << 30) && a->Tk < (1ll << 30) && a->N * a->Tq < (1ll << 31) && a->N * a->Tk < (1ll << 31) &&
                 a->N * a->Tq * a->Hq < (1ll << 31) && a->N * a->Tk * a->Hk < (1ll << 31) && a->N * a->Hk < (1ll << 31),
             RC_EINVAL, "rc_cross_attn: more than 2^31 heads");
  // (scale log2 e has to be finite too: an infinite factor makes NaN of a score of zero)
  RC_REQUIRE(a->scale > 0.0f && a->scale < 0x1p127f, RC_EINVAL, "rc_cross_attn: scale must be positive and below 2^127");
  const int64_t es = a->dtype == RC_F32 ? 4 : 2;
  const int64_t* st[3] = {a->q_stride, a->k_stride, a->v_stride};
  for (int o = 0; o < 3; ++o)
    for (int i = 0; i < 3; ++i)
      RC_REQUIRE(st[o][i] >= 0 && st[o][i] * es % 16 == 0 && (i == 0 || st[o][i] * es < (1ll << 23)), RC_EINVAL,
                 "rc_cross_attn: stride %lld of %c is negative, no multiple of 16 bytes, or 8 MiB or more between tokens "
                 "or heads", (long long)st[o][i], "qkv"[o]);
  RC_REQUIRE((int64_t)a->Hq * a->q_stride[2] * es < (1ll << 30), RC_EINVAL,
             "rc_cross_attn: the heads of a query token span 1 GiB or more");
  RC_REQUIRE((int64_t)a->Hq * a->D * es < (1ll << 23), RC_EINVAL, "rc_cross_attn: a query token of 8 MiB or more");
  RC_REQUIRE(a->key_mask == nullptr || a->mask_stride >= 0, RC_EINVAL, "rc_cross_attn: negative mask stride");
  return RC_OK;
}

int at_check_operand(const rc_attn* a, int64_t rows, const void* p) {
  RC_REQUIRE(rows == 0 || (p != nullptr && (uintptr_t)p % 16 == 0), RC_EINVAL,
             "rc_cross_attn: an operand is null or not aligned to 16 bytes");
  return RC_OK;
}

at_args at_to_dev(const rc_attn* a, void* bits) {
  at_args d;
  for (int i = 0; i < 3; ++i) {
    d.qs[i] = a->q_stride[i];
    d.ks[i] = a->k_stride[i];
    d.vs[i] = a->v_stride[i];
  }
  d.lengths = a->key_lengths;
  d.bits = a->key_mask && a->Tk ? (const uint64_t*)bits : nullptr;
  d.words = (a->Tk + 63) / 64;
  d.N = (int32_t)a->N;
  d.Tq = (int32_t)a->Tq;
  d.Tk = (int32_t)a->Tk;
  d.Hq = a->Hq;
  d.Hk = a->Hk;
  d.G = a->Hq / a->Hk;
  d.D = a->D;
  d.by_Hk = at_div((uint32_t)d.Hk);
  d.by_G = at_div((uint32_t)d.G);
  d.lengths_i64 = a->lengths_i64;
  d.scale = a->scale;
  d.scale_log2 = a->scale * 1.44269504088896340736f;
  return d;
}

int64_t at_bits_bytes(const rc_attn* a) {
  return a->key_mask ? (a->N * ((a->Tk + 63) / 64) * 8 + 255) / 256 * 256 : 0;
}

int at_launch_bits(const rc_attn* a, void* bits, hipStream_t st) {
  const int64_t words = (a->Tk + 63) / 64, total = a->N * words;
  if (a->key_mask == nullptr || total == 0) return RC_OK;
  at_bits_kernel<<<at_grid((total + 3) / 4), 256, 0, st>>>(a->key_mask, a->mask_stride, (uint64_t*)bits, words, (int)a->Tk, total);
  return rc_check_launch("rc_cross_attn (mask)");
}

extern "C" int64_t rc_cross_attn_fwd_work_bytes(const rc_attn* a) {
  const int rc = at_check(a);
  if (rc) return rc < 0 ? rc : RC_EINVAL;
  const at_plan p = at_make_plan(a);
  const int64_t parts = p.sp.n > 1 ? p.items * p.sp.n * p.tile_rows * (a->D + 2) * (int64_t)sizeof(float) : 0;
  return at_bits_bytes(a) + parts;
}

extern "C" int rc_cross_attn_fwd(const rc_attn* a, const void* q, const void* k, const void* v, void* out, void* rest, float* lse,
                                 void* work, void* stream) {
  int rc = at_check(a);
  if (rc) return rc;
  for (const void* p : {q, (const void*)out})
    if ((rc = at_check_operand(a, a->N * a->Tq, p))) return rc;
  RC_REQUIRE((uintptr_t)rest % 16 == 0, RC_EINVAL, "rc_cross_attn_fwd: rest is not aligned to 16 bytes");
  for (const void* p : {k, v})
    if ((rc = at_check_operand(a, a->N * a->Tk, p))) return rc;
  if (a->N * a->Tq == 0) return RC_OK;
  at_plan p = at_make_plan(a);
  RC_REQUIRE((p.sp.n == 1 && at_bits_bytes(a) == 0) || (work != nullptr && (uintptr_t)work % 16 == 0), RC_EINVAL,
             "rc_cross_attn_fwd: work is null or not aligned to 16 bytes");
  RC_REQUIRE(p.items * p.sp.n < (1ll << 31) - 8, RC_EINVAL, "rc_cross_attn_fwd: too many rows");
  hipStream_t st = (hipStream_t)stream;
  if ((rc = at_launch_bits(a, work, st))) return rc;
  p.sp.o = reinterpret_cast<float*>(reinterpret_cast<char*>(work) + at_bits_bytes(a));
  p.sp.ml = p.sp.o + p.items * p.sp.n * p.tile_rows * a->D;
  const at_args d = at_to_dev(a, work);
  if (a->dtype == RC_F32) return at_run_d<float>(a, d, q, k, v, out, rest, lse, p, st);
  if (a->dtype == RC_F16) return at_run_d<rc_half>(a, d, q, k, v, out, rest, lse, p, st);
  return at_run_d<rc_bf16>(a, d, q, k, v, out, rest, lse, p, st);
}
