// Attention of query tokens over the tokens of another sequence, backward.
//
//   P = exp2(S c - lse2),  delta = sum_d dO O,  dS = P (dO V^T - delta)
//   dV = P^T dO,  dQ = scale dS K,  dK = scale dS^T Q
//
// Two kernels, each of which owns what it adds up, so there are no atomics and every run gives the same bits; the price
// is that S and dO V^T are worked out twice (7 products instead of 5).
//   at_dq_kernel   a wave has 32 query rows and goes through the keys: S^T = K Q^T and dP^T = V dO^T leave a query in
//                  each lane, dS^T is the right operand of dQ^T = K^T dS^T as it stands.  It also works out delta (and that
//                  alone where dq is not wanted).
//   at_dkv_kernel  a wave has 32 keys and goes through the query rows of all heads that share them: S = Q K^T and
//                  dP = dO V^T leave a key in each lane; dV^T = dO^T P, dK^T = Q^T dS.
//
// Bound by latency: a wave's blocks of scores go through product, exponential, product, difference and product one after
// the other, with two or four waves a SIMD, and no unit is full.  2 x 2048 x 4096 ragged keys, 16/4 heads of 128, bf16
// (medians of 300 launches): 189 us (dq; matrix pipe busy 40 %, vector pipe 29 %, LDS 20 %) and 254 us (dk and dv; 37 %,
// 25 %, 28 %), 890 and 880 TFLOP/s of the products that they work out; with the forward's 139 us 574 us a training step.
// Each product's left operand comes from LDS, once for every 32 queries or keys of a wave (with 64, the sums alone would
// take all registers).  16-bit heads of 96 and 128: two waves share 32 keys, with the values in LDS, so that four waves run
// on a SIMD instead of two (650 -> 615 us).
#include "attention.h"

#include <initializer_list>

namespace {

struct at_parts {
  float* p;       // [split][...]: fp32 parts in the result's layout; NULL: one split, the result itself is written
  int64_t part;   // elements of one split
  int32_t n;      // splits
  int32_t per;    // keys, or tiles of query rows, of one split
};

template <typename T, int DC, int KT, int WAVES> struct at_dq_lds {
  static constexpr int TILE = at_row<T, DC>::tile(KT);
  static constexpr int BYTES = 4 * TILE;
};

template <typename T, int DC, int NW, int NKB, int OCC>
__global__ __launch_bounds__(64 * NW, OCC) void at_dq_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                             const T* __restrict__ v, const T* __restrict__ out,
                                                             const T* __restrict__ rest_out, const float* __restrict__ lse, const T* __restrict__ dout,
                                                             float* __restrict__ delta, T* __restrict__ dq, at_parts sp,
                                                             at_args a, at_order order, at_div by_tiles, at_div by_splits) {
  using R = at_row<T, DC>;
  constexpr int NDB = DC / 32, KT = 32 * NKB;
  constexpr int TILE = at_dq_lds<T, DC, KT, NW>::TILE;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int item = order.item();
  if (item < 0) return;
  const int rest = by_tiles.of(item), rt = item - rest * (int)by_tiles.d;
  const int nh = by_splits.of(rest), split = rest - nh * (int)by_splits.d;
  const int n = a.by_Hk.of(nh), hk = nh - n * a.Hk;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 31, h = lane >> 5;
  const int row0 = (rt * NW + wave) * 32, row = row0 + c;
  const bool live = row < a.Tq * a.G;
  const int first = min(a.by_G.of(row0), a.Tq - 1);  // the wave's first token
  const int t = live ? a.by_G.of(row) : first, g = live ? row - t * a.G : 0, hq = hk * a.G + g;

  const int len = at_length(a, n);
  const int k_begin = split * sp.per, k_end = min(len, k_begin + sp.per);
  // (without dq only delta is wanted: no keys)
  const int tiles = dq != nullptr && k_end > k_begin ? (k_end - k_begin + KT - 1) / KT : 0;
  at_key_tiles<T, DC, KT, NW> kv;
  kv.init(a, k, v, n, hk, k_begin, k_end, wave, lane);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(at_lds)smem;
  if (tiles > 0) kv.template fetch<true, true>(a, lds0, lds0 + 2 * TILE, wave, lane);

  const int64_t orow = (((int64_t)n * a.Tq + t) * a.Hq + hq) * a.D, srow = ((int64_t)n * a.Hq + hq) * a.Tq + t;
  at_u4 qf[R::STEPS], gf[R::STEPS];
  at_rows_of(q + (int64_t)n * a.qs[0] + (int64_t)first * a.qs[1] + (int64_t)hk * a.G * a.qs[2])
      .row<T, DC>(live ? (uint32_t)(t - first) * (uint32_t)(a.qs[1] * sizeof(T)) + (uint32_t)g * (uint32_t)(a.qs[2] * sizeof(T))
                       : AT_OUTSIDE,
                  a.D, lane, qf);
  const int64_t obase = (((int64_t)n * a.Tq + first) * a.Hq + hk * a.G) * a.D;
  const uint32_t ooff = live ? (uint32_t)(orow - obase) * (uint32_t)sizeof(T) : AT_OUTSIDE;
  at_rows_of(dout + obase).row<T, DC>(ooff, a.D, lane, gf);
  const float ls = live ? lse[srow] : INFINITY;
  float dl = 0.0f;
  {
    const at_rows_of of(out + obase);
#pragma unroll
    for (int s = 0; s < R::STEPS; ++s) {
      dl += at_dot(T(), of.chunk<T>(ooff, a.D, s, h), gf[s]);
      if (s % 8 == 7) asm volatile("" ::: "memory");  // (not all of the row at once: registers)
    }
    if (sizeof(T) == 2 && rest_out != nullptr) {
      const at_rows_of rf(rest_out + obase);
#pragma unroll
      for (int s = 0; s < R::STEPS; ++s) {
        dl += at_dot(T(), rf.chunk<T>(ooff, a.D, s, h), gf[s]);
        if (s % 8 == 7) asm volatile("" ::: "memory");
      }
    }
    dl = at_half_sum(dl);
    if (live && h == 0 && split == 0) delta[srow] = dl;
  }
  at_places<T, DC> at;
  at.init(lane);
  at_f16 acc[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i) acc[i] = (at_f16)(0.0f);
  at_fit<T> fit;
  uint32_t any = 0;

  for (int j = 0; j < tiles; ++j) {
    at_landed();
    if (j + 1 < tiles) kv.template fetch<true, true>(a, lds0 + ((j + 1) & 1) * TILE, lds0 + (2 + ((j + 1) & 1)) * TILE, wave, lane);
    const unsigned char* kt = smem + (j & 1) * TILE;
    const unsigned char* vt = smem + (2 + (j & 1)) * TILE;
    if (DC <= 64 && row0 >= a.Tq * a.G) continue;  // (this wave only helps with the loads)
#pragma unroll
    for (int b = 0; b < NKB; ++b) {
      // (a key that takes no part has the score -inf, so P = 0, and zeros for its value, so dP = 0)
      const uint32_t take = at_key_bits(a, n, k_end, k_begin + j * KT + 32 * b);
      any |= take;
      at_f16 s = at_start<T>(take, lane), dp = (at_f16)(0.0f);
#pragma unroll
      for (int st = 0; st < R::STEPS; ++st) {
        s = at_mma(T(), at.rows(kt, 32 * b, st), qf[st], s);
        dp = at_mma(T(), at.rows(vt, 32 * b, st), gf[st], dp);
        if (R::RB >= 1024 && st % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // registers: no reading further ahead
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(s[i] * a.scale_log2 - ls) * (dp[i] - dl);
      fit.template fit<NDB>(s, acc);
      at_mma_cols<T, DC>(at, kt, 32 * b, s, acc);
    }
  }
  if (dq == nullptr) return;
  const float f = a.scale * fit.undo();
  if (sp.n > 1) at_store_rows<float, DC>(sp.p + split * sp.part + orow, live, any != 0, acc, f, a.D, lane);
  else at_store_rows<T, DC>(dq + orow, live, any != 0, acc, f, a.D, lane);
}

// HALVES = 2: two waves share 32 keys and take every other block of query rows; their values lie in LDS
template <typename T, int DC, int RT, int NW, int HALVES> struct at_dkv_lds {
  static constexpr int TILE = at_row<T, DC>::tile(RT);
  static constexpr int STAT = 256;  // bytes of a tile's lse2 (delta): 64 floats, what one load moves
  static constexpr int V = 4 * TILE + 4 * STAT;
  static constexpr int K = V + at_row<T, DC>::tile(32 * NW);  // (fp16: its scaling takes the registers that K has in bf16)
  static constexpr int BYTES = HALVES == 1 ? V : at_fit<T>::ON ? K + at_row<T, DC>::tile(32 * NW) : K;
  static_assert(HALVES == 1 || NW * DC / 32 * 16 * 64 * 4 <= V, "a wave's sums pass through the tiles' place");
};

// rows t0 .. of one query head: Q, dO, lse2 and delta (behind the last row: its Q and lse2 again, zeros for the others)
template <typename T, int DC, int RT, int NW> struct at_query_tiles {
  using S = at_stage<T, DC, RT, NW>;
  S sq, sg;

  __device__ __forceinline__ void init(const at_args& a, int wave, int lane) {
    sq.init(wave, lane, a.D, (uint32_t)(a.qs[1] * sizeof(T)));
    sg.init(wave, lane, a.D, (uint32_t)(a.Hq * a.D * (int)sizeof(T)));
  }
  __device__ __forceinline__ void fetch(const at_args& a, const T* q, const T* dout, const float* lse, const float* delta, int n,
                                        int hq, int t0, uint32_t lds_q, uint32_t lds_g, uint32_t lds_l, uint32_t lds_d, int wave,
                                        int lane) const {
    const int left = a.Tq - t0;
    const char* qp = reinterpret_cast<const char*>(q + (int64_t)n * a.qs[0] + (int64_t)t0 * a.qs[1] + (int64_t)hq * a.qs[2]);
    const char* gp = reinterpret_cast<const char*>(dout + (((int64_t)n * a.Tq + t0) * a.Hq + hq) * a.D);
    uint32_t outside[S::N];
    if (left >= RT) {
      sq.template issue<true>(qp, lds_q, wave, outside);
      sg.template issue<true>(gp, lds_g, wave, outside);
    } else {
      uint32_t words[RT / 32];
#pragma unroll
      for (int i = 0; i < RT / 32; ++i) words[i] = at_first_bits(left - 32 * i);
      S::spread(words, wave, lane, outside);
      sq.issue_repeat(qp, lds_q, wave, lane, left - 1);
      sg.template issue<false>(gp, lds_g, wave, outside);
    }
    const int64_t srow = ((int64_t)n * a.Hq + hq) * a.Tq + t0;
    if (wave == 0) at_fetch_floats<true>(lse + srow, left, lds_l, lane);
    if (wave == NW - 1) at_fetch_floats(delta + srow, left, lds_d, lane);
  }
};

template <typename T, int DC, int NW, int HALVES, int NRB, bool DO_K, bool DO_V, int OCC>
__global__ __launch_bounds__(64 * NW * HALVES, OCC) void at_dkv_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                              const T* __restrict__ v, const float* __restrict__ lse,
                                                              const T* __restrict__ dout, const float* __restrict__ delta,
                                                              T* __restrict__ dk, T* __restrict__ dv, at_parts sp, at_args a,
                                                              at_order order, at_div by_tiles, at_div by_splits, at_div by_rows) {
  using R = at_row<T, DC>;
  constexpr int NDB = DC / 32, RT = 32 * NRB;
  using L = at_dkv_lds<T, DC, RT, NW, HALVES>;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int item = order.item();
  if (item < 0) return;
  const int rest = by_tiles.of(item), kt = item - rest * (int)by_tiles.d;
  const int nh = by_splits.of(rest), split = rest - nh * (int)by_splits.d;
  const int n = a.by_Hk.of(nh), hk = nh - n * a.Hk, row_tiles = (int)by_rows.d;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 31, h = lane >> 5;
  const int kw = wave % NW, half = wave / NW;
  const int key0 = (kt * NW + kw) * 32, key = key0 + c;
  const int len = at_length(a, n);
  const uint32_t mine = at_key_bits(a, n, len, key0);
  const bool live = key < a.Tk, takes = (mine >> c) & 1;

  // tiles of query rows, all heads of the group one after the other; none if no key of the workgroup takes part
  uint32_t some = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) some |= at_key_bits(a, n, len, (kt * NW + w) * 32);
  const int begin = split * sp.per, end = some ? min(a.G * row_tiles, begin + sp.per) : begin;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(at_lds)smem;
  const uint32_t stat0 = lds0 + 4 * L::TILE;
  at_query_tiles<T, DC, RT, NW * HALVES> qt;
  qt.init(a, wave, lane);
  int g = row_tiles ? by_rows.of(begin) : 0, t0 = (begin - g * row_tiles) * RT;  // of the tile that is fetched next
  auto fetch = [&](int buf) {
    qt.fetch(a, q, dout, lse, delta, n, hk * a.G + g, t0, lds0 + buf * L::TILE, lds0 + (2 + buf) * L::TILE, stat0 + buf * L::STAT,
             stat0 + (2 + buf) * L::STAT, wave, lane);
    t0 += RT;
    if (t0 >= a.Tq) {
      t0 = 0;
      ++g;
    }
  };
  if (begin < end) fetch(0);

  constexpr bool V_LDS = HALVES > 1, K_LDS = HALVES > 1 && at_fit<T>::ON;
  at_u4 kf[K_LDS ? 1 : R::STEPS], vf[V_LDS ? 1 : R::STEPS];
  const T* kp = k + (int64_t)n * a.ks[0] + (int64_t)key0 * a.ks[1] + (int64_t)hk * a.ks[2];
  const T* vp = v + (int64_t)n * a.vs[0] + (int64_t)key0 * a.vs[1] + (int64_t)hk * a.vs[2];
  const uint32_t kst = (uint32_t)(a.ks[1] * sizeof(T)), vst = (uint32_t)(a.vs[1] * sizeof(T));
  const unsigned char *vs = smem + L::V + R::at(32) * kw, *ks = smem + L::K + R::at(32) * kw;
#pragma unroll
  for (int i = 0; i < 32 * R::RB / 1024; ++i) {
    if (i % HALVES != half) continue;
    if constexpr (V_LDS) at_fetch_rows<T, DC>(vp, vst, a.D, mine, lds0 + L::V + R::at(32) * kw, i, lane);
    if constexpr (K_LDS) at_fetch_rows<T, DC>(kp, kst, a.D, mine, lds0 + L::K + R::at(32) * kw, i, lane);
  }
  if constexpr (!K_LDS) at_rows_of(kp).row<T, DC>(takes ? (uint32_t)c * kst : AT_OUTSIDE, a.D, lane, kf);
  if constexpr (!V_LDS && DO_K) at_rows_of(vp).row<T, DC>(takes ? (uint32_t)c * vst : AT_OUTSIDE, a.D, lane, vf);
  at_places<T, DC> at;
  at.init(lane);
  at_f16 acck[DO_K ? NDB : 1], accv[DO_V ? NDB : 1];
#pragma unroll
  for (int i = 0; i < NDB; ++i) {
    if constexpr (DO_K) acck[i] = (at_f16)(0.0f);
    if constexpr (DO_V) accv[i] = (at_f16)(0.0f);
  }
  at_fit<T> fit;

  for (int j = begin; j < end; ++j) {
    const int buf = (j - begin) & 1;
    at_landed();
    if (j + 1 < end) fetch(buf ^ 1);
    const unsigned char* qs = smem + buf * L::TILE;
    const unsigned char* gs = smem + (2 + buf) * L::TILE;
    const float* ls = reinterpret_cast<const float*>(smem + 4 * L::TILE + buf * L::STAT);
    const float* ds = reinterpret_cast<const float*>(smem + 4 * L::TILE + (2 + buf) * L::STAT);
    if (DC <= 64 && mine == 0) continue;  // (none of this wave's keys takes part: it only helps with the loads)
#pragma unroll
    for (int bb = 0; bb < NRB / HALVES; ++bb) {
      const int b = bb + half * (NRB / HALVES);
      // (a key that takes no part has the score -inf, so P = 0, and zeros for its value, so dP = 0)
      at_f16 s = at_start<T, true>(mine, lane);
#pragma unroll
      for (int st = 0; st < R::STEPS; ++st) s = at_mma(T(), at.rows(qs, 32 * b, st), K_LDS ? at.rows(ks, 0, st) : kf[K_LDS ? 0 : st], s);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const at_f4 l4 = *reinterpret_cast<const at_f4*>(ls + 32 * b + 8 * x + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * x + i] = __builtin_amdgcn_exp2f(s[4 * x + i] * a.scale_log2 - (l4[i] - AT_P_LIFT<T>));
      }
      if constexpr (DO_V) at_mma_cols<T, DC>(at, gs, 32 * b, s, accv);
      if constexpr (DO_K) {
        at_f16 dp = (at_f16)(0.0f);
#pragma unroll
        for (int st = 0; st < R::STEPS; ++st) dp = at_mma(T(), at.rows(gs, 32 * b, st), V_LDS ? at.rows(vs, 0, st) : vf[V_LDS ? 0 : st], dp);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const at_f4 d4 = *reinterpret_cast<const at_f4*>(ds + 32 * b + 8 * x + 4 * h);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[4 * x + i] *= dp[4 * x + i] - d4[i];
        }
        fit.template fit<NDB>(s, acck);
        at_mma_cols<T, DC>(at, qs, 32 * b, s, acck);
      }
    }
  }
  const int64_t o = (((int64_t)n * a.Tk + key) * a.Hk + hk) * a.D;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the values' loads to LDS, where no row has waited for them)
  if constexpr (HALVES > 1) {
    // the other wave's sums, one of the two at a time
    float* meet = reinterpret_cast<float*>(smem) + kw * NDB * 1024 + lane;
    const float uk = fit.undo();
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      at_f16* acc = x ? accv : acck;
      const float u = x ? 1.0f : uk;
      at_sync();
      if (half == 1) {
#pragma unroll
        for (int i = 0; i < NDB; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) meet[(i * 16 + r) * 64] = acc[i][r] * u;
      }
      at_sync();
      if (half == 0) {
#pragma unroll
        for (int i = 0; i < NDB; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][r] = acc[i][r] * u + meet[(i * 16 + r) * 64];
      }
    }
    if (half == 1) return;
    fit = at_fit<T>();
  }
  const float unlift = at_fit<T>::ON ? 1.0f / 4096.0f : 1.0f;
  const float fk = a.scale * fit.undo() * unlift, fv = unlift;
  const bool keep = (mine >> c) & 1;
  if (sp.n > 1) {
    float* p = sp.p + (int64_t)split * 2 * sp.part + o;
    if constexpr (DO_K) at_store_rows<float, DC>(p, live, keep, acck, fk, a.D, lane);
    if constexpr (DO_V) at_store_rows<float, DC>(p + sp.part, live, keep, accv, fv, a.D, lane);
  } else {
    if constexpr (DO_K) at_store_rows<T, DC>(dk + o, live, keep, acck, fk, a.D, lane);
    if constexpr (DO_V) at_store_rows<T, DC>(dv + o, live, keep, accv, fv, a.D, lane);
  }
}

// The splits' parts, added in their order; four elements per thread.
template <typename T>
__global__ __launch_bounds__(256) void at_add_kernel(const float* __restrict__ p, int64_t stride, int n, T* __restrict__ out,
                                                     int64_t quads) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads) return;
  at_f4 s = *reinterpret_cast<const at_f4*>(p + 4 * i);
  for (int x = 1; x < n; ++x) s += *reinterpret_cast<const at_f4*>(p + x * stride + 4 * i);
  typedef T t4 __attribute__((ext_vector_type(4)));
  t4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = rc_from_float<T>(s[e]);
  *reinterpret_cast<t4*>(out + 4 * i) = o;
}

// What a call of these sizes needs: splits where there are too few work items, and the scratch of their parts.
struct at_bwd_plan {
  int64_t q_tiles, k_tiles, q_items, k_items;
  int q_splits, k_splits, q_per;
  int64_t bits, delta, parts;  // bytes
};

constexpr int AT_TILE_ROWS = 128;  // query rows, or keys, of a work item

at_bwd_plan at_make_bwd_plan(const rc_attn* a) {
  at_bwd_plan p = {};
  const int64_t rows = a->Tq * (a->Hq / a->Hk), groups = a->N * a->Hk;
  p.q_tiles = (rows + AT_TILE_ROWS - 1) / AT_TILE_ROWS;
  p.k_tiles = (a->Tk + AT_TILE_ROWS - 1) / AT_TILE_ROWS;
  p.q_items = groups * p.q_tiles;
  p.k_items = groups * p.k_tiles;
  // work items that fill the card: narrow heads have two workgroups or more per CU (2048 x 4096, 16/4 heads of 128 with
  // ragged keys, a training step: 622 us, filled twice 641; 4096 x 2048, 8 heads of 64: 155 us, filled twice 142)
  const int64_t fill = a->D * (a->dtype == RC_F32 ? 4 : 2) > 128 ? 256 : 512;
  auto splits = [fill](int64_t items, int64_t most) {
    if (items == 0 || items >= fill) return 1;
    const int64_t n = fill / items;  // (no more than fill the card: the rest would be a second turn)
    return (int)(n < most ? n : most < 1 ? 1 : most);
  };
  // a split has 256 keys at least, or 256 query rows; 64 in fp32, whose products take sixteen times as long
  const int64_t least = a->dtype == RC_F32 ? 64 : 256;
  const int qs = splits(p.q_items, a->Tk / least);
  p.q_per = (int)(((a->Tk + qs - 1) / qs + 63) / 64 * 64);
  if (p.q_per < 64) p.q_per = 64;
  p.q_splits = a->Tk ? (int)((a->Tk + p.q_per - 1) / p.q_per) : 1;
  p.k_splits = splits(p.k_items, rows / least);
  p.bits = at_bits_bytes(a);
  p.delta = (a->N * a->Tq * a->Hq * 4 + 255) / 256 * 256;
  const int64_t pq = p.q_splits > 1 ? (int64_t)p.q_splits * a->N * a->Tq * a->Hq * a->D * 4 : 0;
  const int64_t pk = p.k_splits > 1 ? (int64_t)p.k_splits * 2 * a->N * a->Tk * a->Hk * a->D * 4 : 0;
  p.parts = pq > pk ? pq : pk;  // one after the other
  return p;
}

struct at_bwd_call {
  const rc_attn* a;
  at_args d;
  at_bwd_plan p;
  const void *q, *k, *v, *out, *rest, *dout;
  const float* lse;
  void *dq, *dk, *dv;
  float *delta, *parts;
  hipStream_t st;
};

template <typename T, int DC, int HALVES, int NRB, bool DO_K, bool DO_V, int OCC> int at_launch_dkv(const at_bwd_call& c) {
  constexpr int RT = 32 * NRB;
  using L = at_dkv_lds<T, DC, RT, 4, HALVES>;
  static_assert(L::BYTES <= 160 * 1024, "LDS");
  constexpr auto kernel = at_dkv_kernel<T, DC, 4, HALVES, NRB, DO_K, DO_V, OCC>;
  int rc = at_allow_lds<kernel>(L::BYTES);
  if (rc) return rc;
  const int64_t row_tiles = (c.a->Tq + RT - 1) / RT, all = row_tiles * c.d.G;
  at_parts sp = {};
  sp.per = (int)((all + c.p.k_splits - 1) / c.p.k_splits);
  if (sp.per < 1) sp.per = 1;
  sp.n = c.p.k_splits;
  sp.p = c.parts;
  sp.part = c.a->N * c.a->Tk * c.a->Hk * c.a->D;
  const at_order order(c.a->N, c.a->Hk, c.p.k_tiles * sp.n);
  kernel<<<order.grid(), 256 * HALVES, L::BYTES, c.st>>>((const T*)c.q, (const T*)c.k, (const T*)c.v, c.lse, (const T*)c.dout, c.delta,
                                                  (T*)c.dk, (T*)c.dv, sp, c.d, order,
                                               at_div((uint32_t)c.p.k_tiles), at_div((uint32_t)sp.n), at_div((uint32_t)row_tiles));
  return rc_check_launch("rc_cross_attn_bwd (keys)");
}

template <typename T> int at_add(const at_bwd_call& c, int64_t offset, int64_t stride, int n, void* out, int64_t elems) {
  at_add_kernel<T><<<(uint32_t)((elems / 4 + 255) / 256), 256, 0, c.st>>>(c.parts + offset, stride, n, (T*)out, elems / 4);
  return rc_check_launch("rc_cross_attn_bwd (parts)");
}

template <typename T, int DC> int at_bwd(const at_bwd_call& c) {
  // tiles and resident workgroups: what registers (512 per lane and SIMD) and 160 KiB of LDS allow
  constexpr int RB = at_row<T, DC>::RB;
  constexpr int NB = RB >= 512 ? 1 : 2;
  constexpr int OCC = RB >= 512 ? 1 : 2;
  constexpr int HALVES = sizeof(T) == 2 && DC > 64 && DC <= 128 ? 2 : 1;
  constexpr int KOCC = HALVES == 2 || DC * sizeof(T) <= 128 ? 2 : 1;
  int rc = RC_OK;
  if (c.p.q_items) {  // (the gradients of keys and values need delta)
    constexpr int bytes = at_dq_lds<T, DC, 32 * NB, 4>::BYTES;
    static_assert(bytes <= 160 * 1024, "LDS");
    constexpr auto kernel = at_dq_kernel<T, DC, 4, NB, OCC>;
    if ((rc = at_allow_lds<kernel>(bytes))) return rc;
    at_parts sp = {};
    sp.n = c.dq ? c.p.q_splits : 1;
    sp.per = c.p.q_per;
    sp.p = c.parts;
    sp.part = c.a->N * c.a->Tq * c.a->Hq * c.a->D;
    const at_order order(c.a->N, c.a->Hk, c.p.q_tiles * sp.n);
    kernel<<<order.grid(), 256, bytes, c.st>>>((const T*)c.q, (const T*)c.k, (const T*)c.v, (const T*)c.out,
                                                 (const T*)c.rest, c.lse,
                                                 (const T*)c.dout, c.delta, (T*)c.dq, sp, c.d, order,
                                                 at_div((uint32_t)c.p.q_tiles), at_div((uint32_t)sp.n));
    if ((rc = rc_check_launch("rc_cross_attn_bwd (queries)"))) return rc;
    if (c.dq && sp.n > 1 && (rc = at_add<T>(c, 0, sp.part, sp.n, c.dq, sp.part))) return rc;
  }
  if (!c.dk || !c.p.k_items) return RC_OK;
  // wide heads in fp32, and in fp16 with its scaling: registers for one of the two at a time
  if constexpr (RB >= 1024 || (at_fit<T>::ON && DC > 128)) {
    if ((rc = at_launch_dkv<T, DC, 1, 1, true, false, 1>(c))) return rc;
    if ((rc = at_launch_dkv<T, DC, 1, 1, false, true, 1>(c))) return rc;
  } else {
    if ((rc = at_launch_dkv<T, DC, HALVES, NB, true, true, KOCC>(c))) return rc;
  }
  if (c.p.k_splits > 1) {
    const int64_t part = c.a->N * c.a->Tk * c.a->Hk * c.a->D;
    if ((rc = at_add<T>(c, 0, 2 * part, c.p.k_splits, c.dk, part))) return rc;
    if ((rc = at_add<T>(c, part, 2 * part, c.p.k_splits, c.dv, part))) return rc;
  }
  return RC_OK;
}

template <typename T> int at_bwd_d(const at_bwd_call& c) {
  const int D = c.a->D;
  if (D <= 32) return at_bwd<T, 32>(c);
  if (D <= 64) return at_bwd<T, 64>(c);
  if (D <= 96) return at_bwd<T, 96>(c);
  if (D <= 128) return at_bwd<T, 128>(c);
  if (D <= 192) return at_bwd<T, 192>(c);
  return at_bwd<T, 256>(c);
}

}  // namespace

extern "C" int64_t rc_cross_attn_bwd_work_bytes(const rc_attn* a) {
  const int rc = at_check(a);
  if (rc) return rc < 0 ? rc : RC_EINVAL;
  const at_bwd_plan p = at_make_bwd_plan(a);
  return p.bits + p.delta + p.parts;
}

extern "C" int rc_cross_attn_bwd(const rc_attn* a, const void* q, const void* k, const void* v, const void* out,
                                 const void* rest, const float* lse, const void* dout, void* dq, void* dk, void* dv, void* work,
                                 void* stream) {
  int rc = at_check(a);
  if (rc) return rc;
  for (const void* p : {q, out, (const void*)lse, dout, (const void*)work})
    if ((rc = at_check_operand(a, a->N * a->Tq, p))) return rc;
  for (const void* p : {k, v})
    if ((rc = at_check_operand(a, a->N * a->Tk, p))) return rc;
  RC_REQUIRE((dk == nullptr) == (dv == nullptr), RC_EINVAL, "rc_cross_attn_bwd: dk and dv are wanted together or not at all");
  RC_REQUIRE(((uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)rest) % 16 == 0, RC_EINVAL,
             "rc_cross_attn_bwd: a gradient is not aligned to 16 bytes");
  if (a->N == 0) return RC_OK;
  at_bwd_call c = {};
  c.a = a;
  c.p = at_make_bwd_plan(a);
  RC_REQUIRE(c.p.bits == 0 || (work != nullptr && (uintptr_t)work % 16 == 0), RC_EINVAL,
             "rc_cross_attn_bwd: work is null or not aligned to 16 bytes");
  RC_REQUIRE(c.p.q_items * c.p.q_splits < (1ll << 31) - 8 && c.p.k_items * c.p.k_splits < (1ll << 31) - 8 &&
                 a->N * a->Tq * a->Hq * a->D / 4 < (1ll << 39) && a->N * a->Tk * a->Hk * a->D / 4 < (1ll << 39),
             RC_EINVAL, "rc_cross_attn_bwd: too many rows");
  c.q = q;
  c.k = k;
  c.v = v;
  c.out = out;
  c.rest = rest;
  c.dout = dout;
  c.lse = lse;
  c.dq = dq;
  c.dk = dk;
  c.dv = dv;
  c.delta = reinterpret_cast<float*>(reinterpret_cast<char*>(work) + c.p.bits);
  c.parts = reinterpret_cast<float*>(reinterpret_cast<char*>(work) + c.p.bits + c.p.delta);
  c.st = (hipStream_t)stream;
  c.d = at_to_dev(a, work);
  if ((rc = at_launch_bits(a, work, c.st))) return rc;
  if (dq && dk && a->N * a->Tq && a->N * a->Tk && at_rows_fit(a))
    return at_rows_bwd(a, c.d, q, k, v, out, rest, lse, dout, dq, dk, dv, c.st);
  if (a->dtype == RC_F32) return at_bwd_d<float>(c);
  if (a->dtype == RC_F16) return at_bwd_d<rc_half>(c);
  return at_bwd_d<rc_bf16>(c);
}
