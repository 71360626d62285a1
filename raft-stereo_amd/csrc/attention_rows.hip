// Attention backward in one kernel, for sequences whose keys fit a workgroup (the rows of an image).
//
//   P = exp2(S c - lse2),  delta = sum_d dO O,  dS = P (dO V^T - delta),  dV = P^T dO,  dQ = scale dS K,  dK = scale dS^T Q
//
// A workgroup has all keys of one key head, a wave 32 of them: K as a tile in LDS, V and the sums of dK and dV in
// registers.  The query rows of the group's heads come in batches of as many rows, all of a batch in one go (one memory
// latency; fetched tile by tile, each tile would wait for the loads and for the stores of the one before).  Of each 32
// query rows every wave multiplies its share of S and dP and adds to its dK and dV; its share of dS goes to LDS, where
// after a barrier the waves take blocks of 16 x 16 of dQ = dS K, each over all keys.  Everything is read once and written
// once, and S and dP are worked out once (the two kernels for long sequences read the operands twice and multiply 7
// products instead of 5).
//
// 640 x 180 x 180, 8 heads of 32, bf16: 177 us (median of 300 launches), 2.3 TB/s of operands and gradients (in a call 227
// instead of 267 with the two kernels, when it was measured); the matrix pipe is busy 14 % of the time, the vector pipe and
// LDS 39 %, nearly half of LDS in bank conflicts of the 64-byte rows: the waves of a workgroup wait for each other at each 32
// query rows, and two or three workgroups on a CU fill each other's gaps.  96 x 128 x 117, 4 heads of 64, fp32: 81 us, matrix
// pipe 29 %: 384 workgroups of 135 KB of LDS, one to a CU, are one turn and half of another.
#include "attention.h"

namespace {

template <typename T, int DC, int NW> struct at_rows_lds {
  using R = at_row<T, DC>;
  using RS = at_row<T, 32>;
  static constexpr int KEYS = R::tile(32 * NW), DS = RS::tile(32 * NW), STAT = 256;
  static constexpr int Q = KEYS, G = 2 * KEYS;         // a batch of query rows and of dO: 32 NW
  static constexpr int DSS = 3 * KEYS;                 // [2]: dS of 32 query rows, a key per row
  static constexpr int LSE = DSS + 2 * DS;             // [NW] 64 floats each, as one load moves them
  static constexpr int DELTA = LSE + NW * STAT;        // [NW][32]
  static constexpr int FACTOR = DELTA + NW * STAT / 2; // [NW][32]; fp16: what a row of dS is scaled by
  static constexpr int NORM = FACTOR + NW * STAT / 2;  // fp16: each wave's largest |V|^2
  // fp16 heads of 32: V too, its scaling takes V's registers
  static constexpr bool V_LDS = at_fit<T>::ON && DC == 32;
  static constexpr int V = (NORM + 64 + 1023) / 1024 * 1024;
  static constexpr int BYTES = V_LDS ? V + KEYS : NORM + 64;
};

// A lane's place of an operand of a 16 x 16 product across a tile's rows: 32 rows a step (16-bit types: rows 8 g + 0..3
// and + 4..7 of column i, g = lane / 16), columns 16 ct ..; fp32: 8 rows a step, row g and 4 + g.
template <typename T, int DC> struct at_cols16 {
  using R = at_row<T, DC>;
  uint32_t lo, hi;
  __device__ __forceinline__ void init(int ct, int lane) {
    const int i = lane & 15, g = lane >> 4;
    if constexpr (sizeof(T) == 2) {
      const int chunk = 2 * ct + ((i >> 1) & 1);
      lo = at_chunk<T, DC>(8 * g + (i >> 2), chunk) + (i & 1) * 8;
      hi = at_chunk<T, DC>(8 * g + 4 + (i >> 2), chunk) + (i & 1) * 8;
    } else {
      lo = at_chunk<T, DC>(g, 4 * ct + (i >> 2)) + (i & 3) * 4;
      hi = at_chunk<T, DC>(4 + g, 4 * ct + (i >> 2)) + (i & 3) * 4;
    }
  }
  __device__ __forceinline__ at_u4 read(const unsigned char* tile, int step) const {
    typedef at_s4 __attribute__((address_space(3))) * lds_s4p;
    const at_s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4p)(tile + lo + step * R::at(32)));
    const at_s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4p)(tile + hi + step * R::at(32)));
    return __builtin_bit_cast(at_u4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  __device__ __forceinline__ at_f2 read_f32(const unsigned char* tile, int step) const {
    return at_f2{*reinterpret_cast<const float*>(tile + lo + step * R::at(8)), *reinterpret_cast<const float*>(tile + hi + step * R::at(8))};
  }
};

__device__ __forceinline__ at_f4 at_mma16(rc_half, at_u4 a, at_u4 b, at_f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(at_h8, a), __builtin_bit_cast(at_h8, b), c, 0, 0, 0);
}
__device__ __forceinline__ at_f4 at_mma16(rc_bf16, at_u4 a, at_u4 b, at_f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(at_b8, a), __builtin_bit_cast(at_b8, b), c, 0, 0, 0);
}

template <typename T, int DC, int NW, int OCC>
__global__ __launch_bounds__(64 * NW, OCC) void at_rows_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                               const T* __restrict__ v, const T* __restrict__ out,
                                                               const T* __restrict__ rest_out, const float* __restrict__ lse, const T* __restrict__ dout,
                                                               T* __restrict__ dq, T* __restrict__ dk, T* __restrict__ dv,
                                                               at_args a, at_order order, at_div by_batches) {
  using R = at_row<T, DC>;
  using L = at_rows_lds<T, DC, NW>;
  constexpr int NDB = DC / 32, LOADS = 32 * R::RB / 1024;
  constexpr bool FIT = at_fit<T>::ON;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int nh = order.item();
  if (nh < 0) return;
  const int n = a.by_Hk.of(nh), hk = nh - n * a.Hk;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 31, h = lane >> 5;
  const int key0 = wave * 32, key = key0 + c;
  const uint32_t mine = at_key_bits(a, n, at_length(a, n), key0);
  const bool live = key < a.Tk, takes = (mine >> c) & 1;
  uint32_t some = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) some |= at_key_bits(a, n, at_length(a, n), 32 * w);
  const int batches = (int)by_batches.d;  // of one head's query rows
  const uint32_t lds0 = (uint32_t)(uintptr_t)(at_lds)smem;

  // this wave's keys to LDS
#pragma unroll
  for (int i = 0; i < LOADS; ++i)
    at_fetch_rows<T, DC>(k + (int64_t)n * a.ks[0] + (int64_t)key0 * a.ks[1] + (int64_t)hk * a.ks[2], (uint32_t)(a.ks[1] * sizeof(T)), a.D,
                         mine, lds0 + R::at(32) * wave, i, lane);
  at_u4 vf[R::STEPS];
  const T* vp = v + (int64_t)n * a.vs[0] + (int64_t)key0 * a.vs[1] + (int64_t)hk * a.vs[2];
  const uint32_t vst = (uint32_t)(a.vs[1] * sizeof(T));
  at_rows_of(vp).row<T, DC>(takes ? (uint32_t)c * vst : AT_OUTSIDE, a.D, lane, vf);
  if constexpr (L::V_LDS) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) at_fetch_rows<T, DC>(vp, vst, a.D, mine, lds0 + L::V + R::at(32) * wave, i, lane);
  }
  const unsigned char *ks = smem + R::at(32) * wave, *vs = smem + L::V + R::at(32) * wave;
  at_places<T, DC> at;
  at.init(lane);
  at_f16 acck[NDB], accv[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i) acck[i] = accv[i] = (at_f16)(0.0f);
  at_fit<T> fit;
  float* lses = reinterpret_cast<float*>(smem + L::LSE);
  float* deltas = reinterpret_cast<float*>(smem + L::DELTA);
  float* factors = reinterpret_cast<float*>(smem + L::FACTOR);
  float fv = 1.0f;  // fp16: 1 / a power of two beyond every |V|
  if constexpr (FIT) {
    float n2 = 0.0f;
#pragma unroll
    for (int s = 0; s < R::STEPS; ++s) n2 += at_dot(T(), vf[s], vf[s]);
    n2 = at_half_sum(n2);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) n2 = fmaxf(n2, __shfl_xor(n2, x));
    if (lane == 0) reinterpret_cast<float*>(smem + L::NORM)[wave] = n2;
  }

  for (int b = 0; b < a.G * batches; ++b) {
    const int g = by_batches.of(b), hq = hk * a.G + g, t0 = (b - g * batches) * 32 * NW;
    const int tiles = min(NW, (a.Tq - t0 + 31) >> 5);
    if (b > 0) at_sync();  // nobody reads the last batch any more
    // 32 rows a wave: Q, dO and lse2 to LDS (behind the last row: its Q and lse2 again); delta, as soon as the wave's own
    // loads have landed
    if (wave < tiles) {
      const int t = t0 + 32 * wave, left = a.Tq - t;
      const uint32_t take = at_first_bits(left);
      const int64_t o = (((int64_t)n * a.Tq + t) * a.Hq + hq) * a.D;
      const uint32_t ost = (uint32_t)(a.Hq * a.D * (int)sizeof(T));
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        at_fetch_rows<T, DC>(q + (int64_t)n * a.qs[0] + (int64_t)t * a.qs[1] + (int64_t)hq * a.qs[2], (uint32_t)(a.qs[1] * sizeof(T)), a.D,
                             0xffffffffu, lds0 + L::Q + R::at(32) * wave, i, lane, left - 1);
        at_fetch_rows<T, DC>(dout + o, ost, a.D, take, lds0 + L::G + R::at(32) * wave, i, lane);
      }
      at_fetch_floats<true>(lse + ((int64_t)n * a.Hq + hq) * a.Tq + t, left, lds0 + L::LSE + L::STAT * wave, lane);
      at_u4 of[R::STEPS];
      at_rows_of(out + o).row<T, DC>(c < left ? (uint32_t)c * ost : AT_OUTSIDE, a.D, lane, of);
      constexpr int RESTS = sizeof(T) == 2 ? R::STEPS : 1;
      at_u4 rf[RESTS];
      const bool both = sizeof(T) == 2 && rest_out != nullptr;
      if (both) at_rows_of(rest_out + o).row<T, sizeof(T) == 2 ? DC : 8>(c < left ? (uint32_t)c * ost : AT_OUTSIDE, a.D, lane, rf);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      float s = 0.0f, n2 = 0.0f;
#pragma unroll
      for (int st = 0; st < R::STEPS; ++st) {
        const at_u4 x = at.rows(smem + L::G + R::at(32) * wave, 0, st);
        s += at_dot(T(), x, of[st]);
        if (both) s += at_dot(T(), x, rf[sizeof(T) == 2 ? st : 0]);
        if constexpr (FIT) n2 += at_dot(T(), x, x);
      }
      s = at_half_sum(s);
      if (h == 0) deltas[32 * wave + c] = s;
      if constexpr (FIT) {
        // a power of two beyond |dO|: with the one beyond |V|, |P (dP - delta)| <= 2 |dO| max |V| stays in fp16's range
        n2 = at_half_sum(n2);
        const int e = n2 > 0.0f ? (__builtin_amdgcn_frexp_expf(n2) + 1) >> 1 : 0;
        if (h == 0) factors[32 * wave + c] = ldexpf(1.0f, -e);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    at_landed();
    if (FIT && b == 0) {
      float n2 = 0.0f;
      for (int w = 0; w < NW; ++w) n2 = fmaxf(n2, reinterpret_cast<const float*>(smem + L::NORM)[w]);
      if (n2 > 0.0f) fv = ldexpf(1.0f, -((__builtin_amdgcn_frexp_expf(n2) + 1) >> 1));
    }

    for (int j = 0; j < tiles; ++j) {
      const unsigned char* qs = smem + L::Q + R::at(32) * j;
      const unsigned char* gs = smem + L::G + R::at(32) * j;
      const float *ls = lses + 64 * j, *dl = deltas + 32 * j, *fr = factors + 32 * j;
      // (a key that takes no part has the score -inf, so P = 0, and zeros for its value, so dP = 0)
      at_f16 s = at_start<T, true>(mine, lane);
#pragma unroll
      for (int st = 0; st < R::STEPS; ++st) s = at_mma(T(), at.rows(qs, 0, st), at.rows(ks, 0, st), s);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const at_f4 l4 = *reinterpret_cast<const at_f4*>(ls + 8 * x + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * x + i] = __builtin_amdgcn_exp2f(s[4 * x + i] * a.scale_log2 - (l4[i] - AT_P_LIFT<T>));
      }
      at_mma_cols<T, DC>(at, gs, 0, s, accv);
      at_f16 dp = (at_f16)(0.0f);
#pragma unroll
      for (int st = 0; st < R::STEPS; ++st) dp = at_mma(T(), at.rows(gs, 0, st), L::V_LDS ? at.rows(vs, 0, st) : vf[st], dp);
      unsigned char* dss = smem + L::DSS + (j & 1) * L::DS;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const at_f4 d4 = *reinterpret_cast<const at_f4*>(dl + 8 * x + 4 * h);
        at_f4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = s[4 * x + i] *= dp[4 * x + i] - d4[i];
        if constexpr (FIT) w *= *reinterpret_cast<const at_f4*>(fr + 8 * x + 4 * h) * fv;
        if constexpr (sizeof(T) == 2)
          *reinterpret_cast<at_u2*>(dss + at_chunk<T, 32>(key, x) + 8 * h) = at_u2{at_pack(T(), w[0], w[1]), at_pack(T(), w[2], w[3])};
        else
          *reinterpret_cast<at_f4*>(dss + at_chunk<T, 32>(key, 2 * x + h)) = w;
      }
      fit.template fit<NDB>(s, acck);
      at_mma_cols<T, DC>(at, qs, 0, s, acck);
      at_sync();
      // dQ of these rows: blocks of 16 elements by 16 rows.  (Their places are worked out here each time: there are no
      // registers to keep them in.)
      int ln = lane;
      asm volatile("" : "+v"(ln));
      for (int x = wave; x < 4 * NDB; x += NW) {
        if (16 * (x >> 1) >= a.D) break;
        at_cols16<T, DC> ka;
        at_cols16<T, 32> sb;
        ka.init(x >> 1, ln);
        sb.init(x & 1, ln);
        at_f4 acc = (at_f4)(0.0f);
        if constexpr (sizeof(T) == 2) {
#pragma unroll 2
          for (int i = 0; i < NW; ++i) acc = at_mma16(T(), ka.read(smem, i), sb.read(dss, i), acc);
        } else {
#pragma unroll 4
          for (int i = 0; i < 4 * NW; ++i) {
            const at_f2 u = ka.read_f32(smem, i), w = sb.read_f32(dss, i);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(u[0], w[0], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(u[1], w[1], acc, 0, 0, 0);
          }
        }
        if (!some) acc = (at_f4)(0.0f);  // (no key at all: not even what 0 times NaN leaves)
        const int r = 16 * (x & 1) + (ln & 15), d = 16 * (x >> 1) + 4 * (ln >> 4), t = t0 + 32 * j + r;
        float f = a.scale;
        if constexpr (FIT) f = f / (fr[r] * fv) * (1.0f / 4096.0f);
        T* o = dq + (((int64_t)n * a.Tq + t) * a.Hq + hq) * a.D + d;
        if (t < a.Tq && d < a.D) {
          if constexpr (sizeof(T) == 2) *reinterpret_cast<at_u2*>(o) = at_u2{at_pack(T(), acc[0] * f, acc[1] * f), at_pack(T(), acc[2] * f, acc[3] * f)};
          else *reinterpret_cast<at_f4*>(o) = acc * f;
        }
      }
    }
  }

  const float unlift = FIT ? 1.0f / 4096.0f : 1.0f;
  const bool keep = (mine >> c) & 1;
  const int64_t o = (((int64_t)n * a.Tk + key) * a.Hk + hk) * a.D;
  at_store_rows<T, DC>(dk + o, live, keep, acck, a.scale * fit.undo() * unlift, a.D, lane);
  at_store_rows<T, DC>(dv + o, live, keep, accv, unlift, a.D, lane);
}

template <typename T, int DC, int NW, int OCC>
int at_launch_rows(const rc_attn* a, const at_args& d, const void* q, const void* k, const void* v, const void* out,
                   const void* rest, const float* lse, const void* dout, void* dq, void* dk, void* dv, hipStream_t st) {
  using L = at_rows_lds<T, DC, NW>;
  static_assert(L::BYTES <= 160 * 1024, "LDS");
  constexpr auto kernel = at_rows_kernel<T, DC, NW, OCC>;
  const int rc = at_allow_lds<kernel>(L::BYTES);
  if (rc) return rc;
  const at_order order(a->N, a->Hk, 1);
  kernel<<<order.grid(), 64 * NW, L::BYTES, st>>>((const T*)q, (const T*)k, (const T*)v, (const T*)out, (const T*)rest, lse, (const T*)dout, (T*)dq,
                                                  (T*)dk, (T*)dv, d, order, at_div((uint32_t)((a->Tq + 32 * NW - 1) / (32 * NW))));
  return rc_check_launch("rc_cross_attn_bwd (rows)");
}

// waves (32 keys each) of a workgroup, 0: too many keys
int at_rows_waves(const rc_attn* a) {
  const int need = (int)((a->Tk + 31) / 32);
  const bool f32 = a->dtype == RC_F32;
  const int most = a->D <= 32 ? (f32 ? 6 : 12) : a->D <= 64 ? (f32 ? 4 : 8) : 0;  // registers, and 160 KiB of LDS
  if (need > most) return 0;
  return need <= 4 ? 4 : need <= 6 ? 6 : need <= 8 ? 8 : 12;
}

template <typename T, int DC, typename... Args> int at_rows_nw(int waves, Args... args) {
  // Waves per SIMD.  16-bit heads of 32: four, 128 registers.  (Six waves spread over the SIMDs as 2, 2, 1, 1: with room
  // for three on each, a second workgroup often found no place, and 640 sequences of 180 took 215 instead of 155 us.)
  constexpr int OCC = sizeof(T) == 2 && DC == 32 ? 4 : sizeof(T) == 4 && DC > 32 ? 1 : 2;
  if constexpr (sizeof(T) == 2 || DC == 32)
    if (waves == 6) return at_launch_rows<T, DC, 6, OCC>(args...);
  if constexpr (sizeof(T) == 2)
    if (waves == 8) return at_launch_rows<T, DC, 8, 2>(args...);  // (one workgroup per CU: LDS)
  if constexpr (sizeof(T) == 2 && DC == 32)
    if (waves == 12) return at_launch_rows<T, DC, 12, 3>(args...);
  return at_launch_rows<T, DC, 4, OCC>(args...);
}

}  // namespace

bool at_rows_fit(const rc_attn* a) { return at_rows_waves(a) > 0 && a->N * a->Hk >= 256; }

int at_rows_bwd(const rc_attn* a, const at_args& d, const void* q, const void* k, const void* v, const void* out, const void* rest,
                const float* lse, const void* dout, void* dq, void* dk, void* dv, hipStream_t st) {
  const int w = at_rows_waves(a);
  if (a->dtype == RC_F32)
    return a->D <= 32 ? at_rows_nw<float, 32>(w, a, d, q, k, v, out, rest, lse, dout, dq, dk, dv, st)
                      : at_rows_nw<float, 64>(w, a, d, q, k, v, out, rest, lse, dout, dq, dk, dv, st);
  if (a->dtype == RC_F16)
    return a->D <= 32 ? at_rows_nw<rc_half, 32>(w, a, d, q, k, v, out, rest, lse, dout, dq, dk, dv, st)
                      : at_rows_nw<rc_half, 64>(w, a, d, q, k, v, out, rest, lse, dout, dq, dk, dv, st);
  return a->D <= 32 ? at_rows_nw<rc_bf16, 32>(w, a, d, q, k, v, out, rest, lse, dout, dq, dk, dv, st)
                    : at_rows_nw<rc_bf16, 64>(w, a, d, q, k, v, out, rest, lse, dout, dq, dk, dv, st);
}
