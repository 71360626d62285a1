// RMS norm of query and key heads and their rotation by position, in one pass, and its adjoint.
//
//   r = 1 / sqrt(mean_d x_d^2 + eps),  y_d = x_d r w_d,  (y_a, y_b) -> (y_a cos A - y_b sin A, y_b cos A + y_a sin A)
//   with A = pos * freqs[i] for pair i.  With u = the rotation's transpose applied to the incoming gradient g:
//   dw_d = sum u_d x_d r,   dx = r (w u) - x r^3 mean_d(w u x)
//
// Streaming kernels: every head is read once and written once (backward: x and g read, dx written), so they are bound
// by memory bandwidth as long as the angles stay cheap.  A group of G lanes (G the power of two from D / 8 on) holds
// one head, 8 elements per lane; the sum of squares is a butterfly over the group.  A lane owns BOTH elements of each
// of its four pairs -- elements 4 j .. 4 j + 3 and the ones n_freqs further on (or 8 j .. 8 j + 7 when neighbours are
// paired) -- so the rotation needs no exchange between lanes, and its four angles are worked out once and serve all
// heads of the token that the group goes through.  Lanes of 8 elements rather than 16 bytes each: one form for all
// types, and 8-byte loads of neighbouring lanes fill their cache lines together.
//
// Measured (kernels, medians of 300 launches; a large copy reaches 4.8 TB/s; what the 256 MiB cache still holds comes
// faster): forward, 768 x 312 fp16 queries and keys, 4 heads of 64 each: 110 us, 4.5 TB/s.  640 x 180 fp32, 8 and 8 heads of
// 32: forward 88 us, 5.3 TB/s, backward 141 us, 5.0 TB/s.  8 x 2047 and 4095 bf16, 16 and 4 heads of 128: 47 us, 4.3 TB/s,
// and 67 us, 4.5 TB/s, and 6 us for the sum of the weights' gradients.  One token in 16 sequences, 32 heads of 128: 5.4 us,
// in 12.8 of the call.
#include "rc_common.h"

#include <math.h>

namespace {

constexpr int NR_THREADS = 256;
constexpr int NR_MAX_BLOCKS = 1024;  // of one side's backward pass: rows of partial weight gradients
constexpr uint32_t NR_GRID_X = 1u << 22;  // a launch holds fewer than 2^32 threads along x
constexpr int NR_UNROLL = 4;         // heads whose loads are in flight together

struct nr_side {
  const void* x;
  const void* g;  // backward only
  void* y;        // y, or dx
  const void* w;
  const void* pos;
  int64_t stride[3];
  int64_t pos_stride;
  uint32_t T, tokens;
  int32_t H, w_dtype, pos_dtype;
  int32_t heads_per_group, chunks;
  uint32_t groups;  // tokens * chunks
  uint32_t blocks;
};

struct nr_common {
  const void* freqs;
  int32_t freqs_f64, n_freqs, D;
  float eps;
};

template <typename T> struct nr_quad {
  typedef T type __attribute__((ext_vector_type(4)));
};

template <typename T> __device__ __forceinline__ void nr_load4(const T* p, float* o) {
  const auto v = *reinterpret_cast<const typename nr_quad<T>::type*>(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = rc_to_float(v[j]);
}
template <typename T> __device__ __forceinline__ void nr_store4(T* p, const float* v) {
  typename nr_quad<T>::type o;
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = rc_from_float<T>(v[j]);
  *reinterpret_cast<typename nr_quad<T>::type*>(p) = o;
}

__device__ __forceinline__ float nr_weight(const void* w, int dtype, int d) {
  if (w == nullptr) return 1.0f;
  if (dtype == RC_F32) return reinterpret_cast<const float*>(w)[d];
  if (dtype == RC_F16) return (float)reinterpret_cast<const rc_half*>(w)[d];
  return (float)reinterpret_cast<const rc_bf16*>(w)[d];
}

__device__ __forceinline__ double nr_pos(const nr_side& s, int64_t n, uint32_t t) {
  if (s.pos == nullptr) return (double)t;
  const int64_t i = n * s.pos_stride + t;
  if (s.pos_dtype == RC_POS_I32) return (double)reinterpret_cast<const int32_t*>(s.pos)[i];
  if (s.pos_dtype == RC_POS_I64) return (double)reinterpret_cast<const int64_t*>(s.pos)[i];
  return (double)reinterpret_cast<const float*>(s.pos)[i];
}

template <int G> __device__ __forceinline__ float nr_sum(float v) {
#pragma unroll
  for (int m = G / 2; m > 0; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

// What a lane holds of every head: two runs of four elements, and the four pairs' turns per position.
template <bool IL> struct nr_lane {
  int a, b;         // first element of each run
  bool on, turned;  // the lane has elements; they are rotated
  float wa[4], wb[4];
  double turn[4];

  __device__ __forceinline__ void init(const nr_common& c, const nr_side& s, int j) {
    const int n = c.n_freqs;
    on = j < c.D / 8;
    turned = on && j < n / 4;
    a = IL || !turned ? 8 * j : 4 * j;  // (2 n + 8 (j - n / 4) = 8 j behind the rotated elements)
    b = IL || !turned ? a + 4 : a + n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      wa[i] = on ? nr_weight(s.w, s.w_dtype, a + i) : 0.0f;
      wb[i] = on ? nr_weight(s.w, s.w_dtype, b + i) : 0.0f;
      turn[i] = 0.0;
      if (turned)
        turn[i] = (c.freqs_f64 ? reinterpret_cast<const double*>(c.freqs)[4 * j + i]
                               : (double)reinterpret_cast<const float*>(c.freqs)[4 * j + i]) *
                  0.15915494309189533577;  // 1 / (2 pi)
    }
  }
  // cos and sin of the four angles: the angle in turns, reduced to [-1/2, 1/2] in double
  __device__ __forceinline__ void angles(double pos, float* co, float* si) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double p = pos * turn[i];
      sincospif(2.0f * (float)(p - rint(p)), &si[i], &co[i]);
    }
  }
};

// (a, b) <- rotated by (co, si); INV: by the opposite angle
template <bool IL, bool INV>
__device__ __forceinline__ void nr_rotate(float* a, float* b, const float* co, const float* si) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float& p = IL ? (i < 2 ? a[2 * i] : b[2 * i - 4]) : a[i];
    float& q = IL ? (i < 2 ? a[2 * i + 1] : b[2 * i - 3]) : b[i];
    const float s = INV ? -si[i] : si[i];
    const float x = p * co[i] - q * s, y = q * co[i] + p * s;
    p = x;
    q = y;
  }
}

template <typename T, int G, bool IL>
__device__ __forceinline__ void nr_fwd_body(const nr_side& s, const nr_common& c, uint32_t block) {
  const int j = threadIdx.x % G;
  const uint32_t gi = block * (NR_THREADS / G) + threadIdx.x / G;
  const bool live = gi < s.groups;
  const uint32_t gc = live ? gi : s.groups - 1;  // idle groups repeat the last one's work and store nothing
  const uint32_t token = gc / (uint32_t)s.chunks;
  const int h0 = (int)(gc - token * (uint32_t)s.chunks) * s.heads_per_group;
  const uint32_t n = token / s.T, t = token - n * s.T;
  nr_lane<IL> lane;
  lane.init(c, s, j);
  float co[4], si[4];
  lane.angles(nr_pos(s, n, t), co, si);
  const T* x = reinterpret_cast<const T*>(s.x) + (int64_t)n * s.stride[0] + (int64_t)t * s.stride[1];
  T* y = reinterpret_cast<T*>(s.y) + (int64_t)token * s.H * c.D;
  const float inv_d = 1.0f / (float)c.D;
  for (int hb = 0; hb < s.heads_per_group; hb += NR_UNROLL) {
    float xa[NR_UNROLL][4], xb[NR_UNROLL][4];
#pragma unroll
    for (int u = 0; u < NR_UNROLL; ++u) {
      const int h = h0 + hb + u;
      const bool ok = lane.on && hb + u < s.heads_per_group && h < s.H;
#pragma unroll
      for (int i = 0; i < 4; ++i) xa[u][i] = xb[u][i] = 0.0f;
      if (ok) {
        nr_load4(x + (int64_t)h * s.stride[2] + lane.a, xa[u]);
        nr_load4(x + (int64_t)h * s.stride[2] + lane.b, xb[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < NR_UNROLL; ++u) {
      const int h = h0 + hb + u;
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss += xa[u][i] * xa[u][i] + xb[u][i] * xb[u][i];
      ss = nr_sum<G>(ss);
      const float r = rsqrtf(ss * inv_d + c.eps);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        xa[u][i] = xa[u][i] * r * lane.wa[i];
        xb[u][i] = xb[u][i] * r * lane.wb[i];
      }
      if (lane.turned) nr_rotate<IL, false>(xa[u], xb[u], co, si);
      if (live && lane.on && hb + u < s.heads_per_group && h < s.H) {
        nr_store4(y + (int64_t)h * c.D + lane.a, xa[u]);
        nr_store4(y + (int64_t)h * c.D + lane.b, xb[u]);
      }
    }
  }
}

template <typename T, int G, bool IL>
__global__ __launch_bounds__(NR_THREADS) void nr_fwd_kernel(nr_side q, nr_side k, nr_common c) {
  const uint32_t block = blockIdx.y * NR_GRID_X + blockIdx.x;
  if (block < q.blocks) nr_fwd_body<T, G, IL>(q, c, block);
  else if (block - q.blocks < k.blocks) nr_fwd_body<T, G, IL>(k, c, block - q.blocks);
}

// A group goes through many tokens, so that its lanes' weight gradients are summed in registers; the groups of a block
// are then added in LDS, and the block's row goes to `partial`.  Bound by memory; two heads' loads in flight are what the
// registers of four waves per SIMD hold.
template <typename T, int G, bool IL>
__device__ __forceinline__ void nr_bwd_body(const nr_side& s, const nr_common& c, uint32_t block, float* partial,
                                            float* lds) {
  constexpr int GROUPS = NR_THREADS / G;
  const int j = threadIdx.x % G, grp = threadIdx.x / G;
  nr_lane<IL> lane;
  lane.init(c, s, j);
  const float inv_d = 1.0f / (float)c.D;
  float dwa[4] = {0, 0, 0, 0}, dwb[4] = {0, 0, 0, 0};
  for (uint32_t base = block * GROUPS; base < s.groups; base += s.blocks * GROUPS) {
    const bool live = base + grp < s.groups;
    const uint32_t gc = live ? base + grp : s.groups - 1;
    const uint32_t token = gc / (uint32_t)s.chunks;
    const int h0 = (int)(gc - token * (uint32_t)s.chunks) * s.heads_per_group;
    const uint32_t n = token / s.T, t = token - n * s.T;
    float co[4], si[4];
    lane.angles(nr_pos(s, n, t), co, si);
    const T* x = reinterpret_cast<const T*>(s.x) + (int64_t)n * s.stride[0] + (int64_t)t * s.stride[1];
    const int64_t row = (int64_t)token * s.H * c.D;
    const T* g = reinterpret_cast<const T*>(s.g) + row;
    T* dx = reinterpret_cast<T*>(s.y) + row;
    for (int hb = 0; hb < s.heads_per_group; hb += 2) {
      float xa[2][4], xb[2][4], ga[2][4], gb[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int h = h0 + hb + u;
        const bool ok = live && lane.on && hb + u < s.heads_per_group && h < s.H;
#pragma unroll
        for (int i = 0; i < 4; ++i) xa[u][i] = xb[u][i] = ga[u][i] = gb[u][i] = 0.0f;
        if (ok) {
          nr_load4(x + (int64_t)h * s.stride[2] + lane.a, xa[u]);
          nr_load4(x + (int64_t)h * s.stride[2] + lane.b, xb[u]);
          nr_load4(g + (int64_t)h * c.D + lane.a, ga[u]);
          nr_load4(g + (int64_t)h * c.D + lane.b, gb[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int h = h0 + hb + u;
        const bool ok = live && lane.on && hb + u < s.heads_per_group && h < s.H;
        if (lane.turned) nr_rotate<IL, true>(ga[u], gb[u], co, si);
        float ss = 0.0f, dot = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ss += xa[u][i] * xa[u][i] + xb[u][i] * xb[u][i];
          dot += xa[u][i] * (ga[u][i] * lane.wa[i]) + xb[u][i] * (gb[u][i] * lane.wb[i]);
        }
        ss = nr_sum<G>(ss);
        dot = nr_sum<G>(dot);
        const float r = rsqrtf(ss * inv_d + c.eps);
        const float m = dot * inv_d * r * r * r;
        if (ok) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dwa[i] += ga[u][i] * (xa[u][i] * r);
            dwb[i] += gb[u][i] * (xb[u][i] * r);
            xa[u][i] = ga[u][i] * lane.wa[i] * r - xa[u][i] * m;
            xb[u][i] = gb[u][i] * lane.wb[i] * r - xb[u][i] * m;
          }
          nr_store4(dx + (int64_t)h * c.D + lane.a, xa[u]);
          nr_store4(dx + (int64_t)h * c.D + lane.b, xb[u]);
        }
      }
    }
  }
  if (partial == nullptr) return;  // uniform over the launch: no weight gradient is wanted
  if (lane.on) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lds[grp * c.D + lane.a + i] = dwa[i];
      lds[grp * c.D + lane.b + i] = dwb[i];
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < c.D; d += NR_THREADS) {
    float sum = 0.0f;
    for (int k = 0; k < GROUPS; ++k) sum += lds[k * c.D + d];
    partial[(int64_t)block * c.D + d] = sum;
  }
}

template <typename T, int G, bool IL>
__global__ __launch_bounds__(NR_THREADS) void nr_bwd_kernel(nr_side q, nr_side k, nr_common c, float* pq, float* pk) {
  __shared__ float lds[NR_THREADS * 8];  // [groups][D], D <= 8 G
  if (blockIdx.x < q.blocks) nr_bwd_body<T, G, IL>(q, c, blockIdx.x, pq, lds);
  else nr_bwd_body<T, G, IL>(k, c, blockIdx.x - q.blocks, pk, lds);
}

// Sums the blocks' rows of partial weight gradients in double: a block takes 8 elements of one side, 32 threads per
// element take every 32nd row, and their sums are added in order.
__global__ __launch_bounds__(NR_THREADS) void nr_weight_sum_kernel(const float* pq, const float* pk, float* dwq,
                                                                   float* dwk, uint32_t rows_q, uint32_t rows_k, int D) {
  __shared__ double part[32][8];
  const int slices = D / 8;
  const bool is_k = (int)blockIdx.x >= slices;
  const float* p = is_k ? pk : pq;
  float* out = is_k ? dwk : dwq;
  const uint32_t rows = is_k ? rows_k : rows_q;
  if (out == nullptr) return;
  const int e = threadIdx.x % 8, r0 = threadIdx.x / 8;
  const int d = ((int)blockIdx.x - (is_k ? slices : 0)) * 8 + e;
  double sum = 0.0;
  for (uint32_t r = r0; r < rows; r += 32 * 16) {  // sixteen loads in flight
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = r + 32 * i < rows ? p[(int64_t)(r + 32 * i) * D + d] : 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += (double)v[i];
  }
  part[r0][e] = sum;
  __syncthreads();
  if (r0 == 0) {
#pragma unroll
    for (int i = 1; i < 32; ++i) sum += part[i][e];
    out[d] = (float)sum;
  }
}

int nr_group(int D) {
  int g = 1;
  while (g * 8 < D) g *= 2;
  return g;
}

int nr_check_side(const rc_heads* s, const char* who, const void* y, int64_t N, int D, int dtype) {
  const int es = dtype == RC_F32 ? 4 : 2;
  RC_REQUIRE(s->T >= 0 && s->H >= 0, RC_EINVAL, "rc_qk_norm_rotate: negative size of %s", who);
  RC_REQUIRE(s->T < (1ll << 31) && N * s->T < (1ll << 31) && N * s->T * s->H < (1ll << 31), RC_EINVAL,
             "rc_qk_norm_rotate: %s has more than 2^31 heads", who);
  if (N * s->T * s->H == 0) return RC_OK;
  RC_REQUIRE(s->x != nullptr && y != nullptr, RC_EINVAL, "rc_qk_norm_rotate: null %s", who);
  RC_REQUIRE(((uintptr_t)s->x | (uintptr_t)y) % 16 == 0, RC_EINVAL, "rc_qk_norm_rotate: %s is not aligned to 16 bytes", who);
  for (int i = 0; i < 3; ++i)
    RC_REQUIRE(s->stride[i] >= 0 && s->stride[i] * es % 16 == 0, RC_EINVAL,
               "rc_qk_norm_rotate: stride %lld of %s is negative or no multiple of 16 bytes", (long long)s->stride[i], who);
  RC_REQUIRE(s->weight == nullptr || s->weight_dtype == RC_F32 || s->weight_dtype == RC_F16 || s->weight_dtype == RC_BF16,
             RC_EUNSUPPORTED, "rc_qk_norm_rotate: unknown weight dtype %d", s->weight_dtype);
  RC_REQUIRE(s->pos == nullptr || (s->pos_dtype >= RC_POS_I32 && s->pos_dtype <= RC_POS_F32), RC_EUNSUPPORTED,
             "rc_qk_norm_rotate: unknown position dtype %d", s->pos_dtype);
  return RC_OK;
}

int nr_check(const rc_heads* q, const rc_heads* k, const void* yq, const void* yk, int64_t N, int D, int dtype,
             const void* freqs, int n_freqs) {
  RC_REQUIRE(q != nullptr, RC_EINVAL, "rc_qk_norm_rotate: null queries");
  RC_REQUIRE(dtype == RC_F32 || dtype == RC_F16 || dtype == RC_BF16, RC_EUNSUPPORTED, "unknown dtype %d", dtype);
  RC_REQUIRE(N >= 0 && N < (1ll << 31), RC_EINVAL, "rc_qk_norm_rotate: N=%lld", (long long)N);
  RC_REQUIRE(D >= 8 && D <= RC_HEAD_DIM_MAX && D % 8 == 0, RC_EUNSUPPORTED,
             "head dimension %d is no multiple of 8 in 8..%d", D, RC_HEAD_DIM_MAX);
  RC_REQUIRE(n_freqs >= 0 && n_freqs % 4 == 0 && 2 * n_freqs <= D, RC_EUNSUPPORTED,
             "rc_qk_norm_rotate: %d frequencies for D=%d (a multiple of 4, at most D / 2)", n_freqs, D);
  RC_REQUIRE(n_freqs == 0 || freqs != nullptr, RC_EINVAL, "rc_qk_norm_rotate: null frequencies");
  int rc = nr_check_side(q, "q", yq, N, D, dtype);
  if (rc) return rc;
  return k == nullptr ? RC_OK : nr_check_side(k, "k", yk, N, D, dtype);
}

// Heads per group: a group that goes through more heads works its angles out fewer times, but a launch of few tokens
// needs every lane it can get.
nr_side nr_plan(const rc_heads* s, void* y, const void* g, int64_t N, int D, uint32_t max_blocks) {
  nr_side d = {};
  if (s == nullptr || N * s->T * s->H == 0) return d;
  d.x = s->x;
  d.y = y;
  d.g = g;
  d.w = s->weight;
  d.pos = s->pos;
  for (int i = 0; i < 3; ++i) d.stride[i] = s->stride[i];
  d.pos_stride = s->pos_stride;
  d.T = (uint32_t)s->T;
  d.tokens = (uint32_t)(N * s->T);
  d.H = s->H;
  d.w_dtype = s->weight_dtype;
  d.pos_dtype = s->pos_dtype;
  const int per = NR_THREADS / nr_group(D);
  int hp = s->H;
  while (hp > 1 && (int64_t)d.tokens * ((s->H + hp - 1) / hp) < 2048ll * per) hp = (hp + 1) / 2;
  d.heads_per_group = hp;
  d.chunks = (s->H + hp - 1) / hp;
  d.groups = d.tokens * (uint32_t)d.chunks;
  d.blocks = (d.groups + per - 1) / per;
  if (d.blocks > max_blocks) d.blocks = max_blocks;
  return d;
}

template <typename T, int G, bool IL>
void nr_launch(const nr_side& q, const nr_side& k, const nr_common& c, bool bwd, float* pq, float* pk, hipStream_t st) {
  if (bwd) nr_bwd_kernel<T, G, IL><<<q.blocks + k.blocks, NR_THREADS, 0, st>>>(q, k, c, pq, pk);
  else {
    const uint32_t blocks = q.blocks + k.blocks;
    const dim3 grid = blocks <= NR_GRID_X ? dim3(blocks) : dim3(NR_GRID_X, (blocks - 1) / NR_GRID_X + 1);
    nr_fwd_kernel<T, G, IL><<<grid, NR_THREADS, 0, st>>>(q, k, c);
  }
}

template <typename T, bool IL>
void nr_launch_g(const nr_side& q, const nr_side& k, const nr_common& c, bool bwd, float* pq, float* pk, hipStream_t st) {
  switch (nr_group(c.D)) {
    case 1: return nr_launch<T, 1, IL>(q, k, c, bwd, pq, pk, st);
    case 2: return nr_launch<T, 2, IL>(q, k, c, bwd, pq, pk, st);
    case 4: return nr_launch<T, 4, IL>(q, k, c, bwd, pq, pk, st);
    case 8: return nr_launch<T, 8, IL>(q, k, c, bwd, pq, pk, st);
    case 16: return nr_launch<T, 16, IL>(q, k, c, bwd, pq, pk, st);
    default: return nr_launch<T, 32, IL>(q, k, c, bwd, pq, pk, st);
  }
}

void nr_dispatch(int dtype, int interleaved, const nr_side& q, const nr_side& k, const nr_common& c, bool bwd, float* pq,
                 float* pk, hipStream_t st) {
  if (dtype == RC_F32) {
    if (interleaved) nr_launch_g<float, true>(q, k, c, bwd, pq, pk, st);
    else nr_launch_g<float, false>(q, k, c, bwd, pq, pk, st);
  } else if (dtype == RC_F16) {
    if (interleaved) nr_launch_g<rc_half, true>(q, k, c, bwd, pq, pk, st);
    else nr_launch_g<rc_half, false>(q, k, c, bwd, pq, pk, st);
  } else {
    if (interleaved) nr_launch_g<rc_bf16, true>(q, k, c, bwd, pq, pk, st);
    else nr_launch_g<rc_bf16, false>(q, k, c, bwd, pq, pk, st);
  }
}

}  // namespace

extern "C" int rc_qk_norm_rotate_fwd(const rc_heads* q, const rc_heads* k, void* yq, void* yk, int64_t N, int D,
                                     int dtype, const void* freqs, int freqs_f64, int n_freqs, int interleaved,
                                     float eps, void* stream) {
  const int rc = nr_check(q, k, yq, yk, N, D, dtype, freqs, n_freqs);
  if (rc) return rc;
  const nr_side sq = nr_plan(q, yq, nullptr, N, D, UINT32_MAX), sk = nr_plan(k, yk, nullptr, N, D, UINT32_MAX);
  if (sq.blocks + sk.blocks == 0) return RC_OK;
  const nr_common c = {freqs, freqs_f64, n_freqs, D, eps};
  nr_dispatch(dtype, interleaved, sq, sk, c, false, nullptr, nullptr, (hipStream_t)stream);
  return rc_check_launch("rc_qk_norm_rotate_fwd");
}

extern "C" int64_t rc_qk_norm_rotate_bwd_work_bytes(int D) {
  if (D < 8 || D > RC_HEAD_DIM_MAX || D % 8 != 0) return RC_EUNSUPPORTED;
  return 2ll * NR_MAX_BLOCKS * D * (int64_t)sizeof(float);
}

extern "C" int rc_qk_norm_rotate_bwd(const rc_heads* q, const rc_heads* k, const void* gq, const void* gk, void* dq,
                                     void* dk, float* dwq, float* dwk, void* work, int64_t N, int D, int dtype,
                                     const void* freqs, int freqs_f64, int n_freqs, int interleaved, float eps,
                                     void* stream) {
  int rc = nr_check(q, k, dq, dk, N, D, dtype, freqs, n_freqs);
  if (rc) return rc;
  RC_REQUIRE(N * q->T * q->H == 0 || (gq != nullptr && (uintptr_t)gq % 16 == 0), RC_EINVAL,
             "rc_qk_norm_rotate_bwd: gq is null or not aligned to 16 bytes");
  RC_REQUIRE(k == nullptr || N * k->T * k->H == 0 || (gk != nullptr && (uintptr_t)gk % 16 == 0), RC_EINVAL,
             "rc_qk_norm_rotate_bwd: gk is null or not aligned to 16 bytes");
  RC_REQUIRE((dwq == nullptr && dwk == nullptr) || (work != nullptr && (uintptr_t)work % 16 == 0), RC_EINVAL,
             "rc_qk_norm_rotate_bwd: work is null or not aligned to 16 bytes");
  RC_REQUIRE(k != nullptr || dwk == nullptr, RC_EINVAL, "rc_qk_norm_rotate_bwd: dwk without keys");
  // (two sides share the card: half the blocks each, so that both are resident at once, and half the rows to add up)
  const uint32_t most = k == nullptr ? NR_MAX_BLOCKS : NR_MAX_BLOCKS / 2;
  const nr_side sq = nr_plan(q, dq, gq, N, D, most), sk = nr_plan(k, dk, gk, N, D, most);
  const nr_common c = {freqs, freqs_f64, n_freqs, D, eps};
  float* pq = dwq ? reinterpret_cast<float*>(work) : nullptr;
  float* pk = dwk ? reinterpret_cast<float*>(work) + (int64_t)NR_MAX_BLOCKS * D : nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (sq.blocks + sk.blocks) {
    nr_dispatch(dtype, interleaved, sq, sk, c, true, pq, pk, st);
    rc = rc_check_launch("rc_qk_norm_rotate_bwd");
    if (rc) return rc;
  }
  if (dwq || dwk) {
    nr_weight_sum_kernel<<<2 * (D / 8), NR_THREADS, 0, st>>>(pq, pk, dwq, dwk, sq.blocks, sk.blocks, D);
    rc = rc_check_launch("rc_qk_norm_rotate_bwd (weights)");
  }
  return rc;
}
