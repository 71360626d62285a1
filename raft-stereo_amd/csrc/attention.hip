// Attention of query tokens over the tokens of another sequence, and its adjoint.
//
//   S = scale Q K^T,  P = softmax(S) over the allowed keys,  O = P V
//   lse2 = log2 sum exp2(S log2 e);   delta = sum_d dO O;   dS = P (dO V^T - delta)
//   dV = P^T dO,   dQ = scale dS K,   dK = scale dS^T Q
#include "rc_common.h"

#include <math.h>

#include <initializer_list>

namespace {

constexpr int AT_WAVES = 4;

struct at_args {
  int64_t qs[3], ks[3], vs[3];
  int64_t mask_stride;
  const void* lengths;
  const unsigned char* mask;
  int64_t N;
  int32_t Tq, Tk, Hq, Hk, D;
  int32_t lengths_i64;
  float scale, scale_log2;
};

// keys of sequence n that may be attended to by its length alone
__device__ __forceinline__ int at_length(const at_args& a, int64_t n) {
  if (a.lengths == nullptr) return a.Tk;
  int64_t l = a.lengths_i64 ? reinterpret_cast<const int64_t*>(a.lengths)[n]
                            : (int64_t) reinterpret_cast<const int32_t*>(a.lengths)[n];
  l = l < 0 ? 0 : l;
  return (int)(l > a.Tk ? a.Tk : l);
}
__device__ __forceinline__ bool at_allowed(const at_args& a, int64_t n, int key, int len) {
  return key < len && (a.mask == nullptr || a.mask[n * a.mask_stride + key] != 0);
}

__device__ __forceinline__ float at_wave_max(float v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}
__device__ __forceinline__ float at_wave_sum(float v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

template <typename T> __device__ __forceinline__ float at_dot(const float* a, const T* b, int D) {
  float s = 0.0f;
  for (int d = 0; d < D; ++d) s += a[d] * rc_to_float(b[d]);
  return s;
}

// One wave per query row: 64 keys at a time, a lane for each, then the lanes take 4 output elements each.
template <typename T>
__global__ __launch_bounds__(AT_WAVES * 64) void at_fwd_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                               const T* __restrict__ v, T* __restrict__ out,
                                                               float* __restrict__ lse, at_args a) {
  __shared__ float qrow[AT_WAVES][RC_HEAD_DIM_MAX];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t rows = a.N * a.Tq * a.Hq;
  int64_t row = (int64_t)blockIdx.x * AT_WAVES + wave;
  const bool live = row < rows;
  row = live ? row : rows - 1;
  const int h = (int)(row % a.Hq);
  const int64_t nt = row / a.Hq, n = nt / a.Tq, t = nt - n * a.Tq;
  const int hk = h / (a.Hq / a.Hk);
  const T* qp = q + n * a.qs[0] + t * a.qs[1] + h * a.qs[2];
  for (int d = lane; d < a.D; d += 64) qrow[wave][d] = rc_to_float(qp[d]);
  __syncthreads();
  const int len = at_length(a, n);
  float m = -INFINITY, l = 0.0f, acc[4] = {0, 0, 0, 0};
  bool any = false;
  for (int k0 = 0; k0 < len; k0 += 64) {
    const int key = k0 + lane;
    const bool ok = at_allowed(a, n, key, len);
    float s = -INFINITY;
    if (ok) s = at_dot(qrow[wave], k + n * a.ks[0] + key * a.ks[1] + hk * a.ks[2], a.D) * a.scale_log2;
    const unsigned long long okm = __ballot(ok);
    any = any || okm != 0;
    const float mn = fmaxf(m, at_wave_max(s));
    const float mu = mn == -INFINITY ? 0.0f : mn;
    const float f = exp2f(m - mu), p = ok ? exp2f(s - mu) : 0.0f;
    m = mn;
    l = l * f + at_wave_sum(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= f;
    for (int j = 0; j < 64 && k0 + j < len; ++j) {
      if (!((okm >> j) & 1)) continue;
      const float pj = __shfl(p, j);
      const T* vp = v + n * a.vs[0] + (int64_t)(k0 + j) * a.vs[1] + hk * a.vs[2];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < a.D) acc[i] += pj * rc_to_float(vp[lane + 64 * i]);
    }
  }
  if (!live) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < a.D) out[row * a.D + lane + 64 * i] = rc_from_float<T>(any ? acc[i] / l : 0.0f);
  if (lse != nullptr && lane == 0) lse[(n * a.Hq + h) * a.Tq + t] = any ? m + log2f(l) : INFINITY;
}

// delta[n, h, t] = sum_d dO O, one wave per row
template <typename T>
__global__ __launch_bounds__(AT_WAVES * 64) void at_delta_kernel(const T* __restrict__ out, const T* __restrict__ dout,
                                                                 float* __restrict__ delta, at_args a) {
  const int64_t row = (int64_t)blockIdx.x * AT_WAVES + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= a.N * a.Tq * a.Hq) return;
  float s = 0.0f;
  for (int d = lane; d < a.D; d += 64) s += rc_to_float(out[row * a.D + d]) * rc_to_float(dout[row * a.D + d]);
  s = at_wave_sum(s);
  const int h = (int)(row % a.Hq);
  const int64_t nt = row / a.Hq, n = nt / a.Tq, t = nt - n * a.Tq;
  if (lane == 0) delta[(n * a.Hq + h) * a.Tq + t] = s;
}

template <typename T>
__global__ __launch_bounds__(AT_WAVES * 64) void at_dq_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                              const T* __restrict__ v, const T* __restrict__ dout,
                                                              const float* __restrict__ lse,
                                                              const float* __restrict__ delta, T* __restrict__ dq,
                                                              at_args a) {
  __shared__ float qrow[AT_WAVES][RC_HEAD_DIM_MAX], grow[AT_WAVES][RC_HEAD_DIM_MAX];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t rows = a.N * a.Tq * a.Hq;
  int64_t row = (int64_t)blockIdx.x * AT_WAVES + wave;
  const bool live = row < rows;
  row = live ? row : rows - 1;
  const int h = (int)(row % a.Hq);
  const int64_t nt = row / a.Hq, n = nt / a.Tq, t = nt - n * a.Tq;
  const int hk = h / (a.Hq / a.Hk);
  const T* qp = q + n * a.qs[0] + t * a.qs[1] + h * a.qs[2];
  for (int d = lane; d < a.D; d += 64) {
    qrow[wave][d] = rc_to_float(qp[d]);
    grow[wave][d] = rc_to_float(dout[row * a.D + d]);
  }
  __syncthreads();
  const int len = at_length(a, n);
  const float L = lse[(n * a.Hq + h) * a.Tq + t], dl = delta[(n * a.Hq + h) * a.Tq + t];
  float acc[4] = {0, 0, 0, 0};
  for (int k0 = 0; k0 < len; k0 += 64) {
    const int key = k0 + lane;
    const bool ok = at_allowed(a, n, key, len);
    float ds = 0.0f;
    if (ok) {
      const float s = at_dot(qrow[wave], k + n * a.ks[0] + key * a.ks[1] + hk * a.ks[2], a.D) * a.scale_log2;
      const float dp = at_dot(grow[wave], v + n * a.vs[0] + key * a.vs[1] + hk * a.vs[2], a.D);
      ds = exp2f(s - L) * (dp - dl);
    }
    const unsigned long long okm = __ballot(ok);
    for (int j = 0; j < 64 && k0 + j < len; ++j) {
      if (!((okm >> j) & 1)) continue;
      const float dj = __shfl(ds, j);
      const T* kp = k + n * a.ks[0] + (int64_t)(k0 + j) * a.ks[1] + hk * a.ks[2];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < a.D) acc[i] += dj * rc_to_float(kp[lane + 64 * i]);
    }
  }
  if (!live) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < a.D) dq[row * a.D + lane + 64 * i] = rc_from_float<T>(acc[i] * a.scale);
}

// One wave per key row: 64 query rows of the group at a time.
template <typename T>
__global__ __launch_bounds__(AT_WAVES * 64) void at_dkv_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                               const T* __restrict__ v, const T* __restrict__ dout,
                                                               const float* __restrict__ lse,
                                                               const float* __restrict__ delta, T* __restrict__ dk,
                                                               T* __restrict__ dv, at_args a) {
  __shared__ float krow[AT_WAVES][RC_HEAD_DIM_MAX], vrow[AT_WAVES][RC_HEAD_DIM_MAX];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t rows = a.N * a.Tk * a.Hk;
  int64_t row = (int64_t)blockIdx.x * AT_WAVES + wave;
  const bool live = row < rows;
  row = live ? row : rows - 1;
  const int hk = (int)(row % a.Hk), group = a.Hq / a.Hk;
  const int64_t nt = row / a.Hk, n = nt / a.Tk, t = nt - n * a.Tk;
  const bool ok = at_allowed(a, n, (int)t, at_length(a, n));
  for (int d = lane; d < a.D; d += 64) {
    krow[wave][d] = rc_to_float(k[n * a.ks[0] + t * a.ks[1] + hk * a.ks[2] + d]);
    vrow[wave][d] = rc_to_float(v[n * a.vs[0] + t * a.vs[1] + hk * a.vs[2] + d]);
  }
  __syncthreads();
  float ak[4] = {0, 0, 0, 0}, av[4] = {0, 0, 0, 0};
  if (ok) {
    for (int g = 0; g < group; ++g) {
      const int h = hk * group + g;
      for (int t0 = 0; t0 < a.Tq; t0 += 64) {
        const int tq = t0 + lane;
        float p = 0.0f, ds = 0.0f;
        if (tq < a.Tq) {
          const float s = at_dot(krow[wave], q + n * a.qs[0] + tq * a.qs[1] + h * a.qs[2], a.D) * a.scale_log2;
          const float dp = at_dot(vrow[wave], dout + ((n * a.Tq + tq) * a.Hq + h) * a.D, a.D);
          p = exp2f(s - lse[(n * a.Hq + h) * a.Tq + tq]);
          ds = p * (dp - delta[(n * a.Hq + h) * a.Tq + tq]);
        }
        for (int j = 0; j < 64 && t0 + j < a.Tq; ++j) {
          const float pj = __shfl(p, j), dj = __shfl(ds, j);
          const T* qp = q + n * a.qs[0] + (t0 + j) * a.qs[1] + h * a.qs[2];
          const T* gp = dout + ((n * a.Tq + t0 + j) * a.Hq + h) * a.D;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < a.D) {
              ak[i] += dj * rc_to_float(qp[lane + 64 * i]);
              av[i] += pj * rc_to_float(gp[lane + 64 * i]);
            }
        }
      }
    }
  }
  if (!live) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < a.D) {
      dk[row * a.D + lane + 64 * i] = rc_from_float<T>(ak[i] * a.scale);
      dv[row * a.D + lane + 64 * i] = rc_from_float<T>(av[i]);
    }
}

int at_check(const rc_attn* a) {
  RC_REQUIRE(a != nullptr, RC_EINVAL, "rc_cross_attn: null description");
  RC_REQUIRE(a->dtype == RC_F32 || a->dtype == RC_F16 || a->dtype == RC_BF16, RC_EUNSUPPORTED, "unknown dtype %d", a->dtype);
  RC_REQUIRE(a->D >= 8 && a->D <= RC_HEAD_DIM_MAX && a->D % 8 == 0, RC_EUNSUPPORTED,
             "head dimension %d is no multiple of 8 in 8..%d", a->D, RC_HEAD_DIM_MAX);
  RC_REQUIRE(a->N >= 0 && a->N < (1ll << 31) && a->Tq >= 0 && a->Tk >= 0 && a->Hq >= 1 && a->Hk >= 1, RC_EINVAL,
             "rc_cross_attn: negative size, or no head");
  RC_REQUIRE(a->Hq % a->Hk == 0, RC_EINVAL, "rc_cross_attn: %d query heads are no multiple of %d key heads", a->Hq, a->Hk);
  RC_REQUIRE(a->Tq < (1ll << 30) && a->Tk < (1ll << 30) && a->N * a->Tq < (1ll << 31) && a->N * a->Tk < (1ll << 31) &&
                 a->N * a->Tq * a->Hq < (1ll << 31) && a->N * a->Tk * a->Hk < (1ll << 31),
             RC_EINVAL, "rc_cross_attn: more than 2^31 heads");
  RC_REQUIRE(a->scale > 0.0f && a->scale < INFINITY, RC_EINVAL, "rc_cross_attn: scale must be positive and finite");
  const int64_t es = a->dtype == RC_F32 ? 4 : 2;
  const int64_t* st[3] = {a->q_stride, a->k_stride, a->v_stride};
  for (int o = 0; o < 3; ++o)
    for (int i = 0; i < 3; ++i)
      RC_REQUIRE(st[o][i] >= 0 && st[o][i] * es % 16 == 0 && (i == 0 || st[o][i] * es < (1ll << 24)), RC_EINVAL,
                 "rc_cross_attn: stride %lld of %c is negative, no multiple of 16 bytes, or 16 MiB or more between tokens "
                 "or heads", (long long)st[o][i], "qkv"[o]);
  RC_REQUIRE(a->key_mask == nullptr || a->mask_stride >= 0, RC_EINVAL, "rc_cross_attn: negative mask stride");
  return RC_OK;
}

at_args at_to_dev(const rc_attn* a) {
  at_args d;
  for (int i = 0; i < 3; ++i) {
    d.qs[i] = a->q_stride[i];
    d.ks[i] = a->k_stride[i];
    d.vs[i] = a->v_stride[i];
  }
  d.mask_stride = a->mask_stride;
  d.lengths = a->key_lengths;
  d.mask = a->key_mask;
  d.N = a->N;
  d.Tq = (int32_t)a->Tq;
  d.Tk = (int32_t)a->Tk;
  d.Hq = a->Hq;
  d.Hk = a->Hk;
  d.D = a->D;
  d.lengths_i64 = a->lengths_i64;
  d.scale = a->scale;
  d.scale_log2 = a->scale * 1.44269504088896340736f;
  return d;
}

int at_check_ptrs(const rc_attn* a, std::initializer_list<const void*> query_side, std::initializer_list<const void*> key_side) {
  if (a->N * a->Tq)
    for (const void* p : query_side)
      RC_REQUIRE(p != nullptr && (uintptr_t)p % 16 == 0, RC_EINVAL, "rc_cross_attn: an operand is null or not aligned to 16 bytes");
  if (a->N * a->Tk)
    for (const void* p : key_side)
      RC_REQUIRE(p != nullptr && (uintptr_t)p % 16 == 0, RC_EINVAL, "rc_cross_attn: an operand is null or not aligned to 16 bytes");
  return RC_OK;
}

int64_t at_blocks(int64_t rows) { return (rows + AT_WAVES - 1) / AT_WAVES; }

template <typename T>
int at_fwd(const rc_attn* a, const void* q, const void* k, const void* v, void* out, float* lse, hipStream_t st) {
  const int64_t rows = a->N * a->Tq * a->Hq;
  at_fwd_kernel<T><<<at_blocks(rows), AT_WAVES * 64, 0, st>>>((const T*)q, (const T*)k, (const T*)v, (T*)out, lse, at_to_dev(a));
  return rc_check_launch("rc_cross_attn_fwd");
}

template <typename T>
int at_bwd(const rc_attn* a, const void* q, const void* k, const void* v, const void* out, const float* lse,
           const void* dout, void* dq, void* dk, void* dv, float* delta, hipStream_t st) {
  const at_args d = at_to_dev(a);
  const int64_t rows = a->N * a->Tq * a->Hq, keys = a->N * a->Tk * a->Hk;
  if (rows) {  // (the gradients of keys and values need delta too)
    at_delta_kernel<T><<<at_blocks(rows), AT_WAVES * 64, 0, st>>>((const T*)out, (const T*)dout, delta, d);
    if (dq) at_dq_kernel<T><<<at_blocks(rows), AT_WAVES * 64, 0, st>>>((const T*)q, (const T*)k, (const T*)v, (const T*)dout, lse,
                                                               delta, (T*)dq, d);
  }
  if (keys && dk)
    at_dkv_kernel<T><<<at_blocks(keys), AT_WAVES * 64, 0, st>>>((const T*)q, (const T*)k, (const T*)v, (const T*)dout,
                                                                lse, delta, (T*)dk, (T*)dv, d);
  return rc_check_launch("rc_cross_attn_bwd");
}

}  // namespace

extern "C" int64_t rc_cross_attn_fwd_work_bytes(const rc_attn* a) {
  const int rc = at_check(a);
  return rc ? (rc < 0 ? rc : RC_EINVAL) : 0;
}

extern "C" int rc_cross_attn_fwd(const rc_attn* a, const void* q, const void* k, const void* v, void* out, float* lse,
                                 void* work, void* stream) {
  int rc = at_check(a);
  if (rc) return rc;
  rc = at_check_ptrs(a, {q, out}, {k, v});
  if (rc || a->N * a->Tq == 0) return rc;
  if (a->dtype == RC_F32) return at_fwd<float>(a, q, k, v, out, lse, (hipStream_t)stream);
  if (a->dtype == RC_F16) return at_fwd<rc_half>(a, q, k, v, out, lse, (hipStream_t)stream);
  return at_fwd<rc_bf16>(a, q, k, v, out, lse, (hipStream_t)stream);
}

extern "C" int64_t rc_cross_attn_bwd_work_bytes(const rc_attn* a) {
  const int rc = at_check(a);
  if (rc) return rc < 0 ? rc : RC_EINVAL;
  return a->N * a->Tq * a->Hq * (int64_t)sizeof(float);
}

extern "C" int rc_cross_attn_bwd(const rc_attn* a, const void* q, const void* k, const void* v, const void* out,
                                 const float* lse, const void* dout, void* dq, void* dk, void* dv, void* work,
                                 void* stream) {
  int rc = at_check(a);
  if (rc) return rc;
  rc = at_check_ptrs(a, {q, out, lse, dout, work}, {k, v});
  if (rc) return rc;
  RC_REQUIRE((dk == nullptr) == (dv == nullptr), RC_EINVAL, "rc_cross_attn_bwd: dk and dv are wanted together or not at all");
  RC_REQUIRE(((uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16 == 0, RC_EINVAL,
             "rc_cross_attn_bwd: a gradient is not aligned to 16 bytes");
  if (rc || a->N == 0) return rc;
  if (a->dtype == RC_F32) return at_bwd<float>(a, q, k, v, out, lse, dout, dq, dk, dv, (float*)work, (hipStream_t)stream);
  if (a->dtype == RC_F16) return at_bwd<rc_half>(a, q, k, v, out, lse, dout, dq, dk, dv, (float*)work, (hipStream_t)stream);
  return at_bwd<rc_bf16>(a, q, k, v, out, lse, dout, dq, dk, dv, (float*)work, (hipStream_t)stream);
}
