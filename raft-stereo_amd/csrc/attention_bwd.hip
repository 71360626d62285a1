// Attention of query tokens over the tokens of another sequence, and its adjoint.
//
//   S = scale Q K^T,  P = softmax(S) over the allowed keys,  O = P V
//   lse2 = log2 sum exp2(S log2 e);   delta = sum_d dO O;   dS = P (dO V^T - delta)
//   dV = P^T dO,   dQ = scale dS K,   dK = scale dS^T Q
#include "attention.h"

namespace {

constexpr int AT_WAVES = 4;

__device__ __forceinline__ bool at_allowed(const at_args& a, int n, int key, int len) {
  return key < len && (a.bits == nullptr || (a.bits[(int64_t)n * a.words + (key >> 6)] >> (key & 63)) & 1);
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

// delta[n, h, t] = sum_d dO O, one wave per row
template <typename T>
__global__ __launch_bounds__(AT_WAVES * 64) void at_delta_kernel(const T* __restrict__ out, const T* __restrict__ dout,
                                                                 float* __restrict__ delta, at_args a) {
  const int64_t row = (int64_t)blockIdx.x * AT_WAVES + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= (int64_t)a.N * a.Tq * a.Hq) return;
  float s = 0.0f;
  for (int d = lane; d < a.D; d += 64) s += rc_to_float(out[row * a.D + d]) * rc_to_float(dout[row * a.D + d]);
  s = at_wave_sum(s);
  const int h = (int)(row % a.Hq);
  const int64_t nt = row / a.Hq;
  const int n = (int)(nt / a.Tq), t = (int)(nt - (int64_t)n * a.Tq);
  if (lane == 0) delta[((int64_t)n * a.Hq + h) * a.Tq + t] = s;
}

template <typename T>
__global__ __launch_bounds__(AT_WAVES * 64) void at_dq_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                              const T* __restrict__ v, const T* __restrict__ dout,
                                                              const float* __restrict__ lse,
                                                              const float* __restrict__ delta, T* __restrict__ dq,
                                                              at_args a) {
  __shared__ float qrow[AT_WAVES][RC_HEAD_DIM_MAX], grow[AT_WAVES][RC_HEAD_DIM_MAX];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t rows = (int64_t)a.N * a.Tq * a.Hq;
  int64_t row = (int64_t)blockIdx.x * AT_WAVES + wave;
  const bool live = row < rows;
  row = live ? row : rows - 1;
  const int h = (int)(row % a.Hq);
  const int64_t nt = row / a.Hq;
  const int n = (int)(nt / a.Tq), t = (int)(nt - (int64_t)n * a.Tq);
  const int hk = h / (a.Hq / a.Hk);
  const T* qp = q + n * a.qs[0] + t * a.qs[1] + h * a.qs[2];
  for (int d = lane; d < a.D; d += 64) {
    qrow[wave][d] = rc_to_float(qp[d]);
    grow[wave][d] = rc_to_float(dout[row * a.D + d]);
  }
  __syncthreads();
  const int len = at_length(a, n);
  const float L = lse[((int64_t)n * a.Hq + h) * a.Tq + t], dl = delta[((int64_t)n * a.Hq + h) * a.Tq + t];
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
  const int64_t rows = (int64_t)a.N * a.Tk * a.Hk;
  int64_t row = (int64_t)blockIdx.x * AT_WAVES + wave;
  const bool live = row < rows;
  row = live ? row : rows - 1;
  const int hk = (int)(row % a.Hk), group = a.Hq / a.Hk;
  const int64_t nt = row / a.Hk;
  const int n = (int)(nt / a.Tk), t = (int)(nt - (int64_t)n * a.Tk);
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
          const float dp = at_dot(vrow[wave], dout + (((int64_t)n * a.Tq + tq) * a.Hq + h) * a.D, a.D);
          p = exp2f(s - lse[((int64_t)n * a.Hq + h) * a.Tq + tq]);
          ds = p * (dp - delta[((int64_t)n * a.Hq + h) * a.Tq + tq]);
        }
        for (int j = 0; j < 64 && t0 + j < a.Tq; ++j) {
          const float pj = __shfl(p, j), dj = __shfl(ds, j);
          const T* qp = q + n * a.qs[0] + (t0 + j) * a.qs[1] + h * a.qs[2];
          const T* gp = dout + (((int64_t)n * a.Tq + t0 + j) * a.Hq + h) * a.D;
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

int64_t at_blocks(int64_t rows) { return (rows + AT_WAVES - 1) / AT_WAVES; }

template <typename T>
int at_bwd(const rc_attn* a, const void* q, const void* k, const void* v, const void* out, const float* lse,
           const void* dout, void* dq, void* dk, void* dv, void* work, hipStream_t st) {
  const at_args d = at_to_dev(a, work);
  float* delta = reinterpret_cast<float*>(reinterpret_cast<char*>(work) + at_bits_bytes(a));
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

extern "C" int64_t rc_cross_attn_bwd_work_bytes(const rc_attn* a) {
  const int rc = at_check(a);
  if (rc) return rc < 0 ? rc : RC_EINVAL;
  return at_bits_bytes(a) + a->N * a->Tq * a->Hq * (int64_t)sizeof(float);
}

extern "C" int rc_cross_attn_bwd(const rc_attn* a, const void* q, const void* k, const void* v, const void* out,
                                 const float* lse, const void* dout, void* dq, void* dk, void* dv, void* work,
                                 void* stream) {
  int rc = at_check(a);
  if (rc) return rc;
  for (const void* p : {q, out, (const void*)lse, dout, (const void*)work})
    if ((rc = at_check_operand(a, a->N * a->Tq, p))) return rc;
  for (const void* p : {k, v})
    if ((rc = at_check_operand(a, a->N * a->Tk, p))) return rc;
  RC_REQUIRE(at_bits_bytes(a) == 0 || (work != nullptr && (uintptr_t)work % 16 == 0), RC_EINVAL,
             "rc_cross_attn_bwd: work is null or not aligned to 16 bytes");
  RC_REQUIRE((dk == nullptr) == (dv == nullptr), RC_EINVAL, "rc_cross_attn_bwd: dk and dv are wanted together or not at all");
  RC_REQUIRE(((uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16 == 0, RC_EINVAL,
             "rc_cross_attn_bwd: a gradient is not aligned to 16 bytes");
  if (a->N == 0) return RC_OK;
  if ((rc = at_launch_bits(a, work, (hipStream_t)stream))) return rc;
  if (a->dtype == RC_F32) return at_bwd<float>(a, q, k, v, out, lse, dout, dq, dk, dv, work, (hipStream_t)stream);
  if (a->dtype == RC_F16) return at_bwd<rc_half>(a, q, k, v, out, lse, dout, dq, dk, dv, work, (hipStream_t)stream);
  return at_bwd<rc_bf16>(a, q, k, v, out, lse, dout, dq, dk, dv, work, (hipStream_t)stream);
}
