// What the attention kernels share: arguments, the matrix-instruction fragments, and the staging of tiles of rows.
//
// A tile is a number of rows (tokens of one head) in LDS, RB bytes each (the head padded with zeros to a power of
// two), cut into 16-byte chunks, with PAD bytes behind every eight rows: chunk c of row r lies at
// r * RB + r / 8 * PAD + ((c ^ f(r)) << 4).  LDS has 64 banks, 256 bytes a cycle.  The transposing read (a fragment whose
// reduction runs across rows) takes 64 bytes of each of four consecutive rows in a cycle: f sends them to the four
// quarters of the 256 bytes.  A fragment whose reduction runs along the row takes the same chunk of sixteen consecutive
// rows: f has eight values for them, and the pad moves the second eight to the places between.  (f by itself could take
// sixteen values, at twice the address registers.)  Rows of 64 bytes go without the pad, and two of the sixteen meet.
//
// The 32x32 matrix instructions give lane l = 32 h + c the column c and, in register i, the row 8 (i / 4) + 4 h + i % 4
// of the result.  As the order of the reduction index is free as long as both operands agree, a result (probabilities,
// keys by queries) is the right operand of the next product as it stands: slot (h, j) of the 16 keys from 16 b is key
// 16 b + 8 (j / 4) + 4 h + j % 4, and the left operand's rows are read in that order.
#pragma once
#include "rc_common.h"

#include <atomic>
#include <math.h>

typedef short at_s4 __attribute__((ext_vector_type(4)));
typedef short at_s8 __attribute__((ext_vector_type(8)));
typedef float at_f16 __attribute__((ext_vector_type(16)));
typedef float at_f4 __attribute__((ext_vector_type(4)));
typedef float at_f2 __attribute__((ext_vector_type(2)));
typedef uint32_t at_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t at_u2 __attribute__((ext_vector_type(2)));
typedef _Float16 at_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 at_h2 __attribute__((ext_vector_type(2)));
typedef __bf16 at_b8 __attribute__((ext_vector_type(8)));
typedef __bf16 at_b2 __attribute__((ext_vector_type(2)));

// n / d for 0 <= n < 2^31 by one multiplication: m = ceil(2^(31 + s) / d), s = ceil(log2 d).
struct at_div {
  uint32_t m, s, d;
  __host__ at_div() : m(0), s(0), d(0) {}
  __host__ explicit at_div(uint32_t by) : s(0), d(by) {
    while (s < 31 && (1u << s) < d) ++s;
    m = (uint32_t)(((1ull << (31 + s)) + d - 1) / (d ? d : 1));
  }
  __device__ __forceinline__ int of(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n, m) >> (s - 1)); }
};

// A launch holds fewer than 2^32 threads along x: larger grids go along y too, in rows of 2^22 blocks (a multiple of the
// XCDs that block ids go round).
inline dim3 at_grid(int64_t blocks) {
  return blocks <= 1 << 22 ? dim3((uint32_t)blocks) : dim3(1u << 22, (uint32_t)((blocks + (1 << 22) - 1) >> 22));
}
__device__ __forceinline__ uint32_t at_block() { return (blockIdx.y << 22) + blockIdx.x; }

struct at_args {
  int64_t qs[3], ks[3], vs[3];  // elements between sequences, tokens, heads
  const void* lengths;
  const uint64_t* bits;  // [N][words], bit t % 64 of word t / 64: key t takes part; NULL: the lengths say it
  int64_t words;
  int32_t N, Tq, Tk, Hq, Hk, G, D;
  at_div by_Hk, by_G;
  int32_t lengths_i64;
  float scale, scale_log2;
};

// Raises KERNEL's limit of dynamic LDS, once per device (the call is idempotent: two first calls at once do it twice).
template <auto KERNEL> int at_allow_lds(int bytes) {
  static std::atomic<bool> done[64];
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e == hipSuccess && dev >= 0 && dev < 64 && done[dev]) return RC_OK;
  if (e == hipSuccess)
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) {
    rc_set_error("rc_cross_attn: %d bytes of LDS refused: %s", bytes, hipGetErrorString(e));
    return (int)e;
  }
  if (dev >= 0 && dev < 64) done[dev] = true;
  return RC_OK;
}

// host side (attention_rows.hip): the backward pass in one kernel where a sequence's keys fit a workgroup
bool at_rows_fit(const rc_attn* a);
int at_rows_bwd(const rc_attn* a, const at_args& d, const void* q, const void* k, const void* v, const void* out,
                const void* rest, const float* lse, const void* dout, void* dq, void* dk, void* dv, hipStream_t st);
// host side (attention_fwd.hip)
int at_check(const rc_attn* a);
int at_check_operand(const rc_attn* a, int64_t rows, const void* p);
at_args at_to_dev(const rc_attn* a, void* bits);
int64_t at_bits_bytes(const rc_attn* a);  // scratch of the mask's bits, a multiple of 256
int at_launch_bits(const rc_attn* a, void* bits, hipStream_t st);

__device__ __forceinline__ int at_length(const at_args& a, int n) {
  if (a.lengths == nullptr) return a.Tk;
  int64_t l = a.lengths_i64 ? reinterpret_cast<const int64_t*>(a.lengths)[n]
                            : (int64_t) reinterpret_cast<const int32_t*>(a.lengths)[n];
  l = l < 0 ? 0 : l;
  return __builtin_amdgcn_readfirstlane((int)(l > a.Tk ? a.Tk : l));
}

// one bit for each of the first `left` of 32 rows
__device__ __forceinline__ uint32_t at_first_bits(int left) {
  return left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
}

// the keys k0 .. k0 + 31 (k0 a multiple of 32) that take part, one bit each
__device__ __forceinline__ uint32_t at_key_bits(const at_args& a, int n, int len, int k0) {
  const int left = len - k0;
  uint32_t w = at_first_bits(left);
  // (the address is the same for the whole wave and nothing writes there: a scalar load, which does not wait behind the
  // tiles' loads)
  if (a.bits != nullptr && left > 0)
    w &= reinterpret_cast<const uint32_t __attribute__((address_space(4)))*>((uint64_t)a.bits)[((int64_t)n * a.words) * 2 + (k0 >> 5)];
  return __builtin_amdgcn_readfirstlane(w);
}

// ------------------------------------------------------------------------------------------------ matrix fragments
// One step of a product: 16 bytes per lane of each operand, elements along the reduction.
__device__ __forceinline__ at_f16 at_mma(rc_half, at_u4 a, at_u4 b, at_f16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(at_h8, a), __builtin_bit_cast(at_h8, b), c, 0, 0, 0);
}
__device__ __forceinline__ at_f16 at_mma(rc_bf16, at_u4 a, at_u4 b, at_f16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(at_b8, a), __builtin_bit_cast(at_b8, b), c, 0, 0, 0);
}
__device__ __forceinline__ at_f16 at_mma(float, at_u4 a, at_u4 b, at_f16 c) {
  // (whole vectors are cast: __builtin_bit_cast of one element takes the first)
  const at_f4 x = __builtin_bit_cast(at_f4, a), y = __builtin_bit_cast(at_f4, b);
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
  return c;
}

// What a block of 32 keys' scores start from: 0, or -inf for the keys whose bit in `take` is not set (the same for the
// whole wave).  The mask costs a select and a product of one column by one row: -inf or 0 of this lane's key by 1.
// COLS: the keys are the result's columns.
template <typename T, bool COLS = false> __device__ __forceinline__ at_f16 at_start(uint32_t take, int lane) {
  at_f16 s = (at_f16)(0.0f);
  if (take != 0xffffffffu) {
    const bool out = lane < 32 && !((take >> lane) & 1);
    const uint32_t inf = sizeof(T) == 4 ? 0xff800000u : __is_same(T, rc_half) ? 0xfc00u : 0xff80u;
    const uint32_t one = sizeof(T) == 4 ? 0x3f800000u : __is_same(T, rc_half) ? 0x3c00u : 0x3f80u;
    const at_u4 keys = {out ? inf : 0u, 0u, 0u, 0u}, ones = {lane < 32 ? one : 0u, 0u, 0u, 0u};
    const at_u4 x = COLS ? ones : keys, y = COLS ? keys : ones;
    if constexpr (sizeof(T) == 4) {
      const at_f4 u = __builtin_bit_cast(at_f4, x), w = __builtin_bit_cast(at_f4, y);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(u[0], w[0], s, 0, 0, 0);
    } else {
      s = at_mma(T(), x, y, s);
    }
  }
  return s;
}

// products of 16 bytes of elements, summed in fp32
__device__ __forceinline__ float at_dot(rc_half, at_u4 a, at_u4 b) {
  const at_h8 x = __builtin_bit_cast(at_h8, a), y = __builtin_bit_cast(at_h8, b);
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += (float)x[i] * (float)y[i];
  return s;
}
__device__ __forceinline__ float at_dot(rc_bf16, at_u4 a, at_u4 b) {
  const at_b8 x = __builtin_bit_cast(at_b8, a), y = __builtin_bit_cast(at_b8, b);
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += (float)x[i] * (float)y[i];
  return s;
}
__device__ __forceinline__ float at_dot(float, at_u4 a, at_u4 b) {
  const at_f4 x = __builtin_bit_cast(at_f4, a), y = __builtin_bit_cast(at_f4, b);
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) s += x[i] * y[i];
  return s;
}

__device__ __forceinline__ uint32_t at_pack(rc_half, float x, float y) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((at_f2){x, y}, at_h2));
}
__device__ __forceinline__ uint32_t at_pack(rc_bf16, float x, float y) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((at_f2){x, y}, at_b2));
}

// The halves of the wave exchange: afterwards a holds the lower halves of both, b the upper ones.
__device__ __forceinline__ void at_swap(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
__device__ __forceinline__ at_f2 at_unpack(rc_half, uint32_t x) {
  const at_h2 v = __builtin_bit_cast(at_h2, x);
  return at_f2{(float)v[0], (float)v[1]};
}
__device__ __forceinline__ at_f2 at_unpack(rc_bf16, uint32_t x) {
  const at_b2 v = __builtin_bit_cast(at_b2, x);
  return at_f2{(float)v[0], (float)v[1]};
}

// both halves see their two values
__device__ __forceinline__ void at_both(float x, float& lo, float& hi) {
  uint32_t a = __builtin_bit_cast(uint32_t, x), b = a;
  at_swap(a, b);
  lo = __builtin_bit_cast(float, a);
  hi = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float at_half_max(float x) {
  float lo, hi;
  at_both(x, lo, hi);
  return fmaxf(lo, hi);
}
__device__ __forceinline__ float at_half_sum(float x) {
  float lo, hi;
  at_both(x, lo, hi);
  return lo + hi;
}

// ------------------------------------------------------------------------------------------------- rows in LDS
template <typename T, int DC> struct at_row {
  static constexpr int ES = sizeof(T);
  static constexpr int DS = DC <= 32 ? 32 : DC <= 64 ? 64 : DC <= 128 ? 128 : 256;
  static constexpr int RB = DS * ES;    // bytes of a row
  static constexpr int CH = RB / 16;    // chunks of a row
  static constexpr int STEPS = DC * ES / 32;  // of a product along the row (two chunks each)
  static constexpr int PAD = CH >= 8 ? 32 : 0;
  static constexpr int at(int row) { return row * RB + row / 8 * PAD; }  // row: a multiple of 8
  static constexpr int tile(int rows) { return at(rows); }               // bytes, rows: a multiple of 32
};

template <int CH> __device__ __forceinline__ int at_swizzle(int row) {
  return CH >= 16 ? ((row & 3) << 2) | ((row >> 2) & 1) : CH == 8 ? ((row & 2) << 1) | ((row >> 2) & 1) : (row >> 2) & 1;
}
template <typename T, int DC> __device__ __forceinline__ uint32_t at_chunk(int row, int chunk) {
  using R = at_row<T, DC>;
  return (uint32_t)(row * R::RB + (row >> 3) * R::PAD + ((chunk ^ at_swizzle<R::CH>(row)) << 4));
}

typedef unsigned char __attribute__((address_space(3))) * at_lds;

// A lane's places in a tile.  The swizzle goes by the lowest three bits of the row's number and leaves some bits of the
// chunk's alone, so a few offsets, worked out once, reach everything with constant distances.
template <typename T, int DC> struct at_places {
  using R = at_row<T, DC>;
  static constexpr int NA = R::CH >= 16 ? 4 : R::CH == 8 ? 2 : 1;       // chunk bits 2 and 3 are mixed with the row's
  static constexpr int NX = sizeof(T) == 4 ? 4 : NA;
  uint32_t along[NA];   // row c, chunk 4 i + h
  uint32_t across[NX];  // 16-bit: the transposing read's row and chunk, columns 32 i ..; fp32: row 4 h + i, column c

  __device__ __forceinline__ void init(int lane) {
    const int c = lane & 31, h = lane >> 5;
#pragma unroll
    for (int i = 0; i < NA; ++i) along[i] = at_chunk<T, DC>(c, 4 * i + h);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < NX; ++i) across[i] = at_chunk<T, DC>(4 * h + i, c >> 2) + (c & 3) * 4;
    } else {
      const int i = lane & 15, g = lane >> 4;
#pragma unroll
      for (int x = 0; x < NX; ++x)
        across[x] = at_chunk<T, DC>(4 * (g >> 1) + (i >> 2), 4 * x + 2 * (g & 1) + ((i >> 1) & 1)) + (i & 1) * 8;
    }
  }
  // left operand of step st of a product along the rows: rows row .. row + 31 (a multiple of 32)
  __device__ __forceinline__ at_u4 rows(const unsigned char* tile, int row, int st) const {
    return *reinterpret_cast<const at_u4*>(tile + along[st / 2 % NA] + (R::at(row) + st % 2 * 32 + st / (2 * NA) * (NA * 64)));
  }
  // left operand of a product across the rows (16-bit types): the 16 rows from `row` (a multiple of 16), in the order of
  // a result's registers, columns 32 db .. 32 db + 31
  __device__ __forceinline__ at_u4 cols(const unsigned char* tile, int row, int db) const {
    typedef at_s4 __attribute__((address_space(3))) * lds_s4p;
    const unsigned char* p = tile + across[db % NX] + (R::at(row) + db / NX * (NX * 64));
    const at_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4p)p);
    const at_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4p)(p + R::at(8)));
    return __builtin_bit_cast(at_u4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  // the same in fp32: row 8 (i / 4) + 4 h + i % 4 behind `row`.  The column's chunk 8 db + (c >> 2): its bit 3 is mixed
  // too where a row has more than eight
  __device__ __forceinline__ float col(const unsigned char* tile, int row, int i, int db) const {
    constexpr int MIX = R::CH >= 16 ? 128 : 0;
    const uint32_t o = MIX && (db & 1) ? across[i % 4] ^ MIX : across[i % 4];
    return *reinterpret_cast<const float*>(tile + o + (R::at(row + 8 * (i / 4)) + (MIX ? db / 2 * 256 : db * 128)));
  }
};

// acc[db] += (32 rows of the tile from `row`)^T x, for all columns of the head: x is a result of 32 rows by 32 columns.
// In 16-bit types x (probabilities, or scores' gradients) is rounded to T, as the matrix instructions multiply nothing wider
// by T: of independent roundings a sum keeps about the relative error of one, so that with the result's own the outputs are
// 1.4 times as far from 64 bits as fp32 throughout (bf16: 0.0024 and 0.0017, fp16: 0.00030 and 0.00021), dq and dk up to 1.6
// times where their sums cancel.  A second product with what rounding takes brings dq and dk back to 1.0 and costs a training
// step of 2 x 2048 x 4096, 16/4 heads of 128, 15 % (629 -> 724 us on one card), 768 x 312 x 312, 4 heads of 64, 9 %.
template <typename T, int DC>
__device__ __forceinline__ void at_mma_cols(const at_places<T, DC>& at, const unsigned char* tile, int row, const at_f16& x,
                                            at_f16* acc) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      at_u4 p;
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = at_pack(T(), x[8 * b + 2 * j], x[8 * b + 2 * j + 1]);
#pragma unroll
      for (int db = 0; db < DC / 32; ++db) acc[db] = at_mma(T(), at.cols(tile, row + 16 * b, db), p, acc[db]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int db = 0; db < DC / 32; ++db)
        acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(at.col(tile, row, i, db), x[i], acc[db], 0, 0, 0);
  }
}

// Tiles are filled by loads that go straight to LDS: one instruction moves 1 KiB, lane l's 16 bytes land at 16 l, so
// the swizzle is applied to the addresses that the lanes fetch from.  Chunks behind the head's end and rows that do
// not take part are fetched from beyond the buffer's range, which gives zeros (so whatever those rows hold, NaN
// included, never meets a product).
// Behind the last query row it is that row, and its lse2, that the backward pass's tiles repeat, beside zeros for dO and
// delta: P is then the row's own, and adds P times zero.  (Zeros for the query would make P NaN at an infinite key.)
// (128 rows under 8 MiB apart: offsets and scalar offsets stay under 2^30, and AT_OUTSIDE outside without a wrap)
constexpr uint32_t AT_RANGE = 0x80010000u, AT_OUTSIDE = 0xc0000000u;

typedef int at_i4 __attribute__((ext_vector_type(4)));

// one load of 1 KiB (ONE: 256 bytes, four per lane) to LDS: base + off (AT_OUTSIDE or more: zeros) + soff.  (m0 is the
// compiler's for no longer than an instruction that it sets it for: it needs no saving.)
__device__ __forceinline__ at_i4 at_buffer(const void* base) {
  const uint64_t b = (uint64_t)base;
  return at_i4{__builtin_amdgcn_readfirstlane((int)b), __builtin_amdgcn_readfirstlane((int)(b >> 32) & 0xffff), (int)AT_RANGE,
               0x00020000};
}
template <bool ONE = false> __device__ __forceinline__ void at_load_lds(at_i4 rs, uint32_t off, uint32_t soff, uint32_t lds) {
  if constexpr (ONE)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, %3 offen lds"
                 :
                 : "v"(off), "s"(rs), "s"(lds), "s"(soff)
                 : "memory");
  else
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %3 offen lds"
                 :
                 : "v"(off), "s"(rs), "s"(lds), "s"(soff)
                 : "memory");
}

template <typename T, int DC, int ROWS, int WAVES> struct at_stage {
  using R = at_row<T, DC>;
  static constexpr int PER = 1024 / R::RB;                  // rows per instruction
  static constexpr int N = ROWS * R::RB / 1024 / WAVES;     // instructions per wave, STEP rows apart
  static constexpr int STEP = PER * WAVES;
  static constexpr int PD = STEP >= 8 ? 1 : 8 / STEP;       // instructions after which the swizzle repeats
  static_assert(R::PAD == 0 || 8 % PER == 0, "an instruction's rows have no pad between them");
  static_assert(R::RB <= 1024 && ROWS * R::RB % (1024 * WAVES) == 0 && N % PD == 0, "whole instructions for every wave");
  uint32_t off[PD];
  uint32_t ahead;  // bytes from one group of PD instructions to the next

  // D: elements of a head; stride: bytes between rows (under 8 MiB)
  __device__ __forceinline__ void init(int wave, int lane, int D, uint32_t stride) {
    ahead = PD * STEP * stride;
#pragma unroll
    for (int p = 0; p < PD; ++p) {
      const int r = p * STEP + wave * PER + lane / R::CH, chunk = (lane % R::CH) ^ at_swizzle<R::CH>(r);
      off[p] = chunk * 16 < D * R::ES ? (uint32_t)r * stride + (uint32_t)chunk * 16u : AT_OUTSIDE;
    }
  }
  // words[i], bit r: row 32 i + r takes part -> outside[p]: 0 where this lane's row of instruction p does, else AT_OUTSIDE
  static __device__ __forceinline__ void spread(const uint32_t (&words)[ROWS / 32], int wave, int lane, uint32_t (&outside)[N]) {
#pragma unroll
    for (int p = 0; p < N; ++p) {
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < ROWS / 32; ++i) w |= words[i] & (0u - (uint32_t)((p * STEP + wave * PER) >> 5 == i));
      outside[p] = (uint32_t)__builtin_amdgcn_sbfe((int)~w, (p * STEP + wave * PER + lane / R::CH) & 31, 1) & AT_OUTSIDE;
    }
  }
  // base: the tile's first row; in place of the rows behind `last`, that row again
  __device__ __forceinline__ void issue_repeat(const char* base, uint32_t lds, int wave, int lane, int last) const {
    const at_i4 rs = at_buffer(base);
    const uint32_t stride = ahead / (PD * STEP);
#pragma unroll
    for (int p = 0; p < N; ++p) {
      const int behind = max(p * STEP + wave * PER + lane / R::CH - last, 0);
      const uint32_t at = off[p % PD] + (uint32_t)(p / PD) * ahead - (uint32_t)behind * stride;
      at_load_lds(rs, off[p % PD] == AT_OUTSIDE ? AT_OUTSIDE : at, 0u,
                  __builtin_amdgcn_readfirstlane(lds + (uint32_t)((p * WAVES + wave) * 1024 + (((p * WAVES + wave) * PER) >> 3) * R::PAD)));
    }
  }
  // base: the tile's first row; FULL: every row takes part
  template <bool FULL> __device__ __forceinline__ void issue(const char* base, uint32_t lds, int wave, const uint32_t (&outside)[N]) const {
    const at_i4 rs = at_buffer(base);
#pragma unroll
    for (int p = 0; p < N; ++p)
      at_load_lds(rs, FULL ? off[p % PD] : off[p % PD] | outside[p], (p / PD) * ahead,
                  __builtin_amdgcn_readfirstlane(lds + (uint32_t)((p * WAVES + wave) * 1024 + (((p * WAVES + wave) * PER) >> 3) * R::PAD)));
  }
};

// instruction i of the loads of 32 rows from `base` (bit r of take: row r takes part; behind `last`, that row again)
template <typename T, int DC>
__device__ __forceinline__ void at_fetch_rows(const void* base, uint32_t stride, int D, uint32_t take, uint32_t lds, int i, int lane,
                                              int last = 31) {
  using R = at_row<T, DC>;
  constexpr int PER = 1024 / R::RB;
  const int r = i * PER + lane / R::CH, chunk = (lane % R::CH) ^ at_swizzle<R::CH>(r);
  const uint32_t off = chunk * 16 < D * R::ES && ((take >> r) & 1) ? (uint32_t)min(r, last) * stride + (uint32_t)chunk * 16u : AT_OUTSIDE;
  at_load_lds(at_buffer(base), off, 0u, __builtin_amdgcn_readfirstlane(lds + (uint32_t)(i * 1024 + ((i * PER) >> 3) * R::PAD)));
}

// The key and value tiles of a work item, in the order that it goes through them.
template <typename T, int DC, int KT, int WAVES> struct at_key_tiles {
  using S = at_stage<T, DC, KT, WAVES>;
  S k, v;
  const char *kp, *vp;
  int64_t kstep, vstep;
  int n, next_k, next_v, k_end;  // sequence, first keys of the tiles that are fetched next, end of the item's keys

  __device__ __forceinline__ void init(const at_args& a, const T* kb, const T* vb, int seq, int hk, int begin, int end,
                                       int wave, int lane) {
    n = seq;
    next_k = next_v = begin;
    k_end = end;
    kp = reinterpret_cast<const char*>(kb + (int64_t)n * a.ks[0] + (int64_t)hk * a.ks[2] + (int64_t)begin * a.ks[1]);
    vp = reinterpret_cast<const char*>(vb + (int64_t)n * a.vs[0] + (int64_t)hk * a.vs[2] + (int64_t)begin * a.vs[1]);
    kstep = a.ks[1] * (int64_t)(sizeof(T) * KT);
    vstep = a.vs[1] * (int64_t)(sizeof(T) * KT);
    k.init(wave, lane, a.D, (uint32_t)(a.ks[1] * sizeof(T)));
    v.init(wave, lane, a.D, (uint32_t)(a.vs[1] * sizeof(T)));
  }
  template <bool DO_K, bool DO_V>
  __device__ __forceinline__ void fetch(const at_args& a, uint32_t lds_k, uint32_t lds_v, int wave, int lane) {
    const int k0 = DO_K ? next_k : next_v;
    uint32_t outside[S::N];
    if (a.bits == nullptr && k_end - k0 >= KT) {
      if constexpr (DO_K) k.template issue<true>(kp, lds_k, wave, outside);
      if constexpr (DO_V) v.template issue<true>(vp, lds_v, wave, outside);
    } else {
      uint32_t words[KT / 32];
#pragma unroll
      for (int i = 0; i < KT / 32; ++i) words[i] = at_key_bits(a, n, k_end, k0 + 32 * i);
      S::spread(words, wave, lane, outside);
      if constexpr (DO_K) k.template issue<false>(kp, lds_k, wave, outside);
      if constexpr (DO_V) v.template issue<false>(vp, lds_v, wave, outside);
    }
    if constexpr (DO_K) {
      kp += kstep;
      next_k += KT;
    }
    if constexpr (DO_V) {
      vp += vstep;
      next_v += KT;
    }
  }
};

// every load of this wave has landed, its reads of LDS are done (the tile that they read may be filled next), and every
// wave has said so
__device__ __forceinline__ void at_landed() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void at_sync() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// up to 64 floats to LDS; behind the first `left`, zeros, or (REPEAT) the last of them
template <bool REPEAT = false> __device__ __forceinline__ void at_fetch_floats(const float* base, int left, uint32_t lds, int lane) {
  const uint32_t off = REPEAT ? (uint32_t)min(lane, left - 1) * 4u : lane < left ? (uint32_t)lane * 4u : AT_OUTSIDE;
  at_load_lds<true>(at_buffer(base), off, 0u, __builtin_amdgcn_readfirstlane(lds));
}

// Block id -> work item.  Ids go round the 8 XCDs; items that share keys stay on one XCD and its L2, and units of them
// are dealt out in turn, so that sequences of different lengths spread.  A unit is a sequence, whose heads share cache
// lines, or one key head of it where there are too few sequences to go round (dealing out heads of 64 bytes a token to
// eight XCDs costs 15 % at 640 sequences of 180; dealing out four sequences leaves half the card idle).  The items of
// the last units (fewer than 8) are divided evenly.
struct at_order {
  at_div subs;    // items of a unit
  int32_t units;
  __host__ at_order(int64_t N, int64_t Hk, int64_t items_of_head)
      : subs((uint32_t)(N >= 16 ? Hk * items_of_head : items_of_head)), units((int32_t)(N >= 16 ? N : N * Hk)) {}
  // units that are given
  __host__ at_order(int64_t units_, int64_t subs_) : subs((uint32_t)subs_), units((int32_t)units_) {}
  __host__ dim3 grid() const { return at_grid(8 * ((int64_t)(units / 8) * subs.d + ((int64_t)(units % 8) * subs.d + 7) / 8)); }
  // -1: none
  __device__ __forceinline__ int item() const {
    const uint32_t id = at_block();
    const int xcd = id & 7, pos = id >> 3, whole = (units >> 3) * (int)subs.d;
    if (pos < whole) {
      const int u = subs.of(pos);
      return (u * 8 + xcd) * (int)subs.d + pos - u * (int)subs.d;
    }
    const int rest = (units & 7) * (int)subs.d, per = (rest + 7) >> 3, i = xcd * per + pos - whole;
    return pos - whole < per && i < rest ? (units & ~7) * (int)subs.d + i : -1;
  }
};

// Writes a result (rows: elements 32 db .. of the head, column: this lane's row of memory at p) times f; REST: and what
// rounding took from it.  Without `keep`, zeros: where no key takes part, the sums may hold 0 times an infinity or NaN.
template <typename T, int DC, bool REST = false>
__device__ __forceinline__ void at_store_rows(T* p, bool live, bool keep, const at_f16* acc, float f, int D, int lane,
                                              T* rest = nullptr) {
  const int h = lane >> 5;
#pragma unroll
  for (int db = 0; db < DC / 32; ++db) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        // registers 8 b .. + 3 hold elements 4 h + 0..3 of 16, the next four 8 + 4 h + 0..3: the halves swap, and each
        // lane has eight in a row
        at_u4 w, r;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const at_f2 u = {acc[db][8 * b + 2 * j] * f, acc[db][8 * b + 2 * j + 1] * f};
          const at_f2 v = {acc[db][8 * b + 4 + 2 * j] * f, acc[db][8 * b + 5 + 2 * j] * f};
          uint32_t x = at_pack(T(), u[0], u[1]), y = at_pack(T(), v[0], v[1]);
          if constexpr (REST) {
            const at_f2 a = u - at_unpack(T(), x), c = v - at_unpack(T(), y);
            uint32_t ra = at_pack(T(), a[0], a[1]), rc = at_pack(T(), c[0], c[1]);
            at_swap(ra, rc);
            r[j] = keep ? ra : 0u;
            r[2 + j] = keep ? rc : 0u;
          }
          at_swap(x, y);
          w[j] = keep ? x : 0u;
          w[2 + j] = keep ? y : 0u;
        }
        const int d = 32 * db + 16 * b + 8 * h;
        if (live && d < D) {
          *reinterpret_cast<at_u4*>(p + d) = w;
          if constexpr (REST) *reinterpret_cast<at_u4*>(rest + d) = r;
        }
      }
    } else {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int d = 32 * db + 8 * b + 4 * h;
        at_f4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = keep ? acc[db][4 * b + j] * f : 0.0f;
        if (live && d < D) *reinterpret_cast<at_f4*>(p + d) = w;
      }
    }
  }
}

// Right operand of a product along rows: this lane's row, STEPS chunks.  base: the same for the whole wave; off: bytes to
// this lane's row, AT_OUTSIDE if it has none (zeros then).
struct at_rows_of {
  __amdgpu_buffer_rsrc_t rs;
  __device__ __forceinline__ explicit at_rows_of(const void* base) {
    const uint64_t b = (uint64_t)base;
    const uint64_t u = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32) |
                       (uint32_t)__builtin_amdgcn_readfirstlane((int)b);
    rs = __builtin_amdgcn_make_buffer_rsrc((void*)u, 0, (int)AT_RANGE, 0x00020000);
  }
  template <typename T> __device__ __forceinline__ at_u4 chunk(uint32_t off, int D, int st, int h) const {
    const uint32_t b = (uint32_t)(2 * st + h) * 16u;
    const uint32_t o = b < (uint32_t)D * (uint32_t)sizeof(T) ? off + b : AT_OUTSIDE;
    return __builtin_bit_cast(at_u4, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)o, 0, 0));
  }
  template <typename T, int DC> __device__ __forceinline__ void row(uint32_t off, int D, int lane, at_u4* f) const {
#pragma unroll
    for (int st = 0; st < at_row<T, DC>::STEPS; ++st) f[st] = chunk<T>(off, D, st, lane >> 5);
  }
};

// fp16 has no room for scores' gradients as they come (of a long row they lie below its smallest normal number, of a
// scaled loss beyond its largest).  Each lane's column has a power of two of its own, that of the running largest, and
// its sums are rescaled when a larger one comes along, like a softmax's.  (P is at most 1: 2^12 throughout.)
template <typename T> struct at_fit {
  static constexpr bool ON = sizeof(T) == 2 && __is_same(T, rc_half);
  float s = ON ? 0.0f : 1.0f;
  template <int NDB> __device__ __forceinline__ void fit(at_f16& x, at_f16* acc) {
    if constexpr (ON) {
      float mx = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(x[i]));
      mx = at_half_max(mx);
      const bool need = mx * s > 32768.0f || (s == 0.0f && mx > 0.0f);
      if (__any(need)) {
        const int e = max(__builtin_amdgcn_frexp_expf(mx), -110);
        const float to = need ? ldexpf(1.0f, 11 - e) : s;
        const float f = s == 0.0f ? 1.0f : to / s;
#pragma unroll
        for (int i = 0; i < NDB; ++i) acc[i] *= f;
        s = to;
      }
      x *= s;
    }
  }
  __device__ __forceinline__ float undo() const { return ON ? (s == 0.0f ? 1.0f : 1.0f / s) : 1.0f; }
};
template <typename T> constexpr float AT_P_LIFT = at_fit<T>::ON ? 12.0f : 0.0f;
