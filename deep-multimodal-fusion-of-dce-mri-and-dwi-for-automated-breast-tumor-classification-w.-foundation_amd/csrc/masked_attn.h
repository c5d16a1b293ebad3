// Shared pieces of the masked attention kernels (masked_attn_fwd.h, masked_attn_bwd.h; entry points in
// masked_attn.hip). For one (batch row, query head), over keys j of query i at position a = kv_len - Lq + i:
//
//   z = scale q.k,  s = cap tanh(z / cap) - slope |a - j|,  p = softmax of s over lo_i <= j < hi_i,  o = p v
//
// Every mask is one span [lo, hi) per query (AtSpan): key lengths, causal, a prefix that all queries see, and
// documents packed into a row. A query whose span is empty has o = 0 and no gradient.
//
// Rows: query heads that share a key head are packed into one list, row r = i * group + g, so that the tiles of a
// group read K and V once, and dK / dV sum over the group inside the accumulators.
//
// Matrix layout (32x32 tiles; v_mfma_f32_32x32x16 for 16-bit types, 32x32x2 for f32): an operand lane holds row
// (lane & 31) and, per step, 8 (16-bit) or 1 (f32) elements of the contracted index chosen by lane >> 5; the result lane
// holds column (lane & 31), rows 8 b + 4 (lane >> 5) + r in register 4 b + r. A score tile is computed with the keys (or
// in dK / dV the queries) as rows, so that its registers already are the operand of the next product: the
// contracted index may be taken in any order as long as both operands agree, and the other operand, read transposed
// from LDS (ds_read_b64_tr_b16), takes the order 4 h + {0..3}, 8 + 4 h + {0..3} that the registers have. No shuffle and
// no LDS round trip moves the probabilities.
#pragma once
#include "dmf_common.h"

namespace dmf {

struct AtArgs {
  const void *q, *k, *v;
  long long q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh;  // element strides: batch, token, head
  int batch, lq, lk, hq, hk, d, group;
  float scale, cap;            // cap 0: none
  const float* slopes;         // [hq], null: none
  int causal;
  const int* kv_lens;          // [batch], null: lk
  const int* prefix;           // [batch], null: 0
  const int2* spans;           // [batch][lq] (documents), null: from the fields above
  void* o;                     // [batch][lq][hq][d]
  void* o_lo;                  // what rounding o to 16 bits left over (training: the backward's row sums), null: none
  float* lse;                  // [batch][hk][lq * group]: log sum exp of s (log2 domain; natural for f32), null: none
  int chunk, splits;           // keys per split, splits (1: the whole row in one workgroup)
  float *po, *pml;             // partials [splits][batch * hk][rows][d], [..][2] (max, sum)
  // backward
  const void* go;              // [batch][lq][hq][d]
  float* delta;                // [batch][hk][rows]
  void *dq, *dk, *dv;          // contiguous [batch][l][h][d]
};

constexpr float AT_LOG2E = 1.4426950408889634f;
constexpr unsigned AT_RECORDS = 0x7ffffff0u;  // buffer range: offsets within a tile stay below, BUF_OOB is past it

template <typename T> struct AtT { static constexpr int E = sizeof(T), CH = 16 / E; };

typedef __attribute__((ext_vector_type(16))) float at_f32x16;
typedef short at_v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) at_v4s at_lds_v4s;

template <typename T>
__device__ __forceinline__ at_f32x16 at_mfma(const uint4& a, const uint4& b, at_f32x16 c) {
  if constexpr (__is_same(T, f16_t))
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(dmf_h16x8, a), __builtin_bit_cast(dmf_h16x8, b), c,
                                                  0, 0, 0);
  else if constexpr (__is_same(T, bf16_t)) {
    typedef __attribute__((ext_vector_type(8))) __bf16 b8;
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  } else {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  }
}
__device__ __forceinline__ at_f32x16 at_zero() {
  return at_f32x16{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
}

// value of the other half wave's lane (lane ^ 32) combined with this one's
__device__ __forceinline__ float at_half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float at_half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---------------------------------------------------------------- LDS tiles
// A tile is rows of DP elements (DP = 32, 64 or 128, the head dim padded with zeros), each row's 16-B chunks XORed by
// at_swz(row): 16 consecutive rows at one chunk, and 4 consecutive rows at 4 consecutive chunks (the transposed reads),
// fall into distinct banks.
template <int DF> struct AtPad { static constexpr int DP = DF <= 32 ? 32 : DF <= 64 ? 64 : 128; };

template <typename T, int DP>
__device__ __forceinline__ int at_swz(int row) {
  constexpr int NC = DP * AtT<T>::E / 16;
  if constexpr (sizeof(T) == 4)
    return NC >= 16 ? ((row & 3) | ((row >> 3) & 1) << 2 | ((row >> 2) & 1) << 3) : ((row >> 1) & 7);
  else if constexpr (NC == 16)
    return ((row & 3) << 2) | ((row >> 2) & 3);
  else if constexpr (NC == 8)
    return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  else
    return (row >> 2) & 3;
}
template <typename T, int DP>
__device__ __forceinline__ int at_off(int row, int ch) {
  return row * (DP * AtT<T>::E) + ((ch ^ at_swz<T, DP>(row)) << 4);
}

// LDS-DMA of rows r0 .. r0 + ROWS - 1 of a strided matrix into a tile; rows outside [lo, hi) and the dims from d to DP
// arrive as zeros from the buffer range check. `base` is row 0, sl the row stride in elements; all but the lane is
// wave-uniform. NW waves share the work.
template <typename T, int DP, int ROWS, int NW>
__device__ __forceinline__ void at_load_rows(const T* base, long long sl, int r0, int lo, int hi, int d, unsigned lds,
                                             int wid, int lane) {
  constexpr int NC = DP * AtT<T>::E / 16, PIECES = ROWS * NC / 64;
  static_assert(PIECES % NW == 0, "pieces per wave");
  const v4i_t rs = buf_rsrc(base + (long long)r0 * sl, AT_RECORDS);
#pragma unroll
  for (int i = 0; i < PIECES / NW; ++i) {
    const int p = wid * (PIECES / NW) + i, pos = p * 64 + lane, row = pos / NC;
    const int ch = (pos % NC) ^ at_swz<T, DP>(row);
    const bool ok = r0 + row >= lo && r0 + row < hi && ch * AtT<T>::CH < d;
    dma16(rs, ok ? (unsigned)(row * (int)sl * AtT<T>::E + ch * 16) : BUF_OOB, 0, lds + p * 1024);
  }
}
// Bytes one wave's vmcnt counts per at_load_rows call are PIECES / NW instructions.

// one row operand: 8 (16-bit) or 4 (f32) consecutive dims of `row`, step ks (the steps cover DF dims)
template <typename T, int DF>
struct AtSteps { static constexpr int N = DF / (2 * AtT<T>::CH); };  // row-operand steps over the head dim
template <typename T, int DP>
__device__ __forceinline__ uint4 at_row(const char* tile, int row, int ks, int h) {
  return *(const uint4*)(tile + at_off<T, DP>(row, 2 * ks + h));
}

// acc[fd] += X^T P for the 32 tile rows r0 .. r0 + 31: X's column block fd (32 dims) as the row operand, read transposed
// from its tile; P (32 rows x 32 columns) as a result tile whose registers are p[0..15]
template <typename T, int DF>
__device__ __forceinline__ void at_accumulate(const char* tile, int r0, const float* p, at_f32x16* acc, int lane) {
  constexpr int DP = AtPad<DF>::DP;
  const int h = lane >> 5;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint4 b = make_uint4(B16<T>::pack(p[8 * c], p[8 * c + 1]), B16<T>::pack(p[8 * c + 2], p[8 * c + 3]),
                                 B16<T>::pack(p[8 * c + 4], p[8 * c + 5]), B16<T>::pack(p[8 * c + 6], p[8 * c + 7]));
      const int row = r0 + 16 * c + 4 * h + ((lane >> 2) & 3);
      const int ch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
      for (int fd = 0; fd < DF / 32; ++fd) {
        const at_v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (at_lds_v4s*)(tile + at_off<T, DP>(row, 4 * fd + ch) + 8 * (lane & 1)));
        const at_v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (at_lds_v4s*)(tile + at_off<T, DP>(row + 8, 4 * fd + ch) + 8 * (lane & 1)));
        const uint2 l = __builtin_bit_cast(uint2, lo), g = __builtin_bit_cast(uint2, hi);
        acc[fd] = at_mfma<T>(make_uint4(l.x, l.y, g.x, g.y), b, acc[fd]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = r0 + 8 * (i >> 2) + 4 * h + (i & 3);
#pragma unroll
      for (int fd = 0; fd < DF / 32; ++fd) {
        const int e = 32 * fd + (lane & 31);
        const float x = *(const float*)(tile + at_off<T, DP>(row, e >> 2) + 4 * (e & 3));
        acc[fd] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p[i], acc[fd], 0, 0, 0);
      }
    }
  }
}

// ------------------------------------------------------------------- spans
struct AtSpan {
  int lo, hi;  // hi <= lo: nothing
  int at;      // the query's position
};
__device__ __forceinline__ AtSpan at_span(const AtArgs& a, int b, int i) {
  const int n = a.kv_lens ? min(max(a.kv_lens[b], 0), a.lk) : a.lk;
  AtSpan s;
  s.at = n - a.lq + i;
  if (a.spans) {
    const int2 v = a.spans[(long long)b * a.lq + i];
    s.lo = v.x;
    s.hi = v.y;
  } else {
    s.lo = 0;
    s.hi = a.causal ? min(n, max(s.at + 1, a.prefix ? a.prefix[b] : 0)) : n;
  }
  if (s.hi <= s.lo) s.lo = s.hi = 0;
  return s;
}

// wave-wide minimum / maximum of an int
__device__ __forceinline__ int at_wave_min(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int at_wave_max(int v) { return -at_wave_min(-v); }

// ------------------------------------------------------------------ scores
// CAP: tanh(x) = 1 - 2 / (exp(2 x) + 1): one v_exp, one v_rcp (absolute error ~1e-7, below the 16-bit rounding of the
// probabilities); f32 calls tanhf, since cap * 1e-7 would be several f32 units of the exponent.
template <typename T>
__device__ __forceinline__ float at_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
template <typename T>
__device__ __forceinline__ float at_tanh(float x) {  // of x = z / cap
  if constexpr (sizeof(T) == 4)
    return tanhf(x);
  else
    return fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * (2.f * AT_LOG2E)) + 1.f), 1.f);
}
// The exponent's unit is the log2 domain for 16-bit types (v_exp_f32 is 2^x: one multiply saved per score) and the
// natural one for f32, where scaling s before the maximum is subtracted would round it at |s| log2 e.
template <typename T> struct AtUnit { static constexpr float U = sizeof(T) == 4 ? 1.f : AT_LOG2E; };
template <typename T>
__device__ __forceinline__ float at_exp(float x) {
  if constexpr (sizeof(T) == 4)
    return __builtin_amdgcn_exp2f(x * AT_LOG2E);
  else
    return __builtin_amdgcn_exp2f(x);
}
template <typename T>
__device__ __forceinline__ float at_log(float x) {
  if constexpr (sizeof(T) == 4)
    return logf(x);
  else
    return __builtin_amdgcn_logf(x);  // log2
}
struct AtScore {
  float scale_u;      // scale * U
  float scale_cap;    // scale / cap
  float cap_u;        // cap * U
  float slope_u;      // slope * U (this lane's head)
};
template <typename T>
__device__ __forceinline__ AtScore at_score_of(const AtArgs& a, int head) {
  AtScore s;
  s.scale_u = a.scale * AtUnit<T>::U;
  s.scale_cap = a.cap > 0.f ? a.scale / a.cap : 0.f;
  s.cap_u = a.cap * AtUnit<T>::U;
  s.slope_u = a.slopes ? a.slopes[head] * AtUnit<T>::U : 0.f;
  return s;
}
// s (in units U) of the raw product; dist = |a - j|
template <typename T, bool CAP, bool SLOPE>
__device__ __forceinline__ float at_score(const AtScore& c, float raw, float dist) {
  float s;
  if constexpr (CAP)
    s = c.cap_u * at_tanh<T>(raw * c.scale_cap);
  else
    s = raw * c.scale_u;
  if constexpr (SLOPE) s = fmaf(-c.slope_u, dist, s);
  return s;
}

}  // namespace dmf
