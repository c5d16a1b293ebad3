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
#include <type_traits>

#include "dmf_common.h"

namespace dmf {

struct AtScore {
  float scale_u;    // scale * U (AtUnit)
  float scale_cap;  // scale / cap
  float cap_u;      // cap * U
  float bend;       // -1 / cap_u^2
  float poly[6];    // cap * U * tanh(x) = raw * poly(raw^2) for |x| = |raw| scale / cap <= 1 (16-bit types)
  float half[4];    // the same for |x| <= 0.5
  float one_to, half_to;  // where they hold: 1 and 0.5, or less where a coefficient leaves f32's range (at_score_args)
};

struct AtArgs {
  const void *q, *k, *v;
  long long q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh;  // element strides: batch, token, head
  int batch, lq, lk, hq, hk, d, group;
  unsigned group_m;            // ceil(2^32 / group) (0 for 1): r / group = mulhi(r, group_m) while r * group < 2^32
  float scale, cap;            // cap 0: none
  AtScore sc;                  // the score's constants (at_score_args)
  const float* slopes;         // [hq], null: none
  int causal;
  const int* kv_lens;          // [batch], null: lk
  const int* prefix;           // [batch], null: 0
  const int2* spans;           // [batch][lq] (documents), null: from the fields above
  void* o;                     // [batch][lq][hq][d]
  void* o_lo;                  // what rounding o to 16 bits left over (training: the backward's row sums), null: none
  float* lse;                  // [batch][hq][lq]: log sum exp of s (log2 domain; natural for f32), null: none
  int chunk, splits;           // keys per split, splits (1: the whole row in one workgroup)
  float *po, *pml;             // partials [splits][batch * hk][rows][d], [..][4] (max, o's sum, sum)
  // backward
  const void* go;              // [batch][lq][hq][d]
  float* rowws;                // backward scratch: delta [batch][hq][lq], span lo [batch][lq], hi [batch][lq]
  void *dq, *dk, *dv;          // contiguous [batch][l][h][d]
  int rows_first;              // launch order: row workgroups before key workgroups
};

// forward launch: row waves and key groups per workgroup, keys per split, splits; 32-key tiles for three workgroups a CU
struct AtPlan {
  int nw, ng, chunk, splits;
  bool three;
};

constexpr float AT_LOG2E = 1.4426950408889634f;

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

// two floats rounded to a pair of 16-bit elements (one v_cvt_pk); sum of a pair's elements added to c (one v_dot2)
template <typename T> struct AtPair;
template <> struct AtPair<bf16_t> {
  typedef __attribute__((ext_vector_type(2))) __bf16 V;
  __device__ __forceinline__ static uint32_t pack(float l, float h) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((dmf_f2{l, h}), V));
  }
  __device__ __forceinline__ static float add(uint32_t w, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(V, w), V{(__bf16)1.f, (__bf16)1.f}, c, false);
  }
};
template <> struct AtPair<f16_t> {
  typedef __attribute__((ext_vector_type(2))) _Float16 V;
  __device__ __forceinline__ static uint32_t pack(float l, float h) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((dmf_f2{l, h}), V));
  }
  __device__ __forceinline__ static float add(uint32_t w, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(V, w), V{(_Float16)1.f, (_Float16)1.f}, c, false);
  }
};

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

// LDS-DMA of ROWS rows of a strided matrix into a tile, shared by NW waves. The lanes' byte offsets within a tile of rows
// are computed once; a tile then costs scalar work only: its first row's address and, as the buffer's range, the bytes up to
// row hi, past which rows arrive as zeros. The dims from d to DP get an offset past any range: zeros too. Needs a row stride
// of at least d elements, and ROWS rows within 2 GiB.
template <typename T, int DP, int ROWS, int NW>
struct AtLoad {
  static constexpr int NC = DP * AtT<T>::E / 16, PIECES = ROWS * NC / 64, PW = (PIECES + NW - 1) / NW;
  unsigned voff[PW];
  unsigned row_bytes;
  __device__ __forceinline__ AtLoad(long long sl, int d, int wid, int lane) : row_bytes((unsigned)sl * AtT<T>::E) {
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int pos = (wid * PW + i) * 64 + lane, row = pos / NC, ch = (pos % NC) ^ at_swz<T, DP>(row);
      voff[i] = ch * AtT<T>::CH < d ? row * row_bytes + ch * 16 : BUF_OOB;
    }
  }
  // rows r0 .. of base (row 0), valid below hi, to LDS address lds
  __device__ __forceinline__ void issue(const T* base, int r0, int hi, unsigned lds, int wid) const {
    const unsigned n = (unsigned)min(max(hi - r0, 0), ROWS);
    const unsigned long long at = (unsigned long long)base + (unsigned long long)(unsigned)r0 * row_bytes;
    // (wave-uniform by contract: readfirstlane keeps the descriptor in SGPRs where the compiler cannot prove it)
    const v4i_t rs = {__builtin_amdgcn_readfirstlane((int)at), __builtin_amdgcn_readfirstlane((int)(at >> 32)),
                      __builtin_amdgcn_readfirstlane((int)(n * row_bytes)), BUF_FLAGS};
#pragma unroll
    for (int i = 0; i < PW; ++i)
      if (PIECES % NW == 0 || wid * PW + i < PIECES) dma16(rs, voff[i], 0, lds + (wid * PW + i) * 1024);
  }
};

// one LDS-DMA wave-instruction of 4 B a lane: LDS [lds, lds + 256) (see dma16)
__device__ __forceinline__ void at_dma4(v4i_t rsrc, unsigned voff, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\tbuffer_load_dword %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "v"(voff), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(lds))
               : "memory");
}

// This lane's byte offsets into any tile of these dims: row operands (row lane & 31, step ks) and transposed operands
// (column block fd, see at_accumulate). The XOR depends only on the row modulo 16, so other rows, tiles and stages are
// constants added to these, which the LDS instructions take as immediates.
template <typename T, int DF>
struct AtOffsets {
  static constexpr int DP = AtPad<DF>::DP, KS = DF / (2 * AtT<T>::CH), FD = DF / 32;
  static constexpr int RB = DP * AtT<T>::E;
  int row[KS];
  int col[sizeof(T) == 2 ? 2 * FD : 1];
  __device__ __forceinline__ explicit AtOffsets(int lane) {
    const int h = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) row[ks] = at_off<T, DP>(lane & 31, 2 * ks + h);
    if constexpr (sizeof(T) == 2) {
      const int r = 4 * h + ((lane >> 2) & 3), ch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
      for (int fd = 0; fd < FD; ++fd) {
        col[2 * fd] = at_off<T, DP>(r, 4 * fd + ch) + 8 * (lane & 1);
        col[2 * fd + 1] = at_off<T, DP>(r + 8, 4 * fd + ch) + 8 * (lane & 1);
      }
    }
  }
};
// one row operand: 8 (16-bit) or 4 (f32) consecutive dims of row r0 + (lane & 31) (r0 a multiple of 16), step ks
template <typename T, int DF>
__device__ __forceinline__ uint4 at_row(const char* tile, const AtOffsets<T, DF>& o, int r0, int ks) {
  return *(const uint4*)(tile + r0 * AtOffsets<T, DF>::RB + o.row[ks]);
}

// A 32 x 32 result tile as the operand of the next product: 16-bit types rounded to pairs, f32 as it is
template <typename T> struct AtP {
  uint32_t w[8];
  __device__ __forceinline__ explicit AtP(const float* p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = AtPair<T>::pack(p[2 * i], p[2 * i + 1]);
  }
  // what rounding p to `r` left over, rounded in turn
  __device__ __forceinline__ AtP(const float* p, const AtP& r) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      w[i] = AtPair<T>::pack(p[2 * i] - B16<T>::lo(r.w[i]), p[2 * i + 1] - B16<T>::hi(r.w[i]));
  }
};
template <> struct AtP<float> {
  float w[16];
  __device__ __forceinline__ explicit AtP(const float* p) {
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = p[i];
  }
};

// acc[fd] += X^T P for the 32 tile rows r0 .. r0 + 31: X's column block fd (32 dims) as the row operand, read transposed
// from its tile. TWO: P is p + rest.
template <typename T, int DF, bool TWO = false>
__device__ __forceinline__ void at_accumulate(const char* tile, const AtOffsets<T, DF>& o, int r0, const AtP<T>& p,
                                              at_f32x16* acc, int lane, const AtP<T>* rest = nullptr) {
  constexpr int DP = AtPad<DF>::DP, RB = AtOffsets<T, DF>::RB;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint4 b = make_uint4(p.w[4 * c], p.w[4 * c + 1], p.w[4 * c + 2], p.w[4 * c + 3]);
      const char* t = tile + (r0 + 16 * c) * RB;
#pragma unroll
      for (int fd = 0; fd < DF / 32; ++fd) {
        const uint2 l = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_v4s*)(t + o.col[2 * fd])));
        const uint2 g =
            __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_v4s*)(t + o.col[2 * fd + 1])));
        acc[fd] = at_mfma<T>(make_uint4(l.x, l.y, g.x, g.y), b, acc[fd]);
        if constexpr (TWO)
          acc[fd] = at_mfma<T>(make_uint4(l.x, l.y, g.x, g.y),
                               make_uint4(rest->w[4 * c], rest->w[4 * c + 1], rest->w[4 * c + 2], rest->w[4 * c + 3]),
                               acc[fd]);
      }
    }
  } else {
    const int h = lane >> 5;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = r0 + 8 * (i >> 2) + 4 * h + (i & 3);
#pragma unroll
      for (int fd = 0; fd < DF / 32; ++fd) {
        const int e = 32 * fd + (lane & 31);
        const float x = *(const float*)(tile + at_off<T, DP>(row, e >> 2) + 4 * (e & 3));
        acc[fd] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p.w[i], acc[fd], 0, 0, 0);
      }
    }
  }
}

// What a mask hides. A masked pair has weight 0 exactly, but 0 * NaN is NaN: in a tile that some row sees in part, an element
// of X that is not finite reaches the columns that may not see its row. Where accumulators end up non-finite under a mask, a
// workgroup therefore walks its tiles once more, and takes at_accumulate_seen in such tiles with such an element (at_has_nonfinite):
// the same sum row by row on the vector ALU, over the pairs that sees(row) lets through. Columns that are NaN in every dim by
// what they see (a score of NaN, a delta of NaN) ask for no second walk. Finite inputs cost nothing but the check at the end. 4096 causal tokens, 16 heads of 128, bf16, forward and backward: 138 + 259 us; with one key of NaN that all see, or with
// every operand NaN, the same; with all values NaN 603 + 854, with all output gradients infinite 133 + 2254 (each diagonal tile pair
// by pair).
template <typename T, int DF>
__device__ __forceinline__ bool at_has_nonfinite(const char* tile, int r0, int lane) {
  constexpr int RB = AtOffsets<T, DF>::RB;
  const uint4* p = (const uint4*)(tile + r0 * RB) + lane;
  uint32_t most = 0, most2 = 0;  // of the magnitudes' bits: those of infinities and NaN are the largest
#pragma unroll
  for (int i = 0; i < 32 * RB / 1024; ++i) {
    const uint4 u = p[64 * i];
    for (uint32_t w : {u.x, u.y, u.z, u.w}) {
      if constexpr (sizeof(T) == 4) {
        most = max(most, w & 0x7fffffffu);
      } else {
        most = max(most, w & 0x7fffffffu);
        most2 = max(most2, (w & 0x7fffu) << 16);
      }
    }
  }
  constexpr uint32_t INF = sizeof(T) == 4 ? 0x7f800000u : __is_same(T, f16_t) ? 0x7c000000u : 0x7f800000u;
  return __any(max(most, most2) >= INF);
}
template <typename T, int DF, typename F>
__device__ __forceinline__ void at_accumulate_seen(const char* tile, int r0, const float* p, at_f32x16* acc, int lane,
                                                   F&& sees) {
  constexpr int DP = AtPad<DF>::DP, E = AtT<T>::E, CH = AtT<T>::CH;
  const int h = lane >> 5;
#pragma unroll 1
  for (int r = 0; r < 32; ++r) {  // its weight is in register 4 (r >> 3) + (r & 3) of half (r >> 2) & 1
    const int n = 4 * (r >> 3) + (r & 3);
    float w = p[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) w = n == i ? p[i] : w;
    w = __shfl(w, (lane & 31) + 32 * ((r >> 2) & 1), 64);
    const bool on = sees(r);
#pragma unroll
    for (int f = 0; f < DF / 32; ++f)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int e = 32 * f + 8 * g + 4 * h;
        const T* x = (const T*)(tile + at_off<T, DP>(r0 + r, e / CH) + e % CH * E);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[f][4 * g + i] = on ? fmaf(w, ld(x + i), acc[f][4 * g + i]) : acc[f][4 * g + i];
      }
  }
}

// ------------------------------------------------------------------- spans
struct AtSpan {
  int lo, hi;  // hi <= lo: nothing
  int at;      // the query's position
};
__device__ __forceinline__ int at_keys(const AtArgs& a, int b) {
  return a.kv_lens ? min(max(a.kv_lens[b], 0), a.lk) : a.lk;
}
__device__ __forceinline__ AtSpan at_span(const AtArgs& a, int b, int i) {
  const int n = at_keys(a, b);
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

// packed row r of key head kh: query qi, query head
struct AtRow {
  int qi, head;
};
__device__ __forceinline__ AtRow at_packed(const AtArgs& a, int kh, int r) {
  AtRow x;
  x.qi = a.group_m ? (int)__umulhi((unsigned)r, a.group_m) : r;
  x.head = kh * a.group + r - x.qi * a.group;
  return x;
}

// Union and intersection of the spans of packed rows r0 .. r0 + 31 that see anything, one lane pair per row (`sp`; dead
// rows excluded), uniform over the wave. Spans by position only widen with the row, so the first and last row tell; document
// spans are reduced over the lanes.
struct AtBounds {
  int lo, hi;      // union; hi 0: nothing
  int i_lo, i_hi;  // intersection (by position: or less of it)
};
__device__ __forceinline__ int at_wave_min(int v);
__device__ __forceinline__ int at_wave_max(int v);
__device__ __forceinline__ AtBounds at_bounds(const AtArgs& a, int b, int kh, int r0, int rows, const AtSpan& sp) {
  AtBounds w;
  if (a.spans) {
    const bool live = sp.hi > sp.lo;
    w.lo = at_wave_min(live ? sp.lo : 0x7fffffff), w.hi = at_wave_max(live ? sp.hi : 0);
    w.i_lo = at_wave_max(live ? sp.lo : 0), w.i_hi = at_wave_min(live ? sp.hi : 0x7fffffff);
  } else if (r0 >= rows) {
    w.lo = w.hi = w.i_lo = 0;
    w.i_hi = 0x7fffffff;
  } else {
    const AtSpan first = at_span(a, b, at_packed(a, kh, r0).qi), last = at_span(a, b, at_packed(a, kh, min(r0 + 31, rows - 1)).qi);
    w.lo = w.i_lo = 0;
    w.hi = __builtin_amdgcn_readfirstlane(last.hi);
    w.i_hi = __builtin_amdgcn_readfirstlane(max(first.hi, 1));  // (rows that see nothing come first, then 1, 2, .. keys)
  }
  return w;
}

// wave-wide minimum / maximum of an int
__device__ __forceinline__ int at_wave_min(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int at_wave_max(int v) { return -at_wave_min(-v); }

// columns (lane & 31) for which either half wave's lane says yes
__device__ __forceinline__ unsigned at_columns(bool yes) {
  const unsigned long long m = __ballot(yes);
  return (unsigned)m | (unsigned)(m >> 32);
}
// columns with an accumulator that is not finite
template <int FD>
__device__ __forceinline__ unsigned at_bad_columns(const at_f32x16* acc) {
  float bad = 0.f;
#pragma unroll
  for (int f = 0; f < FD; ++f)
#pragma unroll
    for (int i = 0; i < 16; ++i) bad = fmaf(acc[f][i], 0.f, bad);
  return at_columns(bad != bad);
}
// does any wave of the workgroup say yes? `flag` (LDS) is 0 from before the tiles' barriers on; every wave is done with its tiles
// after this
__device__ __forceinline__ bool at_vote(bool yes, int* flag) {
  if (yes) *flag = 1;
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*flag);
}

// ------------------------------------------------------------------ scores
// The exponent's unit U is the log2 domain for 16-bit types (v_exp_f32 is 2^x: one multiply saved per score) and the
// natural one for f32, where scaling s before the maximum is subtracted would round it at |s| log2 e.
template <typename T> struct AtUnit { static constexpr float U = sizeof(T) == 4 ? 1.f : AT_LOG2E; };
template <typename T>
__device__ __forceinline__ float at_exp(float x) {
  return __builtin_amdgcn_exp2f(sizeof(T) == 4 ? x * AT_LOG2E : x);
}
template <typename T>
__device__ __forceinline__ float at_log(float x) {
  if constexpr (sizeof(T) == 4)
    return logf(x);
  else
    return __builtin_amdgcn_logf(x);  // log2
}

// f16 probabilities below 2^-14 would be subnormal as operands and those of a long flat tail beside one dominant key vanish, so
// they are multiplied by 2^LIFT: in the forward p <= 2^8 (the maximum's lag) becomes at most 2^15, through the exponent; in the
// backward p <= 1 does. What is left is 2^-32 (2^-40) a key. bf16 has f32's exponents.
template <typename T> struct AtLift { static constexpr float FWD = __is_same(T, f16_t) ? 7.f : 0.f, BWD = __is_same(T, f16_t) ? 32768.f : 1.f; };

// CAP. The scores are bound by the vector ALU, and there by v_exp / v_rcp (a quarter of the rate): tanh as
// 1 - 2 / (exp(2 x) + 1) takes two of them and four more operations. While no score of a tile exceeds the cap
// (|x| <= 1, checked per wave and tile with half an operation a score), tanh(x) / x is a polynomial of degree 5 in x^2
// instead: minimax, off by 4.6e-7 at most (6.1e-7 of tanh), no transcendental, and its coefficients carry scale and cap; within
// half the cap (|x| <= 0.5, where trained scores mostly are) degree 3 does, off by 2.5e-7 (5.4e-7). Every form of the score is off
// by less than 10 * 2^-24 * cap (6.0e-7 cap), below the 16-bit rounding of the probabilities while the cap is below a few thousand;
// f32 calls tanhf, since that would be several f32 units of the exponent. The form is a wave's choice for a tile, so a score's
// last bits within that error depend on what else the tile holds.
// A coefficient of x^(2 i + 1) carries cap (scale / cap)^(2 i + 1): under a large cap the last ones fall below f32's normal
// numbers (the eleventh power from cap = 250 at scale 0.088), under a tiny one they pass its largest. The degree-5 form is then
// left out, and the degree-3 one taken up to the x at which the terms that are left out reach 2^-24 of the first.
template <typename T>
inline void at_score_args(AtArgs& a) {
  static const double C[6] = {0.9999994039535522,    -0.3332904279232025,  0.13281433284282684,
                              -0.051605671644210815, 0.016743114218115807, -0.0030670599082022196};
  static const double H[4] = {0.9999994557707791, -0.3332631793480118, 0.131902965910994, -0.0444022258055833};
  a.sc.scale_u = a.scale * AtUnit<T>::U;
  a.sc.scale_cap = a.cap > 0.f ? a.scale / a.cap : 0.f;
  a.sc.cap_u = a.cap * AtUnit<T>::U;
  a.sc.bend = a.cap > 0.f ? -1.f / (a.sc.cap_u * a.sc.cap_u) : 0.f;
  double x = a.sc.scale_cap;
  for (int i = 0; i < 6; ++i) {
    a.sc.poly[i] = (float)(C[i] * a.sc.cap_u * x);
    if (i < 4) a.sc.half[i] = (float)(H[i] * a.sc.cap_u * x);
    x *= (double)a.sc.scale_cap * a.sc.scale_cap;
  }
  auto normal = [](float c) { return fabsf(c) >= 1.17549435e-38f && fabsf(c) < INFINITY; };
  a.sc.one_to = 1.f;
  for (float c : a.sc.poly)
    if (!normal(c)) a.sc.one_to = -1.f;
  // |H[i]| x^(2 i) = 2^-24 for i = 1, 2, 3
  static const float TO[4] = {-1.f, 4.2e-4f, 0.0259f, 0.105f};
  a.sc.half_to = 0.5f;
  for (int i = 3; i >= 0; --i) {
    if (normal(a.sc.half[i])) continue;
    a.sc.half_to = a.sc.scale_cap < 1.f ? TO[i] : -1.f;
    for (int k = i; k < 4; ++k) a.sc.half[k] = 0.f;
  }
}
template <typename T>
__device__ __forceinline__ float at_slope(const AtArgs& a, int head) {
  return a.slopes ? a.slopes[head] * AtUnit<T>::U : 0.f;
}
// cap tanh(z / cap), or z, in units U, of the raw product; FORM: what is known of |x| = |raw| scale / cap
enum { AT_ANY = 0, AT_ONE = 1, AT_HALF = 2 };
template <int FORM>
__device__ __forceinline__ float at_poly(const AtScore& c, float t) {  // of t = raw^2
  if constexpr (FORM == AT_HALF) return fmaf(fmaf(fmaf(c.half[3], t, c.half[2]), t, c.half[1]), t, c.half[0]);
  float p = fmaf(c.poly[5], t, c.poly[4]);
  p = fmaf(p, t, c.poly[3]);
  p = fmaf(p, t, c.poly[2]);
  p = fmaf(p, t, c.poly[1]);
  return fmaf(p, t, c.poly[0]);
}
template <typename T, bool CAP, int FORM>
__device__ __forceinline__ float at_bent(const AtScore& c, float raw) {
  if constexpr (!CAP) {
    return raw * c.scale_u;
  } else if constexpr (sizeof(T) == 4) {
    return c.cap_u * tanhf(raw * c.scale_cap);
  } else if constexpr (FORM != AT_ANY) {
    return raw * at_poly<FORM>(c, raw * raw);
  } else {
    const float e = __builtin_amdgcn_exp2f(raw * (c.scale_cap * (2.f * AT_LOG2E))) + 1.f;
    return fmaf(-2.f * c.cap_u, __builtin_amdgcn_rcpf(e), c.cap_u);
  }
}
// calls f with a (wave-uniform) form as a constant; the form that the wave's largest |x| allows (a NaN among them: it is NaN in
// every form)
template <typename F>
__device__ __forceinline__ void at_by_form(int form, F&& f) {
  if (form == AT_HALF)
    f(std::integral_constant<int, AT_HALF>{});
  else if (form == AT_ONE)
    f(std::integral_constant<int, AT_ONE>{});
  else
    f(std::integral_constant<int, AT_ANY>{});
}
__device__ __forceinline__ int at_form(const AtScore& c, float x) {
  return !__any(!(x <= c.half_to)) ? AT_HALF : !__any(!(x <= c.one_to)) ? AT_ONE : AT_ANY;
}
// raw products of N result tiles -> cap tanh(z / cap) or z in units U, in place, by the form that the whole wave's tile
// allows
template <typename T, bool CAP, int N>
__device__ __forceinline__ void at_bend_tiles(const AtScore& c, at_f32x16* s) {
  auto all = [&](auto form) {
#pragma unroll
    for (int f = 0; f < N; ++f)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[f][i] = at_bent<T, CAP, form.value>(c, s[f][i]);
  };
  if constexpr (CAP && sizeof(T) == 2) {
    float big = 0.f;
#pragma unroll
    for (int f = 0; f < N; ++f)
#pragma unroll
      for (int i = 0; i < 16; ++i) big = fmaxf(big, fabsf(s[f][i]));
    at_by_form(at_form(c, big * c.scale_cap), all);
  } else {
    all(std::integral_constant<int, AT_ANY>{});
  }
}
}  // namespace dmf
