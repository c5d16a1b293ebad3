// Masked attention backward (see masked_attn.h for the mathematics and the layouts).
//
//   delta_i = sum_d do_i o_i          (k_mattn_rows; o with the part its 16-bit rounding left over, so that rounding does
//                                      not enter dS through the whole row)
//   p_ij = exp(s_ij - lse_i),  dp_ij = do_i . v_j,  ds_ij = p_ij (dp_ij - delta_i) (1 - tanh^2(z_ij / cap))
//   dv_j = sum_i p_ij do_i,  dk_j = scale sum_i ds_ij q_i,  dq_i = scale sum_j ds_ij k_j
//
// One launch holds two kinds of workgroups: those of 128 (or 64) keys, which walk the queries that see them and keep dK and
// dV in registers, and those of 256 (or 128) packed rows, which walk their keys and keep dQ. The key workgroups' longest
// walk (all queries of all heads of a group) decides how evenly a launch ends: where that weighs, groups of waves take a
// workgroup's query tiles in turn and add up at the end (mattn_bwd_df). The scores are computed in
// both (7 products for the 5 that one pass with dQ in atomics would take): no atomics, so the same bits every run, no
// f32 dQ in HBM, and the sum over a group's query heads happens inside the dK / dV accumulators.
//
// Bound: no unit is full; a step of 32 x 32 has 32 matrix instructions, about 250 vector ones and 24 + 32 LDS reads one after the
// other, and two waves a SIMD overlap them in part (busy, 32 x 576: matrix pipe 0.32, vector ALU 0.46, LDS 0.21; 8192 tokens in
// documents: 0.35, 0.31, 0.25). 8192 tokens, 32 heads over 8 of 128, bf16: 3.46 to 3.52 ms, 1.09 to 1.11 PFLOP/s of the 7 products;
// 32 x 576, 4 heads, capped: 127 to 134 us (0.58), of which a third is the workgroups' start and end.
#pragma once
#include "masked_attn.h"
#include "masked_attn_fwd.h"

namespace dmf {

// What the backward needs of each row beside lse (a.rowws): -delta, and the query's span. One lane group of 16 per row. HBM:
// o, its rest and do are read once (32 x 576 tokens, 4 heads of 128: 12 us, 4.7 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) k_mattn_rows(AtArgs a) {
  const long long g = ((long long)blockIdx.x * 256 + threadIdx.x) >> 4;  // (b, query, head)
  const int l16 = threadIdx.x & 15;
  const long long n = (long long)a.batch * a.lq * a.hq;
  if (g >= n) return;  // (whole groups leave: the shuffles below stay within 16 lanes)
  const T* go = (const T*)a.go + g * a.d;
  const T* o = (const T*)a.o + g * a.d;
  const T* lo = a.o_lo ? (const T*)a.o_lo + g * a.d : nullptr;
  float t = 0.f;
  for (int e = 8 * l16; e < a.d; e += 128) {
    float x[8], y[8], z[8];
    ld8(go + e, x);
    ld8(o + e, y);
    if (lo) {
      ld8(lo + e, z);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] += z[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) t = fmaf(x[i], y[i], t);
  }
#pragma unroll
  for (int k = 1; k < 16; k <<= 1) t += __shfl_xor(t, k, 64);
  if (l16 == 0) {
    const int head = (int)(g % a.hq);
    const long long bq = g / a.hq;
    const int qi = (int)(bq % a.lq), b = (int)(bq / a.lq);
    a.rowws[((long long)b * a.hq + head) * a.lq + qi] = -t;
    if (head == 0) {
      const AtSpan sp = at_span(a, b, qi);
      ((int*)a.rowws)[n + bq] = sp.lo;
      ((int*)a.rowws)[n + (long long)a.batch * a.lq + bq] = sp.hi;
    }
  }
}

// p and ds of one score s = cap tanh(z / cap) (units U); dist = |a - j|; dpd = dp - delta
template <typename T, bool CAP, bool SLOPE>
__device__ __forceinline__ void at_grad(const AtArgs& a, float slope_u, float s, float dist, float lse, float dpd,
                                        float& p, float& ds) {
  float e = s - lse;
  if constexpr (SLOPE) e = fmaf(-slope_u, dist, s) - lse;
  p = at_exp<T>(e);
  ds = p * dpd;
  if constexpr (CAP) ds *= fmaf(s * s, a.sc.bend, 1.f);  // 1 - tanh^2
}
// f16 holds dS up to 65504, and an output gradient that carries a loss scale may pass that where dq, dk and dv do not. Such
// accumulators end up non-finite too, and the second walk (at_accumulate_seen) brings dS into range: each lane's column (one key, or
// one packed row) has a power of two that its ds and accumulators are in, lowered whenever a tile's largest ds passes 2^15
// in it. What falls below f16's normal numbers is then off by a 2^-39th of the column's largest. bf16 has f32's exponents.
template <typename T> constexpr bool AT_FIT = false;
template <> inline constexpr bool AT_FIT<f16_t> = true;
template <int FD>
__device__ __forceinline__ void at_fit(float* ds, at_f32x16* acc, float& unit) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    ds[i] *= unit;
    most = fmaxf(most, fabsf(ds[i]) < INFINITY ? fabsf(ds[i]) : 0.f);
  }
  most = at_half_max(most);
  if (!__any(most > 32768.f)) return;
  // 2^(14 + e) <= most < 2^(15 + e): times 2^-e
  const float down = most > 32768.f ? __uint_as_float((unsigned)(2 * 127 + 14 - (int)(__float_as_uint(most) >> 23)) << 23) : 1.f;
  unit *= down;
#pragma unroll
  for (int i = 0; i < 16; ++i) ds[i] *= down;
#pragma unroll
  for (int f = 0; f < FD; ++f) acc[f] *= down;
}
// LDS of the key workgroups: their V tile, two stages of (Q, dO) tiles of 32 queries of one head, two of the rows'
// values (one DMA instruction each, whose upper 32 lanes bring zeros). K stays in registers as the score's operand; V does
// not fit there beside the two accumulators (192 registers) and is read from LDS for each dP.
struct AtRowData {
  float lse[64], nd[64];  // nd: -delta
  int lo[64], hi[64];
};
constexpr int AT_QT = 32;
// NW: waves of a workgroup; KW: those along the keys, 32 each
template <typename T, int DF, int NW, int KW> struct AtBwdLds {
  static constexpr int RB = AtPad<DF>::DP * AtT<T>::E;
  static constexpr int NG = NW / KW;                        // groups of waves that take the query tiles in turn
  static constexpr int KT = sizeof(T) == 4 ? 32 : 64;       // keys per tile of the row workgroups
  static constexpr int QTILE = AT_QT * RB, VT = 32 * KW * RB;
  static constexpr int GROUP = 4 * QTILE + 2 * (int)sizeof(AtRowData);  // a group's stages
  static constexpr int SUM = KW * 64 * DF / 2;                          // floats of a group's dK or dV
  static constexpr int KEYS = VT + NG * GROUP, ROWS = 4 * KT * RB, ADD = NG > 1 ? (NG > 2 ? 4 : 2) * SUM * 4 : 0;
  static constexpr int MOST = KEYS > ROWS ? KEYS : ROWS;
  static constexpr int BYTES = (MOST > ADD ? MOST : ADD) + 32 * (int)sizeof(int);  // (and 32 ints: ranges, a vote)
};

template <typename T, int DF, bool CAP, bool SLOPE, int NW, int KW>
__device__ __forceinline__ void at_bwd_keys(const AtArgs& a, int bh, int ktile, char* smem) {
  typedef AtBwdLds<T, DF, NW, KW> L;
  constexpr int DP = AtPad<DF>::DP, KS = AtOffsets<T, DF>::KS, FD = DF / 32;
  constexpr int TILE = L::QTILE, STAGE = 2 * TILE;
  constexpr int NG = L::NG, NT = 64 * NW;
  int* range = (int*)(smem + L::BYTES) - 32;
  if (threadIdx.x == 0) range[16] = 0;
  const int lane = threadIdx.x & 63, w8 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int wid = w8 % KW, grp = w8 / KW;  // 32 keys; which of the query tiles
  const int b = bh / a.hk, kh = bh - b * a.hk;
  const int kb0 = ktile * 32 * KW, kw0 = kb0 + 32 * wid, key = kw0 + (lane & 31);
  const unsigned lds0 = (unsigned)(uintptr_t)((__attribute__((address_space(3))) char*)smem);
  const T* kb = (const T*)a.k + b * a.k_sb + kh * a.k_sh;
  const T* vb = (const T*)a.v + b * a.v_sb + kh * a.v_sh;

  // the queries that see any of the keys lie in [q0, q1]
  const long long nrows = (long long)a.batch * a.hq * a.lq, nq = (long long)a.batch * a.lq;
  const int* w_lo = (const int*)a.rowws + nrows + (long long)b * a.lq;
  const int* w_hi = w_lo + nq;
  int q0 = 0x7fffffff, q1 = -1;
  if (a.spans) {
    for (int i = threadIdx.x; i < a.lq; i += 4 * NT) {
      int lo[4], hi[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = min(i + NT * u, a.lq - 1);
        lo[u] = w_lo[r];
        hi[u] = w_hi[r];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i + NT * u < a.lq && hi[u] > kb0 && lo[u] < kb0 + 32 * KW) {
          q0 = min(q0, i + NT * u);
          q1 = max(q1, i + NT * u);
        }
    }
    q0 = at_wave_min(q0), q1 = at_wave_max(q1);
    if (lane == 0) range[w8] = q0, range[8 + w8] = q1;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) q0 = min(q0, range[w]), q1 = max(q1, range[8 + w]);
    q0 = __builtin_amdgcn_readfirstlane(q0);
    q1 = __builtin_amdgcn_readfirstlane(q1);
  } else {  // spans by position start at 0 and only widen: the last query, and the first whose end is past the keys' start
    const int n = at_keys(a, b);
    if (a.lq > 0 && at_span(a, b, a.lq - 1).hi > kb0) {
      q1 = a.lq - 1;
      // hi(i) = min(n, max(n - lq + i + 1, prefix)) under causal: past kb0 for all queries, or from i = kb0 - (n - lq)
      q0 = at_span(a, b, 0).hi > kb0 ? 0 : max(kb0 - (n - a.lq), 0);
    }
    q0 = __builtin_amdgcn_readfirstlane(q0);
    q1 = __builtin_amdgcn_readfirstlane(q1);
  }

  const AtLoad<T, DP, AT_QT, KW> ql(a.q_sl, a.d, wid, lane), gl((long long)a.hq * a.d, a.d, wid, lane);
  // the tile's lse / delta / lo / hi: one a wave, or one pair
  const long long rv0 = ((long long)b * a.hq + kh * a.group) * a.lq;
  const unsigned rvo = lane < AT_QT ? (unsigned)lane * 4 : BUF_OOB;
  auto issue = [&](int stage, int g, int i0) {
    const unsigned S = lds0 + L::VT + grp * L::GROUP + stage * STAGE;
    const int head = kh * a.group + g;
    ql.issue((const T*)a.q + b * a.q_sb + head * a.q_sh, i0, q1 + 1, S, wid);
    gl.issue((const T*)a.go + ((long long)b * a.lq * a.hq + head) * a.d, i0, q1 + 1, S + TILE, wid);
    // queries past the last arrive as zeros: an empty span
#pragma unroll
    for (int n = 0; n < 4; n += KW) {
      const int x = n + wid;
      const float* rv = x < 2 ? (x == 0 ? a.lse : a.rowws) + rv0 + (long long)g * a.lq : (const float*)(x == 2 ? w_lo : w_hi);
      at_dma4(buf_rsrc(rv + i0, __builtin_amdgcn_readfirstlane(min(q1 + 1 - i0, AT_QT) * 4)), rvo,
              lds0 + L::VT + grp * L::GROUP + 2 * STAGE + stage * (unsigned)sizeof(AtRowData) + x * 256);
    }
  };

  // tiles of 32 queries, head after head; the groups take them in turn
  int g = 0, i0 = q0;  // the tile in hand: head (a.group or more: none), first query
  auto advance = [&](int n, int& hd, int& i) {
    for (; n > 0; --n) {
      i += AT_QT;
      if (i > q1) i = q0, ++hd;
    }
  };
  if (q1 >= 0) {  // (first: the rest of the set-up runs under the loads' latency)
    advance(grp, g, i0);
    if (g < a.group) issue(0, g, i0);
    const AtLoad<T, DP, 32 * KW, NW> vl(a.v_sl, a.d, w8, lane);
    vl.issue(vb, kb0, a.lk, lds0, w8);
  }
  uint4 kf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int e = (2 * ks + h) * AtT<T>::CH;
    kf[ks] = key < a.lk && e < a.d ? *(const uint4*)(kb + key * a.k_sl + e) : make_uint4(0, 0, 0, 0);
  }
  at_f32x16 dk[FD], dv[FD];
#pragma unroll
  for (int f = 0; f < FD; ++f) dk[f] = at_zero(), dv[f] = at_zero();
  const AtOffsets<T, DF> off(lane);
  const char* V = smem + wid * 32 * L::RB;
  float unit = 1.f;  // that ds and dk are in (at_fit)
  const int n0 = (at_keys(a, b)) - a.lq;  // position of query 0
  const char* const base = smem + L::VT + grp * L::GROUP;
  auto step = [&](auto stage, auto again) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    int g1 = g, i1 = i0;  // the next one
    advance(NG, g1, i1);
    if (g1 < a.group) issue(1 - stage, g1, i1);
    const char* Q = base + stage * STAGE;
    const char* G = Q + TILE;
    const AtRowData& x = *(const AtRowData*)(base + 2 * STAGE + stage * (int)sizeof(AtRowData));
    const int f_lo = x.lo[lane & 31], f_hi = x.hi[lane & 31];
    if (g < a.group && __any(f_hi > kw0 && f_lo < kw0 + 32)) {      // some row sees some of this wave's keys
      const bool full = __all(f_lo <= kw0 && f_hi >= kw0 + 32);     // every row sees all of them
      at_f32x16 s = at_zero(), dp = at_zero();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = at_mfma<T>(at_row<T, DF>(Q, off, 0, ks), kf[ks], s);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) dp = at_mfma<T>(at_row<T, DF>(G, off, 0, ks), at_row<T, DF>(V, off, 0, ks), dp);
      at_bend_tiles<T, CAP, 1>(a.sc, &s);
      const float slope = SLOPE ? at_slope<T>(a, kh * a.group + g) : 0.f;
      const float x0 = (float)(n0 + i0 + 4 * h - key);  // position of this lane's first row minus its key
      float p[16], ds[16];
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const float4 lse = *(const float4*)(x.lse + 8 * r4 + 4 * h);
        const float4 nd = *(const float4*)(x.nd + 8 * r4 + 4 * h);
        const float lp[4] = {lse.x, lse.y, lse.z, lse.w}, dl[4] = {nd.x, nd.y, nd.z, nd.w};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 4 * r4 + r;
          at_grad<T, CAP, SLOPE>(a, slope, s[i], fabsf(x0 + (float)(8 * r4 + r)), lp[r],
                                 dp[i] + dl[r], p[i], ds[i]);
        }
      }
      if (!full) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int4 lo = *(const int4*)(x.lo + 8 * r4 + 4 * h), hi = *(const int4*)(x.hi + 8 * r4 + 4 * h);
          const int out[4] = {(key < lo.x) | (key >= hi.x), (key < lo.y) | (key >= hi.y), (key < lo.z) | (key >= hi.z),
                              (key < lo.w) | (key >= hi.w)};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            p[4 * r4 + r] = out[r] ? 0.f : p[4 * r4 + r];
            ds[4 * r4 + r] = out[r] ? 0.f : ds[4 * r4 + r];
          }
        }
      }
#pragma unroll
      for (int i = 0; AtLift<T>::BWD != 1.f && i < 16; ++i) p[i] *= AtLift<T>::BWD;
      // p and ds are rounded to the 16-bit operand type (half a step each)
      const auto sees = [&](int r) { return key >= x.lo[r] && key < x.hi[r]; };
      if (again.value && !full && at_has_nonfinite<T, DF>(G, 0, lane))
        at_accumulate_seen<T, DF>(G, 0, p, dv, lane, sees);
      else
        at_accumulate<T, DF>(G, off, 0, AtP<T>(p), dv, lane);
      if constexpr (again.value && AT_FIT<T>) at_fit<FD>(ds, dk, unit);
      if (again.value && !full && at_has_nonfinite<T, DF>(Q, 0, lane))
        at_accumulate_seen<T, DF>(Q, 0, ds, dk, lane, sees);
      else
        at_accumulate<T, DF>(Q, off, 0, AtP<T>(ds), dk, lane);
    }
    g = g1, i0 = i1;
  };
  auto walk = [&](auto again) {
    if (q1 < 0) return;
    // (uniform over the workgroup: the first group's count)
    const int nt = (a.group * ((q1 - q0) / AT_QT + 1) + NG - 1) / NG;
    if constexpr (again.value) {  // (one copy of the code: its stages need not be constants)
#pragma unroll 1
      for (int t = 0; t < nt; ++t) step(t & 1, again);
    } else {
      for (int t = 0; t < nt; t += 2) {
        step(std::integral_constant<int, 0>{}, again);
        if (t + 1 < nt) step(std::integral_constant<int, 1>{}, again);
      }
    }
  };
  walk(std::false_type{});
  const bool masked = a.causal || a.spans || a.kv_lens;
  if (masked || AT_FIT<T>) {
    bool bad = at_bad_columns<FD>(dk) != 0 || (masked && at_bad_columns<FD>(dv) != 0);
    if (bad) {  // (a row that sees all of the wave's keys and whose lse is NaN makes both sums NaN in every dim)
      bool nan = false;
      for (int i = q0 + lane; i <= q1; i += 64)
        if (w_lo[i] <= kw0 && w_hi[i] >= kw0 + 32)
          for (int n = 0; n < a.group; ++n) nan |= a.lse[rv0 + (long long)n * a.lq + i] != a.lse[rv0 + (long long)n * a.lq + i];
      bad = !__any(nan);
    }
    if (__builtin_expect(at_vote(bad, range + 16), 0)) {  // (unlikely: its spills stay out of the first walk)
#pragma unroll
      for (int f = 0; f < FD; ++f) dk[f] = at_zero(), dv[f] = at_zero();
      g = 0, i0 = q0;
      advance(grp, g, i0);
      if (q1 >= 0 && g < a.group) issue(0, g, i0);
      walk(std::true_type{});
      unit = 1.f / unit;
#pragma unroll
      for (int f = 0; AT_FIT<T> && f < FD; ++f) dk[f] *= unit;
    }
  }
  if constexpr (NG > 1) {  // the groups' sums through LDS: dK's to the first group, dV's to the second
    float* sum = (float*)smem + wid * 64 * (DF / 2) + lane;
    constexpr int HALF = L::SUM;
    if constexpr (NG > 2) {  // first the upper two groups' to the lower two
      float* two = sum + (grp & 1) * 2 * HALF;
      __syncthreads();
      if (grp > 1) {
#pragma unroll
        for (int f = 0; f < FD; ++f)
#pragma unroll
          for (int i = 0; i < 16; ++i) two[(16 * f + i) * 64] = dk[f][i], two[HALF + (16 * f + i) * 64] = dv[f][i];
      }
      __syncthreads();
      if (grp < 2) {
#pragma unroll
        for (int f = 0; f < FD; ++f)
#pragma unroll
          for (int i = 0; i < 16; ++i) dk[f][i] += two[(16 * f + i) * 64], dv[f][i] += two[HALF + (16 * f + i) * 64];
      }
    }
    __syncthreads();
#pragma unroll
    for (int f = 0; f < FD; ++f)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (grp == 0)
          sum[HALF + (16 * f + i) * 64] = dv[f][i];
        else if (grp == 1)
          sum[(16 * f + i) * 64] = dk[f][i];
      }
    __syncthreads();
    if (grp > 1) return;
#pragma unroll
    for (int f = 0; f < FD; ++f)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (grp == 0)
          dk[f][i] += sum[(16 * f + i) * 64];
        else
          dk[f][i] = sum[HALF + (16 * f + i) * 64] + dv[f][i];
      }
  }
  // with two groups each stores one of the two (dv of the second group now in dk)
  const long long ko = ((long long)b * a.lk * a.hk + kh) * a.d, ks = (long long)a.hk * a.d;
  const bool mine = key < a.lk;
  if constexpr (NG > 1) {
    at_store_row<T, DF>((T*)(grp ? a.dv : a.dk) + ko + key * ks, dk, a.d, h, grp ? 1.f / AtLift<T>::BWD : a.scale, mine);
  } else {
    at_store_row<T, DF>((T*)a.dk + ko + key * ks, dk, a.d, h, a.scale, mine);
    at_store_row<T, DF>((T*)a.dv + ko + key * ks, dv, a.d, h, 1.f / AtLift<T>::BWD, mine);
  }
}

template <typename T, int DF, bool CAP, bool SLOPE, int NW, int KW>
__device__ __forceinline__ void at_bwd_rows(const AtArgs& a, int bh, int tile, char* smem) {
  typedef AtBwdLds<T, DF, NW, KW> L;
  constexpr int DP = AtPad<DF>::DP, KS = AtOffsets<T, DF>::KS, FD = DF / 32, KT = L::KT;
  constexpr int TILE = KT * L::RB, STAGE = 2 * TILE;
  int* range = (int*)(smem + L::BYTES) - 32;
  if (threadIdx.x == 0) range[16] = 0;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int b = bh / a.hk, kh = bh - b * a.hk, rows = a.lq * a.group;
  const int row = tile * 32 * NW + wid * 32 + (lane & 31);
  const AtRow pr = at_packed(a, kh, row < rows ? row : 0);
  AtSpan sp = {0, 0, 0};
  float lse = INFINITY, nd = 0.f;
  if (row < rows) {
    sp = at_span(a, b, pr.qi);
    const long long r = ((long long)b * a.hq + pr.head) * a.lq + pr.qi;
    lse = a.lse[r];
    nd = a.rowws[r];
  }
  const bool live = sp.hi > sp.lo;
  const AtBounds w = at_bounds(a, b, kh, tile * 32 * NW + wid * 32, rows, sp);
  const int w_lo = w.lo, w_hi = w.hi, i_lo = w.i_lo, i_hi = w.i_hi;
  int k_lo = w_lo, k_hi = w_hi;
  if (a.spans) {
    if (lane == 0) range[wid] = w_lo, range[8 + wid] = w_hi;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) k_lo = min(k_lo, range[i]), k_hi = max(k_hi, range[8 + i]);
    k_lo = __builtin_amdgcn_readfirstlane(k_lo);
    k_hi = __builtin_amdgcn_readfirstlane(k_hi);
  } else {
    k_lo = 0;
    k_hi = __builtin_amdgcn_readfirstlane(max(at_span(a, b, at_packed(a, kh, min(tile * 32 * NW + 32 * NW, rows) - 1).qi).hi, 0));
  }
  const unsigned lds0 = (unsigned)(uintptr_t)((__attribute__((address_space(3))) char*)smem);
  const T* kb = (const T*)a.k + b * a.k_sb + kh * a.k_sh;
  const T* vb = (const T*)a.v + b * a.v_sb + kh * a.v_sh;
  const T* qp = (const T*)a.q + b * a.q_sb + (long long)pr.qi * a.q_sl + pr.head * a.q_sh;
  const long long orow = (((long long)b * a.lq + pr.qi) * a.hq + pr.head) * a.d;
  const T* gp = (const T*)a.go + orow;
  const AtLoad<T, DP, KT, NW> kl(a.k_sl, a.d, wid, lane), vl(a.v_sl, a.d, wid, lane);
  auto issue = [&](int stage, int k0) {
    kl.issue(kb, k0, k_hi, lds0 + stage * STAGE, wid);
    vl.issue(vb, k0, k_hi, lds0 + stage * STAGE + TILE, wid);
  };
  const int nt = k_hi > k_lo ? (k_hi - k_lo + KT - 1) / KT : 0;
  if (nt > 0) issue(0, k_lo);
  uint4 qf[KS], gf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int e = (2 * ks + h) * AtT<T>::CH;
    qf[ks] = live && e < a.d ? *(const uint4*)(qp + e) : make_uint4(0, 0, 0, 0);
    gf[ks] = live && e < a.d ? *(const uint4*)(gp + e) : make_uint4(0, 0, 0, 0);
  }
  const float slope = SLOPE ? at_slope<T>(a, pr.head) : 0.f;
  const AtOffsets<T, DF> off(lane);
  float unit = 1.f;  // that ds and dq are in (at_fit)
  at_f32x16 dq[FD];
#pragma unroll
  for (int f = 0; f < FD; ++f) dq[f] = at_zero();
  auto step = [&](auto stage, auto again, int t) {
    const int k0 = k_lo + t * KT;
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + 1 < nt) issue(1 - stage, k0 + KT);
    if (k0 >= w_hi || k0 + KT <= w_lo) return;
    const char* K = smem + stage * STAGE;
    const char* V = K + TILE;
    const bool part = k0 < i_lo || k0 + KT > i_hi;
#pragma unroll
    for (int f = 0; f < KT / 32; ++f) {
      at_f32x16 s = at_zero(), dp = at_zero();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = at_mfma<T>(at_row<T, DF>(K, off, 32 * f, ks), qf[ks], s);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) dp = at_mfma<T>(at_row<T, DF>(V, off, 32 * f, ks), gf[ks], dp);
      at_bend_tiles<T, CAP, 1>(a.sc, &s);
      const float x0 = (float)(sp.at - k0 - 32 * f - 4 * h);
      float ds[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float p;
        at_grad<T, CAP, SLOPE>(a, slope, s[i], fabsf(x0 - (float)(8 * (i >> 2) + (i & 3))), lse,
                               dp[i] + nd, p, ds[i]);
      }
      if (part) {
        const int lo = sp.lo - k0 - 32 * f - 4 * h, hi = sp.hi - k0 - 32 * f - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i >> 2) + (i & 3) < lo || 8 * (i >> 2) + (i & 3) >= hi) ds[i] = 0.f;
      }
      if constexpr (again.value && AT_FIT<T>) at_fit<FD>(ds, dq, unit);
      if (again.value && part && at_has_nonfinite<T, DF>(K, 32 * f, lane))
        at_accumulate_seen<T, DF>(K, 32 * f, ds, dq, lane,
                                  [&](int r) { return k0 + 32 * f + r >= sp.lo && k0 + 32 * f + r < sp.hi; });
      else
        at_accumulate<T, DF>(K, off, 32 * f, AtP<T>(ds), dq, lane);
    }
  };
  auto walk = [&](auto again) {
    if constexpr (again.value) {
#pragma unroll 1
      for (int t = 0; t < nt; ++t) step(t & 1, again, t);
    } else {
      for (int t = 0; t < nt; t += 2) {
        step(std::integral_constant<int, 0>{}, again, t);
        if (t + 1 < nt) step(std::integral_constant<int, 1>{}, again, t + 1);
      }
    }
  };
  walk(std::false_type{});
  if (a.causal || a.spans || AT_FIT<T>) {
    const bool bad = (at_bad_columns<FD>(dq) & ~at_columns(!live || lse != lse || nd != nd)) != 0;
    if (__builtin_expect(at_vote(bad, range + 16), 0)) {
#pragma unroll
      for (int f = 0; f < FD; ++f) dq[f] = at_zero();
      if (nt > 0) issue(0, k_lo);
      walk(std::true_type{});
      unit = 1.f / unit;
#pragma unroll
      for (int f = 0; AT_FIT<T> && f < FD; ++f) dq[f] *= unit;
    }
  }
  if (!live) {
#pragma unroll
    for (int f = 0; f < FD; ++f) dq[f] = at_zero();
  }
  at_store_row<T, DF>((T*)a.dq + orow, dq, a.d, h, a.scale, row < rows);
}

// blockIdx.y first counts the workgroups of 32 KW keys (the first keys are seen by most queries), then those of 32 NW packed
// rows, the last rows first, or the other way round (rows_first); heads vary fastest, as in the forward
// (waves a SIMD: what the first walk's registers allow; the second one's would allow fewer, and spills instead)
template <typename T, int DF, bool CAP, bool SLOPE, int NW, int KW>
__global__ void __launch_bounds__(64 * NW, sizeof(T) == 4 ? (DF > 64 ? 1 : 2) : DF == 32 ? 4 : DF == 64 ? 3 : 2) k_mattn_bwd(AtArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int ktiles = (a.lk + 32 * KW - 1) / (32 * KW), y = blockIdx.y;
  const int t = !a.rows_first ? y : y + ktiles < (int)gridDim.y ? y + ktiles : y + ktiles - gridDim.y;
  if (t < ktiles)
    at_bwd_keys<T, DF, CAP, SLOPE, NW, KW>(a, blockIdx.x, t, smem);
  else
    at_bwd_rows<T, DF, CAP, SLOPE, NW, KW>(a, blockIdx.x, gridDim.y - 1 - t, smem);
}

template <typename T, int DF, bool CAP, bool SLOPE, int NW, int KW>
static int mattn_bwd_kw(AtArgs a, hipStream_t stream) {
  typedef AtBwdLds<T, DF, NW, KW> L;
  // Without a mask the kind with the longer walks starts first: 4 lq group / groups products of a tile for a key workgroup's
  // waves against 3 lk for a row workgroup's (1187 tokens, 12 heads of 64: 52 -> 41 us). Under a mask the first keys do (an
  // order by the longest walks left was measured: even for causal masks, 20 % slower for documents).
  a.rows_first = !a.causal && !a.spans && 3LL * a.lk * L::NG > 4LL * a.lq * a.group;
  const dim3 grid((unsigned)(a.batch * a.hk), (unsigned)(cdiv(a.lk, 32 * KW) + cdiv((long long)a.lq * a.group, 32 * NW)));
  hipLaunchKernelGGL((k_mattn_bwd<T, DF, CAP, SLOPE, NW, KW>), grid, dim3(64 * NW), L::BYTES, stream, a);
  DMF_LAUNCH_CHECK("dmf_mattn_bwd");
  return 0;
}
// The workgroups, from sizes and the kind of mask (bf16, 128 dims unless said, the whole backward):
//   4 waves, two workgroups a CU: their loads, barriers and stores fall apart in time and overlap. 32 x 576 tokens, 4 heads, capped:
//     135 -> 132 us against the next form; 32 x 257, 12 heads of 64: 92 -> 67.
//   8 waves, two groups that share a key block's walk, one workgroup a CU: where a mask makes walks unequal and the longest
//     one, which grows with the heads of a group, would end long after the others. 4096 causal tokens, 32 heads over 8 (256 key
//     blocks): 514 us against 791 with 4 waves, 6144 (384): 1094 against 1293; with 512 key blocks the two meet (8192:
//     1895 against 1905) and then turn (3 x 4096: 1503 against 1476), and one head a group gains
//     from 4 waves or comes out even. Documents turn later (16384 tokens in 12, 16 heads over 4, 512 blocks: 684 against 784;
//     32768 in 60, 1024 blocks: 844 against 844).
//   8 waves over 64 keys, four groups: while 128-key blocks would leave half of the 256 CUs without one: twice the workgroups
//     with half the walk, for twice the loads a product. 2048 causal tokens, 32 heads over 8 (128 key blocks): 232 -> 158 us
//     against the second form; at 4096 (256) 514 -> 524. f32, 64 dims: 2 x 1024 causal tokens, 16 heads over 4: 519 -> 276 us;
//     4 x 329 tokens, 4 heads: 59.6 -> 54.8.
//     Up to one block a CU under a document mask, whose longest document is the longest walk (8192 tokens, 16 heads over 4,
//     second form -> this: 3 documents 655 -> 543, 12: 333 -> 278, 64: 115 -> 121), not beyond
//     (4 x 4096 tokens, 8 documents each, 512 blocks: 354 -> 389).
constexpr int AT_FEW_KEY_BLOCKS = 128, AT_EVEN_KEY_BLOCKS = 512;
template <typename T, int DF, bool CAP, bool SLOPE>
static int mattn_bwd_df(const AtArgs& a, hipStream_t stream) {
  const long long blocks = (long long)a.batch * a.hk * cdiv(a.lk, 128);
  if constexpr (sizeof(T) == 2 || DF <= 64) {  // (f32 of more dims: LDS for one group of 4 waves)
    if (blocks <= (a.spans && a.group > 1 ? 2 : 1) * AT_FEW_KEY_BLOCKS) return mattn_bwd_kw<T, DF, CAP, SLOPE, 8, 2>(a, stream);
    const bool uneven = a.group > 1 && (a.causal || a.spans || a.kv_lens);
    if (!uneven || blocks >= (a.spans ? 2 : 1) * AT_EVEN_KEY_BLOCKS) return mattn_bwd_kw<T, DF, CAP, SLOPE, 4, 4>(a, stream);
  }
  return mattn_bwd_kw<T, DF, CAP, SLOPE, (sizeof(T) == 4 && DF > 64 ? 4 : 8), 4>(a, stream);
}

template <typename T>
static int mattn_bwd_t(AtArgs a, hipStream_t stream) {
  at_score_args<T>(a);
  const long long n = (long long)a.batch * a.lq * a.hq;
  if (n > 0) {
    hipLaunchKernelGGL((k_mattn_rows<T>), dim3((unsigned)((n + 15) / 16)), dim3(256), 0, stream, a);
    DMF_LAUNCH_CHECK("dmf_mattn_bwd (rows)");
  }
#define DMF_AT_MODE(DF)                                                                                 \
  return a.cap > 0.f ? (a.slopes ? mattn_bwd_df<T, DF, true, true>(a, stream)                           \
                                 : mattn_bwd_df<T, DF, true, false>(a, stream))                         \
                     : (a.slopes ? mattn_bwd_df<T, DF, false, true>(a, stream)                          \
                                 : mattn_bwd_df<T, DF, false, false>(a, stream))
  if (a.d <= 32) DMF_AT_MODE(32);
  if (a.d <= 64) DMF_AT_MODE(64);
  if (a.d <= 96) DMF_AT_MODE(96);
  DMF_AT_MODE(128);
#undef DMF_AT_MODE
}

}  // namespace dmf
