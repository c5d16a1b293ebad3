// Masked attention backward (see masked_attn.h for the mathematics and the layouts).
//
//   delta_i = sum_d do_i o_i          (k_mattn_delta; o with the part its 16-bit rounding left over, so that rounding does
//                                      not enter dS through the whole row)
//   p_ij = exp(s_ij - lse_i),  dp_ij = do_i . v_j,  ds_ij = p_ij (dp_ij - delta_i) (1 - tanh^2(z_ij / cap))
//   dv_j = sum_i p_ij do_i,  dk_j = scale sum_i ds_ij q_i,  dq_i = scale sum_j ds_ij k_j
//
// One launch holds two kinds of workgroups: those of 128 keys, which walk the packed query rows that see them and keep
// dK and dV in registers, and those of 128 packed rows, which walk their keys and keep dQ. The scores are computed in
// both (7 products for the 5 that one pass with dQ in atomics would take): no atomics, so the same bits every run, no
// f32 dQ in HBM, and the sum over a group's query heads happens inside the dK / dV accumulators.
#pragma once
#include "masked_attn.h"
#include "masked_attn_fwd.h"

namespace dmf {

// packed row r of a (batch row, key head): query r / group, head kh * group + r % group
struct AtRow {
  int qi, head;
};
__device__ __forceinline__ AtRow at_packed(const AtArgs& a, int kh, int r) {
  AtRow x;
  x.qi = r / a.group;
  x.head = kh * a.group + r - x.qi * a.group;
  return x;
}

// delta: one lane group of 16 per packed row
template <typename T>
__global__ void __launch_bounds__(256) k_mattn_delta(AtArgs a) {
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
    const int qi = (int)(bq % a.lq), b = (int)(bq / a.lq), kh = head / a.group;
    a.delta[((long long)b * a.hk + kh) * a.lq * a.group + qi * a.group + head - kh * a.group] = t;
  }
}

// ds and p of one score (p masked to 0 by the caller)
template <typename T, bool CAP, bool SLOPE>
__device__ __forceinline__ void at_grad(const AtScore& c, float slope_u, float raw, float dist, float lse, float dp,
                                        float delta, float& p, float& ds) {
  float s, bend = 1.f;
  if constexpr (CAP) {
    const float t = at_tanh<T>(raw * c.scale_cap);
    s = c.cap_u * t;
    bend = fmaf(-t, t, 1.f);
  } else {
    s = raw * c.scale_u;
  }
  if constexpr (SLOPE) s = fmaf(-slope_u, dist, s);
  p = at_exp<T>(s - lse);
  ds = p * (dp - delta);
  if constexpr (CAP) ds *= bend;
}

// LDS of the 128-key workgroups: two stages of (Q, dO) tiles, then two stages of the per-row values
template <int QT> struct AtRowData {
  float lse[QT], delta[QT], at[QT], slope[QT];
  int lo[QT], hi[QT];
  unsigned full[4], none[4];  // bit s of [w]: every row of 32-row subtile s sees all / none of wave w's keys
};

template <typename T> struct AtBwdTile { static constexpr int QT = sizeof(T) == 4 ? 32 : 64, KT = QT; };

// Q / dO rows r0 .. r0 + QT - 1 (packed) into a tile: as at_load_rows, with the packed row's address per lane
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void at_load_packed(const AtArgs& a, const T* base, long long sl, long long sh, int r0, int r1,
                                               unsigned lds, int wid, int lane) {
  constexpr int NC = DP * AtT<T>::E / 16, PIECES = ROWS * NC / 64;
  const int i0 = r0 / a.group;
  const v4i_t rs = buf_rsrc(base + (long long)i0 * sl, AT_RECORDS);
#pragma unroll
  for (int i = 0; i < PIECES / 4; ++i) {
    const int p = wid * (PIECES / 4) + i, pos = p * 64 + lane, row = pos / NC;
    const int ch = (pos % NC) ^ at_swz<T, DP>(row);
    const int r = r0 + row, qi = r / a.group, g = r - qi * a.group;
    const bool ok = r < r1 && ch * AtT<T>::CH < a.d;
    dma16(rs, ok ? (unsigned)(((qi - i0) * (int)sl + g * (int)sh) * AtT<T>::E + ch * 16) : BUF_OOB, 0, lds + p * 1024);
  }
}

// dk, dv of one key over the packed rows that see it: each lane holds dims lane and lane + 64
template <typename T, bool CAP, bool SLOPE>
__device__ void at_key_alone(const AtArgs& a, int b, int kh, int j, int r0, int r1, int lane, float dk[2], float dv[2]) {
  const T* kj = (const T*)a.k + b * a.k_sb + kh * a.k_sh + j * a.k_sl;
  const T* vj = (const T*)a.v + b * a.v_sb + kh * a.v_sh + j * a.v_sl;
  const bool on0 = lane < a.d, on1 = lane + 64 < a.d;
  const float k0 = on0 ? ld(kj + lane) : 0.f, k1 = on1 ? ld(kj + lane + 64) : 0.f;
  const float v0 = on0 ? ld(vj + lane) : 0.f, v1 = on1 ? ld(vj + lane + 64) : 0.f;
  dk[0] = dk[1] = dv[0] = dv[1] = 0.f;
  const long long rows = (long long)a.lq * a.group, rb = ((long long)b * a.hk + kh) * rows;
  for (int r = r0; r < r1; ++r) {
    const AtRow x = at_packed(a, kh, r);
    const AtSpan sp = at_span(a, b, x.qi);
    if (j < sp.lo || j >= sp.hi) continue;
    const T* q = (const T*)a.q + b * a.q_sb + (long long)x.qi * a.q_sl + x.head * a.q_sh;
    const T* g = (const T*)a.go + (((long long)b * a.lq + x.qi) * a.hq + x.head) * a.d;
    const float q0 = on0 ? ld(q + lane) : 0.f, q1 = on1 ? ld(q + lane + 64) : 0.f;
    const float g0 = on0 ? ld(g + lane) : 0.f, g1 = on1 ? ld(g + lane + 64) : 0.f;
    const float raw = wave_sum(fmaf(q0, k0, q1 * k1)), dp = wave_sum(fmaf(g0, v0, g1 * v1));
    const AtScore sc = at_score_of<T>(a, x.head);
    float p, ds;
    at_grad<T, CAP, SLOPE>(sc, sc.slope_u, raw, fabsf((float)(sp.at - j)), a.lse[rb + r], dp, a.delta[rb + r], p, ds);
    dk[0] = fmaf(ds, q0, dk[0]), dk[1] = fmaf(ds, q1, dk[1]);
    dv[0] = fmaf(p, g0, dv[0]), dv[1] = fmaf(p, g1, dv[1]);
  }
}

// dq of one packed row over its own span
template <typename T, bool CAP, bool SLOPE>
__device__ void at_query_alone(const AtArgs& a, int b, int kh, int r, int lo, int hi, int at, int lane, float dq[2]) {
  const AtRow x = at_packed(a, kh, r);
  const T* q = (const T*)a.q + b * a.q_sb + (long long)x.qi * a.q_sl + x.head * a.q_sh;
  const T* g = (const T*)a.go + (((long long)b * a.lq + x.qi) * a.hq + x.head) * a.d;
  const bool on0 = lane < a.d, on1 = lane + 64 < a.d;
  const float q0 = on0 ? ld(q + lane) : 0.f, q1 = on1 ? ld(q + lane + 64) : 0.f;
  const float g0 = on0 ? ld(g + lane) : 0.f, g1 = on1 ? ld(g + lane + 64) : 0.f;
  const long long rb = ((long long)b * a.hk + kh) * a.lq * a.group + r;
  const float lse = a.lse[rb], delta = a.delta[rb];
  const AtScore sc = at_score_of<T>(a, x.head);
  dq[0] = dq[1] = 0.f;
  for (int j = lo; j < hi; ++j) {
    const T* kj = (const T*)a.k + b * a.k_sb + kh * a.k_sh + j * a.k_sl;
    const T* vj = (const T*)a.v + b * a.v_sb + kh * a.v_sh + j * a.v_sl;
    const float k0 = on0 ? ld(kj + lane) : 0.f, k1 = on1 ? ld(kj + lane + 64) : 0.f;
    const float v0 = on0 ? ld(vj + lane) : 0.f, v1 = on1 ? ld(vj + lane + 64) : 0.f;
    const float raw = wave_sum(fmaf(q0, k0, q1 * k1)), dp = wave_sum(fmaf(g0, v0, g1 * v1));
    float p, ds;
    at_grad<T, CAP, SLOPE>(sc, sc.slope_u, raw, fabsf((float)(at - j)), lse, dp, delta, p, ds);
    dq[0] = fmaf(ds, k0, dq[0]), dq[1] = fmaf(ds, k1, dq[1]);
  }
}

// one lane's column of a transposed accumulator, times `scale`, to its row of the output
template <typename T, int DF>
__device__ __forceinline__ void at_store_row(T* out, const at_f32x16* acc, int d, int h, float scale) {
#pragma unroll
  for (int f = 0; f < DF / 32; ++f)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int e = 32 * f + 8 * g + 4 * h;
      if (e >= d) continue;
      const float v[4] = {acc[f][4 * g] * scale, acc[f][4 * g + 1] * scale, acc[f][4 * g + 2] * scale,
                          acc[f][4 * g + 3] * scale};
      at_store4(out + e, v);
    }
}

template <typename T, int DF, bool CAP, bool SLOPE>
__device__ __forceinline__ void at_bwd_keys(const AtArgs& a, int bh, int ktile, char* smem) {
  constexpr int DP = AtPad<DF>::DP, KS = AtSteps<T, DF>::N, FD = DF / 32, QT = AtBwdTile<T>::QT;
  constexpr int TILE = QT * DP * AtT<T>::E, STAGE = 2 * TILE;
  AtRowData<QT>* rd = (AtRowData<QT>*)(smem + 2 * STAGE);
  int* range = (int*)(rd + 2);  // [8]
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int b = bh / a.hk, kh = bh - b * a.hk, rows = a.lq * a.group;
  const int kb0 = ktile * 128, kw0 = kb0 + 32 * wid, key = kw0 + (lane & 31);
  const unsigned lds0 = (unsigned)(uintptr_t)((__attribute__((address_space(3))) char*)smem);
  const T* qb = (const T*)a.q + b * a.q_sb + kh * a.group * a.q_sh;
  const T* gb = (const T*)a.go + ((long long)b * a.lq * a.hq + kh * a.group) * a.d;
  const long long rb = (long long)bh * rows;

  // the queries that see any of the 128 keys lie in [q0, q1]
  int q0 = 0x7fffffff, q1 = -1;
  for (int i = threadIdx.x; i < a.lq; i += 256) {
    const AtSpan sp = at_span(a, b, i);
    if (sp.hi > kb0 && sp.lo < kb0 + 128 && sp.hi > sp.lo) {
      q0 = min(q0, i);
      q1 = max(q1, i);
    }
  }
  q0 = at_wave_min(q0), q1 = at_wave_max(q1);
  if (lane == 0) range[wid] = q0, range[4 + wid] = q1;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) q0 = min(q0, range[w]), q1 = max(q1, range[4 + w]);
  q0 = __builtin_amdgcn_readfirstlane(q0);
  q1 = __builtin_amdgcn_readfirstlane(q1);
  const int r0 = q1 >= 0 ? q0 * a.group : 0, r1 = (q1 + 1) * a.group;

  uint4 kf[KS], vf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int e = (2 * ks + h) * AtT<T>::CH;
    const bool ok = key < a.lk && e < a.d;
    kf[ks] = ok ? *(const uint4*)((const T*)a.k + b * a.k_sb + kh * a.k_sh + key * a.k_sl + e) : make_uint4(0, 0, 0, 0);
    vf[ks] = ok ? *(const uint4*)((const T*)a.v + b * a.v_sb + kh * a.v_sh + key * a.v_sl + e) : make_uint4(0, 0, 0, 0);
  }
  auto issue = [&](int stage, int r) {
    at_load_packed<T, DP, QT>(a, qb, a.q_sl, a.q_sh, r, r1, lds0 + stage * STAGE, wid, lane);
    at_load_packed<T, DP, QT>(a, gb, (long long)a.hq * a.d, a.d, r, r1, lds0 + stage * STAGE + TILE, wid, lane);
  };
  // the rows' values for one tile, by the first QT threads (wave 0)
  auto row_data = [&](int stage, int r) {
    if (wid != 0) return;
    AtRowData<QT>& x = rd[stage];
    const int rr = r + lane;
    const bool in = lane < QT && rr < r1;
    AtSpan sp = {0, 0, 0};
    float lse = INFINITY, delta = 0.f, slope = 0.f;
    if (in) {
      const AtRow pr = at_packed(a, kh, rr);
      sp = at_span(a, b, pr.qi);
      lse = a.lse[rb + rr];
      delta = a.delta[rb + rr];
      if (SLOPE) slope = a.slopes[pr.head] * AtUnit<T>::U;
    }
    const bool live = sp.hi > sp.lo;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int kw = kb0 + 32 * w;
      const unsigned long long f = __ballot(live && sp.lo <= kw && sp.hi >= kw + 32);
      const unsigned long long n = __ballot(!live || sp.hi <= kw || sp.lo >= kw + 32);
      if (lane == 0) {
        x.full[w] = ((unsigned)f == ~0u ? 1 : 0) | ((unsigned)(f >> 32) == ~0u ? 2 : 0);
        x.none[w] = ((unsigned)n == ~0u ? 1 : 0) | ((unsigned)(n >> 32) == ~0u ? 2 : 0);
      }
    }
    if (lane < QT) {
      x.lse[lane] = lse;
      x.delta[lane] = delta;
      x.at[lane] = (float)sp.at;
      x.slope[lane] = slope;
      x.lo[lane] = sp.lo;
      x.hi[lane] = sp.hi;
    }
  };

  const AtScore sc = at_score_of<T>(a, kh * a.group);
  at_f32x16 dk[FD], dv[FD];
#pragma unroll
  for (int f = 0; f < FD; ++f) dk[f] = at_zero(), dv[f] = at_zero();
  const int nt = r1 > r0 ? (r1 - r0 + QT - 1) / QT : 0;
  if (nt > 0) {
    row_data(0, r0);
    issue(0, r0);
  }
  for (int t = 0; t < nt; ++t) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + 1 < nt) {
      row_data((t + 1) & 1, r0 + (t + 1) * QT);
      issue((t + 1) & 1, r0 + (t + 1) * QT);
    }
    const char* Q = smem + (t & 1) * STAGE;
    const char* G = Q + TILE;
    const AtRowData<QT>& x = rd[t & 1];
    const unsigned full = __builtin_amdgcn_readfirstlane(x.full[wid]), none = __builtin_amdgcn_readfirstlane(x.none[wid]);
#pragma unroll
    for (int f = 0; f < QT / 32; ++f) {
      if ((none >> f) & 1) continue;
      at_f32x16 s = at_zero(), dp = at_zero();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = at_mfma<T>(at_row<T, DP>(Q, 32 * f + (lane & 31), ks, h), kf[ks], s);
        dp = at_mfma<T>(at_row<T, DP>(G, 32 * f + (lane & 31), ks, h), vf[ks], dp);
      }
      float p[16], ds[16];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int rr = 32 * f + 8 * g + 4 * h;
        const float4 lse = *(const float4*)(x.lse + rr), delta = *(const float4*)(x.delta + rr);
        float4 at = make_float4(0.f, 0.f, 0.f, 0.f), slope = at;
        if constexpr (SLOPE) at = *(const float4*)(x.at + rr), slope = *(const float4*)(x.slope + rr);
        const float* lp = &lse.x;
        const float* dl = &delta.x;
        const float* ap = &at.x;
        const float* sp = &slope.x;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          at_grad<T, CAP, SLOPE>(sc, sp[r], s[4 * g + r], fabsf(ap[r] - (float)key), lp[r], dp[4 * g + r], dl[r],
                                 p[4 * g + r], ds[4 * g + r]);
      }
      if (!((full >> f) & 1)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int rr = 32 * f + 8 * (i >> 2) + 4 * h + (i & 3);
          if (key < x.lo[rr] || key >= x.hi[rr]) p[i] = ds[i] = 0.f;
        }
      }
      // p and ds are rounded to the 16-bit operand type (half a step each)
      at_accumulate<T, DF>(G, 32 * f, p, dv, lane);
      at_accumulate<T, DF>(Q, 32 * f, ds, dk, lane);
    }
  }
  float bad = 0.f;
#pragma unroll
  for (int f = 0; f < FD; ++f)
#pragma unroll
    for (int i = 0; i < 16; ++i) bad = fmaf(dk[f][i], 0.f, fmaf(dv[f][i], 0.f, bad));
  const unsigned long long redo = __ballot(key < a.lk && bad != bad);
  const unsigned alone = (unsigned)redo | (unsigned)(redo >> 32);
  const long long ko = ((long long)b * a.lk * a.hk + kh) * a.d, ks = (long long)a.hk * a.d;
  if (key < a.lk && !((alone >> (lane & 31)) & 1)) {
    at_store_row<T, DF>((T*)a.dk + ko + key * ks, dk, a.d, h, a.scale);
    at_store_row<T, DF>((T*)a.dv + ko + key * ks, dv, a.d, h, 1.f);
  }
  for (unsigned todo = alone; todo; todo &= todo - 1) {
    const int j = kw0 + __builtin_ctz(todo);
    float gk[2], gv[2];
    at_key_alone<T, CAP, SLOPE>(a, b, kh, j, r0, r1, lane, gk, gv);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (lane + 64 * e < a.d) {
        st((T*)a.dk + ko + j * ks + lane + 64 * e, gk[e] * a.scale);
        st((T*)a.dv + ko + j * ks + lane + 64 * e, gv[e]);
      }
  }
}

template <typename T, int DF, bool CAP, bool SLOPE>
__device__ __forceinline__ void at_bwd_rows(const AtArgs& a, int bh, int tile, char* smem) {
  constexpr int DP = AtPad<DF>::DP, KS = AtSteps<T, DF>::N, FD = DF / 32, KT = AtBwdTile<T>::KT;
  constexpr int TILE = KT * DP * AtT<T>::E, STAGE = 2 * TILE;
  int* range = (int*)(smem + 2 * STAGE);
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int b = bh / a.hk, kh = bh - b * a.hk, rows = a.lq * a.group;
  const int row = tile * 128 + wid * 32 + (lane & 31);
  const AtRow pr = at_packed(a, kh, row < rows ? row : 0);
  AtSpan sp = {0, 0, 0};
  float lse = INFINITY, delta = 0.f;
  if (row < rows) {
    sp = at_span(a, b, pr.qi);
    lse = a.lse[(long long)bh * rows + row];
    delta = a.delta[(long long)bh * rows + row];
  }
  const bool live = sp.hi > sp.lo;
  const int w_lo = at_wave_min(live ? sp.lo : 0x7fffffff), w_hi = at_wave_max(live ? sp.hi : 0);
  const int i_lo = at_wave_max(live ? sp.lo : 0), i_hi = at_wave_min(live ? sp.hi : 0x7fffffff);
  int k_lo = w_lo, k_hi = w_hi;
  if (lane == 0) range[wid] = w_lo, range[4 + wid] = w_hi;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) k_lo = min(k_lo, range[w]), k_hi = max(k_hi, range[4 + w]);
  k_lo = __builtin_amdgcn_readfirstlane(k_lo);
  k_hi = __builtin_amdgcn_readfirstlane(k_hi);
  const unsigned lds0 = (unsigned)(uintptr_t)((__attribute__((address_space(3))) char*)smem);
  const T* kb = (const T*)a.k + b * a.k_sb + kh * a.k_sh;
  const T* vb = (const T*)a.v + b * a.v_sb + kh * a.v_sh;
  const T* qp = (const T*)a.q + b * a.q_sb + (long long)pr.qi * a.q_sl + pr.head * a.q_sh;
  const long long orow = (((long long)b * a.lq + pr.qi) * a.hq + pr.head) * a.d;
  const T* gp = (const T*)a.go + orow;
  uint4 qf[KS], gf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int e = (2 * ks + h) * AtT<T>::CH;
    qf[ks] = live && e < a.d ? *(const uint4*)(qp + e) : make_uint4(0, 0, 0, 0);
    gf[ks] = live && e < a.d ? *(const uint4*)(gp + e) : make_uint4(0, 0, 0, 0);
  }
  auto issue = [&](int stage, int k0) {
    at_load_rows<T, DP, KT, 4>(kb, a.k_sl, k0, k_lo, k_hi, a.d, lds0 + stage * STAGE, wid, lane);
    at_load_rows<T, DP, KT, 4>(vb, a.v_sl, k0, k_lo, k_hi, a.d, lds0 + stage * STAGE + TILE, wid, lane);
  };
  const AtScore sc = at_score_of<T>(a, pr.head);
  at_f32x16 dq[FD];
#pragma unroll
  for (int f = 0; f < FD; ++f) dq[f] = at_zero();
  const int nt = k_hi > k_lo ? (k_hi - k_lo + KT - 1) / KT : 0;
  if (nt > 0) issue(0, k_lo);
  for (int t = 0; t < nt; ++t) {
    const int k0 = k_lo + t * KT;
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + 1 < nt) issue((t + 1) & 1, k0 + KT);
    if (k0 >= w_hi || k0 + KT <= w_lo) continue;
    const char* K = smem + (t & 1) * STAGE;
    const char* V = K + TILE;
    const bool part = k0 < i_lo || k0 + KT > i_hi;
    const float x0 = (float)(sp.at - k0 - 4 * h);
#pragma unroll
    for (int f = 0; f < KT / 32; ++f) {
      at_f32x16 s = at_zero(), dp = at_zero();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = at_mfma<T>(at_row<T, DP>(K, 32 * f + (lane & 31), ks, h), qf[ks], s);
        dp = at_mfma<T>(at_row<T, DP>(V, 32 * f + (lane & 31), ks, h), gf[ks], dp);
      }
      float ds[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int c = 32 * f + 8 * (i >> 2) + (i & 3);
        float p;
        at_grad<T, CAP, SLOPE>(sc, sc.slope_u, s[i], fabsf(x0 - (float)c), lse, dp[i], delta, p, ds[i]);
        if (part && (k0 + c + 4 * h < sp.lo || k0 + c + 4 * h >= sp.hi)) ds[i] = 0.f;
      }
      at_accumulate<T, DF>(K, 32 * f, ds, dq, lane);
    }
  }
  float bad = 0.f;
#pragma unroll
  for (int f = 0; f < FD; ++f)
#pragma unroll
    for (int i = 0; i < 16; ++i) bad = fmaf(dq[f][i], 0.f, bad);
  const unsigned long long redo = __ballot(live && bad != bad);
  const unsigned alone = (unsigned)redo | (unsigned)(redo >> 32);
  if (row < rows && !((alone >> (lane & 31)) & 1)) {
    if (!live) {
#pragma unroll
      for (int f = 0; f < FD; ++f) dq[f] = at_zero();
    }
    at_store_row<T, DF>((T*)a.dq + orow, dq, a.d, h, a.scale);
  }
  for (unsigned todo = alone; todo; todo &= todo - 1) {
    const int n = __builtin_ctz(todo);
    const int r = __shfl(row, n, 64);
    const AtRow x = at_packed(a, kh, r);
    float g[2];
    at_query_alone<T, CAP, SLOPE>(a, b, kh, r, __shfl(sp.lo, n, 64), __shfl(sp.hi, n, 64), __shfl(sp.at, n, 64), lane, g);
    T* out = (T*)a.dq + (((long long)b * a.lq + x.qi) * a.hq + x.head) * a.d;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (lane + 64 * e < a.d) st(out + lane + 64 * e, g[e] * a.scale);
  }
}

// workgroups [0, nk): 128 keys each (the longer ones: they start first); [nk, ..): 128 packed rows each
template <typename T, int DF, bool CAP, bool SLOPE>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2) k_mattn_bwd(AtArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int nbh = a.batch * a.hk;
  const int ktiles = (a.lk + 127) / 128, rtiles = gridDim.x / nbh - ktiles;
  const int bh = blockIdx.x % nbh, t = blockIdx.x / nbh;
  if (t < ktiles)
    at_bwd_keys<T, DF, CAP, SLOPE>(a, bh, t, smem);
  else
    at_bwd_rows<T, DF, CAP, SLOPE>(a, bh, rtiles - 1 - (t - ktiles), smem);
}

template <typename T, int DF, bool CAP, bool SLOPE>
static int mattn_bwd_df(const AtArgs& a, hipStream_t stream) {
  constexpr int QT = AtBwdTile<T>::QT;
  constexpr size_t LDS = 4 * QT * AtPad<DF>::DP * AtT<T>::E + 2 * sizeof(AtRowData<QT>) + 8 * sizeof(int);
  const long long nbh = (long long)a.batch * a.hk;
  const long long blocks = nbh * (cdiv(a.lk, 128) + cdiv((long long)a.lq * a.group, 128));
  hipLaunchKernelGGL((k_mattn_bwd<T, DF, CAP, SLOPE>), dim3((unsigned)blocks), dim3(256), LDS, stream, a);
  DMF_LAUNCH_CHECK("dmf_mattn_bwd");
  return 0;
}

template <typename T>
static int mattn_bwd_t(const AtArgs& a, hipStream_t stream) {
  const long long n = (long long)a.batch * a.lq * a.hq;
  if (n > 0) {
    hipLaunchKernelGGL((k_mattn_delta<T>), dim3((unsigned)((n + 15) / 16)), dim3(256), 0, stream, a);
    DMF_LAUNCH_CHECK("dmf_mattn_bwd (delta)");
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
