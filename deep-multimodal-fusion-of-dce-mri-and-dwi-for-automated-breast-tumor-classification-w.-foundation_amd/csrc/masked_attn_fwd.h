// Masked attention forward (see masked_attn.h for the mathematics and the layouts).
//
// A workgroup of NW waves takes 32 NW packed rows of one (batch row, key head); the keys of the union of their spans
// stream through two LDS stages of KT keys (LDS-DMA, the next tile in flight under the current one's products). A wave
// holds its 32 queries and their output accumulators in registers and keeps a running maximum and sum per row. The
// maximum may lag by 2^8 before the accumulators are rescaled (p <= 256 is exact enough in f32 and in range in f16), which
// takes the rescale out of almost every tile. NW = 4, KT = 64 for rows that fill it (KT = 32 where three on a CU pay, at_three); NW = 1, KT = 32 for up to 32 rows
// (single tokens: one wave per workgroup, five in a CU's LDS, so that enough loads are in flight to draw on HBM).
//
// Splits: with few workgroups along the rows the keys are cut into chunks of a.chunk, each workgroup writes its
// unnormalised accumulators with (max, sum), and k_mattn_join adds them. Chunks are cut at absolute keys, so a short row of a
// long cache leaves workgroups that exit at once instead of long ones that hold the others up.
//
// Keys outside the union of the workgroup's spans are zero-filled on load; a value inside it that is not finite stays with the
// rows that see it by a second walk (at_accumulate_seen).
//
// Bound: for many rows the order of a wave's own work, score product, cap and exponential, value product, which only the SIMD's other
// wave overlaps: neither unit is full (vector ALU 0.6 and matrix pipe 0.4 busy under a cap, 0.5 and 0.4 without).
// 8192 x 8192 tokens, 32 heads over 8 of 128, bf16: 1.03 to 1.08 ms by the inputs' scale (1.02 to 1.07 PFLOP/s; a large matrix
// product reaches 1.2 to 1.3), capped 1.26 to 1.42, for training 1.42 to 1.48; short rows also start and end: 32 x 576, 4 heads, capped,
// for training: 55 to 60 us. For single queries HBM: 8 rows of up to 65536 keys, 32 heads over 8: 249 us + 9 us of join (5.2 TB/s).
#pragma once
#include "masked_attn.h"

namespace dmf {

template <typename T>
__device__ __forceinline__ void at_store4(T* p, const float* v) {  // p aligned to 4 elements
  if constexpr (sizeof(T) == 4)
    *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
  else
    *(uint2*)p = make_uint2(AtPair<T>::pack(v[0], v[1]), AtPair<T>::pack(v[2], v[3]));
}
// One lane's column of transposed accumulators, times `scale`, to its row `out` of d elements (and what the rounding left
// over to `rest`, if REST). The two half waves hold alternate fours of a row's dims; 16-bit types swap halves of pairs of
// them, so that each lane stores 16 B. All 64 lanes call this; `on` says whether a lane's row is stored.
template <typename T, int DF, bool REST = false>
__device__ __forceinline__ void at_store_row(T* out, const at_f32x16* acc, int d, int h, float scale, bool on,
                                             T* rest = nullptr) {
#pragma unroll
  for (int f = 0; f < DF / 32; ++f) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int e = 32 * f + 8 * g + 4 * h;
        const float v[4] = {acc[f][4 * g] * scale, acc[f][4 * g + 1] * scale, acc[f][4 * g + 2] * scale,
                            acc[f][4 * g + 3] * scale};
        if (on && e < d) at_store4(out + e, v);
      }
    } else {
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        const int e = 32 * f + 8 * (g + h);
        float v[8];
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = acc[f][4 * g + i] * scale;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = AtPair<T>::pack(v[2 * i], v[2 * i + 1]);
        auto put = [&](T* p, const uint32_t* x) {
          const auto a = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false);
          const auto b = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
          if (on && e < d) *(uint4*)(p + e) = make_uint4(a[0], b[0], a[1], b[1]);
        };
        put(out, w);
        if constexpr (REST) {
          uint32_t r[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) r[i] = AtPair<T>::pack(v[2 * i] - B16<T>::lo(w[i]), v[2 * i + 1] - B16<T>::hi(w[i]));
          put(rest, r);
        }
      }
    }
  }
}

// waves a SIMD: what the first walk's registers allow (the second one's would allow fewer, and spills instead)
template <typename T> constexpr int at_fwd_waves(int df, bool cap, int nw, int kt) {
  if (sizeof(T) == 4) return df == 32 ? 4 : df == 64 ? (nw == 1 ? 2 : 3) : df == 96 ? 2 : 1;
  if (nw == 1) return df == 32 ? 5 : df == 64 ? 3 : 2;  // (LDS for no more)
  return df == 32 ? 5 : df == 64 ? 4 : df == 96 ? 3 : kt == 32 && (nw == 4 || !cap) ? 3 : 2;
}
template <typename T, int DF, bool CAP, bool SLOPE, bool TRAIN, int NW, int NG, int KT>
__global__ void __launch_bounds__(64 * NW * NG, at_fwd_waves<T>(DF, CAP, NW, KT)) k_mattn_fwd(AtArgs a) {
  constexpr int DP = AtPad<DF>::DP, KS = AtOffsets<T, DF>::KS, FD = DF / 32, KF = KT / 32;
  constexpr int TILE = KT * DP * AtT<T>::E, STAGE = 2 * TILE;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int range[2 * NW], again_flag;
  if (threadIdx.x == 0) again_flag = 0;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int wid = NG > 1 ? wave % NW : wave, grp = NG > 1 ? wave / NW : 0;  // 32 rows; which of the key tiles
  const int nbh = a.batch * a.hk, rows = a.lq * a.group;
  // Workgroups go to the eight XCDs in turn: splits, then heads vary fastest, so that an XCD gets a share of every batch
  // row (ragged lengths) and row block, and the last row blocks, the longest under a causal mask, start first.
  const int bh = a.splits > 1 ? blockIdx.x / a.splits : blockIdx.x, split = blockIdx.x - bh * a.splits;
  const int tile = gridDim.y - 1 - blockIdx.y;
  const int b = bh / a.hk, kh = bh - b * a.hk;
  const int row = tile * 32 * NW + wid * 32 + (lane & 31);
  const AtRow pr = at_packed(a, kh, row < rows ? row : 0);
  const int qi = pr.qi, head = pr.head;
  AtSpan sp = row < rows ? at_span(a, b, qi) : AtSpan{0, 0, 0};
  const bool live = sp.hi > sp.lo;
  const AtBounds w = at_bounds(a, b, kh, tile * 32 * NW + wid * 32, rows, sp);
  const int w_lo = w.lo, w_hi = w.hi, i_lo = w.i_lo;
  int i_hi = w.i_hi;
  int k_lo = w_lo, k_hi = w_hi;
  if constexpr (NW > 1) {
    if (a.spans) {
      if (lane == 0) range[wid] = w_lo, range[NW + wid] = w_hi;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NW; ++i) k_lo = min(k_lo, range[i]), k_hi = max(k_hi, range[NW + i]);
      k_lo = __builtin_amdgcn_readfirstlane(k_lo);
      k_hi = __builtin_amdgcn_readfirstlane(k_hi);
    } else {
      k_lo = 0;
      k_hi = __builtin_amdgcn_readfirstlane(
          max(at_span(a, b, at_packed(a, kh, min(tile * 32 * NW + 32 * NW, rows) - 1).qi).hi, 0));
    }
  }
  if (a.splits > 1) {
    k_lo = max(k_lo, split * a.chunk);
    k_hi = (int)min((long long)k_hi, (long long)(split + 1) * a.chunk);
    if (k_lo >= k_hi) return;
    sp.hi = min(sp.hi, k_hi);  // (a tile that starts off the chunk's grid may reach past its end)
    i_hi = min(i_hi, k_hi);
  }
  const T* kb = (const T*)a.k + b * a.k_sb + kh * a.k_sh;
  const T* vb = (const T*)a.v + b * a.v_sb + kh * a.v_sh;
  const T* qb = (const T*)a.q + b * a.q_sb + (long long)qi * a.q_sl + head * a.q_sh;
  const float slope = SLOPE ? at_slope<T>(a, head) / (!CAP && sizeof(T) == 2 ? a.sc.scale_u : 1.f) : 0.f;
  const unsigned lds0 = (unsigned)(uintptr_t)((__attribute__((address_space(3))) char*)smem);

  const AtLoad<T, DP, KT, NW> kl(a.k_sl, a.d, wid, lane), vl(a.v_sl, a.d, wid, lane);
  auto issue = [&](int stage, int k0) {
    const unsigned S = lds0 + (grp * 2 + stage) * STAGE;
    kl.issue(kb, k0, k_hi, S, wid);
    vl.issue(vb, k0, k_hi, S + TILE, wid);
  };
  const int nt = k_hi > k_lo ? (k_hi - k_lo + KT - 1) / KT : 0;
  if (grp < nt) issue(0, k_lo + grp * KT);  // (first: the rest of the set-up runs under its latency)
  uint4 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int e = (2 * ks + h) * AtT<T>::CH;
    qf[ks] = live && e < a.d ? *(const uint4*)(qb + e) : make_uint4(0, 0, 0, 0);
  }
  at_f32x16 acc[FD];
#pragma unroll
  for (int f = 0; f < FD; ++f) acc[f] = at_zero();
  // ms: m (0 while there is none) less the lift; the sum that o is divided by: l, of the probabilities as the products take them
  // (rounded: then the rounding of a dominant key cancels), or lx, of the unrounded ones, where their rest is taken too
  float m = -INFINITY, ms = 0.f, l = 0.f, lx = 0.f;
  const AtOffsets<T, DF> off(lane);
  // uncapped 16-bit scores stay raw, a bias divided by the scale, and are scaled in the exponent's FMA (scale > 0); others
  // become s in units U in place
  constexpr bool RAW = !CAP && sizeof(T) == 2;
  // capped 16-bit scores without a bias stay raw too: tanh does not change their order, so the maximum is taken of the raw
  // products and bent alone
  constexpr bool LATE = CAP && !SLOPE && sizeof(T) == 2;
  const char* const base = smem + grp * 2 * STAGE;
  auto step = [&](auto stage, auto again, int t) {  // tile t of all, or none (t >= nt: a group that has run out keeps the barriers)
    const int k0 = k_lo + t * KT;
    // this tile has landed (in every wave: the barrier); the other stage's last readers are past it too
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + NG < nt) issue(1 - stage, k0 + NG * KT);
    if (t >= nt || k0 >= w_hi || k0 + KT <= w_lo) return;  // (wave-uniform) nothing here for these rows
    const char* K = base + stage * STAGE;
    const char* V = K + TILE;
    at_f32x16 s[KF];
#pragma unroll
    for (int f = 0; f < KF; ++f) {
      s[f] = at_zero();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[f] = at_mfma<T>(at_row<T, DF>(K, off, 32 * f, ks), qf[ks], s[f]);
    }
    if constexpr (!RAW && !LATE) at_bend_tiles<T, CAP, KF>(a.sc, s);
    if constexpr (SLOPE) {
      const float x0 = (float)(sp.at - k0 - 4 * h);  // position minus this lane's first key
#pragma unroll
      for (int f = 0; f < KF; ++f)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[f][i] = fmaf(-slope, fabsf(x0 - (float)(32 * f + 8 * (i >> 2) + (i & 3))), s[f][i]);
    }
    const bool part = k0 < i_lo || k0 + KT > i_hi;  // (wave-uniform) some row does not see the whole tile
    const int lo = sp.lo - k0 - 4 * h, hi = sp.hi - k0 - 4 * h;
    float big = 0.f, mt = -INFINITY;
    if constexpr (LATE) {
#pragma unroll
      for (int f = 0; f < KF; ++f)
#pragma unroll
        for (int i = 0; i < 16; ++i) big = fmaxf(big, fabsf(s[f][i]));
    }
    if (part) {
#pragma unroll
      for (int f = 0; f < KF; ++f)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = 32 * f + 8 * (i >> 2) + (i & 3);
          const float x = j < lo || j >= hi ? -INFINITY : s[f][i];
          if constexpr (!LATE) s[f][i] = x;
          mt = fmaxf(mt, x);
        }
    } else {
#pragma unroll
      for (int f = 0; f < KF; ++f)
#pragma unroll
        for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[f][i]);
    }
    mt = at_half_max(mt);
    if (RAW) mt *= a.sc.scale_u;
    // (-inf may be a product too, whose score is -cap: only a row that sees none of the tile has no maximum)
    // (and bent as the tile's scores will be: under a large cap the forms differ by more than the lag)
    const int form = LATE ? at_form(a.sc, big * a.sc.scale_cap) : AT_ANY;
    if constexpr (LATE) {
      at_by_form(form, [&](auto of) { mt = at_bent<T, CAP, of.value>(a.sc, mt); });
      if (sp.hi <= k0 || sp.lo >= k0 + KT) mt = -INFINITY;
    }
    if (__any(mt > m + 8.f * AtUnit<T>::U / AT_LOG2E)) {
      const float mn = fmaxf(m, mt);
      ms = mn == -INFINITY ? 0.f : mn;
      const float alpha = at_exp<T>(m - ms);
      m = mn;
      ms -= AtLift<T>::FWD;
      l *= alpha;
      lx *= alpha;
#pragma unroll
      for (int f = 0; f < FD; ++f) acc[f] *= alpha;
    }
    if constexpr (LATE) {
      at_by_form(form, [&](auto of) {
#pragma unroll
        for (int f = 0; f < KF; ++f)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if constexpr (of.value == AT_ANY)
              s[f][i] = at_exp<T>(at_bent<T, CAP, AT_ANY>(a.sc, s[f][i]) - ms);
            else  // the polynomial's last product and the subtraction in one FMA
              s[f][i] = at_exp<T>(fmaf(s[f][i], at_poly<of.value>(a.sc, s[f][i] * s[f][i]), -ms));
          }
      });
      if (part) {
        int lo2 = lo, hi2 = hi;  // (opaque: the comparisons above would be kept for here, two scalar registers each)
        asm volatile("" : "+v"(lo2), "+v"(hi2));
#pragma unroll
        for (int f = 0; f < KF; ++f)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int j = 32 * f + 8 * (i >> 2) + (i & 3);
            s[f][i] = j < lo2 || j >= hi2 ? 0.f : s[f][i];
          }
      }
    } else {
#pragma unroll
      for (int f = 0; f < KF; ++f)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[f][i] = at_exp<T>(RAW ? fmaf(s[f][i], a.sc.scale_u, -ms) : s[f][i] - ms);
    }
#pragma unroll
    for (int f = 0; f < KF; ++f) {
      const float* p = (const float*)&s[f];
      // p is rounded to the 16-bit operand type: half a step, random in sign over the keys. For a backward what that leaves
      // is multiplied too: its delta = do.o stands for sum_j p dp, and an error of o would pass into dS through whole rows
      // (dq's error against 64 bits 1.47 to 1.52 times a rounding's instead of 1.42).
      const AtP<T> pk(p);
      if constexpr (again.value)
        if (part && at_has_nonfinite<T, DF>(V, 32 * f, lane)) {
          float w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            w[i] = sizeof(T) == 4 || TRAIN ? p[i] : Cvt<T>::load(Cvt<T>::store(p[i]));
            (sizeof(T) == 4 || TRAIN ? lx : l) += w[i];
          }
          at_accumulate_seen<T, DF>(V, 32 * f, w, acc, lane,
                                    [&](int r) { return k0 + 32 * f + r >= sp.lo && k0 + 32 * f + r < sp.hi; });
          continue;
        }
      if constexpr (sizeof(T) == 2) {
        if constexpr (TRAIN) {
#pragma unroll
          for (int i = 0; i < 16; ++i) lx += p[i];
          const AtP<T> rest(p, pk);
          at_accumulate<T, DF, true>(V, off, 32 * f, pk, acc, lane, &rest);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) l = AtPair<T>::add(pk.w[i], l);
          at_accumulate<T, DF>(V, off, 32 * f, pk, acc, lane);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) lx += p[i];
        at_accumulate<T, DF>(V, off, 32 * f, pk, acc, lane);
      }
    }
  };
  auto walk = [&](auto again) {
    if constexpr (again.value) {  // (one copy of the code: its stages need not be constants)
#pragma unroll 1
      for (int t = 0, s = 0; t < nt; t += NG, s ^= 1) step(s, again, t + grp);
    } else {
      for (int t = 0; t < nt; t += 2 * NG) {
        step(std::integral_constant<int, 0>{}, again, t + grp);
        if (t + NG < nt) step(std::integral_constant<int, 1>{}, again, t + NG + grp);
      }
    }
  };
  walk(std::false_type{});
  if (a.causal || a.spans) {
    // (a row whose sum is NaN saw a score of NaN)
    const bool bad = (at_bad_columns<FD>(acc) & ~at_columns(!live || (l + lx) != (l + lx))) != 0;
    if (at_vote(bad, &again_flag)) {
      m = -INFINITY, ms = l = lx = 0.f;
#pragma unroll
      for (int f = 0; f < FD; ++f) acc[f] = at_zero();
      if (grp < nt) issue(0, k_lo + grp * KT);
      walk(std::true_type{});
    }
  }
  lx = at_half_sum(lx);
  l = sizeof(T) == 4 || TRAIN ? lx : at_half_sum(l);
  if constexpr (NG > 1) {  // the second group's maxima, sums and accumulators through LDS
    float* part = (float*)smem + wid * 64 * (DF / 2 + 3) + lane;
    __syncthreads();
    if (grp == 1) {
      part[0] = m, part[64] = l, part[128] = lx;
#pragma unroll
      for (int f = 0; f < FD; ++f)
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(16 * f + i + 3) * 64] = acc[f][i];
    }
    __syncthreads();
    if (grp == 1) return;
    const float m1 = part[0], mn = fmaxf(m, m1);
    ms = mn == -INFINITY ? 0.f : mn;
    const float w0 = at_exp<T>(m - ms), w1 = at_exp<T>(m1 - ms);
    m = mn;
    ms -= AtLift<T>::FWD;
    l = l * w0 + part[64] * w1;
    lx = lx * w0 + part[128] * w1;
#pragma unroll
    for (int f = 0; f < FD; ++f)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[f][i] = acc[f][i] * w0 + part[(16 * f + i + 3) * 64] * w1;
  }
  const long long prow = ((long long)split * nbh + bh) * rows + row;  // partials
  T* ob = (T*)a.o + (((long long)b * a.lq + qi) * a.hq + head) * a.d;
  T* olo = TRAIN ? (T*)a.o_lo + (((long long)b * a.lq + qi) * a.hq + head) * a.d : nullptr;
  const bool mine = row < rows;
  if (a.splits > 1) {
    if (mine) {
      float* po = a.po + prow * a.d;
#pragma unroll
      for (int f = 0; f < FD; ++f)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int e = 32 * f + 8 * g + 4 * h;
          if (e < a.d) *(float4*)(po + e) = make_float4(acc[f][4 * g], acc[f][4 * g + 1], acc[f][4 * g + 2], acc[f][4 * g + 3]);
        }
      if (h == 0) *(float4*)(a.pml + 4 * prow) = make_float4(m, l, lx, 0.f);
    }
  } else {
    if (!live) {
#pragma unroll
      for (int f = 0; f < FD; ++f) acc[f] = at_zero();
    }
    at_store_row<T, DF, TRAIN>(ob, acc, a.d, h, live ? 1.f / l : 0.f, mine, olo);
    if (a.lse && mine && h == 0) a.lse[((long long)b * a.hq + head) * a.lq + qi] = live ? ms + at_log<T>(lx) : INFINITY;
  }
}

// o of one packed row from its splits: sum exp(m_s - m) O_s / sum exp(m_s - m) l_s over the splits its span touches.
// G groups of 32 lanes (four dims a lane) per row take every G-th split and are added up through LDS in a fixed order:
// 8 for few rows of many splits, 1 for many rows.
template <typename T, int G>
__global__ void __launch_bounds__(256) k_mattn_join(AtArgs a) {
  __shared__ float4 part[8][32];
  __shared__ float sums[8][2];
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, nbh = a.batch * a.hk, rows = a.lq * a.group;
  const long long r0 = (long long)blockIdx.x * (8 / G) + grp / G, step = (long long)nbh * rows;  // r0 = bh * rows + row
  const int g = grp % G;
  const bool on = 4 * lane < a.d, in = r0 < step;
  const int bh = in ? (int)(r0 / rows) : 0, row = in ? (int)(r0 - (long long)bh * rows) : 0;
  const int b = bh / a.hk, kh = bh - b * a.hk;
  const AtRow pr = at_packed(a, kh, row);
  const AtSpan sp = at_span(a, b, pr.qi);
  const bool live = in && sp.hi > sp.lo;
  const int s0 = sp.lo / a.chunk, s1 = live ? (sp.hi - 1) / a.chunk + 1 : s0;
  float m = -INFINITY;
  for (int s = s0 + lane; s < s1; s += 32) m = fmaxf(m, a.pml[4 * (s * step + r0)]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float ms = m == -INFINITY ? 0.f : m;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f, lx = 0.f;
#pragma unroll 4
  for (int s = s0 + g; s < s1; s += G) {
    const long long at = s * step + r0;
    const float4 ml = *(const float4*)(a.pml + 4 * at);
    const float4 x = on ? *(const float4*)(a.po + at * a.d + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
    // (a split whose keys are all -inf for this row has w = 0 and finite sums)
    const float w = at_exp<T>(ml.x - ms);
    l = fmaf(w, ml.y, l);
    lx = fmaf(w, ml.z, lx);
    o.x = fmaf(w, x.x, o.x), o.y = fmaf(w, x.y, o.y), o.z = fmaf(w, x.z, o.z), o.w = fmaf(w, x.w, o.w);
  }
  if constexpr (G > 1) {
    part[grp][lane] = o;
    if (lane == 0) sums[grp][0] = l, sums[grp][1] = lx;
    __syncthreads();
    if (g != 0) return;
    for (int k = 1; k < G; ++k) {
      const float4 x = part[grp + k][lane];
      o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
      l += sums[grp + k][0], lx += sums[grp + k][1];
    }
  }
  if (!in) return;
  if (a.lse && lane == 0) a.lse[((long long)b * a.hq + pr.head) * a.lq + pr.qi] = live ? ms - AtLift<T>::FWD + at_log<T>(lx) : INFINITY;
  if (!on) return;
  const long long orow = (((long long)b * a.lq + pr.qi) * a.hq + pr.head) * a.d + 4 * lane;
  const float inv = live ? 1.f / l : 0.f;
  float v[4] = {live ? o.x * inv : 0.f, live ? o.y * inv : 0.f, live ? o.z * inv : 0.f, live ? o.w * inv : 0.f};
  at_store4((T*)a.o + orow, v);
  if (a.o_lo) {
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] -= Cvt<T>::load(Cvt<T>::store(v[r]));
    at_store4((T*)a.o_lo + orow, v);
  }
}

template <typename T, int DF, bool CAP, bool SLOPE, bool TRAIN>
static int mattn_fwd_df(const AtArgs& a, AtPlan p, hipStream_t stream) {
  constexpr int RB = AtPad<DF>::DP * AtT<T>::E;
  constexpr int KT = sizeof(T) == 4 ? 32 : 64;  // f32 rows are twice as wide: the same LDS for half the keys
  constexpr size_t LDS = 4 * KT * RB;
  const int rows = a.lq * a.group, nbh = a.batch * a.hk;
  const dim3 grid((unsigned)(nbh * a.splits), (unsigned)cdiv(rows, 32 * p.nw));
  if (p.nw == 1)
    hipLaunchKernelGGL((k_mattn_fwd<T, DF, CAP, SLOPE, TRAIN, 1, 1, 32>), grid, dim3(64), 4 * 32 * RB, stream, a);
  else if (p.nw == 3)
    hipLaunchKernelGGL((k_mattn_fwd<T, DF, CAP, SLOPE, TRAIN, 3, 1, 32>), grid, dim3(192), 4 * 32 * RB, stream, a);
  else if (sizeof(T) == 2 && p.three)
    hipLaunchKernelGGL((k_mattn_fwd<T, DF, CAP, SLOPE, TRAIN, 4, 1, 32>), grid, dim3(256), 4 * 32 * RB, stream, a);
  else if (p.ng == 1)
    hipLaunchKernelGGL((k_mattn_fwd<T, DF, CAP, SLOPE, TRAIN, 4, 1, KT>), grid, dim3(256), LDS, stream, a);
  else if constexpr (sizeof(T) == 4)  // (16-bit workgroups of 8 waves lose: two of 4 overlap better)
    hipLaunchKernelGGL((k_mattn_fwd<T, DF, CAP, SLOPE, TRAIN, 4, 2, KT>), grid, dim3(512), 2 * LDS, stream, a);
  DMF_LAUNCH_CHECK("dmf_mattn_fwd");
  return 0;
}
template <typename T, int DF, bool CAP, bool SLOPE>
static int mattn_fwd_train(const AtArgs& a, AtPlan p, hipStream_t stream) {
  // (f32 keeps no o_lo: one kernel for both)
  if constexpr (sizeof(T) == 2)
    if (a.o_lo) return mattn_fwd_df<T, DF, CAP, SLOPE, true>(a, p, stream);
  return mattn_fwd_df<T, DF, CAP, SLOPE, false>(a, p, stream);
}

template <typename T>
static int mattn_fwd_t(AtArgs a, AtPlan p, hipStream_t stream) {
  at_score_args<T>(a);
  int rc = 0;
#define DMF_AT_MODE(DF)                                                                  \
  rc = a.cap > 0.f ? (a.slopes ? mattn_fwd_train<T, DF, true, true>(a, p, stream)          \
                               : mattn_fwd_train<T, DF, true, false>(a, p, stream))        \
                   : (a.slopes ? mattn_fwd_train<T, DF, false, true>(a, p, stream)         \
                               : mattn_fwd_train<T, DF, false, false>(a, p, stream))
  if (a.d <= 32) DMF_AT_MODE(32);
  else if (a.d <= 64) DMF_AT_MODE(64);
  else if (a.d <= 96) DMF_AT_MODE(96);
  else DMF_AT_MODE(128);
#undef DMF_AT_MODE
  if (rc) return rc;
  if (a.splits > 1) {
    const long long n = (long long)a.lq * a.group * a.batch * a.hk;
    if (n >= 4096)
      hipLaunchKernelGGL((k_mattn_join<T, 1>), dim3((unsigned)((n + 7) / 8)), dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((k_mattn_join<T, 8>), dim3((unsigned)n), dim3(256), 0, stream, a);
    DMF_LAUNCH_CHECK("dmf_mattn_fwd (join)");
  }
  return 0;
}

}  // namespace dmf
