// Per-head RMS norm of queries and keys with the position rotation in the same pass, and its gradient
// (the step between a token block's qkv projection and its attention, transformer_model.py:100-116).
//
//   y = rot(x * r * w),  r = rsqrt(mean(x^2) + eps) over the D elements of one head
//   rot turns pair p of the first `rot` dims by the table's (cos, sin)[pos][p]; the pair is dims
//   (p, p + rot/2) or, interleaved, (2p, 2p + 1); dims >= rot pass through
//   gradient: g = rot^T dy, xh = x r:  dw = sum g xh,  dx = r (g w - xh mean(g w xh))
//
// Bound: HBM (x in, y out; the tables and weights are read once per group of heads). All arithmetic is f32
// and a value is rounded once, on its store. Measured, bf16, 128 dims, against the 4.9 TB/s of a large copy: 2 x 8192
// tokens, 32 + 8 heads: forward 70 us (4.8 TB/s), backward 122 us (4.1 TB/s) and 5 us to sum the weight gradients' partials;
// 32 x 576 tokens, 4 + 4 heads out of packed rows: forward 15 us (5.0 TB/s).
//
// Layout: a row (one head of one token) is held by G lanes, each with "units" of 2 V elements: V of each half of a
// pair block (or 2 V consecutive ones, interleaved and in the unrotated tail), so a rotation never leaves its lane,
// the loads are 16 B, and the row sum is log2 G shuffles. A lane group keeps its token's cos / sin (V floats each per
// unit, twice the bytes of a 16-bit row) in registers over up to HPG heads; those are chosen so that the launch still
// has enough groups to fill the card.
#include "dmf_common.h"

namespace dmf {

// V elements of T at p (aligned to min(16, V * sizeof(T)) bytes) <-> floats
template <typename T, int V> struct QkVec;
template <typename T> struct QkVec<T, 8> {
  __device__ __forceinline__ static void load(const T* p, float* v) { ld8(p, v); }
  __device__ __forceinline__ static void store(T* p, const float* v) { st8(p, v); }
};
template <typename T> struct QkVec<T, 4> {
  __device__ __forceinline__ static void load(const T* p, float* v) {
    if constexpr (sizeof(T) == 4) {
      const float4 u = *(const float4*)p;
      v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    } else {
      const uint2 u = *(const uint2*)p;
      v[0] = B16<T>::lo(u.x); v[1] = B16<T>::hi(u.x); v[2] = B16<T>::lo(u.y); v[3] = B16<T>::hi(u.y);
    }
  }
  __device__ __forceinline__ static void store(T* p, const float* v) {
    if constexpr (sizeof(T) == 4)
      *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
    else
      *(uint2*)p = make_uint2(B16<T>::pack(v[0], v[1]), B16<T>::pack(v[2], v[3]));
  }
};
template <typename T> struct QkVec<T, 1> {
  __device__ __forceinline__ static void load(const T* p, float* v) { v[0] = ld(p); }
  __device__ __forceinline__ static void store(T* p, const float* v) { st(p, v[0]); }
};

struct QkSide {           // queries or keys
  const void* x;          // element (b, l, h, i) at b sb + l sl + h sh + i
  long long sb, sl, sh;
  const float* w;         // [d], null: ones
  void* y;                // [tokens][heads][d]: forward output, or dx
  const void* dy;         // [tokens][heads][d] (backward)
  int heads, chunks;      // chunks = ceil(heads / hpg)
};
struct QkArgs {
  QkSide s[2];
  int tokens, len, d, rot, norm, hpg, lg;  // lg: log2 of the lanes per row
  float eps;
  const float* cs;        // [rows][rot/2]
  const float* sn;
  const void* pos;        // null: the token's index in its sequence
  long long pos_sb;
  int pos64;
  long long rows;
  float* part;            // backward: [gridDim.x][2][d] weight-gradient partials, null without weights
};

// offset of the two V-element halves of unit u
template <int V, bool INTER>
__device__ __forceinline__ void qk_unit(const QkArgs& a, int u, int& oa, int& ob) {
  const int ur = a.rot / (2 * V);  // rotated units
  if (!INTER && u < ur) {
    oa = u * V;
    ob = a.rot / 2 + u * V;
  } else {
    oa = u * 2 * V;
    ob = oa + V;
  }
}

// cos / sin of a token's position for one unit; a position outside the table makes the row NaN
template <int V>
__device__ __forceinline__ void qk_angles(const QkArgs& a, int b, int l, int u, float* c, float* s) {
  if (u * 2 * V >= a.rot) {
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = 1.f, s[i] = 0.f;
    return;
  }
  long long p = l;
  if (a.pos)
    p = a.pos64 ? ((const long long*)a.pos)[b * a.pos_sb + l] : (long long)((const int*)a.pos)[b * a.pos_sb + l];
  if (p < 0 || p >= a.rows) {
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = s[i] = __builtin_nanf("");
    return;
  }
  const long long o = p * (a.rot / 2) + u * V;
  QkVec<float, V>::load(a.cs + o, c);
  QkVec<float, V>::load(a.sn + o, s);
}

template <int V, bool INTER, bool BACK>
__device__ __forceinline__ void qk_turn(float* x, const float* c, const float* s) {  // x[0..V), x[V..2V)
  if constexpr (INTER && V > 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float p = x[2 * i], q = x[2 * i + 1], sn = BACK ? -s[i] : s[i];
      x[2 * i] = p * c[i] - q * sn;
      x[2 * i + 1] = q * c[i] + p * sn;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float p = x[i], q = x[V + i], sn = BACK ? -s[i] : s[i];
      x[i] = p * c[i] - q * sn;
      x[V + i] = q * c[i] + p * sn;
    }
  }
}

__device__ __forceinline__ float qk_group_sum(float v, int lg) {
  for (int o = 1; o < (1 << lg); o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// NU units per lane (4 only with V = 1, for head dims over 128), NB rows in flight per lane group
template <typename T, int V, bool INTER, int NU, int NB>
__global__ void __launch_bounds__(256) k_qk_norm_rope(QkArgs a) {
  const int lane = threadIdx.x & ((1 << a.lg) - 1);
  const int tok = blockIdx.x * (256 >> a.lg) + (threadIdx.x >> a.lg);
  const int side = blockIdx.y >= (unsigned)a.s[0].chunks;
  const QkSide& q = a.s[side];
  const int h0 = (blockIdx.y - (side ? a.s[0].chunks : 0)) * a.hpg, h1 = min(h0 + a.hpg, q.heads);
  const bool live = tok < a.tokens;
  const int tk = live ? tok : 0, b = tk / a.len, l = tk - b * a.len;
  const T* x = (const T*)q.x + b * q.sb + l * q.sl;
  T* y = (T*)q.y + (long long)tk * q.heads * a.d;
  int oa[NU], ob[NU];
  bool on[NU];
  float c[NU][V], s[NU][V], w[NU][2 * V];
#pragma unroll
  for (int n = 0; n < NU; ++n) {
    const int u = lane + (n << a.lg);
    on[n] = live && u * 2 * V < a.d;
    qk_unit<V, INTER>(a, u, oa[n], ob[n]);
    if (!on[n]) {
      oa[n] = ob[n] = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) c[n][i] = 1.f, s[n][i] = 0.f, w[n][i] = w[n][V + i] = 1.f;
      continue;
    }
    qk_angles<V>(a, b, l, u, c[n], s[n]);
    if (q.w) {
      QkVec<float, V>::load(q.w + oa[n], w[n]);
      QkVec<float, V>::load(q.w + ob[n], w[n] + V);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) w[n][i] = 1.f;
    }
  }
  for (int h = h0; h < h1; h += NB) {
    float v[NB][NU][2 * V];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        if (on[n] && h + j < h1) {
          QkVec<T, V>::load(x + (h + j) * q.sh + oa[n], v[j][n]);
          QkVec<T, V>::load(x + (h + j) * q.sh + ob[n], v[j][n] + V);
        } else {
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) v[j][n][i] = 0.f;
        }
      }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      float r = 1.f;
      if (a.norm) {
        float ss = 0.f;
#pragma unroll
        for (int n = 0; n < NU; ++n)
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) ss = fmaf(v[j][n][i], v[j][n][i], ss);
        r = rsqrtf(qk_group_sum(ss, a.lg) / (float)a.d + a.eps);
      }
#pragma unroll
      for (int n = 0; n < NU; ++n) {
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) v[j][n][i] *= r * w[n][i];
        qk_turn<V, INTER, false>(v[j][n], c[n], s[n]);
        if (on[n] && h + j < h1) {
          QkVec<T, V>::store(y + (long long)(h + j) * a.d + oa[n], v[j][n]);
          QkVec<T, V>::store(y + (long long)(h + j) * a.d + ob[n], v[j][n] + V);
        }
      }
    }
  }
}

// Backward: the same mapping, the token blocks walked with a grid stride so that a workgroup leaves one weight-gradient
// partial per side; a lane sums its dims over its heads and tokens in f32, the groups of the block are added in a fixed
// order through LDS, and k_qk_dw adds the blocks' partials in a fixed order (no atomics: the same bits every run).
template <typename T, int V, bool INTER, int NU, int NB>
__global__ void __launch_bounds__(256) k_qk_norm_rope_bwd(QkArgs a) {
  extern __shared__ float red[];  // [256 >> lg][d]
  const int lane = threadIdx.x & ((1 << a.lg) - 1), grp = threadIdx.x >> a.lg, ngrp = 256 >> a.lg;
  const int side = blockIdx.y >= (unsigned)a.s[0].chunks;
  const QkSide& q = a.s[side];
  const int h0 = (blockIdx.y - (side ? a.s[0].chunks : 0)) * a.hpg, h1 = min(h0 + a.hpg, q.heads);
  int oa[NU], ob[NU];
  bool in[NU];
  float w[NU][2 * V], dw[NU][2 * V];
#pragma unroll
  for (int n = 0; n < NU; ++n) {
    const int u = lane + (n << a.lg);
    in[n] = u * 2 * V < a.d;
    qk_unit<V, INTER>(a, u, oa[n], ob[n]);
    if (!in[n]) oa[n] = ob[n] = 0;
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) w[n][i] = 1.f, dw[n][i] = 0.f;
    if (q.w && in[n]) {
      QkVec<float, V>::load(q.w + oa[n], w[n]);
      QkVec<float, V>::load(q.w + ob[n], w[n] + V);
    }
  }
  for (long long t0 = (long long)blockIdx.x * ngrp; t0 < a.tokens; t0 += (long long)gridDim.x * ngrp) {
    const bool live = t0 + grp < a.tokens;
    const int tk = live ? (int)(t0 + grp) : 0, b = tk / a.len, l = tk - b * a.len;
    const T* x = (const T*)q.x + b * q.sb + l * q.sl;
    const T* dy = (const T*)q.dy + (long long)tk * q.heads * a.d;
    T* dx = (T*)q.y + (long long)tk * q.heads * a.d;
    float c[NU][V], s[NU][V];
    bool on[NU];
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      on[n] = live && in[n];
      if (on[n])
        qk_angles<V>(a, b, l, lane + (n << a.lg), c[n], s[n]);
      else
#pragma unroll
        for (int i = 0; i < V; ++i) c[n][i] = 1.f, s[n][i] = 0.f;
    }
    for (int h = h0; h < h1; h += NB) {
      float v[NB][NU][2 * V], g[NB][NU][2 * V];
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int n = 0; n < NU; ++n) {
          if (on[n] && h + j < h1) {
            QkVec<T, V>::load(x + (h + j) * q.sh + oa[n], v[j][n]);
            QkVec<T, V>::load(x + (h + j) * q.sh + ob[n], v[j][n] + V);
            QkVec<T, V>::load(dy + (long long)(h + j) * a.d + oa[n], g[j][n]);
            QkVec<T, V>::load(dy + (long long)(h + j) * a.d + ob[n], g[j][n] + V);
          } else {
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) v[j][n][i] = g[j][n][i] = 0.f;
          }
        }
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        float r = 1.f, mean = 0.f;
        if (a.norm) {
          float ss = 0.f;
#pragma unroll
          for (int n = 0; n < NU; ++n)
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) ss = fmaf(v[j][n][i], v[j][n][i], ss);
          // (rows that are not there are zeros: without an eps their r would be infinite, and 0 * r would enter dw)
          ss = qk_group_sum(ss, a.lg) / (float)a.d + a.eps;
          r = live && h + j < h1 ? rsqrtf(ss) : 0.f;
        }
#pragma unroll
        for (int n = 0; n < NU; ++n) {
          qk_turn<V, INTER, true>(g[j][n], c[n], s[n]);
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) {
            v[j][n][i] *= r;
            dw[n][i] = fmaf(g[j][n][i], v[j][n][i], dw[n][i]);
            g[j][n][i] *= w[n][i];
            mean = fmaf(g[j][n][i], v[j][n][i], mean);
          }
        }
        if (a.norm) mean = qk_group_sum(mean, a.lg) / (float)a.d;
#pragma unroll
        for (int n = 0; n < NU; ++n) {
          if (a.norm) {
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) g[j][n][i] = r * fmaf(-v[j][n][i], mean, g[j][n][i]);
          }
          if (on[n] && h + j < h1) {
            QkVec<T, V>::store(dx + (long long)(h + j) * a.d + oa[n], g[j][n]);
            QkVec<T, V>::store(dx + (long long)(h + j) * a.d + ob[n], g[j][n] + V);
          }
        }
      }
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int n = 0; n < NU; ++n)
    if (in[n]) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        red[grp * a.d + oa[n] + i] = dw[n][i];
        red[grp * a.d + ob[n] + i] = dw[n][V + i];
      }
    }
  __syncthreads();
  float* part = a.part + ((long long)blockIdx.y * gridDim.x + blockIdx.x) * a.d;
  for (int i = threadIdx.x; i < a.d; i += 256) {
    float t = 0.f;
    for (int k = 0; k < ngrp; ++k) t += red[k * a.d + i];
    part[i] = t;
  }
}

// dw of side blockIdx.y: the sum over its (head chunk, block) partials; 16 columns x 64 row lanes
__global__ void __launch_bounds__(1024) k_qk_dw(const float* part, int d, long long rows0, long long rows1, float* dwq,
                                                float* dwk) {
  __shared__ float red[64][17];
  const int col = blockIdx.x * 16 + (threadIdx.x & 15), rl = threadIdx.x >> 4;
  const long long first = blockIdx.y ? rows0 : 0, n = blockIdx.y ? rows1 : rows0;
  float t = 0.f;
  if (col < d)
    for (long long r = rl; r < n; r += 64) t += part[(first + r) * d + col];
  red[rl][threadIdx.x & 15] = t;
  __syncthreads();
  if (rl == 0 && col < d) {
    t = 0.f;
    for (int k = 0; k < 64; ++k) t += red[k][threadIdx.x & 15];
    (blockIdx.y ? dwk : dwq)[col] = t;
  }
}

constexpr int QK_BWD_BLOCKS = 1024;  // most workgroups along the tokens in the backward

struct QkPlan {
  int v, nu, lg;
};
static bool qk_aligned(const void* p, int bytes) { return (uintptr_t)p % bytes == 0; }
// the widest V whose units tile the head and whose loads are aligned in every operand
static QkPlan qk_plan(const QkArgs& a, int dtype) {
  const int e = dtype == DMF_F32 ? 4 : 2;
  for (int v = 8; v > 1; v /= 2) {
    if (v == 2) continue;
    const int al = v * e > 16 ? 16 : v * e;
    bool ok = (a.rot / 2) % v == 0 && (a.d - a.rot) % (2 * v) == 0 && a.d / (2 * v) <= 64;
    for (int i = 0; i < 2; ++i) {
      const QkSide& s = a.s[i];
      ok = ok && qk_aligned(s.x, al) && s.sb * e % al == 0 && s.sl * e % al == 0 && s.sh * e % al == 0 &&
           qk_aligned(s.y, al) && qk_aligned(s.dy, al) && qk_aligned(s.w, 16) && a.d * e % al == 0;
    }
    ok = ok && qk_aligned(a.cs, 16) && qk_aligned(a.sn, 16);
    if (!ok) continue;
    int lg = 0;
    while ((1 << lg) < a.d / (2 * v)) ++lg;
    return {v, 1, lg};
  }
  int lg = 0;
  while (lg < 6 && (1 << lg) < a.d / 2) ++lg;
  return {1, a.d / 2 > 64 ? 4 : 1, lg};
}

static int qk_check(const char* who, const QkArgs& a, int dtype, int batch) {
  DMF_CHECK_ARG(dtype == DMF_F32 || dtype == DMF_BF16 || dtype == DMF_F16, "%s: dtype %d", who, dtype);
  DMF_CHECK_ARG(a.d >= 2 && a.d <= 512 && a.d % 2 == 0, "%s: head dim %d must be even and at most 512", who, a.d);
  DMF_CHECK_ARG(a.rot >= 0 && a.rot <= a.d && a.rot % 2 == 0, "%s: rotated dims %d must be even and at most the head dim %d",
                who, a.rot, a.d);
  DMF_CHECK_ARG(a.s[0].heads >= 1 && a.s[1].heads >= 1 && a.s[0].heads <= 4096 && a.s[1].heads <= 4096,
                "%s: heads %d / %d must be in 1..4096", who, a.s[0].heads, a.s[1].heads);
  DMF_CHECK_ARG(batch >= 0 && a.len >= 0 && (long long)batch * a.len < (1LL << 31), "%s: %d x %d tokens", who, batch,
                a.len);
  DMF_CHECK_ARG(a.rot == 0 || (a.cs && a.sn && a.rows >= 1), "%s: the rotation needs cos / sin tables", who);
  DMF_CHECK_ARG(a.rot == 0 || a.pos || a.rows >= a.len, "%s: the table has %lld rows for %d positions", who, a.rows,
                a.len);
  DMF_CHECK_ARG(a.norm || (!a.s[0].w && !a.s[1].w), "%s: weights without the norm", who);
  return 0;
}

// heads per lane group: as many as leave 16384 groups (8 waves on each CU at 8 rows a wave), so that the cos / sin
// loads are shared without leaving CUs idle; powers of two, in the forward up to the first that reaches the heads of the side
// with fewer (or 8), so that its groups do not end long before the others' (2 x 8192 tokens, 32 query and 8 key heads of 128,
// bf16: 32 heads a group 76 us, 16: 80, 8: 72, 4: 74). The backward's groups take several tokens each and leave a weight-gradient partial per chunk of heads: there
// more chunks lose (the same sizes: 122 + 5 us for the partials' sum against 130 + 6).
static void qk_split(QkArgs& a, long long tokens, bool even) {
  const int h0 = a.s[0].heads, h1 = a.s[1].heads, few = h0 < h1 ? h0 : h1;
  int most = h0 > h1 ? h0 : h1;
  if (even && most > few) most = few > 8 ? few : most < 8 ? most : 8;
  int hpg = 1;
  while (hpg < most && tokens * (a.s[0].heads + a.s[1].heads) >= 16384LL * 2 * hpg) hpg *= 2;
  a.hpg = hpg;
  for (int i = 0; i < 2; ++i) a.s[i].chunks = cdiv(a.s[i].heads, hpg);
}

#define DMF_QK_LAUNCH(KERNEL, GRID, LDS)                                                                              \
  do {                                                                                                                \
    if (p.v == 8) {                                                                                                   \
      if (interleaved) hipLaunchKernelGGL((KERNEL<T, 8, true, 1, 2>), GRID, dim3(256), LDS, (hipStream_t)stream, a);  \
      else hipLaunchKernelGGL((KERNEL<T, 8, false, 1, 2>), GRID, dim3(256), LDS, (hipStream_t)stream, a);             \
    } else if (p.v == 4) {                                                                                            \
      if (interleaved) hipLaunchKernelGGL((KERNEL<T, 4, true, 1, 2>), GRID, dim3(256), LDS, (hipStream_t)stream, a);  \
      else hipLaunchKernelGGL((KERNEL<T, 4, false, 1, 2>), GRID, dim3(256), LDS, (hipStream_t)stream, a);             \
    } else if (p.nu == 1) {                                                                                           \
      if (interleaved) hipLaunchKernelGGL((KERNEL<T, 1, true, 1, 2>), GRID, dim3(256), LDS, (hipStream_t)stream, a);  \
      else hipLaunchKernelGGL((KERNEL<T, 1, false, 1, 2>), GRID, dim3(256), LDS, (hipStream_t)stream, a);             \
    } else {                                                                                                          \
      if (interleaved) hipLaunchKernelGGL((KERNEL<T, 1, true, 4, 2>), GRID, dim3(256), LDS, (hipStream_t)stream, a);  \
      else hipLaunchKernelGGL((KERNEL<T, 1, false, 4, 2>), GRID, dim3(256), LDS, (hipStream_t)stream, a);             \
    }                                                                                                                 \
  } while (0)

static QkArgs qk_args(const void* q, long long qsb, long long qsl, long long qsh, int hq, const void* k, long long ksb,
                      long long ksl, long long ksh, int hk, int batch, int len, int d, int rot, int norm, float eps,
                      const float* wq, const float* wk, const float* cs, const float* sn, const void* pos,
                      long long pos_sb, int pos64, long long rows) {
  QkArgs a = {};
  a.s[0] = {q, qsb, qsl, qsh, wq, nullptr, nullptr, hq, 0};
  a.s[1] = {k, ksb, ksl, ksh, wk, nullptr, nullptr, hk, 0};
  a.tokens = batch * len;
  a.len = len, a.d = d, a.rot = rot, a.norm = norm, a.eps = eps;
  a.cs = cs, a.sn = sn, a.pos = pos, a.pos_sb = pos_sb, a.pos64 = pos64, a.rows = rows;
  return a;
}

}  // namespace dmf

using namespace dmf;

extern "C" int dmf_qk_norm_rope(int dtype, const void* q, long long q_sb, long long q_sl, long long q_sh, int hq,
                                const void* k, long long k_sb, long long k_sl, long long k_sh, int hk, int batch,
                                int len, int d, int rot, int interleaved, int norm, float eps, const float* wq,
                                const float* wk, const float* cos_t, const float* sin_t, const void* pos,
                                long long pos_sb, int pos64, long long table_rows, void* q_out, void* k_out,
                                void* stream) {
  QkArgs a = qk_args(q, q_sb, q_sl, q_sh, hq, k, k_sb, k_sl, k_sh, hk, batch, len, d, rot, norm, eps, wq, wk, cos_t,
                     sin_t, pos, pos_sb, pos64, table_rows);
  a.s[0].y = q_out, a.s[1].y = k_out;
  if (int rc = qk_check("dmf_qk_norm_rope", a, dtype, batch)) return rc;
  if (a.tokens == 0) return 0;
  DMF_CHECK_ARG(q && k && q_out && k_out, "dmf_qk_norm_rope: null operand");
  qk_split(a, a.tokens, true);
  const QkPlan p = qk_plan(a, dtype);
  a.lg = p.lg;
  const dim3 grid((unsigned)cdiv(a.tokens, 256 >> p.lg), (unsigned)(a.s[0].chunks + a.s[1].chunks));
  DMF_DISPATCH_DTYPE(dtype, T, DMF_QK_LAUNCH(k_qk_norm_rope, grid, 0));
  DMF_LAUNCH_CHECK("dmf_qk_norm_rope");
  return 0;
}

static int qk_bwd_blocks(long long tokens, int lg, int chunks) {
  const long long n = (tokens + (256 >> lg) - 1) / (256 >> lg);
  const long long most = QK_BWD_BLOCKS / chunks > 0 ? QK_BWD_BLOCKS / chunks : 1;
  return (int)(n < most ? n : most);
}

extern "C" long long dmf_qk_norm_rope_bwd_ws_floats(int hq, int hk, int d) {
  // partials [<= max(QK_BWD_BLOCKS, chunks)][d]
  const long long chunks = (long long)hq + hk;
  return (chunks > QK_BWD_BLOCKS ? chunks : QK_BWD_BLOCKS) * d;
}

extern "C" int dmf_qk_norm_rope_bwd(int dtype, const void* q, long long q_sb, long long q_sl, long long q_sh, int hq,
                                    const void* k, long long k_sb, long long k_sl, long long k_sh, int hk, int batch,
                                    int len, int d, int rot, int interleaved, int norm, float eps, const float* wq,
                                    const float* wk, const float* cos_t, const float* sin_t, const void* pos,
                                    long long pos_sb, int pos64, long long table_rows, const void* dq_out,
                                    const void* dk_out, void* dq, void* dk, float* dwq, float* dwk, float* ws,
                                    void* stream) {
  QkArgs a = qk_args(q, q_sb, q_sl, q_sh, hq, k, k_sb, k_sl, k_sh, hk, batch, len, d, rot, norm, eps, wq, wk, cos_t,
                     sin_t, pos, pos_sb, pos64, table_rows);
  a.s[0].y = dq, a.s[1].y = dk;
  a.s[0].dy = dq_out, a.s[1].dy = dk_out;
  if (int rc = qk_check("dmf_qk_norm_rope_bwd", a, dtype, batch)) return rc;
  DMF_CHECK_ARG((dwq != nullptr) == (dwk != nullptr) && (!dwq || (ws && norm)),
                "dmf_qk_norm_rope_bwd: weight gradients need both outputs, the norm and a workspace");
  if (a.tokens) DMF_CHECK_ARG(q && k && dq_out && dk_out && dq && dk, "dmf_qk_norm_rope_bwd: null operand");
  long long n0 = 0, n1 = 0;
  if (a.tokens) {
    a.part = dwq ? ws : nullptr;
    qk_split(a, a.tokens, false);
    const QkPlan p = qk_plan(a, dtype);
    a.lg = p.lg;
    const int chunks = a.s[0].chunks + a.s[1].chunks, nb = qk_bwd_blocks(a.tokens, p.lg, chunks);
    n0 = (long long)nb * a.s[0].chunks, n1 = (long long)nb * a.s[1].chunks;
    const dim3 grid((unsigned)nb, (unsigned)chunks);
    const size_t lds = dwq ? (size_t)(256 >> p.lg) * d * sizeof(float) : 0;
    DMF_DISPATCH_DTYPE(dtype, T, DMF_QK_LAUNCH(k_qk_norm_rope_bwd, grid, lds));
    DMF_LAUNCH_CHECK("dmf_qk_norm_rope_bwd");
  }
  if (dwq) {
    hipLaunchKernelGGL(k_qk_dw, dim3((unsigned)cdiv(d, 16), 2), dim3(1024), 0, (hipStream_t)stream, ws, d, n0, n1, dwq,
                       dwk);
    DMF_LAUNCH_CHECK("dmf_qk_norm_rope_bwd (weights)");
  }
  return 0;
}
