// Entry points of the masked attention (masked_attn.h): argument checks, the split of the keys, the spans of a
// document mask. The kernels are instantiated per storage type in masked_attn_{fwd,bwd}_{bf16,f16,f32}.hip.
#include "masked_attn.h"

namespace dmf {

int mattn_fwd_bf16(const AtArgs& a, AtPlan p, hipStream_t stream);
int mattn_fwd_f16(const AtArgs& a, AtPlan p, hipStream_t stream);
int mattn_fwd_f32(const AtArgs& a, AtPlan p, hipStream_t stream);
int mattn_bwd_bf16(const AtArgs& a, hipStream_t stream);
int mattn_bwd_f16(const AtArgs& a, hipStream_t stream);
int mattn_bwd_f32(const AtArgs& a, hipStream_t stream);

// Spans of a document mask: a document is a maximal run of equal ids >= 0 in the first kv_len positions; query i stands
// at position p = kv_len - lq + i and sees its document, under `causal` only up to itself or the document's first
// `prefix` tokens. One workgroup per 1024 positions and batch row: the run starts among them are bit masks (one ballot a
// wave), a run that enters from the left or leaves to the right is followed 1024 positions at a time.
template <typename I>
__global__ void __launch_bounds__(1024) k_mattn_spans(const I* __restrict__ docs, long long doc_sb,
                                                      const int* kv_lens, const int* prefix, int lq, int lk, int causal,
                                                      int2* __restrict__ spans) {
  __shared__ unsigned long long starts[16];
  __shared__ int found[16];
  const int b = blockIdx.y, t = threadIdx.x, lane = t & 63, wv = t >> 6;
  const int n = kv_lens ? min(max(kv_lens[b], 0), lk) : lk;
  const int q0 = n - lq;  // position of query 0
  const I* id = docs + b * doc_sb;
  int2* out = spans + (long long)b * lq;
  if (blockIdx.x == 0)  // queries before the first position
    for (int i = t; i < min(lq, -q0); i += 1024) out[i] = make_int2(0, 0);
  const long long base = (long long)blockIdx.x * 1024;
  if (base >= n) return;
  auto starts_at = [&](long long j) { return j == 0 || id[j] != id[j - 1]; };
  // largest (sign 1) or smallest (sign -1) v * sign over the workgroup
  auto most = [&](int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if (lane == 0) found[wv] = v;
    __syncthreads();
    int r = found[0];
    for (int w = 1; w < 16; ++w) r = max(r, found[w]);
    return r;
  };
  const int j = (int)base + t;
  const bool in = j < n;
  const unsigned long long mask = __ballot(in && starts_at(j));
  if (lane == 0) starts[wv] = mask;
  __syncthreads();
  int enter = -1, leave = 0x7fffffff;  // start of the run that enters the stretch; end of the one that leaves it
  if (!(starts[0] & 1))
    for (long long x = base - 1; x >= 0 && enter < 0; x -= 1024) enter = most(x - t >= 0 && starts_at(x - t) ? (int)(x - t) : -1);
  const long long past = base + 1024;
  if (past >= n)
    leave = n;
  else
    for (long long x = past; leave == 0x7fffffff; x += 1024) {
      const long long y = x + t;
      leave = -most(y >= n ? -n : starts_at(y) ? -(int)y : (int)0x80000001);
    }
  if (!in || j < q0) return;
  int start = enter, end = leave;
  for (int w = wv; w >= 0; --w) {
    const unsigned long long m = w == wv ? starts[w] & (~0ull >> (63 - lane)) : starts[w];
    if (m) {
      start = (int)base + w * 64 + 63 - __builtin_clzll(m);
      break;
    }
  }
  for (int w = wv; w < 16; ++w) {
    const unsigned long long m = w == wv ? (lane == 63 ? 0ull : starts[w] & (~0ull << (lane + 1))) : starts[w];
    if (m) {
      end = (int)base + w * 64 + __builtin_ctzll(m);
      break;
    }
  }
  end = min(end, n);
  if (causal) end = (int)min((long long)end, max((long long)j + 1, (long long)start + max(prefix ? prefix[b] : 0, 0)));
  out[j - q0] = id[j] < 0 ? make_int2(0, 0) : make_int2(start, end);
}

// The forward's launch, from sizes alone.
//
// Up to 32 rows per key head (single tokens): one-wave workgroups, the keys cut until about AT_FEW_BLOCKS of them run (five
// fit a CU; 8 x 32 query heads over 65536 keys: 282 us with 4096, 256 with 8192, 268 with 16384).
//
// More rows: 4 row waves (3, with 32-key tiles, where short rows would leave one of four without work and half a key tile
// empty: 257 x 257 tokens, 12 heads of 64, batch 32: 29 -> 27 us capped f16, 24 -> 21 bf16; and the grid holds that many row blocks). The keys are cut where that evens out the CUs: a CU's
// n = ceil(workgroups / 256) run two at a time (an odd one out has the CU to itself, a third faster), each costs its key
// tiles and about four tiles' time to start and end, and the cut costs the partials' traffic and a second launch (batch 2, 413
// queries, 16 heads over 4, 32768 keys: 1 cut 798 us, 5: 408, 7: 306, 9: 294, 12: 298). Ragged lengths leave whole cuts without
// work, which two more even out (lengths 32768 and 8192: 7 cuts 304 us, 9: 244, 11: 211, 13: 208).
// f32 tiles take about four times as long, and two key groups share a workgroup's rows while workgroups are scarce.
constexpr long long AT_FEW_BLOCKS = 8192, AT_CUS = 256;
static AtPlan at_plan(int dtype, int batch, int lq, int lk, int hk, int group, int d, bool ragged) {
  const long long rows = (long long)lq * group, nbh = (long long)batch * hk, r32 = (rows + 31) / 32;
  AtPlan p = {4, 1, lk > 0 ? lk : 1, 1, false};
  long long chunk = 0;
  if (rows <= 32) {
    p.nw = 1;
    if (nbh * 2 <= AT_FEW_BLOCKS) {
      chunk = ((long long)lk * nbh + AT_FEW_BLOCKS - 1) / AT_FEW_BLOCKS;
      chunk = chunk < 64 ? 64 : (chunk + 63) / 64 * 64;
    }
  } else {
    const long long b4 = (r32 + 3) / 4 * nbh;
    if ((r32 + 2) / 3 * 3 * nbh < b4 * 4 && lk <= 512 && (lk + 63) / 64 * 64 - lk >= 32 && (r32 + 2) / 3 < 65536) {
      p.nw = 3;
      return p;
    }
    const double fixed = dtype == DMF_F32 ? 1.0 : 4.0, tile_bytes = dtype == DMF_F32 ? 32e6 : 8e6;
    double best = 0;
    for (int s = 1; s <= 64 && (s == 1 || (long long)s * b4 <= 16 * AT_CUS); ++s) {
      long long c = ((long long)lk + s - 1) / s;
      c = (c + 63) / 64 * 64;
      if (s > 1 && c < 128) break;
      const long long n = c > 0 ? ((long long)lk + c - 1) / c : 1;
      const long long turns = (b4 * n + AT_CUS - 1) / AT_CUS;
      double cost = (turns + (turns % 2 ? 0.3 : 0.0)) * (c / 64.0 + fixed);
      if (n > 1) cost += fixed + (double)n * rows * nbh * (d + 4) * 8 / tile_bytes;
      if (s == 1 || cost < best) best = cost, chunk = n > 1 ? c : 0;
    }
    if (ragged && chunk > 0) {
      const long long n = ((long long)lk + chunk - 1) / chunk + 2, c = ((long long)lk + n - 1) / n;
      if (c >= 256) chunk = (c + 63) / 64 * 64;
    }
    if (dtype == DMF_F32 && lk > 64 && b4 * (chunk ? ((long long)lk + chunk - 1) / chunk : 1) <= AT_CUS) p.ng = 2;
  }
  if (chunk > 0 && lk > chunk && nbh * (((long long)lk + chunk - 1) / chunk) < (1LL << 31)) {
    p.chunk = (int)chunk;
    p.splits = (int)(((long long)lk + chunk - 1) / chunk);
  }
  return p;
}

// Workgroups of 4 waves with 64-key tiles run two on a CU, with 32-key tiles (half the LDS, at most 168 registers) three, at
// 3 to 10 % more time for the same work. (Those 168 registers are a few too few for 128 dims under a cap or with slopes for training,
// which spill 12 to 24 bytes in the first walk.) That pays where all are equally long (no mask) and three or five come to a CU, which two at a time
// leave an odd one of: bf16, 128 dims, 576 tokens, 4 heads, batch 32 (640 workgroups): 43 -> 36 us, capped and for training 57 -> 55;
// 64 (1280): 72 -> 62, 99 -> 95; but 48 (960): 50 -> 55, 74 -> 79; 8 (160): 18 -> 20, 25 -> 30. Seven and nine gain as well (88 rows: 97 ->
// 91, 134 -> 133; 112: 125 -> 113, 173 -> 169) and are not taken yet.
static bool at_three(const AtArgs& a) {
  const long long n = ((long long)a.batch * a.hk * (((long long)a.lq * a.group + 127) / 128) + AT_CUS - 1) / AT_CUS;
  return n == 3 || n == 5;
}

static int at_check(const char* who, AtArgs& a, int dtype) {
  DMF_CHECK_ARG(dtype == DMF_F32 || dtype == DMF_BF16 || dtype == DMF_F16, "%s: dtype %d", who, dtype);
  DMF_CHECK_ARG(a.batch >= 0 && a.lq >= 0 && a.lk >= 0 && a.hk >= 1 && a.hq >= 1 && a.hq % a.hk == 0,
                "%s: %d query heads must be a multiple of %d key heads", who, a.hq, a.hk);
  DMF_CHECK_ARG(a.d >= 8 && a.d <= 128 && a.d % 8 == 0, "%s: head dim %d must be a multiple of 8 up to 128", who, a.d);
  // (inside these the score's constants stay normal numbers of f32: scale / cap, its inverse square and a slope over the scale)
  DMF_CHECK_ARG(a.scale >= 0x1p-60f && a.scale <= 0x1p60f, "%s: scale %g must be in 2^-60 .. 2^60", who, a.scale);
  DMF_CHECK_ARG(a.cap == 0.f || (a.cap >= 0x1p-60f && a.cap <= 0x1p60f), "%s: softcap %g must be 0 (none) or in 2^-60 .. 2^60",
                who, a.cap);
  DMF_CHECK_ARG(a.causal || !a.prefix, "%s: a prefix needs causal", who);
  const long long rows = (long long)a.lq * a.group, nbh = (long long)a.batch * a.hk;
  DMF_CHECK_ARG(rows * a.group < (1LL << 31) && nbh < (1LL << 31) && (rows + 127) / 128 + (a.lk + 127LL) / 128 < 65536,
                "%s: %d queries x %d heads x %d rows exceed the launch", who, a.lq, a.hq, a.batch);
  const int e = dtype == DMF_F32 ? 4 : 2;
  const long long st[] = {a.q_sb, a.q_sl, a.q_sh, a.k_sb, a.k_sl, a.k_sh, a.v_sb, a.v_sl, a.v_sh};
  DMF_CHECK_ARG((a.lq <= 1 || a.q_sl >= a.d) && (a.lk <= 1 || (a.k_sl >= a.d && a.v_sl >= a.d)),
                "%s: token strides %lld / %lld / %lld must be at least the head dim", who, a.q_sl, a.k_sl, a.v_sl);
  for (long long s : st) DMF_CHECK_ARG(s >= 0 && s * e % 16 == 0, "%s: stride %lld is not a multiple of 16 bytes", who, s);
  DMF_CHECK_ARG((uintptr_t)a.q % 16 == 0 && (uintptr_t)a.k % 16 == 0 && (uintptr_t)a.v % 16 == 0,
                "%s: q, k and v must be aligned to 16 bytes", who);
  // (offsets within a tile of one head; heads, batch rows and tiles are added in 64 bits)
  DMF_CHECK_ARG(130 * a.k_sl * e < (1LL << 31) && 130 * a.v_sl * e < (1LL << 31) && 130 * a.q_sl * e < (1LL << 31) &&
                    (130LL * a.hq * a.d + (long long)a.hq * a.d) * e < (1LL << 31),
                "%s: a tile of rows spans more than 2 GiB", who);
  if (a.lq <= 1) a.q_sl = a.d;  // (a length of one: any stride says the same)
  if (a.lk <= 1) a.k_sl = a.v_sl = a.d;
  return 0;
}

}  // namespace dmf

using namespace dmf;

template <typename I>
static int mattn_spans(const char* who, const I* documents, long long doc_sb, const int* kv_lens, const int* prefix,
                       int batch, int lq, int lk, int causal, int* spans, void* stream) {
  // (the kernel steps over positions 1024 at a time, in ints)
  DMF_CHECK_ARG(batch >= 0 && batch < 65536 && lq >= 0 && lk >= 0 && lq < (1LL << 31) - 1024 && lk < (1LL << 31) - 1024,
                "%s: batch %d, lengths %d / %d", who, batch, lq, lk);
  if (batch == 0 || lq == 0) return 0;
  DMF_CHECK_ARG((documents || lk == 0) && spans && (uintptr_t)spans % 8 == 0, "%s: null operand", who);
  hipLaunchKernelGGL((k_mattn_spans<I>), dim3((unsigned)cdiv(lk > 0 ? lk : 1, 1024), (unsigned)batch), dim3(1024), 0,
                     (hipStream_t)stream, documents, doc_sb, kv_lens, prefix, lq, lk, causal, (int2*)spans);
  DMF_LAUNCH_CHECK(who);
  return 0;
}
extern "C" int dmf_mattn_spans(const int* documents, long long doc_sb, const int* kv_lens, const int* prefix, int batch,
                               int lq, int lk, int causal, int* spans, void* stream) {
  return mattn_spans("dmf_mattn_spans", documents, doc_sb, kv_lens, prefix, batch, lq, lk, causal, spans, stream);
}
extern "C" int dmf_mattn_spans64(const long long* documents, long long doc_sb, const int* kv_lens, const int* prefix,
                                 int batch, int lq, int lk, int causal, int* spans, void* stream) {
  return mattn_spans("dmf_mattn_spans64", documents, doc_sb, kv_lens, prefix, batch, lq, lk, causal, spans, stream);
}

extern "C" long long dmf_mattn_fwd_ws_floats(int dtype, int batch, int lq, int lk, int hq, int hk, int d, int ragged) {
  if (batch <= 0 || lq <= 0 || lk <= 0 || hk <= 0 || hq < hk) return 0;
  const AtPlan p = at_plan(dtype, batch, lq, lk, hk, hq / hk, d, ragged != 0);
  return p.splits > 1 ? (long long)p.splits * batch * lq * hq * (d + 4) : 0;
}

extern "C" int dmf_mattn_fwd(int dtype, const void* q, long long q_sb, long long q_sl, long long q_sh, const void* k,
                             long long k_sb, long long k_sl, long long k_sh, const void* v, long long v_sb,
                             long long v_sl, long long v_sh, int batch, int lq, int lk, int hq, int hk, int d,
                             float scale, float softcap, const float* slopes, int causal, const int* kv_lens,
                             const int* prefix, const int* spans, void* o, void* o_lo, float* lse, float* ws,
                             void* stream) {
  AtArgs a = {};
  a.q = q, a.k = k, a.v = v;
  a.q_sb = q_sb, a.q_sl = q_sl, a.q_sh = q_sh, a.k_sb = k_sb, a.k_sl = k_sl, a.k_sh = k_sh;
  a.v_sb = v_sb, a.v_sl = v_sl, a.v_sh = v_sh;
  a.batch = batch, a.lq = lq, a.lk = lk, a.hq = hq, a.hk = hk, a.d = d, a.group = hk > 0 ? hq / hk : 0;
  a.group_m = a.group > 1 ? (unsigned)(((1ULL << 32) + a.group - 1) / a.group) : 0;
  a.scale = scale, a.cap = softcap, a.slopes = slopes, a.causal = causal, a.kv_lens = kv_lens, a.prefix = prefix;
  a.spans = (const int2*)spans, a.o = o, a.o_lo = o_lo, a.lse = lse;
  if (int rc = at_check("dmf_mattn_fwd", a, dtype)) return rc;
  if (batch == 0 || lq == 0) return 0;
  DMF_CHECK_ARG(q && o && (lk == 0 || (k && v)), "dmf_mattn_fwd: null operand");
  DMF_CHECK_ARG(!lse || o_lo || dtype == DMF_F32, "dmf_mattn_fwd: lse of a 16-bit type goes with o_lo");
  DMF_CHECK_ARG(!o_lo || dtype != DMF_F32, "dmf_mattn_fwd: f32 has no o_lo");
  DMF_CHECK_ARG((uintptr_t)o % 16 == 0 && (uintptr_t)o_lo % 16 == 0 && (uintptr_t)spans % 8 == 0,
                "dmf_mattn_fwd: outputs must be aligned to 16 bytes");
  AtPlan p = at_plan(dtype, batch, lq, lk, hk, a.group, d, kv_lens != nullptr);
  a.chunk = p.chunk, a.splits = p.splits;
  p.three = p.nw == 4 && p.splits == 1 && !causal && !kv_lens && !spans && at_three(a);
  if (p.splits > 1) {
    DMF_CHECK_ARG(ws && (uintptr_t)ws % 16 == 0, "dmf_mattn_fwd: this size needs a workspace (dmf_mattn_fwd_ws_floats)");
    a.po = ws;
    a.pml = ws + (long long)p.splits * batch * lq * hq * d;
  }
  hipStream_t s = (hipStream_t)stream;
  return dtype == DMF_BF16 ? mattn_fwd_bf16(a, p, s) : dtype == DMF_F16 ? mattn_fwd_f16(a, p, s)
                                                                          : mattn_fwd_f32(a, p, s);
}

extern "C" int dmf_mattn_bwd(int dtype, const void* q, long long q_sb, long long q_sl, long long q_sh, const void* k,
                             long long k_sb, long long k_sl, long long k_sh, const void* v, long long v_sb,
                             long long v_sl, long long v_sh, int batch, int lq, int lk, int hq, int hk, int d,
                             float scale, float softcap, const float* slopes, int causal, const int* kv_lens,
                             const int* prefix, const int* spans, const void* o, const void* o_lo, const float* lse,
                             const void* go, float* ws, void* dq, void* dk, void* dv, void* stream) {
  AtArgs a = {};
  a.q = q, a.k = k, a.v = v;
  a.q_sb = q_sb, a.q_sl = q_sl, a.q_sh = q_sh, a.k_sb = k_sb, a.k_sl = k_sl, a.k_sh = k_sh;
  a.v_sb = v_sb, a.v_sl = v_sl, a.v_sh = v_sh;
  a.batch = batch, a.lq = lq, a.lk = lk, a.hq = hq, a.hk = hk, a.d = d, a.group = hk > 0 ? hq / hk : 0;
  a.group_m = a.group > 1 ? (unsigned)(((1ULL << 32) + a.group - 1) / a.group) : 0;
  a.scale = scale, a.cap = softcap, a.slopes = slopes, a.causal = causal, a.kv_lens = kv_lens, a.prefix = prefix;
  a.spans = (const int2*)spans, a.o = (void*)o, a.o_lo = (void*)o_lo, a.lse = (float*)lse, a.go = go, a.rowws = ws;
  a.dq = dq, a.dk = dk, a.dv = dv;
  if (int rc = at_check("dmf_mattn_bwd", a, dtype)) return rc;
  if (batch == 0 || (lq == 0 && lk == 0)) return 0;
  DMF_CHECK_ARG((lq == 0 || (q && o && lse && go && ws && dq)) && (lk == 0 || (k && v && dk && dv)),
                "dmf_mattn_bwd: null operand");
  DMF_CHECK_ARG(!o_lo || dtype != DMF_F32, "dmf_mattn_bwd: f32 has no o_lo");
  const uintptr_t al = (uintptr_t)o | (uintptr_t)o_lo | (uintptr_t)go | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv;
  DMF_CHECK_ARG(al % 16 == 0 && (uintptr_t)spans % 8 == 0, "dmf_mattn_bwd: operands must be aligned to 16 bytes");
  hipStream_t s = (hipStream_t)stream;
  return dtype == DMF_BF16 ? mattn_bwd_bf16(a, s) : dtype == DMF_F16 ? mattn_bwd_f16(a, s) : mattn_bwd_f32(a, s);
}
