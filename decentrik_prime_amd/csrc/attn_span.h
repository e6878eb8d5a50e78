#pragma once
// Attention of the packed batch in which key n is seen by the queries n .. kend[n] - 1 (a sliding
// window with sinks; answers behind a shared prompt): what the forward (span_fwd.hip) and the
// backward (span_bwd.hip) share.
//
// spans [n_tokens][4] int32 holds, per token m, as query (a0, a1, kbeg) and as key kend: it sees the
// keys [a0, a1) (a sequence's sinks or a group's prompt) and [kbeg, m] (its window or its own answer),
// and as a key it is seen by the queries m .. kend - 1.  The two descriptions are the same set.
#include "attn_dev.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct SpanArgs {
  const f16* qkv;
  const int32_t* spans;
  int64_t n_tokens;
  int nq, nkv;
  float qk_scale, sm_scale;
};

// A block of up to kBM stacked query rows and the keys that they see (SPAN_ITEM_INTS int32, written by
// k_attn.SpanMeta).  The rows of a run of tokens are stacked (token, query head of one KV head's
// group): row i of the block is token t0 + (phase + i) / gin, head g gin + (phase + i) % gin, so one
// K / V tile serves a group's heads, and a block spans few tokens, whatever their number.  Its keys are
// numbered j = 0 .. nk - 1: na rows from a0 (sinks or prompt), then rows b0 .. up to the last token.
// A tile is kBN keys; those of [0, f0) and [f1, f2) are seen by every row.  The item walks tiles
// [tb, te); slot: the partial that it writes, or -1 for the outputs themselves.
constexpr int kItemInts = DK_ATTN_SPAN_ITEM_INTS;
struct SpanItem {
  int t0, phase, rows, g;
  int a0, na, b0, nk;
  int f0, f1, f2, tb;
  int te, slot;
};
__device__ __forceinline__ bool span_item(const SpanArgs& a, const int32_t* items, int i, int n_slots,
                                          SpanItem* it) {
  const int32_t* p = items + (int64_t)i * kItemInts;
  auto u = [&](int k) { return __builtin_amdgcn_readfirstlane(p[k]); };
  *it = SpanItem{u(0), u(1), u(2), u(3), u(4), u(5), u(6), u(7), u(8), u(9), u(10), u(11), u(12), u(13)};
  const int gin = a.nq / a.nkv;
  // an entry that names rows outside the batch is skipped before any load
  return it->t0 >= 0 && it->phase >= 0 && it->phase < gin && it->rows >= 1 && it->rows <= kBM &&
         it->g >= 0 && it->g < a.nkv &&
         (int64_t)it->t0 + (it->phase + it->rows - 1) / gin < a.n_tokens && it->a0 >= 0 &&
         it->na >= 0 && (int64_t)it->a0 + it->na <= a.n_tokens && it->b0 >= 0 && it->nk > it->na &&
         (int64_t)it->b0 + it->nk - it->na <= a.n_tokens &&
         (it->na % kBN == 0 || (it->b0 >= it->a0 + it->na &&
                          ((int64_t)it->b0 - it->a0 - it->na + kBN) * (a.nq + 2 * a.nkv) * kHD * 2 <
                              (int64_t)DK_ATTN_SPAN_REACH_BYTES)) && it->tb >= 0 && it->tb < it->te &&
         it->te <= (it->nk + kBN - 1) / kBN && it->slot < n_slots;
}
__device__ __forceinline__ bool full_tile(const SpanItem& it, int t) {
  return t < it.f0 || (t >= it.f1 && t < it.f2);
}

// A tile of the item's keys, one operand, by LDS DMA: instruction i fills rows 4 (W i + wave) .. + 3 of
// the tile (W waves), 16 lanes a row, from a scalar base per tile and a 32-bit offset per lane.  In the
// tile that holds keys of both runs the second run's lie a gap further on (span_item: it fits).  Keys
// past the last one read its row (finite, and masked).
struct KeySource {
  unsigned rowb, r0, off0, chunk;   // bytes per row; this lane's row, offset and chunk for instruction 0
};
__device__ __forceinline__ KeySource key_source(int64_t row_halves, int wave, int lane) {
  KeySource s;
  s.rowb = (unsigned)(row_halves * (int64_t)sizeof(f16));
  s.r0 = (unsigned)(4 * wave + (lane >> 4));
  s.chunk = (unsigned)(((lane & 15) ^ swz16((int)s.r0)) << 4);
  s.off0 = s.r0 * s.rowb + s.chunk;
  return s;
}
// One operand's tiles in order: where key 0 would lie in each run, and the bytes of the tiles before.
struct KeyWalk {
  uint64_t pa, pb, adv;
  int t;
};
__device__ __forceinline__ KeyWalk key_walk(const SpanItem& it, uint64_t base, unsigned rowb) {
  return KeyWalk{base + (uint64_t)it.a0 * rowb, base + (uint64_t)((int64_t)it.b0 - it.na) * rowb,
                 (uint64_t)it.tb * kBN * rowb, it.tb};
}
template <int W>
__device__ __forceinline__ void next_key_tile(const SpanItem& it, KeyWalk& k, const KeySource& s,
                                              const f16* stage, int wave) {
  const int j0 = k.t * kBN;
  const bool second = j0 >= it.na;
  const uint64_t tb = (second ? k.pb : k.pa) + k.adv;
  const unsigned dst = __builtin_amdgcn_readfirstlane(lds_addr(stage + wave * 512));
  if ((second || j0 + kBN <= it.na) && j0 + kBN <= it.nk) {
#pragma unroll
    for (int i = 0; i < kBN / 4 / W; ++i) dma16s(tb, s.off0 + (unsigned)(4 * W * i) * s.rowb, dst + W * i * 1024);
  } else {
    const unsigned thr = second ? kBN : (unsigned)(it.na - j0);   // the second run's first row here
    const unsigned gap = (unsigned)(it.b0 - it.a0 - it.na) * s.rowb;
    const unsigned rows = (unsigned)(it.nk - 1 - j0);
    const unsigned last = (rows < kBN ? rows * s.rowb + (rows >= thr ? gap : 0u) : ~0u - 4096u) + s.chunk;
#pragma unroll
    for (int i = 0; i < kBN / 4 / W; ++i) {
      unsigned off = s.off0 + (unsigned)(4 * W * i) * s.rowb;
      off += s.r0 + 4 * W * i >= thr ? gap : 0u;
      dma16s(tb, off < last ? off : last, dst + W * i * 1024);
    }
  }
  k.adv += (uint64_t)kBN * s.rowb;
  ++k.t;
}
// the keys' ends, by one wave
__device__ __forceinline__ void key_ends_load(const SpanArgs& a, const SpanItem& it, int t, const int* dst,
                                              int lane) {
  const int jj = t * kBN + lane, j = jj < it.nk ? jj : it.nk - 1;
  const int64_t row = j < it.na ? it.a0 + j : it.b0 + (j - it.na);
  dma4(a.spans + 4 * row + 3, __builtin_amdgcn_readfirstlane(lds_addr(dst)));
}

constexpr int kStride16 = kHD + 8;   // halves per staged row of a result

// Where quad q of result block hb of wave w's rows stands in a partial: 16 bytes per lane, lane-major.
__device__ __forceinline__ int part_off(int w, int hb, int q, int lane) {
  return ((w * (kHD / 32) + hb) * 4 + q) * 256 + 4 * lane;
}
__device__ __forceinline__ f32x4 quad(const f32x16& x, int q) {
  return f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
}

// One query row or one key row at a time, a wave each, over exactly the keys (or queries) that it
// sees: nothing else is read, so whatever a masked row holds cannot reach the result.  Where a token's
// term with itself, which it always sees, is NaN already, so is the whole row, and the walk is spared: a
// batch of nothing but NaN (a diverged step) costs no walks.
struct RowScratch {
  float a[kHD], b[kHD];   // the wave's row (q or k) and its partner (dO or v)
  float p[64], ds[64];
};

__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) v = __fadd_rn(v, __shfl_xor(v, x));
  return v;
}

__device__ __forceinline__ void row_to_lds(float* dst, const f16* src) {
  const int lane = threadIdx.x & 63;
  const f16x2 v = *reinterpret_cast<const f16x2*>(src + 2 * lane);
  dst[2 * lane] = (float)v[0];
  dst[2 * lane + 1] = (float)v[1];
}

// dot product of a row in LDS with this lane's row in memory
__device__ __forceinline__ float row_dot(const float* a, const f16* row) {
  float s = 0.0f;
#pragma unroll 4
  for (int i = 0; i < kHD / 8; ++i) {
    const f16x8 x = *reinterpret_cast<const f16x8*>(row + 8 * i);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fmaf(a[8 * i + e], (float)x[e], s);
  }
  return s;
}

// The keys that query m sees, as na keys from a0 and nb from b0 (kept within [0, m] whatever spans
// holds, so every row read exists).
struct KeyRuns {
  int64_t a0, b0;
  int64_t na, nb;
  __device__ __forceinline__ int64_t row(int64_t i) const { return i < na ? a0 + i : b0 + (i - na); }
};
__device__ __forceinline__ KeyRuns key_runs(const SpanArgs& a, int64_t m) {
  const int32_t* s = a.spans + 4 * m;
  KeyRuns r;
  r.a0 = s[0] > 0 ? s[0] : 0;
  const int64_t a1 = s[1] < m + 1 ? s[1] : m + 1;
  r.na = a1 > r.a0 ? a1 - r.a0 : 0;
  r.b0 = s[2] > 0 ? s[2] : 0;
  if (r.na > 0 && r.b0 < a1) r.b0 = a1;
  r.nb = m + 1 > r.b0 ? m + 1 - r.b0 : 0;
  return r;
}
__device__ __forceinline__ int64_t key_end(const SpanArgs& a, int64_t n) {
  const int64_t e = a.spans[4 * n + 3];
  return e < a.n_tokens ? e : a.n_tokens;
}

// out and lse of query m, head h
__device__ __forceinline__ void span_row_fwd(const SpanArgs& a, int64_t m, int h, f16* out, float* lse,
                                          RowScratch& s) {
  const int lane = threadIdx.x & 63;
  const int64_t ROW = (int64_t)(a.nq + 2 * a.nkv) * kHD;
  const int kvh = h / (a.nq / a.nkv);
  const f16* kb = a.qkv + (int64_t)(a.nq + kvh) * kHD;
  const f16* vb = kb + (int64_t)a.nkv * kHD;
  wave_sync();
  row_to_lds(s.a, a.qkv + m * ROW + (int64_t)h * kHD);
  wave_sync();
  f16* orow = out + m * (int64_t)a.nq * kHD + (int64_t)h * kHD + 2 * lane;
  const float own = __fmul_rn(row_dot(s.a, kb + m * ROW), a.qk_scale);
  if (own != own || own == INFINITY) {   // 2^(inf - inf)
    *reinterpret_cast<f16x2*>(orow) = f16x2{(f16)NAN, (f16)NAN};
    if (lane == 0) lse[(int64_t)h * a.n_tokens + m] = NAN;
    return;
  }
  const KeyRuns kr = key_runs(a, m);
  const int64_t n = kr.na + kr.nb;
  float mx = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  for (int64_t i0 = 0; i0 < n; i0 += 64) {
    const bool on = i0 + lane < n;
    float x = -INFINITY;
    if (on) x = __fmul_rn(row_dot(s.a, kb + kr.row(i0 + lane) * ROW), a.qk_scale);
    // a NaN score has to reach the sum: the maximum leaves it out, 2^(x - max) below does not
    float t = x;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) t = fmaxf(t, __shfl_xor(t, d));
    const float m_new = fmaxf(mx, t);
    const float ref = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = mx == -INFINITY ? 0.0f : exp2f(__fsub_rn(mx, ref));
    const float p = on ? exp2f(__fsub_rn(x, ref)) : 0.0f;
    mx = m_new;
    l = __fadd_rn(__fmul_rn(l, alpha), wave_sum(p));
    o0 = __fmul_rn(o0, alpha);
    o1 = __fmul_rn(o1, alpha);
    wave_sync();
    s.p[lane] = p;
    wave_sync();
    const int cnt = n - i0 < 64 ? (int)(n - i0) : 64;
    for (int j = 0; j < cnt; ++j) {
      const f16x2 v = *reinterpret_cast<const f16x2*>(vb + kr.row(i0 + j) * ROW + 2 * lane);
      o0 = __builtin_fmaf(s.p[j], (float)v[0], o0);
      o1 = __builtin_fmaf(s.p[j], (float)v[1], o1);
    }
  }
  const float inv = __fdiv_rn(1.0f, l);
  f16x2 r;
  r[0] = (f16)__fmul_rn(o0, inv);
  r[1] = (f16)__fmul_rn(o1, inv);
  *reinterpret_cast<f16x2*>(orow) = r;
  if (lane == 0) lse[(int64_t)h * a.n_tokens + m] = __fadd_rn(mx, log2f(l));
}

// dq of query m, head h
__device__ __forceinline__ void span_row_dq(const SpanArgs& a, int64_t m, int h, const f16* dout,
                                         const float* lse, const float* delta, f16* dq,
                                         RowScratch& s) {
  const int lane = threadIdx.x & 63;
  const int64_t ROW = (int64_t)(a.nq + 2 * a.nkv) * kHD, OROW = (int64_t)a.nq * kHD;
  const int kvh = h / (a.nq / a.nkv);
  const f16* kb = a.qkv + (int64_t)(a.nq + kvh) * kHD;
  const f16* vb = kb + (int64_t)a.nkv * kHD;
  wave_sync();
  row_to_lds(s.a, a.qkv + m * ROW + (int64_t)h * kHD);
  row_to_lds(s.b, dout + m * OROW + (int64_t)h * kHD);
  wave_sync();
  const float lm = lse[(int64_t)h * a.n_tokens + m], dm = delta[(int64_t)h * a.n_tokens + m];
  f16* grow = dq + m * OROW + (int64_t)h * kHD + 2 * lane;
  const float own = __fmul_rn(exp2f(__builtin_fmaf(row_dot(s.a, kb + m * ROW), a.qk_scale, -lm)),
                              __fsub_rn(row_dot(s.b, vb + m * ROW), dm));
  if (own != own) {
    *reinterpret_cast<f16x2*>(grow) = f16x2{(f16)NAN, (f16)NAN};
    return;
  }
  const KeyRuns kr = key_runs(a, m);
  const int64_t n = kr.na + kr.nb;
  float g0 = 0.0f, g1 = 0.0f;
  for (int64_t i0 = 0; i0 < n; i0 += 64) {
    float ds = 0.0f;
    if (i0 + lane < n) {
      const int64_t off = kr.row(i0 + lane) * ROW;
      const float p = exp2f(__builtin_fmaf(row_dot(s.a, kb + off), a.qk_scale, -lm));
      ds = __fmul_rn(p, __fsub_rn(row_dot(s.b, vb + off), dm));
    }
    wave_sync();
    s.ds[lane] = ds;
    wave_sync();
    const int cnt = n - i0 < 64 ? (int)(n - i0) : 64;
    for (int j = 0; j < cnt; ++j) {
      const f16x2 k = *reinterpret_cast<const f16x2*>(kb + kr.row(i0 + j) * ROW + 2 * lane);
      g0 = __builtin_fmaf(s.ds[j], (float)k[0], g0);
      g1 = __builtin_fmaf(s.ds[j], (float)k[1], g1);
    }
  }
  f16x2 r;
  r[0] = (f16)__fmul_rn(g0, a.sm_scale);
  r[1] = (f16)__fmul_rn(g1, a.sm_scale);
  *reinterpret_cast<f16x2*>(grow) = r;
}

// dk and dv of key n, KV head g, summed over the queries that see it and the heads of its group
__device__ __forceinline__ void span_key_dkdv(const SpanArgs& a, int64_t n, int g, const f16* dout,
                                           const float* lse, const float* delta, f16* dk, f16* dv,
                                           RowScratch& s) {
  const int lane = threadIdx.x & 63;
  const int64_t ROW = (int64_t)(a.nq + 2 * a.nkv) * kHD, OROW = (int64_t)a.nq * kHD;
  const int gin = a.nq / a.nkv;
  const f16* krow = a.qkv + n * ROW + (int64_t)(a.nq + g) * kHD;
  wave_sync();
  row_to_lds(s.a, krow);
  row_to_lds(s.b, krow + (int64_t)a.nkv * kHD);
  wave_sync();
  const int64_t off = n * (int64_t)a.nkv * kHD + (int64_t)g * kHD + 2 * lane;
  // dk is NaN where the token's own dS is, dv where its own P is or, by columns, its own dO
  bool p_nan = false, ds_nan = false, col0 = false, col1 = false;
  for (int hh = g * gin; hh < (g + 1) * gin; ++hh) {
    const f16* orow = dout + n * OROW + (int64_t)hh * kHD;
    const float p = exp2f(__builtin_fmaf(row_dot(s.a, a.qkv + n * ROW + (int64_t)hh * kHD), a.qk_scale,
                                         -lse[(int64_t)hh * a.n_tokens + n]));
    const float ds = __fmul_rn(p, __fsub_rn(row_dot(s.b, orow), delta[(int64_t)hh * a.n_tokens + n]));
    const f16x2 o = *reinterpret_cast<const f16x2*>(orow + 2 * lane);
    p_nan |= p != p;
    ds_nan |= ds != ds;
    col0 |= o[0] != o[0];
    col1 |= o[1] != o[1];
  }
  if (ds_nan && (p_nan || __builtin_amdgcn_ballot_w64(!(col0 && col1)) == 0)) {
    *reinterpret_cast<f16x2*>(dk + off) = f16x2{(f16)NAN, (f16)NAN};
    *reinterpret_cast<f16x2*>(dv + off) = f16x2{(f16)NAN, (f16)NAN};
    return;
  }
  const int64_t end = key_end(a, n);
  float dk0 = 0.0f, dk1 = 0.0f, dv0 = 0.0f, dv1 = 0.0f;
  for (int hh = g * gin; hh < (g + 1) * gin; ++hh)
    for (int64_t m0 = n; m0 < end; m0 += 64) {
      const int64_t m = m0 + lane;
      const f16* qb = a.qkv + (int64_t)hh * kHD;
      const f16* ob = dout + (int64_t)hh * kHD;
      float p = 0.0f, ds = 0.0f;
      if (m < end) {
        p = exp2f(__builtin_fmaf(row_dot(s.a, qb + m * ROW), a.qk_scale,
                                 -lse[(int64_t)hh * a.n_tokens + m]));
        ds = __fmul_rn(p, __fsub_rn(row_dot(s.b, ob + m * OROW), delta[(int64_t)hh * a.n_tokens + m]));
      }
      wave_sync();
      s.p[lane] = p;
      s.ds[lane] = ds;
      wave_sync();
      const int cnt = end - m0 < 64 ? (int)(end - m0) : 64;
      for (int j = 0; j < cnt; ++j) {
        const f16x2 q = *reinterpret_cast<const f16x2*>(qb + (m0 + j) * ROW + 2 * lane);
        const f16x2 o = *reinterpret_cast<const f16x2*>(ob + (m0 + j) * OROW + 2 * lane);
        dk0 = __builtin_fmaf(s.ds[j], (float)q[0], dk0);
        dk1 = __builtin_fmaf(s.ds[j], (float)q[1], dk1);
        dv0 = __builtin_fmaf(s.p[j], (float)o[0], dv0);
        dv1 = __builtin_fmaf(s.p[j], (float)o[1], dv1);
      }
    }
  f16x2 r;
  r[0] = (f16)__fmul_rn(dk0, a.sm_scale);
  r[1] = (f16)__fmul_rn(dk1, a.sm_scale);
  *reinterpret_cast<f16x2*>(dk + off) = r;
  r[0] = (f16)dv0;
  r[1] = (f16)dv1;
  *reinterpret_cast<f16x2*>(dv + off) = r;
}

// the launch arguments, with the checks both entry points share
inline int span_args(SpanArgs& a, const void* qkv, const int32_t* spans, int64_t n_tokens, int32_t nq,
                     int32_t nkv, int32_t hd) {
  if (hd != kHD || nq < 1 || nkv < 1 || nq % nkv || nq > 65535 || n_tokens < 0 ||
      n_tokens > INT32_MAX / 2)
    return DK_ERR_INVALID;
  if (n_tokens > 0 && (!qkv || !spans)) return DK_ERR_INVALID;
  if (!dk_aligned(qkv, 16) || !dk_aligned(spans, 16)) return DK_ERR_ALIGN;
  const double log2e = 1.4426950408889634;
  a = SpanArgs{(const f16*)qkv, spans, n_tokens, nq, nkv, (float)(log2e / __builtin_sqrt((double)hd)),
               (float)(1.0 / __builtin_sqrt((double)hd))};
  return 0;
}

}  // namespace
