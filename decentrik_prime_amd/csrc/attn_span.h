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

constexpr int kStride16 = kHD + 8;   // halves per staged row of a result

// The wave's 32 staged rows of a result [n_tokens, nq, hd], those that are in the block and not bad, 16
// bytes a lane, four whole rows per store.  One division, and the flags read before the first store: on
// their own in every step they took 0.13 us a step.
__device__ __forceinline__ void store_rows(const SpanArgs& a, const SpanItem& it, int wave, int lane,
                                           const f16* stage, const int* bad, f16* dst) {
  const int gin = a.nq / a.nkv, srow = 32 * wave + (lane >> 4), sr = it.phase + srow;
  int t = sr / gin, h = sr - t * gin;
  const int dt = 4 / gin, dh = 4 - dt * gin;
  int keep[8];
  f16x8 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    keep[i] = (srow + 4 * i < it.rows) & !bad[srow + 4 * i];
    v[i] = *reinterpret_cast<const f16x8*>(stage + (4 * i + (lane >> 4)) * kStride16 + 8 * (lane & 15));
  }
  f16* const base = dst + ((int64_t)it.t0 * a.nq + it.g * gin) * kHD + 8 * (lane & 15);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (keep[i]) *reinterpret_cast<f16x8*>(base + ((int64_t)t * a.nq + h) * kHD) = v[i];
    t += dt;
    h += dh;
    if (h >= gin) {
      h -= gin;
      ++t;
    }
  }
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


// Where quad q of result block hb of wave w's rows stands in a partial: 16 bytes per lane, lane-major.
__device__ __forceinline__ int part_off(int w, int hb, int q, int lane) {
  return ((w * (kHD / 32) + hb) * 4 + q) * 256 + 4 * lane;
}
__device__ __forceinline__ f32x4 quad(const f32x16& x, int q) {
  return f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
}

// One query row or one key row at a time, a wave each, over exactly the keys (or queries) that it
// sees: nothing else is read, so whatever a masked row holds cannot reach the result.  16 lanes hold a
// row, 8 columns each, so a wave takes four rows of a walk at a time, each quarter sums every fourth,
// and the loads of kWalk such steps are in flight.  A walk ends where nothing but NaN can come of
// it; a query's first look is at its term with itself, where a key's walk begins, so a batch of nothing
// but NaN (a diverged step) costs no walks.
constexpr int kWalk = 4;

// redo(i) for the flagged rows of a block, every fourth to a wave.  All flags are read at once: one
// after the other, for a block without any, took 1.6 us.
template <class F>
__device__ __forceinline__ void bad_rows(const int* bad, int rows, F redo) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const uint64_t lo = __builtin_amdgcn_ballot_w64(lane < rows && bad[lane]);
  const uint64_t hi = __builtin_amdgcn_ballot_w64(64 + lane < rows && bad[64 + lane]);
  if ((lo | hi) == 0) return;
  for (int i = wave; i < rows; i += 4)
    if ((i < 64 ? lo : hi) >> (i & 63) & 1) redo(i);
}

struct Row8 {
  float x[8];
};
__device__ __forceinline__ f16x8 row_load(const f16* row) {
  return *reinterpret_cast<const f16x8*>(row + 8 * (threadIdx.x & 15));
}
__device__ __forceinline__ Row8 row8(const f16* row) {
  const f16x8 v = row_load(row);
  Row8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.x[i] = (float)v[i];
  return r;
}
__device__ __forceinline__ void store8(f16* row, const Row8& r) {   // by the first quarter
  f16x8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (f16)r.x[i];
  if ((threadIdx.x & 63) < 16) *reinterpret_cast<f16x8*>(row + 8 * (threadIdx.x & 15)) = v;
}
__device__ __forceinline__ Row8 fill8(float x) { return Row8{{x, x, x, x, x, x, x, x}}; }

// x and its value in another lane of the 16, by a DPP control
template <int kCtrl>
__device__ __forceinline__ float add_dpp(float x) {
  return __fadd_rn(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), kCtrl, 0xf, 0xf, true)));
}
// the dot product of the quarter's row with one held the same way: lanes 1 and 2 further in a quad,
// then the other quad of the half (half mirror) and the other half (mirror), the same sum in every lane
__device__ __forceinline__ float row_dot(const Row8& a, const f16x8& b) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = __builtin_fmaf(a.x[i], (float)b[i], s);
  return add_dpp<0x140>(add_dpp<0x141>(add_dpp<0x4e>(add_dpp<0xb1>(s))));
}
__device__ __forceinline__ void row_add(Row8& r, float w, const f16x8& b) {
#pragma unroll
  for (int i = 0; i < 8; ++i) r.x[i] = __builtin_fmaf(w, (float)b[i], r.x[i]);
}
// the quarters' sums together, times scale
__device__ __forceinline__ Row8 row_sum(Row8 r, float scale) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    r.x[i] = __fadd_rn(r.x[i], __shfl_xor(r.x[i], 16));
    r.x[i] = __fmul_rn(__fadd_rn(r.x[i], __shfl_xor(r.x[i], 32)), scale);
  }
  return r;
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
__device__ __forceinline__ void span_row_fwd(const SpanArgs& a, int64_t m, int h, f16* out, float* lse) {
  const int64_t ROW = (int64_t)(a.nq + 2 * a.nkv) * kHD;
  const int kvh = h / (a.nq / a.nkv), quarter = (threadIdx.x >> 4) & 3;
  const f16* kb = a.qkv + (int64_t)(a.nq + kvh) * kHD;
  const f16* vb = kb + (int64_t)a.nkv * kHD;
  const Row8 q = row8(a.qkv + m * ROW + (int64_t)h * kHD);
  f16* orow = out + m * (int64_t)a.nq * kHD + (int64_t)h * kHD;
  const float own = __fmul_rn(row_dot(q, row_load(kb + m * ROW)), a.qk_scale);
  bool nan = own != own || own == INFINITY;   // 2^(inf - inf)
  const KeyRuns kr = key_runs(a, m);
  const int64_t n = kr.na + kr.nb;
  float mx = -INFINITY, l = 0.0f;
  Row8 o = fill8(0.0f);
  for (int64_t i0 = 0; i0 < n && !nan; i0 += 4 * kWalk) {
    f16x8 k[kWalk], v[kWalk];
#pragma unroll
    for (int u = 0; u < kWalk; ++u) {
      const int64_t i = i0 + 4 * u + quarter, off = kr.row(i < n ? i : n - 1) * ROW;
      k[u] = row_load(kb + off);
      v[u] = row_load(vb + off);
    }
    float sc[kWalk];
#pragma unroll
    for (int u = 0; u < kWalk; ++u) sc[u] = __fmul_rn(row_dot(q, k[u]), a.qk_scale);
#pragma unroll
    for (int u = 0; u < kWalk; ++u) {
      const float x = sc[u];
      if (i0 + 4 * u + quarter < n) {
        // a NaN score has to reach the sum: the maximum leaves it out, 2^(x - max) below does not
        const float m_new = fmaxf(mx, x), ref = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = mx == -INFINITY ? 0.0f : exp2f(__fsub_rn(mx, ref));
        const float p = exp2f(__fsub_rn(x, ref));
        mx = m_new;
        l = __builtin_fmaf(l, alpha, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) o.x[e] = __fmul_rn(o.x[e], alpha);
        row_add(o, p, v[u]);
      }
    }
    nan = __builtin_amdgcn_ballot_w64(l != l) != 0;
  }
  if (nan) {
    store8(orow, fill8(NAN));
    if ((threadIdx.x & 63) == 0) lse[(int64_t)h * a.n_tokens + m] = NAN;
    return;
  }
  // a quarter without keys has added nothing: its sums stay out
  float all = fmaxf(mx, __shfl_xor(mx, 16));
  all = fmaxf(all, __shfl_xor(all, 32));
  const float w = mx == -INFINITY ? 0.0f : exp2f(__fsub_rn(mx, all));
  l = __fmul_rn(l, w);
  l = __fadd_rn(l, __shfl_xor(l, 16));
  l = __fadd_rn(l, __shfl_xor(l, 32));
#pragma unroll
  for (int e = 0; e < 8; ++e) o.x[e] = __fmul_rn(o.x[e], w);
  store8(orow, row_sum(o, __fdiv_rn(1.0f, l)));
  if ((threadIdx.x & 63) == 0) lse[(int64_t)h * a.n_tokens + m] = __fadd_rn(all, log2f(l));
}

// dq of query m, head h
__device__ __forceinline__ void span_row_dq(const SpanArgs& a, int64_t m, int h, const f16* dout,
                                            const float* lse, const float* delta, f16* dq) {
  const int64_t ROW = (int64_t)(a.nq + 2 * a.nkv) * kHD, OROW = (int64_t)a.nq * kHD;
  const int kvh = h / (a.nq / a.nkv), quarter = (threadIdx.x >> 4) & 3;
  const f16* kb = a.qkv + (int64_t)(a.nq + kvh) * kHD;
  const f16* vb = kb + (int64_t)a.nkv * kHD;
  const Row8 q = row8(a.qkv + m * ROW + (int64_t)h * kHD), d = row8(dout + m * OROW + (int64_t)h * kHD);
  const float lm = lse[(int64_t)h * a.n_tokens + m], dm = delta[(int64_t)h * a.n_tokens + m];
  auto grad = [&](const f16x8& k, const f16x8& v) {
    const float p = exp2f(__builtin_fmaf(row_dot(q, k), a.qk_scale, -lm));
    return __fmul_rn(p, __fsub_rn(row_dot(d, v), dm));
  };
  const float own = grad(row_load(kb + m * ROW), row_load(vb + m * ROW));
  bool nan = own != own;   // in every column
  const KeyRuns kr = key_runs(a, m);
  const int64_t n = kr.na + kr.nb;
  Row8 g = fill8(0.0f);
  for (int64_t i0 = 0; i0 < n && !nan; i0 += 4 * kWalk) {
    f16x8 k[kWalk], v[kWalk];
#pragma unroll
    for (int u = 0; u < kWalk; ++u) {
      const int64_t i = i0 + 4 * u + quarter, off = kr.row(i < n ? i : n - 1) * ROW;
      k[u] = row_load(kb + off);
      v[u] = row_load(vb + off);
    }
    float ds[kWalk];
    bool any = false;
#pragma unroll
    for (int u = 0; u < kWalk; ++u) ds[u] = grad(k[u], v[u]);
#pragma unroll
    for (int u = 0; u < kWalk; ++u)
      if (i0 + 4 * u + quarter < n) {
        any |= ds[u] != ds[u];
        row_add(g, ds[u], k[u]);
      }
    nan = __builtin_amdgcn_ballot_w64(any) != 0;
  }
  store8(dq + m * OROW + (int64_t)h * kHD, nan ? fill8(NAN) : row_sum(g, a.sm_scale));
}

// dk and dv of key n, KV head g, summed over the queries that see it and the heads of its group
__device__ __forceinline__ void span_key_dkdv(const SpanArgs& a, int64_t n, int g, const f16* dout,
                                              const float* lse, const float* delta, f16* dk, f16* dv) {
  const int64_t ROW = (int64_t)(a.nq + 2 * a.nkv) * kHD, OROW = (int64_t)a.nq * kHD;
  const int gin = a.nq / a.nkv, quarter = (threadIdx.x >> 4) & 3;
  const f16* krow = a.qkv + n * ROW + (int64_t)(a.nq + g) * kHD;
  const Row8 k = row8(krow), v = row8(krow + (int64_t)a.nkv * kHD);
  Row8 gk = fill8(0.0f), gv = fill8(0.0f);
  bool dk_nan = false, dv_nan = false;   // in every column
  const int64_t end = key_end(a, n);
  for (int hh = g * gin; hh < (g + 1) * gin; ++hh) {
    const f16* qb = a.qkv + (int64_t)hh * kHD;
    const f16* ob = dout + (int64_t)hh * kHD;
    const float* lb = lse + (int64_t)hh * a.n_tokens;
    const float* db = delta + (int64_t)hh * a.n_tokens;
    for (int64_t m0 = n; m0 < end && !(dk_nan && dv_nan); m0 += 4 * kWalk) {
      f16x8 q[kWalk], o[kWalk];
      float lm[kWalk], dm[kWalk];
#pragma unroll
      for (int u = 0; u < kWalk; ++u) {
        const int64_t i = m0 + 4 * u + quarter, m = i < end ? i : end - 1;
        q[u] = row_load(qb + m * ROW);
        o[u] = row_load(ob + m * OROW);
        lm[u] = lb[m];
        dm[u] = db[m];
      }
      float p[kWalk], ds[kWalk];
      bool p_nan = false, ds_nan = false;
#pragma unroll
      for (int u = 0; u < kWalk; ++u) {
        p[u] = exp2f(__builtin_fmaf(row_dot(k, q[u]), a.qk_scale, -lm[u]));
        ds[u] = __fmul_rn(p[u], __fsub_rn(row_dot(v, o[u]), dm[u]));
      }
#pragma unroll
      for (int u = 0; u < kWalk; ++u)
        if (m0 + 4 * u + quarter < end) {
          p_nan |= p[u] != p[u];
          ds_nan |= ds[u] != ds[u];
          row_add(gk, ds[u], q[u]);
          row_add(gv, p[u], o[u]);
        }
      // every column of dv is NaN where each is in a quarter's sum
      bool all = true;
#pragma unroll
      for (int e = 0; e < 8; ++e) all &= gv.x[e] != gv.x[e];
      uint64_t cols = __builtin_amdgcn_ballot_w64(all);
      cols |= cols >> 32;
      cols |= cols >> 16;
      dk_nan |= __builtin_amdgcn_ballot_w64(ds_nan) != 0;
      dv_nan |= __builtin_amdgcn_ballot_w64(p_nan) != 0 || (cols & 0xffff) == 0xffff;
    }
  }
  const int64_t off = n * (int64_t)a.nkv * kHD + (int64_t)g * kHD;
  store8(dk + off, dk_nan ? fill8(NAN) : row_sum(gk, a.sm_scale));
  store8(dv + off, dv_nan ? fill8(NAN) : row_sum(gv, 1.0f));
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
