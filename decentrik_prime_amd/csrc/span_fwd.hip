// Forward of the attention over part of the keys (attn_span.h): with s = scale q . k over the keys that a
// row sees (log2 units), m a reference near max s, l = sum 2^(s - m): out = sum 2^(s - m) v / l,
// lse = m + log2 l, m and l running over the tiles.  P = 2^(s - m) is rounded to fp16 for its product (the
// sum l takes it unrounded), everything else is fp32 up to the one rounding of out.  That rounding is half a
// step, 2^-11 of each value, down to 2^-21 of the row's largest P, and 2^-32 of the largest below: m lies
// kUp under the largest score, so the largest P is 2^7 to 2^15 and the type's subnormals begin that much
// further down (behind a sink that takes a row's weight and has no value, small P are all there is).
// Built with the MFMA accumulators in VGPRs like attn_fwd.hip.
#include "attn_span.h"

namespace {

constexpr int kStages = 2;   // of each operand's ring
// A row's reference m is set kUp (log2 units) under its largest score, and again once a score exceeds m by
// more than kTop: P stays below 2^15, half of fp16's range.
constexpr float kUp = 7.0f, kTop = 15.0f;
// a partial: O (part_off) and the rows' m and l
constexpr int kPartFloats = kBM * kHD + 2 * kBM;

// max over the two lanes l, l ^ 32 (the two key halves of one query)
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The rows whose result is not finite, recomputed over exactly the keys that they see: a masked key's
// probability is 0, but 0 times a NaN or infinity in its value row is not.  bad [kBM]: row flags in
// LDS, written before a barrier.
__device__ __forceinline__ void redo_rows(const SpanArgs& a, int t0, int phase, int rows, int g,
                                          const int* bad, f16* out, float* lse) {
  const int gin = a.nq / a.nkv;
  bad_rows(bad, rows, [&](int i) {
    span_row_fwd(a, t0 + (phase + i) / gin, g * gin + (phase + i) % gin, out, lse);
  });
}

// A workgroup per item: 4 waves of 32 stacked rows, lane l % 32 a row, over 64-key tiles.
//
// Bound: per tile a wave has 32 MFMAs (1024 clocks), about as many clocks of exponentials and
// conversions, and 48 LDS operand reads, one after the other for a wave on its own.  So the scores of
// the next tile stand beside the exponentials of the current one (K runs a tile ahead of V), and a CU
// holds two workgroups (two stages of K and V, 66 KB; 227 registers), whose first loads, barriers and
// stores stand beside the other's products.  Stacking a group's heads on the rows makes a block span
// 128 / gin tokens: fewer masked keys at a window's edges, and answers of a token fill blocks.
// Measured on MI355X, 12 query / 2 KV heads (passes back to back): 16384 tokens, window 4096, 4 sinks
// 424 us (851 TFLOP/s); 8192 tokens, window 1024, 78; a prompt of 8192 with 64 answers of a token 248; one
// workgroup of 8 waves to a CU, the waves of a SIMD on alternate tiles, took 1.17 to 1.2 times as long.
// 20 tokens, one tile, take 7.4: launch 2.2, the item 0.5, first loads 1.9, the tile's code, run for the
// first time, 2.5, the rows' stores 0.3; the second tile 2.1, later ones 1.1 and 2.0 in turn.  A last tile without the next one's scores, or a
// whole tile on its own unmasked, spilled registers.
// Walks are cut where one would outlast the rest (k_attn._fwd_tiles): that prompt uncut 360 us.
__global__ __launch_bounds__(kAThreads, 2) void span_fwd_kernel(
    SpanArgs a, const int32_t* __restrict__ items, int n_slots, f16* __restrict__ out,
    float* __restrict__ lse, float* __restrict__ parts) {
  SpanItem it;
  if (!span_item(a, items, (int)blockIdx.x, n_slots, &it)) return;
  const int lane = threadIdx.x & 63, hl = lane >> 5, c = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int gin = a.nq / a.nkv;
  const int64_t ROW = (int64_t)(a.nq + 2 * a.nkv) * kHD;
  const int row = 32 * wave + c;             // this lane's stacked row
  const bool mval = row < it.rows;
  const int rr = it.phase + (mval ? row : 0);
  const int m = it.t0 + rr / gin, h = it.g * gin + rr % gin;
  const int jlim = mval ? m - it.b0 + it.na : -1;   // its last key
  __shared__ __attribute__((aligned(1024))) f16 ring[2 * kStages * kTileHalves];
  __shared__ __attribute__((aligned(16))) int ends[kStages][kBN];
  f16* const Ks = ring;
  f16* const Vs = ring + kStages * kTileHalves;
  __shared__ int bad[kBM];

  f32x16 oacc[kHD / 32];
#pragma unroll
  for (int hb = 0; hb < kHD / 32; ++hb) oacc[hb] = zero16();
  constexpr float kMasked = -3.0e38f;
  float m_i = -1.0e30f, l_i = 0.0f;   // l_i: this lane's half of the keys (joined at the end)
  const int n_tiles = it.te - it.tb;
  const uint64_t kbase = uniform64((uint64_t)(a.qkv + (int64_t)(a.nq + it.g) * kHD));
  const uint64_t vbase = kbase + (uint64_t)a.nkv * kHD * sizeof(f16);
  const KeySource src = key_source(ROW, wave, lane);
  KeyWalk kw = key_walk(it, kbase, src.rowb), vw = key_walk(it, vbase, src.rowb);
  // the next tile of one operand into stage t % 2
  auto issue = [&](KeyWalk& x, f16* stages) {
    if (x.t < it.te) next_key_tile<4>(it, x, src, stages + ((x.t - it.tb) % kStages) * kTileHalves, wave);
  };
  auto issue_v = [&](int t) {
    issue(vw, Vs);
    if (wave == 0 && t < n_tiles) key_ends_load(a, it, it.tb + t, ends[t % kStages], lane);
  };
  issue(kw, Ks);
  issue_v(0);
  issue(kw, Ks);
  // this lane's query row as the B operand (rows past the block: zeros).  Loaded unconditionally and
  // selected at once, so the compiler's wait for these loads stands here and not inside the loop.
  f16x8 qf[kHD / 16];
  {
    const f16* qrow = a.qkv + (int64_t)m * ROW + (int64_t)h * kHD + 8 * hl;
#pragma unroll
    for (int s = 0; s < kHD / 16; ++s) qf[s] = *reinterpret_cast<const f16x8*>(qrow + 16 * s);
#pragma unroll
    for (int s = 0; s < kHD / 16; ++s) asm volatile("" : "+v"(qf[s]));
#pragma unroll
    for (int s = 0; s < kHD / 16; ++s) qf[s] = mval ? qf[s] : zero8();
  }
  if (threadIdx.x < kBM) bad[threadIdx.x] = 0;
  wait_vmem<0>();
  __syncthreads();
  const unsigned krow = lds_addr(Ks) + row_base(lane), vcol = lds_addr(Vs) + col_base(lane);
  // S^T = K Q^T of tile t: keys kb * 32 + (row of the result), queries on the lanes
  auto scores = [&](f32x16 (&sc)[2], int t) {
    const unsigned ka = fresh(krow + (unsigned)((t % kStages) * kTileHalves * 2));
    sc[0] = sc[1] = zero16();
#pragma unroll
    for (int s = 0; s < kHD / 16; ++s)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        sc[kb] = mfma(lds_read8(ka ^ (unsigned)(32 * s), kb * 32 * kHD * 2), qf[s], sc[kb]);
  };
  f32x16 sc[2], sn[2];
  scores(sc, 0);
  __syncthreads();   // every wave is done with K of tile 0
  // tile t, whose scores are in sc: its softmax and O^T += V^T P^T, beside the scores of tile t + 1
  // into sn (after the last tile: of a stale stage, never used).  MASK: key j of the tile counts iff
  // j <= jlim and the key's end lies past this lane's token; the others' probabilities come out as 0, also
  // where a lane has seen no key yet: kMasked, scaled, lies far below m_i's start, and that below any score.
  auto tile = [&](int t, f32x16 (&sc)[2], f32x16 (&sn)[2], auto mask_c) {
    constexpr bool MASK = decltype(mask_c)::value;
    const unsigned va = fresh(vcol + (unsigned)((t % kStages) * kTileHalves * 2));
    const int lim = jlim - (it.tb + t) * kBN - 4 * hl;
    if constexpr (MASK) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const i32x4 e4 = *reinterpret_cast<const i32x4*>(&ends[t % kStages][8 * q + 4 * hl]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool seen = (8 * q + e <= lim) & (m < e4[e]);
          sc[q >> 2][4 * (q & 3) + e] = seen ? sc[q >> 2][4 * (q & 3) + e] : kMasked;
        }
      }
    }
    // the row maximum of the raw scores, scaled once (the scaling is monotonic)
    float mx = -1.0e30f;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int v = 0; v < 16; ++v) mx = fmaxf(mx, sc[kb][v]);
    mx = half_max(mx);
    // m_i moves (and O and l are rescaled) only when some lane's maximum exceeds it by more than kTop
    const float mt = __fmul_rn(mx, a.qk_scale);
    if (__builtin_amdgcn_ballot_w64(mt > m_i + kTop) != 0) {
      const float m_new = fmaxf(m_i, __fsub_rn(mt, kUp));
      const float alpha = ex2(__fsub_rn(m_i, m_new));
      l_i = __fmul_rn(l_i, alpha);
      m_i = m_new;
#pragma unroll
      for (int hb = 0; hb < kHD / 32; ++hb)
#pragma unroll
        for (int v = 0; v < 16; ++v) oacc[hb][v] = __fmul_rn(oacc[hb][v], alpha);
    }
    scores(sn, t + 1);
    float rs[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    f16x8 pf[kBN / 16];   // P^T as the B operand: keys 16 tt .. + 15
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const float p = ex2(__builtin_fmaf(sc[kb][v], a.qk_scale, -m_i));
        rs[v & 3] = __fadd_rn(rs[v & 3], p);
        pf[2 * kb + (v >> 3)][v & 7] = (f16)p;
      }
    l_i = __fadd_rn(l_i, __fadd_rn(__fadd_rn(rs[0], rs[1]), __fadd_rn(rs[2], rs[3])));
    // O^T += V^T P^T over the tile's 64 keys, 16 per step
#pragma unroll
    for (int tt = 0; tt < kBN / 16; ++tt)
#pragma unroll
      for (int hb = 0; hb < kHD / 32; ++hb)
        oacc[hb] = mfma(lds_col8(va, hb, 16 * tt * kHD * 2), pf[tt], oacc[hb]);
    // the next tile's scores spread over the exponentials, their operands read four MFMAs ahead;
    // then O, its operands four MFMAs (eight reads) ahead
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < 12; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
  };
  using Mask = std::integral_constant<bool, true>;
  using Full = std::integral_constant<bool, false>;
  // V of tile t and K of tile t + 1 are in LDS; K of tile t + 2 goes where tile t's was (its scores are
  // done), V of tile t + 1 where tile t - 1's was
  auto fetch = [&](int t) {
    issue_v(t + 1);
    issue(kw, Ks);
  };
  auto next = [&]() {
    wait_vmem<0>();
    __syncthreads();
  };
  // seen whole by every row (and not the last: without that test the compiler spilled registers)
  auto full = [&](int t) { return t + 1 < n_tiles && full_tile(it, it.tb + t); };
  int t = 0;
  while (t < n_tiles) {
    for (; full(t) && full(t + 1); t += 2) {   // the two score buffers need no copies
      fetch(t);
      tile(t, sc, sn, Full{});
      next();
      fetch(t + 1);
      tile(t + 1, sn, sc, Full{});
      next();
    }
    if (t < n_tiles) {
      fetch(t);
      tile(t, sc, sn, Mask{});
      sc[0] = sn[0];
      sc[1] = sn[1];
      next();
      ++t;
    }
  }
  l_i = __fadd_rn(l_i, __shfl_xor(l_i, 32));
  if (it.slot >= 0) {
    float* part = parts + (int64_t)it.slot * kPartFloats;
#pragma unroll
    for (int hb = 0; hb < kHD / 32; ++hb)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(part + part_off(wave, hb, q, lane)) = quad(oacc[hb], q);
    if (hl == 0) {
      part[kBM * kHD + row] = m_i;
      part[kBM * kHD + kBM + row] = l_i;
    }
    return;
  }
  // the wave's 32 x 128 block of O staged in the (now free) ring, one correctly rounded reciprocal per
  // row, and written back 16 bytes per lane, four whole 256-byte rows per store
  static_assert(4 * 32 * kStride16 <= 2 * kStages * kTileHalves, "O staging in the ring");
  f16* ostage = ring + wave * 32 * kStride16;
  const float inv_l = __fdiv_rn(1.0f, l_i);   // rows past the block: not stored
  // NaN if anything is not finite, also where P's rounding took a mean of values at the type's maximum
  // past it (the redone row holds P in fp32)
  f16x4 chk = {0, 0, 0, 0};
#pragma unroll
  for (int hb = 0; hb < kHD / 32; ++hb)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f16x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = (f16)__fmul_rn(oacc[hb][4 * q + e], inv_l);
      }
      chk = __builtin_elementwise_fma(o, f16x4{0, 0, 0, 0}, chk);
      *reinterpret_cast<f16x4*>(ostage + c * kStride16 + hb * 32 + 8 * q + 4 * hl) = o;
    }
  float sum = __fadd_rn((float)(chk[0] + chk[1]), (float)(chk[2] + chk[3]));
  sum = __fadd_rn(__builtin_fmaf(l_i, 0.0f, sum), __shfl_xor(sum, 32));
  if (sum != 0.0f) bad[row] = 1;
  else if (mval && hl == 0) lse[(int64_t)h * a.n_tokens + m] = __fadd_rn(m_i, log2f(l_i));
  __syncthreads();
  store_rows(a, it, wave, lane, ostage, bad, out);
  redo_rows(a, it.t0, it.phase, it.rows, it.g, bad, out, lse);
}

// The partials of a block put together: O = sum_s O_s 2^(m_s - m) / l, m = max m_s, l likewise, in slot
// order.  A workgroup per 32 rows, a wave per 32 columns, four partials' loads in flight.
__global__ __launch_bounds__(kAThreads) void span_join_kernel(SpanArgs a, const int32_t* __restrict__ joins,
                                                              int n_slots, f16* __restrict__ out,
                                                              float* __restrict__ lse,
                                                              const float* __restrict__ parts) {
  const int32_t* j = joins + (int64_t)(blockIdx.x >> 2) * DK_ATTN_SPAN_JOIN_INTS;
  const int qw = blockIdx.x & 3;   // the row group
  auto u = [&](int k) { return __builtin_amdgcn_readfirstlane(j[k]); };
  int t0 = u(0), phase = u(1), rows = u(2);
  const int g = u(3), s0 = u(4), cnt = u(5);
  const int gin = a.nq / a.nkv;
  if (t0 < 0 || phase < 0 || phase >= gin || rows < 1 || rows > kBM || g < 0 || g >= a.nkv ||
      (int64_t)t0 + (phase + rows - 1) / gin >= a.n_tokens || s0 < 0 || cnt < 1 || cnt > n_slots - s0 ||
      rows <= 32 * qw)
    return;
  rows = rows - 32 * qw < 32 ? rows - 32 * qw : 32;   // the group's own rows
  t0 += (phase + 32 * qw) / gin;
  phase = (phase + 32 * qw) % gin;
  __shared__ __attribute__((aligned(16))) f16 stage[32 * kStride16];
  __shared__ int bad[32];
  if (threadIdx.x < 32) bad[threadIdx.x] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 63, hb = threadIdx.x >> 6, hl = lane >> 5, c = lane & 31;
  const float* p0 = parts + (int64_t)s0 * kPartFloats;
  const float* ml = p0 + kBM * kHD + 32 * qw + c;
  float mm = -1.0e30f, l = 0.0f;
  for (int s = 0; s < cnt; ++s) mm = fmaxf(mm, ml[(int64_t)s * kPartFloats]);
  f32x4 o[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) o[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const float* p = p0 + part_off(qw, hb, 0, lane);
  for (int s = 0; s < cnt; s += 4) {
    f32x4 t[4][4];
    float w[4], ls[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t x = (int64_t)(s + i < cnt ? s + i : cnt - 1) * kPartFloats;
#pragma unroll
      for (int q = 0; q < 4; ++q) t[i][q] = *reinterpret_cast<const f32x4*>(p + x + 256 * q);
      w[i] = ml[x];
      ls[i] = ml[x + kBM];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (s + i >= cnt) break;
      w[i] = ex2(__fsub_rn(w[i], mm));
      l = __builtin_fmaf(ls[i], w[i], l);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[q][e] = __builtin_fmaf(t[i][q][e], w[i], o[q][e]);
    }
  }
  const float inv_l = __fdiv_rn(1.0f, l);
  float chk = __fmul_rn(l, 0.0f);   // NaN if a value is not finite, rounded
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    f16x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = (f16)__fmul_rn(o[q][e], inv_l);
      chk = __builtin_fmaf((float)x[e], 0.0f, chk);
    }
    *reinterpret_cast<f16x4*>(stage + c * kStride16 + hb * 32 + 8 * q + 4 * hl) = x;
  }
  if (chk != 0.0f) bad[c] = 1;
  __syncthreads();
  if (threadIdx.x < rows && !bad[threadIdx.x]) {   // wave 0, its first half: c is the row
    const int rr = phase + c;
    lse[(int64_t)(g * gin + rr % gin) * a.n_tokens + t0 + rr / gin] = __fadd_rn(mm, log2f(l));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 16 * i + (threadIdx.x >> 4), cc = lane & 15, rr = phase + r;
    const f16x8 v = *reinterpret_cast<const f16x8*>(stage + r * kStride16 + 8 * cc);
    if (r < rows && !bad[r])
      *reinterpret_cast<f16x8*>(out + ((int64_t)t0 + rr / gin) * a.nq * kHD +
                                (int64_t)(g * gin + rr % gin) * kHD + 8 * cc) = v;
  }
  redo_rows(a, t0, phase, rows, g, bad, out, lse);
}

}  // namespace

extern "C" int64_t dk_attn_span_workspace(int64_t n_slots) {
  return n_slots > 0 ? n_slots * (int64_t)(kPartFloats * sizeof(float)) : 0;
}

extern "C" int dk_attn_span_fwd(const void* qkv, const int32_t* spans, const int32_t* items,
                                int32_t n_items, const int32_t* joins, int32_t n_joins,
                                int32_t n_slots, int64_t n_tokens, int32_t nq, int32_t nkv, int32_t hd,
                                void* out, float* lse, void* workspace, int64_t workspace_bytes,
                                hipStream_t stream) {
  SpanArgs a;
  if (int e = span_args(a, qkv, spans, n_tokens, nq, nkv, hd)) return e;
  if (n_items < 0 || n_joins < 0 || n_slots < 0) return DK_ERR_INVALID;
  if (n_tokens == 0 || n_items == 0) return 0;
  if (!items || !out || !lse || (n_joins > 0 && !joins)) return DK_ERR_INVALID;
  if (!dk_aligned(out, 16) || !dk_aligned(lse, 4) || !dk_aligned(items, 4) || !dk_aligned(joins, 4) ||
      !dk_aligned(workspace, 256))
    return DK_ERR_ALIGN;
  if (n_slots > 0 && (!workspace || workspace_bytes < dk_attn_span_workspace(n_slots)))
    return DK_ERR_WORKSPACE;
  if (n_items > INT32_MAX / kAThreads || n_joins > INT32_MAX / (4 * kAThreads)) return DK_ERR_INVALID;
  hipLaunchKernelGGL(span_fwd_kernel, dim3((unsigned)n_items), dim3(kAThreads), 0, stream, a, items,
                     n_slots, (f16*)out, lse, (float*)workspace);
  DK_CHECK_LAUNCH();
  if (n_joins > 0) {
    hipLaunchKernelGGL(span_join_kernel, dim3((unsigned)(4 * n_joins)), dim3(kAThreads), 0, stream, a, joins,
                       n_slots, (f16*)out, lse, (const float*)workspace);
    DK_CHECK_LAUNCH();
  }
  return 0;
}
