// Backward of the attention over part of the keys (attn_span.h): P = 2^(s - lse), delta = out . dout,
// dS = P (dout V^T - delta), dq = dS K / sqrt(hd), dk = dS^T q / sqrt(hd) and dv = P^T dout, the last two
// summed over the queries that see a key and the heads of its group.  Three launches: delta; dK/dV
// and dQ on MFMA tiles; the partials of walks that were split, if any.
//
// P and dS are rounded to fp16 for their products, half a step, 2^-11 of each value.  dS is P, about 1 over
// the keys that a row sees, times dout's size, so as it stands it would lie below 2^-14, where fp16's steps
// no longer shrink, for ordinary windows and gradients: both are held 2^up up (P by a larger exponent,
// which costs nothing for a row on a lane and one subtraction a value in dK/dV; the sums are scaled back
// in fp32), which puts the end of the shrinking steps at 2^-30 of its dO row's norm for dQ, and for dK and
// dV at 2^-34 of the walk's largest |delta| (up 15 at most: at 2^-40).  up is taken from dout and, for a
// block of keys, from the rows that see any of them, and moves nothing but where those steps end.
// out, which delta is taken from, is the returned fp16 one; sums, statistics and results are fp32 up to one
// rounding of dq, dk and dv.  Against 64 bits (2-norms) dq comes out 3.0 to 3.6e-4 off and dk 3.1 to 3.4e-4,
// of which dS 2.2e-4, their own rounding 2.1e-4 and delta 1.2e-4 (more where rows see few keys: 9e-4 in all at two),
// dv 2.9e-4, for any size of dout whose gradients fp16 holds (at dout ~ 1e-4 their own rounding is 2 to 4e-3
// of them, and nearly all of it).
//
// Bound: a tile's step (64 queries x 128 keys, or 128 rows x 64 keys) keeps attn.hip's order at one wave
// per SIMD, the next tile's products (in dK/dV all of S before dP) beside this tile's P and dS; it takes
// 2.1 us (dQ 1.7) at the clock that power allows, 40 % of the matrix rate, S and dP computed for dK/dV and
// again for dQ.  An item begins with 3 to 5 us for its rows and first tile and ends with 2 to 3 us of
// stores.  Neither the operand reads (left out, a tile is 0 to 4 % faster) nor the exponentials beside S
// and dP (half of them beside dK and dV: unchanged) bound a tile on their own; what the rest of a tile
// waits for is not known.
// Measured on MI355X, 12 query / 2 KV heads (the three launches, back to back): 8192 tokens, window 1024,
// 4 sinks 235 us; 2048 tokens, window 256, 41; a prompt of 4096 with 16 answers of 512 1098 (617 TFLOP/s).
// A subtraction a value more in dK/dV's P is 1 % of a tile; begun with delta in its accumulators, dP needs
// none.  dQ in a launch of its own (two workgroups to a CU) took 267, 53 and 1014 when these took 258, 47
// and 1088: its blocks fill the ends of the dK/dV walks.
#include "attn_delta.h"
#include "attn_span.h"

namespace {

constexpr int kUnitFloats = kBM * kHD;   // a partial of dQ; dK and dV take two
constexpr int64_t kDeltaWgs = 1 << 16;   // of the delta launch at most: 2^20 rows a round

// The tile ring of both backward kernels: a tile of two operands (kBN rows each) in one of four
// LDS stages, filled by LDS DMA.  Wave w's instruction i fills chunks (4 i + w) 64 + lane of an
// operand: row 16 i + 4 w + lane / 16, with a wave-uniform base per tile and a 32-bit offset per
// lane; rows past `rows` (the rows left in the sequence, less one) read that row (finite, masked
// to p = 0).
constexpr int kBwdStages = 4;
constexpr int kBwdLoads = kTileHalves / 8 / kAThreads;   // per operand per lane: 4
constexpr unsigned kStageBytes = kTileHalves * 2;

struct TileSource {
  uint64_t base;      // first row of tile 0
  unsigned rowb;      // bytes per row
  unsigned off0;      // this lane's offset for instruction 0
  unsigned chunk;     // this lane's (swizzled) chunk offset inside a row
};
__device__ __forceinline__ TileSource tile_source(const f16* base, int64_t row_halves, int wave,
                                                  int lane) {
  TileSource t;
  t.base = uniform64((uint64_t)base);
  t.rowb = (unsigned)(row_halves * (int64_t)sizeof(f16));
  const int r0 = 4 * wave + (lane >> 4);
  t.chunk = (unsigned)(((lane & 15) ^ swz16(r0)) << 4);
  t.off0 = (unsigned)r0 * t.rowb + t.chunk;
  return t;
}
__device__ __forceinline__ void tile_load(const TileSource& src, int64_t first_row, uint64_t more, int rows,
                                          const f16* stage, int wave) {
  const uint64_t tb = src.base + (uint64_t)first_row * src.rowb + more;
  const unsigned last = (unsigned)(rows < kBN ? rows : kBN) * src.rowb + src.chunk;
#pragma unroll
  for (int i = 0; i < kBwdLoads; ++i) {
    const unsigned off = src.off0 + (unsigned)(16 * i) * src.rowb;
    dma16s(tb, off < last ? off : last,
           __builtin_amdgcn_readfirstlane(lds_addr(stage + (4 * i + wave) * 512)));
  }
}

// A barrier that orders the LDS DMA waited for before it, without a wait for the operand reads in
// flight (they are of stages that no load in flight touches).
__device__ __forceinline__ void tile_barrier() {
  wait_vmem<0>();
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

constexpr int kAhead1 = 6, kAhead2 = 4;

// The up of the top.  dQ, per query row with |dO| = r: 2^up r lies in [2^5, 2^6) (up from 0 to 24).  |dS| is
// at most max |dP| / 2 (P (1 - P) of a difference of two), so it fits where the values' norms stay below
// 2^11; a row that does not is redone, as for any overflow.
constexpr int kUpRows = 24;
__device__ __forceinline__ int clamp_up(int up, int most) { return up < 0 ? 0 : up > most ? most : up; }
__device__ __forceinline__ int exponent(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }   // x >= 0
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }
__device__ __forceinline__ int up_of_row(float r2) { return clamp_up(5 - (exponent(r2) >> 1), kUpRows); }
__device__ __forceinline__ float norm2(const f16x8 (&x)[kHD / 16]) {   // of a row whose halves two lanes hold
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < kHD / 16; ++i)
#pragma unroll
    for (int e = 0; e < 8; e += 2)
      s = __builtin_amdgcn_fdot2(f16x2{x[i][e], x[i][e + 1]}, f16x2{x[i][e], x[i][e + 1]}, s, false);
  return __fadd_rn(s, __shfl_xor(s, 32));
}

// dK and dV, per walk: 2^up times the walk's largest |delta| lies in [2^9, 2^10) (up from 0 to 15, for P
// itself), so that dS fits up to 2^6 times that.  delta is the mean of a row's dP under P, about |dP| times the
// root of the sum of P^2, which is no less than P, so over a walk's rows no dS comes out larger by much: over
// 5686 blocks of drawn batches by 1.4 at most, 11 in a walk of a few rows.  Where one is 2^6 times larger,
// in a walk of a row or two whose delta happens to vanish, its key is redone as for any overflow.  A walk
// reads its deltas once before its first tile's P, behind the first products.  Setting up tile by tile
// instead (looking at the next tile beside dK's products and rescaling the sums where it was too much)
// took 9 to 13 % of the whole; norms' exponents in the deltas' last bits, for a bound, left noise in dS
// where it cancels to 0 (a row that sees one key).
constexpr int kUpKeys = 15;
__device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned finite_bits(float x) {   // of |x|, which they order; 0 where it is not finite
  const unsigned b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
// The deltas of the walk over query tiles [tb, te) (per_head to a head) of the heads from h0 on, kFlight to a
// thread at a time: 8 heads by 256 rows, 4 by 512, 2 by 1024 or 1 by 2048.  Where the walk has more than one
// head each is taken whole; what lies past the last row or head is that row or head again.
struct WalkScan {
  static constexpr int kFlight = 8;
  const float* row;
  int64_t n_tokens;
  int rows, heads, shift, r0, hb;
  __device__ __forceinline__ WalkScan(const float* delta, int64_t n, int h0, int k0, int qend, int per_head,
                                      int tb, int te)
      : n_tokens(n), r0(0), hb(0) {
    const int first = tb / per_head;
    heads = (te - 1) / per_head - first + 1;
    const int lo = heads > 1 ? 0 : (tb - first * per_head) * kBN;
    const int hi = heads > 1 ? qend - k0 : (te - first * per_head) * kBN;
    rows = (hi < qend - k0 ? hi : qend - k0) - lo;
    shift = heads > 4 ? 3 : heads > 2 ? 2 : heads - 1;
    row = delta + (int64_t)(h0 + first) * n + k0 + lo;
  }
  __device__ __forceinline__ void load(float (&d)[kFlight]) const {
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const int h = hb + (u & ((1 << shift) - 1));
      const unsigned r = (unsigned)r0 + (unsigned)(u >> shift) * kAThreads + threadIdx.x, last = (unsigned)rows - 1;
      d[u] = *reinterpret_cast<const float*>(
          reinterpret_cast<const char*>(row + (h < heads ? h : heads - 1) * n_tokens) + (r < last ? r : last) * 4u);
    }
  }
  __device__ __forceinline__ bool next() {
    r0 += (kFlight >> shift) * kAThreads;
    if (r0 < rows) return true;
    r0 = 0;
    hb += kFlight;
    return hb < heads;
  }
};
// The bits of this thread's largest, from its first loads and the rest of the walk's.
__device__ __forceinline__ unsigned walk_peak(WalkScan scan, float (&d)[WalkScan::kFlight]) {
  unsigned p = 0;
  for (;;) {
#pragma unroll
    for (int u = 0; u < WalkScan::kFlight; ++u) p = larger(p, finite_bits(d[u]));
    if (!scan.next()) return p;
    scan.load(d);
  }
}
// the largest of the wave's lanes, in every lane: within the rows of 16, then on to the next rows
template <int kCtrl>
__device__ __forceinline__ unsigned larger_dpp(unsigned x) {
  return larger(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, 0xf, 0xf, false));
}
__device__ __forceinline__ unsigned wave_largest(unsigned x) {
  x = larger_dpp<0x118>(larger_dpp<0x114>(larger_dpp<0x112>(larger_dpp<0x111>(x))));
  return (unsigned)__builtin_amdgcn_readlane((int)larger_dpp<0x143>(larger_dpp<0x142>(x)), 63);
}
// the wave's part into peaks, read behind a barrier
__device__ __forceinline__ void peak_out(unsigned p, int wave, unsigned* peaks) {
  p = wave_largest(p);
  if ((threadIdx.x & 63) == 0) peaks[wave] = p;
}
__device__ __forceinline__ int up_of_walk(const unsigned* peaks) {
  const unsigned p = larger(larger(peaks[0], peaks[1]), larger(peaks[2], peaks[3]));
  return __builtin_amdgcn_readfirstlane(clamp_up(9 - exponent(__uint_as_float(p)), kUpKeys));
}

// The rows (or keys) whose result is not finite, recomputed over exactly what they see: 0 times a NaN
// or infinity of a masked row is not 0.  bad: row flags in LDS, written before a barrier.
__device__ __forceinline__ void redo_dq(const SpanArgs& a, int t0, int phase, int rows, int g,
                                        const int* bad, const f16* dout, const float* lse,
                                        const float* delta, f16* dq) {
  const int gin = a.nq / a.nkv;
  bad_rows(bad, rows, [&](int i) {
    span_row_dq(a, t0 + (phase + i) / gin, g * gin + (phase + i) % gin, dout, lse, delta, dq);
  });
}
__device__ __forceinline__ void redo_dkdv(const SpanArgs& a, int k0, int nk, int g, const int* bad,
                                          const f16* dout, const float* lse, const float* delta,
                                          f16* dk, f16* dv) {
  bad_rows(bad, nk, [&](int i) { span_key_dkdv(a, (int64_t)k0 + i, g, dout, lse, delta, dk, dv); });
}

// The wave's 32 keys of dK and dV, rounded, staged in its quarter of two LDS buffers and written back
// 16 bytes per lane, four whole rows per store.  Result register v of block hb: key 32 w +
// 8 (v / 4) + 4 (l / 32) + v % 4, column 32 hb + l % 32.
__device__ __forceinline__ void store_dkdv(const SpanArgs& a, int k0, int nk, int g,
                                           const f32x16 (&dkacc)[kHD / 32], const f32x16 (&dvacc)[kHD / 32],
                                           f16* s0, f16* s1, int* bad, f16* dk, f16* dv) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, hl = lane >> 5, c = lane & 31;
  f16* kst = s0 + w * 32 * kStride16;
  f16* vst = s1 + w * 32 * kStride16;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int r = 8 * (v >> 2) + 4 * hl + (v & 3);
    float chk = 0.0f;   // NaN if a value is not finite
#pragma unroll
    for (int hb = 0; hb < kHD / 32; ++hb) {
      chk = __builtin_fmaf(dkacc[hb][v], 0.0f, __builtin_fmaf(dvacc[hb][v], 0.0f, chk));
      kst[r * kStride16 + hb * 32 + c] = (f16)__fmul_rn(dkacc[hb][v], a.sm_scale);
      vst[r * kStride16 + hb * 32 + c] = (f16)dvacc[hb][v];
    }
    if (chk != 0.0f) bad[32 * w + r] = 1;
  }
  __syncthreads();
  const int key = 32 * w + (lane >> 4), cc = lane & 15;
  int keep[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) keep[i] = (key + 4 * i < nk) & !bad[key + 4 * i];
  const int64_t o = (((int64_t)k0 + key) * a.nkv + g) * kHD + 8 * cc;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + (lane >> 4);
    const f16x8 kv = *reinterpret_cast<const f16x8*>(kst + r * kStride16 + 8 * cc);
    const f16x8 vv = *reinterpret_cast<const f16x8*>(vst + r * kStride16 + 8 * cc);
    if (keep[i]) {
      *reinterpret_cast<f16x8*>(dk + o + (int64_t)(4 * i) * a.nkv * kHD) = kv;
      *reinterpret_cast<f16x8*>(dv + o + (int64_t)(4 * i) * a.nkv * kHD) = vv;
    }
  }
}

// Up to 32 rows of dQ (or keys of dK and dV), wave hb holding columns 32 hb .. + 31 of them as quads,
// rounded, staged and written back.  bad [32] is zero before.
__device__ __forceinline__ void store_group(const SpanArgs& a, bool keys, int t0, int phase, int rows,
                                            int g, int hb, const f32x4 (&x)[4], const f32x4 (&y)[4],
                                            f16* S0, f16* S1, int* bad, f16* dq, f16* dk, f16* dv) {
  const int lane = threadIdx.x & 63, hl = lane >> 5, c = lane & 31, gin = a.nq / a.nkv;
  // staged as rows of 128: dq's lane holds 16 columns of its row, dK's and dV's a column of 16 keys
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (!keys) {
      f16x4 o;
      float chk = 0.0f;   // NaN if a value is not finite
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        chk = __builtin_fmaf(x[q][e], 0.0f, chk);
        o[e] = (f16)__fmul_rn(x[q][e], a.sm_scale);
      }
      if (chk != 0.0f) bad[c] = 1;
      *reinterpret_cast<f16x4*>(S0 + c * kStride16 + hb * 32 + 8 * q + 4 * hl) = o;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 8 * q + 4 * hl + e;
        if (__builtin_fmaf(x[q][e], 0.0f, __fmul_rn(y[q][e], 0.0f)) != 0.0f) bad[r] = 1;
        S0[r * kStride16 + hb * 32 + c] = (f16)__fmul_rn(x[q][e], a.sm_scale);
        S1[r * kStride16 + hb * 32 + c] = (f16)y[q][e];
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 16 * i + (threadIdx.x >> 4), cc = lane & 15;
    if (r >= rows || bad[r]) continue;
    const f16x8 v = *reinterpret_cast<const f16x8*>(S0 + r * kStride16 + 8 * cc);
    if (keys) {
      const int64_t o = ((int64_t)t0 + r) * a.nkv * kHD + (int64_t)g * kHD + 8 * cc;
      *reinterpret_cast<f16x8*>(dk + o) = v;
      *reinterpret_cast<f16x8*>(dv + o) = *reinterpret_cast<const f16x8*>(S1 + r * kStride16 + 8 * cc);
    } else {
      const int rr = phase + r;
      *reinterpret_cast<f16x8*>(dq + ((int64_t)t0 + rr / gin) * a.nq * kHD +
                                (int64_t)(g * gin + rr % gin) * kHD + 8 * cc) = v;
    }
  }
}

// dQ of a block of stacked query rows, over the key tiles of its item
__device__ __forceinline__ void dq_item(const SpanArgs& a, const int32_t* items, int idx, int n_units,
                                        const f16* __restrict__ dout, const float* __restrict__ lse,
                                        const float* __restrict__ delta, f16* __restrict__ dq,
                                        float* __restrict__ parts, f16* Ks, f16* Vs, int (*ends)[kBN],
                                        int* bad) {
  SpanItem it;
  if (!span_item(a, items, idx, n_units, &it)) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, hl = lane >> 5, c = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(w);
  const int64_t ROW = (int64_t)(a.nq + 2 * a.nkv) * kHD, OROW = (int64_t)a.nq * kHD;
  const int gin = a.nq / a.nkv, row = 32 * w + c;
  const bool mval = row < it.rows;
  const int rr = it.phase + (mval ? row : 0);
  const int m = it.t0 + rr / gin, h = it.g * gin + rr % gin;
  const int jlim = mval ? m - it.b0 + it.na : -1;   // this lane's last key

  const int n_tiles = it.te - it.tb;
  const KeySource src = key_source(ROW, wave, lane);
  const uint64_t kbase = uniform64((uint64_t)(a.qkv + (int64_t)(a.nq + it.g) * kHD));
  const uint64_t vbase = kbase + (uint64_t)a.nkv * kHD * sizeof(f16);
  KeyWalk kw = key_walk(it, kbase, src.rowb), vw = key_walk(it, vbase, src.rowb);
  auto issue = [&](int t) {
    if (t >= n_tiles) return;
    const int st = t % kBwdStages;
    next_key_tile<4>(it, kw, src, Ks + st * kTileHalves, wave);
    next_key_tile<4>(it, vw, src, Vs + st * kTileHalves, wave);
    if (wave == 0) key_ends_load(a, it, it.tb + t, ends[st], lane);
  };
  issue(0);
  // this lane's query and dO rows and statistics, loaded unconditionally and selected at once (the
  // compiler's wait for them stands here, not in the loop)
  f16x8 qf[kHD / 16], dof[kHD / 16];
  float lse_m, dl_m;
  {
    const f16* qrow = a.qkv + (int64_t)m * ROW + (int64_t)h * kHD + 8 * hl;
    const f16* drow = dout + (int64_t)m * OROW + (int64_t)h * kHD + 8 * hl;
#pragma unroll
    for (int s = 0; s < kHD / 16; ++s) {
      qf[s] = *reinterpret_cast<const f16x8*>(qrow + 16 * s);
      dof[s] = *reinterpret_cast<const f16x8*>(drow + 16 * s);
    }
    lse_m = lse[(int64_t)h * a.n_tokens + m];
    dl_m = delta[(int64_t)h * a.n_tokens + m];
#pragma unroll
    for (int s = 0; s < kHD / 16; ++s) asm volatile("" : "+v"(qf[s]), "+v"(dof[s]));
    asm volatile("" : "+v"(lse_m), "+v"(dl_m));
#pragma unroll
    for (int s = 0; s < kHD / 16; ++s) {
      qf[s] = mval ? qf[s] : zero8();
      dof[s] = mval ? dof[s] : zero8();
    }
    lse_m = mval ? lse_m : 0.0f;
    dl_m = mval ? dl_m : 0.0f;
  }
  const int up = up_of_row(norm2(dof));
  const float up_lse = __fsub_rn((float)up, lse_m);
  if (threadIdx.x < kBM) bad[threadIdx.x] = 0;
  f32x16 dqacc[kHD / 32];
#pragma unroll
  for (int hb = 0; hb < kHD / 32; ++hb) dqacc[hb] = zero16();
  const unsigned krow = lds_addr(Ks) + row_base(lane), vrow = lds_addr(Vs) + row_base(lane);
  const unsigned kcol = lds_addr(Ks) + col_base(lane);
  // operand i of a tile's products: S^T = K Q^T and dP^T = V dO^T (keys kb * 32 + (row), queries
  // on the lanes): sub-step i / 4, dP^T for i / 2 odd, key half i % 2
  auto rd1 = [&](unsigned ka, unsigned va, int i) {
    return lds_read8((((i >> 1) & 1) ? va : ka) ^ (unsigned)(32 * (i >> 2)), (i & 1) * 32 * kHD * 2);
  };
  f32x16 delta0;   // what dP^T begins with, for dP - delta
#pragma unroll
  for (int v = 0; v < 16; ++v) delta0[v] = -dl_m;
  auto product = [&](f32x16 (&sacc)[2], f32x16 (&dpacc)[2], const f16x8& f, int i) {
    const int s = i >> 2, kb = i & 1;
    if ((i >> 1) & 1) dpacc[kb] = mfma(f, dof[s], s == 0 ? delta0 : dpacc[kb]);
    else sacc[kb] = mfma(f, qf[s], s == 0 ? zero16() : sacc[kb]);
  };
  f16x8 fr[kAhead1];
  tile_barrier();
  issue(1);   // behind the rows and tile 0, which the first products wait for
  f32x16 s_a[2], d_a[2], s_b[2], d_b[2];
  {
    const unsigned ka = fresh(krow), va = fresh(vrow);
#pragma unroll
    for (int i = 0; i < kAhead1; ++i) fr[i] = rd1(ka, va, i);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      product(s_a, d_a, fr[i % kAhead1], i);
      if (i + kAhead1 < 32) fr[i % kAhead1] = rd1(ka, va, i + kAhead1);
      __builtin_amdgcn_sched_barrier(0);
    }
    tile_barrier();
    issue(2);
    const unsigned ka1 = fresh(krow + kStageBytes), va1 = fresh(vrow + kStageBytes);
#pragma unroll
    for (int i = 0; i < kAhead1; ++i) fr[i] = rd1(ka1, va1, i);
  }
  auto step = [&](int t, f32x16 (&sc)[2], f32x16 (&dc)[2], f32x16 (&sn)[2], f32x16 (&dn)[2],
                  auto more_c) {
    constexpr bool MORE = decltype(more_c)::value;   // tile t + 1 exists
    // key j of a tile that some row of the block does not see whole is kept iff j <= jlim and its end
    // lies past this lane's token; the others' probabilities come out as 0.  Rows past the block have
    // zero q, dO and delta, so their dS is zero whatever P is.
    if (!full_tile(it, it.tb + t)) {
      const int lim = jlim - (it.tb + t) * kBN - 4 * hl;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const i32x4 e4 = *reinterpret_cast<const i32x4*>(&ends[t % kBwdStages][8 * q + 4 * hl]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sc[q >> 2][4 * (q & 3) + e] =
              ((8 * q + e <= lim) & (m < e4[e])) ? sc[q >> 2][4 * (q & 3) + e] : -1.0e30f;
      }
    }
    const unsigned nst = (unsigned)((t + 1) % kBwdStages) * kStageBytes;
    const unsigned ka = fresh(krow + nst), va = fresh(vrow + nst);
    const unsigned kc = fresh(kcol + (unsigned)(t % kBwdStages) * kStageBytes);
    auto rd2 = [&](int i) { return lds_col8(kc, i & 3, 16 * (i >> 2) * kHD * 2); };
    Frag8 dsf[kBN / 16];
    f16x8 gr[kAhead2];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if constexpr (MORE) {
        product(sn, dn, fr[i % kAhead1], i);
        if (i + kAhead1 < 32) fr[i % kAhead1] = rd1(ka, va, i + kAhead1);
      }
      const int kb = i >> 4, v = i & 15;
      const float p = ex2(__builtin_fmaf(sc[kb][v], a.qk_scale, up_lse));
      dc[kb][v] = __fmul_rn(p, dc[kb][v]);
      if (i & 1) dsf[i >> 3].h[(i >> 1) & 3] = pinned(dc[kb][v - 1], dc[kb][v]);
      if (i >= 32 - kAhead2) gr[i - (32 - kAhead2)] = rd2(i - (32 - kAhead2));
      if constexpr (MORE) __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (MORE) {
      tile_barrier();
      issue(t + 3);
    }
    const unsigned nst2 = (unsigned)((t + 2) % kBwdStages) * kStageBytes;
    const unsigned ka2 = fresh(krow + nst2), va2 = fresh(vrow + nst2);
    // dQ^T += K^T dS^T
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      dqacc[i & 3] = mfma(gr[i % kAhead2], dsf[i >> 2].get(), dqacc[i & 3]);
      if (i + kAhead2 < 16) gr[i % kAhead2] = rd2(i + kAhead2);
      // (past the last tile: a stale stage, never used)
      if (MORE && i >= 16 - kAhead1) fr[i - (16 - kAhead1)] = rd1(ka2, va2, i - (16 - kAhead1));
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using More = std::integral_constant<bool, true>;
  using Last = std::integral_constant<bool, false>;
  int t = 0;
  for (; t + 2 < n_tiles; t += 2) {
    step(t, s_a, d_a, s_b, d_b, More{});
    step(t + 1, s_b, d_b, s_a, d_a, More{});
  }
  if (t + 1 < n_tiles) {
    step(t, s_a, d_a, s_b, d_b, More{});
    ++t;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      s_a[kb] = s_b[kb];
      d_a[kb] = d_b[kb];
    }
  }
  step(t, s_a, d_a, s_b, d_b, Last{});
  const float back = pow2(-up);
#pragma unroll
  for (int hb = 0; hb < kHD / 32; ++hb)
#pragma unroll
    for (int v = 0; v < 16; ++v) dqacc[hb][v] = __fmul_rn(dqacc[hb][v], back);
  __syncthreads();
  if (it.slot >= 0) {
    float* part = parts + (int64_t)it.slot * kUnitFloats;
#pragma unroll
    for (int hb = 0; hb < kHD / 32; ++hb)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(part + part_off(w, hb, q, lane)) = quad(dqacc[hb], q);
    return;
  }
  // the wave's 32 x 128 block of dQ staged in the (now free) tile ring, then written back 16 bytes per
  // lane, four whole 256-byte rows per store instruction
  f16* stage = Ks + w * 32 * kStride16;
  float chk = 0.0f;   // NaN if a value is not finite
#pragma unroll
  for (int hb = 0; hb < kHD / 32; ++hb)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f16x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        chk = __builtin_fmaf(dqacc[hb][4 * q + e], 0.0f, chk);
        o[e] = (f16)__fmul_rn(dqacc[hb][4 * q + e], a.sm_scale);
      }
      *reinterpret_cast<f16x4*>(stage + c * kStride16 + hb * 32 + 8 * q + 4 * hl) = o;
    }
  if (chk != 0.0f) bad[row] = 1;
  __syncthreads();
  store_rows(a, it, w, lane, stage, bad, dq);
  redo_dq(a, it.t0, it.phase, it.rows, it.g, bad, dout, lse, delta, dq);
}

// dK and dV of a block of up to kBM keys, summed over the heads of the KV head's group: K and V stay in
// registers while the walk goes over every head's query tiles, from the block's first key to the last
// query that sees any of its keys.  The Q and dO tiles and the tiles' lse and delta rows (by dword DMA,
// one lane per query, waves 0 and 1) come through the four-stage ring.
__device__ __forceinline__ void dkdv_item(const SpanArgs& a, const int32_t* items, int idx, int n_units,
                                          const f16* __restrict__ dout, const float* __restrict__ lse,
                                          const float* __restrict__ delta, f16* __restrict__ dk,
                                          f16* __restrict__ dv, float* __restrict__ parts, f16* Qs,
                                          f16* Ds, float (*lse_s)[kBN], float (*dl_s)[kBN], int* bad,
                                          unsigned* peaks) {
  const int32_t* p = items + (int64_t)idx * kItemInts;
  auto u = [&](int k) { return __builtin_amdgcn_readfirstlane(p[k]); };
  const int k0 = u(0), nk = u(2), g = u(3), qend = u(4), tb = u(11), te = u(12), slot = u(13);
  const int gin = a.nq / a.nkv;
  if (k0 < 0 || nk < 1 || nk > kBM || g < 0 || g >= a.nkv || (int64_t)k0 + nk > a.n_tokens ||
      qend <= k0 || qend > a.n_tokens || tb < 0 || tb >= te || (slot >= 0 && slot > n_units - 2))
    return;
  const int per_head = (qend - k0 + kBN - 1) / kBN;   // query tiles of a head's walk
  if (te > (int64_t)gin * per_head) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, hl = lane >> 5, c = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(w);
  const int64_t ROW = (int64_t)(a.nq + 2 * a.nkv) * kHD, OROW = (int64_t)a.nq * kHD;
  const bool nval = 32 * w + c < nk;
  const int n = k0 + (nval ? 32 * w + c : 0);   // this lane's key

  const int n_tiles = te - tb;
  if (tid < kBN) lse_s[kBwdStages][tid] = 0.0f;
  if (tid < kBM) bad[tid] = 0;
  const TileSource qsrc = tile_source(a.qkv + (int64_t)k0 * ROW + (int64_t)g * gin * kHD, ROW, wave, lane);
  const TileSource dsrc = tile_source(dout + (int64_t)k0 * OROW + (int64_t)g * gin * kHD, OROW, wave, lane);
  // The walk: every head of the group in turn, each over the query tiles k0 + 64 i up to qend.  Tiles
  // are issued in order: (head, tile of the head) of the next one.
  int ihead = tb / per_head, itile = tb % per_head;
  int walk = itile;   // and of the next step
  auto issue = [&](int t) {
    if (t >= n_tiles) return;
    const int st = t % kBwdStages, m0 = k0 + itile * kBN;
    tile_load(qsrc, (int64_t)itile * kBN, (uint64_t)ihead * kHD * 2, qend - 1 - m0, Qs + st * kTileHalves, wave);
    tile_load(dsrc, (int64_t)itile * kBN, (uint64_t)ihead * kHD * 2, qend - 1 - m0, Ds + st * kTileHalves, wave);
    if (wave < 2) {
      const int qq = m0 + lane < qend ? m0 + lane : qend - 1;
      const float* src = (wave == 0 ? lse : delta) + (int64_t)(g * gin + ihead) * a.n_tokens + qq;
      dma4(src, __builtin_amdgcn_readfirstlane(lds_addr(wave == 0 ? lse_s[st] : dl_s[st])));
    }
    if (++itile == per_head) {
      itile = 0;
      ++ihead;
    }
  };
  issue(0);

  // this lane's key row and its value row negated as B operands, loaded unconditionally and selected at
  // once (the compiler's wait for them, and for the walk's first deltas, stands here, not in the loop)
  const int end = (int)key_end(a, n);
  f16x8 kf[kHD / 16], vf[kHD / 16];
  const WalkScan scan(delta, a.n_tokens, g * gin, k0, qend, per_head, tb, te);
  float first[WalkScan::kFlight];
  {
    const f16* krow = a.qkv + (int64_t)n * ROW + (int64_t)(a.nq + g) * kHD + 8 * hl;
    const f16* vrow = krow + (int64_t)a.nkv * kHD;
#pragma unroll
    for (int s = 0; s < kHD / 16; ++s) {
      kf[s] = *reinterpret_cast<const f16x8*>(krow + 16 * s);
      vf[s] = *reinterpret_cast<const f16x8*>(vrow + 16 * s);
    }
    scan.load(first);
#pragma unroll
    for (int s = 0; s < kHD / 16; ++s) asm volatile("" : "+v"(kf[s]), "+v"(vf[s]));
#pragma unroll
    for (int s = 0; s < kHD / 16; ++s) {
      kf[s] = nval ? kf[s] : zero8();
      vf[s] = nval ? -vf[s] : zero8();
    }
  }
  // the first end among the wave's keys
  int end_min = nval ? end : INT32_MAX;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) end_min = min(end_min, __shfl_xor(end_min, x));
  end_min = __builtin_amdgcn_readfirstlane(end_min);
  f32x16 dkacc[kHD / 32], dvacc[kHD / 32];
#pragma unroll
  for (int hb = 0; hb < kHD / 32; ++hb) dkacc[hb] = dvacc[hb] = zero16();
  const unsigned qrow = lds_addr(Qs) + row_base(lane), drow = lds_addr(Ds) + row_base(lane);
  const unsigned qcol = lds_addr(Qs) + col_base(lane), dcol = lds_addr(Ds) + col_base(lane);
  // operand i of a tile's products S = Q K^T and then delta - dP = delta + dO (-V)^T (queries qb * 32 +
  // (row of the result), keys on the lanes): sub-step i % 16 / 2, query half i % 2.  The second begin with
  // delta in their accumulators, read beside the first.
  auto rd1 = [&](unsigned qa, unsigned da, int i) {
    return lds_read8((i < 16 ? qa : da) ^ (unsigned)(32 * ((i & 15) >> 1)), (i & 1) * 32 * kHD * 2);
  };
  auto product = [&](f32x16 (&sacc)[2], f32x16 (&dpacc)[2], const f16x8& f, int i) {
    const int s = (i & 15) >> 1, qb = i & 1;
    if (i >= 16) dpacc[qb] = mfma(f, vf[s], dpacc[qb]);
    else sacc[qb] = mfma(f, kf[s], s == 0 ? zero16() : sacc[qb]);
  };
  // the statistics of rows 8 g + 4 (l / 32) + 0..3 of the tile in stage st (g = 0..7)
  auto stat = [&](const float (*tab)[kBN], int st, int g) {
    return *reinterpret_cast<const f32x4*>(&tab[st][8 * g + 4 * hl]);
  };
  f16x8 fr[kAhead1];
  f32x4 ls[2];
  auto delta_in = [&](f32x16 (&d)[2], int st, int g) {
    const f32x4 x = stat(dl_s, st, g);
#pragma unroll
    for (int e = 0; e < 4; ++e) d[g >> 2][4 * (g & 3) + e] = x[e];
  };
  tile_barrier();
  issue(1);   // behind the rows and tile 0, which the first products wait for
  f32x16 s_a[2], d_a[2], s_b[2], d_b[2];
  {
    const unsigned qa = fresh(qrow), da = fresh(drow);
#pragma unroll
    for (int g = 0; g < 8; ++g) delta_in(d_a, 0, g);
#pragma unroll
    for (int i = 0; i < kAhead1; ++i) fr[i] = rd1(qa, da, i);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      product(s_a, d_a, fr[i % kAhead1], i);
      if (i + kAhead1 < 32) fr[i % kAhead1] = rd1(qa, da, i + kAhead1);
      __builtin_amdgcn_sched_barrier(0);
    }
    peak_out(walk_peak(scan, first), wave, peaks);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the row of zeros and the peaks are written
    tile_barrier();
    issue(2);
    const unsigned qa1 = fresh(qrow + kStageBytes), da1 = fresh(drow + kStageBytes);
#pragma unroll
    for (int i = 0; i < kAhead1; ++i) fr[i] = rd1(qa1, da1, i);
    ls[0] = stat(lse_s, 0, 0);
  }
  const int up = up_of_walk(peaks);
  const float upf = (float)up;
  auto step = [&](int t, f32x16 (&sc)[2], f32x16 (&dc)[2], f32x16 (&sn)[2], f32x16 (&dn)[2],
                  auto more_c) {
    constexpr bool MORE = decltype(more_c)::value;   // tile t + 1 exists
    const int st = t % kBwdStages, m0 = k0 + walk * kBN;
    walk = walk + 1 == per_head ? 0 : walk + 1;
    // Keys past the block only reach rows that are not stored; queries before a key or at its end and
    // past it are masked only on the tiles that hold such a query for this wave (a wave-uniform
    // test): query m0 + off + 4 (l / 32) is kept iff lo <= off < hi.  There the exponent is formed before
    // the selection and the loop below is given scale 1 and a row of zeros for lse, so that the others'
    // probabilities are 0 whatever their lse is.
    float scale = a.qk_scale;
    int lrow = st;
    if (m0 < k0 + 32 * wave + 31 || m0 + kBN > end_min) {
      const int lo = n - m0 - 4 * hl, hi = end - m0 - 4 * hl;
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const f32x4 l = g == 0 ? ls[0] : stat(lse_s, st, g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int off = 8 * g + e;
          const float x = __builtin_fmaf(sc[g >> 2][4 * (g & 3) + e], a.qk_scale, -l[e]);
          sc[g >> 2][4 * (g & 3) + e] = ((off >= lo) & (off < hi)) ? x : -1.0e30f;
        }
      }
      scale = 1.0f;
      lrow = kBwdStages;
      ls[0] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const unsigned nst = (unsigned)((t + 1) % kBwdStages) * kStageBytes;
    const unsigned qa = fresh(qrow + nst), da = fresh(drow + nst);
    const unsigned qc = fresh(qcol + (unsigned)st * kStageBytes), dc_ = fresh(dcol + (unsigned)st * kStageBytes);
    auto rd2 = [&](int i) { return lds_col8((i & 1) ? qc : dc_, (i >> 1) & 3, 16 * (i >> 3) * kHD * 2); };
    Frag8 pf[kBN / 16], dsf[kBN / 16];
    f16x8 gr[kAhead2];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if constexpr (MORE) {
        product(sn, dn, fr[i % kAhead1], i);
        if (i + kAhead1 < 32) fr[i % kAhead1] = rd1(qa, da, i + kAhead1);
        if (i < 8) delta_in(dn, (t + 1) % kBwdStages, i);
      }
      const int qb = i >> 4, v = i & 15, g = i >> 2;
      if ((i & 3) == 0 && g + 1 < 8) ls[(g + 1) & 1] = stat(lse_s, lrow, g + 1);
      sc[qb][v] = ex2(__builtin_fmaf(sc[qb][v], scale, __fsub_rn(upf, ls[g & 1][i & 3])));
      dc[qb][v] = __fmul_rn(sc[qb][v], dc[qb][v]);
      if (i & 1) {
        pf[i >> 3].h[(i >> 1) & 3] = pinned(sc[qb][v - 1], sc[qb][v]);
        dsf[i >> 3].h[(i >> 1) & 3] = pinned(dc[qb][v - 1], dc[qb][v]);
      }
      if (i >= 32 - kAhead2) gr[i - (32 - kAhead2)] = rd2(i - (32 - kAhead2));
      if constexpr (MORE) __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (MORE) {
      tile_barrier();
      issue(t + 3);
    }
    const unsigned nst2 = (unsigned)((t + 2) % kBwdStages) * kStageBytes;
    const unsigned qa2 = fresh(qrow + nst2), da2 = fresh(drow + nst2);
    // dV += P^T dO, -dK += -dS^T Q over the tile's 64 queries, 16 per step
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int hb = (i >> 1) & 3;
      if (i & 1) dkacc[hb] = mfma(dsf[i >> 3].get(), gr[i % kAhead2], dkacc[hb]);
      else dvacc[hb] = mfma(pf[i >> 3].get(), gr[i % kAhead2], dvacc[hb]);
      if (i + kAhead2 < 32) gr[i % kAhead2] = rd2(i + kAhead2);
      if constexpr (MORE) {
        // (past the last tile: a stale stage, never used)
        if (i >= 32 - kAhead1) fr[i - (32 - kAhead1)] = rd1(qa2, da2, i - (32 - kAhead1));
        if (i == 28) ls[0] = stat(lse_s, (t + 1) % kBwdStages, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using More = std::integral_constant<bool, true>;
  using Last = std::integral_constant<bool, false>;
  int t = 0;
  for (; t + 2 < n_tiles; t += 2) {
    step(t, s_a, d_a, s_b, d_b, More{});
    step(t + 1, s_b, d_b, s_a, d_a, More{});
  }
  if (t + 1 < n_tiles) {
    step(t, s_a, d_a, s_b, d_b, More{});
    ++t;
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      s_a[qb] = s_b[qb];
      d_a[qb] = d_b[qb];
    }
  }
  step(t, s_a, d_a, s_b, d_b, Last{});
  const float back = pow2(-up);
#pragma unroll
  for (int hb = 0; hb < kHD / 32; ++hb)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      dkacc[hb][v] = __fmul_rn(dkacc[hb][v], -back);
      dvacc[hb][v] = __fmul_rn(dvacc[hb][v], back);
    }
  __syncthreads();
  if (slot >= 0) {
    float* part = parts + (int64_t)slot * kUnitFloats;
#pragma unroll
    for (int hb = 0; hb < kHD / 32; ++hb)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int o = part_off(w, hb, q, lane);
        *reinterpret_cast<f32x4*>(part + o) = quad(dkacc[hb], q);
        *reinterpret_cast<f32x4*>(part + kUnitFloats + o) = quad(dvacc[hb], q);
      }
    return;
  }
  store_dkdv(a, k0, nk, g, dkacc, dvacc, Qs, Ds, bad, dk, dv);
  redo_dkdv(a, k0, nk, g, bad, dout, lse, delta, dk, dv);
}

// The same for a block of at most 32 keys (sinks, whose walk is the whole sequence): a step takes two
// tiles, 32 queries of them to each wave, every wave against all the keys; the waves' sums are put
// together at the end.  Per 64 queries that is a quarter of the products that four groups of 32
// keys, three of them empty, would take: 2048 tokens with 4 sinks 54 -> 47 us.
__device__ __forceinline__ void dkdv_narrow(const SpanArgs& a, const int32_t* items, int idx, int n_units,
                                            const f16* __restrict__ dout, const float* __restrict__ lse,
                                            const float* __restrict__ delta, f16* __restrict__ dk,
                                            f16* __restrict__ dv, float* __restrict__ parts, f16* Qs,
                                            f16* Ds, float (*lse_s)[kBN], float (*dl_s)[kBN], int* bad,
                                            unsigned* peaks) {
  const int32_t* p = items + (int64_t)idx * kItemInts;
  auto u = [&](int k) { return __builtin_amdgcn_readfirstlane(p[k]); };
  const int k0 = u(0), nk = u(2), g = u(3), qend = u(4), tb = u(11), te = u(12), slot = u(13);
  const int gin = a.nq / a.nkv;
  if (k0 < 0 || nk < 1 || nk > 32 || g < 0 || g >= a.nkv || (int64_t)k0 + nk > a.n_tokens ||
      qend <= k0 || qend > a.n_tokens || tb < 0 || tb >= te || (slot >= 0 && slot > n_units - 2))
    return;
  const int per_head = (qend - k0 + kBN - 1) / kBN;
  if (te > (int64_t)gin * per_head) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, hl = lane >> 5, c = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(w);
  const int64_t ROW = (int64_t)(a.nq + 2 * a.nkv) * kHD, OROW = (int64_t)a.nq * kHD;
  const bool nval = c < nk;
  const int n = k0 + (nval ? c : 0);   // this lane's key
  if (tid < kBM) bad[tid] = 0;

  const int n_tiles = te - tb, n_steps = (n_tiles + 1) / 2;
  const TileSource qsrc = tile_source(a.qkv + (int64_t)k0 * ROW + (int64_t)g * gin * kHD, ROW, wave, lane);
  const TileSource dsrc = tile_source(dout + (int64_t)k0 * OROW + (int64_t)g * gin * kHD, OROW, wave, lane);
  int ihead = tb / per_head, itile = tb % per_head;
  auto issue = [&](int t) {
    if (t >= n_tiles) return;
    const int st = t % kBwdStages, m0 = k0 + itile * kBN;
    tile_load(qsrc, (int64_t)itile * kBN, (uint64_t)ihead * kHD * 2, qend - 1 - m0, Qs + st * kTileHalves, wave);
    tile_load(dsrc, (int64_t)itile * kBN, (uint64_t)ihead * kHD * 2, qend - 1 - m0, Ds + st * kTileHalves, wave);
    if (wave < 2) {
      const int qq = m0 + lane < qend ? m0 + lane : qend - 1;
      const float* src = (wave == 0 ? lse : delta) + (int64_t)(g * gin + ihead) * a.n_tokens + qq;
      dma4(src, __builtin_amdgcn_readfirstlane(lds_addr(wave == 0 ? lse_s[st] : dl_s[st])));
    }
    if (++itile == per_head) {
      itile = 0;
      ++ihead;
    }
  };
  issue(0);
  issue(1);
  const int end = (int)key_end(a, n);
  f16x8 kf[kHD / 16], vf[kHD / 16];
  const WalkScan scan(delta, a.n_tokens, g * gin, k0, qend, per_head, tb, te);
  float first[WalkScan::kFlight];
  {
    const f16* krow = a.qkv + (int64_t)n * ROW + (int64_t)(a.nq + g) * kHD + 8 * hl;
    const f16* vrow = krow + (int64_t)a.nkv * kHD;
#pragma unroll
    for (int s = 0; s < kHD / 16; ++s) {
      kf[s] = *reinterpret_cast<const f16x8*>(krow + 16 * s);
      vf[s] = *reinterpret_cast<const f16x8*>(vrow + 16 * s);
    }
    scan.load(first);
#pragma unroll
    for (int s = 0; s < kHD / 16; ++s) asm volatile("" : "+v"(kf[s]), "+v"(vf[s]));
#pragma unroll
    for (int s = 0; s < kHD / 16; ++s) {
      kf[s] = nval ? kf[s] : zero8();
      vf[s] = nval ? vf[s] : zero8();
    }
  }
  int end_min = nval ? end : INT32_MAX;
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) end_min = min(end_min, __shfl_xor(end_min, x));
  end_min = __builtin_amdgcn_readfirstlane(end_min);
  f32x16 dkacc[kHD / 32], dvacc[kHD / 32];
#pragma unroll
  for (int hb = 0; hb < kHD / 32; ++hb) dkacc[hb] = dvacc[hb] = zero16();
  const int half = wave & 1;   // this wave's 32 queries of its tile
  const unsigned hoff = (unsigned)(half * 32 * kHD * 2);
  const unsigned qrow = lds_addr(Qs) + row_base(lane) + hoff, drow = lds_addr(Ds) + row_base(lane) + hoff;
  const unsigned qcol = lds_addr(Qs) + col_base(lane) + hoff, dcol = lds_addr(Ds) + col_base(lane) + hoff;
  int walk = tb % per_head;   // the step's first tile within its head
  peak_out(walk_peak(scan, first), wave, peaks);
  __syncthreads();            // the peaks are written
  const int up = up_of_walk(peaks);
  const float upf = (float)up;
  for (int s = 0; s < n_steps; ++s) {
    tile_barrier();   // the step's tiles are there, and every wave is done with those before
    issue(2 * s + 2);
    issue(2 * s + 3);
    const int t = 2 * s + (wave >> 1);
    int tile = walk + (wave >> 1);
    tile = tile >= per_head ? tile - per_head : tile;
    walk += 2;
    while (walk >= per_head) walk -= per_head;
    if (t >= n_tiles) continue;
    const int st = t % kBwdStages, m0 = k0 + (per_head == 1 ? 0 : tile) * kBN + 32 * half;
    const unsigned so = (unsigned)st * kStageBytes;
    const unsigned qa = fresh(qrow + so), da = fresh(drow + so);
    f32x16 sc = zero16(), dc = zero16();
#pragma unroll
    for (int i = 0; i < kHD / 16; ++i) {
      sc = mfma(lds_read8(qa ^ (unsigned)(32 * i), 0), kf[i], sc);
      dc = mfma(lds_read8(da ^ (unsigned)(32 * i), 0), vf[i], dc);
    }
    // query m0 + off + 4 (l / 32) counts iff lo <= off < hi; the others' P is 0
    const bool masked = m0 < k0 + 31 || m0 + 32 > end_min;
    const int lo = n - m0 - 4 * hl, hi = end - m0 - 4 * hl;
    f16x8 pf[2], dsf[2];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 l = *reinterpret_cast<const f32x4*>(&lse_s[st][32 * half + 8 * q + 4 * hl]);
      const f32x4 d = *reinterpret_cast<const f32x4*>(&dl_s[st][32 * half + 8 * q + 4 * hl]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = 4 * q + e, off = 8 * q + e;
        float x = __builtin_fmaf(sc[v], a.qk_scale, __fsub_rn(upf, l[e]));
        if (masked) x = ((off >= lo) & (off < hi)) ? x : -1.0e30f;
        const float pv = ex2(x);
        pf[v >> 3][v & 7] = (f16)pv;
        dsf[v >> 3][v & 7] = (f16)__fmul_rn(pv, __fsub_rn(dc[v], d[e]));
      }
    }
    // dV += P^T dO, dK += dS^T Q over the wave's 32 queries, 16 per product
    const unsigned qc = fresh(qcol + so), dc_ = fresh(dcol + so);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int hb = 0; hb < kHD / 32; ++hb) {
        dvacc[hb] = mfma(pf[i], lds_col8(dc_, hb, 16 * i * kHD * 2), dvacc[hb]);
        dkacc[hb] = mfma(dsf[i], lds_col8(qc, hb, 16 * i * kHD * 2), dkacc[hb]);
      }
  }
  __syncthreads();
  // the waves' sums, in wave order: 16 KB a wave of each, then wave w takes columns 32 w .. + 31
  const float back = pow2(-up);
#pragma unroll
  for (int hb = 0; hb < kHD / 32; ++hb)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      dkacc[hb][v] = __fmul_rn(dkacc[hb][v], back);
      dvacc[hb][v] = __fmul_rn(dvacc[hb][v], back);
    }
  float* kx = reinterpret_cast<float*>(Qs);
  float* vx = reinterpret_cast<float*>(Ds);
#pragma unroll
  for (int hb = 0; hb < kHD / 32; ++hb)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      *reinterpret_cast<f32x4*>(kx + part_off(w, hb, q, lane)) = quad(dkacc[hb], q);
      *reinterpret_cast<f32x4*>(vx + part_off(w, hb, q, lane)) = quad(dvacc[hb], q);
    }
  __syncthreads();
  f32x4 x[4], y[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    x[q] = y[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int o = 0; o < 4; ++o) {
      const f32x4 kq = *reinterpret_cast<const f32x4*>(kx + part_off(o, w, q, lane));
      const f32x4 vq = *reinterpret_cast<const f32x4*>(vx + part_off(o, w, q, lane));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[q][e] = __fadd_rn(x[q][e], kq[e]);
        y[q][e] = __fadd_rn(y[q][e], vq[e]);
      }
    }
  }
  if (slot >= 0) {
    float* part = parts + (int64_t)slot * kUnitFloats;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      *reinterpret_cast<f32x4*>(part + part_off(0, w, q, lane)) = x[q];
      *reinterpret_cast<f32x4*>(part + kUnitFloats + part_off(0, w, q, lane)) = y[q];
    }
    return;
  }
  __syncthreads();   // the sums have been read
  store_group(a, true, k0, 0, nk, g, w, x, y, Qs, Ds, bad, nullptr, dk, dv);
  redo_dkdv(a, k0, nk, g, bad, dout, lse, delta, dk, dv);
}

// Every item of the backward in one launch, longest walks first (the plan's order): dK/dV walks and
// dQ walks share the CUs, one workgroup each.
__global__ __launch_bounds__(kAThreads) void span_bwd_kernel(
    SpanArgs a, const int32_t* __restrict__ items, int n_units, const f16* __restrict__ dout,
    const float* __restrict__ lse, const float* __restrict__ delta, f16* __restrict__ dq,
    f16* __restrict__ dk, f16* __restrict__ dv, float* __restrict__ parts) {
  static_assert(kBwdStages == kFwdStages, "dK/dV and dQ share the tile ring");
  __shared__ __attribute__((aligned(1024))) f16 T0[kBwdStages * kTileHalves];
  __shared__ __attribute__((aligned(1024))) f16 T1[kBwdStages * kTileHalves];
  __shared__ __attribute__((aligned(16))) float lse_s[kBwdStages + 1][kBN], dl_s[kBwdStages][kBN];
  __shared__ int bad[kBM];
  __shared__ unsigned peaks[kAThreads / 64];
  const int idx = (int)blockIdx.x;
  const int kind = __builtin_amdgcn_readfirstlane(items[(int64_t)idx * kItemInts + 14]);
  if (kind == 2)
    dkdv_narrow(a, items, idx, n_units, dout, lse, delta, dk, dv, parts, T0, T1, lse_s, dl_s, bad,
                peaks);
  else if (kind == 1)
    dkdv_item(a, items, idx, n_units, dout, lse, delta, dk, dv, parts, T0, T1, lse_s, dl_s, bad,
              peaks);
  else
    dq_item(a, items, idx, n_units, dout, lse, delta, dq, parts, T0, T1,
            reinterpret_cast<int (*)[kBN]>(lse_s), bad);
}

// The partials of a split walk summed in slot order: a workgroup per 32 rows (or keys) of a block, a
// wave per 32 columns, four partials' loads in flight (a workgroup per block took 200 us where this
// takes 7: 1300 partials of 2048 tokens).
__global__ __launch_bounds__(kAThreads) void span_bwd_join_kernel(
    SpanArgs a, const int32_t* __restrict__ joins, int n_units, const f16* __restrict__ dout,
    const float* __restrict__ lse, const float* __restrict__ delta, f16* __restrict__ dq,
    f16* __restrict__ dk, f16* __restrict__ dv, const float* __restrict__ parts) {
  const int32_t* j = joins + (int64_t)(blockIdx.x >> 2) * DK_ATTN_SPAN_JOIN_INTS;
  const int w = blockIdx.x & 3;   // the row group
  auto u = [&](int k) { return __builtin_amdgcn_readfirstlane(j[k]); };
  int t0 = u(0), phase = u(1), rows = u(2);
  const int g = u(3), s0 = u(4), cnt = u(5), keys = u(6);
  const int gin = a.nq / a.nkv, step = keys ? 2 : 1;
  if (t0 < 0 || phase < 0 || phase >= gin || rows < 1 || rows > kBM || g < 0 || g >= a.nkv ||
      (int64_t)t0 + (keys ? rows - 1 : (phase + rows - 1) / gin) >= a.n_tokens || s0 < 0 || cnt < 1 ||
      (int64_t)s0 + (int64_t)cnt * step > n_units || rows <= 32 * w)
    return;
  // the group's own rows
  rows = rows - 32 * w < 32 ? rows - 32 * w : 32;
  if (keys) {
    t0 += 32 * w;
  } else {
    t0 += (phase + 32 * w) / gin;
    phase = (phase + 32 * w) % gin;
  }
  __shared__ __attribute__((aligned(16))) f16 S0[32 * kStride16], S1[32 * kStride16];
  __shared__ int bad[32];
  if (threadIdx.x < 32) bad[threadIdx.x] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 63, hb = threadIdx.x >> 6;
  f32x4 x[4], y[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) x[q] = y[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const float* p = parts + (int64_t)s0 * kUnitFloats + part_off(w, hb, 0, lane);
  auto sum = [&](f32x4 (&acc)[4], const float* base) {
    int s = 0;
    for (; s + 4 <= cnt; s += 4) {
      f32x4 t[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          t[i][q] = *reinterpret_cast<const f32x4*>(base + (int64_t)(s + i) * step * kUnitFloats + 256 * q);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[q][e] = __fadd_rn(acc[q][e], t[i][q][e]);
    }
    for (; s < cnt; ++s)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(base + (int64_t)s * step * kUnitFloats + 256 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[q][e] = __fadd_rn(acc[q][e], t[e]);
      }
  };
  sum(x, p);
  if (keys) sum(y, p + kUnitFloats);
  store_group(a, keys, t0, phase, rows, g, hb, x, y, S0, S1, bad, dq, dk, dv);
  if (keys) redo_dkdv(a, t0, rows, g, bad, dout, lse, delta, dk, dv);
  else redo_dq(a, t0, phase, rows, g, bad, dout, lse, delta, dq);
}

}  // namespace

extern "C" int64_t dk_attn_span_bwd_workspace(int64_t n_units) {
  return n_units > 0 ? n_units * (int64_t)(kUnitFloats * sizeof(float)) : 0;
}

extern "C" int dk_attn_span_bwd(const void* qkv, const void* out, const float* lse, const void* dout,
                                const int32_t* spans, const int32_t* items, int32_t n_items,
                                const int32_t* joins, int32_t n_joins, int32_t n_units,
                                int64_t n_tokens, int32_t nq, int32_t nkv, int32_t hd, float* delta,
                                void* dq, void* dk, void* dv, void* workspace,
                                int64_t workspace_bytes, hipStream_t stream) {
  SpanArgs a;
  if (int e = span_args(a, qkv, spans, n_tokens, nq, nkv, hd)) return e;
  if (n_items < 0 || n_joins < 0 || n_units < 0) return DK_ERR_INVALID;
  if (n_tokens == 0 || n_items == 0) return 0;
  if (!out || !lse || !dout || !items || (n_joins > 0 && !joins) || !delta || !dq || !dk || !dv)
    return DK_ERR_INVALID;
  if (!dk_aligned(out, 16) || !dk_aligned(dout, 16) || !dk_aligned(lse, 4) || !dk_aligned(delta, 4) ||
      !dk_aligned(dq, 16) || !dk_aligned(dk, 16) || !dk_aligned(dv, 16) || !dk_aligned(items, 4) ||
      !dk_aligned(joins, 4) || !dk_aligned(workspace, 256))
    return DK_ERR_ALIGN;
  if (n_units > 0 && (!workspace || workspace_bytes < dk_attn_span_bwd_workspace(n_units)))
    return DK_ERR_WORKSPACE;
  const int64_t pairs = n_tokens * nq, wgs = (pairs + 15) / 16 < kDeltaWgs ? (pairs + 15) / 16 : kDeltaWgs;
  if (n_items > INT32_MAX / kAThreads || n_joins > INT32_MAX / (4 * kAThreads)) return DK_ERR_INVALID;
  hipLaunchKernelGGL(attn_delta_kernel, dim3((unsigned)wgs), dim3(kAThreads), 0, stream,
                     (const f16*)out, (const f16*)dout, delta, n_tokens, nq);
  DK_CHECK_LAUNCH();
  hipLaunchKernelGGL(span_bwd_kernel, dim3((unsigned)n_items), dim3(kAThreads), 0, stream, a, items,
                     n_units, (const f16*)dout, lse, delta, (f16*)dq, (f16*)dk, (f16*)dv,
                     (float*)workspace);
  DK_CHECK_LAUNCH();
  if (n_joins > 0) {
    hipLaunchKernelGGL(span_bwd_join_kernel, dim3((unsigned)(4 * n_joins)), dim3(kAThreads), 0, stream, a,
                       joins, n_units, (const f16*)dout, lse, delta, (f16*)dq, (f16*)dk, (f16*)dv,
                       (const float*)workspace);
    DK_CHECK_LAUNCH();
  }
  return 0;
}
