// Token log-probabilities of the language-model head without its logits: for selected rows y_i of the
// final norm's output and the embedding E [V, D] (fp16)
//   x_v = scale <y_i, E_v>,   lse_i = log sum_v e^{x_v},   logp_i = x_{t_i} - lse_i,
//   entropy_i = lse_i - sum_v e^{x_v - lse_i} x_v
// One pass over E: the products stay in MFMA accumulators and each lane folds its own into a running
// (r, s, t) per token, in log2 units z = x log2(e):  r = the largest z so far,  s = sum 2^(z - r),
// t = sum 2^(z - r) (z - r).  Two such states join as
//   r = max(r1, r2),  a_i = 2^(r_i - r),  s = sum a_i s_i,  t = sum a_i (t_i + s_i (r_i - r))
// and at the end logp = ln2 (z_t - r - log2 s), lse = ln2 (r + log2 s), entropy = ln2 (log2 s - t / s).
//
// Bound: the matrix product (2 n V D operations) from some 300 tokens on, below that reading E once.
// A workgroup of 8 waves holds a tile of tokens (64, 128 or 256) and walks a run of E in pieces of 128 or
// 256 rows; (tile, run) pairs fill the 256 CUs (lp_plan).  The walk is one loop over K steps of 64, through
// the borders of the pieces: operands come by LDS DMA (lds_dma.h), the loads NST - 1 steps ahead, so that
// the first steps of a piece arrive while the last one's accumulators are folded.  The MFMA takes E's rows as
// its first operand and the tokens as its second, so that a lane's accumulators are 16 vocabulary entries
// of each of its tokens: the folding needs no exchange between lanes, and the four lanes, the waves and
// the workgroups that share a token meet once, at the end.  Few tokens take small tiles with many stages
// (up to 80 KB of E in flight on a CU), many the 256 x 256 tile of the framework's GEMMs.
//
// Measured on MI355X, 151936 x 1536 (a call's two launches): one token 84 us (5.5 TB/s of E; a copy reaches
// 5.1), 853 tokens 406, 2048 tokens 806 (1.19 PFLOP/s, at the clock that power allows; the library's product
// alone, which writes the logits, 958 to 979); 37 tokens of 32003 x 1024 18.1 us (15.5 the walk).  Folding
// takes about 4 % of a large piece, the two steps behind a tile's border nothing that shows.
#include <algorithm>
#include <utility>

#include "dk_common.h"
#include "lds_dma.h"

namespace dk {
namespace {

constexpr int kLpThreads = 512;
constexpr int kLpBK = 64;      // K per step
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;
// below every z of finite inputs: the r of a state without entries (2^(kNone - r) is 0, and 1 against itself)
constexpr float kNone = -1e30f;

// The 16-byte chunks of a 64-half row are permuted by row: no bank conflict in the operand reads
__device__ __forceinline__ int lp_swz(int r) { return ((r >> 1) & 7) ^ ((r & 1) << 2); }

// How the launch is cut: `tiles` tiles of `bm` tokens, each over `runs` runs of E, and (tail > 0) the tokens
// behind them as one tile of 128 over `tail` runs.  A run is a whole number of pieces of bn rows of E.
struct LpPlan {
  int bm, bn, tiles, runs, tail, pieces;
};

struct LpParams {
  const f16* y;            // [*, D], row stride ldy
  int64_t ldy;
  const int32_t* rows;     // [n] rows of y, or null (0 .. n - 1)
  int64_t total;           // rows of y that `rows` may name
  const f16* e;            // [V, D]
  const int32_t* tgt;      // [n]
  int64_t n, V, D;
  float c;                 // scale log2(e)
  LpPlan plan;
  float* part;             // per token and run: (r, s, t, unused)
  float* xt;               // [n] the target's product, where there is a target
};

// f(0), ..., f(N - 1) with constant arguments (a loop of this size is past the compiler's limit for unrolling,
// and an array indexed by a loop that stays one is kept in memory)
template <class F, int... I>
__device__ __forceinline__ void each(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}

struct LpState {
  float r, s, t;
};

__device__ __forceinline__ LpState lp_join(const LpState& a, const LpState& b) {
  const float r = fmaxf(a.r, b.r);
  const float da = a.r - r, db = b.r - r;
  const float wa = __builtin_amdgcn_exp2f(da), wb = __builtin_amdgcn_exp2f(db);
  return {r, wa * a.s + wb * b.s, wa * (a.t + a.s * da) + wb * (b.t + b.s * db)};
}

__device__ __forceinline__ int lp_runs(const LpPlan& pl, int64_t m) {
  return m < (int64_t)pl.tiles * pl.bm ? pl.runs : pl.tail;
}

// token m's first state in LpParams::part
__device__ __forceinline__ int64_t lp_part(const LpPlan& pl, int64_t m) {
  const int64_t whole = (int64_t)pl.tiles * pl.bm;
  return m < whole ? m * pl.runs : whole * pl.runs + (m - whole) * pl.tail;
}

// The walk of tokens m0 .. m0 + BM - 1 over run `run` of `runs`, in pieces of BN rows of E; WAVES_M x
// 8 / WAVES_M waves; NST stages of operands in LDS
template <int BM, int BN, int WAVES_M, int NST>
__device__ __forceinline__ void lp_walk(const LpParams& p, f16* As, int32_t* tgts, int64_t m0, int run, int runs) {
  constexpr int WAVES_N = 8 / WAVES_M;
  constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N;
  constexpr int TM = WM / 16, TN = WN / 16;          // 16 x 16 blocks of a wave: tokens, vocabulary
  constexpr int SA = BM * kLpBK, SB = BN * kLpBK;   // halves of a stage
  constexpr int LA = BM / 64, LB = BN / 64;         // DMA instructions per lane and step
  constexpr int LOADS = LA + LB;
  constexpr int NMFMA = TM * TN;
  f16* Bs = As + NST * SA;
  static_assert(WAVES_N * BM * 16 <= NST * SA * 2, "the waves' states at the end");

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WAVES_N, wn = wave % WAVES_N;
  // the run's rows of E: [v0, v1)
  const int v0 = __builtin_amdgcn_readfirstlane((int)((int64_t)p.plan.pieces * run / runs) * BN);
  int v1 = __builtin_amdgcn_readfirstlane((int)((int64_t)p.plan.pieces * (run + 1) / runs) * BN);
  v1 = v1 < p.V ? v1 : (int)p.V;
  const int nk = (int)(p.D / kLpBK);
  const int steps = (v1 - v0 + BN - 1) / BN * nk;

  for (int i = tid; i < BM; i += kLpThreads) tgts[i] = m0 + i < p.n ? p.tgt[m0 + i] : -1;

  // ---- loads: instruction j of wave w fills chunks [(8 j + w) 64, +64) of a stage
  const uint64_t a_base = uniform64((uint64_t)(p.rows ? p.y : p.y + m0 * p.ldy));
  unsigned a_off[LA];
#pragma unroll
  for (int j = 0; j < LA; ++j) {
    const int q = (j * 8 + wave) * 64 + lane, row = q >> 3;
    const int64_t m = m0 + row < p.n ? m0 + row : p.n - 1;   // tokens past n: never stored
    int64_t r = m - m0;
    if (p.rows) {
      const int64_t at = p.rows[m];
      r = at < 0 ? 0 : at < p.total ? at : p.total - 1;      // outside: NaN at the end
    }
    a_off[j] = (unsigned)((r * p.ldy + ((q & 7) ^ lp_swz(row)) * 8) * (int64_t)sizeof(f16));
  }
  int ld_kt = 0;                     // the step that is loaded next
  int ld_v = v0;
  uint64_t b_base = 0;
  int b_last = 0;                    // the piece's last row in E: rows past the run are this one again
  auto set_piece = [&]() {
    b_base = uniform64((uint64_t)(p.e + (int64_t)ld_v * p.D));
    b_last = v1 - 1 - ld_v < BN ? v1 - 1 - ld_v : BN;
  };
  // E's offsets are formed load by load (three instructions beside 16 or more MFMAs): held in registers
  // they would push the accumulators' kernel into scratch memory
  const int b_row = wave * 8 + (lane >> 3), b_chunk = ((lane & 7) ^ lp_swz(b_row)) * 16;
  const unsigned d2 = (unsigned)p.D * (unsigned)sizeof(f16);   // below 2^24, as is a row's number
  auto issue = [&](int st, int d) {
    const uint64_t k = (uint64_t)ld_kt * (kLpBK * sizeof(f16));
    if (d < LA) {
      dma16s(a_base + k, a_off[d],
             __builtin_amdgcn_readfirstlane(lds_addr(As + st * SA + (d * 8 + wave) * 512)));
    } else {
      const int j = d - LA, row = b_row + 64 * j < b_last ? b_row + 64 * j : b_last;
      dma16s(b_base + k, __umul24(row, d2) + b_chunk,
             __builtin_amdgcn_readfirstlane(lds_addr(Bs + st * SB + (j * 8 + wave) * 512)));
    }
  };
  auto advance = [&]() {
    if (++ld_kt == nk) {
      ld_kt = 0;
      if ((ld_v += BN) < v1) set_piece();
    }
  };
  auto wait_loads = [&](int later) {   // at most `later` steps of this wave's loads still in flight
    if (NST > 5 && later >= 5) wait_vmem<5 * LOADS>();
    else if (NST > 4 && later >= 4) wait_vmem<4 * LOADS>();
    else if (NST > 3 && later >= 3) wait_vmem<3 * LOADS>();
    else if (NST > 2 && later >= 2) wait_vmem<2 * LOADS>();
    else if (later >= 1) wait_vmem<LOADS>();
    else wait_vmem<0>();
  };
  auto stage_of = [](int s) { return NST == 2 ? s & 1 : s % NST; };

  set_piece();
#pragma unroll
  for (int q = 0; q < NST; ++q)
    if (q < steps) {
#pragma unroll
      for (int d = 0; d < LOADS; ++d) issue(q, d);
      advance();
    }
  wait_loads((steps < NST ? steps : NST) - 1);
  __syncthreads();

  // ---- operands of v_mfma_f32_16x16x32_f16: lane l holds row l % 16 of a 16-row block, k 8 (l / 16) ..
  // + 7 of a 32-wide sub-step.  The tokens' fragments single-buffered where a sub-step has 32 MFMAs (each
  // read again after its last use), else double-buffered like E's.
  const int r16 = lane & 15, g4 = 4 * (lane >> 4);
  int fo[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) fo[q] = r16 * kLpBK + ((4 * q + (lane >> 4)) ^ lp_swz(r16)) * 8;
  constexpr bool A2 = NMFMA <= 16;
  f16x8 fa[A2 ? 2 : 1][TM], fb[2][TN];
  auto kj = [](int k) { return (k / TN) & 1 ? TN - 1 - k % TN : k % TN; };
  auto read_a = [&](int st, int s, int i, int buf) {
    fa[A2 ? buf : 0][i] = *reinterpret_cast<const f16x8*>(As + st * SA + (wm * WM + 16 * i) * kLpBK + fo[s]);
  };
  auto read_b = [&](int st, int s, int j, int buf) {
    fb[buf][j] = *reinterpret_cast<const f16x8*>(Bs + st * SB + (wn * WN + 16 * j) * kLpBK + fo[s]);
  };
  auto a_slot = [](int i) {
    return A2 ? (TN + i < NMFMA ? TN + i : NMFMA - 1) : (i + 1) * TN - 1;
  };
  auto reads_after = [&](int k, int st, int s, int buf) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
      if (j == k) read_b(st, s, j, buf);
#pragma unroll
    for (int i = 0; i < TM; ++i)
      if (a_slot(i) == k) read_a(st, s, i, buf);
  };
  auto mfma_group = [&](int k) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    int n = 0;
#pragma unroll
    for (int j = 0; j < TN; ++j) n += j == k;
#pragma unroll
    for (int i = 0; i < TM; ++i) n += a_slot(i) == k;
    if (n == 1) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    else if (n == 2) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
  };

  f32x4 acc[TM][TN];   // [token block][vocabulary block]: lane l: token l % 16, entries 4 (l / 16) + 0..3
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  LpState state[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) state[i] = {kNone, 0.0f, 0.0f};

  // the accumulators of the piece that begins at entry v into the states.  Entries past v1 are entry v1 - 1
  // again: they leave the largest as it is, and their 2^(z - r) is dropped.
  auto fold = [&](int v) {
    const int first = v + wn * WN + g4;                      // this lane's first vocabulary entry
    // a target's product, from the one lane of the launch that holds it
    bool mine = false;
#pragma unroll
    for (int i = 0; i < TM; ++i)
      mine |= (unsigned)tgts[wm * WM + 16 * i + r16] - (unsigned)first < (unsigned)WN;
    if (__builtin_amdgcn_ballot_w64(mine)) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const unsigned at = (unsigned)tgts[wm * WM + 16 * i + r16] - (unsigned)first;
        float x = acc[i][0][0];
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) x = at == 16u * j + q ? acc[i][j][q] : x;
        if (at < (unsigned)WN && (at & 15) < 4 && (int)at + first < v1)
          p.xt[m0 + wm * WM + 16 * i + r16] = x;
      }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      float mx = acc[i][0][0];
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) mx = fmaxf(mx, acc[i][j][q]);
      const LpState old = state[i];
      const float r = fmaxf(old.r, mx * p.c);
      const float d = old.r - r, w = __builtin_amdgcn_exp2f(d);
      float s = w * old.s, t = w * (old.t + old.s * d);
#pragma unroll
      for (int k = 0; k < 4 * TN; ++k) {
        const float z = __builtin_fmaf(acc[i][k >> 2][k & 3], p.c, -r);
        float ez = __builtin_amdgcn_exp2f(z);
        ez = first + 16 * (k >> 2) + (k & 3) < v1 ? ez : 0.0f;
        s += ez;
        t = __builtin_fmaf(ez, z, t);
      }
      state[i] = {r, s, t};
      __builtin_amdgcn_sched_barrier(0);      // one token block's temporaries at a time
    }
  };

#pragma unroll
  for (int i = 0; i < TM; ++i) read_a(0, 0, i, 0);
#pragma unroll
  for (int j = 0; j < TN; ++j) read_b(0, 0, j, 0);
  int kt = 0, v = v0;
  for (int s = 0; s < steps; ++s) {
    const int st = stage_of(s);
#pragma unroll
    for (int k = 0; k < NMFMA; ++k) {
      acc[k / TN][kj(k)] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb[0][kj(k)], fa[0][k / TN],
                                                                  acc[k / TN][kj(k)], 0, 0, 0);
      reads_after(k, st, 1, 1);
    }
#pragma unroll
    for (int k = 0; k < NMFMA; ++k) mfma_group(k);
    wait_loads((steps - 1 < s + NST - 1 ? steps - 1 : s + NST - 1) - (s + 1));
    __syncthreads();
    const bool more = s + 1 < steps, refill = s + NST < steps;
    const int st1 = stage_of(s + 1);
    __builtin_amdgcn_s_setprio(1);
    each([&](auto kc) __attribute__((always_inline)) {
      constexpr int k = decltype(kc)::value;
      acc[k / TN][kj(k)] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
          fb[1][kj(k)], fa[A2 ? 1 : 0][k / TN], acc[k / TN][kj(k)], 0, 0, 0);
      if (more) reads_after(k, st1, 0, 0);
#pragma unroll
      for (int d = k * LOADS / NMFMA; d < (k + 1) * LOADS / NMFMA; ++d)
        if (refill) issue(st, d);
      __builtin_amdgcn_sched_barrier(0);
    }, std::make_integer_sequence<int, NMFMA>{});
    __builtin_amdgcn_s_setprio(0);
    if (refill) advance();
    if (++kt == nk) {
      fold(v);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      kt = 0;
      v += BN;
    }
  }

  // ---- the four lanes, then the WAVES_N waves that share a token
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int x = 16; x < 64; x *= 2) {
      const LpState o = {__shfl_xor(state[i].r, x), __shfl_xor(state[i].s, x), __shfl_xor(state[i].t, x)};
      state[i] = lp_join(state[i], o);
    }
  __syncthreads();   // no wave reads a stage any more, and no load is in flight
  f32x4* meet = reinterpret_cast<f32x4*>(As);
#pragma unroll
  for (int i = 0; i < TM; ++i)
    if (lane < 16)
      meet[wn * BM + wm * WM + 16 * i + lane] = f32x4{state[i].r, state[i].s, state[i].t, 0.0f};
  __syncthreads();
  if (tid < BM && m0 + tid < p.n) {
    LpState a = {meet[tid][0], meet[tid][1], meet[tid][2]};
#pragma unroll
    for (int w = 1; w < WAVES_N; ++w) {
      const f32x4 b = meet[w * BM + tid];
      a = lp_join(a, {b[0], b[1], b[2]});
    }
    reinterpret_cast<f32x4*>(p.part)[lp_part(p.plan, m0 + tid) + run] = f32x4{a.r, a.s, a.t, 0.0f};
  }
}

constexpr int lp_halves(int bm, int bn, int nst) { return nst * (bm + bn) * kLpBK; }

template <int BM, int BN, int WAVES_M, int NST, bool TAIL>
__global__ __launch_bounds__(kLpThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
void head_logp_kernel(LpParams p) {
  constexpr int mine = lp_halves(BM, BN, NST), tail = TAIL ? lp_halves(128, BN, 3) : 0;
  __shared__ __attribute__((aligned(1024))) f16 S[mine > tail ? mine : tail];
  __shared__ int32_t tgts[BM];
  // each XCD (workgroups are dealt to the 8 of them in turn) a contiguous share of (tile, run) with the
  // tiles fastest, so that the tiles of a run read E through one L2
  const int total = gridDim.x, o = blockIdx.x & 7, q = total >> 3, r = total & 7;
  const int u = o * q + (o < r ? o : r) + ((int)blockIdx.x >> 3);
  const int whole = p.plan.tiles * p.plan.runs;
  if (!TAIL || u < whole) {
    lp_walk<BM, BN, WAVES_M, NST>(p, S, tgts, (int64_t)(u % p.plan.tiles) * BM, u / p.plan.tiles,
                                  p.plan.runs);
  } else if constexpr (TAIL) {
    lp_walk<128, BN, 2, 3>(p, S, tgts, (int64_t)p.plan.tiles * BM, u - whole, p.plan.tail);
  }
}

// The runs' states of a token joined (lane i takes runs i, i + 64, ...; then a butterfly: a fixed order),
// one wave per token.
__global__ __launch_bounds__(256) void head_logp_join_kernel(LpParams p, float* __restrict__ logp,
                                                             float* __restrict__ entropy,
                                                             float* __restrict__ lse) {
  const int lane = threadIdx.x & 63;
  const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= p.n) return;
  // what the result needs beside the states, loaded with them
  const int64_t t = p.tgt[m];
  const int64_t at = p.rows ? p.rows[m] : 0;
  const float xt = p.xt[m];                    // (unwritten where there is no target: not used)
  const f32x4* mine = reinterpret_cast<const f32x4*>(p.part) + lp_part(p.plan, m);
  const int runs = lp_runs(p.plan, m);
  LpState a = {kNone, 0.0f, 0.0f};
  for (int i = lane; i < runs; i += 256) {     // four loads in flight; a run past the last joins as nothing
    f32x4 b[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) b[u] = mine[i + 64 * u < runs ? i + 64 * u : lane < runs ? lane : 0];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool in = i + 64 * u < runs;
      a = lp_join(a, {in ? b[u][0] : kNone, in ? b[u][1] : 0.0f, in ? b[u][2] : 0.0f});
    }
  }
#pragma unroll
  for (int x = 1; x < 64; x *= 2) {
    const LpState o = {__shfl_xor(a.r, x), __shfl_xor(a.s, x), __shfl_xor(a.t, x)};
    a = lp_join(a, o);
  }
  if (lane) return;
  const float l2 = log2f(a.s);
  float lp = 0.0f, en = kLn2 * (l2 - a.t / a.s), ls = kLn2 * (a.r + l2);
  if (t >= p.V) lp = NAN;
  else if (t >= 0) lp = kLn2 * (__builtin_fmaf(xt, p.c, -a.r) - l2);
  // rounding takes neither past what it can be (NaN stays)
  lp = lp > 0.0f ? 0.0f : lp;
  en = en < 0.0f ? 0.0f : en;
  if (p.rows && (at < 0 || at >= p.total)) lp = en = ls = NAN;
  logp[m] = lp;
  entropy[m] = en;
  lse[m] = ls;
}

constexpr int kLpSlots = 256;   // workgroups at once, one per CU

// Estimated microseconds of a plan: fixed, and for every round of workgroups its pieces of E, each of D / 64
// steps (step + load * busy; busy: the share of the CUs that the round fills) and a fold; never below reading
// E once.  The constants are fits to 40 to 1600 tokens over vocabularies of 1000 to 64000 and D of 256 and
// 1536 on MI355X (graph replays).  The small tiles take the small calls (100 tokens, 4000 x 1536: 20 us
// against 41 on 256 x 256), the large ones from a few hundred tokens and some 10^4 entries on (1600 tokens of
// 64000 x 1536: 310 against 377 on 128 x 256, 408 on 128 x 128).
struct LpCost {
  int bm, bn;
  float fixed, step, load, fold;
};
constexpr LpCost kLpCost[] = {{64, 128, 7.4f, 0.475f, 0.035f, 0.3f},
                              {128, 128, 7.5f, 0.52f, 0.115f, 0.5f},
                              {128, 256, 8.3f, 0.85f, 0.25f, 0.9f},
                              {256, 256, 10.5f, 1.2f, 0.57f, 1.8f}};
constexpr float kReadUs = 5.4e6f;   // bytes of E a microsecond

float lp_pieces_us(const LpCost& c, int64_t pieces, int64_t workgroups, float steps) {
  const float busy = workgroups < kLpSlots ? (float)workgroups / kLpSlots : 1.0f;
  return (float)pieces * (steps * (c.step + c.load * busy) + c.fold);
}

// The plan of least estimated time: tiles of one shape over as many runs of E as give one to four rounds of
// workgroups; for 256 x 256 also whole tiles with up to 128 tokens behind them as a tile of 128 x 256 in the
// same launch (853 tokens of 151936 x 1536 423 -> 409 us, 300 246 -> 218).
LpPlan lp_plan(int64_t n, int64_t V, int64_t D) {
  const float steps = (float)(D / kLpBK), read = (float)(2 * V * D) / kReadUs;
  LpPlan best{};
  float best_us = -1.0f, best_work = 0.0f;
  auto consider = [&](float work, const LpPlan& pl, float fixed) {
    const float us = fixed + (work > read ? work : read);
    if (best_us < 0.0f || us < best_us || (us == best_us && work < best_work)) {
      best_us = us;
      best_work = work;
      best = pl;
    }
  };
  for (const LpCost& c : kLpCost) {
    const uint32_t tiles = ((uint32_t)n + c.bm - 1) / c.bm, pieces = ((uint32_t)V + c.bn - 1) / c.bn;
    for (uint32_t rounds = 1; rounds <= 4; ++rounds) {
      uint32_t g = rounds * kLpSlots / tiles;
      g = g < 1 ? 1 : g < pieces ? g : pieces;
      const uint32_t each = (pieces + g - 1) / g;
      const uint32_t runs = (pieces + each - 1) / each;   // the fewest runs of that many pieces
      const int64_t all = ((int64_t)tiles * runs + kLpSlots - 1) / kLpSlots;
      consider(lp_pieces_us(c, all * each, (int64_t)tiles * runs, steps),
               LpPlan{c.bm, c.bn, (int)tiles, (int)runs, 0, (int)pieces}, c.fixed);
      if (g == pieces) break;
    }
  }
  const LpCost &big = kLpCost[3], &small = kLpCost[2];
  const int64_t whole = n / 256, rest = n % 256, pieces = (V + 255) / 256;
  if (rest >= 1 && rest <= 128 && whole >= 1 && whole < kLpSlots) {
    const int64_t most = (kLpSlots - 1) / whole, least = (pieces + most - 1) / most;
    for (int64_t each = least; each < least + 4; ++each) {
      const int64_t g = (pieces + each - 1) / each;
      int64_t left = kLpSlots - whole * g;
      if (left > pieces) left = pieces;
      const int64_t behind = (pieces + left - 1) / left;
      const float a = lp_pieces_us(big, each, kLpSlots, steps), b = lp_pieces_us(small, behind, kLpSlots, steps);
      consider(a > b ? a : b,
               LpPlan{256, 256, (int)whole, (int)g, (int)((pieces + behind - 1) / behind), (int)pieces},
               big.fixed);
    }
  }
  return best;
}

// (token, run) states of a plan
int64_t lp_states(const LpPlan& pl, int64_t n) {
  const int64_t whole = (int64_t)pl.tiles * pl.bm;
  return pl.tail ? whole * pl.runs + (n - whole) * pl.tail : n * pl.runs;
}

// Tokens of a launch: a wave per token in the join, and 2^32 work items are more than a launch takes
constexpr int64_t kLpSlice = (int64_t)1 << 24;

int64_t lp_bytes(int64_t n, int64_t V, int64_t D) { return 16 * lp_states(lp_plan(n, V, D), n) + 4 * n; }

bool lp_sizes_ok(int64_t n, int64_t V, int64_t D) {
  // the grid, 32-bit pieces and steps, and 32-bit offsets inside a piece of E
  return n >= 0 && n <= (int64_t)1 << 30 && V >= 1 && V <= (int64_t)1 << 30 && D >= kLpBK &&
         D % kLpBK == 0 && D <= (int64_t)1 << 20;
}

}  // namespace
}  // namespace dk

using namespace dk;

extern "C" int64_t dk_head_logprobs_workspace(int64_t n, int64_t vocab, int64_t d) {
  if (n <= 0 || !lp_sizes_ok(n, vocab, d)) return 0;
  if (n <= kLpSlice) return lp_bytes(n, vocab, d);
  const int64_t whole = lp_bytes(kLpSlice, vocab, d), rest = n % kLpSlice;
  return rest ? std::max(whole, lp_bytes(rest, vocab, d)) : whole;
}

extern "C" int dk_head_logprobs(const void* y, int64_t ldy, int64_t total, const int32_t* rows, int64_t n,
                                const void* emb, int64_t vocab, int64_t d, const int32_t* tgt, float scale,
                                float* logp, float* entropy, float* lse, void* ws, int64_t ws_bytes,
                                hipStream_t stream) {
  if (!lp_sizes_ok(n, vocab, d) || ldy < d || ldy % 8 || total < 0 || (!rows && n > total) ||
      !(scale > 0.0f) || scale > 1e6f)
    return DK_ERR_INVALID;
  if (n == 0) return 0;
  if (!y || !emb || !tgt || !logp || !entropy || !lse || total == 0) return DK_ERR_INVALID;
  // 32-bit byte offsets: of a tile's rows of y, or of all of y where rows are picked from it
  const int64_t reach = rows ? total : n < 256 ? n : 256;
  if (reach > 1 && ldy > (((int64_t)1 << 31) - 1 - d) / (reach - 1)) return DK_ERR_INVALID;
  if (!dk_aligned(y, 16) || !dk_aligned(emb, 16) || !dk_aligned(tgt, 4) || !dk_aligned(rows, 4) ||
      !dk_aligned(logp, 4) || !dk_aligned(entropy, 4) || !dk_aligned(lse, 4))
    return DK_ERR_ALIGN;
  if (!ws || ws_bytes < dk_head_logprobs_workspace(n, vocab, d) || !dk_aligned(ws, 16))
    return DK_ERR_WORKSPACE;
  for (int64_t i = 0; i < n; i += kLpSlice) {
    const int64_t m = n - i < kLpSlice ? n - i : kLpSlice;
    const LpPlan pl = lp_plan(m, vocab, d);
    LpParams p{(const f16*)y + (rows ? 0 : i * ldy), ldy, rows ? rows + i : nullptr, total, (const f16*)emb,
               tgt + i, m, vocab, d, scale * kLog2e, pl, (float*)ws, (float*)ws + 4 * lp_states(pl, m)};
    const dim3 grid((unsigned)(pl.tiles * pl.runs + pl.tail)), block(kLpThreads);
    if (pl.bm == 64)
      hipLaunchKernelGGL((head_logp_kernel<64, 128, 2, 6, false>), grid, block, 0, stream, p);
    else if (pl.bm == 128 && pl.bn == 128)
      hipLaunchKernelGGL((head_logp_kernel<128, 128, 4, 4, false>), grid, block, 0, stream, p);
    else if (pl.bm == 128)
      hipLaunchKernelGGL((head_logp_kernel<128, 256, 2, 3, false>), grid, block, 0, stream, p);
    else if (pl.tail == 0)
      hipLaunchKernelGGL((head_logp_kernel<256, 256, 2, 2, false>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((head_logp_kernel<256, 256, 2, 2, true>), grid, block, 0, stream, p);
    DK_CHECK_LAUNCH();
    hipLaunchKernelGGL(head_logp_join_kernel, dim3((unsigned)((m + 3) / 4)), dim3(256), 0, stream, p, logp + i,
                       entropy + i, lse + i);
    DK_CHECK_LAUNCH();
  }
  return 0;
}
