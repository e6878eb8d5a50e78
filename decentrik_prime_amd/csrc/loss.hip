// Losses over the log-probabilities of a packed batch's answers, forward and gradient in one call: the
// clipped policy loss with a KL term, and the preference loss over pairs of answers.
//
// A batch is rows (answers) of consecutive tokens; the host cuts them into items (k_loss.RowMeta), a wave
// each: {first token (two words), tokens, row, the row's tokens, its items, the item's place among them, 0}.
// One 32-byte load tells a wave all that it needs before its tokens.  An empty row has one item without tokens.
//
// Policy, per token with advantage A:  r = e^(logp - old),  clipped where A > 0 and r > 1 + high or A < 0
// and r < 1 - low,  p = -A r (clipped: -A times the bound),  f = ref - logp,  k = e^f - f - 1
//   loss = sum w (p + beta k),   dlogp = w (-[not clipped] A r - beta (e^f - 1))
// Preference, S = a row's sum (or mean) of logp - ref, h = beta (S_chosen - S_rejected) - margin:
//   loss = mean over pairs of L(h),   dlogp of a row's tokens = sum over its pairs of +-beta L'(h) / pairs
//
// Differences of log-probabilities and the clip's borders are formed in 64 bits (a token within rounding
// of a border would gain or lose its whole gradient), exponentials in 32 (in 64 where they would pass that),
// sums over tokens in 64 and in an order that the sizes alone give.
//
// Bound: latency.  Up to 64 items and 32768 tokens one workgroup does everything in one launch: 1024 tokens'
// policy loss 4.1 us, 237 tokens' preference loss 4.0, 32 answers in 112 pairs 10.0 (in three launches 14 with
// their gaps).  Beyond, a wave per item and a second launch for what crosses items: one million tokens'
// policy loss 8.4 to 9.3 + 3.9 us (29 MB, half of them the stats' other columns; some 80 vector instructions
// a token are a third of it), the preference loss of 1024 answers 3.7 + 6.2.  A call's host time, some 10
// us, is longer than most of these.
#include "dk_common.h"

namespace {

constexpr int kWaves = 4;        // items of a workgroup
constexpr int kOneWaves = 16;    // the single workgroup of a call with few items
constexpr int kOneItems = 64;
constexpr int64_t kOneTokens = 1 << 15;
constexpr int kAhead = 8;        // tokens of a lane in flight
constexpr int kPairs = 1024;     // pairs of a workgroup

struct Tokens {          // a token array: element i at p[i * stride], negated where it holds losses
  const float* p;
  uint32_t stride;
  float sign;
  // an item's first element (in scalar registers), and element i behind it (one multiply-add)
  __device__ __forceinline__ const float* from(int64_t begin) const { return p + begin * stride; }
  __device__ __forceinline__ float at(const float* first, int i) const {
    return first[(uint64_t)(uint32_t)i * stride];
  }
};

__device__ __forceinline__ int wave_of() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

struct Item {
  int64_t begin;
  int count, row;
  int len, of, at;       // its row's tokens and items, and which of them it is
};

__device__ __forceinline__ Item item_of(const int4* items, int i) {
  const int4 v = items[2 * (int64_t)i], w = items[2 * (int64_t)i + 1];
  return {(int64_t)(((uint64_t)(uint32_t)v.y << 32) | (uint32_t)v.x), v.z, v.w, w.x, w.y, w.z};
}

// the sum over the wave's lanes (a butterfly: every lane gets it, in one order)
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int x = 1; x < 64; x *= 2) v += __shfl_xor(v, x);
  return v;
}

// k = e^f - f - 1 and its slope e^f - 1.  Near 0 k by its series (the terms up to f^9: the next is below 2^-34
// of the sum at 1/2), where the difference would leave few digits, and the slope as f + k; elsewhere k from
// the slope, which f + k would lose behind a large k (e^f of a token that the reference all but rules out).
struct Kl {
  float k, slope;
};

__device__ __forceinline__ Kl kl_of(float f) {
  if (fabsf(f) >= 0.5f) {
    const float slope = expf(f) - 1.0f;
    return {slope - f, slope};
  }
  float q = 1.0f / 362880;
  q = q * f + 1.0f / 40320;
  q = q * f + 1.0f / 5040;
  q = q * f + 1.0f / 720;
  q = q * f + 1.0f / 120;
  q = q * f + 1.0f / 24;
  q = q * f + 1.0f / 6;
  q = q * f + 0.5f;
  const float k = q * f * f;
  return {k, f + k};
}

struct PolicyParams {
  const int4* items;
  const int32_t* row_items;   // [rows + 1] a row's items
  int n_items, rows;
  Tokens logp, old, ref;      // ref.p null: none
  const float* adv;
  int adv_per_token;
  double log_low, log_high;   // log(1 - low), log(1 + high)
  float low, high;            // 1 - low, 1 + high
  float beta;
  int reduction;              // 0: a row's mean, then over rows with tokens; 1: all tokens' mean; 2: sum
  double inv;                 // 1 / rows with tokens, 1 / tokens, 1
  float* dlogp;
  float* stats;               // [rows, 4]
  float* loss;
  double* part;               // [n_items, 4] sums of p, k, clipped, r; then a loss per workgroup
};

struct Sums {
  double v[4];
};

// One token in 32 bits: its slope for logp (before the weight), p, k, r and whether it is clipped
struct PolicyTerms {
  float g, pol, k, r;
  bool cut;
};

__device__ __forceinline__ PolicyTerms policy_token(const PolicyParams& p, double d, double f, float av) {
  const bool up = av > 0.0f && d > p.log_high, down = av < 0.0f && d < p.log_low;
  const float r = expf((float)d);
  // (an advantage of 0 leaves nothing of any ratio, an infinite one included; of NaN it leaves NaN)
  const float kept = up || down || (av == 0.0f && d == d) ? 0.0f : r * av;
  PolicyTerms o{-kept, up ? p.high * av : down ? p.low * av : kept, 0.0f, r, up || down};
  if (p.ref.p) {
    const Kl kl = kl_of((float)f);
    o.k = kl.k;
    if (p.beta != 0.0f) o.g -= p.beta * kl.slope;   // (a reference that is watched alone: at any distance)
  }
  return o;
}

// e^d or e^f past 10^26 is formed in 64 bits: its product with a small advantage, weight or kl_coef may be an
// ordinary number where fp32 has only infinity.  A lane does its tokens of an item again when its sums say
// that there is one; the others come out as before.
constexpr double kFar = 60.0, kFarSum = 1e30;

__device__ __forceinline__ void policy_again(const PolicyParams& p, const Item& it, double weight, Sums& s,
                                             int& clipped) {
  const float *xp = p.logp.from(it.begin), *op = p.old.from(it.begin);
  const float* rp = p.ref.p ? p.ref.from(it.begin) : xp;
  s = Sums{};
  clipped = 0;
#pragma unroll 1
  for (int t = threadIdx.x & 63; t < it.count; t += 64) {
    const double x = (double)(p.logp.sign * p.logp.at(xp, t));
    const double d = x - (double)(p.old.sign * p.old.at(op, t));
    const double f = p.ref.p ? (double)(p.ref.sign * p.ref.at(rp, t)) - x : 0.0;
    const float av = p.adv_per_token ? p.adv[it.begin + t] : p.adv[it.row];
    const PolicyTerms o = policy_token(p, d, f, av);
    double pol = (double)o.pol, k = (double)o.k, r = (double)o.r;
    if (d > kFar || f > kFar) {
      double e[2] = {d, f};
#pragma unroll 1
      for (int q = 0; q < 2; ++q) {             // (one copy of the exponential: it holds many registers)
        const double v = exp(e[0]);
        e[0] = e[1];
        e[1] = v;
      }
      r = e[0];
      const double kept = o.cut || (av == 0.0f && d == d) ? 0.0 : r * (double)av;
      pol = o.cut ? pol : kept;
      double g = -kept;
      if (p.ref.p) {
        // (there e^f - f - 1 and e^f - 1 are e^f but for its last digits, and f may be infinite)
        const double slope = f > kFar ? e[1] : (double)kl_of((float)f).slope;
        k = f > kFar ? e[1] : k;
        if (p.beta != 0.0f) g -= (double)p.beta * slope;
      }
      p.dlogp[it.begin + t] = (float)(g * weight);
    }
    s.v[0] -= pol;
    s.v[1] += k;
    clipped += o.cut;
    s.v[3] += r;
  }
}

// One item: dlogp, and the sums of p, k, clipped and r.  Returns its share of the loss.
__device__ __forceinline__ double policy_item(const PolicyParams& p, const Item& it, Sums& s) {
  const int lane = threadIdx.x & 63;
  s = Sums{};
  if (it.count == 0) return 0.0;
  const double weight = p.reduction == 0 ? p.inv / (double)it.len : p.inv;   // a token's share of the loss
  const float w = (float)weight;
  const float* adv = p.adv_per_token ? p.adv + it.begin : p.adv + it.row;
  const float *xp = p.logp.from(it.begin), *op = p.old.from(it.begin);
  const float* rp = p.ref.p ? p.ref.from(it.begin) : xp;
  int clipped = 0;
  for (int t0 = 0; t0 < it.count; t0 += 64 * kAhead) {
    float x[kAhead], o[kAhead], rf[kAhead], a[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {   // every load before the first use, at tokens inside the item
      const int t = t0 + 64 * u + lane, in = t < it.count ? t : it.count - 1;
      x[u] = p.logp.at(xp, in);
      o[u] = p.old.at(op, in);
      rf[u] = p.ref.p ? p.ref.at(rp, in) : 0.0f;
      a[u] = adv[p.adv_per_token ? in : 0];
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int t = t0 + 64 * u + lane;
      if (t >= it.count) continue;
      const double xs = (double)(p.logp.sign * x[u]);
      const PolicyTerms v = policy_token(p, xs - (double)(p.old.sign * o[u]),
                                         (double)(p.ref.sign * rf[u]) - xs, a[u]);
      p.dlogp[it.begin + t] = v.g * w;
      s.v[0] -= (double)v.pol;
      s.v[1] += (double)v.k;
      clipped += v.cut;
      s.v[3] += (double)v.r;
    }
  }
  if (!(s.v[1] + s.v[3] < kFarSum)) policy_again(p, it, weight, s, clipped);
  s.v[2] = (double)clipped;
#pragma unroll
  for (int q = 0; q < 4; ++q) s.v[q] = wave_sum(s.v[q]);
  return weight * (p.beta != 0.0f ? s.v[0] + (double)p.beta * s.v[1] : s.v[0]);
}

__device__ __forceinline__ void store_stats(const PolicyParams& p, int64_t row, int len, const Sums& s) {
  const double inv = len > 0 ? 1.0 / (double)len : 0.0;
#pragma unroll
  for (int q = 0; q < 4; ++q) p.stats[4 * row + q] = (float)(s.v[q] * inv);
}

// Up to kOneItems items: everything in one workgroup and launch.
__global__ __launch_bounds__(64 * kOneWaves) void policy_one_kernel(PolicyParams p) {
  __shared__ Sums sums[kOneItems];
  __shared__ double loss[kOneItems];
  const int lane = threadIdx.x & 63, wave = wave_of();
  for (int i = wave; i < p.n_items; i += kOneWaves) {
    Sums s;
    const double l = policy_item(p, item_of(p.items, i), s);
    if (lane == 0) {
      sums[i] = s;
      loss[i] = l;
    }
  }
  __syncthreads();
  if (threadIdx.x < p.n_items) {     // a row's first item
    const Item it = item_of(p.items, threadIdx.x);
    if (it.at == 0) {
      Sums s{};
      for (int i = threadIdx.x; i < (int)threadIdx.x + it.of; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) s.v[q] += sums[i].v[q];
      store_stats(p, it.row, it.len, s);
    }
  }
  if (wave == kOneWaves - 1) {
    const double total = wave_sum(lane < p.n_items ? loss[lane] : 0.0);
    if (lane == 0) *p.loss = (float)total;
  }
}

// kWaves items per workgroup.  Rows of one item write their stats; the second launch sums the workgroups'
// losses and the other rows' items.
__global__ __launch_bounds__(64 * kWaves) void policy_kernel(PolicyParams p) {
  __shared__ double loss[kWaves];
  const int lane = threadIdx.x & 63, wave = wave_of();
  const int i = blockIdx.x * kWaves + wave;
  double mine = 0.0;
  if (i < p.n_items) {
    const Item it = item_of(p.items, i);
    Sums s;
    mine = policy_item(p, it, s);
    if (lane == 0) {
      if (it.of == 1) {
        store_stats(p, it.row, it.len, s);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) p.part[4 * (int64_t)i + q] = s.v[q];
      }
    }
  }
  if (lane == 0) loss[wave] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += loss[w];
    p.part[4 * (int64_t)p.n_items + blockIdx.x] = total;
  }
}

constexpr int kSumThreads = 1024;

// the sum of THREADS threads' values, in a fixed order; thread 0 has it
template <int THREADS>
__device__ __forceinline__ double block_sum(double s, double* red) {
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  double total = 0.0;
  if (threadIdx.x == 0)
    for (int w = 0; w < THREADS / 64; ++w) total += red[w];
  return total;
}

// n numbers' sum over a workgroup of kSumThreads; thread 0 has it
__device__ __forceinline__ double array_sum(const double* v, int64_t n, double* red) {
  double s = 0.0;
  int64_t i = threadIdx.x;
  for (; i + 3 * kSumThreads < n; i += 4 * kSumThreads) {
    double a[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) a[u] = v[i + u * kSumThreads];
#pragma unroll
    for (int u = 0; u < 4; ++u) s += a[u];
  }
  for (; i < n; i += kSumThreads) s += v[i];
  return block_sum<kSumThreads>(s, red);
}

// Workgroup 0: the loss.  The others: a wave per row of several items (its items by lane; a row has at
// most 64).
__global__ __launch_bounds__(kSumThreads) void policy_sum_kernel(PolicyParams p, int workgroups) {
  __shared__ double red[kSumThreads / 64];
  if (blockIdx.x == 0) {
    const double total = array_sum(p.part + 4 * (int64_t)p.n_items, workgroups, red);
    if (threadIdx.x == 0) *p.loss = (float)total;
    return;
  }
  const int lane = threadIdx.x & 63;
  const int64_t row = ((int64_t)blockIdx.x - 1) * (kSumThreads / 64) + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  const int b = p.row_items[row], e = p.row_items[row + 1];
  if (e - b < 2) return;
  Sums s{};
  for (int i = b + lane; i < e; i += 64)
#pragma unroll
    for (int q = 0; q < 4; ++q) s.v[q] += p.part[4 * (int64_t)i + q];
#pragma unroll
  for (int q = 0; q < 4; ++q) s.v[q] = wave_sum(s.v[q]);
  if (lane == 0) store_stats(p, row, item_of(p.items, b).len, s);
}

// ---------------------------------------------------------------------------------------------
struct PrefParams {
  const int4* items;
  const int32_t* row_items;    // [rows + 1]
  const int32_t* row_pairs;    // [rows + 1] a row's entries in `entries`
  const int2* entries;         // (other row, pair + 1: this row is chosen, -(pair + 1): rejected)
  const int2* pairs;           // (chosen, rejected)
  int n_items, rows, n_pairs;
  Tokens logp, ref;            // ref.p null: none
  double beta, margin, smoothing;
  int kind;                    // 0 sigmoid, 1 hinge, 2 ipo
  int average;
  float* dlogp;
  float* rewards;              // [rows]
  float* margins;              // [pairs]
  float* loss;
  double* part;                // [n_items] items' sums of logp - ref; then a loss per workgroup of pairs
};

__device__ __forceinline__ double pref_item(const PrefParams& p, const Item& it) {
  const int lane = threadIdx.x & 63;
  const float* xp = p.logp.from(it.begin);
  const float* rp = p.ref.p ? p.ref.from(it.begin) : xp;
  double s = 0.0;
  for (int t0 = 0; t0 < it.count; t0 += 64 * kAhead) {
    float x[kAhead], r[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int t = t0 + 64 * u + lane, in = t < it.count ? t : it.count - 1;
      x[u] = p.logp.at(xp, in);
      r[u] = p.ref.p ? p.ref.at(rp, in) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (t0 + 64 * u + lane < it.count)
        s += (double)(p.logp.sign * x[u]) - (double)(p.ref.sign * r[u]);
  }
  return wave_sum(s);
}

// S of a row from its items' sums, one lane (items in order)
__device__ __forceinline__ double row_score(const PrefParams& p, const double* part, int row) {
  const int b = p.row_items[row], e = p.row_items[row + 1];
  const int len = p.items[2 * (int64_t)b + 1].x;
  double s = 0.0;
  for (int i = b; i < e; ++i) s += part[i];
  return p.average && len > 0 ? s / (double)len : s;
}

// L(h) and L'(h)
__device__ __forceinline__ double pref_loss(const PrefParams& p, double h, double* slope) {
  if (p.kind == 0) {
    // -(1 - e) log s(h) - e log s(-h) = (1 - e) max(-h, 0) + e max(h, 0) + log(1 + e^-|h|); its slope is
    // e s(h) - (1 - e) s(-h), both from e^-|h|
    const double u = exp(-fabs(h)), tail = log1p(u), near = 1.0 / (1.0 + u), far = u * near;
    *slope = h < 0.0 ? p.smoothing * far - (1.0 - p.smoothing) * near
                     : p.smoothing * near - (1.0 - p.smoothing) * far;
    const double with = (1.0 - p.smoothing) * (fmax(-h, 0.0) + tail);
    return p.smoothing == 0.0 ? with : with + p.smoothing * (fmax(h, 0.0) + tail);   // (0 times infinity is 0)
  }
  if (p.kind == 1) {
    *slope = h < 1.0 ? -1.0 : h >= 1.0 ? 0.0 : h;   // NaN stays
    return h < 1.0 ? 1.0 - h : h >= 1.0 ? 0.0 : h;
  }
  const double u = (h - 0.5) / p.beta;
  *slope = 2.0 * u / p.beta;
  return u * u;
}

__device__ __forceinline__ double pref_h(const PrefParams& p, double chosen, double rejected) {
  return p.beta * (chosen - rejected) - p.margin;
}

// a row's score in the rewards, and the coefficient of its tokens from the sum of its pairs' slopes
__device__ __forceinline__ void pref_tokens(const PrefParams& p, const Item& it, double own, double slopes) {
  const int lane = threadIdx.x & 63;
  if (it.at == 0 && lane == 0) p.rewards[it.row] = (float)(p.beta * own);
  if (it.count == 0) return;
  const double g = slopes * p.beta / (double)p.n_pairs;
  const float gf = (float)(p.average ? g / (double)it.len : g);
  for (int t = lane; t < it.count; t += 64) p.dlogp[it.begin + t] = gf;
}

// Up to kOneItems items and kPairs pairs: everything in one workgroup and launch, the rows' scores and the
// pairs' slopes in LDS.
__global__ __launch_bounds__(64 * kOneWaves) void pref_one_kernel(PrefParams p) {
  __shared__ double sums[kOneItems], scores[kOneItems], slopes[kPairs];
  __shared__ double red[kOneWaves];
  const int lane = threadIdx.x & 63, wave = wave_of();
  for (int i = wave; i < p.n_items; i += kOneWaves) {
    const double s = pref_item(p, item_of(p.items, i));
    if (lane == 0) sums[i] = s;
  }
  __syncthreads();
  if (threadIdx.x < p.rows) scores[threadIdx.x] = row_score(p, sums, threadIdx.x);   // rows <= items
  __syncthreads();
  double l = 0.0;
  static_assert(64 * kOneWaves == kPairs, "a thread per pair");
  if (threadIdx.x < p.n_pairs) {
    const int2 pr = p.pairs[threadIdx.x];
    const double h = pref_h(p, scores[pr.x], scores[pr.y]);
    l = pref_loss(p, h, &slopes[threadIdx.x]);
    p.margins[threadIdx.x] = (float)h;
  }
  const double total = block_sum<64 * kOneWaves>(l, red);   // (its barrier publishes the slopes)
  if (threadIdx.x == 0) *p.loss = (float)(total / (double)p.n_pairs);
  for (int i = wave; i < p.n_items; i += kOneWaves) {
    const Item it = item_of(p.items, i);
    double g = 0.0;
    for (int e = p.row_pairs[it.row] + lane; e < p.row_pairs[it.row + 1]; e += 64) {
      const int k = p.entries[e].y;
      g += k > 0 ? slopes[k - 1] : -slopes[-k - 1];
    }
    pref_tokens(p, it, scores[it.row], wave_sum(g));
  }
}

__global__ __launch_bounds__(64 * kWaves) void pref_sum_kernel(PrefParams p) {
  const int i = blockIdx.x * kWaves + wave_of();
  if (i >= p.n_items) return;
  const double s = pref_item(p, item_of(p.items, i));
  if ((threadIdx.x & 63) == 0) p.part[i] = s;
}

// The first pair_wgs workgroups: kPairs pairs each (one alone: the loss too); the others: kWaves items, the
// slopes of a row's pairs by lane.
__global__ __launch_bounds__(64 * kWaves) void pref_apply_kernel(PrefParams p, int pair_wgs) {
  __shared__ double red[kWaves];
  const int b = blockIdx.x;
  if (b < pair_wgs) {
    const int end = (b + 1) * kPairs < p.n_pairs ? (b + 1) * kPairs : p.n_pairs;
    double l = 0.0;
    for (int i = b * kPairs + threadIdx.x; i < end; i += 64 * kWaves) {
      const int2 pr = p.pairs[i];
      const double h = pref_h(p, row_score(p, p.part, pr.x), row_score(p, p.part, pr.y));
      double slope;
      l += pref_loss(p, h, &slope);
      p.margins[i] = (float)h;
    }
    const double total = block_sum<64 * kWaves>(l, red);
    if (threadIdx.x == 0) {
      if (pair_wgs == 1) *p.loss = (float)(total / (double)p.n_pairs);
      else p.part[p.n_items + b] = total;
    }
    return;
  }
  const int i = (b - pair_wgs) * kWaves + wave_of();
  if (i >= p.n_items) return;
  const Item it = item_of(p.items, i);
  const double own = row_score(p, p.part, it.row);
  double g = 0.0;
  for (int e = p.row_pairs[it.row] + (threadIdx.x & 63); e < p.row_pairs[it.row + 1]; e += 64) {
    const int2 en = p.entries[e];
    const double other = row_score(p, p.part, en.x);
    double slope;
    pref_loss(p, en.y > 0 ? pref_h(p, own, other) : pref_h(p, other, own), &slope);
    g += en.y > 0 ? slope : -slope;
  }
  pref_tokens(p, it, own, wave_sum(g));
}

__global__ __launch_bounds__(kSumThreads) void pref_loss_kernel(PrefParams p, int pair_wgs) {
  __shared__ double red[kSumThreads / 64];
  const double total = array_sum(p.part + p.n_items, pair_wgs, red);
  if (threadIdx.x == 0) *p.loss = (float)(total / (double)p.n_pairs);
}

// factors[rows] = 0, but -dlogp[i] / unit at row at[i]; unit is the largest power of two up to the largest
// |dlogp| (1 where that is 0 or not finite), so the division is exact.  One workgroup, bound by its loads'
// latency: 4.7 us for 1520 answer tokens of 2048.
__global__ __launch_bounds__(kSumThreads) void row_factors_kernel(const float* __restrict__ dlogp,
                                                                  const int32_t* __restrict__ at, int64_t n,
                                                                  float* factors, int64_t rows, float* unit) {
  __shared__ uint32_t red[kSumThreads / 64];
  uint32_t top = 0;                       // |x|'s bits are in order, infinity and NaN above all numbers
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < n; i += kSumThreads) {
    const uint32_t bits = __float_as_uint(dlogp[i]) & 0x7fffffffu;
    top = bits > top ? bits : top;
  }
  for (int64_t i = threadIdx.x; i < rows; i += kSumThreads) factors[i] = 0.0f;
#pragma unroll
  for (int x = 1; x < 64; x *= 2) {
    const uint32_t o = __shfl_xor(top, x);
    top = o > top ? o : top;
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();                        // (the zeros are written, too)
#pragma unroll
  for (int w = 0; w < kSumThreads / 64; ++w) top = red[w] > top ? red[w] : top;
  constexpr uint32_t inf = 0x7f800000u, least = 0x00800000u;
  const float u = top == 0 || top >= inf ? 1.0f : __uint_as_float(top < least ? least : top & inf);
  if (threadIdx.x == 0) *unit = u;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < n; i += kSumThreads)
    if ((uint64_t)(int64_t)at[i] < (uint64_t)rows) factors[at[i]] = -dlogp[i] / u;
}

// a token array that is there, or (ref alone) may be absent
bool tokens_ok(const dk_token_array& t, int64_t n, bool absent) {
  return (t.data || n == 0 || absent) && t.stride >= 0 && t.stride <= INT32_MAX;
}

Tokens tokens_of(const dk_token_array& t) {
  return {t.data, (uint32_t)t.stride, t.negated ? -1.0f : 1.0f};
}

// (a wave per item, and kSumThreads per 16 rows: 2^32 work items are more than a launch takes)
bool rows_ok(int64_t n_items, int64_t rows) {
  return rows >= 1 && rows <= n_items && n_items <= (int64_t)1 << 25;
}

}  // namespace

// Few items and tokens take one workgroup and launch (see the top); 64 items of long rows would keep its CU
// busy for far longer than two launches take.
static bool one_group(int64_t n_items, int64_t n_tokens) {
  return n_items <= kOneItems && n_tokens <= kOneTokens;
}

extern "C" int64_t dk_policy_loss_workspace(int64_t n_items, int64_t n_tokens) {
  if (n_items <= 0 || one_group(n_items, n_tokens)) return 0;
  return (4 * n_items + (n_items + kWaves - 1) / kWaves) * (int64_t)sizeof(double);
}

extern "C" int dk_policy_loss(const dk_policy_args* args, hipStream_t stream) {
  if (!args) return DK_ERR_INVALID;
  const dk_policy_args& a = *args;
  const int64_t n_items = a.n_items, rows = a.rows, n_tokens = a.n_tokens;
  if (!rows_ok(n_items, rows) || n_tokens < 0 || !a.items || !a.row_items ||
      !tokens_ok(a.logp, n_tokens, false) || !tokens_ok(a.old, n_tokens, false) ||
      !tokens_ok(a.ref, n_tokens, true) || (n_tokens > 0 && !a.dlogp) || !a.stats || !a.loss ||
      (!a.advantages && (n_tokens > 0 || !a.per_token)) || !(a.clip_low >= 0.0 && a.clip_low <= 1.0) ||
      !(a.clip_high >= 0.0) || !(a.kl_coef - a.kl_coef == 0.0) ||
      (a.kl_coef != 0.0 && !a.ref.data && n_tokens > 0) || a.reduction < 0 || a.reduction > 2 ||
      !(a.denominator > 0.0))
    return DK_ERR_INVALID;
  if (!dk_aligned(a.items, 16) || !dk_aligned(a.row_items, 4)) return DK_ERR_ALIGN;
  const int64_t need = dk_policy_loss_workspace(n_items, n_tokens);
  if (need && (!a.workspace || a.workspace_bytes < need || !dk_aligned(a.workspace, 8)))
    return DK_ERR_WORKSPACE;
  PolicyParams p{reinterpret_cast<const int4*>(a.items), a.row_items, (int)n_items, (int)rows,
                 tokens_of(a.logp), tokens_of(a.old), tokens_of(a.ref), a.advantages, a.per_token != 0,
                 log1p(-a.clip_low), log1p(a.clip_high), (float)(1.0 - a.clip_low),
                 (float)(1.0 + a.clip_high), (float)a.kl_coef, (int)a.reduction, 1.0 / a.denominator, a.dlogp,
                 a.stats, a.loss, (double*)a.workspace};
  if (need == 0) {
    hipLaunchKernelGGL(policy_one_kernel, dim3(1), dim3(64 * kOneWaves), 0, stream, p);
    DK_CHECK_LAUNCH();
    return 0;
  }
  const int wgs = (int)((n_items + kWaves - 1) / kWaves);
  hipLaunchKernelGGL(policy_kernel, dim3(wgs), dim3(64 * kWaves), 0, stream, p);
  DK_CHECK_LAUNCH();
  const int64_t more = n_items > rows ? (rows + kSumThreads / 64 - 1) / (kSumThreads / 64) : 0;
  hipLaunchKernelGGL(policy_sum_kernel, dim3((unsigned)(1 + more)), dim3(kSumThreads), 0, stream, p, wgs);
  DK_CHECK_LAUNCH();
  return 0;
}

static int64_t pair_groups(int64_t pairs) { return (pairs + kPairs - 1) / kPairs; }

extern "C" int64_t dk_preference_loss_workspace(int64_t n_items, int64_t n_tokens, int64_t pairs) {
  if (n_items <= 0 || (one_group(n_items, n_tokens) && pairs <= kPairs)) return 0;
  return (n_items + pair_groups(pairs)) * (int64_t)sizeof(double);
}

extern "C" int dk_preference_loss(const dk_preference_args* args, hipStream_t stream) {
  if (!args) return DK_ERR_INVALID;
  const dk_preference_args& a = *args;
  const int64_t n_items = a.n_items, n_tokens = a.n_tokens, n_pairs = a.n_pairs;
  if (!rows_ok(n_items, a.rows) || n_tokens < 0 || n_pairs < 1 || n_pairs > (int64_t)1 << 28 || !a.items ||
      !a.row_items || !a.row_pairs || !a.entries || !a.pairs || !tokens_ok(a.logp, n_tokens, false) ||
      !tokens_ok(a.ref, n_tokens, true) || (n_tokens > 0 && !a.dlogp) || !a.rewards || !a.margins || !a.loss ||
      !(a.beta > 0.0) || !(1.0 / a.beta > 0.0) || a.kind < 0 || a.kind > 2 ||
      !(a.label_smoothing >= 0.0 && a.label_smoothing <= 0.5) || !(a.margin - a.margin == 0.0))
    return DK_ERR_INVALID;
  if (!dk_aligned(a.items, 16) || !dk_aligned(a.row_items, 4) || !dk_aligned(a.row_pairs, 4) ||
      !dk_aligned(a.entries, 8) || !dk_aligned(a.pairs, 8))
    return DK_ERR_ALIGN;
  const int64_t need = dk_preference_loss_workspace(n_items, n_tokens, n_pairs);
  if (need && (!a.workspace || a.workspace_bytes < need || !dk_aligned(a.workspace, 8)))
    return DK_ERR_WORKSPACE;
  PrefParams p{reinterpret_cast<const int4*>(a.items), a.row_items, a.row_pairs,
               reinterpret_cast<const int2*>(a.entries), reinterpret_cast<const int2*>(a.pairs), (int)n_items,
               (int)a.rows, (int)n_pairs, tokens_of(a.logp), tokens_of(a.ref), a.beta, a.margin,
               a.label_smoothing, (int)a.kind, a.average != 0, a.dlogp, a.rewards, a.margins, a.loss,
               (double*)a.workspace};
  if (need == 0) {
    hipLaunchKernelGGL(pref_one_kernel, dim3(1), dim3(64 * kOneWaves), 0, stream, p);
    DK_CHECK_LAUNCH();
    return 0;
  }
  const int wgs = (int)((n_items + kWaves - 1) / kWaves), pair_wgs = (int)pair_groups(n_pairs);
  hipLaunchKernelGGL(pref_sum_kernel, dim3(wgs), dim3(64 * kWaves), 0, stream, p);
  DK_CHECK_LAUNCH();
  hipLaunchKernelGGL(pref_apply_kernel, dim3(pair_wgs + wgs), dim3(64 * kWaves), 0, stream, p, pair_wgs);
  DK_CHECK_LAUNCH();
  if (pair_wgs > 1) {
    hipLaunchKernelGGL(pref_loss_kernel, dim3(1), dim3(kSumThreads), 0, stream, p, pair_wgs);
    DK_CHECK_LAUNCH();
  }
  return 0;
}

extern "C" int dk_row_factors(const float* dlogp, const int32_t* at, int64_t n, float* factors, int64_t rows,
                              float* unit, hipStream_t stream) {
  if (n < 0 || rows < 0 || !unit || (n > 0 && (!dlogp || !at)) || (rows > 0 && !factors)) return DK_ERR_INVALID;
  if (!dk_aligned(dlogp, 4) || !dk_aligned(at, 4) || !dk_aligned(factors, 4) || !dk_aligned(unit, 4))
    return DK_ERR_ALIGN;
  hipLaunchKernelGGL(row_factors_kernel, dim3(1), dim3(kSumThreads), 0, stream, dlogp, at, n, factors, rows,
                     unit);
  DK_CHECK_LAUNCH();
  return 0;
}
