// Losses over the log-probabilities of a packed batch's answers, forward and gradient in one call: the
// clipped policy loss with a KL term, and the preference loss over pairs of answers.
//
// A batch is rows (answers) of consecutive tokens; the host cuts them into items of at most a few
// thousand tokens of one row (k_loss.RowMeta), a wave each.  An item is {first token (two words), tokens,
// row}; an empty row has one item without tokens.
//
// Policy, per token with advantage A:  r = e^(logp - old),  clipped where A > 0 and r > 1 + high or A < 0
// and r < 1 - low,  p = -A r (clipped: -A times the bound),  f = ref - logp,  k = e^f - f - 1
//   loss = sum w (p + beta k),   dlogp = w (-[not clipped] A r - beta (f + k))        (e^f - 1 = f + k)
// Preference, S = a row's sum (or mean) of logp - ref, h = beta (S_chosen - S_rejected) - margin:
//   loss = mean over pairs of L(h),   dlogp of a row's tokens = sum over its pairs of +-beta L'(h) / pairs
//
// Differences of log-probabilities and the clip's borders are formed in 64 bits (a token within rounding
// of a border would gain or lose its whole gradient), exponentials in 32, sums over tokens in 64 and in an
// order that the sizes alone give.  Bound: latency up to some 10^5 tokens (one or two launches), beyond
// that reading the token arrays once.
#include "dk_common.h"

namespace {

constexpr int kWaves = 4;        // items of a workgroup
constexpr int kOneWaves = 16;    // items that a single workgroup takes in one launch
constexpr int kAhead = 8;        // tokens of a lane in flight

struct Tokens {          // a token array: element i at p[i * stride], negated where it holds losses
  const float* p;
  int64_t stride;
  float sign;
  __device__ __forceinline__ float at(int64_t i) const { return sign * p[i * stride]; }
};

struct Item {
  int64_t begin;
  int count, row;
};

__device__ __forceinline__ Item item_of(const int4* items, int i) {
  const int4 v = items[i];
  return {(int64_t)(((uint64_t)(uint32_t)v.y << 32) | (uint32_t)v.x), v.z, v.w};
}

// the sum over the wave's lanes (a butterfly: every lane gets it, in one order)
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int x = 1; x < 64; x *= 2) v += __shfl_xor(v, x);
  return v;
}

// e^f - f - 1.  Near 0 by its series (the terms up to f^9: the next is below 2^-34 of the sum at 1/2),
// where the difference would leave few digits.
__device__ __forceinline__ float expm1_minus(float f) {
  if (fabsf(f) >= 0.5f) return (expf(f) - 1.0f) - f;
  float q = 1.0f / 362880;
  q = q * f + 1.0f / 40320;
  q = q * f + 1.0f / 5040;
  q = q * f + 1.0f / 720;
  q = q * f + 1.0f / 120;
  q = q * f + 1.0f / 24;
  q = q * f + 1.0f / 6;
  q = q * f + 0.5f;
  return q * f * f;
}

struct PolicyParams {
  const int4* items;
  const int32_t* row_items;   // [rows + 1] a row's items
  const int64_t* lens;        // [rows]
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

// a token's share of the loss
__device__ __forceinline__ double policy_weight(const PolicyParams& p, int row) {
  const int64_t len = p.lens[row];
  return p.reduction == 0 && len > 0 ? p.inv / (double)len : p.inv;
}

// one item: dlogp, and the sums of p, k, clipped and r
__device__ __forceinline__ Sums policy_item(const PolicyParams& p, const Item& it, double weight) {
  const int lane = threadIdx.x & 63;
  const float w = (float)weight;
  const float row_adv = p.adv_per_token ? 0.0f : p.adv[it.row];
  Sums s{};
  for (int t0 = 0; t0 < it.count; t0 += 64 * kAhead) {
    float x[kAhead], o[kAhead], rf[kAhead], a[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {   // every load before the first use, at tokens inside the item
      const int t = t0 + 64 * u + lane;
      const int64_t i = it.begin + (t < it.count ? t : it.count - 1);
      x[u] = p.logp.at(i);
      o[u] = p.old.at(i);
      rf[u] = p.ref.p ? p.ref.at(i) : 0.0f;
      a[u] = p.adv_per_token ? p.adv[i] : row_adv;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int t = t0 + 64 * u + lane;
      if (t >= it.count) continue;
      const double d = (double)x[u] - (double)o[u];
      const bool up = a[u] > 0.0f && d > p.log_high, down = a[u] < 0.0f && d < p.log_low;
      const float r = expf((float)d);
      const float kept = up || down ? 0.0f : r * a[u];
      const float pol = up ? p.high * a[u] : down ? p.low * a[u] : kept;
      float g = -kept, k = 0.0f;
      if (p.ref.p) {
        const float f = (float)((double)rf[u] - (double)x[u]);
        k = expm1_minus(f);
        g -= p.beta * (f + k);
      }
      p.dlogp[it.begin + t] = g * w;
      s.v[0] -= (double)pol;
      s.v[1] += (double)k;
      s.v[2] += up || down ? 1.0 : 0.0;
      s.v[3] += (double)r;
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) s.v[q] = wave_sum(s.v[q]);
  return s;
}

__device__ __forceinline__ void store_stats(const PolicyParams& p, int row, const Sums& s) {
  const int64_t len = p.lens[row];
  const double inv = len > 0 ? 1.0 / (double)len : 0.0;
#pragma unroll
  for (int q = 0; q < 4; ++q) p.stats[4 * (int64_t)row + q] = (float)(s.v[q] * inv);
}

// WAVES items per workgroup.  One workgroup (WAVES = kOneWaves) writes everything; otherwise rows of one
// item write their stats, and the second launch sums the workgroups' losses and the other rows' items.
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void policy_kernel(PolicyParams p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = blockIdx.x * WAVES + wave;
  __shared__ double loss[WAVES];
  __shared__ Sums sums[WAVES];
  __shared__ int row_of[WAVES];
  double mine = 0.0;
  if (i < p.n_items) {
    const Item it = item_of(p.items, i);
    const double w = policy_weight(p, it.row);
    const Sums s = policy_item(p, it, w);
    mine = it.count > 0 ? w * (s.v[0] + (double)p.beta * s.v[1]) : 0.0;
    const bool whole = p.row_items[it.row + 1] - p.row_items[it.row] == 1;
    if (lane == 0) {
      if (whole) store_stats(p, it.row, s);
      if (WAVES == kOneWaves) {
        sums[wave] = s;
        row_of[wave] = whole ? -1 : it.row;
      } else if (!whole) {
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
    for (int w = 0; w < WAVES; ++w) total += loss[w];
    if (WAVES == kOneWaves) *p.loss = (float)total;
    else p.part[4 * (int64_t)p.n_items + blockIdx.x] = total;
  }
  if (WAVES == kOneWaves && lane == 0 && i < p.n_items && row_of[wave] >= 0 &&
      p.row_items[row_of[wave]] == i) {
    Sums s{};
    for (int w = wave; w < WAVES && w < p.n_items && row_of[w] == row_of[wave]; ++w)
#pragma unroll
      for (int q = 0; q < 4; ++q) s.v[q] += sums[w].v[q];
    store_stats(p, row_of[wave], s);
  }
}

constexpr int kSumThreads = 1024;

// n numbers' sum over a workgroup of kSumThreads, in a fixed order; thread 0 has it
__device__ __forceinline__ double block_sum(const double* v, int64_t n, double* red) {
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
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  double total = 0.0;
  if (threadIdx.x == 0)
    for (int w = 0; w < kSumThreads / 64; ++w) total += red[w];
  return total;
}

// Workgroup 0: the loss.  The others: a wave per row of several items (its items by lane; a row has at
// most 64).
__global__ __launch_bounds__(kSumThreads) void policy_sum_kernel(PolicyParams p, int workgroups) {
  __shared__ double red[kSumThreads / 64];
  if (blockIdx.x == 0) {
    const double total = block_sum(p.part + 4 * (int64_t)p.n_items, workgroups, red);
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
  if (lane == 0) store_stats(p, (int)row, s);
}

// ---------------------------------------------------------------------------------------------
struct PrefParams {
  const int4* items;
  const int32_t* row_items;    // [rows + 1]
  const int64_t* lens;         // [rows]
  const int32_t* row_pairs;    // [rows + 1] a row's entries in `entries`
  const int2* entries;         // (other row, pair + 1: this row is chosen, -(pair + 1): rejected)
  int n_items, rows, n_pairs;
  Tokens logp, ref;            // ref.p null: none
  double beta, margin, smoothing;
  int kind;                    // 0 sigmoid, 1 hinge, 2 ipo
  int average;
  float* dlogp;
  float* rewards;              // [rows]
  float* margins;              // [pairs]
  float* loss;
  double* part;                // [n_items] items' sums of logp - ref; then a loss per pair
};

__device__ __forceinline__ double pref_item(const PrefParams& p, const Item& it) {
  const int lane = threadIdx.x & 63;
  double s = 0.0;
  for (int t0 = 0; t0 < it.count; t0 += 64 * kAhead) {
    float x[kAhead], r[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int t = t0 + 64 * u + lane;
      const int64_t i = it.begin + (t < it.count ? t : it.count - 1);
      x[u] = p.logp.at(i);
      r[u] = p.ref.p ? p.ref.at(i) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (t0 + 64 * u + lane < it.count) s += (double)x[u] - (double)r[u];
  }
  return wave_sum(s);
}

// S of a row from its items' sums, one lane (items in order)
__device__ __forceinline__ double row_score(const PrefParams& p, const double* part, int row) {
  const int b = p.row_items[row], e = p.row_items[row + 1];
  double s = 0.0;
  for (int i = b; i < e; ++i) s += part[i];
  const int64_t len = p.lens[row];
  return p.average && len > 0 ? s / (double)len : s;
}

// L(h) and L'(h)
__device__ __forceinline__ double pref_loss(const PrefParams& p, double h, double* slope) {
  if (p.kind == 0) {
    // -(1 - e) log s(h) - e log s(-h): log(1 + e^-|h|) is one of the two softplus terms' part
    const double tail = log1p(exp(-fabs(h)));
    *slope = p.smoothing / (1.0 + exp(-h)) - (1.0 - p.smoothing) / (1.0 + exp(h));
    return (1.0 - p.smoothing) * (fmax(-h, 0.0) + tail) + p.smoothing * (fmax(h, 0.0) + tail);
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

// The item's gradient from the items' sums: the row's coefficient (its pairs by lane), then the tokens.
// The row's first item also writes its reward, and the margins and losses of the pairs that it is the
// chosen row of.
__device__ __forceinline__ void pref_apply(const PrefParams& p, const double* part, int i, const Item& it,
                                           double* pair_loss) {
  const int lane = threadIdx.x & 63;
  const double own = row_score(p, part, it.row);
  const bool first = p.row_items[it.row] == i;
  if (first && lane == 0) p.rewards[it.row] = (float)(p.beta * own);
  double g = 0.0;
  for (int e = p.row_pairs[it.row] + lane; e < p.row_pairs[it.row + 1]; e += 64) {
    const int2 en = p.entries[e];
    const double other = row_score(p, part, en.x);
    const bool chosen = en.y > 0;
    double slope;
    const double h = chosen ? pref_h(p, own, other) : pref_h(p, other, own);
    const double l = pref_loss(p, h, &slope);
    g += chosen ? slope : -slope;
    if (chosen && first) {
      p.margins[en.y - 1] = (float)h;
      pair_loss[en.y - 1] = l;
    }
  }
  g = wave_sum(g) * p.beta / (double)p.n_pairs;
  const int64_t len = p.lens[it.row];
  const float gf = (float)(p.average && len > 0 ? g / (double)len : g);
  for (int t = lane; t < it.count; t += 64) p.dlogp[it.begin + t] = gf;
}

// every item and pair in one workgroup
__global__ __launch_bounds__(64 * kOneWaves) void pref_one_kernel(PrefParams p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __shared__ double sums[kOneWaves];
  __shared__ double red[kSumThreads / 64];
  static_assert(64 * kOneWaves == kSumThreads, "block_sum's threads");
  Item it{0, 0, 0};
  if (wave < p.n_items) {
    it = item_of(p.items, wave);
    const double s = pref_item(p, it);
    if (lane == 0) sums[wave] = s;
  }
  __syncthreads();
  double* pair_loss = p.part + p.n_items;
  if (wave < p.n_items) pref_apply(p, sums, wave, it, pair_loss);
  __syncthreads();
  const double total = block_sum(pair_loss, p.n_pairs, red);
  if (threadIdx.x == 0) *p.loss = (float)(total / (double)p.n_pairs);
}

__global__ __launch_bounds__(64 * kWaves) void pref_sum_kernel(PrefParams p) {
  const int i = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (i >= p.n_items) return;
  const double s = pref_item(p, item_of(p.items, i));
  if ((threadIdx.x & 63) == 0) p.part[i] = s;
}

__global__ __launch_bounds__(64 * kWaves) void pref_apply_kernel(PrefParams p) {
  const int i = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (i >= p.n_items) return;
  pref_apply(p, p.part, i, item_of(p.items, i), p.part + p.n_items);
}

__global__ __launch_bounds__(kSumThreads) void pref_loss_kernel(PrefParams p) {
  __shared__ double red[kSumThreads / 64];
  const double total = block_sum(p.part + p.n_items, p.n_pairs, red);
  if (threadIdx.x == 0) *p.loss = (float)(total / (double)p.n_pairs);
}

bool tokens_ok(const dk_token_array* t, int64_t n) {
  return t && n >= 0 && (n == 0 || t->data) && t->stride >= 0;
}

Tokens tokens_of(const dk_token_array* t) {
  return t ? Tokens{t->data, t->stride, t->negated ? -1.0f : 1.0f} : Tokens{nullptr, 1, 1.0f};
}

bool rows_ok(int64_t n_items, int64_t rows) {
  return rows >= 1 && rows <= n_items && n_items <= (int64_t)1 << 28;
}

}  // namespace

extern "C" int64_t dk_policy_loss_workspace(int64_t n_items) {
  return n_items <= 0 ? 0 : (4 * n_items + (n_items + kWaves - 1) / kWaves) * (int64_t)sizeof(double);
}

extern "C" int dk_policy_loss(const int32_t* items, int64_t n_items, const int32_t* row_items,
                              const int64_t* lens, int64_t rows, int64_t n_tokens,
                              const dk_token_array* logp, const dk_token_array* old, const dk_token_array* ref, const float* advantages,
                              int per_token, double clip_low, double clip_high, double kl_coef,
                              int reduction, double denominator, float* dlogp, float* stats, float* loss,
                              void* ws, int64_t ws_bytes, hipStream_t stream) {
  if (!rows_ok(n_items, rows) || !items || !row_items || !lens || !tokens_ok(logp, n_tokens) ||
      !tokens_ok(old, n_tokens) || (ref && !tokens_ok(ref, n_tokens)) || (n_tokens > 0 && !dlogp) || !stats ||
      !loss || (!advantages && (n_tokens > 0 || !per_token)) ||
      !(clip_low >= 0.0 && clip_low <= 1.0) ||
      !(clip_high >= 0.0) || !(kl_coef - kl_coef == 0.0) || (kl_coef != 0.0 && !ref) || reduction < 0 ||
      reduction > 2 || !(denominator > 0.0))
    return DK_ERR_INVALID;
  if (!dk_aligned(items, 16) || !dk_aligned(lens, 8)) return DK_ERR_ALIGN;
  if (!ws || ws_bytes < dk_policy_loss_workspace(n_items) || !dk_aligned(ws, 8)) return DK_ERR_WORKSPACE;
  PolicyParams p{reinterpret_cast<const int4*>(items), row_items, lens, (int)n_items, (int)rows,
                 tokens_of(logp), tokens_of(old), tokens_of(ref), advantages, per_token,
                 log1p(-clip_low), log1p(clip_high), (float)(1.0 - clip_low), (float)(1.0 + clip_high),
                 (float)kl_coef, reduction, 1.0 / denominator, dlogp, stats, loss, (double*)ws};
  if (n_items <= kOneWaves) {
    hipLaunchKernelGGL((policy_kernel<kOneWaves>), dim3(1), dim3(64 * kOneWaves), 0, stream, p);
    DK_CHECK_LAUNCH();
    return 0;
  }
  const int wgs = (int)((n_items + kWaves - 1) / kWaves);
  hipLaunchKernelGGL((policy_kernel<kWaves>), dim3(wgs), dim3(64 * kWaves), 0, stream, p);
  DK_CHECK_LAUNCH();
  const int64_t more = n_items > rows ? (rows + kSumThreads / 64 - 1) / (kSumThreads / 64) : 0;
  hipLaunchKernelGGL(policy_sum_kernel, dim3((unsigned)(1 + more)), dim3(kSumThreads), 0, stream, p, wgs);
  DK_CHECK_LAUNCH();
  return 0;
}

extern "C" int64_t dk_preference_loss_workspace(int64_t n_items, int64_t pairs) {
  return n_items <= 0 || pairs <= 0 ? 0 : (n_items + pairs) * (int64_t)sizeof(double);
}

extern "C" int dk_preference_loss(const int32_t* items, int64_t n_items, const int32_t* row_items,
                                  const int64_t* lens, int64_t rows, int64_t n_tokens,
                                  const int32_t* row_pairs, const int32_t* entries, int64_t n_pairs,
                                  const dk_token_array* logp,
                                  const dk_token_array* ref, double beta, int kind, double label_smoothing,
                                  double margin, int average, float* dlogp, float* rewards,
                                  float* margins, float* loss, void* ws, int64_t ws_bytes,
                                  hipStream_t stream) {
  if (!rows_ok(n_items, rows) || n_pairs < 1 || n_pairs > (int64_t)1 << 28 || !items || !row_items ||
      !lens || !row_pairs || !entries || !tokens_ok(logp, n_tokens) ||
      (ref && !tokens_ok(ref, n_tokens)) || (n_tokens > 0 && !dlogp) || !rewards || !margins || !loss || !(beta > 0.0) || kind < 0 ||
      kind > 2 || !(label_smoothing >= 0.0 && label_smoothing <= 0.5) || !(margin - margin == 0.0))
    return DK_ERR_INVALID;
  if (!dk_aligned(items, 16) || !dk_aligned(lens, 8) || !dk_aligned(entries, 8)) return DK_ERR_ALIGN;
  if (!ws || ws_bytes < dk_preference_loss_workspace(n_items, n_pairs) || !dk_aligned(ws, 8))
    return DK_ERR_WORKSPACE;
  PrefParams p{reinterpret_cast<const int4*>(items), row_items, lens, row_pairs,
               reinterpret_cast<const int2*>(entries), (int)n_items, (int)rows, (int)n_pairs,
               tokens_of(logp), tokens_of(ref), beta, margin, label_smoothing, kind, average, dlogp, rewards,
               margins, loss, (double*)ws};
  if (n_items <= kOneWaves) {
    hipLaunchKernelGGL(pref_one_kernel, dim3(1), dim3(64 * kOneWaves), 0, stream, p);
    DK_CHECK_LAUNCH();
    return 0;
  }
  const int wgs = (int)((n_items + kWaves - 1) / kWaves);
  hipLaunchKernelGGL(pref_sum_kernel, dim3(wgs), dim3(64 * kWaves), 0, stream, p);
  DK_CHECK_LAUNCH();
  hipLaunchKernelGGL(pref_apply_kernel, dim3(wgs), dim3(64 * kWaves), 0, stream, p);
  DK_CHECK_LAUNCH();
  hipLaunchKernelGGL(pref_loss_kernel, dim3(1), dim3(kSumThreads), 0, stream, p);
  DK_CHECK_LAUNCH();
  return 0;
}
