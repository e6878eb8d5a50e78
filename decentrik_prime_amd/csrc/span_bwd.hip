// Backward of the attention over part of the keys (attn_span.h): delta, then a wave per (query, head)
// for dq and per (key, KV head) for dk and dv.
#include "attn_delta.h"
#include "attn_span.h"

namespace {

__global__ __launch_bounds__(kAThreads) void span_bwd_rows_kernel(
    SpanArgs a, const f16* __restrict__ dout, const float* __restrict__ lse,
    const float* __restrict__ delta, f16* __restrict__ dq, f16* __restrict__ dk, f16* __restrict__ dv) {
  __shared__ RowScratch s[kAThreads / 64];
  const int w = threadIdx.x >> 6;
  int64_t i = (int64_t)blockIdx.x * (kAThreads / 64) + w;
  if (i < a.n_tokens * a.nkv) {
    span_key_dkdv(a, i / a.nkv, (int)(i % a.nkv), dout, lse, delta, dk, dv, s[w]);
    return;
  }
  i -= a.n_tokens * a.nkv;
  if (i < a.n_tokens * a.nq) span_row_dq(a, i / a.nq, (int)(i % a.nq), dout, lse, delta, dq, s[w]);
}

}  // namespace

extern "C" int dk_attn_span_bwd(const void* qkv, const void* out, const float* lse, const void* dout,
                                const int32_t* spans, int64_t n_tokens, int32_t nq, int32_t nkv,
                                int32_t hd, float* delta, void* dq, void* dk, void* dv,
                                hipStream_t stream) {
  SpanArgs a;
  if (int e = span_args(a, qkv, spans, n_tokens, nq, nkv, hd)) return e;
  if (n_tokens == 0) return 0;
  if (!out || !lse || !dout || !delta || !dq || !dk || !dv) return DK_ERR_INVALID;
  if (!dk_aligned(out, 16) || !dk_aligned(dout, 16) || !dk_aligned(lse, 4) || !dk_aligned(delta, 4) ||
      !dk_aligned(dq, 16) || !dk_aligned(dk, 16) || !dk_aligned(dv, 16))
    return DK_ERR_ALIGN;
  const int64_t pairs = n_tokens * nq, wgs = (pairs + n_tokens * nkv + 3) / 4;
  if (wgs > INT32_MAX / kAThreads) return DK_ERR_INVALID;
  hipLaunchKernelGGL(attn_delta_kernel, dim3((unsigned)((pairs + 15) / 16)), dim3(kAThreads), 0,
                     stream, (const f16*)out, (const f16*)dout, delta, n_tokens, nq);
  DK_CHECK_LAUNCH();
  hipLaunchKernelGGL(span_bwd_rows_kernel, dim3((unsigned)wgs), dim3(kAThreads), 0, stream, a,
                     (const f16*)dout, lse, delta, (f16*)dq, (f16*)dk, (f16*)dv);
  DK_CHECK_LAUNCH();
  return 0;
}
