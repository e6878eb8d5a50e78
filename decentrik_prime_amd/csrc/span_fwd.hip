// Forward of the attention over part of the keys (attn_span.h), one wave per (query, head).
#include "attn_span.h"

namespace {

__global__ __launch_bounds__(kAThreads) void span_fwd_rows_kernel(SpanArgs a, f16* __restrict__ out,
                                                                  float* __restrict__ lse) {
  __shared__ RowScratch s[kAThreads / 64];
  const int w = threadIdx.x >> 6;
  const int64_t pair = (int64_t)blockIdx.x * (kAThreads / 64) + w;
  if (pair >= a.n_tokens * a.nq) return;
  span_row_fwd(a, pair / a.nq, (int)(pair % a.nq), out, lse, s[w]);
}

}  // namespace

extern "C" int dk_attn_span_fwd(const void* qkv, const int32_t* spans, int64_t n_tokens, int32_t nq,
                                int32_t nkv, int32_t hd, void* out, float* lse, hipStream_t stream) {
  SpanArgs a;
  if (int e = span_args(a, qkv, spans, n_tokens, nq, nkv, hd)) return e;
  if (n_tokens == 0) return 0;
  if (!out || !lse) return DK_ERR_INVALID;
  if (!dk_aligned(out, 16) || !dk_aligned(lse, 4)) return DK_ERR_ALIGN;
  const int64_t wgs = (n_tokens * nq + 3) / 4;
  if (wgs > INT32_MAX / kAThreads) return DK_ERR_INVALID;
  hipLaunchKernelGGL(span_fwd_rows_kernel, dim3((unsigned)wgs), dim3(kAThreads), 0, stream, a,
                     (f16*)out, lse);
  DK_CHECK_LAUNCH();
  return 0;
}
