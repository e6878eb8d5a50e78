"""LM head over the vocabulary without full logits: loss, entropy, argmax accuracy, lse and
d(hidden) in one pass over vocabulary chunks.

Drop-in for the streamed head of the reference's solution/k_head.py (``ResidentEmbedding``,
``streamed_head``, ``STATE_W``: same names, arguments and results).  Per chunk of the embedding:
    logits_c = Y E_c^T          dk_h16_linear_fwd_lora (fp16 out, the 256-tile GEMM)
    dk_head_chunk               running (max, sum, entropy sum, argmax, target logit) per row;
                                P = p_scale e^(x - m) written in place for rows with a target
    acc += P E_c                dk_h16_linear_bwd_dx_lora with fp32 accumulation
then dk_head_finalize gives (loss, entropy, hit, lse) per row and d(hidden) in token order.  Only
[N, chunk] logits exist at a time.  The embedding stays resident in HBM (288 GB per GPU holds it
many times over): the reference's host-memory EmbeddingStream is not needed on this GPU.
"""

import torch

from . import _lib
from .w4linear import _h16_workspace, _needed

STATE_W = 8          # per-row running state: m, s, t, argmax, x_target, (pad)
CHUNK = 32768        # vocabulary rows per chunk (a multiple of 64): at 2048 tokens a 134 MB
                     # logits buffer; measured 2.81 / 2.49 / 2.45 ms per full-vocabulary call at
                     # 8192 / 16384 / 32768 (fewer split-K reduces and launches per call)
OFFSETS = 1 << 31    # elements of yf that the scoring head's offsets reach


class ResidentEmbedding:
    """The embedding on the GPU: chunk c is a view of it (solution/k_head.py:180-199)."""

    def __init__(self, emb, chunk=CHUNK):
        if emb.dtype != torch.float16 or not emb.is_cuda or not emb.is_contiguous() or emb.dim() != 2:
            raise ValueError("the embedding must be a contiguous CUDA fp16 [vocab, hidden] tensor")
        if chunk % 64 or emb.shape[0] % 64 or emb.shape[1] % 64:
            raise ValueError("chunk, vocabulary and hidden size must be multiples of 64")
        self.emb, self.chunk = emb, int(chunk)
        self.vocab = emb.shape[0]
        self.n_chunks = -(-self.vocab // self.chunk)

    def start(self):
        pass

    def get(self, c):
        v0 = c * self.chunk
        return self.emb[v0:min(v0 + self.chunk, self.vocab)]

    def release(self, c):
        pass

    def rows(self, idx_dev, idx_cpu=None):
        return self.emb.index_select(0, idx_dev)


def _logits(ys, e_c, out):
    """out [N, vc] = fp16(ys e_c^T).  A chunk whose size is not a multiple of 256 (the
    vocabulary's last) runs as two GEMMs, the columns up to the last multiple of 256 on the
    256 x 256-tile kernel and the rest on their own: one GEMM over all of them would take the
    smaller tiles throughout (measured on MI355X, 2048 x 20,864 x 1536: 280 us)."""
    n, d = ys.shape
    vc = e_c.shape[0]
    split = vc - vc % 256 if vc > 256 else vc
    for c0, c1 in ((0, split), (split, vc)):
        if c1 == c0:
            continue
        ws, nbytes = _h16_workspace(n, c1 - c0, d, _lib.DK_OP_LINEAR_FWD, ys.device)
        rc = _lib.lib().dk_h16_linear_fwd_lora(_lib.ptr(ys), d, n, _lib.ptr(e_c[c0:]), c1 - c0, d,
                                               None, None, 0, 0, _lib.ptr(out[:, c0:]), vc,
                                               _lib.ptr(ws), nbytes, None,
                                               _lib.stream_handle(ys.device))
        _lib.check(rc, "dk_h16_linear_fwd_lora (logits)")


def _accumulate(acc, p16, e_c):
    """acc [n_lab, d] (fp32) += p16 [n_lab, vc] e_c [vc, d], fp16 inputs, fp32 accumulation in place
    (solution/k_head.py:164-175)."""
    m, vc = p16.shape
    d = e_c.shape[1]
    ws, nbytes = _h16_workspace(m, vc, d, _lib.DK_OP_LINEAR_BWD_DX, acc.device)
    rc = _lib.lib().dk_h16_linear_bwd_dx_lora(_lib.ptr(p16), p16.stride(0), m, _lib.ptr(e_c), vc, d,
                                              None, 0, 0, _lib.ptr(acc), d, _lib.DK_OUT_F32_ACCUM,
                                              _lib.ptr(ws), nbytes, None,
                                              _lib.stream_handle(acc.device))
    _lib.check(rc, "dk_h16_linear_bwd_dx_lora (head accumulate)")


def streamed_head(yf, source, tgt_sorted, perm, n_lab, e_target, grad_scale, dummy32=None):
    """LM head of the packed batch (solution/k_head.py:277-311).

    yf [N, D] fp16 final-norm output in token order; source: ResidentEmbedding; tgt_sorted [N]
    int32 targets (-1 = none) in the order `perm` (tokens with a target first, n_lab of them);
    e_target [n_lab, D] fp16 embedding rows of those targets.  Returns (loss_sum fp32 scalar,
    stats [N, 4] (loss, entropy, hit, lse) in sorted order, dY [N, D] fp16 = grad_scale *
    d(sum CE)/d(yf) in token order)."""
    n, d = yf.shape
    dev = yf.device
    if yf.dtype != torch.float16 or not yf.is_contiguous() or d % 64:
        raise ValueError("yf must be a contiguous fp16 [N, D] tensor, D a multiple of 64")
    for t, nm in ((tgt_sorted, "tgt_sorted"), (perm, "perm")):
        if t.dtype != torch.int32 or tuple(t.shape) != (n,) or not t.is_contiguous():
            raise ValueError(f"{nm} must be a contiguous int32 [{n}] tensor")
    if not 0 <= n_lab <= n:
        raise ValueError("n_lab must be within [0, N]")
    if n_lab > 0 and (e_target.dtype != torch.float16 or tuple(e_target.shape) != (n_lab, d)
                      or not e_target.is_contiguous()):
        raise ValueError(f"e_target must be a contiguous fp16 [{n_lab}, {d}] tensor")
    ys = yf.index_select(0, perm)
    state = torch.zeros((n, STATE_W), dtype=torch.float32, device=dev)
    state[:, 0] = float("-inf")
    acc = torch.zeros((max(n_lab, 1), d), dtype=torch.float32, device=dev)
    buf = torch.empty((n * source.chunk,), dtype=torch.float16, device=dev)
    lib = _lib.lib()
    for c in range(source.n_chunks):
        e_c = source.get(c)
        vc = e_c.shape[0]
        logits = buf[:n * vc].view(n, vc)
        _logits(ys, e_c, logits)
        rc = lib.dk_head_chunk(_lib.ptr(logits), _lib.ptr(tgt_sorted), _lib.ptr(state),
                               _lib.ptr(acc), n, n_lab, vc, c * source.chunk, float(grad_scale), d,
                               _lib.stream_handle(dev))
        _lib.check(rc, "dk_head_chunk")
        if n_lab > 0:
            _accumulate(acc[:n_lab], logits[:n_lab], e_c)
        source.release(c)
    del buf, ys
    stats = torch.empty((n, 4), dtype=torch.float32, device=dev)
    dy = torch.empty((n, d), dtype=torch.float16, device=dev)
    rc = lib.dk_head_finalize(_lib.ptr(state), _lib.ptr(tgt_sorted), _lib.ptr(perm), _lib.ptr(acc),
                              _lib.ptr(e_target) if n_lab > 0 else None, _lib.ptr(stats),
                              _lib.ptr(dy), n, n_lab, float(grad_scale), 1.0 / float(grad_scale),
                              d, _lib.stream_handle(dev))
    _lib.check(rc, "dk_head_finalize")
    return stats[:, 0].sum(), stats, dy


def token_logprobs(yf, emb, tgt, *, rows=None, scale=1.0):
    """Log-probabilities of given tokens under the head, without its gradient and without logits in memory
    (the reference's or an earlier policy's scores; no counterpart in the reference).

    yf [N, D] fp16 final-norm output (rows may be strided); emb: ResidentEmbedding or [V, D] fp16;
    tgt int32 [n] token ids (below 0: none, logp 0; V or more: NaN); rows: None (n = N) or int32 [n], the
    rows of yf that are scored; scale: a factor of the logits (1 / temperature).  Returns (logp, entropy,
    lse) fp32 [n] of the softmax of scale * yf E^T, the logits in fp32."""
    if isinstance(emb, ResidentEmbedding):
        emb = emb.emb
    if yf.dtype != torch.float16 or not yf.is_cuda or yf.dim() != 2:
        raise ValueError("yf must be a CUDA fp16 [N, D] tensor")
    dev = yf.device
    total, d = yf.shape
    if emb.dtype != torch.float16 or emb.device != dev or emb.dim() != 2 or emb.shape[1] != d or \
            emb.shape[0] < 1 or not emb.is_contiguous():
        raise ValueError(f"the embedding must be a contiguous fp16 [vocab, {d}] tensor on {dev}")
    if d % 64 or d == 0:
        raise ValueError("the hidden size must be a multiple of 64")
    if total > 1 and (yf.stride(1) != 1 or yf.stride(0) < d or yf.stride(0) % 8):
        raise ValueError("yf's rows must be contiguous, their stride at least D and a multiple of 8")
    n = total
    if rows is not None:
        n = rows.shape[0] if rows.dim() == 1 else -1
    for t, nm in ((tgt, "tgt"), (rows, "rows")):
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (n,) or t.device != dev or
                              not t.is_contiguous()):
            raise ValueError(f"{nm} must be a contiguous int32 [n] tensor on {dev}")
    if not 0.0 < scale <= 1e6:
        raise ValueError(f"scale must be within (0, 10^6] (got {scale})")
    logp, entropy, lse = torch.empty(3, n, dtype=torch.float32, device=dev).unbind(0)
    if n == 0:
        return logp, entropy, lse
    if total == 0:
        raise ValueError("rows of an empty yf")
    if total == 1 and (yf.stride(1) != 1 or yf.stride(0) < d or yf.stride(0) % 8):
        yf = yf.reshape(d).clone().view(1, d)
    # the kernel's row offsets are 32 bits wide, over all of yf or (without rows) over 256 rows
    if ((total if rows is not None else min(total, 256)) - 1) * yf.stride(0) + d >= OFFSETS:
        if rows is None:
            yf = yf.contiguous()
        elif n > (OFFSETS - 1) // d:
            for i in range(0, n, (OFFSETS - 1) // d):
                part = slice(i, i + (OFFSETS - 1) // d)
                for whole, piece in zip((logp, entropy, lse),
                                        token_logprobs(yf, emb, tgt[part], rows=rows[part], scale=scale)):
                    whole[part] = piece
            return logp, entropy, lse
        else:                  # the picked rows alone (an index outside stays one)
            inside = (rows >= 0) & (rows < total)
            yf = yf.index_select(0, torch.where(inside, rows, 0))
            rows = torch.where(inside, torch.arange(n, dtype=torch.int32, device=dev), -1)
            total = n
    lib = _lib.lib()
    vocab = emb.shape[0]
    nbytes = _needed(("logprobs", n, vocab, d), lambda: lib.dk_head_logprobs_workspace(n, vocab, d))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _lib.launch(dev, lib.dk_head_logprobs, "dk_head_logprobs", yf.data_ptr(), yf.stride(0), total,
                _lib.ptr(rows), n, emb.data_ptr(), vocab, d, tgt.data_ptr(), scale,
                logp.data_ptr(), entropy.data_ptr(), lse.data_ptr(), ws.data_ptr(), nbytes)
    return logp, entropy, lse


def warmup_specs(hidden=1536, chunk=CHUNK, impl="chunks"):
    """Nothing to warm up: the kernels are compiled ahead of time into libdk.so."""
    return []
