"""Losses over the log-probabilities of a packed batch's answers, with their gradients: the clipped policy
loss with a KL term and the preference loss over pairs of answers (no counterpart in the reference, whose
step trains on cross entropy alone).

The tokens are the batch's labelled ones in sorted order (trainer.pack, trainer.pack_answers), row after
row; ``row_meta`` is their plan, made once per batch from the rows' lengths (trainer.answer_lens):

    meta = row_meta(lens, device)                                   # or row_meta(lens, device, pairs=...)
    loss, dlogp, stats = policy_loss(stats_now, old, advantages, meta, ref=ref, kl_coef=0.04)
    loss, dlogp, rewards, margins = preference_loss(stats_now, ref, meta, beta=0.1)

Log-probabilities are fp32: [n] (any stride) as k_head.token_logprobs returns them, or the streamed head's
stats [N >= n, 4], whose first column is their negative.  16-bit log-probabilities are refused: their
rounding (2^-9 of a value of some units) is of the size of the clip range.  dlogp [n] is the loss's
gradient for the log-probabilities; as the streamed head's gradient is that of the summed cross entropy,
-dlogp are the factors of its rows (row_factors, k_norm.rms_backward's row_scale;
model.QwenQLoRAStep.policy_step).
"""

import math

import numpy as np
import torch

from . import _lib

ITEM_TOKENS = 512    # tokens that a wave takes; longer rows than ROW_ITEMS of these in larger items
ROW_ITEMS = 64
MAX_ITEMS = 1 << 25  # a wave each: 2^32 work items are more than a launch takes
REDUCTIONS = ("row", "token", "sum")
KINDS = ("sigmoid", "hinge", "ipo")


def _whole(values, what, shape):
    """A list of whole numbers, or of pairs of them, as int64."""
    values = np.asarray(values)
    if values.size and (values.dtype.kind not in "iu" or values.shape[1:] != shape or values.ndim == 0):
        raise ValueError(f"{what} must be whole numbers" if not shape else f"{what} must be pairs of whole numbers")
    return values.astype(np.int64).reshape(-1, *shape)


class RowMeta:
    """The plan of rows of consecutive tokens (see row_meta): on the device the kernels' items, each row's
    items, and the pairs with each row's share of them."""

    def __init__(self, lens, device, pairs=None):
        size = _whole(lens, "lens", ())
        rows = size.size
        if rows == 0 or size.min() < 0 or size.max() > 1 << 30:
            raise ValueError("at least one row, each of 0 to 2^30 tokens")
        self.n_rows, self.n_tokens = int(rows), int(size.sum())
        self.n_filled = int(np.count_nonzero(size))
        step = np.maximum(ITEM_TOKENS, -(-(-(-size // ROW_ITEMS)) // 64) * 64)
        count = np.maximum(1, -(-size // step))
        last = np.cumsum(count)
        n = self.n_items = int(last[-1])
        if n > MAX_ITEMS:
            raise ValueError(f"a plan takes up to 2^25 items (here {n}: one for each {ITEM_TOKENS} tokens of a row, "
                             f"up to {ROW_ITEMS} a row, and at least one a row)")
        self.n_pairs = None
        both = None
        if pairs is not None:
            both = _whole(pairs, "pairs", (2,))
            if both.size == 0 or both.min() < 0 or both.max() >= rows or len(both) > 1 << 28:
                raise ValueError(f"at least one pair of rows 0 .. {rows - 1}")
            self.n_pairs = len(both)
        # one buffer: items, the pairs' entries and the pairs, row_pairs, row_items
        k = self.n_pairs or 0
        first = np.cumsum([0, 8 * n, 4 * k, 2 * k, (rows + 1) if k else 0]).tolist()
        flat = np.empty(first[-1] + rows + 1, np.int32)
        items = flat[:8 * n].reshape(n, 8)
        row = np.repeat(np.arange(rows), count)
        of = count[row]
        place = np.arange(n) - (last - count)[row]
        at = place * step[row]                                        # first token within the row
        begin = (np.cumsum(size) - size)[row] + at
        items[:, 0], items[:, 1] = begin.astype(np.uint32).view(np.int32), begin >> 32
        items[:, 2], items[:, 3] = np.minimum(step[row], size[row] - at), row
        items[:, 4], items[:, 5], items[:, 6], items[:, 7] = size[row], of, place, 0
        flat[first[4]] = 0
        flat[first[4] + 1:] = last
        if k:
            own = both.T.reshape(-1)                                  # chosen rows, then rejected ones
            index = np.arange(1, k + 1)
            order = np.argsort(own, kind="stable")
            entries = flat[first[1]:first[2]].reshape(2 * k, 2)
            entries[:, 0] = both[:, ::-1].T.reshape(-1)[order]
            entries[:, 1] = np.concatenate([index, -index])[order]
            flat[first[2]:first[3]] = both.reshape(-1)
            flat[first[3]] = 0
            flat[first[3] + 1:first[4]] = np.cumsum(np.bincount(own, minlength=rows))
        self._buffer = torch.from_numpy(flat).to(torch.device(device))
        self.device = self._buffer.device
        base = self._buffer.data_ptr()
        self.at = {name: base + 4 * i for name, i in
                   zip(("items", "entries", "pairs", "row_pairs", "row_items"), first)}
        self._stream = _lib.stream_handle(self.device) if self.device.type == "cuda" else None
        lib = _lib.lib()
        self.policy_bytes = lib.dk_policy_loss_workspace(n, self.n_tokens)
        self.preference_bytes = lib.dk_preference_loss_workspace(n, self.n_tokens, k)

    def kept(self):
        """The kernels' addresses; a plan used on another stream than the one it was made on keeps its memory
        until that stream is done with it, also when it is dropped before."""
        if _lib.stream_handle(self.device) != self._stream:
            self._buffer.record_stream(torch.cuda.current_stream(self.device))
        return self.at


def row_meta(lens, device, pairs=None):
    """The plan of a batch with rows of `lens` tokens (zeros allowed, 2^25 rows at most), and for
    preference_loss of the pairs (chosen row, rejected row); a row may be in any number of pairs."""
    return RowMeta(lens, device, pairs)


def _tokens(t, what, meta):
    """A token array's (address, stride, negated): [n] log-probabilities, or the head's stats."""
    if t is None:
        return 0, 0, 0
    if t.dtype != torch.float32 or t.get_device() != meta.device.index:   # (a CPU tensor's is -1)
        raise ValueError(f"{what} must be a CUDA fp32 tensor on the plan's device ({meta.device})")
    if t.dim() == 1 and t.shape[0] == meta.n_tokens:
        return t.data_ptr(), t.stride(0), 0
    if t.dim() == 2 and t.shape[0] >= meta.n_tokens and t.shape[1] == 4:
        return t.data_ptr(), t.stride(0), 1
    raise ValueError(f"{what} must be [{meta.n_tokens}] log-probabilities, or the head's stats [N, 4] with "
                     f"these tokens first (got {tuple(t.shape)})")


def policy_loss(logp, old, advantages, meta, *, ref=None, kl_coef=0.0, clip_low=0.2, clip_high=None,
                reduction="row", per_token=False):
    """Clipped policy loss: with r = e^(logp - old) and A a token's advantage
        sum w (-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (e^f - f - 1)),  f = ref - logp
    (clip_high None: clip_low).  advantages fp32 [rows], or [n] with per_token.  reduction "row": the mean
    over rows (that have tokens) of their tokens' means; "token": the mean over all tokens; "sum".
    Returns (loss, dlogp [n], stats [rows, 4]): stats are a row's means of the policy term, of the KL
    estimate e^f - f - 1 (0 without ref), of clipped tokens and of r; 0 for a row without tokens.  A token
    that lies on a border is not clipped.  An advantage of 0, and a kl_coef of 0, leave nothing of their
    terms, infinite ones included.  All fp32."""
    clip_high = clip_low if clip_high is None else clip_high
    if not (0.0 <= clip_low <= 1.0 and clip_high >= 0.0):
        raise ValueError(f"clip_low must be within [0, 1], clip_high at least 0 (got {clip_low}, {clip_high})")
    if not math.isfinite(kl_coef) or (kl_coef and ref is None):
        raise ValueError("kl_coef must be finite, and needs ref")
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {REDUCTIONS}")
    if logp is None or old is None:
        raise ValueError("logp and old are needed")
    n, rows, dev = meta.n_tokens, meta.n_rows, meta.device
    tokens = _tokens(logp, "logp", meta) + _tokens(old, "old", meta) + _tokens(ref, "ref", meta)
    if advantages.dtype != torch.float32 or advantages.device != dev or not advantages.is_contiguous() or \
            tuple(advantages.shape) != ((n,) if per_token else (rows,)):
        raise ValueError(f"advantages must be a contiguous fp32 [{n if per_token else rows}] tensor on {dev}")
    dlogp = torch.empty(n, dtype=torch.float32, device=dev)
    stats = torch.empty(rows, 4, dtype=torch.float32, device=dev)
    loss = torch.empty_strided((), (), dtype=torch.float32, device=dev)
    nbytes = meta.policy_bytes
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    which, at = REDUCTIONS.index(reduction), meta.kept()
    args = _lib.POLICY_ARGS.pack(
        at["items"], meta.n_items, at["row_items"], rows, n, *tokens, advantages.data_ptr(),
        1 if per_token else 0, clip_low, clip_high, kl_coef, which, (meta.n_filled, n, 1)[which] or 1,
        dlogp.data_ptr(), stats.data_ptr(), loss.data_ptr(), ws.data_ptr() if nbytes else 0, nbytes)
    _lib.launch(dev, _lib.lib().dk_policy_loss, "dk_policy_loss", args)
    return loss, dlogp, stats


def preference_loss(logp, ref, meta, *, beta=0.1, kind="sigmoid", label_smoothing=0.0, margin=0.0,
                    average=False):
    """Loss over the plan's pairs of rows: with S a row's sum (average: mean) of logp - ref (ref None:
    logp) and h = beta (S_chosen - S_rejected) - margin, the mean over pairs of
        "sigmoid"  -(1 - e) log s(h) - e log s(-h), s the logistic function, e = label_smoothing
        "hinge"    max(0, 1 - h)
        "ipo"      ((h - 1/2) / beta)^2
    Returns (loss, dlogp [n], rewards [rows] = beta S, margins [pairs] = h), fp32; a row without tokens has
    S = 0."""
    if meta.n_pairs is None:
        raise ValueError("the plan has no pairs (row_meta(..., pairs=...))")
    if not 0.0 < beta < math.inf or not math.isfinite(margin):
        raise ValueError(f"beta must be positive and margin finite (got {beta}, {margin})")
    if kind not in KINDS:
        raise ValueError(f"kind must be one of {KINDS}")
    if not 0.0 <= label_smoothing <= 0.5 or (label_smoothing and kind != "sigmoid"):
        raise ValueError("label_smoothing must be within [0, 1/2], and is the sigmoid loss's alone")
    if logp is None:
        raise ValueError("logp is needed")
    n, rows, dev = meta.n_tokens, meta.n_rows, meta.device
    tokens = _tokens(logp, "logp", meta) + _tokens(ref, "ref", meta)
    dlogp = torch.empty(n, dtype=torch.float32, device=dev)
    rewards = torch.empty(rows, dtype=torch.float32, device=dev)
    margins = torch.empty(meta.n_pairs, dtype=torch.float32, device=dev)
    loss = torch.empty_strided((), (), dtype=torch.float32, device=dev)
    nbytes, at = meta.preference_bytes, meta.kept()
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    args = _lib.PREFERENCE_ARGS.pack(
        at["items"], meta.n_items, at["row_items"], rows, n, at["row_pairs"], at["entries"], at["pairs"],
        meta.n_pairs, *tokens, beta, KINDS.index(kind), label_smoothing, margin, 1 if average else 0,
        dlogp.data_ptr(), rewards.data_ptr(), margins.data_ptr(), loss.data_ptr(),
        ws.data_ptr() if nbytes else 0, nbytes)
    _lib.launch(dev, _lib.lib().dk_preference_loss, "dk_preference_loss", args)
    return loss, dlogp, rewards, margins


def row_factors(dlogp, rows, n):
    """A loss's gradient dlogp [k] as factors of the head's rows (k_norm.rms_backward's row_scale): fp32 [n], 0
    but for -dlogp / unit at rows (int32 [k], none twice; those outside are left out), and unit, the largest
    power of two up to the largest |dlogp| (an fp32 scalar; 1 if that is 0 or not finite).  Losses that are
    means over many tokens have gradients of 1e-4 and less, which a backward in fp16 would lose: divided by
    unit it has the range of the cross entropy's, and k_grad.scale_grads(gradients, unit) undoes it in fp32."""
    dev = dlogp.device
    if dlogp.dtype != torch.float32 or dlogp.dim() != 1 or not dlogp.is_cuda:
        raise ValueError("dlogp must be a CUDA fp32 [k] tensor")
    if rows.dtype != torch.int32 or rows.shape != dlogp.shape or rows.device != dev or not rows.is_contiguous():
        raise ValueError(f"rows must be a contiguous int32 [{dlogp.shape[0]}] tensor on {dev}")
    if n < 0:
        raise ValueError("n must be at least 0")
    dlogp = dlogp.contiguous()
    factors = torch.empty(n, dtype=torch.float32, device=dev)
    unit = torch.empty_strided((), (), dtype=torch.float32, device=dev)
    _lib.launch(dev, _lib.lib().dk_row_factors, "dk_row_factors", dlogp.data_ptr(), rows.data_ptr(),
                dlogp.shape[0], factors.data_ptr(), n, unit.data_ptr())
    return factors, unit
