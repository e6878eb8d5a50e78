"""Variable-length causal GQA attention of the padding-free packed batch, forward and backward.

Drop-in for the attention kernels of the reference's solution/k_attn.py (``block_table``,
``AttnMeta``, ``attention_forward``, ``attention_backward``, ``warmup_specs``: same names,
arguments and results), running the gfx950 kernels ``dk_attn_fwd`` / ``dk_attn_bwd`` of
libdk.so.  The packed tokens' queries, keys and values live in one row of the fused QKV buffer
[N, (nq + 2 nkv) hd] fp16; blocks of 128 rows (queries in the forward and dQ, keys in dK/dV) never
straddle two sequences, so the mask is ``key <= query`` inside a sequence.

forward   online softmax in the exp2 domain (scores scaled by log2(e) / sqrt(hd)), fp32 running
          max and sum, P rounded to fp16 for the P V product; out fp16 [N, nq hd], lse fp32
          [nq, N] = m + log2(l)
backward  delta = rowsum(O dO); dQ fp32 [N, nq hd]; dK, dV fp32 per query head [N, nq hd], which
          the QKV epilogue backward sums over each group of nq / nkv heads (gin)

The reference's block sizes are parameters of its Triton kernels; here the blocks are fixed by
the kernels (128 rows per workgroup, tiles of 64), and ``block_table`` must be built for
FWD_BLOCK_M and BWD_BLOCK.

``span_attention_forward`` / ``span_attention_backward`` (no counterpart in the reference) run the
same attention over part of the keys, named by a plan built once per batch:
``window_meta``   query i of a sequence sees its keys j <= i with i - j < window or j < sinks
``prefix_meta``   groups of a prompt and several answers, the prompt packed once: an answer's token
                  sees the whole prompt and its own answer up to itself
Both are batches in which key n is seen by the queries n .. kend[n] - 1.  The gradients come back in
fp16 (the products behind them take fp16 P and dS), dK and dV summed over each group's heads: the QKV
epilogue backward takes them with gin = 1.
"""

import numpy as np
import torch

from . import _lib

FWD_BLOCK_M, FWD_BLOCK_N = 128, 64
BWD_BLOCK = 128
ATTN_WARPS = 4
HEAD_DIM = 128


def block_table(lens, block):
    """Flat [seq, start, seq, start, ...] for every block of `block` rows of every sequence
    (solution/k_attn.py:185-191)."""
    tab = []
    for s, n in enumerate(lens):
        for start in range(0, n, block):
            tab += (s, start)
    return tab


def bwd_block_table(lens, block):
    """``block_table``'s blocks ordered by the rows from a block's start to its sequence's end,
    longest first (stable).  The backward launch runs its dK/dV blocks in table order and its dQ
    blocks in reverse order, dealt to the XCDs round-robin, so this order starts the longest walks
    first and gives every XCD a balanced share; any order gives the same results."""
    tab = block_table(lens, block)
    pairs = [(tab[i], tab[i + 1]) for i in range(0, len(tab), 2)]
    pairs.sort(key=lambda p: -(int(lens[p[0]]) - p[1]))
    return [v for p in pairs for v in p]


class AttnMeta:
    """Per-batch tables (device int32 tensors) for the attention kernels
    (solution/k_attn.py:194-199)."""

    def __init__(self, cu, tab_fwd, tab_bwd, n_fwd, n_bwd, n_tokens):
        self.cu, self.tab_fwd, self.tab_bwd = cu, tab_fwd, tab_bwd
        self.n_fwd, self.n_bwd, self.n_tokens = n_fwd, n_bwd, n_tokens


def meta_for(lens, device):
    """AttnMeta of a packed batch with sequence lengths `lens` (as solution/test_kernels.py:261-269
    builds it)."""
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + int(n))
    tf, tb = block_table(lens, FWD_BLOCK_M), bwd_block_table(lens, BWD_BLOCK)
    i32 = dict(dtype=torch.int32, device=device)
    return AttnMeta(torch.tensor(cu, **i32), torch.tensor(tf, **i32), torch.tensor(tb, **i32),
                    len(tf) // 2, len(tb) // 2, cu[-1])


def _t(t, dtypes, what, shape=None):
    if t.dtype not in dtypes or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous CUDA tensor of {dtypes}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t


def _check(qkv, meta, nq, nkv, hd, tab, n_blocks):
    if hd != HEAD_DIM or nq % nkv:
        raise ValueError(f"head size {HEAD_DIM} and nq a multiple of nkv (got {hd}, {nq}, {nkv})")
    n = meta.n_tokens
    _t(qkv, (torch.float16,), "qkv", (n, (nq + 2 * nkv) * hd))
    _t(meta.cu, (torch.int32,), "meta.cu")
    _t(tab, (torch.int32,), "block table", (2 * n_blocks,))
    if meta.cu.dim() != 1 or meta.cu.numel() < 2:
        raise ValueError("meta.cu must hold at least one sequence")


def attention_forward(qkv, meta, nq, nkv, hd, block_m=FWD_BLOCK_M, block_n=FWD_BLOCK_N,
                      warps=ATTN_WARPS):
    """(out [N, nq hd] fp16, lse [nq, N] fp32).  meta.tab_fwd must be the block table for
    FWD_BLOCK_M (solution/k_attn.py:202-212)."""
    if (block_m, block_n) != (FWD_BLOCK_M, FWD_BLOCK_N):
        raise ValueError(f"the forward kernel's blocks are {FWD_BLOCK_M} x {FWD_BLOCK_N}")
    _check(qkv, meta, nq, nkv, hd, meta.tab_fwd, meta.n_fwd)
    n = meta.n_tokens
    out = torch.empty((n, nq * hd), dtype=torch.float16, device=qkv.device)
    lse = torch.empty((nq, n), dtype=torch.float32, device=qkv.device)
    rc = _lib.lib().dk_attn_fwd(_lib.ptr(qkv), _lib.ptr(meta.cu), meta.cu.numel() - 1,
                                _lib.ptr(meta.tab_fwd), meta.n_fwd, n, nq, nkv, hd, _lib.ptr(out),
                                _lib.ptr(lse), _lib.stream_handle(qkv.device))
    _lib.check(rc, "dk_attn_fwd")
    return out, lse


def attention_backward(qkv, out, lse, dout, meta, nq, nkv, hd, block=BWD_BLOCK, warps=ATTN_WARPS):
    """fp32 dq [N, nq hd] and per-query-head dk, dv partials [N, nq hd].  meta.tab_bwd must be
    the block table for BWD_BLOCK (solution/k_attn.py:215-245)."""
    if block != BWD_BLOCK:
        raise ValueError(f"the backward kernels' block is {BWD_BLOCK}")
    _check(qkv, meta, nq, nkv, hd, meta.tab_bwd, meta.n_bwd)
    n = meta.n_tokens
    _t(out, (torch.float16,), "out", (n, nq * hd))
    _t(dout, (torch.float16,), "dout", (n, nq * hd))
    _t(lse, (torch.float32,), "lse", (nq, n))
    dev = qkv.device
    delta = torch.empty((nq, n), dtype=torch.float32, device=dev)
    dq = torch.empty((n, nq * hd), dtype=torch.float32, device=dev)
    dkp = torch.empty((n, nq * hd), dtype=torch.float32, device=dev)
    dvp = torch.empty((n, nq * hd), dtype=torch.float32, device=dev)
    rc = _lib.lib().dk_attn_bwd(_lib.ptr(qkv), _lib.ptr(out), _lib.ptr(lse), _lib.ptr(dout),
                                _lib.ptr(meta.cu), meta.cu.numel() - 1, _lib.ptr(meta.tab_bwd),
                                meta.n_bwd, n, nq, nkv, hd, _lib.ptr(delta), _lib.ptr(dq),
                                _lib.ptr(dkp), _lib.ptr(dvp), _lib.stream_handle(dev))
    _lib.check(rc, "dk_attn_bwd")
    return dq, dkp, dvp


class SpanMeta:
    """Plan of one packed batch for the attention over part of the keys (window_meta, prefix_meta).

    spans [n, 4] int32 on the device: token m sees, as a query, the keys [a0, a1) and [kbeg, m]; as a
    key it is seen by the queries m .. kend - 1.  positions [n] int32: each token's position (an
    answer's go on from its prompt's), for the rotary embedding.  n_pairs: visible (query, key) pairs of
    a head.  The other tables are the kernels' work, cut into items here on the host (include/dk.h).  A
    plan serves any number of calls, on any streams of its device, captured or not."""

    def __init__(self, runs, key_runs, spans, positions, nq, nkv, device):
        """runs: (first, past the last) token arrays of the runs whose tokens share [a0, a1) and whose kbeg
        does not fall; key_runs: of the runs whose kend does not fall."""
        n = int(spans.shape[0])
        if nq < 1 or nkv < 1 or nq % nkv:
            raise ValueError(f"nq must be a multiple of nkv (got {nq}, {nkv})")
        if n > MAX_SPAN_TOKENS:
            raise ValueError(f"at most {MAX_SPAN_TOKENS} tokens (got {n})")
        self.n_tokens, self.nq, self.nkv = n, int(nq), int(nkv)
        self.n_pairs = int((spans[:, 3] - np.arange(n)).sum())
        blocks = _query_blocks(runs, spans, nq, nkv)
        items, joins, self.n_slots = _split_items(blocks, blocks[:, _TE], _fwd_tiles(blocks))
        blocks = np.concatenate([_key_blocks(key_runs, spans, nq // nkv, nkv), blocks])
        cost = blocks[:, _TE] * _TILE_COST[blocks[:, _KIND]]
        items_b, joins_b, self.n_units = _split_items(blocks, cost, _bwd_cost(cost))
        if max(len(items), len(items_b)) > MAX_SPAN_ITEMS or max(len(joins), len(joins_b)) > MAX_SPAN_JOINS:
            raise ValueError(f"a batch of {max(len(items), len(items_b))} items and {max(len(joins), len(joins_b))} "
                             f"split walks (at most {MAX_SPAN_ITEMS} and {MAX_SPAN_JOINS})")
        lib = _lib.lib()
        self.fwd_bytes = lib.dk_attn_span_workspace(self.n_slots)
        self.bwd_bytes = lib.dk_attn_span_bwd_workspace(self.n_units)
        # one copy to the device, every table 16-byte aligned in it
        tables = (spans, items, joins, items_b, joins_b, positions)
        ends = np.cumsum([t.size + -t.size % 4 for t in tables])
        flat = np.zeros(int(ends[-1]), np.int32)
        for t, end in zip(tables, ends):
            end -= t.size + -t.size % 4
            flat[end:end + t.size] = t.reshape(-1)
        flat = torch.from_numpy(flat).to(device)
        (self.spans, self.items, self.joins, self.items_bwd, self.joins_bwd, self.positions) = (
            flat[end - (t.size + -t.size % 4):][:t.size].view(t.shape) for t, end in zip(tables, ends))


MAX_SPAN_TOKENS = (1 << 30) - 1
# what a launch takes (include/dk.h): blocks of 128 rows of every run and KV head, their cuts, and twice that
# in the backward; runs are sequences, sinks, prompts and groups' answers
MAX_SPAN_ITEMS = ((1 << 31) - 1) // 256
MAX_SPAN_JOINS = ((1 << 31) - 1) // 1024
_KEYS = 64            # keys of a tile
_ROWS = 128           # stacked query rows of a block
_REACH = 0xfff00000   # DK_ATTN_SPAN_REACH_BYTES
# columns of an item (include/dk.h)
_T0, _PHASE, _N_ROWS, _G, _A0, _NA, _B0, _NK, _F0, _F1, _F2, _TB, _TE, _SLOT, _KIND = range(15)
_QEND = 4             # of a block of keys
# a tile of a dQ walk, of a dK/dV walk of 128 keys and of 32: 48, 64 and 16 MFMAs a wave, the last not
# overlapped
_TILE_COST = np.array([3, 4, 2])


def _blocks_of(runs, per_token, size):
    """(run, first) of every block of `size` of each run's per_token elements per token."""
    n = -(-(runs[1] - runs[0]) * per_token // size)
    run = np.repeat(np.arange(n.size), n)
    return run, (np.arange(run.size) - np.repeat(np.cumsum(n) - n, n)) * size


def _each_head(x, nkv):
    """The items x for every KV head."""
    y = np.tile(x, (nkv, 1))
    y[:, _G] = np.repeat(np.arange(nkv), len(x))
    return y


def _query_blocks(runs, spans, nq, nkv):
    """The blocks of stacked query rows of every run and KV head, as items [n, 16] that walk all of their
    tiles."""
    gin, row_bytes = nq // nkv, 2 * HEAD_DIM * (nq + 2 * nkv)
    run, j0 = _blocks_of(runs, gin, _ROWS)
    r0, r1 = runs[0][run], runs[1][run]
    rows = np.minimum(_ROWS, (r1 - r0) * gin - j0)
    t0, last = r0 + j0 // gin, r0 + (j0 + rows - 1) // gin
    a0, a1, kbeg = (spans[t0, i] for i in range(3))
    # the window of the first row meets the sinks: one run of keys from a0
    one = (a1 > a0) & (kbeg <= a1)
    b0 = np.where(one, a0, kbeg)
    seen = np.where(one | (a1 <= a0), 0, a1 - a0)
    # A tile of both runs' keys needs them within the kernels' 32-bit offsets.  Beyond, the first run
    # goes on to the end of its tile: keys that no row of the block sees.
    far = (b0 - a0 - seen + _KEYS) * row_bytes >= _REACH
    na = np.where(far, -(-seen // _KEYS) * _KEYS, seen)
    if (a0 + na > b0)[far].any():
        raise ValueError(f"rows of {row_bytes} bytes are too long for keys that far apart")
    nk = na + last + 1 - b0
    # every row sees the first run up to t0, also where both are one, and the keys from the last row's kbeg
    # to t0
    first = np.where(one, np.minimum(a1, t0 + 1) - a0, seen)
    lo = np.maximum(spans[last, 2], b0) - b0 + na
    hi = t0 - b0 + na + 1
    x = np.zeros((j0.size, 16), np.int64)
    x[:, _T0], x[:, _PHASE], x[:, _N_ROWS] = t0, j0 % gin, rows
    x[:, _A0], x[:, _NA], x[:, _B0], x[:, _NK] = a0, na, b0, nk
    x[:, _F0] = np.where(lo <= first, hi, first) // _KEYS
    x[:, _F1] = -(-lo // _KEYS)
    x[:, _F2] = np.maximum(hi // _KEYS, x[:, _F1])
    x[:, _TE], x[:, _SLOT] = -(-nk // _KEYS), -1
    return _each_head(x, nkv)


def _key_blocks(key_runs, spans, gin, nkv):
    """The blocks of keys of every run and KV head, as items whose walk over the group's heads and their
    queries is whole."""
    run, k0 = _blocks_of(key_runs, 1, _ROWS)
    k0 = k0 + key_runs[0][run]
    nk = np.minimum(_ROWS, key_runs[1][run] - k0)
    x = np.zeros((k0.size, 16), np.int64)
    x[:, _T0], x[:, _N_ROWS], x[:, _SLOT] = k0, nk, -1
    x[:, _KIND] = np.where(nk <= 32, 2, 1)     # few keys (sinks): the walk of 32
    x[:, _QEND] = spans[k0 + nk - 1, 3]
    x[:, _TE] = gin * -(-(x[:, _QEND] - k0) // _KEYS)
    return _each_head(x, nkv)


def _fwd_tiles(blocks):
    """Tiles per item of the forward at most: a little over the share of one of the 512 workgroups that run
    at a time, two to a CU, and no fewer than make up for a partial (over 15 batches 23.4 us; 24.1 with at
    least 4, 24.3 with 8)."""
    return max(5, int(0.6 * blocks[:, _TE].sum() / 256) + 1)


def _bwd_cost(cost):
    """Cost per item of the backward at most: a CU's share of the whole (256 CUs, an item each at a time)
    and a little, so that no walk (a prompt's or a sink's keys over every later query) outlasts the rest,
    and few partials are written (over 13 batches 49.4 us; 50.4 with + 4 or + 12, 51.8 with + 18, 51.3 with a
    factor of 1, 52.6 with 1.6)."""
    return int(1.25 * cost.sum() / 256) + 8


def _split_items(blocks, cost, most):
    """(items, joins, partials): blocks that cost more than `most` cut into walks of as many tiles each,
    the costliest walks first."""
    n = blocks[:, _TE]
    cut = np.minimum(n, -(-cost // most))
    idx = np.repeat(np.arange(n.size), cut)
    part = np.arange(idx.size) - np.repeat(np.cumsum(cut) - cut, cut)
    items = blocks[idx].copy()
    items[:, _TB] = part * n[idx] // cut[idx]
    items[:, _TE] = (part + 1) * n[idx] // cut[idx]
    split = cut > 1
    size = np.where(blocks[:, _KIND] > 0, 2, 1)   # units of a partial: dK and dV take two
    units = np.where(split, cut * size, 0)
    first = np.cumsum(units) - units
    items[:, _SLOT] = np.where(split[idx], first[idx] + part * size[idx], -1)
    joins = np.zeros((int(split.sum()), 8), np.int64)
    joins[:, :4] = blocks[split][:, [_T0, _PHASE, _N_ROWS, _G]]
    joins[:, 4], joins[:, 5], joins[:, 6] = first[split], cut[split], blocks[split][:, _KIND] > 0
    order = np.argsort(-cost[idx] // cut[idx], kind="stable")
    return items[order], joins, int(units.sum())


def _runs(first, last):
    """The runs that hold tokens, of arrays of first and past-the-last tokens."""
    some = last > first
    return first[some], last[some]


def _lengths(lens, what):
    lens = [int(n) for n in lens]
    if any(n < 0 for n in lens):
        raise ValueError(f"{what} must not be negative")
    return lens


def window_meta(lens, window, sinks, nq, nkv, device):
    """Plan of a packed batch with sequence lengths `lens` (zeros allowed) under a causal sliding
    window: query i sees keys j <= i with i - j < window (window >= 1: itself at least) or
    j < sinks (the sequence's first tokens, sinks >= 0)."""
    lens = _lengths(lens, "lens")
    window, sinks = int(window), int(sinks)
    if window < 1 or sinks < 0:
        raise ValueError(f"window must be at least 1 and sinks at least 0 (got {window}, {sinks})")
    window, sinks = min(window, sum(lens) + 1), min(sinks, sum(lens))
    size = np.asarray(lens, np.int64)
    start = np.cumsum(size) - size
    s0, end = np.repeat(start, size), np.repeat(start + size, size)
    m = np.arange(size.sum(), dtype=np.int64)
    spans = np.empty((m.size, 4), np.int64)
    spans[:, 0] = s0
    spans[:, 1] = np.minimum(s0 + sinks, end)
    spans[:, 2] = np.maximum(s0, m - (window - 1))
    spans[:, 3] = np.where(m - s0 < sinks, end, np.minimum(m + window, end))
    last = start + size
    sunk = np.minimum(start + sinks, last)
    key_runs = _runs(np.concatenate([start, sunk]), np.concatenate([sunk, last]))
    return SpanMeta(_runs(start, last), key_runs, spans, m - s0, nq, nkv, device)


def prefix_meta(groups, nq, nkv, device):
    """Plan of a packed batch of groups (prompt length, [answer lengths]), packed as the prompt's tokens
    and then each answer's (zeros allowed).  Prompt tokens are causal; an answer's token sees the
    group's whole prompt and its own answer up to itself, and nothing of the other answers."""
    size, lead = [], []        # the pieces' lengths; 1 at a prompt
    for prompt, answers in groups:
        size += _lengths([prompt], "prompt lengths") + _lengths(answers, "answer lengths")
        lead += [1] + [0] * (len(size) - len(lead) - 1)
    size, lead = np.asarray(size, np.int64), np.asarray(lead, np.int64)
    start = np.cumsum(size) - size
    group = np.cumsum(lead) - 1
    at = np.nonzero(lead)[0]                                   # the prompts
    g0, p1 = start[at], start[at] + size[at]                   # group and prompt ends
    g1 = np.append(g0[1:], size.sum())[:g0.size]
    piece = np.repeat(np.arange(size.size), size)
    g, is_prompt = group[piece], lead[piece] == 1
    m = np.arange(size.sum(), dtype=np.int64)
    spans = np.empty((m.size, 4), np.int64)
    spans[:, 0] = g0[g]
    spans[:, 1] = np.where(is_prompt, g0[g], p1[g])
    spans[:, 2] = start[piece]
    spans[:, 3] = np.where(is_prompt, g1[g], (start + size)[piece])
    positions = m - start[piece] + np.where(is_prompt, 0, size[at][g])
    runs = _runs(np.concatenate([g0, p1]), np.concatenate([p1, g1]))
    return SpanMeta(runs, runs, spans, positions, nq, nkv, device)


def _check_span(qkv, meta, nq, nkv, hd):
    if hd != HEAD_DIM:
        raise ValueError(f"head size {HEAD_DIM} (got {hd})")
    if (nq, nkv) != (meta.nq, meta.nkv):
        raise ValueError(f"the plan is for {meta.nq} / {meta.nkv} heads (got {nq}, {nkv})")
    _t(qkv, (torch.float16,), "qkv", (meta.n_tokens, (nq + 2 * nkv) * hd))
    if meta.spans.device != qkv.device:
        raise ValueError(f"the plan is on {meta.spans.device}, qkv on {qkv.device}")


def span_attention_forward(qkv, meta, nq, nkv, hd):
    """(out [N, nq hd] fp16, lse [nq, N] fp32) of the attention whose plan is `meta`; layouts as for
    attention_forward."""
    _check_span(qkv, meta, nq, nkv, hd)
    n, dev = meta.n_tokens, qkv.device
    out = torch.empty(n, nq * hd, dtype=torch.float16, device=dev)
    lse = torch.empty(nq, n, dtype=torch.float32, device=dev)
    ws = torch.empty(meta.fwd_bytes, dtype=torch.uint8, device=dev) if meta.fwd_bytes else None
    _lib.launch(dev, _lib.lib().dk_attn_span_fwd, "dk_attn_span_fwd", qkv.data_ptr(),
                meta.spans.data_ptr(), meta.items.data_ptr(), meta.items.shape[0], meta.joins.data_ptr(),
                meta.joins.shape[0], meta.n_slots, n, nq, nkv, hd, out.data_ptr(), lse.data_ptr(),
                _lib.ptr(ws), meta.fwd_bytes)
    return out, lse


def span_attention_backward(qkv, out, lse, dout, meta, nq, nkv, hd):
    """(dq [N, nq hd], dk [N, nkv hd], dv [N, nkv hd]) fp16 from the forward's out and lse and the
    gradient dout of out."""
    _check_span(qkv, meta, nq, nkv, hd)
    n, dev = meta.n_tokens, qkv.device
    for t, dt, what, shape in ((out, torch.float16, "out", (n, nq * hd)),
                               (dout, torch.float16, "dout", (n, nq * hd)),
                               (lse, torch.float32, "lse", (nq, n))):
        _t(t, (dt,), what, shape)
        if t.device != dev:
            raise ValueError(f"{what} is on {t.device}, qkv on {dev}")
    delta = torch.empty(nq, n, dtype=torch.float32, device=dev)
    dq = torch.empty(n, nq * hd, dtype=torch.float16, device=dev)
    dk = torch.empty(n, nkv * hd, dtype=torch.float16, device=dev)
    dv = torch.empty(n, nkv * hd, dtype=torch.float16, device=dev)
    ws = torch.empty(meta.bwd_bytes, dtype=torch.uint8, device=dev) if meta.bwd_bytes else None
    _lib.launch(dev, _lib.lib().dk_attn_span_bwd, "dk_attn_span_bwd", qkv.data_ptr(), out.data_ptr(),
                lse.data_ptr(), dout.data_ptr(), meta.spans.data_ptr(), meta.items_bwd.data_ptr(),
                meta.items_bwd.shape[0], meta.joins_bwd.data_ptr(), meta.joins_bwd.shape[0],
                meta.n_units, n, nq, nkv, hd, delta.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                dv.data_ptr(), _lib.ptr(ws), meta.bwd_bytes)
    return dq, dk, dv


def warmup_specs(nq, nkv, hd):
    """Nothing to warm up: the kernels are compiled ahead of time into libdk.so."""
    return []
