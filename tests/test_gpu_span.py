"""GPU parity of the attention over part of the keys (a sliding window with sinks; answers behind a
shared prompt), forward and backward, against the definition in 64 bits."""

import math

import numpy as np
import pytest

from tests.helpers import log

pytestmark = pytest.mark.gpu
HD = 128


@pytest.fixture(scope="module")
def torch():
    import torch as t
    return t


def _meta(spec, nq, nkv):
    from decentrik_prime_amd import k_attn
    if spec[0] == "window":
        return k_attn.window_meta(spec[1], spec[2], spec[3], nq, nkv, "cuda")
    return k_attn.prefix_meta(spec[1], nq, nkv, "cuda")


def _visible(spec):
    from oracle import attn
    return attn.window_visible(*spec[1:]) if spec[0] == "window" else attn.prefix_visible(spec[1])


def _inputs(torch, n, nq, nkv, seed, scale=0.8):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    qkv = (torch.randn(n, (nq + 2 * nkv) * HD, device="cuda", generator=g) * scale).half()
    return qkv, torch.randn(n, nq * HD, device="cuda", generator=g).half()


def _run(qkv, dout, meta, nq, nkv):
    from decentrik_prime_amd import k_attn
    out, lse = k_attn.span_attention_forward(qkv, meta, nq, nkv, HD)
    return (out, lse) + k_attn.span_attention_backward(qkv, out, lse, dout, meta, nq, nkv, HD)


def _near(got, want, lim, what):
    over = (got.double() - want).abs() - lim
    assert bool((over <= 0).all()), f"{what}: {int((~(over <= 0)).sum())} of {over.numel()} outside, " \
                                    f"worst by {float(over.max()):.3g}"


def _check(torch, spec, nq, nkv, qkv, dout, got):
    """Every output against the formulas, with what the roundings may move it by: P and dS are rounded
    to fp16 (half a step, 2^-11 of the value, 2^-25 below the normal range), the scores' fp32 sums move
    P by at most HD 2^-24 of the products' magnitudes and the fp32 sums over the keys by less than
    2^-12 (together under 2^-10 of the magnitudes summed), and the result itself is rounded to fp16
    (2^-11; 2^-25 below the normal range).  delta is taken from the returned out, off by what out is, and
    moves dS by that times P."""
    vis = torch.from_numpy(_visible(spec)).cuda()
    n, gin, sm = qkv.shape[0], nq // nkv, HD ** -0.5
    x = qkv.double().view(n, nq + 2 * nkv, HD)
    out, lse, dq, dk, dv = (t.view(n, -1, HD) if t.dtype == torch.float16 else t for t in got)
    wk, wv, lk, lv = (torch.zeros(n, nkv, HD, dtype=torch.float64, device="cuda") for _ in range(4))
    for h in range(nq):
        g = h // gin
        q, k, v = x[:, h], x[:, nq + g], x[:, nq + nkv + g]
        do = dout.view(n, nq, HD)[:, h].double()
        sc = torch.where(vis, sm * (q @ k.t()), -float("inf"))
        p = torch.softmax(sc, 1)
        dl = ((p @ v) * do).sum(1, keepdim=True)
        ds = p * (do @ v.t() - dl)
        off = ((2.0 ** -10 * (p @ v.abs()) + 2.0 ** -11 * (p @ v).abs() + 2.0 ** -24) * do.abs()).sum(1, keepdim=True)
        what = f"{spec}, {nq}/{nkv} heads, head {h}: "
        _near(out[:, h], p @ v, 2.0 ** -10 * (p @ v.abs()) + 2.0 ** -11 * (p @ v).abs() + 2.0 ** -24,
              what + "out")
        _near(lse[h], torch.logsumexp(sc, 1) / math.log(2.0), 2.0 ** -12, what + "lse")
        eds = torch.where(vis, 2.0 ** -10 * ds.abs() + 2.0 ** -25 + HD * 2.0 ** -23 * p * (
            do.abs() @ v.abs().t() + ((p @ v) * do).abs().sum(1, keepdim=True)) + off * p, 0.0)
        want = sm * (ds @ k)
        _near(dq[:, h], want, sm * (eds @ k.abs()) + 2.0 ** -11 * want.abs() + 2.0 ** -24, what + "dq")
        wk[:, g] += sm * (ds.t() @ q)
        lk[:, g] += sm * (eds.t() @ q.abs())
        wv[:, g] += p.t() @ do
        lv[:, g] += torch.where(vis, 2.0 ** -10 * p + 2.0 ** -25, 0.0).t() @ do.abs()
    _near(dk, wk, lk + 2.0 ** -11 * wk.abs() + 2.0 ** -24, f"{spec}, {nq}/{nkv} heads: dk")
    _near(dv, wv, lv + 2.0 ** -11 * wv.abs() + 2.0 ** -24, f"{spec}, {nq}/{nkv} heads: dv")


CASES = [
    # one token; an empty sequence; a window of one token with and without sinks
    (("window", [1], 1, 0), 12, 2), (("window", [0, 3, 0, 1], 1, 0), 4, 2), (("window", [70, 200], 1, 1), 2, 1),
    # windows that end inside, at and past a tile; sinks fewer and more than a tile, than the window,
    # than the sequence; blocks whose window meets the sinks
    (("window", [300, 65], 64, 4), 12, 2), (("window", [513], 63, 0), 3, 3), (("window", [700, 1, 129], 200, 70), 4, 2),
    (("window", [400], 17, 130), 8, 1), (("window", [257, 30], 5, 600), 6, 2), (("window", [260, 128], 4096, 3), 5, 1),
    (("window", [1300], 256, 4), 14, 2), (("window", [2100], 1000, 64), 2, 2),
    # a prompt alone, answers alone, one-token answers, answers that share a tile, empty ones
    (("prefix", [(130, [])]), 4, 2), (("prefix", [(0, [5, 130])]), 12, 2), (("prefix", [(1, [1])]), 4, 1),
    (("prefix", [(200, [1] * 70)]), 12, 2), (("prefix", [(64, [64, 128, 0, 63])]), 2, 2),
    (("prefix", [(500, [40, 3, 77, 0, 190]), (0, [33]), (17, [1, 300]), (300, [0])]), 28, 4),
    (("prefix", [(1100, [150, 90, 301])]), 6, 1), (("prefix", [(77, [9] * 33)]), 8, 8),
    # a group of more heads than a block has rows
    (("window", [70, 3], 5, 2), 130, 1), (("prefix", [(40, [1, 7, 30])]), 400, 2),
]


@pytest.mark.parametrize("spec,nq,nkv", CASES)
def test_against_the_definition(torch, spec, nq, nkv):
    log(f"span attention fwd+bwd, {spec}, {nq}/{nkv} heads")
    meta = _meta(spec, nq, nkv)
    qkv, dout = _inputs(torch, meta.n_tokens, nq, nkv, seed=meta.n_tokens + nq)
    _check(torch, spec, nq, nkv, qkv, dout, _run(qkv, dout, meta, nq, nkv))


@pytest.mark.parametrize("spec,nq,nkv", [CASES[i] for i in (0, 3, 5, 6, 7, 9, 11, 14, 15, 16)])
@pytest.mark.parametrize("tiles", [1, 3])
def test_walks_cut_in_parts(torch, monkeypatch, spec, nq, nkv, tiles):
    """The same with every walk cut after a few tiles and joined again."""
    from decentrik_prime_amd import k_attn
    log(f"span attention fwd+bwd in walks of {tiles} tiles, {spec}, {nq}/{nkv} heads")
    monkeypatch.setattr(k_attn, "_fwd_tiles", lambda blocks: tiles)
    monkeypatch.setattr(k_attn, "_bwd_cost", lambda cost: 4 * tiles)
    meta = _meta(spec, nq, nkv)
    assert meta.n_units > 0 or meta.n_tokens < 64
    qkv, dout = _inputs(torch, meta.n_tokens, nq, nkv, seed=meta.n_tokens + nq)
    _check(torch, spec, nq, nkv, qkv, dout, _run(qkv, dout, meta, nq, nkv))


@pytest.mark.parametrize("spec,nq,nkv", [CASES[i] for i in (3, 5, 6, 9, 15)])
def test_runs_of_keys_too_far_apart_for_a_tile(torch, monkeypatch, spec, nq, nkv):
    """The plan of sinks or prompts more than 4 GiB of rows before the window or answer."""
    from decentrik_prime_amd import k_attn
    monkeypatch.setattr(k_attn, "_REACH", 127 * 2 * HD * (nq + 2 * nkv))
    meta = _meta(spec, nq, nkv)
    assert bool(((meta.items[:, 5] > 0) & (meta.items[:, 5] % 64 == 0)).any())
    qkv, dout = _inputs(torch, meta.n_tokens, nq, nkv, seed=meta.n_tokens + nq)
    _check(torch, spec, nq, nkv, qkv, dout, _run(qkv, dout, meta, nq, nkv))


def test_table_entries_that_name_no_rows_are_skipped(torch):
    """Items and joins outside the batch, the heads or the workspace change nothing."""
    nq, nkv = 4, 2
    meta = _meta(("window", [300, 77], 90, 3), nq, nkv)
    n = meta.n_tokens
    qkv, dout = _inputs(torch, n, nq, nkv, seed=9)
    want = _run(qkv, dout, meta, nq, nkv)

    def entries(width, rows):
        return torch.tensor([r + [0] * (width - len(r)) for r in rows], dtype=torch.int32, device="cuda")
    query = [[n, 0, 1, 0, 0, 0, 0, 1, 0, 0, 0, 0, 1, -1], [-1, 0, 1, 0, 0, 0, 0, 1, 0, 0, 0, 0, 1, -1],
             [n - 1, 0, 128, 0, 0, 0, 0, 5, 0, 0, 0, 0, 1, -1], [0, 0, 1, nkv, 0, 0, 0, 1, 0, 0, 0, 0, 1, -1],
             [0, 2, 1, 0, 0, 0, 0, 1, 0, 0, 0, 0, 1, -1], [0, 0, 0, 0, 0, 0, 0, 1, 0, 0, 0, 0, 1, -1],
             [0, 0, 1, 0, 0, 0, n, 1, 0, 0, 0, 0, 1, -1], [0, 0, 1, 0, 0, 0, 0, 1, 0, 0, 0, 0, 2, -1],
             [0, 0, 1, 0, 0, 0, 0, 1, 0, 0, 0, 1, 1, -1], [0, 0, 1, 0, 0, 0, 0, 1, 0, 0, 0, 0, 1, 1 << 20],
             [0, 0, 1, 0, -1, 3, 5, 4, 0, 0, 0, 0, 1, -1], [0, 0, 1, 0, 4, 3, 5, 4, 0, 0, 0, 0, 1, -1]]
    keys = [[n, 0, 1, 0, n + 1, 0, 0, 0, 0, 0, 0, 0, 1, -1], [0, 0, 129, 0, n, 0, 0, 0, 0, 0, 0, 0, 1, -1],
            [0, 0, 1, 0, n + 1, 0, 0, 0, 0, 0, 0, 0, 1, -1], [5, 0, 1, 0, 5, 0, 0, 0, 0, 0, 0, 0, 1, -1],
            [0, 0, 1, 0, 64, 0, 0, 0, 0, 0, 0, 0, 3, -1], [0, 0, 1, 0, 64, 0, 0, 0, 0, 0, 0, 0, 1, 1 << 20],
            [0, 0, 1, -1, 64, 0, 0, 0, 0, 0, 0, 0, 1, -1]]
    joins = [[n, 0, 1, 0, 0, 1], [0, 0, 1, 0, -1, 1], [0, 0, 1, 0, 0, 1 << 20], [0, 2, 1, 0, 0, 1],
             [0, 0, 129, 0, 0, 1], [0, 0, 1, 0, 1 << 20, 1], [0, 0, 1, 0, 0, 0]]
    bad = entries(16, query + [k + [kind] for k in keys + [[0, 0, 33, 0, n, 0, 0, 0, 0, 0, 0, 0, 1, -1]]
                               for kind in ((2,) if k[2] == 33 else (1, 2))])
    meta.items = torch.cat([entries(16, query), meta.items])
    meta.joins = torch.cat([meta.joins, entries(8, joins)])
    meta.items_bwd = torch.cat([bad, meta.items_bwd])
    meta.joins_bwd = torch.cat([meta.joins_bwd, entries(8, joins + [j[:6] + [1] for j in joins if j[1] == 0])])
    for a, b in zip(_run(qkv, dout, meta, nq, nkv), want):
        assert torch.equal(a, b)


def test_many_short_sequences(torch):
    """2^17 sequences of one token and 2^14 answers of one token to a prompt of one: a key or two each."""
    from decentrik_prime_amd import k_attn
    nq, nkv = 4, 1
    n = 1 << 17
    log(f"span attention, {n} one-token sequences")
    qkv, dout = _inputs(torch, n, nq, nkv, seed=4)
    got = _run(qkv, dout, k_attn.window_meta([1] * n, 5, 1, nq, nkv, "cuda"), nq, nkv)
    v = qkv[:, (nq + 1) * HD:]
    assert torch.equal(got[0].view(n, nq, HD), v[:, None].expand(-1, nq, -1))
    # dS = P (dO V - out dO): 0 but for the two sums' rounding, HD 2^-24 of their magnitudes, twice
    mag = (dout.view(n, nq, HD).double().abs() * v[:, None].double().abs()).sum(2)
    lim = 2 * HD * 2.0 ** -24 * mag.amax() * 8 * HD ** -0.5 * nq
    assert float(got[2].abs().max()) <= lim and float(got[3].abs().max()) <= lim
    want = dout.view(n, nq, HD).double().sum(1)
    _near(got[4], want, 2.0 ** -10 * dout.view(n, nq, HD).double().abs().sum(1) + 2.0 ** -11 * want.abs() + 2.0 ** -24, "dv")
    answers = 1 << 14
    meta = k_attn.prefix_meta([(1, [1] * answers)], nq, nkv, "cuda")
    qkv, dout = qkv[:answers + 1].contiguous(), dout[:answers + 1].contiguous()
    got = _run(qkv, dout, meta, nq, nkv)
    x = qkv.double().view(-1, nq + 2, HD)
    k, v = x[:, nq], x[:, nq + 1]
    s = torch.stack([(x[1:, :nq] @ k[0]), (x[1:, :nq] * k[1:, None]).sum(2)], 2) * HD ** -0.5
    p = torch.softmax(s, 2)
    want = p[..., :1] * v[0] + p[..., 1:] * v[1:, None]
    mag = p[..., :1] * v[0].abs() + p[..., 1:] * v[1:, None].abs()
    _near(got[0].view(-1, nq, HD)[1:], want, 2.0 ** -10 * mag + 2.0 ** -11 * want.abs() + 2.0 ** -24, "out")
    do = dout.double().view(-1, nq, HD)
    want = do[0].sum(0) + (p[..., :1] * do[1:]).sum((0, 1))
    mag = do[0].abs().sum(0) + (p[..., :1] * do[1:].abs()).sum((0, 1))
    _near(got[4][0], want, 2.0 ** -10 * mag + 2.0 ** -11 * want.abs(), "dv of the prompt")


def test_rows_past_four_gigabytes(torch):
    """A sequence of 4.6 GB of qkv rows: sinks further from the window than a 32-bit offset reaches.  The
    last rows and keys against their own definition."""
    from decentrik_prime_amd import k_attn
    nq, nkv, window, sinks = 12, 2, 70, 5
    n = (1 << 32) // (2 * HD * (nq + 2 * nkv)) + 70000
    log(f"span attention, one sequence of {n} tokens")
    meta = k_attn.window_meta([n], window, sinks, nq, nkv, "cuda")
    far = meta.items[:, 5] == 64
    assert bool(far.any()) and bool((meta.items[:, 5] == sinks).any())
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    qkv = torch.randn(n, (nq + 2 * nkv) * HD, device="cuda", generator=g, dtype=torch.float16)
    dout = torch.randn(n, nq * HD, device="cuda", generator=g, dtype=torch.float16)
    out, lse, dq, dk, dv = _run(qkv, dout, meta, nq, nkv)
    for t in (out, lse, dq, dk, dv):
        assert bool(torch.isfinite(t[-1000:] if t.shape[0] == n else t).all())
    # the last 300 queries, and the last 300 - window keys, whose queries are all among them
    rows = 300
    m = torch.arange(n - rows, n, device="cuda")
    cols = torch.cat([torch.arange(sinks, device="cuda"), torch.arange(n - rows - window, n, device="cuda")])
    vis = (cols[None] <= m[:, None]) & ((m[:, None] - cols[None] < window) | (cols[None] < sinks))
    x = qkv[cols].double().view(cols.numel(), nq + 2 * nkv, HD)
    q_all = qkv[m].double().view(rows, nq + 2 * nkv, HD)
    gk, gv = (torch.zeros(cols.numel(), nkv, HD, dtype=torch.float64, device="cuda") for _ in range(2))
    lk, lv = torch.zeros_like(gk), torch.zeros_like(gk)
    sm = HD ** -0.5
    for h in range(nq):
        kv = h // (nq // nkv)
        q, k, v = q_all[:, h], x[:, nq + kv], x[:, nq + nkv + kv]
        do = dout[m].double().view(rows, nq, HD)[:, h]
        sc = torch.where(vis, sm * (q @ k.t()), -float("inf"))
        p = torch.softmax(sc, 1)
        o = p @ v
        dl = (o * do).sum(1, keepdim=True)
        ds = p * (do @ v.t() - dl)
        # the tolerances of _check
        lo = 2.0 ** -10 * (p @ v.abs()) + 2.0 ** -11 * o.abs() + 2.0 ** -24
        eds = torch.where(vis, 2.0 ** -10 * ds.abs() + 2.0 ** -25 + HD * 2.0 ** -23 * p * (
            do.abs() @ v.abs().t() + (o * do).abs().sum(1, keepdim=True)) +
            (lo * do.abs()).sum(1, keepdim=True) * p, 0.0)
        _near(out[m].view(rows, nq, HD)[:, h], o, lo, f"head {h}: out")
        _near(lse[h, m], torch.logsumexp(sc, 1) / math.log(2.0), 2.0 ** -12, f"head {h}: lse")
        want = sm * (ds @ k)
        _near(dq[m].view(rows, nq, HD)[:, h], want, sm * (eds @ k.abs()) + 2.0 ** -11 * want.abs() + 2.0 ** -24,
              f"head {h}: dq")
        gk[:, kv] += sm * (ds.t() @ q)
        lk[:, kv] += sm * (eds.t() @ q.abs())
        gv[:, kv] += p.t() @ do
        lv[:, kv] += torch.where(vis, 2.0 ** -10 * p + 2.0 ** -25, 0.0).t() @ do.abs()
    own = slice(sinks + window + window, None)
    for t, w, lim, what in ((dk, gk, lk, "dk"), (dv, gv, lv, "dv")):
        t = t[cols[own]].view(-1, nkv, HD)
        _near(t, w[own], lim[own] + 2.0 ** -11 * w[own].abs() + 2.0 ** -24, what)


def test_no_tokens(torch):
    for spec in (("window", [], 4, 1), ("prefix", [(0, [0])])):
        meta = _meta(spec, 4, 2)
        qkv, dout = _inputs(torch, 0, 4, 2, seed=0)
        for t in _run(qkv, dout, meta, 4, 2):
            assert t.numel() == 0


def test_growing_scores(torch):
    """Scores that grow along the keys by far more than a rescaling's threshold per tile, and a window
    that leaves the largest behind."""
    for spec in (("window", [700], 150, 3), ("prefix", [(300, [100, 200])])):
        log(f"span attention, growing scores, {spec}")
        meta = _meta(spec, 2, 1)
        qkv, dout = _inputs(torch, meta.n_tokens, 2, 1, seed=5, scale=0.3)
        qkv[:, 2 * HD] = (0.25 * meta.positions).half()
        qkv[:, 0] = qkv[:, HD] = 8.0
        got = _run(qkv, dout, meta, 2, 1)
        vis = torch.from_numpy(_visible(spec)).cuda()
        sc = torch.where(vis, HD ** -0.5 * (qkv[:, :HD].double() @ qkv[:, 2 * HD:3 * HD].double().t()),
                         -float("inf"))
        p = torch.softmax(sc, 1)
        v = qkv[:, 3 * HD:].double()
        # scores up to 130 in sums of fp32: P off by 2^-24 HD 2^7, below 2^-10
        _near(got[0][:, :HD], p @ v, 2.0 ** -9 * (p @ v.abs()) + 2.0 ** -24, "out")


def test_wide_window_is_plain_causal_attention(torch):
    from decentrik_prime_amd import k_attn
    lens, nq, nkv = [1, 37, 64, 500], 12, 2
    qkv, dout = _inputs(torch, sum(lens), nq, nkv, seed=3)
    plain = k_attn.attention_forward(qkv, k_attn.meta_for(lens, "cuda"), nq, nkv, HD)
    for spec in (("window", lens, 500, 0), ("window", lens, 1, 500), ("prefix", [(0, lens)])):
        got = k_attn.span_attention_forward(qkv, _meta(spec, nq, nkv), nq, nkv, HD)
        # both within 2^-10 of the same sums of |p v| (at most max |v|, 4) and one fp16 rounding
        assert float((got[0].double() - plain[0].double()).abs().max()) < 2 * 4 * (2.0 ** -10 + 2.0 ** -11)
        assert float((got[1] - plain[1]).abs().max()) < 2.0 ** -11


@pytest.mark.parametrize("spec,bad,clean", [
    # an answer's token, which nothing of the other answers or the prompt sees
    (("prefix", [(40, [20, 30, 9]), (3, [50])]), 65, lambda m: (m < 65) | (m >= 90)),
    # a token in the middle of a sequence: earlier queries, and those past the window
    (("window", [20, 300, 40], 50, 4), 20 + 100, lambda m: (m < 120) | (m >= 170)),
    # a token of the second sequence's end
    (("window", [20, 300, 40], 50, 4), 319, lambda m: m != 319)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), 65504.0])
@pytest.mark.parametrize("cut", [False, True])
def test_unseen_rows_have_no_influence(torch, monkeypatch, spec, bad, clean, value, cut):
    """A row full of NaN, infinities or the type's largest value changes nothing for the queries that do
    not see it, nor for the keys that it does not see."""
    nq, nkv = 4, 2
    log(f"span attention with {value} in row {bad}, {spec}")
    if cut:
        from decentrik_prime_amd import k_attn
        monkeypatch.setattr(k_attn, "_fwd_tiles", lambda blocks: 2)
        monkeypatch.setattr(k_attn, "_bwd_cost", lambda cost: 8)
    meta = _meta(spec, nq, nkv)
    n = meta.n_tokens
    qkv, dout = _inputs(torch, n, nq, nkv, seed=11)
    want = _run(qkv, dout, meta, nq, nkv)
    bad_qkv, bad_dout = qkv.clone(), dout.clone()
    bad_qkv[bad], bad_dout[bad] = value, value
    got = _run(bad_qkv, bad_dout, meta, nq, nkv)
    vis = torch.from_numpy(_visible(spec)).cuda()
    m = torch.arange(n, device="cuda")
    same = ~vis[:, bad]                         # queries that do not see the row
    assert bool((same == clean(m)).all())
    # keys whose queries (and what those saw) are all untouched
    keys = ~vis[~same].any(0)
    for t, w, rows, what in ((got[0], want[0], same, "out"), (got[1].t(), want[1].t(), same, "lse"),
                             (got[2], want[2], same, "dq"), (got[3], want[3], keys, "dk"),
                             (got[4], want[4], keys, "dv")):
        assert bool(torch.isfinite(t[rows].float()).all()), what
        # the same sums, in another order at the most where a row was recomputed on its own
        lim = 2.0 ** -9 * w[rows].double().abs() + 2.0 ** -9
        assert bool(((t[rows].double() - w[rows].double()).abs() <= lim).all()), what
    if value != value:
        assert bool(torch.isnan(got[0][~same]).all())


@pytest.mark.parametrize("what", ["all", "q", "k", "v", "dout"])
def test_batches_of_nothing_but_nan(torch, what):
    """What the definition makes of a batch whose queries, keys, values or gradients are all NaN."""
    nq, nkv = 4, 2
    meta = _meta(("window", [700, 41], 100, 4), nq, nkv)
    qkv, dout = _inputs(torch, meta.n_tokens, nq, nkv, seed=12)
    cols = {"q": slice(0, nq * HD), "k": slice(nq * HD, (nq + nkv) * HD), "v": slice((nq + nkv) * HD, None)}
    for name, c in cols.items():
        if what in (name, "all"):
            qkv[:, c] = float("nan")
    if what in ("dout", "all"):
        dout[:] = float("nan")
    out, lse, dq, dk, dv = _run(qkv, dout, meta, nq, nkv)
    nan = lambda t: bool(torch.isnan(t).all())     # noqa: E731
    finite = lambda t: bool(torch.isfinite(t).all())   # noqa: E731
    assert finite(out) if what == "dout" else nan(out)
    assert nan(lse) if what in ("q", "k", "all") else finite(lse)
    assert nan(dq) and nan(dk)
    assert finite(dv) if what == "v" else nan(dv)


@pytest.mark.parametrize("spec,up,down", [(("window", [30, 400], 90, 3), 130, 141),
                                          (("prefix", [(150, [40, 5, 77])]), 20, 155)])
@pytest.mark.parametrize("cut", [False, True])
def test_infinities_reach_who_sees_them(torch, monkeypatch, spec, up, down, cut):
    """+inf in one value row and one gradient row and -inf in another of each: +inf, -inf, or NaN where
    both come together, in out and dv; lse as without them."""
    nq, nkv = 4, 2
    if cut:
        from decentrik_prime_amd import k_attn
        monkeypatch.setattr(k_attn, "_fwd_tiles", lambda blocks: 1)
        monkeypatch.setattr(k_attn, "_bwd_cost", lambda cost: 4)
    log(f"span attention with infinities in rows {up} and {down}, {spec}")
    meta = _meta(spec, nq, nkv)
    qkv, dout = _inputs(torch, meta.n_tokens, nq, nkv, seed=14)
    want = _run(qkv, dout, meta, nq, nkv)
    vis = torch.from_numpy(_visible(spec)).cuda()
    bad = qkv.clone()
    for row, x in ((up, float("inf")), (down, -float("inf"))):
        bad[row, (nq + nkv) * HD:] = x
        dout[row] = x
    out, lse, _, _, dv = _run(bad, dout, meta, nq, nkv)
    # the same sums, in another order at the most
    assert bool(((lse - want[1]).abs() <= 2.0 ** -12).all())
    for t, sees_up, sees_down, what in ((out, vis[:, up], vis[:, down], "out"),
                                        (dv, vis[up], vis[down], "dv")):
        t = t.float()
        for rows, f in ((sees_up & ~sees_down, torch.isposinf), (sees_down & ~sees_up, torch.isneginf),
                        (sees_up & sees_down, torch.isnan), (~sees_up & ~sees_down, torch.isfinite)):
            assert bool(f(t[rows]).all()), what
        assert bool((sees_up ^ sees_down).any()) and bool((sees_up & sees_down).any())


def test_one_column_of_nan_stays_one(torch):
    """A NaN in one column of every value row and of every gradient row: that column of out and of dv."""
    nq, nkv = 4, 2
    meta = _meta(("prefix", [(70, [30, 45])]), nq, nkv)
    qkv, dout = _inputs(torch, meta.n_tokens, nq, nkv, seed=13)
    want = _run(qkv, dout, meta, nq, nkv)
    qkv.view(-1, nq + 2 * nkv, HD)[:, nq + nkv:, 5] = float("nan")
    dout.view(-1, nq, HD)[:, :, 7] = float("nan")
    got = _run(qkv, dout, meta, nq, nkv)
    for t, w, heads, col in ((got[0], want[0], nq, 5), (got[4], want[4], nkv, 7)):
        t, w = t.view(-1, heads, HD), w.view(-1, heads, HD)
        assert bool(torch.isnan(t[..., col]).all())
        rest = [c for c in range(HD) if c != col]
        # the same sums, in another order at the most
        assert bool(((t - w)[..., rest].double().abs() <= 2.0 ** -9 * w[..., rest].double().abs() + 2.0 ** -9).all())


def test_repeats_and_streams(torch):
    """The same bits on every call, on a stream of its own, and on two streams at once."""
    nq, nkv = 12, 2
    for spec in (("window", [1500, 200], 300, 4), ("prefix", [(900, [40, 60, 300])])):
        meta = _meta(spec, nq, nkv)
        qkv, dout = _inputs(torch, meta.n_tokens, nq, nkv, seed=1)
        want = _run(qkv, dout, meta, nq, nkv)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for st in streams:
            with torch.cuda.stream(st):
                got.append(_run(qkv, dout, meta, nq, nkv))
        torch.cuda.synchronize()
        for res in got:
            for a, b in zip(res, want):
                assert torch.equal(a, b)


def test_captured_and_replayed(torch):
    """A training step's two calls in one graph, replayed on new inputs with eager calls between."""
    nq, nkv = 12, 2
    for spec in (("window", [900, 1, 333], 200, 4), ("prefix", [(700, [1, 40, 260])])):
        meta = _meta(spec, nq, nkv)
        qkv, dout = _inputs(torch, meta.n_tokens, nq, nkv, seed=2)
        _run(qkv, dout, meta, nq, nkv)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = _run(qkv, dout, meta, nq, nkv)
        for r in range(3):
            a, b = _inputs(torch, meta.n_tokens, nq, nkv, seed=30 + r)
            qkv.copy_(a)
            dout.copy_(b)
            want = _run(qkv, dout, meta, nq, nkv)
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(res, want):
                assert torch.equal(x, y), f"replay {r}"


def test_refusals(torch):
    from decentrik_prime_amd import k_attn
    nq, nkv = 4, 2
    meta = k_attn.window_meta([5, 7], 4, 1, nq, nkv, "cuda")
    qkv, dout = _inputs(torch, 12, nq, nkv, seed=0)
    out, lse = k_attn.span_attention_forward(qkv, meta, nq, nkv, HD)
    on_cpu = k_attn.window_meta([5, 7], 4, 1, nq, nkv, "cpu")
    for call in (lambda: k_attn.span_attention_forward(qkv[:11], meta, nq, nkv, HD),
                 lambda: k_attn.span_attention_forward(qkv.float(), meta, nq, nkv, HD),
                 lambda: k_attn.span_attention_forward(qkv.t().contiguous().t(), meta, nq, nkv, HD),
                 lambda: k_attn.span_attention_forward(qkv, meta, nq, nkv, 64),
                 lambda: k_attn.span_attention_forward(qkv, meta, 2, 2, HD),
                 lambda: k_attn.span_attention_forward(qkv, on_cpu, nq, nkv, HD),
                 lambda: k_attn.span_attention_backward(qkv, out, lse.half(), dout, meta, nq, nkv, HD),
                 lambda: k_attn.span_attention_backward(qkv, out, lse.t(), dout, meta, nq, nkv, HD),
                 lambda: k_attn.span_attention_backward(qkv, out, lse, dout[:, :HD], meta, nq, nkv, HD),
                 lambda: k_attn.span_attention_backward(qkv, out.cpu(), lse, dout, meta, nq, nkv, HD)):
        with pytest.raises(ValueError):
            call()


def test_a_layer_around_it(torch):
    """The QKV epilogue, the attention and their backwards together, as a layer runs them: the rotary
    positions of the plan, dk and dv already summed (gin = 1)."""
    from decentrik_prime_amd import k_attn, k_rope
    from decentrik_prime_amd.model import rope_tables
    nq, nkv = 12, 2
    spec = ("prefix", [(90, [20, 33]), (0, [40])])
    meta = _meta(spec, nq, nkv)
    n = meta.n_tokens
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    raw = (torch.randn(n, (nq + 2 * nkv) * HD, device="cuda", generator=g) * 0.8).half()
    dout = torch.randn(n, nq * HD, device="cuda", generator=g).half()
    cos, sin = rope_tables(int(meta.positions.max()) + 1)
    zq = torch.zeros(n, nq * HD, dtype=torch.float16, device="cuda")
    qkv = raw.clone()
    k_rope.qkv_epilogue_forward(qkv, zq, zq[:, :nkv * HD].contiguous(), meta.positions, cos, sin, 0.0,
                                nq, nkv, HD)
    out, lse, dq, dk, dv = got = _run(qkv, dout, meta, nq, nkv)
    _check(torch, spec, nq, nkv, qkv, dout, got)
    dqkv = torch.empty_like(qkv)
    k_rope.qkv_epilogue_backward(dq, dk, dv, meta.positions, cos, sin, dqkv, nq, nkv, HD, 1)
    # the transposed rotation of dq and dk (fp32 products, one fp16 rounding), dv as it is
    c, s = cos[meta.positions.long()][:, None], sin[meta.positions.long()][:, None]
    for lo, d in ((0, dq), (nq, dk)):
        heads = d.view(n, -1, HD).double()
        a, b = heads[..., :HD // 2], heads[..., HD // 2:]
        c1, s1 = c[..., :HD // 2].double(), s[..., :HD // 2].double()
        want = torch.cat([a * c1 + b * s1, b * c1 - a * s1], 2)
        have = dqkv.view(n, -1, HD)[:, lo:lo + heads.shape[1]]
        _near(have, want, 2.0 ** -11 * want.abs() + 2.0 ** -22 * (heads.abs().amax(2, keepdim=True)) + 2.0 ** -24,
              "rotated gradient")
    assert torch.equal(dqkv[:, (nq + nkv) * HD:], dv)


def test_more_rows_than_the_delta_launch_has_lanes(torch):
    """2^20 and some (token, query head) rows of a backward: delta's workgroups go round more than once.
    One-token sequences, whose dv is the sum of the group's gradients and whose dq and dk are 0, behind
    some longer ones that repeat at the end."""
    nq, nkv = 48, 2
    ones = (1 << 20) // nq
    lens = [70, 3] + [1] * ones + [70, 3]
    log(f"span attention, {sum(lens) * nq} rows")
    meta = _meta(("window", lens, 40, 2), nq, nkv)
    qkv, dout = _inputs(torch, meta.n_tokens, nq, nkv, seed=21)
    qkv[-73:], dout[-73:] = qkv[:73], dout[:73]
    got = _run(qkv, dout, meta, nq, nkv)
    for t in (got[0], got[2], got[3], got[4]):
        assert torch.equal(t[:73], t[-73:])
    v, do = qkv[73:-73, (nq + nkv) * HD:].double().view(-1, nkv, HD), dout[73:-73].double().view(-1, nkv, nq // nkv, HD)
    # dS = P (dO V - out dO): 0 but for the two sums' rounding, HD 2^-24 of their magnitudes, twice
    mag = float((do.abs() * v[:, :, None].abs()).sum(3).amax())
    lim = 2 * HD * 2.0 ** -24 * mag * 8 * HD ** -0.5 * (nq // nkv)
    assert float(got[2][73:-73].abs().max()) <= lim and float(got[3][73:-73].abs().max()) <= lim
    _near(got[4][73:-73].view(-1, nkv, HD), do.sum(2),
          2.0 ** -10 * do.abs().sum(2) + 2.0 ** -11 * do.sum(2).abs() + 2.0 ** -24, "dv")


@pytest.mark.parametrize("cut", [False, True])
def test_values_at_the_types_maximum(torch, monkeypatch, cut):
    """Values of +-65504 throughout, most of a row's weight on one key of a later tile: their mean is
    +-65504 whatever the weights, and no rounding of the weights (2^-11 of each, where 2^-12 more would
    round to infinity) takes it past the type's range."""
    from decentrik_prime_amd import k_attn
    nq, nkv, n = 4, 1, 300
    if cut:
        monkeypatch.setattr(k_attn, "_fwd_tiles", lambda blocks: 2)
    meta = _meta(("window", [n], n, 0), nq, nkv)
    g = torch.Generator(device="cuda")
    g.manual_seed(15)
    qkv = torch.zeros(n, (nq + 2 * nkv) * HD, device="cuda", dtype=torch.float16)
    x = qkv.view(n, nq + 2 * nkv, HD)
    x[:, :nq, 0] = 4 + 4 * torch.rand(n, nq, device="cuda", generator=g).half()
    x[:, nq, 0] = -200.0
    x[0, nq, 0], x[100, nq, 0] = 0.0, 6.0      # 3 to 6 in log2 units above key 0's score
    x[:, nq + 1] = 65504.0
    x[:, nq + 1, ::3] = -65504.0
    out, lse = k_attn.span_attention_forward(qkv, meta, nq, nkv, HD)
    assert bool(torch.isfinite(lse).all()) and bool(torch.isfinite(out).all())
    _near(out.view(n, nq, HD), x[:, nq + 1:].double().expand(n, nq, HD), (2.0 ** -10 + 2.0 ** -11) * 65504, "out")


@pytest.mark.parametrize("spec,cut", [(("window", [5000], 4500, 1), False), (("window", [5000], 4500, 1), True),
                                      (("prefix", [(4500, [300, 1])]), False)])
def test_small_weights_behind_a_sink(torch, monkeypatch, spec, cut):
    """A first key that takes nearly all of every row's weight and has no value of its own, as sinks do:
    the output is what the thousands of others, 2^-18 to 2^-26 each, add up to.  P's rounding to fp16 is
    2^-11 of the value, or 2^-32 of the row's largest below its normal range (the tiles hold P times 2^7)."""
    from decentrik_prime_amd import k_attn
    nq, nkv = 4, 2
    if cut:
        monkeypatch.setattr(k_attn, "_fwd_tiles", lambda blocks: 9)
    log(f"span attention, small weights behind a sink, {spec}")
    meta = _meta(spec, nq, nkv)
    n = meta.n_tokens
    qkv, _ = _inputs(torch, n, nq, nkv, seed=16, scale=0.1)
    x = qkv.view(n, nq + 2 * nkv, HD)
    x[:, :nq, 0] = torch.tensor([6.5, 7.3, 8.1, 9.4], device="cuda").half()
    x[:, nq:nq + nkv, 0] = 0.0
    x[0, nq:nq + nkv, 0] = 21.6
    x[:, nq + nkv:] = 1.0 + x[:, nq + nkv:].abs()
    x[0, nq + nkv:] = 0.0
    out, lse = k_attn.span_attention_forward(qkv, meta, nq, nkv, HD)
    vis = torch.from_numpy(_visible(spec)).cuda()
    for h in range(nq):
        q, k, v = (x[:, i].double() for i in (h, nq + h // 2, nq + nkv + h // 2))
        sc = torch.where(vis, HD ** -0.5 * (q @ k.t()), -float("inf"))
        p = torch.softmax(sc, 1)
        floor = 2.0 ** -32 * p.amax(1, keepdim=True) * (vis.double() @ v.abs())
        # the scores' fp32 sums: up to 26 in log2 units, P off by 2^-24 HD 2^5 at the most, below 2^-11
        _near(out.view(n, nq, HD)[:, h], p @ v, 1.5 * 2.0 ** -10 * (p @ v) + floor + 2.0 ** -25, f"head {h}: out")
        _near(lse[h], torch.logsumexp(sc, 1) / math.log(2.0), 2.0 ** -12, f"head {h}: lse")


def _spread(x, y=1.0):
    """The square of a 2-norm's expected error when every value of x is rounded to fp16 on its own (at most
    half a step, 2^-11, evenly spread: a third of the square) and weighted by y."""
    return 2.0 ** -22 / 3 * (x.square() * y).sum()


def _check_norms(torch, spec, nq, nkv, qkv, dout, got, rows=None, what=""):
    """dq, dk and dv of the tokens `rows` (all) against the formulas in 2-norms: P and dS rounded to fp16 on
    their own, delta from the returned out (rounded, and P before it), and the results' own rounding, which
    is taken as it is.  Half as much again is allowed for what the sums' errors, 2^-24 a term, and the
    chance of the rest may add."""
    vis = torch.from_numpy(_visible(spec)).cuda()
    n, gin, sm = qkv.shape[0], nq // nkv, HD ** -0.5
    rows = slice(0, n) if rows is None else rows
    x = qkv.double().view(n, nq + 2 * nkv, HD)
    dq, dk, dv = (t.double().view(n, -1, HD)[rows] for t in got[2:])
    wk, wv = (torch.zeros(n, nkv, HD, dtype=torch.float64, device="cuda") for _ in range(2))
    ek, ev = [0.0] * nkv, [0.0] * nkv
    part = torch.zeros(n, 1, dtype=torch.float64, device="cuda")
    part[rows] = 1.0

    def near(got, want, spread, name):
        own = (want.half().double() - want).square().sum()
        err, lim = float((got - want).norm()), 1.5 * float((own + spread).sqrt())
        log(f"{what}{name}: 2-norm error {err / float(want.norm()):.3g}, at most {lim / float(want.norm()):.3g}")
        assert err <= lim, f"{what}{name}: {err:.3g} > {lim:.3g}"
    for h in range(nq):
        g = h // gin
        q, k, v = x[:, h], x[:, nq + g], x[:, nq + nkv + g]
        do = dout.view(n, nq, HD)[:, h].double()
        p = torch.softmax(torch.where(vis, sm * (q @ k.t()), -float("inf")), 1)
        o = p @ v
        ds = p * (do @ v.t() - (o * do).sum(1, keepdim=True))
        # delta's error per row: out's rounding and, before it, P's
        off = 2.0 ** -22 / 3 * ((o.square() + p.square() @ v.square()) * do.square()).sum(1, keepdim=True)
        near(dq[:, h], (sm * (ds @ k))[rows], sm * sm * (_spread(ds * part, k.square().sum(1)) +
                                                         (off * part * (p @ k).square()).sum()), f"head {h} dq")
        wk[:, g] += sm * (ds.t() @ q)
        wv[:, g] += p.t() @ do
        ek[g] += sm * sm * (_spread(ds * part.t(), q.square().sum(1, keepdim=True)) +
                            ((p * part.t()).square() * off * q.square().sum(1, keepdim=True)).sum())
        ev[g] += _spread(p * part.t(), do.square().sum(1, keepdim=True))
    for g in range(nkv):
        near(dk[:, g], wk[rows, g], ek[g], f"KV head {g} dk")
        near(dv[:, g], wv[rows, g], ev[g], f"KV head {g} dv")


@pytest.mark.parametrize("size", [300.0, 1.0, 1e-3, 1e-4])
@pytest.mark.parametrize("spec,cut", [(("window", [2500], 1500, 4), False), (("window", [2500, 40], 2500, 0), True),
                                      (("prefix", [(1400, [300, 1, 200]), (0, [90])]), False)])
def test_gradients_of_any_size(torch, monkeypatch, spec, cut, size):
    """Walks of some thousand keys with dout large and small: dS is P times dout's size, and the roundings
    stay those of each value whatever that is."""
    from decentrik_prime_amd import k_attn
    nq, nkv = 4, 2
    if cut:
        monkeypatch.setattr(k_attn, "_fwd_tiles", lambda blocks: 7)
        monkeypatch.setattr(k_attn, "_bwd_cost", lambda cost: 60)
    log(f"span attention, dout ~ {size}, {spec}")
    meta = _meta(spec, nq, nkv)
    qkv, dout = _inputs(torch, meta.n_tokens, nq, nkv, seed=17)
    dout = (dout.float() * size).half()
    _check_norms(torch, spec, nq, nkv, qkv, dout, _run(qkv, dout, meta, nq, nkv))


@pytest.mark.parametrize("cut", [False, True])
def test_gradients_of_several_sizes_in_a_batch(torch, monkeypatch, cut):
    """Small gradients beside large ones of another sequence or group, and behind a prompt whose own are 0
    (a loss over the answers alone)."""
    from decentrik_prime_amd import k_attn
    nq, nkv = 4, 2
    if cut:
        monkeypatch.setattr(k_attn, "_bwd_cost", lambda cost: 40)
    for spec, small in ((("window", [70, 1100, 300], 900, 4), slice(70, 1170)),
                        (("prefix", [(300, [20, 7]), (900, [200, 150])]), slice(327, 1577))):
        log(f"span attention, gradients of several sizes, {spec}")
        meta = _meta(spec, nq, nkv)
        qkv, dout = _inputs(torch, meta.n_tokens, nq, nkv, seed=18)
        sizes = torch.full((meta.n_tokens, 1), 200.0, device="cuda")
        sizes[small] = 1e-4
        if spec[0] == "prefix":
            sizes[327:327 + 900] = 0.0
        dout = (dout.float() * sizes).half()
        _check_norms(torch, spec, nq, nkv, qkv, dout, _run(qkv, dout, meta, nq, nkv), small, "the small ones, ")


def test_even_weights_over_many_keys(torch):
    """Queries of 0 give every key that they see the same weight, 2^-16 at the end: out and dv are plain
    sums."""
    nq, nkv, n = 1, 1, 70000
    log(f"span attention, even weights over {n} keys")
    meta = _meta(("window", [n], n, 0), nq, nkv)
    qkv, dout = _inputs(torch, n, nq, nkv, seed=19)
    qkv[:, :HD] = 0.0
    qkv[:, 2 * HD:] += 1.0
    out, lse, _, dk, dv = _run(qkv, dout, meta, nq, nkv)
    m = torch.arange(1, n + 1, device="cuda", dtype=torch.float64)[:, None]
    v, do = qkv[:, 2 * HD:].double(), dout.double()
    want = v.cumsum(0) / m
    # P is 2^7 exactly: the sums' errors of fp32 (n 2^-24 of the magnitudes at the most) and out's rounding
    _near(out, want, n * 2.0 ** -24 * v.abs().cumsum(0) / m + 2.0 ** -11 * want.abs() + 2.0 ** -25, "out")
    _near(lse[0], m[:, 0].log2(), 2.0 ** -12, "lse")
    assert float(dk.abs().max()) == 0.0
    sums = (do / m).flip(0).cumsum(0).flip(0)
    spread = 2.0 ** -22 / 3 * ((do / m).square().flip(0).cumsum(0)).sum()
    own = (sums.half().double() - sums).square().sum()
    err, lim = float((dv.double() - sums).norm()), 1.5 * float((own + spread).sqrt())
    assert err <= lim, f"dv: {err:.3g} > {lim:.3g}"


@pytest.mark.parametrize("scale", [1e-2, 1e3])
def test_gradients_with_values_of_any_size(torch, scale):
    """Small and very large values: dS in fp16 overflows for the largest, and those rows are redone."""
    nq, nkv = 4, 2
    spec = ("window", [1200], 1000, 4)
    log(f"span attention, values ~ {scale}")
    meta = _meta(spec, nq, nkv)
    qkv, dout = _inputs(torch, meta.n_tokens, nq, nkv, seed=20)
    qkv[:, (nq + nkv) * HD:] *= scale
    dout = (dout.float() * (1.0 if scale < 1 else 1e-2)).half()
    _check_norms(torch, spec, nq, nkv, qkv, dout, _run(qkv, dout, meta, nq, nkv))


def test_sinks_of_rows_past_four_gigabytes(torch):
    """dk and dv of the sinks of a sequence of 4.6 GB of qkv rows: the walks whose query tiles lie furthest
    from their first, cut and joined, each value a sum over six million rows.  P from the returned lse and
    delta from the returned out; the other rows' results are at least finite."""
    nq, nkv, window, sinks = 12, 2, 70, 5
    gin, sm = nq // nkv, HD ** -0.5
    n = (1 << 32) // (2 * HD * (nq + 2 * nkv)) + 70000
    log(f"span attention, sinks of one sequence of {n} tokens")
    meta = _meta(("window", [n], window, sinks), nq, nkv)
    g = torch.Generator(device="cuda")
    g.manual_seed(23)
    qkv = torch.randn(n, (nq + 2 * nkv) * HD, device="cuda", generator=g, dtype=torch.float16)
    dout = torch.randn(n, nq * HD, device="cuda", generator=g, dtype=torch.float16)
    out, lse, dq, dk, dv = _run(qkv, dout, meta, nq, nkv)
    for t in (out, lse, dq, dk, dv):
        assert bool(torch.isfinite(t).all())
    wk, wv = (torch.zeros(nkv, sinks, HD, dtype=torch.float64, device="cuda") for _ in range(2))
    ek, ev = [0.0] * nkv, [0.0] * nkv
    keys = qkv[:sinks].double().view(sinks, nq + 2 * nkv, HD)
    for m0 in range(0, n, 1 << 15):
        m = torch.arange(m0, min(m0 + (1 << 15), n), device="cuda")
        seen = m[:, None] >= torch.arange(sinks, device="cuda")
        for h in range(nq):
            kv, cols = h // gin, slice(h * HD, (h + 1) * HD)
            q, o, do = (t[m0:m0 + m.numel(), cols].double() for t in (qkv, out, dout))
            p = torch.where(seen, torch.exp2(q @ keys[:, nq + kv].t() * (sm / math.log(2.0)) -
                                             lse[h, m, None].double()), 0.0)
            ds = p * (do @ keys[:, nq + nkv + kv].t() - (o * do).sum(1, keepdim=True))
            wk[kv] += sm * (ds.t() @ q)
            wv[kv] += p.t() @ do
            ek[kv] += sm * sm * _spread(ds, q.square().sum(1, keepdim=True))
            ev[kv] += _spread(p, do.square().sum(1, keepdim=True))
    for t, want, spread, what in ((dk, wk, ek, "dk"), (dv, wv, ev, "dv")):
        for kv in range(nkv):
            got = t[:sinks].view(sinks, nkv, HD)[:, kv].double()
            # the fp32 sums' errors, 2^-24 a step of walks of some thousand steps, are far below the roundings
            own = (want[kv].half().double() - want[kv]).square().sum()
            err, lim = float((got - want[kv]).norm()), 1.5 * float((own + spread[kv]).sqrt())
            log(f"KV head {kv} {what}: {err / float(want[kv].norm()):.3g}, at most {lim / float(want[kv].norm()):.3g}")
            assert err <= lim, what


@pytest.mark.parametrize("cut", [False, True])
def test_growing_scores_forward_and_backward(torch, monkeypatch, cut):
    """test_growing_scores for both heads, lse and the gradients, and with walks cut so that the partials'
    maxima lie far apart: the backward forms P again from lse, at scores up to 190 in log2 units."""
    from decentrik_prime_amd import k_attn
    nq, nkv, sm = 2, 1, HD ** -0.5
    if cut:
        monkeypatch.setattr(k_attn, "_fwd_tiles", lambda blocks: 2)
        monkeypatch.setattr(k_attn, "_bwd_cost", lambda cost: 8)
    for spec in (("window", [700], 150, 3), ("prefix", [(300, [100, 200])])):
        log(f"span attention, growing scores forward and backward, {spec}, cut {cut}")
        meta = _meta(spec, nq, nkv)
        n = meta.n_tokens
        qkv, dout = _inputs(torch, n, nq, nkv, seed=5, scale=0.3)
        qkv[:, 2 * HD] = (0.25 * meta.positions).half()
        qkv[:, 0] = qkv[:, HD] = 8.0
        out, lse, dq, dk, dv = _run(qkv, dout, meta, nq, nkv)
        vis = torch.from_numpy(_visible(spec)).cuda()
        x = qkv.double().view(n, nq + 2, HD)
        k, v = x[:, 2], x[:, 3]
        wk, wv, lk, lv = (torch.zeros(n, HD, dtype=torch.float64, device="cuda") for _ in range(4))
        # s is off by HD 2^-24 of its 190 at most, lse by 2^-23 of its size and the sum's log2: P, relative,
        # by HD 2^-24 190 ln 2 < 2^-9.9; with its rounding, 2^-11, and the sums', below 2^-9
        rel = 2.0 ** -9
        for h in range(nq):
            q, do = x[:, h], dout.view(n, nq, HD)[:, h].double()
            sc = torch.where(vis, sm * (q @ k.t()), -float("inf"))
            assert float(sc[vis].max()) / math.log(2.0) < 190
            p = torch.softmax(sc, 1)
            o = p @ v
            lo = rel * (p @ v.abs()) + 2.0 ** -11 * o.abs() + 2.0 ** -24
            _near(out.view(n, nq, HD)[:, h], o, lo, f"head {h}: out")
            _near(lse[h], torch.logsumexp(sc, 1) / math.log(2.0), HD * 2.0 ** -24 * 190 + 2.0 ** -12, f"head {h}: lse")
            dl = (o * do).sum(1, keepdim=True)
            ds = p * (do @ v.t() - dl)
            eds = torch.where(vis, 1.5 * rel * ds.abs() + 2.0 ** -30 + HD * 2.0 ** -23 * p * (
                do.abs() @ v.abs().t() + (o * do).abs().sum(1, keepdim=True)) +
                (lo * do.abs()).sum(1, keepdim=True) * p + 2.0 ** -19 * dl.abs() * p, 0.0)
            want = sm * (ds @ k)
            _near(dq.view(n, nq, HD)[:, h], want, sm * (eds @ k.abs()) + 2.0 ** -11 * want.abs() + 2.0 ** -24,
                  f"head {h}: dq")
            wk += sm * (ds.t() @ q)
            lk += sm * (eds.t() @ q.abs())
            wv += p.t() @ do
            lv += torch.where(vis, rel * p + 2.0 ** -30, 0.0).t() @ do.abs()
        _near(dk, wk, lk + 2.0 ** -11 * wk.abs() + 2.0 ** -24, "dk")
        _near(dv, wv, lv + 2.0 ** -11 * wv.abs() + 2.0 ** -24, "dv")


@pytest.mark.parametrize("spec", [("window", [700, 1, 90], 1, 0), ("window", [1] * 300, 5, 2), ("prefix", [(0, [1] * 200)])])
@pytest.mark.parametrize("size", [1.0, 0.1])
def test_rows_that_see_one_key_have_no_gradient(torch, spec, size):
    """P = 1 and out = v, so dS = dout . v - delta is 0 but for the rounding of two fp32 sums of HD products:
    sqrt(HD) half steps of partial sums at random in each, together 2^-21 of the products' norm."""
    nq, nkv = 8, 2
    log(f"span attention, one key to a row, dout ~ {size}, {spec[0]}")
    meta = _meta(spec, nq, nkv)
    n, gin = meta.n_tokens, nq // nkv
    qkv, dout = _inputs(torch, n, nq, nkv, seed=25)
    dout = (dout.float() * size).half()
    out, _, dq, dk, _ = _run(qkv, dout, meta, nq, nkv)
    x, do = qkv.view(n, nq + 2 * nkv, HD).double(), dout.view(n, nq, HD).double()
    k, v = (x[:, i:i + nkv].repeat_interleave(gin, 1) for i in (nq, nq + nkv))
    assert torch.equal(out.view(n, nq, HD).double(), v)
    ds = 2.0 ** -21 * (do * v).norm(dim=2)
    for got, by, what in ((dq, k, "dq"), (dk, x[:, :nq], "dk")):
        err, lim = float(got.double().norm()), float((ds * by.norm(dim=2)).norm()) * HD ** -0.5
        assert err <= lim, f"{what}: {err:.3g} > {lim:.3g}"
