"""CPU checks of the attention over part of the keys: the oracle against autograd and differences, the
plans (k_attn.window_meta, prefix_meta) against the definition of what sees what, and refusals before
any launch."""

import ctypes

import numpy as np
import pytest
import torch

from decentrik_prime_amd import _lib, k_attn
from oracle import attn

NQ, NKV, HD = 4, 2, 128
WINDOWS = [([1], 1, 0), ([5, 0, 3], 1, 0), ([40], 7, 3), ([17, 64, 1, 30], 16, 0), ([50, 9], 8, 60),
           ([33, 70], 1 << 70, 4), ([90], 1, 1), ([0], 4, 4), ([30], 5, 1 << 70)]
GROUPS = [[(5, [1])], [(0, [1])], [(0, [7, 3])], [(12, [])], [(12, [0, 0])], [(30, [4, 0, 9, 1]), (0, [6]),
          (1, [1, 1, 1])], [(64, [64, 64])], []]


def _visible_from_spans(spans):
    """The pairs a plan's spans name, once as seen by each query and once as seen from each key."""
    s = np.asarray(spans, np.int64)
    m, n = np.arange(len(s))[:, None], np.arange(len(s))[None]
    as_query = ((n >= s[:, :1]) & (n < s[:, 1:2]) & (n <= m)) | ((n >= s[:, 2:3]) & (n <= m))
    as_key = (m >= n) & (m < s[None, :, 3])
    return as_query, as_key


@pytest.mark.parametrize("lens,window,sinks", WINDOWS)
def test_window_plan_names_the_visible_pairs(lens, window, sinks):
    meta = k_attn.window_meta(lens, window, sinks, NQ, NKV, "cpu")
    want = attn.window_visible(lens, window, sinks)
    for got in _visible_from_spans(meta.spans):
        np.testing.assert_array_equal(got, want)
    np.testing.assert_array_equal(meta.positions, np.concatenate([np.arange(n) for n in lens]))


@pytest.mark.parametrize("groups", GROUPS)
def test_prefix_plan_names_the_visible_pairs(groups):
    meta = k_attn.prefix_meta(groups, NQ, NKV, "cpu")
    want = attn.prefix_visible(groups)
    for got in _visible_from_spans(meta.spans):
        np.testing.assert_array_equal(got, want)
    pos = [np.concatenate([np.arange(p)] + [p + np.arange(a) for a in ans]) for p, ans in groups]
    np.testing.assert_array_equal(meta.positions, np.concatenate(pos) if pos else [])


def test_oracle_gradients_against_autograd_and_differences():
    lens, window, sinks = [9, 1, 20], 5, 2
    vis = attn.window_visible(lens, window, sinks)
    rng = np.random.default_rng(0)
    n = sum(lens)
    qkv = rng.standard_normal((n, (NQ + 2 * NKV) * HD)) * 0.5
    dout = rng.standard_normal((n, NQ * HD))
    out, lse, dq, dk, dv = attn.span_attention(qkv, vis, NQ, NKV, HD, dout)
    t = torch.from_numpy(qkv).requires_grad_(True)
    x = t.view(n, NQ + 2 * NKV, HD).transpose(0, 1)
    k, v = (x[i:i + NKV].repeat_interleave(NQ // NKV, 0) for i in (NQ, NQ + NKV))
    ref = torch.nn.functional.scaled_dot_product_attention(x[:NQ], k, v, torch.from_numpy(vis))
    ref = ref.transpose(0, 1).reshape(n, -1)
    ref.backward(torch.from_numpy(dout))
    # 64-bit sums of at most 128 x 20 terms of size 1: 2560 x 2^-53
    np.testing.assert_allclose(out, ref.detach().numpy(), rtol=1e-11, atol=1e-12)
    np.testing.assert_allclose(np.concatenate([dq, dk, dv], 1), t.grad.numpy(), rtol=1e-10, atol=1e-11)
    step = rng.standard_normal(qkv.shape)
    step /= np.linalg.norm(step)
    h = 1e-4   # error of a central difference: h^2 / 6 of the third derivative, about 1e-8 here
    f = [(attn.span_attention(qkv + e * step, vis, NQ, NKV, HD)[0] * dout).sum() for e in (h, -h)]
    want = (np.concatenate([dq, dk, dv], 1) * step).sum()
    assert abs((f[0] - f[1]) / (2 * h) - want) < 1e-6 * max(1.0, abs(want))
    full = attn.span_attention(qkv, attn.window_visible(lens, 100, 0), NQ, NKV, HD)
    for a, b in zip(full, attn.attention_fwd(qkv, lens, NQ, NKV, HD)):
        np.testing.assert_allclose(a, b, rtol=1e-12, atol=1e-12)


def test_plan_refusals():
    for lens, window, sinks, nq, nkv in (([4], 0, 0, 4, 2), ([4], 2, -1, 4, 2), ([-1], 2, 0, 4, 2),
                                         ([4], 2, 0, 4, 3), ([4], 2, 0, 4, 0), ([4], 2, 0, 0, 1)):
        with pytest.raises(ValueError):
            k_attn.window_meta(lens, window, sinks, nq, nkv, "cpu")
    for groups in ([(-1, [2])], [(3, [2, -2])]):
        with pytest.raises(ValueError):
            k_attn.prefix_meta(groups, 4, 2, "cpu")


def test_plan_refuses_keys_out_of_reach(monkeypatch):
    monkeypatch.setattr(k_attn, "_REACH", 65 * 2 * HD * (NQ + 2 * NKV))
    with pytest.raises(ValueError):
        k_attn.window_meta([300], 100, 3, NQ, NKV, "cpu")


def test_call_refusals_before_any_launch():
    meta = k_attn.window_meta([5, 7], 4, 1, NQ, NKV, "cpu")
    qkv = torch.zeros(12, (NQ + 2 * NKV) * HD, dtype=torch.float16)
    for call in (lambda: k_attn.span_attention_forward(qkv, meta, NQ, NKV, HD),            # not on a GPU
                 lambda: k_attn.span_attention_forward(qkv, meta, NQ, NKV, 64),            # head size
                 lambda: k_attn.span_attention_forward(qkv, meta, 2, 2, HD)):              # other heads
        with pytest.raises(ValueError):
            call()


def _pairs_of_items(meta, rows_seen):
    """Walks a plan's items as the kernel does and counts, per stacked row, the keys it visits."""
    gin, s = meta.nq // meta.nkv, np.asarray(meta.spans, np.int64)
    count = np.zeros((meta.nkv, gin, meta.n_tokens, meta.n_tokens), np.int64)
    for it in np.asarray(meta.items, np.int64):
        t0, phase, rows, g, a0, na, b0, nk, f0, f1, f2, tb, te, slot = it[:14]
        assert 1 <= rows <= 128 and 0 <= phase < gin and 0 <= tb < te <= -(-nk // 64)
        j = np.arange(64 * tb, min(64 * te, nk))
        key = np.where(j < na, a0 + j, b0 + j - na)
        full = (j // 64 < f0) | ((j // 64 >= f1) & (j // 64 < f2))
        for i in range(rows):
            m, e = t0 + (phase + i) // gin, (phase + i) % gin
            seen = (j <= m - b0 + na) & (m < s[key, 3])
            assert na % 64 == 0 or (b0 - a0 - na + 64) * 2 * HD * (meta.nq + 2 * meta.nkv) < k_attn._REACH
            assert not (full & ~seen).any(), "a tile named full holds a masked key"
            count[g, e, m, key[seen]] += 1
            rows_seen[g * gin + e, m] += slot < 0 or tb == 0
    return count


@pytest.mark.parametrize("nq,nkv", [(4, 2), (5, 1), (3, 3)])
@pytest.mark.parametrize("near", [False, True])
def test_items_visit_every_visible_pair_once(monkeypatch, nq, nkv, near):
    """near: as if two runs of keys 63 rows apart were too far from each other for one tile."""
    if near:
        monkeypatch.setattr(k_attn, "_REACH", 127 * 2 * HD * (nq + 2 * nkv))
    for make, spec in ([(attn.window_visible, w) for w in WINDOWS + [([300, 41], 100, 3), ([260], 30, 90)]] +
                       [(attn.prefix_visible, (g,)) for g in GROUPS + [[(200, [40, 3, 70]), (9, [150])]]]):
        build = k_attn.window_meta if make is attn.window_visible else k_attn.prefix_meta
        meta = build(*spec, nq, nkv, "cpu")
        rows = np.zeros((nq, meta.n_tokens), np.int64)
        count = _pairs_of_items(meta, rows)
        assert (rows == 1).all()
        assert (count == make(*spec)[None, None]).all()


def test_split_items_cover_the_walks():
    meta = k_attn.window_meta([700, 20], 400, 4, 12, 2, "cpu")
    blocks = k_attn._query_blocks((np.array([0, 700]), np.array([700, 720])), np.asarray(meta.spans, np.int64), 12, 2)
    for most in (1, 2, 3, 100):
        items, joins, slots = k_attn._split_items(blocks, blocks[:, 12], most)
        assert (items[:, 12] - items[:, 11]).max() <= most and (items[:, 12] > items[:, 11]).all()
        assert sorted(x for x in items[:, 13] if x >= 0) == list(range(slots))
        for t0, phase, rows, g, first, cnt, keys, _ in joins:
            assert keys == 0
            own = items[(items[:, 13] >= first) & (items[:, 13] < first + cnt)]
            own = own[np.argsort(own[:, 13])]
            assert len(own) == cnt > 1 and (own[:, [0, 1, 2, 3]] == [t0, phase, rows, g]).all()
            assert own[0, 11] == 0 and (own[1:, 11] == own[:-1, 12]).all()
            assert own[-1, 12] == -(-own[-1, 7] // 64)


@pytest.mark.parametrize("nq,nkv", [(4, 2), (3, 1)])
def test_key_items_visit_every_visible_pair_once(nq, nkv):
    gin = nq // nkv
    for make, spec in ([(attn.window_visible, w) for w in WINDOWS + [([300, 41], 100, 3), ([260], 30, 90)]] +
                       [(attn.prefix_visible, (g,)) for g in GROUPS + [[(200, [40, 3, 70]), (9, [150])]]]):
        build = k_attn.window_meta if make is attn.window_visible else k_attn.prefix_meta
        meta = build(*spec, nq, nkv, "cpu")
        s = np.asarray(meta.spans, np.int64)
        count = np.zeros((nq, meta.n_tokens, meta.n_tokens), np.int64)
        units, rows = set(), np.zeros((nq, meta.n_tokens), np.int64)
        for it in np.asarray(meta.items_bwd, np.int64):
            t0, phase, n, g, qend = it[:5]
            tb, te, slot, kind = it[11:15]
            if slot >= 0:
                own = set(range(slot, slot + (2 if kind else 1)))
                assert not units & own
                units |= own
            if not kind:
                for i in range(n if tb == 0 else 0):
                    rows[g * gin + (phase + i) % gin, t0 + (phase + i) // gin] += 1
                continue
            assert n <= (128 if kind == 1 else 32)
            per_head = -(-(qend - t0) // 64)
            assert 0 <= tb < te <= gin * per_head
            for t in range(tb, te):
                q0 = t0 + 64 * (t % per_head)
                q = np.arange(q0, min(q0 + 64, qend))[:, None]
                k = np.arange(t0, t0 + n)[None]
                count[g * gin + t // per_head, q, k] += (q >= k) & (q < s[k, 3])
        assert (rows == 1).all() and len(units) == meta.n_units
        assert (count == make(*spec)[None]).all()


def test_c_entry_refusals_before_any_launch():
    lib, p, odd = _lib.lib(), ctypes.c_void_p(256), ctypes.c_void_p(8)

    def fwd(qkv=p, spans=p, items=p, n_items=1, joins=p, n_joins=0, n_slots=0, n=4, nq=4, nkv=2, hd=128,
            out=p, lse=p, ws=None, nbytes=0):
        return lib.dk_attn_span_fwd(qkv, spans, items, n_items, joins, n_joins, n_slots, n, nq, nkv, hd, out,
                                    lse, ws, nbytes, None)

    def bwd(qkv=p, out=p, lse=p, dout=p, spans=p, items=p, n_items=1, joins=p, n_joins=0, n_units=0, n=4, nq=4,
            nkv=2, hd=128, delta=p, dq=p, dk=p, dv=p, ws=None, nbytes=0):
        return lib.dk_attn_span_bwd(qkv, out, lse, dout, spans, items, n_items, joins, n_joins, n_units, n, nq,
                                    nkv, hd, delta, dq, dk, dv, ws, nbytes, None)
    both = [dict(hd=64), dict(nq=3), dict(nkv=0), dict(nq=0), dict(nq=65536, nkv=1), dict(n=-1),
            dict(n=1 << 31), dict(qkv=None), dict(spans=None), dict(items=None), dict(n_items=-1),
            dict(n_joins=-1), dict(n_joins=1, joins=None), dict(out=None), dict(lse=None),
            dict(n_items=1 << 30), dict(n_joins=1 << 30)]
    for call, more in ((fwd, [dict(n_slots=-1)]),
                       (bwd, [dict(n_units=-1)] + [{k: None} for k in ("dout", "delta", "dq", "dk", "dv")])):
        for bad in both + more:
            assert call(**bad) == _lib.DK_ERR_INVALID, bad
        for k in ("qkv", "spans", "out") + (("dout", "dq", "dk", "dv") if call is bwd else ()):
            assert call(**{k: odd}) == _lib.DK_ERR_ALIGN, k
        assert call(ws=odd) == _lib.DK_ERR_ALIGN
        assert call(n=0, qkv=None, spans=None, items=None, out=None, lse=None) == 0
    for slots in (1, 3):
        need = lib.dk_attn_span_workspace(slots)
        assert need == slots * (128 * 128 + 256) * 4
        assert fwd(n_slots=slots) == fwd(n_slots=slots, ws=p, nbytes=need - 1) == _lib.DK_ERR_WORKSPACE
        need = lib.dk_attn_span_bwd_workspace(slots)
        assert need == slots * 128 * 128 * 4
        assert bwd(n_units=slots) == bwd(n_units=slots, ws=p, nbytes=need - 1) == _lib.DK_ERR_WORKSPACE
    assert lib.dk_attn_span_workspace(0) == lib.dk_attn_span_bwd_workspace(0) == 0


@pytest.mark.parametrize("nq,nkv", [(12, 2), (2, 2), (300, 2)])
@pytest.mark.parametrize("near", [False, True])
def test_tiles_that_every_row_sees_are_named_full(monkeypatch, nq, nkv, near):
    """A tile of 64 keys that all rows of a block see whole runs without a mask: none is missed, whether
    the block's keys are two runs or have grown together (a prompt with its first or only answer, a window
    that meets the sinks)."""
    if near:
        monkeypatch.setattr(k_attn, "_REACH", 127 * 2 * HD * (nq + 2 * nkv))
    gin = nq // nkv
    metas = [k_attn.prefix_meta(g, nq, nkv, "cpu") for g in (
        [(500, [200])], [(64, [64])], [(63, [1])], [(300, [1, 200, 70])], [(0, [150]), (200, [130])])]
    metas += [k_attn.window_meta(*w, nq, nkv, "cpu") for w in (
        ([700], 200, 130), ([700], 100, 600), ([300, 90], 64, 64), ([400], 1000, 0), ([400], 130, 4))]
    for meta in metas:
        s = np.asarray(meta.spans, np.int64)
        named = 0
        for it in np.asarray(meta.items, np.int64):
            t0, phase, rows, g, a0, na, b0, nk, f0, f1, f2 = it[:11]
            m = t0 + (phase + np.arange(rows))[:, None] // gin
            j = np.arange(nk // 64 * 64)
            key = np.where(j < na, a0 + j, b0 + j - na)
            seen = ((j <= m - b0 + na) & (m < s[key, 3])).all(0).reshape(-1, 64).all(1)
            t = np.arange(nk // 64)
            np.testing.assert_array_equal((t < f0) | ((t >= f1) & (t < f2)), seen)
            named += int(seen.sum())
        assert named or meta.n_tokens < 128


def test_plan_refuses_more_items_than_a_launch_takes(monkeypatch):
    """A plan that is built can be run in both directions: what the launches do not take is refused here."""
    meta = k_attn.window_meta([700, 1, 1], 90, 3, NQ, NKV, "cpu")
    most = max(len(meta.items), len(meta.items_bwd))
    assert len(meta.items_bwd) > len(meta.items)
    assert k_attn.MAX_SPAN_ITEMS <= (1 << 31) // 256 and k_attn.MAX_SPAN_JOINS <= (1 << 31) // 1024
    for limit in (most - 1, len(meta.items) - 1):
        monkeypatch.setattr(k_attn, "MAX_SPAN_ITEMS", limit)
        with pytest.raises(ValueError):
            k_attn.window_meta([700, 1, 1], 90, 3, NQ, NKV, "cpu")
    monkeypatch.setattr(k_attn, "MAX_SPAN_ITEMS", most)
    k_attn.window_meta([700, 1, 1], 90, 3, NQ, NKV, "cpu")
    monkeypatch.setattr(k_attn, "_fwd_tiles", lambda blocks: 1)
    monkeypatch.setattr(k_attn, "MAX_SPAN_ITEMS", 1 << 20)
    joins = len(k_attn.window_meta([700], 400, 3, NQ, NKV, "cpu").joins)
    monkeypatch.setattr(k_attn, "MAX_SPAN_JOINS", joins - 1)
    with pytest.raises(ValueError):
        k_attn.window_meta([700], 400, 3, NQ, NKV, "cpu")
