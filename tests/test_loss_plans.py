"""CPU checks of the losses over log-probabilities, the scoring head and gradient clipping: the plans the
kernels walk, and what is refused before any launch."""

import ctypes
import re

import pytest
import torch

from decentrik_prime_amd import _lib, k_grad, k_head, k_loss


def read_plan(meta):
    """(items [n, 8], row_items, entries, pairs, row_pairs) as the kernels read them."""
    raw, first = meta._buffer.numpy(), meta._buffer.data_ptr()

    def part(name, n):
        at = (meta.at[name] - first) // 4
        return raw[at:at + n]
    items = part("items", 8 * meta.n_items).reshape(-1, 8)
    row_items = part("row_items", meta.n_rows + 1)
    assert row_items.size == meta.n_rows + 1
    if meta.n_pairs is None:
        return items, row_items, None, None, None
    return (items, row_items, part("entries", 4 * meta.n_pairs).reshape(-1, 2),
            part("pairs", 2 * meta.n_pairs).reshape(-1, 2), part("row_pairs", meta.n_rows + 1))


@pytest.mark.parametrize("lens", [[0], [1], [0, 0, 5, 0], [511, 512, 513, 1, 0, 1025], [32768, 32769, 100000],
                                  list(range(70)), [1 << 30] * 5 + [3]])
def test_items_cover_every_token_once(lens):
    meta = k_loss.row_meta(lens, "cpu")
    items, row_items = read_plan(meta)[:2]
    assert meta.n_rows == len(lens) and meta.n_tokens == sum(lens)
    assert meta.n_filled == sum(n > 0 for n in lens)
    assert row_items[0] == 0 and row_items[-1] == meta.n_items == len(items)
    start = 0
    for r, n in enumerate(lens):
        mine = items[row_items[r]:row_items[r + 1]]
        assert 1 <= len(mine) <= k_loss.ROW_ITEMS
        at = start
        for place, (lo, hi, count, row, size, of, which, _) in enumerate(mine.tolist()):
            assert (row, size, of, which) == (r, n, len(mine), place)
            assert (hi << 32) + (lo & 0xffffffff) == at
            assert count > 0 or n == 0
            at += count
        start += n
        assert at == start
    assert meta.at["items"] % 16 == 0


@pytest.mark.parametrize("lens, pairs", [([3, 4], [(0, 1)]), ([3, 4, 0], [(0, 1), (2, 1), (1, 0), (0, 1)]),
                                         ([1] * 9, [(i, j) for i in range(9) for j in range(9)])])
def test_every_row_names_its_pairs(lens, pairs):
    meta = k_loss.row_meta(lens, "cpu", pairs=pairs)
    _, _, entries, kept, row_pairs = read_plan(meta)
    assert meta.at["entries"] % 8 == 0 and meta.at["pairs"] % 8 == 0
    assert list(map(tuple, kept.tolist())) == pairs
    want = {r: sorted([(b, i + 1) for i, (a, b) in enumerate(pairs) if a == r] +
                      [(a, -i - 1) for i, (a, b) in enumerate(pairs) if b == r]) for r in range(len(lens))}
    for r in range(len(lens)):
        assert sorted(map(tuple, entries[row_pairs[r]:row_pairs[r + 1]].tolist())) == want[r]


def test_plans_refuse_what_they_cannot_hold():
    for lens in ([], [-1], [3, -2], [(1 << 30) + 1], [1.5], ["a"], [[1, 2]], 3, [True]):
        with pytest.raises(ValueError):
            k_loss.row_meta(lens, "cpu")
    for pairs in ([], [(0, 2)], [(-1, 0)], [(0.0, 1.0)], [0, 1], [(0, 1, 1, 0)], [(0, 1), (1,)]):
        with pytest.raises(ValueError):
            k_loss.row_meta([1, 2], "cpu", pairs=pairs)


def test_plans_hold_what_a_launch_takes():
    """2^25 items: their waves stay below 2^32 work items."""
    import numpy as np
    for lens in (np.zeros((1 << 25) + 1, np.int8), np.full((1 << 19) + 1, 1 << 30)):
        with pytest.raises(ValueError, match="items"):
            k_loss.row_meta(lens, "cpu")
    lib = _lib.lib()
    for entry, struct_name, packed in ((lib.dk_policy_loss, "dk_policy_args", _lib.POLICY_ARGS),
                                       (lib.dk_preference_loss, "dk_preference_args", _lib.PREFERENCE_ARGS)):
        fields = _fields(struct_name)
        for n, want in ((1 << 25, _lib.DK_ERR_WORKSPACE), ((1 << 25) + 1, _lib.DK_ERR_INVALID)):
            values = {name: 4096 if f == "Q" else 0.25 if f == "d" else 1 for name, f in fields}
            values.update(n_items=n, rows=1 << 20, n_tokens=5, workspace_bytes=0)
            assert entry(packed.pack(*(values[name] for name, _ in fields)), None) == want


def test_losses_refuse_bad_arguments():
    meta = k_loss.row_meta([2, 3], "cpu", pairs=[(0, 1)])
    x, a = torch.zeros(5), torch.zeros(2)
    for kwargs in (dict(clip_low=1.5), dict(clip_low=-0.1), dict(clip_high=-1.0), dict(kl_coef=0.1),
                   dict(kl_coef=float("nan"), ref=x), dict(reduction="mean"), {}):   # {}: not on a GPU
        with pytest.raises(ValueError):
            k_loss.policy_loss(x, x, a, meta, **kwargs)
    for kwargs in (dict(beta=0.0), dict(beta=float("inf")), dict(kind="dpo"), dict(label_smoothing=0.6),
                   dict(label_smoothing=0.1, kind="hinge"), dict(margin=float("inf")), {}):
        with pytest.raises(ValueError):
            k_loss.preference_loss(x, x, meta, **kwargs)
    with pytest.raises(ValueError, match="no pairs"):
        k_loss.preference_loss(x, x, k_loss.row_meta([2, 3], "cpu"))


def test_scoring_head_refuses_bad_arguments():
    y, e, t = torch.zeros(2, 64).half(), torch.zeros(8, 64).half(), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        k_head.token_logprobs(y, e, t)          # not on a GPU
    lib = _lib.lib()
    p = ctypes.c_void_p(4096)

    def call(y=p, ldy=64, total=2, rows=None, n=2, emb=p, vocab=8, d=64, tgt=p, scale=1.0, out=p, ws=p,
             nbytes=1 << 20):
        return lib.dk_head_logprobs(y, ldy, total, rows, n, emb, vocab, d, tgt, scale, out, out, out, ws,
                                    nbytes, None)
    assert lib.dk_head_logprobs_workspace(2, 8, 64) == 2 * 20
    assert lib.dk_head_logprobs_workspace(0, 8, 64) == 0
    for bad in (dict(y=None), dict(ldy=32), dict(ldy=68), dict(total=1), dict(n=-1), dict(emb=None),
                dict(vocab=0), dict(d=32), dict(d=96), dict(d=0), dict(tgt=None), dict(scale=0.0),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(out=None),
                dict(rows=p, total=1 << 25), dict(rows=p, total=0), dict(vocab=1 << 31), dict(n=1 << 31)):
        assert call(**bad) == _lib.DK_ERR_INVALID, bad
    for bad in (dict(y=ctypes.c_void_p(4104)), dict(emb=ctypes.c_void_p(4104)), dict(tgt=ctypes.c_void_p(2)),
                dict(out=ctypes.c_void_p(2)), dict(rows=ctypes.c_void_p(4098))):
        assert call(**bad) == _lib.DK_ERR_ALIGN, bad
    for bad in (dict(ws=None), dict(nbytes=39), dict(ws=ctypes.c_void_p(4104))):
        assert call(**bad) == _lib.DK_ERR_WORKSPACE, bad
    assert call(n=0, y=None, ws=None) == 0


@pytest.mark.parametrize("d, most", [(64, 1 << 25), (1536, (1 << 31) // 1536 + 1), (2048, 1 << 20)])
def test_scoring_head_takes_rows_up_to_32_bits_of_offsets(d, most):
    """The last row's end is what counts: below 2^31 elements with `rows`, within a tile of 256 without."""
    lib, p = _lib.lib(), ctypes.c_void_p(4096)

    def call(total, n=2, ldy=d, rows=p):           # (a workspace of 0 bytes: the next refusal, before any launch)
        return lib.dk_head_logprobs(p, ldy, total, rows, n, p, 8, d, p, 1.0, p, p, p, p, 0, None)
    assert call(most) == _lib.DK_ERR_INVALID
    assert call(most - 1) == _lib.DK_ERR_WORKSPACE
    assert call(2, ldy=(1 << 31) - d) == _lib.DK_ERR_INVALID
    assert call(2, ldy=(1 << 31) - d - 8) == _lib.DK_ERR_WORKSPACE
    assert call(1, ldy=1 << 40) == _lib.DK_ERR_WORKSPACE
    assert call(1 << 62, ldy=1 << 40) == call(1 << 62, n=1 << 20, ldy=1 << 40, rows=None) == _lib.DK_ERR_INVALID
    for n, ldy, fits in ((128, 1 << 24, True), (129, 1 << 24, False), (1000, 1 << 23, True),
                         (1000, (1 << 23) + (1 << 16), False), (2, (1 << 31) - d, False), (1, 1 << 40, True)):
        want = _lib.DK_ERR_WORKSPACE if fits else _lib.DK_ERR_INVALID
        assert call(1 << 20, n, ldy, None) == want, (n, ldy)


def test_scoring_head_takes_many_tokens_in_launches_of_2_to_the_24():
    """Their waves stay below 2^32 work items; the scratch memory is one launch's."""
    need = _lib.lib().dk_head_logprobs_workspace
    one = need(1 << 24, 8, 64)
    assert one >= 20 << 24
    for n in ((1 << 24) + 1, 1 << 26, (1 << 26) + 70, (1 << 30) - 5, 1 << 30):
        assert need(n, 8, 64) == one


def _fields(struct_name):
    """The fields of a struct of dk.h, token arrays as three, and the format of each."""
    text = re.sub(r"/\*.*?\*/", "", open(_lib.HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct_name, struct_name), text, re.S).group(1)
    out = []
    for line in filter(None, (x.strip() for x in body.split(";"))):
        kind, names = re.match(r"((?:const )?\w+\*?) (.*)", line, re.S).groups()
        for name in names.split(","):
            if kind == "dk_token_array":
                out += [(name.strip() + s, f) for s, f in (("", "Q"), ("_stride", "q"), ("_negated", "q"))]
            else:
                out.append((name.strip(), "Q" if kind.endswith("*") else {"int64_t": "q", "double": "d"}[kind]))
    return out


@pytest.mark.parametrize("name, packed", [("dk_policy_args", _lib.POLICY_ARGS),
                                          ("dk_preference_args", _lib.PREFERENCE_ARGS)])
def test_packed_arguments_are_the_headers_structs(name, packed):
    fields = _fields(name)
    assert packed.format == "".join(f for _, f in fields) and packed.size == 8 * len(fields)


def test_loss_entries_refuse_bad_arguments():
    lib = _lib.lib()
    p = 4096

    def call(entry, struct_name, packed, good, bad):
        names = [n for n, _ in _fields(struct_name)]
        assert set(good) <= set(names) and set(bad) <= set(names)
        values = {**{n: p for n in names}, **good, **bad}
        return entry(packed.pack(*(values[n] for n in names)), None)

    def policy(**bad):
        good = dict(n_items=100, rows=2, n_tokens=5, per_token=0, clip_low=0.2, clip_high=0.2, kl_coef=0.1,
                    reduction=0, denominator=2.0, workspace_bytes=1 << 12,
                    **{f"{t}_{k}": v for t in ("logp", "old", "ref") for k, v in (("stride", 1), ("negated", 0))})
        return call(lib.dk_policy_loss, "dk_policy_args", _lib.POLICY_ARGS, good, bad)
    for bad in (dict(items=0), dict(row_items=0), dict(n_items=0), dict(n_items=1), dict(rows=0),
                dict(n_tokens=-1), dict(logp=0), dict(old=0), dict(ref=0), dict(logp_stride=-1),
                dict(ref_stride=1 << 31), dict(advantages=0), dict(clip_low=1.1), dict(clip_low=-0.1),
                dict(clip_high=-0.1), dict(clip_high=float("nan")), dict(kl_coef=float("inf")),
                dict(reduction=3), dict(reduction=-1), dict(denominator=0.0), dict(dlogp=0), dict(stats=0),
                dict(loss=0)):
        assert policy(**bad) == _lib.DK_ERR_INVALID, bad
    assert lib.dk_policy_loss(None, None) == _lib.DK_ERR_INVALID
    assert policy(items=4100) == policy(row_items=4097) == _lib.DK_ERR_ALIGN
    assert lib.dk_policy_loss_workspace(64, 1 << 15) == 0        # one workgroup
    need = lib.dk_policy_loss_workspace(100, 5)
    assert need == lib.dk_policy_loss_workspace(100, 1 << 20) > 0
    for bad in (dict(workspace=0), dict(workspace_bytes=need - 1), dict(workspace=4100)):
        assert policy(**bad) == _lib.DK_ERR_WORKSPACE, bad

    def preference(**bad):
        good = dict(n_items=2, rows=2, n_tokens=5, n_pairs=5000, beta=0.1, kind=0, label_smoothing=0.0,
                    margin=0.0, average=0, workspace_bytes=1 << 16, logp_stride=1, logp_negated=0,
                    ref_stride=1, ref_negated=0)
        return call(lib.dk_preference_loss, "dk_preference_args", _lib.PREFERENCE_ARGS, good, bad)
    for bad in (dict(n_pairs=0), dict(entries=0), dict(pairs=0), dict(row_pairs=0), dict(logp=0),
                dict(ref_stride=-1), dict(beta=0.0), dict(beta=float("nan")), dict(beta=float("inf")),
                dict(kind=3), dict(label_smoothing=0.51), dict(margin=float("nan")), dict(dlogp=0),
                dict(rewards=0), dict(margins=0), dict(loss=0)):
        assert preference(**bad) == _lib.DK_ERR_INVALID, bad
    assert lib.dk_preference_loss(None, None) == _lib.DK_ERR_INVALID
    assert preference(entries=4100) == preference(pairs=4100) == _lib.DK_ERR_ALIGN
    assert lib.dk_preference_loss_workspace(64, 1 << 15, 1024) == 0
    for bad in (dict(workspace=0), dict(workspace_bytes=lib.dk_preference_loss_workspace(2, 5, 5000) - 1)):
        assert preference(**bad) == _lib.DK_ERR_WORKSPACE, bad


def test_clipping_refuses_bad_arguments():
    g = torch.ones(4)
    for grads in ([], [g], [g.long()]):
        with pytest.raises(ValueError):
            k_grad.clip_grads(grads, 1.0)
    for kwargs in (dict(max_norm=0.0), dict(max_norm=float("nan")), dict(max_norm=-1.0),
                   dict(max_norm=1.0, scale=0.0), dict(max_norm=1.0, scale=float("inf"))):
        with pytest.raises(ValueError):
            k_grad.clip_grads([g], **kwargs)
    lib = _lib.lib()

    def call(src, dst, numel, types, max_norm=1.0, scale=1.0, norm=64, ws=4096, nbytes=1 << 16):
        n = len(src)
        arrays = [(ctypes.c_int64 * n)(*src), (ctypes.c_int64 * n)(*dst) if dst else None,
                  (ctypes.c_int64 * n)(*numel), (ctypes.c_int32 * n)(*[t & 15 for t in types]),
                  (ctypes.c_int32 * n)(*[t >> 4 for t in types])]
        return lib.dk_grad_clip(*arrays, n, max_norm, scale, norm, ws, nbytes, None)
    f32, f16 = _lib.DK_TYPE_F32 * 17, _lib.DK_TYPE_F16 * 17
    up = _lib.DK_TYPE_F16 | _lib.DK_TYPE_F32 << 4
    a, b = 1 << 20, 1 << 21
    assert lib.dk_grad_clip_workspace(0) == 0
    for bad in (([], None, [], []), ([a], [a], [-1], [f32]), ([0], [a], [4], [f32]), ([a], [0], [4], [f32]),
                ([a], [a], [4], [0]), ([a], [a], [4], [4 * 17]), ([a], [a], [4], [up]),      # in place, two types
                ([a, a], [a, a], [4, 4], [f32, f32]),                                   # a tensor twice
                ([a, a + 8], [a, a + 8], [4, 4], [f32, f32]),                           # overlapping ones
                ([a, b], [b, b + 64], [4, 4], [f32, f32]),                              # an output over a source
                ([a, b], [a + 4, b], [4, 4], [f32, f32]),                               # shifted in place
                ([a, b], [b + 64, b + 72], [4, 4], [f32, f32])):                        # overlapping outputs
        assert call(*bad) == _lib.DK_ERR_INVALID, bad
    for kwargs in (dict(max_norm=0.0), dict(max_norm=float("nan")), dict(scale=0.0),
                   dict(scale=float("inf")), dict(scale=float("nan")), dict(norm=None)):
        assert call([a], [a], [4], [f32], **kwargs) == _lib.DK_ERR_INVALID, kwargs
    assert call([a + 2], [a + 2], [4], [f32]) == _lib.DK_ERR_ALIGN
    assert call([a + 1], [a + 1], [4], [f16]) == _lib.DK_ERR_ALIGN
    assert call([a], [b + 2], [4], [up]) == _lib.DK_ERR_ALIGN
    for kwargs in (dict(ws=None), dict(nbytes=8), dict(ws=4100)):
        assert call([a], [a], [4], [f32], **kwargs) == _lib.DK_ERR_WORKSPACE, kwargs


def test_dense_tensors():
    x = torch.zeros(4, 6)
    for t, want in ((x, True), (x.t(), True), (x[:, :3], False), (x[::2], False), (x[1:3], True),
                    (torch.zeros(1, 5).expand(3, 5), False), (torch.zeros(2, 3, 4).permute(2, 0, 1), True),
                    (torch.zeros(0, 4), True), (torch.zeros(3, 0)[:, :0], True), (torch.zeros(()), True)):
        assert k_grad._dense(t) is want, (t.shape, t.stride())


def test_row_factors_and_scaling_refuse_bad_arguments():
    g, t = torch.ones(4), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        k_loss.row_factors(g, t, 4)             # not on a GPU
    with pytest.raises(ValueError):
        k_grad.scale_grads([g], torch.ones(()))
    with pytest.raises(ValueError):
        k_grad.scale_grads([], torch.ones(()))
    lib, p = _lib.lib(), 4096

    def factors(dlogp=p, at=p, n=4, out=p, rows=9, unit=p):
        return lib.dk_row_factors(dlogp, at, n, out, rows, unit, None)
    for bad in (dict(dlogp=None), dict(at=None), dict(n=-1), dict(out=None), dict(rows=-1), dict(unit=None)):
        assert factors(**bad) == _lib.DK_ERR_INVALID, bad
    for bad in (dict(dlogp=4098), dict(at=4097), dict(out=4098), dict(unit=4099)):
        assert factors(**bad) == _lib.DK_ERR_ALIGN, bad

    def scale(at, numel, types, factor=p):
        n = len(at)
        return lib.dk_grad_scale((ctypes.c_int64 * n)(*at), (ctypes.c_int64 * n)(*numel),
                                 (ctypes.c_int32 * n)(*types), n, factor, 1.0, None)
    a, f32 = 1 << 20, _lib.DK_TYPE_F32
    for bad in (([], [], []), ([0], [4], [f32]), ([a], [-1], [f32]), ([a], [4], [0]), ([a, a], [4, 4], [f32, f32]),
                ([a, a + 8], [4, 4], [f32, f32]), ([a], [4], [f32], None)):
        assert scale(*bad) == _lib.DK_ERR_INVALID, bad
    for inside in (a, a + 12, a + 1024):                                    # a factor that is scaled itself
        assert scale([a, a + 1024], [4, 4], [f32, f32], inside) == _lib.DK_ERR_INVALID
    assert scale([a + 2], [4], [f32]) == scale([a], [4], [f32], p + 2) == _lib.DK_ERR_ALIGN
