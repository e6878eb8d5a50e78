"""Token log-probabilities of the head (k_head.token_logprobs) against the softmax of the logits in 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24          # half a step of fp32


def definition(y, e, tgt, scale):
    """(logp, entropy, lse, and how far logits summed in fp32 may move each) in 64 bits."""
    y, e = y.double(), e.double()
    x = (y @ e.t()) * scale
    lse = torch.logsumexp(x, 1)
    logq = x - lse[:, None]
    q = logq.exp()
    entropy = -(q * logq).sum(1)
    at = tgt.long().clamp(0, e.shape[0] - 1)
    logp = logq.gather(1, at[:, None])[:, 0]
    # products of fp16 are exact in fp32.  A sum of D of them over 32 at a time: D / 32 additions to the
    # accumulator, at most 32 inside one product instruction, each within a step (2 U) of the sum of
    # magnitudes; the scaling by a rounded factor and the difference from the reference add 4 U of |x|
    dx = ((y.abs() @ e.abs().t()) * scale * (2 * U * (y.shape[1] / 32 + 32)) + 4 * U * x.abs()).amax(1)
    # 2^z is within 2 steps, the sums over the vocabulary within their count of joins (16 entries a
    # lane, 2^10 pieces at most, 2^9 joins): all terms are positive
    rel = 2 * U * (16 + 2 ** 10 + 2 ** 9)
    dev = (q * (logq + entropy[:, None]).abs()).sum(1)       # sum p |x - mean|: entropy's slope
    spread = (q * (x - x.amax(1, keepdim=True)).abs()).sum(1)
    return (logp, entropy, lse), (2 * dx + rel + 4 * U * logp.abs(),
                                  dx * dev + rel * (1 + 2 * spread + dev) + 4 * U * entropy,
                                  dx + rel + 4 * U * lse.abs())


def inputs(n, vocab, d, seed=0, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    e = (torch.randn(vocab, d, generator=g, device="cuda") * (spread / math.sqrt(d))).half()
    y = torch.randn(n, d, generator=g, device="cuda").half()
    tgt = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    return y, e, tgt


def check(got, want, tol):
    for name, a, b, t in zip(("logp", "entropy", "lse"), got, want, tol):
        assert a.dtype == torch.float32 and a.shape == b.shape
        off = (a.double() - b).abs() - t
        assert bool((off <= 0).all()), (name, float(off.max()), int(off.argmax()))


@pytest.mark.parametrize("n, vocab, d", [
    (1, 1, 64), (1, 2, 64), (3, 255, 64), (2, 256, 128), (127, 257, 192), (128, 1000, 64), (129, 511, 128),
    (255, 513, 64), (256, 4096, 256), (257, 5000, 64), (700, 32003, 128), (1, 40001, 1024), (33, 70000, 64),
    (64, 300, 2048), (1030, 769, 64)])
def test_logprobs_match_the_definition(n, vocab, d):
    from decentrik_prime_amd import k_head
    y, e, tgt = inputs(n, vocab, d, seed=n + vocab)
    tgt[0], tgt[-1] = 0, vocab - 1
    check(k_head.token_logprobs(y, e, tgt), *definition(y, e, tgt, 1.0))


@pytest.mark.parametrize("scale", [0.3, 1.7, 40.0])
def test_scale_is_a_factor_of_the_logits(scale):
    from decentrik_prime_amd import k_head
    y, e, tgt = inputs(50, 3000, 128, seed=3)
    check(k_head.token_logprobs(y, e, tgt, scale=scale), *definition(y, e, tgt, scale))


def test_peaked_rows_and_far_targets():
    """Logits to +-6 * 10^4: probabilities that are 1 or nothing, and scores of -10^5."""
    from decentrik_prime_amd import k_head
    y, e, tgt = inputs(40, 600, 64, seed=4, spread=40.0)
    y = (y * 60).half()
    best = (y.double() @ e.double().t()).argmax(1)
    tgt[::2] = best[::2].int()
    got = k_head.token_logprobs(y, e, tgt)
    check(got, *definition(y, e, tgt, 1.0))
    assert float(got[0].min()) < -1e4 and bool((got[0] <= 0).all())


@pytest.mark.parametrize("n, total", [(1, 9), (130, 64), (300, 1000), (5, 5)])
def test_rows_pick_from_yf(n, total):
    """Any rows in any order, some of them twice; rows behind each other in a wider buffer."""
    from decentrik_prime_amd import k_head
    y, e, tgt = inputs(total, 900, 128, seed=n)
    wide = torch.full((total, 160), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, :128] = y
    rows = torch.randint(0, total, (n,), device="cuda", dtype=torch.int32,
                         generator=torch.Generator(device="cuda").manual_seed(n))
    tgt = torch.randint(0, 900, (n,), device="cuda", dtype=torch.int32)
    got = k_head.token_logprobs(wide[:, :128], e, tgt, rows=rows)
    check(got, *definition(y[rows.long()], e, tgt, 1.0))


def test_targets_and_rows_outside():
    from decentrik_prime_amd import k_head
    y, e, tgt = inputs(200, 700, 64)
    clean = [t.clone() for t in k_head.token_logprobs(y, e, tgt)]
    tgt[3], tgt[77], tgt[150] = -1, 700, -100
    rows = torch.arange(200, device="cuda", dtype=torch.int32)
    rows[9], rows[10] = -1, 200
    logp, entropy, lse = k_head.token_logprobs(y, e, tgt, rows=rows)
    assert logp[3] == 0 and logp[150] == 0 and torch.isnan(logp[77])
    keep = torch.ones(200, dtype=torch.bool, device="cuda")
    keep[9:11] = False
    for t in (logp, entropy, lse):
        assert bool(torch.isnan(t[9:11]).all())
    assert torch.equal(entropy[keep], clean[1][keep]) and torch.equal(lse[keep], clean[2][keep])
    keep[[3, 77, 150]] = False
    assert torch.equal(logp[keep], clean[0][keep])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_row_that_is_not_finite_stays_alone(bad):
    from decentrik_prime_amd import k_head
    y, e, tgt = inputs(140, 999, 128)
    clean = [t.clone() for t in k_head.token_logprobs(y, e, tgt)]
    y[5, 17] = bad
    keep = torch.arange(140, device="cuda") != 5
    for got, want in zip(k_head.token_logprobs(y, e, tgt), clean):
        assert not bool(torch.isfinite(got[5])) and torch.equal(got[keep], want[keep])


def test_no_tokens_one_row_and_repeats():
    from decentrik_prime_amd import k_head
    y, e, tgt = inputs(300, 50001, 64)
    for t in k_head.token_logprobs(y[:0], e, tgt[:0]):
        assert t.shape == (0,)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert k_head.token_logprobs(y, e, none, rows=none)[0].shape == (0,)
    first = [t.clone() for t in k_head.token_logprobs(y, e, tgt)]
    for a, b in zip(k_head.token_logprobs(y, e, tgt), first):
        assert torch.equal(a, b)
    # a row by itself, from a tensor whose only row has any stride, and a row of ones' expansion
    one = k_head.token_logprobs(y[7:8], e, tgt[7:8])
    check(one, *definition(y[7:8], e, tgt[7:8], 1.0))
    odd = torch.empty(1, 2 * 64 + 1, dtype=torch.float16, device="cuda")[:, 1:65]
    odd.copy_(y[7:8])
    for a, b in zip(k_head.token_logprobs(odd.as_strided((1, 64), (3, 1), 1), e, tgt[7:8]), one):
        assert torch.equal(a, b)


def test_embedding_and_rows_past_4_gib():
    from decentrik_prime_amd import k_head
    vocab, d = 1_100_003, 2048                       # 4.5 GB
    e = torch.zeros(vocab, d, dtype=torch.float16, device="cuda")
    e[:, :64] = torch.randn(vocab, 64, device="cuda").half() * 0.2
    y = torch.randn(5, d, device="cuda").half()
    tgt = torch.tensor([0, vocab - 1, 1 << 20, 5, vocab - 2], dtype=torch.int32, device="cuda")
    want, tol = definition(y[:, :64], e[:, :64], tgt, 1.0)
    tol = [t * (d / 64) for t in tol]
    check(k_head.token_logprobs(y, e, tgt), want, tol)
    # e's own rows as the hidden states: row indices whose offsets pass 32 bits
    small = e[:500].clone()
    rows = torch.tensor([vocab - 1, 3, vocab, 1 << 20], dtype=torch.int32, device="cuda")
    t4 = torch.tensor([7, 499, 0, 3], dtype=torch.int32, device="cuda")
    got = k_head.token_logprobs(e, small, t4, rows=rows)
    ok = torch.tensor([True, True, False, True], device="cuda")
    want, tol = definition(e[rows.long()[ok], :64], small[:, :64], t4[ok], 1.0)
    check([g[ok] for g in got], want, [t * (d / 64) for t in tol])
    assert all(bool(torch.isnan(g[2])) for g in got)


@pytest.mark.parametrize("n, stride", [(200, 1 << 24), (2, 1 << 31), (300, 1 << 23)])
def test_rows_far_apart(n, stride):
    """Rows whose offsets within 256 of them pass 32 bits, and rows at the last stride that does not."""
    from decentrik_prime_amd import k_head
    y, e, tgt = inputs(n, 500, 64, seed=n)
    wide = torch.empty((n - 1) * stride + 64, dtype=torch.float16, device="cuda").as_strided((n, 64), (stride, 1))
    wide.copy_(y)
    for a, b in zip(k_head.token_logprobs(wide, e, tgt), k_head.token_logprobs(y, e, tgt)):
        assert torch.equal(a, b)
    rows = torch.randint(0, n, (77,), dtype=torch.int32, device="cuda")
    rows[5] = n
    tgt = torch.randint(0, 500, (77,), dtype=torch.int32, device="cuda")
    for a, b in zip(k_head.token_logprobs(wide, e, tgt, rows=rows), k_head.token_logprobs(y, e, tgt, rows=rows)):
        assert torch.equal(a.nan_to_num(nan=5.0), b.nan_to_num(nan=5.0)) and bool(a[5].isnan())


def some_rows(n, around):
    """The first and last tokens, those around given ones, and 500 more."""
    near = torch.cat([torch.arange(max(0, a - 3), min(n, a + 3)) for a in (0, n - 1, *around)])
    return torch.cat([near, torch.randint(0, n, (500,), generator=torch.Generator().manual_seed(1))]).cuda()


def test_picked_rows_of_more_than_2_to_the_31_elements():
    """Rows picked from 4 GiB of hidden states, more of them than 32-bit offsets reach."""
    from decentrik_prime_amd import k_head
    total, n = (1 << 25) + 8, (1 << 25) + 1000
    _, e, _ = inputs(1, 7, 64, seed=1)
    y = torch.randn(1 << 12, 64, device="cuda").half().repeat((total >> 12) + 1, 1)[:total]
    rows = (torch.arange(n, device="cuda", dtype=torch.int64) * 7 % total).int()
    rows[1 << 20], rows[n - 2] = total, -1
    tgt = (torch.arange(n, device="cuda") % 7).int()
    got = k_head.token_logprobs(y, e, tgt, rows=rows)
    some = some_rows(n, [(1 << 25) - 1])
    some = some[(rows[some] >= 0) & (rows[some] < total)]
    check([g[some] for g in got], *definition(y[rows[some].long()], e, tgt[some], 1.0))
    for g in got:
        bad = torch.nonzero(~g.isfinite())[:, 0]
        assert bad.tolist() == [1 << 20, n - 2]


def test_more_tokens_than_a_launch_takes():
    """2^26 tokens and some: a wave each would be 2^32 work items in one launch."""
    from decentrik_prime_amd import k_head
    n = (1 << 26) + 70
    _, e, _ = inputs(1, 5, 64, seed=2)
    y = torch.randn(1 << 12, 64, device="cuda").half().repeat((n >> 12) + 1, 1)[:n]
    tgt = (torch.arange(n, device="cuda") % 5).int()
    got = k_head.token_logprobs(y, e, tgt)
    some = some_rows(n, [1 << 24, 1 << 25, 3 << 24, 1 << 26])
    check([g[some] for g in got], *definition(y[some], e, tgt[some], 1.0))
    assert all(bool(g.isfinite().all()) for g in got)


def test_captured_and_on_another_stream():
    from decentrik_prime_amd import k_head
    y, e, tgt = inputs(300, 20000, 128)
    y2, _, tgt2 = inputs(300, 20000, 128, seed=9)
    want = [[t.clone() for t in k_head.token_logprobs(a, e, b)] for a, b in ((y, tgt), (y2, tgt2))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = k_head.token_logprobs(y, e, tgt)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graph = torch.cuda.CUDAGraph()
    sy, st = y.clone(), tgt.clone()
    with torch.cuda.graph(graph):
        out = k_head.token_logprobs(sy, e, st)
    for turn in range(4):
        sy.copy_((y, y2)[turn % 2])
        st.copy_((tgt, tgt2)[turn % 2])
        k_head.token_logprobs(y2, e, tgt2)           # eager work between the replays
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[turn % 2])), turn


def test_refusals():
    from decentrik_prime_amd import k_head
    y, e, tgt = inputs(4, 100, 64)
    for args, kwargs in (((y.float(), e, tgt), {}), ((y, e.float(), tgt), {}), ((y, e[:, :32], tgt), {}),
                         ((y[:, :32], e[:, :32].contiguous(), tgt), {}), ((y, e, tgt.long()), {}),
                         ((y, e, tgt[:3]), {}), ((y, e, tgt), dict(rows=tgt[:3])),
                         ((y, e, tgt), dict(rows=tgt.long())), ((y, e, tgt), dict(scale=0.0)),
                         ((y, e, tgt), dict(scale=float("nan"))), ((y, e.cpu(), tgt), {}),
                         ((y.repeat(2, 1)[::2, :], e[:0], tgt), {}), ((y.t().contiguous().t(), e, tgt), {})):
        with pytest.raises(ValueError):
            k_head.token_logprobs(*args, **kwargs)


def test_agrees_with_the_streamed_head():
    """The training head's loss, entropy and lse, whose logits are rounded to fp16 on the way."""
    from decentrik_prime_amd import k_head
    y, e, tgt = inputs(96, 1024, 128, seed=8)
    tgt[60:] = -1
    perm = torch.arange(96, device="cuda", dtype=torch.int32)
    src = k_head.ResidentEmbedding(e, 512)
    _, stats, _ = k_head.streamed_head(y, src, tgt, perm, 60, e[tgt[:60].long()].contiguous(), 1024.0)
    logp, entropy, lse = k_head.token_logprobs(y, src, tgt)
    top = float((y.double() @ e.double().t()).abs().max())
    atol = 3 * top * 2.0 ** -11                      # half a step of the largest fp16 logit, twice in logp
    for a, b in ((-logp, stats[:, 0]), (entropy, stats[:, 1]), (lse, stats[:, 3])):
        assert float((a - b).abs().max()) <= atol
