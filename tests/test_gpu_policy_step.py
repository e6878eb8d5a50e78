"""Training steps from rewards and preferences (model.QwenQLoRAStep.score, policy_step, preference_step,
clip_grads) on packed answers, against float64 autograd of the decoder with the same token weights."""

import numpy as np
import pytest
import torch

from tests.helpers import host, log
from tests.test_gpu_model import _reference_inputs

pytestmark = pytest.mark.gpu

VOCAB = 4096


def _groups(seed=3):
    rng = np.random.default_rng(seed)
    return [(rng.integers(0, VOCAB, p), [rng.integers(0, VOCAB, a) for a in ans])
            for p, ans in ((70, (30, 1, 45)), (9, (40, 12)))]


def _step(shared=True, **kw):
    """(batch, step) of the groups' answers, behind shared prompts or in rows of their own."""
    from decentrik_prime_amd import model, trainer
    if shared:
        batch = trainer.pack_answers(_groups(), VOCAB)
    else:
        whole = [(np.concatenate([p, a]), len(p)) for p, ans in _groups() for a in ans]
        ids, mask, labels = (torch.zeros(len(whole), 130, dtype=torch.int64) for _ in range(3))
        labels -= 100
        for b, (w, n) in enumerate(whole):
            ids[b, :len(w)], mask[b, :len(w)] = torch.from_numpy(w), 1
            labels[b, n:len(w)] = torch.from_numpy(w[n:])
        batch = trainer.pack(ids, mask, labels, VOCAB)
    return batch, model.QwenQLoRAStep.for_batch(batch, n_layers=2, vocab=VOCAB, seed=5, head_chunk=1024, **kw)


def _visible(batch):
    from oracle import attn
    return None if batch.groups is None else torch.from_numpy(attn.prefix_visible(batch.groups))


def _check_grads(st, want):
    """LoRA gradients as the causal step's test holds them: within 1e-2 of their largest."""
    for i in range(2):
        for nm, got, ref in zip(("dA_q", "dB_q", "dA_v", "dB_v"), st.grads[i], want[i]):
            g, r = host(got).astype(np.float64), ref.numpy()
            err = float(np.abs(g - r).max()) / float(np.abs(r).max())
            assert err <= 1e-2, f"layer {i} {nm}: {err:.3g}"


@pytest.mark.parametrize("shared", [True, False])
def test_policy_step_matches_float64(shared):
    from decentrik_prime_amd import k_loss, k_nf4, trainer
    from oracle import model as ref
    batch, st = _step(shared)
    log(f"policy step, shared prompts {shared}")
    lens = trainer.answer_lens(batch)
    assert lens == [30, 1, 45, 40, 12]
    meta = k_loss.row_meta(lens, "cuda")
    old, _ = st.score()
    base, _ = st.score(adapters=False)
    adv = torch.tensor([1.0, -0.5, 0.25, -2.0, 0.0], device="cuda")
    old = old + 0.1 * torch.randn(old.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    loss, rows, stats = st.policy_step(meta, old, adv, ref=base, kl_coef=0.1)
    again, dlogp, rows2 = k_loss.policy_loss(stats, old, adv, meta, ref=base, kl_coef=0.1)
    assert torch.equal(loss, again) and torch.equal(rows, rows2)
    weights = torch.zeros(st.m)
    weights[st.labelled.cpu()] = -dlogp.cpu()
    _, want = ref.qwen_step(_reference_inputs(torch, st, k_nf4), st.lens, visible=_visible(batch),
                            weights=weights)
    _check_grads(st, want)
    # the norm, and the gradients scaled to a quarter of it
    before = [g.clone() for layer in st.grads for g in layer]
    norm = float(torch.cat([g.reshape(-1) for g in before]).double().norm())
    assert float(st.clip_grads(norm / 4)) == pytest.approx(norm, rel=1e-6)
    for a, b in zip((g for layer in st.grads for g in layer), before):
        assert torch.allclose(a, b * 0.25, rtol=1e-4, atol=0)     # (1e-6 beside the norm)


def test_preference_step_matches_float64():
    from decentrik_prime_amd import k_loss, k_nf4, trainer
    from oracle import model as ref
    batch, st = _step()
    log("preference step")
    meta = k_loss.row_meta(trainer.answer_lens(batch), "cuda", pairs=[(0, 1), (2, 0), (3, 4)])
    base, _ = st.score(adapters=False)
    loss, rewards, margins, stats = st.preference_step(meta, base, beta=0.3, label_smoothing=0.1)
    again, dlogp, r2, m2 = k_loss.preference_loss(stats, base, meta, beta=0.3, label_smoothing=0.1)
    assert torch.equal(loss, again) and torch.equal(rewards, r2) and torch.equal(margins, m2)
    weights = torch.zeros(st.m)
    weights[st.labelled.cpu()] = -dlogp.cpu()
    _, want = ref.qwen_step(_reference_inputs(torch, st, k_nf4), st.lens, visible=_visible(batch),
                            weights=weights)
    _check_grads(st, want)


def test_unit_weights_are_the_cross_entropy_step():
    """dlogp of -1 throughout: the gradients of backward() without it, bit for bit, and halved with it."""
    _, st = _step()
    _, _, dy = st.forward()
    plain = [g.clone() for layer in st.backward(dy) for g in layer]
    _, _, dy = st.forward()
    ones = torch.full((st.n_lab,), -1.0, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip((g for la in st.backward(dy, dlogp=ones) for g in la), plain))
    with pytest.raises(ValueError):
        st.backward(dy, dlogp=ones[1:])


@pytest.mark.parametrize("shift", [-40, -20, -3, 30])
def test_gradients_keep_their_digits_at_any_size_of_the_loss(shift):
    """A loss's gradient times a power of two: the LoRA gradients times it, bit for bit."""
    _, st = _step()
    g = torch.Generator("cuda").manual_seed(2)
    dlogp = torch.randn(st.n_lab, generator=g, device="cuda")
    _, _, dy = st.forward()
    want = [t.double() * 2.0 ** shift for layer in st.backward(dy, dlogp=dlogp) for t in layer]
    _, _, dy = st.forward()
    got = [t.double() for layer in st.backward(dy, dlogp=dlogp * 2.0 ** shift) for t in layer]
    for a, b in zip(got, want):
        assert float(b.abs().max()) > 0 and torch.equal(a, b)
    _, _, dy = st.forward()
    got = [t.double() for layer in st.backward(dy, 2.0 ** shift, dlogp=dlogp) for t in layer]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_small_weights_match_float64():
    """2048 tokens in 16 answers, advantages near 1e-2 and means over rows and tokens (a token's weight is
    near 5e-6), and a preference loss over 40 pairs with beta 0.1."""
    from decentrik_prime_amd import k_loss, k_nf4, model, trainer
    from oracle import model as ref
    rng = np.random.default_rng(8)
    groups = [(rng.integers(0, VOCAB, 65), [rng.integers(0, VOCAB, 112) for _ in range(4)]) for _ in range(4)]
    batch = trainer.pack_answers(groups, VOCAB)
    st = model.QwenQLoRAStep.for_batch(batch, n_layers=2, vocab=VOCAB, seed=5, head_chunk=1024)
    assert st.m == 2064
    lens = trainer.answer_lens(batch)
    pairs = [(int(a), int(b)) for a, b in rng.integers(0, 16, (40, 2)) if a != b]
    meta = k_loss.row_meta(lens, "cuda", pairs=pairs)
    old, _ = st.score()
    base, _ = st.score(adapters=False)
    adv = 1e-2 * torch.randn(16, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    p = _reference_inputs(torch, st, k_nf4)
    for which in ("policy", "preference"):
        if which == "policy":
            _, _, stats = st.policy_step(meta, old, adv, ref=base, kl_coef=1e-3)
            _, dlogp, _ = k_loss.policy_loss(stats, old, adv, meta, ref=base, kl_coef=1e-3)
        else:
            _, _, _, stats = st.preference_step(meta, base, beta=0.1, average=True)
            _, dlogp, _, _ = k_loss.preference_loss(stats, base, meta, beta=0.1, average=True)
        log(f"{which}: largest weight {float(dlogp.abs().max()):.3g}")
        assert 0 < float(dlogp.abs().max()) < 1e-3
        weights = torch.zeros(st.m)
        weights[st.labelled.cpu()] = -dlogp.cpu()
        _, want = ref.qwen_step(p, st.lens, visible=_visible(batch), weights=weights)
        _check_grads(st, want)


def test_a_step_on_log_probabilities_of_fp32():
    """The step in its parts, with the current log-probabilities from token_logprobs as score's are: without
    dropout the ratio is 1 but for the adapters' input (no rounding of the logits to fp16 in between)."""
    from decentrik_prime_amd import k_head, k_loss, k_nf4, trainer
    from oracle import model as ref
    batch, st = _step()
    for i in range(2):
        for k in ("mq", "mv"):
            st.lora[i][k] = torch.ones_like(st.lora[i][k])
    st.keep_scale = 1.0
    meta = k_loss.row_meta(trainer.answer_lens(batch), "cuda")
    old, _ = st.score()
    base, _ = st.score(adapters=False)
    adv = torch.tensor([1.0, -0.5, 0.25, -2.0, 0.0], device="cuda")
    _, _, dy = st.forward()
    logp, _, _ = k_head.token_logprobs(st.yf, st.source, st.tgt_sorted[:st.n_lab], rows=st.perm[:st.n_lab])
    _, dlogp, rows = k_loss.policy_loss(logp, old, adv, meta, ref=base, kl_coef=0.1)
    st.backward(dy, dlogp=dlogp)
    assert float((logp - old).abs().max()) <= 5e-3 and float((rows[:, 3] - 1).abs().max()) <= 5e-3
    weights = torch.zeros(st.m)
    weights[st.labelled.cpu()] = -dlogp.cpu()
    _, want = ref.qwen_step(_reference_inputs(torch, st, k_nf4), st.lens, visible=_visible(batch),
                            weights=weights)
    _check_grads(st, want)


def test_a_captured_policy_step_replays():
    """The whole step in a graph, on advantages of two sizes in turn, with eager steps between the replays."""
    from decentrik_prime_amd import k_loss, trainer
    batch, st = _step()
    meta = k_loss.row_meta(trainer.answer_lens(batch), "cuda")
    old, _ = st.score()
    base, _ = st.score(adapters=False)
    both = [torch.tensor(a, device="cuda") for a in ([1.0, -0.5, 0.25, -2.0, 0.0], [-1e-6, 2e-6, 0.0, 0.0, 5e-6])]

    def run(a):
        loss, rows, _ = st.policy_step(meta, old, a, ref=base, kl_coef=1e-7)
        return [loss, rows, *(g for layer in st.grads for g in layer)]
    want = [[t.clone() for t in run(a)] for a in both]
    graph, adv = torch.cuda.CUDAGraph(), both[0].clone()
    with torch.cuda.graph(graph):
        out = run(adv)
    for turn in range(4):
        adv.copy_(both[turn % 2])
        run(both[1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[turn % 2])), turn


def test_losses_that_are_nothing_or_not_finite():
    """No gradient at all gives zeros, as does a batch without targets; an infinite one is not hidden."""
    from decentrik_prime_amd import k_loss, trainer
    batch, st = _step()
    for dlogp in (torch.zeros(st.n_lab, device="cuda"), torch.full((st.n_lab,), np.inf, device="cuda")):
        _, _, dy = st.forward()
        grads = [g for layer in st.backward(dy, dlogp=dlogp) for g in layer]
        for g in grads:
            assert bool((g == 0).all()) if not bool(dlogp.isinf().any()) else not bool(g.isfinite().all())
    st.use_tokens(batch.ids, torch.full_like(batch.tgt, -1))
    meta = k_loss.row_meta([0] * batch.B, "cuda")
    none = torch.zeros(0, device="cuda")
    loss, rows, _ = st.policy_step(meta, none, torch.ones(batch.B, device="cuda"))
    assert float(loss) == 0 and bool((rows == 0).all())
    assert all(bool((g == 0).all()) for layer in st.grads for g in layer)


@pytest.mark.parametrize("ahead", ["layer", "carried", ("gu", "d", "qkv", "o")])
def test_score_between_forward_and_backward(ahead):
    """Scoring, with adapters and without, before a step and inside it: the step's loss and gradients stay
    the same bits, and so do the scores; without dropout they are the step's own log-probabilities."""
    _, st = _step(ahead=ahead)
    for i in range(2):
        for k in ("mq", "mv"):
            st.lora[i][k] = torch.ones_like(st.lora[i][k])
    st.keep_scale = 1.0
    loss = st.step()
    want = [g.clone() for layer in st.grads for g in layer]
    first = [t.clone() for a in (True, False) for t in st.score(adapters=a)]
    again, stats, dy = st.forward()
    middle = [t.clone() for a in (True, False) for t in st.score(adapters=a)]
    grads = [g for layer in st.backward(dy) for g in layer]
    assert torch.equal(loss, again) and all(torch.equal(a, b) for a, b in zip(grads, want))
    assert all(torch.equal(a, b) for a, b in zip(first, middle))
    # the training head's logits are rounded to fp16; hidden states alike but for the adapters' input,
    # rounded once there
    n = st.n_lab
    tol = 2.0 ** -11 * 2 * float(stats[:, 3].abs().max() + stats[:n, 0].max()) + 5e-3
    assert float((first[0] + stats[:n, 0]).abs().max()) <= tol
    assert float((first[1] - stats[:n, 1]).abs().max()) <= tol
    assert float((first[2] - first[0]).abs().max()) > 1e-3          # the adapters matter


def test_score_without_adapters_is_the_base_model():
    _, st = _step()
    base = [t.clone() for t in st.score(adapters=False)]
    for i in range(2):
        st.lora[i]["Bq"].zero_()
        st.lora[i]["Bv"].zero_()
    for a, b in zip(st.score(), base):
        assert torch.equal(a, b)
    warm = st.score(scale=0.5)
    assert float((warm[1] - base[1]).min()) > 0                     # a higher temperature: more entropy


def test_plans_of_another_batch_are_refused():
    from decentrik_prime_amd import k_loss
    _, st = _step()
    meta = k_loss.row_meta([3, 4], "cuda", pairs=[(0, 1)])
    x = torch.zeros(7, device="cuda")
    with pytest.raises(ValueError):
        st.policy_step(meta, x, torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError):
        st.preference_step(meta, x)
    with pytest.raises(ValueError, match="no gradients"):
        st.clip_grads(1.0)


@pytest.mark.parametrize("d", [64, 1536, 4096])
@pytest.mark.parametrize("fp32", [False, True])
def test_norm_backward_with_a_factor_per_row(d, fp32):
    from decentrik_prime_amd import k_norm
    from oracle import norm
    g = torch.Generator(device="cuda").manual_seed(d)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    n = 37
    x, w, dres = randn(n, d), 1 + 0.1 * randn(d), randn(n, d)
    dy = randn(n, d) if fp32 else randn(n, d).half()
    rstd = torch.rsqrt(x.square().mean(1) + 1e-6)
    gscale, scale = torch.full((1,), 0.5, device="cuda"), randn(n)
    scale[3] = 0.0
    out, plain, one = dres.clone(), dres.clone(), dres.clone()
    k_norm.rms_backward(dy, gscale, x, w, rstd, out, dres=out, row_scale=scale)
    up = host(dy).astype(np.float64) * 0.5 * host(scale).astype(np.float64)[:, None]
    want = norm.rms_bwd_float64(up, host(x).astype(np.float64), host(w), 1e-6) + host(dres)
    assert np.allclose(host(out), want, rtol=1e-4, atol=1e-4)      # as without factors
    assert torch.equal(out[3], dres[3])
    k_norm.rms_backward(dy, gscale, x, w, rstd, plain, dres=plain)
    k_norm.rms_backward(dy, gscale, x, w, rstd, one, dres=one, row_scale=torch.ones_like(scale))
    assert torch.equal(one, plain)
    for bad in (scale[1:], scale.double(), scale.cpu(), scale.view(n, 1)):
        with pytest.raises(ValueError):
            k_norm.rms_backward(dy, gscale, x, w, rstd, out, row_scale=bad)
