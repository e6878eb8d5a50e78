"""The trainer integration's tensor part on the CPU (decentrik_prime_amd/trainer.py): packing of a
right-padded batch (solution/fast_qwen.py:803-871), batch_metrics over per-token stats in the
packing's sorted order (solution/fast_qwen.py:1551-1565) against a walk of the padded batch
(oracle/trainer.py), and compute_loss's normalisation (solution/integration.py:657-664)."""

import numpy as np
import pytest
import torch

from decentrik_prime_amd import trainer
from oracle import trainer as ref


def _batch(seed=0, lens=(5, 3, 7), T=8, vocab=50):
    rng = np.random.default_rng(seed)
    B = len(lens)
    ids = torch.from_numpy(rng.integers(0, vocab, (B, T)))
    mask = (torch.arange(T)[None, :] < torch.tensor(lens)[:, None]).to(torch.int64)
    labels = ids.clone()
    labels[mask == 0] = -100
    labels[0, :2] = -100          # a prompt the loss ignores
    labels[2, 3] = -100
    return ids, mask, labels


def test_pack_tokens_targets_and_order():
    ids, mask, labels = _batch()
    b = trainer.pack(ids, mask, labels, vocab=50)
    assert b.lens == [5, 3, 7] and b.n_real == 15 and b.B == 3 and b.T == 8
    assert torch.equal(b.ids, torch.cat([ids[0, :5], ids[1, :3], ids[2, :7]]))
    # target of token (r, t) = labels[r, t + 1] (ignore index and past the end: none)
    want = []
    for r, n in enumerate(b.lens):
        for t in range(n):
            lab = int(labels[r, t + 1]) if t + 1 < 8 else -100
            want.append(lab if lab != -100 else -1)
    assert b.tgt.tolist() == want
    has = np.array(want) >= 0
    assert b.n_lab == int(has.sum())
    # sorted order: tokens with a target first, each group in token order
    assert b.perm.tolist() == list(np.nonzero(has)[0]) + list(np.nonzero(~has)[0])
    assert b.valid_sorted.tolist() == [True] * b.n_lab + [False] * (15 - b.n_lab)
    rows = np.repeat(np.arange(3), b.lens)
    assert b.row_sorted.tolist() == rows[b.perm.numpy()].tolist()
    assert b.tgt_sorted.tolist() == np.array(want)[b.perm.numpy()].tolist()


@pytest.mark.parametrize("seed", range(6))
def test_pack_against_a_token_walk(seed):
    """Random batches, full rows included, against a walk over every (row, position): the target
    of a real token is the row's next label, even when that label sits at a padded position (the
    collator's -100 there is what makes it none), and -1 past the padded length."""
    rng = np.random.default_rng(100 + seed)
    B, T, vocab = int(rng.integers(1, 5)), int(rng.integers(2, 12)), 40
    lens = [int(v) for v in rng.integers(1, T + 1, B)]
    ids = torch.from_numpy(rng.integers(0, vocab, (B, T)))
    mask = (torch.arange(T)[None, :] < torch.tensor(lens)[:, None]).to(torch.int64)
    labels = torch.from_numpy(np.where(rng.random((B, T)) < 0.3, -100,
                                       rng.integers(0, vocab, (B, T))))
    b = trainer.pack(ids, mask, labels, vocab)
    toks, tg, rows = [], [], []
    for r in range(B):
        for t in range(T):
            if mask[r, t] == 1:
                toks.append(int(ids[r, t]))
                nxt = int(labels[r, t + 1]) if t + 1 < T else -100
                tg.append(nxt if nxt >= 0 else -1)
                rows.append(r)
    assert b.lens == lens and b.ids.tolist() == toks and b.tgt.tolist() == tg
    order = [i for i, v in enumerate(tg) if v >= 0] + [i for i, v in enumerate(tg) if v < 0]
    assert b.perm.tolist() == order
    assert b.row_sorted.tolist() == [rows[i] for i in order]
    assert b.n_lab == sum(v >= 0 for v in tg) and b.n_real == len(toks)
    # a mask value other than 0 and 1 makes the batch unpackable
    mask[0, 0] = 2
    assert trainer.pack(ids, mask, labels, vocab) is None


@pytest.mark.parametrize("case", ["gap", "empty_row", "id_range", "label_range", "shape"])
def test_pack_refuses_what_it_cannot_pack(case):
    ids, mask, labels = _batch()
    if case == "gap":
        mask[0, 1] = 0                       # not one run of ones from the start
    elif case == "empty_row":
        mask[1] = 0
    elif case == "id_range":
        ids[2, 0] = 50
    elif case == "label_range":
        labels[1, 1] = 50
    elif case == "shape":
        labels = labels[:, :-1]
    assert trainer.pack(ids, mask, labels, vocab=50) is None


def test_batch_metrics_against_the_padded_walk():
    ids, mask, labels = _batch(seed=3, lens=(8, 1, 6, 4), T=8)
    b = trainer.pack(ids, mask, labels, vocab=50)
    rng = np.random.default_rng(4)
    tok = np.stack([rng.uniform(0, 9, b.n_real), rng.uniform(0, 5, b.n_real),
                    rng.integers(0, 2, b.n_real), rng.uniform(0, 12, b.n_real)], 1)
    start = np.concatenate([[0], np.cumsum(b.lens)[:-1]])
    got = trainer.batch_metrics(b, torch.from_numpy(tok[b.perm.numpy()]))
    want = ref.padded_metrics(lambda r, t: tok[start[r] + t, :3], b.lens, labels.numpy())
    assert got["n_lab"] == want["n_lab"] == b.n_lab
    assert got["row_tokens"] == want["row_tokens"]
    assert got["entropy"] == pytest.approx(want["entropy"], rel=1e-12)
    assert got["accuracy"] == pytest.approx(want["accuracy"], rel=1e-12)
    assert got["row_loss"] == pytest.approx(want["row_loss"], rel=1e-12)
    # a row whose only token has no target gets loss 0 over 0 tokens
    assert got["row_tokens"][1] == 0 and got["row_loss"][1] == 0.0


def test_batch_metrics_without_targets_and_bad_stats():
    ids, mask, labels = _batch()
    labels[:] = -100
    b = trainer.pack(ids, mask, labels, vocab=50)
    assert b.n_lab == 0
    m = trainer.batch_metrics(b, torch.ones(b.n_real, 4))
    assert m["accuracy"] == 0.0 and m["entropy"] == 1.0 and m["row_tokens"] == [0, 0, 0]
    with pytest.raises(ValueError):
        trainer.batch_metrics(b, torch.ones(b.n_real - 1, 4))


def test_compute_loss_normalisation():
    ids, mask, labels = _batch()
    b = trainer.pack(ids, mask, labels, vocab=50)
    s = torch.tensor(12.0)
    assert float(trainer.compute_loss(s, b)) == pytest.approx(12.0 / b.n_lab)
    assert float(trainer.compute_loss(s, b, num_items_in_batch=4)) == pytest.approx(12.0 / b.n_lab)
    assert float(trainer.compute_loss(s, b, num_items_in_batch=4,
                                      model_accepts_loss_kwargs=True)) == pytest.approx(3.0)
    assert float(trainer.compute_loss(s, b, num_items_in_batch=torch.tensor(6),
                                      model_accepts_loss_kwargs=True)) == pytest.approx(2.0)


def test_padded_walk_known_answer():
    """The padded-batch walk and the packed metrics on a batch small enough to work by hand.
    Row 0 has 3 real tokens, row 1 has 2 (T = 4).  A token's target is the next position's label:
    row 0 -> (none: -100, 7, none: -100), row 1 -> (3, none: -100), so tokens (0, 1) and (1, 0)
    carry the loss.  Per-token (loss, entropy, hit) = (1, 2, 0), (3, 4, 1), (5, 6, 1) | (7, 8, 1),
    (9, 10, 0): entropy = (2 + 4 + 6 + 8 + 10) / 5 = 6, accuracy = (1 + 1) / 2 = 1, row losses 3
    and 7 over one token each."""
    lens = [3, 2]
    labels = np.array([[5, -100, 7, -100], [9, 3, -100, -100]])
    stats = {(0, 0): (1, 2, 0), (0, 1): (3, 4, 1), (0, 2): (5, 6, 1), (1, 0): (7, 8, 1),
             (1, 1): (9, 10, 0)}
    want = {"entropy": 6.0, "accuracy": 1.0, "n_lab": 2, "row_loss": [3.0, 7.0],
            "row_tokens": [1, 1]}
    assert ref.padded_metrics(lambda b, t: stats[(b, t)], lens, labels) == want
    ids = torch.tensor([[1, 2, 3, 0], [4, 5, 0, 0]])
    mask = torch.tensor([[1, 1, 1, 0], [1, 1, 0, 0]])
    b = trainer.pack(ids, mask, torch.from_numpy(labels), vocab=10)
    assert b.tgt.tolist() == [-1, 7, -1, 3, -1]
    tok = [stats[(0, 0)], stats[(0, 1)], stats[(0, 2)], stats[(1, 0)], stats[(1, 1)]]
    st = torch.tensor([list(tok[i]) + [0.0] for i in b.perm.tolist()], dtype=torch.float64)
    assert trainer.batch_metrics(b, st) == want


def test_pack_answers_against_a_token_walk():
    """Every answer's row of targets is that of the prompt and the answer packed alone with the prompt's
    labels ignored; the prompt stands once; what an answer's token sees are the tokens before it."""
    from decentrik_prime_amd import k_attn
    from oracle import attn
    rng = np.random.default_rng(5)
    groups = [(rng.integers(0, 40, p), [rng.integers(0, 40, a) for a in ans])
              for p, ans in ((6, (3, 1, 4)), (1, (5,)), (9, (2, 2)))]
    b = trainer.pack_answers(groups, vocab=40)
    assert b.groups == [(5, [4, 2, 5]), (0, [6]), (8, [3, 3])] and b.B == 6 and b.T == 11
    assert sum(b.lens) == b.n_real == b.ids.numel() and b.n_lab == 17
    vis = attn.prefix_visible(b.groups)
    meta = k_attn.prefix_meta(b.groups, 2, 1, "cpu")
    at, row = 0, 0
    for prompt, answers in groups:
        first = at
        assert b.ids[at:at + len(prompt) - 1].tolist() == prompt[:-1].tolist()
        assert (b.tgt[at:at + len(prompt) - 1] == -1).all()
        at += len(prompt) - 1
        for a in answers:
            whole = np.concatenate([prompt, a])
            lab = np.concatenate([np.full(len(prompt), -100), a])
            alone = trainer.pack(torch.from_numpy(whole)[None], torch.ones(1, len(whole), dtype=torch.int64),
                                 torch.from_numpy(lab)[None], 40)
            end = at + 1 + len(a)
            assert b.ids[at:end].tolist() == whole[len(prompt) - 1:].tolist()
            assert b.tgt[at:end].tolist() == alone.tgt[len(prompt) - 1:].tolist()
            for t in range(at, end):
                seen = np.nonzero(vis[t])[0]
                assert b.ids[seen].tolist() == whole[:len(prompt) + t - at].tolist()
                assert int(meta.positions[t]) == len(seen) - 1
            of_row = b.row_sorted[(b.perm >= at) & (b.perm < end)]
            assert (of_row == row).all()
            at, row = end, row + 1
        assert at > first
    assert at == b.n_real


def test_pack_answers_refuses():
    for groups in ([], [([1, 2], [])], [([], [[1]])], [([1], [[]])], [([1], [[40]])], [([-1], [[3]])],
                   [([[1, 2]], [[3]])]):
        assert trainer.pack_answers(groups, vocab=40) is None


def test_metrics_of_shared_prompts_are_those_of_rows_of_their_own():
    """batch_metrics of a batch packed by pack_answers equal those of the same answers as rows with a
    prompt each: a prompt's token counts once for every answer behind it."""
    rng = np.random.default_rng(8)
    groups = [(rng.integers(0, 40, p), [rng.integers(0, 40, a) for a in ans])
              for p, ans in ((6, (3, 1, 4)), (1, (5,)), (9, (2, 2)))]
    shared = trainer.pack_answers(groups, vocab=40)
    whole = [(np.concatenate([p, a]), len(p)) for p, ans in groups for a in ans]
    T = max(len(w) for w, _ in whole)
    ids, mask, labels = (torch.zeros(len(whole), T, dtype=torch.int64) for _ in range(3))
    labels -= 100
    for b, (w, n) in enumerate(whole):
        ids[b, :len(w)], mask[b, :len(w)] = torch.from_numpy(w), 1
        labels[b, n:len(w)] = torch.from_numpy(w[n:])
    rows = trainer.pack(ids, mask, labels, 40)
    # (loss, entropy, hit, lse) of a token, by what stands before it and what comes next
    known = {}

    def stats(batch, before):
        out = torch.zeros(batch.n_real, 4, dtype=torch.float64)
        for i, t in enumerate(batch.perm.tolist()):
            seen = tuple(before(t))
            ent = known.setdefault(seen, rng.random())
            tgt = int(batch.tgt[t])
            loss, hit = known.setdefault((seen, tgt), (rng.random(), float(rng.integers(0, 2))))
            out[i] = torch.tensor([loss if tgt >= 0 else 0.0, ent, hit if tgt >= 0 else 0.0, 0.0])
        return out
    from oracle import attn
    vis = attn.prefix_visible(shared.groups)
    ends = np.cumsum(rows.lens)
    starts = ends - np.asarray(rows.lens)

    def in_row(t):
        return rows.ids[starts[np.searchsorted(ends, t, side="right")]:t + 1].tolist()
    a = trainer.batch_metrics(shared, stats(shared, lambda t: shared.ids[np.nonzero(vis[t])[0]].tolist()))
    b = trainer.batch_metrics(rows, stats(rows, in_row))
    # sums of at most 60 values in [0, 1) in 64 bits, in another order
    assert abs(a["entropy"] - b["entropy"]) < 60 * 2.0 ** -52
    assert abs(a["accuracy"] - b["accuracy"]) < 2.0 ** -52
    np.testing.assert_allclose(a["row_loss"], b["row_loss"], rtol=1e-14)
    assert a["row_tokens"] == b["row_tokens"] and a["n_lab"] == b["n_lab"]
