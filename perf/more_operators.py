"""Training from preferences and rewards: token log-probabilities of the language-model head, the clipped
policy loss with a KL term, the preference loss over pairs of answers, and clipping by the global gradient
norm.

``run`` with ``own`` true makes the calls of decentrik_prime_amd (k_head, k_loss, k_grad); with ``own``
false it computes the same outputs in elementary torch operations, in 32 bits (the clip's borders, sums over
tokens and sums of squares in 64), rounded once at the end.  ``exact`` computes them from the definitions in
64 bits.

  logprobs    x_v = scale <y, E_v>: log p of a target, the entropy and log sum e^x, for each token
  policy      r = e^(logp - old), p = -min(r A, clip(r) A), k = e^(ref - logp) - (ref - logp) - 1; the
              weighted sum of p + kl k, its gradient for logp, and each row's means of (p, k, clipped, r)
  preference  S = a row's sum (or mean) of logp - ref, h = beta (S_chosen - S_rejected) - margin; the mean
              over pairs, its gradient for logp, beta S and h
  clip        the norm of all gradients together, and the gradients scaled to at most max_norm
"""

import math

import torch

own = False

VOCAB, HIDDEN = 151936, 1536


def listed():
    return [
        # scoring one token: the embedding is read once
        dict(name="logprobs_one", op="logprobs", n=1, total=1, vocab=VOCAB, hidden=HIDDEN, scale=1.0),
        # a few tokens of a smaller model with an odd vocabulary: latency
        dict(name="logprobs_few", op="logprobs", n=37, total=64, vocab=32003, hidden=1024, scale=1.0),
        # the labelled tokens of a packed batch, sampled at a temperature
        dict(name="logprobs_labelled", op="logprobs", n=853, total=2048, vocab=VOCAB, hidden=HIDDEN,
             scale=1.25),
        # every token of a packed batch
        dict(name="logprobs_packed", op="logprobs", n=2048, total=2048, vocab=VOCAB, hidden=HIDDEN,
             scale=1.0),
        # eight answers to one prompt, the current log-probabilities from the head's stats: latency
        dict(name="policy_answers", op="policy", lens="128,97,160,33,255,128,95,128", per_token=False,
             ref=True, kl=0.04, low=0.2, high=0.2, reduction="row", stats=True),
        # a batch of 64 answers, one of them empty, advantages per token, no reference
        dict(name="policy_batch", op="policy", lens="0," + ",".join(str(37 + 15 * i) for i in range(63)),
             per_token=True, ref=False, kl=0.0, low=0.2, high=0.28, reduction="token", stats=False),
        # a rollout of 2048 answers in one call
        dict(name="policy_rollout", op="policy",
             lens=",".join(str(1 + (i * 379) % 1021) for i in range(2048)), per_token=False, ref=True,
             kl=0.001, low=0.2, high=0.2, reduction="row", stats=True),
        # one pair of answers: the least work
        dict(name="preference_pair", op="preference", lens="200,37", pairs="0-1", ref=True, beta=0.1,
             kind="sigmoid", smoothing=0.0, margin=0.0, average=False),
        # all pairs among groups of eight answers to one prompt, rows in several pairs
        dict(name="preference_groups", op="preference", lens=",".join(str(64 + 29 * i) for i in range(32)),
             pairs=",".join("%d-%d" % (8 * g + i, 8 * g + j) for g in range(4) for i in range(8)
                            for j in range(i + 1, 8)),
             ref=True, beta=0.1, kind="sigmoid", smoothing=0.1, margin=0.0, average=False),
        # 512 pairs of long answers, by their mean log-probability, without a reference
        dict(name="preference_long", op="preference",
             lens=",".join(str(1 + (i * 379) % 2039) for i in range(1024)),
             pairs=",".join("%d-%d" % (i, 512 + i) for i in range(512)), ref=False, beta=2.0,
             kind="sigmoid", smoothing=0.0, margin=0.5, average=True),
        # the adapters' gradients of a 28-layer step (rank 16 on the query and value projections), in place
        dict(name="clip_adapters", op="clip", sizes=",".join(["24576,24576,24576,4096"] * 28), types="fp32",
             rms=1e-3, max_norm=1.0, scale=1.0, to_fp32=False),
        # half-precision gradients of a whole embedding and its norms, unscaled into fp32
        dict(name="clip_embedding", op="clip", sizes="1536,%d,1536,8960" % (VOCAB * HIDDEN), types="fp16",
             rms=0.5, max_norm=1.0, scale=1.0 / 1024, to_fp32=True),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], its logarithm evenly spread."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_lens(rng, rows, tokens):
    """Lengths of `rows` rows, about `tokens` in all, some empty."""
    mean = max(1, tokens // rows)
    return [0 if rng.random() < 0.05 else _spread(rng, max(1, mean // 8), 2 * mean) for _ in range(rows)]


def draw(rng):
    op = rng.choice(["logprobs", "policy", "preference", "clip"])
    case = dict(op=op)
    if op == "logprobs":
        hidden = 64 * _spread(rng, 1, 32)
        vocab = _spread(rng, 500, VOCAB)
        most = min(2048, 2048 * VOCAB * HIDDEN // (vocab * hidden))
        n = _spread(rng, 1, most)
        case.update(n=n, total=rng.choice([n, n + rng.randint(1, 100)]), vocab=vocab, hidden=hidden,
                    scale=rng.choice([1.0, round(rng.uniform(0.5, 2.0), 3)]))
    elif op == "policy":
        lens = _draw_lens(rng, _spread(rng, 1, 512), _spread(rng, 1, 500000))
        lens[rng.randrange(len(lens))] += 1
        ref = rng.random() < 0.6
        case.update(lens=",".join(map(str, lens)), per_token=rng.random() < 0.4, ref=ref,
                    kl=rng.choice([0.0, 0.001, 0.04]) if ref else 0.0, low=0.2,
                    high=rng.choice([0.2, 0.28]), reduction=rng.choice(["row", "token", "sum"]),
                    stats=rng.random() < 0.5)
    elif op == "preference":
        rows = _spread(rng, 2, 512)
        lens = _draw_lens(rng, rows, _spread(rng, 2, 500000))
        pairs = [rng.sample(range(rows), 2) for _ in range(_spread(rng, 1, rows))]
        average = rng.random() < 0.3
        if average:
            lens = [max(1, n) for n in lens]
        lens[pairs[0][0]] += 1
        case.update(lens=",".join(map(str, lens)), pairs=",".join("%d-%d" % tuple(p) for p in pairs),
                    ref=rng.random() < 0.7, beta=rng.choice([0.05, 0.1, 0.5]),
                    kind=rng.choice(["sigmoid", "hinge", "ipo"]), smoothing=0.0, margin=0.0,
                    average=average)
        if case["kind"] == "sigmoid":
            case.update(smoothing=rng.choice([0.0, 0.1]), margin=rng.choice([0.0, 0.5]))
    else:
        count, total = _spread(rng, 1, 200), _spread(rng, 1, 50000000)
        sizes = [_spread(rng, 1, max(2, 2 * total // count)) for _ in range(count)]
        case.update(sizes=",".join(map(str, sizes)), types=rng.choice(["fp32", "fp16", "bf16", "mixed"]),
                    rms=round(math.exp(rng.uniform(math.log(2e-3), math.log(0.5))), 5),
                    max_norm=rng.choice([0.5, 1.0, 1000000.0]), scale=rng.choice([1.0, 1.0 / 1024]),
                    to_fp32=rng.random() < 0.5)
        if not case["to_fp32"] and case["types"] != "fp32":
            case["scale"] = 1.0       # 16-bit gradients stay scaled: unscaled they would underflow
    return case


def _ints(text):
    return [int(x) for x in str(text).split(",") if x != ""]


def _pairs(case):
    return [tuple(int(x) for x in p.split("-")) for p in str(case["pairs"]).split(",")]


def work(case):
    if case["op"] == "logprobs":
        n, v, d = case["n"], case["vocab"], case["hidden"]
        return {"bytes": 2 * d * (n + v) + 4 * n + 12 * n + (4 * n if case["total"] != n else 0),
                "flops": 2 * n * v * d}
    if case["op"] == "clip":
        # the gradients once (a second reading finds them in the caches, or does not), the scaled ones once
        sizes, types = _ints(case["sizes"]), _types(case)
        width = [4 if t == torch.float32 else 2 for t in types]
        read = sum(s * w for s, w in zip(sizes, width))
        written = 4 * sum(sizes) if case["to_fp32"] else read
        return {"bytes": read + written, "flops": 3 * sum(sizes)}
    lens = _ints(case["lens"])
    n, rows = sum(lens), len(lens)
    if case["op"] == "policy":
        per = 12 + (4 if case["ref"] else 0) + (4 if case["per_token"] else 0)
        return {"bytes": per * n + (0 if case["per_token"] else 4 * rows) + 16 * rows + 4, "flops": 12 * n}
    pairs = len(_pairs(case))
    return {"bytes": (12 if case["ref"] else 8) * n + 4 * rows + 12 * pairs + 4, "flops": 3 * n + 20 * pairs}


def _types(case):
    every = {"fp32": [torch.float32], "fp16": [torch.float16], "bf16": [torch.bfloat16],
             "mixed": [torch.float32, torch.float16, torch.bfloat16]}[case["types"]]
    return [every[i % len(every)] for i in range(len(_ints(case["sizes"])))]


def _inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)
    state = dict(case=case)
    if case["op"] == "logprobs":
        n, total, v, d = case["n"], case["total"], case["vocab"], case["hidden"]
        # hidden states of a trained model lean towards the row of the token that they predict
        emb = (randn(v, d) * (2.0 / math.sqrt(d))).half()
        tgt = torch.randint(0, v, (n,), generator=g, device=dev, dtype=torch.int32)
        rows = None
        if total != n:
            rows = torch.randperm(total, generator=g, device=dev)[:n].sort().values.to(torch.int32)
        y = randn(total, d)
        lean = torch.rand(n, 1, generator=g, device=dev) * 3.0
        y[rows.long() if rows is not None else slice(None)] += lean * emb[tgt.long()].float()
        state.update(y=y.half(), emb=emb, tgt=tgt, rows=rows)
    elif case["op"] == "clip":
        sizes, types = _ints(case["sizes"]), _types(case)
        # one buffer for each type, as buckets hold them; each gradient is a piece of its type's buffer
        buffers, grads, outs = {}, [], []
        for t in dict.fromkeys(types):
            size = sum(s for s, u in zip(sizes, types) if u == t)
            buffers[t] = (randn(size) * case["rms"]).to(t)
        at = dict.fromkeys(buffers, 0)
        out = torch.empty(sum(sizes), device=dev) if case["to_fp32"] else None
        first = 0
        for s, t in zip(sizes, types):
            grads.append(buffers[t][at[t]:at[t] + s])
            at[t] += s
            if out is not None:
                outs.append(out[first:first + s])
            first += s
        state.update(buffers=list(buffers.values()), grads=grads, out=out, outs=outs)
    else:
        lens = torch.tensor(_ints(case["lens"]), device=dev)
        n = int(lens.sum())
        # log-probabilities of sampled tokens: most near 0, a tail of rare ones
        old = -torch.empty(n, device=dev).exponential_(1.2, generator=g)
        ref = old + 0.1 * randn(n)
        logp = old + 0.15 * randn(n)
        row = torch.repeat_interleave(torch.arange(len(lens), device=dev), lens)
        state.update(lens=lens, row=row, logp=logp, old=old, ref=ref if case["ref"] else None)
        if case["op"] == "policy":
            state["adv"] = randn(n if case["per_token"] else len(lens))
            if case["stats"]:
                # the head's stats (loss, entropy, hit, lse), tokens without a target behind the others
                stats = torch.rand(n + 5, 4, generator=g, device=dev)
                stats[:n, 0] = -logp
                stats[n:] = 0.0
                state["logp"] = stats
        else:
            state["pairs"] = torch.tensor(_pairs(case), device=dev)
    return state


def prepare(case, seed):
    """The inputs, and for the losses the batch's plan, which a training program makes with the batch."""
    state = _inputs(case, seed)
    if own and case["op"] in ("policy", "preference"):
        from decentrik_prime_amd import k_loss
        pairs = _pairs(case) if case["op"] == "preference" else None
        state["meta"] = k_loss.row_meta(_ints(case["lens"]), state["lens"].device, pairs=pairs)
    return state


def _plain_logprobs(state):
    y, tgt, rows = state["y"], state["tgt"].long(), state["rows"]
    y = y if rows is None else y[rows.long()]
    x = y.float() @ state["emb"].float().t() * state["case"]["scale"]
    m = x.amax(1, keepdim=True)
    z = x - m
    e = z.exp()
    s = e.sum(1)
    logp = z.gather(1, tgt[:, None])[:, 0] - s.log()
    return logp, s.log() - (e * z).sum(1) / s, m[:, 0] + s.log()


def _row_sums(values, lens):
    """Sums over each row's tokens, in 64 bits."""
    total = torch.cat([lens.new_zeros(1, dtype=torch.float64), values.double().cumsum(0)])
    ends = lens.cumsum(0)
    return total[ends] - total[ends - lens]


def _plain_policy(state):
    case, row, lens = state["case"], state["row"], state["lens"]
    n = row.numel()
    logp = -state["logp"][:n, 0] if case["stats"] else state["logp"]
    a = state["adv"] if case["per_token"] else state["adv"][row]
    d = logp.double() - state["old"].double()
    clipped = torch.where(a > 0, d > math.log1p(case["high"]), (a < 0) & (d < math.log1p(-case["low"])))
    r = d.float().exp()
    bound = torch.where(a > 0, 1.0 + case["high"], 1.0 - case["low"])
    p = -torch.where(clipped, bound, r) * a
    grad = -torch.where(clipped, 0.0, r) * a
    k = torch.zeros_like(p)
    if case["ref"]:
        f = (state["ref"].double() - logp.double())
        k = (f.expm1() - f).float()
        grad = grad - case["kl"] * f.expm1().float()
    count = lens.double().clamp(min=1.0)
    w = {"row": 1.0 / (count * (lens > 0).sum()), "token": torch.full_like(count, 1.0 / n),
         "sum": torch.ones_like(count)}[case["reduction"]]
    sp, sk = _row_sums(p, lens), _row_sums(k, lens)
    loss = ((sp + case["kl"] * sk) * w).sum().float()
    stats = torch.stack([sp, sk, _row_sums(clipped, lens), _row_sums(r, lens)], 1) / count[:, None]
    return loss, grad * w.float()[row], stats.float()


def _plain_preference(state):
    case, row, lens, pairs = state["case"], state["row"], state["lens"], state["pairs"]
    beta = case["beta"]
    v = state["logp"].double() if state["ref"] is None else state["logp"].double() - state["ref"].double()
    share = 1.0 / lens.double() if case["average"] else torch.ones_like(lens, dtype=torch.float64)
    s = _row_sums(v, lens) * share
    h = beta * (s[pairs[:, 0]] - s[pairs[:, 1]]) - case["margin"]
    eps = case["smoothing"]
    if case["kind"] == "sigmoid":
        up, down = (-h).clamp(min=0) + (-h.abs()).exp().log1p(), h.clamp(min=0) + (-h.abs()).exp().log1p()
        loss = (1 - eps) * up + eps * down
        slope = 1.0 / (1.0 + (-h).exp()) - (1 - eps)
    elif case["kind"] == "hinge":
        loss, slope = (1 - h).clamp(min=0), -(h < 1).double()
    else:
        loss, slope = (h / beta - 0.5 / beta).square(), 2 * (h / beta - 0.5 / beta) / beta
    slope = slope * beta / pairs.shape[0]
    g = torch.zeros_like(s).index_add_(0, pairs[:, 0], slope).index_add_(0, pairs[:, 1], -slope)
    return loss.mean().float(), (g * share).float()[row], (beta * s).float(), h.float()


def _plain_clip(state):
    case, grads = state["case"], state["grads"]
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt() * case["scale"]
    factor = (case["scale"] * (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)).float()
    for g, o in zip(grads, state["outs"] or grads):
        o.copy_(g.float() * factor)
    return (norm.float(),) + ((state["out"],) if case["to_fp32"] else tuple(state["buffers"]))


def run(state):
    case = state["case"]
    if not own:
        return {"logprobs": _plain_logprobs, "policy": _plain_policy, "preference": _plain_preference,
                "clip": _plain_clip}[case["op"]](state)
    from decentrik_prime_amd import k_grad, k_head, k_loss
    if case["op"] == "logprobs":
        return k_head.token_logprobs(state["y"], state["emb"], state["tgt"], rows=state["rows"],
                                     scale=case["scale"])
    if case["op"] == "policy":
        return k_loss.policy_loss(state["logp"], state["old"], state["adv"], state["meta"], ref=state["ref"],
                                  kl_coef=case["kl"], clip_low=case["low"], clip_high=case["high"],
                                  reduction=case["reduction"], per_token=case["per_token"])
    if case["op"] == "preference":
        return k_loss.preference_loss(state["logp"], state["ref"], state["meta"], beta=case["beta"],
                                      kind=case["kind"], label_smoothing=case["smoothing"],
                                      margin=case["margin"], average=case["average"])
    norm = k_grad.clip_grads(state["grads"], case["max_norm"], scale=case["scale"],
                             out=state["outs"] if case["to_fp32"] else None)
    return (norm,) + ((state["out"],) if case["to_fp32"] else tuple(state["buffers"]))


def exact(case, seed):
    state = _inputs(case, seed)
    if case["op"] == "logprobs":
        y = state["y"].double()
        if state["rows"] is not None:
            y = y.index_select(0, state["rows"].long())
        logits = (y @ state["emb"].double().t()).mul_(case["scale"])
        lse = torch.logsumexp(logits, 1)
        chosen = logits[torch.arange(case["n"], device=y.device), state["tgt"].long()]
        logq = logits.sub_(lse[:, None])
        return chosen - lse, -(logq.exp() * logq).sum(1), lse
    if case["op"] == "clip":
        whole = torch.cat([b.double() for b in state["buffers"]])
        norm = torch.linalg.vector_norm(whole).item() * case["scale"]
        factor = case["scale"] * min(1.0, case["max_norm"] / (norm + 1e-6))
        norm = torch.tensor(norm, dtype=torch.float64)
        if not case["to_fp32"]:
            return (norm,) + tuple(b.double() * factor for b in state["buffers"])
        return norm, torch.cat([g.double() for g in state["grads"]]) * factor
    lens = _ints(case["lens"])
    n, dev = sum(lens), state["row"].device

    def row_sum(x):
        return torch.stack([piece.sum() for piece in x.split(lens)])
    filled = torch.tensor([max(1, x) for x in lens], dtype=torch.float64, device=dev)
    ref = None if state["ref"] is None else state["ref"].double()
    if case["op"] == "policy":
        x = (state["logp"][:n, 0].double().neg() if case["stats"] else state["logp"].double())
        x.requires_grad_(True)
        adv = state["adv"].double()
        if not case["per_token"]:
            adv = torch.repeat_interleave(adv, torch.tensor(lens, device=dev))
        ratio = torch.exp(x - state["old"].double())
        surrogate = torch.minimum(ratio * adv, ratio.clamp(1 - case["low"], 1 + case["high"]) * adv)
        kl = torch.zeros_like(x) if ref is None else torch.exp(ref - x) - (ref - x) - 1
        token = case["kl"] * kl - surrogate
        if case["reduction"] == "row":
            loss = (row_sum(token) / filled).sum() / max(1, sum(1 for k in lens if k))
        else:
            loss = token.sum() / (n if case["reduction"] == "token" else 1)
        (grad,) = torch.autograd.grad(loss, x)
        cut = (ratio * adv > ratio.clamp(1 - case["low"], 1 + case["high"]) * adv).double()
        stats = [row_sum(v.detach()) / filled for v in (-surrogate, kl, cut, ratio)]
        return loss.detach(), grad, torch.stack(stats, 1)
    x = state["logp"].double().requires_grad_(True)
    score = row_sum(x if ref is None else x - ref) / (filled if case["average"] else 1.0)
    pairs = _pairs(case)
    win, lose = (torch.tensor([p[i] for p in pairs], device=dev) for i in (0, 1))
    h = case["beta"] * (score[win] - score[lose]) - case["margin"]
    if case["kind"] == "sigmoid":
        each = -(1 - case["smoothing"]) * torch.nn.functional.logsigmoid(h) \
            - case["smoothing"] * torch.nn.functional.logsigmoid(-h)
    elif case["kind"] == "hinge":
        each = torch.relu(1 - h)
    else:
        each = (score[win] - score[lose] - 1 / (2 * case["beta"])) ** 2
    loss = each.mean()
    (grad,) = torch.autograd.grad(loss, x)
    return loss.detach(), grad, (case["beta"] * score).detach(), h.detach()
