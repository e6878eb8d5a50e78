"""Attention of the packed batch over part of the keys, forward and backward: a sliding window with
first tokens that stay visible (sinks), and groups of answers behind one shared prompt.

``run`` with ``own`` true makes the calls of decentrik_prime_amd.k_attn; with ``own`` false it
computes the same outputs in elementary torch operations in 32 bits, rounded once at the end.
``exact`` computes them from the definitions in 64 bits.

A window case has sequences of lengths ``lens``; query i of a sequence sees its keys j <= i with
i - j < window or j < sinks.  A prefix case has groups: a prompt of ``prompts[g]`` tokens followed by
``answers[g]`` (lengths); prompt tokens are causal, an answer's token sees the whole prompt and its own
answer up to itself.  lse is in log2 units.  kind "fwd" returns (out, lse); "train" a training step's
(out, lse, dq, dk, dv).
"""

import math

import torch

own = False

HD = 128
ROWS = 1024   # query rows per piece of the plain form


def listed():
    return [
        # a ragged batch of short rows: latency
        dict(name="window_fwd_short", op="window", kind="fwd", nq=12, nkv=2, lens="1,37,64,200",
             window=48, sinks=4),
        # an ordinary packed batch of 2048 tokens
        dict(name="window_train_packed", op="window", kind="train", nq=12, nkv=2,
             lens="853,612,401,182", window=256, sinks=4),
        # one long document, wide window, no gradient (evaluation)
        dict(name="window_fwd_long", op="window", kind="fwd", nq=12, nkv=2, lens="16384",
             window=4096, sinks=4),
        # long-context training of one document
        dict(name="window_train_long", op="window", kind="train", nq=12, nkv=2, lens="8192",
             window=1024, sinks=4),
        # a key head per query head, odd lengths, many sinks
        dict(name="window_train_mha", op="window", kind="train", nq=16, nkv=16, lens="4001,2500,1",
             window=511, sinks=65),
        # one answer token behind a prompt: the least work
        dict(name="prefix_fwd_one", op="prefix", kind="fwd", nq=12, nkv=2, prompts="0", answers="1"),
        # scoring of choices: one token each behind a long prompt
        dict(name="prefix_fwd_choices", op="prefix", kind="fwd", nq=12, nkv=2, prompts="8192",
             answers=",".join(["1"] * 64)),
        # eight sampled answers to a prompt, 2048 tokens in all
        dict(name="prefix_train_answers", op="prefix", kind="train", nq=12, nkv=2, prompts="1024",
             answers="128,97,160,33,255,128,95,128"),
        # several groups, one without a prompt, seven query heads per key head
        dict(name="prefix_train_groups", op="prefix", kind="train", nq=28, nkv=4,
             prompts="300,0,1500", answers="77,150,9;500;" + ",".join(["33"] * 10)),
        # sixteen long answers to a long prompt
        dict(name="prefix_train_long", op="prefix", kind="train", nq=12, nkv=2, prompts="4096",
             answers="512,500,512,471,512,512,640,512,384,512,513,511,512,512,512,575"),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], its logarithm evenly spread."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["window", "prefix"])
    nq, nkv = rng.choice([(12, 2), (16, 16), (28, 4), (8, 1), (14, 2), (6, 3)])
    case = dict(op=op, kind=rng.choice(["fwd", "train"]), nq=nq, nkv=nkv)
    if op == "window":
        total = _spread(rng, 1, 8192 if nq > 14 else 12288)
        cuts = sorted(rng.randint(0, total) for _ in range(rng.randint(0, 6)))
        lens = [b - a for a, b in zip([0] + cuts, cuts + [total])]
        case.update(lens=",".join(map(str, lens)), window=_spread(rng, 1, 4096),
                    sinks=rng.choice([0, 1, 4, rng.randint(2, 200)]))
    else:
        prompts, answers = [], []
        for _ in range(rng.randint(1, 3)):
            prompts.append(rng.choice([0, _spread(rng, 1, 2500), _spread(rng, 64, 2500)]))
            n = _spread(rng, 1, 40)
            size = _spread(rng, 1, max(1, 2500 // n))
            sizes = [max(0, size - rng.randint(0, max(1, size // 3))) for _ in range(n - 1)]
            answers.append(",".join(map(str, sizes + [size])))
        case.update(prompts=",".join(map(str, prompts)), answers=";".join(answers))
    return case


def _ints(text):
    return [int(x) for x in str(text).split(",") if x != ""]


def _groups(case):
    return [(p, _ints(a)) for p, a in zip(_ints(case["prompts"]), str(case["answers"]).split(";"))]


def _tokens(case):
    if case["op"] == "window":
        return sum(_ints(case["lens"]))
    return sum(p + sum(a) for p, a in _groups(case))


def _pairs(case):
    """Visible (query, key) pairs of one head."""
    if case["op"] == "prefix":
        return sum(p * (p + 1) // 2 + sum(a * (a + 1) // 2 + a * p for a in ans)
                   for p, ans in _groups(case))
    w, s, total = case["window"], case["sinks"], 0
    for n in _ints(case["lens"]):
        full = min(w, n)
        total += full * (full + 1) // 2 + (n - full) * w       # the window
        far = max(0, n - w)                                    # queries that have left key 0
        total += sum(max(0, far - j) for j in range(min(s, n)))
    return total


def work(case):
    n, nq, nkv = _tokens(case), case["nq"], case["nkv"]
    qkv, o, lse = 2 * n * (nq + 2 * nkv) * HD, 2 * n * nq * HD, 4 * n * nq
    flops = 4 * HD * nq * _pairs(case)
    total = qkv + o + lse
    if case["kind"] == "train":
        total += o + qkv                                       # dout in, dq, dk, dv out
        flops += 10 * HD * nq * _pairs(case)
    return {"bytes": total, "flops": flops}


def _inputs(case, seed):
    """The packed q|k|v rows as the projection leaves them (queries and keys share a direction that the
    first keys carry more of, as first tokens do), and dout for a training step."""
    n, nq, nkv = _tokens(case), case["nq"], case["nkv"]
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    qkv = torch.randn(n, nq + 2 * nkv, HD, generator=g, device=dev)
    mean = torch.randn(nkv, HD, generator=g, device=dev) * 0.4
    qkv[:, :nq] += mean.repeat_interleave(nq // nkv, 0)
    start = 0
    spans = _ints(case["lens"]) if case["op"] == "window" else [p + sum(a) for p, a in _groups(case)]
    for size in spans:
        qkv[start:start + min(4, size), nq:nq + nkv] += 1.5 * mean
        start += size
    qkv[:, nq + nkv:] *= 0.8
    state = dict(case=case, qkv=qkv.view(n, -1).half(), n=n)
    if case["kind"] == "train":
        state["dout"] = (torch.randn(n, nq * HD, generator=g, device=dev) * 0.1).half()
    return state


def prepare(case, seed):
    """The inputs and the batch's plan, which a training program keeps for all layers of a step."""
    state = _inputs(case, seed)
    nq, nkv, dev = case["nq"], case["nkv"], state["qkv"].device
    if own:
        from decentrik_prime_amd import k_attn
        if case["op"] == "window":
            state["meta"] = k_attn.window_meta(_ints(case["lens"]), case["window"], case["sinks"], nq,
                                               nkv, dev)
        else:
            state["meta"] = k_attn.prefix_meta(_groups(case), nq, nkv, dev)
    else:
        state["pieces"] = _pieces(case, dev)
    return state


def _pieces(case, dev):
    """The plain form's plan: per piece of query rows (first row, last row + 1, keys [n], visible [rows,
    n]); a piece's keys are its rows' window or own answers and the sinks or prompt before them."""
    out = []

    def piece(r0, r1, a0, a1, b0, kend):
        cols = torch.arange(a0, r1, device=dev) if b0 <= a1 else torch.cat(
            [torch.arange(a0, a1, device=dev), torch.arange(b0, r1, device=dev)])
        rows = torch.arange(r0, r1, device=dev)[:, None]
        out.append((r0, r1, cols, (cols[None] <= rows) & (rows < kend[cols][None])))

    n = _tokens(case)
    kend = torch.empty(n, dtype=torch.int64, device=dev)
    s0 = 0
    if case["op"] == "window":
        w, s = case["window"], case["sinks"]
        for size in _ints(case["lens"]):
            end = s0 + size
            kend[s0:end] = (torch.arange(s0, end, device=dev) + w).clamp(max=end)
            kend[s0:min(s0 + s, end)] = end
            for r0 in range(s0, end, ROWS):
                piece(r0, min(r0 + ROWS, end), s0, min(s0 + s, r0), max(s0, r0 - w + 1), kend)
            s0 = end
        return out
    for p, ans in _groups(case):
        kend[s0:s0 + p] = s0 + p + sum(ans)
        for r0 in range(s0, s0 + p, ROWS):
            piece(r0, min(r0 + ROWS, s0 + p), s0, s0, s0, kend)
        starts, b = [], s0 + p
        for a in ans:
            kend[b:b + a] = b + a
            starts.append(b)
            b += a
        for r0 in range(s0 + p, b, ROWS):
            piece(r0, min(r0 + ROWS, b), s0, s0 + p, max(x for x in starts if x <= r0), kend)
        s0 = b
    return out


def _heads(x, heads, gin):
    """[n, heads hd] -> fp32 [heads gin, n, hd], every head gin times."""
    return x.float().view(x.shape[0], heads, HD).transpose(0, 1).repeat_interleave(gin, 0)


def _plain(state):
    case, qkv, n = state["case"], state["qkv"], state["n"]
    nq, nkv = case["nq"], case["nkv"]
    gin, sm = nq // nkv, HD ** -0.5
    q = _heads(qkv[:, :nq * HD], nq, 1)
    k = _heads(qkv[:, nq * HD:(nq + nkv) * HD], nkv, gin)
    v = _heads(qkv[:, (nq + nkv) * HD:], nkv, gin)
    out, lse = torch.empty_like(q), torch.empty(nq, n, device=q.device)
    train = case["kind"] == "train"
    if train:
        do = _heads(state["dout"], nq, 1)
        dq, dk, dv = torch.empty_like(q), torch.zeros_like(q), torch.zeros_like(q)
    for r0, r1, cols, vis in state["pieces"]:
        kk, vv = k[:, cols], v[:, cols]
        s = (q[:, r0:r1] @ kk.transpose(1, 2) * sm).masked_fill_(~vis, -float("inf"))
        m = s.amax(2, keepdim=True)
        p = (s - m).exp_()
        l = p.sum(2, keepdim=True)
        p /= l
        o = p @ vv
        out[:, r0:r1] = o
        lse[:, r0:r1] = ((m + l.log()) / math.log(2.0))[..., 0]
        if not train:
            continue
        g = do[:, r0:r1]
        ds = (g @ vv.transpose(1, 2) - (o * g).sum(2, keepdim=True)) * p
        dq[:, r0:r1] = ds @ kk * sm
        dk[:, cols] += ds.transpose(1, 2) @ q[:, r0:r1] * sm
        dv[:, cols] += p.transpose(1, 2) @ g

    def rows(x, heads):
        x = x.view(heads, -1, n, HD).sum(1) if heads != nq else x
        return x.transpose(0, 1).reshape(n, heads * HD).half()
    if not train:
        return rows(out, nq), lse
    return rows(out, nq), lse, rows(dq, nq), rows(dk, nkv), rows(dv, nkv)


def run(state):
    if not own:
        return _plain(state)
    from decentrik_prime_amd import k_attn
    case = state["case"]
    args = (state["meta"], case["nq"], case["nkv"], HD)
    out, lse = k_attn.span_attention_forward(state["qkv"], *args)
    if case["kind"] == "fwd":
        return out, lse
    return (out, lse) + tuple(k_attn.span_attention_backward(state["qkv"], out, lse, state["dout"],
                                                             *args))


def exact(case, seed):
    """The definition in 64 bits, one sequence (or one answer with its prompt) at a time."""
    state = _inputs(case, seed)
    n, nq, nkv = state["n"], case["nq"], case["nkv"]
    gin = nq // nkv
    x = state["qkv"].double().view(n, nq + 2 * nkv, HD)
    train = case["kind"] == "train"
    go = state["dout"].double().view(n, nq, HD) if train else None
    out = torch.zeros(n, nq, HD, dtype=torch.float64, device=x.device)
    lse = torch.zeros(nq, n, dtype=torch.float64, device=x.device)
    grad = torch.zeros_like(x)

    def attend(rows, keys, visible):
        """Query rows (a slice) over the key rows (an index) with visible [rows, keys]."""
        for h in range(nq):
            j = nq + h // gin
            qh, kh, vh = x[rows, h], x[keys, j], x[keys, j + nkv]
            s = (qh @ kh.t()) / math.sqrt(HD)
            s = torch.where(visible, s, torch.full_like(s, -float("inf")))
            z = torch.logsumexp(s, 1)
            lse[h, rows] = z / math.log(2.0)
            p = torch.exp(s - z[:, None])
            out[rows, h] = p @ vh
            if train:
                gh = go[rows, h]
                dp = gh @ vh.t()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(HD)
                grad[rows, h] = ds @ kh
                grad[:, j].index_add_(0, keys, ds.t() @ qh)
                grad[:, j + nkv].index_add_(0, keys, p.t() @ gh)

    def positions(lo, hi):
        return torch.arange(lo, hi, device=x.device)

    s0 = 0
    if case["op"] == "window":
        for size in _ints(case["lens"]):
            for i0 in range(0, size, 2048):
                i1 = min(i0 + 2048, size)
                i, j = positions(i0, i1)[:, None], positions(0, i1)[None]
                attend(slice(s0 + i0, s0 + i1), s0 + positions(0, i1),
                       (j <= i) & ((i - j < case["window"]) | (j < case["sinks"])))
            s0 += size
    else:
        for p, ans in _groups(case):
            prompt = s0 + positions(0, p)
            for size, first, before in [(p, s0, 0)] + [
                    (a, s0 + p + sum(ans[:b]), p) for b, a in enumerate(ans)]:
                i = positions(0, size)[:, None]
                j = positions(0, before + size)[None] - before
                if size:
                    attend(slice(first, first + size),
                           torch.cat([prompt[:before], first + positions(0, size)]), j <= i)
            s0 += p + sum(ans)
    result = (out.view(n, -1), lse)
    if train:
        result += (grad[:, :nq].reshape(n, -1), grad[:, nq:nq + nkv].reshape(n, -1),
                   grad[:, nq + nkv:].reshape(n, -1))
    return result
