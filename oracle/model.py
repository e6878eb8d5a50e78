"""CPU float64 reference of a whole Qwen2 QLoRA step (torch autograd), the end-to-end check of
decentrik_prime_amd.model.  TEST INFRASTRUCTURE ONLY: imported by tests/ only, never by the
product path.

The Qwen2 decoder as Hugging Face's modelling code defines it, with the reference's LoRA on q and
v (solution/fast_qwen.py:940-952, 985-1140): per layer
    y = w_in * x * rsqrt(mean(x^2) + eps)
    q|k|v = y W_qkv^T + b, q += s (dropout(y) A_q^T) B_q^T, v += s (dropout(y) A_v^T) B_v^T
    q, k rotated (rotate-half, cos/sin of each token's position in its sequence)
    out = causal softmax(q k^T / sqrt(hd)) v per sequence, key/value head h // (nq / nkv)
    h = x + out W_o^T;  y2 = w_post * RMSNorm(h);  x' = h + (silu(y2 W_g^T) * (y2 W_u^T)) W_d^T
then y_f = w_final * RMSNorm(x_L), logits = y_f E^T, loss = sum of the rows' cross-entropy (rows
with a target), and the LoRA gradients of that loss.  Exact arithmetic here (float64 from the
fp16 weights and inputs): the kernels' fp16 roundings are what the comparison's tolerance covers.
"""

import math

import torch


def qwen_step(p, lens, nq=12, nkv=2, hd=128, visible=None, weights=None):
    """p: CPU tensors x0 [n, D] fp32, emb [V, D], tgt [n] (-1 = none), pos [n], cos / sin
    [positions, hd], w_final [D], eps, ks (dropout keep scale), s (LoRA scale), and layers: dicts
    of wqkv [(nq + 2 nkv) hd, D], bias, wo [D, nq hd], wgu [2 I, D] (gate rows, then up rows),
    wd [D, I], w_in, w_post [D], Aq [r, D], Bq [nq hd, r], Av [r, D], Bv [nkv hd, r], mq / mv
    [n, D] (nonzero = keep).  visible [n, n] bool: the keys that each query sees, in place of causal
    attention inside sequences of lengths lens.  weights [n]: factors of the tokens' cross entropies (1).
    Returns (loss_sum, [(dA_q, dB_q, dA_v, dB_v) per layer])."""
    dt = torch.float64
    eps, ks, s = float(p["eps"]), float(p["ks"]), float(p["s"])
    n = p["x0"].shape[0]
    g = nq // nkv
    half = hd // 2
    c = p["cos"].to(dt)[p["pos"].long(), :half][:, None, :]
    sn = p["sin"].to(dt)[p["pos"].long(), :half][:, None, :]

    def rms(h, w):
        return w.to(dt) * (h * torch.rsqrt((h * h).mean(-1, keepdim=True) + eps))

    def rope(x):
        x1, x2 = x[..., :half], x[..., half:]
        return torch.cat((x1 * c - x2 * sn, x2 * c + x1 * sn), -1)

    x = p["x0"].to(dt)
    params = []
    for L in p["layers"]:
        A = {k: L[k].to(dt).clone().requires_grad_(True) for k in ("Aq", "Bq", "Av", "Bv")}
        params.append(A)
        y = rms(x, L["w_in"])
        qd = nq * hd
        kvd = nkv * hd
        qkv = y @ L["wqkv"].to(dt).T + L["bias"].to(dt)
        xq = y * (L["mq"] != 0).to(dt) * ks
        xv = y * (L["mv"] != 0).to(dt) * ks
        q = qkv[:, :qd] + s * ((xq @ A["Aq"].T) @ A["Bq"].T)
        k = qkv[:, qd:qd + kvd]
        v = qkv[:, qd + kvd:] + s * ((xv @ A["Av"].T) @ A["Bv"].T)
        q = rope(q.view(n, nq, hd))
        k = rope(k.view(n, nkv, hd))
        v = v.view(n, nkv, hd)
        outs, s0 = [], 0
        for ln in ([n] if visible is not None else lens):
            sl = slice(s0, s0 + ln)
            qq = q[sl].transpose(0, 1)
            kk = k[sl].transpose(0, 1).repeat_interleave(g, 0)
            vv = v[sl].transpose(0, 1).repeat_interleave(g, 0)
            o = torch.nn.functional.scaled_dot_product_attention(
                qq[None], kk[None], vv[None], visible, is_causal=visible is None,
                scale=1.0 / math.sqrt(hd))[0]
            outs.append(o.transpose(0, 1).reshape(ln, qd))
            s0 += ln
        h = x + torch.cat(outs) @ L["wo"].to(dt).T
        y2 = rms(h, L["w_post"])
        gu = y2 @ L["wgu"].to(dt).T
        inter = gu.shape[1] // 2
        act = torch.nn.functional.silu(gu[:, :inter]) * gu[:, inter:]
        x = h + act @ L["wd"].to(dt).T
    yf = rms(x, p["w_final"])
    logits = yf @ p["emb"].to(dt).T
    tgt = p["tgt"].long()
    valid = tgt >= 0
    each = torch.nn.functional.cross_entropy(logits[valid], tgt[valid], reduction="none")
    loss = each.sum() if weights is None else (each * weights.to(dt)[valid]).sum()
    loss.backward()
    return float(loss.detach()), [tuple(A[k].grad for k in ("Aq", "Bq", "Av", "Bv")) for A in params]
