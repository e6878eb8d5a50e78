"""A whole Qwen2.5 QLoRA training step of the packed batch on this package's kernels.

The linear stack (stack.NF4LinearStack: NF4 weights, LoRA adapters and keep-masks, the dequant
slot and its dequant schedule) with everything around it, in the order of the reference's
FastQwen2.forward / backward (solution/fast_qwen.py:985-1390):
  forward   x_0 = E[ids] (fp32 residual stream)
            per layer: y = RMSNorm(x_i) (+ the previous MLP output added on the way, x_i kept),
            xq, xv = fp16(dropout(y)) of the fp32 y, z_q, z_v = LoRA-down(xq, xv), qkv = y W_qkv^T + b + LoRA-up, rotated (one GEMM),
            attention, o = out W_o^T, y2 = RMSNorm(x_i + o), act, gu = SwiGLU(y2 W_gu^T),
            d = act W_d^T
            y_f = RMSNorm(x_L + d), LM head over vocabulary chunks: loss, stats, d(y_f)
  backward  final norm, then per layer: down^T + SwiGLU', gate|up^T dX, norm 2 (residual in
            place), o^T, attention, QKV epilogue backward (rotation^T, GQA sums), q+v LoRA
            gradients, q|k|v^T with the masked LoRA input terms (fp32), norm 1 (layer 0 only its
            LoRA gradients, as the reference)
Every activation the backward needs is kept in HBM (about 120 MB per layer at 2048 tokens): the
reference's host arenas, recompute plans and offload options exist for a 16 GB card and are not
built.  Weights are random (W ~ N(0, 0.02) NF4, norm weights near 1, embedding ~ N(0, 0.02));
the tokens and targets are random ids, each sequence's targets its next token (-1 at its end).

``window`` (and ``sinks``) or ``groups`` select k_attn's attention over part of the keys in place of
causal attention: a sliding window in every layer, or answers behind shared prompts.

``policy_step`` and ``preference_step`` train on k_loss's losses over the tokens' log-probabilities in
place of cross entropy, ``score`` gives the log-probabilities that they compare with, and ``clip_grads``
bounds the gradients' global norm.
"""

import torch

from . import k_attn, k_grad, k_head, k_loss, k_norm, k_rope
from .stack import D, KV, NF4LinearStack, layer_flops
from .w4linear import (down_swiglu_backward, gateup_swiglu_forward, linear_backward_dx,
                       linear_backward_dx_lora, linear_forward, linear_forward_rope,
                       lora_down_multi, lora_dz_multi, lora_grads_multi)

NQ, NKV, HD = 12, 2, 128
VOCAB = 151936


def rope_tables(positions, hd=HD, theta=1.0e6, device="cuda"):
    """cos/sin [positions, hd] fp32 as Qwen2's rotary embedding builds them (angles p theta^(-2i/hd),
    the half-width table repeated)."""
    inv = 1.0 / (theta ** (torch.arange(0, hd, 2, dtype=torch.float32, device=device) / hd))
    fr = torch.arange(positions, dtype=torch.float32, device=device)[:, None] * inv[None, :]
    emb = torch.cat((fr, fr), 1)
    return emb.cos().contiguous(), emb.sin().contiguous()


class QwenQLoRAStep(NF4LinearStack):
    """Random-init Qwen2.5-1.5B (n_layers decoder layers, the LM head over `vocab`) with rank-16
    LoRA on q and v, one packed batch of sequences of lengths `lens`.  window, sinks: causal attention
    inside a sliding window and to a sequence's first tokens (k_attn.window_meta).  groups: the batch is
    groups (prompt length, [answer lengths]) in place of sequences (k_attn.prefix_meta; lens is None)."""

    def __init__(self, lens, n_layers=28, vocab=VOCAB, seed=0, device="cuda", eps=1e-6,
                 head_grad_scale=1024.0, head_chunk=k_head.CHUNK, ahead="layer", window=None, sinks=0,
                 groups=None):
        if (lens is None) == (groups is None):
            raise ValueError("either lens or groups")
        if groups is not None:
            if window is not None:
                raise ValueError("a window over groups is not supported")
            lens = [n for prompt, answers in groups for n in (prompt, *answers)]
        if sinks and window is None:
            raise ValueError("sinks need a window")
        m = int(sum(lens))
        super().__init__(n_layers, m, seed=seed, device=device, ahead=ahead)
        dev, f16, f32 = self.device, torch.float16, torch.float32
        self.lens, self.eps, self.head_grad_scale = list(lens), float(eps), float(head_grad_scale)
        gen = torch.Generator(device=dev)
        gen.manual_seed(seed + 1)

        def norm_w():
            return (1.0 + 0.1 * torch.randn(D, generator=gen, device=dev)).contiguous()
        self.w_in = [norm_w() for _ in range(n_layers)]
        self.w_post = [norm_w() for _ in range(n_layers)]
        self.w_final = norm_w()
        if groups is not None:
            self.meta = k_attn.prefix_meta(groups, NQ, NKV, dev)
        elif window is not None:
            self.meta = k_attn.window_meta(lens, window, sinks, NQ, NKV, dev)
        else:
            self.meta = k_attn.meta_for(lens, dev)
        self.span = isinstance(self.meta, k_attn.SpanMeta)
        if self.span:
            self.pos = self.meta.positions
            positions = int(self.pos.max()) + 1
        else:
            self.pos = torch.cat([torch.arange(n, dtype=torch.int32, device=dev) for n in lens])
            positions = max(lens)
        self.cos, self.sin = rope_tables(positions, device=dev)
        # embedding, tokens and next-token targets (sorted: rows with a target first)
        self.emb = (torch.randn(vocab, D, generator=gen, device=dev) * 0.02).half()
        ids = torch.randint(0, vocab, (m,), generator=gen, device=dev)
        tgt = torch.cat([ids[1:], ids[:1]])
        ends = torch.cumsum(torch.tensor(lens, device=dev), 0) - 1
        tgt[ends] = -1
        self.source = k_head.ResidentEmbedding(self.emb, head_chunk)
        self.use_tokens(ids, tgt)
        # activations kept for the backward, per layer
        L = n_layers
        self.xin = [self.x0] + [torch.empty(m, D, dtype=f32, device=dev) for _ in range(L - 1)]
        self.y16 = [torch.empty(m, D, dtype=f16, device=dev) for _ in range(L)]
        # the LoRA inputs: fp16(dropout(y)) of the fp32 norm output, per adapter
        self.xq = [torch.empty(m, D, dtype=f16, device=dev) for _ in range(L)]
        self.xv = [torch.empty(m, D, dtype=f16, device=dev) for _ in range(L)]
        self.qkv_b = [torch.empty(m, (NQ + 2 * NKV) * HD, dtype=f16, device=dev) for _ in range(L)]
        self.att = [None] * L
        self.lse = [None] * L
        self.op = [torch.empty(m, D, dtype=f16, device=dev) for _ in range(L)]
        self.d16 = [torch.empty(m, D, dtype=f16, device=dev) for _ in range(L)]
        self.rstd1 = [torch.empty(m, dtype=f32, device=dev) for _ in range(L)]
        self.rstd2 = [torch.empty(m, dtype=f32, device=dev) for _ in range(L)]
        # per-step scratch
        self.y2 = torch.empty(m, D, dtype=f16, device=dev)
        self.h1 = torch.empty(m, D, dtype=f32, device=dev)
        self.hf = torch.empty(m, D, dtype=f32, device=dev)
        self.yf = torch.empty(m, D, dtype=f16, device=dev)
        self.rstd_f = torch.empty(m, dtype=f32, device=dev)
        self.dh = torch.empty(m, D, dtype=f32, device=dev)
        self.dh16 = torch.empty(m, D, dtype=f16, device=dev)
        self.dy2 = torch.empty(m, D, dtype=f16, device=dev)
        self.dout = torch.empty(m, NQ * HD, dtype=f16, device=dev)
        self.dx32 = torch.empty(m, D, dtype=f32, device=dev)
        self.one = torch.ones(1, dtype=f32, device=dev)

    @classmethod
    def for_batch(cls, batch, **kwargs):
        """The step on the tokens of a packed batch (trainer.pack): its rows' lengths, token ids
        and next-token targets; the weights are random-init as for any instance."""
        st = cls(None if batch.groups else batch.lens, groups=batch.groups, **kwargs)
        st.use_tokens(batch.ids, batch.tgt)
        return st

    def use_tokens(self, ids, tgt):
        """Token ids [m] and next-token targets [m] (-1: none), in token order: the embedding rows
        the first layer reads, and the head's targets in sorted order (tokens with a target
        first, the order trainer.pack's perm gives)."""
        dev = self.device
        ids = torch.as_tensor(ids, device=dev).long()
        tgt = torch.as_tensor(tgt, device=dev).to(torch.int32)
        if ids.shape != (self.m,) or tgt.shape != (self.m,):
            raise ValueError(f"ids and targets must be [{self.m}] (the step's token count)")
        self.x0 = self.emb.index_select(0, ids).float()
        if hasattr(self, "xin"):
            self.xin[0] = self.x0
        has = tgt >= 0
        self.perm = torch.cat([torch.nonzero(has)[:, 0], torch.nonzero(~has)[:, 0]]).to(torch.int32)
        self.tgt_sorted = tgt.index_select(0, self.perm.long()).contiguous()
        self.n_lab = int(has.sum())
        self.labelled = self.perm[:self.n_lab].long()
        self.e_target = self.emb.index_select(0, self.tgt_sorted[:self.n_lab].long()).contiguous()
        self.tgt = tgt

    @property
    def flops_per_step(self):
        """Algorithmic FLOPs: the linear layers, the causal attention (2 hd L(L+1) per sequence and
        head forward, 2.5 times that backward), the LM head (logits and P E, 2 M V D each)."""
        pairs = self.meta.n_pairs if self.span else sum(n * (n + 1) // 2 for n in self.lens)
        att = 4 * HD * pairs * NQ * 3.5
        return self.n_layers * (layer_flops(self.m) + att) + 2 * 2 * self.m * self.emb.shape[0] * D

    def forward(self):
        """Returns (loss_sum, stats [N, 4] in sorted order, d(y_f) [N, D] fp16)."""
        self._pass = getattr(self, "_pass", 0) + 1
        self._forward = True
        w16, side, done = self._w16, self._side, self._done
        x, d_prev = self.x0, None
        for i in range(self.n_layers):
            Lw, lo, z = self.layers[i], self.lora[i], self.z[i]
            # norm 1 with the previous layer's MLP output added on the way (x_i materialised), and
            # the two LoRA inputs dropped out from its fp32 output (solution/k_norm.py:49-53)
            k_norm.rms_forward(x, self.w_in[i], self.y16[i], self.rstd1[i], self.eps, delta=d_prev,
                               xout=self.xin[i] if d_prev is not None else None,
                               xq=self.xq[i], xv=self.xv[i], mq=lo["mq"], mv=lo["mv"],
                               keep_scale=self.keep_scale)
            y = self.y16[i]
            self._lora_downs(i, lambda dq: lora_down_multi(
                None, [(lo["Aq"], None, 1.0, self.xq[i]), (lo["Av"], None, 1.0, self.xv[i])],
                outs=[z["q"], z["v"]], dequant=dq))
            linear_forward_rope(y, Lw["qkv"], lo["bias"], self.qkv_terms(i), self.pos, self.cos,
                                self.sin, (NQ + NKV) * HD, out=self.qkv_b[i], w16=w16("qkv", i),
                                side=side("qkv", i + 1))
            done("qkv", i + 1)
            attend = k_attn.span_attention_forward if self.span else k_attn.attention_forward
            self.att[i], self.lse[i] = attend(self.qkv_b[i], self.meta, NQ, NKV, HD)
            linear_forward(self.att[i], Lw["o"], out=self.op[i], w16=w16("o", i), side=side("o", i + 1))
            done("o", i + 1)
            k_norm.rms_forward(self.xin[i], self.w_post[i], self.y2, self.rstd2[i], self.eps,
                               delta=self.op[i], xout=self.h1)
            gateup_swiglu_forward(self.y2, Lw["gu"], act=self.act, gu=self.gu[i], w16=w16("gu", i),
                                  side=side("gu", i + 1))
            done("gu", i + 1)
            linear_forward(self.act, Lw["d"], out=self.d16[i], w16=w16("d", i), side=side("d", i + 1))
            done("d", i + 1)
            x, d_prev = self.h1, self.d16[i]
        k_norm.rms_forward(x, self.w_final, self.yf, self.rstd_f, self.eps, delta=d_prev,
                           xout=self.hf)
        return k_head.streamed_head(self.yf, self.source, self.tgt_sorted, self.perm, self.n_lab,
                                    self.e_target, self.head_grad_scale)

    def backward(self, dy_head, g_loss=1.0, dlogp=None):
        """LoRA gradients of g_loss * loss_sum: self.grads[i] = (dA_q, dB_q, dA_v, dB_v) fp32.  dlogp [n_lab]
        (fp32, sorted order): of g_loss * a loss with this gradient for the tokens' log-probabilities
        instead (loss_sum's is -1 each); dlogp may be of any size, and g_loss is a factor in fp32 there."""
        dh, dh16 = self.dh, self.dh16
        row_scale, up = None, float(g_loss)
        if dlogp is not None:
            if dlogp.dtype != torch.float32 or tuple(dlogp.shape) != (self.n_lab,) or dlogp.device != dh.device:
                raise ValueError(f"dlogp must be fp32 [{self.n_lab}] (the tokens with a target) on {dh.device}")
            # the gradients between here and the adapters' are fp16: the largest factor is 1 to 2, and the
            # adapters' fp32 gradients get the rest
            row_scale, unit = k_loss.row_factors(dlogp, self.perm[:self.n_lab], self.m)
            up = 1.0
        self._pass = getattr(self, "_pass", 0) + 1
        self._forward = False
        w16, side, done = self._w16, self._side, self._done
        gscale = torch.full((1,), up / self.head_grad_scale, dtype=torch.float32, device=self.device)
        k_norm.rms_backward(dy_head, gscale, self.hf, self.w_final, self.rstd_f, dh, out16=dh16,
                            row_scale=row_scale)
        ks = self.keep_scale
        for i in reversed(range(self.n_layers)):
            Lw, lo, z = self.layers[i], self.lora[i], self.z[i]
            down_swiglu_backward(dh16, Lw["d"], self.gu[i], w16=w16("d", i), side=side("d", i - 1))
            done("d", i - 1)
            linear_backward_dx(self.gu[i], Lw["gu"], out=self.dy2, out_dtype=torch.float16,
                               w16=w16("gu", i), side=side("gu", i - 1))
            done("gu", i - 1)
            # norm 2: its input x_i + o rebuilt in registers; the residual gradient in place
            k_norm.rms_backward(self.dy2, self.one, self.xin[i], self.w_post[i], self.rstd2[i], dh,
                                dres=dh, out16=dh16, delta=self.op[i])
            linear_backward_dx(dh16, Lw["o"], out=self.dout, out_dtype=torch.float16,
                               w16=w16("o", i), side=side("o", i - 1))
            done("o", i - 1)
            attend = k_attn.span_attention_backward if self.span else k_attn.attention_backward
            dq, dkp, dvp = attend(self.qkv_b[i], self.att[i], self.lse[i], self.dout, self.meta, NQ,
                                  NKV, HD)
            dqkv = self.qkv_b[i]      # the QKV epilogue backward writes d(qkv) over the forward's qkv
            k_rope.qkv_epilogue_backward(dq, dkp, dvp, self.pos, self.cos, self.sin, dqkv, NQ, NKV,
                                         HD, 1 if self.span else NQ // NKV)
            del dq, dkp, dvp
            terms = [(dqkv[:, :D], z["q"], lo["Bq"], self.s, None, 1.0, self.xq[i]),
                     (dqkv[:, D + KV:], z["v"], lo["Bv"], self.s, None, 1.0, self.xv[i])]
            w16q = w16("qkv", i) if i > 0 else None
            sums = None
            if w16q is not None:
                # dz now; the q|k|v dX launch carries the column sums (dA, dB) on its idle CUs
                sums = lora_dz_multi(None, terms)
                (daq, dbq, dzq), (dav, dbv, dzv) = sums.grads
            else:
                (daq, dbq, dzq), (dav, dbv, dzv) = lora_grads_multi(None, terms)
            if i > 0:
                # d(y) = dqkv W_qkv + the masked LoRA input terms, in fp32, into norm 1's backward
                linear_backward_dx_lora(dqkv, Lw["qkv"], [(dzq, lo["Aq"], lo["mq"], ks),
                                                          (dzv, lo["Av"], lo["mv"], ks)],
                                        out=self.dx32, w16=w16q, side=side("qkv", i - 1),
                                        sums=sums)
                done("qkv", i - 1)
                k_norm.rms_backward(self.dx32, self.one, self.xin[i], self.w_in[i], self.rstd1[i],
                                    dh, dres=dh, out16=dh16)
            self.grads[i] = (daq, dbq, dav, dbv)
        if dlogp is not None:
            k_grad.scale_grads([g for layer in self.grads for g in layer], unit, scale=float(g_loss))
        return self.grads

    def step(self):
        loss, stats, dy_head = self.forward()
        self.backward(dy_head)
        return loss

    def score(self, adapters=True, scale=1.0):
        """(logp, entropy) fp32 [n_lab] of the batch's targets in sorted order, without dropout: under the
        adapters (a policy's scores of its own samples) or, with adapters False, under the frozen weights
        alone (the reference).  scale: a factor of the logits (1 / temperature); the training steps have none,
        their old and ref are scores at scale 1.  The logits are summed in fp32, where forward()'s stats
        round them to fp16.  What a pending backward() reads stays as it is."""
        self._pass = getattr(self, "_pass", 0) + 1
        self._forward = True
        dev, f16, f32 = self.device, torch.float16, torch.float32
        w16, side, done, m = self._w16, self._side, self._done, self.m
        attend = k_attn.span_attention_forward if self.span else k_attn.attention_forward
        x, xsum, h = self.x0, torch.empty(m, D, dtype=f32, device=dev), torch.empty(m, D, dtype=f32, device=dev)
        y, op, d16 = (torch.empty(m, D, dtype=f16, device=dev) for _ in range(3))
        qkv = torch.empty(m, (NQ + 2 * NKV) * HD, dtype=f16, device=dev)
        act = torch.empty_like(self.act)
        rstd = torch.empty(m, dtype=f32, device=dev)
        z = [torch.empty_like(self.z[0][t]) for t in ("q", "v")]
        d_prev = None
        for i in range(self.n_layers):
            Lw, lo = self.layers[i], self.lora[i]
            k_norm.rms_forward(x, self.w_in[i], y, rstd, self.eps, delta=d_prev,
                               xout=xsum if d_prev is not None else None)
            x = x if d_prev is None else xsum
            terms = []
            if adapters:
                self._lora_downs(i, lambda dq: lora_down_multi(
                    y, [(lo["Aq"], None, 1.0), (lo["Av"], None, 1.0)], outs=z, dequant=dq))
                terms = [(z[0], lo["Bq"], 0, D, self.s), (z[1], lo["Bv"], D + KV, D + 2 * KV, self.s)]
            else:
                self._deferred = None     # (a dequant that waits for the downs: w16 below runs it)
            linear_forward_rope(y, Lw["qkv"], lo["bias"], terms, self.pos, self.cos, self.sin,
                                (NQ + NKV) * HD, out=qkv, w16=w16("qkv", i), side=side("qkv", i + 1))
            done("qkv", i + 1)
            att, _ = attend(qkv, self.meta, NQ, NKV, HD)
            linear_forward(att, Lw["o"], out=op, w16=w16("o", i), side=side("o", i + 1))
            done("o", i + 1)
            k_norm.rms_forward(x, self.w_post[i], y, rstd, self.eps, delta=op, xout=h)
            gateup_swiglu_forward(y, Lw["gu"], act=act, save_gu=False, w16=w16("gu", i),
                                  side=side("gu", i + 1))
            done("gu", i + 1)
            linear_forward(act, Lw["d"], out=d16, w16=w16("d", i), side=side("d", i + 1))
            done("d", i + 1)
            x, d_prev = h, d16
        k_norm.rms_forward(x, self.w_final, y, rstd, self.eps, delta=d_prev)
        logp, entropy, _ = k_head.token_logprobs(y, self.source, self.tgt_sorted[:self.n_lab],
                                                 rows=self.perm[:self.n_lab], scale=scale)
        return logp, entropy

    def _check_rows(self, meta):
        if meta.n_tokens != self.n_lab:
            raise ValueError(f"the plan has {meta.n_tokens} tokens, the batch {self.n_lab} with a target")

    def policy_step(self, meta, old, advantages, *, ref=None, g_loss=1.0, **options):
        """A training step on the clipped policy loss: meta the plan of the batch's answers
        (k_loss.row_meta(trainer.answer_lens(batch), ...)), old (and ref) log-probabilities in sorted order
        (score() at scale 1, or the head's stats of an earlier forward()), options as k_loss.policy_loss.  The
        current log-probabilities are the head's, from logits rounded to fp16 (2^-11 of a logit).  Returns
        (loss, its stats per answer, the head's stats); the gradients of g_loss * loss are in self.grads."""
        self._check_rows(meta)
        _, stats, dy = self.forward()
        loss, dlogp, rows = k_loss.policy_loss(stats, old, advantages, meta, ref=ref, **options)
        self.backward(dy, g_loss, dlogp=dlogp)
        return loss, rows, stats

    def preference_step(self, meta, ref, *, g_loss=1.0, **options):
        """A training step on the preference loss over meta's pairs of answers (options as
        k_loss.preference_loss; ref, as for policy_step, None: without a reference).  Returns (loss, rewards,
        margins, the head's stats); the gradients of g_loss * loss are in self.grads."""
        self._check_rows(meta)
        _, stats, dy = self.forward()
        loss, dlogp, rewards, margins = k_loss.preference_loss(stats, ref, meta, **options)
        self.backward(dy, g_loss, dlogp=dlogp)
        return loss, rewards, margins, stats

    def clip_grads(self, max_norm):
        """Scales self.grads in place to a global norm of at most max_norm; returns the norm before."""
        if any(layer is None for layer in self.grads):
            raise ValueError("no gradients yet (backward)")
        return k_grad.clip_grads([g for layer in self.grads for g in layer], max_norm)
