"""End-to-end parity of the whole QLoRA step (decentrik_prime_amd.model: norms, the rotary q|k|v
GEMM with the LoRA terms, attention, o, SwiGLU MLP, the LM head, and the backward through all of
it) with the float64 torch reference (oracle/model.py) on the same weights: two layers, a
4096-token vocabulary in chunks of 1024; three ragged sequences (the small-M GEMM plans) and four
512-token sequences (M = 2048: the 256-tile GEMM plans of the bench).  The weights the reference uses are the
GPU's own NF4 dequant (bit-exact to the oracle, pinned in tests/test_gpu_nf4.py)."""

import numpy as np
import pytest

from tests.helpers import host, log

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    return t


@pytest.mark.parametrize("lens", [[37, 100, 64], [512, 512, 512, 512]])
def test_qlora_step_matches_float64_reference(torch, lens):
    from decentrik_prime_amd import k_nf4, model
    from oracle import model as ref
    log(f"whole QLoRA step, 2 layers, lens {lens}")
    st = model.QwenQLoRAStep(lens, n_layers=2, vocab=4096, seed=5, head_chunk=1024)
    loss = st.step()
    loss2 = st.step()             # a second step over the same batch: the schedule's steady state
    torch.cuda.synchronize()
    assert float(loss) == float(loss2), "the step is deterministic"
    layers = []
    for i in range(2):
        pk = st.layers[i]["packed"]
        buf = torch.empty(pk.numel, dtype=torch.float16, device="cuda")
        k_nf4.dequant_layer(pk, st.code2, st.nf4, buf)

        def w(kind):
            start, n = st.views[kind]
            W = st.layers[i][kind]
            return buf[start:start + n].view(W.rows, W.cols).cpu()
        lo = st.lora[i]
        layers.append(dict(wqkv=w("qkv"), wo=w("o"), wgu=w("gu"), wd=w("d"), bias=lo["bias"].cpu(),
                           w_in=st.w_in[i].cpu(), w_post=st.w_post[i].cpu(),
                           **{k: lo[k].cpu() for k in ("Aq", "Bq", "Av", "Bv", "mq", "mv")}))
    p = dict(x0=st.x0.cpu(), emb=st.emb.cpu(), tgt=st.tgt.cpu(), pos=st.pos.cpu(), cos=st.cos.cpu(),
             sin=st.sin.cpu(), w_final=st.w_final.cpu(), eps=st.eps, ks=st.keep_scale, s=st.s,
             layers=layers)
    ref_loss, ref_grads = ref.qwen_step(p, lens)
    # measured: loss to ~1e-5 relative, gradients to ~2e-3 of their maximum, at both sizes
    assert abs(float(loss) - ref_loss) <= 1e-4 * abs(ref_loss), (float(loss), ref_loss)
    errs = []
    for i in range(2):
        for nm, got, want in zip(("dA_q", "dB_q", "dA_v", "dB_v"), st.grads[i], ref_grads[i]):
            g, r = host(got).astype(np.float64), want.numpy()
            scale = float(np.abs(r).max())
            err = float(np.abs(g - r).max()) / scale
            errs.append(err)
            assert err <= 1e-2, f"layer {i} {nm}: max error {err:.3g} of the gradient's max {scale:.3g}"
    log(f"  loss {float(loss):.6g} vs {ref_loss:.6g}; LoRA gradients max error / max: "
        f"{max(errs):.3g}")


def test_lora_inputs_from_the_fp32_norm_output(torch):
    """The whole step's LoRA-down input is the reference's xq / xv: the fp32 norm output dropped out
    and rounded to fp16 once, fp16(keep ? y * ks : 0) (solution/k_norm.py:49-53), not the dropout
    of the already rounded fp16 output.  Checked per layer against the oracle's norm -> dropout ->
    lora_down chain on the layer's fp32 input: xq / xv equal to the single rounding in all but a
    handful of elements (those where the GPU's fp32 y differs in its last bit) and unequal to the
    double rounding wherever the two roundings differ; z_q / z_v within 2e-3 of their scale."""
    from decentrik_prime_amd import model
    from oracle import linear, norm
    lens = [512, 512, 512, 512]
    log(f"whole step: LoRA inputs from the fp32 norm output, 2 layers, lens {lens}")
    st = model.QwenQLoRAStep(lens, n_layers=2, vocab=4096, seed=6, head_chunk=1024)
    st.forward()
    torch.cuda.synchronize()
    f16, f32 = np.float16, np.float32
    for i in range(2):
        lo = {k: host(v) for k, v in st.lora[i].items()}
        _, _, y16, xq, xv = norm.rms_fwd(host(st.xin[i]), host(st.w_in[i]), st.eps, mq=lo["mq"],
                                         mv=lo["mv"], keep_scale=st.keep_scale)
        for t, want, mask, z in (("q", xq, lo["mq"], st.z[i]["q"]), ("v", xv, lo["mv"], st.z[i]["v"])):
            got = host((st.xq if t == "q" else st.xv)[i])
            # the double rounding the step must not use: the dropout of the fp16 output
            double = np.where(mask != 0, (y16.astype(f32) * f32(st.keep_scale)).astype(f32),
                              f32(0)).astype(f16)
            differ = want != double
            same = got.view(np.uint16) == want.view(np.uint16)
            assert (~same).sum() <= 1e-4 * got.size, f"layer {i} x{t}: {(~same).sum()} elements differ"
            assert differ.sum() > 100 and (got[differ] != double[differ]).mean() > 0.99, \
                f"layer {i} x{t}: follows the double rounding"
            zr = linear.lora_down(want, None, 1.0, lo["A" + t])
            zs = float(np.abs(zr).max())
            err = float(np.abs(host(z).astype(np.float64) - zr).max()) / zs
            assert err <= 2e-3, f"layer {i} z_{t}: max error {err:.3g} of its scale"


def test_trainer_metrics_of_a_packed_batch(torch):
    """A right-padded batch with prompt tokens the loss ignores, packed (trainer.pack) and run
    through the whole step (two layers, a 4096-token vocabulary): batch_metrics of the head's
    per-token stats against the padded-batch walk (oracle/trainer.py) over the float64 head oracle
    (oracle/head.py) on the step's final hidden state, and compute_loss against the mean of the
    oracle's per-token losses."""
    from decentrik_prime_amd import model, trainer
    from oracle import head
    from oracle import trainer as ref
    rng = np.random.default_rng(8)
    B, T, vocab = 3, 320, 4096
    lens = [300, 150, 62]
    ids = torch.from_numpy(rng.integers(0, vocab, (B, T)))
    mask = (torch.arange(T)[None, :] < torch.tensor(lens)[:, None]).to(torch.int64)
    labels = ids.clone()
    labels[mask == 0] = -100
    labels[0, :40] = -100
    labels[1, :100] = -100
    log(f"trainer metrics of a packed batch, lens {lens}")
    batch = trainer.pack(ids, mask, labels, vocab)
    st = model.QwenQLoRAStep.for_batch(batch, n_layers=2, vocab=vocab, seed=9, head_chunk=1024)
    loss_sum, stats, _ = st.forward()
    torch.cuda.synchronize()
    got = trainer.batch_metrics(batch, stats.cpu())
    # the oracle's per-token stats on the step's final hidden state, in token order
    tok, _ = head.head(host(st.yf), host(st.emb), batch.tgt.numpy(), 1.0)
    start = np.concatenate([[0], np.cumsum(lens)[:-1]])
    want = ref.padded_metrics(lambda b, t: tok[start[b] + t, :3], lens, labels.numpy())
    assert got["n_lab"] == want["n_lab"] and got["row_tokens"] == want["row_tokens"]
    assert abs(got["entropy"] - want["entropy"]) <= 2e-3 * abs(want["entropy"])
    for g, w in zip(got["row_loss"], want["row_loss"]):
        assert abs(g - w) <= 2e-3 * abs(w) + 1e-6
    # accuracy: hits agree except where the top two logits are within a GEMM rounding
    x = np.sort(head.logits16(host(st.yf), host(st.emb)).astype(np.float64), 1)
    near = int(((x[:, -1] - x[:, -2]) <= 2e-2).sum())
    assert abs(got["accuracy"] - want["accuracy"]) <= near / max(want["n_lab"], 1) + 1e-12
    mean = float(trainer.compute_loss(loss_sum, batch))
    ref_mean = float(tok[batch.tgt.numpy() >= 0, 0].sum()) / batch.n_lab
    assert abs(mean - ref_mean) <= 2e-3 * abs(ref_mean)


def _reference_inputs(torch, st, k_nf4):
    layers = []
    for i in range(st.n_layers):
        pk = st.layers[i]["packed"]
        buf = torch.empty(pk.numel, dtype=torch.float16, device="cuda")
        k_nf4.dequant_layer(pk, st.code2, st.nf4, buf)

        def w(kind):
            start, n = st.views[kind]
            W = st.layers[i][kind]
            return buf[start:start + n].view(W.rows, W.cols).cpu()
        lo = st.lora[i]
        layers.append(dict(wqkv=w("qkv"), wo=w("o"), wgu=w("gu"), wd=w("d"), bias=lo["bias"].cpu(),
                           w_in=st.w_in[i].cpu(), w_post=st.w_post[i].cpu(),
                           **{k: lo[k].cpu() for k in ("Aq", "Bq", "Av", "Bv", "mq", "mv")}))
    return dict(x0=st.x0.cpu(), emb=st.emb.cpu(), tgt=st.tgt.cpu(), pos=st.pos.cpu(), cos=st.cos.cpu(),
                sin=st.sin.cpu(), w_final=st.w_final.cpu(), eps=st.eps, ks=st.keep_scale, s=st.s,
                layers=layers)


@pytest.mark.parametrize("kind", ["window", "groups"])
def test_step_over_part_of_the_keys(torch, kind):
    """The whole step under a sliding window with sinks, and over groups of answers behind shared
    prompts, against the float64 reference with the same visible pairs; tolerances as for the causal
    step."""
    from decentrik_prime_amd import k_nf4, model
    from oracle import attn
    from oracle import model as ref
    if kind == "window":
        lens, window, sinks = [37, 210, 64], 50, 4
        st = model.QwenQLoRAStep(lens, n_layers=2, vocab=4096, seed=5, head_chunk=1024, window=window,
                                 sinks=sinks)
        vis = attn.window_visible(lens, window, sinks)
    else:
        groups = [(70, [30, 1, 45]), (0, [40]), (33, [20, 20])]
        st = model.QwenQLoRAStep(None, n_layers=2, vocab=4096, seed=5, head_chunk=1024, groups=groups)
        vis = attn.prefix_visible(groups)
    log(f"whole QLoRA step over part of the keys: {kind}")
    loss = st.step()
    loss2 = st.step()
    torch.cuda.synchronize()
    assert float(loss) == float(loss2), "the step is deterministic"
    ref_loss, ref_grads = ref.qwen_step(_reference_inputs(torch, st, k_nf4), st.lens,
                                        visible=torch.from_numpy(vis))
    assert abs(float(loss) - ref_loss) <= 1e-4 * abs(ref_loss), (float(loss), ref_loss)
    for i in range(2):
        for nm, got, want in zip(("dA_q", "dB_q", "dA_v", "dB_v"), st.grads[i], ref_grads[i]):
            g, r = host(got).astype(np.float64), want.numpy()
            err = float(np.abs(g - r).max()) / float(np.abs(r).max())
            assert err <= 1e-2, f"layer {i} {nm}: {err:.3g}"


def test_shared_prompts_train_as_rows_of_their_own(torch):
    """A batch packed by trainer.pack_answers gives the loss and the LoRA gradients of the same answers as
    rows with a prompt each (trainer.pack), without dropout: both within the causal step's tolerance of
    the same float64 values."""
    from decentrik_prime_amd import model, trainer
    rng = np.random.default_rng(3)
    vocab = 4096
    groups = [(rng.integers(0, vocab, p), [rng.integers(0, vocab, a) for a in ans])
              for p, ans in ((120, (30, 7, 55)), (40, (60, 1)))]
    log("shared prompts against rows of their own")
    kw = dict(n_layers=2, vocab=vocab, seed=9, head_chunk=1024)
    shared = model.QwenQLoRAStep.for_batch(trainer.pack_answers(groups, vocab), **kw)
    whole = [(np.concatenate([p, a]), len(p)) for p, ans in groups for a in ans]
    T = max(len(w) for w, _ in whole)
    ids, mask, labels = (torch.zeros(len(whole), T, dtype=torch.int64) for _ in range(3))
    labels -= 100
    for b, (w, n) in enumerate(whole):
        ids[b, :len(w)], mask[b, :len(w)] = torch.from_numpy(w), 1
        labels[b, n:len(w)] = torch.from_numpy(w[n:])
    rows = model.QwenQLoRAStep.for_batch(trainer.pack(ids, mask, labels, vocab), **kw)
    for st in (shared, rows):
        st.keep_scale = 1.0
        for i in range(2):
            st.layers[i] = shared.layers[i]
            for k, v in shared.lora[i].items():
                st.lora[i][k] = v if k not in ("mq", "mv") else torch.ones_like(st.lora[i][k])
    a, b = shared.step(), rows.step()
    torch.cuda.synchronize()
    assert shared.n_lab == rows.n_lab and shared.m < rows.m
    assert abs(float(a) - float(b)) <= 2e-4 * abs(float(b)), (float(a), float(b))
    for i in range(2):
        for nm, x, y in zip(("dA_q", "dB_q", "dA_v", "dB_v"), shared.grads[i], rows.grads[i]):
            x, y = host(x).astype(np.float64), host(y).astype(np.float64)
            err = float(np.abs(x - y).max()) / float(np.abs(y).max())
            assert err <= 2e-2, f"layer {i} {nm}: {err:.3g}"
