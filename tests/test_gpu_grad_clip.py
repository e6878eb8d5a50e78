"""The global gradient norm and clipping (k_grad) against the definition in 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"fp32": [torch.float32], "fp16": [torch.float16], "bf16": [torch.bfloat16],
         "mixed": [torch.bfloat16, torch.float32, torch.float16]}


def make(sizes, types, seed=0, rms=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, generator=g, device="cuda") * rms).to(types[i % len(types)])
            for i, s in enumerate(sizes)]


def definition(grads, max_norm, scale):
    norm = scale * math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    factor = scale * min(1.0, max_norm / (norm + 1e-6))
    return norm, [g.double() * factor for g in grads]


def check(norm, outs, want_norm, want):
    assert norm.dtype == torch.float32 and norm.shape == ()
    assert abs(float(norm) - want_norm) <= 2 * U * want_norm
    for o, w in zip(outs, want):
        # the factor's and the product's rounding to fp32, and the result's own: half a step, or half
        # of the type's smallest number
        info = torch.finfo(o.dtype)
        tol = w.abs() * (3 * U + info.eps / 2) + info.tiny * info.eps / 2
        assert o.shape == w.shape and bool(((o.double() - w).abs() <= tol).all())


SIZES = {"one": [1], "few": [3, 1, 7, 8, 9], "adapters": [24576, 24576, 24576, 4096] * 6,
         "ragged": [0, 8191, 8192, 8193, 0, 2047, 2049, 100001, 1, 0], "many": [17 + i for i in range(300)],
         "large": [9_000_001, 5], "none": [0, 0]}


@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("max_norm, scale", [(0.25, 1.0), (1e6, 1.0), (0.25, 1.0 / 64), (math.inf, 4.0)])
def test_clipping_matches_the_definition(sizes, types, max_norm, scale):
    from decentrik_prime_amd import k_grad
    grads = make(SIZES[sizes], TYPES[types], seed=len(SIZES[sizes]))
    before = [g.clone() for g in grads]
    norm, want = definition(grads, max_norm, scale)
    outs = [torch.empty(g.shape, device="cuda") for g in grads]
    check(k_grad.clip_grads(grads, max_norm, scale=scale, out=outs), outs, norm, want)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    check(k_grad.grad_norm(grads, scale=scale), [], norm, [])
    check(k_grad.clip_grads(grads, max_norm, scale=scale), grads, norm, want)
    if norm <= max_norm and scale == 1.0:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.parametrize("n", [111, 127, 128, 129, 255, 256, 257, 1000])
def test_any_number_of_tensors(n):
    """Lists that fill launches exactly, and by one tensor more or fewer; every third without elements."""
    from decentrik_prime_amd import k_grad
    grads = make([0 if i % 3 == 2 else 1 + 37 * i for i in range(n)], TYPES["mixed"], seed=n)
    norm, want = definition(grads, 0.5, 1.0)
    outs = [torch.empty(g.shape, device="cuda") for g in grads]
    check(k_grad.clip_grads(grads, 0.5, out=outs), outs, norm, want)
    full = make([5] * n, TYPES["fp32"], seed=n + 1)
    norm, want = definition(full, 0.5, 1.0)
    check(k_grad.clip_grads(full, 0.5), full, norm, want)


@pytest.mark.parametrize("types", list(TYPES))
def test_pieces_of_buffers_at_any_element(types):
    """Gradients that begin anywhere in a buffer; what lies between them is left as it was."""
    from decentrik_prime_amd import k_grad
    buffers = {t: torch.full((30000,), 7.0, device="cuda").to(t) for t in TYPES[types]}
    grads, at = [], dict.fromkeys(buffers, 1)
    for i, n in enumerate([1, 5, 2048, 2049, 8200, 33, 8, 15]):
        t = TYPES[types][i % len(TYPES[types])]
        piece = buffers[t][at[t]:at[t] + n]
        piece.copy_(torch.randn(n, device="cuda"))
        grads.append(piece)
        at[t] += n + 1 + i % 3
    norm, want = definition(grads, 1.0, 1.0)
    check(k_grad.clip_grads(grads, 1.0), grads, norm, want)
    taken = {t: torch.zeros(30000, dtype=torch.bool, device="cuda") for t in buffers}
    for g in grads:
        first = (g.data_ptr() - buffers[g.dtype].data_ptr()) // g.element_size()
        taken[g.dtype][first:first + g.numel()] = True
    for t, b in buffers.items():
        assert bool((b[~taken[t]] == 7.0).all())


def test_output_types_and_shapes():
    from decentrik_prime_amd import k_grad
    src = [torch.randn(5, 700, device="cuda").half(), torch.randn(64, 33, device="cuda").t(),
           torch.randn(2, 3, 5, device="cuda").bfloat16(), torch.randn((), device="cuda")]
    norm, want = definition(src, 2.0, 0.5)
    for t in (torch.float32, torch.float16, torch.bfloat16):
        outs = [torch.empty_like(g, dtype=t) for g in src]
        assert outs[1].stride() == src[1].stride()
        check(k_grad.clip_grads(src, 2.0, scale=0.5, out=outs), outs, norm, want)
    # some in place, some elsewhere
    outs = [src[0], torch.empty_like(src[1]), src[2], torch.empty_like(src[3])]
    check(k_grad.clip_grads(src, 2.0, scale=0.5, out=outs), outs, norm, want)


@pytest.mark.parametrize("size", [1e30, 1e-30])
def test_norms_beyond_the_squares_of_fp32(size):
    from decentrik_prime_amd import k_grad
    grads = [torch.full((1000,), size, device="cuda"), torch.full((24,), -size, device="cuda")]
    assert float(k_grad.grad_norm(grads)) == pytest.approx(32 * size, rel=1e-6)
    if size > 1:
        norm, want = definition(grads, 1.0, 1.0)
        check(k_grad.clip_grads(grads, 1.0), grads, norm, want)


def test_a_gradient_of_more_than_2_to_the_31_elements():
    from decentrik_prime_amd import k_grad
    n = (1 << 31) + 5
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    for at in (0, 1 << 20, (1 << 31) - 1, 1 << 31, n - 1):
        g[at] = 3.0
    assert float(k_grad.clip_grads([g], 1.0)) == pytest.approx(math.sqrt(45), rel=1e-6)
    assert int((g != 0).sum()) == 5
    for at in (0, 1 << 20, (1 << 31) - 1, 1 << 31, n - 1):
        assert float(g[at]) == pytest.approx(3 / math.sqrt(45), rel=2.0 ** -8)


def test_what_is_not_finite():
    from decentrik_prime_amd import k_grad
    for bad, rest in ((float("inf"), 0.0), (float("nan"), float("nan"))):
        grads = [torch.ones(3000, device="cuda"), torch.ones(10, device="cuda").half()]
        grads[0][2999] = bad
        norm = k_grad.clip_grads(grads, 1.0)
        assert not math.isfinite(float(norm)) and bool(torch.isnan(grads[0][2999]))
        for t in (grads[0][:2999], grads[1]):
            assert bool(torch.isnan(t).all()) if math.isnan(rest) else bool((t == 0).all())


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_no_largest_norm_scales_alone(bad):
    from decentrik_prime_amd import k_grad
    grads = [torch.ones(3000, device="cuda"), torch.ones(10, device="cuda").half()]
    grads[0][7] = bad
    assert not math.isfinite(float(k_grad.clip_grads(grads, math.inf, scale=0.5)))
    assert not math.isfinite(float(grads[0][7]))
    grads[0][7] = 0.5
    assert all(bool((g == 0.5).all()) for g in grads)


def test_captured_and_on_another_stream():
    from decentrik_prime_amd import k_grad
    sizes = [24576, 4096, 77] * 60                    # two batches of tensors
    first, second = make(sizes, TYPES["mixed"], 1), make(sizes, TYPES["mixed"], 2, rms=0.5)

    def run(src):
        outs = [torch.empty(g.shape, device="cuda") for g in src]
        return (k_grad.clip_grads(src, 1.0, out=outs), *outs)
    want = [run(first), run(second)]
    assert all(torch.equal(a, b) for a, b in zip(run(first), want[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(second)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    held = [g.clone() for g in first]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(held)
    for turn in range(4):
        for h, g in zip(held, (first, second)[turn % 2]):
            h.copy_(g)
        run(second)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[turn % 2])), turn


@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("types", list(TYPES))
def test_scaling_by_a_number_on_the_device(sizes, types):
    from decentrik_prime_amd import k_grad
    for by, scale in ((0.3, 1.0), (2.0 ** -20, -3.0), (1.0, 1.0), (0.0, 2.0), (4.0, 0.0)):
        grads = make(SIZES[sizes], TYPES[types], seed=2)
        want = [g.double() * float(torch.tensor(by)) * scale for g in grads]
        k_grad.scale_grads(grads, torch.tensor(by, device="cuda"), scale=scale)
        for g, w in zip(grads, want):
            info = torch.finfo(g.dtype)      # the factor's and the product's rounding, and the result's own
            tol = w.abs() * (3 * U + info.eps / 2) + info.tiny * info.eps / 2
            assert bool(((g.double() - w).abs() <= tol).all()), (by, scale)
    one = [torch.ones(4, device="cuda")]
    for bad in (torch.ones(2, device="cuda"), torch.ones((), device="cuda").half(), torch.ones(())):
        with pytest.raises(ValueError):
            k_grad.scale_grads(one, bad)
    with pytest.raises(ValueError):
        k_grad.scale_grads(one + one, torch.ones((), device="cuda"))


def test_refusals():
    from decentrik_prime_amd import k_grad
    g = torch.ones(8, 8, device="cuda")
    for grads, kwargs in (([g, g], {}), ([g, g[2:]], {}), ([g[:, :4]], {}), ([g.cpu()], {}), ([g, g.cpu()], {}),
                          ([g], dict(out=[])), ([g], dict(out=[torch.ones(64, device="cuda")])),
                          ([g], dict(out=[torch.ones(8, 8, device="cuda").t()])),
                          ([g], dict(out=[g.double()])), ([g.half()], dict(out=[g.cpu()])),
                          ([g.view(-1)[:32]], dict(out=[g.view(-1)[1:33]]))):
        with pytest.raises(ValueError):
            k_grad.clip_grads(grads, 1.0, **kwargs)
    assert bool((g == 1).all())


def test_overlaps_are_named():
    from decentrik_prime_amd import k_grad
    g = torch.ones(8, 8, device="cuda")
    for call in (lambda: k_grad.clip_grads([g, g], 1.0), lambda: k_grad.clip_grads([g, g[2:]], 1.0),
                 lambda: k_grad.clip_grads([g.view(-1)[:32]], 1.0, out=[g.view(-1)[1:33]]),
                 lambda: k_grad.scale_grads([g, g[2:]], torch.ones((), device="cuda")),
                 lambda: k_grad.scale_grads([g], g[7, 7])):
        with pytest.raises(ValueError, match="overlap"):
            call()
    assert bool((g == 1).all()) and float(k_grad.grad_norm([g, g])) == pytest.approx(math.sqrt(128))
