"""Global gradient norm and clipping on the GPU against float64.

Tolerances: the norm is summed in 64 bits from 32-value sums in 32 bits (each off by
at most 32 * 2^-24 of itself) and rounded once: 2^-18 covers both.  A clipped value is
g c rounded once, c off by that and one rounding: half a step of the type, 2^-18, and one
denormal step of the type.
"""
import math

import pytest
import torch

import scao_b200
from scao_b200 import clip_grad_norm_, clip_grads_with_norm_, get_total_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def params_of(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, dtype=g.dtype, device=g.device))
        p.grad = g
        out.append(p)
    return out


def norm64(grads, kind):
    x = torch.cat([g.detach().reshape(-1).double() for g in grads]) if grads else torch.zeros(1).double()
    return x.norm().item() if kind == 2 else x.abs().sum().item() if kind == 1 else x.abs().max().item()


def close(got, before, coef):
    want = before.double() * coef
    tol = (torch.finfo(got.dtype).eps / 2 + 2.0 ** -18) * want.abs() + TINY[got.dtype]
    assert ((got.double() - want).abs() <= tol).all()


def check(grads, kind, max_norm):
    before = [g.clone() for g in grads]
    want = norm64(before, kind)
    total = clip_grad_norm_(params_of(grads), max_norm, norm_type=kind)
    assert total.dtype == torch.float32 and total.shape == () and total.device == grads[0].device
    assert abs(total.item() - want) <= 2.0 ** -18 * want + 2.0 ** -149
    coef = min(1.0, max_norm / (want + 1e-6))
    for g, b in zip(grads, before):
        if coef == 1.0:
            assert torch.equal(g, b)
        else:
            close(g, b, coef)


def make(sizes, kinds, scale=1e-2, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(n, generator=gen, device=DEV) * scale).to(T[kinds[i % len(kinds)]])
            for i, n in enumerate(sizes)]


@pytest.mark.parametrize("kind", [1, 2, math.inf])
@pytest.mark.parametrize("kinds", [["f32"], ["bf16"], ["f16"], ["f32", "bf16", "f16"]])
@pytest.mark.parametrize("max_norm", [1e-3, 1e6])
def test_sizes(kind, kinds, max_norm):
    check(make([1, 2, 3, 5, 7, 8, 9, 16, 17, 511, 2047, 2049, 4097, 100003, 300000], kinds), kind, max_norm)


@pytest.mark.parametrize("count", [1, 2, 199, 200, 201, 1599, 1601, 3300])
def test_many_tensors(count):
    check(make([1 + (i * 37) % 300 for i in range(count)], ["f32", "bf16"]), 2, 0.01)


@pytest.mark.parametrize("kinds", [["f32"], ["bf16"]])
def test_one_large_tensor_and_many_small(kinds):
    check(make([9_000_001] + [33] * 40, kinds), 2, 0.5)


@pytest.mark.parametrize("offset", [1, 2, 3, 5, 7])
def test_unaligned_views_leave_their_neighbours(offset):
    for t in T.values():
        flat = torch.randn(70001, device=DEV).to(t)
        keep = flat.clone()
        g = flat[offset:offset + 60001]
        check([g], 2, 0.1)
        assert torch.equal(flat[:offset], keep[:offset]) and torch.equal(flat[offset + 60001:], keep[offset + 60001:])


@pytest.mark.parametrize("scale", [1e-30, 1e-22, 1e15, 1e25])
def test_range_of_float32(scale):
    """Squares of these under- or overflow in 32 bits."""
    check(make([5000, 77], ["f32", "bf16"], scale), 2, scale * 1e-2)


def test_mixed_magnitudes():
    g = make([4096, 4096], ["f32"], 1.0)
    g[0][:100] *= 1e-25
    g[1][5] = 3e38
    check(g, 2, 1.0)


def test_zeros_and_empty():
    g = [torch.zeros(1000, device=DEV), torch.zeros(0, device=DEV), torch.zeros(33, device=DEV, dtype=torch.bfloat16)]
    check(g, 2, 1.0)
    assert get_total_norm([torch.zeros(0, device=DEV)]).item() == 0
    assert clip_grad_norm_([], 1.0).item() == 0 and get_total_norm([]).item() == 0
    assert clip_grad_norm_([torch.nn.Parameter(torch.ones(3, device=DEV))], 1.0).item() == 0   # no gradient


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kind", [1, 2, math.inf])
def test_nonfinite(bad, kind):
    """As torch.nn.utils.clip_grad_norm_: a NaN norm makes everything NaN, an infinite one
    makes finite values 0; error_if_nonfinite raises before anything is written."""
    g = make([5000, 300], ["f32", "bf16"])
    g[1][7] = bad
    before = [x.clone() for x in g]
    with pytest.raises(RuntimeError, match="not finite"):
        clip_grad_norm_(params_of(g), 1.0, kind, error_if_nonfinite=True)
    assert all(torch.equal(x.nan_to_num(), b.nan_to_num()) for x, b in zip(g, before))
    with pytest.raises(RuntimeError, match="not finite"):
        get_total_norm(g, kind, error_if_nonfinite=True)
    total = clip_grad_norm_(params_of(g), 1.0, kind)
    if math.isnan(bad):
        assert total.isnan() and all(x.isnan().all() for x in g)
    else:
        assert total.item() == math.inf and (g[0] == 0).all() and g[1][7].isnan()
        assert g[1].nan_to_num().eq(0).all()


def test_strided_gradients():
    base = torch.randn(64, 100, device=DEV)
    dense = torch.randn(40, 30, device=DEV).t()                 # dense, permuted
    keep = base.clone()
    check([base[:, 3:50], dense], 2, 0.5)
    assert torch.equal(base[:, :3], keep[:, :3]) and torch.equal(base[:, 50:], keep[:, 50:])


def test_infinite_threshold_and_zero_threshold():
    g = make([1000], ["f32"])
    b = g[0].clone()
    clip_grad_norm_(params_of(g), math.inf)
    assert torch.equal(g[0], b)
    clip_grad_norm_(params_of(g), 0.0)
    assert (g[0] == 0).all()


def test_two_step_form_matches():
    a, b = make([3000, 501], ["f32", "bf16"]), make([3000, 501], ["f32", "bf16"])
    total = get_total_norm(a)
    clip_grads_with_norm_(params_of(a), 0.1, total)
    assert torch.equal(total, clip_grad_norm_(params_of(b), 0.1))
    for x, y in zip(a, b):      # the coefficient from the rounded norm: one more half step
        assert ((x.double() - y.double()).abs() <= torch.finfo(x.dtype).eps * y.double().abs()).all()
    c = make([100], ["f32"])
    clip_grads_with_norm_(params_of(c), 0.1, torch.tensor([2.0], dtype=torch.float64, device=DEV))
    close(c[0], make([100], ["f32"])[0], 0.05)


def test_same_inputs_same_bits():
    runs = []
    for _ in range(3):
        g = make([700001, 33, 5000], ["f32", "bf16"])
        runs.append((clip_grad_norm_(params_of(g), 0.1), g))
    for total, g in runs[1:]:
        assert torch.equal(total, runs[0][0]) and all(torch.equal(x, y) for x, y in zip(g, runs[0][1]))


def test_side_stream_and_graph():
    """On a stream of its own, and captured with another graph over other gradients:
    replays in turn give what eager calls give."""
    s = torch.cuda.Stream()
    sets = [make([100000, 77], ["f32", "bf16"], seed=i) for i in range(2)]
    keep = [[g.clone() for g in gs] for gs in sets]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        check(make([12345], ["bf16"], seed=9), 2, 0.1)
    torch.cuda.current_stream().wait_stream(s)
    graphs, totals = [], []
    for gs in sets:
        graph = torch.cuda.CUDAGraph()
        ps = params_of(gs)
        with torch.cuda.graph(graph):
            totals.append(clip_grad_norm_(ps, 0.1))
        graphs.append(graph)
    for round_ in range(2):
        for gs, ks in zip(sets, keep):
            for g, k in zip(gs, ks):
                g.copy_(k * (1 + round_))
        for graph in graphs:
            graph.replay()
        for gs, ks, total in zip(sets, keep, totals):
            eager = [k * (1 + round_) for k in ks]
            assert torch.equal(total, clip_grad_norm_(params_of(eager), 0.1))
            assert all(torch.equal(g, e) for g, e in zip(gs, eager))


def test_counts_as_a_write():
    g = torch.ones(10, device=DEV)
    v = g._version
    clip_grad_norm_(params_of([g]), 0.1)
    assert g._version > v


def test_train_step_clips():
    """train_step(max_grad_norm=...) hands SCAO the clipped gradients: the same update
    as clipping by hand."""
    from scao_b200 import SCAO, gpt
    c = gpt.GPTConfig(n_layer=1, d_model=64, n_head=2, d_ff=128, vocab=128, seq_len=16)
    kw = dict(lr=1e-3, sparsity=0.0, noise_std_init=0.0, async_precond=False)
    a, b = gpt.GPT(c).to(DEV), gpt.GPT(c).to(DEV)
    oa, ob = SCAO(a.parameters(), **kw), SCAO(b.parameters(), **kw)
    tokens = gpt.token_batch(c, 4, seed=1, device=DEV)
    gpt.train_step(a, oa, tokens, max_grad_norm=1e-2)
    gpt.loss_fn(b, tokens).backward()
    before = norm64([p.grad for p in b.parameters()], 2)
    scao_b200.clip_grad_norm_(b.parameters(), 1e-2)
    assert before > 1e-2 and abs(norm64([p.grad for p in b.parameters()], 2) - 1e-2) < 1e-4
    ob.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)


def test_column_halves():
    """Gradients that interleave in memory without sharing are clipped as any; sharing ones are
    refused and stay as they are."""
    base = torch.randn(64, 100, device=DEV)
    check([base[:, :50], base[:, 50:]], 2, 0.5)
    check([base[::2], base[1::2, 3:9]], math.inf, 0.01)
    keep = base.clone()
    for a, b in ((base[:, :51], base[:, 50:]), (base, base[:, ::2])):
        with pytest.raises(ValueError, match="share memory"):
            clip_grad_norm_(params_of([a, b]), 1e-3)
        with pytest.raises(ValueError, match="share memory"):
            clip_grads_with_norm_(params_of([a, b]), 1e-3, torch.ones((), device=DEV))
    assert torch.equal(base, keep)
    want = norm64([base, base[:, ::2]], 2)              # a norm only reads
    assert abs(get_total_norm([base, base[:, ::2]]).item() - want) <= 2.0 ** -18 * want
