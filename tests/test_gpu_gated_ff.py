"""The gated feed-forward product and its gradients on the GPU against float64.

Tolerances.  A product of two 16-bit values is exact in 32 bits; a 32-bit sum of n of
them is off by at most n 2^-23 (tensor cores may cut instead of round) of the sum of the
magnitudes: E below, carried through the activation, whose derivative is below 1.2
and whose own error in 32 bits is below 2^-19 of its argument's size.  Each rounding to
the type adds half a step (r = eps / 2): one for h, one for dg and du (operands) and one
for the gradients, which read g and u rounded to 24 bits (16 of the significand): K = 2^-16
of each.
"""
import math

import pytest
import torch

from gated_ff_shapes import PATHS, plan
from scao_b200 import GatedFeedForward, _lib, gated_ff, gpt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T = {"bf16": torch.bfloat16, "f16": torch.float16}
K = 2.0 ** -16
ACTS = ["silu", "gelu", "gelu_tanh"]


def act64(g, kind):
    if kind == "silu":
        return g * torch.sigmoid(g)
    if kind == "gelu":
        return g * torch.special.ndtr(g)
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))


def tiny(t):
    return 2.0 ** -24 if t == torch.float16 else 2.0 ** -133


def forward64(x, wg, wu, kind):
    """(h, bound on its error, g, u, bounds on theirs)."""
    x, wg, wu = x.detach().double(), wg.detach().double(), wu.detach().double()
    n = x.shape[-1] * 2.0 ** -23
    g, u = x @ wg.T, x @ wu.T
    eg, eu = n * (x.abs() @ wg.abs().T), n * (x.abs() @ wu.abs().T)
    a = act64(g, kind)
    ea = 1.2 * eg + 2.0 ** -19 * g.abs()
    h = a * u
    return h, ea * u.abs() + eu * a.abs() + ea * eu, (g, u, a, eg, eu, ea)


def close(got, want, err):
    t = got.dtype
    r = torch.finfo(t).eps / 2
    bad = (got.double() - want).abs() > (1 + r) * err + r * want.abs() + tiny(t)
    assert not bad.any(), (bad.sum().item(), bad.nonzero()[:4].tolist())


def backward64(x, wg, wu, dh, kind):
    """[(value, bound)] of dx, dwg, dwu."""
    _, _, (g, u, a, eg, eu, ea) = forward64(x, wg, wu, kind)
    t = x.dtype
    r = torch.finfo(t).eps / 2
    x, wg, wu, dh = (v.detach().double() for v in (x, wg, wu, dh))
    gr = g.clone().requires_grad_()
    with torch.enable_grad():
        (d,) = torch.autograd.grad(act64(gr, kind).sum(), [gr])
    dg, du = dh * u * d, dh * a
    eg, eu = eg + K * g.abs(), eu + K * u.abs()
    ed = 1.2 * eg + 2.0 ** -19 * (1 + g.abs())        # act'' is below 1.2
    ea = 1.2 * eg + 2.0 ** -19 * g.abs()
    edg = dh.abs() * (eu * d.abs() + ed * u.abs() + ed * eu)
    edu = dh.abs() * ea
    edg, edu = edg * (1 + r) + r * dg.abs() + tiny(t), edu * (1 + r) + r * du.abs() + tiny(t)
    nf, nm = 2 * wg.shape[0] * 2.0 ** -23, x.shape[0] * 2.0 ** -23
    mag = lambda a, b: a.abs() @ b.abs()  # noqa: E731
    out = [(dg @ wg + du @ wu, (1 + nf) * (mag(edg, wg) + mag(edu, wu)) + nf * (mag(dg, wg) + mag(du, wu)))]
    for y, e in ((dg, edg), (du, edu)):
        out.append((y.T @ x, (1 + nm) * mag(e.T, x) + nm * mag(y.T, x)))
    return out


def randn(*shape, t=torch.bfloat16, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(t)


def inputs(m, d, f, t, seed=0):
    return (randn(m, d, t=t, seed=seed), randn(f, d, t=t, seed=seed + 1, scale=d ** -0.5),
            randn(f, d, t=t, seed=seed + 2, scale=d ** -0.5))


def check(x, wg, wu, kind, train, seed=7):
    if not train:
        with torch.no_grad():
            h = gated_ff(x, wg, wu, activation=kind)
        want, err, _ = forward64(x, wg, wu, kind)
        assert h.dtype == x.dtype and h.is_contiguous()
        close(h, want, err)
        return
    ins = [v.detach().requires_grad_() for v in (x, wg, wu)]
    h = gated_ff(*ins, activation=kind)
    want, err, _ = forward64(x, wg, wu, kind)
    close(h, want, err)
    dh = randn(*h.shape, t=x.dtype, seed=seed, scale=0.1)
    for got, (want, err) in zip(torch.autograd.grad(h, ins, dh), backward64(x, wg, wu, dh, kind)):
        close(got, want, err)


SHAPES = [(1, 64, 64), (1, 2048, 512), (2, 200, 7), (7, 8, 1000), (8, 65, 129), (15, 1, 1), (16, 712, 320),
          (17, 63, 8), (33, 512, 128), (127, 128, 127), (128, 64, 128), (129, 72, 136), (255, 1000, 64),
          (256, 256, 256), (257, 264, 264), (1000, 130, 520), (513, 96, 2048), (3000, 64, 40)]


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("kind", list(T))
@pytest.mark.parametrize("m,d,f", SHAPES)
def test_shapes(m, d, f, kind, train):
    check(*inputs(m, d, f, T[kind]), "silu", train)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [3, 300])
def test_activations(m, act, train):
    x, wg, wu = inputs(m, 128, 200, torch.bfloat16)
    check(x, wg * 4, wu, act, train)         # gates up to about 15 both ways


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [2, 100])
def test_huge_gates(m, act):
    """Gates of 1e19 and more either way: the activation is the gate or nothing, its
    derivative 1 or 0."""
    x, wg, wu = (torch.ones(n, 8, dtype=torch.bfloat16, device=DEV) for n in (m, 16, 16))
    wg[:8] *= 2.0 ** 62
    wg[8:] *= -(2.0 ** 66)
    ins = [v.requires_grad_() for v in (x, wg, wu)]
    h = gated_ff(*ins, activation=act)
    assert (h[:, :8] == 8 * 2.0 ** 62 * 8).all() and (h[:, 8:] == 0).all()
    dx, dg, du = torch.autograd.grad(h, ins, torch.ones_like(h))
    assert (dg[:8] == 8 * m).all() and (dg[8:] == 0).all() and (du[8:] == 0).all()
    assert torch.isfinite(dx).all()


@pytest.mark.parametrize("m", range(1, 70))
def test_every_small_row_count(m):
    check(*inputs(m, 136, 72, torch.float16), "silu", False)


@pytest.mark.parametrize("m", [1, 12, 30, 60])
@pytest.mark.parametrize("d,f", [(33, 9000), (1100, 1000), (2500, 17), (4, 300)])
def test_few_rows_of_other_widths(m, d, f):
    """One to sixteen warps share a contraction; widths that leave warps without a step."""
    check(*inputs(m, d, f, torch.bfloat16), "gelu", False)


@pytest.mark.parametrize("m,d,f", [(2100, 320, 1500), (1500, 700, 1600), (3000, 1100, 2100), (600, 2000, 700),
                                   (5000, 136, 136), (200, 64, 9000), (9000, 64, 200),
                                   (4000, 72, 4000), (4100, 700, 2500)])
def test_many_tiles(m, d, f):
    """More tiles than SMs: the persistent loop and both accumulators; results of one CTA
    and of pairs, whole and split contractions, either product the longer one."""
    check(*inputs(m, d, f, torch.bfloat16), "silu", True)


def test_long_contraction():
    check(*inputs(20000, 72, 136, torch.bfloat16), "gelu", True)


def test_rounding_errors_do_not_pile_up():
    """In the 2-norm roundings are independent: two of them (operand and result) stay
    below sqrt(2) r, h below r; r is the largest of a rounding, its mean is lower."""
    x, wg, wu = inputs(512, 512, 640, torch.bfloat16)
    ins = [v.requires_grad_() for v in (x, wg, wu)]
    h = gated_ff(*ins)
    dh = randn(512, 640, seed=5)
    r = torch.finfo(torch.bfloat16).eps / 2
    rel = lambda a, b: ((a.double() - b).norm() / b.norm()).item()  # noqa: E731
    assert rel(h, forward64(x, wg, wu, "silu")[0]) <= r
    for got, (want, _) in zip(torch.autograd.grad(h, ins, dh), backward64(x, wg, wu, dh, "silu")):
        assert rel(got, want) <= math.sqrt(2) * r


def test_leading_dimensions_and_strides():
    d, f = 72, 136
    _, wg, wu = inputs(1, d, f, torch.bfloat16)
    fused = randn(2 * f, d + 8, scale=0.1)
    for x in (randn(2, 3, 5, d), randn(d), randn(4, 6, d + 24)[..., 8:8 + d], randn(4, 6, d + 1)[..., 1:],
              randn(d, 9).t(), randn(1, d).expand(40, d), randn(40, 2 * d)[:, ::2]):
        for a, b in ((wg, wu), (fused[:f, :d], fused[f:, :d]), (fused[0::2, 3:d + 3], fused[1::2, 3:d + 3]),
                     (wg, wg), (randn(d, f, scale=0.1).t(), wu)):
            h = gated_ff(x, a, b)
            assert h.shape == (*x.shape[:-1], f)
            want, err, _ = forward64(x.reshape(-1, d), a, b, "silu")
            close(h.reshape(-1, f), want, err)


@pytest.mark.parametrize("offset", range(8))
@pytest.mark.parametrize("cols", [1, 7, 9, 16, 23, 40])
def test_packed_copies(cols, offset):
    """The copies of unaligned operands: every value, zeros behind the rows."""
    from scao_b200.feedforward import _operands
    flat = randn(40 * 50 + 64, seed=cols)
    views = [flat[offset:offset + 40 * 49].view(40, 49)[:, :cols], flat[offset:offset + 3 * cols].view(3, cols),
             flat[offset:offset + cols].view(1, cols)]
    ins, _ = _operands(views)
    torch.cuda.synchronize()
    for (t, p, pitch, *_), v in zip(ins, views):
        assert t.data_ptr() == p and p % 16 == 0 and pitch % 8 == 0 and torch.equal(t[:, :cols], v)
        if t is not v:
            assert (t[:, cols:] == 0).all()


def test_odd_widths_keep_copies_for_the_gradient():
    x, wg, wu = inputs(50, 43, 64, torch.bfloat16)
    ins = [v.requires_grad_() for v in (x, wg, wu)]
    h = gated_ff(*ins)
    with torch.no_grad():
        wg += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(h, ins, torch.ones_like(h))


def test_values_beside_a_view_are_not_read():
    """NaN behind odd rows of x and of the weights reaches no result."""
    m, d, f = 20, 43, 50
    for rows in (3, m):
        bx, bg, bu = (torch.full((n, 48), math.nan, dtype=torch.bfloat16, device=DEV) for n in (rows, f, f))
        x, wg, wu = inputs(rows, d, f, torch.bfloat16)
        for b, v in ((bx, x), (bg, wg), (bu, wu)):
            b[:, :d] = v
        check(bx[:, :d], bg[:, :d], bu[:, :d], "silu", False)
        check(bx[:, :d], bg[:, :d], bu[:, :d], "silu", True)


def test_gradient_layouts_and_subsets():
    x, wg, wu = inputs(50, 64, 96, torch.bfloat16)
    ins = [v.requires_grad_() for v in (x, wg, wu)]
    for dh in (randn(96, 50).t(), randn(1, 96).expand(50, 96), randn(50, 1).expand(50, 96), randn(50, 99)[:, 2:98]):
        h = gated_ff(*ins)
        for got, (want, err) in zip(torch.autograd.grad(h, ins, dh), backward64(x, wg, wu, dh, "silu")):
            close(got, want, err)
    dh = randn(50, 96, seed=3)
    want = backward64(x, wg, wu, dh, "silu")
    for which in ([0], [1], [2], [0, 2], [1, 2]):
        ins = [v.detach().requires_grad_(i in which) for i, v in enumerate((x, wg, wu))]
        h = gated_ff(*ins)
        for i, got in zip(which, torch.autograd.grad(h, [ins[i] for i in which], dh)):
            close(got, *want[i])


def test_shared_weights_sum_their_gradients():
    x, w, _ = inputs(30, 64, 40, torch.float16)
    w.requires_grad_()
    dh = randn(30, 40, t=torch.float16, scale=0.1)
    (got,) = torch.autograd.grad(gated_ff(x, w, w), [w], dh)
    (_, _), (a, ea), (b, eb) = backward64(x, w, w, dh, "silu")
    r = torch.finfo(torch.float16).eps / 2
    close(got, a + b, ea + eb + r * (a.abs() + b.abs()) * (1 + r) + 2 * tiny(torch.float16))


def test_gradient_against_differences():
    """Central differences of the float64 form: off by step^2 / 6 of the third
    derivative (below 2 of the inputs' sizes here) beside the gradient's own bound."""
    x, wg, wu = inputs(5, 24, 9, torch.float16)
    ins = [v.requires_grad_() for v in (x, wg, wu)]
    dh = randn(5, 9, t=torch.float16, seed=4)
    grads = torch.autograd.grad(gated_ff(*ins, activation="gelu_tanh"), ins, dh)
    bounds = backward64(x, wg, wu, dh, "gelu_tanh")
    base = [v.detach().double() for v in ins]
    step = 2.0 ** -12
    r = torch.finfo(torch.float16).eps / 2

    def loss(vs):
        return ((act64(vs[0] @ vs[1].T, "gelu_tanh") * (vs[0] @ vs[2].T)) * dh.double()).sum()

    for k, (g, (want, err)) in enumerate(zip(grads, bounds)):
        for i in range(0, g.numel(), 7):
            vs = [[b.clone() for b in base] for _ in range(2)]
            vs[0][k].view(-1)[i] += step
            vs[1][k].view(-1)[i] -= step
            diff = ((loss(vs[0]) - loss(vs[1])) / (2 * step)).item()
            tol = err.reshape(-1)[i].item() * (1 + r) + r * abs(diff) + 2.0 ** -24 + 100 * step * step
            assert abs(g.reshape(-1)[i].item() - diff) <= tol, (k, i)


def test_second_derivative_is_refused():
    ins = [v.requires_grad_() for v in inputs(9, 64, 40, torch.bfloat16)]
    dh = randn(9, 40, seed=2)
    plain = torch.autograd.grad(gated_ff(*ins), ins, dh)
    graph = torch.autograd.grad(gated_ff(*ins), ins, dh, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, graph))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(graph[0].float().sum(), ins)


def test_empty_rows():
    _, wg, wu = inputs(1, 64, 40, torch.bfloat16)
    for shape in ((0, 64), (2, 0, 64)):
        ins = [torch.empty(shape, dtype=torch.bfloat16, device=DEV).requires_grad_(), wg.requires_grad_(),
               wu.requires_grad_()]
        h = gated_ff(*ins)
        assert h.shape == (*shape[:-1], 40)
        dx, dg, du = torch.autograd.grad(h.sum(), ins)
        assert dx.shape == shape and (dg == 0).all() and (du == 0).all()


@pytest.mark.parametrize("m", [3, 40])
def test_nonfinite_rows_stay_alone(m):
    x, wg, wu = inputs(m, 64, 40, torch.bfloat16)
    clean = gated_ff(x, wg, wu)
    x[1, 3], x[2, 5] = math.nan, math.inf
    h = gated_ff(x, wg, wu)
    assert h[1].isnan().all() and not torch.isfinite(h[2]).any()
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(h[keep], clean[keep])


@pytest.mark.parametrize("f", [40, 41])
@pytest.mark.parametrize("m", [3, 40, 130])
def test_writes_nothing_else(m, f):
    """Through the C entry: guards before and behind every result stay."""
    d = 64
    x, wg, wu = inputs(m, d, f, torch.bfloat16)
    L, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    guard = lambda n: torch.full((n + 1024,), 7.0, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    bufs = {"h": guard(m * f), "dx": guard(m * d), "dw_gate": guard(f * d), "dw_up": guard(f * d)}
    saved = torch.empty(int(L.scao_gated_ff_saved_bytes(m, f)), dtype=torch.uint8, device=DEV)
    ws = torch.empty(int(L.scao_gated_ff_workspace_bytes(m, d, f, 3)), dtype=torch.uint8, device=DEV)
    dh = randn(m, f, seed=4)
    import ctypes
    a = _lib.GatedFfArgs()
    a.x, a.w_gate, a.w_up, a.dh = (t.data_ptr() for t in (x, wg, wu, dh))
    a.saved, a.workspace = saved.data_ptr(), ws.data_ptr()
    a.ldx = a.ldg = a.ldu = d
    a.lddh, a.rows, a.d, a.ff, a.dtype, a.act = f, m, d, f, _lib.BF16, 0
    for k, b in bufs.items():
        setattr(a, k, b[512:].data_ptr())
    assert L.scao_gated_ff_forward(ctypes.byref(a), stream) == 0
    assert L.scao_gated_ff_backward(ctypes.byref(a), stream) == 0
    ins = [v.requires_grad_() for v in (x, wg, wu)]
    h = gated_ff(*ins)
    for (k, b), want in zip(bufs.items(), [h, *torch.autograd.grad(h, ins, dh)]):
        n = want.numel()
        assert (b[:512] == 7).all() and (b[512 + n:] == 7).all(), k
        assert torch.equal(b[512:512 + n], want.detach().reshape(-1)), k


def test_same_inputs_same_bits():
    x, wg, wu = inputs(700, 200, 300, torch.bfloat16)
    ins = [v.requires_grad_() for v in (x, wg, wu)]
    dh = randn(700, 300, seed=4)
    runs = []
    for _ in range(3):
        h = gated_ff(*ins)
        runs.append([h.detach(), *torch.autograd.grad(h, ins, dh)])
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(run, runs[0]))


def test_side_streams_and_graphs():
    """Two captured steps over one set of weights, replayed in turn and beside an eager
    call on another stream."""
    _, wg, wu = inputs(1, 64, 96, torch.bfloat16)
    sets = []
    for m in (5, 300):
        x = randn(m, 64, seed=m).requires_grad_()
        leaves = [x, wg.detach().requires_grad_(), wu.detach().requires_grad_()]
        dh = randn(m, 96, seed=m + 1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            h = gated_ff(*leaves)
            out = [h.detach(), *torch.autograd.grad(h, leaves, dh)]
        sets.append((graph, leaves, dh, out))
    side = torch.cuda.Stream()
    for round_ in range(2):
        for graph, leaves, dh, _ in sets:
            with torch.no_grad():
                leaves[0].copy_(randn(*leaves[0].shape, seed=20 + round_))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            xs = randn(300, 64, seed=50)
            eager_side = gated_ff(xs, wg, wu)
        for graph, *_ in sets:
            graph.replay()
        torch.cuda.synchronize()
        want, err, _ = forward64(xs, wg, wu, "silu")
        close(eager_side, want, err)
        for _, leaves, dh, out in sets:
            fresh = [v.detach().clone().requires_grad_() for v in leaves]
            h = gated_ff(*fresh)
            for a, b in zip(out, [h.detach(), *torch.autograd.grad(h, fresh, dh)]):
                assert torch.equal(a, b)


def test_first_call_inside_a_capture():
    """The first call of a process may be captured (status word, kernel attributes)."""
    import subprocess
    import sys
    code = ("import torch; from scao_b200 import gated_ff\n"
            "x = torch.randn(40, 64, device='cuda').bfloat16(); w = torch.randn(48, 64, device='cuda').bfloat16()\n"
            "g = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(g):\n"
            "    h = gated_ff(x, w, w)\n"
            "g.replay()\n"
            "assert torch.equal(h, gated_ff(x, w, w))\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_timed_out_wait_is_reported_once():
    """The word that a kernel sets when a wait runs out (set here by the host) makes the
    next call raise; the one after it runs."""
    x, wg, wu = inputs(40, 64, 40, torch.bfloat16)
    want = gated_ff(x, wg, wu)
    torch.cuda.synchronize()
    _lib.lib().scao_gated_ff_status_word()[0] = 2
    with pytest.raises(_lib.ScaoError, match="timed out"):
        gated_ff(x, wg, wu)
    assert torch.equal(gated_ff(x, wg, wu), want)


def test_autocast_casts():
    x, w = randn(10, 64, t=torch.float32), randn(48, 64, t=torch.float32, scale=0.1).requires_grad_()
    with torch.autocast("cuda", dtype=torch.float16):
        h = gated_ff(x, w, w)
    assert h.dtype == torch.float16
    (g,) = torch.autograd.grad(h.float().sum(), [w])
    assert g.dtype == torch.float32 and torch.isfinite(g).all()
    with pytest.raises(TypeError):
        gated_ff(x, w, w)


def test_saves_nothing_without_gradients():
    x, wg, wu = inputs(4096, 64, 1024, torch.bfloat16)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    h = gated_ff(x, wg, wu)
    assert torch.cuda.max_memory_allocated() - base < 2 * h.numel() * 2
    w = wg.detach().requires_grad_()
    with torch.no_grad():
        assert not gated_ff(x, w, wu).requires_grad


# ------------------------------------------------------- together, in the model
SMALL = gpt.GPTConfig(n_layer=2, d_model=128, n_head=4, d_ff=200, vocab=300, seq_len=48, mlp="gated",
                      positions="rotary", n_kv_head=2)


def plain_loss(model, c, tokens):
    """The model in float64 from its parameters alone: own rotation, own gating."""
    p = {n: v.detach().double().requires_grad_() for n, v in model.named_parameters()}
    idx, B = tokens[:, :-1], tokens.shape[0]
    n, hd, kv = idx.shape[1], c.d_model // c.n_head, c.n_kv_head
    w = c.rotary_base ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)
    ang = torch.arange(n, device=DEV).double()[:, None] * w
    cos, sin = ang.cos(), ang.sin()

    def rot(t):
        a, b = t[..., :hd // 2], t[..., hd // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    ln = lambda t, name: torch.nn.functional.layer_norm(t, (c.d_model,), p[name + ".weight"],  # noqa: E731
                                                        p[name + ".bias"])
    x = p["tok.weight"][idx]
    mask = torch.full((n, n), -math.inf, device=DEV, dtype=torch.float64).triu(1)
    for i in range(c.n_layer):
        b = f"blocks.{i}."
        q, k, v = (ln(x, b + "ln1") @ p[b + "attn.qkv.weight"].T).split([c.d_model, kv * hd, kv * hd], -1)
        q, k, v = (t.view(B, n, -1, hd).transpose(1, 2) for t in (q, k, v))
        q, k = rot(q), rot(k)
        k, v = (t.repeat_interleave(c.n_head // kv, 1) for t in (k, v))
        att = torch.softmax(q @ k.transpose(-1, -2) / math.sqrt(hd) + mask, -1) @ v
        x = x + att.transpose(1, 2).reshape(B, n, -1) @ p[b + "attn.proj.weight"].T
        y = ln(x, b + "ln2")
        h = act64(y @ p[b + "ff.gate.weight"].T, c.activation) * (y @ p[b + "ff.up.weight"].T)
        x = x + h @ p[b + "ff.out.weight"].T
    logits = ln(x, "ln_f") @ p["tok.weight"].T
    loss = torch.nn.functional.cross_entropy(logits.reshape(-1, c.vocab), tokens[:, 1:].reshape(-1))
    return loss, dict(zip(p, torch.autograd.grad(loss, list(p.values()))))


def test_model_matches_float64():
    """Loss and every gradient of the gated, rotary model under bf16 autocast.  A
    layer rounds about eight times on its way (r = 2^-8 at most, about a third of it in
    the mean, independent): over two layers there and back sqrt(32) r / 3, doubled for
    the softmax and the normalisations; 4 r."""
    model = gpt.GPT(SMALL).to(DEV)
    tokens = gpt.token_batch(SMALL, 4, seed=1, device=DEV)
    loss = gpt.loss_fn(model, tokens)
    loss.backward()
    want, grads = plain_loss(model, SMALL, tokens)
    r = 2.0 ** -8
    assert abs(loss.item() - want.item()) <= r * want.item()
    for n, p in model.named_parameters():
        rel = ((p.grad.double() - grads[n]).norm() / grads[n].norm()).item()
        assert rel <= 4 * r, (n, rel)


def test_model_trains_with_clipping():
    """The three together: gated block, rotary positions, clipped SCAO steps run, the
    gradients of every parameter are finite and the weights move."""
    from scao_b200 import SCAO
    model = gpt.GPT(SMALL).to(DEV)
    opt = SCAO(model.parameters(), lr=1e-3, warmup_steps=2, precond_freq=2, min_precond_updates=1,
               blend_steps=2, k_min=4, k_max=16, max_precond_dim=256, sparsity=0.0, noise_std_init=0.0,
               async_precond=False)
    start = [p.detach().clone() for p in model.parameters()]
    for s in range(6):
        loss = gpt.train_step(model, opt, gpt.token_batch(SMALL, 4, seed=s, device=DEV), max_grad_norm=1.0)
        assert torch.isfinite(loss)
    torch.cuda.synchronize()
    opt._plan.check_error()
    for a, p in zip(start, model.parameters()):
        assert torch.isfinite(p).all() and not torch.equal(a, p)


def test_block_matches_its_parts():
    block = GatedFeedForward(64, 96, "gelu", device=DEV, dtype=torch.bfloat16)
    x = randn(2, 7, 64)
    h = gated_ff(x, block.gate.weight, block.up.weight, "gelu")
    assert torch.equal(block(x), block.out(h))


def test_calls_from_two_threads():
    """Forward, gradient, rotation and clipping at the same time on two streams."""
    import threading

    from scao_b200 import Rotary, clip_grad_norm_
    sets = [inputs(m, 72, 136, torch.bfloat16, seed=m) for m in (40, 300)]
    rotary = Rotary(24)

    def work(x, wg, wu):
        ins = [v.detach().clone().requires_grad_() for v in (x, wg, wu)]
        h = gated_ff(*ins)
        params = [torch.nn.Parameter(v.detach().clone()) for v in ins]
        for p, g in zip(params, torch.autograd.grad(h, ins, torch.ones_like(h))):
            p.grad = g
        total = clip_grad_norm_(params, 0.5)
        q = rotary(h.detach()[:, :120].reshape(1, -1, 5, 24).transpose(1, 2))
        return [h.detach(), q, total, *(p.grad for p in params)]

    want = [work(*s) for s in sets]
    got, errors = [[], []], []
    torch.cuda.synchronize()

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(30):
                    got[i].append(work(*sets[i]))
            stream.synchronize()
        except Exception as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_checkpointed_and_offloaded():
    """Recomputed in the backward pass, or with what is kept moved to the host and back:
    the same gradients; a graph used twice too."""
    from torch.utils.checkpoint import checkpoint
    block = GatedFeedForward(64, 96, device=DEV, dtype=torch.bfloat16)
    x = randn(50, 64).requires_grad_()
    leaves = [x, *block.parameters()]
    dy = randn(50, 64, seed=2)
    y = block(x)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy)
    other = torch.autograd.grad(checkpoint(block, x, use_reentrant=False), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = block(x)
    moved = torch.autograd.grad(y, leaves, dy)
    for grads in (again, other, moved):
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_backward_accumulates_into_grad():
    ins = [v.requires_grad_() for v in inputs(20, 43, 50, torch.float16)]
    one = torch.autograd.grad(gated_ff(*ins).sum(), ins)
    for _ in range(2):
        gated_ff(*ins).sum().backward()
    for v, g in zip(ins, one):
        assert torch.equal(v.grad, g + g)


def test_forward_mode_is_refused():
    """A tangent is refused, as an input's and as a gradient's; a level without one changes nothing."""
    from torch.autograd import forward_ad
    x, wg, wu = inputs(40, 64, 48, torch.bfloat16)
    leaf, dh = x.clone().requires_grad_(), randn(40, 48, seed=5)
    want = gated_ff(leaf, wg, wu)
    (dx,) = torch.autograd.grad(want, leaf, dh, retain_graph=True)
    with forward_ad.dual_level():
        for i in range(3):
            ins = [forward_ad.make_dual(v, v) if k == i else v for k, v in enumerate((x, wg, wu))]
            with pytest.raises(NotImplementedError), torch.no_grad():
                gated_ff(*ins)
            with pytest.raises(NotImplementedError):
                gated_ff(*ins)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(want, leaf, forward_ad.make_dual(dh, dh), retain_graph=True)
        h = gated_ff(leaf, wg, wu)
        assert torch.equal(h, want) and torch.equal(gated_ff(x, wg, wu), want)
        assert torch.equal(torch.autograd.grad(h, leaf, dh)[0], dx)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("d", [64, 63])
@pytest.mark.parametrize("grad", [False, True])
def test_traces(grad, d):
    """A torch.jit trace calls the operator again, in both directions; an FX trace is refused."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, wg, wu = inputs(40, d, 48, torch.bfloat16)
    call = lambda v: gated_ff(v, wg, wu)  # noqa: E731
    traced = torch.jit.trace(call, x.clone().requires_grad_(grad), check_trace=False)
    other = randn(40, d, seed=9).requires_grad_()
    h, want = traced(other), call(other)
    assert torch.equal(h, want)
    assert torch.equal(torch.autograd.grad(h.sum(), other)[0], torch.autograd.grad(want.sum(), other)[0])
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(call)(x.clone().requires_grad_(grad))


def test_first_calls_from_threads():
    """The first calls of a process may come from several threads at once."""
    import subprocess
    import sys
    code = ("import sys, threading, torch; from scao_b200 import _lib, gated_ff\n"
            "_lib.lib(); sys.setswitchinterval(1e-6)\n"
            "x = torch.randn(100, 64, device='cuda').bfloat16(); w = torch.randn(48, 64, device='cuda').bfloat16()\n"
            "torch.cuda.synchronize(); gate = threading.Barrier(16); out = [None] * 16\n"
            "def run(i):\n"
            "    torch.cuda.set_device(0); gate.wait()\n"
            "    out[i] = gated_ff(x, w, w)\n"
            "threads = [threading.Thread(target=run, args=(i,)) for i in range(16)]\n"
            "[t.start() for t in threads]; [t.join() for t in threads]\n"
            "assert all(torch.equal(h, gated_ff(x, w, w)) for h in out)\n")
    for _ in range(3):
        r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]


def test_first_work_of_a_thread():
    """A call may be the first GPU work of its thread."""
    import threading
    x, wg, wu = inputs(100, 64, 48, torch.bfloat16)
    want = gated_ff(x, wg, wu)
    leaf = x.clone().requires_grad_()
    kept = gated_ff(leaf, wg, wu)
    (dx,) = torch.autograd.grad(kept, leaf, want, retain_graph=True)
    torch.cuda.synchronize()
    got = {}

    def run(name, call):
        try:
            got[name] = call()
        except Exception as e:      # noqa: BLE001
            got[name] = e

    for name, call in (("forward", lambda: gated_ff(x, wg, wu)),
                       ("gradient", lambda: torch.autograd.grad(kept, leaf, want)[0])):
        t = threading.Thread(target=run, args=(name, call))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert not any(isinstance(v, Exception) for v in got.values()), got
    assert torch.equal(got["forward"], want) and torch.equal(got["gradient"], dx)


def test_copies_for_the_gradient_are_saved_tensors():
    """Aligned copies go where saved tensors go: to the host and back, recomputed, and freed
    with them; operands that lie right are not kept twice."""
    from torch.utils.checkpoint import checkpoint
    m, d, f = 300, 1021, 520
    ins = [v.requires_grad_() for v in inputs(m, d, f, torch.float16)]
    dh = randn(m, f, t=torch.float16, seed=5)
    saved = (m + 127) // 128 * ((f + 127) // 128) * 128 * 128 * 6
    copies = (m + 2 * f) * 1024 * 2
    used = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]  # noqa: E731

    def kept(context):
        """(memory held between the passes, after the backward pass, the gradients)"""
        torch.cuda.synchronize()
        start = used()
        with context:
            h = gated_ff(*ins)
        held = used() - start - h.numel() * 2
        loss = (h * dh).sum()       # holds the graph
        del h
        grads = torch.autograd.grad(loss, ins)
        after = used() - start - sum(g.numel() * 2 for g in grads)
        return held, after, grads, loss

    import contextlib
    held, after, want, loss = kept(contextlib.nullcontext())
    assert saved + copies <= held < saved + copies + 8192
    assert after < 8192, after
    held, _, grads, loss = kept(torch.autograd.graph.save_on_cpu())
    assert held < 8192, held
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    torch.cuda.synchronize()
    start = used()
    h = checkpoint(gated_ff, *ins, use_reentrant=False)
    assert used() - start - h.numel() * 2 < 8192
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad((h * dh).sum(), ins), want))
    x = ins[0].detach()
    wide = torch.empty(m, 1024, dtype=x.dtype, device=DEV)[:, :d].copy_(x).requires_grad_()     # only the weights lie odd
    torch.cuda.synchronize()
    start = used()
    h = gated_ff(wide, *ins[1:])
    assert used() - start - h.numel() * 2 < saved + 2 * f * 1024 * 2 + 8192
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(h, [wide, *ins[1:]], dh), want))


@pytest.mark.parametrize("f", [40, 41, 42])
@pytest.mark.parametrize("m,d", [(40, 64), (130, 63), (300, 66)])
@pytest.mark.parametrize("at", [(1, 1, 1, 1), (2, 2, 2, 1), (3, 5, 1, 4), (4, 6, 7, 7)])
def test_results_anywhere(at, m, d, f):
    """Through the C entry: results that begin between two 32-bit words, of even and odd
    pitch, each of its own alignment; the same bits, and nothing beside them."""
    import ctypes
    x, wg, wu = (torch.nn.functional.pad(v, (0, -d % 8)) for v in inputs(m, d, f, torch.bfloat16))
    L, stream, ld = _lib.lib(), torch.cuda.current_stream().cuda_stream, x.shape[1]
    saved = torch.empty(int(L.scao_gated_ff_saved_bytes(m, f)), dtype=torch.uint8, device=DEV)
    ws = torch.empty(int(L.scao_gated_ff_workspace_bytes(m, d, f, 3)), dtype=torch.uint8, device=DEV)
    dh = randn(m, f, seed=4)
    a = _lib.GatedFfArgs()
    a.x, a.w_gate, a.w_up, a.dh = (t.data_ptr() for t in (x, wg, wu, dh))
    a.saved, a.workspace = saved.data_ptr(), ws.data_ptr()
    a.ldx = a.ldg = a.ldu = ld
    a.lddh, a.rows, a.d, a.ff, a.dtype, a.act = f, m, d, f, _lib.BF16, 0
    bufs = {k: torch.full((n + 1024,), 7.0, dtype=torch.bfloat16, device=DEV)
            for k, n in (("h", m * f), ("dx", m * d), ("dw_gate", f * d), ("dw_up", f * d))}
    for (k, b), off in zip(bufs.items(), at):
        setattr(a, k, b[512 + off:].data_ptr())
    assert L.scao_gated_ff_forward(ctypes.byref(a), stream) == 0
    assert L.scao_gated_ff_backward(ctypes.byref(a), stream) == 0
    ins = [v[:, :d].detach().requires_grad_() for v in (x, wg, wu)]
    h = gated_ff(*ins)
    for (k, b), off, want in zip(bufs.items(), at, [h, *torch.autograd.grad(h, ins, dh)]):
        n, lo = want.numel(), 512 + off
        assert (b[:lo] == 7).all() and (b[lo + n:] == 7).all(), k
        assert torch.equal(b[lo:lo + n], want.detach().reshape(-1)), k


@pytest.mark.parametrize("d", [64, 61])
@pytest.mark.parametrize("m", [5, 200])
def test_saved_tensor_hooks(m, d):
    """Hooks may hand back what was saved anywhere in memory; of another size, type or
    device it is refused."""
    ins = [v.requires_grad_() for v in inputs(m, d, 48, torch.bfloat16)]
    dh = randn(m, 48, seed=5)
    want = torch.autograd.grad(gated_ff(*ins), ins, dh)

    def through(unpack):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            h = gated_ff(*ins)
        return torch.autograd.grad(h, ins, dh)

    def moved(t, by):
        buf = torch.empty(t.numel() + 16, dtype=t.dtype, device=DEV)
        return buf[by:by + t.numel()].view(t.shape).copy_(t)

    for by in (1, 2, 4, 7):
        assert all(torch.equal(a, b) for a, b in zip(through(lambda t: moved(t, by)), want))
    spread = lambda t: torch.stack([t, t], -1)[..., 0]  # noqa: E731
    assert all(torch.equal(a, b) for a, b in zip(through(spread), want))
    for bad in (lambda t: t.cpu(), lambda t: t.float(), lambda t: t[:t.shape[0] - 1]):
        with pytest.raises(RuntimeError, match="another size, type or device"):
            through(bad)


def test_widest():
    """The largest inner width: more blocks of columns than a grid has places in that direction."""
    f = (1 << 23) - 1
    x, wg, wu = inputs(2, 8, f, torch.bfloat16)
    check(x, wg, wu, "silu", True)
    with pytest.raises(ValueError, match="widths below"):
        gated_ff(x, wg.new_empty(f + 1, 8), wu.new_empty(f + 1, 8))


@pytest.mark.parametrize("sizes", list(PATHS))
def test_tile_paths(sizes):
    """Every tile with several items a CTA or pair, and whole and cut contractions, for both
    gradient products together and for each alone."""
    assert [(w, *plan(*sizes, w)) for w, *_ in PATHS[sizes]] == PATHS[sizes]
    x, wg, wu = inputs(*sizes, torch.float16 if sizes[2] % 2 else torch.bfloat16)
    check(x, wg, wu, "silu", True)
    dh = randn(sizes[0], sizes[2], t=x.dtype, seed=7, scale=0.1)
    want = backward64(x, wg, wu, dh, "silu")
    for which in (1, 2):
        ins = [v.detach().requires_grad_(which == (1 if i == 0 else 2)) for i, v in enumerate((x, wg, wu))]
        need = [v for v in ins if v.requires_grad]
        grads = torch.autograd.grad(gated_ff(*ins), need, dh)
        for got, (value, err) in zip(grads, want[:1] if which == 1 else want[1:]):
            close(got, value, err)


@pytest.mark.parametrize("kind", list(T))
def test_gradients_are_two_roundings_off(kind):
    """In the 2-norm, as above, in both types, against the rounding that the result alone has: a
    second, independent one of dg and du of the same mean makes sqrt(2) of it; K of g and u adds
    (K / r)^2 / 2 of that, 2^-11 in float16.  Within 3 %: the mean over 10^5 values."""
    m, d, f = 512, 512, 640
    x, wg, wu = inputs(m, d, f, T[kind])
    ins = [v.requires_grad_() for v in (x, wg, wu)]
    dh = randn(m, f, t=T[kind], seed=5, scale=0.1)
    h = gated_ff(*ins)
    for got, (want, _) in zip(torch.autograd.grad(h, ins, dh), backward64(x, wg, wu, dh, "silu")):
        one = (want.to(T[kind]).double() - want).norm()
        assert (got.double() - want).norm() <= 1.03 * math.sqrt(2) * one
