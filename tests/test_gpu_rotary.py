"""Rotary positions on the GPU against the rotation in complex float64.

Tolerances: cos and sin come from a remainder of turns rounded to 32 bits (below half a
turn: off by at most pi 2^-24) and sincospif (2 steps): 2^-21 of the pair's length covers
both and the two products' roundings; then one rounding to the type, half a step of the
value.
"""
import math

import pytest
import torch

from scao_b200 import Rotary, RotaryScaling

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def frequencies(dim, base, s):
    """(frequencies, magnitude) written apart from the library's."""
    j = torch.arange(dim // 2, dtype=torch.float64, device=DEV)
    if s is not None and s.kind == "ntk":
        base = base * s.factor ** (dim / (dim - 2))
    w = torch.exp(-2 * j / dim * math.log(base))
    if s is None or s.kind == "ntk":
        return w, 1.0
    if s.kind == "linear":
        return w / s.factor, 1.0
    r = s.original_len * w / (2 * math.pi)
    keep = torch.clamp((r - s.slow) / (s.fast - s.slow), 0, 1)
    return w / s.factor + keep * (w - w / s.factor), 0.1 * math.log(s.factor) + 1


def turned(x, pos, rotary, inverse=False):
    """(the rotation in float64, the length of each value's pair)."""
    w, m = frequencies(rotary.dim, rotary.base, rotary.scaling)
    n = rotary.dim // 2
    x = x.detach().double()
    angle = pos.double().reshape(-1 if pos.dim() == 2 else 1, 1, pos.shape[-1], 1) * w
    spin = m * torch.exp(1j * angle)
    if inverse:
        spin = spin.conj()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if rotary.interleaved else (x[..., :n], x[..., n:2 * n])
    z = torch.complex(a, b) * spin
    out, size = x.clone(), torch.zeros_like(x)
    if rotary.interleaved:
        out[..., 0:2 * n:2], out[..., 1:2 * n:2] = z.real, z.imag
        size[..., 0:2 * n:2] = size[..., 1:2 * n:2] = z.abs()
    else:
        out[..., :n], out[..., n:2 * n] = z.real, z.imag
        size[..., :n] = size[..., n:2 * n] = z.abs()
    return out, size


def close(got, x, pos, rotary, inverse=False):
    want, size = turned(x, pos, rotary, inverse)
    assert got.shape == x.shape and got.dtype == x.dtype
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 0.0
    tol = 2.0 ** -21 * size + (torch.finfo(got.dtype).eps / 2) * (want.abs() + 2.0 ** -21 * size) + tiny
    assert ((got.double() - want).abs() <= tol).all()
    assert torch.equal(got[..., rotary.dim:], x[..., rotary.dim:])


def randn(*shape, t=torch.float32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).to(t)


@pytest.mark.parametrize("kind", list(T))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("head_dim,dim", [(64, 64), (128, 128), (80, 64), (100, 100), (100, 50), (96, 2),
                                          (7, 6), (33, 32), (512, 512), (40, 24), (36, 12)])
def test_dims(kind, interleaved, head_dim, dim):
    r = Rotary(dim, interleaved=interleaved)
    q, k = randn(2, 3, 9, head_dim, t=T[kind]), randn(2, 1, 9, head_dim, t=T[kind], seed=1)
    yq, yk = r(q, k)
    pos = torch.arange(9, device=DEV)
    close(yq, q, pos, r)
    close(yk, k, pos, r)


@pytest.mark.parametrize("batch,heads,kv,length", [(1, 1, 1, 1), (1, 32, 8, 1), (33, 5, 1, 1), (2, 12, 4, 1000),
                                                   (1, 2, 2, 30001), (3, 1, 1, 17), (1, 300, 7, 3)])
def test_shapes(batch, heads, kv, length):
    r = Rotary(32)
    q, k = randn(batch, heads, length, 32, t=torch.bfloat16), randn(batch, kv, length, 32, t=torch.bfloat16, seed=1)
    for t, y in zip((q, k), r(q, k)):
        close(y, t, torch.arange(length, device=DEV), r)
    close(r(q), q, torch.arange(length, device=DEV), r)


@pytest.mark.parametrize("kind,head_dim,dim", [("bf16", 100, 50), ("f16", 96, 40), ("f32", 36, 14),
                                               ("f32", 4096, 6), ("f32", 4100, 6), ("bf16", 8192, 22)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("batch,heads,kv,length", [(1, 1, 1, 1), (2, 300, 7, 3), (3, 5, 2, 700)])
def test_rows_wider_than_their_pairs(batch, heads, kv, length, interleaved, kind, head_dim, dim):
    """Whole rows through shared memory: heads in several blocks, rows as long as a block's
    memory and longer."""
    if batch * length * heads * head_dim > 1 << 26:
        length = 5
    r = Rotary(dim, interleaved=interleaved)
    q, k = (randn(batch, h, length, head_dim, t=T[kind], seed=h) for h in (heads, kv))
    ids = torch.randint(0, 1 << 20, (batch, length), device=DEV)
    for t, y in zip((q, k), r(q, k, positions=ids)):
        close(y, t, ids, r)


@pytest.mark.parametrize("scaling", [None, RotaryScaling("linear", 4.0), RotaryScaling("ntk", 8.0),
                                     RotaryScaling("yarn", 16.0, original_len=4096),
                                     RotaryScaling("yarn", 2.5, original_len=100, fast=8, slow=0.5)])
@pytest.mark.parametrize("start", [0, 1_000_000, 2_000_000_011, -5])
def test_far_positions_and_scalings(scaling, start):
    r = Rotary(64, base=500000.0, scaling=scaling)
    q = randn(1, 2, 50, 64)
    close(r(q, positions=start), q, start + torch.arange(50, device=DEV), r)


@pytest.mark.parametrize("pos_type", [torch.int32, torch.int64])
def test_position_tensors(pos_type):
    r = Rotary(16)
    q, k = randn(3, 2, 11, 16), randn(3, 1, 11, 16, seed=1)
    ids = torch.randint(0, 100000, (3, 11), device=DEV).to(pos_type)
    ids[0] = 7                                       # the same position twice, out of order
    for p in (ids, ids[:1], ids[1], ids.t().contiguous().t(), torch.stack([ids, ids], -1)[..., 0]):
        for t, y in zip((q, k), r(q, k, positions=p)):
            close(y, t, p, r)


@pytest.mark.parametrize("kind", list(T))
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides(kind, interleaved):
    """Views of a fused projection, transposed heads, odd offsets, expanded batches."""
    r = Rotary(32, interleaved=interleaved)
    t, pos = T[kind], torch.arange(6, device=DEV)
    qkv = randn(2, 6, 5, 40, t=t)
    flat = randn(2 * 3 * 6 * 41 + 5, t=t)
    for x in (qkv[:, :, 1:4].transpose(1, 2), qkv.transpose(1, 2)[..., 3:38],
              flat[5:].view(2, 3, 6, 41)[..., 1:], randn(1, 3, 6, 32, t=t).expand(4, 3, 6, 32),
              randn(2, 3, 32, 6, t=t).transpose(2, 3), randn(2, 3, 6, 64, t=t)[..., ::2]):
        keep = x.clone()
        close(r(x), x, pos, r)
        assert torch.equal(x, keep)


def test_empty():
    r = Rotary(16)
    for shape in ((0, 2, 5, 16), (2, 0, 5, 16), (2, 2, 0, 16)):
        q = torch.empty(shape, device=DEV)
        assert r(q).shape == q.shape
    q = randn(2, 2, 5, 16)
    yq, yk = r(q, q[:, :0])
    assert yk.shape == (2, 0, 5, 16)
    close(yq, q, torch.arange(5, device=DEV), r)


def test_nonfinite_values_stay_in_their_pair():
    r = Rotary(8)
    q = randn(1, 1, 4, 10)
    q[0, 0, 2, 1] = math.inf
    y = r(q)
    bad = ~torch.isfinite(y)
    assert bad[0, 0, 2, [1, 5]].all() and bad.sum() == 2


@pytest.mark.parametrize("kind", list(T))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("scaling", [None, RotaryScaling("yarn", 4.0, original_len=64)])
def test_gradient(kind, interleaved, scaling):
    r = Rotary(24, interleaved=interleaved, scaling=scaling)
    q, k = (randn(2, h, 7, 32, t=T[kind], seed=h).requires_grad_() for h in (4, 2))
    gq, gk = randn(2, 4, 7, 32, t=T[kind], seed=5), randn(2, 7, 2, 32, t=T[kind], seed=6).transpose(1, 2)
    ids = torch.randint(0, 5000, (2, 7), device=DEV)
    yq, yk = r(q, k, positions=ids)
    dq, dk = torch.autograd.grad([yq, yk], [q, k], [gq, gk])
    close(dq, gq, ids, r, inverse=True)
    close(dk, gk, ids, r, inverse=True)
    (only,) = torch.autograd.grad(r(q, k)[1].sum(), [k])     # an expanded gradient, q unused
    close(only, torch.ones_like(k), torch.arange(7, device=DEV), r, inverse=True)


def test_gradient_against_differences():
    """Float32 values and central differences of the float64 rotation; and the second
    derivative of a square, which is a rotation there and back: m^2."""
    r = Rotary(6, scaling=RotaryScaling("yarn", 4.0, original_len=16))
    q = randn(1, 1, 3, 8).requires_grad_()
    pos = torch.tensor([0, 5, 3], device=DEV)
    w = randn(1, 1, 3, 8, seed=2)
    (g,) = torch.autograd.grad((r(q, positions=pos) * w).sum(), [q])
    eps = 2.0 ** -10
    for i in range(q.numel()):
        d = torch.zeros(q.numel(), dtype=torch.float64, device=DEV)
        d[i] = eps
        d = d.view(q.shape)
        up, down = (turned(q.double() + s * d, pos, r)[0] for s in (1, -1))
        want = (((up - down) / (2 * eps)) * w.double()).sum().item()    # linear: no truncation
        assert abs(g.reshape(-1)[i].item() - want) <= 2.0 ** -18 * w.abs().max().item()
    y = r(q, positions=pos)
    (g,) = torch.autograd.grad((y * y).sum(), [q], create_graph=True)
    (h,) = torch.autograd.grad(g.sum(), [q])
    m = r.magnitude
    want = torch.tensor([2 * m * m] * 6 + [2.0] * 2, device=DEV).expand_as(h)
    assert ((h - want).abs() <= 2.0 ** -18 * want).all()


def test_graph_and_side_stream():
    r = Rotary(32)
    q, ids = randn(2, 3, 5, 32), torch.randint(0, 1000, (2, 5), device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = r(q, positions=ids)
    torch.cuda.current_stream().wait_stream(s)
    close(y, q, ids, r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = r(q, positions=ids)
    for i in range(2):
        q.copy_(randn(2, 3, 5, 32, seed=10 + i))
        ids += 17
        graph.replay()
        close(y, q, ids, r)


def test_long_batch_offsets_pass_32_bits():
    """A view whose last token lies beyond 2^31 values."""
    n = (1 << 31) + 4096
    base = torch.empty(n, dtype=torch.bfloat16, device=DEV)
    x = base.as_strided((1, 2, 3, 64), (0, 64, (1 << 30) + 1024, 1))
    x.copy_(randn(1, 2, 3, 64, t=torch.bfloat16))
    r = Rotary(64)
    y = torch.empty(1, 2, 3, 64, dtype=torch.bfloat16, device=DEV)
    y = r(x)
    close(y, x, torch.arange(3, device=DEV), r)


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad
    r, q, k = Rotary(16), randn(1, 2, 5, 16), randn(1, 1, 5, 16, seed=1)
    leaf = q.clone().requires_grad_()
    want = r(leaf)
    (dq,) = torch.autograd.grad(want, leaf, q, retain_graph=True)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, q)
        for args in ((dual,), (dual, k), (k, dual)):
            with pytest.raises(NotImplementedError):
                r(*args)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(want, leaf, dual, retain_graph=True)
        y = r(leaf)
        assert torch.equal(y, want) and torch.equal(r(q), want)
        assert torch.equal(torch.autograd.grad(y, leaf, q)[0], dq)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("grad", [False, True])
def test_traces(grad):
    """A torch.jit trace calls the operator again, in both directions; an FX trace is refused."""
    from torch.fx.experimental.proxy_tensor import make_fx
    r, ids = Rotary(16), torch.arange(5, device=DEV) + 9
    for call in (lambda t: r(t), lambda t: r(t, t[:, :1], positions=ids)[1], lambda t: r(t, t, positions=3)[0]):
        traced = torch.jit.trace(call, randn(1, 2, 5, 16).requires_grad_(grad), check_trace=False)
        other = randn(1, 2, 5, 16, seed=9).requires_grad_()
        y, want = traced(other), call(other)
        assert torch.equal(y, want)
        assert torch.equal(torch.autograd.grad(y.sum(), other)[0], torch.autograd.grad(want.sum(), other)[0])
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(call)(randn(1, 2, 5, 16).requires_grad_(grad))


def test_saved_tensor_hooks():
    """Positions that hooks hand back on another device, in another type or size are refused."""
    r, ids = Rotary(16), torch.arange(5, device=DEV)
    q = randn(1, 2, 5, 16).requires_grad_()
    (want,) = torch.autograd.grad(r(q, positions=ids), q, torch.ones_like(q))

    def through(unpack):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = r(q, positions=ids)
        return torch.autograd.grad(y, q, torch.ones_like(q))[0]

    assert torch.equal(through(lambda t: t.clone()), want)
    for bad in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t[:4]):
        with pytest.raises(RuntimeError, match="another size, type or device"):
            through(bad)


@pytest.mark.parametrize("dim", [8, 128])
@pytest.mark.parametrize("pos", [1 << 29, -(1 << 29) - 7, 1 << 33, (1 << 40) + 12345, -(1 << 45) + 1, (1 << 50) + 3])
def test_angles_of_very_far_positions(pos, dim):
    """Against angles in rational numbers: off by at most |p| 2^-55 of a turn on top of the
    float32 bound at the head of this file."""
    from fractions import Fraction
    two_pi = Fraction(628318530717958647692528676655900576839433879875021, 10 ** 50)
    r = Rotary(dim)
    x = randn(1, 1, 1, dim, seed=3)
    turns = [Fraction(float(w)) * pos / two_pi for w in r.frequencies]
    angle = torch.tensor([float(t - math.floor(t)) for t in turns], dtype=torch.float64, device=DEV) * (2 * math.pi)
    a, b = x.double().chunk(2, -1)
    want = torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1)
    size = torch.hypot(a, b).repeat(1, 1, 1, 2)
    tol = size * (2.0 ** -21 + 2 * math.pi * abs(pos) * 2.0 ** -55) + 2.0 ** -24 * want.abs()
    for y in (r(x, positions=pos), r(x, positions=torch.tensor([pos], device=DEV))):
        assert ((y.double() - want).abs() <= tol).all()
