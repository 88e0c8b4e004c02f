"""Refusals and host logic of the operators around the optimizer step; no GPU."""
import copy
import ctypes
import math
import pickle
from array import array

import pytest
import torch

from gated_ff_shapes import PAIR, PATHS, SINGLE, TALL, plan
from scao_b200 import (GatedFeedForward, Rotary, RotaryScaling, _lib, clip_grad_norm_,
                       clip_grads_with_norm_, gated_ff, get_total_norm, gpt)
from scao_b200.clip import _layout


def param(grad):
    p = torch.nn.Parameter(torch.empty(grad.shape, dtype=grad.dtype))
    p.grad = grad
    return p


# ------------------------------------------------------------------- clipping
@pytest.mark.parametrize("norm_type", [0, 3, 0.5, -1, math.nan, -math.inf])
def test_clip_refuses_norms(norm_type):
    with pytest.raises(ValueError, match="norm_type"):
        clip_grad_norm_([param(torch.ones(3))], 1.0, norm_type)
    with pytest.raises(ValueError, match="norm_type"):
        get_total_norm([torch.ones(3)], norm_type)


@pytest.mark.parametrize("max_norm", [-1.0, math.nan, -math.inf])
def test_clip_refuses_thresholds(max_norm):
    with pytest.raises(ValueError, match="max_norm"):
        clip_grad_norm_([param(torch.ones(3))], max_norm)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads_with_norm_([param(torch.ones(3))], max_norm, torch.ones(()))


def test_clip_refuses_types_and_devices():
    with pytest.raises(TypeError, match="dtype"):
        clip_grad_norm_([param(torch.ones(3, dtype=torch.float64))], 1.0)
    with pytest.raises(TypeError, match="layout"):
        get_total_norm([torch.eye(3).to_sparse()])
    with pytest.raises(ValueError, match="one device"):
        get_total_norm([torch.ones(3), torch.ones(3, device="meta")])
    with pytest.raises(RuntimeError, match="CUDA"):
        clip_grad_norm_([param(torch.ones(3))], 1.0)


def test_clip_refuses_shared_memory():
    base = torch.ones(20)
    for a, b in ((base[:10], base[9:]), (base, base), (base[3:5], base)):
        with pytest.raises(ValueError, match="share memory"):
            clip_grad_norm_([param(a), param(b)], 1.0)
    with pytest.raises(ValueError, match="with itself"):
        clip_grad_norm_([param(torch.ones(1).expand(5))], 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):            # neighbours do not share
        clip_grad_norm_([param(base[:10]), param(base[10:])], 1.0)


@pytest.mark.parametrize("a,b,shares", [
    (lambda x: x[:, :5], lambda x: x[:, 3:], True), (lambda x: x, lambda x: x[:, ::2], True),
    (lambda x: x[:, :5], lambda x: x[:, 5:], False), (lambda x: x[:, ::2], lambda x: x[:, 1::2], False),
    (lambda x: x[:, ::2], lambda x: x[:, ::3], True), (lambda x: x[::2], lambda x: x[1::2, 2:5], False),
    (lambda x: x[::2], lambda x: x[1::3], True), (lambda x: x[1::4, :3], lambda x: x[::2], False),
    (lambda x: x[2:4], lambda x: x[:, 1:3], True), (lambda x: x[9:], lambda x: x[:9, 1:3], False),
    (lambda x: x[:, 1], lambda x: x[7], True), (lambda x: x[:, 1].bfloat16, lambda x: x[:, 1], False)])
def test_clip_refuses_shared_memory_of_views(a, b, shares):
    base = torch.ones(12, 8)
    a, b = a(base), b(base)
    pair = [param(v() if callable(v) else v) for v in (a, b)]
    for grads in (pair, pair[::-1], [param(torch.ones(3)), *pair]):
        with pytest.raises(ValueError if shares else RuntimeError, match="share memory" if shares else "CUDA"):
            clip_grad_norm_(grads, 1.0)


def test_sharing_of_views_is_exact():
    """Against the sets of the bytes, for many pairs of views."""
    import random

    from scao_b200.clip import _meet, _places
    rng = random.Random(5)
    base = torch.zeros(600, dtype=torch.float32)
    half = base.view(torch.bfloat16)

    def view():
        flat = rng.choice([base, half])
        while True:
            shape = [rng.choice([1, 2, 3, 4, 7]) for _ in range(rng.randint(1, 3))]
            stride, need = [], rng.choice([1, 1, 2, 3, 5])
            for n in shape:
                stride.append(need)
                need = need * n + rng.choice([0, 0, 1, 4])
            order = list(range(len(shape)))
            rng.shuffle(order)
            shape, stride = [shape[i] for i in order], [stride[i] for i in order]
            if need < 500:
                return flat.as_strided(shape, stride, rng.randrange(40 * flat.numel() // 600))

    def bytes_of(t):
        at = torch.zeros(t.shape, dtype=torch.long) + t.data_ptr()
        for i, (n, st) in enumerate(zip(t.shape, t.stride())):
            at = at + (torch.arange(n) * st * t.element_size()).view([-1 if k == i else 1 for k in range(t.dim())])
        return {int(x) + k for x in at.flatten() for k in range(t.element_size())}

    found = [0, 0]
    for _ in range(3000):
        a, b = view(), view()
        if _layout(a)[1] or _layout(b)[1]:
            continue
        want = not bytes_of(a).isdisjoint(bytes_of(b))
        assert _meet(*_places(a), *_places(b)) == want, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride())
        found[want] += 1
    assert min(found) > 500, found


def test_sharing_of_long_views_is_quick():
    """Two halves of the columns of a tall matrix: a few steps, not one a row."""
    import time
    base = torch.zeros(1 << 20, 8)
    pair = [param(base[:, :4]), param(base[:, 4:])]
    with pytest.raises(RuntimeError, match="CUDA"):
        clip_grad_norm_(pair, 1.0)
    from scao_b200.clip import _refuse_sharing
    start = time.perf_counter()
    _refuse_sharing([p.grad for p in pair], {0, 1})
    assert time.perf_counter() - start < 0.1


def test_clip_refuses_forward_mode():
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        g = forward_ad.make_dual(torch.ones(3), torch.ones(3))
        with pytest.raises(NotImplementedError, match="tangents"):
            clip_grad_norm_([param(torch.ones(2)), param(g)], 1.0)
        with pytest.raises(NotImplementedError, match="tangents"):
            get_total_norm([g])
        with pytest.raises(RuntimeError, match="CUDA"):
            get_total_norm([torch.ones(3)])


def test_clip_without_gradients():
    assert clip_grad_norm_([torch.nn.Parameter(torch.ones(2))], 1.0).item() == 0
    assert clip_grads_with_norm_([], 1.0, torch.ones(())) is None


@pytest.mark.parametrize("view,want", [
    (lambda x: x, (True, False)), (lambda x: x.t(), (True, False)), (lambda x: x[:, 1:], (False, False)),
    (lambda x: x[::2], (False, False)), (lambda x: x[:1].expand(4, 6), (False, True)),
    (lambda x: x.as_strided((4, 4), (2, 1)), (False, True)), (lambda x: x[:, :1], (False, False)),
    (lambda x: x[1:2], (True, False))])
def test_layout(view, want):
    assert _layout(view(torch.zeros(8, 6))) == want


def test_clip_c_entry_checks():
    L = _lib.lib()
    bad = [(0, 5, 0), (4096, -1, 0), (4096, 5, 3), (4097, 5, 0), (4096, 1 << 48, 0)]
    for row in bad:
        t = array("q", row)
        assert L.scao_grads_overlap(t.buffer_info()[0], 1) == -1
        assert L.scao_grad_norm(t.buffer_info()[0], 1, 1, 4096, 4096, None) == 1
    t = array("q", (4096, 5, 0, 4096 + 20, 3, 1, 0, 0, 0))
    assert L.scao_grads_overlap(t.buffer_info()[0], 3) == 0
    t[3] = 4096 + 18
    assert L.scao_grads_overlap(t.buffer_info()[0], 3) == 1
    assert L.scao_grad_norm(t.buffer_info()[0], 3, 7, 4096, 4096, None) == 1       # no such norm
    assert L.scao_grad_norm(t.buffer_info()[0], 3, 1, 4096, None, None) == 1       # nowhere to write
    assert L.scao_grad_norm_clip(t.buffer_info()[0], 3, 1, -1.0, 4096, 4096, None) == 1
    assert L.scao_grad_norm_workspace_bytes(1) <= L.scao_grad_norm_workspace_bytes(5000)


def test_c_entries_refuse_misaligned_addresses():
    """Scalars, workspaces and positions that do not lie as their types need."""
    L = _lib.lib()
    t = array("q", (4096, 5, 0))
    at = t.buffer_info()[0]
    for ws, total in ((4100, 4096), (4096, 4098)):
        assert L.scao_grad_norm(at, 1, 1, ws, total, None) == 1
        assert L.scao_grad_norm_clip(at, 1, 1, 1.0, ws, total, None) == 1
    assert L.scao_grad_clip(at, 1, 1.0, 4097, None) == 1
    turns = (ctypes.c_double * 4)(*[0.1] * 4)
    for pos, wide in ((4098, 0), (4097, 0), (4100, 1)):
        a = _lib.RotaryArgs()
        a.turns, a.dim, a.head_dim, a.batch, a.len, a.dtype = ctypes.addressof(turns), 8, 8, 1, 1, 0
        a.heads[0], a.positions, a.positions_64 = 1, pos, wide
        a.src[0] = a.dst[0] = 4096
        assert L.scao_rotary(ctypes.byref(a), None) == 1, (pos, wide)


@pytest.mark.filterwarnings("ignore")
def test_clip_refuses_traces():
    """torch.jit.trace would record the norm as it was allocated."""
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda g: get_total_norm([g]), torch.ones(3), check_trace=False)
    p = param(torch.ones(3))
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda g: clip_grad_norm_([p], 1.0) * g, torch.ones(3), check_trace=False)


@pytest.mark.parametrize("pre_dispatch", [False, True])
def test_fx_traces_are_refused(pre_dispatch):
    from torch.fx.experimental.proxy_tensor import make_fx

    from scao_b200.cuda import _launch

    def call(x):
        y = x.new_empty(3)
        _launch("scao_rotary", 0, lambda *args: 0)
        return y

    with pytest.raises(RuntimeError, match="scao_rotary cannot be traced"):
        make_fx(call, pre_dispatch=pre_dispatch)(torch.ones(3))


# -------------------------------------------------------------------- rotary
@pytest.mark.parametrize("dim", [0, 1, 3, -2, 514])
def test_rotary_refuses_dims(dim):
    with pytest.raises(ValueError, match="dim"):
        Rotary(dim)


@pytest.mark.parametrize("make", [
    lambda: Rotary(8, base=0.0), lambda: Rotary(8, base=math.inf), lambda: RotaryScaling("cubic", 2.0),
    lambda: RotaryScaling("linear", 0.5), lambda: RotaryScaling("linear", math.nan),
    lambda: RotaryScaling("yarn", 2.0), lambda: RotaryScaling("yarn", 2.0, original_len=0),
    lambda: RotaryScaling("yarn", 2.0, original_len=9, fast=1, slow=2),
    lambda: Rotary(2, scaling=RotaryScaling("ntk", 2.0))])
def test_rotary_refuses_settings(make):
    with pytest.raises(ValueError):
        make()


def test_rotary_refuses_tensors():
    r = Rotary(8)
    q = torch.zeros(2, 3, 5, 8)
    for args in ((q[0],), (q[..., :6],), (q, q[:1]), (q, q[:, :, :4]), (q, q.double().float()[..., :7]),
                 (q, q.half())):
        with pytest.raises(ValueError):
            r(*args)
    with pytest.raises(TypeError, match="dtype"):
        r(q.double())
    for p in (torch.zeros(4, dtype=torch.long), torch.zeros(3, 5, dtype=torch.long),
              torch.zeros(1, 1, 5, dtype=torch.long), 1 << 60):
        with pytest.raises(ValueError):
            r(q, positions=p)
    with pytest.raises(TypeError, match="int32 or int64"):
        r(q, positions=torch.zeros(5))
    with pytest.raises(TypeError):
        r(q, positions=2.5)
    with pytest.raises(RuntimeError, match="CUDA"):
        r(q)


def test_rotary_frequencies():
    plain = Rotary(64).frequencies
    assert plain[0] == 1.0 and math.isclose(plain[-1], 10000 ** (-62 / 64))
    ntk = Rotary(64, scaling=RotaryScaling("ntk", 8.0)).frequencies
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / 8)
    yarn = Rotary(64, scaling=RotaryScaling("yarn", 8.0, original_len=8192))
    assert yarn.frequencies[0] == plain[0] and math.isclose(yarn.frequencies[-1], plain[-1] / 8)
    assert math.isclose(yarn.magnitude, 0.1 * math.log(8) + 1)
    assert all(p / 8 <= y <= p for p, y in zip(plain, yarn.frequencies))


def test_rotary_copies_and_pickles():
    r = Rotary(8, base=500.0, scaling=RotaryScaling("linear", 2.0))
    for c in (copy.deepcopy(r), pickle.loads(pickle.dumps(r))):
        assert c._turns == r._turns and c.scaling == r.scaling and c.dim == 8


# --------------------------------------------------------------- gated_ff
def test_gated_ff_refusals():
    b = torch.bfloat16
    x, w = torch.zeros(3, 8, dtype=b), torch.zeros(5, 8, dtype=b)
    with pytest.raises(ValueError, match="activation"):
        gated_ff(x, w, w, activation="relu")
    with pytest.raises(ValueError, match="activation"):
        GatedFeedForward(8, 16, "tanh")
    for args in ((x, w, w[:4]), (x[:, :7], w, w), (x, w[0], w[0]), (x[0, 0], w, w), (x, w[:, :7], w)):
        with pytest.raises(ValueError, match="must be"):
            gated_ff(*args)
    with pytest.raises(ValueError, match="no values"):
        gated_ff(x, w[:0], w[:0])
    for args in ((x.float(), w.float(), w.float()), (x, w.half(), w), (x.half(), w, w), (x.double(),) * 3):
        with pytest.raises((TypeError, ValueError)):
            gated_ff(*args)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_ff(x, w, w)


def test_gated_ff_c_entry_checks():
    L = _lib.lib()
    good = dict(x=4096, w_gate=4096, w_up=4096, h=4096, saved=4096, dh=4096, dx=4096, workspace=4096,
                ldx=8, ldg=8, ldu=8, lddh=5, rows=3, d=8, ff=5, dtype=_lib.BF16, act=0)

    def call(f, **kw):
        a = _lib.GatedFfArgs()
        for k, v in {**good, **kw}.items():
            setattr(a, k, v)
        return f(ctypes.byref(a), None)

    both = (dict(x=4104), dict(x=None), dict(w_gate=4098), dict(ldx=12), dict(ldg=0), dict(ldu=-8), dict(d=0),
            dict(ff=0), dict(rows=-1), dict(dtype=0), dict(dtype=3), dict(act=3), dict(act=-1), dict(d=9))
    for kw in both:
        assert call(L.scao_gated_ff_forward, **kw) == 1, kw
        assert call(L.scao_gated_ff_backward, **kw) == 1, kw
    assert call(L.scao_gated_ff_forward, h=None) == 1
    assert call(L.scao_gated_ff_forward, rows=0) == 0
    for kw in (dict(saved=None), dict(dh=None), dict(workspace=None), dict(workspace=4104), dict(dw_gate=4096),
               dict(dw_up=4096), dict(rows=0)):
        assert call(L.scao_gated_ff_backward, **kw) == 1, kw
    assert L.scao_gated_ff_forward(None, None) == 1
    assert L.scao_gated_ff_saved_bytes(1, 1) == 128 * 128 * 6
    assert L.scao_gated_ff_workspace_bytes(0, 1, 1, 3) == L.scao_gated_ff_workspace_bytes(1, 1, 1, 0) == 0
    for which in (1, 2, 3):         # dg and du at least
        assert L.scao_gated_ff_workspace_bytes(300, 65, 129, which) >= 2 * 2 * 300 * 136
    good = [4096, 8192, 3, 5, 7]
    for i, v in ((0, 0), (0, 4097), (1, 0), (1, 8200), (2, 0), (3, 0), (3, 1 << 25), (4, -1)):
        t = array("q", good[:i] + [v] + good[i + 1:])
        assert L.scao_gated_ff_pack(t.buffer_info()[0], 1, None) == 1, (i, v)
    t = array("q", good * 4)
    assert L.scao_gated_ff_pack(t.buffer_info()[0], 4, None) == 1
    assert L.scao_gated_ff_pack(t.buffer_info()[0], 0, None) == 1


def test_gated_ff_c_entry_alignment():
    """Addresses that the kernels cannot read or write are refused: values of 16 bits at odd
    bytes, what is kept for the gradient off its 16 bytes."""
    L = _lib.lib()
    good = dict(x=4096, w_gate=4096, w_up=4096, h=4096, saved=4096, dh=4096, dx=4096, dw_gate=4096, dw_up=4096,
                workspace=4096, ldx=8, ldg=8, ldu=8, lddh=5, rows=3, d=8, ff=5, dtype=_lib.BF16, act=0)

    def call(f, **kw):
        a = _lib.GatedFfArgs()
        for k, v in {**good, **kw}.items():
            setattr(a, k, v)
        return f(ctypes.byref(a), None)

    for at in (4097, 4098, 4100, 4104):
        assert call(L.scao_gated_ff_forward, saved=at) == 1
        assert call(L.scao_gated_ff_backward, saved=at) == 1
    assert call(L.scao_gated_ff_forward, h=4097) == 1
    for k in ("dh", "dx", "dw_gate", "dw_up"):
        assert call(L.scao_gated_ff_backward, **{k: 4097}) == 1, k


def test_gated_ff_tile_paths():
    """The sizes of the GPU tests still reach the tile paths that they stand for; together all."""
    seen = set()
    for sizes, paths in PATHS.items():
        for which, *want in paths:
            assert plan(*sizes, which) == tuple(want), (sizes, which)
            tile, dx, dw, several = want
            seen.add((which > 0, tile, several))
            if which:
                seen.add((tile, "dx", dx > 1))
                seen.add((tile, "dw", dw > 1))
    assert {(False, t, True) for t in range(3)} | {(True, PAIR, True), (True, TALL, True)} <= seen
    assert {(PAIR, "dx", True), (PAIR, "dw", True), (SINGLE, "dx", True), (SINGLE, "dw", True)} <= seen


def test_gated_ff_plan_checks():
    L, out = _lib.lib(), (ctypes.c_int32 * 5)()
    for args in ((0, 8, 8, 3), (8, 0, 8, 3), (8, 8, -1, 0), (8, 8, 8, 4), (8, 8, 8, -1)):
        assert L.scao_gated_ff_plan(*args, out) == 1, args
    assert L.scao_gated_ff_plan(8, 8, 8, 3, None) == 1
    assert L.scao_gated_ff_plan((1 << 31) - 1, 8, 1 << 22, 0, out) == 1        # more tiles than a launch takes


# ----------------------------------------------------------------- the model
@pytest.mark.parametrize("kw", [dict(mlp="moe"), dict(positions="none"), dict(n_kv_head=5), dict(n_kv_head=0)])
def test_gpt_config_refuses(kw):
    with pytest.raises(ValueError):
        gpt.GPTConfig(**kw)


def test_gpt_shapes():
    c = gpt.GPTConfig(n_layer=1, d_model=32, n_head=4, d_ff=48, vocab=50, seq_len=8, mlp="gated",
                      positions="rotary", n_kv_head=2)
    names = {n: tuple(p.shape) for n, p in gpt.GPT(c).named_parameters()}
    assert names["blocks.0.attn.qkv.weight"] == (64, 32) and names["blocks.0.ff.gate.weight"] == (48, 32)
    assert names["blocks.0.ff.out.weight"] == (32, 48) and not any("pos" in n or ".fc" in n for n in names)
    plain = dict(n_layer=1, d_model=32, n_head=4, d_ff=48, vocab=50, seq_len=8)
    logits = gpt.GPT(gpt.GPTConfig(**plain))(torch.arange(8)[None])          # the default runs on the CPU
    assert logits.shape == (1, 8, 50)


def test_rotary_c_entry_checks():
    L = _lib.lib()
    turns = (ctypes.c_double * 4)(*[0.1] * 4)

    def call(**kw):
        a = _lib.RotaryArgs()
        a.turns, a.dim, a.head_dim, a.batch, a.len, a.dtype = ctypes.addressof(turns), 8, 8, 1, 1, 0
        a.heads[0] = 1
        a.src[0] = a.dst[0] = 4096
        for k, v in kw.items():
            if k in ("src", "dst"):
                getattr(a, k)[0] = v
            else:
                setattr(a, k, v)
        return L.scao_rotary(ctypes.byref(a), None)

    for kw in (dict(dim=7), dict(dim=0), dict(dim=10), dict(dtype=3), dict(batch=-1), dict(turns=None),
               dict(src=None), dict(dst=4098)):
        assert call(**kw) == 1, kw
    assert call(batch=0) == 0
    assert L.scao_rotary(None, None) == 1


def test_packed_arguments_match_the_structs():
    """The packed forms that the calls pass have the fields of the C structs."""
    from scao_b200 import feedforward, rotary
    assert rotary._ARGS.size == ctypes.sizeof(_lib.RotaryArgs)
    assert feedforward._ARGS.size == ctypes.sizeof(_lib.GatedFfArgs)
    a = _lib.GatedFfArgs.from_buffer_copy(feedforward._ARGS.pack(*range(1, 21)))
    assert [getattr(a, n) for n, _ in a._fields_] == list(range(1, 21))
    b = _lib.RotaryArgs.from_buffer_copy(rotary._ARGS.pack(*range(1, 34)))
    assert [b.src[0], b.dst[1], b.src_stride[1][0], b.dst_stride[1][2], b.turns, b.positions, b.pos_stride_b,
            b.start, b.heads[1], b.dtype, b.inverse, b.factor] == [1, 4, 8, 16, 17, 18, 19, 21, 23, 24, 31, 32]


def test_model_copies_and_saves(tmp_path):
    c = gpt.GPTConfig(n_layer=1, d_model=32, n_head=4, d_ff=48, vocab=50, seq_len=8, mlp="gated",
                      positions="rotary", rotary_scaling=RotaryScaling("yarn", 4.0, original_len=8))
    m = gpt.GPT(c)
    torch.save(m, tmp_path / "m.pt")
    for other in (copy.deepcopy(m), torch.load(tmp_path / "m.pt", weights_only=False)):
        assert other.blocks[0].attn.rotary._turns == m.blocks[0].attn.rotary._turns
        assert all(torch.equal(a, b) for a, b in zip(m.parameters(), other.parameters()))
    with pytest.raises(RuntimeError, match="CUDA"):
        m(torch.arange(8)[None])
