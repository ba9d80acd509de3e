"""rotary against its definition in 64 bits, and its gradient against the formula's and
differences.

Bounds.  The angle's fraction of a turn is rounded to fp32 from 64 bits (|t| <= 1 half turns: 2^-25
of one, pi * 2^-25 < 2^-23 rad), sine and cosine are off by 2 steps of 2^-24 and their product with the
gain by one: (2^-23 + 3 * 2^-24) * gain * (|a| + |b|), with three roundings of the products
and sum 2^-24 of that each: below 8 * 2^-24 = 2^-21 of gain * (|a| + |b|); then half a step of the
type.  64 bits themselves leave |position * turns| * 2^-53 turns twice: 2^-20 rad at 2^31 for
turns of 1, added where it counts."""
import math

import pytest
import torch

from oracle import page_select as S

DEV = "cuda"
pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def freqs_of(R, base=10000.0, gain=1.0):
    from flashvsr_sm89_ops import RotaryFrequencies
    return RotaryFrequencies(base ** (-torch.arange(0, R, 2).double() / max(R, 1)) / (2 * math.pi), gain)


def on_gpu(f):
    return type(f)(f.turns.to(DEV), f.gain)


def check(got, x, f, pos, pairs, back=False):
    """got of x [B, S, H, D] (CPU)."""
    R = 2 * f.turns.numel()
    want = S.rotated(x, f.turns, f.gain, pos, pairs, back)
    size = x.double().abs().clone()
    half = R // 2
    a, b = (size[..., :half], size[..., half:R]) if pairs == "half" else \
        (size[..., 0:R:2], size[..., 1:R:2])
    both = a + b
    size[..., :R] = torch.cat([both, both], -1) if pairs == "half" else both.repeat_interleave(2, -1)
    far = 0 if pos is None else float(pos.abs().max())
    angle = 2 * math.pi * far * 2.0 ** -52 * float(f.turns.max() if R else 0)
    t = torch.finfo(x.dtype)
    tol = t.eps / 2 * want.abs() + (2.0 ** -21 + angle) * abs(f.gain) * size + t.smallest_normal * t.eps
    got = got.cpu()
    assert got.dtype == x.dtype and got.shape == x.shape
    ok = ((got.double() - want).abs() <= tol) | (torch.isnan(got) & torch.isnan(want)) | \
        (got.double() == want)
    assert bool(ok.all()), float((got.double() - want).abs().nan_to_num().max())
    assert torch.equal(got[..., R:].nan_to_num(nan=7.0), x[..., R:].nan_to_num(nan=7.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("D,R", [(128, 128), (128, 64), (64, 64), (64, 16), (80, 32), (96, 96),
                                 (40, 36), (24, 8), (2, 2), (7, 4), (5, 0), (256, 240)])
def test_heads(dtype, pairs, D, R):
    """Whole and part heads, widths that vectors hold and that they do not."""
    from flashvsr_sm89_ops import rotary
    B, T, Hq, Hk = 2, 5, 3, 2
    q, k = (torch.randn(B, T, h, D, generator=gen(h)).to(dtype) for h in (Hq, Hk))
    f, pos = freqs_of(R, gain=1.25), torch.tensor([0, 1, 77, 100000, -3], dtype=torch.int32)
    oq, ok = rotary(q.to(DEV), k.to(DEV), on_gpu(f), pos.to(DEV), pairs=pairs)
    check(oq, q, f, pos, pairs)
    check(ok, k, f, pos, pairs)
    alone = rotary(q.to(DEV), None, on_gpu(f), pos.to(DEV), pairs=pairs)
    assert torch.equal(alone, oq)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,pshape", [((1, 1, 4, 128), (1,)), ((3, 7, 2, 64), (3, 7)),
                                          ((2, 300, 5, 64), (300,)), ((9, 2, 64), (9,)),
                                          ((2, 33, 3, 64), None), ((700, 12, 128), None)])
def test_positions(dtype, shape, pshape):
    from flashvsr_sm89_ops import rotary
    x = torch.randn(shape, generator=gen(1)).to(dtype)
    f = freqs_of(shape[-1])
    pos = None if pshape is None else torch.randint(-50000, 1000000, pshape, generator=gen(2)).int()
    out = rotary(x.to(DEV), None, on_gpu(f), None if pos is None else pos.to(DEV))
    four = x if x.dim() == 4 else x[None]
    check(out if out.dim() == 4 else out[None], four, f, pos, "half")


def test_far_positions():
    """Up to the ends of int32, where 32-bit angles would be off by whole turns."""
    from flashvsr_sm89_ops import rotary
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, 16777217, 1], dtype=torch.int32)
    x = torch.randn(1, 5, 2, 64, generator=gen(0))
    for base in (10000.0, 1.5):
        f = freqs_of(64, base)
        check(rotary(x.to(DEV), None, on_gpu(f), pos.to(DEV)), x, f, pos, "half")


@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", TYPES)
def test_strides(pairs, dtype):
    """Columns of one projection, heads before tokens, odd offsets, rows that share their place."""
    from flashvsr_sm89_ops import rotary
    D, f = 64, freqs_of(32)
    base = torch.randn(2, 9, 8 * D + 6, generator=gen(0)).to(dtype)
    views = [base[..., :6 * D].unflatten(-1, (6, D)), base[..., 3:3 + 4 * D].unflatten(-1, (4, D)),
             base[..., 8:8 + 4 * D].unflatten(-1, (4, D)).transpose(1, 2),
             base[:1, :, :4 * D].unflatten(-1, (4, D)).expand(2, 9, 4, D),
             base[..., :2 * D:2].unflatten(-1, (1, D)),
             base[0, 0, :D].expand(2, 9, 3, D)]
    dev = base.to(DEV)
    for v in views:
        d = torch.as_strided(dev, v.shape, v.stride(), v.storage_offset())
        out = rotary(d, d, on_gpu(f), pairs=pairs)
        for o in out:
            check(o, v, f, None, pairs)
            assert o.is_contiguous()


def test_special_values():
    """Infinities and NaN stay in their pair; subnormals; copied channels keep their bits."""
    from flashvsr_sm89_ops import rotary
    for dtype in TYPES:
        x = torch.randn(1, 4, 2, 64, generator=gen(0)).to(dtype)
        x[0, 1, 0, 3], x[0, 2, 1, 40], x[0, 3, 0, 63] = math.nan, math.nan, math.nan
        x[0, 0, 0] = torch.finfo(dtype).smallest_normal / 4
        f = freqs_of(32)
        check(rotary(x.to(DEV), None, on_gpu(f)), x, f, None, "half")
        x[0, 1, 1, 0] = math.inf
        out = rotary(x.to(DEV), None, on_gpu(f))
        assert not bool(torch.isfinite(out[0, 1, 1, 0])) and bool(torch.isfinite(out[0, 1, 1, 1:16]).all())


def test_nothing():
    from flashvsr_sm89_ops import rotary
    f = on_gpu(freqs_of(64))
    for shape in ((0, 4, 64), (2, 0, 3, 64), (5, 0, 64), (0, 3, 2, 64)):
        assert rotary(torch.empty(shape, device=DEV), None, f).shape == shape


@pytest.fixture(params=["native", "general"])
def path(request, monkeypatch):
    """Both ways that a call can take on the host."""
    from flashvsr_sm89_ops import _lib
    _lib.selected_host()
    if request.param == "general":
        monkeypatch.setattr(_lib, "_selected_host", _lib._GeneralPath)
    return request.param


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("D,R", [(128, 128), (64, 32), (24, 20)])
def test_gradient(dtype, pairs, D, R, path):
    """dq and dk are the rotation back of the gradients, whatever their layout, and q's or k's
    alone where only one is asked for."""
    from flashvsr_sm89_ops import rotary
    B, T, Hq, Hk = 2, 6, 4, 2
    f = freqs_of(R, gain=1.5)
    pos = torch.randint(0, 5000, (B, T), generator=gen(4)).int()
    x = torch.randn(B, T, Hq + Hk, D, generator=gen(0)).to(dtype).to(DEV)
    q, k = x[:, :, :Hq].detach().requires_grad_(), x[:, :, Hq:].detach().requires_grad_()
    oq, ok = rotary(q, k, on_gpu(f), pos.to(DEV), pairs=pairs)
    gq, gk = (torch.randn(B, T, h, D, generator=gen(h)).to(dtype) for h in (Hq, Hk))
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq.to(DEV), gk.to(DEV)), retain_graph=True)
    check(dq, gq, f, pos, pairs, back=True)
    check(dk, gk, f, pos, pairs, back=True)
    strided = gq.transpose(1, 2).contiguous().transpose(1, 2)
    d2, = torch.autograd.grad(oq, q, strided.to(DEV), retain_graph=True)
    assert torch.equal(d2, dq)
    d3, = torch.autograd.grad(ok.sum(), k, retain_graph=True)  # one value for every element
    check(d3, torch.ones_like(gk), f, pos, pairs, back=True)
    d4, = torch.autograd.grad((oq, ok), k, (gq.to(DEV), gk.to(DEV)))
    assert torch.equal(d4, dk)


def test_gradient_of_one_input_and_shared_heads(path):
    """k without a gradient; one k spread over heads (a broadcast) gets the sum."""
    from flashvsr_sm89_ops import rotary
    f = on_gpu(freqs_of(64))
    q = torch.randn(3, 2, 64, device=DEV, requires_grad=True)
    k = torch.randn(3, 2, 64, device=DEV)
    oq, ok = rotary(q, k, f)
    assert ok.requires_grad and oq.requires_grad  # (outputs of one node)
    oq.backward(torch.ones_like(oq))
    assert q.grad is not None and k.grad is None
    one = torch.randn(3, 1, 64, device=DEV, requires_grad=True)
    g = torch.randn(3, 4, 64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))
    out = rotary(one.expand(3, 4, 64), None, f)
    d, = torch.autograd.grad(out, one, g)
    want = S.rotated(g.cpu()[None], freqs_of(64).turns, 1.0, None, "half", True)[0].sum(1, keepdim=True)
    assert bool(((d.cpu().double() - want).abs() <= 2.0 ** -20 * g.cpu().abs().sum(1).max()).all())


def test_gradient_by_differences(path):
    """fp32, the derivative of a random product along a random direction.  The map is linear, so a
    difference over a step of 1 has no error of its own: both sides are sums of 768 products
    that fp32 rounds, 2^-21 of their magnitudes each (the bound above)."""
    from flashvsr_sm89_ops import rotary
    f = on_gpu(freqs_of(48, gain=1.3))
    g = torch.Generator(device=DEV).manual_seed(0)
    q, d, w = (torch.randn(4, 3, 64, device=DEV, generator=g) for _ in range(3))
    q.requires_grad_()
    out = rotary(q, None, f, pairs="interleaved")
    dq, = torch.autograd.grad(out, q, w)
    slope = ((rotary(q.detach() + d, None, f, pairs="interleaved") - out.detach()).double() * w).sum()
    size = (w.abs().double() * (q.abs() + d.abs()).double()).sum() + (dq * d).abs().double().sum()
    assert float((slope - (dq.double() * d).sum()).detach().abs()) <= 3 * 2.0 ** -21 * 2 * 1.3 * float(size)


def test_second_gradient(path):
    from flashvsr_sm89_ops import rotary
    f = on_gpu(freqs_of(64))
    q = torch.randn(4, 2, 64, device=DEV, requires_grad=True)
    g = torch.randn(4, 2, 64, device=DEV, requires_grad=True)
    dq, = torch.autograd.grad(rotary(q, None, f), q, g, create_graph=True)
    w = torch.randn(4, 2, 64, device=DEV)
    dg, = torch.autograd.grad(dq, g, w)  # the rotation of w
    check(dg[None], w.cpu()[None], freqs_of(64), None, "half")


def test_nodes(path):
    """What a graph holds: no gradient without being asked, outputs of one node, positions changed
    between the two ways refused, backward on another thread's stream as on the caller's."""
    from flashvsr_sm89_ops import rotary
    f = on_gpu(freqs_of(64))
    q = torch.randn(4, 2, 64, device=DEV, requires_grad=True)
    pos = torch.arange(4, dtype=torch.int32, device=DEV)
    assert not rotary(q.detach(), None, f, pos).requires_grad
    with torch.no_grad():
        assert not rotary(q, None, f, pos).requires_grad
    with torch.inference_mode():
        rotary(q, None, f, pos)
    out, k = rotary(q, q.detach(), f, pos)
    assert out.grad_fn is not None and out.requires_grad and out.is_leaf is False
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out2 = rotary(q, None, f, pos)
        d2, = torch.autograd.grad(out2, q, torch.ones_like(out2))
    torch.cuda.current_stream().wait_stream(side)
    d, = torch.autograd.grad(out, q, torch.ones_like(out), retain_graph=True)
    assert torch.equal(d, d2)
    pos += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, q, torch.ones_like(out))
    empty = torch.empty(0, 2, 64, device=DEV, requires_grad=True)
    d, = torch.autograd.grad(rotary(empty, None, f).sum(), empty)
    assert d.shape == empty.shape


def test_graph_of_forward_and_backward(path):
    """Captured with leaves of its own, replayed with other inputs between eager steps."""
    from flashvsr_sm89_ops import rotary
    f = on_gpu(freqs_of(128))
    x, g = (torch.randn(2, 40, 4, 128, device=DEV).bfloat16() for _ in range(2))
    pos = torch.arange(40, dtype=torch.int32, device=DEV)

    def step(x):
        leaf = x.detach().requires_grad_()
        out = rotary(leaf, None, f, pos)
        return out.detach(), torch.autograd.grad(out, leaf, g)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step(x)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        x.normal_()
        g.normal_()
        pos += 1000
        want = step(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_capture_with_a_live_graph(monkeypatch):
    """Refused before anything is captured; once the outputs are gone the same leaf does."""
    from flashvsr_sm89_ops import rotary
    f = on_gpu(freqs_of(64))
    q = torch.randn(6, 2, 64, device=DEV, requires_grad=True)
    g = torch.randn(6, 2, 64, device=DEV)
    out = rotary(q, None, f)
    want, = torch.autograd.grad(out, q, g, retain_graph=True)
    with pytest.raises(RuntimeError, match="graph from another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            rotary(q, None, f)
    with pytest.raises(RuntimeError, match="graph from another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            rotary(q.detach(), q, f)
    from flashvsr_sm89_ops import _lib
    monkeypatch.setattr(_lib, "_selected_host", _lib._GeneralPath)  # by way of Python too
    with pytest.raises(RuntimeError, match="graph from another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            rotary(q.detach(), q, f)
    monkeypatch.undo()
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first, second = rotary(q, q, f)  # (a graph of the same stream is none to refuse)
        got, = torch.autograd.grad(rotary(q, None, f), q, g)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(first, second)


def test_no_forward_mode():
    from flashvsr_sm89_ops import rotary
    f = on_gpu(freqs_of(64))
    q = torch.randn(6, 2, 64, device=DEV)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(ValueError, match="forward-mode"):
            rotary(dual, None, f)
        with pytest.raises(ValueError, match="forward-mode"):
            rotary(q, dual, f)


def test_on_another_stream():
    from flashvsr_sm89_ops import rotary
    f = on_gpu(freqs_of(128))
    x = torch.randn(500, 8, 128, device=DEV)
    want = rotary(x, None, f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = x * 1.0
        out = rotary(y, None, f)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)


def test_offsets_past_32_bits():
    """2.2e9 values: rows at the end against the same rows alone."""
    from flashvsr_sm89_ops import rotary
    f = on_gpu(freqs_of(128))
    T, H = 70000, 250
    x = torch.zeros(T, H, 128, dtype=torch.bfloat16, device=DEV)
    x[-3:] = torch.randn(3, H, 128, device=DEV)
    pos = torch.arange(T, dtype=torch.int32, device=DEV)
    out = rotary(x, None, f, pos)
    assert torch.equal(out[-3:], rotary(x[-3:].clone(), None, f, pos[-3:]))
    assert not bool(out[:5].any())


@pytest.mark.parametrize("grad", [False, True])
def test_out_of_memory(path, grad):
    """Outputs that memory cannot hold are an exception like any other, and the next call works."""
    from flashvsr_sm89_ops import rotary
    f = on_gpu(freqs_of(128))
    one = torch.ones(1, 1, 128, device=DEV, requires_grad=grad)
    want = rotary(one, None, f)
    huge = one.expand(1 << 22, 1 << 10, 128)  # 2 TiB of results
    for args in ((huge, None), (one.expand(1 << 22, 1, 128), huge)):
        with pytest.raises(torch.OutOfMemoryError):
            rotary(*args, f)
    assert torch.equal(rotary(one, None, f), want)


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
@pytest.mark.filterwarnings("ignore:The AccumulateGrad node's stream")
def test_capture_with_a_live_graph_further_up(path, monkeypatch):
    """A leaf behind q and k (a projection's weight, or the rows that they are slices of) with an eager
    graph from another stream: its gradient is refused inside the capture, the call itself and gradients
    that stop before it are not."""
    from flashvsr_sm89_ops import _lib, rotary
    f = on_gpu(freqs_of(64))
    x = torch.randn(6, 4, 64, device=DEV, requires_grad=True)
    g = torch.randn(6, 3, 64, device=DEV)

    def step():
        y = x * 2
        return y, *rotary(y[:, :3], y[:, 3:], f)
    live = step()
    want_q, want_k = live[1].detach(), live[2].detach()
    want, = torch.autograd.grad(live[1], x, g, retain_graph=True)
    for inputs in ((x,), None):
        with pytest.raises(RuntimeError, match="graph from another stream"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                y, q, k = step()
                torch.autograd.grad(q, x, g) if inputs else q.backward(g)
        del y, q, k
    assert x.grad is None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, q, k = step()
        dy, = torch.autograd.grad(q, y, g)
    for _ in range(3):
        dy.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(2 * dy, want)
    del live, y, q, k, dy, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, q, k = step()
        dx, = torch.autograd.grad(q, x, g)
    for _ in range(3):
        dx.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, want)
    del y, q, k, dx, graph
    monkeypatch.setattr(_lib, "_host", _lib._GeneralPath)  # (leaves are not seen from there)
    monkeypatch.setattr(_lib, "_selected_host", _lib._GeneralPath)
    with pytest.raises(RuntimeError, match="native extension"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(step()[1], x, g)
    dx, = torch.autograd.grad(step()[1], x, g)
    assert torch.equal(dx, want)


@pytest.mark.filterwarnings("ignore:The AccumulateGrad node's stream")
def test_capture_over_two_streams(path):
    """A captured step that goes over two streams: a leaf's graph from the other one is of the same
    capture."""
    from flashvsr_sm89_ops import rotary
    f = on_gpu(freqs_of(64))
    x, g = (torch.randn(6, 3, 64, device=DEV) for _ in range(2))
    side = torch.cuda.Stream()

    def step(x):
        leaf = x.detach().requires_grad_()
        here = torch.cuda.current_stream()
        first = rotary(leaf, None, f)
        side.wait_stream(here)
        with torch.cuda.stream(side):
            second = rotary(leaf, None, f, pairs="interleaved")
        here.wait_stream(side)
        d, = torch.autograd.grad((first, second), leaf, (g, g))
        return first.detach(), second.detach(), d
    step(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x)
    for i in range(3):
        x.normal_()
        g.normal_()
        want = step(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("D", [64, 66])
@pytest.mark.parametrize("pos", [1, 1000003])
@pytest.mark.parametrize("back", [False, True])
def test_angles_of_fp32(pairs, D, pos, back):
    """Angles 0.001 to 0.01 turns beside a quarter: the cosine is small, so a rounding of the angle to 24
    bits, up to 2^-25 half turns, would be far more than steps of its own.  Of (1, 0) and (0, 1): sine and
    cosine 2 units of the last place, 2^-22 of themselves, one more rounding; products with 1 and 0
    are exact.  What 64 bits leave of the angle is below 2^-30 turns of 2^-10."""
    from flashvsr_sm89_ops import RotaryFrequencies, rotary
    g = gen(D)
    off = (0.001 + 0.009 * torch.rand(32, generator=g).double()) * (1 - 2 * (torch.arange(32) % 2))
    turns = (torch.randint(0, 1000, (32,), generator=g) * (pos > 1) + 0.25 + off) / pos
    f, p = RotaryFrequencies(turns, 1.0), torch.tensor([pos], dtype=torch.int32)
    x = torch.zeros(1, 1, 2, D)
    x[0, 0, 0, :32] = 1.0
    x[0, 0, 1, 32:64] = 1.0
    if pairs == "interleaved":
        x[..., :64] = x[..., :64].unflatten(-1, (2, 32)).transpose(-1, -2).flatten(-2)
    if back:
        q = torch.zeros_like(x, device=DEV).requires_grad_()
        got, = torch.autograd.grad(rotary(q, None, on_gpu(f), p.to(DEV), pairs=pairs), q, x.to(DEV))
    else:
        got = rotary(x.to(DEV), None, on_gpu(f), p.to(DEV), pairs=pairs)
    want = S.rotated(x, turns, 1.0, p, pairs, back)
    tol = 2.0 ** -21 * want.abs() + 2.0 ** -40
    assert bool(((got.cpu().double() - want).abs() <= tol).all()), \
        float(((got.cpu().double() - want).abs() / tol).max())
