"""GPU parity of the rotary operator against the 64-bit oracle, through the public API.

Tolerance, derived: the kernel rounds once to the output type (half a step, eps / 2 of the value;
for fp16 at least half its smallest step, 2^-25) after 32-bit arithmetic.  cos and sin, from an
angle reduced in 64 bits, are off by less than 2^-22 (the reduced angle's rounding to 32 bits,
pi 2^-25, and the function's last places), a product and the sum add 2^-24 of each term, so the
32-bit value is off by less than scale (|x| + |y|) 2^-21.
"""
import pytest
import torch

from oracle import serving_oracle as orc
from tests._pkg import pkg, submodule

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def table(n, base=150000.0):
    return (base ** (-torch.arange(n, dtype=torch.float64) / max(1, n))).float()


def tolerance(x, ref, n, scale, interleaved):
    """Elementwise bound for outputs ref of inputs x."""
    eps = torch.finfo(x.dtype).eps / 2
    size = x.double().cpu().abs()
    pair = size.clone()
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    pair[..., a] = pair[..., b] = size[..., a] + size[..., b]
    floor = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    wide = abs(scale) * pair * 2.0 ** -21
    return (eps * (ref.abs() + wide)).clamp_min(floor) + wide


def check(x, y, pos, inv, axes, interleaved, scale, inverse=False):
    ref = orc.rotary(x, pos, inv, axes, interleaved, scale, inverse)
    err = (y.detach().double().cpu() - ref).abs()
    n = inv.numel()
    assert bool((err <= tolerance(x.detach(), ref, n, scale, interleaved)).all()), err.max()
    # what is not rotated is copied
    assert torch.equal(y[..., 2 * n:].cpu(), x[..., 2 * n:].cpu())


def positions(g, axes, b, l, first, dtype=torch.int64):
    return torch.randint(0, 5000, (axes, b, l), generator=g).to(dtype) + first


CASES = [
    # b, hq, hkv, l, d, sections, interleaved, scale, first position
    (2, 8, 2, 300, 64, (32,), False, 1.0, 0),
    (1, 4, 4, 1, 64, (32,), False, 1.0, 0),
    (1, 64, 8, 129, 64, (12, 10, 10), False, 1.25, 120000),
    (3, 5, 1, 33, 128, (16, 24, 24), False, 1.0, 1 << 20),
    (2, 4, 2, 65, 128, (64,), True, 0.5, 1 << 30),
    (2, 3, 3, 17, 16, (2, 3, 3), True, 1.0, 0),
    (1, 2, 1, 257, 32, (6, 8), False, 1.0, 7),           # 28 of 32 values turned
    (2, 6, 2, 40, 80, (20, 10, 10), False, 1.0, 0),      # heads that are no kernel size
    (1, 3, 1, 50, 10, (2, 1), False, 2.0, 3),            # rows that are not 16-byte aligned
    (1, 2, 2, 5, 64, (), False, 1.0, 0),                 # nothing is turned
    (1, 1, 1, 2050, 64, (32,), False, 1.0, 0),
    (70, 8, 8, 1, 64, (32,), False, 1.0, 4000),          # one token each
    (300, 2, 1, 3, 48, (8, 8), True, 1.0, 100),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=[f"{c[0]}x{c[1]}x{c[3]}x{c[4]}-{'i' if c[6] else 'h'}{len(c[5])}" for c in CASES])
def test_rotary_forward_and_gradient(case, dtype):
    b, hq, hkv, l, d, sections, interleaved, scale, first = case
    g = torch.Generator().manual_seed(b + l + d)
    n = sum(sections)
    inv = table(n)
    axes = [a for a, x in enumerate(sections) for _ in range(x)]
    pos = positions(g, max(1, len(sections)), b, l, first)
    rot = pkg().Rotary(inv.to(DEV), sections=sections or None, interleaved=interleaved, scale=scale)
    q, k, dq, dk = (torch.randn(b, h, l, d, generator=g).to(dtype) for h in (hq, hkv, hq, hkv))
    qd, kd = (t.to(DEV).requires_grad_() for t in (q, k))
    shaped = pos.to(DEV) if len(sections) > 1 else pos[0].to(DEV)
    yq, yk = pkg().apply_rotary(qd, kd, shaped, rot)
    assert yq.shape == q.shape and yk.shape == k.shape and yq.dtype == dtype
    gq, gk = torch.autograd.grad((yq, yk), (qd, kd), (dq.to(DEV), dk.to(DEV)))
    p = pos[:, :, None]
    for x, y, inverse in ((q, yq, False), (k, yk, False), (dq, gq, True), (dk, gk, True)):
        check(x, y, p, inv, axes, interleaved, scale, inverse)


def test_gradient_against_differences():
    # the map is linear: <L(x + u) - L(x - u)> / 2 = <gradient, u> whatever the step, up to the
    # roundings of the four kernel results (half a step each)
    g = torch.Generator().manual_seed(2)
    rot = pkg().Rotary(table(32).to(DEV), sections=(12, 10, 10), scale=1.5)
    pos = positions(g, 3, 2, 37, 1000).to(DEV)
    q, u, w = (torch.randn(2, 4, 37, 64, generator=g).to(DEV) for _ in range(3))
    q, u, w = q.half(), (u / 8).half(), w.half()
    plus, minus = (q + u).requires_grad_(), (q - u)
    y1, _ = pkg().apply_rotary(plus, None, pos, rot)
    y0, _ = pkg().apply_rotary(minus, None, pos, rot)
    (grad,) = torch.autograd.grad(y1, plus, w)
    step = plus.detach().double() - minus.double()
    left = ((y1.detach().double() - y0.double()) * w.double()).sum()
    right = (grad.double() * step).sum()
    half = torch.finfo(torch.float16).eps / 2
    bound = half * (((y1.detach().double().abs() + y0.double().abs()) * w.double().abs()).sum()
                    + (grad.double().abs() * step.abs()).sum()) * 1.01
    assert abs(float(left - right)) <= float(bound)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_positions_shapes_and_types(dtype):
    g = torch.Generator().manual_seed(3)
    inv = table(16)
    rot1, rot3 = (pkg().Rotary(inv.to(DEV), sections=s) for s in ((16,), (6, 5, 5)))
    x = torch.randn(3, 2, 20, 32, generator=g).bfloat16()
    pos = positions(g, 3, 3, 20, 0, dtype)
    a1, a3 = [0] * 16, [0] * 6 + [1] * 5 + [2] * 5
    for p, rot, axes, full in ((pos[0], rot1, a1, pos[:1]), (pos[:1], rot1, a1, pos[:1]), (pos[0, 0], rot1, a1, pos[:1, :1]),
                               (pos, rot3, a3, pos), (pos[:, 0], rot3, a3, pos[:, :1]),
                               (pos.flip(2).transpose(1, 2).contiguous().transpose(1, 2), rot3, a3, pos.flip(2))):
        y, _ = pkg().apply_rotary(x.to(DEV), None, p.to(DEV), rot)
        check(x, y, full[:, :, None], inv, axes, False, 1.0)
    packed = x.permute(0, 2, 1, 3).reshape(60, 2, 32)
    y, z = pkg().apply_rotary(packed.to(DEV), packed.to(DEV), pos.reshape(3, 60).to(DEV), rot3)
    ref = pos.reshape(3, 1, 60)
    check(packed.transpose(0, 1), y.transpose(0, 1), ref, inv, a3, False, 1.0)
    assert torch.equal(y, z)


def test_axes_in_any_order():
    g = torch.Generator().manual_seed(4)
    inv = table(24)
    axes = [i % 3 for i in range(24)]
    rot = pkg().Rotary(inv.to(DEV), axes=axes)
    x = torch.randn(1, 3, 41, 64, generator=g).half()
    pos = positions(g, 3, 1, 41, 0)
    y, _ = pkg().apply_rotary(x.to(DEV), None, pos.to(DEV), rot)
    check(x, y, pos[:, :, None], inv, axes, False, 1.0)


def test_strides_broadcasts_and_offsets():
    # slices of one projection, transposed and expanded heads, a base that is not 16-byte aligned
    g = torch.Generator().manual_seed(5)
    inv, axes = table(32), [0] * 32
    rot = pkg().Rotary(inv.to(DEV))
    pos = positions(g, 1, 2, 77, 0)
    qkv = torch.randn(2, 77, 12, 64, generator=g).bfloat16().to(DEV)
    q, k = qkv[:, :, :8].transpose(1, 2), qkv[:, :, 8:10].transpose(1, 2)
    odd = torch.randn(2 * 3 * 77 * 64 + 1, generator=g).bfloat16().to(DEV)[1:].view(2, 3, 77, 64)
    wide = torch.randn(2, 1, 77, 64, generator=g).bfloat16().to(DEV).expand(2, 4, 77, 64)
    reverse = torch.randn(2, 3, 64, 77, generator=g).bfloat16().to(DEV).transpose(2, 3)
    for x, z in ((q, k), (odd, None), (wide, odd), (reverse, wide)):
        y, w = pkg().apply_rotary(x, z, pos[0].to(DEV), rot)
        check(x, y, pos[:, :, None], inv, axes, False, 1.0)
        if z is not None:
            check(z, w, pos[:, :, None], inv, axes, False, 1.0)
    # a broadcast input's gradient is the sum over its copies
    leaf = torch.randn(2, 1, 77, 64, generator=g).half().to(DEV).requires_grad_()
    y, _ = pkg().apply_rotary(leaf.expand(2, 4, 77, 64), None, pos[0].to(DEV), rot)
    y.sum().backward()
    one = torch.ones(2, 4, 77, 64, dtype=torch.float16)
    ref = orc.rotary(one, pos[:, :, None], inv, axes, inverse=True).sum(1, keepdim=True)
    # four equal terms, each off by half a step, summed by torch in fp16 (half a step of each partial sum)
    assert float((leaf.grad.double().cpu() - ref).abs().max()) <= 2.0 ** -11 * 1.42 * (4 + 2 + 3 + 4)


def test_in_place_through_the_library():
    import ctypes
    L, R = submodule("_lib"), submodule("rotary")
    g = torch.Generator().manual_seed(6)
    inv, pos = table(32), positions(g, 1, 2, 50, 9)
    rot = pkg().Rotary(inv.to(DEV))
    x = torch.randn(2, 4, 50, 64, generator=g).half()
    y = x.to(DEV)
    p = pos[0].to(DEV)
    t = R._tensor(y)
    t.ptr = y.data_ptr()
    none = L.SwaTensor(None, 0, 0, 0)
    args = L.SwaRotaryArgs(2, 4, 0, 50, 64, L.SWA_F16, 0, rot._bind(p, 2, 50), t, none, t, none)
    args.r.positions = p.data_ptr()
    assert L.lib().swa_rotary(ctypes.byref(args), torch.cuda.current_stream().cuda_stream) == 0
    check(x, y, pos[:, :, None], inv, [0] * 32, False, 1.0)


def test_empty_and_other_stream_and_graph():
    g = torch.Generator().manual_seed(7)
    inv = table(32)
    rot = pkg().Rotary(inv.to(DEV))
    e = torch.empty(2, 4, 0, 64, device=DEV, dtype=torch.float16)
    y, _ = pkg().apply_rotary(e, None, torch.empty(0, dtype=torch.int64, device=DEV), rot)
    assert y.shape == e.shape
    x = torch.randn(1, 4, 60, 64, generator=g).half().to(DEV)
    pos = positions(g, 1, 1, 60, 0)
    p = pos[0, 0].to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, _ = pkg().apply_rotary(x, None, p, rot)
    side.synchronize()
    check(x.cpu(), y, pos[:, :, None], inv, [0] * 32, False, 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z, _ = submodule("rotary").rotate(x, None, p, rot)
    x.copy_(torch.randn(1, 4, 60, 64, generator=g).half())
    p.add_(17)
    graph.replay()
    torch.cuda.synchronize()
    check(x.cpu(), z, pos[:, :, None] + 17, inv, [0] * 32, False, 1.0)


def test_refusals_and_second_gradient():
    rot = pkg().Rotary(table(32).to(DEV), sections=(16, 16))
    q = torch.randn(1, 2, 8, 64, device=DEV, dtype=torch.float16)
    pos = torch.zeros(2, 1, 8, dtype=torch.int64, device=DEV)
    for bad in (pos[:1], pos[:, :, :7], pos[0], pos.cpu(), torch.zeros(2, 2, 8, dtype=torch.int64, device=DEV)):
        with pytest.raises(ValueError):
            pkg().apply_rotary(q, None, bad, rot)
    with pytest.raises(TypeError):
        pkg().apply_rotary(q, None, pos.float(), rot)
    with pytest.raises(TypeError):
        pkg().apply_rotary(q.float(), None, pos, rot)
    for k in (q[:, :, :4], q[..., :32], q[0], q.cpu()):
        with pytest.raises(ValueError):
            pkg().apply_rotary(q, k, pos, rot)
    for x in (q[:, :0], q[..., :32], q[..., :63]):
        with pytest.raises(ValueError):
            pkg().apply_rotary(x, None, pos, rot)
    for kw in (dict(sections=(5, 5)), dict(sections=(33, -1)), dict(axes=[0] * 31), dict(axes=[0] * 32, sections=(32,)),
               dict(axes=[300] * 32), dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            pkg().Rotary(table(32).to(DEV), **kw)
    # the gradient of a gradient: the map and its transpose, once more
    x = q.clone().requires_grad_()
    u = torch.randn_like(q).requires_grad_()
    y, _ = pkg().apply_rotary(x, None, pos + 3, rot)
    (g,) = torch.autograd.grad(y, x, u, create_graph=True)
    (h,) = torch.autograd.grad(g, u, q)
    assert torch.equal(h, y.detach())


def test_attention_takes_the_rotation():
    g = torch.Generator().manual_seed(8)
    rot = pkg().Rotary(table(32).to(DEV), sections=(12, 10, 10))
    q, k, v, do = (torch.randn(2, h, 150, 64, generator=g).bfloat16().to(DEV).requires_grad_(h != 9)
                   for h in (8, 2, 2, 8))
    pos = positions(g, 3, 2, 150, 0).to(DEV)
    o = pkg().flash_swda_with_sink(q, k, v, 40, 4, rotary=rot, positions=pos)
    one = torch.autograd.grad(o, (q, k, v), do)
    yq, yk = pkg().apply_rotary(q, k, pos, rot)
    ref = pkg().flash_swda_with_sink(yq, yk, v, 40, 4)
    two = torch.autograd.grad(ref, (q, k, v), do)
    assert torch.equal(o, ref) and all(torch.equal(a, b) for a, b in zip(one, two))
    pack = lambda t: t.detach().transpose(1, 2).reshape(300, -1, 64)  # noqa: E731
    flat = pos.reshape(3, 300)
    o = pkg().flash_swda_with_sink_varlen(pack(q), pack(k), pack(v), [0, 150, 300], 40, 4, rotary=rot, positions=flat)
    assert torch.equal(o.view(2, 150, 8, 64).transpose(1, 2), ref)


def test_forward_mode_derivatives():
    fw = torch.autograd.forward_ad
    rot = pkg().Rotary(table(32).to(DEV), scale=1.5)
    pos = torch.arange(9, device=DEV) + 100
    q, k, u, w = (torch.randn(1, h, 9, 64, device=DEV).half() for h in (4, 2, 4, 2))
    turn = submodule("rotary").rotate
    want, values = turn(u, w, pos, rot), turn(q, k, pos, rot)
    for grad in (False, True):
        with torch.set_grad_enabled(grad), fw.dual_level():
            # both, one of them, and a leaf of a backward pass too
            for du, dw in ((u, w), (u, None), (None, w)):
                a = q if du is None else fw.make_dual(q.clone().requires_grad_(grad), du)
                b = k if dw is None else fw.make_dual(k, dw)
                ys = pkg().apply_rotary(a, b, pos, rot)
                for y, value, tangent, ref in zip(ys, values, (du, dw), want):
                    y = fw.unpack_dual(y)
                    assert torch.equal(y.primal, value)
                    if tangent is not None:
                        assert torch.equal(y.tangent, ref)
                    else:
                        assert y.tangent is None or not y.tangent.any()
            y, none = pkg().apply_rotary(fw.make_dual(q, u), None, pos, rot)
            assert none is None and torch.equal(fw.unpack_dual(y).tangent, want[0])
    # the attention has no forward mode and says so
    with fw.dual_level(), pytest.raises(RuntimeError):
        pkg().flash_swda_with_sink(fw.make_dual(q, u), k, k, 4, rotary=rot, positions=pos)
    # a tangent through the backward pass
    x = q.clone().requires_grad_()
    y, _ = pkg().apply_rotary(x, None, pos, rot)
    with fw.dual_level():
        (g,) = torch.autograd.grad(y, x, fw.make_dual(torch.zeros_like(q), u))
        assert torch.equal(fw.unpack_dual(g).tangent, turn(u, None, pos, rot, inverse=True)[0])


def test_gradients_that_nobody_asks_for(monkeypatch):
    R = submodule("rotary")
    rot = pkg().Rotary(table(32).to(DEV))
    pos = torch.arange(9, device=DEV)
    q, k, dq, dk = (torch.randn(1, h, 9, 64, device=DEV).half() for h in (4, 2, 4, 2))
    refs = R.rotate(dq, dk, pos, rot, inverse=True)
    turned = []
    plain = R.rotate

    def counted(a, b, *rest, **kw):
        turned.append([x.shape[1] for x in (a, b) if x is not None])
        return plain(a, b, *rest, **kw)

    monkeypatch.setattr(R, "rotate", counted)
    for a, b, heads in ((1, 0, [4]), (0, 1, [2]), (1, 1, [4, 2])):
        x, z = q.clone().requires_grad_(bool(a)), k.clone().requires_grad_(bool(b))
        ys = R.apply_rotary(x, z, pos, rot)
        turned.clear()
        torch.autograd.backward(ys, (dq, dk))
        assert turned == [heads]
        assert (x.grad is None) == (not a) and (z.grad is None) == (not b)
        assert all(y.grad is None or torch.equal(y.grad, ref) for y, ref in zip((x, z), refs))


def test_gradient_in_a_graph():
    rot = pkg().Rotary(table(32).to(DEV))
    pos = torch.arange(40, device=DEV)
    q, dq = (torch.randn(1, 4, 40, 64, device=DEV).half() for _ in range(2))
    x = q.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = pkg().apply_rotary(x, None, pos, rot)
        (g,) = torch.autograd.grad(y, x, dq)
    pos.add_(1000)
    dq.mul_(2)
    graph.replay()
    turn = submodule("rotary").rotate
    assert torch.equal(y.detach(), turn(q, None, pos, rot)[0]) and torch.equal(g, turn(dq, None, pos, rot, inverse=True)[0])
