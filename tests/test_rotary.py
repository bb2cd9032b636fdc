"""Rotary positions against their definition in 64 bits: layouts, parts of a head,
odd sizes, strides, in place, far positions, scaled frequencies, gradients and refusals.

Tolerance of a turned value y = x1 c + x2 s: half a unit of the output type on y, and
2^-20 (|x1| + |x2|) m for the fp32 products, sums and tables (four roundings of 2^-24
each, with room), m the factor on cos and sin; fp16 adds half its smallest step."""
import math

import pytest
import torch

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _pairs(rot, layout):
    i = torch.arange(rot // 2)
    return (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)


def _turned(x, angle, mul, layout, rot, back=False):
    """x (rows, heads, d) float64, angle (rows, rot/2) float64 on the CPU."""
    one, two = _pairs(rot, layout)
    c, s = angle.cos()[:, None] * mul, angle.sin()[:, None] * mul * (-1 if back else 1)
    y = x.clone()
    y[..., one] = x[..., one] * c + x[..., two] * s
    y[..., two] = x[..., two] * c - x[..., one] * s
    return y


def _check(y, x, ref, dtype, mul, layout, rot):
    one, two = _pairs(rot, layout)
    room = torch.zeros_like(x)
    room[..., one] = room[..., two] = (x[..., one].abs() + x[..., two].abs()) * mul * 2.0 ** -20
    tol = ref.abs() * UNIT[dtype] * 1.001 + room + (2.0 ** -25 if dtype == torch.float16 else 0)
    err = (y.double().cpu() - ref).abs()
    assert (err <= tol).all(), (err - tol).max().item()
    assert torch.equal(y.cpu()[..., rot:].double(), x[..., rot:])  # the rest passes through


def _angle(pos, rot, base=10000.0):
    w = torch.tensor([base ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64)
    return pos.double()[:, None].cpu() * w


def test_tables_match_the_definition_cpu():
    from rs_nanogpt_b200.ops import rotary
    cos, sin = rotary.tables(32, 50000, device="cpu")
    a = _angle(torch.arange(50000), 32)
    assert cos.shape == (50000, 16) and cos.dtype == torch.float32
    assert (cos.double() - a.cos()).abs().max() < 2.0 ** -23
    assert (sin.double() - a.sin()).abs().max() < 2.0 ** -23


def test_scaled_tables_cpu():
    from rs_nanogpt_b200.ops import rotary
    rot, f, n = 64, 4.0, 300
    plain = _angle(torch.arange(n), rot)
    cos, _ = rotary.tables(rot, n, scaling=rotary.Scaling("linear", f), device="cpu")
    assert (cos.double() - (plain / f).cos()).abs().max() < 1e-6
    cos, _ = rotary.tables(rot, n, scaling=rotary.Scaling("ntk", f), device="cpu")
    # The fastest pair keeps its frequency, the slowest turns f times slower.
    assert (cos[:, 0].double() - plain[:, 0].cos()).abs().max() < 1e-6
    assert (cos[:, -1].double() - (plain[:, -1] / f).cos()).abs().max() < 1e-6
    cos, sin = rotary.tables(rot, n, scaling=rotary.Scaling("parts", f, original_len=128), device="cpu")
    mul = 0.1 * math.log(f) + 1
    assert (cos ** 2 + sin ** 2 - mul ** 2).abs().max() < 1e-5
    for i in range(rot // 2):
        w = 10000.0 ** (-2 * i / rot)
        keep = min(1.0, max(0.0, (128 * w / (2 * math.pi) - 1) / 31))
        ref = torch.arange(n).double() * w * (keep + (1 - keep) / f)
        assert (cos[:, i].double() - ref.cos() * mul).abs().max() < 1e-6


@pytest.mark.parametrize("make", [
    lambda r: r.tables(7, 4, device="cpu"), lambda r: r.tables(0, 4, device="cpu"), lambda r: r.tables(8, 0, device="cpu"),
    lambda r: r.tables(2, 4, scaling=r.Scaling("ntk", 2.0), device="cpu"), lambda r: r.Scaling("other", 2.0),
    lambda r: r.Scaling("linear", 0.5), lambda r: r.Scaling("parts", 2.0, original_len=0),
    lambda r: r.rotate(torch.zeros(1, 1, 8), None, torch.zeros(1), None, None, layout="diagonal")])
def test_refusals_cpu(make):
    from rs_nanogpt_b200.ops import rotary
    with pytest.raises(ValueError):
        make(rotary)


gpu = [pytest.mark.gpu, pytest.mark.usefixtures("kernel_ok")]


def _gpu(fn):
    for m in gpu:
        fn = m(fn)
    return fn


@_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows,hq,hk,d,rot", [(1, 1, 1, 128, 128), (257, 10, 10, 128, 128), (33, 7, 1, 64, 32),
                                              (19, 3, 2, 80, 20), (5, 2, 2, 66, 66), (70, 4, 0, 128, 2),
                                              (3, 9, 3, 6, 4), (1000, 1, 1, 256, 64)])
def test_rotate_and_gradient(rows, hq, hk, d, rot, layout, dtype):
    from rs_nanogpt_b200.ops import rotary
    torch.manual_seed(rows)
    cos, sin = rotary.tables(rot, 4096)
    pos = torch.randint(0, 4096, (rows,), device="cuda", dtype=torch.int32)
    q = torch.randn(rows, hq, d, device="cuda").to(dtype)
    k = torch.randn(rows, hk, d, device="cuda").to(dtype) if hk else None
    for fn, back in ((rotary.rotate, False), (rotary.rotate_bwd, True)):
        outs = fn(q, k, pos, cos, sin, layout)
        for x, y in zip((q, k), outs):
            if x is None:
                assert y is None
                continue
            x = x.double().cpu()
            _check(y, x, _turned(x, _angle(pos, rot), 1.0, layout, rot, back), dtype, 1.0, layout, rot)


@_gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strided_views_and_in_place(layout):
    from rs_nanogpt_b200.ops import rotary
    torch.manual_seed(1)
    n, h, d, rot = 37, 3, 64, 48
    cos, sin = rotary.tables(rot, 64)
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    for shift in (0, 1, 4):  # starts at any alignment
        fused = torch.randn(n, 3 * h * d + 7 + shift, device="cuda").bfloat16()
        q, k = (fused[:, shift + i * h * d:shift + (i + 1) * h * d].view(n, h, d) for i in range(2))
        before = fused.clone()
        want = [_turned(x.double().cpu(), _angle(pos, rot), 1.0, layout, rot) for x in (q, k)]
        xs = [x.double().cpu() for x in (q, k)]
        rotary.rotate(q, k, pos, cos, sin, layout, q_out=q, k_out=k)
        for x, ref, y in zip(xs, want, (q, k)):
            _check(y, x, ref, torch.bfloat16, 1.0, layout, rot)
        rest = torch.ones(fused.shape[1], dtype=torch.bool, device="cuda")
        rest[shift:shift + 2 * h * d] = False
        assert torch.equal(fused[:, rest], before[:, rest])
    heads_first = torch.randn(h, n, d, device="cuda").transpose(0, 1)  # any order of rows and heads
    y, _ = rotary.rotate(heads_first, None, pos, cos, sin, layout)
    x = heads_first.double().cpu()
    _check(y, x, _turned(x, _angle(pos, rot), 1.0, layout, rot), torch.float32, 1.0, layout, rot)


@_gpu
def test_gradient_against_differences():
    """<dy, rotate(x + e) - rotate(x - e)> / 2 = <rotate_bwd(dy), e>: the turn is linear, so the
    difference is exact up to fp32 rounding, 2^-20 of the sums of magnitudes."""
    from rs_nanogpt_b200.ops import rotary
    torch.manual_seed(2)
    scaling = rotary.Scaling("parts", 8.0, original_len=64)
    cos, sin = rotary.tables(24, 512, scaling=scaling)
    pos = torch.randint(0, 512, (65,), device="cuda", dtype=torch.int32)
    for layout in rotary.LAYOUTS:
        x, dy = torch.randn(65, 3, 32, device="cuda"), torch.randn(65, 3, 32, device="cuda")
        dx, _ = rotary.rotate_bwd(dy, None, pos, cos, sin, layout)
        for _ in range(4):
            e = torch.randn_like(x)
            hi, _ = rotary.rotate(x + e, None, pos, cos, sin, layout)
            lo, _ = rotary.rotate(x - e, None, pos, cos, sin, layout)
            left = (dy.double() * (hi.double() - lo.double()) / 2).sum().item()
            right = (dx.double() * e.double()).sum().item()
            room = (dy.double().norm() * (x.double().norm() + e.double().norm())).item() * 2 * 2.0 ** -20
            assert abs(left - right) <= room


@_gpu
def test_inverse_far_positions_and_empty():
    from rs_nanogpt_b200.ops import rotary
    torch.manual_seed(3)
    cos, sin = rotary.tables(64, 1 << 18)
    pos = torch.tensor([0, 1, 131072, (1 << 18) - 1], device="cuda", dtype=torch.int32)
    q = torch.randn(4, 2, 64, device="cuda")
    y, _ = rotary.rotate(q, None, pos, cos, sin)
    x = q.double().cpu()
    _check(y, x, _turned(x, _angle(pos, 64), 1.0, "half", 64), torch.float32, 1.0, "half", 64)
    z, _ = rotary.rotate_bwd(y, None, pos, cos, sin)
    assert (z - q).abs().max() < 1e-5
    empty, _ = rotary.rotate(q[:0], None, pos[:0], cos, sin)
    assert empty.shape == (0, 2, 64)


@pytest.mark.gpu
def test_position_outside_the_tables_is_reported():
    from rs_nanogpt_b200.ops import rotary
    from rs_nanogpt_b200.ops._ext import kernel_status
    kernel_status(True)
    cos, sin = rotary.tables(32, 16)
    q = torch.randn(3, 2, 32, device="cuda")
    out = torch.zeros_like(q)
    rotary.rotate(q, None, torch.tensor([3, 16, -1], device="cuda", dtype=torch.int32), cos, sin, q_out=out)
    assert kernel_status(True) == 5
    assert out[0].abs().sum() > 0 and out[1:].abs().sum() == 0


@pytest.mark.gpu
def test_refusals():
    from rs_nanogpt_b200.ops import rotary
    cos, sin = rotary.tables(32, 16)
    q, pos = torch.zeros(4, 2, 64, device="cuda"), torch.zeros(4, device="cuda", dtype=torch.int32)
    buf = torch.zeros(5 * 2 * 64, device="cuda")
    for args in [
        (q.double(), None, pos, cos, sin),                       # dtype
        (q[..., :31], None, pos, cos, sin),                      # odd heads, more turned than there is
        (q[..., :16], None, pos, cos, sin),
        (q, q.bfloat16(), pos, cos, sin),                        # k unlike q
        (q, None, pos.long(), cos, sin),
        (q, None, pos[:3], cos, sin),
        (q, None, pos.cpu(), cos, sin),
        (q, None, pos, cos.half(), sin.half()),
        (q, None, pos, cos, sin[:8]),
        (q.transpose(1, 2), None, pos, cos, sin),                # last dimension not contiguous
        (buf[:512].view(4, 2, 64), None, pos, cos, sin, "half", buf[64:576].view(4, 2, 64)),  # shifted over itself
    ]:
        with pytest.raises(RuntimeError):
            rotary.rotate(*args)
