"""Rotary positions against exact angles and float64 products."""
import math
from fractions import Fraction

import pytest
import torch

from maxsim_amd import Rotary

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ROUND = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}
TURN = 2 * Fraction("3.14159265358979323846264338327950288419716939937511")


def _angles(frequencies, axes, positions):
    """[rows, pairs] in float64, whole turns taken off exactly."""
    positions = positions.cpu().view(-1, positions.shape[-1]).tolist()
    turns = [Fraction(f) / TURN for f in frequencies]
    return torch.tensor([[2 * math.pi * float(positions[a][r] * t % 1) for a, t in zip(axes, turns)]
                         for r in range(len(positions[0]))], dtype=torch.float64).view(len(positions[0]), len(turns))


def _check(got, x, angles, adjacent):
    """Sine and cosine come within 4 x 2^-24 (their angle within a quarter turn's half has
    three roundings of it, their polynomials two and a remainder of 2^-28); a product and the sum
    round too; the result once."""
    x, pairs = x.cpu().double(), angles.shape[1]
    c, s = angles.cos()[:, None], angles.sin()[:, None]
    at = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if adjacent else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b = x[..., at[0]], x[..., at[1]]
    got = got.cpu()
    for part, exp in zip(at, (a * c - b * s, a * s + b * c)):
        tol = ROUND[got.dtype] * exp.abs() + 6 * 2.0**-24 * (a.abs() + b.abs()) + 1e-37
        if got.dtype == F16:
            tol = tol + 2.0**-25
        diff = (got[..., part].double() - exp).abs()
        assert bool((diff <= tol).all()), float((diff / tol).max())
    assert torch.equal(got[..., 2 * pairs:].double(), x[..., 2 * pairs:])


def _inputs(rows, heads, dim, kind, seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return (2 * torch.randn((rows, heads, dim), generator=g)).to(kind).cuda()


def _positions(axes, rows, most, seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randint(-3, most, (axes, rows), generator=g).to(torch.int32).cuda()


def _default(part):
    return [10000.0 ** (-2.0 * i / part) for i in range(part // 2)]


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("rows,heads,kv_heads,dim,part,num_axes", [
    (1, 1, 1, 64, 64, 1), (3, 32, 8, 128, 128, 1), (7, 6, 2, 96, 96, 3), (17, 5, 1, 256, 128, 2), (2, 3, 3, 80, 32, 1),
    (5, 2, 1, 10, 6, 3), (4, 7, 7, 2, 2, 1), (9, 40, 8, 100, 50, 2), (6, 4, 4, 256, 256, 3), (3, 2, 1, 255, 6, 1),
    (700, 9, 3, 64, 48, 3)])
def test_rows(gpu, kind, adjacent, rows, heads, kv_heads, dim, part, num_axes):
    axes = [(i * 5 + i // 3) % num_axes for i in range(part // 2)]
    axes[-1] = num_axes - 1
    rotary = Rotary(dim, rotary_dim=part, axes=axes, adjacent=adjacent)
    assert rotary.num_axes == num_axes
    q, k = _inputs(rows, heads, dim, kind, 1), _inputs(rows, kv_heads, dim, kind, 2)
    positions = _positions(num_axes, rows, 200000, 3)
    got = rotary(q, k, positions)
    angles = _angles(_default(part), axes, positions)
    for g, x in zip(got, (q, k)):
        assert g.shape == x.shape and g.dtype == kind
        _check(g, x, angles, adjacent)
    alone = rotary(q, None, positions if num_axes > 1 else positions[0])
    assert alone[1] is None and torch.equal(alone[0], got[0])
    # In place, and into rows of wider buffers.
    wide = torch.full((rows, heads + 2, dim + 8), 7.0, dtype=kind, device="cuda")
    q_out, k_out = wide[:, 1:heads + 1, 3:dim + 3], k.clone()
    rotary(q, k_out, positions, out=(q_out, k_out))
    assert torch.equal(q_out, got[0]) and torch.equal(k_out, got[1])
    wide[:, 1:heads + 1, 3:dim + 3] = 7.0
    assert bool((wide == 7.0).all())


@pytest.mark.parametrize("shift", [0, 1, 8])
def test_views_of_a_fused_projection(gpu, shift):
    rows, heads, kv_heads, dim = 33, 8, 2, 64
    fused = _inputs(rows, 1, (heads + 2 * kv_heads) * dim + shift, BF16, 4)[:, 0, shift:]
    q = fused[:, :heads * dim].view(rows, heads, dim)
    k = fused[:, heads * dim:(heads + kv_heads) * dim].view(rows, kv_heads, dim)
    positions = _positions(1, rows, 5000, 5)
    rotary = Rotary(dim)
    got = rotary(q, k, positions[0])
    assert all(torch.equal(a, b) for a, b in zip(got, rotary(q.contiguous(), k.contiguous(), positions)))
    rotary(q, k, positions[0], out=(q, k))  # neighbours in one buffer
    assert torch.equal(q, got[0]) and torch.equal(k, got[1])


def test_far_positions_and_odd_frequencies(gpu):
    frequencies = [1.0, 6.283185307179586, -0.3, 1e-9, 0.0, 1234.5678, 1e-30, 2.0**-7]
    rotary = Rotary(16, frequencies=frequencies)
    ends = [0, 1, -1, 2**31 - 1, -2**31, 2**30 + 12345, 1000003, -77777777, 131071]
    positions = torch.tensor([ends], dtype=torch.int32).cuda()
    for kind in (F32, F16, BF16):
        x = _inputs(len(ends), 3, 16, kind, 6)
        # A product of 2^31 and a frequency rounded to 2^-64 turns is within 2^-34.
        _check(rotary(x, None, positions)[0], x, _angles(frequencies, [0] * 8, positions), False)
    quarters = Rotary(2, frequencies=[math.pi / 2])
    x = torch.tensor([1.0, 0.0], device="cuda").expand(8, 1, 2).contiguous()
    got = quarters(x, None, torch.arange(8, dtype=torch.int32, device="cuda"))[0][:, 0].cpu()
    exp = torch.tensor([[1.0, 0], [0, 1], [-1, 0], [0, -1]] * 2)
    assert bool(((got - exp).abs() <= 2.0**-23).all())


def test_values_at_the_ends(gpu):
    rotary = Rotary(8)
    positions = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    x = torch.zeros((3, 2, 8), device="cuda")
    x[1, 0, 2] = math.nan
    x[2, 1, 5] = math.inf
    got = rotary(x, None, positions)[0].cpu()
    assert bool(torch.isnan(got[1, 0, [2, 6]]).all()) and not bool(torch.isfinite(got[2, 1, [1, 5]]).any())
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[1, 0, [2, 6]] = rest[2, 1, [1, 5]] = False
    assert bool((got[rest] == 0).all())
    for kind in (F32, F16, BF16):
        small = (_inputs(3, 2, 8, F32, 7) * {F32: 1e-36, F16: 1e-6, BF16: 1e-36}[kind]).to(kind)
        _check(rotary(small, None, positions)[0], small, _angles(_default(8), [0] * 4, positions), False)
    assert rotary(x[:0], x[:0], positions[:0])[0].shape == (0, 2, 8)
    assert rotary(x, x[:, :0], positions)[1].shape == (3, 0, 8)


def test_rows_past_32_bits(gpu):
    """Rows that begin past 2^31 elements."""
    wide = torch.zeros(2**31 + 2**20, dtype=F16, device="cuda")
    q = wide[:2**31 + 1024].as_strided((3, 4, 64), (2**30, 64, 1))
    q.copy_(_inputs(3, 4, 64, F16, 8))
    positions = _positions(1, 3, 900, 3)
    rotary = Rotary(64)
    want = rotary(q.contiguous(), None, positions)[0]
    assert torch.equal(rotary(q, None, positions)[0], want)
    rotary(q, None, positions, out=(q, None))
    assert torch.equal(q, want)


def test_graph_replays(gpu):
    rotary = Rotary(64, axes=[0] * 16 + [1] * 16)
    q, k, positions = _inputs(5, 4, 64, BF16, 1), _inputs(5, 2, 64, BF16, 2), _positions(2, 5, 900, 3)
    rotary(q, k, positions)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary(q, k, positions)
    for i in range(4):
        q.copy_(_inputs(5, 4, 64, BF16, 10 + i))
        positions.copy_(_positions(2, 5, 900, 20 + i))
        eager = rotary(q, k, positions)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


def test_refusals(gpu):
    for args, kw in (((64,), {"rotary_dim": 63}), ((64,), {"rotary_dim": 66}), ((64,), {"rotary_dim": 0}), ((1,), {}),
                     ((64,), {"base": 0.0}), ((64,), {"base": math.inf}), ((64,), {"axes": [0] * 31}),
                     ((64,), {"frequencies": [1.0]}), ((4,), {"frequencies": [1.0, math.nan]}),
                     ((4,), {"axes": [0, -1]}), ((4,), {"axes": [0, 2]}), ((64,), {"device": "cpu"})):
        with pytest.raises(ValueError):
            Rotary(*args, **kw)
    with pytest.raises(NotImplementedError):
        Rotary(258)
    rotary, two = Rotary(8), Rotary(8, axes=[0, 0, 1, 1])
    q, p = torch.zeros((3, 2, 8), device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    wide = torch.zeros((3, 4, 8), device="cuda")
    for r, args, kw in ((rotary, (q[..., :6], None, p), {}), (rotary, (q, q.half(), p), {}),
                        (rotary, (q, q[:2], p), {}), (rotary, (q, None, p.long()), {}), (rotary, (q, None, p[:2]), {}), (two, (q, None, p), {}),
                        (two, (q, None, p.expand(3, 3)), {}), (rotary, (q, None, p.cpu()), {}),
                        (rotary, (q.double(), None, p), {}), (rotary, (q.cpu(), None, p), {}),
                        (rotary, (q.transpose(1, 2).contiguous().transpose(1, 2), None, p), {}),
                        (rotary, (q, q, p), {"out": (q, q)}), (rotary, (q, q, p), {"out": (q, None)}),
                        (rotary, (q, None, p), {"out": (q, q)}), (rotary, (q, None, p), {"out": (q.half(), None)}),
                        (rotary, (wide[:, :2], None, p), {"out": (wide[:, 1:3], None)}),
                        (rotary, (q, None, p), {"out": (q[:1].expand(3, 2, 8), None)}),
                        (rotary, (wide[:, :2], wide[:, 2:], p), {"out": (wide[:, 2:], wide[:, :2])})):
        with pytest.raises(ValueError):
            r(*args, **kw)
