"""Products with a matrix in 4 bits and group scales against float64."""
import math

import pytest
import torch

from maxsim_amd import Int4Linear, pack_int4_groups

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _matrix(n, k, group, seed=0):
    g = torch.Generator()
    g.manual_seed(seed)
    c = torch.randint(-7, 8, (n, k), generator=g)
    s = (0.01 * torch.exp(0.5 * torch.randn((n, k // group), generator=g))).to(BF16)
    nib = (c & 15).to(torch.uint8)
    return nib[:, 0::2] | (nib[:, 1::2] << 4), s, c.double() * s.double().repeat_interleave(group, 1)


def _rows(m, k, kind, seed=1):
    g = torch.Generator()
    g.manual_seed(seed)
    x = torch.randn((m, k), generator=g)
    x[:, :: max(1, k // 7)] *= 20.0
    return x.to(kind)


def _check(got, x, w, s, group, bias=None):
    """Each group's sum is group products of single precision (bfloat16: with an
    offset of 24 on codes of up to 7), then one rounding per group."""
    x, kind = x.double(), got.dtype
    exp = x @ w.T + (0 if bias is None else bias.double())
    groups = w.shape[1] // group
    scale = s.double().repeat_interleave(group, 1)
    most = (31.0 if kind == BF16 else 7.0) * (x.abs() @ scale.T)
    tol = 2.0**-24 * ((group / 2 + 4) * most + (groups + 20) * (x.abs() @ w.abs().T + exp.abs()))
    tol += {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}[kind] * exp.abs() + (2.0**-25 if kind == F16 else 1e-30)
    # A result that is no number of the type (an input may be infinite) is none here either.
    finite = exp.abs() <= torch.finfo(kind).max
    assert bool(torch.isfinite(got.cpu())[finite].all()) and not bool(torch.isfinite(got.cpu())[~finite].any())
    diff = (got.cpu().double() - exp).abs()[finite]
    assert bool((diff <= tol[finite]).all()), float((diff / tol[finite]).max())


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 1, 128), (1, 16, 256), (1, 100, 128), (2, 129, 640), (4, 48, 128), (5, 17, 384),
                                   (16, 33, 256), (17, 40, 128), (33, 70, 512), (64, 16, 128), (100, 50, 256)])
def test_products(gpu, kind, group, m, n, k):
    codes, scales, w = _matrix(n, k, group)
    linear = Int4Linear(codes.cuda(), scales.cuda())
    x = _rows(m, k, kind)
    got = linear(x.cuda())
    assert got.shape == (m, n) and got.dtype == kind
    _check(got, x, w, scales, group)
    assert torch.equal(linear(x.cuda()), got)


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("group,k", [(32, 32), (32, 96), (32, 160), (64, 64), (64, 320), (32, 4128)])
@pytest.mark.parametrize("m", [1, 3, 19])
def test_columns_that_end_inside_a_tile(gpu, kind, group, k, m):
    codes, scales, w = _matrix(21, k, group, seed=k)
    x = _rows(m, k, kind)
    _check(Int4Linear(codes.cuda(), scales.cuda())(x.cuda()), x, w, scales, group)


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (3, 5000, 1024), (16, 2048, 8192), (1, 33, 16384)])
def test_larger_products(gpu, kind, m, n, k):
    codes, scales, w = _matrix(n, k, 64)
    x = _rows(m, k, kind)
    _check(Int4Linear(codes.cuda(), scales.cuda())(x.cuda()), x, w, scales, 64)


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_shapes_strides_bias_and_out(gpu, kind, shift):
    codes, scales, w = _matrix(45, 192, 64)
    bias = torch.linspace(-2, 2, 45)
    linear = Int4Linear(codes.cuda(), scales.cuda(), bias=bias.cuda())
    wide = _rows(6, 192 + 10 + shift, kind)
    x = wide.cuda()[:, shift:shift + 192]
    out = torch.empty((6, 45), dtype=kind, device="cuda")
    assert linear(x, out=out) is out
    _check(out, wide[:, shift:shift + 192], w, scales, 64, bias)
    assert torch.equal(linear(x.reshape(2, 3, 192)), out.view(2, 3, 45))
    assert torch.equal(linear(x[4]), linear(x[4:5])[0])
    assert torch.equal(linear(x.t().contiguous().t()), out)
    assert linear(x[:0]).shape == (0, 45)


def test_values_at_the_ends_of_their_range(gpu):
    codes, scales, w = _matrix(20, 128, 32)
    linear = Int4Linear(codes.cuda(), scales.cuda())
    for kind, size in ((F32, 1e30), (F32, 1e-30), (BF16, 1e30), (BF16, 1e-30), (F16, 3e3), (F16, 1e-4)):
        x = (_rows(3, 128, F32) * size).to(kind)
        _check(linear(x.cuda()), x, w, scales, 32)
    for kind in (F32, F16, BF16):
        x = _rows(3, 128, kind)
        x[1, 9] = math.nan
        got = linear(x.cuda()).cpu()
        assert bool(torch.isnan(got[1]).all()) and bool(torch.isfinite(got[[0, 2]]).all())
        x[1, 9] = math.inf
        got = linear(x.cuda()).cpu()
        assert not bool(torch.isfinite(got[1]).any()) and bool(torch.isfinite(got[[0, 2]]).all())


def test_quantised_matrix(gpu):
    w = torch.randn((70, 256), device="cuda") * torch.exp(torch.randn((70, 1), device="cuda"))
    w[3, 64:128] = 0.0
    for group in (32, 64, 128):
        codes, scales = pack_int4_groups(w, group)
        assert codes.shape == (70, 128) and scales.shape == (70, 256 // group)
        c = torch.stack((codes & 15, codes >> 4), -1).flatten(1).to(torch.int16)
        c = torch.where(c > 7, c - 16, c)
        assert int(c.abs().max()) <= 7
        back = c.double() * scales.double().repeat_interleave(group, 1)
        # Half a step, and what the rounding of a scale adds at the ends.
        assert bool(((back - w.double()).abs() <= scales.double().repeat_interleave(group, 1) * 0.53).all())
        x = torch.randn((2, 256), device="cuda")
        _check(Int4Linear.from_float(w, group)(x), x.cpu(), back.cpu(), scales.cpu(), group)


def test_graph_replays(gpu):
    codes, scales, w = _matrix(300, 1024, 128)
    linear = Int4Linear(codes.cuda(), scales.cuda())
    x = _rows(2, 1024, BF16).cuda()
    linear(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = linear(x)
    for i in range(4):
        x.copy_(_rows(2, 1024, BF16, seed=i))
        eager = linear(x)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_refusals(gpu):
    codes, scales, _ = _matrix(20, 128, 32)
    codes, scales = codes.cuda(), scales.cuda()
    for bad in ((codes.cpu(), scales), (codes.int(), scales), (codes, scales.float()), (codes, scales[:, :3]),
                (codes, scales[:, :0]), (codes[:5], scales), (codes[0], scales), (codes, scales.cpu()),
                (codes, scales, torch.zeros(19, device="cuda")), (codes, scales, torch.zeros(20))):
        with pytest.raises(ValueError):
            Int4Linear(*bad)
    linear = Int4Linear(codes, scales)
    x = torch.zeros((2, 128), device="cuda")
    for bad, kw in ((x[:, :64], {}), (x.cpu(), {}), (x.double(), {}), (x, {"out": x}), (x, {"out": x[:, :20].half()})):
        with pytest.raises(ValueError):
            linear(bad, **kw)
    for args in ((torch.zeros((4, 100), device="cuda"), 32), (torch.zeros((4, 64), device="cuda"), 16),
                 (torch.zeros(64, device="cuda"), 32), (torch.full((4, 64), math.nan, device="cuda"), 32)):
        with pytest.raises(ValueError):
            pack_int4_groups(*args)


# ------------------------------------------------- product by product
#
# No product may weigh on another column's: bounds by the products themselves.


def _between(got, exp, tol):
    """Every value is the rounding of one within tol of the expected (float64)."""
    low, high = (exp - tol).to(got.dtype), (exp + tol).to(got.dtype)
    off = ~((low <= got) & (got <= high))
    assert not bool(off.any()), float(((got.double() - exp).abs() / tol)[off].max())


def _check_by_products(got, x, w, group, bias=None):
    """A group's sum is group exact products added in single precision; groups, waves
    and the bias are added to it.  ``w`` is [n, k]; all in float64 on the GPU."""
    x, w = x.cuda().double(), w.cuda().t().contiguous()
    exp = x @ w + (0 if bias is None else bias.cuda().double())
    mass = x.abs() @ w.abs() + (0 if bias is None else bias.cuda().double().abs())
    _between(got, exp, 2.0**-24 * (group + w.shape[0] // group + 20) * mass + 1e-37)


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("m", [1, 7, 24])
def test_large_inputs_under_zero_codes(gpu, kind, m):
    """A column far larger than the others weighs nothing where its code is zero."""
    codes, scales, w = _matrix(300, 512, 128)
    codes[::2, 50] = 0  # columns 100 and 101
    w[::2, 100:102] = 0.0
    x = _rows(m, 512, kind)
    x[:, 100] = 6e4 if kind == F16 else 1e7
    x[:, 101] = -3e4 if kind == F16 else 1e8
    _check_by_products(Int4Linear(codes.cuda(), scales.cuda())(x.cuda()), x, w, 128)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 20])
def test_largest_inputs(gpu, kind, group, m):
    """Inputs up to the largest of their type, results well inside it."""
    codes, scales, w = _matrix(40, 384, group)
    scales, w = (scales.float() / 4096).to(BF16), w / 4096  # exactly
    g = torch.Generator()
    g.manual_seed(2)
    x = ((2 * torch.rand((m, 384), generator=g) - 1) * 3.38e38).to(kind)
    x[0] = torch.finfo(kind).max
    _check_by_products(Int4Linear(codes.cuda(), scales.cuda())(x.cuda()), x, w, group)


def test_outputs_that_overlap_inputs(gpu):
    """An output over x is refused; one between the rows of x is not."""
    codes, scales, w = _matrix(128, 128, 32)
    linear = Int4Linear(codes.cuda(), scales.cuda())
    wide = _rows(3, 500, F32)
    flat = wide.cuda().view(-1)
    x = flat.view(3, 500)[:, :128]
    for out in (flat[:384], flat[127:511], flat[500:884], flat[1000 + 100:1000 + 484], flat[400:784]):
        with pytest.raises(ValueError, match="overlap"):
            linear(x, out=out.view(3, 128))
    with pytest.raises(ValueError, match="overlap"):
        linear(x[0], out=x[0])
    square = x.contiguous()
    with pytest.raises(ValueError, match="overlap"):
        linear(square, out=square)
    _check_by_products(linear(x, out=torch.empty_like(square)), x.cpu(), w, 32)
    _check_by_products(linear(x[:2], out=flat[128:128 + 256].view(2, 128)), wide[:2, :128], w, 32)  # in row 0's gap
    assert torch.equal(x.cpu(), wide[:, :128])


# ------------------------------------------------------- shapes of tiles


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("group,k", [(32, 416), (64, 448), (128, 384)])
def test_row_tiles_of_a_workgroup(gpu, kind, group, k):
    """Widths at which workgroups have one, two, four and seven row tiles (256 CUs), the
    last of them partly or wholly past the end; rows of one and two column tiles."""
    g = torch.Generator(device="cuda")
    g.manual_seed(k)
    for n in (4081, 8163, 16345, 28629):
        w = torch.randn((n, k), generator=g, device="cuda")
        codes, scales = pack_int4_groups(w, group)
        bias = torch.randn(n, generator=g, device="cuda")
        linear = Int4Linear(codes, scales, bias)
        c = torch.stack((codes & 15, codes >> 4), -1).flatten(1).to(torch.int8)
        w = torch.where(c > 7, c - 16, c).double() * scales.double().repeat_interleave(group, 1)
        for m in (1, 5, 16, 19, 32, 75):
            x = torch.randn((m, k), generator=g, device="cuda").to(kind)
            out = torch.full((m + 1, n), 7.0, dtype=kind, device="cuda")
            linear(x, out=out[:m])
            _check_by_products(out[:m], x, w, group, bias)
            assert bool((out[m] == 7).all())


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("m,n", [(32, 28672), (17, 28629), (1, 28672), (16, 16345)])
def test_row_tiles_and_many_waves(gpu, kind, m, n):
    """As many row tiles as the registers hold and eight or sixteen waves, which join in
    up to 112 KiB of LDS."""
    g = torch.Generator(device="cuda")
    g.manual_seed(n + m)
    codes = torch.randint(0, 256, (n, 512), generator=g, device="cuda", dtype=torch.uint8)  # -8 too
    scales = (0.01 * (1 + torch.rand((n, 8), generator=g, device="cuda"))).to(BF16)
    linear = Int4Linear(codes, scales)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(1).to(torch.int8)
    w = torch.where(c > 7, c - 16, c).double() * scales.double().repeat_interleave(128, 1)
    x = torch.randn((m, 1024), generator=g, device="cuda").to(kind)
    _check_by_products(linear(x), x, w, 128)
