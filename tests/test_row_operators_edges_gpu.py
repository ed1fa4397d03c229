"""The row operators (group norm, linear layer, Newton-Schulz) where values, sizes or calls are at the edge of what they take, against
64 bits.  u = 2^-24; HALF_STEP is half a step of the stored type."""
import math

import pytest
import torch

from panopticsegforlargescalepointcloud_amd import modules, ops
from test_groupnorm_gpu import HALF_STEP, TINY, act64, dact64

pytestmark = pytest.mark.gpu

u = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def far_values(dtype):
    return torch.tensor([-5.5, -6.0, -6.5, -7.0, -8.0, -9.5, -11.0, -12.5, -15.0, -20.0, -1e4, torch.finfo(dtype).min, 6.5, 20.0, 1e4]).to(dtype)


def check_gelu(z, y, dz, dtype):
    """Phi(z) behind -6 is kept to 1 % (0.7 % by its fit, and the hardware's exponential), z^2 / 2 is rounded once (z^2 u of the density),
    and what is below 2^-126 may be 0; in front of it 16 u as everywhere"""
    z, y, dz = z.double().cpu(), y.double().cpu(), dz.double().cpu()
    U, tiny = HALF_STEP[dtype], TINY[dtype]
    want, slope = act64(z, "gelu"), dact64(z, "gelu")
    density = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    near_zero = 2.0 ** -126 * (z > -40) * (1 + z.abs())  # farther out nothing but 0 will do
    rel = torch.where(z < -6, 0.01, 0.0) * want.abs() + torch.where(z < -6, 0.0, 16 * u) * z.abs()
    assert bool(((y - want).abs() <= rel + U * (want.abs() + rel) + tiny * (z > -40) + near_zero).all()), (y, want)
    phi = 0.5 * torch.erfc(-z / math.sqrt(2.0))
    rel = torch.where(z < -6, 0.01, 0.0) * phi + torch.where(z < -6, 0.0, 16 * u) + (8 + 2 * z * z) * u * (z.abs() * density)
    rel = torch.where(z.abs() < 40, rel, 16 * u * (z > 0))
    assert bool(((dz - slope).abs() <= rel + U * (slope.abs() + rel) + tiny * (z > -40) + near_zero).all()), (dz, slope)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("copies", [1, 40])  # few rows, and enough for the kernel that streams them
def test_gelu_goes_to_zero_in_the_far_tail_linear(dtype, copies):
    z = far_values(dtype).repeat(copies).cuda().view(-1, 1)
    one = torch.ones((1, 1), dtype=dtype, device="cuda")
    y = ops.linear_act_fwd(z, one, None, 4)
    dx = ops.linear_act_bwd(z, torch.ones_like(z), one, None, 4)[0]
    check_gelu(z, y, dx, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 3000])
def test_gelu_goes_to_zero_in_the_far_tail_group_norm(dtype, rows):
    """weight 0: z is the bias, whatever the rows are; the bias gradient of one gradient of 1 is act'(z)"""
    z = far_values(torch.float32)
    c = z.numel()
    x = torch.randn((rows, c), device="cuda").to(dtype)
    off = torch.tensor([0, rows], device="cuda")
    w, b = torch.zeros(c, device="cuda"), z.cuda()
    y, mean, rstd = ops.group_norm_fwd(x, off, 1, w, b, 1e-5, 4)
    dy = torch.zeros_like(x)
    dy[rows // 2] = 1
    db = ops.group_norm_bwd(x, dy, off, 1, w, b, mean, rstd, 4)[2]
    assert bool((y == y[:1]).all())
    keep = z.abs() <= torch.finfo(dtype).max
    check_gelu(z[keep], y[0].cpu()[keep].float(), db.cpu()[keep], dtype)
    far = torch.tensor([-math.inf, math.inf, 0.0], device="cuda").repeat(c // 3)
    y = ops.group_norm_fwd(x, off, 1, w, far, 1e-5, 4)[0].float()
    assert bool(torch.isnan(y[:, 0]).all()) and bool((y[:, 1] == math.inf).all()) and bool((y[:, 2] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["none", "relu", "silu"])
def test_rows_equal_to_their_mean_come_out_as_the_bias(dtype, kind):
    """one-row elements under instance norm, and constant channels: x is its mean, so z is the bias whatever the size of x"""
    act = ops.activation_id(kind)
    size = torch.tensor([0.3, 10.3, 1000.1, 30000.0], device="cuda")
    torch.manual_seed(9)
    for c, rows in ((8, 1), (7, 1), (64, 300), (300, 40), (12, 70_000)):
        sign = torch.where(torch.arange(c, device="cuda") % 3 == 0, -1.0, 1.0)
        x = (size.repeat(-(-c // 4))[:c] * sign).repeat(3 * rows, 1).to(dtype)
        off = torch.tensor([0, rows, rows, 3 * rows], device="cuda")
        w, b = 1 + torch.rand(c, device="cuda"), torch.randn(c, device="cuda")
        y, mean, rstd = ops.group_norm_fwd(x, off, c, w, b, 1e-5, act)
        assert bool((y == y[:1]).all())
        want = act64(b.double(), kind)
        # (a result below the type's smallest normal number is rounded to half of its smallest step: 3e-5 in fp16 is off by 2^-25, not by 2^-11 of itself)
        room = HALF_STEP[dtype] * want.abs() + (16 * u if kind == "silu" else 0) * b.double().abs() + TINY[dtype] / 2
        assert bool(((y[0].double() - want).abs() <= room).all())
        y, mean, rstd = ops.group_norm_fwd(x, off, c, w, None, 1e-5, act)
        assert int(y.count_nonzero()) == 0
        assert int(ops.group_norm_bwd(x, torch.ones_like(x), off, c, w, None, mean, rstd, 1)[2].count_nonzero()) == 0  # relu at 0: slope 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c,groups", [(32, 8), (7, 7), (300, 300)])
@pytest.mark.parametrize("lengths", [[20_000], [1, 2, 3, 500, 9494, 10_000]])
def test_forward_and_backward_agree_about_the_side_of_a_kink(dtype, c, groups, lengths):
    """with gradients of one the bias gradient of relu counts the values whose z is positive: those that are in the result"""
    n = sum(lengths)
    gen = torch.Generator(device="cuda").manual_seed(c + n)
    x = (200 + 3 * torch.randn((n, c), generator=gen, device="cuda")).to(dtype)
    off = torch.tensor([0] + lengths, device="cuda").cumsum(0)
    w = 1 + torch.rand(c, generator=gen, device="cuda")
    for b in (None, 1e-6 * torch.randn(c, generator=gen, device="cuda")):
        _, mean, rstd = ops.group_norm_fwd(x, off, groups, w, b, 1e-5, 1)
        db = ops.group_norm_bwd(x, torch.ones_like(x), off, groups, w, b, mean, rstd, 1)[2]
        positive = ops.group_norm_fwd(x.float(), off, groups, w, b, 1e-5, 1)[0] > 0  # (16-bit values are fp32 values)
        assert torch.equal(db.double(), positive.sum(0).double())


def test_more_statistics_than_a_launch_has_threads_for():
    """65600 batch elements x 1024 groups = 2^26 statistics and more, of elements of one and two rows.  Instance norm of two rows: the
    values are d and -d around their mean, so xh = +- d / sqrt(d^2 + eps)"""
    b, c = 65_600, 1024
    gen = torch.Generator(device="cuda").manual_seed(3)
    lengths = torch.ones(b, dtype=torch.int64, device="cuda")
    lengths[::40] = 2
    lengths[7::40] = 0
    off = torch.zeros(b + 1, dtype=torch.int64, device="cuda")
    off[1:] = lengths.cumsum(0)
    n = int(off[-1])
    x = torch.randn((n, c), generator=gen, device="cuda")
    w, bias = 1 + torch.rand(c, generator=gen, device="cuda"), torch.randn(c, generator=gen, device="cuda")
    assert b * c >= 2 ** 26
    y, mean, rstd = ops.group_norm_fwd(x, off, c, w, bias, 1e-5)
    first = off[:-1][lengths == 2]
    pair = torch.zeros(n, dtype=torch.bool, device="cuda")
    pair[first] = pair[first + 1] = True
    assert torch.equal(y[~pair], bias.expand(n, c)[~pair]) and int(rstd[7::40].count_nonzero()) == 0
    p, q = x[first].double(), x[first + 1].double()
    d, m = (p - q) / 2, (p + q) / 2
    r = 1 / torch.sqrt(d * d + 1e-5)
    ez = w.double() * 4 * u * (r * (p.abs() + m.abs()) + 1) + 2 * u * (w.double() + bias.abs().double())
    assert bool(((y[first].double() - (d * r * w + bias)).abs() <= ez + u * 4).all())
    assert bool(((mean[lengths == 2].double() - m).abs() <= 2 * u * m.abs() + 1e-30).all()) and bool(((rstd[lengths == 2].double() - r).abs() <= 2 * u * r).all())
    # one row: every value is its own mean, so its gradient is 0; two rows: dx = r (1 - xh^2) (dy1 - dy2) / 2 w
    dy = torch.randn((n, c), generator=gen, device="cuda")
    dx, dw, db = ops.group_norm_bwd(x, dy, off, c, w, bias, mean, rstd)
    assert int(dx[~pair].count_nonzero()) == 0
    xh, h1, h2 = d * r, dy[first].double() * w, dy[first + 1].double() * w
    exh = 4 * u * (r * (p.abs() + m.abs()) + 1)
    want = r * (1 - xh * xh) * (h1 - h2) / 2
    size = h1.abs() + h2.abs()
    assert bool(((dx[first].double() - want).abs() <= r * (20 * u * size + 4 * exh * size)).all())
    assert bool(((db.double() - dy.double().sum(0)).abs() <= 2 * u * dy.double().abs().sum(0)).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,c,groups,shuffled", [([900, 0, 1, 300], 64, 8, True), ([40_000] * 3, 20, 5, False), ([], 8, 2, False),
                                                      ([0], 16, 4, False), ([3, 5], 300, 300, False)])
def test_group_norm_makes_the_gradients_that_are_wanted(dtype, lengths, c, groups, shuffled):
    n = sum(lengths) + 30 * (len(lengths) > 2)  # rows behind the last element
    gen = torch.Generator(device="cuda").manual_seed(n + c)
    draw = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    x, dy, w, b = draw(n, c).to(dtype), draw(n, c).to(dtype), 1 + 0.2 * draw(c), draw(c)
    off = torch.tensor([0] + lengths, device="cuda").cumsum(0)
    order = torch.randperm(n, generator=gen, device="cuda") if shuffled else None
    _, mean, rstd = ops.group_norm_fwd(x, off, groups, w, b, 1e-5, 3, 0.0, order)
    full = ops.group_norm_bwd(x, dy, off, groups, w, b, mean, rstd, 3, 0.0, order)
    for k in range(8):
        want = [bool(k & 1), bool(k & 2), bool(k & 4)]
        got = ops.group_norm_bwd(x, dy, off, groups, w, b, mean, rstd, 3, 0.0, order, *want)
        assert all((g is None) != k and (g is None or torch.equal(g, f)) for g, f, k in zip(got, full, want)), want
    for frozen in range(1, 8):
        leaves = [t.clone().requires_grad_(not frozen >> i & 1) for i, t in enumerate((x, w, b))]
        y = modules.group_norm_act(leaves[0], off, groups, leaves[1], leaves[2], activation="silu", order=order)
        assert y.requires_grad == (frozen != 7)
        if frozen != 7:
            y.backward(dy)
        assert all(leaf.grad is None if frozen >> i & 1 else torch.equal(leaf.grad, f) for i, (leaf, f) in enumerate(zip(leaves, full))), frozen


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,cin,cout", [(1_250_000, 8, 8), (5_000_000, 8, 16), (1_250_001, 4, 200), (70_003, 16, 70)])
@pytest.mark.parametrize("kind", ["none", "silu"])
def test_bias_gradients_of_one_sign_over_many_rows(dtype, n, cin, cout, kind):
    """dy near 0.1 everywhere.  Sums of positive terms: a chain of k fp32 additions is off by k u / 2 of the sum at most (its partial sums grow
    evenly); no chain is longer than 1024 whatever n is, and what is added to it in fp64 rounds twice.  act' is off by 16 u."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn((n, cin), generator=gen, device="cuda").to(dtype)
    w = torch.zeros((cout, cin), device="cuda", dtype=dtype)  # z is the bias
    b = torch.linspace(0.5, 3, cout, device="cuda").to(dtype)
    room = (64 if dtype == torch.float32 else 512 + 16) * u
    for scale in (1.0, 1 / 64):
        dy = (scale * (0.1 + 0.001 * torch.arange(cout, device="cuda"))).to(dtype).expand(n, cout).contiguous()
        db = ops.linear_act_bwd(x, dy, w, b, ops.activation_id(kind), want_input=False, want_weight=False)[2]
        want = dy[0].double() * dact64(b.double(), kind) * n
        over = want > torch.finfo(dtype).max * (1 + HALF_STEP[dtype])  # (the sum itself is none of the type's numbers)
        assert bool((db[over] == math.inf).all())
        off = (db.double() / want - 1).abs()[~over]
        assert bool((off <= room + HALF_STEP[dtype] * (1 + room)).all()), off.max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,cin,cout", [(5, 8, 6), (300, 75, 133), (300, 64, 64), (400, 200, 392), (70_000, 40, 24)])
def test_infinities_do_what_they_do_in_a_sum(dtype, n, cin, cout):
    """rows, weights and gradients with infinities and the largest finite numbers: where the sum of 64 bits is infinite or NaN the result is,
    and where act makes a number of it, it is that number"""
    gen = torch.Generator(device="cuda").manual_seed(n)
    draw = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    x, w, b, dy = draw(n, cin).to(dtype), (0.1 + draw(cout, cin).abs()).to(dtype), draw(cout).to(dtype), draw(n, cout).to(dtype)
    x[0], x[n // 2, 3], x[n // 2, 5], x[n - 1, 0], x[2, 1] = -math.inf, math.inf, -math.inf, math.inf, math.nan
    w[2, 4] = 0.0
    x[3, 4] = math.inf  # times 0
    finite = torch.isfinite(x).all(1)
    plain_y = ops.linear_act_fwd(torch.where(finite[:, None], x, 0), w, b)
    plain = ops.linear_act_bwd(torch.where(finite[:, None], x, 0), dy, w, b, 1)
    z = x.double() @ w.double().t() + b.double()
    for kind in ("none", "relu", "leaky_relu"):
        y = ops.linear_act_fwd(x, w, b, ops.activation_id(kind), 0.2).double()
        want = torch.where(torch.isnan(z), z, z.clamp(min=0) if kind == "relu" else torch.where(z > 0, z, 0.2 * z) if kind == "leaky_relu" else z)
        special = ~finite
        assert torch.equal(torch.isnan(y[special]), torch.isnan(want[special])), kind
        keep = ~torch.isnan(want) & special[:, None]
        assert torch.equal(y[keep], want[keep].to(dtype).double()), kind  # infinities, and relu's zeros
    assert torch.equal(ops.linear_act_fwd(x, w, b)[finite], plain_y[finite])
    # relu of a row of -inf or +inf: slopes 0 and 1, so dx is finite; the row's part of dW is 0 * inf = NaN or inf
    dx, dw, db = ops.linear_act_bwd(x, dy, w, b, 1)
    assert torch.equal(dx[finite], plain[0][finite]) and int(dx[0].count_nonzero()) == 0 and bool(torch.isfinite(dx[n - 1]).all())
    assert bool(torch.isnan(dw).all()) and bool(torch.isfinite(db).all())  # (row 0: 0 * -inf in every entry)
    d = dy.clone()
    d[1, 2] = math.inf
    clean = torch.where(finite[:, None], x, 0)
    dx, dw, _ = ops.linear_act_bwd(clean, d, w, b, 0)
    assert torch.equal(torch.isnan(dx[1]), w[2] == 0) and bool((dx[1][w[2] > 0] == math.inf).all())
    want = math.inf * clean[1].double()
    assert torch.equal(torch.isnan(dw[2].double()), torch.isnan(want)) and torch.equal(dw[2].double()[want.abs() == math.inf], want[want.abs() == math.inf])
    same = torch.arange(cout, device="cuda") != 2
    assert torch.equal(dw[same], ops.linear_act_bwd(clean, dy, w, b, 0)[1][same])


def test_largest_numbers_of_fp32():
    """values above the largest bfloat16, and partial sums that pass the range but come back"""
    top = torch.finfo(torch.float32).max
    x = torch.tensor([[top, 1.0, 0.0], [-top, 0.0, 2.0], [top, top, 0.0], [3.4e38, 0.0, 1e38]], device="cuda")
    w = torch.tensor([[0.5, 0.0, 0.0], [1.0, 0.0, 0.0], [-0.25, -0.125, 1.0], [0.0, 2.0, 3.0]], device="cuda")
    y = ops.linear_act_fwd(x, w).double()
    want = (x.double() @ w.double().t())
    assert torch.equal(y, want.float().double()), (y, want)


def test_fp32_products_leave_out_little_and_on_both_sides():
    """one product per result: three bf16 terms of each operand, the middle one at most 2^-8 and the last 2^-16 of it, so the three products that
    are left out are at most (2 2^-24 + 2^-32) = 2.01 u of it; the addition of the largest rounds once more, by a whole step (2 u) at most"""
    gen = torch.Generator(device="cuda").manual_seed(0)
    x, w = (1 + torch.rand((2000, 1), generator=gen, device="cuda")), (1 + torch.rand((1000, 1), generator=gen, device="cuda"))
    off = ops.linear_act_fwd(x, w).double() / (x.double() @ w.double().t()) - 1
    assert float(off.abs().max()) <= 4.01 * u, float(off.abs().max() / u)
    # sums of positive terms: a step of 32 terms is six additions, each off by a whole step (2 u) at most of partial sums that grow evenly, and
    # at most one more inside it
    x, w = (0.5 + torch.rand((300, 512), generator=gen, device="cuda")), (0.5 + torch.rand((200, 512), generator=gen, device="cuda"))
    off = ops.linear_act_fwd(x, w).double() / (x.double() @ w.double().t()) - 1
    assert float(off.abs().max()) <= (2.01 + 512 / 32 * 6 * 2) * u


@pytest.mark.parametrize("n,cin,cout", [(10_000_000, 64, 32), (3_000_001, 130, 260), (300_000, 20, 600)])
def test_weight_gradients_of_one_sign_over_many_rows(n, cin, cout):
    """fp32, every product the same.  At most 2048 rows are one chain of fp32 additions, 64 steps of six: each is off by a whole step (2 u) at most
    of partial sums that grow evenly.  The split leaves out 2.01 u, and the parts are rounded, added in fp64 and rounded"""
    x, dy = torch.full((n, cin), 0.1, device="cuda"), torch.full((n, cout), 0.3, device="cuda")
    w = torch.zeros((cout, cin), device="cuda")
    dw = ops.linear_act_bwd(x, dy, w, None, 0, want_input=False, want_bias=False)[1]
    off = dw.double() / (x[0, 0].double() * dy[0, 0].double() * n) - 1
    assert float(off.abs().max()) <= (64 * 6 + 2.01 + 4) * u, float(off.abs().max() / u)
    assert int((dw != dw[0, 0]).sum()) == 0


def test_linear_layers_take_what_their_parent_takes():
    """any leading dimensions, and mixed types under autocast (which gives the result its type; operands of one type keep theirs)"""
    torch.manual_seed(1)
    layer = modules.LinearAct(24, 40, activation="silu").cuda()
    for shape in ((24,), (5, 24), (3, 7, 24), (2, 3, 4, 24), (0, 24), (4, 0, 24)):
        x = torch.randn(shape, device="cuda", requires_grad=True)
        res = torch.randn(*shape[:-1], 40, device="cuda", requires_grad=True)
        y = layer(x, res)
        assert y.shape == (*shape[:-1], 40)
        rows = ops.linear_act_fwd(x.detach().reshape(-1, 24), layer.weight.detach(), layer.bias.detach(), 3, 0.0, res.detach().reshape(-1, 40))
        assert torch.equal(y.detach().reshape(-1, 40), rows)
        dy = torch.randn_like(y)
        gx, gr = torch.autograd.grad(y, (x, res), dy)
        want = ops.linear_act_bwd(x.detach().reshape(-1, 24), dy.reshape(-1, 40), layer.weight.detach(), layer.bias.detach(), 3)[0]
        assert torch.equal(gx.reshape(-1, 24), want) and torch.equal(gr, dy)
    strided = torch.randn(6, 24, 5, device="cuda").transpose(1, 2)
    assert torch.equal(layer(strided), layer(strided.contiguous()))
    for bad in ((torch.randn((), device="cuda"), None), (torch.randn(3, 7, 23, device="cuda"), None),
                (torch.randn(3, 7, 24, device="cuda"), torch.randn(7, 3, 40, device="cuda"))):
        with pytest.raises(ValueError):
            layer(*bad)
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.randn(300, 24, device="cuda", requires_grad=True)
        with torch.autocast("cuda", dtype=dtype):
            y = layer(x.to(dtype))
            inner = layer(x.to(dtype), torch.zeros(300, 40, device="cuda"))
            full = layer(x)
        assert y.dtype == inner.dtype == dtype and torch.equal(full, layer(x))
        low = lambda t: t.detach().to(dtype)  # noqa: E731
        assert torch.equal(y, ops.linear_act_fwd(low(x), low(layer.weight), low(layer.bias), 3)) and torch.equal(inner, y)
        dy = torch.randn_like(y)
        grads = torch.autograd.grad(y, (x, layer.weight, layer.bias), dy)
        want = ops.linear_act_bwd(low(x), dy, low(layer.weight), low(layer.bias), 3)
        assert all(g.dtype == torch.float32 and torch.equal(g, w.float()) for g, w in zip(grads, want))
        with pytest.raises(TypeError):
            layer(x.to(dtype))  # without autocast: types are not mixed


def test_tangents_are_refused_not_dropped():
    x, t = torch.randn(6, 8, device="cuda"), torch.randn(6, 8, device="cuda")
    w, off = torch.randn(8, 8, device="cuda"), torch.tensor([0, 6], device="cuda")
    scale = torch.ones(8, device="cuda")
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        dual = torch.autograd.forward_ad.make_dual(x, t)
        for call in (lambda: modules.linear_act(dual, w), lambda: modules.linear_act(x, torch.autograd.forward_ad.make_dual(w, w)),
                     lambda: modules.linear_act(x, w, None, residual=dual), lambda: modules.group_norm_act(dual, off, 2),
                     lambda: modules.group_norm_act(x, off, 2, torch.autograd.forward_ad.make_dual(scale, scale))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert torch.equal(modules.linear_act(x, w), ops.linear_act_fwd(x, w))
    assert torch.equal(modules.group_norm_act(x, off, 2), ops.group_norm_fwd(x, off, 2)[0])


def rounds(g, steps, coefficients):
    """the iteration in 64 bits, and what the rounding of X to fp32 after every fifth step can make of it: an error grows by at most
    max |p'(sigma)| over the singular values that a step meets, p(x) = a x + b x^3 + c x^5"""
    a, b, c = coefficients
    x = g.double().cpu()
    x = x / (x.norm() + 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    bound = 0.0
    for k in range(steps):
        s = x @ x.t()
        lam = torch.linalg.eigvalsh(s).clamp(min=0)
        bound = bound * float((a + 3 * b * lam + 5 * c * lam * lam).abs().max()) + 1e-11  # (a round of five in fp64)
        x = a * x + (b * s + c * (s @ s)) @ x
        if steps > 8 and (k + 1) % 5 == 0 and k + 1 < steps:
            bound += u * float(x.norm())
    return (x.t() if tall else x), bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n", [(64, 64), (300, 48), (40, 333), (128, 1000)])
def test_newton_schulz_of_many_steps(dtype, m, n):
    gen = torch.Generator().manual_seed(m + n)
    g = torch.randn((m, n), generator=gen)
    if m == n:
        g = g + 8 * torch.eye(m)
    g = g.to(dtype)
    for coefficients in (ops.NEWTON_SCHULZ_COEFFICIENTS, (1.5, -0.5, 0.0), (2.0, -1.5, 0.5)):
        for steps in (8, 9, 10, 11, 13, 30):
            if steps == 30 and coefficients[0] > 3:
                continue  # (its singular values never settle: errors go on growing, in every precision)
            want, bound = rounds(g, steps, coefficients)
            got = ops.newton_schulz(g.cuda(), steps, coefficients).double().cpu()
            assert float((got - want).norm()) <= bound + (u + HALF_STEP[dtype]) * float(want.norm()) + TINY[dtype] * want.numel() ** 0.5, (steps, coefficients)


@pytest.mark.parametrize("dtype", DTYPES)
def test_newton_schulz_of_many_steps_keeps_missing_directions_small(dtype):
    """a matrix that lacks directions: they stay what rounding makes of them, and no singular value leaves the range that the polynomial maps
    to itself (p has its largest value, 1.21, at 0.56, and stays above 0.68 from there to 1.21)"""
    gen = torch.Generator().manual_seed(7)
    draw = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    twice, zero = draw(64, 64), draw(200, 48)
    twice[:, :32] = twice[:, 32:]
    zero[:, 5] = zero[:, 9] = 0
    for g in (twice, zero, draw(90, 1) @ draw(1, 60), draw(300, 10) @ draw(10, 64), draw(7, 1), torch.zeros(20, 30)):
        for steps in (9, 12, 16, 20, 40, 100):
            out = ops.newton_schulz(g.to(dtype).cuda(), steps)
            assert bool(torch.isfinite(out).all()), (tuple(g.shape), steps)
            # bfloat16's half step of every entry: at most 2^-8 |out|_F, with |out|_F^2 <= 64 values of 1.21^2
            assert float(torch.linalg.svdvals(out.double().cpu()).max()) <= 1.21 + (HALF_STEP[dtype] + 4 * u) * 1.21 * 8, (tuple(g.shape), steps)
            if g is zero:
                assert int(out[:, 5].count_nonzero()) == 0
    static = twice.to(dtype).cuda()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.newton_schulz(static, 21)
    for k in range(3):
        static.copy_(twice.roll(k, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.newton_schulz(static, 21)), k


@pytest.mark.parametrize("dtype,batch,m,n", [(torch.float32, 1, 70_001, 40), (torch.bfloat16, 5, 33, 15_000), (torch.float16, 1100, 200, 24),
                                            (torch.float32, 2, 65_600, 128)])
def test_newton_schulz_of_more_parts_than_workgroups(dtype, batch, m, n):
    """a workgroup takes several parts of 64 of the long side (whole numbers of them, and a short last one)"""
    gen = torch.Generator().manual_seed(n)
    g = torch.randn((batch, m, n), generator=gen).to(dtype)
    out = ops.newton_schulz(g.cuda()).double().cpu()
    for k in {0, batch // 2, batch - 1}:
        want, bound = rounds(g[k], 5, ops.NEWTON_SCHULZ_COEFFICIENTS)
        assert float((out[k] - want).norm()) <= bound + (u + HALF_STEP[dtype]) * float(want.norm()) + TINY[dtype] * want.numel() ** 0.5, k


@pytest.mark.parametrize("batch,m,n", [(4, 160, 4_194_304), (4, 4_194_304, 160)])
def test_newton_schulz_above_a_short_side_of_128_past_32_bits(batch, m, n):
    """more than 2^31 elements on the plane form: the same matrix at the start and at the end of a batch"""
    s, l = min(m, n), max(m, n)
    one = torch.zeros((l, s), dtype=torch.bfloat16, device="cuda")
    rows = torch.arange(l // s * s, device="cuda")
    one[rows, rows % s] = 0.5
    g = (one if m > n else one.t()).repeat(batch, 1, 1)
    assert g.numel() > 2 ** 31  # (the last matrix passes it)
    out = ops.newton_schulz(g)
    assert all(torch.equal(out[0], out[i]) for i in range(1, batch))
    # orthogonal columns of one length: every singular value is t = 1 / sqrt(s) of the norm, and so is every result
    t = s ** -0.5
    for _ in range(5):
        a, b, c = ops.NEWTON_SCHULZ_COEFFICIENTS
        t = a * t + b * t ** 3 + c * t ** 5
    value = t / (l // s) ** 0.5
    have = out[batch - 1] if m > n else out[batch - 1].t()
    # bfloat16's half step, and two planes: 2^-16 of three operands a step, 4 times as much in the later ones: below 2^-8 in all
    assert float((have[rows, rows % s].double() / value - 1).abs().max()) <= 2 ** -7
    assert int(have.count_nonzero()) == rows.numel()


@pytest.mark.parametrize("c,groups", [(8, 8), (8, 2), (7, 7), (96, 32), (300, 100)])
@pytest.mark.parametrize("lengths,shuffled", [([70_000], False), ([3, 40, 0, 30_000, 1], True), ([400_000, 200_000], False)])
def test_statistics_far_from_zero(c, groups, lengths, shuffled):
    """channels of one value, and of a small spread, around numbers up to 1e7: the mean is rounded once, 1 / std is off by what fp64 sums of
    distances to a value of the group leave, far below u, and its own rounding; without a spread it is 1 / sqrt(eps)"""
    n = sum(lengths)
    gen = torch.Generator(device="cuda").manual_seed(n + c)
    at = torch.tensor([0.3, 1000.1, 30000.7, 100000.3, 1000001.0, 1e7 + 1], device="cuda").repeat_interleave(c // groups).repeat(c)[:c]
    off = torch.tensor([0] + lengths, device="cuda").cumsum(0)
    order = torch.randperm(n, generator=gen, device="cuda") if shuffled else None
    w = 1 + torch.rand(c, generator=gen, device="cuda")
    dy = torch.randn((n, c), generator=gen, device="cuda")
    for spread in (0.0, 3.0):
        x = at + spread * torch.randn((n, c), generator=gen, device="cuda") if spread else at.expand(n, c).contiguous()
        _, mean, rstd = ops.group_norm_fwd(x, off, groups, w, None, 1e-5, 0, 0.0, order)
        dx = ops.group_norm_bwd(x, dy, off, groups, w, None, mean, rstd, 0, 0.0, order)[0]
        for e, (lo, hi) in enumerate(zip(off[:-1].tolist(), off[1:].tolist())):
            if hi == lo:
                assert int(rstd[e].count_nonzero()) == 0
                continue
            rows = torch.arange(lo, hi, device="cuda") if order is None else order[lo:hi]
            v = x[rows].double().view(hi - lo, groups, -1)
            want = v.mean((0, 2))
            var = ((v - want[:, None]) ** 2).mean((0, 2))
            r = 1 / torch.sqrt(var + 1e-5)
            assert bool(((mean[e].double() - want).abs() <= 2 * u * want.abs()).all())
            # a group of one value has mean v itself (n v / n rounds in this reference only)
            r = torch.where(torch.tensor(spread == 0.0, device="cuda"), 1e-5 ** -0.5, r)
            assert bool(((rstd[e].double() - r).abs() <= 2 * u * r).all()), (rstd[e].double() / r - 1).abs().max()
            if spread == 0.0:  # xh is 0: dx = rstd (h - mean(h))
                h = (dy[rows].double() * w).view(hi - lo, groups, -1)
                m = h.mean((0, 2), keepdim=True)
                d = dx[rows].double().view(hi - lo, groups, -1)
                assert bool(((d - r[:, None] * (h - m)).abs() <= 8 * u * r[:, None] * (h.abs() + m.abs())).all())
