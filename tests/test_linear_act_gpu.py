"""Linear layer with a fused epilogue and its gradients (ops.linear_act_fwd / _bwd, modules.linear_act) against 64 bits.

Error bounds.  u = 2^-24, U = half a step of the stored type.  A sum of N products whose partial sums stay below R has, from N
independent roundings of at most u R each, an error below 4 sqrt(N) u R in every one of 1e6 results; with terms of random sign
R <= 4 sqrt(sum of squares) + |sum|.  fp32 operands make six products of each (N = 6 K) and leave out less than 3 u of it.  act' is
good to 16 u and |act''| <= 0.8; dz is rounded once to the element type.  At the kink of relu / leaky an element whose |z| is below
its error may take either slope.  Whole-number inputs make every sum exact: there the results have to be equal."""
import pytest
import torch

from panopticsegforlargescalepointcloud_amd import _lib, modules, ops
from test_groupnorm_gpu import HALF_STEP, SLOPE, act64, dact64, kinked, near

pytestmark = pytest.mark.gpu

u = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def product(a, b, six):
    """a @ b and a bound of the fp32 evaluation's error"""
    n = a.shape[1] * (6 if six else 1)
    p = a @ b
    if a.shape[1] == 0:
        return p, torch.zeros_like(p)
    rms = torch.sqrt((a * a) @ (b * b))
    return p, 4 * u * n ** 0.5 * (4 * rms + p.abs()) + (3 * u * (a.abs() @ b.abs()) if six else 0)


def reference(x, w, b, kind, residual, dy):
    six, U = x.dtype == torch.float32, HALF_STEP[x.dtype]
    X, W = x.detach().double().cpu(), w.detach().double().cpu()
    z, ez = product(X, W.t(), six)
    if b is not None:
        z = z + b.detach().double().cpu()
        ez = ez + u * z.abs()
    y, ey = act64(z, kind), 1.13 * ez + 16 * u * z.abs()
    if residual is not None:
        y = y + residual.detach().double().cpu()
        ey = ey + u * y.abs()
    D = dy.double().cpu()
    dz = D * dact64(z, kind)
    edz = torch.zeros_like(dz) if kind == "none" else D.abs() * (0.8 * ez + 16 * u) + U * dz.abs()
    if kinked(kind):
        edz = edz + D.abs() * (z.abs() <= ez)
    dx, edx = product(dz, W, six)
    dw, edw = product(dz.t(), X, six)
    db, edb = product(torch.ones((1, dz.shape[0]), dtype=torch.float64), dz, False)
    return ((y, ey), (dx, edx + edz @ W.abs()), (dw, edw + edz.t() @ X.abs()), (db[0], edb[0] + edz.sum(0)))


def tensors(n, cin, cout, dtype, seed, bias=True, residual=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    x, w = r(n, cin), r(cout, cin) / cin ** 0.5
    b, res, dy = (0.3 * r(cout) if bias else None), (r(n, cout) if residual else None), 0.3 * r(n, cout)
    return [None if t is None else t.to(dtype).cuda() for t in (x, w, b, res, dy)]


def check(n, cin, cout, dtype, kind, bias=True, residual=True):
    x, w, b, res, dy = tensors(n, cin, cout, dtype, n + cin + cout, bias, residual)
    act = ops.activation_id(kind)
    y = ops.linear_act_fwd(x, w, b, act, SLOPE, res)
    dx, dw, db = ops.linear_act_bwd(x, dy, w, b, act, SLOPE)
    for got, want, what in zip((y, dx, dw, db), reference(x, w, b, kind, res, dy), ("y", "dx", "dweight", "dbias")):
        assert got.dtype == dtype
        near(got, *want, dtype, what)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["none", "relu", "leaky_relu", "silu", "gelu"])
def test_types_and_activations(dtype, kind):
    check(700, 96, 160, dtype, kind)
    check(300, 64, 48, dtype, kind, bias=False, residual=False)


@pytest.mark.parametrize("n,cin,cout", [
    (0, 16, 16), (1, 1, 1), (1, 64, 64), (2, 7, 3), (64, 112, 7), (64, 7, 112), (127, 33, 65), (129, 128, 129), (1000, 4, 16),
    (513, 75, 133), (260, 1024, 20), (90, 20, 1030), (300, 130, 64), (4097, 16, 5), (20_001, 64, 32), (9000, 36, 200), (33, 2050, 17),
    (700, 200, 392), (1030, 512, 264), (16_500, 128, 512),
])
@pytest.mark.parametrize("dtype", DTYPES)
def test_shapes(n, cin, cout, dtype):
    check(n, cin, cout, dtype, "silu")


@pytest.mark.parametrize("n", [1, 2, 3, 130])
@pytest.mark.parametrize("cin,cout", [(1, 1), (2, 3), (3, 2), (5, 7), (7, 5), (1, 7), (7, 1)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_shorter_than_a_vector(n, cin, cout, dtype):
    """Rows of fewer than eight elements: what a load takes beside its own row still lies inside the tensor."""
    check(n, cin, cout, dtype, "silu")


@pytest.mark.parametrize("n,cin,cout", [(1, 5, 9), (131, 64, 64), (300, 75, 133), (640, 192, 96), (1025, 40, 260), (5000, 16, 24),
                                        (12_000, 130, 70), (700, 200, 392), (1030, 512, 264), (16_500, 128, 512), (70_000, 256, 512),
                                        (520, 264, 1160)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_whole_numbers_are_exact(n, cin, cout, dtype):
    g = torch.Generator().manual_seed(n)
    draw = lambda *s: torch.randint(-3, 4, s, generator=g).double()  # noqa: E731
    x, w, b, res, dy = draw(n, cin), draw(cout, cin), draw(cout), draw(n, cout), draw(n, cout)
    up = lambda t: t.to(dtype).cuda()  # noqa: E731
    stored = lambda t: t.float().to(dtype).cpu()  # noqa: E731  (sums below 2^24: exact in fp32, then one rounding)
    z = x @ w.t() + b
    assert torch.equal(ops.linear_act_fwd(up(x), up(w), up(b), 1, 0.0, up(res)).cpu(), stored(z.clamp(min=0) + res))
    dz = dy * (z > 0)
    dx, dw, db = ops.linear_act_bwd(up(x), up(dy), up(w), up(b), 1)
    assert torch.equal(dx.cpu(), stored(dz @ w))
    assert torch.equal(dw.cpu(), stored(dz.t() @ x).clamp(-65504, 65504) if dtype == torch.float16 else stored(dz.t() @ x))
    assert torch.equal(db.cpu(), stored(dz.sum(0)))
    dx, dw, db = ops.linear_act_bwd(up(x), up(dy), up(w), None, 0)
    assert torch.equal(dx.cpu(), stored(dy @ w)) and torch.equal(dw.cpu(), stored(dy.t() @ x)) and torch.equal(db.cpu(), stored(dy.sum(0)))


@pytest.mark.parametrize("n,cin,cout", [(64, 1, 1), (8193, 3, 5), (9001, 31, 33), (65_537, 64, 64), (8200, 96, 96), (70_001, 75, 133), (65_536, 128, 128), (12_345, 75, 133), (8192, 160, 160), (65_600, 159, 160),
                                        (8211, 129, 40), (8299, 40, 129), (20_000, 128, 128), (9000, 7, 160), (9000, 160, 7), (8192, 97, 96)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_narrow_layers_over_many_rows(n, cin, cout, dtype):
    check(n, cin, cout, dtype, "gelu")
    check(n, cin, cout, dtype, "none", bias=False, residual=False)
    g = torch.Generator().manual_seed(n)
    draw = lambda *s: torch.randint(-3, 4, s, generator=g).double()  # noqa: E731
    x, w, b, res, dy = draw(n, cin), draw(cout, cin), draw(cout), draw(n, cout), draw(n, cout)
    up, stored = (lambda t: t.to(dtype).cuda()), (lambda t: t.float().to(dtype).cpu())  # noqa: E731
    z = x @ w.t() + b
    assert torch.equal(ops.linear_act_fwd(up(x), up(w), up(b), 1, 0.0, up(res)).cpu(), stored(z.clamp(min=0) + res))
    dz = dy * (z > 0)
    for act, d in ((1, dz), (0, dy)):
        dx, dw, db = ops.linear_act_bwd(up(x), up(dy), up(w), up(b), act)
        assert torch.equal(dx.cpu(), stored(d @ w)) and torch.equal(dw.cpu(), stored(d.t() @ x)) and torch.equal(db.cpu(), stored(d.sum(0)))
        for want in ((True, False, False), (False, True, False), (False, False, True)):
            got = ops.linear_act_bwd(up(x), up(dy), up(w), up(b), act, want_input=want[0], want_weight=want[1], want_bias=want[2])
            assert all((p is None) != k and (not k or torch.equal(p, q)) for p, q, k in zip(got, (dx, dw, db), want))


def test_narrow_layers_keep_non_finite_rows_apart_and_repeat():
    x, w, b, res, dy = tensors(9000, 75, 133, torch.bfloat16, 11)
    clean = ops.linear_act_bwd(x, dy, w, b, 3)
    again = ops.linear_act_bwd(x, dy, w, b, 3)
    assert all(torch.equal(p, q) for p, q in zip(clean, again))
    bad = x.clone()
    bad[7, 3], bad[8999, 74] = float("nan"), float("inf")
    y, dx = ops.linear_act_fwd(bad, w, b, 3, 0.0, res), ops.linear_act_bwd(bad, dy, w, b, 3)[0]
    keep = torch.ones(9000, dtype=torch.bool, device="cuda")
    keep[7] = keep[8999] = False
    assert torch.equal(y[keep], ops.linear_act_fwd(x, w, b, 3, 0.0, res)[keep]) and torch.equal(dx[keep], clean[0][keep])


def test_fp32_keeps_all_bits_of_its_operands():
    """one product per result: fp32 operands of 24 significant bits against a power of two come back unchanged"""
    x = torch.randn(200, 64, device="cuda")
    x = x * torch.exp2(torch.randint(-30, 30, x.shape, device="cuda").float())
    w = 0.5 * torch.eye(64, device="cuda")
    assert torch.equal(ops.linear_act_fwd(x, w), 0.5 * x)
    dx, dw, _ = ops.linear_act_bwd(x, x, w)
    assert torch.equal(dx, 0.5 * x)


def test_non_finite_rows_stay_rows():
    x, w, b, res, dy = tensors(300, 75, 133, torch.bfloat16, 1)
    for act in (0, 1, 3, 4):
        clean, cdx = ops.linear_act_fwd(x, w, b, act, 0.0, res), ops.linear_act_bwd(x, dy, w, b, act)[0]
        bad = x.clone()
        bad[7, 3], bad[200, 74] = float("nan"), float("inf")
        y, dx = ops.linear_act_fwd(bad, w, b, act, 0.0, res), ops.linear_act_bwd(bad, dy, w, b, act)[0]
        keep = torch.ones(300, dtype=torch.bool, device="cuda")
        keep[7] = keep[200] = False
        assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], cdx[keep])
        assert torch.isnan(y[7]).all()
    # relu of a row of +inf: slope 1, so the input gradient is finite, the padding columns of dz notwithstanding
    big = torch.full((4, 75), float("inf"), device="cuda", dtype=torch.bfloat16)
    ones = torch.ones((133, 75), device="cuda", dtype=torch.bfloat16)
    assert torch.equal(ops.linear_act_bwd(big, dy[:4].contiguous(), ones, None, 1)[0].float(),
                       ops.linear_act_bwd(torch.ones_like(big), dy[:4].contiguous(), ones, None, 1)[0].float())


def test_module_gradients_and_what_is_wanted():
    x, w, b, res, dy = tensors(500, 40, 72, torch.float32, 2)
    full = ops.linear_act_bwd(x, dy, w, b, 3)
    for frozen in range(4):
        leaves = [t.clone().requires_grad_(i != frozen) for i, t in enumerate((x, w, b, res))]
        y = modules.linear_act(leaves[0], leaves[1], leaves[2], activation="silu", residual=leaves[3])
        y.backward(dy)
        for i, (leaf, want) in enumerate(zip(leaves, (*full, dy))):
            assert leaf.grad is None if i == frozen else torch.equal(leaf.grad, want), (frozen, i)
    with torch.no_grad():
        assert not modules.linear_act(x.requires_grad_(), w, b).requires_grad
    # a weight used twice and a bias of a broadcast gradient: autograd adds what the two calls give
    wl = w.clone().requires_grad_()
    (modules.linear_act(x.detach(), wl, b, activation="gelu").sum() + modules.linear_act(2 * x.detach(), wl, b, activation="gelu").sum()).backward()
    one = torch.ones_like(dy)
    assert torch.equal(wl.grad, ops.linear_act_bwd(x.detach(), one, w, b, 4)[1] + ops.linear_act_bwd(2 * x.detach(), one, w, b, 4)[1])


def test_gradients_against_differences():
    x, w, b, res, dy = tensors(60, 20, 30, torch.float32, 3)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, res)]
    modules.linear_act(leaves[0], leaves[1], leaves[2], activation="gelu", residual=leaves[3]).backward(dy)
    bounds = [e for _, e in reference(x, w, b, "gelu", res, dy)[1:]] + [torch.zeros(60, 30, dtype=torch.float64)]
    g = torch.Generator().manual_seed(1)
    for at, leaf in enumerate(leaves):
        v = torch.randn(leaf.shape, generator=g, dtype=torch.float64)
        h, vals = 1e-5, []
        for sign in (1, -1):
            t = [p.double().cpu() for p in (x, w, b, res)]
            t[at] = t[at] + sign * h * v
            vals.append(((act64(t[0] @ t[1].t() + t[2], "gelu") + t[3]) * dy.double().cpu()).sum())
        want, got = (vals[0] - vals[1]) / (2 * h), (leaf.grad.double().cpu() * v).sum()
        room = ((bounds[at] + u * leaf.grad.double().cpu().abs()) * v.abs()).sum() + 1e-6 * want.abs() + 1e-6
        assert abs(got - want) <= room, (at, float(got), float(want), float(room))


def test_unaligned_strided_and_broadcast():
    base = torch.randn(3 + 200 * 64, device="cuda")
    x, w = base[3:].view(200, 64), torch.randn(65 * 64 + 1, device="cuda")[1:].view(65, 64)
    want = reference(x, w, None, "relu", None, torch.ones(200, 65))
    near(ops.linear_act_fwd(x, w, None, 1), *want[0], torch.float32, "unaligned")
    wide = torch.randn((200, 100), device="cuda")
    near(ops.linear_act_fwd(wide[:, 5:69], w, None, 1), *reference(wide[:, 5:69], w, None, "relu", None, torch.ones(200, 65))[0],
         torch.float32, "strided")
    got = ops.linear_act_bwd(x, torch.ones((1, 1), device="cuda").expand(200, 65), w, None, 1)
    for g, wnt in zip(got, want[1:]):
        near(g, *wnt, torch.float32, "broadcast gradient")
    wt = torch.randn((64, 65), device="cuda").t()
    near(ops.linear_act_fwd(x, wt, None, 1), *reference(x, wt, None, "relu", None, torch.ones(200, 65))[0], torch.float32, "transposed weight")


def test_repeats_stream_and_graph():
    x, w, b, res, dy = tensors(30_000, 64, 96, torch.bfloat16, 5)
    one = ops.linear_act_bwd(x, dy, w, b, 3)
    assert all(torch.equal(p, q) for p, q in zip(one, ops.linear_act_bwd(x, dy, w, b, 3)))
    want = ops.linear_act_fwd(x, w, b, 3, 0.0, res)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.linear_act_fwd(x, w, b, 3, 0.0, res)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    sx, sdy = x.clone(), dy.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fy = ops.linear_act_fwd(sx, w, b, 3, 0.0, res)
        by = ops.linear_act_bwd(sx, sdy, w, b, 3)
    for k in range(3):
        sx.copy_(x * (k + 1))
        sdy.copy_(dy * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(fy, ops.linear_act_fwd(sx, w, b, 3, 0.0, res)), k
        assert all(torch.equal(p, q) for p, q in zip(by, ops.linear_act_bwd(sx, sdy, w, b, 3))), k


@pytest.mark.parametrize("dtype,blocks,cin,cout", [(torch.bfloat16, 4200, 128, 8), (torch.float16, 4200, 8, 128), (torch.bfloat16, 4200, 128, 128),
                                                  (torch.float32, 4200, 128, 8), (torch.bfloat16, 530, 1024, 256)])
def test_offsets_past_32_bits(dtype, blocks, cin, cout):
    """More than 2^31 elements: 4096 rows of small whole numbers again and again give the same results again and again.  Every sum is a
    whole number below 2^24 (weight gradient: blocks times one block's, which is below 2^10), so fp32 holds it whatever the order."""
    g = torch.Generator().manual_seed(blocks + cin)
    draw = lambda *s: torch.randint(-1, 2, s, generator=g).double()  # noqa: E731
    x, w, b, dy = draw(4096, cin), draw(cout, cin), draw(cout), draw(4096, cout)
    up = lambda t: t.to(dtype).cuda()  # noqa: E731
    same = lambda t, want: bool((t.view(blocks, 4096, -1) == up(want)).all())  # noqa: E731
    many = lambda t: up(t).repeat(blocks, 1)  # noqa: E731
    assert max(cin, cout) * 4096 * blocks > 2 ** 31
    z = x @ w.t() + b
    big, big_dy = many(x), many(dy)
    assert same(ops.linear_act_fwd(big, up(w), up(b), 1), z.clamp(min=0))
    for act, dz in ((1, dy * (z > 0)), (0, dy)):
        dw_one = dz.t() @ x
        assert dw_one.abs().max() < 2 ** 10 and dz.sum(0).abs().max() < 2 ** 10
        dx, dw, db = ops.linear_act_bwd(big, big_dy, up(w), up(b), act)
        assert same(dx, dz @ w)
        assert torch.equal(dw, up((dw_one * blocks).float())) and torch.equal(db, up((dz.sum(0) * blocks).float()))
        del dx


def test_refusals():
    x, w, b, res, dy = tensors(10, 12, 8, torch.float32, 6)
    for args, err in (((x, w[:, :11].contiguous()), ValueError), ((x.view(-1), w), ValueError), ((x, w.half()), TypeError),
                      ((x.double(), w.double()), TypeError), ((x, w, b[:7].contiguous()), ValueError), ((x, w, b.cpu()), _lib.PanopticHipError),
                      ((x, w, b, 0, 0.0, res[:9].contiguous()), ValueError), ((x, w, b, 0, 0.0, res[:1]), ValueError)):
        with pytest.raises(err):
            ops.linear_act_fwd(*args)
    with pytest.raises(ValueError):
        ops.linear_act_bwd(x, dy[:, :7].contiguous(), w, b)
    with pytest.raises(_lib.PanopticHipError):
        ops.linear_act_fwd(x, w, b, 9)
