"""Newton-Schulz orthogonalisation (ops.newton_schulz) and the optimiser built on it against the iteration in 64 bits.

Error bound.  The steps run in fp64 on the Gram matrix S of the shorter side s.  An error of S grows by at most a^2 = 11.9 a step
(in the directions where S is near 0; elsewhere the iteration contracts), a product of s terms rounds by s 2^-53 at most, and a step
has four of them: 4 s 2^-53 (1 + 11.9 + .. + 11.9^(steps - 1)) < 4 s 2^-53 1.1 a^(2 steps - 2), taken relative to the largest value an
entry can have (the largest singular value, 1.3).  The result is rounded to fp32 and to its type.

Shorter sides above 128 run the iteration in operands of two (16-bit types) or three bf16 planes, e = 2^-18 or 2^-26 of a value (each
plane rounds to half a step of 8 bits).  In a step, X, P and S are rounded to planes and the products leave out pairs below e: less than
9 e |P| |X|_F in all (S enters P with |b + 2 c S| < 5), and fp32 sums of 6 s products of random sign add sqrt(6 s) u |P| |X|_F.  What a
step brings grows in the later ones by at most max |p'(sigma)| over the singular values they meet, p(x) = a x + b x^3 + c x^5."""
import pytest
import torch

from panopticsegforlargescalepointcloud_amd import _lib, ops
from test_groupnorm_gpu import HALF_STEP, TINY

pytestmark = pytest.mark.gpu
A, B, C = ops.NEWTON_SCHULZ_COEFFICIENTS
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def iterate(g, steps=5, coefficients=(A, B, C), eps=1e-7, planes=None):
    """the definition, one matrix, 64 bits on the CPU; with `planes`, and the bound of the plane form's error (Frobenius norm)"""
    a, b, c = coefficients
    x = g.detach().double().cpu()
    x = x / (x.norm() + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    e = {None: 0.0, 2: 2.0 ** -18, 3: 2.0 ** -26}[planes]
    bound = 0.0
    for _ in range(steps):
        s = x @ x.t()
        p = a * torch.eye(len(s), dtype=torch.float64) + b * s + c * (s @ s)
        if planes:
            lam = torch.linalg.eigvalsh(s).clamp(min=0)
            bound = bound * float((a + 3 * b * lam + 5 * c * lam * lam).abs().max())
            bound += (9 * e + (6 * len(s)) ** 0.5 * 2.0 ** -24) * float(torch.linalg.matrix_norm(p, 2)) * float(x.norm())
        x = p @ x
    x = x.t() if tall else x
    return (x, bound) if planes else x


def check(g, steps=5, coefficients=(A, B, C), eps=1e-7):
    out = ops.newton_schulz(g, steps, coefficients, eps)
    assert out.shape == g.shape and out.dtype == g.dtype
    U = HALF_STEP[g.dtype]
    s = min(g.shape[-2:])
    for o, x in zip(out.view(-1, *g.shape[-2:]), g.view(-1, *g.shape[-2:])):
        if s > 128:
            want, bound = iterate(x, steps, coefficients, eps, 3 if g.dtype == torch.float32 else 2)
            off = float((o.double().cpu() - want).norm())
            assert off <= bound + (U + 2.0 ** -24) * float(want.norm()) + TINY[g.dtype] * want.numel() ** 0.5, (tuple(g.shape), off, bound)
            continue
        want = iterate(x, steps, coefficients, eps)
        room = (U + 2.0 ** -24) * want.abs() + 4 * s * 2.0 ** -53 * 1.1 * abs(coefficients[0]) ** (2 * steps - 2) * 1.3 + TINY[g.dtype]
        over = (o.double().cpu() - want).abs() - room
        assert bool((over <= 0).all()), (tuple(g.shape), float(over.max()))


def matrices(batch, m, n, dtype, seed=0, scale=1e-3):
    """a few strong directions over a floor of noise"""
    gen = torch.Generator().manual_seed(seed)
    k = max(1, min(m, n) // 8)
    strong = torch.randn((batch, m, k), generator=gen) / (1 + torch.arange(k)) @ torch.randn((batch, k, n), generator=gen)
    return ((strong + torch.randn((batch, m, n), generator=gen)) * scale).to(dtype).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,m,n", [(1, 129, 129), (2, 300, 260), (3, 140, 1000), (1, 1030, 520), (1, 512, 512), (2, 256, 2049), (1, 3000, 131)])
def test_long_short_sides(batch, m, n, dtype):
    check(matrices(batch, m, n, dtype, seed=m + n))
    gen = torch.Generator().manual_seed(m)
    check(torch.randn((1, m, n), generator=gen).to(dtype).cuda())  # singular values near each other: nothing grows


def test_scales_of_large_matrices():
    for scale in (1e-30, 1e-6, 1e6, 1e25):
        check(matrices(2, 300, 200, torch.float32, scale=scale), eps=0.0)
    check(matrices(1, 300, 200, torch.float16, scale=1.0))
    for steps in (1, 2):
        check(matrices(1, 200, 300, torch.bfloat16), steps=steps)
    g = matrices(4, 200, 190, torch.float32)
    clean = ops.newton_schulz(g)
    h = g.clone()
    h[0] = 0
    h[1, 3, 4] = float("nan")
    h[2, 60, 0] = float("inf")
    out = ops.newton_schulz(h)
    assert torch.equal(out[0], torch.zeros_like(out[0])) and torch.equal(out[3], clean[3])
    assert torch.isnan(out[1]).all() and torch.isnan(out[2]).all()
    want = ops.newton_schulz(g)
    static = g.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.newton_schulz(static)
    for k in range(3):
        static.copy_(g * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.newton_schulz(static)), k
    assert torch.equal(want, clean)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,m,n", [
    (1, 1, 1), (1, 1, 9), (2, 9, 1), (3, 5, 5), (1, 16, 64), (2, 64, 64), (4, 65, 64), (1, 63, 200), (2, 130, 75), (3, 432, 16),
    (2, 1728, 64), (1, 864, 112), (2, 96, 700), (1, 257, 129), (1, 200, 256), (5, 33, 31), (2, 500, 128), (1, 127, 1000), (1, 1001, 97), (2, 48, 333), (1, 80, 81),
])
def test_shapes(batch, m, n, dtype):
    check(matrices(batch, m, n, dtype, seed=m + n))


def test_one_matrix_and_other_polynomials():
    g = matrices(1, 80, 48, torch.float32)[0]
    check(g)
    for steps in (1, 2, 3, 8):
        check(g, steps=steps)
    check(g, coefficients=(1.5, -0.5, 0.0))  # the cubic iteration
    check(g, eps=0.0)
    check(g, eps=1.0)


def test_scales_and_strong_directions():
    for scale in (1e-18, 1e-6, 1e6, 1e18):  # squares of the small ones vanish in fp32
        check(matrices(2, 100, 40, torch.float32, scale=scale), eps=0.0)
    g = torch.randn(60, 1, device="cuda") @ torch.randn(1, 90, device="cuda")  # rank one: all other directions are rounding noise
    check(g)


def test_zero_nan_and_inf_stay_in_their_matrix():
    g = matrices(4, 70, 90, torch.float32)
    clean = ops.newton_schulz(g)
    h = g.clone()
    h[0] = 0
    h[1, 3, 4] = float("nan")
    h[2, 60, 0] = float("inf")
    out = ops.newton_schulz(h)
    assert torch.equal(out[0], torch.zeros_like(out[0])) and torch.equal(out[3], clean[3])
    assert torch.isnan(out[1]).all() and torch.isnan(out[2]).all()


def test_singular_values_come_near_one():
    g = torch.randn(3, 300, 64, device="cuda")
    sv = torch.linalg.svdvals(ops.newton_schulz(g).double().cpu())
    assert float(sv.min()) > 0.6 and float(sv.max()) < 1.3


def test_batch_strides_repeats_stream_and_graph():
    g = matrices(6, 200, 96, torch.bfloat16)
    want = ops.newton_schulz(g)
    assert torch.equal(want, ops.newton_schulz(g))
    assert torch.equal(want[2], ops.newton_schulz(g[2])) or torch.allclose(want[2].float(), ops.newton_schulz(g[2]).float(), rtol=2.0 ** -7)
    assert torch.equal(ops.newton_schulz(g.transpose(1, 2)), ops.newton_schulz(g.transpose(1, 2).contiguous()))
    assert torch.equal(ops.newton_schulz(g[:, ::2]), ops.newton_schulz(g[:, ::2].contiguous()))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.newton_schulz(g)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    static = g.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.newton_schulz(static)
    for k in range(3):
        static.copy_(g.flip(0) * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.newton_schulz(static)), k


@pytest.mark.parametrize("dtype,batch,m,n", [(torch.bfloat16, 6, 4_000_000, 96), (torch.bfloat16, 3, 160, 4_194_304)])
def test_offsets_past_32_bits(dtype, batch, m, n):
    """More than 2^31 elements: the same matrix at the start and at the end of a batch; diagonals of one value below each other, so
    that the result is a multiple of it."""
    s, l = min(m, n), max(m, n)
    one = torch.zeros((l, s), dtype=dtype, device="cuda")
    rows = torch.arange(l // s * s, device="cuda")
    one[rows, rows % s] = 0.5
    g = (one if m > n else one.t()).repeat(batch, 1, 1)
    assert g.numel() > 2 ** 30 and (batch - 1) * m * n * g.element_size() > 2 ** 31
    out = ops.newton_schulz(g)
    assert all(torch.equal(out[0], out[i]) for i in range(1, batch))
    # columns of one length, orthogonal: all singular values are one number t = 1 / sqrt(s) of the norm, and so are they in the result
    t = s ** -0.5
    for _ in range(5):
        a, b, c = ops.NEWTON_SCHULZ_COEFFICIENTS
        t = a * t + b * t ** 3 + c * t ** 5
    value = t / (l // s) ** 0.5  # every column has l // s entries
    have = out[0] if m > n else out[0].t()
    # bf16's half step; two planes of 8 bits leave 2^-16 of an operand, three operands a step, of which the later steps make no more than
    # |t f'(t) / f(t)| <= 4 times as much: below 2^-8 in all
    assert float((have[rows, rows % s].double() / value - 1).abs().max()) <= 2 ** -7
    assert int(have.count_nonzero()) == rows.numel()


def test_refusals():
    g = torch.randn(8, 8, device="cuda")
    for bad, err in ((torch.zeros(8, device="cuda"), ValueError), (torch.zeros(2, 2, 2, 2, device="cuda"), ValueError),
                     (torch.zeros(0, 8, device="cuda"), ValueError), (g.double(), TypeError), (g.cpu(), _lib.PanopticHipError)):
        with pytest.raises(err):
            ops.newton_schulz(bad)
    with pytest.raises(ValueError):
        ops.newton_schulz(g, steps=0)
    with pytest.raises(_lib.PanopticHipError):
        ops.newton_schulz(g, eps=-1.0)
    with pytest.raises(ValueError):
        ops.newton_schulz(g, coefficients=(1.0, 2.0))
    assert ops.newton_schulz(torch.zeros(0, 4, 4, device="cuda")).shape == (0, 4, 4)
