"""CPU: argument checks of the row operators -- the C entries refuse bad arguments before anything is launched, the Python entries
refuse tensors that do not live on a HIP device."""
import ctypes as C

import pytest
import torch

from panopticsegforlargescalepointcloud_amd import _lib, modules, ops, training

INVALID, WORKSPACE = 1, 4
P = C.c_void_p(4096)  # never read: every call below is refused before a launch


def group_norm(**kw):
    a = dict(x=P, dtype=0, n=10, c=8, groups=2, offsets=P, b=1, order=None, weight=None, bias=None, eps=1e-5, act=0, slope=0.0, y=P,
             mean=P, rstd=P, ws=P, wsb=1 << 20, stream=None)
    a.update(kw)
    return _lib.load().pp_group_norm_fwd(*a.values())


@pytest.mark.parametrize("kw", [{"dtype": 3}, {"dtype": -1}, {"act": 5}, {"act": -1}, {"c": 0}, {"c": 1025, "groups": 1}, {"groups": 3},
                                {"groups": 0}, {"n": -1}, {"b": -1}, {"b": 1 << 40}, {"offsets": None}, {"x": None}, {"y": None},
                                {"mean": None}, {"ws": None}])
def test_group_norm_entry_refuses(kw):
    assert group_norm(**kw) == INVALID
    assert b"pp_group_norm" in _lib.load().pp_last_error()


def test_group_norm_workspace():
    lib = _lib.load()
    assert group_norm(wsb=8) == WORKSPACE
    assert lib.pp_group_norm_workspace(-1, 1, 8, 2, 0) == 0
    for n in (0, 1, 65536, 65537, 1 << 33):
        for b in (0, 1, 5000):
            chunks = -(-n // max(32, -(-n // 1024)))  # a slot per chunk and element that meet, two fp64 sums per group; backward two per channel and chunk
            assert lib.pp_group_norm_workspace(n, b, 64, 8, 0) >= (chunks + b) * 8 * 16
            assert lib.pp_group_norm_workspace(n, b, 64, 8, 1) >= (chunks + b) * 8 * 16 + chunks * 64 * 16 + b * 8 * 8


def test_cpu_tensors_are_refused():
    x = torch.zeros((4, 8))
    with pytest.raises(_lib.PanopticHipError):
        ops.group_norm_fwd(x, torch.tensor([0, 4]), 2)
    with pytest.raises(_lib.PanopticHipError):
        modules.group_norm_act(x.requires_grad_(), torch.tensor([0, 4]), 2)


def test_activation_names():
    assert ops.activation_id(None) == ops.activation_id("none") == 0
    with pytest.raises(ValueError):
        ops.activation_id("swish2")


def linear(**kw):
    a = dict(x=P, dtype=0, n=10, cin=8, w=P, cout=8, bias=None, act=0, slope=0.0, residual=None, y=P, stream=None)
    a.update(kw)
    return _lib.load().pp_linear_act_fwd(*a.values())


@pytest.mark.parametrize("kw", [{"dtype": 3}, {"act": 5}, {"cin": 0}, {"cout": 0}, {"cout": (1 << 20) + 1}, {"n": -1}, {"w": None},
                                {"x": None}, {"y": None}, {"n": 1 << 31}])
def test_linear_act_entry_refuses(kw):
    assert linear(**kw) == INVALID


def test_linear_act_backward_entry_refuses():
    lib = _lib.load()
    a = [P, P, 0, 10, 8, P, 8, None, 3, 0.0, P, P, P, P, lib.pp_linear_act_bwd_workspace(0, 10, 8, 8, 3), None]
    for at, value, rc in ((1, None, INVALID), (13, None, INVALID), (14, 100, WORKSPACE), (13, C.c_void_p(4100), INVALID), (8, 7, INVALID)):
        assert lib.pp_linear_act_bwd(*(a[:at] + [value] + a[at + 1:])) == rc
    with pytest.raises(_lib.PanopticHipError):
        modules.linear_act(torch.zeros((4, 8)), torch.zeros((3, 8)))


def test_newton_schulz_entry_refuses():
    lib = _lib.load()
    a = [P, 0, 2, 40, 30, 5, 3.4, -4.7, 2.0, 1e-7, P, P, lib.pp_newton_schulz_workspace(2, 40, 30), None]
    for at, value, rc in ((1, 4, INVALID), (2, -1, INVALID), (2, 1 << 17, INVALID), (3, 0, INVALID), (4, 1 << 40, INVALID), (5, 0, INVALID),
                          (5, 101, INVALID), (9, -1.0, INVALID), (0, None, INVALID), (11, C.c_void_p(4104), INVALID), (12, 10, WORKSPACE)):
        assert lib.pp_newton_schulz(*(a[:at] + [value] + a[at + 1:])) == rc, at
    assert lib.pp_newton_schulz(*(a[:3] + [9000, 9000] + a[5:])) == INVALID
    assert lib.pp_newton_schulz_workspace(1, 0, 4) == 0
    with pytest.raises(_lib.PanopticHipError):
        ops.newton_schulz(torch.zeros(4, 4))


def test_newton_schulz_workspace_stays_near_the_input():
    """short sides up to 128: partial Gram matrices of at most 1024 workgroups (one a matrix in larger batches), five more matrices a batch
    element; more than eight steps: two fp32 copies beside them.  Above 128: two X and two S-sized matrices of two (16 bits) or three planes"""
    lib = _lib.load()
    for batch, m, n in ((6, 4_000_000, 96), (1, 128, 4_194_304), (8, 1728, 64), (3, 5184, 96), (3000, 100, 100), (1, 7, 1)):
        s, l = min(m, n), max(m, n)
        gram = min(batch * -(-l // 64), max(1024, batch)) * s * s * 8
        for dtype in (0, 1, 2):
            short = lib.pp_newton_schulz_workspace_for(dtype, batch, m, n, 5)
            assert 4 * batch * s * s * 8 <= short <= gram + 4 * batch * s * s * 8 + 4096
            assert short + 8 * batch * m * n <= lib.pp_newton_schulz_workspace_for(dtype, batch, m, n, 9) <= lib.pp_newton_schulz_workspace(batch, m, n)
    assert lib.pp_newton_schulz_workspace_for(1, 6, 4_000_000, 96, 5) < 100 << 20
    low, full = (lib.pp_newton_schulz_workspace_for(dtype, 2, 4096, 1024, 5) for dtype in (1, 0))
    assert low < full == lib.pp_newton_schulz_workspace(2, 4096, 1024) and low >= 2 * 2 * 2 * (4096 * 1024 + 1024 * 1024) * 2
    assert lib.pp_newton_schulz_workspace_for(0, -1, 4, 4, 5) == 0


def test_muon_refuses_before_it_changes_anything():
    def param(*shape):
        return torch.nn.Parameter(torch.ones(shape))
    good = param(4, 3)
    for bad in (param(4), param(0, 3), param(3, 0), param(2, 0, 3), param(9000, 1).expand(9000, 9000).detach().requires_grad_()):
        with pytest.raises(ValueError, match="Muon"):
            training.Muon([good, bad])
        opt = training.Muon([good])
        with pytest.raises(ValueError, match="Muon"):
            opt.add_param_group({"params": [bad]})
        assert len(opt.param_groups) == 1
    sparse = param(4, 3)
    sparse.grad = torch.ones(4, 3).to_sparse()
    good.grad = torch.ones(4, 3)
    opt = training.Muon([good, sparse], weight_decay=0.1)
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    opt = training.Muon([good], weight_decay=0.1)
    with pytest.raises(RuntimeError, match="device"):
        opt.step()
    assert not opt.state and bool((good == 1).all())
    matrices, others = training.matrix_parameters(torch.nn.ParameterList([good, param(3, 0), param(0, 3), param(2, 0, 3), param(5)]))
    assert len(matrices) == 1 and len(others) == 4


@pytest.mark.parametrize("n,cin,cout", [(1_000_000, 8192, 8192), (1_000_000, 16384, 4096), (10_000_000, 64, 64), (300_000, 4096, 4096), ((1 << 31) - 1, 8, 8)])
def test_linear_act_workspace_stays_near_the_input(n, cin, cout):
    """parts of the weight gradient: no more than the rows of x and dz, or two workgroups' worth of every compute unit; dz; parts of the bias"""
    lib = _lib.load()
    tiles = -(-cout // 128) * -(-cin // (128 if cin > 64 else 64))
    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        parts = max(4 * n * (cin + cout), -(-512 // tiles) * cin * cout * 4) + 33 * cin * cout * 4
        dz = n * -(-cout // 8) * 8 * size
        bias = (max(n // 128 + 1, 512, n // 131072 + 1) + 32) * cout * 4
        assert lib.pp_linear_act_bwd_workspace(dtype, n, cin, cout, 3) <= parts + dz + bias + 4096


def test_matrix_parameters_are_what_muon_takes():
    def param(*shape):
        return torch.nn.Parameter(torch.empty(shape, device="meta"))
    model = torch.nn.ParameterList([param(8192, 9000), param(9000, 8193), param(27, 400, 8193), param(27, 64, 96), param(2, 2), param(1, 7), param(6)])
    matrices, others = training.matrix_parameters(model)
    assert [tuple(p.shape) for p in matrices] == [(8192, 9000), (27, 64, 96), (2, 2)] and len(others) == 4
    training.Muon(matrices)
