"""Cases of three operators that train and serve blocks which do not depend on the batch: group normalisation with an activation
over the rows of each batch element, a linear layer whose epilogue adds the bias, the activation and a residual, and the
orthogonalisation of a weight's update by Newton-Schulz products.  `run` computes them in elementary torch operations, or, where
`own` is true, through the package's entry points."""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NORM_EPS = 1e-5
LEAK = 0.2
NS_EPS = 1e-7


def _norm(name, dtype, batch, rows, channels, groups, activation, train, ragged=False, shuffled=False):
    return {"name": name, "op": "group_norm", "dtype": dtype, "batch": batch, "rows": rows, "channels": channels, "groups": groups,
            "activation": activation, "train": train, "ragged": ragged, "shuffled": shuffled}


def _linear(name, dtype, rows, cin, cout, activation, residual, train):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "cin": cin, "cout": cout, "activation": activation,
            "residual": residual, "train": train}


def _orthogonal(name, dtype, batch, m, n):
    return {"name": name, "op": "newton_schulz", "dtype": dtype, "batch": batch, "m": m, "n": n}


def listed():
    return [
        # the deepest level of one cylinder when a single tile is served: a call that is all latency
        _norm("norm_coarse_level", "float32", 1, 1021, 112, 8, "relu", False),
        # four training cylinders at the second level of the backbone; the level's rows are in the order of its kernel map
        _norm("norm_train_backbone", "float32", 4, 325_000, 32, 8, "silu", True, shuffled=True),
        # the scorer's batch: one batch element per proposal, most of them short, some without rows
        _norm("norm_train_proposals", "bfloat16", 1500, 180_003, 64, 16, "silu", True, ragged=True),
        # a scene of 64 cylinders served as one batch
        _norm("norm_scene", "bfloat16", 64, 2_500_000, 96, 32, "gelu", False),
        # the squeeze layer of a squeeze-and-excite block: one row per batch element
        _linear("linear_squeeze", "float32", 64, 112, 7, "relu", False, False),
        # a pointwise residual layer over the voxels of a scene
        _linear("linear_scene_rows", "bfloat16", 1_250_000, 64, 64, "gelu", True, False),
        # a hidden layer over the voxels of four training cylinders
        _linear("linear_train_rows", "float32", 325_000, 96, 96, "gelu", False, True),
        # a hidden layer of a wide block
        _linear("linear_train_wide", "bfloat16", 8192, 1024, 4096, "silu", False, True),
        # sizes that fit no tile
        _linear("linear_train_odd", "float16", 50_021, 75, 133, "silu", True, True),
        # the kernels [27, 64, 64] of the levels with 64 channels, flattened to [27 * 64, 64]
        _orthogonal("orthogonal_level4", "float32", 8, 1728, 64),
        # the first decoder kernels [27, 192, 96]
        _orthogonal("orthogonal_decoder", "float32", 3, 5184, 96),
        # the two matrices of a wide block
        _orthogonal("orthogonal_wide", "bfloat16", 2, 1024, 4096),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        op = rng.choice(("group_norm", "linear", "newton_schulz"))
        dtype = rng.choice(tuple(DTYPES))
        if op == "group_norm":
            groups = rng.choice((1, 2, 4, 8, 16, 32))
            case = _norm("", dtype, _log(rng, 1, 2000), _log(rng, 500, 2_500_000), groups * max(1, _log(rng, 16, 256) // groups), groups,
                         rng.choice(("none", "relu", "leaky_relu", "silu", "gelu")), rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.3)
        elif op == "linear":
            case = _linear("", dtype, _log(rng, 1, 1_250_000), _log(rng, 4, 1024), _log(rng, 4, 4096),
                           rng.choice(("none", "relu", "leaky_relu", "silu", "gelu")), rng.random() < 0.5, rng.random() < 0.5)
        else:
            case = _orthogonal("", dtype, _log(rng, 1, 16), _log(rng, 16, 6000), _log(rng, 16, 4096))
        del case["name"]
        if dtype == "float32" and case.get("train") and "relu" in case["activation"]:
            continue  # the slope jumps at 0: which side a 32-bit sum next to it falls on is no property of the operator
        w = work(case)
        small = min(case.get("m", 0), case.get("n", 0)) <= 1024
        if small and w["bytes"] <= 0.9e9 and w["flops"] <= 1.9e11:
            return case


def _offsets(case, gen):
    """first row of every batch element: [batch + 1], the last entry is the number of rows"""
    if case["ragged"]:
        share = torch.exp(1.5 * torch.randn(case["batch"], generator=gen))
        share[torch.rand(case["batch"], generator=gen) < 0.05] = 0.0
        share[0] += 1.0
    else:
        share = 0.5 + torch.rand(case["batch"], generator=gen)
    ends = torch.round(torch.cumsum(share.double(), 0) / share.double().sum() * case["rows"]).long()
    ends[-1] = case["rows"]
    return torch.cat([torch.zeros(1, dtype=torch.int64), ends])


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    gpu = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gpu, device="cuda")

    state = {"case": dict(case)}
    if case["op"] == "newton_schulz":
        # an update as it is met in training: a few strong directions over a floor of noise, scales that differ by batch element
        b, m, n = case["batch"], case["m"], case["n"]
        k = max(1, min(m, n) // 8)
        strong = torch.bmm(normal(b, m, k) / (1.0 + torch.arange(k, device="cuda")), normal(b, k, n))
        state["g"] = ((strong / math.sqrt(k) + normal(b, m, n)) * 1e-3 * (1.0 + torch.rand((b, 1, 1), generator=gpu, device="cuda"))).to(dtype)
        return state
    train = case["train"]
    if case["op"] == "group_norm":
        n, c = case["rows"], case["channels"]
        state["offsets"] = _offsets(case, gen).cuda()
        # a level's rows are nearly sorted by batch element: blocks of 8192 rows are in an order of their own
        state["order"] = None
        if case["shuffled"]:
            key = torch.arange(n, device="cuda") // 8192 + torch.rand(n, generator=gpu, device="cuda", dtype=torch.float64)
            state["order"] = torch.argsort(torch.argsort(key) // 8192 * 8192 + torch.rand(n, generator=gpu, device="cuda", dtype=torch.float64) * 8192)
        state["x"] = (normal(n, c) * (0.5 + torch.rand(c, generator=gpu, device="cuda")) + normal(c)).to(dtype).requires_grad_(train)
        state["weight"] = (1.0 + 0.2 * normal(c)).requires_grad_(train)
        state["bias"] = (0.2 * normal(c)).requires_grad_(train)
        state["dy"] = normal(n, c).to(dtype) if train else None
        return state
    n, cin, cout = case["rows"], case["cin"], case["cout"]
    state["x"] = normal(n, cin).to(dtype).requires_grad_(train)
    state["weight"] = (normal(cout, cin) / math.sqrt(cin)).to(dtype).requires_grad_(train)
    state["bias"] = (0.2 * normal(cout)).to(dtype).requires_grad_(train)
    state["residual"] = normal(n, cout).to(dtype).requires_grad_(train) if case["residual"] else None
    state["dy"] = (0.1 * normal(n, cout)).to(dtype) if train else None
    return state


def _activation(z, kind):
    if kind == "relu":
        return torch.clamp(z, min=0.0)
    if kind == "leaky_relu":
        return torch.where(z > 0, z, LEAK * z)
    if kind == "silu":
        return z / (1.0 + torch.exp(-z))
    if kind == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _slope(z, kind):
    """derivative of the activation"""
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "leaky_relu":
        return torch.where(z > 0, 1.0, LEAK)
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if kind == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    return torch.ones_like(z)


def _plain_norm(s):
    case, x = s["case"], s["x"]
    n, c, g = case["rows"], case["channels"], case["groups"]
    off = s["offsets"]
    counts = off[1:] - off[:-1]
    ids = torch.repeat_interleave(torch.arange(case["batch"], device=x.device), counts, output_size=n)
    if s["order"] is not None:
        ids = torch.empty_like(ids).index_copy_(0, s["order"], ids)
    m = (counts.clamp(min=1) * (c // g)).double()[:, None]

    def per_group(v):  # means over the rows of a batch element and the channels of a group: differences of running sums, in 64 bits
        v = v.view(n, g, c // g).sum(2, dtype=torch.float64)
        v = v if s["order"] is None else v[s["order"]]
        run = torch.cat([torch.zeros((g, 1), dtype=torch.float64, device=x.device), torch.cumsum(v.t().contiguous(), 1)], 1)
        return (run[:, off[1:]] - run[:, off[:-1]]).t() / m

    mean = per_group(x.float()).float()
    centred = x.float().view(n, g, c // g) - mean[ids][:, :, None]
    rstd = (1.0 / torch.sqrt(per_group((centred * centred).view(n, c)) + NORM_EPS)).float()
    hat = (centred * rstd[ids][:, :, None]).view(n, c)
    z = hat * s["weight"] + s["bias"]
    y = _activation(z, case["activation"]).to(x.dtype)
    if not case["train"]:
        return [y]
    dz = s["dy"].float() * _slope(z, case["activation"])
    dbias = dz.sum(0, dtype=torch.float64).float()
    dweight = (dz * hat).sum(0, dtype=torch.float64).float()
    dhat = dz * s["weight"]
    a, b = per_group(dhat).float(), per_group(dhat * hat).float()
    dx = rstd[ids][:, :, None] * (dhat.view(n, g, -1) - a[ids][:, :, None] - hat.view(n, g, -1) * b[ids][:, :, None])
    return [y, dx.view(n, c).to(x.dtype), dweight, dbias]


def _weight_gradient(dz, x, dtype):
    """dz^T x; for 32-bit outputs the long sum over the rows is taken in parts of 2048 rows, which are added in 64 bits"""
    k = dz.shape[0] // 2048
    if dtype != torch.float32 or k < 2:
        return torch.mm(dz.t(), x)
    n = 2048 * k
    parts = torch.bmm(dz[:n].view(k, 2048, -1).transpose(1, 2).contiguous(), x[:n].view(k, 2048, -1))
    return parts.sum(0, dtype=torch.float64) + torch.mm(dz[n:].t(), x[n:])


def _plain_linear(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = torch.mm(x, w.t()) + s["bias"].float()
    y = _activation(z, case["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    y = y.to(dtype)
    if not case["train"]:
        return [y]
    dz = s["dy"].float() * _slope(z, case["activation"])
    grads = [torch.mm(dz, w), _weight_gradient(dz, x, dtype), dz.sum(0)] + ([s["dy"]] if s["residual"] is not None else [])
    return [y] + [v.to(dtype) for v in grads]


def _plain_newton_schulz(s):
    a, b, c = COEFFICIENTS
    g = s["g"].float()
    x = g / (torch.sqrt((g * g).sum((1, 2), keepdim=True)) + NS_EPS)
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2).contiguous() if tall else x
    for _ in range(5):
        p = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * p + c * torch.bmm(p, p), x)
    return [(x.transpose(1, 2).contiguous() if tall else x).to(s["g"].dtype)]


def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return {"group_norm": _plain_norm, "linear": _plain_linear, "newton_schulz": _plain_newton_schulz}[case["op"]](state)
    from panopticsegforlargescalepointcloud_amd import modules, ops
    if case["op"] == "newton_schulz":
        return [ops.newton_schulz(state["g"], steps=5, coefficients=COEFFICIENTS, eps=NS_EPS)]
    if case["op"] == "group_norm":
        y = modules.group_norm_act(state["x"], state["offsets"], case["groups"], state["weight"], state["bias"], eps=NORM_EPS,
                                   activation=case["activation"], slope=LEAK, order=state["order"])
        leaves = [state["x"], state["weight"], state["bias"]]
    else:
        y = modules.linear_act(state["x"], state["weight"], state["bias"], activation=case["activation"], slope=LEAK,
                               residual=state["residual"])
        leaves = [state["x"], state["weight"], state["bias"]] + ([] if state["residual"] is None else [state["residual"]])
    return [y.detach()] + (list(torch.autograd.grad(y, leaves, state["dy"])) if case["train"] else [])


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "newton_schulz":
        # the Gram matrix of the short side once, its polynomials on the short side, their product with the matrix once
        small, large = min(case["m"], case["n"]), max(case["m"], case["n"])
        return {"bytes": 2.0 * case["batch"] * small * large * size,
                "flops": case["batch"] * min(3.0 * small * small * large + 20.0 * small ** 3, 15.0 * small * small * large + 5.0 * small ** 3)}
    both = 2.0 if case["train"] else 1.0
    if case["op"] == "group_norm":
        n = case["rows"] * case["channels"]
        return {"bytes": both * 2.0 * n * size + (8.0 * case["rows"] if case["shuffled"] else 0.0), "flops": both * 10.0 * n}
    n, cin, cout = case["rows"], case["cin"], case["cout"]
    read = n * cin + cin * cout + cout + (n * cout if case["residual"] else 0)
    more = (n * cout + n * cin + cin * cout + cout) if case["train"] else 0
    return {"bytes": float(size) * (read + n * cout + more), "flops": (6.0 if case["train"] else 2.0) * n * cin * cout}


def exact(case, seed):
    """the definitions in 64 bits; gradients by automatic differentiation of the definition"""
    s = prepare(case, seed)
    if case["op"] == "newton_schulz":
        if case["batch"] * min(case["m"], case["n"]) ** 2 * max(case["m"], case["n"]) > 1e11:
            return None
        a, b, c = COEFFICIENTS
        out = []
        for g in s["g"]:
            x = g.double()
            x = x / (torch.linalg.vector_norm(x) + NS_EPS)
            for _ in range(5):
                eye = torch.eye(min(x.shape), dtype=torch.float64, device=x.device)
                if x.shape[0] <= x.shape[1]:
                    p = x @ x.mT
                    x = (a * eye + p @ (b * eye + c * p)) @ x
                else:
                    p = x.mT @ x
                    x = x @ (a * eye + p @ (b * eye + c * p))
            out.append(x)
        return [torch.stack(out)]
    x = s["x"].detach().double().requires_grad_(case["train"])
    w = s["weight"].detach().double().requires_grad_(case["train"])
    bias = s["bias"].detach().double().requires_grad_(case["train"])

    def act(z):
        kind = case["activation"]
        if kind == "relu":
            return z.relu()
        if kind == "leaky_relu":
            return torch.nn.functional.leaky_relu(z, LEAK)
        if kind == "silu":
            return z * torch.sigmoid(z)
        if kind == "gelu":
            return z * (0.5 * torch.erfc(-z / math.sqrt(2.0)))
        return z

    leaves = [x, w, bias]
    if case["op"] == "linear":
        y = act(torch.addmm(bias, x, w.mT))
        if s["residual"] is not None:
            leaves.append(s["residual"].detach().double().requires_grad_(case["train"]))
            y = y + leaves[-1]
    else:
        bounds, g = s["offsets"].tolist(), case["groups"]
        rows = x if s["order"] is None else x[s["order"]]
        parts = []
        for lo, hi in zip(bounds[:-1], bounds[1:]):
            if hi > lo:
                v = rows[lo:hi].reshape(hi - lo, g, -1)
                var, mean = torch.var_mean(v, dim=(0, 2), keepdim=True, correction=0)
                parts.append(((v - mean) * torch.rsqrt(var + NORM_EPS)).reshape(hi - lo, -1))
        y = act(torch.cat(parts) * w + bias)
        if s["order"] is not None:
            y = torch.empty_like(y).index_copy(0, s["order"], y)
    if not case["train"]:
        return [y]
    return [y.detach()] + list(torch.autograd.grad(y, leaves, s["dy"].double()))
