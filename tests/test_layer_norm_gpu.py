"""layer_norm on the GPU against its formulas in float64, and the scan and the norm together as a block runs them.

Bounds (u = 2^-24): a float32 sum of n terms in any order is off by at most n u times the sum of their absolute values; here a lane adds
at most dim / 32 terms before lanes are joined, so S = dim / 32 + 16 covers a row's sums, and the number of rows those over the rows.  From
there the errors are carried through the formulas term by term; the sigmoid is off by 16 units (float32) or, with the fast
exponential of 16-bit inputs, by 64 (see gated_reference).
"""
import pytest
import torch

import cs2d
import gated_reference as R
from conftest import check_close

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def expected(x, weight, bias, gate, dy, eps=1e-5):
    """{name: (value, tolerance)} for rows (rows, dim); everything on the CPU in float64."""
    dtype, D = x.dtype, x.shape[-1]
    wdtype = weight.dtype if weight is not None else F32
    f = lambda t, none=None: none if t is None else t.detach().double().cpu()
    x, dy, w, b, z = f(x), f(dy), f(weight, torch.ones(D, dtype=torch.float64)), f(bias, torch.zeros(D, dtype=torch.float64)), f(gate)
    S, ks = (D / 32 + 16) * U, R.K[dtype] * U
    mean = lambda t: t.mean(-1, keepdim=True)
    mu = mean(x)
    m = x - mu
    em = S * mean(x.abs()) + U * mu.abs() + U * m.abs()
    v = mean(m * m)
    rstd = (v + eps).rsqrt()
    er = 0.55 * (mean(2 * m.abs() * em + em * em) + (S + 2 * U) * v) / (v + eps) + 4 * U
    xh = m * rstd
    eh = em * rstd + xh.abs() * (er + 2 * U)
    n = xh * w + b
    en = w.abs() * eh + 2 * U * ((xh * w).abs() + b.abs())
    sg = torch.sigmoid(z) if z is not None else None
    s = z * sg if z is not None else torch.ones_like(x)
    kd = ks + 2 * U
    val = {"y": n * s}
    tol = {"y": en * s.abs() + (n * s).abs() * kd}
    dn = dy * s
    t = dn * w
    m1, m2 = mean(t), mean(t * xh)
    e1 = (S + kd + U) * mean(t.abs())
    e2 = (S + kd + 3 * U) * mean((t * xh).abs()) + mean(t.abs() * eh)
    dx = rstd * (t - m1 - xh * m2)
    val["dx"] = dx
    tol["dx"] = rstd * ((kd + U) * t.abs() + e1 + xh.abs() * e2 + eh * m2.abs() + 4 * U * (t.abs() + m1.abs() + (xh * m2).abs())) * (1 + er) + dx.abs() * (er + 2 * U)
    rows = x.shape[0]
    val["dweight"], val["dbias"] = (dn * xh).sum(0), dn.sum(0)
    tol["dweight"] = (dn.abs() * eh + (rows * U + kd + 2 * U) * (dn * xh).abs()).sum(0)
    tol["dbias"] = (rows * U + kd) * dn.abs().sum(0)
    if z is not None:
        slope, sl = sg + s * (1 - sg), sg + (s * (1 - sg)).abs()
        val["dgate"] = dy * n * slope
        tol["dgate"] = dy.abs() * (en * slope.abs() + n.abs() * (2 * ks + 4 * U) * sl) + (dy * n).abs() * sl * 4 * U
    out = {}
    for k in val:
        ty = wdtype if k in ("dweight", "dbias") else dtype
        r = 0.0 if ty == F32 else R.half_step(ty)
        tiny = 1e-38 if ty == F32 else torch.finfo(ty).smallest_normal * torch.finfo(ty).eps / 2
        out[k] = (val[k], tol[k] * (1 + r) + r * val[k].abs() + tiny)
    return out


def inputs(lead, dim, dtype, gated=True, wdtype=F32, seed=0, image=False):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen)
    x = n(*lead, dim) * (0.5 + torch.rand(dim, generator=gen)) + 2 * n(dim)
    x = x.to(dtype).cuda()
    if image:
        x = x.movedim(-1, 1).contiguous().movedim(1, -1)
    return {"x": x, "weight": (1 + 0.2 * n(dim)).to(wdtype).cuda(), "bias": (0.3 * n(dim)).to(wdtype).cuda(),
            "gate": (3 * n(*lead, dim)).to(dtype).cuda() if gated else None, "dy": n(*lead, dim).to(dtype).cuda()}


def run(d, eps=1e-5):
    got = step(d, eps)
    with torch.no_grad():
        y = cs2d.layer_norm(*[d[k] for k in ("x", "weight", "bias", "gate")], eps)
    assert torch.allclose(got["y"], y, rtol=0, atol=0, equal_nan=True) and y.is_contiguous()     # with and without statistics to keep
    return got


def step(d, eps=1e-5):
    names = [k for k in ("x", "weight", "bias", "gate") if d[k] is not None]
    leaves = {k: d[k].detach().requires_grad_(True) for k in names}
    args = [leaves.get(k) for k in ("x", "weight", "bias", "gate")]
    y = cs2d.layer_norm(*args, eps)
    g = torch.autograd.grad(y, [leaves[k] for k in names], d["dy"])
    return {"y": y.detach(), **{"d" + k: t for k, t in zip(names, g)}}


def check(d, got, eps=1e-5):
    rows = lambda t: None if t is None else t.reshape(-1, t.shape[-1])
    want = expected(rows(d["x"]), d["weight"], d["bias"], rows(d["gate"]), rows(d["dy"]), eps)
    for k, v in got.items():
        R.check(k, v if k in ("dweight", "dbias") else rows(v), want[k])


DIMS = (1, 2, 7, 31, 32, 64, 96, 100, 192, 255, 256, 384, 387, 513, 768, 1000, 1024, 1536, 2050, 4096, 9000)


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("dim", DIMS)
def test_widths_of_token_rows(dim, dtype):
    for gated, lead in ((False, (37,)), (True, (3, 11))):
        d = inputs(lead, dim, dtype, gated, seed=dim)
        check(d, run(d))
    assert cs2d.device_status() == 0


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("dim", (1, 3, 31, 32, 51, 64, 96, 192, 200, 384, 387, 768, 1536, 2000, 4096, 9000))
def test_widths_of_images(dim, dtype):
    for gated, lead in ((False, (2, 3, 5)), (True, (2, 6, 8)), (True, (1, 7, 9))):
        d = inputs(lead, dim, dtype, gated, seed=dim, image=True)
        got = run(d)
        assert got["dx"].stride(-1) == lead[1] * lead[2] or dim == 1
        check(d, got)


@pytest.mark.parametrize("rows", (1, 2, 31, 32, 33, 1000, 5000))
@pytest.mark.parametrize("image", (False, True))
def test_numbers_of_rows(rows, image):
    for dim, dtype in ((48, F32), (64, BF16)):
        d = inputs((1, rows) if image else (rows,), dim, dtype, True, seed=rows, image=image)
        check(d, run(d))


@pytest.mark.parametrize("image", (False, True))
@pytest.mark.parametrize("have", ("", "w", "b", "z", "wz", "bz"))
def test_absent_parameters(have, image):
    d = inputs((2, 4, 4), 72, BF16, True, image=image)
    for k, c in (("weight", "w"), ("bias", "b"), ("gate", "z")):
        if c not in have:
            d[k] = None
    check(d, run(d))


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("image", (False, True))
def test_parameters_in_the_type_of_x(dtype, image):
    d = inputs((2, 5, 9), 136, dtype, True, wdtype=dtype, image=image)
    check(d, run(d))


def test_strides():
    B, H, W, D = 2, 5, 6, 40
    d = inputs((B, H, W), 3 * D + 1, BF16)
    views = {"halves": lambda t: t[..., D:2 * D], "odd start": lambda t: t[..., 1:D + 1], "columns left out": lambda t: t[:, :, :4, :D],
             "channels apart": lambda t: t[..., :2 * D:2], "expanded": lambda t: t[:, :1, :, :D].expand(B, H, W, D), "two axes": lambda t: t[0, 0, :, :D],
             "one axis": lambda t: t[0, 0, 0, :D], "five axes": lambda t: t[..., :D].reshape(B, H, 2, 3, D),
             "an image's first rows": lambda t: t[..., :D].permute(0, 3, 1, 2).contiguous()[:, :, :3].permute(0, 2, 3, 1),
             "an image's columns": lambda t: t[..., :D].permute(0, 3, 1, 2).contiguous()[..., 1:].permute(0, 2, 3, 1),
             "channels of an image": lambda t: t.permute(0, 3, 1, 2).contiguous()[:, 3:3 + D].permute(0, 2, 3, 1),
             "one image": lambda t: t[0, :, :, :D].permute(2, 0, 1).contiguous().permute(1, 2, 0),
             "a matrix's columns": lambda t: t[0, 0, :, :D].t().contiguous().t()}
    for name, view in views.items():
        e = {k: view(d[k]) for k in ("x", "gate", "dy")}
        e["weight"], e["bias"] = d["weight"][:D], d["bias"][1:D + 1]
        got = run(e)
        check(e, got)
        for k, v in run({k: v.contiguous() for k, v in e.items()}).items():
            if k == "y" or got["dx"].stride() == v.stride():
                check_close(f"{name} {k}", got[k].float().cpu(), v.float().cpu(), R.half_step(BF16) * 4, 1e-3)


def test_rows_that_vary_little_or_not_at_all():
    for image in (False, True):
        d = inputs((4, 8), 96, F32, True, image=image)
        d["x"] = d["x"] * 1e-3 + 100.0                            # the variance of the centred values
        check(d, run(d))
        d["x"] = torch.full_like(d["x"], 3.0)
        got = run(d)
        assert torch.isfinite(got["dx"]).all()
        want = d["bias"] * torch.nn.functional.silu(d["gate"])
        check_close("y", got["y"].cpu(), want.cpu(), 1e-5, 1e-6)


def test_values_far_out():
    d = inputs((3, 9), 64, F32, True)
    d["gate"][0] = 200.0
    d["gate"][1] = -200.0
    got = run(d)
    check(d, got)
    d["x"][2, 4, 5] = float("nan")
    d["x"][1, 2, 3] = float("inf")
    got = run(d)
    for r in ((2, 4), (1, 2)):
        assert torch.isnan(got["y"][r]).all() and torch.isnan(got["dx"][r]).all()
    ok = torch.ones(3, 9, dtype=torch.bool)
    ok[2, 4] = ok[1, 2] = False
    assert torch.isfinite(got["y"].cpu()[ok]).all() and torch.isfinite(got["dx"].cpu()[ok]).all()


def test_empty_and_refusals():
    w = torch.ones(8, device="cuda", requires_grad=True)
    y = cs2d.layer_norm(torch.zeros(0, 8, device="cuda"), w)
    assert y.shape == (0, 8) and not torch.autograd.grad(y.sum(), w)[0].any()
    x = torch.zeros(4, 8, device="cuda")
    for args, msg in [((x.double(),), "input type"), ((x, w[:4]), "shape"), ((x, w.half()), "float32"), ((x, w.cpu()), "device"), ((x, None, w.half()), "float32"),
                      ((x.half(), w, w.half()), "one dtype"), ((x, None, None, x.half()), "dtype of x"), ((x, None, None, x[:2]), "shape of x"),
                      ((x, None, None, None, -1.0), "eps"), ((x[:, :0],), "channel")]:
        with pytest.raises(RuntimeError, match=msg):
            cs2d.layer_norm(*args)
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(cs2d.layer_norm(x).sum(), x, create_graph=True)


def test_first_calls_of_a_process_inside_a_capture():
    """Nothing has been launched before: the recorded step prepares its kernels itself."""
    import subprocess
    import sys
    from conftest import ROOT
    code = """
import sys, torch
sys.path.insert(0, "official-cross-scan_b200")
import cs2d
u, g, z = (torch.randn(1, 700, 64, device="cuda") for _ in range(3))
w = torch.ones(64, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    a = [t.requires_grad_(True) for t in (u, g, z, w)]
    y = cs2d.layer_norm(cs2d.gated_scan_1d(a[0], a[1])[0], a[3], None, a[2])
    grads = torch.autograd.grad(y, a, torch.ones_like(y))
graph.replay()
torch.cuda.synchronize()
kept = [t.clone() for t in (y, *grads)]
y = cs2d.layer_norm(cs2d.gated_scan_1d(a[0], a[1])[0], a[3], None, a[2])
print(all(torch.equal(p, q) for p, q in zip(kept, (y, *torch.autograd.grad(y, a, torch.ones_like(y))))))
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["True"], r.stdout + r.stderr


def test_same_bits_every_time_on_other_streams_and_from_a_graph():
    for image in (False, True):
        d = inputs((4, 30, 31), 192, BF16, image=image)
        first = run(d)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = run(d)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = cs2d.layer_norm(*[d[k] for k in ("x", "weight", "bias", "gate")])
            kept = step(d)
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, first["y"])
        for k in first:
            assert torch.equal(first[k], again[k]) and torch.equal(first[k], kept[k]), k


def test_gradient_against_differences():
    """As for the scan: rounding 2 |f| 30 u / 2e, truncation below e^2 |f| for inputs and directions of order one."""
    d = inputs((7, 5), 48, F32)
    d["x"] = d["x"] / d["x"].std()
    got = run(d)
    names = ("x", "weight", "bias", "gate")
    f = lambda *a: (cs2d.layer_norm(*a).double() * d["dy"].double()).sum()
    size = (got["y"].double() * d["dy"].double()).abs().sum()
    gen, e = torch.Generator().manual_seed(2), 2.0 ** -7
    for k, name in enumerate(names):
        v = torch.randn(d[name].shape, generator=gen).cuda()
        v /= v.abs().max()
        lo, hi = [[d[n] if n != name else d[n] + s * e * v for n in names] for s in (-1, 1)]
        slope = (f(*hi) - f(*lo)) / (2 * e)
        want = (got["d" + name].double() * v.double()).sum()
        assert abs(slope - want) < size * (30 * U / e + e * e), name


def test_scan_and_norm_as_a_block_runs_them():
    """Gates and values from one projection, the scan of packed sequences, the gated norm, a projection back: against the same in float64."""
    gen = torch.Generator().manual_seed(0)
    dim, lengths = 24, [30, 0, 1, 97]
    off = torch.tensor([0, 30, 30, 31, 128], dtype=torch.int32)
    n = lambda *s: torch.randn(*s, generator=gen)
    par = {"win": 0.3 * n(3 * dim, 16), "w": 1 + 0.1 * n(dim), "b": 0.1 * n(dim), "wout": 0.3 * n(16, dim), "h0": n(4, dim)}
    x, dy = n(128, 16), n(128, 16)

    def block(scan, norm, x, p):
        u, g, z = (x @ p["win"].t()).split(dim, -1)
        y, last = scan(u, g + 1, p["h0"])
        return norm(y, p["w"], p["b"], z) @ p["wout"].t(), last

    dev = {k: v.cuda().requires_grad_(True) for k, v in par.items()}
    xd = x.cuda().requires_grad_(True)
    y, last = block(lambda u, g, h: cs2d.gated_scan_1d(u, g, h, off.cuda()), cs2d.layer_norm, xd, dev)
    got = torch.autograd.grad([y, last], [xd, *dev.values()], [dy.cuda(), torch.ones_like(last)])

    def scan64(u, g, h):
        parts = [R.scan(u[a:b], g[a:b], h[i], "sigmoid", True) for i, (a, b) in enumerate(zip(off[:-1], off[1:]))]
        return torch.cat([p[0] for p in parts]), torch.stack([p[1] for p in parts])

    ref = {k: v.double().requires_grad_(True) for k, v in par.items()}
    xr = x.double().requires_grad_(True)
    norm64 = lambda y, w, b, z: torch.nn.functional.layer_norm(y, (dim,), w, b) * torch.nn.functional.silu(z)
    y64, last64 = block(scan64, norm64, xr, ref)
    want = torch.autograd.grad([y64, last64], [xr, *ref.values()], [dy.double(), torch.ones_like(last64)])
    # float32 through two small products, a scan with a memory of a few tokens and a norm: a block-level tolerance
    check_close("y", y.detach().cpu(), y64.detach(), 1e-3, 1e-4)
    for name, a, b in zip(("x", *par), got, want):
        check_close("d" + name, a.cpu(), b, 1e-3, 1e-3)
    assert cs2d.device_status() == 0


@pytest.mark.parametrize("dtype", (F32, BF16))
def test_ss2d_with_the_fused_norm(dtype):
    """The block with its norm and gate in one operator: the same step as with the three, to the roundings between them."""
    import copy
    from cs2d.nn import SS2D
    torch.manual_seed(5)
    m = SS2D(d_model=16, d_state=4).cuda()
    f = SS2D(d_model=16, d_state=4, fused_norm=True).cuda()
    f.load_state_dict(m.state_dict())
    x = torch.randn(2, 8, 12, 16, device="cuda")
    dy = torch.randn(2, 8, 12, 16, device="cuda")
    if dtype == BF16:      # projections and norm in 16 bits, the scan's parameters in 32 as everywhere
        for b in (m, f):
            for p in (b.in_proj, b.conv2d, b.x_proj, b.out_norm, b.out_proj):
                p.to(BF16)
        x, dy = x.to(BF16), dy.to(BF16)
    outs = []
    for b in (m, f):
        xl = x.clone().requires_grad_(True)
        y = b(xl)
        outs.append((y, *torch.autograd.grad(y, [xl, *b.parameters()], dy)))
    # fp32: a block-level tolerance; bf16: the three operators round the norm and the gate's value on the way, half a step each
    tol = 1e-4 if dtype == F32 else 12 * R.half_step(BF16)
    for name, a, c in zip(("y", "x", *dict(m.named_parameters())), *outs):
        scale = float(a.float().abs().max())
        check_close(name, c.detach().float().cpu(), a.detach().float().cpu(), tol, tol * max(scale, 1e-3))
    assert cs2d.device_status() == 0
