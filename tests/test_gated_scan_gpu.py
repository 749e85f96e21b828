"""gated_scan_1d and gated_scan_step on the GPU against the token-by-token definition in float64."""
import subprocess
import sys
import textwrap

import pytest
import torch

import cs2d
import gated_reference as R
from conftest import ROOT

pytestmark = pytest.mark.gpu
FORMS = ("sigmoid", "log", "direct")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def inputs(shape, states, dtype, form, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen)
    gate = 2 + 2 * n(*shape) if form == "sigmoid" else -torch.exp(n(*shape) - 2)
    if form == "direct":
        gate = gate.exp() * (1 - 2 * (torch.rand(*shape, generator=gen) < 0.2).float())     # of either sign
    d = {"u": n(*shape) * scale, "gate": gate.clamp(-8, 8), "dy": n(*shape)}
    d = {k: v.to(dtype).cuda() for k, v in d.items()}
    d["h0"], d["dlast"] = n(states, shape[-1]).cuda(), n(states, shape[-1]).cuda()
    return d


def run(d, form, weighted, h0=True, dlast=True, offsets=None):
    leaves = [d["u"], d["gate"]] + ([d["h0"]] if h0 else [])
    leaves = [t.detach().requires_grad_(True) for t in leaves]
    y, last = cs2d.gated_scan_1d(leaves[0], leaves[1], leaves[2] if h0 else None, offsets, form=form, weighted=weighted)
    outs, gos = ([y, last], [d["dy"], d["dlast"]]) if dlast else ([y], [d["dy"]])
    g = torch.autograd.grad(outs, leaves, gos)
    with torch.no_grad():
        y2, last2 = cs2d.gated_scan_1d(d["u"], d["gate"], d["h0"] if h0 else None, offsets, form=form, weighted=weighted)
    assert torch.equal(y, y2) and torch.equal(last, last2)       # with and without a state to keep
    return dict(zip(("y", "h_last", "du", "dgate", "dh0"), (y, last, *g)))


def check_dense(d, got, form, weighted, h0=True, dlast=True):
    for b in range(d["u"].shape[0]):
        want = R.expected(d["u"][b], d["gate"][b], d["h0"][b] if h0 else None, d["dy"][b], d["dlast"][b] if dlast else None, form, weighted,
                          d["u"].dtype)
        for k, v in got.items():
            R.check(f"{k}[{b}]", v[b], want[k])


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 1, 7), (3, 8, 64), (2, 9, 2), (33, 16, 31), (2, 17, 66), (1, 64, 192), (5, 100, 32),
                                   (2, 128, 33), (1, 129, 130), (2, 256, 64), (1, 257, 97), (2, 1037, 51), (1, 2500, 96)])
def test_sizes(shape, dtype):
    form = FORMS[(shape[1] + shape[2]) % 3]
    for weighted in (True, False):
        d = inputs(shape, shape[0], dtype, form, seed=shape[1])
        check_dense(d, run(d, form, weighted), form, weighted)
    assert cs2d.device_status() == 0


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("weighted", (True, False))
@pytest.mark.parametrize("form", FORMS)
def test_forms_without_states(form, weighted, dtype):
    d = inputs((2, 300, 70), 2, dtype, form, seed=5)
    check_dense(d, run(d, form, weighted, h0=False, dlast=False), form, weighted, h0=False, dlast=False)


# lengths of many tiles: few channels (one or more CTAs of a cluster along the rows), many channels
@pytest.mark.parametrize("shape", [(1, 9001, 8), (1, 6000, 64), (4, 4100, 130)])
@pytest.mark.parametrize("dtype", (F32, BF16))
def test_long(shape, dtype):
    d = inputs(shape, shape[0], dtype, "sigmoid", seed=2)
    check_dense(d, run(d, "sigmoid", True), "sigmoid", True)


def packed(lengths, dim, dtype, form, before=0, behind=0, seed=3, garbage=float("nan")):
    total = before + sum(lengths) + behind
    d = inputs((total, dim), len(lengths), dtype, form, seed=seed)
    off = [before]
    for n in lengths:
        off.append(off[-1] + n)
    for k in ("u", "gate", "dy"):
        d[k][:off[0]] = garbage
        d[k][off[-1]:] = garbage
    return d, off


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("lengths,before,behind", [([1], 0, 0), ([0, 0, 5, 0], 0, 0), ([3, 1, 0, 1, 1, 7, 16, 15, 17], 0, 3), ([40, 0, 260, 1, 128], 5, 20),
                                                   ([700, 0, 0, 1, 299, 1800], 0, 129), ([2, 2, 2], 300, 300), ([1] * 70, 0, 0), ([0, 0], 0, 4), ([], 0, 6)])
def test_packed(lengths, before, behind, dtype):
    form = FORMS[len(lengths) % 3]
    for h0, garbage, kind in ((True, float("nan"), torch.int32), (False, float("inf"), torch.int64)):
        d, off = packed(lengths, 65 if dtype == F32 else 66, dtype, form, before, behind, garbage=garbage)
        got = run(d, form, True, h0=h0, offsets=torch.tensor(off, dtype=kind, device="cuda"))
        for k in ("y", "du", "dgate"):
            assert not got[k][:off[0]].any() and not got[k][off[-1]:].any(), k
        for s in range(len(lengths)):
            r = slice(off[s], off[s + 1])
            want = R.expected(d["u"][r], d["gate"][r], d["h0"][s] if h0 else None, d["dy"][r], d["dlast"][s], form, True, dtype)
            for k, v in got.items():
                R.check(f"{k} of sequence {s}", v[r] if k in ("y", "du", "dgate") else v[s], want[k])
    assert cs2d.device_status() == 0


def test_a_sequence_keeps_its_infinities_to_itself():
    d, off = packed([40, 300, 40], 64, F32, "log")
    d["u"][20], d["dy"][20] = float("inf"), float("nan")
    off_t = torch.tensor(off, dtype=torch.int32, device="cuda")
    got = run(d, "log", False, offsets=off_t)
    assert torch.isinf(got["y"][20:40]).all() and torch.isnan(got["du"][:21]).all()
    for s in (1, 2):
        r = slice(off[s], off[s + 1])
        want = R.expected(d["u"][r], d["gate"][r], d["h0"][s], d["dy"][r], d["dlast"][s], "log", False, F32)
        for k, v in got.items():
            R.check(k, v[r] if k in ("y", "du", "dgate") else v[s], want[k])


def test_offsets_that_cannot_be_followed_are_reported():
    d, _ = packed([100], 64, F32, "sigmoid")
    for bad in ([0, 60, 40, 100], [0, 50, 101], [-3, 50, 100]):
        with torch.no_grad():
            y, last = cs2d.gated_scan_1d(d["u"], d["gate"], None, torch.tensor(bad, device="cuda"))
        torch.cuda.synchronize()
        assert cs2d.device_status() == 8 and "offsets" in cs2d._lib.last_error()
        assert y.shape == (100, 64) and last.shape == (len(bad) - 1, 64)
    assert cs2d.device_status() == 0


@pytest.mark.parametrize("dtype", (F32, BF16))
def test_strides(dtype):
    B, L, D = 2, 150, 48
    d = inputs((B, L, 3 * D + 1), B, dtype, "sigmoid", seed=8)
    views = {"halves": lambda t: t[..., D:2 * D], "odd start": lambda t: t[..., 1:D + 1], "odd rows": lambda t: t[:, 1::2, :D],
             "time first": lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)[..., :D],
             "channels outside": lambda t: t[..., :D].transpose(1, 2).contiguous().transpose(1, 2),
             "one for all": lambda t: t[:1, :, :D].expand(B, L, D)}
    for name, view in views.items():
        e = {k: view(d[k]) for k in ("u", "gate", "dy")}
        e["h0"], e["dlast"] = d["h0"][:, :D], d["dlast"][:, 1:D + 1]
        got = run(e, "sigmoid", True)
        check_dense(e, got, "sigmoid", True)
        dense = run({k: v.contiguous() for k, v in e.items()}, "sigmoid", True)
        for k in got:
            assert torch.equal(got[k], dense[k]), (name, k)


def test_extreme_gates():
    u = torch.randn(1, 600, 32, device="cuda")
    for form, keep, drop in (("sigmoid", 200.0, -200.0), ("sigmoid", float("inf"), float("-inf")), ("log", 0.0, float("-inf")), ("direct", 1.0, 0.0)):
        h0 = torch.randn(1, 32, device="cuda")
        y, last = cs2d.gated_scan_1d(u, torch.full_like(u, keep), h0, form=form, weighted=True)
        assert torch.equal(y, h0[:, None].expand_as(y)) and torch.equal(last, h0)          # a = 1: nothing is let in
        y, last = cs2d.gated_scan_1d(u, torch.full_like(u, drop), h0, form=form, weighted=True)
        assert torch.equal(y, u) and torch.equal(last, u[:, -1])                           # a = 0: nothing is kept
    gate = torch.zeros(1, 600, 32, device="cuda")
    gate[0, 300, 5] = float("nan")
    y, last = cs2d.gated_scan_1d(u, gate, None)
    bad = torch.isnan(y)
    assert bad[0, 300:, 5].all() and int(bad.sum()) == 300 and torch.isnan(last[0, 5])
    # factors above one over an empty state: their product overflows, the state does not
    y, _ = cs2d.gated_scan_1d(torch.zeros_like(u), torch.full_like(u, 3.0), None, form="direct", weighted=False)
    assert not y.any()


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("form", FORMS)
def test_prompt_then_tokens(form, dtype):
    """A prompt through the scan, then tokens one by one on rows of a pool of states: as the scan of the whole."""
    B, L, D, n = 3, 40, 37, 20
    d = inputs((B, L, D), B, dtype, form, seed=1)
    with torch.no_grad():
        whole, last = cs2d.gated_scan_1d(d["u"], d["gate"], None, form=form)
        y, h = cs2d.gated_scan_1d(d["u"][:, :n], d["gate"][:, :n], None, form=form)
        pool = torch.full((7, D + 3), 9.0, device="cuda")
        rows = pool[1:1 + B, :D]
        rows.copy_(h)
        ys = [y] + [cs2d.gated_scan_step(d["u"][:, t], d["gate"][:, t], rows, form=form)[:, None] for t in range(n, L)]
    got = torch.cat(ys, 1)
    for b in range(B):
        want = R.expected(d["u"][b], d["gate"][b], None, d["dy"][b], None, form, True, dtype)
        R.check("y", got[b], want["y"])
        R.check("state", rows[b], want["h_last"])
    pool[1:1 + B, :D] = 9.0
    assert (pool == 9.0).all()


def test_empty_calls():
    for shape in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        u = torch.randn(shape, device="cuda", requires_grad=True)
        g = torch.randn(shape, device="cuda", requires_grad=True)
        h0 = torch.randn(shape[0], shape[2], device="cuda", requires_grad=True)
        y, last = cs2d.gated_scan_1d(u, g, h0)
        assert y.shape == shape and torch.equal(last, h0)
        du, dg, dh = torch.autograd.grad([y, last], [u, g, h0], [torch.ones_like(y), torch.full_like(last, 2.0)])
        assert du.shape == shape and dg.shape == shape and torch.equal(dh, torch.full_like(h0, 2.0))
    u = torch.randn(0, 8, device="cuda")
    y, last = cs2d.gated_scan_1d(u, u, torch.ones(2, 8, device="cuda"), torch.tensor([0, 0, 0], device="cuda"))
    assert y.shape == (0, 8) and (last == 1).all()
    assert cs2d.gated_scan_step(u, u, torch.zeros(0, 8, device="cuda")).shape == (0, 8)


def test_gradient_against_differences():
    """Along random directions: (f(x + e v) - f(x - e v)) / 2e.  Rounding: 2 * |f| * 2^-24 * 30 / 2e; truncation: e^2 / 6 times a third
    derivative that is at most the sum of |terms| for gates of order one (the sigmoid's derivatives are below 1/4)."""
    d = inputs((2, 60, 8), 2, F32, "sigmoid", seed=4)
    got = run(d, "sigmoid", True)
    gen = torch.Generator().manual_seed(1)
    f = lambda u, g, h: [t.double() for t in cs2d.gated_scan_1d(u, g, h)]
    loss = lambda u, g, h: sum((t * w.double()).sum() for t, w in zip(f(u, g, h), (d["dy"], d["dlast"])))
    size = sum((t.abs() * w.double().abs()).sum() for t, w in zip(f(d["u"], d["gate"], d["h0"]), (d["dy"], d["dlast"])))
    e = 2.0 ** -7
    for k, name in enumerate(("u", "gate", "h0")):
        v = torch.randn(d[name].shape, generator=gen).cuda()
        v /= v.abs().max()
        args = [d["u"], d["gate"], d["h0"]]
        lo, hi = list(args), list(args)
        lo[k], hi[k] = args[k] - e * v, args[k] + e * v
        slope = (loss(*hi) - loss(*lo)) / (2 * e)
        want = (got["d" + name].double() * v.double()).sum()
        assert abs(slope - want) < size * (30 * 2.0 ** -24 / e + e * e), name


def test_same_bits_every_time_and_on_another_stream():
    d = inputs((3, 2000, 130), 3, BF16, "sigmoid")
    first = run(d, "sigmoid", True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(d, "sigmoid", True)
    side.synchronize()
    for k in first:
        assert torch.equal(first[k], again[k]), k


def test_two_captured_graphs_at_once():
    """Training steps of two sizes and one token, recorded, then replayed on new inputs, two graphs on two streams at a time."""
    data = [inputs((2, 900, 66), 2, BF16, "sigmoid", seed=s) for s in (0, 1)]
    steps, graphs = [], []
    for d in data:
        leaves = [d[k].requires_grad_(True) for k in ("u", "gate", "h0")]

        def step(d=d, leaves=leaves):
            y, last = cs2d.gated_scan_1d(*leaves)
            g = torch.autograd.grad([y, last], leaves, [d["dy"], d["dlast"]])
            with torch.no_grad():
                h = last.clone()
                return [y, last, *g, cs2d.gated_scan_step(d["u"][:, 0], d["gate"][:, 0], h), h]
        steps.append(step)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for d in data:
        with torch.no_grad():
            for k in ("u", "gate", "dy", "dlast", "h0"):
                d[k].copy_(torch.randn(d[k].shape, device="cuda"))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, out), step in zip(graphs, steps):
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_a_held_eager_graph_of_the_same_leaves_refuses_the_capture():
    """In a process of its own: without the refusal the backward of the recorded step would end it."""
    code = textwrap.dedent("""
        import sys, torch
        sys.path.insert(0, "official-cross-scan_b200")
        import cs2d
        u, g = (torch.randn(1, 50, 8, device="cuda", requires_grad=True) for _ in range(2))
        x = torch.randn(4, 8, device="cuda", requires_grad=True)
        held = cs2d.gated_scan_1d(u, g)[0], cs2d.layer_norm(x)
        for call in (lambda: cs2d.gated_scan_1d(u, g), lambda: cs2d.layer_norm(x)):
            try:
                with torch.cuda.graph(torch.cuda.CUDAGraph()):
                    call()
                print("captured")
            except RuntimeError as e:
                print("refused" if "default stream" in str(e) else e)
        del held
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, _ = cs2d.gated_scan_1d(u, g)
            du, = torch.autograd.grad(y, u, torch.ones_like(y))
        graph.replay()
        torch.cuda.synchronize()
        print("done", bool(torch.isfinite(du).all()))
    """)
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["refused", "refused", "done", "True"], r.stdout + r.stderr


def test_no_second_derivative():
    u, g = (torch.randn(1, 5, 8, device="cuda", requires_grad=True) for _ in range(2))
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(cs2d.gated_scan_1d(u, g)[0].sum(), u, create_graph=True)


def test_refusals():
    u, h = torch.randn(2, 5, 8, device="cuda"), torch.zeros(2, 8, device="cuda")
    off = torch.tensor([0, 5], device="cuda")
    for args, kw, msg in [((u.double(), u.double()), {}, "not implemented for input type"), ((u, u.half()), {}, "dtype of u"), ((u, u[:1]), {}, "shape of u"),
                          ((u, u, h.half()), {}, "h0 must be float32"), ((u, u, h[:1]), {}, "h0 must have shape"), ((u, u.cpu()), {}, "device"),
                          ((u[0, 0], u[0, 0]), {}, "u must have shape"), ((u, u, None, off), {}, "total, dim"), ((u[0], u[0], None, off.float()), {}, "offsets"),
                          ((u[0], u[0], None, off.cpu()), {}, "device"), ((u[0], u[0], None, off[:0]), {}, "offsets"), ((u, u), {"form": "tanh"}, "form must be")]:
        with pytest.raises(RuntimeError, match=msg):
            cs2d.gated_scan_1d(*args, **kw)
    v = u[:, 0]
    for args, msg in [((u, u, h), "batch, dim"), ((v, v, h.half()), "float32"), ((v, v, h[:1].expand(2, 8)), "overlap"), ((v, v, h.t().contiguous().t()), "in place"),
                      ((v.clone().requires_grad_(True), v, h), "no gradient"), ((v, v, h[:1]), "shape of u")]:
        with pytest.raises(RuntimeError, match=msg):
            cs2d.gated_scan_step(*args)


def test_more_elements_than_32_bits_count():
    """2 x 1100000 x 1024 bf16 elements: a gate of zero passes every input on, one of one adds up what a counting input brings."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    u = torch.empty(2, 1100000, 1024, dtype=BF16, device="cuda")
    for b in range(2):
        for i in range(0, u.shape[1], 100000):
            u[b, i:i + 100000].normal_()
    with torch.no_grad():
        y, last = cs2d.gated_scan_1d(u, torch.zeros(1, 1, 1024, dtype=BF16, device="cuda").expand_as(u), None, form="direct", weighted=False)
        assert torch.equal(y, u) and torch.equal(last, u[:, -1].float())
        del y
        n = cs2d.layer_norm(u, eps=1e-5)
        for at in (0, 1048575, 1048576, 1099999):
            for b in range(2):
                row = u[b, at].double()
                want = (row - row.mean()) / (row.var(unbiased=False) + 1e-5).sqrt()
                assert float((n[b, at].double() - want).abs().max()) <= 4 * (R.half_step(BF16) + 1e-5) * float(want.abs().max())


def test_a_state_that_may_not_be_written_stays_as_it_is():
    """An inference tensor outside inference mode: refused, as torch refuses it, before anything is written."""
    u = torch.randn(2, 8, device="cuda")
    with torch.inference_mode():
        h = torch.ones(2, 8, device="cuda")
        before = cs2d.gated_scan_step(u, u, h).clone()
        kept = h.clone()
    with pytest.raises(RuntimeError, match="inference"):
        cs2d.gated_scan_step(u, u, h)
    assert torch.equal(h, kept) and torch.isfinite(before).all()


def test_tangents_are_refused_not_lost():
    """Forward-mode differentiation is not implemented: an input with a tangent raises, whether it wants a gradient or not."""
    import torch.autograd.forward_ad as fw
    u, h, off = torch.randn(2, 5, 8, device="cuda"), torch.randn(2, 8, device="cuda"), torch.tensor([0, 2, 5], device="cuda")
    w = torch.ones(8, device="cuda")
    for needs in (False, True):
        with fw.dual_level():
            dual = lambda t: fw.make_dual(t.clone().requires_grad_(needs), torch.ones_like(t))
            calls = [lambda: cs2d.gated_scan_1d(dual(u), u, h), lambda: cs2d.gated_scan_1d(u, dual(u), h), lambda: cs2d.gated_scan_1d(u, u, dual(h)),
                     lambda: cs2d.gated_scan_1d(u[0], dual(u[0]), None, off), lambda: cs2d.layer_norm(dual(u)), lambda: cs2d.layer_norm(u, dual(w)),
                     lambda: cs2d.layer_norm(u, w, dual(w)), lambda: cs2d.layer_norm(u, w, None, dual(u))]
            for i, call in enumerate(calls):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
                with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
                    call()
            with torch.no_grad():
                for args in ((dual(u[:, 0]), u[:, 0], h), (u[:, 0], dual(u[:, 0]), h), (u[:, 0], u[:, 0], dual(h))):
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        cs2d.gated_scan_step(*args)
    with torch.no_grad():
        assert cs2d.layer_norm(u).shape == u.shape and cs2d.gated_scan_step(u[:, 0], u[:, 0], h).shape == h.shape
