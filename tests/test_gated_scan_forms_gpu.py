"""gated_scan_1d in the forms that large problems take, over many steps of a unit's loop.

A unit is 64 channels wide where there are at least 96 such units or at most 128 rows, else 16; a cluster of CTAs shares a unit's rows
where all clusters fit the GPU at once (at most two CTAs to an SM), else one CTA walks them.  A step of the loop is 128 rows per CTA of a wide
unit of a 16-bit type (64 of float32; the backward half as many), four times as many of a narrow one.
"""
import pytest
import torch

import cs2d
import gated_reference as R
from test_gated_scan_gpu import inputs, packed, run

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def check(d, got, form, weighted, h0=True, dlast=True):
    """All batch rows at once: channels do not know of each other, so the batch is more channels."""
    seq = lambda t: t.transpose(0, 1).reshape(t.shape[1], -1)
    want = R.expected(seq(d["u"]), seq(d["gate"]), d["h0"].reshape(-1) if h0 else None, seq(d["dy"]), d["dlast"].reshape(-1) if dlast else None,
                      form, weighted, d["u"].dtype)
    for k, v in got.items():
        R.check(k, seq(v) if v.dim() == 3 else v.reshape(-1), want[k])
    assert cs2d.device_status() == 0


# wide: clusters of two, one CTA, one CTA and four blocks of channels the last of which has 8 of 64, rows on 4 bytes, clusters of two with one channel
# more than 64, and with 33 for five steps and more; narrow: one CTA (285 units, 180), the last block with 1 and 3 channels
@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("shape,form,weighted", [((96, 400, 64), "sigmoid", True), ((200, 330, 64), "log", True), ((50, 333, 200), "direct", False),
                                                 ((99, 300, 66), "sigmoid", False), ((48, 643, 65), "log", False), ((97, 1300, 33), "direct", True),
                                                 ((95, 1100, 33), "sigmoid", True), ((60, 1100, 35), "log", True)])
def test_many_units_over_many_steps(shape, form, weighted, dtype):
    d = inputs(shape, shape[0], dtype, form, seed=shape[1])
    check(d, run(d, form, weighted), form, weighted)


@pytest.mark.parametrize("dtype", (F32, BF16))
def test_a_wide_form_without_states_and_on_views(dtype):
    d = inputs((98, 600, 3 * 64 + 1), 98, dtype, "sigmoid", seed=1)
    for left in (64, 1):        # rows on 2 (4) bytes in both; with and without a piece on 16 bytes
        e = {k: d[k][..., left:left + 64] for k in ("u", "gate", "dy")}
        e["h0"], e["dlast"] = d["h0"][:, left:left + 64], d["dlast"][:, left:left + 64]
        check(e, run(e, "sigmoid", True, h0=False, dlast=False), "sigmoid", True, h0=False, dlast=False)
        check(e, run(e, "sigmoid", True), "sigmoid", True)


# wide with clusters of two and one CTA, rows on 4 and on 16 bytes; narrow with one CTA: 200 units
@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("dim", (6150, 12800, 3200))
def test_packed_rows_of_many_units(dim, dtype):
    lengths = {6150: [0, 1, 200, 37, 0, 0, 500, 129, 2], 12800: [0, 1, 200, 0, 130], 3200: [500, 0, 1, 700]}[dim]
    form = "sigmoid" if dtype == BF16 else "log"
    d, off = packed(lengths, dim, dtype, form, before=9, behind=70)
    got = run(d, form, True, offsets=torch.tensor(off, dtype=torch.int32, device="cuda"))
    for k in ("y", "du", "dgate"):
        assert not got[k][:off[0]].any() and not got[k][off[-1]:].any(), k
    for s in range(len(lengths)):
        r = slice(off[s], off[s + 1])
        want = R.expected(d["u"][r], d["gate"][r], d["h0"][s], d["dy"][r], d["dlast"][s], form, True, dtype)
        for k, v in got.items():
            R.check(f"{k} of sequence {s}", v[r] if k in ("y", "du", "dgate") else v[s], want[k])
    assert cs2d.device_status() == 0


def test_many_short_sequences():
    """Thousands of sequences, every third of them empty, states of their own; odd rows, two channels more than a narrow unit."""
    gen = torch.Generator().manual_seed(0)
    lengths = torch.randint(1, 6, (3000,), generator=gen)
    lengths[::3] = 0
    lengths = lengths.tolist()
    d, off = packed(lengths, 18, F32, "direct", before=1, behind=2)
    got = run(d, "direct", True, offsets=torch.tensor(off, dtype=torch.int64, device="cuda"))
    a, u, dy = (d[k].double().cpu() for k in ("gate", "u", "dy"))
    h0, dlast = d["h0"].double().cpu(), d["dlast"].double().cpu()
    for s in (0, 1, 2, 3, 4, 1500, 1501, 2996, 2997, 2998, 2999):
        r = slice(off[s], off[s + 1])
        want = R.expected(u[r].float(), a[r].float(), h0[s], dy[r].float(), dlast[s], "direct", True, F32)
        for k, v in got.items():
            R.check(f"{k} of sequence {s}", v[r] if k in ("y", "du", "dgate") else v[s], want[k])
    # and all of them by their padded form, sequence by sequence along a second axis: five steps of the definition
    n = torch.tensor(lengths)
    at = torch.tensor(off[:-1])
    h, H, M = h0.clone(), h0.abs(), torch.zeros_like(h0)         # H, M: as in gated_reference
    ys, tol = torch.zeros_like(u), torch.zeros_like(u)
    for t in range(5):
        on = n > t
        i = at[on] + t
        b = (1 - a[i]) * u[i]
        M[on] = a[i].abs() * (M[on] + H[on]) + b.abs()
        H[on] = a[i].abs() * H[on] + b.abs()
        h[on] = a[i] * h[on] + b
        ys[i], tol[i] = h[on], R.K[F32] * R.UNIT * M[on]
    inside = slice(off[0], off[-1])
    assert ((got["y"].detach().double().cpu() - ys)[inside].abs() <= tol[inside]).all()
    assert ((got["h_last"].detach().double().cpu() - h).abs() <= R.K[F32] * R.UNIT * M).all()


def test_more_elements_than_32_bits_count_forward_and_backward():
    """2 x 1100000 x 1024 bf16 elements with a dense gate of one: y counts up what four rows far apart bring, du counts up from the end what four
    rows of dy bring, dgate is their product: small whole numbers, exact in every type."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    B, L, D = 2, 1100000, 1024
    u, gate, dy = (torch.full((B, L, D), v, dtype=BF16, device="cuda") for v in (0.0, 1.0, 0.0))
    brings = {0: 1, 511: 2, 1048575: 3, 1099998: 1}          # rows of u; the second batch row brings it negated
    asks = {1099999: 2, 1048576: 1, 512: 3, 31: 1}           # rows of dy
    c = (torch.arange(D, device="cuda") % 2 + 1).float()     # channels differ
    for t, v in brings.items():
        u[0, t], u[1, t] = v * c, -v * c
    for t, v in asks.items():
        dy[:, t] = v
    for t in (u, gate):
        t.requires_grad_(True)
    y, last = cs2d.gated_scan_1d(u, gate, None, form="direct", weighted=False)
    du, dgate = torch.autograd.grad(y, [u, gate], dy)
    borders = sorted({0, L} | {t + k for t in brings for k in (0, 1)} | {t + k for t in asks for k in (0, 1)})
    for lo, hi in zip(borders[:-1], borders[1:]):            # constant between
        h = sum(v for t, v in brings.items() if t <= lo)
        before = sum(v for t, v in brings.items() if t < lo)
        e = sum(v for t, v in asks.items() if t >= hi - 1)
        for b, sign in enumerate((1, -1)):
            row = lambda v: v.to(BF16)[None].expand(hi - lo, D)
            assert torch.equal(y[b, lo:hi], row(sign * h * c)), (lo, b)
            assert torch.equal(du[b, lo:hi], row(torch.full_like(c, e))), (lo, b)
            assert torch.equal(dgate[b, lo:hi].float(), row(sign * before * e * c).float()), (lo, b)
    assert torch.equal(last[0], 7 * c) and torch.equal(last[1], -7 * c)
    assert cs2d.device_status() == 0


def test_first_calls_from_several_threads():
    """In a process of its own: threads whose streams launch every kernel for the first time, at the same time."""
    import subprocess
    import sys
    import textwrap
    from conftest import ROOT
    code = textwrap.dedent("""
        import sys, threading, torch
        sys.path.insert(0, "official-cross-scan_b200")
        import cs2d
        u, g, z = (torch.randn(40, 400, 64, device="cuda") for _ in range(3))
        w = torch.ones(64, device="cuda")
        def step():
            a = [t.detach().requires_grad_(True) for t in (u, g, z, w)]
            y = cs2d.layer_norm(cs2d.gated_scan_1d(a[0], a[1])[0], a[3], None, a[2])
            return [y.detach(), *torch.autograd.grad(y, a, torch.ones_like(y))]
        torch.cuda.synchronize()
        gate, outs = threading.Barrier(8), [None] * 8
        def work(i):
            with torch.cuda.stream(torch.cuda.Stream()):
                gate.wait()
                outs[i] = step()
                torch.cuda.current_stream().synchronize()
        threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
        [t.start() for t in threads], [t.join() for t in threads]
        want = step()
        print(all(torch.equal(p, q) for o in outs for p, q in zip(o, want)), cs2d.device_status())
    """)
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["True", "0"], r.stdout + r.stderr


def test_a_launch_that_failed_is_not_reported_twice():
    """In a process of its own: a recording that something else has made invalid refuses the scan's launch; the next call, on a good stream, runs."""
    import subprocess
    import sys
    import textwrap
    from conftest import ROOT
    code = textwrap.dedent("""
        import sys, torch
        sys.path.insert(0, "official-cross-scan_b200")
        import cs2d
        u, x = torch.randn(1, 300, 64, device="cuda"), torch.randn(5, 64, device="cuda")
        want = cs2d.layer_norm(x), cs2d.gated_scan_1d(u, u)[0]
        torch.cuda.synchronize()
        try:
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                try:
                    torch.cuda.synchronize()            # not allowed while recording
                except RuntimeError:
                    pass
                try:
                    cs2d.gated_scan_1d(u, u)
                    print("launched")
                except RuntimeError as e:
                    print("refused" if "launch failed" in str(e) else e)
        except RuntimeError:
            print("invalid")
        print(torch.equal(cs2d.layer_norm(x), want[0]), torch.equal(cs2d.gated_scan_1d(u, u)[0], want[1]))
    """)
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["refused", "invalid", "True", "True"], r.stdout + r.stderr
