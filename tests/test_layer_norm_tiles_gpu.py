"""layer_norm where a CTA works on several tiles and a group of lanes on several rows of a tile: the shapes of training batches.

The backward runs at most four CTAs to an SM (592), the forward six (888); tiles of tokens hold 1, 2, 4 or 8 rows per group of lanes while there are
tiles for all CTAs, those of images up to 64 positions (32 of float32).
"""
import pytest
import torch

import cs2d
import gated_reference as R
from test_layer_norm_gpu import U, check, expected, inputs, run, step

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


# vectors of 16 bytes, pairs of 16-bit elements, single elements; two to eight rows per group, more tiles than CTAs in every backward
@pytest.mark.parametrize("gated", (False, True))
@pytest.mark.parametrize("dim,dtype", [(768, F32), (768, BF16), (768, F16), (770, BF16), (771, F32), (771, BF16), (387, F16)])
def test_tokens_of_several_tiles(dim, dtype, gated):
    d = inputs((5003,), dim, dtype, gated, seed=dim)
    check(d, run(d))
    assert cs2d.device_status() == 0


@pytest.mark.parametrize("dtype", (F32, BF16))
def test_tokens_whose_outer_index_changes_inside_a_cta(dtype):
    d = inputs((2, 10100), 192, dtype, True, seed=1)
    e = {k: d[k][:, :10007] for k in ("x", "gate", "dy")}        # not one run of rows
    e.update(weight=d["weight"], bias=d["bias"])
    check(e, run(e))


# whole tiles of 64 and 32 positions, of 16 (wide rows) and element by element; float32 tiles of 32
@pytest.mark.parametrize("lead,dim,dtype", [((16, 64, 64), 96, BF16), ((16, 64, 64), 96, F32), ((14, 24, 32), 768, F16), ((20, 16, 16), 1536, BF16),
                                            ((60, 33, 31), 51, BF16), ((60, 33, 31), 51, F32), ((3, 104, 104), 100, F16)])
@pytest.mark.parametrize("gated", (False, True))
def test_images_of_several_tiles(lead, dim, dtype, gated):
    d = inputs(lead, dim, dtype, gated, seed=dim, image=True)
    check(d, run(d))
    assert cs2d.device_status() == 0


# a row's values do not depend on the rows beside it: a batch gives the bits of its parts, which run on other tiles, and its sums are theirs
@pytest.mark.parametrize("lead,dim,dtype,image", [((120003,), 192, BF16, False), ((50001,), 387, F32, False), ((30011,), 770, F16, False), ((25088,), 768, F32, False),
                                                  ((24, 96, 96), 384, BF16, True), ((24, 75, 75), 387, F16, True), ((24, 96, 96), 192, F32, True)])
def test_a_batch_gives_the_bits_of_its_parts(lead, dim, dtype, image):
    gen = torch.Generator(device="cuda").manual_seed(dim)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    d = {k: n(*lead, dim).to(dtype) for k in ("x", "gate", "dy")}
    if image:
        d["x"] = d["x"].movedim(-1, 1).contiguous().movedim(1, -1)
    d["weight"], d["bias"] = 1 + 0.2 * n(dim), 0.3 * n(dim)
    got = step(d)
    size = 1 if image else lead[0] // 24 + 1
    parts = []
    for at in range(0, lead[0], size):
        parts.append(step({k: v if v.dim() == 1 else v[at:at + size] for k, v in d.items()}))
    for k in ("y", "dx", "dgate"):
        assert torch.equal(got[k], torch.cat([p[k] for p in parts])), k
    rows = got["y"].numel() // dim
    xh = torch.nn.functional.layer_norm(d["x"].float(), (dim,), eps=1e-5).abs()
    dn = (d["dy"].float() * torch.nn.functional.silu(d["gate"].float())).abs()
    for k, terms in (("dweight", dn * xh), ("dbias", dn)):
        whole = sum(p[k].double() for p in parts)
        # both are sums of the same float32 terms in two orders: a lane adds fewer than `rows` / 32 of them before sums are joined
        bound = 2 * (rows / 32 + 64) * U * terms.double().reshape(-1, dim).sum(0)
        assert ((got[k].double() - whole).abs() <= bound).all(), k


@pytest.mark.parametrize("image", (False, True))
def test_more_elements_than_32_bits_count_backward(image):
    """2 x 1100000 x 1024 bf16 elements: rows from everywhere against float64, the parameters' sums against exact ones."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    B, L, D = 2, 1100000, 1024
    x = torch.empty((B, D, L) if image else (B, L, D), dtype=BF16, device="cuda")
    for b in range(B):       # channels of different means, so that the sums of normalised values grow with every row
        x[b].normal_().add_(torch.linspace(-1, 1, D, device="cuda").view((D, 1) if image else (D,)))
    x = x.movedim(1, 2) if image else x
    w = (1 + 0.2 * torch.randn(D, device="cuda")).requires_grad_(True)
    bias = torch.zeros(D, device="cuda", requires_grad=True)
    dy = torch.ones(B, L, D, dtype=BF16, device="cuda")
    y = cs2d.layer_norm(x.requires_grad_(True), w, bias)
    dx, dw, db = torch.autograd.grad(y, [x, w, bias], dy)
    assert dx.stride() == x.stride()
    assert (db == B * L).all()                       # ones, counted: exact
    for b in range(B):
        rows = torch.tensor([0, 1, 63, 64, 524287, 524288, 1048575, 1048576, 1099967, 1099999], device="cuda")
        want = expected(x[b, rows], w, None, None, dy[b, rows])
        R.check("y", y[b, rows], want["y"])
        R.check("dx", dx[b, rows], want["dx"])
    total, size = torch.zeros(D, dtype=torch.float64, device="cuda"), torch.zeros(D, dtype=torch.float64, device="cuda")
    with torch.no_grad():
        for b in range(B):
            for at in range(0, L, 100000):
                t = x[b, at:at + 100000].double()
                t = t - t.mean(-1, keepdim=True)
                t *= (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
                total += t.sum(0)
                size += t.abs().sum(0)
    # 296 CTAs of four rows at a time: a lane adds fewer than B * L / 1024 terms before sums are joined, each a normalised value off by fewer than
    # D / 32 + 32 units of the largest of its row (below 8)
    assert ((dw.double() - total).abs() <= (B * L / 1024 + 64) * U * size + B * L * 8 * (D / 32 + 32) * U).all()
    assert (total[0] < -0.5 * B * L) and (total[-1] > 0.5 * B * L)


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("dim", (51, 192, 768))
def test_an_axis_of_one_between_rows_and_channels(dim, dtype):
    """(B, 1, dim), as tokens that are decoded together or maps of one position have it, is (B, dim): the same kernels, so the same bits."""
    d = inputs((6001,), dim, dtype, True, seed=dim)
    plain = run(d)
    for shape in ((6001, 1, dim), (6001, 1, 1, dim)):
        e = {k: v.reshape(shape) if v.dim() > 1 else v for k, v in d.items()}
        got = run(e)
        for k, v in got.items():
            assert torch.equal(v, plain[k].reshape(v.shape)), (k, shape)


def test_an_axis_of_one_with_strides_of_each_their_own():
    """x, gate and dy are columns of wider tensors, of one width each; the same for images of one position and for one row."""
    B, D = 700, 96
    d = inputs((B, 1), 3 * D, BF16, True)
    e = {"x": d["x"][..., D:2 * D], "gate": torch.cat([d["gate"], d["gate"]], -1)[..., 8:D + 8], "dy": d["dy"][:, :, :D].contiguous(),
         "weight": d["weight"][:D], "bias": d["bias"][:D]}
    check(e, run(e))
    e["dy"] = d["dy"][..., :D]
    check(e, run(e))
    e["x"] = d["x"][:, 0, :D].t().contiguous().t()[:, None]        # channels apart: a copy
    check(e, run(e))
    one = {k: v[:1] if v.dim() > 1 else v for k, v in e.items()}
    check(one, run(one))
    image = dict(e, x=torch.randn(B, D, 1, 1, device="cuda").to(BF16).permute(0, 2, 3, 1))
    image.update(gate=e["gate"][:, None], dy=e["dy"][:, None])
    check(image, run(image))
