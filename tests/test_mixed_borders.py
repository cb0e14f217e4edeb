"""The 16-bit operators (plnlp_amd/mixed.py) where their kernels change over and where their numbers leave the middle of the range:
sums over many rows compared bit for bit, saturated activations, values at the edge of a type, sorts of more than 2^20 ids, tensors
that cannot be written, operands with a forward-mode tangent.

Where inputs are small whole numbers every sum is exact in f32 (below 2^24) and one rounding to the type is left, so results are
compared for equality; other tolerances are bounds of the arithmetic, with u = finfo(type).eps / 2 for one rounding to the type."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {t: torch.finfo(t).eps / 2 for t in (F32, BF16, F16)}
TINY = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for t in (F32, BF16, F16)}
ADD = 2.0 ** -23               # an f32 addition, on the matrix cores too


@pytest.fixture(scope="module")
def P():
    import plnlp_amd
    from plnlp_amd import _lib
    _lib.load()
    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    return plnlp_amd


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def whole(shape, dtype, seed, lo=-1, hi=1):
    return torch.randint(lo, hi + 1, shape, generator=generator(seed), device="cuda").to(dtype)


# ------------------------------------------------------------------ gradients summed over many rows ------
def backward_of_whole_numbers(P, m, n, k, dtype, act="none", slope=None):
    """(dx, dw, db) through the C ABI from a workspace of NaN, and what they have to be: gy, x and w in {-1, 0, 1}, the slope 1 where it
    is given at all, so every sum is a whole number below 2^24 and the result is its one rounding"""
    from plnlp_amd import _lib as L
    lib = L.load()
    gy, x, w = whole((m, n), dtype, 1), whole((m, k), dtype, 2), whole((n, k), dtype, 3)
    dx, dw, db = (torch.full(s, math.nan, dtype=dtype, device="cuda") for s in ((m, k), (n, k), (n,)))
    code = L.ACTIVATIONS[act]
    n_bytes = lib.plnlp_linear_act_backward_workspace_bytes(m, n, k, code)
    ws = torch.full(((n_bytes + 3) // 4,), math.nan, device="cuda")
    L.check(lib.plnlp_linear_act_backward(gy.data_ptr(), n, L.ptr(slope), n, code, x.data_ptr(), k, w.data_ptr(), k, m, n, k, dx.data_ptr(), k,
                                          dw.data_ptr(), k, db.data_ptr(), L.DTYPE_CODES[dtype], ws.data_ptr(), n_bytes, L.stream_ptr()), "backward")
    gf, xf, wf = gy.float(), x.float(), w.float()
    return (dx, dw, db), ((gf @ wf).to(dtype), (gf.t() @ xf).to(dtype), gf.sum(0).to(dtype))


# rows below, at and past the count from which the weights' gradient of a 256-wide layer is cut into 256 x 256 tiles, whose kernel takes
# no column sums: widths that take them (their product is 57 344 or more) and one that does not
@gpu
@pytest.mark.parametrize("m", [393088, 393216, 400008])
@pytest.mark.parametrize("n,k", [(256, 256), (240, 240), (224, 256), (256, 224), (248, 216)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_bias_gradient_of_very_many_rows(P, m, n, k, dtype):
    got, want = backward_of_whole_numbers(P, m, n, k, dtype)
    for name, a, b in zip(("dx", "dw", "db"), got, want):
        assert torch.equal(a, b), name


@gpu
def test_bias_gradient_of_very_many_rows_through_the_layer(P):
    layer = P.LinearAct(256, 256).cuda()
    x, gy = whole((393216, 256), BF16, 1).requires_grad_(True), whole((393216, 256), BF16, 2)
    dx, dw, db = torch.autograd.grad(layer(x), [x, layer.lin.weight, layer.lin.bias], gy)
    assert torch.equal(db, gy.float().sum(0).to(BF16))
    assert torch.equal(dw, (gy.float().t() @ x.detach().float()).to(BF16))


# The sums over rows (dw, db) and over columns (dx) bit for bit, so that a lost K slice, tile, last step or workgroup's part shows: each
# kernel that takes them (tiles of 128 and 256, rows in LDS or streamed, column sums beside dx, beside dw or on their own), whole and
# ragged rows.  With relu a slope of 1 is written down; without an activation none is read.
@gpu
@pytest.mark.parametrize("m,n,k", [(777, 520, 136), (16384, 1024, 512), (16390, 1280, 576), (12552, 1000, 1032), (1792, 8200, 520), (32770, 256, 256),
                                   (33800, 264, 96), (34000, 72, 264), (65537, 512, 64), (8300, 72, 520), (8209, 33, 64), (131072, 256, 256),
                                   (40001, 200, 200)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", ["none", "relu"])
def test_sums_of_whole_numbers(P, m, n, k, dtype, act):
    slope = torch.full((m, n), 1 << 14, dtype=torch.int16, device="cuda") if act == "relu" else None
    got, want = backward_of_whole_numbers(P, m, n, k, dtype, act, slope)
    for name, a, b in zip(("dx", "dw", "db"), got, want):
        assert torch.equal(a, b), name


@gpu
@pytest.mark.parametrize("m,n,k,act", [(16384, 1024, 512, "silu"), (32770, 256, 256, "gelu"), (65537, 512, 64, "none"), (777, 515, 1003, "gelu_tanh"),
                                       (1, 4096, 4096, "silu"), (40001, 200, 200, "silu")])
def test_the_same_bits_twice(P, m, n, k, act):
    x, w, b = (torch.randn(s, generator=generator(i), device="cuda").to(BF16).requires_grad_(True) for i, s in enumerate(((m, k), (n, k), (n,))))
    gy = torch.randn((m, n), generator=generator(9), device="cuda").to(BF16)

    def run():
        y = P.linear_act(x, w, b, activation=act)
        return [y.detach(), *torch.autograd.grad(y, [x, w, b], gy)]
    for u, v in zip(run(), run()):
        assert torch.equal(u, v)
