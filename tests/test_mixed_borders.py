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


# ------------------------------------------------------------------ saturated units ------
def slope_ref(z, name):
    if name == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c, a = math.sqrt(2 / math.pi), 0.044715
    s = torch.sigmoid(2 * c * (z + a * z ** 3))          # (1 + tanh) / 2 without its cancellation
    return s + z * s * torch.sigmoid(-2 * c * (z + a * z ** 3)) * 2 * c * (1 + 3 * a * z * z)


# Every unit far on the flat side, where the derivative is 10^-2 .. 10^-9: the gradients in RELATIVE terms.  The kept derivative is off by
# 2^-10 of itself there; the f32 exponentials (arguments below 64: 64 * 2^-23 * ln 2) and the fitted normal distribution (1.2e-5, in a sum
# that it is an eighth of) by less than 2e-5; z itself by e_z, which the derivative's logarithm follows at a rate below 10 (gelu: |z|;
# gelu_tanh: 1.6 (1 + 0.13 z^2); silu: 1).  dz is rounded to the type before dx and dw are taken, db sums it unrounded; what
# remains of each is the sums' f32 additions and one rounding.  gy and x are positive: nothing cancels in dw and db.
@gpu
@pytest.mark.parametrize("act,center,spread,dtype,gain", [("gelu", -4.0, 0.15, BF16, 1.0), ("gelu", -5.5, 0.2, BF16, 1.0), ("gelu", -4.2, 0.1, F16, 512.0),
                                                          ("gelu_tanh", -4.0, 0.2, BF16, 1.0), ("gelu_tanh", -5.0, 0.1, BF16, 1.0),
                                                          ("silu", -6.0, 0.3, BF16, 1.0), ("silu", -10.0, 0.5, BF16, 1.0), ("silu", -22.0, 1.0, BF16, 1.0),
                                                          ("silu", -10.0, 0.5, F16, 512.0)])
@pytest.mark.parametrize("m,n,k", [(4, 64, 64), (40, 96, 64), (300, 136, 72), (300, 131, 77), (8200, 200, 72), (8192, 256, 256)])
def test_gradients_of_saturated_units(P, act, center, spread, dtype, gain, m, n, k):
    u, tiny = U[dtype], TINY[dtype]
    x = (0.5 + torch.rand((m, k), generator=generator(1), device="cuda")).to(dtype).requires_grad_(True)
    w = (torch.randn((n, k), generator=generator(2), device="cuda") * spread / math.sqrt(k)).to(dtype).requires_grad_(True)
    b = torch.full((n,), center, dtype=dtype, device="cuda", requires_grad=True)
    gy = ((0.5 + torch.rand((m, n), generator=generator(3), device="cuda")) * gain).to(dtype)
    xd, wd, g = x.detach().double(), w.detach().double(), gy.double()
    z = xd @ wd.t() + b.detach().double()
    assert -30 < float(z.min()) and float(z.max()) < -2.5 and bool((slope_ref(z, act) < 0).all())
    e_z = (xd.abs() @ wd.abs().t()) * (k + 2) * ADD + z.abs() * ADD
    dz = g * slope_ref(z, act)
    relative = 2.0 ** -10 + 2e-5 + 10 * e_z
    e_sum = dz.abs() * relative                                    # of the dz that db sums
    e_dz = dz.abs() * (relative + u * 1.01) + tiny                 # of the rounded one
    dx, dw, db = torch.autograd.grad(P.linear_act(x, w, b, activation=act), [x, w, b], gy)
    for name, got, want, bound in (("db", db, dz.sum(0), e_sum.sum(0) + dz.abs().sum(0) * (m + 2) * ADD),
                                   ("dw", dw, dz.t() @ xd, e_dz.t() @ xd.abs() + (dz.t().abs() @ xd.abs()) * (m + 2) * ADD),
                                   ("dx", dx, dz @ wd, e_dz @ wd.abs() + (dz.abs() @ wd.abs()) * (n + 2) * ADD)):
        bound = bound + want.abs() * u * 1.01 + tiny
        over = (got.double() - want).abs() - bound
        assert not bool(torch.isnan(over).any()) and float(over.max()) <= 0.0, (name, float(((got.double() - want).abs() / want.abs()).max()))
        if name != "dx":                                           # the bounds say something: within 2 % of what they bound
            assert float((bound / want.abs()).median()) <= 0.02, name


# ------------------------------------------------------------------ the edge of a type ------
@gpu
@pytest.mark.parametrize("m,n,k", [(2, 8, 8), (20, 24, 64)])
@pytest.mark.parametrize("dtype,most", [(F16, 60000.0), (BF16, 2.9e38)])
def test_small_dz_at_the_edge_of_the_type(P, m, n, k, dtype, most):
    """few elements of dz, kept as two terms: dy * act'(z) past the type's largest number (act' = 1.129 at z = 1.414, gelu) gives the
    product's own finite values, an infinite dy gives infinities and a NaN stays in its row, in all three gradients"""
    x = torch.zeros(m, k, dtype=dtype, device="cuda")
    x[:, 0] = 1.0
    w = torch.full((n, k), 2.0 ** -10, dtype=dtype, device="cuda")
    w[:, 0] = 1.4140625
    x.requires_grad_(True), w.requires_grad_(True)
    b = torch.zeros(n, dtype=dtype, device="cuda", requires_grad=True)
    gy = torch.zeros(m, n, dtype=dtype, device="cuda")
    gy[0, 0] = most
    slope = float(0.5 * (1 + math.erf(1.4140625 * math.sqrt(0.5))) + 1.4140625 * math.exp(-1.4140625 ** 2 / 2) / math.sqrt(2 * math.pi))
    dz = float(gy[0, 0]) * slope
    limit = torch.finfo(dtype).max
    if dtype == F16:
        assert dz > limit
    dx, dw, db = torch.autograd.grad(P.linear_act(x, w, b, activation="gelu"), [x, w, b], gy)
    # the slope is kept in steps of 2^-14 and computed to 2e-5, two terms hold dz to u^2, the result is rounded once
    for got in dx[0, 1:].double():
        assert abs(float(got) - dz * 2.0 ** -10) <= dz * 2.0 ** -10 * (2.0 ** -15 + 2e-5 + 2 * U[dtype])
    assert not bool(dx[1:].any())
    if dtype == F16:
        assert float(dw[0, 0]) == math.inf and float(db[0]) == math.inf          # (these are dz itself: past the type)
    assert not bool(torch.isnan(dx).any() or torch.isnan(dw[1:]).any() or torch.isnan(db).any())
    gy[0, 0] = math.inf
    dx, dw, db = torch.autograd.grad(P.linear_act(x, w, b, activation="gelu"), [x, w, b], gy)
    assert bool((dx[0] == math.inf).all()) and not bool(dx[1:].any())
    assert float(dw[0, 0]) == math.inf and not bool(dw[1:].any()) and float(db[0]) == math.inf and not bool(db[1:].any())
    gy[0, 0] = math.nan
    dx, dw, db = torch.autograd.grad(P.linear_act(x, w, b, activation="gelu"), [x, w, b], gy)
    assert bool(torch.isnan(dx[0]).all()) and not bool(dx[1:].any()) and bool(torch.isnan(dw[0]).all()) and math.isnan(float(db[0]))


# ------------------------------------------------------------------ refusals ------
def test_a_forward_mode_tangent_is_refused():
    """no operator has a forward-mode derivative: an operand that carries a tangent is refused, with a graph and without, before anything
    else is looked at (no device needed)"""
    import torch.autograd.forward_ad as fwd
    import plnlp_amd as P
    x, w, b, r = (torch.ones(s, dtype=BF16) for s in ((4, 8), (6, 8), (6,), (4, 6)))
    table, ids = torch.ones(5, 8), torch.zeros(3, dtype=torch.int64)
    with fwd.dual_level():
        dual = [fwd.make_dual(t, torch.ones_like(t)) for t in (x, w, b, r)]
        for i in range(4):
            args = [d if j == i else t for j, (t, d) in enumerate(zip((x, w, b, r), dual))]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                P.linear_act(*args[:3], residual=args[3], activation="gelu")
            with pytest.raises(NotImplementedError, match="forward-mode"), torch.no_grad():
                P.linear_act(*args[:3], residual=args[3], activation="gelu")
        with pytest.raises(NotImplementedError, match="forward-mode"):
            P.embedding_lookup(fwd.make_dual(table, torch.ones_like(table)), ids)
        g = fwd.make_dual(table, torch.ones_like(table))
        for call in (lambda: P.grad_norm([table, g]), lambda: P.clip_grads([g], 1.0), lambda: P.clip_grads([table], 1.0, out=[g])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(P._lib.PlnlpHipError):          # (operands without a tangent go on as ever: there is no CPU path)
            P.linear_act(x, w, b, residual=r)


@gpu
def test_operands_without_a_tangent_inside_a_dual_level(P):
    import torch.autograd.forward_ad as fwd
    x, w = whole((4, 8), BF16, 1), whole((6, 8), BF16, 2)
    want = P.linear_act(x, w)
    with fwd.dual_level():
        assert torch.equal(P.linear_act(x, w), want)


@gpu
def test_clip_refuses_an_expanded_tensor_before_it_writes(P):
    """a tensor whose elements share memory cannot be written: the call is refused as a whole, the other tensors stay as they were"""
    a, one = torch.ones(40, device="cuda"), torch.ones(1, 3, dtype=BF16, device="cuda")
    for grads, out in (([a, one.expand(5, 3)], None), ([a, a.clone()], [a.clone(), torch.zeros(1, device="cuda").expand(40)]),
                       ([one.expand(5, 3)], None)):
        keep = [g.clone() for g in grads + (out or [])]
        with pytest.raises(ValueError, match="share memory"):
            P.clip_grads(grads, 0.5, out=out)
        assert all(torch.equal(g, k) for g, k in zip(grads + (out or []), keep))
    out = [torch.zeros(5, 3, device="cuda")]                       # (read, it counts as the elements it shows)
    assert float(P.clip_grads([one.expand(5, 3)], 1.0, out=out)) == pytest.approx(math.sqrt(15), rel=1e-6)
    assert float(out[0].norm()) == pytest.approx(1.0, rel=1e-5)
    P.clip_grads([torch.ones(0, 3, device="cuda").expand(0, 3), torch.ones(1, 1, device="cuda").expand(1, 1)], 1.0)      # nothing shared
    a = torch.arange(240, device="cuda").float().view(30, 8)
    want = a.clone()
    n = P.clip_grads([a.t(), a[3:5]], 1.0)                         # a strided view and a part of its memory: scaled once, from the old values
    ref = math.sqrt(float(want.double().square().sum() + want[3:5].double().square().sum()))
    assert float(n) == pytest.approx(ref, rel=1e-6)
    assert float((a.double() - want.double() / (ref + 1e-6)).abs().max()) <= 4 * U[F32]          # (elements below 1; factor and product in f32)


# ------------------------------------------------------------------ the lookup's gradient over many ids ------
# 2^20 ids and more (the sort's larger tiles), tables whose keys take one, two and three passes; a third of the batch is one id, whose run
# crosses many ranges, some ids lie outside.  dy is small whole numbers: every sum is exact and rounded once.
@gpu
@pytest.mark.parametrize("n", [2 ** 20, 2 ** 20 + 1, 3000017])
@pytest.mark.parametrize("rows", [1500, 300007, 4300001])
@pytest.mark.parametrize("width,id_t", [(8, torch.int64), (5, torch.int32), (40, torch.int64)])
@pytest.mark.parametrize("frequent", [False, True])
def test_lookup_gradient_of_many_ids(P, n, rows, width, id_t, frequent):
    ids = torch.randint(-3, rows + 3, (n,), generator=generator(n + rows), device="cuda")
    if frequent:
        ids[torch.rand(n, generator=generator(7), device="cuda") < 1 / 3] = rows // 2
    gy = whole((n, width), BF16, 5, -3, 3)
    table = torch.zeros(rows, width, device="cuda", requires_grad=True)
    got, = torch.autograd.grad(P.embedding_lookup(table, ids.to(id_t), padding_idx=rows - 1, out_dtype=BF16), [table], gy)
    ok = (ids >= 0) & (ids < rows - 1)
    want = torch.zeros(rows, width, dtype=torch.int64, device="cuda").index_add_(0, ids[ok], gy.long()[ok])
    assert int(want.abs().max()) < 2 ** 24
    assert torch.equal(got.long(), want)
