"""The 16-bit operators (plnlp_amd/mixed.py) against plain float64 formulas.

Tolerances are bounds of the arithmetic, written down per test: u = finfo(type).eps / 2 is the largest relative error of one rounding
to the stored type, TINY[type] the largest absolute one below its normal range, and a sum of c terms held in f32 is off by at most
c * 2^-23 of the sum of their magnitudes (2^-24 an addition if it rounds to nearest; the matrix cores promise no more than
faithful)."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {t: torch.finfo(t).eps / 2 for t in (F32, BF16, F16)}
TINY = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for t in (F32, BF16, F16)}
ADD = 2.0 ** -23


@pytest.fixture(scope="module")
def P():
    import plnlp_amd
    from plnlp_amd import _lib
    _lib.load()
    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    return plnlp_amd


def within(got, want, bound):
    assert got.shape == want.shape
    over = (got.double() - want).abs() - bound
    assert not bool(torch.isnan(over).any()) and float(over.max() if over.numel() else 0) <= 0.0, float(over.max())


def rand(shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


# ------------------------------------------------------------------ lookup ------
def lookup_ref(table, ids, scale):
    v = table.shape[0]
    ok = (ids >= 0) & (ids < v)
    rows = torch.zeros(v + 1, table.shape[1], dtype=torch.float64, device=table.device)
    rows[:v] = table.double() * scale
    return rows[torch.where(ok, ids.long(), torch.full_like(ids.long(), v))]


def lookup_grad_ref(gy, ids, v, scale, padding=None):
    """(gradient, sum of magnitudes, ids per row) in float64"""
    flat, g = ids.reshape(-1).long(), gy.reshape(ids.numel(), gy.shape[-1]).double()
    ok = (flat >= 0) & (flat < v)
    if padding is not None:
        ok &= flat != padding
    flat, g = flat[ok], g[ok]
    out = torch.zeros(v, gy.shape[-1], dtype=torch.float64, device=gy.device).index_add_(0, flat, g) * scale
    mag = torch.zeros_like(out).index_add_(0, flat, g.abs()) * abs(scale)
    return out, mag, torch.bincount(flat, minlength=v).double()[:, None]


# widths: one element, odd, even without 16-byte rows, one pack, several packs a lane; ids: none, one, a wave, the most that are
# placed in one launch and one more, several counting tiles
@gpu
@pytest.mark.parametrize("n_ids,rows,width", [(0, 5, 8), (1, 1, 1), (1, 7, 3), (3, 300, 50), (64, 65, 64), (257, 1000, 8), (4096, 100, 33),
                                              (4097, 3, 256), (5000, 70001, 40), (8192, 9001, 33), (8193, 40, 5), (20000, 2047, 17), (20000, 2048, 24), (9000, 4200000, 2),
                                              (70000, 500, 1100)])
@pytest.mark.parametrize("table_t,out_t,id_t", [(BF16, BF16, torch.int64), (F16, F16, torch.int32), (F32, BF16, torch.int32), (F32, F32, torch.int64)])
def test_lookup(P, n_ids, rows, width, table_t, out_t, id_t):
    g = torch.Generator(device="cuda").manual_seed(n_ids + width)
    table = rand((rows, width), table_t, 1).requires_grad_(True)
    ids = torch.randint(-2, rows + 2, (n_ids,), generator=g, device="cuda").to(id_t)       # a few outside the table
    gy = rand((n_ids, width), out_t, 2)
    y = P.embedding_lookup(table, ids, scale=0.37, out_dtype=out_t)
    want = lookup_ref(table.detach(), ids, 0.37)
    # scale is rounded to f32, the product in f32, then to the type
    within(y.detach(), want, want.abs() * (U[out_t] + 2 * U[F32]) + TINY[out_t])
    got, = torch.autograd.grad(y, [table], gy)
    ref, mag, count = lookup_grad_ref(gy, ids, rows, 0.37)
    assert got.dtype == table_t and got.shape == table.shape
    within(got, ref, ref.abs() * U[table_t] + mag * (count + 4) * ADD + TINY[table_t])


# a frequent id: runs longer than the pieces that are summed beforehand, beginning and ending inside one; the rest spread
@gpu
@pytest.mark.parametrize("width,dtype", [(8, BF16), (96, F32), (1024, BF16), (7, F16)])
@pytest.mark.parametrize("run", [511, 512, 513, 900, 6001])
def test_lookup_gradient_of_a_frequent_id(P, width, dtype, run):
    g = torch.Generator(device="cuda").manual_seed(run)
    ids = torch.cat([torch.full((run,), 41, device="cuda"), torch.randint(0, 90, (1500,), generator=g, device="cuda"),
                     torch.full((700,), -1, device="cuda"), torch.full((900,), 77, device="cuda")])
    ids = ids[torch.randperm(ids.numel(), generator=g, device="cuda")]
    table = torch.zeros(90, width, dtype=dtype, device="cuda", requires_grad=True)
    gy = rand((ids.numel(), width), dtype, 3, 0.1)
    for padding in (None, 77):
        y = P.embedding_lookup(table, ids, padding_idx=padding)
        got, = torch.autograd.grad(y, [table], gy)
        ref, mag, count = lookup_grad_ref(gy, ids, 90, 1.0, padding)
        within(got, ref, ref.abs() * U[dtype] + mag * (count + 4) * ADD + TINY[dtype])
        if padding is not None:
            assert not bool(got[padding].any())
        again, = torch.autograd.grad(P.embedding_lookup(table, ids, padding_idx=padding), [table], gy)
        assert torch.equal(got, again)                       # the same bits every time


@gpu
def test_lookup_all_ids_equal_none_valid_and_padding(P):
    table = rand((6, 16), BF16, 4).requires_grad_(True)
    gy = rand((3000, 16), BF16, 5)
    for ids, padding in ((torch.full((3000,), 5, device="cuda"), None), (torch.full((3000,), -1, device="cuda"), None),
                         (torch.full((3000,), 5, device="cuda"), -1)):
        y = P.embedding_lookup(table, ids, padding_idx=padding)
        assert torch.equal(y.detach(), lookup_ref(table.detach(), ids, 1.0).to(BF16))       # (the padding row is read like any other)
        got, = torch.autograd.grad(y, [table], gy)
        ref, mag, count = lookup_grad_ref(gy, ids, 6, 1.0, None if padding is None else padding % 6)
        within(got, ref, ref.abs() * U[BF16] + mag * (count + 4) * ADD)


@gpu
def test_lookup_strides_shapes_and_neighbours(P):
    """a table kept padded, ids of two dimensions that are a transposed view, an unaligned gradient, a gradient that is an expanded
    scalar; NaN in an unread row stays there; memory around the result is left as it was"""
    big = rand((50, 24), F32, 6)
    big[13] = math.nan
    table = big[:, 3:21].detach().requires_grad_(True)       # 18 columns, rows 24 apart, 12 bytes off
    ids = torch.arange(12, device="cuda").view(4, 3).t()
    y = P.embedding_lookup(table, ids, scale=-2.0)
    assert y.shape == (3, 4, 18) and torch.equal(y.detach(), table.detach()[ids] * -2.0)
    gy = rand((3, 4, 19), F32, 7)[..., 1:]
    got, = torch.autograd.grad(y, [table], gy)
    ref, _, _ = lookup_grad_ref(gy, ids, 50, -2.0)
    assert torch.equal(got.double(), ref)                    # one id a row: a product with a power of two is exact
    got, = torch.autograd.grad(P.embedding_lookup(table, ids).sum(), [table])
    assert torch.equal(got, (torch.arange(50, device="cuda") < 12).float()[:, None].expand(50, 18))
    assert P.embedding_lookup(table, torch.zeros(0, 3, dtype=torch.int32, device="cuda")).shape == (0, 3, 18)
    got, = torch.autograd.grad(P.embedding_lookup(table, torch.zeros(0, dtype=torch.int64, device="cuda")).sum(), [table])
    assert got.shape == table.shape and not bool(got.any())
    lib, L = P._lib.load(), P._lib
    grad = torch.full((50, 32), 7.0, device="cuda")
    ws = torch.empty(lib.plnlp_embedding_grad_workspace_bytes(12, 18), dtype=torch.uint8, device="cuda")
    flat, g2 = ids.contiguous(), gy.reshape(12, 18).contiguous()
    assert lib.plnlp_embedding_grad(g2.data_ptr(), 18, 0, flat.data_ptr(), 8, 12, -1, -2.0, grad.data_ptr(), 32, 0, 50, 18, ws.data_ptr(),
                                    ws.numel(), L.stream_ptr()) == 0
    assert torch.equal(grad[:, :18].double(), ref) and bool((grad[:, 18:] == 7.0).all())


@gpu
def test_lookup_past_32_bit_offsets(P):
    """rows whose elements begin past 2^32 bytes and 2^31 elements of the table and of the result's gradient"""
    v, d = 2 ** 21 + 3, 1032
    table = torch.zeros(v, d, dtype=BF16, device="cuda")
    ids = torch.tensor([v - 1, 0, v - 2, 2 ** 21, v - 1], device="cuda")
    table[ids] = rand((5, d), BF16, 8)
    table.requires_grad_(True)
    y = P.embedding_lookup(table, ids)
    assert torch.equal(y.detach(), table.detach()[ids])
    gy = rand((5, d), BF16, 9)
    got, = torch.autograd.grad(y, [table], gy)
    assert torch.equal(got[ids[1:4]], gy[1:4])
    assert torch.equal(got[v - 1], (gy[0].float() + gy[4].float()).to(BF16))
    assert not bool(got[1:1000].any()) and not bool(got[2 ** 21 - 1000:2 ** 21].any())


# ------------------------------------------------------------------ linear ------
def act_ref(z, name):
    """(activation, derivative) in float64"""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        phi = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


# the activation's own error in f32: the fitted normal distribution is good to 4e-6 relative, the exponentials' arguments reach
# |z|^2 / 2 (|z| <= 12 here: 72 * 2^-24 * log2 e) and the reciprocals are good to an ulp: 2e-5 of max(|z|, 1) covers all of them
ACT_ERR = 2e-5
SLOPE_LIP = 1.0        # |act''| is at most 0.8 (gelu, gelu_tanh), 0.5 (silu)
SLOPE_ROUND = 2.0 ** -15       # the slope is kept in steps of 2^-14


def linear_case(P, m, n, k, dtype, act, bias, residual, pad=0, seed=0):
    x = rand((m, k + pad), dtype, seed + 1)[:, :k].detach().requires_grad_(True)
    w = rand((n, k + pad), dtype, seed + 2, 1 / math.sqrt(max(k, 1)))[:, :k].detach().requires_grad_(True)
    b = rand((n,), dtype, seed + 3).requires_grad_(True) if bias else None
    r = rand((m, n + pad), dtype, seed + 4)[:, :n].detach().requires_grad_(True) if residual else None
    gy = rand((m, n), dtype, seed + 5)
    return x, w, b, r, gy


def check_linear(P, x, w, b, r, gy, act, dtype):
    u, tiny = U[dtype], TINY[dtype]
    k = x.shape[1]
    xd, wd = x.detach().double(), w.detach().double()
    z = xd @ wd.t()
    e_z = (xd.abs() @ wd.abs().t()) * (k + 2) * ADD
    if b is not None:
        z = z + b.detach().double()
        e_z = e_z + z.abs() * ADD
    a, slope = act_ref(z, act)
    y_ref = a if r is None else a + r.detach().double()
    err = 0.0 if act in ("none", "relu") else ACT_ERR
    e_y = 1.13 * e_z + err * z.abs().clamp_min(1) + y_ref.abs() * (u + 2 * ADD) + a.abs() * ADD + tiny      # |act'| <= 1.13
    y = P.linear_act(x, w, b, residual=r, activation=act)
    within(y.detach(), y_ref, e_y)
    with torch.no_grad():
        assert torch.equal(P.linear_act(x, w, b, residual=r, activation=act), y)      # the same bits without a graph
    leaves = [t for t in (x, w, b, r) if t is not None]
    got = list(torch.autograd.grad(y, leaves, gy))
    g = gy.double()
    dz = g * slope
    e_dz = torch.zeros_like(dz)
    if act != "none":
        # the slope is taken at z as summed and kept in steps, dz is rounded to the type
        e_dz = g.abs() * (SLOPE_LIP * e_z + SLOPE_ROUND + err * z.abs().clamp_min(1)) + dz.abs() * (u + 2 * ADD) + tiny
        if act == "relu":
            e_dz = torch.zeros_like(dz)                       # (exact: the inputs are small whole numbers there)
    dx, dw = dz @ wd, dz.t() @ xd
    m, n = dz.shape
    within(got[0], dx, e_dz @ wd.abs() + (dz.abs() @ wd.abs()) * (n + 2) * ADD * 1.1 + dx.abs() * u + tiny)
    within(got[1], dw, e_dz.t() @ xd.abs() + (dz.t().abs() @ xd.abs()) * (m + 2) * ADD * 1.1 + dw.abs() * u + tiny)
    if b is not None:
        db = dz.sum(0)
        within(got[2], db, e_dz.sum(0) + dz.abs().sum(0) * (m + 2) * ADD * 1.1 + db.abs() * u + tiny)
    if r is not None:
        assert torch.equal(got[-1], gy)
    for t, gt in zip(leaves, got):
        assert gt.shape == t.shape and gt.dtype == dtype
    return y, got


# rows: one, the few-rows kernel's three sizes and their edges, one tile, ragged tiles, K cut into slices; widths odd, even, whole
# groups of eight, ragged against the 128-wide tile; depths below, at and past a 64-step
LINEAR_SHAPES = [(32, 1024, 4104), (64, 2049, 2056), (1, 1, 1), (1, 16, 64), (1, 200, 4096), (3, 17, 72), (16, 256, 256), (17, 40, 1024), (32, 8, 8), (33, 136, 520), (64, 128, 128),
                 (65, 128, 128), (100, 64, 64), (128, 128, 64), (129, 130, 65), (300, 520, 8), (257, 72, 2056), (777, 515, 130), (5, 515, 1003),
                 (1500, 200, 200), (4000, 24, 48)]
# many rows and weights that fit LDS: full and ragged groups of 64 columns, K of whole and ragged 32-pieces up to the deepest taken
# (and the first that is not), rows that end inside a group of 16; the last two fall back for their strides and widths
MANY_ROWS = [(8192, 256, 256), (8200, 200, 72), (10007, 8, 8), (9000, 136, 264), (8195, 64, 512), (8192, 264, 96), (8300, 512, 64), (8300, 72, 520), (8201, 40, 36), (8209, 33, 64), (32770, 256, 256), (33800, 264, 96), (34000, 72, 264), (9001, 64, 200),
             (65537, 512, 64), (8208, 8, 384)]


@gpu
@pytest.mark.parametrize("m,n,k", LINEAR_SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_shapes(P, m, n, k, dtype):
    act = ("gelu", "silu", "none", "gelu_tanh")[(m + n + k) % 4]
    check_linear(P, *linear_case(P, m, n, k, dtype, act, True, True), act, dtype)


@gpu
@pytest.mark.parametrize("m,n,k", MANY_ROWS)
@pytest.mark.parametrize("dtype,act,pad", [(BF16, "gelu", 0), (F16, "silu", 8), (BF16, "none", 0), (F16, "gelu_tanh", 3)])
def test_linear_many_rows(P, m, n, k, dtype, act, pad):
    check_linear(P, *linear_case(P, m, n, k, dtype, act, True, (m + pad) % 2 == 0, pad), act, dtype)


@gpu
def test_linear_many_rows_some_gradients(P):
    """each gradient alone: which of them brings the others' sums differs"""
    x, w, b, r, gy = linear_case(P, 8500, 96, 64, BF16, "silu", True, True)
    full = torch.autograd.grad(P.linear_act(x, w, b, residual=r, activation="silu"), [x, w, b, r], gy)
    for i, leaf in enumerate((x, w, b, r)):
        args = [t if j == i else t.detach() for j, t in enumerate((x, w, b, r))]
        got, = torch.autograd.grad(P.linear_act(*args[:3], residual=args[3], activation="silu"), [leaf], gy)
        if i == 2:        # summed in another order
            within(got, full[2].double(), (gy.double().abs() * 1.13).sum(0) * 8502 * ADD + 2 * U[BF16] * full[2].double().abs())
        else:
            assert torch.equal(got, full[i])


@gpu
@pytest.mark.parametrize("act", ["none", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("m,n,k,pad", [(20, 64, 64, 0), (200, 96, 136, 8), (200, 96, 136, 3)])
def test_linear_epilogues_and_strides(P, act, bias, residual, m, n, k, pad):
    check_linear(P, *linear_case(P, m, n, k, BF16, act, bias, residual, pad), act, BF16)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,k", [(8, 64, 64), (150, 130, 66), (700, 128, 256)])
def test_linear_relu_at_its_border(P, m, n, k, dtype):
    """whole numbers: z is exact, often 0 (slope 0 there), and so is every gradient below 2^24 before its one rounding"""
    g = torch.Generator(device="cuda").manual_seed(k)
    x, w, b, gy = (torch.randint(-1, 2, s, generator=g, device="cuda").to(dtype) for s in ((m, k), (n, k), (n,), (m, n)))
    z = x.double() @ w.double().t() + b.double()
    assert bool((z == 0).any())
    check_linear(P, *(t.requires_grad_(True) for t in (x, w, b)), None, gy, "relu", dtype)


@gpu
@pytest.mark.parametrize("m,n,k,dtype", [(16384, 1024, 512, BF16), (16390, 1280, 576, F16), (12552, 1000, 1032, BF16), (1792, 8200, 520, F16),
                                         (512, 2048, 3000, BF16)])
def test_linear_large_tiles(P, m, n, k, dtype):
    """the 256 x 256 tiles, forward and both gradients, alone and with K in slices, with ragged rows, columns and depths; dx checked on
    sampled rows"""
    x, w, b, r, gy = linear_case(P, m, n, k, dtype, "silu", True, True)
    y = P.linear_act(x, w, b, residual=r, activation="silu")
    dx, dw, db, dr = torch.autograd.grad(y, [x, w, b, r], gy)
    u, tiny = U[dtype], TINY[dtype]
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.cat([torch.tensor([0, m - 1, m - 2], device="cuda"), torch.randint(0, m, (253,), generator=g, device="cuda")])
    xd, wd = x.detach().double(), w.detach().double()
    z = xd @ wd.t() + b.detach().double()
    a, slope = act_ref(z, "silu")
    e_z = (xd.abs() @ wd.abs().t()) * (k + 3) * ADD
    y_ref = a + r.detach().double()
    within(y.detach()[rows], y_ref[rows], (1.13 * e_z + ACT_ERR * z.abs().clamp_min(1) + y_ref.abs() * (u + 2 * ADD) + a.abs() * ADD + tiny)[rows])
    gd = gy.double()
    dz = gd * slope
    e_dz = gd.abs() * (SLOPE_LIP * e_z + SLOPE_ROUND + ACT_ERR * z.abs().clamp_min(1)) + dz.abs() * (u + 2 * ADD) + tiny
    ref = dz[rows] @ wd
    within(dx[rows], ref, e_dz[rows] @ wd.abs() + (dz[rows].abs() @ wd.abs()) * (n + 2) * ADD * 1.1 + ref.abs() * u + tiny)
    ref = dz.t() @ xd
    within(dw, ref, e_dz.t() @ xd.abs() + (dz.t().abs() @ xd.abs()) * (m + 2) * ADD * 1.1 + ref.abs() * u + tiny)
    ref = dz.sum(0)
    within(db, ref, e_dz.sum(0) + dz.abs().sum(0) * (m + 2) * ADD * 1.1 + ref.abs() * u + tiny)
    assert torch.equal(dr, gy)


@gpu
def test_linear_against_differences(P):
    """the gradients of a smooth layer against central differences of the float64 formula along random directions"""
    x, w, b, r, gy = linear_case(P, 40, 48, 56, F16, "gelu", True, True)
    got = torch.autograd.grad(P.linear_act(x, w, b, residual=r, activation="gelu"), [x, w, b, r], gy)

    def f(x, w, b, r):
        return ((act_ref(x @ w.t() + b, "gelu")[0] + r) * gy.double()).sum()
    at = [t.detach().double() for t in (x, w, b, r)]
    for i, t in enumerate(at):
        d = rand(t.shape, F32, 60 + i).double()
        step = 1e-5
        hi, lo = list(at), list(at)
        hi[i], lo[i] = t + step * d, t - step * d
        want = float((f(*hi) - f(*lo)) / (2 * step))
        # each element of a gradient is off by u of itself and by what the 16-bit dz carries into it (a few u of its terms)
        assert abs(float((got[i].double() * d).sum()) - want) <= 8 * U[F16] * float((got[i].double().abs() * d.abs()).sum()) + 1e-6


@gpu
def test_linear_shapes_of_more_dimensions_and_empty_ones(P):
    w, b = rand((24, 16), BF16, 1).requires_grad_(True), rand((24,), BF16, 2).requires_grad_(True)
    x, r = rand((2, 3, 16), BF16, 3), rand((2, 3, 24), BF16, 4)
    y = P.linear_act(x, w, b, residual=r, activation="silu")
    assert y.shape == (2, 3, 24) and torch.equal(y.view(6, 24), P.linear_act(x.view(6, 16), w, b, residual=r.view(6, 24), activation="silu"))
    assert P.linear_act(x[0, 0], w, b).shape == (24,)
    empty = torch.zeros(0, 16, dtype=BF16, device="cuda", requires_grad=True)
    y = P.linear_act(empty, w, b, activation="gelu")
    dx, dw, db = torch.autograd.grad(y, [empty, w, b], torch.zeros_like(y))
    assert y.shape == (0, 24) and dx.shape == (0, 16) and not bool(dw.any()) and not bool(db.any())
    x0, w0 = torch.zeros(5, 0, dtype=BF16, device="cuda"), torch.zeros(24, 0, dtype=BF16, device="cuda")
    assert torch.equal(P.linear_act(x0, w0, b), b.detach().expand(5, 24))
    none = torch.zeros(0, 16, dtype=BF16, device="cuda", requires_grad=True)          # a layer without outputs
    some = x.view(6, 16).clone().requires_grad_(True)
    y = P.linear_act(some, none, activation="gelu")
    dx, dw = torch.autograd.grad(y, [some, none], torch.zeros_like(y))
    assert y.shape == (6, 0) and dx.shape == (6, 16) and not bool(dx.any()) and dw.shape == (0, 16)
    # a bias and a residual shared by broadcasting: the caller expands, autograd sums
    one = rand((1, 24), BF16, 5).requires_grad_(True)
    y = P.linear_act(x.view(6, 16), w, b, residual=one.expand(6, 24))
    got, = torch.autograd.grad(y, [one], torch.ones_like(y))
    assert torch.equal(got, torch.full_like(got, 6.0))
    # only some gradients wanted
    y = P.linear_act(x.view(6, 16), w.detach(), b, activation="gelu")
    assert torch.autograd.grad(y.sum(), [b])[0].shape == (24,)


@gpu
@pytest.mark.parametrize("m", [4, 90])
def test_linear_special_values(P, m):
    """NaN and infinity stay in their row; a value past the type's range becomes infinite; far negative arguments of the smooth
    activations come out as their tiny values, not as NaN"""
    for act in ("none", "relu", "gelu", "gelu_tanh", "silu"):
        x = torch.zeros(m, 64, dtype=BF16, device="cuda")
        x[1, 0], x[2, 0], x[3, 0] = math.nan, math.inf, -60.0
        w = torch.ones(32, 64, dtype=BF16, device="cuda")
        y = P.linear_act(x, w, activation=act)
        assert bool(torch.isnan(y[1]).all()) and bool((y[2] == math.inf).all()) and not bool(y[0].any()) and not bool(y[4:].any())
        assert bool((y[3] == -60).all()) if act == "none" else float(y[3].abs().max()) <= 1e-20
    big = torch.full((m, 64), 30000.0, dtype=F16, device="cuda")
    assert bool((P.linear_act(big, torch.ones(8, 64, dtype=F16, device="cuda")) == math.inf).all())
    # columns and depths past the matrix are not read into it: the memory around x and w holds NaN
    xb = torch.full((m + 2, 80), math.nan, dtype=BF16, device="cuda")
    wb = torch.full((40, 80), math.nan, dtype=BF16, device="cuda")
    xb[1:m + 1, 8:32], wb[1:34, 8:32] = 1.0, 1.0
    y = P.linear_act(xb[1:m + 1, 8:32], wb[1:34, 8:32])
    assert bool((y == 24).all())


# ------------------------------------------------------------------ clipping ----
def norm_ref(grads, p):
    parts = [g.double().abs().reshape(-1) for g in grads]
    v = torch.cat(parts) if parts else torch.zeros(0, dtype=torch.float64)
    if v.numel() == 0:
        return 0.0
    return float(v.max()) if p == math.inf else float((v ** p).sum() ** (1 / p))


def grad_list(sizes, types, seed, std=0.1):
    return [rand(s, types[i % len(types)], seed + i, std) for i, s in enumerate(sizes)]


SIZES = {"one": [(1,)], "odd": [(7,), (1, 1), (0,), (13, 5), (4097,), (8191,)], "wide": [(300, 257), (100000,), (3,)],
         "many": [(i % 40 + 1,) for i in range(400)]}


@gpu
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("types", [[BF16], [F16], [F32], [F32, BF16, F16]])
@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_clip(P, sizes, types, p):
    grads = grad_list(SIZES[sizes], types, 1)
    ref = norm_ref(grads, p)
    for limit in (0.3 * ref, 2 * ref):
        coef = min(1.0, limit / (ref + 1e-6))
        wide = [torch.full_like(g, math.nan, dtype=F32) for g in grads]
        n = P.clip_grads(grads, limit, norm_type=p, out=wide)
        assert n.dtype == F32 and n.dim() == 0
        assert abs(float(n) - ref) <= ref * 2 * U[F32]       # f64 sums, rounded to f32 once
        assert float(P.grad_norm(grads, norm_type=p)) == float(n)
        for g, o in zip(grads, wide):                         # the factor and the product in f32
            within(o, g.double() * coef, g.double().abs() * coef * 4 * U[F32])
        mine = [g.clone() for g in grads]
        n2 = P.clip_grads(mine, limit, norm_type=p)
        assert float(n2) == float(n)
        for g, o, c in zip(grads, wide, mine):
            assert torch.equal(c, o.to(g.dtype))              # in place: the same values, rounded once
            if coef == 1.0:
                assert torch.equal(c, g)


@gpu
def test_clip_special_values(P):
    for t, v, kind in ((F32, math.nan, "nan"), (BF16, math.inf, "inf"), (F16, -math.inf, "inf"), (BF16, math.nan, "nan")):
        for p in (2.0, 1.0, math.inf):
            g = [torch.ones(5000, dtype=t, device="cuda"), torch.ones(3, dtype=F32, device="cuda")]
            g[0][4321] = v
            n = float(P.clip_grads(g, 1.0, norm_type=p))
            if kind == "nan":
                assert math.isnan(n) and all(bool(torch.isnan(x).all()) for x in g)
            else:
                assert n == math.inf and not bool(g[1].any()) and bool(torch.isnan(g[0][4321])) and int((g[0] == 0).sum()) == 4999
    # squares that leave f32's range on both sides
    assert abs(float(P.grad_norm([torch.full((4,), 1e30, device="cuda")])) / 2e30 - 1) < 1e-6
    assert abs(float(P.grad_norm([torch.full((4,), 1e-30, device="cuda")])) / 2e-30 - 1) < 1e-6
    g = [torch.ones(10, dtype=BF16, device="cuda")]
    assert float(P.clip_grads(g, 0.0)) == pytest.approx(math.sqrt(10)) and not bool(g[0].any())
    g = [torch.ones(10, dtype=BF16, device="cuda")]
    P.clip_grads(g, math.inf)
    assert bool((g[0] == 1).all())
    assert float(P.clip_grads([], 1.0)) == 0.0 and float(P.grad_norm([torch.zeros(0, device="cuda")])) == 0.0


@gpu
def test_clip_views_alignment_and_neighbours(P):
    """tensors that begin anywhere in a buffer and end before its other values; transposed and strided ones"""
    for t in (BF16, F16, F32):
        for off in range(0, 9):
            buf = rand((5000,), t, off)
            keep = buf.clone()
            out = torch.full((5100,), 9.0, dtype=F32, device="cuda")
            n = P.clip_grads([buf[off:off + 4321]], 0.5, out=[out[off + 1:off + 4322]])
            ref = norm_ref([buf[off:off + 4321]], 2.0)
            assert abs(float(n) - ref) <= ref * 2 * U[F32]
            assert bool((out[:off + 1] == 9).all()) and bool((out[off + 4322:] == 9).all()) and torch.equal(buf, keep)
            P.clip_grads([buf[off:off + 4321]], 0.5)
            assert torch.equal(buf[off:off + 4321], out[off + 1:off + 4322].to(t))
            assert torch.equal(buf[:off], keep[:off]) and torch.equal(buf[off + 4321:], keep[off + 4321:])
    a = rand((40, 30), F32, 3)
    views = [a.t()[:, 5:20], a[:, 25:]]                       # strided views of one buffer that do not overlap
    want = [v.clone() for v in views]
    n = P.clip_grads(views, 0.1)
    plain = [v.contiguous() for v in want]
    assert float(P.clip_grads(plain, 0.1)) == float(n)
    for v, q in zip(views, plain):
        assert torch.equal(v, q)


# rows of the gradient apart from each other and at every alignment; dE cleared beside the sort (few ids) or behind it (many); what lies
# between the rows and around them stays
@gpu
@pytest.mark.parametrize("n_ids,rows", [(0, 70), (5, 700), (60, 70), (9000, 30000), (9000, 300)])
@pytest.mark.parametrize("width,ld,shift", [(8, 8, 0), (7, 7, 0), (7, 7, 1), (24, 32, 0), (33, 40, 3), (64, 66, 2), (5, 4100, 1)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_lookup_gradient_between_other_memory(P, n_ids, rows, width, ld, shift, dtype):
    from plnlp_amd import _lib as L
    lib, code = L.load(), L.DTYPE_CODES[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    ids = torch.randint(-1, rows + 1, (n_ids,), generator=g, device="cuda")
    gy = rand((n_ids, width), dtype, 3)
    memory = torch.full((rows * ld + 64,), 7.0, dtype=dtype, device="cuda")
    ws = torch.empty(lib.plnlp_embedding_grad_workspace_bytes(n_ids, width) + 16, dtype=torch.uint8, device="cuda")
    grad = memory[shift:shift + rows * ld].view(rows, ld)
    for _ in range(2):                                      # (over the first call's result as well)
        L.check(lib.plnlp_embedding_grad(gy.data_ptr(), width, code, ids.data_ptr(), 8, n_ids, 2, 0.5, grad.data_ptr(), ld, code, rows, width,
                                         ws.data_ptr(), ws.numel(), L.stream_ptr()), "grad")
        ref, mag, count = lookup_grad_ref(gy, ids, rows, 0.5, padding=2)
        within(grad[:, :width], ref, ref.abs() * U[dtype] + mag * (count + 4) * ADD + TINY[dtype])
        assert bool((grad[:, width:] == 7).all()) and bool((memory[:shift] == 7).all()) and bool((memory[shift + rows * ld:] == 7).all())


# more workgroups than one dimension of a grid takes (2^32 threads): rows too narrow to share one, too wide for several
@gpu
def test_lookup_of_many_rows(P):
    n = 2 ** 26 + 5
    table = rand((1000, 129), BF16, 8)
    ids = torch.randint(0, 1000, (n,), generator=torch.Generator(device="cuda").manual_seed(9), device="cuda", dtype=torch.int32)
    y = P.embedding_lookup(table, ids)
    for lo in range(0, n, 2 ** 22):                      # (scale 1: copies)
        part = y[lo:lo + 2 ** 22]
        assert torch.equal(part, table[ids[lo:lo + 2 ** 22].long()]), lo


@gpu
def test_clip_refuses_what_it_would_scale_twice(P):
    a, b = rand((30, 8), BF16, 1), rand((20,), F32, 2)
    for grads, out in (([a, b, a], None), ([a.t(), a.t()], None), ([a[:, ::2], a[:, ::2]], None), ([a, a[3:5]], None),
                       ([a, b], [b.new_empty(240), a.view(-1)[:20]])):
        keep = [g.clone() for g in grads]
        with pytest.raises(ValueError):
            P.clip_grads(grads, 0.1, out=out)
        assert all(torch.equal(g, k) for g, k in zip(grads, keep))
    with torch.inference_mode():
        c = torch.ones(10, device="cuda")
        P.clip_grads([c], 1.0)
        assert float(c.norm()) == pytest.approx(1.0, abs=1e-5)
    version = a._version
    P.clip_grads([a], 0.1)
    assert a._version > version                               # autograd is told that the gradient changed


@gpu
def test_clip_more_partials_than_a_workgroup_joins(P):
    grads = [torch.full((1,), 0.5, dtype=(BF16, F32)[i % 2], device="cuda") for i in range(4300)]
    want = 0.5 * math.sqrt(4300)
    n = P.clip_grads(grads, 1.0)
    assert abs(float(n) - want) <= want * 2 * U[F32]
    c = torch.tensor(0.5 / (want + 1e-6))
    assert all(abs(float(g) - float(c)) <= float(c) * 4 * U[g.dtype] for g in grads[::97])


@gpu
def test_clip_of_parameters(P):
    from plnlp_amd.optim import clip_grad_norm_
    ps = [torch.nn.Parameter(rand((30, 7), t, i)) for i, t in enumerate((BF16, F32, F16))]
    assert float(clip_grad_norm_(ps, 1.0)) == 0.0
    for i, p in enumerate(ps[:2]):
        p.grad = rand((30, 7), p.dtype, 10 + i)
    ref = norm_ref([p.grad for p in ps[:2]], 2.0)
    assert float(clip_grad_norm_(iter(ps), 1.0)) == pytest.approx(ref, rel=2e-7)
    assert norm_ref([p.grad for p in ps[:2]], 2.0) <= 1.0 + 2 * U[BF16]
    assert float(clip_grad_norm_(ps[0], 5.0, norm_type=math.inf)) == float(ps[0].grad.abs().max())


# ------------------------------------------------------------------ together ----
@gpu
def test_a_training_step_of_all_three(P):
    """endpoint rows of an fp32 table in bf16 -> a residual layer -> a head -> squared loss; gradients of the working copies, clipped into
    fp32 ones, stepped by FusedAdam.  The gradients against the same formulas in float64 on the same 16-bit weights: between the table and
    a gradient lie eight tensors that are rounded to bf16 (rows, z, y, score, and four gradients on the way back), each by at most u of its
    elements, and no map of the step enlarges a relative change by more than a factor of two (its products sum terms of random sign)."""
    from plnlp_amd.optim import FusedAdam
    torch.manual_seed(0)
    table = torch.nn.Parameter(rand((500, 48), F32, 1, 0.5))
    emb = P.ScaledEmbedding(500, 48, scale=1.5, dtype=F32, out_dtype=BF16).cuda()
    emb.weight = table
    hidden, head = P.LinearAct(48, 48, activation="gelu").cuda(), P.LinearAct(48, 1, bias=False).cuda()
    work = [hidden.lin.weight, hidden.lin.bias, head.lin.weight]
    master = [torch.nn.Parameter(w.detach().float()) for w in work]
    opt = FusedAdam(master + [table], lr=0.01)
    src, dst = (torch.randint(0, 500, (700,), generator=torch.Generator(device="cuda").manual_seed(s), device="cuda") for s in (2, 3))
    target = rand((700, 1), F32, 4)

    def loss64(table, w1, b1, w2):
        x = table[src] * 1.5 + table[dst] * 1.5
        y = act_ref(x @ w1.t() + b1, "gelu")[0] + x
        return ((y @ w2.t() - target.double()) ** 2).mean()

    for step in range(3):
        leaves = [t.detach().double().requires_grad_(True) for t in (table, *work)]
        ref = torch.autograd.grad(loss64(*leaves), leaves)
        x = emb(src) + emb(dst)
        score = head(hidden(x, residual=x))
        loss = ((score.float() - target) ** 2).mean()
        grads = torch.autograd.grad(loss, [table, *work])
        for g, want in zip(grads, ref):
            assert g.shape == want.shape
            assert float((g.double() - want).norm()) <= 16 * U[BF16] * float(want.norm())
        for p, g in zip(master, grads[1:]):
            p.grad = torch.empty_like(p)
        table.grad = torch.empty_like(table)
        norm = P.clip_grads(grads, 0.05, out=[table.grad] + [p.grad for p in master])
        assert abs(float(norm) - norm_ref(grads, 2.0)) <= 2 * U[F32] * norm_ref(grads, 2.0)
        assert norm_ref([table.grad] + [p.grad for p in master], 2.0) <= 0.05 * (1 + 8 * U[F32])
        before = table.detach().clone()
        opt.step()
        assert bool((table.detach() != before)[src].any())
        with torch.no_grad():
            for w, p in zip(work, master):
                w.copy_(p)


@gpu
@pytest.mark.parametrize("n,width", [(5000, 64), (40000, 256), (7, 96), (2048, 1024)])
def test_captured_and_replayed(P, n, width):
    """the three operators with their gradients in one graph, replayed with other inputs and eager work between: eager's bits each time"""
    table = rand((300, width), BF16, 1).requires_grad_(True)
    w, b = rand((width, width), BF16, 2, 0.1).requires_grad_(True), rand((width,), BF16, 3).requires_grad_(True)
    ids, gy = torch.zeros(n, dtype=torch.int64, device="cuda"), torch.zeros(n, width, dtype=BF16, device="cuda")

    def step():
        x = P.embedding_lookup(table, ids, scale=0.5)
        y = P.linear_act(x, w, b, residual=x, activation="gelu")
        grads = torch.autograd.grad(y, [table, w, b], gy)
        out = [torch.empty_like(g, dtype=F32) for g in grads]
        return [y.detach(), P.clip_grads(grads, 1.0, out=out), *out]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        ids.copy_(torch.randint(-1, 300 if i % 2 else 4, (n,), generator=torch.Generator(device="cuda").manual_seed(i), device="cuda"))
        gy.copy_(rand((n, width), BF16, 20 + i, 0.1))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        eager = step()
        torch.cuda.synchronize()
        for u, v in zip(got, eager):
            assert torch.equal(u, v)


@gpu
def test_gradients_of_gradients_are_refused(P):
    x, w, table = rand((5, 8), BF16, 1).requires_grad_(True), rand((4, 8), BF16, 2).requires_grad_(True), rand((7, 8), BF16, 3).requires_grad_(True)
    for y, leaf in ((P.linear_act(x, w, activation="silu"), x), (P.embedding_lookup(table, torch.arange(3, device="cuda")), table)):
        g, = torch.autograd.grad(y.float().square().sum(), [leaf], create_graph=True)      # (allowed: the gradient itself is right)
        assert bool(torch.isfinite(g).all())
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.float().sum(), [leaf])


@gpu
def test_two_streams_at_once(P):
    """the same calls on two streams, each with its own tensors, give what one stream gives"""
    def work(seed):
        table = rand((5000, 96), BF16, seed).requires_grad_(True)
        ids = torch.randint(0, 5000, (20000,), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
        w = rand((96, 96), BF16, seed + 1, 0.1).requires_grad_(True)
        gy = rand((20000, 96), BF16, seed + 2)
        return table, ids, w, gy

    def run(table, ids, w, gy):
        y = P.linear_act(P.embedding_lookup(table, ids), w, activation="silu")
        g = list(torch.autograd.grad(y, [table, w], gy))
        return [y.detach(), P.clip_grads(g, 1.0), *g]
    a, b = work(1), work(50)
    want = run(*a), run(*b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            ra = run(*a)
        with torch.cuda.stream(s2):
            rb = run(*b)
        torch.cuda.synchronize()
        for got, ref in ((ra, want[0]), (rb, want[1])):
            for u, v in zip(got, ref):
                assert torch.equal(u, v)


# ------------------------------------------------------------------ refusals (no device needed) ----
def test_refusals():
    import plnlp_amd as P
    from plnlp_amd._lib import PlnlpHipError
    x, w = torch.zeros(4, 8, dtype=BF16), torch.zeros(6, 8, dtype=BF16)
    ids = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(TypeError, match="ops.LinearFn"):
        P.linear_act(x.float(), w.float())
    for kw in (dict(weight=torch.zeros(6, 7, dtype=BF16)), dict(bias=torch.zeros(5, dtype=BF16)), dict(residual=torch.zeros(1, 6, dtype=BF16)),
               dict(activation="tanh")):
        with pytest.raises(ValueError):
            P.linear_act(x, **{"weight": w, **kw})
    for kw in (dict(weight=w.half()), dict(bias=torch.zeros(6)), dict(residual=torch.zeros(4, 6))):
        with pytest.raises(TypeError):
            P.linear_act(x, **{"weight": w, **kw})
    with pytest.raises(ValueError):
        P.embedding_lookup(torch.zeros(3), ids)
    with pytest.raises(ValueError):
        P.embedding_lookup(torch.zeros(3, 4, dtype=torch.float64), ids)
    with pytest.raises(ValueError):
        P.embedding_lookup(torch.zeros(3, 4), ids, padding_idx=3)
    with pytest.raises(TypeError):
        P.embedding_lookup(torch.zeros(3, 4), ids.float())
    with pytest.raises(TypeError):
        P.embedding_lookup(torch.zeros(3, 4), ids, out_dtype=torch.float64)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            P.clip_grads([torch.zeros(3)], bad)
    with pytest.raises(ValueError):
        P.clip_grads([torch.zeros(3)], 1.0, norm_type=3)
    with pytest.raises(TypeError):
        P.clip_grads([torch.zeros(3, dtype=torch.float64)], 1.0)
    for call in (lambda: P.linear_act(x, w), lambda: P.embedding_lookup(torch.zeros(3, 4), ids), lambda: P.clip_grads([torch.zeros(3)], 1.0),
                 lambda: P.grad_norm([torch.zeros(3)])):
        with pytest.raises(PlnlpHipError):                   # no CPU path
            call()


def test_overlaps_are_found():
    """the host's check of written ranges, on made-up addresses"""
    import numpy as np
    from plnlp_amd import mixed

    def check(*entries):
        src, dst, n, st, dt = (np.array([e[i] for e in entries], dtype=np.int64) for i in range(5))
        return mixed._overlap(src, dst, n, st, dt)
    F, H = 0, 1                                                              # four bytes, two bytes
    assert not check() and not check((1000, 1000, 10, F, F), (1040, 1040, 10, F, F))          # in place, side by side
    assert not check((1000, 2000, 10, H, F), (1010, 2040, 10, H, F))         # sources may overlap: they are only read
    assert not check((1000, 1000, 10, F, F), (1000, 1000, 0, F, F))          # nothing in an empty one
    assert not check((1000, 3000, 10, H, F), (5000, 5000, 4, F, F))
    assert check((1000, 1000, 10, F, F), (1000, 1000, 10, F, F))             # listed twice
    assert check((1000, 1000, 10, F, F), (1036, 1036, 10, F, F))
    assert check((1000, 2000, 10, F, F), (1100, 2039, 10, F, F))             # written ranges overlap
    assert check((1000, 1020, 10, F, F)) and check((1020, 1000, 10, F, F))   # its own source, shifted
    assert check((1000, 2000, 10, F, F), (2000, 3000, 10, F, F))             # one's result over another's source
    assert check((2036, 3000, 10, F, F), (1000, 2000, 10, F, F))


def test_argument_checks_of_the_library():
    """each call is refused before anything is launched (addresses are made up and never read)"""
    from plnlp_amd import _lib as L
    lib = L.load()
    A = 0x10000
    look = lambda **k: lib.plnlp_embedding_lookup(*{**dict(t=A, ld=8, td=1, v=4, w=8, ids=A, ib=8, n=2, s=1.0, o=A, ldo=8, od=1, st=None), **k}.values())
    assert look(n=-1) == -2 and look(ld=7) == -2 and look(ldo=7) == -2 and look(v=2 ** 31) == -2 and look(td=3) == -4 and look(ib=2) == -4
    assert look(t=None) == -1 and look(ids=None) == -1 and look(o=None) == -1 and look(t=A + 1) == -3 and look(ids=A + 4) == -3 and look(n=0) == 0
    grad = lambda **k: lib.plnlp_embedding_grad(*{**dict(g=A, ldg=8, gd=1, ids=A, ib=8, n=5000, p=-1, s=1.0, e=A, lde=8, ed=1, v=9, w=8, ws=A, b=10 ** 7,
                                                         st=None), **k}.values())
    assert grad(b=100) == -5 and grad(ws=None) == -5 and grad(ws=A + 8) == -3 and grad(ldg=7) == -2 and grad(lde=7) == -2 and grad(e=None) == -1
    assert grad(g=None) == -1 and grad(gd=7) == -4 and grad(v=0) == 0 and grad(w=0) == 0
    lin = lambda **k: lib.plnlp_linear_act(*{**dict(x=A, ldx=64, w=A, ldw=64, b=None, r=None, ldr=0, act=0, m=512, n=64, k=64, p=None, ldp=0, o=A, ldo=64,
                                                    d=1, ws=None, wb=0, st=None), **k}.values())
    assert lin(d=0) == -4 and lin(act=9) == -4 and lin(m=-1) == -2 and lin(ldx=63) == -2 and lin(ldo=63) == -2 and lin(x=None) == -1 and lin(o=None) == -1
    assert lin(x=A + 1) == -3 and lin(b=A + 1) == -3 and lin(r=A, ldr=3) == -2 and lin(m=0) == 0
    assert lin(m=512, k=4096, ldx=4096, ldw=4096) == -5      # K is cut: the slices need their workspace
    assert lin(m=2 ** 31) == -2 and lin(n=2 ** 26, ldo=2 ** 26) == -2 and lin(k=2 ** 31, ldx=2 ** 31, ldw=2 ** 31) == -2
    assert lin(m=2 ** 25, n=2 ** 25, ldo=2 ** 25) == -2      # more tiles than a launch holds
    back = lambda **k: lib.plnlp_linear_act_backward(*{**dict(g=A, ldg=64, p=A, ldp=64, act=2, x=A, ldx=64, w=A, ldw=64, m=512, n=64, k=64, dx=A, lddx=64,
                                                              dw=A, lddw=64, db=A, d=1, ws=A, wb=10, st=None), **k}.values())
    assert back() == -5 and back(ws=None) == -5 and back(p=None) == -1 and back(lddx=3) == -2 and back(d=0) == -4 and back(g=None) == -1
    t = (L.GradTensor * 2)()
    for i in range(2):
        t[i].src, t[i].dst, t[i].n, t[i].src_dtype, t[i].dst_dtype = A, A + 64, 8, 1, 0
    clip = lambda n=2, kind=0, m=1.0, ws=A, wd=100, o=A: lib.plnlp_grad_clip(t, n, kind, m, ws, wd, o, None)
    assert lib.plnlp_grad_norm_workspace_doubles(t, 2) == 3
    assert clip(kind=5) == -2 and clip(m=-1.0) == -2 and clip(m=float("nan")) == -2 and clip(wd=2) == -5 and clip(ws=None) == -1 and clip(o=None) == -1
    t[1].dst_dtype = 4
    assert clip() == -4
    t[1].dst_dtype, t[1].dst = 0, A                           # in place, of another type
    assert clip() == -4
    t[1].dst, t[1].src = A + 64, None
    assert clip() == -1
