"""The operators of a training step with 16-bit storage, as a user's program calls them, and their plain forms.

  lookup  -- rows of an embedding table by id, times a scale; its gradient summed by id
             (plnlp_amd.embedding_lookup)
  linear  -- activation(x W^T + bias) + residual, and its gradients (plnlp_amd.linear_act)
  clip    -- the global norm of many gradients, and the gradients clipped by it (plnlp_amd.clip_grads)

`own` chooses between the framework's operators and the plain forms (elementary torch operations in 32 bits,
rounded once at the end)."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # ---- rows of a table by id
        # serving: the two endpoints of a few candidate edges on a small graph's 512-wide table
        dict(name="lookup-serve", op="lookup", train=False, tokens=16, rows=4267, width=512, table="bf16", out="bf16",
             ids="int64", skew=1.0, invalid=0.0, scale=1.0, pad=0),
        # a training batch's positives and negatives (65 536 + 65 536 edges, both endpoints) on a 235 868-node table
        dict(name="lookup-train-batch", op="lookup", train=True, tokens=262144, rows=235868, width=256, table="bf16",
             out="bf16", ids="int64", skew=1.0, invalid=0.0, scale=1.0, pad=0),
        # a 50-wide fp32 master table kept padded to 64 columns, 16-bit rows out, a padded batch (some ids are -1)
        dict(name="lookup-train-narrow", op="lookup", train=True, tokens=131071, rows=1000003, width=50, table="fp32",
             out="bf16", ids="int32", skew=1.5, invalid=0.05, scale=0.5, pad=14),
        # token ids of a skewed vocabulary: the first ids hold a few percent of the batch each
        dict(name="lookup-train-skewed", op="lookup", train=True, tokens=524288, rows=32000, width=1024, table="bf16",
             out="bf16", ids="int64", skew=4.0, invalid=0.0, scale=32.0, pad=0),
        # ---- product with bias, activation and residual
        # one query through one layer of a serving stack: the weights are read once
        dict(name="linear-serve-one", op="linear", train=False, m=1, n=4096, k=4096, dtype="bf16", act="silu", bias=True,
             residual=True, pad=0),
        # a small ragged batch, odd sizes, a strided input
        dict(name="linear-ragged", op="linear", train=False, m=777, n=515, k=1003, dtype="fp16", act="gelu_tanh",
             bias=True, residual=True, pad=5),
        # the edge predictor over a step's 131 072 edges at its width of 256, forward and backward
        dict(name="linear-train-edges", op="linear", train=True, m=131072, n=256, k=256, dtype="bf16", act="gelu",
             bias=True, residual=True, pad=0),
        # a 200-wide layer, forward and backward, in fp16
        dict(name="linear-train-narrow", op="linear", train=True, m=40001, n=200, k=200, dtype="fp16", act="silu",
             bias=True, residual=False, pad=0),
        # a large product, bound by the matrix cores, forward and backward
        dict(name="linear-train-large", op="linear", train=True, m=8192, n=4096, k=4096, dtype="bf16", act="gelu",
             bias=True, residual=True, pad=0),
        # ---- global gradient norm and clipping
        # a small model's gradients, below the limit: the norm alone is needed
        dict(name="clip-small", op="clip", layers=3, hidden=256, rows=1000, dtype="bf16", out="inplace", norm=2.0,
             limit=2.0, align=64),
        # many tensors of a deep stack, 16-bit gradients clipped into 32-bit ones for the optimiser
        dict(name="clip-many", op="clip", layers=150, hidden=300, rows=4267, dtype="mixed", out="fp32", norm=2.0,
             limit=0.3, align=64),
        # a large model: a table's gradient and the layers', clipped
        dict(name="clip-large", op="clip", layers=24, hidden=2048, rows=235868, dtype="bf16", out="same", norm=2.0,
             limit=0.3, align=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "linear", "linear", "clip"])
    while True:
        if op == "lookup":
            case = dict(op=op, train=rng.random() < 0.7, tokens=_log(rng, 1, 524288), rows=_log(rng, 2, 1000003),
                        width=_log(rng, 1, 2048), table=rng.choice(["bf16", "fp16", "fp32"]), out="bf16",
                        ids=rng.choice(["int64", "int32"]), skew=rng.choice([1.0, 1.5, 4.0]),
                        invalid=rng.choice([0.0, 0.05]), scale=rng.choice([1.0, 0.5, 11.3]), pad=rng.choice([0, 0, 3, 8]))
            case["out"] = case["table"] if case["table"] != "fp32" else rng.choice(["fp32", "bf16"])
            if rng.random() < 0.5:
                case["width"] = max(8, case["width"] // 8 * 8)
        elif op == "linear":
            case = dict(op=op, train=rng.random() < 0.5, m=_log(rng, 1, 131072), n=_log(rng, 1, 4096),
                        k=_log(rng, 1, 4096), dtype=rng.choice(["bf16", "fp16"]), act="none",
                        bias=rng.random() < 0.8, residual=rng.random() < 0.5, pad=rng.choice([0, 0, 3, 8]))
            # the derivative of relu jumps where its argument is 0, where every rounding decides: forward cases only
            case["act"] = rng.choice(["none", "gelu", "gelu_tanh", "silu"] + ([] if case["train"] else ["relu"]))
            if rng.random() < 0.6:
                case["n"], case["k"] = max(8, case["n"] // 8 * 8), max(8, case["k"] // 8 * 8)
        else:
            case = dict(op=op, layers=_log(rng, 1, 150), hidden=_log(rng, 8, 2048), rows=_log(rng, 1, 235868),
                        dtype=rng.choice(["bf16", "fp16", "fp32", "mixed"]), out=rng.choice(["same", "fp32", "inplace"]),
                        norm=rng.choice([2.0, 2.0, 1.0, math.inf]), limit=0.3, align=rng.choice([64, 64, 1]))
            if case["out"] == "inplace":
                case["limit"] = 2.0         # (a clipped gradient is not clipped again by the next pass: below the limit)
        w = work(case)
        caps = [work(c) for c in listed() if c["op"] == op]
        if w["bytes"] <= max(c["bytes"] for c in caps) and w["flops"] <= max(c["flops"] for c in caps):
            return case


# ---------------------------------------------------------------- what a user's program has in hand ----------
def _grad_shapes(case):
    h = case["hidden"]
    shapes = [(case["rows"], h)]
    for _ in range(case["layers"]):
        shapes += [(h, h), (h,), (h, h)]
    return shapes


def _grad_dtypes(case, count):
    if case["dtype"] != "mixed":
        return [DTYPES[case["dtype"]]] * count
    return [torch.float32 if i % 3 == 0 else torch.bfloat16 for i in range(count)]      # the table's and one in three


def _buckets(shapes, dtypes, align):
    """the tensors as views of one flat buffer a type, each beginning at a multiple of `align` elements"""
    at, views = {}, []
    for x, dt in zip(shapes, dtypes):
        at[dt] = -(-at.get(dt, 0) // align) * align + math.prod(x)
    flat = {dt: torch.zeros(n, dtype=dt, device="cuda") for dt, n in at.items()}
    at = dict.fromkeys(flat, 0)
    for x, dt in zip(shapes, dtypes):
        lo = -(-at[dt] // align) * align
        at[dt] = lo + math.prod(x)
        views.append(flat[dt][lo:at[dt]].view(x))
    return flat, views


def _randn(shape, gen, std, dtype):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "lookup":
        t, v, d = case["tokens"], case["rows"], case["width"]
        buf = _randn((v, d + case["pad"]), gen, 0.05, DTYPES[case["table"]])
        s["table"] = buf[:, :d]
        u = torch.rand(t, generator=gen, device="cuda", dtype=torch.float64)
        ids = (u.pow(case["skew"]) * v).long().clamp_(0, v - 1)
        if case["invalid"] > 0.0:
            ids[torch.rand(t, generator=gen, device="cuda") < case["invalid"]] = -1
        s["ids"] = ids.to(torch.int64 if case["ids"] == "int64" else torch.int32)
        if case["train"]:
            s["gy"] = _randn((t, d), gen, 0.01, DTYPES[case["out"]])
            s["table"].requires_grad_(True)
    elif case["op"] == "linear":
        m, n, k, dt = case["m"], case["n"], case["k"], DTYPES[case["dtype"]]
        s["x"] = _randn((m, k + case["pad"]), gen, 1.0, dt)[:, :k]
        s["w"] = _randn((n, k), gen, 1.0 / math.sqrt(k), dt)
        s["b"] = _randn((n,), gen, 0.1, dt) if case["bias"] else None
        s["r"] = _randn((m, n), gen, 1.0, dt) if case["residual"] else None
        if case["train"]:
            s["gy"] = _randn((m, n), gen, 0.1, dt)
            for name in ("x", "w", "b", "r"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    else:
        shapes = _grad_shapes(case)
        dts = _grad_dtypes(case, len(shapes))
        count = sum(math.prod(x) for x in shapes)
        s["flat"], s["grads"] = _buckets(shapes, dts, case["align"])
        for g in s["grads"]:
            g.copy_(_randn(g.shape, gen, 0.01, torch.float32))
        expect = {2.0: 0.01 * math.sqrt(count), 1.0: 0.01 * count * math.sqrt(2 / math.pi), math.inf: 0.04}[case["norm"]]
        s["max_norm"] = case["limit"] * expect
        if case["out"] == "inplace":
            s["out"] = None
        else:
            wide = [torch.float32] * len(dts) if case["out"] == "fp32" else dts
            s["flat"], s["out"] = _buckets(shapes, wide, case["align"])
    return s


# ---------------------------------------------------------------- one pass -----------------------------------
def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    with torch.no_grad():
        return {"lookup": _plain_lookup, "linear": _plain_linear, "clip": _plain_clip}[case["op"]](case, state)


def _own(case, s):
    import plnlp_amd as P
    if case["op"] == "lookup":
        y = P.embedding_lookup(s["table"], s["ids"], scale=case["scale"], out_dtype=DTYPES[case["out"]])
        if not case["train"]:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, [s["table"]], s["gy"])]
    if case["op"] == "linear":
        y = P.linear_act(s["x"], s["w"], s["b"], residual=s["r"], activation=case["act"])
        if not case["train"]:
            return [y]
        leaves = [t for t in (s["x"], s["w"], s["b"], s["r"]) if t is not None]
        return [y.detach(), *torch.autograd.grad(y, leaves, s["gy"])]
    norm = P.clip_grads(s["grads"], s["max_norm"], norm_type=case["norm"], out=s["out"])
    return [norm, *s["flat"].values()]


def _plain_lookup(case, s):
    table, ids, v = s["table"], s["ids"].long(), case["rows"]
    valid = (ids >= 0) & (ids < v)
    at = torch.where(valid, ids, torch.zeros_like(ids))
    y = torch.where(valid[:, None], table[at].float() * case["scale"], torch.zeros((), device=ids.device))
    out = [y.to(DTYPES[case["out"]])]
    if case["train"]:
        gy = torch.where(valid[:, None], s["gy"].float(), torch.zeros((), device=ids.device))
        g = torch.zeros(v, case["width"], device=ids.device).index_add_(0, at, gy)
        out.append((g * case["scale"]).to(table.dtype))
    return out


def _act(z, name):
    """the activation and its derivative"""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if name == "silu":
        e = 1.0 / (1.0 + torch.exp(-z))
        return z * e, e * (1.0 + z * (1.0 - e))
    if name == "gelu":
        cdf = 0.5 * torch.erfc(z * -math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    c, a = math.sqrt(2.0 / math.pi), 0.044715
    e = 1.0 / (1.0 + torch.exp(-2.0 * c * (z + a * z * z * z)))
    return z * e, e + z * e * (1.0 - e) * 2.0 * c * (1.0 + 3.0 * a * z * z)


def _plain_linear(case, s):
    dt = DTYPES[case["dtype"]]
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y, dy = _act(z, case["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    out = [y.to(dt)]
    if case["train"]:
        gy = s["gy"]
        dz = gy.float() * dy
        out += [(dz @ w).to(dt), (dz.t() @ x).to(dt)]
        if s["b"] is not None:
            out.append(dz.sum(0).to(dt))
        if s["r"] is not None:
            out.append(gy)
    return out


def _norm_of(grads, kind):
    if kind == math.inf:
        return torch.stack([g.abs().max() for g in grads]).max()
    if kind == 1.0:
        return torch.stack([g.abs().sum() for g in grads]).sum()
    return torch.stack([g.square().sum() for g in grads]).sum().sqrt()


def _plain_clip(case, s):
    wide = [g.float() for g in s["grads"]]
    norm = _norm_of(wide, case["norm"])
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    into = s["grads"] if s["out"] is None else s["out"]
    for o, g in zip(into, wide):
        o.copy_(g * coef)
    return [norm, *s["flat"].values()]


# ---------------------------------------------------------------- what a pass cannot do without --------------
def work(case):
    if case["op"] == "lookup":
        t, v, d = case["tokens"], case["rows"], case["width"]
        idb = 8 if case["ids"] == "int64" else 4
        # rows that t draws touch: every row once where the ids are even, fewer where they are skewed
        touched = v * -math.expm1(-t / v) if case["skew"] == 1.0 else min(t, v)
        b = t * idb + touched * d * BYTES[case["table"]] + t * d * BYTES[case["out"]]
        f = t * d
        if case["train"]:
            b += t * d * BYTES[case["out"]] + v * d * BYTES[case["table"]]
            f += 2 * t * d
        return {"bytes": int(b), "flops": int(f)}
    if case["op"] == "linear":
        m, n, k, e = case["m"], case["n"], case["k"], BYTES[case["dtype"]]
        tensors = m * k + n * k + m * n + (m * n if case["residual"] else 0) + (n if case["bias"] else 0)
        f = 2 * m * n * k
        if case["train"]:
            tensors += m * n + m * k + n * k + (n if case["bias"] else 0)
            f *= 3
        return {"bytes": int(tensors * e), "flops": int(f)}
    shapes = _grad_shapes(case)
    dts = _grad_dtypes(case, len(shapes))
    b = 0
    for x, dt in zip(shapes, dts):
        e = 4 if dt == torch.float32 else 2
        b += math.prod(x) * e
        if case["out"] != "inplace":
            b += math.prod(x) * (4 if case["out"] == "fp32" else e)
    return {"bytes": int(b), "flops": int(3 * sum(math.prod(x) for x in shapes))}


# ---------------------------------------------------------------- the definition, in 64 bits -----------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"lookup": _exact_lookup, "linear": _exact_linear, "clip": _exact_clip}[case["op"]](case, s)


def _exact_lookup(case, s):
    v, d = case["rows"], case["width"]
    ids = s["ids"].long()
    wide = torch.zeros(v + 1, d, dtype=torch.float64, device=ids.device)        # row v stands for every invalid id
    wide[:v] = s["table"].double() * case["scale"]
    row = torch.where((ids < 0) | (ids >= v), torch.full_like(ids, v), ids)
    out = [wide.index_select(0, row)]
    if case["train"]:
        acc = torch.zeros_like(wide)
        for lo in range(0, ids.numel(), 1 << 17):
            acc.index_add_(0, row[lo:lo + (1 << 17)], s["gy"][lo:lo + (1 << 17)].double())
        out.append(acc[:v] * case["scale"])
    return out


def _exact_linear(case, s):
    x, w = s["x"].double(), s["w"].double()
    z = torch.matmul(x, w.t().contiguous())
    if s["b"] is not None:
        z += s["b"].double()
    name = case["act"]
    if name == "none":
        a, da = z, torch.ones_like(z)
    elif name == "relu":
        a, da = torch.maximum(z, torch.zeros_like(z)), (z > 0).double()
    elif name == "silu":
        sg = torch.sigmoid(z)
        a, da = z * sg, sg + z * sg * (1 - sg)
    elif name == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        a, da = z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        a, da = 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    y = a + s["r"].double() if s["r"] is not None else a
    if not case["train"]:
        return [y]
    gy = s["gy"].double()
    dz = gy * da
    out = [y, torch.matmul(dz, w), torch.matmul(dz.t().contiguous(), x)]
    if s["b"] is not None:
        out.append(torch.sum(dz, 0))
    if s["r"] is not None:
        out.append(gy)
    return out


def _exact_clip(case, s):
    p = case["norm"]
    parts = [g.double().abs() for g in s["grads"]]
    if p == math.inf:
        norm = max(float(x.max()) for x in parts)
    else:
        norm = sum(float((x ** p).sum()) for x in parts) ** (1.0 / p)
    coef = min(1.0, s["max_norm"] / (norm + 1e-6))
    into = s["grads"] if s["out"] is None else s["out"]
    flat, views = _buckets([g.shape for g in into], [g.dtype for g in into], case["align"])
    flat = {dt: torch.zeros_like(f, dtype=torch.float64) for dt, f in flat.items()}
    for g, o, v in zip(s["grads"], into, views):
        flat[o.dtype].as_strided(v.shape, v.stride(), v.storage_offset()).copy_(g.double() * coef)
    return [torch.tensor(norm, dtype=torch.float64, device="cuda"), *flat.values()]
