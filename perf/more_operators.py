"""Timed cases of the feed-forward operators over atoms: layer norm with its gradients, a dense
layer with bias, activation and residual, and the same with a weight of each atom's group (its
species, or the expert that it is routed to), each in its plain form and through the framework's
own calls.

``listed()`` are the cases that are timed, ``draw(rng)`` gives more of the same ranges.
``prepare(case, seed)`` is what a program holds before the call, ``run(state)`` one pass,
``exact(case, seed)`` the same outputs from the definitions in 64 bits.
"""
from __future__ import annotations

import math
import types

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
# of the largest listed case: 3 products of 24,000 x 1,024 x 4,096, in a plain form in 32 bits
MAX_PRODUCT = 24000 * 1024 * 4096
MAX_ROW_ELEMENTS = 24000 * 2048


def listed() -> list:
    return [
        # one molecule (21 atoms) of a dynamics run, energies and forces: the latency of a norm
        # forward and backward
        dict(name="norm_molecule_21", kind="norm", tokens=21, channels=128, dtype="f32", affine=True,
             packed=True, train=True),
        # fitting on the 9,000-atom water box at 128 channels
        dict(name="norm_water_9000", kind="norm", tokens=9000, channels=128, dtype="f32", affine=True,
             packed=True, train=True),
        # screening the 72,000-atom box in 16 bits, a norm without weights of odd width that is a
        # part of wider rows
        dict(name="norm_odd_72000_serve", kind="norm", tokens=72000, channels=511, dtype="f16",
             affine=False, packed=False, train=False),
        # training a wide model in 16 bits
        dict(name="norm_wide_24000", kind="norm", tokens=24000, channels=2048, dtype="bf16", affine=True,
             packed=True, train=True),
        # a single atom through the wide layer: the weight's bytes
        dict(name="linear_wide_1_serve", kind="linear", tokens=1, inputs=1024, outputs=4096, dtype="bf16",
             bias=True, activation="gelu", residual=False, train=False),
        # the molecule's first feed-forward product with its gradients
        dict(name="linear_molecule_21", kind="linear", tokens=21, inputs=128, outputs=512, dtype="f32",
             bias=True, activation="silu", residual=False, train=True),
        # the water box's second one, onto the residual
        dict(name="linear_water_9000", kind="linear", tokens=9000, inputs=512, outputs=128, dtype="f32",
             bias=True, activation="none", residual=True, train=True),
        # training a wide model in 16 bits: three large products
        dict(name="linear_wide_24000", kind="linear", tokens=24000, inputs=1024, outputs=4096,
             dtype="bf16", bias=True, activation="gelu", residual=False, train=True),
        # a molecule's atoms, each with the weights of its species (four of nine)
        dict(name="grouped_molecule_21", kind="grouped", tokens=21, groups=9, ids="species", inputs=128,
             outputs=128, dtype="f32", bias=True, activation="silu", residual=False, train=True),
        # fitting with weights a species on the 72,000-atom water box: two groups hold all rows
        dict(name="grouped_water_72000", kind="grouped", tokens=72000, groups=9, ids="species",
             inputs=128, outputs=512, dtype="f32", bias=True, activation="silu", residual=False,
             train=True),
        # screening organic molecules in 16 bits, odd widths
        dict(name="grouped_odd_5000_serve", kind="grouped", tokens=5000, groups=119, ids="species",
             inputs=250, outputs=511, dtype="f16", bias=True, activation="silu", residual=False,
             train=False),
        # training 64 experts, to which a router sends very different numbers of rows (some none)
        dict(name="grouped_experts_16384", kind="grouped", tokens=16384, groups=64, ids="zipf",
             inputs=1024, outputs=1024, dtype="bf16", bias=False, activation="none", residual=True,
             train=True),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo: int, hi: int) -> int:
    """Half of the widths are multiples of 64 or 16, the others any number."""
    n = _log_int(rng, lo, hi)
    unit = rng.choice([64, 16, 1, 1])
    return max(unit, n // unit * unit)


def draw(rng) -> dict:
    """One more case of the listed kinds, sizes log-uniform over each kind's range."""
    kind = rng.choice(["norm", "linear", "linear", "grouped", "grouped"])
    dtype = rng.choice(["f32", "f32", "bf16", "bf16", "f16"])
    train = rng.random() < 0.7
    if kind == "norm":
        channels = _width(rng, 1, 8192)
        tokens = min(_log_int(rng, 1, 72000), MAX_ROW_ELEMENTS * 2 // (channels * BYTES[dtype]))
        return dict(kind=kind, tokens=tokens, channels=channels, dtype=dtype,
                    affine=rng.random() < 0.8, packed=rng.random() < 0.7, train=train)
    inputs, outputs = _width(rng, 8, 4096), _width(rng, 8, 4096)
    tokens = max(1, min(_log_int(rng, 1, 72000), MAX_PRODUCT // (inputs * outputs)))
    case = dict(kind=kind, tokens=tokens, inputs=inputs, outputs=outputs, dtype=dtype,
                bias=rng.random() < 0.7, activation=rng.choice(["none", "silu", "gelu", "tanh"]),
                residual=rng.random() < 0.4, train=train)
    if kind == "grouped":
        ids = rng.choice(["species", "zipf"])
        groups = rng.choice([9, 19, 119]) if ids == "species" else _log_int(rng, 1, 256)
        # the weights and their gradient in 32 bits: 1 GB each at most
        case.update(ids=ids, groups=max(1, min(groups, (1 << 28) // (inputs * outputs))))
    return case


# --------------------------------------------------------------------------- inputs
def _generator(seed: int):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _leaf(x):
    return x.detach().requires_grad_(True)


def _groups(case, rng) -> np.ndarray:
    T, G = case["tokens"], case["groups"]
    if case["ids"] == "species":
        known = np.array([z for z in (1, 8, 6, 7, 16, 17) if z < G] or [0])
        if T > 10000:                              # water: two hydrogens an oxygen
            known = known[:2]
        weight = np.array([2.0 if z == 1 else 1.0 for z in known])
        return rng.choice(known, size=T, p=weight / weight.sum()).astype(np.int64)
    ids = np.minimum(rng.zipf(1.3, size=T) - 1, G - 1)
    return rng.permutation(G)[ids].astype(np.int64)


def _group_counts(case) -> int:
    """Groups that have rows, about (the draws of the ids are another each time)."""
    if case["ids"] == "species":
        known = max(1, sum(z < case["groups"] for z in (1, 8, 6, 7, 16, 17)))
        return min(case["tokens"], known, 2 if case["tokens"] > 10000 else 6)
    return min(case["tokens"], case["groups"])


def prepare(case, seed):
    gen, rng = _generator(seed), np.random.default_rng(seed)
    s = types.SimpleNamespace(case=case)
    dt, T = DTYPES[case["dtype"]], case["tokens"]
    if case["kind"] == "norm":
        C = case["channels"]
        # features of an atom have an offset and a spread of their own
        x = torch.randn((T, C if case["packed"] else C + 8), generator=gen, device="cuda")
        x = x * (0.5 + torch.rand((T, 1), generator=gen, device="cuda")) + torch.randn(
            (T, 1), generator=gen, device="cuda")
        s.x = _leaf(x.to(dt)[:, :C])
        s.weight = s.bias = None
        if case["affine"]:
            s.weight = _leaf((1 + 0.1 * _normal(gen, (C,), torch.float32)).to(dt))
            s.bias = _leaf(_normal(gen, (C,), dt, 0.1))
        s.grad = _normal(gen, (T, C), dt)
        return s
    K, N = case["inputs"], case["outputs"]
    lead = (case["groups"],) if case["kind"] == "grouped" else ()
    s.x = _leaf(_normal(gen, (T, K), dt))
    s.weight = _leaf(_normal(gen, lead + (K, N), dt, K ** -0.5))
    s.bias = _leaf(_normal(gen, lead + (N,), dt, 0.1)) if case["bias"] else None
    s.residual = _leaf(_normal(gen, (T, N), dt)) if case["residual"] else None
    s.grad = _normal(gen, (T, N), dt)
    s.activation = None if case["activation"] == "none" else case["activation"]
    if case["kind"] == "grouped":
        ids = _groups(case, rng)
        s.ids = torch.from_numpy(ids).cuda()
        # the plain form's layout: the rows of each group that has some
        order = np.argsort(ids, kind="stable")
        s.rows = {int(g): torch.from_numpy(order[ids[order] == g]).cuda() for g in np.unique(ids)}
        if own:
            import xnn_amd as xa
            s.plan = xa.group_plan(s.ids, case["groups"])
    return s


# --------------------------------------------------------------------------- one pass
def run(s):
    case = s.case
    if own:
        return _OWN[case["kind"]](s)
    with torch.no_grad():
        return _PLAIN[case["kind"]](s)


def _own_call(s, call, leaves):
    if not s.case["train"]:
        with torch.no_grad():
            return call()
    out = call()
    return (out.detach(), *torch.autograd.grad(out, [t for t in leaves if t is not None], s.grad))


def _own_norm(s):
    import xnn_amd as xa
    return _own_call(s, lambda: xa.layer_norm(s.x, s.weight, s.bias, EPS), (s.x, s.weight, s.bias))


def _own_linear(s):
    import xnn_amd as xa
    return _own_call(s, lambda: xa.linear(s.x, s.weight, s.bias, s.activation, s.residual),
                     (s.x, s.weight, s.bias, s.residual))


def _own_grouped(s):
    import xnn_amd as xa
    return _own_call(s, lambda: xa.grouped_linear(s.x, s.weight, s.plan, s.bias, s.activation, s.residual),
                     (s.x, s.weight, s.bias, s.residual))


_OWN = {"norm": _own_norm, "linear": _own_linear, "grouped": _own_grouped}


def _plain_norm(s):
    dt, x = s.x.dtype, s.x.float()
    centered = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((centered * centered).mean(1, keepdim=True) + EPS)
    n = centered * r
    w = None if s.weight is None else s.weight.float()
    out = (n if w is None else n * w + s.bias.float()).to(dt)
    if not s.case["train"]:
        return out
    g = s.grad.float()
    gw = g if w is None else g * w
    dx = r * (gw - gw.mean(1, keepdim=True) - n * (gw * n).mean(1, keepdim=True))
    if w is None:
        return out, dx.to(dt)
    return out, dx.to(dt), (g * n).sum(0).to(dt), g.sum(0).to(dt)


def _activated(z, name):
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    return torch.tanh(z) if name == "tanh" else z


def _slope(z, name):
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    t = torch.tanh(z)
    return 1 - t * t


def _plain_rows(x, w, b, residual, g, name):
    """Rows of one weight in 32 bits: the output, and with a cotangent the gradients."""
    z = x @ w
    if b is not None:
        z = z + b
    y = _activated(z, name)
    if residual is not None:
        y = y + residual
    if g is None:
        return y, None, None, None
    d = g if name == "none" else g * _slope(z, name)
    return y, d @ w.t(), x.t() @ d, None if b is None else d.sum(0)


def _plain_linear(s):
    case, dt = s.case, s.x.dtype
    x, w, b, r = (None if t is None else t.float() for t in (s.x, s.weight, s.bias, s.residual))
    y, dx, dw, db = _plain_rows(x, w, b, r, s.grad.float() if case["train"] else None, case["activation"])
    if not case["train"]:
        return y.to(dt)
    out = (y.to(dt), dx.to(dt), dw.to(dt))
    if b is not None:
        out += (db.to(dt),)
    return out if r is None else (*out, s.grad)


def _plain_grouped(s):
    case, dt = s.case, s.x.dtype
    train = case["train"]
    y = torch.empty((case["tokens"], case["outputs"]), dtype=dt, device=s.x.device)
    if train:
        dx, dw = torch.empty_like(s.x), torch.zeros_like(s.weight)
        db = None if s.bias is None else torch.zeros_like(s.bias)
    for g, rows in s.rows.items():
        b = None if s.bias is None else s.bias[g].float()
        r = None if s.residual is None else s.residual[rows].float()
        part = _plain_rows(s.x[rows].float(), s.weight[g].float(), b, r,
                           s.grad[rows].float() if train else None, case["activation"])
        y[rows] = part[0].to(dt)
        if train:
            dx[rows], dw[g] = part[1].to(dt), part[2].to(dt)
            if db is not None:
                db[g] = part[3].to(dt)
    if not train:
        return y
    out = (y, dx, dw) if s.bias is None else (y, dx, dw, db)
    return out if s.residual is None else (*out, s.grad)


_PLAIN = {"norm": _plain_norm, "linear": _plain_linear, "grouped": _plain_grouped}


# --------------------------------------------------------------------------- floors
def work(case):
    size, T = BYTES[case["dtype"]], case["tokens"]
    if case["kind"] == "norm":
        n = T * case["channels"]
        b = 2 * n * size + (2 * case["channels"] * size if case["affine"] else 0)
        if case["train"]:                          # the cotangent in, the gradients out
            b += 2 * n * size + (2 * case["channels"] * size if case["affine"] else 0)
        return {"bytes": float(b), "flops": float(n * (18 if case["train"] else 7))}
    K, N = case["inputs"], case["outputs"]
    weights = _group_counts(case) if case["kind"] == "grouped" else 1
    b = T * (K + N) * size + weights * K * N * size
    b += (weights * N * size if case["bias"] else 0) + (T * N * size if case["residual"] else 0)
    if case["kind"] == "grouped":
        b += 8 * T
    if case["train"]:                              # the cotangent in, the gradients out
        b += T * (N + K) * size
        b += (case["groups"] if case["kind"] == "grouped" else 1) * (K + (1 if case["bias"] else 0)) * N * size
    return {"bytes": float(b), "flops": float((6 if case["train"] else 2) * T * K * N)}


# --------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s)


def _double(*tensors):
    return [None if t is None else t.detach().double().requires_grad_(True) for t in tensors]


def _with_gradients(s, out, leaves):
    if not s.case["train"]:
        return out.detach()
    return (out.detach(), *torch.autograd.grad(out, [t for t in leaves if t is not None], s.grad.double()))


def _exact_norm(s):
    x, w, b = leaves = _double(s.x, s.weight, s.bias)
    n = (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + EPS)
    return _with_gradients(s, n if w is None else torch.addcmul(b, n, w), leaves)


_FUNCTIONS = {"none": lambda z: z, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
              "tanh": torch.tanh}


def _exact_linear(s):
    x, w, b, r = leaves = _double(s.x, s.weight, s.bias, s.residual)
    z = torch.mm(x, w) if b is None else torch.addmm(b, x, w)
    y = _FUNCTIONS[s.case["activation"]](z)
    return _with_gradients(s, y if r is None else r + y, leaves)


def _exact_grouped(s):
    x, w, b, r = leaves = _double(s.x, s.weight, s.bias, s.residual)
    order = torch.argsort(s.ids, stable=True)
    counts = torch.bincount(s.ids, minlength=s.case["groups"]).tolist()
    ws, bs = w.unbind(0), None if b is None else b.unbind(0)
    parts = []
    for g, rows in enumerate(torch.split(order, counts)):
        if len(rows):
            z = torch.mm(x[rows], ws[g])
            parts.append(z if bs is None else z + bs[g])
    back = torch.argsort(order)
    y = _FUNCTIONS[s.case["activation"]](torch.cat(parts)[back])
    return _with_gradients(s, y if r is None else r + y, leaves)


_EXACT = {"norm": _exact_norm, "linear": _exact_linear, "grouped": _exact_grouped}
