"""Timed cases of the attention operators over atoms: species embedding with its gradient,
normalized and rotated heads, attention within structures with its gradient, and dropout
with a residual, each in its plain form and through the framework's own calls.

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
EPS = 1e-6
# scores of the padded plain form: the largest listed case has 4 x 24,000^2
MAX_SCORES = 4 * 24000 ** 2


def listed() -> list:
    return [
        # one molecule (21 atoms) of a dynamics run, energies and forces: the latency of a call
        # forward and backward
        dict(name="attention_molecule_21", kind="attention", structures=1, lo=21, hi=21, heads=4,
             kv_heads=4, head_dim=32, dtype="f32", masked=0.0, packed=False, train=True),
        # fitting on a batch of 1,024 molecules of 10 to 60 atoms, 64 channels
        dict(name="attention_batch_1024", kind="attention", structures=1024, lo=10, hi=60, heads=4,
             kv_heads=4, head_dim=16, dtype="f32", masked=0.0, packed=True, train=True),
        # the 9,000-atom water box at 128 channels, every atom attending to every other
        dict(name="attention_water_9000", kind="attention", structures=1, lo=9000, hi=9000, heads=4,
             kv_heads=4, head_dim=32, dtype="f32", masked=0.0, packed=True, train=True),
        # screening in 16 bits: structures of 10 to 1,000 atoms side by side, shared key and
        # value heads, padding atoms masked out, one structure with nothing left
        dict(name="attention_mixed_64_serve", kind="attention", structures=64, lo=10, hi=1000,
             heads=8, kv_heads=2, head_dim=64, dtype="bf16", masked=0.1, packed=True, train=False),
        # training on one large box in 16 bits
        dict(name="attention_box_24000", kind="attention", structures=1, lo=24000, hi=24000,
             heads=4, kv_heads=4, head_dim=64, dtype="bf16", masked=0.0, packed=True, train=True),
        # the species rows of one molecule, no gradient: the smallest lookup
        dict(name="embedding_molecule_21", kind="embedding", tokens=21, vocab=119, channels=128,
             dtype="f32", ids="species", train=False),
        # species rows of the 72,000-atom water box and the table's gradient: two ids hold all
        # the tokens
        dict(name="embedding_water_72000", kind="embedding", tokens=72000, vocab=119, channels=128,
             dtype="f32", ids="species", train=True),
        # a large vocabulary (fragments, text): most rows of the gradient are empty
        dict(name="embedding_vocabulary_50000", kind="embedding", tokens=16384, vocab=50000,
             channels=1024, dtype="bf16", ids="zipf", train=True),
        # heads of the 9,000-atom box rotated by each atom's own phases, gradients of the phases
        # (which lead to the forces) among the outputs
        dict(name="rotate_water_9000", kind="rotate", tokens=9000, heads=4, kv_heads=4, head_dim=32,
             rotated=32, dtype="f32", positions=0, interleaved=False, packed=True, train=True),
        # wide heads in 16 bits, rows of a table by position, keys shared by four heads each
        dict(name="rotate_wide_24000", kind="rotate", tokens=24000, heads=16, kv_heads=4,
             head_dim=128, rotated=128, dtype="bf16", positions=4096, interleaved=False,
             packed=True, train=True),
        # the residual branch of the 9,000-atom box, forward and backward
        dict(name="dropout_water_9000", kind="dropout", rows=9000, channels=128, dtype="f32", p=0.1,
             residual=True, train=True),
        # the same of a wide model over the 72,000-atom box in 16 bits
        dict(name="dropout_wide_72000", kind="dropout", rows=72000, channels=512, dtype="bf16",
             p=0.1, residual=True, train=True),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    """One more case of the listed kinds, sizes log-uniform over each kind's range."""
    kind = rng.choice(["attention", "attention", "attention", "embedding", "rotate", "dropout"])
    dtype = rng.choice(["f32", "f32", "bf16", "bf16", "f16"])
    train = rng.random() < 0.7
    if kind == "attention":
        kv = rng.choice([1, 2, 4])
        heads = kv * rng.choice([1, 1, 2, 4])
        heads, kv = (4, 4) if heads > 8 else (heads, kv)
        dim = rng.choice([8, 16, 20, 32, 33, 48, 64, 64, 96, 128])
        if rng.random() < 0.5:
            structures, lo = 1, _log_int(rng, 1, 24000)
            lo = min(lo, int(math.sqrt(MAX_SCORES * 64 / (heads * dim))), int(math.sqrt(MAX_SCORES / heads)))
            hi = lo
        else:
            structures = _log_int(rng, 2, 1024)
            lo = rng.randint(1, 20)
            hi = lo + _log_int(rng, 1, 2000)
            hi = max(lo, min(hi, int(math.sqrt(MAX_SCORES / (structures * heads)))))
        return dict(kind=kind, structures=structures, lo=lo, hi=hi, heads=heads, kv_heads=kv,
                    head_dim=dim, dtype=dtype, masked=rng.choice([0.0, 0.0, 0.1, 0.5]),
                    packed=rng.random() < 0.5, train=train)
    if kind == "embedding":
        ids = rng.choice(["species", "zipf"])
        tokens = _log_int(rng, 1, 72000)
        channels = rng.choice([32, 64, 65, 128, 250, 512, 1024])
        tokens = min(tokens, 16384 * 2048 // (channels * BYTES[dtype]))
        vocab = rng.choice([9, 19, 119]) if ids == "species" else _log_int(rng, 100, 50000)
        return dict(kind=kind, tokens=tokens, vocab=vocab, channels=channels, dtype=dtype, ids=ids,
                    train=train)
    if kind == "rotate":
        kv = rng.choice([1, 2, 4])
        heads = kv * rng.choice([1, 2, 4])
        dim = rng.choice([16, 32, 48, 64, 80, 128])
        tokens = min(_log_int(rng, 1, 24000),
                     24000 * 20 * 256 // ((heads + kv) * dim * BYTES[dtype]))
        return dict(kind=kind, tokens=tokens, heads=heads, kv_heads=kv, head_dim=dim,
                    rotated=rng.choice([dim, dim, dim // 2]), dtype=dtype,
                    positions=rng.choice([0, 0, 512, 4096]), interleaved=rng.random() < 0.3,
                    packed=rng.random() < 0.5, train=train)
    channels = rng.choice([1, 33, 64, 128, 256, 511, 512])
    rows = min(_log_int(rng, 1, 72000), 72000 * 1024 // (channels * BYTES[dtype]))
    return dict(kind=kind, rows=rows, channels=channels, dtype=dtype,
                p=rng.choice([0.0, 0.1, 0.25, 0.5]), residual=rng.random() < 0.7, train=train)


# --------------------------------------------------------------------------- inputs
def _generator(seed: int):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _counts(case) -> np.ndarray:
    """Atoms of each structure, spread over the logarithm of the case's range."""
    B, lo, hi = case["structures"], case["lo"], case["hi"]
    x = (np.arange(B) + 0.5) / B
    return np.clip(np.rint(lo * (hi / lo) ** x), lo, hi).astype(np.int64)


def _valid(case, counts, rng):
    """The atoms that may be attended to (None: all); of several structures one has none."""
    if case["masked"] == 0.0:
        return None
    total = int(counts.sum())
    valid = rng.random(total) >= case["masked"]
    if len(counts) > 1:
        start = int(counts[: len(counts) // 2].sum())
        valid[start:start + counts[len(counts) // 2]] = False
    return valid


def _split(x, packed, *heads):
    """Head blocks of one projection's output: views of it, or each a tensor of its own."""
    parts = x.split(list(heads), 1)
    return [(p if packed else p.contiguous()).detach().requires_grad_(True) for p in parts]


def prepare(case, seed):
    gen, rng = _generator(seed), np.random.default_rng(seed)
    s = types.SimpleNamespace(case=case)
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "attention":
        counts = rng.permutation(_counts(case))
        total, H, K, D = int(counts.sum()), case["heads"], case["kv_heads"], case["head_dim"]
        qkv = _normal(gen, (total, H + 2 * K, D), dt)
        s.q, s.k, s.v = _split(qkv, case["packed"], H, K, K)
        s.grad = _normal(gen, (total, H, D), dt)
        valid = _valid(case, counts, rng)
        s.mask = None if valid is None else torch.from_numpy(valid).cuda()
        s.n_atoms = torch.from_numpy(counts).cuda()
        # the plain form's layout: row of each atom in the padded batch
        longest = int(counts.max())
        rows = np.repeat(np.arange(len(counts)) * longest, counts) + np.concatenate(
            [np.arange(n) for n in counts])
        s.shape, s.rows = (len(counts), longest), torch.from_numpy(rows).cuda()
        if own:
            import xnn_amd as xa
            s.plan = xa.attention_plan(s.n_atoms, total)
    elif case["kind"] == "embedding":
        V, C, T = case["vocab"], case["channels"], case["tokens"]
        s.table = _normal(gen, (V, C), dt).requires_grad_(True)
        if case["ids"] == "species":
            known = np.array([z for z in (1, 8, 6, 7, 16, 17, 18) if z < V])[:2 if T > 4000 else 7]
            ids = rng.choice(known, size=T)
        else:
            ids = np.minimum(rng.zipf(1.2, size=T) - 1, V - 1)
            ids = rng.permutation(V)[ids]
        s.ids = torch.from_numpy(ids.astype(np.int64)).cuda()
        s.scale = float(math.sqrt(C))
        s.grad = _normal(gen, (T, C), dt)
    elif case["kind"] == "rotate":
        T, H, K, D, R = (case[k] for k in ("tokens", "heads", "kv_heads", "head_dim", "rotated"))
        qk = _normal(gen, (T, H + K, D), dt)
        s.q, s.k = _split(qk, case["packed"], H, K)
        s.q_weight, s.k_weight = ((1 + 0.1 * _normal(gen, (D,), torch.float32)).to(dt)
                                  .requires_grad_(True) for _ in range(2))
        P = case["positions"]
        angle = torch.rand((P or T, R // 2), generator=gen, device="cuda") * (2 * math.pi)
        s.cos, s.sin = torch.cos(angle), torch.sin(angle)
        s.positions = None
        if P:
            s.positions = torch.from_numpy(np.arange(T, dtype=np.int64) % P).cuda()
        elif case["train"]:
            s.cos.requires_grad_(True)
            s.sin.requires_grad_(True)
        s.grad_q, s.grad_k = _normal(gen, (T, H, D), dt), _normal(gen, (T, K, D), dt)
    else:
        n = (case["rows"], case["channels"])
        s.x, s.grad = (_normal(gen, n, dt) for _ in range(2))
        s.residual = _normal(gen, n, dt).requires_grad_(True) if case["residual"] else None
        s.x.requires_grad_(True)
        # a seed of 64 bits, a counter that has passed 32
        s.seed, s.offset = int(rng.integers(0, 2 ** 63)), int(rng.integers(2 ** 32, 2 ** 40))
    return s


# --------------------------------------------------------------------------- one pass
def run(s):
    case = s.case
    if own:
        return _OWN[case["kind"]](s)
    with torch.no_grad():
        return _PLAIN[case["kind"]](s)


def _own_attention(s):
    import xnn_amd as xa
    if not s.case["train"]:
        with torch.no_grad():
            return xa.structure_attention(s.q, s.k, s.v, s.plan, mask=s.mask)
    out = xa.structure_attention(s.q, s.k, s.v, s.plan, mask=s.mask)
    return (out.detach(), *torch.autograd.grad(out, (s.q, s.k, s.v), s.grad))


def _own_embedding(s):
    import xnn_amd as xa
    if not s.case["train"]:
        with torch.no_grad():
            return xa.embedding(s.ids, s.table, s.scale)
    out = xa.embedding(s.ids, s.table, s.scale)
    return (out.detach(), *torch.autograd.grad(out, (s.table,), s.grad))


def _own_rotate(s):
    import xnn_amd as xa
    args = (s.q, s.k, s.q_weight, s.k_weight, s.cos, s.sin)
    kw = dict(positions=s.positions, eps=EPS, interleaved=s.case["interleaved"])
    if not s.case["train"]:
        with torch.no_grad():
            return xa.head_norm_rotate(*args, **kw)
    q, k = xa.head_norm_rotate(*args, **kw)
    wanted = args if s.positions is None else args[:4]
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), wanted, (s.grad_q, s.grad_k)))


def _own_dropout(s):
    import xnn_amd as xa
    if not s.case["train"]:
        with torch.no_grad():
            return xa.dropout_add(s.x, s.residual, s.case["p"], s.seed, s.offset)
    out = xa.dropout_add(s.x, s.residual, s.case["p"], s.seed, s.offset)
    wanted = (s.x,) if s.residual is None else (s.x, s.residual)
    return (out.detach(), *torch.autograd.grad(out, wanted, s.grad))


_OWN = {"attention": _own_attention, "embedding": _own_embedding, "rotate": _own_rotate,
        "dropout": _own_dropout}


def _padded(x, s, groups=1):
    """(T, H, D) as (B, H, L, D) in float32, zeros beyond a structure's atoms; a shared head
    repeated for each of its group."""
    B, L = s.shape
    out = x.new_zeros((B * L, x.shape[1], x.shape[2]), dtype=torch.float32)
    out[s.rows] = x.float()
    out = out.view(B, L, *x.shape[1:]).transpose(1, 2)
    return out if groups == 1 else out.repeat_interleave(groups, 1)


def _unpadded(x, s, groups=1):
    """The inverse of :func:`_padded`; a shared head gets the sum over its group."""
    B, H, L, D = x.shape
    if groups > 1:
        x = x.view(B, H // groups, groups, L, D).sum(2)
    return x.transpose(1, 2).reshape(B * L, H // groups, D)[s.rows]


def _plain_attention(s):
    c = s.case
    B, L = s.shape
    groups = c["heads"] // c["kv_heads"]
    dt = s.q.dtype
    q, k, v = _padded(s.q, s), _padded(s.k, s, groups), _padded(s.v, s, groups)
    allowed = torch.zeros(B * L, dtype=torch.bool, device=q.device)
    allowed[s.rows] = True if s.mask is None else s.mask
    allowed = allowed.view(B, 1, 1, L)
    scale = c["head_dim"] ** -0.5
    scores = (q * scale) @ k.transpose(2, 3)
    scores.masked_fill_(~allowed, -math.inf)
    top = scores.amax(3, keepdim=True)
    scores -= torch.where(top == -math.inf, 0.0, top)
    prob = scores.exp_()
    total = prob.sum(3, keepdim=True)
    prob /= torch.where(total == 0, 1.0, total)
    out = prob @ v
    result = _unpadded(out, s).to(dt)
    if not c["train"]:
        return result
    g = _padded(s.grad, s)
    dv = prob.transpose(2, 3) @ g
    ds = g @ v.transpose(2, 3)
    ds -= (g * out).sum(3, keepdim=True)
    ds *= prob
    del prob, scores
    dq = (ds @ k) * scale
    dk = ds.transpose(2, 3) @ (q * scale)
    return (result, _unpadded(dq, s).to(dt), _unpadded(dk, s, groups).to(dt),
            _unpadded(dv, s, groups).to(dt))


def _plain_embedding(s):
    out = (s.table[s.ids].float() * s.scale).to(s.table.dtype)
    if not s.case["train"]:
        return out
    grad = torch.zeros(s.table.shape, device=s.table.device)
    grad.index_add_(0, s.ids, s.grad.float())
    return out, (grad * s.scale).to(s.table.dtype)


def _pairs(x, R, interleaved):
    """The two members of each rotated pair, and what is left as it is."""
    turned, rest = x[..., :R], x[..., R:]
    if interleaved:
        return turned[..., 0::2], turned[..., 1::2], rest
    return turned[..., :R // 2], turned[..., R // 2:], rest


def _joined(a, b, rest, interleaved):
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, rest), -1)


def _plain_heads(x, weight, cos, sin, g, case):
    """One of queries and keys: its output, and its gradients where ``g`` is given."""
    R, inter = case["rotated"], case["interleaved"]
    dt, x, w = x.dtype, x.float(), weight.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x * r
    a, b, rest = _pairs(n * w, R, inter)
    out = _joined(a * cos - b * sin, a * sin + b * cos, rest, inter).to(dt)
    if g is None:
        return (out,)
    ga, gb, grest = _pairs(g.float(), R, inter)
    d_cos, d_sin = (ga * a + gb * b).sum(1), (gb * a - ga * b).sum(1)
    gu = _joined(ga * cos + gb * sin, gb * cos - ga * sin, grest, inter)
    gn = gu * w
    dx = r * (gn - n * (gn * n).mean(-1, keepdim=True))
    return out, dx.to(dt), (gu * n).sum((0, 1)).to(dt), d_cos, d_sin


def _plain_rotate(s):
    case = s.case
    cos, sin = s.cos, s.sin
    if s.positions is not None:
        cos, sin = cos[s.positions], sin[s.positions]
    cos, sin = cos[:, None, :], sin[:, None, :]
    gq, gk = (s.grad_q, s.grad_k) if case["train"] else (None, None)
    q = _plain_heads(s.q, s.q_weight, cos, sin, gq, case)
    k = _plain_heads(s.k, s.k_weight, cos, sin, gk, case)
    if not case["train"]:
        return q[0], k[0]
    out = (q[0], k[0], q[1], k[1], q[2], k[2])
    return out if s.positions is not None else (*out, q[3] + k[3], q[4] + k[4])


def _philox_round(c, key):
    """One round of Philox4x32 (Salmon et al., SC 2011) on int64 tensors of 32-bit words."""
    m = 0xFFFFFFFF
    p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
    return (((p1 >> 32) & m) ^ c[1] ^ key[0], p1 & m, ((p0 >> 32) & m) ^ c[3] ^ key[1], p0 & m)


def _draws16(n, seed, offset, device):
    """``n`` 16-bit draws: element e has half word e % 8 of the Philox block with counter
    (e / 8, offset) and key ``seed``."""
    m = 0xFFFFFFFF
    i = torch.arange((n + 7) // 8, device=device)
    c = (i & m, i >> 32, torch.full_like(i, offset & m), torch.full_like(i, (offset >> 32) & m))
    k = [(((seed & m) + j * 0x9E3779B9) & m, (((seed >> 32) & m) + j * 0xBB67AE85) & m)
         for j in range(10)]
    c = _philox_round(_philox_round(_philox_round(_philox_round(_philox_round(
        c, k[0]), k[1]), k[2]), k[3]), k[4])
    c = _philox_round(_philox_round(_philox_round(_philox_round(_philox_round(
        c, k[5]), k[6]), k[7]), k[8]), k[9])
    words = torch.stack(c, 1)
    return torch.stack((words & 0xFFFF, words >> 16), 2).flatten()[:n]


def _plain_dropout(s):
    drop = int(round(s.case["p"] * 65536))
    keep = _draws16(s.x.numel(), s.seed, s.offset, s.x.device).view(s.x.shape) >= drop
    factor = 65536.0 / (65536 - drop)
    out = torch.where(keep, s.x.float() * factor, 0.0)
    if s.residual is not None:
        out = out + s.residual.float()
    out = out.to(s.x.dtype)
    if not s.case["train"]:
        return out
    dx = torch.where(keep, s.grad.float() * factor, 0.0).to(s.x.dtype)
    return (out, dx) if s.residual is None else (out, dx, s.grad)


_PLAIN = {"attention": _plain_attention, "embedding": _plain_embedding, "rotate": _plain_rotate,
          "dropout": _plain_dropout}


# --------------------------------------------------------------------------- floors
def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"] == "attention":
        counts = _counts(case)
        T, H, K, D = int(counts.sum()), case["heads"], case["kv_heads"], case["head_dim"]
        pairs = float((counts ** 2).sum()) * (1 - case["masked"])
        io = (2 * H + 2 * K) * T * D * size
        if not case["train"]:
            return {"bytes": float(io), "flops": 4 * pairs * H * D}
        # the gradient reads q, k, v and the cotangent, writes three gradients
        return {"bytes": float(2 * io), "flops": 14 * pairs * H * D}
    if case["kind"] == "embedding":
        T, V, C = case["tokens"], case["vocab"], case["channels"]
        rows = min(T, 7 if case["ids"] == "species" else V)
        b = rows * C * size + T * 8 + T * C * size
        if case["train"]:
            b += T * C * size + V * C * size
        return {"bytes": float(b), "flops": float(T * C * (2 if case["train"] else 1))}
    if case["kind"] == "rotate":
        T, heads, D = case["tokens"], case["heads"] + case["kv_heads"], case["head_dim"]
        tables = (case["positions"] or T) * case["rotated"] * 4
        b = 2 * T * heads * D * size + tables
        if case["train"]:
            b += 2 * T * heads * D * size + (0 if case["positions"] else tables)
        return {"bytes": float(b), "flops": float(T * heads * D * (24 if case["train"] else 7))}
    n = case["rows"] * case["channels"]
    b = n * size * (3 if case["residual"] else 2)
    if case["train"]:
        b += 2 * n * size
    return {"bytes": float(b), "flops": float(n * (3 if case["train"] else 2))}


# --------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s)


def _exact_attention(s):
    case = s.case
    groups, train = case["heads"] // case["kv_heads"], case["train"]
    q, k, v = (t.detach().double() for t in (s.q, s.k, s.v))
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    mask = torch.ones(len(q), dtype=torch.bool, device=q.device) if s.mask is None else s.mask
    start = 0
    for n in s.n_atoms.tolist():
        own_rows = torch.arange(start, start + n, device=q.device)
        start += n
        keys = own_rows[mask[own_rows]]
        if len(keys) == 0:
            continue
        # heads together in small structures, one at a time in large ones
        step = case["heads"] if n <= 2000 else 1
        for h in range(0, case["heads"], step):
            mine = torch.arange(h, h + step, device=q.device)
            shared = mine // groups
            a = q[own_rows][:, mine].transpose(0, 1).contiguous().requires_grad_(train)
            b = k[keys][:, shared].transpose(0, 1).contiguous().requires_grad_(train)
            c = v[keys][:, shared].transpose(0, 1).contiguous().requires_grad_(train)
            weights = torch.softmax((a @ b.transpose(1, 2)) / math.sqrt(case["head_dim"]), -1)
            o = weights @ c
            out[own_rows[:, None], mine] = o.detach().transpose(0, 1)
            if train:
                g = s.grad[own_rows][:, mine].double().transpose(0, 1)
                ga, gb, gc = torch.autograd.grad(o, (a, b, c), g)
                dq[own_rows[:, None], mine] = ga.transpose(0, 1)
                rows, cols = keys[:, None].expand(-1, step), shared.expand(len(keys), -1)
                dk.index_put_((rows, cols), gb.transpose(0, 1), accumulate=True)
                dv.index_put_((rows, cols), gc.transpose(0, 1), accumulate=True)
            del weights, o
    return (out, dq, dk, dv) if train else out


def _exact_embedding(s):
    table = s.table.detach().double().requires_grad_(True)
    out = torch.nn.functional.embedding(s.ids, table) * s.scale
    if not s.case["train"]:
        return out.detach()
    return out.detach(), torch.autograd.grad(out, table, s.grad.double())[0]


def _exact_rotate(s):
    case = s.case
    R, D = case["rotated"], case["head_dim"]
    leaves = [t.detach().double().requires_grad_(True)
              for t in (s.q, s.k, s.q_weight, s.k_weight, s.cos, s.sin)]
    q, k, wq, wk, cos, sin = leaves
    if s.positions is not None:
        cos, sin = cos[s.positions], sin[s.positions]
    turn = torch.complex(cos, sin)[:, None, :]
    order = list(range(D))
    if not case["interleaved"]:
        order[:R] = [i // 2 + (i % 2) * (R // 2) for i in range(R)]
    back = torch.tensor(np.argsort(order), device=q.device)
    order = torch.tensor(order, device=q.device)

    def heads(x, w):
        y = (x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + EPS) * w)[..., order]
        z = torch.view_as_complex(y[..., :R].unflatten(-1, (R // 2, 2)).contiguous()) * turn
        return torch.cat((torch.view_as_real(z).flatten(-2), y[..., R:]), -1)[..., back]

    outs = heads(q, wq), heads(k, wk)
    if not case["train"]:
        return tuple(o.detach() for o in outs)
    wanted = leaves if s.positions is None else leaves[:4]
    grads = torch.autograd.grad(outs, wanted, (s.grad_q.double(), s.grad_k.double()))
    return (*(o.detach() for o in outs), *grads)


def _exact_dropout(s):
    n, u32 = s.x.numel(), np.uint64(0xFFFFFFFF)
    i = np.arange((n + 7) // 8, dtype=np.uint64)
    c = [i & u32, i >> np.uint64(32), np.full_like(i, s.offset & 0xFFFFFFFF),
         np.full_like(i, s.offset >> 32)]
    key = [s.seed & 0xFFFFFFFF, s.seed >> 32]
    for _ in range(10):
        low, high = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(high >> np.uint64(32)) ^ c[1] ^ np.uint64(key[0]), high & u32,
             (low >> np.uint64(32)) ^ c[3] ^ np.uint64(key[1]), low & u32]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    halves = np.stack([h for w in c for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], 1)
    drop = int(round(s.case["p"] * 65536))
    keep = torch.from_numpy(halves.reshape(-1)[:n] >= np.uint64(drop)).to(s.x.device)
    factor = keep.view(s.x.shape).double() * (65536.0 / (65536 - drop))
    out = s.x.detach().double() * factor
    if s.residual is not None:
        out = out + s.residual.detach().double()
    if not s.case["train"]:
        return out
    dx = s.grad.double() * factor
    return (out, dx) if s.residual is None else (out, dx, s.grad.double())


_EXACT = {"attention": _exact_attention, "embedding": _exact_embedding, "rotate": _exact_rotate,
          "dropout": _exact_dropout}
