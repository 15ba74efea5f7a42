"""Timed and checked cases of the rotary-position and differential-attention operators.

Two operators, each in the forms a program meets them in:

  rotary    q and k of a projection turned by their token positions (forward, and forward + gradient)
  dattn     differential attention: softmax(q1 k1^T) - lambda * softmax(q2 k2^T) times v, its sub-normalisation,
            and the gradients of everything that is learned

`own = False` computes them from elementary torch operations in float32, `own = True` through uniter_amd.  `exact` computes them
a third time in float64, gradients by their formulas.
"""
import math
import random

import torch

own = False

BF16 = torch.bfloat16
EPS = 1e-5


def _dev():
    return "cuda" if torch.cuda.is_available() else "cpu"


# --------------------------------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # q | k of the base encoder's projection (hidden 768, two 32-wide maps per 64-wide head), one training step
        _rotary("rotary_base_step", B=32, L=96, heads=48, dim=32, rot=32, train=True),
        # one new token of one request, far into its context
        _rotary("rotary_one_token", B=1, L=1, heads=24, dim=64, rot=64, interleaved=True, first=131_071),
        # a long prompt: half of each head turned, frequencies stretched for a context 16 times the trained one
        _rotary("rotary_long_prompt", B=1, L=32_749, heads=24, dim=64, rot=32, scaling="yarn", factor=16.0),
        # 24-layer configuration's sequences (128 + 50 tokens) in the interleaved layout, one training step
        _rotary("rotary_large_step", B=16, L=178, heads=32, dim=64, rot=64, interleaved=True, scaling="linear", factor=4.0, train=True),
        # the class token alone against its own sequence: the smallest serving call
        _dattn("dattn_cls_token", B=1, Lq=1, Lk=96, heads=12, dim=32),
        # one token of each request against a long context
        _dattn("dattn_token_long", B=4, Lq=1, Lk=16_381, heads=12, dim=32),
        # the base encoder's shape, padded batch, forward only (evaluation, retrieval)
        _dattn("dattn_base_eval", B=32, Lq=96, Lk=96, heads=12, dim=32, mask="pad"),
        # the base encoder's shape, one training step of the operator
        _dattn("dattn_base_step", B=32, Lq=96, Lk=96, heads=12, dim=32, mask="pad", train=True),
        # 24-layer configuration (hidden 1024) at 128 + 50 tokens with 128-wide heads, one training step
        _dattn("dattn_large_step", B=16, Lq=178, Lk=178, heads=8, dim=64, mask="pad", train=True),
        # ragged sequences up to the position table's 512, stored back to back, one training step
        _dattn("dattn_packed_step", B=24, Lq=509, Lk=509, heads=12, dim=32, packed=True, train=True),
        # a long document, forward only
        _dattn("dattn_long_eval", B=1, Lq=8_191, Lk=8_191, heads=6, dim=64),
        # long training sequences; the rear part of each is masked out for good (-inf)
        _dattn("dattn_long_step", B=2, Lq=2_050, Lk=2_050, heads=12, dim=32, mask="inf", train=True),
    ]


def _rotary(name, B, L, heads, dim, rot, interleaved=False, scaling="none", factor=1.0, first=0, train=False):
    c = dict(op="rotary", B=B, L=L, heads=heads, dim=dim, rot=rot, interleaved=interleaved, scaling=scaling, factor=factor,
             first=first, train=train)
    return dict(c, name=name) if name else c


def _dattn(name, B, Lq, Lk, heads, dim, mask="none", packed=False, cross=False, norm=True, depth=5, train=False):
    c = dict(op="dattn", B=B, Lq=Lq, Lk=Lk, heads=heads, dim=dim, mask=mask, packed=packed, cross=cross or Lq != Lk, norm=norm,
             depth=depth, train=train)
    return dict(c, name=name) if name else c


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.35:
        dim = rng.choice([32, 64, 128])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        heads = rng.choice([8, 12, 16, 24, 32, 48])
        rows = max(1, _log(rng, 1, 32_768) * 64 // dim * 24 // heads)
        L = min(rows, _log(rng, 1, 32_768))
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return _rotary(None, B=max(1, rows // L), L=L, heads=heads, dim=dim, rot=rot, interleaved=rng.random() < 0.5,
                       scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 16.0]),
                       first=rng.choice([0, 0, _log(rng, 1, 200_000)]), train=rng.random() < 0.5)
    dim, heads = rng.choice([(32, 12), (32, 16), (64, 6), (64, 8), (32, 5), (64, 3)])
    kind = rng.choice(["token", "self", "self", "packed", "cross"])
    train = kind != "token" and rng.random() < 0.6
    if kind == "token":
        return _dattn(None, B=_log(rng, 1, 8), Lq=1, Lk=_log(rng, 1, 16_384), heads=heads, dim=dim,
                      mask=rng.choice(["none", "pad", "inf"]), depth=rng.randrange(24))
    if kind == "packed":
        L = _log(rng, 16 if train else 2, 1_024)
        return _dattn(None, B=max(1, min(32, _log(rng, 1, 8_192) // L + 1)), Lq=L, Lk=L, heads=heads, dim=dim, packed=True,
                      norm=rng.random() < 0.8, depth=rng.randrange(24), train=train)
    # (a lone key's attention weight is 1 whatever its score: training sequences have some keys to choose from)
    L = _log(rng, 24, 2_048) if train else _log(rng, 1, 4_096)
    Lk = max(1, int(L * rng.uniform(0.3, 1.0))) if kind == "cross" else L
    return _dattn(None, B=max(1, min(32, 4_096 // L)), Lq=L, Lk=Lk, heads=heads, dim=dim, mask=rng.choice(["none", "pad", "inf"]),
                  cross=kind == "cross", norm=rng.random() < 0.8, depth=rng.randrange(24), train=train)


# --------------------------------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Ragged lengths spread over 1 .. Lq (a golden-ratio sequence), the longest among them; every batch shuffles the same ones."""
    return [case["Lq"]] + [1 + int((case["Lq"] - 1) * ((i * 0.6180339887498949) % 1.0)) for i in range(1, case["B"])]


def prepare(case, seed):
    g = torch.Generator(device=_dev()).manual_seed(int(seed) * 2 + 1)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device=_dev(), generator=g) * std).to(BF16)

    s = dict(case)
    if case["op"] == "rotary":
        B, L, w = case["B"], case["L"], case["heads"] * case["dim"]
        # q | k are the first two thirds of a fused projection's rows
        s["proj"] = normal(B, L, w + w // 2)
        jitter = torch.randint(0, 9, (B, 1), device=_dev(), generator=g)              # requests do not start at one position
        s["positions"] = torch.arange(L, device=_dev())[None, :] + case["first"] + jitter
        if case["train"]:
            s["dout"] = normal(B, L, case["heads"], case["dim"])
        return s
    B, Lq, Lk, heads, dim = case["B"], case["Lq"], case["Lk"], case["heads"], case["dim"]
    H = heads * 2 * dim
    s["lambdas"] = tuple(normal(heads, dim, std=0.1) for _ in range(4))
    s["lambda_init"] = 0.8 - 0.6 * math.exp(-0.3 * case["depth"])
    s["norm_weight"] = (1.0 + normal(2 * dim, std=0.1).float()).to(BF16) if case["norm"] else None
    rows = (B, Lq)
    s["cu"], s["max_len"] = None, None
    if case["packed"]:
        lens = _lengths(case)
        random.Random(seed).shuffle(lens)
        s["cu"] = torch.tensor([sum(lens[:i]) for i in range(B + 1)], dtype=torch.int32, device=_dev())
        s["max_len"] = Lq
        rows = (sum(lens),)
    if case["cross"]:
        s["q"] = normal(B, Lq, H)
        s["kv"] = normal(B, Lk, 2 * H)
    else:
        s["qkv"] = normal(*rows, 3 * H)
    s["mask_bias"] = None
    if case["mask"] != "none":
        low = -10000.0 if case["mask"] == "pad" else -math.inf
        real = torch.randint((Lk + 1) // 2, Lk + 1, (B, 1), device=_dev(), generator=g)
        s["mask_bias"] = torch.where(torch.arange(Lk, device=_dev())[None, :] < real, 0.0, low).to(torch.float32)
    if case["train"]:
        s["dout"] = normal(*rows, H)
    return s


# --------------------------------------------------------------------------------------------------------------------------
# rotary positions
# --------------------------------------------------------------------------------------------------------------------------
BASE = 10000.0
TRAINED = 2048               # positions that the frequencies were trained for ("yarn")


def _frequencies(c):
    """(angle per position of each turned pair, factor on the result) in Python floats: the published scaling formulas."""
    n = c["rot"] // 2
    base = BASE
    if c["scaling"] == "ntk":
        base = BASE * c["factor"] ** (c["rot"] / (c["rot"] - 2))
    f = [base ** (-2.0 * i / c["rot"]) for i in range(n)]
    if c["scaling"] == "linear":
        return [x / c["factor"] for x in f], 1.0
    if c["scaling"] != "yarn":
        return f, 1.0

    def pair_of(turns):      # the (fractional) pair that makes this many turns over the trained positions
        return c["rot"] * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(BASE))

    lo, hi = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), c["rot"] - 1)
    out = []
    for i, x in enumerate(f):
        keep = 1.0 - min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
        out.append(x / c["factor"] * (1.0 - keep) + x * keep)
    return out, 0.1 * math.log(c["factor"]) + 1.0


def _qk(s):
    w = s["heads"] * s["dim"]
    return s["proj"][..., :w].unflatten(-1, (s["heads"], s["dim"]))


def _turn(x, cos, sin, rot, interleaved):
    """x [..., heads, dim], cos / sin [..., 1, rot / 2]."""
    t, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = t[..., 0::2], t[..., 1::2]
        t = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = t[..., : rot // 2], t[..., rot // 2:]
        t = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((t, rest), dim=-1)


def _run_rotary(s):
    if own:
        from uniter_amd import ops
        from uniter_amd.model.rotary import RotaryPositions
        if "plan" not in s:                  # what a model holds: built once from its configuration
            s["plan"] = RotaryPositions(s["dim"], rotary_dim=s["rot"], base=BASE, interleaved=s["interleaved"],
                                        scaling=None if s["scaling"] == "none" else
                                        {"type": s["scaling"], "factor": s["factor"], "original_max_position": TRAINED})
        x = _qk(s)
        if not s["train"]:
            return ops.rotary(x, s["positions"], s["plan"])
        x = x.detach().requires_grad_(True)
        y = ops.rotary(x, s["positions"], s["plan"])
        return y, torch.autograd.grad(y, x, s["dout"])[0]
    f, mult = _frequencies(s)
    angle = s["positions"].double()[..., None, None] * torch.tensor(f, dtype=torch.float64, device=s["proj"].device)
    cos, sin = (torch.cos(angle) * mult).float(), (torch.sin(angle) * mult).float()
    x = _qk(s).float()
    if not s["train"]:
        return _turn(x, cos, sin, s["rot"], s["interleaved"]).to(BF16)
    x = x.detach().requires_grad_(True)
    y = _turn(x, cos, sin, s["rot"], s["interleaved"])
    return y.to(BF16), torch.autograd.grad(y, x, s["dout"].float())[0].to(BF16)


# --------------------------------------------------------------------------------------------------------------------------
# differential attention
# --------------------------------------------------------------------------------------------------------------------------
def _plain_dattn(q, k, v, lambdas, lambda_init, weight, bias, heads, dim):
    """q [B, Lq, H], k / v [B, Lk, H], bias [B, Lk] or None; all float32.  [B, Lq, H]."""
    B, Lq, H = q.shape
    Lk = k.shape[1]
    q = q.view(B, Lq, heads, 2, dim).permute(0, 2, 3, 1, 4).reshape(B * heads * 2, Lq, dim)
    k = k.view(B, Lk, heads, 2, dim).permute(0, 2, 3, 4, 1).reshape(B * heads * 2, dim, Lk)
    v = v.view(B, Lk, heads, 2 * dim).permute(0, 2, 1, 3).reshape(B * heads, Lk, 2 * dim)
    sc = torch.bmm(q, k).view(B, heads, 2, Lq, Lk) * dim ** -0.5
    if bias is not None:
        sc = sc + bias[:, None, None, None, :]
    top = sc.amax(dim=-1, keepdim=True)
    e = torch.exp(sc - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)                    # a row without keys attends to nothing
    lq1, lk1, lq2, lk2 = lambdas
    lam = torch.exp((lq1 * lk1).sum(-1)) - torch.exp((lq2 * lk2).sum(-1)) + lambda_init
    a = p[:, :, 0] - lam[None, :, None, None] * p[:, :, 1]
    o = torch.bmm(a.reshape(B * heads, Lq, Lk), v).view(B, heads, Lq, 2 * dim)
    if weight is not None:
        o = o * torch.rsqrt(o.square().mean(dim=-1, keepdim=True) + EPS) * weight * (1.0 - lambda_init)
    return o.permute(0, 2, 1, 3).reshape(B, Lq, H)


def _run_dattn(s):
    heads, dim = s["heads"], s["dim"]
    H = heads * 2 * dim
    if own:
        from uniter_amd import ops
        lams, weight = s["lambdas"], s["norm_weight"]
        data = (s["q"], s["kv"]) if s["cross"] else (s["qkv"],)
        if s["train"]:
            data = tuple(t.detach().requires_grad_(True) for t in data)
            lams = tuple(t.detach().requires_grad_(True) for t in lams)
            weight = None if weight is None else weight.detach().requires_grad_(True)
        if s["cross"]:
            if s["train"]:                   # k and v of one projection, as two gradients
                k, v = (t.detach().requires_grad_(True) for t in data[1].split(H, dim=-1))
                data = (data[0], k, v)
            else:
                data = (data[0],) + tuple(data[1].split(H, dim=-1))
            out = ops.differential_attention(*data, heads, lams, s["lambda_init"], norm_weight=weight, mask_bias=s["mask_bias"])
        else:
            out = ops.differential_self_attention(data[0], heads, lams, s["lambda_init"], norm_weight=weight,
                                                  mask_bias=s["mask_bias"], cu_seqlens=s["cu"], max_len=s["max_len"])
        if not s["train"]:
            return out
        leaves = data + lams + (() if weight is None else (weight,))
        return (out,) + torch.autograd.grad(out, leaves, s["dout"])
    data = (s["q"],) + tuple(s["kv"].split(H, dim=-1)) if s["cross"] else (s["qkv"],)
    leaves = [t.float() for t in data + s["lambdas"] + (() if s["norm_weight"] is None else (s["norm_weight"],))]
    if s["train"]:
        leaves = [t.detach().requires_grad_(True) for t in leaves]
    n = len(data)
    lams = leaves[n:n + 4]
    weight = leaves[n + 4] if s["norm_weight"] is not None else None
    q, k, v = leaves[:n] if n == 3 else leaves[0].split(H, dim=-1)
    bias = s["mask_bias"]
    if s["cu"] is not None:                  # rows back to back -> one padded row block per sequence, and back
        cu = s["cu"].long()
        t = torch.arange(q.shape[0], device=q.device)
        b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
        at = cu[:-1, None] + torch.arange(s["max_len"], device=q.device)[None, :]
        bias = torch.where(at < cu[1:, None], 0.0, -math.inf)
        at = at.clamp(max=q.shape[0] - 1)
        q, k, v = q[at], k[at], v[at]
    out = _plain_dattn(q, k, v, lams, s["lambda_init"], weight, bias, heads, dim)
    if s["cu"] is not None:
        out = out[b, t - cu[b]]
    if not s["train"]:
        return out.to(BF16)
    return (out.to(BF16),) + tuple(x.to(BF16) for x in torch.autograd.grad(out, leaves, s["dout"].float()))


def run(state):
    return _run_rotary(state) if state["op"] == "rotary" else _run_dattn(state)


# --------------------------------------------------------------------------------------------------------------------------
# work and exact results
# --------------------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "rotary":
        n = c["B"] * c["L"] * c["heads"] * c["dim"]
        times = 2 if c["train"] else 1
        return {"bytes": times * (4 * n + 8 * c["B"] * c["L"]), "flops": times * 3 * c["B"] * c["L"] * c["heads"] * c["rot"]}
    H = c["heads"] * 2 * c["dim"]
    lens = [(n, n) for n in _lengths(c)] if c["packed"] else [(c["Lq"], c["Lk"])] * c["B"]
    rows_q, rows_k = (sum(n[i] for n in lens) for i in (0, 1))
    pairs = c["heads"] * sum(n * m for n, m in lens)
    flops = 8 * c["dim"] * pairs                                                      # two maps' scores, one product with v
    moved = 2 * H * (2 * rows_q + 2 * rows_k) + (4 * c["B"] * c["Lk"] if c["mask"] != "none" else 0)
    if c["train"]:
        flops += 16 * c["dim"] * pairs                                                # dA, dV, dQ and dK
        moved += 2 * H * (2 * rows_q + 2 * rows_k)                                    # dout read; dq, dk, dv written
    return {"bytes": float(moved), "flops": float(flops)}


def _exact_head(q, k, v, bias, lam, weight, scale_out, dim, dout):
    """One head of one sequence in float64: (out, and with dout: dq, dk, dv, dlambda, dweight)."""
    z = dim ** -0.5
    maps = []
    for j in range(2):
        sc = q[:, j * dim:(j + 1) * dim] @ k[:, j * dim:(j + 1) * dim].T * z
        if bias is not None:
            sc = sc + bias[None, :]
        if sc.shape[1] and bool(torch.isneginf(sc).all()):
            maps.append(torch.zeros_like(sc))
        else:
            maps.append(torch.softmax(sc, dim=-1))
    a = maps[0] - lam * maps[1]
    o = a @ v
    r = (o.square().mean(dim=-1, keepdim=True) + EPS).rsqrt()
    out = o if weight is None else o * r * weight * scale_out
    if dout is None:
        return (out,)
    dw = None
    do = dout
    if weight is not None:
        dw = (dout * o * r * scale_out).sum(dim=0)
        du = dout * weight * scale_out
        do = r * (du - o * r * r * (du * o).mean(dim=-1, keepdim=True))
    dv = a.T @ do
    da = do @ v.T
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    for j, dp in ((0, da), (1, -lam * da)):
        ds = maps[j] * (dp - (dp * maps[j]).sum(dim=-1, keepdim=True)) * z
        dq[:, j * dim:(j + 1) * dim] = ds @ k[:, j * dim:(j + 1) * dim]
        dk[:, j * dim:(j + 1) * dim] = ds.T @ q[:, j * dim:(j + 1) * dim]
    return out, dq, dk, dv, -(da * maps[1]).sum(), dw


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        f, mult = _frequencies(case)
        rot = case["rot"]
        x = _qk(s).double()
        angle = s["positions"].double()[..., None, None] * torch.tensor(f, dtype=torch.float64, device=x.device)
        turn = torch.polar(torch.full_like(angle, mult), angle)                       # a turned pair is a complex product

        def apply(t, by):
            y = t.clone()
            at = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
            w = torch.complex(t[..., at[0]].contiguous(), t[..., at[1]].contiguous()) * by
            y[..., at[0]], y[..., at[1]] = w.real, w.imag
            return y

        y = apply(x, turn)
        return (y, apply(s["dout"].double(), turn.conj())) if case["train"] else y
    heads, dim, train = case["heads"], case["dim"], case["train"]
    w = 2 * dim
    H = heads * w
    if case["cross"]:
        q = s["q"].double()
        k, v = (t.double() for t in s["kv"].split(H, dim=-1))
    else:
        q, k, v = (t.double() for t in s["qkv"].split(H, dim=-1))
    lq1, lk1, lq2, lk2 = (t.double() for t in s["lambdas"])
    e1, e2 = (lq1 * lk1).sum(-1).exp(), (lq2 * lk2).sum(-1).exp()
    lam = e1 - e2 + s["lambda_init"]
    weight = None if s["norm_weight"] is None else s["norm_weight"].double()
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dlam, dweight = torch.zeros_like(lam), torch.zeros(w, dtype=torch.float64, device=q.device)
    cu = None if s["cu"] is None else s["cu"].tolist()
    for b in range(case["B"]):
        at = slice(cu[b], cu[b + 1]) if cu is not None else b
        bias = None if s["mask_bias"] is None else s["mask_bias"][b].double()
        for h in range(heads):
            c = slice(h * w, (h + 1) * w)
            got = _exact_head(q[at][:, c], k[at][:, c], v[at][:, c], bias, lam[h], weight, 1.0 - s["lambda_init"], dim,
                              s["dout"][at][:, c].double() if train else None)
            out[at][:, c] = got[0]
            if train:
                dq[at][:, c], dk[at][:, c], dv[at][:, c] = got[1:4]
                dlam[h] += got[4]
                if weight is not None:
                    dweight += got[5]
    if not train:
        return out
    d1, d2 = (dlam * e1)[:, None], (-dlam * e2)[:, None]
    data = (dq, dk, dv) if case["cross"] else (torch.cat((dq, dk, dv), dim=-1),)
    return (out,) + data + (d1 * lk1, d1 * lq1, d2 * lk2, d2 * lq2) + (() if weight is None else (dweight,))
