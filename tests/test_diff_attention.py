"""Differential attention (ops.differential_attention, ops.differential_self_attention) against its formula in 64 bits.

Tolerances: every comparison is element by element against a bound that is computed, in 64 bits, from the roundings the kernels make
on purpose — the weights P (and dS, and the gradient of o) become bf16 operands, outputs are rounded once — carried through the formula
with absolute values.  U = half a step of bf16, relative.  SLACK covers what is held in 32 bits: a score shifted by a mask of -10000
(14427 in log2 units) is held to 2^-11, which is 2^-11.5 of its exponential; score sums of up to 64 products, exponentials and running
sums add less.
"""
import math

import pytest
import torch

from uniter_amd import _lib, ops

BF16 = torch.bfloat16
U = torch.finfo(BF16).eps / 2
SLACK = 2.0 ** -10
LOWEST = torch.finfo(torch.float32).min


# --------------------------------------------------------------------------------------------------------------------------
# the formula, its gradients and their bounds
# --------------------------------------------------------------------------------------------------------------------------
def one_head(q, k, v, bias, lam, lam_init, w, eps, dim, dy=None, keep=None):
    """One head of one sequence, float64 CPU.  q [Lq, 2 d], k / v [Lk, 2 d], bias [Lk] or None, keep [Lq, Lk] dropout multipliers or None.
    Returns a dict name -> (value, bound)."""
    z = dim ** -0.5
    Lq, Lk = q.shape[0], k.shape[0]
    gone = torch.zeros(Lk, dtype=torch.bool) if bias is None else torch.isneginf(bias)
    k, v = (torch.where(gone[:, None], 0.0, t) for t in (k, v))
    P = []
    for j in range(2):
        s = q[:, j * dim:(j + 1) * dim] @ k[:, j * dim:(j + 1) * dim].T * z
        if bias is not None:
            s = torch.where(gone, -math.inf, (s + bias) if not (bias < -1e30).any() else torch.where(bias < -1e30, LOWEST * 1.0, s + bias))
        e = torch.where(torch.isneginf(s), 0.0, (s - s.amax(1, keepdim=True)).exp()) if Lk else s
        t = e.sum(1, keepdim=True)
        P.append(e / torch.where(t == 0, 1.0, t))
    M = torch.ones(Lq, Lk, dtype=torch.float64) if keep is None else keep
    so = 1.0 - lam_init
    O = [(M * p) @ v for p in P]
    E = [(U + SLACK) * ((M * p) @ v.abs()) for p in P]                                  # weights rounded to bf16
    o, Eo = O[0] - lam * O[1], E[0] + abs(lam) * E[1]
    Eo = Eo + SLACK * (O[0].abs() + abs(lam) * O[1].abs())                              # lambda in 32 bits
    n = o.shape[1]
    if w is None:
        y, Ey = o, Eo
    else:
        r = (o.square().mean(1, keepdim=True) + eps).rsqrt()
        dr = r ** 3 * (o.abs() * Eo).mean(1, keepdim=True)
        y = so * w * o * r
        Ey = so * w.abs() * (r * Eo + o.abs() * dr)
    out = {"out": (y, Ey + (U + SLACK) * y.abs())}
    if dy is None:
        return out
    if w is None:
        do, Edo = dy, torch.zeros_like(dy)
    else:
        du = so * w * dy
        c = r * r * (du * o).mean(1, keepdim=True)
        Ec = 2 * r * dr * (du * o).abs().mean(1, keepdim=True) + r * r * (du.abs() * Eo).mean(1, keepdim=True)
        do = r * (du - o * c)
        Edo = dr * (du - o * c).abs() + r * (Eo * c.abs() + o.abs() * Ec) + SLACK * (r * (du.abs() + o.abs() * c.abs()))
        out["w"] = ((so * dy * o * r).sum(0), (so * dy.abs() * (r * Eo + o.abs() * dr)).sum(0) + SLACK * (so * dy * o * r).abs().sum(0))
    Eg = Edo + (U if w is not None else 0.0) * do.abs()                                 # as an operand
    A = P[0] - lam * P[1]
    Ap = P[0] + abs(lam) * P[1]
    out["v"] = ((M * A).T @ do, (M * (U * A.abs() + SLACK * Ap)).T @ do.abs() + (M * A.abs()).T @ Eg)
    G, EG = M * (do @ v.T), M * (Eg @ v.abs().T) + SLACK * M * (do.abs() @ v.abs().T)
    dq, dk, Eq, Ek = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(q), torch.zeros_like(k)
    for j, f in ((0, 1.0), (1, -lam)):
        c = slice(j * dim, (j + 1) * dim)
        D = (do * O[j]).sum(1, keepdim=True)
        ED = (Edo * O[j].abs() + do.abs() * E[j]).sum(1, keepdim=True) + SLACK * (do * O[j]).abs().sum(1, keepdim=True)
        S = P[j] * (G - D)
        ES = P[j] * (EG + ED) + (U + SLACK) * S.abs() + SLACK * P[j] * (G.abs() + D.abs())
        dq[:, c], Eq[:, c] = f * z * (S @ k[:, c]), abs(f) * z * (ES @ k[:, c].abs())
        dk[:, c], Ek[:, c] = f * z * (S.T @ q[:, c]), abs(f) * z * (ES.T @ q[:, c].abs())
        if j == 1:
            out["lam"] = (-D.sum(), ED.sum())
    out["q"], out["k"] = (dq, Eq), (dk, Ek)
    return out


def whole(q, k, v, heads, lams, lam_init, w, eps, bias=None, spans=None, dy=None, keep=None):
    """All heads and sequences: dict name -> (value, bound) shaped as the op returns them.  spans: [(q slice, k slice)] of packed rows;
    keep: function (sequence, head) -> multipliers."""
    D = torch.float64
    q, k, v = (t.detach().cpu().to(D) for t in (q, k, v))
    lams = [t.detach().cpu().to(D) for t in lams]
    w = None if w is None else w.detach().cpu().to(D)
    dy = None if dy is None else dy.detach().cpu().to(D)
    bias = None if bias is None else bias.cpu().to(D)
    W = q.shape[-1] // heads
    dim = W // 2
    lq1, lk1, lq2, lk2 = (t.expand(heads, dim) for t in lams)
    e1, e2 = (lq1 * lk1).sum(-1).exp(), (lq2 * lk2).sum(-1).exp()
    lam = e1 - e2 + lam_init
    res = {n: [torch.zeros_like(t), torch.zeros_like(t)] for n, t in (("out", q), ("q", q), ("k", k), ("v", v))}
    dl, El = torch.zeros(heads, dtype=D), torch.zeros(heads, dtype=D)
    dw, Ew = torch.zeros(W, dtype=D), torch.zeros(W, dtype=D)
    for b, (sq, sk) in enumerate(spans if spans is not None else [(i, i) for i in range(q.shape[0])]):
        for h in range(heads):
            c = slice(h * W, (h + 1) * W)
            got = one_head(q[sq][:, c], k[sk][:, c], v[sk][:, c], None if bias is None else bias[b], float(lam[h]), lam_init, w, eps, dim,
                           None if dy is None else dy[sq][:, c], None if keep is None else keep(b, h))
            for n, at in (("out", sq), ("q", sq), ("k", sk), ("v", sk)):
                if n in got:
                    for i in range(2):
                        res[n][i][at][:, c] = got[n][i]
            if dy is not None:
                dl[h] += got["lam"][0]
                El[h] += got["lam"][1]
                if w is not None:
                    dw += got["w"][0]
                    Ew += got["w"][1]
    if dy is None:
        return {"out": res["out"]}
    for n, d, s, e, o in (("lq1", dl, 1, e1, lk1), ("lk1", dl, 1, e1, lq1), ("lq2", dl, -1, e2, lk2), ("lk2", dl, -1, e2, lq2)):
        val, bnd = s * (d * e)[:, None] * o, (El * e)[:, None] * o.abs()
        bnd = bnd + SLACK * val.abs()
        if lams[0].dim() == 1:
            val, bnd = val.sum(0), bnd.sum(0)
        res[n] = [val, bnd]
    if w is not None:
        res["w"] = [dw, Ew]
    for n in res:
        if n != "out":
            res[n][1] = res[n][1] + (U + SLACK) * res[n][0].abs()                       # the result's own rounding
    return res


def check(name, got, want):
    val, bound = want
    got = got.detach().cpu().double()
    assert got.shape == val.shape, (name, got.shape, val.shape)
    off = (got - val).abs()
    bad = ~(off <= bound * 1.01 + 1e-30)
    assert not bad.any(), "%s: %d of %d off, worst %.3g at a bound of %.3g (value %.3g)" % (
        name, int(bad.sum()), bad.numel(), float(off[bad].max()), float(bound[bad][off[bad].argmax()]), float(val[bad][off[bad].argmax()]))


# --------------------------------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------------------------------
def params(g, heads, dim, per_head=True, norm=True, std=0.2):
    shape = (heads, dim) if per_head else (dim,)
    lams = tuple((torch.randn(*shape, generator=g) * std).to(BF16).cuda() for _ in range(4))
    w = (1 + 0.2 * torch.randn(2 * dim, generator=g)).to(BF16).cuda() if norm else None
    return lams, w


def mask_of(kind, B, Lk, g):
    if kind == "none" or Lk == 0:
        return None
    m = torch.zeros(B, Lk)
    if kind == "random":
        m = torch.randn(B, Lk, generator=g) * 3
    low = {"pad": -10000.0, "lowest": LOWEST, "inf": -math.inf}.get(kind)
    if low is not None:
        for b in range(B):
            m[b, int(torch.randint(1, Lk + 1, (1,), generator=g)):] = low
        m[0] = low                              # a whole sequence masked: uniform weights, or (-inf) no keys at all
        if kind == "inf" and B > 1:             # and holes in the middle of one
            m[1] = torch.where(torch.rand(Lk, generator=g) < 0.5, low, 0.0)
    return m.cuda()


def leaf(t):
    return None if t is None else t.detach().requires_grad_(True)


def run_all(q, k, v, heads, lams, lam_init, w, dy, **kw):
    """(out, dict of gradients) of differential_attention"""
    q, k, v, w = leaf(q), leaf(k), leaf(v), leaf(w)
    lams = tuple(leaf(t) for t in lams)
    out = ops.differential_attention(q, k, v, heads, lams, lam_init, norm_weight=w, **kw)
    names = ["q", "k", "v", "lq1", "lk1", "lq2", "lk2"] + ([] if w is None else ["w"])
    grads = torch.autograd.grad(out, (q, k, v) + lams + (() if w is None else (w,)), dy)
    return out, dict(zip(names, grads))


CASES = [
    # B, Lq, Lk, heads, dim, mask, per head, norm
    (1, 1, 1, 1, 32, "none", True, True),
    (1, 1, 1, 2, 64, "none", True, False),
    (2, 1, 33, 3, 32, "pad", True, True),
    (3, 31, 65, 1, 64, "inf", True, True),
    (2, 64, 64, 2, 32, "none", False, True),
    (1, 129, 95, 2, 64, "random", True, False),
    (2, 33, 1, 2, 32, "inf", True, True),
    (2, 97, 96, 2, 32, "lowest", True, True),
    (3, 40, 257, 2, 32, "inf", True, False),
    (1, 260, 130, 1, 64, "pad", False, False),
    (2, 300, 200, 1, 32, "random", True, True),
    (1, 5, 700, 2, 64, "inf", True, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Lq,Lk,heads,dim,mask,per_head,norm", CASES)
def test_forward_and_gradients(B, Lq, Lk, heads, dim, mask, per_head, norm):
    g = torch.Generator().manual_seed(Lq * 1000 + Lk)
    H = heads * 2 * dim
    q, k, v, dy = (torch.randn(B, n, H, generator=g).to(BF16).cuda() for n in (Lq, Lk, Lk, Lq))
    lams, w = params(g, heads, dim, per_head, norm)
    bias = mask_of(mask, B, Lk, g)
    want = whole(q, k, v, heads, lams, 0.35, w, 1e-5, bias=bias, dy=dy)
    if mask == "inf":                           # whatever stands in a key that is out for good is not used
        hole = torch.isneginf(bias)[..., None]
        k, v = torch.where(hole, math.nan, k), torch.where(hole, math.inf, v)
    out, grads = run_all(q, k, v, heads, lams, 0.35, w, dy, mask_bias=bias)
    check("out", out, want["out"])
    for n, t in grads.items():
        check("gradient of " + n, t, want[n])
    with torch.no_grad():                       # the form that keeps nothing for a backward pass gives the same bits
        assert torch.equal(out, ops.differential_attention(q, k, v, heads, lams, 0.35, norm_weight=w, mask_bias=bias))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,Lk", [(32, 1), (32, 1000), (64, 4097), (32, 20_011)])
def test_single_tokens_against_long_keys(dim, Lk):
    g = torch.Generator().manual_seed(Lk)
    heads, B = 3, 2
    H = heads * 2 * dim
    q, kv = torch.randn(B, 1, H, generator=g).to(BF16).cuda(), torch.randn(B, Lk, 2 * H, generator=g).to(BF16).cuda()
    k, v = kv.split(H, dim=-1)
    lams, w = params(g, heads, dim)
    for kind in ("none", "inf"):
        bias = mask_of(kind, B, Lk, g)
        want = whole(q, k, v, heads, lams, 0.5, w, 1e-5, bias=bias)
        with torch.no_grad():
            check("out", ops.differential_attention(q, k, v, heads, lams, 0.5, norm_weight=w, mask_bias=bias), want["out"])


@pytest.mark.gpu
@pytest.mark.parametrize("dim,lens_q,lens_k", [(32, [5, 1, 0, 130, 33], None), (64, [64, 3], None), (32, [7, 40, 1, 9], [65, 0, 3, 200])])
def test_packed_rows(dim, lens_q, lens_k):
    g = torch.Generator().manual_seed(len(lens_q) + dim)
    heads, behind = 2, 3                        # rows behind the last sequence
    H = heads * 2 * dim
    same = lens_k is None
    lens_k = lens_q if same else lens_k
    cu = [torch.tensor([0] + list(torch.tensor(n).cumsum(0)), dtype=torch.int32).cuda() for n in (lens_q, lens_k)]
    spans = [(slice(sum(lens_q[:i]), sum(lens_q[:i + 1])), slice(sum(lens_k[:i]), sum(lens_k[:i + 1]))) for i in range(len(lens_q))]
    q, k, v, dy = (torch.randn(sum(n) + behind, H, generator=g).to(BF16).cuda() for n in (lens_q, lens_k, lens_k, lens_q))
    for t in (q, k, v, dy):
        t[-behind:] = math.nan
    lams, w = params(g, heads, dim)
    want = whole(*(torch.nan_to_num(t) for t in (q, k, v)), heads, lams, 0.6, w, 1e-5, spans=spans, dy=torch.nan_to_num(dy))
    kw = dict(cu_seqlens=cu[0], max_len=max(lens_q))
    if not same:
        kw.update(cu_seqlens_k=cu[1], max_len_k=max(lens_k))
    out, grads = run_all(q, k, v, heads, lams, 0.6, w, dy, **kw)
    check("out", out, want["out"])
    for n, t in grads.items():
        check("gradient of " + n, t, want[n])
    if same:
        qkv, w2 = leaf(torch.cat((q, k, v), dim=-1)), leaf(w)
        l2 = tuple(leaf(t) for t in lams)
        out2 = ops.differential_self_attention(qkv, heads, l2, 0.6, norm_weight=w2, **kw)
        d = torch.autograd.grad(out2, (qkv,) + l2 + (w2,), dy)
        assert torch.equal(out2, out) and torch.equal(d[0], torch.cat([grads[n] for n in "qkv"], dim=-1))
        assert all(torch.equal(a, grads[n]) for a, n in zip(d[1:], ("lq1", "lk1", "lq2", "lk2", "w")))


@pytest.mark.gpu
def test_bad_boundaries_read_and_write_nothing_outside():
    """cu_seqlens that do not ascend, or leave the rows there are, are cut to them."""
    g = torch.Generator().manual_seed(3)
    q = torch.randn(50, 128, generator=g).to(BF16).cuda()
    lams, w = params(g, 1, 64)
    for cu in ([0, 30, 20, 50], [0, 10, 10_000_000, 50], [-5, 10, 20, 50]):
        cu = torch.tensor(cu, dtype=torch.int32).cuda()
        out, grads = run_all(q, q, q, 1, lams, 0.5, w, q, cu_seqlens=cu, max_len=50)
        assert torch.isfinite(out).all() and all(torch.isfinite(t).all() for t in grads.values())
    cu = torch.tensor([0, 20, 50], dtype=torch.int32).cuda()               # a sequence longer than max_len says: its first rows only
    out, grads = run_all(q, q, q, 1, lams, 0.5, w, q, cu_seqlens=cu, max_len=20)
    assert not out[40:].any() and not grads["q"][40:].any() and not grads["v"][40:].any() and out[20:40].any()


@pytest.mark.gpu
def test_empty_sizes():
    lams, w = params(torch.Generator().manual_seed(0), 2, 32)
    for B, Lq, Lk in ((0, 4, 4), (2, 0, 3), (2, 3, 0), (1, 0, 0)):
        q, k, dy = (torch.randn(B, n, 128).to(BF16).cuda() for n in (Lq, Lk, Lq))
        out, grads = run_all(q, k, k, 2, lams, 0.5, w, dy)
        assert out.shape == q.shape and not out.any()
        assert all(not t.any() for t in grads.values()) and grads["k"].shape == k.shape


@pytest.mark.gpu
def test_packed_batches_without_rows():
    """A batch of empty examples, and examples without keys, whose tensors have no memory at all."""
    lams, w = params(torch.Generator().manual_seed(1), 2, 32)
    none, cu0 = torch.empty(0, 128, dtype=BF16, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda")
    x = torch.randn(9, 128).to(BF16).cuda()
    for q, k, cq, ck in ((none, none, cu0, cu0), (x, none, cu, cu0), (none, x, cu0, cu)):
        out, grads = run_all(q, k, k, 2, lams, 0.5, w, q, cu_seqlens=cq, cu_seqlens_k=ck, max_len=5, max_len_k=5)
        assert out.shape == q.shape and not out.any()
        assert all(not t.any() for t in grads.values()) and grads["k"].shape == k.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dim,Lq,Lk", [(32, 1, 5000), (64, 130, 700), (32, 300, 300)])
def test_no_key_left_among_many(dim, Lq, Lk):
    """Example 0 has no key at all, example 1 its very last one only, example 2 its first: many tiles (and splits) with nothing in them."""
    g = torch.Generator().manual_seed(Lk)
    H = 2 * 2 * dim
    q, k, v, dy = (torch.randn(3, n, H, generator=g).to(BF16).cuda() for n in (Lq, Lk, Lk, Lq))
    k[0], v[0] = math.nan, math.inf                                        # never used
    bias = torch.full((3, Lk), -math.inf).cuda()
    bias[1, -1], bias[2, 0] = 0.0, 0.0
    lams, w = params(g, 2, dim)
    out, grads = run_all(q, k, v, 2, lams, 0.5, w, dy, mask_bias=bias)
    want = whole(q, k.nan_to_num(0.0), v.nan_to_num(0.0, 0.0), 2, lams, 0.5, w, 1e-5, bias.cpu(), dy=dy)
    assert not out[0].any() and not grads["q"][0].any() and not grads["k"][0].any() and not grads["v"][0].any()
    for n in ("out", "q", "k", "v"):
        value, bound = want[n]
        got = (out if n == "out" else grads[n]).cpu().double()
        over = (got - value).abs() - bound - U * value.abs() - 1e-30
        assert (over <= 0).all(), (n, float(over.max()))


def with_roundings(q, k, v, lam, lam_init, w, dim, dy, rnd):
    """One head in float64, (out, dq, dk, dv); rnd: applied where the kernels round to bf16."""
    S = [q[:, j * dim:(j + 1) * dim] @ k[:, j * dim:(j + 1) * dim].T * dim ** -0.5 for j in range(2)]
    e = [(s - s.amax(1, keepdim=True)).exp() for s in S]
    P = [x / x.sum(1, keepdim=True) for x in e]
    O = [rnd(x) @ v / x.sum(1, keepdim=True) for x in e]
    o = O[0] - lam * O[1]
    r = (o.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    du = (1 - lam_init) * w * dy
    do = rnd(r * (du - o * r * r * (du * o).mean(1, keepdim=True)))
    dS = [rnd(p * (do @ v.T - (do * x).sum(1, keepdim=True))) * f * dim ** -0.5 for f, p, x in ((1.0, P[0], O[0]), (-lam, P[1], O[1]))]
    dq = torch.cat([t @ k[:, j * dim:(j + 1) * dim] for j, t in enumerate(dS)], 1)
    dk = torch.cat([t.T @ q[:, j * dim:(j + 1) * dim] for j, t in enumerate(dS)], 1)
    return rnd((1 - lam_init) * w * o * r), rnd(dq), rnd(dk), rnd(rnd(P[0] - lam * P[1]).T @ do)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,L,shift", [(32, 130, 16.0), (64, 70, 16.0), (32, 40, 4.0), (64, 200, 1.0)])
def test_values_with_a_common_part(dim, L, shift):
    """What all values have in common cancels in G - D, so it must not come back as an error of dQ and dK: these are held to 1.5 times what the
    formula with the kernels' roundings written out is off by (other draws of the same sizes, and the fp32 sums beside them)."""
    g = torch.Generator().manual_seed(L)
    H = 2 * dim
    q, k, v, dy = (torch.randn(L, H, generator=g) for _ in range(4))
    q, k, v, dy = (t.to(BF16) for t in (q, k, v + shift, dy))
    lams, w = params(g, 1, dim)
    out, grads = run_all(*(t[None].cuda() for t in (q, k, v)), 1, lams, 0.5, w, dy[None].cuda())
    l = [t.double().cpu()[0] for t in lams]
    lam = float((l[0] * l[1]).sum().exp() - (l[2] * l[3]).sum().exp() + 0.5)
    args = [t.double() for t in (q, k, v)] + [lam, 0.5, w.double().cpu(), dim, dy.double()]
    exact, rounded = (with_roundings(*args, rnd) for rnd in (lambda t: t, lambda t: t.to(BF16).double()))
    for n, got, x, y in zip(("out", "q", "k", "v"), (out, grads["q"], grads["k"], grads["v"]), exact, rounded):
        off, room = float((got[0].double().cpu() - x).norm() / x.norm()), float((y - x).norm() / x.norm())
        assert off < 1.5 * room, (n, off, room)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,Lq,Lk", [(32, 1, 3000), (64, 40, 70), (32, 70, 40), (64, 1, 3000)])
def test_a_mask_entry_that_is_nan_shows(dim, Lq, Lk):
    """Every score sum of that example holds it: NaN in all its rows and gradients, as in the formula; the other example is as without it."""
    g = torch.Generator().manual_seed(Lk + dim)
    H = 2 * 2 * dim
    q, k, v, dy = (torch.randn(2, n, H, generator=g).to(BF16).cuda() for n in (Lq, Lk, Lk, Lq))
    lams, w = params(g, 2, dim)
    bias = torch.zeros(2, Lk).cuda()
    want, grads = run_all(q, k, v, 2, lams, 0.5, w, dy, mask_bias=bias)
    for at in (0, Lk // 2, Lk - 1):
        bad = bias.clone()
        bad[1, at] = math.nan
        assert whole(q[1:], k[1:], v[1:], 2, lams, 0.5, w, 1e-5, bias=bad[1:])["out"][0].isnan().all()
        out, d = run_all(q, k, v, 2, lams, 0.5, w, dy, mask_bias=bad)
        assert out[1].isnan().all() and all(d[n][1].isnan().all() for n in "qkv") and all(d[n].isnan().all() for n in ("lq1", "w"))
        assert torch.equal(out[0], want[0]) and all(torch.equal(d[n][0], grads[n][0]) for n in "qkv")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [32, 64])
def test_one_token_after_the_other_against_a_cache(dim):
    """Serving: a prompt of 37 tokens, then single ones; keys are turned straight into a cache that is longer than what it holds (NaN behind),
    queries attend to what is there.  Every step against the formula on the same turned queries and keys."""
    from uniter_amd.model.rotary import RotaryPositions
    g = torch.Generator().manual_seed(dim)
    B, heads, room, prompt, end = 2, 3, 80, 37, 66
    H = heads * 2 * dim
    rot = RotaryPositions(dim, scaling={"type": "linear", "factor": 2.0})
    lams, w = params(g, heads, dim)
    x = torch.randn(B, end, 3 * H, generator=g).to(BF16).cuda()
    cache = torch.full((2, B, room, H), math.nan, dtype=BF16, device="cuda")
    at = 0
    with torch.no_grad():
        for n in [prompt] + [1] * (end - prompt):
            q, k, v = x[:, at:at + n].split(H, dim=-1)
            q = ops.rotary(q.unflatten(-1, (2 * heads, dim)), None, rot, offset=at).flatten(2)
            ops.rotary(k.unflatten(-1, (2 * heads, dim)), None, rot, offset=at, out=cache[0, :, at:at + n].unflatten(-1, (2 * heads, dim)))
            cache[1, :, at:at + n] = v
            at += n
            out = ops.differential_attention(q, cache[0, :, :at], cache[1, :, :at], heads, lams, 0.4, norm_weight=w)
            value, bound = whole(q, cache[0, :, :at], cache[1, :, :at], heads, lams, 0.4, w, 1e-5)["out"]
            over = (out.cpu().double() - value).abs() - bound - U * value.abs()
            assert (over <= 0).all(), (at, float(over.max()))
    whole_prompt = ops.rotary(x[..., H:2 * H].unflatten(-1, (2 * heads, dim)), None, rot).flatten(2)
    assert torch.equal(cache[0, :, :end], whole_prompt) and cache[0, :, end:].isnan().all()


@pytest.mark.gpu
def test_strides_and_alignment():
    g = torch.Generator().manual_seed(9)
    heads, dim, B, L = 2, 32, 2, 45
    H = heads * 2 * dim
    qkv, dy = torch.randn(B, L, 3 * H, generator=g).to(BF16).cuda(), torch.randn(B, L, H, generator=g).to(BF16).cuda()
    lams, w = params(g, heads, dim)
    bias = mask_of("pad", B, L, g)
    parts = [t.contiguous() for t in qkv.split(H, dim=-1)]
    out, grads = run_all(*parts, heads, lams, 0.4, w, dy, mask_bias=bias)
    views = [
        qkv.split(H, dim=-1),                                                                       # slices of one projection
        [t.transpose(0, 1).contiguous().transpose(0, 1) for t in parts],                            # [L, B, H] underneath
        [torch.empty(B, L, H + 1, dtype=BF16, device="cuda")[..., 1:].copy_(t) for t in parts],     # rows on 2 bytes
        [t.transpose(1, 2).contiguous().transpose(1, 2) for t in parts],                            # columns strided
        [torch.stack((t, t), dim=1)[:, 0] for t in parts],                                          # batch stride twice the size
    ]
    wide = torch.empty(B, L + 3, device="cuda")[:, :L].copy_(bias)
    for vs in views:
        o2, g2 = run_all(*vs, heads, lams, 0.4, w, dy.transpose(0, 1).contiguous().transpose(0, 1), mask_bias=wide)
        assert torch.equal(o2, out) and all(torch.equal(g2[n], grads[n]) for n in grads)
    q = leaf(qkv)
    o2 = ops.differential_self_attention(q, heads, lams, 0.4, norm_weight=w, mask_bias=bias[:, None, None, :])
    assert torch.equal(o2, out)
    assert torch.equal(torch.autograd.grad(o2, q, dy)[0], torch.cat([grads[n] for n in "qkv"], dim=-1))
    one = qkv[:1].expand(3, L, 3 * H)                                                               # a broadcast batch: its gradient adds up
    q1 = leaf(qkv[:1])
    d3 = dy[:1].expand(3, L, H)
    d, = torch.autograd.grad(ops.differential_self_attention(q1.expand(3, L, 3 * H), heads, lams, 0.4, norm_weight=w), q1, d3)
    o1 = ops.differential_self_attention(q1, heads, lams, 0.4, norm_weight=w)
    ref, = torch.autograd.grad(o1, q1, dy[:1])
    assert torch.equal(ops.differential_self_attention(one, heads, lams, 0.4, norm_weight=w)[2], o1[0])
    # three equal bf16 terms: two additions, each rounded by at most U of a sum of up to three terms
    assert ((d - 3 * ref.float()).abs() <= 2 * U * 3 * ref.float().abs() * 1.01 + 1e-30).all()


@pytest.mark.gpu
@pytest.mark.parametrize("B,L", [(1, 7), (3, 1), (1, 1)])
def test_strides_that_nothing_steps_over(B, L):
    """A dimension of one has a stride that no address uses: any value of it is taken."""
    g = torch.Generator().manual_seed(31)
    heads, dim = 2, 32
    H = heads * 2 * dim
    lams, w = params(g, heads, dim)
    parts = [torch.randn(B, L, H, generator=g).to(BF16).cuda() for _ in range(4)]

    def odd(t):                     # the strides of dimensions of one are 5 and 2^24 + 3
        room = torch.zeros(B * L * H, dtype=BF16, device="cuda")
        return room.as_strided((B, L, H), (L * H if B > 1 else 5, H if L > 1 else (1 << 24) + 3, 1)).copy_(t)

    def both(q, k, v, dy):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        y = ops.differential_attention(q, k, v, heads, lams, 0.4, norm_weight=w)
        return [y.detach(), *torch.autograd.grad(y, (q, k, v), dy)]

    for a, b in zip(both(*map(odd, parts)), both(*parts)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_scores_of_any_size():
    """Large scores: one key takes all the weight of a map; the running maximum moves late in the row."""
    g = torch.Generator().manual_seed(4)
    heads, dim, L = 1, 32, 200
    q = torch.randn(1, L, 64, generator=g)
    k = torch.randn(1, L, 64, generator=g)
    k *= torch.linspace(0.01, 40, L)[None, :, None]                       # scores up to several hundred, growing along the row
    v, dy = torch.randn(1, L, 64, generator=g), torch.randn(1, L, 64, generator=g)
    q, k, v, dy = (t.to(BF16).cuda() for t in (q, k, v, dy))
    lams, w = params(g, heads, dim)
    want = whole(q, k, v, heads, lams, 0.3, None, 1e-5, dy=dy)
    out, grads = run_all(q, k, v, heads, lams, 0.3, None, dy)
    # scores of size 2^9 carry 2^9 * 2^-24 * a few into the exponent: SLACK covers it
    check("out", out, want["out"])
    check("gradient of v", grads["v"], want["v"])
    big = torch.full((1, 70, 64), 200.0).to(BF16).cuda()                   # equal scores of 226 000: no overflow, uniform weights
    out = ops.differential_attention(big, big, v[:, :70], 1, lams, 0.3)
    mean = v[:, :70].double().mean(1, keepdim=True)
    lam = sum(s * (a.double() * b.double()).sum().exp() for s, a, b in ((1, lams[0], lams[1]), (-1, lams[2], lams[3]))) + 0.3
    bound = (U + SLACK) * ((1 + abs(float(lam))) * v[:, :70].double().abs().mean(1, keepdim=True)) + U * mean.abs()
    assert ((out.double() - (1 - lam) * mean).abs() <= bound * 1.01).all()


# ---- dropout: the kernels' counter-based draws, restated -------------------------------------------------------------------
def philox(c, key, rounds=7):
    """c: four int64 tensors holding 32 bits each."""
    m32 = 0xFFFFFFFF
    c0, c1, c2, c3 = c
    k0, k1 = key
    for _ in range(rounds):
        p0, p1 = 0xD2511F53 * c0, 0xCD9E8D57 * c2                          # (low 64 bits; the high word by shift)
        hi0, lo0, hi1, lo1 = (p0 >> 32) & m32, p0 & m32, (p1 >> 32) & m32, p1 & m32
        c0, c1, c2, c3 = hi1 ^ c1 ^ k0, lo1, hi0 ^ c3 ^ k1, lo0
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    return c0, c1, c2, c3


def keep_of(seed, offset, p, bh, Lq_max, Lk_max, Lq, Lk):
    """Multipliers [Lq, Lk] of one (sequence, head): one call per (row, 16 keys, half of every 8)."""
    thresh = int(p * 65536.0 + 0.5)
    q, k = torch.arange(Lq)[:, None], torch.arange(Lk)[None, :]
    group = ((bh * Lq_max + q) * ((Lk_max + 15) // 16) + k // 16) * 2 + (k // 4) % 2
    field = ((k // 8) % 2) * 4 + k % 4
    zero = torch.zeros_like(group)
    words = torch.stack(philox((group & 0xFFFFFFFF, group >> 32, zero + (offset & 0xFFFFFFFF), zero + (offset >> 32)),
                               (seed & 0xFFFFFFFF, seed >> 32)))
    word = words.gather(0, (field // 2).expand(Lq, Lk)[None])[0]
    bits = (word >> (16 * (field % 2))) & 0xFFFF
    return torch.where(bits >= thresh, 65536.0 / (65536 - thresh), 0.0).double()


def test_restated_generator_is_the_published_one():
    """Known-answer vectors of the generator's 10-round form (Salmon et al., SC'11)."""
    def run(c, k):
        return [int(x) for x in philox([torch.tensor(v) for v in c], k, rounds=10)]
    assert run([0, 0, 0, 0], (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    f = 0xFFFFFFFF
    assert run([f, f, f, f], (f, f)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.gpu
@pytest.mark.parametrize("dim,Lq,Lk,packed", [(32, 45, 70, False), (64, 33, 130, False), (32, 60, 60, True), (64, 1, 40, False)])
def test_dropout(dim, Lq, Lk, packed):
    g = torch.Generator().manual_seed(dim + Lq)
    heads, p, seed = 2, 0.25, 1234567890123
    H = heads * 2 * dim
    lams, w = params(g, heads, dim)
    if packed:
        lens = [Lq, 7, 20]
        cu = torch.tensor([0, Lq, Lq + 7, Lq + 27], dtype=torch.int32).cuda()
        q, k, v, dy = (torch.randn(sum(lens), H, generator=g).to(BF16).cuda() for _ in range(4))
        spans = [(slice(int(a), int(b)),) * 2 for a, b in zip(cu[:-1], cu[1:])]
        kw, sizes = dict(cu_seqlens=cu, max_len=Lq), [(n, n) for n in lens]
    else:
        q, k, v, dy = (torch.randn(2, n, H, generator=g).to(BF16).cuda() for n in (Lq, Lk, Lk, Lq))
        spans, kw, sizes = None, {}, [(Lq, Lk)] * 2
    ops.manual_seed(seed)
    ops._next_offsets(5)
    want = whole(q, k, v, heads, lams, 0.45, w, 1e-5, spans=spans, dy=dy,
                 keep=lambda b, h: keep_of(seed, 5, p, b * heads + h, Lq, Lk, *sizes[b]))
    out, grads = run_all(q, k, v, heads, lams, 0.45, w, dy, p_drop=p, **kw)
    check("out", out, want["out"])
    for n, t in grads.items():
        check("gradient of " + n, t, want[n])
    assert not torch.equal(out, run_all(q, k, v, heads, lams, 0.45, w, dy, p_drop=p, **kw)[0])    # the next call draws anew


# ---- how it is called ------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_same_bits_every_time_on_any_stream_and_from_graphs():
    g = torch.Generator().manual_seed(77)
    heads, dim = 3, 32
    qkv = torch.randn(4, 150, 3 * heads * 64, generator=g).to(BF16).cuda()
    dy = torch.randn(4, 150, heads * 64, generator=g).to(BF16).cuda()
    lams, w = params(g, heads, dim)

    def step(x):
        x = leaf(x)
        out = ops.differential_self_attention(x, heads, lams, 0.5, norm_weight=w)
        return out, torch.autograd.grad(out, x, dy)[0]

    want = step(qkv)
    again = step(qkv)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    other = [qkv, qkv.flip(0).contiguous()]
    want2 = step(other[1])
    torch.cuda.synchronize()
    got = []
    for i in range(6):                          # two streams at work at once
        with torch.cuda.stream(streams[i % 2]):
            got.append(step(other[i % 2]))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(o, (want, want2)[i % 2]))
    # one token against many keys, two captured graphs that share the pool, replayed in turn
    q1 = [torch.randn(2, 1, heads * 64, generator=g).to(BF16).cuda() for _ in range(2)]
    kv = torch.randn(2, 5000, 2 * heads * 64, generator=g).to(BF16).cuda()
    k, v = kv.split(heads * 64, dim=-1)
    graphs, outs = [], []
    with torch.no_grad():
        ops.differential_attention(q1[0], k, v, heads, lams, 0.5, norm_weight=w)
        torch.cuda.synchronize()
        pool = torch.cuda.graph_pool_handle()
        for i in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, pool=pool):
                outs.append(ops.differential_attention(q1[i], k, v, heads, lams, 0.5, norm_weight=w))
            graphs.append(gr)
        for r in range(3):
            kv.mul_(0.5 + r)
            for i in range(2):
                graphs[i].replay()
                torch.cuda.synchronize()
                assert torch.equal(outs[i], ops.differential_attention(q1[i], k, v, heads, lams, 0.5, norm_weight=w))


@pytest.mark.gpu
def test_captured_training_step():
    g = torch.Generator().manual_seed(5)
    heads, dim = 2, 64
    x = torch.randn(2, 70, 3 * heads * 128, generator=g).to(BF16).cuda().requires_grad_(True)
    dy = torch.randn(2, 70, heads * 128, generator=g).to(BF16).cuda()
    lams, w = params(g, heads, dim)
    lams = tuple(leaf(t) for t in lams)

    def step():
        out = ops.differential_self_attention(x, heads, lams, 0.5, norm_weight=w)
        return (out,) + torch.autograd.grad(out, (x,) + lams, dy)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = step()
    for i in range(3):
        with torch.no_grad():
            x.mul_(0.9)
            dy.mul_(-1)
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
def test_gradient_against_differences():
    """<out(x + h) - out(x - h), dy> / 2 against <grad, h> for steps h in q, k, v, lambda and w together.  Both outs carry their bound
    from whole(); the third-order term of the difference is bounded by the same difference of the 64-bit formula."""
    g = torch.Generator().manual_seed(12)
    heads, dim, L = 2, 32, 48
    H = heads * 2 * dim
    base = [torch.randn(1, L, H, generator=g).to(BF16).double() for _ in range(3)]
    lam = [(torch.randn(heads, dim, generator=g) * 0.2).to(BF16).double() for _ in range(4)]
    w = [(1 + 0.2 * torch.randn(2 * dim, generator=g)).to(BF16).double()]
    dy = torch.randn(1, L, H, generator=g).to(BF16).cuda()
    point = base + lam + w
    h = [torch.randn(t.shape, generator=g).to(BF16).double() * 2.0 ** -5 for t in point]

    def at(s):
        return [(t + s * d).to(BF16).cuda() for t, d in zip(point, h)]

    def args(ts):
        return (*ts[:3], heads, tuple(ts[3:7]), 0.4)

    up, down, mid = at(1.0), at(-1.0), at(0.0)
    step = [(a.double() - b.double()).cpu() / 2 for a, b in zip(up, down)]            # the step really taken, after rounding
    with torch.no_grad():
        diff = ops.differential_attention(*args(up), norm_weight=up[7]).double() - ops.differential_attention(*args(down), norm_weight=down[7]).double()
    got = float((diff * dy.double()).sum()) / 2
    _, grads = run_all(*args(mid), mid[7], dy)
    lin = sum(float((grads[n].double().cpu() * d).sum()) for n, d in zip(("q", "k", "v", "lq1", "lk1", "lq2", "lk2", "w"), step))
    f = [whole(*args(ts), ts[7], 1e-5, dy=dy) for ts in (up, down, mid)]
    true = float(((f[0]["out"][0] - f[1]["out"][0]) * dy.double().cpu()).sum()) / 2
    slope = sum(float((f[2][n][0] * d).sum()) for n, d in zip(("q", "k", "v", "lq1", "lk1", "lq2", "lk2", "w"), step))
    noise = float(((f[0]["out"][1] + f[1]["out"][1]) * dy.double().cpu().abs()).sum()) / 2
    slack = sum(float((f[2][n][1] * d.abs()).sum()) for n, d in zip(("q", "k", "v", "lq1", "lk1", "lq2", "lk2", "w"), step))
    assert abs(slope - true) <= 0.1 * abs(true)                                       # the step is small enough to say something
    assert abs(got - lin) <= noise + slack + abs(true - slope)


def test_formula_gradients_against_differences():
    """The 64-bit gradients of whole() against central differences of its own output, over every input (CPU)."""
    g = torch.Generator().manual_seed(1)
    heads, dim, Lq, Lk = 2, 32, 5, 7
    H = heads * 2 * dim
    names = ("q", "k", "v", "lq1", "lk1", "lq2", "lk2", "w")
    point = [torch.randn(1, n, H, generator=g).double() for n in (Lq, Lk, Lk)] + [torch.randn(heads, dim, generator=g).double() * 0.2 for _ in range(4)]
    point.append(1 + 0.2 * torch.randn(2 * dim, generator=g).double())
    dy = torch.randn(1, Lq, H, generator=g).double()
    bias = torch.tensor([[0.0, -1.0, -math.inf, 0.5, 0.0, -10000.0, 0.0]])
    keep = (torch.rand(heads, Lq, Lk, generator=g) > 0.3).double() / 0.7

    def f(ts, dy=None):
        return whole(*ts[:3], heads, tuple(ts[3:7]), 0.4, ts[7], 1e-5, bias=bias, dy=dy, keep=lambda b, h: keep[h])

    res = f(point, dy)
    for i, n in enumerate(names):
        for _ in range(3):
            d = torch.randn(point[i].shape, generator=g).double()
            up, down = ([t + s * d if j == i else t for j, t in enumerate(point)] for s in (1e-6, -1e-6))
            num = float(((f(up)["out"][0] - f(down)["out"][0]) * dy).sum()) / 2e-6
            ana = float((res[n][0] * d).sum())
            assert abs(num - ana) <= 1e-5 * (abs(ana) + float((res[n][0] * d).abs().sum())), (n, num, ana)


# ---- refusals --------------------------------------------------------------------------------------------------------------
def test_bad_c_arguments_are_refused():
    import ctypes
    lib = _lib.load()

    def args(**kw):
        a = _lib.UniterDiffAttention()
        a.q = a.k = a.v = a.lambda_q1 = a.lambda_k1 = a.lambda_q2 = a.lambda_k2 = 4096
        a.q_row = a.k_row = a.v_row = 64
        a.B = a.Lq = a.Lk = a.heads = 1
        a.head_dim = 32
        for n, x in kw.items():
            setattr(a, n, x)
        return a

    def refused(text, out=4096, row=64, stats=None, maps=None, **kw):
        a = args(**kw)
        assert lib.uniter_diff_attention_fwd(ctypes.byref(a), out, row, 0, stats, maps, None, 0, None) < 0, kw
        assert text in lib.uniter_hip_last_error(), (kw, lib.uniter_hip_last_error())

    refused(b"head_dim", head_dim=48)
    refused(b"head", heads=0)
    refused(b"length", Lq=-1)
    refused(b"length", Lk=1 << 31)
    refused(b"cu_seqlens", cu_seqlens_q=4096)
    refused(b"mask", cu_seqlens_q=4096, cu_seqlens_k=4096, mask_bias=4096)
    refused(b"dropout", p_drop=1.0)
    refused(b"strides", k_row=60)
    refused(b"strides", row=4)
    refused(b"aligned", q=4100)
    refused(b"aligned", out=4104)
    refused(b"null", q=None)
    refused(b"null", lambda_k2=None)
    refused(b"null", out=None)
    refused(b"together", stats=4096)
    refused(b"2^24", k_row=1 << 24)
    refused(b"workspace", Lk=100_000)
    refused(b"too many", B=1 << 20, heads=64, Lq=1 << 12)
    a, g = args(), _lib.UniterDiffAttentionGrads()
    n = lib.uniter_diff_attention_bwd_workspace_bytes(ctypes.byref(a))
    assert n > 0 and lib.uniter_diff_attention_bwd_workspace_bytes(ctypes.byref(args(head_dim=40))) == 0
    assert lib.uniter_diff_attention_bwd(ctypes.byref(a), 4096, 4096, 4096, 64, 0, ctypes.byref(g), 4096, n, None) < 0      # no dq
    g.q = g.k = g.v = 4096
    g.q_row = g.k_row = g.v_row = 64
    assert lib.uniter_diff_attention_bwd(ctypes.byref(a), 4096, 4096, 4096, 64, 0, ctypes.byref(g), 4096, n - 1, None) < 0
    assert b"workspace" in lib.uniter_hip_last_error()
    g.norm_weight = 4096
    assert lib.uniter_diff_attention_bwd(ctypes.byref(a), 4096, 4096, 4096, 64, 0, ctypes.byref(g), 4096, n, None) < 0
    assert lib.uniter_diff_attention_fwd(ctypes.byref(args(B=0)), None, 0, 0, None, None, None, 0, None) == 0


def test_bad_c_arguments_of_empty_calls_are_refused():
    """Key rows without query rows: dK and dV are written (zeros), so k, v and their gradients have to be there."""
    import ctypes
    lib = _lib.load()
    a, g = _lib.UniterDiffAttention(), _lib.UniterDiffAttentionGrads()
    a.lambda_q1 = a.lambda_k1 = a.lambda_q2 = a.lambda_k2 = 4096
    a.B = a.heads = a.Lk = 1
    a.head_dim, a.k_row, a.v_row, g.k_row, g.v_row, g.k, g.v = 32, 64, 64, 64, 64, 4096, 4096

    def bwd():
        n = lib.uniter_diff_attention_bwd_workspace_bytes(ctypes.byref(a))
        return lib.uniter_diff_attention_bwd(ctypes.byref(a), None, None, None, 0, 0, ctypes.byref(g), 4096, n, None), lib.uniter_hip_last_error()

    assert bwd()[0] < 0 and b"null" in bwd()[1]                            # k and v missing
    a.k = a.v = 4096
    g.v = None
    assert bwd()[0] < 0 and b"null" in bwd()[1]
    a.Lq, a.q, a.q_row, a.norm_weight = 1, 4096, 64, 4096                  # an eps of 0 with a norm: a row of zeros would be 0 / 0
    assert lib.uniter_diff_attention_fwd(ctypes.byref(a), 4096, 64, 0, None, None, None, 0, None) < 0
    assert b"norm_eps" in lib.uniter_hip_last_error()
    a.norm_weight, a.cu_seqlens_q, a.cu_seqlens_k, a.q, a.k = None, 4096, 4096, None, None
    assert lib.uniter_diff_attention_fwd(ctypes.byref(a), None, 64, 0, None, None, None, 0, None) == 0        # no rows at all


def test_cpu_tensors_are_refused():
    t, l = torch.zeros(1, 2, 64, dtype=BF16), torch.zeros(1, 32, dtype=BF16)
    with pytest.raises(_lib.UniterHipError, match="CUDA"):
        ops.differential_attention(t, t, t, 1, (l, l, l, l), 0.5)


def _modes_are_refused(q, k, v, lams, w, bias):
    import torch.autograd.forward_ad as fwAD
    args = [q, k, v, *lams, w, bias]

    def call(ts):
        return ops.differential_attention(*ts[:3], 1, ts[3:7], 0.5, norm_weight=ts[7], mask_bias=ts[8])

    with fwAD.dual_level():
        for i, t in enumerate(args):
            with pytest.raises(_lib.UniterHipError, match="forward-mode"):
                call([fwAD.make_dual(a, torch.ones_like(a)) if a is t else a for a in args])
    with pytest.raises(_lib.UniterHipError, match="trace"):
        torch.jit.trace(lambda a: call([a] + args[1:]), (q,), check_trace=False)


def _mode_inputs(dev):
    c = dict(dtype=BF16, device=dev)
    return [torch.zeros(1, 2, 64, **c) for _ in range(3)] + [tuple(torch.zeros(1, 32, **c) for _ in range(4)), torch.ones(64, **c), torch.zeros(1, 2, device=dev)]


def test_forward_mode_and_tracing_are_refused_first():
    """(whatever else the call may have wrong: here, tensors on the CPU)"""
    import torch.autograd.forward_ad as fwAD
    q, k, v, lams, w, bias = _mode_inputs("cpu")
    with fwAD.dual_level():
        with pytest.raises(_lib.UniterHipError, match="forward-mode"):
            ops.differential_attention(q, fwAD.make_dual(k, torch.ones_like(k)), v, 1, lams, 0.5)
    with pytest.raises(_lib.UniterHipError, match="trace"):
        torch.jit.trace(lambda a: ops.differential_attention(a, k, v, 1, lams, 0.5), (q,), check_trace=False)


@pytest.mark.gpu
def test_forward_mode_and_tracing_are_refused():
    args = _mode_inputs("cuda")
    _modes_are_refused(*args)
    q, k, v, lams, w, bias = args
    assert ops.differential_attention(q, k, v, 1, lams, 0.5, norm_weight=w, mask_bias=bias).shape == q.shape      # nothing is left over


@pytest.mark.gpu
def test_a_mask_that_wants_a_gradient_is_refused():
    q, k, v, lams, w, bias = _mode_inputs("cuda")
    learned = bias.clone().requires_grad_(True)
    for m in (learned, 2 * learned, learned[:, None, None, :]):
        with pytest.raises(_lib.UniterHipError, match="mask_bias"):
            ops.differential_attention(q, k, v, 1, lams, 0.5, mask_bias=m)
        with torch.no_grad():
            assert torch.equal(ops.differential_attention(q, k, v, 1, lams, 0.5, mask_bias=m), ops.differential_attention(q, k, v, 1, lams, 0.5, mask_bias=m.detach()))
    ops.differential_attention(q, k, v, 1, lams, 0.5, mask_bias=learned.detach())


@pytest.mark.gpu
def test_refusals():
    c = dict(dtype=BF16, device="cuda")
    q, k, l = torch.zeros(2, 3, 128, **c), torch.zeros(2, 4, 128, **c), torch.zeros(2, 32, **c)
    lam, w = (l, l, l, l), torch.ones(64, **c)
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    f = ops.differential_attention
    for bad in (lambda: f(q, k, k, 3, lam, 0.5), lambda: f(q.float(), k, k, 2, lam, 0.5), lambda: f(q, k[:1], k[:1], 2, lam, 0.5),
                lambda: f(q, k, k[:, :3], 2, lam, 0.5), lambda: f(q, k, k, 2, lam[:3], 0.5), lambda: f(q, k, k, 2, (l, l, l, l[0]), 0.5),
                lambda: f(q, k, k, 2, (l.float(),) * 4, 0.5), lambda: f(q, k, k, 2, lam, 0.5, norm_weight=w[:32]),
                lambda: f(q, k, k, 2, lam, 0.5, mask_bias=torch.zeros(2, 3, device="cuda")),
                lambda: f(q, k, k, 2, lam, 0.5, mask_bias=torch.zeros(2, 4, **c)), lambda: f(q, k, k, 2, lam, 0.5, p_drop=1.0),
                lambda: f(q, k, k, 2, lam, 0.5, cu_seqlens=cu, max_len=3), lambda: f(q[0], k[0], k[0], 2, lam, 0.5, cu_seqlens=cu),
                lambda: f(q[0], k[0], k[0], 2, lam, 0.5, cu_seqlens=cu.long(), max_len=3), lambda: f(q[0], k[0], k[0], 2, lam, 0.5),
                lambda: f(q[0], k[0], k[0], 2, lam, 0.5, cu_seqlens_k=cu, max_len=3),
                lambda: f(q[0], k[0], k[0], 2, lam, 0.5, cu_seqlens=cu, max_len=3, mask_bias=torch.zeros(1, 3, device="cuda")),
                lambda: f(q, k.cpu(), k, 2, lam, 0.5), lambda: f(q, k, None, 2, lam, 0.5), lambda: f(q, None, None, 2, lam, 0.5),
                lambda: f(q, k, k, 2, (l, l, l, l.cpu()), 0.5), lambda: f(q, k, k, 2, lam, 0.5, norm_weight=w.float()),
                lambda: f(q, k, k, 2, lam, 0.5, mask_bias=torch.zeros(2, 4)),
                lambda: f(q, k, k, 2, lam, 0.5, mask_bias=torch.zeros(2, 1, 3, 4, device="cuda")), lambda: ops.differential_self_attention(q, 2, lam, 0.5)):
        with pytest.raises(_lib.UniterHipError):
            bad()
    with pytest.raises(_lib.UniterHipError, match="eps"):
        f(q, k, k, 2, lam, 0.5, norm_weight=w, eps=0.0)
    x = q.clone().requires_grad_(True)
    first, = torch.autograd.grad(f(x, k, k, 2, lam, 0.5), x, q, create_graph=True)
    with pytest.raises(RuntimeError):                                       # no second derivative
        torch.autograd.grad(first.sum(), x)
    dy = q.clone().requires_grad_(True)
    first, = torch.autograd.grad(f(x, k, k, 2, lam, 0.5), x, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.float().square().sum(), dy)
