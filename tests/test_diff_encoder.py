"""The encoder with differential attention and rotary positions (config.attention_type = "differential"), as a model uses them:
projection, rotary positions, differential attention, output block, intermediate, output — against the same layers in plain float32."""
import copy
import math

import pytest
import torch

from tests.common import cosine, rel_l2
from uniter_amd import _lib, ops
from uniter_amd.model.layer import BertDifferentialSelfAttention, BertLayer, BertSelfAttention, is_differential
from uniter_amd.model.model import UniterConfig, UniterEncoder, UniterModel
from uniter_amd.utils.arena import flatten_model

BF16 = torch.bfloat16
U = torch.finfo(BF16).eps / 2


def config(heads=2, hidden=128, layers=2, rotary=None, p=0.0, **kw):
    c = UniterConfig(100, hidden_size=hidden, num_hidden_layers=layers, num_attention_heads=heads, intermediate_size=2 * hidden,
                     hidden_dropout_prob=p, attention_probs_dropout_prob=p, max_position_embeddings=64)
    c.attention_type = "differential"
    c.rotary = rotary
    for k, v in kw.items():
        setattr(c, k, v)
    return c


ROTARY = {"rotary_dim": 16, "scaling": {"type": "yarn", "factor": 4.0, "original_max_position": 128}}


# ---- construction (CPU) ----------------------------------------------------------------------------------------------------
def test_default_configuration_builds_what_it_always_did():
    c = UniterConfig(100, hidden_size=128, num_hidden_layers=2, num_attention_heads=2, intermediate_size=256)
    e = UniterEncoder(c)
    assert all(type(l.attention.self) is BertSelfAttention and not is_differential(l) for l in e.layer)
    assert not any("lambda" in n for n in e.state_dict())
    assert "attention_type" not in c.to_dict()


def test_differential_configuration():
    e = UniterEncoder(config(rotary=ROTARY, layers=3))
    for i, l in enumerate(e.layer):
        att = l.attention.self
        assert type(att) is BertDifferentialSelfAttention and abs(att.lambda_init - (0.8 - 0.6 * math.exp(-0.3 * i))) < 1e-12
        assert att.lambda_q1.shape == (2, 32) and att.LayerNorm.weight.shape == (64,) and att.rotary.rotary_dim == 16
    names = set(e.state_dict())
    assert {"layer.0.attention.self.%s" % n for n in ("lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2", "LayerNorm.weight", "query.weight")} <= names
    again = UniterEncoder(config(rotary=ROTARY, layers=3))
    again.load_state_dict(e.state_dict())
    assert BertLayer(config(heads=1, hidden=128)).attention.self.map_size == 64
    d = config(rotary=ROTARY).to_dict()
    assert UniterConfig.from_dict(d).rotary == ROTARY


@pytest.mark.parametrize("kw", [dict(heads=4), dict(attention_type="other"), dict(rotary={"rotary_dim": 5}),
                                dict(attention_type="softmax", rotary=ROTARY)])
def test_bad_configurations_are_refused(kw):
    with pytest.raises(_lib.UniterHipError):
        BertLayer(config(**kw))


def test_arena_holds_every_parameter():
    e = UniterEncoder(config(rotary=ROTARY)).bfloat16()
    before = {n: p.detach().clone() for n, p in e.named_parameters()}
    arena = flatten_model(e)
    assert len(arena.params) == len(before) and arena.check()
    for n, p in e.named_parameters():
        assert torch.equal(p, before[n]) and p.untyped_storage().data_ptr() == arena.data.untyped_storage().data_ptr()
    w, b = e.layer[0].attention.self.fused_qkv()
    assert w.data_ptr() == e.layer[0].attention.self.query.weight.data_ptr()      # still adjacent


def test_reducer_leaves_a_differential_encoder_to_finish():
    from uniter_amd.utils.distributed import GradientReducer
    e = UniterEncoder(config()).bfloat16()
    r = GradientReducer(flatten_model(e), e)
    assert r.encoder is None and e.grad_ready_hook is None and not r.buckets


def test_no_weight_decay_on_the_head_norm():
    from uniter_amd.optim.misc import build_optimizer

    class O:
        optim, learning_rate, betas, weight_decay = "adamw", 1e-3, (0.9, 0.98), 0.01
    m = UniterEncoder(config())
    opt = build_optimizer(m, O)
    plain = {id(p) for g in opt.param_groups if g["weight_decay"] == 0.0 for p in g["params"]}
    assert id(m.layer[0].attention.self.LayerNorm.weight) in plain


@pytest.mark.parametrize("cu,total", [([0, 5, 10], 10), ([0, 5, 10], 13), ([0, 5, 10], 8), ([0, 0, 3, 3, 3, 9, 9], 12), ([0], 4), ([0, 0], 3),
                                      ([2, 4], 6), ([-5, 3, 50], 7), ([0, 10_000_000], 4), ([0, 6], 0)])
def test_positions_of_packed_rows(cu, total):
    """Rows of a sequence count from its first row (bounds cut to the rows there are), those behind the last one from its end; others are 0."""
    want = [0] * total
    last = min(max(cu[-1], 0), total)
    want[last:] = range(total - last)
    for a, b in zip(cu[:-1], cu[1:]):
        a, b = (min(max(x, 0), total) for x in (a, b))
        want[a:b] = range(b - a)
    got = ops.packed_positions(torch.tensor(cu, dtype=torch.int32), total)
    assert got.dtype == torch.int64 and got.tolist() == want


def test_positions_of_bounds_that_do_not_ascend_stay_in_range():
    for cu in ([0, 30, 20, 50], [7, 2, 9], [40, 0, 0], [-3, -9, 4]):
        got = ops.packed_positions(torch.tensor(cu, dtype=torch.int32), 33)
        assert got.shape == (33,) and ((got >= 0) & (got < 33)).all()


# ---- against plain float32 layers ------------------------------------------------------------------------------------------
class _Round(torch.autograd.Function):
    """Round to bf16 and go on in float32, values and gradients."""

    @staticmethod
    def forward(ctx, t):
        return t.to(BF16).float()

    @staticmethod
    def backward(ctx, g):
        return g.to(BF16).float()


def plain_attention(att, x, bias, pos, rnd, seen):
    """BertDifferentialSelfAttention in float32; x [B, L, H], bias [B, L], pos [B, L]; rnd: applied where the kernels store bf16; seen:
    takes (o, P_2 V), [B, L, heads, 2 d]."""
    B, L, H = x.shape
    n, d = att.num_attention_heads, att.map_size
    q, k, v = (rnd(torch.nn.functional.linear(x, m.weight, m.bias)) for m in (att.query, att.key, att.value))
    q, k = (t.view(B, L, 2 * n, d) for t in (q, k))
    if att.rotary is not None:
        r = att.rotary.rotary_dim
        ang = pos.double()[..., None, None] * torch.tensor(att.rotary.inv_freq, dtype=torch.float64)
        c, s = ((f(ang) * att.rotary.multiplier).float() for f in (torch.cos, torch.sin))

        def turn(t):
            a, b = t[..., :r // 2], t[..., r // 2:r]
            return rnd(torch.cat((a * c - b * s, b * c + a * s, t[..., r:]), dim=-1))
        q, k = turn(q), turn(k)
    sc = torch.einsum("blhd,bmhd->bhlm", q, k) * d ** -0.5 + bias[:, None, None, :]
    e = (sc - sc.detach().amax(-1, keepdim=True)).exp()
    p = (rnd(e) / e.sum(-1, keepdim=True)).view(B, n, 2, L, L)
    lam = (att.lambda_q1 * att.lambda_k1).sum(-1).exp() - (att.lambda_q2 * att.lambda_k2).sum(-1).exp() + att.lambda_init
    a = p[:, :, 0] - lam[None, :, None, None] * p[:, :, 1]
    v = v.view(B, L, n, 2 * d)
    o = torch.einsum("bhlm,bmhe->blhe", a, v)
    o.retain_grad()
    seen.append((o, torch.einsum("bhlm,bmhe->blhe", p[:, :, 1], v).detach()))
    o = o * (o.square().mean(-1, keepdim=True) + att.LayerNorm.eps).rsqrt() * att.LayerNorm.weight * (1 - att.lambda_init)
    return rnd(o.reshape(B, L, H))


def plain_layers(layers, x, bias, pos, rnd=lambda t: t, seen=None):
    seen = [] if seen is None else seen
    for l in layers:
        a = l.attention.output
        h = rnd(a.LayerNorm(rnd(a.dense(plain_attention(l.attention.self, x, bias, pos, rnd, seen))) + x))
        x = rnd(l.output.LayerNorm(rnd(l.output.dense(rnd(l.intermediate.intermediate_act_fn(l.intermediate.dense(h))))) + h))
    return x


def encoder(cfg, seed=0):
    torch.manual_seed(seed)
    e = UniterEncoder(cfg)
    with torch.no_grad():
        for n, p in e.named_parameters():
            if "LayerNorm" in n and n.endswith("weight"):
                p.copy_(1 + 0.1 * torch.randn_like(p))
            elif "lambda" not in n:
                p.copy_(torch.randn_like(p) * (0.08 if p.dim() > 1 else 0.02))
    return e.bfloat16()


# Tolerances.  How far the bf16 roundings at the kernels' borders carry is computed for each case: the same layers run once more with
# these roundings written out (`_Round`).  Counting roundings alone is not enough: eight per layer of 0.42 half steps give 0.8 % over
# three layers, but the scores' errors are relative to the scores (standard deviation 0.8 - 1.9 in these cases), exp makes them relative
# errors of P, and o1 - lambda o2 raises them by |o1| / |o1 - lambda o2| (up to 1.9 in the last layer).  Written out, the four cases give
# 0.57, 0.53, 0.65 and 1.03 % for the output and 0.8, 0.7, 1.2 and 2.1 % for dx.  The kernels' roundings are other draws of the same
# sizes, with a few more inside (q times 1 / sqrt(d), P and dS as operands of the backward products): 1.5 times for the output, twice for
# dx.  Parameter gradients: the 5e-2 that the encoder's tests allow (written out: up to 2.7 %), but not for lambda's: they are multiples of
# ONE sum per head, dlambda = -sum dO . (P_2 V) over all rows and columns, which may come out at a small part of its terms (one of these
# layers: 3.9, where its neighbours have 50 and the terms' absolute values sum to 4700; moving x by 0.3 % moves it by up to 0.8).  With
# relative errors e of dO and of P_2 V, independent from row to row, its standard deviation is sqrt(2) e times the root of the terms'
# squares (terms of a row summed, or each for itself: whichever is more); e: twice the written-out error of dx, four deviations allowed.
# A single call's lambda gradients are held to strict bounds in the tests of the operator.
@pytest.mark.gpu
@pytest.mark.parametrize("heads,hidden,rotary,L", [(2, 128, ROTARY, 50), (1, 128, None, 33), (3, 192, {"interleaved": False}, 130), (2, 256, ROTARY, 64),
                                                   (6, 384, None, 64), (4, 256, None, 64)])
def test_encoder_against_plain_layers(heads, hidden, rotary, L):
    cfg = config(heads, hidden, 3, rotary)
    e = encoder(cfg)
    ref = copy.deepcopy(e).float()
    e = e.cuda().train()
    g = torch.Generator().manual_seed(L)
    x = torch.randn(3, L, hidden, generator=g).to(BF16)
    dy = torch.randn(3, L, hidden, generator=g).to(BF16)
    valid = torch.tensor([L, L - 7, L // 2])
    mask = (torch.arange(L)[None] >= valid[:, None]).float() * -10000.0
    dy = dy * (torch.arange(L)[None, :, None] < valid[:, None, None])
    xr = x.float().requires_grad_(True)
    seen = []
    want = plain_layers(ref.layer, xr, mask, torch.arange(L).expand(3, L), seen=seen)
    want.backward(dy.float())
    xs = x.float().requires_grad_(True)
    rounded = plain_layers(copy.deepcopy(ref).layer, xs, mask, torch.arange(L).expand(3, L), _Round.apply)
    rounded.backward(dy.float())
    xg = x.cuda().requires_grad_(True)
    outs = e(xg, mask.cuda()[:, None, None, :])
    assert len(outs) == 3
    outs[-1].backward(dy.cuda())
    live = torch.arange(L)[None] < valid[:, None]
    assert rel_l2(outs[-1].float().cpu()[live], want[live].detach()) < 1.5 * rel_l2(rounded[live].detach(), want[live].detach())
    assert rel_l2(xg.grad.float().cpu(), xr.grad) < 2 * rel_l2(xs.grad, xr.grad)
    for (n, p), (_, q) in zip(e.named_parameters(), ref.named_parameters()):
        if "lambda" in n:
            lay, at = ref.layer[int(n.split(".")[1])].attention.self, n.split("lambda_")[1]
            o, o2 = seen[int(n.split(".")[1])]
            # |g - g'| = |dlambda - dlambda'| exp(q . k) |other vector|
            term = o.grad * o2
            room = torch.maximum(term.square().sum((0, 1, 3)), term.sum(-1).square().sum((0, 1))).sqrt() * 4 * 2 ** 0.5 * 2 * rel_l2(xs.grad, xr.grad)
            a, b = getattr(lay, "lambda_q" + at[1]).detach(), getattr(lay, "lambda_k" + at[1]).detach()
            room = room * (a * b).sum(-1).exp() * (b if at[0] == "q" else a).norm(dim=-1) + U * q.grad.norm(dim=-1)
            off = (p.grad.float().cpu() - q.grad).norm(dim=-1)
            assert (off < room).all(), (n, off, room)
            continue
        if n.endswith("key.bias") and rotary is None:
            continue                             # a shift of all scores of a row: its gradient is zero but for rounding
        assert rel_l2(p.grad.float().cpu(), q.grad) < 5e-2 and cosine(p.grad.float().cpu(), q.grad) > 0.998, (n, rel_l2(p.grad.float().cpu(), q.grad))
    with torch.no_grad():                        # eval gives the same bits; without mask entries too
        assert torch.equal(e.eval()(x.cuda(), mask.cuda())[-1], outs[-1])
    # gradients accumulate over micro-steps: a second pass doubles them (a bf16 sum of equal values is exact)
    first = {n: p.grad.clone() for n, p in e.named_parameters()}
    e.train()
    e(x.cuda(), mask.cuda(), output_all_encoded_layers=False)[0].backward(dy.cuda())
    for n, p in e.named_parameters():
        assert rel_l2(p.grad, 2 * first[n]) < 8e-3, n


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.2])
def test_one_node_per_layer_does_what_the_blocks_do(p):
    """The blocks on their own round two residual sums more, and gelu's derivative once more: three roundings among the 20 of a layer's
    backward pass, well under its tolerance of 5e-2 to the formula.  Dropout draws are the same."""
    cfg = config(2, 128, 2, ROTARY, p=p)
    one = encoder(cfg).cuda().train()
    two = copy.deepcopy(one)
    for l in two.layer:                          # a frozen bias: block by block
        l.output.dense.bias.requires_grad_(False)
    g = torch.Generator().manual_seed(2)
    x, dy = (torch.randn(2, 40, 128, generator=g).to(BF16).cuda() for _ in range(2))
    got = []
    for e in (one, two):
        ops.manual_seed(5)
        xg = x.clone().requires_grad_(True)
        y = e(xg, torch.zeros(2, 40).cuda())[-1]
        y.backward(dy)
        got.append((y.detach(), xg.grad))
    assert torch.equal(got[0][0], got[1][0])
    assert rel_l2(got[1][1], got[0][1]) < 2e-2
    for (n, q), (_, r) in zip(one.named_parameters(), two.named_parameters()):
        if r.requires_grad and not n.endswith("key.bias"):
            assert cosine(q.grad, r.grad) > 0.995, n
        elif not r.requires_grad:
            assert r.grad is None and q.grad.any(), n


@pytest.mark.gpu
def test_frozen_encoders_and_what_the_blocks_refuse():
    x = torch.randn(2, 9, 64).to(BF16).cuda()
    for kw in (dict(intermediate_size=96), dict(hidden_act="relu")):
        with pytest.raises(_lib.UniterHipError):
            encoder(config(1, 64, 1, **kw)).cuda().train()(x, torch.zeros(2, 9).cuda())
    e = encoder(config(1, 64, 2)).cuda().train()
    for q in e.parameters():
        q.requires_grad_(False)
    xg = x.clone().requires_grad_(True)
    e(xg, torch.zeros(2, 9).cuda())[-1].backward(x)
    assert xg.grad.any() and all(q.grad is None for q in e.parameters())
    y = e(x, torch.zeros(2, 9).cuda())[-1]
    assert not y.requires_grad


def test_projections_fused_in_inference_mode_stay_trainable():
    att = BertDifferentialSelfAttention(config())
    before = [q.detach().clone() for q in att.parameters()]
    with torch.inference_mode():
        w, b = att.fused_qkv()
    assert not w.is_inference() and not any(q.is_inference() or q.data.is_inference() for q in att.parameters())
    assert all(torch.equal(q, o) for q, o in zip(att.parameters(), before)) and w.data_ptr() == att.query.weight.data_ptr()
    att.query(torch.ones(1, 128)).sum().backward()
    assert att.query.weight.grad.any()


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [ROTARY, None])
def test_evaluation_in_inference_mode_before_training(rotary):
    e = encoder(config(rotary=rotary)).cuda()
    other = copy.deepcopy(e)
    x, dy = (torch.randn(2, 40, 128).to(BF16).cuda() for _ in range(2))
    mask = torch.zeros(2, 40).cuda()
    with torch.inference_mode():
        seen = e.eval()(x, mask)[-1]
    got = []
    for m in (e, other):
        y = m.train()(x, mask)[-1]
        y.backward(dy)
        got.append([y.detach()] + [q.grad for q in m.parameters()])
    assert torch.equal(seen, got[0][0]) and all(torch.equal(a, b) for a, b in zip(*got))


def test_tile_indices_are_those_of_the_gemm_kernels():
    """ops asks for the deep-pipelined tiles by index; gemm.hip asserts that these entries of its table are the tiles that they are named for."""
    import os
    import re
    with open(os.path.join(os.path.dirname(ops.__file__), "csrc", "gemm.hip")) as f:
        found = re.search(r"constexpr int kTileG8 = (\d+), kTileG6 = (\d+);", f.read())
    assert (ops._TILE_256, ops._TILE_192) == tuple(int(x) for x in found.groups())


def test_a_mask_that_wants_a_gradient_is_refused():
    x, learned = torch.zeros(2, 3, 128), torch.zeros(2, 3, requires_grad=True)
    for m in (learned, 2 * learned[:, None, None, :]):
        with pytest.raises(_lib.UniterHipError, match="detached"):
            ops.key_mask(m, x)
        with torch.no_grad():
            assert ops.key_mask(m, x).shape == (2, 3)
    assert ops.key_mask(learned.detach(), x).shape == (2, 3) and ops.key_mask(None, x) is None


PROJECTIONS = ["query.weight", "key.weight", "value.weight", "query.bias", "key.bias", "value.bias"]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["differential", "softmax"])
@pytest.mark.parametrize("arena", [False, True])
@pytest.mark.parametrize("trained", [PROJECTIONS[3:], PROJECTIONS[:1], ["key.weight", "value.bias"], PROJECTIONS[:3], []])
def test_partly_frozen_projections(trained, arena, kind):
    """Trained ones get the gradient that they have when all are trained, bit for bit and over two passes; frozen ones get none."""
    torch.manual_seed(5)
    make = BertDifferentialSelfAttention if kind == "differential" else BertSelfAttention
    x, dy = (torch.randn(2, 40, 128).to(BF16).cuda() for _ in range(2))
    mask = torch.zeros(2, 40).cuda()
    full = make(config()).cuda().bfloat16().train()
    part = copy.deepcopy(full)
    arenas = [flatten_model(m) for m in (full, part)] if arena else []
    for n, q in part.named_parameters():
        q.requires_grad_(n in trained)
    for _ in range(2):
        got = []
        for m in (full, part):
            xg = x.clone().requires_grad_(True)
            y = m(xg, mask)
            y.backward(dy)
            got.append((y.detach(), xg.grad))
        assert all(torch.equal(a, b) for a, b in zip(*got))
        for (n, q), (_, r) in zip(full.named_parameters(), part.named_parameters()):
            assert torch.equal(q.grad, r.grad) if n in trained else r.grad is None, n
    assert full.query.weight.grad.any() and all(a.check() for a in arenas)


@pytest.mark.gpu
@pytest.mark.parametrize("blocks", [False, True])
def test_two_layers_at_work_on_two_streams(blocks):
    """No scratch is shared: every pass gives the bits of a pass alone, as one node per layer and block by block (a frozen bias)."""
    cfg = config(2, 128, 2, ROTARY)
    nets = [encoder(cfg, seed).cuda().train() for seed in (0, 1)]
    for e in nets:
        if blocks:
            for l in e.layer:
                l.output.dense.bias.requires_grad_(False)
    g = torch.Generator().manual_seed(9)
    data = [tuple(torch.randn(3, 40 + 24 * i, 128, generator=g).to(BF16).cuda() for _ in range(2)) for i in range(2)]

    def step(i):
        x, dy = data[i]
        for q in nets[i].parameters():
            q.grad = None
        xg = x.clone().requires_grad_(True)
        y = nets[i](xg, torch.zeros(x.shape[:2], device="cuda"))[-1]
        y.backward(dy)
        return [y.detach(), xg.grad] + [q.grad for q in nets[i].parameters() if q.requires_grad]

    want = [step(i) for i in range(2)]
    ops._scratch_cache.clear()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for r in range(8):
        with torch.cuda.stream(streams[r % 2]):
            got.append(step(r % 2))
    torch.cuda.synchronize()
    assert not ops._scratch_cache                # (buffers of the process, whatever the stream)
    for r, ts in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(ts, want[r % 2]))


@pytest.mark.gpu
def test_packed_rows_give_what_padded_rows_give():
    cfg = config(2, 128, 2, ROTARY)
    e = encoder(cfg).cuda().eval()
    lens = [50, 7, 31]
    x = torch.randn(3, 50, 128).to(BF16).cuda()
    mask = torch.arange(50).cuda()[None] < torch.tensor(lens).cuda()[:, None]
    with torch.no_grad():
        a = e(x, torch.where(mask, 0.0, -math.inf))[-1]
        b = e.forward_packed(x, mask.long(), seq_lens=lens)[-1]
    assert rel_l2(b.float()[mask], a.float()[mask]) < 4e-3 and not b[~mask].any()


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [ROTARY, None])
def test_packed_layer_with_rows_behind_the_last_sequence(rotary):
    """Rows that belong to no sequence: zeros, and the others come out as where those rows are a sequence of their own, bit for bit (rows
    are independent of each other in every product, and the sizes are the same)."""
    torch.manual_seed(3)
    att = BertDifferentialSelfAttention(config(rotary=rotary)).cuda().bfloat16().train()
    x, dy = (torch.randn(15, 128).to(BF16).cuda() for _ in range(2))
    got = []
    for cu in ([0, 5, 5, 12], [0, 5, 5, 12, 15]):
        xg = x.clone().requires_grad_(True)
        y = att(xg, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_len=7)
        got.append((y, torch.autograd.grad(y, xg, dy)[0]))
    for a, b in zip(*got):
        assert torch.equal(a[:12], b[:12]) and not a[12:].any() and b[12:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("loss", ["square", "linear"])
def test_model_trains_with_the_optimizer_and_dropout(loss):
    from uniter_amd.optim.adamw import AdamW
    cfg = config(2, 128, 2, {"rotary_dim": 32}, p=0.1)
    torch.manual_seed(3)
    m = UniterModel(cfg, 16).cuda().bfloat16().train()
    flatten_model(m)
    opt = AdamW(m.parameters(), lr=1e-3)
    opt.fuse_zero_grad = True
    m.encoder.grad_ready_hook = ops.DeferWgradJoin()
    ops.manual_seed(11)
    ids, pos = torch.randint(1, 100, (4, 20)).cuda(), torch.arange(20)[None].cuda()
    am = torch.ones(4, 20, dtype=torch.long).cuda()
    before = {n: p.detach().clone() for n, p in m.named_parameters()}
    to = torch.randn(4, 20, 128).to(BF16).cuda()
    seen = []
    for _ in range(2):
        y = m(ids, pos, None, None, am, output_all_encoded_layers=False)
        (y.float().square().mean() if loss == "square" else (y * to).sum()).backward()
        seen.append(y.detach())
        grads = {n: p.grad for n, p in m.encoder.named_parameters()}
        assert all(g is not None and torch.isfinite(g).all() for g in grads.values())
        opt.step()
        opt.zero_grad()
    # A norm's weight of 1 stays where it is: a step of at most lr = 1e-3 is less than half a bf16 step below 1, 2^-9 = 1.95e-3.  The
    # mean square of LayerNorm's rows (weight 1, bias 0) is 1 whatever goes in, so that loss has no gradient but rounding's (1e-6 and
    # less, at or under the optimizer's eps): its lambda vectors need not move by half a bf16 step of theirs.
    fixed = ("key.bias", "LayerNorm.weight") + (("lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2") if loss == "square" else ())
    still = [n for n, p in m.encoder.named_parameters() if torch.equal(p, before["encoder." + n]) and not n.endswith(fixed)]
    assert not still
    assert not torch.equal(seen[0], seen[1])


@pytest.mark.gpu
def test_positions_in_every_form_that_rotary_takes():
    torch.manual_seed(1)
    att = BertDifferentialSelfAttention(config(rotary=ROTARY)).cuda().bfloat16()
    x = torch.randn(3, 9, 128).to(BF16).cuda()
    pos = torch.randint(0, 500, (9,)).cuda()
    want = att(x, positions=pos.expand(3, 9).contiguous())
    for p in (pos, pos[None], pos.int()[None], pos.expand(3, 9)):
        assert torch.equal(att(x, positions=p), want)
    assert torch.equal(att(x[:1], positions=pos[None]), want[:1])
    for bad in (pos[None, None], pos[None, :8], pos.expand(2, 9)):
        with pytest.raises(_lib.UniterHipError, match="positions"):
            att(x, positions=bad)


@pytest.mark.gpu
def test_module_refusals():
    att = BertDifferentialSelfAttention(config(rotary=ROTARY)).cuda().bfloat16()
    x = torch.zeros(2, 5, 128, dtype=BF16, device="cuda")
    plain = BertDifferentialSelfAttention(config()).cuda().bfloat16()
    cu = torch.tensor([0, 5, 10], dtype=torch.int32, device="cuda")
    assert att(x).shape == x.shape and att(x.flatten(0, 1), cu_seqlens=cu, max_len=5).shape == (10, 128)
    for bad in (lambda: att(x[..., :64]), lambda: att(x.float()), lambda: att(x, torch.zeros(2, 4).cuda()), lambda: att(x, positions=torch.zeros(4).long().cuda()), lambda: plain(x, positions=torch.arange(5).cuda()),
                lambda: att(x.flatten(0, 1)), lambda: att(x.flatten(0, 1), cu_seqlens=cu), lambda: att(x.cpu())):
        with pytest.raises(_lib.UniterHipError):
            bad()
    e = UniterEncoder(config()).cuda().bfloat16()
    e.grad_ready_hook = lambda l: None
    with pytest.raises(_lib.UniterHipError, match="hook"):
        e(x, torch.zeros(2, 5).cuda())
