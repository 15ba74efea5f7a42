"""Rotary positions (ops.rotary, model/rotary.py) against the formula in 64 bits."""
import math

import pytest
import torch

from uniter_amd import _lib, ops
from uniter_amd.model.rotary import RotaryPositions

BF16 = torch.bfloat16
U = torch.finfo(BF16).eps / 2

SCALINGS = [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
            {"type": "yarn", "factor": 16.0, "original_max_position": 2048}]


# ---- frequencies (CPU) -----------------------------------------------------------------------------------------------------
def test_frequencies_of_each_scaling():
    plain = RotaryPositions(64).inv_freq
    assert len(plain) == 32 and plain[0] == 1.0 and abs(plain[31] - 10000.0 ** (-62 / 64)) < 1e-18
    lin = RotaryPositions(64, scaling={"type": "linear", "factor": 4.0})
    assert all(abs(a * 4 - b) < 1e-15 for a, b in zip(lin.inv_freq, plain)) and lin.multiplier == 1.0
    ntk = RotaryPositions(64, scaling={"type": "ntk", "factor": 8.0})
    assert ntk.inv_freq[0] == 1.0 and abs(ntk.inv_freq[31] * 8 / plain[31] - 1) < 1e-12        # fastest kept, slowest divided by f
    yarn = RotaryPositions(64, scaling={"type": "yarn", "factor": 16.0, "original_max_position": 2048})
    ratio = [a / b for a, b in zip(yarn.inv_freq, plain)]
    assert ratio[0] == 1.0 and abs(ratio[31] - 1 / 16) < 1e-15 and all(x >= y for x, y in zip(ratio, ratio[1:]))
    assert abs(yarn.multiplier - (0.1 * math.log(16.0) + 1.0)) < 1e-15
    for i, f in enumerate(plain):                                      # turns over the trained length against the two borders
        turns = 2048 * f / (2 * math.pi)
        if turns > 64:
            assert ratio[i] == 1.0
        if turns < 0.5:
            assert abs(ratio[i] - 1 / 16) < 1e-15
    assert RotaryPositions(64, rotary_dim=16).inv_freq == [10000.0 ** (-2.0 * i / 16) for i in range(8)]


@pytest.mark.parametrize("kw", [
    dict(head_dim=64, rotary_dim=3), dict(head_dim=64, rotary_dim=66), dict(head_dim=1), dict(head_dim=2048), dict(head_dim=64, base=0.0),
    dict(head_dim=64, scaling={"type": "cubic", "factor": 2.0}), dict(head_dim=64, scaling={"type": "linear"}),
    dict(head_dim=64, scaling={"type": "linear", "factor": 0.5}), dict(head_dim=64, scaling={"type": "yarn", "factor": 2.0}),
    dict(head_dim=64, scaling={"type": "linear", "factor": 2.0, "beta_fast": 3.0}), dict(head_dim=2, scaling={"type": "ntk", "factor": 2.0}),
    dict(head_dim=64, scaling={"type": "yarn", "factor": 2.0, "original_max_position": 64, "beta_fast": 1.0, "beta_slow": 2.0})])
def test_bad_configurations_are_refused(kw):
    with pytest.raises(_lib.UniterHipError):
        RotaryPositions(**kw)


def test_the_table_is_an_ordinary_tensor_whatever_makes_it():
    for mode in (torch.inference_mode, torch.no_grad, torch.enable_grad):
        rot = RotaryPositions(8)
        with mode():
            made = rot.turns(torch.device("cpu"))
        assert not made.is_inference() and rot.turns(torch.device("cpu")) is made
        assert made.tolist() == [f / (2 * math.pi) for f in rot.inv_freq]


def test_cpu_tensors_and_bad_c_arguments_are_refused():
    with pytest.raises(_lib.UniterHipError, match="CUDA"):
        ops.rotary(torch.zeros(1, 2, 1, 64, dtype=BF16), None, RotaryPositions(64))
    lib = _lib.load()
    import ctypes
    s = (ctypes.c_int64 * 3)(64, 64, 64)
    r = _lib.UniterRotary()
    r.B, r.L, r.heads, r.head_dim, r.rot_dim = 1, 1, 1, 64, 64
    assert lib.uniter_rotary(ctypes.byref(r), None, s, None, s, None) < 0 and b"null" in lib.uniter_hip_last_error()
    r.rot_dim = 7
    assert lib.uniter_rotary(ctypes.byref(r), 64, s, 64, s, None) < 0 and b"rot_dim" in lib.uniter_hip_last_error()
    r.rot_dim, r.head_dim = 64, 4096
    assert lib.uniter_rotary(ctypes.byref(r), 64, s, 64, s, None) < 0
    r.head_dim, r.B = 64, 0
    assert lib.uniter_rotary(ctypes.byref(r), None, s, None, s, None) == 0           # nothing to do
    r.B, r.freq = 1, 8
    r.L = 1 << 27
    assert lib.uniter_rotary(ctypes.byref(r), 64, s, 64, s, None) < 0 and b"too many" in lib.uniter_hip_last_error()
    r.L = 1
    t = (ctypes.c_int64 * 3)(64, 64, 128)
    assert lib.uniter_rotary(ctypes.byref(r), 64, s, 64, t, None) < 0 and b"in place" in lib.uniter_hip_last_error()


def _verdict(lib, sizes, dim, x, sx, y, sy):
    """What uniter_rotary says of x and y (element addresses) before anything is launched: without frequencies it ends at the null pointer."""
    import ctypes
    r = _lib.UniterRotary()
    r.B, r.L, r.heads = sizes
    r.head_dim = r.rot_dim = dim
    A = ctypes.c_int64 * 3
    assert lib.uniter_rotary(ctypes.byref(r), 2 * x, A(*sx), 2 * y, A(*sy), None) < 0
    text = lib.uniter_hip_last_error()
    assert b"overlap" in text or b"null" in text, text
    return b"overlap" in text


def _elements(sizes, dim, at, st):
    return [at + b * st[0] + l * st[1] + h * st[2] + e for b in range(sizes[0]) for l in range(sizes[1]) for h in range(sizes[2]) for e in range(dim)]


def test_overlapping_outputs_are_refused_and_others_are_not():
    """Against the elements themselves.  Whatever meets is refused; of equal strides, whatever does not meet is taken."""
    lib = _lib.load()
    # [L, B, heads, dim] underneath, one row of the batch on: x's second row is y's first
    assert _verdict(lib, (2, 8, 2), 32, 4096, (64, 256, 32), 4096 + 64, (64, 256, 32))
    assert not _verdict(lib, (2, 8, 2), 32, 4096, (64, 256, 32), 4096 + 128, (64, 256, 32))
    import random
    rng = random.Random(5)
    seen = [0, 0, 0]
    for _ in range(6000):
        sizes, dim = tuple(rng.choice((1, 2, 3)) for _ in range(3)), 2 * rng.choice((1, 1, 2))
        if rng.random() < 0.7:                       # nested in some order, with gaps or without
            st, span = [0, 0, 0], dim
            for i in rng.sample(range(3), 3):
                st[i] = span + rng.choice((0, 0, 1, dim, 3 * dim))
                span += (sizes[i] - 1) * st[i]
        else:
            st = [rng.randrange(0, 20) for _ in range(3)]
        if rng.random() < 0.1:
            st = [-s for s in st]
        sy = list(st) if rng.random() < 0.8 else [rng.randrange(1, 20) for _ in range(3)]
        x, y = 4096, 4096 + rng.randrange(-40, 41)
        if x == y and sy != st:
            continue                                 # (refused for its strides)
        ex, ey = _elements(sizes, dim, x, st), _elements(sizes, dim, y, sy)
        refused = _verdict(lib, sizes, dim, x, st, y, sy)
        itself = len(set(ey)) < len(ey)
        if itself or (x != y and set(ex) & set(ey)):
            assert refused, (sizes, dim, st, sy, y - x)
            seen[0] += 1
        elif sy == st:
            order = sorted((abs(s), n) for s, n in zip(st, sizes) if n > 1)
            span, nested = dim, True
            for s, n in order:
                nested, span = nested and s >= span, span + (n - 1) * s
            if nested:
                assert not refused, (sizes, dim, st, sy, y - x)
                seen[1] += 1
        elif not refused:
            seen[2] += 1
    assert min(seen) > 50, seen


# ---- kernels ---------------------------------------------------------------------------------------------------------------
def turned(x, positions, rot, sign=1.0):
    """float64 result on the CPU: a turned pair is a complex product.  x [.., heads, dim], positions [..]."""
    n = rot.rotary_dim
    x = x.detach().cpu().double()
    ang = positions.cpu().double()[..., None, None] * torch.tensor(rot.inv_freq, dtype=torch.float64) * sign
    by = torch.polar(torch.full_like(ang, rot.multiplier), ang)
    a, b = (slice(0, n, 2), slice(1, n, 2)) if rot.interleaved else (slice(0, n // 2), slice(n // 2, n))
    w = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * by
    y = x.clone()
    y[..., a], y[..., b] = w.real, w.imag
    return y


def close(got, want, x, rot):
    """One rounding of the result to bf16, and the sine and cosine to 2^-18 of a turn's scale: the hardware functions are good to about
    2^-20 absolutely, the angle's fraction reaches them rounded to 2^-25 of a turn (2 pi 2^-25 < 2^-22), each multiplied by an element
    of the pair; products and their sum add 3 roundings of 2^-24."""
    n = rot.rotary_dim
    size = x.detach().cpu().double().abs()
    a, b = (slice(0, n, 2), slice(1, n, 2)) if rot.interleaved else (slice(0, n // 2), slice(n // 2, n))
    pair = size[..., a] + size[..., b]
    bound = torch.zeros_like(size)
    bound[..., a] = bound[..., b] = pair * rot.multiplier * 2.0 ** -18
    bound += U * want.abs() * 1.001
    bad = (got.detach().cpu().double() - want).abs() > bound
    assert not bad.any(), "%d of %d off, worst %.3g over its bound" % (
        int(bad.sum()), bad.numel(), float(((got.detach().cpu().double() - want).abs() - bound).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,L,heads,dim,n", [(1, 1, 1, 64, 64), (2, 5, 3, 32, 32), (3, 97, 24, 64, 32), (1, 33, 5, 80, 48), (2, 7, 2, 128, 128),
                                             (1, 3, 2, 96, 6), (1, 4, 1, 2, 2), (1, 6, 70, 16, 16), (1, 2, 2, 1024, 1024), (1, 9, 3, 30, 20)])
def test_forward_and_gradient(B, L, heads, dim, n, interleaved):
    g = torch.Generator().manual_seed(L * 31 + dim)
    for scaling in SCALINGS if n > 2 else SCALINGS[:2]:
        rot = RotaryPositions(dim, rotary_dim=n, interleaved=interleaved, scaling=scaling)
        x = torch.randn(B, L, heads, dim, generator=g).to(BF16).cuda().requires_grad_(True)
        pos = torch.randint(0, 200_000, (B, L), generator=g).cuda()
        dy = torch.randn(B, L, heads, dim, generator=g).to(BF16).cuda()
        y = ops.rotary(x, pos, rot)
        dx, = torch.autograd.grad(y, x, dy)
        close(y, turned(x, pos, rot), x, rot)
        close(dx, turned(dy, pos, rot, -1.0), dy, rot)


@pytest.mark.gpu
def test_positions_forms_offsets_and_far_positions():
    rot = RotaryPositions(64, rotary_dim=32)
    x = torch.randn(3, 11, 4, 64).to(BF16).cuda()
    ar = torch.arange(11).expand(3, 11)
    close(ops.rotary(x, None, rot), turned(x, ar, rot), x, rot)
    close(ops.rotary(x, None, rot, offset=77), turned(x, ar + 77, rot), x, rot)
    p1 = torch.randint(0, 9999, (11,)).cuda()
    for p in (p1, p1[None], p1.int(), p1.expand(3, 11)):
        assert torch.equal(ops.rotary(x, p, rot), ops.rotary(x, p1.expand(3, 11).contiguous(), rot))
    wide = torch.randint(0, 9999, (3, 22)).cuda()
    assert torch.equal(ops.rotary(x, wide[:, ::2], rot), ops.rotary(x, wide[:, ::2].contiguous(), rot))
    for far in (2 ** 20 + 1, 2 ** 31 + 5, 2 ** 40 + 3):
        p = torch.arange(11).cuda() + far
        close(ops.rotary(x, p, rot), turned_exact(x, p.cpu(), rot), x, rot)
    close(ops.rotary(x, p1 - 12000, rot), turned(x, (p1 - 12000).expand(3, 11), rot), x, rot)       # before the origin


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,L,heads,dim,n", [(1, 3, 37, 64, 32), (2, 2, 9, 512, 512), (1, 2, 7, 384, 256), (1, 5, 11, 200, 16), (1, 2, 3, 520, 64)])
def test_more_heads_than_a_wave_holds(B, L, heads, dim, n, interleaved):
    rot = RotaryPositions(dim, rotary_dim=n, interleaved=interleaved)
    g = torch.Generator().manual_seed(dim)
    x = torch.randn(B, L, heads, dim, generator=g).to(BF16).cuda()
    pos = torch.randint(0, 5000, (B, L), generator=g).cuda()
    y = ops.rotary(x, pos, rot)
    close(y, turned(x, pos, rot), x, rot)
    guard = torch.full((B, L + 1, heads, dim + 8), 7.0, dtype=BF16, device="cuda")
    view = guard[:, :L, :, :dim].copy_(x)
    assert torch.equal(ops.rotary(view, pos, rot, out=view), y)                      # in place, between rows that stay as they were
    assert (guard[:, L] == 7).all() and (guard[..., dim:] == 7).all()


def turned_exact(x, pos, rot):
    """As turned(), with the angle reduced in whole-number arithmetic: far positions lose nothing."""
    from fractions import Fraction
    frac = [[float((Fraction(f / (2 * math.pi)) * int(p)) % 1) * 2 * math.pi for f in rot.inv_freq] for p in pos.tolist()]
    n = rot.rotary_dim
    x = x.cpu().double()
    ang = torch.tensor(frac, dtype=torch.float64)[:, None, :]
    w = torch.complex(x[..., :n // 2].contiguous(), x[..., n // 2:n].contiguous()) * torch.polar(torch.full_like(ang, rot.multiplier), ang)
    y = x.clone()
    y[..., :n // 2], y[..., n // 2:n] = w.real, w.imag
    return y


@pytest.mark.gpu
def test_strides_packed_rows_in_place_and_out():
    rot = RotaryPositions(32, interleaved=True)
    proj = torch.randn(2, 9, 3 * 128).to(BF16).cuda()
    qk = proj[..., :256].unflatten(-1, (8, 32))
    pos = torch.randint(0, 5000, (2, 9)).cuda()
    want = ops.rotary(qk.contiguous(), pos, rot)
    assert torch.equal(ops.rotary(qk, pos, rot), want)
    assert torch.equal(ops.rotary(qk.transpose(0, 1), pos.t(), rot), want.transpose(0, 1))
    assert torch.equal(ops.rotary(qk.flatten(0, 1), pos.flatten(), rot), want.flatten(0, 1))        # back to back
    odd = torch.empty(2, 9, 8 * 32 + 1, dtype=BF16, device="cuda")[..., 1:].unflatten(-1, (8, 32)).copy_(qk)   # 2-byte aligned
    assert torch.equal(ops.rotary(odd, pos, rot), want)
    tr = qk.transpose(-1, -2).contiguous().transpose(-1, -2)                                        # heads not contiguous
    assert torch.equal(ops.rotary(tr, pos, rot), want)
    rest = proj[..., 256:].clone()
    with torch.no_grad():
        assert ops.rotary(qk, pos, rot, out=qk).data_ptr() == qk.data_ptr()
    assert torch.equal(qk, want) and torch.equal(proj[..., 256:], rest)
    k_of_q = proj[..., 128:256].unflatten(-1, (4, 32))
    with torch.no_grad():
        src = proj[..., :128].unflatten(-1, (4, 32))
        w2 = ops.rotary(src, pos, rot)
        assert torch.equal(ops.rotary(src, pos, rot, out=k_of_q), w2) and torch.equal(proj[..., 256:], rest)
    empty = torch.empty(2, 0, 8, 32, dtype=BF16, device="cuda")
    assert ops.rotary(empty, None, rot).shape == empty.shape


@pytest.mark.gpu
def test_refusals():
    rot = RotaryPositions(64)
    x = torch.zeros(2, 3, 4, 64, dtype=BF16, device="cuda")
    for bad in (lambda: ops.rotary(x.float(), None, rot), lambda: ops.rotary(x[0, 0], None, rot), lambda: ops.rotary(x, None, RotaryPositions(32)),
                lambda: ops.rotary(x[0], None, rot), lambda: ops.rotary(x, torch.zeros(4, dtype=torch.int64, device="cuda"), rot),
                lambda: ops.rotary(x, torch.zeros(3, device="cuda"), rot), lambda: ops.rotary(x, torch.zeros(3, dtype=torch.int64), rot),
                lambda: ops.rotary(x.clone().requires_grad_(True), None, rot, out=x), lambda: ops.rotary(x, None, rot, out=x[:1]),
                lambda: ops.rotary(x[:, :2], None, rot, out=x[:, 1:]), lambda: ops.rotary(x, None, rot, out=x[:1].expand(2, 3, 4, 64)),
                lambda: ops.rotary(x[:, :1].expand(2, 3, 4, 64), None, rot, out=x[:, :1].expand(2, 3, 4, 64))):
        with pytest.raises(_lib.UniterHipError):
            bad()


@pytest.mark.gpu
def test_outputs_beside_their_input_in_one_storage():
    rot = RotaryPositions(32)
    t = torch.randn(8, 4, 2, 32).to(BF16).cuda()             # [L, B, heads, dim] underneath
    v = t.transpose(0, 1)
    want = ops.rotary(v[:2], None, rot)
    with pytest.raises(_lib.UniterHipError, match="overlap"):
        ops.rotary(v[:2], None, rot, out=v[1:3])
    with torch.no_grad():
        assert torch.equal(ops.rotary(v[:2], None, rot, out=v[2:]), want) and torch.equal(v[2:], want)
        flat = torch.zeros(400, dtype=BF16, device="cuda")
        with pytest.raises(_lib.UniterHipError, match="overlap"):      # windows of one another
            ops.rotary(want[0, :8], torch.arange(8).cuda(), rot, out=flat.as_strided((8, 2, 32), (40, 32, 1)))


@pytest.mark.gpu
def test_strides_that_nothing_steps_over():
    """A dimension of one has a stride that no address uses: any value of it is taken, also where out is x under another name."""
    rot = RotaryPositions(32)
    for shape in ((1, 5, 3, 32), (2, 1, 3, 32), (3, 4, 1, 32), (1, 1, 1, 32)):
        x = torch.randn(shape).to(BF16).cuda()
        strange = [s if n > 1 else 7 + i for i, (n, s) in enumerate(zip(shape, x.stride()))]
        strange[3] = 1
        want = ops.rotary(x, None, rot, offset=3)
        assert torch.equal(ops.rotary(x.as_strided(shape, strange), None, rot, offset=3), want)
        with torch.no_grad():
            assert torch.equal(ops.rotary(x.as_strided(shape, strange), None, rot, offset=3, out=x), want) and torch.equal(x, want)


@pytest.mark.gpu
def test_an_entry_that_refuses_raises_the_packages_error():
    """Past the checks of the call: the status of the C entry, with its message."""
    rot = RotaryPositions(64)
    rot.rotary_dim = 7
    x = torch.zeros(1, 2, 3, 64, dtype=BF16, device="cuda")
    for leaf in (x, x.clone().requires_grad_(True)):
        with pytest.raises(_lib.UniterHipError, match="rot_dim"):
            ops.rotary(leaf, None, rot)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    rot = RotaryPositions(64)
    x = torch.randn(1, 2, 3, 64).to(BF16).cuda().requires_grad_(True)
    dy = torch.randn(1, 2, 3, 64).to(BF16).cuda().requires_grad_(True)
    dx, = torch.autograd.grad(ops.rotary(x, None, rot), x, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.float().square().sum(), dy)


@pytest.mark.gpu
def test_gradient_against_differences():
    """The map is linear: y(x + h) - y(x) = y(h).  With x = 0 the difference is the derivative itself, so <y(h), dy> = <h, dx(dy)> up to
    the roundings of y and dx: half a step each, on every product."""
    rot = RotaryPositions(64, rotary_dim=32, scaling=SCALINGS[3])
    h = torch.randn(2, 17, 3, 64).to(BF16).cuda()
    dy = torch.randn(2, 17, 3, 64).to(BF16).cuda()
    pos = torch.randint(0, 100_000, (2, 17)).cuda()
    x = torch.zeros_like(h).requires_grad_(True)
    dx, = torch.autograd.grad(ops.rotary(x, pos, rot), x, dy)
    yh = ops.rotary(h, pos, rot)
    a, b = (yh.double() * dy.double()), (h.double() * dx.double())
    assert abs(float(a.sum() - b.sum())) <= 1.01 * U * float(a.abs().sum() + b.abs().sum())


@pytest.mark.gpu
def test_other_streams_and_captured_graphs():
    rot = RotaryPositions(64)
    x = torch.randn(2, 50, 6, 64).to(BF16).cuda()
    pos = torch.arange(50).cuda()
    want = ops.rotary(x, pos, rot)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.rotary(x, pos, rot)
    s.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.rotary(x, pos, rot)
    for i in range(3):
        x.mul_(-1)
        pos.add_(3)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.rotary(x, pos, rot))


@pytest.mark.gpu
def test_written_outputs_are_seen_by_autograd():
    """A tensor that a node has saved and that is then turned in place (or written to) makes that node's backward pass an error, as any
    in-place operation does; what is only read does not."""
    rot = RotaryPositions(64)
    scale = torch.ones(64, dtype=BF16, device="cuda", requires_grad=True)
    for write in ("x", "out", "view", "read"):
        cache = torch.randn(2, 9, 3, 64).to(BF16).cuda()
        y = (cache * scale).sum()                # saves `cache`
        with torch.no_grad():
            before = cache._version
            if write == "x":
                ops.rotary(cache, None, rot, out=cache)
            elif write == "out":
                ops.rotary(torch.zeros_like(cache), None, rot, out=cache)
            elif write == "view":
                ops.rotary(torch.zeros_like(cache[:, 2:5]), None, rot, out=cache[:, 2:5])
            else:
                ops.rotary(cache, None, rot)
            assert cache._version == before + (write != "read")
        if write == "read":
            y.backward()
        else:
            with pytest.raises(RuntimeError, match="inplace"):
                y.backward()
    with torch.inference_mode():                 # tensors without a version counter
        z = torch.zeros(1, 2, 3, 64, dtype=BF16, device="cuda")
        assert ops.rotary(z, None, rot, out=z) is z


@pytest.mark.gpu
def test_forward_mode_and_tracing_are_refused():
    import torch.autograd.forward_ad as fwAD
    rot = RotaryPositions(64)
    x, t = (torch.randn(1, 2, 3, 64).to(BF16).cuda() for _ in range(2))
    with fwAD.dual_level():
        d = fwAD.make_dual(x, t)
        for bad in (lambda: ops.rotary(d, None, rot), lambda: ops.rotary(d[:, 1:], None, rot), lambda: ops.rotary(x.clone(), None, rot, out=d),
                    lambda: ops.rotary(fwAD.make_dual(x.clone().requires_grad_(True), t), None, rot)):
            with pytest.raises(_lib.UniterHipError, match="forward-mode"):
                bad()
        assert torch.equal(ops.rotary(x, None, rot), ops.rotary(x.clone(), None, rot))        # others go on
    with pytest.raises(_lib.UniterHipError, match="trace"):
        torch.jit.trace(lambda a: ops.rotary(a, None, rot), (x,), check_trace=False)
    ops.rotary(x, None, rot)


@pytest.mark.gpu
def test_first_call_in_inference_mode_then_gradients():
    rot = RotaryPositions(64)
    x = torch.randn(1, 7, 3, 64).to(BF16).cuda()
    with torch.inference_mode():
        ops.rotary(x, None, rot)
    y = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(ops.rotary(y, None, rot), y, x)
    close(dx, turned(x, torch.arange(7)[None], rot, -1.0), x, rot)


@pytest.mark.gpu
def test_a_first_call_under_capture_is_refused_and_the_capture_goes_on():
    rot = RotaryPositions(64)
    x = torch.randn(1, 7, 3, 64).to(BF16).cuda()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(_lib.UniterHipError, match="capture"):
            ops.rotary(x, None, rot)
        y = x * 2
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, x * 2)
    want = ops.rotary(x, None, rot)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.rotary(x, None, rot)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
