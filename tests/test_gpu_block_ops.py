"""The block operators (group norm with an activation, gated recurrence, dropout) on the GPU against their 64-bit forms, whose
bounds follow the arithmetic (tests/block_oracle.py)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from speech_separation_amd import _lib, autograd, ops  # noqa: E402
from tests import block_oracle as oracle  # noqa: E402
from tests.block_oracle import close  # noqa: E402

DEV = "cuda:0"
F32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16
NAN = float("nan")


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g).to(dtype)


def place(t, how):
    """t on the GPU under other strides: "plain", "wide" (a slice of wider rows at an odd offset, so no row is aligned),
    "frames" (frame-major, [S, B, C] in memory)."""
    B, S, C = t.shape
    if how == "wide":
        w = torch.full((B, S, 2 * C + 3), NAN, dtype=t.dtype, device=DEV)
        w[..., 3:3 + C] = t.to(DEV)
        return w[..., 3:3 + C]
    if how == "frames":
        return t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    return t.to(DEV)


def lengths_of(kind, B, S):
    if kind is None:
        return None
    n = torch.tensor([(S, 1, 0, S // 2, S + 9, -3)[i % 6] for i in range(B)], dtype=torch.int32)
    return n.roll(1) if kind == "rolled" else n


def poison(t, lengths):
    """What stands behind an utterance's end is never read into a result."""
    if lengths is not None:
        for b, n in enumerate(lengths.clamp(0, t.shape[1]).tolist()):
            t[b, n:] = torch.tensor([NAN, float("inf"), -float("inf"), torch.finfo(t.dtype).min])[torch.arange(t.shape[2]) % 4].to(t.dtype)
    return t


# ------------------------------------------------------------------ group norm with an activation
NORM = [  # B, S, C, groups, type, act, act_first, lengths, strides
    (1, 1, 8, 1, F32, 1, False, None, "plain"),
    (2, 1, 4, 4, F32, 0, False, None, "plain"),             # one value a group
    (1, 7, 3, 3, BF16, 2, False, None, "plain"),
    (3, 65, 96, 8, F32, 1, True, "ends", "plain"),
    (6, 66, 96, 32, BF16, 1, False, "ends", "wide"),        # 3 channels a group
    (2, 300, 131, 1, F32, 3, False, None, "wide"),
    (2, 300, 131, 131, FP16, 1, False, "rolled", "plain"),  # one channel a group
    (2, 513, 64, 32, FP16, 2, True, None, "frames"),
    (1, 2000, 512, 1, F32, 1, True, None, "plain"),
    (7, 40, 1030, 10, BF16, 0, False, "rolled", "frames"),
    (1, 31, 2048, 4, F32, 1, False, None, "plain"),
    (2, 4099, 16, 2, BF16, 3, True, None, "wide"),
    (65, 9, 40, 5, F32, 2, False, "ends", "plain"),
    (3, 1000, 512, 16, BF16, 1, False, "ends", "plain"),
    (2, 700, 520, 2, FP16, 1, True, "rolled", "wide"),
    (1, 9000, 8, 1, F32, 1, False, None, "plain"),
    (300, 3, 64, 4, F32, 1, False, None, "plain"),
    (2, 3000, 1024, 8, BF16, 1, False, None, "plain"),
    (2, 20, 4100, 1, F32, 1, False, "ends", "plain"),
    (2, 20, 4100, 4100, BF16, 2, False, None, "plain"),     # every channel a group, more of them than a workgroup takes
    (1, 70, 9001, 1, FP16, 0, False, None, "wide"),
    (1, 20, 65537, 65537, F32, 1, False, None, "plain"),    # the last slice holds one channel, and its lane is moved into the one before
    (2, 20, 131075, 1, BF16, 0, False, "ends", "plain"),
    (1, 20, 131078, 65539, FP16, 2, True, None, "plain"),
    (3, 200, 2, 1, BF16, 1, True, "ends", "plain"),         # frames narrower than a vector
    (3, 200, 1, 1, F32, 2, False, None, "wide"),
]


@pytest.mark.parametrize("B,S,C,G,dtype,act,first,ends,strides", NORM)
def test_group_norm_act(B, S, C, G, dtype, act, first, ends, strides):
    g = torch.Generator().manual_seed(B + S + C)
    lengths = lengths_of(ends, B, S)
    x = poison((randn(g, B, S, C) * torch.exp(0.3 * randn(g, C)) + 0.5 * randn(g, C)).to(dtype), lengths)
    dy = poison(randn(g, B, S, C, dtype=dtype), lengths)
    gamma, beta = 1 + 0.2 * randn(g, C), 0.2 * randn(g, C)
    # A group without spread has 1/sqrt(eps) as its factor, which makes every rounding of x one of y: a large eps keeps the
    # bounds of the groups of one value meaningful.
    eps = 0.1 if S * C // G < 16 else 1e-5
    want = oracle.group_norm(x, gamma, beta, G, eps, act, first, lengths, dy)
    xd, dyd, gd, bd = place(x, strides), place(dy, strides), gamma.to(DEV), beta.to(DEV)
    ld = None if lengths is None else lengths.to(DEV)
    y, stats = ops.group_norm_act(xd, gd, bd, G, eps=eps, act=act, act_first=first, lengths=ld)
    close(y, *want["y"], "y")
    close(stats, *want["stats"], "stats")
    dx, dgamma, dbeta = ops.group_norm_act_backward(dyd, xd, gd, bd, stats, G, act=act, act_first=first, lengths=ld)
    close(dx, *want["dx"], "dx")
    close(dgamma, *want["dgamma"], "dgamma")
    close(dbeta, *want["dbeta"], "dbeta")
    # the same call gives the same bits
    again = ops.group_norm_act_backward(dyd, xd, gd, bd, stats, G, act=act, act_first=first, lengths=ld)
    assert all(torch.equal(a, b) for a, b in zip((dx, dgamma, dbeta), again))
    assert torch.equal(y, ops.group_norm_act(xd, gd, bd, G, eps=eps, act=act, act_first=first, lengths=ld)[0])


@pytest.mark.parametrize("gamma,beta", [(False, False), (True, False), (False, True)])
def test_group_norm_act_without_gains(gamma, beta):
    g = torch.Generator().manual_seed(5)
    x, dy, ga, be = randn(g, 2, 50, 24), randn(g, 2, 50, 24), randn(g, 24), randn(g, 24)
    ga, be = ga if gamma else None, be if beta else None
    want = oracle.group_norm(x, ga, be, 3, 1e-5, 1, False, None, dy)
    gd, bd = (None if t is None else t.to(DEV) for t in (ga, be))
    y, stats = ops.group_norm_act(x.to(DEV), gd, bd, 3, act=1)
    close(y, *want["y"])
    dx, dgamma, dbeta = ops.group_norm_act_backward(dy.to(DEV), x.to(DEV), gd, bd, stats, 3, act=1)
    close(dx, *want["dx"])
    assert (dgamma is None) == (ga is None) and (dbeta is None) == (be is None)
    if gamma:
        close(dgamma, *want["dgamma"])
    if beta:
        close(dbeta, *want["dbeta"])


@pytest.mark.parametrize("level", [300.0, 1e4])
def test_group_norm_act_far_from_zero(level):
    """Values whose mean is many times their spread: the variance must not come out of a difference of squares."""
    g = torch.Generator().manual_seed(6)
    x = randn(g, 2, 3000, 64) + level
    y, stats = ops.group_norm_act(x.to(DEV), None, None, 2)
    want = oracle.group_norm(x, None, None, 2, 1e-5, 0, False)
    close(y, *want["y"])
    var = x.double().view(2, 3000, 2, 32).var((1, 3), unbiased=False)
    assert float(((stats[..., 1].cpu().double() ** -2 - 1e-5) / var - 1).abs().max()) < 1e-4 * max(1, level / 1e3)


def test_group_norm_act_empty():
    for shape in ((0, 5, 8), (2, 0, 8)):
        x = torch.zeros(shape, device=DEV)
        w = torch.ones(8, device=DEV)
        y, stats = ops.group_norm_act(x, w, w, 2)
        dx, dgamma, dbeta = ops.group_norm_act_backward(x, x, w, w, stats, 2)
        assert y.shape == dx.shape == x.shape and not bool(stats.any()) and not bool(dgamma.any()) and not bool(dbeta.any())
    x = torch.full((2, 4, 8), NAN, device=DEV)
    y, stats = ops.group_norm_act(x, w, w, 2, lengths=torch.zeros(2, dtype=torch.int32, device=DEV))
    dx, dgamma, _ = ops.group_norm_act_backward(x, x, w, w, stats, 2, lengths=torch.zeros(2, dtype=torch.int32, device=DEV))
    assert not bool(y.any()) and not bool(stats.any()) and not bool(dx.any()) and not bool(dgamma.any())


def test_group_norm_act_keeps_a_bad_value_in_its_group():
    x = torch.randn(2, 40, 32, device=DEV)
    x[0, 3, 9] = NAN
    x[1, 5, 20] = float("inf")
    y, _ = ops.group_norm_act(x, None, None, 4, act=1)
    bad = ~torch.isfinite(y.view(2, 40, 4, 8))
    assert bool(bad[0, :, 1].all()) and bool(bad[1, :, 2].any())
    bad[0, :, 1] = bad[1, :, 2] = False
    assert not bool(bad.any())


# ------------------------------------------------------------------ gated recurrence
REC = [  # B, S, C, type, lengths, reverse, strides, h0, dlast
    (1, 1, 1, F32, None, False, "plain", True, True),
    (64, 1, 512, F32, None, False, "plain", True, True),
    (3, 2, 33, BF16, None, True, "plain", False, False),
    (3, 31, 33, F32, "ends", False, "wide", True, True),
    (2, 32, 64, FP16, None, False, "plain", True, False),
    (2, 33, 64, F32, None, True, "plain", False, True),
    (6, 63, 40, BF16, "ends", True, "frames", True, True),
    (6, 129, 7, F32, "rolled", False, "plain", True, True),
    (1, 1000, 130, F32, None, False, "plain", True, True),
    (2, 1025, 300, BF16, "rolled", True, "wide", True, True),
    (2, 4097, 40, F32, None, False, "frames", True, True),
    (1, 9001, 24, FP16, None, True, "plain", True, True),
    (33, 257, 96, BF16, "ends", False, "plain", False, True),
    (1, 3000, 513, BF16, None, False, "plain", True, True),
    (8, 513, 512, FP16, "rolled", True, "wide", True, True),
    (2, 70, 4100, BF16, "ends", False, "plain", True, True),
    (2, 300, 3, BF16, None, True, "wide", True, True),
    (300, 40, 129, F32, "ends", False, "frames", True, True),
    (70000, 2, 5, FP16, "ends", True, "plain", True, True),
    (40, 300, 501, BF16, "ends", False, "plain", False, True),
]


def rec_inputs(g, B, S, C, dtype, lengths):
    level = 6 * torch.rand(C, generator=g) - 1
    x, dh = randn(g, B, S, C, dtype=dtype), randn(g, B, S, C, dtype=dtype)
    gate = (1.5 * randn(g, B, S, C) + level).to(dtype)
    return poison(x, lengths), poison(gate, lengths), poison(dh, lengths), randn(g, B, C), randn(g, B, C)


def to_dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


@pytest.mark.parametrize("B,S,C,dtype,ends,reverse,strides,with_h0,with_dlast", REC)
def test_gated_recurrence(B, S, C, dtype, ends, reverse, strides, with_h0, with_dlast):
    g = torch.Generator().manual_seed(B + S + C)
    lengths = lengths_of(ends, B, S)
    x, gate, dh, h0, dlast = rec_inputs(g, B, S, C, dtype, lengths)
    h0, dlast = h0 if with_h0 else None, dlast if with_dlast else None
    want = oracle.recurrence(x, gate, h0, lengths, reverse, dh, dlast)
    xd, gd, dhd = (place(t, strides) for t in (x, gate, dh))
    h0d, dld, ld = to_dev(h0, dlast, lengths)
    h, last, none = ops.gated_recurrence(xd, gd, h0d, ld, reverse)
    assert none is None
    close(h, *want["h"], "h")
    close(last, *want["last"], "last")
    h2, last2, saved = ops.gated_recurrence(xd, gd, h0d, ld, reverse, save=True)
    assert torch.equal(h, h2) and torch.equal(last, last2)
    got = ops.gated_recurrence_backward(dhd, xd, gd, saved, dld, ld, reverse)
    for name, v in zip(("dx", "dgate", "dh0"), got):
        close(v, *want[name], name)
    assert all(torch.equal(a, b) for a, b in zip(got, ops.gated_recurrence_backward(dhd, xd, gd, saved, dld, ld, reverse)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gated_recurrence_saturated_gates(dtype):
    """Gates that open or shut for good: infinite, beyond what an exponential holds, and close to 1 for a whole sequence."""
    g = torch.Generator().manual_seed(11)
    B, S, C = 2, 700, 16
    x, dh, h0, dlast = randn(g, B, S, C, dtype=dtype), randn(g, B, S, C, dtype=dtype), randn(g, B, C), randn(g, B, C)
    kinds = torch.tensor([float("inf"), -float("inf"), 200.0, -200.0, 88.0, -88.0, 104.0, -104.0, 17.0, -17.0, 12.0, 9.0, 0.0, 1e-30, 3e38, -3e38])
    gate = kinds.expand(B, S, C).clone()
    gate[:, ::97] = randn(g, B, gate[:, ::97].shape[1], C)
    gate = gate.to(dtype)
    want = oracle.recurrence(x, gate, h0, None, False, dh, dlast)
    xd, gd, dhd, h0d, dld = to_dev(x, gate, dh, h0, dlast)
    h, last, saved = ops.gated_recurrence(xd, gd, h0d, save=True)
    close(h, *want["h"], "h")
    close(last, *want["last"], "last")
    for name, v in zip(("dx", "dgate", "dh0"), ops.gated_recurrence_backward(dhd, xd, gd, saved, dld)):
        value, err = want[name]
        if name == "dgate":                    # a (1 - a) of a gate beyond 87 is a subnormal number: the kernel may call it 0
            err = err + 1e-36
        close(v, value, err + 1e-36, name)


def test_gated_recurrence_frame_by_frame_and_in_pieces():
    """A stream: one state, updated in place, one frame or some frames a call."""
    g = torch.Generator().manual_seed(12)
    B, S, C = 3, 70, 48
    x, gate, _, h0, _ = rec_inputs(g, B, S, C, F32, None)
    want = oracle.recurrence(x, gate, h0)
    xd, gd, state = to_dev(x, gate, h0)
    parts, s = [], 0
    for k in (1, 1, 1, 5, 32, 1, 29):
        h, last, _ = ops.gated_recurrence(xd[:, s:s + k], gd[:, s:s + k], state, last=state)
        assert last is state
        parts.append(h)
        s += k
    assert s == S
    close(torch.cat(parts, 1), *want["h"])
    close(state, *want["last"])


def test_gated_recurrence_state_in_place_over_a_long_sequence():
    g = torch.Generator().manual_seed(13)
    for reverse in (False, True):
        x, gate, dh, h0, dlast = to_dev(*rec_inputs(g, 1, 20000, 24, BF16, None))
        h, last, saved = ops.gated_recurrence(x, gate, h0, reverse=reverse, save=True)
        state = h0.clone()
        h2, _, saved2 = ops.gated_recurrence(x, gate, state, reverse=reverse, last=state, save=True)
        assert torch.equal(h, h2) and torch.equal(last, state) and torch.equal(saved, saved2)


@pytest.mark.parametrize("C,dtype", [(33, F32), (65, BF16), (129, F32), (131, FP16)])
def test_gated_recurrence_state_in_place_where_slices_share_channels(C, dtype):
    """Widths whose last lanes are moved left over channels of the slice before, which another workgroup may have finished."""
    g = torch.Generator().manual_seed(15)
    x, gate, dh, h0, dlast = to_dev(*rec_inputs(g, 70, 90, C, dtype, None))
    h, last, saved = ops.gated_recurrence(x, gate, h0, save=True)
    for _ in range(5):
        state = h0.clone()
        h2, _, saved2 = ops.gated_recurrence(x, gate, state, last=state, save=True)
        assert torch.equal(h, h2) and torch.equal(last, state) and torch.equal(saved, saved2)


def test_gated_recurrence_gradients_into_one_tensor():
    g = torch.Generator().manual_seed(14)
    both = randn(g, 3, 200, 2 * 40, dtype=BF16).to(DEV)
    x, gate, dh = both[..., :40], both[..., 40:], randn(g, 3, 200, 40, dtype=BF16).to(DEV)
    _, _, saved = ops.gated_recurrence(x, gate, save=True)
    dx, dgate, dh0 = ops.gated_recurrence_backward(dh, x, gate, saved)
    d = torch.full((3, 200, 83), 7.0, dtype=BF16, device=DEV)
    got = ops.gated_recurrence_backward(dh, x, gate, saved, out=(d[..., 1:41], d[..., 41:81]))
    assert torch.equal(d[..., 1:41], dx) and torch.equal(d[..., 41:81], dgate) and torch.equal(got[2], dh0)
    assert bool((d[..., 0] == 7).all()) and bool((d[..., 81:] == 7).all())


@pytest.mark.parametrize("S,C,dtype", [(50, 33, F32), (3000, 131, F32), (3000, 66, BF16)])
def test_gated_recurrence_keeps_a_bad_value_in_its_channel(S, C, dtype):
    """Not a number from one frame on in the channels it came in by, forward and backward, and nowhere else."""
    g = torch.Generator().manual_seed(16)
    x, gate, dh, _, _ = rec_inputs(g, 2, S, C, dtype, None)
    x[0, 7, C - 1], gate[1, 20, 3], dh[0, S - 9, 0] = NAN, NAN, NAN
    xd, gd, dhd = to_dev(x, gate, dh)
    h, last, saved = ops.gated_recurrence(xd, gd, save=True)
    want = torch.zeros(2, S, C, dtype=torch.bool)
    want[0, 7:, C - 1] = want[1, 20:, 3] = True
    assert torch.equal(torch.isnan(h).cpu(), want) and torch.equal(torch.isnan(last).cpu(), want[:, -1])
    dx, dgate, dh0 = ops.gated_recurrence_backward(dhd, xd, gd, saved)
    back = torch.zeros(2, S, C, dtype=torch.bool)
    back[0, :S - 8, 0] = back[1, :21, 3] = True
    assert torch.equal(torch.isnan(dx).cpu(), back)
    back[0, 7:, C - 1] = back[1, 20:, 3] = True              # h_{t-1} - x_t
    assert torch.equal(torch.isnan(dgate).cpu(), back) and bool(torch.isnan(dh0[0, 0])) and int(torch.isnan(dh0).sum()) == 2


def test_gated_recurrence_empty():
    for B, S in ((0, 4), (3, 0)):
        x = torch.zeros(B, S, 8, device=DEV)
        h0 = torch.randn(B, 8, device=DEV)
        h, last, saved = ops.gated_recurrence(x, x, h0, save=True)
        assert h.shape == x.shape and torch.equal(last, h0)
        dx, dgate, dh0 = ops.gated_recurrence_backward(x, x, x, saved, dlast=h0)
        assert dx.shape == x.shape and torch.equal(dh0, h0)
        assert not bool(ops.gated_recurrence(x, x)[1].any())


# ------------------------------------------------------------------ dropout
@pytest.mark.parametrize("B,S,C,tx,tr,p,strides", [
    (1, 1, 1, F32, None, 0.5, "plain"), (2, 33, 40, F32, F32, 0.1, "plain"), (3, 17, 37, BF16, F32, 0.25, "wide"), (2, 50, 257, FP16, None, 0.1, "plain"),
    (5, 31, 16, BF16, BF16, 0.9, "frames"), (2, 100, 512, FP16, F32, 0.1, "plain"), (2, 9, 7, FP16, FP16, 0.3, "wide"), (1, 4000, 24, F32, None, 0.01, "wide"),
    (300, 1, 64, BF16, F32, 0.1, "plain"), (2, 3, 8, F32, F32, 0.0, "plain"), (2, 3, 8, F32, F32, 1.0, "plain"), (2, 3, 8, BF16, None, 2.0 ** -17, "plain"),
    (2, 3, 8, BF16, None, 1.0 - 2.0 ** -16, "plain")])
def test_dropout(B, S, C, tx, tr, p, strides):
    g = torch.Generator().manual_seed(B + S + C)
    x, r = randn(g, B, S, C, dtype=tx), None if tr is None else randn(g, B, S, C, dtype=tr)
    for seed, step, site in ((0, 0, 0), (-7, 3, 1), (2 ** 63 - 1, 2 ** 40 + 17, 2 ** 32 - 1)):
        rng = torch.tensor([seed, step], device=DEV)
        y = ops.dropout(place(x, strides), p, rng, site, None if r is None else place(r, strides))
        assert y.dtype == (tr or tx)
        close(y, *oracle.dropout(x, p, seed, step, site, r))
        dy = randn(g, B, S, C, dtype=tr or tx)
        dx = ops.dropout_backward(place(dy, strides), p, rng, site, dtype=tx)
        assert dx.dtype == tx
        close(dx, *oracle.dropout(dy, p, seed, step, site))


def test_dropout_drops_what_is_not_finite():
    x = torch.full((2, 20, 64), NAN, device=DEV)
    rng = torch.tensor([1, 2], device=DEV)
    y = ops.dropout(x, 0.5, rng, residual=torch.ones_like(x))
    kept = oracle.keep((2, 20, 64), 0.5, 1, 2, 0).to(DEV)
    assert torch.equal(torch.isnan(y), kept) and bool((y[~kept] == 1).all())
    assert not bool(ops.dropout(x, 1.0, rng).any())


def test_dropout_in_place():
    g = torch.Generator().manual_seed(3)
    x, r, rng = randn(g, 2, 30, 44).to(DEV), randn(g, 2, 30, 44).to(DEV), torch.tensor([5, 6], device=DEV)
    want = ops.dropout(x, 0.2, rng, 4, r)
    r2, x2 = r.clone(), x.clone()
    assert ops.dropout(x, 0.2, rng, 4, r2, out=r2) is r2 and torch.equal(r2, want)
    assert torch.equal(ops.dropout(x2, 0.2, rng, 4, r, out=x2), want)
    wide = torch.zeros(2, 30, 100, device=DEV)
    wide[..., :44], wide[..., 50:94] = x, r
    assert torch.equal(ops.dropout(wide[..., :44], 0.2, rng, 4, wide[..., 50:94], out=wide[..., 50:94]), want)
    assert torch.equal(wide[..., :44], x) and not bool(wide[..., 44:50].any()) and not bool(wide[..., 94:].any())


def test_dropout_many_utterances_that_do_not_follow_one_another():
    """More utterances than a grid's second dimension counts."""
    B, S, C = 70000, 2, 9
    x = place(torch.arange(B * S * C, dtype=F32).view(B, S, C) % 97 - 48, "frames")
    rng = torch.tensor([8, 9], device=DEV)
    y = ops.dropout(x, 0.4, rng, 1)
    close(y, *oracle.dropout(x.cpu(), 0.4, 8, 9, 1))


# ------------------------------------------------------------------ all of them
def test_refusals():
    x, f64, i32 = torch.zeros(2, 3, 8, device=DEV), torch.zeros(2, 3, 8, dtype=torch.float64, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    w, rng, st = torch.zeros(8, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(2, 2, 2, device=DEV)
    hs, sv = torch.zeros(2, 8, device=DEV), torch.zeros(2, 1, 8, device=DEV)
    half = x.to(BF16)
    turned = torch.zeros(2, 8, 3, device=DEV).transpose(1, 2)
    bad = [
        lambda: ops.group_norm_act(f64, None, None, 2), lambda: ops.group_norm_act(turned, None, None, 2), lambda: ops.group_norm_act(x, None, None, 3),
        lambda: ops.group_norm_act(x, None, None, 0), lambda: ops.group_norm_act(x, w[:4], None, 2), lambda: ops.group_norm_act(x, w.to(BF16), None, 2),
        lambda: ops.group_norm_act(x, w.cpu(), None, 2), lambda: ops.group_norm_act(x, w, w, 2, lengths=i32.long()),
        lambda: ops.group_norm_act(x, w, w, 2, lengths=i32[:1]), lambda: ops.group_norm_act(x, w, w, 2, act=4), lambda: ops.group_norm_act(x, w, w, 2, eps=-1.0),
        lambda: ops.group_norm_act(x, w, w, 2, eps=NAN), lambda: ops.group_norm_act(x[0], w, w, 2),
        lambda: ops.group_norm_act_backward(half, x, w, w, st, 2), lambda: ops.group_norm_act_backward(x[:1], x, w, w, st, 2),
        lambda: ops.group_norm_act_backward(x, x, w, w, st[:1], 2), lambda: ops.group_norm_act_backward(x, x, w, w, None, 2),
        lambda: ops.gated_recurrence(x, half), lambda: ops.gated_recurrence(x, x[:, :2]), lambda: ops.gated_recurrence(x, x, hs[:1]),
        lambda: ops.gated_recurrence(x, x, hs.to(BF16)), lambda: ops.gated_recurrence(x, x, last=hs.t().contiguous().t()), lambda: ops.gated_recurrence(turned, turned),
        lambda: ops.gated_recurrence_backward(x, x, x, None), lambda: ops.gated_recurrence_backward(x, x, x, sv[:, :, :4]),
        lambda: ops.gated_recurrence_backward(x, x, x, sv, out=(x, torch.empty_like(x))), lambda: ops.gated_recurrence_backward(x, x, x, sv, dlast=hs[:1]),
        lambda: ops.gated_recurrence_backward(x, x, x, sv, out=(hs[:1, None].expand(2, 3, 8), torch.empty_like(x))),
        lambda: ops.dropout(x, 1.1, rng), lambda: ops.dropout(x, -0.1, rng), lambda: ops.dropout(x, NAN, rng), lambda: ops.dropout(x, 0.1, rng.int()),
        lambda: ops.dropout(x, 0.1, None), lambda: ops.dropout(x, 0.1, rng[:1]), lambda: ops.dropout(x, 0.1, rng, site=-1), lambda: ops.dropout(x, 0.1, rng, site=2 ** 32),
        lambda: ops.dropout(half, 0.1, rng, residual=x.to(FP16)), lambda: ops.dropout(x, 0.1, rng, residual=x[:, :2]), lambda: ops.dropout(x, 0.1, rng, residual=3.0),
        lambda: ops.dropout(x[:, :2], 0.1, rng, out=x[:, 1:]), lambda: ops.dropout_backward(half, 0.1, rng, dtype=FP16), lambda: ops.dropout_backward(None, 0.1, rng),
    ]
    leaf = torch.zeros(2, 8, device=DEV, requires_grad=True)
    dx = torch.empty_like(x)
    bad += [lambda: ops.gated_recurrence(x, x, last=leaf), lambda: ops.gated_recurrence(x, x, hs, last=x.view(-1)[8:24].view(2, 8)),
            lambda: ops.gated_recurrence_backward(x, x, x, sv, out=(dx, dx)), lambda: ops.dropout(x, 0.1, rng, out=x.clone().requires_grad_()),
            lambda: ops.dropout(x, 0.1, rng, out=torch.empty(2, 3, 4, device=DEV)), lambda: ops.gated_recurrence_backward(x, x, x, sv, out=(dx, half))]
    for f in bad:
        with pytest.raises(ValueError):
            f()


def test_writing_in_place_is_noticed_by_autograd():
    w = torch.randn(2, 3, 8, device=DEV, requires_grad=True)
    r = torch.randn(2, 3, 8, device=DEV)
    y = (w * r).sum()
    ops.dropout(torch.randn(2, 3, 8, device=DEV), 0.1, torch.tensor([1, 2], device=DEV), residual=r, out=r)
    with pytest.raises(RuntimeError):
        y.backward()


def test_autograd_refuses_its_backward_under_capture(monkeypatch):
    x = torch.randn(2, 3, 8, device=DEV, requires_grad=True)
    outs = [autograd.group_norm_act(x, None, None, 2), autograd.gated_recurrence(x, x)[0], autograd.dropout(x, 0.1, torch.tensor([1, 2], device=DEV))]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for y in outs:
        with pytest.raises(RuntimeError):
            y.sum().backward()


def test_inference_mode():
    with torch.inference_mode():
        x, state, rng = torch.randn(2, 3, 8, device=DEV), torch.zeros(2, 8, device=DEV), torch.tensor([1, 2], device=DEV)
        h, last, _ = ops.gated_recurrence(x, x, state.clone())
        assert torch.equal(ops.gated_recurrence(x, x, state, last=state)[0], h) and torch.equal(state, last)
        y = ops.dropout(h, 0.1, rng, residual=x)
        assert torch.equal(ops.dropout(h, 0.1, rng, residual=x, out=x), y)
        assert torch.equal(autograd.gated_recurrence(x, x)[0], ops.gated_recurrence(x, x)[0])


def test_autograd_without_gradients_saves_nothing():
    x = torch.randn(2, 40, 8, device=DEV)
    with torch.no_grad():
        h, last = autograd.gated_recurrence(x, x)
    assert torch.equal(h, ops.gated_recurrence(x, x)[0]) and not h.requires_grad


def block(x, w, lengths, state, rng):
    """The operators as a gated recurrent block uses them: norm, projection to value | gate, recurrence, projection back, dropout
    onto the residual stream."""
    y, stats = ops.group_norm_act(x, w["gamma"], w["beta"], 4, act=1, lengths=lengths)
    vg = ops.linear(y, w["vg"])
    C = w["vg"].shape[0] // 2
    h, last, saved = ops.gated_recurrence(vg[..., :C], vg[..., C:], state, lengths, save=True)
    z = ops.linear(h, w["out"])
    return ops.dropout(z, 0.1, rng, site=2, residual=x), (y, stats, vg, h, last, saved)


def block_inputs(B=3, S=150, C=64, seed=21):
    g = torch.Generator().manual_seed(seed)
    x, dout, state = randn(g, B, S, C), randn(g, B, S, C), randn(g, B, 2 * C)
    w = {"gamma": 1 + 0.2 * randn(g, C), "beta": 0.2 * randn(g, C), "vg": randn(g, 4 * C, C) / 8, "out": randn(g, C, 2 * C) / 8}
    lengths = torch.tensor([S, 0, S // 2][:B], dtype=torch.int32)
    return x, dout, state, w, lengths


def test_block_forward_and_gradients():
    """A run of the operators together, forward and backward by hand, against autograd in 64 bits.  One block's chain of
    fp32 results: each stage keeps 2e-6 of its scale (its own bound above), the products add theirs (K <= 128, 2e-6), five stages."""
    x, dout, state, w, lengths = block_inputs()
    B, S, C = x.shape
    wd = {k: v.to(DEV) for k, v in w.items()}
    xd, doutd, stated, ld = to_dev(x, dout, state, lengths)
    rng = torch.tensor([77, 3], device=DEV)
    out, (y, stats, vg, h, last, saved) = block(xd, wd, ld, stated, rng)
    dz = ops.dropout_backward(doutd, 0.1, rng, site=2)
    dh = dz @ wd["out"]
    dvg = torch.empty_like(vg)
    _, _, dstate = ops.gated_recurrence_backward(dh, vg[..., :2 * C], vg[..., 2 * C:], saved, None, ld, out=(dvg[..., :2 * C], dvg[..., 2 * C:]))
    dy = dvg @ wd["vg"]
    dx, dgamma, dbeta = ops.group_norm_act_backward(dy, xd, wd["gamma"], wd["beta"], stats, 4, act=1, lengths=ld)
    dx = dx + doutd
    got = {"out": out, "last": last, "dx": dx, "dgamma": dgamma, "dbeta": dbeta, "dstate": dstate,
           "dvg": (dvg.flatten(0, 1).t() @ y.flatten(0, 1)), "dout": (dz.flatten(0, 1).t() @ h.flatten(0, 1))}

    leaf = {k: v.double().requires_grad_() for k, v in dict(w, x=x, state=state).items()}
    o, la = reference_block(leaf, lengths, oracle.keep((B, S, C), 0.1, 77, 3, 2))
    o.backward(dout.double())
    want = {"out": o, "last": la, "dx": leaf["x"].grad, "dgamma": leaf["gamma"].grad, "dbeta": leaf["beta"].grad, "dstate": leaf["state"].grad,
            "dvg": leaf["vg"].grad, "dout": leaf["out"].grad}
    for k in want:
        v = want[k].detach()
        assert float((got[k].double().cpu() - v).abs().max()) <= 2e-5 * float(v.abs().max()), k


def reference_block(leaf, lengths, keep):
    x = leaf["x"]
    B, S, C = x.shape
    y = torch.zeros_like(x)
    h = torch.zeros(B, S, 2 * C, dtype=torch.float64)
    rows, lasts, ys = [], [], []
    for b in range(B):
        n = int(lengths[b])
        v = leaf["state"][b]
        hb, yb = [], torch.zeros(0, C, dtype=torch.float64)
        if n:
            u = x[b, :n].view(n, 4, -1)
            var, mean = torch.var_mean(u, dim=(0, 2), unbiased=False, keepdim=True)
            yb = torch.nn.functional.silu(((u - mean) / torch.sqrt(var + 1e-5)).reshape(n, C) * leaf["gamma"] + leaf["beta"])
        vg = yb @ leaf["vg"].t()
        for t in range(n):
            a = torch.sigmoid(vg[t, 2 * C:])
            v = a * v + (1 - a) * vg[t, :2 * C]
            hb.append(v)
        hb = torch.cat([torch.stack(hb) if n else torch.zeros(0, 2 * C, dtype=torch.float64), torch.zeros(S - n, 2 * C, dtype=torch.float64)])
        rows.append(hb @ leaf["out"].t())
        lasts.append(v)
    z = torch.stack(rows)
    return x + torch.where(keep, z * (65536 / (65536 - 6554)), 0.0), torch.stack(lasts)


def test_autograd_block():
    """The same block through speech_separation_amd.autograd."""
    x, dout, state, w, lengths = block_inputs(seed=22)
    B, S, C = x.shape
    leaf = {k: v.to(DEV).requires_grad_() for k, v in dict(w, x=x, state=state).items()}
    rng, ld = torch.tensor([78, 4], device=DEV), lengths.to(DEV)
    y = autograd.group_norm_act(leaf["x"], leaf["gamma"], leaf["beta"], 4, act=1, lengths=ld)
    vg = torch.nn.functional.linear(y, leaf["vg"])
    h, last = autograd.gated_recurrence(vg[..., :2 * C], vg[..., 2 * C:], leaf["state"], ld)
    o = autograd.dropout(torch.nn.functional.linear(h, leaf["out"]), 0.1, rng, 2, leaf["x"])
    (o * dout.to(DEV)).sum().backward()
    ref = {k: v.double().requires_grad_() for k, v in dict(w, x=x, state=state).items()}
    ro, rl = reference_block(ref, lengths, oracle.keep((B, S, C), 0.1, 78, 4, 2))
    ro.backward(dout.double())
    assert float((last.detach().double().cpu() - rl.detach()).abs().max()) <= 2e-5 * float(rl.detach().abs().max())
    for k in leaf:
        v = ref[k].grad
        assert float((leaf[k].grad.double().cpu() - v).abs().max()) <= 2e-5 * float(v.abs().max()), k


def test_autograd_notices_an_advanced_step():
    x, rng = torch.randn(2, 4, 8, device=DEV, requires_grad=True), torch.tensor([1, 0], device=DEV)
    y = autograd.dropout(x, 0.5, rng)
    rng[1] += 1
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_captured_graph_replays_with_new_inputs():
    """Forward and backward of all three operators in one graph: each replay agrees with the eager calls on what its buffers
    hold by then, with other work and synchronisation in between."""
    sets = [block_inputs(seed=30 + k) for k in range(3)]
    wd = {k: v.to(DEV) for k, v in sets[0][3].items()}
    C = sets[0][0].shape[2]
    x, dout, state, ld = to_dev(*sets[0][:3], sets[0][4])
    rng = torch.tensor([9, 0], device=DEV)

    def step(x, dout, state, lengths, rng):
        out, (y, stats, vg, h, last, saved) = block(x, wd, lengths, state, rng)
        dz = ops.dropout_backward(dout, 0.1, rng, site=2)
        dh = dz @ wd["out"]
        dv, dg, ds = ops.gated_recurrence_backward(dh, vg[..., :2 * C], vg[..., 2 * C:], saved, None, lengths)
        return out, last, dv, dg, ds, *ops.group_norm_act_backward(x, x, wd["gamma"], wd["beta"], stats, 4, act=1, lengths=lengths)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(x, dout, state, ld, rng)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, dout, state, ld, rng)
    for k, (nx, nd, ns, _, nl) in enumerate(sets):
        for t, v in ((x, nx), (dout, nd), (state, ns), (ld, nl.roll(k))):
            t.copy_(v.to(DEV))
        rng[1] = k
        graph.replay()
        torch.cuda.synchronize()
        want = step(x, dout, state, ld, rng)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_two_streams_at_once():
    g = torch.Generator().manual_seed(40)
    a, b = (rec_inputs(g, 2, 3000, 96, F32, None) for _ in range(2))
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    data = [to_dev(*v) for v in (a, b)]
    torch.cuda.synchronize()
    for s, (x, gate, dh, h0, dlast) in zip(streams, data):
        with torch.cuda.stream(s):
            h, last, saved = ops.gated_recurrence(x, gate, h0, save=True)
            y, stats = ops.group_norm_act(h, None, None, 4, act=1)
            outs.append((h, last, y, *ops.gated_recurrence_backward(dh, x, gate, saved, dlast), ops.group_norm_act_backward(dh, h, None, None, stats, 4, act=1)[0]))
    torch.cuda.synchronize()
    for (x, gate, dh, h0, dlast), got in zip(data, outs):
        h, last, saved = ops.gated_recurrence(x, gate, h0, save=True)
        y, stats = ops.group_norm_act(h, None, None, 4, act=1)
        want = (h, last, y, *ops.gated_recurrence_backward(dh, x, gate, saved, dlast), ops.group_norm_act_backward(dh, h, None, None, stats, 4, act=1)[0])
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_offsets_beyond_32_bits():
    """Utterances more than 2^31 elements apart in one buffer."""
    apart, B, S, C = (1 << 31) + 64, 2, 40, 64
    buf = torch.empty(apart + S * C, dtype=BF16, device=DEV)
    g = torch.Generator().manual_seed(50)
    x, gate, dh, h0, dlast = rec_inputs(g, B, S, C, BF16, None)
    xd = buf.as_strided((B, S, C), (apart, C, 1))
    xd.copy_(x.to(DEV))
    gd, dhd, h0d, dld = to_dev(gate, dh, h0, dlast)
    want = oracle.recurrence(x, gate, h0, None, False, dh, dlast)
    h, last, saved = ops.gated_recurrence(xd, gd, h0d, save=True)
    close(h, *want["h"])
    for name, v in zip(("dx", "dgate", "dh0"), ops.gated_recurrence_backward(dhd, xd, gd, saved, dld)):
        close(v, *want[name])
    want = oracle.group_norm(x, None, None, 2, 1e-5, 1, False, None, dh)
    y, stats = ops.group_norm_act(xd, None, None, 2, act=1)
    close(y, *want["y"])
    close(ops.group_norm_act_backward(dhd, xd, None, None, stats, 2, act=1)[0], *want["dx"])
    rng = torch.tensor([3, 4], device=DEV)
    close(ops.dropout(xd, 0.3, rng), *oracle.dropout(x, 0.3, 3, 4, 0))
    ops.dropout(gd, 0.3, rng, out=xd)
    close(xd, *oracle.dropout(gate, 0.3, 3, 4, 0))
    assert np.isfinite(float(last.sum()))


def test_rows_beyond_32_bits():
    """A tensor of more than 2^31 elements: its last rows agree with the same rows alone where rows are independent."""
    S, C = 33000000, 66
    rng = torch.tensor([3, 4], device=DEV)
    x = torch.empty(1, S, C, dtype=FP16, device=DEV)
    x.fill_(1.0)
    y = ops.dropout(x, 0.25, rng, site=5)
    tail = torch.from_numpy(_tail_keep(S, C, 20)).to(DEV)
    assert torch.equal(y[0, -20:], torch.where(tail, 65536 / 49152, 0.0).to(FP16))
    del y
    gate = torch.zeros_like(x)
    gate[0, -30:] = 2.0
    x[0, -30] = -3.0
    h, last, _ = ops.gated_recurrence(x, gate)
    want = oracle.recurrence(x[:, -90:].cpu(), gate[:, -90:].cpu(), torch.ones(1, C))        # 0.5^60 of what came before is left
    close(h[:, -30:], want["h"][0][:, -30:], want["h"][1][:, -30:] + 1e-12)
    close(last, want["last"][0], want["last"][1] + 1e-12)


def test_group_norm_act_beyond_32_bits():
    S, C = 33000000, 66
    x = torch.empty(1, S, C, dtype=BF16, device=DEV)
    x.fill_(1.0)
    x[..., 1::2] = -1.0
    y, stats = ops.group_norm_act(x, None, None, 1)
    r = 1 / (1 + 1e-5) ** 0.5
    assert abs(float(stats[0, 0, 0])) < 1e-6 and abs(float(stats[0, 0, 1]) - r) < 1e-6
    assert bool((y[0, -50:].float().abs() == torch.tensor(r).to(BF16).float().item()).all()) and bool((y[0, -50:, 0] > 0).all())
    dy = torch.zeros_like(x)
    dy[0, -1, 0] = 1.0
    dx, dgamma, dbeta = ops.group_norm_act_backward(dy, x, torch.ones(C, device=DEV), torch.zeros(C, device=DEV), stats, 1)
    assert abs(float(dx[0, -1, 0]) - 1) < 0.01 and abs(float(dx[0, -1, 1])) < 1e-6       # one of 2 10^9 values
    assert abs(float(dgamma[0]) - r) < 1e-5 and float(dbeta[0]) == 1.0 and not bool(dbeta[1:].any())


def _tail_keep(S, C, rows):
    per = -(-C // 8)
    block = np.arange((S - rows) * per, S * per, dtype=np.uint64)
    w = oracle.philox([block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), np.full_like(block, 4), np.full_like(block, 5)], [3, 0])
    return np.stack(w, -1).astype("<u4").view("<u2").reshape(rows, per * 8)[:, :C] >= 16384


# A thread sums n <= 64 values of one channel about the first of them, K: d = u - K, s = sum d, q = sum d^2, M2 = q - s^2 / n.  In 32
# bits q is off by (n + 2) U q and s by n U sum |d|, which changes s^2 / n by 2 n U q at most (|s| sum |d| <= n q); so M2 is off by
# (3 n + 4) U q.  K is one of the values, so (K - mean)^2 <= M2 (n - 1) / n and q = M2 + n (K - mean)^2 <= n M2.  The thread's mean is
# off by e = U sum |d| <= U sqrt(n q), and that of all values by the sum of 2 n e |its mean - theirs| more: by Cauchy, with M2 of all
# of them, 2 U n sqrt(n) M2 at most.
NORM_M2 = ((3 * 64 + 4) * 64 + 2 * 64 * 8) * oracle.U


@pytest.mark.parametrize("B,S,C,dtype,first", [(257, 16384, 4, F32, 1000.0), (257, 16384, 8, BF16, 1000.0), (300, 4096, 64, F32, -3000.0), (2, 4000, 512, F32, 1000.0)])
def test_group_norm_act_outlying_first_frame(B, S, C, dtype, first):
    """One frame unlike all others at the head of every utterance, in chunks of thousands of frames: it costs no digits of the variance."""
    g = torch.Generator(device=DEV).manual_seed(61)
    x = torch.randn(B, S, C, generator=g, device=DEV)
    x[:, 0] = first
    x = x.to(dtype)
    _, stats = ops.group_norm_act(x, None, None, 1)
    for b in range(0, B, 50):
        v = x[b].double()
        mean, var = v.mean(), v.var(unbiased=False)
        # a channel's, a thread's and the group's mean are rounded to 32 bits: 3 U of the largest each, twice as a factor of a deviation
        m = float(v.abs().mean())
        assert abs(float(stats[b, 0, 0]) - float(mean)) <= 70 * oracle.U * (m + abs(float(mean)) + float(var) ** 0.5)
        got = float(stats[b, 0, 1].double() ** -2 - 1e-5)
        assert abs(got / float(var) - 1) <= NORM_M2 + 16 * oracle.U, (b, got, float(var))


def test_group_norm_act_sums_of_many_threads():
    """Narrow frames, whose channels are summed by 256 threads: one large sum first, then 255 of less than half its last bit each.  No
    more than 64 terms are added one after the other in 32 bits, so no sum is off by more than 64 U of its terms."""
    S, C = 1024, 4
    many = torch.zeros(1, S, C, device=DEV)
    many[0, 1], many[0, 2:256] = 2.0 ** 24, 1.0
    total = 2.0 ** 24 + 254
    _, stats = ops.group_norm_act(many, None, None, 1)
    assert abs(float(stats[0, 0, 0]) - total / S) <= 65 * oracle.U * total / S
    x = torch.randn(1, S, C, device=DEV)
    w = torch.ones(C, device=DEV)
    _, stats = ops.group_norm_act(x, w, w, 1)
    _, _, dbeta = ops.group_norm_act_backward(many, x, w, w, stats, 1)
    assert bool(((dbeta.double() - total).abs() <= 65 * oracle.U * total).all()), dbeta


@pytest.mark.parametrize("C,G", [(512, 512), (131, 131), (256, 32)])
def test_group_norm_relu_gradient_goes_by_the_forward(C, G):
    """Values within roundings of the corner of a ReLU: the gradient passes exactly where the forward's result is above zero."""
    B, S = 1, 64
    g = torch.Generator().manual_seed(62)
    x, gamma = randn(g, B, S, C).to(DEV), (1 + 0.2 * randn(g, C)).to(DEV)
    _, stats = ops.group_norm_act(x, None, None, G)
    mean, rstd = (stats[0, :, k].repeat_interleave(C // G) for k in (0, 1))
    at = torch.arange(C, device=DEV) % S                    # the frame of channel c that beta moves to the corner
    c = torch.arange(C, device=DEV)
    beta = -((x[0, at, c] - mean) * rstd * gamma)
    y, stats = ops.group_norm_act(x, gamma, beta, G, act=_lib.ACT_RELU)
    above = y[0, at, c] > 0
    assert 0 < int(above.sum()) < C                         # of such values some lie on either side
    dy = torch.zeros_like(x)
    dy[0, at, c] = 1.0
    dx, _, dbeta = ops.group_norm_act_backward(dy, x, gamma, beta, stats, G, act=_lib.ACT_RELU)
    assert torch.equal(dbeta, above.float())
    if C == G:                                              # a channel that lets nothing through has no gradient anywhere
        assert torch.equal((dx[0] != 0).any(0), above)


def test_outputs_into_parts_of_frame_major_and_one_frame_tensors():
    g = torch.Generator().manual_seed(64)
    for B, S in ((3, 200), (5, 1)):
        both = randn(g, S, B, 80, dtype=BF16).to(DEV).transpose(0, 1)
        x, gate, dh = both[..., :40], both[..., 40:], place(randn(g, B, S, 40, dtype=BF16), "frames")
        _, _, saved = ops.gated_recurrence(x, gate, save=True)
        want = ops.gated_recurrence_backward(dh, x, gate, saved)
        d = torch.full((S, B, 83), 7.0, dtype=BF16, device=DEV).transpose(0, 1)
        dh0 = ops.gated_recurrence_backward(dh, x, gate, saved, out=(d[..., 1:41], d[..., 41:81]))[2]
        assert torch.equal(d[..., 1:41], want[0]) and torch.equal(d[..., 41:81], want[1]) and torch.equal(dh0, want[2])
        assert bool((d[..., 0] == 7).all()) and bool((d[..., 81:] == 7).all())
        rng = torch.tensor([5, 6], device=DEV)
        drop = ops.dropout(x, 0.2, rng, 4, gate)
        assert ops.dropout(x, 0.2, rng, 4, gate, out=gate) is gate and torch.equal(both[..., 40:], drop)
        with pytest.raises(ValueError):
            ops.dropout(x, 0.2, rng, 4, out=both[..., 20:60])


def test_the_most_utterances():
    """As many one-frame utterances as a launch's threads count: the last of them agree with the same rows alone; one more is refused."""
    B, C, last = (1 << 24) - 1, 2, 1000
    g = torch.Generator(device=DEV).manual_seed(65)
    x, dy = (torch.randn(B, 1, C, generator=g, device=DEV) for _ in range(2))
    y, stats = ops.group_norm_act(x, None, None, 1, eps=0.1, act=1)
    want = oracle.group_norm(x[-last:].cpu(), None, None, 1, 0.1, 1, False, None, dy[-last:].cpu())
    close(y[-last:], *want["y"])
    close(stats[-last:], *want["stats"])
    close(ops.group_norm_act_backward(dy, x, None, None, stats, 1, act=1)[0][-last:], *want["dx"])
    B = (1 << 25) - 1
    x, gate, h0 = (torch.randn(B, 1, 1, generator=g, device=DEV) for _ in range(3))
    x, gate, h0 = x.to(BF16), gate.to(BF16), h0[:, 0]
    h, state, saved = ops.gated_recurrence(x, gate, h0, save=True)
    want = oracle.recurrence(x[-last:].cpu(), gate[-last:].cpu(), h0[-last:].cpu(), None, False, x[-last:].cpu())
    close(h[-last:], *want["h"])
    close(state[-last:], *want["last"])
    for name, v in zip(("dx", "dgate", "dh0"), ops.gated_recurrence_backward(x, x, gate, saved)):
        close(v[-last:], *want[name], name)
    with pytest.raises(_lib.Msf2Error):
        ops.group_norm_act(torch.zeros(1 << 24, 1, C, device=DEV), None, None, 1)
    x = torch.zeros(1 << 25, 1, 1, dtype=BF16, device=DEV)
    with pytest.raises(_lib.Msf2Error):
        ops.gated_recurrence(x, x)


def test_refused_calls_leave_outputs_unannounced():
    """A call that is refused has written nothing: autograd still takes the tensors it was to write for unchanged."""
    x, rng = torch.randn(2, 3, 8, device=DEV), torch.tensor([1, 2], device=DEV)
    _, last, saved = ops.gated_recurrence(x, x, save=True)
    a, b = torch.empty_like(x), torch.empty_like(x)
    long = torch.zeros(2, dtype=torch.int64, device=DEV)
    calls = [lambda: ops.dropout(x, 2.0, rng, out=a), lambda: ops.dropout(x, 0.1, rng, site=-1, out=a), lambda: ops.dropout(x, 0.1, rng.int(), out=a),
             lambda: ops.dropout(x, 0.1, 5, out=a), lambda: ops.dropout(x, 0.1, rng, residual=x.double(), out=a), lambda: ops.dropout(x, 0.1, rng, out=3.0),
             lambda: ops.gated_recurrence_backward(x, x, x, saved[:1], out=(a, b)), lambda: ops.gated_recurrence_backward(x, x, x, 3.0, out=(a, b)),
             lambda: ops.gated_recurrence_backward(x, x, x, saved, dlast=last[:1], out=(a, b)), lambda: ops.gated_recurrence_backward(x, x, x, saved, dlast=1, out=(a, b)),
             lambda: ops.gated_recurrence_backward(x, x, x, saved, lengths=long, out=(a, b)), lambda: ops.gated_recurrence_backward(x, x, x, saved, out=(a, None)),
             lambda: ops.gated_recurrence_backward(x, x, x, saved, out=(a, torch.zeros_like(x, requires_grad=True))),
             lambda: ops.gated_recurrence_backward(x, x, x, saved, out=a), lambda: ops.gated_recurrence(x, x, lengths=long, last=last)]
    for f in calls:
        with pytest.raises(ValueError):
            f()
        assert a._version == b._version == last._version == 0
