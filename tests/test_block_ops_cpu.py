"""What the block operators refuse, and the 64-bit forms that their kernels are tested against: all of it without a GPU."""
import numpy as np
import pytest
import torch

from tests import block_oracle as oracle
from speech_separation_amd import _lib, ops

P = 4096            # an address that no entry point may get as far as to use


def _norm(lib, **kw):
    a = dict(x=P, gamma=P, beta=P, lengths=None, y=P, stats=P, B=2, S=3, C=8, groups=2, eps=1e-5, act=1, first=0, type=0, ws=P, n=1 << 30)
    a.update(kw)
    return lib.msf2_group_norm_act(a["x"], 24, 8, a["gamma"], a["beta"], a["lengths"], a["y"], 24, 8, a["stats"], a["B"], a["S"], a["C"],
                                   a["groups"], a["eps"], a["act"], a["first"], a["type"], a["ws"], a["n"], None)


def _norm_backward(lib, **kw):
    a = dict(dy=P, x=P, stats=P, dx=P, B=2, S=3, C=8, groups=2, act=1, type=0, ws=P, n=1 << 30)
    a.update(kw)
    return lib.msf2_group_norm_act_backward(a["dy"], 24, 8, a["x"], 24, 8, P, P, a["stats"], None, a["dx"], 24, 8, P, P, a["B"], a["S"], a["C"],
                                            a["groups"], a["act"], 0, a["type"], a["ws"], a["n"], None)


def _rec(lib, **kw):
    a = dict(x=P, gate=P, h=P, B=2, S=3, C=8, type=0, ws=P, n=1 << 30)
    a.update(kw)
    return lib.msf2_gated_recurrence(a["x"], 24, 8, a["gate"], 24, 8, P, None, a["h"], 24, 8, P, P, a["B"], a["S"], a["C"], 0, a["type"],
                                     a["ws"], a["n"], None)


def _rec_backward(lib, **kw):
    a = dict(dh=P, x=P, gate=P, saved=P, dx=P, dgate=P, B=2, S=3, C=8, type=0, ws=P, n=1 << 30)
    a.update(kw)
    return lib.msf2_gated_recurrence_backward(a["dh"], 24, 8, a["x"], 24, 8, a["gate"], 24, 8, a["saved"], P, None, a["dx"], 24, 8, a["dgate"],
                                              24, 8, P, a["B"], a["S"], a["C"], 0, a["type"], a["ws"], a["n"], None)


def _drop(lib, **kw):
    a = dict(x=P, r=None, y=P, rng=P, p=0.1, B=2, S=3, C=8, x_type=0, y_type=0)
    a.update(kw)
    return lib.msf2_dropout(a["x"], 24, 8, a["r"], 24, 8, a["y"], 24, 8, a["rng"], 0, a["p"], a["B"], a["S"], a["C"], a["x_type"], a["y_type"], None)


BAD_SIZES = [dict(B=0), dict(S=0), dict(C=0), dict(B=-1), dict(S=-5), dict(C=-8), dict(B=2 ** 31 - 1, S=2 ** 31 - 1, C=2 ** 20), dict(type=3), dict(type=-1)]


@pytest.mark.parametrize("call,bad", [
    *[(_norm, b) for b in BAD_SIZES + [dict(x=None), dict(y=None), dict(stats=None), dict(groups=3), dict(groups=0), dict(groups=-2), dict(eps=-1.0),
                                       dict(eps=float("nan")), dict(act=4), dict(act=-1)]],
    *[(_norm_backward, b) for b in BAD_SIZES + [dict(dy=None), dict(x=None), dict(stats=None), dict(dx=None), dict(groups=5), dict(act=9), dict(ws=None)]],
    *[(_rec, b) for b in BAD_SIZES + [dict(x=None), dict(gate=None), dict(h=None)]],
    *[(_rec_backward, b) for b in BAD_SIZES + [dict(dh=None), dict(x=None), dict(gate=None), dict(saved=None), dict(dx=None), dict(dgate=None)]],
    *[(_drop, b) for b in BAD_SIZES[:7] + [dict(x_type=3), dict(y_type=-1), dict(x_type=1, y_type=2), dict(x_type=2, y_type=1), dict(x=None), dict(y=None),
                                           dict(rng=None), dict(p=-0.1), dict(p=1.5), dict(p=float("nan"))]],
])
def test_entry_points_refuse(call, bad):
    assert call(_lib.load(), **bad) == -1


def test_entry_points_refuse_a_short_workspace():
    lib = _lib.load()
    need = lib.msf2_group_norm_act_backward_ws_bytes(2, 3, 8, 2, 0)
    assert need > 0 and _norm_backward(lib, n=need - 1) == -2
    for call, need in ((_norm, lib.msf2_group_norm_act_ws_bytes(4, 5000, 512, 2, 0)), (_rec, lib.msf2_gated_recurrence_ws_bytes(4, 5000, 512, 0)),
                       (_rec_backward, lib.msf2_gated_recurrence_backward_ws_bytes(4, 5000, 512, 0))):
        if need:
            assert call(lib, B=4, S=5000, C=512, n=need - 1) == -2


def test_workspace_queries_refuse_bad_sizes():
    lib = _lib.load()
    for B, S, C in ((0, 3, 8), (2, 0, 8), (2, 3, 0), (-1, 3, 8)):
        assert lib.msf2_group_norm_act_ws_bytes(B, S, C, 1, 0) == 0
        assert lib.msf2_group_norm_act_backward_ws_bytes(B, S, C, 1, 0) == 0
        assert lib.msf2_gated_recurrence_ws_bytes(B, S, C, 0) == 0
        assert lib.msf2_gated_recurrence_backward_ws_bytes(B, S, C, 0) == 0
    assert lib.msf2_group_norm_act_backward_ws_bytes(2, 3, 8, 0, 0) == 0
    assert lib.msf2_group_norm_act_backward_ws_bytes(2, 3, 8, 3, 0) == 0


@pytest.mark.parametrize("call", [
    lambda x: ops.group_norm_act(x, None, None, 2), lambda x: ops.group_norm_act_backward(x, x, None, None, x, 2),
    lambda x: ops.gated_recurrence(x, x), lambda x: ops.gated_recurrence_backward(x, x, x, x),
    lambda x: ops.dropout(x, 0.1, torch.zeros(2, dtype=torch.int64)), lambda x: ops.dropout_backward(x, 0.1, torch.zeros(2, dtype=torch.int64))])
@pytest.mark.parametrize("x", [torch.zeros(2, 3, 8), None, torch.zeros(6, 8)])
def test_wrappers_refuse_what_is_not_on_the_gpu(call, x):
    with pytest.raises(ValueError):
        call(x)


def test_overlap_check():
    both = torch.zeros(2, 5, 16)
    x, g = both[..., :8], both[..., 8:]
    assert not ops._clash(x, g) and not ops._clash(g, x)
    assert ops._clash(x, x) and ops._clash(both[..., 1:9], x) and ops._clash(both[..., 4:12], g)
    assert not ops._clash(both[:1], both[1:]) and not ops._clash(both[0], both[1])
    assert ops._clash(both[:, 1:], both[:, :-1])
    assert not ops._clash(both, torch.zeros(2, 5, 16)) and not ops._clash(both[:0], both)


def test_oracle_philox_gives_the_published_words():
    """The known answers of the generator's authors for ten rounds: all zero, all ones, and the digits of pi."""
    known = [((0,) * 4, (0,) * 2, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
             ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
             ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))]
    for c, k, want in known:
        assert tuple(int(v) for v in oracle.philox(c, k)) == want


def test_oracle_gradients_agree_with_differences():
    """The formulas of the oracle's backward passes against central differences of its forward passes."""
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    lengths = torch.tensor([5, 0, 3], dtype=torch.int32)

    def check(f, arg, grad, at):
        for i in at:
            d = torch.zeros_like(arg).view(-1)
            d[i] = 1e-6
            d = d.view_as(arg)
            assert abs(float(f(arg + d) - f(arg - d)) / 2e-6 - float(grad.reshape(-1)[i])) < 1e-7

    x, dy, ga, be = r(3, 5, 6), r(3, 5, 6), r(6), r(6)
    for which in (0, 1, 2, 3):
        for first in (False, True):
            def f(x=x, ga=ga, be=be):
                return (oracle.group_norm(x, ga, be, 2, 1e-5, which, first, lengths)["y"][0] * dy).sum()
            o = oracle.group_norm(x, ga, be, 2, 1e-5, which, first, lengths, dy)
            check(lambda v: f(x=v), x, o["dx"][0], (0, 7, 29, 45, 60, 77, 89))
            check(lambda v: f(ga=v), ga, o["dgamma"][0], range(6))
            check(lambda v: f(be=v), be, o["dbeta"][0], range(6))
    gate, h0, dl = r(3, 5, 6), r(3, 6), r(3, 6)
    for reverse in (False, True):
        def f(x=x, gate=gate, h0=h0):
            o = oracle.recurrence(x, gate, h0, lengths, reverse)
            return (o["h"][0] * dy).sum() + (o["last"][0] * dl).sum()
        o = oracle.recurrence(x, gate, h0, lengths, reverse, dy, dl)
        check(lambda v: f(x=v), x, o["dx"][0], (0, 7, 29, 45, 60, 77, 89))
        check(lambda v: f(gate=v), gate, o["dgate"][0], (0, 7, 29, 45, 60, 77, 89))
        check(lambda v: f(h0=v), h0, o["dh0"][0], range(18))


def test_oracle_keep_rate():
    for p in (0.1, 0.5):
        k = oracle.keep((4, 250, 512), p, 1234567890123, 5, 3).double()
        sigma = (p * (1 - p) / k.numel()) ** 0.5
        assert abs(float(k.mean()) - (1 - p)) < 5 * sigma
    assert np.array_equal(oracle.keep((1, 6, 17), 0.3, 1, 2, 3)[0, 3:].numpy(), oracle.keep((2, 3, 17), 0.3, 1, 2, 3)[1].numpy())


def test_overlap_check_of_other_layouts():
    """Frame-major halves, one-frame halves whose unused strides differ, frames before and behind one another: apart; a part of any of them
    moved by less than its own width, or onto itself: not."""
    turned = torch.zeros(5, 4, 35).transpose(0, 1)                       # [S, B, C] in memory
    x, g = turned[..., :16], turned[..., 16:32]
    assert not ops._clash(x, g) and not ops._clash(g, x)
    assert ops._clash(x, x) and ops._clash(x, turned[..., 15:31]) and ops._clash(turned[..., 17:33], g) and ops._clash(turned, turned)
    assert not ops._clash(turned[:, :2], turned[:, 2:4]) and not ops._clash(turned[:2], turned[2:]) and ops._clash(turned[:, 1:], turned[:, :-1])
    assert ops._clash(turned[:3, :, :16], turned[1:, :, 10:26]) and not ops._clash(turned[:3, :, :16], turned[1:, :, 16:32])
    one = torch.zeros(4, 1, 32)
    x, g = one[..., :16].as_strided((4, 1, 16), (32, 7, 1)), one[..., 16:]
    assert not ops._clash(x, g) and not ops._clash(g, x) and ops._clash(x, one[..., :16]) and ops._clash(x, one[..., 3:19])
    both = torch.zeros(3, 10, 8)
    assert not ops._clash(both[:, :5], both[:, 5:]) and ops._clash(both[:, :6], both[:, 4:])
    one = torch.zeros(3, 10, 2)
    assert not ops._clash(one[..., :1], one[..., 1:]) and ops._clash(one[..., :1], one[..., :1])


def test_overlap_check_agrees_with_the_addresses():
    rng = np.random.default_rng(63)
    n = 0
    for _ in range(3000):
        B, S, C = (int(v) for v in rng.integers(1, 5, 3))
        order = rng.permutation(2)
        inner = C + int(rng.integers(0, 4))
        st = [0, 0]
        st[order[0]] = inner
        st[order[1]] = inner * (S if order[0] else B) + int(rng.integers(0, 7))
        base = torch.zeros(400)
        t, u = (base.as_strided((B, S, C), (st[0], st[1], 1), int(rng.integers(0, 60))) for _ in range(2))
        at = [{int(v.storage_offset() + b * st[0] + s * st[1] + c) for b in range(B) for s in range(S) for c in range(C)} for v in (t, u)]
        assert ops._clash(t, u) == bool(at[0] & at[1]), (B, S, C, st, t.storage_offset(), u.storage_offset())
        n += bool(at[0] & at[1])
    assert 500 < n < 2500


@pytest.mark.parametrize("call,bad", [
    *[(call, dict(B=1, S=1, C=C, **kw)) for call, kw in ((_norm, dict(groups=1)), (_norm_backward, dict(groups=1)), (_rec, {}), (_rec_backward, {}), (_drop, {}))
      for C in (2 ** 30, 2 ** 31 - 8, 2 ** 31 - 1)],
    (_norm, dict(B=2 ** 24, S=1)), (_norm_backward, dict(B=2 ** 24, S=1, n=1 << 40)), (_norm, dict(B=2 ** 31 - 1, S=1, n=1 << 40)),
    (_rec, dict(B=2 ** 26, S=1)), (_rec_backward, dict(B=2 ** 26, S=1)), (_rec, dict(B=2 ** 31 - 1, S=1))])
def test_entry_points_refuse_what_their_indices_do_not_hold(call, bad):
    """Channels whose index would pass 2^31 within the last lanes, and launches of more threads than the hardware counts."""
    assert call(_lib.load(), **bad) == -1


def test_autograd_keeps_states_for_a_backward_pass_only(monkeypatch):
    """With a learned first state, say: its gradient is asked for, but not under no_grad or inference_mode."""
    from speech_separation_amd import autograd
    asked = []

    def fake(x, gate, h0, lengths, reverse, save):
        asked.append(save)
        return x * 1, h0 * 1, torch.zeros(1) if save else None

    monkeypatch.setattr(ops, "gated_recurrence", fake)
    x, h0 = torch.zeros(2, 3, 8), torch.zeros(2, 8, requires_grad=True)
    for mode, want in ((torch.enable_grad, True), (torch.no_grad, False), (torch.inference_mode, False)):
        with mode():
            autograd.gated_recurrence(x, x, h0)
        assert asked.pop() is want, mode
    autograd.gated_recurrence(x, x, h0.detach())
    assert asked.pop() is False
