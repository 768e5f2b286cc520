"""The training and streaming operators of a gated recurrent block, as they are measured: group norm with an activation
(channels last), the gated linear recurrence, and dropout from a counter-based generator with the residual addition.

``run`` computes a case in elementary torch operations, or, where ``own`` is true, through speech_separation_amd.ops.
Activations are token-major [B, S, C].  Sizes follow the separation model: 512 channels, 256 in the FSMN-family block,
3999 frames for 4 s at 8 kHz, 61499 for the longest input that is separated in one piece, batches of 16 and 64.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ACTS = {"none": 0, "silu": 1, "sigmoid": 2, "relu": 3}
EPS = 1e-5
MOST = 64 * 3999 * 512           # elements of one activation in the largest case


# ------------------------------------------------------------------ cases
def _norm(name, B, S, C, groups, act, act_first, dtype, ragged, train):
    return {"name": name, "op": "norm", "B": B, "S": S, "C": C, "groups": groups, "act": act, "act_first": act_first,
            "dtype": dtype, "ragged": ragged, "train": train}


def _rec(name, B, S, C, dtype, ragged, reverse, packed, train):
    return {"name": name, "op": "rec", "B": B, "S": S, "C": C, "dtype": dtype, "ragged": ragged, "reverse": reverse,
            "packed": packed, "train": train}


def _drop(name, B, S, C, p, dtype, residual, train):
    return {"name": name, "op": "drop", "B": B, "S": S, "C": C, "p": p, "dtype": dtype, "residual": residual, "train": train}


def listed():
    return [
        # half a second of one speaker pair, normalised while it streams: a call that costs little but its launch
        _norm("norm_half_second", 1, 499, 512, 1, "silu", False, "fp32", False, False),
        # the TCN block's order, SiLU then a norm over all channels of an utterance, in a training step of 16 x 4 s
        _norm("norm_tcn_train_fp32", 16, 3999, 512, 1, "silu", True, "fp32", False, True),
        # a batch of utterances of 0 to 7.5 s padded to one length, the FSMN-family block's width, 8 groups
        _norm("norm_ragged_train_bf16", 12, 7499, 256, 8, "silu", False, "bf16", True, True),
        # a batch of 64 x 4 s in inference, 16 groups
        _norm("norm_batch_bf16", 64, 3999, 512, 16, "silu", False, "bf16", False, False),
        # one frame for each of 64 live streams: the state goes in and comes out
        _rec("rec_one_frame", 64, 1, 512, "fp32", False, False, False, False),
        # an odd width and padded utterances, right to left (the second half of a bidirectional block)
        _rec("rec_ragged_train_fp32", 7, 1875, 131, "fp32", True, True, False, True),
        # the longest recording in one piece: one sequence, so the work is split over its length
        _rec("rec_long_bf16", 1, 61499, 512, "bf16", False, False, True, False),
        # training on 16 x 4 s, value and gate side by side as one projection writes them
        _rec("rec_train_fp32", 16, 3999, 512, "fp32", False, False, True, True),
        # training on 64 x 4 s
        _rec("rec_train_bf16", 64, 3999, 512, "bf16", False, False, True, True),
        # half a second of one utterance onto the fp32 residual stream
        _drop("drop_half_second", 1, 499, 512, 0.1, "bf16", "fp32", False),
        # an odd width without a residual
        _drop("drop_odd_train_fp16", 5, 7499, 257, 0.25, "fp16", "none", True),
        # training on 64 x 4 s: bf16 branch, fp32 residual stream
        _drop("drop_train_bf16", 64, 3999, 512, 0.1, "bf16", "fp32", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rec", "drop"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    B, train = _log(rng, 1, 64), rng.random() < 0.5
    if op == "norm":
        groups = rng.choice([1, 1, 2, 4, 8, 16, 32])
        C = groups * _log(rng, max(4, 64 // groups), 1024 // groups)
        S = min(_log(rng, 16, 65536), max(16, MOST // (B * C)))
        act, first = rng.choice(["none", "silu", "silu", "sigmoid", "relu"]), rng.random() < 0.4
        if act == "relu" and train:
            first = True         # a step of the gradient at z = 0 would compare roundings of z, not gradients
        return {k: v for k, v in _norm("", B, S, C, groups, act, first, dtype, rng.random() < 0.4, train).items() if k != "name"}
    C = _log(rng, 33, 1024)
    if op == "rec":
        S = 1 if rng.random() < 0.1 else min(_log(rng, 2, 65536), max(2, MOST // (B * C)))
        return {k: v for k, v in _rec("", B, S, C, dtype, rng.random() < 0.4, rng.random() < 0.4, rng.random() < 0.5,
                                      train).items() if k != "name"}
    S = min(_log(rng, 1, 65536), max(1, MOST // (B * C)))
    return {k: v for k, v in _drop("", B, S, C, rng.choice([0.05, 0.1, 0.25, 0.5]), dtype,
                                   rng.choice(["none", "same", "fp32"]), train).items() if k != "name"}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _lengths(case, g):
    """Utterance lengths of a padded batch: the longest fills it, one is a single frame and one is empty where there is room."""
    if not case["ragged"]:
        return None
    n = (torch.rand(case["B"], generator=g, device=DEV) * case["S"]).to(torch.int32) + 1
    n[0] = case["S"]
    if case["B"] > 2:
        n[1], n[2] = 1, 0
    return n


def prepare(case, seed):
    g, t = _gen(seed), TYPES[case["dtype"]]
    B, S, C = case["B"], case["S"], case["C"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    st = {"case": dict(case)}
    if case["op"] == "norm":
        # activations of a trained network: every channel has its own level and spread
        st["x"] = (randn(B, S, C) * torch.exp(0.3 * randn(C)) + 0.5 * randn(C)).to(t)
        st["gamma"], st["beta"] = 1 + 0.2 * randn(C), 0.2 * randn(C)
        st["lengths"] = _lengths(case, g)
        if case["train"]:
            st["dy"] = randn(B, S, C).to(t)
    elif case["op"] == "rec":
        # gates whose time constants run from one frame to some hundreds
        level = 6 * torch.rand(C, generator=g, device=DEV) - 1
        if case["packed"]:
            both = torch.empty(B, S, 2 * C, device=DEV, dtype=t)
            st["x"], st["gate"] = both[..., :C], both[..., C:]
            st["x"].copy_(randn(B, S, C))
            st["gate"].copy_(randn(B, S, C) * 1.5 + level)
        else:
            st["x"], st["gate"] = randn(B, S, C).to(t), (randn(B, S, C) * 1.5 + level).to(t)
        st["h0"] = randn(B, C)
        st["lengths"] = _lengths(case, g)
        if case["train"]:
            st["dh"], st["dlast"] = randn(B, S, C).to(t), randn(B, C)
    else:
        st["x"] = randn(B, S, C).to(t)
        st["residual"] = None if case["residual"] == "none" else randn(B, S, C).to(torch.float32 if case["residual"] == "fp32" else t)
        st["rng"] = torch.randint(0, 2 ** 62, (2,), generator=g, device=DEV, dtype=torch.int64)
        st["site"] = int(seed) % 97
        if case["train"]:
            st["dy"] = randn(B, S, C).to(t if st["residual"] is None else st["residual"].dtype)
    return st


# ------------------------------------------------------------------ plain forms
def _act(v, act):
    return {"none": lambda: v, "silu": lambda: v / (1 + torch.exp(-v)), "sigmoid": lambda: 1 / (1 + torch.exp(-v)),
            "relu": lambda: torch.clamp(v, min=0)}[act]()


def _act_grad(v, act):
    if act == "none":
        return torch.ones_like(v)
    if act == "relu":
        return (v > 0).to(v.dtype)
    p, q = 1 / (1 + torch.exp(-v)), 1 / (1 + torch.exp(v))
    return p * q if act == "sigmoid" else p * (1 + v * q)


def _rows(st):
    """[B, S, 1]: whether a frame belongs to its utterance."""
    c = st["case"]
    if st["lengths"] is None:
        return None
    return (torch.arange(c["S"], device=DEV) < st["lengths"][:, None])[..., None]


def _plain_norm(st):
    c = st["case"]
    B, S, C, G = c["B"], c["S"], c["C"], c["groups"]
    act, first, t = c["act"], c["act_first"], TYPES[c["dtype"]]
    valid = _rows(st)
    x = st["x"].float()
    n = torch.full((B, 1, 1, 1), S * (C // G), device=DEV, dtype=torch.float32)
    if valid is not None:
        x = torch.where(valid, x, 0.0)
        n = st["lengths"].float().clamp(min=1).view(B, 1, 1, 1) * (C // G)

    def per_group(v):                       # sum over the frames and channels of a group
        v = v if valid is None else torch.where(valid, v, 0.0)
        return v.view(B, S, G, C // G).sum(dim=(1, 3), keepdim=True)

    def spread(s):                          # a group's value at each of its channels
        return s.expand(B, 1, G, C // G).reshape(B, 1, C)

    u = _act(x, act) if first else x
    mean = spread(per_group(u) / n)
    rstd = spread(1 / torch.sqrt(per_group((u - mean) ** 2) / n + EPS))
    xh = (u - mean) * rstd
    z = xh * st["gamma"] + st["beta"]
    y = z if first else _act(z, act)
    if valid is not None:
        y = torch.where(valid, y, 0.0)
    if not c["train"]:
        return [y.to(t)]
    dz = st["dy"].float() * (1 if first else _act_grad(z, act))
    if valid is not None:
        dz = torch.where(valid, dz, 0.0)
    dbeta, dgamma = dz.sum(dim=(0, 1)), (dz * xh).sum(dim=(0, 1))
    k = dz * st["gamma"]
    dx = rstd * (k - spread(per_group(k) / n) - xh * spread(per_group(k * xh) / n))
    if first:
        dx = dx * _act_grad(x, act)
    if valid is not None:
        dx = torch.where(valid, dx, 0.0)
    return [y.to(t), dx.to(t), dgamma, dbeta]


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from h_{-1} = 0, by doubling: after k passes a row holds the last 2^k terms."""
    d = 1
    while d < a.shape[1]:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return b


def _plain_rec(st):
    c = st["case"]
    t, valid = TYPES[c["dtype"]], _rows(st)
    x, gate = st["x"].float(), st["gate"].float()
    a, na = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
    b = na * x
    if valid is not None:                   # a frame past the end hands the state on
        a, b = torch.where(valid, a, 1.0), torch.where(valid, b, 0.0)
    flip = (lambda v: v.flip(1)) if c["reverse"] else (lambda v: v)
    af, bf = flip(a), flip(b).clone()
    bf[:, 0] += af[:, 0] * st["h0"]
    hf = _scan(af, bf)
    h, last = flip(hf), hf[:, -1].contiguous()
    out = h if valid is None else torch.where(valid, h, 0.0)
    if not c["train"]:
        return [out.to(t), last]
    before = flip(torch.cat([st["h0"][:, None], hf[:, :-1]], 1))
    dh = st["dh"].float()
    if valid is not None:
        dh = torch.where(valid, dh, 0.0)
    dhf = flip(dh)
    # E_t = a_t (dh_t + E_{t+1}), the gradient that a frame hands to the one before it
    eb = (af * dhf).flip(1)
    eb[:, 0] += af[:, -1] * st["dlast"]
    E = _scan(af.flip(1), eb).flip(1)
    D = flip(dhf + torch.cat([E[:, 1:], st["dlast"][:, None]], 1))
    dx, dgate, dh0 = na * D, a * na * (before - x) * D, E[:, 0].contiguous()
    if valid is not None:
        dx, dgate = torch.where(valid, dx, 0.0), torch.where(valid, dgate, 0.0)
    return [out.to(t), last, dx.to(t), dgate.to(t), dh0]


def _philox(c0, c1, c2, c3, k0, k1):
    """Philox4x32-10 (Salmon et al. 2011) on int64 tensors that hold 32-bit words."""
    low = 0xFFFFFFFF

    def mul(m, v):                          # high and low word of a 32 x 32 bit product
        part = v * (m & 0xFFFF)
        top = (part >> 16) + v * (m >> 16)
        return top >> 16, ((top & 0xFFFF) << 16) | (part & 0xFFFF)

    for _ in range(10):
        h0, l0 = mul(0xD2511F53, c0)
        h1, l1 = mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c0, c1, c2, c3


def _kept(st):
    c = st["case"]
    rows, C, low = c["B"] * c["S"], c["C"], 0xFFFFFFFF
    per = -(-C // 8)
    block = torch.arange(rows * per, device=DEV, dtype=torch.int64)
    seed, step = st["rng"][0], st["rng"][1]
    words = _philox(block & low, block >> 32, (step & low).expand_as(block), torch.full_like(block, st["site"]),
                    seed & low, (seed >> 32) & low)
    bits = torch.stack([v for w in words for v in (w & 0xFFFF, w >> 16)], -1)
    return (bits >= round(c["p"] * 65536)).view(c["B"], c["S"], per * 8)[..., :C]


def _plain_drop(st):
    c = st["case"]
    kept, thr = _kept(st), round(c["p"] * 65536)
    scale = 65536 / (65536 - thr)
    y = torch.where(kept, st["x"].float() * scale, 0.0)
    if st["residual"] is None:
        y = y.to(TYPES[c["dtype"]])
    else:
        y = (st["residual"].float() + y).to(st["residual"].dtype)
    if not c["train"]:
        return [y]
    return [y, torch.where(kept, st["dy"].float() * scale, 0.0).to(TYPES[c["dtype"]])]


# ------------------------------------------------------------------ the framework's operators
def _own_norm(st):
    from speech_separation_amd import ops
    c = st["case"]
    kw = {"act": ACTS[c["act"]], "act_first": c["act_first"], "lengths": st["lengths"]}
    y, stats = ops.group_norm_act(st["x"], st["gamma"], st["beta"], c["groups"], eps=EPS, **kw)
    if not c["train"]:
        return [y]
    return [y, *ops.group_norm_act_backward(st["dy"], st["x"], st["gamma"], st["beta"], stats, c["groups"], **kw)]


def _own_rec(st):
    from speech_separation_amd import ops
    c = st["case"]
    kw = {"lengths": st["lengths"], "reverse": c["reverse"]}
    h, last, saved = ops.gated_recurrence(st["x"], st["gate"], h0=st["h0"], save=c["train"], **kw)
    if not c["train"]:
        return [h, last]
    return [h, last, *ops.gated_recurrence_backward(st["dh"], st["x"], st["gate"], saved, dlast=st["dlast"], **kw)]


def _own_drop(st):
    from speech_separation_amd import ops
    c = st["case"]
    y = ops.dropout(st["x"], c["p"], st["rng"], site=st["site"], residual=st["residual"])
    if not c["train"]:
        return [y]
    return [y, ops.dropout_backward(st["dy"], c["p"], st["rng"], site=st["site"], dtype=st["x"].dtype)]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "rec": _own_rec, "drop": _own_drop}[op](state)
    return {"norm": _plain_norm, "rec": _plain_rec, "drop": _plain_drop}[op](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    B, S, C = case["B"], case["S"], case["C"]
    e, n = 4 if case["dtype"] == "fp32" else 2, B * S * C
    if case["op"] == "norm":
        if not case["train"]:
            return {"bytes": 2 * n * e + 8 * C, "flops": 12 * n}
        return {"bytes": 4 * n * e + 16 * C, "flops": 32 * n}                   # x, dy | y, dx
    if case["op"] == "rec":
        if not case["train"]:
            return {"bytes": 3 * n * e + 8 * B * C, "flops": 10 * n}            # x, gate | h
        return {"bytes": 6 * n * e + 16 * B * C, "flops": 30 * n}               # x, gate, dh | h, dx, dgate
    r = {"none": e, "same": e, "fp32": 4}[case["residual"]]
    there = n * (e + r + (0 if case["residual"] == "none" else r))
    return {"bytes": there + (n * (r + e) if case["train"] else 0), "flops": 15 * n * (2 if case["train"] else 1)}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_norm(case, st):
    B, S, C, G = case["B"], case["S"], case["C"], case["groups"]
    f = {"none": lambda v: v, "silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, "relu": torch.relu}[case["act"]]
    gamma, beta = (st[k].double().requires_grad_() for k in ("gamma", "beta"))
    y = torch.zeros(B, S, C, device=DEV, dtype=torch.float64)
    dx, dgamma, dbeta = torch.zeros_like(y), torch.zeros_like(gamma), torch.zeros_like(beta)
    lengths = [S] * B if st["lengths"] is None else st["lengths"].tolist()
    for b, n in enumerate(lengths):
        if not n:
            continue
        x = st["x"][b, :n].double().requires_grad_()
        u = (f(x) if case["act_first"] else x).reshape(n, G, -1)
        var, mean = torch.var_mean(u, dim=(0, 2), unbiased=False, keepdim=True)
        z = ((u - mean) / torch.sqrt(var + EPS)).reshape(n, C) * gamma + beta
        z = z if case["act_first"] else f(z)
        y[b, :n] = z.detach()
        if case["train"]:
            d = torch.autograd.grad(z, (x, gamma, beta), st["dy"][b, :n].double())
            dx[b, :n] = d[0]
            dgamma, dbeta = dgamma + d[1], dbeta + d[2]
    return [y, dx, dgamma.detach(), dbeta.detach()] if case["train"] else [y]


def _exact_rec(case, st):
    B, S, C = case["B"], case["S"], case["C"]
    order = range(S - 1, -1, -1) if case["reverse"] else range(S)
    x, a = (st[k].double().transpose(0, 1).contiguous() for k in ("x", "gate"))
    a = torch.sigmoid(a)
    n = torch.full((B,), S, device=DEV) if st["lengths"] is None else st["lengths"]
    live = torch.arange(S, device=DEV)[:, None] < n
    a[~live], x[~live] = 1.0, 0.0
    b = (1 - a) * x
    h, before, state = torch.empty_like(a), torch.empty_like(a) if case["train"] else None, st["h0"].double()
    for t in order:
        if case["train"]:
            before[t] = state
        state = torch.addcmul(b[t], a[t], state, out=h[t])
    last = state.clone()
    h[~live] = 0.0
    h = h.transpose(0, 1)
    if not case["train"]:
        return [h, last]
    dh = st["dh"].double().transpose(0, 1).contiguous()
    dh[~live] = 0.0
    carry = st["dlast"].double()
    for t in reversed(order):
        carry = dh[t].add_(carry) * a[t]     # dh[t] is from here on the whole gradient of h_t
    dx = (1 - a) * dh
    dgate = dx * a * (before - x)
    dgate[~live] = 0.0
    return [h, last, dx.transpose(0, 1), dgate.transpose(0, 1), carry]


def _exact_drop(case, st):
    B, S, C = case["B"], case["S"], case["C"]
    per, thr = (C + 7) // 8, math.floor(case["p"] * 65536 + 0.5)
    seed, step = (int(v) for v in st["rng"].tolist())
    word = np.uint64(0xFFFFFFFF)
    kept = torch.empty(B * S, per * 8, dtype=torch.bool)
    at = max(1, (1 << 20) // per)
    for r in range(0, B * S, at):
        rows = min(at, B * S - r)
        block = np.arange(r * per, (r + rows) * per, dtype=np.uint64)
        ctr = [block & word, block >> np.uint64(32), np.full_like(block, step & 0xFFFFFFFF), np.full_like(block, st["site"])]
        key = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
        for i in range(10):
            p, q = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
            k = [np.uint64((key[0] + i * 0x9E3779B9) & 0xFFFFFFFF), np.uint64((key[1] + i * 0xBB67AE85) & 0xFFFFFFFF)]
            ctr = [(q >> np.uint64(32)) ^ ctr[1] ^ k[0], q & word, (p >> np.uint64(32)) ^ ctr[3] ^ k[1], p & word]
        bits = np.stack(ctr, -1).astype("<u4").view("<u2")
        kept[r:r + rows] = torch.from_numpy(bits.reshape(rows, per * 8) >= thr)
    kept = kept[:, :C].to(DEV).view(B, S, C)
    scale = 65536 / (65536 - thr)
    y = st["x"].double() * scale * kept
    if st["residual"] is not None:
        y += st["residual"].double()
    return [y, st["dy"].double() * scale * kept] if case["train"] else [y]


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "rec": _exact_rec, "drop": _exact_drop}[case["op"]](case, st)
