"""Thin torch-tensor wrappers over the single-operator entry points of libmsf2
(include/msf2.h).  Host plumbing only: shape checks, output / workspace
allocation from torch's allocator, the current HIP stream.  Every function
raises if the library is missing and requires CUDA (HIP) tensors: contiguous
fp32 ones, except for the block operators at the end (group norm, gated
recurrence, dropout), which take fp32, bf16 and fp16 and any batch and frame
strides as long as channels are contiguous.  Those run on the device of their
operands, whichever device is current, and on its current stream."""
import torch

from . import _lib


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _ws(nbytes, dev):
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=dev)


def _chk(*ts):
    for t in ts:
        if not (t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()):
            raise ValueError("expected contiguous fp32 tensors on the GPU")


def encoder(mix, enc_w_tapmajor, eps=1e-8):
    """mix [B,T], enc_w [16,C] -> (enc [B,S,C], stats [B,2] = (mean, rstd))."""
    lib = _lib.load()
    _chk(mix, enc_w_tapmajor)
    B, T = mix.shape
    C = enc_w_tapmajor.shape[1]
    S = lib.msf2_num_frames(T)
    enc = torch.empty((B, S, C), device=mix.device)
    stats = torch.empty((B, 2), device=mix.device)
    n = lib.msf2_stats_ws_bytes(B, S)
    ws = _ws(n, mix.device)
    _lib.check(lib.msf2_encoder(mix.data_ptr(), enc_w_tapmajor.data_ptr(), enc.data_ptr(), stats.data_ptr(),
                                eps, B, T, C, ws.data_ptr(), ws.numel(), _stream(mix)), "msf2_encoder")
    return enc, stats


def dwconv17(x, dw_tapmajor, out=None, accumulate=False):
    """x [B,S,C] -> x + dwconv17(x); with accumulate, added onto `out`."""
    lib = _lib.load()
    _chk(x, dw_tapmajor)
    B, S, C = x.shape
    if out is None:
        out = torch.empty_like(x)
    _chk(out)
    _lib.check(lib.msf2_dwconv17(x.data_ptr(), C, dw_tapmajor.data_ptr(), out.data_ptr(), C, B, S, C,
                                 int(accumulate), _stream(x)), "msf2_dwconv17")
    return out


def linear(x, W, b=None, shift=False, scale_norm=False, act=0, precision=_lib.PREC_FP32):
    """x [B,S,K], W [N,K] -> act(rowscale(shift(x)) W^T + b) [B,S,N]."""
    lib = _lib.load()
    _chk(x, W)
    B, S, K = x.shape
    N = W.shape[0]
    if precision == _lib.PREC_BF16:          # the bf16 kernels take the weight matrix as bf16
        W = W.to(torch.bfloat16).contiguous()
    y = torch.empty((B, S, N), device=x.device)
    n = lib.msf2_linear_ws_bytes(B, S)
    ws = _ws(n, x.device)
    _lib.check(lib.msf2_linear(x.data_ptr(), K, W.data_ptr(), b.data_ptr() if b is not None else None, y.data_ptr(),
                               N, B, S, K, N, int(shift), int(scale_norm), act, precision, ws.data_ptr(), ws.numel(),
                               _stream(x)), "msf2_linear")
    return y


def flash_attention(hu, gamma, beta, freqs, precision=_lib.PREC_FP32):
    """hu [B,S,2E+128] = v|u|qk -> o [B,S,E]."""
    lib = _lib.load()
    _chk(hu, gamma, beta, freqs)
    B, S, W = hu.shape
    E = (W - _lib.QK_DIM) // 2
    o = torch.empty((B, S, E), device=hu.device)
    n = lib.msf2_flash_attention_ws_bytes(B, S, E)
    ws = _ws(n, hu.device)
    _lib.check(lib.msf2_flash_attention(hu.data_ptr(), W, gamma.data_ptr(), beta.data_ptr(), freqs.data_ptr(),
                                        o.data_ptr(), B, S, E, precision, ws.data_ptr(), ws.numel(), _stream(hu)),
               "msf2_flash_attention")
    return o


def gated_tcn(x, layer_weights, precision=_lib.PREC_FP32):
    """In place on x [B,S,C]; layer_weights: a _lib.LayerWeights (from PackedWeights.layers[i])."""
    lib = _lib.load()
    _chk(x)
    B, S, C = x.shape
    n = lib.msf2_gated_tcn_ws_bytes(B, S, C)
    ws = _ws(n, x.device)
    _lib.check(lib.msf2_gated_tcn(x.data_ptr(), layer_weights, B, S, C, precision, ws.data_ptr(), ws.numel(),
                                  _stream(x)), "msf2_gated_tcn")
    return x


def decoder(sep, dec_w, T):
    """sep [B,S,C] (encoder output times mask), dec_w [C,16] -> est [B,T]."""
    lib = _lib.load()
    _chk(sep, dec_w)
    B, S, C = sep.shape
    est = torch.empty((B, T), device=sep.device)
    n = lib.msf2_decoder_ws_bytes(B, S)
    ws = _ws(n, sep.device)
    _lib.check(lib.msf2_decoder(sep.data_ptr(), dec_w.data_ptr(), est.data_ptr(), B, S, C, T, ws.data_ptr(),
                                ws.numel(), _stream(sep)), "msf2_decoder")
    return est


def tcn_pointwise(h, t, bstat, tcn_weights, precision=_lib.PREC_FP32):
    """h, t [B,S,C]; bstat [B,2]; tcn_weights: a _lib.TcnWeights -> new h (one kernel launch)."""
    lib = _lib.load()
    _chk(h, t, bstat)
    B, S, C = h.shape
    out = torch.empty_like(h)
    _lib.check(lib.msf2_tcn_pointwise(h.data_ptr(), t.data_ptr(), bstat.data_ptr(), tcn_weights, out.data_ptr(),
                                      B, S, C, precision, _stream(h)), "msf2_tcn_pointwise")
    return out


def pit_si_snr(est, src):
    """est, src: [2, B, T] fp32 on the GPU -> (si_snr [B, 2 (source), 2 (estimate)] dB, best [B] dB,
    perm [B] int32: 0 identity, 1 swapped).  Reference: losses/loss.py:653-723 with the 2-source PitWrapper."""
    lib = _lib.load()
    _chk(est, src)
    assert est.shape == src.shape and est.shape[0] == 2 and est.dim() == 3
    _, B, T = est.shape
    si = torch.empty((B, 2, 2), dtype=torch.float32, device=est.device)
    best = torch.empty((B,), dtype=torch.float32, device=est.device)
    perm = torch.empty((B,), dtype=torch.int32, device=est.device)
    ws = _ws(lib.msf2_pit_si_snr_ws_bytes(B, T), est.device)
    _lib.check(lib.msf2_pit_si_snr(est.data_ptr(), src.data_ptr(), si.data_ptr(), best.data_ptr(), perm.data_ptr(), B, T,
                                   ws.data_ptr(), ws.numel(), _stream(est)), "msf2_pit_si_snr")
    return si, best, perm


def pit_si_snr_noalloc(est, src, si, best, perm):
    """pit_si_snr for callers that cannot allocate: every buffer, outputs included, comes from the caller and the
    library's partial sums live in its fixed device array (msf2_pit_si_snr_noalloc).  Nothing is allocated here.
    The library uses the array of the thread's current device, so the call is made with the operands' device current."""
    lib = _lib.load()
    _chk(est, src, si, best)
    if est.shape != src.shape or est.dim() != 3 or est.shape[0] != 2:
        raise ValueError("est and src must both be [2, B, T]")
    _, B, T = est.shape
    if not (perm.is_cuda and perm.dtype == torch.int32 and perm.is_contiguous() and tuple(perm.shape) == (B,)):
        raise ValueError("perm must be a contiguous int32 tensor [B] on the GPU")
    if tuple(si.shape) != (B, 2, 2) or tuple(best.shape) != (B,):
        raise ValueError("si must be [B, 2, 2] and best [B]")
    if any(t.device != est.device for t in (src, si, best, perm)):
        raise ValueError("all tensors must live on one GPU")
    with torch.cuda.device(est.device):
        _lib.check(lib.msf2_pit_si_snr_noalloc(est.data_ptr(), src.data_ptr(), si.data_ptr(), best.data_ptr(), perm.data_ptr(),
                                               B, T, _stream(est)), "msf2_pit_si_snr_noalloc")


def gated_fsmn(x, packed):
    """x: [B, S, dim] fp32 on the GPU; packed = packing.pack_fsmn_block(...).  Reference:
    Gated_FSMN_Block_Dilated.forward (mossformer2_block.py:456-463)."""
    import ctypes as C
    lib = _lib.load()
    w, dim, inner, _keep = packed
    _chk(x)
    B, S, D = x.shape
    assert D == dim
    y = torch.empty_like(x)
    ws = _ws(lib.msf2_gated_fsmn_ws_bytes(B, S, dim, inner), x.device)
    _lib.check(lib.msf2_gated_fsmn(x.data_ptr(), C.byref(w), y.data_ptr(), B, S, dim, inner, ws.data_ptr(), ws.numel(),
                                   _stream(x)), "msf2_gated_fsmn")
    return y


# The current stream's handle without the Python object around it: 2 us less in a call that takes about 10.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


# ---- operators of a gated recurrent block: group norm with an activation, gated recurrence, dropout ------------------
# Plain functions: they record nothing for autograd (speech_separation_amd.autograd does) and they may be captured into a
# HIP graph, workspaces included, which come from torch's allocator for every call.
_TYPES = {torch.float32: _lib.TYPE_FP32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_FP16}


def _rows(t, name, like=None, same_type=True):
    """Address, batch stride and frame stride of a [B, S, C] operand, `like` another one."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 3 and t.dtype in _TYPES):
        raise ValueError(f"{name}: expected a [B, S, C] fp32, bf16 or fp16 tensor on the GPU")
    if like is not None and (t.shape != like.shape or t.device != like.device or (same_type and t.dtype != like.dtype)):
        raise ValueError(f"{name}: expected shape {tuple(like.shape)}, {like.dtype} on {like.device}, "
                         f"got {tuple(t.shape)}, {t.dtype} on {t.device}")
    b, s, c = t.stride()
    if c != 1 and t.shape[2] > 1:
        raise ValueError(f"{name}: channels must be contiguous (stride 1), got strides {t.stride()}")
    return t.data_ptr(), b, s


def _span(t):
    """First address and the one past the last of a tensor's elements."""
    n = sum((k - 1) * st for k, st in zip(t.shape, t.stride())) + 1 if t.numel() else 0
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def _meets(off, axes):
    """Whether off = sum d_i stride_i with |d_i| < size_i, axes = (stride, size) from the widest stride down.  Of a tensor whose
    elements do not share addresses the rest reaches less than a stride, so three steps of an axis are tried at most."""
    if not axes:
        return off == 0
    (st, n), rest = axes[0], axes[1:]
    reach = sum((k - 1) * t for t, k in rest)
    if st == 0:
        return _meets(off, rest)
    return any(_meets(off - d * st, rest) for d in range(max(1 - n, -((reach - off) // st)), min(n - 1, (off + reach) // st) + 1))


def _clash(t, u):
    """Whether two tensors share memory.  Those of one shape and the same strides (those of one-element dimensions aside) are
    compared element by element, so parts of one larger tensor are told apart however it is laid out."""
    (a, b), (c, d) = _span(t), _span(u)
    if b <= c or d <= a or a == b or c == d:
        return False
    e = t.element_size()
    axes = [sorted(((st, n) for st, n in zip(v.stride(), v.shape) if n > 1), reverse=True) for v in (t, u)]
    if t.shape == u.shape and axes[0] == axes[1] and e == u.element_size() and (c - a) % e == 0:
        return _meets((c - a) // e, axes[0])
    return True


def _out_rows(t, name, like, same_type=True, apart=(), same=()):
    """_rows of an operand that is written: no two of its elements share an address, nor with those of `apart`; `same` may
    be the very same tensor."""
    r = _rows(t, name, like, same_type)
    (B, S, C), (_, b, s) = t.shape, r
    if t.numel() and not ((S == 1 or s >= C) and (B == 1 or b >= C) and
                          (B == 1 or S == 1 or b >= (S - 1) * s + C or s >= (B - 1) * b + C)):
        raise ValueError(f"{name}: rows of the output overlap (strides {t.stride()})")
    for u in (*apart, *same):
        if u is not None and _clash(t, u):
            if any(u is v for v in same) and u.data_ptr() == t.data_ptr() and u.stride() == t.stride() and u.dtype == t.dtype:
                continue
            raise ValueError(f"{name}: the output shares memory with another operand")
    return r


def _new(x):
    """A contiguous tensor of x's shape and type (empty_like is the quicker call, but keeps other strides)."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _written(*ts):
    """Tensors of the caller's that a kernel is about to write: autograd is told, as by any operation in place."""
    for t in ts:
        if t.requires_grad and (t.is_leaf or torch.is_grad_enabled()):
            raise ValueError("a tensor that requires a gradient cannot be written in place here")
    for t in ts:
        if not t.is_inference():             # those have no version to count
            torch.autograd.graph.increment_version(t)


def _aside(t, name, shape, device, dtype=torch.float32):
    """Address of a contiguous side operand (None: null)."""
    if t is None:
        return None
    if not (isinstance(t, torch.Tensor) and t.device == device and t.dtype == dtype and tuple(t.shape) == shape and t.is_contiguous()):
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor {shape} on {device}")
    return t.data_ptr()


def _call(name, dev, ws_bytes, args):
    """Run an entry point on `dev`, with a workspace of that many bytes if it takes one, on dev's current stream."""
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _call(name, dev, ws_bytes, args)
    if ws_bytes is not None:
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
        args = (*args, ws.data_ptr() if ws_bytes else None, ws_bytes)
    rc = getattr(_lib.load(), name)(*args, _raw_stream(dev.index))
    if rc:
        _lib.check(rc, name)


def group_norm_act(x, gamma, beta, groups, eps=1e-5, act=_lib.ACT_NONE, act_first=False, lengths=None):
    """y = act(norm(x)) of x [B, S, C], or norm(act(x)) with act_first: (y, stats [B, groups, 2] = mean and 1/sqrt(var + eps)
    for the backward pass).  act: _lib.ACT_*.  gamma, beta: fp32 [C] or None; lengths: int32 [B] or None, the frames of each
    utterance: frames past them count for nothing and are zero in y.  Reference: TCNBlock.net, mossformer2_block.py:508-531."""
    lib = _lib.load()
    xr = _rows(x, "x")
    B, S, C = x.shape
    if groups < 1 or C % groups or C < 1:
        raise ValueError(f"groups = {groups} does not divide {C} channels")
    if not 0.0 <= eps < float("inf"):
        raise ValueError("eps must be finite and not negative")
    if act not in (0, 1, 2, 3):
        raise ValueError(f"unknown activation {act}")
    dev = x.device
    side = (_aside(gamma, "gamma", (C,), dev), _aside(beta, "beta", (C,), dev), _aside(lengths, "lengths", (B,), dev, torch.int32))
    y = _new(x)
    if not (B and S):
        return y, torch.zeros((B, groups, 2), device=dev)
    stats = torch.empty((B, groups, 2), device=dev)
    t = _TYPES[x.dtype]
    _call("msf2_group_norm_act", dev, lib.msf2_group_norm_act_ws_bytes(B, S, C, groups, t),
          (*xr, *side, y.data_ptr(), S * C, C, stats.data_ptr(), B, S, C, groups, eps, act, int(act_first), t))
    return y, stats


def group_norm_act_backward(dy, x, gamma, beta, stats, groups, act=_lib.ACT_NONE, act_first=False, lengths=None):
    """(dx, dgamma, dbeta) of group_norm_act for the gradient dy of y; stats as the forward returned them.  dgamma and dbeta
    are fp32 [C], summed over utterances and frames (None where gamma or beta is)."""
    lib = _lib.load()
    xr, dyr = _rows(x, "x"), _rows(dy, "dy", x)
    B, S, C = x.shape
    if groups < 1 or C % groups or C < 1:
        raise ValueError(f"groups = {groups} does not divide {C} channels")
    if act not in (0, 1, 2, 3):
        raise ValueError(f"unknown activation {act}")
    dev = x.device
    side = (_aside(gamma, "gamma", (C,), dev), _aside(beta, "beta", (C,), dev), _aside(stats, "stats", (B, groups, 2), dev),
            _aside(lengths, "lengths", (B,), dev, torch.int32))
    if side[2] is None:
        raise ValueError("stats: expected what group_norm_act returned")
    dx = _new(x)
    new = torch.empty if B and S else torch.zeros
    dgamma = None if gamma is None else new((C,), device=dev)
    dbeta = None if beta is None else new((C,), device=dev)
    if B and S:
        t = _TYPES[x.dtype]
        _call("msf2_group_norm_act_backward", dev, lib.msf2_group_norm_act_backward_ws_bytes(B, S, C, groups, t),
              (*dyr, *xr, *side, dx.data_ptr(), S * C, C, None if dgamma is None else dgamma.data_ptr(),
               None if dbeta is None else dbeta.data_ptr(), B, S, C, groups, act, int(act_first), t))
    return dx, dgamma, dbeta


def gated_recurrence(x, gate, h0=None, lengths=None, reverse=False, last=None, save=False):
    """h_t = a_t h_{t-1} + (1 - a_t) x_t with a = sigmoid(gate), per channel of x, gate [B, S, C], from h0 (fp32 [B, C], None:
    zeros): (h, last, saved).  last: fp32 [B, C], the state after the last frame, written into `last` if given, which may be h0
    itself (a stream that keeps one state).  reverse walks from an utterance's last frame to its first.  lengths: int32 [B] or
    None, as in group_norm_act; an empty utterance hands h0 on.  saved: with save=True the states that
    gated_recurrence_backward starts from (fp32, one row in _lib.RECURRENCE_SAVE), else None."""
    lib = _lib.load()
    xr, gr = _rows(x, "x"), _rows(gate, "gate", x)
    B, S, C = x.shape
    if C < 1:
        raise ValueError("x has no channels")
    dev = x.device
    h0p, lp = _aside(h0, "h0", (B, C), dev), _aside(lengths, "lengths", (B,), dev, torch.int32)
    if last is None:
        last = torch.empty((B, C), device=dev)
        lastp = last.data_ptr()
    else:
        lastp = _aside(last, "last", (B, C), dev)
        if any(_clash(last, u) for u in (x, gate, lengths) if u is not None) or (h0 is not None and _clash(last, h0) and lastp != h0p):
            raise ValueError("last: the output shares memory with another operand")
        _written(last)                       # after all checks: a refused call leaves it as it was
    h = _new(x)
    saved = torch.empty((B, -(-S // _lib.RECURRENCE_SAVE), C), device=dev) if save else None
    if B and S:
        t = _TYPES[x.dtype]
        _call("msf2_gated_recurrence", dev, lib.msf2_gated_recurrence_ws_bytes(B, S, C, t),
              (*xr, *gr, h0p, lp, h.data_ptr(), S * C, C, lastp, saved.data_ptr() if save else None, B, S, C, int(reverse), t))
    elif h0 is None:
        last.zero_()
    elif lastp != h0p:
        last.copy_(h0)
    return h, last, saved


def gated_recurrence_backward(dh, x, gate, saved, dlast=None, lengths=None, reverse=False, out=None):
    """(dx, dgate, dh0) of gated_recurrence for the gradients dh of h and dlast (fp32 [B, C] or None) of last; saved as the
    forward returned it with save=True.  out: a pair of tensors to write dx and dgate into, for instance the two halves of the
    gradient of the projection that x and gate were cut from."""
    lib = _lib.load()
    xr, gr, dhr = _rows(x, "x"), _rows(gate, "gate", x), _rows(dh, "dh", x)
    B, S, C = x.shape
    if C < 1:
        raise ValueError("x has no channels")
    dev = x.device
    dlp, lp = _aside(dlast, "dlast", (B, C), dev), _aside(lengths, "lengths", (B,), dev, torch.int32)
    savedp = _aside(saved, "saved", (B, -(-S // _lib.RECURRENCE_SAVE), C), dev)
    if savedp is None:
        raise ValueError("saved: expected what gated_recurrence returned with save=True")
    if out is None:
        dx, dgate = _new(x), _new(x)
        dxr, dgr = (dx.data_ptr(), S * C, C), (dgate.data_ptr(), S * C, C)
    else:
        if not (isinstance(out, (tuple, list)) and len(out) == 2):
            raise ValueError("out: expected a pair of tensors")
        dx, dgate = out
        dgr = _out_rows(dgate, "dgate", x, apart=(dh, x, gate, saved, dlast, lengths))
        dxr = _out_rows(dx, "dx", x, apart=(dh, x, gate, saved, dlast, lengths, dgate))
        _written(dx, dgate)
    if not (B and S):
        return dx, dgate, torch.zeros((B, C), device=dev) if dlast is None else dlast.clone()
    dh0 = torch.empty((B, C), device=dev)
    t = _TYPES[x.dtype]
    _call("msf2_gated_recurrence_backward", dev, lib.msf2_gated_recurrence_backward_ws_bytes(B, S, C, t),
          (*dhr, *xr, *gr, savedp, dlp, lp, *dxr, *dgr, dh0.data_ptr(), B, S, C, int(reverse), t))
    return dx, dgate, dh0


def _dropout(x, p, rng, site, residual, y, given=False):
    xr = _rows(x, "x")
    B, S, C = x.shape
    dev = x.device
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p = {p} is no probability")
    if not 0 <= site < 1 << 32:
        raise ValueError("site must be in [0, 2^32)")
    if y.dtype not in _TYPES or (y.dtype != x.dtype and torch.float32 not in (x.dtype, y.dtype)):
        raise ValueError(f"no conversion from {x.dtype} to {y.dtype}")
    rr = (None, 0, 0) if residual is None else _rows(residual, "residual", y)
    rngp = _aside(rng, "rng", (2,), dev, torch.int64)
    if rngp is None:
        raise ValueError("rng: expected an int64 tensor (seed, step) on the GPU")
    if given:
        yr = _out_rows(y, "out", x, same_type=False, apart=(rng,), same=(x, residual))
        _written(y)
    else:
        yr = (y.data_ptr(), S * C, C)
    if B and S and C:
        _call("msf2_dropout", dev, None, (*xr, *rr, *yr, rngp, site, p, B, S, C, _TYPES[x.dtype], _TYPES[y.dtype]))
    return y


def dropout(x, p, rng, site=0, residual=None, out=None):
    """residual + x keep / (1 - p) (no residual: x keep / (1 - p)) of x [B, S, C]; residual is of x's type or fp32, and so is the
    result.  The mask comes from a counter-based generator and is never stored: it depends on rng = (seed, step), an int64
    tensor on the GPU, on site, which tells the dropouts of one step apart, and on an element's place, not on strides or
    types (include/msf2.h).  p counts in steps of 2^-16.  Advance rng[1] after a step's backward pass; a captured graph
    draws new masks when the program does.  out: where to write, x or residual themselves if wanted."""
    if not all(isinstance(t, torch.Tensor) for t in (x, *(t for t in (residual, out) if t is not None))):
        raise ValueError("x, residual, out: expected tensors")
    if out is not None:
        return _dropout(x, p, rng, site, residual, out, True)
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual: expected shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    return _dropout(x, p, rng, site, residual, _new(x if residual is None else residual))


def dropout_backward(dy, p, rng, site=0, dtype=None):
    """The gradient of dropout's x (of type `dtype`, None: dy's) for the gradient dy of its result: dy keep / (1 - p), with
    the forward's p, rng and site.  The residual's gradient is dy itself."""
    if not isinstance(dy, torch.Tensor):
        raise ValueError("dy: expected a tensor")
    dx = _new(dy) if dtype in (None, dy.dtype) else torch.empty(dy.shape, dtype=dtype, device=dy.device)
    return _dropout(dy, p, rng, site, None, dx)
