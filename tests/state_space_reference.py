"""TEST INFRASTRUCTURE: the state-space layer's operators in plain 64-bit torch, step by step, differentiable by autograd, and
stand-ins of dp_timeautodiff_amd._native's entry points built from them (host logic on the CPU)."""
import torch
import torch.nn.functional as F

BLOCK = 128


def rms_norm(x, weight, residual=None, eps=1e-6):
    r = x if residual is None else x + residual
    return r / torch.sqrt((r * r).mean(-1, keepdim=True) + eps) * weight, r


def _live(lengths, B, T):
    end = torch.full((B,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    return end, torch.arange(T)[None, :] < end[:, None]


def causal_conv(x, weight, bias=None, silu=True, state=None, lengths=None):
    """Returns y and the state behind each sequence."""
    B, T, D = x.shape
    W = weight.shape[1]
    end, live = _live(lengths, B, T)
    x = torch.where(live[..., None], x, torch.zeros((), dtype=x.dtype))
    before = x.new_zeros(B, W - 1, D) if state is None else state
    line = torch.cat([before, x], 1)
    ys = []
    for t in range(T):
        p = sum(weight[:, i] * line[:, t + i] for i in range(W))
        if bias is not None:
            p = p + bias
        ys.append((F.silu(p) if silu else p) * live[:, t, None])
    y = torch.stack(ys, 1) if ys else x
    new = torch.stack([line[b, int(end[b]):int(end[b]) + W - 1] for b in range(B)]) if B else before
    return y, new


def selective_scan(u, delta, A_log, B, C, D=None, z=None, dt_bias=None, softplus=True, state=None, lengths=None):
    """Returns out and the final state."""
    nb, T, d = u.shape
    _, live = _live(lengths, nb, T)
    zero = torch.zeros((), dtype=u.dtype)
    u, delta, B, C = (torch.where(live[..., None], t, zero) for t in (u, delta, B, C))
    z = None if z is None else torch.where(live[..., None], z, zero)
    A = -torch.exp(A_log)
    h = u.new_zeros(nb, d, A_log.shape[1]) if state is None else state
    outs = []
    for t in range(T):
        pre = delta[:, t] if dt_bias is None else delta[:, t] + dt_bias
        dt = (torch.logaddexp(pre, torch.zeros_like(pre)) if softplus else pre) * live[:, t, None]
        h = torch.exp(dt[..., None] * A) * h + (dt * u[:, t])[..., None] * B[:, t, None]
        y = (h * C[:, t, None]).sum(-1)
        if D is not None:
            y = y + D * u[:, t]
        if z is not None:
            y = y * F.silu(z[:, t])
        outs.append(y * live[:, t, None])
    return (torch.stack(outs, 1) if outs else u), h


def compress(x):
    """(q, exponent byte) of the last dimension's blocks, in 64 bits."""
    x = x.double()
    C = x.shape[-1]
    blocks = F.pad(x, (0, -C % BLOCK)).unflatten(-1, (-1, BLOCK))
    top = blocks.abs().amax(-1)
    bad = ~torch.isfinite(blocks).all(-1)
    k = torch.full_like(top, -126)
    for e in range(-126, 123):  # the least k with top <= 127 * 2^k, by trying
        k = torch.where(top > 127.0 * 2.0 ** e, torch.full_like(k, e + 1), k)
    q = torch.where(bad[..., None], torch.zeros_like(blocks), torch.round(blocks / 2.0 ** k[..., None]))
    q = torch.where(k[..., None] == 122, q.clamp(-63, 63), q)  # 64 * 2^122 is no fp32 number
    return q.flatten(-2)[..., :C].to(torch.int8), torch.where(bad, torch.full_like(k, 255), k + 127).to(torch.uint8)


def restore(q, e):
    C = q.shape[-1]
    scale = torch.where(e == 255, torch.full(e.shape, float("nan"), dtype=torch.float64), 2.0 ** (e.double() - 127))
    return q.double() * scale.repeat_interleave(BLOCK, -1)[..., :C]


# ---- stand-ins of the ctypes wrappers (CPU tensors in, what the kernels would return out) ---------------------------------------


def _rms_norm_forward(x, residual, weight, eps, want_rstd, quantize):
    y, r = rms_norm(x.double(), weight.double(), None if residual is None else residual.double(), eps)
    rstd = 1 / torch.sqrt((r * r).mean(-1) + eps)
    q, e = compress(y) if quantize else (None, None)
    return y.to(x.dtype), None if residual is None else r.to(x.dtype), rstd.float().reshape(-1) if want_rstd else None, q, e


def _write(window, B, g, scale, accumulate):
    rows = window.base[:B, window.offset:window.offset + window.numel]
    g = (g.reshape(B, -1) * scale).to(rows.dtype)
    rows.copy_(rows + g if accumulate else g)


def _per_sample(fn, B, *grads_of):
    """fn(b) -> gradients of sample b."""
    return [torch.stack(g) for g in zip(*(fn(b) for b in range(B)))]


def _rms_norm_backward(r, residual, dy, dr, weight, rstd, want_dx, want_dw, window=None, scale=1.0, accumulate=False):
    r64, s = r.double() + (0 if residual is None else residual.double()), rstd.double().view(*r.shape[:-1], 1)
    n, g = r64 * s, dy.double() * weight.double()
    dx = s * (g - n * (g * n).mean(-1, keepdim=True)) + (0 if dr is None else dr.double())
    dw = dy.double() * n
    if window is not None:
        if r.shape[0]:
            _write(window, r.shape[0], dw.reshape(r.shape[0], -1, r.shape[-1]).sum(1), scale, accumulate)
        return (dx.to(r.dtype) if want_dx else None), None
    return (dx.to(r.dtype) if want_dx else None), dw.reshape(-1, r.shape[-1]).sum(0).float()


def _causal_conv_forward(x, weight, bias, state, lengths, silu, want_state):
    y, s = causal_conv(x.double(), weight.double(), None if bias is None else bias.double(), silu,
                       None if state is None else state.double(), lengths)
    return y.to(x.dtype), s.to(x.dtype) if want_state else None


def _differentiate(fn, tensors, seeds):
    leaves = [None if t is None else t.detach().double().requires_grad_() for t in tensors]
    with torch.enable_grad():
        outs = fn(*leaves)
        total = sum(((o * s.double()).sum() for o, s in zip(outs, seeds) if s is not None), torch.zeros((), dtype=torch.float64))
        total = total + sum((t.sum() * 0 for t in leaves if t is not None), torch.zeros((), dtype=torch.float64))
        grads = iter(torch.autograd.grad(total, [t for t in leaves if t is not None]))
    return [None if t is None else next(grads) for t in leaves]


def _causal_conv_backward(x, weight, bias, state, lengths, silu, dy, dstate_out, want_dstate, want_par, windows=None, scale=1.0,
                          accumulate=False):
    cut = lambda t, b: None if t is None else t[b:b + 1]  # noqa: E731
    rows = [_differentiate(lambda a, w, c, s: causal_conv(a, w, c, silu, s, cut(lengths, b)), (x[b:b + 1], weight, bias, cut(state, b)),
                           (dy[b:b + 1], cut(dstate_out, b))) for b in range(x.shape[0])]
    dx = torch.cat([r[0] for r in rows]).to(x.dtype) if rows else torch.empty_like(x)
    ds = torch.cat([r[3] for r in rows]).to(x.dtype) if want_dstate and state is not None else None
    if windows is None:
        return dx, ds, (sum(r[1] for r in rows).float(), None if bias is None else sum(r[2] for r in rows).float())
    if rows:
        for k, w in ((1, windows[0]), (2, windows[1])):
            if w is not None:
                _write(w, len(rows), torch.stack([r[k] for r in rows]), scale, accumulate)
    return dx, ds, None


class _ScanInputs:
    def __init__(self, u, delta, A_log, B, C, D, z, dt_bias, h0, lengths, softplus, step=False):
        self.u, self.delta, self.A_log, self.B, self.C, self.D, self.z, self.dt_bias = u, delta, A_log, B, C, D, z, dt_bias
        self.h0, self.lengths, self.softplus = h0, lengths, softplus

    checked = classmethod(lambda cls, *a: cls(*a))

    def tensors(self, rows=slice(None)):
        cut = lambda t: None if t is None else t[rows]  # noqa: E731
        return cut(self.u), cut(self.delta), self.A_log, cut(self.B), cut(self.C), self.D, cut(self.z), self.dt_bias, cut(self.h0)


def _selective_scan_forward(inp, want_kept, want_state):
    *a, h0 = [None if t is None else t.double() for t in inp.tensors()]
    out, h = selective_scan(*a, softplus=inp.softplus, state=h0, lengths=inp.lengths)
    return out.to(inp.u.dtype), h.float() if want_state else None, torch.zeros(()) if want_kept else None


def _selective_scan_backward(inp, kept, dout, dhT, want_dh0, want_par, windows=None, scale=1.0, accumulate=False):
    rows = []
    for b in range(inp.u.shape[0]):
        one = slice(b, b + 1)
        run = lambda *a: selective_scan(*a[:8], softplus=inp.softplus, state=a[8],  # noqa: E731
                                        lengths=None if inp.lengths is None else inp.lengths[one])
        rows.append(_differentiate(run, inp.tensors(one), (dout[one], None if dhT is None else dhT[one])))
    col = lambda k, like: (torch.cat([r[k] for r in rows]).to(like.dtype) if rows else torch.empty_like(like))  # noqa: E731
    du, dd, dB, dC = (col(k, t) for k, t in ((0, inp.u), (1, inp.delta), (3, inp.B), (4, inp.C)))
    dz = None if inp.z is None else col(6, inp.z)
    dh0 = col(8, inp.h0) if want_dh0 and inp.h0 is not None else None
    grads = None
    if windows is None:
        grads = tuple(None if t is None else sum(r[k] for r in rows).float() for k, t in ((2, inp.A_log), (5, inp.D), (7, inp.dt_bias)))
    elif rows:
        for k, w in zip((2, 5, 7), windows):
            if w is not None:
                _write(w, len(rows), torch.stack([r[k] for r in rows]), scale, accumulate)
    return du, dd, dB, dC, dz, dh0, grads


def _normsq_slots(P):
    return 1


def _normsq_partials(gs, B, part, slot0):
    part[:B, slot0] = (gs.base[:B, gs.offset:gs.offset + gs.numel].double() ** 2).sum(1).float()


def install(monkeypatch):
    """Patches dp_timeautodiff_amd._native with the stand-ins, those of cpu_backend among them (CPU tests only)."""
    import cpu_backend
    from dp_timeautodiff_amd import _native
    cpu_backend.install(monkeypatch)
    for name, fn in (("rms_norm_forward", _rms_norm_forward), ("rms_norm_backward", _rms_norm_backward),
                     ("causal_conv_forward", _causal_conv_forward), ("causal_conv_backward", _causal_conv_backward),
                     ("ScanInputs", _ScanInputs), ("selective_scan_forward", _selective_scan_forward),
                     ("selective_scan_backward", _selective_scan_backward), ("normsq_slots", _normsq_slots),
                     ("normsq_partials", _normsq_partials), ("compress_activation", compress),
                     ("restore_activation", lambda q, e, dtype: restore(q, e).to(dtype))):
        monkeypatch.setattr(_native, name, fn)
