"""Calls of the state-space operators at the edges of what they take: layouts of parameters, infinite steps, the types' largest
values, sizes past what a launch can count, other ways of differentiating.  Oracle and tolerances: those of
tests/test_state_space_gpu.py (1e-5 of a tensor's largest value, half a step of a 16-bit result)."""
import ctypes

import pytest
import torch
import torch.nn as nn

import state_space_reference as R

F32 = 1e-5


# ---- parameters that are not dense ------------------------------------------------------------------------------------------------


def test_norm_backward_reads_a_dense_weight(monkeypatch):
    """What the launch is handed, seen on the host: C floats of the weight's own values, wherever they stood."""
    from dp_timeautodiff_amd import _native
    _native.load()
    seen = {}

    def call(name, device, *args):
        if name == "dpk_rms_norm_backward":
            address = args[8]
            seen["address"] = address
            if seen.get("read"):
                seen["weight"] = torch.frombuffer(bytearray(ctypes.string_at(address, 4 * 6)), dtype=torch.float32)

    monkeypatch.setattr(_native, "_call", call)
    r, dy, rstd = torch.ones(3, 6), torch.ones(3, 6), torch.ones(3)
    wide = torch.arange(12.0)
    seen["read"] = True
    _native.rms_norm_backward(r, None, dy, None, wide[::2], rstd, True, True)
    assert torch.equal(seen["weight"], wide[::2])
    one = torch.tensor([3.0])
    seen["read"] = False   # (of an expanded weight's own storage only the first float may be read)
    _native.rms_norm_backward(r, None, dy, None, one.expand(6), rstd, True, True)
    assert seen["address"] != one.data_ptr()


def _layouts(dense):
    """The same values: every second element of a wider tensor, a transposed one, and the tensor itself."""
    wide = torch.stack([dense, torch.full_like(dense, 7.0)], -1).flatten(-2)
    yield wide[..., ::2]
    if dense.dim() == 2:
        yield dense.t().contiguous().t()
    yield dense


@pytest.mark.gpu
def test_parameters_of_any_layout_give_the_same_results():
    from dp_timeautodiff_amd.layers import causal_conv, rms_norm, selective_scan
    g = torch.Generator().manual_seed(0)
    B, T, D, N = 3, 9, 40, 6
    rnd = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    x, res, delta, z, dy = (rnd(B, T, D) for _ in range(5))
    Bm, Cm = rnd(B, T, N), rnd(B, T, N)
    calls = [
        (lambda u, w: rms_norm(u, w, res)[0], [rnd(D)]),
        (lambda u, w: rms_norm(u, w)[0], [rnd(D)]),
        (lambda u, w, b: causal_conv(u, w, b), [rnd(D, 4), rnd(D)]),
        (lambda u, a, d, b, h: selective_scan(u, delta, a, Bm, Cm, d, z, b, state=h), [rnd(D, N), rnd(D), rnd(D), rnd(B, D, N)])]
    for k, (fn, params) in enumerate(calls):
        want = None
        for views in zip(*([p] + [v for v in _layouts(p)] for p in params)):
            u = x.clone().requires_grad_()
            leaves = [v.detach().requires_grad_() for v in views]
            assert all(v.stride() == w.stride() for v, w in zip(views, leaves))
            y = fn(u, *leaves)
            y.backward(dy)
            got = [y.detach(), u.grad] + [t.grad for t in leaves]
            want = got if want is None else want
            assert all(torch.equal(a, b) for a, b in zip(got, want)), k
    # one number for all channels
    one = torch.tensor([1.5], device="cuda", requires_grad=True)
    u = x.clone().requires_grad_()
    rms_norm(u, one.expand(D), res)[0].backward(dy)
    u64, one64 = x.cpu().double().requires_grad_(), torch.tensor([1.5], dtype=torch.float64, requires_grad=True)
    (R.rms_norm(u64, one64.expand(D), res.cpu().double())[0] * dy.cpu().double()).sum().backward()
    assert float((u.grad.cpu().double() - u64.grad).abs().max()) <= F32 * float(u64.grad.abs().max())
    # its gradient is a sum of D channels' gradients, each within F32 of the largest
    dw = rms_grad_terms(x, res, dy)
    assert float((one.grad.cpu().double() - one64.grad).abs().max()) <= F32 * D * float(dw.abs().max())


def rms_grad_terms(x, res, dy):
    w = torch.full((x.shape[-1],), 1.5, dtype=torch.float64, requires_grad=True)
    (R.rms_norm(x.cpu().double(), w, res.cpu().double())[0] * dy.cpu().double()).sum().backward()
    return w.grad


# ---- forward-mode derivatives ------------------------------------------------------------------------------------------------------


@pytest.fixture(params=[pytest.param("hip", marks=pytest.mark.gpu), "oracle"])
def dev(request, monkeypatch):
    if request.param == "hip":
        assert torch.cuda.is_available()
        from dp_timeautodiff_amd import _native
        _native.load()
        return torch.device("cuda:0")
    R.install(monkeypatch)
    return torch.device("cpu")


@pytest.mark.parametrize("record", [True, False])
def test_a_forward_mode_tangent_is_refused_and_not_dropped(dev, record):
    from torch.autograd import forward_ad
    from dp_timeautodiff_amd.layers import causal_conv, causal_conv_step, rms_norm, selective_scan, selective_scan_step
    t = lambda *s: torch.ones(*s, device=dev)  # noqa: E731
    x, w, cw, a, b = t(2, 3, 4), t(4), t(4, 2), t(4, 5), t(2, 3, 5)
    calls = [(rms_norm, [x, w]), (rms_norm, [x, w, x]), (causal_conv, [x, cw]), (causal_conv, [x, cw, w]),
             (selective_scan, [x, x, a, b, b]), (selective_scan, [x, x, a, b, b, w, x, w]),
             (causal_conv_step, [t(2, 4), t(2, 1, 4), cw, w]),
             (selective_scan_step, [t(2, 4), t(2, 4), a, t(2, 5), t(2, 5), t(2, 4, 5), w, t(2, 4), w])]
    with torch.set_grad_enabled(record), forward_ad.dual_level():
        for fn, args in calls:
            for k, arg in enumerate(args):
                dual = forward_ad.make_dual(arg, torch.ones_like(arg))
                with pytest.raises(NotImplementedError):
                    fn(*[dual if i == k else v for i, v in enumerate(args)])
        rms_norm(x, w)   # a level without a tangent is of no account


# ---- 8 bits at the ends of a type's range ------------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_finite_fp16_values_restore_as_finite():
    """65056 is 63.53 * 2^10: it is held as 64 * 2^10 = 2^16, which fp16 has no number for.  Off by at most max / 127 all the same."""
    from dp_timeautodiff_amd.activation8 import compress_activation, restore_activation
    for top in (65024.0, 65056.0, 65504.0):
        for C in (1, 5, 128, 260):
            x = torch.linspace(-1.0, 1.0, 2 * C).reshape(2, C)
            x[0, 0], x[1, C // 2] = top, -top
            x[0, C - 1] = 65024.0   # just on the border of q = 63 and 64 where the block has a larger value
            x = x.to(torch.float16)
            a = compress_activation(x.cuda())
            q, e = R.compress(x)
            assert torch.equal(a.data.cpu(), q) and torch.equal(a.exponent.cpu(), e)
            back = restore_activation(a).cpu().double()
            assert torch.equal(back, R.restore(q, e).clamp(-65504, 65504).to(torch.float16).double())
            assert bool(torch.isfinite(back).all())
            most = torch.nn.functional.pad(x.double().abs(), (0, -C % 128)).unflatten(-1, (-1, 128)).amax(-1)
            assert bool(((back - x.double()).abs() <= most.repeat_interleave(128, -1)[..., :C] / 127).all())
            assert torch.equal(restore_activation(a, torch.float32).cpu().double(), R.restore(q, e))
    # what fp16 never held goes by fp16's own rounding
    a = compress_activation(torch.tensor([[131072.0, -1.0]], device="cuda"))
    assert restore_activation(a, torch.float16)[0, 0].isinf() and torch.isfinite(restore_activation(a)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_errors_at_both_ends_of_the_scales(dev, dtype):
    """At k = 122, q is held to 63 and an element is off by at most 2^122; under the least scale by at most 2^-127."""
    from dp_timeautodiff_amd.activation8 import compress_activation, restore_activation
    big = torch.full((1, 128), torch.finfo(dtype).max, dtype=dtype)
    big[0, 1:64] = -torch.rand(63, generator=torch.Generator().manual_seed(0)).to(dtype) * torch.finfo(dtype).max
    small = torch.linspace(-2.0 ** -125, 2.0 ** -125, 128).reshape(1, 128).to(dtype)
    for x, most in ((big, 2.0 ** 122), (small, 2.0 ** -127)):
        back = restore_activation(compress_activation(x.to(dev)))
        assert back.dtype == dtype and bool(torch.isfinite(back).all())
        assert float((back.cpu().double() - x.double()).abs().max()) <= most


# ---- steps of size 0 by an infinite delta ------------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_softplus_at_the_ends_of_the_range():
    """Below -87 e^x leaves fp32's normal numbers and may come out as 0: 2^-126 of allowance there."""
    from dp_timeautodiff_amd.layers import selective_scan
    x = torch.tensor([-float("inf"), -3.4e38, -2.5e38, -1e30, -1e4, -151.0, -150.0, -149.0, -104.0, -90.0, -87.0, -20.0, 0.0, 19.999, 20.0, 20.001,
                      88.0, 1e4])
    d = x.numel()
    one = torch.ones(1, 1, 1)
    delta = x.view(1, 1, d).cuda().requires_grad_()
    _, h = selective_scan(torch.ones(1, 1, d).cuda(), delta, torch.zeros(d, 1).cuda(), one.cuda(), one.cuda(), return_state=True)
    ref = torch.logaddexp(x.double(), torch.zeros((), dtype=torch.float64))
    off = (h.detach().view(d).double().cpu() - ref).abs()
    assert bool((off <= 16 * 2.0 ** -24 * ref + 2.0 ** -126).all())
    h.sum().backward()
    assert bool(((delta.grad.view(d).double().cpu() - torch.sigmoid(x.double())).abs() <= F32 * torch.sigmoid(x.double()) + 2.0 ** -126).all())
    for bad, seen in ((float("inf"), torch.isinf), (float("nan"), torch.isnan)):
        _, h = selective_scan(one.cuda(), torch.full((1, 1, 1), bad).cuda(), torch.zeros(1, 1).cuda(), one.cuda(), one.cuda(), return_state=True)
        assert bool(seen(h).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", [(3, 20, 70, 16, "zdbsh", None), (1, 700, 40, 16, "zdsh", [611]), (2, 9, 65, 4, "zdbs", [9, 3])], ids=str)
def test_steps_masked_by_an_infinite_delta_leave_the_state(dtype, case):
    import test_state_space_gpu as G
    from dp_timeautodiff_amd.layers import selective_scan, selective_scan_step
    args, dout, dh, lengths = G.scan_inputs(case, dtype)
    args[1][:, ::3] = -float("inf")
    args[1][0, 1, 0] = -float("inf")
    l64 = G.leaf64(*args)
    o_ref, h_ref = R.selective_scan(*l64[:8], state=l64[8], lengths=lengths)
    lg = G.leaf(*args)
    out, h = selective_scan(*lg[:8], state=lg[8], lengths=None if lengths is None else lengths.cuda(), return_state=True)
    G.close(out, o_ref, "out")
    G.close(h, h_ref, "state")
    ((o_ref * dout.double()).sum() + (h_ref * dh.double()).sum()).backward()
    torch.autograd.backward((out, h), (dout.cuda(), dh.cuda()))
    for n, a, b in zip(G.NAMES, lg, l64):
        if a is not None:
            assert bool(torch.isfinite(b.grad).all()), n
            extra = 0.0
            if n == "u":   # two terms that may cancel: 1e-5 of each
                skip = (dout.double() * (1.0 if args[6] is None else torch.nn.functional.silu(args[6].double())) * args[5].double()).abs()
                extra = F32 * (2 * skip + b.grad.abs())
            G.close(a.grad, b.grad, "d" + n, extra)
    state = torch.randn(2, 5, 3, device="cuda")
    kept = state.clone()
    y = selective_scan_step(torch.ones(2, 5, device="cuda"), torch.full((2, 5), -float("inf"), device="cuda"), torch.zeros(5, 3, device="cuda"),
                            torch.ones(2, 3, device="cuda"), torch.ones(2, 3, device="cuda"), state)
    assert torch.equal(state, kept) and bool(torch.isfinite(y).all())


# ---- states kept for the backward pass ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("T,carried,groups", [(0, False, 0), (1, False, 0), (8, False, 0), (9, False, 1), (17, False, 2), (0, True, 0), (1, True, 1),
                                              (8, True, 1), (9, True, 2)])
def test_no_memory_is_held_for_groups_without_a_kept_state(monkeypatch, T, carried, groups):
    from dp_timeautodiff_amd import _native
    _native.load()
    monkeypatch.setattr(_native, "_call", lambda *a: None)
    B, D, N = 6, 10, 5
    u, bc = torch.zeros(B, T, D), torch.zeros(B, T, N)
    inp = _native.ScanInputs.checked(u, u, torch.zeros(D, N), bc, bc, None, None, None, torch.zeros(B, D, N) if carried else None, None, True)
    _, _, kept = _native.selective_scan_forward(inp, True, False)
    assert kept.numel() == (B * groups if groups else 1) * 8 * D   # N = 5 takes 8 rows


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 7, 8, 9])
def test_many_short_sequences(T):
    import test_state_space_gpu as G
    from dp_timeautodiff_amd.layers import selective_scan
    args, dout, _, _ = G.scan_inputs((130, T, 70, 6, "zdbs", None), torch.float32)
    l64, lg = G.leaf64(*args), G.leaf(*args)
    ref, _ = R.selective_scan(*l64[:8])
    (ref * dout.double()).sum().backward()
    selective_scan(*lg[:8]).backward(dout.cuda())
    for n, a, b in zip(G.NAMES[:8], lg, l64):
        extra = 0.0
        if n == "u":   # two terms that may cancel: 1e-5 of each
            skip = (dout.double() * torch.nn.functional.silu(args[6].double()) * args[5].double()).abs()
            extra = F32 * (2 * skip + b.grad.abs())
        G.close(a.grad, b.grad, "d" + n, extra)


# ---- under the engine -----------------------------------------------------------------------------------------------------------------


def _engine_net(dev, B=4, T=6, **kw):
    import test_state_space_layers as L
    net = L.make_net(dev, **kw)
    x, w = L.data(B, T)
    return net, x, w, L.reference(net, x, w), L.check


@pytest.mark.parametrize("shared", [False, True])
def test_summed_gradients_are_left_to_autograd_when_asked(dev, shared):
    """skip_autograd_param_grads=False: p.grad beside p.grad_sample, for these layers as for Linear ones."""
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    net, x, w, want, check = _engine_net(dev, shared=shared)
    gsm = GradSampleModule(net, loss_reduction="sum", skip_autograd_param_grads=False)
    (gsm(x.to(dev)) * w.to(dev)).sum().backward()
    gsm.check_complete()
    check(net, want)
    for n, p in net.named_parameters():
        total = want[n].sum(0)
        # each sample's gradient is within F32 of the largest, so their sum is within B times that
        assert p.grad is not None, n
        assert float((p.grad.cpu().double() - total).abs().max()) <= F32 * x.shape[0] * float(want[n].abs().max()), n


def test_removed_hooks_leave_all_layers_to_autograd(dev):
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    net, x, w, want, _ = _engine_net(dev)
    gsm = GradSampleModule(net)
    gsm.remove_hooks()
    (gsm(x.to(dev)) * w.to(dev)).sum().backward()
    for n, p in net.named_parameters():
        assert p.grad_sample is None and p.grad is not None, n
        assert float((p.grad.cpu().double() - want[n].sum(0)).abs().max()) <= F32 * x.shape[0] * float(want[n].abs().max()), n


def test_an_eight_bit_input_of_another_tensor_is_refused(dev):
    from dp_timeautodiff_amd.activation8 import compress_activation
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    from dp_timeautodiff_amd.layers import DPSelectiveSSM
    gsm = GradSampleModule(DPSelectiveSSM(12, 4).to(dev).train(), activation_bits=8)
    x = torch.randn(3, 5, 12, device=dev)
    own = compress_activation(x)
    bad = [compress_activation(x[:, :4]), compress_activation(x.to(torch.bfloat16)), own._replace(exponent=own.exponent[:, :3]),
           compress_activation(torch.randn(3, 5, 140, device=dev)), own.data]
    if dev.type == "cuda":
        bad.append(own._replace(data=own.data.cpu(), exponent=own.exponent.cpu()))
    for kept in bad:
        with pytest.raises(ValueError, match="8 bits"):
            gsm(x, kept=kept)
    assert gsm._layers[0].acts == []
    gsm(x, kept=own).sum().backward()
    gsm.check_complete()


def test_validator_leaves_a_frozen_rms_norm_alone():
    from dp_timeautodiff_amd.validators import ModuleValidator
    net = nn.Sequential(nn.Linear(4, 9), nn.RMSNorm(9), nn.Linear(9, 2))
    net[1].weight.requires_grad_(False)
    assert ModuleValidator.is_valid(net)
    fixed = ModuleValidator.fix(net)
    assert type(fixed[1]) is nn.RMSNorm and not fixed[1].weight.requires_grad and ModuleValidator.is_valid(fixed)


def test_validator_reports_a_norm_too_wide_to_replace():
    from dp_timeautodiff_amd.validators import ModuleValidator
    net = nn.Sequential(nn.Linear(4, 9), nn.RMSNorm(16385), nn.RMSNorm((3, 4)))
    fixed = ModuleValidator.fix(net)   # and does not fail over it
    assert type(fixed[1]) is nn.RMSNorm and len(ModuleValidator.validate(fixed)) == len(ModuleValidator.validate(net)) == 2


# ---- sizes past what a launch can count -------------------------------------------------------------------------------------------------


def test_launches_of_too_many_threads_are_refused():
    """A launch counts its threads in 32 bits.  Every call is refused before anything is launched (no GPU needed)."""
    from dp_timeautodiff_amd import _native
    lib = _native.load()
    p = ctypes.c_void_p(4096)   # never dereferenced
    norm = lambda rows, C: lib.dpk_rms_norm_forward(p, C, None, 0, p, p, None, None, None, None, rows, C, 1e-6, 0, None)  # noqa: E731
    # a row takes 32, 64, 256 or 1024 threads
    assert norm(2 ** 27, 8) == norm(2 ** 26, 200) == norm(2 ** 24, 1025) == norm(2 ** 22, 5000) == -2
    assert lib.dpk_rms_norm_backward(p, 8, None, 0, p, 8, None, 0, p, p, p, p, 8, 2 ** 24, 4, 1, 8, 1.0, 0, 0, None) == -2
    assert lib.dpk_rms_norm_backward(p, 8, None, 0, p, 8, None, 0, p, p, p, p, 8, 2 ** 20, 4, 16, 8, 1.0, 0, 0, None) == -2
    assert lib.dpk_rms_norm_backward(p, 5000, None, 0, p, 5000, None, 0, p, p, p, p, 5000, 2 ** 22, 4, 1, 5000, 1.0, 0, 0, None) == -2
    conv = lambda B, T, D: lib.dpk_causal_conv_forward(p, 24, 8, p, None, None, None, p, None, B, T, D, 4, 1, 0, None)  # noqa: E731
    assert conv(2 ** 24, 1, 8) == conv(1, 2 ** 30 + 1, 8) == conv(1, 4, 2 ** 30 + 1) == -2
    assert lib.dpk_causal_conv_backward(p, 24, 8, p, 24, 8, p, None, None, None, None, p, None, None, 0, -1, 1, 2 ** 24, 1, 8, 4, 1, 1.0, 0, 0,
                                        None) == -2
    assert lib.dpk_causal_conv_step(p, 2 ** 20, p, p, None, p, 2 ** 12, 2 ** 20, 4, 1, 0, None) == -2

    def scan(**k):
        s = _native._ScanDesc()
        for n, v in dict(dict(B=2, T=8, D=8, N=4, dtype=0, nchunk=1, chunk=8, u=4096, delta=4096, Bm=4096, Cm=4096, A_log=4096, kept=4096,
                              edge=4096, span=4096), **k).items():
            setattr(s, n, v)
        return s

    g = _native._ScanGrads()
    for n in ("dout", "du", "ddelta", "dB", "dC", "dbc"):
        setattr(g, n, 4096)
    fwd = lambda **k: lib.dpk_selective_scan_forward(ctypes.byref(scan(**k)), p, None, None)  # noqa: E731
    back = lambda **k: lib.dpk_selective_scan_backward(ctypes.byref(scan(**k)), ctypes.byref(g), None)  # noqa: E731
    assert fwd(B=2 ** 26) == back(B=2 ** 26) == fwd(B=2 ** 24, D=256) == fwd(T=2 ** 30 + 1, chunk=2 ** 30 + 8) == -2
    assert back(B=2 ** 22, D=256, N=16) == -2                                        # four workgroups of 256 threads a sequence
    assert fwd(B=2 ** 22, T=24, nchunk=16, chunk=8) == -2                            # 64 threads a chunk
    assert fwd(B=2 ** 20, T=64 * 33, nchunk=33, chunk=64, D=64, N=32) == -2          # chunks, and eight lanes a state to join them
    assert back(B=2 ** 20, T=2 ** 12, chunk=2 ** 12, D=300) == -2                    # 2^32 sums over channel blocks and more
    step = lambda **k: lib.dpk_selective_scan_step(ctypes.byref(scan(T=1, **k)), p, p, None)  # noqa: E731
    assert step(B=2 ** 20, D=2 ** 12) == step(B=2 ** 20, D=2 ** 10, N=16) == -2
    assert lib.dpk_compress_activation(p, 1, p, p, 2 ** 29 + 1, 1, 0, None) == lib.dpk_restore_activation(p, p, p, 2 ** 29 + 1, 1, 0, None) == -2
    assert lib.dpk_compress_activation(p, 2 ** 31 - 1, p, p, 1, 2 ** 31 - 1, 0, None) == -2
    out, n, st = (ctypes.c_void_p * 3)(4096, None, None), (ctypes.c_int64 * 3)(2 ** 29, 0, 0), (ctypes.c_int64 * 3)(2 ** 29, 0, 0)
    assert lib.dpk_sum_rows(p, 1, 4, 2 ** 29, out, n, st, 1.0, 0, None) == -2


@pytest.mark.parametrize("size", [2 ** 30 + 1, 2 ** 32 + 3])
def test_sizes_past_a_c_int_are_refused(monkeypatch, size):
    """(The tensors are one element seen over and over; ctypes would pass 2^32 + 3 on as 3.)"""
    from dp_timeautodiff_amd import _native
    monkeypatch.setattr(_native, "_act", lambda *a: None)
    monkeypatch.setattr(_native, "_req", lambda *a: None)
    one = torch.zeros(1)
    wide = lambda *s, dtype=torch.float32: one.to(dtype).expand(*s)  # noqa: E731
    for call in (lambda: _native._conv_args(wide(1, size, 1), one.view(1, 1), None, None, None),
                 lambda: _native._conv_args(wide(size, 1, 1), one.view(1, 1), None, None, None),
                 lambda: _native._conv_args(wide(1, 1, size), wide(size, 1), None, None, None),
                 lambda: _native.causal_conv_step(wide(size, 1), wide(size, 0, 1), one.view(1, 1), None, True),
                 lambda: _native.ScanInputs(wide(1, size, 1), wide(1, size, 1), one.view(1, 1), wide(1, size, 1), wide(1, size, 1), *[None] * 5, True),
                 lambda: _native.ScanInputs(wide(size, 1), wide(size, 1), one.view(1, 1), wide(size, 1), wide(size, 1), *[None] * 5, True, step=True),
                 lambda: _native.compress_activation(wide(size)), lambda: _native.compress_activation(wide(2, size)),
                 lambda: _native.restore_activation(wide(1, size, dtype=torch.int8), wide(1, -(-size // 128), dtype=torch.uint8), torch.float32)):
        with pytest.raises(_native.DpkError, match="along a dimension"):
            call()


# ---- rows spread over several waves, many to a workgroup ----------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,C", [(4200, 600), (4200, 1025), (4200, 2100), (2100, 4100)])
def test_wide_norms_over_many_rows(dtype, rows, C):
    """From 513 (16 bits) or 1025 features on, four or sixteen waves share a row and meet in LDS; here every workgroup of the backward
    pass goes through that at least four times."""
    import test_state_space_gpu as G
    from dp_timeautodiff_amd.layers import rms_norm
    x, res, dy, dr = G.make(rows + C, dtype, *[(rows, C)] * 4)
    w, = G.make(1, torch.float32, (C,))
    x64, r64, w64 = G.leaf64(x, res, w)
    y_ref, r_ref = R.rms_norm(x64, w64, r64)
    ((y_ref * dy.double()).sum() + (r_ref * dr.double()).sum()).backward()
    xg, rg, wg = G.leaf(x, res, w)
    y, r = rms_norm(xg, wg, rg)
    torch.autograd.backward((y, r), (dy.cuda(), dr.cuda()))
    G.close(y, y_ref, "y")
    G.close(r, r_ref, "r")
    G.close(xg.grad, x64.grad, "dx")
    G.close(rg.grad, r64.grad, "dresidual")
    G.close(wg.grad, w64.grad, "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("C", [1025, 2049, 4100])
def test_wide_norms_per_sample(C):
    """Seven rows of one sample to a workgroup."""
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    from dp_timeautodiff_amd.layers import DPRMSNorm
    B, T = 600, 7
    g = torch.Generator().manual_seed(C)
    x, dy = torch.randn(B, T, C, generator=g), torch.randn(B, T, C, generator=g)
    norm = DPRMSNorm(C).cuda().train()
    with torch.no_grad():
        norm.weight.copy_(torch.rand(C, generator=g) + 0.5)
    gsm = GradSampleModule(norm, loss_reduction="sum")
    xg = x.cuda().requires_grad_()
    gsm(xg)[0].backward(dy.cuda())
    gsm.check_complete()
    x64 = x.double().requires_grad_()
    y, _ = R.rms_norm(x64, norm.weight.detach().cpu().double())
    (y * dy.double()).sum().backward()
    want = (dy.double() * (y.detach() / norm.weight.detach().cpu().double())).sum(1)
    got = norm.weight.grad_sample.cpu().double()
    assert got.shape == want.shape and float((got - want).abs().max()) <= F32 * float(want.abs().max())
    assert float((xg.grad.cpu().double() - x64.grad).abs().max()) <= F32 * float(x64.grad.abs().max())


@pytest.mark.gpu
def test_grad_samples_on_a_side_stream():
    """overlap_grad_sample=True: Linear layers write the arena on a stream of their own, the state-space layers on the current one."""
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    net, x, w, want, check = _engine_net(torch.device("cuda:0"))
    gsm = GradSampleModule(net, loss_reduction="sum", overlap_grad_sample=True)
    for _ in range(3):
        gsm.zero_grad()
        (gsm(x.cuda()) * w.cuda()).sum().backward()
        gsm.check_complete()
        check(net, want)


# ---- parameters that no kernel, or more than one layer, would write -----------------------------------------------------------------------


def test_a_subclass_with_a_parameter_of_its_own_is_refused(dev):
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    from dp_timeautodiff_amd.layers import DPCausalConv, DPRMSNorm, DPSelectiveScan

    def more(base):
        class More(base):
            def __init__(self, *a):
                super().__init__(*a)
                self.shift = nn.Parameter(torch.zeros(4))
        return More(4)

    class Renamed(DPRMSNorm):
        pass

    for base in (DPRMSNorm, DPCausalConv, DPSelectiveScan):
        with pytest.raises(NotImplementedError):
            GradSampleModule(more(base).to(dev))
    GradSampleModule(Renamed(4).to(dev))
    GradSampleModule(DPCausalConv(4, bias=False).to(dev))


def test_a_parameter_of_two_layers_is_refused(dev):
    """(One layer called twice adds up; two layers with one parameter would each write its rows.)"""
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    from dp_timeautodiff_amd.layers import DPRMSNorm
    pair = nn.ModuleList([DPRMSNorm(4), DPRMSNorm(4)]).to(dev)
    pair[1].weight = pair[0].weight
    with pytest.raises(NotImplementedError, match="shared"):
        GradSampleModule(pair)
    mixed = nn.ModuleList([nn.LayerNorm(4), DPRMSNorm(4)]).to(dev)
    mixed[1].weight = mixed[0].weight
    with pytest.raises(NotImplementedError, match="shared"):
        GradSampleModule(mixed)


def test_a_refused_model_keeps_its_layers_to_itself(dev):
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    from dp_timeautodiff_amd.layers import DPRMSNorm
    net = nn.ModuleDict({"norm": DPRMSNorm(4), "table": nn.Embedding(5, 4, padding_idx=0)}).to(dev)
    with pytest.raises(NotImplementedError):
        GradSampleModule(net)
    x = torch.randn(3, 2, 4, device=dev)
    net["norm"](x)[0].sum().backward()
    assert net["norm"].weight.grad is not None and net["norm"]._dpk_claim is None


# ---- the same tensor twice, and nothing at all --------------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_one_tensor_as_several_operands():
    import test_state_space_gpu as G
    from dp_timeautodiff_amd.layers import rms_norm, selective_scan
    x, dy, dr, bc = G.make(3, torch.float32, (3, 7, 20), (3, 7, 20), (3, 7, 20), (3, 7, 20))
    w, a = G.make(4, torch.float32, (20,), (20, 20))
    (xg, wg), (x64, w64) = G.leaf(x, w), G.leaf64(x, w)
    y, r = rms_norm(xg, wg, xg)
    y_ref, r_ref = R.rms_norm(x64, w64, x64)
    torch.autograd.backward((y, r), (dy.cuda(), dr.cuda()))
    ((y_ref * dy.double()).sum() + (r_ref * dr.double()).sum()).backward()
    G.close(xg.grad, x64.grad, "dx")
    G.close(wg.grad, w64.grad, "dw")
    # u, delta and z are one tensor, B and C another: its gradient is the sum of theirs, each within F32 of its largest value
    xg, bg, ag = G.leaf(x, bc, a)
    parts = G.leaf64(x, x, a, bc, bc, x)
    ref = R.selective_scan(*parts[:5], None, parts[5])[0]
    out = selective_scan(xg, xg, ag, bg, bg, None, xg)
    out.backward(dy.cuda())
    (ref * dy.double()).sum().backward()
    G.close(out, ref, "out")
    for n, got, of in (("x", xg, (0, 1, 5)), ("bc", bg, (3, 4)), ("A_log", ag, (2,))):
        G.close(got.grad, sum(parts[k].grad for k in of), "d" + n, F32 * sum(float(parts[k].grad.abs().max()) for k in of))


@pytest.mark.gpu
@pytest.mark.parametrize("skip", [True, False])
def test_an_empty_batch(skip):
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    dev = torch.device("cuda:0")
    net, _, _, _, _ = _engine_net(dev)
    gsm = GradSampleModule(net, skip_autograd_param_grads=skip)
    gsm(torch.zeros(0, 5, 5, device=dev)).sum().backward()
    gsm.check_complete()
    for n, p in net.named_parameters():
        assert p.grad_sample.shape[0] == 0, n
        assert (p.grad is None) if skip else (p.grad is not None and not p.grad.any()), n
