"""The state-space layers under the DP engine: per-sample gradients, clipping, accumulation, shared layers, 8-bit stash, graphs.

Oracle: the same module arithmetic in float64 (tests/state_space_reference.py), one sample at a time, by autograd.  Every test runs
twice: "hip" (gpu: the kernels) and "oracle" (CPU: the same host code on stand-ins of the kernels).  Tolerance: 1e-5 of the
tensor's largest value, the framework's bar for per-sample gradients."""
import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import state_space_reference as R
from conftest import rel_err

TOL = 1e-5


@pytest.fixture(params=[pytest.param("hip", marks=pytest.mark.gpu), "oracle"])
def dev(request, monkeypatch):
    if request.param == "hip":
        assert torch.cuda.is_available()
        from dp_timeautodiff_amd import _native
        _native.load()
        return torch.device("cuda:0")
    R.install(monkeypatch)
    return torch.device("cpu")


class Net(nn.Module):
    """Two state-space blocks on a residual stream, a final norm, a head."""

    def __init__(self, d_in=5, d=12, d_out=3, state=6, shared=False):
        super().__init__()
        from dp_timeautodiff_amd.layers import DPRMSNorm, DPSelectiveSSMBlock
        self.embed = nn.Linear(d_in, d)
        self.first = DPSelectiveSSMBlock(d, state)
        self.second = self.first if shared else DPSelectiveSSMBlock(d, state)
        self.norm = DPRMSNorm(d)
        self.head = nn.Linear(d, d_out)

    def forward(self, x, lengths=None):
        h, r = self.first(self.embed(x), None, lengths)
        h, r = self.second(h, r, lengths)
        return self.head(self.norm(h, r)[0])


def ref_mixer(m, p, pre, x, lengths):
    xr, z = F.linear(x, p[pre + "in_proj.weight"]).chunk(2, -1)
    u, _ = R.causal_conv(xr, p[pre + "conv.weight"], p[pre + "conv.bias"], True, None, lengths)
    dt, B, C = torch.split(F.linear(u, p[pre + "x_proj.weight"]), [m.dt_rank, m.state_size, m.state_size], -1)
    y, _ = R.selective_scan(u, F.linear(dt, p[pre + "dt_proj.weight"]), p[pre + "scan.A_log"], B, C, p[pre + "scan.D"], z,
                            p[pre + "scan.dt_bias"], True, None, lengths)
    return F.linear(y, p[pre + "out_proj.weight"])


def ref_net(net, p, x, lengths=None):
    def block(name, x, res):
        y, r = R.rms_norm(x, p[name + ".norm.weight"], res, net.first.norm.eps)
        return ref_mixer(getattr(net, name).mixer, p, name + ".mixer.", y, lengths), r

    h, r = block("first", F.linear(x, p["embed.weight"], p["embed.bias"]), None)
    h, r = block("first" if net.second is net.first else "second", h, r)
    y, _ = R.rms_norm(h, p["norm.weight"], r, net.norm.eps)
    return F.linear(y, p["head.weight"], p["head.bias"])


def reference(net, x, w, lengths=None):
    """Per-sample gradients of sum(w * net(x)) in float64, one sample at a time."""
    rows = {n: [] for n, _ in net.named_parameters()}
    for b in range(x.shape[0]):
        p = {n: v.detach().cpu().double().requires_grad_() for n, v in net.named_parameters()}
        y = ref_net(net, p, x[b:b + 1].double(), None if lengths is None else lengths[b:b + 1])
        (y * w[b:b + 1].double()).sum().backward()
        for n in rows:
            rows[n].append(p[n].grad)
    return {n: torch.stack(v) for n, v in rows.items()}


def make_net(dev, seed=0, **kw):
    torch.manual_seed(seed)
    net = Net(**kw)
    with torch.no_grad():
        for n, p in net.named_parameters():
            if n.endswith("norm.weight"):
                p.uniform_(0.5, 1.5)
    return net.to(dev).train()


def data(B, T, d_in=5, d_out=3, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(B, T, d_in, generator=g), torch.randn(B, T, d_out, generator=g)


def check(net, want):
    for n, p in net.named_parameters():
        got = p.grad_sample
        got = torch.cat([g for g in got]) if isinstance(got, list) else got
        got = got.detach().cpu().numpy()
        assert got.shape == tuple(want[n].shape), n
        assert rel_err(got, want[n].numpy()) < TOL, n


@pytest.mark.parametrize("B,T,ragged", [(5, 9, False), (3, 1, False), (4, 20, True)])
def test_per_sample_gradients_and_the_optimizer_tail(dev, B, T, ragged):
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    from dp_timeautodiff_amd.optimizer import DPOptimizer
    from dp_timeautodiff_amd.validators import ModuleValidator
    net = make_net(dev)
    assert ModuleValidator.is_valid(net)
    x, w = data(B, T)
    lengths = torch.tensor([T, 3, 1, 11], dtype=torch.int32)[:B] if ragged else None
    if ragged:
        w = w * (torch.arange(T)[None, :, None] < lengths[:, None, None])
    want = reference(net, x, w, lengths)
    gsm = GradSampleModule(net)
    y = gsm(x.to(dev), None if lengths is None else lengths.to(dev))
    ((y * w.to(dev)).sum() / B).backward()   # loss_reduction="mean": rows are those of the sum
    gsm.check_complete()
    check(net, want)
    assert all(p.grad is None for p in net.parameters())   # the summed gradients nobody reads are not computed
    C = 0.5
    opt = DPOptimizer(torch.optim.SGD(net.parameters(), lr=0.0), noise_multiplier=0.0, max_grad_norm=C, expected_batch_size=B)
    opt.attach_grad_sample_module(gsm)
    opt.step()
    flat = torch.cat([want[n].reshape(B, -1) for n, _ in net.named_parameters()], 1)
    norms = flat.norm(dim=1)
    assert rel_err(opt.per_sample_norms.cpu().numpy(), norms.numpy()) < TOL
    clip = (C / (norms + 1e-6)).clamp(max=1.0)
    got = torch.cat([p.grad.reshape(-1).cpu() for p in net.parameters()]).numpy()
    assert rel_err(got, ((flat * clip[:, None]).sum(0) / B).numpy()) < TOL


@pytest.mark.parametrize("shared", [False, True])
def test_per_sample_gradients_of_few_long_sequences(dev, shared):
    """A sample's rows are spread over workgroups (norm, convolution) and chunks of time (scan), whose parts are joined; a layer's
    second call adds to the joined rows."""
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    T = 300 if dev.type == "cuda" else 40
    net = make_net(dev, shared=shared)
    x, w = data(2, T)
    lengths = torch.tensor([T, T - 27], dtype=torch.int32)
    w = w * (torch.arange(T)[None, :, None] < lengths[:, None, None])
    want = reference(net, x, w, lengths)
    gsm = GradSampleModule(net, loss_reduction="sum")
    (gsm(x.to(dev), lengths.to(dev)) * w.to(dev)).sum().backward()
    gsm.check_complete()
    check(net, want)


def test_privacy_engine_hands_the_stash_width_on(dev):
    from torch.utils.data import DataLoader, TensorDataset
    from dp_timeautodiff_amd.privacy_engine import PrivacyEngine
    net = make_net(dev)
    loader = DataLoader(TensorDataset(torch.randn(16, 5, 5), torch.randn(16, 5, 3)), batch_size=8)
    gsm, opt, _ = PrivacyEngine().make_private(module=net, optimizer=torch.optim.SGD(net.parameters(), lr=0.1), data_loader=loader,
                                               noise_multiplier=1.0, max_grad_norm=1.0, poisson_sampling=False, activation_bits=8)
    assert gsm.activation_bits == 8
    x, w = data(4, 5)
    (gsm(x.to(dev)) * w.to(dev)).mean().backward()
    opt.step()
    assert all(torch.isfinite(p).all() for p in net.parameters())


def test_without_the_engine_the_layers_train_as_any_other(dev):
    net = make_net(dev)
    x, w = data(4, 7)
    want = reference(net, x, w)
    (net(x.to(dev)) * w.to(dev)).sum().backward()
    for n, p in net.named_parameters():
        assert rel_err(p.grad.cpu().numpy(), want[n].sum(0).numpy()) < TOL, n


def test_a_layer_called_twice_in_a_pass_adds_up(dev):
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    net = make_net(dev, shared=True)
    x, w = data(4, 6)
    want = reference(net, x, w)
    gsm = GradSampleModule(net, loss_reduction="sum")
    for _ in range(2):  # a second step starts anew
        gsm.zero_grad()
        (gsm(x.to(dev)) * w.to(dev)).sum().backward()
        gsm.check_complete()
        check(net, want)


def test_two_passes_before_one_step_append_their_samples(dev):
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    net = make_net(dev)
    x, w = data(7, 5)
    want = reference(net, x, w)
    gsm = GradSampleModule(net, loss_reduction="sum")
    for lo, hi in ((0, 3), (3, 7)):
        (gsm(x[lo:hi].to(dev)) * w[lo:hi].to(dev)).sum().backward()
    gsm.check_complete()
    check(net, want)


def test_an_incomplete_pass_leaves_nothing_behind(dev):
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    net = make_net(dev)
    x, w = data(4, 5)
    want = reference(net, x, w)
    gsm = GradSampleModule(net, loss_reduction="sum")
    y = gsm.head(gsm.norm(gsm.embed(x.to(dev)))[0])   # a pass that does not reach the blocks
    (y * w.to(dev)).sum().backward()
    with pytest.raises(ValueError):
        gsm.check_complete()
    gsm.zero_grad()
    (gsm(x.to(dev)) * w.to(dev)).sum().backward()
    gsm.check_complete()
    check(net, want)


def test_empty_poisson_batch_and_frozen_hooks(dev):
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    net = make_net(dev)
    gsm = GradSampleModule(net)
    gsm(torch.zeros(0, 5, 5, device=dev)).sum().backward()
    gsm.check_complete()
    assert all(p.grad_sample.shape[0] == 0 for p in net.parameters())
    gsm.zero_grad()
    gsm.disable_hooks()
    x, w = data(2, 3)
    (gsm(x.to(dev)) * w.to(dev)).sum().backward()
    assert all(p.grad_sample is None and p.grad is not None for p in net.parameters())
    gsm.enable_hooks()
    gsm.eval()
    with torch.no_grad():
        gsm(x.to(dev))
    assert isinstance(gsm.to_standard_module(), Net) and net.norm._dpk_claim is None


def test_sequence_first_norm_and_data_as_its_input(dev):
    """batch_first=False: DPRMSNorm takes its samples from dimension 1; its input is data (nothing upstream needs a gradient)."""
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    from dp_timeautodiff_amd.layers import DPRMSNorm

    class One(nn.Module):
        def __init__(self):
            super().__init__()
            self.norm = DPRMSNorm(10)
            self.fc = nn.Linear(10, 2)

        def forward(self, x):
            return self.fc(self.norm(x)[0])

    net = One().to(dev).train()
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(6, 4, 10, generator=g), torch.randn(6, 4, 2, generator=g)  # [T, B, C]
    gsm = GradSampleModule(net, batch_first=False, loss_reduction="sum")
    (gsm(x.to(dev)) * w.to(dev)).sum().backward()
    gsm.check_complete()
    for b in range(4):
        p = {n: v.detach().cpu().double().requires_grad_() for n, v in net.named_parameters()}
        y = F.linear(R.rms_norm(x[:, b].double(), p["norm.weight"])[0], p["fc.weight"], p["fc.bias"])
        (y * w[:, b].double()).sum().backward()
        for n, v in net.named_parameters():
            assert rel_err(v.grad_sample[b].cpu().numpy(), p[n].grad.numpy()) < TOL, n


def test_a_single_row_has_no_samples(dev):
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    from dp_timeautodiff_amd.layers import DPRMSNorm
    gsm = GradSampleModule(DPRMSNorm(8).to(dev))
    with pytest.raises(ValueError, match="samples"):
        gsm(torch.randn(8, device=dev))


def test_validator_replaces_torch_rms_norm(dev):
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    from dp_timeautodiff_amd.layers import DPRMSNorm
    from dp_timeautodiff_amd.validators import ModuleValidator
    torch.manual_seed(0)
    net = nn.Sequential(nn.Linear(4, 9), nn.RMSNorm(9, eps=1e-4), nn.Linear(9, 2))
    with torch.no_grad():
        net[1].weight.uniform_(0.5, 2.0)
    assert not ModuleValidator.is_valid(net)
    fixed = ModuleValidator.fix(net)
    assert isinstance(fixed[1], DPRMSNorm) and ModuleValidator.is_valid(fixed)
    assert list(fixed.state_dict()) == list(net.state_dict())
    x = torch.randn(3, 5, 4)
    fixed = fixed.to(dev).train()
    gsm = GradSampleModule(fixed, loss_reduction="sum")
    y = gsm(x.to(dev))
    assert rel_err(y.detach().cpu().numpy(), net.double()(x.double()).detach().numpy()) < TOL
    y.square().sum().backward()
    gsm.check_complete()
    for b in range(3):
        net.zero_grad()
        net(x[b:b + 1].double()).square().sum().backward()
        for (n, p), q in zip(net.named_parameters(), fixed.parameters()):
            assert rel_err(q.grad_sample[b].cpu().numpy(), p.grad.numpy()) < TOL, n


def test_eight_bit_stash_contracts_the_restored_activations(dev):
    """activation_bits=8: a Linear's per-sample gradient is the contraction of its restored input; everything else is untouched.
    in_proj's stash is the norm's own 8-bit output."""
    from dp_timeautodiff_amd.activation8 import Activation8, compress_activation, restore_activation
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    x, w = data(4, 6)
    grads, stash = {}, {}
    for bits in (32, 8):
        net = make_net(dev)
        gsm = GradSampleModule(net, loss_reduction="sum", activation_bits=bits)
        y = gsm(x.to(dev))
        stash[bits] = {layer.name: list(layer.acts) for layer in gsm._layers if layer.kind == "linear"}
        (y * w.to(dev)).sum().backward()
        gsm.check_complete()
        grads[bits] = {n: p.grad_sample.cpu().clone() for n, p in net.named_parameters()}
    linear = {n for n in stash[8]}
    for name in linear:
        (full,), (kept,) = stash[32][name], stash[8][name]
        assert isinstance(kept, Activation8)
        again = compress_activation(full)
        assert torch.equal(kept.data, again.data) and torch.equal(kept.exponent, again.exponent), name
        back = restore_activation(kept).cpu().double()
        top = F.pad(full.cpu().double().abs(), (0, -full.shape[-1] % 128)).unflatten(-1, (-1, 128)).amax(-1)
        assert bool(((back - full.cpu().double()).abs() <= top.repeat_interleave(128, -1)[..., :full.shape[-1]] / 127).all())
    for n in grads[32]:
        owner, _, leaf = n.rpartition(".")
        if owner in linear and leaf == "weight":
            # G^T (A8 - A): every backprop's weight is at most max|A8 - A| = 1/127 of the block's largest activation
            assert rel_err(grads[8][n].numpy(), grads[32][n].numpy()) < 0.1, n
            assert not torch.equal(grads[8][n], grads[32][n]), n
        else:
            assert torch.equal(grads[8][n], grads[32][n]), n
    with pytest.raises(ValueError):
        GradSampleModule(make_net(dev), activation_bits=4)


def test_deepcopy_and_state_dict(dev):
    import copy
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    net = make_net(dev)
    gsm = GradSampleModule(net)
    twin = copy.deepcopy(net)
    assert twin.first.norm._dpk_claim is None and twin.first.mixer.conv._dpk_claim is None
    assert list(twin.state_dict()) == list(net.state_dict())
    assert gsm.first.mixer.scan._dpk_claim is not None


def test_constructor_refusals():
    from dp_timeautodiff_amd.layers import DPCausalConv, DPRMSNorm, DPSelectiveScan
    for make in (lambda: DPRMSNorm(0), lambda: DPRMSNorm(16385), lambda: DPCausalConv(0), lambda: DPCausalConv(4, 5),
                 lambda: DPCausalConv(4, activation="tanh"), lambda: DPSelectiveScan(4, 33), lambda: DPSelectiveScan(0),
                 lambda: DPSelectiveScan(4, dt_min=0.0), lambda: DPSelectiveScan(4, dt_min=0.2, dt_max=0.1)):
        with pytest.raises(ValueError):
            make()


def test_product_refuses_cpu_tensors():
    from dp_timeautodiff_amd import activation8, layers
    from dp_timeautodiff_amd._native import DpkError
    z = torch.zeros
    for call in (lambda: layers.rms_norm(z(2, 4), z(4)), lambda: layers.causal_conv(z(1, 2, 4), z(4, 2)),
                 lambda: layers.causal_conv_step(z(1, 4), z(1, 1, 4), z(4, 2)),
                 lambda: layers.selective_scan(z(1, 2, 4), z(1, 2, 4), z(4, 2), z(1, 2, 2), z(1, 2, 2)),
                 lambda: layers.selective_scan_step(z(1, 4), z(1, 4), z(4, 2), z(1, 2), z(1, 2), z(1, 4, 2)),
                 lambda: activation8.compress_activation(z(2, 4)),
                 lambda: activation8.restore_activation(activation8.Activation8(z(2, 4).to(torch.int8), z(2, 1).to(torch.uint8), torch.float32))):
        with pytest.raises(DpkError, match="CUDA/HIP"):
            call()


def test_c_entry_refusals():
    """Argument errors come back as codes before anything is launched (no GPU needed)."""
    import ctypes
    from dp_timeautodiff_amd import _native
    lib = _native.load()
    p = ctypes.c_void_p(4096)   # never dereferenced: every call below is refused
    ok = lambda **k: dict(dict(rows=4, C=8, eps=1e-6, dtype=0, X=p, W=p, Y=p, Q=None, E=None), **k)  # noqa: E731

    def norm(rows, C, eps, dtype, X, W, Y, Q, E):
        return lib.dpk_rms_norm_forward(X, 8, None, 0, W, Y, None, None, Q, E, rows, C, eps, dtype, None)

    assert norm(**ok(X=None)) == norm(**ok(W=None)) == norm(**ok(Y=None)) == norm(**ok(C=0)) == norm(**ok(rows=-1)) == -1
    assert norm(**ok(eps=-1.0)) == norm(**ok(eps=float("nan"))) == norm(**ok(dtype=3)) == norm(**ok(Q=p)) == norm(**ok(E=p)) == -1
    assert norm(**ok(C=16385)) == norm(**ok(rows=2 ** 31)) == -2
    assert lib.dpk_rms_norm_backward(p, 8, None, 0, p, 8, None, 0, p, p, p, p, 7, 1, 4, 1, 8, 1.0, 0, 0, None) == -1   # dw_stride < C
    assert lib.dpk_rms_norm_backward(p, 8, None, 0, p, 8, None, 0, p, p, p, p, 8, 1, 4, 0, 8, 1.0, 0, 0, None) == -1   # no part
    assert lib.dpk_rms_norm_backward(p, 8, p, 8, p, 8, None, 0, p, p, p, p, 8, 1, 4, 1, 8, 1.0, 0, 0, None) == -1   # fp32: R is the sum
    conv = lambda x=p, w=p, T=3, D=8, W=4, dt=0: lib.dpk_causal_conv_forward(x, 24, 8, w, None, None, None, p, None, 2, T, D, W, 1, dt, None)  # noqa: E731
    assert conv(x=None) == conv(w=None) == conv(T=-1) == conv(D=0) == conv(W=0) == conv(dt=9) == -1 and conv(W=5) == -2
    assert lib.dpk_causal_conv_step(p, 8, None, p, None, p, 2, 8, 4, 1, 0, None) == -1

    def scan(**k):
        s = _native._ScanDesc()
        for n, v in dict(dict(B=2, T=16, D=8, N=4, dtype=0, nchunk=1, chunk=16, u=4096, delta=4096, Bm=4096, Cm=4096, A_log=4096), **k).items():
            setattr(s, n, v)
        return s

    def fwd(out=p, **k):
        return lib.dpk_selective_scan_forward(ctypes.byref(scan(**k)), out, None, None)

    assert fwd(out=None) == fwd(u=None) == fwd(A_log=None) == fwd(D=0) == fwd(N=0) == fwd(T=-1) == fwd(dtype=5) == fwd(u_sb=-1) == -1
    assert fwd(u_st=1 << 24) == fwd(z_st=1 << 24) == fwd(B_st=1 << 24) == fwd(C_st=1 << 24) == -2   # a lane's offsets would not reach
    assert fwd(N=33) == -2 and fwd(nchunk=0) == fwd(chunk=12) == fwd(chunk=8) == fwd(nchunk=2) == -1   # chunks that miss rows, no scratch
    g = _native._ScanGrads()
    assert lib.dpk_selective_scan_backward(ctypes.byref(scan()), ctypes.byref(g), None) == -1
    assert lib.dpk_selective_scan_backward(ctypes.byref(scan()), None, None) == -1 and lib.dpk_selective_scan_forward(None, p, None, None) == -1
    assert lib.dpk_selective_scan_step(ctypes.byref(scan()), p, p, None) == -1   # T is not 1
    assert lib.dpk_compress_activation(None, 8, p, p, 4, 8, 0, None) == lib.dpk_compress_activation(p, 8, p, p, 4, 0, 0, None) == -1
    assert lib.dpk_restore_activation(p, p, p, 4, 8, 7, None) == -1
    out, n, st = (ctypes.c_void_p * 3)(4096, None, None), (ctypes.c_int64 * 3)(8, 0, 0), (ctypes.c_int64 * 3)(8, 0, 0)
    assert lib.dpk_sum_rows(p, 1, 4, 7, out, n, st, 1.0, 0, None) == lib.dpk_sum_rows(p, 1, 4, 8, out, None, st, 1.0, 0, None) == -1
    n[1] = 3   # columns without a destination
    assert lib.dpk_sum_rows(p, 1, 4, 16, out, n, st, 1.0, 0, None) == -1
    # and what is empty is done
    assert norm(**ok(rows=0)) == 0 and lib.dpk_compress_activation(None, 8, None, None, 0, 8, 0, None) == 0 and fwd(B=0) == 0


def test_chunk_rule_covers_the_sequence():
    import ctypes
    from dp_timeautodiff_amd import _native
    lib = _native.load()
    g = lib.dpk_selective_scan_group()
    for B in (1, 2, 7, 64, 5000):
        for T in (0, 1, 8, 63, 64, 65, 1000, 8192, 100_003):
            for D in (1, 64, 500, 4096):
                for back in (0, 1):
                    c = ctypes.c_int(-1)
                    n = lib.dpk_selective_scan_chunks(B, T, D, back, ctypes.byref(c))
                    assert n >= 1 and c.value % g == 0 and n * c.value >= T and (n - 1) * c.value < max(T, 1)
                s = lib.dpk_causal_conv_segments(B, T, D)
                assert 1 <= s <= max(T, 1)
    assert lib.dpk_rms_norm_split(1, 1) == 1 and lib.dpk_rms_norm_split(0, 5) == 1
    assert 1 <= lib.dpk_rms_norm_split(3, 1000) <= 1000


@pytest.mark.gpu
def test_whole_step_replays_from_a_graph():
    """GraphedDPStep over the blocks: replays equal eager steps bit for bit, with eager work between them."""
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    from dp_timeautodiff_amd.graphed import GraphedDPStep
    from dp_timeautodiff_amd.optimizer import DPOptimizer
    dev = torch.device("cuda:0")

    def build():
        net = make_net(dev)
        gsm = GradSampleModule(net, activation_bits=8)
        opt = DPOptimizer(torch.optim.SGD(net.parameters(), lr=0.1), noise_multiplier=0.0, max_grad_norm=0.5, expected_batch_size=6)
        opt.attach_grad_sample_module(gsm)
        return net, gsm, opt

    x, w = (t.to(dev) for t in data(6, 11))
    net, gsm, opt = build()
    step = GraphedDPStep(gsm, opt, lambda: (gsm(x) * w).sum() / 6, warmup=2)
    step.capture()
    eager_net, eager, eopt = build()
    for _ in range(2):
        eopt.zero_grad()
        ((eager(x) * w).sum() / 6).backward()
        eopt.step()
    for k in range(4):
        nx, nw = (t.to(dev) for t in data(6, 11, seed=10 + k))
        x.copy_(nx)
        w.copy_(nw)
        eopt.zero_grad()
        ((eager(x) * w).sum() / 6).backward()
        eopt.step()
        torch.cuda.synchronize()
        step()
        torch.cuda.synchronize()
        for (n, a), b in zip(net.named_parameters(), eager_net.parameters()):
            assert torch.equal(a, b), (k, n)


@pytest.mark.gpu
def test_tokens_one_by_one_match_the_prompt():
    from dp_timeautodiff_amd.layers import DPSelectiveSSM, DPSelectiveSSMBlock
    torch.manual_seed(0)
    m = DPSelectiveSSM(20, 8).cuda().eval()
    block = DPSelectiveSSMBlock(20, 8).cuda().eval()
    x = torch.randn(3, 10, 20, device="cuda")
    with torch.no_grad():
        whole, end = m(x, return_state=True)
        head, state = m(x[:, :4], return_state=True)
        got = [head]
        for t in range(4, 10):
            got.append(m.step(x[:, t], state)[:, None])
        # the projections run as other library products for one token: each of three errs by a few 2^-24 of its terms
        assert rel_err(torch.cat(got, 1).cpu().numpy(), whole.cpu().numpy()) < TOL
        assert rel_err(state.scan.cpu().numpy(), end.scan.cpu().numpy()) < TOL and rel_err(state.conv.cpu().numpy(), end.conv.cpu().numpy()) < TOL
        out, res = block(x)
        st = block.mixer.initial_state(3)
        for t in range(10):
            o, r = block.step(x[:, t], st)
            assert rel_err(o.cpu().numpy(), out[:, t].cpu().numpy()) < 10 * TOL and torch.equal(r, res[:, t])
        # ragged prompts, then tokens
        lengths = torch.tensor([10, 4, 7], dtype=torch.int32, device="cuda")
        _, ragged = m(x, lengths=lengths, return_state=True)
        for b, n in enumerate((10, 4, 7)):
            _, one = m(x[b:b + 1, :n], return_state=True)
            assert rel_err(ragged.scan[b:b + 1].cpu().numpy(), one.scan.cpu().numpy()) < TOL
            assert rel_err(ragged.conv[b:b + 1].cpu().numpy(), one.conv.cpu().numpy()) < TOL


@pytest.mark.gpu
def test_eight_bit_stash_holds_a_quarter():
    from dp_timeautodiff_amd.grad_sample import GradSampleModule
    held = {}
    for bits in (32, 8):
        torch.manual_seed(0)
        net = nn.Sequential(nn.Linear(8, 1024), nn.Linear(1024, 4)).cuda().train()  # nothing but the stash holds the wide tensor
        gsm = GradSampleModule(net, activation_bits=bits)
        x = torch.randn(64, 128, 8, device="cuda")
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = gsm(x)
        held[bits] = torch.cuda.memory_allocated() - before
        y.sum().backward()
    wide = 64 * 128 * 1024
    assert held[32] - held[8] > 2.8 * wide   # 4 bytes against 1 + 1/128
    assert math.isfinite(float(net[1].weight.grad_sample.sum()))
