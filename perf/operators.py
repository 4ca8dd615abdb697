"""Timed cases of the state-space layer's operators: RMS norm with the residual's addition and an 8-bit output, the short
causal convolution, the selective scan (training, prompts, single tokens) and 8-bit activation checkpoints.

`run` computes a case in elementary torch operations in 32 bits where `own` is false, and through
dp_timeautodiff_amd's entry points where it is true."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
BLOCK = 128


def listed():
    return [
        # one token of one sequence through a block's norm: launch latency
        {"name": "norm_token", "op": "norm", "B": 1, "T": 1, "C": 512, "dtype": "bf16", "train": False, "q8": False},
        # the denoiser's width and batch (B=4096, T=48, H=250): forward and backward of a training step
        {"name": "norm_train", "op": "norm", "B": 4096, "T": 48, "C": 250, "dtype": "fp32", "train": True, "q8": False},
        # the long-horizon model (T=256, H=512) in bf16, the following layer's input kept in 8 bits and restored
        {"name": "norm_q8", "op": "norm", "B": 1024, "T": 256, "C": 512, "dtype": "bf16", "train": False, "q8": True},
        # the VAE's batch (B=1024, T=24), twice its width of 128
        {"name": "conv_train", "op": "conv", "B": 1024, "T": 24, "D": 256, "W": 4, "dtype": "fp32", "train": True, "ragged": False},
        # long prompts of unequal lengths in one padded batch
        {"name": "conv_prompt", "op": "conv", "B": 8, "T": 4096, "D": 1024, "W": 4, "dtype": "bf16", "train": False, "ragged": True},
        # a training step of the VAE's size
        {"name": "scan_train", "op": "scan", "B": 1024, "T": 24, "D": 256, "N": 16, "dtype": "fp32", "train": True, "ragged": False},
        # a training step of the long-horizon size (T=256, twice H=512), a physical chunk of it
        {"name": "scan_train_long", "op": "scan", "B": 256, "T": 256, "D": 1024, "N": 16, "dtype": "fp32", "train": True, "ragged": False},
        # few long sequences in training: the work has to be split over time
        {"name": "scan_train_few", "op": "scan", "B": 2, "T": 4096, "D": 500, "N": 16, "dtype": "bf16", "train": True, "ragged": False},
        # one long prompt, state kept for the tokens that follow
        {"name": "scan_prompt", "op": "scan", "B": 1, "T": 8192, "D": 1024, "N": 16, "dtype": "bf16", "train": False, "ragged": False},
        # a token each of many sequences: convolution and scan, states updated in place
        {"name": "token", "op": "token", "B": 64, "D": 512, "N": 16, "W": 4, "dtype": "fp32"},
        # the dp_job batch (B=64, T=24, H=200): a small stash
        {"name": "checkpoint_small", "op": "checkpoint", "B": 64, "T": 24, "C": 200, "dtype": "fp32"},
        # the denoiser's widest Linear input (B=4096, T=48, 2H=500)
        {"name": "checkpoint", "op": "checkpoint", "B": 4096, "T": 48, "C": 500, "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "conv", "scan", "scan", "scan", "token", "checkpoint"])
    dtype = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    B = _log(rng, 1, 4096)
    if op == "norm":
        C = _log(rng, 5, 4096)
        T = _log(rng, 1, max(1, min(4096, 50_000_000 // (B * C))))
        train = rng.random() < 0.5
        return {"op": op, "B": B, "T": T, "C": C, "dtype": dtype, "train": train, "q8": not train and rng.random() < 0.5}
    if op == "conv":
        D = _log(rng, 7, 2048)
        T = _log(rng, 1, max(1, min(8192, 33_000_000 // (B * D))))
        return {"op": op, "B": B, "T": T, "D": D, "W": rng.randint(2, 4), "dtype": dtype, "train": rng.random() < 0.5, "ragged": rng.random() < 0.5}
    if op == "scan":
        D = _log(rng, 7, 2048)
        N = rng.choice([4, 8, 13, 16, 16, 16])
        T = _log(rng, 1, max(1, min(8192, 400_000_000 // (B * D * N))))
        return {"op": op, "B": B, "T": T, "D": D, "N": N, "dtype": dtype, "train": rng.random() < 0.6, "ragged": rng.random() < 0.3}
    if op == "token":
        return {"op": op, "B": _log(rng, 1, 1024), "D": _log(rng, 16, 2048), "N": rng.choice([8, 16]), "W": rng.randint(2, 4), "dtype": dtype}
    C = _log(rng, 5, 2048)
    return {"op": op, "B": B, "T": _log(rng, 1, max(1, min(4096, 90_000_000 // (B * C)))), "C": C, "dtype": dtype}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dt)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    op, B = case["op"], case["B"]
    s = {"case": dict(case)}
    if op == "norm":
        T, C = case["T"], case["C"]
        s |= {"x": randn(B, T, C), "residual": randn(B, T, C), "weight": 0.5 + rand(C)}
        if case["train"]:
            s |= {"dy": randn(B, T, C), "dr": randn(B, T, C)}
        return s
    if op == "checkpoint":
        return s | {"x": randn(B, case["T"], case["C"])}
    D = case["D"]
    if op in ("conv", "token"):
        W = case["W"]
        s |= {"conv_weight": (rand(D, W) * 2 - 1) / math.sqrt(W), "conv_bias": (rand(D) * 2 - 1) / math.sqrt(W)}
    if op in ("scan", "token"):
        N = case["N"]
        # steps between 1e-3 and 1e-1 at delta = 0, decay rates 1 .. N with a spread
        first = torch.exp(rand(D) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        s |= {"A_log": torch.log(torch.arange(1, N + 1, device="cuda", dtype=torch.float32) * (0.75 + 0.5 * rand(D, N))),
              "D": 0.5 + rand(D), "dt_bias": first + torch.log(-torch.expm1(-first))}
    if op == "token":
        return s | {"x": randn(B, D), "conv_state": randn(B, W - 1, D), "u": randn(B, D), "delta": randn(B, D) * 0.5,
                    "B": randn(B, N), "C": randn(B, N), "z": randn(B, D), "state": randn(B, D, N).float()}
    T = case["T"]
    if case["ragged"]:
        s["lengths"] = torch.randint(max(1, T // 4), T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    if op == "conv":
        s["x"] = randn(B, T, D)
    else:
        s |= {"u": randn(B, T, D), "delta": randn(B, T, D) * 0.5, "B": randn(B, T, N), "C": randn(B, T, N), "z": randn(B, T, D)}
    if case["train"]:
        s["dout"] = randn(B, T, D)
    return s


def run(s):
    op = s["case"]["op"]
    if own:
        return {"norm": _own_norm, "conv": _own_conv, "scan": _own_scan, "token": _own_token, "checkpoint": _own_checkpoint}[op](s)
    return {"norm": _plain_norm, "conv": _plain_conv, "scan": _plain_scan, "token": _plain_token, "checkpoint": _plain_checkpoint}[op](s)


# ---- the framework's operators ------------------------------------------------------------------------------------------


def _leaves(s, *names):
    return [s[n].detach().requires_grad_() for n in names]


def _own_norm(s):
    from dp_timeautodiff_amd.activation8 import restore_activation
    from dp_timeautodiff_amd.layers import rms_norm
    c = s["case"]
    if c["train"]:
        x, residual, weight = _leaves(s, "x", "residual", "weight")
        y, r = rms_norm(x, weight, residual, eps=EPS)
        dx, dw = torch.autograd.grad((y, r), (x, weight), (s["dy"], s["dr"]))
        return {"y": y.detach(), "r": r.detach(), "dx": dx, "dw": dw}
    if c["q8"]:
        y, r, a = rms_norm(s["x"], s["weight"], s["residual"], eps=EPS, quantize=True)
        return {"y": y, "r": r, "kept": restore_activation(a, torch.bfloat16)}
    y, r = rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
    return {"y": y, "r": r}


def _own_conv(s):
    from dp_timeautodiff_amd.layers import causal_conv
    if s["case"]["train"]:
        x, w, b = _leaves(s, "x", "conv_weight", "conv_bias")
        y = causal_conv(x, w, b, activation="silu", lengths=s.get("lengths"))
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dout"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    y, state = causal_conv(s["x"], s["conv_weight"], s["conv_bias"], activation="silu", lengths=s.get("lengths"), return_state=True)
    return {"y": y, "state": state}


def _own_scan(s):
    from dp_timeautodiff_amd.layers import selective_scan
    names = ("u", "delta", "A_log", "B", "C", "D", "z", "dt_bias")
    if s["case"]["train"]:
        leaves = _leaves(s, *names)
        out = selective_scan(*leaves, softplus=True, lengths=s.get("lengths"))
        grads = torch.autograd.grad(out, leaves, s["dout"])
        return {"out": out.detach(), **{"d" + n: g for n, g in zip(names, grads)}}
    out, state = selective_scan(*(s[n] for n in names), softplus=True, lengths=s.get("lengths"), return_state=True)
    return {"out": out, "state": state}


def _own_token(s):
    from dp_timeautodiff_amd.layers import causal_conv_step, selective_scan_step
    y = causal_conv_step(s["x"], s["conv_state"], s["conv_weight"], s["conv_bias"], activation="silu")
    out = selective_scan_step(s["u"], s["delta"], s["A_log"], s["B"], s["C"], s["state"], s["D"], s["z"], s["dt_bias"], softplus=True)
    return {"y": y, "conv_state": s["conv_state"], "out": out, "state": s["state"]}


def _own_checkpoint(s):
    from dp_timeautodiff_amd.activation8 import compress_activation, restore_activation
    return restore_activation(compress_activation(s["x"]), s["x"].dtype)


# ---- plain forms: elementary operations in 32 bits, rounded once at the end --------------------------------------------------


def _keep8(v):
    """The values that 8 bits hold of v: q * 2^k, per block of 128 of the last dimension the least k with max <= 127 * 2^k."""
    C = v.shape[-1]
    blocks = torch.nn.functional.pad(v, (0, -C % BLOCK)).unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(blocks.abs().amax(-1, keepdim=True))
    k = torch.where(m <= 127 / 128, e - 7, e - 6).clamp(min=-126)
    return torch.ldexp(torch.round(torch.ldexp(blocks, -k)), k).flatten(-2)[..., :C]


def _plain_norm(s):
    c, dt = s["case"], s["x"].dtype
    w = s["weight"]
    r = s["x"].float() + s["residual"].float()
    rstd = 1 / torch.sqrt((r * r).mean(-1, keepdim=True) + EPS)
    n = r * rstd
    y = n * w
    out = {"y": y.to(dt), "r": r.to(dt)}
    if c["q8"]:
        out["kept"] = _keep8(y).to(torch.bfloat16)
    if c["train"]:
        dy = s["dy"].float()
        g = dy * w
        out["dx"] = (rstd * (g - n * (g * n).mean(-1, keepdim=True)) + s["dr"].float()).to(dt)
        out["dw"] = (dy * n).sum((0, 1))
    return out


def _mask(s, B, T):
    if "lengths" not in s:
        return None
    return (torch.arange(T, device="cuda") < s["lengths"][:, None])[..., None]


def _plain_conv(s):
    c, dt = s["case"], s["x"].dtype
    B, T, D, W = c["B"], c["T"], c["D"], c["W"]
    w, x = s["conv_weight"], s["x"].float()
    mask = _mask(s, B, T)
    xp = torch.cat([x.new_zeros(B, W - 1, D), x], 1)
    p = s["conv_bias"] + sum(w[:, i] * xp[:, i:i + T] for i in range(W))
    sig = 1 / (1 + torch.exp(-p))
    y = p * sig
    out = {"y": (y if mask is None else torch.where(mask, y, 0)).to(dt)}
    if not c["train"]:
        end = s["lengths"].long() if mask is not None else torch.full((B,), T, device="cuda")
        at = end[:, None] + torch.arange(W - 1, device="cuda")
        out["state"] = xp.gather(1, at[..., None].expand(B, W - 1, D)).to(dt)
        return out
    g = s["dout"].float() * sig * (1 + p * (1 - sig))
    if mask is not None:
        g = torch.where(mask, g, 0)
    gp = torch.cat([g, g.new_zeros(B, W - 1, D)], 1)
    out["dx"] = sum(w[:, i] * gp[:, W - 1 - i:W - 1 - i + T] for i in range(W)).to(dt)
    out["dw"] = torch.stack([(g * xp[:, i:i + T]).sum((0, 1)) for i in range(W)], 1)
    out["db"] = g.sum((0, 1))
    return out


def _prefix(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1, by doubling: after the pass of stride k an entry spans 2k steps."""
    k = 1
    while k < b.shape[1]:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], 1)
        if 2 * k < b.shape[1]:
            a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _plain_scan(s):
    c, dt = s["case"], s["u"].dtype
    u, z, Bm, Cm = (s[n].float() for n in ("u", "z", "B", "C"))
    x = s["delta"].float() + s["dt_bias"]
    step = torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))
    mask = _mask(s, c["B"], c["T"])
    if mask is not None:
        step = torch.where(mask, step, 0)
    A = -torch.exp(s["A_log"])
    a = torch.exp(step[..., None] * A)
    h = _prefix(a, (step * u)[..., None] * Bm[:, :, None])
    y = (h * Cm[:, :, None]).sum(-1) + s["D"] * u
    sig = 1 / (1 + torch.exp(-z))
    out = y * z * sig
    res = {"out": (out if mask is None else torch.where(mask, out, 0)).to(dt)}
    if not c["train"]:
        res["state"] = h[:, -1].contiguous()
        return res
    dout = s["dout"].float()
    if mask is not None:
        dout = torch.where(mask, dout, 0)
    dz = dout * y * sig * (1 + z * (1 - sig))
    dy = dout * z * sig
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    dh = _prefix(after.flip(1), (dy[..., None] * Cm[:, :, None]).flip(1)).flip(1)
    del after
    dC = (dy[..., None] * h).sum(2)
    e = dh * a
    del a
    e[:, 1:] *= h[:, :-1]
    e[:, 0] = 0
    del h
    q = (dh * Bm[:, :, None]).sum(-1)
    dB = (dh * (step * u)[..., None]).sum(2)
    del dh
    dstep = q * u + (e * A).sum(-1)
    ddelta = dstep / (1 + torch.exp(-x))
    if mask is not None:
        ddelta = torch.where(mask, ddelta, 0)
    res |= {"du": (q * step + s["D"] * dy).to(dt), "ddelta": ddelta.to(dt), "dA_log": A * (e * step[..., None]).sum((0, 1)),
            "dB": dB.to(dt), "dC": dC.to(dt), "dD": (dy * u).sum((0, 1)), "dz": dz.to(dt), "ddt_bias": ddelta.sum((0, 1))}
    return res


def _plain_token(s):
    dt = s["x"].dtype
    line = torch.cat([s["conv_state"], s["x"][:, None]], 1)
    p = s["conv_bias"] + (line.float() * s["conv_weight"].t()).sum(1)
    s["conv_state"].copy_(line[:, 1:])
    u, z = s["u"].float(), s["z"].float()
    x = s["delta"].float() + s["dt_bias"]
    step = torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))
    a = torch.exp(step[..., None] * -torch.exp(s["A_log"]))
    s["state"].copy_(a * s["state"] + (step * u)[..., None] * s["B"].float()[:, None])
    y = (s["state"] * s["C"].float()[:, None]).sum(-1) + s["D"] * u
    return {"y": (p / (1 + torch.exp(-p))).to(dt), "conv_state": s["conv_state"], "out": (y * z / (1 + torch.exp(-z))).to(dt), "state": s["state"]}


def _plain_checkpoint(s):
    return _keep8(s["x"].float()).to(s["x"].dtype)


# ---- the definitions in 64 bits, step by step ---------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    d = {n: v.double() for n, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    lengths = s.get("lengths")
    return {"norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan, "token": _exact_token, "checkpoint": _exact_checkpoint}[case["op"]](case, d, lengths)


def _exact_norm(c, d, lengths):
    r = d["x"] + d["residual"]
    ms = torch.linalg.vector_norm(r, dim=-1, keepdim=True).square() / c["C"] + EPS
    out = {"y": d["weight"] * r * ms.rsqrt(), "r": r}
    if c["q8"]:
        out["kept"] = None  # which of two neighbours a computed value rounds to goes by its last bits
    if c["train"]:
        # y = w r ms^(-1/2) and d ms / d r = 2 r / C
        along = (d["dy"] * d["weight"] * r).sum(-1, keepdim=True)
        out["dx"] = d["dy"] * d["weight"] * ms.rsqrt() - r * along * ms.pow(-1.5) / c["C"] + d["dr"]
        out["dw"] = (d["dy"] * r * ms.rsqrt()).flatten(0, 1).sum(0)
    return out


def _ends(c, lengths):
    return torch.full((c["B"],), c["T"], device="cuda") if lengths is None else lengths.long()


def _exact_conv(c, d, lengths):
    T, W, x, w = c["T"], c["W"], d["x"], d["conv_weight"]
    end = _ends(c, lengths)
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    dw, db = torch.zeros_like(w), torch.zeros_like(d["conv_bias"])
    for lo in range(0, T, 512):  # pieces of the time axis, so that a long prompt needs no more memory than it has to
        hi = min(T, lo + 512)
        live = (torch.arange(lo, hi, device="cuda") < end[:, None])[..., None]
        p = d["conv_bias"].expand(c["B"], hi - lo, c["D"]).clone()
        for j in range(W):
            first = max(lo, j)  # input t - j reaches output t through tap W - 1 - j
            if first < hi:
                p[:, first - lo:] += x[:, first - j:hi - j] * w[:, W - 1 - j]
        sig = torch.sigmoid(p)
        y[:, lo:hi] = p * sig * live
        if c["train"]:
            g = d["dout"][:, lo:hi] * (sig + p * sig * (1 - sig)) * live
            db += g.sum((0, 1))
            for j in range(W):
                first = max(lo, j)
                if first < hi:
                    dx[:, first - j:hi - j] += g[:, first - lo:] * w[:, W - 1 - j]
                    dw[:, W - 1 - j] += (g[:, first - lo:] * x[:, first - j:hi - j]).sum((0, 1))
    if c["train"]:
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    state = torch.zeros(c["B"], W - 1, c["D"], device="cuda", dtype=torch.float64)
    rows = torch.arange(c["B"], device="cuda")
    for j in range(W - 1):
        at = end - (W - 1) + j
        state[:, j] = torch.where((at >= 0)[:, None], x[rows, at.clamp(min=0)], 0)
    return {"y": y, "state": state}


def _exact_scan(c, d, lengths):
    B, T, D, N = c["B"], c["T"], c["D"], c["N"]
    if T * B * D * N > 1_200_000_000 or T > 10_000:
        return None
    end = _ends(c, lengths)
    A = -d["A_log"].exp()
    h = torch.zeros(B, D, N, device="cuda", dtype=torch.float64)
    out, kept = torch.zeros_like(d["u"]), []
    for t in range(T):
        live = (t < end)[:, None].double()
        dt = torch.logaddexp(d["delta"][:, t] + d["dt_bias"], torch.zeros_like(d["dt_bias"])) * live
        if c["train"]:
            kept.append(h)
        h = torch.exp(dt[..., None] * A) * h + (dt * d["u"][:, t])[..., None] * d["B"][:, t, None]
        y = torch.matmul(h, d["C"][:, t, :, None])[..., 0] + d["D"] * d["u"][:, t]
        out[:, t] = y * d["z"][:, t] * torch.sigmoid(d["z"][:, t]) * live
    if not c["train"]:
        return {"out": out, "state": h}
    g = {n: torch.zeros_like(d[n]) for n in ("u", "delta", "A_log", "B", "C", "D", "z", "dt_bias")}
    dh = torch.zeros_like(h)
    for t in range(T - 1, -1, -1):
        live = (t < end)[:, None].double()
        u, z, pre = d["u"][:, t], d["z"][:, t], d["delta"][:, t] + d["dt_bias"]
        dt = torch.logaddexp(pre, torch.zeros_like(pre)) * live
        decay = torch.exp(dt[..., None] * A)
        before = kept.pop()
        y = torch.matmul(h, d["C"][:, t, :, None])[..., 0] + d["D"] * u
        sig, do = torch.sigmoid(z), d["dout"][:, t] * live
        dy = do * z * sig
        g["z"][:, t] = do * y * (sig + z * sig * (1 - sig))
        g["D"] += (dy * u).sum(0)
        dh = dh + dy[..., None] * d["C"][:, t, None]
        g["C"][:, t] = torch.matmul(dy[:, None], h)[:, 0]
        g["B"][:, t] = torch.matmul((dt * u)[:, None], dh)[:, 0]
        into = torch.matmul(dh, d["B"][:, t, :, None])[..., 0]
        back = dh * before * decay
        g["u"][:, t] = into * dt + d["D"] * dy
        g["delta"][:, t] = (into * u + (back * A).sum(-1)) * torch.sigmoid(pre) * live
        g["A_log"] += (back * dt[..., None]).sum(0) * A
        g["dt_bias"] += g["delta"][:, t].sum(0)
        dh, h = dh * decay, before
    return {"out": out, **{"d" + n: v for n, v in g.items()}}


def _exact_token(c, d, lengths):
    W = c["W"]
    p = d["conv_bias"] + d["x"] * d["conv_weight"][:, W - 1]
    for j in range(W - 1):
        p = p + d["conv_state"][:, j] * d["conv_weight"][:, j]
    conv_state = torch.cat([d["conv_state"][:, 1:], d["x"][:, None]], 1)
    pre = d["delta"] + d["dt_bias"]
    dt = torch.logaddexp(pre, torch.zeros_like(pre))
    h = d["state"] * torch.exp(-d["A_log"].exp() * dt[..., None]) + (dt * d["u"])[..., None] * d["B"][:, None]
    y = torch.matmul(h, d["C"][..., None])[..., 0] + d["D"] * d["u"]
    return {"y": p * torch.sigmoid(p), "conv_state": conv_state, "out": y * d["z"] * torch.sigmoid(d["z"]), "state": h}


def _exact_checkpoint(c, d, lengths):
    x = d["x"]
    out = torch.empty_like(x)
    for lo in range(0, c["C"], BLOCK):
        v = x[..., lo:lo + BLOCK]
        top = v.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -140)
        k = torch.ceil(torch.log2(top) - math.log2(127))  # corrected where the logarithm was off by its last bit
        k = torch.where(top > 127 * 2.0 ** k, k + 1, torch.where(top <= 127 * 2.0 ** (k - 1), k - 1, k)).clamp(min=-126)
        out[..., lo:lo + BLOCK] = torch.round(v / 2.0 ** k) * 2.0 ** k
    return out


def work(case):
    e = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    op, B = case["op"], case["B"]
    if op == "token":
        D, N, W = case["D"], case["N"], case["W"]
        return {"bytes": B * D * (6 * e + 2 * (W - 1) * e + 8 * N) + 2 * B * N * e + 4 * D * (N + W + 3), "flops": B * D * (2 * W + 7 * N + 20)}
    rows = B * case["T"]
    if op == "checkpoint":
        return {"bytes": 2 * rows * case["C"] * e, "flops": 4 * rows * case["C"]}
    if op == "norm":
        n = rows * case["C"]
        return {"bytes": n * (7 * e if case["train"] else 4 * e + (2 if case["q8"] else 0)), "flops": n * (14 if case["train"] else 5)}
    n = rows * case["D"]
    if op == "conv":
        return {"bytes": n * e * (4 if case["train"] else 2), "flops": n * (6 * case["W"] + 15 if case["train"] else 2 * case["W"] + 5)}
    N = case["N"]
    if case["train"]:
        return {"bytes": n * e * 8 + rows * N * e * 4 + 8 * case["D"] * (N + 2), "flops": n * (25 * N + 40)}
    return {"bytes": n * e * 4 + rows * N * e * 2 + 4 * case["D"] * N * (B + 1), "flops": n * (7 * N + 20)}
