"""Workloads of the gated linear recurrence and of the 4-bit mat-vecs, each with its plain form.

The recurrence (``wavenet_vocoder_amd.recurrence``), z = (f | v | o) along the channels:

    a = sigmoid(f)    h_t = a_t h_{t-1} + (1 - a_t) v_t    y_t = h_t sigmoid(o_t)      (without an output gate: y = h)

the state read as zero where an utterance of a packed slot begins, and handed on unchanged behind a row's length.
The mat-vec (``wavenet_vocoder_amd.engine.Q4Linear``), weights of 4 bits in groups along the inputs:

    W[n, k] = scale[n, k / g] (code[n, k] - zero[n, k / g])        y = x W^T + bias

and the two in one step: the gates z of one time step straight out of the product.

``own`` false: elementary torch operations; true: the package's calls on the same inputs."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # scoring one utterance with a layer of the 128-channel models, 24064 samples (one second at 24 kHz)
        dict(name="scan_1x24064x128_f32", op="scan", B=1, T=24064, C=128, gated=True, rows="full", dtype="f32"),
        # slots of several utterances back to back, the 512-channel geometry
        dict(name="scan_packed_8x24064x512_bf16", op="scan", B=8, T=24064, C=512, gated=True, rows="packed", dtype="bf16"),
        # a training batch of clips, 128 channels
        dict(name="train_8x7680x128_bf16", op="train", B=8, T=7680, C=128, gated=True, rows="full", dtype="bf16"),
        # a padded batch of odd sizes, one row of it empty, without an output gate
        dict(name="train_ragged_5x3001x201_f16", op="train", B=5, T=3001, C=201, gated=False, rows="lengths", dtype="f16"),
        # the longest clips and the widest geometry
        dict(name="train_8x24064x512_f32", op="train", B=8, T=24064, C=512, gated=True, rows="full", dtype="f32"),
        # one time step: the benchmark's batch, and a full one
        dict(name="step_8x128_f32", op="step", B=8, C=128, gated=True, dtype="f32"),
        dict(name="step_64x512_bf16", op="step", B=64, C=512, gated=True, dtype="bf16"),
        # a 1x1 convolution of the 512-channel geometry, one utterance
        dict(name="q4_1x512x512_f32", op="q4", B=1, K=512, N=512, group=64, dtype="f32"),
        # three taps of 512 channels and 80 of conditioning as one product, the benchmark's batch
        dict(name="q4_8x1616x512_bf16", op="q4", B=8, K=1616, N=512, group=32, dtype="bf16"),
        # a product bound by its weights, one row
        dict(name="q4_1x8192x8192_bf16", op="q4", B=1, K=8192, N=8192, group=64, dtype="bf16"),
        # the fused step of one utterance, and of a batch at the 512-channel geometry
        dict(name="cell_1x128x128_f32", op="cell", B=1, K=128, C=128, gated=True, group=32, dtype="f32"),
        dict(name="cell_48x512x512_bf16", op="cell", B=48, K=512, C=512, gated=True, group=64, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("scan", "train", "step", "q4", "cell"))
    c = dict(op=op, dtype=rng.choice(sorted(TYPES)))
    if op in ("scan", "train"):
        c.update(B=_spread(rng, 1, 16), T=_spread(rng, 1, 24064), C=_spread(rng, 1, 512), gated=rng.random() < 0.7,
                 rows=rng.choice(("full", "lengths", "packed")))
        while c["B"] * c["T"] * c["C"] > 8 * 24064 * 512:
            c["B"] -= 1
    elif op == "step":
        c.update(B=_spread(rng, 1, 64), C=_spread(rng, 1, 2048), gated=rng.random() < 0.7)
    elif op == "q4":
        c.update(B=_spread(rng, 1, 64), K=_spread(rng, 16, 8192), N=_spread(rng, 16, 8192), group=rng.choice((32, 64, 128)))
    else:
        c.update(B=_spread(rng, 1, 64), K=_spread(rng, 16, 2048), C=_spread(rng, 16, 2048), gated=rng.random() < 0.7,
                 group=rng.choice((32, 64, 128)))
    return c


# ---- inputs ---------------------------------------------------------------------------------------------------------------------
def _gates(c):
    return 3 if c["gated"] else 2


def _gate_inputs(c, lead, g, dt):
    z = torch.randn(*lead, _gates(c) * c["C"], generator=g, device="cuda")
    z[..., :c["C"]].mul_(1.5).add_(2.0)             # gates that remember some ten to some hundred steps
    return z.to(dt)


def _weights(n, k, group, g):
    """Random weights in groups: the codes, scales and zero points that asymmetric rounding gives."""
    n_g = -(-k // group)
    w = torch.randn(n, n_g * group, generator=g, device="cuda") / math.sqrt(k)
    w = w.view(n, n_g, group)
    lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
    scales = ((hi - lo) / 15).to(torch.bfloat16)
    s = scales.float()
    zeros = torch.round(-lo / s).clamp(0, 15)
    codes = (torch.round(w / s[..., None]) + zeros[..., None]).clamp(0, 15)
    return codes.view(n, n_g * group)[:, :k].to(torch.uint8).contiguous(), scales, zeros.to(torch.uint8)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[c["dtype"]]
    s = dict(c)
    B = c["B"]
    if c["op"] in ("scan", "train"):
        T, C = c["T"], c["C"]
        s["z"] = _gate_inputs(c, (B, T), g, dt)
        s["h0"] = torch.randn(B, C, generator=g, device="cuda")
        s["lengths"] = s["seg_start"] = None
        if c["rows"] == "lengths":
            n = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
            n[0] = T
            if B > 2:
                n[1], n[2] = 0, 1
            s["lengths"] = n
        elif c["rows"] == "packed":                 # utterances of some thousand steps; every other row goes on with an earlier one
            first = torch.rand(B, T, generator=g, device="cuda") < 1 / 4000
            first[::2, 0] = True
            at = torch.arange(T, device="cuda").expand(B, T)
            s["seg_start"] = torch.where(first, at, -1).cummax(1).values.to(torch.int32)
        if c["op"] == "train":
            s["dy"] = torch.randn(B, T, C, generator=g, device="cuda").to(dt)
            s["dh"] = torch.randn(B, C, generator=g, device="cuda")
            s["z"].requires_grad_()
            s["h0"].requires_grad_()
        return s
    if c["op"] in ("step", "cell"):
        s["state"] = torch.randn(B, c["C"], generator=g, device="cuda")
    if c["op"] == "step":
        s["z"] = _gate_inputs(c, (B,), g, dt)
        return s
    n = c["N"] if c["op"] == "q4" else _gates(c) * c["C"]
    s["x"] = torch.randn(B, c["K"], generator=g, device="cuda").to(dt)
    s["codes"], s["scales"], s["zeros"] = _weights(n, c["K"], c["group"], g)
    s["bias"] = torch.randn(n, generator=g, device="cuda") * 0.1
    if c["op"] == "cell":
        s["bias"][:c["C"]] += 2.0
    if own:
        from wavenet_vocoder_amd.engine import Q4Linear
        q = Q4Linear(c["K"], n, s["x"].device, group_size=c["group"], gates=1 if c["op"] == "q4" else _gates(c))
        q.set_codes(s["codes"], s["scales"], s["zeros"], s["bias"])
        s["layer"] = q
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------------------
def run(state):
    s = state
    return (_own if own else _plain)(s)


def _own(s):
    from wavenet_vocoder_amd.recurrence import gated_recurrence, gated_recurrence_step
    if s["op"] in ("scan", "train"):
        y, h = gated_recurrence(s["z"], s["h0"], output_gate=s["gated"], lengths=s["lengths"], seg_start=s["seg_start"])
        if s["op"] == "scan":
            return y, h
        dz, dh0 = torch.autograd.grad((y, h), (s["z"], s["h0"]), (s["dy"], s["dh"]))
        return y.detach(), h.detach(), dz, dh0
    if s["op"] == "step":
        return gated_recurrence_step(s["z"], s["state"], output_gate=s["gated"]), s["state"]
    if s["op"] == "q4":
        return s["layer"].step(s["x"])
    return s["layer"].recurrence_step(s["x"], s["state"]), s["state"]


@torch.no_grad()
def _plain(s):
    if s["op"] in ("scan", "train"):
        return _plain_scan(s)
    if s["op"] == "step":
        z = s["z"].float()
    else:
        w = _plain_weights(s)
        z = s["x"].float() @ w.t() + s["bias"]
        if s["op"] == "q4":
            return z.to(s["x"].dtype)
    C = s["C"]
    h = s["state"] * _sigmoid(z[:, :C]) + _sigmoid(-z[:, :C]) * z[:, C:2 * C]
    s["state"].copy_(h)
    y = h * _sigmoid(z[:, 2 * C:]) if s["gated"] else h
    return y.to(s["z" if s["op"] == "step" else "x"].dtype), s["state"]


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _plain_weights(s):
    k, g = s["K"], s["group"]
    at = torch.arange(k, device="cuda") // g
    return (s["codes"].float() - s["zeros"].float()[:, at]) * s["scales"].float()[:, at]


def _affine_scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, h_{-1} = 0, by doubling the reach of every step; overwrites its arguments."""
    d, T = 1, a.shape[1]
    while d < T:
        b[:, d:] = b[:, d:] + a[:, d:] * b[:, :-d]
        a[:, d:] = a[:, d:] * a[:, :-d]
        d *= 2
    return b


def _plain_scan(s):
    z, h0, C = s["z"], s["h0"], s["C"]
    B, T = z.shape[:2]
    f, v = z[..., :C].float(), z[..., C:2 * C].float()
    a, u = _sigmoid(f), _sigmoid(-f)
    at = torch.arange(T, device=z.device)
    live = None if s["lengths"] is None else (at < s["lengths"][:, None])[..., None]
    cut = None if s["seg_start"] is None else (s["seg_start"] == at)[..., None]
    keep = a                                        # what a step keeps of the state before it
    put = u * v
    if cut is not None:
        keep = torch.where(cut, 0.0, keep)
    if live is not None:
        keep, put = torch.where(live, keep, 1.0), torch.where(live, put, 0.0)
    put[:, 0] += keep[:, 0] * h0
    h = _affine_scan(keep.clone(), put)
    last = h[:, -1].clone()
    so = _sigmoid(z[..., 2 * C:].float()) if s["gated"] else None
    y = h * so if s["gated"] else h
    if live is not None:
        y = torch.where(live, y, 0.0)
    y = y.to(z.dtype)
    if s["op"] == "scan":
        return y, last
    dy = s["dy"].float()
    if live is not None:
        dy = torch.where(live, dy, 0.0)
    dh = dy * so if s["gated"] else dy.clone()
    dh[:, -1] += s["dh"]
    back = torch.zeros_like(keep)                   # from the end: dh_t = g_t + keep_{t+1} dh_{t+1}
    back[:, 1:] = keep[:, 1:].flip(1)
    dh = _affine_scan(back, dh.flip(1)).flip(1)
    before = torch.cat((h0[:, None], h[:, :-1]), 1)
    if cut is not None:
        before = torch.where(cut, 0.0, before)
    dz = [dh * (before - v) * a * u, dh * u]
    if s["gated"]:
        dz.append(dy * h * so * (1 - so))
    dz = torch.cat(dz, -1)
    if live is not None:
        dz = torch.where(live, dz, 0.0)
    return y, last, dz.to(z.dtype), keep[:, 0] * dh[:, 0]


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------
def work(case):
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    B = c["B"]
    if c["op"] in ("scan", "train"):
        n, G = B * c["T"] * c["C"], _gates(c)
        ends = B * c["C"] * 4
        maps = 4 * B * c["T"] if c["rows"] == "packed" else 0
        if c["op"] == "scan":
            return dict(bytes=n * (G + 1) * e + 2 * ends + maps, flops=n * (6 + 4 * (G - 2) + 4))
        return dict(bytes=n * (2 * G + 2) * e + 4 * ends + maps, flops=n * 3 * (6 + 4 * (G - 2) + 4))
    if c["op"] == "step":
        n = B * c["C"]
        return dict(bytes=n * (_gates(c) + 1) * e + 8 * n, flops=n * 14)
    k, n = c["K"], c["N"] if c["op"] == "q4" else _gates(c) * c["C"]
    weights = n * k / 2 + n * -(-k // c["group"]) * 2.5 + 4 * n
    if c["op"] == "q4":
        return dict(bytes=weights + B * (k + n) * e, flops=2.0 * B * n * k)
    return dict(bytes=weights + B * (k + c["C"]) * e + 8 * B * c["C"], flops=2.0 * B * n * k + 14 * B * c["C"])


# ---- the definition, step by step, in 64 bits -----------------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] in ("scan", "train"):
        return _exact_scan(s)
    if s["op"] in ("q4", "cell"):
        g, k = s["group"], s["K"]
        x = s["x"].double()
        z = s["bias"].double().repeat(s["B"], 1)
        for i in range(0, k, g):                    # group by group
            q = s["codes"][:, i:i + g].double() - s["zeros"][:, i // g].double()[:, None]
            z += (x[:, i:i + g] @ q.t()) * s["scales"][:, i // g].double()
        if s["op"] == "q4":
            return z
    else:
        z = s["z"].double()
    parts = z.split(s["C"], -1)
    keep = torch.sigmoid(parts[0])
    h = keep * s["state"].double() + torch.sigmoid(-parts[0]) * parts[1]
    return (h * torch.sigmoid(parts[2]) if s["gated"] else h), h


def _exact_scan(s):
    z = s["z"].detach().double().transpose(0, 1).contiguous()       # time first
    T, B, _ = z.shape
    parts = z.split(s["C"], -1)
    h = s["h0"].detach().double()
    start = h
    one = torch.ones(T, B, 1, dtype=torch.float64, device=z.device)
    live = one if s["lengths"] is None else (torch.arange(T, device=z.device)[:, None] < s["lengths"]).double()[..., None]
    cut = 0 * one if s["seg_start"] is None else (s["seg_start"].t() == torch.arange(T, device=z.device)[:, None]).double()[..., None]
    a = torch.sigmoid(parts[0])
    new = torch.sigmoid(-parts[0]) * parts[1] * live
    keep = a * (1 - cut) * live + (1 - live)
    hs = torch.empty_like(new)
    for k, b, to in zip(keep.unbind(0), new.unbind(0), hs.unbind(0)):
        h = torch.addcmul(b, k, h, out=to)
    gate = torch.sigmoid(parts[2]) if s["gated"] else one
    y = (hs * gate * live).transpose(0, 1)
    if s["op"] == "scan":
        return y, hs[-1]
    dy = s["dy"].double().transpose(0, 1) * live
    dhs = dy * gate
    r = s["dh"].double()
    for k, d in zip(reversed(keep.unbind(0)), reversed(dhs.unbind(0))):
        r = k * d.add_(r)
    before = torch.cat((start[None], hs[:-1])) * (1 - cut)
    da = dhs * (before - parts[1]) * live
    dz = [da * a * torch.sigmoid(-parts[0]), dhs * live * torch.sigmoid(-parts[0])]
    if s["gated"]:
        dz.append(dy * hs * gate * torch.sigmoid(-parts[2]))
    return y, hs[-1], torch.cat(dz, -1).transpose(0, 1), r
