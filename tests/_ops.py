"""Plain 64-bit forms of the gated recurrence and of the 4-bit products, and the error bounds that the tests hold the kernels to.

Bounds, M = max(|v|, |h0|), S = max|dh|, u = 1 - sigmoid(f), eps = 2^-24 (half a step of float32):
  * a gate is off by at most delta = (1.5 |f| + 8) eps of itself, next to 0 and next to 1: the exponent f log2(e) is rounded (|f| eps at
    most, 1.5 with the change of base), exp2 and the reciprocal are within an ulp, and three more operations follow;
  * h is a convex combination of the v and h0, so |h| <= M.  A step a h + u v rounds twice (2 eps M) and carries delta of a h and of u v, of
    which an older share shrinks by 1 - u per step: at most N = 1 / u_min or T of them live at a time, 2 eps M N for the roundings and
    2 delta M for the gates, whose shares u v add up to M and whose shares a h are held as 1 - U over stretches.  The joins of stretches,
    quads, blocks, chunks, groups and sections round a state no more than 40 times on its way, a few eps of M each; where N < 8, next to
    nothing of it is left behind the first of them, and else 40 < 10 N.  So |h - exact| <= k M with k = 2 delta + 12 eps N + 12 eps;
  * dh_t = s, what goes back is a s: the same recursion with S in place of M, |dh - exact| <= k S;
  * df = dh (h_{t-1} - v) sigmoid(f) u: k S 2 M + S k M + S 2 M (2 delta + 4 eps), times sigmoid(f) u <= 1/4: within k S M;
    dv = dh u: (k + delta + eps) S <= 2 k S;  do = dy h sigmoid(o)(1 - sigmoid(o)): (k M + M (2 delta + 4 eps)) |dy| / 4 <= k M |dy|.
  * the result's own type rounds by finfo.eps / 2 of the value (half a step of the smallest number near zero)."""
import numpy as np
import torch

EPS = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def oracle_scan(z, h0=None, output_gate=True, lengths=None, seg_start=None, dy=None, dh_last=None):
    """float64 on the CPU, step by step.  -> dict(y, h_last, dz, dh0, h, dh) (gradients where dy is given)."""
    z = z.detach().double().cpu()
    B, T, n = z.shape
    C = n // (3 if output_gate else 2)
    live = torch.ones(B, T, dtype=torch.bool)
    if lengths is not None:
        live = torch.arange(T) < lengths.cpu().long()[:, None]
    begins = torch.zeros(B, T, dtype=torch.bool)
    if seg_start is not None:
        begins = seg_start.cpu().long() == torch.arange(T)
    begins &= live
    z = torch.where(live[..., None], z, torch.zeros(()).double())
    f, v = z[..., :C], z[..., C:2 * C]
    a, u = torch.sigmoid(f), torch.sigmoid(-f)
    so = torch.sigmoid(z[..., 2 * C:]) if output_gate else torch.ones(B, T, C).double()
    h = torch.zeros(B, C).double() if h0 is None else h0.detach().double().cpu()
    hs, before = [], []
    for t in range(T):
        p = torch.where(begins[:, t, None], torch.zeros(()).double(), h)
        before.append(p)
        h = torch.where(live[:, t, None], a[:, t] * p + u[:, t] * v[:, t], h)
        hs.append(h)
    hs, before = torch.stack(hs, 1), torch.stack(before, 1)
    out = dict(y=torch.where(live[..., None], hs * so, torch.zeros(()).double()), h_last=h, h=hs)
    if dy is None and dh_last is None:
        return out
    dy = torch.zeros(B, T, C).double() if dy is None else torch.where(live[..., None], dy.double().cpu(), torch.zeros(()).double())
    r = torch.zeros(B, C).double() if dh_last is None else dh_last.double().cpu()
    dhs = [None] * T
    for t in reversed(range(T)):
        d = dy[:, t] * so[:, t] + r
        dhs[t] = torch.where(live[:, t, None], d, torch.zeros(()).double())
        d = torch.where(begins[:, t, None], torch.zeros(()).double(), a[:, t] * d)
        r = torch.where(live[:, t, None], d, r)
    dh = torch.stack(dhs, 1)
    dz = [dh * (before - v) * a * u, dh * u]
    if output_gate:
        dz.append(torch.where(live[..., None], dy * hs * so * torch.sigmoid(-z[..., 2 * C:]), torch.zeros(()).double()))
    dz = torch.where(live[..., None], torch.cat(dz, -1), torch.zeros(()).double())
    out.update(dz=dz, dh0=r, dh=dh)
    return out


def scan_bounds(z, want, h0=None, output_gate=True, lengths=None, dy=None, dh_last=None):
    """k and the scales M, S, |dy| of the module's text, from the inputs and the exact result."""
    z = z.detach().double().cpu()
    T, C = z.shape[1], z.shape[2] // (3 if output_gate else 2)
    if lengths is not None:
        z = torch.where((torch.arange(T) < lengths.cpu().long()[:, None])[..., None], z, torch.zeros(()).double())
    f, v, o = z[..., :C], z[..., C:2 * C], z[..., 2 * C:]
    top = max(float(f.abs().max()), float(o.abs().max()) if output_gate else 0.0)
    delta = (1.5 * top + 8) * EPS
    k = 2 * delta + 12 * EPS * min(T, 1 / float(torch.sigmoid(-f).min())) + 12 * EPS
    M = max(float(v.abs().max()), 0.0 if h0 is None else float(h0.abs().max()))
    S = 0.0
    if "dh" in want:
        S = max(float(want["dh"].abs().max()), 0.0 if dh_last is None else float(dh_last.abs().max()))
    D = 0.0 if dy is None else float(dy.double().abs().max())
    return k, M, S, D


def near(got, want, bound, what=""):
    """|got - want| <= bound + the rounding to got's own type."""
    info = torch.finfo(got.dtype)
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()) == bool(torch.isfinite(want).all()), f"{what}: not finite"
    allowed = bound + info.eps / 2 * (want.abs() + bound) + info.smallest_normal * info.eps / 2
    over = (got - want).abs() / allowed
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times its bound (error {float((got - want).abs().max()):.3g}, bound {bound:.3g})"


def check_scan(got, want, z, h0=None, output_gate=True, lengths=None, dy=None, dh_last=None):
    """got: dict with y, h_last and, for gradients, dz, dh0."""
    k, M, S, D = scan_bounds(z, want, h0, output_gate, lengths, dy, dh_last)
    near(got["y"], want["y"], 2 * k * M, "y")       # the output gate multiplies once more: delta + eps
    near(got["h_last"], want["h_last"], k * M, "h_last")
    if "dz" in got:
        C = want["h"].shape[-1]
        near(got["dz"][..., :C], want["dz"][..., :C], 2 * k * S * M, "df")
        near(got["dz"][..., C:2 * C], want["dz"][..., C:2 * C], 2 * k * S, "dv")
        if output_gate:
            near(got["dz"][..., 2 * C:], want["dz"][..., 2 * C:], k * M * D, "do")
    if got.get("dh0") is not None:
        near(got["dh0"], want["dh0"], k * S, "dh0")


def q4_weight(codes, scales, zeros, group):
    at = torch.arange(codes.shape[1]) // group
    zp = torch.full_like(scales.double().cpu(), 8.0) if zeros is None else zeros.double().cpu()
    return scales.double().cpu()[:, at] * (codes.double().cpu() - zp[:, at])


def q4_bound(x, codes, scales, zeros, group, bias):
    """Of the products' sums in float32, per output: the codes enter with an offset of up to 16 (24 with the zero point's own 16 + 15
    against it), sums of 32 inputs are joined one after the other, then the groups: at most 64 + K / 32 roundings of a running sum of
    the magnitudes, and the bias."""
    K = codes.shape[1]
    at = torch.arange(K) // group
    s = scales.double().cpu().abs()[:, at]
    mass = x.double().cpu().abs() @ (s * 62).t()
    return (64 + K / 32) * EPS * mass + 2 * EPS * (0 if bias is None else bias.double().cpu().abs())


def random_q4(n, k, group, seed, zeros=True):
    g = torch.Generator().manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = (torch.rand(n, groups, generator=g) * 0.1 + 0.01).to(torch.bfloat16)
    zp = torch.randint(0, 16, (n, groups), generator=g, dtype=torch.uint8) if zeros else None
    return codes, scales, zp


# ---- bounds by what is left of each input ---------------------------------------------------------------------------------------
# The bounds above go by the largest v, h0 and dh of the whole call.  These go by m_t = sigmoid(f) m_{t-1} + sigmoid(-f) |v|, m_{-1} = |h0|: what
# the inputs still weigh at step t, so that a state that a gate forgot, or a spike long ago, does not excuse an error now.
# One step: sigmoid(-|f|) is off by delta = (1.5 |f| + 8) eps of itself (as above), 1 - sigmoid(-|f|) by no more than that and a rounding, two sums
# follow, and below 2^-126 a gate may read as 0: within (delta + 4 eps) m + 2^-126 (|h| + |v|).
TINY = 2.0 ** -126


def gate_ends(dtype):
    """f, h, v: every combination of gates that remember, forget and do neither with states and inputs of all sizes."""
    big = min(float(torch.finfo(dtype).max) * 0.9, 3e38)
    f = torch.tensor([-float("inf"), -200.0, -88.0, -40.0, -20.0, -16.0, -12.0, -10.0, -3.0, 0.0, 3.0, 9.0, 20.0, 88.0, 200.0, float("inf")])
    h = torch.tensor([0.0, 1e-3, -1.0, 1000.0, -1e6, 1e8, 3e38, -3e38])
    v = torch.tensor([0.0, 1.2345, -1.0, 1e-3, 6e4, big, -big])
    f, h, v = (t.reshape(-1) for t in torch.meshgrid(f, h, v, indexing="ij"))
    return f.to(dtype), h, v.to(dtype)


def check_blend(got, f, h, v):
    """One step's state against sigmoid(f) h + sigmoid(-f) v in 64 bits; at the infinite gates exactly h and v."""
    f, h, v, got = f.double(), h.double(), v.double(), got.double().cpu()
    keep, new = torch.sigmoid(f), torch.sigmoid(-f)
    want = torch.where(f == float("inf"), h, torch.where(f == -float("inf"), v, keep * h + new * v))
    bound = ((1.5 * f.abs().clamp(max=200) + 8) + 4) * EPS * (keep * h.abs() + new * v.abs()) + TINY * (h.abs() + v.abs())
    bound = torch.where(f.isinf(), 0.0, bound)
    over = (got - want).abs() > bound
    assert not (over | got.isnan()).any(), [(float(f[i]), float(h[i]), float(v[i]), float(got[i]), float(want[i])) for i in (over | got.isnan()).nonzero()[:5, 0]]


# A whole sequence: h_t is a sum of the v_s (and h0), each times a product of gates, and every operation of the kernels but 1 - U (below) adds or
# multiplies such terms, so that the error of a term is its own relative one: delta_l + 3 eps for each gate on its way (an operation for the
# gate, one for the sum), and the joins of stretches, of a wave's rows, a chunk's waves, a group's chunks (15 at most), a section's groups
# (15) and a state's start: 64 eps in all (a section more is 32768 steps more, whose own 3 eps each pay for it).  The product P of a
# stretch's gates may be taken as 1 - U with U = sum of u_l times the product before it, U <= 1/2: off by eps + U times U's relative error,
# no more than delta + eps a step.  So with m_t as above
#     d_t = a_t (d_{t-1} + (delta_t + 3 eps) m_{t-1}) + u_t |v_t| (delta_t + 3 eps),    |h_t - exact| <= d_t + 64 eps m_t
# and the same from the end for dh.  The products behind them: y = h sigmoid(o), dv = dh u, df = dh (h_{t-1} - v) a u, do = dy h so (1 - so), add
# their gates' deltas and an eps an operation (of t h - t v, t = a u, by the magnitudes).  1.01 for what is quadratic, TINY M for gates that
# read as 0.
#
# Long sequences of gates that remember (`long`) need less than delta a step.  A stretch keeps P = 1 - U of the state: off by eps of itself for
# the subtraction and, U being a sum of its 8 u with at most 16 roundings each, by U (delta + 16 eps); a block of 128 steps, which takes its
# P from 1 - U again, multiplies 16 such P by 15 products: within 31 eps, and U (delta + 30 eps) with the 14 roundings of its sums.  That is
# eps / 4 a step and u (delta + 30 eps); the joins of chunks, groups and sections behind it are fewer than one in 128 steps.  P >= 1/2 there:
# twice that, relative to P, so a step loses no more than 2 u (delta + 30 eps) + eps / 2, or delta + 3 eps as above.  The constant is 128 eps:
# within its own stretch a state has gone through up to 8 steps of a h + u v, 5 eps each.
def local_scan(z, h0=None, output_gate=True, lengths=None, seg_start=None, dy=None, dh_last=None, long=False):
    """(exact results, their bounds), float64 on the CPU step by step: dicts of y, h_last and, where dy is given, dz and dh0."""
    FIXED = (128 if long else 64) * EPS
    z = z.detach().double().cpu().numpy()
    B, T, n = z.shape
    C = n // (3 if output_gate else 2)
    n_live = np.full(B, T) if lengths is None else lengths.cpu().long().clamp(0, T).numpy()
    live = np.arange(T) < n_live[:, None]
    begins = np.zeros((B, T), bool) if seg_start is None else seg_start.cpu().long().numpy() == np.arange(T)
    begins &= live
    z = np.where(live[..., None], z, 0.0)
    f, v = z[..., :C], z[..., C:2 * C]
    delta = lambda x: (1.5 * np.abs(x) + 8) * EPS  # noqa: E731
    sig = lambda x: 1 / (1 + np.exp(np.minimum(-x, 700)))  # noqa: E731
    a, u = sig(f), sig(-f)
    K = delta(f) + 3 * EPS
    h = np.zeros((B, C)) if h0 is None else h0.detach().double().cpu().numpy().copy()
    M = max(np.abs(v).max(), np.abs(h).max())
    keep = np.where(live[..., None], np.where(begins[..., None], 0.0, a), 1.0)
    new, own = np.where(live[..., None], u * v, 0.0), np.where(live[..., None], K, 0.0)
    loss = np.where(live[..., None], np.minimum(K, 2 * u * (delta(f) + 30 * EPS) + EPS / 2), 0.0) if long else own
    hs, ms, ds = np.empty((T + 1, B, C)), np.empty((T + 1, B, C)), np.empty((T + 1, B, C))
    hs[0], ms[0], ds[0] = h, np.abs(h), 0
    for t in range(T):
        k, l, w, o = keep[:, t], loss[:, t], new[:, t], own[:, t]
        hs[t + 1] = k * hs[t] + w
        ms[t + 1] = k * ms[t] + np.abs(w)
        ds[t + 1] = k * (ds[t] + l * ms[t]) + np.abs(w) * o
    hs, ms, eh = (x.transpose(1, 0, 2) for x in (hs, ms, 1.01 * (ds + FIXED * ms) + 8 * TINY * M))
    o = z[..., 2 * C:] if output_gate else None
    so, do = (sig(o), delta(o)) if output_gate else (np.ones((B, T, C)), np.zeros((B, T, C)))
    L = live[..., None]
    want = dict(y=np.where(L, hs[:, 1:] * so, 0), h_last=hs[:, -1])
    bound = dict(y=np.where(L, so * (eh[:, 1:] + (do + 2 * EPS) * ms[:, 1:]), 0), h_last=eh[:, -1])
    if dy is not None:
        dy = np.where(L, dy.double().cpu().numpy(), 0)
        r = np.zeros((B, C)) if dh_last is None else dh_last.double().cpu().numpy()
        mr, dr = np.abs(r), np.zeros((B, C))
        S = max(np.abs(dy).max(), mr.max())
        g, dh, mb, db = dy * so, np.empty((B, T, C)), np.empty((B, T, C)), np.empty((B, T, C))
        for t in reversed(range(T)):
            k, l, gt = keep[:, t], loss[:, t], g[:, t]
            dh[:, t] = gt + r
            mb[:, t] = np.abs(gt) + mr
            db[:, t] = (do[:, t] + 2 * EPS) * np.abs(gt) + dr
            r, mr, dr = k * dh[:, t], k * mb[:, t], k * (db[:, t] + l * mb[:, t])
        eb = 1.01 * (db + FIXED * mb) + 8 * TINY * S
        before, mbe, ebe = (np.where(begins[..., None], 0, x[:, :-1]) for x in (hs, ms, eh))
        t, K2 = a * u, 2 * delta(f) + 6 * EPS
        dz = [dh * (before - v) * t, dh * u]
        bz = [t * (eb * (mbe + np.abs(v)) + mb * (ebe + K2 * (mbe + np.abs(v)))), u * (eb + K * mb)]
        if output_gate:
            so1 = so * sig(-o)
            dz.append(dy * hs[:, 1:] * so1)
            bz.append(np.abs(dy) * so1 * (eh[:, 1:] + (2 * do + 6 * EPS) * ms[:, 1:]))
        want.update(dz=np.concatenate([np.where(L, x, 0) for x in dz], -1), dh0=r)
        bound.update(dz=np.concatenate([np.where(L, 1.01 * x + 8 * TINY * M * S, 0) for x in bz], -1), dh0=1.01 * (dr + FIXED * mr) + 8 * TINY * S)
    return tuple({k: torch.from_numpy(np.ascontiguousarray(x)) for k, x in d.items()} for d in (want, bound))


def check_local(got, local, only=None):
    """Every number within its own bound and the rounding to its type."""
    want, bound = local
    for k in want:
        if got.get(k) is None or (only and k not in only):
            continue
        x, w, b = got[k].detach(), want[k], bound[k]
        info = torch.finfo(x.dtype)
        over = (x.double().cpu() - w).abs() / (b + info.eps / 2 * (w.abs() + b) + info.smallest_normal * info.eps / 2)
        assert x.shape == w.shape and not x.isnan().any(), k
        assert float(over.max()) <= 1.0, f"{k}: {float(over.max()):.3g} times its bound at {np.unravel_index(int(over.argmax()), over.shape)}"
