"""The gated recurrence on the GPU against its plain 64-bit form (tests/_ops.py, with the bounds' derivation)."""
import pytest
import torch

from tests._ops import DTYPES, check_blend, check_local, check_scan, gate_ends, local_scan, near, oracle_scan
from wavenet_vocoder_amd.recurrence import gated_recurrence, gated_recurrence_step

pytestmark = pytest.mark.gpu


def inputs(B, T, C, gates, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(B, T, gates * C, generator=g)
    z[..., :C] = z[..., :C] * 1.5 + 2.0
    return (z.to(dt), torch.randn(B, C, generator=g), torch.randn(B, T, C, generator=g).to(dt), torch.randn(B, C, generator=g))


def maps(kind, B, T, seed=0):
    g = torch.Generator().manual_seed(seed + 77)
    if kind == "lengths":
        n = torch.randint(0, T + 1, (B,), generator=g)
        n[0] = 0
        n[-1] = T
        if B > 2:
            n[1] = 1
        return dict(lengths=n.to(torch.int32))
    if kind in ("packed", "both"):
        first = torch.rand(B, T, generator=g) < 0.02
        first[::2, 0] = True
        at = torch.arange(T).expand(B, T)
        m = dict(seg_start=torch.where(first, at, torch.tensor(-1)).cummax(1).values.to(torch.int32))
        if kind == "both":
            m["lengths"] = torch.randint(0, T + 1, (B,), generator=g).to(torch.int32)
        return m
    return {}


def run(z, h0, dy, dh, gates, m, grads=True):
    """One forward and backward pass through the public function; outputs as check_scan takes them."""
    zc = z.cuda().requires_grad_(grads)
    hc = None if h0 is None else h0.cuda().requires_grad_(grads)
    mc = {k: v.cuda() for k, v in m.items()}
    y, h_last = gated_recurrence(zc, hc, output_gate=gates == 3, **mc)
    got = dict(y=y, h_last=h_last)
    if grads:
        leaves = (zc,) if hc is None else (zc, hc)
        d = torch.autograd.grad((y, h_last), leaves, (dy.cuda(), dh.cuda()))
        got.update(dz=d[0], dh0=d[1] if hc is not None else None)
    torch.cuda.synchronize()
    return got


SHAPES = [(1, 1, 1), (2, 2, 3), (3, 7, 20), (2, 127, 64), (2, 128, 65), (3, 129, 33), (1, 300, 128), (2, 513, 17), (4, 1000, 72),
          (1, 2500, 8), (2, 1025, 201), (1, 4097, 40), (2, 511, 2), (1, 513, 3), (3, 1500, 4), (2, 9000, 16), (1, 2100, 17),
          (2, 300, 130), (1, 512, 67), (12, 400, 700), (2, 200, 300), (1, 256, 500), (2, 257, 300), (3, 1024, 33), (2, 1024, 2), (2, 1025, 256),
          (12, 1000, 130), (40, 1000, 70), (3, 500, 1300), (80, 1000, 30), (2, 513, 600)]


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("gates", [2, 3])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_scan_and_gradients(shape, gates, dtype):
    B, T, C = shape
    z, h0, dy, dh = inputs(B, T, C, gates, DTYPES[dtype], seed=T)
    want = oracle_scan(z, h0, gates == 3, dy=dy, dh_last=dh)
    check_scan(run(z, h0, dy, dh, gates, {}), want, z, h0, gates == 3, None, dy, dh)


@pytest.mark.parametrize("kind", ["lengths", "packed", "both"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(5, 1, 8), (4, 130, 24), (3, 700, 129), (5, 2049, 16), (4, 400, 70), (4, 1000, 40), (4, 200, 260), (4, 1000, 3)], ids=lambda s: "x".join(map(str, s)))
def test_padded_batches_and_packed_slots(shape, dtype, kind):
    B, T, C = shape
    z, h0, dy, dh = inputs(B, T, C, 3, DTYPES[dtype], seed=T + 1)
    m = maps(kind, B, T, seed=T)
    want = oracle_scan(z, h0, True, dy=dy, dh_last=dh, **m)
    got = run(z, h0, dy, dh, 3, m)
    check_scan(got, want, z, h0, True, m.get("lengths"), dy, dh)
    if "lengths" in m:
        behind = torch.arange(T) >= m["lengths"][:, None]
        assert not got["y"].cpu()[behind].any() and not got["dz"].cpu()[behind].any()
        empty = m["lengths"] == 0
        assert torch.equal(got["h_last"].cpu()[empty], h0[empty]) and torch.equal(got["dh0"].cpu()[empty], dh[empty])


@pytest.mark.parametrize("shape", [(9, 100, 70), (9, 1500, 70), (9, 3000, 20), (90, 1025, 80)], ids=lambda s: "x".join(map(str, s)))
def test_a_rows_bits_do_not_depend_on_its_batch(shape):
    """Neither within short sequences (128 steps) nor within long ones (more than 1024); between them the cut goes by the amount of data."""
    B, T, C = shape
    z, h0, dy, dh = inputs(B, T, C, 3, torch.bfloat16, seed=3)
    all_ = run(z, h0, dy, dh, 3, {})
    for b in (0, 4, B - 1):
        one = run(z[b:b + 1], h0[b:b + 1], dy[b:b + 1], dh[b:b + 1], 3, {})
        for k in all_:
            assert torch.equal(one[k][0], all_[k][b]), k


@pytest.mark.parametrize("T", [40, 1500])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
def test_what_stands_behind_a_length_is_not_looked_at(poison, T):
    B, C = 3, 40
    z, h0, dy, dh = inputs(B, T, C, 3, torch.float32, seed=5)
    n = torch.tensor([0, T // 2, T - 1], dtype=torch.int32)
    clean = run(z, h0, dy, dh, 3, dict(lengths=n))
    behind = torch.arange(T) >= n[:, None]
    z[behind] = poison
    dy[behind] = poison
    got = run(z, h0, dy, dh, 3, dict(lengths=n))
    for k in clean:
        assert torch.equal(got[k], clean[k]), k


@pytest.mark.parametrize("T", [60, 1500])
def test_a_broken_utterance_stays_its_own(T):
    """NaN and infinities of one utterance of a packed slot reach neither the next one's outputs nor the earlier one's gradients."""
    z, h0, dy, dh = inputs(1, T, 16, 3, torch.float32, seed=6)
    a, b = T // 3, 2 * T // 3
    start = torch.zeros(1, T, dtype=torch.int32)
    start[:, a:b], start[:, b:] = a, b
    clean = run(z, h0, dy, dh, 3, dict(seg_start=start))
    z[:, a + 2], z[:, b - 3] = float("nan"), float("inf")
    dy[:, b - 2] = float("nan")
    got = run(z, h0, dy, dh, 3, dict(seg_start=start))
    for k in ("y", "dz"):
        assert torch.equal(got[k][:, :a], clean[k][:, :a]) and torch.equal(got[k][:, b:], clean[k][:, b:]), k
        assert torch.isnan(got[k][:, a:b]).any()
    assert torch.equal(got["h_last"], clean["h_last"]) and torch.equal(got["dh0"], clean["dh0"])


def test_a_nan_input_is_seen():
    z, h0, dy, dh = inputs(1, 700, 4, 3, torch.float32)
    z[0, 300, 1] = float("nan")                     # the gate of channel 1
    got = run(z, h0, dy, dh, 3, {})
    assert torch.isnan(got["y"][0, 300:, 1]).all() and torch.isnan(got["h_last"][0, 1])
    assert torch.isfinite(got["y"][..., [0, 2, 3]]).all() and torch.isfinite(got["y"][0, :300]).all()
    assert torch.isnan(got["dh0"][0, 1])


@pytest.mark.parametrize("f", [-200.0, -30.0, 30.0, 200.0])
@pytest.mark.parametrize("T", [5, 900])
def test_gates_at_their_ends(f, T):
    z, h0, dy, dh = inputs(2, T, 12, 3, torch.float32, seed=9)
    z[..., :12] = f
    want = oracle_scan(z, h0, True, dy=dy, dh_last=dh)
    check_scan(run(z, h0, dy, dh, 3, {}), want, z, h0, True, None, dy, dh)


@pytest.mark.parametrize("T", [5, 900])
@pytest.mark.parametrize("gate", ["f", "o"])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_infinite_gates_are_their_limits(sign, dtype, gate, T):
    """Infinities and the type's ends give the bits of 300, whose sigmoid is 0 or 1 in 32 bits."""
    z, h0, dy, dh = inputs(2, T, 12, 3, DTYPES[dtype], seed=10)
    at, c = (slice(0, 12) if gate == "f" else slice(24, 36)), slice(1, T, 2)
    outs = []
    for x in (300.0, float("inf"), torch.finfo(DTYPES[dtype]).max):
        z[:, c, at] = sign * x
        outs.append(run(z, h0, dy, dh, 3, {}))
    for k in outs[0]:
        assert torch.isfinite(outs[0][k]).all() and torch.equal(outs[0][k], outs[1][k]) and torch.equal(outs[0][k], outs[2][k]), k


def test_the_state_before_may_be_written_to_before_the_backward_pass():
    z, h0, dy, dh = inputs(2, 300, 20, 3, torch.float32, seed=12)
    want = run(z, h0, dy, dh, 3, {})
    zc, state = z.cuda().requires_grad_(), h0.cuda()
    y, h = gated_recurrence(zc, state)
    state.copy_(h.detach())
    dz, = torch.autograd.grad((y, h), zc, (dy.cuda(), dh.cuda()))
    assert torch.equal(dz, want["dz"])


def test_long_memory_keeps_its_precision():
    """f = 9 remembers 8000 steps: a gate held only as sigmoid(f) in float32 would be 2e-4 off here."""
    T, C = 12000, 8
    z, h0, dy, dh = inputs(1, T, C, 2, torch.float32, seed=11)
    z[..., :C] = 9.0
    z[..., C:] += 1.0
    want = oracle_scan(z, h0, False, dy=dy, dh_last=dh)
    got = run(z, h0, dy, dh, 2, {})
    check_scan(got, want, z, h0, False, None, dy, dh)
    # random roundings: eps sqrt(8000) each way, far below the bound's sum of them and below 2e-4
    assert float((got["h_last"].double().cpu() - want["h_last"]).abs().max()) < 2e-5 * float(z[..., C:].abs().max())


def test_optional_arguments_and_partial_gradients():
    z, h0, dy, dh = inputs(2, 333, 24, 3, torch.float32, seed=3)
    want = oracle_scan(z, None, True, dy=dy)
    zc = z.cuda().requires_grad_()
    y, h_last = gated_recurrence(zc)
    dz, = torch.autograd.grad(y, zc, dy.cuda(), retain_graph=True)
    check_scan(dict(y=y, h_last=h_last, dz=dz), want, z, None, True, None, dy, None)
    dz, = torch.autograd.grad(h_last, zc, dh.cuda())            # no gradient at y
    want = oracle_scan(z, None, True, dh_last=dh)
    check_scan(dict(y=y, h_last=h_last, dz=dz), want, z, None, True, None, None, dh)
    hc = h0.cuda().requires_grad_()                             # the state alone
    y, h_last = gated_recurrence(z.cuda(), hc)
    d, = torch.autograd.grad((y, h_last), hc, (dy.cuda(), dh.cuda()))
    near(d, oracle_scan(z, h0, True, dy=dy, dh_last=dh)["dh0"], 1e-3, "dh0")
    with torch.no_grad():
        assert torch.equal(gated_recurrence(zc)[0], gated_recurrence(z.cuda())[0])
    assert not gated_recurrence(z.cuda())[0].requires_grad


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("how", ["offset", "wide", "time", "broadcast_time", "broadcast_batch", "columns"])
def test_strides(how, dtype):
    """Views of other alignments and orders give the bits of the same values laid out densely."""
    B, T, C, dt = 3, 300, 24, DTYPES[dtype]
    z, h0, dy, dh = (t.cuda() for t in inputs(B, T, C, 3, dt, seed=13))
    if how == "offset":                 # one element behind an aligned address
        v = torch.empty(z.numel() + 1, dtype=dt, device="cuda")[1:].view(z.shape).copy_(z)
    elif how == "wide":                 # a slice of wider rows
        v = torch.zeros(B, T, 3 * C + 7, dtype=dt, device="cuda")[..., 3:3 + 3 * C].copy_(z)
    elif how == "time":                 # time first in memory
        v = torch.empty(T, B, 3 * C, dtype=dt, device="cuda").transpose(0, 1).copy_(z)
    elif how == "broadcast_time":
        z = z[:, :1].expand(B, T, 3 * C).contiguous()
        v = z[:, :1].contiguous().expand(B, T, 3 * C)
    elif how == "broadcast_batch":
        z = z[:1].expand(B, T, 3 * C).contiguous()
        v = z[:1].contiguous().expand(B, T, 3 * C)
    else:                               # channels are not contiguous: copied once
        v = torch.empty(B, 3 * C, T, dtype=dt, device="cuda").transpose(1, 2).copy_(z)
    dyv = torch.empty(T, B, C, dtype=dt, device="cuda").transpose(0, 1).copy_(dy)
    outs = []
    for a, d in ((z, dy), (v, dyv)):
        a = a.detach().requires_grad_()
        y, h = gated_recurrence(a, h0)
        outs.append((y, h, *torch.autograd.grad((y, h), a, (d, dh))))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_gradients_of_broadcast_inputs():
    """One row of gates for the whole batch, one initial state for all rows: their gradients are the sums over the batch."""
    B, T, C = 4, 150, 16
    z, h0, dy, dh = inputs(B, T, C, 3, torch.float32, seed=17)
    z, h0 = z[:1], h0[:1]
    want = oracle_scan(z.expand(B, -1, -1), h0.expand(B, -1), True, dy=dy, dh_last=dh)
    zc, hc = z.cuda().requires_grad_(), h0.cuda().requires_grad_()
    y, h = gated_recurrence(zc.expand(B, -1, -1), hc.expand(B, -1))
    dz, dh0 = torch.autograd.grad((y, h), (zc, hc), (dy.cuda(), dh.cuda()))
    near(dz, want["dz"].sum(0, keepdim=True), 1e-3, "dz")
    near(dh0, want["dh0"].sum(0, keepdim=True), 1e-3, "dh0")


@pytest.mark.parametrize("gates", [2, 3])
def test_gradient_against_differences(gates):
    """<gradient, d> = (L(x + e d) - L(x - e d)) / 2 e of the exact forward pass, to e^2 and the gradient's own float32 error."""
    B, T, C = 2, 200, 6
    z, h0, dy, dh = inputs(B, T, C, gates, torch.float32, seed=19)
    got = run(z, h0, dy, dh, gates, {})
    g = torch.Generator().manual_seed(1)
    for _ in range(4):
        d, e = torch.randn(z.shape, generator=g).double(), 1e-4
        d0 = torch.randn(h0.shape, generator=g).double()
        L = []
        for s in (e, -e):
            o = oracle_scan(z.double() + s * d, h0.double() + s * d0, gates == 3)
            L.append(float((o["y"] * dy.double()).sum() + (o["h_last"] * dh.double()).sum()))
        diff = (L[0] - L[1]) / (2 * e)
        dot = float((got["dz"].double().cpu() * d).sum() + (got["dh0"].double().cpu() * d0).sum())
        mass = float((got["dz"].double().cpu() * d).abs().sum() + (got["dh0"].double().cpu() * d0).abs().sum())
        assert abs(diff - dot) <= 1e-5 * mass, (diff, dot, mass)


def test_batch_strides_over_32_bits():
    C, T = 8, 40
    z, h0, dy, dh = inputs(2, T, C, 3, torch.bfloat16, seed=23)
    far = (1 << 31) + 8                 # elements between the two rows
    buf = torch.empty(far + T * 3 * C, dtype=torch.bfloat16, device="cuda")
    v = buf.as_strided((2, T, 3 * C), (far, 3 * C, 1))
    v.copy_(z)
    v.requires_grad_()
    y, h = gated_recurrence(v, h0.cuda())
    dz, = torch.autograd.grad((y, h), v, (dy.cuda(), dh.cuda()))
    want = run(z, h0, dy, dh, 3, {})
    assert torch.equal(y, want["y"]) and torch.equal(h, want["h_last"]) and torch.equal(dz, want["dz"])


def test_outputs_over_32_bits():
    """dz of 2.6e9 values: the last row and a middle one against the same rows alone."""
    B, T, C = 18, 24064, 2000
    g = torch.Generator(device="cuda").manual_seed(3)
    z = torch.randn(B, T, 3 * C, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_()
    dy = torch.randn(B, T, C, generator=g, device="cuda", dtype=torch.bfloat16)
    y, h = gated_recurrence(z)
    dz, = torch.autograd.grad(y, z, dy)
    for b in (B // 2, B - 1):
        zb = z[b:b + 1].detach().clone().requires_grad_()
        yb, hb = gated_recurrence(zb)
        dzb, = torch.autograd.grad(yb, zb, dy[b:b + 1])
        # one row alone may be cut into stretches elsewhere: equal to the roundings of bf16 and of the sums behind them
        for p, q in ((y[b], yb[0]), (dz[b], dzb[0]), (h[b], hb[0])):
            assert float((p.float() - q.float()).abs().max()) <= 2.0 ** -8 * float(q.float().abs().max()) * 1.01


def test_the_same_call_gives_the_same_bits():
    z, h0, dy, dh = inputs(3, 2000, 96, 3, torch.bfloat16, seed=29)
    first = run(z, h0, dy, dh, 3, {})
    for _ in range(5):
        again = run(z, h0, dy, dh, 3, {})
        for k in first:
            assert torch.equal(first[k], again[k]), k


def test_two_streams_at_once():
    args = [inputs(2, 3000, 64, 3, torch.float32, seed=s) for s in (31, 37)]
    want = [run(*a, 3, {}) for a in args]
    dev = [[t.cuda() for t in a] for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        got = []
        for (z, h0, dy, dh), s in zip(dev, streams):
            with torch.cuda.stream(s):
                a, b = z.detach().requires_grad_(), h0.detach().requires_grad_()
                y, h = gated_recurrence(a, b)
                got.append((y, h, *torch.autograd.grad((y, h), (a, b), (dy, dh))))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for x, k in zip(g, ("y", "h_last", "dz", "dh0")):
                assert torch.equal(x, w[k]), k


@pytest.mark.parametrize("T", [50, 3000])
def test_captured_and_replayed(T):
    """Forward and backward of two graphs with inputs of their own, replayed in turn and side by side with eager work between."""
    args = [inputs(2, T, 48, 3, torch.bfloat16, seed=s) for s in (41, 43)]
    start = maps("packed", 2, T)["seg_start"].cuda()
    graphs, bufs, outs = [], [], []
    for a in args:
        z, h0, dy, dh = (t.cuda() for t in a)
        z, h0 = z.requires_grad_(), h0.requires_grad_()

        def once(z=z, h0=h0, dy=dy, dh=dh):
            y, h = gated_recurrence(z, h0, seg_start=start)
            return (y, h, *torch.autograd.grad((y, h), (z, h0), (dy, dh)))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            once()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(once())
        graphs.append(g)
        bufs.append((z, h0, dy, dh, once))
    other = torch.cuda.Stream()
    for rep in range(4):
        with torch.no_grad():
            for z, h0, dy, dh, _ in bufs:
                z.copy_(torch.randn_like(z) + 1)
                h0.copy_(torch.randn_like(h0))
        want = [b[4]() for b in bufs]
        for o in outs:
            for t in o:
                t.detach().zero_()
        torch.cuda.synchronize()
        if rep % 2:
            with torch.cuda.stream(other):
                graphs[1].replay()
            graphs[0].replay()
        else:
            graphs[0].replay()
            graphs[1].replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            for x, y in zip(o, w):
                assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("gates", [2, 3])
@pytest.mark.parametrize("shape", [(1, 1), (8, 128), (3, 17), (65, 130), (1, 2049)], ids=lambda s: "x".join(map(str, s)))
def test_step_is_the_scan(shape, gates, dtype):
    B, C = shape
    T, dt = 5, DTYPES[dtype]
    z, h0, _, _ = inputs(B, T, C, gates, dt, seed=47)
    want = oracle_scan(z, h0, gates == 3)
    state, ys = h0.cuda(), []
    for t in range(T):
        at = state.data_ptr()
        ys.append(gated_recurrence_step(z.cuda()[:, t], state, output_gate=gates == 3))       # a strided view of the sequence
        assert state.data_ptr() == at
    check_scan(dict(y=torch.stack(ys, 1), h_last=state), want, z, h0, gates == 3)


def test_step_captured():
    z, h0, _, _ = inputs(4, 6, 40, 3, torch.float32, seed=53)
    want = oracle_scan(z, h0, True)
    zt, state = z[:, 0].cuda(), h0.cuda()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = gated_recurrence_step(zt, state)
    state.copy_(h0)
    ys = []
    for t in range(6):
        zt.copy_(z[:, t])
        g.replay()
        ys.append(y.clone())
    check_scan(dict(y=torch.stack(ys, 1), h_last=state), want, z, h0, True)


def test_offsets_of_the_step_over_32_bits():
    far = (1 << 31) + 8
    z, h0, _, _ = inputs(2, 1, 8, 3, torch.bfloat16, seed=59)
    v = torch.empty(far + 24, dtype=torch.bfloat16, device="cuda").as_strided((2, 24), (far, 1))
    v.copy_(z[:, 0])
    a, b = h0.cuda(), h0.cuda()
    assert torch.equal(gated_recurrence_step(v, a), gated_recurrence_step(z[:, 0].cuda(), b)) and torch.equal(a, b)


def test_steps_far_apart():
    """Time strides of 2^20 elements and more are copied once."""
    z, h0, dy, dh = inputs(1, 3, 8, 3, torch.bfloat16, seed=61)
    far = (1 << 22) + 16
    v = torch.empty(2 * far + 24, dtype=torch.bfloat16, device="cuda").as_strided((1, 3, 24), (3 * far, far, 1))
    v.copy_(z)
    assert torch.equal(gated_recurrence(v, h0.cuda())[0], gated_recurrence(z.cuda(), h0.cuda())[0])


def test_refusals_on_the_device():
    z = torch.zeros(2, 5, 12, device="cuda")
    ok = torch.zeros(2, 4, device="cuda")
    i32 = torch.int32
    for bad, err in ((dict(z=z[0]), ValueError), (dict(z=z[..., :11]), ValueError), (dict(z=z[:0]), ValueError), (dict(z=z[:, :0]), ValueError),
                     (dict(z=z[..., :0]), ValueError), (dict(z=z.double()), TypeError), (dict(h0=ok[:1]), ValueError),
                     (dict(h0=ok.double()), TypeError), (dict(h0=ok.cpu()), ValueError), (dict(lengths=torch.zeros(3, dtype=i32, device="cuda")), ValueError),
                     (dict(lengths=torch.zeros(2, device="cuda")), TypeError), (dict(lengths=torch.zeros(2, dtype=i32)), ValueError),
                     (dict(seg_start=torch.zeros(2, 4, dtype=i32, device="cuda")), ValueError),
                     (dict(z=z[:1].expand(65536, 5, 12)), ValueError), (dict(z=z[:1, :1].expand(1, (1 << 30) + 1, 12)), ValueError)):
        a = dict(z=z)
        a.update(bad)
        with pytest.raises(err):
            gated_recurrence(a.pop("z"), a.pop("h0", None), **a)
    zs, st = torch.zeros(2, 12, device="cuda"), torch.zeros(2, 4, device="cuda")
    for zz, ss, err in ((zs[:, :11], st, ValueError), (zs[0], st, ValueError), (zs[:0], st[:0], ValueError), (zs.double(), st, TypeError),
                        (zs, st[:1], ValueError), (zs, st.double(), TypeError), (zs, st.cpu(), ValueError), (zs.cpu(), st, RuntimeError),
                        (zs, torch.zeros(2, 8, device="cuda")[:, ::2], ValueError), (zs, torch.zeros(1, 4, device="cuda").expand(2, 4), ValueError),
                        (zs.clone().requires_grad_(), st, RuntimeError), (zs, st.clone().requires_grad_(), RuntimeError)):
        with pytest.raises(err):
            gated_recurrence_step(zz, ss)
    w = z.clone().requires_grad_()
    y, _ = gated_recurrence(w)
    g, = torch.autograd.grad(y.sum(), w, create_graph=True)     # asked for, though nothing goes through it
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), w)


def test_lengths_outside_the_sequence_and_of_64_bits():
    z, h0, dy, dh = inputs(4, 90, 12, 3, torch.float32, seed=71)
    want = run(z, h0, dy, dh, 3, dict(lengths=torch.tensor([0, 90, 7, 90], dtype=torch.int32)))
    got = run(z, h0, dy, dh, 3, dict(lengths=torch.tensor([-5, 2 ** 40, 7, 91])))
    for k in want:
        assert torch.equal(got[k], want[k]), k


def test_work_under_way_on_another_stream():
    """The call runs on the current stream and waits there for the inputs' producer."""
    z, h0, _, _ = (t.cuda() for t in inputs(2, 2000, 64, 3, torch.float32, seed=73))
    want = gated_recurrence(z, h0)
    s = torch.cuda.Stream()
    for _ in range(5):
        late = torch.zeros_like(z)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(20):
                late.copy_(z * 0.5)
            late.copy_(z)
            y, h = gated_recurrence(late, h0)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(y, want[0]) and torch.equal(h, want[1])


@pytest.mark.parametrize("kind", ["full", "both"])
@pytest.mark.parametrize("gates,dtype", [(2, "f32"), (3, "bf16")])
def test_data_larger_than_the_caches(gates, dtype, kind):
    """Rows of whole lines, more than the last-level cache holds, take another path to memory than the same values an element off:
    the same bits."""
    B, T, C, dt = 8, 12100, 512, DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(79)
    n = B * T * gates * C
    z = torch.randn(n + 1, generator=g, device="cuda").to(dt)
    off = z[1:].view(B, T, gates * C)
    on = off.clone()
    dy = torch.randn(B, T, C, generator=g, device="cuda").to(dt)
    dh = torch.randn(B, C, generator=g, device="cuda")
    h0 = torch.randn(B, C, generator=g, device="cuda")
    m = {k: v.cuda() for k, v in maps(kind, B, T, seed=3).items()}
    outs = []
    for a in (on, off):
        a = a.detach().requires_grad_()
        y, h = gated_recurrence(a, h0, output_gate=gates == 3, **m)
        outs.append((y, h, *torch.autograd.grad((y, h), a, (dy, dh))))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    row = B - 1                         # and one row against the definition
    k = {n: v[row:row + 1].cpu() for n, v in m.items()}
    zr, hr = on[row:row + 1].cpu(), h0[row:row + 1].cpu()
    want = oracle_scan(zr, hr, gates == 3, dy=dy[row:row + 1].cpu(), dh_last=dh[row:row + 1].cpu(), **k)
    got = dict(y=outs[0][0][row:row + 1], h_last=outs[0][1][row:row + 1], dz=outs[0][2][row:row + 1])
    check_scan(got, want, zr, hr, gates == 3, k.get("lengths"), dy[row:row + 1], dh[row:row + 1])


@pytest.mark.parametrize("gates", [2, 3])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_step_with_gates_at_both_ends(dtype, gates):
    """A gate that forgets leaves of the state what the formula leaves, not 2^-24 of what it was; one that replaces it gives v."""
    f, h, v = gate_ends(DTYPES[dtype])
    state = h[None].cuda()
    z = torch.cat([f, v] + [torch.zeros_like(v)] * (gates - 2))[None].cuda()
    y = gated_recurrence_step(z, state, output_gate=gates == 3)
    check_blend(state[0], f, h, v)
    assert torch.equal(y, (state * (0.5 if gates == 3 else 1.0)).to(y.dtype))


LOCAL_SHAPES = [(1, 1, 4), (2, 9, 3), (3, 130, 40), (2, 1000, 20), (2, 1000, 70), (1, 3000, 24), (1, 3000, 67)]


@pytest.mark.parametrize("kind", ["full", "lengths", "both"])
@pytest.mark.parametrize("what", ["h0", "dh_last", "v", "dy", "all"])
@pytest.mark.parametrize("shape", LOCAL_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_large_values_leave_what_the_gates_leave(shape, what, kind):
    """A state, gradient, input or gradient of an output 1e6 times the others: what is left of it after its gates, no more."""
    B, T, C = shape
    z, h0, dy, dh = inputs(B, T, C, 3, torch.float32, seed=T + C)
    z[..., :C] = (z[..., :C] - 2.0) / 1.5           # gates about 1/2
    if what in ("h0", "all"):
        h0 *= 1e6
    if what in ("dh_last", "all"):
        dh *= 1e6
    if what in ("v", "all"):
        z[:, T // 3, C:2 * C] *= 1e6
    if what in ("dy", "all"):
        dy[:, T // 2] *= 1e6
    m = maps(kind, B, T, seed=T)
    check_local(run(z, h0, dy, dh, 3, m), local_scan(z, h0, True, dy=dy, dh_last=dh, **m))


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("f", [-80.0, -20.0, -16.0, -12.0, -10.0, -6.0, -1.0, 0.0, 1.0, 6.0, 10.0])
@pytest.mark.parametrize("shape", [(2, 1, 8), (2, 2, 40), (1, 5, 130), (2, 300, 20), (2, 300, 70)], ids=lambda s: "x".join(map(str, s)))
def test_gates_hold_their_precision_at_both_ends(shape, f, dtype):
    """Every output of gates around f, dh0 of gates that forget among them: (2^-24 |f|) of itself, not of 1."""
    B, T, C = shape
    z, h0, dy, dh = inputs(B, T, C, 3, torch.float32, seed=7)
    z[..., :C] = f + 0.1 * z[..., :C]
    z = z.to(DTYPES[dtype])
    dy = dy.to(DTYPES[dtype])
    check_local(run(z, h0, dy, dh, 3, {}), local_scan(z, h0, True, dy=dy, dh_last=dh))


@pytest.mark.parametrize("T", [3, 200, 700, 3000])
@pytest.mark.parametrize("C", [12, 70])
def test_infinite_gates_replace_and_keep(C, T):
    """f = -inf: the state is v, whatever it was.  f = inf: the state stays."""
    z, h0, dy, dh = inputs(2, T, C, 2, torch.float32, seed=10)
    h0 *= 1e8
    z[..., :C] = -float("inf")
    got = run(z, h0, dy, dh, 2, {})
    assert torch.equal(got["y"].cpu(), z[..., C:]) and torch.equal(got["h_last"].cpu(), z[:, -1, C:]) and not got["dh0"].any()
    assert torch.equal(got["dz"][..., C:].cpu()[:, :-1], dy[:, :-1])
    z[:, :, :C] = float("inf")
    z[:, T // 2, :C] = -float("inf")
    got = run(z, h0, dy, dh, 2, {})
    want = h0[:, None].repeat(1, T, 1)
    want[:, T // 2:] = z[:, T // 2, None, C:]
    assert torch.equal(got["y"].cpu(), want) and torch.equal(got["h_last"].cpu(), want[:, -1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [4, 200, 700, 3000])
@pytest.mark.parametrize("C", [12, 70])
def test_values_at_the_type_s_ends(C, T, dtype):
    """v, h0 and dh_last of both signs next to the largest number: a convex combination of them is none larger."""
    z, h0, dy, dh = inputs(2, T, C, 2, torch.float32, seed=10)
    sign = torch.where(torch.arange(T) % 2 == 0, 1.0, -1.0)[:, None]
    z[..., :C] = (z[..., :C] - 2.0) / 1.5
    z[..., C:] = 3e38 * sign
    z = z.to(DTYPES[dtype])
    h0 = torch.full_like(h0, -3e38)
    dy *= 1e-20
    dh = torch.full_like(dh, 1e-20)
    check_local(run(z, h0, dy.to(z.dtype), dh, 2, {}), local_scan(z, h0, False, dy=dy.to(z.dtype), dh_last=dh))


@pytest.mark.parametrize("T", [4, 200, 700, 3000])
@pytest.mark.parametrize("C", [12, 70])
def test_an_infinite_state_is_handed_on(C, T):
    """Empty rows, and what stands behind a length, hand on what they are given, whatever it is: forward the state, backward its gradient."""
    z, h0, dy, dh = inputs(3, T, C, 3, torch.float32, seed=14)
    inf = float("inf")
    for x in (h0, dh):
        x[0, ::2], x[0, 1::3] = inf, -inf
    n = torch.tensor([0, T // 2, T - 1], dtype=torch.int32)
    z[1, T // 2 - 1, C:2 * C] = inf                 # the last live step's input: the state behind it is infinite, or
    z[1, T // 2 - 1, :C] = 0.0
    dh[2] = inf                                     # the gradient that arrives at row 2's end
    got = run(z, h0, dy, dh, 3, dict(lengths=n))
    assert torch.equal(got["h_last"][0].cpu(), h0[0]) and torch.equal(got["dh0"][0].cpu(), dh[0])
    assert (got["h_last"][1] == inf).all()
    assert torch.equal(got["dz"][2, T - 2, C:2 * C].cpu(), torch.full((C,), inf)) and not got["y"][0].any()


@pytest.mark.parametrize("kind", ["full", "both"])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("shape", [(90, 300, 100), (30, 300, 300), (9, 512, 700), (60, 1000, 40), (40, 700, 130), (20, 1024, 256), (80, 513, 67), (200, 129, 130),
                                   (100, 1000, 30), (600, 700, 8), (700, 1024, 3), (100, 900, 32), (5000, 513, 1)],
                         ids=lambda s: "x".join(map(str, s)))
def test_a_rows_bits_do_not_depend_on_its_batch_at_any_length(shape, dtype, kind):
    """Sequences that a small batch runs in one workgroup and a large one in several, whose joins are the same."""
    B, T, C = shape
    z, h0, dy, dh = inputs(B, T, C, 3, DTYPES[dtype], seed=3)
    m = maps(kind, B, T, seed=5)
    all_ = run(z, h0, dy, dh, 3, m)
    for b, n in ((0, 1), (B // 2, 2), (B - 1, 1)):
        part = run(z[b:b + n], h0[b:b + n], dy[b:b + n], dh[b:b + n], 3, {k: v[b:b + n] for k, v in m.items()})
        for k in all_:
            assert torch.equal(part[k], all_[k][b:b + n]), (k, b)


# Chunks of 128 steps (512 of rows up to 32 channels), groups of 16 chunks, sections of 16 groups: from chunk 144 on a chunk takes the maps of its
# section's groups 8 and up, from chunk 256 on a state that a section handed out, from 512 on one that had another's before it.
LONG = [(1, 20000, 33), (2, 33000, 40), (1, 70000, 36), (1, 80000, 20), (2, 135000, 5), (1, 270000, 2)]


@pytest.mark.parametrize("kind", ["full", "ends"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", LONG, ids=lambda s: "x".join(map(str, s)))
def test_long_sequences_against_the_definition(shape, dtype, kind):
    """Every level of the hand-over between chunks, with gates that remember 8000 steps, so that each is seen far behind it."""
    B, T, C = shape
    z, h0, dy, dh = inputs(B, T, C, 2, torch.float32, seed=T)
    z[..., :C] = 9.0 + 0.1 * z[..., :C]
    z[..., C:] += 1.0
    z, dy = z.to(DTYPES[dtype]), dy.to(DTYPES[dtype])
    h0, dh = 30 * h0, 30 * dh
    m = {}
    if kind == "ends":                  # a length inside the last chunks, utterances that begin on both sides of the hand-overs
        start = torch.full((B, T), -1, dtype=torch.int32)
        for at in (T // 3, T // 2 + 1, T - 700):
            start[:, at:] = at
        m = dict(lengths=torch.full((B,), T - 300, dtype=torch.int32), seg_start=start)
    check_local(run(z, h0, dy, dh, 2, m), local_scan(z, h0, False, dy=dy, dh_last=dh, long=True, **m))
