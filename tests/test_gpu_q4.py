"""Products with 4-bit weights on the GPU against their plain 64-bit form (tests/_ops.py, with the bounds' derivation)."""
import pytest
import torch

from tests._ops import DTYPES, EPS, check_blend, gate_ends, near, q4_bound, q4_weight, random_q4
from wavenet_vocoder_amd.engine import Q4Linear

pytestmark = pytest.mark.gpu


def layer(cin, cout, group, gates=1, seed=0, zeros=True, bias=True):
    codes, scales, zp = random_q4(cout, cin, group, seed, zeros)
    b = torch.randn(cout, generator=torch.Generator().manual_seed(seed + 1)) if bias else None
    q = Q4Linear(cin, cout, "cuda", group_size=group, gates=gates)
    q.set_codes(codes.cuda(), scales.cuda(), None if zp is None else zp.cuda(), None if b is None else b.cuda())
    return q, (codes, scales, zp, b)


def exact(x, parts, group):
    codes, scales, zp, b = parts
    y = x.double().cpu() @ q4_weight(codes, scales, zp, group).t()
    return y if b is None else y + b.double()


def check(y, x, parts, group):
    want = exact(x, parts, group)
    bound = q4_bound(x, parts[0], parts[1], parts[2], group, parts[3])
    info = torch.finfo(y.dtype)
    allowed = bound * (1 + info.eps) + info.eps / 2 * want.abs() + info.smallest_normal * info.eps / 2
    got = y.double().cpu()
    over = float(((got - want).abs() / allowed).max())
    assert got.shape == want.shape and over <= 1.0, f"{over:.3g} times its bound"


SHAPES = [(1, 1, 1), (1, 16, 16), (2, 33, 17), (3, 127, 15), (5, 128, 48), (8, 129, 100), (16, 300, 31), (17, 512, 64), (31, 80, 256),
          (33, 1616, 40), (48, 257, 96), (64, 640, 130), (65, 96, 24), (130, 200, 50), (1, 4100, 33), (4, 2048, 1000), (48, 130, 2100), (64, 2200, 1100), (9, 4100, 40), (5, 2100, 20)]


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_products(shape, group, dtype):
    B, cin, cout = shape
    q, parts = layer(cin, cout, group, seed=cin + group)
    x = torch.randn(B, cin, generator=torch.Generator().manual_seed(B)).to(DTYPES[dtype])
    check(q.step(x.cuda()), x, parts, group)


@pytest.mark.parametrize("zeros,bias", [(False, False), (True, False), (False, True)])
def test_without_zero_points_or_bias(zeros, bias):
    q, parts = layer(200, 70, 64, zeros=zeros, bias=bias)
    x = torch.randn(6, 200, generator=torch.Generator().manual_seed(2))
    check(q.step(x.cuda()), x, parts, 64)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("gates", [1, 2, 3])
def test_weight_is_what_was_given(group, gates):
    for cin, cout in ((1, 6), (130, 30), (257, 96)):
        q, parts = layer(cin, cout, group, gates=gates, seed=cin)
        assert torch.equal(q.weight().double().cpu(), q4_weight(*parts[:3], group))       # 8-bit scale x 5-bit difference: exact


@pytest.mark.parametrize("gates", [2, 3])
def test_gates_give_the_same_product(gates):
    codes, scales, zp = random_q4(gates * 21, 150, 32, 5)
    x = torch.randn(4, 150, generator=torch.Generator().manual_seed(3))
    q, parts = layer(150, gates * 21, 32, gates=gates, seed=5)
    check(q.step(x.cuda()), x, parts, 32)


@pytest.mark.parametrize("code", [0, 15])
def test_ends_of_the_codes(code):
    cin, cout = 160, 32
    codes = torch.full((cout, cin), code, dtype=torch.uint8)
    scales = torch.full((cout, 5), 0.125, dtype=torch.bfloat16)
    zp = torch.full((cout, 5), 15 - code, dtype=torch.uint8)
    q = Q4Linear(cin, cout, "cuda", group_size=32)
    q.set_codes(codes.cuda(), scales.cuda(), zp.cuda())
    x = torch.ones(1, cin)
    assert torch.equal(q.step(x.cuda()).cpu(), torch.full((1, cout), (2 * code - 15) * 0.125 * cin))      # exact in float32


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e6, 1e30])
def test_float32_rows_of_any_magnitude(scale):
    """float32 inputs keep their 24 bits whatever their size."""
    q, parts = layer(257, 40, 64, seed=9, bias=False)
    x = torch.randn(3, 257, generator=torch.Generator().manual_seed(4)) * scale
    check(q.step(x.cuda()), x, parts, 64)


def test_float32_inputs_are_not_rounded():
    """One input of 1 + 2^-23 against one of -1 with the same weight: what is left is the last bit alone."""
    cin = 64
    q = Q4Linear(cin, 16, "cuda", group_size=32)
    q.set_codes(torch.full((16, cin), 9, dtype=torch.uint8).cuda(), torch.ones(16, 2, dtype=torch.bfloat16).cuda())
    x = torch.zeros(1, cin)
    x[0, 0], x[0, 40] = 1 + 2.0 ** -23, -1.0
    # two groups' sums of at most 25 each way, rounded to 24 bits: 2^-19 is their last bit, 2^-23 the answer
    assert float((q.step(x.cuda()).cpu() - 2.0 ** -23).abs().max()) <= 3 * 2.0 ** -19


def test_rounding_of_weights():
    """set_weights: every weight within half a scale (and the rounding of the zero point within the range), the scale a 15th of the
    group's range up to bf16's step."""
    g = torch.Generator().manual_seed(6)
    cout, cin, group = 40, 200, 64
    w = torch.randn(cout, cin, generator=g) * 0.05
    w[3] = 0
    w[4] = 0.25
    w[5] = -torch.rand(cin, generator=g)
    q = Q4Linear(cin, cout, "cuda", group_size=group)
    q.set_weights(w.cuda())
    got = q.weight().cpu()
    for k in range(0, cin, group):
        part, back = w[:, k:k + group], got[:, k:k + group]
        span = part.amax(1).clamp(min=0) - part.amin(1).clamp(max=0)
        # scale <= span / 15 (1 + 2^-7); code and zero point are each off by half a scale at most
        assert ((part - back).abs().amax(1) <= span / 15 * (1 + 2.0 ** -7) * 1.001).all()
    assert not got[3].any()
    assert torch.equal(got[4], torch.full((cin,), float(got[4, 0])))
    q2 = Q4Linear(cin, cout, "cuda", group_size=group)
    q2.set_weights(w[..., None].cuda())
    assert torch.equal(q2.weight().cpu(), got)
    x = torch.randn(2, cin, generator=g)
    near(q.step(x.cuda()), x.double() @ got.double().t(), 1e-4, "y")


def test_bad_codes_are_refused():
    q = Q4Linear(40, 8, "cuda", group_size=32)
    ok = torch.full((8, 40), 3, dtype=torch.uint8, device="cuda")
    s = torch.ones(8, 2, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="not set"):
        q.step(torch.ones(1, 40, device="cuda"))
    bad = ok.clone()
    bad[7, 39] = 16
    with pytest.raises(ValueError, match="over 15"):
        q.set_codes(bad, s)
    with pytest.raises(RuntimeError, match="not set"):
        q.step(torch.ones(1, 40, device="cuda"))
    with pytest.raises(ValueError, match="over 15"):
        q.set_codes(ok, s, torch.full((8, 2), 200, dtype=torch.uint8, device="cuda"))
    w = torch.ones(8, 40, device="cuda")
    w[2, 3] = float("nan")
    with pytest.raises(ValueError, match="not finite"):
        q.set_weights(w)
    q.set_codes(ok, s)
    assert torch.equal(q.step(torch.ones(1, 40, device="cuda")).cpu(), torch.full((1, 8), -5.0 * 40))
    with pytest.raises(RuntimeError, match="not differentiable"):
        q.step(torch.ones(1, 40, device="cuda", requires_grad=True))
    for x, err in ((torch.ones(1, 41, device="cuda"), ValueError), (torch.ones(40, device="cuda"), ValueError),
                   (torch.ones(0, 40, device="cuda"), ValueError), (torch.ones(1, 40, device="cuda", dtype=torch.float64), TypeError),
                   (torch.ones(1, 40), RuntimeError)):
        with pytest.raises(err):
            q.step(x)
    with pytest.raises(ValueError, match="one gate"):
        q.recurrence_step(torch.ones(1, 40, device="cuda"), torch.zeros(1, 8, device="cuda"))


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_strides_of_x(dtype):
    q, parts = layer(200, 48, 64, seed=7)
    x = torch.randn(5, 200, generator=torch.Generator().manual_seed(8)).to(DTYPES[dtype]).cuda()
    want = q.step(x)
    wide = torch.full((5, 215), float("nan"), dtype=x.dtype, device="cuda")
    for off in (0, 1, 4, 8):            # NaN around the rows: nothing but the rows is read into a product
        wide.fill_(float("nan"))
        wide[:, off:off + 200] = x
        assert torch.equal(q.step(wide[:, off:off + 200]), want), off
    assert torch.equal(q.step(x.t().contiguous().t()), want)
    assert torch.equal(q.step(x[:1].expand(5, 200)), q.step(x[:1].expand(5, 200).contiguous()))


def test_nan_stays_in_its_row():
    q, _ = layer(200, 48, 64, seed=7)
    x = torch.randn(20, 200, device="cuda")
    want = q.step(x)
    x[3, 17], x[18, 5] = float("nan"), float("inf")
    got = q.step(x)
    keep = [i for i in range(20) if i not in (3, 18)]
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[3]).all() and not torch.isfinite(got[18]).any()


@pytest.mark.parametrize("cin,cout", [(700, 100), (4100, 40), (260, 2100)])
def test_a_row_does_not_depend_on_its_batch(cin, cout):
    """Whatever form the kernel takes for so many rows (through LDS or not, one tile a wave or two): the same bits."""
    q, _ = layer(cin, cout, 64, seed=8)
    for dt in DTYPES.values():
        x = torch.randn(64, cin, device="cuda").to(dt)
        full = q.step(x)
        for lo, n in ((0, 1), (5, 3), (7, 9), (16, 16), (20, 33)):
            assert torch.equal(q.step(x[lo:lo + n]), full[lo:lo + n]), (dt, lo, n)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("gates", [2, 3])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 128, 128), (8, 80, 20), (3, 130, 33), (17, 512, 64), (48, 257, 50), (70, 64, 16)],
                         ids=lambda s: "x".join(map(str, s)))
def test_recurrence_step(shape, gates, dtype):
    """The fused step against the exact one: errors ez of the gate inputs move keep and the output gate by ez / 4 of |v - h| and |h|,
    and v by ez, on top of the step's own roundings (tests/_ops.py, T = 1)."""
    B, cin, C = shape
    q, parts = layer(cin, gates * C, 32, gates=gates, seed=cin)
    g = torch.Generator().manual_seed(B)
    x, state = (torch.randn(B, cin, generator=g) * 0.2).to(DTYPES[dtype]), torch.randn(B, C, generator=g)
    z, ez = exact(x, parts, 32), q4_bound(x, *parts[:3], 32, parts[3])
    f, v = z[:, :C], z[:, C:2 * C]
    h = state.double() * torch.sigmoid(f) + torch.sigmoid(-f) * v
    delta = (1.5 * float(z.abs().max()) + 8) * EPS
    e = float(ez.max())
    M = max(float(v.abs().max()), float(state.abs().max()))
    eh = e * (M / 2 + 1) + (2 * delta + 12 * EPS) * M
    y = h * torch.sigmoid(z[:, 2 * C:]) if gates == 3 else h
    sc = state.cuda()
    got = q.recurrence_step(x.cuda(), sc)
    near(sc, h, eh, "state")
    near(got, y, eh + M * (e / 4 + delta + EPS), "y")


def test_recurrence_step_captured_and_on_two_streams():
    q, _ = layer(128, 3 * 64, 64, gates=3, seed=11)
    x = torch.randn(4, 128, device="cuda")
    state = torch.zeros(4, 64, device="cuda")
    want_state = torch.zeros(4, 64, device="cuda")
    wants = [q.recurrence_step(x, want_state).clone() for _ in range(5)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = q.recurrence_step(x, state)
    state.zero_()
    for w in wants:
        g.replay()
        assert torch.equal(y, w)
        q.step(x)
    assert torch.equal(state, want_state)
    streams = [torch.cuda.Stream() for _ in range(2)]
    states = [torch.zeros(4, 64, device="cuda") for _ in streams]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, st in zip(streams, states):
            with torch.cuda.stream(s):
                q.recurrence_step(x, st)
    torch.cuda.synchronize()
    for st in states:
        assert torch.equal(st, want_state)


def test_weights_are_not_set_while_capturing():
    q, parts = layer(64, 32, 32)
    codes, scales, zp, b = (t.cuda() for t in parts)
    x = torch.randn(2, 64, device="cuda")
    want = q.step(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = q.step(x)
        with pytest.raises(NotImplementedError, match="captured"):
            q.set_codes(codes, scales, zp, b)
    for _ in range(3):
        g.replay()
        assert torch.equal(y, want)


@pytest.mark.parametrize("B", [1, 7, 20])
@pytest.mark.parametrize("gates", [2, 3])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_recurrence_step_with_gates_at_both_ends(dtype, gates, B):
    """All weights are zero, so that the bias alone is z, in float32 for every type of x."""
    f, h, v = gate_ends(torch.float32)
    C = f.numel()
    q = Q4Linear(40, gates * C, "cuda", group_size=32, gates=gates)
    q.set_codes(torch.full((gates * C, 40), 8, dtype=torch.uint8, device="cuda"), torch.ones(gates * C, 2, dtype=torch.bfloat16, device="cuda"), None,
                torch.cat([f, v] + [torch.zeros(C)] * (gates - 2)).cuda())
    state = h.expand(B, C).contiguous().cuda()
    y = q.recurrence_step(torch.randn(B, 40, generator=torch.Generator().manual_seed(1)).to(DTYPES[dtype]).cuda(), state)
    for row in state:
        check_blend(row, f, h, v)
    assert torch.equal(y, (state * (0.5 if gates == 3 else 1.0)).to(y.dtype))


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("shape", [(1, 300, 40), (4, 128, 16), (40, 257, 33), (5, 2100, 20)], ids=lambda s: "x".join(map(str, s)))
def test_finite_inputs_of_any_size(shape, group, dtype):
    """Rows next to the largest number of their type: what is summed on the way overflows where the result does, not before it."""
    B, cin, cout = shape
    codes, scales, zp = random_q4(cout, cin, group, 3)
    scales = (scales.float() * 2.0 ** -10).to(torch.bfloat16)
    q = Q4Linear(cin, cout, "cuda", group_size=group)
    q.set_codes(codes.cuda(), scales.cuda(), zp.cuda())
    g = torch.Generator().manual_seed(B)
    sign = torch.where(torch.rand(B, cin, generator=g) < 0.5, -1.0, 1.0)
    x = (sign * (0.5 + 0.5 * torch.rand(B, cin, generator=g)) * float(torch.finfo(DTYPES[dtype]).max)).to(DTYPES[dtype])
    x[0] = x[0].abs()
    parts = (codes, scales, zp, None)
    want = exact(x, parts, group)
    assert torch.isfinite(x).all()
    assert float(want.abs().max()) < float(torch.finfo(DTYPES[dtype]).max)
    check(q.step(x.cuda()), x, parts, group)
