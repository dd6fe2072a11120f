"""What the recurrence and the 4-bit products refuse, the C structure against its ctypes mirror, and the oracle's own definition --
without a GPU."""
import ctypes
import os
import shutil
import subprocess
import sys

import pytest
import torch

from tests._ops import oracle_scan, q4_weight, random_q4
from wavenet_vocoder_amd import _lib
from wavenet_vocoder_amd.engine import Q4Linear
from wavenet_vocoder_amd.modules import ResidualRecurrentGLU
from wavenet_vocoder_amd.recurrence import gated_recurrence, gated_recurrence_step

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INC = os.path.join(ROOT, "include")


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="HIP device"):
        gated_recurrence(torch.zeros(1, 2, 6))
    with pytest.raises(RuntimeError, match="HIP device"):
        gated_recurrence_step(torch.zeros(1, 6), torch.zeros(1, 2))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        Q4Linear(64, 64, torch.device("cpu"))
    m = ResidualRecurrentGLU(8, 12, skip_out_channels=4).eval()
    with pytest.raises(RuntimeError, match="HIP device"):
        m(torch.zeros(1, 8, 3))
    with pytest.raises(RuntimeError, match="HIP device"):
        m.incremental_forward(torch.zeros(1, 1, 8))
    with pytest.raises(RuntimeError, match="HIP device"):
        m.quantize_(32).incremental_forward(torch.zeros(1, 1, 8))
    assert sorted(m.state_dict()) == ["conv1x1_in.bias", "conv1x1_in.weight", "conv1x1_out.bias", "conv1x1_out.weight", "conv1x1_skip.bias",
                                      "conv1x1_skip.weight"]


def status(fn, *args):
    st = getattr(_lib.lib(), fn)(*args)
    return st, _lib.lib().wnv_last_error().decode()


def fake(**kw):
    """Arguments that are whole but for what a test changes; the addresses are never looked at: every case is refused before a launch."""
    a = dict(B=1, C=4, T=2, gates=3, dtype=0, z=4096, z_batch_stride=24, z_time_stride=12, y=4096, h_last=4096, saved=4096,
             workspace=4096, dz=4096)
    a.update(kw)
    r = _lib.RecurrenceArgs()
    for k, v in a.items():
        setattr(r, k, v)
    return ctypes.byref(r)


@pytest.mark.parametrize("entry", ["wnv_recurrence_forward", "wnv_recurrence_backward"])
@pytest.mark.parametrize("kw,code", [
    (dict(z=None), 1), (dict(B=0), 1), (dict(T=0), 1), (dict(C=0), 1), (dict(B=-1), 1), (dict(gates=1), 1), (dict(gates=4), 1),
    (dict(dtype=3), 1), (dict(dtype=-1), 1), (dict(B=65536), 5), (dict(C=(1 << 20) + 1), 5), (dict(T=1 << 31), 5),
    (dict(z_batch_stride=-1), 1), (dict(z_time_stride=-12), 1), (dict(h0=4096, h0_batch_stride=-4), 1)])
def test_recurrence_refuses(entry, kw, code):
    st, msg = status(entry, 0, fake(**kw))
    assert st == code and entry in msg, (st, msg)


def test_recurrence_refuses_missing_outputs():
    assert status("wnv_recurrence_forward", 0, None)[0] == 1
    assert status("wnv_recurrence_forward", 0, fake(y=None))[0] == 1
    assert status("wnv_recurrence_forward", 0, fake(h_last=None))[0] == 1
    assert status("wnv_recurrence_forward", -1, fake())[0] == 1
    assert status("wnv_recurrence_backward", 0, fake(saved=None))[0] == 1
    assert status("wnv_recurrence_backward", 0, fake(dz=None))[0] == 1
    assert status("wnv_recurrence_backward", 0, fake(dy=4096, dy_time_stride=-1))[0] == 1
    assert status("wnv_recurrence_step", 0, None, 12, 4096, 4096, 1, 4, 3, 0, None)[0] == 1
    assert status("wnv_recurrence_step", 0, 4096, 12, None, 4096, 1, 4, 3, 0, None)[0] == 1
    assert status("wnv_recurrence_step", 0, 4096, 12, 4096, 4096, 0, 4, 3, 0, None)[0] == 1
    assert status("wnv_recurrence_step", 0, 4096, -12, 4096, 4096, 1, 4, 3, 0, None)[0] == 1
    assert status("wnv_recurrence_step", 0, 4096, 12, 4096, 4096, 1, 4, 3, 9, None)[0] == 1


def test_sizes_of_the_buffers():
    lib = _lib.lib()
    for fn in (lib.wnv_recurrence_saved_bytes, lib.wnv_recurrence_workspace_bytes):
        assert fn(0, 1, 1, 3, 0) == -1 and fn(1, 1, 1, 5, 0) == -1 and fn(1, 1, 1, 3, 7) == -1
        for B, T, C in ((1, 1, 1), (3, 129, 40), (8, 24064, 512), (2, 1 << 20, 8)):
            for gates in (2, 3):
                for dt in (0, 1, 2):
                    assert fn(B, T, C, gates, dt) >= 0


def test_q4_refuses():
    h = ctypes.c_void_p()
    lib = _lib.lib()
    for args, code in (((0, 8, 1, 32, 0), 1), ((8, 0, 1, 32, 0), 1), ((8, 8, 0, 32, 0), 1), ((8, 8, 4, 32, 0), 1), ((8, 8, 3, 32, 0), 1),
                       ((8, 8, 1, 48, 0), 5), ((8, 8, 1, 256, 0), 5), ((8, 8, 1, 32, -1), 1), (((1 << 20) + 1, 8, 1, 32, 0), 5)):
        assert lib.wnv_q4_create(*args, ctypes.byref(h)) == code, args
        assert not h.value
    assert lib.wnv_q4_create(8, 8, 1, 32, 0, None) == 1
    assert lib.wnv_q4_create(40, 9, 3, 32, 0, ctypes.byref(h)) == 0 and h.value
    try:
        assert lib.wnv_q4_step(h, 4096, 40, 4096, 1, 0, None) == 2                 # weights are not set
        assert lib.wnv_q4_recurrence_step(h, 4096, 40, 4096, 4096, 1, 0, None) == 2
        assert lib.wnv_q4_dequantise(h, 4096, None) == 2
        assert lib.wnv_q4_set_codes(h, None, 4096, None, None, None) == 1
        assert lib.wnv_q4_set_weights(h, None, None, None) == 1
        assert lib.wnv_q4_step(None, 4096, 40, 4096, 1, 0, None) == 1
    finally:
        assert lib.wnv_q4_destroy(h) == 0
    assert lib.wnv_q4_destroy(None) == 0


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_the_argument_structure_has_the_layout_of_the_header(tmp_path):
    fields = [n for n, _ in _lib.RecurrenceArgs._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "wnv.h"\nint main(void) {\n'
                   '  printf("%zu\\n", sizeof(wnv_recurrence_args));\n'
                   + "".join(f'  printf("%zu\\n", offsetof(wnv_recurrence_args, {f}));\n' for f in fields)
                   + '  printf("%d %d %d\\n", WNV_F32, WNV_BF16, WNV_F16);\n  return 0;\n}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", INC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()
    assert int(out[0]) == ctypes.sizeof(_lib.RecurrenceArgs)
    assert [int(v) for v in out[1:-1]] == [getattr(_lib.RecurrenceArgs, f).offset for f in fields]
    assert out[-1] == "{float32} {bfloat16} {float16}".format(**_lib.DTYPE)


def test_the_oracle_is_its_definition():
    """Its gradients against torch's own through its own forward formula, in 64 bits; a step by hand."""
    g = torch.Generator().manual_seed(0)
    z, h0 = torch.randn(2, 9, 12, generator=g).double().requires_grad_(), torch.randn(2, 4, generator=g).double().requires_grad_()
    dy, dh = torch.randn(2, 9, 4, generator=g).double(), torch.randn(2, 4, generator=g).double()
    start = torch.tensor([[-1, -1, -1, 3, 3, 3, 6, 6, 6], [0] * 9])
    n = torch.tensor([8, 4])
    h, ys = h0, []
    for t in range(9):
        keep, new, gate = torch.sigmoid(z[:, t, :4]), z[:, t, 4:8], torch.sigmoid(z[:, t, 8:])
        live = (t < n).double()[:, None]
        p = h * (start[:, t] != t).double()[:, None]
        h = live * (keep * p + (1 - keep) * new) + (1 - live) * h
        ys.append(h * gate * live)
    y = torch.stack(ys, 1)
    dz, dh0 = torch.autograd.grad((y, h), (z, h0), (dy, dh))
    o = oracle_scan(z, h0, True, n, start, dy, dh)
    for a, b in ((o["y"], y), (o["h_last"], h), (o["dz"], dz), (o["dh0"], dh0)):
        assert float((a - b.detach()).abs().max()) < 1e-13
    codes, scales, zp = random_q4(3, 70, 32, 1)
    w = q4_weight(codes, scales, zp, 32)
    assert float(w[2, 69]) == float(scales[2, 2]) * (int(codes[2, 69]) - int(zp[2, 2]))


def test_the_package_imports_without_a_gpu_build_of_torch():
    """A torch built for the CPU has none of torch._C's _cuda_* functions."""
    code = ("import torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda_getCurrentRawStream')]:\n"
            "    delattr(torch._C, n)\n"
            "import wavenet_vocoder_amd, wavenet_vocoder_amd.engine, wavenet_vocoder_amd.modules, wavenet_vocoder_amd.recurrence\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


@pytest.mark.parametrize("which", [0, 1])
def test_forward_mode_derivatives_are_refused(which):
    """A dual tensor does not require grad; its tangent has to end in an error, not in an output without one."""
    from torch.autograd import forward_ad

    def duals(*shapes):
        return [forward_ad.make_dual(torch.zeros(s), torch.ones(s)) if i == which else torch.zeros(s) for i, s in enumerate(shapes)]
    layer = Q4Linear.__new__(Q4Linear)
    layer._h, layer._index, layer.cin, layer.channels = ctypes.c_void_p(), -1, 6, 2      # as a handle on the CPU would be, had it one
    with forward_ad.dual_level():
        for call in (lambda: gated_recurrence(*duals((1, 3, 6), (1, 2))), lambda: gated_recurrence_step(*duals((1, 6), (1, 2))),
                     lambda: layer.recurrence_step(*duals((1, 6), (1, 2)))) + (() if which else (lambda: layer.step(*duals((1, 6))),)):
            with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
                call()
