"""8-bit integers by row, their product and products grouped by expert, without a GPU: descriptors, refusals, the order of launch controls."""
import ctypes
import os
import re
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DESCRIPTORS = {"exb_rows_desc": ("RowsDesc", "@q2i2q"), "exb_int8_desc": ("Int8Desc", "@q4i3q"), "exb_grouped_desc": ("GroupedDesc", "@q6i4q")}


def offsets_agree(descriptors, tmp_path):
    """Every field lies where the header has it, in the ctypes structure and in the packed bytes."""
    from excalibur_b200 import capi
    lines = []
    for c_name, (py, fmt) in sorted(descriptors.items()):
        lines.append('printf("%%zu", sizeof(%s));' % c_name)
        lines += ['printf(" %%zu", offsetof(%s, %s));' % (c_name, f) for f, _ in getattr(capi, py)._fields_]
        lines.append('printf("\\n");')
    src = tmp_path / "offsets.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "excalibur_b200.h"\nint main(void) {%s return 0; }\n' % "".join(lines))
    exe = str(tmp_path / "offsets")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe])
    out = subprocess.check_output([exe], text=True).strip().split("\n")
    for (c_name, (py, fmt)), line in zip(sorted(descriptors.items()), out):
        cls, got = getattr(capi, py), list(map(int, line.split()))
        assert got[0] == ctypes.sizeof(cls) == struct.calcsize(fmt), c_name
        assert got[1:] == [getattr(cls, f).offset for f, _ in cls._fields_], c_name
        values = [i + 1 for i in range(len(cls._fields_))]
        assert struct.pack(fmt, *values) == bytes(cls(*values)), c_name


def test_descriptors_are_laid_out_alike(tmp_path):
    offsets_agree(DESCRIPTORS, tmp_path)


class Fake:
    """A context that no call gets past: the library's own checks come before it is used."""

    def __init__(self):
        self.device = -1                                     # what torch says of a CPU tensor
        self._room = ctypes.create_string_buffer(4096)
        self._h = ctypes.addressof(self._room)


def refusal(call, *args):
    """The library's answer to a call with a descriptor and addresses that nobody reads; without a GPU a call that passes all checks ends at the device."""
    from excalibur_b200 import capi
    rc = getattr(capi.lib(), call)(Fake()._h, *args, None)
    return rc, capi.last_error()


A, W, Y, S, T, B, E = (0x10000000 * i for i in range(1, 8))      # addresses far apart


def grouped(**changed):
    from excalibur_b200 import capi
    d = dict(M=100, N=64, K=48, dtype=capi.EXB_F16, y_dtype=capi.EXB_F16, experts=4, reserved=0, a_stride=48, w_stride=48, expert_stride=64 * 48, y_stride=64)
    at = dict(a=A, sa=None, w=W, sw=None, ends=E, bias=None, y=Y)
    for k, v in changed.items():
        (d if k in d else at)[k] = v
    return refusal("exb_grouped_matmul_fwd", ctypes.byref(capi.GroupedDesc(**d)), *(at[k] for k in ("a", "sa", "w", "sw", "ends", "bias", "y")))


def int8(**changed):
    from excalibur_b200 import capi
    d = dict(M=100, N=64, K=48, y_dtype=capi.EXB_F16, reserved=0, a_stride=48, w_stride=48, y_stride=64)
    at = dict(a=A, sa=S, w=W, sw=T, bias=None, y=Y)
    for k, v in changed.items():
        (d if k in d else at)[k] = v
    return refusal("exb_int8_matmul_fwd", ctypes.byref(capi.Int8Desc(**d)), *(at[k] for k in ("a", "sa", "w", "sw", "bias", "y")))


def rows(**changed):
    from excalibur_b200 import capi
    d = dict(rows=100, C=48, in_dtype=capi.EXB_F16, x_stride=48, q_stride=48)
    at = dict(x=A, q=W, scales=S)
    for k, v in changed.items():
        (d if k in d else at)[k] = v
    return refusal("exb_quantize_rows_fwd", ctypes.byref(capi.RowsDesc(**d)), *(at[k] for k in ("x", "q", "scales")))


BAD, UNSUPPORTED = -1, -2


def _no_gpu():
    import torch
    return not torch.cuda.is_available()


@pytest.mark.skipif(not _no_gpu(), reason="the addresses are not real")
@pytest.mark.parametrize("call", [grouped, int8, rows])
def test_a_good_call_gets_as_far_as_the_device(call):
    assert call()[0] == -3      # EXB_ERR_CUDA: there is none


@pytest.mark.parametrize("call,changed,code", [
    (grouped, dict(dtype=2), BAD), (grouped, dict(dtype=5), BAD), (grouped, dict(y_dtype=1), BAD), (grouped, dict(y_dtype=9), BAD),
    (grouped, dict(M=-1), BAD), (grouped, dict(N=0), BAD), (grouped, dict(K=0), BAD), (grouped, dict(experts=0), BAD), (grouped, dict(experts=1025), UNSUPPORTED),
    (grouped, dict(a=None), BAD), (grouped, dict(w=None), BAD), (grouped, dict(ends=None), BAD), (grouped, dict(y=None), BAD),
    (grouped, dict(sa=S), BAD), (grouped, dict(sw=T), BAD), (grouped, dict(dtype=1), BAD), (grouped, dict(dtype=1, sa=S), BAD),
    (grouped, dict(a_stride=40), BAD), (grouped, dict(w_stride=40), BAD), (grouped, dict(y_stride=63), BAD), (grouped, dict(expert_stride=63 * 48), BAD),
    (grouped, dict(a_stride=52), BAD), (grouped, dict(w_stride=52, expert_stride=64 * 52), BAD), (grouped, dict(expert_stride=64 * 48 + 4), BAD),
    (grouped, dict(a=A + 8), BAD), (grouped, dict(w=W + 8), BAD), (grouped, dict(y=Y + 1), BAD), (grouped, dict(ends=E + 2), BAD), (grouped, dict(bias=B + 2), BAD),
    (grouped, dict(y=A + 64), BAD), (grouped, dict(y=W + 128), BAD), (grouped, dict(y=E), BAD), (grouped, dict(y=W + 48 * 2, expert_stride=1 << 20), BAD),
    (grouped, dict(M=1 << 31), UNSUPPORTED), (grouped, dict(K=1 << 30, a_stride=1 << 30, w_stride=1 << 30), UNSUPPORTED),
    (int8, dict(y_dtype=1), BAD), (int8, dict(M=-1), BAD), (int8, dict(N=0), BAD), (int8, dict(K=0), BAD),
    (int8, dict(K=131072, a_stride=131072, w_stride=131072), UNSUPPORTED),
    (int8, dict(a=None), BAD), (int8, dict(w=None), BAD), (int8, dict(y=None), BAD), (int8, dict(sa=None), BAD), (int8, dict(sw=None), BAD),
    (int8, dict(a_stride=32), BAD), (int8, dict(a_stride=56), BAD), (int8, dict(w_stride=56), BAD), (int8, dict(y_stride=60), BAD),
    (int8, dict(a=A + 4), BAD), (int8, dict(sa=S + 1), BAD), (int8, dict(y=S), BAD), (int8, dict(y=T + 16), BAD), (int8, dict(bias=Y + 4), BAD),
    (rows, dict(in_dtype=1), BAD), (rows, dict(rows=-1), BAD), (rows, dict(C=0), BAD), (rows, dict(x=None), BAD), (rows, dict(q=None), BAD), (rows, dict(scales=None), BAD),
    (rows, dict(x_stride=47), BAD), (rows, dict(q_stride=32), BAD), (rows, dict(q_stride=56), BAD), (rows, dict(q=W + 8), BAD), (rows, dict(x=A + 1), BAD),
    (rows, dict(scales=S + 2), BAD), (rows, dict(q=A + 16), BAD), (rows, dict(scales=W + 64), BAD), (rows, dict(rows=1 << 32), UNSUPPORTED),
])
def test_bad_calls_are_refused(call, changed, code):
    assert call(**changed)[0] == code, changed


@pytest.mark.parametrize("call", [grouped, int8])
def test_no_rows_are_no_error(call):
    assert call(M=0, a=None, w=None, y=None)[0] == 0
    assert rows(rows=0, x=None)[0] == 0


def test_null_contexts_and_descriptors_are_refused():
    from excalibur_b200 import capi
    L, d = capi.lib(), ctypes.byref(capi.GroupedDesc())
    for call, n in (("exb_quantize_rows_fwd", 4), ("exb_int8_matmul_fwd", 7), ("exb_grouped_matmul_fwd", 8)):
        assert getattr(L, call)(None, d, *[None] * n) == BAD
        assert getattr(L, call)(Fake()._h, None, *[None] * n) == BAD
        assert "null context" in capi.last_error()


def test_the_binding_refuses_tensors_that_do_not_fit():
    import torch
    from excalibur_b200 import capi
    capi._torch()
    ctx = Fake()
    i8, f16, f32, i32 = torch.int8, torch.float16, torch.float32, torch.int32

    def z(*shape, dtype=f16):
        return torch.zeros(shape, dtype=dtype)
    for x, kw in [(z(3), {}), (z(3, 4, 5), {}), (z(4, 6).t(), {}), (z(4, 32), dict(q=z(4, 16, dtype=i8))), (z(4, 32), dict(q=z(4, 32))), (z(4, 20), dict(q=z(4, 20, dtype=i8))),
                  (z(4, 32), dict(scales=z(5, dtype=f32))), (z(4, 32), dict(scales=z(4))), (z(4, 32), dict(scales=z(8, dtype=f32)[::2]))]:
        with pytest.raises(capi.ExbError):
            capi.quantize_rows(ctx, x, **kw)
    a, w, sa, sw = z(4, 32, dtype=i8), z(6, 32, dtype=i8), z(4, dtype=f32), z(6, dtype=f32)
    for args, kw in [((z(4, 32), sa, w, sw), {}), ((a, sa, z(6, 32), sw), {}), ((a, sa, z(6, 16, dtype=i8), sw), {}), ((a, z(3, dtype=f32), w, sw), {}),
                     ((a, sa, w, z(6)), {}), ((a, z(4, 1, dtype=f32), w, sw), {}), ((a, sa, w, sw), dict(bias=z(5, dtype=f32))), ((a, sa, w, sw), dict(y=z(4, 5))),
                     ((a, sa, w, sw), dict(y=z(4, 6, dtype=f32))), ((z(4, 40, dtype=i8)[:, :32], sa, w, sw), {})]:
        with pytest.raises(capi.ExbError):
            capi.int8_matmul(ctx, *args, **kw)
    a, w, ends = z(4, 32), z(3, 6, 32), z(3, dtype=i32)
    for args, kw in [((z(4, 32, dtype=f32), z(3, 6, 32, dtype=f32), ends), {}), ((a, z(6, 32), ends), {}), ((a, z(3, 6, 32, dtype=torch.bfloat16), ends), {}),
                     ((a, z(3, 6, 16), ends), {}), ((a, w, z(2, dtype=i32)), {}), ((a, w, z(3, dtype=torch.int64)), {}), ((a, w, z(6, dtype=i32)[::2]), {}),
                     ((a, w, ends), dict(a_scales=z(4, dtype=f32))), ((a, w, ends), dict(bias=z(6, dtype=f32))), ((a, w, ends), dict(bias=z(3, 6))),
                     ((a, w, ends), dict(y=z(4, 7))), ((a, w, ends), dict(out_dtype=capi.EXB_F32, y=z(4, 6))), ((z(4, 36)[:, :32], w, ends), {}),
                     ((a, z(3, 6, 36)[:, :, :32], ends), {}), ((a, z(3, 32, 6).transpose(1, 2), ends), {}),
                     ((a.to(i8), w.to(i8), ends), {}), ((a.to(i8), w.to(i8), ends), dict(a_scales=z(4, dtype=f32))),
                     ((a.to(i8), w.to(i8), ends), dict(a_scales=z(4, dtype=f32), w_scales=z(18, dtype=f32)))]:
        with pytest.raises(capi.ExbError):
            capi.grouped_matmul(ctx, *args, **kw)


def test_tensor_memory_is_taken_between_the_two_launch_controls():
    """As the 8-bit floating point product's: waited for the previous kernel first, tensor memory taken, and only then the next one let in."""
    text = open(os.path.join(ROOT, "excalibur_b200", "csrc", "grouped_matmul.cu")).read()
    kernels = re.findall(r"__global__ .*?\n}\n", text, re.S)
    assert len(kernels) == 2
    for body in kernels:
        wait, alloc, let_in = (body.index(w) for w in ("pdl_wait();", "ptx::tmem_alloc", "pdl_launch_dependents();"))
        assert wait < alloc < let_in
        assert all(body.count(w) == 1 for w in ("pdl_wait();", "ptx::tmem_alloc", "pdl_launch_dependents();"))
