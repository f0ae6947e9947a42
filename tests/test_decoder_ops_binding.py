"""The binding of the operators behind a decoder (no GPU): descriptors as the header lays them out."""
import ctypes
import os
import struct
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DESCRIPTORS = {"exb_norm_desc": ("NormDesc", "@q4i2f7q"), "exb_blocks_desc": ("BlocksDesc", "@q4i3q"), "exb_matmul_desc": ("MatmulDesc", "@q4i5q"),
               "exb_logprobs_desc": ("LogprobsDesc", "@2q4ifi")}


def test_descriptors_are_laid_out_alike(tmp_path):
    """Every field lies where the header has it, in the ctypes structure and in the packed bytes."""
    from excalibur_b200 import capi
    lines = []
    for c_name, (py, fmt) in sorted(DESCRIPTORS.items()):
        lines.append('printf("%%zu", sizeof(%s));' % c_name)
        lines += ['printf(" %%zu", offsetof(%s, %s));' % (c_name, f) for f, _ in getattr(capi, py)._fields_]
        lines.append('printf("\\n");')
    src = tmp_path / "offsets.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "excalibur_b200.h"\nint main(void) {%s return 0; }\n' % "".join(lines))
    exe = str(tmp_path / "offsets")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe])
    out = subprocess.check_output([exe], text=True).strip().split("\n")
    for (c_name, (py, fmt)), line in zip(sorted(DESCRIPTORS.items()), out):
        cls, got = getattr(capi, py), list(map(int, line.split()))
        assert got[0] == ctypes.sizeof(cls) == struct.calcsize(fmt), c_name
        assert got[1:] == [getattr(cls, f).offset for f, _ in cls._fields_], c_name
        values = [i + 1 for i in range(len(cls._fields_))]
        assert struct.pack(fmt, *values) == bytes(cls(*values)), c_name


def test_calls_without_a_context_are_refused():
    from excalibur_b200 import capi
    L = capi.lib()
    d = ctypes.byref(capi.BlocksDesc())
    assert L.exb_quantize_blocks_fwd(None, d, None, None, None, None) == capi.EXB_ERR_BAD_ARG
    assert L.exb_fp8_matmul_fwd(None, d, None, None, None, None, None, None, None) == capi.EXB_ERR_BAD_ARG
    assert L.exb_residual_norm_fwd(None, *[None] * 12) == capi.EXB_ERR_BAD_ARG
    assert L.exb_token_logprobs_fwd(None, d, None, None, None, None, None, None, None) == capi.EXB_ERR_BAD_ARG
    assert "null context" in capi.last_error()


def test_tensor_memory_is_taken_between_the_two_launch_controls():
    """A kernel that holds tensor memory while it waits for the previous one could keep from that one what it still needs: waited for
    first, taken, and only then the next kernel is let in.  No run shows it: the window is a fraction of a microsecond."""
    import re
    text = open(os.path.join(ROOT, "excalibur_b200", "csrc", "fp8_matmul.cu")).read()
    kernels = re.findall(r"__global__ .*?\n}\n", text, re.S)
    assert len(kernels) == 2
    for body in kernels:
        wait, alloc, let_in = (body.index(w) for w in ("pdl_wait();", "ptx::tmem_alloc", "pdl_launch_dependents();"))
        assert wait < alloc < let_in
        assert all(body.count(w) == 1 for w in ("pdl_wait();", "ptx::tmem_alloc", "pdl_launch_dependents();"))
