"""CPU: the transformer-block calls' struct layouts, and what Backend refuses before the library is reached.

The Backend here has no context (there is no GPU) and takes CPU tensors for its own: an argument it refuses raises ValueError, a
call it would make ends at the library's check of the null context."""
import ctypes as C
import os
import struct
import subprocess

import pytest
import torch

import swcompiler_b200 as swc
from swcompiler_b200 import _lib as L
from swcompiler_b200 import kernels as K

BF16, F32 = torch.bfloat16, torch.float32
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def be():
    b = K.Backend.__new__(K.Backend)
    b.lib, b.device, b._index, b._ctx, b.torch_stream = L.lib(), torch.device("cpu"), -1, C.c_void_p(), None
    return b


FIELDS = {
    "swcb200_fc_epilogue": (K._FC_EPILOGUE, ["bias", "act", "scale", "residual", "residual_dtype", "ld_residual"]),
    "swcb200_norm_block": (K._NORM_BLOCK, ["x", "x_dtype", "ldx", "post.kind", "post.weight", "post.bias", "post.eps", "gate", "gate_dtype",
                                           "ld_gate", "gate_rows", "scale", "residual", "residual_dtype", "ld_residual", "sum", "sum_dtype",
                                           "ld_sum", "pre.kind", "pre.weight", "pre.bias", "pre.eps", "y", "y_dtype", "ldy"]),
    "swcb200_attention": (K._ATTENTION, ["q", "k", "v", "o", "lse", "q_row", "q_head", "k_row", "k_head", "v_row", "v_head", "o_row", "o_head",
                                         "batch", "total_q", "total_k", "heads_q", "heads_kv", "head_dim", "q_offsets", "k_offsets", "k_lens",
                                         "scale", "causal", "workspace", "workspace_bytes"]),
}


@pytest.mark.parametrize("name", FIELDS)
def test_packed_structs_are_the_headers(name, tmp_path):
    """Every field at the offset the C compiler gives it."""
    packer, fields = FIELDS[name]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "swc_b200.h"\nint main(void) { printf("%zu", sizeof(' + name + "));\n" +
                   "".join(f'printf(" %zu", offsetof({name}, {f}));\n' for f in fields) + "return 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    size, *offsets = map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split())
    assert packer.size <= size < packer.size + 8
    for i, offset in enumerate(offsets):
        values = [0] * len(fields)
        values[i] = 1
        packed = packer.pack(*values)
        assert next(j for j, byte in enumerate(packed) if byte) in range(offset, offset + 4), fields[i]


def reaches_library(call):
    with pytest.raises(swc.SwcError) as e:
        call()
    assert e.value.status == L.ERR_BAD_ARG


def test_fc_bf16_residual_refusals(be):
    a, wp, bias = torch.zeros(4, 64, dtype=BF16), torch.zeros(24, 64, dtype=BF16), torch.zeros(24)
    be._check = lambda rc, what: (_ for _ in ()).throw(swc.SwcError(rc, what))
    reaches_library(lambda: be.fc_bf16_residual(a, wp, bias, swc.ACT_SILU, residual=torch.zeros(4, 24)))
    for bad in (dict(a=a.float()), dict(wp=wp.float()), dict(a=a[:, :56]), dict(a=a.t()), dict(a=a[0]), dict(bias=bias[:23]),
                dict(bias=bias.to(BF16)), dict(residual=torch.zeros(4, 23)), dict(residual=torch.zeros(4, 24).double()),
                dict(out=torch.zeros(3, 24)), dict(out=torch.zeros(24, 4).t()), dict(residual=torch.zeros(24).expand(4, 24))):
        with pytest.raises(ValueError):
            be.fc_bf16_residual(**{**dict(a=a, wp=wp, bias=bias), **bad})


def test_norm_residual_refusals(be):
    x, w = torch.zeros(4, 24, dtype=BF16), torch.ones(24)
    rms = (swc.NORM_RMS, w, None, 1e-6)
    be._check = lambda rc, what: (_ for _ in ()).throw(swc.SwcError(rc, what))
    reaches_library(lambda: be.norm_residual(x, residual=x.float(), post=rms, gate=torch.ones(2, 24), gate_rows=2, pre=rms))
    for bad in (dict(x=x.double()), dict(x=x.t()), dict(residual=x[:3]), dict(residual=x[:, :23]), dict(gate=torch.ones(1, 24), gate_rows=2),
                dict(gate=torch.ones(2, 23)), dict(gate=torch.ones(2, 24), gate_rows=-1), dict(pre=(swc.NORM_RMS, w[:23], None, 1e-6)),
                dict(pre=(swc.NORM_RMS, w.to(BF16), None, 1e-6)), dict(pre=None, y=torch.zeros(4, 24)), dict(sum=torch.zeros(5, 24)),
                dict(y=torch.zeros(4, 25))):
        with pytest.raises(ValueError):
            be.norm_residual(**{**dict(x=x, pre=rms), **bad})


def test_attention_bf16_refusals(be):
    q, k = torch.zeros(6, 4, 32, dtype=BF16), torch.zeros(9, 2, 32, dtype=BF16)
    off = torch.zeros(3, dtype=torch.int32)
    be._check = lambda rc, what: (_ for _ in ()).throw(swc.SwcError(rc, what))
    good = dict(q=q, k=k, v=k, q_offsets=off, k_offsets=off)
    reaches_library(lambda: be.attention_bf16(**good, k_lens=off[:2], lse=torch.zeros(6, 4)))
    for bad in (dict(q=q.float()), dict(k=k[0]), dict(v=k[:8]), dict(k=k[:, :, :24]), dict(q=q.transpose(1, 2)), dict(q_offsets=off.long()),
                dict(k_offsets=off[:2]), dict(k_lens=off), dict(q_offsets=off[:0], k_offsets=off[:0]), dict(out=torch.zeros(6, 4, 24, dtype=BF16)),
                dict(out=torch.zeros(6, 4, 32)), dict(lse=torch.zeros(4, 6)), dict(lse=torch.zeros(6, 4, dtype=BF16))):
        with pytest.raises(ValueError):
            be.attention_bf16(**{**good, **bad})


def test_null_context_is_refused():
    lib = L.lib()
    assert lib.swcb200_fc_bf16_residual(None, 1, 1, 1, None, 8, None, 8, b"", None, 0, 1) == L.ERR_BAD_ARG
    assert lib.swcb200_norm_residual(None, 1, 1, b"") == L.ERR_BAD_ARG
    assert lib.swcb200_attention_bf16(None, b"") == L.ERR_BAD_ARG
    assert lib.swcb200_attention_workspace(None, b"", C.byref(C.c_size_t())) == L.ERR_BAD_ARG
    assert struct.calcsize("P") == 8
