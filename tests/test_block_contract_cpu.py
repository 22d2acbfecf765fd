"""CPU: arguments that the transformer-block calls must not let through to the library."""
import ctypes as C
import glob
import os
import re

import pytest
import torch

import swcompiler_b200 as swc
from swcompiler_b200 import _lib as L
from swcompiler_b200 import kernels as K

BF16, F32 = torch.bfloat16, torch.float32
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "swcompiler_b200", "csrc")


@pytest.fixture
def be():
    """A Backend without a context, for tensors of no GPU: what it lets through ends at the library's check of the context."""
    b = K.Backend.__new__(K.Backend)
    b.lib, b.device, b._index, b._ctx, b.torch_stream = L.lib(), torch.device("meta"), -1, C.c_void_p(), None
    b._check = lambda rc, what: (_ for _ in ()).throw(swc.SwcError(rc, what))
    return b


def reaches_library(call):
    with pytest.raises(swc.SwcError) as e:
        call()
    assert e.value.status == L.ERR_BAD_ARG


def meta(*shape, dtype=BF16, pitch=None):
    if pitch is None:
        return torch.empty(shape, dtype=dtype, device="meta")
    return torch.empty_strided(shape, (pitch, 1), dtype=dtype, device="meta")


BIG = 1 << 32  # a C int keeps the low 32 bits of what is passed for it


@pytest.mark.parametrize("more", [8, 64])
def test_fc_bf16_residual_sizes_that_a_c_int_cannot_hold(be, more):
    a, wp = meta(4, 64), meta(24, 64)
    reaches_library(lambda: be.fc_bf16_residual(a, wp, residual=meta(4, 24, pitch=(1 << 31) - 1), out=meta(4, 24, pitch=(1 << 31) - 1)))
    for bad in (dict(a=meta(BIG + more, 64)), dict(a=meta(1 << 31, 64)), dict(wp=meta(BIG + more, 64)), dict(a=meta(4, BIG + more), wp=meta(24, BIG + more)),
                dict(a=meta(1, BIG + more), wp=meta(1, BIG + more)), dict(a=meta(4, 64, pitch=BIG + more)), dict(wp=meta(24, 64, pitch=BIG + more)),
                dict(out=meta(4, 24, pitch=BIG + more)), dict(residual=meta(4, 24, pitch=BIG + more)), dict(out=meta(4, 24, pitch=1 << 31))):
        with pytest.raises(ValueError):
            be.fc_bf16_residual(**{**dict(a=a, wp=wp), **bad})


def test_norm_residual_sizes_that_a_c_int_cannot_hold(be):
    rms = (swc.NORM_RMS, None, None, 1e-6)
    reaches_library(lambda: be.norm_residual(meta(4, 24, pitch=BIG + 8), pre=rms))  # a pitch is a size_t
    for cols in (BIG + 8, BIG + 64, 1 << 31):
        with pytest.raises(ValueError):
            be.norm_residual(meta(1, cols), pre=rms)
        with pytest.raises(ValueError):
            be.norm_residual(meta(2, cols))


def test_kernels_that_start_early_use_ordinary_loads():
    """A kernel that starts while its predecessor still writes must not read through non-coherent loads, which are for memory that
    nobody writes while the kernel runs: neither by name nor by a const __restrict__ parameter, from which the compiler makes them."""
    early = [f for f in glob.glob(os.path.join(CSRC, "*.cu")) if "swc_after_previous()" in open(f).read()]
    assert len(early) >= 3
    todo, seen = list(early), set()
    while todo:
        path = todo.pop()
        if path in seen:
            continue
        seen.add(path)
        text = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(path).read(), flags=re.S)
        todo += [os.path.join(CSRC, h) for h in re.findall(r'#include "(\w+\.cuh)"', text)]
        found = re.findall(r"__ldg|__ldcs|\.global\.nc|ld_nc|__restrict__", text)
        assert not found, (os.path.basename(path), found)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64, torch.int32])
def test_results_of_other_types_are_refused(be, dtype):
    x, rms = meta(4, 64), (swc.NORM_RMS, None, None, 1e-6)
    for call in (lambda: be.fc_bf16_residual(x, meta(24, 64), out_dtype=dtype), lambda: be.norm_residual(x, pre=rms, sum_dtype=dtype),
                 lambda: be.norm_residual(x, pre=rms, y_dtype=dtype), lambda: be.norm_residual(x, pre=rms, want_sum=False, y_dtype=dtype)):
        with pytest.raises(ValueError):
            call()
