"""Host-side mirror of the reference's kernel interface, on torch CUDA tensors.

`Backend` owns one library context (device + stream) and exposes one method per function of the
reference's kernel header (src/codegen/utils/kernels.h), same name, same argument meaning, with
tensors in place of raw pointers and shapes taken from the tensors.  Every method only validates,
allocates the output with torch and calls through the C-ABI; all arithmetic happens in the CUDA
library.  torch is used for device memory and streams, nothing else.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L


def _p(t):
    return C.c_void_p(t.data_ptr() if t is not None else 0)


def _dims(seq):
    return (C.c_size_t * len(seq))(*[int(x) for x in seq])


def conv_out_dims(idims, fdims, kernels, strides, pads):
    """Conv2dOp shape inference, src/op/dlOp.cpp:195-196."""
    n, h, w, _ = idims
    return (n, (h + pads[0] + pads[2] - kernels[0]) // strides[0] + 1,
            (w + pads[1] + pads[3] - kernels[1]) // strides[1] + 1, fdims[0])


def pool_out_dims(idims, kernels, strides, pads):
    n, h, w, c = idims
    return (n, (h + pads[0] + pads[2] - kernels[0]) // strides[0] + 1,
            (w + pads[1] + pads[3] - kernels[1]) // strides[1] + 1, c)


class _Norm(C.Structure):
    _fields_ = [("kind", C.c_int), ("weight", C.c_void_p), ("bias", C.c_void_p), ("eps", C.c_float)]


class _NormBlock(C.Structure):
    _fields_ = [("x", C.c_void_p), ("x_dtype", C.c_int), ("ldx", C.c_size_t), ("post", _Norm), ("gate", C.c_void_p),
                ("gate_dtype", C.c_int), ("ld_gate", C.c_size_t), ("gate_rows", C.c_longlong), ("scale", C.c_float),
                ("residual", C.c_void_p), ("residual_dtype", C.c_int), ("ld_residual", C.c_size_t), ("sum", C.c_void_p),
                ("sum_dtype", C.c_int), ("ld_sum", C.c_size_t), ("pre", _Norm), ("y", C.c_void_p), ("y_dtype", C.c_int),
                ("ldy", C.c_size_t)]


class _Attention(C.Structure):
    _fields_ = ([(n, C.c_void_p) for n in ("q", "k", "v", "o", "lse")] +
                [(n, C.c_size_t) for n in ("q_row", "q_head", "k_row", "k_head", "v_row", "v_head", "o_row", "o_head")] +
                [(n, C.c_int) for n in ("batch", "total_q", "total_k", "heads_q", "heads_kv", "head_dim")] +
                [(n, C.c_void_p) for n in ("q_offsets", "k_offsets", "k_lens")] +
                [("scale", C.c_float), ("causal", C.c_int), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)])


class _FcEpilogue(C.Structure):
    _fields_ = [("bias", C.c_void_p), ("act", C.c_int), ("scale", C.c_float), ("residual", C.c_void_p),
                ("residual_dtype", C.c_int), ("ld_residual", C.c_int)]


class Backend:
    def __init__(self, device: int | torch.device = 0, precision: int = L.STRICT_F32, own_stream: bool = False,
                 stream: "torch.cuda.Stream | None" = None):
        """Work is issued on `stream` if given, else on torch's current stream of the device (own_stream=True:
        on a stream the library creates, which torch knows nothing about -- synchronise with `sync()`)."""
        if not torch.cuda.is_available():
            raise RuntimeError("swcompiler_b200 needs a CUDA device; there is no CPU path")
        self.lib = L.lib()
        self.device = torch.device("cuda", device if isinstance(device, int) else device.index or 0)
        self._ctx = C.c_void_p()
        self.torch_stream = None
        with torch.cuda.device(self.device):
            if own_stream:
                rc = self.lib.swcb200_init(C.c_int(self.device.index), C.c_int(precision), C.byref(self._ctx))
            else:
                self.torch_stream = stream if stream is not None else torch.cuda.current_stream(self.device)
                rc = self.lib.swcb200_init_on_stream(C.c_int(self.device.index), C.c_int(precision),
                                                     C.c_void_p(self.torch_stream.cuda_stream), C.byref(self._ctx))
        if rc != L.OK:
            raise L.SwcError(rc, "swcb200_init")
        self.precision = precision

    # ---- plumbing -----------------------------------------------------------
    def close(self):
        if self._ctx:
            self.lib.swcb200_destroy(self._ctx)
            self._ctx = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc: int, what: str):
        if rc != L.OK:
            raise L.SwcError(rc, what, self.lib.swcb200_last_error(self._ctx).decode())

    def _call(self, name: str, *args):
        self._check(getattr(self.lib, "swcb200_" + name)(self._ctx, *args), name)

    def sync(self):
        self._call("sync")

    def set_wait_limit(self, cycles: int):
        """Limit, in SM clock cycles, of every wait inside the tensor-core kernels launched through this context."""
        self._call("set_wait_limit", C.c_longlong(cycles))

    def set_sm_limit(self, sms: int):
        """The persistent tensor-core kernels of this context take at most `sms` SMs (0 = all): leaves room for a
        collective of another stream to run beside them."""
        self._call("set_sm_limit", C.c_int(sms))

    def selftest_wait_timeout(self):
        """Launches a kernel whose bounded wait can only run out; `sync()` then raises with status ERR_TIMEOUT."""
        self._call("selftest_wait_timeout")

    def _issue_stream(self):
        if self.torch_stream is None:
            return torch.cuda.ExternalStream(self.lib.swcb200_stream(self._ctx), self.device)
        return self.torch_stream

    def set_precision(self, precision: int):
        self._call("set_precision", C.c_int(precision))
        self.precision = precision

    @property
    def launches(self) -> int:
        return int(self.lib.swcb200_launch_count(self._ctx))

    def _f32(self, *ts):
        for t in ts:
            if t is None:
                continue
            if not (t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()):
                raise ValueError("expected a contiguous fp32 CUDA tensor")

    def _on_device(self, what, *ts):
        for t in ts:
            if t is not None and t.device != self.device:
                raise ValueError(f"{what}: expected a tensor on {self.device}, got one on {t.device}")

    def _rows(self, what, *ts):
        """[rows, cols] tensors, fp32 or bf16, each row contiguous, at any row pitch."""
        self._on_device(what, *ts)
        for t in ts:
            if t is None:
                continue
            if t.dim() != 2 or t.dtype not in (torch.float32, torch.bfloat16):
                raise ValueError(f"{what}: expected a 2-D fp32 or bf16 tensor")
            if t.numel() and ((t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1])):
                raise ValueError(f"{what}: expected contiguous rows that do not overlap, got strides {t.stride()}")

    def _vector(self, what, t, n):
        self._on_device(what, t)
        if t is not None and (t.dtype != torch.float32 or t.shape != (n,) or not t.is_contiguous()):
            raise ValueError(f"{what}: expected a contiguous fp32 tensor of {n} elements")

    @staticmethod
    def _ld(t):
        return 0 if t is None else t.stride(0) if t.shape[0] > 1 else t.shape[1]

    @staticmethod
    def _dt(t):
        return L.F32 if t is None or t.dtype == torch.float32 else L.BF16

    def _new(self, shape, dtype=torch.float32):
        return torch.empty(tuple(int(s) for s in shape), dtype=dtype, device=self.device)

    # ---- dense --------------------------------------------------------------
    def matrixMatrixMul_f(self, a, b, out=None):
        self._f32(a, b)
        (m, k), (k2, n) = a.shape, b.shape
        if k != k2:
            raise ValueError("inner dimensions differ")
        c = out if out is not None else self._new((m, n))
        self._call("matrixMatrixMul_f", C.c_int(m), C.c_int(n), C.c_int(k), _p(a), C.c_int(k), _p(b), C.c_int(n),
                   _p(c), C.c_int(n))
        return c

    def batchedadd_f(self, batch, slice_, out=None):
        self._f32(batch, slice_)
        rows, cols = batch.shape
        out = out if out is not None else torch.empty_like(batch)
        self._call("batchedadd_f", _p(out), _p(batch), _p(slice_), C.c_size_t(rows), C.c_size_t(cols))
        return out

    def matrixTanh_f(self, a, out=None):
        self._f32(a)
        m, n = a.shape
        out = out if out is not None else torch.empty_like(a)
        self._call("matrixTanh_f", C.c_int(m), C.c_int(n), _p(a), C.c_int(n), _p(out), C.c_int(n))
        return out

    def matrixSoftmax_f(self, a, out=None):
        self._f32(a)
        m, n = a.shape
        out = out if out is not None else torch.empty_like(a)
        self._call("matrixSoftmax_f", C.c_int(m), C.c_int(n), _p(a), C.c_int(n), _p(out), C.c_int(n))
        return out

    def argMax_i(self, a, top_k: int):
        self._f32(a)
        m, n = a.shape
        idx = self._new((m, top_k), torch.int32)
        self._call("argMax_i", _p(a), _p(idx), C.c_int(m), C.c_int(n), C.c_int(top_k))
        return idx

    def accuracy_i(self, pred, label, accum=None):
        """accum [2] int32 += (rows whose label is among their predictions pred[i, :], rows); a fresh zeroed
        counter pair if `accum` is None."""
        m, n = pred.shape
        if accum is None:
            accum = torch.zeros(2, dtype=torch.int32, device=self.device)
            if self.torch_stream is None:  # the library's own stream knows nothing of torch's fill kernel
                torch.cuda.current_stream(self.device).synchronize()
        self._call("accuracy_i", _p(pred), _p(label), _p(accum), C.c_int(m), C.c_int(n))
        return accum

    def relu_f(self, a, out=None):
        self._f32(a)
        out = out if out is not None else torch.empty_like(a)
        self._call("relu_f", _p(a), _p(out), C.c_size_t(a.numel()))
        return out

    def vecAdd_f(self, a, b, out=None):
        self._f32(a, b)
        out = out if out is not None else torch.empty_like(a)
        self._call("vecAdd_f", C.c_int(a.numel()), _p(a), _p(b), _p(out))
        return out

    # ---- NHWC ---------------------------------------------------------------
    def conv2d_f(self, x, filt, bias, kernels, strides, pads, group=1, out=None):
        self._f32(x, filt, bias)
        odims = conv_out_dims(x.shape, filt.shape, kernels, strides, pads)
        out = out if out is not None else self._new(odims)
        self._call("conv2d_f", _p(out), _p(x), _p(filt), _p(bias), _dims(odims), _dims(x.shape), _dims(filt.shape),
                   _dims(bias.shape), _dims(kernels), _dims(strides), _dims(pads), C.c_size_t(group))
        return out

    def maxpool_f(self, x, kernels, strides, pads, out=None):
        self._f32(x)
        odims = pool_out_dims(x.shape, kernels, strides, pads)
        out = out if out is not None else self._new(odims)
        self._call("maxpool_f", _p(x), _p(out), _dims(x.shape), _dims(odims), _dims(kernels), _dims(strides),
                   _dims(pads))
        return out

    def avgpool_f(self, x, kernels, strides, pads, out=None):
        self._f32(x)
        odims = pool_out_dims(x.shape, kernels, strides, pads)
        out = out if out is not None else self._new(odims)
        self._call("avgpool_f", _p(x), _p(out), _dims(x.shape), _dims(odims), _dims(kernels), _dims(strides),
                   _dims(pads))
        return out

    def batchnormalization_f(self, x, mean, var, scale, bias, eps, out=None):
        self._f32(x, mean, var, scale, bias)
        out = out if out is not None else torch.empty_like(x)
        self._call("batchnormalization_f", _p(out), _p(x), _p(mean), _p(var), _p(scale), _p(bias), _dims(x.shape),
                   C.c_float(eps))
        return out

    def transpose2d_f(self, x, shuffle):
        self._f32(x)
        odims = tuple(x.shape[s] for s in shuffle)
        out = self._new(odims)
        self._call("transpose2d_f", _p(x), _p(out), _dims(x.shape), _dims(odims), _dims(shuffle))
        return out

    def transpose4d_f(self, x, shuffle):
        self._f32(x)
        odims = tuple(x.shape[s] for s in shuffle)
        out = self._new(odims)
        self._call("transpose4d_f", _p(x), _p(out), _dims(x.shape), _dims(odims), _dims(shuffle))
        return out

    # ---- chains as the lowered graph has them ---------------------------------
    def fc(self, x, w, b=None):
        """MatrixMatrixMul then MatrixVectorAdd (src/op/dlOp/dlOpEinsum.cpp:154-237); a 4-D NHWC input is
        viewed as [N, H*W*C] (src/tensor/tensor.cpp:128-138)."""
        y = self.matrixMatrixMul_f(x.reshape(x.shape[0], -1), w)
        return y if b is None else self.batchedadd_f(y, b)

    def mlp_forward(self, x, w0, b0, w1, b1):
        return self.matrixSoftmax_f(self.fc(self.matrixTanh_f(self.fc(x, w0, b0)), w1, b1))

    # ---- bf16 storage / tensor-core path ---------------------------------------
    def cast_f32_to_bf16(self, x, out=None):
        self._f32(x)
        out = out if out is not None else self._new(x.shape, torch.bfloat16)
        self._call("cast_f32_to_bf16", _p(x), _p(out), C.c_size_t(x.numel()))
        return out

    def cast_bf16_to_f32(self, x, out=None):
        out = out if out is not None else self._new(x.shape, torch.float32)
        self._call("cast_bf16_to_f32", _p(x), _p(out), C.c_size_t(x.numel()))
        return out

    def pack_weight_bf16(self, w):
        """fp32 W[k, n] -> bf16 Wp[n, k]."""
        self._f32(w)
        k, n = w.shape
        wp = self._new((n, k), torch.bfloat16)
        self._call("pack_weight_bf16", _p(w), C.c_int(k), C.c_int(n), C.c_int(n), _p(wp))
        return wp

    def fc_bf16(self, a, wp, bias=None, act=L.ACT_NONE, out_dtype=torch.bfloat16, out=None, a_lo=None, out_lo=None):
        """act(A[m,k] . Wp[n,k]^T + bias) in one launch; A, Wp bf16.  With `a_lo` the input is a split activation
        (A = a + a_lo, two bf16 terms); with `out_lo` (bf16 outputs) the output's second term is written there."""
        if a.dtype != torch.bfloat16 or wp.dtype != torch.bfloat16 or not (a.is_contiguous() and wp.is_contiguous()):
            raise ValueError("fc_bf16 wants contiguous bf16 operands")
        (m, k), (n, k2) = a.shape, wp.shape
        if k != k2:
            raise ValueError("inner dimensions differ")
        out = out if out is not None else self._new((m, n), out_dtype)
        dt = C.c_int(L.BF16 if out.dtype == torch.bfloat16 else L.F32)
        if a_lo is None and out_lo is None:
            self._call("fc_bf16", C.c_int(m), C.c_int(n), C.c_int(k), _p(a), C.c_int(k), _p(wp), C.c_int(k), _p(bias),
                       C.c_int(act), _p(out), dt, C.c_int(n))
            return out
        for t in (a_lo, out_lo):
            if t is not None and not (t.dtype == torch.bfloat16 and t.is_contiguous()):
                raise ValueError("the second term of a split activation is a contiguous bf16 tensor")
        if (a_lo is not None and a_lo.shape != a.shape) or (out_lo is not None and out_lo.shape != out.shape):
            raise ValueError("the two terms of a split activation have the same shape")
        self._call("fc_bf16_split", C.c_int(m), C.c_int(n), C.c_int(k), _p(a), _p(a_lo), C.c_int(k), _p(wp), C.c_int(k),
                   _p(bias), C.c_int(act), _p(out), _p(out_lo), dt, C.c_int(n))
        return out

    def fc_bf16_scatter_rows(self, a, wp, slot_table, nranks: int, rank: int, ld_slot: int):
        """A[m,k] . Wp[n,k]^T with fp32 rows scattered to the ranks that own them: row i goes into slot `rank` of the
        slot array of rank i // (m // nranks) (`slot_table` from `NcclComm.peer_slots_setup`)."""
        if a.dtype != torch.bfloat16 or wp.dtype != torch.bfloat16 or not (a.is_contiguous() and wp.is_contiguous()):
            raise ValueError("fc_bf16_scatter_rows wants contiguous bf16 operands")
        (m, k), (n, k2) = a.shape, wp.shape
        if k != k2:
            raise ValueError("inner dimensions differ")
        self._call("fc_bf16_scatter_rows", C.c_int(m), C.c_int(n), C.c_int(k), _p(a), C.c_int(k), _p(wp), C.c_int(k),
                   slot_table, C.c_int(nranks), C.c_int(rank), C.c_int(ld_slot))

    def sum_slots(self, slots, out):
        """out = slots[0] + slots[1] + ... in that order; slots [p, ...] fp32 contiguous, out one slot's shape."""
        self._f32(slots, out)
        n = out.numel()
        self._call("sum_slots", _p(slots), C.c_size_t(n), C.c_int(slots.shape[0]), _p(out), C.c_size_t(n))
        return out

    def pack_filter_bf16(self, filt):
        """fp32 filter [oC, kh, kw, iC] -> bf16, same layout."""
        self._f32(filt)
        fp = self._new(filt.shape, torch.bfloat16)
        self._call("pack_filter_bf16", _p(filt), _dims(filt.shape), _p(fp))
        return fp

    def conv2d_bf16(self, x, fp, bias, kernels, strides, pads, bn=None, residual=None, relu=False, out=None, pool=False):
        """Conv2d [-> BatchNormalization] [-> ElementAdd(residual)] [-> Relu] [-> MaxPool 2x2/2] in one tensor-core
        launch.  x, fp (packed filter), residual, out: bf16 NHWC.  bn = (scale, bias, mean, var, eps) or None.
        With `pool` the result is [N, OH/2, OW/2, oC] (3x3 filters over 64 -> 64 channels only)."""
        odims = conv_out_dims(x.shape, fp.shape, kernels, strides, pads)
        out_shape = (odims[0], odims[1] // 2, odims[2] // 2, odims[3]) if pool else odims
        out = out if out is not None else self._new(out_shape, torch.bfloat16)

        class Ep(C.Structure):
            _fields_ = [("bn_scale", C.c_void_p), ("bn_bias", C.c_void_p), ("bn_mean", C.c_void_p),
                        ("bn_var", C.c_void_p), ("bn_eps", C.c_float), ("residual", C.c_void_p), ("relu", C.c_int),
                        ("pool2x2", C.c_int)]

        ep = Ep()
        if bn is not None:
            ep.bn_scale, ep.bn_bias, ep.bn_mean, ep.bn_var = (t.data_ptr() for t in bn[:4])
            ep.bn_eps = float(bn[4])
        ep.residual = residual.data_ptr() if residual is not None else None
        ep.relu = 1 if relu else 0
        ep.pool2x2 = 1 if pool else 0
        self._call("conv2d_bf16", _p(out), _p(x), _p(fp), _p(bias), _dims(odims), _dims(x.shape), _dims(fp.shape),
                   _dims(kernels), _dims(strides), _dims(pads), C.byref(ep))
        return out

    def maxpool_bf16(self, x, kernels, strides, pads, out=None):
        odims = pool_out_dims(x.shape, kernels, strides, pads)
        out = out if out is not None else self._new(odims, torch.bfloat16)
        self._call("maxpool_bf16", _p(x), _p(out), _dims(x.shape), _dims(odims), _dims(kernels), _dims(strides),
                   _dims(pads))
        return out

    # ---- transformer blocks -----------------------------------------------------
    def fc_bf16_residual(self, a, wp, bias=None, act=L.ACT_NONE, residual=None, scale=1.0, out_dtype=torch.bfloat16, out=None):
        """residual + scale * act(A[m,k] . Wp[n,k]^T + bias) in one launch.  A, Wp bf16, rows at any pitch that is a multiple
        of 8; bias fp32 [n]; residual and `out` [m, n] fp32 or bf16, which may be one tensor.  All six activations."""
        self._rows("fc_bf16_residual", a, wp, residual, out)
        if a.dtype != torch.bfloat16 or wp.dtype != torch.bfloat16:
            raise ValueError("fc_bf16_residual wants bf16 operands")
        (m, k), (n, k2) = a.shape, wp.shape
        if k != k2:
            raise ValueError("inner dimensions differ")
        self._vector("fc_bf16_residual", bias, n)
        out = out if out is not None else self._new((m, n), out_dtype)
        if out.shape != (m, n) or (residual is not None and residual.shape != (m, n)):
            raise ValueError("fc_bf16_residual: residual and out are [m, n]")
        ep = _FcEpilogue(bias.data_ptr() if bias is not None else None, act, scale,
                         residual.data_ptr() if residual is not None else None, self._dt(residual), self._ld(residual))
        pitch = lambda t: -(-t.shape[1] // 8) * 8 if t.shape[0] <= 1 else t.stride(0)  # one row has no pitch of its own
        self._call("fc_bf16_residual", C.c_int(m), C.c_int(n), C.c_int(k), _p(a), C.c_int(pitch(a)), _p(wp), C.c_int(pitch(wp)),
                   C.byref(ep), _p(out), C.c_int(self._dt(out)), C.c_int(self._ld(out)))
        return out

    def norm_residual(self, x, residual=None, post=None, gate=None, gate_rows=0, scale=1.0, pre=None, sum_dtype=None,
                      y_dtype=torch.bfloat16, sum=None, y=None, want_sum=True):
        """What lies between two blocks, in one launch: t = residual + scale * gate * post(x), y = pre(t).

        x, residual [rows, cols] and gate [gates, cols] fp32 or bf16, rows at any pitch.  post and pre are norms
        (kind, weight, bias, eps) with kind NORM_RMS or NORM_LAYER, weight and bias fp32 [cols] or None.  Gate row
        r // gate_rows multiplies row r (gate_rows 0: one gate row for all).  Returns (t, y); t is None without
        want_sum, y without pre.  `sum` (t's tensor) and `y` may be x or residual, which are then overwritten."""
        self._rows("norm_residual", x, residual, gate, sum, y)
        rows, cols = x.shape
        if gate_rows < 0:
            raise ValueError("norm_residual: negative gate_rows")
        if gate is not None and (gate.shape[1] != cols or gate.shape[0] < (-(-rows // gate_rows) if gate_rows else 1)):
            raise ValueError("norm_residual: too few gate rows, or of another width")
        block = _NormBlock()
        for name, n in (("post", post), ("pre", pre)):
            if n is not None:
                kind, weight, bias, eps = n
                self._vector("norm_residual", weight, cols)
                self._vector("norm_residual", bias, cols)
                setattr(block, name, _Norm(kind, weight.data_ptr() if weight is not None else None,
                                           bias.data_ptr() if bias is not None else None, eps))
        if pre is None and y is not None:
            raise ValueError("norm_residual: y goes with the norm that writes it")
        if want_sum and sum is None:
            sum = self._new((rows, cols), sum_dtype or (residual if residual is not None else x).dtype)
        if pre is not None and y is None:
            y = self._new((rows, cols), y_dtype)
        for t in (residual, sum, y):
            if t is not None and t.shape != x.shape:
                raise ValueError("norm_residual: tensors of different shapes")
        block.x, block.x_dtype, block.ldx = x.data_ptr(), self._dt(x), self._ld(x)
        block.gate_rows, block.scale = gate_rows, scale
        for name, ld, t in (("gate", "ld_gate", gate), ("residual", "ld_residual", residual), ("sum", "ld_sum", sum), ("y", "ldy", y)):
            if t is not None:
                setattr(block, name, t.data_ptr())
            setattr(block, name + "_dtype", self._dt(t))
            setattr(block, ld, self._ld(t))
        self._call("norm_residual", C.c_size_t(rows), C.c_int(cols), C.byref(block))
        return sum, y

    def attention_bf16(self, q, k, v, q_offsets, k_offsets, k_lens=None, scale=None, causal=True, out=None, lse=None):
        """softmax(scale * q . k^T) . v over packed sequences.  q [total_q, heads_q, d], k, v [total_k, heads_kv, d] bf16 at any
        row and head strides (multiples of 8), d a multiple of 8 up to 128; q_offsets, k_offsets int32 [batch + 1] on the
        device; k_lens int32 [batch]: only that many of a sequence's key rows are filled.  scale: d ** -0.5 unless given.
        causal: query i of n_q sees keys j <= i + n_k - n_q.  `lse` fp32 [total_q, heads_q] receives the log of each softmax's
        sum.  Rows of `out` that belong to no sequence keep what they held."""
        self._on_device("attention_bf16", q, k, v, q_offsets, k_offsets, k_lens, out, lse)
        for t in (q, k, v, out):
            if t is not None and (t.dim() != 3 or t.dtype != torch.bfloat16 or (t.numel() and t.shape[2] > 1 and t.stride(2) != 1)):
                raise ValueError("attention_bf16: q, k, v and out are bf16 [rows, heads, d] with contiguous d")
        (tq, hq, d), (tk, hkv, dk) = q.shape, k.shape
        if v.shape != k.shape or dk != d or (out is not None and out.shape != q.shape):
            raise ValueError("attention_bf16: q, out [total_q, heads_q, d] and k, v [total_k, heads_kv, d]")
        batch = q_offsets.numel() - 1
        for t, n in ((q_offsets, batch + 1), (k_offsets, batch + 1), (k_lens, batch)):
            if t is not None and (t.dtype != torch.int32 or not t.is_contiguous() or t.dim() != 1 or t.numel() != n or batch < 0):
                raise ValueError("attention_bf16: offsets are contiguous int32 [batch + 1], k_lens [batch]")
        if lse is not None and (lse.dtype != torch.float32 or lse.shape != (tq, hq) or not lse.is_contiguous()):
            raise ValueError("attention_bf16: lse is a contiguous fp32 tensor [total_q, heads_q]")
        out = out if out is not None else self._new(q.shape, torch.bfloat16)
        a = _Attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else None,
                       q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), out.stride(0), out.stride(1),
                       batch, tq, tk, hq, hkv, d, q_offsets.data_ptr(), k_offsets.data_ptr(),
                       k_lens.data_ptr() if k_lens is not None else None, d ** -0.5 if scale is None else scale, int(causal))
        need = C.c_size_t()
        self._call("attention_workspace", C.byref(a), C.byref(need))
        if need.value:
            # from the memory pool of the stream that the kernels run on: handed out again only to work behind them
            with torch.cuda.stream(self._issue_stream()):
                ws = torch.empty(need.value, dtype=torch.uint8, device=self.device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need.value
        self._call("attention_bf16", C.byref(a))
        return out
