"""GPU: the transformer-block operators against their definitions in 64 bits.

Tolerances count roundings.  eps(t) / 2 is half a step of type t relative to the value.  Sums: a chain of n fp32 additions is off
by at most n * 2^-24 of the sum of magnitudes; tensor-core products add 16 terms at a time, with at most two steps of the running
magnitude each, so k terms are off by at most (k / 16) * 2 * 2^-23 of it."""
import math

import pytest
import torch

import swcompiler_b200 as swc
from swcompiler_b200 import _lib as L

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
ACTS = ["NONE", "RELU", "TANH", "GELU", "GELU_TANH", "SILU"]


@pytest.fixture(scope="module")
def be():
    return swc.Backend(0, swc.TC_BF16)


def gen(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *shape, dtype=F32, s=1.0: (torch.randn(shape, generator=g, device="cuda") * s).to(dtype)


def half_step(t):
    return torch.finfo(t.dtype).eps / 2


def check(got, want, tol):
    """tol: without the rounding to got's type."""
    err = (got.double() - want).abs()
    bad = ~(err <= tol + half_step(got) * (want.abs() + tol))
    assert not bad.any(), (int(bad.sum()), float(err[bad].max()), float(want[bad].abs().max()))


# ------------------------------------------------------------------ fc_bf16_residual

def act64(t, act):
    return {"NONE": lambda: t, "RELU": lambda: t.clamp_min(0), "TANH": lambda: torch.tanh(t), "GELU": lambda: t * torch.special.ndtr(t),
            "GELU_TANH": lambda: 0.5 * t * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3))),
            "SILU": lambda: t * torch.sigmoid(t)}[act]()


def fc_check(got, a, wp, bias, act, residual, scale):
    a, wp = a.double(), wp.double()
    z, mass, k = a @ wp.t(), a.abs() @ wp.abs().t(), a.shape[1]
    if bias is not None:
        z, mass = z + bias.double(), mass + bias.double().abs()
    # no activation is steeper than 1.13; 2^-19: exponential, division and error function in fp32, of a value no larger than |z| + 1
    tol = scale * (1.13 * (k / 16 + 9) * 2 ** -22 * mass + 2 ** -19 * (z.abs() + 1) * (act != "NONE"))
    want = act64(z, act) * scale
    if residual is not None:
        want = want + residual.double()
        tol = tol + 2 ** -24 * (want.abs() + residual.double().abs())
    check(got, want, tol + 2 ** -23 * want.abs())


# sizes around the forms' edges: up to 4 rows; undivided and divided k; tiles of 16 to 256 rows; CTA pairs
@pytest.mark.parametrize("m,n,k", [(1, 1, 8), (1, 1000, 784), (2, 37, 4096), (3, 300, 72), (4, 4096, 520), (5, 33, 64), (16, 128, 4096), (17, 130, 200),
                                   (31, 1000, 1024), (64, 257, 2048), (129, 257, 264), (300, 1000, 4096), (777, 65, 128), (600, 2000, 64),
                                   (2300, 2200, 136), (20000, 264, 72)])
def test_fc_bf16_residual(be, m, n, k):
    rn = gen(m * 31 + n * 7 + k)
    act = ACTS[(m + n + k) % 6]
    a, wp, bias = rn(m, k, dtype=BF16), rn(n, k, dtype=BF16, s=k ** -0.5), rn(n, s=0.3)
    fc_check(be.fc_bf16_residual(a, wp), a, wp, None, "NONE", None, 1.0)
    for rdt, odt in ((BF16, F32), (F32, BF16)):
        r = rn(m, n, dtype=rdt)
        fc_check(be.fc_bf16_residual(a, wp, bias, getattr(swc, "ACT_" + act), residual=r, scale=0.4, out_dtype=odt), a, wp, bias, act, r, 0.4)
    be.sync()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [2, 40, 2500])
def test_fc_bf16_residual_activations(be, m, act):
    """Arguments from deep in the negative tail to far positive, fp32 out."""
    rn = gen(m)
    a, wp = rn(m, 64, dtype=BF16, s=2.0), rn(1500, 64, dtype=BF16, s=0.3)
    fc_check(be.fc_bf16_residual(a, wp, None, getattr(swc, "ACT_" + act), out_dtype=F32), a, wp, None, act, None, 1.0)


@pytest.mark.parametrize("m", [1, 3, 20, 200, 3000])
def test_fc_bf16_residual_pitches(be, m):
    """Odd k and n as columns of wider tensors, at every alignment of the output; what lies beside a row is neither read nor written."""
    rn = gen(m)
    n, k = 301, 93
    wide_a, wide_w = torch.full((m, 104), float("nan"), dtype=BF16, device="cuda"), torch.full((n, 112), float("inf"), dtype=BF16, device="cuda")
    a, wp = wide_a[:, :k], wide_w[:, :k]
    a.copy_(rn(m, k)), wp.copy_(rn(n, k, s=0.1))
    wide_r, wide_c = rn(m, n + 5), torch.full((m, n + 9), 7.0, dtype=BF16, device="cuda")
    r, c = wide_r[:, 2:2 + n], wide_c[:, 3:3 + n]
    assert be.fc_bf16_residual(a, wp, None, swc.ACT_RELU, residual=r, out=c) is c
    fc_check(c, a, wp, None, "RELU", r, 1.0)
    assert (wide_c[:, :3] == 7).all() and (wide_c[:, 3 + n:] == 7).all()


@pytest.mark.parametrize("m", [1, 50, 3000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_fc_bf16_residual_in_place(be, m, dtype):
    rn = gen(5)
    a, wp, r = rn(m, 256, dtype=BF16), rn(700, 256, dtype=BF16, s=0.06), rn(m, 700, dtype=dtype)
    want = be.fc_bf16_residual(a, wp, None, residual=r, out_dtype=dtype)
    assert torch.equal(be.fc_bf16_residual(a, wp, None, residual=r, out=r), want)


def test_fc_bf16_residual_empty_and_refused(be):
    a, wp = torch.zeros(4, 64, dtype=BF16, device="cuda"), torch.zeros(24, 64, dtype=BF16, device="cuda")
    assert be.fc_bf16_residual(a[:0], wp).shape == (0, 24)
    assert be.fc_bf16_residual(a, wp[:0]).shape == (4, 0)
    big = torch.zeros(4, 48, dtype=F32, device="cuda")
    for status, call in ((L.ERR_BAD_ARG, lambda: be.fc_bf16_residual(a, wp, None, 6)),
                         (L.ERR_BAD_ARG, lambda: be.fc_bf16_residual(a, wp, None, -1)),
                         (L.ERR_BAD_ARG, lambda: be.fc_bf16_residual(a, wp, residual=big[:, :24], out=big[:, 8:32])),
                         (L.ERR_MISALIGNED, lambda: be.fc_bf16_residual(a[:, :60].contiguous(), wp[:, :60].contiguous())),
                         (L.ERR_MISALIGNED, lambda: be.fc_bf16_residual(a[:, 1:57], wp[:, 8:])),
                         (L.ERR_BAD_ARG, lambda: be.fc_bf16_residual(a[:, :0], wp[:, :0]))):
        with pytest.raises(swc.SwcError) as e:
            call()
        assert e.value.status == status
    assert be.fc_bf16_residual(a, wp, residual=big[:, :24], out=big[:, 24:]).shape == (4, 24)  # side by side is no overlap
    with pytest.raises(ValueError):
        be.fc_bf16_residual(a.cpu(), wp)


@pytest.mark.parametrize("m", [1, 4, 200])
def test_fc_bf16_residual_refuses_to_overwrite_its_operands(be, m):
    a, wide, room = torch.zeros(m, 64, dtype=BF16, device="cuda"), torch.zeros(m, 128, dtype=BF16, device="cuda"), torch.zeros(m * 64 + 64, device="cuda")
    weights = torch.zeros(64 * 64 + m * 64, dtype=BF16, device="cuda")
    wp = weights[:64 * 64].view(64, 64)
    for args in (dict(a=a, out=a), dict(a=wide[:, :64], out=wide[:, 8:72]), dict(a=a, out=weights[64 * 63:64 * (63 + m)].view(m, 64)),
                 dict(a=a, bias=room[32:96], out=room[:m * 64].view(m, 64))):
        with pytest.raises(swc.SwcError) as e:
            be.fc_bf16_residual(wp=wp, **args)
        assert e.value.status == L.ERR_BAD_ARG
    # side by side is no overlap
    be.fc_bf16_residual(wide[:, :64], wp, bias=room[m * 64:], out=wide[:, 64:])
    be.fc_bf16_residual(a, wp, out=weights[64 * 64:].view(m, 64))
    be.fc_bf16_residual(a, wp, bias=room[m * 64:], out=room[:m * 64].view(m, 64))


# ------------------------------------------------------------------ norm_residual

def norm64(t, tol, norm):
    """norm(t) for t known to tol, and the tolerance of the result."""
    kind, w, b, eps = norm
    cols = t.shape[1]
    w = torch.ones(cols, device="cuda", dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(cols, device="cuda", dtype=torch.float64) if b is None else b.double()
    n = 64 + cols / 32                  # additions that a term of a row sum passes at most: 32 in a thread, then a tree
    u = n * 2 ** -24
    if kind == swc.NORM_LAYER:
        mean = t.mean(1, keepdim=True)
        tol = tol + tol.mean(1, keepdim=True) + u * t.abs().mean(1, keepdim=True) + 2 ** -24 * t.abs()
        t = t - mean
    var = t.square().mean(1, keepdim=True) + eps
    rstd = var.rsqrt()
    # d rstd / rstd = -d var / (2 var);  d var = mean(2 t dt + dt^2) and the sum's own rounding
    rel = (2 * t.abs() * tol + tol * tol).mean(1, keepdim=True) / (2 * var) + u + 4 * 2 ** -24
    y = t * rstd * w
    return y + b, (rstd * tol * w.abs() + y.abs() * rel) * (1 + rel) + 4 * 2 ** -24 * (y.abs() + b.abs())


def norm_check(got, x, residual, post, gate, gate_rows, scale, pre):
    t, tol = x.double(), torch.zeros_like(x, dtype=torch.float64)
    if post:
        t, tol = norm64(t, tol, post)
    f = scale
    if gate is not None:
        rows = torch.arange(x.shape[0], device="cuda")
        f = f * gate.double()[rows // gate_rows if gate_rows else rows * 0]
    t, tol = t * f, (tol + 3 * 2 ** -24 * t.abs()) * (f.abs() if torch.is_tensor(f) else abs(f))
    if residual is not None:
        t = t + residual.double()
        tol = tol + 2 ** -24 * t.abs()
    if got[0] is not None:
        check(got[0], t, tol)
    if pre:
        y, tol = norm64(t, tol, pre)
        check(got[1], y, tol)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (1, 8), (5, 64), (130, 75), (77, 264), (9, 1000), (2, 1003), (40, 1024), (33, 1032), (4, 4096),
                                       (3, 5001), (2, 16384), (1, 16383), (700, 40)])
def test_norm_residual(be, rows, cols):
    rn = gen(rows * 13 + cols)
    w, b = 1 + rn(cols, s=0.2), rn(cols, s=0.2)
    rms, layer = (swc.NORM_RMS, w, None, 1e-5), (swc.NORM_LAYER, w, b, 1e-5)
    per = max(1, rows // 3)
    gates = [rn(-(-rows // per), cols), rn(1, cols, dtype=BF16)]
    for i, (xt, rt, st, yt) in enumerate(((BF16, BF16, BF16, BF16), (BF16, F32, F32, BF16), (F32, F32, BF16, F32), (F32, BF16, F32, BF16))):
        x, r = rn(rows, cols, dtype=xt), rn(rows, cols, dtype=rt, s=2.0)
        post, pre = ((None, rms), (rms, layer), (layer, rms), (layer, layer))[i]
        args = dict(residual=r, post=post, gate=gates[i % 2] if i else None, gate_rows=per if i and i % 2 == 0 else 0, scale=0.7, pre=pre)
        norm_check(be.norm_residual(x, sum_dtype=st, y_dtype=yt, **args), x, **args)
    x = rn(rows, cols)
    none = dict(residual=None, post=None, gate=None, gate_rows=0, scale=1.0)
    norm_check(be.norm_residual(x, pre=layer, want_sum=False), x, **none, pre=layer)                  # a norm alone
    norm_check(be.norm_residual(x, pre=(swc.NORM_RMS, None, b, 0.0), y_dtype=F32), x, **none, pre=(swc.NORM_RMS, None, b, 0.0))
    t, y = be.norm_residual(x, residual=rn(rows, cols))                                               # a sum alone
    assert y is None and t.dtype == F32
    be.sync()


@pytest.mark.parametrize("cols", [96, 97, 2048, 2050])
def test_norm_residual_pitches_and_places(be, cols):
    """Columns of wider tensors at every alignment, sum over the residual and y over x in place."""
    rn = gen(cols)
    rows = 21
    pre = (swc.NORM_RMS, None, None, 1e-6)
    for shift in (0, 1, 8):
        wx, wr = rn(rows, cols + 24, dtype=BF16), rn(rows, cols + 24)
        x, r = wx[:, shift:shift + cols], wr[:, shift:shift + cols]
        keep_x, keep_r = wx.clone(), wr.clone()
        was_x, was_r = x.clone(), r.clone()
        norm_check(be.norm_residual(x, residual=r, pre=pre), was_x, was_r, None, None, 0, 1.0, pre)
        # (aligned copies take the form in chunks of 8, whose row sums add up in another order: compared within the tolerance)
        got = be.norm_residual(x, residual=r, pre=pre, sum=r, y=x)
        assert got[0] is r and got[1] is x
        norm_check(got, was_x, was_r, None, None, 0, 1.0, pre)
        beside = torch.ones(cols + 24, dtype=torch.bool, device="cuda")
        beside[shift:shift + cols] = False
        assert torch.equal(wx[:, beside], keep_x[:, beside]) and torch.equal(wr[:, beside], keep_r[:, beside])


def test_norm_residual_refuses_to_overwrite_its_vectors(be):
    room = torch.zeros(5 * 64, device="cuda")
    x, w = torch.zeros(4, 64, device="cuda"), room[4 * 64 - 8:5 * 64 - 8]
    for norm in ((swc.NORM_LAYER, w, None, 1e-6), (swc.NORM_RMS, None, w, 1e-6)):
        for args in (dict(pre=norm, y=room[:256].view(4, 64)), dict(pre=norm, sum=room[:256].view(4, 64)), dict(post=norm, sum=room[:256].view(4, 64))):
            with pytest.raises(swc.SwcError) as e:
                be.norm_residual(x, **args)
            assert e.value.status == L.ERR_BAD_ARG
    be.norm_residual(x, pre=(swc.NORM_RMS, room[256:], None, 1e-6), y_dtype=F32, sum=room[:256].view(4, 64))  # behind it is no overlap


@pytest.mark.parametrize("rows,cols", [(5, 256), (1, 40), (13, 33), (3, 1000)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_residual_gate_per_row(be, rows, cols, dtype):
    """A gate row for every row, at row counts that leave a CTA's last rows without one; what lies behind the last one may be anything."""
    rn = gen(rows + cols)
    x, room = rn(rows, cols, dtype=BF16), torch.full((rows + 8, cols), float("nan"), dtype=dtype, device="cuda")
    room[:rows] = rn(rows, cols, dtype=dtype)
    args = dict(residual=rn(rows, cols), post=(swc.NORM_RMS, None, None, 1e-6), gate=room[:rows], gate_rows=1, scale=1.0,
                pre=(swc.NORM_LAYER, None, None, 1e-6))
    norm_check(be.norm_residual(x, **args), x, **args)


def test_norm_residual_large_mean_and_constant_rows(be):
    """A layer norm of rows far from zero does not lose the variance; of constant rows it is the bias."""
    rn = gen(3)
    w, b = 1 + rn(512, s=0.1), rn(512)
    layer = (swc.NORM_LAYER, w, b, 1e-5)
    x = rn(20, 512) + 3000
    norm_check(be.norm_residual(x, pre=layer, y_dtype=F32), x, None, None, None, 0, 1.0, layer)
    x = torch.full((3, 512), 4.0, device="cuda")
    assert torch.equal(be.norm_residual(x, pre=layer, y_dtype=F32)[1], b.expand(3, 512))


def test_norm_residual_empty_and_refused(be):
    x = torch.zeros(4, 64, device="cuda")
    pre = (swc.NORM_RMS, None, None, 1e-6)
    t, y = be.norm_residual(x[:0], pre=pre)
    assert t.shape == (0, 64) and y.shape == (0, 64)
    wide = torch.zeros(4, 96, device="cuda")
    for status, call in ((L.ERR_BAD_ARG, lambda: be.norm_residual(x, pre=(3, None, None, 1e-6))),
                         (L.ERR_BAD_ARG, lambda: be.norm_residual(x, pre=(swc.NORM_RMS, None, None, -1.0))),
                         (L.ERR_BAD_ARG, lambda: be.norm_residual(x, pre=(swc.NORM_RMS, None, None, float("nan")))),
                         (L.ERR_BAD_ARG, lambda: be.norm_residual(x, want_sum=False)),
                         (L.ERR_BAD_ARG, lambda: be.norm_residual(wide[:, :64], sum=wide[:, 32:])),
                         (L.ERR_BAD_ARG, lambda: be.norm_residual(x, pre=pre, sum=wide[:, :64], y=wide[:, 16:80])),
                         (L.ERR_TOO_LARGE, lambda: be.norm_residual(torch.zeros(1, 16385, device="cuda")))):
        with pytest.raises(swc.SwcError) as e:
            call()
        assert e.value.status == status


# ------------------------------------------------------------------ attention_bf16

def offsets(lengths, extra=0):
    o = [0]
    for n in lengths:
        o.append(o[-1] + n)
    return torch.tensor([v + extra for v in o], dtype=torch.int32, device="cuda")


def attention64(q, k, v, nq, nk, causal, scale):
    """One sequence: output, its tolerance without the rounding at the end, log-sum."""
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    q, k, v = (t.double().transpose(0, 1) for t in (q, k, v))
    k, v = k.repeat_interleave(hq // hkv, 0), v.repeat_interleave(hq // hkv, 0)
    s = scale * (q @ k.transpose(1, 2))
    ds = scale * (d / 16 + 1) * 2 ** -22 * (q.abs() @ k.abs().transpose(1, 2)) + 2 ** -23 * s.abs()
    if causal:
        hidden = torch.arange(nk, device="cuda") > torch.arange(nq, device="cuda")[:, None] + (nk - nq)
        s, ds = s.masked_fill(hidden, -math.inf), ds.masked_fill(hidden, 0)
    lse = torch.logsumexp(s, 2) if nk else torch.full((hq, nq), -math.inf, device="cuda", dtype=torch.float64)
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0)[..., None])
    top = ds.amax(2, keepdim=True) if nk else torch.zeros(hq, nq, 1, device="cuda", dtype=torch.float64)
    # a weight: rounded to bf16 (2^-8), off by its score's error and by the normaliser's, and by the fp32 exponential (2^-20); sums
    tol = (2 ** -8 + 2 * top + 2 ** -20 + (nk / 16 + 8) * 2 ** -22 + nk * 2 ** -24) * (p @ v.abs()) * 1.01
    return (p @ v).transpose(0, 1), tol.transpose(0, 1), lse.t(), (top[..., 0] + 2 ** -18).t()


def attention_check(be, q, k, v, nq, nk, causal, scale=None, out=None, k_lens=None, k_room=None, first_q=0, **kw):
    """k_room: rows that each sequence owns in k, of which nk are filled."""
    k_room = k_room or nk
    off_q, off_k = offsets(nq, first_q), offsets(k_room)
    lse = torch.full(q.shape[:2], 5.0, device="cuda")
    keep = None if out is None else out.clone()
    got = be.attention_bf16(q, k, v, off_q, off_k, k_lens=k_lens, scale=scale, causal=causal, out=out, lse=lse)
    at_q, at_k = first_q, 0
    for n, m, room in zip(nq, nk, k_room):
        rows = slice(at_q, at_q + n)
        want, tol, ls, ltol = attention64(q[rows], k[at_k:at_k + m], v[at_k:at_k + m], n, m, causal, scale or q.shape[2] ** -0.5)
        check(got[rows], want, tol)
        empty = ls == -math.inf
        assert (got[rows][empty] == 0).all() and torch.equal(lse[rows] == -math.inf, empty)
        err = (lse[rows].double() - ls).abs()[~empty]
        assert (err <= (ltol + 2 ** -21 * ls.abs())[~empty]).all()
        at_q, at_k = at_q + n, at_k + room
    for a, b in ((0, first_q), (at_q, q.shape[0])):  # rows of no sequence
        assert (lse[a:b] == 5).all()
        if keep is not None:
            assert torch.equal(got[a:b], keep[a:b])
    return got


PROMPTS = [  # lengths, heads_q, heads_kv, d
    ([1], 1, 1, 8), ([70], 1, 1, 64), ([128], 2, 2, 128), ([129, 1, 255], 4, 2, 128), ([300, 64, 0, 17], 7, 1, 72), ([513], 8, 1, 40),
    ([200, 31], 48, 1, 16), ([400], 130, 1, 24), ([1000, 3], 3, 3, 128), ([90, 700], 16, 8, 104), ([260], 5, 5, 56)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,hq,hkv,d", PROMPTS)
def test_attention_prompts(be, lengths, hq, hkv, d, causal):
    rn = gen(sum(lengths) + d)
    total = sum(lengths)
    # strided: columns of one projection's output
    t = rn(total, (hq + 2 * hkv) * d + 16, dtype=BF16)
    q = t[:, :hq * d].unflatten(1, (hq, d))
    k, v = (t[:, hq * d + i * hkv * d: hq * d + (i + 1) * hkv * d].unflatten(1, (hkv, d)) for i in (0, 1))
    attention_check(be, q, k, v, lengths, lengths, causal)


# more than 1024 keys per sequence take another form of the kernel
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,hq,hkv,d", [([1025], 2, 2, 64), ([1024], 2, 2, 64), ([2100, 130], 8, 2, 128), ([1500], 7, 1, 72),
                                              ([3000, 0, 520], 6, 3, 40), ([1, 2303, 1700], 4, 1, 96)])
def test_attention_long_prompts(be, lengths, hq, hkv, d, causal):
    rn = gen(sum(lengths) + d)
    q, k, v = rn(sum(lengths), hq, d, dtype=BF16), rn(sum(lengths), hkv, d, dtype=BF16), rn(sum(lengths), hkv, d, dtype=BF16)
    attention_check(be, q, k, v, lengths, lengths, causal)


@pytest.mark.parametrize("flip", [False, True])
def test_attention_long_prompts_scores_far_apart_and_not_finite(be, flip):
    """As the two tests of that below, beyond 1024 keys."""
    rn = gen(19)
    new, n, d = 200, 2300, 64
    q, k, v = rn(new, 2, d, dtype=BF16).abs(), rn(n, 2, d, dtype=BF16).abs(), rn(n, 2, d, dtype=BF16)
    k = (k.float() * torch.linspace(-4, 40, n, device="cuda")[:, None, None]).to(BF16)
    attention_check(be, q, k.flip(0).contiguous() if flip else k, v, [new], [n], False, scale=1.0)
    clean = be.attention_bf16(q, k, v, offsets([new]), offsets([n]), causal=False)
    q[5, 1, 3] = float("nan")
    got = be.attention_bf16(q, k, v, offsets([new]), offsets([n]), causal=False)
    assert got[5, 1].isnan().all() and torch.equal(got[:5], clean[:5]) and torch.equal(got[6:], clean[6:])


@pytest.mark.parametrize("n", [300, 1500])
def test_attention_keys_with_infinite_scores_below(be, n):
    """Keys of score -infinity at the front, more than a block of them, weigh nothing."""
    rn = gen(n)
    new, d = 150, 64
    q, k, v = rn(new, 2, d, dtype=BF16).abs() + 0.1, rn(n, 2, d, dtype=BF16), rn(n, 2, d, dtype=BF16)
    k[:140, 0, :] = float("-inf")  # q > 0: every product is -infinity
    got = be.attention_bf16(q, k, v, offsets([new]), offsets([n]), causal=False)
    want, tol, _, _ = attention64(q[:, :1].contiguous(), k[140:, :1].contiguous(), v[140:, :1].contiguous(), new, n - 140, False, d ** -0.5)
    check(got[:, :1], want, tol)


@pytest.mark.parametrize("nq,nk,hq,hkv,d", [([1], [1], 1, 1, 8), ([1], [64], 4, 1, 128), ([1, 1, 1], [3000, 1, 700], 8, 2, 128), ([1] * 40, list(range(1, 2000, 50)), 8, 1, 64),
                                            ([4, 2], [1500, 2], 16, 2, 72), ([1], [5000], 64, 1, 128), ([1, 1], [900, 1300], 96, 1, 32),
                                            ([3, 0, 30, 1], [600, 5, 400, 0], 4, 4, 128), ([1], [9000], 128, 1, 16)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_few_tokens(be, nq, nk, hq, hkv, d, causal):
    rn = gen(sum(nk) + d)
    attention_check(be, rn(sum(nq), hq, d, dtype=BF16), rn(sum(nk), hkv, d, dtype=BF16), rn(sum(nk), hkv, d, dtype=BF16), nq, nk, causal)


@pytest.mark.parametrize("nq,nk", [([70], [4000]), ([40, 90], [3000, 2100]), ([300], [100]), ([65], [0]), ([20, 100], [7, 33])])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_chunks(be, nq, nk, d):
    """New tokens behind (or more than) the keys: divided keys, and rows that the mask leaves nothing."""
    rn = gen(sum(nk) + d)
    attention_check(be, rn(sum(nq), 8, d, dtype=BF16), rn(sum(nk), 2, d, dtype=BF16), rn(sum(nk), 2, d, dtype=BF16), nq, nk, True)


@pytest.mark.parametrize("new", [1, 100])
def test_attention_unfilled_cache_rows_may_hold_anything(be, new):
    rn = gen(new)
    nk, room, hkv, d = [130, 1000, 101, 100], [1024] * 4, 2, 128
    q = rn(4 * new + 5, 8, d, dtype=BF16)
    k, v = (torch.full((sum(room) + 3, hkv, d), x, dtype=BF16, device="cuda") for x in (float("nan"), float("inf")))
    for i, n in enumerate(nk):
        k[i * 1024:i * 1024 + n], v[i * 1024:i * 1024 + n] = rn(n, hkv, d, dtype=BF16), rn(n, hkv, d, dtype=BF16)
    out = torch.full_like(q, 3.0)
    lens = torch.tensor(nk, dtype=torch.int32, device="cuda")
    attention_check(be, q, k, v, [new] * 4, nk, True, out=out, k_lens=lens, k_room=room, first_q=2)


@pytest.mark.parametrize("new", [1, 200])
def test_attention_scores_far_apart(be, new):
    """Scores that grow along the keys, so that the maximum is replaced block after block, and ones beyond what exp takes."""
    rn = gen(9)
    n, d = 900, 64
    q, k, v = rn(new, 2, d, dtype=BF16).abs(), rn(n, 2, d, dtype=BF16).abs(), rn(n, 2, d, dtype=BF16)
    k = (k.float() * torch.linspace(-4, 40, n, device="cuda")[:, None, None]).to(BF16)
    for order in (k, k.flip(0)):
        attention_check(be, q, order.contiguous(), v, [new], [n], False, scale=1.0)


@pytest.mark.parametrize("new", [1, 200])
def test_attention_non_finite_inputs(be, new):
    """A NaN or an infinite score reaches its own row and head only."""
    rn = gen(2)
    n, d = 500, 128
    q, k, v = rn(new, 2, d, dtype=BF16), rn(n, 1, d, dtype=BF16), rn(n, 1, d, dtype=BF16)
    clean = be.attention_bf16(q, k, v, offsets([new]), offsets([n]), causal=False)
    q[0, 1, 3] = float("nan")
    got = be.attention_bf16(q, k, v, offsets([new]), offsets([n]), causal=False)
    assert got[0, 1].isnan().all() and torch.equal(got[0, 0], clean[0, 0]) and torch.equal(got[1:], clean[1:])
    q[0, 1, 3] = float("inf")
    got = be.attention_bf16(q, k, v, offsets([new]), offsets([n]), causal=False)
    assert got[0, 1].isnan().all() and torch.equal(got[0, 0], clean[0, 0])
    be.sync()


@pytest.mark.parametrize("new", [1, 150])
def test_attention_wrong_offsets_stay_inside(be, new):
    """Offsets beyond the tensors are clamped to them: nothing outside is touched, the good sequence's rows are right."""
    rn = gen(4)
    q, k, v = rn(2 * new, 4, 64, dtype=BF16), rn(300, 2, 64, dtype=BF16), rn(300, 2, 64, dtype=BF16)
    off_q = torch.tensor([0, new, 1 << 30], dtype=torch.int32, device="cuda")
    off_k = torch.tensor([0, 300, 1 << 30], dtype=torch.int32, device="cuda")
    got = be.attention_bf16(q, k, v, off_q, off_k, causal=False)
    want, tol, _, _ = attention64(q[:new], k, v, new, 300, False, 0.125)
    check(got[:new], want, tol)
    assert (got[new:] == 0).all()  # the second one has no keys
    back = torch.tensor([2 * new, -5, 7], dtype=torch.int32, device="cuda")
    be.attention_bf16(q, k, v, back, back)
    be.sync()


@pytest.mark.parametrize("new", [1, 150])
def test_attention_extreme_offsets(be, new):
    """The least and largest integers as offsets and lengths: sequences of nothing, or up to the tensors' ends."""
    rn = gen(14)
    q, k, v = rn(2 * new, 4, 64, dtype=BF16), rn(300, 2, 64, dtype=BF16), rn(300, 2, 64, dtype=BF16)
    low, high = -(1 << 31), (1 << 31) - 1
    at = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    want, tol, _, _ = attention64(q[:new], k, v, new, 300, False, 0.125)
    out = torch.full_like(q, 7)
    be.attention_bf16(q, k, v, at(0, new, low), at(low, high, low), causal=False, out=out)  # (the second one: no rows)
    check(out[:new], want, tol)
    assert (out[new:] == 7).all()
    out = torch.full_like(q, 7)
    be.attention_bf16(q, k, v, at(new, low, new), at(200, low, 300), causal=False, out=out)  # no rows; rows 0 .. new, all keys
    check(out[:new], want, tol)
    assert (out[new:] == 7).all()
    out = be.attention_bf16(q, k, v, at(0, new, high), at(0, 300, low), k_lens=at(high, low), causal=False)
    check(out[:new], want, tol)
    assert (out[new:] == 0).all()


@pytest.mark.parametrize("new", [1, 5])
def test_attention_sequences_that_overlap_stay_inside(be, new):
    """Offsets that name the same rows again and again ask for more pieces of work than the workspace has room for; the call after
    it is not harmed."""
    rn = gen(15)
    n = 200 * new
    q, k, v = rn(n, 8, 64, dtype=BF16), rn(4000, 2, 64, dtype=BF16), rn(4000, 2, 64, dtype=BF16)
    off = torch.zeros(201, dtype=torch.int32, device="cuda")
    for rows in (new, n):  # every second sequence has the same rows and all keys
        off_q, off_k = off.clone(), off.clone()
        off_q[1::2], off_k[1::2] = rows, 4000
        be.attention_bf16(q, k, v, off_q, off_k, causal=False)
    be.sync()
    got = be.attention_bf16(q[:new], k, v, offsets([new]), offsets([4000]), causal=False)
    want, tol, _, _ = attention64(q[:new], k, v, new, 4000, False, 0.125)
    check(got, want, tol)


def test_attention_lengths_change_under_a_graph():
    """One captured call, replayed for other lengths; a second graph in flight has a workspace of its own."""
    s = torch.cuda.Stream()
    rn = gen(6)
    with torch.cuda.stream(s):
        be = swc.Backend(0, swc.TC_BF16, stream=s)
        q, k, v = rn(3, 8, 128, dtype=BF16), rn(3 * 2048, 2, 128, dtype=BF16), rn(3 * 2048, 2, 128, dtype=BF16)
        lens = torch.tensor([5, 2048, 700], dtype=torch.int32, device="cuda")
        off_q, off_k = offsets([1] * 3), offsets([2048] * 3)
        be.attention_bf16(q, k, v, off_q, off_k, k_lens=lens)
        s.synchronize()
        graphs, outs = [], []
        for _ in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=s):
                outs.append(be.attention_bf16(q, k, v, off_q, off_k, k_lens=lens))
        other = torch.cuda.Stream()
        for nk in ([5, 2048, 700], [2048, 1, 0], [64, 65, 2047]):
            lens.copy_(torch.tensor(nk, dtype=torch.int32))
            other.wait_stream(s)
            graphs[0].replay()
            with torch.cuda.stream(other):
                graphs[1].replay()
            s.wait_stream(other)
            for i, n in enumerate(nk):
                rows = slice(i * 2048, i * 2048 + n)
                want, tol, _, _ = attention64(q[i:i + 1], k[rows], v[rows], 1, n, True, 128 ** -0.5)
                check(outs[0][i:i + 1], want, tol)
            assert torch.equal(outs[0], outs[1])
    s.synchronize()
    be.sync()


def test_attention_on_the_librarys_own_stream():
    be = swc.Backend(0, swc.TC_BF16, own_stream=True)
    rn = gen(8)
    q, k, v = rn(2, 16, 128, dtype=BF16), rn(6000, 2, 128, dtype=BF16), rn(6000, 2, 128, dtype=BF16)
    off_q, off_k = offsets([1, 1]), offsets([2900, 3100])
    torch.cuda.synchronize()
    got = be.attention_bf16(q, k, v, off_q, off_k)
    be.sync()
    for i, (a, b) in enumerate(((0, 2900), (2900, 6000))):
        want, tol, _, _ = attention64(q[i:i + 1], k[a:b], v[a:b], 1, b - a, True, 128 ** -0.5)
        check(got[i:i + 1], want, tol)


def test_attention_repeats_bit_for_bit(be):
    rn = gen(10)
    for nq, nk in (([1] * 6, [3000, 10, 700, 2000, 64, 65]), ([200, 300], [200, 300]), ([80], [5000])):
        q, k, v = rn(sum(nq), 8, 128, dtype=BF16), rn(sum(nk), 2, 128, dtype=BF16), rn(sum(nk), 2, 128, dtype=BF16)
        first = be.attention_bf16(q, k, v, offsets(nq), offsets(nk))
        for _ in range(3):
            assert torch.equal(be.attention_bf16(q, k, v, offsets(nq), offsets(nk)), first)


def test_attention_empty_and_refused(be):
    z = lambda *shape: torch.zeros(shape, dtype=BF16, device="cuda")
    off = offsets([2, 2])
    assert be.attention_bf16(z(0, 4, 32), z(4, 2, 32), z(4, 2, 32), off, off).shape == (0, 4, 32)
    assert (be.attention_bf16(z(4, 4, 32), z(0, 2, 32), z(0, 2, 32), off, offsets([0, 0])) == 0).all()
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = z(4, 4, 32) + 1
    assert (be.attention_bf16(z(4, 4, 32), z(4, 2, 32), z(4, 2, 32), none, none, out=out) == 1).all()
    q, k = z(4, 4, 32), z(4, 2, 32)
    wide = z(4, 4, 40)
    for status, call in ((L.ERR_BAD_SHAPE, lambda: be.attention_bf16(z(4, 5, 32), k, k, off, off)),
                         (L.ERR_UNSUPPORTED, lambda: be.attention_bf16(z(4, 4, 12), z(4, 2, 12), z(4, 2, 12), off, off)),
                         (L.ERR_UNSUPPORTED, lambda: be.attention_bf16(z(4, 4, 136), z(4, 2, 136), z(4, 2, 136), off, off)),
                         (L.ERR_BAD_ARG, lambda: be.attention_bf16(q, k, k, off, off, scale=0.0)),
                         (L.ERR_BAD_ARG, lambda: be.attention_bf16(q, k, k, off, off, scale=float("nan"))),
                         (L.ERR_BAD_ARG, lambda: be.attention_bf16(q, k, k, off, off, out=q)),
                         (L.ERR_MISALIGNED, lambda: be.attention_bf16(wide[:, :, 4:36], k, k, off, off)),
                         (L.ERR_MISALIGNED, lambda: be.attention_bf16(z(4, 4, 36)[:, :, :32], k, k, off, off)),
                         (L.ERR_BAD_SHAPE, lambda: be.attention_bf16(q, k[:, :1].expand(4, 2, 32), k, off, off))):
        with pytest.raises(swc.SwcError) as e:
            call()
        assert e.value.status == status, e.value
    import ctypes as C
    from swcompiler_b200 import kernels as K
    long_k = z(4000, 2, 32)
    a = (q.data_ptr(), long_k.data_ptr(), long_k.data_ptr(), out.data_ptr(), 0, 128, 32, 64, 32, 64, 32, 128, 32, 2, 4, 4000, 4, 2, 32,
         off.data_ptr(), off.data_ptr(), 0, 0.2, 1)
    need = C.c_size_t()
    assert be.lib.swcb200_attention_workspace(be._ctx, K._ATTENTION.pack(*a, 0, 0), C.byref(need)) == L.OK and need.value > 0
    assert be.lib.swcb200_attention_bf16(be._ctx, K._ATTENTION.pack(*a, 0, 0)) == L.ERR_BAD_ARG
    for i in (13, 14, 15):  # batch, total_q, total_k
        assert be.lib.swcb200_attention_workspace(be._ctx, K._ATTENTION.pack(*a[:i], (1 << 30) + 1, *a[i + 1:], 0, 0), C.byref(need)) == L.ERR_TOO_LARGE
    assert be.lib.swcb200_attention_workspace(be._ctx, K._ATTENTION.pack(*a, 0, 0), C.byref(need)) == L.OK
    ws = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    assert be.lib.swcb200_attention_bf16(be._ctx, K._ATTENTION.pack(*a, ws.data_ptr(), need.value - 1)) == L.ERR_BAD_ARG
    assert be.lib.swcb200_attention_bf16(be._ctx, K._ATTENTION.pack(*a, ws.data_ptr() + 8, need.value)) == L.ERR_MISALIGNED


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("decode", [False, True])
def test_a_block_of_a_transformer(be, decode):
    """norm, projection, attention over a cache, projection onto the stream, norm, activation, projection onto the stream: each call
    on what the calls before it left, in place where a program would."""
    rn = gen(20 + decode)
    width, hq, hkv, d, hidden = 512, 8, 2, 64, 1280
    nq = [1, 1, 1] if decode else [150, 33, 260]
    nk = [700, 40, 513] if decode else nq
    rows, room = sum(nq), 1024
    w = lambda n, k: rn(n, k, dtype=BF16, s=k ** -0.5)
    w_qkv, w_o, w_up, w_down = w((hq + 2 * hkv) * d, width), w(width, hq * d), w(hidden, width), w(width, hidden)
    b_qkv, b_up = rn((hq + 2 * hkv) * d, s=0.1), rn(hidden, s=0.1)
    norm1, norm2 = (swc.NORM_RMS, 1 + rn(width, s=0.1), None, 1e-6), (swc.NORM_LAYER, 1 + rn(width, s=0.1), rn(width, s=0.1), 1e-6)
    stream = rn(rows, width, s=2.0)
    cache_k, cache_v = rn(3 * room, hkv, d, dtype=BF16), rn(3 * room, hkv, d, dtype=BF16)
    lens = torch.tensor(nk, dtype=torch.int32, device="cuda")
    where = torch.cat([torch.arange(i * room + m - n, i * room + m, device="cuda") for i, (n, m) in enumerate(zip(nq, nk))])

    before = stream.clone()
    _, h = be.norm_residual(stream, pre=norm1, want_sum=False)
    norm_check((None, h), before, None, None, None, 0, 1.0, norm1)
    qkv = be.fc_bf16_residual(h, w_qkv, b_qkv)
    fc_check(qkv, h, w_qkv, b_qkv, "NONE", None, 1.0)
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split((hq * d, hkv * d, hkv * d), 1))
    cache_k[where], cache_v[where] = k, v
    o = attention_check(be, q, cache_k, cache_v, nq, nk, True, k_lens=lens, k_room=[room] * 3)
    be.fc_bf16_residual(o.flatten(1), w_o, residual=stream, out=stream)
    fc_check(stream, o.flatten(1), w_o, None, "NONE", before, 1.0)
    before = stream.clone()
    _, h = be.norm_residual(stream, pre=norm2, want_sum=False)
    norm_check((None, h), before, None, None, None, 0, 1.0, norm2)
    up = be.fc_bf16_residual(h, w_up, b_up, swc.ACT_GELU)
    fc_check(up, h, w_up, b_up, "GELU", None, 1.0)
    down = be.fc_bf16_residual(up, w_down)
    t, y = be.norm_residual(down, residual=stream, post=norm1, scale=0.5, pre=norm2, sum=stream)  # the next block's way in
    norm_check((t, y), down, before, norm1, None, 0, 0.5, norm2)
    be.sync()


def test_two_streams_with_captured_blocks_at_once():
    """The same chain eager, and captured by two contexts whose graphs are replayed side by side, again and again: the same bits."""
    hq, hkv, d, width = 8, 2, 128, 1024
    norm = (swc.NORM_RMS, None, None, 1e-6)

    def block(be, x, w_qkv, w_o, q_off, k_off, cache_k, cache_v, n):
        _, h = be.norm_residual(x, pre=norm, want_sum=False)
        qkv = be.fc_bf16_residual(h, w_qkv)
        q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split((hq * d, hkv * d, hkv * d), 1))
        whole = be.attention_bf16(q, k, v, q_off, q_off)                          # the rows as prompts
        cached = be.attention_bf16(q[:n], cache_k, cache_v, k_off[0], k_off[1])   # the first ones as new tokens over a cache
        x2 = be.fc_bf16_residual(whole.flatten(1), w_o, residual=x, out_dtype=F32)
        x3 = be.fc_bf16_residual(cached.flatten(1), w_o, act=swc.ACT_SILU)
        return be.norm_residual(x2, pre=norm) + (x3,)

    cases = []
    for i, (lengths, n) in enumerate((([300, 5, 170], 3), ([64, 700], 1))):
        rn = gen(30 + i)
        rows = sum(lengths)
        cases.append((rn(rows, width), rn((hq + 2 * hkv) * d, width, dtype=BF16, s=0.03), rn(width, hq * d, dtype=BF16, s=0.03), offsets(lengths),
                      (offsets([1] * n), offsets([2500] * n)), rn(2500 * n, hkv, d, dtype=BF16), rn(2500 * n, hkv, d, dtype=BF16), n))
    be = swc.Backend(0, swc.TC_BF16)
    want = [[t.clone() for t in block(be, *c)] for c in cases]
    torch.cuda.synchronize()
    lanes = []
    for c in cases:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            lane = swc.Backend(0, swc.TC_BF16, stream=s)
            block(lane, *c)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                out = block(lane, *c)
        lanes.append((s, lane, g, out))
    for _ in range(5):
        for s, _, g, out in lanes:
            with torch.cuda.stream(s):
                for t in out:
                    t.zero_()
                g.replay()
                g.replay()
    torch.cuda.synchronize()
    for (_, lane, _, out), expect in zip(lanes, want):
        lane.sync()
        for got, ref in zip(out, expect):
            assert torch.equal(got, ref)
