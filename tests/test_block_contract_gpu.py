"""GPU: what the transformer-block calls promise beside their results: bounded waits, limits, order on a stream."""
import ctypes as C

import pytest
import torch

import swcompiler_b200 as swc
from swcompiler_b200 import _lib as L
from swcompiler_b200 import kernels as K
from test_block_ops_gpu import attention64, be, check, fc_check, gen, offsets  # noqa: F401 (be: a fixture)

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("hq,d", [(4, 64), (24, 128), (64, 64)])
def test_attention_waits_that_run_out_end_the_call(hq, d):
    """The last of 65536 sequences is the only one with rows, and looking for it takes about a millisecond: waits limited to less run
    out (in all warps, or around that time in some of a group).  The call ends either way, and the context stays usable."""
    be = swc.Backend(0, swc.TC_BF16)
    rn = gen(hq)
    batch, n = 1 << 16, 1900
    q, k, v = rn(1, hq, d, dtype=BF16), rn(n, 1, d, dtype=BF16), rn(n, 1, d, dtype=BF16)
    off_q, off_k = torch.zeros(batch + 1, dtype=torch.int32, device="cuda"), torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
    off_q[-1], off_k[-1] = 1, n
    want, tol, _, _ = attention64(q, k, v, 1, n, True, d ** -0.5)
    ran_out = []
    for limit in [20_000] + [int(100_000 * 1.2 ** i) for i in range(24)] + [4_000_000_000]:
        be.set_wait_limit(limit)
        got = be.attention_bf16(q, k, v, off_q, off_k)
        try:
            be.sync()
        except swc.SwcError as e:
            assert e.status == L.ERR_TIMEOUT
            ran_out.append(limit)
        else:
            check(got, want, tol)
    assert 20_000 in ran_out and 4_000_000_000 not in ran_out


@pytest.mark.parametrize("m", [1, 2, 24])
def test_a_chain_reads_what_the_call_before_it_wrote(m):
    """Layers of a gated block over the same few buffers, captured and replayed with new inputs: every call's operands (rows, gate,
    bias, norm weights) were rewritten just before.  The bits are those of the calls one by one with a wait behind each."""
    d, layers = 1024, 5
    s = torch.cuda.Stream()
    rn = gen(m)
    with torch.cuda.stream(s):
        be = swc.Backend(0, swc.TC_BF16, stream=s)
        w = [[rn(d, d, dtype=BF16, s=d ** -0.5) for _ in range(4)] for _ in range(layers)]
        x0, x = rn(m, d), torch.empty(m, d, device="cuda")
        h, a, g, y = (torch.empty(m, d, dtype=BF16, device="cuda") for _ in range(4))
        vector = torch.empty(1, d, device="cuda")
        keep = [torch.empty(m, d, device="cuda") for _ in range(layers)]

        def run(behind):
            be.norm_residual(x0, pre=(swc.NORM_RMS, None, None, 1e-6), sum=x, y=h), behind()
            for i, (w1, w2, w3, w4) in enumerate(w):
                be.fc_bf16_residual(h, w1, out=a), behind()
                be.fc_bf16_residual(h, w2, act=swc.ACT_SILU, out=g), behind()
                be.fc_bf16_residual(h[:1], w3, act=swc.ACT_TANH, out=vector), behind()
                be.norm_residual(a, gate=g, gate_rows=1, pre=(swc.NORM_LAYER, vector[0], vector[0], 1e-5), want_sum=False, y=y), behind()
                be.fc_bf16_residual(y, w4, vector[0], residual=x, out=x), behind()
                be.norm_residual(x, post=(swc.NORM_RMS, vector[0], None, 1e-6), pre=(swc.NORM_RMS, None, vector[0], 1e-6), sum=keep[i], y=h), behind()

        run(lambda: None)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            run(lambda: None)
        for step in range(12):
            for _ in range(2):  # (the first one leaves other values in all of the buffers)
                x0.copy_(rn(m, d))
                graph.replay()
            got = [t.clone() for t in keep + [h]]
            run(s.synchronize)
            assert all(torch.equal(p, q) for p, q in zip(got, keep + [h])), step
        be.sync()
    s.synchronize()


def least_ms(be, call, times=6):
    call()
    best = float("inf")
    for _ in range(times):
        e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        e[0].record()
        call()
        e[1].record()
        e[1].synchronize()
        best = min(best, e[0].elapsed_time(e[1]))
    return best


@pytest.mark.parametrize("what", ["split", "pairs", "tokens", "many rows", "prompts", "long prompt", "chunk"])
def test_an_sm_limit_holds(be, what):
    """With eight SMs of all of them a call takes many times as long (a quarter of the SMs' ratio is asked for), and its results are
    right under any limit."""
    rn = gen(len(what))
    if what in ("split", "pairs"):
        m, n, k = (64, 8192, 4096) if what == "split" else (4096, 4096, 2048)
        a, wp, out = rn(m, k, dtype=BF16), rn(n, k, dtype=BF16, s=k ** -0.5), torch.empty(m, n, device="cuda")
        want = a.double() @ wp.double().t()
        tol = k / 16 * 2 ** -22 * (a.double().abs() @ wp.double().abs().t())

        def call():
            be.fc_bf16_residual(a, wp, out=out)
    else:
        nq, nk, hq, hkv, d = {"tokens": ([1] * 64, [2000] * 64, 8, 8, 128), "many rows": ([2] * 16, [3000] * 16, 64, 2, 64),
                              "prompts": ([200] * 64, [200] * 64, 16, 8, 64), "long prompt": ([4000], [4000], 16, 2, 128),
                              "chunk": ([70], [40000], 8, 2, 128)}[what]
        q, k, v = rn(sum(nq), hq, d, dtype=BF16), rn(sum(nk), hkv, d, dtype=BF16), rn(sum(nk), hkv, d, dtype=BF16)
        off_q, off_k, out = offsets(nq), offsets(nk), torch.empty(sum(nq), hq, d, dtype=BF16, device="cuda")
        parts = [attention64(q[i * nq[0]:(i + 1) * nq[0]], k[i * nk[0]:(i + 1) * nk[0]], v[i * nk[0]:(i + 1) * nk[0]], nq[0], nk[0], True, d ** -0.5)[:2]
                 for i in range(len(nq))]
        want, tol = (torch.cat(t) for t in zip(*parts))

        def call():
            be.attention_bf16(q, k, v, off_q, off_k, out=out)

    sms = torch.cuda.get_device_properties(0).multi_processor_count
    try:
        free = least_ms(be, call)
        for limit in (1, 8, 21, sms + 1):
            be.set_sm_limit(limit)
            out.fill_(float("nan"))
            t = least_ms(be, call)
            check(out, want, tol)
            if limit == 8:
                assert t > free * sms / 8 / 4, (t, free)
    finally:
        be.set_sm_limit(0)
    be.sync()


def test_attention_workspace_reads_no_more_than_it_says(be):
    """Batch, totals, heads and width, in a description that is zero otherwise: the bytes of the whole description."""
    fields = [0] * 26
    fields[13:19] = 1, 1, 60000, 32, 8, 128
    need, whole = C.c_size_t(), C.c_size_t()
    assert be.lib.swcb200_attention_workspace(be._ctx, K._ATTENTION.pack(*fields), C.byref(need)) == L.OK and need.value > 0
    fields[22] = 0.1
    assert be.lib.swcb200_attention_workspace(be._ctx, K._ATTENTION.pack(*fields), C.byref(whole)) == L.OK and whole.value == need.value
    q, k = torch.zeros(1, 32, 128, dtype=BF16, device="cuda"), torch.zeros(600, 8, 128, dtype=BF16, device="cuda")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(swc.SwcError) as e:
            be.attention_bf16(q, k, k, offsets([1]), offsets([600]), scale=scale)
        assert e.value.status == L.ERR_BAD_ARG
    with pytest.raises(swc.SwcError):
        be.attention_bf16(q[:0], k, k, offsets([0]), offsets([600]), scale=0.0)  # empty calls, too


@pytest.mark.parametrize("new,n", [(1, 900), (30, 700), (200, 900), (200, 2300), (70, 6000)])
@pytest.mark.parametrize("size", [3e3, 3e4, 1e6, 1e12])
def test_attention_scores_far_beyond_the_exponential(be, new, n, size):
    """Scores of 1e7 up to 1e25: a row is the value of its largest score.  All terms of a score are positive, so it is known to
    (d / 16 + 1) * 2^-22 of itself; rows whose two largest scores are nearer than four times that are left out.  The one weight left is
    rounded to bf16."""
    d, h = 64, 2
    rn = gen(new + n)
    q, k, v = (rn(new, h, d).abs() * size).to(BF16), (rn(n, h, d).abs() * size).to(BF16), rn(n, h, d, dtype=BF16)
    slope = torch.linspace(0.5, 2, n, device="cuda")[:, None, None]
    for keys in (k, (k.float() * slope).to(BF16), (k.float() * slope.flip(0)).to(BF16)):
        lse = torch.empty(new, h, device="cuda")
        got = be.attention_bf16(q, keys, v, offsets([new]), offsets([n]), causal=False, lse=lse)
        s = d ** -0.5 * q.double().transpose(0, 1) @ keys.double().permute(1, 2, 0)
        first, second = s.topk(2, 2).values.unbind(2)
        known = (d / 16 + 1) * 2 ** -22
        clear = (first - second > 4 * known * first).t()
        assert clear.float().mean() > 0.9
        want = torch.stack([v[s[i].argmax(1), i] for i in range(h)], 1).double()
        check(got[clear], want[clear], 2 ** -8 * want[clear].abs())
        assert ((lse.double() - first.t()).abs() <= (known + 2 ** -21) * first.t()).all()
    be.sync()


@pytest.mark.parametrize("new", [1, 100])
def test_attention_largest_and_smallest_scales(be, new):
    """The softmax runs on powers of two: a scale that is finite, but not times log2(e), is refused; smaller ones give no NaN."""
    rn = gen(new)
    q, k, v = rn(new, 2, 64, dtype=BF16), rn(300, 2, 64, dtype=BF16), rn(300, 2, 64, dtype=BF16)
    for scale in (2.4e38, 3.3e38):
        with pytest.raises(swc.SwcError) as e:
            be.attention_bf16(q * 0, k, v, offsets([new]), offsets([300]), scale=scale)
        assert e.value.status == L.ERR_BAD_ARG
    uniform = v.double().mean(0, keepdim=True).expand(new, 2, 64)
    # equal weights: 300 of them, rounded to bf16 (1 is a bf16), and 300 additions of the products
    tol = 300 * 2 ** -24 * v.double().abs().mean(0)
    check(be.attention_bf16(q * 0, k, v, offsets([new]), offsets([300]), scale=2e38, causal=False), uniform, tol)
    check(be.attention_bf16(q, k, v, offsets([new]), offsets([300]), scale=1e-30, causal=False), uniform, tol)


@pytest.mark.parametrize("m,n,k", [(1900, 6500, 4104), (700, 4700, 5600)])
def test_fc_bf16_residual_tiles_in_bands(be, m, n, k):
    """Weights of more than 48 MiB in tiles of 256 whose number is no multiple of 8: tiles are taken in bands, the last one narrower.
    Every tile is written, once (in place, a second time would add its product again)."""
    rn = gen(n)
    a, wp, bias, r = rn(m, k, dtype=BF16), rn(n, k, dtype=BF16, s=k ** -0.5), rn(n), rn(m, n)
    out = r.clone()
    be.fc_bf16_residual(a, wp, bias, residual=out, out=out)
    fc_check(out, a, wp, bias, "NONE", r, 1.0)


@pytest.mark.parametrize("new", [2, 90])
def test_attention_outputs_that_overlap_themselves_are_refused(be, new):
    rn = gen(new)
    q, k, v = rn(new, 4, 32, dtype=BF16), rn(200, 2, 32, dtype=BF16), rn(200, 2, 32, dtype=BF16)
    room = torch.zeros(new * 4 * 64, dtype=BF16, device="cuda")
    want = be.attention_bf16(q, k, v, offsets([new]), offsets([200]))
    for strides in ((32, 32, 1), (96, 32, 1), (32, 32 * new - 8, 1), (40, 40, 1)):
        with pytest.raises(swc.SwcError) as e:
            be.attention_bf16(q, k, v, offsets([new]), offsets([200]), out=room.as_strided((new, 4, 32), strides))
        assert e.value.status == L.ERR_BAD_SHAPE
    for strides in ((128, 32, 1), (32, 32 * new, 1), (40, 40 * new, 1), (160, 40, 1)):  # rows or heads first, dense or not
        assert torch.equal(be.attention_bf16(q, k, v, offsets([new]), offsets([200]), out=room.as_strided((new, 4, 32), strides)), want)
    for t in (q[:1], q[:, :2].contiguous()):  # a dimension of one element has no stride
        be.attention_bf16(t, k, v, offsets([len(t)]), offsets([200]), out=torch.empty_like(t))


@pytest.mark.parametrize("limit", [1, 2, 3])
def test_fc_bf16_under_the_smallest_sm_limits(be, limit):
    rn = gen(limit)
    a, wp = rn(700, 256, dtype=BF16), rn(900, 256, dtype=BF16, s=256 ** -0.5)
    be.set_sm_limit(limit)
    try:
        fc_check(be.fc_bf16(a, wp, out_dtype=F32), a, wp, None, "NONE", None, 1.0)
        fc_check(be.fc_bf16_residual(a, wp, out_dtype=F32), a, wp, None, "NONE", None, 1.0)
    finally:
        be.set_sm_limit(0)
    be.sync()
