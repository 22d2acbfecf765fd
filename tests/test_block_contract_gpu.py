"""GPU: what the transformer-block calls promise beside their results: bounded waits, limits, order on a stream."""
import pytest
import torch

import swcompiler_b200 as swc
from swcompiler_b200 import _lib as L
from test_block_ops_gpu import attention64, check, gen, offsets

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
