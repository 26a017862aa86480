"""Waits of the tensor cores' attention kernels that run out: the call reports it, each element of the forward
pass's outputs holds its result or is not written, and the context stays usable."""
import numpy as np
import pytest

from helpers import d, dev, host
from quasarml_b200 import abi, datagen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
def test_waits_that_run_out(D):
    import torch
    torch.cuda.set_device(0)
    c = abi.Context(0)
    q, k, v, do = (dev(datagen.normal(i, (2, 700, 4 if i in (1, 4) else 2, D), 0, 1).astype(np.float16)) for i in range(1, 5))
    o, lse = torch.empty_like(q), torch.empty(2, 4, 700, device="cuda")
    grads = [torch.empty_like(x) for x in (q, k, v)]

    def forward():
        c.attention(d(q), d(k), d(v), d(o), D ** -0.5, window=300, sinks=2, lse=d(lse))

    def backward():
        c.attention_backward(d(q), d(k), d(v), d(o), d(lse), d(do), *[d(x) for x in grads], D ** -0.5, window=300, sinks=2)

    forward()
    assert c.last_kernel() == "k_attention_tc"
    c.synchronize()
    want = [host(o), host(lse)]
    backward()
    c.synchronize()
    want_grads = [host(x) for x in grads]
    flush, expired, kept = torch.empty(2**26, device="cuda"), 0, 0
    for limit in [1] + sorted(int(1000 * 1.12 ** i) for i in range(45)):
        o.fill_(77.0)
        lse.fill_(77.0)
        flush.zero_()
        torch.cuda.synchronize()
        c.set_wait_limit(limit)
        forward()
        try:
            c.synchronize()
        except abi.QsmlError as e:
            assert e.status == abi.E_TIMEOUT
            expired += 1
        for x, w in zip((o, lse), want):
            got = host(x)
            assert np.all((got == w) | (got == 77.0)), limit
        kept += int(np.any(host(o) == want[0]))
    assert expired and kept  # some limits ran out, some CTAs finished
    o.copy_(dev(want[0]))
    lse.copy_(dev(want[1]))
    expired = 0
    for limit in [1] + sorted(int(1000 * 1.3 ** i) for i in range(20)):
        flush.zero_()
        torch.cuda.synchronize()
        c.set_wait_limit(limit)
        backward()
        try:
            c.synchronize()
        except abi.QsmlError as e:
            assert e.status == abi.E_TIMEOUT
            expired += 1
    assert expired
    c.set_wait_limit(0)
    forward()
    backward()
    c.synchronize()
    for x, w in zip([o, lse] + grads, want + want_grads):
        assert np.array_equal(host(x), w)
    c.close()
