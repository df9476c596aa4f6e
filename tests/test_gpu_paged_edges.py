"""The paged cache where it is easily wrong, against the 64-bit oracle.  Pools,
checks and tolerances are test_gpu_paged's unless a test derives its own."""
import numpy as np
import pytest

import paged_oracle as po
from test_gpu_paged import ATOL, DT, Pool, check_decode, table, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def test_a_cache_made_on_a_side_stream_while_the_default_stream_is_busy(torch):
    """Long enough that ranges are kept back: their counters have to be zero when the first call starts."""
    from mxmoe.paged import PagedKvCache
    P = Pool(torch, [5000] * 8, 8, 8, 64, 16)
    q = torch.randn(8, 8, 64, device="cuda").bfloat16()
    want = P.cache.decode(q, P.tables, P.lens)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    torch.cuda._sleep(400_000_000)  # about 0.2 s on the default stream
    with torch.cuda.stream(s):
        cache = PagedKvCache.over(P.k, P.v, 8)
        got = [cache.decode(q, P.tables, P.lens) for _ in range(3)]
        cache.sync_status()
    torch.cuda.synchronize()
    got.append(cache.decode(q, P.tables, P.lens))
    for x in got:
        assert torch.equal(x, want)
