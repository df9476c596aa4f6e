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


@pytest.mark.parametrize("T,nH,H,hd,rot,cache", [(4, 64, 8, 64, 64, "bf16"), (4, 6, 2, 72, 36, "f32"), (2001, 3, 1, 16, 16, "bf16")])
def test_append_skips_positions_outside_the_table(torch, T, nH, H, hd, rot, cache):
    """Nothing of such a token enters the cache (its query turns as position 0), whatever kernel the sizes choose; the
    others do.  Without `positions` the cache index is the position."""
    from mxmoe import MxMoeError
    n, page = 50, 16
    P = Pool(torch, [n] * 3, nH, H, hd, page, cache, track=True, max_pages=-(-(n + T) // page))
    t = np.arange(T)
    rows, index = (t % 3).astype(np.int32), (n + t // 3).astype(np.int32)
    pos = np.array([100, 7, -1, 2 ** 31 - 1], np.int32)[t % 4]
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(T, h, hd, generator=g).bfloat16().cuda() for h in (nH, H, H))
    r = table(torch, rot, 100)
    before = [x.clone() for x in (P.k, P.v, P.weight, P.position)]
    args = (P.tables, torch.from_numpy(index).cuda(), r)
    got = P.cache.append(q, k, v, *args, torch.from_numpy(pos).cuda(), torch.from_numpy(rows).cuda())
    with pytest.raises(MxMoeError, match="position"):
        P.cache.sync_status()
    ok = np.flatnonzero(pos == 7)
    page_of, slot = (torch.from_numpy(x.astype(np.int64)).cuda() for x in po.place(P.htab, page, rows[ok], index[ok]))
    assert torch.all(P.position[page_of, :, slot] == 7) and torch.all(P.weight[page_of, :, slot] == 0)
    assert torch.equal(P.v[page_of, :, slot], v[ok].to(P.v.dtype))
    for now, was in zip((P.k, P.v, P.weight, P.position), before):
        now, was = now.clone(), was.clone()
        now[page_of, :, slot] = was[page_of, :, slot] = 0
        raw = {2: torch.int16, 4: torch.int32}[now.element_size()]
        assert torch.equal(now.view(raw), was.view(raw))
    assert torch.equal(got[pos != 7], q[pos != 7])
    # indexes as positions, the table too short for all of them
    for x, was in zip((P.k, P.v, P.weight, P.position), before):
        x.copy_(was)
    P.cache.append(q, k, v, P.tables, args[1], table(torch, rot, n), rows=torch.from_numpy(rows).cuda())
    with pytest.raises(MxMoeError, match="position"):
        P.cache.sync_status()
    for now, was in zip((P.k, P.v, P.weight, P.position), before):
        raw = {2: torch.int16, 4: torch.int32}[now.element_size()]
        assert torch.equal(now.view(raw), was.view(raw))
