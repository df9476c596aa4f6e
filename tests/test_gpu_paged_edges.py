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


@pytest.mark.parametrize("dtype,hd", [("f32", 64), ("bf16", 64), ("f32", 80)])
@pytest.mark.parametrize("shift", [0, 1])
def test_append_8_bit_rounds_the_quotient(torch, dtype, hd, shift):
    """An 8-bit code is the one nearest to x / scale, ties to even, also where x is a rounded tie times the scale: the
    bits of a correctly rounded quotient rounded again.  shift: off the alignment of wide loads."""
    T, H = 512, 8
    P = Pool(torch, [0], H, H, hd, 16, "e4m3", max_pages=T // 16)
    codes = torch.arange(0, 126, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    ties = (codes[1:] + codes[:-1]) / 2
    g = torch.Generator().manual_seed(3)
    x = ties[torch.randint(len(ties), (T, H, hd), generator=g)] * (torch.randint(0, 2, (T, H, hd), generator=g) * 2 - 1)
    ks, vs = (s.double().cpu()[:, None] for s in (P.ks, P.vs))
    dt = getattr(torch, DT[dtype])
    k, v = (x * ks).to(dt), (x * vs).to(dt)
    k[0, 0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), -0.0])

    def off(t):
        return torch.cat([torch.zeros(shift, dtype=dt), t.flatten()]).cuda()[shift:].view(t.shape)

    P.cache.append(None, off(k), off(v), P.tables, torch.arange(T, dtype=torch.int32, device="cuda"),
                   rows=torch.zeros(T, dtype=torch.int32, device="cuda"))
    P.cache.sync_status()
    pg, sl = po.place(P.htab, 16, 0, np.arange(T))
    for pool, t, s in ((P.k, k, ks), (P.v, v, vs)):
        want = (t.float() / s.float()).clamp(-448, 448).to(torch.float8_e4m3fn)
        got = pool.cpu().view(torch.uint8)[pg, :, sl].view(torch.float8_e4m3fn)
        nan = want.float().isnan()
        assert torch.equal(got.float().isnan(), nan)
        assert torch.equal(got.view(torch.uint8)[~nan], want.view(torch.uint8)[~nan])


def test_numbers_past_32_bits_are_refused(torch):
    """They do not wrap around on their way to the C structs."""
    from mxmoe import MxMoeError
    from mxmoe.paged import PagedKvCache, RotaryConfig, RotaryTable
    P = Pool(torch, [40, 40], 8, 2, 64, 16, track=True)
    q = torch.randn(2, 8, 64, device="cuda")
    before = [x.clone() for x in (P.k, P.v, P.weight, P.position)]
    w = 1 << 32
    for f in (lambda: P.cache.decode(q, P.tables, P.lens, window=w + 5),
              lambda: P.cache.evict(P.tables, P.lens, P.lens, w + 30),
              lambda: P.cache.evict(P.tables, P.lens, P.lens, 30, sink=w),
              lambda: P.cache.evict(P.tables, P.lens, P.lens, 30, recent=w),
              lambda: PagedKvCache(4, 16, w + 8, 2, 64), lambda: PagedKvCache.over(P.k, P.v, w + 8),
              lambda: RotaryTable.of(RotaryConfig(w + 64), 1)):
        with pytest.raises(MxMoeError):
            f()
    for now, was in zip((P.k, P.v, P.weight, P.position), before):
        raw = {2: torch.int16, 4: torch.int32}[now.element_size()]
        assert torch.equal(now.view(raw), was.view(raw))


@pytest.mark.parametrize("gap", [14.0, 17.5, 20.0, 24.0])
@pytest.mark.parametrize("n,hd,every", [(20, 16, 20), (256, 64, 256), (200, 128, 200), (100, 256, 100), (30000, 64, 300)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decode_8_bit_keeps_small_shares(torch, gap, n, hd, every, dtype):
    """One key in `every` holds nearly all of the softmax and has a value of 0; the others, `gap` below it, make up the
    output.  A share is held to half a step of the second of its two terms, 2^-39 of the largest, and as it is held
    in 22 bits otherwise to 1e-5 of itself."""
    from mxmoe.paged import PagedKvCache
    page = 16
    pages = -(-n // page)
    k = torch.zeros(pages, 1, page, hd)
    v = torch.full((pages, 1, page, hd), 448.0)
    at = np.arange(0, n, every)
    k[at // page, 0, at % page, 0] = 16.0
    v[at // page, 0, at % page] = 0.0
    q = torch.zeros(1, 2, hd, dtype=getattr(torch, DT[dtype]))
    q[0, :, 0] = gap / 16  # exact in bf16
    e4 = torch.float8_e4m3fn
    cache = PagedKvCache.over(k.to(e4).cuda(), v.to(e4).cuda(), 2)
    tab = np.arange(pages, dtype=np.int32)[None]
    got = cache.decode(q.cuda(), torch.from_numpy(tab).cuda(), torch.tensor([n], dtype=torch.int32, device="cuda"), scale=1.0)
    want, _ = po.decode(q.double().numpy(), k.double().numpy(), v.double().numpy(), tab, np.array([n]), 1.0)
    tol = 448 * every * 2.0 ** -39 + 1e-5 * want + (2.0 ** -8 * want if dtype == "bf16" else 0)
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= tol)


def odd_close(got, want, tol):
    """Alike where NaN or infinite, within tol elsewhere."""
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)])
    assert np.all(np.abs(got[fin] - want[fin]) <= tol[fin])


@pytest.mark.parametrize("cache,q_dtype", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32"), ("e4m3", "bf16"), ("e4m3", "f32")])
@pytest.mark.parametrize("lens,nH,H,hd", [([40, 100], 8, 2, 64), ([5000, 333], 12, 1, 128), ([70, 1000], 2, 1, 80), ([300, 90], 4, 2, 256)])
def test_decode_infinite_and_nan_keys_and_values(torch, cache, q_dtype, lens, nH, H, hd):
    """As the formula has it: a key of score -inf, and what lies at it, does not count; an infinite value with a share
    gives infinity in its column, both signs give NaN; a NaN value its column; a NaN score the head."""
    P = Pool(torch, lens, nH, H, hd, 16, cache, track=True)
    rng = np.random.default_rng(7)
    q = torch.randn(2, nH, hd, generator=torch.Generator().manual_seed(1)).to(getattr(torch, DT[q_dtype]))
    bias = np.zeros((2, nH, max(lens)), np.float32)
    inf, nan = (np.inf, np.nan) if cache != "e4m3" else (np.nan, np.nan)  # e4m3 has no infinities
    for row, n in enumerate(lens):
        pg, sl = po.place(P.htab, 16, row, np.arange(n))
        # values: +inf in column 1, -inf in 2, both in 3, NaN in 5
        for col, x in ((1, inf), (2, -inf), (3, inf), (3, -inf), (5, nan)):
            i = rng.integers(n)
            P.hv[pg[i], H - 1, sl[i], col] = x
        # masked by the bias: whatever lies there
        for i in rng.choice(n, 7, replace=False):
            bias[row, :, i] = -np.inf
            P.hv[pg[i], :, sl[i]] = rng.choice([inf, -inf, nan], hd)
    # row 1, first key head: an infinite key, a score of +-inf for each head by its query's sign
    if cache != "e4m3":
        pg, sl = po.place(P.htab, 16, 1, 11)
        bias[1, :, 11] = 0
        P.hv[pg, 0, sl] = 1.0
        P.hk[pg, 0, sl, 2] = inf
    P.k.copy_(torch.from_numpy(P.hk).to(P.k.dtype))
    P.v.copy_(torch.from_numpy(P.hv).to(P.v.dtype))
    used = P.hw.copy()
    lse = torch.empty(2, nH, device="cuda")
    out = P.cache.decode(q.cuda(), P.tables, P.lens, bias=torch.from_numpy(bias).cuda(), track=True, lse=lse)
    P.cache.sync_status()
    w = P.hw.astype(np.float64)
    with np.errstate(invalid="ignore"):
        want, want_lse = po.decode(q.double().numpy(), P.hk, P.hv, P.htab, P.hlens, 1 / np.sqrt(hd), bias=bias, weight=w,
                                   k_scale=P.hks, v_scale=P.hvs)
    assert np.isfinite(want).any() and not np.isfinite(want).all()
    tol = 2 * ATOL + (2.0 ** -8 if q_dtype == "bf16" else 2.0 ** -24) * np.abs(want)
    odd_close(out.double().cpu().numpy(), want, tol)
    odd_close(lse.cpu().numpy(), want_lse, 2 * ATOL + 2e-6 * np.abs(want_lse))
    odd_close(P.weight.cpu().numpy(), w, 2e-5 * (w - used) + 2.0 ** -23 * np.abs(w))


TYPES = [("bf16", "bf16"), ("bf16", "f32"), ("e4m3", "bf16"), ("e4m3", "f32"), ("f32", "f32")]


@pytest.mark.parametrize("cache,q_dtype,nH,H,hd,longest", [(*t, 8, 4, 16, 12000) for t in TYPES]
                         + [("bf16", "bf16", 18, 2, 16, 12000), ("e4m3", "f32", 18, 2, 16, 12000), ("bf16", "bf16", 4, 4, 128, 6000),
                            ("e4m3", "bf16", 4, 4, 128, 6000), ("f32", "f32", 2, 2, 256, 6000)])
def test_decode_ranges_kept_back(torch, cache, q_dtype, nH, H, hd, longest):
    """More than eight tiles a warp (148 SMs of 8 warps at most, tiles of 16 or 32 keys): a quarter of the list goes to
    whoever is done, the counters are set back at the end, by calls of every size in turn."""
    rng = np.random.default_rng(2)
    lens = [int(x) for x in rng.integers(1, longest, 26)] + [0, 1, 40000, 31, 32, 33]
    tile = 16 if hd == 256 else 32
    assert sum(-(-n // tile) for n in lens) * H * -(-nH // H // 8) >= 8 * 8 * 148
    P, out = check_decode(torch, lens, nH, H, hd, 16, cache, q_dtype, sinks=True)
    q = torch.randn(len(lens), nH, hd, device="cuda").to(getattr(torch, DT[q_dtype]))
    few = P.cache.decode(q[:3], P.tables[:3], P.lens[:3])
    want = P.cache.decode(q, P.tables, P.lens)
    for _ in range(5):
        assert torch.equal(P.cache.decode(q[:3], P.tables[:3], P.lens[:3]), few)
        assert torch.equal(P.cache.decode(q, P.tables, P.lens), want)


@pytest.mark.parametrize("cache,q_dtype", [("bf16", "bf16"), ("e4m3", "f32"), ("f32", "f32")])
def test_decode_track_with_ranges_kept_back(torch, cache, q_dtype):
    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.integers(1, 12000, 28)] + [0, 20000, 1]
    check_decode(torch, lens, 8, 4, 16, 16, cache, q_dtype, sinks=True, track=True)


@pytest.mark.parametrize("rows,longest", [(513, 200), (1100, 200), (513, 1200), (1100, 1200)])
@pytest.mark.parametrize("cache,q_dtype", [("bf16", "bf16"), ("f32", "f32"), ("e4m3", "f32")])
@pytest.mark.parametrize("track", [False, True])
def test_decode_rows_of_several_launches(torch, rows, longest, cache, q_dtype, track):
    """More than 512 rows: whole segments under a table of 200 tokens, cut ones (kept back among them) under one of 1200;
    bias and lse by row, weights of one launch while the next begins."""
    rng = np.random.default_rng(rows)
    lens = [int(x) for x in rng.integers(0, longest + 1, rows)]
    lens[0] = lens[511] = lens[-1] = 0
    lens[512] = longest
    bias = rng.standard_normal((rows, 1, longest // 2)).astype(np.float32)
    check_decode(torch, lens, 6, 3, 16, 8, cache, q_dtype, sinks=True, bias=bias, track=track)


def test_decode_rows_of_several_launches_by_strides(torch):
    rows = 700
    lens = [(37 * i) % 300 for i in range(rows)]
    P = Pool(torch, lens, 4, 2, 32, 8)
    q = torch.randn(rows, 4, 32, device="cuda").bfloat16()
    lse, out_lse = torch.empty(rows, 4, device="cuda"), torch.empty(rows, 4, device="cuda")
    want = P.cache.decode(q, P.tables, P.lens, lse=lse)
    wide = torch.zeros(4, rows, 40, device="cuda").bfloat16()
    wide[:, :, 4:36] = q.transpose(0, 1)
    room = torch.zeros(4, rows, 48, device="cuda").bfloat16()
    tables = torch.zeros(rows, P.tables.shape[1] + 3, dtype=torch.int32, device="cuda")
    tables[:, : P.tables.shape[1]] = P.tables
    P.cache.decode(wide.transpose(0, 1)[..., 4:36], tables[:, : P.tables.shape[1]], P.lens,
                   out=room.transpose(0, 1)[..., 8:40], lse=out_lse)
    assert torch.equal(room.transpose(0, 1)[..., 8:40], want) and torch.equal(out_lse, lse)
    assert torch.count_nonzero(room) == torch.count_nonzero(want)


@pytest.mark.parametrize("cache,q_dtype,out_dtype", [("bf16", "bf16", "f32"), ("bf16", "f32", "bf16"), ("e4m3", "bf16", "f32"),
                                                     ("e4m3", "f32", "bf16"), ("f32", "bf16", "f32"), ("f32", "bf16", "bf16"),
                                                     ("f32", "f32", "bf16")])
@pytest.mark.parametrize("nH,H,hd", [(8, 2, 64), (9, 1, 128), (6, 2, 256)])
def test_decode_output_types(torch, cache, q_dtype, out_dtype, nH, H, hd):
    check_decode(torch, [0, 1, 17, 300, 5000], nH, H, hd, 16, cache, q_dtype, out_dtype, sinks=True)


@pytest.mark.parametrize("cache,q_dtype", TYPES + [("f32", "bf16")])
@pytest.mark.parametrize("shape", [(3, 16, 3000), (1, 1, 40)])
def test_decode_bias_by_type(torch, cache, q_dtype, shape):
    bias = np.random.default_rng(1).standard_normal(shape).astype(np.float32)
    check_decode(torch, [3000, 39, 41], 16, 2, 64, 16, cache, q_dtype, bias=bias)


@pytest.mark.parametrize("cache,q_dtype", TYPES + [("f32", "bf16")])
@pytest.mark.parametrize("window", [1, 17, 300])
def test_decode_window_by_type(torch, cache, q_dtype, window):
    check_decode(torch, [1, 16, 129, 7000, 0], 16, 2, 64, 24, cache, q_dtype, window=window, sinks=True)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,rot", [(64, 64), (80, 20), (7, 6)])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary_bf16(torch, interleaved, hd, rot, inverse):
    """The turn and its gradient in bf16: one rounding of the 32-bit result."""
    x = torch.randn(300, 5, hd, generator=torch.Generator().manual_seed(4)).bfloat16()
    pos = (np.arange(300) * 13 % 1000).astype(np.int32)
    inv, f = po.frequencies(rot, scaling="yarn", factor=8.0)
    want = po.rotate(x.double().numpy(), pos, inv, f, interleaved, inverse=inverse)
    r = table(torch, rot, 1000, interleaved, scaling="yarn", scaling_factor=8.0)
    got = r.apply(x.cuda(), torch.from_numpy(pos).cuda(), inverse=inverse)
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= 6e-6 + (2.0 ** -8 + 2.0 ** -20) * np.abs(want))


@pytest.mark.parametrize("over", ["lens", "seen", "askew"])
def test_evict_writes_lengths_over_others(torch, over):
    """Into lens, where it is seen too; into seen; over seen by one element."""
    lens = [700, 90, 3000, 40, 1500]
    P, R = (Pool(torch, lens, 8, 4, 32, 16, track=True) for _ in range(2))
    want = R.cache.evict(R.tables, R.lens, R.lens, 300, 4, 50)
    room = torch.cat([P.lens, P.lens])
    seen, new = {"lens": (P.lens, P.lens), "seen": (room[:5], room[:5]), "askew": (room[:5], room[1:6])}[over]
    got = P.cache.evict(P.tables, P.lens, seen, 300, 4, 50, new_lens=new)
    P.cache.sync_status()
    assert torch.equal(got, want) and torch.equal(P.position, R.position) and torch.equal(P.weight, R.weight)
