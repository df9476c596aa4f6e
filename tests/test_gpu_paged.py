"""GPU parity of the paged key-value cache (mxmoe.paged over the C ABI) against
the 64-bit oracle (oracle/paged_oracle.py).

Tolerances, from the formulas.  A score is a sum of head_dim products of 32-bit
or exact terms: with |q . k| scale of about 10 in sum of magnitudes it is off by
at most a few 2^-22 x 10, so a share by 5e-6 of itself, and an output by 5e-6 of
max |v| (below 6 in these inputs): 3e-5 absolute covers it, twice that with a
bias or 8-bit scales.  A bf16 output adds half a step, 2^-8 of itself
at most.  A
share added to a weight is off by 2e-5 of itself, the sum by one rounding.  A
rotation in 32 bits is off by 3 roundings of max(|a|, |b|): 4 x 2^-24 x 2 x the
factor, and one rounding of the table's entries: 1e-6 of 6.  An 8-bit value lies
within half a step of the exact one (1e-3 of the step for the product before
it).  Moves are exact."""
import numpy as np
import pytest

import paged_oracle as po

pytestmark = pytest.mark.gpu

ATOL = 3e-5


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


DT = {"f32": "float32", "bf16": "bfloat16", "e4m3": "float8_e4m3fn"}


class Pool:
    """A random cache on the device and what it stands for on the host; unused slots hold NaN and infinity."""

    def __init__(self, torch, lens, nH, H, hd, page, cache="bf16", track=False, seed=0, max_pages=None, spare=3, share=0):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        rows = len(lens)
        mp = max_pages or max(1, -(-max(lens) // page))
        n_pages = rows * mp + spare
        tab = rng.permutation(n_pages)[: rows * mp].reshape(rows, mp).astype(np.int32)
        if share:  # the first `share` pages are every row's
            tab[:, :share] = tab[0, :share]
        dt = getattr(torch, DT[cache])
        used = np.zeros((n_pages, page), bool)
        for r, n in enumerate(lens):
            at = np.arange(n)
            used[tab[r, at // page], at % page] = True
        junk = ~torch.from_numpy(used)[:, None, :, None].expand(n_pages, H, page, hd)

        def pool(bad):
            x = torch.randn((n_pages, H, page, hd), generator=g)
            x = (x * 90).clamp(-448, 448) if cache == "e4m3" else x
            x[junk] = bad
            return x.to(dt)

        k, v = pool(float("nan")), pool(float("nan") if cache == "e4m3" else float("inf"))
        self.k, self.v = k.cuda(), v.cuda()
        self.hk, self.hv = (x.to(torch.float64).numpy() for x in (k, v))
        self.ks = self.vs = None
        self.hks = self.hvs = None
        if cache == "e4m3":
            self.hks, self.hvs = ((rng.random(H) + 0.5).astype(np.float32) / np.float32(90) for _ in range(2))
            self.ks, self.vs = (torch.from_numpy(x).cuda() for x in (self.hks, self.hvs))
        self.weight = self.position = self.hw = self.hp = None
        if track:
            self.hw = (rng.exponential(size=(n_pages, H, page)) ** 2).astype(np.float32)
            self.hp = np.zeros((n_pages, H, page), np.int32)
            for r, n in enumerate(lens):
                at = np.arange(mp * page)
                self.hp[tab[r, at // page], :, at % page] = at[:, None]
            self.weight, self.position = torch.from_numpy(self.hw.copy()).cuda(), torch.from_numpy(self.hp.copy()).cuda()
        self.htab, self.hlens = tab, np.array(lens, np.int64)
        self.tables, self.lens = torch.from_numpy(tab).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
        from mxmoe.paged import PagedKvCache
        self.cache = PagedKvCache.over(self.k, self.v, nH, self.weight, self.position, self.ks, self.vs)


def check_decode(torch, lens, nH, H, hd, page, cache="bf16", q_dtype="bf16", out_dtype=None, window=0, sinks=False,
                 quiet=False, bias=None, track=False, seed=0, share=0, max_pages=None, scale=None, q_scale=2.0):
    P = Pool(torch, lens, nH, H, hd, page, cache, track, seed, share=share, max_pages=max_pages)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(len(lens), nH, hd, generator=g) * q_scale).to(getattr(torch, DT[q_dtype]))
    sk = torch.randn(nH, generator=g) if sinks else None
    lse = torch.empty(len(lens), nH, device="cuda")
    out = P.cache.decode(q.cuda(), P.tables, P.lens, scale=scale, window=window, sinks=None if sk is None else sk.cuda(),
                         quiet=quiet, bias=None if bias is None else torch.from_numpy(bias).cuda(), track=track,
                         out_dtype=getattr(torch, DT[out_dtype]) if out_dtype else None, lse=lse)
    again = P.cache.decode(q.cuda(), P.tables, P.lens, scale=scale, window=window, sinks=None if sk is None else sk.cuda(),
                           quiet=quiet, bias=None if bias is None else torch.from_numpy(bias).cuda(),
                           out_dtype=getattr(torch, DT[out_dtype]) if out_dtype else None)
    P.cache.sync_status()
    w = P.hw.astype(np.float64) if track else None
    want, want_lse = po.decode(q.to(torch.float64).numpy(), P.hk, P.hv, P.htab, P.hlens,
                               1 / np.sqrt(hd) if scale is None else scale, window,
                               None if sk is None else sk.numpy().astype(np.float64), quiet, bias, w, P.hks, P.hvs)
    got = out.to(torch.float64).cpu().numpy()
    kind = out_dtype or q_dtype
    atol = ATOL * (2 if bias is not None or cache == "e4m3" else 1) * max(1.0, q_scale / 2)
    assert np.all(np.isfinite(got))
    err = np.abs(got - want) - (2.0 ** -8 * np.abs(want) if kind == "bf16" else 0)
    assert err.max() <= atol, err.max()
    fin = np.isfinite(want_lse)
    got_lse = lse.cpu().numpy()
    assert np.array_equal(fin, np.isfinite(got_lse))
    assert np.all(np.abs(got_lse[fin] - want_lse[fin]) <= atol + 2e-6 * np.abs(want_lse[fin]))
    assert torch.equal(out.view(torch.uint8), again.view(torch.uint8))  # the same bits every time
    if track:
        gw = P.weight.cpu().numpy()
        assert np.all(np.abs(gw - w) <= 2e-5 * (w - P.hw) + 2.0 ** -23 * w)
    return P, out


HEADS = [(64, 8, 64), (8, 8, 64), (12, 4, 128), (10, 2, 80), (9, 1, 64), (16, 1, 128), (40, 1, 64), (4, 2, 256),
         (5, 5, 72), (6, 2, 8), (24, 2, 96)]


@pytest.mark.parametrize("nH,H,hd", HEADS)
@pytest.mark.parametrize("cache,q_dtype", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32"), ("e4m3", "bf16"),
                                           ("e4m3", "f32")])
def test_decode_heads_and_types(torch, nH, H, hd, cache, q_dtype):
    if cache == "e4m3" and hd % 16:
        pytest.skip("an 8-bit cache's heads are multiples of 16")
    check_decode(torch, [0, 1, 2, 15, 16, 17, 33, 130], nH, H, hd, 16, cache, q_dtype, sinks=True)


@pytest.mark.parametrize("page", [1, 3, 7, 8, 16, 24, 100, 256])
@pytest.mark.parametrize("cache", ["bf16", "e4m3", "f32"])
def test_decode_pages(torch, page, cache):
    check_decode(torch, [1, 95, 200, 0, 64], 8, 2, 64, page, cache, "f32")


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 128, 1000, 5000])
def test_decode_window(torch, window):
    check_decode(torch, [1, 16, 129, 700, 0], 16, 2, 64, 16, window=window, sinks=True)


@pytest.mark.parametrize("lens", [[6001], [3000, 1], [1] * 300, [20000, 0, 37, 4096, 511]])
@pytest.mark.parametrize("cache,hd", [("bf16", 64), ("e4m3", 128), ("f32", 80)])
def test_decode_long_and_many(torch, lens, cache, hd):
    check_decode(torch, lens, 8, 2, hd, 16, cache, "f32", quiet=True)


@pytest.mark.parametrize("H,nH", [(8, 64), (1, 9), (2, 2), (2, 32)])
@pytest.mark.parametrize("cache,q_dtype", [("bf16", "bf16"), ("e4m3", "bf16"), ("f32", "f32")])
def test_decode_track(torch, H, nH, cache, q_dtype):
    check_decode(torch, [0, 1, 17, 2500, 300], nH, H, 64, 16, cache, q_dtype, sinks=True, track=True)


def test_decode_track_with_quiet_softmax_and_bias(torch):
    rng = np.random.default_rng(3)
    bias = rng.standard_normal((3, 8, 700)).astype(np.float32)
    check_decode(torch, [700, 10, 333], 8, 2, 64, 8, quiet=True, bias=bias, track=True, q_dtype="f32")


@pytest.mark.parametrize("shape", [(3, 16, 600), (1, 16, 600), (3, 1, 600), (1, 1, 40)])
def test_decode_bias_shapes(torch, shape):
    bias = np.random.default_rng(1).standard_normal(shape).astype(np.float32)
    check_decode(torch, [600, 39, 41], 16, 2, 64, 16, q_dtype="f32", bias=bias)


def test_decode_rows_that_the_bias_empties(torch):
    """-inf for every key: zeros without sinks (or the formula with them); the type's lowest value for every key is
    a score like another, so the keys share evenly."""
    bias = np.zeros((3, 1, 100), np.float32)
    bias[0] = -np.inf
    bias[1] = np.finfo(np.float32).min
    bias[2, 0, :99] = -np.inf
    P, out = check_decode(torch, [100, 100, 100], 4, 2, 64, 16, q_dtype="f32", bias=bias)
    assert np.all(out[0].cpu().numpy() == 0)
    check_decode(torch, [100, 100, 100], 4, 2, 64, 16, q_dtype="f32", bias=bias, sinks=True)
    check_decode(torch, [100, 100, 100], 4, 2, 64, 16, q_dtype="f32", bias=bias, quiet=True)


def test_decode_sinks_of_minus_infinity_and_large_scores(torch):
    check_decode(torch, [50, 0], 8, 2, 64, 16, q_dtype="f32", scale=1e-30)
    check_decode(torch, [300, 5], 8, 2, 64, 16, q_dtype="f32", q_scale=60.0)
    P = Pool(torch, [40, 0], 4, 2, 64, 16)
    q = torch.randn(2, 4, 64, device="cuda")
    gone = torch.full((4,), float("-inf"), device="cuda")
    a = P.cache.decode(q, P.tables, P.lens, sinks=gone)
    assert torch.equal(a, P.cache.decode(q, P.tables, P.lens)) and torch.all(a[1] == 0)


def test_decode_nan_stays_in_its_row(torch):
    P = Pool(torch, [300, 300, 40], 8, 2, 64, 16)
    q = torch.randn(3, 8, 64, device="cuda").bfloat16()
    want = P.cache.decode(q, P.tables, P.lens)
    q[1, 3, 5] = float("nan")
    got = P.cache.decode(q, P.tables, P.lens)
    assert torch.all(got[1, 3].isnan())
    keep = torch.ones(3, 8, dtype=torch.bool)
    keep[1, 3] = False
    assert torch.equal(got[keep], want[keep])


def test_decode_shared_prefix_and_several_tokens_of_one_sequence(torch):
    check_decode(torch, [70, 90, 65], 8, 2, 64, 16, share=4)
    P = Pool(torch, [200], 8, 2, 64, 16)
    q = torch.randn(4, 8, 64, device="cuda")
    lens = torch.tensor([197, 198, 199, 200], dtype=torch.int32, device="cuda")
    got = P.cache.decode(q, P.tables.expand(4, -1), lens)
    want, _ = po.decode(q.double().cpu().numpy(), P.hk, P.hv, P.htab.repeat(4, 0), [197, 198, 199, 200], 1 / 8)
    assert np.abs(got.cpu().numpy() - want).max() <= ATOL


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decode_strides_alignment_and_stream(torch, dtype):
    P = Pool(torch, [100, 33], 8, 2, 64, 16)
    dt = getattr(torch, DT[dtype])
    base = torch.randn(2 * 8 * 100 + 1, device="cuda").to(dt)
    q = base[1:].view(2, 8, 100)[:, :, 3:67]  # heads 100 apart, one element off every wider alignment
    want = P.cache.decode(q.contiguous(), P.tables, P.lens)
    hole = torch.zeros(2 * 8 * 77 + 1, device="cuda", dtype=dt)
    out = hole[1:].view(8, 2, 77).transpose(0, 1)[:, :, :64]
    wide = torch.zeros(2, P.tables.shape[1] + 5, dtype=torch.int32, device="cuda")
    wide[:, : P.tables.shape[1]] = P.tables
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        P.cache.decode(q, wide[:, : P.tables.shape[1]], P.lens, out=out)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want)
    assert torch.count_nonzero(hole) == torch.count_nonzero(out)  # nothing beside it


def test_calls_in_a_cuda_graph(torch):
    P = Pool(torch, [100, 2000], 16, 2, 64, 16, track=True)
    q = torch.randn(2, 16, 64, device="cuda").bfloat16()
    want = P.cache.decode(q, P.tables, P.lens)
    out = torch.empty_like(want)
    new = torch.empty_like(P.lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        P.cache.decode(q, P.tables, P.lens, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            P.cache.decode(q, P.tables, P.lens, out=out)
            P.cache.evict(P.tables, P.lens, P.lens, 1000, recent=10, new_lens=new)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and new.tolist() == [100, 1000]


def test_what_is_out_of_range_is_skipped_and_reported(torch):
    from mxmoe import MxMoeError
    P = Pool(torch, [40, 40], 8, 2, 64, 16, track=True)
    q = torch.randn(2, 8, 64, device="cuda")
    P.cache.decode(q, P.tables, P.lens)
    P.cache.sync_status()
    want = P.cache.decode(q, P.tables, P.lens)
    tab = P.tables.clone()
    tab[0, 1] = 1 << 30
    tab[0, 2] = -5
    got = P.cache.decode(q, tab, P.lens)
    with pytest.raises(MxMoeError, match="table entry"):
        P.cache.sync_status()
    P.cache.sync_status()
    assert torch.equal(got[1], want[1])
    first = torch.tensor([16, 40], dtype=torch.int32, device="cuda")
    assert torch.allclose(got[0], P.cache.decode(q, P.tables, first)[0], atol=ATOL)
    lens = torch.tensor([1 << 30, -3], dtype=torch.int32, device="cuda")
    P.v.zero_()
    P.k.zero_()
    got = P.cache.decode(q, P.tables, lens)
    with pytest.raises(MxMoeError, match="length"):
        P.cache.sync_status()
    assert torch.all(got == 0)
    before = P.k.clone(), P.v.clone(), P.weight.clone(), P.position.clone()
    k = torch.randn(4, 2, 64, device="cuda")
    P.cache.append(None, k, k, tab, torch.tensor([1 << 29, 20, 5, 5], dtype=torch.int32, device="cuda"),
                   rows=torch.tensor([1, 0, 7, -1], dtype=torch.int32, device="cuda"))
    with pytest.raises(MxMoeError, match="index"):
        P.cache.sync_status()
    for a, b in zip(before, (P.k, P.v, P.weight, P.position)):
        assert torch.equal(a, b)
    P.cache.evict(tab, P.lens, P.lens, 30)
    with pytest.raises(MxMoeError, match="table entry"):
        P.cache.sync_status()


# ---- append ----


def e4m3_close(got, x):
    """got is x to within half a step of its binade (and a little of the product before)."""
    e = np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -20))), -6)
    step = 2.0 ** (e - 3)
    x = np.clip(x, -448, 448)
    return np.abs(got - x) <= step * (0.5 + 1e-3)


def same_values(kind, got, want):
    if kind == "e4m3":
        return e4m3_close(got, want).all()
    tol = 6e-6 + (2.0 ** -8 + 2.0 ** -20) * np.abs(want) * (kind == "bf16")
    return (np.abs(got - want) <= tol).all()


def table(torch, rot, n, interleaved=False, **kw):
    from mxmoe.paged import RotaryConfig, RotaryTable
    return RotaryTable.of(RotaryConfig(rot, **kw), n, interleaved)


@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 32), (128, 128), (80, 80), (72, 36), (96, 6), (16, 2), (256, 256),
                                    (64, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f32", "e4m3"), ("f32", "f32"), ("bf16", "e4m3"),
                                         ("f32", "bf16"), ("bf16", "f32")])
def test_append(torch, hd, rot, interleaved, dtype, cache):
    if cache == "e4m3" and hd % 16:
        pytest.skip("an 8-bit cache's heads are multiples of 16")
    nH, H, page = 6, 2, 7
    P = Pool(torch, [30, 12, 0], nH, H, hd, page, cache, track=True, max_pages=8)
    rows = np.array([0, 0, 1, 2, 2, 1, 0, 2, 0], np.int32)
    index = np.array([30, 31, 12, 0, 1, 13, -1, 55, 33], np.int32)
    pos = np.array([30, 31, 500, 1000, 3, 13, 77, 55, 2047], np.int32)
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(9, (nH + 2 * H) * hd, generator=g).to(getattr(torch, DT[dtype])).cuda()
    q, k, v = (x.unflatten(1, (-1, hd)) for x in qkv.split([nH * hd, H * hd, H * hd], 1))
    r = table(torch, rot, 2048, interleaved) if rot else None
    inv, f = po.frequencies(rot) if rot else (np.zeros(0), 1.0)
    k_out = torch.zeros(9, H, hd, dtype=k.dtype, device="cuda")
    keep = [x.cpu().clone() for x in (qkv, P.weight, P.position)]
    got = P.cache.append(q, k, v, P.tables, torch.from_numpy(index).cuda(), r, torch.from_numpy(pos).cuda(),
                         torch.from_numpy(rows).cuda(), k_out=k_out)
    P.cache.sync_status()
    assert torch.equal(qkv.cpu(), keep[0])

    def host(x):
        return x.detach().to(torch.float64).cpu().numpy()

    wq, wk = (po.rotate(host(x), pos, inv, f, interleaved) for x in (q, k))
    assert same_values(dtype, host(got), wq) and same_values(dtype, host(k_out), wk)
    nk, nv, written = host(P.k), host(P.v), np.zeros(P.hk.shape[:3], bool)
    for t in range(9):
        if index[t] < 0:
            continue
        pg, sl = po.place(P.htab, page, rows[t], index[t])
        written[pg, :, sl] = True
        s = 1.0 if P.hks is None else P.hks[:, None].astype(np.float64)
        z = 1.0 if P.hvs is None else P.hvs[:, None].astype(np.float64)
        assert same_values(cache, nk[pg, :, sl], wk[t] / s)
        assert same_values(cache, nv[pg, :, sl], host(v)[t] / z)
        assert torch.all(P.weight[pg, :, sl] == 0) and torch.all(P.position[pg, :, sl] == int(pos[t]))
    other = torch.from_numpy(~written)
    for now, was in ((nk, P.hk), (nv, P.hv)):
        assert np.array_equal(now[~written], was[~written], equal_nan=True)
    assert torch.equal(P.weight.cpu()[other], keep[1][other]) and torch.equal(P.position.cpu()[other], keep[2][other])


@pytest.mark.parametrize("tokens", [1, 2, 63, 700])
def test_append_token_by_row_in_place(torch, tokens):
    """Without rows and positions: token t is row t, its position its cache index; queries and keys in place."""
    lens = [(7 * i) % 50 + 1 for i in range(tokens)]
    P = Pool(torch, lens, 64, 8, 64, 16, max_pages=5)
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(tokens, n, 64, generator=g).bfloat16().cuda() for n in (64, 8, 8))
    hq, hk = (x.double().cpu().numpy() for x in (q, k))
    index = P.lens.clone()
    out = P.cache.append(q, k, v, P.tables, index, table(torch, 64, 64), q_out=q, k_out=k)
    assert out is q
    inv, f = po.frequencies(64)
    wk = po.rotate(hk, lens, inv, f)
    assert same_values("bf16", q.double().cpu().numpy(), po.rotate(hq, lens, inv, f))
    assert same_values("bf16", k.double().cpu().numpy(), wk)
    for t in range(tokens):
        pg, sl = po.place(P.htab, 16, t, lens[t])
        assert torch.equal(P.k[pg, :, sl], k[t]) and torch.equal(P.v[pg, :, sl], v[t])


@pytest.mark.parametrize("dtype,cache,interleaved", [("bf16", "bf16", False), ("f32", "e4m3", True), ("f32", "f32", False)])
def test_append_more_tokens_than_blocks(torch, dtype, cache, interleaved):
    """Blocks that take one token after another, more than they look up together, places among them that are not written."""
    T, hd, nH, H = 13001, 16, 3, 1
    lens = [4334, 4334, 4334]
    P = Pool(torch, lens, nH, H, hd, 16, cache)
    t = np.arange(T)
    rows, index = (t % 3).astype(np.int32), np.where(t % 11 == 5, -1, t // 3).astype(np.int32)
    pos = (t * 7 % 4001).astype(np.int32)
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(T, n, hd, generator=g).to(getattr(torch, DT[dtype])).cuda() for n in (nH, H, H))
    got = P.cache.append(q, k, v, P.tables, torch.from_numpy(index).cuda(), table(torch, 8, 4001, interleaved),
                         torch.from_numpy(pos).cuda(), torch.from_numpy(rows).cuda())
    P.cache.sync_status()
    inv, f = po.frequencies(8)
    wq, wk = (po.rotate(x.double().cpu().numpy(), pos, inv, f, interleaved) for x in (q, k))
    assert same_values(dtype, got.double().cpu().numpy(), wq)
    s, z = (1.0, 1.0) if P.hks is None else (P.hks[0].astype(np.float64), P.hvs[0].astype(np.float64))
    hk, hv = (x.to(torch.float64).cpu().numpy() for x in (P.k, P.v))
    on = index >= 0
    page, slot = P.htab[rows[on], index[on] // 16], index[on] % 16
    assert same_values(cache, hk[page, 0, slot], wk[on, 0] / s)
    assert same_values(cache, hv[page, 0, slot], v.double().cpu().numpy()[on, 0] / z)
    off = P.htab[rows[~on], (t // 3)[~on] // 16], (t // 3)[~on] % 16
    assert np.array_equal(hk[off[0], 0, off[1]], P.hk[off[0], 0, off[1]], equal_nan=True)


@pytest.mark.parametrize("shift", [0, 1, 3])
def test_append_strides_and_alignment(torch, shift):
    hd, nH, H = 64, 4, 2
    P = Pool(torch, [5, 5, 5], nH, H, hd, 4, max_pages=4)
    buf = torch.randn(3 * (nH + 2 * H) * 70 + shift, device="cuda").bfloat16()
    x = buf[shift:].view(nH + 2 * H, 3, 70).transpose(0, 1)[..., :hd]
    q, k, v = x[:, :nH], x[:, nH:nH + H], x[:, nH + H:]
    r = table(torch, 64, 100)
    room = torch.zeros(nH * 3 * 66 + shift, device="cuda").bfloat16()
    out = room[shift:].view(nH, 3, 66).transpose(0, 1)[..., :hd]
    P.cache.append(q, k, v, P.tables, P.lens, r, q_out=out)
    a = (P.k.clone(), P.v.clone())
    want = P.cache.append(q.contiguous(), k.contiguous(), v.contiguous(), P.tables, P.lens, r)
    assert torch.equal(out, want)
    assert torch.equal(a[0].view(torch.int16), P.k.view(torch.int16)) and torch.equal(a[1].view(torch.int16), P.v.view(torch.int16))
    assert torch.count_nonzero(room) == torch.count_nonzero(out)


@pytest.mark.parametrize("scaling", ["plain", "linear", "ntk", "yarn", "streaming"])
def test_rotary_tables(torch, scaling):
    from mxmoe.paged import RotaryConfig, RotaryTable
    n = 131072
    r = RotaryTable.of(RotaryConfig(64, scaling=scaling, scaling_factor=32.0), n)
    inv, f = po.frequencies(64, scaling=scaling, factor=32.0)
    pos = np.array([0, 1, 2, 100, 4095, 131071] if scaling != "streaming" else [0, 1, 2, 100])
    angle = pos[:, None] * inv
    # 2^-24 of an entry; the oracle's "streaming" frequencies are rounded to 32 bits, 4e-7 of the angle
    tol = 1e-7 * f if scaling != "streaming" else 1e-7 * f + 4e-7 * angle
    assert np.all(np.abs(r.cos.cpu().numpy()[pos] - f * np.cos(angle)) <= tol)
    assert np.all(np.abs(r.sin.cpu().numpy()[pos] - f * np.sin(angle)) <= tol)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,rot", [(64, 64), (80, 20), (7, 6)])
def test_rotary_gradient(torch, interleaved, hd, rot):
    """The inverse turn is the gradient: against the transposed formula, and against differences of the turn (it is
    linear, so central differences of a power of two have rounding error only: 2 x 1e-6 over a step of 2)."""
    g = torch.Generator().manual_seed(2)
    x, up = (torch.randn(5, 3, hd, generator=g).cuda() for _ in range(2))
    pos = torch.tensor([0, 1, 77, 500, 999], dtype=torch.int32, device="cuda")
    r = table(torch, rot, 1000, interleaved, scaling="yarn", scaling_factor=8.0)
    inv, f = po.frequencies(rot, scaling="yarn", factor=8.0)
    grad = r.apply(up, pos, inverse=True).cpu().numpy()
    want = po.rotate(up.cpu().numpy(), pos.cpu().numpy(), inv, f, interleaved, inverse=True)
    assert np.abs(grad - want).max() <= 6e-6
    for col in range(hd):
        step = torch.zeros_like(x)
        step[..., col] = 1.0
        diff = (r.apply(x + step, pos) - r.apply(x - step, pos)) / 2
        assert np.abs((diff * up).sum(-1).cpu().numpy() - grad[..., col]).max() <= 2e-5
    back = r.apply(r.apply(x, pos), pos, inverse=True) / f ** 2
    assert np.abs((back[..., :rot] - x[..., :rot]).cpu().numpy()).max() <= 1.2e-5
    y = x.clone()
    assert torch.equal(r.apply(y, pos, out=y), r.apply(x, pos))


# ---- evict ----


def check_evict(torch, lens, budget, sink, recent, H=2, hd=64, page=16, cache="bf16", seed=0, mutate=None, seen=None,
                in_place=False):
    P = Pool(torch, lens, H * 2, H, hd, page, cache, track=True, seed=seed)
    seen = np.array(lens if seen is None else seen, np.int32)
    if mutate:
        mutate(P)
        P.weight.copy_(torch.from_numpy(P.hw))
        P.position.copy_(torch.from_numpy(P.hp))
    new = P.lens if in_place else None
    got = P.cache.evict(P.tables, P.lens, torch.from_numpy(seen).cuda(), budget, sink, recent, new_lens=new)
    P.cache.sync_status()
    hk, hv = P.hk.copy(), P.hv.copy()
    want = po.evict(hk, hv, P.hw, P.hp, P.htab, P.hlens, seen, budget, sink, recent)
    assert np.array_equal(got.cpu().numpy(), want)
    assert np.array_equal(P.position.cpu().numpy(), P.hp)
    assert np.array_equal(P.weight.cpu().numpy(), P.hw, equal_nan=True)
    for x, y in ((P.k, hk), (P.v, hv)):
        assert np.array_equal(x.to(torch.float64).cpu().numpy(), y, equal_nan=True)


@pytest.mark.parametrize("cache,hd", [("bf16", 64), ("f32", 8), ("e4m3", 16), ("e4m3", 128), ("bf16", 72), ("f32", 256)])
@pytest.mark.parametrize("page", [1, 7, 16])
def test_evict_types_and_pages(torch, cache, hd, page):
    check_evict(torch, [100, 0, 40, 41, 64, 1], 40, 4, 10, hd=hd, page=page, cache=cache)


@pytest.mark.parametrize("lens,budget", [([2049], 2048), ([2048, 2047], 2048), ([5000, 1025, 3000], 1024),
                                         ([12000], 11000), ([9000], 17), ([40000, 33000], 20000), ([2, 1, 0, 3], 1)])
def test_evict_lengths(torch, lens, budget):
    check_evict(torch, lens, budget, min(4, budget // 2), budget // 4, H=1)


@pytest.mark.parametrize("alike", [False, True])
@pytest.mark.parametrize("lens,budget", [([9000], 8800), ([16380, 8193, 40], 8192), ([20000], 4001), ([24570, 100], 16000)])
def test_evict_rows_of_several_blocks(torch, lens, budget, alike):
    """Three to six blocks of a row, shares that end short, weights that are nearly all alike."""
    def few(P):
        P.hw[:] = np.random.default_rng(2).integers(0, 2, P.hw.shape).astype(np.float32)

    check_evict(torch, lens, budget, 4, budget // 4, mutate=few if alike else None)


@pytest.mark.parametrize("length,budget", [(160000, 40000), (190000, 189000), (200000, 150000)])
def test_evict_the_longest_rows(torch, length, budget):
    """Seven and eight blocks of a row, and rows too long for that."""
    check_evict(torch, [length, 300], budget, 4, 1000, H=1, hd=16)


def test_evict_ties_zeros_and_nan(torch):
    def ties(P):
        P.hw[:] = np.random.default_rng(0).integers(0, 3, P.hw.shape).astype(np.float32)
        P.hw[P.hw == 1] = -0.0

    def odd(P):
        u = np.random.default_rng(1).random(P.hw.shape)
        P.hw[u < 0.2] = np.nan
        P.hw[(u >= 0.2) & (u < 0.4)] = np.inf
        P.hw[(u >= 0.4) & (u < 0.5)] = -np.inf
        P.hw[(u >= 0.5) & (u < 0.6)] = -2.5
        P.hw[(u >= 0.6) & (u < 0.7)] = 1e-42

    def same(P):
        P.hw[:] = 0.25

    for m in (ties, odd, same):
        for lens, budget in (([300, 90], 70), ([3000], 2500), ([3000], 300)):
            check_evict(torch, lens, budget, 2, 20, mutate=m)


def test_evict_positions_out_of_order(torch):
    def shuffle(P):
        rng = np.random.default_rng(4)
        for r, n in enumerate(P.hlens):
            at = np.arange(n)
            for h in range(P.hp.shape[1]):
                P.hp[P.htab[r, at // 16], h, at % 16] = rng.permutation(3 * n)[:n]

    check_evict(torch, [500, 1300], 400, 30, 200, mutate=shuffle, seen=[1500, 3900])

    def guarded(P):  # more protected than the budget holds: the first of them leave
        P.hp[:] = 0

    check_evict(torch, [500, 1300], 400, 30, 200, mutate=guarded)


def test_evict_in_place_lens(torch):
    check_evict(torch, [500, 20, 130], 100, 4, 50, H=8, in_place=True)


@pytest.mark.parametrize("max_pages", [300, 2000, 13000])
def test_evict_under_wide_tables(torch, max_pages):
    """Tables far wider than the rows: the work is laid out by what a row could hold."""
    P = Pool(torch, [900, 30, 513], 4, 2, 64, 16, track=True)
    wide = torch.full((3, max_pages), -1, dtype=torch.int32, device="cuda")
    wide[:, : P.tables.shape[1]] = P.tables
    got = P.cache.evict(wide, P.lens, P.lens, 300, 4, 50)
    P.cache.sync_status()
    want = po.evict(P.hk, P.hv, P.hw, P.hp, P.htab, P.hlens, P.hlens, 300, 4, 50)
    assert np.array_equal(got.cpu().numpy(), want) and np.array_equal(P.position.cpu().numpy(), P.hp)
    assert np.array_equal(P.weight.cpu().numpy(), P.hw)
    for x, y in ((P.k, P.hk), (P.v, P.hv)):
        assert np.array_equal(x.to(torch.float64).cpu().numpy(), y, equal_nan=True)


def test_steps_of_a_thinned_conversation(torch):
    """append, decode and evict together over 40 steps against the oracle: the cache never grows past its budget."""
    nH, H, hd, page, budget, rows = 8, 2, 64, 8, 24, 3
    from mxmoe.paged import PagedKvCache
    mp = budget // page + 1
    cache = PagedKvCache(rows * mp, page, nH, H, hd, torch.float32, track=True)
    tab = np.random.default_rng(0).permutation(rows * mp).reshape(rows, mp).astype(np.int32)
    tables = torch.from_numpy(tab).cuda()
    hk, hv = (np.zeros(cache.k.shape) for _ in range(2))
    hw, hp = np.zeros(cache.k.shape[:3]), np.zeros(cache.k.shape[:3], np.int32)
    r = table(torch, hd, 64)
    inv, f = po.frequencies(hd)
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    hl = np.zeros(rows, np.int64)
    g = torch.Generator().manual_seed(9)
    for step in range(40):
        q, k, v = (torch.randn(rows, n, hd, generator=g) for n in (nH, H, H))
        pos = np.full(rows, step, np.int32)
        qr = cache.append(q.cuda(), k.cuda(), v.cuda(), tables, lens, r, torch.from_numpy(pos).cuda())
        lens = lens + 1
        out = cache.decode(qr, tables, lens, track=True)
        wq, wk = (po.rotate(x.numpy(), pos, inv, f) for x in (q, k))
        for i in range(rows):
            pg, sl = po.place(tab, page, i, hl[i])
            hk[pg, :, sl], hv[pg, :, sl], hw[pg, :, sl], hp[pg, :, sl] = wk[i], v[i].numpy(), 0, step
        hl += 1
        want, _ = po.decode(wq, hk, hv, tab, hl, 1 / np.sqrt(hd), weight=hw)
        assert np.abs(out.cpu().numpy() - want).max() <= 1e-4
        lens = cache.evict(tables, lens, torch.full((rows,), step + 1, dtype=torch.int32, device="cuda"), budget, 2, 8)
        hl = po.evict(hk, hv, hw, hp, tab, hl, np.full(rows, step + 1), budget, 2, 8)
        assert np.array_equal(cache.position.cpu().numpy(), hp)
    cache.sync_status()
    assert lens.tolist() == [budget] * rows


def test_offsets_past_32_bits(torch):
    """Pages whose byte and element offsets pass 2^32 (two pools of 4.3 GB, left unwritten but for what the test uses)."""
    from mxmoe.paged import PagedKvCache
    page, H, hd = 64, 2, 256
    n_pages = (1 << 32) // (page * H * hd) + 8
    k = torch.empty(n_pages, H, page, hd, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    v = torch.empty_like(k)
    w = torch.zeros(n_pages, H, page, device="cuda")
    p = torch.zeros(n_pages, H, page, dtype=torch.int32, device="cuda")
    cache = PagedKvCache.over(k, v, 4, w, p)
    tables = torch.tensor([[n_pages - 1, n_pages - 3], [0, 1]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(3)
    n = 100
    kk, vv = (torch.randn(n, H, hd, generator=g).cuda() for _ in range(2))
    for row in range(2):
        cache.append(None, kk, vv, tables, torch.arange(n, dtype=torch.int32, device="cuda"),
                     rows=torch.full((n,), row, dtype=torch.int32, device="cuda"))
    q = torch.randn(1, 4, hd, generator=g).cuda()
    lens = torch.tensor([n, n], dtype=torch.int32, device="cuda")
    out = [cache.decode(q, tables[i:i + 1], lens[i:i + 1], track=True) for i in range(2)]
    assert torch.equal(out[0], out[1]) and float(out[0].abs().max()) > 0
    cache.evict(tables, lens, lens, 60, 2, 5)
    cache.sync_status()
    for x in (k.view(torch.uint8), v.view(torch.uint8), w, p):
        assert torch.equal(x[n_pages - 1], x[0]) and torch.equal(x[n_pages - 3][:, : n - page], x[1][:, : n - page])


def test_refusals_with_a_device(torch):
    from mxmoe import MxMoeError
    from mxmoe.paged import PagedKvCache, RotaryConfig, RotaryTable
    P = Pool(torch, [40, 40], 8, 2, 64, 16)
    q = torch.randn(2, 8, 64, device="cuda")
    k = torch.randn(2, 2, 64, device="cuda")

    def refused(f, match):
        with pytest.raises(MxMoeError, match=match):
            f()

    d = P.cache.decode
    refused(lambda: d(q[:, :7], P.tables, P.lens), "q: expected")
    refused(lambda: d(q.half(), P.tables, P.lens), "unsupported dtype")
    refused(lambda: d(q.cpu(), P.tables, P.lens), "expected a tensor")
    refused(lambda: d(q, P.tables[:1], P.lens), "tables")
    refused(lambda: d(q, P.tables.long(), P.lens), "tables")
    refused(lambda: d(q, P.tables, P.lens.long()), "lens")
    refused(lambda: d(q, P.tables, P.lens[:1]), "lens")
    refused(lambda: d(q, P.tables, P.lens, window=-1), "window")
    refused(lambda: d(q, P.tables, P.lens, sinks=torch.zeros(7, device="cuda")), "sinks")
    refused(lambda: d(q, P.tables, P.lens, bias=torch.zeros(2, 3, 40, device="cuda")), "bias")
    refused(lambda: d(q, P.tables, P.lens, track=True), "weight buffer")
    refused(lambda: d(q, P.tables, P.lens, scale=float("nan")), "finite")
    refused(lambda: d(q, P.tables, P.lens, out=torch.zeros(2, 8, 63, device="cuda")), "out")
    refused(lambda: P.cache.evict(P.tables, P.lens, P.lens, 10), "weight and position")
    T = Pool(torch, [40, 40], 8, 2, 64, 16, track=True)
    refused(lambda: T.cache.evict(T.tables, T.lens, T.lens, 10, 4, 7), "above the budget")
    refused(lambda: T.cache.evict(T.tables, T.lens, T.lens, 0, 0, 0), "budget")
    refused(lambda: T.cache.decode(q, T.tables, T.lens, track=True, window=5), "window must be 0")
    r = table(torch, 64, 10)
    a = P.cache.append
    refused(lambda: a(q, k, k, P.tables, P.lens[:1], r), "index")
    refused(lambda: a(q, k, k.bfloat16(), P.tables, P.lens, r), "v: expected")
    refused(lambda: a(q.bfloat16(), k, k, P.tables, P.lens, r), "q: expected")
    refused(lambda: a(None, k, k, P.tables[:1], P.lens, r), "need `rows`")
    refused(lambda: a(None, k, k, P.tables, P.lens, r, q_out=q), "q_out without q")
    refused(lambda: a(q, k, k, P.tables, P.lens, table(torch, 66, 10)), "rot_dim")
    refused(lambda: RotaryTable.of(RotaryConfig(63), 10), "rot_dim")
    refused(lambda: RotaryTable.of(RotaryConfig(64, scaling="cubic"), 10), "scaling")
    refused(lambda: RotaryTable.of(RotaryConfig(64, theta=-1.0), 10), "theta")
    refused(lambda: r.apply(q[0], P.lens), "x: expected")
    refused(lambda: PagedKvCache(4, 16, 8, 3, 64), "divisible")
    refused(lambda: PagedKvCache(4, 16, 8, 2, 60), "multiple of 8")
    refused(lambda: PagedKvCache(4, 16, 8, 2, 264), "at most 256")
    refused(lambda: PagedKvCache(4, 16, 8, 2, 24, torch.float8_e4m3fn), "multiple of 8")
    refused(lambda: PagedKvCache(4, 16, 8, 2, 64, torch.float16), "unsupported cache dtype")
    refused(lambda: PagedKvCache(4, 16, 8, 2, 64, k_scale=torch.ones(2, device="cuda")), "8-bit cache")
    refused(lambda: PagedKvCache(0, 16, 8, 2, 64), "zero dimension")
    # nothing to do is not an error
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert d(q[:0], P.tables[:0], none).shape == (0, 8, 64)
    assert a(q[:0], k[:0], k[:0], P.tables, none, r, rows=none).shape == (0, 8, 64)
