"""rai_b200.paged.attention against plain attention in 64 bits: types, head
layouts, ragged lengths, masks, and what masked places may hold."""
import itertools
import math

import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def run(cache, q, rows, *, scale=None, softcap=0.0, window=0, first=0, max_rows=None, with_lse=True, **kw):
    from rai_b200 import paged
    dev = q.device
    lse = torch.full(q.shape[:2], 7.0, device=dev) if with_lse else None
    out = kw.pop("out", None)
    if out is None:
        out = torch.full(q.shape, 3.0, dtype=q.dtype, device=dev)
    got = paged.attention(q, cache.k, cache.v, cache.table, cache.kv_len, ref.starts_of(rows, dev, first),
                          max(rows) if max_rows is None else max_rows, scale=scale, softcap=softcap, window=window, out=out,
                          lse=lse, **kw)
    paged.status()
    return got, lse


def agree(cache, q, rows, got, lse, *, scale=None, softcap=0.0, window=0, first=0):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, bound, wlse = ref.attention(q, cache, rows, scale, softcap, window, first)
    a, b = first, first + sum(rows)
    g, w = got[a:b].double(), want[a:b]
    fine = torch.isfinite(w)
    assert torch.equal(torch.isfinite(g), fine), "finite where it should not be, or the other way"
    assert torch.equal(torch.isnan(g), torch.isnan(w))
    over = torch.where(fine, (g - w).abs() / bound[a:b], 0.0)
    assert over.max() <= 1.0, f"off by {over.max():.3g} times the bound at {over.argmax()}"
    if lse is not None:
        d = (lse[a:b].double() - wlse[a:b])
        empty = wlse[a:b] == -math.inf
        assert torch.equal(lse[a:b] == -math.inf, empty)
        # Scores off by d, sums of up to n terms in f32.
        tol = 2.0 ** -18 * (1 + wlse[a:b].abs()) + softcap * 2.0 ** -20
        assert (d[~empty].abs() <= tol[~empty]).all(), d[~empty].abs().max()
    # Rows of no sequence are left as they were.
    assert (got[:a] == 3.0).all() and (got[b:] == 3.0).all()


def make_q(T, H, D, dtype, dev, seed=1, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn((T, H, D), generator=g)).to(dtype).to(dev)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("heads,nkv,hd", [(14, 2, 64), (32, 8, 128), (4, 4, 32), (6, 2, 96), (15, 5, 80), (4, 2, 256),
                                          (8, 1, 16), (5, 1, 136)])
@pytest.mark.parametrize("wide", [0, 2000])
def test_shapes_and_lengths(dtype, heads, nkv, hd, wide):
    """A table for longer sequences than there are (wide) may choose another
    kernel."""
    dev = torch.device("cuda", 0)
    rows = [1, 2, 0, 9, 1, 5, 1, 1]
    lens = [1, 64, 7, 65, 200, 5, 63, 129]
    c = ref.Cache(lens, nkv, hd, 16, dtype, dev, seed=hd, wide=wide)
    q = make_q(sum(rows) + 4, heads, hd, dtype, dev)
    got, lse = run(c, q, rows, first=2)
    agree(c, q, rows, got, lse, first=2)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("page", [1, 3, 16, 100, 256])
@pytest.mark.parametrize("softcap,window", [(0.0, 0), (20.0, 0), (0.0, 1), (0.0, 70), (5.0, 33)])
@pytest.mark.parametrize("rows", [[3, 1, 12, 40], [3, 1, 12, 20]], ids=["many", "few"])
def test_pages_caps_and_windows(dtype, page, softcap, window, rows):
    dev = torch.device("cuda", 0)
    lens = [3, 300, 130, 140]
    hd = 64 if sum(rows) > 50 else 128
    c = ref.Cache(lens, 2, hd, page, dtype, dev, seed=page, wide=1 + 40000 // page)
    q = make_q(sum(rows), 6, hd, dtype, dev, scale=2.0)
    got, lse = run(c, q, rows, softcap=softcap, window=window)
    agree(c, q, rows, got, lse, softcap=softcap, window=window)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("heads,nkv,hd", [(8, 2, 64), (8, 2, 128), (2, 2, 256)])
@pytest.mark.parametrize("softcap,window", [(0.0, 0), (30.0, 100)])
def test_long_chunks(dtype, heads, nkv, hd, softcap, window):
    """Hundreds of rows: several row tiles, cut over the CTAs."""
    dev = torch.device("cuda", 0)
    rows = [300, 1, 129, 64, 257]
    lens = [300, 900, 700, 64, 1025]
    c = ref.Cache(lens, nkv, hd, 32, dtype, dev, seed=hd + 1)
    q = make_q(sum(rows) + 3, heads, hd, dtype, dev)
    got, lse = run(c, q, rows, softcap=softcap, window=window)
    agree(c, q, rows, got, lse, softcap=softcap, window=window)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,lens", [([1], [5000]), ([1, 1], [9000, 3]), ([9, 4, 1], [4000, 6500, 2500]),
                                       ([33], [3000]), ([1] * 40, list(range(200, 4200, 100))), ([2, 1, 3] * 9, [1500, 1100, 4000] * 9)])
def test_few_long_sequences_are_cut(dtype, rows, lens):
    dev = torch.device("cuda", 0)
    c = ref.Cache(lens, 2, 64, 16, dtype, dev, seed=len(lens))
    q = make_q(sum(rows), 8, 64, dtype, dev)
    got, lse = run(c, q, rows)
    agree(c, q, rows, got, lse)
    again, _ = run(c, q, rows)
    assert torch.equal(got, again)  # the same bits every time


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [[5, 3, 150, 200], [5, 3, 40, 7]], ids=["many", "few"])
@pytest.mark.parametrize("wide", [0, 2000])
def test_rows_that_see_nothing(dtype, hd, rows, wide):
    """kv_len below the row count: the first rows stand before the sequence."""
    dev = torch.device("cuda", 0)
    lens = [2, 0, 30, 1]
    c = ref.Cache(lens, 2, hd, 16, dtype, dev, wide=wide)
    q = make_q(sum(rows), 4, hd, dtype, dev)
    got, lse = run(c, q, rows)
    agree(c, q, rows, got, lse)
    assert (got[:3] == 0).all() and (lse[5:8] == -math.inf).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,window", [(6, 0), (6, 40), (160, 0), (300, 90)])
@pytest.mark.parametrize("wide", [0, 10000])
def test_what_is_masked_does_not_matter(dtype, hd, rows, window, wide):
    """NaN and infinities in later tokens, in tokens behind the window, in
    unused slots: only rows that see them change."""
    dev = torch.device("cuda", 0)
    n = rows + 300
    c = ref.Cache([n], 2, hd, 16, dtype, dev, seed=rows, wide=wide)
    q = make_q(rows, 4, hd, dtype, dev)

    def token(t):
        return c.rows[0][t // 16], t % 16
    p, s = token(n - 3)
    c.v[p, :, s, 5] = math.nan
    c.k[p, 0, s] = math.inf
    p, s = token(n - 2)
    c.v[p, 1, s] = math.inf
    p, s = token(n - rows // 2)
    c.v[p, 0, s, :3] = -math.inf
    if window:
        p, s = token(10)
        c.v[p, :, s] = math.nan
        c.k[p, :, s] = math.nan
    got, _ = run(c, q, [rows], window=window, with_lse=False)
    want, bound, _ = ref.attention(q, c, [rows], hd ** -0.5, 0.0, window)
    # K of KV head 0 at n - 3 is infinite: its rows from there on are NaN or
    # saturated; the others are held to their bounds.
    g, w = got.double(), want
    safe = torch.ones(rows, 4, dtype=torch.bool, device=dev)
    safe[rows - 3:, :2] = False
    fine = torch.isfinite(w) & safe[:, :, None]
    assert ((g - w).abs() <= bound)[fine].all()
    assert not torch.isfinite(g[(~torch.isfinite(w)) & safe[:, :, None]]).any()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_scores_of_the_lowest_value_and_large(dtype):
    """Scores near the largest the type can make, and all equal ones."""
    dev = torch.device("cuda", 0)
    c = ref.Cache([90, 90], 1, 64, 16, dtype, dev)
    q = make_q(2, 2, 64, dtype, dev, scale=60.0)
    q[1] = 0
    got, lse = run(c, q, [1, 1], with_lse=False)
    agree(c, q, [1, 1], got, None)


def test_strided_rows_and_slot_major_pages():
    """q as a view of a projection's output, out in a wider buffer, pages
    [page, slot, head, dim], a table cut from a wider one."""
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    rows, lens = [2, 130, 1], [50, 200, 777]
    for dtype in DTYPES:
        c = ref.Cache(lens, 2, 64, 16, dtype, dev, nhd=True, wide=4)
        T = sum(rows)
        big = make_q(T, 12, 64, dtype, dev)
        q = big[:, 2:10]
        store = torch.full((T, 9, 72), 3.0, dtype=dtype, device=dev)
        out = store[:, :8, :64]
        got, lse = run(c, q, rows, out=out)
        agree(c, q, rows, got, lse)
        assert (store[:, 8] == 3.0).all() and (store[:, :, 64:] == 3.0).all()


def test_other_stream_graph_and_shared_workspace():
    """A captured call replays on new contents; two graphs that share a
    workspace run one after the other."""
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    rows, lens = [1, 3], [2000, 900]
    cs = [ref.Cache(lens, 2, 128, 16, torch.bfloat16, dev, seed=s) for s in (1, 2)]
    qs = [make_q(4, 8, 128, torch.bfloat16, dev, seed=s) for s in (3, 4)]
    starts = ref.starts_of(rows, dev)
    ws = torch.empty(paged.attention_workspace_bytes(qs[0], cs[0].k, cs[0].table, 3), dtype=torch.uint8, device=dev)
    want = [paged.attention(q, c.k, c.v, c.table, c.kv_len, starts, 3) for q, c in zip(qs, cs)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], [torch.zeros_like(q) for q in qs]
    with torch.cuda.stream(side):
        for q, c, o in zip(qs, cs, outs):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                paged.attention(q, c.k, c.v, c.table, c.kv_len, starts, 3, out=o, workspace=ws)
            graphs.append(g)
        for _ in range(3):
            for g in graphs:
                g.replay()
    side.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    # New lengths in the same memory.
    cs[0].kv_len.copy_(torch.tensor([1500, 40], dtype=torch.int32))
    cs[0].lens = [1500, 40]
    with torch.cuda.stream(side):
        graphs[0].replay()
    side.synchronize()
    agree(cs[0], qs[0], rows, outs[0], None)


def test_bad_values_on_the_device_are_cut_and_reported():
    """Page numbers outside the pool read as masked; lengths and row ranges
    outside the tensors are cut."""
    import rai_b200
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    rows, lens = [1, 2], [100, 64]
    c = ref.Cache(lens, 2, 64, 16, torch.bfloat16, dev)
    q = make_q(3, 4, 64, torch.bfloat16, dev)
    starts = ref.starts_of(rows, dev)
    want = paged.attention(q, c.k, c.v, c.table, c.kv_len, starts, 2)
    paged.status()
    for cell in (-1, c.n_pages, 1 << 30):
        t = c.table.clone()
        t[0, 2] = cell
        got = paged.attention(q, c.k, c.v, t, c.kv_len, starts, 2)
        with pytest.raises(rai_b200.RaiError):
            paged.status()
        assert torch.equal(got[1:], want[1:]) and torch.isfinite(got.float()).all()
    for bad in ([0, 1, 1000], [-5, 1, 3], [2, 1, 3]):
        paged.attention(q, c.k, c.v, c.table, c.kv_len, torch.tensor(bad, dtype=torch.int32, device=dev), 2)
        with pytest.raises(rai_b200.RaiError):
            paged.status()
    paged.attention(q, c.k, c.v, c.table, torch.tensor([1 << 30, -4], dtype=torch.int32, device=dev), starts, 2)
    with pytest.raises(rai_b200.RaiError):
        paged.status()
    paged.status()  # the query clears it


def test_offsets_past_32_bits():
    """A page whose elements lie beyond 2^32 bytes of the pool."""
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    pages, nkv, page, hd = 18000, 8, 64, 256  # 4.7 GB a pool
    k = torch.zeros((pages, nkv, page, hd), dtype=torch.bfloat16, device=dev)
    v = torch.zeros((pages, nkv, page, hd), dtype=torch.bfloat16, device=dev)
    c = ref.Cache([130], nkv, hd, page, torch.bfloat16, dev, extra=0)
    far = [pages - 1, 16500, pages - 7]
    for j, p in enumerate(far):
        k[p], v[p] = c.k[c.rows[0][j]], c.v[c.rows[0][j]]
    q = make_q(1, 8, hd, torch.bfloat16, dev)
    table = torch.tensor([far], dtype=torch.int32, device=dev)
    got = paged.attention(q, k, v, table, c.kv_len, ref.starts_of([1], dev), 1)
    want = paged.attention(q, c.k, c.v, c.table, c.kv_len, ref.starts_of([1], dev), 1)
    assert torch.equal(got, want)


@pytest.mark.parametrize("heads,nkv", [(2, 2), (8, 1), (7, 1), (32, 2)])
@pytest.mark.parametrize("hd", [64, 80, 128])
def test_chunks_shorter_than_a_query_tile(heads, nkv, hd):
    """Row tensors with fewer rows than a tile of queries has, groups that do
    and do not divide it."""
    dev = torch.device("cuda", 0)
    for rows, lens in (([70], [70]), ([129, 66], [400, 66]), ([300], [1000])):
        c = ref.Cache(lens, nkv, hd, 16, torch.bfloat16, dev, seed=hd)
        q = make_q(sum(rows), heads, hd, torch.bfloat16, dev)
        got, lse = run(c, q, rows)
        agree(c, q, rows, got, lse)


def test_two_streams_at_once():
    """Calls of both kernels that may overlap, each with its own workspace."""
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    jobs = []
    for hd, rows, lens in ((64, [1] * 8, [700] * 8), (128, [200, 90], [2000, 90]), (128, [1, 3], [9000, 9000])):
        c = ref.Cache(lens, 2, hd, 16, torch.bfloat16, dev, seed=hd, wide=4000)
        q = make_q(sum(rows), 8, hd, torch.bfloat16, dev)
        jobs.append((q, c.k, c.v, c.table, c.kv_len, ref.starts_of(rows, dev), max(rows)))
    want = [paged.attention(*j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[] for _ in jobs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for s, j, g in zip(streams, jobs, got):
            with torch.cuda.stream(s):
                g.append(paged.attention(*j))
    torch.cuda.synchronize()
    paged.status()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=str)
@pytest.mark.parametrize("heads,nkv,hd", [(16, 16, 64), (16, 16, 128), (12, 4, 64), (16, 4, 64)])
@pytest.mark.parametrize("window", [40, 256])
def test_many_masked_tiles_in_a_row(dtype, heads, nkv, hd, window):
    """Long chunks behind a window of a few tiles: nearly every tile of V is
    looked through by two warps that have to stay together, in items of a few
    tiles each, whose queries come by TMA or by copies."""
    dev = torch.device("cuda", 0)
    rows, lens = [3000, 300, 2500, 2999, 1], [3000, 800, 2600, 4000, 900]
    c = ref.Cache(lens, nkv, hd, 16, dtype, dev, seed=window)
    q = make_q(sum(rows), heads, hd, dtype, dev)
    first, lse = run(c, q, rows, window=window)
    for _ in range(20):
        got, _ = run(c, q, rows, window=window)
        assert torch.equal(got, first)
    agree(c, q, rows, first, lse, window=window)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)], ids=str)
def test_an_infinite_value_at_the_end_of_a_million_tokens(dtype, hd):
    """Sequences that share one long context, a whole item or a third of one to
    a CTA: giving the value back to the rows that see it walks the masked tiles
    alone, so that no other warp's wait runs out meanwhile."""
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    n, seqs, page = 1_000_003, 150, 128
    g = torch.Generator(device=dev).manual_seed(hd)
    pages = -(-n // page)
    k, v = (torch.randn((pages, 1, page, hd), device=dev, generator=g).to(dtype) for _ in range(2))
    t = n - 2
    v[t // page, 0, t % page, 1] = math.inf
    v[t // page, 0, t % page, hd - 1] = math.nan
    table = torch.arange(pages, dtype=torch.int32, device=dev).expand(seqs, pages).contiguous()
    q = torch.randn((1, 2, hd), device=dev, generator=g).to(dtype).expand(seqs, 2, hd).contiguous()
    lens = torch.full((seqs,), n, dtype=torch.int32, device=dev)
    got = paged.attention(q, k, v, table, lens, torch.arange(seqs + 1, dtype=torch.int32, device=dev), 1)
    paged.status()
    kk, vv = (x.view(-1, hd)[:n].double() for x in (k, v))
    p = torch.softmax(hd ** -0.5 * (q[0].double() @ kk.T), 1)
    seen = torch.isfinite(vv)
    want = p @ torch.where(seen, vv, 0.0)
    size = p @ torch.where(seen, vv, 0.0).abs()
    assert (got[:, :, 1] == math.inf).all() and torch.isnan(got[:, :, hd - 1]).all()
    cols = [c for c in range(hd) if c not in (1, hd - 1)]
    # Roundings of the output and the probabilities, sums of n terms in f32
    # (random: their square root), scores off by hd + 4 roundings.
    u = ref.EPS[dtype]
    bound = u * want.abs() + size * (1.01 * u + 2 * (hd + 4) * 2.0 ** -24 * 10 + n ** 0.5 * 2.0 ** -22) + 2.0 ** -24 * (dtype == torch.float16)
    assert ((got[:, :, cols].double() - want[:, cols]).abs() <= bound[:, cols]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("hd,rows", [(64, [1, 3]), (128, [1, 3]), (128, [70, 3])], ids=str)
@pytest.mark.parametrize("cap", [2.0, 100.0, 1e4, 1e6, 1e12, 3e38])
def test_caps_far_above_the_scores(dtype, hd, rows, cap):
    """A cap may be off by a part of the score, not of the cap."""
    dev = torch.device("cuda", 0)
    lens = [200, 90]
    c = ref.Cache(lens, 2, hd, 16, dtype, dev, seed=hd)
    q = make_q(sum(rows), 4, hd, dtype, dev, scale=2.0)
    got, lse = run(c, q, rows, softcap=cap)
    want, _, wlse = ref.attention(q, c, rows, hd ** -0.5, cap)
    # What the roundings around the cap may make of the same scores uncapped;
    # the cap moves each score by 2^-17 of itself at most.
    _, bound, _ = ref.attention(q, c, rows, hd ** -0.5)
    top = max(q.double().norm(dim=-1).max() * k.norm(dim=-1).max() for k, _ in (c.tokens(s) for s in range(2))) * hd ** -0.5
    size = max(v.abs().max() for _, v in (c.tokens(s) for s in range(2)))
    # (bound holds the probabilities' and the output's roundings relative to
    # the uncapped ones: 2 u of the largest value covers the capped ones.)
    assert ((got.double() - want).abs() <= torch.clamp(bound, min=2.1 * ref.EPS[dtype] * size) + 2.0 ** -16 * top * size).all()
    assert ((lse.double() - wlse).abs() <= 2.0 ** -18 * (1 + wlse.abs()) + 2.0 ** -17 * top).all()


class Without:
    """A cache of one sequence without its token t."""

    def __init__(self, cache, t):
        self.lens, self.c, self.t = [cache.lens[0] - 1], cache, t

    def tokens(self, s):
        k, v = self.c.tokens(0)
        keep = torch.arange(k.shape[1], device=k.device) != self.t
        return k[:, keep], v[:, keep]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 8, 40, 90])
def test_infinite_keys_and_values_that_rows_see(dtype, hd, rows):
    """A key of -inf has weight 0 and an infinite value is its rows' output,
    also where the factor beside it is a power of two (a probability of 1, a
    query of small integers), in tiles that no mask touches."""
    dev = torch.device("cuda", 0)
    n = 700
    c = ref.Cache([n], 2, hd, 16, dtype, dev, seed=hd + rows)
    q = torch.randint(1, 4, (rows, 4, hd), generator=torch.Generator().manual_seed(rows)).to(dtype).to(dev)

    def token(t):
        return c.rows[0][t // 16], t % 16
    p, s = token(37)
    c.k[p, :, s] = -math.inf
    p, s = token(90)
    c.k[p, :, s] = 40.0  # its probability is 1
    c.v[p, :, s, 3] = math.inf
    c.v[p, 0, s, 5] = -math.inf
    c.v[p, 1, s, 7] = math.nan
    got, lse = run(c, q, [rows])
    agree(Without(c, 37), q, [rows], got, lse)
    assert (got[:, :, 3] == math.inf).all() and (got[:, :2, 5] == -math.inf).all() and torch.isnan(got[:, 2:, 7]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("hd,rows,lens", [(64, [1, 5, 1], [3000, 900, 40]), (128, [2, 300, 1], [9000, 700, 64]), (128, [1, 9, 4], [9000, 9000, 700])])
def test_output_in_place_of_the_queries(dtype, hd, rows, lens):
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    c = ref.Cache(lens, 2, hd, 16, dtype, dev, seed=hd, wide=3000)
    big = make_q(sum(rows), 12, hd, dtype, dev)
    q = big[:, 2:10]
    want = paged.attention(q, c.k, c.v, c.table, c.kv_len, ref.starts_of(rows, dev), max(rows))
    rest = big[:, 10:].clone()
    got = paged.attention(q, c.k, c.v, c.table, c.kv_len, ref.starts_of(rows, dev), max(rows), out=q)
    paged.status()
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want) and torch.equal(big[:, 10:], rest)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("hd,rows", [(64, [1, 5]), (128, [2, 200])])
def test_pages_that_heads_share(dtype, hd, rows):
    """One KV head's pages expanded to four (a stride of 0) are read as if
    copied; the same as an output is refused."""
    import rai_b200
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    c = ref.Cache([700, 300], 1, hd, 16, dtype, dev, seed=hd)
    q = make_q(sum(rows), 8, hd, dtype, dev)
    starts = ref.starts_of(rows, dev)
    k, v = (t.expand(-1, 4, -1, -1) for t in (c.k, c.v))
    got = paged.attention(q, k, v, c.table, c.kv_len, starts, max(rows))
    full = ref.Cache([700, 300], 4, hd, 16, dtype, dev)
    full.k, full.v, full.rows = k, v, c.rows
    want, bound, _ = ref.attention(q, full, rows, hd ** -0.5)
    assert ((got.double() - want).abs() <= bound).all()
    with pytest.raises(rai_b200.RaiError):
        paged.attention(q, k, v, c.table, c.kv_len, starts, max(rows), out=torch.zeros_like(q[:, :1]).expand(-1, 8, -1))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("page", [8, 16, 24, 128])
@pytest.mark.parametrize("hd,rows", [(64, [1, 2]), (128, [1, 2]), (128, [80, 2])])
def test_pages_outside_the_pool_read_as_zeros(dtype, page, hd, rows):
    """Also after calls whose tiles left NaN behind them in shared memory."""
    import rai_b200
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    c = ref.Cache([400, 300], 2, hd, page, dtype, dev, seed=hd, wide=40000 // page)
    q = make_q(sum(rows), 8, hd, dtype, dev)
    starts = ref.starts_of(rows, dev)
    table, k, v = c.table.clone(), c.k.clone(), c.v.clone()
    for s, cell in ((0, 1), (0, 2), (1, 0)):
        k[c.rows[s][cell]] = 0
        v[c.rows[s][cell]] = 0
        table[s, cell] = -1 if cell else c.n_pages
    want = paged.attention(q, k, v, c.table, c.kv_len, starts, max(rows))
    paged.status()
    junk = [torch.full_like(t, math.nan) for t in (c.k, c.v)]
    for _ in range(4):
        paged.attention(q, *junk, c.table, c.kv_len, starts, max(rows))
        got = paged.attention(q, c.k, c.v, table, c.kv_len, starts, max(rows))
        with pytest.raises(rai_b200.RaiError):
            paged.status()
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.float32, 128), (torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float16, 64)], ids=str)
def test_weights_do_not_drift_along_a_context(dtype, hd):
    """Equal scores of several hundred: each token's weight is the same however
    many tiles lie behind it. Values of 1 in the first half and -1 in the second
    cancel."""
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    n, seqs, page, H = 100_000, 150, 100 if hd == 64 else 128, 4
    n = n // (2 * page) * 2 * page
    pages = n // page
    k = torch.full((pages, 1, page, hd), 2.0 ** -4, dtype=dtype, device=dev)
    v = torch.ones((pages, 1, page, hd), dtype=dtype, device=dev)
    v[pages // 2:, :, :, ::2] = -1
    q = torch.empty((seqs, H, hd), dtype=dtype, device=dev)
    for h in range(H):
        q[:, h] = 180.0 + 7 * h  # (exact in every type)
    table = torch.arange(pages, dtype=torch.int32, device=dev).expand(seqs, pages).contiguous()
    lens = torch.full((seqs,), n, dtype=torch.int32, device=dev)
    lse = torch.zeros((seqs, H), device=dev)
    scale = 0.7137
    got = paged.attention(q, k, v, table, lens, torch.arange(seqs + 1, dtype=torch.int32, device=dev), 1, scale=scale, lse=lse)
    paged.status()
    score = scale * hd * q[0, :, 0].double() * 2.0 ** -4  # 514 to 574
    # Sums of n / 3 equal terms in f32, by threads that add some hundred tiles
    # of up to 32 terms: 2^-24 of the sum for each addition, 2^13 of them. The
    # score is rounded twice, times log2(e) once more.
    tol = 2.0 ** -11
    assert ((lse.double() - (score + math.log(n))).abs() <= tol + score * 2.0 ** -21).all()
    assert (got[:, :, ::2].double().abs() <= tol).all()
    assert ((got[:, :, 1::2].double() - 1).abs() <= tol + ref.EPS[dtype]).all()
