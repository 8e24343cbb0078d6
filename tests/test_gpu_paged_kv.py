"""rai_b200.paged: rotary positions with the store, and the page operations,
against plain forms (64 bits; lists); a beam decoding loop over all of them."""
import math
import random

import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("src", DTYPES, ids=str)
@pytest.mark.parametrize("dst", DTYPES, ids=str)
@pytest.mark.parametrize("hd,rot", [(64, 64), (128, 64), (80, 20), (96, 96), (256, 256), (32, 6)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_append(src, dst, hd, rot, interleaved):
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    rows, lens = [1, 4, 0, 37, 5], [1, 100, 9, 37, 5000]
    H, G, T = 6, 2, sum(rows) + 2
    c = ref.Cache(lens, G, hd, 16, dst, dev, junk=9.0)
    g = torch.Generator().manual_seed(hd)
    qkv = torch.randn((T, (H + 2 * G) * hd), generator=g).to(src).to(dev)
    q, k, v = (x.view(T, -1, hd) for x in qkv.split([H * hd, G * hd, G * hd], 1))
    freq, m = paged.rope_frequencies(rot, 500000.0, "yarn", factor=4.0, low=1.0, high=32.0, original=2048.0)
    inv = torch.from_numpy(freq).to(dev)
    before_k, before_v = c.k.clone(), c.v.clone()
    out = torch.full((T, H, hd), 3.0, dtype=dst, device=dev)
    got = paged.rope_append(q, k, v, c.k, c.v, c.table, c.kv_len, ref.starts_of(rows, dev), inv, interleaved=interleaved,
                            mscale=m, q_out=out)
    paged.status()
    pos = torch.cat([torch.arange(t - n, t) for n, t in zip(rows, lens)]).to(dev)
    n = sum(rows)
    u = ref.EPS[dst]

    def close(a, x):
        # One rounding to the type, the angle's sine and cosine and two
        # products and a sum in f32 (each 2^-24 of either term, the functions
        # 2 ulp), halves below the normal range.
        w = ref.rope(x.double(), pos, inv, interleaved, m)
        size = x.double().abs().amax(-1, keepdim=True) * 2 * m
        assert ((a.double() - w).abs() <= u * w.abs() + 2.0 ** -21 * size + 2.0 ** -25 * (dst == torch.float16)).all()
    close(got[:n], q[:n])
    assert (got[n:] == 3.0).all()
    page = torch.cat([torch.tensor([c.rows[s][t // 16] for t in range(lens[s] - r, lens[s])], dtype=torch.long)
                      for s, r in enumerate(rows)]).to(dev)
    close(c.k[page, :, pos % 16], k[:n])
    assert torch.equal(c.v[page, :, pos % 16], v[:n].to(dst))
    before_k[page, :, pos % 16] = c.k[page, :, pos % 16]
    before_v[page, :, pos % 16] = c.v[page, :, pos % 16]
    assert torch.equal(before_k, c.k) and torch.equal(before_v, c.v)  # nothing else was written


def test_rope_in_place_and_far_positions():
    """q_out = q; a million tokens in, where 32-bit angles are off by 0.06."""
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    hd, n = 64, 1_000_003
    c = ref.Cache([10], 1, hd, 16, torch.float32, dev, junk=0.0)
    table = torch.zeros((1, 70000), dtype=torch.int32, device=dev)
    inv = torch.from_numpy(paged.rope_frequencies(hd, 10000.0)[0]).to(dev)
    q = torch.randn((2, 3, hd), device=dev)
    k = torch.randn((2, 1, hd), device=dev)
    want = ref.rope(q.double(), torch.tensor([n - 2, n - 1], device=dev), inv, False)
    got = paged.rope_append(q, k, k, c.k, c.v, table, torch.tensor([n], dtype=torch.int32, device=dev),
                            ref.starts_of([2], dev), inv, q_out=q)
    assert got.data_ptr() == q.data_ptr()
    assert (got.double() - want).abs().max() <= 2.0 ** -20 * 8


def test_rope_rows_before_the_sequence_and_bad_pages():
    import rai_b200
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    c = ref.Cache([2, 20], 1, 64, 16, torch.bfloat16, dev, junk=4.0)
    inv = torch.from_numpy(paged.rope_frequencies(64)[0]).to(dev)
    q = torch.randn((7, 2, 64), device=dev).bfloat16()
    k = torch.randn((7, 1, 64), device=dev).bfloat16()
    paged.rope_append(q, k, k, c.k, c.v, c.table, c.kv_len, ref.starts_of([5, 2], dev), inv)
    paged.status()
    assert torch.equal(c.v[c.rows[0][0], 0, :2], k[3:5, 0])
    before = c.v.clone()
    t = c.table.clone()
    t[1, 1] = c.n_pages + 5
    paged.rope_append(q, k, k * 2, c.k, c.v, t, c.kv_len, ref.starts_of([0, 2], dev), inv)
    with pytest.raises(rai_b200.RaiError):
        paged.status()
    assert torch.equal(before, c.v)


def lists(t):
    return t.tolist()


def check_pages(want, table, lens, refs):
    assert lists(lens) == want.lens
    got = lists(table)
    for s, n in enumerate(want.lens):
        c = want.cells(n)
        assert got[s][:c] == want.table[s][:c], s
    assert lists(refs) == want.refs


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("page", [1, 16, 24])
def test_fork_resize_compact_in_turn(seed, page):
    """Random forks, growths, truncations, frees and compactions of a pool of
    two layers, against lists; the tokens every sequence holds are followed
    through all of it."""
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    r = random.Random(seed * 100 + page)
    n, layers, nkv, hd = r.choice([3, 9, 40]), 2, 2, 16
    lens = [r.randrange(0, 70) for _ in range(n)]
    c = ref.Cache(lens, nkv, hd, page, torch.bfloat16, dev, seed=seed, junk=0.0, extra=40 + 500 // page, wide=200 // page + 2)
    k = torch.stack([c.k, c.k + 1]).contiguous()
    v = torch.stack([c.v, c.v + 2]).contiguous()
    table, refs = c.table.clone(), c.refs.clone()
    kv = c.kv_len.clone()
    want = ref.Pages(c.rows, lens, lists(refs), page)
    width = table.shape[1]

    def content(s):
        m = want.lens[s]
        return [torch.cat([x[:, p] for p in want.table[s][: want.cells(m)]], 2)[:, :, :m].clone() if m else None for x in (k, v)]
    held = [content(s) for s in range(n)]
    for step in range(14):
        what = r.choice(["fork", "grow", "any", "compact", "shrink"])
        if what == "fork":
            parents = [r.randrange(-1, n) if r.random() < 0.2 else r.randrange(n) for _ in range(n)]
            want.fork(parents, width)
            table, kv = paged.fork(table, kv, refs, torch.tensor(parents, dtype=torch.int32, device=dev), page)
            held = [held[p] if p >= 0 else [None, None] for p in parents]
        elif what == "compact":
            moves, used = want.compact()
            got = paged.compact(table, kv, refs, k, v)
            assert got.item() == used
        else:
            cap = min(width * page, 190)
            if what == "grow":
                d = r.choice([1, 1, 5])
                d = min(d, cap - max(want.lens))
                new = [m + d for m in want.lens]
                _, short = want.resize(new)
                got = paged.resize(table, kv, refs, k, v, delta=d)
            else:
                new = [r.randrange(0, cap) if what == "any" else r.randrange(0, m + 1) for m in want.lens]
                _, short = want.resize(new)
                got = paged.resize(table, kv, refs, k, v, new_lens=torch.tensor(new, dtype=torch.int32, device=dev))
            assert got.item() == short
        paged.status()
        check_pages(want, table, kv, refs)
        # What a sequence held it still holds.
        for s in range(n):
            now = content(s)
            for i in range(2):
                if held[s][i] is not None and now[i] is not None:
                    m = min(held[s][i].shape[2], now[i].shape[2])
                    assert torch.equal(held[s][i][:, :, :m], now[i][:, :, :m]), (step, what, s)
            held[s] = now


def test_resize_reports_missing_pages():
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    c = ref.Cache([30, 16], 1, 16, 16, torch.bfloat16, dev, extra=2, wide=8, junk=0.0)
    k, v = c.k.contiguous(), c.v.contiguous()
    want = ref.Pages(c.rows, c.lens, lists(c.refs), 16)
    new = torch.tensor([80, 5], dtype=torch.int32, device=dev)
    _, short = want.resize([80, 5])
    got = paged.resize(c.table, c.kv_len, c.refs, k, v, new_lens=new)
    assert got.item() == short == 1
    check_pages(want, c.table, c.kv_len, c.refs)


def test_many_sequences_and_a_large_pool():
    """The most sequences a call takes, pages beyond one scan of the block."""
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    n = 4096
    r = random.Random(5)
    lens = [r.randrange(1, 60) for _ in range(n)]
    c = ref.Cache(lens, 1, 8, 16, torch.bfloat16, dev, extra=70000, wide=2, junk=0.0)
    want = ref.Pages(c.rows, lens, lists(c.refs), 16)
    parents = [r.randrange(n) for _ in range(n)]
    want.fork(parents, c.table.shape[1])
    table, kv = paged.fork(c.table, c.kv_len, c.refs, torch.tensor(parents, dtype=torch.int32, device=dev), 16)
    check_pages(want, table, kv, c.refs)
    copies, short = want.resize([m + 1 for m in want.lens])
    k0 = c.k.clone()
    got = paged.resize(table, kv, c.refs, c.k, c.v, delta=1)
    assert got.item() == short == 0
    check_pages(want, table, kv, c.refs)
    src, dst = (torch.tensor(x, device=dev) for x in zip(*copies))
    assert torch.equal(c.k[dst], k0[src])
    moves, used = want.compact()
    k1 = c.k.clone()
    assert paged.compact(table, kv, c.refs, c.k, c.v).item() == used
    check_pages(want, table, kv, c.refs)
    src, dst = (torch.tensor(x, device=dev) for x in zip(*moves))
    assert torch.equal(c.k[dst], k1[src])


@pytest.mark.parametrize("hd,page,dtype", [(64, 16, torch.bfloat16), (8, 1, torch.float16), (256, 128, torch.float32)])
def test_copy_pages(hd, page, dtype):
    import rai_b200
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    k = torch.randn((3, 50, 2, page, hd), device=dev).to(dtype)
    v = torch.randn((3, 50, 2, page, hd), device=dev).to(dtype)
    k0, v0 = k.clone(), v.clone()
    src, dst = [3, 3, 40], [7, 8, 49]
    paged.copy_pages(k, v, torch.tensor(src, dtype=torch.int32, device=dev), torch.tensor(dst, dtype=torch.int32, device=dev))
    paged.status()
    k0[:, dst], v0[:, dst] = k0[:, src], v0[:, src]
    assert torch.equal(k, k0) and torch.equal(v, v0)
    paged.copy_pages(k, v, torch.tensor([50, -1], dtype=torch.int32, device=dev), torch.tensor([1, 2], dtype=torch.int32, device=dev))
    with pytest.raises(rai_b200.RaiError):
        paged.status()
    assert torch.equal(k, k0) and torch.equal(v, v0)
    # One layer's four dimensions.
    paged.copy_pages(k[1], v[1], torch.tensor([0], dtype=torch.int32, device=dev), torch.tensor([1], dtype=torch.int32, device=dev))
    assert torch.equal(k[1, 1], k0[1, 0]) and torch.equal(k[0], k0[0]) and torch.equal(k[2], k0[2])


def test_fork_ignores_parents_out_of_range():
    import rai_b200
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    c = ref.Cache([20, 33], 1, 16, 16, torch.bfloat16, dev, junk=0.0)
    t, n = paged.fork(c.table, c.kv_len, c.refs, torch.tensor([5, 1, -3], dtype=torch.int32, device=dev), 16)
    with pytest.raises(rai_b200.RaiError):
        paged.status()
    assert lists(n) == [0, 33, 0] and lists(t[1])[:3] == c.rows[1][:3]
    assert c.refs.sum().item() == 3


def test_beam_decoding_over_a_paged_cache():
    """The operators as they are used together: a tiny attention model decodes
    with beam search over forked pages, step for step as a plain search that
    keeps each beam's whole history and recomputes everything in 64 bits."""
    from rai_b200 import beams, paged
    dev = torch.device("cuda", 0)
    V, H, G, D, B, N, page, layers = 53, 4, 2, 32, 2, 3, 4, 2
    g = torch.Generator().manual_seed(3)
    emb = torch.randn((V, H * D), generator=g).to(dev)
    wq = [(torch.randn((H * D, H * D), generator=g) / 8).to(dev) for _ in range(layers)]
    wk = [(torch.randn((H * D, G * D), generator=g) / 8).to(dev) for _ in range(layers)]
    wv = [(torch.randn((H * D, G * D), generator=g) / 8).to(dev) for _ in range(layers)]
    head = (torch.randn((H * D, V), generator=g) / 6).to(dev)
    inv = torch.from_numpy(paged.rope_frequencies(D)[0]).to(dev)
    prompts = [[1, 5, 9, 2, 30, 7], [4, 4, 8]]

    def plain_logits(tokens):
        """Logits after the last token, everything recomputed."""
        x = emb[tokens].double()
        T = len(tokens)
        pos = torch.arange(T, device=dev)
        for l in range(layers):
            q = ref.rope((x @ wq[l].double()).view(T, H, D), pos, inv, False)
            k = ref.rope((x @ wk[l].double()).view(T, G, D), pos, inv, False)
            v = (x @ wv[l].double()).view(T, G, D)
            o = torch.zeros_like(q)
            for h in range(H):
                s = (q[:, h] @ k[:, h // 2].T) * D ** -0.5
                s[torch.triu(torch.ones(T, T, dtype=torch.bool, device=dev), 1)] = -math.inf
                o[:, h] = torch.softmax(s, 1) @ v[:, h // 2]
            x = x + o.reshape(T, -1)
        return x[-1] @ head.double()

    S, width, pages = B * N, 16, 100
    k = torch.zeros((layers, pages, G, page, D), device=dev)
    v = torch.zeros_like(k)
    table = torch.full((S, width), -1, dtype=torch.int32, device=dev)
    lens = torch.zeros(S, dtype=torch.int32, device=dev)
    refs = torch.zeros(pages, dtype=torch.int32, device=dev)

    def forward(tokens, rows):
        """tokens of every sequence's new rows, one after the other -> logits of the rows."""
        x = emb[tokens]
        starts = ref.starts_of(rows, dev)
        for l in range(layers):
            qkv = torch.cat([x @ wq[l], x @ wk[l], x @ wv[l]], 1)
            q, kk, vv = (y.view(len(tokens), -1, D) for y in qkv.split([H * D, G * D, G * D], 1))
            q = paged.rope_append(q, kk, vv, k[l], v[l], table, lens, starts, inv)
            o = paged.attention(q, k[l], v[l], table, lens, starts, max(rows))
            x = x + o.reshape(len(tokens), -1)
        return x @ head
    # Prefill the first beam of each request, then fork it to all of them.
    rows = [len(prompts[s // N]) if s % N == 0 else 0 for s in range(S)]
    assert paged.resize(table, lens, refs, k, v, new_lens=torch.tensor(rows, dtype=torch.int32, device=dev)).item() == 0
    logits = forward([t for p in prompts for t in p], rows)
    last = torch.tensor(rows).cumsum(0)[::N] - 1
    logits = logits[last.to(dev)].repeat_interleave(N, 0)
    scores = torch.tensor([[0.0] + [-math.inf] * (N - 1)] * B, device=dev)
    table, lens = paged.fork(table, lens, refs, torch.tensor([s // N * N for s in range(S)], dtype=torch.int32, device=dev), page)
    assert refs.max().item() == N  # the prompts' pages are shared
    hist = torch.zeros((S, 32), dtype=torch.int32, device=dev)
    hist_len = torch.zeros(S, dtype=torch.int32, device=dev)
    plain = [[(0.0, p)] for p in prompts]
    for step in range(7):
        r = beams.select(logits.view(B, N, V), scores, eos=0, history=hist, hist_len=hist_len)
        hist, hist_len, scores = r.history, r.hist_len, r.scores
        table, lens = paged.fork(table, lens, refs, r.parents.view(-1), page)
        assert paged.resize(table, lens, refs, k, v, delta=1).item() == 0
        logits = forward(r.tokens.view(-1).tolist(), [1] * S)
        paged.status()
        for b in range(B):
            best = []
            for score, toks in plain[b]:
                lp = torch.log_softmax(plain_logits(toks), 0)
                best += [(score + lp[t].item(), toks + [t]) for t in range(1, V)]
            plain[b] = sorted(best, reverse=True)[:N]
            for i, (score, toks) in enumerate(plain[b]):
                s = b * N + i
                assert hist[s, : step + 1].tolist() == toks[len(prompts[b]):]
                assert abs(score - scores[b, i].item()) < 1e-3
    # Ending every sequence leaves no page in use.
    paged.resize(table, lens, refs, k, v, new_lens=torch.zeros(S, dtype=torch.int32, device=dev))
    assert refs.abs().sum().item() == 0
    assert paged.compact(table, lens, refs, k, v).item() == 0


def test_a_beam_step_in_a_graph():
    """Fork, resize and rope captured once and replayed on new contents of the
    same memory; the eager calls on copies give the same."""
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    n, hd, page = 6, 64, 16
    lens = [33, 33, 20, 48, 5, 64]
    c = ref.Cache(lens, 2, hd, page, torch.bfloat16, dev, extra=40, wide=3, junk=0.0)
    k, v = c.k.contiguous(), c.v.contiguous()
    first = [x.clone() for x in (c.table, c.kv_len, c.refs, k, v)]
    parents = torch.tensor([0, 0, 2, 3, 3, 3], dtype=torch.int32, device=dev)
    inv = torch.from_numpy(paged.rope_frequencies(hd)[0]).to(dev)
    q = torch.randn((n, 4, hd), device=dev).bfloat16()
    kk = torch.randn((n, 2, hd), device=dev).bfloat16()
    starts = ref.starts_of([1] * n, dev)

    def step(table, lens, refs, k, v):
        t, m = paged.fork(table, lens, refs, parents, page)
        short = paged.resize(t, m, refs, k, v, delta=1)
        r = paged.rope_append(q, kk, kk, k, v, t, m, starts, inv)
        o = paged.attention(r, k, v, t, m, starts, 1)
        return t, m, refs, k, v, short, r, o
    step(*[x.clone() for x in first])  # looks up the status word
    state = [x.clone() for x in first]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*state)
    for trial in range(2):
        for a, b in zip(state, first):
            a.copy_(b)
        q.normal_()
        parents.copy_(torch.tensor([trial, 0, 2, 3, 5, 5 - trial], dtype=torch.int32))
        graph.replay()
        want = step(*[x.clone() for x in first])
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(got, want)):
            if i == 0:  # cells behind the lengths are not compared
                for s, m in enumerate(want[1].tolist()):
                    assert torch.equal(a[s, : -(-m // page)], b[s, : -(-m // page)])
            else:
                assert torch.equal(a, b), i


def test_resize_gives_nothing_when_pages_are_short():
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    n = 4096
    k = torch.zeros((3, 1, 1, 8), dtype=torch.bfloat16, device=dev)
    lens = torch.zeros(n, dtype=torch.int32, device=dev)
    refs = torch.zeros(3, dtype=torch.int32, device=dev)
    table = torch.full((n, 600), -1, dtype=torch.int32, device=dev)
    assert paged.resize(table, lens, refs, k, k.clone(), delta=600).item() == n * 600 - 3
    assert lens.sum().item() == 0 and refs.sum().item() == 0 and (table == -1).all()


@pytest.mark.parametrize("children", [1, 2, 5])
def test_fork_into_given_outputs(children):
    """out_table (a part of a wider one) and out_lens, more or fewer children
    than parents."""
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    lens = [20, 33, 7]
    c = ref.Cache(lens, 1, 16, 16, torch.bfloat16, dev, junk=0.0)
    want = ref.Pages(c.rows, lens, lists(c.refs), 16)
    parents = [1, 0, 1, -1, 2][:children]
    width = c.table.shape[1]
    want.fork(parents, width)
    wide = torch.full((children, width + 3), 77, dtype=torch.int32, device=dev)
    out, n = wide[:, :width], torch.full((children,), 77, dtype=torch.int32, device=dev)
    got = paged.fork(c.table, c.kv_len, c.refs, torch.tensor(parents, dtype=torch.int32, device=dev), 16, out_table=out, out_lens=n)
    paged.status()
    assert got[0].data_ptr() == out.data_ptr() and got[1].data_ptr() == n.data_ptr()
    check_pages(want, out, n, c.refs)
    assert (wide[:, width:] == 77).all()


def test_a_graph_notices_pages_that_were_written():
    """Pages saved for a backward pass and written since: an error, as for any
    operation in place; inference tensors stay allowed."""
    from rai_b200 import paged
    dev = torch.device("cuda", 0)
    c = ref.Cache([20, 9], 1, 64, 16, torch.float32, dev, junk=0.0)
    inv = torch.from_numpy(paged.rope_frequencies(64)[0]).to(dev)
    q, k = torch.randn((2, 2, 64), device=dev), torch.randn((2, 1, 64), device=dev)
    starts = ref.starts_of([1, 1], dev)
    one = torch.zeros(1, dtype=torch.int32, device=dev)
    out = torch.zeros_like(q)
    calls = [(lambda: paged.rope_append(q, k, k, c.k, c.v, c.table, c.kv_len, starts, inv), (c.k, c.v)),
             (lambda: paged.rope_append(q, k, k, c.k, c.v, c.table, c.kv_len, starts, inv, q_out=out), (out, c.k)),
             (lambda: paged.attention(q, c.k, c.v, c.table, c.kv_len, starts, 1, out=out), (out,)),
             (lambda: paged.copy_pages(c.k, c.v, one, one + 1), (c.k, c.v)),
             (lambda: paged.resize(c.table, c.kv_len, c.refs, c.k, c.v, delta=0), (c.k, c.v, c.table, c.kv_len, c.refs)),
             (lambda: paged.compact(c.table, c.kv_len, c.refs, c.k, c.v), (c.k, c.v, c.table, c.refs))]
    for call, tensors in calls:
        before = [t._version for t in tensors]
        call()
        assert all(t._version > b for t, b in zip(tensors, before))
    w = torch.ones(64, device=dev, requires_grad=True)
    loss = (w * c.k).sum()
    paged.copy_pages(c.k, c.v, one, one + 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        ks, vs = c.k.clone(), c.v.clone()
    paged.copy_pages(ks, vs, one, one + 1)
    assert torch.equal(ks[1], ks[0])
