"""rai_b200.beams.select against a plain selection in 64 bits."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def plain(logits, scores, keep, eos):
    """The definition, one request at a time on the host."""
    out = []
    B, N, V = logits.shape
    for b in range(B):
        x = logits[b].double()
        x = torch.where(torch.isnan(x), -math.inf, x)
        m = x.amax(1, keepdim=True)
        d = torch.where(x == m, 0.0, x - m)
        s = scores[b].double()
        s = torch.where(torch.isnan(s), -math.inf, s)
        key = s[:, None] + (d - torch.log(torch.where(x == m, 1.0, torch.exp(x - m)).sum(1, keepdim=True)))
        raw, key = x.flatten(), key.flatten()
        o = torch.sort(raw, dim=0, descending=True, stable=True)[1]
        o = o[torch.sort(key[o], dim=0, descending=True, stable=True)[1]][:keep]
        cand = [(key[i].item(), i.item() // V, i.item() % V) for i in o]
        cand += [(-math.inf, -1, -1)] * (keep - len(cand))
        go = [c for c in cand if c[1] >= 0 and c[2] != eos][:N]
        go += [(-math.inf, -1, -1)] * (N - len(go))
        out.append((cand, go))
    return out


def check(logits, scores, keep=None, eos=-1):
    from rai_b200 import beams
    r = beams.select(logits, scores, keep=keep, eos=eos)
    B, N, V = logits.shape
    keep = 2 * N if keep is None else keep
    for b, (cand, go) in enumerate(plain(logits.cpu(), scores.cpu(), keep, eos)):
        assert r.cand_beams[b].tolist() == [c[1] for c in cand], b
        assert r.cand_tokens[b].tolist() == [c[2] for c in cand], b
        assert r.tokens[b].tolist() == [c[2] for c in go]
        assert r.parents[b].tolist() == [c[1] + b * N if c[1] >= 0 else -1 for c in go]
        for got, want in ((r.cand_scores[b], cand), (r.scores[b], go)):
            w = torch.tensor([c[0] for c in want], dtype=torch.float64)
            g = got.double().cpu()
            assert torch.equal(torch.isfinite(g), torch.isfinite(w))
            f = torch.isfinite(w)
            # One rounding to f32; the sums' 2-ulp exponentials.
            assert ((g - w).abs()[f] <= 2.0 ** -24 * w.abs()[f] + 2.0 ** -22).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,N,V", [(1, 1, 1), (1, 1, 2), (2, 3, 7), (1, 4, 100), (3, 5, 1237), (2, 8, 32001), (1, 32, 2049),
                                   (1, 2, 151936), (40, 2, 513)])
def test_sizes(dtype, B, N, V):
    g = torch.Generator().manual_seed(V + N)
    x = (3 * torch.randn((B, N, V), generator=g)).to(dtype).cuda()
    s = -5 * torch.rand((B, N), generator=g)
    check(x, s.cuda(), eos=V // 2)
    check(x, s.cuda(), keep=N)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_ties_take_the_lowest(dtype):
    """Few values, so that most logits are equal: within a beam the lowest
    token, between equal beams the lowest beam."""
    g = torch.Generator().manual_seed(1)
    x = torch.randint(-2, 3, (2, 4, 5000), generator=g).to(dtype).cuda()
    x[1, 1:] = x[1, :1]
    check(x, torch.zeros((2, 4)).cuda(), eos=3)
    check(torch.zeros((1, 3, 9000), dtype=dtype).cuda(), torch.zeros((1, 3)).cuda())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_order_of_the_vocabulary(dtype):
    """Rising logits: every step of the pass has better ones than the last."""
    x = (torch.arange(20000) / 3000.0).to(dtype).repeat(1, 2, 1).cuda()
    check(x, torch.tensor([[0.0, -0.3]]).cuda())
    check(x.flip(-1).contiguous(), torch.tensor([[0.0, -0.3]]).cuda())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_infinities_and_nan(dtype):
    g = torch.Generator().manual_seed(2)
    x = torch.randn((6, 3, 3000), generator=g).to(dtype)
    x[0, :, 10:] = -math.inf       # fewer finite ones than are kept
    x[1, 0] = -math.inf            # a row with nothing: uniform
    x[2, 1, [5, 900, 2999]] = math.inf
    x[3, :, ::2] = math.nan
    x[4, :, 7] = torch.finfo(dtype).min
    x[5] = math.nan
    s = -torch.rand((6, 3), generator=g)
    s[4, 0] = -math.inf
    s[3, 2] = math.nan
    check(x.cuda(), s.cuda(), eos=2)


def test_rows_of_any_alignment_and_spacing():
    g = torch.Generator().manual_seed(3)
    for dtype in DTYPES:
        big = torch.randn((2 * 3, 1011), generator=g).to(dtype).cuda()
        x = big[:, 3:1004].view(2, 3, 1001) if False else big[:, 3:1004].unflatten(0, (2, 3))
        check(x, torch.zeros((2, 3)).cuda())
        check(big.unflatten(0, (2, 3))[:, :, 1:], torch.zeros((2, 3)).cuda())


def test_all_candidates_end():
    """Fewer continuations than beams when eos takes the best."""
    x = torch.full((1, 2, 3), -math.inf)
    x[0, 0, 1] = 0.0
    x[0, 1, 1] = 0.0
    check(x.cuda(), torch.zeros((1, 2)).cuda(), eos=1)
    check(x.cuda(), torch.zeros((1, 2)).cuda(), keep=2, eos=1)


def test_histories():
    import rai_b200
    from rai_b200 import beams, paged
    g = torch.Generator().manual_seed(4)
    x = torch.randn((3, 4, 50), generator=g).cuda()
    h = torch.randint(0, 50, (12, 9), generator=g).int().cuda()
    n = torch.tensor([0, 3, 8, 1, 2, 2, 2, 2, 5, 5, 5, 5], dtype=torch.int32).cuda()
    r = beams.select(x, torch.zeros((3, 4)).cuda(), history=h, hist_len=n)
    paged.status()
    for i, (p, t) in enumerate(zip(r.parents.view(-1).tolist(), r.tokens.view(-1).tolist())):
        m = n[p].item()
        assert r.hist_len[i].item() == m + 1
        assert r.history[i, : m + 1].tolist() == h[p, :m].tolist() + [t]
    n.fill_(9)
    r = beams.select(x, torch.zeros((3, 4)).cuda(), history=h, hist_len=n)
    with pytest.raises(rai_b200.RaiError):
        paged.status()
    assert r.hist_len.tolist() == [9] * 12 and r.history[0].tolist() == h[r.parents.view(-1)[0]].tolist()


def test_in_a_graph_and_twice_the_same():
    from rai_b200 import beams
    x = torch.randn((4, 4, 40000), device="cuda")
    s = torch.zeros((4, 4), device="cuda")
    want = beams.select(x, s, eos=5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = beams.select(x, s, eos=5)
    x.mul_(0.5)
    graph.replay()
    second = beams.select(x, s, eos=5)
    torch.cuda.synchronize()
    for a, b in zip(got[:6], second[:6]):
        assert torch.equal(a, b)
    assert not torch.equal(want.cand_scores, got.cand_scores)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_more_equal_logits_than_a_buffer_holds(dtype):
    """Long runs of the best value, and steps that each beat the last."""
    x = torch.zeros((2, 3, 70001), dtype=dtype)
    x[0, 0, 9000:60000] = 3.0
    x[0, 1] = torch.arange(70001).div(8192, rounding_mode="floor").to(dtype)
    x[0, 2, ::2] = 1.0
    x[1, 0, 65000:] = 2.0
    x[1, 1] = -math.inf
    x[1, 1, 69990:] = 1.0
    s = torch.tensor([[0.0, -1.0, -0.5], [0.0, 0.0, 0.0]])
    check(x.cuda(), s.cuda(), eos=9001)
    check(x.cuda(), s.cuda(), keep=64, eos=3)


def test_on_two_streams_at_once():
    from rai_b200 import beams
    xs = [torch.randn((8, 4, 50000), device="cuda") for _ in range(2)]
    s = torch.zeros((8, 4), device="cuda")
    want = [beams.select(x, s) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(beams.select(xs[i], s))
    torch.cuda.synchronize()
    for w, rs in zip(want, got):
        for r in rs:
            for a, b in zip(w[:6], r[:6]):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N,V", [(4, 3001), (8, 500), (2, 152001), (32, 4097)])
@pytest.mark.parametrize("peak", [0.0, 12.0])
def test_beams_nearer_than_32_bits(dtype, N, V, peak):
    """Beam scores set so that the best candidates of different beams are at
    the same sum but for the scores' own rounding (1e-7 and less), on flat
    rows and on rows where a few tokens hold the mass."""
    g = torch.Generator().manual_seed(V)
    B = 24 if V < 10000 else 6
    x = 2 * torch.randn((B, N, V), generator=g)
    for i in range(3):
        at = torch.randint(0, V, (B, N, 1), generator=g)
        x.scatter_(2, at, peak + torch.rand((B, N, 1), generator=g))
    x = x.to(dtype)
    y = x.double()
    s = (-4.0 - (y.amax(2) - torch.logsumexp(y, 2))).float()
    check(x.cuda(), s.cuda(), eos=V // 2)
    check(x.cuda(), s.cuda(), keep=N)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_beams_of_infinite_score(dtype):
    """What a grammar took out of a beam of +infinity is not chosen before what
    it left."""
    from rai_b200 import beams
    g = torch.Generator().manual_seed(9)
    x = torch.randn((1, 2, 500), generator=g).to(dtype)
    x[:, :, 7:] = -math.inf
    s = torch.tensor([[-1.0, math.inf]])
    r = beams.select(x.cuda(), s.cuda(), keep=16)
    left = sorted(range(7), key=lambda t: (-x[0, 1, t].item(), t))
    assert r.cand_beams[0, :7].tolist() == [1] * 7 and r.cand_tokens[0, :7].tolist() == left
    assert (r.cand_scores[0, :7] == math.inf).all()
    other = sorted(range(7), key=lambda t: (-x[0, 0, t].item(), t))
    assert r.cand_beams[0, 7:14].tolist() == [0] * 7 and r.cand_tokens[0, 7:14].tolist() == other
    assert (r.cand_scores[0, 14:] == -math.inf).all() and not torch.isnan(r.scores).any()
    assert r.parents[0].tolist() == [1, 1] and r.tokens[0].tolist() == left[:2]
    one = beams.select(x[:, 1:].cuda(), s[:, 1:].cuda(), keep=16)
    assert one.cand_tokens[0].tolist() == left + list(range(7, 16))
    assert (one.cand_scores[0, :7] == math.inf).all() and (one.cand_scores[0, 7:] == -math.inf).all()
