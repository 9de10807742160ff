"""GPU tests of sampling (btf_sample) against a plain implementation in 64 bits (numpy).

Tokens have to be equal. The masses differ by 2^-45 of the largest one (fixed point) and 2^-52 relative (exp), so a
token can differ only where u lies within about V 2^-45 of a border of the running mass: below 10^-8 for the rows
here. Log-probabilities: the exponent and the log are taken in 64 bits and rounded once (2^-24 relative); the fixed
point moves a mass w by 2^-45 (2^-45 / w relative, w > e^-20 here: 2^-16 at most) and Z >= 1 by V 2^-45 < 2^-26."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _reference(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """(token, logprob) of one row of float values."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return 0, np.nan
    order = np.argsort(-x, kind="stable")
    if not T > 0:
        return int(order[0]), 0.0
    with np.errstate(invalid="ignore"):
        e = np.where(x == top, 0.0, (x - top) / np.float64(T))
    e = np.where(np.isnan(e), -np.inf, e)
    w = np.exp(e)
    n = len(x) if k <= 0 else min(k, len(x))
    if p < 1:
        c = np.cumsum(w[order[:n]])
        n = min(n, int(np.searchsorted(c, np.float64(p) * c[-1])) + 1)
    keep = np.zeros(len(x), bool)
    keep[order[:max(n, 1)]] = True
    if m > 0:
        keep &= e >= min(np.log(np.float64(m)), 0.0)
    c = np.cumsum(np.where(keep, w, 0.0))
    t = int(np.searchsorted(c, np.float64(u) * c[-1], side="right"))
    return t, e[t] - np.log(c[-1])


def _run(btf, cuda, x, u, T=None, k=None, p=None, m=None):
    f = lambda a, t: None if a is None else torch.as_tensor(np.asarray(a), dtype=t).to(cuda)  # noqa: E731
    tok, lp = btf.sample(x, f(u, torch.float32), f(T, torch.float32), f(k, torch.int32), f(p, torch.float32),
                         f(m, torch.float32))
    assert btf.device_error() == 0
    return tok.cpu().numpy(), lp.cpu().numpy()


def _compare(btf, cuda, x, u, T=None, k=None, p=None, m=None):
    x = x.to(cuda)
    tok, lp = _run(btf, cuda, x, u, T, k, p, m)
    rows = x.float().cpu().numpy()
    for b in range(len(rows)):
        at = lambda a, d, t=np.float32: d if a is None else t(np.asarray(a)[b])  # noqa: E731
        t, l = _reference(rows[b], np.float32(np.asarray(u)[b]), at(T, 1.0), at(k, 0, int), at(p, 1.0), at(m, 0.0))
        assert tok[b] == t, (b, tok[b], t)
        np.testing.assert_allclose(lp[b], l, rtol=2.0 ** -23, atol=2.0 ** -15, err_msg=str(b))


def _logits(B, V, seed, scale=2.2, hot=40):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=g) * scale
    at = torch.randint(V, (B, hot), generator=g)
    return x.scatter_add(1, at, torch.rand(B, hot, generator=g) * 9)


FILTERS = [dict(), dict(k=50), dict(p=0.9), dict(m=0.05), dict(k=200, p=0.95, m=0.01), dict(k=1), dict(p=0.0),
           dict(m=1.0), dict(k=5000, p=0.999)]


@pytest.mark.parametrize("f", FILTERS, ids=str)
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 33), (4, 1000), (3, 16384), (2, 16385), (7, 50257), (2, 128003),
                                 (3, 248320), (1, 524288)])
def test_shapes_and_filters(cuda, btf, B, V, f):
    rng = np.random.default_rng(V + B)
    a = {n: np.full(B, v) for n, v in f.items()}
    _compare(btf, cuda, _logits(B, V, V), rng.random(B, dtype=np.float32), T=rng.uniform(0.3, 1.5, B), **a)


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("f", FILTERS[:5], ids=str)
def test_types_with_many_ties(cuda, btf, t, f):
    """16-bit logits: thousands of equal values, cut in index order."""
    B, V = 6, 50257
    rng = np.random.default_rng(11)
    _compare(btf, cuda, _logits(B, V, 9).to(t), rng.random(B, dtype=np.float32), T=np.full(B, 1.7),
             **{n: np.full(B, v) for n, v in f.items()})


@pytest.mark.parametrize("V", [5, 300, 40000, 248320])
@pytest.mark.parametrize("f", [dict(), dict(k=3), dict(k=257), dict(p=0.5), dict(k=400, p=0.25), dict(m=1.0)], ids=str)
def test_all_equal(cuda, btf, V, f):
    """One key: every cut falls among ties."""
    u = np.array([0.0, 0.3, 0.99999994], np.float32)
    _compare(btf, cuda, torch.full((3, V), -1.25), u, **{n: np.full(3, v) for n, v in f.items()})


@pytest.mark.parametrize("f", [dict(k=1000), dict(p=0.7), dict(k=30000, p=0.6)], ids=str)
def test_cuts_among_close_values(cuda, btf, f):
    """Tens of thousands of different values in one bin of the first histogram, and two tied plateaus."""
    g = torch.Generator().manual_seed(12)
    x = 5.0 + torch.rand(4, 60000, generator=g) * 1e-3
    x[1] = torch.where(torch.rand(60000, generator=g) < 0.5, 5.0, 5.0 + 2 ** -20)
    x[2, ::2] = 4.999
    x[3] = torch.arange(60000) * 1e-7 + 1.0
    _compare(btf, cuda, x, np.array([0.1, 0.5, 0.7, 0.95], np.float32), **{n: np.full(4, v) for n, v in f.items()})


def test_rows_with_their_own_parameters(cuda, btf):
    B, V = 24, 4099
    rng = np.random.default_rng(3)
    _compare(btf, cuda, _logits(B, V, 2), rng.random(B, dtype=np.float32),
             T=rng.choice([0.0, -1.0, 0.2, 1.0, 3.0], B), k=rng.choice([0, -3, 1, 7, 4099, 9999], B),
             p=rng.choice([0.0, 0.2, 0.9, 1.0, 2.0], B), m=rng.choice([0.0, -1.0, 0.1, 1.0, 5.0], B))


def test_special_values(cuda, btf):
    """NaN and infinities, zeros of both signs, extreme temperatures, and random numbers at and outside their ends."""
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(14, 9)
    x[0] = nan
    x[1] = -inf
    x[2, :] = torch.tensor([nan, -inf, 3, nan, 3, -inf, 1, 2, nan])
    x[3, 4] = inf
    x[4, 2] = x[4, 7] = inf
    x[5] = torch.tensor([0.0, -0.0] * 4 + [0.0])
    x[6, 3] = 1e30
    x[7] = torch.linspace(-1e30, 1e30, 9)
    x[8, 1] = -inf
    x[9] = torch.arange(9)
    x[10] = torch.arange(9)
    x[11] = torch.arange(9)
    x[12] = torch.arange(9)
    x[13, 5] = 3e38
    T = np.array([1, 1, 1, 1, 1, 0, 1, 1e30, inf, 1e-45, 1e-30, 1e30, nan, 1], np.float32)
    u = np.array([.5, .5, .6, .5, .7, .5, .5, .9, .95, .5, .5, 0.0, .5, .99], np.float32)
    _compare(btf, cuda, x, u, T=T)
    _compare(btf, cuda, x, u, T=T, k=np.full(14, 2), p=np.full(14, 0.9), m=np.full(14, 0.1))
    # u outside [0, 1): the nearest draw there is; NaN parameters are off
    y = torch.arange(6.0).repeat(4, 1).to(cuda)
    tok, _ = _run(btf, cuda, y, [-1.0, nan, 1.0, 7.0], p=[nan, nan, nan, nan], m=[nan] * 4)
    assert tok.tolist() == [0, 0, 5, 5]


def test_ends_of_u(cuda, btf):
    """u = 0 draws the first kept token, the largest u below 1 the last, and every kept token is drawn in between."""
    x = torch.tensor([[1.0, 5.0, 2.0, 5.0, 4.0, -3.0]]).repeat(2, 1).to(cuda)
    tok, _ = _run(btf, cuda, x, [0.0, 0.99999994], k=[3, 3])
    assert tok.tolist() == [1, 4]
    n = 4096
    tok, lp = _run(btf, cuda, x[:1].repeat(n, 1), (np.arange(n) + 0.5) / n, k=np.full(n, 3))
    w = np.exp([0.0, 0.0, -1.0])
    got = np.array([(tok == t).sum() for t in (1, 3, 4)])
    assert got.sum() == n and np.abs(got - n * w / w.sum()).max() <= 1
    np.testing.assert_allclose(np.exp(lp), (w / w.sum())[np.searchsorted([1, 3, 4], tok)], rtol=2.0 ** -21)


def test_strided_rows_and_offsets(cuda, btf):
    V = 1003
    buf = _logits(5, 2 * V + 1, 5)
    u = np.linspace(0.05, 0.95, 5).astype(np.float32)
    _compare(btf, cuda, buf[:, 1:1 + V], u, k=np.full(5, 20))
    d = buf.to(cuda)
    tok, _ = _run(btf, cuda, d[:, 1:1 + V], u, k=np.full(5, 20))
    again, _ = _run(btf, cuda, d[:, 1:1 + V].contiguous(), u, k=np.full(5, 20))
    assert np.array_equal(tok, again)
    big = torch.empty(2, 2 ** 31 // 2 + 8, dtype=torch.float16, device=cuda)  # the second row begins behind 2^30 values
    rows = big[:, :V]
    rows.copy_(buf[:2, :V].half())
    tok, _ = _run(btf, cuda, rows, u[:2], k=[9, 9])
    again, _ = _run(btf, cuda, buf[:2, :V].half().to(cuda), u[:2], k=[9, 9])
    assert np.array_equal(tok, again)


def test_streams_and_graph(cuda, btf):
    """Two calls at once on two streams, and a captured call replayed on changed logits, parameters and numbers."""
    B, V = 8, 100003
    x = _logits(B, V, 6).to(cuda)
    u = torch.rand(B, device=cuda)
    p = torch.full((B,), 0.8, device=cuda)
    want = btf.sample(x, u, top_p=p)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        got.append([btf.sample(x, u, top_p=p, stream=s) for _ in range(3)])
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for calls in got:
        for tok, lp in calls:
            assert torch.equal(tok, want[0]) and torch.equal(lp, want[1])
    tok, lp = torch.empty_like(want[0]), torch.empty_like(want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        btf.sample(x, u, top_p=p, tokens=tok, logprobs=lp)
    for seed in (7, 8):
        x.copy_(_logits(B, V, seed))
        u.copy_(torch.rand(B, generator=torch.Generator().manual_seed(seed)))
        p.fill_(0.5 + seed / 100)
        graph.replay()
        want = btf.sample(x, u, top_p=p)
        assert torch.equal(tok, want[0]) and torch.equal(lp, want[1])


def test_refusals(cuda, btf):
    x, u = torch.zeros(2, 10, device=cuda), torch.zeros(2, device=cuda)
    for fn in (lambda: btf.sample(x, u.double()), lambda: btf.sample(x, u[:1]), lambda: btf.sample(x.double(), u),
               lambda: btf.sample(x, u, top_k=torch.zeros(2, device=cuda)), lambda: btf.sample(x, u.cpu()),
               lambda: btf.sample(x[:, ::2], u), lambda: btf.sample(x[:1].expand(2, 10), u),
               lambda: btf.sample(x, u, tokens=torch.zeros(2, dtype=torch.int64, device=cuda))):
        with pytest.raises(RuntimeError):
            fn()
    assert btf.sample(x[:0], u[:0])[0].shape == (0,)


@pytest.mark.parametrize("f", [dict(), dict(k=50), dict(k=3000, p=0.9), dict(p=0.9), dict(p=0.9999), dict(m=0.05), dict(m=1e-9),
                               dict(k=200, p=0.95, m=0.01)], ids=str)
@pytest.mark.parametrize("B,V,off,t", [(100, 60001, 0, torch.float32), (100, 60001, 1, torch.float16),
                                       (20, 248321, 3, torch.bfloat16), (310, 20000, 0, torch.float16),
                                       (75, 8192, 0, torch.float32), (300, 524288, 0, torch.bfloat16)])
def test_many_rows(cuda, btf, B, V, off, t, f):
    """More rows than the card holds in shared memory: the token and the log-probability of a row are those that it has
    in a call of its own, to the last bit, and those of the plain form."""
    g = torch.Generator(device=cuda).manual_seed(V + B)
    x = (torch.randn(B, V + off, generator=g, device=cuda) * 2.2).to(t)[:, off:]
    x[1] = -3.0
    x[2, ::3] = float("nan")
    x[3] = float("-inf")
    x[4, V // 2:] = float("-inf")
    x[5] = x[5].round()
    x[6, :V - 1] = -100.0
    x[7, V // 3] = float("inf")
    x[8] *= 0.01
    rng = np.random.default_rng(B)
    u, T = rng.random(B, dtype=np.float32), rng.choice([0.0, 0.5, 1.0, 1.3], B).astype(np.float32)
    T[1:9] = 1.0
    a = {n: np.full(B, v) for n, v in f.items()}
    tok, lp = _run(btf, cuda, x, u, T, **a)
    rows = list(range(12)) + [B // 2, B - 2, B - 1]
    for b in rows:
        one, lpo = _run(btf, cuda, x[b:b + 1], u[b:b + 1], T[b:b + 1], **{n: v[b:b + 1] for n, v in a.items()})
        assert tok[b] == one[0] and np.array_equal(lp[b:b + 1], lpo, equal_nan=True), b
    for b in [1, 2, 4, 5, 8, 10, B - 1]:
        r, l = _reference(x[b].float().cpu().numpy(), u[b], T[b], f.get("k", 0), np.float32(f.get("p", 1.0)),
                          np.float32(f.get("m", 0.0)))
        assert tok[b] == r, b
        np.testing.assert_allclose(lp[b], l, rtol=2.0 ** -23, atol=2.0 ** -15, err_msg=str(b))


@pytest.mark.parametrize("f", FILTERS[:5], ids=str)
@pytest.mark.parametrize("B,V", [(1, 70000), (2, 131073), (3, 33000), (9, 66000), (1, 4097)])
def test_ctas_without_logits(cuda, btf, B, V, f):
    """Rows whose last CTAs of the cluster have nothing to read (70000 values: 12 parts of 6144 for 16 CTAs), launched
    back to back: those CTAs reach the cluster's first exchange before the others have begun to read."""
    rng = np.random.default_rng(V)
    x, u, T = _logits(B, V, V), rng.random(B, dtype=np.float32), rng.uniform(0.3, 1.5, B)
    a = {n: np.full(B, v) for n, v in f.items()}
    _compare(btf, cuda, x, u, T=T, **a)
    xd, ud, t = x.to(cuda), torch.from_numpy(u).to(cuda), torch.from_numpy(T.astype(np.float32)).to(cuda)
    par = {dict(k="top_k", p="top_p", m="min_p")[n]: torch.as_tensor(v, dtype=torch.int32 if n == "k" else torch.float32).to(cuda)
           for n, v in a.items()}
    outs = [btf.sample(xd, ud, temperature=t, **par) for _ in range(50)]
    for tok, lp in outs[1:]:
        assert torch.equal(tok, outs[0][0]) and torch.equal(lp, outs[0][1])
    assert btf.device_error() == 0


@pytest.mark.parametrize("V", [4, 4099, 248320])
def test_tokens_without_mass_are_not_drawn(cuda, btf, V):
    """Masses are 2^-44 fixed point: e^-30 of the largest is 1.6 of a unit, e^-31.5 is 0.4 and rounds to none, so u = 0
    draws the first token that has one."""
    x = torch.full((3, V), -100.0)
    x[:, 1], x[:, 2], x[:, 3] = -31.5, torch.tensor([-30.0, -31.5, -30.0]), 0.0
    x[2, 0] = -30.0
    tok, lp = _run(btf, cuda, x.to(cuda), np.zeros(3, np.float32))
    assert tok.tolist() == [2, 3, 0]
    np.testing.assert_allclose(lp, [-30.0, 0.0, -30.0], atol=1e-9, rtol=2.0 ** -23)
