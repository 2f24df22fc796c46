"""Drawing tokens on the device against the definition in 64 bits.

The kernel's weights are f32 (expf's 2 steps, a subtraction and a division: a relative 2^-21 where a weight matters, more
only below e^-20), its sums exact.  So a token is right when uniform lies in its interval widened by 2e-6 of the mass;
where a token's place lies within 2e-6 of top_p's border or its weight within 2e-6 of min_p, either decision about it is
right, and its mass widens the intervals too.  All other choices (ties, orders, masks) are held to exactly."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
SLACK = 2e-6


def right_tokens(l, t, k, p, m, u):
    """The tokens that may come back for one row."""
    l = np.where(np.isnan(l), -np.inf, l.astype(np.float64)) + 0.0
    if not (l > -np.inf).any():
        return {-1}
    if not t > 0:
        return {int(np.argmax(l))}
    with np.errstate(all="ignore"):
        w = np.exp(np.where(l == l.max(), 0.0, (l - l.max()) / t))
    order = np.lexsort((np.arange(l.size), -l))
    order = order[l[order] > -np.inf]
    if 0 < k < order.size:
        order = order[:k]
    before = np.concatenate([[0.0], np.cumsum(w[order])])
    total, loose = before[-1], 0.0
    if p < 1:
        near = np.abs(before[:-1] - p * total) < SLACK * total
        near[0] = False
        loose += w[order][near].sum()
        keep = before[:-1] < p * total
        keep[0] = True
        order = order[keep]
    m = min(m, 1.0)
    loose += w[order][np.abs(w[order] - m) < SLACK * m].sum() if 0 < m < 1 else 0.0
    order = np.sort(order[w[order] >= m])
    up = np.cumsum(w[order])
    slack = SLACK * up[-1] + loose
    at = min(max(u, 0.0), 1.0) * up[-1]
    ok = (up > at - slack) & (np.concatenate([[0.0], up[:-1]]) <= at + slack)
    return set(int(i) for i in order[ok & (w[order] > 0)])


def draw(nne, ctx, logits, u, t=None, k=None, p=None, m=None, gap=0):
    import torch
    rows, vocab = logits.shape
    wide = np.full((rows, vocab + gap), 99.0, np.float32)
    wide[:, :vocab] = logits
    d = lambda a, ty: None if a is None else torch.from_numpy(np.broadcast_to(np.asarray(a, ty), (rows,)).copy()).cuda()  # noqa: E731
    x = torch.from_numpy(wide).cuda()
    keep = [d(t, np.float32), d(k, np.int32), d(p, np.float32), d(m, np.float32), d(u, np.float32)]
    out = torch.full((rows + 1,), -9, device="cuda", dtype=torch.int32)
    ptr = [0 if a is None else a.data_ptr() for a in keep]
    call = nne.Sampler(ctx, rows, vocab, x.data_ptr(), ptr[4], out.data_ptr(), ptr[0], ptr[1], ptr[2], ptr[3], row_stride=vocab + gap)
    call.run(torch.cuda.current_stream().cuda_stream)
    got = out.cpu().numpy()
    call.run(torch.cuda.current_stream().cuda_stream)
    assert np.array_equal(got, out.cpu().numpy()) and got[rows] == -9
    return got[:rows]


def check(nne, ctx, logits, u, t=None, k=None, p=None, m=None, gap=0):
    got = draw(nne, ctx, logits, u, t, k, p, m, gap)
    rows = logits.shape[0]
    full = lambda a, off, ty: np.broadcast_to(np.asarray(off if a is None else a, ty), (rows,))  # noqa: E731
    t, k, p, m = full(t, 1, np.float32), full(k, 0, np.int64), full(p, 1, np.float32), full(m, 0, np.float32)
    u = full(u, 0, np.float32)
    for r in range(rows):
        right = right_tokens(logits[r], float(t[r]), int(k[r]), float(p[r]), float(m[r]), float(u[r]))
        assert int(got[r]) in right, (r, int(got[r]), sorted(right)[:5], t[r], k[r], p[r], m[r], u[r])


@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 4096, 4097, 32000, 50257, 128000, 300001])
def test_settings_mixed(nne, ctx, vocab):
    rng = np.random.default_rng(vocab)
    rows = 40 if vocab < 60000 else 16
    logits = (rng.standard_normal((rows, vocab)) * rng.choice([0.5, 2, 6], (rows, 1))).astype(np.float32)
    t = rng.choice([0.0, 0.3, 0.8, 1.0, 2.5], rows).astype(np.float32)
    k = rng.choice([0, 1, 2, 7, 50, 1000, 10 ** 6, -3], rows)
    p = rng.choice([1.0, 0.95, 0.5, 0.1, 0.999, 0.0, 1.5], rows).astype(np.float32)
    m = rng.choice([0.0, 0.0, 0.01, 0.3, 1.0, 2.0, -1.0], rows).astype(np.float32)
    check(nne, ctx, logits, rng.random(rows).astype(np.float32), t, k, p, m)


@pytest.mark.parametrize("vocab", [100, 9000])
def test_everything_off_and_one_at_a_time(nne, ctx, vocab):
    rng = np.random.default_rng(1)
    logits = (rng.standard_normal((30, vocab)) * 3).astype(np.float32)
    u = rng.random(30).astype(np.float32)
    check(nne, ctx, logits, u)
    check(nne, ctx, logits, u, t=0.7, gap=5)
    check(nne, ctx, logits, u, k=20)
    check(nne, ctx, logits, u, p=0.9, gap=1)
    check(nne, ctx, logits, u, m=0.05)


@pytest.mark.parametrize("vocab", [257, 20000])
def test_ties(nne, ctx, vocab):
    """Few distinct values: top-k and top-p end inside runs of equal logits, which are cut off by index."""
    rng = np.random.default_rng(2)
    rows = 48
    logits = rng.integers(-2, 3, (rows, vocab)).astype(np.float32)
    logits[:8] = 1.5                                       # all equal
    logits[8:12] = np.where(rng.random((4, vocab)) < 0.5, 0.0, -0.0)
    k = rng.choice([0, 1, 3, vocab // 7, vocab // 2, vocab - 1], rows)
    p = rng.choice([1.0, 0.7, 0.31, 0.05, 0.0], rows).astype(np.float32)
    check(nne, ctx, logits, rng.random(rows).astype(np.float32), 1.0, k, p)
    check(nne, ctx, logits, np.float32(0.9999), 0.5, k, p, 0.2)


@pytest.mark.parametrize("vocab", [20000, 70000])
def test_a_top_k_beyond_the_threads(nne, ctx, vocab):
    """More places than a cluster has threads (2048 at this many rows), with and without top-p."""
    rng = np.random.default_rng(6)
    rows = 64
    logits = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    logits[::2, : vocab // 2] -= 12.0                      # a cluster's parts that differ in their work
    logits[1::4] = np.round(logits[1::4])
    k = rng.choice([2049, 3000, 4100, 9001, vocab - 1], rows)
    for _ in range(4):
        u = rng.random(rows).astype(np.float32)
        check(nne, ctx, logits, u, 1.0, k, rng.choice([0.9, 0.5, 0.1, 1.0], rows).astype(np.float32))
        check(nne, ctx, logits, u, 0.7, k)


@pytest.mark.parametrize("vocab", [64, 12345])
def test_masked_and_special_logits(nne, ctx, vocab):
    rng = np.random.default_rng(3)
    base = (rng.standard_normal((12, vocab)) * 3).astype(np.float32)
    low = np.finfo(np.float32).min
    x = base.copy()
    x[0, rng.random(vocab) < 0.9] = -np.inf
    x[1] = -np.inf                                         # nothing to choose: -1
    x[2] = np.nan
    x[3, 1::2] = np.nan
    x[4, rng.random(vocab) < 0.9] = low
    x[5] = low
    x[6], x[6, 40] = -np.inf, -5.0                         # one choice
    x[7, 13], x[7, 50] = np.inf, np.inf                    # infinities share the mass
    x[8] *= 1e30
    x[9] = 1e-42
    x[10, 5] = np.finfo(np.float32).max
    u = rng.random(12).astype(np.float32)
    for s in (dict(), dict(k=5), dict(p=0.8), dict(k=30, p=0.5), dict(m=0.1), dict(t=0.0), dict(t=1e-3, k=5, p=0.9), dict(t=1e6, p=0.5),
              dict(t=float("inf"), p=0.25, k=40), dict(t=float("nan")), dict(t=1e-42, k=9, p=0.9)):
        check(nne, ctx, x, u, **s)


def test_ends_of_the_uniform_number(nne, ctx):
    logits = np.tile(np.array([0.0, 1.0, -np.inf, 2.0, -1.0, -np.inf], np.float32), (5, 1))
    assert draw(nne, ctx, logits, np.array([0.0, 1.0, 0.99999994, -3.0, np.nan], np.float32)).tolist() == [0, 4, 4, 0, 0]


def test_the_inverse_of_the_distribution(nne, ctx):
    """Every token comes back exactly on its interval of a fine grid of uniform numbers."""
    rng = np.random.default_rng(4)
    row = (rng.standard_normal(300) * 2).astype(np.float32)
    n = 4096
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    check(nne, ctx, np.tile(row, (n, 1)), u, 0.9, 100, 0.9, 0.01)


def test_another_stream_and_a_captured_call(nne, ctx):
    import torch
    rng = np.random.default_rng(5)
    rows, vocab = 7, 40000
    x = torch.from_numpy((rng.standard_normal((rows, vocab)) * 3).astype(np.float32)).cuda()
    u = torch.from_numpy(rng.random(rows).astype(np.float32)).cuda()
    k, p = torch.full((rows,), 50, device="cuda", dtype=torch.int32), torch.full((rows,), 0.9, device="cuda")
    out = torch.zeros(rows, device="cuda", dtype=torch.int32)
    call = nne.Sampler(ctx, rows, vocab, x.data_ptr(), u.data_ptr(), out.data_ptr(), top_k=k.data_ptr(), top_p=p.data_ptr())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        x.mul_(1.01)
        call.run(s.cuda_stream)
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        for r, row in enumerate(x.cpu().numpy()):
            assert int(out[r]) in right_tokens(row, 1.0, 50, float(np.float32(0.9)), 0.0, float(u[r]))


def test_refusals(nne, ctx):
    good = dict(rows=1, vocab=10, logits=16, uniform=16, tokens=16)
    for change in (dict(vocab=0), dict(vocab=2 ** 22 + 1), dict(row_stride=9), dict(rows=2 ** 40), dict(logits=0), dict(uniform=0), dict(tokens=0),
                   dict(logits=18), dict(tokens=18), dict(top_k=17), dict(uniform=19)):
        with pytest.raises(nne.InvalidArgument):
            nne.Sampler(ctx, **{**good, **change}).run()
    nne.Sampler(ctx, **{**good, "rows": 0}).run()
