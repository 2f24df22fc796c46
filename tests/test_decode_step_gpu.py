"""The decode-step operators together, as a program runs them: 4-bit projections (q, k and v fused in one layer), norm,
rotation and storing, attention over the cache, output projection with the plan's residual add, logits, a token - a prompt
first, in chains, then a tree of drafted tokens - captured into one graph, against the same model in 64 bits.

The reference computes in 64 bits and rounds keys and values to f16 as the cache does.  A key or value that lies next to
a rounding border may come out one step (2^-10 of its size) apart: scores then differ by at most
ds = 2^-10 * scale * sum|q k| <= 2^-10 * max|s|_1, probabilities by e^{2 ds}, the attention's output by
max|v| * (2 ds + 2^-10); every product after that passes it on as a plain sum of magnitudes."""
import numpy as np
import pytest

import oracle

pytestmark = pytest.mark.gpu

HID, HQ, HKV, D, VOCAB, PAGE, GROUP = 256, 8, 2, 64, 999, 16, 64
PROMPT, NODES = 70, 6
PARENT = [-1, 0, 0, 1, 1, 2]


def rotate(x, pos):
    half = D // 2
    angle = pos[:, None] * 10000.0 ** (-2.0 * np.arange(half) / D)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * c - b * s, b * c + a * s], axis=2)


def norm(x, gamma):
    return x / np.sqrt((x * x).mean(axis=2, keepdims=True) + 1e-6) * gamma


def test_a_prompt_and_a_drafted_tree(nne, ctx):
    import torch
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    layer = lambda n, k, seed: nne.QLinear4.from_linear(nne.Linear(oracle.normal(800, seed, (n, k), 0.0, 0.08)), GROUP, ctx)  # noqa: E731
    width = (HQ + 2 * HKV) * D
    qkv, proj, head = layer(width, HID, 1), layer(HID, HQ * D, 2), layer(VOCAB, HID, 3)
    wq, wo, wh = (x.to_linear().weight.astype(np.float64) for x in (qkv, proj, head))
    gq, gk = oracle.normal(801, 0, (D,), 1.0, 0.1), oracle.normal(801, 1, (D,), 1.0, 0.1)
    tokens = PROMPT + NODES
    h = oracle.normal(802, 0, (tokens, HID))
    depth = [0] * NODES
    for i, p in enumerate(PARENT):
        depth[i] = 0 if p < 0 else depth[p] + 1
    position = np.array(list(range(PROMPT)) + [PROMPT + x for x in depth], np.int32)
    masks = []
    for i, p in enumerate(PARENT):
        masks.append((masks[p] if p >= 0 else 0) | 1 << i)

    # the model in 64 bits
    rows = (h.astype(np.float64) @ wq.T).reshape(tokens, -1, D)
    q = rotate(norm(rows[:, :HQ], gq.astype(np.float64)), position)
    k = rotate(norm(rows[:, HQ:HQ + HKV], gk.astype(np.float64)), position).astype(np.float16).astype(np.float64)
    v = rows[:, HQ + HKV:].astype(np.float16).astype(np.float64)
    att, ds = np.zeros((tokens, HQ, D)), 0.0
    for t in range(tokens):
        sees = list(range(t + 1)) if t < PROMPT else list(range(PROMPT)) + [PROMPT + j for j in range(NODES) if masks[t - PROMPT] >> j & 1]
        for x in range(HQ):
            kk, vv = k[sees, x // (HQ // HKV)], v[sees, x // (HQ // HKV)]
            s = kk @ q[t, x] * D ** -0.5
            ds = max(ds, 2.0 ** -10 * D ** -0.5 * float((np.abs(kk) @ np.abs(q[t, x])).max()))
            w = np.exp(s - s.max())
            att[t, x] = (w / w.sum()) @ vv
    off = np.abs(v).max() * (2 * ds + 2.0 ** -10) * 1.05
    hidden = att.reshape(tokens, -1) @ wo.T + h
    logits = hidden @ wh.T
    far = np.abs(wh) @ (np.abs(wo).sum(axis=1) * off)  # per token of the vocabulary
    far = far + 1e-4 * np.abs(logits).max()            # f32 arithmetic of four products

    # the same on the device
    pages = -(-tokens // PAGE) + 1
    cache = nne.PagedKvCache(ctx, pages, PAGE, HKV, D, "f16", rope_dims=D)
    hd, table = dev(h), dev(np.random.default_rng(0).permutation(pages).astype(np.int32)[None, :-1])
    buf = torch.empty(tokens, width, device="cuda")
    qo, at, hid, lg = (torch.empty(tokens, n, device="cuda") for n in (HQ * D, HQ * D, HID, VOCAB))
    gqd, gkd, pos = dev(gq), dev(gk), dev(position)
    seq, place = torch.zeros(tokens, device="cuda", dtype=torch.int32), torch.arange(tokens, device="cuda", dtype=torch.int32)
    vis, u = dev(np.array(masks, np.int64)), torch.zeros(tokens, device="cuda")
    tok, temp = torch.full((tokens,), -5, device="cuda", dtype=torch.int32), torch.zeros(tokens, device="cuda")
    pieces = [(0, 64), (64, PROMPT), (PROMPT, tokens)]
    keep = []

    def step(lo, hi, tree):
        n, p = hi - lo, lambda t, w: t.data_ptr() + 4 * w * lo
        start, context = dev(np.array([0, n], np.int32)), dev(np.array([lo], np.int32))
        keep.append((start, context))
        append = nne.KvAppend(cache, n, HQ, p(buf, width), p(buf, width) + 4 * HQ * D, p(buf, width) + 4 * (HQ + HKV) * D, p(qo, HQ * D),
                              width, width, width, gqd.data_ptr(), gkd.data_ptr(), 1e-6, table.data_ptr(), pages - 1, 1, p(seq, 1), p(place, 1),
                              p(pos, 1))
        attend = nne.TreeAttention(cache, n, HQ, p(qo, HQ * D), p(at, HQ * D), 1, start.data_ptr(), context.data_ptr(), table.data_ptr(),
                                   pages - 1, n, lo, vis.data_ptr() if tree else 0)
        sample = nne.Sampler(ctx, n, VOCAB, p(lg, VOCAB), p(u, 1), p(tok, 1), p(temp, 1))

        def run(s):
            qkv.forward_device(p(hd, HID), n, p(buf, width), s)
            append.run(s)
            attend.run(s)
            proj.forward_device(p(at, HQ * D), n, p(hid, HID), s)
            nne.add_device(ctx, p(hid, HID), p(hd, HID), n * HID, p(hid, HID), s)
            head.forward_device(p(hid, HID), n, p(lg, VOCAB), s)
            sample.run(s)
        return run

    steps = [step(lo, hi, i == 2) for i, (lo, hi) in enumerate(pieces)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for f in steps:
        f(s.cuda_stream)
    s.synchronize()

    def verify():
        assert np.all(np.abs(lg.cpu().numpy() - logits) <= far)
        got = tok.cpu().numpy()
        assert np.all(logits[np.arange(tokens), got] >= (logits - far).max(axis=1) - far[got])
    verify()
    first = lg.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        for f in steps:
            f(s.cuda_stream)
    for t in (buf, qo, at, hid, lg):
        t.fill_(float("nan"))
    g.replay()
    torch.cuda.synchronize()
    verify()
    assert torch.equal(first, lg)
    ctx.check()


def test_a_pool_beyond_32_bits(nne, ctx):
    """Keys and values at the end of a pool of more than 2^32 elements: stored there, read from there."""
    import torch
    page, d, pages = 1024, 256, 16400
    k, v = (torch.empty(pages, 1, page, d, device="cuda", dtype=torch.float16) for _ in range(2))
    assert k.numel() > 2 ** 32
    cache = nne.PagedKvCache(ctx, pages, page, 1, d, "f16", k.data_ptr(), v.data_ptr())
    n = 40
    x = torch.randn(3, n, d, device="cuda")
    table = torch.tensor([[pages - 1]], device="cuda", dtype=torch.int32)
    seq, at = torch.zeros(n, device="cuda", dtype=torch.int32), torch.arange(n, device="cuda", dtype=torch.int32)
    s = torch.cuda.current_stream().cuda_stream
    nne.KvAppend(cache, n, k=x[1].data_ptr(), v=x[2].data_ptr(), page_table=table.data_ptr(), table_stride=1, sequences=1,
                 sequence=seq.data_ptr(), index=at.data_ptr()).run(s)
    assert torch.equal(k[-1, 0, :n], x[1].half()) and torch.equal(v[-1, 0, :n], x[2].half())
    out = torch.empty(n, d, device="cuda")
    start, context = torch.tensor([0, n], device="cuda", dtype=torch.int32), torch.zeros(1, device="cuda", dtype=torch.int32)
    for rows in (n, 1):  # both kernels
        start[1] = rows
        nne.TreeAttention(cache, n, 1, x[0].data_ptr(), out.data_ptr(), 1, start.data_ptr(), context.data_ptr(), table.data_ptr(), 1, rows,
                          0).run(s)
        for r in range(rows):
            # Scores are off by (D / 16 + 8) 2^-22 of scale * sum |q k|, which enters numerator and denominator; the probabilities'
            # parts and the sums over one tile of keys by fewer than 40 steps of 2^-22 more.
            keys, values, q = x[1, :r + 1].half().double(), x[2, :r + 1].half().double(), x[0, r].double()
            w = torch.softmax(keys @ q * d ** -0.5, dim=0)
            size = float((keys.abs() @ q.abs()).max()) * d ** -0.5
            bound = (2 * (d / 16 + 8) * size + 40) * 2.0 ** -22 * (w @ values.abs())
            assert bool(((out[r].double() - w @ values).abs() <= bound).all())


FIRST_CALL = """
import importlib, sys
sys.path.insert(0, %r)
import torch
nne = importlib.import_module("neural-network-engine_b200")
ctx = nne.default_context(0)
k, v = (torch.randn(8, 2, 16, 64, device="cuda").half() for _ in range(2))
q, out = torch.randn(1, 8, 64, device="cuda"), torch.zeros(1, 8, 64, device="cuda")
i = lambda *x: torch.tensor(x, device="cuda", dtype=torch.int32)
start, context, table = i(0, 1), i(100), i(*range(8))
cache = nne.PagedKvCache(ctx, 8, 16, 2, 64, "f16", k.data_ptr(), v.data_ptr())
call = nne.TreeAttention(cache, 1, 8, q.data_ptr(), out.data_ptr(), 1, start.data_ptr(), context.data_ptr(), table.data_ptr(), 8, 1, 100)
logits, u, tok = torch.randn(1, 9000, device="cuda"), torch.zeros(1, device="cuda"), i(-1)
draw = nne.Sampler(ctx, 1, 9000, logits.data_ptr(), u.data_ptr(), tok.data_ptr())
w, x, y = torch.randn(64, 64, device="cuda"), torch.randn(9, 64, device="cuda"), torch.zeros(9, 64, device="cuda")
layer = nne.QLinear4.from_linear_device(ctx, w.data_ptr(), 0, 64, 64, 32)
torch.cuda.synchronize()
s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    call.run(s.cuda_stream)
    draw.run(s.cuda_stream)
    layer.forward_device(x.data_ptr(), 9, y.data_ptr(), s.cuda_stream)
g.replay()
torch.cuda.synchronize()
a, b, c = out.clone(), tok.clone(), y.clone()
out.zero_(), tok.zero_(), y.zero_()
call.run(), draw.run(), layer.forward_device(x.data_ptr(), 9, y.data_ptr())
torch.cuda.synchronize()
assert torch.equal(a, out) and torch.equal(b, tok) and torch.equal(c, y) and bool(a.any()) and bool(c.any())
"""


def test_a_first_call_may_be_captured(nne):
    """In a process of its own: what the library asks the driver once is asked while a stream is being captured."""
    import subprocess
    import sys
    root = oracle.ROOT
    r = subprocess.run([sys.executable, "-c", FIRST_CALL % root], cwd=root, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
