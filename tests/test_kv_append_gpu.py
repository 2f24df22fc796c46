"""Filling the paged key/value cache on the device against numpy in 64 bits.

Bound, per element of a rotated pair (a, b), in units of |a| + |b|:  the angle is off by 2^-25 (its f32 rounding within
a quarter of a half turn), sin and cos by 2 steps of 2^-24 each, two products and a sum by 2^-24 each; a normed head
adds (d / 8 + 8) * 2^-24 (the sum of d squares over 32 lanes and five shuffles, a division and a root, halved by the
root, and two products).  Storing adds half a step of the type: 2^-8 (bf16), 2^-11 (f16) of the value, at least 2^-25
(f16's smallest step)."""
import ctypes as C

import numpy as np
import pytest

import oracle

pytestmark = pytest.mark.gpu
STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def torch_dtype(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16}[name]


def head_exact(x, gamma, eps, position, dims, pairs, freq):
    """(value, sum of magnitudes of the pair) of [tokens, heads, d] in 64 bits."""
    x = x.astype(np.float64)
    if gamma is not None:
        x = x / np.sqrt((x * x).mean(axis=2, keepdims=True) + eps) * gamma.astype(np.float64)
    y, mag = x.copy(), np.abs(x)
    if dims:
        angle = position.astype(np.float64)[:, None] * freq
        c, s = np.cos(angle)[:, None, :], np.sin(angle)[:, None, :]
        first, second = (slice(0, dims, 2), slice(1, dims, 2)) if pairs else (slice(0, dims // 2), slice(dims // 2, dims))
        a, b = x[..., first], x[..., second]
        y[..., first], y[..., second] = a * c - b * s, b * c + a * s
        mag[..., first] = mag[..., second] = np.abs(a) + np.abs(b)
    return y, mag


class Setup:
    def __init__(self, nne, ctx, tokens, hq, hkv, d, dims, pairs, norm, dtype, page, start, offset=0, gap=0, seed=0, freq=None):
        import torch
        rng = np.random.default_rng(seed + tokens * 7 + d)
        self.shape = (tokens, hq, hkv, d)
        width = (hq + 2 * hkv) * d + gap
        self.buf = torch.zeros(tokens * width + 8, device="cuda")
        self.host = rng.standard_normal((tokens, width)).astype(np.float32) * 3
        self.buf[offset:offset + tokens * width] = torch.from_numpy(self.host.reshape(-1))
        self.seqs = 3 if tokens > 4 else 1
        self.sequence = np.sort(rng.integers(0, self.seqs, tokens)).astype(np.int32)
        self.index = np.zeros(tokens, np.int32)
        for s in range(self.seqs):
            at = self.sequence == s
            self.index[at] = np.arange(at.sum()) + 5 * s  # the first places of later sequences stay as they were
        per = (int(self.index.max()) + page) // page
        self.pages = self.seqs * per + 2
        self.table = rng.permutation(self.pages)[:self.seqs * per].astype(np.int32).reshape(self.seqs, per)
        self.position = self.index + start
        self.dtype, self.page, self.eps = dtype, page, 1e-5
        self.k0 = torch.randn(self.pages, hkv, page, d, device="cuda").to(torch_dtype(dtype))
        self.v0 = torch.randn(self.pages, hkv, page, d, device="cuda").to(torch_dtype(dtype))
        self.k, self.v = self.k0.clone(), self.v0.clone()
        self.gq = rng.standard_normal(d).astype(np.float32) if norm else None
        self.gk = rng.standard_normal(d).astype(np.float32) if norm else None
        self.cache = nne.PagedKvCache(ctx, self.pages, page, hkv, d, dtype, self.k.data_ptr(), self.v.data_ptr(), rope_dims=dims,
                                      rope_interleaved=pairs, rope_base=10000.0, rope_freq=freq)
        self.dims, self.pairs = dims, pairs
        self.freq = 10000.0 ** (-2.0 * np.arange(dims // 2) / dims) if freq is None else np.asarray(freq) if dims else None
        self.q_out = torch.full((tokens, hq, d), 9.0, device="cuda")
        self.dev = {n: torch.from_numpy(getattr(self, n)).cuda() for n in ("sequence", "index", "position", "table")}
        self.g = [torch.from_numpy(g).cuda() if g is not None else None for g in (self.gq, self.gk)]
        at = self.buf.data_ptr() + 4 * offset
        self.call = nne.KvAppend(
            self.cache, tokens=tokens, q_heads=hq, q=at if hq else 0, k=at + 4 * hq * d, v=at + 4 * (hq + hkv) * d,
            q_out=self.q_out.data_ptr() if hq else 0, q_stride=width, k_stride=width, v_stride=width,
            q_gamma=self.g[0].data_ptr() if norm else 0, k_gamma=self.g[1].data_ptr() if norm else 0, eps=self.eps,
            page_table=self.dev["table"].data_ptr(), table_stride=per, sequences=self.seqs, sequence=self.dev["sequence"].data_ptr(),
            index=self.dev["index"].data_ptr(), position=self.dev["position"].data_ptr())

    def check(self, stored=None):
        """Everything against the definition; `stored`: which tokens' keys and values are there (all)."""
        tokens, hq, hkv, d = self.shape
        rows = self.host[:, :(hq + 2 * hkv) * d].reshape(tokens, -1, d)
        unit = 2.0 ** -25 + 2 * 2.0 ** -23 + 3 * 2.0 ** -24 + ((d / 8 + 8) * 2.0 ** -24 if self.gq is not None else 0.0)
        turn = (self.eps, self.position, self.dims, self.pairs, self.freq)
        stored = np.ones(tokens, bool) if stored is None else stored
        if hq:
            want, mag = head_exact(rows[:, :hq], self.gq, *turn)
            got = self.q_out.cpu().numpy()
            live = self.index >= 0
            assert np.all(np.abs(got - want)[live] <= (mag * unit)[live])
            assert np.all(got[~live] == 9.0)
        want, mag = head_exact(rows[:, hq:hq + hkv], self.gk, *turn)
        kp, vp = self.k0.double().cpu().numpy(), self.v0.double().cpu().numpy()
        kb, vb = np.zeros_like(kp), np.zeros_like(vp)
        for t in np.nonzero(stored)[0]:
            at = self.table[self.sequence[t], self.index[t] // self.page]
            o = self.index[t] % self.page
            kp[at, :, o], vp[at, :, o] = want[t], rows[t, hq + hkv:]
            kb[at, :, o] = mag[t] * unit * 2 + np.abs(want[t]) * STEP[self.dtype] + 2.0 ** -25
            vb[at, :, o] = np.abs(rows[t, hq + hkv:]) * STEP[self.dtype] + 2.0 ** -25
        assert np.all(np.abs(self.k.double().cpu().numpy() - kp) <= kb)
        assert np.all(np.abs(self.v.double().cpu().numpy() - vp) <= vb)


def now():
    import torch
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,hq,hkv,d,dims,pairs,norm,page,start", [
    (1, 1, 1, 64, 64, False, True, 8, 0), (1, 32, 8, 128, 128, False, True, 64, 4000), (7, 12, 3, 96, 96, True, False, 16, 1),
    (5, 8, 8, 256, 256, False, True, 32, 130000), (300, 4, 2, 128, 64, True, True, 16, 70000), (33, 16, 1, 64, 32, False, False, 128, 2 ** 20),
    (9, 3, 1, 256, 128, True, True, 8, 17), (40, 6, 2, 96, 40, False, True, 1024, 999999), (500, 0, 4, 128, 128, True, True, 16, 3),
    (20, 4, 4, 128, 0, False, True, 16, 0)])
def test_append(nne, ctx, dtype, tokens, hq, hkv, d, dims, pairs, norm, page, start):
    s = Setup(nne, ctx, tokens, hq, hkv, d, dims, pairs, norm, dtype, page, start)
    s.call.run(now())
    s.check()


@pytest.mark.parametrize("offset,gap", [(1, 0), (0, 3), (2, 5), (4, 64)])
@pytest.mark.parametrize("d", [64, 256])
def test_unaligned_rows(nne, ctx, offset, gap, d):
    s = Setup(nne, ctx, 11, 4, 2, d, d, False, True, "bf16", 16, 55, offset, gap)
    s.call.run(now())
    s.check()


def test_given_frequencies(nne, ctx):
    freq = np.concatenate([np.ones(8), np.linspace(0.5, 1e-4, 24)])
    s = Setup(nne, ctx, 20, 4, 2, 128, 64, False, False, "f16", 16, 5000, freq=freq)
    s.call.run(now())
    s.check()


def test_padding_and_places_that_do_not_exist(nne, ctx):
    """Padded tokens, sequences and places outside the table, pages outside the pool: nothing is written for them."""
    import torch
    s = Setup(nne, ctx, 30, 4, 2, 128, 128, False, True, "bf16", 8, 100)
    stored = np.ones(30, bool)
    for t in (0, 7, 29):
        s.index[t], stored[t] = -1, False
    index = s.index.copy()
    index[3] = 2 ** 30                                   # behind the table's row
    sequence = s.sequence.copy()
    sequence[5], sequence[6] = -1, s.seqs                # no such sequence
    stored[[3, 5, 6]] = False
    table = s.table.copy()
    bad = [(s.sequence[10], s.index[10] // 8, s.pages), (s.sequence[20], s.index[20] // 8, -1), (s.sequence[25], s.index[25] // 8, 2 ** 30)]
    for b, slot, value in bad:
        table[b, slot] = value
        stored &= ~((s.sequence == b) & (s.index // 8 == slot))
    s.dev["index"].copy_(torch.from_numpy(index))
    s.dev["sequence"].copy_(torch.from_numpy(sequence))
    s.dev["table"].copy_(torch.from_numpy(table))
    s.call.run(now())
    s.check(stored)


def test_parts_of_the_step(nne, ctx):
    """Queries alone (in place, without places), keys and values alone, positions by the places."""
    import torch
    q = torch.randn(6, 4, 64, device="cuda")
    host = q.cpu().numpy()
    cache = nne.PagedKvCache(ctx, 4, 16, 2, 64, "f16", rope_dims=64)
    pos = torch.tensor([0, 1, 5, 100, 1000, 70000], device="cuda", dtype=torch.int32)
    nne.KvAppend(cache, 6, 4, q=q.data_ptr(), q_out=q.data_ptr(), position=pos.data_ptr()).run(now())
    freq = 10000.0 ** (-2.0 * np.arange(32) / 64)
    want, mag = head_exact(host, None, 0, pos.cpu().numpy(), 64, False, freq)
    assert np.all(np.abs(q.cpu().numpy() - want) <= mag * 2.0 ** -21)
    kv = torch.randn(2, 3, 2, 64, device="cuda")
    table, seq = torch.tensor([[3, 1]], device="cuda", dtype=torch.int32), torch.zeros(3, device="cuda", dtype=torch.int32)
    idx = torch.tensor([0, 17, 31], device="cuda", dtype=torch.int32)
    nne.KvAppend(cache, 3, k=kv[0].data_ptr(), v=kv[1].data_ptr(), page_table=table.data_ptr(), table_stride=2, sequences=1,
                 sequence=seq.data_ptr(), index=idx.data_ptr()).run(now())
    want, mag = head_exact(kv[0].cpu().numpy(), None, 0, idx.cpu().numpy(), 64, False, freq)
    kp, vp, n = cache.pools()
    assert n == 4 * 2 * 16 * 64 * 2
    pool = np.zeros(n // 2, np.float16)
    assert nne.load().nne_device_download(ctx.handle, pool.ctypes.data_as(C.c_void_p), kp, n) == 0
    pool = pool.reshape(4, 2, 16, 64).astype(np.float64)
    for t, (page, o) in enumerate([(3, 0), (1, 1), (1, 15)]):
        assert np.all(np.abs(pool[page, :, o] - want[t]) <= np.abs(want[t]) * 2.0 ** -11 + mag[t] * 2.0 ** -20 + 2.0 ** -25)
        pool[page, :, o] = 0
    assert not pool.any()  # the rest is as it was created


def test_another_stream_and_a_captured_call(nne, ctx):
    import torch
    s = Setup(nne, ctx, 16, 8, 2, 128, 128, False, True, "bf16", 16, 9)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        s.call.run(st.cuda_stream)
    assert torch.equal(s.k, s.k0)
    g.replay()
    torch.cuda.synchronize()
    s.check()
    s.position += 1000
    s.dev["position"].copy_(torch.from_numpy(s.position))
    s.k.copy_(s.k0)
    g.replay()
    torch.cuda.synchronize()
    s.check()


def test_refusals(nne, ctx):
    ok = dict(pages=4, page_size=16, kv_heads=2, head_dim=64, dtype="f16")
    for change in (dict(head_dim=80), dict(page_size=12), dict(page_size=4), dict(page_size=2048), dict(kv_heads=0), dict(rope_dims=12),
                   dict(rope_dims=72), dict(rope_dims=64, rope_base=-1.0), dict(k_pages=16), dict(k_pages=8, v_pages=8),
                   dict(pages=2 ** 27), dict(dtype="f32"), dict(rope_dims=64, rope_freq=[1.0])):
        with pytest.raises(nne.InvalidArgument):
            nne.PagedKvCache(ctx, **{**ok, **change})
    c = nne.PagedKvCache(ctx, **ok, rope_dims=64)
    good = dict(tokens=2, q_heads=4, q=16, q_out=16, k=16, v=16, page_table=16, table_stride=1, sequences=1, sequence=16, index=16)
    for change in (dict(v=0), dict(q_out=0), dict(q_heads=0), dict(q_stride=100), dict(k_stride=64), dict(page_table=0), dict(index=0),
                   dict(sequence=0), dict(table_stride=0), dict(q=18), dict(tokens=2 ** 32), dict(index=17), dict(page_table=18), dict(q_gamma=18),
                   dict(position=19)):
        with pytest.raises(nne.InvalidArgument):
            nne.KvAppend(c, **{**good, **change}).run()
    nne.KvAppend(c, **{**good, "tokens": 0}).run()
    c.close()
    with pytest.raises(nne.GpuError):
        nne.KvAppend.run(nne.KvAppend(c, **good))
