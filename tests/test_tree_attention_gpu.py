"""Tree attention over the paged cache on the device against the definition in 64 bits.

Bound, per element, in units of A = sum p |v| (p the probabilities).  A score is a dot product of D f32-like products
summed by D / 16 MMAs in three chains: off by at most (D / 16 + 8) * 2^-22 of M = scale * sum |q k| (the unit may truncate;
q's parts 2^-22; scale * log2 e and its product with q 2^-23), and its exp2 argument by 2^-23 of its size beside that; a
probability is off by that times ln 2 * log2 e = 1 plus 2^-22 (exp2).  It enters numerator and denominator: twice.  P's parts: 2^-21.  The
sums over keys: within a tile at most 64 / 16 * 3 + 2 steps of 2^-23, then one f32 step a tile of 64 keys in a CTA, joins of 4
warps and 16 CTAs."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def now():
    import torch
    return torch.cuda.current_stream().cuda_stream


class Setup:
    """Sequences of given contexts and node counts; `visible`: "tree", "chain" (None passed) or a list of masks."""

    def __init__(self, nne, ctx, contexts, nodes, hq, hkv, d, dtype, page, visible="tree", gap=0, behind=0, seed=0, spread=1.0, max_nodes=None):
        import torch
        g = torch.Generator(device="cuda")
        g.manual_seed(seed + hq * d)
        rng = np.random.default_rng(seed)
        self.contexts, self.nodes, self.hq, self.hkv, self.d, self.page = contexts, nodes, hq, hkv, d, page
        per = [max(1, -(-(c + n) // page)) for c, n in zip(contexts, nodes)]
        self.pages = sum(per) + 2
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(per), max(per)), -7, np.int32)
        at = 0
        for b, n in enumerate(per):
            self.table[b, :n] = order[at:at + n]
            at += n
        dt = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
        # places that no sequence has hold NaN: nothing may read them
        self.k = torch.full((self.pages, hkv, page, d), float("nan"), device="cuda", dtype=dt)
        self.v = self.k.clone()
        for b, (c, n) in enumerate(zip(contexts, nodes)):
            i = np.arange(c + n)
            p, o = torch.from_numpy(self.table[b, i // page].astype(np.int64)).cuda(), torch.from_numpy(i % page).cuda()
            self.k[p, :, o] = torch.randn(c + n, hkv, d, device="cuda", generator=g).to(dt)
            self.v[p, :, o] = torch.randn(c + n, hkv, d, device="cuda", generator=g).to(dt)
        self.start = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
        self.tokens = int(self.start[-1]) + behind
        self.width = hq * d + gap
        self.q = torch.randn(self.tokens, self.width, device="cuda", generator=g) * spread
        self.out = torch.full((self.tokens, self.width), 5.0, device="cuda")
        masks = []
        for n in nodes:
            rows = []
            for i in range(n):
                parent = int(rng.integers(0, i)) if i else -1
                rows.append((rows[parent] if i else 0) | 1 << i)
            masks += rows
        if visible == "chain":
            masks = [(2 << i) - 1 for n in nodes for i in range(n)]
        elif visible != "tree":
            masks = list(visible)
        self.masks = masks
        self.dev = [torch.from_numpy(x).cuda() for x in (self.table, self.start, np.array(contexts, np.int32))]
        bits = np.array([m & (2 ** 64 - 1) for m in masks] + [0] * behind, np.uint64).view(np.int64)
        self.vis = None if visible == "chain" else torch.from_numpy(bits).cuda()
        self.scale = d ** -0.5
        self.cache = nne.PagedKvCache(ctx, self.pages, page, hkv, d, dtype, self.k.data_ptr(), self.v.data_ptr())
        self.call = nne.TreeAttention(
            self.cache, self.tokens, hq, self.q.data_ptr(), self.out.data_ptr(), len(nodes), self.dev[1].data_ptr(), self.dev[2].data_ptr(),
            self.dev[0].data_ptr(), self.table.shape[1], max(nodes) if max_nodes is None else max_nodes, max(contexts),
            0 if self.vis is None else self.vis.data_ptr(), None, self.width, self.width)

    def exact(self):
        """(out, bound) [tokens, hq, d] in 64 bits; a row that sees nothing is 0."""
        import torch
        hq, hkv, d, group = self.hq, self.hkv, self.d, self.hq // self.hkv
        out = torch.zeros(self.tokens, hq, d, device="cuda", dtype=torch.float64)
        bound = out.clone()
        for b, (c, n) in enumerate(zip(self.contexts, self.nodes)):
            i = np.arange(c + n)
            p, o = torch.from_numpy(self.table[b, i // self.page].astype(np.int64)).cuda(), torch.from_numpy(i % self.page).cuda()
            keys, values = self.k[p, :, o].double(), self.v[p, :, o].double()  # [length, hkv, d]
            for r in range(n):
                row = int(self.start[b]) + r
                see = torch.tensor([j < c or bool(self.masks[row] >> (j - c) & 1) for j in range(c + n)], device="cuda")
                if not bool(see.any()):
                    continue
                q = self.q[row, :hq * d].view(hq, d).double()
                k, v = keys[see].repeat_interleave(group, 1), values[see].repeat_interleave(group, 1)
                s = torch.einsum("hd,lhd->hl", q, k) * self.scale
                w = torch.softmax(s, dim=1)
                out[row] = torch.einsum("hl,lhd->hd", w, v)
                big = torch.einsum("hd,lhd->hl", q.abs(), k.abs()) * self.scale
                ds = big * (d / 16 + 8) * 2.0 ** -22 + (s.abs() + s.abs().amax(dim=1, keepdim=True)) * 2.0 ** -22 + 2.0 ** -22
                steps = 2.0 ** -21 + (14 + (c + n) / 64 + 24) * 2.0 ** -23
                bound[row] = torch.einsum("hl,lhd->hd", w * (2 * ds.amax(dim=1, keepdim=True) + 2 * steps), v.abs())
        return out, bound

    def got(self):
        return self.out[:, :self.hq * self.d].view(self.tokens, self.hq, self.d)

    def check(self):
        import torch
        self.call.run(now())
        want, bound = self.exact()
        live = int(self.start[-1])
        far = (self.got()[:live].double() - want[:live]).abs()
        assert bool((far <= bound[:live] + 1e-30).all()), float((far / (bound[:live] + 1e-30)).nan_to_num(nan=9e9).max())
        assert bool((self.out[live:] == 5.0).all()) and bool((self.out[:, self.hq * self.d:] == 5.0).all())
        first = self.out.clone()
        self.call.run(now())
        assert torch.equal(first, self.out)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("contexts,nodes,hq,hkv,d,page", [
    ([0], [1], 1, 1, 64, 8), ([1], [1], 4, 1, 128, 16), ([63], [1], 8, 8, 128, 64), ([64], [1], 32, 8, 128, 32), ([500, 1, 77], [1, 1, 1], 8, 2, 96, 16),
    ([5000], [1], 8, 2, 128, 64), ([3000], [1], 4, 1, 256, 1024), ([200, 9], [7, 3], 4, 2, 256, 8), ([1000], [16], 2, 2, 64, 16),
    ([333, 40], [4, 2], 16, 4, 128, 8), ([130, 700, 0], [33, 7, 64], 8, 2, 128, 16), ([2000], [64], 8, 1, 64, 128), ([90], [40], 8, 1, 96, 32),
    ([100], [20], 4, 1, 256, 16), ([17], [30], 1, 1, 128, 8), ([61, 62, 63, 64, 65], [5, 5, 5, 5, 5], 4, 4, 64, 64)])
def test_trees(nne, ctx, dtype, contexts, nodes, hq, hkv, d, page):
    Setup(nne, ctx, contexts, nodes, hq, hkv, d, dtype, page, seed=len(contexts) + hq).check()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
def test_long_contexts_split_over_a_cluster(nne, ctx, dtype, d):
    Setup(nne, ctx, [20011], [3], 4, 1, d, dtype, 64, seed=5).check()


@pytest.mark.parametrize("gap,behind", [(0, 3), (1, 0), (4, 2)])
def test_chains_strides_and_rows_behind(nne, ctx, gap, behind):
    Setup(nne, ctx, [70, 10], [6, 64], 8, 2, 64, "bf16", 16, "chain", gap, behind).check()


def test_steep_and_flat_scores(nne, ctx):
    """Scores far apart (one key takes nearly all) and all equal (queries of zeros)."""
    Setup(nne, ctx, [300, 100], [5, 3], 4, 2, 128, "f16", 16, spread=40.0).check()
    Setup(nne, ctx, [300, 100], [5, 3], 4, 2, 128, "bf16", 16, spread=40.0).check()
    Setup(nne, ctx, [300], [5], 4, 2, 128, "f16", 16, spread=0.0).check()
    Setup(nne, ctx, [300], [5], 4, 2, 128, "f16", 16, spread=1e-20).check()


def test_rows_that_see_nothing(nne, ctx):
    s = Setup(nne, ctx, [0, 0], [4, 3], 8, 2, 128, "bf16", 16, [0, 1, 0, 0b1111, 0b100, 0, 1])
    s.check()
    got = s.got()
    assert bool((got[[0, 2, 5]] == 0).all()) and bool(got[[1, 3, 4, 6]].any(dim=2).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("d,nodes", [(128, 9), (64, 40), (256, 5)])
def test_what_a_row_does_not_see_does_not_reach_it(nne, ctx, dtype, bad, d, nodes):
    """A drafted node whose key and value are not finite: rows that see it are not finite, all others exactly as they
    were with ordinary numbers in its place."""
    s = Setup(nne, ctx, [100], [nodes], 8, 2, d, dtype, 16, seed=3)
    s.check()
    clean = s.got().clone()
    sees = np.array([bool(m >> 2 & 1) for m in s.masks])
    page, o = int(s.table[0, 102 // 16]), 102 % 16
    s.v[page, :, o, :5] = bad
    s.call.run(now())
    got = s.got().cpu().numpy()
    assert np.array_equal(got[~sees], clean.cpu().numpy()[~sees])
    assert not np.isfinite(got[sees][:, :, :5]).any()
    far = np.abs(got[sees][:, :, 5:] - clean.cpu().numpy()[sees][:, :, 5:])
    assert np.all(far <= 1e-5 * np.abs(clean.cpu().numpy()).max())
    s.k[page, :, o] = bad
    s.call.run(now())
    got = s.got().cpu().numpy()
    assert np.array_equal(got[~sees], clean.cpu().numpy()[~sees])
    assert np.isnan(got[sees]).all() or not np.isnan(bad)


def test_a_row_of_nan_stays_alone(nne, ctx):
    s = Setup(nne, ctx, [100], [9], 8, 2, 128, "f16", 16, seed=3)
    s.call.run(now())
    clean = s.got().clone()
    s.q[4, 7] = float("nan")          # head 0 of node 4
    s.call.run(now())
    got = s.got()
    assert bool(got[4, 0].isnan().all())
    keep = [i for i in range(9) if i != 4]
    import torch
    assert torch.equal(got[keep], clean[keep]) and torch.equal(got[4, 1:], clean[4, 1:])


def test_places_without_a_page_are_seen_by_nobody(nne, ctx):
    import torch
    s = Setup(nne, ctx, [100, 60], [3, 2], 4, 2, 64, "bf16", 16, "chain", seed=11)
    table = s.table.copy()
    table[0, 2], table[0, 4], table[1, 0] = -1, s.pages, 2 ** 30
    s.dev[0].copy_(torch.from_numpy(table))
    s.call.run(now())
    got = s.got().double()
    for b, gone in ((0, [2, 4]), (1, [0])):
        c, n = s.contexts[b], s.nodes[b]
        for r in range(n):
            keep = [i for i in range(c + r + 1) if i // 16 not in gone]
            p, o = torch.tensor(s.table[b][[i // 16 for i in keep]].astype(np.int64)).cuda(), torch.tensor([i % 16 for i in keep]).cuda()
            k, v = s.k[p, :, o].double().repeat_interleave(2, 1), s.v[p, :, o].double().repeat_interleave(2, 1)
            q = s.q[s.start[b] + r].view(4, 64).double()
            w = torch.softmax(torch.einsum("hd,lhd->hl", q, k) * s.scale, dim=1)
            want = torch.einsum("hl,lhd->hd", w, v)
            assert bool(((got[s.start[b] + r] - want).abs() <= 1e-5).all())


def test_nodes_above_the_bound_and_odd_tables(nne, ctx):
    """max_nodes below a sequence's nodes: the rows beyond are not written.  Contexts longer than the table: its places
    are all there is."""
    s = Setup(nne, ctx, [50], [12], 4, 1, 128, "f16", 16, "chain", max_nodes=8, seed=2)
    s.call.run(now())
    want, bound = s.exact()
    # the last four nodes' keys are not counted either, and no row sees a later node in a chain
    assert bool(((s.got()[:8].double() - want[:8]).abs() <= bound[:8]).all()) and bool((s.out[8:] == 5.0).all())
    t = Setup(nne, ctx, [64], [0], 4, 1, 128, "f16", 16, "chain", behind=1, max_nodes=4)
    t.call.run(now())
    assert bool((t.out == 5.0).all())
    u = Setup(nne, ctx, [60], [4], 4, 1, 128, "f16", 16, "chain", seed=8)
    import torch
    u.dev[2].copy_(torch.tensor([2 ** 31 - 5], dtype=torch.int32))
    u.call.run(now())
    assert bool(u.got().isfinite().all())


def test_captured_beside_another_stream(nne, ctx):
    """A captured call replayed while eager calls of another setup run on another stream."""
    import torch
    a, b = (Setup(nne, ctx, [900], [5], 8, 2, 128, t, 16, seed=i) for i, t in enumerate(("bf16", "f16")))
    a.check(), b.check()
    want_a, want_b = a.out.clone(), b.out.clone()
    st, other = torch.cuda.Stream(), torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream()), other.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        a.call.run(st.cuda_stream)
    a.out.fill_(0), b.out.fill_(0)
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(st):
            g.replay()
        b.call.run(other.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(a.out, want_a) and torch.equal(b.out, want_b)


def test_refusals(nne, ctx):
    c = nne.PagedKvCache(ctx, 4, 16, 2, 64, "f16")
    good = dict(tokens=2, q_heads=4, q=16, out=16, sequences=1, node_start=16, context=16, page_table=16, table_stride=1, max_nodes=2,
                max_context=10)
    for change in (dict(q_heads=3), dict(q_heads=0), dict(max_nodes=65), dict(max_nodes=-1), dict(q_stride=100), dict(out_stride=64), dict(q=0),
                   dict(out=0), dict(node_start=0), dict(context=0), dict(page_table=0), dict(table_stride=0), dict(scale=float("nan")),
                   dict(visible=12), dict(q=18), dict(context=18), dict(page_table=17), dict(node_start=19), dict(tokens=2 ** 31), dict(max_context=-1), dict(sequences=-1)):
        with pytest.raises(nne.InvalidArgument):
            nne.TreeAttention(c, **{**good, **change}).run()
    for change in (dict(tokens=0), dict(sequences=0), dict(max_nodes=0)):
        nne.TreeAttention(c, **{**good, **change}).run()
