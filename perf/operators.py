"""The decode-step operators beside QLinear: plain forms, inputs and sizes for measuring them.

Four operators, in the order a decode step meets them:
  q4       forward of a linear layer with 4-bit weights and one f32 scale a group of inputs
  quant4   the quantizer of such a layer
  append   per-head RMSNorm of queries and keys, rotation by position, keys and values into a paged cache
  tree     attention of a tree of drafted tokens (one node: ordinary decoding) over the paged cache
  sample   temperature, top-k, top-p and min-p sampling from given uniform numbers
"""
import importlib
import math

import torch

own = False

PACKAGE = "neural-network-engine_b200"


# ---- cases ----------------------------------------------------------------------------------------------

def listed():
    return [
        # one token through an attention projection of a 7B-shaped stack: the smallest layer, latency counts
        dict(name="q4 4096x4096 m1 g128", op="q4", n=4096, k=4096, m=1, group=128, bias=False),
        # one token through the down projection of a 70B-shaped FFN: the longest rows
        dict(name="q4 8192x28672 m1 g64", op="q4", n=8192, k=28672, m=1, group=64, bias=False),
        # a batch of sequences at once, ragged sizes, the smallest group, with a bias
        dict(name="q4 11003x4091 m12 g32", op="q4", n=11003, k=4091, m=12, group=32, bias=True),
        # quantizing an FFN matrix at load time
        dict(name="quant4 11008x4096 g64", op="quant4", n=11008, k=4096, group=64),
        # the same for a small ragged layer: latency counts
        dict(name="quant4 257x1001 g32", op="quant4", n=257, k=1001, group=32),
        # one decode step of eight sequences, normed heads: latency counts
        dict(name="append 8 tokens bf16", op="append", tokens=8, seqs=8, hq=32, hkv=8, d=128, dims=128, pairs=False,
             norm=True, dtype="bf16", page=64, start=4000),
        # a long prompt's chunk at far positions, pairs rotated, packed q/k/v rows
        dict(name="append 6001 tokens f16", op="append", tokens=6001, seqs=3, hq=32, hkv=8, d=128, dims=128,
             pairs=True, norm=False, dtype="f16", page=16, start=120000),
        # ordinary decoding of one long sequence: the work has to be split over the context
        dict(name="tree 1x1 ctx 16001 bf16", op="tree", seqs=1, nodes=1, ctx=16001, hq=32, hkv=8, d=128, dtype="bf16", page=64),
        # ordinary decoding of a batch of unlike lengths
        dict(name="tree 24x1 ctx 8192 f16", op="tree", seqs=24, nodes=1, ctx=8192, hq=32, hkv=8, d=128, dtype="f16", page=32),
        # drafted trees of a few sequences
        dict(name="tree 4x33 ctx 3000 bf16", op="tree", seqs=4, nodes=33, ctx=3000, hq=32, hkv=8, d=128, dtype="bf16", page=16),
        # one row of logits of a 7B-shaped model's vocabulary: latency counts
        dict(name="sample 1x32000", op="sample", rows=1, vocab=32000, top_k=50, mixed=False),
        # a batch over a large vocabulary, every row with settings of its own
        dict(name="sample 64x128000", op="sample", rows=64, vocab=128000, top_k=0, mixed=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["q4", "q4", "quant4", "append", "append", "tree", "tree", "tree", "sample", "sample"])
    if op == "q4":
        n, m = _log(rng, 64, 28672), rng.choice([1, 1, 2, 3, 4, 7, 8, 16, 21, 48, 64])
        k = _log(rng, 64, min(28672, 8192 * 28672 // n, (14 << 30) // (n * m)))
        return dict(op=op, n=n, k=k, m=m, group=rng.choice([32, 64, 128]),
                    bias=rng.random() < 0.5)
    if op == "quant4":
        return dict(op=op, n=_log(rng, 64, 11008), k=_log(rng, 64, 8192), group=rng.choice([32, 64, 128]))
    if op == "append":
        hkv = rng.choice([1, 2, 4, 8])
        d = rng.choice([64, 96, 128, 256])
        return dict(op=op, tokens=_log(rng, 1, 6000) + 3, seqs=rng.choice([1, 2, 3]), hq=hkv * rng.choice([1, 4, 8] if hkv < 8 else [1, 4]),
                    hkv=hkv, d=d, dims=rng.choice([d, d, d // 2]), pairs=rng.random() < 0.5, norm=rng.random() < 0.5,
                    dtype=rng.choice(["bf16", "f16"]), page=rng.choice([16, 32, 64, 128]), start=_log(rng, 1, 130000))
    if op == "tree":
        hkv, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 96, 128, 256])
        seqs, nodes = rng.choice([1, 1, 2, 3, 5, 8]), rng.choice([1, 1, 2, 7, 16, 33, 64])
        hq = hkv * rng.choice([1, 4, 8] if hkv < 8 else [1, 4])
        longest = min(131072, (1 << 28) // (4 * hkv * d * seqs), 7000000000 // (nodes * hq * d * seqs))
        return dict(op=op, seqs=seqs, nodes=nodes, ctx=_log(rng, 16, longest), hq=hq, hkv=hkv, d=d, dtype=rng.choice(["bf16", "f16"]), page=rng.choice([16, 32, 64, 128]))
    return dict(op=op, rows=_log(rng, 1, 64), vocab=_log(rng, 1000, 152000), top_k=rng.choice([0, 1, 5, 50, 400]),
                mixed=rng.random() < 0.5)


# ---- inputs -----------------------------------------------------------------------------------------------

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=g)


def _quant4_plain(w, group):
    """Codes -8..7 (int8, [n, k]) and scales [n, ceil(k / group)]: scale = max|w| / 7 (1 where that is 0),
    code = w / scale by way of the f32 reciprocal, halves away from zero."""
    n, k = w.shape
    groups = -(-k // group)
    padded = torch.zeros(n, groups * group, device=w.device, dtype=torch.float32)
    padded[:, :k] = w
    v = padded.view(n, groups, group)
    top = v.abs().amax(dim=2)
    scales = torch.where(top > 0, top / torch.full_like(top, 7.0), torch.ones_like(top))  # by a tensor: IEEE division
    t = (v * (1.0 / scales)[:, :, None]).double()  # 64 bits: the halves are a border
    codes = (torch.sign(t) * torch.floor(t.abs() + 0.5)).clamp(-8, 7).to(torch.int8)
    return codes.view(n, groups * group)[:, :k].contiguous(), scales


def _pack4(codes):
    """[n, k] codes as bytes [n, ceil(k / 2)], two's complement, the even column in the low four bits."""
    n, k = codes.shape
    c = torch.zeros(n, k + (k & 1), device=codes.device, dtype=torch.int32)
    c[:, :k] = codes
    c &= 15
    return (c[:, 0::2] | (c[:, 1::2] << 4)).to(torch.uint8)


def _unpack4(packed, k):
    b = packed.to(torch.int32)
    c = torch.stack([b & 15, b >> 4], dim=2).view(b.shape[0], -1)[:, :k]
    return c - 16 * (c >= 8).to(torch.int32)


def _pages_for(g, lengths, page):
    """A page table for sequences of these lengths, pages handed out in a shuffled order, two spare pages left."""
    per = [max(1, -(-n // page)) for n in lengths]
    total, width = sum(per) + 2, max(per)
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(len(lengths), width, device="cuda", dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def _ragged(most, seqs, step):
    return [max(1, most - (most // 2) * (b * step % 8) // 7) for b in range(seqs)]


def prepare(case, seed):
    return {"q4": _prepare_q4, "quant4": _prepare_quant4, "append": _prepare_append, "tree": _prepare_tree,
            "sample": _prepare_sample}[case["op"]](case, seed)


def _context():
    nne = importlib.import_module(PACKAGE)
    return nne, nne.default_context(torch.cuda.current_device()), torch.cuda.current_stream().cuda_stream


def _prepare_q4(case, seed):
    g = _generator(seed)
    n, k, m, group = case["n"], case["k"], case["m"], case["group"]
    codes, scales = _quant4_plain(_normal(g, n, k) * 0.02, group)
    s = dict(op="q4", k=k, group=group, packed=_pack4(codes), scales=scales, x=_normal(g, m, k),
             bias=_normal(g, n) * 0.1 if case["bias"] else None)
    if own:
        nne, ctx, stream = _context()
        s["layer"] = nne.QLinear4.from_packed_device(ctx, s["packed"].data_ptr(), scales.data_ptr(),
                                                     s["bias"].data_ptr() if case["bias"] else 0, n, k, group, stream)
        s["y"] = torch.empty(m, n, device="cuda", dtype=torch.float32)
        s["stream"] = stream
    return s


def _prepare_quant4(case, seed):
    g = _generator(seed)
    n, k, group = case["n"], case["k"], case["group"]
    s = dict(op="quant4", w=_normal(g, n, k) * 0.02, group=group)
    if own:
        nne, ctx, stream = _context()
        s["packed"] = torch.empty(n, (k + 1) // 2, device="cuda", dtype=torch.uint8)
        s["scales"] = torch.empty(n, -(-k // group), device="cuda", dtype=torch.float32)
        s["call"], s["ctx"], s["stream"] = nne.quantize_rows4_device, ctx, stream
    return s


def _prepare_append(case, seed):
    g = _generator(seed)
    tokens, seqs, hq, hkv, d = case["tokens"], min(case["seqs"], case["tokens"]), case["hq"], case["hkv"], case["d"]
    dt = DTYPES[case["dtype"]]
    share = [tokens // seqs + (1 if b < tokens % seqs else 0) for b in range(seqs)]
    table, pages = _pages_for(g, share, case["page"])
    sequence = torch.cat([torch.full((n,), b, device="cuda", dtype=torch.int32) for b, n in enumerate(share)])
    index = torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in share])
    s = dict(op="append", qkv=_normal(g, tokens, (hq + 2 * hkv) * d), hq=hq, hkv=hkv, d=d, dims=case["dims"], pairs=case["pairs"],
             q_gamma=1 + 0.1 * _normal(g, d) if case["norm"] else None, k_gamma=1 + 0.1 * _normal(g, d) if case["norm"] else None,
             eps=1e-6, base=10000.0, page=case["page"], table=table, sequence=sequence, index=index,
             position=index + case["start"],
             k_pages=_normal(g, pages, hkv, case["page"], d).to(dt), v_pages=_normal(g, pages, hkv, case["page"], d).to(dt))
    if own:
        nne, ctx, stream = _context()
        s["q_out"] = torch.empty(tokens, hq, d, device="cuda", dtype=torch.float32)
        at, row = s["qkv"].data_ptr(), (hq + 2 * hkv) * d
        s["cache"] = nne.PagedKvCache(ctx, pages, case["page"], hkv, d, case["dtype"], s["k_pages"].data_ptr(), s["v_pages"].data_ptr(),
                                      rope_dims=case["dims"], rope_interleaved=case["pairs"], rope_base=s["base"])
        s["call"] = nne.KvAppend(
            s["cache"], tokens=tokens, q_heads=hq, q=at, k=at + 4 * hq * d, v=at + 4 * (hq + hkv) * d, q_out=s["q_out"].data_ptr(),
            q_stride=row, k_stride=row, v_stride=row, q_gamma=s["q_gamma"].data_ptr() if case["norm"] else 0,
            k_gamma=s["k_gamma"].data_ptr() if case["norm"] else 0, eps=s["eps"], page_table=table.data_ptr(), sequences=seqs,
            table_stride=table.shape[1], sequence=sequence.data_ptr(), index=index.data_ptr(), position=s["position"].data_ptr())
        s["stream"] = stream
    return s


def _prepare_tree(case, seed):
    g = _generator(seed)
    seqs, most, hq, hkv, d, page = case["seqs"], case["nodes"], case["hq"], case["hkv"], case["d"], case["page"]
    dt = DTYPES[case["dtype"]]
    # the first sequence has the full context and tree, the others down to half of them
    ctx_len, nodes = _ragged(case["ctx"], seqs, 3), _ragged(most, seqs, 5)
    table, pages = _pages_for(g, [a + b for a, b in zip(ctx_len, nodes)], page)
    start = [0]
    for n in nodes:
        start.append(start[-1] + n)
    tokens = start[-1]
    # each node's parent is one of the nodes before it; a node sees its ancestors and itself
    r = torch.rand(tokens, device="cuda", generator=g).tolist()
    seen = []
    for b in range(seqs):
        own_rows = []
        for i in range(nodes[b]):
            parent = int(r[start[b] + i] * i) if i else -1
            own_rows.append((own_rows[parent] if i else 0) | (1 << i))
        seen += own_rows
    seen = [v - (1 << 64) if v >= 1 << 63 else v for v in seen]
    s = dict(op="tree", q=_normal(g, tokens, hq, d), hq=hq, hkv=hkv, d=d, page=page, table=table, scale=d ** -0.5,
             start=torch.tensor(start, device="cuda", dtype=torch.int32), context=torch.tensor(ctx_len, device="cuda", dtype=torch.int32),
             visible=torch.tensor(seen, device="cuda", dtype=torch.int64), seqs=seqs, most=most, longest=max(ctx_len),
             k_pages=_normal(g, pages, hkv, page, d).to(dt), v_pages=_normal(g, pages, hkv, page, d).to(dt))
    if own:
        nne, ctx, stream = _context()
        s["out"] = torch.empty(tokens, hq, d, device="cuda", dtype=torch.float32)
        s["cache"] = nne.PagedKvCache(ctx, pages, page, hkv, d, case["dtype"], s["k_pages"].data_ptr(), s["v_pages"].data_ptr())
        s["call"] = nne.TreeAttention(
            s["cache"], tokens=tokens, q_heads=hq, q=s["q"].data_ptr(), out=s["out"].data_ptr(), sequences=seqs,
            node_start=s["start"].data_ptr(), context=s["context"].data_ptr(), visible=s["visible"].data_ptr(),
            page_table=table.data_ptr(), table_stride=table.shape[1], max_nodes=most, max_context=max(ctx_len), scale=s["scale"])
        s["stream"] = stream
    return s


def _prepare_sample(case, seed):
    g = _generator(seed)
    rows, vocab = case["rows"], case["vocab"]
    # logits of a language model: a broad bulk, and a few tokens well above it
    logits = 2.0 * _normal(g, rows, vocab)
    top = torch.randint(0, vocab, (rows, 24), device="cuda", generator=g)
    logits.scatter_add_(1, top, 4.0 + 3.0 * _normal(g, rows, 24).abs())
    s = dict(op="sample", logits=logits, u=torch.rand(rows, device="cuda", dtype=torch.float32, generator=g))
    i = torch.arange(rows, device="cuda")
    if case["mixed"]:  # every request brings its own settings, some of them switched off
        s["temperature"] = torch.where(i % 7 == 6, 0.0, 0.6 + 0.9 * torch.rand(rows, device="cuda", generator=g)).float()
        s["top_k"] = torch.where(i % 3 == 0, 0, 1 + (i * 37) % 500).to(torch.int32)
        s["top_p"] = torch.where(i % 4 == 0, 1.0, 0.5 + 0.49 * torch.rand(rows, device="cuda", generator=g)).float()
        s["min_p"] = torch.where(i % 5 == 0, 0.02, 0.0).float()
    else:
        s["temperature"] = torch.full((rows,), 0.8, device="cuda")
        s["top_k"] = torch.full((rows,), case["top_k"], device="cuda", dtype=torch.int32)
        s["top_p"] = torch.full((rows,), 0.95, device="cuda")
        s["min_p"] = torch.zeros(rows, device="cuda")
    if own:
        nne, ctx, stream = _context()
        s["tokens"] = torch.empty(rows, device="cuda", dtype=torch.int32)
        s["call"] = nne.Sampler(ctx, rows=rows, vocab=vocab, logits=logits.data_ptr(), temperature=s["temperature"].data_ptr(),
                                top_k=s["top_k"].data_ptr(), top_p=s["top_p"].data_ptr(), min_p=s["min_p"].data_ptr(),
                                uniform=s["u"].data_ptr(), tokens=s["tokens"].data_ptr())
        s["stream"] = stream
    return s


# ---- one pass ---------------------------------------------------------------------------------------------

def run(state):
    return {"q4": _run_q4, "quant4": _run_quant4, "append": _run_append, "tree": _run_tree, "sample": _run_sample}[state["op"]](state)


def _run_q4(s):
    if own:
        s["layer"].forward_device(s["x"].data_ptr(), s["x"].shape[0], s["y"].data_ptr(), s["stream"])
        return s["y"]
    n, k = s["packed"].shape[0], s["k"]
    scale = s["scales"].repeat_interleave(s["group"], dim=1)[:, :k]
    y = s["x"] @ (_unpack4(s["packed"], k).float() * scale).t()
    return y if s["bias"] is None else y + s["bias"]


def _run_quant4(s):
    if own:
        w = s["w"]
        s["call"](s["ctx"], w.data_ptr(), w.shape[0], w.shape[1], s["group"], s["packed"].data_ptr(), s["scales"].data_ptr(), s["stream"])
        return dict(packed=s["packed"], scales=s["scales"])
    codes, scales = _quant4_plain(s["w"], s["group"])
    return dict(packed=_pack4(codes), scales=scales)


def _norm_rotate_plain(x, gamma, eps, position, dims, pairs, base):
    """[tokens, heads, d]: RMSNorm over d, then the first `dims` of each head rotated by position * base^(-2i/dims)."""
    if gamma is not None:
        x = x * torch.rsqrt((x * x).mean(dim=2, keepdim=True) + eps) * gamma
    half = dims // 2
    freq = base ** (-torch.arange(half, device=x.device, dtype=torch.float64) * 2 / dims)
    angle = position.double()[:, None] * freq  # 64 bits: far positions are many turns
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    if pairs:
        a, b = x[:, :, 0:dims:2], x[:, :, 1:dims:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=3).flatten(2)
    else:
        a, b = x[:, :, :half], x[:, :, half:dims]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=2)
    return torch.cat([turned, x[:, :, dims:]], dim=2)


def _run_append(s):
    if own:
        s["call"].run(s["stream"])
        return dict(q=s["q_out"], k_pages=s["k_pages"], v_pages=s["v_pages"])
    hq, hkv, d, page = s["hq"], s["hkv"], s["d"], s["page"]
    rows = s["qkv"].view(-1, hq + 2 * hkv, d)
    turn = (s["eps"], s["position"], s["dims"], s["pairs"], s["base"])
    q = _norm_rotate_plain(rows[:, :hq], s["q_gamma"], *turn)
    k = _norm_rotate_plain(rows[:, hq:hq + hkv], s["k_gamma"], *turn)
    index = s["index"].long()
    at = s["table"][s["sequence"].long(), index // page].long()
    s["k_pages"][at, :, index % page] = k.to(s["k_pages"].dtype)
    s["v_pages"][at, :, index % page] = rows[:, hq + hkv:].to(s["v_pages"].dtype)
    return dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"])


def _gathered(s):
    """The sequences' nodes and keys side by side, padded: q [b, hkv, nodes, group, d], keys and values
    [b, hkv, length, d], and which key a node sees [b, nodes, length]."""
    seqs, most, page, hq, hkv, d = s["seqs"], s["most"], s["page"], s["hq"], s["hkv"], s["d"]
    dev = s["q"].device
    node = torch.arange(most, device=dev)
    row = (s["start"][:-1, None] + node).long()
    there = node < (s["start"][1:] - s["start"][:-1])[:, None]
    row = row.clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].view(seqs, most, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4)
    table = s["table"].long()
    k = s["k_pages"][table].permute(0, 2, 1, 3, 4).reshape(seqs, hkv, -1, d)
    v = s["v_pages"][table].permute(0, 2, 1, 3, 4).reshape(seqs, hkv, -1, d)
    at = torch.arange(k.shape[2], device=dev)
    behind = at - s["context"][:, None]  # which node's key, from 0
    bit = (s["visible"][row][:, :, None] >> behind.clamp(0, 63)[:, None, :]) & 1
    see = (behind < 0)[:, None, :] | ((behind >= 0) & (behind < most))[:, None, :] & (bit == 1)
    return q, k, v, see & there[:, :, None], row[there], there


def _run_tree(s):
    if own:
        s["call"].run(s["stream"])
        return s["out"]
    q, k, v, see, row, there = _gathered(s)
    b, hkv, most, group, d = q.shape
    score = (q.reshape(b, hkv, most * group, d) @ k.float().transpose(2, 3)).view(b, hkv, most, group, -1) * s["scale"]
    score = score.masked_fill(~see[:, None, :, None, :], -math.inf)
    top = score.amax(dim=4, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim=4, keepdim=True)
    o = (p.view(b, hkv, most * group, -1) @ v.float()).view(b, hkv, most, group, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 2, 1, 3, 4).reshape(b, most, -1, d)
    return o[there].view(-1, s["hq"], d)


def _run_sample(s):
    if own:
        s["call"].run(s["stream"])
        return s["tokens"]
    logits = s["logits"].double()  # 64 bits: the ends of the kept set and the drawn place are borders
    rows, vocab = logits.shape
    greedy = s["temperature"] == 0
    w = torch.exp((logits - logits.amax(dim=1, keepdim=True)) / torch.where(greedy, 1.0, s["temperature"].double())[:, None])
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices  # equal logits: the lowest index first
    place = torch.arange(vocab, device=logits.device)
    k = torch.where((s["top_k"] <= 0) | (s["top_k"] > vocab), vocab, s["top_k"])
    sorted_w = torch.gather(w, 1, order) * (place < k[:, None])
    before = torch.cumsum(sorted_w, dim=1) - sorted_w
    keep = (place < k[:, None]) & ((before < s["top_p"].double()[:, None] * sorted_w.sum(dim=1, keepdim=True)) | (place == 0)
                                   | (s["top_p"] >= 1)[:, None])
    keep &= sorted_w >= s["min_p"].double()[:, None]
    keep &= ~greedy[:, None] | (place == 0)
    kept = torch.zeros_like(w).scatter(1, order, torch.gather(w, 1, order) * keep)
    upto = torch.cumsum(kept, dim=1)
    past = (upto > s["u"].double()[:, None] * upto[:, -1:]) & (kept > 0)
    return past.to(torch.int8).argmax(dim=1).to(torch.int32)


# ---- what a pass cannot do without -------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "q4":
        n, k, m = case["n"], case["k"], case["m"]
        return {"bytes": n * k / 2 + 4 * n * -(-k // case["group"]) + 4 * m * (n + k) + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if op == "quant4":
        n, k = case["n"], case["k"]
        return {"bytes": 4.5 * n * k + 4 * n * -(-k // case["group"]), "flops": 3 * n * k}
    if op == "append":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
        return {"bytes": t * d * (8 * hq + 12 * hkv), "flops": 8 * t * d * (hq + hkv)}
    if op == "tree":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        each = [(c + n, n * hq) for c, n in zip(_ragged(case["ctx"], case["seqs"], 3), _ragged(case["nodes"], case["seqs"], 5))]
        return {"bytes": sum(4 * keys * hkv * d + 8 * rows * d for keys, rows in each), "flops": sum(4 * rows * keys * d for keys, rows in each)}
    return {"bytes": 4 * case["rows"] * case["vocab"], "flops": 4 * case["rows"] * case["vocab"]}


# ---- the definitions in 64 bits, for how far either form is off ---------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"q4": _exact_q4, "quant4": _exact_quant4, "append": _exact_append, "tree": _exact_tree, "sample": lambda s: None}[case["op"]](s)


def _exact_q4(s):
    byte = s["packed"].double()
    code = torch.stack([byte % 16, torch.floor(byte / 16)], dim=2).flatten(1)[:, :s["k"]]
    code = torch.where(code > 7, code - 16, code)
    total = torch.zeros(s["x"].shape[0], code.shape[0], device="cuda", dtype=torch.float64)
    for j in range(s["scales"].shape[1]):
        part = slice(j * s["group"], min(s["k"], (j + 1) * s["group"]))
        total += (s["x"][:, part].double() @ code[:, part].t()) * s["scales"][:, j].double()
    return total if s["bias"] is None else total + s["bias"].double()


def _exact_quant4(s):
    n, k = s["w"].shape
    scales = torch.stack([p.abs().amax(dim=1) for p in s["w"].double().split(s["group"], dim=1)], dim=1) / 7
    return dict(packed=None, scales=torch.where(scales == 0, 1.0, scales))


def _exact_append(s):
    hq, hkv, d, dims, page = s["hq"], s["hkv"], s["d"], s["dims"], s["page"]
    z = s["qkv"].double().view(-1, hq + 2 * hkv, d)
    i = torch.arange(dims // 2, device="cuda", dtype=torch.float64)
    turn = torch.polar(torch.ones_like(i)[None], s["position"].double()[:, None] / s["base"] ** (2 * i / dims))

    def head(x, gamma):
        if gamma is not None:
            x = x / (x.square().sum(dim=-1, keepdim=True) / d + s["eps"]).sqrt() * gamma.double()
        x = x.clone()
        first, second = (slice(0, dims, 2), slice(1, dims, 2)) if s["pairs"] else (slice(0, dims // 2), slice(dims // 2, dims))
        c = torch.complex(x[..., first], x[..., second]) * turn[:, None]
        x[..., first], x[..., second] = c.real, c.imag
        return x

    q, k, v = head(z[:, :hq], s["q_gamma"]), head(z[:, hq:hq + hkv], s["k_gamma"]), z[:, hq + hkv:]
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    slot = s["table"].long()[s["sequence"].long(), s["index"].long().div(page, rounding_mode="floor")]
    kp[slot, :, s["index"].long() % page] = k
    vp[slot, :, s["index"].long() % page] = v
    return dict(q=q, k_pages=kp, v_pages=vp)


def _exact_tree(s):
    start, context, group, page = s["start"].tolist(), s["context"].tolist(), s["hq"] // s["hkv"], s["page"]
    out = torch.zeros(s["q"].shape[0], s["hq"], s["d"], device="cuda", dtype=torch.float64)
    for b in range(s["seqs"]):
        n = start[b + 1] - start[b]
        length = context[b] + n
        pages = s["table"][b, :-(-length // page)].long()
        bits = s["visible"][start[b]:start[b + 1]]
        see = torch.ones(n, length, device="cuda", dtype=torch.bool)
        see[:, context[b]:] = torch.stack([(bits >> j) & 1 for j in range(n)], dim=1) == 1
        for h in range(s["hkv"]):
            k = s["k_pages"][pages, h].reshape(-1, s["d"])[:length].double()
            v = s["v_pages"][pages, h].reshape(-1, s["d"])[:length].double()
            heads = slice(h * group, (h + 1) * group)
            t = torch.einsum("nhd,ld->nhl", s["q"][start[b]:start[b + 1], heads].double(), k) * s["scale"]
            out[start[b]:start[b + 1], heads] = torch.einsum(
                "nhl,ld->nhd", torch.softmax(t.masked_fill(~see[:, None], -math.inf), dim=2), v)
    return out
