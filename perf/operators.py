"""The operators of a drafted step, as cases that can be timed.

A serving step that checks several drafted tokens per request runs them in
this order: the attention of every request's tree of drafted tokens over the
paged cache, a token sampled after every node from given random numbers, the
path of the tree that those tokens accept, and the accepted rows moved together
in the cache. Forks of requests copy pages of the cache.

Each operator has a plain form in elementary tensor operations, which says what
it computes, and a call through the package's public entry points. Sizes are
those of the repository's model shapes (0.8B: 8 query and 2 KV heads, 6 layers
with a cache; 4B: 16 and 4, 8 layers; head dimension 256; vocabulary 248,320)
and of its benchmark's batches and contexts.
"""
import ctypes
import math

import numpy as np
import torch

own = False

SIGMAS = 2.2  # spread of a vocabulary's logits around their mean
VOCAB = 248320

# ------------------------------------------------------------------ the cases


def listed():
    return [
        # one request, a chain of four drafted tokens behind its pending one (0.8B): latency
        {"name": "tree_chain_1", "kind": "tree", "batch": 1, "heads": 8, "kv_heads": 2, "head_dim": 256, "page_tokens": 16,
         "min_context": 611, "max_context": 611, "min_nodes": 5, "max_nodes": 5, "gated": True},
        # the usual decode batch of 16 with small trees (0.8B)
        {"name": "tree_16", "kind": "tree", "batch": 16, "heads": 8, "kv_heads": 2, "head_dim": 256, "page_tokens": 16,
         "min_context": 64, "max_context": 4096, "min_nodes": 8, "max_nodes": 16, "gated": True},
        # 64 requests of ragged contexts and trees, some of one node alone (4B)
        {"name": "tree_64_ragged", "kind": "tree", "batch": 64, "heads": 16, "kv_heads": 4, "head_dim": 256,
         "page_tokens": 16, "min_context": 1, "max_context": 8192, "min_nodes": 1, "max_nodes": 23, "gated": True},
        # one long document with a full tree of 64 nodes (4B)
        {"name": "tree_long", "kind": "tree", "batch": 1, "heads": 16, "kv_heads": 4, "head_dim": 256, "page_tokens": 16,
         "min_context": 100003, "max_context": 100003, "min_nodes": 64, "max_nodes": 64, "gated": True},
        # one request's next token under the default sampling options
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": VOCAB, "temperature": 0.7, "top_k": 20, "top_p": 0.95,
         "min_p": 0.0, "penalty": 1.05, "masked": 0.0, "mixed": False},
        # a decode batch that keeps a nucleus of any width
        {"name": "sample_16_nucleus", "kind": "sample", "rows": 16, "vocab": VOCAB, "temperature": 1.0, "top_k": 0,
         "top_p": 0.95, "min_p": 0.02, "penalty": 1.0, "masked": 0.0, "mixed": False},
        # every node of 16 small trees, each request with options of its own and
        # a grammar that leaves out part of the vocabulary
        {"name": "sample_256_mixed", "kind": "sample", "rows": 256, "vocab": VOCAB, "temperature": 0.8, "top_k": 50,
         "top_p": 0.9, "min_p": 0.05, "penalty": 1.1, "masked": 0.3, "mixed": True},
        # the accepted path of one small tree, and of a full batch of large ones
        {"name": "accept_1", "kind": "accept", "batch": 1, "min_nodes": 16, "max_nodes": 16},
        {"name": "accept_64", "kind": "accept", "batch": 64, "min_nodes": 9, "max_nodes": 64},
        # the shared tail pages of 8 requests copied before they are written (0.8B)
        {"name": "copy_tails_8", "kind": "copy", "pairs": 8, "layers": 6, "kv_heads": 2, "head_dim": 256, "page_tokens": 16,
         "partial": True},
        # the whole pages of a long request copied (4B): 2000-odd pages in 8 layers
        {"name": "copy_2047", "kind": "copy", "pairs": 2047, "layers": 8, "kv_heads": 4, "head_dim": 256, "page_tokens": 16,
         "partial": False},
        # the accepted rows of a batch's trees moved together (0.8B)
        {"name": "compact_64", "kind": "compact", "batch": 64, "layers": 6, "kv_heads": 2, "head_dim": 256,
         "page_tokens": 16, "min_nodes": 9, "max_nodes": 40},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "sample", "sample", "accept", "copy", "compact"])
    if kind == "tree":
        heads, kv = rng.choice([(8, 2), (16, 4), (4, 4), (16, 2), (6, 2), (5, 1)])
        batch = _log_int(rng, 1, 64)
        top = _log_int(rng, 16, min(60000, 250000 // batch))
        nodes = _log_int(rng, 1, 64 if batch * top < 60000 else 24)
        return {"kind": "tree", "batch": batch, "heads": heads, "kv_heads": kv, "head_dim": rng.choice([256, 256, 256, 128, 64]),
                "page_tokens": rng.choice([4, 16, 16, 64]), "min_context": rng.randint(0, top), "max_context": top,
                "min_nodes": rng.randint(1, nodes), "max_nodes": nodes, "gated": rng.random() < 0.8}
    if kind == "sample":
        return {"kind": "sample", "rows": _log_int(rng, 1, 128), "vocab": rng.choice([VOCAB, VOCAB, _log_int(rng, 100, VOCAB)]),
                "temperature": rng.choice([0.0, 0.6, 0.7, 1.0, 1.3]), "top_k": rng.choice([0, 0, 1, 20, 50, 300]),
                "top_p": rng.choice([1.0, 0.8, 0.95]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]),
                "penalty": rng.choice([1.0, 1.05, 1.1]), "masked": rng.choice([0.0, 0.0, 0.5, 0.99]),
                "mixed": rng.random() < 0.4}
    nodes = _log_int(rng, 4, 128)
    if kind == "accept":
        return {"kind": "accept", "batch": _log_int(rng, 1, 256), "min_nodes": rng.randint(1, nodes), "max_nodes": nodes}
    heads, dim = rng.choice([(2, 256), (4, 256), (4, 64), (1, 128), (3, 20)])
    layers = rng.choice([1, 6, 8])
    if kind == "copy":
        return {"kind": "copy", "pairs": _log_int(rng, 1, 1500), "layers": layers, "kv_heads": heads, "head_dim": dim,
                "page_tokens": rng.choice([4, 16, 16, 64 if layers == 1 else 16]), "partial": rng.random() < 0.5}
    return {"kind": "compact", "batch": _log_int(rng, 1, 64), "layers": layers, "kv_heads": heads, "head_dim": dim,
            "page_tokens": rng.choice([4, 16, 16]), "min_nodes": rng.randint(4, nodes), "max_nodes": nodes}


# ------------------------------------------------------------------- material


_PROGRAM = {}


def _stream():
    """The program's one stream, torch's current one from here on and the context's: inputs, operators and whatever
    reads the outputs follow one another on it."""
    if "stream" not in _PROGRAM:
        _PROGRAM["stream"] = torch.cuda.Stream()
    stream, current = _PROGRAM["stream"], torch.cuda.current_stream()
    if current != stream:
        stream.wait_stream(current)
        torch.cuda.set_stream(stream)
    return stream


def _generators(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g, np.random.default_rng(int(seed))


class _Arg:
    """A torch tensor as a buffer argument of the package's operators."""

    def __init__(self, tensor):
        assert tensor.is_contiguous()
        self.tensor, self.ptr = tensor, ctypes.c_void_p(tensor.data_ptr())


def _dev(array):
    return _Arg(torch.from_numpy(np.ascontiguousarray(array)).to("cuda"))


def _tree(r, n):
    """Parents of a tree of n nodes, parents before children (node 0 the root,
    the others below one of the last few nodes)."""
    i = np.arange(1, n)
    return np.concatenate([[-1], i - r.integers(1, np.minimum(i, 6) + 1)]).astype(np.int32)


def _ancestors(parents, words):
    """Bit j of row i: node j is node i or above it."""
    bits = []
    for i, p in enumerate(parents):
        bits.append((1 << i) | (bits[p] if p >= 0 else 0))
    out = np.array([[(b >> (64 * w)) & 0xFFFFFFFFFFFFFFFF for w in range(words)] for b in bits], np.uint64)
    return out.view(np.int64).reshape(len(parents), words)


def _spread(r, low, high, n):
    """n whole numbers spread evenly over low..high, in an order of the seed's:
    every seed has the same numbers, so its outputs have the same shapes."""
    return r.permutation(np.rint(np.linspace(high, low, n)).astype(np.int32))


def _starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def _pages(r, rows, page_tokens):
    """A page table whose requests hold the given numbers of rows in pages of
    their own, in any order, and the number of pages."""
    need = [(int(n) + page_tokens - 1) // page_tokens for n in rows]
    perm = r.permutation(sum(need)).astype(np.int32)
    table = np.zeros((len(need), max(max(need), 1)), np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, max(sum(need), 1)


def _halves(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(torch.float16)


def prepare(case, seed):
    _stream()
    g, r = _generators(seed)
    kind = case["kind"]
    s = {"case": case, "kind": kind}
    if kind in ("tree", "accept", "compact"):
        nodes = _spread(r, case["min_nodes"], case["max_nodes"], case["batch"])
        start = _starts(nodes)
        parents = [_tree(r, int(n)) for n in nodes]
        rows = int(start[-1])
        s.update(rows=rows, max_nodes=int(nodes.max()), node_start=_dev(start), batch=case["batch"])
    if kind == "tree":
        pt, hd, kv, heads = (case[k] for k in ("page_tokens", "head_dim", "kv_heads", "heads"))
        context = _spread(r, case["min_context"], case["max_context"], case["batch"])
        table, total = _pages(r, context + nodes, pt)
        words = (s["max_nodes"] + 63) // 64
        s.update(total_pages=total, max_len=int((context + nodes).max()), table=_dev(table), context=_dev(context),
                 masks=_dev(np.concatenate([_ancestors(p, words) for p in parents])),
                 k=_Arg(_halves(g, total, pt, kv, hd)), v=_Arg(_halves(g, total, pt, kv, hd)),
                 q=_Arg(torch.randn(rows, heads, hd, generator=g, device="cuda")),
                 gates=_Arg(torch.randn(rows, heads, hd, generator=g, device="cuda")) if case["gated"] else None,
                 out=_Arg(torch.zeros(rows, heads, hd, device="cuda")))
    elif kind == "sample":
        n, vocab = case["rows"], case["vocab"]
        x = torch.randn(n, vocab, generator=g, device="cuda") * SIGMAS
        # a few tokens stand out, as after most contexts
        peaks = torch.randint(0, vocab, (n, 24), generator=g, device="cuda")
        x.scatter_add_(1, peaks, 6.0 + 10.0 * torch.rand(n, 24, generator=g, device="cuda"))
        if case["masked"] > 0:
            x.masked_fill_(torch.rand(n, vocab, generator=g, device="cuda") < case["masked"], -math.inf)
        options = {"temperature": np.full(n, case["temperature"], np.float32), "top_k": np.full(n, case["top_k"], np.int32),
                   "top_p": np.full(n, case["top_p"], np.float32), "min_p": np.full(n, case["min_p"], np.float32),
                   "penalty": np.full(n, case["penalty"], np.float32)}
        if case["mixed"]:
            for name, off in (("temperature", 0.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0), ("penalty", 1.0)):
                options[name][r.random(n) < 0.25] = off
        s.update({k: _dev(v) for k, v in options.items()})
        s.update(logits=_Arg(x), uniforms=_Arg(torch.rand(n, generator=g, device="cuda")), counts=None,
                 token=_Arg(torch.zeros(n, dtype=torch.int32, device="cuda")), probability=_Arg(torch.zeros(n, device="cuda")))
        if case["penalty"] > 1.0:
            seen = torch.randint(0, vocab, (n, 512), generator=g, device="cuda")
            s["counts"] = _Arg(torch.zeros(n, vocab, dtype=torch.int32, device="cuda").scatter_(1, seen, 1))
    elif kind == "accept":
        # siblings hold different tokens; most nodes' sampled token is a child's
        draft = np.concatenate([(r.integers(0, VOCAB) + 7919 * np.arange(n)) % VOCAB for n in nodes]).astype(np.int32)
        sampled = r.integers(0, VOCAB, size=rows).astype(np.int32)
        up = np.concatenate([np.where(p < 0, -1, start[b] + p) for b, p in enumerate(parents)])
        child = r.permutation(np.flatnonzero((up >= 0) & (r.random(rows) < 0.85)))
        sampled[up[child]] = draft[child]
        s.update(parents=_dev(np.concatenate(parents)), draft=_dev(draft), sampled=_dev(sampled),
                 path=_Arg(torch.zeros(case["batch"], s["max_nodes"], dtype=torch.int32, device="cuda")),
                 count=_Arg(torch.zeros(case["batch"], dtype=torch.int32, device="cuda")),
                 next=_Arg(torch.zeros(case["batch"], dtype=torch.int32, device="cuda")))
    else:
        pt, layers, width = case["page_tokens"], case["layers"], case["kv_heads"] * case["head_dim"]
        if kind == "copy":
            n = case["pairs"]
            ids = r.permutation(2 * n + 3).astype(np.int32)
            s["src"], s["dst"] = ids[:n].copy(), ids[n:2 * n].copy()
            s["tokens"] = r.integers(1, pt + 1, size=n).astype(np.int32) if case["partial"] else np.full(n, pt, np.int32)
            total = 2 * n + 3
        else:
            context = r.integers(0, 200, size=case["batch"]).astype(np.int32)
            table, total = _pages(r, np.full(case["batch"], 200 + s["max_nodes"]), pt)
            # accepted paths whose nodes other than the root and those already
            # in place lie behind the rows that are written: the same pass can
            # then be made again on its own result
            path = np.full((case["batch"], s["max_nodes"]), -1, np.int32)
            count = np.zeros(case["batch"], np.int32)
            for b, m in enumerate(nodes):
                c = int(r.integers(1, int(m) // 2 + 1)) if m > 1 else 1
                path[b, :c] = np.concatenate([[0], np.sort(r.permutation(np.arange(c, int(m)))[:c - 1])])
                count[b] = c
            s.update(table=_dev(table), context=_dev(context), path=_dev(path), count=_dev(count))
        s.update(total_pages=total, k=_Arg(_halves(g, layers, total, pt, width)), v=_Arg(_halves(g, layers, total, pt, width)))
    return s


# ------------------------------------------------------------- the plain forms


def _visible(masks, context, owner, node, length, nodes, words):
    """[rows, length]: which rows of its request's cache a node sees."""
    t = torch.arange(length, device="cuda")
    j = t - context[owner].unsqueeze(1)
    bits = masks.gather(1, (j.clamp(0, 64 * words - 1) >> 6)) >> (j.clamp(min=0) & 63)
    return (j < 0) | ((j < nodes[owner].unsqueeze(1)) & ((bits & 1) == 1))


def _plain_tree(s):
    c, n = s["case"], s["max_nodes"]
    heads, kv, hd, pt, batch, length = c["heads"], c["kv_heads"], c["head_dim"], c["page_tokens"], c["batch"], s["max_len"]
    qpk = heads // kv
    start = s["node_start"].tensor.long()
    nodes = start[1:] - start[:-1]
    owner = torch.repeat_interleave(torch.arange(batch, device="cuda"), nodes, output_size=s["rows"])
    node = torch.arange(s["rows"], device="cuda") - start[owner]
    context, table = s["context"].tensor.long(), s["table"].tensor.long()
    t = torch.arange(length, device="cuda")
    at = table[:, (t // pt).clamp(max=table.shape[1] - 1)] * pt + t % pt
    keys = s["k"].tensor.view(-1, kv, hd)[at].float().permute(0, 2, 3, 1).contiguous()   # [batch, kv, hd, length]
    values = s["v"].tensor.view(-1, kv, hd)[at].float().permute(0, 2, 1, 3).contiguous()  # [batch, kv, length, hd]
    q = torch.zeros(batch, n, heads, hd, device="cuda")
    q[owner, node] = s["q"].tensor
    seen = torch.zeros(batch, n, length, dtype=torch.bool, device="cuda")
    seen[owner, node] = _visible(s["masks"].tensor, context, owner, node, length, nodes, s["masks"].tensor.shape[1])
    q = q.view(batch, n, kv, qpk, hd).permute(0, 2, 1, 3, 4).reshape(batch, kv, n * qpk, hd)
    score = torch.matmul(q, keys) * (1.0 / math.sqrt(hd))
    score = score.view(batch, kv, n, qpk, length).masked_fill_(~seen.view(batch, 1, n, 1, length), -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3.0e38)
    p = torch.exp(score - top).view(batch, kv, n * qpk, length)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, values) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.view(batch, kv, n, qpk, hd).permute(0, 2, 1, 3, 4).reshape(batch, n, heads, hd)[owner, node]
    return out / (1.0 + torch.exp(-s["gates"].tensor)) if s["gates"] is not None else out


def _plain_sample(s):
    x = s["logits"].tensor
    if s["counts"] is not None:
        r = s["penalty"].tensor.unsqueeze(1)
        hit = (s["counts"].tensor > 0) & (r > 1.0)
        # the quotient rounded once to 32 bits
        x = torch.where(hit, torch.where(x > 0, (x.double() / r.double()).float(), x * r), x)
    vocab = x.shape[1]
    x, order = torch.sort(torch.where(torch.isnan(x), -math.inf, x), dim=1, descending=True, stable=True)
    x = x.double()
    t = s["temperature"].tensor.double().unsqueeze(1)
    greedy = t <= 1e-6
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, 1.0, t))
    rank = torch.arange(vocab, device="cuda").unsqueeze(0)
    k = s["top_k"].tensor.long().unsqueeze(1)
    k = torch.where((k <= 0) | (k > vocab), vocab, k)
    cum = torch.cumsum(w, 1)
    before = cum - w
    nucleus = s["top_p"].tensor.double().unsqueeze(1)
    enough = nucleus * cum.gather(1, k - 1)
    keep = (rank < k) & ((nucleus >= 1.0) | (before < enough)) & (w >= s["min_p"].tensor.double().unsqueeze(1))
    keep = (keep & ~greedy) | (rank == 0)
    last = keep.sum(1, keepdim=True) - 1
    mass = cum.gather(1, last)
    at = torch.minimum((cum <= s["uniforms"].tensor.double().unsqueeze(1) * mass).sum(1, keepdim=True), last)
    token, p = order.gather(1, at), w.gather(1, at) / mass
    none = torch.isinf(x[:, :1]) & (x[:, :1] < 0)
    return {"token": torch.where(none, -1, token).squeeze(1).int(), "probability": torch.where(none, 0.0, p).squeeze(1).float()}


def _plain_accept(s):
    start, rows = s["node_start"].tensor.long(), s["rows"]
    parents, draft, sampled = (s[k].tensor.long() for k in ("parents", "draft", "sampled"))
    batch, width = s["batch"], s["max_nodes"]
    owner = torch.repeat_interleave(torch.arange(batch, device="cuda"), start[1:] - start[:-1], output_size=rows)
    node = torch.arange(rows, device="cuda") - start[owner]
    up = torch.where(parents >= 0, start[owner] + parents, -1)
    agrees = (up >= 0) & (draft == sampled[up.clamp(min=0)])
    path = torch.full((batch, width + 1), -1, dtype=torch.long, device="cuda")
    path[:, 0] = 0
    at, count = start[:-1].clone(), torch.ones(batch, dtype=torch.long, device="cuda")
    for depth in range(1, width):
        child = torch.where(agrees & (up == at[owner]), node, rows)
        child = torch.full((batch,), rows, device="cuda").scatter_reduce_(0, owner, child, "amin")
        found = (child < rows) & (count == depth)
        path[:, depth] = torch.where(found, child, -1)
        at = torch.where(found, start[:-1] + child, at)
        count += found
    return {"path": path[:, :width].int(), "count": count.int(), "next": sampled[at].int()}


def _plain_copy(s):
    pt = s["case"]["page_tokens"]
    src, dst, tokens = (torch.from_numpy(s[k]).to("cuda").long() for k in ("src", "dst", "tokens"))
    keep = (torch.arange(pt, device="cuda") < tokens.unsqueeze(1)).view(1, -1, pt, 1)
    for pool in (s["k"].tensor, s["v"].tensor):
        pool[:, dst] = torch.where(keep, pool[:, src], pool[:, dst])


def _plain_compact(s):
    pt, path = s["case"]["page_tokens"], s["path"].tensor.long()
    context, table = s["context"].tensor.long().unsqueeze(1), s["table"].tensor.long()
    j = torch.arange(path.shape[1], device="cuda").unsqueeze(0)
    moved = j < s["count"].tensor.unsqueeze(1)
    last = table.shape[1] - 1

    def row(t):
        return table.gather(1, (t // pt).clamp(0, last)) * pt + t % pt

    to, of = row(context + j)[moved], row(context + path)[moved]
    for pool in (s["k"].tensor, s["v"].tensor):
        flat = pool.view(pool.shape[0], -1, pool.shape[-1])
        flat[:, to] = flat[:, of]


# ------------------------------------------------------------- the framework's


def _program():
    """The package and the program's one context (one device, the program's stream)."""
    if "ctx" not in _PROGRAM:
        import importlib

        q = importlib.import_module("qwen35-cpu_amd")
        _PROGRAM["q"], _PROGRAM["ctx"] = q, q.Context(0, _stream().cuda_stream)
    return _PROGRAM["q"], _PROGRAM["ctx"]


def run(s):
    c, kind = s["case"], s["kind"]
    if kind == "tree":
        if not own:
            return _plain_tree(s)
        q, ctx = _program()
        q.attention_tree_paged(ctx, s["q"], s["gates"], s["k"], s["v"], s["total_pages"], s["table"],
                               s["table"].tensor.shape[1], c["page_tokens"], s["context"], s["node_start"], s["masks"],
                               s["out"], s["batch"], s["rows"], s["max_nodes"], s["max_len"], c["heads"], c["kv_heads"],
                               c["head_dim"], 1.0 / math.sqrt(c["head_dim"]))
        return s["out"].tensor
    if kind == "sample":
        if not own:
            return _plain_sample(s)
        q, ctx = _program()
        q.sample_logits(ctx, s["logits"], c["vocab"], s["counts"], s["penalty"], s["temperature"], s["top_k"], s["top_p"],
                        s["min_p"], s["uniforms"], c["rows"], c["vocab"], s["token"], s["probability"])
        return {"token": s["token"].tensor, "probability": s["probability"].tensor}
    if kind == "accept":
        if not own:
            return _plain_accept(s)
        q, ctx = _program()
        q.tree_accept(ctx, s["node_start"], s["parents"], s["draft"], s["sampled"], s["path"], s["max_nodes"], s["count"],
                      s["next"], s["batch"], s["rows"], s["max_nodes"])
        return {"path": s["path"].tensor, "count": s["count"].tensor, "next": s["next"].tensor}
    width = c["kv_heads"] * c["head_dim"]
    stride = s["total_pages"] * c["page_tokens"] * width
    if kind == "copy":
        if not own:
            _plain_copy(s)
        else:
            q, ctx = _program()
            q.cache_copy_pages(ctx, s["k"], s["v"], c["layers"], stride, s["total_pages"], c["page_tokens"], width, s["src"],
                               s["dst"], s["tokens"])
    elif not own:
        _plain_compact(s)
    else:
        q, ctx = _program()
        q.cache_compact_rows(ctx, s["k"], s["v"], c["layers"], stride, s["total_pages"], c["page_tokens"], width, s["table"],
                             s["table"].tensor.shape[1], s["context"], s["path"], s["max_nodes"], s["count"], s["batch"])
    # the cache's binary16 rows as the bits they are: a copy changes none
    return {"k": s["k"].tensor.view(torch.int16), "v": s["v"].tensor.view(torch.int16)}


# ------------------------------------------------------ what it cannot do without


def _mean(case, what):
    return float(np.linspace(case["max_" + what], case["min_" + what], case["batch"]).mean())


def work(case):
    kind = case["kind"]
    if kind == "tree":
        nodes, tokens = _mean(case, "nodes"), _mean(case, "context") + _mean(case, "nodes")
        rows = case["batch"] * nodes
        return {"bytes": case["batch"] * tokens * case["kv_heads"] * case["head_dim"] * 4.0 +
                rows * case["heads"] * case["head_dim"] * (12.0 if case["gated"] else 8.0) + rows * 8,
                "flops": 4.0 * rows * tokens * case["heads"] * case["head_dim"]}
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (8.0 if case["penalty"] > 1.0 else 4.0) + case["rows"] * 32.0, "flops": 30.0 * n}
    if kind == "accept":
        rows = case["batch"] * _mean(case, "nodes")
        return {"bytes": rows * 12.0 + case["batch"] * (12.0 + 4.0 * case["max_nodes"]), "flops": rows * 2.0}
    width = case["layers"] * case["kv_heads"] * case["head_dim"] * 2.0 * 2.0  # bytes of a token's rows, K and V
    if kind == "copy":
        tokens = case["pairs"] * ((case["page_tokens"] + 1) / 2 if case["partial"] else case["page_tokens"])
        return {"bytes": 2.0 * tokens * width, "flops": 0.0}
    return {"bytes": 2.0 * case["batch"] * max(1.0, _mean(case, "nodes") / 4) * width, "flops": 0.0}


# ------------------------------------------------- the definitions in 64 bits


def _exact_tree(s, case):
    """Request by request and head by head, each node over the rows it sees."""
    host = {k: s[k].tensor.cpu().numpy() for k in ("node_start", "context", "masks", "table")}
    pt, qpk = case["page_tokens"], case["heads"] // case["kv_heads"]
    out = torch.zeros_like(s["q"].tensor, dtype=torch.float64)
    for b in range(case["batch"]):
        r0, r1, c = int(host["node_start"][b]), int(host["node_start"][b + 1]), int(host["context"][b])
        t = np.arange(c + r1 - r0)
        at = torch.from_numpy(host["table"][b][t // pt].astype(np.int64) * pt + t % pt).to("cuda")
        bits = np.unpackbits(host["masks"][r0:r1].astype("<i8").view(np.uint8), axis=1, bitorder="little")[:, :r1 - r0]
        hidden = torch.from_numpy(np.concatenate([np.zeros((r1 - r0, c), bool), bits == 0], axis=1)).to("cuda")
        for h in range(case["heads"]):
            k = s["k"].tensor.flatten(0, 1)[at, h // qpk].double()
            v = s["v"].tensor.flatten(0, 1)[at, h // qpk].double()
            a = (s["q"].tensor[r0:r1, h].double() @ k.T.contiguous()) / math.sqrt(case["head_dim"])
            a = torch.softmax(a.masked_fill(hidden, -math.inf), dim=1)
            out[r0:r1, h] = torch.nan_to_num(a) @ v
    return out * torch.sigmoid(s["gates"].tensor.double()) if case["gated"] else out


def _exact_sample(s):
    """Row by row: the tokens in order, cut from the end, then walked to the number."""
    host = {k: s[k].tensor.cpu().numpy() for k in ("logits", "temperature", "top_k", "top_p", "min_p", "penalty", "uniforms")}
    counts = s["counts"].tensor.cpu().numpy() if s["counts"] is not None else None
    tokens, probabilities = [], []
    for i, x in enumerate(host["logits"]):
        x = x.copy()
        r = host["penalty"][i]
        if counts is not None and r > 1.0:
            hit = counts[i] > 0
            x[hit] = np.where(x[hit] > 0, x[hit] / r, x[hit] * r)
        order = np.argsort(-x, kind="stable")
        order = order[np.isfinite(x[order])]
        if order.size == 0:
            tokens.append(-1)
            probabilities.append(0.0)
            continue
        if host["temperature"][i] <= 1e-6:
            tokens.append(int(order[0]))
            probabilities.append(1.0)
            continue
        if 0 < host["top_k"][i] < order.size:
            order = order[:host["top_k"][i]]
        v = x[order].astype(np.float64)
        w = np.exp((v - v[0]) / np.float64(host["temperature"][i]))
        total, n = math.fsum(w), order.size
        if host["top_p"][i] < 1.0:
            n = min(n, int(np.searchsorted(np.cumsum(w), np.float64(host["top_p"][i]) * total, side="left")) + 1)
        n = max(1, min(n, int((w >= np.float64(host["min_p"][i])).sum())))
        w = w[:n]
        mass = math.fsum(w)
        at = min(n - 1, int(np.searchsorted(np.cumsum(w), np.float64(host["uniforms"][i]) * mass, side="right")))
        tokens.append(int(order[at]))
        probabilities.append(w[at] / mass)
    return {"token": np.array(tokens, np.int32), "probability": np.array(probabilities, np.float64)}


def exact(case, seed):
    if case["kind"] not in ("tree", "sample"):
        return None  # whole numbers and copied bits
    s = prepare(case, seed)
    return _exact_tree(s, case) if case["kind"] == "tree" else _exact_sample(s)
