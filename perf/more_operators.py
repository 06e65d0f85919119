"""Decoding with drafted tokens and sampling, in elementary torch operations and
through the entry points of `spissa_amd.device`.

Kinds:

  tree    attention of a tree of drafted tokens over a KV cache, for each of a batch
          of sequences. Node t of a sequence has a parent among the nodes before it
          (-1: none); its position is the cache's length plus its depth, and it sees
          the cached rows, its ancestors and itself (with a window W: those less than
          W positions before it). Queries and keys are (Gemma: RMS-normed first) rotated
          by their position, and the nodes' rows appended to the cache:
          out_t = sum_j p_tj v_j,  p_t = softmax_j(q_t . k_j / sqrt(d))
  sample  one token of each row of logits. With w_i = exp((x_i - max x) / T), in the
          order of falling logits (equal ones by index): the first top_k, of those the
          shortest run whose weights reach top_p of their sum, of those the ones with
          w_i >= min_p. The token is the first index whose running sum of kept weights,
          in index order, is above u times their sum; its probability is its share of
          that sum. T = 0 takes the largest logit.
  accept  the drafted tokens that the sampled ones confirm: from node 0, the first child
          whose drafted token is the one sampled at its parent, and so on down
  keep    the accepted nodes' rows moved together in the caches of several layers:
          row P + i is what row P + path[i] was

Head shapes are the Llama 3.2 and Gemma 3 ones that this repository's benchmark uses,
or generic; so are the vocabularies.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-6

# query heads, KV heads, head dim
HEADS = {"llama1b": (32, 8, 64), "llama3b": (24, 8, 128), "gemma1b": (4, 1, 256), "gemma4b": (8, 4, 256)}


def listed():
    return [
        # A short chat turn with a draft of five tokens in a row: all latency.
        _tree("tree_chain_5", "llama1b", 1, 499, 5, "chain", 0),
        # One sequence's tree over a long context.
        _tree("tree_26_8192", "llama3b", 1, 8192, 26, "tree", 0),
        # A serving batch, ragged lengths and trees.
        _tree("tree_batch16", "llama3b", 16, 8192, 12, "tree", 0),
        # A sliding-window layer with the QK-norm.
        _tree("tree_window_32", "gemma4b", 1, 5000, 32, "tree", 1024),
        # One KV head, a long context and the widest tree.
        _tree("tree_256_32768", "gemma1b", 1, 32768, 256, "tree", 0),
        # The token after a step of one sequence.
        _sample("sample_1", 1, 128256, "all", False),
        # A batch whose requests each have their own settings; logits of a bf16 head, with ties.
        _sample("sample_64", 64, 128256, "rows", True),
        # The nodes of a small tree over the largest vocabulary, temperature alone.
        _sample("sample_plain_5", 5, 262144, "none", False),
        # One sequence's draft.
        {"name": "accept_1", "kind": "accept", "batch": 1, "nodes": 5},
        # A serving batch's trees.
        {"name": "accept_64", "kind": "accept", "batch": 64, "nodes": 64},
        # A whole model's caches after one sequence's draft.
        {"name": "keep_28_layers", "kind": "keep", "layers": 28, "batch": 1, "kv": 8, "dim": 128, "cached": 777, "nodes": 26, "kept": 4},
        # A layer of a batch, large trees of which much is accepted.
        {"name": "keep_batch32", "kind": "keep", "layers": 1, "batch": 32, "kv": 8, "dim": 128, "cached": 500, "nodes": 64, "kept": 12},
    ]


def _tree(name, model, batch, cached, nodes, shape, window):
    hq, hkv, d = HEADS[model]
    return {"name": name, "kind": "tree", "batch": batch, "cached": cached, "nodes": nodes, "shape": shape, "q": hq, "kv": hkv,
            "dim": d, "window": window, "norm": model.startswith("gemma")}


def _sample(name, rows, vocab, settings, ties):
    return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "settings": settings, "ties": ties}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "tree", "sample", "sample", "sample", "accept", "keep"])
    if kind == "sample":
        vocab = _log(rng, 1000, 262144)
        case = _sample("", rng.choice([1, _log(rng, 2, max(2, min(256, 8.2e6 / vocab)))]), vocab,
                       rng.choice(["none", "all", "all", "rows", "rows"]), rng.random() < 0.5)
        del case["name"]
        return case
    if kind == "accept":
        return {"kind": kind, "batch": _log(rng, 1, 64), "nodes": _log(rng, 2, 256)}
    if kind == "keep":
        layers = rng.choice([1, rng.randint(2, 32)])
        nodes = _log(rng, 2, 96)
        return {"kind": kind, "layers": layers, "batch": rng.randint(1, 32 // layers), "kv": rng.randint(1, 8),
                "dim": rng.choice([64, 128, 256]), "cached": _log(rng, 1, 1500), "nodes": nodes, "kept": rng.randint(1, min(16, (nodes + 1) // 2))}
    if rng.random() < 0.5:
        model = rng.choice(sorted(HEADS))
        (hq, kv, d), norm = HEADS[model], model.startswith("gemma")
    else:
        kv, d, norm = rng.randint(1, 8), rng.choice([64, 128, 256]), rng.random() < 0.3
        hq = kv * rng.choice([1, 2, 3, 4, 5, 8])
    batch = rng.choice([1, 1, rng.randint(2, 16)])
    cached = rng.choice([_log(rng, 1, 512), _log(rng, 256, max(256, min(32768, 1.3e8 / (batch * kv * d))))])
    nodes = rng.choice([rng.randint(1, 8), _log(rng, 4, max(4, min(256, 7.0e9 / (batch * hq * d * (cached + 64)))))])
    return {"kind": kind, "batch": batch, "cached": cached, "nodes": nodes, "shape": rng.choice(["chain", "tree", "tree", "tree"]),
            "q": hq, "kv": kv, "dim": d, "window": rng.choice([0, 0, 0, _log(rng, 16, 2048)]), "norm": norm}


# ---------------------------------------------------------------------------
# inputs


def _lens(case):
    """Rows of each sequence's cache: a batch's lengths spread down to a quarter of the longest, odd ones among them."""
    n, b = case["cached"], case["batch"]
    return [max(1, n - (3 * n * i) // (4 * b)) for i in range(b)]


def _nodes(case):
    """Nodes of each sequence's tree, down to half of the largest."""
    t, b = case["nodes"], case["batch"]
    return [max(1, t - (t * i) // (2 * b)) for i in range(b)]


def _parents(case):
    """Each sequence's tree: a matter of the case, as a program's draft has a fixed form."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    chain = case.get("shape") == "chain"
    return [[-1] + [i - 1 if chain else rng.randrange(max(0, i - 9), i) for i in range(1, n)] for n in _nodes(case)]


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def _inputs(case, seed):
    """Every input tensor of a case from the seed alone, the same for prepare() and exact()."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=DEV)  # noqa: E731
    uniform = lambda *shape: torch.rand(*shape, generator=gen, device=DEV)  # noqa: E731
    whole = lambda lo, hi, *shape: torch.randint(lo, hi, shape, generator=gen, device=DEV, dtype=torch.int32)  # noqa: E731
    kind = case["kind"]
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a broad base, and some tokens well above it
        x = normal(rows, vocab) * 2.0
        at = torch.randint(0, vocab, (rows, 96), generator=gen, device=DEV)
        x.scatter_reduce_(1, at, torch.linspace(14.0, 4.0, 96, device=DEV) + normal(rows, 96), "amax")
        got = {"logits": x.bfloat16().float() if case["ties"] else x, "u": uniform(rows)}
        if case["settings"] == "all":
            return got | {"temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.02}
        if case["settings"] == "none":
            return got | {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
        pick = lambda values: torch.tensor(values, device=DEV)[whole(0, len(values), rows).long()]  # noqa: E731
        return got | {"temperature": pick([0.0, 0.6, 0.7, 0.8, 1.0, 1.0, 1.3]), "top_k": pick([0, 0, 1, 20, 50, 1000]).int(),
                      "top_p": pick([1.0, 1.0, 0.5, 0.8, 0.9, 0.95, 0.99]), "min_p": pick([0.0, 0.0, 0.02, 0.1])}
    if kind == "accept":
        parents = torch.tensor(sum(_parents(case), []), device=DEV, dtype=torch.int32)
        # few tokens, so that children often hold the one sampled
        return {"parents": parents, "tokens": whole(0, 3, len(parents)), "sampled": whole(0, 3, len(parents))}
    kv, d = case["kv"], case["dim"]
    if kind == "keep":
        n, t = case["layers"] * case["batch"], case["nodes"]
        path = torch.full((case["batch"], t), -1, device=DEV, dtype=torch.int32)
        # node 0, then rising nodes behind the rows they move to
        for row in path:
            row[0] = 0
            row[1:case["kept"]] = case["kept"] + torch.randperm(t - case["kept"], generator=gen, device=DEV)[:case["kept"] - 1].sort().values
        count = torch.full((case["batch"],), case["kept"], device=DEV, dtype=torch.int32)
        return {"rows": normal(n, 2, t, kv, d), "path": path.reshape(-1), "count": count}
    lens, total = _lens(case), sum(_nodes(case))
    bk, bv = normal(kv, d), normal(kv, d) * 0.25  # channels' own offsets
    got = {"past_k": [normal(p, kv, d) + bk for p in lens], "past_v": [normal(p, kv, d) + bv for p in lens],
           "q": normal(total, case["q"], d), "k": normal(total, kv, d) + bk, "v": normal(total, kv, d) + bv,
           "parents": torch.tensor(sum(_parents(case), []), device=DEV, dtype=torch.int32)}
    if case["norm"]:
        got |= {"q_norm": 1.0 + 0.25 * normal(d), "k_norm": 1.0 + 0.25 * normal(d)}
    return got


def _base(case):
    """The rotation's base, by the kind of model."""
    return 1000000.0 if case["norm"] else 500000.0


def _angles(case, positions):
    """The angles as the tables define them, in single precision: position times 1 / base^(2 i / d)."""
    d = case["dim"]
    power = torch.tensor([_base(case) ** (2 * i / d) for i in range(d // 2)], dtype=torch.float64).float()
    return positions.float()[:, None] * (1.0 / power).to(positions.device)


# ---------------------------------------------------------------------------
# the plain form


def _ancestors(parents):
    """[b, t, t]: whether column's node is the row's or one above it; parents [b, t], -1 for none."""
    t = parents.shape[1]
    up = torch.eye(t, device=DEV) + (parents[..., None] == torch.arange(t, device=DEV)).float()
    for _ in range((t - 1).bit_length()):
        up = (up @ up).clamp(max=1.0)
    return up > 0


def _norm(x, weight):
    return x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * weight


def _rotate(x, cos, sin):
    """Halves as pairs; cos, sin [n, d / 2]."""
    a, b = x.chunk(2, -1)
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_tree(st):
    case = st["case"]
    hq, hkv, d, window = case["q"], case["kv"], case["dim"], case["window"]
    at, first, (b, t) = st["at"], st["first"], st["shape"]  # rows of the padded batch that are there
    up = _ancestors(torch.full((b * t,), -1, device=DEV, dtype=torch.int32).index_copy(0, at, st["parents"]).reshape(b, t))
    depth = up.sum(-1) - 1
    pos = first[:, None] + depth
    q, k = st["q"], st["k"]
    if case["norm"]:
        q, k = _norm(q, st["q_norm"]), _norm(k, st["k_norm"])
    rows = pos.reshape(-1)[at]
    q, k = _rotate(q, st["cos"][rows], st["sin"][rows]), _rotate(k, st["cos"][rows], st["sin"][rows])
    keys, values = st["cache"]
    n = keys.shape[1] - t
    keys[:, n:] = torch.zeros(b * t, hkv, d, device=DEV).index_copy(0, at, k).reshape(b, t, hkv, d)
    values[:, n:] = torch.zeros(b * t, hkv, d, device=DEV).index_copy(0, at, st["v"]).reshape(b, t, hkv, d)
    qt = torch.zeros(b * t, hq, d, device=DEV).index_copy(0, at, q).reshape(b, t, hkv, hq // hkv, d)
    qt = qt.permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d).contiguous()
    scores = (qt @ keys.permute(0, 2, 3, 1).contiguous()).reshape(b, hkv, -1, t, n + t) * (1.0 / math.sqrt(d))
    past = torch.arange(n, device=DEV)
    seen = (past < first[:, None, None]).expand(b, t, n)
    if window:
        seen = seen & (past > pos[..., None] - window)
        up = up & (depth[:, None, :] > depth[..., None] - window)
    scores = scores.masked_fill(~torch.cat([seen, up], -1)[:, None, None], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    out = (p.reshape(b, hkv, -1, n + t) @ values.permute(0, 2, 1, 3).contiguous()).reshape(b, hkv, -1, t, d)
    out = out.permute(0, 3, 1, 2, 4).reshape(b * t, hq, d)[at]
    return [out, [list(r.split(st["nodes"])) for r in (k, st["v"])]]


def _plain_sample(st):
    x, rows = st["logits"], st["logits"].shape[0]
    col = lambda v: (v if torch.is_tensor(v) else torch.full((rows,), v, device=DEV)).double()[:, None]  # noqa: E731
    temperature, top_k, top_p, min_p = (col(st[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    v, order = x.sort(stable=True, dim=-1, descending=True)
    rank = torch.arange(x.shape[1], device=DEV)
    top_k = torch.where(top_k > 0, top_k, float(x.shape[1]))
    w = ((v.double() - v[:, :1].double()) / torch.where(temperature > 0, temperature, 1.0)).exp()
    w = torch.where(rank < torch.where(temperature > 0, top_k, 1.0), w, 0.0)
    run = w.cumsum(-1)
    w = torch.where((top_p >= 1) | (rank == 0) | (run - w < top_p * run[:, -1:]), w, 0.0)
    w = torch.where(w >= min_p, w, 0.0)
    kept = torch.zeros_like(w).scatter_(1, order, w)
    run = kept.cumsum(-1)
    token = (run <= st["u"].double()[:, None] * run[:, -1:]).sum(-1, keepdim=True)
    return [token[:, 0].int(), (kept.gather(1, token) / run[:, -1:])[:, 0].float()]


def _plain_accept(st):
    (b, t), at = st["shape"], st["at"]
    pad = lambda x, fill: torch.full((b * t,), fill, device=DEV, dtype=torch.int64).index_copy(0, at, x.long()).reshape(b, t)  # noqa: E731
    parents, tokens, sampled = pad(st["parents"], -1), pad(st["tokens"], -1), pad(st["sampled"], -2)
    up = parents.clamp(min=0)
    right = (parents >= 0) & (tokens == sampled.gather(1, up))
    # of siblings that hold the token the first
    twin = right[:, None, :] & (parents[:, None, :] == parents[..., None])
    node = torch.arange(t, device=DEV)
    taken = (right & ~(twin & (node < node[:, None])).any(-1)) | (node == 0)
    for _ in range((t - 1).bit_length()):
        taken, up = taken & taken.gather(1, up), up.gather(1, up)
    count = taken.sum(-1)
    path = torch.where(taken, node, t).sort(-1).values
    last = path.gather(1, count[:, None] - 1)
    path = torch.where(path < t, path, -1)
    return [path.reshape(-1)[at].int(), count.int(), sampled.gather(1, last)[:, 0].int()]


def _plain_keep(st):
    rows, b = st["rows"], st["count"].shape[0]
    t = rows.shape[2]
    node = torch.arange(t, device=DEV)
    of = torch.where(node < st["count"][:, None], st["path"].reshape(b, t).long(), node)
    of = of.repeat(rows.shape[0] // b, 1)[:, None, :, None, None].expand_as(rows)
    rows.copy_(rows.gather(2, of))
    return list(rows.flatten(0, 1).unbind(0))


# ---------------------------------------------------------------------------
# state and a pass

_sessions = []


def _session():
    """A program's one session, on a stream of its own."""
    if not _sessions:
        from spissa_amd.device import Session

        stream = torch.cuda.Stream()
        _sessions.append((Session(0, stream=stream), stream))
    return _sessions[0][0]


class _Rows:
    """Rows of a cache's keys or values as the tensor library takes them, in place; they hold the cache."""

    def __init__(self, cache, pointer, shape):
        self.cache = cache
        self.__cuda_array_interface__ = {"data": (pointer, False), "shape": tuple(shape), "typestr": "<f4", "version": 2}


def _view(cache, first, count):
    """A cache's rows first..first + count: keys and values."""
    h, d = cache.num_heads(), cache.head_dim()
    return [torch.as_tensor(_Rows(cache, p + first * h * d * 4, (count, h, d)), device=DEV) for p in (cache.device_keys_ptr(), cache.device_values_ptr())]


def _padded(rows, n):
    """Rows of several sequences as one tensor, the shorter ones filled up with zeros."""
    return torch.stack([torch.nn.functional.pad(r, (0, 0, 0, 0, 0, n - r.shape[0])) for r in rows])


def prepare(case, seed):
    inp = _inputs(case, seed)
    kind = case["kind"]
    st = {"case": case} | {n: v for n, v in inp.items() if not n.startswith("past")}
    if kind in ("tree", "accept"):
        st["nodes"] = nodes = _nodes(case)
        st["shape"] = (case["batch"], max(nodes))
        st["at"] = torch.cat([torch.arange(n, device=DEV) + i * max(nodes) for i, n in enumerate(nodes)])
    if kind == "tree":
        st["first"] = torch.tensor(_lens(case), device=DEV)
        at = _angles(case, torch.arange(max(_lens(case)) + max(nodes), device=DEV)).double()
        st["cos"], st["sin"] = at.cos().float(), at.sin().float()
    if own:
        _prepare_own(case, inp, st)
    elif kind == "tree":
        st["cache"] = [_padded(inp[t], max(_lens(case)) + max(st["nodes"])) for t in ("past_k", "past_v")]
    torch.cuda.synchronize()
    return st


def _prepare_own(case, inp, st):
    from spissa_amd import _ffi
    from spissa_amd.device import SamplingConfig
    from spissa_amd.rotary import KvAttentionConfig

    ses, kind = _session(), case["kind"]
    torch.cuda.synchronize()
    if kind == "sample":
        st["config"] = SamplingConfig(*(inp[n] for n in ("temperature", "top_k", "top_p", "min_p")))
        st["outputs"] = [torch.zeros(case["rows"], device=DEV, dtype=torch.int32), torch.zeros(case["rows"], device=DEV)]
    elif kind == "accept":
        n = len(inp["parents"])
        st["outputs"] = [torch.zeros(m, device=DEV, dtype=torch.int32) for m in (n, case["batch"], case["batch"])]
    elif kind == "keep":
        st["nodes"] = [case["nodes"]] * case["batch"]
        st["cache"], p = [], case["cached"]
        past = torch.zeros(p, case["kv"], case["dim"], device=DEV)
        torch.cuda.synchronize()
        for k, v in inp["rows"]:
            c = ses.kv_cache(case["kv"], case["dim"], p + case["nodes"] + 64)
            ses.append(c, past, past, p)
            ses.append(c, k, v, case["nodes"])
            st["cache"].append(c)
        ses.sync()
        st["outputs"] = [v for c in st["cache"] for v in _view(c, p, case["nodes"])]
    else:
        lens, nodes = _lens(case), st["nodes"]
        hq, kv, d = case["q"], case["kv"], case["dim"]
        st["config"] = KvAttentionConfig(sum(nodes), hq, kv, d, True, case["window"])
        st["table"] = ses.rope_table(_ffi.ROPE_GEMMA if case["norm"] else _ffi.ROPE_LLAMA, d, _base(case), max_positions=max(lens) + max(nodes))
        st["cache"] = []
        for k, v in zip(inp["past_k"], inp["past_v"]):
            c = ses.kv_cache(kv, d, len(k) + max(nodes) + 64)
            ses.append(c, k, v, len(k))
            st["cache"].append(c)
        ses.sync()
        rows = [_view(c, p, n) for c, p, n in zip(st["cache"], lens, nodes)]
        st["outputs"] = [torch.zeros_like(inp["q"]), [list(r) for r in zip(*rows)]]
        st["lens"] = lens


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"tree": _plain_tree, "sample": _plain_sample, "accept": _plain_accept, "keep": _plain_keep}[kind](state)
    ses, out = _session(), state["outputs"]
    if kind == "sample":
        ses.sample(state["logits"], state["u"], state["config"], *out)
    elif kind == "accept":
        ses.tree_accept(state["parents"], state["tokens"], state["sampled"], state["nodes"], *out)
    elif kind == "keep":
        ses.keep_rows(state["cache"], state["nodes"], state["path"], state["count"])
    else:
        for c, p in zip(state["cache"], state["lens"]):
            c.truncate(p)  # the nodes of the pass before
        what = (state["table"], state["q"], state["k"], state["v"], state["cache"], state["nodes"], state["parents"], state["config"])
        if state["case"]["norm"]:
            ses.gemma_tree_step(*what, state["q_norm"], state["k_norm"], EPS, 1.0, out[0])
        else:
            ses.tree_step(*what, out[0])
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 4 * n}
    if kind == "accept":
        return {"bytes": 16 * sum(_nodes(case)) + 8 * case["batch"], "flops": 2 * sum(_nodes(case))}
    kv, d = case["kv"], case["dim"]
    if kind == "keep":
        moved = case["layers"] * case["batch"] * (case["kept"] - 1)
        return {"bytes": 16 * moved * kv * d + 4 * case["batch"] * (case["kept"] + 1), "flops": 0}
    size, flops, window = 0, 0, case["window"]
    for p, parents in zip(_lens(case), _parents(case)):
        # queries in and out, new rows in and out, the cached rows that any node sees
        size += 8 * len(parents) * (case["q"] + 2 * kv) * d + 8 * kv * d * min(p, window - 1 if window else p)
        seen = sum(min(p + e + 1, window) if window else p + e + 1 for e in _depths(parents))
        flops += 4 * d * case["q"] * seen
    return {"bytes": size, "flops": flops}


# ---------------------------------------------------------------------------
# the same in 64 bits


def _turn_64(x, angles):
    """Channel i and i + d / 2 of rows [n, h, d] turned by their row's angle."""
    h = x.shape[-1] // 2
    c, s = torch.cos(angles.double()).unsqueeze(1), torch.sin(angles.double()).unsqueeze(1)
    out = torch.empty_like(x)
    out[..., :h] = x[..., :h] * c - x[..., h:] * s
    out[..., h:] = x[..., h:] * c + x[..., :h] * s
    return out


def _exact_tree(case, inp):
    hq, hkv, d, window = case["q"], case["kv"], case["dim"], case["window"]
    outs, rows_k, rows_v, at = [], [], [], 0
    for p, parents, pk, pv in zip(_lens(case), _parents(case), inp["past_k"], inp["past_v"]):
        n = len(parents)
        q, k, v = (inp[t][at:at + n].double() for t in "qkv")
        at += n
        if case["norm"]:
            q = q / torch.sqrt(torch.sum(q * q, -1, True) / d + EPS) * inp["q_norm"].double()
            k = k / torch.sqrt(torch.sum(k * k, -1, True) / d + EPS) * inp["k_norm"].double()
        depth = _depths(parents)
        turn = _angles(case, torch.tensor([p + e for e in depth], device=DEV))
        q, k = _turn_64(q, turn), _turn_64(k, turn)
        seen = torch.zeros(n, p + n, dtype=torch.bool)
        for t in range(n):
            seen[t, max(0, p + depth[t] - window + 1) if window else 0:p] = True
            a = t
            while a >= 0 and (not window or depth[t] - depth[a] < window):
                seen[t, p + a] = True
                a = parents[a]
        seen = seen.to(DEV)
        out = torch.empty(n, hq, d, dtype=torch.float64, device=DEV)
        for g in range(hkv):
            kk, vv = torch.cat([pk[:, g].double(), k[:, g]]), torch.cat([pv[:, g].double(), v[:, g]])
            kt = kk.t().contiguous()
            for h in range(g * hq // hkv, (g + 1) * hq // hkv):
                sc = torch.where(seen, q[:, h].contiguous() @ kt / math.sqrt(d), -math.inf)
                out[:, h] = torch.softmax(sc, -1) @ vv
        outs.append(out)
        rows_k.append(k)
        rows_v.append(v)
    return [torch.cat(outs), [rows_k, rows_v]]


def _exact_sample(case, inp):
    tokens, probs = [], []
    of = lambda n, i: float(inp[n][i]) if torch.is_tensor(inp[n]) else float(torch.tensor(inp[n], dtype=torch.float32))  # noqa: E731
    for i, x in enumerate(inp["logits"].double()):
        t, k, p, least = of("temperature", i), int(of("top_k", i)), of("top_p", i), of("min_p", i)
        best = x.max()
        if t == 0:
            tokens.append(int((x == best).nonzero()[0]))
            probs.append(1.0)
            continue
        w = torch.exp((x - best) / t)
        order = torch.sort(-x, stable=True).indices  # falling, equal ones by index
        if 0 < k < len(x):
            order = order[:k]
        if p < 1:
            before = torch.cumsum(w[order], 0) - w[order]
            order = order[:max(1, int((before < p * w[order].sum()).sum()))]
        order = order[w[order] >= least]
        index = torch.sort(order).values
        run = torch.cumsum(w[index], 0)
        j = int(torch.searchsorted(run, inp["u"][i].double() * run[-1], right=True))
        tokens.append(int(index[j]))
        probs.append(float(w[index[j]] / run[-1]))
    return [torch.tensor(tokens, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64)]


def _exact_accept(case, inp):
    paths, counts, nexts, at = [], [], [], 0
    for parents in _parents(case):
        n = len(parents)
        tokens, sampled = (inp[t][at:at + n].tolist() for t in ("tokens", "sampled"))
        at += n
        path = [0]
        while True:
            more = [t for t in range(n) if parents[t] == path[-1] and tokens[t] == sampled[path[-1]]]
            if not more:
                break
            path.append(more[0])
        paths += path + [-1] * (n - len(path))
        counts.append(len(path))
        nexts.append(sampled[path[-1]])
    return [torch.tensor(v, dtype=torch.int32) for v in (paths, counts, nexts)]


def exact(case, seed):
    inp = _inputs(case, seed)
    if case["kind"] == "tree":
        return _exact_tree(case, inp)
    if case["kind"] == "sample":
        return _exact_sample(case, inp)
    if case["kind"] == "accept":
        return _exact_accept(case, inp)
    out, t = [], case["nodes"]
    for i, rows in enumerate(inp["rows"].double()):
        b = i % case["batch"]
        path = inp["path"][b * t:(b + 1) * t].tolist()[:int(inp["count"][b])]
        for r in rows:
            out.append(torch.cat([r[path], r[len(path):]]))
    return out
