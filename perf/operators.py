"""Serving in four bits: the calls whose weights or whose cache hold 4-bit codes,
in elementary torch operations and through the entry points of `spissa_amd.device`.

Kinds:

  linear  a projection of weights held as 4-bit codes with a scale (and, if the
          checkpoint has them, a zero point) for each group of input channels:
          out = x W^T + bias,  W[n, k] = scale[n, k / group] * (code[n, k] - zero[n, k / group])
  append  rows of keys and values into a cache that holds them in 4 bits, and
          those rows back as the values they then stand for. Of each token and
          head, every 32 channels have a minimum and a step of their own:
          min = half(lo), step = half((hi - lo) * float(1 / 15)),
          code = clamp(rne((x - min) * (1 / step)), 0, 15), value = min + step * code
  attend  attention of one token of each of a batch of sequences over such caches
          (the token's own row is the cache's last)
  step    one sequence's decode step or prompt chunk: append, then attention of
          the new rows over the whole cache; the output and the appended rows

Head shapes are the Llama 3.2 and Gemma 3 ones that this repository's benchmark
uses, or generic.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
GROUP = 32  # channels of a row with one minimum and step

# query heads, KV heads, head dim
HEADS = {"llama1b": (32, 8, 64), "llama3b": (24, 8, 128), "gemma1b": (4, 1, 256), "gemma4b": (8, 4, 256)}
SCALES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # The key projection of the smallest model for one token: half a megabyte of codes, all latency.
        _linear("linear_key_1", 1, 512, 2048, 32, "f16", False, False),
        # A layer's largest matrix for one token, with the zero points of an asymmetric checkpoint.
        _linear("linear_down_1", 1, 2048, 8192, 128, "f16", True, False),
        # The tied table after the last layer of every generated token: 151 MB of codes.
        _linear("linear_table_1", 1, 262144, 1152, 64, "f16", False, False),
        # Sixteen sequences' tokens through one projection.
        _linear("linear_batch16", 16, 2560, 2048, 128, "bf16", False, True),
        # A ragged prompt, scales in single precision, channels that fill no whole group.
        _linear("linear_prompt_1500", 1500, 4097, 2500, 64, "f32", True, True),
        # The row of one generated token.
        {"name": "append_1", "kind": "append", "tokens": 1, "cached": 777, "kv": 8, "dim": 64},
        # A prompt's rows.
        {"name": "append_4096", "kind": "append", "tokens": 4096, "cached": 0, "kv": 8, "dim": 128},
        # Sixteen sequences of differing lengths, one launch.
        _attend("attend_batch16", "llama3b", 16, 8192, 0),
        # One KV head and a long context: all parallelism from the keys.
        _attend("attend_32768", "gemma1b", 1, 32768, 0),
        # A short chat turn's decode step.
        _step("step_decode_512", "llama1b", 1, 512, 0),
        # A new turn against a long resident cache.
        _step("step_chunk_512", "llama3b", 512, 7680, 0),
        # A prompt through a sliding-window layer.
        _step("step_prompt_2048", "gemma4b", 2048, 0, 1024),
    ]


def _linear(name, tokens, out, inner, group, scale, zeros, bias):
    return {"name": name, "kind": "linear", "tokens": tokens, "out": out, "in": inner, "group": group, "scale": scale,
            "zeros": zeros, "bias": bias}


def _attend(name, model, batch, cached, window):
    hq, hkv, d = HEADS[model]
    return {"name": name, "kind": "attend", "batch": batch, "cached": cached, "q": hq, "kv": hkv, "dim": d,
            "window": window}


def _step(name, model, tokens, cached, window):
    hq, hkv, d = HEADS[model]
    return {"name": name, "kind": "step", "tokens": tokens, "cached": cached, "q": hq, "kv": hkv, "dim": d,
            "window": window}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "append", "attend", "attend", "step", "step", "step"])
    if kind == "linear":
        inner, group = _log(rng, 48, 9000), rng.choice([32, 64, 128])
        out = _log(rng, 16, min(65536, 3.0e8 / inner))
        tokens = rng.choice([1, _log(rng, 2, 32), _log(rng, 16, max(17, min(2048, 1.5e10 / (inner * out))))])
        case = _linear("", tokens, out, inner, group, rng.choice(sorted(SCALES)), rng.random() < 0.5, rng.random() < 0.5)
        del case["name"]
        return case
    if kind == "append":
        d = rng.choice([64, 128, 256])
        kv = rng.randint(1, 16)
        return {"kind": kind, "tokens": _log(rng, 1, min(4096, 4.19e6 / (kv * d))), "cached": rng.choice([0, _log(rng, 1, 8192)]),
                "kv": kv, "dim": d}
    if rng.random() < 0.5:
        hq, kv, d = HEADS[rng.choice(sorted(HEADS))]
    else:
        kv, d = rng.randint(1, 8), rng.choice([64, 128, 256])
        hq = kv * rng.choice([1, 2, 3, 4, 5, 8])
    window = rng.choice([0, 0, _log(rng, 16, 2048)])
    case = {"kind": kind, "q": hq, "kv": kv, "dim": d, "window": window}
    if kind == "attend":
        batch = rng.choice([1, rng.randint(2, 16)])
        case |= {"batch": batch, "cached": _log(rng, 1, min(32768, 1.3e8 / (batch * kv * d)))}
        return case
    cached = rng.choice([0, _log(rng, 1, 8192)])
    most = int((math.sqrt(cached * cached + 4 * 1.0e8 / hq) - cached) / 2)  # (cached + tokens) * tokens scores a head
    case |= {"cached": cached, "tokens": rng.choice([1, _log(rng, 2, min(2048, max(2, most)))])}
    return case


# ---------------------------------------------------------------------------
# inputs


def _lens(case):
    """Rows of each sequence's cache: a batch's lengths spread down to a quarter of the longest, odd ones among them."""
    n, b = case["cached"], case["batch"]
    return [max(1, n - (3 * n * i) // (4 * b)) for i in range(b)]


def _inputs(case, seed):
    """Every input tensor of a case from the seed alone, the same for prepare() and exact()."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=DEV)  # noqa: E731
    if case["kind"] == "linear":
        m, n, k = case["tokens"], case["out"], case["in"]
        groups = -(-k // case["group"])
        # activations with a few channels far above the rest, as a layer's are
        x = normal(m, k) * torch.where(torch.rand(k, generator=gen, device=DEV) < 0.01, 20.0, 1.0)
        codes = torch.randint(0, 256, (n, (k + 1) // 2), generator=gen, device=DEV, dtype=torch.uint8)
        scales = ((0.5 + torch.rand(n, groups, generator=gen, device=DEV)) * 0.005).to(SCALES[case["scale"]])
        zeros = torch.randint(4, 13, (n, groups), generator=gen, device=DEV, dtype=torch.uint8) if case["zeros"] else None
        return {"x": x, "codes": codes, "scales": scales, "zeros": zeros, "bias": normal(n) if case["bias"] else None}
    kv, d = case["kv"], case["dim"]
    bk, bv = normal(kv, d), normal(kv, d) * 0.25  # channels' own offsets
    if case["kind"] == "attend":
        lens = _lens(case)
        return {"k": [normal(p, kv, d) + bk for p in lens], "v": [normal(p, kv, d) + bv for p in lens],
                "q": normal(case["batch"], case["q"], d)}
    p, s = case["cached"], case["tokens"]
    got = {"past_k": normal(p, kv, d) + bk, "past_v": normal(p, kv, d) + bv, "k": normal(s, kv, d) + bk, "v": normal(s, kv, d) + bv}
    if case["kind"] == "step":
        got["q"] = normal(s, case["q"], d)
    return got


# ---------------------------------------------------------------------------
# the plain form


def _pack(x):
    """Rows [..., d] as packed codes [..., d / 2] (even channels in the low four bits), steps and minima [..., d / 32]."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.amin(-1), g.amax(-1)
    low, step = lo.half(), ((hi - lo) * (1.0 / 15.0)).half()
    inv = torch.where(step > 0, 1.0 / step.float(), 0.0)
    code = ((g - low.float()[..., None]) * inv[..., None]).round().clamp(0, 15).to(torch.uint8).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), step, low


def _unpack(codes, step, low):
    """The rows that codes, steps and minima stand for."""
    c = torch.stack([codes & 15, codes >> 4], -1).float().reshape(*step.shape, GROUP)
    return (low.float()[..., None] + step.float()[..., None] * c).flatten(-2)


def _plain_linear(st):
    n, group, k = st["codes"].shape[0], st["group"], st["x"].shape[1]
    c = torch.stack([st["codes"] & 15, st["codes"] >> 4], -1).reshape(n, -1)[:, :k].float()
    z = 8.0 if st["zeros"] is None else st["zeros"].float().repeat_interleave(group, 1)[:, :k]
    out = st["x"] @ ((c - z) * st["scales"].float().repeat_interleave(group, 1)[:, :k]).t()
    return out if st["bias"] is None else out + st["bias"]


def _plain_attend(q, k, v, first, window):
    """q [b, s, hq, d] over k, v [b, n, hkv, d]; first [b]: the position of each sequence's first query."""
    b, s, hq, d = q.shape
    n, hkv = k.shape[1:3]
    qt = q.reshape(b, s, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d).contiguous()
    scores = (qt @ k.permute(0, 2, 3, 1).contiguous()).reshape(b, hkv, -1, s, n) * (1.0 / math.sqrt(d))
    at = first[:, None, None] + torch.arange(s, device=DEV)[None, :, None]
    key = torch.arange(n, device=DEV)[None, None, :]
    hidden = key > at
    if window:
        hidden = hidden | (key <= at - window)
    scores = scores.masked_fill(hidden[:, None, None], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    out = p.reshape(b, hkv, -1, n) @ v.permute(0, 2, 1, 3).contiguous()
    return out.reshape(b, hkv, -1, s, d).permute(0, 3, 1, 2, 4).reshape(b, s, hq, d)


def _plain(st):
    case = st["case"]
    if case["kind"] == "linear":
        return _plain_linear(st)
    if case["kind"] == "append":
        return [_unpack(*_pack(st["k"])), _unpack(*_pack(st["v"]))]
    if case["kind"] == "attend":
        return _plain_attend(st["q"][:, None], _unpack(*st["cache"][0]), _unpack(*st["cache"][1]), st["first"], case["window"])[:, 0]
    p, new = case["cached"], [_pack(st["k"]), _pack(st["v"])]
    for held, rows in zip(st["cache"], new):
        for t, r in zip(held, rows):
            t[0, p:] = r
    out = _plain_attend(st["q"][None], _unpack(*st["cache"][0]), _unpack(*st["cache"][1]), st["first"], case["window"])[0]
    return [out, _unpack(*new[0]), _unpack(*new[1])]


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


def _padded(rows, n):
    """Rows of several sequences as one tensor, the shorter ones filled up with zeros."""
    return torch.stack([torch.nn.functional.pad(r, (0, 0, 0, 0, 0, n - r.shape[0])) for r in rows])


def prepare(case, seed):
    inp = _inputs(case, seed)
    kind = case["kind"]
    st = {"case": case}
    if kind == "linear":
        st |= inp | {"group": case["group"]}
        if own:
            st["weight"] = _session().q4_linear_weight(inp["codes"], inp["scales"], case["out"], case["in"], case["group"],
                                                       inp["zeros"])
            st["outputs"] = torch.zeros(case["tokens"], case["out"], device=DEV)
        torch.cuda.synchronize()
        return st
    kv, d = case["kv"], case["dim"]
    st |= {t: inp[t] for t in ("k", "v", "q") if t in inp and kind != "attend" or t == "q" and t in inp}
    if kind == "attend":
        lens = _lens(case)
        st["first"] = torch.tensor([p - 1 for p in lens], device=DEV)
    elif kind == "step":
        st["first"] = torch.tensor([case["cached"]], device=DEV)
    if own:
        from spissa_amd.rotary import KvAttentionConfig

        ses = _session()
        if kind != "append":
            st["cfg"] = KvAttentionConfig(case.get("tokens", 1), case["q"], kv, d, True, case["window"])
        torch.cuda.synchronize()
        if kind == "attend":
            st["cache"] = []
            for rk, rv in zip(inp["k"], inp["v"]):
                c = ses.q4_kv_cache(kv, d, rk.shape[0] + 64)
                ses.append(c, rk, rv, rk.shape[0])
                st["cache"].append(c)
            st["outputs"] = torch.zeros_like(inp["q"])
        else:
            c = st["cache"] = ses.q4_kv_cache(kv, d, case["cached"] + case["tokens"] + 64)
            if case["cached"]:
                ses.append(c, inp["past_k"], inp["past_v"], case["cached"])
            st["outputs"] = ([torch.zeros_like(inp["q"])] if kind == "step" else []) + [torch.zeros_like(inp["k"]) for _ in range(2)]
    elif kind == "attend":
        st["cache"] = [_pack(_padded(inp[t], max(_lens(case)))) for t in ("k", "v")]
    elif kind == "step":
        rows = case["cached"] + case["tokens"]
        st["cache"] = [_pack(_padded([inp[t]], rows)) for t in ("past_k", "past_v")]
    torch.cuda.synchronize()
    return st


def run(state):
    if not own:
        return _plain(state)
    case, ses, out = state["case"], _session(), state["outputs"]
    kind = case["kind"]
    if kind == "linear":
        ses.linear(state["weight"], state["x"], state["bias"], case["tokens"], out)
    elif kind == "attend":
        ses.attention_cached_batch(state["q"], state["cache"], state["cfg"], out)
    else:
        c, p, s = state["cache"], case["cached"], case["tokens"]
        c.truncate(p)  # the rows of the pass before
        if kind == "append":
            ses.append(c, state["k"], state["v"], s)
        elif s == 1:
            ses.decode_step(None, state["q"], state["k"], state["v"], [c], state["cfg"], out[0])
        else:
            ses.prefill_step(None, state["q"], state["k"], state["v"], c, state["cfg"], out[0])
        ses.cache_rows(c, p, s, out[-2], out[-1])
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without


def _row_bytes(kv, d):
    """A token's keys or values in 4 bits: codes, and a minimum and a step for every 32 channels."""
    return kv * (d // 2 + d // GROUP * 4)


def _seen(first, s, window):
    """Visible (query, key) pairs of s queries at positions first.., and the rows that any of them sees."""
    pairs = sum(min(p + 1, window) if window else p + 1 for p in range(first, first + s))
    return pairs, min(first + s, window + s - 1) if window else first + s


def work(case):
    kind = case["kind"]
    if kind == "linear":
        m, n, k = case["tokens"], case["out"], case["in"]
        groups = -(-k // case["group"])
        size = n * ((k + 1) // 2) + n * groups * (4 if case["scale"] == "f32" else 2) + (n * groups // 2 if case["zeros"] else 0)
        return {"bytes": size + 4 * m * (n + k) + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    kv, d = case["kv"], case["dim"]
    if kind == "attend":
        size = flops = 0
        for p in _lens(case):
            pairs, rows = _seen(p - 1, 1, case["window"])
            size += 2 * rows * _row_bytes(kv, d) + 8 * case["q"] * d
            flops += 4 * d * case["q"] * pairs
        return {"bytes": size, "flops": flops}
    s = case["tokens"]
    # new rows read in f32, held in 4 bits, and given back
    size = 2 * s * (8 * kv * d + _row_bytes(kv, d))
    if kind == "append":
        return {"bytes": size, "flops": 8 * s * kv * d}
    pairs, rows = _seen(case["cached"], s, case["window"])
    size += 2 * max(0, rows - s) * _row_bytes(kv, d) + 8 * s * case["q"] * d
    return {"bytes": size, "flops": 4 * d * case["q"] * pairs}


# ---------------------------------------------------------------------------
# the same in 64 bits


def _held(x):
    """The values that rows stand for once held in 4 bits. The codes' decisions are single precision, as the format defines them."""
    d = x.shape[-1]
    out = torch.empty_like(x, dtype=torch.float64)
    for c in range(0, d, GROUP):
        part = x[..., c:c + GROUP]
        lo, hi = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        base = lo.to(torch.float16).float()
        width = ((hi - lo) * torch.tensor(1 / 15, dtype=torch.float32, device=DEV)).to(torch.float16).float()
        code = torch.where(width > 0, torch.round((part - base) * torch.reciprocal(width)), torch.zeros_like(part))
        code = torch.minimum(torch.maximum(code, torch.zeros_like(code)), torch.full_like(code, 15.0))
        out[..., c:c + GROUP] = base.double() + width.double() * code.double()
    return out


def _attend_64(q, keys, values, first, window):
    """q [s, hq, d] at positions first.. over keys, values [n, hkv, d], head by head."""
    s, hq, d = q.shape
    n, hkv = keys.shape[:2]
    dist = (first + torch.arange(s, device=DEV))[:, None] - torch.arange(n, device=DEV)[None, :]
    seen = (dist >= 0) & (dist < window if window else True)
    out = torch.empty(s, hq, d, dtype=torch.float64, device=DEV)
    for h in range(hq):
        k, v = keys[:, h * hkv // hq].contiguous(), values[:, h * hkv // hq].contiguous()
        sc = torch.where(seen, q[:, h].double() @ k.t().contiguous() / math.sqrt(d), -math.inf)
        out[:, h] = torch.softmax(sc, -1) @ v
    return out


def exact(case, seed):
    inp = _inputs(case, seed)
    if case["kind"] == "linear":
        k, parts = case["in"], []
        of = torch.arange(k, device=DEV) // case["group"]
        rows = max(1, 40_000_000 // k)
        for a in range(0, case["out"], rows):
            b = inp["codes"][a:a + rows].to(torch.int64)
            code = torch.empty(b.shape[0], 2 * b.shape[1], dtype=torch.float64, device=DEV)
            code[:, 0::2], code[:, 1::2] = b % 16, b // 16
            zero = 8 if inp["zeros"] is None else inp["zeros"][a:a + rows].double()[:, of]
            w = (code[:, :k] - zero) * inp["scales"][a:a + rows].double()[:, of]
            parts.append(inp["x"].double() @ w.t().contiguous())
        out = torch.cat(parts, 1)
        return out if inp["bias"] is None else out + inp["bias"].double()
    if case["kind"] == "append":
        return [_held(inp["k"]), _held(inp["v"])]
    if case["kind"] == "attend":
        return torch.cat([_attend_64(inp["q"][i:i + 1], _held(inp["k"][i]), _held(inp["v"][i]), p - 1, case["window"])
                          for i, p in enumerate(_lens(case))])
    new = [_held(inp["k"]), _held(inp["v"])]
    keys, values = (torch.cat([_held(inp["past_" + t]), r]) for t, r in zip("kv", new))
    return [_attend_64(inp["q"], keys, values, case["cached"], case["window"]), new[0], new[1]]
