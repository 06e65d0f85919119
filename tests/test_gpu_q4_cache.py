"""The KV cache held in 4 bits: rows in and back bit for bit, and the attention
over it against 64-bit sums over the same held rows.

Attention tolerance. A score is a sum of D products, in f32, over at most 16
products, log2(D / 16) exchanges, the step and the minimum: 24 roundings of at
most 2^-24 of sum |q k| / sqrt(D), which for these N(0, 1) rows (channel offsets
included) stays under 28 at D 256. That is 4e-5 in a score, twice that in a
weight against the others; the weighted sum adds roundings that average out.
So 8e-5 of the largest |value|, about twice the largest output.
"""
import numpy as np
import pytest
import torch

import oracle as o
import spissa_amd as sa
from spissa_amd.device import Session
from spissa_amd.rotary import KvAttentionConfig
from tests.helpers import assert_bitwise as flat_bitwise
from tests.q4 import attend, hold

pytestmark = pytest.mark.gpu

TOL = 8e-5


def assert_bitwise(got, ref, what=""):
    assert got.shape == ref.shape, what
    flat_bitwise(got.ravel(), ref.ravel(), what)


def rows(rng, n, h, d, spread=1.0):
    """Rows with an offset of their own for each channel, as keys have."""
    off = rng.standard_normal((h, d)).astype(np.float32)
    return (rng.standard_normal((n, h, d)).astype(np.float32) * np.float32(spread) + off).astype(np.float32)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.fixture(scope="module")
def ses(gpu):
    # the tests' own tensors are made, filled and freed on the session's stream
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        yield Session(0, stream=stream)


def held(ses, cache, first=0, n=None):
    n = len(cache) - first if n is None else n
    k = torch.full((n, cache.num_heads(), cache.head_dim()), np.nan, device="cuda")
    v = torch.full_like(k, np.nan)
    ses.cache_rows(cache, first, n, k, v)
    ses.sync()
    return k.cpu().numpy(), v.cpu().numpy()


def filled(ses, rng, n, hkv, d, room=0):
    """A cache of n rows, and the values they stand for."""
    k, v = rows(rng, n, hkv, d), rows(rng, n, hkv, d, 0.5)
    c = ses.q4_kv_cache(hkv, d, n + room)
    ses.append(c, dev(k), dev(v), n)
    return c, hold(k), hold(v)


def check(got, ref, values, what):
    got = got.cpu().numpy().astype(np.float64).reshape(ref.shape)
    err = np.max(np.abs(got - ref)) / np.max(np.abs(values))
    print(f"[q4] {what}: {err:.2e}", flush=True)
    assert err <= TOL, (what, err)


# ---- rows ----

@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,h", [(1, 1), (1, 8), (3, 5), (33, 2), (257, 3)])
def test_rows_come_back_as_the_format_has_them(ses, d, n, h):
    rng = np.random.default_rng(n * 1000 + h * 10 + d)
    k, v = rows(rng, n, h, d), rows(rng, n, h, d, 0.02)
    c = ses.q4_kv_cache(h, d, n + 7)
    ses.append(c, dev(k), dev(v), n)
    gk, gv = held(ses, c)
    assert_bitwise(gk, hold(k), "keys")
    assert_bitwise(gv, hold(v), "values")
    assert_bitwise(c.keys(), hold(k).ravel(), "keys on the host")
    assert_bitwise(c.values(), hold(v).ravel(), "values on the host")
    assert c.resident_bytes() == 2 * n * h * (d // 2 + d // 8)


def test_rows_of_every_kind(ses):
    """Constant groups, zeros of both signs, the range's ends, steps below binary16's normal numbers."""
    rng = np.random.default_rng(5)
    k = np.zeros((8, 2, 64), np.float32)
    k[0] = 3.25
    k[1] = -0.0
    k[2, :, ::2], k[2, :, 1::2] = 65504.0, -65504.0
    k[3] = rng.standard_normal((2, 64)) * 1e-5
    k[4] = rng.standard_normal((2, 64)) * 1e-9
    k[5] = 1000.0 + rng.standard_normal((2, 64)) * 0.01
    k[6] = rng.standard_normal((2, 64)) * 1e4
    k[7] = np.repeat(np.arange(16, dtype=np.float32) / 2, 4)[:64] - 1  # halfway cases of the rounding
    c = ses.q4_kv_cache(2, 64, 8)
    ses.append(c, dev(k), dev(-k), 8)
    gk, gv = held(ses, c)
    assert_bitwise(gk, hold(k), "keys")
    assert_bitwise(gv, hold(-k), "values")


def test_rows_in_pieces_truncated_and_written_again(ses):
    rng = np.random.default_rng(6)
    k, v = rows(rng, 40, 3, 128), rows(rng, 40, 3, 128)
    c = ses.q4_kv_cache(3, 128, 40)
    for a, b in ((0, 1), (1, 18), (18, 40)):
        ses.append(c, dev(k[a:b]), dev(v[a:b]), b - a)
    gk, gv = held(ses, c)
    assert_bitwise(gk, hold(k), "keys")
    twin = c.clone()
    c.truncate(17)
    k2, v2 = rows(rng, 5, 3, 128), rows(rng, 5, 3, 128)
    c.append(k2.ravel(), v2.ravel(), 5)  # host rows
    gk, gv = held(ses, c)
    assert_bitwise(gk, hold(np.concatenate([k[:17], k2])), "keys written again")
    assert_bitwise(gv, hold(np.concatenate([v[:17], v2])), "values written again")
    gk, _ = held(ses, twin)
    assert_bitwise(gk, hold(k), "the clone keeps its rows")
    assert isinstance(twin, sa.Q4KvCache) and len(twin) == 40
    gk, _ = held(ses, twin, 39, 1)
    assert_bitwise(gk, hold(k[39:]), "one row")


def test_f32_caches_give_their_rows_too(ses):
    rng = np.random.default_rng(8)
    k, v = rows(rng, 12, 2, 64), rows(rng, 12, 2, 64)
    c = ses.kv_cache(2, 64, 12)
    ses.append(c, dev(k), dev(v), 12)
    gk, gv = held(ses, c, 4, 5)
    assert_bitwise(gk, k[4:9], "keys")
    assert_bitwise(gv, v[4:9], "values")


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 65520.0, 1e30])
def test_values_outside_the_format(ses, bad):
    k = np.ones((2, 2, 64), np.float32)
    v = k.copy()
    v[1, 1, 40] = bad
    c = ses.q4_kv_cache(2, 64, 4)
    with pytest.raises(sa.InvalidTensorDataError):
        c.append(k.ravel(), v.ravel(), 2)
    assert len(c) == 0
    ses.append(c, dev(k), dev(v), 2)
    with pytest.raises(sa.InvalidTensorDataError):
        ses.sync()
    ses.sync()
    _, gv = held(ses, c)
    assert np.isfinite(gv).all()


def test_heads_past_four_gigabytes(ses):
    rng = np.random.default_rng(9)
    c = ses.q4_kv_cache(3, 256, 1 << 24)  # 2 GiB of codes a head
    k, v = rows(rng, 70, 3, 256), rows(rng, 70, 3, 256)
    ses.append(c, dev(k), dev(v), 70)
    gk, gv = held(ses, c)
    assert_bitwise(gk, hold(k), "keys")
    assert_bitwise(gv, hold(v), "values")
    q = rng.standard_normal((5, 6, 256)).astype(np.float32)
    out = torch.empty(5, 6, 256, device="cuda")
    ses.attention_cached(dev(q), c, KvAttentionConfig(5, 6, 3, 256, True), out)
    ses.sync()
    check(out, attend(q, hold(k), hold(v)), hold(v), "heads past 4 GiB")


# ---- attention of single tokens ----

@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 2), (9, 3), (8, 2), (5, 1), (7, 1), (16, 2)])
@pytest.mark.parametrize("n", [1, 2, 31, 129, 1030])
def test_one_token(ses, d, hq, hkv, n):
    rng = np.random.default_rng(d + 17 * hq + n)
    c, k, v = filled(ses, rng, n, hkv, d)
    q = rng.standard_normal((1, hq, d)).astype(np.float32)
    for window in (0, 1, 30, 2000):
        out = torch.full((1, hq, d), np.nan, device="cuda")
        ses.attention_cached(dev(q), c, KvAttentionConfig(1, hq, hkv, d, True, window), out)
        ses.sync()
        check(out, attend(q, k, v, True, window), v, f"d {d} heads {hq}/{hkv} n {n} window {window}")


@pytest.mark.parametrize("n", [8192, 40001])
def test_one_token_long(ses, n):
    rng = np.random.default_rng(n)
    c, k, v = filled(ses, rng, n, 1, 128)
    q = rng.standard_normal((1, 3, 128)).astype(np.float32) * 3
    out = torch.empty(1, 3, 128, device="cuda")
    for window in (0, 4097):
        ses.attention_cached(dev(q), c, KvAttentionConfig(1, 3, 1, 128, True, window), out)
        ses.sync()
        check(out, attend(q, k, v, True, window), v, f"n {n} window {window}")


@pytest.mark.parametrize("d,hq,hkv", [(64, 32, 8), (128, 6, 2), (256, 4, 1)])
@pytest.mark.parametrize("batch", [2, 16, 19])
def test_batch_of_ragged_caches(ses, d, hq, hkv, batch):
    rng = np.random.default_rng(batch + d)
    lens = [1 + int(x) for x in rng.integers(0, 700, batch)]
    lens[0], lens[-1] = 1, 700
    made = [filled(ses, rng, n, hkv, d) for n in lens]
    made[1] = made[0]  # two queries of one context
    q = rng.standard_normal((batch, hq, d)).astype(np.float32)
    for window in (0, 64):
        out = torch.full((batch, hq, d), np.nan, device="cuda")
        ses.attention_cached_batch(dev(q), [m[0] for m in made], KvAttentionConfig(1, hq, hkv, d, True, window), out)
        ses.sync()
        for b, (_, k, v) in enumerate(made):
            check(out[b], attend(q[b:b + 1], k, v, True, window)[0], v, f"sequence {b} of {lens[b]} rows window {window}")


def test_no_sequences(ses):
    out = torch.zeros(1, 2, 64, device="cuda")
    ses.attention_cached_batch(out, [], KvAttentionConfig(1, 2, 2, 64, True), out)
    ses.sync()


# ---- attention of several tokens ----

CHUNKS = [(2, 0), (3, 5), (16, 0), (17, 63), (64, 64), (65, 200), (130, 1), (200, 1000)]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (4, 2), (6, 2), (8, 2), (5, 1)])
@pytest.mark.parametrize("s,past", CHUNKS)
def test_chunks(ses, d, hq, hkv, s, past):
    rng = np.random.default_rng(d + 31 * s + past + hq)
    c, k, v = filled(ses, rng, s + past, hkv, d, room=3)
    q = rng.standard_normal((s, hq, d)).astype(np.float32)
    for causal, window in ((True, 0), (True, 1), (True, 50), (False, 0), (False, 40)):
        out = torch.full((s, hq, d), np.nan, device="cuda")
        ses.attention_cached(dev(q), c, KvAttentionConfig(s, hq, hkv, d, causal, window), out)
        ses.sync()
        check(out, attend(q, k, v, causal, window), v, f"d {d} heads {hq}/{hkv} {s}+{past} causal {causal} window {window}")


def test_long_prompt(ses):
    rng = np.random.default_rng(12)
    c, k, v = filled(ses, rng, 1500, 2, 128)
    q = rng.standard_normal((1500, 6, 128)).astype(np.float32)
    out = torch.empty(1500, 6, 128, device="cuda")
    ses.attention_cached(dev(q), c, KvAttentionConfig(1500, 6, 2, 128, True), out)
    ses.sync()
    check(out, attend(q, k, v), v, "prompt")


@pytest.mark.parametrize("scale", [1e-3, 300.0])
def test_values_of_any_size(ses, scale):
    """Values far from 1, and a row far beyond the others, keep their digits."""
    rng = np.random.default_rng(13)
    k, v = rows(rng, 150, 2, 64), (rows(rng, 150, 2, 64) * scale).astype(np.float32)
    c = ses.q4_kv_cache(2, 64, 150)
    big = np.full((1, 2, 64), 60000.0, np.float32)
    ses.append(c, dev(big), dev(big), 1)  # rolled back: only the rows that stay count
    c.truncate(0)
    ses.append(c, dev(k), dev(v), 150)
    q = rng.standard_normal((150, 4, 64)).astype(np.float32)
    out = torch.empty(150, 4, 64, device="cuda")
    ses.attention_cached(dev(q), c, KvAttentionConfig(150, 4, 2, 64, True), out)
    ses.sync()
    check(out, attend(q, hold(k), hold(v)), hold(v), f"values of {scale}")


def test_large_scores(ses):
    """Queries and keys whose scores reach hundreds: one key takes all the weight."""
    rng = np.random.default_rng(14)
    c, k, v = filled(ses, rng, 90, 1, 64)
    q = (rng.standard_normal((40, 2, 64)) * 256).astype(np.float32)
    q[:20] = np.rint(q[:20])
    out = torch.empty(40, 2, 64, device="cuda")
    ses.attention_cached(dev(q), c, KvAttentionConfig(40, 2, 1, 64, True), out)
    ses.sync()
    ref = attend(q, k, v)
    # a score's error grows with it: 256 times the tolerance's sum |q k|
    err = np.max(np.abs(out.cpu().numpy() - ref)) / np.max(np.abs(v))
    assert err <= 256 * TOL, err


def test_nan_query_is_reported(ses):
    rng = np.random.default_rng(15)
    c, _, _ = filled(ses, rng, 40, 1, 64)
    for s in (1, 5):
        q = np.ones((s, 2, 64), np.float32)
        q[s - 1, 1, 3] = np.nan
        out = torch.empty(s, 2, 64, device="cuda")
        ses.attention_cached(dev(q), c, KvAttentionConfig(s, 2, 1, 64, True), out)
        with pytest.raises(sa.InvalidTensorDataError):
            ses.sync()
    ses.sync()


# ---- fused steps ----

@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 2), (128, 6, 2), (256, 4, 1)])
@pytest.mark.parametrize("s,past", [(1, 0), (1, 77), (5, 0), (70, 33)])
def test_llama_step(ses, d, hq, hkv, s, past):
    rng = np.random.default_rng(d + s + past)
    c, k0, v0 = filled(ses, rng, past, hkv, d, s) if past else (ses.q4_kv_cache(hkv, d, s), np.zeros((0, hkv, d)), np.zeros((0, hkv, d)))
    q, k, v = rows(rng, s, hq, d), rows(rng, s, hkv, d), rows(rng, s, hkv, d)
    table = ses.rope_table(0, d, 500000.0, max_positions=past + s)
    cfg = KvAttentionConfig(s, hq, hkv, d, True)
    out = torch.full((s, hq, d), np.nan, device="cuda")
    dq, dk, dv = dev(q), dev(k), dev(v)
    if s == 1:
        ses.decode_step(table, dq, dk, dv, [c], cfg, out)
    else:
        ses.prefill_step(table, dq, dk, dv, c, cfg, out)
    ses.sync()
    qr, kr = q.ravel().copy(), k.ravel().copy()
    sa.apply_llama_rotary_inplace(qr, kr, hq, hkv, sa.RotaryEmbeddingConfig(s, hq, d, d, 500000.0, past))
    gk, gv = held(ses, c, past, s)
    assert len(c) == past + s
    assert_bitwise(gk, hold(kr.reshape(s, hkv, d)), "appended keys")
    assert_bitwise(gv, hold(v), "appended values")
    assert_bitwise(dq.cpu().numpy(), q, "q is read only")
    ref = attend(qr.reshape(s, hq, d), np.concatenate([k0, gk]), np.concatenate([v0, gv]))
    check(out, ref, np.concatenate([v0, gv]), f"step {s}+{past}")


@pytest.mark.parametrize("s,past", [(1, 50), (40, 50)])
def test_gemma_step(ses, s, past):
    d, hq, hkv, eps = 256, 4, 2, 1e-6
    rng = np.random.default_rng(s + past)
    c, k0, v0 = filled(ses, rng, past, hkv, d, s)
    q, k, v = rows(rng, s, hq, d), rows(rng, s, hkv, d), rows(rng, s, hkv, d)
    qn, kn = (1 + 0.1 * rng.standard_normal((2, d))).astype(np.float32)
    table = ses.rope_table(1, d, 10000.0, 8.0, max_positions=past + s)
    cfg = KvAttentionConfig(s, hq, hkv, d, True, 64)
    out = torch.empty(s, hq, d, device="cuda")
    args = (table, dev(q), dev(k), dev(v))
    if s == 1:
        ses.gemma_decode_step(*args, [c], cfg, dev(qn), dev(kn), eps, 0.5, out)
    else:
        ses.gemma_prefill_step(*args, c, cfg, dev(qn), dev(kn), eps, 0.5, out)
    ses.sync()
    qr = sa.rms_norm(q.ravel(), qn, s * hq, d, eps)
    kr = sa.rms_norm(k.ravel(), kn, s * hkv, d, eps)
    sa.apply_gemma_rotary_inplace(qr, kr, hq, hkv, sa.RotaryEmbeddingConfig(s, hq, d, d, 10000.0, past), 8.0)
    gk, gv = held(ses, c, past, s)
    assert_bitwise(gv, hold(v), "appended values")
    want = hold(kr.reshape(s, hkv, d))
    # the norm's sum is a tree: a key may differ in its last place, and so land one code beside a tie
    step = np.repeat((kr.reshape(-1, 32).max(1) - kr.reshape(-1, 32).min(1)) / 15, 32).reshape(want.shape)
    assert np.all(np.abs(gk - want) <= 1.01 * step + 1e-3 * np.abs(want))
    assert np.mean(np.abs(gk - want) > 1e-2 * step + 2e-3 * np.abs(want)) <= 1e-3
    ref = attend((qr * np.float32(0.5)).reshape(s, hq, d), np.concatenate([k0, gk]), np.concatenate([v0, gv]), True, 64)
    check(out, ref, np.concatenate([v0, gv]), f"gemma step {s}+{past}")


def test_batched_decode_steps(ses):
    d, hq, hkv, batch = 64, 4, 2, 18
    rng = np.random.default_rng(20)
    made = [filled(ses, rng, 1 + 13 * b, hkv, d, 2) for b in range(batch)]
    keep = [[m[1], m[2]] for m in made]
    cfg = KvAttentionConfig(1, hq, hkv, d, True)
    for _ in range(2):
        q, k, v = rows(rng, batch, hq, d), rows(rng, batch, hkv, d), rows(rng, batch, hkv, d)
        out = torch.empty(batch, hq, d, device="cuda")
        ses.decode_step(None, dev(q), dev(k), dev(v), [m[0] for m in made], cfg, out)
        ses.sync()
        for b in range(batch):
            keep[b][0] = np.concatenate([keep[b][0], hold(k[b:b + 1])])
            keep[b][1] = np.concatenate([keep[b][1], hold(v[b:b + 1])])
            check(out[b], attend(q[b:b + 1], *keep[b])[0], keep[b][1], f"sequence {b}")


def test_chunks_of_a_prompt_agree(ses):
    """A prompt in one step, in chunks, and token by token: the same rows, the same outputs to rounding."""
    d, hq, hkv, n = 64, 4, 2, 90
    rng = np.random.default_rng(21)
    q, k, v = rows(rng, n, hq, d), rows(rng, n, hkv, d), rows(rng, n, hkv, d)
    table = ses.rope_table(0, d, 10000.0, max_positions=n)
    outs = []
    for parts in ([n], [33, 1, 56], [1] * n):
        c, at, got = ses.q4_kv_cache(hkv, d, n), 0, []
        for s in parts:
            out = torch.empty(s, hq, d, device="cuda")
            ses.prefill_step(table, dev(q[at:at + s]), dev(k[at:at + s]), dev(v[at:at + s]), c,
                             KvAttentionConfig(s, hq, hkv, d, True), out)
            got.append(out)
            at += s
        ses.sync()
        outs.append((torch.cat(got).cpu().numpy(), *held(ses, c)))
    for other in outs[1:]:
        assert_bitwise(other[1], outs[0][1], "keys")
        assert_bitwise(other[2], outs[0][2], "values")
        assert np.max(np.abs(other[0] - outs[0][0])) <= 2 * TOL * np.max(np.abs(v))


# ---- streams, capture, refusals ----

def test_captured_step_replays(ses):
    """A step and the attention in a graph, replayed with eager work between."""
    d, hq, hkv = 128, 6, 2
    rng = np.random.default_rng(22)
    stream = torch.cuda.Stream()
    own = Session(0, stream=stream)
    c, k0, v0 = filled(own, rng, 600, hkv, d, 1)
    table = own.rope_table(0, d, 10000.0, max_positions=700)
    cfg = KvAttentionConfig(1, hq, hkv, d, True)
    q, k, v = (dev(rows(rng, 1, h, d)) for h in (hq, hkv, hkv))
    out = torch.empty(1, hq, d, device="cuda")
    torch.cuda.synchronize()

    def step():
        c.truncate(600)
        own.decode_step(table, q, k, v, [c], cfg, out)

    with torch.cuda.stream(stream):
        step()
    own.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for _ in range(3):
        nq, nk, nv = rows(rng, 1, hq, d), rows(rng, 1, hkv, d), rows(rng, 1, hkv, d)
        q.copy_(dev(nq))
        k.copy_(dev(nk))
        v.copy_(dev(nv))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        own.sync()
        got = out.clone()
        with torch.cuda.stream(stream):
            step()
        own.sync()
        assert_bitwise(got.cpu().numpy(), out.cpu().numpy(), "replay against eager")
        qr, kr = nq.ravel().copy(), nk.ravel().copy()
        sa.apply_llama_rotary_inplace(qr, kr, hq, hkv, sa.RotaryEmbeddingConfig(1, hq, d, d, 10000.0, 600))
        keys = np.concatenate([k0, hold(kr.reshape(1, hkv, d))])
        check(got, attend(qr.reshape(1, hq, d), keys, np.concatenate([v0, hold(nv)])), v0, "replay")


def test_same_results_on_every_call(ses):
    rng = np.random.default_rng(23)
    c, _, _ = filled(ses, rng, 3000, 2, 128)
    for s in (1, 40):
        q = dev(rng.standard_normal((s, 6, 128)).astype(np.float32))
        outs = []
        for _ in range(3):
            out = torch.empty(s, 6, 128, device="cuda")
            ses.attention_cached(q, c, KvAttentionConfig(s, 6, 2, 128, True), out)
            ses.sync()
            outs.append(out.cpu().numpy())
        assert_bitwise(outs[1], outs[0])
        assert_bitwise(outs[2], outs[0])


def test_refusals(ses):
    d, hq, hkv = 64, 4, 2
    rng = np.random.default_rng(24)
    c, _, _ = filled(ses, rng, 10, hkv, d, 2)
    full = filled(ses, rng, 3, hkv, d)[0]
    empty = ses.q4_kv_cache(hkv, d, 4)
    f32 = ses.kv_cache(hkv, d, 16)
    t = torch.zeros(4, hq, d, device="cuda")
    one = KvAttentionConfig(1, hq, hkv, d, True)
    two = KvAttentionConfig(2, hq, hkv, d, True)
    table = ses.rope_table(0, d, 10000.0, max_positions=5)
    odd = torch.zeros(4 * hq * d + 1, device="cuda")[1:]
    neox = ses.rope_table(2, d // 2, 10000.0, max_positions=64)
    for exc, call in [
        (sa.ArgumentError, lambda: ses.attention(t, t, t, c, one, t)),
        (sa.ArgumentError, lambda: ses.attention_decode_batch(t, t, t, [c], one, t)),
        (sa.ArgumentError, lambda: ses.decode_step_noalloc(None, t, t, t, [c], one, t)),
        (sa.ArgumentError, lambda: ses.attention_cached_batch(t, [f32], one, t)),
        (sa.ArgumentError, lambda: ses.decode_step(None, t, t, t, [c, f32], one, t)),
        (sa.ArgumentError, lambda: ses.decode_step(None, t, t, t, [c, c], one, t)),
        (sa.ArgumentError, lambda: ses.attention_cached(odd, c, one, t)),
        (sa.ArgumentError, lambda: ses.decode_step(None, t, odd, t, [c], one, t)),
        (sa.ArgumentError, lambda: ses.append(c, odd, t, 1)),
        (sa.ArgumentError, lambda: ses.cache_rows(c, 0, 1, odd, t)),
        (sa.ShapeError, lambda: ses.attention_cached_batch(t, [empty], one, t)),
        (sa.ShapeError, lambda: ses.attention_cached_batch(t, [c], two, t)),
        (sa.ShapeError, lambda: ses.attention_cached(t, empty, one, t)),
        (sa.ShapeError, lambda: ses.attention_cached(t, c, KvAttentionConfig(11, hq, hkv, d, True), t)),
        (sa.ShapeError, lambda: ses.attention_cached(t, c, KvAttentionConfig(1, hq, hkv, 128, True), t)),
        (sa.ShapeError, lambda: ses.attention_cached(t, c, KvAttentionConfig(1, 3, 2, d, True), t)),
        (sa.ShapeError, lambda: ses.decode_step(None, t, t, t, [full], one, t)),
        (sa.ShapeError, lambda: ses.decode_step(None, t, t, t, [c], two, t)),
        (sa.ShapeError, lambda: ses.decode_step(table, t, t, t, [c], one, t)),
        (sa.ShapeError, lambda: ses.decode_step(neox, t, t, t, [c], one, t)),
        (sa.ShapeError, lambda: ses.prefill_step(None, t, t, t, full, two, t)),
        (sa.ShapeError, lambda: ses.append(full, t, t, 1)),
        (sa.ShapeError, lambda: ses.append(c, t, t, 0)),
        (sa.ShapeError, lambda: ses.cache_rows(c, 8, 3, t, t)),
        (TypeError, lambda: ses.cache_rows(c, 0, 10, t[0, 0], t)),
        (sa.ShapeError, lambda: c.truncate(11)),
    ]:
        with pytest.raises(exc):
            call()
    host = np.zeros(hq * d, np.float32)
    with pytest.raises(sa.ArgumentError):
        sa.scaled_dot_product_attention_with_cache(host, host[:hkv * d], host[:hkv * d], c, one)
    assert len(c) == 10 and len(full) == 3 and len(empty) == 0
    assert not c.device_keys_ptr() and not c.device_values_ptr()
    ses.sync()


def test_more_rows_than_a_launch_takes(ses):
    """Refused before anything runs: the small tensors are never read."""
    n, t = 140000, torch.zeros(64, device="cuda")
    c = ses.q4_kv_cache(1, 64, n)
    cfg = KvAttentionConfig(n, 64, 1, 64, True)
    with pytest.raises(sa.ShapeError):
        ses.prefill_step(None, t, t, t, c, cfg, t)
    assert len(c) == 0
    k = torch.zeros(n, 64, device="cuda")
    ses.append(c, k, k, n)
    with pytest.raises(sa.ShapeError):
        ses.attention_cached(t, c, cfg, t)
    ses.sync()


@pytest.mark.parametrize("d,hq,hkv", [(64, 32, 2), (64, 3, 3), (128, 12, 1), (128, 6, 2), (256, 8, 1), (256, 3, 1)])
@pytest.mark.parametrize("size", [1.0, 3000.0])
def test_steps_over_several_key_ranges(ses, d, hq, hkv, size):
    """A ragged batch whose longest caches are split, with a new value row far beyond the held ones."""
    rng = np.random.default_rng(d + hq)
    lens = [0, 1, 255, 900, 2600]
    made = [filled(ses, rng, n, hkv, d, 1) if n else
            (ses.q4_kv_cache(hkv, d, 1), np.zeros((0, hkv, d)), np.zeros((0, hkv, d))) for n in lens]
    b = len(lens)
    q, k, v = rows(rng, b, hq, d), rows(rng, b, hkv, d), (rows(rng, b, hkv, d) * np.float32(size)).astype(np.float32)
    for window in (0, 1000):
        out = torch.full((b, hq, d), np.nan, device="cuda")
        for m, n in zip(made, lens):
            m[0].truncate(n)
        ses.decode_step(None, dev(q), dev(k), dev(v), [m[0] for m in made], KvAttentionConfig(1, hq, hkv, d, True, window), out)
        ses.sync()
        for i, (c, k0, v0) in enumerate(made):
            keys, values = np.concatenate([k0, hold(k[i:i + 1])]), np.concatenate([v0, hold(v[i:i + 1])])
            gk, gv = held(ses, c)
            assert_bitwise(gk, keys.astype(np.float32), f"keys of {lens[i]}")
            assert_bitwise(gv, values.astype(np.float32), f"values of {lens[i]}")
            check(out[i], attend(q[i:i + 1], keys, values, True, window)[0], values, f"step over {lens[i]} window {window}")


def test_steps_report_values_outside_the_format(ses):
    d, hq, hkv = 128, 4, 2
    rng = np.random.default_rng(31)
    for which in (0, 1):
        c, _, _ = filled(ses, rng, 20, hkv, d, 1)
        kv = [rows(rng, 1, hkv, d), rows(rng, 1, hkv, d)]
        kv[which][0, 1, 77] = np.inf
        q, out = dev(rows(rng, 1, hq, d)), torch.empty(1, hq, d, device="cuda")
        ses.decode_step(None, q, dev(kv[0]), dev(kv[1]), [c], KvAttentionConfig(1, hq, hkv, d, True), out)
        with pytest.raises(sa.InvalidTensorDataError):
            ses.sync()
        ses.sync()


def test_two_graphs_share_the_workspaces(ses):
    """Replays in turn, of a split step, of a chunk with ranges, and of the step's chunk form."""
    d, hq, hkv = 128, 6, 2
    rng = np.random.default_rng(32)
    stream = torch.cuda.Stream()
    own = Session(0, stream=stream)
    with torch.cuda.stream(stream):
        made = [filled(own, rng, n, hkv, d, 40)[0] for n in (3000, 1800)]
        q1, k1, v1 = (dev(rows(rng, 1, h, d)) for h in (hq, hkv, hkv))
        q2, k2, v2 = (dev(rows(rng, 40, h, d)) for h in (hq, hkv, hkv))
        outs = [torch.zeros(1, hq, d, device="cuda"), torch.zeros(40, hq, d, device="cuda")]
    table = own.rope_table(0, d, 10000.0, max_positions=4000)

    def one():
        made[0].truncate(3000)
        own.decode_step(table, q1, k1, v1, [made[0]], KvAttentionConfig(1, hq, hkv, d, True), outs[0])

    def many():
        made[1].truncate(1800)
        own.prefill_step(table, q2, k2, v2, made[1], KvAttentionConfig(40, hq, hkv, d, True), outs[1])

    calls, graphs, want = (one, many), [], []
    for call, out in zip(calls, outs):
        call()
        own.sync()
        want.append(out.cpu().numpy())
    for call in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            call()
    for turn in (0, 1, 0, 0, 1, 1):
        with torch.cuda.stream(stream):
            outs[turn].zero_()
        torch.cuda.synchronize()
        graphs[turn].replay()
        torch.cuda.synchronize()
        assert_bitwise(outs[turn].cpu().numpy(), want[turn], f"graph {turn}")
        own.sync()


@pytest.mark.parametrize("d,hq,hkv,s,past", [(64, 9, 3, 401, 333), (128, 5, 1, 450, 77), (256, 4, 2, 300, 513), (128, 16, 2, 129, 2000)])
def test_chunks_of_many_rows(ses, d, hq, hkv, s, past):
    test_chunks(ses, d, hq, hkv, s, past)


@pytest.mark.parametrize("d,hq,hkv", [(64, 9, 3), (128, 4, 2), (256, 3, 1), (64, 5, 5)])
@pytest.mark.parametrize("s,past", [(2, 2600), (7, 1500), (33, 800)])
def test_a_few_queries_over_several_key_ranges(ses, d, hq, hkv, s, past):
    test_chunks(ses, d, hq, hkv, s, past)


@pytest.mark.parametrize("s", [1, 3])
@pytest.mark.parametrize("scale", [1e-3, 300.0])
def test_few_queries_of_values_of_any_size(ses, s, scale):
    """As test_values_of_any_size, and with one row of large values among small ones."""
    rng = np.random.default_rng(33)
    k, v = rows(rng, 900, 2, 64), (rows(rng, 900, 2, 64) * scale).astype(np.float32)
    c = ses.q4_kv_cache(2, 64, 900)
    big = np.full((1, 2, 64), 60000.0, np.float32)
    ses.append(c, dev(big), dev(big), 1)
    c.truncate(0)
    ses.append(c, dev(k), dev(v), 900)
    q = rng.standard_normal((s, 4, 64)).astype(np.float32)
    out = torch.empty(s, 4, 64, device="cuda")
    cfg = KvAttentionConfig(s, 4, 2, 64, True)
    ses.attention_cached(dev(q), c, cfg, out)
    ses.sync()
    check(out, attend(q, hold(k), hold(v)), hold(v), f"values of {scale}")
    c.truncate(0)
    v[400] *= np.float32(40.0)  # (the range's scale moves in the middle; 300 * 40 * 5 is within the format's 65504)
    ses.append(c, dev(k), dev(v), 900)
    ses.attention_cached(dev(q), c, cfg, out)
    ses.sync()
    check(out, attend(q, hold(k), hold(v)), hold(v), f"values of {scale}, one row far larger")


def test_rows_past_a_launch(ses):
    """More rows in one append than a grid has threads for, which is under 2^32."""
    n, h, d = 15900000, 17, 64
    if torch.cuda.mem_get_info()[0] < 130 << 30:
        pytest.skip("needs 130 GiB of device memory")
    rng = np.random.default_rng(41)
    x = torch.zeros(n, h, d, device="cuda")
    places = [0, 7895159, 7895160, 7895161, 15790319, 15790320, 15790321, n - 1]
    some = rows(rng, len(places), h, d)
    x[torch.tensor(places, device="cuda")] = dev(some)
    c = ses.q4_kv_cache(h, d, n)
    ses.append(c, x, x, n)
    ses.sync()
    for i, at in enumerate(places):
        gk, gv = held(ses, c, at, 1)
        assert_bitwise(gk, hold(some[i:i + 1]), f"key {at}")
        assert_bitwise(gv, hold(some[i:i + 1]), f"value {at}")
    gk, _ = held(ses, c, 7895100, 60)
    assert not np.any(gk[:59])
    del x
    torch.cuda.empty_cache()
