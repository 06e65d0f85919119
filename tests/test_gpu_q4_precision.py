"""How far attention over the 4-bit cache is from 64-bit sums over the same held
rows, by the root mean square (RMS) of the errors against that of the outputs.

A score takes at most 24 roundings of 2^-24 (tests/test_gpu_q4_cache.py counts
them) of partial sums that are at most A = sum |q k| / sqrt(D). Each is off by
at most half a step and unbiased, so of RMS 2^-24 A / sqrt(3): together sqrt(8)
2^-24 A, which is the relative error of a weight. Weights, values and outputs
add a few roundings of 2^-24 of their own: 2^-22 holds sixteen of them at their
worst, or more at their RMS. An error that all outputs of a row share is at most that too.
"""
import numpy as np
import pytest
import torch

from spissa_amd import InvalidTensorDataError, RotaryEmbeddingConfig, apply_gemma_rotary_inplace, rms_norm
from spissa_amd.device import Session
from spissa_amd.rotary import KvAttentionConfig
from tests.q4 import attend, hold

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ses(gpu):
    # the tests' own tensors are made, filled and freed on the session's stream
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        yield Session(0, stream=stream)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def attention(ses, q, cache, hkv, causal=True, window=0):
    s, hq, d = q.shape
    out = torch.full((s, hq, d), np.nan, device="cuda")
    ses.attention_cached(dev(q), cache, KvAttentionConfig(s, hq, hkv, d, causal, window), out)
    ses.sync()
    return out.cpu().numpy()


def rms(a):
    return float(np.sqrt(np.mean(np.square(np.asarray(a, np.float64)))))


def score_size(q, keys):
    """A: the largest sum |q k| / sqrt(D) of a query and a key of its KV head."""
    hq, hkv, d = q.shape[1], keys.shape[1], q.shape[2]
    q, keys = np.abs(q).astype(np.float64), np.abs(keys).astype(np.float64)
    return max(np.max(q[:, h] @ keys[:, h * hkv // hq].T) for h in range(hq)) / np.sqrt(d)


def check(got, ref, a, what, more=0.0):
    off, tol = rms(got - ref) / rms(ref), np.sqrt(8.0) * 2.0**-24 * a + 2.0**-22 + more
    print(f"[q4 precision] {what}: {off:.2e} of {tol:.2e}", flush=True)
    assert off <= tol, (what, off, tol)


@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 1), (128, 6, 2), (256, 2, 1)])
@pytest.mark.parametrize("s", [1, 5, 550])
@pytest.mark.parametrize("nats", [9.0, 11.0, 13.0])
def test_a_sink(ses, d, hq, hkv, s, nats):
    """The first key takes the weight and has no value: the output is the rest, which has little weight each."""
    rng = np.random.default_rng(d + s)
    n = 6000
    k = rng.standard_normal((n, hkv, d)).astype(np.float32)
    v = (1 + 0.3 * rng.standard_normal((n, hkv, d))).astype(np.float32)
    q = rng.standard_normal((s, hq, d)).astype(np.float32)
    k[:, :, 0], q[:, :, 0] = 0, 4
    k[0], v[0] = 0, 0
    k[0, :, 0] = nats * np.sqrt(d) / 4  # (the others' scores are about N(0, 1))
    c = ses.q4_kv_cache(hkv, d, n)
    ses.append(c, dev(k), dev(v), n)
    keys, values = hold(k), hold(v)
    check(attention(ses, q, c, hkv), attend(q, keys, values), score_size(q, keys), f"d {d} s {s} {nats} nats")


@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 1), (128, 6, 2), (256, 2, 1)])
@pytest.mark.parametrize("s,past", [(1, 39), (5, 35), (550, 0)])
@pytest.mark.parametrize("nats", [5.0, 9.0, 13.0])
def test_a_sink_before_few_keys(ses, d, hq, hkv, s, past, nats):
    """As test_a_sink, with each row's error against that row's output: few keys do not
    average their weights' roundings. The weights are about e^-nats of the largest, so
    2^-19 at the least; a second piece that ends 2^-38 below the largest is a rounding
    of 2^-20 there: off by at most half of that, 2^-22 in RMS over two keys and more."""
    rng = np.random.default_rng(d + s)
    n = s + past
    k = rng.standard_normal((n, hkv, d)).astype(np.float32)
    v = (1 + 0.3 * rng.standard_normal((n, hkv, d))).astype(np.float32)
    q = rng.standard_normal((s, hq, d)).astype(np.float32)
    k[:, :, 0], q[:, :, 0] = 0, 4
    k[0], v[0] = 0, 0
    k[0, :, 0] = nats * np.sqrt(d) / 4
    c = ses.q4_kv_cache(hkv, d, n)
    ses.append(c, dev(k), dev(v), n)
    keys, values = hold(k), hold(v)
    got, ref = attention(ses, q, c, hkv), attend(q, keys, values)
    if past == 0:  # (the first query sees the sink alone)
        assert not np.any(got[0]) and not np.any(ref[0])
        got, ref = got[1:], ref[1:]
    size = np.sqrt(np.mean(ref * ref, axis=2, keepdims=True))
    check(got / size, ref / size, score_size(q, keys), f"d {d} s {s} {nats} nats, few keys", 2.0**-22)


@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 4), (128, 2, 2), (256, 1, 1), (128, 8, 1)])
@pytest.mark.parametrize("s", [40, 1100])
def test_roundings_have_no_side(ses, d, hq, hkv, s):
    """Queries that see one key each give its value back. Weights and values of two
    pieces, each the nearest, are off to either side alike: over the 320 (key, group)
    pairs or more of a case, a mean of roundings of 2^-24 at most (2^-25 in RMS) stays
    within 2^-29, and four times that is allowed. Cut pieces are off to one side."""
    rng = np.random.default_rng(d + s)
    k, v = rng.standard_normal((2, s, hkv, d)).astype(np.float32)
    q = rng.standard_normal((s, hq, d)).astype(np.float32)
    c = ses.q4_kv_cache(hkv, d, s)
    ses.append(c, dev(k), dev(v), s)
    ref = np.repeat(hold(v).astype(np.float64), hq // hkv, axis=1)
    got = attention(ses, q, c, hkv, window=1)
    gain = float(np.sum((got - ref) * ref) / np.sum(ref * ref))
    print(f"[q4 precision] d {d} heads {hq}/{hkv} s {s}: 1 + {gain:.2e}", flush=True)
    assert abs(gain) <= 2.0**-27, gain
    check(got, ref, 0.0, "one key")


@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 2), (128, 6, 2), (256, 4, 1)])
@pytest.mark.parametrize("how", ["clear", "truncate", "roll back", "not finite"])
def test_a_used_cache_is_as_a_new_one(ses, d, hq, hkv, how):
    """Rows that are gone leave nothing behind, bit for bit."""
    rng = np.random.default_rng(d)
    n, half = 700, 300
    k, v = rng.standard_normal((2, n, hkv, d)).astype(np.float32) * np.float32(0.01)
    q = rng.standard_normal((n, hq, d)).astype(np.float32)
    new, used = (ses.q4_kv_cache(hkv, d, n) for _ in range(2))
    ses.append(new, dev(k), dev(v), n)
    at = half if how in ("roll back", "not finite") else 0
    if at:
        ses.append(used, dev(k[:at]), dev(v[:at]), at)
    gone = torch.full((100, hkv, d), np.inf if how == "not finite" else 65504.0, device="cuda")
    gone[:, :, ::2] = -65504.0
    ses.append(used, gone, gone, 100)
    if how == "not finite":
        with pytest.raises(InvalidTensorDataError):
            ses.sync()
    if how == "clear":
        used.clear()
    else:
        used.truncate(at)
    ses.append(used, dev(k[at:]), dev(v[at:]), n - at)
    want, got = attention(ses, q, new, hkv), attention(ses, q, used, hkv)
    assert np.array_equal(want.view(np.uint32), got.view(np.uint32))
    keys, values = hold(k), hold(v)
    check(got, attend(q, keys, values), score_size(q, keys), f"d {d} {how}")


@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 2), (128, 6, 2), (256, 4, 1)])
@pytest.mark.parametrize("s", [1, 5, 550])
@pytest.mark.parametrize("at", [0, 333])
def test_small_values_beside_a_large_one(ses, d, hq, hkv, s, at):
    """A row of large values that no query looks at costs the others what the pieces
    cannot hold: 2^-38 of the largest value, for each of the weights and the values."""
    rng = np.random.default_rng(d + s + at)
    n = 900
    k, v = rng.standard_normal((2, n, hkv, d)).astype(np.float32)
    v = 1 + np.float32(0.1) * v
    q = rng.standard_normal((s, hq, d)).astype(np.float32)
    k[:, :, 0], q[:, :, 0] = 0, 4
    k[at] = 0
    k[at, :, 0] = -10.0 * np.sqrt(d)  # 40 nats below
    v[at] = 3000 * rng.standard_normal((hkv, d))
    c = ses.q4_kv_cache(hkv, d, n)
    ses.append(c, dev(k), dev(v), n)
    keys, values = hold(k), hold(v)
    ref = attend(q, keys, values)
    check(attention(ses, q, c, hkv), ref, score_size(q, keys), f"d {d} s {s}, a large row", 2 * 2.0**-38 * np.max(np.abs(values)) / rms(ref))


@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 2), (128, 6, 2), (256, 4, 1)])
@pytest.mark.parametrize("s", [1, 5, 550])
@pytest.mark.parametrize("size", [1e5, 1e7, 1e9, 1e30])
@pytest.mark.parametrize("value", [1.0, 0.02])
def test_scores_of_any_size(ses, d, hq, hkv, s, size, value):
    """Scores whose largest takes the whole weight: its value comes back, to a weight of two
    pieces and seven roundings of the step's part, the minimum's and their sum over the
    weight's, each at most 1.1 of the largest value: under sixteen of 2^-24 together. Where
    two scores are within their roundings of each other the row says nothing: 24 of 2^-24 A
    each, and 30 to make the second's weight vanish."""
    rng = np.random.default_rng(d + s)
    n = 600
    k, v = rng.standard_normal((2, n, hkv, d)).astype(np.float32)
    v *= np.float32(value)  # (and with them the scale that the weights are held at)
    q = (rng.standard_normal((s, hq, d)) * size).astype(np.float32)
    c = ses.q4_kv_cache(hkv, d, n)
    ses.append(c, dev(k), dev(v), n)
    keys, values = hold(k), hold(v)
    got, ref = attention(ses, q, c, hkv), attend(q, keys, values)
    assert np.isfinite(got).all()
    sc = np.einsum("shd,nhd->shn", q.astype(np.float64), np.repeat(keys, hq // hkv, axis=1)) / np.sqrt(d)
    pos = np.arange(n - s, n)[:, None, None]
    sc = np.sort(np.where(np.arange(n) > pos, -np.inf, sc), axis=2)
    clear = sc[:, :, -1] - sc[:, :, -2] > 30 + 48 * 2.0**-24 * score_size(q, keys)
    assert clear.mean() > 0.5
    off = np.max(np.abs(got - ref)[clear]) / np.max(np.abs(values))
    print(f"[q4 precision] d {d} s {s} scores of {size}: {off:.2e}, {clear.mean():.2f} of the rows", flush=True)
    assert off <= 2.0**-20, off


@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 2), (128, 6, 2), (256, 4, 2)])
@pytest.mark.parametrize("batch", [1, 5, 17])
@pytest.mark.parametrize("window", [0, 64])
def test_gemma_steps_of_a_batch(ses, d, hq, hkv, batch, window):
    """Norm, rotation, prescale, append and attention of a token of each of several
    sequences. The norm's sum is a tree where the plain form's is a chain: each is off by
    at most d / 2 roundings of 2^-24, so queries and keys may differ by 2^-16 of themselves
    (d 256) at worst, and by 2^-21 in RMS. The reference takes the keys as they were held."""
    eps, prescale = 1e-6, 0.5
    rng = np.random.default_rng(d + batch)
    lens = [int(x) for x in rng.integers(0, 900, batch)]
    lens[0] = 0
    q, k, v = (rng.standard_normal((batch, h, d)).astype(np.float32) for h in (hq, hkv, hkv))
    qn, kn = (1 + 0.1 * rng.standard_normal((2, d))).astype(np.float32)
    table = ses.rope_table(1, d, 10000.0, 8.0, max_positions=max(lens) + 1)
    caches, held = [], []
    for n in lens:
        pk, pv = rng.standard_normal((2, n, hkv, d)).astype(np.float32)
        caches.append(ses.q4_kv_cache(hkv, d, n + 1))
        if n:
            ses.append(caches[-1], dev(pk), dev(pv), n)
        held.append((hold(pk), hold(pv)))
    out = torch.full((batch, hq, d), np.nan, device="cuda")
    ses.gemma_decode_step(table, dev(q), dev(k), dev(v), caches, KvAttentionConfig(1, hq, hkv, d, True, window), dev(qn), dev(kn), eps,
                          prescale, out)
    ses.sync()
    got = out.cpu().numpy()
    for b, n in enumerate(lens):
        qr = rms_norm(q[b].ravel(), qn, hq, d, eps)
        kr = rms_norm(k[b].ravel(), kn, hkv, d, eps)
        apply_gemma_rotary_inplace(qr, kr, hq, hkv, RotaryEmbeddingConfig(1, hq, d, d, 10000.0, n), 8.0)
        assert len(caches[b]) == n + 1
        keys, values = caches[b].keys().reshape(n + 1, hkv, d), caches[b].values().reshape(n + 1, hkv, d)
        assert np.array_equal(keys[:n].view(np.uint32), held[b][0].view(np.uint32))
        assert np.array_equal(values.view(np.uint32), np.concatenate([held[b][1], hold(v[b:b + 1])]).view(np.uint32))
        near, step = hold(kr.reshape(1, hkv, d)), np.ptp(kr.reshape(-1, 32), axis=1).repeat(32).reshape(1, hkv, d) / 15
        assert np.all(np.abs(keys[n:] - near) <= 1.01 * step + 1e-3 * np.abs(near)), f"key of sequence {b}"
        qr = (qr * np.float32(prescale)).reshape(1, hq, d)
        a = score_size(qr, keys)
        check(got[b:b + 1], attend(qr, keys, values, True, window), a, f"d {d} sequence {b} of {n}", 2.0**-21 * a)


@pytest.mark.parametrize("d,hq,hkv", [(64, 32, 8), (128, 6, 2), (256, 4, 1)])
@pytest.mark.parametrize("s,past", [(1, 0), (1, 40), (1, 5000), (6, 700), (40, 3000), (300, 20), (530, 900)])
def test_outputs(ses, d, hq, hkv, s, past):
    """Ordinary rows, against the outputs' own size: a second piece left out anywhere
    (2^-12 of a query, a weight or a value) is tens of times the tolerance."""
    rng = np.random.default_rng(d + s + past)
    n = s + past
    k, v = rng.standard_normal((2, n, hkv, d)).astype(np.float32)
    k += rng.standard_normal((hkv, d)).astype(np.float32)  # channels' own offsets
    q = rng.standard_normal((s, hq, d)).astype(np.float32)
    c = ses.q4_kv_cache(hkv, d, n)
    if past:
        ses.append(c, dev(k[:past]), dev(v[:past]), past)
    keys, values = hold(k), hold(v)
    a = score_size(q, keys)
    out = torch.full((s, hq, d), np.nan, device="cuda")
    for window in (0, 100):
        c.truncate(past)
        cfg = KvAttentionConfig(s, hq, hkv, d, True, window)
        args = dev(q), dev(k[past:]), dev(v[past:])
        ses.decode_step(None, *args, [c], cfg, out) if s == 1 else ses.prefill_step(None, *args, c, cfg, out)
        ses.sync()
        ref = attend(q, keys, values, True, window)
        check(out.cpu().numpy(), ref, a, f"d {d} step {s}+{past} window {window}")
        got = attention(ses, q, c, hkv, window=window)
        assert np.array_equal(got.view(np.uint32), out.cpu().numpy().view(np.uint32)), "the attention alone"
    check(attention(ses, q, c, hkv, causal=False), attend(q, keys, values, False), a, f"d {d} {s}+{past} not causal")
