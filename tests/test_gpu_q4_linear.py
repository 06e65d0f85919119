"""Projections of 4-bit weights against 64-bit sums.

Tolerance, for each output, of sum |x w|. An activation is held to 2^-22 of
itself (down to 2^-28 of the largest of its row, below that to 2^-38 of that
largest: the second term). The sums run over at most K / 32 steps of two
instructions in f32, each of 32 products and a rounding, and then 16 ranges:
(K / 16 + 64) roundings of 2^-24 at worst.
"""
import threading

import numpy as np
import pytest
import torch

import spissa_amd as sa
from spissa_amd.device import AttentionLayer, Session
from spissa_amd.linear import DTYPE_BF16, DTYPE_Q4, StreamingLinearConfig, StreamingTileLinearConfig
from spissa_amd.rotary import KvAttentionConfig
from tests.q4 import attend

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ses(gpu):
    # the tests' own tensors are made, filled and freed on the session's stream
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        yield Session(0, stream=stream)


SCALES = {"f16": np.float16, "bf16": None, "f32": np.float32}


class Weight:
    """A checkpoint's arrays and the float64 matrix they stand for."""

    def __init__(self, rng, n, k, group, scale="f16", zeros=False, size=0.01):
        groups = -(-k // group)
        self.n, self.k, self.group = n, k, group
        self.codes = rng.integers(0, 256, (n, (k + 1) // 2), dtype=np.uint8)
        s = ((0.2 + rng.random((n, groups))) * size * rng.choice([-1, 1], (n, groups), p=[0.1, 0.9])).astype(np.float32)
        if scale == "bf16":
            self.scales = (s.view(np.uint32) >> 16).astype(np.uint16)
            s = (self.scales.astype(np.uint32) << 16).view(np.float32)
        else:
            self.scales = s.astype(SCALES[scale])
        self.zeros = rng.integers(0, 16, (n, groups), dtype=np.uint8) if zeros else None
        c = np.empty((n, 2 * self.codes.shape[1]))
        c[:, 0::2], c[:, 1::2] = self.codes & 15, self.codes >> 4
        of = np.arange(k) // group
        z = 8 if self.zeros is None else self.zeros[:, of].astype(np.float64)
        real = s if scale == "bf16" else self.scales
        self.w = (c[:, :k] - z) * real.astype(np.float64)[:, of]

    def on(self, ses):
        return ses.q4_linear_weight(self.codes, self.scales, self.n, self.k, self.group, self.zeros)


def bound(x, w, bias):
    k = x.shape[1]
    most = np.max(np.abs(x), axis=1, keepdims=True)
    b = (k / 16 + 64) * 2.0**-24 * (np.abs(x) @ np.abs(w).T) + 2.0**-22 * (np.abs(x) @ np.abs(w).T)
    b += 2.0**-38 * most * np.abs(w).sum(1)[None, :]
    return b + 2.0**-23 * (0 if bias is None else np.abs(bias))


def call(ses, weight, x, bias=None, offset=0):
    m, n = x.shape[0], weight.out_features
    room = torch.empty(x.size + offset, device="cuda")
    dx = room[offset:].view(m, x.shape[1])
    dx.copy_(torch.from_numpy(x))
    out = torch.full((m + 1, n), np.nan, device="cuda")
    ses.linear(weight, dx, None if bias is None else torch.from_numpy(bias).cuda(), m, out[:m])
    ses.sync()
    assert torch.isnan(out[m]).all(), "a row past the last was written"
    return out[:m].cpu().numpy()


def check(ses, wt, x, bias=None, weight=None, offset=0, what=""):
    got = call(ses, weight or wt.on(ses), x, bias, offset).astype(np.float64)
    x = x.astype(np.float64)
    ref = x @ wt.w.T + (0 if bias is None else bias.astype(np.float64))
    off = np.abs(got - ref) / (bound(x, wt.w, bias) + 1e-300)
    print(f"[q4 linear] {what} {wt.n}x{wt.k}/{wt.group} m {x.shape[0]}: {off.max():.3f} of the bound", flush=True)
    assert off.max() <= 1, (what, off.max())


def acts(rng, m, k):
    return rng.standard_normal((m, k)).astype(np.float32)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 16, 17, 33, 65, 130])
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (15, 31, 32), (16, 128, 128), (17, 129, 64), (100, 300, 32),
                                       (33, 1000, 128), (512, 2048, 32), (260, 777, 96), (48, 640, 256), (64, 256, 4096)])
def test_sizes(ses, m, n, k, group):
    rng = np.random.default_rng(m + 7 * n + k)
    wt = Weight(rng, n, k, group)
    check(ses, wt, acts(rng, m, k), rng.standard_normal(n).astype(np.float32))


@pytest.mark.parametrize("scale", list(SCALES))
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 4, 9, 70])
def test_types(ses, m, scale, zeros, group):
    rng = np.random.default_rng(group + m)
    wt = Weight(rng, 90, 600, group, scale, zeros)
    check(ses, wt, acts(rng, m, 600), None, what=f"{scale} zeros {zeros}")


@pytest.mark.parametrize("m", [1, 3, 20, 300])
@pytest.mark.parametrize("k", [64, 512, 1000, 1001])
def test_rows_of_any_alignment(ses, m, k):
    rng = np.random.default_rng(k + m)
    wt = Weight(rng, 70, k, 64)
    w = wt.on(ses)
    x = acts(rng, m, k)
    for offset in (0, 1, 2, 3):
        check(ses, wt, x, None, w, offset)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (2, 2048, 8192), (16, 2560, 2048), (333, 1151, 2500), (1, 40001, 576),
                                   (1030, 2048, 2048)])
def test_large(ses, m, n, k):
    rng = np.random.default_rng(n)
    wt = Weight(rng, n, k, 128, "f16", True)
    check(ses, wt, acts(rng, m, k), rng.standard_normal(n).astype(np.float32))


@pytest.mark.parametrize("m", [16, 17, 24, 32, 33, 47, 64])
@pytest.mark.parametrize("n,k,group", [(70, 8192, 128), (130, 8200, 64), (1000, 9000, 32), (2100, 500, 128)])
def test_some_tokens(ses, m, n, k, group):
    """Either side of where the tiles of many tokens begin."""
    rng = np.random.default_rng(n + m)
    wt = Weight(rng, n, k, group, "f16", True)
    check(ses, wt, acts(rng, m, k), rng.standard_normal(n).astype(np.float32))


@pytest.mark.parametrize("n,k,group", [(98337, 200, 64), (98305, 129, 32), (99000, 640, 128), (20005, 1100, 64), (33000, 515, 32)])
@pytest.mark.parametrize("scale,zeros", [("f16", False), ("f32", True)])
@pytest.mark.parametrize("m", [1, 3])
def test_one_token_of_many_rows(ses, n, k, group, scale, zeros, m):
    rng = np.random.default_rng(n)
    wt = Weight(rng, n, k, group, scale, zeros)
    check(ses, wt, acts(rng, m, k), rng.standard_normal(n).astype(np.float32), what=f"{scale} zeros {zeros}")


@pytest.mark.parametrize("scale,zeros,group", [("f16", False, 128), ("f16", True, 64), ("f32", True, 32), ("bf16", False, 128),
                                               ("f32", False, 128), ("f16", False, 32), ("bf16", True, 64)])
@pytest.mark.parametrize("k", [1, 130, 257, 700])
def test_many_tokens_and_many_rows(ses, scale, zeros, group, k):
    """The tiles of many tokens, their last ones ragged, over one block of K and more."""
    rng = np.random.default_rng(k + group)
    wt = Weight(rng, 4100, k, group, scale, zeros)
    check(ses, wt, acts(rng, 1545, k), rng.standard_normal(4100).astype(np.float32), what=f"{scale} zeros {zeros}")


@pytest.mark.parametrize("m", [1, 4, 5, 40])
def test_activations_of_every_size(ses, m):
    """Outliers, a row of zeros, rows at the ends of the f32 range."""
    rng = np.random.default_rng(m)
    wt = Weight(rng, 50, 512, 32, "f32")
    w = wt.on(ses)
    x = acts(rng, m, 512)
    x[:, ::100] *= 3000
    check(ses, wt, x, None, w, what="outliers")
    x[0] = 0
    assert not call(ses, w, x)[0].any()
    x[0] = acts(rng, 1, 512)[0] * np.float32(1e30)
    check(ses, wt, x, None, w, what="1e30")
    small = (acts(rng, m, 512).astype(np.float64) * 1e-30).astype(np.float32)
    check(ses, wt, small, None, w, what="1e-30")
    tiny = (acts(rng, m, 512).astype(np.float64) * 1e-40).astype(np.float32)
    got = call(ses, w, tiny).astype(np.float64)
    # below the normal range a term may lose all but 2^-149
    assert np.max(np.abs(got - tiny.astype(np.float64) @ wt.w.T)) <= 512 * 15 * 0.012 * 2.0**-126 * 2.0**-20 + 2.0**-140


@pytest.mark.parametrize("m", [2, 6, 40])
def test_infinities_and_nan_stay_in_their_row(ses, m):
    rng = np.random.default_rng(m)
    wt = Weight(rng, 40, 300, 64)
    w = wt.on(ses)
    x = acts(rng, m, 300)
    clean = call(ses, w, x)
    x[0, 100] = np.inf
    x[1, 200] = np.nan
    got = call(ses, w, x)
    with np.errstate(invalid="ignore"):
        ref = x[:2].astype(np.float64) @ wt.w.T
        # one infinity: its products decide
        want = np.where(wt.w[:, 100] == 0, np.nan, np.sign(wt.w[:, 100]) * np.inf)
    assert np.array_equal(got[0], want.astype(np.float32), equal_nan=True)
    assert np.isnan(got[1]).all() and np.isnan(ref[1]).all()
    assert np.array_equal(got[2:], clean[2:])


def test_a_row_of_infinite_scale(ses):
    """An infinite scale is its row's alone, groups past the last channel included."""
    rng = np.random.default_rng(3)
    wt = Weight(rng, 20, 40, 32)
    wt.scales[3, 1] = np.inf
    x = acts(rng, 2, 40)
    got = call(ses, ses.q4_linear_weight(wt.codes, wt.scales, 20, 40, 32), x)
    assert not np.isfinite(got[:, 3]).any() and np.isfinite(np.delete(got, 3, 1)).all()
    assert np.isinf(got[:, 3]).all()


def test_device_and_host_arrays_are_the_same(ses):
    rng = np.random.default_rng(4)
    wt = Weight(rng, 37, 333, 64, "bf16", True)
    x = acts(rng, 3, 333)
    a = call(ses, wt.on(ses), x)
    dev = lambda t: torch.from_numpy(t).cuda()  # noqa: E731
    b = call(ses, ses.q4_linear_weight(dev(wt.codes), dev(wt.scales.view(np.int16)).view(torch.bfloat16), 37, 333, 64,
                                       dev(wt.zeros)), x)
    assert np.array_equal(a, b)


def test_drop_in_and_lm_head(ses):
    rng = np.random.default_rng(5)
    wt = Weight(rng, 1000, 256, 32)
    w = sa.Q4LinearWeight(wt.codes, wt.scales, 1000, 256, 32)
    x = acts(rng, 2, 256)
    bias = rng.standard_normal(1000).astype(np.float32)
    model = sa.LinearModel({"w": w})
    got = sa.streaming_tile_linear_from_model(model, "w", x.ravel(), bias,
                                              StreamingTileLinearConfig(StreamingLinearConfig(2, 256, 1000), 64))
    ref = x.astype(np.float64) @ wt.w.T + bias
    assert np.all(np.abs(got.reshape(2, 1000) - ref) <= bound(x.astype(np.float64), wt.w, bias))
    logits = sa.lm_head_logits_q4(x[0].copy(), w, 1000, 256)
    dl, tok = torch.empty(1000, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    ses.lm_head(wt.on(ses), torch.from_numpy(x[0]).cuda(), dl, tok)
    ses.sync()
    assert np.array_equal(dl.cpu().numpy(), logits) and tok.item() == sa.sample_argmax(logits)


@pytest.mark.parametrize("m", [1, 7, 100])
def test_captured_and_replayed(ses, m):
    rng = np.random.default_rng(m)
    wt = Weight(rng, 300, 700, 64)
    stream = torch.cuda.Stream()
    own = Session(0, stream=stream)
    w = wt.on(own)
    x, out = torch.zeros(m, 700, device="cuda"), torch.zeros(m, 300, device="cuda")
    torch.cuda.synchronize()
    own.linear(w, x, None, m, out)
    own.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        own.linear(w, x, None, m, out)
    for _ in range(3):
        nx = acts(rng, m, 700)
        x.copy_(torch.from_numpy(nx))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), call(ses, wt.on(ses), nx))


def test_several_threads_on_one_session(ses):
    rng = np.random.default_rng(8)
    own = Session(0)
    wt = Weight(rng, 200, 1000, 128)
    w = wt.on(own)
    xs = [acts(rng, m, 1000) for m in (1, 6, 30, 90, 12, 200)]
    want = [call(ses, wt.on(ses), x) for x in xs]
    dx = [torch.from_numpy(x).cuda() for x in xs]
    outs = [torch.zeros(x.shape[0], 200, device="cuda") for x in xs]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            for _ in range(20):
                own.linear(w, dx[i], None, xs[i].shape[0], outs[i])
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    own.sync()
    assert not failed
    for o, r in zip(outs, want):
        assert np.array_equal(o.cpu().numpy(), r)


def test_one_token_beside_a_growing_workspace(ses):
    """One thread's calls need no workspace while another's replace it by larger ones."""
    rng = np.random.default_rng(11)
    own = Session(0)
    wt = Weight(rng, 48, 512, 64)
    w = wt.on(own)
    one, many = acts(rng, 1, 512), acts(rng, 400, 512)
    want = call(ses, wt.on(ses), one)
    d_one, d_many = torch.from_numpy(one).cuda(), torch.from_numpy(many).cuda()
    outs = [torch.zeros(1, 48, device="cuda") for _ in range(64)]
    out = torch.zeros(400, 48, device="cuda")
    torch.cuda.synchronize()
    failed = []

    def run(calls):
        try:
            for c in calls:
                own.linear(w, *c)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=([(d_one, None, 1, o) for o in outs],)),
               threading.Thread(target=run, args=([(d_many, None, m, out) for m in range(5, 401, 9)],))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    own.sync()
    assert not failed
    for o in outs:
        assert np.array_equal(o.cpu().numpy(), want)
    assert np.array_equal(out[:392].cpu().numpy(), call(ses, wt.on(ses), many[:392]))


def test_refusals(ses):
    rng = np.random.default_rng(9)
    wt = Weight(rng, 20, 100, 32, "f16", True)
    new = ses.q4_linear_weight
    cases = [
        (sa.ShapeError, lambda: new(wt.codes, wt.scales, 20, 100, 0)),
        (sa.ShapeError, lambda: new(wt.codes, wt.scales, 20, 100, 16)),
        (sa.ShapeError, lambda: new(wt.codes, wt.scales, 0, 100, 32)),
        (sa.ShapeError, lambda: new(wt.codes, wt.scales, 20, 0, 32)),
        (sa.ShapeError, lambda: new(wt.codes, wt.scales, 1 << 31, 100, 32)),
        (sa.InvalidTensorDataError, lambda: new(wt.codes, wt.scales, 20, 102, 32)),
        (sa.InvalidTensorDataError, lambda: new(wt.codes, wt.scales, 20, 100, 64)),
        (sa.InvalidTensorDataError, lambda: new(wt.codes, wt.scales, 20, 100, 32, wt.zeros[:10])),
        (sa.InvalidTensorDataError, lambda: new(wt.codes, wt.scales, 20, 100, 32, wt.zeros + np.uint8(16))),
        (TypeError, lambda: new(wt.codes.astype(np.int32), wt.scales, 20, 100, 32)),
        (TypeError, lambda: new(wt.codes, wt.scales.astype(np.float64), 20, 100, 32)),
        (TypeError, lambda: new(wt.codes[:, ::2], wt.scales, 20, 100, 32)),
        (TypeError, lambda: sa.lm_head_logits_parallel(np.zeros(100, np.float32), wt.on(ses), 20, 100)),
        (sa.ShapeError, lambda: sa.linear(wt.on(ses), np.zeros(99, np.float32), None, StreamingLinearConfig(1, 99, 20))),
    ]
    for exc, make in cases:
        with pytest.raises(exc):
            make()
    other = ses.q4_linear_weight(wt.codes, wt.scales, 20, 100, 32, wt.zeros)
    ses.linear(other, torch.zeros(1, device="cuda"), None, 0, torch.zeros(1, device="cuda"))  # no tokens: nothing
    assert other.dtype == DTYPE_Q4
    ses.sync()


# ---- run together: a layer's attention sublayer ----

def norm(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)


@pytest.mark.parametrize("mixed", [False, True])
def test_sublayer_of_4_bit_weights_over_a_4_bit_cache(ses, mixed):
    """A prompt, a chunk and two tokens through a Llama layer's sublayer, against the same in 64
    bits over the rows the cache holds. mixed: bf16 weights beside the 4-bit ones."""
    hidden, hq, hkv, d, eps = 192, 6, 2, 64, 1e-5
    rng = np.random.default_rng(10)
    made = {t: Weight(rng, n, k, 64, size=0.02) for t, (n, k) in
            {"q": (hq * d, hidden), "k": (hkv * d, hidden), "v": (hkv * d, hidden), "o": (hidden, hq * d)}.items()}
    w = {t: m.on(ses) for t, m in made.items()}
    mat = {t: m.w for t, m in made.items()}
    if mixed:
        bits = (rng.standard_normal((hkv * d, hidden)).astype(np.float32) * np.float32(0.05)).view(np.uint32) >> 16
        w["v"] = ses.linear_weight(bits.astype(np.uint16).ravel(), DTYPE_BF16, hkv * d, hidden)
        mat["v"] = (bits << 16).view(np.float32).astype(np.float64)
    nw = (1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32)
    table = ses.rope_table(0, d, 10000.0, max_positions=200)
    layer = AttentionLayer(hidden, hq, hkv, d, w["q"], w["k"], w["v"], w["o"], input_norm=torch.from_numpy(nw).cuda(),
                           eps=eps, rope=table)
    cache = ses.q4_kv_cache(hkv, d, 128)
    inv = 1.0 / 10000.0 ** (np.arange(0, d, 2) / d)
    at = 0
    for s in (70, 9, 1, 1):
        x = acts(rng, s, hidden)
        out = torch.empty(s, hidden, device="cuda")
        ses.attention_sublayer(layer, torch.from_numpy(x).cuda(), s, cache, out)
        rows = [torch.empty(at + s, hkv, d, device="cuda") for _ in range(2)]
        ses.cache_rows(cache, 0, at + s, *rows)
        ses.sync()
        keys, values = (r.cpu().numpy() for r in rows)
        xn = norm(x.astype(np.float64), nw, eps)
        q = (xn @ mat["q"].T).reshape(s, hq, d)
        ang = (np.arange(at, at + s)[:, None] * inv)[:, None, :]
        a, b = q[..., :d // 2], q[..., d // 2:]
        q = np.concatenate([a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)], -1)
        ref = attend(q, keys, values).reshape(s, hq * d) @ mat["o"].T
        err = np.max(np.abs(out.cpu().numpy() - ref)) / np.max(np.abs(ref))
        print(f"[q4 sublayer] {s} tokens: {err:.2e}", flush=True)
        # f32 angles at positions below 200: 200 * 2^-24 in a rotation; the rest is the sums' 1e-5
        assert err <= 1e-4, (s, err)
        v = (xn @ mat["v"].T).reshape(s, hkv, d)
        step = (v.reshape(-1, 32).max(1) - v.reshape(-1, 32).min(1)) / 15
        assert np.all(np.abs(values[at:].reshape(-1, 32) - v.reshape(-1, 32)) <= 0.52 * step[:, None] + 2e-3)
        at += s
    assert len(cache) == at


def test_gemma_sublayer_of_4_bit_weights_over_a_4_bit_cache(ses):
    """The same through a Gemma layer's: norms of queries and keys, a prescale, positions
    divided by eight, a window, a norm behind. Scores reach A = 16 / 4 = 4 at most (rows of
    norm 16, sqrt(256), a prescale of 1/4), off by the angles' 25 * 2^-24 and the sums' 1e-5
    of them: under 5e-5 in a weight; the output's own sums and norms are 2e-5."""
    hidden, hq, hkv, d, eps, prescale, window = 320, 4, 2, 256, 1e-6, 0.25, 60
    rng = np.random.default_rng(12)
    made = {t: Weight(rng, n, k, 32, "f16", True, size=0.02) for t, (n, k) in
            {"q": (hq * d, hidden), "k": (hkv * d, hidden), "v": (hkv * d, hidden), "o": (hidden, hq * d)}.items()}
    w = {t: m.on(ses) for t, m in made.items()}
    nw, pw = (1 + 0.1 * rng.standard_normal((2, hidden))).astype(np.float32)
    qn, kn = (1 + 0.1 * rng.standard_normal((2, d))).astype(np.float32)
    on = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    layer = AttentionLayer(hidden, hq, hkv, d, w["q"], w["k"], w["v"], w["o"], input_norm=on(nw), q_norm=on(qn), k_norm=on(kn),
                           post_norm=on(pw), eps=eps, rope=ses.rope_table(1, d, 10000.0, 8.0, max_positions=200),
                           q_prescale=prescale, window=window)
    cache = ses.q4_kv_cache(hkv, d, 200)
    inv = 1.0 / 10000.0 ** (np.arange(0, d, 2) / d)
    at = 0

    def rotated(y, s):
        ang = (np.arange(at, at + s)[:, None] / 8.0 * inv)[:, None, :]
        a, b = y[..., :d // 2], y[..., d // 2:]
        return np.concatenate([a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)], -1)

    for s in (90, 1, 6, 40, 1):
        x = acts(rng, s, hidden)
        out = torch.empty(s, hidden, device="cuda")
        ses.attention_sublayer(layer, on(x), s, cache, out)
        rows = [torch.empty(at + s, hkv, d, device="cuda") for _ in range(2)]
        ses.cache_rows(cache, 0, at + s, *rows)
        ses.sync()
        keys, values = (r.cpu().numpy() for r in rows)
        xn = norm(x.astype(np.float64), nw, eps)
        q = rotated(norm((xn @ made["q"].w.T).reshape(s, hq, d), qn, eps), s) * prescale
        ref = norm(attend(q, keys, values, True, window).reshape(s, hq * d) @ made["o"].w.T, pw, eps)
        err = np.max(np.abs(out.cpu().numpy() - ref)) / np.max(np.abs(ref))
        print(f"[q4 sublayer] gemma, {s} tokens: {err:.2e}", flush=True)
        assert err <= 1e-4, (s, err)
        k = rotated(norm((xn @ made["k"].w.T).reshape(s, hkv, d), kn, eps), s)
        for got, y in ((keys, k), (values, (xn @ made["v"].w.T).reshape(s, hkv, d))):
            g = y.reshape(-1, 32)
            step = (g.max(1) - g.min(1)) / 15
            assert np.all(np.abs(got[at:].reshape(-1, 32) - g) <= 0.52 * step[:, None] + 2e-3 * np.max(np.abs(g), axis=1, keepdims=True))
        at += s
    assert len(cache) == at
