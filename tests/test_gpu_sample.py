"""Sampling on the device (spissa_sample_device) against the same in 64 bits.

Tokens have to be equal: the settings' limits and the random number's place are
compared on sums that are exact to 2^-38 of the largest weight or better, and a number
drawn this near a border of the definition's own (64-bit) sums is left out of the
comparison: BORDER, 2^-36 of the sum. Probabilities: one rounding to f32 (2^-24 of the
value), and weights in steps of 2^-(62 - log2 vocab) of the largest.
"""
import numpy as np
import pytest

from spissa_amd import _ffi
from tests import drafts

pytestmark = pytest.mark.gpu

BORDER = 2.0 ** -36
ROWS = [  # temperature, top_k, top_p, min_p
    (1.0, 0, 1.0, 0.0), (0.7, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 20, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (0.8, 50, 0.95, 0.05),
    (1.0, 0, 1.0, 0.3), (0.0, 0, 1.0, 0.0), (0.0, 5, 0.5, 0.5), (1.0, 0, 0.0, 0.0), (1.0, 0, 0.5, 1.0), (2.5, 300, 0.99, 0.001),
    (1e-3, 0, 0.9, 0.0), (100.0, 0, 0.5, 0.0), (1.0, 10**6, 0.8, 0.0), (1.0, 7, 0.999999, 0.0)]


@pytest.fixture(scope="module")
def s(gpu):
    import torch

    from spissa_amd.device import Session

    stream = torch.cuda.Stream()
    session = Session(0, stream=stream)
    with torch.cuda.stream(stream):
        yield session


def run(s, x, u, rows, per_row=True):
    """tokens, probs of logits x [n, vocab] under the settings rows [n]."""
    import torch

    from spissa_amd.device import SamplingConfig

    n = len(x)
    cols = list(zip(*rows))
    if per_row:
        cfg = SamplingConfig(*(torch.tensor(c, dtype=torch.int32 if i == 1 else torch.float32, device="cuda") for i, c in enumerate(cols)))
    else:
        cfg = SamplingConfig(*rows[0])
    tokens = torch.full((n,), -7, dtype=torch.int32, device="cuda")
    probs = torch.full((n,), -7.0, device="cuda")
    s.sample(torch.as_tensor(x, device="cuda"), torch.as_tensor(np.asarray(u, np.float32), device="cuda"), cfg, tokens, probs)
    return tokens.cpu().numpy(), probs.cpu().numpy()


def compare(x, u, rows, got):
    left_out = 0
    for i, (row, setting) in enumerate(zip(x, rows)):
        token, prob, near = drafts.sample(row, u[i], *setting)
        if near < BORDER:
            left_out += 1
            continue
        assert got[0][i] == token, (i, setting, got[0][i], token, prob)
        unit = 2.0 ** -min(51, 62 - int(np.ceil(np.log2(max(2, len(row))))))
        assert abs(got[1][i] - prob) <= prob * 2.0 ** -23 + 2 * unit * len(row), (i, setting)
    assert left_out * 4 <= len(rows)


def logits(rng, n, vocab, kind):
    if kind == "flat":
        return rng.normal(size=(n, vocab)).astype(np.float32) * 0.01
    if kind == "equal":
        return np.full((n, vocab), -3.25, np.float32)
    x = rng.normal(size=(n, vocab)).astype(np.float32) * 3
    if kind == "ties":  # few values, each many times; both zeros among them
        x = np.round(x)
        x[:, ::3] *= np.where(x[:, ::3] == 0, -1, 1).astype(np.float32)
        x = np.where((x == 0) & (rng.random(x.shape) < 0.5), np.float32(-0.0), x)
    if kind == "banned":
        x[:, rng.random(vocab) < 0.7] = -np.inf
        x[:, vocab // 2] = 0.5
    if kind == "wide":
        x *= 1e4
    return x.astype(np.float32)


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 255, 1000, 1023, 1024, 1025, 4099, 32003, 128256, 262144])
@pytest.mark.parametrize("kind", ["plain", "ties", "flat", "equal", "banned", "wide"])
def test_rows_of_settings(s, vocab, kind):
    print(f"[case] sample vocab={vocab} {kind}", flush=True)
    rng = np.random.default_rng(vocab * 7 + len(kind))
    x = logits(rng, len(ROWS), vocab, kind)
    u = rng.random(len(ROWS)).astype(np.float32)
    u = np.minimum(u, np.float32(1 - 2.0 ** -24))
    compare(x, u, ROWS, run(s, x, u, ROWS))
    s.sync()


@pytest.mark.parametrize("setting", ROWS)
def test_one_setting_for_all_rows_gives_the_same(s, setting):
    rng = np.random.default_rng(5)
    x = logits(rng, 7, 5003, "plain")
    u = rng.random(7).astype(np.float32)
    a, b = run(s, x, u, [setting] * 7), run(s, x, u, [setting] * 7, per_row=False)
    compare(x, u, [setting] * 7, a)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("vocab", [77, 5001, 128256])
def test_uniform_numbers_at_their_ends(s, vocab):
    rng = np.random.default_rng(3)
    x = np.repeat(logits(rng, 1, vocab, "plain"), 2, 0)
    rows = [(1.0, 0, 1.0, 0.0)] * 2
    u = np.array([0.0, 1 - 2.0 ** -24], np.float32)
    tokens, _ = run(s, x, u, rows)
    # u = 0: the first token whose weight counts
    w = np.exp(x[0].astype(np.float64) - x[0].max())
    assert tokens[0] == int(np.nonzero(w >= 2.0 ** -40)[0][0])
    assert tokens[1] == drafts.sample(x[1], u[1], *rows[1])[0]


def test_every_token_comes_as_often_as_its_weight(s):
    """Evenly spaced numbers: each token's count is its probability's, to one at either end of its range."""
    rng = np.random.default_rng(11)
    n = 4096
    x = np.repeat(logits(rng, 1, 37, "plain"), n, 0)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    for setting in [(1.0, 0, 1.0, 0.0), (0.7, 9, 0.9, 0.0)]:
        tokens, probs = run(s, x, u, [setting] * n)
        for t in np.unique(tokens):
            assert abs((tokens == t).sum() - probs[tokens == t][0] * n) <= 1 + 1e-3


def test_rows_do_not_depend_on_their_neighbours(s):
    rng = np.random.default_rng(2)
    x = logits(rng, 48, 9001, "plain")
    u = rng.random(48).astype(np.float32)
    rows = [ROWS[i % len(ROWS)] for i in range(48)]
    whole = run(s, x, u, rows)
    for i in (0, 17, 47):
        one = run(s, x[i:i + 1], u[i:i + 1], rows[i:i + 1])
        assert one[0][0] == whole[0][i] and one[1][0] == whole[1][i]


def test_no_probabilities_and_an_offset_buffer(s):
    import torch

    from spissa_amd.device import SamplingConfig

    rng = np.random.default_rng(9)
    x = logits(rng, 3, 4099, "plain")
    u = rng.random(3).astype(np.float32)
    buf = torch.empty(3 * 4099 + 1, device="cuda")
    buf[1:] = torch.as_tensor(x.reshape(-1), device="cuda")  # rows at no multiple of 16 bytes
    tokens = torch.full((5,), -7, dtype=torch.int32, device="cuda")
    s.sample(buf[1:], torch.as_tensor(u, device="cuda"), SamplingConfig(0.9, 40, 0.9, 0.0), tokens)
    s.sync()
    assert tokens.tolist() == [drafts.sample(x[i], u[i], 0.9, 40, 0.9, 0.0)[0] for i in range(3)] + [-7, -7]


@pytest.mark.parametrize("what", ["nan", "inf", "none", "u1", "u-", "unan", "t-", "tnan", "p", "m"])
def test_bad_rows_are_reported_and_leave_the_others(gpu, s, what):
    print(f"[case] bad row {what}", flush=True)
    rng = np.random.default_rng(4)
    x = logits(rng, 3, 3001, "plain")
    u = rng.random(3).astype(np.float32)
    rows = [(0.8, 50, 0.95, 0.05)] * 3
    if what == "nan":
        x[1, 2999] = np.nan
    elif what == "inf":
        x[1, 5] = np.inf
    elif what == "none":
        x[1] = -np.inf
    elif what[0] == "u":
        u[1] = {"u1": 1.0, "u-": -0.25, "unan": np.nan}[what]
    else:
        rows[1] = {"t-": (-1.0, 0, 1.0, 0.0), "tnan": (np.nan, 0, 1.0, 0.0), "p": (1.0, 0, 1.5, 0.0), "m": (1.0, 0, 1.0, -1.0)}[what]
    tokens, probs = run(s, x, u, rows)
    with pytest.raises(gpu.InvalidTensorDataError):
        s.sync()
    s.sync()  # reported once
    assert tokens[1] == -1 and probs[1] == 0
    for i in (0, 2):
        assert tokens[i] == drafts.sample(x[i], u[i], *rows[i])[0]


def test_no_rows(s):
    import torch

    from spissa_amd.device import SamplingConfig

    none = torch.empty(0, device="cuda")
    s.sample(none, none, SamplingConfig(), none.int())
    s.sync()


def test_refusals(gpu, s):
    import torch

    from spissa_amd.device import SamplingConfig

    x, u, t = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (SamplingConfig(-1.0), SamplingConfig(top_p=2.0), SamplingConfig(min_p=-0.5)):
        with pytest.raises(gpu.InvalidTensorDataError):
            s.sample(x, u, bad, t)
    with pytest.raises(TypeError):
        s.sample(x, u, SamplingConfig(temperature=torch.ones(1, device="cuda")), t)
    with pytest.raises(TypeError):
        s.sample(x, u, SamplingConfig(top_k=torch.ones(2, device="cuda")), t)
    with pytest.raises(TypeError):
        s.sample(x, u, SamplingConfig(), t[:1])
    with pytest.raises(TypeError):
        s.sample(x[:, :5], u, SamplingConfig(), t)
    assert _ffi.load().spissa_sample_device(s.handle, None, u.data_ptr(), SamplingConfig()._c(2, 8), t.data_ptr(), None) == _ffi.ERR_ARGUMENT


def test_two_captured_calls_in_turn_with_eager_ones(gpu):
    """Two graphs of one session share its workspace: replayed in turn, with new inputs and eager calls between."""
    import torch

    from spissa_amd.device import SamplingConfig, Session

    stream = torch.cuda.Stream()
    ses = Session(0, stream=stream)
    rng = np.random.default_rng(8)
    shapes, sets = [(3, 128256), (40, 5003)], []
    with torch.cuda.stream(stream):
        for n, vocab in shapes:
            rows = [ROWS[i % len(ROWS)] for i in range(n)]
            cols = list(zip(*rows))
            cfg = SamplingConfig(*(torch.tensor(c, dtype=torch.int32 if i == 1 else torch.float32, device="cuda") for i, c in enumerate(cols)))
            st = {"rows": rows, "cfg": cfg, "x": torch.zeros(n, vocab, device="cuda"), "u": torch.zeros(n, device="cuda"),
                  "t": torch.zeros(n, dtype=torch.int32, device="cuda"), "p": torch.zeros(n, device="cuda")}
            ses.sample(st["x"], st["u"], cfg, st["t"], st["p"])
            sets.append(st)
        ses.sync()
        for st in sets:
            st["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(st["graph"], stream=stream):
                ses.sample(st["x"], st["u"], st["cfg"], st["t"], st["p"])
        for _ in range(3):
            for st in sets:
                n, vocab = st["x"].shape
                x, u = logits(rng, n, vocab, "plain"), rng.random(n).astype(np.float32)
                st["x"].copy_(torch.as_tensor(x, device="cuda"))
                st["u"].copy_(torch.as_tensor(u, device="cuda"))
                st["t"].fill_(-9)
                st["graph"].replay()
                got = st["t"].cpu().numpy(), st["p"].cpu().numpy()
                compare(x, u, st["rows"], got)
                eager = torch.zeros_like(st["t"])
                ses.sample(st["x"], st["u"], st["cfg"], eager)
                ses.sync()
                assert np.array_equal(eager.cpu().numpy(), got[0])


HARD = [(1.0, 20000, 1.0, 0.0), (0.8, 20000, 0.9, 0.0), (0.8, 9000, 1.0, 0.001), (1.5, 1000, 0.7, 0.0), (50.0, 0, 0.3, 0.0),
        (1.0, 300, 0.999, 0.0), (1e-4, 5000, 0.9, 0.0), (0.05, 257, 1.0, 0.0), (1.0, 256, 0.5, 0.0), (20.0, 12000, 0.99, 0.0)]


@pytest.mark.parametrize("vocab", [300, 1537, 8191, 8192, 8193, 40001, 131073, 300001])
@pytest.mark.parametrize("kind", ["plain", "ties", "flat", "equal"])
def test_limits_among_thousands(s, vocab, kind):
    """Lists that fill, overflow, or end among many equal tokens, on either side of the longest row of one workgroup."""
    print(f"[case] sample vocab={vocab} {kind} limits among thousands", flush=True)
    rng = np.random.default_rng(vocab + len(kind))
    x = logits(rng, len(HARD), vocab, kind)
    u = np.minimum(rng.random(len(HARD)), 1 - 2.0 ** -24).astype(np.float32)
    compare(x, u, HARD, run(s, x, u, HARD))
    s.sync()


def test_the_longest_rows(s):
    """2^22 logits a row: runs of several granules a thread."""
    rng = np.random.default_rng(22)
    x = logits(rng, 4, 1 << 22, "plain")
    rows = [(1.0, 0, 1.0, 0.0), (0.9, 50, 0.95, 0.0), (1.2, 0, 0.9, 0.0), (3.0, 20000, 0.9, 0.0)]
    for u in ([0.0, 0.25, 0.5, 0.999], [0.75, 0.9, 0.125, 0.3]):
        compare(x, u, rows, run(s, x, u, rows))
    s.sync()


@pytest.mark.parametrize("n,vocab", [(1025, 9001), (2049, 1000), (65535, 5)])
def test_more_rows_than_a_round_of_launches(s, n, vocab):
    rng = np.random.default_rng(n)
    x = logits(rng, 16, vocab, "plain")[np.arange(n) % 16]
    u = np.minimum(rng.random(n), 1 - 2.0 ** -24).astype(np.float32)
    rows = [ROWS[i % 7] for i in range(n)]
    tokens, probs = run(s, x, u, rows)
    at = np.unique(np.concatenate([[0, 1022, 1023, 1024, n - 1], rng.integers(0, n, 20)]))
    compare(x[at], u[at], [rows[i] for i in at], (tokens[at], probs[at]))
    assert (tokens >= 0).all() and (tokens < vocab).all()
    s.sync()


def test_two_sessions_at_once():
    """Two sessions of two threads and streams: workspaces of their own, and the same tokens as alone."""
    import threading

    import torch

    from spissa_amd.device import SamplingConfig, Session

    rng = np.random.default_rng(6)
    x = torch.as_tensor(logits(rng, 8, 50001, "plain"), device="cuda")
    u = torch.as_tensor(rng.random(8).astype(np.float32), device="cuda")
    cfgs = [SamplingConfig(0.9, 40, 0.9, 0.0), SamplingConfig(1.2, 0, 0.8, 0.01)]
    torch.cuda.synchronize()
    want, got, failed = [None] * 2, [[], []], []

    def work(i, rounds):
        try:
            stream = torch.cuda.Stream()
            ses = Session(0, stream=stream)
            with torch.cuda.stream(stream):
                for _ in range(rounds):
                    t = torch.zeros(8, dtype=torch.int32, device="cuda")
                    ses.sample(x, u, cfgs[i], t)
                    got[i].append(t)
                ses.sync()
        except Exception as e:  # (shown by the main thread)
            failed.append(e)

    for i in range(2):
        work(i, 1)
        want[i] = got[i].pop().tolist()
    threads = [threading.Thread(target=work, args=(i, 30)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    assert all(t.tolist() == want[i] for i in range(2) for t in got[i])


@pytest.mark.parametrize("vocab", [2047, 2049, 10007, 12287, 12288, 12289])
@pytest.mark.parametrize("kind", ["plain", "ties", "banned", "equal", "wide"])
def test_rows_about_the_longest_of_one_workgroup(s, vocab, kind):
    print(f"[case] sample vocab={vocab} {kind} about the longest row of one workgroup", flush=True)
    rng = np.random.default_rng(vocab * 3 + len(kind))
    rows = ROWS + HARD
    x = logits(rng, len(rows), vocab, kind)
    u = np.minimum(rng.random(len(rows)), 1 - 2.0 ** -24).astype(np.float32)
    compare(x, u, rows, run(s, x, u, rows))
    s.sync()


def within(x, setting, tokens, probs):
    """Each probability against the definition's of that token: weights off by (1 + 60) * 2^-52 of themselves in 64 bits
    (logits up to 60 temperatures down), their sum by half a step of 2^-shift a token, one rounding to f32."""
    for row, token, prob in zip(x.astype(np.float64), tokens, probs):
        w = np.exp((row - row.max()) / np.float64(np.float32(setting[0])))
        order = np.argsort(-row, kind="stable")[:setting[1] or None]
        if setting[2] < 1:
            run = np.cumsum(w[order])
            order = order[:max(1, int(((run - w[order]) < np.float64(np.float32(setting[2])) * run[-1]).sum()))]
        want = w[token] / w[order].sum()
        lost = len(row) * 2.0 ** -(1 + min(51, 62 - int(np.ceil(np.log2(max(2, len(row)))))))
        assert token in order and abs(prob - want) <= want * (2.0 ** -24 + 2.0 ** -45 + lost), (setting, token, prob, want)


@pytest.mark.parametrize("vocab", [700, 12288, 12289, 262144, 1 << 22])
@pytest.mark.parametrize("down", [18.0, 24.0, 27.0])
@pytest.mark.parametrize("filters", [False, True])
def test_probabilities_of_rare_tokens(s, vocab, down, filters):
    """All but one logit `down` temperatures below it and the number above its share: one of them is drawn, with its own
    probability (weights there are few steps of the whole numbers that are summed)."""
    print(f"[case] sample vocab={vocab} rare tokens {down} down filters={filters}", flush=True)
    rng = np.random.default_rng(vocab)
    x = (np.float32(-down) + rng.uniform(-0.3, 0.3, (3, vocab))).astype(np.float32)
    x[:, vocab // 3] = 0.0
    x *= np.float32(0.75)
    share = vocab * np.exp(-down)
    # the largest token comes after a third of the others: numbers before and behind its share
    u = np.array([0.0, 0.2 * share / (1 + share), 1 - 2.0 ** -24], np.float32)
    setting = (0.75, 0, 1.0, 0.0) if not filters else (0.75, vocab - 1, 1.0, 0.0)
    tokens, probs = run(s, x, u, [setting] * 3)
    s.sync()
    assert tokens[0] != vocab // 3
    within(x, setting, tokens, probs)


def test_rows_by_the_logits_shape(s):
    """[rows, vocab], further leading dimensions, or all in one: the same tokens; another number of rows is refused."""
    import torch

    from spissa_amd.device import SamplingConfig

    rng = np.random.default_rng(14)
    x, u = torch.as_tensor(logits(rng, 4, 1000, "plain"), device="cuda"), torch.as_tensor(rng.random(4).astype(np.float32), device="cuda")
    got = []
    for view in (x, x.view(2, 2, 1000), x.view(-1)):
        t = torch.full((4,), -7, dtype=torch.int32, device="cuda")
        s.sample(view, u, SamplingConfig(0.9, 40, 0.9, 0.0), t)
        got.append(t.tolist())
    s.sync()
    assert got[0] == got[1] == got[2] and min(got[0]) >= 0
    t = torch.full((4,), -7, dtype=torch.int32, device="cuda")
    with pytest.raises(TypeError, match="rows"):
        s.sample(x, u[:2], SamplingConfig(), t)
    assert t.tolist() == [-7] * 4


# ---- rows of several workgroups: the calls above, past the longest row of one


def border(vocab):
    """How far the sums of whole numbers may be off: half a step of each token's weight, and 2^-45 for the weights
    themselves in 64 bits, over a sum of at least 1."""
    return vocab * 2.0 ** -(1 + min(51, 62 - int(np.ceil(np.log2(max(2, vocab)))))) + 2.0 ** -45


def same(x, u, rows, got):
    left_out = 0
    for i, (row, setting) in enumerate(zip(x, rows)):
        token, prob, near = drafts.sample(row, u[i], *setting)
        if near < border(len(row)):
            left_out += 1
            continue
        assert got[0][i] == token, (i, setting, got[0][i], token, prob)
        assert abs(got[1][i] - prob) <= prob * (2.0 ** -24 + border(len(row))), (i, setting)
    assert left_out * 4 <= len(rows)


@pytest.mark.parametrize("vocab", [12289, 32003, 262144])
@pytest.mark.parametrize("setting", ROWS)
def test_one_setting_for_all_long_rows(s, vocab, setting):
    print(f"[case] sample vocab={vocab} by numbers {setting}", flush=True)
    rng = np.random.default_rng(15)
    x = logits(rng, 3, vocab, "plain")
    u = rng.random(3).astype(np.float32)
    a, b = run(s, x, u, [setting] * 3), run(s, x, u, [setting] * 3, per_row=False)
    s.sync()
    same(x, u, [setting] * 3, a)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("vocab", [32003, 128256])
def test_long_rows_do_not_depend_on_their_neighbours(s, vocab):
    rng = np.random.default_rng(16)
    x = logits(rng, 48, vocab, "plain")
    u = rng.random(48).astype(np.float32)
    rows = [ROWS[i % len(ROWS)] for i in range(48)]
    whole = run(s, x, u, rows)
    for i in (0, 17, 31, 47):
        one = run(s, x[i:i + 1], u[i:i + 1], rows[i:i + 1])
        assert one[0][0] == whole[0][i] and one[1][0] == whole[1][i]
    s.sync()


@pytest.mark.parametrize("vocab", [12289, 40003])
@pytest.mark.parametrize("setting", [(0.9, 40, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (0.7, 0, 0.8, 0.01), (0.0, 0, 1.0, 0.0)])
def test_long_rows_without_probabilities_in_an_offset_buffer(s, vocab, setting):
    import torch

    from spissa_amd.device import SamplingConfig

    rng = np.random.default_rng(17)
    x = logits(rng, 3, vocab, "plain")
    u = rng.random(3).astype(np.float32)
    buf = torch.full((3 * vocab + 9,), float("nan"), device="cuda")
    buf[1:1 + 3 * vocab] = torch.as_tensor(x.reshape(-1), device="cuda")  # rows at no multiple of 16 bytes, none behind them
    tokens = torch.full((5,), -7, dtype=torch.int32, device="cuda")
    s.sample(buf[1:1 + 3 * vocab], torch.as_tensor(u, device="cuda"), SamplingConfig(*setting), tokens)
    s.sync()
    assert tokens.tolist() == [drafts.sample(x[i], u[i], *setting)[0] for i in range(3)] + [-7, -7]


@pytest.mark.parametrize("filters", [False, True])
@pytest.mark.parametrize("what", ["nan", "inf", "none", "u1", "u-", "unan", "t-", "tnan", "p", "m"])
def test_bad_long_rows_are_reported_and_leave_the_others(gpu, s, what, filters):
    """The bad number in a slice that is not the first, or in the settings."""
    print(f"[case] bad long row {what} filters={filters}", flush=True)
    rng = np.random.default_rng(18)
    x = logits(rng, 3, 40001, "plain")
    u = rng.random(3).astype(np.float32)
    rows = [(0.8, 50, 0.95, 0.05) if filters else (0.8, 0, 1.0, 0.0)] * 3
    if what == "nan":
        x[1, 39999] = np.nan
    elif what == "inf":
        x[1, 20005] = np.inf
    elif what == "none":
        x[1] = -np.inf
    elif what[0] == "u":
        u[1] = {"u1": 1.0, "u-": -0.25, "unan": np.nan}[what]
    else:
        rows[1] = {"t-": (-1.0, 0, 1.0, 0.0), "tnan": (np.nan, 0, 1.0, 0.0), "p": (1.0, 0, 1.5, 0.0), "m": (1.0, 0, 1.0, -1.0)}[what]
    tokens, probs = run(s, x, u, rows)
    with pytest.raises(gpu.InvalidTensorDataError):
        s.sync()
    s.sync()
    assert tokens[1] == -1 and probs[1] == 0
    for i in (0, 2):
        assert tokens[i] == drafts.sample(x[i], u[i], *rows[i])[0]


@pytest.mark.parametrize("n,vocab", [(1025, 12289), (2051, 16001)])
@pytest.mark.parametrize("per_row", [False, True])
def test_more_long_rows_than_a_round_of_launches(s, n, vocab, per_row):
    """The second round's workspace is the first's; its pointers go on where the first ended."""
    print(f"[case] sample {n} x {vocab} per_row={per_row}", flush=True)
    rng = np.random.default_rng(n)
    x = logits(rng, 16, vocab, "plain")[np.arange(n) % 16]
    u = np.minimum(rng.random(n), 1 - 2.0 ** -24).astype(np.float32)
    for setting in [None] if per_row else [(1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.05)]:
        rows = [ROWS[i % 7] for i in range(n)] if per_row else [setting] * n
        tokens, probs = run(s, x, u, rows, per_row)
        s.sync()
        at = np.unique(np.concatenate([[0, 1022, 1023, 1024, n - 1], rng.integers(0, n, 12)]))
        same(x[at], u[at], [rows[i] for i in at], (tokens[at], probs[at]))
        assert (tokens >= 0).all() and (tokens < vocab).all()


def test_captured_calls_of_long_rows_and_the_walk_behind_them(gpu):
    """Two graphs of one session, each sampling long rows (by arrays, by numbers without filters) and walking a tree by what
    came: replayed in turn with new inputs, eager calls between."""
    import torch

    from spissa_amd.device import SamplingConfig, Session

    stream = torch.cuda.Stream()
    ses = Session(0, stream=stream)
    rng = np.random.default_rng(19)
    parents = drafts.make_tree(rng, 12, 4)
    with torch.cuda.stream(stream):
        sets = []
        for n, vocab, arrays in [(12, 20011, True), (12, 128256, False)]:
            rows = [ROWS[i % len(ROWS)] if arrays else (0.02, 0, 1.0, 0.0) for i in range(n)]
            cols = list(zip(*rows))
            cfg = SamplingConfig(*(torch.tensor(c, dtype=torch.int32 if i == 1 else torch.float32, device="cuda") for i, c in enumerate(cols))
                                 if arrays else rows[0])
            i32 = lambda m: torch.zeros(m, dtype=torch.int32, device="cuda")  # noqa: E731
            st = {"rows": rows, "x": torch.zeros(n, vocab, device="cuda"), "u": torch.zeros(n, device="cuda"), "p": torch.zeros(n, device="cuda"),
                  "parents": torch.tensor(parents, dtype=torch.int32, device="cuda"), "drafted": i32(n), "t": i32(n), "walk": [i32(n), i32(1), i32(1)]}

            def step(st=st, cfg=cfg, n=n):
                ses.sample(st["x"], st["u"], cfg, st["t"], st["p"])
                ses.tree_accept(st["parents"], st["drafted"], st["t"], [n], *st["walk"])

            step()
            sets.append((st, step))
        ses.sync()
        graphs = []
        for st, step in sets:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                step()
        walked = 0
        for _ in range(3):
            for (st, step), g in zip(sets, graphs):
                n, vocab = st["x"].shape
                x, u = logits(rng, n, vocab, "plain"), rng.random(n).astype(np.float32)
                # drafts that sampling often confirms: the largest logit after the parent
                drafted = np.array([x[max(0, p)].argmax() for p in parents], np.int32)
                for name, v in (("x", x), ("u", u), ("drafted", drafted)):
                    st[name].copy_(torch.as_tensor(v, device="cuda"))
                st["t"].fill_(-9)
                g.replay()
                got = [v.cpu().numpy().copy() for v in (st["t"], st["p"], *st["walk"])]
                same(x, u, st["rows"], got)
                path, last = drafts.accept(parents, drafted, got[0])
                assert got[2].tolist() == path + [-1] * (n - len(path)) and got[3][0] == len(path) and got[4][0] == last
                walked = max(walked, len(path))
                step()
                ses.sync()
                assert all(np.array_equal(a, b.cpu().numpy()) for a, b in zip(got, (st["t"], st["p"], *st["walk"])))
        assert walked > 1
