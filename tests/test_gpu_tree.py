"""Drafted tokens on the device: the tree step, the walk along confirmed nodes and the
move of their rows, against plain forms in 64 bits.

Tolerance of the attention: of each output row (a node and head, D channels) the
2-norm of the difference over the row's own 2-norm, at most ROW. The products take
queries, keys, weights and values as two pieces, off by 2^-23 of themselves each
(2^-24.8 in the mean square), the sums of up to D products and of a row's keys are f32,
off by at most sqrt(256) * 2^-24.8 of their terms' root of squares: for inputs N(0, 1)
a score is off by about 7e-7 in the mean square, a weight by that share of itself, and
the output, a sum of values with independent signs, likewise: 1e-6, of which one row
of a few thousand may be some five times off. 1e-5 leaves a factor of two above that.
Rows that are appended are bit for bit what the rotation alone gives.
"""
import numpy as np
import pytest

from spissa_amd import _ffi
from tests import drafts

pytestmark = pytest.mark.gpu

ROW = 1e-5
HEADS = [(4, 4, 64), (32, 8, 64), (24, 8, 128), (5, 1, 128), (4, 1, 256), (8, 4, 256), (16, 1, 64)]


@pytest.fixture(scope="module")
def s(gpu):
    import torch

    from spissa_amd.device import Session

    stream = torch.cuda.Stream()
    session = Session(0, stream=stream)
    with torch.cuda.stream(stream):
        yield session


def dev(x):
    import torch

    return torch.as_tensor(np.ascontiguousarray(x), device="cuda")


def tables(s, kind, d, rows):
    """A rope table and its rows on the host, from rotating (1, 0) pairs."""
    import torch

    t = s.rope_table(kind, d, 500000.0, max_positions=rows)
    unit = torch.zeros(rows, 1, d, device="cuda")
    unit[..., :d // 2] = 1.0
    other = torch.zeros_like(unit)
    s.rope_apply(t, unit, other, rows, 1, 1, d, 0)
    u = unit.cpu().numpy()[:, 0]
    return t, u[:, :d // 2].copy(), u[:, d // 2:].copy()


class Draft:
    """Caches, trees and inputs of one step, on the device and as the plain form has them."""

    def __init__(self, s, rng, heads, past, nodes, reach=5, roots=0.0, scale=1.0, vscale=1.0, room=4):
        self.hq, self.hkv, self.d = heads
        self.past, self.nodes = past, nodes
        self.parents = [drafts.make_tree(rng, n, reach, roots) for n in nodes]
        f = lambda *shape: rng.normal(size=shape).astype(np.float32)  # noqa: E731
        self.pk = [f(p, self.hkv, self.d) * np.float32(scale) for p in past]
        self.pv = [f(p, self.hkv, self.d) * np.float32(vscale) for p in past]
        n = sum(nodes)
        self.q, self.k, self.v = f(n, self.hq, self.d), f(n, self.hkv, self.d) * np.float32(scale), f(n, self.hkv, self.d) * np.float32(vscale)
        self.caches = [self.cache(s, i, room) for i in range(len(past))]

    def cache(self, s, i, room=4):
        c = s.kv_cache(self.hkv, self.d, self.past[i] + self.nodes[i] + room)
        if self.past[i]:
            s.append(c, dev(self.pk[i]), dev(self.pv[i]), self.past[i])
        return c

    def config(self, window=0):
        from spissa_amd.rotary import KvAttentionConfig

        return KvAttentionConfig(sum(self.nodes), self.hq, self.hkv, self.d, True, window)

    def flat_parents(self):
        return dev(np.array(sum(self.parents, []), np.int32))

    def run(self, s, table=None, window=0, norm=None, prescale=1.0, eps=1e-6, parents=None):
        out = dev(np.full(self.q.shape, np.nan, np.float32))
        args = (table, dev(self.q), dev(self.k), dev(self.v), self.caches, self.nodes, self.flat_parents() if parents is None else parents, self.config(window))
        if norm:
            s.gemma_tree_step(*args, dev(norm[0]), dev(norm[1]), eps, prescale, out)
        else:
            s.tree_step(*args, out)
        return out

    def plain(self, tab=None, window=0, norm=None, prescale=1.0, eps=1e-6):
        """Outputs and rows [n, hkv, d] of keys."""
        outs, rows, at = [], [], 0
        for p, parents, pk, pv in zip(self.past, self.parents, self.pk, self.pv):
            n = len(parents)
            q, k, v = (x[at:at + n] for x in (self.q, self.k, self.v))
            at += n
            if n == 0:
                continue
            if norm:
                q, k = drafts.norm(q, norm[0], eps), drafts.norm(k, norm[1], eps)
            if tab:
                pos = p + np.array(drafts.depths(parents))
                q, k = drafts.rotate(q, pos, *tab), drafts.rotate(k, pos, *tab)
            rows.append(k)
            outs.append(drafts.attend(q * prescale, np.concatenate([pk, k]), np.concatenate([pv, v]), drafts.seen(parents, p, window)))
        return np.concatenate(outs), np.concatenate(rows)


def rows_off(got, want):
    d = got.astype(np.float64) - want
    return float((np.linalg.norm(d, axis=-1) / np.linalg.norm(want, axis=-1)).max())


def held(s, cache, first, count):
    import torch

    k, v = (torch.zeros(count, cache.num_heads(), cache.head_dim(), device="cuda") for _ in range(2))
    s.cache_rows(cache, first, count, k, v)
    return k.cpu().numpy(), v.cpu().numpy()


STEPS = [  # past, nodes, window
    ([0], [1], 0), ([0], [7], 0), ([1], [1], 0), ([5], [3], 0), ([31], [33], 0), ([32], [32], 0), ([63], [2], 0), ([64], [64], 0),
    ([65], [65], 0), ([127], [5], 0), ([128], [31], 0), ([129], [129], 0), ([500], [256], 0), ([1000], [17], 0), ([2049], [26], 0),
    ([300], [20], 1), ([300], [20], 2), ([300], [40], 7), ([513], [30], 64), ([777], [12], 200), ([10], [25], 100), ([700], [90], 65),
    ([0, 3, 700, 64], [4, 1, 9, 64], 0), ([40, 0, 333], [0, 5, 3], 0), ([100] * 17, [2] * 17, 0), ([900, 20, 1], [3, 70, 11], 33)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("past,nodes,window", STEPS)
def test_step(s, heads, past, nodes, window):
    print(f"[case] tree step heads={heads} past={past[:4]} nodes={nodes[:4]} window={window}", flush=True)
    rng = np.random.default_rng(sum(past) * 31 + sum(nodes) + heads[0])
    dr = Draft(s, rng, heads, past, nodes, roots=0.1 if window % 2 else 0.0)
    table, cos, sin = tables(s, _ffi.ROPE_LLAMA, heads[2], max(past) + max(nodes) + 1)
    out = dr.run(s, table, window)
    s.sync()
    want, _ = dr.plain((cos, sin), window)
    assert rows_off(out.cpu().numpy(), want) <= ROW
    at = 0
    for c, p, n, parents, pk, pv in zip(dr.caches, past, nodes, dr.parents, dr.pk, dr.pv):
        assert len(c) == p + n
        k, v = held(s, c, 0, p + n)
        # the rows before stay, the new ones are the rotation's to the bit
        assert np.array_equal(k[:p], pk) and np.array_equal(v[:p], pv) and np.array_equal(v[p:], dr.v[at:at + n])
        for t, e in enumerate(drafts.depths(parents)):
            row, none = dev(dr.k[at + t:at + t + 1]), dev(np.zeros((1, heads[1], heads[2]), np.float32))
            s.rope_apply(table, row, none, 1, heads[1], heads[1], heads[2], p + e)
            if t % 7 == 0:
                assert np.array_equal(row.cpu().numpy()[0], k[p + t])
        at += n


@pytest.mark.parametrize("heads", [(24, 8, 128), (8, 4, 256), (4, 2, 64)])
@pytest.mark.parametrize("past,nodes,window", [([0], [1], 0), ([70], [33], 0), ([600, 9], [12, 40], 64)])
def test_gemma_step(s, heads, past, nodes, window):
    print(f"[case] gemma tree step heads={heads} past={past} nodes={nodes} window={window}", flush=True)
    rng = np.random.default_rng(sum(past) + heads[2])
    dr = Draft(s, rng, heads, past, nodes)
    norm = [(1 + 0.25 * rng.normal(size=heads[2])).astype(np.float32) for _ in range(2)]
    table, cos, sin = tables(s, _ffi.ROPE_GEMMA, heads[2], max(past) + max(nodes) + 1)
    out = dr.run(s, table, window, norm, 0.75)
    s.sync()
    want, rows = dr.plain((cos, sin), window, norm, 0.75)
    assert rows_off(out.cpu().numpy(), want) <= ROW
    at = 0
    for c, p, n in zip(dr.caches, past, nodes):
        # the sum of squares as a tree (8 roundings), the root, the division, two products, the rotation: 16 roundings
        assert rows_off(held(s, c, p, n)[0], rows[at:at + n]) <= 16 * 2.0 ** -24
        at += n


def test_no_table(s):
    dr = Draft(s, np.random.default_rng(0), (24, 8, 128), [100], [9])
    out = dr.run(s)
    s.sync()
    assert rows_off(out.cpu().numpy(), dr.plain()[0]) <= ROW


@pytest.mark.parametrize("heads", [(24, 8, 128), (32, 8, 64), (4, 1, 256)])
@pytest.mark.parametrize("past", [3, 700])
def test_a_chain_is_as_many_decode_steps(s, heads, past):
    from spissa_amd.rotary import KvAttentionConfig

    rng = np.random.default_rng(past)
    dr = Draft(s, rng, heads, [past], [6])
    dr.parents = [[-1, 0, 1, 2, 3, 4]]
    table, *_ = tables(s, _ffi.ROPE_LLAMA, heads[2], past + 8)
    one = dr.cache(s, 0)
    out = dr.run(s, table).cpu().numpy()
    cfg = KvAttentionConfig(1, *heads, True, 0)
    for t in range(6):
        o = dev(np.zeros_like(dr.q[:1]))
        s.decode_step(table, dev(dr.q[t:t + 1]), dev(dr.k[t:t + 1]), dev(dr.v[t:t + 1]), [one], cfg, o)
        assert rows_off(out[t:t + 1], o.cpu().numpy().astype(np.float64)) <= 2 * ROW  # (each side's own)
    a, b = held(s, dr.caches[0], 0, past + 6), held(s, one, 0, past + 6)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    s.sync()


@pytest.mark.parametrize("heads", [(24, 8, 128), (8, 2, 64), (4, 1, 256)])
@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_what_is_not_finite_reaches_only_those_that_see_it(gpu, s, heads, where, what):
    print(f"[case] {what} in a drafted {where} {heads}", flush=True)
    rng = np.random.default_rng(1)
    dr = Draft(s, rng, heads, [150, 40], [40, 7])
    bad = 11
    (dr.k if where == "key" else dr.v)[bad, heads[1] - 1, 5] = what
    out = dr.run(s).cpu().numpy()
    with pytest.raises(gpu.InvalidTensorDataError):
        s.sync()
    s.sync()
    dr.k[bad] = dr.v[bad] = 0
    want, _ = dr.plain()
    sees = np.zeros(47, bool)
    sees[:40] = drafts.seen(dr.parents[0], 0)[:, bad]
    assert sees.any() and not sees.all()
    assert rows_off(out[~sees], want[~sees]) <= ROW
    group = heads[0] // heads[1]
    assert np.isnan(out[sees][:, -group:]).all()  # the heads of the KV head that has it


@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("what", [np.nan, np.inf])
def test_what_is_not_finite_in_the_cache(gpu, s, where, what):
    """Outside the window it takes no part; inside, those that see it are NaN."""
    rng = np.random.default_rng(6)
    dr = Draft(s, rng, (8, 2, 128), [400], [30])
    depth = np.array(drafts.depths(dr.parents[0]))
    window = 100
    at = 400 + 4 + 1 - window - 1  # seen by depths 0..3
    (dr.pk if where == "key" else dr.pv)[0][at] = what
    dr.caches = [dr.cache(s, 0)]
    out = dr.run(s, window=window).cpu().numpy()
    with pytest.raises(gpu.InvalidTensorDataError):
        s.sync()
    dr.pk[0][at] = dr.pv[0][at] = 0
    want, _ = dr.plain(window=window)
    sees = depth <= 3
    assert (~sees).any() and rows_off(out[~sees], want[~sees]) <= ROW and np.isnan(out[sees]).all()
    # a window that ends before it, for all
    dr.caches[0].truncate(400)
    out = dr.run(s, window=50).cpu().numpy()
    s.sync()
    assert rows_off(out, dr.plain(window=50)[0]) <= ROW


@pytest.mark.parametrize("heads", [(24, 8, 128), (8, 2, 64), (4, 1, 256)])
@pytest.mark.parametrize("scale,vscale", [(1e-6, 1e-6), (30.0, 1e6), (1e-3, 1e30), (1e-30, 1e-30)])
def test_values_of_any_size(s, heads, scale, vscale):
    rng = np.random.default_rng(3)
    dr = Draft(s, rng, heads, [333], [21], scale=scale, vscale=vscale)
    # scores as for N(0, 1), but for keys of a size to make one token take nearly all
    dr.q /= np.float32(min(scale, 1.0))
    out = dr.run(s)
    s.sync()
    # (scores of up to 30 times the size are off by as much more, relative to the weights)
    assert rows_off(out.cpu().numpy(), dr.plain()[0]) <= ROW * max(1.0, scale)


@pytest.mark.parametrize("heads", [(24, 8, 128), (8, 2, 64), (4, 1, 256)])
def test_keys_and_values_whose_size_grows_along_the_cache(s, heads):
    """Blocks of rows from 2^-20 to 2^20 in size, values with them."""
    rng = np.random.default_rng(4)
    dr = Draft(s, rng, heads, [1300], [21])
    steps = np.float32(2.0) ** np.linspace(-20, 20, 14).round().astype(np.float32).repeat(100)[:1300, None, None]
    dr.pv[0] *= steps
    dr.pk[0][::3] *= np.float32(1e-4)
    dr.caches = [dr.cache(s, 0)]
    out = dr.run(s)
    s.sync()
    want = dr.plain()[0]
    # every output is of the size of the largest values
    assert rows_off(out.cpu().numpy(), want) <= ROW
    # and with their sizes falling
    dr.pv[0] = dr.pv[0][::-1].copy()
    dr.caches = [dr.cache(s, 0)]
    out = dr.run(s)
    s.sync()
    assert rows_off(out.cpu().numpy(), dr.plain()[0]) <= ROW


def test_one_huge_key_among_ordinary_ones(s):
    rng = np.random.default_rng(12)
    dr = Draft(s, rng, (24, 8, 128), [600], [21])
    dr.pk[0][[0, 333]] *= np.float32(-1e5)
    dr.q = np.abs(dr.q)
    dr.pk[0][[0, 333]] = -np.abs(dr.pk[0][[0, 333]])  # so far below that it takes no weight
    dr.caches = [dr.cache(s, 0)]
    out = dr.run(s)
    s.sync()
    # (ordinary keys are then held to 2^-32 of 4e5: scores of |q| sqrt(128) 1e-4 / sqrt(128))
    assert rows_off(out.cpu().numpy(), dr.plain()[0]) <= 4e5 * 2.0 ** -32 * 8 + ROW


def test_parents_out_of_range_count_as_none(gpu, s):
    rng = np.random.default_rng(2)
    dr = Draft(s, rng, (8, 2, 64), [50, 20], [9, 5])
    wrong = [list(p) for p in dr.parents]
    wrong[0][4], wrong[0][6], wrong[1][2] = 4, 200, -2
    out = dr.run(s, parents=dev(np.array(sum(wrong, []), np.int32)))
    got = out.cpu().numpy()
    with pytest.raises(gpu.InvalidTensorDataError):
        s.sync()
    s.sync()
    dr.parents[0][4] = dr.parents[0][6] = dr.parents[1][2] = -1
    assert rows_off(got, dr.plain()[0]) <= ROW


def test_rows_behind_the_nodes_stay(s):
    import torch

    rng = np.random.default_rng(7)
    dr = Draft(s, rng, (24, 8, 128), [77], [10], room=20)
    c = dr.caches[0]
    s.append(c, torch.full((30, 8, 128), 7.0, device="cuda"), torch.full((30, 8, 128), 9.0, device="cuda"), 30)
    c.truncate(77)
    dr.run(s)
    s.sync()
    view = torch.as_tensor(type("R", (), {"__cuda_array_interface__": {"data": (c.device_keys_ptr(), False), "shape": (107, 8, 128),
                                                                        "typestr": "<f4", "version": 2}})(), device="cuda")
    assert (view[87:] == 7.0).all() and not (view[77:87] == 7.0).any()


def test_long_cache_past_32_bit_offsets(s):
    """Rows behind the first 4 GiB of a cache's keys."""
    import torch

    from spissa_amd.rotary import KvAttentionConfig

    hq, hkv, d, n, t = 8, 8, 128, (1 << 20) + 3000, 9
    c = s.kv_cache(hkv, d, n + t)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    half = n // 4
    for first in range(0, n, half):
        m = min(half, n - first)
        s.append(c, torch.zeros(m, hkv, d, device="cuda"), torch.zeros(m, hkv, d, device="cuda"), m)
    c.truncate(n - 2500)
    k, v = (torch.randn(2500, hkv, d, generator=gen, device="cuda") for _ in range(2))
    s.append(c, k, v, 2500)
    q, nk, nv = (torch.randn(t, hq, d, generator=gen, device="cuda") for _ in range(3))
    parents = [-1, 0, 0, 1, 2, 3, 3, 4, 7]
    out = torch.zeros_like(q)
    for window in (2000, 0):
        c.truncate(n)
        s.tree_step(None, q, nk, nv, [c], [t], dev(np.array(parents, np.int32)), KvAttentionConfig(t, hq, hkv, d, True, window), out)
        s.sync()
        kk, vv = (torch.cat([a, b]).cpu().numpy() for a, b in ((k, nk), (v, nv)))
        if window:
            want = drafts.attend(q.cpu().numpy(), kk, vv, drafts.seen(parents, 2500, window))
        else:  # the zeros before weigh exp(0) each and hold nothing
            qs = q.cpu().numpy().astype(np.float64)
            vis = drafts.seen(parents, 2500)
            want = np.empty(qs.shape)
            for i in range(t):
                sc = np.einsum("hd,mhd->hm", qs[i], kk[vis[i]].astype(np.float64)) / np.sqrt(d)
                top = np.maximum(0, sc.max(1, keepdims=True))
                p = np.exp(sc - top)
                want[i] = np.einsum("hm,mhd->hd", p, vv[vis[i]].astype(np.float64)) / (p.sum(1, keepdims=True) + (n - 2500) * np.exp(-top))
        # (a sum over 2^20 equal weights: 2^-24 for each of the rounds in which a workgroup and the merge add them)
        assert rows_off(out.cpu().numpy(), want) <= ROW * (1 if window else 4)


def test_refusals(gpu, s):
    from spissa_amd.device import Session
    from spissa_amd.rotary import KvAttentionConfig

    rng = np.random.default_rng(0)
    dr = Draft(s, rng, (8, 2, 64), [5, 6], [3, 4], room=0)
    table, *_ = tables(s, _ffi.ROPE_LLAMA, 64, 9)  # one position short
    before = [len(c) for c in dr.caches]

    def refused(error, caches=None, nodes=None, table=None, cfg=None, q=None, k=None):
        out = dev(np.zeros_like(dr.q))
        with pytest.raises(error):
            s.tree_step(table, dev(dr.q) if q is None else q, dev(dr.k) if k is None else k, dev(dr.v), caches or dr.caches,
                        nodes or dr.nodes, dr.flat_parents(), cfg or dr.config(), out)
        assert [len(c) for c in dr.caches] == before

    refused(gpu.ShapeError, table=table)
    refused(gpu.ShapeError, table=s.rope_table(_ffi.ROPE_NEOX, 64, 1e4, max_positions=64))
    refused(gpu.ShapeError, table=s.rope_table(_ffi.ROPE_LLAMA, 32, 1e4, max_positions=64))
    refused(gpu.ShapeError, nodes=[4, 3])  # past the first cache's capacity
    refused(gpu.ArgumentError, caches=[dr.caches[0], dr.caches[0]], nodes=[3, 4])
    refused(gpu.ArgumentError, caches=[dr.caches[0], s.q4_kv_cache(2, 64, 32)])
    refused(gpu.ShapeError, caches=[dr.caches[0], s.kv_cache(4, 64, 32)])
    refused(gpu.ShapeError, caches=[dr.caches[0], s.kv_cache(2, 128, 32)])
    refused(gpu.ShapeError, cfg=KvAttentionConfig(7, 8, 2, 64, False, 0))
    odd = dev(np.zeros(dr.q.size + 1, np.float32))[1:]
    refused(gpu.ArgumentError, q=odd)
    refused(TypeError, q=dev(dr.q[:6]))
    refused(TypeError, k=dev(dr.k[:6]))
    refused(TypeError, nodes=[7])
    g = s.rope_table(_ffi.ROPE_GEMMA, 64, 1e4, max_positions=64)
    w = dev(np.ones(64, np.float32))
    args = (dev(dr.q), dev(dr.k), dev(dr.v), dr.caches, dr.nodes, dr.flat_parents(), dr.config())
    with pytest.raises(gpu.ArgumentError):
        s.gemma_tree_step(s.rope_table(_ffi.ROPE_LLAMA, 64, 1e4, max_positions=64), *args, w, w, 1e-6, 1.0, dev(np.zeros_like(dr.q)))
    with pytest.raises(TypeError):
        s.gemma_tree_step(g, *args, w[:32], w, 1e-6, 1.0, dev(np.zeros_like(dr.q)))
    assert [len(c) for c in dr.caches] == before
    # nothing to do
    s.tree_step(None, dev(dr.q), dev(dr.k), dev(dr.v), [], [], dr.flat_parents(), KvAttentionConfig(0, 8, 2, 64, True, 0), dev(dr.q))
    s.tree_step(None, dev(dr.q), dev(dr.k), dev(dr.v), dr.caches, [0, 0], dr.flat_parents(), KvAttentionConfig(0, 8, 2, 64, True, 0), dev(dr.q))
    s.sync()
    assert [len(c) for c in dr.caches] == before
    other = Session(0)
    with pytest.raises(gpu.ArgumentError):
        other.close()
        other.tree_step(None, dev(dr.q), dev(dr.k), dev(dr.v), dr.caches, dr.nodes, dr.flat_parents(), dr.config(), dev(dr.q))


def test_the_same_call_gives_the_same_bits(s):
    rng = np.random.default_rng(21)
    dr = Draft(s, rng, (24, 8, 128), [3000, 70], [26, 50])
    first = dr.run(s).cpu().numpy()
    for _ in range(3):
        for c, p in zip(dr.caches, dr.past):
            c.truncate(p)
        assert np.array_equal(dr.run(s).cpu().numpy(), first)
    s.sync()


def test_captured_steps_in_turn_with_eager_ones(gpu):
    """Two graphs of one session, replayed with new inputs and eager calls between."""
    import torch

    from spissa_amd.device import Session

    stream = torch.cuda.Stream()
    ses = Session(0, stream=stream)
    rng = np.random.default_rng(8)
    with torch.cuda.stream(stream):
        sets = []
        for heads, past, nodes, window in [((24, 8, 128), [2000], [26], 0), ((8, 4, 256), [700, 90], [5, 64], 64)]:
            dr = Draft(ses, rng, heads, past, nodes)
            q, k, v, out = (torch.zeros(*x.shape, device="cuda") for x in (dr.q, dr.k, dr.v, dr.q))
            args = (None, q, k, v, dr.caches, nodes, dr.flat_parents(), dr.config(window), out)
            ses.tree_step(*args)
            sets.append((dr, args, window))
        ses.sync()
        graphs = []
        for dr, args, window in sets:
            for c, p in zip(dr.caches, dr.past):
                c.truncate(p)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                ses.tree_step(*args)
            graphs.append(g)
        for turn in range(3):
            for (dr, args, window), g in zip(sets, graphs):
                dr.q, dr.k, dr.v = (rng.normal(size=x.shape).astype(np.float32) for x in (dr.q, dr.k, dr.v))
                for t, x in zip(args[1:4], (dr.q, dr.k, dr.v)):
                    t.copy_(dev(x))
                args[-1].fill_(np.nan)
                g.replay()
                got = args[-1].cpu().numpy()
                assert rows_off(got, dr.plain(window=window)[0]) <= ROW, turn
                for c, p in zip(dr.caches, dr.past):
                    c.truncate(p)
                assert np.array_equal(dr.run(ses, window=window).cpu().numpy(), got)
        ses.sync()


# ---- the walk


@pytest.mark.parametrize("nodes", [[1], [2], [5], [63], [64], [65], [256], [0], [0, 4, 0], [7, 256, 1, 30], [26] * 64, [3] * 65, [12] * 200])
def test_accept(s, nodes):
    import torch

    print(f"[case] accept nodes={nodes[:4]} of {len(nodes)}", flush=True)
    rng = np.random.default_rng(sum(nodes) + len(nodes))
    n, b = sum(nodes), len(nodes)
    parents = [drafts.make_tree(rng, m, 6, 0.05) for m in nodes]
    tokens, sampled = rng.integers(0, 3, n).astype(np.int32), rng.integers(-1, 3, n).astype(np.int32)
    path = torch.full((max(1, n),), -5, dtype=torch.int32, device="cuda")
    count, last = (torch.full((b + 1,), -5, dtype=torch.int32, device="cuda") for _ in range(2))
    s.tree_accept(dev(np.array(sum(parents, []) or [0], np.int32)), dev(np.append(tokens, 0).astype(np.int32)),
                  dev(np.append(sampled, 0).astype(np.int32)), nodes, path, count, last)
    s.sync()
    path, count, last = (x.cpu().numpy() for x in (path, count, last))
    at = 0
    for i, m in enumerate(nodes):
        if m:
            want, token = drafts.accept(parents[i], tokens[at:at + m], sampled[at:at + m])
        else:
            want, token = [], -1
        assert path[at:at + m].tolist() == want + [-1] * (m - len(want)) and count[i] == len(want) and last[i] == token
        at += m
    assert count[b] == last[b] == -5


def test_accept_a_whole_chain_and_a_bad_parent(gpu, s):
    import torch

    n = 256
    parents = np.arange(-1, n - 1).astype(np.int32)
    tokens = np.arange(n).astype(np.int32)
    path, count, last = (torch.zeros(m, dtype=torch.int32, device="cuda") for m in (n, 1, 1))
    s.tree_accept(dev(parents), dev(tokens), dev(tokens + 1), [n], path, count, last)
    s.sync()
    assert path.tolist() == list(range(n)) and count.item() == n and last.item() == n
    parents[100] = 100
    s.tree_accept(dev(parents), dev(tokens), dev((tokens + 1).astype(np.int32)), [n], path, count, last)
    with pytest.raises(gpu.InvalidTensorDataError):
        s.sync()
    assert count.item() == 100 and path.tolist() == list(range(100)) + [-1] * 156


# ---- the rows


def random_paths(rng, nodes):
    path, count = [], []
    for n in nodes:
        m = int(rng.integers(0, n + 1))
        path += sorted(rng.choice(n, m, replace=False).tolist()) + [-1] * (n - m)
        count.append(m)
    return np.array(path or [0], np.int32), np.array(count, np.int32)


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("heads,dim", [(8, 128), (1, 256), (3, 64), (5, 64)])
@pytest.mark.parametrize("layers,nodes", [(1, [9]), (3, [26]), (28, [5]), (2, [4, 0, 256, 64]), (5, [7] * 11)])
def test_keep(s, q4, heads, dim, layers, nodes):
    print(f"[case] keep q4={q4} heads={heads} dim={dim} layers={layers} nodes={nodes[:4]}", flush=True)
    rng = np.random.default_rng(layers * 100 + sum(nodes))
    path, count = random_paths(rng, nodes)
    caches, before, past = [], [], []
    for i in range(layers):
        for n in nodes:
            p = int(rng.integers(0, 40))
            c = (s.q4_kv_cache if q4 else s.kv_cache)(heads, dim, p + n + 3)
            x, y = (rng.normal(size=(p + n, heads, dim)).astype(np.float32) for _ in range(2))
            if p + n:
                s.append(c, dev(x), dev(y), p + n)
            caches.append(c), past.append(p), before.append(held(s, c, 0, p + n) if p + n else None)
    s.keep_rows(caches, nodes, dev(path), dev(count))
    s.sync()
    for i, (c, p, rows) in enumerate(zip(caches, past, before)):
        b = i % len(nodes)
        n, first = nodes[b], sum(nodes[:b])
        assert len(c) == p + n
        if not n:
            continue
        for got, was in zip(held(s, c, 0, p + n), rows):
            want = was.copy()
            want[p:p + count[b]] = was[p + path[first:first + count[b]]]
            assert np.array_equal(got, want)


@pytest.mark.parametrize("heads,dim", [(1, 5), (3, 20), (7, 80), (2, 1), (1, 6)])
def test_keep_rows_of_other_widths(s, heads, dim):
    rng = np.random.default_rng(dim)
    c = s.kv_cache(heads, dim, 40)
    x, y = (rng.normal(size=(30, heads, dim)).astype(np.float32) for _ in range(2))
    s.append(c, dev(x), dev(y), 30)
    s.keep_rows([c], [20], dev(np.array([1, 2, 5, 19] + [-1] * 16, np.int32)), dev(np.array([4], np.int32)))
    s.sync()
    for got, was in zip(held(s, c, 0, 30), (x, y)):
        want = was.copy()
        want[10:14] = was[[11, 12, 15, 29]]
        assert np.array_equal(got, want)


@pytest.mark.parametrize("path,count,kept", [([0, 2, 2, 5], 4, 2), ([0, 3, 1, 5], 4, 2), ([0, 6, 7, 9], 4, 1), ([-1, 1, 2, 3], 3, 0),
                                             ([0, 2, 3, 4], 9, 4), ([1, 2, 3, 4], -3, 0)])
def test_keep_ends_at_a_wrong_path(gpu, s, path, count, kept):
    rng = np.random.default_rng(0)
    c, other = (s.kv_cache(2, 64, 40) for _ in range(2))
    x, y = (rng.normal(size=(20, 2, 64)).astype(np.float32) for _ in range(2))
    for cc in (c, other):
        s.append(cc, dev(x), dev(y), 20)
    full = path + [5, 5] if count == 9 else path + [-1, -1]
    s.keep_rows([c, other], [6, 2], dev(np.array(full + [1, -1], np.int32)), dev(np.array([count, 1], np.int32)))
    with pytest.raises(gpu.InvalidTensorDataError):
        s.sync()
    s.sync()
    want = x.copy()
    at = full[:kept + (1 if count == 9 else 0)]
    want[14:14 + len(at)] = x[[14 + p for p in at]]
    assert np.array_equal(held(s, c, 0, 20)[0], want)
    want = x.copy()
    want[18] = x[19]
    assert np.array_equal(held(s, other, 0, 20)[0], want)


def test_keep_refusals(gpu, s):
    c, d = s.kv_cache(2, 64, 16), s.kv_cache(2, 64, 16)
    x = dev(np.zeros((8, 2, 64), np.float32))
    for cc in (c, d):
        s.append(cc, x, x, 8)
    path, count = dev(np.zeros(16, np.int32)), dev(np.zeros(2, np.int32))
    with pytest.raises(gpu.ShapeError):
        s.keep_rows([c], [9], path, count)
    with pytest.raises(gpu.ArgumentError):
        s.keep_rows([c, c], [2], path, count)
    with pytest.raises(TypeError):
        s.keep_rows([c, d, c], [2, 2], path, count)
    with pytest.raises(TypeError):
        s.keep_rows([c, d], [9, 9], path, count)
    with pytest.raises(TypeError):
        s.keep_rows([c], [], path, count)
    s.keep_rows([], [], path, count)
    s.keep_rows([c, d], [0, 0], path, count)
    s.sync()


@pytest.mark.parametrize("heads", [(8, 2, 64), (24, 8, 128), (4, 1, 256)])
def test_the_prefill_operands_follow(s, heads):
    """A prompt through the bf16 prefill, a draft, its kept rows, another chunk: as with rows appended one after the other."""
    from spissa_amd.rotary import KvAttentionConfig

    rng = np.random.default_rng(1)
    dr = Draft(s, rng, heads, [0], [21], room=400)
    hq, hkv, d = heads
    f = lambda n, h: dev(rng.normal(size=(n, h, d)).astype(np.float32))  # noqa: E731
    table, *_ = tables(s, _ffi.ROPE_LLAMA, d, 400)
    c, plain = dr.caches[0], dr.cache(s, 0, 400)
    q, k, v = f(90, hq), f(90, hkv), f(90, hkv)
    for cc in (c, plain):
        s.prefill_step(table, q, k, v, cc, KvAttentionConfig(90, hq, hkv, d, True, 0), dev(np.zeros((90, hq, d), np.float32)))
    dr.run(s, table)
    rows = held(s, c, 90, 21)
    path = [0, 1, 4, 7, 8, 15, 20]
    s.keep_rows([c], [21], dev(np.array(path + [-1] * 14, np.int32)), dev(np.array([7], np.int32)))
    c.truncate(97)
    s.append(plain, dev(rows[0][path]), dev(rows[1][path]), 7)
    q, k, v = f(33, hq), f(33, hkv), f(33, hkv)
    outs = []
    for cc in (c, plain):
        out = dev(np.zeros((33, hq, d), np.float32))
        s.prefill_step(table, q, k, v, cc, KvAttentionConfig(33, hq, hkv, d, True, 0), out)
        outs.append(out.cpu().numpy())
    s.sync()
    assert np.array_equal(outs[0], outs[1])


# ---- all of them together


@pytest.mark.parametrize("settings", ["greedy", "sampled"])
def test_drafted_decoding_writes_what_decoding_writes(s, settings):
    """A model of two layers and a small vocabulary, decoded a token a step and by drafted
    trees: the same tokens, and the same rows in its caches. Each step's tree holds the true
    next tokens among wrong ones, or wrong ones alone. The random number of a position is
    the same on both ways."""
    import torch

    from spissa_amd.device import SamplingConfig
    from spissa_amd.rotary import KvAttentionConfig

    hq, hkv, d, vocab, layers, prompt, steps = 8, 2, 64, 211, 2, 19, 24
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    r = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    embed, head = r(vocab, hq * d), r(vocab, hq * d) * 0.2
    wq, wk, wv = ([r(hq * d, n * d) / 22 for _ in range(layers)] for n in (hq, hkv, hkv))
    table, *_ = tables(s, _ffi.ROPE_LLAMA, d, 128)
    weight = s.linear_weight(head.cpu().numpy(), _ffi.DTYPE_F32, vocab, hq * d)
    uniform = torch.rand(256, generator=gen, device="cuda")
    cfg = SamplingConfig(0.0) if settings == "greedy" else SamplingConfig(0.9, 40, 0.95, 0.01)
    mm = lambda x, w: (x.double() @ w.double()).float().contiguous()  # noqa: E731  (the same bits for one row as for many)
    prompt_tokens = torch.randint(0, vocab, (prompt,), generator=gen, device="cuda")

    def layer_pass(tokens, caches, attend):
        x = embed[tokens]
        for i in range(layers):
            out = torch.zeros(len(tokens), hq, d, device="cuda")
            attend(i, *(mm(x, w[i]).view(len(tokens), -1, d) for w in (wq, wk, wv)), caches[i], out)
            x = x + out.view(len(tokens), -1).double().mul(64).round().div(64).float()  # (both ways' roundings fall together)
        logits = torch.zeros(len(tokens), vocab, device="cuda")
        s.linear(weight, x.contiguous(), None, len(tokens), logits)
        return logits.mul(256).round().div(256)

    def decode(i, q, k, v, c, out):
        s.decode_step(table, q, k, v, [c], KvAttentionConfig(1, hq, hkv, d, True, 0), out)

    def sampled(logits, positions):
        t = torch.zeros(len(positions), dtype=torch.int32, device="cuda")
        s.sample(logits.contiguous(), uniform[positions].contiguous(), cfg, t)
        return t

    plain = [s.kv_cache(hkv, d, 128) for _ in range(layers)]
    tokens = prompt_tokens.tolist()
    for p in range(prompt + steps):
        got = sampled(layer_pass(torch.tensor([tokens[p]], device="cuda"), plain, decode), torch.tensor([p], device="cuda"))
        if p >= prompt - 1:
            tokens.append(int(got))

    rng = np.random.default_rng(5)
    caches = [s.kv_cache(hkv, d, 160) for _ in range(layers)]
    for p in range(prompt - 1):
        layer_pass(torch.tensor([tokens[p]], device="cuda"), caches, decode)
    mine, accepted = tokens[:prompt], []
    while len(mine) < len(tokens) - 8:
        p = len(mine) - 1  # the last known token, not in the caches yet
        parents, draft = [-1], [mine[p]]
        spine = 0
        for e in range(int(rng.integers(0, 5))):  # a level: wrong children, the true one among them
            level = spine
            right = int(rng.integers(0, 3))
            for j in range(3):
                parents.append(level)
                draft.append(tokens[p + 1 + e] if j == right else (tokens[p + 1 + e] + 1 + j) % vocab)
                if j == right:
                    spine = len(parents) - 1
        n = len(parents)
        par, tok = dev(np.array(parents, np.int32)), dev(np.array(draft, np.int32))
        pos = p + torch.tensor(drafts.depths(parents), device="cuda")

        def tree(i, q, k, v, c, out):
            s.tree_step(table, q, k, v, [c], [n], par, KvAttentionConfig(n, hq, hkv, d, True, 0), out)

        got = sampled(layer_pass(tok.long(), caches, tree), pos)
        path, count, last = (torch.zeros(m, dtype=torch.int32, device="cuda") for m in (n, 1, 1))
        s.tree_accept(par, tok, got, [n], path, count, last)
        s.keep_rows(caches, [n], path, count)
        s.sync()
        m = int(count)
        for c in caches:
            c.truncate(p + m)
        mine += [draft[t] for t in path.tolist()[1:m]] + [int(last)]
        accepted.append(m)
    assert mine == tokens[:len(mine)] and max(accepted) > 2
    for a, b in zip(caches, plain):
        n = len(a)
        assert n == len(mine) - 1
        for x, y in zip(held(s, a, 0, n), held(s, b, 0, n)):
            assert np.abs(x - y).max() <= 1e-3


@pytest.mark.parametrize("heads", [(24, 8, 128), (8, 2, 64), (4, 1, 256)])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_a_query_that_is_not_finite_is_its_rows_alone(gpu, s, heads, what):
    print(f"[case] {what} in a query {heads}", flush=True)
    rng = np.random.default_rng(12)
    dr = Draft(s, rng, heads, [333], [13])
    dr.q[6, 1, 3] = what
    out = dr.run(s).cpu().numpy()
    with pytest.raises(gpu.InvalidTensorDataError):
        s.sync()
    s.sync()
    assert not np.isfinite(out[6, 1]).any()
    dr.q[6, 1] = 0
    others = np.ones(out.shape[:2], bool)
    others[6, 1] = False
    want, _ = dr.plain()
    assert rows_off(out[others], want[others]) <= ROW


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e4])
def test_queries_of_any_size(s, scale):
    """Small ones weigh all keys alike; large ones take one key, their scores' error 2^-22 of some 1e5: a weight that is
    another's neighbour within 2^-22 * 1e5 = 0.03 could be off by that much, which N(0, 1) keys of 64 channels are not (the
    two largest of 260 scores lie some 1e4 * 8 * 0.3 apart), so the row is the key's value to the pieces' 2^-23."""
    rng = np.random.default_rng(13)
    dr = Draft(s, rng, (4, 2, 64), [250], [10])
    dr.q *= np.float32(scale)
    out = dr.run(s).cpu().numpy()
    s.sync()
    assert rows_off(out, dr.plain()[0]) <= ROW


def test_two_sessions_at_once(gpu):
    """Two sessions of two threads and streams, each with caches and a workspace of its own: the same outputs as alone."""
    import threading

    import torch

    from spissa_amd.device import Session

    got, failed = [[], []], []

    def work(i, rounds):
        try:
            stream = torch.cuda.Stream()
            ses = Session(0, stream=stream)
            with torch.cuda.stream(stream):
                dr = Draft(ses, np.random.default_rng(20 + i), [(24, 8, 128), (8, 4, 256)][i], [[900], [40, 700]][i], [[12], [30, 3]][i])
                for _ in range(rounds):
                    got[i].append(dr.run(ses))
                    for c, p in zip(dr.caches, dr.past):
                        c.truncate(p)
                ses.sync()
        except Exception as e:  # (shown by the main thread)
            failed.append(e)

    want = []
    for i in range(2):
        work(i, 1)
        want.append(got[i].pop())
    threads = [threading.Thread(target=work, args=(i, 25)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_a_closed_cache_is_refused(gpu, s):
    dr = Draft(s, np.random.default_rng(0), (4, 2, 64), [5, 6, 7], [2, 1, 3])
    dr.caches[1].close()
    with pytest.raises(gpu.ArgumentError):
        dr.run(s)
    assert [len(dr.caches[0]), len(dr.caches[2])] == [5, 7]


def test_a_whole_drafted_step_in_a_graph(gpu):
    """Two layers' tree steps, sampling, the walk and the move captured as one graph: replayed with new inputs, with
    eager calls of the same session between the replays, each replay equal to the same calls made eagerly."""
    import torch

    from spissa_amd.device import SamplingConfig, Session

    rng = np.random.default_rng(31)
    stream = torch.cuda.Stream()
    ses = Session(0, stream=stream)
    past, nodes, vocab, heads = [40, 333], [7, 12], 9001, (8, 2, 64)
    n = sum(nodes)
    with torch.cuda.stream(stream):
        layers = [Draft(ses, rng, heads, past, nodes) for _ in range(2)]
        twins = [[d.cache(ses, b) for b in range(2)] for d in layers]
        ins = [{k: dev(getattr(d, k)) for k in "qkv"} for d in layers]
        parents, drafted = layers[0].flat_parents(), torch.zeros(n, dtype=torch.int32, device="cuda")
        logits, u = torch.zeros(n, vocab, device="cuda"), torch.zeros(n, device="cuda")
        cfg = SamplingConfig(0.8, 3, 0.9, 0.0)

        def step(caches):
            """(outputs, sampled, path, count, next): new tensors."""
            outs = [torch.zeros(n, 8, 64, device="cuda") for _ in layers]
            ints = [torch.zeros(m, dtype=torch.int32, device="cuda") for m in (n, n, 2, 2)]
            for i in range(2):
                ses.tree_step(None, ins[i]["q"], ins[i]["k"], ins[i]["v"], caches[i], nodes, parents, layers[i].config(), outs[i])
            ses.sample(logits, u, cfg, ints[0])
            ses.tree_accept(parents, drafted, ints[0], nodes, *ints[1:])
            ses.keep_rows([c for cs in caches for c in cs], nodes, ints[1], ints[2])
            return outs + ints

        def back(caches):
            for cs in caches:
                for c, p in zip(cs, past):
                    c.truncate(p)

        mine = [d.caches for d in layers]
        step(mine)
        back(mine)
        ses.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step(mine)
        walked = set()
        for _ in range(4):
            for i in ins:
                for x in i.values():
                    x.copy_(torch.as_tensor(rng.normal(size=tuple(x.shape)).astype(np.float32)))
            logits.copy_(torch.as_tensor(rng.normal(size=(n, vocab)).astype(np.float32)))
            u.copy_(torch.as_tensor(rng.random(n).astype(np.float32)))
            # drafts that sampling often confirms: the largest logit after the parent
            best = logits.argmax(1).int()
            drafted.copy_(torch.where(parents >= 0, best[torch.cat([parents[:7].clamp(min=0), parents[7:].clamp(min=0) + 7]).long()], best))
            graph.replay()
            want = step(twins)
            ses.sync()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            walked |= set(got[4].tolist())
            for i in range(2):
                for b in range(2):
                    for x, y in zip(held(ses, mine[i][b], past[b], nodes[b]), held(ses, twins[i][b], past[b], nodes[b])):
                        assert np.array_equal(x, y)
            back(twins)
        assert max(walked) > 1  # (some walks go on)


@pytest.mark.parametrize("heads", [(24, 8, 128), (8, 2, 64), (4, 1, 256)])
@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("past,window", [([0, 0], 0), ([150, 40], 0), ([0, 0], 3), ([150, 40], 60)])
@pytest.mark.parametrize("size", [0.01, 0.25, 0.0])
def test_what_is_not_finite_beside_values_below_one(gpu, s, heads, where, past, window, size):
    """As models' values are: the scale that the rest of a first tile takes is far above the one that a number
    which is not finite leads to. (size 0: all other values nothing; then the outputs are nothing.)"""
    print(f"[case] NaN in a drafted {where} {heads} past={past} window={window} size={size}", flush=True)
    rng = np.random.default_rng(17)
    dr = Draft(s, rng, heads, past, [40, 7], vscale=size)
    bad = 11
    (dr.k if where == "key" else dr.v)[bad, heads[1] - 1, 5] = np.nan
    out = dr.run(s, window=window).cpu().numpy()
    with pytest.raises(gpu.InvalidTensorDataError):
        s.sync()
    s.sync()
    dr.k[bad] = dr.v[bad] = 0
    want, _ = dr.plain(window=window)
    sees = np.zeros(47, bool)
    sees[:40] = drafts.seen(dr.parents[0], 0, window)[:, bad]
    assert sees.any() and not sees.all()
    if size:
        assert rows_off(out[~sees], want[~sees]) <= ROW
    else:
        assert (out[~sees] == 0).all()
    assert np.isnan(out[sees][:, -(heads[0] // heads[1]):]).all()


@pytest.mark.parametrize("heads", [(24, 8, 128), (8, 2, 64), (4, 1, 256)])
@pytest.mark.parametrize("what", [np.nan, np.inf])
def test_a_cached_value_that_is_not_finite_and_that_deeper_nodes_do_not_see(gpu, s, heads, what):
    rng = np.random.default_rng(18)
    dr = Draft(s, rng, heads, [400], [30], vscale=0.01)
    depth = np.array(drafts.depths(dr.parents[0]))
    at = 400 + 4 + 1 - 100 - 1  # with a window of 100 seen by depths 0..3
    dr.pv[0][at, 0, 3] = what
    dr.caches = [dr.cache(s, 0)]
    out = dr.run(s, window=100).cpu().numpy()
    with pytest.raises(gpu.InvalidTensorDataError):
        s.sync()
    dr.pv[0][at] = 0
    want, _ = dr.plain(window=100)
    sees, group = depth <= 3, heads[0] // heads[1]
    assert (~sees).any() and rows_off(out[~sees], want[~sees]) <= ROW and np.isnan(out[sees][:, :group]).all()
    if heads[1] > 1:  # (the other KV heads' rows do not see it either)
        assert np.isfinite(out[:, group:]).all()


@pytest.mark.parametrize("heads", [(24, 8, 128), (8, 2, 64), (4, 1, 256)])
@pytest.mark.parametrize("past", [250, 3000])
@pytest.mark.parametrize("scale", [1e6, 1e7, 1e8, 1e9, 1e10, 1e12, 1e30])
def test_scores_of_any_size(s, heads, past, scale):
    """Scores of 2^20 and more, between whose numbers in f32 lie 8, 16 and more: every row is the value of its largest
    score, to the pieces' 2^-23, as the two largest of a row lie far more than 2^-20 of themselves apart."""
    print(f"[case] queries of {scale} {heads} past={past}", flush=True)
    rng = np.random.default_rng(28)
    dr = Draft(s, rng, heads, [past], [10])
    dr.q *= np.float32(scale)
    out = dr.run(s).cpu().numpy()
    s.sync()
    assert rows_off(out, dr.plain()[0]) <= ROW


def with_rows(s, dr):
    """The draft's caches from its rows as they are now."""
    dr.caches = [dr.cache(s, i) for i in range(len(dr.past))]
    return dr


def by_scores(dr, window=0):
    """What the scores' own errors may do to each output row, over the row's 2-norm. A score is a sum of D products
    of pieces (off by 5 * 2^-24 of each) by 3 D / 32 instructions, off by half a step of their sum at most: for
    huge keys far more than for the others. An output follows an error e_j of score j by p_j e_j (v_j - out);
    twice that for errors up to 1."""
    offs, at = [], 0
    for p, parents, pk, pv in zip(dr.past, dr.parents, dr.pk, dr.pv):
        n, r = len(parents), dr.hq // dr.hkv
        k, v = (np.concatenate([a, b[at:at + n]]).astype(np.float64).repeat(r, 1) for a, b in ((pk, dr.k), (pv, dr.v)))
        for t, seen in enumerate(drafts.seen(parents, p, window)):
            q, kk, vv = dr.q[at + t].astype(np.float64), k[seen], v[seen]
            sc = np.einsum("hd,mhd->mh", q, kk) / np.sqrt(dr.d)
            w = np.exp(sc - sc.max(0))
            w /= w.sum(0)
            e = np.einsum("hd,mhd->mh", np.abs(q), np.abs(kk)) / np.sqrt(dr.d) * (5 + 3 * dr.d / 32) * 2.0 ** -24
            out = np.einsum("mh,mhd->hd", w, vv)
            offs.append(2 * np.einsum("mh,mh->h", w * e, np.linalg.norm(vv - out, axis=-1)) / np.linalg.norm(out, axis=-1))
        at += n
    return np.stack(offs)


def each_off(got, want):
    return np.linalg.norm(got.astype(np.float64) - want, axis=-1) / np.linalg.norm(want, axis=-1)


OUTLIERS = [(24, 8, 128), (8, 2, 64), (4, 1, 256)]


@pytest.mark.parametrize("heads", OUTLIERS)
@pytest.mark.parametrize("where", ["key", "value", "both"])
@pytest.mark.parametrize("size", [1e5, 1e8, 1e30])
@pytest.mark.parametrize("past", [[0, 0], [150, 40]])
def test_a_drafted_row_of_any_size_leaves_the_others(s, heads, where, size, past):
    """Rows that do not see it are off by no more than without it; those that see it by what its score is off besides."""
    print(f"[case] {where} of {size} {heads} past={past}", flush=True)
    rng = np.random.default_rng(19)
    dr = Draft(s, rng, heads, past, [40, 7])
    for x, name in ((dr.k, "key"), (dr.v, "value")):
        if where in (name, "both"):
            x[11] *= np.float32(size)
    out = dr.run(s).cpu().numpy()
    s.sync()
    want, _ = dr.plain()
    sees = np.zeros(47, bool)
    sees[:40] = drafts.seen(dr.parents[0], 0)[:, 11]
    assert sees.any() and not sees.all()
    assert rows_off(out[~sees], want[~sees]) <= ROW
    assert (each_off(out, want) <= ROW + by_scores(dr))[sees].all()


@pytest.mark.parametrize("heads", OUTLIERS)
@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("size", [1e8, 1e30])
def test_a_cached_row_of_any_size_leaves_nodes_that_do_not_see_it(s, heads, where, size):
    rng = np.random.default_rng(20)
    dr = Draft(s, rng, heads, [400], [30])
    at = 400 + 4 + 1 - 100 - 1  # with a window of 100 seen by depths 0..3
    (dr.pk if where == "key" else dr.pv)[0][at] *= np.float32(size)
    out = with_rows(s, dr).run(s, window=100).cpu().numpy()
    s.sync()
    want, _ = dr.plain(window=100)
    deep = np.array(drafts.depths(dr.parents[0])) > 3
    assert deep.any() and not deep.all()
    assert rows_off(out[deep], want[deep]) <= ROW
    assert (each_off(out, want) <= ROW + by_scores(dr, 100))[~deep].all()


@pytest.mark.parametrize("heads", [(24, 8, 128), (16, 8, 64), (8, 4, 256)])
@pytest.mark.parametrize("past", [600, 9000])
@pytest.mark.parametrize("size", [1e5, 1e10, 1e30])
def test_huge_values_of_no_weight(s, heads, past, size):
    """Seen, but with scores some 100 below the others': in a first tile with more of them behind it in the same
    workgroup, and in the middle."""
    print(f"[case] values of {size} without weight {heads} past={past}", flush=True)
    rng = np.random.default_rng(21)
    dr = Draft(s, rng, heads, [past], [5])
    dr.q = np.abs(dr.q)
    for at in (0, 300):
        dr.pk[0][at] = -20 * np.abs(dr.pk[0][at])
        dr.pv[0][at] *= np.float32(size)
    out = with_rows(s, dr).run(s).cpu().numpy()
    s.sync()
    assert rows_off(out, dr.plain()[0]) <= ROW


@pytest.mark.parametrize("heads", OUTLIERS)
@pytest.mark.parametrize("size", [1e5, 1e30])
def test_huge_keys_of_no_weight(s, heads, size):
    rng = np.random.default_rng(22)
    dr = Draft(s, rng, heads, [5000], [21])
    dr.q = np.abs(dr.q)
    for at in (0, 333, 4999):
        dr.pk[0][at] = -np.abs(dr.pk[0][at]) * np.float32(size)
    out = with_rows(s, dr).run(s).cpu().numpy()
    s.sync()
    assert rows_off(out, dr.plain()[0]) <= ROW


@pytest.mark.parametrize("heads", OUTLIERS)
@pytest.mark.parametrize("at", [0, 250, 699])
def test_a_huge_value_of_small_weight(s, heads, at):
    """A weight of e^-28 of the others' and a value of 1e14: shares of the same size."""
    rng = np.random.default_rng(23)
    dr = Draft(s, rng, heads, [700], [9])
    u = rng.normal(size=heads[2])
    dr.q[:] = u
    dr.pk[0][at] = u * (-28 * np.sqrt(heads[2]) / (u @ u))
    dr.pv[0][at] *= np.float32(1e14)
    out = with_rows(s, dr).run(s).cpu().numpy()
    s.sync()
    # (its score is the sum of 3 D / 32 matrix instructions, each off by half a step of 28 at most, and its weight by that share)
    assert rows_off(out, dr.plain()[0]) <= ROW + 3 * heads[2] / 32 * 28 * 2.0 ** -24


@pytest.mark.parametrize("heads", OUTLIERS)
@pytest.mark.parametrize("past,nodes", [([0], [100]), ([1000], [30]), ([3000, 77], [40, 9])])
@pytest.mark.parametrize("where", ["values", "small keys", "both"])
def test_rows_of_all_sizes_in_a_tile(s, heads, past, nodes, where):
    """Sizes from 2^-40 to 2^40 (keys: to 2^2) without order, a tile's rows held in many parts."""
    print(f"[case] sizes without order: {where} {heads} past={past} nodes={nodes}", flush=True)
    rng = np.random.default_rng(24)
    dr = Draft(s, rng, heads, past, nodes)
    for keys, rows in ((True, dr.pk + [dr.k]), (False, dr.pv + [dr.v])):
        for x in rows:
            if where in ("both", "small keys" if keys else "values"):
                x *= np.float32(2) ** rng.integers(-40, 3 if keys else 41, (len(x), 1, 1)).astype(np.float32)
    out = with_rows(s, dr).run(s).cpu().numpy()
    s.sync()
    assert rows_off(out, dr.plain()[0]) <= ROW


@pytest.mark.parametrize("heads", OUTLIERS)
def test_a_huge_row_beside_one_that_is_not_finite(gpu, s, heads):
    rng = np.random.default_rng(25)
    dr = Draft(s, rng, heads, [90], [40], vscale=0.01)
    dr.v[11] *= np.float32(1e30)
    dr.k[17] *= np.float32(-1e12)
    dr.v[23, 0, 1], dr.k[31, 0, 2] = np.nan, -np.inf
    out = dr.run(s).cpu().numpy()
    with pytest.raises(gpu.InvalidTensorDataError):
        s.sync()
    s.sync()
    seen = drafts.seen(dr.parents[0], 0)
    poisoned = seen[:, 23] | seen[:, 31]
    dr.v[23] = dr.k[31] = 0
    want, _ = dr.plain()
    assert poisoned.any() and rows_off(out[~poisoned], want[~poisoned]) <= ROW
    assert np.isnan(out[poisoned][:, :heads[0] // heads[1]]).all()


@pytest.mark.parametrize("heads", [(24, 8, 128), (8, 2, 64), (4, 1, 256)])
@pytest.mark.parametrize("past", [0, 333])
@pytest.mark.parametrize("scale,vscale", [(1.0, 1e-33), (1.0, 1e-36), (1e-34, 1e-36), (1e-34, 1.0)])
def test_the_smallest_values(s, heads, past, scale, vscale):
    """Down to outputs of 2^-126, whose last bit is 2^-149: 2^-24 of the larger half of a row of some 1e-37."""
    rng = np.random.default_rng(27)
    dr = Draft(s, rng, heads, [past], [21], scale=scale, vscale=vscale)
    dr.q /= np.float32(scale)
    out = dr.run(s).cpu().numpy()
    s.sync()
    assert rows_off(out, dr.plain()[0]) <= ROW


@pytest.mark.parametrize("heads", [(24, 8, 128), (8, 4, 256), (8, 2, 64)])
@pytest.mark.parametrize("window,size", [(0, 1.0), (64, 1.0), (0, 1e6)])
def test_a_gemma_chain_is_as_many_gemma_decode_steps(s, heads, window, size):
    """With the norm, the prescale and a window; and with a value of 1e6 in the cache."""
    from spissa_amd.rotary import KvAttentionConfig

    rng = np.random.default_rng(29)
    dr = Draft(s, rng, heads, [200], [6])
    dr.pv[0][150] *= np.float32(size)
    dr.parents = [[-1, 0, 1, 2, 3, 4]]
    norm = [dev((1 + 0.25 * rng.normal(size=heads[2])).astype(np.float32)) for _ in range(2)]
    table, *_ = tables(s, _ffi.ROPE_GEMMA, heads[2], 208)
    with_rows(s, dr)
    one = dr.cache(s, 0)
    out = dev(np.zeros_like(dr.q))
    s.gemma_tree_step(table, dev(dr.q), dev(dr.k), dev(dr.v), dr.caches, [6], dr.flat_parents(), dr.config(window), *norm, 1e-6, 0.75, out)
    out = out.cpu().numpy()
    cfg = KvAttentionConfig(1, *heads, True, window)
    for t in range(6):
        o = dev(np.zeros_like(dr.q[:1]))
        s.gemma_decode_step(table, dev(dr.q[t:t + 1]), dev(dr.k[t:t + 1]), dev(dr.v[t:t + 1]), [one], cfg, *norm, 1e-6, 0.75, o)
        # each side's own error, and 16 * 2^-24 of the rows of keys, whose norms are summed in different orders
        assert rows_off(out[t:t + 1], o.cpu().numpy().astype(np.float64)) <= 2 * ROW + 16 * 2.0 ** -24 * np.sqrt(heads[2])
    a, b = held(s, dr.caches[0], 0, 206), held(s, one, 0, 206)
    assert rows_off(a[0], b[0].astype(np.float64)) <= 2 * 16 * 2.0 ** -24 and np.array_equal(a[1], b[1])
    s.sync()


@pytest.mark.parametrize("heads", OUTLIERS)
def test_a_captured_step_replayed_with_huge_rows_and_such_as_are_not_finite(gpu, heads):
    """Captured with ordinary rows; which tiles take turns of their own is found on the device in each replay."""
    import torch

    from spissa_amd.device import Session

    rng = np.random.default_rng(30)
    stream = torch.cuda.Stream()
    ses = Session(0, stream=stream)
    with torch.cuda.stream(stream):
        dr = Draft(ses, rng, heads, [500, 70], [20, 9])
        q, k, v, out = (torch.zeros(*x.shape, device="cuda") for x in (dr.q, dr.k, dr.v, dr.q))
        args = (None, q, k, v, dr.caches, dr.nodes, dr.flat_parents(), dr.config(), out)
        ses.tree_step(*args)
        for c, p in zip(dr.caches, dr.past):
            c.truncate(p)
        ses.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ses.tree_step(*args)
        sees = np.zeros(29, bool)
        sees[:20] = drafts.seen(dr.parents[0], 0)[:, 7]
        for size in (1.0, 1e8, np.nan, 1e-30, 1e30, 1.0):
            dr.q, dr.k, dr.v = (rng.normal(size=x.shape).astype(np.float32) for x in (dr.q, dr.k, dr.v))
            dr.v[7] *= np.float32(size)
            for t, x in zip((q, k, v), (dr.q, dr.k, dr.v)):
                t.copy_(dev(x))
            out.fill_(np.nan)
            graph.replay()
            got = out.cpu().numpy()
            if np.isnan(size):
                with pytest.raises(gpu.InvalidTensorDataError):
                    ses.sync()
                dr.v[7] = 0
                assert np.isnan(got[sees]).all()
            else:
                ses.sync()
            want, _ = dr.plain()
            at = ~sees if np.isnan(size) else np.ones(29, bool)
            assert rows_off(got[at], want[at]) <= ROW, size
            # and the call made eagerly has the same bits
            for c, p in zip(dr.caches, dr.past):
                c.truncate(p)
            ses.tree_step(None, q, k, v, dr.caches, dr.nodes, dr.flat_parents(), dr.config(), out)
            assert np.array_equal(out.cpu().numpy(), got, equal_nan=True)
            if np.isnan(size):
                with pytest.raises(gpu.InvalidTensorDataError):
                    ses.sync()
        ses.sync()
