"""The operators of a tree step on the GPU against plain 64-bit forms
(tree_reference.py): attention of drafted trees over paged histories,
verification of the drafts, append of the accepted path, and the three together
as a server runs them (DecodeBatch.prepare_tree .. accept_tree).

Attention is held to the tolerance of every attention entry point of the
library: max-abs 2e-5 plus rel 1e-4, on the values the pages hold.  Accepted
paths and tokens are equal, and appended rows equal bit by bit."""

import numpy as np
import pytest
import torch

import helix_runtime_amd as hx
import oracle
import tree_reference as ref

pytestmark = pytest.mark.gpu

ATOL, RTOL = 2e-5, 1e-4
D, P = 128, 16
KS, VS = 0.037, 0.011
DTYPES = ["f32", "bf16", "fp8"]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")


def host(t):
    return t.detach().cpu().numpy()


def on_pages(dtype, x, scale):
    if dtype == "bf16":
        return oracle.round_bf16(x)
    if dtype == "fp8":
        return oracle.round_fp8(x, scale)
    return x


def to_pool(dtype, x, scale):
    """A pool tensor of fp32 values."""
    t = dev(x)
    if dtype == "bf16":
        return t.to(torch.bfloat16)
    if dtype == "fp8":
        by = torch.full((), scale, device="cuda:0")
        return (t / by).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return t


class Problem:
    """Scattered pages, histories and trees of one attention call."""

    def __init__(self, dtype, hists, hq, hkv, nodes, seed, parents=None, counts=None):
        rng = self.rng = np.random.default_rng(seed)
        self.dtype, self.hists, self.hq, self.hkv, self.T = dtype, list(hists), hq, hkv, nodes
        B = self.B = len(hists)
        self.pages = [(h + P - 1) // P for h in hists]
        self.N = sum(self.pages) + 3
        normal = lambda *s: rng.standard_normal(s, dtype=np.float32)  # noqa: E731
        self.kp, self.vp = normal(self.N, hkv, P, D), normal(self.N, hkv, P, D)
        order = rng.permutation(self.N)
        self.tables = np.zeros((B, max(1, max(self.pages)) + 1), np.int32)
        at = 0
        for b, n in enumerate(self.pages):
            self.tables[b, :n] = order[at:at + n]
            at += n
        self.q = normal(B, hq, nodes, D)
        self.tk, self.tv = normal(B, hkv, nodes, D), normal(B, hkv, nodes, D)
        self.parents = ref.random_trees(rng, B, nodes) if parents is None else parents
        self.counts = counts

    def scales(self):
        return dict(k_scale=KS, v_scale=VS) if self.dtype == "fp8" else {}

    def want(self, before=7.0):
        out = np.full((self.B, self.hq, self.T, D), before, np.float64)
        kp, vp = on_pages(self.dtype, self.kp, KS), on_pages(self.dtype, self.vp, VS)
        tk, tv = on_pages(self.dtype, self.tk, KS), on_pages(self.dtype, self.tv, VS)
        for b, n in enumerate(self.hists):
            ids = self.tables[b, :self.pages[b]]
            k = kp[ids].transpose(1, 0, 2, 3).reshape(self.hkv, -1, D)[:, :n]
            v = vp[ids].transpose(1, 0, 2, 3).reshape(self.hkv, -1, D)[:, :n]
            count = self.T if self.counts is None else min(max(int(self.counts[b]), 0), self.T)
            ref.tree_attention(self.q[b], k, v, tk[b], tv[b], self.parents[b], count, out[b])
        return out

    def tensors(self):
        self.d = dict(query=dev(self.q), key_pool=to_pool(self.dtype, self.kp, KS),
                      value_pool=to_pool(self.dtype, self.vp, VS), tables=dev(self.tables),
                      lengths=dev(np.array(self.hists, np.int32)), tree_key=dev(self.tk),
                      tree_value=dev(self.tv), parents=dev(self.parents),
                      output=torch.full((self.B, self.hq, self.T, D), 7.0, device="cuda:0"),
                      workspace=hx.tree_workspace(self.B, self.hq, self.hkv, self.T),
                      node_counts=None if self.counts is None else dev(
                          np.asarray(self.counts, np.int32)),
                      page_dtype=self.dtype, **self.scales())
        return self.d

    def run(self):
        d = self.tensors()
        # What an earlier call left in a workspace is not read.
        d["workspace"].fill_(255)
        hx.paged_tree_attention(**d)
        torch.cuda.synchronize()
        return host(d["output"])


def close(got, want):
    np.testing.assert_allclose(got, want, atol=ATOL, rtol=RTOL)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,nodes", [
    (4, 4, 1), (8, 8, 5), (8, 4, 16), (6, 2, 7), (8, 2, 4), (8, 2, 17), (10, 2, 13), (16, 2, 16),
    (32, 2, 3), (8, 2, 33), (8, 2, 64), (16, 2, 64), (24, 2, 43), (5, 1, 31)])
def test_attention_over_groups_and_tree_sizes(device, dtype, hq, hkv, nodes):
    p = Problem(dtype, [0, 1, 15, 16, 33, 200, 517], hq, hkv, nodes, hq * 100 + nodes)
    close(p.run(), p.want())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hists", [[0], [1], [31], [32], [1000], [5000], [0, 0, 0],
                                   [3, 0, 2047, 0, 64, 65], list(range(0, 90))])
def test_attention_over_histories(device, dtype, hists):
    p = Problem(dtype, hists, 8, 2, 6, 1000 + sum(hists))
    close(p.run(), p.want())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nodes", [9, 40, 64])
def test_rows_behind_a_sequences_nodes_stay(device, dtype, nodes):
    """Ragged trees (none, one and more nodes than there are rows among them),
    forests, chains given as None."""
    counts = [nodes, 0, 1, nodes // 2, nodes + 5, -3, 33]
    hists = [40, 300, 0, 17, 5, 100, 600]
    rng = np.random.default_rng(nodes)
    p = Problem(dtype, hists, 8, 2, nodes, 5 + nodes, counts=counts,
                parents=ref.random_trees(rng, len(hists), nodes, forest=True))
    got = p.run()
    close(got, p.want())
    p.parents = ref.chain(p.B, nodes)
    d = p.tensors()
    d["parents"] = None
    hx.paged_tree_attention(**d)
    close(host(d["output"]), p.want())


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_histories_split_over_the_device(device, dtype):
    """Few rows over a long axis, and a long beside short ones."""
    for hists, hq, hkv, nodes in (([20011], 4, 1, 3), ([9000, 3, 0, 700], 8, 2, 20)):
        p = Problem(dtype, hists, hq, hkv, nodes, 77)
        close(p.run(), p.want())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,nodes", [(2, 8), (4, 16), (4, 29), (8, 16), (4, 33), (4, 64)])
def test_results_are_fp32_results(device, dtype, hq, nodes):
    """Every bit of the fp32 factors takes part, in each shape of the kernel (16 to
    256 rows a head).  A score's partial sums lie below 4 (in powers of two), so
    each of its 12 roundings is off by 2^-22 / sqrt(12) in the mean square, and the
    score by 2^-22: a weight by 2^-22.5 of itself, the row's sums and quotient by
    2^-23 or so each.  A factor cut to 16 bits moves the scores by 2^-18."""
    p = Problem(dtype, [3001], hq, 1, nodes, 300 + nodes)
    got, want = p.run(), p.want()
    assert np.linalg.norm(got - want) <= 2.0 ** -20 * np.linalg.norm(want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_a_row_does_not_see_does_not_reach_it(device, dtype):
    """NaN and infinities in the slots behind a history, in pages of no
    sequence, in tree rows outside a node's way to its root and behind the
    node count leave the other rows as they are; rows that see a NaN are NaN."""
    nodes = 12
    parents = np.array([[-1, 0, 0, 1, 2, 3, 4, 0, 7, 8, 2, 10]] * 4, np.int32)
    p = Problem(dtype, [5, 40, 0, 333], 8, 2, nodes, 3, parents=parents, counts=[12, 12, 12, 9])
    own = np.zeros((p.N, P), bool)
    for b, n in enumerate(p.hists):
        for i in range(n):
            own[p.tables[b, i // P], i % P] = True
    for pool in (p.kp, p.vp):
        pool.transpose(0, 2, 1, 3)[~own] = np.nan
    for x, bad in ((p.tv, np.nan), (p.tk, np.nan), (p.tv, np.inf)):
        at = int(p.rng.integers(0, D))
        keep = x[:, :, 4].copy(), x[:, :, 9:].copy()
        x[:, :, 4, at] = bad  # seen by nodes 4 and 6 alone
        x[3, :, 9:] = bad     # behind sequence 3's count
        got, want = p.run(), p.want()
        rest = [t for t in range(nodes) if t not in (4, 6)]
        assert np.isfinite(want[:, :, rest]).all()
        close(got[:, :, rest], want[:, :, rest])
        if not (dtype == "fp8" and np.isinf(bad)):  # (fp8 pages saturate)
            assert not np.isfinite(want[:, :, [4, 6]]).all(axis=-1).any()
        np.testing.assert_allclose(got, want, atol=ATOL, rtol=RTOL)
        x[:, :, 4], x[:, :, 9:] = keep


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nodes,long", [(3, 700), (20, 90)])
def test_infinities_in_the_history(device, dtype, nodes, long):
    """A key whose score is -inf takes no part, values of +-inf reach every
    row, fp32's largest values stay finite: as plain arithmetic has it."""
    p = Problem(dtype, [long, 64, 30], 4, 1, nodes, 8)
    p.q = np.abs(p.q) + 0.1
    p.kp[p.tables[0, 1], 0, 3, 17] = -np.inf
    p.vp[p.tables[1, 2], 0, 5, 40] = np.inf
    p.vp[p.tables[1, 2], 0, 5, 41] = -np.inf
    p.kp[p.tables[2, 0], 0, 1, 8] = -3.3e38
    got, want = p.run(), p.want()
    assert np.isfinite(want[0]).all() and np.isfinite(want[2]).all()
    close(got, want)


@pytest.mark.parametrize("scale", [1e-6, 1e-3, 3e3])
@pytest.mark.parametrize("dtype", DTYPES)
def test_small_and_large_magnitudes(device, dtype, scale):
    """Queries shrunk and keys grown by the same factor (scores stay as they
    are), values grown: results to the same relative tolerance."""
    p = Problem(dtype, [50, 0, 400], 8, 2, 10, 4)
    if dtype != "fp8":  # fp8 codes cover their scale's range only
        p.kp *= np.float32(scale)
        p.tk *= np.float32(scale)
        p.vp *= np.float32(scale)
        p.tv *= np.float32(scale)
    p.q *= np.float32(1 / scale if dtype != "fp8" else 1.0)
    if dtype == "fp8":
        p.q *= np.float32(min(scale, 20.0))
    got, want = p.run(), p.want()
    unit = scale if dtype != "fp8" else 1.0
    np.testing.assert_allclose(got[:] / unit, want / unit, atol=ATOL, rtol=RTOL)


def test_bad_pages_lengths_and_parents_give_nan_where_they_reach(device):
    parents = np.array([[-1, 0, 1, 0, 3, 2]] * 5, np.int32)
    parents[3, 2] = 4    # behind its node: nodes 2 and 5 hang from it
    parents[4, 3] = -7
    p = Problem("bf16", [100, 40, 40, 40, 40], 4, 2, 6, 21, parents=parents)
    want = p.want()
    d = p.tensors()
    d["tables"][0, 3] = p.N          # outside the pool
    d["tables"][0, 4] = -1
    d["lengths"][1] = -1
    d["lengths"][2] = 16 * d["tables"].shape[1] + 1
    hx.paged_tree_attention(**d)
    got = host(d["output"])
    assert np.isnan(got[:3]).all()
    close(got[3:], want[3:])
    assert np.isnan(got[3][:, [2, 5]]).all() and np.isnan(got[4][:, [3, 4]]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_page_offsets_past_32_bits(device, dtype):
    """Pages at the end of a pool of more than 2^32 elements."""
    hkv = 2
    N = (1 << 32) // (hkv * P * D) + 70
    pool = lambda: torch.empty(N, hkv, P, D, device="cuda:0", dtype={  # noqa: E731
        "f32": torch.float32, "bf16": torch.bfloat16, "fp8": torch.uint8}[dtype])
    p = Problem(dtype, [700, 90], 4, hkv, 5, 31)
    want = p.want()
    d = p.tensors()
    kp, vp = pool(), pool()
    kp[N - p.N:], vp[N - p.N:] = d["key_pool"], d["value_pool"]
    d.update(key_pool=kp, value_pool=vp, tables=d["tables"] + (N - p.N))
    hx.paged_tree_attention(**d)
    close(host(d["output"]), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_calls_are_bit_identical_and_streams_apart(device, dtype):
    p = Problem(dtype, [2000, 17, 900, 0], 8, 2, 16, 55)
    first = p.run()
    d = p.tensors()
    side = torch.cuda.Stream()
    other = Problem(dtype, [1200, 3, 0, 45], 8, 2, 16, 56)
    e = other.tensors()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):  # two calls at once, a workspace each
        hx.paged_tree_attention(**d)
    hx.paged_tree_attention(**e)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(host(d["output"]), first)
    close(host(e["output"]), other.want())


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_call_replays_with_other_lengths_and_trees(device, dtype):
    p = Problem(dtype, [300, 900, 64, 0], 8, 2, 16, 91)
    d = p.tensors()
    d["node_counts"] = torch.full((p.B,), 16, dtype=torch.int32, device="cuda:0")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        hx.paged_tree_attention(**d)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        hx.paged_tree_attention(**d)
    for step in range(3):
        p.hists = [[300, 900, 64, 0], [7, 890, 33, 0], [300, 0, 50, 0]][step]
        p.pages = [(h + P - 1) // P for h in p.hists]
        p.counts = [[16] * 4, [3, 16, 0, 9], [1, 2, 16, 16]][step]
        d["lengths"].copy_(dev(np.array(p.hists, np.int32)))
        d["node_counts"].copy_(dev(np.array(p.counts, np.int32)))
        d["output"].fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = host(d["output"])
        close(got, p.want())
        eager = p.tensors()
        hx.paged_tree_attention(**eager)
        np.testing.assert_array_equal(host(eager["output"]), got)


# ---------------------------------------------------------- verification ----
def drafts(rng, b, t, v, parents, certain, flat=False):
    """Random target and drafter rows and the drafter's tokens."""
    logits = rng.standard_normal((b, t, v)) * (0.1 if flat else 2.0)
    soft = lambda x: (np.exp(x) / np.exp(x).sum(-1, keepdims=True)).astype(np.float32)  # noqa: E731
    target = soft(logits)
    draft = soft(logits + 0.7 * rng.standard_normal((b, t, v)))
    tokens = np.zeros((b, t), np.int32)
    for i in range(b):
        for c in range(t):
            row = draft[i, max(0, min(parents[i, c], t - 1))].astype(np.float64)
            tokens[i, c] = (rng.choice(v, p=row / row.sum()) if v < 3000 else
                            min(v - 1, np.searchsorted(np.cumsum(row), rng.random() * row.sum())))
    return target, None if certain else draft, tokens


class Check:
    """One verification and its plain form."""

    def __init__(self, target, draft, tokens, parents, uniforms, bonus, counts=None):
        self.a = (target, draft, tokens, parents, uniforms, bonus, counts)
        b, t, v = target.shape
        i32 = dict(dtype=torch.int32, device="cuda:0")
        self.d = dict(target=dev(target), draft=None if draft is None else dev(draft),
                      tokens=dev(tokens), parents=dev(parents), uniforms=dev(uniforms),
                      bonus_uniforms=dev(bonus), path=torch.full((b, t), 99, **i32),
                      accepted=torch.full((b,), 99, **i32), next_token=torch.full((b,), 99, **i32),
                      workspace=hx.verify_workspace(b, t, v),
                      node_counts=None if counts is None else dev(np.asarray(counts, np.int32)))
        self.d["workspace"].fill_(255)

    def run(self):
        hx.verify_tree(**self.d)
        torch.cuda.synchronize()
        return self.compare()

    def compare(self):
        target, draft, tokens, parents, uniforms, bonus, counts = self.a
        b, t, _ = target.shape
        path, accepted, after = (host(self.d[n]) for n in ("path", "accepted", "next_token"))
        for i in range(b):
            n = t if counts is None else min(max(int(counts[i]), 0), t)
            way, follow = ref.verify(target[i], None if draft is None else draft[i], tokens[i],
                                     parents[i], n, uniforms[i], bonus[i])
            assert list(path[i]) == way + [-1] * (t - len(way)), i
            assert (accepted[i], after[i]) == (len(way), follow), i
        return accepted


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("b,t,v", [(1, 1, 1), (3, 2, 2), (40, 8, 17), (7, 64, 63), (5, 13, 1000),
                                   (30, 6, 257), (2, 5, 32000), (3, 16, 128257)])
def test_verification_equals_the_plain_form(device, certain, b, t, v):
    rng = np.random.default_rng(b * 1000 + t + v)
    for parents in (ref.random_trees(rng, b, t), ref.chain(b, t)):
        target, draft, tokens = drafts(rng, b, t, v, parents, certain)
        u, bonus = rng.random((b, t), np.float32), rng.random(b, np.float32)
        Check(target, draft, tokens, parents, u, bonus).run()


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("v", [20011, 49153, 90001, 131072])
def test_verification_of_many_rejections(device, certain, v):
    """All nodes are the root's children, hard to accept: a sum over the vocabulary
    for each, some of the sequences' first children accepted."""
    rng = np.random.default_rng(v)
    b, t = 3, 12
    parents = np.zeros((b, t), np.int32)
    parents[:, 0] = -1
    target, draft, tokens = drafts(rng, b, t, v, parents, certain)
    u = np.full((b, t), 0.9999, np.float32)
    u[1, 1] = 0.0
    accepted = Check(target, draft, tokens, parents, u, rng.random(b, np.float32)).run()
    assert accepted[1] == 2


@pytest.mark.parametrize("certain", [False, True])
def test_verification_at_its_edges(device, certain):
    """Siblings with one token, tokens and parents out of range, ragged counts,
    a bonus number of 0 and just below 1, rows with zeros, a target equal to
    the drafter, a drafter whose token the target rules out."""
    rng = np.random.default_rng(9)
    b, t, v = 24, 12, 301
    parents = ref.random_trees(rng, b, t, forest=True)
    target, draft, tokens = drafts(rng, b, t, v, parents, certain, flat=True)
    tokens[:, 3] = tokens[:, 2]
    tokens[0:3, 4] = [-1, v, 2**31 - 1]
    parents[3:6, 5] = [5, 11, -9]
    counts = rng.integers(-1, t + 3, b)
    bonus = rng.random(b, np.float32)
    bonus[:6] = [0.0, 0.0, np.nextafter(np.float32(1), np.float32(0)), 0.99999, 0.0, 1e-30]
    target[6:9, :, : v // 2] = 0
    target[9, :, tokens[9]] = 0
    if draft is not None:
        draft[10:13] = target[10:13]
        draft[13] = 0
    u = rng.random((b, t), np.float32)
    u[14] = 0
    u[15] = np.nextafter(np.float32(1), np.float32(0))
    Check(target, draft, tokens, parents, u, bonus, counts).run()


def test_verification_where_nothing_is_left(device):
    """The whole of a row rejected: its own probabilities stand; a row without
    any: no token."""
    target = np.zeros((3, 2, 70), np.float32)
    target[0, 0, [5, 9]] = 0.25, 0.5
    draft = np.zeros((3, 2, 70), np.float32)
    draft[:, 0, [5, 9]] = 0.5, 1.0
    tokens = np.array([[0, 9]] * 3, np.int32)
    u = np.full((3, 2), 0.75, np.float32)
    bonus = np.array([0.5, 0.5, 0.0], np.float32)
    c = Check(target, draft, tokens, ref.chain(3, 2), u, bonus)
    c.run()
    assert list(host(c.d["next_token"])) == [9, -1, -1]
    assert list(host(c.d["accepted"])) == [1, 1, 1]


def test_verification_of_strided_rows_on_another_stream_and_captured(device):
    rng = np.random.default_rng(12)
    b, t, v = 6, 9, 5003
    parents = ref.random_trees(rng, b, t)
    target, draft, tokens = drafts(rng, b, t, v, parents, False)
    c = Check(target, draft, tokens, parents, rng.random((b, t), np.float32),
              rng.random(b, np.float32))
    wide = torch.full((b, t + 2, v + 5), float("nan"), device="cuda:0")
    wide[:, 1:t + 1, 3:v + 3] = c.d["target"]
    c.d["target"] = wide[:, 1:t + 1, 3:v + 3]
    turned = torch.empty(t, b, v, device="cuda:0")
    turned.copy_(c.d["draft"].transpose(0, 1))
    c.d["draft"] = turned.transpose(0, 1)
    c.run()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        hx.verify_tree(**c.d)
    for step in range(3):
        u = rng.random((b, t), np.float32)
        bonus = rng.random(b, np.float32)
        c.a = (*c.a[:4], u, bonus, None)
        c.d["uniforms"].copy_(dev(u))
        c.d["bonus_uniforms"].copy_(dev(bonus))
        c.d["path"].fill_(99)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.compare()
    with torch.cuda.stream(side):
        hx.verify_tree(**c.d)
    side.synchronize()
    c.compare()


def test_verification_of_a_large_batch(device):
    rng = np.random.default_rng(14)
    b, t, v = 1500, 4, 40
    parents = ref.random_trees(rng, b, t)
    target, draft, tokens = drafts(rng, b, t, v, parents, False)
    accepted = Check(target, draft, tokens, parents, rng.random((b, t), np.float32),
                     rng.random(b, np.float32)).run()
    assert len(set(accepted)) > 2


# ---------------------------------------------------------------- append ----
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layers,b,hkv,t,page,dim,shift", [
    (1, 1, 1, 1, 16, 128, 0), (3, 5, 2, 7, 16, 128, 0), (2, 3, 3, 5, 7, 37, 0),
    (2, 2, 8, 64, 16, 128, 1), (4, 9, 2, 3, 32, 80, 0), (1, 70, 4, 2, 4, 64, 0)])
def test_append_path_writes_the_accepted_rows_alone(device, dtype, layers, b, hkv, t, page, dim,
                                                    shift):
    rng = np.random.default_rng(layers * 10 + t)
    each = (t + page - 1) // page + 1
    N = b * each + 1
    width = {"f32": torch.float32, "bf16": torch.bfloat16, "fp8": torch.uint8}[dtype]
    src = [rng.standard_normal((layers, b, hkv, t, dim), dtype=np.float32) for _ in range(2)]
    slots = np.zeros((b, t), np.int64)
    path = np.full((b, t), -1, np.int32)
    accepted = rng.integers(0, t + 1, b).astype(np.int32)
    for i in range(b):
        pos = int(rng.integers(0, page)) + np.arange(t)
        slots[i] = (i * each + pos // page) * page + pos % page
        path[i, :accepted[i]] = np.sort(rng.permutation(t)[:accepted[i]])
    if t > 1:
        path[0, 0], accepted[0] = t, max(accepted[0], 1)      # a node past the tree
        slots[-1, 0], accepted[-1] = N * page, max(accepted[-1], 1)  # a slot past the pool
        path[-1, 0] = 0
    if b > 2 and t > 1:
        slots[1, 0], path[1, 0], accepted[1] = -5, 0, max(accepted[1], 1)
    pools, want = [], []
    for x in src:
        base = torch.randint(0, 100, (layers + 1, N, hkv, page, dim), device="cuda:0").to(width)
        pool = base[:layers]  # layers a stride apart
        expect = pool.clone()
        rows = to_pool(dtype, x, 1.0 if dtype != "fp8" else (KS if x is src[0] else VS))
        for i in range(b):
            for j in range(accepted[i]):
                s, n = int(slots[i, j]), int(path[i, j])
                if 0 <= s < N * page and 0 <= n < t:
                    expect[:, s // page, :, s % page] = rows[:, i, :, n]
        pools.append(pool)
        want.append(expect)
    moved = []
    for x in src:  # rows at any 4-byte address
        flat = torch.empty(x.size + shift, device="cuda:0")
        flat[shift:] = dev(x).flatten()
        moved.append(flat[shift:].view(x.shape))
    kw = dict(k_scale=KS, v_scale=VS) if dtype == "fp8" else {}
    hx.append_path(*moved, *pools, dev(slots), dev(path), dev(accepted), page_dtype=dtype, **kw)
    torch.cuda.synchronize()
    for got, expect in zip(pools, want):
        assert torch.equal(got, expect)
    if layers == 1:  # the one-layer form
        again = [p.clone()[0] for p in want]
        hx.append_path(moved[0][0], moved[1][0], *again, dev(slots), dev(path), dev(accepted),
                       page_dtype=dtype, **kw)
        assert all(torch.equal(a, w[0]) for a, w in zip(again, want))


# --------------------------------------------------------- the whole step ----
class Server:
    """A cache of a few sequences beside host copies of their rows."""

    def __init__(self, dtype, hists, layers=2, hq=8, hkv=2, seed=1, max_tokens=512, spare=40):
        self.rng = np.random.default_rng(seed)
        self.dtype, self.layers, self.hq, self.hkv = dtype, layers, hq, hkv
        self.B = len(hists)
        kw = dict(k_scale=KS, v_scale=VS) if dtype == "fp8" else {}
        blocks = sum((h + P - 1) // P for h in hists) + spare
        self.cache = hx.PagedKvCache(layers, hkv, D, P, blocks, page_dtype=dtype, **kw)
        self.seqs, self.k, self.v = [], [], []
        for h in hists:
            s = self.cache.create_sequence()
            k, v = self.normal(layers, hkv, h, D), self.normal(layers, hkv, h, D)
            if h:
                self.cache.append_layer_major(s, [dev(x) for x in k], [dev(x) for x in v])
            self.seqs.append(s)
            self.k.append(on_pages(dtype, k, KS))
            self.v.append(on_pages(dtype, v, VS))
        self.batch = hx.DecodeBatch(self.cache, self.seqs, hq, max_tokens)

    def normal(self, *shape):
        return self.rng.standard_normal(shape, dtype=np.float32)

    def tree_step(self, nodes, counts=None, commit="accept"):
        """One step; returns the accepted numbers."""
        B, L = self.B, self.layers
        parents = ref.random_trees(self.rng, B, nodes)
        q = self.normal(L, B, self.hq, nodes, D)
        k, v = self.normal(L, B, self.hkv, nodes, D), self.normal(L, B, self.hkv, nodes, D)
        dk, dv, dp = dev(k), dev(v), dev(parents)
        dc = None if counts is None else dev(np.array(counts, np.int32))
        self.batch.prepare_tree(nodes)
        for layer in range(L):
            out = torch.zeros(B, self.hq, nodes, D, device="cuda:0")
            self.batch.tree_layer(layer, dev(q[layer]), dk[layer], dv[layer], dp, out,
                                  node_counts=dc)
            for b in range(B):
                want = np.zeros((self.hq, nodes, D))
                ref.tree_attention(q[layer, b], self.k[b][layer], self.v[b][layer],
                                   on_pages(self.dtype, k[layer, b], KS),
                                   on_pages(self.dtype, v[layer, b], VS), parents[b],
                                   nodes if counts is None else counts[b], want)
                close(host(out[b]), want)
        i32 = dict(dtype=torch.int32, device="cuda:0")
        path = torch.empty(B, nodes, **i32)
        accepted, after = torch.empty(B, **i32), torch.empty(B, **i32)
        if commit is None:
            return None
        if commit == "accept":
            target, draft, tokens = drafts(self.rng, B, nodes, 50, parents, False)
            u, bonus = self.rng.random((B, nodes), np.float32), self.rng.random(B, np.float32)
            self.batch.accept_tree(dev(target), dev(draft), dev(tokens), dp, dev(u), dev(bonus),
                                   dk, dv, path, accepted, after, node_counts=dc)
            for b in range(B):
                way, follow = ref.verify(target[b], draft[b], tokens[b], parents[b],
                                         nodes if counts is None else counts[b], u[b], bonus[b])
                assert list(host(path[b])[:len(way)]) == way and int(after[b]) == follow
                assert int(accepted[b]) == len(way)
        else:
            for b in range(B):
                t = int(self.rng.integers(0, nodes))
                way = sorted(ref.ancestors(parents[b], t))
                path[b, :len(way)] = torch.tensor(way, **i32)
                accepted[b] = len(way)
            self.batch.commit_path(dk, dv, path, accepted)
        for b in range(B):
            way = host(path[b])[:int(accepted[b])]
            self.k[b] = np.concatenate([self.k[b], on_pages(self.dtype, k[:, b][:, :, way], KS)], 2)
            self.v[b] = np.concatenate([self.v[b], on_pages(self.dtype, v[:, b][:, :, way], VS)], 2)
        self.compare()
        return host(accepted)

    def decode_step(self):
        q = self.normal(self.layers, self.B, self.hq, D)
        k, v = self.normal(self.layers, self.B, self.hkv, D), self.normal(self.layers, self.B,
                                                                        self.hkv, D)
        self.batch.prepare()
        for layer in range(self.layers):
            out = torch.empty(self.B, self.hq, D, device="cuda:0")
            self.batch.append_attention_layer(layer, dev(q[layer]), dev(k[layer]), dev(v[layer]),
                                              out)
            for b in range(self.B):
                want = np.zeros((self.hq, 1, D))
                ref.tree_attention(q[layer, b][:, None], self.k[b][layer], self.v[b][layer],
                                   on_pages(self.dtype, k[layer, b][:, None], KS),
                                   on_pages(self.dtype, v[layer, b][:, None], VS), [-1], 1, want)
                close(host(out[b]), want[:, 0])
        for b in range(self.B):
            self.k[b] = np.concatenate([self.k[b], on_pages(self.dtype, k[:, b][:, :, None], KS)], 2)
            self.v[b] = np.concatenate([self.v[b], on_pages(self.dtype, v[:, b][:, :, None], VS)], 2)
        torch.cuda.synchronize()
        self.compare()

    def compare(self):
        used = 0
        for b, s in enumerate(self.seqs):
            n = self.k[b].shape[2]
            assert self.cache.length(s) == n
            assert len(self.cache.block_table(s)) == (n + P - 1) // P
            used += (n + P - 1) // P
            for layer in range(self.layers):
                gk, gv = self.cache.retrieve_layer(s, layer)
                np.testing.assert_array_equal(host(gk), self.k[b][layer])
                np.testing.assert_array_equal(host(gv), self.v[b][layer])
        assert self.cache.stats()["used_blocks"] == used


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_server_of_tree_steps(device, dtype):
    """Tree steps of several sizes, an ordinary decode step between them, trees
    of no nodes for some sequences, a dropped step, a truncated member: tables,
    pages and results stay those of the accepted tokens."""
    s = Server(dtype, [0, 1, 15, 16, 100, 37])
    s.tree_step(6)
    s.tree_step(20, counts=[20, 0, 3, 1, 20, 7])
    s.decode_step()
    s.tree_step(64, commit="path")
    s.tree_step(5, commit=None)  # dropped by the next prepare
    s.decode_step()
    s.tree_step(9, commit=None)
    s.tree_step(13)
    cut = s.cache.length(s.seqs[4]) - 30
    s.cache.truncate_sequence(s.seqs[4], cut)
    s.k[4], s.v[4] = s.k[4][:, :, :cut], s.v[4][:, :, :cut]
    s.tree_step(1)
    s.decode_step()
    s.batch.close()
    s.cache.close()


def test_tree_step_refusals_and_order(device):
    s = Server("f32", [20, 33], layers=1, spare=7)
    b, t = s.batch, 4
    z = lambda *n, **kw: torch.zeros(*n, device="cuda:0", **kw)  # noqa: E731
    i32 = dict(dtype=torch.int32)
    q, rows = z(2, 8, t, D), z(2, 2, t, D)
    parents, path, accepted = z(2, t, **i32), z(2, t, **i32), z(2, **i32)
    keys = z(1, 2, 2, t, D)

    def refused(call, status=hx.INVALID_ARGUMENT):
        with pytest.raises(hx.HelixError) as e:
            call()
        assert e.value.status == status

    b._nodes = t
    refused(lambda: b.tree_layer(0, q, rows, rows, parents, torch.empty_like(q)))  # not prepared
    refused(lambda: b.commit_path(keys, keys, path, accepted))
    b.prepare_chunk(t)  # a chunk step is no tree step
    refused(lambda: b.tree_layer(0, q, rows, rows, parents, torch.empty_like(q)))
    for seq, n in zip(s.seqs, (20, 33)):
        s.cache.truncate_sequence(seq, n)
    refused(lambda: b.prepare_tree(65))
    refused(lambda: b.prepare_tree(0))
    b.prepare_tree(t)
    refused(lambda: b.tree_layer(1, q, rows, rows, parents, torch.empty_like(q)), hx.OUT_OF_RANGE)
    refused(lambda: b.tree_layer(0, q, rows, rows, parents, q))  # output is the query
    refused(lambda: b.tree_layer(0, q[:, :, :3], rows, rows, parents, torch.empty_like(q)))
    accepted.fill_(t + 1)
    refused(lambda: b.commit_path(keys, keys, path, accepted))
    accepted.fill_(1)
    s.cache.truncate_sequence(s.seqs[0], 22)  # below the step
    refused(lambda: b.commit_path(keys, keys, path, accepted))
    refused(lambda: b.tree_layer(0, q, rows, rows, parents, torch.empty_like(q)))
    s.cache.truncate_sequence(s.seqs[0], 20)
    b.prepare_tree(t)
    b.commit_path(keys, keys, path, accepted)
    assert [s.cache.length(x) for x in s.seqs] == [21, 34]
    refused(lambda: b.commit_path(keys, keys, path, accepted))  # once
    # A pool too small for the trees leaves everything as it was.
    refused(lambda: b.prepare_tree(64), hx.RESOURCE_EXHAUSTED)
    assert [s.cache.length(x) for x in s.seqs] == [21, 34]
    b.prepare()
    assert [s.cache.length(x) for x in s.seqs] == [22, 35]


def test_tree_layers_on_other_streams_and_captured(device):
    """A layer's call on a side stream waits for the step's upload, and a
    captured one replays."""
    s = Server("bf16", [60, 5, 200], layers=1)
    nodes = 7
    parents = ref.random_trees(s.rng, 3, nodes)
    q, k, v = s.normal(3, 8, nodes, D), s.normal(3, 2, nodes, D), s.normal(3, 2, nodes, D)
    want = np.zeros((3, 8, nodes, D))
    for b in range(3):
        ref.tree_attention(q[b], s.k[b][0], s.v[b][0], on_pages("bf16", k[b], 1),
                           on_pages("bf16", v[b], 1), parents[b], nodes, want[b])
    args = dev(q), dev(k), dev(v), dev(parents)
    side, out = torch.cuda.Stream(), torch.zeros(3, 8, nodes, D, device="cuda:0")
    torch.cuda.synchronize()
    s.batch.prepare_tree(nodes)
    s.batch.tree_layer(0, *args, out, stream=side)
    side.synchronize()
    close(host(out), want)
    s.batch.prepare_tree(nodes, stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s.batch.tree_layer(0, *args, out)
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        close(host(out), want)


def refused(call, status=hx.INVALID_ARGUMENT):
    with pytest.raises(hx.HelixError) as e:
        call()
    assert e.value.status == status


def cut_and_grow(s, b, keep, more):
    """Truncates member b to `keep` tokens and appends `more` others."""
    k, v = s.normal(s.layers, s.hkv, more, D), s.normal(s.layers, s.hkv, more, D)
    s.cache.truncate_sequence(s.seqs[b], keep)
    s.cache.append_layer_major(s.seqs[b], [dev(x) for x in k], [dev(x) for x in v])
    s.k[b] = np.concatenate([s.k[b][:, :, :keep], on_pages(s.dtype, k, KS)], 2)
    s.v[b] = np.concatenate([s.v[b][:, :, :keep], on_pages(s.dtype, v, VS)], 2)


@pytest.mark.parametrize("dtype", ["f32", "fp8"])
@pytest.mark.parametrize("keep", [0, 16, 18])
def test_a_member_cut_after_prepare_ends_an_ordinary_step(device, dtype, keep):
    """Also where it has grown back to the step's length by then: its tokens, on
    other pages or on the step's, are not the step's to write."""
    s = Server(dtype, [20, 33, 16], spare=8)
    b, B, L = s.batch, s.B, s.layers
    rows, all_rows = torch.ones(B, s.hkv, D, device="cuda:0"), torch.ones(L, B, s.hkv, 1, D,
                                                                         device="cuda:0")
    q = torch.ones(B, s.hq, D, device="cuda:0")
    b.prepare()
    cut_and_grow(s, 0, keep, 21 - keep)
    other = s.cache.create_sequence()  # takes pages that the cut freed
    filler = [torch.full((s.hkv, 30, D), 5.0, device="cuda:0")] * L
    s.cache.append_layer_major(other, filler, filler)
    assert s.cache.length(s.seqs[0]) == 21
    before = [host(s.cache.retrieve_layer(other, 1)[i]) for i in (0, 1)]
    refused(lambda: b.append_layer(0, rows, rows))
    refused(lambda: b.append_all_layers(all_rows, all_rows))
    refused(lambda: b.attention_layer(0, q, rows, rows, torch.empty_like(q)))
    refused(lambda: b.append_attention_layer(0, q, rows, rows, torch.empty_like(q)))
    torch.cuda.synchronize()
    for i in (0, 1):
        np.testing.assert_array_equal(host(s.cache.retrieve_layer(other, 1)[i]), before[i])
    s.cache.release_sequence(other)
    for i in (1, 2):  # (the refused step's slots)
        s.cache.truncate_sequence(s.seqs[i], s.k[i].shape[2])
    s.compare()
    s.decode_step()
    s.tree_step(5)
    s.decode_step()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("keep", [0, 17, 20])
def test_a_member_cut_and_grown_after_prepare_tree_keeps_its_tokens(device, dtype, keep):
    """The step is refused, and the next prepare takes back the other members'
    reserved slots only."""
    s = Server(dtype, [20, 33, 16])
    b, B, t = s.batch, s.B, 4
    z = lambda *n, **kw: torch.zeros(*n, device="cuda:0", **kw)  # noqa: E731
    keys, q, rows = z(s.layers, B, s.hkv, t, D), z(B, s.hq, t, D), z(B, s.hkv, t, D)
    path, one = z(B, t, dtype=torch.int32), torch.ones(B, dtype=torch.int32, device="cuda:0")
    for _ in range(2):
        lengths = [s.k[i].shape[2] for i in range(B)]
        b.prepare_tree(t)
        cut_and_grow(s, 0, keep, lengths[0] + t - keep)
        assert s.cache.length(s.seqs[0]) == lengths[0] + t
        refused(lambda: b.tree_layer(0, q, rows, rows, None, torch.empty_like(q)))
        refused(lambda: b.commit_path(keys, keys, path, one))
        assert [s.cache.length(x) for x in s.seqs] == [n + t for n in lengths]
        s.decode_step()  # (compares every row)
        s.tree_step(6)


def test_two_batches_over_one_sequence_see_each_others_cuts(device):
    """A step that another batch's commit cuts into is refused; a cut of no tokens
    is none."""
    s = Server("f32", [20, 33], spare=20)
    other = hx.DecodeBatch(s.cache, s.seqs[:1], s.hq, 512)
    rows = torch.ones(1, s.hkv, D, device="cuda:0")
    z = lambda *n, **kw: torch.zeros(*n, device="cuda:0", **kw)  # noqa: E731
    s.batch.prepare_tree(4)
    other.prepare()  # behind the tree's slots
    refused(lambda: s.batch.commit_path(z(2, 2, 2, 4, D), z(2, 2, 2, 4, D),
                                        z(2, 4, dtype=torch.int32), z(2, dtype=torch.int32)))
    s.cache.truncate_sequence(s.seqs[0], 25)
    other.append_layer(0, rows, rows)
    s.cache.truncate_sequence(s.seqs[0], 24)
    refused(lambda: other.append_layer(0, rows, rows))
    s.cache.truncate_sequence(s.seqs[0], 20)
    s.decode_step()
    refused(lambda: other.append_layer(0, rows, rows))
    s.tree_step(3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hists", [[0, 7], [3001, 40], [20011]])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_wrong_parent_beside_values_that_are_no_numbers(device, dtype, hists, bad):
    """A tile of rows that a value of an unseen node makes NaN is computed again;
    its rows with a wrong parent on their way stay NaN, in units of one range and
    in joined ones, and the others come out as they are."""
    nodes = 12
    parents = np.array([[-1, 0, 0, 1, 2, 9, 4, 0, 7, 5, 2, 10]] * len(hists), np.int32)
    p = Problem(dtype, hists, 8, 2, nodes, 17, parents=parents)
    p.tv[:, :, 4, 77] = bad  # seen by nodes 4 and 6 alone
    got, want = p.run(), p.want()
    lost, seen = [5, 9], [4, 6]
    rest = [t for t in range(nodes) if t not in lost + seen]
    assert np.isnan(want[:, :, lost]).all() and np.isfinite(want[:, :, rest]).all()
    assert np.isnan(got[:, :, lost]).all()
    close(got, want)


def test_a_captured_layer_outlives_larger_steps(device):
    """What a captured launch reads and writes stays where it is: a graph of trees
    of 7 nodes is replayed behind trees of 64 and a chunk, and the batch's device
    state keeps its addresses from the batch's first step on."""
    s = Server("bf16", [60, 5, 200], layers=1, spare=60)
    b, nodes = s.batch, 7
    first = b.device_state()
    parents = ref.random_trees(s.rng, 3, nodes)
    q, k, v = s.normal(3, 8, nodes, D), s.normal(3, 2, nodes, D), s.normal(3, 2, nodes, D)
    args = dev(q), dev(k), dev(v), dev(parents)
    side, out = torch.cuda.Stream(), torch.zeros(3, 8, nodes, D, device="cuda:0")
    torch.cuda.synchronize()
    b.prepare_tree(nodes, stream=side)
    b.tree_layer(0, *args, out, stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        b.tree_layer(0, *args, out)
    for step in range(3):
        s.tree_step(64)
        assert b.device_state() == first
        lengths = [s.k[i].shape[2] for i in range(3)]
        b.prepare_chunk(100)
        for seq, n in zip(s.seqs, lengths):
            s.cache.truncate_sequence(seq, n)
        b.prepare_tree(nodes, stream=side)
        side.synchronize()
        assert b.device_state() == first
        want = np.zeros((3, 8, nodes, D))
        for i in range(3):
            ref.tree_attention(q[i], s.k[i][0], s.v[i][0], on_pages("bf16", k[i], 1),
                               on_pages("bf16", v[i], 1), parents[i], nodes, want[i])
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        close(host(out), want)


@pytest.mark.parametrize("nodes", [1, 4])
def test_a_tree_step_takes_tree_calls_alone(device, nodes):
    """The calls of the other steps would write rows that the next prepare drops,
    or attend as if the nodes were a chunk."""
    s = Server("f32", [20, 33])
    b, B, L = s.batch, s.B, s.layers
    one = lambda *n: torch.ones(*n, device="cuda:0")  # noqa: E731
    q, rows = one(B, s.hq, nodes, D), one(B, s.hkv, nodes, D)
    out = torch.full_like(q, 7.0)
    b.prepare_tree(nodes)
    refused(lambda: b.append_layer(0, rows, rows))
    refused(lambda: b.append_all_layers(one(L, *rows.shape), one(L, *rows.shape)))
    refused(lambda: b.prefill_layer(0, q, rows, rows, out))
    refused(lambda: b.attention_layer(0, q, rows, rows, out))
    refused(lambda: b.append_attention_layer(0, q, rows, rows, out))
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    s.tree_step(nodes)  # the step before is dropped
    s.decode_step()


def test_closing_a_batch_drops_its_uncommitted_tree_step(device):
    """As the next prepare would: members that changed since are left alone."""
    s = Server("f32", [20, 33, 16, 7])
    s.batch.prepare_tree(20)
    assert [s.cache.length(x) for x in s.seqs] == [40, 53, 36, 27]
    cut_and_grow(s, 0, 18, 22)
    s.cache.release_sequence(s.seqs[3])
    del s.seqs[3], s.k[3], s.v[3]
    s.batch.close()
    assert [s.cache.length(x) for x in s.seqs] == [40, 33, 16]
    s.compare()
    s.B = 3
    s.batch = hx.DecodeBatch(s.cache, s.seqs, s.hq, 512)
    s.tree_step(5)
    s.batch.prepare()  # an ordinary step's slots stay the members'
    s.batch.close()
    assert [s.cache.length(x) for x in s.seqs] == [s.k[i].shape[2] + 1 for i in range(3)]


def test_a_batch_with_a_tree_step_closes_inside_a_read_lease(device):
    s = Server("f32", [20, 33])
    s.batch.prepare_tree(20)
    with s.cache.read_sequence(s.seqs[1]) as view:
        s.batch.close()
        assert view.length() == 53  # the lease's copy
    assert [s.cache.length(x) for x in s.seqs] == [20, 33]
    s.compare()
    s.batch = hx.DecodeBatch(s.cache, s.seqs, s.hq, 512)
    with s.cache.read_sequence(s.seqs[0]):
        pass
    s.tree_step(4)
