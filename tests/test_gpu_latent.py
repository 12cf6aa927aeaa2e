"""Attention over a latent cache on the GPU, absorbed (paged_latent_attention) and
expanded (latent_prefill_attention), against plain 64-bit forms
(latent_reference.py), and a run of the operators as a model would make it.

Held to the tolerance of every attention entry point of the library: max-abs 2e-5
plus rel 1e-4, on the values the pages hold.  (Scores here have a standard
deviation of about 1.7 and are sums of 576 or 192 products, each rounded to 2^-24:
their error stays near 2e-6, which outputs of up to 5 take over.)"""

import numpy as np
import pytest
import torch

import helix_runtime_amd as hx
import latent_reference as ref
import oracle

pytestmark = pytest.mark.gpu

ATOL, RTOL = 2e-5, 1e-4
P, ROPE = 16, 64
SCALE = 192 ** -0.5
PS = 0.037
DTYPES = ["f32", "bf16", "fp8"]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")


def host(t):
    return t.detach().cpu().numpy()


def close(got, want):
    np.testing.assert_allclose(got, want, atol=ATOL, rtol=RTOL)


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda:0")


def held(dtype, x):
    if dtype == "bf16":
        return oracle.round_bf16(x)
    if dtype == "fp8":
        return oracle.round_fp8(x, PS)
    return x


def to_pool(dtype, x):
    t = dev(x)
    if dtype == "bf16":
        return t.to(torch.bfloat16)
    if dtype == "fp8":
        by = torch.full((), PS, device="cuda:0")
        return (t / by).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return t


def pytest_generate_tests(metafunc):
    """Each test of the absorbed form with tables as long as they have to be and with
    longer ones: the kernel's units may be of 64 or of 16 rows."""
    if metafunc.function.__name__.startswith("test_absorbed"):
        metafunc.fixturenames.append("room")
        metafunc.parametrize("room", [0, 1040], indirect=True)


@pytest.fixture
def room(request, monkeypatch):
    monkeypatch.setattr(Latent, "room", request.param)


class Latent:
    """Scattered pages and queries of one call; slots that hold no token, and pages
    that no table names, are NaN."""

    room = 0  # pages that the table could name besides

    def __init__(self, dtype, latent, lengths, hq, t, seed=0, counts=None):
        rng = self.rng = np.random.default_rng(seed + 31 * hq + t)
        self.dtype, self.n, self.hq, self.t = dtype, latent, hq, t
        self.lengths, self.counts = list(lengths), counts
        b = self.b = len(self.lengths)
        pages = [(x + P - 1) // P for x in self.lengths]
        physical = sum(pages) + 3
        self.rows = [rng.standard_normal((x, latent + ROPE), dtype=np.float32) for x in self.lengths]
        pool = np.full((physical, P, latent + ROPE), np.nan, np.float32)
        order = rng.permutation(physical)
        self.tables = np.full((b, max(1, max(pages)) + 1 + self.room), 0xffffffff, np.uint32)
        at = 0
        for i, n in enumerate(pages):
            ids = order[at:at + n]
            at += n
            self.tables[i, :n] = ids
            for j in range(n):
                part = self.rows[i][j * P:(j + 1) * P]
                pool[ids[j], :len(part)] = part
        self.pool = to_pool(dtype, pool)
        self.q = rng.standard_normal((b, hq, t, latent + ROPE), dtype=np.float32)

    def want(self, before=7.0):
        out = np.full((self.b, self.hq, self.t, self.n), before, np.float64)
        for i, x in enumerate(self.lengths):
            count = self.t if self.counts is None else min(max(int(self.counts[i]), 0), self.t)
            ref.latent_attention(self.q[i], held(self.dtype, self.rows[i]), x, count, SCALE, self.n,
                                 out[i])
        return out

    def arguments(self):
        return dict(query=dev(self.q), pool=self.pool, tables=dev(self.tables.view(np.int32)),
                    lengths=i32(self.lengths),
                    output=torch.full((self.b, self.hq, self.t, self.n), 7.0, device="cuda:0"),
                    workspace=hx.latent_workspace(self.b, self.hq, self.t, self.n), scale=SCALE,
                    token_counts=None if self.counts is None else i32(self.counts),
                    page_dtype=self.dtype, **(dict(page_scale=PS) if self.dtype == "fp8" else {}))

    def run(self, **other):
        d = {**self.arguments(), **other}
        d["workspace"].fill_(255)  # what an earlier call left is not read
        hx.paged_latent_attention(**d)
        torch.cuda.synchronize()
        return host(d["output"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("latent", [256, 512])
@pytest.mark.parametrize("hq,t", [(1, 1), (5, 1), (16, 1), (16, 2), (20, 1), (16, 3), (64, 1), (8, 9),
                                  (128, 1), (3, 33), (100, 2), (16, 16)])
def test_absorbed_over_rows(device, dtype, latent, hq, t):
    p = Latent(dtype, latent, [t, t + 1, 33 + t, 200, 517], hq, t)
    close(p.run(), p.want())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", [[1], [15], [16], [17], [31], [32], [33], [63], [64], [65], [1000],
                                     [5000], [3, 1, 2047, 1, 64, 65], list(range(1, 90))])
def test_absorbed_over_lengths(device, dtype, lengths):
    p = Latent(dtype, 512, lengths, 16, 1, seed=sum(lengths))
    close(p.run(), p.want())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,t", [(16, 5), (40, 2), (2, 70)])
def test_absorbed_rows_that_see_nothing_or_lie_behind(device, dtype, hq, t):
    """Counts of none, some, more than there are rows, and more than there are
    tokens: rows without a token are 0, rows behind the count stay."""
    counts = [t, 0, 1, t // 2, t + 5, -3, t]
    p = Latent(dtype, 512, [40, 300, 1, 17, 600, 100, t // 2 + 1], hq, t, seed=5, counts=counts)
    got, want = p.run(), p.want()
    close(got, want)
    assert (got[1] == 7).all() and (got[5] == 7).all() and (got[2, :, 1:] == 7).all()
    none = t - (t // 2 + 1)  # rows of the last sequence before its first token
    assert (got[6, :, :none] == 0).all() and (want[6, :, :none] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_absorbed_empty_sequences(device, dtype):
    p = Latent(dtype, 256, [0, 5, 0], 4, 2, counts=[2, 2, 0])
    got = p.run()
    close(got, p.want())
    assert (got[0] == 0).all() and (got[2] == 7).all()
    p = Latent(dtype, 256, [0], 4, 1)
    assert (p.run() == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp8"])
@pytest.mark.parametrize("hq,t", [(16, 4), (4, 40)])
def test_absorbed_later_tokens_do_not_reach_earlier_rows(device, dtype, hq, t):
    """The step's second token is NaN in its latent part, the third infinite in its
    rotated part (fp8: NaN): the first row is as without them, later rows NaN."""
    p = Latent(dtype, 512, [t, 30 + t, 95], hq, t, seed=9)
    want = p.want()
    for i, x in enumerate(p.lengths):
        page = lambda pos: (int(p.tables[i, pos // P]), pos % P)  # noqa: E731
        a, b = page(x - t + 1), page(x - t + 2)
        if dtype == "fp8":
            p.pool[a[0], a[1], 7] = 0x7f
            p.pool[b[0], b[1], 520] = 0x7f
        else:
            p.pool[a[0], a[1], 7] = float("nan")
            p.pool[b[0], b[1], 520] = float("inf")
    got = p.run()
    close(got[:, :, 0], want[:, :, 0])
    # (The NaN stands in a score of every row that sees it.)
    assert np.isnan(got[:, :, 1:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,t", [(16, 4), (5, 20), (40, 3), (128, 2)])
def test_absorbed_unseen_numbers_change_no_bit(device, dtype, hq, t):
    """Queries behind the counts, slots that hold no token, and the step's last token:
    rows that do not see them are equal bit by bit whatever they hold."""
    counts = [t, 1, t // 2, t, 2]
    p = Latent(dtype, 512, [300, 1000, 37, 90, 2100], hq, t, seed=11, counts=counts)
    got = []
    for size in (0.0, 1.0, 5.0, 40.0):
        rng = np.random.default_rng(int(size))
        some = lambda *s: size * rng.standard_normal(s, dtype=np.float32)  # noqa: E731
        for i, (n, count) in enumerate(zip(p.lengths, counts)):
            p.q[i, :, count:] = some(hq, t - count, p.n + ROPE)
            page, at = int(p.tables[i, (n - 1) // P]), (n - 1) % P
            p.pool[page, at:] = to_pool(dtype, some(P - at, p.n + ROPE))
        got.append(p.run())
    for i, count in enumerate(counts):
        for other in got[1:]:
            assert (other[i, :, :count - 1] == got[0][i, :, :count - 1]).all()
            assert (other[i, :, count:] == 7).all()


def test_absorbed_special_queries_stay_in_their_rows(device):
    p = Latent("bf16", 512, [50, 100], 20, 2)
    want = p.want()
    p.q[0, 3, 1, 5] = np.nan
    p.q[1, 17, 0, 570] = np.nan
    got = p.run()
    assert np.isnan(got[0, 3, 1]).all() and np.isnan(got[1, 17, 0]).all()
    got[0, 3, 1], got[1, 17, 0] = want[0, 3, 1], want[1, 17, 0]
    close(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_absorbed_large_scores(device, dtype):
    """Queries of which each follows one key: maxima that move far from block to
    block, and probabilities that are all but one 0."""
    p = Latent(dtype, 512, [300], 16, 1, seed=2)
    rows = held(dtype, p.rows[0])
    for h in range(16):
        p.q[0, h, 0] = rows[(h * 37) % 300] * np.float32(0.5 + h)
    got = p.run()
    # Scores up to 16 * 576 / 13.9 = 660, off by 660 * 2^-22 = 1.6e-4 at most in 32
    # bits; the weights of keys that matter are off by as much of themselves.
    np.testing.assert_allclose(got, p.want(), atol=1e-3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_absorbed_largest_queries(device, dtype):
    """Queries up to fp32's largest numbers, whose scores are of size 1."""
    p = Latent(dtype, 512, [40, 700, 3000], 16, 1, seed=4)
    p.q[:] = 0
    p.q[..., 520] = np.exp2(p.rng.uniform(125, 127.99, p.q.shape[:3]))
    for i, n in enumerate(p.lengths):
        at = torch.arange(n)
        page = torch.from_numpy(p.tables[i, :(n + P - 1) // P].astype(np.int64))[at // P]
        p.rows[i][:, 520] = p.rng.uniform(-0.25, 0.25, n) * PS
        p.pool[page, at % P, 520] = to_pool(dtype, p.rows[i][:, 520])
    got = p.run(scale=1e-36)
    p.q *= np.float32(1e-36 / SCALE)
    close(got, p.want())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,hq,t", [([3, 40, 700], 16, 4), ([5000], 16, 1), ([100] * 30 + [9000], 20, 2)])
def test_absorbed_scores_that_are_all_minus_infinity(device, dtype, lengths, hq, t):
    """Scores of -16 times 6e37 leave 32 bits' range: weights that are 0 / 0, so NaN and
    not the 0 of a row that sees nothing, in whole units and in parts of one."""
    p = Latent(dtype, 512, lengths, hq, t, seed=3)
    p.q[..., 516] = 0
    want = p.want()
    p.q *= np.float32(SCALE)
    p.q[:, ::2, :, 516] = 6e37
    for i, n in enumerate(lengths):
        at = torch.arange(n)
        page = torch.from_numpy(p.tables[i, :(n + P - 1) // P].astype(np.int64))[at // P]
        # (-416 PS, which fp8 pages hold, is -15.4.)
        p.pool[page, at % P, 516] = 0xfd if dtype == "fp8" else -16
    got = p.run(scale=1.0)
    for i, n in enumerate(lengths):
        none = max(t - n, 0)
        assert (got[i, :, :none] == 0).all()
        assert np.isnan(got[i, ::2, none:]).all()
        close(got[i, 1::2], want[i, 1::2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_absorbed_bad_lengths_and_pages(device, dtype):
    """A length past the table, a negative one, and a page outside the pool make
    their sequence NaN and leave the others."""
    p = Latent(dtype, 512, [40, 40, 40, 40, 40], 8, 2)
    want = p.want()
    d = p.arguments()
    d["lengths"] = i32([40, -1, d["tables"].shape[1] * P + 1, 40, 40])
    d["tables"][3, 1] = p.pool.shape[0]
    hx.paged_latent_attention(**d)
    got = host(d["output"])
    assert np.isnan(got[1:4]).all()
    close(got[[0, 4]], want[[0, 4]])


@pytest.mark.parametrize("hq,t", [(16, 1), (20, 3), (64, 2)])
def test_absorbed_strides(device, hq, t):
    """Queries as a product over heads leaves them, outputs as the next one takes
    them, and a buffer with gaps."""
    p = Latent("bf16", 512, [70, 5, 130], hq, t)
    q = torch.zeros(hq, 3, t, 600, device="cuda:0")
    q[..., 12:588] = dev(p.q).transpose(0, 1)
    out = torch.full((3, t, hq, 520), 7.0, device="cuda:0")
    got = p.run(query=q.transpose(0, 1)[..., 12:588], output=out.transpose(1, 2)[..., 4:516])
    close(got, p.want())
    assert (host(out)[..., :4] == 7).all() and (host(out)[..., 516:] == 7).all()


@pytest.mark.parametrize("dtype,hq,t", [("bf16", 16, 3), ("fp8", 128, 1), ("f32", 16, 1)])
def test_absorbed_long_sequences(device, dtype, hq, t):
    """131071 tokens beside short ones."""
    p = Latent(dtype, 512, [131071, 3, 70], hq, t)
    q = p.q[:, :4]  # (the reference takes some of the heads)
    got = p.run()
    p.q, p.hq = q, 4
    close(got[:, :4], p.want())


def test_absorbed_calls_are_equal_bit_by_bit(device):
    p = Latent("bf16", 512, [4000, 17, 900, 2500], 128, 1)
    first = p.run()
    for _ in range(3):
        assert (p.run() == first).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,t", [(16, 1), (40, 2)])
@pytest.mark.parametrize("sign", [-1, 0])
def test_absorbed_other_scales(device, dtype, hq, t, sign):
    """A negative scale turns the scores about; with none every token counts alike."""
    p = Latent(dtype, 512, [100, 0, 33], hq, t)
    got = p.run(scale=sign * SCALE)
    p.q = p.q * np.float32(sign)
    close(got, p.want())


@pytest.mark.parametrize("dtype,hq,t", [("f32", 16, 1), ("fp8", 8, 2), ("bf16", 40, 2)])
def test_absorbed_many_sequences(device, dtype, hq, t):
    """More units than workgroups, empty ones and one of many parts among them."""
    rng = np.random.default_rng(5)
    lengths = [int(x) for x in rng.integers(0, 40, 300)]
    lengths[7], lengths[150], lengths[299] = 30000, 0, 700
    counts = [int(x) for x in rng.integers(-1, t + 2, 300)]
    counts[7] = t
    p = Latent(dtype, 256, lengths, hq, t, counts=counts)
    close(p.run(), p.want())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,hq,t", [([300, 50, 700, 33], 128, 20), ([300, 50, 1700, 33], 64, 9),
                                          ([90, 200, 0, 1000], 64, 17), ([700, 3], 16, 40), ([2000, 30], 16, 17),
                                          ([5000], 20, 54)])
def test_absorbed_many_row_blocks(device, dtype, lengths, hq, t):
    """9 to 80 units of a sequence, with one list of tiles for all of them and with one
    each, ragged, sequences without rows among them."""
    counts = [t, 0, t // 3, t + 1][:len(lengths)]
    p = Latent(dtype, 512, lengths, hq, t, seed=13, counts=counts)
    got = p.run()
    heads = sorted({0, 1, hq // 3, hq - 2, hq - 1})
    p.q, p.hq = p.q[:, heads], len(heads)
    close(got[:, heads], p.want())
    for i, count in enumerate(counts):
        assert (got[i, :, min(count, t):] == 7).all() and np.isfinite(got[i]).all()


def test_absorbed_pools_past_32_bits(device):
    """Pages whose elements lie past 2^32 of the pool."""
    n = (1 << 32) // (P * 576) + 40
    pool = torch.zeros(n, P, 576, dtype=torch.uint8, device="cuda:0")
    p = Latent("fp8", 512, [100, 60], 16, 1)
    count = p.pool.shape[0]
    pool[n - count:] = p.pool
    tables = p.tables.astype(np.int64)
    tables[tables < count] += n - count
    got = p.run(pool=pool, tables=dev(tables.astype(np.uint32).view(np.int32)))
    close(got, p.want())


def test_absorbed_captured_and_replayed(device):
    """Two graphs with a workspace each, replayed side by side and in turns with
    other lengths and contents, against eager calls."""
    p, o = Latent("bf16", 512, [700, 40, 3], 16, 2), Latent("fp8", 512, [90, 1000], 128, 1)
    sets = [x.arguments() for x in (p, o)]
    graphs = []
    for d in sets:
        hx.paged_latent_attention(**d)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            hx.paged_latent_attention(**d)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    for i in range(3):
        for d in sets:
            d["query"].mul_(-1.1)
            d["lengths"].sub_(i)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for d, x in zip(sets, (p, o)):
            e = dict(d, output=torch.full_like(d["output"], 7.0),
                     workspace=hx.latent_workspace(x.b, x.hq, x.t))
            hx.paged_latent_attention(**e)
            torch.cuda.synchronize()
            assert torch.equal(torch.nan_to_num(e["output"]), torch.nan_to_num(d["output"]))


# --------------------------------------------------------------- expanded ----
class Expanded:
    def __init__(self, b, h, t, s, seed=0, counts=None, lengths=None):
        rng = self.rng = np.random.default_rng(seed + t + s)
        self.shape, self.counts, self.lengths = (b, h, t, s), counts, lengths
        normal = lambda *x: rng.standard_normal(x, dtype=np.float32)  # noqa: E731
        self.q, self.k, self.v = normal(b, h, t, 192), normal(b, h, s, 128), normal(b, h, s, 128)
        self.r = normal(b, s, 64)

    def want(self, before=7.0):
        b, h, t, s = self.shape
        out = np.full((b, h, t, 128), before, np.float64)
        for i in range(b):
            count = t if self.counts is None else min(max(int(self.counts[i]), 0), t)
            n = s if self.lengths is None else int(self.lengths[i])
            ref.expanded_attention(self.q[i], self.k[i], self.r[i], self.v[i], n, count, SCALE,
                                   out[i])
        return out

    def arguments(self):
        b, h, t, s = self.shape
        return dict(query=dev(self.q), key=dev(self.k), rope_key=dev(self.r), value=dev(self.v),
                    output=torch.full((b, h, t, 128), 7.0, device="cuda:0"),
                    workspace=hx.latent_prefill_workspace(b, h, t, s), scale=SCALE,
                    key_lengths=None if self.lengths is None else i32(self.lengths),
                    token_counts=None if self.counts is None else i32(self.counts))

    def run(self, **other):
        d = {**self.arguments(), **other}
        d["workspace"].fill_(255)
        hx.latent_prefill_attention(**d)
        torch.cuda.synchronize()
        return host(d["output"])


@pytest.mark.parametrize("b,h,t,s", [
    (1, 1, 1, 1), (1, 2, 1, 100), (2, 1, 5, 5), (1, 3, 16, 16), (2, 2, 17, 33), (1, 1, 63, 64),
    (1, 2, 64, 64), (1, 1, 65, 65), (3, 1, 33, 200), (1, 2, 128, 128), (1, 1, 130, 257), (1, 1, 300, 301),
    (2, 5, 40, 600)])
def test_expanded_over_sizes(device, b, h, t, s):
    p = Expanded(b, h, t, s)
    close(p.run(), p.want())


@pytest.mark.parametrize("t,s", [(70, 70), (33, 150)])
def test_expanded_ragged(device, t, s):
    """Counts and key lengths of each sequence: none, one, all; keys behind a
    sequence's are NaN and reach nothing; rows without a key are 0."""
    counts = [t, 0, 1, t // 2, t + 5, -3, t]
    lengths = [s, 0, 1, t // 2 + 3, s, 5, t // 2]
    p = Expanded(7, 2, t, s, counts=counts, lengths=lengths)
    for i, n in enumerate(lengths):
        p.k[i, :, n:], p.v[i, :, n:], p.r[i, n:] = np.nan, np.inf, np.nan
    got, want = p.run(), p.want()
    close(got, want)
    assert (got[1] == 7).all() and (got[5] == 7).all()
    assert (got[6, :, :t - t // 2] == 0).all()


def test_expanded_later_keys_do_not_reach_earlier_rows(device):
    """NaN, infinities and the type's extremes in keys and values of later tokens."""
    p = Expanded(1, 2, 70, 100)
    want = p.want()
    p.v[0, :, 60, 5], p.k[0, :, 75, 3], p.r[0, 90, 0] = np.inf, np.nan, -np.inf
    got = p.run()
    close(got[:, :, :30], want[:, :, :30])
    assert np.isnan(got[:, :, 45:]).all()
    assert not np.isfinite(got[:, :, 30:45, 5]).any()
    p = Expanded(1, 1, 20, 20)
    want = p.want()
    p.k[0, :, 15:], p.v[0, :, 15:] = -3.4e38, 3.4e38
    got = p.run()
    close(got[:, :, :15], want[:, :, :15])


@pytest.mark.parametrize("b,h,t,s", [(4, 3, 70, 100), (4, 2, 200, 500), (4, 70, 30, 300)])
def test_expanded_unseen_numbers_change_no_bit(device, b, h, t, s):
    """As in the absorbed form, with numbers of a size that no part is computed again
    for."""
    counts, lengths = [t, 1, t // 2, t - 1], [s, s - 1, s // 2, 2 * t // 3]
    p = Expanded(b, h, t, s, counts=counts, lengths=lengths)
    got = []
    for size in (0.1, 1.0, 3.0):
        rng = np.random.default_rng(int(10 * size))
        for i, (n, count) in enumerate(zip(lengths, counts)):
            for x in (p.q[i, :, count:], p.k[i, :, n - 1:], p.r[i, n - 1:], p.v[i, :, n - 1:]):
                x[...] = size * rng.standard_normal(x.shape, dtype=np.float32)
        got.append(p.run())
    for i, count in enumerate(counts):
        for other in got[1:]:
            assert (other[i, :, :count - 1] == got[0][i, :, :count - 1]).all()
            assert (other[i, :, count:] == 7).all()


@pytest.mark.parametrize("b,h,t,s", [(1, 2, 20, 300), (2, 1, 30, 20), (4, 40, 130, 140), (1, 1, 20, 3000)])
def test_expanded_scores_that_are_all_minus_infinity(device, b, h, t, s):
    """As in the absorbed form: NaN, not the 0 of a row that sees nothing."""
    p = Expanded(b, h, t, s)
    p.q[..., 3], p.k[..., 3] = 0, -16
    want = p.want()
    p.q *= np.float32(SCALE)
    p.q[:, :, ::3, 3] = 6e37
    got = p.run(scale=1.0)
    none = max(t - s, 0)
    assert (got[:, :, :none] == 0).all()
    large = np.arange(t) % 3 == 0
    assert np.isnan(got[:, :, large & (np.arange(t) >= none)]).all()
    close(got[:, :, ~large], want[:, :, ~large])


def test_expanded_sizes_of_numbers(device):
    """Keys and values a thousand times larger and smaller than each other, from
    block to block and from element to element."""
    p = Expanded(1, 2, 40, 300)
    p.v *= np.exp(p.rng.uniform(-7, 7, p.v.shape[:3] + (1,))).astype(np.float32)
    p.k *= np.exp(p.rng.uniform(-3, 0.5, p.k.shape)).astype(np.float32)
    got, want = p.run(), p.want()
    # Outputs are sums of values up to 4000: held to 2^-18 of the largest that a row
    # weighs, far above 32-bit rounding and far below 16 bits'.
    assert (np.abs(got - want) <= 2.0 ** -18 * np.abs(p.v).max()).all()
    assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want)


@pytest.mark.parametrize("b,h,t,s", [(1, 2, 40, 300), (4, 40, 130, 140)])
@pytest.mark.parametrize("kind", ["large keys", "large values", "a large dim", "large later values", "small values",
                                  "small later values", "zero keys first", "weightless values first"])
def test_expanded_range_of_numbers(device, b, h, t, s, kind):
    """Numbers past 16 bits' range, units alone and in parts: as precise as 32 bits
    are.  Scores keep their size, so their error stays near 2e-6 as above; an
    output's is twice that of the values' sizes that it weighs, held to five times
    that."""
    p = Expanded(b, h, t, s)
    first = slice(0, 33)
    if kind == "large keys":
        p.q, p.k, p.r = p.q * 2.0 ** -60, p.k * 2.0 ** 60, p.r * 2.0 ** 60
    elif kind == "large values":
        p.v *= np.float32(2.0 ** 90)
    elif kind == "a large dim":
        # (2^-33 of 2^12 times 4 is a tenth of what the others are held to.)
        p.v[..., 5] *= np.float32(2.0 ** 12)
    elif kind == "large later values":
        p.v[:, :, 100:] *= np.float32(2.0 ** 40)
    elif kind == "small values":
        p.v *= np.float32(2.0 ** -90)
    elif kind == "small later values":
        p.v[:, :, 33:] *= np.float32(2.0 ** -40)
    elif kind == "zero keys first":
        p.q, p.k, p.r = p.q * 2.0 ** 30, p.k * 2.0 ** -30, p.r * 2.0 ** -30
        p.k[:, :, first], p.r[:, first] = 0, 0
    else:
        # Scores of about -57 beside the others' of 2.
        p.q[..., 0], p.k[:, :, first, 0] = 8, -100
        p.k[:, :, 33:, 0] = 0
        p.v[:, :, first] *= np.float32(2.0 ** 30)
    p.q, p.k, p.r = (x.astype(np.float32) for x in (p.q, p.k, p.r))
    got, want = p.run(), p.want()
    p.v = np.abs(p.v)
    held_to = np.full(t, 2e-5)
    if kind == "weightless values first":
        # Rows that see those keys alone have scores of size 58, not of size 2.  The sum
        # is rounded at each matrix step, 6 steps of up to 6 products: to 58 * 2^-24 / 3 **
        # 0.5 in the mean, 36 ** 0.5 times that together, 1.2e-5; twice that for an output,
        # and five times that again for the largest of 80 thousand.
        held_to[:max(33 - (s - t), 0)] = 1.2e-4
    assert (np.abs(got - want) <= held_to[:, None] * p.want()).all()


def test_expanded_empty_rows_beside_nan(device):
    """Rows without a key are 0 whatever the keys and values of the unit's other rows,
    of the sequence before and behind the sequence are."""
    t, s = 70, 90
    lengths = [20, 0, s, 0, 65] * 20
    p = Expanded(100, 3, t, s, lengths=lengths)
    for i, n in enumerate(lengths):
        p.v[i, :, n:], p.k[i, :, n:], p.r[i, n:] = np.nan, np.nan, np.nan
        if i % 10 < 5:
            p.v[i, :, 0] = np.inf if i % 2 else np.nan
    got, want = p.run(), p.want()
    for i, n in enumerate(lengths):
        empty = max(t - n, 0)
        assert (got[i, :, :empty] == 0).all(), i
        if i % 10 < 5:
            assert not np.isfinite(got[i, :, empty:]).any(), i
        else:
            close(got[i], want[i])


@pytest.mark.parametrize("t", [10, 100])
def test_nothing_to_do(device, t):
    """No sequence has a row, or a key: outputs stay, or are 0."""
    p = Expanded(3, 2, t, 40, counts=[0, -1, 0])
    assert (p.run() == 7).all()
    p = Expanded(3, 2, t, 40, lengths=[0, 0, 0])
    assert (p.run() == 0).all()
    for room in (0, 1040):
        p = Latent("bf16", 256, [0, 0], 16, t)
        p.tables = np.full((2, 1 + room), 0xffffffff, np.uint32)
        assert (p.run() == 0).all()
        assert (p.run(token_counts=i32([0, -1])) == 7).all()


def test_expanded_bad_lengths(device):
    p = Expanded(4, 2, 10, 30)
    want = p.want()
    got = p.run(key_lengths=i32([30, -1, 31, 30]))
    assert np.isnan(got[1:3]).all()
    close(got[[0, 3]], want[[0, 3]])


def test_expanded_strides(device):
    """As projections leave queries, keys and values."""
    b, h, t, s = 2, 3, 50, 90
    p = Expanded(b, h, t, s)
    q = dev(p.q.transpose(0, 2, 1, 3))
    kv = dev(np.concatenate([p.k, p.v], axis=-1).transpose(0, 2, 1, 3))
    down = torch.zeros(b, s, 512 + 64, device="cuda:0")
    down[..., 512:] = dev(p.r)
    out = torch.full((b, t, h, 128), 7.0, device="cuda:0")
    got = p.run(query=q.transpose(1, 2), key=kv.transpose(1, 2)[..., :128],
                value=kv.transpose(1, 2)[..., 128:], rope_key=down[..., 512:],
                output=out.transpose(1, 2))
    close(got, p.want())


@pytest.mark.parametrize("t,s", [(50, 90), (130, 200)])
@pytest.mark.parametrize("sign", [-1, 0])
def test_expanded_other_scales(device, t, s, sign):
    p = Expanded(1, 2, t, s)
    got = p.run(scale=sign * SCALE)
    p.q = p.q * np.float32(sign)
    close(got, p.want())


@pytest.mark.parametrize("b,h,t,s", [(20, 20, 50, 300), (6, 50, 130, 400), (70, 3, 20, 60)])
def test_expanded_many_units(device, b, h, t, s):
    """More units than workgroups, or more sequences than a wavefront has lanes; some
    without rows or keys."""
    rng = np.random.default_rng(b)
    p = Expanded(b, h, t, s, counts=[int(x) for x in rng.integers(-1, t + 2, b)],
                 lengths=[int(x) for x in rng.integers(0, s + 1, b)])
    close(p.run(), p.want())


@pytest.mark.parametrize("b,h,t,s", [(5, 61, 130, 300), (13, 61, 50, 120), (2, 400, 65, 140)])
def test_expanded_heads_that_no_number_divides(device, b, h, t, s):
    """Histories longer than the step, and units of several heads to a workgroup: some
    sequences without rows, or shorter than their tables say."""
    rng = np.random.default_rng(h)
    p = Expanded(b, h, t, s, counts=[int(x) for x in rng.integers(t // 2, t + 2, b)],
                 lengths=[int(x) for x in rng.integers(s // 2, s + 1, b)])
    p.counts[0] = 0
    close(p.run(), p.want())


@pytest.mark.parametrize("b,h,t,s", [(1, 1, 20, 3000), (2, 1, 114, 2500), (1, 3, 130, 2000),
                                     (1, 16, 70, 1500)])
def test_expanded_few_units_in_many_parts(device, b, h, t, s):
    p = Expanded(b, h, t, s)
    close(p.run(), p.want())


@pytest.mark.parametrize("h,t,s", [(1, 8300, 8400), (9, 8250, 17000), (2, 8200, 300)])
def test_expanded_many_row_blocks(device, h, t, s):
    """More than 64 units of a head, whose heads take turns in the second case: sampled
    rows."""
    p = Expanded(1, h, t, s)
    got = p.run()
    assert np.isfinite(got).all()
    for head in {0, h // 2, h - 1}:
        key = np.concatenate([p.k[0, head], p.r[0]], axis=-1).astype(np.float64)
        for row in [0, 1, 127, 128, 4000, 8000, 8063, 8064, 8191, 8192, t - 2, t - 1]:
            n = max(s - t + row + 1, 0)
            x = (p.q[0, head, row].astype(np.float64) @ key[:n].T * SCALE)[None]
            close(got[0, head, row], ref.softmax_sum(x, p.v[0, head, :n].astype(np.float64))[0])


def test_expanded_one_long_sequence_among_many(device):
    """Broadcast keys of 300 sequences, of which one sees all and is in many parts."""
    b, t, s = 300, 20, 4000
    p = Expanded(b, 1, t, 1, lengths=[25] * b)
    p.lengths[100] = s
    d = p.arguments()
    p.shape = (b, 1, t, s)
    for name, key, tail in (("k", "key", (1, s, 128)), ("v", "value", (1, s, 128)),
                            ("r", "rope_key", (s, 64))):
        one = p.rng.standard_normal((1, *tail), dtype=np.float32)
        setattr(p, name, np.broadcast_to(one, (b, *tail)))
        d[key] = dev(one).expand(b, *tail)
    d["workspace"] = hx.latent_prefill_workspace(b, 1, t, s)
    d["workspace"].fill_(255)
    hx.latent_prefill_attention(**d)
    close(host(d["output"]), p.want())


@pytest.mark.parametrize("t", [20, 100])
def test_expanded_rows_far_apart(device, t):
    """Keys' rows as far apart as they may be, and sequences past 2^32 bytes."""
    b, h, s, far = 2, 1, 40, (1 << 25) - 4
    p = Expanded(b, h, t, s)
    d = p.arguments()
    room = torch.zeros(s * far, device="cuda:0")
    value = room.as_strided((b, h, s, 128), (256, 256, far, 1))
    value.copy_(d["value"])
    key = room.as_strided((b, h, s, 128), ((1 << 30) + 64, 128, 512, 1), 1024)
    key.copy_(d["key"])
    close(p.run(value=value, key=key), p.want())


def test_calls_on_streams_at_once(device):
    """Calls of both forms on two streams, a workspace each, on tensors of a third."""
    sets = [(hx.paged_latent_attention, Latent("bf16", 512, [900, 33, 5000], 16, 3).arguments()),
            (hx.paged_latent_attention, Latent("fp8", 512, [5000, 33], 16, 1).arguments()),
            (hx.latent_prefill_attention, Expanded(2, 9, 150, 700).arguments())]
    outs = []
    for call, d in sets:
        call(**d)
        torch.cuda.synchronize()
        outs.append(d["output"].clone())
        d["output"].fill_(7.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for (call, d), stream in zip(sets, streams):
            call(**d, stream=stream)
    torch.cuda.synchronize()
    for (_, d), out in zip(sets, outs):
        assert torch.equal(d["output"], out)


def test_expanded_captured_and_replayed(device):
    p = Expanded(3, 2, 65, 129, counts=[65, 10, 33], lengths=[129, 100, 33])
    d = p.arguments()
    hx.latent_prefill_attention(**d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hx.latent_prefill_attention(**d)
    for i in range(3):
        d["query"].mul_(-1.1)
        d["value"].add_(0.25)
        d["key_lengths"].sub_(i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        e = dict(d, output=torch.full_like(d["output"], 7.0),
                 workspace=hx.latent_prefill_workspace(*p.shape))
        hx.latent_prefill_attention(**e)
        torch.cuda.synchronize()
        assert torch.equal(e["output"], d["output"])


# ------------------------------------------------- as a model would run them ----
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_model_layer_over_prompt_and_steps(device, dtype):
    """One layer of latent attention: a prompt in the expanded form, then steps of one
    and of three tokens in the absorbed form over the pages that the appends filled,
    all against a recomputation in 64 bits from the values the pages hold."""
    h, n, batch = 4, 256, 3
    rng = np.random.default_rng(11)
    up_k, up_v = (rng.standard_normal((h, n, 128)).astype(np.float32) / 16 for _ in range(2))
    cos, sin = (torch.empty(64, 32, device="cuda:0") for _ in range(2))
    hx.rope_tables(cos, sin, base=10000.0, scaling="bands", factor=4.0, original_length=32)
    manager = hx.BlockManager(1, 1, n + ROPE, P, 40)
    pool = to_pool(dtype, np.full((40, P, n + ROPE), np.nan, np.float32))
    seqs = [manager.create_sequence() for _ in range(batch)]
    scale = dict(page_scale=PS) if dtype == "fp8" else {}
    past = [np.zeros((0, n + ROPE)) for _ in range(batch)]
    hc, hs = host(cos), host(sin)

    for step, counts in enumerate(([20, 7, 1], [1, 1, 1], [3, 0, 2], [1, 1, 1])):
        t = max(counts)
        starts = [manager.length(s) for s in seqs]
        slots = np.full((batch, t), -1, np.int64)
        for b, s in enumerate(seqs):
            if counts[b]:
                slots[b, :counts[b]] = manager.append(s, counts[b])
        width = max(len(manager.block_table(s)) for s in seqs)
        tables = np.zeros((batch, width), np.int32)
        for b, s in enumerate(seqs):
            table = manager.block_table(s)
            tables[b, :len(table)] = table
        latent = rng.standard_normal((batch, t, n), dtype=np.float32)
        rope_key = rng.standard_normal((batch, t, ROPE), dtype=np.float32)
        q = rng.standard_normal((batch, t, h, 192), dtype=np.float32)
        token_counts, dq = i32(counts), dev(q).transpose(1, 2)
        absorbed = torch.zeros(batch, h, t, n + ROPE, device="cuda:0")
        for b in range(h):
            absorbed[:, b, :, :n] = dq[:, b, :, :128] @ dev(up_k[b]).T
        hx.latent_append(dev(latent), dev(rope_key), pool, i32(starts), dev(slots), cos, sin,
                         query=dq[..., 128:], query_out=absorbed[..., n:], layout="halves",
                         token_counts=token_counts, page_dtype=dtype, **scale)
        # What the pages hold, in 64 bits.
        for b in range(batch):
            for j in range(counts[b]):
                turned = ref.rotate32(rope_key[b, j], hc[starts[b] + j], hs[starts[b] + j], "halves")
                row = held(dtype, np.concatenate([latent[b, j], turned])[None].astype(np.float32))
                past[b] = np.concatenate([past[b], row.astype(np.float64)])
        out = torch.full((batch, h, t, n), 7.0, device="cuda:0")
        hx.paged_latent_attention(absorbed, pool, dev(tables), i32([len(x) for x in past]), out,
                                  hx.latent_workspace(batch, h, t, n), SCALE,
                                  token_counts=token_counts, page_dtype=dtype, **scale)
        heads = torch.stack([out[:, i] @ dev(up_v[i]) for i in range(h)], dim=1)
        want = np.zeros((batch, h, t, 128))
        for b in range(batch):
            k, v = past[b][:, :n] @ up_k.astype(np.float64), past[b][:, :n] @ up_v.astype(np.float64)
            turned = np.stack([ref.rotate32(q[b, j, :, 128:], hc[starts[b] + j], hs[starts[b] + j],
                                            "halves") for j in range(counts[b])] or
                              [np.zeros((h, ROPE), np.float32)])
            whole = np.concatenate([q[b, :len(turned), :, :128], turned], axis=-1)
            ref.expanded_attention(whole.transpose(1, 0, 2), k, past[b][:, n:], v, len(past[b]),
                                   counts[b], SCALE, want[b])
        for b in range(batch):
            # The two products around the attention are fp32 sums of 128 and 256 terms.
            np.testing.assert_allclose(host(heads)[b, :, :counts[b]], want[b, :, :counts[b]],
                                       atol=1e-4, rtol=1e-4)
        if step == 0:
            rows = torch.zeros(batch, t, n + ROPE, device="cuda:0")
            for b in range(batch):
                rows[b, :counts[b]] = dev(past[b].astype(np.float32))
            key, value = (torch.stack([rows[..., :n] @ dev(u[i]) for i in range(h)], dim=1)
                          for u in (up_k, up_v))
            whole = torch.cat([dq[..., :128], absorbed[..., n:]], dim=-1)
            expanded = torch.zeros(batch, h, t, 128, device="cuda:0")
            hx.latent_prefill_attention(whole, key, rows[..., n:], value, expanded,
                                        hx.latent_prefill_workspace(batch, h, t, t), SCALE,
                                        key_lengths=token_counts, token_counts=token_counts)
            for b in range(batch):
                np.testing.assert_allclose(host(expanded)[b, :, :counts[b]],
                                           want[b, :, :counts[b]], atol=1e-4, rtol=1e-4)
