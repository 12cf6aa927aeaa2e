"""Rotary positions on the GPU: tables against 64-bit ones, rows and appends bit by
bit against the formula with every product and sum rounded to fp32, in both
layouts, over all of a head or a part, strided, in place, ragged, on every page
type, alone and as a step of DecodeBatch."""

import ctypes
import math

import numpy as np
import pytest
import torch

import helix_runtime_amd as hx
import latent_reference as ref
import oracle

pytestmark = pytest.mark.gpu

KS, VS = 0.037, 0.011
DTYPES = ["f32", "bf16", "fp8"]
LAYOUTS = ["pairs", "halves"]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")


def host(t):
    return t.detach().cpu().numpy()


def normal(rng, *shape):
    return rng.standard_normal(shape, dtype=np.float32)


def same_bits(got, want):
    np.testing.assert_array_equal(np.ascontiguousarray(got).view(np.uint32),
                                  np.ascontiguousarray(want, dtype=np.float32).view(np.uint32))


def on_pages(dtype, x, scale):
    """What a page holds of fp32 rows, as a pool tensor holds it."""
    if dtype == "bf16":
        return oracle.bf16_bits(x)
    if dtype == "fp8":
        return oracle.fp8_bits(x, scale)
    return np.ascontiguousarray(x, dtype=np.float32)


def pool_of(dtype, rng, *shape):
    """Pages of arbitrary contents, and their bits."""
    x = normal(rng, *shape)
    bits = on_pages(dtype, x, 1.0)
    t = dev(bits.view(np.int16) if dtype == "bf16" else bits)
    return t, bits


def bits_of(pool):
    x = host(pool)
    return x.view(np.uint16) if x.dtype == np.int16 else x


# ---------------------------------------------------------------- tables ----
@pytest.mark.parametrize("scaling", [
    dict(), dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
    dict(scaling="ramp", factor=16.0, original=4096), dict(scaling="ramp", factor=1.0, original=10),
    dict(scaling="ramp", factor=2.0, original=8192, low=2.0, high=5.5),
    dict(scaling="bands", factor=8.0, original=8192),
    dict(scaling="bands", factor=3.0, original=512, low=0.5, high=9.0)])
@pytest.mark.parametrize("rows,rotary,first", [(1, 128, 0), (17, 2, 5), (100, 50, 131072 - 3),
                                               (1000, 64, 0), (33, 256, 2**31 - 33)])
def test_tables(device, scaling, rows, rotary, first):
    if scaling.get("scaling") == "ntk" and rotary == 2:
        pytest.skip("one pair has no such scaling")
    base, amplitude = 500000.0, 1.25
    cos, sin = (torch.full((rows, rotary // 2), 9.0, device="cuda:0") for _ in range(2))
    names = dict(original="original_length")
    hx.rope_tables(cos, sin, base=base, first_position=first, amplitude=amplitude,
                   **{names.get(k, k): v for k, v in scaling.items()})
    want = ref.tables(rows, rotary, base, first, **scaling)
    # One rounding to fp32, and angles whose 64-bit products are off by 2^-53 of
    # themselves: up to a few 2^-53 of the last position on either side.
    tol = 2.0 ** -50 * (first + rows) + 2.0 ** -40
    for got, exact in zip((cos, sin), want):
        exact = exact * amplitude
        assert (np.abs(host(got) - exact) <= 2.0 ** -24 * np.abs(exact) + tol).all()


def wide_frequencies(rotary, base, scaling="none", factor=1.0, original_length=0):
    wide = np.longdouble
    i = np.arange(rotary // 2, dtype=wide)
    f = wide(base) ** (-2 * i / rotary)
    if scaling == "linear":
        return f / factor
    if scaling == "ntk":
        return f * wide(factor) ** (-2 * i / (rotary - 2))
    if scaling == "ramp":
        def pair(turns):
            return rotary * math.log(original_length / (2 * math.pi * turns)) / (2 * math.log(base))
        a, b = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rotary - 1)
        w = np.clip((i - a) / max(b - a, 0.001), 0, 1)
        return (1 - w) * f + w * f / factor
    if scaling == "bands":
        w = np.clip((original_length * f / (2 * np.arccos(wide(-1))) - 1) / 3, 0, 1)
        return (1 - w) * f / factor + w * f
    return f


@pytest.mark.parametrize("scaling", [
    dict(), dict(scaling="linear", factor=3.0), dict(scaling="ntk", factor=7.0),
    dict(scaling="ramp", factor=5.0, original_length=4096), dict(scaling="bands", factor=7.0, original_length=8192)])
@pytest.mark.parametrize("rotary", [4, 64, 128, 250])
@pytest.mark.parametrize("base", [1.5, 10000.0, 1e6])
def test_tables_against_wider_numbers(device, scaling, rotary, base):
    """Against angles of 64-bit mantissas (off by position * 2^-60 at most): one rounding,
    and angles that are off by position * 2^-50 (bands: 2^-48)."""
    if np.finfo(np.longdouble).nmant < 63:
        pytest.skip("no wider numbers here")
    f = wide_frequencies(rotary, base, **scaling)
    share = 2.0 ** -48 if scaling.get("scaling") == "bands" else 2.0 ** -50
    for last in (1, 2**17, 2**20, 2**24, 2**31):
        first = max(last - 40, 0)
        cos, sin = (torch.empty(last - first, rotary // 2, device="cuda:0") for _ in range(2))
        hx.rope_tables(cos, sin, base=base, first_position=first, **scaling)
        angles = np.arange(first, last, dtype=np.longdouble)[:, None] * f
        for got, exact in zip((cos, sin), (np.cos(angles), np.sin(angles))):
            off = np.abs(host(got) - exact)
            # (Rounded to the nearest: half a step of what lies below the next power of two.)
            step = np.exp2(np.floor(np.log2(np.maximum(np.abs(exact), 2.0 ** -126))) - 24)
            assert (off <= step + share * last + 2.0 ** -45).all()


def test_tables_are_what_the_rotation_takes(device):
    """Row r of tables from position p on is row p + r of those from 0 on."""
    whole = [torch.empty(300, 32, device="cuda:0") for _ in range(2)]
    part = [torch.empty(41, 32, device="cuda:0") for _ in range(2)]
    hx.rope_tables(*whole)
    hx.rope_tables(*part, first_position=256)
    for w, p in zip(whole, part):
        assert (w[256:297] - p).abs().max() <= 2.0 ** -24


# ------------------------------------------------------------------ rows ----
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("tokens,vectors,dim,rotary", [
    (1, 1, 2, 2), (1, 32, 128, 128), (7, 5, 128, 64), (65, 3, 96, 48), (300, 40, 80, 80),
    (9, 2, 40, 18), (33, 1, 192, 64), (5, 64, 256, 2), (2049, 1, 64, 8), (4, 6, 10, 10)])
def test_rows(device, layout, tokens, vectors, dim, rotary):
    rng = np.random.default_rng(dim + tokens)
    x = normal(rng, tokens, vectors, dim)
    rows = max(tokens, 50)
    cos, sin = (t.astype(np.float32) for t in ref.tables(rows, rotary))
    pos = rng.integers(0, rows, tokens).astype(np.int32)
    at = (cos[pos][:, None], sin[pos][:, None])
    got = hx.rope_rows(dev(x), dev(cos), dev(sin), positions=dev(pos), layout=layout)
    same_bits(host(got), ref.rotate32(x, *at, layout))
    back = hx.rope_rows(dev(x), dev(cos), dev(sin), positions=dev(pos), layout=layout, inverse=True)
    same_bits(host(back), ref.rotate32(x, *at, layout, inverse=True))
    got = hx.rope_rows(dev(x), dev(cos), dev(sin), layout=layout, rotary_dim=rotary)
    same_bits(host(got), ref.rotate32(x, cos[:tokens, None], sin[:tokens, None], layout))


def test_whole_heads_of_pairs_are_what_rope_gives(device):
    rng = np.random.default_rng(1)
    x, (cos, sin) = normal(rng, 37, 6, 128), ref.tables(64, 128)
    pos = dev(rng.integers(0, 64, 37).astype(np.int32))
    c, s = dev(cos.astype(np.float32)), dev(sin.astype(np.float32))
    same_bits(host(hx.rope_rows(dev(x), c, s, positions=pos)), host(hx.rope(dev(x), c, s, pos)))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_rows_of_a_projection(device, layout, shift):
    """Rows among others, on 16 bytes or not, written into a buffer of other strides
    and in place; what lies beside them stays."""
    rng = np.random.default_rng(shift)
    whole = normal(rng, 21, 9, 96 + 8)
    cos, sin = (t.astype(np.float32) for t in ref.tables(21, 64))
    want = ref.rotate32(whole[:, 2:7, shift:shift + 96], cos[:, None], sin[:, None], layout)
    x = dev(whole)
    out = torch.full((9, 21, 100), 5.0, device="cuda:0")
    view = out.transpose(0, 1)[:, 1:6, shift % 2:shift % 2 + 96]
    hx.rope_rows(x[:, 2:7, shift:shift + 96], dev(cos), dev(sin), view, layout=layout)
    same_bits(host(view), want)
    left = host(out)
    assert (left[0] == 5).all() and (left[6:] == 5).all() and (left[:, :, 97:] == 5).all()
    same_bits(host(x), whole)
    hx.rope_rows(x[:, 2:7, shift:shift + 96], dev(cos), dev(sin),
                 x[:, 2:7, shift:shift + 96], layout=layout)
    whole[:, 2:7, shift:shift + 96] = want
    same_bits(host(x), whole)


def test_positions_outside_the_tables_give_nan(device):
    x = torch.ones(4, 2, 8, device="cuda:0")
    cos, sin = (torch.ones(3, 2, device="cuda:0") for _ in range(2))
    pos = torch.tensor([0, -1, 3, 2], dtype=torch.int32, device="cuda:0")
    y = host(hx.rope_rows(x, cos, sin, positions=pos))
    assert np.isnan(y[1:3, :, :4]).all() and np.isfinite(y[[0, 3]]).all()
    assert (y[:, :, 4:] == 1).all()


@pytest.mark.parametrize("layout", LAYOUTS)
def test_the_inverse_is_the_gradient(device, layout):
    """g . d rotate(x) / dx, by differences of a linear map: (rotate(x + h e) -
    rotate(x - h e)) / 2 h . g for each e."""
    rng = np.random.default_rng(3)
    cos, sin = (dev(t.astype(np.float32)) for t in ref.tables(3, 8))
    g = normal(rng, 3, 1, 12)
    eye = np.eye(36, dtype=np.float32).reshape(36, 3, 1, 12)
    x = normal(rng, 3, 1, 12)
    want = np.empty(36)
    for i in range(36):
        up, down = (host(hx.rope_rows(dev(x + h * eye[i]), cos, sin, layout=layout))
                    for h in (0.5, -0.5))
        want[i] = ((up.astype(np.float64) - down) * g).sum()
    got = host(hx.rope_rows(dev(g), cos, sin, layout=layout, inverse=True)).ravel()
    # Values up to 4 rounded by up to 3 * 2^-24 of themselves, on either side, times
    # g, in 2 terms.
    np.testing.assert_allclose(got, want, atol=2 * 6 * 4 * 2.0 ** -24 * 4)


# ---------------------------------------------------------------- append ----
class Append:
    """A step's rows among a projection's, scattered slots, ragged counts."""

    def __init__(self, dtype, layout, b, t, hq, hkv, d, rotary, seed=0, ragged=False, page=16):
        rng = self.rng = np.random.default_rng(seed + b * 100 + t)
        self.dtype, self.layout, self.page = dtype, layout, page
        self.shape = (b, t, hq, hkv, d)
        self.counts = rng.integers(0, t + 1, b) if ragged else np.full(b, t)
        self.rows = normal(rng, b, t, hq + 2 * hkv, d)
        self.cos, self.sin = (x.astype(np.float32) for x in ref.tables(200 + t, rotary))
        self.starts = rng.integers(0, 200, b).astype(np.int32)
        n = (b * t + page - 1) // page + 3
        self.slots = rng.permutation(n * page)[:b * t].reshape(b, t).astype(np.int64)
        self.kp, self.kbits = pool_of(dtype, rng, n, hkv, page, d)
        self.vp, self.vbits = pool_of(dtype, rng, n, hkv, page, d)

    def want(self, fill=3.0):
        b, t, hq, hkv, d = self.shape
        q, k, v = (np.full((b, h, t, d), fill, np.float32) for h in (hq, hkv, hkv))
        for i in range(b):
            for j in range(self.counts[i]):
                at = self.starts[i] + j
                r = self.rows[i, j]
                turned = ref.rotate32(r[:hq + hkv], self.cos[at], self.sin[at], self.layout)
                q[i, :, j], k[i, :, j], v[i, :, j] = turned[:hq], turned[hq:], r[hq + hkv:]
                page, row = divmod(int(self.slots[i, j]), self.page)
                if 0 <= page < len(self.kbits):
                    self.kbits[page, :, row] = on_pages(self.dtype, k[i, :, j], KS)
                    self.vbits[page, :, row] = on_pages(self.dtype, v[i, :, j], VS)
        return q, k, v

    def views(self, rows):
        hq, hkv = self.shape[2:4]
        x = rows.transpose(1, 2)
        return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]

    def call(self, rows, q, k, v, **other):
        x, y, z = self.views(rows)
        counts = None if (self.counts == self.shape[1]).all() else dev(self.counts.astype(np.int32))
        hx.rope_append(x, y, z, self.kp, self.vp, dev(self.starts), dev(self.slots), dev(self.cos),
                       dev(self.sin), query_out=q, key_out=k, value_out=v, layout=self.layout,
                       token_counts=counts, page_dtype=self.dtype,
                       **(dict(k_scale=KS, v_scale=VS) if self.dtype == "fp8" else {}), **other)

    def check_pages(self):
        np.testing.assert_array_equal(bits_of(self.kp), self.kbits)
        np.testing.assert_array_equal(bits_of(self.vp), self.vbits)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("b,t,hq,hkv,d,rotary,page", [
    (1, 1, 32, 8, 128, 128, 16), (3, 1, 4, 2, 128, 64, 16), (2, 33, 6, 3, 64, 64, 16),
    (5, 7, 5, 1, 80, 40, 16), (2, 9, 2, 1, 18, 6, 5), (64, 2, 8, 8, 32, 32, 16),
    (1, 500, 3, 1, 128, 128, 32)])
def test_append(device, dtype, layout, b, t, hq, hkv, d, rotary, page):
    for ragged in (False, True):
        a = Append(dtype, layout, b, t, hq, hkv, d, rotary, ragged=ragged, page=page)
        out = [torch.full((b, h, t, d), 3.0, device="cuda:0") for h in (hq, hkv, hkv)]
        a.call(dev(a.rows), *out)
        for got, want in zip(out, a.want()):
            same_bits(host(got), want)
        a.check_pages()


def test_append_without_row_outputs_and_out_of_pool_slots(device):
    a = Append("bf16", "halves", 4, 5, 2, 2, 64, 64, ragged=True)
    a.slots[0, 0], a.slots[1, 2], a.slots[3, 4] = -1, a.kbits.shape[0] * 16, 2**40
    x, k, v = a.views(dev(a.rows))
    hx.rope_append(None, k, v, a.kp, a.vp, dev(a.starts), dev(a.slots), dev(a.cos), dev(a.sin),
                   layout="halves", token_counts=dev(a.counts.astype(np.int32)), page_dtype="bf16")
    a.want()
    a.check_pages()


def test_append_in_place(device):
    """Every output is its own input, inside one projection's output."""
    a = Append("f32", "halves", 3, 6, 4, 2, 64, 32)
    rows = dev(a.rows)
    a.call(rows, *a.views(rows))
    for got, want in zip(a.views(rows), a.want()):
        same_bits(host(got), want)
    a.check_pages()


def test_append_of_counts_past_the_ends(device):
    a = Append("f32", "pairs", 4, 3, 2, 1, 8, 8)
    a.counts = np.array([3, 0, 2, 3])
    out = [torch.full((4, h, 3, 8), 3.0, device="cuda:0") for h in (2, 1, 1)]
    x, k, v = a.views(dev(a.rows))
    hx.rope_append(x, k, v, a.kp, a.vp, dev(a.starts), dev(a.slots), dev(a.cos), dev(a.sin),
                   query_out=out[0], key_out=out[1], value_out=out[2],
                   token_counts=torch.tensor([9, -5, 2, 3], dtype=torch.int32, device="cuda:0"))
    for got, want in zip(out, a.want()):
        same_bits(host(got), want)
    a.check_pages()


def test_positions_outside_the_tables_reach_only_their_rows(device):
    a = Append("bf16", "pairs", 3, 2, 2, 1, 16, 8)
    a.starts[:] = [-1, 201, 5]  # tables of 202 rows
    out = [torch.full((3, h, 2, 16), 3.0, device="cuda:0") for h in (2, 1, 1)]
    a.call(dev(a.rows), *out)
    q = host(out[0])
    assert np.isnan(q[0, :, 0, :8]).all() and np.isnan(q[1, :, 1, :8]).all()
    assert np.isfinite(q[:, :, :, 8:]).all() and np.isfinite(q[[0, 1], :, [1, 0]]).all()
    assert np.isfinite(q[2]).all() and np.isfinite(host(out[2])).all()
    held = a.kp.view(torch.bfloat16).float()
    for b, t in ((0, 0), (1, 1)):
        page, row = divmod(int(a.slots[b, t]), 16)
        assert torch.isnan(held[page, :, row, :8]).all()
        assert torch.isfinite(held[page, :, row, 8:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("latent", [256, 512])
@pytest.mark.parametrize("b,t,hq,ragged", [(1, 1, 16, False), (3, 5, 3, True), (2, 70, 1, True)])
def test_latent_append(device, dtype, latent, b, t, hq, ragged):
    rng = np.random.default_rng(latent + t)
    counts = rng.integers(0, t + 1, b) if ragged else np.full(b, t)
    lat, down, q = normal(rng, b, t, latent), normal(rng, b, t, 100), normal(rng, b, t, hq, 192)
    cos, sin = (x.astype(np.float32) for x in ref.tables(100 + t, 64))
    starts = rng.integers(0, 100, b).astype(np.int32)
    n = (b * t + 15) // 16 + 2
    slots = rng.permutation(n * 16)[:b * t].reshape(b, t).astype(np.int64)
    pool, bits = pool_of(dtype, rng, n, 16, latent + 64)
    whole = torch.full((b, hq, t, latent + 64), 3.0, device="cuda:0")
    hx.latent_append(dev(lat), dev(down)[..., 36:], pool, dev(starts), dev(slots), dev(cos), dev(sin),
                     query=dev(q).transpose(1, 2)[..., 128:], query_out=whole[..., latent:],
                     token_counts=dev(counts.astype(np.int32)) if ragged else None,
                     page_dtype=dtype, **(dict(page_scale=KS) if dtype == "fp8" else {}))
    want = np.full((b, hq, t, latent + 64), 3.0, np.float32)
    for i in range(b):
        for j in range(counts[i]):
            c, s = cos[starts[i] + j], sin[starts[i] + j]
            want[i, :, j, latent:] = ref.rotate32(q[i, j, :, 128:], c, s, "pairs")
            row = np.concatenate([lat[i, j], ref.rotate32(down[i, j, 36:], c, s, "pairs")])
            bits[slots[i, j] // 16, slots[i, j] % 16] = on_pages(dtype, row, KS)
    same_bits(host(whole), want)
    np.testing.assert_array_equal(bits_of(pool), bits)


# ------------------------------------------------------------ DecodeBatch ----
@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_of_a_batch_are_the_calls_they_replace(device, dtype):
    """Decode and chunk steps with rope_append_layer against rope_rows, append_layer
    and the same attention: every output and every page equal."""
    L, hq, hkv, d = 2, 8, 2, 128
    rng = np.random.default_rng(7)
    cos, sin = (dev(x.astype(np.float32)) for x in ref.tables(256, 64))
    caches, batches = [], []
    for _ in range(2):
        scale = dict(k_scale=KS, v_scale=VS) if dtype == "fp8" else {}
        cache = hx.PagedKvCache(L, hkv, d, 16, 64, page_dtype=dtype, **scale)
        seqs = []
        for n in (5, 16, 40):
            s = cache.create_sequence()
            x = [dev(np.random.default_rng(n + i).standard_normal((hkv, n, d), dtype=np.float32))
                 for i in range(2 * L)]
            cache.append_layer_major(s, x[:L], x[L:])
            seqs.append(s)
        caches.append((cache, seqs))
        batches.append(hx.DecodeBatch(cache, seqs, hq, 256))
    one, two = batches
    lengths = np.array([5, 16, 40])
    for step in (1, 6, 1, 1, 70):
        for batch in batches:
            batch.prepare() if step == 1 else batch.prepare_chunk(step)
        for layer in range(L):
            rows = dev(normal(rng, 3, step, hq + 2 * hkv, d)).transpose(1, 2)
            q, k, v = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:]
            qo, ko, vo = (torch.empty(x.shape, device="cuda:0") for x in (q, k, v))
            one.rope_append_layer(layer, q, k, v, cos, sin, qo, ko, vo, layout="halves")
            got = torch.empty_like(qo)
            pos = torch.from_numpy((lengths[:, None] + np.arange(step)).astype(np.int32)).to("cuda:0")
            turned = []
            for x in (q, k):
                flat = x.transpose(1, 2).reshape(3 * step, x.shape[1], d).contiguous()
                y = hx.rope_rows(flat, cos, sin, positions=pos.flatten(), layout="halves")
                turned.append(y.view(3, step, x.shape[1], d).transpose(1, 2).contiguous())
            want = torch.empty_like(got)
            v = v.contiguous()
            two.append_layer(layer, turned[1], v)
            if step == 1:
                one.attention_layer(layer, qo, ko, vo, got)
                two.attention_layer(layer, turned[0], turned[1], v, want)
            else:
                one.prefill_layer(layer, qo, ko, vo, got)
                two.prefill_layer(layer, turned[0], turned[1], v, want)
            assert torch.equal(qo, turned[0]) and torch.equal(ko, turned[1])
            assert torch.equal(vo, v) and torch.equal(got, want)
        lengths += step
    for layer in range(L):
        for (c1, s1), (c2, s2) in [caches]:
            for x, y in zip(s1, s2):
                for mine, other in zip(c1.retrieve_layer(x, layer), c2.retrieve_layer(y, layer)):
                    assert torch.equal(mine, other)
    with pytest.raises(hx.HelixError) as e:
        one.rope_append_layer(L, q, k, v, cos, sin, qo)
    assert e.value.status == hx.OUT_OF_RANGE
    for batch in batches:
        batch.close()
    for cache, _ in caches:
        cache.close()


def test_a_tree_step_refuses_the_call(device):
    cache = hx.PagedKvCache(1, 2, 128, 16, 16)
    batch = hx.DecodeBatch(cache, [cache.create_sequence()], 2, 64)
    x = torch.zeros(1, 2, 3, 128, device="cuda:0")
    cos, sin = (torch.ones(64, 64, device="cuda:0") for _ in range(2))
    with pytest.raises(hx.HelixError):
        batch.rope_append_layer(0, x, x.clone(), x.clone(), cos, sin, x)
    batch.prepare_chunk(3)
    batch.prepare_tree(3)
    with pytest.raises(hx.HelixError) as e:
        batch.rope_append_layer(0, x, x.clone(), x.clone(), cos, sin, x)
    assert "tree step" in str(e.value)
    batch.close()
    cache.close()


def test_a_step_refuses_rows_in_its_own_memory(device):
    """Rows and tables in the cache's pages (of any layer), outputs on the step's lengths
    or slots."""
    lib = hx.load()
    cache = hx.PagedKvCache(2, 2, 128, 16, 16)
    batch = hx.DecodeBatch(cache, [cache.create_sequence()], 4, 64)
    batch.prepare()
    x = torch.zeros(3, 1, 4, 1, 128, device="cuda:0")
    out = torch.zeros_like(x)
    cos, sin = (torch.ones(64, 64, device="cuda:0") for _ in range(2))
    tables, lengths, slots = (ctypes.c_void_p() for _ in range(3))
    hx.check(lib.helix_decode_batch_tables(batch._h, *(ctypes.byref(p) for p in (tables, lengths, slots)),
                                           None, None))
    good = [x[0].data_ptr(), x[1].data_ptr(), x[2].data_ptr(), out[0].data_ptr(), out[1].data_ptr(),
            out[2].data_ptr(), cos.data_ptr(), sin.data_ptr()]

    def call(rows):
        args = [a for p in rows[:6] for a in (p, None)]
        return lib.helix_decode_batch_rope_append_layer(batch._h, 0, *args, *rows[6:], 64, 128, 0, None)

    assert call(good) == 0
    torch.cuda.synchronize()
    before = [[host(p) for p in cache.layer_pools(layer)] for layer in range(2)]
    for i in range(8):
        inside = [p for layer in range(2) for p in cache.layer_pool_pointers(layer)]
        for at in inside + ([lengths.value, slots.value] if 3 <= i < 6 else []):
            assert call(good[:i] + [at] + good[i + 1:]) == hx.INVALID_ARGUMENT
            assert b"alias" in lib.helix_last_error() or b"pools" in lib.helix_last_error()
    for layer in range(2):
        for p, q in zip(before[layer], cache.layer_pools(layer)):
            same_bits(p, host(q))  # (pages that hold nothing yet hold anything)
    batch.close()
    cache.close()


# ------------------------------------------------------- streams, capture ----
def test_other_streams_and_replays(device):
    """Captured on a stream of its own and replayed with other contents, against
    eager calls."""
    a = Append("bf16", "halves", 2, 3, 4, 2, 64, 64)
    rows, starts, slots = dev(a.rows), dev(a.starts), dev(a.slots)
    cos, sin = dev(a.cos), dev(a.sin)
    out = [torch.zeros(2, h, 3, 64, device="cuda:0") for h in (4, 2, 2)]

    def call(kp, vp, to):
        hx.rope_append(*a.views(rows), kp, vp, starts, slots, cos, sin, query_out=to[0],
                       key_out=to[1], value_out=to[2], layout="halves", page_dtype="bf16")

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call(a.kp, a.vp, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call(a.kp, a.vp, out)
    for i in range(3):
        rows.copy_(dev(normal(a.rng, *a.rows.shape)))
        starts.add_(i)
        slots.copy_(slots.roll(1, 1))
        kp, vp = a.kp.clone(), a.vp.clone()
        torch.cuda.synchronize()
        graph.replay()
        want = [torch.zeros_like(x) for x in out]
        torch.cuda.synchronize()
        call(kp, vp, want)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))
        assert torch.equal(a.kp, kp) and torch.equal(a.vp, vp)
