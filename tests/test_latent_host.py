"""What the entry points of rotary rows and of the latent cache refuse before any
launch, without a GPU: sizes, strides, rows that share memory, workspaces."""

import ctypes

import pytest
import torch

import helix_runtime_amd as hx

MB = 1 << 20


def strides(*s):
    return (ctypes.c_size_t * 3)(*s) if s else None


def refused(lib, rc, status, text=b""):
    assert rc == status, (rc, lib.helix_last_error())
    assert lib.helix_last_error() and text in lib.helix_last_error()


def tables(lib, cos=MB, sin=2 * MB, rows=10, first=0, rotary=64, base=1e4, scaling=0, factor=1.0,
           original=0.0, low=1.0, high=32.0, amplitude=1.0):
    return lib.helix_rope_tables(cos, sin, rows, first, rotary, base, scaling, factor, original, low,
                                 high, amplitude, None)


@pytest.mark.parametrize("bad,status", [
    (dict(rotary=0), hx.INVALID_ARGUMENT), (dict(rotary=7), hx.INVALID_ARGUMENT),
    (dict(base=1.0), hx.INVALID_ARGUMENT), (dict(base=float("inf")), hx.INVALID_ARGUMENT),
    (dict(base=float("nan")), hx.INVALID_ARGUMENT), (dict(scaling=5), hx.INVALID_ARGUMENT),
    (dict(scaling=-1), hx.INVALID_ARGUMENT), (dict(factor=0.5), hx.INVALID_ARGUMENT),
    (dict(factor=float("nan")), hx.INVALID_ARGUMENT), (dict(amplitude=float("inf")), hx.INVALID_ARGUMENT),
    (dict(scaling=2, rotary=2), hx.INVALID_ARGUMENT), (dict(scaling=3), hx.INVALID_ARGUMENT),
    (dict(scaling=3, original=100.0, low=2.0, high=2.0), hx.INVALID_ARGUMENT),
    (dict(scaling=4, original=100.0, low=0.0), hx.INVALID_ARGUMENT),
    (dict(scaling=4, original=100.0, high=float("nan")), hx.INVALID_ARGUMENT),
    (dict(first=2**31), hx.OUT_OF_RANGE), (dict(rows=2**32), hx.OUT_OF_RANGE),
    (dict(rows=2**31 - 5, first=6), hx.OUT_OF_RANGE), (dict(cos=None), hx.INVALID_ARGUMENT),
    (dict(sin=MB + 64), hx.INVALID_ARGUMENT)])
def test_tables_refusals(bad, status):
    lib = hx.load()
    refused(lib, tables(lib, **bad), status)


def rows(lib, x=MB, xs=None, y=8 * MB, ys=None, tokens=4, vectors=3, dim=128, rotary=64, layout=0,
         cos=16 * MB, sin=17 * MB, table=10, pos=18 * MB):
    return lib.helix_rope_rows(x, xs, y, ys, tokens, vectors, dim, rotary, layout, 0, cos, sin, table,
                               pos, None)


@pytest.mark.parametrize("bad,status", [
    (dict(dim=0), hx.INVALID_ARGUMENT), (dict(dim=127), hx.INVALID_ARGUMENT),
    (dict(rotary=0), hx.INVALID_ARGUMENT), (dict(rotary=63), hx.INVALID_ARGUMENT),
    (dict(rotary=130), hx.INVALID_ARGUMENT), (dict(layout=2), hx.INVALID_ARGUMENT),
    (dict(table=0), hx.INVALID_ARGUMENT), (dict(x=None), hx.INVALID_ARGUMENT),
    (dict(cos=None), hx.INVALID_ARGUMENT), (dict(tokens=2**31), hx.INVALID_ARGUMENT),
    (dict(tokens=2**26, vectors=100, y=1 << 50, cos=1 << 51, sin=1 << 52), hx.OUT_OF_RANGE),
    (dict(y=MB + 512), hx.INVALID_ARGUMENT),                     # inside the input
    (dict(ys=strides(384, 100, 0)), hx.INVALID_ARGUMENT),        # rows into each other
    (dict(ys=strides(0, 128, 0)), hx.INVALID_ARGUMENT),
    (dict(xs=strides(2**62, 128, 0)), hx.INVALID_ARGUMENT),
    (dict(y=MB, ys=strides(384, 128, 0), xs=strides(500, 128, 0)), hx.INVALID_ARGUMENT),
    (dict(y=16 * MB + 256), hx.INVALID_ARGUMENT)])               # inside the tables
def test_rows_refusals(bad, status):
    lib = hx.load()
    refused(lib, rows(lib, **bad), status)


def test_rows_of_nothing_is_no_call():
    lib = hx.load()
    assert rows(lib, tokens=0) == 0 and rows(lib, vectors=0) == 0 and tables(lib, rows=0) == 0


# One projection's output [batch, tokens, 48, 128] at MB, as its heads lie in it.
FUSED = (10 * 48 * 128, 128, 48 * 128)


def append(lib, q=MB, k=MB + 32 * 512, v=MB + 40 * 512, qs=FUSED, ks=FUSED, vs=FUSED, qo=64 * MB,
           qos=None, ko=None, vo=None, kos=None, batch=2, hq=32, hkv=8, tokens=10, dim=128,
           kp=128 * MB, vp=256 * MB, blocks=100, page=16, slots=512 * MB, starts=513 * MB, cos=514 * MB,
           sin=515 * MB, table=10, rotary=128, layout=1, dtype=1, scale=1.0, launch=False):
    if not launch:
        kp = kp if kp is not None else None
    s = lambda x: strides(*x) if x else None  # noqa: E731
    return lib.helix_paged_rope_append(q, s(qs), k, s(ks), v, s(vs), qo, s(qos), ko, s(kos), vo, None,
                                       batch, hq, hkv, tokens, dim, kp, vp, blocks, page, slots,
                                       starts, None, cos, sin, table, rotary, layout, dtype, scale,
                                       scale, None)


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=3), b"page dtype"), (dict(dtype=2, scale=0.0), b"scales"),
    (dict(blocks=0), b"block count"), (dict(blocks=2**32), b"block count"),
    (dict(page=0), b"page size"), (dict(hkv=0), b"range"), (dict(dim=7), b"even"),
    (dict(rotary=256), b"rotary"), (dict(layout=9), b"layout"), (dict(table=0), b"tables"),
    (dict(k=None), b"non-null"), (dict(qo=None), b"query with query_out"),
    (dict(slots=None), b"non-null"), (dict(vp=128 * MB + 4096), b"must not overlap"),
    (dict(kp=MB), b"rows must not lie in the pools"), (dict(kp=64 * MB), b"rows must not lie"),
    (dict(qo=MB + 512, qos=FUSED), b"share elements"),          # onto the next heads
    (dict(qo=MB + 256, qos=FUSED), b"share elements"),
    (dict(ko=64 * MB), b"share elements"),                       # onto the queries' output
    (dict(ko=MB + 40 * 512, kos=FUSED), b"share elements"),      # keys onto the values
    (dict(qo=64 * MB, qos=(FUSED[0], 100, FUSED[2])), b"share elements"),
    (dict(qo=64 * MB, qos=(0, 128, FUSED[2])), b"share elements"),
    (dict(qo=514 * MB), b"alias the tables"), (dict(qs=(2**41, 128, 6144)), b"strides")])
def test_append_refusals(bad, text):
    lib = hx.load()
    refused(lib, append(lib, **bad), hx.INVALID_ARGUMENT, text)


def test_append_takes_its_inputs_as_outputs():
    """Rows of one projection's output, each written onto itself, are no overlap (the
    call is refused for what comes after)."""
    lib = hx.load()
    refused(lib, append(lib, qo=MB, qos=FUSED, ko=MB + 32 * 512, kos=FUSED, slots=None),
            hx.INVALID_ARGUMENT, b"non-null")
    assert append(lib, batch=0) == 0 and append(lib, tokens=0) == 0


def latent_append(lib, latent=512, page=16, rows_at=MB, rope=2 * MB, q=4 * MB, qs=None, qo=16 * MB,
                  qos=(16 * 10 * 576, 10 * 576, 576), pages=64 * MB, blocks=100, dtype=0, scale=1.0,
                  batch=2, table=10, slots=512 * MB):
    s = lambda x: strides(*x) if x else None  # noqa: E731
    return lib.helix_paged_latent_append(rows_at, None, rope, None, q, s(qs), qo, s(qos), batch, 16,
                                         10, latent, pages, blocks, page, slots, 513 * MB, None,
                                         514 * MB, 515 * MB, table, 0, dtype, scale, None)


@pytest.mark.parametrize("bad,status", [
    (dict(latent=128), hx.UNSUPPORTED), (dict(page=32), hx.UNSUPPORTED),
    (dict(dtype=2, scale=-1.0), hx.INVALID_ARGUMENT), (dict(blocks=0), hx.INVALID_ARGUMENT),
    (dict(pages=None), hx.INVALID_ARGUMENT), (dict(q=None), hx.INVALID_ARGUMENT),
    (dict(slots=None), hx.INVALID_ARGUMENT), (dict(table=0), hx.INVALID_ARGUMENT),
    (dict(pages=MB), hx.INVALID_ARGUMENT), (dict(qo=64 * MB), hx.INVALID_ARGUMENT),
    (dict(qo=MB), hx.INVALID_ARGUMENT), (dict(qos=(16 * 640, 640, 60)), hx.INVALID_ARGUMENT)])
def test_latent_append_refusals(bad, status):
    lib = hx.load()
    refused(lib, latent_append(lib, **bad), status)
    assert latent_append(lib, batch=0) == 0


def latent(lib, q=MB, qs=None, batch=2, hq=16, tokens=1, n=512, pages=8 * MB, blocks=100, page=16,
           tables_at=64 * MB, width=8, lengths=65 * MB, out=66 * MB, os=None, scale=0.1,
           workspace=128 * MB, size=1 << 30, dtype=0, page_scale=1.0):
    return lib.helix_paged_latent_attention(q, qs, batch, hq, tokens, n, pages, blocks, page, tables_at,
                                            width, lengths, None, out, os, scale, workspace, size,
                                            dtype, page_scale, None)


@pytest.mark.parametrize("bad,status", [
    (dict(n=384), hx.UNSUPPORTED), (dict(page=32), hx.UNSUPPORTED),
    (dict(batch=2**40), hx.INVALID_ARGUMENT), (dict(hq=2**20), hx.INVALID_ARGUMENT),
    (dict(tokens=2**30), hx.INVALID_ARGUMENT), (dict(blocks=0), hx.INVALID_ARGUMENT),
    (dict(width=0), hx.INVALID_ARGUMENT), (dict(width=2**27), hx.INVALID_ARGUMENT),
    (dict(scale=float("nan")), hx.INVALID_ARGUMENT), (dict(q=None), hx.INVALID_ARGUMENT),
    (dict(q=MB + 8), hx.INVALID_ARGUMENT), (dict(pages=8 * MB + 4), hx.INVALID_ARGUMENT),
    (dict(qs=strides(578 * 16, 578, 578)), hx.INVALID_ARGUMENT),
    (dict(os=strides(0, 512, 512)), hx.INVALID_ARGUMENT),
    (dict(out=MB), hx.INVALID_ARGUMENT), (dict(out=8 * MB), hx.INVALID_ARGUMENT),
    (dict(out=128 * MB), hx.INVALID_ARGUMENT), (dict(workspace=None), hx.INVALID_ARGUMENT),
    (dict(workspace=128 * MB + 4), hx.INVALID_ARGUMENT), (dict(size=0), hx.INVALID_ARGUMENT),
    (dict(dtype=2, page_scale=float("inf")), hx.INVALID_ARGUMENT)])
def test_latent_attention_refusals(bad, status):
    lib = hx.load()
    refused(lib, latent(lib, **bad), status)


def prefill(lib, q=MB, qs=None, k=16 * MB, r=32 * MB, v=48 * MB, vs=None, batch=2, heads=3, tokens=10,
            keys=20, out=64 * MB, os=None, scale=0.1, workspace=128 * MB, size=1 << 34):
    return lib.helix_latent_prefill_attention(q, qs, k, None, r, None, v, vs, batch, heads, tokens, keys,
                                              None, None, out, os, scale, workspace, size, None)


@pytest.mark.parametrize("bad,status", [
    (dict(batch=2**30), hx.INVALID_ARGUMENT), (dict(heads=2**20), hx.INVALID_ARGUMENT),
    (dict(tokens=2**25), hx.INVALID_ARGUMENT), (dict(keys=2**25), hx.INVALID_ARGUMENT),
    (dict(batch=2**16, heads=2**10, keys=2**10), hx.INVALID_ARGUMENT),
    (dict(scale=float("inf")), hx.INVALID_ARGUMENT), (dict(q=None), hx.INVALID_ARGUMENT),
    (dict(r=None), hx.INVALID_ARGUMENT), (dict(v=48 * MB + 4), hx.INVALID_ARGUMENT),
    (dict(vs=strides(3 * 20 * 129, 20 * 129, 129)), hx.INVALID_ARGUMENT),
    (dict(out=48 * MB), hx.INVALID_ARGUMENT), (dict(os=strides(3840, 0, 128)), hx.INVALID_ARGUMENT),
    (dict(workspace=None), hx.INVALID_ARGUMENT), (dict(size=0), hx.INVALID_ARGUMENT),
    (dict(workspace=64 * MB), hx.INVALID_ARGUMENT)])
def test_latent_prefill_refusals(bad, status):
    lib = hx.load()
    refused(lib, prefill(lib, **bad), status)


def test_latent_indexes_apart():
    """Tables and lengths in the output or the workspace."""
    lib = hx.load()
    for bad in (dict(tables_at=69206016 + 64), dict(lengths=69206016 + 8),
                dict(tables_at=134217728 + 64), dict(lengths=134217728 + (1 << 20))):
        refused(lib, latent(lib, **bad), hx.INVALID_ARGUMENT)
    for at in (64 * MB + 16, 128 * MB + 16):
        out = 64 * MB
        for index in ((at, None), (None, at)):
            refused(lib, lib.helix_latent_prefill_attention(
                MB, None, 16 * MB, None, 32 * MB, None, 48 * MB, None, 2, 3, 10, 20, *index, out, None,
                0.1, 128 * MB, 16 << 30, None), hx.INVALID_ARGUMENT)


def test_latent_prefill_rows_far_apart():
    """Rows of keys 2^25 numbers apart are refused; a single one has no next."""
    far = dict(v=2**50, vs=strides(2**26, 2**26, 2**25), batch=1, heads=1, keys=2)
    refused(hx.load(), prefill(hx.load(), **far), hx.UNSUPPORTED)
    far = dict(far, vs=strides(2**26, 2**26, 2**25), keys=1, tokens=0)
    assert prefill(hx.load(), **far) == 0


def test_attention_of_nothing_is_no_call():
    lib = hx.load()
    assert latent(lib, batch=0) == 0 and latent(lib, hq=0) == 0 and latent(lib, tokens=0) == 0
    assert prefill(lib, batch=0) == 0 and prefill(lib, heads=0) == 0 and prefill(lib, tokens=0) == 0


def test_workspace_sizes():
    assert 0 < hx.latent_workspace_bytes(64, 128, 1) < 1 << 30
    assert hx.latent_workspace_bytes(1, 16, 1, 256) > 0
    assert hx.latent_prefill_workspace_bytes(4, 32, 512, 4096) > 0
    for call in (lambda: hx.latent_workspace_bytes(1, 16, 1, 500),
                 lambda: hx.latent_prefill_workspace_bytes(2**30, 1, 1, 1)):
        with pytest.raises(hx.HelixError):
            call()


@pytest.mark.parametrize("at", [8 * MB - 12, 8 * MB, 8 * MB + 6140])
def test_rows_positions_apart(at):
    """Positions (four) in the output (4 x 3 x 128 numbers)."""
    lib = hx.load()
    refused(lib, rows(lib, pos=at), hx.INVALID_ARGUMENT, b"positions")


# What rope_append writes: query rows, key rows, value rows and both pools.
@pytest.mark.parametrize("at", [64 * MB + 4096, 80 * MB + 128, 90 * MB + 128, 128 * MB + 512, 256 * MB + 512])
@pytest.mark.parametrize("what", [("slots", b"slots"), ("starts", b"starts"), ("counts", b"counts"),
                                  ("cos", b"tables"), ("sin", b"tables")])
def test_append_indexes_apart(what, at):
    lib = hx.load()
    index = {"slots": 512 * MB, "starts": 513 * MB, "counts": 516 * MB, "cos": 514 * MB, "sin": 515 * MB,
             what[0]: at}
    rc = lib.helix_paged_rope_append(
        MB, None, 16 * MB, None, 32 * MB, None, 64 * MB, None, 80 * MB, None, 90 * MB, None, 2, 32, 8, 10,
        128, 128 * MB, 256 * MB, 100, 16, index["slots"], index["starts"], index["counts"], index["cos"],
        index["sin"], 10, 128, 1, 1, 1.0, 1.0, None)
    refused(lib, rc, hx.INVALID_ARGUMENT, what[1])


# And latent_append: query rows, and the pages (100 of 16 x 576 numbers).
@pytest.mark.parametrize("at", [16 * MB + 4096, 64 * MB + 100 * 16 * 576 * 4 - 16])
@pytest.mark.parametrize("what", [("slots", b"slots"), ("starts", b"starts"), ("counts", b"counts"),
                                  ("cos", b"tables"), ("sin", b"tables")])
def test_latent_append_indexes_apart(what, at):
    lib = hx.load()
    index = {"slots": 512 * MB, "starts": 513 * MB, "counts": 516 * MB, "cos": 514 * MB, "sin": 515 * MB,
             what[0]: at}
    rc = lib.helix_paged_latent_append(
        MB, None, 2 * MB, None, 4 * MB, None, 16 * MB, strides(16 * 10 * 576, 10 * 576, 576), 2, 16, 10, 512,
        64 * MB, 100, 16, index["slots"], index["starts"], index["counts"], index["cos"], index["sin"], 10,
        0, 0, 1.0, None)
    refused(lib, rc, hx.INVALID_ARGUMENT, what[1])


# ---------------------------------------------------------- Python checks ----
def wrong(call, text):
    with pytest.raises(hx.HelixError) as e:
        call()
    assert e.value.status == hx.INVALID_ARGUMENT and text in str(e.value)


def test_python_checks_of_rotary_rows():
    z = torch.zeros
    cos, sin = z(8, 4), z(8, 4)
    wrong(lambda: hx.rope_tables(cos, z(8, 5)), "sine")
    wrong(lambda: hx.rope_tables(cos.double(), sin), "cosine")
    wrong(lambda: hx.rope_tables(cos, sin, scaling="other"), "scaling")
    wrong(lambda: hx.rope_tables(cos, sin, first_position=-1), "first_position")
    wrong(lambda: hx.rope_tables(cos, sin), "GPU")
    x = z(3, 2, 16)
    wrong(lambda: hx.rope_rows(z(3, 16), cos, sin), "shape")
    wrong(lambda: hx.rope_rows(x.half(), cos, sin), "float32")
    wrong(lambda: hx.rope_rows(z(3, 16, 2).transpose(1, 2), cos, sin), "last dimension")
    wrong(lambda: hx.rope_rows(x, cos, sin, z(3, 2, 15)), "output")
    wrong(lambda: hx.rope_rows(x, cos, sin, rotary_dim=16), "rotary_dim")
    wrong(lambda: hx.rope_rows(x, cos, sin, layout="rows"), "layout")
    wrong(lambda: hx.rope_rows(x, cos, sin, positions=z(3)), "positions")
    wrong(lambda: hx.rope_rows(z(9, 2, 16), cos, sin), "row per token")
    wrong(lambda: hx.rope_rows(x, cos, sin), "GPU")


def test_python_checks_of_appends():
    z, i = torch.zeros, lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    slots = torch.zeros(2, 3, dtype=torch.int64)
    good = dict(query=z(2, 4, 3, 8), keys=z(2, 2, 3, 8), values=z(2, 2, 3, 8), key_pool=z(5, 2, 16, 8),
                value_pool=z(5, 2, 16, 8), starts=i(2), slots=slots, cosine=z(9, 4), sine=z(9, 4),
                query_out=z(2, 4, 3, 8))
    call = lambda **bad: lambda: hx.rope_append(**{**good, **bad})  # noqa: E731
    wrong(call(), "GPU")
    wrong(call(keys=z(2, 3, 8)), "keys")
    wrong(call(query_out=None), "go together")
    wrong(call(values=z(2, 2, 4, 8)), "values")
    wrong(call(key_out=z(2, 2, 3, 7)), "key_out")
    wrong(call(key_pool=z(5, 3, 16, 8)), "pools")
    wrong(call(value_pool=z(6, 2, 16, 8)), "value_pool")
    wrong(call(key_pool=z(5, 2, 16, 8).half()), "key_pool")
    wrong(call(page_dtype="int4"), "page_dtype")
    wrong(call(slots=slots.int()), "slots")
    wrong(call(starts=z(2)), "starts")
    wrong(call(token_counts=i(3)), "token_counts")
    wrong(call(rotary_dim=6), "rotary_dim")
    good = dict(latent=z(2, 3, 256), rope_key=z(2, 3, 64), pool=z(5, 16, 320), starts=i(2), slots=slots,
                cosine=z(9, 32), sine=z(9, 32))
    call = lambda **bad: lambda: hx.latent_append(**{**good, **bad})  # noqa: E731
    wrong(call(), "GPU")
    wrong(call(latent=z(2, 256)), "latent")
    wrong(call(rope_key=z(2, 3, 32)), "rope_key")
    wrong(call(pool=z(5, 16, 300)), "latent + 64")
    wrong(call(pool=z(16, 320)), "pool")
    wrong(call(query=z(2, 4, 3, 64)), "go together")
    wrong(call(query=z(2, 4, 3, 60), query_out=z(2, 4, 3, 64)), "query")
    wrong(call(cosine=z(9, 16), sine=z(9, 16)), "rotary_dim")


def test_python_checks_of_attention():
    z, i = torch.zeros, lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    good = dict(query=z(2, 4, 3, 320), pool=z(5, 16, 320), tables=i(2, 4), lengths=i(2),
                output=z(2, 4, 3, 256), workspace=z(100), scale=0.1)
    call = lambda **bad: lambda: hx.paged_latent_attention(**{**good, **bad})  # noqa: E731
    wrong(call(), "GPU")
    wrong(call(query=z(2, 4, 320)), "query")
    wrong(call(pool=z(5, 16, 576)), "latent + 64")
    wrong(call(output=z(2, 4, 3, 320)), "output")
    wrong(call(tables=i(3, 4)), "tables")
    wrong(call(tables=z(2, 4)), "tables")
    wrong(call(lengths=i(3)), "lengths")
    wrong(call(token_counts=z(2)), "token_counts")
    wrong(call(page_dtype="bf16"), "pool")
    good = dict(query=z(2, 4, 3, 192), key=z(2, 4, 5, 128), rope_key=z(2, 5, 64), value=z(2, 4, 5, 128),
                output=z(2, 4, 3, 128), workspace=z(100), scale=0.1)
    call = lambda **bad: lambda: hx.latent_prefill_attention(**{**good, **bad})  # noqa: E731
    wrong(call(), "GPU")
    wrong(call(query=z(2, 4, 3, 128)), "query")
    wrong(call(key=z(2, 4, 5, 64)), "key")
    wrong(call(rope_key=z(2, 6, 64)), "rope_key")
    wrong(call(value=z(2, 4, 6, 128)), "value")
    wrong(call(key_lengths=i(3)), "key_lengths")
    wrong(call(token_counts=i(3)), "token_counts")
