"""Host side of a tree step, without a GPU: what the entry points refuse before
any launch, and truncation of sequences against a model of the page
bookkeeping."""

import ctypes

import numpy as np
import pytest
import torch

import helix_runtime_amd as hx
import tree_reference as ref


def attention(lib, batch=4, hq=32, hkv=8, nodes=8, dim=128, page=16, physical=100, max_blocks=8,
              dtype=0, ks=1.0, vs=1.0, pointer=None, workspace=None, size=1 << 40):
    p = pointer
    return lib.helix_paged_tree_attention(p, batch, hq, hkv, nodes, dim, p, p, physical, page, p,
                                          max_blocks, p, p, p, p, None, p, workspace, size, dtype,
                                          ks, vs, None)


@pytest.mark.parametrize("bad,status", [
    (dict(dim=64), hx.UNSUPPORTED), (dict(page=32), hx.UNSUPPORTED),
    (dict(nodes=65), hx.UNSUPPORTED), (dict(hq=30), hx.INVALID_ARGUMENT),
    (dict(hkv=0), hx.INVALID_ARGUMENT), (dict(hq=0), hx.INVALID_ARGUMENT),
    (dict(physical=0), hx.INVALID_ARGUMENT), (dict(physical=2**32), hx.INVALID_ARGUMENT),
    (dict(max_blocks=0), hx.INVALID_ARGUMENT), (dict(max_blocks=2**27), hx.INVALID_ARGUMENT),
    (dict(batch=2**40), hx.INVALID_ARGUMENT), (dict(batch=2**63), hx.INVALID_ARGUMENT),
    (dict(dtype=3), hx.INVALID_ARGUMENT), (dict(dtype=2, ks=0.0), hx.INVALID_ARGUMENT),
    (dict(dtype=2, vs=float("nan")), hx.INVALID_ARGUMENT), (dict(), hx.INVALID_ARGUMENT),
    (dict(pointer=4096), hx.INVALID_ARGUMENT),  # every tensor at one address
])
def test_tree_attention_refuses_before_any_launch(bad, status):
    lib = hx.load()
    assert attention(lib, **bad) == status
    assert lib.helix_last_error()


def test_tree_attention_of_nothing_is_no_call():
    lib = hx.load()
    assert attention(lib, batch=0) == 0 and attention(lib, nodes=0) == 0


def test_workspace_sizes():
    assert hx.tree_workspace_bytes(1, 32, 8, 1) > 0
    assert hx.tree_workspace_bytes(64, 32, 8, 64) < 1 << 30
    assert hx.verify_workspace_bytes(64, 64, 128256) > 0
    for call in (lambda: hx.tree_workspace_bytes(1, 32, 8, 65),
                 lambda: hx.verify_workspace_bytes(1, 65, 10)):
        with pytest.raises(hx.HelixError) as e:
            call()
        assert e.value.status == hx.UNSUPPORTED
    with pytest.raises(hx.HelixError):
        hx.tree_workspace_bytes(1, 7, 2, 4)


def verify(lib, batch=2, nodes=4, vocab=100, stride=None, batch_stride=None, draft=None,
           draft_stride=100, pointer=None, size=1 << 30, workspace=None):
    p = pointer
    stride = vocab if stride is None else stride
    return lib.helix_verify_tree(p, 4 * stride if batch_stride is None else batch_stride, stride,
                                 draft, 400, draft_stride, batch, nodes, vocab, p, None, None, p, p,
                                 p, p, p, workspace, size, None)


@pytest.mark.parametrize("bad,status", [
    (dict(nodes=65), hx.UNSUPPORTED), (dict(vocab=0), hx.INVALID_ARGUMENT),
    (dict(vocab=2**31), hx.INVALID_ARGUMENT), (dict(batch=2**21), hx.INVALID_ARGUMENT),
    (dict(), hx.INVALID_ARGUMENT), (dict(pointer=4096, stride=99), hx.INVALID_ARGUMENT),
    (dict(pointer=4096, draft=4096, draft_stride=99), hx.INVALID_ARGUMENT),
    (dict(pointer=4096, batch_stride=2**50), hx.INVALID_ARGUMENT),
    (dict(pointer=4096), hx.INVALID_ARGUMENT),  # no workspace
    (dict(pointer=4096, workspace=4096, size=0), hx.INVALID_ARGUMENT),
    (dict(pointer=4096, workspace=4100), hx.INVALID_ARGUMENT),
])
def test_verify_refuses_before_any_launch(bad, status):
    lib = hx.load()
    assert verify(lib, **bad) == status
    assert lib.helix_last_error()
    assert verify(lib, batch=0) == 0 and verify(lib, nodes=0) == 0


def append(lib, layers=2, stride=None, physical=10, heads=2, page=16, dim=8, batch=1, nodes=4,
           dtype=0, ks=1.0, pointer=None):
    stride = physical * heads * page * dim if stride is None else stride
    p = pointer
    return lib.helix_paged_append_path(p, p, p, p, layers, stride, physical, heads, page, dim, p, p,
                                       p, batch, nodes, dtype, ks, 1.0, None)


@pytest.mark.parametrize("bad", [
    dict(physical=0), dict(heads=0), dict(page=0), dict(dim=0), dict(stride=10),
    dict(layers=40000), dict(dtype=7), dict(dtype=2, ks=-1.0), dict(batch=2**33), dict(),
    dict(nodes=2**33)])
def test_append_path_refuses_before_any_launch(bad):
    lib = hx.load()
    assert append(lib, **bad) == hx.INVALID_ARGUMENT
    assert lib.helix_last_error()
    assert append(lib, batch=0) == 0 and append(lib, nodes=0) == 0 and append(lib, layers=0) == 0


def test_size_overflow_is_out_of_range():
    assert append(hx.load(), physical=2**40, heads=2**20, page=2**10) == hx.OUT_OF_RANGE


def test_decode_batch_entries_refuse_null_handles():
    lib = hx.load()
    assert lib.helix_decode_batch_prepare_tree(None, 4, None) == hx.INVALID_ARGUMENT
    assert lib.helix_decode_batch_tree_layer(None, 0, *[None] * 7) == hx.INVALID_ARGUMENT
    assert lib.helix_decode_batch_commit_path(None, *[None] * 5) == hx.INVALID_ARGUMENT
    assert lib.helix_decode_batch_accept_tree(None, None, 0, 0, None, 0, 0, 1,
                                              *[None] * 11) == hx.INVALID_ARGUMENT
    assert lib.helix_paged_cache_truncate_sequence(None, hx.Sequence(), 0) == hx.INVALID_ARGUMENT
    assert lib.helix_block_manager_truncate(None, hx.Sequence(), 0) == hx.INVALID_ARGUMENT


def tensors(b=2, hq=4, hkv=2, t=3):
    f = torch.zeros
    return dict(query=f(b, hq, t, 128), key_pool=f(4, hkv, 16, 128), value_pool=f(4, hkv, 16, 128),
                tables=f(b, 2, dtype=torch.int32), lengths=f(b, dtype=torch.int32),
                tree_key=f(b, hkv, t, 128), tree_value=f(b, hkv, t, 128),
                parents=f(b, t, dtype=torch.int32), output=f(b, hq, t, 128),
                workspace=f(1 << 20, dtype=torch.uint8))


@pytest.mark.parametrize("name,value", [
    ("query", torch.zeros(2, 4, 3, 128, dtype=torch.float64)),
    ("query", torch.zeros(4, 3, 128)), ("query", torch.zeros(2, 4, 128, 3).transpose(2, 3)),
    ("output", torch.zeros(2, 4, 4, 128)), ("tree_key", torch.zeros(2, 4, 3, 128)),
    ("tree_value", torch.zeros(2, 2, 3, 128, dtype=torch.bfloat16)),
    ("tables", torch.zeros(2, 2, dtype=torch.int64)), ("tables", torch.zeros(3, 2, dtype=torch.int32)),
    ("lengths", torch.zeros(3, dtype=torch.int32)), ("parents", torch.zeros(2, 4, dtype=torch.int32)),
    ("parents", torch.zeros(2, 3, dtype=torch.int64)), ("value_pool", torch.zeros(5, 2, 16, 128)),
    ("key_pool", torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16)),
    ("workspace", torch.zeros(1 << 20, dtype=torch.uint8)[::2]),
    ("node_counts", torch.zeros(1, dtype=torch.int32)), (None, None)])
def test_python_tree_attention_checks_its_tensors(name, value):
    """(None: everything fits, but the tensors are not on a GPU.)"""
    kw = tensors()
    if name is not None:
        kw[name] = value
    with pytest.raises(hx.HelixError) as e:
        hx.paged_tree_attention(**kw)
    assert e.value.status == hx.INVALID_ARGUMENT


@pytest.mark.parametrize("name,value", [
    ("target", torch.zeros(2, 3, 9).double()), ("target", torch.zeros(2, 9, 3).transpose(1, 2)),
    ("draft", torch.zeros(2, 3, 8)), ("tokens", torch.zeros(2, 3)),
    ("uniforms", torch.zeros(2, 3).double()), ("bonus_uniforms", torch.zeros(3)),
    ("path", torch.zeros(2, 4, dtype=torch.int32)), ("next_token", torch.zeros(2)),
    ("accepted", torch.zeros(2, dtype=torch.int64)), (None, None)])
def test_python_verify_checks_its_tensors(name, value):
    i = dict(dtype=torch.int32)
    kw = dict(target=torch.zeros(2, 3, 9), draft=torch.zeros(2, 3, 9), tokens=torch.zeros(2, 3, **i),
              parents=None, uniforms=torch.zeros(2, 3), bonus_uniforms=torch.zeros(2),
              path=torch.zeros(2, 3, **i), accepted=torch.zeros(2, **i),
              next_token=torch.zeros(2, **i), workspace=torch.zeros(1 << 20, dtype=torch.uint8))
    if name is not None:
        kw[name] = value
    with pytest.raises(hx.HelixError) as e:
        hx.verify_tree(**kw)
    assert e.value.status == hx.INVALID_ARGUMENT


@pytest.mark.parametrize("name,value", [
    ("keys", torch.zeros(2, 1, 2, 3, 9)), ("values", torch.zeros(1, 2, 3, 8)),
    ("key_pool", torch.zeros(2, 4, 2, 16, 9)), ("value_pool", torch.zeros(3, 4, 2, 16, 8)),
    ("key_pool", torch.zeros(2, 4, 2, 8, 16).transpose(3, 4)),
    ("slots", torch.zeros(1, 3, dtype=torch.int32)), ("path", torch.zeros(1, 3, dtype=torch.int64)),
    ("accepted", torch.zeros(2, dtype=torch.int32)), (None, None)])
def test_python_append_path_checks_its_tensors(name, value):
    kw = dict(keys=torch.zeros(2, 1, 2, 3, 8), values=torch.zeros(2, 1, 2, 3, 8),
              key_pool=torch.zeros(2, 4, 2, 16, 8), value_pool=torch.zeros(2, 4, 2, 16, 8),
              slots=torch.zeros(1, 3, dtype=torch.int64), path=torch.zeros(1, 3, dtype=torch.int32),
              accepted=torch.zeros(1, dtype=torch.int32))
    if name is not None:
        kw[name] = value
    with pytest.raises(hx.HelixError) as e:
        hx.append_path(**kw)
    assert e.value.status == hx.INVALID_ARGUMENT


@pytest.mark.parametrize("page_dtype,dtype", [
    ("f32", "int32"), ("bf16", "float16"), ("fp8", "bool"), ("fp8", "float8_e5m2"),
    ("fp8", "float8_e4m3fnuz"), ("f32", "bfloat16"), ("f16", "float16")])
def test_pools_must_hold_the_page_types_elements(page_dtype, dtype):
    """An element type of the right width alone would give wrong numbers without
    an error."""
    dtype = getattr(torch, dtype)
    for names in (("key_pool",), ("value_pool",), ("key_pool", "value_pool")):
        a = tensors()
        b = dict(keys=torch.zeros(1, 2, 3, 8), values=torch.zeros(1, 2, 3, 8),
                 slots=torch.zeros(1, 3, dtype=torch.int64),
                 path=torch.zeros(1, 3, dtype=torch.int32),
                 accepted=torch.zeros(1, dtype=torch.int32))
        right = {"f32": torch.float32, "bf16": torch.bfloat16}.get(page_dtype, torch.uint8)
        for name in ("key_pool", "value_pool"):
            a[name] = a[name].to(dtype if name in names else right)
            b[name] = torch.zeros(4, 2, 16, 8).to(dtype if name in names else right)
        for call, kw in ((hx.paged_tree_attention, a), (hx.append_path, b)):
            with pytest.raises(hx.HelixError) as e:
                call(**kw, page_dtype=page_dtype)
            assert e.value.status == hx.INVALID_ARGUMENT
            assert "pool must" in str(e.value) or "page_dtype" in str(e.value)


@pytest.mark.parametrize("page_dtype,dtypes", [
    ("f32", ["float32"]), ("bf16", ["bfloat16", "int16", "uint16"]),
    ("fp8", ["float8_e4m3fn", "uint8", "int8"])])
def test_pools_may_hold_their_bits(page_dtype, dtypes):
    """(What is refused then is that they are not on a GPU.)"""
    for dtype in dtypes:
        a = tensors()
        a.update(key_pool=a["key_pool"].to(getattr(torch, dtype)),
                 value_pool=a["value_pool"].to(getattr(torch, dtype)))
        with pytest.raises(hx.HelixError, match="on a GPU"):
            hx.paged_tree_attention(**a, page_dtype=page_dtype)


def test_prepare_tree_takes_the_current_stream_of_the_caches_device(monkeypatch):
    """As the step's other calls do, whatever device is the current one."""
    class Stream:
        def __init__(self, device=None):
            self.cuda_stream = 100 + (0 if device is None else torch.device(device).index)

    class Library:
        def helix_decode_batch_prepare_tree(self, handle, nodes, stream):
            self.stream = getattr(stream, "value", stream)
            return 0

    lib = Library()
    monkeypatch.setattr(hx, "_lib", lambda: lib)
    monkeypatch.setattr(torch.cuda, "current_stream", Stream)
    batch = hx.DecodeBatch.__new__(hx.DecodeBatch)
    batch._h, batch._cache = 1, type("Cache", (), {"device": 1})()
    try:
        batch.prepare_tree(4)
        assert lib.stream == 101
        batch.prepare_tree(4, stream=Stream("cuda:2"))
        assert lib.stream == 102
    finally:
        batch._h = None


# ------------------------------------------------------------- truncation ----
def test_truncate_frees_pages_in_table_order():
    m = hx.BlockManager(1, 1, 2, 4, 5)
    s = m.create_sequence()
    m.append(s, 18)  # 5 pages
    m.truncate_sequence(s, 5)
    assert m.length(s) == 5 and m.block_table(s) == [0, 1]
    assert m.block_info(1) == (1, 1) and m.block_info(2) == (0, 0)
    st = m.stats()
    assert (st["used_blocks"], st["active_tokens"], st["resident_tokens"]) == (2, 5, 5)
    m.validate()
    other = m.create_sequence()
    m.append(other, 12)
    assert m.block_table(other) == [2, 3, 4]
    m.truncate_sequence(s, 5)  # nothing to drop
    m.truncate_sequence(s, 0)
    assert m.length(s) == 0 and m.block_table(s) == [] and m.contains(s)
    m.append(s, 3)
    assert m.block_table(s) == [0]
    m.validate()


def test_truncate_refusals():
    m = hx.BlockManager(1, 1, 2, 4, 8)
    s = m.create_sequence()
    m.append(s, 10)
    with pytest.raises(hx.HelixError) as e:
        m.truncate_sequence(s, 11)
    assert e.value.status == hx.OUT_OF_RANGE
    f, _ = m.fork_sequence(s, 8)
    with pytest.raises(hx.HelixError) as e:
        m.truncate_sequence(s, 7)  # inside the second page, which the fork shares
    assert e.value.status == hx.INVALID_ARGUMENT
    assert m.length(s) == 10
    m.validate()
    m.truncate_sequence(s, 4)  # whole pages may go
    assert m.block_table(f) == [0, 1] and m.block_info(1) == (1, 4)
    m.truncate_sequence(f, 7)  # its own now
    m.validate()
    m.release_sequence(s)
    with pytest.raises(hx.HelixError):
        m.truncate_sequence(s, 0)
    with pytest.raises(hx.HelixError):
        m.truncate_sequence(hx.Sequence(), 0)


@pytest.mark.parametrize("seed", range(4))
def test_random_programs_with_truncation_keep_every_invariant(seed):
    rng = np.random.default_rng(seed)
    m = hx.BlockManager(1, 2, 4, int(rng.integers(1, 9)), 40)
    lengths = {}
    for _ in range(300):
        op = rng.integers(0, 5)
        live = list(lengths)
        if op == 0 or not live:
            lengths[m.create_sequence()] = 0
            continue
        s = live[rng.integers(len(live))]
        try:
            if op == 1:
                n = int(rng.integers(1, 20))
                m.append(s, n)
                lengths[s] += n
            elif op == 2 and lengths[s]:
                f, _ = m.fork_sequence(s, int(rng.integers(1, lengths[s] + 1)), allow_cow=True)
                lengths[f] = m.length(f)
            elif op == 3:
                n = int(rng.integers(0, lengths[s] + 1))
                m.truncate_sequence(s, n)
                lengths[s] = n
            elif op == 4:
                m.release_sequence(s)
                del lengths[s]
        except hx.HelixError as e:
            assert e.status in (hx.RESOURCE_EXHAUSTED, hx.INVALID_ARGUMENT)
        m.validate()
        assert {s: m.length(s) for s in lengths} == lengths


# ------------------------------------------------ the verification's rule ----
@pytest.mark.parametrize("certain", [False, True])
def test_the_rule_leaves_the_targets_distribution(certain):
    """The plain verification, as the tests of the kernel use it: over many
    random numbers, the first token after the root is distributed as the
    target's row 0 (5 standard deviations of a binomial)."""
    rng = np.random.default_rng(3)
    V, N = 5, 20000
    target = rng.dirichlet(np.ones(V), size=4).astype(np.float32)
    draft = rng.dirichlet(np.ones(V), size=4).astype(np.float32)
    parents = np.array([-1, 0, 0, 1], np.int32)
    seen = np.zeros(V)
    for _ in range(N):
        d0 = draft[0].astype(np.float64)
        tokens = np.array([0, *rng.choice(V, 2, p=d0 / d0.sum()), 0])
        if certain:
            tokens[1:3] = [2, 4]
        path, after = ref.verify(target, None if certain else draft, tokens, parents, 4,
                                 rng.random(4), rng.random())
        seen[tokens[path[1]] if len(path) > 1 else after] += 1
    p = target[0].astype(np.float64)
    assert np.all(np.abs(seen / N - p) < 5 * np.sqrt(p * (1 - p) / N))
