"""MI355X-native paged-KV hot path of helix-runtime.

Python front end over the C ABI in ``include/helix_paged.h``.  The names and
argument meaning follow the reference's C++ interface
(``include/helix/kv_cache/cuda_paged.hpp``, ``include/helix/kv_cache/paged.hpp``,
``include/helix/attention/cuda_paged.hpp``); errors surface as
:class:`HelixError` carrying the reference's error code.  PyTorch is used
only for device memory and streams: every computation runs in the HIP
kernels of ``libhelix_paged.so``.
"""

from __future__ import annotations

import contextlib
import ctypes
import sys
import os
import subprocess

from . import _native
from ._native import (HelixError, Sequence, INVALID_ARGUMENT, OUT_OF_RANGE, UNSUPPORTED,
                      RESOURCE_EXHAUSTED, RUNTIME, INTERNAL, check)

__all__ = [
    "build", "load", "HelixError", "Sequence", "BlockManager", "PagedKvCache", "DecodeBatch",
    "PagedBlockTable", "paged_attention_out", "paged_attention_with_tail_out",
    "paged_decode_attention", "decode_workspace_bytes", "decode_workspace", "append_slots",
    "paged_tree_attention", "tree_workspace_bytes", "tree_workspace", "verify_tree",
    "verify_workspace_bytes", "verify_workspace", "append_path",
    "rope_tables", "rope_rows", "rope_append", "latent_append", "paged_latent_attention",
    "latent_workspace_bytes", "latent_workspace", "latent_prefill_attention",
    "latent_prefill_workspace_bytes", "latent_prefill_workspace",
    "PagedPrefixCache", "PREFIX_INSERTED", "PREFIX_ALREADY_PRESENT", "PREFIX_REJECTED_TOO_LARGE",
    "INVALID_ARGUMENT", "OUT_OF_RANGE", "UNSUPPORTED", "RESOURCE_EXHAUSTED", "RUNTIME", "INTERNAL",
]


def build(jobs: int = 8) -> str:
    """Compile libhelix_paged.so for gfx950 with the in-tree Makefile."""
    subprocess.run(["make", "-s", "-C", _native.HERE, f"-j{jobs}", "libhelix_paged.so"],
                   check=True)
    return _native.LIB_PATH


def load():
    return _native.load()


def _lib():
    return _native.load()


def _ptr(t):
    """Device (or host) address of a tensor, or None."""
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(stream):
    import torch
    if stream is None:
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


def _require_f32(t, name):
    import torch
    if t.dtype != torch.float32 or not t.is_contiguous():
        raise HelixError(INVALID_ARGUMENT, f"{name} must be a contiguous float32 tensor")


def _cfg(layers, kv_heads, head_dimension, block_tokens, physical_blocks):
    return _native.Config(layers, kv_heads, head_dimension, block_tokens, physical_blocks)


# ------------------------------------------------------------------ host ----
class BlockManager:
    """Host page bookkeeping of the paged pool (no device memory)."""

    def __init__(self, layers, kv_heads, head_dimension, block_tokens, physical_blocks):
        h = ctypes.c_void_p()
        cfg = _cfg(layers, kv_heads, head_dimension, block_tokens, physical_blocks)
        check(_lib().helix_block_manager_create(ctypes.byref(cfg), ctypes.byref(h)))
        self._h = h
        self.block_tokens = block_tokens
        self.physical_blocks = physical_blocks

    def __del__(self, _finalizing=sys.is_finalizing):
        if _finalizing():
            return  # the process is exiting; the driver reclaims device memory
        h = getattr(self, "_h", None)
        if h:
            _lib().helix_block_manager_destroy(h)
            self._h = None

    def create_sequence(self) -> Sequence:
        s = Sequence()
        check(_lib().helix_block_manager_create_sequence(self._h, ctypes.byref(s)))
        return s

    def fork_sequence(self, source, prefix_tokens, allow_cow=False):
        s, c = Sequence(), _native.CowCopy()
        check(_lib().helix_block_manager_fork_sequence(self._h, source, prefix_tokens,
                                                       int(allow_cow), ctypes.byref(s),
                                                       ctypes.byref(c)))
        return s, (c.from_block, c.to_block, c.tokens)

    def append(self, seq, tokens=1):
        slots = (ctypes.c_uint64 * tokens)()
        check(_lib().helix_block_manager_append(self._h, seq, tokens, slots))
        return list(slots)

    def release_sequence(self, seq):
        check(_lib().helix_block_manager_release_sequence(self._h, seq))

    def truncate_sequence(self, seq, length):
        """Drops the tokens from `length` on and frees the pages they alone held."""
        check(_lib().helix_block_manager_truncate(self._h, seq, length))

    def contains(self, seq):
        out = ctypes.c_int()
        check(_lib().helix_block_manager_contains(self._h, seq, ctypes.byref(out)))
        return bool(out.value)

    def length(self, seq):
        out = ctypes.c_size_t()
        check(_lib().helix_block_manager_length(self._h, seq, ctypes.byref(out)))
        return out.value

    def block_table(self, seq):
        n = ctypes.c_size_t()
        buf = (ctypes.c_uint32 * self.physical_blocks)()
        check(_lib().helix_block_manager_block_table(self._h, seq, buf, self.physical_blocks,
                                                     ctypes.byref(n)))
        return list(buf[: n.value])

    def stats(self):
        s = _native.Stats()
        check(_lib().helix_block_manager_stats(self._h, ctypes.byref(s)))
        return s.as_dict()

    def block_info(self, block):
        r, t = ctypes.c_size_t(), ctypes.c_size_t()
        check(_lib().helix_block_manager_block_info(self._h, block, ctypes.byref(r),
                                                    ctypes.byref(t)))
        return r.value, t.value

    def validate(self):
        check(_lib().helix_block_manager_validate(self._h))

    def geometry(self):
        a, b, c = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
        check(_lib().helix_block_manager_geometry(self._h, ctypes.byref(a), ctypes.byref(b),
                                                  ctypes.byref(c)))
        return a.value, b.value, c.value


PAGE_DTYPES = {"f32": 0, "bf16": 1, "fp8": 2}

# ---------------------------------------------------------- prefix cache ----
PREFIX_INSERTED, PREFIX_ALREADY_PRESENT, PREFIX_REJECTED_TOO_LARGE = 0, 1, 2


def _tokens(tokens):
    arr = (ctypes.c_uint32 * max(len(tokens), 1))(*[int(t) for t in tokens])
    return arr, len(tokens)


class PagedPrefixCache:
    """helix::kv_cache::PagedPrefixCache (include/helix/kv_cache/prefix.hpp:
    66-112) over a ``PagedKvCache`` (device pool) or a ``BlockManager`` (host
    bookkeeping only).  ``insert`` returns one of PREFIX_INSERTED,
    PREFIX_ALREADY_PRESENT, PREFIX_REJECTED_TOO_LARGE; ``lookup_longest``
    returns ``(sequence, matched_tokens)`` or None, and the caller releases
    the sequence."""

    def __init__(self, pool, maximum_entries, maximum_block_references):
        h = ctypes.c_void_p()
        cfg = _native.PrefixConfig(maximum_entries, maximum_block_references)
        if isinstance(pool, BlockManager):
            check(_lib().helix_prefix_cache_create_host(pool._h, ctypes.byref(cfg),
                                                        ctypes.byref(h)))
        elif isinstance(pool, PagedKvCache):
            check(_lib().helix_prefix_cache_create(pool._h, ctypes.byref(cfg), ctypes.byref(h)))
        else:
            check(_lib().helix_prefix_cache_create(None, ctypes.byref(cfg), ctypes.byref(h)))
        self._h = h
        self._pool = pool  # the host manager must outlive the index

    def close(self):
        h = getattr(self, "_h", None)
        if h:
            _lib().helix_prefix_cache_destroy(h)
            self._h = None

    def __del__(self, _finalizing=sys.is_finalizing):
        if _finalizing():
            return  # the process is exiting; the driver reclaims device memory
        self.close()

    def insert(self, namespace_id, tokens, source):
        arr, n = _tokens(tokens)
        out = ctypes.c_int()
        check(_lib().helix_prefix_cache_insert(self._h, namespace_id, arr, n, source,
                                               ctypes.byref(out)))
        return out.value

    def lookup_longest(self, namespace_id, tokens, maximum_prefix_tokens=None):
        arr, n = _tokens(tokens)
        limit = (1 << 64) - 1 if maximum_prefix_tokens is None else maximum_prefix_tokens
        hit, seq, matched = ctypes.c_int(), Sequence(), ctypes.c_size_t()
        check(_lib().helix_prefix_cache_lookup_longest(self._h, namespace_id, arr, n, limit,
                                                       ctypes.byref(hit), ctypes.byref(seq),
                                                       ctypes.byref(matched)))
        return (seq, matched.value) if hit.value else None

    def contains(self, namespace_id, tokens):
        arr, n = _tokens(tokens)
        out = ctypes.c_int()
        check(_lib().helix_prefix_cache_contains(self._h, namespace_id, arr, n,
                                                 ctypes.byref(out)))
        return bool(out.value)

    def erase(self, namespace_id, tokens):
        arr, n = _tokens(tokens)
        out = ctypes.c_int()
        check(_lib().helix_prefix_cache_erase(self._h, namespace_id, arr, n, ctypes.byref(out)))
        return bool(out.value)

    def evict_lru(self):
        out = ctypes.c_int()
        check(_lib().helix_prefix_cache_evict_lru(self._h, ctypes.byref(out)))
        return bool(out.value)

    def clear(self):
        check(_lib().helix_prefix_cache_clear(self._h))

    def stats(self):
        s = _native.PrefixStats()
        check(_lib().helix_prefix_cache_stats(self._h, ctypes.byref(s)))
        return s.as_dict()

    def config(self):
        c = _native.PrefixConfig()
        check(_lib().helix_prefix_cache_config(self._h, ctypes.byref(c)))
        return c.maximum_entries, c.maximum_block_references

    def block_tokens(self):
        out = ctypes.c_size_t()
        check(_lib().helix_prefix_cache_block_tokens(self._h, ctypes.byref(out)))
        return out.value


# ---------------------------------------------------------------- device ----
class PagedKvCache:
    """GPU paged KV pool (CudaPagedKvCache + the CPU cache's fork/bulk append)."""

    def __init__(self, layers, kv_heads, head_dimension, block_tokens, physical_blocks,
                 device=0, page_dtype="f32", k_scale=1.0, v_scale=1.0):
        """``page_dtype`` "bf16" stores pages as bf16 (extension: appended
        fp32 rows rounded to nearest even, gathers widen back to fp32);
        "fp8" stores OCP E4M3 codes of x / k_scale (keys) and x / v_scale
        (values), rounded to nearest even and saturating at +-448; gathers
        return decode(code) * scale."""
        h = ctypes.c_void_p()
        cfg = _cfg(layers, kv_heads, head_dimension, block_tokens, physical_blocks)
        if page_dtype not in PAGE_DTYPES:
            raise HelixError(INVALID_ARGUMENT, f"page_dtype must be one of {sorted(PAGE_DTYPES)}")
        if page_dtype != "fp8" and (k_scale != 1.0 or v_scale != 1.0):
            raise HelixError(INVALID_ARGUMENT, "k_scale and v_scale apply to fp8 pages only")
        if page_dtype == "fp8":
            check(_lib().helix_paged_cache_create_fp8(ctypes.byref(cfg), device, float(k_scale),
                                                      float(v_scale), ctypes.byref(h)))
        else:
            check(_lib().helix_paged_cache_create_typed(ctypes.byref(cfg), device,
                                                        PAGE_DTYPES[page_dtype], ctypes.byref(h)))
        self._h = h
        self.page_dtype = page_dtype
        ks, vs = ctypes.c_float(), ctypes.c_float()
        check(_lib().helix_paged_cache_fp8_scales(h, ctypes.byref(ks), ctypes.byref(vs)))
        self.k_scale, self.v_scale = ks.value, vs.value
        self.layers, self.kv_heads, self.head_dimension = layers, kv_heads, head_dimension
        self.block_tokens, self.physical_blocks, self.device = block_tokens, physical_blocks, device

    def close(self):
        h = getattr(self, "_h", None)
        if h:
            _lib().helix_paged_cache_destroy(h)
            self._h = None

    def __del__(self, _finalizing=sys.is_finalizing):
        if _finalizing():
            return  # the process is exiting; the driver reclaims device memory
        self.close()

    def create_sequence(self) -> Sequence:
        s = Sequence()
        check(_lib().helix_paged_cache_create_sequence(self._h, ctypes.byref(s)))
        return s

    def fork_sequence(self, source, prefix_tokens, allow_cow=False, stream=None):
        s = Sequence()
        check(_lib().helix_paged_cache_fork_sequence(self._h, source, prefix_tokens,
                                                     int(allow_cow), _stream(stream),
                                                     ctypes.byref(s)))
        return s

    def append(self, seq, token_keys, token_values, stream=None):
        """token_keys/values: device [layers, kv_heads, head_dimension]."""
        for t, n in ((token_keys, "token keys"), (token_values, "token values")):
            _require_f32(t, n)
            if tuple(t.shape) != (self.layers, self.kv_heads, self.head_dimension):
                raise HelixError(INVALID_ARGUMENT,
                                 f"{n} shape does not match [layers, heads, dimension]")
        check(_lib().helix_paged_cache_append(self._h, seq, _ptr(token_keys), _ptr(token_values),
                                              _stream(stream)))

    def append_layer_major(self, seq, layer_keys, layer_values, stream=None):
        """One device [kv_heads, tokens, head_dimension] tensor per layer."""
        if len(layer_keys) != self.layers or len(layer_values) != self.layers:
            raise HelixError(INVALID_ARGUMENT, "requires one key/value tensor per layer")
        tokens = layer_keys[0].shape[1]
        for t in list(layer_keys) + list(layer_values):
            _require_f32(t, "layer tensor")
            if tuple(t.shape) != (self.kv_heads, tokens, self.head_dimension):
                raise HelixError(INVALID_ARGUMENT, "layer tensor shape mismatch")
        kp = (ctypes.c_void_p * self.layers)(*[t.data_ptr() for t in layer_keys])
        vp = (ctypes.c_void_p * self.layers)(*[t.data_ptr() for t in layer_values])
        check(_lib().helix_paged_cache_append_layer_major(self._h, seq, kp, vp, tokens,
                                                          _stream(stream)))

    def release_sequence(self, seq):
        check(_lib().helix_paged_cache_release_sequence(self._h, seq))

    def truncate_sequence(self, seq, length):
        """Drops the tokens from `length` on and frees the pages they alone held."""
        check(_lib().helix_paged_cache_truncate_sequence(self._h, seq, length))

    def retrieve_layer(self, seq, layer):
        """Allocating gather: returns device (keys, values) [kv_heads, length, dim]."""
        import torch
        n = self.length(seq)
        shape = (self.kv_heads, n, self.head_dimension)
        k = torch.empty(shape, dtype=torch.float32, device=f"cuda:{self.device}")
        v = torch.empty(shape, dtype=torch.float32, device=f"cuda:{self.device}")
        self.copy_layer_out(seq, layer, k, v)
        return k, v

    def copy_layer_out(self, seq, layer, keys, values, stream=None):
        check(_lib().helix_paged_cache_copy_layer_out(self._h, seq, layer, _ptr(keys),
                                                      _ptr(values), _stream(stream)))

    def copy_layer_prefix_out(self, seq, layer, expected_length, keys, values, stream=None):
        check(_lib().helix_paged_cache_copy_layer_prefix_out(
            self._h, seq, layer, expected_length, _ptr(keys), _ptr(values), keys.shape[1],
            _stream(stream)))

    def contains(self, seq):
        out = ctypes.c_int()
        check(_lib().helix_paged_cache_contains(self._h, seq, ctypes.byref(out)))
        return bool(out.value)

    def length(self, seq):
        out = ctypes.c_size_t()
        check(_lib().helix_paged_cache_length(self._h, seq, ctypes.byref(out)))
        return out.value

    def block_table(self, seq):
        n = ctypes.c_size_t()
        buf = (ctypes.c_uint32 * self.physical_blocks)()
        check(_lib().helix_paged_cache_block_table(self._h, seq, buf, self.physical_blocks,
                                                   ctypes.byref(n)))
        return list(buf[: n.value])

    def stats(self):
        s = _native.Stats()
        check(_lib().helix_paged_cache_stats(self._h, ctypes.byref(s)))
        return s.as_dict()

    def is_healthy(self):
        out = ctypes.c_int()
        check(_lib().helix_paged_cache_is_healthy(self._h, ctypes.byref(out)))
        return bool(out.value)

    def geometry(self):
        a, b, c = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
        check(_lib().helix_paged_cache_geometry(self._h, ctypes.byref(a), ctypes.byref(b),
                                                ctypes.byref(c)))
        return a.value, b.value, c.value

    def layer_pool_pointers(self, layer):
        k, v = ctypes.c_void_p(), ctypes.c_void_p()
        check(_lib().helix_paged_cache_layer_pools(self._h, layer, ctypes.byref(k),
                                                   ctypes.byref(v)))
        return k.value, v.value

    def layer_pools(self, layer):
        """Device copies of layer `layer`'s pools [physical, kv_heads, block_tokens, dim]
        (float32, bfloat16 for a bf16 cache, uint8 E4M3 codes for an fp8 cache)."""
        import torch
        kp, vp = self.layer_pool_pointers(layer)
        shape = (self.physical_blocks, self.kv_heads, self.block_tokens, self.head_dimension)
        dtype = {"bf16": torch.bfloat16, "fp8": torch.uint8}.get(self.page_dtype, torch.float32)
        out = []
        for p in (kp, vp):
            t = torch.empty(shape, dtype=dtype, device=f"cuda:{self.device}")
            device_copy(t.data_ptr(), p, t.numel() * t.element_size())
            out.append(t)
        return out[0], out[1]

    def read_sequence(self, seq):
        return DecodeView(self, seq)


class DecodeView:
    """Read lease on one sequence; holds the cache lock until released."""

    def __init__(self, cache, seq):
        h = ctypes.c_void_p()
        check(_lib().helix_paged_cache_read_sequence(cache._h, seq, ctypes.byref(h)))
        self._h = h
        self._cache = cache

    def release(self):
        if getattr(self, "_h", None):
            _lib().helix_decode_view_release(self._h)
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.release()

    def __del__(self, _finalizing=sys.is_finalizing):
        if _finalizing():
            return  # the process is exiting; the driver reclaims device memory
        self.release()

    def length(self):
        out = ctypes.c_size_t()
        check(_lib().helix_decode_view_length(self._h, ctypes.byref(out)))
        return out.value

    def physical_blocks(self):
        p, n = ctypes.POINTER(ctypes.c_uint32)(), ctypes.c_size_t()
        check(_lib().helix_decode_view_physical_blocks(self._h, ctypes.byref(p), ctypes.byref(n)))
        return [p[i] for i in range(n.value)]

    def block_table(self):
        p = ctypes.c_void_p()
        check(_lib().helix_decode_view_block_table(self._h, ctypes.byref(p)))
        return p.value

    def layer_pool_pointers(self, layer):
        k, v = ctypes.c_void_p(), ctypes.c_void_p()
        check(_lib().helix_decode_view_layer_pools(self._h, layer, ctypes.byref(k),
                                                   ctypes.byref(v)))
        return k.value, v.value

    def poison(self):
        _lib().helix_decode_view_poison(self._h)


class PagedBlockTable:
    """Validated device copy of a logical->physical page mapping."""

    def __init__(self, physical_blocks, physical_block_count, device=0):
        ids = (ctypes.c_uint32 * max(1, len(physical_blocks)))(*physical_blocks)
        h = ctypes.c_void_p()
        check(_lib().helix_block_table_create(ids, len(physical_blocks), physical_block_count,
                                              device, ctypes.byref(h)))
        self._h = h
        self.logical_block_count = len(physical_blocks)
        self.physical_block_count = physical_block_count

    def data(self):
        return _lib().helix_block_table_data(self._h)

    def __del__(self, _finalizing=sys.is_finalizing):
        if _finalizing():
            return  # the process is exiting; the driver reclaims device memory
        h = getattr(self, "_h", None)
        if h:
            _lib().helix_block_table_destroy(h)
            self._h = None


# ------------------------------------------------------------- attention ----
def rope_out(input, cosine, sine, output, positions=None, stream=None):
    """kernels::rope / cpu::rope_out (src/kernels/cpu/reference.cpp:490-533) on
    device tensors: input/output [tokens, ..., head_dim] float32 (output may
    be input), cosine/sine [rows, head_dim / 2].  Without positions token t
    uses row t (rows must equal tokens); with int32 positions [tokens] it uses
    row positions[t]."""
    tokens, head_dim = input.shape[0], input.shape[-1]
    vectors = input.numel() // (tokens * head_dim) if tokens and head_dim else 0
    check(_lib().helix_rope(_ptr(input), _ptr(output), tokens, vectors, head_dim, _ptr(cosine),
                            _ptr(sine), cosine.shape[0],
                            None if positions is None else _ptr(positions), _stream(stream)))
    return output


def rope(input, cosine, sine, positions=None, stream=None):
    import torch
    return rope_out(input, cosine, sine, torch.empty_like(input), positions, stream)


def paged_attention_out(query, key_blocks, value_blocks, block_table, kv_tokens,
                        query_position_offset, output, score_workspace, stream=None):
    """paged_scaled_dot_product_attention_out; block_table: device uint32 pointer or tensor."""
    hq, nq, kd = query.shape
    n, hkv, p, vd = value_blocks.shape
    table_ptr = block_table.data_ptr() if hasattr(block_table, "data_ptr") else block_table
    logical = 0 if kv_tokens == 0 else (kv_tokens - 1) // p + 1
    check(_lib().helix_paged_attention_out(
        _ptr(query), hq, nq, kd, _ptr(key_blocks), _ptr(value_blocks), n, hkv, p, vd,
        ctypes.c_void_p(table_ptr), logical, kv_tokens, query_position_offset, _ptr(output),
        _ptr(score_workspace), score_workspace.numel(), _stream(stream)))


def paged_attention_with_tail_out(query, key_blocks, value_blocks, block_table, history_tokens,
                                  tail_key, tail_value, output, score_workspace, stream=None,
                                  logical_blocks=None, probabilities=False):
    """paged_scaled_dot_product_attention_with_tail_out; score_workspace
    [q_heads, tail, history + tail] receives the softmax probabilities, as
    the reference's contract says.  probabilities=True selects the exact
    scalar kernel for every shape
    (helix_paged_attention_with_tail_probabilities_out)."""
    hq, t, kd = query.shape
    n, hkv, p, vd = value_blocks.shape
    table_ptr = block_table.data_ptr() if hasattr(block_table, "data_ptr") else block_table
    if logical_blocks is None:
        logical_blocks = 0 if history_tokens == 0 else (history_tokens - 1) // p + 1
    fn = (_lib().helix_paged_attention_with_tail_probabilities_out if probabilities
          else _lib().helix_paged_attention_with_tail_out)
    check(fn(_ptr(query), hq, t, kd, _ptr(key_blocks), _ptr(value_blocks), n, hkv, p, vd,
             ctypes.c_void_p(table_ptr), logical_blocks, history_tokens, _ptr(tail_key),
             _ptr(tail_value), _ptr(output), _ptr(score_workspace), score_workspace.numel(),
             _stream(stream)))


def decode_workspace_bytes(batch, q_heads, kv_heads, max_blocks, pages_per_split=0):
    out = ctypes.c_size_t()
    check(_lib().helix_paged_decode_workspace_bytes(batch, q_heads, kv_heads, max_blocks,
                                                    pages_per_split, ctypes.byref(out)))
    return out.value


def decode_workspace(batch, q_heads, kv_heads, max_blocks, pages_per_split=0, device="cuda:0",
                     stream=None):
    """Allocate and zero a decode workspace (torch uint8 tensor)."""
    import torch
    n = decode_workspace_bytes(batch, q_heads, kv_heads, max_blocks, pages_per_split)
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device=device)
    check(_lib().helix_paged_decode_workspace_init(_ptr(ws), ws.numel(), _stream(stream)))
    return ws


_PAGE_DTYPES = {"f32": 0, "bf16": 1, "fp8": 2}


def paged_decode_attention(query, key_pool, value_pool, tables, lengths, tail_key, tail_value,
                           output, workspace, pages_per_split=0, stream=None, pool_shape=None,
                           page_dtype="f32", k_scale=1.0, v_scale=1.0):
    """Batched decode: query [B, Hq, 128]; pools [N, Hkv, 16, 128] tensors (or raw
    device addresses with pool_shape) of page_dtype "f32", "bf16" or "fp8"
    (E4M3 codes with scales k_scale / v_scale, pools as uint8 / int16 / any
    tensor whose bytes are the pages); tables [B, max_blocks] int32/uint32;
    lengths [B] int32; tail [B, Hkv, 128]; output [B, Hq, 128]."""
    b, hq, _ = query.shape
    if pool_shape is None:
        pool_shape = tuple(key_pool.shape)
        key_pool, value_pool = key_pool.data_ptr(), value_pool.data_ptr()
    n, hkv, p, d = pool_shape
    dtype = _PAGE_DTYPES.get(page_dtype, page_dtype)
    check(_lib().helix_paged_decode_attention_typed(
        _ptr(query), b, hq, hkv, d, ctypes.c_void_p(key_pool), ctypes.c_void_p(value_pool), n,
        p, _ptr(tables),
        tables.shape[1], _ptr(lengths), _ptr(tail_key), _ptr(tail_value), _ptr(output),
        _ptr(workspace), workspace.numel() * workspace.element_size(), pages_per_split,
        dtype, k_scale, v_scale, _stream(stream)))


def append_slots(keys, values, key_pool, value_pool, slots, stream=None):
    """Write rows [count, Hkv, D] into one layer's pools at int64 slots."""
    n, hkv, p, d = key_pool.shape
    check(_lib().helix_paged_append_slots(_ptr(keys), _ptr(values), _ptr(key_pool),
                                          _ptr(value_pool), n, hkv, p, d, _ptr(slots),
                                          slots.numel(), _stream(stream)))


def paged_prefill_attention(query, key_pool, value_pool, tables, lengths, chunk_key,
                            chunk_value, output, stream=None, pool_shape=None,
                            page_dtype="f32", k_scale=1.0, v_scale=1.0):
    """Batched chunked prefill (MFMA): query [B, Hq, T, 128]; pools [N, Hkv, 16,
    128] tensors (or raw device addresses with pool_shape) of page_dtype
    "f32", "bf16" or "fp8" (scales k_scale / v_scale); tables [B,
    max_blocks] int32/uint32; lengths [B] int32 history tokens; chunk_key /
    chunk_value [B, Hkv, T, 128] fp32; output [B, Hq, T, 128]."""
    b, hq, t, _ = query.shape
    if pool_shape is None:
        pool_shape = tuple(key_pool.shape)
        key_pool, value_pool = key_pool.data_ptr(), value_pool.data_ptr()
    n, hkv, p, d = pool_shape
    dtype = _PAGE_DTYPES.get(page_dtype, page_dtype)
    check(_lib().helix_paged_prefill_attention_typed(
        _ptr(query), b, hq, hkv, t, d, ctypes.c_void_p(key_pool), ctypes.c_void_p(value_pool),
        n, p, _ptr(tables), tables.shape[1], _ptr(lengths), _ptr(chunk_key), _ptr(chunk_value),
        _ptr(output), dtype, k_scale, v_scale, _stream(stream)))


def append_chunk(keys, values, key_pool, value_pool, slots, stream=None):
    """Write rows [B, Hkv, T, D] into one layer's pools at int64 slots [B, T]."""
    n, hkv, p, d = key_pool.shape
    b, t = slots.shape
    check(_lib().helix_paged_append_chunk(_ptr(keys), _ptr(values), _ptr(key_pool),
                                          _ptr(value_pool), n, hkv, p, d, _ptr(slots), b, t,
                                          _stream(stream)))


# ------------------------------------------------------------ tree steps ----
def _require_tensor(t, name, dtypes, shape, device=None, strided=False):
    """A device tensor of one of `dtypes` and of `shape` (None: any size),
    contiguous, or with `strided` contiguous in its last dimension."""
    try:  # (most calls' arguments are right, and a small call is this long)
        if (t.dtype in dtypes and t.shape == shape and t.is_contiguous() and
                (device is None or t.device == device)):
            return
    except (AttributeError, TypeError):
        pass
    import torch
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        names = " or ".join(str(d).replace("torch.", "") for d in dtypes)
        raise HelixError(INVALID_ARGUMENT, f"{name} must be a {names} tensor")
    if t.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape)):
        want = ", ".join("*" if n is None else str(n) for n in shape)
        raise HelixError(INVALID_ARGUMENT,
                         f"{name} must have shape [{want}], got {list(t.shape)}")
    if strided:
        if t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
            raise HelixError(INVALID_ARGUMENT, f"{name} must be contiguous in its last dimension")
    elif not t.is_contiguous():
        raise HelixError(INVALID_ARGUMENT, f"{name} must be contiguous")
    if device is not None and t.device != device:
        raise HelixError(INVALID_ARGUMENT, f"{name} must be on {device}, got {t.device}")


_POOL_DTYPES = {}


def _pool_dtypes(page_dtype):
    """What a pool tensor of page_dtype may be: its values, or their bits."""
    if not _POOL_DTYPES:
        import torch
        _POOL_DTYPES.update(f32=(torch.float32,),
                            bf16=(torch.bfloat16, torch.int16, torch.uint16),
                            fp8=(torch.float8_e4m3fn, torch.uint8, torch.int8))
    if page_dtype not in _POOL_DTYPES:
        raise HelixError(INVALID_ARGUMENT, 'page_dtype must be "f32", "bf16" or "fp8"')
    return _POOL_DTYPES[page_dtype]


_HERE = contextlib.nullcontext()


def _on(device):
    """The device of a call's tensors as the current one."""
    import torch
    if device.type != "cuda":
        raise HelixError(INVALID_ARGUMENT, f"tensors must be on a GPU, got {device}")
    if torch.cuda.current_device() == device.index:
        return _HERE
    return torch.cuda.device(device)


def _device_stream(stream, device):
    import torch
    return (torch.cuda.current_stream(device) if stream is None else stream).cuda_stream


def _address(t):
    return None if t is None else t.data_ptr()


def tree_workspace_bytes(batch, q_heads, kv_heads, nodes):
    out = ctypes.c_size_t()
    check(_lib().helix_paged_tree_workspace_bytes(batch, q_heads, kv_heads, nodes,
                                                  ctypes.byref(out)))
    return out.value


def tree_workspace(batch, q_heads, kv_heads, nodes, device="cuda:0"):
    """A workspace for paged_tree_attention (torch uint8 tensor; no initial
    value needed).  Calls that overlap need one each."""
    import torch
    n = tree_workspace_bytes(batch, q_heads, kv_heads, nodes)
    return torch.empty(max(n, 16), dtype=torch.uint8, device=device)


def paged_tree_attention(query, key_pool, value_pool, tables, lengths, tree_key, tree_value,
                         parents, output, workspace, node_counts=None, stream=None,
                         pool_shape=None, page_dtype="f32", k_scale=1.0, v_scale=1.0):
    """Attention of a tree of up to 64 drafted tokens per sequence: query row
    (h, t) sees the sequence's history, the ancestors of node t and node t.
    query, output [B, Hq, T, 128]; pools [N, Hkv, 16, 128] tensors (or raw
    device addresses with pool_shape) of page_dtype "f32", "bf16" (bfloat16, or
    its bits as int16 / uint16) or "fp8" (float8_e4m3fn, uint8 or int8);
    tables [B, max_blocks] int32/uint32; lengths [B] int32 history tokens;
    tree_key / tree_value [B, Hkv, T, 128]; parents [B, T] int32 (parent of
    each node, before it, or -1 for a root) or None for chains; node_counts [B]
    int32 or None: each sequence's own number of nodes, rows of `output` behind
    it stay as they were.  Any Hq that is a multiple of Hkv."""
    import torch
    if query.dim() != 4:
        raise HelixError(INVALID_ARGUMENT, "query must have shape [batch, q_heads, nodes, dim]")
    b, hq, t, d = query.shape
    f32, i32 = (torch.float32,), (torch.int32,)
    dev = query.device
    if pool_shape is None:
        pool_shape = key_pool.shape
        dtypes = _pool_dtypes(page_dtype)
        for pool, name in ((key_pool, "key_pool"), (value_pool, "value_pool")):
            _require_tensor(pool, name, dtypes, pool_shape, dev)
        key_pool, value_pool = key_pool.data_ptr(), value_pool.data_ptr()
    if len(pool_shape) != 4:
        raise HelixError(INVALID_ARGUMENT, "pools must have shape [blocks, kv_heads, tokens, dim]")
    n, hkv, p, pd = pool_shape
    if pd != d:
        raise HelixError(INVALID_ARGUMENT, "query and pools must have the same head size")
    _require_tensor(query, "query", f32, (b, hq, t, d))
    _require_tensor(output, "output", f32, (b, hq, t, d), dev)
    _require_tensor(tree_key, "tree_key", f32, (b, hkv, t, d), dev)
    _require_tensor(tree_value, "tree_value", f32, (b, hkv, t, d), dev)
    shape = getattr(tables, "shape", ())
    width = shape[1] if len(shape) == 2 else None
    _require_tensor(tables, "tables", (torch.int32, torch.uint32), (b, width), dev)
    _require_tensor(lengths, "lengths", i32, (b,), dev)
    if parents is not None:
        _require_tensor(parents, "parents", i32, (b, t), dev)
    if node_counts is not None:
        _require_tensor(node_counts, "node_counts", i32, (b,), dev)
    _require_tensor(workspace, "workspace", (workspace.dtype,), (workspace.numel(),), dev)
    dtype = _PAGE_DTYPES.get(page_dtype, -1)
    with _on(dev):
        check(_lib().helix_paged_tree_attention(
            _address(query), b, hq, hkv, t, d, key_pool, value_pool,
            n, p, _address(tables), width, _address(lengths), _address(tree_key),
            _address(tree_value), _address(parents), _address(node_counts), _address(output),
            _address(workspace), workspace.nbytes, dtype, k_scale,
            v_scale, _device_stream(stream, dev)))


def verify_workspace_bytes(batch, nodes, vocab):
    out = ctypes.c_size_t()
    check(_lib().helix_verify_tree_workspace_bytes(batch, nodes, vocab, ctypes.byref(out)))
    return out.value


def verify_workspace(batch, nodes, vocab, device="cuda:0"):
    """A workspace for verify_tree (torch uint8 tensor; no initial value
    needed).  Calls that overlap need one each."""
    import torch
    n = verify_workspace_bytes(batch, nodes, vocab)
    return torch.empty(max(n, 16), dtype=torch.uint8, device=device)


def _verify_arguments(target, draft, tokens, parents, uniforms, bonus_uniforms, path, accepted,
                      next_token, node_counts):
    """The checked arguments of a verification up to its strides, and behind
    its sizes."""
    import torch
    f32, i32 = (torch.float32,), (torch.int32,)
    shape = getattr(target, "shape", ())
    b, t, v = shape if len(shape) == 3 else (None, None, None)
    _require_tensor(target, "target", f32, (b, t, v), strided=True)
    dev = target.device
    if draft is not None:
        _require_tensor(draft, "draft", f32, (b, t, v), dev, strided=True)
    _require_tensor(tokens, "tokens", i32, (b, t), dev)
    if parents is not None:
        _require_tensor(parents, "parents", i32, (b, t), dev)
    if node_counts is not None:
        _require_tensor(node_counts, "node_counts", i32, (b,), dev)
    _require_tensor(uniforms, "uniforms", f32, (b, t), dev)
    _require_tensor(bonus_uniforms, "bonus_uniforms", f32, (b,), dev)
    _require_tensor(path, "path", i32, (b, t), dev)
    _require_tensor(accepted, "accepted", i32, (b,), dev)
    _require_tensor(next_token, "next_token", i32, (b,), dev)

    def strides(x):  # a dimension of one row may have any stride
        return (0, 0) if x is None else (x.stride(0) if b > 1 else 0,
                                         x.stride(1) if t > 1 else v)

    rows = (_address(target), *strides(target), _address(draft), *strides(draft))
    lists = (_address(tokens), _address(parents), _address(node_counts), _address(uniforms),
             _address(bonus_uniforms))
    return rows, lists, (_address(path), _address(accepted), _address(next_token))


def verify_tree(target, draft, tokens, parents, uniforms, bonus_uniforms, path, accepted,
                next_token, workspace, node_counts=None, stream=None):
    """Which drafted tokens the target's probabilities accept, and the token
    that follows them.  target [B, T, V]: row n is the target's distribution
    after node n; draft [B, T, V] or None: row n is the distribution the children
    of node n were drawn from (None: they were certain); both may be strided in
    their first two dimensions (nodes share no entries).  tokens [B, T] int32; parents [B, T] int32 or
    None for chains (node 0 is the root); uniforms [B, T] and bonus_uniforms [B]
    in [0, 1); node_counts [B] int32 or None.  Writes path [B, T] (accepted
    nodes from the root, then -1), accepted [B] (their number) and next_token
    [B], all int32."""
    rows, lists, out = _verify_arguments(target, draft, tokens, parents, uniforms, bonus_uniforms,
                                         path, accepted, next_token, node_counts)
    b, t, v = target.shape
    dev = target.device
    _require_tensor(workspace, "workspace", (workspace.dtype,), (workspace.numel(),), dev)
    with _on(dev):
        check(_lib().helix_verify_tree(
            *rows, b, t, v, *lists, *out, _address(workspace),
            workspace.nbytes, _device_stream(stream, dev)))


def append_path(keys, values, key_pool, value_pool, slots, path, accepted, stream=None,
                page_dtype="f32", k_scale=1.0, v_scale=1.0):
    """Write the rows of the accepted nodes, path[b, i] for i < accepted[b], to
    slots[b, i]: keys / values [B, Hkv, T, D] and pools [N, Hkv, P, D] (of the
    types that paged_tree_attention takes), or with a leading dimension of layers
    each (a pool's layers may lie apart); slots [B, T] int64, path [B, T] and
    accepted [B] int32."""
    import torch
    layered = key_pool.dim() == 5
    if key_pool.dim() not in (4, 5):
        raise HelixError(INVALID_ARGUMENT,
                         "pools must have shape [(layers,) blocks, kv_heads, tokens, dim]")
    dev = keys.device
    layers = key_pool.shape[0] if layered else 1
    n, hkv, p, d = key_pool.shape[-4:]
    lead = (layers,) if layered else ()
    shape = getattr(slots, "shape", ())
    b, t = shape if len(shape) == 2 else (None, None)
    _require_tensor(slots, "slots", (torch.int64,), (b, t), dev)
    _require_tensor(keys, "keys", (torch.float32,), (*lead, b, hkv, t, d))
    _require_tensor(values, "values", (torch.float32,), (*lead, b, hkv, t, d), dev)
    _require_tensor(path, "path", (torch.int32,), (b, t), dev)
    _require_tensor(accepted, "accepted", (torch.int32,), (b,), dev)
    dtypes = _pool_dtypes(page_dtype)
    stride = 0
    for pool, name in ((key_pool, "key_pool"), (value_pool, "value_pool")):
        if layered:
            _require_tensor(pool, name, dtypes, key_pool.shape, dev, strided=True)
            if layers and not pool.is_contiguous():  # a layer's pool is, if not all of them
                _require_tensor(pool[0], name, dtypes, key_pool.shape[1:], dev)
            if layers > 1:
                if pool.stride(0) != key_pool.stride(0):
                    raise HelixError(INVALID_ARGUMENT, "pools must have the same layer stride")
                stride = pool.stride(0)
        else:
            _require_tensor(pool, name, dtypes, key_pool.shape, dev)
    with _on(dev):
        check(_lib().helix_paged_append_path(
            _address(keys), _address(values), _address(key_pool), _address(value_pool), layers,
            stride, n, hkv, p, d, _address(slots), _address(path), _address(accepted), b, t,
            _PAGE_DTYPES.get(page_dtype, -1), k_scale, v_scale, _device_stream(stream, dev)))


# --------------------------------------- rotary positions, latent cache ----
ROPE_LAYOUTS = {"pairs": 0, "halves": 1}
ROPE_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "ramp": 3, "bands": 4}
LATENT_ROPE = 64  # rotated elements of a latent cache's row
LATENT_NOPE = 128  # key elements of a head without them, and of its value (expanded form)
_Strides = ctypes.c_size_t * 3


def _rows(t, name, shape, device=None):
    """The address of fp32 rows of `shape` (None: any size), contiguous in their
    last dimension, and their other strides (None: contiguous)."""
    _require_tensor(t, name, (_F32(),), shape, device, strided=True)
    if t.is_contiguous():
        return t.data_ptr(), None
    return t.data_ptr(), _Strides(*t.stride()[:-1])


_f32 = None


def _F32():
    global _f32
    if _f32 is None:
        import torch
        _f32 = torch.float32
    return _f32


def _optional_rows(t, name, shape, device):
    return (None, None) if t is None else _rows(t, name, shape, device)


def _layout(layout):
    if layout not in ROPE_LAYOUTS:
        raise HelixError(INVALID_ARGUMENT, f"layout must be one of {sorted(ROPE_LAYOUTS)}")
    return ROPE_LAYOUTS[layout]


def _rope_cache(cosine, sine, rotary_dim, device):
    """Checks the tables; their rows and the rotary dimension."""
    shape = getattr(cosine, "shape", ())
    rows, pairs = shape if len(shape) == 2 else (None, None)
    _require_tensor(cosine, "cosine", (_F32(),), (rows, pairs), device)
    _require_tensor(sine, "sine", (_F32(),), (rows, pairs), device)
    if rotary_dim is not None and rotary_dim != 2 * pairs:
        raise HelixError(INVALID_ARGUMENT, "tables must have shape [rows, rotary_dim / 2]")
    return rows, 2 * pairs


def rope_tables(cosine, sine, base=10000.0, first_position=0, scaling="none", factor=1.0,
                original_length=0, low=None, high=None, amplitude=1.0, stream=None):
    """Fill cosine and sine [rows, rotary_dim / 2] for positions first_position on:
    amplitude * cos and sin of position * base^(-2 i / rotary_dim), in 64 bits (angles
    are off by position * 2^-50 at most), rounded once.  scaling changes the frequencies for contexts longer than
    original_length, the one a model was trained on: "linear" (divided by factor),
    "ntk" (a larger base), "ramp" (divided where a wave turns at most `low` times
    over the original length, as they are from `high` turns on, a mean between,
    linear in the pair's index; 1 and 32 by default) or "bands" (the same, linear in
    the turns; 1 and 4 by default)."""
    import torch
    if scaling not in ROPE_SCALINGS:
        raise HelixError(INVALID_ARGUMENT, f"scaling must be one of {sorted(ROPE_SCALINGS)}")
    rows, rotary = _rope_cache(cosine, sine, None, None)
    if sine.device != cosine.device:
        raise HelixError(INVALID_ARGUMENT, "cosine and sine must be on one device")
    low = 1.0 if low is None else low
    high = (4.0 if scaling == "bands" else 32.0) if high is None else high
    if not isinstance(first_position, int) or first_position < 0:
        raise HelixError(INVALID_ARGUMENT, "first_position must be a whole number of 0 at least")
    dev = cosine.device
    with _on(dev):
        check(_lib().helix_rope_tables(
            cosine.data_ptr(), sine.data_ptr(), rows, first_position, rotary, base,
            ROPE_SCALINGS[scaling], factor, original_length, low, high, amplitude,
            _device_stream(stream, dev)))


def rope_rows(input, cosine, sine, output=None, positions=None, layout="pairs", rotary_dim=None,
              inverse=False, stream=None):
    """Rotate the first rotary_dim elements of rows [tokens, vectors, head_dim]
    (any strides but the last; the other elements are copied) to output (None: a new
    tensor; may be input itself).  cosine, sine [rows, rotary_dim / 2]; token t uses
    row positions[t] (int32) or t.  layout "pairs" turns elements (2 i, 2 i + 1),
    "halves" (i, i + rotary_dim / 2); inverse turns back (the gradient's way)."""
    import torch
    shape = getattr(input, "shape", ())
    if len(shape) != 3:
        raise HelixError(INVALID_ARGUMENT, "input must have shape [tokens, vectors, head_dim]")
    if output is None:
        output = torch.empty(shape, dtype=torch.float32, device=input.device)
    x, xs = _rows(input, "input", shape)
    dev = input.device
    y, ys = _rows(output, "output", shape, dev)
    rows, rotary = _rope_cache(cosine, sine, rotary_dim, dev)
    tokens, vectors, dim = shape
    if positions is not None:
        _require_tensor(positions, "positions", (torch.int32,), (tokens,), dev)
    elif rows < tokens:
        raise HelixError(INVALID_ARGUMENT, "without positions the tables need a row per token")
    order = _layout(layout)
    with _on(dev):
        check(_lib().helix_rope_rows(
            x, xs, y, ys, tokens, vectors, dim, rotary, order, bool(inverse),
            cosine.data_ptr(), sine.data_ptr(), rows, _address(positions),
            _device_stream(stream, dev)))
    return output


def _append_rows(batch, q_heads, kv_heads, tokens, dim, query, keys, values, query_out, key_out,
                 value_out, dev):
    """Checked addresses and strides of a rope append's rows, inputs then outputs."""
    if (query is None) != (query_out is None):
        raise HelixError(INVALID_ARGUMENT, "query and query_out go together")
    q, kv = (batch, q_heads, tokens, dim), (batch, kv_heads, tokens, dim)
    return (*_optional_rows(query, "query", q, dev), *_rows(keys, "keys", kv, dev),
            *_rows(values, "values", kv, dev), *_optional_rows(query_out, "query_out", q, dev),
            *_optional_rows(key_out, "key_out", kv, dev),
            *_optional_rows(value_out, "value_out", kv, dev))


def rope_append(query, keys, values, key_pool, value_pool, starts, slots, cosine, sine,
                query_out=None, key_out=None, value_out=None, layout="pairs", rotary_dim=None,
                token_counts=None, stream=None, page_dtype="f32", k_scale=1.0, v_scale=1.0):
    """Append a step's new rows with the rotation on the way, in one launch.
    query [B, Hq, T, D] (or None) rotated to query_out; keys [B, Hkv, T, D] rotated to
    their pages, and to key_out where given; values likewise, not rotated.  All of
    any strides but the last (a projection's output as it lies); an output may be its
    input.  Pools [N, Hkv, P, D] of page_dtype; slots [B, T] int64 (outside the
    pool: no page); row t of sequence b stands at position starts[b] + t (int32);
    token_counts [B] int32 or None: each sequence's own number of rows."""
    import torch
    shape = getattr(keys, "shape", ())
    if len(shape) != 4:
        raise HelixError(INVALID_ARGUMENT, "keys must have shape [batch, kv_heads, tokens, dim]")
    b, hkv, t, d = shape
    dev = keys.device
    hq = query.shape[1] if query is not None and query.dim() == 4 else 0
    rows = _append_rows(b, hq, hkv, t, d, query, keys, values, query_out, key_out, value_out, dev)
    dtypes = _pool_dtypes(page_dtype)
    n, _, p, _ = pool_shape = key_pool.shape if key_pool.dim() == 4 else (None, hkv, None, d)
    if pool_shape[1] != hkv or pool_shape[3] != d:
        raise HelixError(INVALID_ARGUMENT, "pools must have the heads and head size of the keys")
    _require_tensor(key_pool, "key_pool", dtypes, pool_shape, dev)
    _require_tensor(value_pool, "value_pool", dtypes, pool_shape, dev)
    _require_tensor(slots, "slots", (torch.int64,), (b, t), dev)
    _require_tensor(starts, "starts", (torch.int32,), (b,), dev)
    if token_counts is not None:
        _require_tensor(token_counts, "token_counts", (torch.int32,), (b,), dev)
    table_rows, rotary = _rope_cache(cosine, sine, rotary_dim, dev)
    order = _layout(layout)
    with _on(dev):
        check(_lib().helix_paged_rope_append(
            *rows, b, hq, hkv, t, d, key_pool.data_ptr(), value_pool.data_ptr(), n, p,
            slots.data_ptr(), starts.data_ptr(), _address(token_counts), cosine.data_ptr(),
            sine.data_ptr(), table_rows, rotary, order, _PAGE_DTYPES[page_dtype],
            k_scale, v_scale, _device_stream(stream, dev)))


def _latent_pool(pool, pool_shape, page_dtype, dev):
    """A latent cache's pages [N, 16, latent + 64]: address and shape."""
    dtypes = _pool_dtypes(page_dtype)
    if pool_shape is None:
        pool_shape = getattr(pool, "shape", ())
        if len(pool_shape) == 3:
            _require_tensor(pool, "pool", dtypes, pool_shape, dev)
            pool = pool.data_ptr()
    if len(pool_shape) != 3:
        raise HelixError(INVALID_ARGUMENT, "pool must have shape [blocks, tokens, latent + 64]")
    return pool, pool_shape


def latent_append(latent, rope_key, pool, starts, slots, cosine, sine, query=None, query_out=None,
                  layout="pairs", token_counts=None, stream=None, pool_shape=None,
                  page_dtype="f32", page_scale=1.0):
    """Append a step's rows to a latent cache, pages [N, 16, latent + 64] of
    page_dtype (or a raw address with pool_shape): latent [B, T, latent], and rope_key
    [B, T, 64] rotated behind it.  query [B, Hq, T, 64], the rotated part of the
    queries, goes to query_out, which may be the last part of the absorbed queries
    ([B, Hq, T, latent + 64][..., latent:]).  The rest as rope_append."""
    import torch
    shape = getattr(latent, "shape", ())
    if len(shape) != 3:
        raise HelixError(INVALID_ARGUMENT, "latent must have shape [batch, tokens, latent]")
    if (query is None) != (query_out is None):
        raise HelixError(INVALID_ARGUMENT, "query and query_out go together")
    b, t, n = shape
    dev = latent.device
    rows = (*_rows(latent, "latent", (b, t, n)),
            *_rows(rope_key, "rope_key", (b, t, LATENT_ROPE), dev))
    hq = query.shape[1] if query is not None and query.dim() == 4 else 0
    q = (b, hq, t, LATENT_ROPE)
    rows += (*_optional_rows(query, "query", q, dev),
             *_optional_rows(query_out, "query_out", q, dev))
    pages, (blocks, p, width) = _latent_pool(pool, pool_shape, page_dtype, dev)
    if width != n + LATENT_ROPE:
        raise HelixError(INVALID_ARGUMENT, "pages must hold rows of latent + 64 elements")
    _require_tensor(slots, "slots", (torch.int64,), (b, t), dev)
    _require_tensor(starts, "starts", (torch.int32,), (b,), dev)
    if token_counts is not None:
        _require_tensor(token_counts, "token_counts", (torch.int32,), (b,), dev)
    table_rows, _ = _rope_cache(cosine, sine, LATENT_ROPE, dev)
    order = _layout(layout)
    with _on(dev):
        check(_lib().helix_paged_latent_append(
            *rows, b, hq, t, n, pages, blocks, p, slots.data_ptr(), starts.data_ptr(),
            _address(token_counts), cosine.data_ptr(), sine.data_ptr(), table_rows,
            order, _PAGE_DTYPES[page_dtype], page_scale, _device_stream(stream, dev)))


def latent_workspace_bytes(batch, q_heads, tokens, latent=512):
    out = ctypes.c_size_t()
    check(_lib().helix_paged_latent_workspace_bytes(batch, q_heads, tokens, latent,
                                                    ctypes.byref(out)))
    return out.value


def latent_workspace(batch, q_heads, tokens, latent=512, device="cuda:0"):
    """A workspace for paged_latent_attention (torch uint8 tensor; no initial
    value needed).  Calls that overlap need one each."""
    import torch
    n = latent_workspace_bytes(batch, q_heads, tokens, latent)
    return torch.empty(max(n, 16), dtype=torch.uint8, device=device)


def paged_latent_attention(query, pool, tables, lengths, output, workspace, scale,
                           token_counts=None, stream=None, pool_shape=None, page_dtype="f32",
                           page_scale=1.0):
    """Attention over a latent cache, absorbed form: query [B, Hq, T, latent + 64],
    output [B, Hq, T, latent] (any strides of four elements but the last); pages [N,
    16, latent + 64] tensors (or a raw address with pool_shape) of page_dtype; tables
    [B, max_blocks] int32/uint32; lengths [B] int32 tokens in the pages, the step's
    own (token_counts [B] int32, or T) the last: row t sees the first lengths[b] -
    token_counts[b] + t + 1.  scale multiplies the scores.  Rows that see nothing are
    0; rows of `output` behind token_counts stay as they were."""
    import torch
    shape = getattr(query, "shape", ())
    if len(shape) != 4:
        raise HelixError(INVALID_ARGUMENT, "query must have shape [batch, q_heads, tokens, dim]")
    b, hq, t, width = shape
    dev = query.device
    pages, (blocks, p, w) = _latent_pool(pool, pool_shape, page_dtype, dev)
    if w != width or width <= LATENT_ROPE:
        raise HelixError(INVALID_ARGUMENT, "query and pages must have rows of latent + 64 elements")
    n = width - LATENT_ROPE
    q = _rows(query, "query", shape)
    o = _rows(output, "output", (b, hq, t, n), dev)
    i32 = (torch.int32,)
    shape = getattr(tables, "shape", ())
    max_blocks = shape[1] if len(shape) == 2 else None
    _require_tensor(tables, "tables", (torch.int32, torch.uint32), (b, max_blocks), dev)
    _require_tensor(lengths, "lengths", i32, (b,), dev)
    if token_counts is not None:
        _require_tensor(token_counts, "token_counts", i32, (b,), dev)
    _require_tensor(workspace, "workspace", (workspace.dtype,), (workspace.numel(),), dev)
    with _on(dev):
        check(_lib().helix_paged_latent_attention(
            *q, b, hq, t, n, pages, blocks, p, tables.data_ptr(), max_blocks, lengths.data_ptr(),
            _address(token_counts), *o, scale, workspace.data_ptr(), workspace.nbytes,
            _PAGE_DTYPES[page_dtype], page_scale, _device_stream(stream, dev)))


def latent_prefill_workspace_bytes(batch, heads, tokens, keys):
    out = ctypes.c_size_t()
    check(_lib().helix_latent_prefill_workspace_bytes(batch, heads, tokens, keys,
                                                      ctypes.byref(out)))
    return out.value


def latent_prefill_workspace(batch, heads, tokens, keys, device="cuda:0"):
    """A workspace for latent_prefill_attention (torch uint8 tensor; no initial
    value needed).  Calls that overlap need one each."""
    import torch
    n = latent_prefill_workspace_bytes(batch, heads, tokens, keys)
    return torch.empty(max(n, 16), dtype=torch.uint8, device=device)


def latent_prefill_attention(query, key, rope_key, value, output, workspace, scale,
                             key_lengths=None, token_counts=None, stream=None):
    """Attention of a latent cache's prompts, expanded form: query [B, H, T, 128 +
    64], key and value [B, H, S, 128], rope_key [B, S, 64] shared by the heads, output
    [B, H, T, 128] (any strides of four elements but the last).  Sequence b has
    key_lengths[b] keys (int32; None: S), its token_counts[b] new tokens' (int32;
    None: T) the last: row t sees the first key_lengths[b] - token_counts[b] + t + 1.
    Rows that see nothing are 0; rows of `output` behind token_counts stay as they
    were.  (Numbers that vary by more than fp16's range within a head take up to two
    and a half times as long.)"""
    import torch
    qs, ks = getattr(query, "shape", ()), getattr(key, "shape", ())
    if len(qs) != 4 or len(ks) != 4:
        raise HelixError(INVALID_ARGUMENT,
                         "query and key must have shape [batch, heads, tokens, dim]")
    b, h, t, _ = qs
    s = ks[2]
    dev = query.device
    args = (*_rows(query, "query", (b, h, t, LATENT_NOPE + LATENT_ROPE)),
            *_rows(key, "key", (b, h, s, LATENT_NOPE), dev),
            *_rows(rope_key, "rope_key", (b, s, LATENT_ROPE), dev),
            *_rows(value, "value", (b, h, s, LATENT_NOPE), dev))
    o = _rows(output, "output", (b, h, t, LATENT_NOPE), dev)
    for x, name in ((key_lengths, "key_lengths"), (token_counts, "token_counts")):
        if x is not None:
            _require_tensor(x, name, (torch.int32,), (b,), dev)
    _require_tensor(workspace, "workspace", (workspace.dtype,), (workspace.numel(),), dev)
    with _on(dev):
        check(_lib().helix_latent_prefill_attention(
            *args, b, h, t, s, _address(key_lengths), _address(token_counts), *o, scale,
            workspace.data_ptr(), workspace.nbytes, _device_stream(stream, dev)))


class DecodeBatch:
    """Batched decode driver over a PagedKvCache (persistent device tables)."""

    def __init__(self, cache, sequences, q_heads, max_tokens, pages_per_split=0):
        arr = (Sequence * len(sequences))(*sequences)
        h = ctypes.c_void_p()
        check(_lib().helix_decode_batch_create(cache._h, arr, len(sequences), q_heads, max_tokens,
                                               pages_per_split, ctypes.byref(h)))
        self._h = h
        self._cache = cache
        self.batch = len(sequences)
        self.q_heads = q_heads

    def close(self):
        h = getattr(self, "_h", None)
        if h:
            _lib().helix_decode_batch_destroy(h)
            self._h = None

    def __del__(self, _finalizing=sys.is_finalizing):
        if _finalizing():
            return  # the process is exiting; the driver reclaims device memory
        self.close()

    def prepare(self, stream=None):
        check(_lib().helix_decode_batch_prepare(self._h, _stream(stream)))
        self._tokens = 1

    def append_attention_layer(self, layer, query, keys, values, output, stream=None):
        """append_layer + attention_layer in one decode launch (the new token
        rows are the attention tail and are written to their slots)."""
        check(_lib().helix_decode_batch_append_attention_layer(
            self._h, layer, _ptr(query), _ptr(keys), _ptr(values), _ptr(output),
            _stream(stream)))

    def prepare_chunk(self, tokens, stream=None):
        """Reserve `tokens` slots per sequence (chunked prefill step)."""
        check(_lib().helix_decode_batch_prepare_chunk(self._h, tokens, _stream(stream)))
        self._tokens = tokens

    def prefill_layer(self, layer, query, chunk_key, chunk_value, output, stream=None):
        check(_lib().helix_decode_batch_prefill_layer(self._h, layer, _ptr(query),
                                                      _ptr(chunk_key), _ptr(chunk_value),
                                                      _ptr(output), _stream(stream)))

    def append_layer(self, layer, keys, values, stream=None):
        check(_lib().helix_decode_batch_append_layer(self._h, layer, _ptr(keys), _ptr(values),
                                                     _stream(stream)))

    def append_all_layers(self, keys, values, stream=None):
        """append_layer for every layer in one launch: rows [layers, batch,
        kv_heads, tokens, head_dim] (the step's token committed after the
        forward pass, as CudaPagedKvCache::append commits [layers, kv_heads,
        head_dim] for one sequence)."""
        check(_lib().helix_decode_batch_append_all_layers(self._h, _ptr(keys), _ptr(values),
                                                          _stream(stream)))

    def rope(self, query, key, cosine, sine, stream=None):
        """Rotary embedding of the step's query [batch, q_heads, dim] and key
        [batch, kv_heads, dim] in place, each sequence at its position (its
        length before the step); cosine/sine [rows, dim / 2]."""
        check(_lib().helix_decode_batch_rope(self._h, _ptr(query), _ptr(key), _ptr(cosine),
                                             _ptr(sine), cosine.shape[0], _stream(stream)))

    def rope_append_layer(self, layer, query, keys, values, cosine, sine, query_out, key_out=None,
                          value_out=None, layout="pairs", rotary_dim=None, stream=None):
        """rope() and append_layer() in one launch, for chunk steps too: query
        [batch, q_heads, tokens, dim] (or None) rotated to query_out, keys [batch,
        kv_heads, tokens, dim] rotated to the step's slots and to key_out, values to
        theirs and to value_out, each sequence from its length before the step on.
        Rows may be strided, outputs may be their inputs; key_out and value_out are
        what attention_layer() or prefill_layer() takes."""
        import torch
        dev = torch.device("cuda", self._cache.device)
        t = getattr(self, "_tokens", 0)
        rows = _append_rows(self.batch, self.q_heads, self._cache.kv_heads, t,
                            self._cache.head_dimension, query, keys, values, query_out, key_out,
                            value_out, dev)
        table_rows, rotary = _rope_cache(cosine, sine, rotary_dim, dev)
        check(_lib().helix_decode_batch_rope_append_layer(
            self._h, layer, *rows, cosine.data_ptr(), sine.data_ptr(), table_rows, rotary,
            _layout(layout), _device_stream(stream, dev)))

    def attention_layer(self, layer, query, tail_key, tail_value, output, stream=None):
        check(_lib().helix_decode_batch_attention_layer(self._h, layer, _ptr(query),
                                                        _ptr(tail_key), _ptr(tail_value),
                                                        _ptr(output), _stream(stream)))

    def prepare_tree(self, nodes, stream=None):
        """Reserve the slots of a tree of `nodes` drafted tokens (up to 64) per
        sequence: tree_layer() in every layer, then accept_tree() or
        commit_path().  An uncommitted tree step is dropped by the next
        prepare call or close()."""
        import torch
        dev = torch.device("cuda", self._cache.device)
        check(_lib().helix_decode_batch_prepare_tree(self._h, nodes, _device_stream(stream, dev)))
        self._nodes = nodes

    def tree_layer(self, layer, query, tree_key, tree_value, parents, output, node_counts=None,
                   stream=None):
        """paged_tree_attention over the batch: query, output [batch, q_heads,
        nodes, dim], tree rows [batch, kv_heads, nodes, dim]."""
        import torch
        t, hkv, d = getattr(self, "_nodes", 0), self._cache.kv_heads, self._cache.head_dimension
        dev = torch.device("cuda", self._cache.device)
        for x, name, heads in ((query, "query", self.q_heads), (tree_key, "tree_key", hkv),
                               (tree_value, "tree_value", hkv), (output, "output", self.q_heads)):
            _require_tensor(x, name, (torch.float32,), (self.batch, heads, t, d), dev)
        for x, name, shape in ((parents, "parents", (self.batch, t)),
                               (node_counts, "node_counts", (self.batch,))):
            if x is not None:
                _require_tensor(x, name, (torch.int32,), shape, dev)
        check(_lib().helix_decode_batch_tree_layer(
            self._h, layer, _ptr(query), _ptr(tree_key), _ptr(tree_value), _ptr(parents),
            _ptr(node_counts), _ptr(output), _device_stream(stream, dev)))

    def _tree_rows(self, keys, values):
        import torch
        shape = (self._cache.layers, self.batch, self._cache.kv_heads, getattr(self, "_nodes", 0),
                 self._cache.head_dimension)
        dev = torch.device("cuda", self._cache.device)
        _require_tensor(keys, "keys", (torch.float32,), shape, dev)
        _require_tensor(values, "values", (torch.float32,), shape, dev)
        return dev

    def commit_path(self, keys, values, path, accepted, stream=None):
        """End a tree step: the rows [layers, batch, kv_heads, nodes, dim] of the
        accepted nodes go to their pages in every layer, and each sequence keeps
        its accepted tokens (path [batch, nodes], accepted [batch] int32, as
        verify_tree leaves them).  Synchronises the stream."""
        import torch
        dev = self._tree_rows(keys, values)
        _require_tensor(path, "path", (torch.int32,), (self.batch, keys.shape[3]), dev)
        _require_tensor(accepted, "accepted", (torch.int32,), (self.batch,), dev)
        check(_lib().helix_decode_batch_commit_path(self._h, _ptr(keys), _ptr(values), _ptr(path),
                                                    _ptr(accepted), _device_stream(stream, dev)))

    def accept_tree(self, target, draft, tokens, parents, uniforms, bonus_uniforms, keys, values,
                    path, accepted, next_token, node_counts=None, stream=None):
        """verify_tree of the step's drafts, then commit_path of what it accepts."""
        dev = self._tree_rows(keys, values)
        rows, lists, out = _verify_arguments(target, draft, tokens, parents, uniforms,
                                             bonus_uniforms, path, accepted, next_token,
                                             node_counts)
        _require_tensor(target, "target", (target.dtype,), (self.batch, keys.shape[3], None), dev,
                        strided=True)
        check(_lib().helix_decode_batch_accept_tree(
            self._h, *rows, target.shape[2], *lists, _ptr(keys), _ptr(values), *out,
            _device_stream(stream, dev)))

    def shared_pages(self):
        """Leading pages the prepared decode step attends once for the batch."""
        n = ctypes.c_size_t()
        check(_lib().helix_decode_batch_shared_pages(self._h, ctypes.byref(n)))
        return n.value

    def set_timing_event(self, event):
        """Record `event` (a torch.cuda.Event or None) between the main decode
        kernel and the merge kernel of every attention_layer()."""
        if event is not None:
            event = ctypes.c_void_p(event.cuda_event if hasattr(event, "cuda_event") else event)
        check(_lib().helix_decode_batch_set_timing_event(self._h, event))

    def device_state(self):
        t, l, s = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
        mb, ps = ctypes.c_size_t(), ctypes.c_size_t()
        check(_lib().helix_decode_batch_tables(self._h, ctypes.byref(t), ctypes.byref(l),
                                               ctypes.byref(s), ctypes.byref(mb),
                                               ctypes.byref(ps)))
        return {"tables": t.value, "lengths": l.value, "slots": s.value,
                "max_blocks": mb.value, "pages_per_split": ps.value}


# ---------------------------------------------------------------- plumbing ----
_hip = None


def device_copy(dst: int, src: int, nbytes: int):
    """hipMemcpy device-to-device (plumbing for reading raw pool memory)."""
    global _hip
    if _hip is None:
        _hip = ctypes.CDLL("libamdhip64.so")
        _hip.hipMemcpy.restype = ctypes.c_int
        _hip.hipMemcpy.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]
    rc = _hip.hipMemcpy(ctypes.c_void_p(dst), ctypes.c_void_p(src), nbytes, 3)
    if rc != 0:
        raise HelixError(RUNTIME, f"hipMemcpy failed with {rc}")
