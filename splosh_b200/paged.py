"""A paged key/value cache of the caller's own, over libsploshcuda's spl_paged_* entry points: append with the rotation applied on the way, and
attention of a chunk of new tokens (single tokens, verify blocks, prompt chunks) over it. Addresses are ints, as in the other primitives. No CPU
fallback: the calls run on the engine's device."""
import ctypes as C

import numpy as np

from .engine import EngineError, lib, stream_handle, _ptr

TYPES = {"f32": 0, "fp16": 1, "bf16": 2, "e4m3": 3}


class _Config(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("heads", "kv_heads", "head_dim", "dtype", "page_tokens", "pages")] + \
               [(n, C.c_int64) for n in ("page_stride", "head_stride", "token_stride")] + \
               [("rotary_dim", C.c_int32), ("rope_theta", C.c_float), ("scale", C.c_float)] + \
               [(n, C.c_int32) for n in ("causal", "window", "max_sequences", "max_rows", "max_context")]


def _type(name):
    if name not in TYPES:
        raise EngineError(10, f"no such type: {name}; one of {', '.join(TYPES)}")
    return TYPES[name]


def _config(heads, kv_heads, head_dim, pages, page_tokens=256, dtype="bf16", layout="head", strides=None, rotary_dim=0, rope_theta=10000.0, scale=0.0, causal=True, window=0,
            max_sequences=8, max_rows=64, max_context=32768):
    if strides is None:
        if layout not in ("head", "token"):
            raise EngineError(10, f"no such layout: {layout}; head or token")
        page = kv_heads * page_tokens * head_dim
        strides = (page, page_tokens * head_dim, head_dim) if layout == "head" else (page, head_dim, kv_heads * head_dim)
    return _Config(heads, kv_heads, head_dim, _type(dtype), page_tokens, pages, *strides, rotary_dim, rope_theta, scale, int(causal), window, max_sequences, max_rows, max_context)


def _batch(rows, lengths, page_table):
    rows, lengths, table = (np.ascontiguousarray(x, np.int32) for x in (rows, lengths, page_table))
    if rows.ndim != 1 or lengths.shape != rows.shape or table.ndim != 2 or table.shape[0] != rows.shape[0]:
        raise EngineError(10, "rows and lengths are one number a sequence, the page table one row a sequence")
    return rows, lengths, table


def _groups(groups):
    groups = np.ascontiguousarray(groups if groups is not None else (), np.int32).reshape(-1, 2)
    return np.ascontiguousarray(groups[:, 0]), np.ascontiguousarray(groups[:, 1])


def paged_check(rows=(), lengths=(), page_table=None, groups=None, **config):
    """What PagedAttention and its batch would say to these arguments, without a GPU (spl_paged_check_shared): whether append would refuse the batch."""
    cfg, message, shared = _config(**config), C.create_string_buffer(256), C.c_int32(0)
    rows, lengths, table = _batch(rows, lengths, np.zeros((len(rows), 0), np.int32) if page_table is None else page_table)
    sequences, tokens = _groups(groups)
    status = lib().spl_paged_check_shared(C.byref(cfg), rows.shape[0], _ptr(rows), _ptr(lengths), _ptr(table), table.shape[1], len(sequences), _ptr(sequences), _ptr(tokens), C.byref(shared), message,
                                          len(message))
    if status:
        raise EngineError(status, message.value.decode() or "spl_paged_check refused its arguments")
    return bool(shared.value)


def debug_paged_plan(rows, lengths, blocks=148, **config):
    """How a batch's attention is dealt to the blocks of a launch (spl_debug_paged_plan): (block_begin, items, merges)."""
    cfg = _config(**config)
    rows, lengths = np.ascontiguousarray(rows, np.int32), np.ascontiguousarray(lengths, np.int32)
    group = cfg.heads // cfg.kv_heads
    capacity = cfg.kv_heads * (int(rows.sum()) * group // 128 + len(rows)) + blocks
    begin, items, merges = np.zeros(blocks + 1, np.int32), np.zeros((capacity, 8), np.int32), np.zeros((blocks, 8), np.int32)
    item_count, merge_count = C.c_int32(0), C.c_int32(0)
    status = lib().spl_debug_paged_plan(C.byref(cfg), blocks, len(rows), _ptr(rows), _ptr(lengths), _ptr(begin), _ptr(items), capacity, C.byref(item_count), _ptr(merges), C.byref(merge_count))
    if status:
        raise EngineError(status, "spl_debug_paged_plan refused its arguments")
    return begin, items[:item_count.value], merges[:merge_count.value]


def debug_paged_plan_shared(rows, lengths, groups, blocks=148, **config):
    """How a batch with groups is dealt to the blocks of a launch (spl_debug_paged_plan_shared): (block_begin, items, records, rows of partial sums, whether some sequences meet a prefix together)."""
    cfg = _config(**config)
    rows, lengths = np.ascontiguousarray(rows, np.int32), np.ascontiguousarray(lengths, np.int32)
    sequences, tokens = _groups(groups)
    capacity = 2 * (cfg.kv_heads * (int(rows.sum()) * (cfg.heads // cfg.kv_heads) // 128 + len(rows)) + blocks)
    begin, items, records = np.zeros(blocks + 1, np.int32), np.zeros((capacity, 8), np.int32), np.zeros((capacity, 10), np.int32)
    item_count, record_count, partial_rows, joint = C.c_int32(0), C.c_int32(0), C.c_int64(0), C.c_int32(0)
    status = lib().spl_debug_paged_plan_shared(C.byref(cfg), blocks, len(rows), _ptr(rows), _ptr(lengths), len(sequences), _ptr(sequences), _ptr(tokens), _ptr(begin), _ptr(items), capacity,
                                               C.byref(item_count), _ptr(records), capacity, C.byref(record_count), C.byref(partial_rows), C.byref(joint))
    if status:
        raise EngineError(status, "spl_debug_paged_plan_shared refused its arguments, or a plan is larger than what is set aside for it")
    return begin, items[:item_count.value], records[:record_count.value], partial_rows.value, bool(joint.value)


class PagedAttention:
    """One layer shape and the batch of a pass (spl_paged). The cache is the caller's: K and V each `pages` pages in the layout "head"
    ([page][kv head][token][channel]) or "token" ([page][token][kv head][channel]), or with `strides` (page, head, token) in elements. With dtype "e4m3" the cache holds 8-bit codes,
    their scales are fp32 [page][kv head][token], and queries are bf16."""

    def __init__(self, engine, heads, kv_heads, head_dim, pages, page_tokens=256, dtype="bf16", layout="head", strides=None, rotary_dim=0, rope_theta=10000.0, scale=0.0,
                 causal=True, window=0, max_sequences=8, max_rows=64, max_context=32768):
        self.handle, self.engine, self.dtype = None, engine, dtype
        self.q_width, self.kv_width = heads * head_dim, kv_heads * head_dim
        cfg = _config(heads, kv_heads, head_dim, pages, page_tokens, dtype, layout, strides, rotary_dim, rope_theta, scale, causal, window, max_sequences, max_rows, max_context)
        handle = C.c_void_p()
        engine._check(lib().spl_paged_create(engine.handle, C.byref(cfg), C.byref(handle)))
        self.handle = handle

    def close(self):
        if getattr(self, "handle", None):
            lib().spl_paged_destroy(self.handle); self.handle = None

    def __del__(self):
        self.close()

    def _handle(self):
        if not self.handle or not self.engine.handle:
            raise EngineError(10, "the engine or this object is closed")
        return self.handle

    def batch(self, rows, lengths, page_table, stream=None, groups=None):
        """The sequences of a pass: new tokens and length (with them) of each, and its pages (int32 [sequences][pages of the longest]). `groups`: (sequences, tokens) pairs, the next so many sequences begin
        with the same pages of so many tokens (spl_paged_batch_shared)."""
        rows, lengths, table = _batch(rows, lengths, page_table)
        sequences, tokens = _groups(groups)
        self.engine._check(lib().spl_paged_batch_shared(self._handle(), rows.shape[0], _ptr(rows), _ptr(lengths), _ptr(table), table.shape[1], len(sequences), _ptr(sequences), _ptr(tokens),
                                                        stream_handle(stream)))

    def append(self, q, k, v, q_out, k_cache, v_cache, dtype="f32", ld=None, q_norm=None, k_norm=None, stream=None, k_scale=None, v_scale=None):
        """Rows of `dtype` at the addresses q, k, v (row stride `ld` elements for all three, or a triple; None: each contiguous) -> rotated queries at q_out,
        keys and values in the cache. q_norm and k_norm are tensors of Engine.tensor_vector. k_scale and v_scale: the scales of an e4m3 cache."""
        q_ld, k_ld, v_ld = (self.q_width, self.kv_width, self.kv_width) if ld is None else (ld,) * 3 if np.isscalar(ld) else ld
        if k_scale is None and v_scale is None:
            self.engine._check(lib().spl_paged_append(self._handle(), _type(dtype), q, q_ld, k, k_ld, v, v_ld, q_norm, k_norm, q_out, k_cache, v_cache, stream_handle(stream)))
        else:
            self.engine._check(lib().spl_paged_append_scaled(self._handle(), _type(dtype), q, q_ld, k, k_ld, v, v_ld, q_norm, k_norm, q_out, k_cache, v_cache, k_scale, v_scale, stream_handle(stream)))

    def attend(self, q, k_cache, v_cache, out, out_dtype=None, stream=None, k_scale=None, v_scale=None):
        """The batch's rows over the cache: q and out [rows][heads][head_dim], out of the queries' type or "f32". k_scale and v_scale: the scales of an e4m3 cache."""
        out_type = _type(out_dtype or ("bf16" if self.dtype == "e4m3" else self.dtype))
        if k_scale is None and v_scale is None:
            self.engine._check(lib().spl_paged_attend(self._handle(), q, k_cache, v_cache, out_type, out, stream_handle(stream)))
        else:
            self.engine._check(lib().spl_paged_attend_scaled(self._handle(), q, k_cache, v_cache, k_scale, v_scale, out_type, out, stream_handle(stream)))
