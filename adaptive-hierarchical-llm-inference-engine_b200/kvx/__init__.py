"""Python front end of libadaptive_engine.so (ctypes over the C ABI in
include/kvx.h and include/adaptive_engine.h).

Tensors are torch CUDA tensors; only their data pointers and the current
CUDA stream cross the ABI.  There is no fallback: importing this module on a
machine where the library cannot be loaded raises, and every call whose
status is not KVX_OK raises KvxError.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import os
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
LIB_PATH = os.path.join(PKG, "libadaptive_engine.so")

KVX_F32, KVX_F16, KVX_I8 = 0, 1, 2
HEAD_DIM, PAGE_TOKENS = 128, 16

STATUS = {0: "ok", -1: "invalid argument", -2: "object pinned", -3: "CUDA error",
          -4: "unsupported geometry or dtype", -5: "bounded device wait expired",
          -6: "workspace or pool too small", -7: "no sm_100 device",
          -8: "request exceeds the static scratch of kvx_decode_noalloc",
          -9: "another rank's part of the multi-GPU step failed"}


class KvxError(RuntimeError):
    def __init__(self, fn, status):
        super().__init__(f"{fn}: {STATUS.get(status, status)} ({status})")
        self.status = status


def build() -> str:
    """Compile the library in-tree (nvcc, sm_100a)."""
    import subprocess
    subprocess.run(["make", "-s", "-C", PKG, "-j8"], check=True)
    return LIB_PATH


def _load():
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is not built; run `make -C {PKG}`")
    return C.CDLL(LIB_PATH)


lib = _load()


class KvPaged(C.Structure):
    _fields_ = [("pool", C.c_void_p), ("stats", C.c_void_p), ("dtype", C.c_int32),
                ("num_pages", C.c_int32), ("num_kv_heads", C.c_int32),
                ("head_dim", C.c_int32), ("page_tokens", C.c_int32)]


_vp, _i32, _sz, _f32 = C.c_void_p, C.c_int32, C.c_size_t, C.c_float
lib.kvx_version.restype = C.c_char_p
lib.kvx_status_string.restype = C.c_char_p
lib.kvx_status_string.argtypes = [C.c_int]
lib.kvx_device_check.restype = C.c_int
lib.kvx_append.argtypes = [C.POINTER(KvPaged), _vp, _i32, _vp, _i32, _vp, _vp, _vp, _vp]
lib.kvx_append_chunk.argtypes = [C.POINTER(KvPaged), _vp, _i32, _vp, _i32, _i32, _vp, _vp, _vp, _vp]
lib.kvx_append_chunk.restype = C.c_int
lib.kvx_decode_workspace_bytes.restype = _sz
lib.kvx_decode_workspace_bytes.argtypes = [_i32, _i32, _i32, _i32]
lib.kvx_decode.argtypes = [C.POINTER(KvPaged), _vp, _i32, _vp, _i32, _i32, _vp, _vp, _i32, _f32,
                           _vp, _sz, _vp, _vp]
lib.kvx_append_decode.argtypes = [C.POINTER(KvPaged), _vp, _i32, _vp, _i32, _vp, _vp, _i32, _vp,
                                  _vp, _i32, _f32, _vp, _sz, _vp, _vp]
lib.kvx_append_decode_signal.argtypes = [C.POINTER(KvPaged), _vp, _i32, _vp, _i32, _vp, _vp, _i32, _vp,
                                         _vp, _i32, _f32, _vp, _sz, _vp, _vp, C.c_uint32, _vp]
lib.kvx_stream_wait_geq.argtypes = [_vp, C.c_uint32, _vp]
lib.kvx_decode_workspace_init.argtypes = [_vp, _sz, _vp]
lib.kvx_decode_noalloc.argtypes = [C.POINTER(KvPaged), _vp, _i32, _vp, _i32, _i32, _vp, _vp, _i32,
                                   _f32, _vp, _vp]
lib.kvx_decode_noalloc.restype = C.c_int
lib.kvx_decode_noalloc_scratch_bytes.restype = _sz
lib.kvx_compress_int8.argtypes = [_vp, _i32, _vp, _vp, _sz, _i32, _vp]
lib.kvx_decompress_int8.argtypes = [_vp, _vp, _vp, _i32, _sz, _i32, _vp]
lib.kvx_compress_nf4.argtypes = [_vp, _i32, _vp, _vp, _sz, _i32, _vp]
lib.kvx_decompress_nf4.argtypes = [_vp, _vp, _vp, _i32, _sz, _i32, _vp]
lib.kvx_fp16_wrap_encode.argtypes = [_vp, _vp, _sz, _vp]
lib.kvx_fp16_wrap_decode.argtypes = [_vp, _vp, _sz, _vp]
lib.kvx_f32_to_f16_trunc.argtypes = [_vp, _vp, _sz, _vp]
lib.kvx_f16_trunc_to_f32.argtypes = [_vp, _vp, _sz, _vp]
lib.kvx_lru_select.argtypes = [_vp, _sz, _vp, _vp]
lib.kvx_migrate_frames.argtypes = [_vp, _i32, _vp, _i32, _vp, _vp, _i32, _sz, _i32, _i32, _vp, _vp]
lib.kvx_evict_select.argtypes = [_i32, _vp, _sz, _f32, _vp, _vp, _vp]
lib.kvx_decode_attn_workspace_bytes.restype = _sz
lib.kvx_decode_attn_workspace_bytes.argtypes = [_i32, _i32, _i32, _i32]
lib.kvx_decode_attn.argtypes = [C.POINTER(KvPaged), _vp, _i32, _vp, _i32, _i32, _vp, _vp, _i32, _f32,
                                _vp, _sz, _vp, _vp, _vp]
lib.kvx_decode_attn.restype = C.c_int
lib.kvx_attn_to_metrics.argtypes = [_vp, _vp, _i32, _vp, _i32, _vp, _i32, C.c_uint64, _vp]
lib.kvx_attn_to_metrics.restype = C.c_int
lib.kvx_evict_select_composite.argtypes = [_vp, _vp, _i32, _vp, _sz, _f32, _vp, _vp, _vp]


class RopeConfig(C.Structure):
    _fields_ = [("rotary_dim", C.c_int32), ("scaling", C.c_int32), ("base", C.c_double), ("factor", C.c_double),
                ("low", C.c_double), ("high", C.c_double), ("original_context", C.c_double)]


class RopeTableC(C.Structure):
    _fields_ = [("turns", C.c_void_p), ("rotary_dim", C.c_int32), ("layout", C.c_int32), ("amplitude", C.c_float)]


class RopeRows(C.Structure):
    _fields_ = [("in_", C.c_void_p), ("out", C.c_void_p), ("heads", C.c_int32), ("in_token_stride", C.c_int64),
                ("in_head_stride", C.c_int64), ("out_token_stride", C.c_int64), ("out_head_stride", C.c_int64)]


_i64 = C.c_int64
lib.kvx_rope_frequencies.argtypes = [C.POINTER(RopeConfig), _vp, C.POINTER(C.c_float)]
lib.kvx_rope.argtypes = [C.POINTER(RopeTableC), _vp, _i32, _i32, _i32, _vp, _i32, _i32, _vp]  # RopeRows, or their bytes
lib.kvx_rope_append.argtypes = [C.POINTER(KvPaged), _vp, _i32, _vp, _vp, _i32, _i32, C.POINTER(RopeTableC), _i32, _vp, _i64,
                                _vp, _i32, _vp, _i64, _vp, _i64, _vp, _vp]
lib.kvx_attend_chunk_workspace_bytes.restype = _sz
lib.kvx_attend_chunk_workspace_bytes.argtypes = [_i32, _i32, _i32, _i32, _i32]
lib.kvx_attend_chunk.argtypes = [C.POINTER(KvPaged), _vp, _i32, _vp, _vp, _i32, _i32, _i32, _vp, _vp, _i32, _f32, _i32, _vp,
                                 _sz, _vp, _vp]
for _fn in ("kvx_rope_frequencies", "kvx_rope", "kvx_rope_append", "kvx_attend_chunk",
            "kvx_append", "kvx_decode", "kvx_append_decode", "kvx_append_decode_signal", "kvx_stream_wait_geq",
            "kvx_decode_workspace_init", "kvx_compress_int8", "kvx_decompress_int8",
            "kvx_compress_nf4", "kvx_decompress_nf4", "kvx_fp16_wrap_encode", "kvx_fp16_wrap_decode",
            "kvx_f32_to_f16_trunc", "kvx_f16_trunc_to_f32", "kvx_lru_select",
            "kvx_migrate_frames", "kvx_evict_select", "kvx_evict_select_composite"):
    getattr(lib, _fn).restype = C.c_int


def _check(fn, rc):
    if rc != 0:
        raise KvxError(fn, rc)


def _torch():
    import torch
    return torch


def _stream(stream):
    if stream is not None:
        return C.c_void_p(stream if isinstance(stream, int) else stream.cuda_stream)
    return C.c_void_p(_torch().cuda.current_stream().cuda_stream)


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _dtype_code(t):
    torch = _torch()
    return {torch.float32: KVX_F32, torch.float16: KVX_F16, torch.int8: KVX_I8}[t.dtype]


def paged(pool, stats=None) -> KvPaged:
    """Describe one layer's pool: a CUDA tensor [pages][2][hkv][16][128], or
    an existing KvPaged view (e.g. from kvx.engine.layer_view)."""
    if isinstance(pool, KvPaged):
        return pool
    assert pool.is_cuda and pool.is_contiguous() and pool.dim() == 5
    pages, two, hkv, pt, dim = pool.shape
    assert two == 2
    return KvPaged(pool.data_ptr(), 0 if stats is None else stats.data_ptr(), _dtype_code(pool),
                   pages, hkv, dim, pt)


class _DeviceArray:
    """__cuda_array_interface__ over a raw device address (no ownership)."""

    def __init__(self, ptr, shape, typestr):
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": tuple(shape), "typestr": typestr,
                                         "version": 3, "strides": None}


def pool_tensor(view):
    """A torch view [pages][2][hkv][16][128] of a KvPaged pool (e.g. an
    engine layer from kvx.engine.layer_view); the memory stays the owner's."""
    torch = _torch()
    typestr = {KVX_F32: "<f4", KVX_F16: "<f2", KVX_I8: "|i1"}[view.dtype]
    shape = (view.num_pages, 2, view.num_kv_heads, view.page_tokens, view.head_dim)
    return torch.as_tensor(_DeviceArray(view.pool, shape, typestr), device="cuda")


def append(pool, block_table, positions, new_k, new_v, error_flag=None, stream=None):
    kv = paged(pool)
    rc = lib.kvx_append(C.byref(kv), _ptr(block_table), block_table.shape[1], _ptr(positions),
                        positions.shape[0], _ptr(new_k), _ptr(new_v), _ptr(error_flag),
                        _stream(stream))
    _check("kvx_append", rc)


def append_chunk(pool, block_table, positions, new_k, new_v, error_flag=None, stream=None):
    """Append new_k / new_v [batch][n_new][hkv][128] at positions[s] ..
    positions[s] + n_new - 1 of each sequence."""
    kv = paged(pool)
    batch, n_new = new_k.shape[0], new_k.shape[1]
    rc = lib.kvx_append_chunk(C.byref(kv), _ptr(block_table), block_table.shape[1], _ptr(positions), batch,
                              n_new, _ptr(new_k), _ptr(new_v), _ptr(error_flag), _stream(stream))
    _check("kvx_append_chunk", rc)


def decode_workspace_bytes(batch, num_q_heads, max_pages):
    return lib.kvx_decode_workspace_bytes(batch, num_q_heads, max_pages, PAGE_TOKENS)


def decode_workspace(batch, num_q_heads, max_pages, device="cuda"):
    """A zero-filled decode workspace (the split counters start at zero)."""
    torch = _torch()
    return torch.zeros(max(decode_workspace_bytes(batch, num_q_heads, max_pages), 16),
                       dtype=torch.uint8, device=device)


def decode(pool, block_table, seq_lens, q, out=None, stats=None, workspace=None,
           error_flag=None, sm_scale=0.0, stream=None):
    """Paged GQA decode.  q: [batch][hq][128] fp32/fp16 CUDA tensor."""
    torch = _torch()
    kv = paged(pool, stats)
    batch, hq, _ = q.shape
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:
        workspace = decode_workspace(batch, hq, block_table.shape[1], q.device)
    rc = lib.kvx_decode(C.byref(kv), _ptr(block_table), block_table.shape[1], _ptr(seq_lens),
                        batch, hq, _ptr(q), _ptr(out), _dtype_code(q), sm_scale,
                        _ptr(workspace), workspace.numel() * workspace.element_size(),
                        _ptr(error_flag), _stream(stream))
    _check("kvx_decode", rc)
    return out


def append_decode(pool, block_table, positions, new_k, new_v, q, out=None, workspace=None,
                  error_flag=None, sm_scale=0.0, stream=None):
    """Append the token at `positions` and decode over positions+1 tokens, one launch."""
    torch = _torch()
    kv = paged(pool)
    batch, hq, _ = q.shape
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:
        workspace = decode_workspace(batch, hq, block_table.shape[1], q.device)
    rc = lib.kvx_append_decode(C.byref(kv), _ptr(block_table), block_table.shape[1],
                               _ptr(positions), batch, _ptr(new_k), _ptr(new_v), hq, _ptr(q),
                               _ptr(out), _dtype_code(q), sm_scale, _ptr(workspace),
                               workspace.numel() * workspace.element_size(), _ptr(error_flag),
                               _stream(stream))
    _check("kvx_append_decode", rc)
    return out


def append_decode_signal(pool, block_table, positions, new_k, new_v, q, done, epoch, out=None,
                         workspace=None, error_flag=None, sm_scale=0.0, stream=None):
    """append_decode that stores `epoch` to done[1] once the whole launch has
    finished (done: int32 CUDA tensor of 2, done[0] zero-filled once)."""
    torch = _torch()
    kv = paged(pool)
    batch, hq, _ = q.shape
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:
        workspace = decode_workspace(batch, hq, block_table.shape[1], q.device)
    rc = lib.kvx_append_decode_signal(C.byref(kv), _ptr(block_table), block_table.shape[1],
                                      _ptr(positions), batch, _ptr(new_k), _ptr(new_v), hq, _ptr(q),
                                      _ptr(out), _dtype_code(q), sm_scale, _ptr(workspace),
                                      workspace.numel() * workspace.element_size(), _ptr(error_flag),
                                      _ptr(done), epoch & 0xFFFFFFFF, _stream(stream))
    _check("kvx_append_decode_signal", rc)
    return out


def stream_wait_geq(word, value, stream=None):
    """Make `stream` wait until the device word reaches `value` (cyclic
    32-bit comparison).  word: a CUDA tensor whose first element is waited on."""
    _check("kvx_stream_wait_geq", lib.kvx_stream_wait_geq(_ptr(word), value & 0xFFFFFFFF, _stream(stream)))


def compress_int8(src, block_elems=PAGE_TOKENS * HEAD_DIM, codes=None, stats=None, stream=None):
    torch = _torch()
    n = src.numel()
    nb = n // block_elems
    if codes is None:
        codes = torch.empty(n, dtype=torch.int8, device=src.device)
    if stats is None:
        stats = torch.empty((nb, 4), dtype=torch.float32, device=src.device)
    rc = lib.kvx_compress_int8(_ptr(src), _dtype_code(src), _ptr(codes), _ptr(stats), nb,
                               block_elems, _stream(stream))
    _check("kvx_compress_int8", rc)
    return codes, stats


def decompress_int8(codes, stats, dtype=None, block_elems=PAGE_TOKENS * HEAD_DIM, out=None,
                    stream=None):
    torch = _torch()
    dtype = dtype or torch.float32
    if out is None:
        out = torch.empty(codes.numel(), dtype=dtype, device=codes.device)
    rc = lib.kvx_decompress_int8(_ptr(codes), _ptr(stats), _ptr(out), _dtype_code(out),
                                 codes.numel() // block_elems, block_elems, _stream(stream))
    _check("kvx_decompress_int8", rc)
    return out


def compress_nf4(src, block_elems=PAGE_TOKENS * HEAD_DIM, codes=None, stats=None, stream=None):
    """KVCompressionEngine NF4 per block: codes (uint8, two per byte) and stats."""
    torch = _torch()
    nb = src.numel() // block_elems
    if codes is None:
        codes = torch.empty(nb * ((block_elems + 1) // 2), dtype=torch.uint8, device=src.device)
    if stats is None:
        stats = torch.empty((nb, 4), dtype=torch.float32, device=src.device)
    rc = lib.kvx_compress_nf4(_ptr(src), _dtype_code(src), _ptr(codes), _ptr(stats), nb, block_elems,
                              _stream(stream))
    _check("kvx_compress_nf4", rc)
    return codes, stats


def decompress_nf4(codes, stats, dtype=None, block_elems=PAGE_TOKENS * HEAD_DIM, out=None, stream=None):
    torch = _torch()
    dtype = dtype or torch.float32
    nb = stats.numel() // 4
    if out is None:
        out = torch.empty(nb * block_elems, dtype=dtype, device=codes.device)
    rc = lib.kvx_decompress_nf4(_ptr(codes), _ptr(stats), _ptr(out), _dtype_code(out), nb, block_elems,
                                _stream(stream))
    _check("kvx_decompress_nf4", rc)
    return out


def fp16_wrap_encode(x, out=None, stream=None):
    """KVCompressionEngine FP16 (exponent-wrapping): fp32 -> uint16 bits as int16 tensor."""
    torch = _torch()
    if out is None:
        out = torch.empty(x.numel(), dtype=torch.int16, device=x.device)
    _check("kvx_fp16_wrap_encode", lib.kvx_fp16_wrap_encode(_ptr(x), _ptr(out), x.numel(), _stream(stream)))
    return out


def fp16_wrap_decode(h, out=None, stream=None):
    torch = _torch()
    if out is None:
        out = torch.empty(h.numel(), dtype=torch.float32, device=h.device)
    _check("kvx_fp16_wrap_decode", lib.kvx_fp16_wrap_decode(_ptr(h), _ptr(out), h.numel(), _stream(stream)))
    return out


def f32_to_f16_trunc(x, out=None, stream=None):
    torch = _torch()
    if out is None:
        out = torch.empty(x.numel(), dtype=torch.int16, device=x.device)
    _check("kvx_f32_to_f16_trunc", lib.kvx_f32_to_f16_trunc(_ptr(x), _ptr(out), x.numel(),
                                                            _stream(stream)))
    return out


def f16_trunc_to_f32(h, out=None, stream=None):
    torch = _torch()
    if out is None:
        out = torch.empty(h.numel(), dtype=torch.float32, device=h.device)
    _check("kvx_f16_trunc_to_f32", lib.kvx_f16_trunc_to_f32(_ptr(h), _ptr(out), h.numel(),
                                                            _stream(stream)))
    return out


def softmax_rows(x, out=None, stream=None):
    """Row softmax of a [rows][cols] fp32 CUDA tensor (TensorOps::softmax)."""
    torch = _torch()
    if out is None:
        out = torch.empty_like(x)
    _check("kvx_softmax_rows", lib.kvx_softmax_rows(_ptr(x), _ptr(out), C.c_int64(x.shape[0]),
                                                    C.c_int64(x.shape[1]), _stream(stream)))
    return out


def attention_dense(q, k, v, out=None, scale=0.0, stream=None):
    """softmax(q k^T * scale) v for fp32 CUDA tensors q [seq_q][dim],
    k / v [seq_k][dim] (TensorOps::attention; scale <= 0 -> 1/sqrt(dim))."""
    torch = _torch()
    if out is None:
        out = torch.empty_like(q)
    _check("kvx_attention_dense",
           lib.kvx_attention_dense(_ptr(q), _ptr(k), _ptr(v), _ptr(out), C.c_int64(q.shape[0]),
                                   C.c_int64(k.shape[0]), C.c_int32(q.shape[1]), C.c_float(scale),
                                   _stream(stream)))
    return out


def lru_select(stamps, victim=None, stream=None):
    torch = _torch()
    if victim is None:
        victim = torch.empty(1, dtype=torch.int32, device=stamps.device)
    _check("kvx_lru_select", lib.kvx_lru_select(_ptr(stamps), stamps.numel(), _ptr(victim),
                                                _stream(stream)))
    return victim


def migrate_frames(dev_base, dev_capacity, host_base, host_capacity, dev_frames, host_frames,
                   frame_bytes, direction, ctas=0, error_flag=None, stream=None):
    """dev_base/host_base: raw addresses (int) or tensors; frames: int32 CUDA tensors."""
    def addr(x):
        return C.c_void_p(x if isinstance(x, int) else x.data_ptr())
    rc = lib.kvx_migrate_frames(addr(dev_base), dev_capacity, addr(host_base), host_capacity,
                                _ptr(dev_frames), _ptr(host_frames), dev_frames.numel(),
                                frame_bytes, direction, ctas, _ptr(error_flag), _stream(stream))
    _check("kvx_migrate_frames", rc)


EVICT_LRU, EVICT_TOKEN_WEIGHTED, EVICT_ATTENTION_BASED, EVICT_PREDICTIVE = 0, 1, 2, 3


def evict_select(policy, pages, decay=0.95, predicted=None, out=None, stream=None):
    """AdvancedEvictionPolicy selectPageToEvict on the device.  pages: CUDA
    uint8 tensor holding n EvictionMetrics records of 48 bytes."""
    torch = _torch()
    if out is None:
        out = torch.empty(1, dtype=torch.int32, device=pages.device)
    _check("kvx_evict_select", lib.kvx_evict_select(policy, _ptr(pages), pages.numel() // 48, decay,
                                                    _ptr(predicted), _ptr(out), _stream(stream)))
    return out


def evict_select_composite(policies, weights, pages, decay=0.95, predicted=None, out=None, stream=None):
    torch = _torch()
    if out is None:
        out = torch.empty(1, dtype=torch.int32, device=pages.device)
    pol = (C.c_int32 * len(policies))(*policies)
    w = (C.c_float * len(weights))(*[float(x) for x in weights])
    _check("kvx_evict_select_composite",
           lib.kvx_evict_select_composite(pol, w, len(policies), _ptr(pages), pages.numel() // 48, decay,
                                          _ptr(predicted), _ptr(out), _stream(stream)))
    return out


def decode_attn(pool, block_table, seq_lens, q, out=None, stats=None, page_mass=None, workspace=None,
                error_flag=None, sm_scale=0.0, stream=None):
    """Paged decode plus each page's attention mass ([batch][max_pages], mean
    over q-heads).  Returns (out, page_mass)."""
    torch = _torch()
    kv = paged(pool, stats)
    batch, hq, _ = q.shape
    mp = block_table.shape[1]
    if out is None:
        out = torch.empty_like(q)
    if page_mass is None:
        page_mass = torch.empty((batch, mp), dtype=torch.float32, device=q.device)
    if workspace is None:
        workspace = torch.zeros(lib.kvx_decode_attn_workspace_bytes(batch, hq, mp, PAGE_TOKENS),
                                dtype=torch.uint8, device=q.device)
    rc = lib.kvx_decode_attn(C.byref(kv), _ptr(block_table), mp, _ptr(seq_lens), batch, hq, _ptr(q), _ptr(out),
                             _dtype_code(q), sm_scale, _ptr(workspace), workspace.numel(), _ptr(page_mass),
                             _ptr(error_flag), _stream(stream))
    _check("kvx_decode_attn", rc)
    return out, page_mass


def attn_to_metrics(page_mass, block_table, seq_lens, metrics, current_token, stream=None):
    """Fold one step's page_mass into EvictionMetrics records (CUDA uint8
    tensor of 48-byte records indexed by physical page)."""
    rc = lib.kvx_attn_to_metrics(_ptr(page_mass), _ptr(block_table), block_table.shape[1], _ptr(seq_lens),
                                 block_table.shape[0], _ptr(metrics), metrics.numel() // 48, current_token,
                                 _stream(stream))
    _check("kvx_attn_to_metrics", rc)


# ---- rotary positions, ragged append, attention of several new tokens

ROPE_LAYOUT = {"half": 0, "interleaved": 1}
ROPE_SCALING = {"none": 0, "linear": 1, "ntk": 2, "llama3": 3, "yarn": 4}


# These calls are made once per layer and step, so their checks are plain
# comparisons and the message is only made when one fails.
#
# stream (None: the device's current one; a torch stream or its handle): where
# the call's work goes, outputs and scratch that the call makes itself included,
# which belong to it.  Order it with the streams of the other tensors.

def _require(cond, what):
    if not cond:
        raise ValueError(what)


_rt = None  # (float16, float32, int32, current raw stream of a device, current device)


def _runtime():
    global _rt
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
    _rt = (torch.float16, torch.float32, torch.int32, raw, getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device))
    return _rt


def _launch(dev, stream, fn, *args):
    """fn(*args, stream) with device `dev` current, so that a launch never
    lands on another device than its operands; stream None: that device's
    current one."""
    rt = _rt or _runtime()
    if dev == rt[4]():
        return fn(*args, rt[3](dev) if stream is None else stream if isinstance(stream, int) else stream.cuda_stream)
    with _torch().cuda.device(dev):
        return fn(*args, rt[3](dev) if stream is None else stream if isinstance(stream, int) else stream.cuda_stream)


def _on(stream, like):
    """Context for tensors that a call on `stream` makes itself: they belong to
    that stream, so their memory is free when its work reaches the call, a fill
    runs before the call's kernels, and memory given back is not taken by
    another stream while those run."""
    if stream is None or like.get_device() < 0:
        return contextlib.nullcontext()
    torch = _torch()
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=like.device) if isinstance(stream, int) else stream)


def _empty_like(x, stream):
    if stream is None:
        return _torch().empty(x.shape, dtype=x.dtype, device=x.device)
    with _on(stream, x):
        return _torch().empty(x.shape, dtype=x.dtype, device=x.device)


def _one_device(first, *others):
    """The CUDA device that all of these tensors (or None) lie on."""
    dev = first.get_device()
    if dev < 0:
        raise ValueError("tensors of one call lie on one CUDA device")
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError("tensors of one call lie on one CUDA device")
    return dev


def _vector(t, n, what):
    """An int32 tensor [n] (n None: any length), contiguous."""
    if t.dtype != (_rt or _runtime())[2] or t.dim() != 1 or not t.is_contiguous() or (n is not None and t.shape[0] != n):
        raise ValueError(what + ": contiguous int32" + ("" if n is None else f" [{n}]"))


def _flag(t):
    if t is None:
        return None
    if t.dtype != (_rt or _runtime())[2] or t.numel() < 1:
        raise ValueError("error_flag: int32, one element")
    return t.data_ptr()


def _io_code(x, what):
    rt = _rt or _runtime()
    if x.dtype == rt[0]:
        return KVX_F16
    if x.dtype == rt[1]:
        return KVX_F32
    raise ValueError(what + ": float16 or float32")


def _kept(name):
    """A property whose object stays: x.name += y of a tensor writes it in place,
    another object is refused."""
    held = "_" + name

    def keep(self, value):
        if value is not getattr(self, held):
            raise AttributeError(f"{name}: written in place, not replaced (the calls hold its address or value)")
    return property(lambda self: getattr(self, held), keep)


class RopeTable:
    """Frequencies of a rotary embedding on the device (see rope_table)."""

    turns, rotary_dim, layout, amplitude = _kept("turns"), _kept("rotary_dim"), _kept("layout"), _kept("amplitude")

    def __init__(self, turns, rotary_dim, layout, amplitude):
        _require(layout in ROPE_LAYOUT, f"layout: one of {sorted(ROPE_LAYOUT)}")
        _require(rotary_dim >= 2 and rotary_dim % 2 == 0, "rotary_dim: even, at least 2")
        _require(turns.dtype == _torch().int64 and turns.is_contiguous() and tuple(turns.shape) == (rotary_dim // 2,),
                 "turns: contiguous int64 [rotary_dim / 2]")
        self._turns, self._rotary_dim, self._layout, self._amplitude = turns, rotary_dim, layout, amplitude
        self.c = RopeTableC(turns.data_ptr(), rotary_dim, ROPE_LAYOUT[layout], amplitude)
        self.ref = C.byref(self.c)


def rope_frequencies(rotary_dim, base=10000.0, scaling="none", factor=1.0, low=1.0, high=4.0, original_context=8192.0):
    """(turns, amplitude): host list of rotary_dim / 2 angles per position in
    units of 2^-64 turns, and the factor on cosine and sine."""
    cfg = RopeConfig(rotary_dim, ROPE_SCALING[scaling], base, factor, low, high, original_context)
    turns, amplitude = (C.c_uint64 * max(rotary_dim // 2, 1))(), C.c_float()
    _check("kvx_rope_frequencies", lib.kvx_rope_frequencies(C.byref(cfg), turns, C.byref(amplitude)))
    return list(turns), amplitude.value


def rope_table(rotary_dim, base=10000.0, layout="half", scaling="none", factor=1.0, low=1.0, high=4.0,
               original_context=8192.0, device="cuda"):
    """Frequencies base^(-2i/rotary_dim), scaled for long contexts: "linear",
    "ntk", "llama3" (low / high: turns within original_context between which
    factor fades in) or "yarn" (low / high likewise, commonly 1 and 32)."""
    torch = _torch()
    _require(layout in ROPE_LAYOUT, f"layout: one of {sorted(ROPE_LAYOUT)}")
    _require(scaling in ROPE_SCALING, f"scaling: one of {sorted(ROPE_SCALING)}")
    turns, amplitude = rope_frequencies(rotary_dim, base, scaling, factor, low, high, original_context)
    signed = [t - (1 << 64) if t >> 63 else t for t in turns]
    return RopeTable(torch.tensor(signed, dtype=torch.int64).to(device), rotary_dim, layout, amplitude)


# kvx_rope_rows as bytes, one and two of them: a quarter of the time that
# ctypes takes to make the structures
_ROWS = {n: struct.Struct("@" + "QQi4xqqqq" * n) for n in (1, 2)}


def _rope_rows(x, out, what):
    """The fields of the RopeRows of a tensor [tokens][heads][dim] and its output."""
    sx, so = x.stride(), out.stride()
    shape = x.shape
    if len(shape) != 3 or (shape[2] > 1 and (sx[2] != 1 or so[2] != 1)):
        raise ValueError(what + ": [tokens][heads][dim], last dimension contiguous")
    if out.shape != shape or out.dtype != x.dtype:
        raise ValueError(what + "_out: shape and dtype of its input")
    if (so[0] == 0 and shape[0] > 1) or (so[1] == 0 and shape[1] > 1):
        raise ValueError(what + "_out: strides without overlap")
    return x.data_ptr(), out.data_ptr(), shape[1], sx[0], sx[1], so[0], so[1]


def rope(q, k, positions, table, q_out=None, k_out=None, inverse=False, stream=None):
    """Rotate q [tokens][hq][dim] and k [tokens][hk][dim] (k may be None) by
    positions [tokens] (int32); any token and head strides.  q_out = q rotates
    in place.  inverse=True turns back, which is the gradient of the rotation.
    Autograd records nothing here, so tensors that require a gradient are
    refused while it records: call under torch.no_grad(), or from the forward
    and backward of an autograd function.  Returns (q_out, k_out)."""
    if (q.requires_grad or (k is not None and k.requires_grad)) and _torch().is_grad_enabled():
        raise ValueError("q, k: a gradient would be lost here; call rope under torch.no_grad() or in an autograd function")
    if q_out is None:
        q_out = _empty_like(q, stream)
    rows = _rope_rows(q, q_out, "q")
    tokens, _, dim = q.shape
    n = 1
    if k is not None:
        if k_out is None:
            k_out = _empty_like(k, stream)
        rows += _rope_rows(k, k_out, "k")
        n = 2
        if k.shape[0] != tokens or k.shape[2] != dim or k.dtype != q.dtype:
            raise ValueError("k: tokens, dim and dtype of q")
    _vector(positions, tokens, "positions")
    code = _io_code(q, "q")
    dev = _one_device(q, q_out, k, k_out, positions, table.turns)
    rc = _launch(dev, stream, lib.kvx_rope, table.ref, positions.data_ptr(), tokens, dim, code, _ROWS[n].pack(*rows), n,
                 1 if inverse else 0)
    if rc:
        raise KvxError("kvx_rope", rc)
    return q_out, k_out


def _packed(x, heads, what):
    """Token stride of [tokens][heads][128] with the heads of a token side by side."""
    shape, st = x.shape, x.stride()
    if len(shape) != 3 or shape[2] != HEAD_DIM or (heads is not None and shape[1] != heads) or (
            shape[0] and (st[2] != 1 or (shape[1] > 1 and st[1] != HEAD_DIM))):
        raise ValueError(what + ": [tokens][heads][128], heads side by side")
    return st[0] if shape[0] > 1 else shape[1] * HEAD_DIM


def _ragged(block_table, q_start, positions):
    if block_table.dtype != (_rt or _runtime())[2] or block_table.dim() != 2 or not block_table.is_contiguous():
        raise ValueError("block_table: contiguous int32 [batch][max_pages]")
    batch, max_pages = block_table.shape
    _vector(positions, batch, "positions")
    _vector(q_start, batch + 1, "q_start")
    return batch, max_pages


def _pool(pool, stats):
    """paged(pool, stats), with the shapes of both checked, and the pool as a
    tensor (None for a KvPaged view)."""
    if isinstance(pool, KvPaged):
        return pool, None
    kv = paged(pool, stats)
    if kv.dtype == KVX_I8 and stats is None:
        raise ValueError("stats: an int8 pool has them")
    if stats is not None and (stats.dtype != (_rt or _runtime())[1] or not stats.is_contiguous() or
                              tuple(stats.shape) != (kv.num_pages, 2, kv.num_kv_heads, 4)):
        raise ValueError("stats: contiguous float32 [pages][2][hkv][4]")
    return kv, pool


def rope_append(pool, block_table, q_start, positions, k, v, q=None, q_out=None, table=None, stats=None, error_flag=None,
                stream=None):
    """Rotate and append a ragged batch: packed rows q_start[s] ..
    q_start[s+1]-1 of k, v ([tokens][hkv][128]) and q ([tokens][hq][128] or
    None) belong to sequence s and start at position positions[s].  k is
    rotated and stored with v in the pages (int8 pools: quantised, stats
    updated); q is rotated into q_out, which is returned.  table None: no
    rotation."""
    kv, tensor = _pool(pool, stats)
    batch, max_pages = _ragged(block_table, q_start, positions)
    tokens = k.shape[0]
    ks, vs = _packed(k, kv.num_kv_heads, "k"), _packed(v, kv.num_kv_heads, "v")
    code = _io_code(k, "k")
    if v.shape[0] != tokens or v.dtype != k.dtype:
        raise ValueError("v: tokens and dtype of k")
    hq = qs = 0
    q_ptr = out_ptr = None
    if q is not None:
        qs, hq = _packed(q, None, "q"), q.shape[1]
        if q.shape[0] != tokens or q.dtype != k.dtype:
            raise ValueError("q: tokens and dtype of k")
        if q_out is None:
            q_out = _empty_like(q, stream)
        if q_out.shape != q.shape or q_out.dtype != q.dtype or not q_out.is_contiguous():
            raise ValueError("q_out: contiguous, shape and dtype of q")
        q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out: only with q")
    dev = _one_device(k, v, q, q_out, block_table, q_start, positions, error_flag, tensor, stats,
                      None if table is None else table.turns)
    rc = _launch(dev, stream, lib.kvx_rope_append, C.byref(kv), block_table.data_ptr(), max_pages, q_start.data_ptr(),
                 positions.data_ptr(), batch, tokens, None if table is None else table.ref, code, q_ptr, qs, out_ptr, hq,
                 k.data_ptr(), ks, v.data_ptr(), vs, _flag(error_flag))
    if rc:
        raise KvxError("kvx_rope_append", rc)
    return q_out


def attend_chunk_workspace(batch, total_tokens, num_q_heads, num_kv_heads, max_pages, device="cuda"):
    """Scratch of attend_chunk for calls up to this size (no initialisation needed)."""
    n = lib.kvx_attend_chunk_workspace_bytes(batch, total_tokens, num_q_heads, num_kv_heads, max_pages)
    return _torch().empty(max(n, 16), dtype=_torch().uint8, device=device)


def attend_chunk(pool, block_table, q_start, positions, q, stats=None, out=None, workspace=None, error_flag=None,
                 sm_scale=0.0, causal=True, stream=None):
    """Attention of a ragged batch of new tokens over an int8 pool that holds
    them already: packed rows q [tokens][hq][128] as in rope_append; the query
    at position p sees keys 0 .. p (causal=False: every key of its sequence,
    positions[s] + its new tokens)."""
    kv, tensor = _pool(pool, stats)
    batch, max_pages = _ragged(block_table, q_start, positions)
    code = _io_code(q, "q")
    if q.dim() != 3 or q.shape[2] != HEAD_DIM or not q.is_contiguous():
        raise ValueError("q: contiguous [tokens][hq][128]")
    tokens, hq, _ = q.shape
    if out is None:
        with _on(stream, q):
            out = _torch().zeros_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError("out: contiguous, shape and dtype of q")
    if workspace is None:
        with _on(stream, q):
            workspace = attend_chunk_workspace(batch, tokens, hq, kv.num_kv_heads, max_pages, q.device)
    elif not workspace.is_contiguous():
        raise ValueError("workspace: contiguous")
    dev = _one_device(q, out, block_table, q_start, positions, workspace, error_flag, tensor, stats)
    rc = _launch(dev, stream, lib.kvx_attend_chunk, C.byref(kv), block_table.data_ptr(), max_pages, q_start.data_ptr(),
                 positions.data_ptr(), batch, tokens, hq, q.data_ptr(), out.data_ptr(), code, sm_scale, 1 if causal else 0,
                 workspace.data_ptr(), workspace.nbytes, _flag(error_flag))
    if rc:
        raise KvxError("kvx_attend_chunk", rc)
    return out
