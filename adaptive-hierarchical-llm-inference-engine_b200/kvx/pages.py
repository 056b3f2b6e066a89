"""Page bookkeeping on the device: ctypes front end of the kvx_pages_* calls
of include/kvx.h.

    pages = Pages.empty(num_pages, num_rows, max_pages, pools, stats)
    pages.reserve(new_tokens)           # pages for every row's next tokens
    pages.seq_lens += new_tokens        # once they are appended
    pages.fork(parents, children)       # samples / beams share a prefix
    pages.free(rows)                    # finished sequences
    pages.compact(num_live)             # live pages to the front of the pools

pools: the layers' page pools (CUDA tensors [pages][2][hkv][16][128], or
KvPaged views), which share the block table; stats: their statistics for int8
pools.  A refused call changes nothing and sets a bit of error_flag.
"""
from __future__ import annotations

import ctypes as C

from . import KvPaged, KvxError, _flag, _kept, _launch, _one_device, _pool, _require, _torch, _vector, lib

_vp, _i32, _sz = C.c_void_p, C.c_int32, C.c_size_t


class PagesC(C.Structure):
    _fields_ = [("refcounts", _vp), ("block_table", _vp), ("seq_lens", _vp), ("num_pages", _i32), ("num_rows", _i32),
                ("max_pages", _i32)]


_pp, _kp = C.POINTER(PagesC), C.POINTER(KvPaged)
lib.kvx_pages_workspace_bytes.argtypes = [_i32, _i32]
lib.kvx_pages_workspace_bytes.restype = _sz
lib.kvx_pages_reserve.argtypes = [_pp, _vp, _vp, _sz, _vp, _vp]
lib.kvx_pages_fork.argtypes = [_pp, _kp, _i32, _vp, _vp, _i32, _vp, _sz, _vp, _vp]
lib.kvx_pages_free.argtypes = [_pp, _vp, _i32, _vp, _vp]
lib.kvx_pages_compact.argtypes = [_pp, _kp, _i32, _vp, _sz, _vp, _vp, _vp]
lib.kvx_pages_copy.argtypes = [_kp, _i32, _vp, _vp, _i32, _vp, _vp]
for _fn in ("kvx_pages_reserve", "kvx_pages_fork", "kvx_pages_free", "kvx_pages_compact", "kvx_pages_copy"):
    getattr(lib, _fn).restype = C.c_int

ERR_RANGE, ERR_LONG, ERR_PAGES, ERR_ROWS = 2, 4, 8, 16  # bits of error_flag


class Pages:
    """The three arrays, the pools and the scratch of one set of pages.  The
    calls hold their addresses, so the tensors are written in place
    (pages.seq_lens += n, pages.block_table.copy_(t)) and never replaced."""

    refcounts, block_table, seq_lens = _kept("refcounts"), _kept("block_table"), _kept("seq_lens")
    pools, stats = _kept("pools"), _kept("stats")

    def __init__(self, refcounts, block_table, seq_lens, pools, stats=None):
        torch = _torch()
        _require(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.is_contiguous(),
                 "block_table: contiguous int32 [rows][max_pages]")
        _vector(refcounts, None, "refcounts")
        _vector(seq_lens, block_table.shape[0], "seq_lens")
        _require(stats is None or len(stats) == len(pools), "stats: one per pool")
        self._refcounts, self._block_table, self._seq_lens = refcounts, block_table, seq_lens
        self._pools, self._stats = tuple(pools), None if stats is None else tuple(stats)
        described = [_pool(p, None if stats is None else stats[i]) for i, p in enumerate(self._pools)]
        _require(all(kv.num_pages == refcounts.shape[0] for kv, _ in described), "refcounts: one per page of the pools")
        self._device = _one_device(refcounts, block_table, seq_lens, *(t for _, t in described), *(self._stats or ()))
        self._layers = (KvPaged * max(len(described), 1))(*(kv for kv, _ in described))
        self._pages = C.byref(PagesC(refcounts.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), refcounts.shape[0],
                                     block_table.shape[0], block_table.shape[1]))
        self._bytes = lib.kvx_pages_workspace_bytes(refcounts.shape[0], block_table.shape[0])
        self._workspace = torch.empty(max(self._bytes, 16), dtype=torch.uint8, device=refcounts.device)

    @classmethod
    def empty(cls, num_pages, num_rows, max_pages, pools, stats=None, device="cuda"):
        """Every page free, every row empty."""
        torch = _torch()
        return cls(torch.zeros(num_pages, dtype=torch.int32, device=device),
                   torch.full((num_rows, max_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(num_rows, dtype=torch.int32, device=device), pools, stats)

    def _run(self, fn, name, stream, tensors, *args):
        for t in tensors:
            if t is not None and t.get_device() != self._device:
                raise ValueError("tensors of one call lie on one CUDA device")
        rc = _launch(self._device, stream, fn, *args)
        if rc:
            raise KvxError(name, rc)

    def reserve(self, new_tokens, error_flag=None, stream=None):
        """Pages for the next new_tokens[row] tokens of every row."""
        _vector(new_tokens, self._block_table.shape[0], "new_tokens")
        self._run(lib.kvx_pages_reserve, "kvx_pages_reserve", stream, (new_tokens, error_flag), self._pages, new_tokens.data_ptr(),
                  self._workspace.data_ptr(), self._bytes, _flag(error_flag))

    def fork(self, parents, children, error_flag=None, stream=None):
        """Row children[i] (empty) becomes a copy of row parents[i]."""
        _vector(parents, None, "parents")
        n = parents.shape[0]
        _vector(children, n, "children")
        self._run(lib.kvx_pages_fork, "kvx_pages_fork", stream, (parents, children, error_flag), self._pages, self._layers,
                  len(self._pools), parents.data_ptr(), children.data_ptr(), n, self._workspace.data_ptr(), self._bytes,
                  _flag(error_flag))

    def free(self, rows, error_flag=None, stream=None):
        """Drop the pages of these rows."""
        _vector(rows, None, "rows")
        self._run(lib.kvx_pages_free, "kvx_pages_free", stream, (rows, error_flag), self._pages, rows.data_ptr(), rows.shape[0],
                  _flag(error_flag))

    def compact(self, num_live=None, error_flag=None, stream=None):
        """Move the held pages to the front; num_live (int32 [1]) gets their number."""
        if num_live is not None:
            _vector(num_live, 1, "num_live")
        self._run(lib.kvx_pages_compact, "kvx_pages_compact", stream, (num_live, error_flag), self._pages, self._layers,
                  len(self._pools), self._workspace.data_ptr(), self._bytes, None if num_live is None else num_live.data_ptr(),
                  _flag(error_flag))

    def copy(self, src, dst, error_flag=None, stream=None):
        """Page src[i] to page dst[i] in every layer."""
        _vector(src, None, "src")
        _vector(dst, src.shape[0], "dst")
        self._run(lib.kvx_pages_copy, "kvx_pages_copy", stream, (src, dst, error_flag), self._layers, len(self._pools), src.data_ptr(),
                  dst.data_ptr(), src.shape[0], _flag(error_flag))
