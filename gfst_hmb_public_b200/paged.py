"""Paged block memory: requests of ragged lengths in one pool of L-token blocks,
a prefix that all of them share, and the softmax attention that reads both.

``memory.BlockMemory`` gives every stream its own ring and moves all streams in
step; here a request holds as many blocks of the pool as its length needs,
takes and returns them on the GPU (no length is read back to the host), and the
blocks of a prefix that every request of the batch starts with (instructions, a
document) are stored once and attended for all requests in one product.

* ``block_tables``     one step of the tables: blocks taken and returned, the
                       slot of every new token, packed offsets
* ``paged_append``     the new tokens' keys and values to their slots
* ``prefix_attention`` attention of the new tokens over the prefix and over
                       each request's own positions, causal within the new ones
* ``PagedMemory``      pool, tables, lengths and prefix of a batch of requests

Layout: pool_K [n_blocks, heads, L, d], pool_V [n_blocks, heads, L, dv]; a block
of one head is one contiguous L x d slab, as in ``memory.BlockMemory``.  Slot
``block * L + offset`` names a token's place in the pool.

Serving operators: nothing here records gradients, and tensors that ask for
them (or carry forward-mode tangents) are refused.  The reference
(pkhairkh/gfst-hmb-public) keeps one Python list of blocks per sample
(src/gfst_hmb_mpuc/state.py:651-815) and has no shared prefix.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _native as nat

_ENTRY: dict = {}  # entry points by name, as the loaded library gives them
_I32 = torch.int32
_DTYPES = {torch.float32: nat.DTYPE_F32, torch.bfloat16: nat.DTYPE_BF16, torch.float16: nat.DTYPE_F16}


def _dtype_code(what: str, *tensors: torch.Tensor) -> int:
    dtype = tensors[0].dtype
    for t in tensors:
        if t.dtype is not dtype:
            raise RuntimeError(f"{what}: mixed dtypes {({t.dtype for t in tensors})}")
    if dtype not in _DTYPES:
        raise RuntimeError(f"{what}: unsupported dtype {dtype} (float32, bfloat16 or float16)")
    return _DTYPES[dtype]


def _no_grad(what: str, *tensors: torch.Tensor | None) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no backward pass; call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} has no forward-mode derivative; pass tensors without tangents")


def _cuda(what: str, *tensors: torch.Tensor | None) -> int:
    """Index of the CUDA device that holds every given tensor; raises as nat.require_cuda does."""
    try:
        index = tensors[0].get_device()  # -1: not on a GPU
        if index >= 0:
            for t in tensors:
                if t is not None and t.get_device() != index:
                    break
            else:
                return index
    except AttributeError:  # no tensor
        pass
    return nat.require_cuda(*tensors, what=what).index


def _call(index: int, name: str, *args) -> None:
    """Entry point ``name`` on device ``index`` and its current stream."""
    fn = _ENTRY.get(name)
    if fn is None:
        fn = _ENTRY[name] = getattr(nat.load(), name)
    stream = torch._C._cuda_getCurrentRawStream(index)  # current_stream(index).cuda_stream, without its 1.2 us
    if torch.cuda.current_device() == index:
        status = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            status = fn(*args, stream)
    if status != nat.GFST_OK:
        nat.check(status, name)


def _int32(what: str, name: str, t: torch.Tensor, shape: tuple) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise RuntimeError(f"{what}: {name} must be int32 (got {t.dtype})")
    if t.shape != shape:
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {shape}")
    return t if t.is_contiguous() else t.contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [n, heads, width] with contiguous 16-byte aligned rows (a copy where it has none)."""
    per = 16 // t.element_size()
    a, b, c = t.stride()
    if c == 1 and a % per == 0 and b % per == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.contiguous().clone() if t.is_contiguous() else t.contiguous()


@functools.lru_cache(maxsize=256)
def _workspace_bytes(n: int, heads: int, group: int, dv: int) -> int:
    nbytes = ctypes.c_size_t(0)
    nat.check(nat.load().gfst_prefix_attention_workspace_bytes(n, heads, group, dv, ctypes.byref(nbytes)),
              "gfst_prefix_attention_workspace_bytes")
    return int(nbytes.value)


class BlockTables(NamedTuple):
    """What one step of ``block_tables`` leaves (all int32 on the device)."""
    tables: torch.Tensor      # [B, W] blocks of each request, -1 behind them
    lens: torch.Tensor        # [B] tokens of each request, the new ones included
    cu_new: torch.Tensor      # [B + 1] first packed position of each request's new tokens
    slot_map: torch.Tensor    # [n_tokens] slot of each new token, -1 behind the last
    free_state: torch.Tensor  # [2] (head, count) of the free ring
    n_short: torch.Tensor     # [1] blocks wanted and not had: 0 in a step that may be used


def block_tables(lens: torch.Tensor, new_lens: torch.Tensor, tables: torch.Tensor, free_ring: torch.Tensor,
                 free_state: torch.Tensor, *, block_len: int, n_tokens: int,
                 tables_out: torch.Tensor | None = None) -> BlockTables:
    """One step of the block tables, on the GPU.

    lens [B] tokens of each request and tables [B, W] its blocks; new_lens [B]
    the tokens it appends (0: idle, negative: the request ends and returns its
    blocks); free_ring [n_blocks] with free_state [2] = (head, count) the free
    blocks.  Blocks are taken in request order from the ring's head; returned
    ones go behind its tail and are handed out from the next step on.
    ``free_ring`` is updated in place (only behind the tail, so a step that is
    not used can be taken again from the same lens, tables and free_state).
    ``n_tokens`` is the number of packed new tokens the caller holds, at least
    the sum of the positive new_lens.  ``tables_out`` (may be ``tables``)
    receives the new tables in place of a new tensor.  All int32.

    A step that wants more blocks than there are has n_short > 0 and is not to
    be used; in place (``tables_out`` is ``tables``) it changes nothing, and no
    token of it has a slot.  So does a step in place with more new tokens than
    ``n_tokens``: n_short counts them too."""
    what = "block_tables"
    index = _cuda(what, lens, new_lens, tables, free_ring, free_state, tables_out)
    if tables.ndim != 2 or free_ring.ndim != 1:
        raise ValueError("block_tables expects tables [B, W] and free_ring [n_blocks]")
    B, W = tables.shape
    n = int(n_tokens)
    if not (lens.dtype is new_lens.dtype is free_state.dtype is _I32 and lens.shape == new_lens.shape == (B,) and
            free_state.shape == (2,) and lens.is_contiguous() and new_lens.is_contiguous() and
            free_state.is_contiguous()):
        lens, new_lens = _int32(what, "lens", lens, (B,)), _int32(what, "new_lens", new_lens, (B,))
        free_state = _int32(what, "free_state", free_state, (2,))
    if free_ring.dtype != torch.int32 or not free_ring.is_contiguous():
        raise RuntimeError("block_tables: free_ring must be contiguous int32")
    if n < 0:
        raise ValueError(f"block_tables: n_tokens {n} is negative")
    if tables_out is None:
        tables = _int32(what, "tables", tables, (B, W))
    else:
        if not (tables.is_contiguous() and tables_out.is_contiguous()):
            raise ValueError("block_tables: tables and tables_out must be contiguous")
        _int32(what, "tables", tables, (B, W))
        _int32(what, "tables_out", tables_out, (B, W))
        a, b, size = tables.data_ptr(), tables_out.data_ptr(), B * W * 4
        if a != b and a < b + size and b < a + size:
            raise ValueError("block_tables: tables_out overlaps tables without being it")
    # one buffer for all that is new; the slots first, at an allocation's alignment
    sizes = [n, B, B + 1, 2, 1]
    if tables_out is None:
        sizes.append(B * W)
    buffer = lens.new_empty((n + 2 * B + 4 + (B * W if tables_out is None else 0),))
    cut = torch.split_with_sizes(buffer, sizes)
    if tables_out is None:
        tables_out = cut[5].view(B, W)
    at_slots = buffer.data_ptr()
    at_lens = at_slots + 4 * n
    at_cu = at_lens + 4 * B
    at_state = at_cu + 4 * (B + 1)
    _call(index, "gfst_block_tables", lens.data_ptr(), new_lens.data_ptr(), tables.data_ptr(), free_ring.data_ptr(),
          free_state.data_ptr(), B, W, int(block_len), free_ring.shape[0], n, tables_out.data_ptr(), at_lens, at_cu,
          at_slots, at_state, at_state + 8)
    return BlockTables(tables_out, cut[1], cut[2], cut[0], cut[3], cut[4])


def _check_pools(what: str, pool_K: torch.Tensor, pool_V: torch.Tensor) -> tuple:
    k, v = pool_K.shape, pool_V.shape
    if len(k) != 4 or len(v) != 4 or k[0] != v[0] or k[1] != v[1] or k[2] != v[2] or k[1] == 0:
        raise ValueError(f"{what} expects pool_K [n_blocks, heads, L, d] and pool_V [n_blocks, heads, L, dv]")
    if not (pool_K.is_contiguous() and pool_V.is_contiguous()):
        raise ValueError(f"{what}: pools must be contiguous")
    return (*k, v[3])


def paged_append(K: torch.Tensor, V: torch.Tensor, pool_K: torch.Tensor, pool_V: torch.Tensor,
                 slot_map: torch.Tensor) -> None:
    """Write K [n, heads, d] and V [n, heads, dv] to their slots of the pools:
    pool[s // L, h, s % L] = row (t, h) with s = slot_map[t] (int32 [n]).  Tokens
    with a negative slot (padding, or a block that was not had) are left out, and
    so is a slot outside the pool; nothing else of the pools changes.  The slots
    that are written must be distinct, as ``block_tables`` gives them.  K and V
    may be strided views (a fused projection's output) with 16-byte rows, but not
    of the pools themselves."""
    what = "paged_append"
    index = _cuda(what, K, V, pool_K, pool_V, slot_map)
    n_blocks, H, L, d, dv = _check_pools(what, pool_K, pool_V)
    if K.ndim != 3 or V.ndim != 3 or K.shape[1:] != (H, d) or V.shape != (K.shape[0], H, dv):
        raise ValueError(f"paged_append: K{tuple(K.shape)} V{tuple(V.shape)} do not match pools of {H} heads, "
                         f"d={d}, dv={dv}")
    code = _dtype_code(what, K, V, pool_K, pool_V)
    _no_grad(what, K, V, pool_K, pool_V)
    n = K.shape[0]
    slot_map = _int32(what, "slot_map", slot_map, (n,))
    K, V = _rows(K), _rows(V)
    kt, kh, _ = K.stride()
    vt, vh, _ = V.stride()
    _call(index, "gfst_paged_append", K.data_ptr(), kt, kh, V.data_ptr(), vt, vh, pool_K.data_ptr(), pool_V.data_ptr(),
          slot_map.data_ptr(), n, n_blocks, L, H, d, dv, code)


def prefix_attention(Q: torch.Tensor, pool_K: torch.Tensor, pool_V: torch.Tensor, tables: torch.Tensor,
                     lens: torch.Tensor, cu_new: torch.Tensor, *, prefix_table: torch.Tensor | None = None,
                     prefix_len: torch.Tensor | None = None, scale: float | None = None,
                     out: torch.Tensor | None = None, return_lse: bool = False):
    """Softmax attention of the new tokens over a shared prefix and over each
    request's own positions.

    Q [n, heads * group, d] in packed order (query head hq reads KV head hq //
    group; rows may be strided); pools as ``paged_append`` writes them; tables
    [B, W], lens [B] and cu_new [B + 1] as ``block_tables`` leaves them (lens
    counts the new tokens, whose keys are already in the pool); prefix_table
    [P] int32 and prefix_len [1] int32 (on the device): the blocks and length of
    the prefix, or None.  The i-th of a request's n_b new tokens sees the whole
    prefix and its own positions up to lens[b] - n_b + i.  ``scale`` defaults to
    d ** -0.5.

    Returns (out [n, heads * group, dv], lse float32 [n, heads * group] or
    None).  A token that sees nothing gets zeros and -inf.  Tokens behind
    cu_new[B] (a padded batch) get the same; with ``out`` given (contiguous,
    Q's dtype) their rows of it stay as they were, and lse is -inf.  A table entry outside the
    pool within a request's length reads as zero keys and values and is
    reported by ``_native.check_device_errors``.  Keys and values that no token
    sees may hold anything; one that is not finite and is seen makes columns of
    the row inf or NaN.  Each call takes a workspace of 8 (dv + 4) bytes per row
    of ``out`` and 42 MB (dv 128) from the caching allocator."""
    what = "prefix_attention"
    index = _cuda(what, Q, pool_K, pool_V, tables, lens, cu_new, prefix_table, prefix_len, out)
    n_blocks, H, L, d, dv = _check_pools(what, pool_K, pool_V)
    if Q.ndim != 3 or Q.shape[2] != d or Q.shape[1] % H != 0 or Q.shape[1] == 0:
        raise ValueError(f"prefix_attention: Q{tuple(Q.shape)} does not match pools of {H} heads, d={d}")
    if tables.ndim != 2:
        raise ValueError("prefix_attention expects tables [B, W]")
    n, heads, _ = Q.shape
    B, W = tables.shape
    if tables.dtype != torch.int32:
        raise RuntimeError("prefix_attention: tables must be int32")
    if W > 0 and tables.stride(1) != 1:
        tables = tables.contiguous()
    if not (lens.dtype is cu_new.dtype is _I32 and lens.shape == (B,) and cu_new.shape == (B + 1,) and
            lens.is_contiguous() and cu_new.is_contiguous()):
        lens, cu_new = _int32(what, "lens", lens, (B,)), _int32(what, "cu_new", cu_new, (B + 1,))
    if (prefix_table is None) != (prefix_len is None):
        raise ValueError("prefix_attention: prefix_table and prefix_len go together")
    P, p_table, p_len = 0, None, None
    if prefix_table is not None:
        P = prefix_table.numel()
        if not (prefix_table.dtype is prefix_len.dtype is _I32 and prefix_len.shape == (1,) and
                prefix_table.ndim == 1 and prefix_table.is_contiguous()):
            prefix_table = _int32(what, "prefix_table", prefix_table, (P,))
            prefix_len = _int32(what, "prefix_len", prefix_len, (1,))
        p_table, p_len = prefix_table.data_ptr(), prefix_len.data_ptr()
    code = _dtype_code(what, Q, pool_K, pool_V)
    _no_grad(what, Q, pool_K, pool_V, out)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"prefix_attention: scale {scale} is not finite")
    given = out is not None
    if given:
        if out.shape != (n, heads, dv) or out.dtype != Q.dtype or not out.is_contiguous():
            raise ValueError(f"prefix_attention: out must be contiguous {Q.dtype} [{n}, {heads}, {dv}]")
    else:
        out = Q.new_empty((n, heads, dv))
    lse = Q.new_empty((n, heads), dtype=torch.float32) if return_lse else None
    Q = _rows(Q)
    qt, qh, _ = Q.stride()
    nbytes = _workspace_bytes(n, H, heads // H, dv)
    ws = tables.new_empty(((nbytes + 3) // 4,))
    _call(index, "gfst_prefix_attention", Q.data_ptr(), qt, qh, pool_K.data_ptr(), pool_V.data_ptr(), n_blocks, L, H,
          heads // H, d, dv, code, tables.data_ptr(), tables.stride(0), W, lens.data_ptr(), cu_new.data_ptr(), B, n,
          p_table, P, p_len, scale, out.data_ptr(), nat.ptr(lse), 0 if given else 1, ws.data_ptr(), nbytes)
    return out, lse


class PagedMemory:
    """Pool, block tables, lengths and shared prefix of up to ``max_requests``
    requests, each of up to ``max_blocks`` blocks (``n_layers`` pools share the
    tables).  A request is an index in [0, max_requests); every step passes one
    entry per index (0: idle, negative: ends).

    A step: ``step = mem.extend(new_lens, n_tokens)``; then for every layer
    ``mem.append(K, V, step, layer)`` and ``mem.attend(Q, step, layer=layer)``.
    A step's tables and lengths are the memory's own: it is over with the next
    ``extend``, ``share``, ``unshare`` or ``reset``.
    Lengths and tables stay on the GPU; shapes depend on ``n_tokens`` alone, so a
    step can be captured in a CUDA graph and replayed with new ``new_lens`` in
    the same tensor (tokens behind the last request are padding)."""

    def __init__(self, n_blocks: int, block_len: int, n_heads: int, d: int, dv: int | None = None, *,
                 max_requests: int, max_blocks: int, n_layers: int = 1, dtype: torch.dtype = torch.bfloat16,
                 device="cuda"):
        if dtype not in _DTYPES:
            raise RuntimeError(f"PagedMemory: unsupported dtype {dtype} (float32, bfloat16 or float16)")
        if min(n_blocks, block_len, n_heads, d, max_requests, max_blocks, n_layers) < 1:
            raise ValueError("PagedMemory: sizes must be positive")
        dv = d if dv is None else dv
        self.n_blocks, self.block_len, self.n_heads, self.d, self.dv = n_blocks, block_len, n_heads, d, dv
        self.max_requests, self.max_blocks, self.n_layers, self.dtype = max_requests, max_blocks, n_layers, dtype
        i32 = dict(dtype=torch.int32, device=device)
        self.pool_K = torch.zeros((n_layers, n_blocks, n_heads, block_len, d), dtype=dtype, device=device)
        self.pool_V = torch.zeros((n_layers, n_blocks, n_heads, block_len, dv), dtype=dtype, device=device)
        self.tables = torch.full((max_requests, max_blocks), -1, **i32)
        self.lens = torch.zeros((max_requests,), **i32)
        self.free_ring = torch.arange(n_blocks, **i32)
        self.free_state = torch.tensor([0, n_blocks], **i32)
        self.prefix_table = torch.full((max_blocks,), -1, **i32)
        self.prefix_len = torch.zeros((1,), **i32)

    @property
    def device(self) -> torch.device:
        return self.pool_K.device

    def extend(self, new_lens: torch.Tensor, n_tokens: int) -> BlockTables:
        """Take and return blocks for one step; updates the memory's tables,
        lengths and free ring in place and returns the step (whose ``tables`` and
        ``lens`` are the memory's own).  ``n_tokens`` is at least the sum of the
        positive new_lens.  ``n_short`` of the step says how many blocks the pool,
        and how many tokens ``n_tokens``, was short of; read it when the host waits
        anyway.  A step with n_short > 0 did nothing: no request grew or ended, its
        tokens have no slots and attend to nothing.  End a request (or pass more
        tokens) and take it again."""
        t = block_tables(self.lens, new_lens, self.tables, self.free_ring, self.free_state,
                         block_len=self.block_len, n_tokens=n_tokens, tables_out=self.tables)
        self.lens.copy_(t.lens)
        self.free_state.copy_(t.free_state)
        return t._replace(lens=self.lens, free_state=self.free_state)

    def append(self, K: torch.Tensor, V: torch.Tensor, step: BlockTables, layer: int = 0) -> None:
        """Keys and values [n_tokens, heads, d / dv] of the step's new tokens."""
        paged_append(K, V, self.pool_K[layer], self.pool_V[layer], step.slot_map)

    def attend(self, Q: torch.Tensor, step: BlockTables, *, layer: int = 0, scale: float | None = None,
               out: torch.Tensor | None = None, return_lse: bool = False):
        """Attention of the step's new tokens, Q [n_tokens, heads * group, d]
        (``prefix_attention``); append the step's keys first."""
        return prefix_attention(Q, self.pool_K[layer], self.pool_V[layer], step.tables, step.lens, step.cu_new,
                                prefix_table=self.prefix_table, prefix_len=self.prefix_len, scale=scale, out=out,
                                return_lse=return_lse)

    def share(self, request: int) -> None:
        """Make request ``request``'s tokens the prefix of all requests: its blocks
        become the prefix's and the index is free again.  The prefix must be
        empty (``unshare`` first) and the other requests are then taken to
        continue it."""
        r = self._index(request)
        if int(self.prefix_len.item()) != 0:
            raise RuntimeError("PagedMemory.share: there is a prefix already; unshare it first")
        self.prefix_table.copy_(self.tables[r])
        self.prefix_len.copy_(self.lens[r:r + 1])
        self.tables[r].fill_(-1)
        self.lens[r:r + 1].zero_()

    def unshare(self, request: int) -> None:
        """Give the prefix's blocks and tokens to the idle request index
        ``request`` (end it to return the blocks)."""
        r = self._index(request)
        if int(self.lens[r].item()) != 0:
            raise RuntimeError(f"PagedMemory.unshare: request {r} holds tokens")
        self.tables[r].copy_(self.prefix_table)
        self.lens[r:r + 1].copy_(self.prefix_len)
        self.prefix_table.fill_(-1)
        self.prefix_len.zero_()

    def reset(self) -> None:
        """Forget every request and the prefix (the pools keep their bytes)."""
        self.tables.fill_(-1)
        self.prefix_table.fill_(-1)
        self.lens.zero_()
        self.prefix_len.zero_()
        self.free_ring.copy_(torch.arange(self.n_blocks, dtype=torch.int32, device=self.device))
        self.free_state.copy_(torch.tensor([0, self.n_blocks], dtype=torch.int32))

    def _index(self, request: int) -> int:
        r = int(request)
        if not 0 <= r < self.max_requests:
            raise ValueError(f"PagedMemory: request {r} outside [0, {self.max_requests})")
        return r
