"""Tree drafts and 8-bit KV caches: the Python face of the ``eesd_tree_*``, ``eesd_kv_*`` and
``eesd_attn_tree`` primitives of ``include/eesd.h``.

One round of a step whose drafts form a tree::

    cache = KVCache(n_layers, max_batch, n_kv_heads, max_seq, head_dim, "int8")
    tree = TreeBatch([(row, ctx, parents), ...], cache)          # once per round
    ws = attention_workspace(tree, cache, n_heads)
    for layer in range(n_layers):
        kv_append(qkv, cache, tree, cos, sin, q_out=q, layer=layer)
        tree_attention(q, cache, tree, out, layer=layer, workspace=ws)
    tree_accept(y, ids, tree, path, n_acc, next_ids)             # y: the head's tokens of all nodes
    kv_compact(cache, tree, path, n_acc)                         # all layers
    tree.check()                                                 # raises what the device found wrong

Everything is enqueued on the current stream of the tensors' device and nothing synchronises but
``check``.  A ``parents`` entry may be a node count instead of a list: a chain (a prefill chunk, a decode
step).  The reference drafts chains over an unquantised cache (solutions/packed.py:142-196,
solutions/engine.py:453-475); a chain over a cache in the model dtype computes the same.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np
import torch

from . import lib
from .model import DTYPES

FORMATS = {"bf16": (lib.KV_MODEL, torch.bfloat16), "f32": (lib.KV_MODEL, torch.float32),
           "e4m3": (lib.KV_E4M3, torch.float8_e4m3fn), "int8": (lib.KV_INT8, torch.int8)}
_FORMAT_OF = {dt: name for name, (_, dt) in FORMATS.items()}


_raw_stream = torch._C._cuda_getCurrentRawStream     # current_stream() builds a Stream object first
_current_device = torch._C._cuda_getDevice
_fn = {}


def _call(dev: torch.device, name: str, *args) -> None:
    """``lib.call`` with ``dev`` current and its current stream as the last argument."""
    fn = _fn.get(name)
    if fn is None:
        fn = _fn[name] = getattr(lib.load(), name)
    i = dev.index
    if _current_device() == i:
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(i))
    if rc:
        lib.check(rc, name)
    lib.direct_launches += 1


def _need(t: torch.Tensor, what: str, dev: torch.device, dtype, shape=None) -> int:
    """Address of ``t``, checked."""
    if t.dtype is not dtype or t.device != dev or not t.is_contiguous() or (shape is not None and t.shape != shape):
        raise ValueError(f"{what}: need a contiguous {dtype} tensor {list(shape) if shape else ''} on {dev}, "
                         f"got {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


class KVCache:
    """K and V of all layers, ``[n_layers, max_batch, n_kv_heads, max_seq, head_dim]``, in the model dtype
    ("bf16", "f32") or in 8 bits ("e4m3", "int8") with one power-of-two exponent byte per vector
    (``k_exp``, ``v_exp``: ``[n_layers, max_batch, n_kv_heads, max_seq]``)."""

    def __init__(self, n_layers: int, max_batch: int, n_kv_heads: int, max_seq: int, head_dim: int, fmt: str = "bf16",
                 device="cuda"):
        if fmt not in FORMATS:
            raise ValueError(f"cache format {fmt!r} (one of {sorted(FORMATS)})")
        shape = (n_layers, max_batch, n_kv_heads, (max_seq + 63) // 64 * 64, head_dim)
        dt = FORMATS[fmt][1]
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dt) if dt.itemsize == 1 else
                torch.zeros(shape, dtype=dt, device=device) for _ in range(2))
        ke, ve = (torch.full(shape[:4], 27, dtype=torch.uint8, device=device) for _ in range(2)) if dt.itemsize == 1 else (None, None)
        self._set(k, v, ke, ve)

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor, k_exp: Optional[torch.Tensor] = None,
             v_exp: Optional[torch.Tensor] = None) -> "KVCache":
        """A cache over existing tensors (e.g. ``DeviceModel.k_cache`` and ``v_cache``), without copying."""
        c = cls.__new__(cls)
        c._set(k, v, k_exp, v_exp)
        return c

    def _set(self, k, v, ke, ve) -> None:
        if k.device.type != "cuda":
            raise ValueError("the KV cache must be on a CUDA device: there is no other compute path")
        if k.dim() != 5 or k.dtype not in _FORMAT_OF:
            raise ValueError(f"k: need a 5-d tensor of one of {sorted(FORMATS)}, got {k.dtype} {list(k.shape)}")
        _need(k, "k", k.device, k.dtype)
        _need(v, "v", k.device, k.dtype, tuple(k.shape))
        self.format = _FORMAT_OF[k.dtype]
        self.k, self.v, self.k_exp, self.v_exp = k, v, ke, ve
        self.device = k.device
        self.quantised = k.dtype.itemsize == 1
        self._dtypes = DTYPES if self.quantised else {k.dtype: DTYPES[k.dtype]}
        if self.quantised:
            for t, what in ((ke, "k_exp"), (ve, "v_exp")):
                if t is None:
                    raise ValueError(f"an 8-bit cache needs {what}")
                _need(t, what, k.device, torch.uint8, tuple(k.shape[:4]))
        L, B, H, S, D = k.shape
        self.n_layers, self.max_batch, self.n_kv_heads, self.max_seq, self.head_dim = L, B, H, S, D
        self.struct = lib.KvCache(FORMATS[self.format][0], L, B, H, S, D, k.data_ptr(), v.data_ptr(),
                                  lib.ptr(ke if self.quantised else None), lib.ptr(ve if self.quantised else None))
        self.ref = C.byref(self.struct)

    def model_dtype(self, t: torch.Tensor, what: str) -> int:
        """The library's dtype of an activation tensor that goes with this cache."""
        dt = self._dtypes.get(t.dtype)
        if dt is None or t.device != self.device:
            raise ValueError(f"{what}: {t.dtype} on {t.device} does not go with a {self.format} cache on {self.device}")
        return dt


class TreeBatch:
    """The blocks of one round on the device.  ``blocks``: ``(row, ctx, parents)`` each, ``parents`` a list with
    ``parents[i] < i`` (-1: a child of the committed context) or a node count (a chain).  Node i sits at cache
    slot ``ctx + i`` and at position ``ctx + depth``.  A batch of chains only has no mask and any number of
    nodes; with a tree in it a block has at most 256 nodes.

    ``blk`` [n_blocks, 4] = (start, T, row, ctx), ``parent``, ``tok_pos``, ``tok_slot``, ``tok_row`` [n_tokens]
    int32 and ``mask`` [n_tokens, words] int64 are device tensors.  A program that advances ``ctx`` on the device
    edits ``blk`` and calls ``update``; ``max_ctx`` (default: the largest ``ctx + T`` given) has to bound ``ctx + T``
    from then on too, as ``max_nodes`` does T.  A block may become shorter: tokens of no block are padding, with -1 for
    position, slot and row, neither written nor read."""

    def __init__(self, blocks: Sequence[tuple], cache: KVCache, max_ctx: Optional[int] = None, max_nodes: Optional[int] = None):
        blk, par, chains, start = [], [], True, 0
        for row, ctx, parents in blocks:
            T = parents if isinstance(parents, (int, np.integer)) else len(parents)
            if T < 1 or not 0 <= row < cache.max_batch or ctx < 0 or ctx + T > cache.max_seq:
                raise ValueError(f"block (row {row}, ctx {ctx}, {T} nodes) does not fit a cache of {cache.max_batch} rows "
                                 f"x {cache.max_seq} slots")
            if isinstance(parents, (int, np.integer)):
                par.append(np.arange(-1, T - 1, dtype=np.int32))
            else:
                p = np.asarray(parents, dtype=np.int32)
                if p.ndim != 1 or (p < -1).any() or (p >= np.arange(T)).any():
                    raise ValueError("parents: need -1 <= parents[i] < i")
                par.append(p)
                chains = False
            blk.append((start, T, row, ctx))
            start += T
        self.n_blocks, self.n_tokens = len(blk), start
        if not blk:
            raise ValueError("a tree batch needs at least one block")
        self.max_nodes = max(max(b[1] for b in blk), max_nodes or 1)
        self.max_ctx = max(max(b[1] + b[3] for b in blk), max_ctx or 1)
        if not chains and self.max_nodes > lib.TREE_MAX_NODES:
            raise ValueError(f"a tree has at most {lib.TREE_MAX_NODES} nodes per block, got {self.max_nodes}")
        self.device, self._cache = cache.device, cache
        n, nb, W = self.n_tokens, self.n_blocks, 0 if chains else (self.max_nodes + 63) // 64
        host = np.concatenate([np.asarray(blk, dtype=np.int32).reshape(-1), *par])
        up = torch.from_numpy(host).pin_memory().to(self.device, non_blocking=True)
        ints = torch.empty(3 * n + 1, dtype=torch.int32, device=self.device)
        self.blk, self.parent = up[:4 * nb].view(nb, 4), up[4 * nb:]
        self.tok_pos, self.tok_slot, self.tok_row = ints[:n], ints[n:2 * n], ints[2 * n:3 * n]
        self.status = ints[3 * n:].zero_()
        self.mask = torch.empty(n, W, dtype=torch.int64, device=self.device) if W else None
        self.struct = lib.Tree(n, nb, self.max_nodes, self.max_ctx, W, 0, self.blk.data_ptr(),
                               None if chains else self.parent.data_ptr(), self.tok_pos.data_ptr(), self.tok_slot.data_ptr(),
                               self.tok_row.data_ptr(), lib.ptr(self.mask))
        self.ref = C.byref(self.struct)
        self.ptr_pos, self.ptr_slot, self.ptr_row = self.tok_pos.data_ptr(), self.tok_slot.data_ptr(), self.tok_row.data_ptr()
        self.ptr_status = self.status.data_ptr()
        self.update()

    def on(self, cache: "KVCache") -> "TreeBatch":
        """The batch itself, if it is on the cache's device."""
        if self.device != cache.device:
            raise ValueError(f"a batch on {self.device} and a cache on {cache.device}")
        return self

    def update(self) -> None:
        """Positions, slots, rows and the mask from ``blk`` and ``parent`` (one launch)."""
        _call(self.device, "eesd_tree_meta", self.ref, self._cache.max_batch, self._cache.max_seq, self.ptr_status)

    def check(self) -> None:
        """Raise if a call on this batch met a bad block, row, slot or path, or a wait that gave up; synchronises."""
        bits = C.c_int(0)
        with torch.cuda.device(self.device):
            rc = lib.load().eesd_status_read(self.status.data_ptr(), C.byref(bits), torch.cuda.current_stream().cuda_stream)
            if rc == lib.ERR_DEVICE:
                self.status.zero_()
            lib.check(rc, f"device status (bits 0x{bits.value:x})")


def kv_append(qkv: torch.Tensor, cache: KVCache, tree: TreeBatch, rope_cos: torch.Tensor, rope_sin: torch.Tensor,
              q_out: Optional[torch.Tensor] = None, layer: int = 0) -> None:
    """RoPE of q and k of ``qkv`` [n_tokens, (Hq + 2 Hkv) D] (rows may be strided) and the (quantising) append of k
    and v.  The rotated q goes to ``q_out`` [n_tokens, Hq D], or back into ``qkv``."""
    dt = cache.model_dtype(qkv, "qkv")
    D, dev, n = cache.head_dim, cache.device, tree.on(cache).n_tokens
    n_heads = _heads(qkv, "qkv", n, D) - 2 * cache.n_kv_heads
    cos = _need(rope_cos, "rope_cos", dev, torch.float32)
    sin = _need(rope_sin, "rope_sin", dev, torch.float32, rope_cos.shape)
    if rope_cos.dim() != 2 or rope_cos.shape[1] != D:
        raise ValueError(f"RoPE tables: need [positions, {D}]")
    q = None if q_out is None else _need(q_out, "q_out", dev, qkv.dtype, (n, n_heads * D))
    _call(dev, "eesd_kv_append", dt, cache.ref, layer, qkv.data_ptr(), _row_stride(qkv), n_heads, tree.ptr_pos, tree.ptr_slot,
          tree.ptr_row, n, cos, sin, rope_cos.shape[0], q, tree.ptr_status)


def _heads(t: torch.Tensor, what: str, n: int, D: int) -> int:
    """Heads in the rows of ``t``: [n, heads D] with unit stride in a row."""
    if t.dim() != 2 or t.shape[0] != n or t.stride(1) != 1 or t.shape[1] % D:
        raise ValueError(f"{what}: need [{n}, heads x {D}] rows with unit stride, got {list(t.shape)}")
    return t.shape[1] // D


def _row_stride(t: torch.Tensor) -> int:
    if t.shape[0] == 1:
        return t.shape[1]
    if t.stride(0) >= 2 ** 31:                           # ctypes would cut it to 32 bits
        raise ValueError(f"rows {t.stride(0)} elements apart: at most 2^31 - 1")
    return t.stride(0)


def kv_read(cache: KVCache, tok_row: torch.Tensor, tok_slot: torch.Tensor, k_out: Optional[torch.Tensor],
            v_out: Optional[torch.Tensor], layer: int = 0, status: Optional[torch.Tensor] = None) -> None:
    """``k_out`` / ``v_out`` [n, Hkv, D] (bf16 or f32; either may be None) = the cached values at
    (tok_row[i], tok_slot[i]).  An index out of range leaves its output as it was and sets ``status``."""
    some = k_out if k_out is not None else v_out
    if some is None:
        raise ValueError("kv_read: both outputs are None")
    dt, dev, n = cache.model_dtype(some, "output"), cache.device, tok_row.numel()
    shape = (n, cache.n_kv_heads, cache.head_dim)
    row, slot = _need(tok_row, "tok_row", dev, torch.int32, (n,)), _need(tok_slot, "tok_slot", dev, torch.int32, (n,))
    k = None if k_out is None else _need(k_out, "k_out", dev, some.dtype, shape)
    v = None if v_out is None else _need(v_out, "v_out", dev, some.dtype, shape)
    st = None if status is None else _need(status, "status", dev, torch.int32, (1,))
    _call(dev, "eesd_kv_read", dt, cache.ref, layer, slot, row, n, k, v, st)


def attention_workspace(tree: TreeBatch, cache: KVCache, n_heads: int, dtype: torch.dtype = torch.bfloat16,
                        split_keys: int = 0) -> torch.Tensor:
    """A workspace for ``tree_attention`` calls of this batch (another batch may need more: a call with too little is
    refused).  Calls that may overlap on the GPU need one each."""
    n = lib.load().eesd_attn_tree_workspace_bytes(DTYPES[dtype], cache.ref, tree.ref, n_heads, split_keys)
    if n == 0:
        raise lib.EesdError(f"attention workspace: {lib.load().eesd_last_error().decode(errors='replace')}")
    return torch.empty(n, dtype=torch.uint8, device=cache.device)


def tree_attention(q: torch.Tensor, cache: KVCache, tree: TreeBatch, out: Optional[torch.Tensor] = None, layer: int = 0,
                   workspace: Optional[torch.Tensor] = None, split_keys: int = 0) -> torch.Tensor:
    """Attention of the batch's nodes over ``layer`` of the cache.  ``q`` [n_tokens, Hq D]: rotated queries (rows may
    be strided, e.g. the q columns of a fused projection); the result is [n_tokens, Hq D] in q's dtype.  See
    ``eesd_attn_tree`` for what a node sees and for ``split_keys``."""
    dt = cache.model_dtype(q, "q")
    dev, n = cache.device, tree.on(cache).n_tokens
    n_heads = _heads(q, "q", n, cache.head_dim)
    if out is None:
        out = torch.empty(n, q.shape[1], dtype=q.dtype, device=dev)
    o = _need(out, "out", dev, q.dtype, (n, q.shape[1]))
    if workspace is None:
        workspace = attention_workspace(tree, cache, n_heads, q.dtype, split_keys)
    ws = _need(workspace, "workspace", dev, torch.uint8)
    _call(dev, "eesd_attn_tree", dt, cache.ref, layer, tree.ref, q.data_ptr(), _row_stride(q), n_heads, o, split_keys, ws,
          workspace.numel(), tree.ptr_status)
    return out


def tree_accept(y: torch.Tensor, ids: torch.Tensor, tree: TreeBatch, path: torch.Tensor, n_acc: torch.Tensor,
                next_ids: torch.Tensor) -> None:
    """Greedy walk through every block's tree: ``ids`` [n_tokens] the nodes' tokens, ``y`` [n_tokens] the model's
    token after each node.  ``path`` [n_blocks, max_nodes] (-1 behind the end), ``n_acc`` and ``next_ids`` [n_blocks]."""
    dev, i32, n, nb = tree.device, torch.int32, (tree.n_tokens,), (tree.n_blocks,)
    _call(dev, "eesd_tree_accept", _need(y, "y", dev, i32, n), _need(ids, "ids", dev, i32, n), tree.ref,
          _need(path, "path", dev, i32, (tree.n_blocks, tree.max_nodes)), _need(n_acc, "n_acc", dev, i32, nb),
          _need(next_ids, "next_ids", dev, i32, nb), tree.ptr_status)


def kv_compact(cache: KVCache, tree: TreeBatch, path: torch.Tensor, n_acc: torch.Tensor) -> None:
    """Move the accepted path's K and V of every layer to the slots behind ``ctx``.  Blocks of one row whose slots
    overlap are left as they are and reported."""
    dev, i32 = tree.on(cache).device, torch.int32
    _call(dev, "eesd_kv_compact", lib.F32 if cache.format == "f32" else lib.BF16, cache.ref, tree.ref,
          _need(path, "path", dev, i32, (tree.n_blocks, tree.max_nodes)), _need(n_acc, "n_acc", dev, i32, (tree.n_blocks,)),
          tree.ptr_status)
