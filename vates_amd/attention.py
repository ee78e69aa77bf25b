"""Full-attention decoder block and quantised GEMV on libvmi.

``AttentionLayer`` is the attention half of a Qwen3-Next decoder layer as the
MTP layer runs it (mlx_streaming/mtp/qwen3_next_mtp.py:34-57, ``self.layer``)
and as the main model's full-attention layers run it in the verify forward
(mlx_streaming/mtp/generate.py:101-220): out = x + attn(rmsnorm(x)) with the KV
cache updated in place.  ``KVCache`` holds one layer's bf16 keys and values
and the number of committed positions, the analogue of mlx-lm's KVCache with
its trim (mlx_streaming/mtp/kv_cache.py:222-251); its storage is blocks of 32
positions in the attention kernel's operand order (``keys``/``values`` and
``write`` convert from and to [n_kv_heads, positions, 256]).
``KVCache8`` holds them in 8 bits with a scale for each position and kv head,
half the bytes; ``norm_rope_append`` forms a batch's heads and appends to it,
``attend`` is the attention over it.
Errors raise ``VmiError``; there is no fallback path.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ._lib import VMI_BF16, VMI_F32, VMI_KV8_TREE_ROW, QMat, VmiError, check, load
from .moe import QuantizedProj, _ptr, _require, _stream_handle, scratch, workspace


class AttnDesc(ctypes.Structure):
    _fields_ = [("hidden", ctypes.c_int), ("n_heads", ctypes.c_int), ("n_kv_heads", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("rope_dim", ctypes.c_int), ("rope_theta", ctypes.c_float),
                ("norm_eps", ctypes.c_float), ("bits", ctypes.c_int), ("group", ctypes.c_int),
                ("input_norm", ctypes.c_void_p), ("q_proj", QMat), ("k_proj", QMat), ("v_proj", QMat),
                ("o_proj", QMat), ("q_norm", ctypes.c_void_p), ("k_norm", ctypes.c_void_p)]


def qgemv(x: torch.Tensor, w: QuantizedProj, *, bits: int = 4, out: Optional[torch.Tensor] = None,
          residual: Optional[torch.Tensor] = None, out_bf16: Optional[torch.Tensor] = None, stream=None):
    """y = W x for x bf16 [T, K] (T <= 8): f32 [T, N] and/or bf16(y + residual)."""
    T, K = x.shape
    N = w.weight.shape[-2]
    dev = x.device
    _require(x, "x", 2, dev)
    if out is None and out_bf16 is None:
        out = torch.empty((T, N), dtype=torch.float32, device=dev)
    rc = load().vmi_qgemv(x.data_ptr(), T, K, w.qmat(), N, bits, 64, None if out is None else out.data_ptr(),
                          None if residual is None else residual.data_ptr(),
                          None if out_bf16 is None else out_bf16.data_ptr(), _stream_handle(stream))
    check(rc, "vmi_qgemv")
    return out if out is not None else out_bf16


def qgemm_workspace_bytes(w: QuantizedProj, T: int, K: int, bits: int = 4) -> int:
    """Workspace of ``qgemm`` (0: a form it is not built for)."""
    return load().vmi_qgemm_workspace_bytes(T, K, w.qmat(), w.weight.shape[-2], bits, 64)


def qgemm(x: torch.Tensor, w: QuantizedProj, out_bf16: torch.Tensor, *, bits: int = 4, stream=None,
          ws: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out_bf16 = bf16(x W^T) for a prompt's rows (vmi_qgemm): x bf16 [T, K]."""
    if x.dim() != 2 or x.shape[1] * bits != 32 * w.weight.shape[-1]:
        raise VmiError(f"x {tuple(x.shape)} does not fit weights of {w.weight.shape[-1] * 32 // bits} columns")
    T, K = x.shape
    _require(x, "x", 2, x.device)
    _require(out_bf16, "out_bf16", 2, x.device)
    if tuple(out_bf16.shape) != (T, w.weight.shape[-2]):
        raise VmiError(f"out_bf16 must be [{T}, {w.weight.shape[-2]}]")
    sh = _stream_handle(stream)
    if ws is None:
        ws = scratch(qgemm_workspace_bytes(w, T, K, bits), x.device, stream)
    check(load().vmi_qgemm(x.data_ptr(), T, K, w.qmat(), w.weight.shape[-2], bits, 64, None, out_bf16.data_ptr(),
                           ws.data_ptr(), ws.numel(), sh), "vmi_qgemm")
    return out_bf16


KV_BLOCK = 32          # positions per cache block
_PERM = {}


def _block_perm(kind: str, device) -> torch.Tensor:
    """Storage offset inside a block (8192 bf16) of (position kt, dim d), flattened
    as kt * 256 + d: keys ((a*8 + kk)*64 + q4*16 + nl)*8 + e with
    kt = 8*(nl>>2) + 4*a + (nl&3), d = 32*kk + 8*q4 + e; values
    ((dt*64 + q4*16 + nl)*8 + e) with kt = 8*q4 + e, d = 16*dt + nl."""
    key = (kind, str(device))
    if key not in _PERM:
        kt = torch.arange(KV_BLOCK).view(-1, 1)
        d = torch.arange(256).view(1, -1)
        if kind == "k":
            nl, a = 4 * (kt >> 3) + (kt & 3), (kt >> 2) & 1
            off = (((a * 8 + (d >> 5)) * 64 + ((d >> 3) & 3) * 16 + nl) << 3) + (d & 7)
        else:
            off = ((((d >> 4) * 64 + (kt >> 3) * 16 + (d & 15)) << 3) + (kt & 7))
        _PERM[key] = off.reshape(-1).to(device)
    return _PERM[key]


class KVCache:
    """bf16 keys and values of one attention layer: k, v [n_kv_heads, blocks, 8192]
    (32 positions per block, kernel operand order); capacity rounds up to 32."""

    def __init__(self, n_kv_heads: int, max_len: int, device, head_dim: int = 256):
        if head_dim != 256:
            raise VmiError(f"head_dim={head_dim} (256 only)")
        self.max_len = -(-max_len // KV_BLOCK) * KV_BLOCK
        nb = self.max_len // KV_BLOCK
        self.k = torch.zeros((n_kv_heads, nb, KV_BLOCK * head_dim), dtype=torch.bfloat16, device=device)
        self.v = torch.zeros_like(self.k)
        self.length = 0  # committed positions
        self.n_kv = n_kv_heads
        self.tree_kv = None  # [paths, n_kv, 2, span, 256] bf16: a draft tree's new keys and values
        # (made here, not by the first tree: that one's stream would not wait for the fill)
        self._tree_flat = torch.zeros(16 * n_kv_heads * 2 * 256, dtype=torch.bfloat16, device=device)

    @property
    def device(self) -> torch.device:
        return self.k.device

    def tree_buffer(self, paths: int, span: int) -> torch.Tensor:
        """The tree forward's keys and values [paths, n_kv, 2, span, 256]: one
        allocation for every tree of at most 16 tokens, so commit tables built
        for different (paths, span) see the same address."""
        if paths * span > 16:
            raise VmiError(f"a tree of {paths} x {span} tokens exceeds 16")
        self.tree_kv = self._tree_flat[:paths * self.n_kv * 2 * span * 256].view(paths, self.n_kv, 2, span, 256)
        return self.tree_kv

    def trim(self, n: int) -> None:
        """Drops the last n positions (kv_cache.py:222-251: rejected drafts)."""
        if n < 0 or n > self.length:
            raise VmiError(f"cannot trim {n} of {self.length} positions")
        self.length -= n

    def _read(self, raw: torch.Tensor, kind: str, start: int, stop: int) -> torch.Tensor:
        b0, b1 = start // KV_BLOCK, -(-stop // KV_BLOCK)
        blk = raw[:, b0:b1]
        logical = blk[:, :, _block_perm(kind, raw.device)].reshape(raw.shape[0], (b1 - b0) * KV_BLOCK, 256)
        return logical[:, start - b0 * KV_BLOCK:stop - b0 * KV_BLOCK]

    def keys(self, start: int = 0, stop: Optional[int] = None) -> torch.Tensor:
        """Keys of positions start..stop-1 as [n_kv_heads, positions, 256] (a copy)."""
        return self._read(self.k, "k", start, self.length if stop is None else stop)

    def values(self, start: int = 0, stop: Optional[int] = None) -> torch.Tensor:
        return self._read(self.v, "v", start, self.length if stop is None else stop)

    def write(self, start: int, keys: torch.Tensor, values: torch.Tensor) -> None:
        """Stores [n_kv_heads, n, 256] keys and values at positions start..start+n-1."""
        n = keys.shape[1]
        if start < 0 or start + n > self.max_len:
            raise VmiError(f"positions {start}..{start + n} outside the capacity {self.max_len}")
        b0, b1 = start // KV_BLOCK, -(-(start + n) // KV_BLOCK)
        for raw, kind, data in ((self.k, "k", keys), (self.v, "v", values)):
            logical = self._read(raw, kind, b0 * KV_BLOCK, b1 * KV_BLOCK).clone()
            logical[:, start - b0 * KV_BLOCK:start - b0 * KV_BLOCK + n] = data
            blk = torch.empty_like(raw[:, b0:b1])
            blk[:, :, _block_perm(kind, raw.device)] = logical.reshape(raw.shape[0], b1 - b0, -1)
            raw[:, b0:b1] = blk


class KVCache8(KVCache):
    """Keys and values of one attention layer in 8 bits (vmi_kv8_*): each
    position's key and value of a kv head is 256 codes and one fp32 scale, the
    codes within half a step (1/254 of the row's largest magnitude) of what was
    written.  A row is stored alike whatever is appended around it.  ``data``
    holds the records (include/vmi.h), ``status`` (int32 [1] on the device) the
    status bits that calls with a position on the device OR in."""

    def __init__(self, n_kv_heads: int, max_len: int, device, head_dim: int = 256):
        if head_dim != 256:
            raise VmiError(f"head_dim={head_dim} (256 only)")
        if max_len < 1 or n_kv_heads < 1:
            raise VmiError(f"a cache of {n_kv_heads} kv heads and {max_len} positions")
        self.max_len = -(-max_len // KV_BLOCK) * KV_BLOCK
        self.n_kv = n_kv_heads
        nbytes = load().vmi_kv8_bytes(n_kv_heads, self.max_len)
        if not nbytes:
            raise VmiError(f"a cache of {n_kv_heads} kv heads and {max_len} positions")
        self.data = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.length = 0
        self.tree_kv = None   # uint8: a draft tree's new rows
        self._tree_flat = torch.zeros(16 * n_kv_heads * VMI_KV8_TREE_ROW, dtype=torch.uint8, device=device)

    @property
    def device(self) -> torch.device:
        return self.data.device

    def tree_buffer(self, paths: int, span: int) -> torch.Tensor:
        """The tree forward's rows, uint8 [paths, n_kv, span, 528]: one
        allocation for every tree of at most 16 tokens, as KVCache's."""
        if paths * span > 16:
            raise VmiError(f"a tree of {paths} x {span} tokens exceeds 16")
        self.tree_kv = self._tree_flat[:paths * self.n_kv * span * VMI_KV8_TREE_ROW].view(paths, self.n_kv, span,
                                                                                          VMI_KV8_TREE_ROW)
        return self.tree_kv

    def read(self, start: int = 0, stop: Optional[int] = None, *, dtype: torch.dtype = torch.bfloat16, stream=None):
        """(keys, values) of positions start..stop-1 (default: all committed
        ones) as [n_kv_heads, positions, 256], float32 or rounded to bfloat16."""
        return self._read8(start, stop, dtype, True, True, stream)

    def keys(self, start: int = 0, stop: Optional[int] = None, *, dtype: torch.dtype = torch.bfloat16,
             stream=None) -> torch.Tensor:
        return self._read8(start, stop, dtype, True, False, stream)[0]

    def values(self, start: int = 0, stop: Optional[int] = None, *, dtype: torch.dtype = torch.bfloat16,
               stream=None) -> torch.Tensor:
        return self._read8(start, stop, dtype, False, True, stream)[1]

    def _read8(self, start, stop, dtype, want_k, want_v, stream):
        stop = self.length if stop is None else stop
        if dtype is not torch.bfloat16 and dtype is not torch.float32:
            raise VmiError(f"dtype {dtype} is not bfloat16 or float32")
        if not 0 <= start <= stop <= self.max_len:
            raise VmiError(f"positions {start}..{stop} outside the capacity {self.max_len}")
        dev = _on_current(self.data)
        rows = _like(self.data, (self.n_kv, stop - start, 256), dtype, stream)
        k = rows if want_k else None
        v = (rows if not want_k else _like(rows, None, dtype, stream)) if want_v else None
        if stop > start:
            check(load().vmi_kv8_read(self.data.data_ptr(), self.n_kv, self.max_len, start, stop - start, _ptr(k),
                                      _ptr(v), VMI_F32 if dtype is torch.float32 else VMI_BF16, _stream_on(dev, stream)),
                  "vmi_kv8_read")
        return k, v

    def write(self, start: int, keys: torch.Tensor, values: torch.Tensor, *, stream=None) -> None:
        """Stores bfloat16 [n_kv_heads, n, 256] keys and values at positions
        start..start+n-1.  Rows of 256 are contiguous; heads and positions may
        be strided (a transposed view of token-major rows; 16-byte aligned).  The
        committed length is the caller's to set."""
        dev = _on_current(self.data)
        n = keys.shape[1] if keys.dim() == 3 else 0
        for name, t in (("keys", keys), ("values", values)):
            if t.device != dev or t.dtype is not torch.bfloat16 or t.shape != (self.n_kv, n, 256) or t.stride(2) != 1:
                raise VmiError(f"{name} must be bfloat16 [{self.n_kv}, {n}, 256] on {dev} with contiguous rows")
        if start < 0 or start + n > self.max_len:
            raise VmiError(f"positions {start}..{start + n} outside the capacity {self.max_len}")
        if n:
            a, b = int(self.n_kv > 1), int(n > 1)   # (one head, or one position, may have any stride)
            check(load().vmi_kv8_write(keys.data_ptr(), keys.stride(0) * a, keys.stride(1) * b, values.data_ptr(),
                                       values.stride(0) * a, values.stride(1) * b, self.n_kv, start, n,
                                       self.data.data_ptr(), self.max_len, _stream_on(dev, stream)), "vmi_kv8_write")


def _like(t: torch.Tensor, shape, dtype: torch.dtype, stream) -> torch.Tensor:
    """An output of a call on `stream`, on t's device (shape None: and of its
    shape), allocated in that stream's order."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return _like(t, shape, dtype, None)
    return torch.empty_like(t) if shape is None else t.new_empty(shape, dtype=dtype)


def _on_current(t: torch.Tensor) -> torch.device:
    """The tensor's device, which has to be the one that the calls go to."""
    dev = t.device
    # (torch.cuda.current_device without its check that the device is initialised: t is on one)
    if dev.type != "cuda" or dev.index != torch._C._cuda_getDevice():
        raise VmiError(f"tensors on {dev} are not on the current HIP device")
    return dev


def _stream_on(dev: torch.device, stream) -> int:
    return torch._C._cuda_getCurrentRawStream(dev.index) if stream is None else stream.cuda_stream


_ATTEND_BYTES: dict = {}   # (device, T, query heads, kv heads) -> bytes of vmi_kv8_attention's workspace


def _position(cache: KVCache8, T: int, pos0: Optional[int], pos_device: Optional[torch.Tensor], dev) -> int:
    if pos_device is not None:
        if pos_device.device != dev or pos_device.dtype is not torch.int32 or pos_device.numel() != 1:
            raise VmiError(f"pos_device must be int32 [1] on {dev}")
        return 0
    pos0 = cache.length if pos0 is None else pos0
    if pos0 < 0 or pos0 + T > cache.max_len:
        raise VmiError(f"positions {pos0}..{pos0 + T} outside the capacity {cache.max_len}")
    return pos0


def norm_rope_append(qkv: torch.Tensor, cache: KVCache8, q_norm: torch.Tensor, k_norm: torch.Tensor, *, n_heads: int,
                     rope_dim: int = 64, rope_theta: float = 1e7, eps: float = 1e-6, pos0: Optional[int] = None,
                     pos_device: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                     stream=None) -> torch.Tensor:
    """The heads of T tokens from their projections (vmi_kv8_append): qkv f32
    [T, (2 n_heads + 2 n_kv) * 256] holds q | gate per head, then the keys, then
    the values.  Queries and keys get their per-head RMSNorm and rotary embedding
    at positions pos0.. (default: cache.length); keys and values go into the cache,
    whose length becomes pos0 + T; returns the queries, bfloat16 [T, n_heads, 256].
    With pos_device (int32 [1] on the device) the position is read there when the
    kernel runs, one outside the capacity is clamped and sets VMI_STATUS_BAD_POS in
    cache.status, and cache.length is left to the caller."""
    dev = _on_current(cache.data)
    _require(qkv, "qkv", 4, dev)
    if qkv.dtype is not torch.float32 or qkv.dim() != 2 or qkv.shape[1] != (2 * n_heads + 2 * cache.n_kv) * 256:
        raise VmiError(f"qkv must be float32 [T, {(2 * n_heads + 2 * cache.n_kv) * 256}]")
    for name, t in (("q_norm", q_norm), ("k_norm", k_norm)):
        _require(t, name, 2, dev)
        if t.dtype is not torch.bfloat16 or t.numel() != 256:
            raise VmiError(f"{name} must be bfloat16 [256]")
    T = qkv.shape[0]
    pos = _position(cache, T, pos0, pos_device, dev)
    if out is None:
        out = _like(q_norm, (T, n_heads, 256), torch.bfloat16, stream)
    else:
        _rows_bf16(out, "out", (T, n_heads, 256), dev)
    if T:
        check(load().vmi_kv8_append(qkv.data_ptr(), T, n_heads, cache.n_kv, q_norm.data_ptr(), k_norm.data_ptr(), eps,
                                    rope_dim, rope_theta, pos, _ptr(pos_device), cache.data.data_ptr(), cache.max_len,
                                    out.data_ptr(), cache.status.data_ptr(), _stream_on(dev, stream)), "vmi_kv8_append")
    if pos_device is None:
        cache.length = pos + T
    return out


def _rows_bf16(t: torch.Tensor, name: str, shape: tuple, dev) -> None:
    _require(t, name, 2, dev)
    if t.dtype is not torch.bfloat16 or t.shape != shape:
        raise VmiError(f"{name} must be bfloat16 {list(shape)}")


def attend(q: torch.Tensor, cache: KVCache8, *, pos0: Optional[int] = None, gate: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None, pos_device: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """softmax(q k / 16) v over an 8-bit cache (vmi_kv8_attention): q bfloat16 [T,
    n_heads, 256], the queries of positions pos0.. (default: the last T committed
    ones), each seeing the positions up to its own; with gate (float32 [T, n_heads,
    256], rows of 256 contiguous) times sigmoid(gate).  Returns bfloat16 [T,
    n_heads, 256].  The result of a token of a batch of T * n_heads / n_kv <= 64
    does not depend on the batch, and no token's on the keys and values behind it.
    Queries count as 16-bit integers, probabilities and value scales as fp16, a scale relative
    to the largest that the query sees (include/vmi.h).  pos_device as for
    ``norm_rope_append``."""
    dev = _on_current(cache.data)
    if q.dim() != 3 or q.shape[1] % cache.n_kv or not q.shape[1]:
        raise VmiError(f"q {tuple(q.shape)} does not fit a cache of {cache.n_kv} kv heads")
    T, n_heads = q.shape[:2]
    _rows_bf16(q, "q", (T, n_heads, 256), dev)
    if pos0 is None and pos_device is None:
        pos0 = cache.length - T
    pos = _position(cache, T, pos0, pos_device, dev)
    if gate is not None and (gate.device != dev or gate.dtype is not torch.float32 or gate.shape != q.shape or
                             gate.stride(2) != 1):
        raise VmiError(f"gate must be float32 {list(q.shape)} on {dev} with contiguous rows")
    if out is None:
        out = _like(q, None, torch.bfloat16, stream)
    else:
        _rows_bf16(out, "out", (T, n_heads, 256), dev)
    if T:
        lib = load()
        key = (dev.index, T, n_heads, cache.n_kv)
        nbytes = _ATTEND_BYTES.get(key)
        if nbytes is None:
            nbytes = _ATTEND_BYTES[key] = lib.vmi_kv8_attention_workspace_bytes(T, n_heads, cache.n_kv)
        ws = _like(cache.data, (nbytes,), torch.uint8, stream)
        check(lib.vmi_kv8_attention(q.data_ptr(), T, n_heads, cache.n_kv, pos, _ptr(pos_device), cache.data.data_ptr(),
                                    cache.max_len, _ptr(gate), 0 if gate is None or T == 1 else gate.stride(0),
                                    0 if gate is None or n_heads == 1 else gate.stride(1), out.data_ptr(), cache.status.data_ptr(),
                                    ws.data_ptr(), nbytes, _stream_on(dev, stream)), "vmi_kv8_attention")
    return out


def layer_cache(attn, max_len: int, bits: int) -> KVCache:
    """A cache of an attention layer.  Layers whose own ``new_cache`` takes the length
    alone give bf16 ones."""
    return attn.new_cache(max_len) if bits == 16 else attn.new_cache(max_len, bits)


def prompt_bytes(attn, T: int, cache: Optional[KVCache]) -> int:
    """An attention layer's prompt workspace for this kind of cache.  Layers whose own
    ``prompt_workspace_bytes`` takes T alone serve bf16 caches."""
    return attn.prompt_workspace_bytes(T, cache) if isinstance(cache, KVCache8) else attn.prompt_workspace_bytes(T)


class AttentionLayer:
    def __init__(self, q_proj: QuantizedProj, k_proj: QuantizedProj, v_proj: QuantizedProj, o_proj: QuantizedProj,
                 input_norm: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor, *, n_heads: int = 16,
                 n_kv_heads: int = 2, rope_dim: int = 64, rope_theta: float = 1e7, eps: float = 1e-6,
                 bits: int = 4):
        dev = input_norm.device
        self.device = dev
        self.hidden = input_norm.numel()
        self.n_heads, self.n_kv = n_heads, n_kv_heads
        for name, p in (("q_proj", q_proj), ("k_proj", k_proj), ("v_proj", v_proj), ("o_proj", o_proj)):
            p.check(name, dev)
        for name, t in (("input_norm", input_norm), ("q_norm", q_norm), ("k_norm", k_norm)):
            _require(t, name, 2, dev)
        self._keep = (q_proj, k_proj, v_proj, o_proj, input_norm, q_norm, k_norm)
        d = AttnDesc()
        d.hidden, d.n_heads, d.n_kv_heads, d.head_dim, d.rope_dim = self.hidden, n_heads, n_kv_heads, 256, rope_dim
        d.rope_theta, d.norm_eps, d.bits, d.group = rope_theta, eps, bits, 64
        d.input_norm = input_norm.data_ptr()
        d.q_proj, d.k_proj, d.v_proj, d.o_proj = q_proj.qmat(), k_proj.qmat(), v_proj.qmat(), o_proj.qmat()
        d.q_norm, d.k_norm = q_norm.data_ptr(), k_norm.data_ptr()
        self.desc = d

    def new_cache(self, max_len: int, bits: int = 16) -> KVCache:
        """A cache for this layer: bf16, or with bits=8 a ``KVCache8``, which
        every call of the layer takes in its place."""
        if bits not in (8, 16):
            raise VmiError(f"a cache of {bits} bits (8 or 16)")
        return (KVCache8 if bits == 8 else KVCache)(self.n_kv, max_len, self.device)

    def _cache8(self, x: torch.Tensor, cache: KVCache8, paths: int, span: int, pos0: Optional[int], out, stream,
                pos_device) -> torch.Tensor:
        """The block over an 8-bit cache: a batch (paths = 0) or a draft tree."""
        dev = _on_current(cache.data)
        if dev != self.device or cache.n_kv != self.n_kv:
            raise VmiError(f"a cache of {cache.n_kv} kv heads on {dev} does not fit the layer")
        T = max(paths, 1) * span
        _rows_bf16(x, "x", (T, self.hidden), dev)
        pos = _position(cache, span, pos0, pos_device, dev)
        if out is None:
            out = _like(x, None, torch.bfloat16, stream)
        else:
            _rows_bf16(out, "out", (T, self.hidden), dev)
        lib = load()
        nbytes = lib.vmi_attention_kv8_workspace_bytes(max(paths, 1), span, self.hidden, self.n_heads, self.n_kv)
        if not nbytes:
            raise VmiError(f"a batch of {max(paths, 1)} x {span} tokens is not built for this layer")
        ws = _like(cache.data, (nbytes,), torch.uint8, stream)
        rest = (out.data_ptr(), cache.status.data_ptr(), ws.data_ptr(), nbytes, _stream_handle(stream))
        if paths:
            check(lib.vmi_attention_tree_kv8(ctypes.byref(self.desc), x.data_ptr(), paths, span, pos, _ptr(pos_device),
                                             cache.data.data_ptr(), cache.max_len, cache.tree_buffer(paths, span).data_ptr(),
                                             *rest), "vmi_attention_tree_kv8")
        else:
            check(lib.vmi_attention_layer_kv8(ctypes.byref(self.desc), x.data_ptr(), span, pos, _ptr(pos_device),
                                              cache.data.data_ptr(), cache.max_len, *rest), "vmi_attention_layer_kv8")
            if pos_device is None:
                cache.length = pos + span
        return out

    def __call__(self, x: torch.Tensor, cache: KVCache, *, pos0: Optional[int] = None,
                 out: Optional[torch.Tensor] = None, stream=None,
                 pos_device: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x bf16 [T, hidden] at cache positions pos0.. (default: cache.length);
        appends k, v there and sets cache.length = pos0 + T.  With pos_device
        (int32 [1] on the device) the position is read there when the kernels
        run and cache.length is left to the caller."""
        T = x.shape[0]
        if isinstance(cache, KVCache8):
            return self._cache8(x, cache, 0, T, pos0, out, stream, pos_device)
        pos0 = cache.length if pos0 is None else pos0
        _require(x, "x", 2, self.device)
        if out is None:
            out = torch.empty_like(x)
        sh = _stream_handle(stream)
        lib = load()
        ws = workspace(lib.vmi_attention_layer_workspace_bytes(T, self.hidden, self.n_heads, self.n_kv, cache.max_len),
                       self.device, sh, tag="attention")
        rc = lib.vmi_attention_layer(ctypes.byref(self.desc), x.data_ptr(), T, pos0,
                                     None if pos_device is None else pos_device.data_ptr(), cache.k.data_ptr(),
                                     cache.v.data_ptr(), cache.max_len, out.data_ptr(), ws.data_ptr(), ws.numel(), sh)
        check(rc, "vmi_attention_layer")
        if pos_device is None:
            cache.length = pos0 + T
        return out

    def prompt_workspace_bytes(self, T: int, cache: Optional[KVCache] = None) -> int:
        """Workspace of ``prompt`` on T tokens (0: a form it is not built for)
        into the cache (None: a bf16 one)."""
        if isinstance(cache, KVCache8):
            return load().vmi_attention_prompt_kv8_workspace_bytes(ctypes.byref(self.desc), T)
        return load().vmi_attention_prompt_workspace_bytes(ctypes.byref(self.desc), T)

    def prompt(self, x: torch.Tensor, cache: KVCache, *, pos0: int, keys_only: bool = False, stream=None,
               ws: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """The block over a prompt's tokens (vmi_attention_prompt), x bf16
        [T, hidden] at positions pos0..; sets cache.length = pos0 + T.
        keys_only: the cache is filled and nothing returned."""
        if x.dim() != 2 or x.shape[1] != self.hidden or cache.n_kv != self.n_kv:
            raise VmiError(f"x {tuple(x.shape)} or a cache of {cache.n_kv} kv heads does not fit the layer")
        T = x.shape[0]
        _require(x, "x", 2, self.device)
        out = None if keys_only else _like(x, None, x.dtype, stream)
        sh = _stream_handle(stream)
        if ws is None:
            ws = scratch(prompt_bytes(self, T, cache), self.device, stream)
        if isinstance(cache, KVCache8):
            if _on_current(cache.data) != self.device or cache.n_kv != self.n_kv:
                raise VmiError(f"a cache of {cache.n_kv} kv heads on {cache.device} does not fit the layer")
            check(load().vmi_attention_prompt_kv8(ctypes.byref(self.desc), x.data_ptr(), T, pos0, cache.data.data_ptr(),
                                                  cache.max_len, _ptr(out), ws.data_ptr(), ws.numel(), sh),
                  "vmi_attention_prompt_kv8")
            cache.length = pos0 + T
            return out
        check(load().vmi_attention_prompt(ctypes.byref(self.desc), x.data_ptr(), T, pos0, cache.k.data_ptr(),
                                          cache.v.data_ptr(), cache.max_len, None if keys_only else out.data_ptr(),
                                          ws.data_ptr(), ws.numel(), sh), "vmi_attention_prompt")
        cache.length = pos0 + T
        return out

    def tree(self, x: torch.Tensor, cache: KVCache, paths: int, *, pos0: Optional[int] = None,
             out: Optional[torch.Tensor] = None, stream=None, pos_device: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The block over a draft tree: x bf16 [paths * span, hidden], path p's
        tokens at rows p*span.. and positions pos0.. (default: cache.length).
        The cache is only read; every path's new keys and values go to
        cache.tree_kv until vmi_tree_commit writes the winner's."""
        T = x.shape[0]
        if T % paths:
            raise VmiError(f"{T} rows do not split into {paths} paths")
        span = T // paths
        if isinstance(cache, KVCache8):
            return self._cache8(x, cache, paths, span, pos0, out, stream, pos_device)
        pos0 = cache.length if pos0 is None else pos0
        _require(x, "x", 2, self.device)
        if out is None:
            out = torch.empty_like(x)
        tkv = cache.tree_buffer(paths, span)
        sh = _stream_handle(stream)
        lib = load()
        ws = workspace(lib.vmi_attention_tree_workspace_bytes(paths, span, self.hidden, self.n_heads, self.n_kv,
                                                              cache.max_len), self.device, sh, tag="attention")
        rc = lib.vmi_attention_tree(ctypes.byref(self.desc), x.data_ptr(), paths, span, pos0,
                                    None if pos_device is None else pos_device.data_ptr(), cache.k.data_ptr(),
                                    cache.v.data_ptr(), cache.max_len, tkv.data_ptr(), out.data_ptr(), ws.data_ptr(),
                                    ws.numel(), sh)
        check(rc, "vmi_attention_tree")
        return out

