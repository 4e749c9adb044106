"""The low-bit decode path: weights and the KV cache held in 4 bits (``evs_q4_*``).

Decoding a block of a few tokens is bound by the bytes of the weights and, at long contexts, of the
keys and values.  Held in 4 bits both shrink to 0.28 of their bf16 size:

* ``quantize_weight`` / ``q4_linear``: tokens times a 4-bit weight;
* ``Q4Cache`` with ``q4_kv_append``, ``q4_kv_read`` and ``q4_attention``: a paged KV cache of 4-bit
  keys and values, written with the position rotation applied, and attention over it.

Format: groups of values share a bf16 scale, absmax / 7 rounded to five significant bits; a code c in
1..15 stands for (c - 8) * scale, which is exact in bf16.  A group whose absmax / 7 is below 2^-120 is
held as zeros; a group with a NaN, an infinity or absmax / 7 above 2^120 is held as NaN.  Weights use
groups of 32, 64 or 128 input features, the cache groups of 32 along head_dim.

All tensors are CUDA tensors; calls run on the current stream of their device, allocate their result
and scratch from torch's allocator and can be captured into CUDA graphs.  The reference has no
counterpart: it runs its target in bf16 (evspark/api.py:94-98).
"""

from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _native as N

KBLOCK = 128  # weights: input features are padded to a multiple of this
KV_GROUP = 32
_DT = {torch.bfloat16: N.EVS_DTYPE_BF16, torch.float32: N.EVS_DTYPE_FP32}


def _dtype(t: torch.Tensor, what: str) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise ValueError(f"{what} must be bf16 or fp32, got {t.dtype}") from None


def _need_cuda(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        if not torch.cuda.is_available():
            raise RuntimeError("evspark_b200 runs on a CUDA B200 (sm_100a); no CUDA device is available")
        raise ValueError(f"{what} must be a CUDA tensor")


# A decode step's calls are a few microseconds long on the device, so the host side counts: the raw stream
# (current_stream() builds a Stream object, 2 us a call), device indices instead of torch.device objects, and
# the C structs packed as bytes.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_fns: dict = {}
_pack_rows = struct.Struct("@PPPqiii4x").pack  # evs_q4_rows
_pack_strides = struct.Struct("@3q").pack


def _call(index: int, name: str, *args) -> None:
    """One library call on the current stream of device ``index``."""
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(N.lib(), name)
    if index == _current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        N.check(status, name)


# Sizes that the library takes.  Checked here, as they go to it as 32-bit integers, which would wrap.
_MOST = 2 ** 31 - 1


def _check_weight_size(n: int, k: int, what: str) -> None:
    if n > _MOST or k > 2 ** 24 or n * k > 2 ** 35:
        raise ValueError(f"{what}: at most 2^31 - 1 rows, 2^24 features and 2^35 values, got [{n}, {k}]")


def padded_features(k: int) -> int:
    return -(-k // KBLOCK) * KBLOCK


class _Fixed:
    """Objects whose calls keep the addresses of their tensors: what those belong to cannot be replaced."""

    _FIXED = frozenset()

    def __setattr__(self, name, value):
        if name in self._FIXED and "_index" in self.__dict__:
            raise AttributeError(f"{type(self).__name__}: {name} cannot be replaced, its address is kept; "
                                 f"write into it or make a new {type(self).__name__}")
        super().__setattr__(name, value)


class Q4Weight(_Fixed):
    """A weight [N, K] held in 4 bits: ``codes`` uint8 [N, Kp / 2] (two input features per byte, the even
    one in the low half, Kp = K rounded up to 128 with codes of 8 behind K), ``scales`` bf16
    [Kp / group, N]."""

    _FIXED = frozenset(("codes", "scales", "shape", "group"))

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape: tuple[int, int], group: int):
        n, k = int(shape[0]), int(shape[1])
        if n < 1 or k < 1:
            raise ValueError(f"Q4Weight: shape must be at least [1, 1], got {tuple(shape)}")
        _check_weight_size(n, k, "Q4Weight")
        if group not in (32, 64, 128):
            raise ValueError(f"Q4Weight: group must be 32, 64 or 128, got {group}")
        kp = padded_features(k)
        if codes.dtype != torch.uint8 or tuple(codes.shape) != (n, kp // 2):
            raise ValueError(f"Q4Weight: codes must be uint8 [{n}, {kp // 2}], got {codes.dtype} {tuple(codes.shape)}")
        if scales.dtype != torch.bfloat16 or tuple(scales.shape) != (kp // group, n):
            raise ValueError(f"Q4Weight: scales must be bf16 [{kp // group}, {n}], "
                             f"got {scales.dtype} {tuple(scales.shape)}")
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.data_ptr() % 16:
            raise ValueError("Q4Weight: codes and scales must be contiguous, codes 16-byte aligned")
        if codes.device != scales.device:
            raise ValueError("Q4Weight: codes and scales on different devices")
        _need_cuda(codes, "Q4Weight: codes")
        self.codes, self.scales, self.shape, self.group = codes, scales, (n, k), int(group)
        self._args = (codes.data_ptr(), scales.data_ptr(), n, k, self.group)
        self._index = codes.get_device()

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 2 * self.scales.numel()

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values that the weight holds [N, K] (exact in bf16)."""
        if dtype not in _DT:
            raise ValueError(f"dequantize: dtype must be bf16 or fp32, got {dtype}")
        n, k = self.shape
        out = torch.empty(n, k, dtype=dtype, device=self.device)
        _call(self._index, "evs_q4_dequantize", self.codes.data_ptr(), self.scales.data_ptr(), n, k, self.group,
              out.data_ptr(), _DT[dtype], k)
        return out


def quantize_weight(w: torch.Tensor, group: int = 64) -> Q4Weight:
    """A weight [N, K] (bf16 or fp32; rows may be strided) -> ``Q4Weight``."""
    if w.dim() != 2 or w.numel() == 0:
        raise ValueError(f"quantize_weight: w must be a non-empty [N, K] matrix, got {tuple(w.shape)}")
    _check_weight_size(*w.shape, "quantize_weight")
    if group not in (32, 64, 128):
        raise ValueError(f"quantize_weight: group must be 32, 64 or 128, got {group}")
    dt = _dtype(w, "quantize_weight: w")
    _need_cuda(w, "quantize_weight: w")
    n, k = w.shape
    if w.stride(1) != 1 or (n > 1 and w.stride(0) < k):
        w = w.contiguous()
    kp = padded_features(k)
    codes = torch.empty(n, kp // 2, dtype=torch.uint8, device=w.device)
    scales = torch.empty(kp // group, n, dtype=torch.bfloat16, device=w.device)
    _call(w.get_device(), "evs_q4_quantize", w.data_ptr(), dt, max(w.stride(0), k), n, k, group, codes.data_ptr(),
          scales.data_ptr())
    return Q4Weight(codes, scales, (n, k), group)


def q4_linear(x: torch.Tensor, w: Q4Weight, *, out_dtype: torch.dtype = torch.float32,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """``x [..., K] @ w.T`` with sums in fp32 -> [..., N] in ``out_dtype`` (fp32 or bf16), or into ``out``.

    bf16 rows multiply the held weight values exactly; fp32 rows are used at full precision.  A row's
    result does not depend on the other rows.  Meant for the few tokens of a decode step or verify
    block: every 32 rows read the weight once."""
    codes, scales, n, k, group = w._args
    dt = _DT.get(x.dtype)
    if dt is None:
        dt = _dtype(x, "q4_linear: x")
    shape = x.shape
    if not shape or shape[-1] != k:
        raise ValueError(f"q4_linear: x must be [..., {k}], got {tuple(shape)}")
    if x.get_device() != w._index:
        raise ValueError(f"q4_linear: x on {x.device}, the weight on {w.codes.device}")
    m = x.numel() // k
    if m > _MOST:
        raise ValueError(f"q4_linear: too many rows ({m})")
    if out is not None:
        if out.shape != shape[:-1] + (n,) or out.get_device() != w._index or not out.is_contiguous():
            raise ValueError(f"q4_linear: out must be a contiguous [..., {n}] tensor of x's batch shape and device")
        odt = _dtype(out, "q4_linear: out")
    else:
        odt = _DT.get(out_dtype)
        if odt is None:
            raise ValueError(f"q4_linear: out_dtype must be bf16 or fp32, got {out_dtype}")
        out = x.new_empty(shape[:-1] + (n,), dtype=out_dtype)
    if m == 0:
        return out
    ldx = k
    if not x.is_contiguous():
        if len(shape) == 2 and x.stride(1) == 1 and x.stride(0) >= k:
            ldx = x.stride(0)
        else:
            x = x.contiguous()
    _call(w._index, "evs_q4_linear", x.data_ptr(), dt, ldx, m, codes, scales, n, k, group, out.data_ptr(), odt, n)
    return out


class Q4Cache(_Fixed):
    """A pool of KV pages in 4 bits, shared by any number of rows and layers' worth of page tables.

    ``pool`` uint8 [num_pages, kv_heads, block]: per page and head K codes [P, D / 2], V codes [P, D / 2],
    K scales bf16 [D / 32, P] and V scales [D / 32, P] (P = page_size tokens, D = head_dim).  Which page
    holds what is the caller's page table's affair; pages may be shared by rows for reading.

    Calls that meet a length outside the page table or a page id outside the pool skip that row (its
    attention result is NaN) and note it on the device; ``check`` reads the note and raises."""

    _FIXED = frozenset(("pool", "num_pages", "kv_heads", "head_dim", "page_size"))

    def __init__(self, num_pages: int, kv_heads: int, head_dim: int, *, page_size: int = 64, device="cuda:0"):
        self._init(None, num_pages, kv_heads, head_dim, page_size, torch.device(device))

    @classmethod
    def from_pool(cls, pool: torch.Tensor, *, head_dim: int, page_size: int) -> "Q4Cache":
        """A cache over an existing pool tensor (kept, not copied)."""
        if pool.dtype != torch.uint8 or pool.dim() != 3 or not pool.is_contiguous():
            raise ValueError("Q4Cache: pool must be a contiguous uint8 [pages, kv_heads, block] tensor")
        self = cls.__new__(cls)
        self._init(pool, pool.shape[0], pool.shape[1], head_dim, page_size, pool.device)
        return self

    @staticmethod
    def block_bytes(head_dim: int, page_size: int) -> int:
        return page_size * head_dim + page_size * head_dim // 8

    def _init(self, pool, num_pages, kv_heads, head_dim, page_size, device):
        num_pages, kv_heads, head_dim, page_size = int(num_pages), int(kv_heads), int(head_dim), int(page_size)
        if head_dim not in (32, 64, 128):
            raise ValueError(f"Q4Cache: head_dim must be 32, 64 or 128, got {head_dim}")
        if page_size < 16 or page_size > 4096 or page_size % 16:
            raise ValueError(f"Q4Cache: page_size must be a multiple of 16 in [16, 4096], got {page_size}")
        if num_pages < 1 or kv_heads < 1:
            raise ValueError("Q4Cache: needs at least one page and one kv head")
        block = self.block_bytes(head_dim, page_size)
        if pool is None:
            if device.type != "cuda" or not torch.cuda.is_available():
                raise RuntimeError("evspark_b200 runs on a CUDA B200 (sm_100a); no CUDA device is available")
            pool = torch.zeros(num_pages, kv_heads, block, dtype=torch.uint8, device=device)
        elif pool.shape[2] != block:
            raise ValueError(f"Q4Cache: a page block of head_dim {head_dim} and page_size {page_size} has {block} bytes, "
                             f"the pool's have {pool.shape[2]}")
        _need_cuda(pool, "Q4Cache: pool")
        if pool.data_ptr() % 16:
            raise ValueError("Q4Cache: the pool must be 16-byte aligned")
        self.pool, self.num_pages, self.kv_heads = pool, num_pages, kv_heads
        self.head_dim, self.page_size = head_dim, page_size
        self._err = torch.zeros(3, dtype=torch.int32, device=pool.device)
        self._desc = N.Q4CacheDesc(pool.data_ptr(), self._err.data_ptr(), num_pages, page_size, kv_heads, head_dim)
        self._ref = C.addressof(self._desc)
        self._index = pool.get_device()
        self._workspace: dict = {}  # attention workspace bytes by call sizes

    @property
    def device(self) -> torch.device:
        return self.pool.device

    def check(self) -> None:
        """Raise if a call since the last ``check`` met a bad length or page id, on whatever stream it ran (waits
        for the device)."""
        torch.cuda.synchronize(self._index)
        code, where, info = self._err.tolist()
        if code:
            self._err.zero_()
            if code == N.EVS_ETIMEOUT:
                raise N.EvsError(f"Q4Cache: a wait inside a kernel ran out at row {info}; what that call returned is not "
                                 f"valid [evs status {code}, kernel {where}]")
            raise N.EvsError(f"Q4Cache: row {info} has a length outside its page table (or above max_length), "
                             f"or a page id outside the pool [evs status {code}, kernel {where}]")


def _rows(cache: Q4Cache, page_table, lengths, counts, batch: int, tokens: int, what: str):
    """The checked evs_q4_rows of a call, packed, and its table's positions."""
    index = cache._index
    shape, strides = page_table.shape, page_table.stride()
    if (page_table.dtype != torch.int32 or len(shape) != 2 or shape[0] != batch or shape[1] < 1
            or (shape[1] > 1 and strides[1] != 1) or (batch > 1 and strides[0] < shape[1])):
        raise ValueError(f"{what}: page_table must be int32 [{batch}, max_pages] with contiguous rows")
    if lengths.dtype != torch.int32 or lengths.shape != (batch,) or not lengths.is_contiguous():
        raise ValueError(f"{what}: lengths must be a contiguous int32 [{batch}] tensor")
    if page_table.get_device() != index or lengths.get_device() != index:
        raise ValueError(f"{what}: page_table and lengths must be on the cache's device {cache.pool.device}")
    cp = 0
    if counts is not None:
        if (counts.dtype != torch.int32 or counts.shape != (batch,) or not counts.is_contiguous()
                or counts.get_device() != index):
            raise ValueError(f"{what}: counts must be a contiguous int32 [{batch}] tensor on {cache.pool.device}")
        cp = counts.data_ptr()
    mp = shape[1]
    if batch > _MOST or tokens > _MOST or mp > _MOST:
        raise ValueError(f"{what}: too large a call")
    return _pack_rows(page_table.data_ptr(), lengths.data_ptr(), cp, max(strides[0], mp), mp, batch, tokens), \
        mp * cache.page_size


def _heads(t: torch.Tensor, shape: tuple, dtype, index: int, name: str) -> bytes:
    """The packed strides of a checked [B, T, heads, D] tensor."""
    if t.shape != shape or t.dtype != dtype or t.get_device() != index:
        raise ValueError(f"{name} must be {dtype} {list(shape)} on cuda:{index}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    sb, st, sh, sd = t.stride()
    if sd != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return _pack_strides(sb, st, sh)


def q4_kv_append(cache: Q4Cache, page_table: torch.Tensor, lengths: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                 q: torch.Tensor | None = None, counts: torch.Tensor | None = None, rope_base: float = 10000.0,
                 q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Rotate the new keys to their positions and put keys and values into the cache.

    k, v [B, T, kv_heads, D] (bf16 or fp32; strided views of a fused projection are fine) are the tokens
    at positions lengths[b] .. lengths[b] + counts[b] - 1 of row b (counts None: T each; tokens from
    counts[b] on are padding).  page_table int32 [B, max_pages] lists row b's pages in order.  With q
    [B, T, heads, D] the rotated queries are returned (or written into ``q_out``, which may be q; its
    padding is left as it was).  The lengths are not changed.  Rotation: rotate-half, angle
    position * rope_base^(-2 j / D) in fp64 for any position; k is quantised unrounded."""
    if k.dim() != 4:
        raise ValueError(f"q4_kv_append: k must be [B, T, kv_heads, D], got {tuple(k.shape)}")
    B, T = k.shape[:2]
    dt, dtype, index, D = _dtype(k, "q4_kv_append: k"), k.dtype, cache._index, cache.head_dim
    shape = (B, T, cache.kv_heads, D)
    ks = _heads(k, shape, dtype, index, "q4_kv_append: k")
    vs = _heads(v, shape, dtype, index, "q4_kv_append: v")
    rows, _ = _rows(cache, page_table, lengths, counts, B, T, "q4_kv_append")
    H, qs, qos, qp, qop = 0, None, None, None, None
    if q is not None:
        H = q.shape[2] if q.dim() == 4 else 0
        shape = (B, T, H, D)
        qs = _heads(q, shape, dtype, index, "q4_kv_append: q")
        if q_out is None:
            q_out = q.new_empty(shape)
        qos = _heads(q_out, shape, dtype, index, "q4_kv_append: q_out")
        qp, qop = q.data_ptr(), q_out.data_ptr()
        if not 1 <= H <= _MOST:
            raise ValueError(f"q4_kv_append: q needs between one and 2^31 - 1 heads, got {H}")
    elif q_out is not None:
        raise ValueError("q4_kv_append: q_out without q")
    if B == 0 or T == 0:
        return q_out
    _call(index, "evs_q4_kv_append", cache._ref, rows, k.data_ptr(), ks, v.data_ptr(), vs, qp, qs, qop, qos, H, dt,
          rope_base)
    return q_out


def q4_kv_read(cache: Q4Cache, page_table: torch.Tensor, starts: torch.Tensor, tokens: int, *,
               counts: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16,
               out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that the cache holds at positions starts[b] .. starts[b] + counts[b] - 1 (counts
    None: ``tokens`` each) -> k, v [B, tokens, kv_heads, D] (padding behind counts[b] is left unwritten)."""
    B, index = starts.shape[0] if starts.dim() == 1 else -1, cache._index
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError(f"q4_kv_read: tokens must not be negative, got {tokens}")
    rows, _ = _rows(cache, page_table, starts, counts, B, tokens, "q4_kv_read")
    shape = (B, tokens, cache.kv_heads, cache.head_dim)
    if out is None:
        if dtype not in _DT:
            raise ValueError(f"q4_kv_read: dtype must be bf16 or fp32, got {dtype}")
        out = tuple(cache.pool.new_empty(shape, dtype=dtype) for _ in range(2))
    k, v = out
    dt = _dtype(k, "q4_kv_read: k")
    ks = _heads(k, shape, k.dtype, index, "q4_kv_read: k")
    vs = _heads(v, shape, k.dtype, index, "q4_kv_read: v")
    if B == 0 or tokens == 0:
        return k, v
    _call(index, "evs_q4_kv_read", cache._ref, rows, k.data_ptr(), ks, v.data_ptr(), vs, dt)
    return k, v


def q4_attention(q: torch.Tensor, cache: Q4Cache, page_table: torch.Tensor, lengths: torch.Tensor, *,
                 counts: torch.Tensor | None = None, scale: float | None = None, max_length: int | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of new tokens over the cache, which holds their own keys already.

    q [B, T, heads, D] (bf16 or fp32, rotated), heads a multiple of kv_heads: query head h reads kv head
    h // (heads / kv_heads).  Token t < counts[b] of row b (counts None: T each) sits at position
    lengths[b] + t and sees positions 0 .. lengths[b] + t.  scale defaults to D^-0.5.  max_length, a host
    bound of lengths + counts, keeps the launch small; without it the page table's size bounds it.
    Returns [B, T, heads, D] in q's dtype, or fills ``out`` (padding behind counts[b] is left unwritten).

    ``out`` may be q.

    A token's result depends only on its position, its q and the keys it sees, bit for bit: not on the
    batch, the other tokens of the call, max_length or the page size.  One size matters: bf16 calls of more
    than 64 rows (T * heads / kv_heads, D = 128) sum in another order from position 4,096 on."""
    if q.dim() != 4:
        raise ValueError(f"q4_attention: q must be [B, T, heads, D], got {tuple(q.shape)}")
    B, T, H, _ = q.shape
    dt, index = _dtype(q, "q4_attention: q"), cache._index
    if not 1 <= H <= _MOST or H % cache.kv_heads:
        raise ValueError(f"q4_attention: heads ({H}) must be a multiple of kv_heads ({cache.kv_heads})")
    shape = (B, T, H, cache.head_dim)
    qs = _heads(q, shape, q.dtype, index, "q4_attention: q")
    if scale is None:
        scale = cache.head_dim ** -0.5
    elif not 0.0 < scale <= 1e38:
        raise ValueError(f"q4_attention: scale must be positive and at most 1e38, got {scale}")
    if max_length is not None and not 1 <= max_length < 2 ** 31:
        raise ValueError(f"q4_attention: max_length must be positive, got {max_length}")
    rows, positions = _rows(cache, page_table, lengths, counts, B, T, "q4_attention")
    if out is None:
        out = q.new_empty(shape)
    os_ = _heads(out, shape, q.dtype, index, "q4_attention: out")
    if B == 0 or T == 0:
        return out
    ml = 0 if max_length is None else max_length
    sizes = (B, T, H, min(ml, positions) if ml else positions)
    need = cache._workspace.get(sizes)
    if need is None:
        need = N.lib().evs_q4_attention_workspace(cache._ref, rows, H, ml)
        if len(cache._workspace) >= 256:
            cache._workspace.clear()
        cache._workspace[sizes] = need
    ws, wp = None, None
    if need > 0:
        ws = cache.pool.new_empty((need,))
        wp = ws.data_ptr()
    else:
        need = 0
    _call(index, "evs_q4_attention", cache._ref, rows, q.data_ptr(), qs, H, scale, ml, out.data_ptr(), os_, dt, wp, need)
    return out
