"""A paged K/V cache held in 4 bits: what ``CuteChronos2Model.enable_turboquant_kv`` simulates, stored.

The TurboQuant hook quantises K and V and restores them in place; this cache keeps the codes.  Vectors of 64 values are
rotated (signs, permutation, Hadamard), each coordinate held as one of 16 Lloyd-Max levels and the norm in 16 bits: 34
bytes a vector where bf16 takes 128.  Tokens live in pages that a block table names per sequence; appending rotates the
keys to their positions on the way (rotate-half, like the model's attention), and attention works on the codes: it
rotates a query into the codes' frame and the result back out, never the cache.

Every method enqueues work on the current stream of the cache's device and returns; lengths, positions and tables stay on
the device (int32; int64 is converted first, a launch an operand).  There is no gradient: what a call returns is detached,
like all of this library's kernels'.  A sequence, position, page or length out of range sets a bit of the library's device status, which stands
until :meth:`PagedKV4Cache.check` reads it.
"""

from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import _native as nat
from .turboquant import TurboQuantParams

DIM = 64
NORMS = {"float16": 0, "bfloat16": 1}
DEV_CACHE_RANGE = nat.DEV_CACHE_RANGE
_CODES = {torch.bfloat16: nat.CC2_BF16, torch.float32: nat.CC2_F32}


def rope_rows(positions: int, theta: float, device) -> torch.Tensor:
    """(positions, 32, 2) float32 (cos, sin) of the fp32 angles position / theta^(2i/64), the model's rotation."""
    inv = 1.0 / theta ** (torch.arange(0, DIM, 2, dtype=torch.int64).float() / DIM)
    ang = torch.arange(positions, dtype=torch.float32, device=device)[:, None] * inv.to(device)[None]
    return torch.stack([ang.double().cos(), ang.double().sin()], -1).float()


def _quant(p: TurboQuantParams, which: str) -> tuple[nat.KV4Quant, np.ndarray, np.ndarray]:
    """-> the rotation, the upper half of the levels, the bounds between them"""
    if p.mode != "mse" or p.bits != 4 or p.rotation != "hadamard" or p.dim != DIM:
        raise ValueError(f"the {which} quantiser must be mode 'mse', 4 bits, rotation 'hadamard', dim {DIM}; got "
                         f"{p.mode!r}, {p.bits}, {p.rotation!r}, {p.dim}")
    if p.norm_dtype not in NORMS:
        raise ValueError(f"the cache holds norms in 16 bits (float16 or bfloat16), got {p.norm_dtype}")
    t = {k: p.tensors[k].cpu().numpy() for k in ("signs", "perm", "codebook", "boundaries")}
    # sign and magnitude: the upper levels and their mirror image (the Lloyd-Max iteration leaves the two halves apart
    # by 6e-5 of the norm at most; the cache keeps their mean)
    half = np.float32(0.5)
    levels = half * (t["codebook"][8:] - t["codebook"][7::-1])
    bounds = half * (t["boundaries"][8:] - t["boundaries"][6::-1])
    if np.abs(t["codebook"][8:] - levels).max() > 1e-3:
        raise ValueError(f"the {which} quantiser's codebook is not symmetric")
    if not (np.diff(levels) > 0).all() or not (np.diff(bounds) > 0).all() or levels[0] < 0 or levels[-1] > 1:
        raise ValueError(f"the {which} quantiser's levels must ascend between 0 and 1")
    if sorted(t["perm"].tolist()) != list(range(DIM)):
        raise ValueError(f"the {which} quantiser's permutation is none")
    signs = sum(1 << i for i in range(DIM) if t["signs"][i] < 0)
    return nat.KV4Quant(signs, (C.c_uint8 * DIM)(*(int(i) for i in t["perm"]))), levels, bounds


_PER = {torch.bfloat16: 7, torch.float32: 3}  # elements of 16 bytes, less one
_BYTES = (torch.bool, torch.uint8)
_raw_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream(i).cuda_stream in a fraction of its time


def _place(t: torch.Tensor, per: int) -> tuple[int, int, int] | None:
    """Address of t (rows, heads, 64), elements from row to row and from head to head, as the kernels take them: last
    axis dense, rows and heads on 16-byte boundaries (``per`` + 1 elements).  None where it does not lie so."""
    (rows, heads, last), at = t.stride(), t.data_ptr()
    return None if last != 1 or (rows | heads) & per or at & 15 else (at, rows, heads)


def _rows(t: torch.Tensor, per: int) -> tuple[torch.Tensor, tuple[int, int, int]]:
    """t, copied where the kernels cannot read it as it is, and where it lies."""
    at = _place(t, per)
    if at is None:
        t = t.clone(memory_format=torch.contiguous_format)
        at = _place(t, per)
    return t, at


class PagedKV4Cache:
    """``num_pages`` pages of ``page_size`` (16, 32, 64, 128, 256) tokens for ``num_heads`` key / value heads of 64.

    ``key`` and ``value`` are the quantisers (:class:`TurboQuantParams`, 4 bits, "mse", "hadamard"; default seeds 0 and
    1).  ``rope_theta`` None appends keys as they come; otherwise positions up to ``max_positions`` can be rotated to.
    ``pages`` is the storage (uint8, ``(num_pages, bytes of a page)``); pages can be copied or shared between sequences.
    """

    def __init__(self, num_pages: int, num_heads: int, *, page_size: int = 64, key: TurboQuantParams | None = None,
                 value: TurboQuantParams | None = None, rope_theta: float | None = 10000.0, max_positions: int = 8192,
                 device="cuda"):
        lib = nat.load()
        key = key or TurboQuantParams.build(DIM, 4, mode="mse", seed=0, device="cpu")
        value = value or TurboQuantParams.build(DIM, 4, mode="mse", seed=1, device="cpu")
        if key.norm_dtype != value.norm_dtype:
            raise ValueError("keys and values must hold their norms in the same type")
        if num_pages < 1 or num_pages > 2**31 - 1:
            raise ValueError(f"num_pages must be positive, got {num_pages}")
        if rope_theta is not None and max_positions < 1:
            raise ValueError(f"max_positions must be positive, got {max_positions}")
        (kq, levels, bounds), (vq, *v_book) = _quant(key, "key"), _quant(value, "value")
        if not (np.array_equal(levels, v_book[0]) and np.array_equal(bounds, v_book[1])):
            raise ValueError("keys and values must share one codebook")
        nbytes = C.c_size_t()
        if lib.cc2_kv4_page_bytes(page_size, num_heads, C.byref(nbytes)) != 0:
            raise ValueError(lib.cc2_last_error().decode())
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("cutechronos_b200 kernels take CUDA tensors only (no CPU path)")
        self._pages = torch.zeros(num_pages, nbytes.value, dtype=torch.uint8, device=device)
        self.device = self._pages.device
        self._at = self._pages.get_device()
        self.num_pages, self.num_heads, self.page_size = num_pages, num_heads, page_size
        self._rope = rope_rows(max_positions, rope_theta, self.device) if rope_theta is not None else None
        self._c = nat.KV4Cache(self._pages.data_ptr(), num_pages, page_size, num_heads, NORMS[key.norm_dtype],
                               self._rope.data_ptr() if self._rope is not None else None,
                               max_positions if self._rope is not None else 0, (C.c_float * 8)(*levels),
                               (C.c_float * 7)(*bounds), kq, vq)
        self._ref = C.byref(self._c)
        self._lib = lib
        self._plan = (None, 0)  # sizes of the last attention call, bytes of its workspace

    # The library holds these two by address: their contents may be written, they cannot be replaced.
    @property
    def pages(self) -> torch.Tensor:
        """The storage: uint8, (num_pages, bytes of a page)."""
        return self._pages

    @property
    def rope(self) -> torch.Tensor | None:
        """(max_positions, 32, 2) float32 (cos, sin) that keys and queries are rotated by; None without a rotation."""
        return self._rope

    # -- arguments ---------------------------------------------------------------------------
    # Plain code on purpose: a single-token step's kernels take about as long as these checks.
    def _call(self, fn, what: str, *args) -> None:
        """fn(cache, *args, stream) on the cache's device and the caller's current stream."""
        i = self._at
        if torch._C._cuda_getDevice() == i:
            status = fn(self._ref, *args, _raw_stream(i))
        else:
            with torch.cuda.device(i):
                status = fn(self._ref, *args, _raw_stream(i))
        if status:
            nat.check(status, what)

    def _index(self, t: torch.Tensor, what: str, dim: int = 1) -> torch.Tensor:
        if t.get_device() != self._at:
            raise RuntimeError(f"{what} must be on {self.device}, got {t.device}")
        if t.dim() != dim:
            raise ValueError(f"{what} must have {dim} axis(es), got shape {tuple(t.shape)}")
        if t.dtype != torch.int32:
            if t.dtype != torch.int64:
                raise TypeError(f"{what} must be int32 or int64, got {t.dtype}")
            return self._narrow(t)
        return t if t.is_contiguous() or t.stride(-1) == 1 else t.contiguous()

    def _narrow(self, t: torch.Tensor) -> torch.Tensor:
        """t in 32 bits; what does not fit stays out of range."""
        i, shape, stride = self._at, t.shape, t.stride()
        out = torch.empty(shape, dtype=torch.int32, device=self.device)
        args = t.data_ptr(), stride[0], stride[-1], shape[0] if len(shape) > 1 else 1, shape[-1], out.data_ptr()
        if torch._C._cuda_getDevice() == i:
            status = self._lib.cc2_kv4_index32(*args, _raw_stream(i))
        else:
            with torch.cuda.device(i):
                status = self._lib.cc2_kv4_index32(*args, _raw_stream(i))
        if status:
            nat.check(status, "cc2_kv4_index32")
        return out

    def _values(self, t: torch.Tensor, what: str) -> int:
        if t.get_device() != self._at:
            raise RuntimeError(f"{what} must be on {self.device}, got {t.device} (no CPU path)")
        if t.dim() != 3 or t.shape[2] != DIM:
            raise ValueError(f"{what} must be (tokens, heads, {DIM}), got {tuple(t.shape)}")
        code = _CODES.get(t.dtype)
        if code is None:
            raise TypeError(f"{what}: dtype {t.dtype} not supported (bfloat16 / float32)")
        return code

    def _table(self, block_table: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
        """-> the table, its rows, its columns, elements from row to row"""
        t = self._index(block_table, "block_table", 2)
        rows, cols = t.shape
        if rows < 1 or cols < 1:
            raise ValueError(f"block_table is empty: {(rows, cols)}")
        ld = t.stride(0) if rows > 1 else cols
        if ld < cols:  # rows that overlap (an expanded row)
            t, ld = t.contiguous(), cols
        return t, rows, cols, ld

    def _places(self, seq_ids, positions, tokens: int | None):
        seq, pos = self._index(seq_ids, "seq_ids"), self._index(positions, "positions")
        n = seq.shape[0]
        if pos.shape[0] != n or (tokens is not None and n != tokens):
            raise ValueError(f"seq_ids and positions must name one place for each token, got {n} and {pos.shape[0]}"
                             + ("" if tokens is None else f" for {tokens}"))
        return seq, pos, n

    # -- operators ---------------------------------------------------------------------------
    def append(self, k: torch.Tensor, v: torch.Tensor, seq_ids: torch.Tensor, positions: torch.Tensor,
               block_table: torch.Tensor, *, token_mask: torch.Tensor | None = None) -> None:
        """Put k and v (tokens, heads, 64; bfloat16 or float32, any strides) at entries ``positions`` of sequences
        ``seq_ids``: page ``block_table[seq, pos // page_size]``, place ``pos % page_size``.  Keys are rotated to their
        positions.  ``token_mask`` 0 / False: attention will not see the token.  A negative sequence or position skips
        the token; no two tokens of a call may have the same place."""
        code = self._values(k, "k")
        if self._values(v, "v") != code or v.shape != k.shape or k.shape[1] != self.num_heads:
            raise ValueError(f"k and v must both be (tokens, {self.num_heads}, {DIM}) of one type, got "
                             f"{tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
        seq, pos, n = self._places(seq_ids, positions, k.shape[0])
        table, seqs, cols, ld = self._table(block_table)
        mask = None
        if token_mask is not None:
            if token_mask.shape != seq.shape or token_mask.device != self.device:
                raise ValueError("token_mask must have one entry for each token, on the cache's device")
            mask = token_mask if token_mask.dtype in _BYTES else token_mask != 0
            if not mask.is_contiguous():
                mask = mask.contiguous()
        per = _PER[k.dtype]
        (k, k_at), (v, v_at) = _rows(k, per), _rows(v, per)
        self._call(self._lib.cc2_kv4_append_cols, "cc2_kv4_append", code, *k_at, *v_at, n, seq.data_ptr(), pos.data_ptr(),
                   None if mask is None else mask.data_ptr(), table.data_ptr(), ld, cols, seqs)

    def read(self, seq_ids: torch.Tensor, positions: torch.Tensor, block_table: torch.Tensor, *,
             dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """What the entries stand for, dense: (k, v), each (tokens, heads, 64), keys as they were rotated.  Masked
        tokens read like others; skipped ones give zeros."""
        code = _CODES.get(dtype)
        if code is None:
            raise TypeError(f"dtype {dtype} not supported (bfloat16 / float32)")
        seq, pos, n = self._places(seq_ids, positions, None)
        table, seqs, cols, ld = self._table(block_table)
        k = torch.empty((n, self.num_heads, DIM), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        self._call(self._lib.cc2_kv4_read_cols, "cc2_kv4_read", code, k.data_ptr(), v.data_ptr(), n, seq.data_ptr(),
                   pos.data_ptr(), table.data_ptr(), ld, cols, seqs)
        return k, v

    def attention(self, q: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor, *,
                  cu_q: torch.Tensor | None = None, max_q: int | None = None, max_len: int | None = None,
                  causal: bool = True, scale: float = 1.0, rotate_q: bool = False, return_lse: bool = False,
                  out: torch.Tensor | None = None):
        """Attention of q (tokens, query heads, 64; bfloat16 or float32) over the cache -> the same shape and type.

        ``seq_lens`` counts each sequence's cached tokens, the queries' own among them.  Sequence s has the rows
        ``cu_q[s] : cu_q[s + 1]``, at most ``max_q`` (with ``cu_q`` the default is all rows of the call, and the kernel is
        chosen for that many: give the real bound), or without ``cu_q`` one equal share each, standing at its last positions;
        ``causal`` lets a row see the entries up to its own.  Query head h reads key head h // (query heads / heads).
        ``scale`` multiplies the scores (1, as in the model's attention); ``rotate_q`` rotates the queries to their
        positions.  ``max_len`` bounds seq_lens (default: what the block table has room for); a tighter bound splits the
        work better.  A row that sees no token gives 0, as does one of no sequence (before ``cu_q[0]``, from ``cu_q[-1]`` on),
        which in an ``out`` of the caller's is left alone.  With ``return_lse`` also the (tokens, query heads) float32
        logarithm of each row's sum of exponentials (-inf for such a row), to join it with attention over other keys.
        bfloat16 calls keep 11 bits of a weight times its value's norm down to 2^-20 of the row's largest weight times the
        sequence's largest norm."""
        code = self._values(q, "q")
        lens = self._index(seq_lens, "seq_lens")
        table, rows, cols, ld = self._table(block_table)
        total, heads, _ = q.shape
        seqs = lens.shape[0]
        if rows != seqs:
            raise ValueError(f"block_table has {rows} rows for {seqs} sequences")
        if heads == 0 or heads % self.num_heads:
            raise ValueError(f"{heads} query heads are no multiple of the cache's {self.num_heads}")
        if cu_q is None:
            if total % seqs or (max_q is not None and max_q != total // seqs):
                raise ValueError(f"{total} query rows are no equal shares of {seqs} sequences: give cu_q")
            max_q, cu = total // seqs, None
        else:
            cu_q = self._index(cu_q, "cu_q")
            if cu_q.shape[0] != seqs + 1:
                raise ValueError(f"cu_q must have {seqs + 1} entries, got {cu_q.shape[0]}")
            max_q, cu = total if max_q is None or max_q > total else int(max_q), cu_q.data_ptr()
        room = cols * self.page_size
        max_len = room if max_len is None or max_len > room else int(max_len)
        if max_q < 0 or max_len < 0:
            raise ValueError("max_q and max_len must not be negative")
        if rotate_q and self._rope is None:
            raise ValueError("the cache was made without a rotation (rope_theta None)")
        per = _PER[q.dtype]
        q, q_at = _rows(q, per)
        fill = 2 if return_lse else 0  # what this call allocates is written whole
        if out is None:
            fill |= 1
            out = torch.empty_like(q) if q.is_contiguous() else torch.empty_like(q, memory_format=torch.contiguous_format)
            out_at = (out.data_ptr(), heads * DIM, DIM)
        else:
            out_at = None
            if out.shape == q.shape and out.dtype == q.dtype and out.device == self.device:
                out_at = _place(out, per)
            if out_at is None or any(n > 1 and st < DIM for n, st in zip(out.shape[:2], out_at[1:])):
                raise ValueError("out must have q's shape, type and device, its rows apart, dense and on 16-byte boundaries")
        lse = torch.empty((total, heads), dtype=torch.float32, device=self.device) if return_lse else None
        sizes = (code, heads, seqs, total, max_q, max_len)
        plan = self._plan  # another thread's call may leave its own at any time
        if plan[0] != sizes:
            nbytes = C.c_size_t()
            self._call(lambda ref, *a: self._lib.cc2_kv4_attention_workspace_bytes(ref, *a[:-1]),
                       "cc2_kv4_attention_workspace_bytes", *sizes, C.byref(nbytes))
            self._plan = plan = (sizes, nbytes.value)
        need = plan[1]
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self._call(self._lib.cc2_kv4_attention_fill, "cc2_kv4_attention", code, *q_at, *out_at, heads, seqs, total, cu,
                   max_q, lens.data_ptr(), max_len,
                   table.data_ptr(), ld, causal, scale, rotate_q, fill, None if lse is None else lse.data_ptr(),
                   None if ws is None else ws.data_ptr(), need)
        return (out, lse) if return_lse else out

    def check(self) -> None:
        """Wait for the device and raise if a cache call on it reported an error since the last check: a sequence,
        position, page or length out of range, or a kernel that gave up waiting.  A forward's errors are its own (see
        :meth:`CuteChronos2Model.set_device_checks`)."""
        with torch.cuda.device(self.device):
            status = self._lib.cc2_device_status_of(nat.DEV_CACHE, 1)
        if status < 0:
            nat.check(status, "cc2_device_status_of")
        if status:
            raise nat.NativeError(f"device status {status}" + (
                ": a sequence, position, page or length of a cache call was out of range"
                if status & DEV_CACHE_RANGE else ": a kernel of a cache call gave up waiting, its outputs are incomplete"))
