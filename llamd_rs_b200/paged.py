"""Many sequences over paged K/V caches: page bookkeeping, the batch of one step, and its two operators.

``Pages`` hands out page ids and counts who holds them; sequences that begin alike hold the beginning's pages together
(``fork``). ``Batch`` is the shape of one step, set once and used by every layer: ``append`` norms, rotates and stores the new
tokens, ``attention`` attends them. Buffers are the caller's, on the device: ``DevBuf``, a plain address, or anything with
``data_ptr()`` (a torch tensor), whose type, shape and strides are then checked. The calls enqueue on the library's stream
and do not wait. Where a tensor is among their buffers they order that stream with torch's current one, both ways: they read what the current stream
has written when they are made, and it reads what they have written. A caller whose buffers are in use on any other stream orders the
two with ``wait_for`` and ``ready_for``.
"""
from __future__ import annotations

import ctypes as C
import math
import operator
import sys

import numpy as np

from . import backend
from ._lib import lib
from .backend import DevBuf, LlamdError, Malformed, Other, ShapeError, Unsupported

TYPES = {"f16": 0, "bf16": 1, "f32": 2}
CACHES = {"i8": 3, "e4m3": 4}  # in 8 bits
SCALE_BLOCK = 16  # positions to a scale of theirs
_SCALES = 5  # (bytes: the exponent plus 127)
_SIZE = {0: 2, 1: 2, 2: 4, 3: 1, 4: 1, 5: 1}
_TORCH = {"torch.float16": 0, "torch.bfloat16": 1, "torch.float32": 2, "torch.int8": 3, "torch.float8_e4m3fn": 4, "torch.float8_e8m0fnu": 5, "torch.uint8": 5}
_seen = {}  # a tensor's dtype -> its number here, filled as they come
SCALING = {"none": 0, "linear": 1, "base": 2, "by_frequency": 3}


class OutOfPages(LlamdError):
    pass


def _type_of(x):
    t = _seen.get(x.dtype)
    if t is None:
        t = _seen[x.dtype] = _TORCH.get(str(x.dtype), -1)
    return t


def _int32s(x, what):
    """x as an int32 array; refused where a conversion would change a value."""
    a = np.asarray(x)
    if a.dtype != np.int32:
        if a.size and (a.dtype.kind not in "iu" or int(a.min()) < -2 ** 31 or int(a.max()) >= 2 ** 31):
            raise Malformed(f"{what}: {a.dtype}, not whole numbers of 32 bits")
        a = a.astype(np.int32)
    return np.ascontiguousarray(a)


def _int(x, what, below=2 ** 31):
    """x as a whole number from 0 on: what the library would else see the low bits of."""
    try:
        n = operator.index(x)
    except TypeError:
        n = -1
    if not 0 <= n < below:
        raise Malformed(f"{what}: {x!r} is not a whole number below {below}")
    return n


def _one_device(*buffers):
    """Refuses tensors that are not all on the current device: the library has that one, and another's memory may be out of a kernel's reach. -> the device, None
    where no buffer is a tensor."""
    here = None
    for x in buffers:
        if x is None:
            continue
        try:
            at = x.get_device()
        except AttributeError:  # (an address, a DevBuf)
            continue
        if at != here:
            if here is not None:
                raise ShapeError(f"tensors on devices {here} and {at}")
            here = at
    if here is not None:
        if here < 0:
            raise ShapeError("a tensor that is not on a device")
        torch = sys.modules["torch"]
        current = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)()
        if here != current:
            raise ShapeError(f"tensors on device {here} where {current} is the current one")
    return here


def _stream_at(device):
    """torch's current stream (a cudaStream_t) on _one_device's device."""
    if device is None:
        return None
    torch = sys.modules["torch"]
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # (0.1 us; the public way makes an object of it, 2.4 us)
    return raw(device) if raw else torch.cuda.current_stream(device).cuda_stream


def _stream_here(x):
    """The same of one tensor that is to be on the current device."""
    c, at = sys.modules["torch"]._C, x.get_device()
    try:
        if at == c._cuda_getDevice():
            return c._cuda_getCurrentRawStream(at)
    except AttributeError:
        pass
    return _stream_at(_one_device(x))


def _refuse(what):
    """The last call's own refusal as an error, read so that the next call starts clean."""
    why = backend._last_error() or what
    if lib().llamd_fwd_last_error() > 0:  # not a refusal: the device's own
        raise Other(why)
    raise Malformed(why)


def rope_table(rows: int, rot: int, freq_base: float, scaling: str = "none", factor: float = 1.0, original: int = 0) -> np.ndarray:
    """[rows][rot / 2][2] sines and cosines for ``Batch.append`` (llamd_cuda_rope_table_scaled). "by_frequency" ramps in the number of turns; a checkpoint
    whose loader ramps over the pair's index needs a table of its own, which append takes as well."""
    if scaling not in SCALING:
        raise Unsupported(f"rope scaling {scaling!r}: one of {', '.join(SCALING)}")
    if rows < 0 or rot < 2 or rot % 2:
        raise ShapeError(f"rope table of {rows} rows, {rot} elements")
    rows, rot, original = _int(rows, "rows"), _int(rot, "rotated elements"), _int(original, "trained positions")
    out = np.empty((rows, rot // 2, 2), dtype=np.float32)
    if lib().llamd_cuda_rope_table_scaled(backend._ptr(out), rows, rot, freq_base, SCALING[scaling], factor, original) != 0:
        _refuse("rope table")
    return out


class Pages:
    """Which pages of a pool are free, and how many sequences hold each of the others."""

    def __init__(self, n_pages: int, page_size: int):
        if n_pages < 1 or page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
            raise ShapeError(f"{n_pages} pages of {page_size} positions")
        self.n_pages, self.page_size = n_pages, page_size
        self._free = list(range(n_pages - 1, -1, -1))
        self._held = [0] * n_pages

    def free(self) -> int:
        return len(self._free)

    def grow(self, table: list, n_pos: int) -> None:
        """Adds pages to ``table`` until it holds n_pos positions; all or none."""
        more = -(-n_pos // self.page_size) - len(table)
        if more > len(self._free):
            raise OutOfPages(f"{more} pages wanted, {len(self._free)} free")
        for _ in range(more):
            table.append(self._free.pop())
            self._held[table[-1]] = 1

    def fork(self, table: list, n_pos: int) -> list:
        """A table of another sequence that begins with the first n_pos positions (whole pages) of this one."""
        if n_pos < 0 or n_pos % self.page_size or n_pos > len(table) * self.page_size:
            raise Malformed(f"{n_pos} positions of {len(table)} pages of {self.page_size} cannot be shared")
        shared = list(table[:n_pos // self.page_size])
        for p in shared:
            if not 0 <= p < self.n_pages or self._held[p] < 1:
                raise Malformed(f"page {p} is nobody's and cannot be shared")
        for p in shared:
            self._held[p] += 1
        return shared

    def release(self, table: list) -> None:
        """The sequence is done: pages that nobody else holds are free again. Where one of them is not held, nothing is released."""
        for i, p in enumerate(table):
            if not 0 <= p < self.n_pages or self._held[p] < 1:
                for x in table[:i]:
                    self._held[x] += 1
                raise Malformed(f"page {p} is released twice")
            self._held[p] -= 1
        self._free.extend(p for p in dict.fromkeys(table) if not self._held[p])
        table.clear()


class Batch:
    """One step's sequences over caches of one geometry (llamd_cuda_paged_new). ``cache``: None, the pools hold ``dtype``, or "i8" or "e4m3", codes in 8 bits
    beside pools of scales [n_pages][n_head_kv][page_size / 16] (llamd_cuda_paged_new8), which ``append`` and ``attention`` then take as well."""

    def __init__(self, n_head: int, n_head_kv: int, head_dim: int, page_size: int, dtype: str = "f16", cache: str | None = None):
        self.ptr = None
        if dtype not in ("f16", "bf16"):
            raise Unsupported(f"a paged cache holds f16 or bf16, not {dtype}")
        if cache is not None and cache not in CACHES:
            raise Unsupported(f"a paged cache in 8 bits holds {' or '.join(CACHES)}, not {cache}")
        backend._need_device()
        n_head, n_head_kv, head_dim, page_size = (_int(x, "paged batch") for x in (n_head, n_head_kv, head_dim, page_size))
        self.type = TYPES[dtype]
        self.n_head, self.n_head_kv, self.head_dim, self.page_size = n_head, n_head_kv, head_dim, page_size
        self.cache = self.type if cache is None else CACHES[cache]
        if cache is None:
            self.ptr = lib().llamd_cuda_paged_new(n_head, n_head_kv, head_dim, page_size, self.type)
        else:
            self.ptr = lib().llamd_cuda_paged_new8(n_head, n_head_kv, head_dim, page_size, self.type, self.cache)
        if not self.ptr:
            _refuse("paged batch")
        self.tokens, self.n_pages, self.scale = 0, 0, 1.0 / math.sqrt(head_dim)
        self._append, self._attention = lib().llamd_fwd_paged_append, lib().llamd_fwd_paged_attention
        if cache is not None:
            self._append, self._attention = lib().llamd_fwd_paged_append8, lib().llamd_fwd_paged_attention8
        self._wait, self._ready = lib().llamd_fwd_wait_stream, lib().llamd_fwd_ready_stream
        self._pool = 0

    def set(self, q_lens, kv_lens, pages, n_pages: int, n_shared: int = 0) -> None:
        """q_lens, kv_lens: new tokens and positions in all of every sequence; pages: their tables, rows of one int32 array or a
        list of lists; n_pages: the pools' size; n_shared: positions at the beginning that all of them have in common."""
        q, kv = _int32s(q_lens, "new-token counts").ravel(), _int32s(kv_lens, "lengths").ravel()
        n_pages, n_shared = _int(n_pages, "pages"), _int(n_shared, "shared positions")
        if not isinstance(pages, np.ndarray):
            rows = [_int32s(r if hasattr(r, "__array__") else list(r), "page ids").ravel() for r in pages]
            pages = np.full((len(rows), max([len(r) for r in rows] + [1])), -1, dtype=np.int32)  # (-1: refused where a sequence reaches it)
            for i, r in enumerate(rows):
                pages[i, :len(r)] = r
        pages = _int32s(pages, "page ids")
        if q.size != kv.size or pages.ndim != 2 or pages.shape[0] != q.size:
            raise ShapeError(f"{q.size} new-token counts, {kv.size} lengths, tables {pages.shape}")
        if lib().llamd_cuda_paged_set(self.ptr, q.size, backend._ptr(q), backend._ptr(kv), backend._ptr(pages), pages.shape[1], n_pages, n_shared) != 0:
            _refuse("paged batch")
        self.tokens, self.n_pages = int(q.sum()), n_pages
        self._pool = n_pages * self.n_head_kv * self.page_size * self.head_dim

    def _call(self, what, call, stream, *args):
        """One of the two calls, between the orders with the caller's stream where there is one."""
        if stream is not None and self._wait(stream) != 0:
            _refuse(what)
        if call(self.ptr, *args) != 0:
            _refuse(what)
        if stream is not None and self._ready(stream) != 0:
            _refuse(what)

    @staticmethod
    def _tensors(*wanted):
        """The addresses of (tensor, type, values at least, rows) that are all as plain as can be and on one device, or None: then each is looked at for itself."""
        found = []
        try:
            device = wanted[0][0].get_device()
            if device < 0:
                return None
            for x, type_, n, rows in wanted:
                if _seen.get(x.dtype) != type_ or x.get_device() != device or not x.is_contiguous() or x.numel() < n or (rows is not None and (x.shape[0] != rows or x.numel() != n)):
                    return None
                found.append(x.data_ptr())
        except (AttributeError, IndexError):
            return None
        return found

    def _rows(self, x, n, type_, what, stride=None):
        """(address, elements between tokens) of `tokens` rows of n elements."""
        try:
            ptr = x.data_ptr()
        except AttributeError:
            stride = n if stride is None else _int(stride, f"{what}: elements between tokens", 2 ** 40)
            if isinstance(x, DevBuf):
                if self.tokens and x.nbytes < ((self.tokens - 1) * stride + n) * _SIZE[type_]:
                    raise ShapeError(f"{what}: {x.nbytes} bytes for {self.tokens} tokens") from None
                return x.ptr, stride
            return x, stride
        if _seen.get(x.dtype) != type_ and _type_of(x) != type_:
            raise ShapeError(f"{what}: {x.dtype}")
        if x.numel() == self.tokens * n:
            if x.is_contiguous() and (not self.tokens or x.shape[0] == self.tokens):
                return ptr, n
            shape, st = x.shape, x.stride()
            if shape[0] == self.tokens and st[-1] == 1 and (len(shape) == 2 or (len(shape) == 3 and shape[2] == self.head_dim and (shape[1] == 1 or st[1] == self.head_dim))):
                return ptr, st[0] if shape[0] > 1 else n
        raise ShapeError(f"{what}: {tuple(x.shape)} with strides {x.stride()} for {self.tokens} tokens of {n // self.head_dim} heads of {self.head_dim}")

    def _whole(self, x, type_, n, what):
        """The address of n contiguous values at least."""
        try:
            ptr = x.data_ptr()
        except AttributeError:
            if isinstance(x, DevBuf):
                if x.nbytes < n * _SIZE[type_]:
                    raise ShapeError(f"{what}: {x.nbytes} bytes for {n} values") from None
                return x.ptr
            return x
        if (_seen.get(x.dtype) != type_ and _type_of(x) != type_) or x.numel() < n or not x.is_contiguous():
            raise ShapeError(f"{what}: {x.dtype}, {tuple(x.shape)} on {x.device} for {n} values")
        return ptr

    def append(self, q, k, v, q_out, k_pages, v_pages, rope=None, rot: int | None = None, interleaved: bool = False, q_norm=None, k_norm=None,
               eps: float = 1e-6, inputs: str | None = None, rope_rows: int | None = None, strides=(None, None, None), k_scales=None, v_scales=None) -> None:
        """llamd_fwd_paged_append, or _append8 with the scales of a cache in 8 bits. ``inputs`` ("f32" or the cache's type) and ``strides`` (elements between tokens of q, k, v)
        describe buffers that are plain addresses or ``DevBuf``; a tensor says so itself, and its table how many rows it has."""
        if inputs is None:
            it = _type_of(q) if hasattr(q, "data_ptr") else 2
        else:
            it = TYPES.get(inputs, -1)
        if it != 2 and it != self.type:
            raise Unsupported("append takes f32 or the cache's type")
        rot = (0 if rope is None else self.head_dim) if rot is None else _int(rot, "rotated elements")
        if rot and rope is None:
            raise Malformed("a rotation without its angles")
        if rope_rows is None:
            if not rot:
                rope_rows = 0
            elif hasattr(rope, "data_ptr"):
                if rope.dim() > 1 and rope.shape[0] * rot != rope.numel():
                    raise ShapeError(f"angles of {tuple(rope.shape)} for {rot} rotated elements")
                rope_rows = rope.numel() // rot
            elif isinstance(rope, DevBuf):
                rope_rows = rope.nbytes // (4 * rot)
            else:
                raise Malformed("rope_rows: how many positions the table has")
        else:
            rope_rows = _int(rope_rows, "rope_rows")
        D, T, t, c = self.head_dim, self.tokens, self.type, self.cache
        nq, nk = self.n_head * D, self.n_head_kv * D
        eight = c != t or k_scales is not None or v_scales is not None
        if eight:
            n_scales = self._scales_given(k_scales, v_scales)
        if rot and q_norm is not None and k_norm is not None:
            plain = (self._tensors((q, it, T * nq, T), (k, it, T * nk, T), (v, it, T * nk, T), (q_norm, 2, D, None), (k_norm, 2, D, None),
                                   (rope, 2, rope_rows * rot, None), (q_out, t, T * nq, T), (k_pages, t, self._pool, None), (v_pages, t, self._pool, None)) if not eight else
                     self._tensors((q, it, T * nq, T), (k, it, T * nk, T), (v, it, T * nk, T), (q_norm, 2, D, None), (k_norm, 2, D, None),
                                   (rope, 2, rope_rows * rot, None), (q_out, t, T * nq, T), (k_pages, c, self._pool, None), (v_pages, c, self._pool, None),
                                   (k_scales, _SCALES, n_scales, None), (v_scales, _SCALES, n_scales, None)))
            if plain and eight:
                self._call("append", self._append, _stream_here(q), plain[0], plain[1], plain[2], it, nq, nk, nk, plain[3], plain[4], eps, plain[5], rope_rows, rot,
                           interleaved, plain[6], nq, plain[7], plain[8], plain[9], plain[10])
                return
            if plain:
                self._call("append", self._append, _stream_here(q), plain[0], plain[1], plain[2], it, nq, nk, nk, plain[3], plain[4], eps, plain[5], rope_rows, rot,
                           interleaved, plain[6], nq, plain[7], plain[8])
                return
        stream = _stream_at(_one_device(q, k, v, q_out, k_pages, v_pages, rope, q_norm, k_norm, k_scales, v_scales))
        scales = self._scales_of(k_scales, v_scales) if eight else ()
        qp, qs = self._rows(q, nq, it, "q", strides[0])
        kp, ks = self._rows(k, nk, it, "k", strides[1])
        vp, vs = self._rows(v, nk, it, "v", strides[2])
        op, os_ = self._rows(q_out, nq, self.type, "q_out")
        self._call("append", self._append, stream, qp, kp, vp, it, qs, ks, vs,
                   None if q_norm is None else self._whole(q_norm, 2, D, "q_norm"), None if k_norm is None else self._whole(k_norm, 2, D, "k_norm"), eps,
                   self._whole(rope, 2, rope_rows * rot, "rope") if rot else None, rope_rows, rot, interleaved, op, os_,
                   self._whole(k_pages, c, self._pool, "k_pages"), self._whole(v_pages, c, self._pool, "v_pages"), *scales)

    def _scales_given(self, k_scales, v_scales):
        """How many scales a pool has of a cache in 8 bits; refused where they are missing, or the cache is not."""
        if self.cache == self.type:
            raise Malformed("scales of a cache that is not in 8 bits")
        if k_scales is None or v_scales is None:
            raise Malformed("a cache in 8 bits without its scales")
        return self._pool // (SCALE_BLOCK * self.head_dim)

    def _scales_of(self, k_scales, v_scales):
        """The scales' addresses where the cache is in 8 bits."""
        if self.cache == self.type and k_scales is None and v_scales is None:
            return ()
        n = self._scales_given(k_scales, v_scales)
        return self._whole(k_scales, _SCALES, n, "k_scales"), self._whole(v_scales, _SCALES, n, "v_scales")

    def attention(self, q, k_pages, v_pages, out, scale: float | None = None, out_f32: bool | None = None, k_scales=None, v_scales=None) -> None:
        """llamd_fwd_paged_attention, or _attention8 with the scales of a cache in 8 bits. ``out_f32`` says of an address that it takes f32; a tensor's type says so itself."""
        if out_f32 is None:
            out_f32 = hasattr(out, "data_ptr") and _type_of(out) == 2
        n = self.n_head * self.head_dim
        scale = self.scale if scale is None else scale
        c = self.cache
        if c != self.type or k_scales is not None or v_scales is not None:
            n_scales = self._scales_given(k_scales, v_scales)
            plain = self._tensors((q, self.type, self.tokens * n, self.tokens), (k_pages, c, self._pool, None), (v_pages, c, self._pool, None),
                                  (out, 2 if out_f32 else self.type, self.tokens * n, self.tokens), (k_scales, _SCALES, n_scales, None), (v_scales, _SCALES, n_scales, None))
            if plain:
                self._call("attention", self._attention, _stream_here(q), plain[0], n, plain[1], plain[2], plain[4], plain[5], plain[3], n, out_f32, scale)
                return
        else:
            plain = self._tensors((q, self.type, self.tokens * n, self.tokens), (k_pages, self.type, self._pool, None), (v_pages, self.type, self._pool, None),
                                  (out, 2 if out_f32 else self.type, self.tokens * n, self.tokens))
            if plain:
                self._call("attention", self._attention, _stream_here(q), plain[0], n, plain[1], plain[2], plain[3], n, out_f32, scale)
                return
        stream = _stream_at(_one_device(q, k_pages, v_pages, out, k_scales, v_scales))
        scales = self._scales_of(k_scales, v_scales)
        qp, qs = self._rows(q, n, self.type, "q")
        op, os_ = self._rows(out, n, 2 if out_f32 else self.type, "out")
        kp, vp = self._whole(k_pages, c, self._pool, "k_pages"), self._whole(v_pages, c, self._pool, "v_pages")
        self._call("attention", self._attention, stream, qp, qs, kp, vp, *scales, op, os_, out_f32, scale)

    def free(self) -> None:
        if self.ptr:
            lib().llamd_cuda_paged_free(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def status() -> int:
    """0 while every bounded wait inside the attention has been met; a failure is handed out once, and append and attention refuse until it has been read
    (llamd_fwd_paged_status; waits for the stream)."""
    return int(lib().llamd_fwd_paged_status())


def wait_limit(seconds: float) -> None:
    """How long a wait inside the attention may take (2 s unless it is set); 0: its tensor-core kernel gives up at once (llamd_fwd_paged_wait_limit)."""
    if not 0 <= seconds < 1e9:
        raise Malformed(f"a limit of {seconds} seconds")
    lib().llamd_fwd_paged_wait_limit(int(round(seconds * 1e9)))


def wait_for(stream: int) -> None:
    """What is enqueued through the library from here on waits for what ``stream`` (a cudaStream_t) holds now."""
    if lib().llamd_fwd_wait_stream(C.c_void_p(stream)) != 0:
        _refuse("wait_for")


def ready_for(stream: int) -> None:
    """What is enqueued on ``stream`` from here on waits for what the library's stream holds now."""
    if lib().llamd_fwd_ready_stream(C.c_void_p(stream)) != 0:
        _refuse("ready_for")
