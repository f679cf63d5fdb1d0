"""The choice of the next tokens from rows of logits by temperature, top-k, top-p and min-p, with uniform numbers that the caller draws (llamd_fwd_sample).

Buffers are the caller's, on the device: ``DevBuf``, a plain address, or anything with ``data_ptr()`` (a torch tensor), whose type, shape and strides are then checked.
The call enqueues on the library's stream and does not wait; where a tensor is among its buffers it orders that stream with torch's current one, both ways.
``ops.sample`` takes and returns numpy arrays, ``model.CudaModel.sample`` a model's own logits.
"""
from __future__ import annotations

from ._lib import lib
from .backend import DevBuf, Malformed, ShapeError, Unsupported
from .paged import TYPES, _int, _one_device, _refuse, _stream_at, _type_of

MOST_TOKENS = 393216
_SIZE = {0: 2, 1: 2, 2: 4}


def _of_rows(x, n, dtype, what):
    """The address of n elements of 32 bits, or None."""
    if x is None:
        return None
    if hasattr(x, "data_ptr"):
        if str(x.dtype) != dtype or x.numel() != n or not x.is_contiguous() or not x.is_cuda:
            raise ShapeError(f"{what}: {x.dtype}, {tuple(x.shape)} on {x.device} for {n} rows")
        return x.data_ptr()
    if isinstance(x, DevBuf):
        if x.nbytes < 4 * n:
            raise ShapeError(f"{what}: {x.nbytes} bytes for {n} rows")
        return x.ptr
    return x


def sample(logits, uniform, token, temperature=None, top_k=None, top_p=None, min_p=None, prob=None, rows: int | None = None, n_vocab: int | None = None,
           dtype: str = "f32", stride: int | None = None) -> None:
    """A token for each row of logits. ``uniform`` f32, ``token`` i32 (out), ``temperature``, ``top_p``, ``min_p`` f32, ``top_k`` i32 and ``prob`` f32 (out):
    one element for each row, None for no limit. ``rows``, ``n_vocab``, ``dtype`` and ``stride`` (elements between rows) describe logits that are a plain address or
    a ``DevBuf``; a tensor [rows][n_vocab], its rows contiguous, says so itself."""
    if hasattr(logits, "data_ptr"):
        t = _type_of(logits)
        if t not in (0, 1, 2):
            raise Unsupported(f"logits in f32, f16 or bf16, not {logits.dtype}")
        if logits.dim() != 2 or not logits.is_cuda or (logits.shape[1] > 1 and logits.stride(1) != 1):
            raise ShapeError(f"logits: {tuple(logits.shape)} with strides {logits.stride()} on {logits.device}")
        rows, n_vocab = logits.shape
        stride = logits.stride(0) if rows > 1 else n_vocab
        ptr = logits.data_ptr()
    else:
        if dtype not in TYPES:
            raise Unsupported(f"logits in f32, f16 or bf16, not {dtype}")
        if rows is None or n_vocab is None:
            raise Malformed("logits at an address: rows and n_vocab")
        t, rows, n_vocab = TYPES[dtype], _int(rows, "rows"), _int(n_vocab, "n_vocab")
        stride = n_vocab if stride is None else _int(stride, "logits: elements between rows", 2 ** 40)
        if isinstance(logits, DevBuf) and rows and logits.nbytes < ((rows - 1) * stride + n_vocab) * _SIZE[t]:
            raise ShapeError(f"logits: {logits.nbytes} bytes for {rows} rows")
        ptr = logits.ptr if isinstance(logits, DevBuf) else logits
    if stride < n_vocab:
        raise ShapeError(f"rows of {n_vocab} logits {stride} apart")
    if uniform is None or token is None:
        raise Malformed("sample: a uniform number and a place for the token of each row")
    at = [_of_rows(x, rows, d, what) for x, d, what in ((temperature, "torch.float32", "temperature"), (top_k, "torch.int32", "top_k"), (top_p, "torch.float32", "top_p"),
                                                        (min_p, "torch.float32", "min_p"), (uniform, "torch.float32", "uniform"), (token, "torch.int32", "token"),
                                                        (prob, "torch.float32", "prob"))]
    stream, L = _stream_at(_one_device(logits, uniform, token, temperature, top_k, top_p, min_p, prob)), lib()
    if stream is not None and L.llamd_fwd_wait_stream(stream) != 0:
        _refuse("sample")
    if L.llamd_fwd_sample(ptr, t, stride, rows, n_vocab, *at) != 0:
        _refuse("sample")
    if stream is not None and L.llamd_fwd_ready_stream(stream) != 0:
        _refuse("sample")
