"""The two ends of a model over a vocabulary of tokens, on the device.

TokenOps has the embedding of tokens (a settling's input rows) and its gradient, and the losses of hidden states (a
settling's top) against labels or a teacher's top logits through an output matrix, with the gradients of both.  The
counterparts in the reference's device trainer are embed_gather, embed_scatter and ce_loss_grad
(PredictiveCoding.Device/Kernels/DeviceTrainKernels.cs:36-55,502-546).

Every operator has two forms: on DeviceTensors, which checks shapes and allocates what it returns, and `*_device` on raw
device pointers with everything named by the caller (dtype names "f32", "bf16", "f16"; pitches of 0 are the row's own
width).  16-bit bf16 tensors are uint16 bit patterns, as everywhere in this package.
"""
from __future__ import annotations

import numpy as np

from ._native import DTYPE, call
from .device import DeviceTensor, Stream
from .errors import ArgumentException

_NAMES = {np.dtype(np.float32): "f32", np.dtype(np.float16): "f16", np.dtype(np.uint16): "bf16"}


def _type(name: str) -> int:
    if name not in DTYPE:
        raise ArgumentException(f"unknown type {name!r}: one of {sorted(DTYPE)}")
    return DTYPE[name]


def _name(t: DeviceTensor, what: str) -> str:
    if t.dtype not in _NAMES:
        raise ArgumentException(f"{what} must be float32, float16 or uint16 (bf16); got {t.dtype}")
    return _NAMES[t.dtype]


def _matrix(t: DeviceTensor, what: str):
    if len(t.shape) != 2 or 0 in t.shape[1:]:
        raise ArgumentException(f"{what} must be a 2-D tensor with columns; got shape {t.shape}")
    return t.shape


def _ints(t: DeviceTensor, shape, what: str):
    if t.dtype != np.int32 or t.shape != tuple(shape):
        raise ArgumentException(f"{what} must be an int32 tensor of shape {tuple(shape)}; got {t.dtype} {t.shape}")


def _weights(t: DeviceTensor | None, rows: int):
    if t is not None and (t.dtype != np.float32 or t.shape != (rows,)):
        raise ArgumentException(f"row_weight must be a float32 tensor of shape {(rows,)}; got {t.dtype} {t.shape}")
    return None if t is None else t.ptr


def _handle(stream: Stream | None):
    return stream.handle if stream else None


def _done(stream: Stream | None):
    if stream is None:
        call("pcd_device_synchronize")


class TokenOps:
    """Embedding, cross entropy and distillation over a vocabulary (pcd_token_* in include/pcdevice.h)."""

    # ------------------------------------------------------------- embedding

    @staticmethod
    def embed_device(dtype: str, table: int, tokens: int, count: int, vocab: int, dim: int, out: int, scale: float = 1.0,
                     out_dtype: str | None = None, ld_table: int = 0, ld_out: int = 0, stream: Stream | None = None) -> None:
        """out[i] = scale * table[tokens[i]] on device pointers; queued on `stream`."""
        call("pcd_token_embed", _type(dtype), table, ld_table, tokens, count, vocab, dim, scale, out,
             _type(out_dtype or dtype), ld_out, _handle(stream))

    @staticmethod
    def embed(table: DeviceTensor, tokens: DeviceTensor, scale: float = 1.0, out: DeviceTensor | None = None,
              out_dtype=None, stream: Stream | None = None) -> DeviceTensor:
        """scale * table[tokens] as [tokens x dim], of the table's type or `out_dtype` (fp32 beside a 16-bit table: what
        a settling takes).  Tokens below 0 are padding: rows of zeros."""
        vocab, dim = _matrix(table, "table")
        _ints(tokens, tokens.shape[:1] or (1,), "tokens")
        n = tokens.shape[0]
        if out is None:
            out = DeviceTensor((n, dim), out_dtype or table.dtype, stream)
        elif out.shape != (n, dim):
            raise ArgumentException(f"out must have shape {(n, dim)}; got {out.shape}")
        if n:
            TokenOps.embed_device(_name(table, "table"), table.ptr, tokens.ptr, n, vocab, dim, out.ptr, float(scale),
                                  _name(out, "out"), stream=stream)
        _done(stream)
        return out

    @staticmethod
    def embed_grad_device(dtype: str, d_out: int, tokens: int, count: int, vocab: int, dim: int, d_table: int,
                          scale: float = 1.0, accumulate: bool = False, out_dtype: str | None = None, ld_out: int = 0,
                          ld_table: int = 0, stream: Stream | None = None) -> None:
        """The gradient of embed_device by its table on device pointers; `dtype` is d_table's, `out_dtype` d_out's."""
        call("pcd_token_embed_grad", _type(dtype), d_table, ld_table, tokens, count, vocab, dim, scale, int(accumulate),
             d_out, _type(out_dtype or dtype), ld_out, _handle(stream))

    @staticmethod
    def embed_grad(d_out: DeviceTensor, tokens: DeviceTensor, vocab: int, scale: float = 1.0,
                   d_table: DeviceTensor | None = None, accumulate: bool = False, dtype=None,
                   stream: Stream | None = None) -> DeviceTensor:
        """The table's gradient [vocab x dim]; with `accumulate` added to the given d_table (tied matrices)."""
        n, dim = _matrix(d_out, "d_out")
        _ints(tokens, (n,), "tokens")
        if d_table is None:
            if accumulate:
                raise ArgumentException("accumulate needs the d_table to add to")
            d_table = DeviceTensor((vocab, dim), dtype or d_out.dtype, stream)
        elif d_table.shape != (vocab, dim):
            raise ArgumentException(f"d_table must have shape {(vocab, dim)}; got {d_table.shape}")
        TokenOps.embed_grad_device(_name(d_table, "d_table"), d_out.ptr, tokens.ptr, n, vocab, dim, d_table.ptr, float(scale),
                                   accumulate, _name(d_out, "d_out"), stream=stream)
        _done(stream)
        return d_table

    # ---------------------------------------------------------------- losses

    @staticmethod
    def keep_logits(nbytes: int) -> None:
        """Most bytes of logits that the losses keep between their two passes (default 1 GiB; 0: none)."""
        if nbytes < 0:
            raise ArgumentException("a number of bytes is not negative")
        call("pcd_token_keep_logits", int(nbytes))

    @staticmethod
    def cross_entropy_device(dtype: str, hidden: int, weight: int, labels: int, rows: int, dim: int, vocab: int, loss: int,
                             d_hidden: int | None = None, d_weight: int | None = None, row_weight: int | None = None,
                             scale: float = 1.0, hidden_dtype: str | None = None, ld_hidden: int = 0, ld_weight: int = 0,
                             ld_dhidden: int = 0, ld_dweight: int = 0, stream: Stream | None = None) -> None:
        """Softmax cross entropy of scale * hidden . weight^T against labels on device pointers; `dtype` is weight's."""
        call("pcd_token_xent", _type(dtype), hidden, _type(hidden_dtype or dtype), ld_hidden, weight, ld_weight, labels,
             row_weight, rows, dim, vocab, scale, loss, d_hidden, ld_dhidden, d_weight, ld_dweight, _handle(stream))

    @staticmethod
    def distill_device(dtype: str, hidden: int, weight: int, teacher_ids: int, teacher_logits: int, top: int, rows: int,
                       dim: int, vocab: int, loss: int, temperature: float = 1.0, d_hidden: int | None = None,
                       d_weight: int | None = None, row_weight: int | None = None, scale: float = 1.0,
                       teacher_dtype: str = "f32", hidden_dtype: str | None = None, ld_hidden: int = 0, ld_weight: int = 0,
                       ld_dhidden: int = 0, ld_dweight: int = 0, stream: Stream | None = None) -> None:
        """The divergence from a teacher's top logits on device pointers; `dtype` is weight's."""
        call("pcd_token_distill", _type(dtype), hidden, _type(hidden_dtype or dtype), ld_hidden, weight, ld_weight,
             teacher_ids, teacher_logits, _type(teacher_dtype), top, row_weight, rows, dim, vocab, scale, temperature, loss,
             d_hidden, ld_dhidden, d_weight, ld_dweight, _handle(stream))

    @staticmethod
    def _head(hidden: DeviceTensor, weight: DeviceTensor):
        rows, dim = _matrix(hidden, "hidden")
        vocab, wide = _matrix(weight, "weight")
        if wide != dim:
            raise ArgumentException(f"hidden states of {dim} and a weight of {wide} columns")
        dtype, hidden_dtype = _name(weight, "weight"), _name(hidden, "hidden")
        if hidden_dtype not in (dtype, "f32"):
            raise ArgumentException(f"hidden states must have the weight's type {dtype} or be fp32; got {hidden_dtype}")
        return rows, dim, vocab, dtype, hidden_dtype

    @staticmethod
    def _outputs(hidden, weight, grads, stream):
        loss = DeviceTensor(hidden.shape[:1], np.float32, stream)
        if not grads:
            return loss, None, None
        return loss, DeviceTensor(hidden.shape, hidden.dtype, stream), DeviceTensor(weight.shape, weight.dtype, stream)

    @staticmethod
    def cross_entropy(hidden: DeviceTensor, weight: DeviceTensor, labels: DeviceTensor,
                      row_weight: DeviceTensor | None = None, scale: float = 1.0, grads: bool = False,
                      stream: Stream | None = None):
        """(loss [rows], d_hidden, d_weight) of softmax(scale * hidden . weight^T) against labels, the gradients None
        unless asked for.  Rows with a negative label or no weight are left out."""
        rows, dim, vocab, dtype, hidden_dtype = TokenOps._head(hidden, weight)
        _ints(labels, (rows,), "labels")
        w = _weights(row_weight, rows)
        loss, dh, dw = TokenOps._outputs(hidden, weight, grads, stream)
        if rows or grads:
            TokenOps.cross_entropy_device(dtype, hidden.ptr, weight.ptr, labels.ptr, rows, dim, vocab, loss.ptr,
                                          dh and dh.ptr, dw and dw.ptr, w, float(scale), hidden_dtype, stream=stream)
        _done(stream)
        return loss, dh, dw

    @staticmethod
    def distill(hidden: DeviceTensor, weight: DeviceTensor, teacher_ids: DeviceTensor, teacher_logits: DeviceTensor,
                temperature: float = 1.0, row_weight: DeviceTensor | None = None, scale: float = 1.0, grads: bool = False,
                stream: Stream | None = None):
        """(loss [rows], d_hidden, d_weight) of the divergence of softmax(scale * hidden . weight^T / temperature) from a
        teacher's top logits [rows x top]; slots with a negative id are not there."""
        rows, dim, vocab, dtype, hidden_dtype = TokenOps._head(hidden, weight)
        _matrix(teacher_logits, "teacher_logits")
        if teacher_logits.shape[0] != rows:
            raise ArgumentException(f"teacher logits of {teacher_logits.shape[0]} rows for {rows} hidden states")
        _ints(teacher_ids, teacher_logits.shape, "teacher_ids")
        teacher_dtype = _name(teacher_logits, "teacher_logits")
        w = _weights(row_weight, rows)
        loss, dh, dw = TokenOps._outputs(hidden, weight, grads, stream)
        if rows or grads:
            TokenOps.distill_device(dtype, hidden.ptr, weight.ptr, teacher_ids.ptr, teacher_logits.ptr,
                                    teacher_logits.shape[1], rows, dim, vocab, loss.ptr, float(temperature), dh and dh.ptr,
                                    dw and dw.ptr, w, float(scale), teacher_dtype, hidden_dtype, stream=stream)
        _done(stream)
        return loss, dh, dw
