"""What the token operators refuse, before any device call (no GPU needed)."""
import math

import numpy as np
import pytest

from predicitivecoding_amd import ArgumentException, TokenOps, _native
from predicitivecoding_amd.errors import DeviceException, DeviceStatus

P = 4096   # an address that no refused call reads


def refused(fn, *args, **kwargs):
    with pytest.raises(DeviceException) as e:
        fn(*args, **kwargs)
    assert e.value.code == DeviceStatus.InvalidValue
    return str(e.value)


def test_embed_refusals():
    ok = dict(dtype="bf16", table=P, tokens=P, count=4, vocab=10, dim=8, out=P)
    for bad in (dict(table=None), dict(tokens=None), dict(out=None), dict(count=-1), dict(vocab=0), dict(dim=0),
                dict(ld_table=7), dict(ld_out=7), dict(ld_out=-8), dict(out_dtype="f16")):
        refused(TokenOps.embed_device, **{**ok, **bad})
    with pytest.raises(ArgumentException):
        TokenOps.embed_device(**{**ok, "dtype": "f8"})
    TokenOps.embed_device(**{**ok, "count": 0, "tokens": None, "out": None})   # nothing to do


def test_embed_grad_refusals():
    ok = dict(dtype="f32", d_out=P, tokens=P, count=4, vocab=10, dim=8, d_table=P)
    for bad in (dict(d_out=None), dict(tokens=None), dict(d_table=None), dict(count=-1), dict(vocab=0), dict(dim=-3),
                dict(ld_table=7), dict(ld_out=7), dict(dtype="bf16", out_dtype="f16")):
        refused(TokenOps.embed_grad_device, **{**ok, **bad})
    TokenOps.embed_grad_device(**{**ok, "count": 0, "tokens": None, "d_out": None, "accumulate": True})


LOSS = dict(dtype="bf16", hidden=P, weight=P, rows=4, dim=8, vocab=10, loss=P)
BAD_LOSS = (dict(hidden=None), dict(weight=None), dict(loss=None), dict(rows=-1), dict(dim=0), dict(vocab=0),
            dict(rows=2 ** 24 + 1), dict(ld_hidden=7), dict(ld_weight=7), dict(ld_dhidden=7), dict(ld_dweight=7),
            dict(scale=math.nan), dict(scale=math.inf), dict(hidden_dtype="f16"), dict(dtype="f32", hidden_dtype="bf16"))


def test_cross_entropy_refusals():
    for bad in BAD_LOSS + (dict(labels=None),):
        refused(TokenOps.cross_entropy_device, **{**LOSS, "labels": P, **bad})
    TokenOps.cross_entropy_device(**{**LOSS, "rows": 0, "hidden": None, "loss": None, "labels": None})   # nothing to do



def test_distill_refusals():
    ok = {**LOSS, "teacher_ids": P, "teacher_logits": P, "top": 4}
    for bad in BAD_LOSS + (dict(teacher_ids=None), dict(teacher_logits=None), dict(top=0), dict(top=1025),
                           dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.nan),
                           dict(temperature=math.inf), dict(temperature=1e-45)):
        refused(TokenOps.distill_device, **{**ok, **bad})
    with pytest.raises(ArgumentException):
        TokenOps.distill_device(**{**ok, "teacher_dtype": "i8"})


def test_unknown_types_are_refused_by_the_library():
    assert _native.lib().pcd_token_embed(7, P, 0, P, 1, 1, 1, 1.0, P, 0, 0, None) == DeviceStatus.InvalidValue
    assert _native.lib().pcd_token_embed_grad(0, P, 0, P, 1, 1, 1, 1.0, 0, P, 9, 0, None) == DeviceStatus.InvalidValue
    assert _native.lib().pcd_token_xent(3, P, 3, 0, P, 0, P, None, 1, 1, 1, 1.0, P, None, 0, None, 0, None) == \
        DeviceStatus.InvalidValue
    assert _native.lib().pcd_token_distill(0, P, 0, 0, P, 0, P, P, 5, 1, None, 1, 1, 1, 1.0, 1.0, P, None, 0, None, 0, None) == \
        DeviceStatus.InvalidValue


def test_a_negative_number_of_bytes_is_refused():
    with pytest.raises(ArgumentException):
        TokenOps.keep_logits(-1)


class Fake:
    """A DeviceTensor's shape and type without its memory."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype, self.ptr = tuple(shape), np.dtype(dtype), P


def test_tensor_forms_check_shapes_and_types():
    f, i = np.float32, np.int32
    h, w, y = Fake((4, 8), f), Fake((10, 8), f), Fake((4,), i)
    bad = [
        lambda: TokenOps.cross_entropy(h, Fake((10, 9), f), y),
        lambda: TokenOps.cross_entropy(h, w, Fake((5,), i)),
        lambda: TokenOps.cross_entropy(h, w, Fake((4,), f)),
        lambda: TokenOps.cross_entropy(h, w, y, row_weight=Fake((3,), f)),
        lambda: TokenOps.cross_entropy(Fake((4, 8), np.float16), w, y),
        lambda: TokenOps.cross_entropy(Fake((4,), f), w, y),
        lambda: TokenOps.distill(h, w, Fake((4, 3), i), Fake((4, 2), f)),
        lambda: TokenOps.distill(h, w, Fake((5, 3), i), Fake((5, 3), f)),
        lambda: TokenOps.distill(h, w, Fake((4, 3), i), Fake((4, 3), i)),
        lambda: TokenOps.embed(w, Fake((4,), f)),
        lambda: TokenOps.embed(Fake((10,), f), y),
        lambda: TokenOps.embed(w, y, out=Fake((5, 8), f)),
        lambda: TokenOps.embed_grad(h, Fake((3,), i), 10),
        lambda: TokenOps.embed_grad(h, y, 10, accumulate=True),
        lambda: TokenOps.embed_grad(h, y, 10, d_table=Fake((9, 8), f)),
    ]
    for call in bad:
        with pytest.raises(ArgumentException):
            call()


def test_more_logits_than_are_counted_are_refused():
    for rows, vocab in ((2 ** 24, 2 ** 15 + 1), (2 ** 15 + 1, 2 ** 24)):
        assert "2^39" in refused(TokenOps.cross_entropy_device, **{**LOSS, "labels": P, "rows": rows, "vocab": vocab})
        assert "2^39" in refused(TokenOps.distill_device, **{**LOSS, "teacher_ids": P, "teacher_logits": P, "top": 4,
                                                             "rows": rows, "vocab": vocab})


def test_factors_that_fp32_does_not_hold_are_refused():
    ok = {**LOSS, "teacher_ids": P, "teacher_logits": P, "top": 4}
    for bad in (dict(scale=3e38), dict(scale=-2.5e38)):   # times log2 e
        refused(TokenOps.cross_entropy_device, **{**LOSS, "labels": P, **bad})
    for bad in (dict(temperature=2e19), dict(temperature=1e-20), dict(scale=1e30, temperature=1e-9),
                dict(scale=-1e30, temperature=1e9)):
        refused(TokenOps.distill_device, **{**ok, **bad})


def test_rows_longer_than_an_int_counts_units_of_are_refused():
    # the last unit of a row, and a wave's last column, end past it
    for dim in (2 ** 30 + 1, 2 ** 31 - 1):
        refused(TokenOps.embed_device, "bf16", P, P, 1, 1, dim, P)
        refused(TokenOps.embed_grad_device, "bf16", P, P, 1, 1, dim, P)


def test_tokens_without_an_axis_are_refused():
    with pytest.raises(ArgumentException):
        TokenOps.embed(Fake((10, 8), np.float32), Fake((), np.int32))
