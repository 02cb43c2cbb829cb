"""CPU: what 8-bit rows say of an input norm, and the encoder that asks."""

import copy
import pickle

import pytest
import torch

from saeflow_amd import Fp8Encoder
from saeflow_amd.kernels import Fp8Rows


@pytest.mark.parametrize("normed", [None, False, True])
def test_views_and_copies_say_what_their_rows_said(normed):
    rows = Fp8Rows.empty(5, 200, "cpu", normed=normed)
    for made in (rows, rows[1:3], rows.to("cpu"), copy.copy(rows), copy.deepcopy(rows), pickle.loads(pickle.dumps(rows)),
                 Fp8Rows(rows.q, rows.scale, 200, normed=normed)):
        assert made.normed is normed
    assert Fp8Rows(rows.q, rows.scale, 200).normed is None
    with pytest.raises(AttributeError):
        rows.normed = True


def test_an_encoder_that_norms_refuses_rows_that_were_not():
    enc = object.__new__(Fp8Encoder)  # (its product needs a GPU)
    enc.input_norm, enc.activation = "layer_norm", "relu"
    rows = Fp8Rows.empty(5, 200, "cpu", normed=False)
    for call in (enc.encode, enc.encode_sparse):
        with pytest.raises(ValueError, match="not normed"):
            call(rows)
