"""A buffer that is accumulated into shares no memory with what is read beside it.  No GPU: the refusals stand in front of the look at the device."""

from __future__ import annotations

import pytest
import torch

from skyrl_amd import embedding as E


@pytest.mark.parametrize("begin,refused", [(0, True), (79, True), (80, False), (40, True)])
def test_a_gradient_inside_the_buffer(begin, refused):
    """80 elements of buffer, 24 of gradient."""
    flat = torch.zeros(200)
    buffer, d = flat[:80].view(10, 8), flat[begin:begin + 24].view(3, 8)
    with pytest.raises(ValueError if refused else RuntimeError) as e:
        E.embedding_backward_accumulate(d, torch.zeros(3, dtype=torch.int64), buffer)
    assert ("shares memory" in str(e.value)) == refused


def test_a_gradient_that_ends_in_the_buffer_and_one_row_of_it():
    flat = torch.zeros(200)
    buffer = flat[20:100].view(10, 8)
    for d in (flat[:24].view(3, 8), flat[24:32].expand(3, 8)):
        with pytest.raises(ValueError):
            E.embedding_backward_accumulate(d, torch.zeros(3, dtype=torch.int64), buffer)
    with pytest.raises(RuntimeError):  # columns that are not side by side are read from a copy, taken in front of the call
        E.embedding_backward_accumulate(flat[:96:4].view(3, 8), torch.zeros(3, dtype=torch.int64), buffer)


def test_ids_inside_the_buffer():
    buffer = torch.zeros(10, 8)
    ids = buffer.view(torch.int64).view(-1)[3:6]
    with pytest.raises(ValueError):
        E.embedding_backward_accumulate(torch.zeros(3, 8), ids, buffer)


def test_half_a_gradient_in_another_type():
    flat = torch.zeros(200)
    d = flat[60:100].view(torch.bfloat16)[:24].view(3, 8)
    with pytest.raises(ValueError):
        E.embedding_backward_accumulate(d, torch.zeros(3, dtype=torch.int64), flat[:80].view(10, 8))
