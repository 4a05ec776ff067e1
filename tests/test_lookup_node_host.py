"""Building and loading of the autograd node.  No GPU."""

from __future__ import annotations

import os

import pytest
import torch

from skyrl_amd import _lib
from skyrl_amd import embedding as E
from skyrl_amd.csrc import build as B


def test_it_loads_beside_the_library():
    node = _lib.load_node()
    assert os.path.samefile(node.__file__, B.node_path()) and node is _lib.load_node()


def test_a_missing_node_is_an_error_and_not_another_path(monkeypatch):
    monkeypatch.setattr(_lib, "_node", None)
    monkeypatch.setattr(_lib, "_NODE_PATH", os.path.join(B.HERE, "not_there.so"))
    with pytest.raises(_lib.LmHeadLibraryError, match="not built"):
        _lib.load_node()


def test_no_gradients_on_the_cpu():
    weight = torch.zeros(4, 8, requires_grad=True)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        E.embedding_lookup(weight, torch.zeros(2, dtype=torch.int64))


def test_the_build_line_is_for_the_host_alone():
    line = B.node_command("out.so")
    assert os.path.basename(line[0]) == "g++" and line[-1].startswith("-l") and not any("offload" in x or x.endswith(".hip") for x in line)
