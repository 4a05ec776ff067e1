"""What the head with adapters does with operands that ask for a gradient: it gives one, or refuses.  No GPU: CPU operands get as far as their refusal."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad

from skyrl_amd import _lib
from skyrl_amd import adapters as AD

NAMES = ("hidden", "weight", "lora_a", "lora_b", "scaling")


def operands():
    b16 = torch.bfloat16
    return {"hidden": torch.ones(3, 64, dtype=b16), "weight": torch.ones(50, 64, dtype=b16), "lora_a": torch.ones(2, 8, 64, dtype=b16),
            "lora_b": torch.ones(2, 50, 8, dtype=b16), "scaling": torch.ones(2), "adapter_ids": torch.zeros(3, dtype=torch.int64)}


@pytest.mark.parametrize("name", NAMES)
def test_logits_are_not_detached_in_silence(name):
    x = operands()
    x[name].requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        AD.adapter_logits(**x)
    x[name] = x[name] * 1.0  # an activation
    with pytest.raises(ValueError, match="no gradient"):
        AD.adapter_logits(**x)
    for quiet in (torch.no_grad, torch.inference_mode):
        with quiet(), FakeTensorMode(allow_non_fake_inputs=True):
            assert AD.adapter_logits(**x).shape == (3, 50)


@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_is_refused(name):
    x = operands()
    with forward_ad.dual_level():
        x[name] = forward_ad.make_dual(x[name], torch.ones_like(x[name]))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(ValueError, match="no gradient"):
                AD.adapter_logits(**x)
        if name in ("hidden", "lora_a", "lora_b"):  # autograd's function has no forward formula and says so
            with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(RuntimeError, match="forward"):
                AD.adapter_logprobs_from_hidden(x["hidden"], x["weight"], torch.zeros(3, dtype=torch.int64), x["lora_a"], x["lora_b"], x["scaling"],
                                                x["adapter_ids"])


def test_a_frozen_batch_gets_logits():
    with FakeTensorMode(allow_non_fake_inputs=True):
        assert AD.adapter_logits(**operands()).shape == (3, 50)


@pytest.mark.parametrize("H,V", [(896, 151936), (3584, 152064)])
def test_no_room_is_taken_for_a_gradient_of_the_weight(H, V):
    """From the second block of 32768 tokens on the head keeps dW's sum, V H fp32; with adapters there is no dW, only dB's sum, N V R fp32."""
    lib = _lib.load()
    head = [lib.skyrl_lmhead_bwd_active_rows_workspace_bytes(T, H, V, 0) for T in (32768, 32769)]
    ours = [lib.skyrl_lmhead_adapter_bwd_workspace_bytes(T, H, V, 1, 8) for T in (32768, 32769)]
    assert head[1] - head[0] >= 4 * V * H
    assert 4 * V * 8 <= ours[1] - ours[0] <= 4 * V * 8 + (1 << 20)
