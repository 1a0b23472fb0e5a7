"""Forward-mode derivatives: the operators have none and say so, instead of an answer without a tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from dsalt_b200 import layers as Y


def calls(device):
    new = lambda *s: torch.ones(*s, device=device)  # noqa: E731
    ffn = [new(4, 64), new(96, 64), new(96, 64), new(64, 96)]
    heads = [new(4, 2, 64), new(4, 1, 64), new(4, 64), new(4, 64), new(64), new(64)]
    rope = lambda q, k, c, s, wq, wk: Y.qk_norm_rope(q, k, c, s, q_weight=wq, k_weight=wk)  # noqa: E731
    return [(Y.gated_ffn, ffn), (rope, heads)]


def refuse(device):
    for call, args in calls(device):
        for i in range(len(args)):
            with fw.dual_level():
                dual = [fw.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
                for enabled in (True, False):
                    with torch.set_grad_enabled(enabled), pytest.raises(RuntimeError, match="forward-mode"):
                        call(*dual)


def test_dual_tensors_are_refused():
    refuse("cpu")  # before anything else is looked at


@pytest.mark.gpu
def test_dual_tensors_are_refused_on_the_gpu():
    refuse("cuda")
    for call, args in calls("cuda"):  # a level without a dual argument changes nothing
        with fw.dual_level():
            call(*args)
