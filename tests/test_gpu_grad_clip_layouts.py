"""Gradients with gaps in the clipping: those that share memory are refused before anything is scaled, those side by side in one
buffer are scaled each once.  Bounds as in test_gpu_grad_clip.py."""
import pytest
import torch

from tests import test_gpu_grad_clip as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("views", [
    lambda b: [b[:, 3:17], b[:, 3:17]], lambda b: [b[:, :4], b[:, 2:6]], lambda b: [b[:, :4], b[4]], lambda b: [b[:, ::2], b[:, ::3]],
    lambda b: [b[:21, 3:17], torch.ones(3, device="cuda"), b[20:, 5:8]]])
def test_gradients_with_gaps_that_share_memory_are_refused(views):
    from transformer_amd import clip_grad_norm_
    buf = torch.ones(40, 24, device="cuda")
    with pytest.raises(ValueError, match="share"):
        clip_grad_norm_(G.params(views(buf)), 1.0)
    assert torch.equal(buf, torch.ones(40, 24, device="cuda"))


def test_gradients_side_by_side_in_one_buffer():
    g = torch.Generator(device="cuda").manual_seed(3)
    buf = torch.randn(300, 96, generator=g, device="cuda")
    keep = buf.clone()
    G.check([buf[:, :31], buf[:, 31:64], buf[:, 64:90].t(), torch.randn(50, generator=g, device="cuda")], 2.0)
    assert torch.equal(buf[:, 90:], keep[:, 90:]) and not torch.equal(buf[:, :90], keep[:, :90])
