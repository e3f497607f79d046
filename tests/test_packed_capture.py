"""A PackedSequences' lists are copied to the device at the first call of their kind, which waits for the copy: a graph
capture cannot hold it, and is told so before anything is added to it."""
import pytest
import torch

from vmonarch_b200 import PackedSequences, gated_residual_norm, packed_attention


def test_refused_while_capturing(monkeypatch):
    seqs = PackedSequences([30, 5], device="cpu")
    monkeypatch.setattr(PackedSequences, "_stream", lambda seqs: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    seqs.device = torch.device("cuda", 0)
    for first in (seqs._starts, lambda: seqs._template((False, True, 0.125, torch.bfloat16, 2, 2, 64))):
        with pytest.raises(AssertionError, match="before the capture"):
            first()
    assert not seqs._cache


@pytest.mark.gpu
def test_first_call_in_a_capture_and_after_it():
    x = torch.randn(35, 2, 64, device="cuda").to(torch.bfloat16)
    scale = torch.randn(2, 64, device="cuda").to(torch.bfloat16)
    seqs = PackedSequences([30, 5])
    for call in (lambda: packed_attention(x, x, x, seqs), lambda: gated_residual_norm(x[:, 0], scale=scale, seqs=seqs)[1]):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(AssertionError, match="before the capture"):
            with torch.cuda.graph(graph):
                call()
        want = call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        graph.replay()
        assert torch.equal(got, want)
