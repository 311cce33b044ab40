"""The packed language model's first call under graph capture: nothing it needs is made, or copied from the host, in it."""

import pytest
import torch

GPU = pytest.mark.gpu


def test_rotary_positions_are_made_with_the_model(pkg):
    # (made in the first packed call they were copied from host memory there, which a capture refuses)
    model = pkg.esmc.HipEsmc(torch.zeros(33, 128), [], torch.ones(128), n_heads=2, device="cpu")
    assert model._rotary.freq.shape == (32,) and model._rotary.freq.device == model.embed.device
    made = model._rotary
    assert model.float()._rotary is made and made.freq.dtype == torch.float64
    assert model.half()._rotary is made and made.freq.dtype == torch.float64
    model._apply(lambda t: t.to("meta"))  # another device
    assert model._rotary is not made and model._rotary.freq.device.type == "meta"
    assert not any("rotary" in n for n in model.state_dict())


@GPU
def test_first_packed_call_captured(gpu_lib, pkg):
    from test_gpu_esmc_packed import _gen, _model
    other, *_ = _model(pkg, 256, 384, 4, 1, seed=3)
    cu = torch.tensor([0, 100, 149, 150], dtype=torch.int32, device="cuda")
    ids = torch.randint(0, 33, (150,), generator=_gen(3)).cuda()
    other.packed_hidden_states(ids, cu)      # (libraries and the scratch are there, as in any program)
    model, *_ = _model(pkg, 256, 384, 4, 2)  # itself called for the first time in the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = model.packed_hidden_states(ids, cu)
    keep = pkg.scratch.current("cuda")
    want = model.packed_hidden_states(ids, cu)
    for _ in range(4):
        got.zero_()
        graph.replay()
        again = model.packed_hidden_states(ids, cu)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(again, want)
    del keep
