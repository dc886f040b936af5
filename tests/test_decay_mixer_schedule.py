"""DecayTokenMixer's schedule: one tensor a device for all of a module's calls, whoever asks first."""

import copy

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F


def test_schedule_asked_for_in_inference_mode_can_be_saved_for_backward():
    layer = F.DecayTokenMixer(16, num_heads=4)
    with torch.inference_mode():
        on_meta = layer.log_decay("meta")  # a device that the module was not made on
        here = layer.log_decay("cpu")
    assert not on_meta.is_inference() and not here.is_inference()

    class Save(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, a):
            ctx.save_for_backward(a)
            return x * a

        @staticmethod
        def backward(ctx, g):
            return g * ctx.saved_tensors[0], None

    x = torch.ones(4, requires_grad=True)
    Save.apply(x, layer.log_decay("cpu")).sum().backward()
    assert torch.equal(x.grad, here)


def test_schedule_stays_fp32_through_casts_and_copies():
    layer = F.DecayTokenMixer(16, num_heads=4)
    want = layer.log_decay("cpu").clone()
    for other in (layer.half(), copy.deepcopy(layer), layer.double()):
        assert other.log_decay("cpu").dtype == torch.float32
        assert torch.equal(other.log_decay("cpu"), want)
    assert set(layer.state_dict()) == {"norm.weight", "norm.bias", "qkv_proj.weight",
                                       "qkv_proj.bias", "out_proj.weight", "out_proj.bias"}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_serving_before_training(dtype):
    torch.manual_seed(0)
    layer = F.DecayTokenMixer(32, num_heads=2).to("cuda", dtype)
    x = torch.randn(2, 70, 32, device="cuda", dtype=dtype)
    with torch.inference_mode():
        served, state = layer(x, return_state=True)
        layer.step(x[:, 0], state)
    y = layer(x)
    assert torch.equal(y, served)
    y.float().square().sum().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in layer.parameters())


@pytest.mark.gpu
def test_schedule_is_there_before_the_first_call():
    """A first call may be captured in a graph, where nothing can be copied from the host."""
    layer = F.DecayTokenMixer(32, num_heads=2).to("cuda:0")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        twice = layer.log_decay(torch.device("cuda:0")) * 2
    graph.replay()
    assert torch.equal(twice.cpu(), layer.log_decay("cpu") * 2)
