"""The operators for several experts per token have no backward pass: inputs that require a gradient are refused, not taken
out of the graph in silence."""
import pytest
import torch

from infmoe_amd import capi, ops


def inputs(device):
    g = torch.Generator().manual_seed(3)
    draw = lambda *shape: torch.randn(shape, generator=g).to(device)
    route = dict(logits=draw(4, 8), bias=draw(8))
    experts = dict(x=draw(4, 16), weights=draw(4, 2), wi=draw(3, 24, 16), wo=draw(3, 16, 24), wi_1=draw(3, 24, 16), out=draw(4, 16))
    lora = dict(x=draw(4, 16), w=draw(24, 16), a=draw(3, 4, 16), b=draw(3, 24, 4), scale=draw(3), out=draw(4, 24))
    return route, experts, lora


def calls(device):
    route, experts, lora = inputs(device)
    ids = torch.tensor([[0, 1], [2, 0], [1, 2], [0, 2]], dtype=torch.int32, device=device)
    adapter = torch.tensor([0, 2, -1, 1], dtype=torch.int32, device=device)
    return [(route, lambda: ops.route_topk(route["logits"], 2, bias=route["bias"])),
            (experts, lambda: ops.experts_topk(experts["x"], ids, experts["weights"], experts["wi"], experts["wo"], experts["wi_1"],
                                               ffn="gated_silu", out=experts["out"])),
            (lora, lambda: ops.lora_project(lora["x"], lora["w"], lora["a"], lora["b"], adapter, lora["scale"], out=lora["out"]))]


def refuses(tensors, call):
    for name, t in tensors.items():
        t.requires_grad_(True)
        with pytest.raises(capi.InfMoEError, match="gradient") as ei:
            call()
        assert ei.value.status == capi.ERR_INVALID_ARGUMENT, name
        t.requires_grad_(False)


def test_inputs_that_require_a_gradient_are_refused():
    for tensors, call in calls("cpu"):  # (before anything looks at the device)
        refuses(tensors, call)
        next(iter(tensors.values())).requires_grad_(True)
        with torch.no_grad(), pytest.raises(capi.InfMoEError, match="on the GPU"):
            call()


@pytest.mark.gpu
def test_with_gradients_off_they_are_inputs_like_others(lib, torch_cuda):
    for tensors, call in calls("cuda"):
        refuses(tensors, call)
        want = [v.clone() for v in (lambda r: r if isinstance(r, tuple) else (r,))(call())]
        for t in tensors.values():
            t.requires_grad_(True)
        for mode in (torch.no_grad, torch.inference_mode):
            with mode():
                got = call()
            got = got if isinstance(got, tuple) else (got,)
            assert all(torch.equal(g, w) for g, w in zip(got, want))
