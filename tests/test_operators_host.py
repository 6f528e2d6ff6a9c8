"""What the entry points for several experts per token refuse, and empty batches; no GPU is touched."""
import ctypes as C

import pytest

from infmoe_amd import capi

P = C.create_string_buffer(64)  # stands for a device buffer: a refused call never looks at it


def route(**change):
    a = dict(T=4, E=8, k=2, dtype=0, logits=P, stride=8, score=0, bias=None, groups=1, top_groups=1, group_top=1,
             renormalize=1, scale=1.0, ids=P, weights=P, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return capi.load().infmoe_route_topk(*[C.cast(v, C.c_void_p) if v is P else v for v in a.values()])


@pytest.mark.parametrize("change", [
    dict(T=-1), dict(E=0), dict(E=1025, stride=1025), dict(k=0), dict(k=9), dict(E=64, stride=64, k=33), dict(dtype=3), dict(dtype=-1),
    dict(score=2), dict(groups=0), dict(groups=3), dict(E=130, stride=130, groups=65), dict(groups=2, top_groups=3), dict(top_groups=0),
    dict(groups=4, top_groups=1, k=3), dict(group_top=0), dict(group_top=3), dict(groups=8, top_groups=8, group_top=2), dict(stride=7),
    dict(logits=None), dict(ids=None), dict(weights=None),
])
def test_route_refuses(change):
    assert route(**change) == capi.ERR_INVALID_ARGUMENT
    assert b"route_topk" in capi.load().infmoe_last_error()


def test_route_of_no_rows_needs_no_memory():
    assert route(T=0, logits=None, ids=None, weights=None) == capi.OK


def experts(**change):
    a = dict(T=4, k=2, E=3, d=16, h=24, ffn=1, dtype=0, x=P, x_stride=16, ids=P, weights=P, wi=P, wi_1=P, wo=P, wi_stride=384,
             wo_stride=384, y=P, y_stride=16, workspace=256 * 1024, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return capi.load().infmoe_experts_topk(*[C.cast(v, C.c_void_p) if v is P else v for v in a.values()])


@pytest.mark.parametrize("change", [
    dict(T=-1), dict(k=0), dict(k=33), dict(E=0), dict(E=1025), dict(T=1 << 30, k=2), dict(d=0), dict(h=0), dict(h=(1 << 24) + 1, wi_stride=1 << 40, wo_stride=1 << 40),
    dict(ffn=3), dict(ffn=-1), dict(dtype=3), dict(x_stride=15), dict(y_stride=15), dict(wi_stride=383), dict(wo_stride=383), dict(x=None),
    dict(ids=None), dict(weights=None), dict(wi=None), dict(wo=None), dict(y=None), dict(workspace=None), dict(workspace=256 * 1024 + 64),
    dict(ffn=0), dict(ffn=1, wi_1=None), dict(ffn=2, wi_1=None),
])
def test_experts_refuse(change):
    assert experts(**change) == capi.ERR_INVALID_ARGUMENT
    assert b"experts_topk" in capi.load().infmoe_last_error()


def test_experts_of_no_rows_need_no_memory():
    assert experts(T=0, x=None, ids=None, weights=None, wi=None, wi_1=None, wo=None, y=None, workspace=None) == capi.OK
    size = capi.load().infmoe_experts_topk_workspace_bytes
    assert size(0, 2, 3, 16, 24, 0) == 0 and size(-1, 2, 3, 16, 24, 0) == 0
    assert 0 < size(1, 2, 3, 16, 24, 2) <= size(2, 2, 3, 16, 24, 2) <= size(2, 2, 3, 16, 24, 0)


def lora(**change):
    a = dict(T=4, d=16, n=24, r=4, L=3, dtype=2, x=P, x_stride=16, w=P, a=P, b=P, adapter=P, scale=P, y=P, y_stride=24, workspace=256 * 1024, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return capi.load().infmoe_lora_project(*[C.cast(v, C.c_void_p) if v is P else v for v in a.values()])


@pytest.mark.parametrize("change", [
    dict(T=-1), dict(d=0), dict(n=0), dict(r=0), dict(r=257), dict(L=0), dict(dtype=3), dict(x_stride=15), dict(y_stride=23), dict(x=None), dict(w=None),
    dict(a=None), dict(b=None), dict(adapter=None), dict(y=None), dict(workspace=None), dict(workspace=256 * 1024 + 64), dict(d=(1 << 24) + 1, x_stride=1 << 25),
])
def test_lora_refuses(change):
    assert lora(**change) == capi.ERR_INVALID_ARGUMENT
    assert b"lora_project" in capi.load().infmoe_last_error()


def test_lora_of_no_rows_needs_no_memory():
    assert lora(T=0, x=None, w=None, a=None, b=None, adapter=None, y=None, workspace=None) == capi.OK
    assert capi.load().infmoe_lora_project_workspace_bytes(0, 16, 24, 4, 0) == 0
