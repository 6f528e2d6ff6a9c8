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
