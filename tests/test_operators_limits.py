"""Sizes that the operators for several experts per token cannot launch are refused before anything is; no GPU is touched."""
import pytest

from infmoe_amd import capi
from tests.test_operators_host import experts


@pytest.mark.parametrize("change", [
    dict(T=1 << 25, k=32, h=1 << 20, wi_stride=1 << 24, wo_stride=1 << 24),
    dict(T=1 << 30, k=1, d=1024, h=64, x_stride=1024, y_stride=1024, wi_stride=1 << 16, wo_stride=1 << 16),
    dict(T=1 << 30, k=1, d=1024, h=1024, dtype=2, x_stride=1024, y_stride=1024, wi_stride=1 << 20, wo_stride=1 << 20),
    dict(T=64, k=16, E=1024, h=1 << 23, wi_stride=1 << 27, wo_stride=1 << 27),
    dict(T=64, k=16, E=1024, d=1 << 23, x_stride=1 << 23, y_stride=1 << 23, wi_stride=1 << 28, wo_stride=1 << 28),
    dict(T=1 << 26, k=16, E=2, d=13, h=29),
])
def test_experts_refuse_more_tiles_than_a_launch_holds(change):
    assert experts(**change) == capi.ERR_INVALID_ARGUMENT
    assert b"experts_topk: more tiles" in capi.load().infmoe_last_error()


@pytest.mark.parametrize("sizes", [
    (4, 33, 8, 16, 24, 0), (4, 2, 1025, 16, 24, 0), (1 << 30, 2, 8, 16, 24, 0), ((1 << 31) - 1, 32, 1024, 1 << 23, 1 << 23, 0),
    (4, 2, 8, (1 << 23) + 1, 24, 0), (4, 2, 8, 16, (1 << 31) - 1, 2), (4, 2, 8, 16, 24, 3), (4, 2, 8, 16, 24, -1)])
def test_no_workspace_for_experts_that_are_refused(sizes):
    assert capi.load().infmoe_experts_topk_workspace_bytes(*sizes) == 0


@pytest.mark.parametrize("sizes", [
    (4, (1 << 23) + 1, 24, 4, 0), (4, 16, (1 << 31) - 1, 4, 0), (4, 16, 24, 257, 0), (4, 16, 24, (1 << 31) - 1, 0), (4, 16, 24, 4, 3), (4, 16, 24, 4, -1)])
def test_no_workspace_for_adapters_that_are_refused(sizes):
    assert capi.load().infmoe_lora_project_workspace_bytes(*sizes) == 0


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
@pytest.mark.parametrize("T", [64, 300])
def test_partial_sums_only_for_rows_of_whole_pieces(dtype, size, T):
    """K is cut over workgroups for rows of whole 16-byte pieces only; others need no more than the adapters' first product."""
    bytes_of = capi.load().infmoe_lora_project_workspace_bytes
    first = (T * 16 * size + 255) // 256 * 256
    assert bytes_of(T, 4096, 1024, 16, dtype) > first
    assert bytes_of(T, 4097, 1024, 16, dtype) == first
