"""infmoe_experts_topk on batches of many slots: the plan over many blocks, tokens beyond what one launch has work items for."""
import numpy as np
import pytest

from oracle import topk_oracle as O
from tests.topk_util import assert_within, draw_experts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,k,E", [(16384, 1, 3), (17409, 1, 70), (9000, 2, 1024), (30011, 3, 130), (70001, 8, 64)])
def test_batches_of_many_blocks(lib, torch_cuda, T, k, E):
    """Up to 548 blocks of 1024 slots, with 1 to 16 stretches of them; slots without an expert, experts without a slot.  A sample
    of the rows against the oracle, the others by a second call on the rows in another order."""
    torch = torch_cuda
    from infmoe_amd import ops
    rng = np.random.default_rng(T)
    c = draw_experts(torch, rng, T, k, E, 16, 24, "relu", "bfloat16")
    ids = rng.integers(-1, max(E - 2, 1), (T, k)).astype(np.int32)
    ids[T // 2:] = np.where(rng.random((T - T // 2, k)) < 0.9, E - 1, ids[T // 2:])  # the last expert has most rows, E - 2 may have none
    c["ids"].copy_(torch.from_numpy(ids))
    y = ops.experts_topk(c["x"], c["ids"], c["weights"], c["wi"], c["wo"])
    some = np.unique(np.concatenate([[0, 1, T - 1], rng.choice(T, 500)]))
    exact = dict(c["exact"], x=c["exact"]["x"][some], ids=ids[some], weights=c["exact"]["weights"][some])
    assert_within(y[torch.from_numpy(some).cuda()], *O.experts_topk(**exact))
    order = torch.from_numpy(rng.permutation(T)).cuda()
    again = ops.experts_topk(c["x"][order], c["ids"][order], c["weights"][order], c["wi"], c["wo"])
    assert torch.equal(again, y[order])


def test_more_tokens_than_one_launch_has_work_items_for(lib, torch_cuda):
    """2^24 + 77 tokens: the weighted sum would be 2^32 work items and more.  Every row is one of 1000, with one of three
    experts or none, so that the whole result is known from 4000 rows."""
    torch = torch_cuda
    from infmoe_amd import ops
    T, E, d, h = (1 << 24) + 77, 3, 8, 16
    rng = np.random.default_rng(1)
    c = draw_experts(torch, rng, 1000, 1, E, d, h, "gated_silu", "float16")
    want, bound = np.zeros((E + 1, 1000, d)), np.zeros((E + 1, 1000, d))
    for e in range(E):
        want[e], bound[e] = O.experts_topk(**dict(c["exact"], ids=np.full((1000, 1), e), weights=np.ones((1000, 1))))
    g = torch.Generator(device="cuda").manual_seed(2)
    row = torch.randint(0, 1000, (T,), device="cuda", generator=g)
    ids = torch.randint(0, E + 1, (T, 1), device="cuda", generator=g, dtype=torch.int32)  # (E: no expert)
    y = ops.experts_topk(c["x"][row], ids, torch.ones(T, 1, device="cuda"), c["wi"], c["wo"], c["wi_1"], ffn="gated_silu")
    want, bound = torch.from_numpy(want).cuda(), torch.from_numpy(bound).cuda()
    for part in torch.arange(T, device="cuda").split(1 << 22):
        at = (ids[part, 0].long(), row[part])
        assert ((y[part].double() - want[at]).abs() <= bound[at]).all()


def test_many_blocks_in_a_graph_and_on_two_streams(lib, torch_cuda):
    """The plan of many blocks captured, replayed with other routings and eager work between, and on two streams at once."""
    torch = torch_cuda
    from infmoe_amd import ops
    rng = np.random.default_rng(4)
    T, k, E = 20011, 2, 100
    c = draw_experts(torch, rng, T, k, E, 16, 24, "gated_silu", "bfloat16")
    call = lambda: ops.experts_topk(c["x"], c["ids"], c["weights"], c["wi"], c["wo"], c["wi_1"], ffn="gated_silu")
    want = call()
    got, sides = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        c["ids"].copy_(torch.from_numpy(rng.integers(-1, E, (T, k)).astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())
        torch.cuda.synchronize()
