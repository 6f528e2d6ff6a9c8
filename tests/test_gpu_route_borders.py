"""infmoe_route_topk where scores meet at a border of the choice: group sums whose terms cancel, a large score without a bias
against a small one with it."""
import numpy as np
import pytest

from oracle import topk_oracle as O

pytestmark = pytest.mark.gpu
RTOL = 2.0 ** -17  # of a weight; derived in test_gpu_route.py


def check(got, want):
    ids, w = (g.cpu().numpy() for g in got)
    np.testing.assert_array_equal(ids, want[0])
    np.testing.assert_allclose(w, want[1], rtol=RTOL, atol=1e-38)


def cancelling_groups(rng, T, groups, per, score, size):
    """Logits and a bias for which the two best of every group of `per` add up to nearly the same number, through a bias of
    +size on the one and -size on the other; the group's other experts are far behind.  Rows in which two groups' sums lie
    closer than 64 bits tell apart (the sums' roundings are 3 * 2^-53 * size, a score's a few 2^-53) are left out."""
    p = np.full((T, groups, per), 0.05 / (groups * per) if score == "softmax" else 0.05)
    pair = 0.9 / groups if score == "softmax" else 0.9
    p[:, :, 0] = pair * rng.uniform(0.2, 0.8, (T, groups))
    p[:, :, 1] = pair * (1 + 10.0 ** rng.uniform(-8.5, -6.5, (T, groups)) * rng.choice([-1, 1], (T, groups))) - p[:, :, 0]
    x = (np.log(p) if score == "softmax" else np.log(p) - np.log1p(-p)).reshape(T, -1).astype(np.float32)
    bias = np.full((groups, per), -8.0 * size, np.float32)
    bias[:, 0], bias[:, 1] = size, -size
    wide = x.astype(np.float64)
    s = np.exp(wide) / np.exp(wide).sum(axis=1, keepdims=True) if score == "softmax" else 1 / (1 + np.exp(-wide))
    sums = np.sort(s.reshape(T, groups, per)[:, :, :2].sum(axis=2), axis=1)
    apart = np.diff(sums, axis=1).min(axis=1) > 1e-15 * (4 * size + 4)
    assert apart.mean() > 0.9
    return x[apart], bias.reshape(-1)


@pytest.mark.parametrize("score,size", [("softmax", 1.0), ("softmax", 30.0), ("softmax", 300.0), ("sigmoid", 1.0), ("sigmoid", 100.0), ("sigmoid", 3e4)])
@pytest.mark.parametrize("T,groups,top_groups,per", [(300, 2, 1, 2), (300, 8, 4, 2), (5000, 2, 1, 2), (5000, 8, 4, 32), (300, 4, 2, 64)])
def test_group_sums_that_cancel_are_ordered_in_64_bits(lib, torch_cuda, score, size, T, groups, top_groups, per):
    torch = torch_cuda
    from infmoe_amd import ops
    x, bias = cancelling_groups(np.random.default_rng(T + groups + per), T, groups, per, score, size)
    kw = dict(score=score, groups=groups, top_groups=top_groups, group_top=2)
    got = ops.route_topk(torch.from_numpy(x).cuda(), 2, bias=torch.from_numpy(bias).cuda(), **kw)
    check(got, O.route_topk(x, 2, bias=bias, **kw))


def test_a_group_sum_whose_terms_cancel(lib, torch_cuda):
    """Group sums 0.832025 and 0.8320276 behind terms of 108: FP32's sums stand the other way round, 4e-6 apart."""
    torch = torch_cuda
    from infmoe_amd import ops
    x = np.array([[0.01374958, -0.7145797, 0.4695681, -1.2847303]], np.float32)
    bias = np.array([107.59555, -107.59555, 0, 0], np.float32)
    kw = dict(score="sigmoid", groups=2, top_groups=1, group_top=2)
    want = O.route_topk(x, 2, bias=bias, **kw)
    assert want[0].tolist() == [[2, 3]]
    check(ops.route_topk(torch.from_numpy(x).cuda(), 2, bias=torch.from_numpy(bias).cuda(), **kw), want)


@pytest.mark.parametrize("T,E,groups", [(300, 1024, 1), (300, 990, 33), (300, 256, 1), (5000, 256, 8), (300, 40, 1), (5000, 1023, 3)])
@pytest.mark.parametrize("spread", [0.0, 1.0, 3.0])
def test_a_large_score_against_a_small_one_with_a_bias(lib, torch_cuda, T, E, groups, spread):
    """Softmax: one expert with half of the row's total against one whose bias is that half, from 1e-8 to 1e-5 apart.  The
    error of the row's total, which all scores share, moves the one and not the other.  (`spread` of the other logits: with
    0.0 all terms of the total are equal, and so are their roundings.)"""
    torch = torch_cuda
    from infmoe_amd import ops
    rng = np.random.default_rng(E + int(10 * spread))
    wide = spread * rng.standard_normal((T, E)) + rng.uniform(-2, 2, (T, 1))
    wide[:, 1] -= 20.0
    x = wide.astype(np.float32)
    total = np.exp(x[:, 1:].astype(np.float64)).sum(axis=1)
    near = 10.0 ** rng.uniform(-8, -5, T) * rng.choice([-1, 1], T)
    x[:, 0] = np.log(total) + np.log((0.5 + near) / (0.5 - near))
    bias = np.zeros(E, np.float32)
    bias[1] = 0.5
    s = np.exp(x.astype(np.float64))
    s /= s.sum(axis=1, keepdims=True)
    x = x[np.abs(s[:, 0] - s[:, 1] - 0.5) > 1e-14]  # (closer ones 64 bits do not tell apart)
    assert len(x) > 0.9 * T
    kw = dict(score="softmax", groups=groups, top_groups=groups)
    got = ops.route_topk(torch.from_numpy(x).cuda(), 2, bias=torch.from_numpy(bias).cuda(), **kw)
    check(got, O.route_topk(x, 2, bias=bias, **kw))


@pytest.mark.parametrize("E,k", [(128, 3), (128, 15), (256, 8), (200, 6)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_the_best_experts_in_a_few_lanes_of_a_row(lib, torch_cuda, E, k, score):
    """Rows of several experts per lane whose best ones are neighbours, so that most lanes list none, up to those where one
    lane has them all; and rows with fewer experts than k left, or with none."""
    torch = torch_cuda
    from infmoe_amd import ops
    rng = np.random.default_rng(E + k)
    T = 4100
    x = rng.standard_normal((T, E)).astype(np.float32)
    for t in range(T):
        at, count = rng.integers(E), rng.integers(1, 17)
        x[t, (at + np.arange(count)) % E] += 10.0
    x[::17] = -np.inf
    x[::17, 5] = np.where(rng.random(len(x[::17])) < 0.5, 1.0, -np.inf)
    for bias in (None, (0.01 * rng.standard_normal(E)).astype(np.float32)):
        got = ops.route_topk(torch.from_numpy(x).cuda(), k, score=score, bias=None if bias is None else torch.from_numpy(bias).cuda())
        check(got, O.route_topk(x, k, score=score, bias=bias))


@pytest.mark.parametrize("T,E,k", [((1 << 31) - 1, 1, 1), ((1 << 26) + 77, 20, 17), ((1 << 27) + 77, 2, 1)])
def test_more_rows_than_one_launch_has_work_items_for(lib, torch_cuda, T, E, k):
    """Rows of 16 lanes and of 64 beyond 2^32 work items, and the largest count there is.  Every row is one of 1000."""
    torch = torch_cuda
    from infmoe_amd import ops
    rng = np.random.default_rng(E)
    x = rng.standard_normal((1000, E)).astype(np.float16)
    ids, w = O.route_topk(x.astype(np.float32), k, renormalize=False)
    ids, w = torch.from_numpy(ids).cuda(), torch.from_numpy(w.astype(np.float32)).cuda()
    row = lambda start, stop: torch.arange(start, stop, device="cuda") * 7 % 1000
    logits = torch.empty(T, E, dtype=torch.float16, device="cuda")
    table, step = torch.from_numpy(x).cuda(), 1 << 26
    for at in range(0, T, step):
        logits[at:at + step] = table[row(at, min(at + step, T))]
    got_ids, got_w = ops.route_topk(logits, k, renormalize=False)
    for at in range(0, T, step):
        r = row(at, min(at + step, T))
        assert torch.equal(got_ids[at:at + step], ids[r])
        assert ((got_w[at:at + step] - w[r]).abs() <= RTOL * w[r]).all()
