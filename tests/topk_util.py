"""Inputs of the tests of the operators for several experts per token, and the comparison with the oracle's bounds."""
import numpy as np

DTYPES = ("float32", "bfloat16", "float16")
FFNS = ("relu", "gated_gelu", "gated_silu")


def typed(torch, a, dtype):
    """(device tensor in dtype, its values in float64)."""
    t = torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda().to(getattr(torch, dtype))
    return t, t.double().cpu().numpy()


def assert_within(got, want, bound, what=""):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(got), nan, err_msg=f"{what}: NaN in other places")
    off = np.where(nan, 0.0, np.abs(got - want))
    over = off > np.where(nan, 1.0, bound)
    assert not over.any(), f"{what}: {over.sum()} of {off.size} beyond their bound, worst {np.max(off / np.where(nan, 1, bound)):.3g} times, first at {np.argwhere(over)[0]}"


def draw_experts(torch, rng, T, k, E, d, h, ffn, dtype):
    """dict of device tensors and, under "exact", the oracle's arrays."""
    x, xe = typed(torch, rng.standard_normal((T, d)), dtype)
    wi, wie = typed(torch, rng.standard_normal((E, h, d)) / np.sqrt(d), dtype)
    wo, woe = typed(torch, rng.standard_normal((E, d, h)) / np.sqrt(h), dtype)
    w1 = w1e = None
    if ffn != "relu":
        w1, w1e = typed(torch, rng.standard_normal((E, h, d)) / np.sqrt(d), dtype)
    ids = np.argsort(rng.random((T, E)) + 0.3 * rng.random(E), axis=1)[:, :k].astype(np.int32) if k <= E else rng.integers(0, E, (T, k)).astype(np.int32)
    weights = rng.random((T, k)).astype(np.float32)
    weights /= weights.sum(axis=1, keepdims=True)
    return dict(x=x, wi=wi, wo=wo, wi_1=w1, ids=torch.from_numpy(ids).cuda(), weights=torch.from_numpy(weights).cuda(), ffn=ffn,
                exact=dict(x=xe, wi=wie, wo=woe, wi_1=w1e, ids=ids, weights=weights, ffn=ffn, dtype=dtype))


def draw_lora(torch, rng, T, d, n, r, L, dtype, order):
    x, xe = typed(torch, rng.standard_normal((T, d)), dtype)
    w, we = typed(torch, rng.standard_normal((n, d)) / np.sqrt(d), dtype)
    a, ae = typed(torch, rng.standard_normal((L, r, d)) / np.sqrt(d), dtype)
    b, be = typed(torch, rng.standard_normal((L, n, r)) / np.sqrt(r), dtype)
    adapter = rng.integers(-1, L + 1, T).astype(np.int32)  # none (-1), beyond the last (L)
    if order == "requests":
        adapter = np.repeat(rng.integers(-1, L, T), rng.integers(1, 60, T))[:T].astype(np.int32)
    scale = rng.uniform(0.5, 2.0, L).astype(np.float32)
    return dict(x=x, w=w, a=a, b=b, adapter=torch.from_numpy(adapter).cuda(), scale=torch.from_numpy(scale).cuda(),
                exact=dict(x=xe, w=we, a=ae, b=be, adapter=adapter, scale=scale, dtype=dtype))
