"""GPU: RansAttention, a decoder layer's attention block with entropy-coded projections and a paged cache, against the same
block computed in 64 bits token by token from the decoded weights and the keys and values that the cache holds.

Tolerance (norm of the difference over the norm): x, q, out and y are rounded to bf16 (2^-8 each at most, and the errors of
q and k move the scores by less than their relative error times the largest score); 3e-2 covers the sum with scores below 4.
"""
import numpy as np
import pytest

from oracle import kv_oracle as orc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(cuda_ok):
    import torch as t
    import rans_b200
    rans_b200.load()
    return t


def _linear(rows, cols, seed):
    import rans_model as rm
    w = np.random.default_rng(seed).standard_normal((rows, cols)) / cols ** 0.5
    codes, step = rm.ecsq_rtn(w, 4.25)
    return rm.RansLinear(rm.EncodedMatrix.encode(codes, step, R=8, C=256))


@pytest.mark.parametrize("kind,batch", [("bf16", 1), ("mxfp4", 1), ("fp16", 3), ("mxfp4", 3)])
def test_layer_against_64_bits(torch, kind, batch):
    import rans_cache as rc
    import rans_model as rm
    hidden, heads, kv_heads, dim, steps = 256, 4, 2, 64, 40
    proj = [_linear(heads * dim, hidden, 1), _linear(kv_heads * dim, hidden, 2), _linear(kv_heads * dim, hidden, 3), _linear(hidden, heads * dim, 4)]
    dense = [p.weight_bf16().double().cpu().numpy() for p in proj]
    cache = rc.KVCache(pages=4 * batch, page=16, kv_heads=kv_heads, dim=dim, batch=batch, max_tokens=64, kind=kind)
    layer = rm.RansAttention(*proj, cache, heads)
    torch.manual_seed(3)
    x = torch.randn(steps, batch, hidden, device="cuda").bfloat16()
    for i in range(steps):
        y = layer(x[i])
        assert y.shape == (batch, hidden) and y.dtype == x.dtype
        total = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * (i + 1)
        k, v = (r.double().cpu().numpy().reshape(batch, i + 1, kv_heads, dim) for r in cache.read(total, batch * (i + 1)))
        for b in range(batch):
            xb = x[i, b].double().cpu().numpy()
            q = (dense[0] @ xb).reshape(heads, dim)
            out = orc.attend(q, k[b].transpose(1, 0, 2), v[b].transpose(1, 0, 2), dim ** -0.5)[0]
            want = dense[3] @ out.reshape(-1)
            got = y[b].double().cpu().numpy()
            assert np.linalg.norm(got - want) <= 3e-2 * np.linalg.norm(want)
    # the newest key is what the projection gives, rounded to the cache's type
    want = (dense[1] @ x[-1, 0].double().cpu().numpy()).reshape(kv_heads, dim)
    if kind == "mxfp4":
        want = orc.values(*orc.quantise(want))
    assert np.linalg.norm(k[0, -1] - want) <= (0.2 if kind == "mxfp4" else 2e-2) * np.linalg.norm(want)
    cache.check()


def test_layer_keeps_its_budget(torch):
    import rans_cache as rc
    import rans_model as rm
    hidden, heads, kv_heads, dim = 256, 4, 2, 64
    proj = [_linear(heads * dim, hidden, 1), _linear(kv_heads * dim, hidden, 2), _linear(kv_heads * dim, hidden, 3), _linear(hidden, heads * dim, 4)]
    cache = rc.KVCache(pages=8, page=16, kv_heads=kv_heads, dim=dim, batch=2, max_tokens=64, kind="mxfp4")
    calls = []

    def rotate(q, k, seen):
        calls.append(seen.tolist())
        return q, k

    layer = rm.RansAttention(*proj, cache, heads, rotate=rotate, budget=24, recent=8, slack=4)
    for i in range(60):
        y = layer(torch.randn(2, hidden, device="cuda").bfloat16())
        assert torch.isfinite(y).all()
        length = cache.length.tolist()
        assert length[0] == length[1] <= 28 and (i < 28 or length[0] >= 24)
        assert calls[-1] == [i, i]
        newest = cache.position[cache.table[:, : -(-length[0] // 16)].long()].transpose(1, 2).reshape(2, kv_heads, -1)[..., :length[0]]
        for t in range(max(0, i - 7), i + 1):
            assert (newest == t).any(-1).all()              # the newest eight are always there
    cache.check()
    assert cache.free_pages == 8 - 2 * 2


def test_layer_refusals(torch):
    import rans_cache as rc
    import rans_model as rm
    hidden, heads, kv_heads, dim = 256, 4, 2, 64
    q, k, v, o = _linear(heads * dim, hidden, 1), _linear(kv_heads * dim, hidden, 2), _linear(kv_heads * dim, hidden, 3), _linear(hidden, heads * dim, 4)
    cache = rc.KVCache(pages=4, page=16, kv_heads=kv_heads, dim=dim, batch=1, max_tokens=64)
    for args, more in (((q, k, v, o, cache, 8), {}), ((q, q, v, o, cache, heads), {}), ((q, k, v, o, cache, heads), dict(budget=0)),
                       ((q, k, v, o, cache, heads), dict(budget=4, recent=5)), ((q, k, v, o, cache, heads), dict(budget=4, slack=-1))):
        with pytest.raises(ValueError):
            rm.RansAttention(*args, **more)
    layer = rm.RansAttention(q, k, v, o, cache, heads)
    with pytest.raises(ValueError):
        layer(torch.zeros(2, hidden, device="cuda"))
