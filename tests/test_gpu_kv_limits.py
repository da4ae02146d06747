"""GPU: the paged key-value cache at the ends of its types, its row ranges and its pages, against the 64-bit oracle."""
import numpy as np
import pytest

from oracle import kv_oracle as orc
from test_gpu_kv_cache import APART, check_attend, fill, rc, seeded, torch     # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu


def i32(torch, x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ probabilities
@pytest.mark.parametrize("dim,heads", [(64, 8), (128, 8), (128, 24), (256, 4)])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "4-bit values far apart"])
def test_attend_rounds_the_output_and_little_else(torch, rc, kind, dim, heads):
    """The error's root mean square beside that of the exact result rounded once to the output's type.  Probabilities held to
    2^-16 (bf16) or 2^-22 (fp16) of themselves and fp32 sums add less than a hundredth of it; probabilities rounded once to
    the type would add about a fifth.  (The squares add up: 2 % is an error of a fifth of the rounding's.)"""
    lens = [2000, 1777, 3001]
    apart = kind.startswith("4-bit")
    cache, truth, _ = fill(torch, rc, lens, 2, dim, 16, "mxfp4" if apart else kind, seed=dim + heads, exponents=APART["far apart"] if apart else None)
    q = torch.randn(len(lens), heads, dim, device="cuda").to(torch.float16 if kind == "fp16" else torch.bfloat16)
    scale = dim ** -0.5 * (0.05 if apart else 1.0)
    out = cache.attend(q, scale=scale)[0].double().cpu()
    want = torch.from_numpy(np.stack([orc.attend(q[b].double().cpu().numpy(), truth["k"][b], truth["v"][b], scale)[0] for b in range(len(lens))]))
    size = want.abs().amax(-1, keepdim=True) if apart else 1.0             # (a row's largest blocks decide)
    rms = lambda x: float((x / size).square().mean().sqrt())                # noqa: E731
    assert rms(out - want) <= 1.02 * rms(want.to(q.dtype).double() - want)


@pytest.mark.parametrize("lens", [[1], [300], [9000], [1, 0, 33, 700]])
@pytest.mark.parametrize("spread", [8.0e37, 2.0 ** -70], ids=["large", "small"])
def test_attend_over_bf16_values_near_the_ends_of_the_type(torch, rc, lens, spread):
    """Sums of values up to the type's largest stay finite, and tiny ones keep their digits, in one part and in many."""
    cache, truth, table = fill(torch, rc, lens, 2, 128, 16, "bf16", seed=sum(lens))
    v = (cache.v.float() * spread).clamp(-3.38e38, 3.38e38).bfloat16()
    cache.v.copy_(v)
    pages = lambda b, n: torch.from_numpy(table[b, :-(-n // 16)]).long().cuda()     # noqa: E731
    for b, n in enumerate(lens):
        truth["v"][b] = v[pages(b, n)].transpose(0, 1).reshape(2, -1, 128)[:, :n].double().cpu().numpy() if n else truth["v"][b]
    q = torch.randn(len(lens), 14, 128, device="cuda").bfloat16()
    got = cache.attend(q, weigh=True)
    check_attend(torch, cache, truth, q, lens, 128 ** -0.5, got, cache.weight, table)


def test_attend_over_bf16_values_that_are_all_the_largest(torch, rc):
    lens = [1, 40, 5000]
    cache, _, _ = fill(torch, rc, lens, 1, 64, 16, "bf16", seed=1)
    top = torch.finfo(torch.bfloat16).max
    cache.v.fill_(top)
    cache.v[..., ::2] = -top
    out, _ = cache.attend(torch.randn(3, 8, 64, device="cuda").bfloat16())
    # the exact answer is the value itself; fp32 sums are off by less than half a unit of bf16
    assert (out[..., 1::2] == top).all() and (out[..., ::2] == -top).all()


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("n", [1, 17, 600])
def test_attend_with_scores_near_the_lowest_number(torch, rc, kind, n):
    """Equal scores of -2.2e38 (finite in powers of two as well): the mean of the values."""
    cache, truth, table = fill(torch, rc, [n], 1, 64, 16, kind, seed=n)
    cache.k.fill_(0.0)
    cache.k[..., 0] = 2.0 ** 10
    q = torch.zeros(1, 4, 64, device="cuda", dtype=cache.k.dtype)
    q[..., 0] = -1.3046875
    scale = 2.0 ** 117                                     # -1.3046875 * 2^127 = -2.2198e38, times log2 e -3.2026e38
    out, log_sum = cache.attend(q, scale=scale, weigh=True)
    want = truth["v"][0][0].mean(0)
    size = np.abs(truth["v"][0][0]).mean(0)
    assert (np.abs(out[0].double().cpu().numpy() - want) <= 2.0 ** -7 * size).all()
    assert np.abs(log_sum.double().cpu().numpy() / (-1.3046875 * 2.0 ** 127) - 1).max() <= 2.0 ** -21
    t = np.arange(n)
    weight = cache.weight.cpu().numpy()[table[0, t // 16], 0, t % 16]
    assert np.abs(weight * n / 4 - 1).max() <= 2.0 ** -18


@pytest.mark.parametrize("dim,heads", [(64, 4), (128, 8), (128, 24), (256, 8)])
def test_attend_over_key_blocks_that_are_not_finite(torch, rc, dim, heads):
    """Scale byte 255 is NaN whatever the block's codes are: the scores, so all of the head's output, are NaN."""
    lens = [40, 40, 40]
    cache, _, table = fill(torch, rc, lens, 2, dim, 16, "mxfp4", seed=dim)
    for b, code in ((0, 0x77), (1, 0xff)):                 # 6 and -6 throughout the row
        cache.k[int(table[b, 1]), 1, 3] = code
        cache.k_scale[int(table[b, 1]), 1, 3, 1] = 255
    q = torch.randn(3, heads, dim, device="cuda").abs().bfloat16()
    out, log_sum = cache.attend(q)
    half = heads // 2
    assert torch.isnan(out[:2, half:]).all() and torch.isnan(log_sum[:2, half:]).all()
    assert torch.isfinite(out[:2, :half]).all() and torch.isfinite(out[2]).all() and torch.isfinite(log_sum[2]).all()


# ------------------------------------------------------------------ row ranges
STARTS = {"past the rows": ([0, 2, 9], [42, 22]), "past the rows at once": ([0, 100, 200], [44, 20]),
          "not from zero": ([1, 2, 4], [41, 22]), "from below zero": ([-3, 2, 4], [42, 22]),
          "falling": ([0, 3, 1], [40, 20]), "falling below zero": ([0, -2, 4], [40, 20])}


@pytest.mark.parametrize("what", list(STARTS))
@pytest.mark.parametrize("kind", ["bf16", "mxfp4"])
def test_append_of_bad_row_ranges_counts_what_it_stored(torch, rc, what, kind):
    """4 rows: those inside both the ranges and the rows are stored and counted, none where the ranges fall; check() tells."""
    starts, lens = STARTS[what]
    cache, _, table = fill(torch, rc, [40, 20], 1, 64, 16, kind, seed=3)
    rows = torch.randn(4, 1, 64, device="cuda").bfloat16()
    cache.append(rows, rows, i32(torch, starts))
    with pytest.raises(rc.CacheError, match="rows"):
        cache.check()
    assert cache.length.tolist() == lens and cache.seen.tolist() == lens
    # what was counted can be read back: the rows of the clamped ranges
    new = [n - m for n, m in zip(lens, (40, 20))]
    got = cache.read(i32(torch, np.cumsum([0] + new)), sum(new))[0].double().cpu().numpy()
    first = [min(max(s, 0), 4) for s in starts]
    want = np.concatenate([rows[first[b]:first[b] + new[b]].double().cpu().numpy() for b in range(2)])
    assert np.array_equal(got, want if kind == "bf16" else orc.values(*orc.quantise(want)))
    cache.check()


@pytest.mark.parametrize("starts", [[0, 2, 9], [1, 2, 4], [0, 3, 1], [-1, 2, 4]])
def test_read_of_bad_row_ranges_is_reported(torch, rc, starts):
    cache, truth, _ = fill(torch, rc, [40, 20], 1, 64, 16, "bf16", seed=3)
    k, _ = cache.read(i32(torch, starts), 4)
    assert torch.isfinite(k).all()
    with pytest.raises(rc.CacheError, match="rows"):
        cache.check()


def test_append_of_falling_ranges_over_many_sequences(torch, rc):
    """Ranges in no order over more sequences than one round of the search takes."""
    batch = 300
    cache, _, _ = fill(torch, rc, [5] * batch, 1, 64, 16, "bf16", seed=4)
    rng = np.random.default_rng(0)
    rows = torch.ones(200, 1, 64, device="cuda")
    for _ in range(5):
        cache.append(rows, rows, i32(torch, rng.integers(0, 201, batch + 1)))
        with pytest.raises(rc.CacheError, match="rows"):
            cache.check()
        assert cache.length.tolist() == [5] * batch and cache.seen.tolist() == [5] * batch
        assert torch.isfinite(cache.read(i32(torch, rng.integers(0, 201, batch + 1)), 200)[0]).all()
        with pytest.raises(rc.CacheError, match="rows"):
            cache.check()
