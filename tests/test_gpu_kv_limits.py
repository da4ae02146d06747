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
