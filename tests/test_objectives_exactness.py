"""The objectives over logits on the CPU: what happens at borders (clip bounds, infinite margins, NaN among the
operands), and what the engine says of their steps. (The device's kernels: test_gpu_objectives_exactness.py.)"""
import numpy as np
import pytest

from rustautograd_b200 import frontend as F


@pytest.fixture
def cpu(oracle):
    F.use(oracle, "cpu")
    return oracle


def run(fn, *args, **kw):
    args = tuple(F.tensor(a) for a in args)
    return F.compile(fn, args, validate="none", **kw)(*args)


def clipped_tokens(rng, n, v=8):
    """Logits, labels, old log-probabilities and advantages of tokens that are all clipped, and their terms' exact values for
    bounds 0.8 and 1.28: -1.28 A for ratios of about e, -0.8 A for ratios of about 1 / e."""
    x = rng.normal(size=(n, v)).astype("float32")
    lab = rng.integers(0, v, n).astype("int32")
    z = x.astype("f8")
    lp = z[np.arange(n), lab] - np.log(np.exp(z).sum(1))
    up = rng.random(n) < 0.5
    adv = (np.where(up, 1, -1) * rng.uniform(0.1, 3, n)).astype("float32")
    return x, lab, (lp + np.where(up, -1, 1)).astype("float32"), adv, -np.where(up, 1 + 0.28, 1 - 0.2) * adv.astype("f8")


def test_clip_bounds_are_not_rounded(cpu):
    # A clipped token's term is the bound times the advantage, rounded once: half a step, 2^-24 relatively.
    x, lab, old, adv, want = clipped_tokens(np.random.default_rng(1), 512)
    one = F.tensor(np.ones(512, "float32"))
    terms = run(lambda x: F.nn.policy_loss(x, F.tensor(lab), F.tensor(old), F.tensor(adv), one, clip_low=0.2, clip_high=0.28)[1], x).numpy()
    assert (np.abs(terms.astype("f8") - want) <= 2.0 ** -24 * (1 + 1e-6) * np.abs(want)).all()
