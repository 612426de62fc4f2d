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


# Pairs of which one answer holds a token that its logits ban: margins of +inf (the rejected one), of -inf (the chosen one) and a
# finite one. By definition the first costs 0 with smoothing 0, the second with smoothing 1; otherwise both cost infinity.
def infinite_margins(dtype, v=6, t=3):
    x = np.random.default_rng(2).normal(size=(6, t, v)).astype(dtype)
    lab = np.zeros((6, t), "int32")
    x[3, 1, 0] = x[1, 2, 0] = -np.inf  # pairs are (0, 3), (1, 4), (2, 5)
    z = x.astype("f8")
    with np.errstate(divide="ignore"):
        lp = z[..., 0] - np.log(np.exp(z).sum(-1))
    return x, lab, np.ones((6, t), dtype), np.zeros(6, dtype), lp.sum(1)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("smoothing", [0.0, 0.25, 1.0])
def test_infinite_margins(cpu, smoothing, dtype):
    x, lab, w, ref, seq = infinite_margins(dtype)
    for pairs, signs in (([0, 2], (np.inf, 0)), ([1, 2], (-np.inf, 0)), ([0, 1, 2], (np.inf, -np.inf, 0))):
        rows = pairs + [p + 3 for p in pairs]

        def f(x):
            out = F.nn.preference_loss(x, F.tensor(lab[rows]), F.tensor(w[rows]), F.tensor(ref[rows]), 0.5, smoothing)
            return out[0], out[1]
        (loss, margins), g = run(F.value_and_grad(f, has_aux=True), x[rows])
        check_infinite_margins(loss.numpy(), margins.numpy(), g.numpy(), signs, seq, smoothing, 20 * np.finfo(dtype).eps)


def check_infinite_margins(loss, margins, g, signs, seq, smoothing, off):
    n = len(signs)
    assert np.array_equal(margins[:-1], signs[:-1])
    h = 0.5 * (seq[2] - seq[5])
    terms = [np.inf if s and not (s > 0 and smoothing == 0 or s < 0 and smoothing == 1) else 0 for s in signs]
    terms[-1] = (1 - smoothing) * np.logaddexp(0, -h) + smoothing * np.logaddexp(0, h)
    want = sum(terms) / n
    # Two sums of three log-probabilities, each off by `off` at most, times beta (the loss's slope is below 1). For a row of v logits
    # within 12 of each other that is u (additions + 2.3 * 12 + 4 for the exponentials + 4 log s + 2 |lp|): 40 u for 6 logits.
    assert loss == want if np.isinf(want) else abs(loss - want) <= 0.5 * 6 * off, (loss, want)
    assert np.isfinite(g).all()
    for k, s in enumerate(signs[:-1]):  # the slope of a side that costs nothing is 0, of one that costs infinity +-beta / n
        still = s > 0 and smoothing == 0 or s < 0 and smoothing == 1
        assert (not g[[k, n + k]].any()) == still


def test_answers_both_out_of_reach_have_no_margin(cpu):
    x, lab, w, ref, _ = infinite_margins("float32")
    rows = [1, 2, 3, 5]  # the banned answers against each other, and a pair of others
    loss, margins, _ = run(lambda x: F.nn.preference_loss(x, F.tensor(lab[rows]), F.tensor(w[rows]), F.tensor(ref[rows])), x[rows])
    assert np.isnan(loss.numpy()) and np.isnan(margins.numpy()[0]) and np.isfinite(margins.numpy()[1])


def nan_operands(rng, v, dtype):
    """Operands of a policy loss of 8 rows with kl, of which rows 1 to 6 hold a NaN: in old_logp (with advantages of both signs), in the
    advantage (with ratios above and below the bounds), in the weight and in the reference."""
    x, lab = rng.normal(size=(8, v)).astype(dtype), rng.integers(0, v, 8).astype("int32")
    z = x.astype("f8")
    lp = z[np.arange(8), lab] - np.log(np.exp(z).sum(1))
    ops = {"old": lp - np.array([0, 0, 0, 1, -1, 0, 0, 0.0]), "adv": np.array([1.0, 1, -1, 1, -1, 1, 1, -1]), "w": np.ones(8), "ref": lp + 0.1}
    bad = {k: a.copy() for k, a in ops.items()}
    bad["old"][1:3] = bad["adv"][3:5] = bad["w"][5] = bad["ref"][6] = np.nan
    return x, lab, *({k: a.astype(dtype) for k, a in o.items()} for o in (ops, bad))


def check_nan_operands(good, bad, kl):
    rows = [1, 2, 3, 4, 5] + ([6] if kl else [])
    fine = [r for r in range(8) if r not in rows]
    (loss, terms, logp, g), (_, good_terms, good_logp, good_g) = bad, good
    assert np.isnan(loss) and np.isnan(terms[rows]).all() and np.isnan(g[rows]).all()
    assert np.array_equal(logp, good_logp) and np.array_equal(terms[fine], good_terms[fine]) and np.array_equal(g[fine], good_g[fine])
    assert np.isfinite(good_g).all()


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("kl", [0.0, 0.1])
def test_nan_among_the_operands_reaches_the_gradient(cpu, kl, dtype):
    x, lab, good, bad = nan_operands(np.random.default_rng(3), 9, dtype)

    def policy(o):
        def f(x):
            out = F.nn.policy_loss(x, F.tensor(lab), F.tensor(o["old"]), F.tensor(o["adv"]), F.tensor(o["w"]), F.tensor(o["ref"]) if kl else None, kl=kl)
            return out[0], out[1:]
        (loss, (terms, logp)), g = run(F.value_and_grad(f, has_aux=True), x)
        return loss.numpy(), terms.numpy(), logp.numpy(), g.numpy()
    check_nan_operands(policy(good), policy(bad), kl)


def test_no_advantage_costs_nothing_at_any_ratio(cpu):
    # A = 0 and a ratio past the largest number: the bound counts, and the term and its gradient are 0.
    x, lab, one = np.zeros((1, 4), "float64"), F.tensor(np.zeros(1, "int32")), F.tensor(np.ones(1))
    loss, g = run(F.value_and_grad(lambda x: F.nn.policy_loss(x, lab, one * -1000.0, one * 0.0, one)[0]), x)
    assert loss.numpy() == 0 and not g.numpy().any()


def test_sizes_past_31_bits_are_refused_without_positions_too(product):
    # Sequences without positions have no rows, but pairs: as many as would wrap the workspace's size around. Before any CUDA call.
    import ctypes

    import rustautograd_b200
    from test_objectives import Logits, Preference
    lib = ctypes.CDLL(rustautograd_b200.LIBRARY)
    lib.rgc_last_error.restype = ctypes.c_char_p
    lib.rgc_preference_workspace.restype = ctypes.c_size_t
    fake = ctypes.c_void_p(1 << 20)  # never dereferenced
    for outer, inner in ((1 << 62, 0), (1 << 31, 0), (0, 1 << 31)):
        for dtype in (0, 1, 256, 257):
            x, p = Logits(1 << 20, outer, inner, 8, 8, 8, dtype), Preference(fake, fake, 0.1, 0.0)
            rc = lib.rgc_preference_loss(ctypes.byref(x), fake, ctypes.byref(p), fake, None, None, None, fake, ctypes.c_size_t(0), None)
            assert rc == -1 and b"too many rows" in lib.rgc_last_error(), (outer, inner, lib.rgc_last_error())
    for n, t in ((1 << 62, 0), (1 << 31, 0), (1 << 16, 1 << 15), (2, 1 << 62)):
        assert lib.rgc_preference_workspace(ctypes.c_int64(n), ctypes.c_int64(t), 1) == 0
    assert lib.rgc_preference_workspace(ctypes.c_int64(2), ctypes.c_int64(0), 1) > 0


def test_step_costs(oracle):
    # Operands and kept results once each, by their own types, whatever the slots' sizes (a row of one logit is as large as its term).
    F.use(oracle, "cuda-plan")
    for v in (1, 2, 50):
        for es, dtype in ((4, "float32"), (8, "float64")):
            n, t, k = 6, 5, 3
            x, row, seq = (F.tensor(np.zeros(s, dtype)) for s in ((n, t, v), (n, t), (n,)))
            lab, index, teacher = F.zeros((n, t), "int32"), F.zeros((n, t, k), "int32"), F.tensor(np.zeros((n, t, k), dtype))

            def cost(f):
                (got,) = [c for c in F.compile(f, (x,), validate="none")._n.step_costs() if c[0] == "objective"]
                return got[1:]
            rows, logits = n * t, n * t * v
            cases = [(lambda x: F.nn.policy_loss(x, lab, row, row, row)[0], 4 * rows + 3 * rows * es + es, 1),
                     (lambda x: F.nn.preference_loss(x, lab, row, seq)[0], 4 * rows + (rows + n) * es + es, 2),
                     (lambda x: F.nn.distillation_loss(x, index, teacher, row)[0], 4 * rows * k + (rows * k + rows) * es + es, 1)]
            for f, small, reads in cases:
                assert cost(f) == (3.0 * logits, logits * es + small)
                assert cost(F.value_and_grad(f)) == (6.0 * logits, logits * es * (reads + 1) + small)
            terms = lambda x: F.nn.policy_loss(x, lab, row, row, row)[:2]
            assert cost(terms) == (3.0 * logits, logits * es + 4 * rows + 3 * rows * es + es + rows * es)
            assert cost(lambda x: F.nn.token_log_prob(x, lab)) == (3.0 * logits, logits * es + 4 * rows + rows * es)


def test_plan_summary_names_the_slots_of_every_result(oracle):
    import json
    F.use(oracle, "cuda-plan")
    x, lab, w = F.zeros((3, 7)), F.zeros((3,), "int32"), F.ones((3,))
    (step,) = json.loads(F.compile(F.value_and_grad(lambda x: F.nn.policy_loss(x, lab, w, w, w)[0]), (x,), validate="none")._n.plan_summary())
    assert len(step["out"]) == 2 and max(step["out"]) < 100 and len(set(step["out"] + step["in"])) == len(step["out"]) + len(set(step["in"]))


def label_cases():
    """(what, function of the logits, whether the engine's check refuses its labels) for logits (4, 3, 6): an index outside the vocabulary
    at a position that counts, and at positions that do not (weight 0, an absent teacher entry)."""
    rng = np.random.default_rng(5)
    row, seq = F.tensor(rng.random((4, 3)).astype("float32")), F.tensor(np.zeros(4, "float32"))
    lab, index, w = rng.integers(0, 6, (4, 3)).astype("int32"), rng.integers(0, 6, (4, 3, 2)).astype("int32"), np.ones((4, 3), "float32")
    teacher = rng.normal(size=(4, 3, 2)).astype("float32")
    for bad in (None, -100, -1, 6):
        for weight in (1.0, -1.0, 0.0):
            l, i, ww, t = lab.copy(), index.copy(), w.copy(), teacher.copy()
            if bad is not None:
                l[2, 1] = i[2, 1, 1] = bad
            ww[2, 1] = weight
            refused = bad is not None and weight != 0
            l, i, ww = F.tensor(l), F.tensor(i), F.tensor(ww)
            yield ("policy", bad, weight), lambda x, l=l, ww=ww: F.nn.policy_loss(x, l, row, row, ww)[0], refused
            yield ("preference", bad, weight), lambda x, l=l, ww=ww: F.nn.preference_loss(x, l, ww, seq)[0], refused
            yield ("distillation", bad, weight), lambda x, i=i, ww=ww: F.nn.distillation_loss(x, i, F.tensor(teacher), ww)[0], refused
            yield ("logp", bad, weight), lambda x, l=l: F.nn.token_log_prob(x, l).sum(), bad is not None
            t[2, 1, 1] = -np.inf
            yield ("absent", bad, weight), lambda x, i=i, ww=ww, t=t: F.nn.distillation_loss(x, i, F.tensor(t), ww)[0], False


def check_labels(device):
    x = F.tensor(np.random.default_rng(6).normal(size=(4, 3, 6)).astype("float32"))
    for what, f, refused in label_cases():
        report = F.compile(lambda x: F.value_and_grad(f)(x), (x,), validate="standard", device=device).report
        codes = [d["code"] for d in report["diagnostics"]]
        assert codes.count("INDEX_OUT_OF_RANGE") == refused and (report["status"] == "validation_failed") == refused, (what, report)


@pytest.mark.parametrize("device", ["cpu", "cuda-plan"])
def test_labels_that_count_are_checked(oracle, device):
    F.use(oracle, device)
    check_labels(device)
